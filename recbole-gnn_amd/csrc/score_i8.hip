// score_i8.hip — rows in 8 bits with a scale each, and scores from them.
//
//   codes[r, j] = rint(x[r, j] / s_r) in [-127, 127],  s_r = fl32(max |x[r, :]| / 127)
//   S[b, j] = su[b] si[j] sum_k qu[b, k] qi[j, k]
//
// The sums run on the integer matrix cores (v_mfma_i32_32x32x32_i8: 16 bytes of a row per lane and operand, K is order-free, both
// operands are K-contiguous) and are exact in 32 bits up to K = 131 071.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lds_dma.h"
#include "vocab_common.h"

namespace rbg {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- rows to 8 bits ------------------------------------------------------------------------------------------------------

// The quotient is the IEEE one (no reciprocal): a code is the nearest whole number to x / s, so whoever restates the operator gets the
// same codes.
struct RowScale {
    float s;    // what the row is divided by; 0: its codes are 0
    float out;  // what is stored
};
__device__ __forceinline__ RowScale row_scale(float m) {  // m: the largest magnitude, infinite for a row that is not finite
    const float s = m / 127.f;
    if (m == INFINITY) return {0.f, NAN};
    return s >= 1.17549435e-38f ? RowScale{s, s} : RowScale{0.f, 0.f};
}
__device__ __forceinline__ uint32_t code_of(float x, float s) { return (uint32_t)(int)fminf(fmaxf(rintf(x / s), -127.f), 127.f) & 255u; }
__device__ __forceinline__ float magnitude(float x) {  // NaN counts as infinite
    const float v = fabsf(x);
    return v < INFINITY ? v : INFINITY;
}

// G lanes per row hold NC vectors each, read once.  Bound by the reads and the quotients: 4 096 x 8 192 bf16, 101 MB in 33 us = 3.1 TB/s;
// 4 096 x 64 fp32 in 5 us, a launch.
template <class T, int G, int NC>
__global__ __launch_bounds__(256) void quantize_kernel(const T *__restrict__ x, int64_t ldx, int64_t n, int K, int8_t *__restrict__ codes,
                                                       int ldc, float *__restrict__ scale) {
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int sub = threadIdx.x % G;
    const bool on = row < n;
    const T *p = x + (on ? row : 0) * ldx;
    Vec<T, E> v[NC];
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        const int c = (u * G + sub) * E;
        if (c + E <= K) {
            v[u] = load_any<T, E>(p + c);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[u].v[e] = c + e < K ? p[c + e] : from_f32<T>(0.f);
        }
    }
#pragma unroll
    for (int u = 0; u < NC; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, magnitude(to_f32(v[u].v[e])));
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if constexpr (G > 64) {
        __shared__ float red[4];
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    if (!on) return;
    const RowScale s = row_scale(m);
    if (sub == 0) scale[row] = s.out;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        const int c = (u * G + sub) * E;
        if (c >= ldc) break;
        Vec<uint32_t, E / 4> w;
#pragma unroll
        for (int k = 0; k < E / 4; ++k) {
            w.v[k] = 0;
            if (s.s != 0.f)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.v[k] |= code_of(to_f32(v[u].v[4 * k + e]), s.s) << (8 * e);
        }
        *reinterpret_cast<Vec<uint32_t, E / 4> *>(codes + row * ldc + c) = w;
    }
}

// Longer rows (of more than 16 384 values in 32 bits, 32 768 in 16): one workgroup per row, which it reads twice and element by element.  512 rows
// of 16 448 fp32 in 36 us where 16 384 take 11, of 32 832 bf16 in 70 where 32 768 take 19: correct at any length, not made for speed.
template <class T>
__global__ __launch_bounds__(256) void quantize_long_kernel(const T *__restrict__ x, int64_t ldx, int64_t K, int8_t *__restrict__ codes, int64_t ldc,
                                                           float *__restrict__ scale) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const T *p = x + row * ldx;
    float m = 0.f;
    for (int64_t j = threadIdx.x; j < K; j += 256) m = fmaxf(m, magnitude(to_f32(p[j])));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    const RowScale s = row_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    if (threadIdx.x == 0) scale[row] = s.out;
    uint32_t *out = reinterpret_cast<uint32_t *>(codes + row * ldc);
    for (int64_t c = threadIdx.x; c < ldc / 4; c += 256) {
        uint32_t w = 0;
        if (s.s != 0.f)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * c + e < K) w |= code_of(to_f32(p[4 * c + e]), s.s) << (8 * e);
        out[c] = w;
    }
}

template <class T>
static int launch_quantize_rows(const T *x, int64_t ldx, int64_t n, int64_t K, int8_t *codes, int64_t ldc, float *scale, hipStream_t s) {
    constexpr int E = 16 / (int)sizeof(T);
    auto blocks = [&](int per) { return dim3((unsigned)((n + per - 1) / per)); };
    if (ldc <= 32 * E) hipLaunchKernelGGL((quantize_kernel<T, 32, 1>), blocks(8), dim3(256), 0, s, x, ldx, n, (int)K, codes, (int)ldc, scale);
    else if (ldc <= 128 * E) hipLaunchKernelGGL((quantize_kernel<T, 64, 2>), blocks(4), dim3(256), 0, s, x, ldx, n, (int)K, codes, (int)ldc, scale);
    else if (ldc <= 1024 * E) hipLaunchKernelGGL((quantize_kernel<T, 256, 4>), blocks(1), dim3(256), 0, s, x, ldx, n, (int)K, codes, (int)ldc, scale);
    else if (ldc <= 4096 * E) hipLaunchKernelGGL((quantize_kernel<T, 256, 16>), blocks(1), dim3(256), 0, s, x, ldx, n, (int)K, codes, (int)ldc, scale);
    else hipLaunchKernelGGL((quantize_long_kernel<T>), blocks(1), dim3(256), 0, s, x, ldx, K, codes, ldc, scale);
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

template <class T>
static int launch_quantize(const T *x, int64_t ldx, int64_t n, int64_t K, int8_t *codes, int64_t ldc, float *scale, hipStream_t s) {
    for (int64_t r0 = 0; r0 < n; r0 += kRowsPerLaunch)
        if (int rc = launch_quantize_rows<T>(x + r0 * ldx, ldx, std::min(kRowsPerLaunch, n - r0), K, codes + r0 * ldc, ldc, scale + r0, s)) return rc;
    return RBG_OK;
}

// ---- the product ---------------------------------------------------------------------------------------------------------

struct ScoreArgs {
    const int8_t *qu, *qi;
    int64_t ldu, ldi;
    const float *su, *si;
    int64_t B, n;
    int kc;        // chunks of 16 bytes in a row of codes
    void *S;
    int64_t lds;
    const void *u;  // rows that a kernel makes the codes of for itself (then ldu counts their elements)
    int K;
};

// acc su si in 32 bits.  acc < 2^31, so acc su may pass the type's end, where the score need not, for su > 2^96 alone: such a scale goes in two
// parts (powers of two: the same roundings).  FAR: some scale of the wave's users is one.  (Two parts for every user: 110 -> 118 us at
// 4 096 x 40 982 x 128 bf16; chosen by wave 110.)
constexpr float kFarScale = 0x1p96f;
template <bool FAR>
__device__ __forceinline__ float score_of(int acc, float su, float si) {
    if constexpr (!FAR) return (float)acc * su * si;
    asm volatile("" : "+v"(su));  // (or the parts of every row's scale are made ahead and kept in registers)
    const bool far = su > kFarScale;
    return (float)acc * (far ? su * 0x1p-64f : su) * si * (far ? 0x1p64f : 1.f);
}
template <int N>
__device__ __forceinline__ bool any_far(const float (&su)[N]) {  // on any lane of the wave
    bool far = false;
#pragma unroll
    for (int i = 0; i < N; ++i) far |= su[i] > kFarScale;
    return __ballot(far) != 0;
}
template <class F>
__device__ __forceinline__ void by_far(bool far, F f) {
    if (far) f(std::true_type{});
    else f(std::false_type{});
}

// The codes of a row that two lanes share, h the even 16-byte chunks or the odd ones, from its K values; its scale.
template <class TU, int KS>
__device__ __forceinline__ float own_codes(const TU *x, int K, int h, i32x4 (&codes)[KS]) {
    constexpr int E = 16 / (int)sizeof(TU);
    TU v[KS][16];
    float mag = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        const int c = 16 * (2 * k + h);
        if (c + 16 <= K) {
#pragma unroll
            for (int q = 0; q < 16 / E; ++q) {
                const Vec<TU, E> t = load_any<TU, E>(x + c + q * E);
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][q * E + e] = t.v[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[k][e] = c + e < K ? x[c + e] : from_f32<TU>(0.f);
        }
    }
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) mag = fmaxf(mag, magnitude(to_f32(v[k][e])));
    const RowScale s = row_scale(fmaxf(mag, __shfl_xor(mag, 32)));
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w = 0;
            if (s.s != 0.f)
#pragma unroll
                for (int e = 0; e < 4; ++e) w |= code_of(to_f32(v[k][4 * q + e]), s.s) << (8 * e);
            codes[k][q] = (int)w;
        }
    return s.out;
}

// Short rows (K <= 32 KS): the scores are written at the rate of the stores and everything else has to hide behind them.  A workgroup
// keeps 32 users' codes in registers and walks item tiles of TB bytes of scores per row: each wave multiplies 32 items' codes at a time,
// taken straight from the table, and puts its scores into LDS, every row shifted by its distance from a 128-byte line.  Whole lines then
// leave as 16-byte stores of consecutive lanes (1 KB of a row per wave and store at TB = 2048), whatever the row stride; what a tile leaves
// over of a row's last line (less than LINE scores) moves to the front of the row for the next tile.  4 096 x 40 982 x 64 into fp32:
// 672 MB in 141 to 147 us behind itself, 138 to 140 a call among other work = 4.6 to 4.9 TB/s; bare whole-line stores into rows of that
// stride take 131 to 138.
template <class TO, class TU, int KS, int TB>
__global__ __launch_bounds__(256, TB == 2048 ? 2 : 4) void score_i8_short_kernel(const ScoreArgs a, int tiles_per_walk) {
    constexpr int E = 16 / (int)sizeof(TO), TILE = TB / (int)sizeof(TO), LINE = 128 / (int)sizeof(TO), PITCH = TILE + LINE;
    __shared__ alignas(16) TO buf[32 * PITCH];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 31, h = lane >> 5;
    const int64_t b0 = (int64_t)blockIdx.y * 32;
    const int64_t t0 = (int64_t)blockIdx.x * tiles_per_walk, t1 = min(t0 + tiles_per_walk, (a.n + TILE - 1) / TILE);
    const int64_t js = t0 * TILE, je = min(t1 * TILE, a.n);
    TO *S = (TO *)a.S + b0 * a.lds;
    const int rows = (int)min<int64_t>(32, a.B - b0);
    // row r starts (off0 + r step) mod LINE scores behind a line, and so does every tile of it (TILE is whole lines)
    const unsigned off0 = (unsigned)((reinterpret_cast<uintptr_t>(S) / sizeof(TO)) % LINE), step = (unsigned)(a.lds % LINE);
    i32x4 fu[KS];
    float own_su = 0.f;
    if constexpr (std::is_void_v<TU>) {
        const i32x4 *pu = reinterpret_cast<const i32x4 *>(a.qu + min(b0 + m, a.B - 1) * a.ldu) + h;
#pragma unroll
        for (int k = 0; k < KS; ++k) fu[k] = pu[2 * k];
    } else {
        own_su = own_codes<TU, KS>((const TU *)a.u + min(b0 + m, a.B - 1) * a.ldu, a.K, h, fu);
    }
    float su[16];
    unsigned at[16];  // where this lane's item of sub-tile 0 goes, for each of its 16 rows
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const unsigned row = (r & 3) + 8 * (r >> 2) + 4 * h;
        if constexpr (std::is_void_v<TU>) su[r] = a.su[min<int64_t>(b0 + row, a.B - 1)];
        else su[r] = __shfl(own_su, row);
        at[r] = row * PITCH + ((off0 + row * step) & (LINE - 1)) + w * 32 + m;
    }
    i32x4 fi[KS];
    float si;
    auto fetch = [&](int64_t sub) {  // sub-tiles of 128 items, 32 for each wave
        const int64_t j = min(sub * 128 + w * 32 + m, a.n - 1);
        const i32x4 *p = reinterpret_cast<const i32x4 *>(a.qi + j * a.ldi);
#pragma unroll
        for (int k = 0; k < KS; ++k) fi[k] = p[min(2 * k + h, a.kc - 1)];  // behind the row's end the users' codes are zero
        si = a.si[j];
    };
    // the scores of a row's last piece of a line: LINE of them from (threadIdx.x / (LINE / KEEP)), KEEP for each thread
    constexpr int KEEP = 32 * LINE / 256;
    const unsigned krow = threadIdx.x / (LINE / KEEP), kcol = threadIdx.x % (LINE / KEEP) * KEEP;
    const bool far = any_far(su);  // (the same rows in all four waves)
    fetch(t0 * (TILE / 128));
    for (int64_t t = t0; t < t1; ++t) {
#pragma unroll
        for (int u = 0; u < TILE / 128; ++u) {
            i32x16 acc = {};
#pragma unroll
            for (int k = 0; k < KS; ++k) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fu[k], fi[k], acc, 0, 0, 0);
            const float sj = si;
            if (u + 1 < TILE / 128 || t + 1 < t1) fetch(t * (TILE / 128) + u + 1);
#pragma unroll
            for (int r = 0; r < 16; ++r) buf[at[r] + u * 128] = from_f32<TO>(score_of<false>(acc[r], su[r], sj));
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) buf[at[r] + u * 128] = from_f32<TO>(score_of<true>(acc[r], su[r], sj));
            }
        }
        __syncthreads();
        const bool first = t == t0, last = t + 1 == t1;
        constexpr int L = TILE / E;  // lanes that store a row's lines of one tile
#pragma unroll
        for (int q = 0; q < 32 / (256 / L); ++q) {
            const unsigned row = q * (256 / L) + threadIdx.x / L;
            const int64_t line = t * TILE - (int)((off0 + row * step) & (LINE - 1));  // the column at the row's front in LDS
            if ((int)row >= rows) continue;
            TO *to = S + row * a.lds + line;
            const TO *from = &buf[row * PITCH];
            const int lo = first ? (int)(js - line) : 0, hi = last ? (int)(je - line) : TILE;
            for (int c = threadIdx.x % L * E; c < hi; c += TILE) {
                if (c >= lo && c + E <= hi) {
                    __builtin_nontemporal_store(*reinterpret_cast<const i32x4 *>(from + c), reinterpret_cast<i32x4 *>(to + c));
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (c + e >= lo && c + e < hi) to[c + e] = from[c + e];
                }
            }
        }
        const Vec<TO, KEEP> keep = *reinterpret_cast<const Vec<TO, KEEP> *>(&buf[krow * PITCH + TILE + kcol]);
        __syncthreads();
        const unsigned ph = (off0 + krow * step) & (LINE - 1);
#pragma unroll
        for (int e = 0; e < KEEP; ++e)
            if (kcol + e < ph) buf[krow * PITCH + kcol + e] = keep.v[e];
    }
}

template <class TO, class TU, int KS, int TB>
static int launch_short(const ScoreArgs &a, int64_t resident, hipStream_t s) {
    constexpr int TILE = TB / (int)sizeof(TO);
    const int64_t tiles = (a.n + TILE - 1) / TILE, panels = (a.B + 31) / 32;
    // once round the workgroups that fit the chip, and walks of at least two tiles (their ends store pieces of lines)
    int64_t walks = std::max<int64_t>(1, std::min<int64_t>((tiles + 1) / 2, resident / panels));
    const int per = (int)((tiles + walks - 1) / walks);
    walks = (tiles + per - 1) / per;
    for (int64_t y0 = 0; y0 < panels; y0 += 65535) {  // (a grid's y dimension ends at 65 535)
        ScoreArgs p = a;
        if constexpr (std::is_void_v<TU>) p.qu += y0 * 32 * a.ldu, p.su += y0 * 32;
        else p.u = (const TU *)a.u + y0 * 32 * a.ldu;
        p.B -= y0 * 32;
        p.S = (TO *)a.S + y0 * 32 * a.lds;
        hipLaunchKernelGGL((score_i8_short_kernel<TO, TU, KS, TB>), dim3((unsigned)walks, (unsigned)std::min<int64_t>(65535, panels - y0)), dim3(256), 0, s, p, per);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

// 2 KB of a row per tile where that leaves every CU work; else 512 bytes: four times the workgroups.
template <class TO, class TU, int KS>
static int launch_short(const ScoreArgs &a, hipStream_t s) {
    const int64_t panels = (a.B + 31) / 32, lines = (a.n * (int64_t)sizeof(TO) + 2047) / 2048;
    return panels * lines >= 1024 ? launch_short<TO, TU, KS, 2048>(a, 512, s) : launch_short<TO, TU, KS, 512>(a, 1024, s);
}

// Few users (B <= 16 UT), or too few scores for the tiles below: 16 x 16 tiles straight from the rows, no staging: a wave's load touches
// 64 bytes of each of 16 items' rows.  A workgroup has 16 UT users (blockIdx.y) and KW of its waves share 16 IT items and split K (their
// sums meet in LDS); the other 4 / KW have items of their own.
// TU other than void: the users' rows are a.u, of that type and at most kOwnCodes values in all; every workgroup makes their codes for
// itself in LDS, and the call is one launch.  (At 8 192 values that takes longer than everything else: 357 us for one user of 131 072
// items x 8 192, 198 with the codes made first.)
// Bound by reading the items: one user of 40 982 x 128 in 4.8 us, most of it the launch, of 131 072 x 8 192 in 198 = 5.4 TB/s.
constexpr int kOwnCodes = 2048;

template <class TO, class TU, int UT, int IT, int KW>
__global__ __launch_bounds__(256) void score_i8_few_kernel(const ScoreArgs a) {
    constexpr int U = 4;  // steps of 64 bytes in flight
    constexpr bool OWN = !std::is_void_v<TU>;
    // a row of codes: K rounded up to 64, and 16 more bytes so that the 16 rows of a fragment spread over the banks
    __shared__ alignas(16) int8_t own[OWN ? kOwnCodes + 16 * 80 : 16];
    __shared__ float own_su[16];
    const int pitch = (a.kc + 3) / 4 * 64 + 16;
    // (w as a scalar: it decides how many steps there are, and a matrix instruction that a mask of lanes alone guards runs all the same)
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
    const int64_t j0 = ((int64_t)blockIdx.x * (4 / KW) + w / KW) * (16 * IT), b0 = (int64_t)blockIdx.y * (16 * UT);
    const i32x4 *pu[UT], *pi[IT];
#pragma unroll
    for (int x = 0; x < UT; ++x) {
        if constexpr (OWN) pu[x] = reinterpret_cast<const i32x4 *>(own + min<int>(m, (int)a.B - 1) * pitch);
        else pu[x] = reinterpret_cast<const i32x4 *>(a.qu + min<int64_t>(b0 + 16 * x + m, a.B - 1) * a.ldu);
    }
#pragma unroll
    for (int y = 0; y < IT; ++y) pi[y] = reinterpret_cast<const i32x4 *>(a.qi + min<int64_t>(j0 + 16 * y + m, a.n - 1) * a.ldi);
    if constexpr (OWN) {
        static_assert(UT == 1);
        for (int r = w; r < (int)a.B; r += 4) {  // a wave per row
            const TU *p = (const TU *)a.u + r * a.ldu;
            float mag = 0.f;
            for (int c = lane; c < a.K; c += 64) mag = fmaxf(mag, magnitude(to_f32(p[c])));
            const RowScale s = row_scale(wave_max(mag));
            for (int c = lane; c < pitch - 16; c += 64)
                own[r * pitch + c] = c < a.K && s.s != 0.f ? (int8_t)code_of(to_f32(p[c]), s.s) : (int8_t)0;
            if (lane == 0) own_su[r] = s.out;
        }
        __syncthreads();
    }
    const float *su = OWN ? own_su : a.su;
    const int steps = (a.kc + 3) / 4, per = (steps + KW - 1) / KW;
    const int s0 = w % KW * per, s1 = min(s0 + per, steps);
    i32x4 acc[UT][IT] = {};
    for (int t = s0; t < s1; t += U) {
        i32x4 fu[U][UT], fi[U][IT];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < s1) {
                const int c = 4 * (t + u) + g;  // behind the row's end the users' codes are zero, up to a multiple of 128 bytes
#pragma unroll
                for (int x = 0; x < UT; ++x) fu[u][x] = pu[x][c];
#pragma unroll
                for (int y = 0; y < IT; ++y) fi[u][y] = pi[y][min(c, a.kc - 1)];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < s1)
#pragma unroll
                for (int x = 0; x < UT; ++x)
#pragma unroll
                    for (int y = 0; y < IT; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fu[u][x], fi[u][y], acc[x][y], 0, 0, 0);
    }
    if constexpr (KW > 1) {
        __shared__ i32x4 part[4][UT * IT][64];
#pragma unroll
        for (int x = 0; x < UT; ++x)
#pragma unroll
            for (int y = 0; y < IT; ++y) part[w][x * IT + y][lane] = acc[x][y];
        __syncthreads();
        if (w % KW) return;
#pragma unroll
        for (int q = 1; q < KW; ++q)
#pragma unroll
            for (int x = 0; x < UT; ++x)
#pragma unroll
                for (int y = 0; y < IT; ++y) acc[x][y] += part[w + q][x * IT + y][lane];
    }
    TO *S = (TO *)a.S;
    float sb[UT * 4];
#pragma unroll
    for (int i = 0; i < UT * 4; ++i) sb[i] = su[min<int64_t>(b0 + 16 * (i / 4) + 4 * g + i % 4, a.B - 1)];
    by_far(any_far(sb), [&](auto far) {
#pragma unroll
        for (int y = 0; y < IT; ++y) {
            const int64_t j = j0 + 16 * y + m;
            if (j >= a.n) continue;
            const float si = a.si[j];
#pragma unroll
            for (int x = 0; x < UT; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t b = b0 + 16 * x + 4 * g + r;
                    if (b < a.B) S[b * a.lds + j] = from_f32<TO>(score_of<decltype(far)::value>(acc[x][y][r], sb[4 * x + r], si));
                }
        }
    });
}

template <class TO, class TU, int UT>
static int launch_few(const ScoreArgs &a, hipStream_t s) {
    const unsigned gy = (unsigned)((a.B + 16 * UT - 1) / (16 * UT));  // (a few)
    auto blocks = [&](int per) { return dim3((unsigned)((a.n + per - 1) / per), gy); };
    if constexpr (UT > 1) {  // (at most 8 192 items and groups of users: see launch_score_items)
        hipLaunchKernelGGL((score_i8_few_kernel<TO, TU, UT, 1, 4>), blocks(16), dim3(256), 0, s, a);
    } else if (a.kc >= 64) {  // 1 KB and more of a row: four waves share it
        // more items per wave read the users' codes less often, but leave fewer waves (16, 32 and 64 items, us: 16 x 32 768 x 2 048 20, 18, 19;
        // 1 x 65 536 x 1 024 25, 22, 20; 1 x 65 536 x 2 048 47, 47, 36; 1 x 131 072 x 2 048 82, 79, 68; 16 x 131 072 x 2 048 70, 59, 56)
        if (a.n * gy <= 16 * 2048) hipLaunchKernelGGL((score_i8_few_kernel<TO, TU, UT, 1, 4>), blocks(16), dim3(256), 0, s, a);
        else if (a.n * gy <= 64 * 1024 || a.kc < 128) hipLaunchKernelGGL((score_i8_few_kernel<TO, TU, UT, 2, 4>), blocks(32), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((score_i8_few_kernel<TO, TU, UT, 4, 4>), blocks(64), dim3(256), 0, s, a);
    } else {  // (1 x 131 072 x 960: 27, and 32 with the row over four waves; 16 x 131 072 x 512: 19.6 and 18.4)
        hipLaunchKernelGGL((score_i8_few_kernel<TO, TU, UT, 2, 1>), blocks(128), dim3(256), 0, s, a);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

// Large products: a 64 W x 64 W tile of S per workgroup (W = 4, or 2 where that leaves CUs without one), one wave per SIMD with a quarter
// of it (W x W accumulators of 32 x 32), K in steps of 128 bytes through two LDS stages that LDS-DMA fills.  A step is four slices of
// 32 bytes: while a slice's W W products run, the next slice's 2 W fragments are read; the barrier that hands over a stage
// stands in front of the last slice's products, so that the next stage's first fragments arrive under them and the old stage's
// refill goes out between them.  Chunk c of row r lies at slot c ^ (r / 2 % 8): any 16 rows' fragments cover the 64 banks.
// Bound by the power the matrix cores draw: the clock falls to between 1.55 and 1.9 GHz, box by box, and 4 096 x 16 384 x 8 192 takes 490
// to 550 us = 2.0 to 2.2 P operations per second, which is also what a plain library product of 8-bit integers of 8 192 cubed reaches.
template <class TO, int W>
__global__ __launch_bounds__(256, W == 4 ? 1 : 2) void score_i8_tile_kernel(const ScoreArgs a, int gx, int gy) {
    constexpr int SIDE = 64 * W, STAGE = 2 * SIDE * 128;
    __shared__ alignas(16) int8_t lds[2 * STAGE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, h = lane >> 5;
    // workgroup i runs on XCD i % 8: give each XCD a run of tiles, four user tiles deep, so that its L2 sees few rows at a time
    const int total = gx * gy, q8 = total / 8, r8 = total % 8, xcd = blockIdx.x % 8;
    const int t = xcd * q8 + min(xcd, r8) + blockIdx.x / 8;
    const int group = t / (4 * gx), y0 = group * 4, deep = min(4, gy - y0), in = t - group * 4 * gx;
    // (the quotients come out of vector registers: told to be the same in all lanes, the operands' bases below are scalar)
    const int64_t b0 = (int64_t)__builtin_amdgcn_readfirstlane(y0 + in % deep) * SIDE, j0 = (int64_t)__builtin_amdgcn_readfirstlane(in / deep) * SIDE;
    const int steps = (a.kc + 7) / 8;
    // this wave fills rows 16 W w .. 16 W w + 16 W - 1 of both operands, eight rows per request
    const int sc = (lane & 7) ^ (lane >> 4);  // its chunk in rows of an even request; ^ 4 in those of an odd one
    const int8_t *bu = a.qu + b0 * a.ldu, *bi = a.qi + j0 * a.ldi;
    uint32_t ou[2 * W], oi[2 * W];
#pragma unroll
    for (int q = 0; q < 2 * W; ++q) {
        const int r = 16 * W * w + 8 * q + (lane >> 3);
        ou[q] = (uint32_t)(min<int64_t>(r, a.B - 1 - b0) * a.ldu) + 16 * (sc ^ (q & 1) * 4);
        oi[q] = (uint32_t)(min<int64_t>(r, a.n - 1 - j0) * a.ldi) + 16 * (sc ^ (q & 1) * 4);
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t *)lds;
    // behind a row's end: the users' codes are zero there, the items' row ends at its last whole chunk
    const int last = a.kc - 1 - 8 * (steps - 1);
    const uint32_t back[2] = {16u * (uint32_t)max(0, sc - last), 16u * (uint32_t)max(0, (sc ^ 4) - last)};
    auto fill = [&](int step, auto part) {  // a W-th of a stage: two requests for either operand
        const unsigned to = lds0 + (step & 1) * STAGE + w * (W * 2048);
        const uint32_t at = (uint32_t)step * 128;
        const bool end = step + 1 == steps;
        constexpr int q = 2 * decltype(part)::value;
        lds_dma16(bu, ou[q] + at, to + q * 1024);
        lds_dma16(bu, ou[q + 1] + at, to + q * 1024 + 1024);
        lds_dma16(bi, oi[q] + at - (end ? back[0] : 0u), to + STAGE / 2 + q * 1024);
        lds_dma16(bi, oi[q + 1] + at - (end ? back[1] : 0u), to + STAGE / 2 + q * 1024 + 1024);
    };
    auto each = [](auto f) {
        f(std::integral_constant<int, 0>{});
        f(std::integral_constant<int, 1>{});
        if constexpr (W == 4) f(std::integral_constant<int, 2>{}), f(std::integral_constant<int, 3>{});
    };
    i32x16 acc[W][W] = {};
    i32x4 f0[2 * W], f1[2 * W];
    const int wu = (w >> 1) * (32 * W), wi = (w & 1) * (32 * W);
    auto read = [&](i32x4(&to)[2 * W], int step, int k) {
        const int8_t *from = lds + (step & 1) * STAGE + (((2 * k + h) ^ ((m >> 1) & 7)) * 16);
#pragma unroll
        for (int x = 0; x < W; ++x) to[x] = *reinterpret_cast<const i32x4 *>(from + (wu + 32 * x + m) * 128);
#pragma unroll
        for (int y = 0; y < W; ++y) to[W + y] = *reinterpret_cast<const i32x4 *>(from + STAGE / 2 + (wi + 32 * y + m) * 128);
    };
    auto multiply = [&](const i32x4(&g)[2 * W], auto part) {
        constexpr int x = decltype(part)::value;
#pragma unroll
        for (int y = 0; y < W; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(g[x], g[W + y], acc[x][y], 0, 0, 0);
    };
    auto slice = [&](const i32x4(&g)[2 * W], i32x4(&next)[2 * W], int step, int k) {  // read (step, k) under the products of g
        read(next, step, k);
        __builtin_amdgcn_sched_barrier(0);
        each([&](auto x) { multiply(g, x); });
        __builtin_amdgcn_sched_barrier(0);
    };
    float wave_su[(W + 1) / 2];  // of the wave's users, one or two for each lane
#pragma unroll
    for (int i = 0; i < (W + 1) / 2; ++i) wave_su[i] = a.su[min<int64_t>(b0 + wu + 64 * i + lane, a.B - 1)];
    const bool far_users = any_far(wave_su);
    each([&](auto q) { fill(0, q); });
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 1) each([&](auto q) { fill(1, q); });
    read(f0, 0, 0);
    for (int st = 0; st < steps; ++st) {
        slice(f0, f1, st, 1);
        slice(f1, f0, st, 2);
        slice(f0, f1, st, 3);
        // The next stage is filled, and nobody reads this one any more: its refill goes out between the products.  (After the last
        // step the fragments read here are of no use, but they are read all the same: no wait then depends on a branch.)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        read(f0, st + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
        const bool more = st + 2 < steps;
        each([&](auto x) {
            multiply(f1, x);
            __builtin_amdgcn_sched_barrier(0);
            if (more) fill(st + 2, x);
        });
    }
    __syncthreads();
    // the wave's tile through its quarter of the LDS, a strip of 32 users at a time, and out in rows
    constexpr int COLS = 32 * W, E = 16 / (int)sizeof(TO), L = COLS / E;
    TO *strip = reinterpret_cast<TO *>(lds + w * (STAGE / 2));
    TO *S = (TO *)a.S;
    const bool inside = j0 + SIDE <= a.n;  // (else the items end in this tile)
    float si[W];
#pragma unroll
    for (int y = 0; y < W; ++y) si[y] = a.si[min<int64_t>(j0 + wi + 32 * y + m, a.n - 1)];
#pragma unroll
    for (int x = 0; x < W; ++x) {
        const int64_t bx = b0 + wu + 32 * x;
        by_far(far_users, [&](auto far) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = (r & 3) + 8 * (r >> 2) + 4 * h;
                const float su = a.su[min<int64_t>(bx + row, a.B - 1)];
#pragma unroll
                for (int y = 0; y < W; ++y) strip[row * COLS + 32 * y + m] = from_f32<TO>(score_of<decltype(far)::value>(acc[x][y][r], su, si[y]));
            }
        });
        if (inside) {
#pragma unroll
            for (int q = 0; q < 32 * L / 64; ++q) {
                const int row = q * (64 / L) + lane / L, c = lane % L * E;
                if (bx + row < a.B) store_any(S + (bx + row) * a.lds + j0 + wi + c, *reinterpret_cast<const Vec<TO, E> *>(strip + row * COLS + c));
            }
        } else {
#pragma unroll 4
            for (int q = 0; q < 32 * COLS / 64; ++q) {
                const int row = q / (COLS / 64), c = q % (COLS / 64) * 64 + lane;
                if (bx + row < a.B && j0 + wi + c < a.n) S[(bx + row) * a.lds + j0 + wi + c] = strip[row * COLS + c];
            }
        }
    }
}

template <class TO, int W>
static int launch_tiles(const ScoreArgs &a, hipStream_t s) {
    constexpr int64_t SIDE = 64 * W;
    const int64_t gx = (a.n + SIDE - 1) / SIDE, all = (a.B + SIDE - 1) / SIDE, most = std::max<int64_t>(1, ((int64_t)1 << 23) / gx);
    for (int64_t y0 = 0; y0 < all; y0 += most) {  // (a grid holds fewer than 2^32 threads)
        ScoreArgs p = a;
        p.qu += y0 * SIDE * a.ldu, p.su += y0 * SIDE, p.B -= y0 * SIDE;
        p.S = (TO *)a.S + y0 * SIDE * a.lds;
        const int64_t gy = std::min(most, all - y0);
        p.B = std::min(p.B, gy * SIDE);
        hipLaunchKernelGGL((score_i8_tile_kernel<TO, W>), dim3((unsigned)(gx * gy)), dim3(256), 0, s, p, (int)gx, (int)gy);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

// TU other than void: rows of users to be made into codes on the way, few ones or short ones.
template <class TO, class TU>
static int launch_score_items(const ScoreArgs &a, hipStream_t s) {
    if (a.B <= 16) return launch_few<TO, TU, 1>(a, s);
    if (a.kc <= 4) return launch_short<TO, TU, 2>(a, s);
    if (a.kc <= 8 || !std::is_void_v<TU>) return launch_short<TO, TU, 4>(a, s);
    if (a.kc <= 16 && a.B * a.n * (int64_t)sizeof(TO) >= 128 << 20) return launch_short<TO, void, 8, 2048>(a, 512, s);  // (4096 x 40 001 x 256: 197 us, 237 in tiles; 100 x 100 001 x 200: 40 and 22)
    const int64_t wide = ((a.n + 255) / 256) * ((a.B + 255) / 256), small = ((a.n + 127) / 128) * ((a.B + 127) / 128);
    // 64 x 16 tiles with K over four waves, many times the workgroups (300 x 300 x 8 192: 31 us against 51; 1 000 x 1 000 x 1 024: 19 against 16)
    if (small <= 32 && a.kc >= 128) return launch_few<TO, void, 4>(a, s);
    // Rounds of 256 x 256 tiles (one per CU) against 128 x 128 ones, whose products cost about 1.37 times as much but which waste less of the
    // last round and of the edges.  (128 and 256 wide, us: 2 000 x 2 000 x 4 096 39 and 74; 3 000 x 3 000 x 2 048 45 and 53; 4 096 x 16 384 x
    // 2 048 199 and 188.  Short rows are the stores' and the small tiles' again, which the rule leaves: 4 096 x 8 192 x 1 024 60 and 70.)
    return (wide + 255) / 256 * 4 <= 1.37 * small / 256 ? launch_tiles<TO, 4>(a, s) : launch_tiles<TO, 2>(a, s);
}

template <class TO, class TU>
static int launch_score(const ScoreArgs &a, hipStream_t s) {
    constexpr int64_t kItemsPerLaunch = 1 << 24;  // (a grid holds fewer than 2^32 threads per dimension)
    for (int64_t j0 = 0; j0 < a.n; j0 += kItemsPerLaunch) {
        ScoreArgs p = a;
        p.qi += j0 * a.ldi, p.si += j0, p.S = (TO *)a.S + j0, p.n = std::min(kItemsPerLaunch, a.n - j0);
        if (int rc = launch_score_items<TO, TU>(p, s)) return rc;
    }
    return RBG_OK;
}

// Bytes between the rows of codes that a call makes for itself.
static int64_t own_stride(int64_t K) { return (K + 127) / 128 * 128; }

// Whether the product's workgroups make the users' codes themselves, in one launch.  Up to 16 users: kOwnCodes.  Rows of up to 128 values of
// more users, against codes made first: 100 x 1 000 x 100 fp16 9.8 us a call and 12.7, 4 096 x 40 982 x 128 bf16 112 and 118, x 64 fp32 140 and
// 141; but x 128 fp32 148 and 144, 600 x 5 000 x 127 fp32 13.3 and 13.0: every workgroup reads its 32 rows before its first product.
static bool makes_codes(int64_t B, int64_t n, int64_t K, int size) {
    if (B <= 16) return B * K <= kOwnCodes;
    return K <= 128 && (K * size <= 256 || B * n <= 1 << 21);
}

constexpr int64_t kMaxStride = 1 << 23;  // 32-bit offsets inside a tile
constexpr int64_t kMaxK = 131071;  // 128 x 128 x K < 2^31

// What both product entries ask of the items and the scores.
static int check_score(int64_t B, const int8_t *qi, int64_t ldi, const float *si, int64_t n, int64_t K, const void *S, int64_t lds, int out_dtype) {
    if (!elem_ok(out_dtype)) return fail(RBG_EINVAL, "out_dtype = %d", out_dtype);
    if (B < 0 || n < 0 || K <= 0 || ldi < K || lds < n)
        return fail(RBG_ESHAPE, "B = %lld, n = %lld, K = %lld, ldi = %lld, lds = %lld", (long long)B, (long long)n, (long long)K, (long long)ldi, (long long)lds);
    if (ldi % 16) return fail(RBG_EINVAL, "ldi = %lld is not a multiple of 16", (long long)ldi);
    if (K > kMaxK) return fail(RBG_EUNSUPPORTED, "K = %lld: sums of more than 131071 products may pass 32 bits", (long long)K);
    if (n > 0x7fffffffll || B > 0x7fffffffll) return fail(RBG_EUNSUPPORTED, "rows beyond 2^31");
    if (ldi > kMaxStride) return fail(RBG_EUNSUPPORTED, "ldi = %lld: at most 2^23 bytes between rows of codes", (long long)ldi);
    if (B && n && (!qi || !si || !S)) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(qi) || reinterpret_cast<uintptr_t>(S) % elem_size(out_dtype)) return fail(RBG_EINVAL, "codes need 16-byte alignment, scores that of their type");
    return RBG_OK;
}

}  // namespace rbg

using namespace rbg;

extern "C" {

int rbg_quantize_rows_i8(const void *x, int64_t ldx, int dtype, int64_t n, int64_t K, int8_t *codes, int64_t ldc, float *scale, void *stream) {
    clear_error();
    if (!elem_ok(dtype)) return fail(RBG_EINVAL, "dtype = %d", dtype);
    if (n < 0 || K <= 0 || ldx < K || ldc < K) return fail(RBG_ESHAPE, "n = %lld, K = %lld, ldx = %lld, ldc = %lld", (long long)n, (long long)K, (long long)ldx, (long long)ldc);
    if (ldc % 16) return fail(RBG_EINVAL, "ldc = %lld is not a multiple of 16", (long long)ldc);
    if (n > 0x7fffffffll) return fail(RBG_EUNSUPPORTED, "rows beyond 2^31");
    if (n == 0) return RBG_OK;
    if (!x || !codes || !scale) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(codes) || reinterpret_cast<uintptr_t>(x) % elem_size(dtype)) return fail(RBG_EINVAL, "codes need 16-byte alignment, rows that of their type");
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        return launch_quantize<E>((const E *)x, ldx, n, K, codes, ldc, scale, (hipStream_t)stream);
    });
}

int rbg_score_i8(const int8_t *qu, int64_t ldu, const float *su, int64_t B, const int8_t *qi, int64_t ldi, const float *si, int64_t n,
                 int64_t K, void *S, int64_t lds, int out_dtype, void *stream) {
    clear_error();
    if (int rc = check_score(B, qi, ldi, si, n, K, S, lds, out_dtype)) return rc;
    if (ldu < K) return fail(RBG_ESHAPE, "K = %lld, ldu = %lld", (long long)K, (long long)ldu);
    if (ldu % 128) return fail(RBG_EINVAL, "ldu = %lld is not a multiple of 128", (long long)ldu);
    if (ldu > kMaxStride) return fail(RBG_EUNSUPPORTED, "ldu = %lld: at most 2^23 bytes between rows of codes", (long long)ldu);
    if (B == 0 || n == 0) return RBG_OK;
    if (!qu || !su) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(qu)) return fail(RBG_EINVAL, "codes need 16-byte alignment");
    const ScoreArgs a{qu, qi, ldu, ldi, su, si, B, n, (int)((K + 15) / 16), S, lds, nullptr, (int)K};
    return with_elem(out_dtype, [&](auto t) { return launch_score<decltype(t), void>(a, (hipStream_t)stream); });
}

int rbg_score_rows_i8_workspace(int64_t B, int64_t K, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(RBG_EINVAL, "bytes is NULL");
    if (B < 0 || K <= 0) return fail(RBG_ESHAPE, "B = %lld, K = %lld", (long long)B, (long long)K);
    const int64_t ldc = own_stride(K);
    *bytes = B * ldc + (4 * B + 15) / 16 * 16;
    return RBG_OK;
}

int rbg_score_rows_i8(const void *u, int64_t ldu, int dtype, int64_t B, const int8_t *qi, int64_t ldi, const float *si, int64_t n, int64_t K,
                      void *S, int64_t lds, int out_dtype, void *workspace, void *stream) {
    clear_error();
    if (!elem_ok(dtype)) return fail(RBG_EINVAL, "dtype = %d", dtype);
    if (int rc = check_score(B, qi, ldi, si, n, K, S, lds, out_dtype)) return rc;
    if (ldu < K) return fail(RBG_ESHAPE, "K = %lld, ldu = %lld", (long long)K, (long long)ldu);
    if (B == 0 || n == 0) return RBG_OK;
    if (!u || !workspace) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(workspace) || reinterpret_cast<uintptr_t>(u) % elem_size(dtype)) return fail(RBG_EINVAL, "workspace is not 16-byte aligned, or rows not to their type");
    const int64_t ldc = own_stride(K);
    int8_t *qu = (int8_t *)workspace;
    float *su = (float *)(qu + B * ldc);
    if (makes_codes(B, n, K, elem_size(dtype))) {
        const ScoreArgs a{nullptr, qi, ldu, ldi, nullptr, si, B, n, (int)((K + 15) / 16), S, lds, u, (int)K};
        return with_elem(out_dtype, [&](auto o) {
            return with_elem(dtype, [&](auto t) { return launch_score<decltype(o), decltype(t)>(a, (hipStream_t)stream); });
        });
    }
    if (int rc = rbg_quantize_rows_i8(u, ldu, dtype, B, K, qu, ldc, su, stream)) return rc;
    return rbg_score_i8(qu, ldc, su, B, qi, ldi, si, n, K, S, lds, out_dtype, stream);
}

}  // extern "C"
