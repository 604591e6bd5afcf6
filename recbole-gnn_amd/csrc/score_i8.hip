// score_i8.hip — rows in 8 bits with a scale each, and scores from them.
//
//   codes[r, j] = rint(x[r, j] / s_r) in [-127, 127],  s_r = fl32(max |x[r, :]| / 127)
//   S[b, j] = su[b] si[j] sum_k qu[b, k] qi[j, k]
//
// The sums run on the integer matrix cores (v_mfma_i32_32x32x32_i8: 16 bytes of a row per lane and operand, K is order-free, both
// operands are K-contiguous) and are exact in 32 bits up to K = 131 071.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "vocab_common.h"

namespace rbg {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- rows to 8 bits ------------------------------------------------------------------------------------------------------

// One workgroup per row.  The quotient is the IEEE one (no reciprocal): a code is the nearest whole number to x / s, so whoever
// restates the operator gets the same codes.
template <class T, int TH>
__global__ __launch_bounds__(TH) void quantize_kernel(const T *__restrict__ x, int64_t ldx, int64_t K, int8_t *__restrict__ codes, int64_t ldc,
                                                      float *__restrict__ scale) {
    __shared__ float red[TH / kWave];
    const int64_t row = blockIdx.x;
    const T *p = x + row * ldx;
    float m = 0.f;
    bool odd = false;  // an infinity or NaN
    for (int64_t j = threadIdx.x; j < K; j += TH) {
        const float v = fabsf(to_f32(p[j]));
        odd |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    m = wave_max(odd ? INFINITY : m);
    if constexpr (TH > kWave) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int i = 1; i < TH / kWave; ++i) m = fmaxf(m, red[i]);
    }
    float s = m / 127.f;
    const bool zero = !(s >= 1.17549435e-38f) || m == INFINITY;
    if (threadIdx.x == 0) scale[row] = m == INFINITY ? NAN : zero ? 0.f : s;
    uint32_t *out = reinterpret_cast<uint32_t *>(codes + row * ldc);
    for (int64_t c = threadIdx.x; c < ldc / 4; c += TH) {
        uint32_t w = 0;
        if (!zero)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t j = 4 * c + e;
                if (j < K) {
                    const float q = fminf(fmaxf(rintf(to_f32(p[j]) / s), -127.f), 127.f);
                    w |= ((uint32_t)(int)q & 255u) << (8 * e);
                }
            }
        out[c] = w;
    }
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
};

// A 128 x 128 tile of S per workgroup of four waves (64 x 64 each: 2 x 2 tiles of 32 x 32); K in steps of 128 bytes, both
// operands' steps staged in LDS (rows of 128 bytes; 16-byte chunk c of row r at slot c ^ (r & 7), so that the 32 rows a
// fragment read touches spread over the banks), the next step in flight in registers.
template <class TO>
__global__ __launch_bounds__(256) void score_i8_kernel(const ScoreArgs a) {
    __shared__ i32x4 lu[128 * 8], li[128 * 8];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t b0 = (int64_t)blockIdx.y * 128, j0 = (int64_t)blockIdx.x * 128;
    const int steps = (a.kc + 7) / 8;
    // this thread stages chunk (tid & 7) of rows tid / 8 + 32 q
    const int sc = threadIdx.x & 7, sr = threadIdx.x >> 3;
    const i32x4 *pu[4], *pi[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        pu[q] = reinterpret_cast<const i32x4 *>(a.qu + min(b0 + sr + 32 * q, a.B - 1) * a.ldu);
        pi[q] = reinterpret_cast<const i32x4 *>(a.qi + min(j0 + sr + 32 * q, a.n - 1) * a.ldi);
    }
    i32x4 ru[4], ri[4];
    auto fetch = [&](int t) {
        const int c = t * 8 + sc;
        const int ci = min(c, a.kc - 1);  // behind the row's end the users' codes are zero
#pragma unroll
        for (int q = 0; q < 4; ++q) ru[q] = pu[q][c], ri[q] = pi[q][ci];
    };
    i32x16 acc[2][2] = {};
    fetch(0);
    const int m = lane & 31, h = lane >> 5, wu = (w >> 1) * 64, wi = (w & 1) * 64;
    for (int t = 0; t < steps; ++t) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = sr + 32 * q;
            lu[r * 8 + (sc ^ (r & 7))] = ru[q];
            li[r * 8 + (sc ^ (r & 7))] = ri[q];
        }
        __syncthreads();
        if (t + 1 < steps) fetch(t + 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            i32x4 fu[2], fi[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int r = 32 * q + m, c = (2 * k + h) ^ (r & 7);
                fu[q] = lu[(wu + r) * 8 + c];
                fi[q] = li[(wi + r) * 8 + c];
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fu[x], fi[y], acc[x][y], 0, 0, 0);
        }
    }
    TO *S = (TO *)a.S;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const int64_t j = j0 + wi + 32 * y + m;
        if (j >= a.n) continue;
        const float si = a.si[j];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t b = b0 + wu + 32 * x + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (b < a.B) S[b * a.lds + j] = from_f32<TO>((float)acc[x][y][r] * a.su[b] * si);
            }
    }
}

template <class TO>
static int launch_score(const ScoreArgs &a, hipStream_t s) {
    const int64_t gy = (a.B + 127) / 128;
    for (int64_t y0 = 0; y0 < gy; y0 += 65535) {  // (a grid's y dimension ends at 65 535)
        ScoreArgs p = a;
        p.qu += y0 * 128 * a.ldu, p.su += y0 * 128, p.B -= y0 * 128;
        p.S = (TO *)a.S + y0 * 128 * a.lds;
        const unsigned rows = (unsigned)std::min<int64_t>(65535, gy - y0);
        hipLaunchKernelGGL((score_i8_kernel<TO>), dim3((unsigned)((a.n + 127) / 128), rows), dim3(256), 0, s, p);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

constexpr int64_t kMaxK = 131071;  // 128 x 128 x K < 2^31

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
        if (K <= 512) hipLaunchKernelGGL((quantize_kernel<E, 64>), dim3((unsigned)n), dim3(64), 0, (hipStream_t)stream, (const E *)x, ldx, K, codes, ldc, scale);
        else hipLaunchKernelGGL((quantize_kernel<E, 256>), dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, (const E *)x, ldx, K, codes, ldc, scale);
        RBG_HIP(hipGetLastError());
        return (int)RBG_OK;
    });
}

int rbg_score_i8(const int8_t *qu, int64_t ldu, const float *su, int64_t B, const int8_t *qi, int64_t ldi, const float *si, int64_t n,
                 int64_t K, void *S, int64_t lds, int out_dtype, void *stream) {
    clear_error();
    if (!elem_ok(out_dtype)) return fail(RBG_EINVAL, "out_dtype = %d", out_dtype);
    if (B < 0 || n < 0 || K <= 0 || ldu < K || ldi < K || lds < n)
        return fail(RBG_ESHAPE, "B = %lld, n = %lld, K = %lld, ldu = %lld, ldi = %lld, lds = %lld", (long long)B, (long long)n, (long long)K, (long long)ldu, (long long)ldi, (long long)lds);
    if (ldu % 128 || ldi % 16) return fail(RBG_EINVAL, "ldu = %lld is not a multiple of 128, or ldi = %lld of 16", (long long)ldu, (long long)ldi);
    if (K > kMaxK) return fail(RBG_EUNSUPPORTED, "K = %lld: sums of more than 131071 products may pass 32 bits", (long long)K);
    if (n > 0x7fffffffll || B > 0x7fffffffll) return fail(RBG_EUNSUPPORTED, "rows beyond 2^31");
    if (B == 0 || n == 0) return RBG_OK;
    if (!qu || !su || !qi || !si || !S) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(qu) || !on_16(qi) || reinterpret_cast<uintptr_t>(S) % elem_size(out_dtype))
        return fail(RBG_EINVAL, "codes need 16-byte alignment, scores that of their type");
    const ScoreArgs a{qu, qi, ldu, ldi, su, si, B, n, (int)((K + 15) / 16), S, lds};
    return with_elem(out_dtype, [&](auto t) { return launch_score<decltype(t)>(a, (hipStream_t)stream); });
}

}  // extern "C"
