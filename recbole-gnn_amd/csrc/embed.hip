// embed.hip — rows of a table looked up by id with a scale, and the table's gradient by sorted ids.
//
//   out[i] = s T[id_i]            dT[v] = s sum_{i : id_i = v, ascending i} G[i]
//
// The lookup is a gather: 8 bytes of id, a row read, a row written.
// The gradient sorts the places by id (stably: equal ids keep their order) and then sums runs.  A lane-group of d / (16 bytes)
// lanes walks a chunk of consecutive sorted places and writes every row whose run lies inside the chunk; a run that crosses a
// chunk's border leaves 32-bit partial sums, one for the chunk's first run and one for its last, which a second launch adds
// in chunk order.  No float atomics: the order of every sum is decided by the sizes alone.  The rows nothing refers to are
// zeroed in the same launch by workgroups of their own, which find them by bisection in the sorted ids, so that every
// row of the gradient is written once.
//
// The sort: up to kRankMax places, a place's rank is counted outright — the number of (id, place) pairs in front of it — from the
// ids staged in LDS: N^2 compares, 64 to an instruction, in one launch.  Above, least-significant-digit radix passes of
// up to nine bits: to kMoveMax places one launch each, which counts the next pass's digits as it goes (and one launch for the first
// pass's); beyond, three each (digit counts per tile, their prefix per digit, a stable scatter).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "vocab_common.h"

namespace rbg {

// ---- lookup --------------------------------------------------------------------------------------------------------------

// The lane-groups below cover a row of d elements with vectors of VEC; the last vector of a row ends where the row ends and overlaps the one
// in front of it (both hold the same values), so that rows of any width and start move 16 bytes at a time.
template <int VEC>
__device__ __forceinline__ int vector_at(int c, int d) { return min(c, d - VEC); }

// G lanes per row, R rows of a lane-group in flight (ids, then rows, then stores).  Bound by memory: 65 536 rows of 2 KB (bf16, d = 1 024) out of
// 131 072 in 47 us, 268 MB of rows read and written at 5.7 TB/s; 32 rows of 128 bytes in 2 us, which is a launch.
template <class T, int VEC, int G>
__global__ __launch_bounds__(256) void lookup_kernel(const T *__restrict__ table, int64_t ldt, int64_t n_rows, const int64_t *__restrict__ ids,
                                                     int64_t n, int d, float scale, T *__restrict__ out, int64_t ldo) {
    constexpr int R = 4;
    const int sub = threadIdx.x % G;
    const int64_t i0 = ((int64_t)blockIdx.x * (256 / G) + threadIdx.x / G) * R;
    if (i0 >= n) return;
    int64_t id[R];
#pragma unroll
    for (int r = 0; r < R; ++r) id[r] = i0 + r < n ? ids[i0 + r] : -1;
    for (int c0 = sub * VEC; c0 < d; c0 += G * VEC) {
        const int c = vector_at<VEC>(c0, d);
        Vec<T, VEC> v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (id[r] >= 0 && id[r] < n_rows) v[r] = load_any<T, VEC>(table + id[r] * ldt + c);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[r].v[e] = from_f32<T>(0.f);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (i0 + r >= n) break;
            const float s = id[r] >= 0 && id[r] < n_rows ? scale : 0.f;  // (zeros stay zeros whatever the scale)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[r].v[e] = from_f32<T>(s * to_f32(v[r].v[e]));
            store_any(out + (i0 + r) * ldo + c, v[r]);
        }
    }
}

// ---- sort ----------------------------------------------------------------------------------------------------------------

// Places ranked by counting (15 565 places of 4 221 rows with their lookup: 41 us this way, 38 by digits; 12 200: 34 and 35.5; 9 000: 29
// and 33.5).
constexpr int kRankMax = 12288;
constexpr int kMaxBits = 9;

// A place's sort key: its row, or n_rows for one that adds to nothing (such places end behind every row).
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, int64_t i, int64_t n_rows, int64_t padding) {
    const int64_t id = ids[i];
    return id >= 0 && id < n_rows && id != padding ? (uint32_t)id : (uint32_t)n_rows;
}

// Rank by counting: a workgroup of 16 waves ranks 16 Q places, a wave Q of them.  The wave holds its places' keys in scalar registers and 64
// other places' in a vector register: one compare for 64 pairs, and a count of its bits.  Every second place's bits are counted by the
// scalar unit, which the CU's 16 waves share, the others lane by lane.  Only the step that holds the wave's own places
// looks at positions: all others lie wholly in front of them (an equal key counts) or wholly behind (it does not).  Bound by the
// compares: 6 144 places in 7.7 us; one launch where radix passes would be four.
template <int Q>
__global__ __launch_bounds__(1024) void rank_kernel(const int64_t *__restrict__ ids, int n, int64_t n_rows, int64_t padding,
                                                    uint32_t *__restrict__ keys, uint32_t *__restrict__ places) {
    constexpr int U = 8;  // steps in flight
    __shared__ uint32_t all[kRankMax];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n64 = (n + 63) & ~63;
#pragma unroll 8
    for (int j = threadIdx.x; j < n64; j += 1024) all[j] = j < n ? key_of(ids, j, n_rows, padding) : 0xffffffffu;
    __syncthreads();
    const int i0 = (blockIdx.x * 16 + w) * Q;
    if (i0 >= n) return;
    uint32_t mine[Q], rank[Q], part[Q];  // (a wave's count of a place, or its lanes' counts)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        mine[q] = __builtin_amdgcn_readfirstlane(all[min(i0 + q, n - 1)]);
        rank[q] = part[q] = 0;
    }
    auto step = [&](uint32_t k, auto ahead) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const bool in_front = ahead.value ? k <= mine[q] : k < mine[q];
            if (q & 1) part[q] += in_front;
            else rank[q] += __popcll(__ballot(in_front));
        }
    };
    auto steps = [&](int from, int to, auto ahead) {  // places [from, to), both multiples of 64
        int j = from;
        for (; j + 64 * U <= to; j += 64 * U) {
            uint32_t k[U];
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = all[j + 64 * u + lane];
#pragma unroll
            for (int u = 0; u < U; ++u) step(k[u], ahead);
        }
        for (; j < to; j += 64) step(all[j + lane], ahead);
    };
    const int own = i0 & ~63;  // (64 is a multiple of Q: one step holds all of the wave's places)
    steps(0, own, std::true_type{});
    {
        const uint32_t k = all[own + lane];
#pragma unroll
        for (int q = 0; q < Q; ++q) rank[q] += __popcll(__ballot(k < mine[q] || (k == mine[q] && own + lane < i0 + q)));
    }
    steps(own + 64, n64, std::false_type{});
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (q & 1)
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) part[q] += __shfl_xor(part[q], o);
        const uint32_t r = rank[q] + (q & 1 ? part[q] : 0u);
        if (lane == 0 && i0 + q < n) keys[r] = mine[q], places[r] = (uint32_t)(i0 + q);
    }
}

// A wave's rank of each of its R x 64 places among those with the same digit, in order; slots[digit] counts them.
template <int R>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[R], const bool (&there)[R], int bits, uint32_t *slots, uint32_t (&rank)[R]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        unsigned long long same = __ballot(there[u]);
        for (int b = 0; b < bits; ++b) {
            const bool set = (digit[u] >> b) & 1u;
            const unsigned long long one = __ballot(set);
            same &= set ? one : ~one;
        }
        const int ahead = __popcll(same & ((1ull << lane) - 1ull));
        volatile uint32_t *slot = &slots[digit[u]];
        const uint32_t before = *slot;  // (a wave's LDS accesses are served in the order it issues them)
        rank[u] = before + ahead;
        if (there[u] && ahead == 0) *slot = before + __popcll(same);
    }
}

// The exclusive prefix of one value per thread over a workgroup of TH threads; `part`: TH / 64 entries of LDS.
template <int TH>
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *part) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) part[w] = x;
    __syncthreads();
    uint32_t r = x - v;
    for (int q = 0; q < w; ++q) r += part[q];
    return r;
}

// One launch per pass.  Tiles of 2 048 places, counts[pass][tile][digit].
constexpr int kBins = 1 << kMaxBits, kMoveTile = 2048, kMoveMax = 1 << 16, kMaxPasses = 4;
constexpr int kMoveTiles = kMoveMax / kMoveTile;

// The first pass's counts; the later passes' are cleared.
__global__ __launch_bounds__(512) void move_count_kernel(const int64_t *ids, int n, int64_t n_rows, int64_t padding, int bits, int passes,
                                                         uint32_t *counts) {
    __shared__ uint32_t h[kBins];
    h[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveTile / 512; ++u) {
        const int i = blockIdx.x * kMoveTile + u * 512 + threadIdx.x;
        if (i < n) atomicAdd(&h[key_of(ids, i, n_rows, padding) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    counts[blockIdx.x * kBins + threadIdx.x] = h[threadIdx.x];
    for (int q = 1; q < passes; ++q) counts[((int64_t)q * gridDim.x + blockIdx.x) * kBins + threadIdx.x] = 0;
}

// A pass: a place moves to (places of smaller digits) + (of its digit in earlier tiles) + (of its digit before it here).  A thread per
// digit adds up the tiles' counts, which are few.  COUNT: the next pass's counts are taken where the places arrive, first in LDS: a place
// in every 50 may be the same row's, and adding each to memory by itself takes 45 us of a pass of 65 536, this way 3.
template <bool COUNT>
__global__ __launch_bounds__(512) void move_kernel(const int64_t *ids, const uint32_t *keys, const uint32_t *places, int n, int64_t n_rows,
                                                   int64_t padding, int shift, int bits, const uint32_t *counts, uint32_t *next_counts,
                                                   uint32_t *keys_out, uint32_t *places_out) {
    constexpr int R = kMoveTile / 512;
    __shared__ uint32_t at[8][kBins];  // places of a digit in each wave's eighth, then where the next one goes
    __shared__ uint32_t part[8];
    __shared__ uint32_t arrive[COUNT ? kMoveTiles : 1][kBins];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t mask = (1u << bits) - 1;
#pragma unroll
    for (int q = 0; q < 8; ++q) at[q][threadIdx.x] = 0;
    if constexpr (COUNT)
        for (int t = 0; t < (int)gridDim.x; ++t) arrive[t][threadIdx.x] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * kMoveTile + w * (64 * R);
    uint32_t key[R], digit[R], rank[R];
    bool there[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int i = i0 + u * 64 + lane;
        there[u] = i < n;
        key[u] = there[u] ? (ids ? key_of(ids, i, n_rows, padding) : keys[i]) : 0u;
        digit[u] = (key[u] >> shift) & mask;
    }
    uint32_t total = 0, before = 0;
    for (int t0 = 0; t0 < (int)gridDim.x; t0 += 16) {
        uint32_t c[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) c[t] = t0 + t < (int)gridDim.x ? counts[(t0 + t) * kBins + threadIdx.x] : 0u;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            total += c[t];
            before += t0 + t < (int)blockIdx.x ? c[t] : 0u;
        }
    }
    wave_ranks<R>(digit, there, bits, at[w], rank);
    uint32_t go = block_prefix<512>(total, part) + before;  // (its barrier also ends the counting)
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const uint32_t c = at[q][threadIdx.x];
        at[q][threadIdx.x] = go;
        go += c;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < R; ++u) {
        if (!there[u]) continue;
        const uint32_t to = at[w][digit[u]] + rank[u];
        keys_out[to] = key[u];
        places_out[to] = places ? places[i0 + u * 64 + lane] : (uint32_t)(i0 + u * 64 + lane);
        if constexpr (COUNT) atomicAdd(&arrive[to / kMoveTile][(key[u] >> (shift + bits)) & mask], 1u);
    }
    if constexpr (COUNT) {  // (integer sums: the order of the additions does not show)
        __syncthreads();
        for (int t = 0; t < (int)gridDim.x; ++t) {
            const uint32_t c = arrive[t][threadIdx.x];
            if (c) atomicAdd(&next_counts[t * kBins + threadIdx.x], c);
        }
    }
}

// Three launches per pass (beyond kMoveMax places).  First: how often each digit occurs in each tile -> hist[digit][tile].  (ids: the first pass.)
constexpr int kTile = 2048;
__global__ __launch_bounds__(256) void digit_count_kernel(const int64_t *ids, const uint32_t *keys, int64_t n, int64_t n_rows, int64_t padding,
                                                          int shift, int bits, uint32_t *hist) {
    __shared__ uint32_t h[1 << kMaxBits];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += 256) h[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * kTile;
#pragma unroll
    for (int u = 0; u < kTile / 256; ++u) {
        const int64_t i = i0 + u * 256 + threadIdx.x;
        if (i < n) {
            const uint32_t k = ids ? key_of(ids, i, n_rows, padding) : keys[i];
            atomicAdd(&h[(k >> shift) & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += 256) hist[(int64_t)d * gridDim.x + blockIdx.x] = h[d];
}

// Second launch: one workgroup per digit turns its counts into their exclusive prefix over the tiles; total[digit].
__global__ __launch_bounds__(256) void digit_prefix_kernel(uint32_t *hist, int tiles, uint32_t *total) {
    __shared__ uint32_t part[4];
    uint32_t *h = hist + (int64_t)blockIdx.x * tiles;
    uint32_t run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const uint32_t v = t < tiles ? h[t] : 0u;
        const uint32_t ahead = block_prefix<256>(v, part);
        if (t < tiles) h[t] = run + ahead;
        run += part[0] + part[1] + part[2] + part[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = run;
}

// Third launch: every place moves to (places of smaller digits) + (of its digit in earlier tiles) + (of its digit before it here).
__global__ __launch_bounds__(256) void digit_scatter_kernel(const int64_t *ids, const uint32_t *keys, const uint32_t *places, int64_t n,
                                                            int64_t n_rows, int64_t padding, int shift, int bits, const uint32_t *hist,
                                                            const uint32_t *total, uint32_t *keys_out, uint32_t *places_out) {
    __shared__ uint32_t at[4][1 << kMaxBits];  // places of a digit in each wave's quarter, then where the next one goes
    __shared__ uint32_t part[4];
    const int bins = 1 << bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < 4 * (1 << kMaxBits); d += 256) (&at[0][0])[d] = 0;
    __syncthreads();
    constexpr int R = kTile / 256;
    const int64_t i0 = (int64_t)blockIdx.x * kTile + w * (64 * R);
    uint32_t key[R], digit[R], rank[R];
    bool there[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int64_t i = i0 + u * 64 + lane;
        there[u] = i < n;
        key[u] = there[u] ? (ids ? key_of(ids, i, n_rows, padding) : keys[i]) : 0u;
        digit[u] = (key[u] >> shift) & (bins - 1);
    }
    wave_ranks<R>(digit, there, bits, at[w], rank);
    __syncthreads();
    // start of each digit: exclusive prefix of the totals, two digits per thread
    const uint32_t a = 2 * threadIdx.x < (unsigned)bins ? total[2 * threadIdx.x] : 0u;
    const uint32_t b = 2 * threadIdx.x + 1 < (unsigned)bins ? total[2 * threadIdx.x + 1] : 0u;
    const uint32_t first = block_prefix<256>(a + b, part);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int d = 2 * threadIdx.x + k;
        if (d < bins) {
            uint32_t go = (k ? first + a : first) + hist[(int64_t)d * gridDim.x + blockIdx.x];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t c = at[q][d];
                at[q][d] = go;
                go += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int64_t i = i0 + u * 64 + lane;
        if (i < n) {
            const uint32_t to = at[w][digit[u]] + rank[u];
            keys_out[to] = key[u];
            places_out[to] = places ? places[i] : (uint32_t)i;
        }
    }
}

// ---- sums of runs ------------------------------------------------------------------------------------------------------

struct RunArgs {
    const void *grad;
    int64_t ldg;
    int64_t n, n_rows;
    int d, chunk;              // sorted places per chunk
    int64_t chunks;
    const uint32_t *keys, *places;
    float scale;
    void *out;
    float *part;               // [chunks][2][d]: sums of the chunk's first run and of its last, where they cross a border
    int64_t run_blocks;        // the launch's workgroups that sum; the rest zero rows,
    int stripe;                // this many each
};

template <class T, int VEC>
__device__ __forceinline__ void store_row(T *p, const float (&acc)[VEC], float scale) {
    Vec<T, VEC> v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v.v[e] = from_f32<T>(scale * acc[e]);
    store_any(p, v);
}

// The first of n sorted keys, `stride` apart, that is not below v, by a whole wave: 64 probes a round.
__device__ __forceinline__ int64_t first_not_below(const uint32_t *keys, int64_t n, uint32_t v, int stride = 1) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, cnt = n;  // the answer is in [lo, lo + cnt]
    while (cnt > 0) {
        const int64_t step = (cnt + 63) / 64;
        const int64_t at = lo + (lane + 1) * step - 1;
        const int below = __popcll(__ballot(at < lo + cnt && keys[at * stride] < v));  // probes 0 .. below - 1 are below v
        const int64_t end = lo + cnt;
        lo += below * step;
        cnt = min(step - 1, end - lo);
    }
    return lo;
}

constexpr int kStripe = 256;  // rows that one workgroup zeroes, at most

// G lanes x VEC elements cover a piece of a row (blockIdx.y: which piece); 256 / G chunks per workgroup.  Bound by reading rows in sorted,
// that is random, order: 65 536 gradient rows of 2 KB (bf16, d = 1 024) and 131 072 rows written, 403 MB in 86 us = 4.7 TB/s; the join
// behind it 7.
template <class TI, class TO, int VEC, int G>
__global__ __launch_bounds__(256) void run_sum_kernel(const RunArgs a) {
    constexpr int U = G < 8 ? G : 8;  // rows in flight per lane-group
    const int sub = threadIdx.x % G, grp = threadIdx.x / G;
    const int piece = (blockIdx.y * G + sub) * VEC, col = vector_at<VEC>(piece, a.d);
    const bool on = piece < a.d;
    TO *out = (TO *)a.out;
    const float zero[VEC] = {};
    if (blockIdx.x >= a.run_blocks) {  // zero the rows of a stripe that no place refers to
        __shared__ uint32_t used[kStripe];
        __shared__ int64_t bounds[2];
        const int64_t r0 = (int64_t)(blockIdx.x - a.run_blocks) * a.stripe;
        const int rows = (int)min<int64_t>(a.stripe, a.n_rows - r0);
        if (threadIdx.x < kStripe) used[threadIdx.x] = 0;
        if (threadIdx.x < 128) {
            const int w = threadIdx.x >> 6;
            const int64_t at = first_not_below(a.keys, a.n, (uint32_t)(r0 + w * rows));
            if ((threadIdx.x & 63) == 0) bounds[w] = at;
        }
        __syncthreads();
        if (bounds[1] - bounds[0] <= 4096) {
            for (int64_t p = bounds[0] + threadIdx.x; p < bounds[1]; p += 256) used[a.keys[p] - (uint32_t)r0] = 1;
        } else if (rows <= 16) {  // long runs: a wave looks for each row
            for (int q = threadIdx.x >> 6; q < rows; q += 4) {
                const int64_t at = bounds[0] + first_not_below(a.keys + bounds[0], bounds[1] - bounds[0], (uint32_t)(r0 + q));
                if ((threadIdx.x & 63) == 0) used[q] = at < bounds[1] && a.keys[at] == (uint32_t)(r0 + q);
            }
        } else if ((int)threadIdx.x < rows) {  // each row looks for itself
            int64_t lo = bounds[0], hi = bounds[1];
            const uint32_t key = (uint32_t)(r0 + threadIdx.x);
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (a.keys[mid] < key) lo = mid + 1;
                else hi = mid;
            }
            used[threadIdx.x] = lo < bounds[1] && a.keys[lo] == key;
        }
        __syncthreads();
        if (on)
            for (int q = grp; q < rows; q += 256 / G)
                if (!used[q]) store_row<TO, VEC>(out + (r0 + q) * a.d + col, zero, 1.f);
        return;
    }
    const int64_t c = (int64_t)blockIdx.x * (256 / G) + grp;
    if (c >= a.chunks) return;
    const int64_t p0 = c * a.chunk, p1 = min(p0 + a.chunk, a.n);
    const TI *grad = (const TI *)a.grad;
    const uint32_t none = (uint32_t)a.n_rows;
    const uint32_t ahead = p0 > 0 ? a.keys[p0 - 1] : 0xffffffffu;  // (no key is 2^32 - 1)
    const uint32_t behind = p1 < a.n ? a.keys[p1] : 0xffffffffu;
    float acc[VEC] = {};
    uint32_t run = a.keys[p0];
    bool first = run == ahead;  // the current run began in an earlier chunk
    // U places at a time, a lane each, one turn ahead of their rows
    auto key_at = [&](int64_t p) { return sub < U && p + sub < p1 ? a.keys[p + sub] : none; };
    auto place_at = [&](int64_t p) { return sub < U && p + sub < p1 ? a.places[p + sub] : 0u; };
    uint32_t next_key = key_at(p0), next_place = place_at(p0);
    for (int64_t p = p0; p < p1; p += U) {
        const uint32_t my_key = next_key, my_place = next_place;
        next_key = key_at(p + U), next_place = place_at(p + U);
        uint32_t key[U];
        Vec<TI, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            key[u] = __shfl(my_key, u, G);
            const uint32_t place = __shfl(my_place, u, G);
            if (key[u] != none && on) v[u] = load_any<TI, VEC>(grad + (int64_t)place * a.ldg + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (key[u] != run) {  // the run ends here (a place behind the chunk's last has no row: `none`)
                if (p + u >= p1) break;
                if (run != none && on) {
                    if (first) {
                        float *to = a.part + (2 * c) * a.d + col;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) to[e] = acc[e];
                    } else {
                        store_row<TO, VEC>(out + (int64_t)run * a.d + col, acc, a.scale);
                    }
                }
                run = key[u];
                first = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
            if (run != none && on) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += to_f32(v[u].v[e]);
            }
        }
    }
    if (run == none) return;
    const bool goes_on = run == behind;
    if (!first && !goes_on) {
        if (on) store_row<TO, VEC>(out + (int64_t)run * a.d + col, acc, a.scale);
        return;
    }
    if (on) {
        float *to = a.part + (2 * c + (first ? 0 : 1)) * a.d + col;
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e] = acc[e];
    }
}

// Few places (n <= kFewPlaces): one launch, no sorted list.  A workgroup owns `stripe` rows (and a piece of their columns), finds the places that
// refer to them, ranks those by (row, place) by counting, and sums a run per lane-group; its other rows are zeroed.  Bound by the rows'
// zeroes where the table is large, by its launch where it is not: 32 places of 40 982 x 64 fp32 in 5.4 us; 256 in 14.6, where three launches
// take 8.4 for 257 (the ranks and the runs of a row's workgroup; the host's time for three calls and a workspace is not in that).
constexpr int kFewPlaces = 256;

template <class TI, class TO, int VEC, int G>
__global__ __launch_bounds__(256) void few_places_kernel(const RunArgs a, const int64_t *__restrict__ ids, int64_t padding, int stripe) {
    constexpr int U = 16;  // rows in flight per lane-group (a row that all places refer to is one group's: 256 of them in 16 turns)
    __shared__ __align__(16) uint32_t row_of[kFewPlaces];  // of a place, from the workgroup's first row; 256: another's
    __shared__ uint32_t run_of[kFewPlaces + 1], place_of[kFewPlaces];
    __shared__ uint32_t used[256];
    __shared__ uint32_t found;
    const int n = (int)a.n, i = threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.x * stripe;
    const int rows = (int)min<int64_t>(stripe, a.n_rows - r0);
    uint32_t mine = 256;
    if (i < n) {
        const int64_t id = ids[i];
        if (id >= r0 && id < r0 + rows && id != padding) mine = (uint32_t)(id - r0);
    }
    row_of[i] = mine;
    used[i] = 0;
    if (i == 0) found = 0;
    __syncthreads();
    if (mine < 256) {
        uint32_t rank = 0;
        const int n4 = (n + 3) & ~3;
        for (int j = 0; j < n4; j += 4) {
            const uint4 k = *reinterpret_cast<const uint4 *>(row_of + j);
            rank += k.x < mine || (k.x == mine && j < i);
            rank += k.y < mine || (k.y == mine && j + 1 < i);
            rank += k.z < mine || (k.z == mine && j + 2 < i);
            rank += k.w < mine || (k.w == mine && j + 3 < i);
        }
        run_of[rank] = mine;
        place_of[rank] = (uint32_t)i;
        used[mine] = 1;
        atomicAdd(&found, 1u);
    }
    __syncthreads();
    const int sub = i % G, grp = i / G, m = (int)found;
    const int piece = (blockIdx.y * G + sub) * VEC, col = vector_at<VEC>(piece, a.d);
    if (piece >= a.d) return;
    const TI *grad = (const TI *)a.grad;
    TO *out = (TO *)a.out;
    const float zero[VEC] = {};
    for (int e0 = grp; e0 < m; e0 += 256 / G) {
        const uint32_t run = run_of[e0];
        if (e0 && run_of[e0 - 1] == run) continue;  // another lane-group has it
        int end = e0 + 1;
        while (end < m && run_of[end] == run) ++end;
        float acc[VEC] = {};
        for (int p = e0; p < end; p += U) {
            Vec<TI, VEC> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p + u < end) v[u] = load_any<TI, VEC>(grad + (int64_t)place_of[p + u] * a.ldg + col);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p + u < end)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[e] += to_f32(v[u].v[e]);
        }
        store_row<TO, VEC>(out + (r0 + run) * a.d + col, acc, a.scale);
    }
    for (int q = grp; q < rows; q += 256 / G)
        if (!used[q]) store_row<TO, VEC>(out + (r0 + q) * a.d + col, zero, 1.f);
}

// Runs over several chunks: the last sum of the chunk they start in, then the first sums of the chunks they reach into.  A workgroup finds
// out for itself whether a run starts in its chunk and goes on (a list of such chunks cost the launch before it an atomic each at one
// address: 5 us for 3 000 of them).
template <class TO, int VEC, int G>
__global__ __launch_bounds__(256) void run_join_kernel(const RunArgs a) {
    constexpr int N = 256 / G;
    __shared__ float sums[256 * VEC];
    const int sub = threadIdx.x % G, grp = threadIdx.x / G;
    const int piece = (blockIdx.y * G + sub) * VEC, col = vector_at<VEC>(piece, a.d);
    const bool on = piece < a.d;
    for (int64_t c = blockIdx.x; c + 1 < a.chunks; c += gridDim.x) {
        const int64_t p0 = c * a.chunk, p1 = p0 + a.chunk;
        const uint32_t key = a.keys[p1], own = a.keys[p1 - 1], ahead = p0 > 0 ? a.keys[p0 - 1] : 0xffffffffu;
        if (key != own || key == ahead || key == (uint32_t)a.n_rows) continue;  // no run, or none of a row, starts in chunk c and goes on
        // the last chunk that starts with the run's key
        const int64_t last = c + first_not_below(a.keys + (c + 1) * a.chunk, a.chunks - c - 1, key + 1u, a.chunk);
        // parts c, c + 1, .., last: an equal piece for each lane-group, the pieces joined in order
        const int64_t cnt = last - c + 1, per = (cnt + N - 1) / N;
        const int64_t q0 = c + grp * per, q1 = min(q0 + per, last + 1);
        float acc[VEC] = {};
        if (on) {
#pragma unroll 8
            for (int64_t q = q0; q < q1; ++q) {
                const float *from = a.part + (2 * q + (q == c ? 1 : 0)) * a.d + col;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += from[e];
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[threadIdx.x * VEC + e] = acc[e];
        __syncthreads();
        if (grp == 0 && on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            for (int q = 0; q < N; ++q)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += sums[(q * G + sub) * VEC + e];
            store_row<TO, VEC>((TO *)a.out + (int64_t)key * a.d + col, acc, a.scale);
        }
        __syncthreads();
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------

static int64_t round16e(int64_t b) { return (b + 15) & ~int64_t(15); }

// Sorted places per chunk: enough chunks for eight waves per SIMD where the places allow it, 64 places at most (long runs leave few parts).
// The gradient with 8, 16, 32 and 64, us (the rule's in brackets): 6 144 of 40 982 x 64 fp32 [15.7], 17, 21, 29; 65 536 of 131 072 x 128 fp32
// [50], 47, 47, 51; 65 536 of 131 072 x 1 024 bf16 128, 125, [122], 128; 1 000 000 of 200 000 x 64 fp32 343, 245, 195, 169 [24 places: 209].
static int chunk_of(int64_t n, int d) {
    const int64_t want = n * std::max(1, d / 8) / (64 * 4096);
    return want <= 8 ? 8 : want >= 64 ? 64 : (int)want / 8 * 8;
}

struct Layout {
    int64_t keys, places, keys2, places2, hist, total, part, bytes;
    int chunk, tiles;
    int64_t chunks;
};

static Layout layout_of(int64_t n, int d) {
    Layout l{};
    l.chunk = chunk_of(n, d);
    l.chunks = (n + l.chunk - 1) / l.chunk;
    l.tiles = (int)((n + kTile - 1) / kTile);
    int64_t at = 0;
    auto take = [&](int64_t b) {
        const int64_t r = at;
        at += round16e(b);
        return r;
    };
    if (n <= kFewPlaces) return l;
    l.keys = take(4 * n), l.places = take(4 * n);
    if (n > kRankMax) {
        l.keys2 = take(4 * n), l.places2 = take(4 * n);
        l.hist = take(4ll * kBins * l.tiles * (n <= kMoveMax ? kMaxPasses : 1));
        l.total = take(4 * kBins);
    }
    l.part = take(4ll * 2 * l.chunks * d);
    l.bytes = at;
    return l;
}

template <class TI, class TO, int VEC, int G>
static void launch_runs(const RunArgs &a0, const int64_t *ids, int64_t padding, hipStream_t s) {
    RunArgs a = a0;
    if (a.n <= kFewPlaces) {
        int stripe = 256;  // fewer rows where there are few, for more workgroups
        while (stripe > 8 && a.n_rows < stripe * 256) stripe /= 2;
        hipLaunchKernelGGL((few_places_kernel<TI, TO, VEC, G>), dim3((unsigned)((a.n_rows + stripe - 1) / stripe), (unsigned)((a.d + G * VEC - 1) / (G * VEC))),
                           dim3(256), 0, s, a, ids, padding, stripe);
        return;
    }
    a.run_blocks = (a.chunks + 256 / G - 1) / (256 / G);
    const unsigned pieces = (unsigned)((a.d + G * VEC - 1) / (G * VEC));
    // rows of about 1 024 places, which a workgroup takes its rows' marks from at once
    a.stripe = kStripe;
    while (a.stripe > 8 && a.n * a.stripe > 1024 * a.n_rows) a.stripe /= 2;
    const int64_t zero_blocks = (a.n_rows + a.stripe - 1) / a.stripe;
    hipLaunchKernelGGL((run_sum_kernel<TI, TO, VEC, G>), dim3((unsigned)(a.run_blocks + zero_blocks), pieces), dim3(256), 0, s, a);
    if (a.chunks > 1)
        hipLaunchKernelGGL((run_join_kernel<TO, VEC, G>), dim3((unsigned)std::min<int64_t>(a.chunks, 16384), pieces), dim3(256), 0, s, a);
}

template <class TI, class TO>
static int launch_runs_of(const RunArgs &a, const int64_t *ids, int64_t padding, bool wide, hipStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(TI);
    const int lanes = wide ? (a.d + VEC - 1) / VEC : a.d;
    if (wide) {
        if (lanes <= 4) launch_runs<TI, TO, VEC, 4>(a, ids, padding, s);
        else if (lanes <= 8) launch_runs<TI, TO, VEC, 8>(a, ids, padding, s);
        else if (lanes <= 16) launch_runs<TI, TO, VEC, 16>(a, ids, padding, s);
        else if (lanes <= 32) launch_runs<TI, TO, VEC, 32>(a, ids, padding, s);
        else launch_runs<TI, TO, VEC, 64>(a, ids, padding, s);
    } else {
        launch_runs<TI, TO, 1, 8>(a, ids, padding, s);  // rows of less than 16 bytes: at most seven elements
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

static int check_places(int64_t n, int64_t n_rows, int d) {
    if (n < 0 || n_rows < 0 || d <= 0) return fail(RBG_ESHAPE, "n = %lld, n_rows = %lld, d = %d", (long long)n, (long long)n_rows, d);
    if (n >= 0x7fff0000ll || n_rows >= 0x7fffffffll || d > 1 << 20)
        return fail(RBG_EUNSUPPORTED, "ids or rows beyond 2^31, or d beyond 2^20: n = %lld, n_rows = %lld, d = %d", (long long)n, (long long)n_rows, d);
    return RBG_OK;
}

}  // namespace rbg

using namespace rbg;

extern "C" {

int rbg_embedding(const void *table, int64_t ldt, int64_t n_rows, int d, int dtype, const int64_t *ids, int64_t n, float scale, void *out,
                  int64_t ldo, void *stream) {
    clear_error();
    if (!elem_ok(dtype)) return fail(RBG_EINVAL, "dtype = %d", dtype);
    if (n < 0 || n_rows < 0 || d <= 0 || ldt < d || ldo < d)
        return fail(RBG_ESHAPE, "n = %lld, n_rows = %lld, d = %d, ldt = %lld, ldo = %lld", (long long)n, (long long)n_rows, d, (long long)ldt, (long long)ldo);
    if (d > 1 << 30) return fail(RBG_EUNSUPPORTED, "d = %d: at most 2^30 columns", d);
    if (n > (int64_t)1 << 34) return fail(RBG_EUNSUPPORTED, "n = %lld: at most 2^34 ids", (long long)n);
    constexpr int64_t kIdsPerLaunch = 1 << 26;  // (a grid holds fewer than 2^32 threads per dimension, a workgroup of 256 at least 16 ids)
    if (n == 0) return RBG_OK;
    if ((n_rows && !table) || !ids || !out) return fail(RBG_EINVAL, "NULL pointer");
    const int size = elem_size(dtype);
    if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) % size) return fail(RBG_EINVAL, "a table is not aligned to its type");
    const bool wide = (int64_t)d * size >= 16;
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        constexpr int VEC = 16 / (int)sizeof(E);
        auto go = [&](auto kernel, int G) {
            const int64_t per = 256 / G * 4;
            for (int64_t i0 = 0; i0 < n; i0 += kIdsPerLaunch) {
                const int64_t cnt = std::min(kIdsPerLaunch, n - i0);
                hipLaunchKernelGGL(kernel, dim3((unsigned)((cnt + per - 1) / per)), dim3(256), 0, (hipStream_t)stream, (const E *)table, ldt, n_rows, ids + i0,
                                   cnt, d, scale, (E *)out + i0 * ldo, ldo);
            }
        };
        const int lanes = wide ? (d + VEC - 1) / VEC : d;
        if (wide) {
            if (lanes <= 4) go(lookup_kernel<E, VEC, 4>, 4);
            else if (lanes <= 16) go(lookup_kernel<E, VEC, 16>, 16);
            else go(lookup_kernel<E, VEC, 64>, 64);
        } else {
            go(lookup_kernel<E, 1, 8>, 8);  // rows of less than 16 bytes: at most seven elements
        }
        RBG_HIP(hipGetLastError());
        return (int)RBG_OK;
    });
}

int rbg_embedding_grad_workspace(int64_t n, int64_t n_rows, int d, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(RBG_EINVAL, "bytes is NULL");
    if (int rc = check_places(n, n_rows, d)) return rc;
    *bytes = layout_of(n, d).bytes;
    return RBG_OK;
}

int rbg_embedding_grad(const void *grad, int64_t ldg, int dtype, const int64_t *ids, int64_t n, int64_t n_rows, int d, float scale,
                       int64_t padding_idx, void *out, int out_dtype, void *workspace, void *stream) {
    clear_error();
    if (!elem_ok(dtype) || (out_dtype != dtype && out_dtype != RBG_F32)) return fail(RBG_EINVAL, "dtype = %d, out_dtype = %d", dtype, out_dtype);
    if (int rc = check_places(n, n_rows, d)) return rc;
    if (ldg < d) return fail(RBG_ESHAPE, "d = %d, ldg = %lld", d, (long long)ldg);
    if (n_rows == 0) return RBG_OK;
    if ((n && (!grad || !ids)) || !out || (n > kFewPlaces && !workspace)) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(workspace)) return fail(RBG_EINVAL, "workspace is not 16-byte aligned");
    const int size = elem_size(dtype), out_size = elem_size(out_dtype);
    if (reinterpret_cast<uintptr_t>(grad) % size || reinterpret_cast<uintptr_t>(out) % out_size) return fail(RBG_EINVAL, "a tensor is not aligned to its type");
    hipStream_t s = (hipStream_t)stream;
    const Layout l = layout_of(n, d);
    char *w = (char *)workspace;
    uint32_t *keys = (uint32_t *)(w + l.keys), *places = (uint32_t *)(w + l.places);
    if (n > kFewPlaces && n <= kRankMax) {
        // places per wave: few where there are few, so that every CU has a workgroup
        if (n <= 4096) hipLaunchKernelGGL((rank_kernel<1>), dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, s, ids, (int)n, n_rows, padding_idx, keys, places);
        else if (n <= 8192) hipLaunchKernelGGL((rank_kernel<2>), dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, s, ids, (int)n, n_rows, padding_idx, keys, places);
        else hipLaunchKernelGGL((rank_kernel<4>), dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, s, ids, (int)n, n_rows, padding_idx, keys, places);
    } else if (n > kRankMax) {
        int bits = 1;
        while (((int64_t)1 << bits) <= n_rows) ++bits;  // keys 0 .. n_rows
        const int passes = (bits + kMaxBits - 1) / kMaxBits, width = (bits + passes - 1) / passes;
        uint32_t *k2 = (uint32_t *)(w + l.keys2), *p2 = (uint32_t *)(w + l.places2);
        uint32_t *hist = (uint32_t *)(w + l.hist), *total = (uint32_t *)(w + l.total);
        const uint32_t *from_k = nullptr, *from_p = nullptr;
        if (n <= kMoveMax) hipLaunchKernelGGL(move_count_kernel, dim3(l.tiles), dim3(512), 0, s, ids, (int)n, n_rows, padding_idx, width, passes, hist);
        // the last pass ends in (keys, places)
        uint32_t *to_k = passes & 1 ? keys : k2, *to_p = passes & 1 ? places : p2;
        for (int q = 0; q < passes; ++q) {
            const int64_t *src = q == 0 ? ids : nullptr;
            if (n <= kMoveMax) {
                uint32_t *counts = hist + (int64_t)q * l.tiles * kBins, *next = counts + (int64_t)l.tiles * kBins;
                if (q + 1 < passes)
                    hipLaunchKernelGGL((move_kernel<true>), dim3(l.tiles), dim3(512), 0, s, src, from_k, from_p, (int)n, n_rows, padding_idx, q * width, width,
                                       counts, next, to_k, to_p);
                else
                    hipLaunchKernelGGL((move_kernel<false>), dim3(l.tiles), dim3(512), 0, s, src, from_k, from_p, (int)n, n_rows, padding_idx, q * width, width,
                                       counts, nullptr, to_k, to_p);
            } else {
                hipLaunchKernelGGL(digit_count_kernel, dim3(l.tiles), dim3(256), 0, s, src, from_k, n, n_rows, padding_idx, q * width, width, hist);
                hipLaunchKernelGGL(digit_prefix_kernel, dim3(1u << width), dim3(256), 0, s, hist, l.tiles, total);
                hipLaunchKernelGGL(digit_scatter_kernel, dim3(l.tiles), dim3(256), 0, s, src, from_k, from_p, n, n_rows, padding_idx, q * width, width,
                                   hist, total, to_k, to_p);
            }
            from_k = to_k, from_p = to_p;
            to_k = to_k == keys ? k2 : keys, to_p = to_p == places ? p2 : places;
        }
    }
    RBG_HIP(hipGetLastError());
    const RunArgs a{grad, ldg, n, n_rows, d, l.chunk, l.chunks, keys, places, scale, out, (float *)(w + l.part), 0, 0};
    const bool wide = (int64_t)d * size >= 16;
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        return out_dtype == dtype ? launch_runs_of<E, E>(a, ids, padding_idx, wide, s) : launch_runs_of<E, float>(a, ids, padding_idx, wide, s);
    });
}

}  // extern "C"
