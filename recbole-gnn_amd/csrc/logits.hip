// logits.hip — losses on whole rows of logits: distillation from a teacher's top list, log-probabilities of targets, and the
// preference loss on pairs of packed sequences, each with its gradient.
//
// Mathematics.  With m = max_j z_j, c = log2(e) / T and e_j = 2^((z_j - m) c), S = sum_j e_j, a row's softmax is q_j = e_j / S and
// log q_j = (z_j - m) / T - ln S.  (z - m is formed before it is scaled: a row whose logits all hold the type's lowest value is a
// uniform row, not a difference of overflows.)  (m, S) is all a gradient needs; a row of nothing but -inf has m = -inf, S = 0.
// Every gradient here is a e_j plus a few sparse terms: the teacher's entries, or the target.
//
// What bounds it.  The rows are read from and written to HBM and nothing else is large: 16 bytes per lane and request, a row's
// elements in front of and behind its 16-byte boundaries one by one (rows of an odd length start anywhere).  Value and gradient of
// the distillation in one call keep the row in registers between the two: one read, one write.  The preference loss needs
// every token of a pair before any gradient of it, so its rows are read twice.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "vocab_common.h"

namespace rbg {

constexpr int kMaxEntries = 256;  // of a teacher's list

// A row of V elements as 16-byte chunks: `head` elements, then nb chunks, then the rest; x-th of the `extra` loose elements = at(x).
template <class T>
struct RowShape {
    static constexpr int E = 16 / (int)sizeof(T);
    int head, nb, extra, tail;
    __device__ __forceinline__ RowShape(const T *p, int V) {
        const int off = (int)((16u - (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / (int)sizeof(T);
        head = min(off, V);
        nb = (V - head) / E;
        tail = head + nb * E;
        extra = head + (V - tail);
    }
    __device__ __forceinline__ int at(int x) const { return x < head ? x : tail + (x - head); }
};

// 16 bytes of a gradient.  Rows that a workgroup writes (NT) go past the caches: what these hold is then logits, of which a second reader
// finds more (value and gradient of the preference loss: 172 us with plain stores and 139 us past the caches at 4 096 x 40 982 bf16, 107
// and 86 at 1 200 x 40 001 fp32; of the distillation 77 and 73 at 2 048 x 40 982 bf16; alike at 600 x 40 001 bf16).  Compile-time:
// with both kinds of store behind a condition the compiler makes one of them, the plain one.
template <bool NT>
__device__ __forceinline__ void put16(void *p, const void *v) {
    u32x4 x;
    __builtin_memcpy(&x, v, 16);
    if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<u32x4 *>(p));
    else *reinterpret_cast<u32x4 *>(p) = x;
}

struct MaxSum {
    float m, s;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// (m, s) of two parts of a row.  A part of nothing but -inf is (-inf, 0); NaN stays in s.
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s};
    return {m, a.s * exp2_fast((a.m - m) * c) + b.s * exp2_fast((b.m - m) * c)};
}

__device__ __forceinline__ MaxSum wave_join(MaxSum v, float c) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join(v, MaxSum{__shfl_xor(v.m, o), __shfl_xor(v.s, o)}, c);
    return v;
}

// Over a workgroup of TH threads; every thread gets the result.  `sh`: TH / 64 entries of LDS nobody else uses meanwhile.
template <int TH>
__device__ __forceinline__ MaxSum block_join(MaxSum v, float c, MaxSum *sh) {
    v = wave_join(v, c);
    if constexpr (TH > kWave) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        if (lane == 0) sh[w] = v;
        __syncthreads();
        v = sh[0];
#pragma unroll
        for (int i = 1; i < TH / kWave; ++i) v = join(v, sh[i], c);
    }
    return v;
}

// The running (m, s) of one thread over U chunks at a time: one rescaling for U E elements.
template <class T, int N>
__device__ __forceinline__ void online(MaxSum &r, const float (&x)[N], float c) {
    float m = r.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    const float mm = m == -INFINITY ? 0.f : m;
    float s = r.s * exp2_fast((r.m - mm) * c);
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2_fast((x[i] - mm) * c);
    r.m = m;
    r.s = s;
}

// The TH threads that share a row: a workgroup, or (TH = 64) a wave of one.
template <int TH>
__device__ __forceinline__ int member() { return TH == kWave ? (int)(threadIdx.x & 63) : (int)threadIdx.x; }

// (m, s) of chunks [c0, c1) of a row, and of its loose elements when `loose`, as far as one of its TH threads sees it.
template <class T, int TH, int U>
__device__ __forceinline__ MaxSum scan_row(const T *__restrict__ z, const RowShape<T> &sh, int c0, int c1, bool loose, float c) {
    constexpr int E = RowShape<T>::E;
    const Vec<T, E> *body = reinterpret_cast<const Vec<T, E> *>(z + sh.head);
    MaxSum r{-INFINITY, 0.f};
    const int tid = member<TH>();
    int i = c0 + tid;
    for (; i + (U - 1) * TH < c1; i += U * TH) {
        Vec<T, E> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = body[i + u * TH];
        float x[U * E];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) x[u * E + e] = to_f32(v[u].v[e]);
        online<T>(r, x, c);
    }
    if (i < c1) {  // at most U more, all in flight at once
        Vec<T, E> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * TH < c1) v[u] = body[i + u * TH];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u * TH >= c1) break;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = to_f32(v[u].v[e]);
            online<T>(r, x, c);
        }
    }
    if (loose && tid < sh.extra) {
        const float x[1] = {to_f32(z[sh.at(tid)])};
        online<T>(r, x, c);
    }
    return r;
}

// g_j = a 2^((z_j - m) c) over chunks [c0, c1) (and the loose elements); element `hot` (or -1) gets `more` on top, before the rounding.
// z and g may be the same row: an element is read and written by the same thread.
template <class T, int TH, int U>
__device__ __forceinline__ void write_row(const T *z, T *g, const RowShape<T> &sh, int c0, int c1, bool loose, float m, float c, float a,
                                          int hot, float more) {
    constexpr int E = RowShape<T>::E;
    const Vec<T, E> *body = reinterpret_cast<const Vec<T, E> *>(z + sh.head);
    Vec<T, E> *out = reinterpret_cast<Vec<T, E> *>(g + sh.head);
    const bool wide = on_16_dev(out);
    const int tid = member<TH>();
    const int hb = hot - sh.head;
    const int hc = hot >= sh.head && hot < sh.tail ? hb / E : -1, he = hb - hc * E;
    for (int i0 = c0; i0 < c1; i0 += U * TH) {
        Vec<T, E> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * TH + tid;
            if (i < c1) v[u] = body[i];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * TH + tid;
            if (i >= c1) break;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = a * exp2_fast((to_f32(v[u].v[e]) - m) * c);
            if (i == hc) {
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] += e == he ? more : 0.f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) v[u].v[e] = from_f32<T>(x[e]);
            if (wide) {
                put16<(TH > kWave)>(out + i, &v[u]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) g[sh.head + i * E + e] = v[u].v[e];
            }
        }
    }
    if (loose && tid < sh.extra) {
        const int j = sh.at(tid);
        float x = a * exp2_fast((to_f32(z[j]) - m) * c);
        if (j == hot) x += more;
        g[j] = from_f32<T>(x);
    }
}

template <class T, int TH>
__device__ __forceinline__ void zero_row(T *g, const RowShape<T> &sh, int c0, int c1, bool loose) {
    constexpr int E = RowShape<T>::E;
    Vec<T, E> *out = reinterpret_cast<Vec<T, E> *>(g + sh.head);
    const bool wide = on_16_dev(out);
    const int tid = member<TH>();
    Vec<T, E> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.v[e] = from_f32<T>(0.f);
    for (int i = c0 + tid; i < c1; i += TH) {
        if (wide) {
            put16<(TH > kWave)>(out + i, &v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) g[sh.head + i * E + e] = v.v[e];
        }
    }
    if (loose && tid < sh.extra) g[sh.at(tid)] = from_f32<T>(0.f);
}

// Part s of S of a row's chunks.
__device__ __forceinline__ void part_of(int nb, int s, int S, int &c0, int &c1) {
    c0 = (int)((int64_t)nb * s / S);
    c1 = (int)((int64_t)nb * (s + 1) / S);
}

// ---- distillation --------------------------------------------------------------------------------------------------------

struct DistillArgs {
    const void *z;
    int64_t ldz;
    int V, k;
    const int64_t *idx;
    const float *val;
    float c, T;  // log2(e) / T
    const float *row_w;
    float *loss, *stats;
    void *grad;
    int64_t ldg;
    MaxSum *part;  // [n][S] when a row is split
    float *zt;     // [n][k] when a row is split: the entries' logits (the gradient may overwrite them)
};

struct Entries {
    int idx[kMaxEntries];    // -1: none
    float p[kMaxEntries];    // teacher's probability
    float z[kMaxEntries];    // student's logit there
    float any;               // 0: a row without entries
    MaxSum red[16];
};

// Wave 0 fills the list: probabilities over the entries that are there.  Ends without a barrier.
template <class T>
__device__ __forceinline__ void load_entries(const DistillArgs &a, int64_t row, const T *z, const float *zt, Entries &sh) {
    if (threadIdx.x >= kWave) return;
    float v[kMaxEntries / kWave];
    float tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < kMaxEntries / kWave; ++u) {
        const int i = u * kWave + threadIdx.x;
        v[u] = -INFINITY;
        if (i < a.k) {
            const int64_t j = a.idx[row * a.k + i];
            const bool there = j >= 0 && j < a.V;
            sh.idx[i] = there ? (int)j : -1;
            sh.z[i] = there ? (zt ? zt[row * a.k + i] : to_f32(z[j])) : 0.f;
            if (there) v[u] = a.val[row * a.k + i];
            tm = fmaxf(tm, v[u]);
        }
    }
    tm = wave_max(tm);
    const float tmm = tm == -INFINITY ? 0.f : tm;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < kMaxEntries / kWave; ++u) {
        v[u] = exp2_fast((v[u] - tmm) * a.c);
        s += v[u];
    }
    s = wave_sum(s);
#pragma unroll
    for (int u = 0; u < kMaxEntries / kWave; ++u) {
        const int i = u * kWave + threadIdx.x;
        if (i < a.k) sh.p[i] = s == 0.f ? 0.f : v[u] / s;
    }
    if (threadIdx.x == 0) sh.any = s;
}

__device__ __forceinline__ bool distill_empty(const Entries &sh, MaxSum st) { return sh.any == 0.f || (st.m == -INFINITY && st.s == 0.f); }

// Wave 0: the row's loss from its list.  The teacher's log-probabilities are taken of the rounded p: p (log p - log q) is then the
// divergence of the p that the gradient uses.
__device__ __forceinline__ void entries_loss(const DistillArgs &a, int64_t row, const Entries &sh, MaxSum st) {
    if (threadIdx.x >= kWave) return;
    const float lns = logf(st.s), inv_t = 1.f / a.T;
    float l = 0.f;
    for (int i = threadIdx.x; i < a.k; i += kWave)
        if (sh.idx[i] >= 0 && sh.p[i] != 0.f) l += sh.p[i] * (logf(sh.p[i]) - ((sh.z[i] - st.m) * inv_t - lns));
    l = wave_sum(l);
    if (threadIdx.x == 0) {
        if (a.loss) a.loss[row] = distill_empty(sh, st) ? 0.f : a.T * a.T * l;
        if (a.stats) a.stats[2 * row] = st.m, a.stats[2 * row + 1] = st.s;
    }
}

// The entries' elements of the gradient, over what write_row stored there (a barrier lies between): w T (q - sum of p).  The first
// entry of an index writes it.  Only elements that part [c0, c1) (+ loose) of the row owns.
template <class T, int TH>
__device__ __forceinline__ void fix_entries(const DistillArgs &a, T *g, const RowShape<T> &rs, int c0, int c1, bool loose, const Entries &sh,
                                            MaxSum st, float w) {
    for (int i = threadIdx.x; i < a.k; i += TH) {
        const int j = sh.idx[i];
        if (j < 0) continue;
        const int b = j - rs.head;
        const bool in_body = b >= 0 && j < rs.tail;
        if (in_body ? (b / RowShape<T>::E < c0 || b / RowShape<T>::E >= c1) : !loose) continue;
        float p = 0.f;
        bool first = true;
        for (int t = 0; t < a.k; ++t) {
            if (sh.idx[t] != j) continue;
            p += sh.p[t];
            first &= t >= i;
        }
        if (first) g[j] = from_f32<T>(w * a.T * (exp2_fast((sh.z[i] - st.m) * a.c) / st.s - p));
    }
}

// The loss alone: one workgroup streams a row.  Bound by the reads: 4 096 x 91 600 fp32, 1.5 GB in 253 us = 5.9 TB/s.
template <class T, int TH>
__global__ __launch_bounds__(TH) void distill_eval_kernel(const DistillArgs a) {
    __shared__ Entries sh;
    const int64_t row = blockIdx.x;
    const T *z = (const T *)a.z + row * a.ldz;
    const RowShape<T> rs(z, a.V);
    load_entries(a, row, z, nullptr, sh);
    const MaxSum st = block_join<TH>(scan_row<T, TH, 4>(z, rs, 0, rs.nb, true, a.c), a.c, sh.red);
    __syncthreads();
    entries_loss(a, row, sh, st);
}

// The passes over a row in registers each convert its elements anew: kept, the converted ones would take twice the registers of a 16-bit row.
template <int N>
__device__ __forceinline__ void forget(u32x4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}
template <class T, int E>
__device__ __forceinline__ Vec<T, E> as_elems(const u32x4 &v) {
    Vec<T, E> r;
    __builtin_memcpy(&r, &v, 16);
    return r;
}

// Value and gradient of a row that fits the registers of its workgroup: NC chunks of 16 bytes per thread.  The teacher's entries are set
// right behind the row's stores and a barrier.  (Finding each thread's entries on a list in LDS before its stores instead: 82 us
// against 74 at 2048 x 40 982 bf16 — the lists' making delays every store of the row, the second look only its last ones.)  Bound by
// memory: at that size 336 MB in 60 us = 5.6 TB/s behind another call of itself, 73 us with other work between.
template <class T, int TH, int NC>
__global__ __launch_bounds__(TH, NC <= 12 ? 5 : 4) void distill_row_kernel(const DistillArgs a) {
    constexpr int E = RowShape<T>::E;
    __shared__ Entries sh;
    const int64_t row = blockIdx.x;
    const T *z = (const T *)a.z + row * a.ldz;
    T *g = (T *)a.grad + row * a.ldg;
    const RowShape<T> rs(z, a.V);
    const u32x4 *body = reinterpret_cast<const u32x4 *>(z + rs.head);
    u32x4 v[NC];
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        const int i = u * TH + threadIdx.x;
        if (i < rs.nb) v[u] = body[i];
    }
    const bool has_loose = (int)threadIdx.x < rs.extra;
    const float loose = has_loose ? to_f32(z[rs.at(threadIdx.x)]) : -INFINITY;
    load_entries(a, row, z, nullptr, sh);
    MaxSum r{loose, 0.f};
#pragma unroll
    for (int u = 0; u < NC; ++u)
        if (u * TH + (int)threadIdx.x < rs.nb)
#pragma unroll
            for (int e = 0; e < E; ++e) r.m = fmaxf(r.m, to_f32(as_elems<T, E>(v[u]).v[e]));
    forget(v);
    const float mm = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
    for (int u = 0; u < NC; ++u)
        if (u * TH + (int)threadIdx.x < rs.nb)
#pragma unroll
            for (int e = 0; e < E; ++e) r.s += exp2_fast((to_f32(as_elems<T, E>(v[u]).v[e]) - mm) * a.c);
    forget(v);
    if (has_loose) r.s += exp2_fast((loose - mm) * a.c);
    const MaxSum st = block_join<TH>(r, a.c, sh.red);
    if constexpr (TH == kWave) __syncthreads();  // (block_join's own barrier hands over the entries elsewhere)
    entries_loss(a, row, sh, st);                // (the other waves are storing meanwhile: at the end it would prolong the workgroup)
    if (distill_empty(sh, st)) {
        zero_row<T, TH>(g, rs, 0, rs.nb, true);
    } else {
        const float w = a.row_w ? a.row_w[row] : 1.f;
        const float s = w * a.T / st.s;
        Vec<T, E> *out = reinterpret_cast<Vec<T, E> *>(g + rs.head);
        const bool wide = on_16_dev(out);
#pragma unroll
        for (int u = 0; u < NC; ++u) {
            const int i = u * TH + threadIdx.x;
            if (i >= rs.nb) break;
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(s * exp2_fast((to_f32(as_elems<T, E>(v[u]).v[e]) - st.m) * a.c));
            if (wide) {
                put16<(TH > kWave)>(out + i, &o);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) g[rs.head + i * E + e] = o.v[e];
            }
        }
        if (has_loose) g[rs.at(threadIdx.x)] = from_f32<T>(s * exp2_fast((loose - st.m) * a.c));
        __syncthreads();
        fix_entries<T, TH>(a, g, rs, 0, rs.nb, true, sh, st, w);
    }
}

// Rows longer than that: the row is read twice, the second time out of the caches where they hold it.
template <class T, int TH>
__global__ __launch_bounds__(TH) void distill_long_kernel(const DistillArgs a) {
    __shared__ Entries sh;
    const int64_t row = blockIdx.x;
    const T *z = (const T *)a.z + row * a.ldz;
    T *g = (T *)a.grad + row * a.ldg;
    const RowShape<T> rs(z, a.V);
    load_entries(a, row, z, nullptr, sh);
    const MaxSum st = block_join<TH>(scan_row<T, TH, 4>(z, rs, 0, rs.nb, true, a.c), a.c, sh.red);
    __syncthreads();
    entries_loss(a, row, sh, st);
    if (distill_empty(sh, st)) {
        zero_row<T, TH>(g, rs, 0, rs.nb, true);
        return;
    }
    const float w = a.row_w ? a.row_w[row] : 1.f;
    write_row<T, TH, 4>(z, g, rs, 0, rs.nb, true, st.m, a.c, w * a.T / st.s, -1, 0.f);
    __syncthreads();
    fix_entries<T, TH>(a, g, rs, 0, rs.nb, true, sh, st, w);
}

// Few rows: S workgroups share one.  First launch: (m, s) of each part; part 0 keeps the entries' logits.
template <class T, int TH>
__global__ __launch_bounds__(TH) void distill_part_kernel(const DistillArgs a) {
    __shared__ MaxSum red[TH / kWave];
    const int64_t row = blockIdx.y;
    const T *z = (const T *)a.z + row * a.ldz;
    const RowShape<T> rs(z, a.V);
    int c0, c1;
    part_of(rs.nb, blockIdx.x, gridDim.x, c0, c1);
    const MaxSum st = block_join<TH>(scan_row<T, TH, 4>(z, rs, c0, c1, blockIdx.x == 0, a.c), a.c, red);
    if (threadIdx.x == 0) a.part[row * gridDim.x + blockIdx.x] = st;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.k; i += TH) {
            const int64_t j = a.idx[row * a.k + i];
            a.zt[row * a.k + i] = j >= 0 && j < a.V ? to_f32(z[j]) : 0.f;
        }
}

// The parts of a row, joined in their order by every wave.
__device__ __forceinline__ MaxSum join_parts(const MaxSum *part, int S, float c) {
    const int lane = threadIdx.x & 63;
    MaxSum v{-INFINITY, 0.f};
    if (lane < S) v = part[lane];  // S <= 64
    return wave_join(v, c);
}

// Second launch: a part's gradient.  Also the backward form, from (m, s) of an earlier call.
template <class T, int TH, bool PARTS>
__global__ __launch_bounds__(TH) void distill_grad_kernel(const DistillArgs a) {
    __shared__ Entries sh;
    const int64_t row = blockIdx.y;
    const T *z = (const T *)a.z + row * a.ldz;
    T *g = (T *)a.grad + row * a.ldg;
    const RowShape<T> rs(z, a.V);
    load_entries(a, row, z, PARTS ? a.zt : nullptr, sh);
    MaxSum st;
    if constexpr (PARTS) st = join_parts(a.part + row * gridDim.x, gridDim.x, a.c);
    else st = MaxSum{a.stats[2 * row], a.stats[2 * row + 1]};
    __syncthreads();
    if constexpr (PARTS)
        if (blockIdx.x == 0) entries_loss(a, row, sh, st);
    if (!a.grad) return;
    int c0, c1;
    part_of(rs.nb, blockIdx.x, gridDim.x, c0, c1);
    const bool loose = blockIdx.x == 0;
    if (distill_empty(sh, st)) {
        zero_row<T, TH>(g, rs, c0, c1, loose);
        return;
    }
    const float w = a.row_w ? a.row_w[row] : 1.f;
    write_row<T, TH, 4>(z, g, rs, c0, c1, loose, st.m, a.c, w * a.T / st.s, -1, 0.f);
    __syncthreads();
    fix_entries<T, TH>(a, g, rs, c0, c1, loose, sh, st, w);
}

// ---- log-probabilities of targets and the preference loss ---------------------------------------------------------------

struct LogpArgs {
    const void *z;
    int64_t ldz;
    int V;
    const int64_t *targets;
    float *logp;         // either
    double *logp64;      // or
    float *coef;         // set to 0 when given
    float *stats;        // [m][2]
    MaxSum *part;        // [m][S] when a row is split
};

__device__ __forceinline__ void store_logp(const LogpArgs &a, int64_t row, bool there, float zt, MaxSum st) {
    double l = 0.0;
    if (there && !(st.m == -INFINITY && st.s == 0.f)) l = ((double)zt - (double)st.m) - log((double)st.s);
    if (a.logp) a.logp[row] = (float)l;
    if (a.logp64) a.logp64[row] = l;
    if (a.coef) a.coef[row] = 0.f;
    if (a.stats) a.stats[2 * row] = st.m, a.stats[2 * row + 1] = st.s;
}

constexpr float kLog2e = 1.44269504088896340736f;

// One workgroup per row and part; a row without a target is not read.  Bound by the reads: 252 MB (4 096 x 40 982 bf16, a quarter
// without a target) in 43 us = 5.9 TB/s, 1.18 GB (6 001 x 131 072 fp16) in 196 = 6.0.
template <class T, int TH, bool PARTS>
__global__ __launch_bounds__(TH) void logp_kernel(const LogpArgs a) {
    __shared__ MaxSum red[TH / kWave];
    const int64_t row = PARTS ? blockIdx.y : blockIdx.x;
    const int64_t t = a.targets[row];
    const bool there = t >= 0 && t < a.V;
    const T *z = (const T *)a.z + row * a.ldz;
    MaxSum st{-INFINITY, 0.f};
    if (there) {
        const RowShape<T> rs(z, a.V);
        int c0 = 0, c1 = rs.nb;
        if constexpr (PARTS) part_of(rs.nb, blockIdx.x, gridDim.x, c0, c1);
        st = block_join<TH>(scan_row<T, TH, 4>(z, rs, c0, c1, !PARTS || blockIdx.x == 0, kLog2e), kLog2e, red);
    }
    if (threadIdx.x) return;
    if constexpr (PARTS) a.part[row * gridDim.x + blockIdx.x] = st;
    else store_logp(a, row, there, there ? to_f32(z[t]) : 0.f, st);
}

template <class T>
__global__ __launch_bounds__(kWave) void logp_join_kernel(const LogpArgs a, int S) {
    const int64_t row = blockIdx.x;
    const int64_t t = a.targets[row];
    const bool there = t >= 0 && t < a.V;
    const MaxSum st = join_parts(a.part + row * S, S, kLog2e);
    if (threadIdx.x == 0) store_logp(a, row, there, there ? to_f32(((const T *)a.z + row * a.ldz)[t]) : 0.f, st);
}

// Part `part` of `parts` of a row's gradient w (onehot - softmax), by TH threads; a row of gradient 0 is not read.
template <class T, int TH>
__device__ __forceinline__ void grad_row(const void *zv, int64_t ldz, int V, const int64_t *targets, const float *stats, int64_t row, float w,
                                         void *gv, int64_t ldg, int part, int parts) {
    const int64_t t = targets[row];
    const T *z = (const T *)zv + row * ldz;
    T *g = (T *)gv + row * ldg;
    const RowShape<T> rs(z, V);
    int c0, c1;
    part_of(rs.nb, part, parts, c0, c1);
    const bool loose = part == 0;
    bool none = t < 0 || t >= V || w == 0.f;
    float m = 0.f, s = 0.f;
    if (!none) {
        m = stats[2 * row], s = stats[2 * row + 1];
        none = m == -INFINITY && s == 0.f;
    }
    if (none) zero_row<T, TH>(g, rs, c0, c1, loose);
    else write_row<T, TH, 4>(z, g, rs, c0, c1, loose, m, kLog2e, -w / s, (int)t, w);
}

template <class T, int TH>
__device__ __forceinline__ void clear_row(const void *zv, int64_t ldz, int V, int64_t row, void *gv, int64_t ldg) {
    const RowShape<T> rs((const T *)zv + row * ldz, V);
    zero_row<T, TH>((T *)gv + row * ldg, rs, 0, rs.nb, true);
}

// One workgroup per row and part; row = the last one first: what the pass before read last is what the caches still hold.  Bound by
// memory: at the sizes above 252 MB read and 336 MB written in 84 us = 7.0 TB/s, much of the reads out of the caches, and 1.18 + 1.57 GB
// in 485 = 5.7.
template <class T, int TH>
__global__ __launch_bounds__(TH) void logp_grad_kernel(const void *z, int64_t ldz, int V, const int64_t *targets, const float *stats,
                                                       const float *row_g, void *g, int64_t ldg) {
    const int64_t row = (int64_t)gridDim.y - 1 - blockIdx.y;
    grad_row<T, TH>(z, ldz, V, targets, stats, row, row_g[row], g, ldg, blockIdx.x, gridDim.x);
}

// A pair's margin h, its loss and d loss / d h are held in 64 bits and rounded once each: they are few, and a margin rounded to 32 bits costs
// a loss of exp(-h) |h| steps.  With t = exp(-|h|): sigmoid(|h|) = 1 / (1 + t), sigmoid(-|h|) = t / (1 + t).
__device__ __forceinline__ double sigmoid_d(double h, double smoothing) {  // d loss / d margin
    const double t = exp(-fabs(h)), r = 1.0 / (1.0 + t);
    const double up = h < 0.0 ? t * r : r, down = h < 0.0 ? r : t * r;  // sigmoid(h), sigmoid(-h)
    return smoothing * up - (1.0 - smoothing) * down;
}

// -log sigmoid(x) = max(-x, 0) + log(1 + exp(-|x|)); a term of weight 0 is left out (its value may be infinite).
__device__ __forceinline__ void store_pair(double h, double smoothing, float *loss, float *margin) {
    const double l = log1p(exp(-fabs(h)));
    double v = 0.0;
    if (smoothing < 1.0) v += (1.0 - smoothing) * (fmax(-h, 0.0) + l);
    if (smoothing > 0.0) v += smoothing * (fmax(h, 0.0) + l);
    *loss = (float)(h != h ? h : v);
    *margin = (float)h;
}

__device__ __forceinline__ void seq_of(const int64_t *offsets, int64_t s, int64_t m, int64_t &lo, int64_t &hi) {
    lo = offsets[s], hi = offsets[s + 1];
    lo = lo < 0 ? 0 : lo > m ? m : lo;
    hi = hi < lo ? lo : hi > m ? m : hi;
}

// The margin of a pair, by the TH threads of a workgroup: both sequences as one list of tokens, 4 TH in flight, both sums in 64 bits.
template <class L, int TH>
__device__ __forceinline__ double pair_margin(const L *logp, int64_t m, const int64_t *offsets, const float *ref, int64_t i, float beta,
                                             int64_t (&lo)[2], int64_t (&hi)[2], double (&red)[2][TH / kWave]) {
    seq_of(offsets, 2 * i, m, lo[0], hi[0]);
    seq_of(offsets, 2 * i + 1, m, lo[1], hi[1]);
    const float r0 = ref[2 * i], r1 = ref[2 * i + 1];
    const int64_t first = hi[0] - lo[0], all = first + hi[1] - lo[1], skip = lo[1] - first;
    double v[2] = {0.0, 0.0};
    for (int64_t u0 = threadIdx.x; u0 < all; u0 += 4 * TH) {
        double l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t u = u0 + TH * q;
            l[q] = u < all ? (double)logp[u + (u < first ? lo[0] : skip)] : 0.0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool second = u0 + TH * q >= first;
            v[0] += second ? 0.0 : l[q], v[1] += second ? l[q] : 0.0;
        }
    }
    double sum[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        sum[k] = wave_sum(v[k]);
        if constexpr (TH > kWave)
            if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = sum[k];
    }
    if constexpr (TH > kWave) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sum[k] = red[k][0];
#pragma unroll
            for (int q = 1; q < TH / kWave; ++q) sum[k] += red[k][q];
        }
    }
    return (double)beta * ((sum[0] - (double)r0) - (sum[1] - (double)r1));
}

// One workgroup per pair: the loss, and (COEF) the tokens' gradients of pair_w loss.  Bound by latency (4 096 tokens of 32 pairs 5 us,
// 6 001 of two 8).
template <class L, bool COEF>
__global__ __launch_bounds__(256) void pair_kernel(const L *logp, int64_t m, const int64_t *offsets, const float *ref, float beta,
                                                   float smoothing, const float *pair_w, float *loss, float *margin, float *coef) {
    __shared__ double red[2][4];
    const int64_t i = blockIdx.x;
    int64_t lo[2], hi[2];
    const double h = pair_margin<L, 256>(logp, m, offsets, ref, i, beta, lo, hi, red);
    if (threadIdx.x == 0) store_pair(h, smoothing, loss + i, margin + i);
    if constexpr (COEF) {
        const float d = (float)((double)beta * sigmoid_d(h, smoothing) * (pair_w ? (double)pair_w[i] : 1.0));
#pragma unroll
        for (int k = 0; k < 2; ++k)
            for (int64_t t = lo[k] + threadIdx.x; t < hi[k]; t += 256) coef[t] = k ? -d : d;
    }
}

// Pairs and gradients in one launch, for few tokens: the workgroups of a row find its sequence (the last one that begins at or before it)
// and form their pair's margin for themselves, which reads kFusedTokens log-probabilities at most; one workgroup per pair behind the
// rows' (blockIdx.y >= m, part 0) writes its loss.
constexpr int64_t kFusedTokens = 1024, kFusedPairs = 256;

template <class T, int TH>
__global__ __launch_bounds__(TH) void pair_rows_kernel(const LogpArgs a, int64_t m, const int64_t *offsets, int64_t pairs, const float *ref,
                                                       float beta, float smoothing, const float *pair_w, float *loss, float *margin, void *gv,
                                                       int64_t ldg) {
    __shared__ double red[2][TH / kWave];
    int64_t lo[2], hi[2];
    if (blockIdx.y >= m) {
        if (blockIdx.x) return;
        const int64_t i = blockIdx.y - m;
        const double h = pair_margin<double, TH>(a.logp64, m, offsets, ref, i, beta, lo, hi, red);
        if (threadIdx.x == 0) store_pair(h, smoothing, loss + i, margin + i);
        return;
    }
    const int64_t row = blockIdx.y, t = a.targets[row];
    float w = 0.f;
    if (t >= 0 && t < a.V) {
        int before = 0;  // offsets at or before the row
        for (int64_t c = threadIdx.x & 63; c - (threadIdx.x & 63) <= 2 * pairs; c += 64)
            before += __popcll(__ballot(c <= 2 * pairs && offsets[min(c, 2 * pairs)] <= row));
        if (before > 0 && before <= 2 * pairs) {
            const int64_t i = (before - 1) >> 1;
            const double h = pair_margin<double, TH>(a.logp64, m, offsets, ref, i, beta, lo, hi, red);
            const float d = (float)((double)beta * sigmoid_d(h, smoothing) * (pair_w ? (double)pair_w[i] : 1.0));
            w = (before - 1) & 1 ? -d : d;
        }
    }
    grad_row<T, TH>(a.z, a.ldz, a.V, a.targets, a.stats, row, w, gv, ldg, blockIdx.x, gridDim.x);
}

// Small calls in one launch: a workgroup per pair, a wave per row.  Both sums meet in LDS, and the rows, read a second time for their
// gradient, are still in the caches.  (m, S) of a row stays with the wave that goes on to write it.  Bound by that chain of latencies: 40
// tokens of 1 683 fp32 logits in 10.8 us.
template <class T>
__global__ __launch_bounds__(1024) void pair_small_kernel(const LogpArgs a, int64_t m, const int64_t *offsets, const float *ref, float beta,
                                                          float smoothing, const float *pair_w, float *loss, float *margin, void *gv, int64_t ldg) {
    __shared__ double red[2][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t i = blockIdx.x;
    int64_t lo[2], hi[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        seq_of(offsets, 2 * i + k, m, lo[k], hi[k]);
        double sum = 0.0;
        for (int64_t row = lo[k] + w; row < hi[k]; row += 16) {
            const int64_t t = a.targets[row];
            if (t < 0 || t >= a.V) continue;
            const T *z = (const T *)a.z + row * a.ldz;
            const RowShape<T> rs(z, a.V);
            const float zt = to_f32(z[t]);
            const MaxSum st = wave_join(scan_row<T, kWave, 4>(z, rs, 0, rs.nb, true, kLog2e), kLog2e);
            if (lane == 0) a.stats[2 * row] = st.m, a.stats[2 * row + 1] = st.s;
            if (!(st.m == -INFINITY && st.s == 0.f)) sum += ((double)zt - (double)st.m) - log((double)st.s);
        }
        if (lane == 0) red[k][w] = sum;
    }
    __syncthreads();
    double sum[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        sum[k] = 0.0;
#pragma unroll
        for (int q = 0; q < 16; ++q) sum[k] += red[k][q];
        sum[k] -= (double)ref[2 * i + k];
    }
    const double h = (double)beta * (sum[0] - sum[1]);
    if (threadIdx.x == 0) store_pair(h, smoothing, loss + i, margin + i);
    const float d = (float)((double)beta * sigmoid_d(h, smoothing) * (pair_w ? (double)pair_w[i] : 1.0));
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (int64_t row = lo[k] + w; row < hi[k]; row += 16)
            grad_row<T, kWave>(a.z, a.ldz, a.V, a.targets, a.stats, row, k ? -d : d, gv, ldg, 0, 1);
    // rows in front of the first sequence and behind the last
    const int64_t r0 = i == 0 ? 0 : hi[1], r1 = i == 0 ? lo[0] : m;
    if (i == 0 || i + 1 == gridDim.x)
        for (int64_t row = r0 + w; row < r1; row += 16) clear_row<T, kWave>(a.z, a.ldz, a.V, row, gv, ldg);
    if (i == 0 && gridDim.x == 1)
        for (int64_t row = hi[1] + w; row < m; row += 16) clear_row<T, kWave>(a.z, a.ldz, a.V, row, gv, ldg);
}

// grad_logp of every token: its sequence is found by bisection (the last one that begins at or before it and is not empty).
__global__ __launch_bounds__(256) void pair_grad_kernel(const float *margin, int64_t m, const int64_t *offsets, int64_t pairs, float beta,
                                                        float smoothing, const float *g_loss, const float *g_margin, float *grad) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= m) return;
    int64_t lo = 0, hi = 2 * pairs;  // offsets[lo] <= t < offsets[hi], if t is in a sequence
    double v = 0.0;
    if (offsets[0] <= t && t < offsets[hi]) {
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (offsets[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int64_t i = lo >> 1;
        if (g_loss) v += (double)g_loss[i] * sigmoid_d(margin[i], smoothing);
        if (g_margin) v += (double)g_margin[i];
        v *= lo & 1 ? -(double)beta : (double)beta;
    }
    grad[t] = (float)v;
}

// ---- host ----------------------------------------------------------------------------------------------------------------

// How many workgroups share a row: one where the rows alone give every CU two; else enough for about four per CU, of at least 4 096
// elements each.  (64 parts at most: one wave joins them.)
static int row_parts(int64_t n, int64_t V) {
    if (n >= 512) return 1;
    const int64_t want = std::min<int64_t>((1024 + n - 1) / std::max<int64_t>(n, 1), V / 4096);
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, 64));
}

static int64_t round16(int64_t b) { return (b + 15) & ~int64_t(15); }

// Workgroups per row of a pass that needs nothing from the rest of the row: 256 threads x 4 chunks each.
static int grad_parts(int64_t V, int elem) { return (int)std::max<int64_t>(1, std::min<int64_t>((V * elem + 16383) / 16384, 1024)); }

static int check_rows(const void *z, int64_t ldz, int dtype, int64_t n, int64_t V) {
    if (!elem_ok(dtype)) return fail(RBG_EINVAL, "dtype = %d", dtype);
    if (n < 0 || V <= 0 || ldz < V) return fail(RBG_ESHAPE, "n = %lld, V = %lld, ldz = %lld", (long long)n, (long long)V, (long long)ldz);
    if (V > 0x7fffff00ll || n > 0x7fffffffll) return fail(RBG_EUNSUPPORTED, "rows or columns beyond 2^31");
    if (n && !z) return fail(RBG_EINVAL, "NULL pointer");
    if (reinterpret_cast<uintptr_t>(z) % elem_size(dtype)) return fail(RBG_EINVAL, "logits are not aligned to their type");
    return RBG_OK;
}

// A gradient is written to rows of its own or, element for element, to the rows it is computed from.
static int check_grad(const void *z, int64_t ldz, int dtype, int64_t n, int64_t V, const void *g, int64_t ldg) {
    if (ldg < V) return fail(RBG_ESHAPE, "V = %lld, ldg = %lld", (long long)V, (long long)ldg);
    if (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) return fail(RBG_EINVAL, "the gradient is not aligned to its type");
    if (g == z) return ldg == ldz ? RBG_OK : fail(RBG_EINVAL, "a gradient in place of the logits needs their row stride");
    const uintptr_t z0 = (uintptr_t)z, g0 = (uintptr_t)g;
    const uintptr_t z1 = z0 + (uintptr_t)((n - 1) * ldz + V) * elem_size(dtype), g1 = g0 + (uintptr_t)((n - 1) * ldg + V) * elem_size(dtype);
    if (z0 < g1 && g0 < z1) return fail(RBG_EINVAL, "the gradient overlaps the logits");
    return RBG_OK;
}

// S: row_parts of the whole call, which its workspace is sized for (a call's last slice of rows may be short).
template <class T>
static int launch_distill_rows(const DistillArgs &a, int64_t n, int64_t V, int S, hipStream_t s) {
    if (S > 1) {
        hipLaunchKernelGGL((distill_part_kernel<T, 256>), dim3(S, (unsigned)n), dim3(256), 0, s, a);
        hipLaunchKernelGGL((distill_grad_kernel<T, 256, true>), dim3(S, (unsigned)n), dim3(256), 0, s, a);
    } else if (!a.grad) {
        if (V * (int64_t)sizeof(T) <= 4096) hipLaunchKernelGGL((distill_eval_kernel<T, 64>), dim3((unsigned)n), dim3(64), 0, s, a);
        else hipLaunchKernelGGL((distill_eval_kernel<T, 256>), dim3((unsigned)n), dim3(256), 0, s, a);
    } else {
        const int64_t chunks = V * (int64_t)sizeof(T) / 16;  // at most this many whole ones
        // The smallest that holds the row; the next one up costs (us, bf16): 4 096 x 2 048 12.5 -> 16, 4 096 x 8 192 29 -> 33, 2 048 x 16 384
        // 28.5 -> 30, x 28 672 42 -> 44, x 40 982 62 -> 67, 1 024 x 65 536 46 -> 48, x 91 600 67 -> 84; a row read twice instead (fp32)
        // 1 024 x 91 600 149 -> 182.
        const dim3 grid((unsigned)n);
        if (chunks <= 64 * 4) hipLaunchKernelGGL((distill_row_kernel<T, 64, 4>), grid, dim3(64), 0, s, a);
        else if (chunks <= 256 * 4) hipLaunchKernelGGL((distill_row_kernel<T, 256, 4>), grid, dim3(256), 0, s, a);
        else if (chunks <= 512 * 4) hipLaunchKernelGGL((distill_row_kernel<T, 512, 4>), grid, dim3(512), 0, s, a);
        else if (chunks <= 512 * 7) hipLaunchKernelGGL((distill_row_kernel<T, 512, 7>), grid, dim3(512), 0, s, a);
        else if (chunks <= 512 * 11) hipLaunchKernelGGL((distill_row_kernel<T, 512, 11>), grid, dim3(512), 0, s, a);
        else if (chunks <= 512 * 16) hipLaunchKernelGGL((distill_row_kernel<T, 512, 16>), grid, dim3(512), 0, s, a);
        else if (chunks <= 512 * 24) hipLaunchKernelGGL((distill_row_kernel<T, 512, 24>), grid, dim3(512), 0, s, a);
        else if (chunks <= 1024 * 24) hipLaunchKernelGGL((distill_row_kernel<T, 1024, 24>), grid, dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((distill_long_kernel<T, 1024>), grid, dim3(1024), 0, s, a);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

template <class T>
static int launch_distill(const DistillArgs &a, int64_t n, int64_t V, int S, hipStream_t s) {
    for (int64_t r0 = 0; r0 < n; r0 += kRowsPerLaunch) {
        DistillArgs p = a;
        p.z = (const T *)a.z + r0 * a.ldz, p.idx += r0 * a.k, p.val += r0 * a.k, p.loss += r0;
        if (a.row_w) p.row_w += r0;
        if (a.stats) p.stats += 2 * r0;
        if (a.grad) p.grad = (T *)a.grad + r0 * a.ldg;
        if (int rc = launch_distill_rows<T>(p, std::min(kRowsPerLaunch, n - r0), V, S, s)) return rc;
    }
    return RBG_OK;
}

template <class T>
static int launch_logp_rows(const LogpArgs &a, int64_t m, int64_t V, int S, hipStream_t s) {
    if (S > 1) {
        hipLaunchKernelGGL((logp_kernel<T, 256, true>), dim3(S, (unsigned)m), dim3(256), 0, s, a);
        hipLaunchKernelGGL((logp_join_kernel<T>), dim3((unsigned)m), dim3(64), 0, s, a, S);
    } else if (V * (int64_t)sizeof(T) <= 4096) {
        hipLaunchKernelGGL((logp_kernel<T, 64, false>), dim3((unsigned)m), dim3(64), 0, s, a);
    } else {
        hipLaunchKernelGGL((logp_kernel<T, 256, false>), dim3((unsigned)m), dim3(256), 0, s, a);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

template <class T>
static int launch_logp(const LogpArgs &a, int64_t m, int64_t V, hipStream_t s) {
    const int S = row_parts(m, V);  // the whole call's, as its workspace
    for (int64_t r0 = 0; r0 < m; r0 += kRowsPerLaunch) {
        LogpArgs p = a;
        p.z = (const T *)a.z + r0 * a.ldz, p.targets += r0;
        if (a.logp) p.logp += r0;
        if (a.logp64) p.logp64 += r0;
        if (a.coef) p.coef += r0;
        if (a.stats) p.stats += 2 * r0;
        if (int rc = launch_logp_rows<T>(p, std::min(kRowsPerLaunch, m - r0), V, S, s)) return rc;
    }
    return RBG_OK;
}

template <class L, bool COEF>
static int launch_pairs(const L *logp, int64_t m, const int64_t *offsets, int64_t pairs, const float *ref, float beta, float smoothing,
                        const float *pair_w, float *loss, float *margin, float *coef, hipStream_t s) {
    for (int64_t i0 = 0; i0 < pairs; i0 += kRowsPerLaunch)
        hipLaunchKernelGGL((pair_kernel<L, COEF>), dim3((unsigned)std::min(kRowsPerLaunch, pairs - i0)), dim3(256), 0, s, logp, m, offsets + 2 * i0,
                           ref + 2 * i0, beta, smoothing, pair_w ? pair_w + i0 : nullptr, loss + i0, margin + i0, coef);
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

// A grid's y dimension ends at 65 535: the rows go in slices of that.
constexpr int64_t kMaxGridY = 65535;

template <class T>
static int launch_logp_grad(const T *z, int64_t ldz, int64_t m, int64_t V, const int64_t *targets, const float *stats, const float *row_g,
                            T *g, int64_t ldg, hipStream_t s) {
    const int S = grad_parts(V, sizeof(T));
    const int64_t slices = (m + kMaxGridY - 1) / kMaxGridY;
    for (int64_t k = slices - 1; k >= 0; --k) {
        const int64_t r0 = k * kMaxGridY, cnt = std::min(kMaxGridY, m - r0);
        const dim3 grid(S, (unsigned)cnt);
        if (V * (int64_t)sizeof(T) <= 4096)
            hipLaunchKernelGGL((logp_grad_kernel<T, 64>), grid, dim3(64), 0, s, z + r0 * ldz, ldz, (int)V, targets + r0, stats + 2 * r0,
                               row_g + r0, g + r0 * ldg, ldg);
        else
            hipLaunchKernelGGL((logp_grad_kernel<T, 256>), grid, dim3(256), 0, s, z + r0 * ldz, ldz, (int)V, targets + r0, stats + 2 * r0,
                               row_g + r0, g + r0 * ldg, ldg);
    }
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

static int check_pairs(int64_t m, const int64_t *offsets, int64_t pairs, float beta, float smoothing) {
    if (m < 0 || pairs < 0 || pairs > 0x3fffffff || m > 0x7fffffffll) return fail(RBG_ESHAPE, "m = %lld, pairs = %lld", (long long)m, (long long)pairs);
    if (!std::isfinite(beta) || !(smoothing >= 0.f && smoothing <= 1.f)) return fail(RBG_EINVAL, "beta = %g, smoothing = %g", beta, smoothing);
    if (!offsets) return fail(RBG_EINVAL, "NULL pointer");
    return RBG_OK;
}

}  // namespace rbg

using namespace rbg;

extern "C" {

int rbg_distill_topk_workspace(int64_t n, int64_t V, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(RBG_EINVAL, "bytes is NULL");
    if (n < 0 || V <= 0) return fail(RBG_ESHAPE, "n = %lld, V = %lld", (long long)n, (long long)V);
    const int S = row_parts(n, V);
    *bytes = S > 1 ? round16(n * S * (int64_t)sizeof(MaxSum)) + round16(n * kMaxEntries * 4) : 0;
    return RBG_OK;
}

int rbg_distill_topk(const void *z, int64_t ldz, int dtype, int64_t n, int64_t V, const int64_t *idx, const float *val, int k, float T,
                     const float *row_w, float *loss, float *stats, void *grad, int64_t ldg, void *workspace, void *stream) {
    clear_error();
    if (int rc = check_rows(z, ldz, dtype, n, V)) return rc;
    if (k < 1 || k > kMaxEntries) return fail(RBG_EUNSUPPORTED, "k = %d: 1 to %d entries per row", k, kMaxEntries);
    if (!(T >= 1e-15f && T <= 1e15f)) return fail(RBG_EINVAL, "T = %g", T);  // (1 / T and T^2 stay normal numbers)
    if (n == 0) return RBG_OK;
    if (!idx || !val || !loss || (!workspace && row_parts(n, V) > 1)) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(workspace)) return fail(RBG_EINVAL, "workspace is not 16-byte aligned");
    if (grad)
        if (int rc = check_grad(z, ldz, dtype, n, V, grad, ldg)) return rc;
    const int S = row_parts(n, V);
    DistillArgs a{z, ldz, (int)V, k, idx, val, (float)(1.4426950408889634 / (double)T), T, row_w, loss, stats, grad, ldg, (MaxSum *)workspace,
                  (float *)((char *)workspace + round16(n * S * (int64_t)sizeof(MaxSum)))};
    return with_elem(dtype, [&](auto t) { return launch_distill<decltype(t)>(a, n, V, S, (hipStream_t)stream); });
}

int rbg_distill_topk_backward(const void *z, int64_t ldz, int dtype, int64_t n, int64_t V, const int64_t *idx, const float *val, int k,
                              float T, const float *stats, const float *row_w, void *grad, int64_t ldg, void *stream) {
    clear_error();
    if (int rc = check_rows(z, ldz, dtype, n, V)) return rc;
    if (k < 1 || k > kMaxEntries) return fail(RBG_EUNSUPPORTED, "k = %d: 1 to %d entries per row", k, kMaxEntries);
    if (!(T >= 1e-15f && T <= 1e15f)) return fail(RBG_EINVAL, "T = %g", T);
    if (n == 0) return RBG_OK;
    if (!idx || !val || !stats || !grad) return fail(RBG_EINVAL, "NULL pointer");
    if (int rc = check_grad(z, ldz, dtype, n, V, grad, ldg)) return rc;
    const int S = grad_parts(V, elem_size(dtype));
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        for (int64_t r0 = 0; r0 < n; r0 += kMaxGridY) {
            const DistillArgs a{(const E *)z + r0 * ldz, ldz, (int)V, k, idx + r0 * k, val + r0 * k, (float)(1.4426950408889634 / (double)T), T,
                                row_w ? row_w + r0 : nullptr, nullptr, const_cast<float *>(stats) + 2 * r0, (E *)grad + r0 * ldg, ldg, nullptr, nullptr};
            const dim3 grid(S, (unsigned)std::min(kMaxGridY, n - r0));
            hipLaunchKernelGGL((distill_grad_kernel<E, 256, false>), grid, dim3(256), 0, (hipStream_t)stream, a);
        }
        RBG_HIP(hipGetLastError());
        return (int)RBG_OK;
    });
}

int rbg_token_logp_workspace(int64_t m, int64_t V, int64_t *bytes) {
    clear_error();
    if (!bytes) return fail(RBG_EINVAL, "bytes is NULL");
    if (m < 0 || V <= 0) return fail(RBG_ESHAPE, "m = %lld, V = %lld", (long long)m, (long long)V);
    const int S = row_parts(m, V);
    *bytes = S > 1 ? round16(m * S * (int64_t)sizeof(MaxSum)) : 0;
    return RBG_OK;
}

int rbg_token_logp(const void *z, int64_t ldz, int dtype, int64_t m, int64_t V, const int64_t *targets, float *logp, float *stats,
                   void *workspace, void *stream) {
    clear_error();
    if (int rc = check_rows(z, ldz, dtype, m, V)) return rc;
    if (m == 0) return RBG_OK;
    if (!targets || !logp || (!workspace && row_parts(m, V) > 1)) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(workspace)) return fail(RBG_EINVAL, "workspace is not 16-byte aligned");
    const LogpArgs a{z, ldz, (int)V, targets, logp, nullptr, nullptr, stats, (MaxSum *)workspace};
    return with_elem(dtype, [&](auto t) { return launch_logp<decltype(t)>(a, m, V, (hipStream_t)stream); });
}

int rbg_token_logp_backward(const void *z, int64_t ldz, int dtype, int64_t m, int64_t V, const int64_t *targets, const float *stats,
                            const float *row_g, void *grad, int64_t ldg, void *stream) {
    clear_error();
    if (int rc = check_rows(z, ldz, dtype, m, V)) return rc;
    if (m == 0) return RBG_OK;
    if (!targets || !stats || !row_g || !grad) return fail(RBG_EINVAL, "NULL pointer");
    if (int rc = check_grad(z, ldz, dtype, m, V, grad, ldg)) return rc;
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        return launch_logp_grad<E>((const E *)z, ldz, m, V, targets, stats, row_g, (E *)grad, ldg, (hipStream_t)stream);
    });
}

int rbg_preference_loss(const float *logp, int64_t m, const int64_t *offsets, int64_t pairs, const float *ref, float beta, float smoothing,
                        float *loss, float *margin, void *stream) {
    clear_error();
    if (int rc = check_pairs(m, offsets, pairs, beta, smoothing)) return rc;
    if (pairs == 0) return RBG_OK;
    if ((m && !logp) || !ref || !loss || !margin) return fail(RBG_EINVAL, "NULL pointer");
    return launch_pairs<float, false>(logp, m, offsets, pairs, ref, beta, smoothing, nullptr, loss, margin, nullptr, (hipStream_t)stream);
}

int rbg_preference_loss_backward(const float *margin, int64_t m, const int64_t *offsets, int64_t pairs, float beta, float smoothing,
                                 const float *g_loss, const float *g_margin, float *grad_logp, void *stream) {
    clear_error();
    if (int rc = check_pairs(m, offsets, pairs, beta, smoothing)) return rc;
    if (m == 0) return RBG_OK;
    if ((pairs && !margin) || !grad_logp) return fail(RBG_EINVAL, "NULL pointer");
    hipLaunchKernelGGL(pair_grad_kernel, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, (hipStream_t)stream, margin, m, offsets, pairs, beta,
                       smoothing, g_loss, g_margin, grad_logp);
    RBG_HIP(hipGetLastError());
    return RBG_OK;
}

int rbg_preference_grad_workspace(int64_t m, int64_t V, int64_t *bytes) {
    if (int rc = rbg_token_logp_workspace(m, V, bytes)) return rc;
    *bytes += round16(8 * m) + round16(8 * m) + round16(4 * m);  // logp in 64 bits, (m, S), the tokens' coefficients
    return RBG_OK;
}

int rbg_preference_grad(const void *z, int64_t ldz, int dtype, int64_t m, int64_t V, const int64_t *targets, const int64_t *offsets,
                        int64_t pairs, const float *ref, float beta, float smoothing, const float *pair_w, float *loss, float *margin,
                        void *grad, int64_t ldg, void *workspace, void *stream) {
    clear_error();
    if (int rc = check_rows(z, ldz, dtype, m, V)) return rc;
    if (int rc = check_pairs(m, offsets, pairs, beta, smoothing)) return rc;
    if (m == 0 && pairs == 0) return RBG_OK;
    if ((pairs && (!ref || !loss || !margin)) || (m && (!targets || !grad || !workspace))) return fail(RBG_EINVAL, "NULL pointer");
    if (!on_16(workspace)) return fail(RBG_EINVAL, "workspace is not 16-byte aligned");
    if (m)
        if (int rc = check_grad(z, ldz, dtype, m, V, grad, ldg)) return rc;
    hipStream_t s = (hipStream_t)stream;
    char *w = (char *)workspace;
    double *logp = (double *)w;
    float *stats = (float *)(w + round16(8 * m));
    float *coef = (float *)(w + 2 * round16(8 * m));
    MaxSum *part = (MaxSum *)(w + 2 * round16(8 * m) + round16(4 * m));
    return with_elem(dtype, [&](auto t) {
        typedef decltype(t) E;
        // Up to 256 tokens, 64 and 128 KB a pair, rows of 16 KB and 1 MB in all: one launch instead of three (40 x 1 683 fp32, four
        // pairs: 13 us a call, 19 with three).  A workgroup takes a pair's rows sixteen at a time, a wave each, and the lengths are on the
        // device: all tokens in one pair cost 16 turns of it at most (4 756 tokens of two pairs would take 560 us), and a wave
        // reads a row of 16 KB in four turns (one of 500 KB would take 80 us).
        const int64_t total = m * V * (int64_t)sizeof(E);
        if (m && m <= 256 && m <= pairs * 64 && pairs <= kRowsPerLaunch && V * (int64_t)sizeof(E) <= 16 << 10 && total <= 1 << 20 && total <= pairs << 17) {
            const LogpArgs a{z, ldz, (int)V, targets, nullptr, nullptr, nullptr, stats, nullptr};
            hipLaunchKernelGGL((pair_small_kernel<E>), dim3((unsigned)pairs), dim3(1024), 0, s, a, m, offsets, ref, beta, smoothing, pair_w, loss, margin,
                               grad, ldg);
            RBG_HIP(hipGetLastError());
            return (int)RBG_OK;
        }
        // Pairs and gradients in one launch: 870 x 135 bf16, 40 pairs, 16.1 us a call against 18.4; 883 x 5 178 fp32, 10 pairs, 16.3 against
        // 18.3; but 1 000 x 40 000 bf16, 200 pairs (80 MB), 41.3 against 39.4, and 1 024 x 131 072 fp32, one pair, 252 against 228.
        const bool fused = m && m <= kFusedTokens && pairs <= kFusedPairs && total <= 32 << 20;
        if (m) {
            const LogpArgs a{z, ldz, (int)V, targets, nullptr, logp, fused ? nullptr : coef, stats, part};
            if (int rc = launch_logp<E>(a, m, V, s)) return rc;
        }
        if (fused) {
            const LogpArgs a{z, ldz, (int)V, targets, nullptr, logp, nullptr, stats, nullptr};
            const dim3 grid(grad_parts(V, sizeof(E)), (unsigned)(m + pairs));
            if (V * (int64_t)sizeof(E) <= 4096)
                hipLaunchKernelGGL((pair_rows_kernel<E, 64>), grid, dim3(64), 0, s, a, m, offsets, pairs, ref, beta, smoothing, pair_w, loss, margin, grad, ldg);
            else
                hipLaunchKernelGGL((pair_rows_kernel<E, 256>), grid, dim3(256), 0, s, a, m, offsets, pairs, ref, beta, smoothing, pair_w, loss, margin, grad, ldg);
            RBG_HIP(hipGetLastError());
            return (int)RBG_OK;
        }
        if (int rc = launch_pairs<double, true>(logp, m, offsets, pairs, ref, beta, smoothing, pair_w, loss, margin, coef, s)) return rc;
        return m ? launch_logp_grad<E>((const E *)z, ldz, m, V, targets, stats, coef, (E *)grad, ldg, s) : (int)RBG_OK;
    });
}

}  // extern "C"
