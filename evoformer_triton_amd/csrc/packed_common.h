// Attention within packed sequences: what its kernels share.
#pragma once

#include "elements.h"
#include "kernels.h"

namespace evo {

// Whether a launch with a wave to a row, four of them to a workgroup, holds so many rows.
static inline bool row_waves_fit(int64_t rows) { return grid_fits((rows + 3) / 4, 256); }

// A kernel's first argument, loaded anew: what its end alone needs is then not kept in registers over its loop.
__device__ __forceinline__ EvoPacked parameters_again() {
    auto *at = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    EvoPacked p;
    __builtin_memcpy(&p, (const void *)at, sizeof p);
    return p;
}

// Rows of a sequence: queries q0 .. q1 - 1, keys k0 .. k1 - 1.  gap: rows of no sequence, before the first and behind the last.
struct Segment {
    int q0, q1, k0, k1;
    bool gap;
    __device__ __forceinline__ int nq() const { return q1 - q0; }
    __device__ __forceinline__ int nk() const { return k1 - k0; }
    // the keys that query i (of the tensor) sees: k0 .. k0 + seen(i) - 1
    __device__ __forceinline__ int seen(int i, bool causal) const { return causal ? max(0, min(nk(), nk() - nq() + (i - q0) + 1)) : nk(); }
    // the first query (of the tensor) that sees key j (of the tensor); q1 or beyond: none does
    __device__ __forceinline__ int first_query(int j, bool causal) const { return causal ? q0 + max(0, (j - k0) - (nk() - nq())) : q0; }
};

// Where segment j of n + 2 begins: 0 before the first sequence, then the sequences, then what is behind the last.  Brought into [0, T] whatever the offsets hold.
__device__ __forceinline__ int segment_begin(const void *offsets, int bytes, int n, int64_t T, int j) {
    if (j <= 0) return 0;
    if (j > n + 1) return (int)T;
    const int64_t v = bytes == 8 ? ((const int64_t *)offsets)[j - 1] : (int64_t)((const int *)offsets)[j - 1];
    return (int)min(max(v, (int64_t)0), T);
}
__device__ __forceinline__ int queries_begin(const EvoPacked &p, int j) { return segment_begin(p.offsets, p.offset_bytes, p.n, p.Tq, j); }
__device__ __forceinline__ int keys_begin(const EvoPacked &p, int j) { return segment_begin(p.key_offsets, p.offset_bytes, p.n, p.Tk, j); }

// The last of `count` indices (at least one) of which `before` holds, which is true up to some index (0 among them) and false from there on: 64 are asked at a time, by
// a whole wave.  (Where `before` is none such: some index.)
template <typename F>
__device__ __forceinline__ int last_where(int count, F before) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (count > 1) {
        const int step = (count + 63) / 64;
        const bool yes = (int64_t)lane * step < count && before(lo + lane * step);
        const int c = max(1, (int)__popcll(__ballot(yes)));
        lo += (c - 1) * step;
        count = min(step, count - (c - 1) * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
__device__ __forceinline__ Segment segment(const EvoPacked &p, int j) {
    Segment s;
    s.gap = j == 0 || j == p.n + 1;
    s.q0 = queries_begin(p, j);
    s.q1 = max(s.q0, queries_begin(p, j + 1));
    s.k0 = keys_begin(p, j);
    s.k1 = max(s.k0, keys_begin(p, j + 1));
    s.q0 = __builtin_amdgcn_readfirstlane(s.q0);
    s.q1 = __builtin_amdgcn_readfirstlane(s.q1);
    s.k0 = __builtin_amdgcn_readfirstlane(s.k0);
    s.k1 = __builtin_amdgcn_readfirstlane(s.k1);
    return s;
}
// Segment j where lane x holds the first query q and the first key k of segment x (up to n + 2).
__device__ __forceinline__ Segment segment_of_lanes(const EvoPacked &p, int q, int k, int j) {
    Segment s;
    s.gap = j == 0 || j == p.n + 1;
    s.q0 = __builtin_amdgcn_readlane(q, j);
    s.q1 = __builtin_amdgcn_readfirstlane(max(s.q0, (int)__builtin_amdgcn_readlane(q, j + 1)));
    s.k0 = __builtin_amdgcn_readlane(k, j);
    s.k1 = __builtin_amdgcn_readfirstlane(max(s.k0, (int)__builtin_amdgcn_readlane(k, j + 1)));
    return s;
}
// The last segment j for which before(begin(j), j) holds, begin(j) being its first query (KEYS: key) and `before` as last_where takes it.  Where a wave has a lane for every segment's begin, those of queries and of
// keys are loaded at once and the segment's own are taken from the lanes: one trip to memory, not two or three.
template <bool KEYS, typename F>
__device__ __forceinline__ Segment find_segment(const EvoPacked &p, F before, int &j) {
    if (p.n + 3 > 64) {
        j = last_where(p.n + 2, [&](int x) { return before(KEYS ? keys_begin(p, x) : queries_begin(p, x), x); });
        return segment(p, j);
    }
    const int lane = threadIdx.x & 63, x = min(lane, p.n + 2), q = queries_begin(p, x), k = keys_begin(p, x);
    j = __builtin_amdgcn_readfirstlane(max(1, (int)__popcll(__ballot(lane < p.n + 2 && before(KEYS ? k : q, lane)))) - 1);
    return segment_of_lanes(p, q, k, j);
}
// The segment that a row of the queries (or, KEYS, of the keys) lies in.
template <bool KEYS>
__device__ __forceinline__ Segment segment_of_row(const EvoPacked &p, int row) {
    int j;
    return find_segment<KEYS>(p, [&](int begin, int) { return begin <= row; }, j);
}

__device__ __forceinline__ float lane_value(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A row of up to 128 values, two to a lane: lane and lane + 64.
struct Row {
    float a, b;
};
template <typename T>
__device__ __forceinline__ Row load_row(const T *x, int D) {
    const int lane = threadIdx.x & 63;
    Row r;
    r.a = lane < D ? (float)x[lane] : 0.0f;
    r.b = lane + 64 < D ? (float)x[lane + 64] : 0.0f;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_row(T *x, Row r, int D) {
    const int lane = threadIdx.x & 63;
    if (lane < D) x[lane] = (T)r.a;
    if (lane + 64 < D) x[lane + 64] = (T)r.b;
}
__device__ __forceinline__ void add_row(Row &r, float w, Row x) {
    r.a = fmaf(w, x.a, r.a);
    r.b = fmaf(w, x.b, r.b);
}
// This lane's own row x times a row that the wave holds
template <typename T>
__device__ __forceinline__ float own_dot(Row r, const T *x, int D) {
    float s = 0.0f;
    for (int d = 0; d < min(D, 64); ++d) s = fmaf(lane_value(r.a, d), (float)x[d], s);
    for (int d = 64; d < D; ++d) s = fmaf(lane_value(r.b, d - 64), (float)x[d], s);
    return s;
}

template <typename T>
__device__ __forceinline__ const T *head_row(const void *x, int64_t row, int64_t stride_t, int h, int64_t stride_h) {
    return (const T *)x + row * stride_t + h * stride_h;
}

// What dQ's kernel leaves for that of dK and dV, [H][Tq] each: -delta and -lse, the latter in units of q . k (16 bits: what their products begin with).
struct BackwardRows {
    float *delta, *base;
};
// The forward's lse is that of rounded probabilities, and its output, of which delta is formed, theirs too.  The sums that dQ's kernel has of probabilities (`sum`, 1 but for that) and of ds (`rest`, 0 but for that) say by how
// much: what dK and dV are formed with is put right by them.
__device__ __forceinline__ void save_row(const BackwardRows &to, int64_t at, float lse, float delta, float sum, float rest, float c) {
    const bool any = sum > 0.0f;
    to.delta[at] = -(any ? delta + rest / sum : delta);
    to.base[at] = -(any ? lse + __log2f(sum) : lse) / c;
}

// ---- One row by one wave, products and sums in fp32: what the matrix kernels leave for rows whose result is no number.  A masked key or query may hold an infinity or a NaN there, which a product
// with a probability of zero does not keep out; here a wave takes the rows alone that are seen, 64 at a time, a row of the other side to a lane.

template <typename T>
__device__ __forceinline__ void row_forward(const EvoPacked &p, const Segment &s, int i, int h) {
    const int lane = threadIdx.x & 63, hk = h / (p.H / p.Hk), seen = s.gap ? 0 : s.seen(i, p.causal);
    const float c = p.scale * kLog2e;
    const Row q = load_row(head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h), p.D);
    float m = -INFINITY, l = 0.0f;
    Row o = {0.0f, 0.0f};
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int n = min(64, seen - j0);
        const float x = lane < n ? own_dot(q, head_row<T>(p.k, s.k0 + j0 + lane, p.k_stride_t, hk, p.k_stride_h), p.D) * c : -INFINITY;
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn, alpha = fast_exp2(m - base), e = lane < n ? fast_exp2(x - base) : 0.0f;
        m = mn;
        l = l * alpha + wave_sum(e);
        o.a *= alpha;
        o.b *= alpha;
        for (int j = 0; j < n; ++j) add_row(o, lane_value(e, j), load_row(head_row<T>(p.v, s.k0 + j0 + j, p.v_stride_t, hk, p.v_stride_h), p.D));
    }
    const float inv = seen ? 1.0f / l : 0.0f;
    o.a *= inv;
    o.b *= inv;
    store_row((T *)p.o + ((int64_t)i * p.H + h) * p.D, o, p.D);
    if (p.o_low) store_row((T *)p.o_low + ((int64_t)i * p.H + h) * p.D, Row{o.a - (float)(T)o.a, o.b - (float)(T)o.b}, p.D);
    if (p.lse && lane == 0) p.lse[(int64_t)h * p.Tq + i] = seen ? m + __log2f(l) : INFINITY;
}

template <typename T>
__device__ __forceinline__ void row_dq(const EvoPacked &p, const Segment &s, int i, int h, float delta) {
    const int lane = threadIdx.x & 63, hk = h / (p.H / p.Hk), seen = s.gap ? 0 : s.seen(i, p.causal);
    const float c = p.scale * kLog2e, lse = p.lse[(int64_t)h * p.Tq + i];
    const Row q = load_row(head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h), p.D), dout = load_row(head_row<T>(p.dout, i, p.dout_stride_t, h, p.dout_stride_h), p.D);
    Row dq = {0.0f, 0.0f};
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int n = min(64, seen - j0);
        float ds = 0.0f;
        if (lane < n) {
            const int j = s.k0 + j0 + lane;
            const float e = fast_exp2(own_dot(q, head_row<T>(p.k, j, p.k_stride_t, hk, p.k_stride_h), p.D) * c - lse);
            ds = e * (own_dot(dout, head_row<T>(p.v, j, p.v_stride_t, hk, p.v_stride_h), p.D) - delta) * p.scale;
        }
        for (int j = 0; j < n; ++j) add_row(dq, lane_value(ds, j), load_row(head_row<T>(p.k, s.k0 + j0 + j, p.k_stride_t, hk, p.k_stride_h), p.D));
    }
    store_row((T *)p.dq + ((int64_t)i * p.H + h) * p.D, dq, p.D);
}

template <typename T>
__device__ __forceinline__ void row_dkdv(const EvoPacked &p, const Segment &s, int j, int hk, const float *minus_delta) {
    const int lane = threadIdx.x & 63, G = p.H / p.Hk;
    const float c = p.scale * kLog2e;
    const Row k = load_row(head_row<T>(p.k, j, p.k_stride_t, hk, p.k_stride_h), p.D), v = load_row(head_row<T>(p.v, j, p.v_stride_t, hk, p.v_stride_h), p.D);
    Row dk = {0.0f, 0.0f}, dv = {0.0f, 0.0f};
    // the first query that sees this key
    const int first = s.gap ? s.q1 : s.first_query(j, p.causal);
    for (int h = hk * G; h < (hk + 1) * G; ++h) {
        for (int i0 = first; i0 < s.q1; i0 += 64) {
            const int n = min(64, s.q1 - i0);
            float e = 0.0f, ds = 0.0f;
            if (lane < n) {
                const int i = i0 + lane;
                e = fast_exp2(own_dot(k, head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h), p.D) * c - p.lse[(int64_t)h * p.Tq + i]);
                ds = e * (own_dot(v, head_row<T>(p.dout, i, p.dout_stride_t, h, p.dout_stride_h), p.D) + minus_delta[(int64_t)h * p.Tq + i]) * p.scale;
            }
            for (int i = 0; i < n; ++i) {
                add_row(dv, lane_value(e, i), load_row(head_row<T>(p.dout, i0 + i, p.dout_stride_t, h, p.dout_stride_h), p.D));
                add_row(dk, lane_value(ds, i), load_row(head_row<T>(p.q, i0 + i, p.q_stride_t, h, p.q_stride_h), p.D));
            }
        }
    }
    store_row((T *)p.dk + ((int64_t)j * p.Hk + hk) * p.D, dk, p.D);
    store_row((T *)p.dv + ((int64_t)j * p.Hk + hk) * p.D, dv, p.D);
}

}  // namespace evo
