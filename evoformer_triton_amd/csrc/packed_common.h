// Attention within packed sequences: what its kernels share.
#pragma once

#include "elements.h"
#include "kernels.h"

namespace evo {

// Whether a launch with a wave to a row, four of them to a workgroup, holds so many rows.
static inline bool row_waves_fit(int64_t rows) { return grid_fits((rows + 3) / 4, 256); }

// A kernel's first argument, loaded anew (by scalar loads): what its end alone needs is then not kept in registers over its loop.
__device__ __forceinline__ EvoPacked parameters_again() {
    typedef const __attribute__((address_space(4))) unsigned Word;
    Word *at = (Word *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    struct Words {
        unsigned x[sizeof(EvoPacked) / 4];
    } words;
#pragma unroll
    for (unsigned i = 0; i < sizeof(EvoPacked) / 4; ++i) words.x[i] = at[i];
    return __builtin_bit_cast(EvoPacked, words);
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
// This lane's own row x times a row that the wave holds; by all lanes of a wave, since each is asked for its part of that
template <typename T>
__device__ __forceinline__ float own_dot(Row r, const T *x, int D) {
    float s = 0.0f;
    if constexpr (sizeof(T) == 2) {   // (pieces of 16 bytes)
        for (int d = 0; d < min(D, 64); d += 8) {
            const auto v = ld8(x + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(lane_value(r.a, d + i), (float)v[i], s);
        }
        for (int d = 64; d < D; d += 8) {
            const auto v = ld8(x + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(lane_value(r.b, d - 64 + i), (float)v[i], s);
        }
    } else {
        for (int d = 0; d < min(D, 64); ++d) s = fmaf(lane_value(r.a, d), (float)x[d], s);
        for (int d = 64; d < D; ++d) s = fmaf(lane_value(r.b, d - 64), (float)x[d], s);
    }
    return s;
}

template <typename T>
__device__ __forceinline__ const T *head_row(const void *x, int64_t row, int64_t stride_t, int h, int64_t stride_h) {
    return (const T *)x + row * stride_t + h * stride_h;
}

// This lane's two columns of a row
template <typename T>
__device__ __forceinline__ Row columns(const T *x, int D) {
    const int lane = threadIdx.x & 63;
    return {(float)x[min(lane, D - 1)], (float)x[min(lane + 64, D - 1)]};
}
// The sum of n rows (up to 64) with weights, lane i's for row `first` + i; N rows are asked for at a time (four where a kernel of few registers does it: eight would leave room for fewer of its waves).
template <typename T, int N>
__device__ __forceinline__ void add_rows(Row &sum, float w, const void *x, int64_t first, int64_t stride_t, int h, int64_t stride_h, int n, int D) {
    for (int i = 0; i < n; i += N) {
        Row v[N];
#pragma unroll
        for (int y = 0; y < N; ++y) v[y] = columns(head_row<T>(x, first + min(i + y, n - 1), stride_t, h, stride_h), D);
#pragma unroll
        for (int y = 0; y < N; ++y)
            if (i + y < n) add_row(sum, lane_value(w, i + y), v[y]);
    }
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

// ---- What the matrix kernels do about results that are no numbers.  A key or a query that a row does not see, but others of its tile do, may hold an infinity or a NaN, which a product with a probability of
// zero does not keep out.  Such a row is formed anew by a wave from the rows alone that it sees, 64 at a time, a row of the other side to a lane, products and sums in fp32: that takes hundreds of times as long as a
// matrix kernel's share, so that it is for rows alone that may have come to it in this way.  All others are what they are because of what they see:
//   nothing that is not seen, of the stages that the tile's causal limits run through, holds anything but numbers; or
//   the row has no number whatever else there is: a sum of its probabilities (forward) or of its dS (dQ) that is no number, lse or delta of a query that sees the key (dK, dV), or, in every
//   column, a NaN or infinities of both signs in what is seen.
// Forward and backward of one causal sequence of 2048 rows, 8 heads of 64, bf16: 0.13 ms; with an incoming gradient of NaN alone 0.20 (every row formed anew: 35), with a row of NaN in it 0.7, with one in the values 1.0.  4 x 4096
// rows, 32 heads (8) of 128: 2.9, 2.8, 97 (the keys just behind that row's place take it in: 62 of each head, 31 to a wave, from all queries behind them) and 5.

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
// Whether rows from .. to - 1 hold numbers alone
template <typename T>
__device__ __forceinline__ bool all_finite(const void *x, int64_t stride_t, int h, int64_t stride_h, int from, int to, int D) {
    for (int i = from; i < to; i += 8) {
        float largest = 0.0f;   // (fmaxf passes a NaN over)
        bool nan = false;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const Row r = columns(head_row<T>(x, min(i + y, to - 1), stride_t, h, stride_h), D);
            largest = fmaxf(largest, fmaxf(fabsf(r.a), fabsf(r.b)));
            nan |= __builtin_isunordered(r.a, r.b);
        }
        if (__any(nan | (largest == INFINITY))) return false;
    }
    return true;
}
// Whether a sum of rows from .. to - 1, and of those that `c` knows of, is a NaN in every column, whatever their positive weights.  c: bits of this lane's two columns, of a NaN and of infinities of either sign
template <typename T>
__device__ __forceinline__ bool no_column_left(unsigned &c, const void *x, int64_t stride_t, int h, int64_t stride_h, int from, int to, int D) {
    auto kind = [](float v) -> unsigned { return !(v == v) ? 7 : v == INFINITY ? 2 : v == -INFINITY ? 4 : 0; };
    for (int i = from; i < to; i += 8) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const Row r = columns(head_row<T>(x, min(i + y, to - 1), stride_t, h, stride_h), D);
            c |= kind(r.a) | kind(r.b) << 3;
        }
        if (__all((c & 54) == 54)) return true;
    }
    return false;
}
// Whether o of rows that see the first `seen` keys, all of them, may have taken in something else: from key `seen` up to `end`.
template <typename T>
__device__ __forceinline__ bool spoilt_forward(const EvoPacked &p, const Segment &s, int hk, int seen, int end) {
    unsigned c = 0;
    return !all_finite<T>(p.v, p.v_stride_t, hk, p.v_stride_h, s.k0 + seen, s.k0 + end, p.D) && !no_column_left<T>(c, p.v, p.v_stride_t, hk, p.v_stride_h, s.k0, s.k0 + seen, p.D);
}
// The same of dQ (of rows whose sums of dS are numbers)
template <typename T>
__device__ __forceinline__ bool spoilt_dq(const EvoPacked &p, const Segment &s, int hk, int seen, int end) {
    return !all_finite<T>(p.k, p.k_stride_t, hk, p.k_stride_h, s.k0 + seen, s.k0 + end, p.D);
}
// Of dK and dV of keys k0 .. k1 - 1, which queries from .. q1 - 1 see: queries begin .. from - 1, and the zeros that stand for queries past the sequence's end, whose products with a key or value that is no number are none.
template <typename T>
__device__ __forceinline__ bool spoilt_dkdv(const EvoPacked &p, const Segment &s, int hk, int k0, int k1, int begin, int from, const float *minus_delta) {
    const int lane = threadIdx.x & 63, G = p.H / p.Hk;
    bool dv = !all_finite<T>(p.k, p.k_stride_t, hk, p.k_stride_h, k0, k1, p.D), dk = dv || !all_finite<T>(p.v, p.v_stride_t, hk, p.v_stride_h, k0, k1, p.D);
    for (int h = hk * G; h < (hk + 1) * G; ++h) {
        dk = dk || !all_finite<T>(p.q, p.q_stride_t, h, p.q_stride_h, begin, from, p.D);
        dv = dv || !all_finite<T>(p.dout, p.dout_stride_t, h, p.dout_stride_h, begin, from, p.D);
    }
    if (!dk && !dv) return false;
    unsigned c = 0;
    for (int h = hk * G; h < (hk + 1) * G; ++h) {
        bool lse = false, delta = false;
        for (int i = from + lane; i < s.q1; i += 64) {
            const float x = minus_delta[(int64_t)h * p.Tq + i];
            lse |= !finite(p.lse[(int64_t)h * p.Tq + i]);
            delta |= !(x == x);
        }
        if (__any(lse)) return false;
        if (__any(delta)) dk = false;
        if (dv && no_column_left<T>(c, p.dout, p.dout_stride_t, h, p.dout_stride_h, from, s.q1, p.D)) dv = false;
        if (!dk && !dv) return false;
    }
    return true;
}

template <typename T, int N = 8>
__device__ __forceinline__ void row_forward(const EvoPacked &p, const Segment &s, int i, int h) {
    const int lane = threadIdx.x & 63, hk = h / (p.H / p.Hk), seen = s.gap ? 0 : s.seen(i, p.causal);
    const float c = p.scale * kLog2e;
    const Row q = load_row(head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h), p.D);
    float m = -INFINITY, l = 0.0f;
    Row o = {0.0f, 0.0f};
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int n = min(64, seen - j0);
        const float dot = own_dot(q, head_row<T>(p.k, s.k0 + j0 + min(lane, n - 1), p.k_stride_t, hk, p.k_stride_h), p.D), x = lane < n ? dot * c : -INFINITY;
        const float mn = fmaxf(m, wave_max(x));
        const float base = mn == -INFINITY ? 0.0f : mn, alpha = fast_exp2(m - base), e = lane < n ? fast_exp2(x - base) : 0.0f;
        m = mn;
        l = l * alpha + wave_sum(e);
        o.a *= alpha;
        o.b *= alpha;
        add_rows<T, N>(o, e, p.v, s.k0 + j0, p.v_stride_t, hk, p.v_stride_h, n, p.D);
    }
    const float inv = seen ? 1.0f / l : 0.0f;
    o.a *= inv;
    o.b *= inv;
    store_row((T *)p.o + ((int64_t)i * p.H + h) * p.D, o, p.D);
    if (sizeof(T) == 2 && p.o_low) store_row((T *)p.o_low + ((int64_t)i * p.H + h) * p.D, Row{o.a - (float)(T)o.a, o.b - (float)(T)o.b}, p.D);
    if (p.lse && lane == 0) p.lse[(int64_t)h * p.Tq + i] = seen ? m + __log2f(l) : INFINITY;
}

template <typename T, int N = 8>
__device__ __forceinline__ void row_dq(const EvoPacked &p, const Segment &s, int i, int h, float delta) {
    const int lane = threadIdx.x & 63, hk = h / (p.H / p.Hk), seen = s.gap ? 0 : s.seen(i, p.causal);
    const float c = p.scale * kLog2e, lse = p.lse[(int64_t)h * p.Tq + i];
    const Row q = load_row(head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h), p.D), dout = load_row(head_row<T>(p.dout, i, p.dout_stride_t, h, p.dout_stride_h), p.D);
    Row dq = {0.0f, 0.0f};
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int n = min(64, seen - j0);
        const int row = s.k0 + j0 + min(lane, n - 1);
        const float e = fast_exp2(own_dot(q, head_row<T>(p.k, row, p.k_stride_t, hk, p.k_stride_h), p.D) * c - lse);
        const float ds = e * (own_dot(dout, head_row<T>(p.v, row, p.v_stride_t, hk, p.v_stride_h), p.D) - delta) * p.scale;
        add_rows<T, N>(dq, ds, p.k, s.k0 + j0, p.k_stride_t, hk, p.k_stride_h, n, p.D);
    }
    store_row((T *)p.dq + ((int64_t)i * p.H + h) * p.D, dq, p.D);
}

template <typename T, int N = 8>
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
            const int row = i0 + min(lane, n - 1);
            const float e = fast_exp2(own_dot(k, head_row<T>(p.q, row, p.q_stride_t, h, p.q_stride_h), p.D) * c - p.lse[(int64_t)h * p.Tq + row]);
            const float ds = e * (own_dot(v, head_row<T>(p.dout, row, p.dout_stride_t, h, p.dout_stride_h), p.D) + minus_delta[(int64_t)h * p.Tq + row]) * p.scale;
            add_rows<T, N>(dv, e, p.dout, i0, p.dout_stride_t, h, p.dout_stride_h, n, p.D);
            add_rows<T, N>(dk, ds, p.q, i0, p.q_stride_t, h, p.q_stride_h, n, p.D);
        }
    }
    store_row((T *)p.dk + ((int64_t)j * p.Hk + hk) * p.D, dk, p.D);
    store_row((T *)p.dv + ((int64_t)j * p.Hk + hk) * p.D, dv, p.D);
}

}  // namespace evo
