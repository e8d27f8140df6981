// Attention within packed sequences on the matrix cores, 16-bit, compiled once per head dim (-DEVO_D=32|64|96|128; a head dim between takes the next, with zeros behind it).
//
// A workgroup of four waves takes 128 rows of a sequence and head (forward, dQ: queries; dK/dV: keys), a wave 32 of them, and the other side's rows stream through LDS, a
// stage ahead of the one that is computed on, brought there by the load path itself.  Scores are formed transposed, S^T = K Q^T: a lane then holds 16 keys of one query, the softmax
// needs one exchange with the lane's other half, and the tile is as it lies the operand of O^T = V^T P^T (common.h), whose other operand, V^T, is read from row-major V by
// transposing reads.  The running maximum moves only when it grows by more than 2^8, so that the sums are rarely multiplied again; probabilities are rounded to the inputs' type to
// multiply V and summed as rounded.
//
// Which rows: tile t of the launch belongs to the last segment j (packed_common.h) with begin(j) / 128 + j <= t; begin(j + 1) / 128 + j + 1 leaves room for all of j's tiles, so that every workgroup finds
// its place by itself, without a sum over the sequences before it and whatever the lengths are; at most one tile per segment finds nothing to do.
//
// A row of V beyond the sequence's end is read as zeros (the load is out of range).  One that causal queries do not see may hold an infinity or a NaN, which a probability of
// zero does not keep out of the sums: results that are no numbers are formed anew, row by row (row_forward and its like), with the rows that are seen alone.
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

constexpr int kPackedRows = 128;   // of a workgroup

// This lane's offset of its first piece of a stage of rows; its further pieces are kPieceRows rows on each.
template <int NW>
struct StagePieces {
    typedef PackedGeo::G G;
    static constexpr int RPP = 1024 / G::ROW;        // rows to a piece of 1 KB
    static constexpr int STEP = RPP * NW;            // rows from one of a wave's pieces to its next
    static_assert(STEP % 16 == 0, "a lane's chunk is the same in all of its pieces");
    static __device__ __forceinline__ int first(int wave, int lane, int stride, int D) {
        const int r = wave * RPP + lane / G::C, c = (lane % G::C) ^ G::x(r);
        return c * 8 < D ? r * stride + c * 16 : kFarOff;
    }
    template <int ROWS>
    static __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t rs, unsigned char *dst, int first, int stride, int wave) {
        constexpr int PIECES = ROWS / RPP;
#pragma unroll
        for (int i = 0; i < (PIECES + NW - 1) / NW; ++i) {
            if (PIECES % NW != 0 && wave + i * NW >= PIECES) break;   // (uniform)
            dma16(rs, dst + (wave + i * NW) * 1024, first + (first == kFarOff ? 0 : i * STEP * stride));
        }
    }
};

// A row's values as operands: step ks holds columns 16 ks + 8 g .. + 7; zeros from D on.
template <typename T>
__device__ __forceinline__ void load_operands(const T *row, int D, int g, typename Mfma<T>::v8 (&x)[PackedGeo::KSD]) {
#pragma unroll
    for (int ks = 0; ks < PackedGeo::KSD; ++ks) x[ks] = ks * 16 + g * 8 < D ? ld8(row + ks * 16 + g * 8) : zero8<T>();
}

// Where a workgroup is: a tile of a segment, and a head.
struct Place {
    Segment s;
    int first;   // its first row (of the tensor), or, where there is nothing to do, s's end or beyond
};
template <bool KEYS>
__device__ __forceinline__ Place place_of(const EvoPacked &p, int t) {
    auto begin = [&](int j) { return KEYS ? keys_begin(p, j) : queries_begin(p, j); };
    const int j = last_where(p.n + 2, [&](int x) { return begin(x) / kPackedRows + x <= t; });
    Place r;
    r.s = segment(p, j);
    const int b = KEYS ? r.s.k0 : r.s.q0, i = t - (b / kPackedRows + j);
    r.first = i < 0 ? INT32_MAX : (int)min((int64_t)INT32_MAX, b + (int64_t)i * kPackedRows);   // (below zero: offsets that do not ascend)
    return r;
}

template <typename T>
__device__ __forceinline__ void zero_rows(T *x, int first, int end, int heads, int h, int D) {
    const int per = D / 8, n = (min(first + kPackedRows, end) - first) * per;
    for (int i = threadIdx.x; i < n; i += 256) *reinterpret_cast<uint4 *>(x + ((int64_t)(first + i / per) * heads + h) * D + i % per * 8) = make_uint4(0, 0, 0, 0);
}

// The lanes (low 32 bits: the rows of the wave) whose accumulators hold something that is no number
__device__ __forceinline__ unsigned rows_without_number(bool nan) {
    const uint64_t b = __ballot(nan);
    return (unsigned)b | (unsigned)(b >> 32);
}

__device__ __forceinline__ f32x16 filled(float v) {
    f32x16 x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = v;
    return x;
}

// ------------------------------------------------------------------ forward

template <typename T>
__global__ void __launch_bounds__(256, EVO_D == 32 ? 4 : EVO_D == 64 ? 3 : 2) packed_fwd(EvoPacked p, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4> Pieces;
    typedef typename Mfma<T>::v8 v8;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][2 * R::ARRAY];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    // A key head's query heads follow each other, then its tiles, the last (under a causal mask the longest) first; consecutive workgroups run on one XCD.
    const int group = p.H / p.Hk;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x), per = (unsigned)tiles * (unsigned)group;
    const int hk = (int)(lid / per), h = hk * group + (int)(lid % per % (unsigned)group);
    const Place at = place_of<false>(p, tiles - 1 - (int)(lid % per / (unsigned)group));
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int D = p.D, rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {
        zero_rows((T *)p.o, at.first, s.q1, p.H, h, D);
        if (p.lse && (int)threadIdx.x < rows) p.lse[(int64_t)h * p.Tq + at.first + threadIdx.x] = INFINITY;
        return;
    }
    const int kst = (int)p.k_stride_t * 2, vst = (int)p.v_stride_t * 2;
    const char *kbase = (const char *)head_row<T>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = (const char *)head_row<T>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    const int koff = Pieces::first(wave, lane, kst, D), voff = Pieces::first(wave, lane, vst, D);
    auto fetch = [&](int stage) {
        const int row = stage * R::STAGE, n = min(R::STAGE, s.nk() - row);
        unsigned char *dst = lds[stage & 1];
        Pieces::fetch<R::STAGE>(rows_at(kbase + (int64_t)row * kst, n, kst, D), dst, koff, kst, wave);
        Pieces::fetch<R::STAGE>(rows_at(vbase + (int64_t)row * vst, n, vst, D), dst + R::ARRAY, voff, vst, wave);
    };
    fetch(0);

    const int q0 = at.first + wave * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1;   // uniform
    v8 qf[R::KSD];
    load_operands(head_row<T>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), D, g, qf);
    const int seen = s.seen(qrow, p.causal);
    // of the wave's queries: the fewest keys and the most
    const int wave_least = active ? s.seen(q0, p.causal) : 0, wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    const float c = p.scale * kLog2e;
    float m = kMaskFloor, l = 0.0f;
    f32x16 o[R::DT];
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) o[dt] = filled(0.0f);
    v8 one;
#pragma unroll
    for (int i = 0; i < 8; ++i) one[i] = (T)1.0f;

    auto step = [&](const unsigned char *buf, int key0) __attribute__((always_inline)) {
        f32x16 a[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            a[t] = filled(0.0f);
#pragma unroll
            for (int ks = 0; ks < R::KSD; ++ks) a[t] = Mfma<T>::mma(*reinterpret_cast<const v8 *>(buf + G::at(32 * t + li, 2 * ks + g)), qf[ks], a[t]);
        }
        if (key0 + R::STAGE > wave_least) {   // (uniform)
            asm volatile("");                 // (a branch: not computed where it is not needed)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) a[t][r] = key0 + 32 * t + crow(r, g) < seen ? a[t][r] : -INFINITY;
        }
        float top = a[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, a[t][r]);
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        // (not below the floor: a query that sees none of these keys has -inf here, and -inf less -inf is no number)
        const float cand = fmaxf(fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * c, kMaskFloor);
        const bool grow = cand > m + 8.0f;
        if (__any(grow)) {
            const float mn = grow ? cand : m, alpha = fast_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
        }
        v8 pf[4];
#pragma unroll
        for (int ts = 0; ts < 4; ++ts) {
#pragma unroll
            for (int i = 0; i < 8; ++i) pf[ts][i] = (T)fast_exp2(fmaf(a[ts / 2][8 * (ts & 1) + i], c, -m));
            l = dot8<T>(pf[ts], one, l);
        }
#pragma unroll
        for (int ts = 0; ts < 4; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) o[dt] = Mfma<T>::mma(transposed<T, R::GD>(buf + R::ARRAY, (ts / 2) * 32, ts & 1, dt, lane), pf[ts], o[dt]);
    };
    const int stages = (seen_most + R::STAGE - 1) / R::STAGE;
    wait_loads();
    wait_lds_barrier();
    for (int st = 0; st < stages; ++st) {
        if (st + 1 < stages) fetch(st + 1);
        if (st * R::STAGE < wave_most) step(lds[st & 1], st * R::STAGE);
        if (st + 1 < stages) {
            wait_loads();
            wait_lds_barrier();
        }
    }
    if (!active) return;
    l += __shfl_xor(l, 32);
    const float inv = seen ? 1.0f / l : 0.0f;
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[dt][r] = seen ? o[dt][r] * inv : 0.0f;
            nan |= !(o[dt][r] == o[dt][r]);
        }
    const bool own = q0 + li < s.q1;
    unsigned again = rows_without_number(nan && own);
    const bool whole = own && !(again >> li & 1);
    if (p.lse && whole && g == 0) p.lse[(int64_t)h * p.Tq + qrow] = seen ? m + __log2f(l) : INFINITY;
    T *out = (T *)p.o + ((int64_t)qrow * p.H + h) * D;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) store_row_tile<T>(out, dt * 32, whole ? D : 0, o[dt], 1.0f, g);
    for (; again; again &= again - 1) row_forward<T>(p, s, q0 + __builtin_ctz(again), h);
}

// ------------------------------------------------------------------ dQ

template <typename T>
__global__ void __launch_bounds__(256, EVO_D == 32 ? 4 : EVO_D == 64 ? 3 : 2) packed_dq(EvoPacked p, float *delta, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4> Pieces;
    typedef typename Mfma<T>::v8 v8;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][2 * R::ARRAY];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int group = p.H / p.Hk;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x), per = (unsigned)tiles * (unsigned)group;
    const int hk = (int)(lid / per), h = hk * group + (int)(lid % per % (unsigned)group);
    const Place at = place_of<false>(p, tiles - 1 - (int)(lid % per / (unsigned)group));
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int D = p.D, rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {
        zero_rows((T *)p.dq, at.first, s.q1, p.H, h, D);
        if ((int)threadIdx.x < rows) delta[(int64_t)h * p.Tq + at.first + threadIdx.x] = 0.0f;
        return;
    }
    const int kst = (int)p.k_stride_t * 2, vst = (int)p.v_stride_t * 2;
    const char *kbase = (const char *)head_row<T>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = (const char *)head_row<T>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    const int koff = Pieces::first(wave, lane, kst, D), voff = Pieces::first(wave, lane, vst, D);
    auto fetch = [&](int stage) {
        const int row = stage * R::STAGE, n = min(R::STAGE, s.nk() - row);
        unsigned char *dst = lds[stage & 1];
        Pieces::fetch<R::STAGE>(rows_at(kbase + (int64_t)row * kst, n, kst, D), dst, koff, kst, wave);
        Pieces::fetch<R::STAGE>(rows_at(vbase + (int64_t)row * vst, n, vst, D), dst + R::ARRAY, voff, vst, wave);
    };
    fetch(0);

    const int q0 = at.first + wave * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1, own = q0 + li < s.q1;
    v8 qf[R::KSD], df[R::KSD];
    load_operands(head_row<T>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), D, g, qf);
    load_operands(head_row<T>(p.dout, qrow, p.dout_stride_t, h, p.dout_stride_h), D, g, df);
    float dl = 0.0f;
    {
        v8 of[R::KSD];
        load_operands((const T *)p.o + ((int64_t)qrow * p.H + h) * D, D, g, of);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) dl = dot8<T>(df[ks], of[ks], dl);
    }
    dl += __shfl_xor(dl, 32);
    if (own && g == 0) delta[(int64_t)h * p.Tq + qrow] = dl;
    const float lse = p.lse[(int64_t)h * p.Tq + qrow];
    const int seen = s.seen(qrow, p.causal);
    const int wave_least = active ? s.seen(q0, p.causal) : 0, wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    const float c = p.scale * kLog2e;
    f32x16 dq[R::DT];
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) dq[dt] = filled(0.0f);

    auto step = [&](const unsigned char *buf, int kb, int key0) __attribute__((always_inline)) {
        f32x16 a = filled(0.0f), d = filled(-dl);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) {
            a = Mfma<T>::mma(*reinterpret_cast<const v8 *>(buf + G::at(kb + li, 2 * ks + g)), qf[ks], a);
            d = Mfma<T>::mma(*reinterpret_cast<const v8 *>(buf + R::ARRAY + G::at(kb + li, 2 * ks + g)), df[ks], d);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] *= fast_exp2(fmaf(a[r], c, -lse));
        if (key0 + 32 > wave_least) {   // (uniform)
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; ++r) d[r] = key0 + crow(r, g) < seen ? d[r] : 0.0f;
        }
        v8 pf[2];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int i = 0; i < 8; ++i) pf[ts][i] = (T)d[8 * ts + i];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) dq[dt] = Mfma<T>::mma(transposed<T, R::GD>(buf, kb, ts, dt, lane), pf[ts], dq[dt]);
    };
    const int stages = (seen_most + R::STAGE - 1) / R::STAGE;
    wait_loads();
    wait_lds_barrier();
    for (int st = 0; st < stages; ++st) {
        if (st + 1 < stages) fetch(st + 1);
#pragma unroll
        for (int t = 0; t < 2; ++t)
            if (st * R::STAGE + 32 * t < wave_most) step(lds[st & 1], 32 * t, st * R::STAGE + 32 * t);
        if (st + 1 < stages) {
            wait_loads();
            wait_lds_barrier();
        }
    }
    if (!active) return;
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan |= !(dq[dt][r] == dq[dt][r]);
    unsigned again = rows_without_number(nan && own);
    const bool whole = own && !(again >> li & 1);
    T *out = (T *)p.dq + ((int64_t)qrow * p.H + h) * D;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) store_row_tile<T>(out, dt * 32, whole ? D : 0, dq[dt], p.scale, g);
    for (; again; again &= again - 1) {
        const int b = __builtin_ctz(again);
        row_dq<T>(p, s, q0 + b, h, lane_value(dl, b));
    }
}

// ------------------------------------------------------------------ dK, dV

template <typename T>
__global__ void __launch_bounds__(256, EVO_D == 32 ? 3 : 2) packed_dkdv(EvoPacked p, const float *delta, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4> Pieces;
    typedef typename Mfma<T>::v8 v8;
    constexpr int ROWS = EVO_D > 64 ? 32 : 64;   // queries of a stage
    constexpr int ARRAY = ROWS * G::ROW, BYTES = 2 * ARRAY + 2 * 256;   // Q, dO, then 64 places each for lse and delta
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][(BYTES + 1023) / 1024 * 1024];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int group = p.H / p.Hk;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x);
    const int hk = (int)(lid / (unsigned)tiles);
    const Place at = place_of<true>(p, (int)(lid % (unsigned)tiles));   // (a sequence's first keys, which causal queries see most of, first)
    const Segment &s = at.s;
    if (at.first >= s.k1) return;
    const int D = p.D;
    // the first query that sees the workgroup's first key
    const int more = s.nk() - s.nq(), begin = s.q0 + (p.causal ? max(0, at.first - s.k0 - more) : 0);
    if (s.gap || begin >= s.q1) {
        zero_rows((T *)p.dk, at.first, s.k1, p.Hk, hk, D);
        zero_rows((T *)p.dv, at.first, s.k1, p.Hk, hk, D);
        return;
    }
    const int qst = (int)p.q_stride_t * 2, dst_ = (int)p.dout_stride_t * 2;
    const int qoff = Pieces::first(wave, lane, qst, D), doff = Pieces::first(wave, lane, dst_, D);
    const int stages = (s.q1 - begin + ROWS - 1) / ROWS;
    auto fetch = [&](int h, int stage, unsigned char *dst) {
        const int row = begin + stage * ROWS, n = min(ROWS, s.q1 - row);
        Pieces::fetch<ROWS>(rows_at(head_row<T>(p.q, row, p.q_stride_t, h, p.q_stride_h), n, qst, D), dst, qoff, qst, wave);
        Pieces::fetch<ROWS>(rows_at(head_row<T>(p.dout, row, p.dout_stride_t, h, p.dout_stride_h), n, dst_, D), dst + ARRAY, doff, dst_, wave);
        if (wave < 2) {   // (a number to a lane; rows past the end: zero)
            const float *x = (wave ? delta : p.lse) + (int64_t)h * p.Tq + row;
            dma4(__builtin_amdgcn_make_buffer_rsrc((void *)x, 0, n * 4, 0x00020000), dst + 2 * ARRAY + wave * 256, lane * 4);
        }
    };
    int h = hk * group, stage = 0;
    fetch(h, 0, lds[0]);
    const int k0 = at.first + wave * 32, krow = min(k0 + li, s.k1 - 1);
    const bool active = k0 < s.k1, own = k0 + li < s.k1;
    v8 kf[R::KSD], vf[R::KSD];
    load_operands(head_row<T>(p.k, krow, p.k_stride_t, hk, p.k_stride_h), D, g, kf);
    load_operands(head_row<T>(p.v, krow, p.v_stride_t, hk, p.v_stride_h), D, g, vf);
    // the first query that sees this lane's key, the wave's first and its last one, as rows of the tensor
    const int from = p.causal ? s.q0 + max(0, krow - s.k0 - more) : s.q0;
    const int wave_from = p.causal ? s.q0 + max(0, k0 - s.k0 - more) : s.q0, wave_to = p.causal ? s.q0 + max(0, min(k0 + 31, s.k1 - 1) - s.k0 - more) : s.q0;
    const float c = p.scale * kLog2e;
    f32x16 dk[R::DT], dv[R::DT];
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) dk[dt] = dv[dt] = filled(0.0f);

    auto step = [&](const unsigned char *buf, int qb, int row0) __attribute__((always_inline)) {
        const float *lse = reinterpret_cast<const float *>(buf + 2 * ARRAY) + qb, *del = lse + 64;
        f32x16 a = filled(0.0f), d, b;
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(lse + 8 * rr + 4 * g), y = *reinterpret_cast<const f32x4 *>(del + 8 * rr + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[4 * rr + i] = x[i];
                d[4 * rr + i] = -y[i];
            }
        }
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) a = Mfma<T>::mma(*reinterpret_cast<const v8 *>(buf + G::at(qb + li, 2 * ks + g)), kf[ks], a);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) d = Mfma<T>::mma(*reinterpret_cast<const v8 *>(buf + ARRAY + G::at(qb + li, 2 * ks + g)), vf[ks], d);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            a[r] = fast_exp2(fmaf(a[r], c, -b[r]));
            d[r] *= a[r];
        }
        if (row0 < wave_to) {   // (uniform)
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool sees = row0 + crow(r, g) >= from;
                a[r] = sees ? a[r] : 0.0f;
                d[r] = sees ? d[r] : 0.0f;
            }
        }
        v8 pf[2], sf[2];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                pf[ts][i] = (T)a[8 * ts + i];
                sf[ts][i] = (T)d[8 * ts + i];
            }
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) {
                dv[dt] = Mfma<T>::mma(transposed<T, R::GD>(buf + ARRAY, qb, ts, dt, lane), pf[ts], dv[dt]);
                dk[dt] = Mfma<T>::mma(transposed<T, R::GD>(buf, qb, ts, dt, lane), sf[ts], dk[dt]);
            }
    };
    wait_loads();
    wait_lds_barrier();
    const int total = stages * group;
    for (int it = 0; it < total; ++it) {
        const int row = begin + stage * ROWS;
        if (++stage == stages) {
            stage = 0;
            ++h;
        }
        if (it + 1 < total) fetch(h, stage, lds[(it + 1) & 1]);
#pragma unroll
        for (int t = 0; t < ROWS / 32; ++t) {
            const int row0 = row + 32 * t;
            if (active && row0 < s.q1 && row0 + 31 >= wave_from) step(lds[it & 1], 32 * t, row0);
        }
        if (it + 1 < total) {
            wait_loads();
            wait_lds_barrier();
        }
    }
    if (!active) return;
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan |= !(dk[dt][r] == dk[dt][r]) || !(dv[dt][r] == dv[dt][r]);
    unsigned again = rows_without_number(nan && own);
    const bool whole = own && !(again >> li & 1);
    const int64_t off = ((int64_t)krow * p.Hk + hk) * D;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) {
        store_row_tile<T>((T *)p.dk + off, dt * 32, whole ? D : 0, dk[dt], p.scale, g);
        store_row_tile<T>((T *)p.dv + off, dt * 32, whole ? D : 0, dv[dt], 1.0f, g);
    }
    for (; again; again &= again - 1) row_dkdv<T>(p, s, k0 + __builtin_ctz(again), hk, delta);
}

// ------------------------------------------------------------------ launches

static int64_t packed_tiles(int64_t rows, int n) { return rows / kPackedRows + n + 2; }

}  // namespace

int EVO_CAT(launch_packed_fwd_d, EVO_D)(const EvoPacked &p, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = tiles * p.H;
    if (!grid_fits(grid, 256)) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        packed_fwd<decltype(t)><<<(unsigned)grid, 256, 0, st>>>(p, (int)tiles);
        return hip_rc();
    });
}
int EVO_CAT(launch_packed_bwd_d, EVO_D)(const EvoPacked &p, float *delta, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const int64_t qt = packed_tiles(p.Tq, p.n), kt = packed_tiles(p.Tk, p.n);
    if (!grid_fits(qt * p.H, 256) || !grid_fits(kt * p.Hk, 256)) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        if (p.Tq) {
            packed_dq<T><<<(unsigned)(qt * p.H), 256, 0, st>>>(p, delta, (int)qt);
            if (const int rc = hip_rc()) return rc;
        }
        if (p.Tk && p.dk) packed_dkdv<T><<<(unsigned)(kt * p.Hk), 256, 0, st>>>(p, delta, (int)kt);
        return hip_rc();
    });
}

}  // namespace evo
