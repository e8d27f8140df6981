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
        zero_rows((T *)p.o, at.first, rows, p.H, h, D);
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

    const Staged staged(lane);
    auto step = [&](const unsigned char *buf, int key0) __attribute__((always_inline)) {
        const unsigned at = Staged::base(buf);
        f32x16 a[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            a[t] = filled(0.0f);
#pragma unroll
            for (int ks = 0; ks < R::KSD; ++ks) a[t] = Mfma<T>::mma(staged.rows<T>(at, 32 * t, ks), qf[ks], a[t]);
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
            for (int dt = 0; dt < R::DT; ++dt) o[dt] = Mfma<T>::mma(staged.cols<T>(at + R::ARRAY, (ts / 2) * 32, ts & 1, dt), pf[ts], o[dt]);
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
__global__ void __launch_bounds__(256, EVO_D == 32 ? 4 : EVO_D == 64 ? 3 : 2) packed_dq(EvoPacked p, BackwardRows out_rows, int tiles) {
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
        zero_rows((T *)p.dq, at.first, rows, p.H, h, D);
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
    const float c = p.scale * kLog2e, lse = p.lse[(int64_t)h * p.Tq + qrow];
    if (own && g == 0) {
        out_rows.delta[(int64_t)h * p.Tq + qrow] = -dl;
        out_rows.base[(int64_t)h * p.Tq + qrow] = -lse / c;
    }
    const int seen = s.seen(qrow, p.causal);
    const int wave_least = active ? s.seen(q0, p.causal) : 0, wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    f32x16 dq[R::DT];
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) dq[dt] = filled(0.0f);

    const Staged staged(lane);
    auto step = [&](const unsigned char *buf, int kb, int key0) __attribute__((always_inline)) {
        const unsigned at = Staged::base(buf);
        f32x16 a = filled(0.0f), d = filled(-dl);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) {
            a = Mfma<T>::mma(staged.rows<T>(at, kb, ks), qf[ks], a);
            d = Mfma<T>::mma(staged.rows<T>(at + R::ARRAY, kb, ks), df[ks], d);
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
            for (int dt = 0; dt < R::DT; ++dt) dq[dt] = Mfma<T>::mma(staged.cols<T>(at, kb, ts, dt), pf[ts], dq[dt]);
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

// ------------------------------------------------------------------ launches

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
int EVO_CAT(launch_packed_dq_d, EVO_D)(const EvoPacked &p, const BackwardRows &rows, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = tiles * p.H;
    if (!grid_fits(grid, 256)) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        packed_dq<decltype(t)><<<(unsigned)grid, 256, 0, st>>>(p, rows, (int)tiles);
        return hip_rc();
    });
}

}  // namespace evo
