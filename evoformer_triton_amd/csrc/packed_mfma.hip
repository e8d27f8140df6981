// Attention within packed sequences on the matrix cores, 16-bit, compiled once per head dim (-DEVO_D=32|64|96|128; a head dim between takes the next, with zeros behind it).
//
// A workgroup of four waves takes 128 rows of a sequence and head (forward, dQ: queries; dK/dV: keys), a wave 32 of them, and the other side's rows stream through LDS, a
// stage ahead of the one that is computed on, brought there by the load path itself.  Scores are formed transposed, S^T = K Q^T: a lane then holds 16 keys of one query, the softmax
// needs one exchange with the lane's other half, and the tile is as it lies the operand of O^T = V^T P^T (common.h), whose other operand, V^T, is read from row-major V by
// transposing reads.  Probabilities are formed relative to the maximum so far, which is looked for again only when a lane's sum of 32 of them passes 2^13; they are rounded to the inputs' type to
// multiply V and summed as rounded.
//
// dQ: P again from the forward's lse, dP^T = V dO^T, dS = P (dP - delta), delta = sum of dO times the output and what rounding left of it (the forward keeps both: the output alone is off by half a
// step, and with it every dS of its row by P times that).  dS multiplies K as two values of the inputs' type, what rounding leaves of it as the second: rounded once its share of the error is as large
// as that of rounding the result.  P's and dS's sums over a row, which should be 1 and 0, put right what the rounded probabilities of the forward left in lse and delta: by them dQ is divided, and dK's
// kernel gets both mended.  Errors of dQ and dK next to the formula's in 64 bits, of their norms (chains of 51 to 768 rows, 8 heads of 32, bf16): 0.0019 and 0.0023, where rounding the exact result gives
// 0.0017; without any of this 0.0035 and 0.0033.
//
// What bounds them: the matrix instructions and, at the same time on the same SIMD, exponentials (a quarter of the rate of other instructions) and additions.  Forward, one causal prompt of 16384 rows,
// 32 heads (8 for keys) of 128: 1.95 ms, 1.1 Pflop/s of the 1.30 that a large library product reaches.  Training, 4 x 4096 rows: forward 0.58 ms, dQ 1.06 (its product of K twice), dK and dV 1.09.
// Inputs of zeros take a quarter less time than random ones: the power that the products take has its part in it.
//
// Which rows: tile t of the launch belongs to the last segment j (packed_common.h) with begin(j) / 128 + j <= t; begin(j + 1) / 128 + j + 1 leaves room for all of j's tiles, so that every workgroup finds
// its place by itself, without a sum over the sequences before it and whatever the lengths are; at most one tile per segment finds nothing to do.  A sequence's last queries (first keys), which under a
// causal mask have the longest walks, begin first; of few long sequences all of them by their walks (place_of).
//
// A row of V beyond the sequence's end is read as zeros (the load is out of range).  One that causal queries do not see may hold an infinity or a NaN, which a probability of
// zero does not keep out of the sums: results that may be no numbers because of such a row are formed anew, row by row (packed_common.h).
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

// Stages in LDS: one that is computed on and the others under way.  (Head dim 64, seven prompts of 90 to 2011: 35.0 us with two, 36.1 with three; head dim 32, chains of 51 to 768, forward and dQ: 49.4 with
// four, or three of twice as many keys, and 51.8 with three and two.)
template <int KG> constexpr int kStageBuffers = EVO_D > 32 ? 2 : KG == 2 ? 3 : 4;

// ------------------------------------------------------------------ forward

// KG: groups of four waves that share the queries and take 64 keys of a stage each, joined at the end.  PART: a part of the stages, of which packed_join makes the result.
template <typename T, int KG, bool PART>
__global__ void __launch_bounds__(KG * 256, KG == 2 ? 2 : EVO_D == 32 ? 4 : EVO_D == 64 ? 3 : 2) packed_fwd(EvoPacked p, Parts parts, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4 * KG> Pieces;
    typedef typename Mfma<T>::v8 v8;
    constexpr int BUFS = kStageBuffers<KG>, KEYS = R::STAGE * KG, ARRAY = R::ARRAY * KG;   // of a stage
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int heads = p.H / p.Hk;
    const Unit unit(blockIdx.x, tiles, p.Hk, heads * (PART ? parts.chunks : 1));
    if (unit.none) return;
    const int hk = unit.hk, h = hk * heads + unit.member % heads, part = PART ? unit.member / heads : 0;
    const Place at = place_of<false>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int D = p.D, rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {   // (with parts: packed_join's)
        if (PART) return;
        zero_rows((T *)p.o, at.first, rows, p.H, h, D);
        if (p.o_low) zero_rows((T *)p.o_low, at.first, rows, p.H, h, D);
        if (p.lse && (int)threadIdx.x < rows) p.lse[(int64_t)h * p.Tq + at.first + threadIdx.x] = INFINITY;
        return;
    }
    const int all = (seen_most + KEYS - 1) / KEYS, from = PART ? part_begin(part, parts.chunks, all) : 0, to = PART ? part_begin(part + 1, parts.chunks, all) : all;
    const int kst = (int)p.k_stride_t * 2, vst = (int)p.v_stride_t * 2;
    const char *kbase = (const char *)head_row<T>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = (const char *)head_row<T>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    const int koff = Pieces::first(wave, lane, kst, D), voff = Pieces::first(wave, lane, vst, D);
    auto fetch = [&](int stage) {   // (a stage past the last reads zeros: a wave's loads are as many in every stage)
        const int row = stage * KEYS, n = min(KEYS, s.nk() - row);
        unsigned char *dst = lds + stage % BUFS * (2 * ARRAY);
        Pieces::template fetch<KEYS>(rows_at(kbase + (int64_t)row * kst, n, kst, D), dst, koff, kst, wave);
        Pieces::template fetch<KEYS>(rows_at(vbase + (int64_t)row * vst, n, vst, D), dst + ARRAY, voff, vst, wave);
    };
#pragma unroll
    for (int i = 0; i < BUFS - 1; ++i) fetch(from + i);

    const int own = KG == 1 ? wave : wave & 3, key_group = KG == 1 ? 0 : wave >> 2;
    const int q0 = at.first + own * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1;   // uniform
    v8 qf[R::KSD];
    load_operands(head_row<T>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), D, g, qf);
    asked_together<R::KSD>(qf);   // (and waited for: in the loop the compiler, which does not count the loads into LDS, would wait for the next stage's with them)
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
        const unsigned at = Staged::base(buf) + key_group * R::ARRAY;
        // All operands of a product are asked for together (left to itself the compiler asks for one, waits for it and multiplies), the values' before the softmax
        v8 kf[2][R::KSD], vf[4][R::DT];
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) kf[t][ks] = staged.rows<T>(at, 32 * t, ks);
        __builtin_amdgcn_sched_barrier(0);
        f32x16 a[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) a[t] = filled(0.0f);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) a[t] = Mfma<T>::mma(kf[t][ks], qf[ks], a[t]);
#pragma unroll
        for (int ts = 0; ts < 4; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) vf[ts][dt] = staged.cols<T>(at + ARRAY, (ts / 2) * 32, ts & 1, dt);
        __builtin_amdgcn_sched_barrier(0);
        if (key0 + R::STAGE > wave_least) {   // (uniform)
            asm volatile("");                 // (a branch: not computed where it is not needed)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) a[t][r] = key0 + 32 * t + crow(r, g) < seen ? a[t][r] : -INFINITY;
        }
        // Probabilities relative to the maximum so far, which is looked for only when their sum shows that some score stands far above it (at first any does)
        v8 pf[4];
        auto probabilities = [&] {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int ts = 0; ts < 4; ++ts) {
#pragma unroll
                for (int i = 0; i < 8; ++i) pf[ts][i] = (T)fast_exp2(fmaf(a[ts / 2][8 * (ts & 1) + i], c, -m));
                sum[ts & 1] = dot8<T>(pf[ts], one, sum[ts & 1]);
            }
            return sum[0] + sum[1];
        };
        float sum = probabilities();
        if (__builtin_expect(__any(!(sum <= 8192.0f)), 0)) {
            float top = a[0][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, a[t][r]);
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const float mn = fmaxf(fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * c, m), alpha = fast_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
            sum = probabilities();
        }
        l += sum;
#pragma unroll
        for (int ts = 0; ts < 4; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) o[dt] = Mfma<T>::mma(vf[ts][dt], pf[ts], o[dt]);
    };
    for (int st = from; st < to; ++st) {
        // this stage is there, and everybody has read the one before, whose place the next one to be asked for takes
        wait_loads_but<(BUFS - 2) * 2 * Pieces::each(KEYS)>();
        wait_lds_barrier();
        fetch(st + BUFS - 1);
        const int key0 = st * KEYS + key_group * R::STAGE;
        if (key0 < wave_most) step(lds + st % BUFS * (2 * ARRAY), key0);
    }
    wait_loads();   // (LDS is the next workgroup's from here on)
    if constexpr (KG == 2) {
        // Both groups' sums relative to the larger maximum, the second's added to the first's
        float *const x = reinterpret_cast<float *>(lds) + own * (R::DT * 16 + 3) * 64, *const ml = x + R::DT * 16 * 64;
        wait_lds_barrier();
        ml[key_group * 64 + lane] = m;
        wait_lds_barrier();
        const float mn = fmaxf(ml[lane], ml[64 + lane]), f = fast_exp2(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] *= f;
        if (key_group) {
            give(o, x, lane);
            ml[128 + lane] = l;
        }
        wait_lds_barrier();
        if (key_group) return;
        take(o, x, lane);
        l += ml[128 + lane];
    }
    if (!active) return;
    l += __shfl_xor(l, 32);
    const bool mine = q0 + li < s.q1;
    if constexpr (PART) {
        const int64_t row = ((int64_t)part * p.Tq + qrow) * p.H + h;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) store_row_part(parts.o + row * D, dt * 32, mine ? D : 0, o[dt], g);
        if (mine && g == 0) parts.ml[row] = make_float2(m, l);
        return;
    }
    const float inv = seen ? 1.0f / l : 0.0f;
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[dt][r] = seen ? o[dt][r] * inv : 0.0f;
            nan |= !(o[dt][r] == o[dt][r]);
        }
    // (a sum of zero: every score lies below what the maximum begins with)
    unsigned again = rows_without_number(nan && mine && l == l);
    const unsigned none = rows_without_number(mine && seen && l == 0.0f);
    if (p.lse && mine && g == 0) p.lse[(int64_t)h * p.Tq + qrow] = seen ? m + __log2f(l) : INFINITY;
    const int64_t row = ((int64_t)qrow * p.H + h) * D;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) store_row_tile<T>((T *)p.o + row, dt * 32, mine ? D : 0, o[dt], 1.0f, g);
    if (p.o_low) {
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] = left<T>(o[dt][r]);
            store_row_tile<T>((T *)p.o_low + row, dt * 32, mine ? D : 0, o[dt], 1.0f, g);
        }
    }
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int end = min(s.nk(), (wave_most + R::STAGE - 1) / R::STAGE * R::STAGE);
    if (!spoilt_forward<T>(late, s, hk, wave_least, end)) again = none;
    wait_loads();   // (and for what has been stored, of which some is overwritten)
    for (; again; again &= again - 1) {
        const int b = __builtin_ctz(again), i = q0 + b;
        if ((none >> b & 1) || !all_finite<T>(late.v, late.v_stride_t, hk, late.v_stride_h, s.k0 + s.seen(i, late.causal), s.k0 + end, late.D)) row_forward<T>(late, s, i, h);
    }
}

// ------------------------------------------------------------------ dQ

template <typename T, int KG, bool PART>
__global__ void __launch_bounds__(KG * 256, KG == 2 ? 2 : EVO_D <= 64 ? 3 : 2) packed_dq(EvoPacked p, BackwardRows out_rows, Parts parts, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4 * KG> Pieces;
    typedef typename Mfma<T>::v8 v8;
    constexpr int BUFS = kStageBuffers<KG>, KEYS = R::STAGE * KG, ARRAY = R::ARRAY * KG;   // of a stage
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int heads = p.H / p.Hk;
    const Unit unit(blockIdx.x, tiles, p.Hk, heads * (PART ? parts.chunks : 1));
    if (unit.none) return;
    const int hk = unit.hk, h = hk * heads + unit.member % heads, part = PART ? unit.member / heads : 0;
    const Place at = place_of<false>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int D = p.D, rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {
        if (!PART) zero_rows((T *)p.dq, at.first, rows, p.H, h, D);
        return;
    }
    const int all = (seen_most + KEYS - 1) / KEYS, from = PART ? part_begin(part, parts.chunks, all) : 0, to = PART ? part_begin(part + 1, parts.chunks, all) : all;
    const int kst = (int)p.k_stride_t * 2, vst = (int)p.v_stride_t * 2;
    const char *kbase = (const char *)head_row<T>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = (const char *)head_row<T>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    const int koff = Pieces::first(wave, lane, kst, D), voff = Pieces::first(wave, lane, vst, D);
    auto fetch = [&](int stage) {   // (a stage past the last reads zeros: a wave's loads are as many in every stage)
        const int row = stage * KEYS, n = min(KEYS, s.nk() - row);
        unsigned char *dst = lds + stage % BUFS * (2 * ARRAY);
        Pieces::template fetch<KEYS>(rows_at(kbase + (int64_t)row * kst, n, kst, D), dst, koff, kst, wave);
        Pieces::template fetch<KEYS>(rows_at(vbase + (int64_t)row * vst, n, vst, D), dst + ARRAY, voff, vst, wave);
    };
#pragma unroll
    for (int i = 0; i < BUFS - 1; ++i) fetch(from + i);

    const int own = KG == 1 ? wave : wave & 3, key_group = KG == 1 ? 0 : wave >> 2;
    const int q0 = at.first + own * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1;   // uniform
    const bool mine = q0 + li < s.q1;
    v8 qf[R::KSD], df[R::KSD];
    load_operands(head_row<T>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), D, g, qf);
    load_operands(head_row<T>(p.dout, qrow, p.dout_stride_t, h, p.dout_stride_h), D, g, df);
    float dl = 0.0f;
    {
        v8 of[R::KSD];
        load_operands((const T *)p.o + ((int64_t)qrow * p.H + h) * D, D, g, of);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) dl = dot8<T>(df[ks], of[ks], dl);
        if (p.o_low) {
            load_operands((const T *)p.o_low + ((int64_t)qrow * p.H + h) * D, D, g, of);
#pragma unroll
            for (int ks = 0; ks < R::KSD; ++ks) dl = dot8<T>(df[ks], of[ks], dl);
        }
    }
    dl += __shfl_xor(dl, 32);
    const float c = p.scale * kLog2e;
    float lse[1] = {p.lse[(int64_t)h * p.Tq + qrow]};
    asked_together<R::KSD>(qf);   // (see packed_fwd)
    asked_together<R::KSD>(df);
    asked_together<1>(lse);
    const int seen = s.seen(qrow, p.causal);
    const int wave_least = active ? s.seen(q0, p.causal) : 0, wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    f32x16 dq[R::DT];
    float sum[2] = {0.0f, 0.0f}, rest[2] = {0.0f, 0.0f};   // of the probabilities, which should be 1, and of ds, which should be 0
    float less = lse[0] - (kShifts<T> ? kShiftQuery : 0);  // (and, with dQ, times what this takes off)
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) dq[dt] = filled(0.0f);

    const Staged staged(lane);
    auto step = [&](const unsigned char *buf, int kb, int key0) __attribute__((always_inline)) {
        const unsigned at = Staged::base(buf) + key_group * R::ARRAY;
        v8 kf[R::KSD];
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) kf[ks] = staged.rows<T>(at, kb, ks);
        __builtin_amdgcn_sched_barrier(0);
        f32x16 a = filled(0.0f), d = filled(-dl);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) a = Mfma<T>::mma(kf[ks], qf[ks], a);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) d = Mfma<T>::mma(staged.rows<T>(at + ARRAY, kb, ks), df[ks], d);
        if (key0 + 32 > wave_least) {   // (uniform)
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool sees = key0 + crow(r, g) < seen;
                a[r] = sees ? a[r] : -INFINITY;
                d[r] = sees ? d[r] : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float e = fast_exp2(fmaf(a[r], c, -less));
            sum[r & 1] += e;
            d[r] *= e;
            rest[r & 1] += d[r];
        }
        if constexpr (kShifts<T>) {
            bool any;
            const int down = shift_down(d, any);
            if (__builtin_expect(any, 0)) {
                const float by = ldexpf(1.0f, -down);
                less += (float)down;
                sum[0] *= by;
                sum[1] *= by;
                rest[0] *= by;
                rest[1] *= by;
                d *= by;
                shift_by(dq, by);
            }
        }
#pragma unroll
        for (int ts = 0; ts < 2; ++ts) {
            v8 hi, lo, kt[R::DT];
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) kt[dt] = staged.cols<T>(at, kb, ts, dt);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                hi[i] = (T)d[8 * ts + i];
                lo[i] = (T)left<T>(d[8 * ts + i]);
            }
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) dq[dt] = Mfma<T>::mma(kt[dt], hi, dq[dt]);
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) dq[dt] = Mfma<T>::mma(kt[dt], lo, dq[dt]);
        }
    };
    for (int st = from; st < to; ++st) {
        wait_loads_but<(BUFS - 2) * 2 * Pieces::each(KEYS)>();
        wait_lds_barrier();
        fetch(st + BUFS - 1);
        // (interleaved for D = 64 they would need more than the 168 registers of three waves to a SIMD: 10 of them would live in memory)
#pragma unroll (EVO_D == 64 ? 1 : 2)
        for (int t = 0; t < 2; ++t) {
            const int key0 = st * KEYS + key_group * R::STAGE + 32 * t;
            if (key0 < wave_most) step(lds + st % BUFS * (2 * ARRAY), 32 * t, key0);
        }
    }
    wait_loads();
    sum[0] += sum[1];
    rest[0] += rest[1];
    if constexpr (kShifts<T>) {   // (of a row that sees nothing there are no sums; the difference is a whole number, but for its rounding)
        const float by = ldexpf(1.0f, seen ? (int)rintf(less - lse[0]) : 0);
        sum[0] *= by;
        rest[0] *= by;
        shift_by(dq, by);
    }
    if constexpr (KG == 2) {
        float *const x = reinterpret_cast<float *>(lds) + own * (R::DT * 16 + 2) * 64, *const more = x + R::DT * 16 * 64;
        wait_lds_barrier();
        if (key_group) {
            give(dq, x, lane);
            more[lane] = sum[0];
            more[64 + lane] = rest[0];
        }
        wait_lds_barrier();
        if (key_group) return;
        take(dq, x, lane);
        sum[0] += more[lane];
        rest[0] += more[64 + lane];
    }
    if (!active) return;
    sum[0] += __shfl_xor(sum[0], 32);
    rest[0] += __shfl_xor(rest[0], 32);
    if constexpr (PART) {
        const int64_t row = ((int64_t)part * p.Tq + qrow) * p.H + h;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) store_row_part(parts.o + row * D, dt * 32, mine ? D : 0, dq[dt], g);
        if (mine && g == 0) {
            parts.ml[row] = make_float2(sum[0], rest[0]);
            if (part == 0) out_rows.delta[(int64_t)h * p.Tq + qrow] = dl;
        }
        return;
    }
    const float inv = seen ? 1.0f / sum[0] : 0.0f;
    if (mine && g == 0) save_row(out_rows, (int64_t)h * p.Tq + qrow, lse[0], dl, sum[0], rest[0], c);
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan |= !(dq[dt][r] == dq[dt][r]);
    // (an infinite dS has no second value)
    unsigned again = rows_without_number(nan && mine && rest[0] == rest[0]);
    const unsigned infinite = rows_without_number(mine && fabsf(rest[0]) == INFINITY) & again;
    T *out = (T *)p.dq + ((int64_t)qrow * p.H + h) * D;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) store_row_tile<T>(out, dt * 32, mine ? D : 0, dq[dt], p.scale * inv, g);
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int end = min(s.nk(), (wave_most + 31) / 32 * 32);
    if (!spoilt_dq<T>(late, s, hk, wave_least, end)) again = infinite;
    wait_loads();   // (see packed_fwd)
    for (; again; again &= again - 1) {
        const int b = __builtin_ctz(again), i = q0 + b;
        if ((infinite >> b & 1) || spoilt_dq<T>(late, s, hk, s.seen(i, late.causal), end)) row_dq<T>(late, s, i, h, lane_value(dl, b));
    }
}

// ------------------------------------------------------------------ launches

}  // namespace

size_t EVO_CAT(packed_fwd_bytes_d, EVO_D)(const EvoPacked &p) { return EVO_CAT(packed_d, EVO_D)::query_plan(p).bytes(p.Tq * p.H, p.D + 2); }
int EVO_CAT(launch_packed_join_d, EVO_D)(const EvoPacked &p, float *o, float2 *ml, int parts, hipStream_t st);
int EVO_CAT(launch_packed_fwd_d, EVO_D)(const EvoPacked &p, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const Plan plan = query_plan(p);
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = Unit::grid(tiles, p.Hk, p.H / p.Hk * plan.parts), rows = p.Tq * p.H;
    if (!grid_fits(grid, 256 * plan.groups) || (plan.parts > 1 && (rows > INT32_MAX || !grid_fits(rows, 256)))) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        return plan.run([&](auto groups, auto part) {
            constexpr int KG = decltype(groups)::value, LDS = kStageBuffers<KG> * 2 * PackedGeo::ARRAY * KG;
            constexpr auto kern = packed_fwd<T, KG, decltype(part)::value>;
            static PerDevice done;
            if (const int rc = ensure_dynamic_lds((const void *)kern, LDS, done, nullptr)) return rc;
            float *const o = (float *)p.workspace;
            const Parts parts = {o, (float2 *)(o + plan.parts * rows * p.D), 0, plan.parts};
            kern<<<(unsigned)grid, 256 * KG, LDS, st>>>(p, parts, (int)tiles);
            const int rc = hip_rc();
            return rc || !decltype(part)::value ? rc : EVO_CAT(launch_packed_join_d, EVO_D)(p, parts.o, parts.ml, parts.chunks, st);
        });
    });
}
size_t EVO_CAT(packed_dq_bytes_d, EVO_D)(const EvoPacked &p) { return EVO_CAT(packed_d, EVO_D)::query_plan(p).bytes(p.Tq * p.H, p.D + 2); }
int EVO_CAT(launch_packed_dq_d, EVO_D)(const EvoPacked &p, const BackwardRows &saved, float *sums, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const Plan plan = query_plan(p);
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = Unit::grid(tiles, p.Hk, p.H / p.Hk * plan.parts), rows = p.Tq * p.H;
    if (!grid_fits(grid, 256 * plan.groups) || (plan.parts > 1 && !row_waves_fit(rows))) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        return plan.run([&](auto groups, auto part) {
            constexpr int KG = decltype(groups)::value, LDS = kStageBuffers<KG> * 2 * PackedGeo::ARRAY * KG;
            constexpr auto kern = packed_dq<T, KG, decltype(part)::value>;
            static PerDevice done;
            if (const int rc = ensure_dynamic_lds((const void *)kern, LDS, done, nullptr)) return rc;
            const Parts parts = {sums, (float2 *)(sums + plan.parts * rows * p.D), 0, plan.parts};
            kern<<<(unsigned)grid, 256 * KG, LDS, st>>>(p, saved, parts, (int)tiles);
            if (const int rc = hip_rc()) return rc;
            if (!decltype(part)::value) return (int)EVO_OK;
            packed_sum<T, false><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, saved, parts, (unsigned)rows);
            return hip_rc();
        });
    });
}

}  // namespace evo
