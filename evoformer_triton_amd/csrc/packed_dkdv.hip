// Attention within packed sequences on the matrix cores: dK and dV (see packed_mfma.hip).
//
// A wave has 32 keys, a column of the products' each, and walks over the queries of all heads that share the key head: S = Q K^T and dP = dO V^T begin with what is subtracted from them (-lse in units of
// q . k, -delta; staged in LDS beside the rows), P and dS as they lie are operands of dV^T = dO^T P and dK^T = Q^T dS.  Four products for each pair of rows, their other operands from LDS: for head dims
// above 64 V's too, since with K's, dK and dV in registers (2 waves to a SIMD) there is no room for them.  4 x 4096 causal rows, 32 heads (8) of 128: 1.09 ms, 1.0 Pflop/s; what is left of the rate of
// a large product goes into LDS's reads, of which each product needs two, and into exponentials.
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

// ------------------------------------------------------------------ dK, dV

// KG: groups of four waves that share the keys and take a part of each stage's queries, joined at the end.  PART: a part of the walk, all of which packed_sum adds up.
template <int KG> struct KeyGeo {
    typedef PackedGeo::G G;
    static constexpr int SUB = EVO_D > 64 ? 32 : 64, ROWS = SUB * KG;                  // queries of a stage to a group, and of a stage
    static constexpr int ARRAY = ROWS * G::ROW, BYTES = 2 * ARRAY + 1024;              // Q, dO, then for each 64 queries what their products begin with, 64 places each
    static constexpr bool VLDS = EVO_D > 64;                                           // V's operands from LDS with each use, else kept in registers
    static constexpr int LDS = 2 * BYTES + (VLDS ? kPackedRows * G::ROW : 0);
    static_assert(4 * PackedGeo::DT * 16 * 64 * 4 <= LDS, "a group's sums of dK or dV fit");
};
template <typename T, int KG, bool PART>
__global__ void __launch_bounds__(KG * 256, KG == 1 && EVO_D == 32 ? 3 : 2) packed_dkdv(EvoPacked p, BackwardRows saved, Parts parts, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef KeyGeo<KG> K;
    typedef StagePieces<4 * KG> Pieces;
    typedef typename Mfma<T>::v8 v8;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];   // two stages, then (VLDS) V
    unsigned char *const vlds = lds + 2 * K::BYTES;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int own = KG == 1 ? wave : wave & 3, row_group = KG == 1 ? 0 : wave >> 2;
    const int group = p.H / p.Hk;
    const Unit unit(blockIdx.x, tiles, p.Hk, PART ? parts.chunks : 1);
    if (unit.none) return;
    const int hk = unit.hk;
    const Place at = place_of<true>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.k1) return;
    const int D = p.D, rows = min(kPackedRows, s.k1 - at.first);
    const int begin = s.first_query(at.first, p.causal);   // that sees any of the workgroup's keys
    if (s.gap || begin >= s.q1) {
        if (PART) return;
        zero_rows((T *)p.dk, at.first, rows, p.Hk, hk, D);
        zero_rows((T *)p.dv, at.first, rows, p.Hk, hk, D);
        return;
    }
    const int qst = (int)p.q_stride_t * 2, dst_ = (int)p.dout_stride_t * 2;
    const int qoff = Pieces::first(wave, lane, qst, D), doff = Pieces::first(wave, lane, dst_, D);
    const int stages = (s.q1 - begin + K::ROWS - 1) / K::ROWS;
    auto fetch = [&](int h, int stage, unsigned char *dst) {
        const int row = begin + stage * K::ROWS, n = min(K::ROWS, s.q1 - row);
        Pieces::template fetch<K::ROWS>(rows_at(head_row<T>(p.q, row, p.q_stride_t, h, p.q_stride_h), n, qst, D), dst, qoff, qst, wave);
        Pieces::template fetch<K::ROWS>(rows_at(head_row<T>(p.dout, row, p.dout_stride_t, h, p.dout_stride_h), n, dst_, D), dst + K::ARRAY, doff, dst_, wave);
        if (wave < (K::ROWS > 64 ? 4 : 2)) {   // (a number to a lane; rows past the end: zero)
            const int first = (wave >> 1) * 64;
            const float *x = (wave & 1 ? saved.delta : saved.base) + (int64_t)h * p.Tq + row + first;
            dma4(__builtin_amdgcn_make_buffer_rsrc((void *)x, 0, max(0, n - first) * 4, 0x00020000), dst + 2 * K::ARRAY + wave * 256, lane * 4);
        }
    };
    const int total = stages * group, from = PART ? part_begin(unit.member, parts.chunks, total) : 0, to = PART ? part_begin(unit.member + 1, parts.chunks, total) : total;
    int h = hk * group + from / stages, stage = from % stages;
    if (from < to) fetch(h, stage, lds);
    const int k0 = at.first + own * 32, krow = min(k0 + li, s.k1 - 1);
    const bool active = k0 < s.k1, mine = k0 + li < s.k1;
    if (K::VLDS) {   // (rows past the sequence's end: zeros)
        const int vst = (int)p.v_stride_t * 2, voff = Pieces::first(wave, lane, vst, D);
        Pieces::template fetch<kPackedRows>(rows_at(head_row<T>(p.v, at.first, p.v_stride_t, hk, p.v_stride_h), rows, vst, D), vlds, voff, vst, wave);
    }
    v8 kf[R::KSD], vf[K::VLDS ? 1 : R::KSD];
    load_operands(head_row<T>(p.k, krow, p.k_stride_t, hk, p.k_stride_h), D, g, kf);
    if constexpr (!K::VLDS) load_operands(head_row<T>(p.v, krow, p.v_stride_t, hk, p.v_stride_h), D, g, vf);
    asked_together<R::KSD>(kf);   // (and waited for: see packed_fwd)
    if constexpr (!K::VLDS) asked_together<R::KSD>(vf);
    // the first query that sees this lane's key, the wave's first one and its last one
    const int key_from = s.first_query(krow, p.causal), wave_from = s.first_query(k0, p.causal), wave_to = s.first_query(min(k0 + 31, s.k1 - 1), p.causal);
    const float c = p.scale * kLog2e;
    f32x16 dk[R::DT], dv[R::DT];
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) dk[dt] = dv[dt] = filled(0.0f);
    float by = 0x1p17f;   // (kShifts: P, and with it dV, are times 2^kShiftKey, dS and dK times this too)

    const Staged staged(lane);
    auto step = [&](const unsigned char *buf, int qb, int row0) __attribute__((always_inline)) {
        const unsigned at = Staged::base(buf), vat = Staged::base(vlds) + own * 32 * G::ROW;
        // (the products begin with what is subtracted from them)
        const float *sub = reinterpret_cast<const float *>(buf + 2 * K::ARRAY + (qb >> 6) * 512) + (qb & 63) + 4 * g;
        auto begin_with = [&](const float *from) __attribute__((always_inline)) {
            f32x16 t;
#pragma unroll
            for (int rr = 0; rr < 4; ++rr) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(from + 8 * rr);
#pragma unroll
                for (int i = 0; i < 4; ++i) t[4 * rr + i] = x[i];
            }
            return t;
        };
        f32x16 a = begin_with(sub);
        const unsigned qat = at + (unsigned)(qb * G::ROW), dat = qat + K::ARRAY;
        v8 x[R::KSD];
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) x[ks] = staged.rows<T>(qat, 0, ks);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) a = Mfma<T>::mma(x[ks], kf[ks], a);
        f32x16 d = begin_with(sub + 64);
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) d = Mfma<T>::mma(staged.rows<T>(dat, 0, ks), K::VLDS ? staged.rows<T>(vat, 0, ks) : vf[K::VLDS ? 0 : ks], d);
#pragma unroll
        for (int r = 0; r < 16; ++r) a[r] = fast_exp2(kShifts<T> ? fmaf(a[r], c, (float)kShiftKey) : a[r] * c);
        if (row0 < wave_to) {   // (uniform)
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool sees = row0 + crow(r, g) >= key_from;
                a[r] = sees ? a[r] : 0.0f;
                d[r] = sees ? d[r] : 0.0f;
            }
        }
        if constexpr (kShifts<T>) {
            d *= a;
            d *= by;
            bool any;
            const int down = shift_down(d, any);
            if (__builtin_expect(any, 0)) {
                const float more = ldexpf(1.0f, -down);
                by *= more;
                d *= more;
                shift_by(dk, more);
            }
        }
        v8 pf[2], sf[2];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int i = 0; i < 8; ++i) pf[ts][i] = (T)a[8 * ts + i];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) dv[dt] = Mfma<T>::mma(staged.cols<T>(dat, 0, ts, dt), pf[ts], dv[dt]);
        // (without this head dim 128 keeps one of K's operands in memory, whose way back is waited for with all that is on its way into LDS: 1.16 ms instead of 1.09 for the size above)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int i = 0; i < 8; ++i) sf[ts][i] = (T)(kShifts<T> ? d[8 * ts + i] : a[8 * ts + i] * d[8 * ts + i]);
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) dk[dt] = Mfma<T>::mma(staged.cols<T>(qat, 0, ts, dt), sf[ts], dk[dt]);
    };
    wait_loads();
    wait_lds_barrier();
    for (int it = from; it < to; ++it) {
        const int row = begin + stage * K::ROWS;
        const unsigned char *const buf = lds + ((it - from) & 1) * K::BYTES;
        if (++stage == stages) {
            stage = 0;
            ++h;
        }
        if (it + 1 < to) fetch(h, stage, lds + ((it + 1 - from) & 1) * K::BYTES);
        for (int t = 0; t < K::SUB / 32; ++t) {
            const int qb = row_group * K::SUB + 32 * t, row0 = row + qb;
            if (active && row0 < s.q1 && row0 + 31 >= wave_from) step(buf, qb, row0);
        }
        if (it + 1 < to) {
            wait_loads();
            wait_lds_barrier();
        }
    }
    wait_loads();
    if constexpr (kShifts<T>) {
        const float back = ldexpf(1.0f, -kShiftKey);
        shift_by(dk, back / by);
        shift_by(dv, back);
    }
    if constexpr (KG == 2) {
        float *const x = reinterpret_cast<float *>(lds) + own * R::DT * 16 * 64;
        wait_lds_barrier();
        if (row_group) give(dk, x, lane);
        wait_lds_barrier();
        if (!row_group) take(dk, x, lane);
        wait_lds_barrier();
        if (row_group) give(dv, x, lane);
        wait_lds_barrier();
        if (row_group) return;
        take(dv, x, lane);
    }
    if (!active) return;
    const int64_t row = (int64_t)krow * p.Hk + hk;
    if constexpr (PART) {
        const int64_t all = p.Tk * p.Hk;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) {
            store_row_part(parts.o + (unit.member * all + row) * D, dt * 32, mine ? D : 0, dk[dt], g);
            store_row_part(parts.o + ((parts.chunks + unit.member) * all + row) * D, dt * 32, mine ? D : 0, dv[dt], g);
        }
        return;
    }
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan |= !(dk[dt][r] == dk[dt][r]) || !(dv[dt][r] == dv[dt][r]);
    unsigned again = rows_without_number(nan && mine);
#pragma unroll
    for (int dt = 0; dt < R::DT; ++dt) {
        store_row_tile<T>((T *)p.dk + row * D, dt * 32, mine ? D : 0, dk[dt], p.scale, g);
        store_row_tile<T>((T *)p.dv + row * D, dt * 32, mine ? D : 0, dv[dt], 1.0f, g);
    }
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int least = max(begin, wave_from - 31);   // (of the queries that a step of the wave's has)
    if (!spoilt_dkdv<T>(late, s, hk, k0, min(k0 + 32, s.k1), least, wave_to, saved.delta)) return;
    wait_loads();   // (see packed_fwd)
    for (; again; again &= again - 1) {
        const int j = k0 + __builtin_ctz(again);
        if (spoilt_dkdv<T>(late, s, hk, j, j + 1, least, s.first_query(j, late.causal), saved.delta)) row_dkdv<T>(late, s, j, hk, saved.delta);
    }
}

}  // namespace

size_t EVO_CAT(packed_dkdv_bytes_d, EVO_D)(const EvoPacked &p) { return EVO_CAT(packed_d, EVO_D)::key_plan(p).bytes(p.Tk * p.Hk, 2 * p.D); }
int EVO_CAT(launch_packed_dkdv_d, EVO_D)(const EvoPacked &p, const BackwardRows &saved, float *sums, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const Plan plan = key_plan(p);
    const int64_t tiles = packed_tiles(p.Tk, p.n), grid = Unit::grid(tiles, p.Hk, plan.parts), rows = p.Tk * p.Hk;
    if (!grid_fits(grid, 256 * plan.groups) || (plan.parts > 1 && !row_waves_fit(rows))) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        return plan.run([&](auto groups, auto part) {
            constexpr int KG = decltype(groups)::value;
            constexpr auto kern = packed_dkdv<T, KG, decltype(part)::value>;
            static PerDevice done;
            if (const int rc = ensure_dynamic_lds((const void *)kern, KeyGeo<KG>::LDS, done, nullptr)) return rc;
            const Parts parts = {sums, nullptr, 0, plan.parts};
            kern<<<(unsigned)grid, 256 * KG, KeyGeo<KG>::LDS, st>>>(p, saved, parts, (int)tiles);
            if (const int rc = hip_rc()) return rc;
            if (!decltype(part)::value) return (int)EVO_OK;
            packed_sum<T, true><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, saved, parts, (unsigned)rows);
            return hip_rc();
        });
    });
}

}  // namespace evo
