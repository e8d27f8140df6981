// Attention within packed sequences on the matrix cores: dK and dV (see packed_mfma.hip).
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

// ------------------------------------------------------------------ dK, dV

// KT: key tiles of 32 to a wave.
template <typename T, int KT>
__global__ void __launch_bounds__(256, KT == 2 ? 1 : 2) packed_dkdv(EvoPacked p, BackwardRows rows, int tiles) {
    typedef PackedGeo R;
    typedef R::G G;
    typedef StagePieces<4> Pieces;
    typedef typename Mfma<T>::v8 v8;
    constexpr int KEYS = 128 * KT;               // of a workgroup
    constexpr int ROWS = EVO_D > 64 && KT == 1 ? 32 : 64;   // queries of a stage
    constexpr int ARRAY = ROWS * G::ROW, BYTES = 2 * ARRAY + 2 * 256;   // Q, dO, then 64 places each for lse and delta
    constexpr bool VLDS = EVO_D > 64;   // V's operands from LDS with each use, else kept in registers
    constexpr int STAGE_BYTES = (BYTES + 1023) / 1024 * 1024;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];   // two stages, then (VLDS) V
    unsigned char *const vlds = lds + 2 * STAGE_BYTES;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int group = p.H / p.Hk;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x);
    const int hk = (int)(lid / (unsigned)tiles);
    const Place at = place_of<true, KEYS>(p, (int)(lid % (unsigned)tiles));   // (a sequence's first keys, which causal queries see most of, first)
    const Segment &s = at.s;
    if (at.first >= s.k1) return;
    const int D = p.D;
    // the first query that sees the workgroup's first key
    const int more = s.nk() - s.nq(), begin = s.q0 + (p.causal ? max(0, at.first - s.k0 - more) : 0);
    if (s.gap || begin >= s.q1) {
        zero_rows((T *)p.dk, at.first, min(KEYS, s.k1 - at.first), p.Hk, hk, D);
        zero_rows((T *)p.dv, at.first, min(KEYS, s.k1 - at.first), p.Hk, hk, D);
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
            const float *x = (wave ? rows.delta : rows.base) + (int64_t)h * p.Tq + row;
            dma4(__builtin_amdgcn_make_buffer_rsrc((void *)x, 0, n * 4, 0x00020000), dst + 2 * ARRAY + wave * 256, lane * 4);
        }
    };
    int h = hk * group, stage = 0;
    fetch(h, 0, lds);
    const int k0 = at.first + wave * 32 * KT;
    const bool active = k0 < s.k1;
    if (VLDS) {   // (rows past the sequence's end: zeros)
        const int vst = (int)p.v_stride_t * 2, voff = Pieces::first(wave, lane, vst, D);
#pragma unroll
        for (int t = 0; t < KEYS / 64; ++t) {
            const int row = at.first + 64 * t;
            Pieces::fetch<64>(rows_at(head_row<T>(p.v, row, p.v_stride_t, hk, p.v_stride_h), min(64, s.k1 - row), vst, D), vlds + t * 64 * G::ROW, voff, vst, wave);
        }
    }
    v8 kf[KT][R::KSD], vf[VLDS ? 1 : KT][R::KSD];
    int from[KT];   // the first query that sees this lane's key, as a row of the tensor
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int krow = min(k0 + 32 * t + li, s.k1 - 1);
        load_operands(head_row<T>(p.k, krow, p.k_stride_t, hk, p.k_stride_h), D, g, kf[t]);
        if constexpr (!VLDS) load_operands(head_row<T>(p.v, krow, p.v_stride_t, hk, p.v_stride_h), D, g, vf[t]);
        from[t] = p.causal ? s.q0 + max(0, krow - s.k0 - more) : s.q0;
    }
    // that of the wave's first key and of its last one
    const int wave_from = p.causal ? s.q0 + max(0, k0 - s.k0 - more) : s.q0, wave_to = p.causal ? s.q0 + max(0, min(k0 + 32 * KT - 1, s.k1 - 1) - s.k0 - more) : s.q0;
    const float c = p.scale * kLog2e;
    f32x16 dk[KT][R::DT], dv[KT][R::DT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) dk[t][dt] = dv[t][dt] = filled(0.0f);

    const Staged staged(lane);
    auto step = [&](const unsigned char *buf, int qb, int row0) __attribute__((always_inline)) {
        const unsigned at = Staged::base(buf), vat = Staged::base(vlds) + wave * 32 * KT * G::ROW;
        // (the products begin with what is subtracted from them)
        const float *sub = reinterpret_cast<const float *>(buf + 2 * ARRAY) + qb + 4 * g;
        f32x16 a[KT], d[KT];
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(sub + 8 * rr), y = *reinterpret_cast<const f32x4 *>(sub + 64 + 8 * rr);
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[t][4 * rr + i] = x[i];
                    d[t][4 * rr + i] = y[i];
                }
        }
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) {
            const v8 x = staged.rows<T>(at, qb, ks);
#pragma unroll
            for (int t = 0; t < KT; ++t) a[t] = Mfma<T>::mma(x, kf[t][ks], a[t]);
        }
#pragma unroll
        for (int ks = 0; ks < R::KSD; ++ks) {
            const v8 x = staged.rows<T>(at + ARRAY, qb, ks);
#pragma unroll
            for (int t = 0; t < KT; ++t) d[t] = Mfma<T>::mma(x, VLDS ? staged.rows<T>(vat, 32 * t, ks) : vf[VLDS ? 0 : t][ks], d[t]);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) a[t][r] = fast_exp2(a[t][r] * c);
        if (row0 < wave_to) {   // (uniform)
            asm volatile("");
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool sees = row0 + crow(r, g) >= from[t];
                    a[t][r] = sees ? a[t][r] : 0.0f;
                    d[t][r] = sees ? d[t][r] : 0.0f;
                }
        }
        v8 pf[KT][2], sf[KT][2];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int ts = 0; ts < 2; ++ts)
#pragma unroll
                for (int i = 0; i < 8; ++i) pf[t][ts][i] = (T)a[t][8 * ts + i];
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) {
                const v8 x = staged.cols<T>(at + ARRAY, qb, ts, dt);
#pragma unroll
                for (int t = 0; t < KT; ++t) dv[t][dt] = Mfma<T>::mma(x, pf[t][ts], dv[t][dt]);
            }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int ts = 0; ts < 2; ++ts)
#pragma unroll
                for (int i = 0; i < 8; ++i) sf[t][ts][i] = (T)(a[t][8 * ts + i] * d[t][8 * ts + i]);
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
#pragma unroll
            for (int dt = 0; dt < R::DT; ++dt) {
                const v8 x = staged.cols<T>(at, qb, ts, dt);
#pragma unroll
                for (int t = 0; t < KT; ++t) dk[t][dt] = Mfma<T>::mma(x, sf[t][ts], dk[t][dt]);
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
        if (it + 1 < total) fetch(h, stage, lds + ((it + 1) & 1) * STAGE_BYTES);
        for (int t = 0; t < ROWS / 32; ++t) {
            const int row0 = row + 32 * t;
            if (active && row0 < s.q1 && row0 + 31 >= wave_from) step(lds + (it & 1) * STAGE_BYTES, 32 * t, row0);
        }
        if (it + 1 < total) {
            wait_loads();
            wait_lds_barrier();
        }
    }
    if (!active) return;
    bool nan[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        nan[t] = false;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) nan[t] |= !(dk[t][dt][r] == dk[t][dt][r]) || !(dv[t][dt][r] == dv[t][dt][r]);
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = k0 + 32 * t + li, krow = min(key, s.k1 - 1);
        unsigned again = rows_without_number(nan[t] && key < s.k1);
        const bool whole = key < s.k1 && !(again >> li & 1);
        const int64_t off = ((int64_t)krow * p.Hk + hk) * D;
#pragma unroll
        for (int dt = 0; dt < R::DT; ++dt) {
            store_row_tile<T>((T *)p.dk + off, dt * 32, whole ? D : 0, dk[t][dt], p.scale, g);
            store_row_tile<T>((T *)p.dv + off, dt * 32, whole ? D : 0, dv[t][dt], 1.0f, g);
        }
        for (; again; again &= again - 1) row_dkdv<T>(p, s, k0 + 32 * t + __builtin_ctz(again), hk, rows.delta);
    }
}

}  // namespace

int EVO_CAT(launch_packed_dkdv_d, EVO_D)(const EvoPacked &p, const BackwardRows &rows, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    constexpr int KT = 1;
    const int64_t tiles = packed_tiles(p.Tk, p.n, 128 * KT), grid = tiles * p.Hk;
    if (!grid_fits(grid, 256)) return EVO_EOVERFLOW;
    return by_half(p.dtype, [&](auto t) {
        constexpr auto kern = packed_dkdv<decltype(t), KT>;
        constexpr int ROWS = EVO_D > 64 && KT == 1 ? 32 : 64, LDS = 2 * ((2 * ROWS * PackedGeo::G::ROW + 512 + 1023) / 1024 * 1024) + (EVO_D > 64 ? 128 * KT * PackedGeo::G::ROW : 0);
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kern, LDS, done, nullptr)) return rc;
        kern<<<(unsigned)grid, 256, LDS, st>>>(p, rows, (int)tiles);
        return hip_rc();
    });
}

}  // namespace evo
