// Attention within packed sequences in fp32 on the matrix cores (v_mfma_f32_32x32x2_f32), compiled once per head dim (-DEVO_D=32|64|96|128; smaller ones: columns of zeros).
//
// A wave has 32 queries (dK and dV: keys), a column of the products' each, and walks over the other side, 32 rows to a stage that the workgroup's four waves share in LDS:
//   S^T = K Q^T with Q's values in registers, lane (column, g) has those 8 s + 4 g .. + 3: a vector of four of K's row, read from LDS, and four of them are four products' operands;
//   O^T = V^T P^T: register r of S^T is row 8 (r / 4) + 4 g + r % 4 of it, so that it is, as it lies, the operand of the product with these two rows (one for each g) of V.
// dQ^T = K^T dS^T, dV^T = dO^T P and dK^T = Q^T dS likewise.  One product takes 64 cycles of a SIMD for the 256 bytes that it reads from LDS, a multiply-add in fp32 for each clock and lane: what
// bounds the kernels is these, and what else there is (exponentials, the next stage's way from memory over registers into the other half of LDS) goes on beside them.  Rows in LDS are four
// values longer than the head dim: vectors of 16 rows then lie in banks of their own.
// Walks are split into parts where tiles are few (the chip is filled, and a causal mask's long walks do not wait for each other); a second kernel joins or adds up the parts, in their order.
// 2 sequences of up to 4096 rows, 16 heads (4 for keys) of 128, causal: 1.21 ms (113 Tflop/s of the 157 that the instruction has), with gradients 5.4 ms; a row by a wave on the
// vector unit instead: one such sequence and 8 heads 30 ms, here 0.39.  One token against 131072 keys, 16 heads (2): 0.10 ms.
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

struct F32Geo {
    static constexpr int STAGE = 32, PITCH = EVO_D + 4, ARRAY = STAGE * PITCH;   // rows of a stage; in values
    static constexpr int KS = EVO_D / 8, DT = EVO_D / 32;
    static constexpr int LDS = 2 * 2 * (ARRAY + STAGE) * 4;                      // two stages of two arrays, and (dK, dV) two numbers to a row
};

// Four values of a row from column c on; zeros from D on.  vec: rows begin at, and D is, a multiple of 16 bytes
__device__ __forceinline__ f32x4 four(const float *row, int c, int D, bool vec) {
    if (vec) return c < D ? *reinterpret_cast<const f32x4 *>(row + c) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = c + i < D ? row[c + i] : 0.0f;
    return x;
}
__device__ __forceinline__ void store_four(float *row, int c, int D, bool vec, f32x4 x) {
    if (vec) {
        if (c < D) *reinterpret_cast<f32x4 *>(row + c) = x;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c + i < D) row[c + i] = x[i];
}
// A row's values as operands
__device__ __forceinline__ void load_values(const float *row, int g, int D, bool vec, f32x4 (&x)[F32Geo::KS]) {
#pragma unroll
    for (int s = 0; s < F32Geo::KS; ++s) x[s] = four(row, 8 * s + 4 * g, D, vec);
}
// A result's row
__device__ __forceinline__ void store_values(float *row, int g, int D, bool vec, const f32x16 (&x)[F32Geo::DT], float scale) {
#pragma unroll
    for (int dt = 0; dt < F32Geo::DT; ++dt)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
            store_four(row, dt * 32 + 8 * rr + 4 * g, D, vec, f32x4{x[dt][4 * rr] * scale, x[dt][4 * rr + 1] * scale, x[dt][4 * rr + 2] * scale, x[dt][4 * rr + 3] * scale});
}
__device__ __forceinline__ void zero_values(float *x, int first, int rows, int heads, int h, int D) {
    for (int i = threadIdx.x; i < rows * D; i += blockDim.x) x[((int64_t)(first + i / D) * heads + h) * D + i % D] = 0.0f;
}
__device__ __forceinline__ bool no_number(const f32x16 (&x)[F32Geo::DT]) {
    bool nan = false;
#pragma unroll
    for (int dt = 0; dt < F32Geo::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan |= !(x[dt][r] == x[dt][r]);
    return nan;
}

// The share of one of THREADS threads in 32 rows on their way into LDS: row threadIdx.x / 8 and every THREADS / 8 on, four values in every 32; zeros from `rows` on.
template <int THREADS = 256>
struct F32Share {
    static constexpr int EACH = 256 / THREADS;
    f32x4 x[EACH][F32Geo::DT];
    __device__ __forceinline__ void ask(const float *base, int64_t stride, int rows, int D, bool vec) {
        const int c = (threadIdx.x & 7) * 4;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int r = (threadIdx.x >> 3) + e * (THREADS / 8);
#pragma unroll
            for (int i = 0; i < F32Geo::DT; ++i) x[e][i] = r < rows ? four(base + r * stride, c + 32 * i, D, vec) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    __device__ __forceinline__ void put(float *to) const {
        const int c = (threadIdx.x & 7) * 4;
#pragma unroll
        for (int e = 0; e < EACH; ++e)
#pragma unroll
            for (int i = 0; i < F32Geo::DT; ++i) *reinterpret_cast<f32x4 *>(to + ((threadIdx.x >> 3) + e * (THREADS / 8)) * F32Geo::PITCH + c + 32 * i) = x[e][i];
    }
};
__device__ __forceinline__ f32x16 mma2(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
// The products of the 32 staged rows with the wave's own
__device__ __forceinline__ f32x16 times(const float *staged, const f32x4 (&own)[F32Geo::KS], int li, int g) {
    f32x16 a = filled(0.0f);
#pragma unroll
    for (int s = 0; s < F32Geo::KS; ++s) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(staged + li * F32Geo::PITCH + 8 * s + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) a = mma2(x[i], own[s][i], a);
    }
    return a;
}
// The staged rows' sum with weights w, a column of the result for each of the wave's own rows
__device__ __forceinline__ void add_weighted(f32x16 (&sum)[F32Geo::DT], const float *staged, const f32x16 &w, int li, int g) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int dt = 0; dt < F32Geo::DT; ++dt) sum[dt] = mma2(staged[crow(r, g) * F32Geo::PITCH + dt * 32 + li], w[r], sum[dt]);
}

// The staged keys from key0 on added to the outputs o and sums l relative to 2^m; of them those below `seen` are seen.
__device__ __forceinline__ void add_keys(f32x16 (&o)[F32Geo::DT], float &m, float &l, const float *K, const float *V, const f32x4 (&q)[F32Geo::KS], int key0, int seen, float c, int li, int g) {
    f32x16 a = times(K, q, li, g);
    if (__any(key0 + F32Geo::STAGE > seen)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) a[r] = key0 + crow(r, g) < seen ? a[r] : -INFINITY;
    }
    float top = a[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, a[r]);
    const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)) * c);
    if (__any(mn > m)) {
        const float alpha = fast_exp2(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < F32Geo::DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        a[r] = fast_exp2(fmaf(a[r], c, -m));
        sum += a[r];
    }
    l += sum;
    add_weighted(o, V, a, li, g);
}

// PART: a part of the stages, of which packed_f32_join makes the result.
template <bool VEC, bool PART>
__global__ void __launch_bounds__(256, 2) packed_f32_fwd(EvoPacked p, Parts parts, int tiles, bool vec_out) {
    typedef F32Geo F;
    extern __shared__ __attribute__((aligned(16))) float mem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int heads = p.H / p.Hk, D = p.D;
    const Unit unit(blockIdx.x, tiles, p.Hk, heads * (PART ? parts.chunks : 1));
    if (unit.none) return;
    const int hk = unit.hk, h = hk * heads + unit.member % heads, part = PART ? unit.member / heads : 0;
    const Place at = place_of<false>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {   // (with parts: packed_f32_join's)
        if (PART) return;
        zero_values((float *)p.o, at.first, rows, p.H, h, D);
        if (p.lse && (int)threadIdx.x < rows) p.lse[(int64_t)h * p.Tq + at.first + threadIdx.x] = INFINITY;
        return;
    }
    const int all = (seen_most + F::STAGE - 1) / F::STAGE, from = PART ? part_begin(part, parts.chunks, all) : 0, to = PART ? part_begin(part + 1, parts.chunks, all) : all;
    const float *kbase = head_row<float>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = head_row<float>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    F32Share<> ks, vs;
    auto ask = [&](int st) {
        const int row = st * F::STAGE;
        ks.ask(kbase + row * p.k_stride_t, p.k_stride_t, s.nk() - row, D, VEC);
        vs.ask(vbase + row * p.v_stride_t, p.v_stride_t, s.nk() - row, D, VEC);
    };
    const int q0 = at.first + wave * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1, mine = q0 + li < s.q1;
    f32x4 q[F::KS];
    load_values(head_row<float>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), g, D, VEC, q);
    const int seen = s.seen(qrow, p.causal);
    const int wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    const float c = p.scale * kLog2e;
    float m = kMaskFloor, l = 0.0f;
    f32x16 o[F::DT];
#pragma unroll
    for (int dt = 0; dt < F::DT; ++dt) o[dt] = filled(0.0f);
    if (from < to) {
        ask(from);
        ks.put(mem);
        vs.put(mem + F::ARRAY);
    }
    __syncthreads();
    for (int st = from; st < to; ++st) {
        const float *const K = mem + ((st - from) & 1) * 2 * F::ARRAY, *const V = K + F::ARRAY;
        if (st + 1 < to) ask(st + 1);
        const int key0 = st * F::STAGE;
        if (key0 < wave_most) {   // (uniform)
            add_keys(o, m, l, K, V, q, key0, seen, c, li, g);
        }
        if (st + 1 < to) {
            float *const next = mem + ((st + 1 - from) & 1) * 2 * F::ARRAY;
            ks.put(next);
            vs.put(next + F::ARRAY);
        }
        __syncthreads();
    }
    if (!active) return;
    l += __shfl_xor(l, 32);
    if constexpr (PART) {
        const int64_t row = ((int64_t)part * p.Tq + qrow) * p.H + h;
        if (mine) store_values(parts.o + row * EVO_D, g, EVO_D, true, o, 1.0f);
        if (mine && g == 0) parts.ml[row] = make_float2(m, l);
        return;
    }
    const float inv = seen ? 1.0f / l : 0.0f;
#pragma unroll
    for (int dt = 0; dt < F::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = seen ? o[dt][r] * inv : 0.0f;
    unsigned again = rows_without_number(no_number(o) && mine && l == l);   // (see packed_fwd)
    const unsigned none = rows_without_number(mine && seen && l == 0.0f);
    if (p.lse && mine && g == 0) p.lse[(int64_t)h * p.Tq + qrow] = seen ? m + __log2f(l) : INFINITY;
    if (mine) store_values((float *)p.o + ((int64_t)qrow * p.H + h) * D, g, D, vec_out, o, 1.0f);
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int end = min(s.nk(), (wave_most + F::STAGE - 1) / F::STAGE * F::STAGE);
    if (!spoilt_forward<float>(late, s, hk, active ? s.seen(q0, late.causal) : 0, end)) again = none;
    wait_loads();
    for (; again; again &= again - 1) {
        const int b = __builtin_ctz(again), i = q0 + b;
        if ((none >> b & 1) || !all_finite<float>(late.v, late.v_stride_t, hk, late.v_stride_h, s.k0 + s.seen(i, late.causal), s.k0 + end, late.D)) row_forward<float>(late, s, i, h);
    }
}

// A sequence's few queries: one wave takes a part of its keys, and the queries of all heads that share a key head are the columns (32 after 32 of them).  A wave has the LDS and the registers of its
// own that a workgroup of packed_f32_fwd shares, and asks for the next keys and values before it computes; packed_f32_join makes the results, of rows of no sequence too.
template <bool VEC>
__global__ void __launch_bounds__(64, 1) packed_f32_few(EvoPacked p, Parts parts) {
    typedef F32Geo F;
    extern __shared__ __attribute__((aligned(16))) float mem[];
    const int lane = threadIdx.x, li = lane & 31, g = lane >> 5, heads = p.H / p.Hk, D = p.D;
    const int part = (int)(blockIdx.x % (unsigned)parts.chunks), unit = (int)(blockIdx.x / (unsigned)parts.chunks), hk = unit % p.Hk;
    const Segment s = segment(p, 1 + unit / p.Hk);
    const int64_t rows = s.nk() ? (int64_t)s.nq() * heads : 0;
    const int all = (s.nk() + F::STAGE - 1) / F::STAGE, from = part_begin(part, parts.chunks, all), to = part_begin(part + 1, parts.chunks, all);
    const float *kbase = head_row<float>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = head_row<float>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    const float c = p.scale * kLog2e;
    for (int64_t r0 = 0; r0 < rows; r0 += 32) {
        const int64_t pair = min(r0 + li, rows - 1);
        const int i = s.q0 + (int)(pair / heads), h = hk * heads + (int)(pair % heads), seen = s.seen(i, p.causal);
        const int most = s.seen(s.q0 + (int)(min(r0 + 31, rows - 1) / heads), p.causal), end = min(to, (most + F::STAGE - 1) / F::STAGE);
        f32x4 q[F::KS];
        load_values(head_row<float>(p.q, i, p.q_stride_t, h, p.q_stride_h), g, D, VEC, q);
        float m = kMaskFloor, l = 0.0f;
        f32x16 o[F::DT];
#pragma unroll
        for (int dt = 0; dt < F::DT; ++dt) o[dt] = filled(0.0f);
        F32Share<64> ks, vs;
        auto ask = [&](int st) {
            const int row = st * F::STAGE;
            ks.ask(kbase + row * p.k_stride_t, p.k_stride_t, s.nk() - row, D, VEC);
            vs.ask(vbase + row * p.v_stride_t, p.v_stride_t, s.nk() - row, D, VEC);
        };
        if (from < end) ask(from);
        for (int st = from; st < end; ++st) {
            __syncthreads();
            ks.put(mem);
            vs.put(mem + F::ARRAY);
            __syncthreads();
            if (st + 1 < end) ask(st + 1);
            add_keys(o, m, l, mem, mem + F::ARRAY, q, st * F::STAGE, seen, c, li, g);
        }
        l += __shfl_xor(l, 32);
        if (r0 + li < rows) {
            const int64_t row = ((int64_t)part * p.Tq + i) * p.H + h;
            store_values(parts.o + row * EVO_D, g, EVO_D, true, o, 1.0f);
            if (g == 0) parts.ml[row] = make_float2(m, l);
        }
    }
}

// The parts of a row joined, in their order, by a wave.
__global__ void __launch_bounds__(256) packed_f32_join(EvoPacked p, Parts parts, unsigned rows) {
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int i = (int)(row / (unsigned)p.H), h = (int)(row % (unsigned)p.H), lane = threadIdx.x & 63;
    const Segment s = segment_of_row<false>(p, i);
    const bool sees = !s.gap && s.seen(i, p.causal) > 0;
    const int n = sees ? parts.chunks : 0;
    float M = kMaskFloor, L = 0.0f;
    for (int x = lane; x < n; x += 64) M = fmaxf(M, parts.ml[(int64_t)x * rows + row].x);
    M = wave_max(M);
    Row o = {0.0f, 0.0f};
#pragma unroll 8
    for (int x = 0; x < n; ++x) {
        const int64_t at = (int64_t)x * rows + row;
        const float2 y = parts.ml[at];
        const float f = fast_exp2(y.x - M);
        L = fmaf(y.y, f, L);
        add_row(o, f, load_row(parts.o + at * EVO_D, EVO_D));
    }
    const float inv = sees ? 1.0f / L : 0.0f;
    o.a *= inv;
    o.b *= inv;
    if (__any(!(o.a == o.a) || !(o.b == o.b)) && L == L) {
        const EvoPacked late = parameters_again();
        const int seen = s.seen(i, late.causal);
        if (L == 0.0f || spoilt_forward<float>(late, s, h / (late.H / late.Hk), seen, min(s.nk(), seen + 62))) {   // (what other rows of a wave see, and the end of a stage)
            row_forward<float, 4>(late, s, i, h);
            return;
        }
    }
    store_row((float *)p.o + ((int64_t)i * p.H + h) * p.D, o, p.D);
    if (p.lse && lane == 0) p.lse[(int64_t)h * p.Tq + i] = sees ? M + __log2f(L) : INFINITY;
}

// PART: a part of the walk, all of which packed_f32_sum adds up (dK's and dV's kernel likewise).
template <bool VEC, bool PART>
__global__ void __launch_bounds__(256, EVO_D <= 64 ? 2 : 1) packed_f32_dq(EvoPacked p, BackwardRows saved, Parts parts, int tiles, bool vec_out) {
    typedef F32Geo F;
    extern __shared__ __attribute__((aligned(16))) float mem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int heads = p.H / p.Hk, D = p.D;
    const Unit unit(blockIdx.x, tiles, p.Hk, heads * (PART ? parts.chunks : 1));
    if (unit.none) return;
    const int hk = unit.hk, h = hk * heads + unit.member % heads, part = PART ? unit.member / heads : 0;
    const Place at = place_of<false>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.q1) return;
    const int rows = min(kPackedRows, s.q1 - at.first);
    const int seen_most = s.gap ? 0 : s.seen(at.first + rows - 1, p.causal);
    if (seen_most == 0) {   // (no key is seen by its rows: nothing reads their delta)
        if (PART) return;
        zero_values((float *)p.dq, at.first, rows, p.H, h, D);
        return;
    }
    const int all = (seen_most + F::STAGE - 1) / F::STAGE, from = PART ? part_begin(part, parts.chunks, all) : 0, to = PART ? part_begin(part + 1, parts.chunks, all) : all;
    const float *kbase = head_row<float>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = head_row<float>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    F32Share<> ks, vs;
    auto ask = [&](int st) {
        const int row = st * F::STAGE;
        ks.ask(kbase + row * p.k_stride_t, p.k_stride_t, s.nk() - row, D, VEC);
        vs.ask(vbase + row * p.v_stride_t, p.v_stride_t, s.nk() - row, D, VEC);
    };
    const int q0 = at.first + wave * 32, qrow = min(q0 + li, s.q1 - 1);
    const bool active = q0 < s.q1, mine = q0 + li < s.q1;
    f32x4 q[F::KS], dout[F::KS];
    load_values(head_row<float>(p.q, qrow, p.q_stride_t, h, p.q_stride_h), g, D, VEC, q);
    load_values(head_row<float>(p.dout, qrow, p.dout_stride_t, h, p.dout_stride_h), g, D, VEC, dout);
    float delta = 0.0f;
    {
        const float *o = (const float *)p.o + ((int64_t)qrow * p.H + h) * D;
#pragma unroll
        for (int x = 0; x < F::KS; ++x) {
            const f32x4 y = four(o, 8 * x + 4 * g, D, vec_out);
#pragma unroll
            for (int i = 0; i < 4; ++i) delta = fmaf(dout[x][i], y[i], delta);
        }
    }
    delta += __shfl_xor(delta, 32);
    const float c = p.scale * kLog2e, lse = p.lse[(int64_t)h * p.Tq + qrow];
    if (mine && g == 0 && part == 0) saved.delta[(int64_t)h * p.Tq + qrow] = -delta;
    const int seen = s.seen(qrow, p.causal);
    const int wave_least = active ? s.seen(q0, p.causal) : 0, wave_most = active ? s.seen(min(q0 + 31, s.q1 - 1), p.causal) : 0;
    f32x16 dq[F::DT];
#pragma unroll
    for (int dt = 0; dt < F::DT; ++dt) dq[dt] = filled(0.0f);
    if (from < to) {
        ask(from);
        ks.put(mem);
        vs.put(mem + F::ARRAY);
    }
    __syncthreads();
    for (int st = from; st < to; ++st) {
        const float *const K = mem + ((st - from) & 1) * 2 * F::ARRAY, *const V = K + F::ARRAY;
        if (st + 1 < to) ask(st + 1);
        const int key0 = st * F::STAGE;
        if (key0 < wave_most) {   // (uniform)
            f32x16 a = times(K, q, li, g);
            const f32x16 d = times(V, dout, li, g);
#pragma unroll
            for (int r = 0; r < 16; ++r) a[r] = fast_exp2(fmaf(a[r], c, -lse)) * (d[r] - delta);
            if (key0 + F::STAGE > wave_least) {
#pragma unroll
                for (int r = 0; r < 16; ++r) a[r] = key0 + crow(r, g) < seen ? a[r] : 0.0f;
            }
            add_weighted(dq, K, a, li, g);
        }
        if (st + 1 < to) {
            float *const next = mem + ((st + 1 - from) & 1) * 2 * F::ARRAY;
            ks.put(next);
            vs.put(next + F::ARRAY);
        }
        __syncthreads();
    }
    if (!active) return;
    if constexpr (PART) {
        if (mine) store_values(parts.o + (((int64_t)part * p.Tq + qrow) * p.H + h) * EVO_D, g, EVO_D, true, dq, 1.0f);
        return;
    }
    unsigned again = rows_without_number(no_number(dq) && mine && lse == lse && delta == delta);   // (of a NaN among them every dS is one)
    if (mine) store_values((float *)p.dq + ((int64_t)qrow * p.H + h) * D, g, D, vec_out, dq, p.scale);
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int end = min(s.nk(), (wave_most + F::STAGE - 1) / F::STAGE * F::STAGE);
    if (!spoilt_dq<float>(late, s, hk, wave_least, end)) return;
    wait_loads();
    for (; again; again &= again - 1) {
        const int b = __builtin_ctz(again), i = q0 + b;
        if (spoilt_dq<float>(late, s, hk, s.seen(i, late.causal), end)) row_dq<float>(late, s, i, h, lane_value(delta, b));
    }
}

template <bool VEC, bool PART>
__global__ void __launch_bounds__(256, EVO_D <= 64 ? 2 : 1) packed_f32_dkdv(EvoPacked p, BackwardRows saved, Parts parts, int tiles, bool vec_out) {
    typedef F32Geo F;
    extern __shared__ __attribute__((aligned(16))) float mem[];   // two stages: Q, dO, lse, -delta
    constexpr int STAGE = 2 * (F::ARRAY + F::STAGE);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int heads = p.H / p.Hk, D = p.D;
    const Unit unit(blockIdx.x, tiles, p.Hk, PART ? parts.chunks : 1);
    if (unit.none) return;
    const int hk = unit.hk;
    const Place at = place_of<true>(p, unit.tile, tiles);
    const Segment &s = at.s;
    if (at.first >= s.k1) return;
    const int rows = min(kPackedRows, s.k1 - at.first);
    const int begin = s.first_query(at.first, p.causal);   // that sees any of the workgroup's keys
    if (s.gap || begin >= s.q1) {
        if (PART) return;
        zero_values((float *)p.dk, at.first, rows, p.Hk, hk, D);
        zero_values((float *)p.dv, at.first, rows, p.Hk, hk, D);
        return;
    }
    F32Share<> qs, ds;
    float number = 0.0f;   // of a row of the stage: lse (the first 32 threads), -delta (the next)
    auto ask = [&](int h, int stage) {
        const int row = begin + stage * F::STAGE, n = s.q1 - row, r = threadIdx.x & 31;
        qs.ask(head_row<float>(p.q, row, p.q_stride_t, h, p.q_stride_h), p.q_stride_t, n, D, VEC);
        ds.ask(head_row<float>(p.dout, row, p.dout_stride_t, h, p.dout_stride_h), p.dout_stride_t, n, D, VEC);
        if (threadIdx.x < 64) {
            const float *x = (threadIdx.x < 32 ? p.lse : saved.delta) + (int64_t)h * p.Tq + row;
            number = r < n ? x[r] : threadIdx.x < 32 ? INFINITY : 0.0f;   // (past the end: probabilities of zero)
        }
    };
    auto put = [&](float *to) {
        qs.put(to);
        ds.put(to + F::ARRAY);
        if (threadIdx.x < 64) to[2 * F::ARRAY + threadIdx.x] = number;
    };
    const int k0 = at.first + wave * 32, krow = min(k0 + li, s.k1 - 1);
    const bool active = k0 < s.k1, mine = k0 + li < s.k1;
    f32x4 k[F::KS], v[F::KS];
    load_values(head_row<float>(p.k, krow, p.k_stride_t, hk, p.k_stride_h), g, D, VEC, k);
    load_values(head_row<float>(p.v, krow, p.v_stride_t, hk, p.v_stride_h), g, D, VEC, v);
    // the first query that sees this lane's key, the wave's first one and its last one
    const int key_from = s.first_query(krow, p.causal), wave_from = s.first_query(k0, p.causal), wave_to = s.first_query(min(k0 + 31, s.k1 - 1), p.causal);
    const float c = p.scale * kLog2e;
    f32x16 dk[F::DT], dv[F::DT];
#pragma unroll
    for (int dt = 0; dt < F::DT; ++dt) dk[dt] = dv[dt] = filled(0.0f);
    const int stages = (s.q1 - begin + F::STAGE - 1) / F::STAGE;
    const int total = stages * heads, from = PART ? part_begin(unit.member, parts.chunks, total) : 0, to = PART ? part_begin(unit.member + 1, parts.chunks, total) : total;
    int stage = from % stages, h = hk * heads + from / stages, half = 0;
    if (from < to) {
        ask(h, stage);
        put(mem);
    }
    __syncthreads();
    for (int it = from; it < to; ++it) {
        const float *const Q = mem + half * STAGE, *const dO = Q + F::ARRAY, *const numbers = Q + 2 * F::ARRAY;
        const int row0 = begin + stage * F::STAGE;
        if (++stage == stages) {
            stage = 0;
            ++h;
        }
        half ^= 1;
        if (it + 1 < to) ask(h, stage);
        if (active && row0 + F::STAGE > wave_from) {   // (uniform)
            f32x16 a = times(Q, k, li, g), d = times(dO, v, li, g);
#pragma unroll
            for (int rr = 0; rr < 4; ++rr) {
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(numbers + 8 * rr + 4 * g), minus = *reinterpret_cast<const f32x4 *>(numbers + 32 + 8 * rr + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[4 * rr + i] = fast_exp2(fmaf(a[4 * rr + i], c, -lse[i]));
                    d[4 * rr + i] += minus[i];
                }
            }
            if (row0 < wave_to) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool sees = row0 + crow(r, g) >= key_from;
                    a[r] = sees ? a[r] : 0.0f;
                    d[r] = sees ? d[r] : 0.0f;
                }
            }
            add_weighted(dv, dO, a, li, g);
#pragma unroll
            for (int r = 0; r < 16; ++r) d[r] *= a[r];
            add_weighted(dk, Q, d, li, g);
        }
        if (it + 1 < to) put(mem + half * STAGE);
        __syncthreads();
    }
    if (!active) return;
    if constexpr (PART) {
        const int64_t all = p.Tk * p.Hk, row = unit.member * all + (int64_t)krow * p.Hk + hk;
        if (mine) {
            store_values(parts.o + row * EVO_D, g, EVO_D, true, dk, 1.0f);
            store_values(parts.o + (row + parts.chunks * all) * EVO_D, g, EVO_D, true, dv, 1.0f);
        }
        return;
    }
    unsigned again = rows_without_number((no_number(dk) || no_number(dv)) && mine);
    if (mine) {
        const int64_t row = ((int64_t)krow * p.Hk + hk) * D;
        store_values((float *)p.dk + row, g, D, vec_out, dk, p.scale);
        store_values((float *)p.dv + row, g, D, vec_out, dv, 1.0f);
    }
    if (!again) return;
    const EvoPacked late = parameters_again();
    const int least = max(begin, wave_from - 31);
    if (!spoilt_dkdv<float>(late, s, hk, k0, min(k0 + 32, s.k1), least, wave_to, saved.delta)) return;
    wait_loads();
    for (; again; again &= again - 1) {
        const int j = k0 + __builtin_ctz(again);
        if (spoilt_dkdv<float>(late, s, hk, j, j + 1, least, s.first_query(j, late.causal), saved.delta)) row_dkdv<float>(late, s, j, hk, saved.delta);
    }
}

// The parts of a row of dQ (KEYS: dK and dV) added up, in their order, by a wave.
template <bool KEYS>
__global__ void __launch_bounds__(256) packed_f32_sum(EvoPacked p, BackwardRows saved, Parts parts, unsigned rows) {
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int heads = KEYS ? p.Hk : p.H, i = (int)(row / (unsigned)heads), h = (int)(row % (unsigned)heads);
    const Segment s = segment_of_row<KEYS>(p, i);
    const int n = s.gap || (KEYS ? s.first_query(i, p.causal) >= s.q1 : s.seen(i, p.causal) == 0) ? 0 : parts.chunks;
    Row sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    bool nan = false;
#pragma unroll
    for (int y = 0; y < (KEYS ? 2 : 1); ++y) {
        for (int x = 0; x < n; ++x) add_row(sum[y], 1.0f, load_row(parts.o + ((int64_t)(x + y * parts.chunks) * rows + row) * EVO_D, EVO_D));
        nan |= !(sum[y].a == sum[y].a) || !(sum[y].b == sum[y].b);
        store_row((float *)(y ? p.dv : KEYS ? p.dk : p.dq) + (int64_t)row * p.D, y ? sum[y] : Row{sum[y].a * p.scale, sum[y].b * p.scale}, p.D);
    }
    if (!__any(nan)) return;
    const EvoPacked late = parameters_again();
    // (what other rows of a wave see, and the end of a stage)
    if constexpr (KEYS) {
        const int from = s.first_query(i, late.causal);
        if (!spoilt_dkdv<float>(late, s, h, i, i + 1, max(s.q0, from - 62), from, saved.delta)) return;
        wait_loads();   // (for what has been stored, too: it is overwritten)
        row_dkdv<float, 4>(late, s, i, h, saved.delta);
    } else {
        const int64_t at = (int64_t)h * late.Tq + i;
        const int seen = s.seen(i, late.causal);
        if (!(late.lse[at] == late.lse[at]) || !(saved.delta[at] == saved.delta[at]) || !spoilt_dq<float>(late, s, h / (late.H / late.Hk), seen, min(s.nk(), seen + 62))) return;
        wait_loads();
        row_dq<float, 4>(late, s, i, h, -saved.delta[at]);
    }
}

// Parts of the keys of few queries: as many as make 16 waves to a CU, which has room for four at once (sequences differ in length), of two stages of an average sequence at least.
static Plan few_f32_plan(const EvoPacked &p) {
    const int64_t units = (int64_t)p.n * p.Hk, room = 4096 / units, worth = p.Tk / p.n / (2 * F32Geo::STAGE), n = room < worth ? room : worth;
    return {1, (int)(n < 1 ? 1 : n > 512 ? 512 : n)};
}
// Parts of a walk of `steps` stages for `units` workgroups without them.
static Plan f32_plan(int64_t units, int64_t steps) {
    const int64_t room = 2048 / (units ? units : 1), worth = steps / 4, n = room < worth ? room : worth;
    return {1, (int)(n < 1 ? 1 : n > 64 ? 64 : n)};
}
static Plan f32_queries(const EvoPacked &p) { return f32_plan((p.Tq / kPackedRows + (p.n + 1) / 2) * p.H, p.Tk / (p.n ? p.n : 1) / F32Geo::STAGE); }
static Plan f32_keys(const EvoPacked &p) { return f32_plan((p.Tk / kPackedRows + (p.n + 1) / 2) * p.Hk, p.Tq / (p.n ? p.n : 1) * (p.H / p.Hk) / F32Geo::STAGE); }

template <typename F>
static int by_flag(bool flag, F &&f) {
    return flag ? f(std::true_type()) : f(std::false_type());
}
// Whether inputs, and results, can be moved 16 bytes at a time
static bool vectors(const EvoPacked &p, bool backward) {
    bool yes = p.D % 4 == 0;
    for (const void *x : {p.q, p.k, p.v, backward ? p.dout : nullptr}) yes = yes && (uintptr_t)x % 16 == 0;
    for (int64_t x : {p.q_stride_t, p.k_stride_t, p.v_stride_t, backward ? p.dout_stride_t : 0, p.q_stride_h, p.k_stride_h, p.v_stride_h, backward ? p.dout_stride_h : 0}) yes = yes && x % 4 == 0;
    return yes;
}
static bool vector_results(const EvoPacked &p) {
    bool yes = p.D % 4 == 0;
    for (const void *x : {(const void *)p.o, (const void *)p.dq, (const void *)p.dk, (const void *)p.dv}) yes = yes && (uintptr_t)x % 16 == 0;
    return yes;
}

}  // namespace

size_t EVO_CAT(packed_f32_fwd_bytes_d, EVO_D)(const EvoPacked &p) { return EVO_CAT(packed_d, EVO_D)::f32_queries(p).bytes(p.Tq * p.H, EVO_D + 2); }
size_t EVO_CAT(packed_f32_bwd_bytes_d, EVO_D)(const EvoPacked &p) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const size_t dq = f32_queries(p).bytes(p.Tq * p.H, EVO_D), dkdv = f32_keys(p).bytes(p.Tk * p.Hk, 2 * EVO_D);
    return dq > dkdv ? dq : dkdv;
}
// (the join makes the results with one part too)
size_t EVO_CAT(packed_f32_few_bytes_d, EVO_D)(const EvoPacked &p) { return (size_t)(EVO_CAT(packed_d, EVO_D)::few_f32_plan(p).parts * p.Tq * p.H * (EVO_D + 2) * (int64_t)sizeof(float)); }
int EVO_CAT(launch_packed_f32_few_d, EVO_D)(const EvoPacked &p, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const int parts = few_f32_plan(p).parts;
    const int64_t grid = (int64_t)p.n * p.Hk * parts, rows = p.Tq * p.H;
    if (!grid_fits(grid, 64) || !row_waves_fit(rows)) return EVO_EOVERFLOW;
    const Parts to = {(float *)p.workspace, (float2 *)((float *)p.workspace + parts * rows * EVO_D), 0, parts};
    const int rc = by_flag(vectors(p, false), [&](auto vec) {
        constexpr auto kern = packed_f32_few<decltype(vec)::value>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kern, F32Geo::LDS / 2, done, nullptr)) return rc;
        kern<<<(unsigned)grid, 64, F32Geo::LDS / 2, st>>>(p, to);
        return hip_rc();
    });
    if (rc) return rc;
    packed_f32_join<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, to, (unsigned)rows);
    return hip_rc();
}
int EVO_CAT(launch_packed_f32_fwd_d, EVO_D)(const EvoPacked &p, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const int parts = f32_queries(p).parts;
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = Unit::grid(tiles, p.Hk, p.H / p.Hk * (int64_t)parts), rows = p.Tq * p.H;
    if (!grid_fits(grid, 256) || (parts > 1 && !row_waves_fit(rows))) return EVO_EOVERFLOW;
    auto go = [&](auto vec, auto part) {
        constexpr auto kern = packed_f32_fwd<decltype(vec)::value, decltype(part)::value>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kern, F32Geo::LDS, done, nullptr)) return rc;
        const Parts to = {(float *)p.workspace, (float2 *)((float *)p.workspace + parts * rows * EVO_D), 0, parts};
        kern<<<(unsigned)grid, 256, F32Geo::LDS, st>>>(p, to, (int)tiles, vector_results(p));
        if (const int rc = hip_rc()) return rc;
        if (!decltype(part)::value) return (int)EVO_OK;
        packed_f32_join<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, to, (unsigned)rows);
        return hip_rc();
    };
    return by_flag(vectors(p, false), [&](auto vec) { return by_flag(parts > 1, [&](auto part) { return go(vec, part); }); });
}
int EVO_CAT(launch_packed_f32_bwd_d, EVO_D)(const EvoPacked &p, const BackwardRows &saved, float *sums, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const bool vec_out = vector_results(p);
    const Parts qparts = {sums, nullptr, 0, f32_queries(p).parts}, kparts = {sums, nullptr, 0, f32_keys(p).parts};
    const int64_t tiles = packed_tiles(p.Tq, p.n), grid = Unit::grid(tiles, p.Hk, p.H / p.Hk * (int64_t)qparts.chunks), rows = p.Tq * p.H;
    const int64_t key_tiles = packed_tiles(p.Tk, p.n), key_grid = Unit::grid(key_tiles, p.Hk, kparts.chunks), keys = p.Tk * p.Hk;
    if (!grid_fits(grid, 256) || !grid_fits(key_grid, 256) || (qparts.chunks > 1 && !row_waves_fit(rows)) || (kparts.chunks > 1 && !row_waves_fit(keys))) return EVO_EOVERFLOW;
    auto dq = [&](auto vec, auto part) {
        constexpr auto kern = packed_f32_dq<decltype(vec)::value, decltype(part)::value>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kern, F32Geo::LDS, done, nullptr)) return rc;
        kern<<<(unsigned)grid, 256, F32Geo::LDS, st>>>(p, saved, qparts, (int)tiles, vec_out);
        if (const int rc = hip_rc()) return rc;
        if (!decltype(part)::value) return (int)EVO_OK;
        packed_f32_sum<false><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, saved, qparts, (unsigned)rows);
        return hip_rc();
    };
    auto dkdv = [&](auto vec, auto part) {
        constexpr auto kern = packed_f32_dkdv<decltype(vec)::value, decltype(part)::value>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kern, F32Geo::LDS, done, nullptr)) return rc;
        kern<<<(unsigned)key_grid, 256, F32Geo::LDS, st>>>(p, saved, kparts, (int)key_tiles, vec_out);
        if (const int rc = hip_rc()) return rc;
        if (!decltype(part)::value) return (int)EVO_OK;
        packed_f32_sum<true><<<(unsigned)((keys + 3) / 4), 256, 0, st>>>(p, saved, kparts, (unsigned)keys);
        return hip_rc();
    };
    return by_flag(vectors(p, true), [&](auto vec) {
        if (p.Tq) {
            if (const int rc = by_flag(qparts.chunks > 1, [&](auto part) { return dq(vec, part); })) return rc;
        }
        return p.Tk && p.dk ? by_flag(kparts.chunks > 1, [&](auto part) { return dkdv(vec, part); }) : (int)EVO_OK;
    });
}

}  // namespace evo
