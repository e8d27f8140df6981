// Packed attention in 16 bits: what its matrix kernels share.  Compiled once per head dim (-DEVO_D=32|64|96|128).
#pragma once

#include "packed_common.h"
#include "stream_common.h"

#ifndef EVO_D
#error "compile with -DEVO_D=<head dim>"
#endif

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {   // (one name for each head dim's kernels)

constexpr int kPackedRows = 128;      // of a workgroup of the forward and of dQ
constexpr int kFarOff = 0x7fffff00;   // an offset past the end of every array

struct PackedGeo {
    static constexpr int GD = EVO_D == 96 ? 128 : EVO_D;   // rows in LDS (96: three quarters of them used)
    typedef StreamGeo<GD> G;
    static constexpr int KSD = EVO_D / 16, DT = EVO_D / 32;
    static constexpr int STAGE = 64;   // keys of a stage
    static constexpr int ARRAY = STAGE * G::ROW;
};

// Rows at `base`, `rows` of them, stride_t bytes apart, as a resource whose end is the end of the last: what is asked for beyond reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void *base, int rows, int stride, int D) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, rows > 0 ? (rows - 1) * stride + D * 2 : 0, 0x00020000);
}

// This lane's offset of its first piece of a stage of rows; its further pieces are STEP rows on each.
template <int NW>
struct StagePieces {
    typedef PackedGeo::G G;
    static constexpr int RPP = 1024 / G::ROW;        // rows to a piece of 1 KB
    static constexpr int STEP = RPP * NW;            // rows from one of a wave's pieces to its next
    static_assert(STEP % 16 == 0, "a lane's chunk is the same in all of its pieces");
    static constexpr int each(int rows) { return rows / RPP / NW; }   // pieces of a wave (where they are shared out evenly)
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

// Where this lane reads staged rows: as offsets in LDS, to which a multiple of 256 is added and of which a few bits are then turned over (StreamGeo stores chunk c of row r at c ^ x(r), and
// what depends on the step, the tile or the half of it is in bits of their own), so that one addition and an exclusive or with a constant, not an address in a register of its own for each read, lead there.
struct Staged {
    typedef PackedGeo::G G;
    unsigned row, col;   // of operands along rows, and of transposed ones
    __device__ __forceinline__ explicit Staged(int lane) {
        const int li = lane & 31, g = lane >> 5, r = 4 * g + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        row = (unsigned)G::at(li, g);
        col = (unsigned)(G::at(r, c) + (lane & 1) * 8);
    }
    static __device__ __forceinline__ unsigned base(const unsigned char *x) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)x; }
    // row kb + li of the array at `at`, columns 16 ks + 8 g .. + 7 (`at` and `kb` multiples of 256 bytes and 32 rows)
    template <typename T>
    __device__ __forceinline__ typename Mfma<T>::v8 rows(unsigned at, int kb, int ks) const {
        return *(const __attribute__((address_space(3))) typename Mfma<T>::v8 *)(uintptr_t)(((at + row) ^ (unsigned)(ks << 5)) + (unsigned)(kb * G::ROW));
    }
    // `transposed` (stream_common.h) of the array at `at`
    template <typename T>
    __device__ __forceinline__ typename Mfma<T>::v8 cols(unsigned at, int kb, int ts, int dt) const {
        typename Mfma<T>::v8 r;
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
            const unsigned a = ((at + col) ^ (unsigned)(dt << 6 | h2 << (PackedGeo::GD == 32 ? 5 : 4))) + (unsigned)((kb + 16 * ts + 8 * h2) * G::ROW);
            const typename Mfma<T>::v4 v = __builtin_bit_cast(typename Mfma<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4s __attribute__((address_space(3))) *)(uintptr_t)a));
#pragma unroll
            for (int i = 0; i < 4; ++i) r[4 * h2 + i] = v[i];
        }
        return r;
    }
};

// A row's values as operands: step ks holds columns 16 ks + 8 g .. + 7; zeros from D on.
template <typename T>
__device__ __forceinline__ void load_operands(const T *row, int D, int g, typename Mfma<T>::v8 (&x)[PackedGeo::KSD]) {
#pragma unroll
    for (int ks = 0; ks < PackedGeo::KSD; ++ks) x[ks] = ks * 16 + g * 8 < D ? ld8(row + ks * 16 + g * 8) : zero8<T>();
}

// Where a workgroup is: a tile of a segment.
struct Place {
    Segment s;
    int first;   // its first row (of the tensor), or, where there is nothing to do, s's end or beyond
};
// The tile that is the `rank`th of `tiles` to begin.  KEYS: of keys, else of queries.
template <bool KEYS>
__device__ __forceinline__ Place place_of(const EvoPacked &p, int rank, int tiles) {
    Place r;
    int j;
    // Of few sequences the tiles with the longest walks begin first.  Under a causal mask a tile of queries i before a sequence's own first one sees i + 1 tiles of keys, one of keys is seen from as many
    // tiles as are behind it and its own: of c_j tiles of sequence j max(0, c_j - w) have walks longer than w, and the rank is that of walks of w where the sum of these reaches it.  Without a mask all of a
    // sequence's tiles have the same walk.  4 x 4096 causal rows, 32 heads (8) of 128: dK and dV 1.19 ms (1.34 with one sequence after the other), forward 0.635 (0.66), dQ 1.08 (1.06: more sequences' keys
    // at once in an L2).  Seven causal sequences of 5 tiles on average: forward 34.0 us (35.1); 16 of 3: with gradients 88 (99); 40 of one: 9 (7), the search takes longer than it
    // gains.  24 chains of 51 to 768 rows without a mask, 8 heads of 32: forward 16.1 us (19.2), dQ 24.7 (31.1), of 64: 17 (22); 60 of 100 to 1000 with 32 heads: 218 (177), hence not for so many.  Where it turns, by sequences of
    // 100 to 1400 rows, with gradients, causal: 8 heads of 32: 16 87 us (109), 29 103 (116), 45 141 (149), 60 188 (174); 32 heads (8) of 64: 8 178 (209), 29 409 (434), 36 508 (513), 45 629 (622); 16 heads of 128: 16 238 (264),
    // 24 354 (357), 29 430 (425), 36 532 (513).  Without a mask the same within 3 in a hundred.
    if (p.n < 30 && (KEYS ? p.Tk : p.Tq) >= (int64_t)2 * kPackedRows * p.n) {
        const int lane = threadIdx.x & 63, x = min(lane, p.n + 2), q = queries_begin(p, x), k = keys_begin(p, x);
        const int nq = max(0, __shfl_down(q, 1) - q), nk = max(0, __shfl_down(k, 1) - k), own = lane < p.n + 2 ? ((KEYS ? nk : nq) + kPackedRows - 1) / kPackedRows : 0;
        int into = 0;         // the tile's place in its sequence, as far as lane j knows
        bool chosen = false;
        if (p.causal) {
            auto longer = [&](int w) {
                int sum = 0;
                for (int y = 0; y < p.n + 2; ++y) sum += max(0, __builtin_amdgcn_readlane(own, y) - w);
                return sum;
            };
            int lo = -1, hi = tiles, at = 0;   // longer(hi) <= rank, and not of lo
            while (hi - lo > 1) {
                const int step = (hi - lo + 63) / 64, w = min(hi, lo + (lane + 1) * step), n = longer(w);
                const int f = __builtin_ctzll(__ballot(n <= rank));   // (the last lane's w is hi)
                hi = __builtin_amdgcn_readlane(w, f);
                at = __builtin_amdgcn_readlane(n, f);
                lo = hi - step;
            }
            const uint64_t those = __ballot(own >= hi && own > 0);
            chosen = hi > 0 && (those >> lane & 1) && __popcll(those & ((1ull << lane) - 1)) == rank - at;
            into = KEYS ? own - hi : hi - 1;
        } else {
            const int walk = lane == 0 || lane > p.n ? -1 : KEYS ? nq : nk;   // (rows of no sequence: last)
            int before = 0;
            for (int y = 0; y < p.n + 2; ++y) {
                const int other = __builtin_amdgcn_readlane(walk, y);
                before += other > walk || (other == walk && y < lane) ? __builtin_amdgcn_readlane(own, y) : 0;
            }
            into = rank - before;
            chosen = into >= 0 && into < own;
        }
        const uint64_t found = __ballot(chosen);
        if (!found) {   // (past the last)
            r.s = Segment{0, 0, 0, 0, true};
            r.first = INT32_MAX;
            return r;
        }
        j = __builtin_ctzll(found);
        r.s = segment_of_lanes(p, q, k, j);
        r.first = (KEYS ? r.s.k0 : r.s.q0) + __builtin_amdgcn_readlane(into, j) * kPackedRows;
        return r;
    }
    const int t = KEYS ? rank : tiles - 1 - rank;
    r.s = find_segment<KEYS>(p, [&](int begin, int x) { return begin / kPackedRows + x <= t; }, j);
    const int b = KEYS ? r.s.k0 : r.s.q0, i = t - (b / kPackedRows + j);
    r.first = i < 0 ? INT32_MAX : (int)min((int64_t)INT32_MAX, b + (int64_t)i * kPackedRows);   // (below zero: offsets that do not ascend)
    return r;
}

template <typename T>
__device__ __forceinline__ void zero_rows(T *x, int first, int rows, int heads, int h, int D) {
    const int per = D / 8, n = rows * per;
    for (int i = threadIdx.x; i < n; i += blockDim.x) *reinterpret_cast<uint4 *>(x + ((int64_t)(first + i / per) * heads + h) * D + i % per * 8) = make_uint4(0, 0, 0, 0);
}

// The lanes (low 32 bits: the rows of the wave) whose accumulators hold something that is no number
__device__ __forceinline__ unsigned rows_without_number(bool nan) {
    const uint64_t b = __ballot(nan);
    return (unsigned)b | (unsigned)(b >> 32);
}

// What rounding leaves
template <typename T>
__device__ __forceinline__ float left(float v) { return v - (float)(T)v; }

// fp16 in the backward.  Below 2^-14 it has fewer bits, below 2^-25 none, and above 65504 it is infinite, while dS = P (dP - delta) has gradients of any size in it and P as small a number as there are keys.  So a lane
// forms dS and its sums times a power of two, which comes down, as the running maximum of a softmax goes up, where dS would pass kShiftTop, and is taken out of the sums at the end.  For dQ, whose P stays in fp32, P has it, and
// it begins at 2^kShiftQuery: an incoming gradient's smallest step, 2^-24, spread over 2^17 keys is a dS of 2^-1 then.  For dV P is an operand, times 2^kShiftKey always (a score of up to 2^24, which fp32 leaves off by
// 2, still has no infinite one; of 2^27 keys alike each has bits), and dS's power is one beside it, 2^17 at first.  Errors of dQ, dK and dV next to the exact result rounded, 4096 rows of D = 64 without a mask, incoming gradients of
// 1e-4: 8.0, 8.0 and 1.0 times without it, 1.0 for all three with it (tests/test_gpu_packed_gradients.py).  What it costs is looking for the largest of 16 values in each tile: 4 x 4096 causal rows, 32 heads (8) of 128,
// forward and backward 2.84 ms instead of 2.74; twelve of 200 to 1500, 16 heads (4) of 64, 194 us instead of 184.  bf16 has fp32's exponents.
template <typename T> constexpr bool kShifts = std::is_same<T, f16_t>::value;
constexpr int kShiftQuery = 40, kShiftKey = 13;
constexpr float kShiftTop = 32768.0f;
// How far (a power of two) this lane's column has to come down for `d`, both of its halves, to be below 2^10; 0 where it is not above kShiftTop.  (An infinity is not: it stays one.)
__device__ __forceinline__ int shift_down(const f32x16 &d, bool &any) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(d[r]));
    any = __any(top > kShiftTop);
    if (__builtin_expect(!any, 1)) return 0;
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    const float most = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
    return most > kShiftTop && most < INFINITY ? __builtin_amdgcn_frexp_expf(most) - 10 : 0;
}
template <int N>
__device__ __forceinline__ void shift_by(f32x16 (&x)[N], float by) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] *= by;
}

__device__ __forceinline__ f32x16 filled(float v) {
    f32x16 x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = v;
    return x;
}

// Which tile and heads a workgroup takes.  Workgroups go round the eight XCDs, each with an L2 of its own; a unit, a tile and a key head, goes to one of them with all of its query heads, and units follow
// each other by tiles first: with a multiple of eight key heads an XCD keeps to its own, with fewer the tiles of one are dealt out one by one, so that all XCDs have long and short ones.  (Seven prompts of 90 to 2011, 16 / 4 heads of 64:
// 36.6 us; in runs of units, a half of a key head's tiles to an XCD, 39.7.)
struct Unit {
    int tile, hk, member;   // member: of the unit's workgroups
    bool none;              // past the last unit
    __device__ __forceinline__ Unit(unsigned id, int tiles, int heads, int members) {
        const unsigned slot = id / 8, u = slot / (unsigned)members * 8 + id % 8;
        member = (int)(slot % (unsigned)members);
        tile = (int)(u / (unsigned)heads);
        hk = (int)(u % (unsigned)heads);
        none = tile >= tiles;
    }
    static int64_t grid(int64_t tiles, int64_t heads, int64_t members) { return (tiles * heads + 7) / 8 * 8 * members; }
};

// Results in parts: [part][row][head] rows of D fp32 (of a softmax: relative to 2^m) and, of a softmax, (m, l).
struct Parts {
    float *o;
    float2 *ml;
    int chunk;   // keys of a part (packed_few), or 0: each row has `chunks` of them
    int chunks;  // the most of a row
};
// What part `x` of `parts` takes of n steps
__device__ __forceinline__ int part_begin(int x, int parts, int n) { return (int)((int64_t)n * x / parts); }

// The accumulators of two waves that have the same rows, through LDS, a register of all lanes after the other: given by one, added by the other
template <int N>
__device__ __forceinline__ void give(const f32x16 (&x)[N], float *to, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(i * 16 + r) * 64 + lane] = x[i][r];
}
template <int N>
__device__ __forceinline__ void take(f32x16 (&x)[N], const float *from, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] += from[(i * 16 + r) * 64 + lane];
}
// A tile's row as fp32 (store_row_tile's, unrounded): columns 8 (r / 4) + 4 g + r % 4
__device__ __forceinline__ void store_row_part(float *row, int c0, int ncols, const f32x16 &x, int g) {
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
        const int c = c0 + 8 * rr + 4 * g;
        if (c < ncols) *reinterpret_cast<f32x4 *>(row + c) = f32x4{x[4 * rr], x[4 * rr + 1], x[4 * rr + 2], x[4 * rr + 3]};
    }
}
__device__ __forceinline__ void zero_parts(float *x, int first, int rows, int heads, int h, int D) {
    const int per = D / 4, n = rows * per;
    for (int i = threadIdx.x; i < n; i += blockDim.x) *reinterpret_cast<f32x4 *>(x + ((int64_t)(first + i / per) * heads + h) * D + i % per * 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

static int64_t packed_tiles(int64_t rows, int n) { return rows / kPackedRows + n + 2; }

// The sums of a row's parts, by a wave for each row: dQ, or (KEYS) dK and dV, whose parts follow those of dK.
template <typename T, bool KEYS>
__global__ void __launch_bounds__(256) packed_sum(EvoPacked p, BackwardRows saved, Parts parts, unsigned rows) {
    const int lane = threadIdx.x & 63;
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int heads = KEYS ? p.Hk : p.H, i = (int)(row / (unsigned)heads), h = (int)(row % (unsigned)heads), D = p.D, d = min(lane * 2, D - 2);
    const Segment s = segment_of_row<KEYS>(p, i);
    const bool any = !s.gap && (KEYS ? s.first_query(i, p.causal) < s.q1 : s.seen(i, p.causal) > 0);
    bool nan = false;
    float2 sum[KEYS ? 2 : 1];
#pragma unroll
    for (int y = 0; y < (KEYS ? 2 : 1); ++y) {
        const float *x = parts.o + ((int64_t)y * parts.chunks * rows + row) * D + d;
        sum[y] = make_float2(0.0f, 0.0f);
        if (any) {
#pragma unroll 4
            for (int c = 0; c < parts.chunks; ++c) {
                const float2 v = *reinterpret_cast<const float2 *>(x + (int64_t)c * rows * D);
                sum[y].x += v.x;
                sum[y].y += v.y;
            }
        }
        nan |= !(sum[y].x == sum[y].x) || !(sum[y].y == sum[y].y);
    }
    float scale = p.scale;
    if constexpr (!KEYS) {   // (of the probabilities and of ds: see packed_dq)
        const int64_t at = (int64_t)h * p.Tq + i;
        const float delta = any ? saved.delta[at] : 0.0f, c = p.scale * kLog2e;
        float total = 0.0f, rest = 0.0f;
        if (any) {
            for (int x = 0; x < parts.chunks; ++x) {
                const float2 y = parts.ml[(int64_t)x * rows + row];
                total += y.x;
                rest += y.y;
            }
        }
        if (lane == 0 && any) save_row(saved, at, p.lse[at], delta, total, rest, c);
        scale = any ? scale / total : 0.0f;
        if (__any(nan) && rest == rest) {
            const EvoPacked late = parameters_again();
            const int seen = s.seen(i, late.causal);
            if (!finite(rest) || spoilt_dq<T>(late, s, h / (late.H / late.Hk), seen, min(s.nk(), seen + 62))) {   // (what other rows of a wave see, and the end of a step)
                row_dq<T, 4>(late, s, i, h, delta);
                return;
            }
        }
    }
    if constexpr (KEYS) {
        if (__any(nan)) {
            const EvoPacked late = parameters_again();
            const int from = s.first_query(i, late.causal);
            if (spoilt_dkdv<T>(late, s, h, i, i + 1, max(s.q0, from - 62), from, saved.delta)) {
                row_dkdv<T, 4>(late, s, i, h, saved.delta);
                return;
            }
        }
    }
    if (lane * 2 >= D) return;
#pragma unroll
    for (int y = 0; y < (KEYS ? 2 : 1); ++y) {
        const float f = y ? 1.0f : scale;
        typename Mfma<T>::v2 v;
        v[0] = (T)(sum[y].x * f);
        v[1] = (T)(sum[y].y * f);
        *reinterpret_cast<typename Mfma<T>::v2 *>((T *)(KEYS ? (y ? p.dv : p.dk) : p.dq) + (int64_t)row * D + lane * 2) = v;
    }
}

// How a launch fills the chip: `groups` (1 or 2) of four waves to a tile of rows, that share its walk over the other side, and `parts` of it, workgroups of their own whose results are joined by a kernel more.
struct Plan {
    int groups, parts;
    size_t bytes(int64_t rows, int columns) const { return parts > 1 ? (size_t)(parts * rows * columns * (int64_t)sizeof(float)) : 0; }
    template <typename F>
    int run(F &&f) const {
        const std::integral_constant<int, 1> one;
        const std::integral_constant<int, 2> two;
        if (parts > 1) return f(two, std::true_type());
        return groups == 2 ? f(two, std::false_type()) : f(one, std::false_type());
    }
};
// units: tiles and heads; steps: of an average sequence's walk, 64 rows each.  Two groups while the workgroups of eight waves all fit at once, two or (D = 32) three of them to a CU: 2048 causal rows
// of 24 heads and D = 128 43 us (53 with one group), of 40 heads 73 (59).  Parts: for `most` units and fewer, as many as make workgroups that all fit at once, two (the keys' side) at least, each of
// `few` steps where a CU is left to itself (up to 64 units), of `more` up to 256 and of 32 beyond: dK and dV of 12 heads (4 for keys) of D = 80, five sequences of up to 1777 rows, 55 us with 3 parts
// and 59 with 5.
constexpr int kAtOnce = EVO_D == 32 ? 768 : 512;
static Plan plan_for(int64_t units, int64_t steps, int64_t least, int64_t most, int64_t few, int64_t more) {
    Plan r = {steps >= 12 && units <= kAtOnce ? 2 : 1, 1};
    if (units && units <= most) {
        const int64_t room = kAtOnce / units < least ? least : kAtOnce / units, worth = steps / (units <= 64 ? few : units <= 256 ? more : 32), n = room < worth ? room : worth;
        r.parts = (int)(n < 1 ? 1 : n > 16 ? 16 : n);
    }
    return r;
}
static Plan query_plan(const EvoPacked &p) {
    return plan_for((p.Tq / kPackedRows + (p.n + 1) / 2) * p.H, p.Tk / (p.n ? p.n : 1) / 64, 1, 256, 8, 32);
}
// (a key's walk is over the queries of all heads that share it)
static Plan key_plan(const EvoPacked &p) {
    return plan_for((p.Tk / kPackedRows + (p.n + 1) / 2) * p.Hk, p.Tq / (p.n ? p.n : 1) * (p.H / p.Hk) / 64, 2, 400, 4, 8);
}

template <typename F>
static int by_half(int dtype, F &&f) {
    return dtype == EVO_BF16 ? f(bf16_t()) : f(f16_t());
}

}  // namespace
}  // namespace evo
