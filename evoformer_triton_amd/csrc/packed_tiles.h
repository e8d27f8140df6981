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

// Where a workgroup is: a tile of a segment, and a head.
struct Place {
    Segment s;
    int first;   // its first row (of the tensor), or, where there is nothing to do, s's end or beyond
};
template <bool KEYS, int ROWS = kPackedRows>
__device__ __forceinline__ Place place_of(const EvoPacked &p, int t) {
    auto begin = [&](int j) { return KEYS ? keys_begin(p, j) : queries_begin(p, j); };
    const int j = last_where(p.n + 2, [&](int x) { return begin(x) / ROWS + x <= t; });
    Place r;
    r.s = segment(p, j);
    const int b = KEYS ? r.s.k0 : r.s.q0, i = t - (b / ROWS + j);
    r.first = i < 0 ? INT32_MAX : (int)min((int64_t)INT32_MAX, b + (int64_t)i * ROWS);   // (below zero: offsets that do not ascend)
    return r;
}

template <typename T>
__device__ __forceinline__ void zero_rows(T *x, int first, int rows, int heads, int h, int D) {
    const int per = D / 8, n = rows * per;
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

static int64_t packed_tiles(int64_t rows, int n, int tile = kPackedRows) { return rows / tile + n + 2; }

template <typename F>
static int by_half(int dtype, F &&f) {
    return dtype == EVO_BF16 ? f(bf16_t()) : f(f16_t());
}

}  // namespace
}  // namespace evo
