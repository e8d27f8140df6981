// What the kernels of the 8-bit products share (csrc/fp8.hip, csrc/fp8_large.hip).
#pragma once

#include "common.h"
#include "bwd_common.h"
#include "kernels.h"

namespace evo {

constexpr int kF8Block = 128;   // elements that share a scale

typedef int i32x8f __attribute__((ext_vector_type(8)));
typedef int i32x4f __attribute__((ext_vector_type(4)));
typedef unsigned u32x2f __attribute__((ext_vector_type(2)));

struct F8Matmul {
    const uint8_t *a, *b;        // [M][kp], [N][kp]
    const uint32_t *sa, *sb;     // [M][sd], [N][sd]: four blocks' scales each
    const void *bias;
    void *out;
    int64_t ldo, kp;
    int M, N, blocks, sd;        // blocks of the contraction
    int mt, nt, slice;           // tiles; blocks of a slice, a multiple of four (or all)
    int bias_dtype;
};

// 16-byte chunk c of row r of a staged tile (rows of 128 bytes): any chunk of 16 rows touches all banks once
__device__ __forceinline__ int f8_swz(int r) { return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1); }
__device__ __forceinline__ int f8_at(int r, int c) { return r * 128 + ((c ^ f8_swz(r)) << 4); }
// output that row r of a 32-row accumulator tile holds: lane group g ends up with outputs 16 g .. 16 g + 15 in register order
__device__ __forceinline__ int f8_deal(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

// 16 bytes per lane from base + offset to dst (uniform) + 16 * lane, as an instruction that the compiler does not count
__device__ __forceinline__ void f8_dma(const uint8_t *base, int offset, unsigned char *dst) {
    const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(offset), "s"(base) : "m0", "memory");
}
// 4 bytes per lane
__device__ __forceinline__ void f8_dma4(const uint32_t *base, int offset, unsigned char *dst) {
    const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(offset), "s"(base) : "m0", "memory");
}
// this wave's loads have landed, everybody's have, and everybody is done with the stage before
__device__ __forceinline__ void f8_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int J>
__device__ __forceinline__ f32x16 f8_mma(i32x8f a, i32x8f b, f32x16 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, J, sa, J, sb);
}

// Eight e4m3 values (two registers) with their scale as bf16.
__device__ __forceinline__ bf16x8 f8_widen(int lo, int hi, float scale) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int w = i ? hi : lo;
        const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false), y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
        r[4 * i] = x[0];
        r[4 * i + 1] = x[1];
        r[4 * i + 2] = y[0];
        r[4 * i + 3] = y[1];
    }
    return r;
}
__device__ __forceinline__ float f8_scale(uint32_t four, int j) {
    const unsigned byte = (four >> (8 * j)) & 0xff;
    return __uint_as_float(byte ? byte << 23 : 0x400000u);
}

__device__ __forceinline__ float f8_bias(const void *b, int i, int dtype) {
    return dtype == EVO_F32 ? ((const float *)b)[i] : dtype == EVO_BF16 ? (float)((const bf16_t *)b)[i] : (float)((const f16_t *)b)[i];
}

// What the lanes of a wave have written to LDS before and read after, or the other way round: LDS takes a wave's accesses in their order, and the compiler, which
// sees that no lane reads what it has written itself, keeps that order only if it is told to.
__device__ __forceinline__ void f8_wave_sync() { asm volatile("" ::: "memory"); }

// Eight results of a row, of which the last may lie beyond it.
template <typename T>
__device__ __forceinline__ void f8_store8(T *p, const T (&e)[8], int left) {
    if (left >= 8) {
        __builtin_memcpy(p, e, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = e[i];
    }
}

// The slice and tile of a workgroup.  Tiles of a band of eight rows of tiles come one below the other: what runs at once on an XCD shares rows of both sides.
__device__ __forceinline__ void f8_tile(const F8Matmul &p, unsigned lid, int &slice, int &mt, int &nt) {
    constexpr unsigned BAND = 8;
    const unsigned tiles = p.mt * p.nt, tile = lid % tiles, band = tile / (BAND * p.nt), in = tile % (BAND * p.nt);
    const unsigned high = min(BAND, p.mt - band * BAND);
    slice = lid / tiles;
    mt = band * BAND + in % high;
    nt = in / high;
}

// A wave's results, TM x TN tiles of 32 x 32, to memory: through LDS, 32 rows at a time, so that neighbouring lanes store a row's pieces.
template <int W, int TM, int TN, typename T>
__device__ __forceinline__ void f8_store_tile(const f32x16 (&acc)[TN][TM], const F8Matmul &p, unsigned char *lds, const float *bias, int wave, int lane, int m0,
                                              int n0, int wm, int wn, int slice) {
    constexpr int ROW = TN * 32 * sizeof(T), CHUNKS = TN * 4;   // bytes of a row, chunks of eight results
    const int li = lane & 31, g = lane >> 5;
    unsigned char *mine = lds + wave * 32 * ROW;
    auto place = [](int r, int c) { return r * ROW + ((c ^ (r & (CHUNKS - 1))) * (int)(8 * sizeof(T))); };
    T *out = (T *)p.out + (int64_t)slice * p.M * p.N;
#pragma unroll
    for (int u = 0; u < TM; ++u) {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 *b = reinterpret_cast<const f32x4 *>(bias + wn + 32 * t + 16 * g + 8 * h);
                T e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = (T)(acc[t][u][8 * h + i] + b[i / 4][i % 4]);
                __builtin_memcpy(__builtin_assume_aligned(mine + place(li, 4 * t + 2 * g + h), 16), e, sizeof e);
            }
        }
        f8_wave_sync();
        constexpr int RPI = 64 / CHUNKS;   // rows that the wave's lanes store at once
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            const int r = i * RPI + lane / CHUNKS, c = lane % CHUNKS, m = m0 + wm + 32 * u + r, o = n0 + wn + 8 * c;
            T e[8];
            __builtin_memcpy(e, __builtin_assume_aligned(mine + place(r, c), 16), sizeof e);
            if (m < p.M && o < p.N) f8_store8(out + (int64_t)m * p.ldo + o, e, p.N - o);
        }
        f8_wave_sync();
    }
}

int launch_fp8_large(const F8Matmul &a, int slices, int dtype, hipStream_t st);

}  // namespace evo
