// Large products of 8-bit matrices: tiles of 256 x 256, four waves of 128 x 128 (4 x 4 tiles of v_mfma_scale_f32_32x32x64, 256 accumulation
// registers), one per SIMD, and one workgroup per CU that stays for several tiles.
//
// A stage is 64 of the contraction of 512 rows, 32 KB, in a ring of four.  Step g multiplies the operands of stage g, which lie in registers, while those
// of stage g + 1 are read from LDS and stage g + 4 is asked for into the place of stage g.  One barrier a step: ahead of it a wave's reads of
// stage g and its loads of stage g + 1 are done (stages g + 2 and g + 3, eight loads each, may be under way).  The stages of a workgroup's tiles follow one another
// without a gap, so that the next tile's first ones are on their way while a tile's results are stored.
//
// A wave of 128 x 128 reads 16 KB of LDS for 16 products of 64 cycles; with eight waves of 128 x 64, whose reads took turns with the products of the other wave
// of a SIMD, LDS had 96 KB to deliver and 32 to take in the 1024 cycles of a step and was what bounded it.
#include <type_traits>

#include "fp8_common.h"

namespace evo {

namespace {
constexpr int SIDE = 256, ROW = 64, STAGE = 2 * SIDE * ROW, RING = 4, PIECES = 8, TT = 4;
constexpr int SCALES = RING * STAGE, BIAS = SCALES + 4 * 2 * SIDE * 4, EPILOGUE = BIAS + 4 * SIDE * 4, LDS = EPILOGUE + 4 * 4096;
// The same value, which the compiler does not carry from one use to the next (a kernel that keeps 256 sums and 104 registers of operands has no room for
// what could be formed ahead of its loops).
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
// Bytes that loads into LDS take, 16 or 4 per lane, from `off` + `more` (uniform) on to dst (uniform) + 16 or 4 * lane; those beyond the end read as zeros.
// Instructions that the compiler does not count.
struct Source {
    __amdgpu_buffer_rsrc_t rs;
    Source() = default;
    __device__ __forceinline__ Source(const void *p, unsigned bytes) : rs(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000)) {}
    __device__ __forceinline__ void dma16(int off, int more, unsigned char *dst) const {
        const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)dst;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(to), "v"(off), "s"(rs), "s"(more) : "m0", "memory");
    }
    __device__ __forceinline__ void dma4(int off, int more, unsigned char *dst) const {
        const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)dst;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(to), "v"(off), "s"(rs), "s"(more) : "m0", "memory");
    }
};
// acc += a b^T times the scales in byte J of sa and sb.  As an instruction that the compiler does not know, with the sums in accumulation
// registers: they take all 256 of them, and the compiler's own copies of sums, for which it keeps some, went through memory.  (Independent products follow
// one another; what else touches a sum keeps the distance itself: `settle`.)
template <int J>
__device__ __forceinline__ void product(f32x16 &acc, const i32x8f &a, const i32x8f &b, int sa, int sb) {
    if constexpr (J == 0) asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (J == 1) asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (J == 2) asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}
// acc = 0, as a product of zeros (256 zeros by way of the vector unit take four times as long)
__device__ __forceinline__ void clear(f32x16 &acc, const i32x4f &zeros) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(zeros)); }
// between a product and what else reads or writes its sum: 20 states at least
__device__ __forceinline__ void settle(f32x16 (&acc)[TT][TT]) {
    asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int n = 0; n < TT * TT; ++n) asm volatile("" : "+a"(acc[n / TT][n % TT]));
}
}  // namespace

template <typename T>
__global__ void __launch_bounds__(256, 1) fp8_matmul_large(F8Matmul p, int slices) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds8[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const int wm = (wave & 1) * 128, wn = (wave >> 1) * 128;

    // this workgroup's tiles: every gx-th of its XCD's
    const unsigned total = p.mt * p.nt * slices, x = blockIdx.x % 8, place = blockIdx.x / 8, gx = (gridDim.x + 7 - x) / 8;
    const unsigned start = x * (total / 8) + min(x, total % 8), size = total / 8 + (x < total % 8 ? 1 : 0);
    const int mine = place < size ? (int)((size - place + gx - 1) / gx) : 0;
    if (mine == 0) return;

    // A wave brings 128 rows, 16 rows of 64 bytes at a time: waves 0 and 1 of a, 2 and 3 of b.  Rows that a tile does not have read as zeros.
    const bool tokens = wave < 2;
    const int at = (wave & 1) * 128, es = p.bias_dtype == EVO_F32 ? 4 : 2;
    struct Tile {
        int slice, m0, n0, ns;
        Source rows, scales, bias;
    };
    auto tile_of = [&](int i) {
        Tile t;
        f8_tile(p, start + place + i * gx, t.slice, t.m0, t.n0);
        t.m0 *= SIDE;
        t.n0 *= SIDE;
        const int first = t.slice * p.slice, r0 = tokens ? t.m0 : t.n0, have = min((tokens ? p.M : p.N) - r0, SIDE);
        t.ns = 2 * min(p.slice, p.blocks - first);
        t.rows = Source((tokens ? p.a : p.b) + r0 * p.kp + (int64_t)first * kF8Block, (unsigned)(have * p.kp - (int64_t)first * kF8Block));
        t.scales = Source((tokens ? p.sa : p.sb) + (int64_t)r0 * p.sd + first / 4, (unsigned)(have * p.sd - first / 4) * 4);
        t.bias = Source((const char *)p.bias + (int64_t)t.n0 * es, p.bias ? (unsigned)(((p.N - t.n0) * (int64_t)es + 3) & ~3) : 0);
        return t;
    };
    int off[PIECES], soff[2];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int r = at + i * 16 + lane / 4, row = tokens ? r : (r & ~31) + f8_deal(r & 31);
        off[i] = row * (int)p.kp + (((lane % 4) ^ ((r >> 2) & 3)) << 4);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = at + i * 64 + lane;
        soff[i] = (tokens ? r : (r & ~31) + f8_deal(r & 31)) * p.sd * 4;
    }
    int fslot = 0, fscale = 0, fbias = 0;
    auto fetch_extra = [&](const Tile &t, int s) {   // what a stage has besides: its eight steps' scales, its tile's bias as it lies
        if (s % 8 == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) t.scales.dma4(soff[i], s / 2, lds8 + SCALES + fscale * (2 * SIDE * 4) + ((tokens ? 0 : SIDE) + at + i * 64) * 4);
            fscale = (fscale + 1) & 3;
            if (s == 0) {
                t.bias.dma4(threadIdx.x * 4, 0, lds8 + BIAS + fbias * (SIDE * 4) + wave * 256);
                fbias = (fbias + 1) & 3;
            }
        }
    };
    auto fetch_piece = [&](const Tile &t, int s, int i) { t.rows.dma16(off[i], s * ROW, lds8 + fslot * STAGE + ((tokens ? 0 : SIDE) + at + i * 16) * ROW); };
    Tile tile = tile_of(0);
#pragma unroll 1
    for (int s = 0; s < 4; ++s) {   // (a tile has four stages at least)
        fetch_extra(tile, s);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) fetch_piece(tile, s, i);
        fslot = (fslot + 1) & 3;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    const int rs = (li >> 2) & 3;
    const unsigned char *ap = lds8 + (wm + li) * ROW, *bp = lds8 + (SIDE + wn + li) * ROW;
    const int c0 = ((2 * g) ^ rs) << 4, c1 = ((2 * g + 1) ^ rs) << 4;
    // Operands: of a two stages' (all of them are wanted until a step's end), of b one stage's and one more: b[t] is read again as soon as its products are under way,
    // the last one's place takes turns with a fifth.
    i32x8f a[2][TT], b[TT + 1];
    int slot = 0, sc = 0, bi = 0;
    auto half = [&](i32x8f &v, const unsigned char *row, int h) {
        const i32x4f x = *reinterpret_cast<const i32x4f *>(row + slot * STAGE + (h ? c1 : c0));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = x[i];
    };
    int xs[TT], ws[TT], xn[TT], wn4[TT];
    auto read_scales = [&]() {
        const int *s = reinterpret_cast<const int *>(lds8 + SCALES + sc * (2 * SIDE * 4));
#pragma unroll
        for (int u = 0; u < TT; ++u) xn[u] = s[wm + 32 * u + li];
#pragma unroll
        for (int t = 0; t < TT; ++t) wn4[t] = s[SIDE + wn + 32 * t + li];
        sc = (sc + 1) & 3;
    };
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            half(a[0][t], ap + t * 32 * ROW, h);
            half(b[t], bp + t * 32 * ROW, h);
        }
    read_scales();

#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
        const bool another = i + 1 < mine;
        const Tile then = another ? tile_of(i + 1) : tile;
        const int ns = tile.ns, slice = tile.slice, m0 = tile.m0, n0 = tile.n0;
        f32x16 acc[TT][TT];
        {
            i32x4f zeros = {fresh(0), fresh(0), fresh(0), fresh(0)};
            asm volatile("s_nop 4" : "+v"(zeros));
#pragma unroll
            for (int n = 0; n < TT * TT; ++n) clear(acc[n / TT][n % TT], zeros);
            settle(acc);
        }
#pragma unroll 1
        for (int s8 = 0; s8 < ns; s8 += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int s = s8 + j, now = j & 1, next = now ^ 1;
                if (j % 2 == 0 && s >= ns) break;
                if (!another && s + 3 >= ns) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                if (j == 0) {
#pragma unroll
                    for (int u = 0; u < TT; ++u) {
                        xs[u] = xn[u];
                        ws[u] = wn4[u];
                    }
                }
                slot = (slot + 1) & 3;
                const bool here = s + 4 < ns, more = here || another;
                const Tile &from = here ? tile : then;
                const int fs = here ? s + 4 : s + 4 - ns;
                if (more) fetch_extra(from, fs);
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const int t = n / TT, u = n % TT;
                    const i32x8f &bo = t == TT - 1 && now ? b[TT] : b[t], &ao = a[now][u];
                    if (j / 2 == 0) product<0>(acc[t][u], bo, ao, ws[t], xs[u]);
                    else if (j / 2 == 1) product<1>(acc[t][u], bo, ao, ws[t], xs[u]);
                    else if (j / 2 == 2) product<2>(acc[t][u], bo, ao, ws[t], xs[u]);
                    else product<3>(acc[t][u], bo, ao, ws[t], xs[u]);
                    if (n < 8) half(a[next][n / 2], ap + n / 2 * 32 * ROW, n & 1);
                    if (n >= 4 && n % 4 < 2 && n < 15) half(b[n / 4 - 1], bp + (n / 4 - 1) * 32 * ROW, n & 1);
                    if (n == 10 || n == 11) half(next ? b[TT] : b[TT - 1], bp + (TT - 1) * 32 * ROW, n & 1);
                    if (n >= 8 && more) fetch_piece(from, fs, n - 8);
                    if (n == 8 && j % 2 == 1 && (j == 7 || s == ns - 1)) read_scales();
                    __builtin_amdgcn_sched_barrier(0);
                }
                fslot = (fslot + 1) & 3;
            }
        }
        settle(acc);
        // The tile's results, 16 rows at a time by way of LDS.  (What was read for a stage beyond the last one is not used.)
        const int lane = fresh(threadIdx.x & 63), li = lane & 31, g = lane >> 5;
        const unsigned char *raw = lds8 + BIAS + bi * (SIDE * 4);
        bi = (bi + 1) & 3;
        auto biased = [&](const f32x16 &v, int t, int h, T (&e)[8]) {
            float w[8];
            const int o = wn + 32 * t + 16 * g + 8 * h;
            if (!p.bias) {
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = 0.0f;
            } else if (p.bias_dtype == EVO_F32) {
                __builtin_memcpy(w, __builtin_assume_aligned(raw + o * 4, 16), sizeof w);
            } else if (p.bias_dtype == EVO_BF16) {
                const bf16x8 x = *reinterpret_cast<const bf16x8 *>(raw + o * 2);
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = (float)x[k];
            } else {
                const f16x8 x = *reinterpret_cast<const f16x8 *>(raw + o * 2);
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = (float)x[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = (T)(v[8 * h + k] + w[k]);
        };
        T *out = (T *)p.out + (int64_t)slice * p.M * p.N;
        unsigned char *hold = lds8 + EPILOGUE + wave * 4096;
#pragma unroll
        for (int u = 0; u < TT; ++u) {
            if constexpr (sizeof(T) == 4) {
                const int m = m0 + wm + 32 * u + li;
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int o = n0 + wn + 32 * t + 16 * g + 8 * h;
                        T e[8];
                        biased(acc[t][u], t, h, e);
                        if (m < p.M && o < p.N) f8_store8(out + (int64_t)m * p.ldo + o, e, p.N - o);
                    }
            } else {
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const int r16 = li & 15;
                    if (li >> 4 == part) {
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                T e[8];
                                biased(acc[t][u], t, h, e);
                                __builtin_memcpy(__builtin_assume_aligned(hold + r16 * 256 + (((4 * t + 2 * g + h) ^ r16) << 4), 16), e, sizeof e);
                            }
                    }
                    f8_wave_sync();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = 4 * k + lane / 16, c = lane % 16, m = m0 + wm + 32 * u + 16 * part + r, o = n0 + wn + 8 * c;
                        T e[8];
                        __builtin_memcpy(e, __builtin_assume_aligned(hold + r * 256 + ((c ^ r) << 4), 16), sizeof e);
                        if (m < p.M && o < p.N) f8_store8(out + (int64_t)m * p.ldo + o, e, p.N - o);
                    }
                    f8_wave_sync();
                }
            }
        }
        tile = then;
    }
}

int launch_fp8_large(const F8Matmul &a, int slices, int dtype, hipStream_t st) {
    auto go = [&](auto t) {
        typedef decltype(t) T;
        static PerDevice done;
        int cus = 0;
        if (const int rc = ensure_dynamic_lds((const void *)fp8_matmul_large<T>, LDS, done, &cus)) return rc;
        const int64_t total = (int64_t)a.mt * a.nt * slices;
        fp8_matmul_large<T><<<(unsigned)(total < cus ? total : cus), 256, LDS, st>>>(a, slices);
        return hip_rc();
    };
    return dtype == EVO_BF16 ? go(bf16_t()) : dtype == EVO_F16 ? go(f16_t()) : go(float());
}

}  // namespace evo
