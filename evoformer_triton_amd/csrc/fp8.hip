// Linear layers in 8 bits: e4m3 operands with a power-of-two scale (E8M0, the exponent + 127) for each block of 128 along the
// contraction, y = Q(x) Q(w)^T + b.  The rounding of a matrix (fp8_quantize, fp8_quantize_two: along its rows, its columns or both in one pass), and products of two
// rounded matrices that both lie with the contraction along their rows: tiles of 128 x 128 (fp8_matmul) and of 256 x 256 (fp8_matmul_big), strips of 128 rows for up to four
// blocks (fp8_strip), up to 64 rows (fp8_few), and the sum of a contraction's slices (fp8_slices).  A training step's products are all of that form:
//   y = Qk(x) Qk(w)^T,  dx = Qn(dy) Qn(w^T)^T,  dw = Qm(dy^T) Qm(x^T)^T
// each operand rounded along the axis that its product contracts.  A copy of 1 GB runs at 5.1 TB/s both ways here, of 67 MB at up to 7.9; the bf16 product of 8192^3 at
// 1211 TFLOP/s, the library's 8-bit one (one scale for a matrix) at 2790 to 2900.
//
// Sums.  On gfx950 all 8-bit products add eight neighbouring values of a lane with what lies 13 bits below the largest of them cut off; between those groups, and to the
// accumulator, 24 bits count.  That is 1.4e-5 of a result on normal data, where the roundings to 8 bits are up to 2^-4 each and that of a bf16 result up to 2^-9 of what
// they round, for half the time that bf16 products take: a bf16 result is another one than with fp32 sums in one entry of 25 to 75, an fp16 one in one of 7 to 13, mostly by a last bit, and
// as far from 64 bits (1.7e-3 and 2.1e-4).  fp32 results are not given that: their operands are widened to bf16, exactly for values from 2^-133 on (a smaller one, of a block
// whose largest is below 2^-115, loses bits) and below 2^128, and take its products, whose sums are fp32 (WIDE).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elements.h"
#include "kernels.h"

namespace evo {

constexpr int kF8Block = 128;   // elements that share a scale

typedef int i32x8f __attribute__((ext_vector_type(8)));
typedef int i32x4f __attribute__((ext_vector_type(4)));
typedef unsigned u32x2f __attribute__((ext_vector_type(2)));

static int64_t f8_pitch(int64_t k) { return (k + kF8Block - 1) / kF8Block * kF8Block; }             // bytes of a rounded row
static int64_t f8_scale_pitch(int64_t k) { return (k + 4 * kF8Block - 1) / (4 * kF8Block) * 4; }   // bytes of its scales

// Eight elements, at any element's address: global memory takes 16 bytes at any alignment.  (As a vector type: copied element by element, the whole and the partial
// store of a row's end became one sequence of two-byte stores, and the results of 256 x 256 took longer than 8 blocks of their products.)
template <typename T>
struct F8Eight {
    typedef T V __attribute__((ext_vector_type(8)));
    typedef V U __attribute__((aligned(sizeof(T))));
    V v;
    __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const U *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<U *>(p) = v; }
    __device__ __forceinline__ void store_some(T *p, int left) const {   // the first `left`
        if (left >= 8) {
            store(p);
            return;
        }
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) p[i] = v[i];
    }
};

// ---- rounding ----

// The exponent e of a block whose largest finite magnitude has these bits: the least with magnitude <= 448 2^e, at least -127 (0 for a block of zeros).
__device__ __forceinline__ int f8_exponent(unsigned amax) {
    const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);   // 448 = 1.75 * 2^8
    return amax ? max(e, -127) : 0;
}
__device__ __forceinline__ float f8_power(int e) { return __uint_as_float(e == -127 ? 0x400000u : (unsigned)(e + 127) << 23); }   // 2^e

// Magnitudes of 16-bit types are compared as whole numbers, two at a time; infinities and NaN, which count for nothing, come out the largest and are looked for only then.
template <typename T>
struct F8Bits {
    static constexpr bool HALF = sizeof(T) == 2;
    typedef typename std::conditional<HALF, uint16_t, uint32_t>::type U;
    typedef U V __attribute__((ext_vector_type(8)));
    static constexpr U INF = !HALF ? 0x7f800000u : std::is_same<T, bf16_t>::value ? 0x7f80 : 0x7c00;
    __device__ __forceinline__ static V of(const F8Eight<T> &e) { return __builtin_bit_cast(V, e.v) & (U)(HALF ? 0x7fff : 0x7fffffff); }
    __device__ __forceinline__ static V finite(V v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] < INF ? v[i] : (U)0;
        return v;
    }
    __device__ __forceinline__ static unsigned most(V v) {
        const auto a = __builtin_elementwise_max(v.lo, v.hi);
        const auto b = __builtin_elementwise_max(a.lo, a.hi);
        return max((unsigned)b[0], (unsigned)b[1]);
    }
    // a magnitude as that of a float
    __device__ __forceinline__ static unsigned wide(unsigned m) {
        if constexpr (!HALF) return m;
        else if constexpr (std::is_same<T, bf16_t>::value) return m << 16;
        else return __float_as_uint((float)__builtin_bit_cast(f16_t, (uint16_t)m));
    }
};
// The largest finite magnitude of each of the eight places, of N times eight values.
template <int N, typename T>
__device__ __forceinline__ typename F8Bits<T>::V f8_magnitudes(const F8Eight<T> (&e)[N]) {
    typename F8Bits<T>::V all = F8Bits<T>::of(e[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) all = __builtin_elementwise_max(all, F8Bits<T>::of(e[i]));
    if (F8Bits<T>::most(all) >= F8Bits<T>::INF) {
        all = F8Bits<T>::finite(F8Bits<T>::of(e[0]));
#pragma unroll
        for (int i = 1; i < N; ++i) all = __builtin_elementwise_max(all, F8Bits<T>::finite(F8Bits<T>::of(e[i])));
    }
    return all;
}

// The largest of all, as that of a float.
template <int N, typename T>
__device__ __forceinline__ unsigned f8_largest(const F8Eight<T> (&e)[N]) {
    typedef F8Bits<T> B;
    if constexpr (B::HALF) return B::wide(B::most(f8_magnitudes(e)));
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) m = max(m, (unsigned)B::of(e[i])[c]);
    if (m >= B::INF) {
        m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int c = 0; c < 8; ++c) m = max(m, (unsigned)B::finite(B::of(e[i]))[c]);
    }
    return m;
}

// Two values over `scale`, a power of two, as e4m3, to nearest, ties to even; infinities and NaN as NaN.
template <bool HI, typename T>
__device__ __forceinline__ int f8_pair(int old, T a, T b, float scale) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    typedef T V __attribute__((ext_vector_type(2)));
    s16x2 o = __builtin_bit_cast(s16x2, old);
    if constexpr (sizeof(T) == 4) o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, a, b, scale, HI);
    else if constexpr (std::is_same<T, bf16_t>::value) o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, V{a, b}, scale, HI);
    else o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, V{a, b}, scale, HI);
    return __builtin_bit_cast(int, o);
}
template <typename T>
__device__ __forceinline__ int f8_pack(T a, T b, T c, T d, float scale) {
    return f8_pair<true>(f8_pair<false>(0, a, b, scale), c, d, scale);
}
template <int N>
__device__ __forceinline__ unsigned f8_max_ror(unsigned v) {   // with the value N lanes further within 16
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 | N, 0xf, 0xf, false));
}
__device__ __forceinline__ unsigned f8_max16(unsigned v) { return f8_max_ror<1>(f8_max_ror<2>(f8_max_ror<4>(f8_max_ror<8>(v)))); }

// over the four groups of 16 lanes
__device__ __forceinline__ unsigned f8_max_rows(unsigned v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}
template <typename V>   // eight values each, of 16 or 32 bits
__device__ __forceinline__ V f8_max_rows(V v) {
    typedef unsigned W __attribute__((ext_vector_type(sizeof(V) / 4)));
    W w = __builtin_bit_cast(W, v), x, y;
#pragma unroll
    for (int i = 0; i < (int)sizeof(V) / 4; ++i) {
        const auto a = __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
        x[i] = a[0];
        y[i] = a[1];
    }
    v = __builtin_elementwise_max(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y));
    w = __builtin_bit_cast(W, v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(V) / 4; ++i) {
        const auto a = __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);
        x[i] = a[0];
        y[i] = a[1];
    }
    return __builtin_elementwise_max(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y));
}
__device__ __forceinline__ float f8_sum_rows(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

struct F8Quantize {
    const void *x;
    int64_t ldx, rows;
    int cols, sp, tiles_k;        // sp: bytes of a row's scales
    int64_t spt, tiles_r;         // of a column's
    int64_t kp, rp;               // bytes of a rounded row, of a rounded column
    uint8_t *q, *s, *qt, *st;
    float *sums;
};

// The scale of block k of a row (or column) of `blocks`; with the last one, the places up to the next multiple of four.
__device__ __forceinline__ void f8_store_scale(uint8_t *s, int64_t k, int64_t blocks, int64_t pitch, uint8_t scale) {
    s[k] = scale;
    if (k == blocks - 1) {
        if (k + 1 < pitch) s[k + 1] = 127;
        if (k + 2 < pitch) s[k + 2] = 127;
        if (k + 3 < pitch) s[k + 3] = 127;
    }
}

// Bound by memory: x once, the bytes once or twice.  A workgroup takes whole blocks both ways, so that one pass gives both roundings and the column sums for the bias's
// gradient; the transposed bytes are turned in LDS.  8192 x 8192 bf16 both ways 50.6 us (5.3 TB/s), 32 768 x 1024 27.6, along its rows alone 8192 x 4096 18.0 (5.6 TB/s).  With one
// float at a time through maxima, scaling and conversion 32 768 x 256 along its rows took 7.9 us instead of 7.3.
// A workgroup rounds R rows x 128 columns, 128 rows where it rounds columns, too: thread t V rows (V (t / 16) ..) of eight columns (8 (t % 16) ..).
template <typename T, int R, int V, bool ROWS, bool COLS>
__device__ __forceinline__ void f8_quantize(const F8Quantize &p, unsigned id) {
    static_assert(R == 128 || !COLS, "a column's block is 128 rows");
    typedef F8Bits<T> B;
    constexpr int WAVES = R / V / 4, THREADS = R / V * 16;
    __shared__ __attribute__((aligned(16))) unsigned char tile[COLS ? 128 * 128 : 16];
    __shared__ unsigned amaxs[COLS ? WAVES : 1][128];
    __shared__ float sums[COLS ? WAVES : 1][128];
    __shared__ __attribute__((aligned(16))) float col_scale[COLS ? 128 : 4];
    __shared__ uint8_t row_scale[R];
    const int t = threadIdx.x, cg = t % 16, rg = t / 16, wave = t / 64;
    const int kt = id % p.tiles_k;
    const int64_t rt = id / p.tiles_k;
    const int c0 = kt * 128 + cg * 8;
    const int64_t r0 = rt * R + rg * V;
    F8Eight<T> e[V];
    const T *x = (const T *)p.x;
    const bool last_rows = (rt + 1) * R >= p.rows, ragged = (kt + 1) * 128 > p.cols;   // uniform
    const bool corner = ragged && last_rows;
    if (p.cols >= 8 && (!corner || p.rows >= 2)) {
        // All loads under way together: rows beyond the last repeat it, and what lies behind a row's end is the next row's; the last row of all, which may not be read
        // beyond, element by element.
        T l[8];
#pragma unroll
        for (int i = 0; i < V; ++i) e[i].load(x + min(r0 + i, p.rows - (corner ? 2 : 1)) * p.ldx + (c0 < p.cols ? c0 : 0));
        if (corner) {
#pragma unroll
            for (int c = 0; c < 8; ++c) l[c] = x[(p.rows - 1) * p.ldx + min(c0 + c, p.cols - 1)];
        }
        if (corner) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int c = 0; c < 8; ++c) e[i].v[c] = r0 + i == p.rows - 1 ? l[c] : e[i].v[c];
        }
        if (last_rows || ragged) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (r0 + i >= p.rows || c0 + c >= p.cols) e[i].v[c] = (T)0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const T one = x[min(r0 + i, p.rows - 1) * p.ldx + min(c0 + c, p.cols - 1)];
                e[i].v[c] = r0 + i < p.rows && c0 + c < p.cols ? one : (T)0.0f;
            }
    }
    if (ROWS && p.q) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const F8Eight<T> one[1] = {e[i]};
            const auto &v = e[i].v;
            const int ex = f8_exponent(f8_max16(f8_largest(one)));
            const float scale = f8_power(ex);
            if (r0 + i < p.rows) {
                *reinterpret_cast<u32x2f *>(p.q + (r0 + i) * p.kp + c0) =
                    u32x2f{(unsigned)f8_pack(v[0], v[1], v[2], v[3], scale), (unsigned)f8_pack(v[4], v[5], v[6], v[7], scale)};
            }
            if (cg == 0) row_scale[rg * V + i] = (uint8_t)(ex + 127);
        }
    }
    if constexpr (COLS) if (p.qt) {
        const typename B::V a = f8_max_rows(f8_magnitudes(e));
        float s[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            s[c] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) s[c] += (float)e[i].v[c];
            s[c] = f8_sum_rows(s[c]);
        }
        if (rg % 4 == 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                amaxs[wave][cg * 8 + c] = a[c];
                sums[wave][cg * 8 + c] = s[c];
            }
        }
        __syncthreads();
        if (t < 128) {
            unsigned most = 0;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                most = max(most, amaxs[w][t]);
                s += sums[w][t];
            }
            const int ex = f8_exponent(B::wide(most));
            col_scale[t] = f8_power(ex);
            if (kt * 128 + t < p.cols) {
                f8_store_scale(p.st + (kt * 128 + t) * p.spt, rt, p.tiles_r, p.spt, (uint8_t)(ex + 127));
                if (p.sums) p.sums[rt * p.cols + kt * 128 + t] = s;
            }
        }
        __syncthreads();
        // byte of row r of column col: 16-byte chunks of a column's 128 rows, moved about so that neighbouring columns' lie in different banks
        auto at = [](int col, int r) { return col * 128 + (((r >> 4) ^ ((col >> 3) & 7)) << 4) + (r & 15); };
        float scales[8];
        __builtin_memcpy(scales, __builtin_assume_aligned(col_scale + cg * 8, 16), sizeof scales);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int col = cg * 8 + c;
            const float scale = scales[c];
            if constexpr (V == 8) {
                *reinterpret_cast<u32x2f *>(tile + at(col, rg * 8)) =
                    u32x2f{(unsigned)f8_pack<T>(e[0].v[c], e[1].v[c], e[2].v[c], e[3].v[c], scale), (unsigned)f8_pack<T>(e[4].v[c], e[5].v[c], e[6].v[c], e[7].v[c], scale)};
            } else {
                static_assert(V == 2, "");
                *reinterpret_cast<uint16_t *>(tile + at(col, rg * 2)) = (uint16_t)f8_pair<false, T>(0, e[0].v[c], e[1].v[c], scale);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 1024 / THREADS; ++k) {
            const int col = t / 8 + THREADS / 8 * k, slot = t % 8;
            if (kt * 128 + col < p.cols)
                *reinterpret_cast<i32x4f *>(p.qt + (int64_t)(kt * 128 + col) * p.rp + rt * 128 + slot * 16) = *reinterpret_cast<const i32x4f *>(tile + at(col, slot * 16));
        }
    }
    if constexpr (ROWS) if (p.q) {
        if (!COLS || !p.qt) __syncthreads();
        if (t < R && rt * R + t < p.rows) f8_store_scale(p.s + (rt * R + t) * p.sp, kt, p.tiles_k, p.sp, row_scale[t]);
    }
}
template <typename T, int R, int V, bool ROWS, bool COLS>
__global__ void __launch_bounds__(R / V * 16) fp8_quantize(F8Quantize p) {
    f8_quantize<T, R, V, ROWS, COLS>(p, blockIdx.x);
}
// Two matrices, each both ways or one, in one launch: a weight of a few tiles takes a launch's time (1024 x 256 6 us) beside its input (32 768 x 256 7).
struct F8Two {
    F8Quantize p[2];
    unsigned first;   // tiles of the first
};
template <typename T, int V>
__global__ void __launch_bounds__(128 / V * 16) fp8_quantize_two(F8Two a) {
    const unsigned second = blockIdx.x >= a.first ? 1 : 0;
    f8_quantize<T, 128, V, true, true>(a.p[second], blockIdx.x - second * a.first);
}

// Column sums from those of 128 rows each.  A launch's time: 256 parts of 1024 columns 3.8 us.
__global__ void __launch_bounds__(1024) sums_of_parts(const float *part, void *out, int cols, int64_t parts, int dtype) { sum_parts<32>(part, out, cols, parts, dtype, blockIdx.x); }
int launch_sum_parts(const float *part, void *out, int cols, int64_t parts, int dtype, hipStream_t st) {
    sums_of_parts<<<(unsigned)((cols + 31) / 32), 1024, 0, st>>>(part, out, cols, parts, dtype);
    return hip_rc();
}

// ---- product ----

struct F8Matmul {
    const uint8_t *a, *b;        // [M][kp], [N][kp]
    const uint32_t *sa, *sb;     // [M][sd], [N][sd]: four blocks' scales each
    const void *bias;
    void *out;
    int64_t ldo, kp;
    int M, N, blocks, sd;        // blocks of the contraction
    int mt, nt, slice;           // tiles; blocks of a slice, a multiple of four (or all)
    int bias_dtype;
    const void *x;               // strips, rounded on the way: [M][k], rows ldx apart
    int64_t ldx;
    int k, pieces, tiles;        // strips: workgroups that share one's columns, tiles of a workgroup
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

// What the lanes of a wave have written to LDS before and read after, or the other way round: LDS takes a wave's accesses in their order, and the compiler, which
// sees that no lane reads what it has written itself, keeps that order only if it is told to.
__device__ __forceinline__ void f8_wave_sync() { asm volatile("" ::: "memory"); }

// A workgroup's slice and tile.  Tiles of a band of eight rows of tiles come one below the other: what runs at once on an XCD shares rows of both sides.
__device__ __forceinline__ void f8_tile(const F8Matmul &p, int &slice, int &mt, int &nt) {
    constexpr unsigned BAND = 8;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x), tiles = p.mt * p.nt, tile = lid % tiles, band = tile / (BAND * p.nt), in = tile % (BAND * p.nt);
    const unsigned high = min(BAND, p.mt - band * BAND);
    slice = lid / tiles;
    mt = band * BAND + in % high;
    nt = in / high;
}

// A wave's results, TM x TN tiles of 32 x 32, to memory: through LDS, 32 rows at a time, so that neighbouring lanes store a row's pieces.
template <int TN, typename T>
constexpr int kF8TileLds = 32 * TN * 32 * sizeof(T);   // bytes that a wave needs for that
template <int TM, int TN, typename T>
__device__ __forceinline__ void f8_store_tile(const f32x16 (&acc)[TN][TM], const F8Matmul &p, unsigned char *mine, const float *bias, int lane, int m0, int n0, int wm,
                                              int wn, int slice) {
    constexpr int ROW = TN * 32 * sizeof(T), CHUNKS = TN * 4;   // bytes of a row, chunks of eight results
    const int li = lane & 31, g = lane >> 5;
    auto place = [](int r, int c) { return r * ROW + ((c ^ (r & (CHUNKS - 1))) * (int)(8 * sizeof(T))); };
    T *out = (T *)p.out + (int64_t)slice * p.M * p.N;
    const bool inside = m0 + wm + 32 * TM <= p.M && n0 + wn + 32 * TN <= p.N;   // uniform
#pragma unroll
    for (int u = 0; u < TM; ++u) {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 *b = reinterpret_cast<const f32x4 *>(bias + wn + 32 * t + 16 * g + 8 * h);
                F8Eight<T> e;
#pragma unroll
                for (int i = 0; i < 8; ++i) e.v[i] = (T)(acc[t][u][8 * h + i] + b[i / 4][i % 4]);
                *reinterpret_cast<typename F8Eight<T>::V *>(mine + place(li, 4 * t + 2 * g + h)) = e.v;
            }
        }
        f8_wave_sync();
        constexpr int RPI = 64 / CHUNKS;   // rows that the wave's lanes store at once
        const int c = lane % CHUNKS, o = n0 + wn + 8 * c;
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            const int r = i * RPI + lane / CHUNKS, m = m0 + wm + 32 * u + r;
            F8Eight<T> e;
            e.v = *reinterpret_cast<const typename F8Eight<T>::V *>(mine + place(r, c));
            T *to = out + (int64_t)m * p.ldo + o;
            if (inside) e.store(to);
            else if (m < p.M && o < p.N) e.store_some(to, p.N - o);
        }
        f8_wave_sync();
    }
}

// out[m][n] (+ slice M N) = sum over the slice's blocks of a[m] . b[n], times the scales, + bias[n].  WM x WN waves of TM x TN tiles
// of 32 x 32; outputs (rows of b) are the accumulators' rows, rows of a their columns: a lane then holds 16 outputs side by side.  128 x 128 with two stages of a block each:
// 64 KB, two workgroups to a unit, one of which multiplies while the other waits for its loads or stores; eight waves of 32 x 64, two of a SIMD in turn (us, instead of four of
// 64 x 64, on one card: 2048^3 13.0 / 14.4, 1024 x 4096 x 1024 9.0 / 9.8, 32 768 x 256 x 1024 15.1 / 15.0; four stages for the one workgroup that then fits: 14.8, 9.8, 14.7).  Bound by those
// loads and stores: 32 768 x 256 x 1024 in 13.6 us on another (1260 TFLOP/s; 50 MB, 3.7 TB/s); results written two bytes at a time instead of 16 made 32 768 x 1024 x 256 30 us instead of 23.
template <int WM, int WN, int TM, int TN, typename T, bool WIDE>
__global__ void __launch_bounds__(WM * WN * 64, 2) fp8_matmul(F8Matmul p) {
    constexpr int W = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32, STAGE = (BM + BN) * 128, PIECES = (BM + BN) / 8 / W, SCALES = 2 * STAGE,
                  BIAS = SCALES + 2 * (BM + BN) * 4;
    static_assert(BM / 8 % PIECES == 0 && PIECES % 4 == 0, "a wave brings rows of one side, 32 at least");
    constexpr int ROWS = (BM + BN) / W;
    static_assert(ROWS <= 64, "a lane brings a row's scales");
    static_assert(W * kF8TileLds<TN, T> <= 2 * STAGE, "what the waves hold of their results at a time");
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds8[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    int slice, m0, n0;
    f8_tile(p, slice, m0, n0);
    m0 *= BM;
    n0 *= BN;
    const int wm = wave % WM * TM * 32, wn = wave / WM * TN * 32;
    const int first = slice * p.slice, nb = min(p.slice, p.blocks - first);

    // this wave's pieces of a stage: eight rows of 128 bytes each
    const bool tokens = wave * PIECES * 8 < BM;
    const int at = wave * PIECES * 8 - (tokens ? 0 : BM), last = (tokens ? p.M - m0 : p.N - n0) - 1;
    const uint8_t *base[PIECES / 4];   // of 32 rows each: what a lane adds to it stays within 32 bits
    int off[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int from = min(at + i / 4 * 32, last), r = at + i * 8 + lane / 8, row = tokens ? r : (r & ~31) + f8_deal(r & 31);
        if (i % 4 == 0) base[i / 4] = (tokens ? p.a + (int64_t)(m0 + from) * p.kp : p.b + (int64_t)(n0 + from) * p.kp) + (int64_t)first * kF8Block;
        off[i] = (min(row, last) - from) * (int)p.kp + (((lane % 8) ^ f8_swz(r)) << 4);
    }
    auto fetch = [&](int s) {
        unsigned char *to = lds8 + (s & 1) * STAGE + wave * PIECES * 1024;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) f8_dma(base[i / 4] + s * kF8Block, off[i], to + i * 1024);
    };
    const uint32_t *sbase = (tokens ? p.sa + (int64_t)m0 * p.sd : p.sb + (int64_t)n0 * p.sd) + first / 4;
    int soff;
    {
        const int r = at + lane % ROWS, row = tokens ? r : (r & ~31) + f8_deal(r & 31);
        soff = min(row, last) * p.sd * 4;
    }
    auto fetch_scales = [&](int s4) {   // of four stages
        if (lane < ROWS) f8_dma4(sbase + s4, soff, lds8 + SCALES + (s4 & 1) * (BM + BN) * 4 + ((tokens ? 0 : BM) + at) * 4);
    };
    int xs[TM], ws[TN];

    f32x16 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int u = 0; u < TM; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][u][r] = 0.0f;

    float *bias = reinterpret_cast<float *>(lds8 + BIAS);
    for (int i = threadIdx.x; i < BN; i += W * 64) bias[i] = p.bias && n0 + i < p.N ? load_as(p.bias, n0 + i, p.bias_dtype) : 0.0f;
    fetch_scales(0);
    fetch(0);
    for (int s4 = 0; s4 < nb; s4 += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (s4 + j >= nb) break;
            f8_sync();
            if (j == 0) {
                const int *x = reinterpret_cast<const int *>(lds8 + SCALES + ((s4 >> 2) & 1) * (BM + BN) * 4);
#pragma unroll
                for (int u = 0; u < TM; ++u) xs[u] = x[wm + 32 * u + li];
#pragma unroll
                for (int t = 0; t < TN; ++t) ws[t] = x[BM + wn + 32 * t + li];
                if (s4 + 4 < nb) fetch_scales(s4 / 4 + 1);
            }
            if (s4 + j + 1 < nb) fetch(s4 + j + 1);
            const unsigned char *buf = lds8 + (j & 1) * STAGE;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                i32x8f b[TN], a[TM];
                auto operand = [&](int row) {
                    const i32x4f lo = *reinterpret_cast<const i32x4f *>(buf + f8_at(row, 4 * ks + 2 * g)),
                                 hi = *reinterpret_cast<const i32x4f *>(buf + f8_at(row, 4 * ks + 2 * g + 1));
                    return i32x8f{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                };
#pragma unroll
                for (int t = 0; t < TN; ++t) b[t] = operand(BM + wn + 32 * t + li);
#pragma unroll
                for (int u = 0; u < TM; ++u) a[u] = operand(wm + 32 * u + li);
                if constexpr (WIDE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bf16x8 bw[TN], aw[TM];
#pragma unroll
                        for (int t = 0; t < TN; ++t) bw[t] = f8_widen(b[t][2 * i], b[t][2 * i + 1], f8_scale(ws[t], j));
#pragma unroll
                        for (int u = 0; u < TM; ++u) aw[u] = f8_widen(a[u][2 * i], a[u][2 * i + 1], f8_scale(xs[u], j));
#pragma unroll
                        for (int t = 0; t < TN; ++t)
#pragma unroll
                            for (int u = 0; u < TM; ++u) acc[t][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[t], aw[u], acc[t][u], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < TN; ++t)
#pragma unroll
                        for (int u = 0; u < TM; ++u)
                            acc[t][u] = j == 0 ? f8_mma<0>(b[t], a[u], acc[t][u], ws[t], xs[u]) : j == 1 ? f8_mma<1>(b[t], a[u], acc[t][u], ws[t], xs[u])
                                      : j == 2 ? f8_mma<2>(b[t], a[u], acc[t][u], ws[t], xs[u]) : f8_mma<3>(b[t], a[u], acc[t][u], ws[t], xs[u]);
                }
            }
        }
    }
    __syncthreads();
    f8_store_tile<TM, TN, T>(acc, p, lds8 + wave * kF8TileLds<TN, T>, bias, lane, m0, n0, wm, wn, slice);
}

struct F8Wide {   // 16 of a lane's values of a row as operands of two products
    bf16x8 k[2];
};

// The same for large products: tiles of 256 x 256, eight waves of 128 x 64, 64 of the contraction at a time in a ring of four stages of 32 KB.
// The two waves of a SIMD take turns: between two barriers one of them reads its operands (and asks for a stage) while the other
// multiplies.  Waves 4 to 7 run one barrier behind waves 0 to 3.
//
// Step s: a wave reads stage s, asks for stage s + 3 into the place of stage s - 1, which the other half has read before the last barrier;
// barrier; eight products; barrier.  Stage s + 1 is first read by waves 0 to 3 after their step s: before that barrier every wave's loads of it
// have landed.  That is the end of step s for waves 0 to 3 and the middle of it for waves 4 to 7, when stages s + 2 and s + 3 are still under way.
//
// 8192 x 4096 x 4096 in 111 to 114 us, 2480 TFLOP/s (128 x 128: 139; 124 on another card), 8192^3 in 417 to 528 by card, 2640 to 2080.  Two bounds share the rest: power (with operands of
// zeros 391 us instead of 528 on one card) and the loads (without them 407 of those 528, 301 of the 391; without LDS reads as well 385 and 292).  The matrix cores are busy for 0.59 to 0.61 of
// the cycles.  9 loads of 10 find L2: 1.07 GB for 8192 x 4096 x 4096, 9.7 TB/s of requests of 64 bytes, some 400 cycles each; 99 MB come from past it, 50 are needed.  fp32 results (WIDE): 224 us,
// 1230 TFLOP/s, the rate of the library's bf16 product (216); widened in one piece before the products instead of by halves 285.  Four waves of 128 x 128 over several tiles in
// turn, with the next tile's loads under the last one's stores: 528 and, for short contractions, 36 us instead of 32.  Loads asked for between the products: no change.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(512, 2) fp8_matmul_big(F8Matmul p) {
    constexpr int W = 8, TM = 4, TN = 2, BM = 256, BN = 256, STAGE = (BM + BN) * 64, RING = 4, PIECES = 4;
    constexpr int SCALES = RING * STAGE, BIAS = SCALES + 2 * (BM + BN) * 4;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds8[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    int slice, m0, n0;
    f8_tile(p, slice, m0, n0);
    m0 *= BM;
    n0 *= BN;
    const bool late = wave >= 4;
    const int wm = (wave & 1) * 128, wn = (wave >> 1) * 64;
    const int first = slice * p.slice, nb = min(p.slice, p.blocks - first), ns = 2 * nb;

    // this wave's pieces of a stage, 16 rows of 64 bytes each: rows of a from waves 0, 2, 4, 6, of b from the others
    const bool tokens = (wave & 1) == 0;
    const int at = (wave >> 1) * 64, last = (tokens ? p.M - m0 : p.N - n0) - 1;
    const uint8_t *base[PIECES / 2];   // of 32 rows each, as above
    const uint32_t *sbase = (tokens ? p.sa + (int64_t)m0 * p.sd : p.sb + (int64_t)n0 * p.sd) + first / 4;
    int off[PIECES], soff;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int from = min(at + i / 2 * 32, last), r = at + i * 16 + lane / 4, row = tokens ? r : (r & ~31) + f8_deal(r & 31);
        if (i % 2 == 0) base[i / 2] = (tokens ? p.a + (int64_t)(m0 + from) * p.kp : p.b + (int64_t)(n0 + from) * p.kp) + (int64_t)first * kF8Block;
        off[i] = (min(row, last) - from) * (int)p.kp + (((lane % 4) ^ ((r >> 2) & 3)) << 4);
    }
    {
        const int r = at + lane, row = tokens ? r : (r & ~31) + f8_deal(r & 31);
        soff = min(row, last) * p.sd * 4;
    }
    unsigned char *to = lds8 + (tokens ? 0 : BM * 64) + at * 64;
    auto fetch = [&](int s) {
        unsigned char *dst = to + (s & 3) * STAGE;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) f8_dma(base[i / 2] + s * 64, off[i], dst + i * 1024);
    };
    auto fetch_scales = [&](int s8) {   // of steps 8 s8 .. 8 s8 + 7
        f8_dma4(sbase + s8, soff, lds8 + SCALES + (s8 & 1) * (BM + BN) * 4 + ((tokens ? 0 : BM) + at) * 4);
    };

    f32x16 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int u = 0; u < TM; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][u][r] = 0.0f;

    float *bias = reinterpret_cast<float *>(lds8 + BIAS);
    if (threadIdx.x < BN) bias[threadIdx.x] = p.bias && n0 + (int)threadIdx.x < p.N ? load_as(p.bias, n0 + threadIdx.x, p.bias_dtype) : 0.0f;
    fetch_scales(0);
    fetch(0);
    fetch(1);                          // (two steps at least)
    if (ns > 2) fetch(2);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (late) asm volatile("s_barrier" ::: "memory");

    const int rs = (li >> 2) & 3;
    const unsigned char *ap = lds8 + (wm + li) * 64, *bp = lds8 + BM * 64 + (wn + li) * 64;
    const int c0 = ((2 * g) ^ rs) << 4, c1 = ((2 * g + 1) ^ rs) << 4;
    int xs[TM], ws[TN];
    auto steps = [&](auto half) {
        constexpr bool LATE = decltype(half)::value;
        for (int s8 = 0; s8 < ns; s8 += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int s = s8 + j;
                if (j % 2 == 0 && s >= ns) break;
                if (j == 0) {
                    const int *x = reinterpret_cast<const int *>(lds8 + SCALES + ((s8 >> 3) & 1) * (BM + BN) * 4);
#pragma unroll
                    for (int u = 0; u < TM; ++u) xs[u] = x[wm + 32 * u + li];
#pragma unroll
                    for (int t = 0; t < TN; ++t) ws[t] = x[BM + wn + 32 * t + li];
                    if (s8 + 8 < ns) fetch_scales(s8 / 8 + 1);
                }
                const int slot = (j & 3) * STAGE;
                // WIDE: half a stage at a time, widened before the barrier, while the other wave of the SIMD multiplies
                constexpr int PARTS = WIDE ? 2 : 1;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    constexpr bool ONCE = PARTS == 1;
                    const bool ends = part == PARTS - 1;
                    typename std::conditional<WIDE, F8Wide, i32x8f>::type b[TN], a[TM];
                    i32x4f lo[TN + TM], hi[TN + TM];
#pragma unroll
                    for (int i = 0; i < TN + TM; ++i) {
                        const unsigned char *row = (i < TN ? bp + i * 2048 : ap + (i - TN) * 2048) + slot;
                        lo[i] = *reinterpret_cast<const i32x4f *>(row + (part == 0 ? c0 : c1));
                        if (ONCE) hi[i] = *reinterpret_cast<const i32x4f *>(row + c1);
                    }
#pragma unroll
                    for (int i = 0; i < TN + TM; ++i) {
                        auto &to_ = i < TN ? b[i] : a[i - TN];
                        if constexpr (ONCE) {
                            to_ = i32x8f{lo[i][0], lo[i][1], lo[i][2], lo[i][3], hi[i][0], hi[i][1], hi[i][2], hi[i][3]};
                        } else {
                            const float f = f8_scale(i < TN ? ws[i] : xs[i - TN], j / 2);
                            to_.k[0] = f8_widen(lo[i][0], lo[i][1], f);
                            to_.k[1] = f8_widen(lo[i][2], lo[i][3], f);
                            asm volatile("" : "+v"(to_.k[0]), "+v"(to_.k[1]));   // here, not where they are wanted
                        }
                    }
                    // stage s + 1 has landed where stages s + 2 and s + 3, four loads each, may be under way; the last stages are waited for altogether
                    if (part == 0 && s + 3 < ns) fetch(s + 3);
                    if (LATE && ends) {
                        if (s + 3 < ns) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier\n\ts_setprio 1" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (WIDE) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int t = 0; t < TN; ++t)
#pragma unroll
                                for (int u = 0; u < TM; ++u) acc[t][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[t].k[i], a[u].k[i], acc[t][u], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int t = 0; t < TN; ++t)
#pragma unroll
                            for (int u = 0; u < TM; ++u)
                                acc[t][u] = j / 2 == 0 ? f8_mma<0>(b[t], a[u], acc[t][u], ws[t], xs[u]) : j / 2 == 1 ? f8_mma<1>(b[t], a[u], acc[t][u], ws[t], xs[u])
                                          : j / 2 == 2 ? f8_mma<2>(b[t], a[u], acc[t][u], ws[t], xs[u]) : f8_mma<3>(b[t], a[u], acc[t][u], ws[t], xs[u]);
                    }
#pragma unroll
                    for (int t = 0; t < TN; ++t)   // the products stay between the barriers
#pragma unroll
                        for (int u = 0; u < TM; ++u) asm volatile("" : "+v"(acc[t][u]));
                    __builtin_amdgcn_sched_barrier(0);
                    if (LATE || !ends) asm volatile("s_setprio 0\n\ts_barrier" ::: "memory");
                    else if (s + 3 < ns) asm volatile("s_setprio 0\n\ts_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
                    else asm volatile("s_setprio 0\n\ts_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
                }
            }
        }
    };
    if (late) steps(std::true_type());
    else steps(std::false_type());
    if (!late) asm volatile("s_barrier" ::: "memory");
    __syncthreads();
    f8_store_tile<TM, TN, T>(acc, p, lds8 + wave * kF8TileLds<TN, T>, bias, lane, m0, n0, wm, wn, slice);
}

// ---- a contraction of up to four blocks ----

// What such products cost is their results, and how soon one tile's are on their way after the last one's.  A workgroup stays on a strip of 128 rows of a, 32 in the
// registers of each wave, as operands, and takes a piece of b's rows in tiles of 64: the next tile is on its way to LDS while this one is multiplied and stored.  ROUND: the
// strip comes as it is and is rounded on the way, once for all tiles.  The sums are those of the other kernels, product for product.
// 32 768 x 1024 x 256 with its rounding 20.1 us (84 MB, 4.2 TB/s; rounding kernel and tiles of 128 x 128 29.3), from a rounded matrix 19.6 (22.7); 131 072 rows 65.7 (103).
// The results go out through the place of the tile that has been read: with one of their own, half as many workgroups fit and 65 536 x 512 x 512 takes 47.8 us instead of 32.0.
// Rows to be rounded are read by the lanes that hold them as operands: neighbouring lanes along a row, turned in LDS, take longer (100 x 1024 x 256 6.4 instead of
// 5.6 us, 32 768 rows 21.3 instead of 20.1); rounded rows, of half the bytes or less, a shorter one (8192 x 1024 x 512 with the rounding
// kernel 17.2 by the lanes that hold them, 15.4 turned).
template <typename T, int NB, bool ROUND>
__global__ void __launch_bounds__(256, 2) fp8_strip(F8Matmul p) {
    constexpr bool WIDE = sizeof(T) == 4;
    constexpr int TN = 2, BM = 128, BN = 64;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds8[];
    __shared__ float bias[4][BN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, g = lane >> 5;
    const unsigned lid = xcd_remap(blockIdx.x, gridDim.x);   // pieces of a strip side by side
    const int m0 = (int)(lid / p.pieces) * BM, first = (int)(lid % p.pieces) * p.tiles, end = min(first + p.tiles, p.nt);
    // A tile of b in LDS: four parts of 16 rows, [block][row]; each wave fetches one, and takes its place, when all have read it, for its results' way out.
    const int part = max(p.blocks * 2048, kF8TileLds<TN, T>);

    // this wave's rows: two pieces of eight for each block
    int row[2], at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = wave * 16 + i * 8 + lane / 8;
        row[i] = (r & ~31) + f8_deal(r & 31);
        at[i] = ((lane % 8) ^ f8_swz(r)) << 4;
    }
    auto fetch = [&](int tile) {
        const uint8_t *base = p.b + (int64_t)tile * BN * p.kp;
        unsigned char *to = lds8 + ((tile & 1) * 4 + wave) * part;
        const int last = p.N - tile * BN - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int off = min(row[i], last) * (int)p.kp + at[i];
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (b < p.blocks) f8_dma(base + b * kF8Block, off, to + b * 2048 + i * 1024);
        }
    };
    int ws[TN], wn[TN];
    float next = 0.0f;
    auto ask = [&](int tile) {   // its scales and this thread's number of its bias
#pragma unroll
        for (int t = 0; t < TN; ++t) wn[t] = (int)p.sb[(int64_t)min(tile * BN + 32 * t + f8_deal(li), p.N - 1) * p.sd];
        const int n = tile * BN + (int)threadIdx.x;
        if (threadIdx.x < BN && p.bias) next = n < p.N ? load_as(p.bias, n, p.bias_dtype) : 0.0f;
    };
    auto take = [&](int tile) {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            asm volatile("" : "+v"(wn[t]));
            ws[t] = wn[t];
        }
        if (threadIdx.x < BN) bias[tile & 3][threadIdx.x] = next;
    };

    ask(first);
    fetch(first);
    const int mw = m0 + wave * 32;
    i32x8f a[2 * NB];
    int xs = 0;
    if constexpr (ROUND) {
        const T *x = (const T *)p.x + (int64_t)min(mw + li, p.M - 1) * p.ldx + 32 * g;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b >= p.blocks) break;
            F8Eight<T> e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = b * kF8Block + 64 * (i / 4) + 8 * (i % 4), left = p.k - c - 32 * g;
                if (left >= 8) {
                    e[i].load(x + c);
                } else {
#pragma unroll
                    for (int w = 0; w < 8; ++w) e[i].v[w] = w < left ? x[c + w] : (T)0.0f;
                }
            }
            const unsigned most = f8_largest(e);
            const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
            const int ex = f8_exponent(max(both[0], both[1]));
            const float scale = f8_power(ex);
            xs |= (ex + 127) << (8 * b);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const auto &v = e[i / 2].v;
                const int c = i % 2 * 4;
                a[2 * b + i / 8][i % 8] = f8_pack<T>(v[c], v[c + 1], v[c + 2], v[c + 3], scale);
            }
        }
    } else {
        // The wave's rows come by neighbouring lanes, and a block at a time through its part of the other tile's place.
        unsigned char *mine = lds8 + (((first + 1) & 1) * 4 + wave) * part;
        xs = (int)p.sa[(int64_t)min(mw + li, p.M - 1) * p.sd];
        i32x4f e[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (b < p.blocks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) e[b][i] = *reinterpret_cast<const i32x4f *>(p.a + (int64_t)min(mw + 8 * i + lane / 8, p.M - 1) * p.kp + b * kF8Block + lane % 8 * 16);
            }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b >= p.blocks) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<i32x4f *>(mine + f8_at(8 * i + lane / 8, lane % 8)) = e[b][i];
            f8_wave_sync();
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const i32x4f lo = *reinterpret_cast<const i32x4f *>(mine + f8_at(li, 4 * ks + 2 * g)),
                             hi = *reinterpret_cast<const i32x4f *>(mine + f8_at(li, 4 * ks + 2 * g + 1));
                a[2 * b + ks] = i32x8f{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
            f8_wave_sync();
        }
    }
    take(first);
    f8_sync();

    for (int tile = first; tile < end; ++tile) {
        const bool more = tile + 1 < end;
        if (more) {
            ask(tile + 1);
            fetch(tile + 1);
        }
        f32x16 acc[TN][1];
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][0][r] = 0.0f;
        unsigned char *buf = lds8 + (tile & 1) * 4 * part;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b >= p.blocks) break;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    const unsigned char *from = buf + (2 * t + li / 16) * part + b * 2048;
                    const i32x4f lo = *reinterpret_cast<const i32x4f *>(from + f8_at(li % 16, 4 * ks + 2 * g)),
                                 hi = *reinterpret_cast<const i32x4f *>(from + f8_at(li % 16, 4 * ks + 2 * g + 1));
                    const i32x8f w = i32x8f{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    const i32x8f &v = a[2 * b + ks];
                    if constexpr (WIDE) {
                        const float wf = f8_scale(ws[t], b), xf = f8_scale(xs, b);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[t][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_widen(w[2 * i], w[2 * i + 1], wf), f8_widen(v[2 * i], v[2 * i + 1], xf), acc[t][0], 0, 0, 0);
                    } else {
                        acc[t][0] = b == 0 ? f8_mma<0>(w, v, acc[t][0], ws[t], xs) : b == 1 ? f8_mma<1>(w, v, acc[t][0], ws[t], xs)
                                  : b == 2 ? f8_mma<2>(w, v, acc[t][0], ws[t], xs) : f8_mma<3>(w, v, acc[t][0], ws[t], xs);
                    }
                }
            }
        }
        // the next tile has landed, the results of the one before are out, and everybody has read this one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (more) take(tile + 1);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        f8_store_tile<1, TN, T>(acc, p, buf + wave * part, bias[tile & 3], lane, m0, tile * BN, wave * 32, 0, 0);
    }
}

// The slices' sums, eight columns per thread, in their order, and column sums that are asked for with them.  16 slices of 1024 x 256: 5 us, a launch and the way to memory;
// the column sums in one of their own 4 more.
struct F8Sums {   // the column sums' parts and where their totals go, if there are any
    const float *part;
    void *out;
    int64_t parts;
    int cols, dtype;
    unsigned first;   // the first workgroup that adds them up
};
template <typename T>
__global__ void __launch_bounds__(256) fp8_slices(const float *part, T *out, const void *bias, int bias_dtype, int64_t M, int N, int64_t ldo, int slices, F8Sums c) {
    if (c.part && blockIdx.x >= c.first) {
        sum_parts<8>(c.part, c.out, c.cols, c.parts, c.dtype, blockIdx.x - c.first);
        return;
    }
    const int pieces = (N + 7) / 8;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / pieces;
    const int o = (int)(id % pieces) * 8;
    if (m >= M) return;
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.0f;
    const float *x = part + m * N + o;
    if (o + 8 <= N) {
#pragma unroll 4
        for (int k = 0; k < slices; ++k) {
            float v[8];
            __builtin_memcpy(v, x + (int64_t)k * M * N, sizeof v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += v[i];
        }
    } else {
        for (int k = 0; k < slices; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (o + i < N) s[i] += x[(int64_t)k * M * N + i];
    }
    F8Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = (T)(bias && o + i < N ? s[i] + load_as(bias, o + i, bias_dtype) : s[i]);
    e.store_some(out + m * ldo + o, N - o);
}

// ---- few rows ----

// Up to 64 rows, rounded on the way: the weight's rows are read once, straight into operands, and what there is to multiply is hidden behind that; one launch where a
// rounding pass and a product of tiles take two or three.  A workgroup takes 16 NT rows of b (outputs) and all rows of x, for a slice of the contraction; its
// waves take turns at the slice's blocks and add up through LDS.  v_mfma_scale_f32_16x16x128: one product per block and 16 rows of either side (lane l, q = l / 16: row
// l % 16, of a block's 128 values 16 q .. 16 q + 15 and 64 + 16 q ..; results of row l % 16 of x, outputs 4 q .. 4 q + 3).  The rows of x are rounded by every
// workgroup again, a block's 32 values of a lane and its three neighbours' at a time.  Bound by the way of one launch where the weight is small (one token through
// 1024 x 256 4.5 us; rounding, product and sums of slices took 10), by memory where it is large (1 x 8192 x 8192 18 us, 3.7 TB/s; 24 x 8192 x 8192 24.6).
struct F8Few {
    const void *x;               // [M][k], rows ldx apart
    const uint8_t *b;
    const uint32_t *sb;
    const void *bias;
    void *out;                   // [slices][M][N] where there are several slices
    int64_t ldx, ldo, kp;
    int M, N, k, blocks, slice, sd, bias_dtype;
};
constexpr int kF8FewRows = 64, kF8FewWaves = 8;

template <typename T, typename O, int MT, int NT, int U>   // U: blocks under way at a time
__global__ void __launch_bounds__(kF8FewWaves * 64) fp8_few(F8Few p) {
    constexpr bool WIDE = sizeof(T) == 4;
    __shared__ f32x4 sums[kF8FewWaves / 2][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, li = lane & 15, q = lane >> 4;
    const int tiles = (p.N + 16 * NT - 1) / (16 * NT), slice = blockIdx.x / tiles, n0 = blockIdx.x % tiles * (16 * NT);
    const int begin = slice * p.slice, end = min(begin + p.slice, p.blocks);
    const uint8_t *b[NT];
    const uint32_t *sb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t row = min(n0 + 16 * t + li, p.N - 1);
        b[t] = p.b + row * p.kp + q * 16;
        sb[t] = p.sb + row * p.sd;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int first = begin + wave; first < end; first += waves * U) {
        i32x8f bo[U][NT];
        int bs[U][NT];
        F8Eight<T> e[U][MT][4];
#pragma unroll
        for (int j = 0; j < U; ++j) {   // (blocks beyond the last repeat it; they are not multiplied)
            const int k = min(first + j * waves, end - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint8_t *from = b[t] + (int64_t)k * kF8Block;
                const i32x4f lo = *reinterpret_cast<const i32x4f *>(from), hi = *reinterpret_cast<const i32x4f *>(from + 64);
                bo[j][t] = i32x8f{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                bs[j][t] = (int)(sb[t][k >> 2] >> (8 * (k & 3)));
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int k = min(first + j * waves, end - 1), c = k * kF8Block + q * 16;
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                const T *x = (const T *)p.x + min(16 * u + li, p.M - 1) * p.ldx + c;
                if ((k + 1) * kF8Block <= p.k) {   // uniform
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[j][u][i].load(x + 64 * (i / 2) + 8 * (i % 2));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int w = 64 * (i / 16) + i % 16;
                        e[j][u][i / 8].v[i % 8] = c + w < p.k ? x[w] : (T)0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (first + j * waves >= end) break;
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                const int ex = f8_exponent(f8_max_rows(f8_largest(e[j][u])));
                const float scale = f8_power(ex);
                i32x8f ao;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const auto &v = e[j][u][i / 2].v;
                    const int c = i % 2 * 4;
                    ao[i] = f8_pack<T>(v[c], v[c + 1], v[c + 2], v[c + 3], scale);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if constexpr (WIDE) {
                        const float as = f8_scale(ex + 127, 0), ws = f8_scale(bs[j][t], 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f8_widen(bo[j][t][2 * i], bo[j][t][2 * i + 1], ws), f8_widen(ao[2 * i], ao[2 * i + 1], as),
                                                                                acc[t][u], 0, 0, 0);
                    } else {
                        acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bo[j][t], ao, acc[t][u], 0, 0, 0, bs[j][t], 0, ex + 127);
                    }
                }
            }
        }
    }
    // the upper half of the waves to the lower, then all four
    constexpr int HALF = kF8FewWaves / 2;
    if (wave >= HALF) {
#pragma unroll
        for (int i = 0; i < NT * MT; ++i) sums[wave - HALF][i][lane] = acc[i / MT][i % MT];
    }
    __syncthreads();
    if (wave < HALF) {
#pragma unroll
        for (int i = 0; i < NT * MT; ++i) {
            f32x4 s = acc[i / MT][i % MT];
            if (wave + HALF < waves) s += sums[wave][i][lane];
            sums[wave][i][lane] = s;
        }
    }
    __syncthreads();
    O *out = (O *)p.out + (int64_t)slice * p.M * p.N;
    for (int i = wave; i < NT * MT; i += waves) {
        f32x4 s = sums[0][i][lane];
        for (int w = 1; w < min(waves, HALF); ++w) s += sums[w][i][lane];
        const int m = 16 * (i % MT) + li, o = n0 + 16 * (i / MT) + 4 * q;
        if (m < p.M) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (o + r < p.N) out[m * p.ldo + o + r] = (O)(s[r] + (p.bias ? load_as(p.bias, o + r, p.bias_dtype) : 0.0f));
        }
    }
}

static bool f8_off(const void *p, int n) { return ((uintptr_t)p & (n - 1)) != 0; }

constexpr int kF8StripBlocks = 4, kF8SumsParts = 1024;   // (of more parts a launch of its own, of four times the threads)
constexpr int64_t kF8MaxK = 1 << 26;   // of the contraction: 32 rows stay within 32-bit offsets

// How a product is cut.  Up to four blocks: strips.  Tiles of 256 x 256 where there is one for each unit, else of 128 x 128 (us, 128 / 256: 8192 x 2048 x 2048, 256 large tiles,
// 41.2 / 35.0, 4096^3 75.6 / 58.2, 8192 x 4096 x 1024 43.2 / 41.0; 8192 x 1024 x 1024, 128 of them, 15.5 / 19.3, 4096 x 2048 x 2048 22.5 / 43.6).  And into slices of
// the contraction where there are fewer tiles than units, one workgroup to each, of eight blocks at least (us, for 512 / 256 workgroups: 1024 x 256 x 32 768
// 27.3 / 25.5, 1024 x 1024 x 8192 28.7 / 25.6, 300 x 700 x 33 000 in fp32 42.8 / 39.6, 512 x 512 x 65 536 35.1 / 37.0).
struct F8Plan {
    int mt, nt, slice, slices;
    bool big, strip;
};
static F8Plan f8_plan(int64_t m, int64_t n, int64_t k) {
    F8Plan q{};
    const int blocks = (int)((k + kF8Block - 1) / kF8Block);
    q.strip = blocks <= kF8StripBlocks;
    q.big = !q.strip && ((m + 255) / 256) * ((n + 255) / 256) >= 256;
    const int side = q.big ? 256 : 128;
    q.mt = (int)((m + side - 1) / side);
    q.nt = (int)((n + side - 1) / side);
    const int64_t tiles = (int64_t)q.mt * q.nt;
    int64_t want = tiles >= 256 ? 1 : 256 / tiles;
    if (want > blocks / 8) want = blocks / 8;
    if (want < 1) want = 1;
    q.slice = (int)((blocks + want - 1) / want + 3) / 4 * 4;
    q.slices = (blocks + q.slice - 1) / q.slice;
    if (q.slices == 1) q.slice = blocks;
    return q;
}

static int f8_check(const EvoFp8Matmul *p) {
    if (!p || p->m <= 0 || p->n <= 0 || p->k <= 0 || !known_dtype(p->dtype)) return EVO_EINVAL;
    if (p->m > INT32_MAX - 512 || p->n > INT32_MAX - 512) return EVO_EOVERFLOW;
    if (p->k > kF8MaxK) return EVO_EUNSUPPORTED;
    const F8Plan q = f8_plan(p->m, p->n, p->k);
    if ((int64_t)q.mt * q.nt > INT32_MAX || (int64_t)q.mt * q.nt * q.slices > INT32_MAX) return EVO_EOVERFLOW;
    return EVO_OK;
}

constexpr int kF8QuantizeFew = 512;   // tiles
static int f8_rounding_check(const void *x, int64_t ldx, const void *q, const void *scales, const void *qt, const void *scales_t, const float *sums, int64_t rows,
                             int64_t cols, int dtype) {
    if (!x || rows <= 0 || cols <= 0 || ldx < cols || !known_dtype(dtype) || !q != !scales || !qt != !scales_t || (!q && !qt) || (sums && !qt)) return EVO_EINVAL;
    if (cols > kF8MaxK || (qt && rows > ((int64_t)1 << 40))) return EVO_EUNSUPPORTED;
    return f8_off(q, 16) || f8_off(qt, 16) ? EVO_EALIGN : EVO_OK;
}
static F8Quantize f8_rounding(const void *x, int64_t ldx, void *q, void *scales, void *qt, void *scales_t, float *sums, int64_t rows, int64_t cols) {
    F8Quantize p{};
    p.x = x;
    p.ldx = ldx;
    p.rows = rows;
    p.cols = (int)cols;
    p.kp = f8_pitch(cols);
    p.sp = (int)f8_scale_pitch(cols);
    p.tiles_k = (int)(p.kp / kF8Block);
    p.rp = f8_pitch(rows);
    p.spt = f8_scale_pitch(rows);
    p.tiles_r = p.rp / kF8Block;
    p.q = (uint8_t *)q;
    p.s = (uint8_t *)scales;
    p.qt = (uint8_t *)qt;
    p.st = (uint8_t *)scales_t;
    p.sums = sums;
    return p;
}
static F8Matmul f8_operands(const EvoFp8Matmul &p) {
    F8Matmul a{};
    a.a = (const uint8_t *)p.a;
    a.b = (const uint8_t *)p.b;
    a.sa = (const uint32_t *)p.scales_a;
    a.sb = (const uint32_t *)p.scales_b;
    a.bias = p.bias;
    a.out = p.out;
    a.ldo = p.ldo;
    a.k = (int)p.k;
    a.kp = f8_pitch(p.k);
    a.M = (int)p.m;
    a.N = (int)p.n;
    a.blocks = (int)(a.kp / kF8Block);
    a.sd = (int)(f8_scale_pitch(p.k) / 4);
    a.bias_dtype = p.bias_dtype;
    return a;
}

template <int WM, int WN, int TM, int TN, typename T, bool WIDE>
static int f8_launch_tiles(const F8Matmul &a, unsigned grid, hipStream_t st) {
    constexpr int side = 32 * (WM * TM + WN * TN), lds = 2 * side * 128 + 2 * side * 4 + 32 * WN * TN * 4;
    constexpr auto kernel = fp8_matmul<WM, WN, TM, TN, T, WIDE>;
    static PerDevice done;
    if (const int rc = ensure_dynamic_lds((const void *)kernel, lds, done, nullptr)) return rc;
    kernel<<<grid, WM * WN * 64, lds, st>>>(a);
    return hip_rc();
}
template <typename T, bool WIDE>
static int f8_launch(const F8Matmul &a, const F8Plan &q, hipStream_t st) {
    if (q.strip) return f8_launch_strip<T, false>(a, st);
    if (!grid_fits((int64_t)q.mt * q.nt * q.slices, 512)) return EVO_EOVERFLOW;
    const unsigned grid = (unsigned)(q.mt * q.nt * q.slices);
    if (q.big) {
        constexpr int lds = 4 * 512 * 64 + 2 * 512 * 4 + 256 * 4;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)fp8_matmul_big<T, WIDE>, lds, done, nullptr)) return rc;
        fp8_matmul_big<T, WIDE><<<grid, 512, lds, st>>>(a);
        return hip_rc();
    }
    return f8_launch_tiles<4, 2, 1, 2, T, WIDE>(a, grid, st);
}

// Strips of 128 rows, their columns in pieces for two workgroups on each unit (one: 32 768 x 1024 x 256 27.3 us instead of 20.1, 8192 x 4096 x 256 26.1 instead of 20.8).
constexpr int kF8StripGroups = 512;
struct F8StripPlan {
    int strips, tiles, pieces;
};
static F8StripPlan f8_strip_plan(int64_t m, int64_t n) {
    F8StripPlan q{};
    q.strips = (int)((m + 127) / 128);
    const int nt = (int)((n + 63) / 64), want = std::min((kF8StripGroups + q.strips - 1) / q.strips, nt);
    q.tiles = (nt + want - 1) / want;
    q.pieces = (nt + q.tiles - 1) / q.tiles;
    return q;
}
// Whether a strip is rounded by its workgroups.  Up to two blocks: always (us, on the way / before, in bf16: 1000 x 1024 x 256 6.5 / 11.0, 4096 x 1024 x 256 in 16 pieces 8.9 /
// 10.9, 17 000 x 700 x 256 15.6 / 16.4, 33 000 x 333 x 256 16.4 / 20.5; 12 000 x 384 x 256 11.4 / 11.1; in fp32 it takes up to a third longer where there are many pieces, 4096 x 1024 x 256
// 15.8 / 12.2, and as long for one or two).  More, which fp32 has no registers for: where a strip is one piece, or up to six are all under way at once, two workgroups to a unit (one piece: 65 536 x
// 512 x 512 30.6 / 42.2, 100 000 x 1024 x 384 75 / 92; at once: 16 384 x 768 x 384, 512 workgroups, 15.6 / 17.7, 11 000 x 320 x 384, 430 in five pieces, 10.6 / 11.2); with a second
// round of them, or more pieces, before (17 000 x 700 x 300, 532 workgroups, 24.4 / 19.5, 13 312 x 1280 x 384 in five pieces 26.0 / 20.2, 22 000 x 1536 x 300 in three 39.0 / 30.9; 8192 x 1024 x 512,
// 512 in eight, 16.4 / 15.2, 300 x 8192 x 512 12.6 / 9.1).
static bool f8_strip_rounds(int64_t m, int64_t n, int64_t k, int dtype) {
    if (k <= 2 * kF8Block) return true;
    if (k > kF8StripBlocks * kF8Block || dtype == EVO_F32) return false;
    const F8StripPlan q = f8_strip_plan(m, n);
    return q.pieces == 1 || (q.pieces <= 6 && q.strips * q.pieces <= kF8StripGroups);
}
template <typename T, bool ROUND>
static int f8_launch_strip(F8Matmul a, hipStream_t st) {
    const F8StripPlan q = f8_strip_plan(a.M, a.N);
    a.nt = (a.N + 63) / 64;
    a.tiles = q.tiles;
    a.pieces = q.pieces;
    auto go = [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        auto lds = [](int blocks) { return 8 * std::max(blocks * 2048, kF8TileLds<2, T>); };
        constexpr auto kernel = fp8_strip<T, NB, ROUND>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kernel, lds(NB), done, nullptr)) return rc;
        kernel<<<(unsigned)(q.strips * q.pieces), 256, lds(a.blocks), st>>>(a);
        return hip_rc();
    };
    if (a.blocks == 1) return go(std::integral_constant<int, 1>());
    if (a.blocks == 2) return go(std::integral_constant<int, 2>());
    if constexpr (ROUND && sizeof(T) == 4) return EVO_EUNSUPPORTED;
    else return go(std::integral_constant<int, kF8StripBlocks>());
}

// Few rows: 64 outputs to a workgroup where there are then enough of them for the chip, or slices of the contraction to make up for it, else 16; of a block at least for each
// wave.  us, 16 / 64 outputs: 24 x 4096 x 4096 14.4 / 12.1 (1 row 8.9 / 9.8), 24 x 8192 x 8192 49 / 25, 48 x 500 x 8000 24.4 / 19.1; 24 x 1024 x 256 4.7 / 6.6,
// 8 x 8192 x 1024 5.9 / 6.5.
struct F8FewPlan {
    int nt, slice, slices;
};
static F8FewPlan f8_few_plan(int64_t n, int64_t k) {
    const int blocks = (int)((k + kF8Block - 1) / kF8Block), most = blocks < kF8FewWaves ? 1 : blocks / kF8FewWaves;
    F8FewPlan q{};
    q.nt = n >= 256 && (most >= 4 || (n + 63) / 64 * most >= 256) ? 4 : 1;
    const int64_t groups = (n + 16 * q.nt - 1) / (16 * q.nt);
    int64_t want = (256 + groups - 1) / groups;
    if (want > most) want = most;
    q.slice = (int)((blocks + want - 1) / want);
    q.slices = (blocks + q.slice - 1) / q.slice;
    return q;
}
template <typename T, typename O>
static int f8_launch_few(const F8Few &a, const F8FewPlan &q, hipStream_t st) {
    const int64_t groups = ((int64_t)a.N + 16 * q.nt - 1) / (16 * q.nt) * q.slices;
    const unsigned grid = (unsigned)groups, threads = 64 * (q.slice < kF8FewWaves ? q.slice : kF8FewWaves);
    if (!grid_fits(groups, (int)threads)) return EVO_EOVERFLOW;
    auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        constexpr int MANY = sizeof(T) == 4 ? 1 : MT > 2 ? 2 : 4;
        if (q.nt == 4) fp8_few<T, O, MT, 4, 1><<<grid, threads, 0, st>>>(a);
        else if (q.slice <= kF8FewWaves) fp8_few<T, O, MT, 1, 1><<<grid, threads, 0, st>>>(a);
        else fp8_few<T, O, MT, 1, MANY><<<grid, threads, 0, st>>>(a);
        return hip_rc();
    };
    const int mt = (a.M + 15) / 16;
    return mt == 1 ? go(std::integral_constant<int, 1>()) : mt == 2 ? go(std::integral_constant<int, 2>()) : mt == 3 ? go(std::integral_constant<int, 3>())
                                                                                                          : go(std::integral_constant<int, 4>());
}
template <typename T>
static int f8_add_slices(const EvoFp8Matmul &p, int slices, F8Sums c, hipStream_t st) {
    const int64_t pieces = p.m * ((p.n + 7) / 8), groups = (pieces + 255) / 256, more = c.part ? (c.cols + 31) / 32 : 0;
    if (!grid_fits(groups + more, 256)) return EVO_EOVERFLOW;
    c.first = (unsigned)groups;
    fp8_slices<T><<<(unsigned)(groups + more), 256, 0, st>>>((const float *)p.workspace, (T *)p.out, p.bias, p.bias_dtype, p.m, (int)p.n, p.ldo, slices, c);
    return hip_rc();
}

}  // namespace evo

extern "C" {

int evoattn_fp8_quantize(const void *x, int64_t ldx, void *q, void *scales, void *qt, void *scales_t, float *sums, int64_t rows, int64_t cols, int32_t dtype,
                         void *hip_stream) {
    using namespace evo;
    if (const int rc = f8_rounding_check(x, ldx, q, scales, qt, scales_t, sums, rows, cols, dtype)) return rc;
    const F8Quantize p = f8_rounding(x, ldx, q, scales, qt, scales_t, sums, rows, cols);
    if (p.tiles_r > INT32_MAX / p.tiles_k || !grid_fits(p.tiles_r * p.tiles_k, 256)) return EVO_EOVERFLOW;
    const unsigned grid = (unsigned)(p.tiles_r * p.tiles_k);
    hipStream_t st = (hipStream_t)hip_stream;
    return by_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        // few tiles: more threads for each (us, more / fewer: 1024 x 256 both ways 5.5 / 5.8, 2048 x 4096 rows 6.9 / 7.5; 8192 x 8192 both ways 53.5 / 50.6)
        const bool few = p.tiles_r * p.tiles_k < kF8QuantizeFew;
        if (q && qt) few ? fp8_quantize<T, 128, 2, true, true><<<grid, 1024, 0, st>>>(p) : fp8_quantize<T, 128, 8, true, true><<<grid, 256, 0, st>>>(p);
        else if (!q) few ? fp8_quantize<T, 128, 2, false, true><<<grid, 1024, 0, st>>>(p) : fp8_quantize<T, 128, 8, false, true><<<grid, 256, 0, st>>>(p);
        else if (few) fp8_quantize<T, 16, 1, true, false><<<(unsigned)((rows + 15) / 16 * p.tiles_k), 256, 0, st>>>(p);
        else fp8_quantize<T, 128, 8, true, false><<<grid, 256, 0, st>>>(p);
        return hip_rc();
    });
}

int evoattn_fp8_quantize_two(const EvoFp8Rounding *a, const EvoFp8Rounding *b, int32_t dtype, void *hip_stream) {
    using namespace evo;
    if (!a || !b || !known_dtype(dtype)) return EVO_EINVAL;
    F8Two both{};
    int64_t tiles = 0;
    for (int i = 0; i < 2; ++i) {
        const EvoFp8Rounding &r = i ? *b : *a;
        if (const int rc = f8_rounding_check(r.x, r.ldx, r.q, r.scales, r.qt, r.scales_t, r.sums, r.rows, r.cols, dtype)) return rc;
        both.p[i] = f8_rounding(r.x, r.ldx, r.q, r.scales, r.qt, r.scales_t, r.sums, r.rows, r.cols);
        if (both.p[i].tiles_r > INT32_MAX / both.p[i].tiles_k) return EVO_EOVERFLOW;
        if (i == 0) both.first = (unsigned)(both.p[0].tiles_r * both.p[0].tiles_k);
        tiles += both.p[i].tiles_r * both.p[i].tiles_k;
    }
    if (!grid_fits(tiles, 256)) return EVO_EOVERFLOW;
    return by_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (tiles < kF8QuantizeFew) fp8_quantize_two<T, 2><<<(unsigned)tiles, 1024, 0, (hipStream_t)hip_stream>>>(both);
        else fp8_quantize_two<T, 8><<<(unsigned)tiles, 256, 0, (hipStream_t)hip_stream>>>(both);
        return hip_rc();
    });
}

int evoattn_fp8_column_sums(const float *sums, void *out, int64_t rows, int64_t cols, int32_t dtype, void *hip_stream) {
    using namespace evo;
    if (!sums || !out || rows <= 0 || cols <= 0 || !known_dtype(dtype)) return EVO_EINVAL;
    if (cols > kF8MaxK) return EVO_EUNSUPPORTED;
    return launch_sum_parts(sums, out, (int)cols, (rows + kF8Block - 1) / kF8Block, dtype, (hipStream_t)hip_stream);
}

size_t evoattn_fp8_matmul_workspace_bytes(const EvoFp8Matmul *p) {
    using namespace evo;
    if (f8_check(p)) return 0;
    const F8Plan q = f8_plan(p->m, p->n, p->k);
    return q.slices == 1 ? 0 : (size_t)q.slices * p->m * p->n * sizeof(float);
}

static int f8_matmul(const EvoFp8Matmul *p, const evo::F8Sums &c, void *hip_stream, bool *added) {
    using namespace evo;
    if (const int rc = f8_check(p)) return rc;
    if (!p->a || !p->b || !p->scales_a || !p->scales_b || !p->out || p->ldo < p->n || (p->bias && !known_dtype(p->bias_dtype))) return EVO_EINVAL;
    if (f8_off(p->a, 16) || f8_off(p->b, 16) || f8_off(p->scales_a, 4) || f8_off(p->scales_b, 4)) return EVO_EALIGN;
    const F8Plan q = f8_plan(p->m, p->n, p->k);
    if (q.slices > 1 && (!p->workspace || p->workspace_bytes < evoattn_fp8_matmul_workspace_bytes(p))) return EVO_EWORKSPACE;
    F8Matmul a = f8_operands(*p);
    if (q.slices > 1) {
        a.bias = nullptr;
        a.out = p->workspace;
        a.ldo = p->n;
    }
    a.mt = q.mt;
    a.nt = q.nt;
    a.slice = q.slice;
    hipStream_t st = (hipStream_t)hip_stream;
    const bool wide = p->dtype == EVO_F32;
    if (q.slices == 1) {
        return p->dtype == EVO_F32 ? f8_launch<float, true>(a, q, st) : p->dtype == EVO_BF16 ? f8_launch<bf16_t, false>(a, q, st) : f8_launch<f16_t, false>(a, q, st);
    }
    if (const int rc = wide ? f8_launch<float, true>(a, q, st) : f8_launch<float, false>(a, q, st)) return rc;
    *added = c.part != nullptr;
    return by_dtype(p->dtype, [&](auto t) { return f8_add_slices<decltype(t)>(*p, q.slices, c, st); });
}
int evoattn_fp8_matmul(const EvoFp8Matmul *p, void *hip_stream) {
    bool added;
    return f8_matmul(p, evo::F8Sums{}, hip_stream, &added);
}
int evoattn_fp8_matmul_sums(const EvoFp8Matmul *p, const float *sums, int64_t rows, void *out, int32_t dtype, void *hip_stream) {
    using namespace evo;
    if (const int rc = f8_check(p)) return rc;
    if (!sums || !out || rows <= 0 || !known_dtype(dtype)) return EVO_EINVAL;
    F8Sums c{};
    c.parts = (rows + kF8Block - 1) / kF8Block;
    if (c.parts <= kF8SumsParts) c.part = sums;
    c.out = out;
    c.cols = (int)p->m;
    c.dtype = dtype;
    bool added = false;
    const int rc = f8_matmul(p, c, hip_stream, &added);
    return rc || added ? rc : evoattn_fp8_column_sums(sums, out, rows, p->m, dtype, hip_stream);
}

int evoattn_fp8_matmul_rounds(const EvoFp8Matmul *p) {
    using namespace evo;
    return !f8_check(p) && (p->m <= kF8FewRows || f8_strip_rounds(p->m, p->n, p->k, p->dtype));
}
size_t evoattn_fp8_matmul_rounding_workspace_bytes(const EvoFp8Matmul *p) {
    using namespace evo;
    if (f8_check(p) || p->m > kF8FewRows) return 0;   // (strips need none)
    const F8FewPlan q = f8_few_plan(p->n, p->k);
    return q.slices == 1 ? 0 : (size_t)q.slices * p->m * p->n * sizeof(float);
}

int evoattn_fp8_matmul_rounding(const EvoFp8Matmul *p, const void *x, int64_t ldx, void *hip_stream) {
    using namespace evo;
    if (const int rc = f8_check(p)) return rc;
    const bool few = p->m <= kF8FewRows;
    if (!evoattn_fp8_matmul_rounds(p)) return EVO_EUNSUPPORTED;
    if (!x || ldx < p->k || !p->b || !p->scales_b || !p->out || p->ldo < p->n || (p->bias && !known_dtype(p->bias_dtype))) return EVO_EINVAL;
    if (f8_off(p->b, 16) || f8_off(p->scales_b, 4)) return EVO_EALIGN;
    hipStream_t st = (hipStream_t)hip_stream;
    if (!few) {
        F8Matmul a = f8_operands(*p);
        a.x = x;
        a.ldx = ldx;
        return by_dtype(p->dtype, [&](auto t) { return f8_launch_strip<decltype(t), true>(a, st); });
    }
    const F8FewPlan q = f8_few_plan(p->n, p->k);
    const bool cut = q.slices > 1;
    if (cut && (!p->workspace || p->workspace_bytes < evoattn_fp8_matmul_rounding_workspace_bytes(p))) return EVO_EWORKSPACE;
    F8Few a{};
    a.x = x;
    a.ldx = ldx;
    a.b = (const uint8_t *)p->b;
    a.sb = (const uint32_t *)p->scales_b;
    a.bias = cut ? nullptr : p->bias;
    a.out = cut ? p->workspace : p->out;
    a.ldo = cut ? p->n : p->ldo;
    a.kp = f8_pitch(p->k);
    a.M = (int)p->m;
    a.N = (int)p->n;
    a.k = (int)p->k;
    a.blocks = (int)(a.kp / kF8Block);
    a.slice = q.slice;
    a.sd = (int)(f8_scale_pitch(p->k) / 4);
    a.bias_dtype = p->bias_dtype;
    return by_dtype(p->dtype, [&](auto t) {
        typedef decltype(t) T;
        if (!cut) return f8_launch_few<T, T>(a, q, st);
        if (const int rc = f8_launch_few<T, float>(a, q, st)) return rc;
        return f8_add_slices<T>(*p, q.slices, F8Sums{}, st);
    });
}

}  // extern "C"
