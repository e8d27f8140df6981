// The learned relative position bias of the attention: a number per head and bucket of the distance between two residues,
//   out[b,h,i,j] = table[bucket(b,i,j), h] (+ pair[b,h,i,j]),  bucket = lut[clamp(pos_q[b,i] - pos_k[b,j], -R, R) + R],
// or the table's last row where i and j lie in different chains; and the table's gradient, the sum of the output's over the pairs of
// each bucket.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elements.h"
#include "kernels.h"

namespace evo {

constexpr int kRbWaves = 4;
constexpr int kRbMaxReach = 4096, kRbMaxRows = 256;
constexpr int kRbMost = INT32_MAX - 1024;      // queries, keys: what is counted up in steps of a workgroup's stays within 32 bits
constexpr int64_t kRbNear = (int64_t)1 << 30;   // positions in (-2^30, 2^30): differences fit in 32 bits

// V elements of T from any element's address on (global memory takes 16 bytes at any alignment).
template <typename T>
struct RbVec {
    static constexpr int V = 16 / sizeof(T);
    T e[V];
    __device__ __forceinline__ static RbVec load(const T *p) {
        RbVec r;
        __builtin_memcpy(&r, p, 16);
        return r;
    }
    __device__ __forceinline__ void store(T *p) const { __builtin_memcpy(p, this, 16); }
};

// Positions or chains of one side, of 4 or 8 bytes each.
struct RbIndex {
    const void *p;
    int64_t b;
    bool wide;
    __device__ __forceinline__ int64_t operator[](int64_t i) const { return wide ? ((const int64_t *)p)[b + i] : (int64_t)((const int32_t *)p)[b + i]; }
};

struct RbArgs {
    const void *pos_q, *pos_k, *chain_q, *chain_k;   // [B or 1, Nq], [B or 1, Nk]
    const uint8_t *lut;
    const void *table;
    int64_t pos_q_b, pos_k_b;     // from one batch to the next (0: the same)
    int64_t pair_b, pair_h, pair_row;
    int B, H, Nq, Nk, rows, reach, table_dtype;
    int lanes;            // forward: that a row takes, a power of two up to 64
    int strips, heads;    // pieces of a row (backward: and of the heads) that a workgroup each takes
    int chunk, chunks;    // rows of a workgroup
    bool wide;            // positions and chains of 8 bytes
    __device__ __forceinline__ RbIndex queries(const void *t, int b) const { return {t, b * pos_q_b, wide}; }
    __device__ __forceinline__ RbIndex keys(const void *t, int b) const { return {t, b * pos_k_b, wide}; }
};

__device__ __forceinline__ bool rb_near(int64_t p) { return p > -kRbNear && p < kRbNear; }

// The clipped distance from 0 on.  Positions near zero in 32 bits, any others in 64, where a difference may overflow.
__device__ __forceinline__ int rb_offset(int q, int k, int reach) { return min(max(q - k, -reach), reach) + reach; }
__device__ __forceinline__ int rb_offset(int64_t q, int64_t k, int reach) {
    const int64_t d = __builtin_elementwise_sub_sat(q, k);
    return (int)min(max(d, (int64_t)-reach), (int64_t)reach) + reach;
}

// Forward.  Bound by memory: the pair bias read and the result written once.  The head's numbers lie in LDS by clipped distance, so that an element costs one subtraction, a clip
// and a look-up; positions of a strip of keys stay in registers over a workgroup's rows.  4 x 32 x 1024^2 in fp32 with a pair bias 187 us (1.07 GB, 5.7 TB/s), 8 x 8 x 512^2 in bf16
// 19.8 (67 MB, 3.4 TB/s).  Distances in 32 bits where the positions allow it: in 64 an element takes five instructions more.
template <typename T, bool PAIR, bool CHAIN>
__global__ void __launch_bounds__(kRbWaves * 64) relative_bias_fwd(RbArgs a, const T *pair, T *out) {
    constexpr int V = RbVec<T>::V, U = 4;
    extern __shared__ float val[];   // [2 R + 1]: this head's number for each clipped distance
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned id = blockIdx.x;
    const int strip = id % a.strips;
    id /= a.strips;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int h = id % a.H, b = id / a.H;
    for (int o = threadIdx.x; o <= 2 * a.reach; o += kRbWaves * 64) {
        const int r = a.lut[o];
        val[o] = r < a.rows ? load_as(a.table, (int64_t)r * a.H + h, a.table_dtype) : 0.0f;
    }
    const float other = CHAIN ? load_as(a.table, (int64_t)(a.rows - 1) * a.H + h, a.table_dtype) : 0.0f;
    const RbIndex qs = a.queries(a.pos_q, b), ks = a.keys(a.pos_k, b), qc = a.queries(a.chain_q, b), kc = a.keys(a.chain_k, b);
    // The last lane of a row that is no whole number of pieces steps back: two lanes write the same values there.
    const int col = (strip * 64 + lane % a.lanes) * V, first = min(col, max(a.Nk - V, 0)), sub = lane / a.lanes, per = 64 / a.lanes;
    const bool mine = col < a.Nk;
    int64_t pk[V], ck[V];
    bool near = true;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t j = min(first + e, a.Nk - 1);
        pk[e] = ks[j];
        ck[e] = CHAIN ? kc[j] : 0;
        near = near && rb_near(pk[e]);
    }
    near = __all(near);
    __syncthreads();
    const int r0 = chunk * a.chunk, r1 = r0 + min(a.chunk, a.Nq - r0);
    const int64_t plane = ((int64_t)b * a.H + h) * a.Nq;
    const bool whole = a.Nk >= V;
    for (int base = r0 + wave * per * U; base < r1; base += kRbWaves * per * U) {
        RbVec<T> in[U];
        int64_t pq[U], cq[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(base + u * per + sub, r1 - 1);
            pq[u] = qs[i];
            cq[u] = CHAIN ? qc[i] : 0;
            if (PAIR && mine) {
                const T *p = pair + b * a.pair_b + h * a.pair_h + i * a.pair_row;
                if (whole) {
                    in[u] = RbVec<T>::load(p + first);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) in[u].e[e] = p[min(e, a.Nk - 1)];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * per + sub;
            int o[V];
            if (near && __all(rb_near(pq[u]))) {
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rb_offset((int)pq[u], (int)pk[e], a.reach);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rb_offset(pq[u], pk[e], a.reach);
            }
            RbVec<T> r;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float v = val[o[e]];
                if (CHAIN) v = ck[e] == cq[u] ? v : other;
                r.e[e] = (T)(PAIR ? v + (float)in[u].e[e] : v);
            }
            if (i < r1 && mine) {
                T *p = out + (plane + i) * a.Nk;
                if (whole) {
                    r.store(p + first);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < a.Nk) p[e] = r.e[e];
                }
            }
        }
    }
}

// Backward: the sums of dout over the pairs of each bucket, as products: buckets x pairs (one where a pair is of the bucket, else zero) times
// pairs x heads, on v_mfma_f32_16x16x32 (lane l, q = l / 16: operands' row or column l % 16, contraction 8q .. 8q + 7; accumulator column l % 16, rows
// 4q .. 4q + 3).  16-bit gradients are operands as they lie; fp32 ones, 2^24 times as large, as three bf16 parts, which hold all of their
// 24 bits (of one below 2^-110 as it is, the smaller parts run out of exponents: sums of gradients around 3e-36 were 1.6e-5 off).  A
// product with one is exact, and sums are fp32 in a fixed order.  Zero times an infinity is no number: a workgroup that ends with a
// sum that is not finite (2^24 times as large, in fp32: from 2^104 on) forms its sums again one by one, and so does one whose positions lie some 2^30 (less 4096) or more from its first query's.
// Such a workgroup takes 40 to 100 times as long (with infinities in all of them 2 x 8 x 251^2 in fp16 0.57 ms instead of 14 us, 4 x 32 x 1024^2 in fp32 11 ms instead of 0.11).
// Chains are names: a query's is compared with those of the workgroup's keys, one to a lane, in all of their bits, and a lane takes its pairs' from the answer.
// Bound by memory: 4 x 32 x 1024^2 in fp32 107 to 109 us (537 MB, 5.0 TB/s), after the forward's results have been written 141 to 148.  As many additions to sums in LDS: 681 us.  32 heads to a
// workgroup, whose buckets are then looked up once: 151 where this took 116.
constexpr int kRbKeys = 64, kRbHeads = 16;   // a workgroup's keys and heads

typedef float f32x4r __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4r rb_mma(bf16x8 a, bf16x8 b, f32x4r c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4r rb_mma(f16x8 a, f16x8 b, f32x4r c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

typedef uint32_t u32x4r __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2r __attribute__((ext_vector_type(2)));

// Eight gradients of a head, and their products.
template <typename T>
struct RbRow {
    typedef typename std::conditional<sizeof(T) == 4, bf16_t, T>::type O;   // operands' type
    typedef typename Mfma<O>::v8 v8;
    static constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
    static constexpr float UP = sizeof(T) == 4 ? 0x1p24f : 1.0f, DOWN = 1.0f / UP;   // what products are the sums' times
    static constexpr uint32_t ONE = std::is_same<O, f16_t>::value ? 0x3c00 : 0x3f80;
    T e[8];
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(e, p, sizeof e); }
    __device__ __forceinline__ void parts(v8 (&out)[PARTS]) const {
        if constexpr (PARTS == 1) {
            out[0] = __builtin_bit_cast(v8, e);
        } else {
            uint32_t x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(e[i] * UP);
#pragma unroll
            for (int k = 0; k < 3; ++k) {   // the upper halves, then what they leave
                u32x4r h;
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302);
                out[k] = __builtin_bit_cast(v8, h);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k < 2) x[i] = __float_as_uint(__uint_as_float(x[i]) - __uint_as_float(x[i] & 0xffff0000u));
            }
        }
    }
};

// min(x, 1) in both halves; not as the compiler would have it, two comparisons and two selections
__device__ __forceinline__ u16x2r rb_any_bits(u16x2r x) {
    u16x2r r;
    asm("v_pk_min_u16 %0, %1, %2" : "=v"(r) : "v"(x), "s"(0x00010001));
    return r;
}

// A position less the workgroup's first, in 32 bits; false where that is not within 2^30 less the largest reach, so that a query's less a key's, and the reach
// on top of it, fit in 32 bits as well.
__device__ __forceinline__ bool rb_from(int64_t p, int64_t base, int &d) {
    constexpr int64_t most = kRbNear - kRbMaxReach;
    int64_t w;
    const bool over = __builtin_sub_overflow(p, base, &w);
    d = (int)w;
    return !over && w > -most && w < most;
}

// Lanes of a workgroup's keys: group g of 32, a lane's eight from `first` on, of which the first `skip` are another lane's (or none).
template <int TILES, typename T, bool CHAIN>
__global__ void __launch_bounds__(kRbWaves * 64) relative_bias_bwd(RbArgs a, const T *dout, float *part, void *dtable) {
    typedef RbRow<T> Row;
    typedef typename Row::v8 v8;
    constexpr int G = kRbKeys / 32, U = 2;
    extern __shared__ float lds[];   // [waves - 1][TILES * 4][64] sums; uint16 [2 R + 2] buckets, the last one of pairs in different chains
    uint16_t *lut = reinterpret_cast<uint16_t *>(lds + (kRbWaves - 1) * TILES * 4 * 64);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, li = lane & 15;
    unsigned id = blockIdx.x;
    const int strip = id % a.strips;
    id /= a.strips;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int b = id % a.B, h0 = id / a.B * kRbHeads, j0 = strip * kRbKeys;
    const RbIndex qs = a.queries(a.pos_q, b), ks = a.keys(a.pos_k, b), qc = a.queries(a.chain_q, b), kc = a.keys(a.chain_k, b);
    const int r0 = chunk * a.chunk, r1 = r0 + min(a.chunk, a.Nq - r0);
    const bool whole = a.Nk >= 8, ragged = j0 + kRbKeys > a.Nk;
    const T *rows = dout + (((int64_t)b * a.H + min(h0 + li, a.H - 1)) * a.Nq) * a.Nk;

    const int64_t p0 = qs[r0], chain = CHAIN ? kc[min(j0 + lane, a.Nk - 1)] : 0;   // of the lane's key of the 64
    int first[G], skip[G], pk[G][8];
    bool near = true;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int col = j0 + 32 * g + 8 * q;
        first[g] = min(col, max(a.Nk - 8, 0));
        skip[g] = min(col - first[g], 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int j = min(first[g] + e, a.Nk - 1);
            near = rb_from(ks[j], p0, pk[g][e]) && near;
            pk[g][e] -= a.reach;
        }
    }
    for (int o = threadIdx.x; o <= 2 * a.reach + 1; o += kRbWaves * 64) lut[o] = o <= 2 * a.reach ? a.lut[o] : a.rows - 1;

    // Sums of a few rows, and of those: in one the roundings of some hundred additions come to three times the error (6.6e-7 of a sum over 131 000 pairs).
    f32x4r acc[TILES], sum[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = sum[t] = f32x4r{0.0f, 0.0f, 0.0f, 0.0f};
    int steps = 0;
    Row next[U][G];
    int pq[U];
    int64_t cq[U];
    auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(base + u * kRbWaves, r1 - 1);
            near = rb_from(qs[i], p0, pq[u]) && near;
            cq[u] = CHAIN ? qc[i] : 0;
            const T *p = rows + (int64_t)i * a.Nk;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (whole) {
                    next[u][g].load(p + first[g]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) next[u][g].e[e] = p[min(e, a.Nk - 1)];
                }
            }
        }
    };
    fetch(r0 + wave);
    __syncthreads();
    for (int base = r0 + wave; base < r1; base += U * kRbWaves) {
        if (++steps % 4 == 0) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                sum[t] += acc[t];
                acc[t] = f32x4r{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        Row now[U][G];
        int pn[U];
        int64_t cn[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            pn[u] = pq[u];
            cn[u] = cq[u];
#pragma unroll
            for (int g = 0; g < G; ++g) now[u][g] = next[u][g];
        }
        if (base + U * kRbWaves < r1) fetch(base + U * kRbWaves);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (base + u * kRbWaves >= r1) break;
            const unsigned long long same = CHAIN ? __builtin_amdgcn_ballot_w64(chain == cn[u]) : 0;   // (the whole wave is here)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                int o[8];
                // (a piece that steps back may begin before the workgroup's first key, with keys that are another's)
                const int at = first[g] - j0;
                const unsigned mine = (unsigned)(same >> max(at, 0)) << max(-at, 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = min(max(pn[u] - pk[g][e], 0), 2 * a.reach);
                    if (CHAIN) o[e] = mine >> e & 1 ? o[e] : 2 * a.reach + 1;
                }
                u16x2r bucket[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) bucket[i] = u16x2r{lut[o[2 * i]], lut[o[2 * i + 1]]};
                if (ragged) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < skip[g] || first[g] + e >= a.Nk) bucket[e / 2][e % 2] = 0xffff;
                }
                v8 d[Row::PARTS];
                now[u][g].parts(d);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint16_t r = (uint16_t)(16 * t + li);
                    u32x4r hot;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {   // ONE where equal: ONE - min(different bits, 1) * ONE
                        const u16x2r off = rb_any_bits(bucket[i] ^ u16x2r{r, r});
                        hot[i] = __builtin_bit_cast(uint32_t, u16x2r{(uint16_t)Row::ONE, (uint16_t)Row::ONE} - off * u16x2r{(uint16_t)Row::ONE, (uint16_t)Row::ONE});
                    }
#pragma unroll
                    for (int k = 0; k < Row::PARTS; ++k) acc[t] = rb_mma(__builtin_bit_cast(v8, hot), d[k], acc[t]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        acc[t] += sum[t];
        if (sizeof(T) == 4) acc[t] *= Row::DOWN;
    }
    bool fine = near;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) fine = fine && __builtin_fabsf(acc[t][r]) < __builtin_inff();
    if (wave > 0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds[((wave - 1) * TILES * 4 + 4 * t + r) * 64 + lane] = acc[t][r];
    }
    const bool again = __syncthreads_or(!fine);
    const int64_t at = ((int64_t)b * a.chunks + chunk) * a.strips + strip;
    auto write = [&](int row, int h, float s) {
        if (part) part[(at * a.rows + row) * a.H + h] = s;
        else store_as(dtable, (int64_t)row * a.H + h, s, a.table_dtype);
    };
    if (!again) {
        if (wave > 0 || h0 + li >= a.H) return;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float s = acc[t][r];
#pragma unroll
                for (int w = 0; w < kRbWaves - 1; ++w) s += lds[(w * TILES * 4 + 4 * t + r) * 64 + lane];
                const int row = 16 * t + 4 * q + r;
                if (row < a.rows) write(row, h0 + li, s);
            }
        return;
    }
    // one entry of the table per thread, pair by pair: rows' sums, then their sum (in one chain of 128 rows of equal numbers the roundings came to 6e-5)
    const int h = h0 + threadIdx.x % kRbHeads;
    if (h >= a.H) return;
    const T *mine = dout + ((int64_t)b * a.H + h) * a.Nq * a.Nk;
    for (int row = threadIdx.x / kRbHeads; row < a.rows; row += kRbWaves * 64 / kRbHeads) {
        float s = 0.0f;
        for (int i = r0; i < r1; ++i) {
            float one = 0.0f;
            for (int j = j0; j < min(j0 + kRbKeys, a.Nk); ++j) {
                const int o = CHAIN && kc[j] != qc[i] ? 2 * a.reach + 1 : rb_offset(qs[i], ks[j], a.reach);
                if (lut[o] == row) one += (float)mine[(int64_t)i * a.Nk + j];
            }
            s += one;
        }
        write(row, h, s);
    }
}

// The gradient of a pair bias that all batches share: the sum of the output's over them.  Bound by memory: 4 x 32 x 1024^2 in fp32 124 us (671 MB, 5.4 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) relative_bias_batch_sum(const T *dout, T *dpair, int64_t n, int batches) {
    constexpr int V = RbVec<T>::V;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (i >= n) return;
    if (i + V <= n) {
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.0f;
#pragma unroll 4
        for (int b = 0; b < batches; ++b) {
            const RbVec<T> v = RbVec<T>::load(dout + b * n + i);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += (float)v.e[e];
        }
        RbVec<T> r;
#pragma unroll
        for (int e = 0; e < V; ++e) r.e[e] = (T)s[e];
        r.store(dpair + i);
        return;
    }
    for (int64_t j = i; j < n; ++j) {
        float s = 0.0f;
        for (int b = 0; b < batches; ++b) s += (float)dout[b * n + j];
        dpair[j] = (T)s;
    }
}

// Rows of a workgroup, a multiple of `step`, so that `want` workgroups cover a call of `each` strips of rows.
static void rb_chunks(RbArgs &a, int64_t each, int step, int want) {
    int64_t chunk = (each * a.Nq + want - 1) / want;
    chunk = (chunk + step - 1) / step * step;
    if (chunk > a.Nq) chunk = a.Nq;
    a.chunk = (int)chunk;
    a.chunks = (int)((a.Nq + chunk - 1) / chunk);
}

static int rb_check(const EvoRelativeBias *p) {
    if (!p) return EVO_EINVAL;
    if (p->B <= 0 || p->H <= 0 || p->Nq <= 0 || p->Nk <= 0 || !known_dtype(p->dtype) || !known_dtype(p->table_dtype)) return EVO_EINVAL;
    if (!p->lut || !p->pos_q || !p->pos_k || (p->pos_bytes != 4 && p->pos_bytes != 8) || !p->chain_q != !p->chain_k) return EVO_EINVAL;
    if (p->reach < 0 || p->rows < 1) return EVO_EINVAL;
    if (p->reach > kRbMaxReach || p->rows > kRbMaxRows) return EVO_EUNSUPPORTED;
    if (p->pos_q_stride_b < 0 || p->pos_k_stride_b < 0) return EVO_EINVAL;
    if (p->Nq > kRbMost || p->Nk > kRbMost) return EVO_EOVERFLOW;
    const int64_t rows = (int64_t)p->B * p->H;
    if (rows > INT32_MAX || rows * p->Nq / p->Nq != rows || rows > INT64_MAX / 8 / p->Nq || rows * p->Nq > INT64_MAX / 8 / p->Nk) return EVO_EOVERFLOW;
    return EVO_OK;
}

static RbArgs rb_args(const EvoRelativeBias &p) {
    RbArgs a{};
    a.pos_q = p.pos_q;
    a.pos_k = p.pos_k;
    a.chain_q = p.chain_q;
    a.chain_k = p.chain_k;
    a.lut = (const uint8_t *)p.lut;
    a.table = p.table;
    a.pos_q_b = p.pos_q_stride_b;
    a.pos_k_b = p.pos_k_stride_b;
    a.pair_b = p.pair_stride_b;
    a.pair_h = p.pair_stride_h;
    a.pair_row = p.pair_stride_row;
    a.B = p.B;
    a.H = p.H;
    a.Nq = p.Nq;
    a.Nk = p.Nk;
    a.rows = p.rows;
    a.reach = p.reach;
    a.table_dtype = p.table_dtype;
    a.wide = p.pos_bytes == 8;
    return a;
}

// Workgroups.  Forward: one for every 64 KB, since each looks its table and positions up first, two for each unit at least and eight at most, that enough is under
// way.  Of 512 / 1024 / 2048 / 4096, us: 2 x 64 x 256^2 with a bias in bf16 12.1 / 12.7 / 17.6 / 24.5, 1 x 32 x 1024^2 in fp32 81 / 58 / 47 / 47.
// Backward: two for each unit, whose parts are few to add up.  Of 256 / 384 / 512 / 1024 / 2048: 4 x 32 x 1024^2 in fp32 140 / 131 / 107 / 116 / 121,
// 2 x 64 x 256^2 in bf16 14.2 / 15.4 / 14.3 / 15.2 / 21.5.
constexpr int kRbBytes = 1 << 16, kRbFwdLeast = 512, kRbFwdMost = 2048, kRbBwdGroups = 512;

static RbArgs rb_fwd_args(const EvoRelativeBias &p) {
    RbArgs a = rb_args(p);
    const int v = p.dtype == EVO_F32 ? 4 : 8;
    const int64_t pieces = ((int64_t)p.Nk + v - 1) / v;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < pieces) a.lanes *= 2;
    a.strips = (int)((pieces + 63) / 64);
    const int64_t bytes = (int64_t)p.B * p.H * p.Nq * p.Nk * (p.dtype == EVO_F32 ? 4 : 2) * (p.pair ? 2 : 1);
    const int want = (int)std::min<int64_t>(std::max<int64_t>(bytes / kRbBytes, kRbFwdLeast), kRbFwdMost);
    rb_chunks(a, (int64_t)p.B * p.H * a.strips, kRbWaves * 64 / a.lanes, want);
    return a;
}

static RbArgs rb_bwd_args(const EvoRelativeBias &p) {
    RbArgs a = rb_args(p);
    a.strips = (p.Nk + kRbKeys - 1) / kRbKeys;
    a.heads = (p.H + kRbHeads - 1) / kRbHeads;
    rb_chunks(a, (int64_t)p.B * a.strips * a.heads, kRbWaves, kRbBwdGroups);
    return a;
}
static int64_t rb_parts(const RbArgs &a) { return (int64_t)a.B * a.chunks * a.strips; }
static bool rb_bwd_fits(const RbArgs &a) { return grid_fits(rb_parts(a) * a.heads, kRbWaves * 64) && (int64_t)a.rows * a.H <= INT32_MAX; }

template <typename T, bool CHAIN>
static int rb_launch_bwd(const RbArgs &a, unsigned grid, const T *dout, float *part, void *dtable, hipStream_t st) {
    auto go = [&](auto n) {
        constexpr int TILES = decltype(n)::value;
        constexpr int sums = (kRbWaves - 1) * TILES * 4 * 64 * sizeof(float), most = sums + (2 * kRbMaxReach + 2) * sizeof(uint16_t);
        constexpr auto kernel = relative_bias_bwd<TILES, T, CHAIN>;
        static PerDevice done;
        if (const int rc = ensure_dynamic_lds((const void *)kernel, most, done, nullptr)) return rc;
        kernel<<<grid, kRbWaves * 64, sums + (2 * a.reach + 2) * sizeof(uint16_t), st>>>(a, dout, part, dtable);
        return hip_rc();
    };
    if (a.rows <= 32) return go(std::integral_constant<int, 2>());
    if (a.rows <= 48) return go(std::integral_constant<int, 3>());
    if (a.rows <= 80) return go(std::integral_constant<int, 5>());
    if (a.rows <= 144) return go(std::integral_constant<int, 9>());
    return go(std::integral_constant<int, 16>());
}

}  // namespace evo

extern "C" {

int evoattn_relative_bias_fwd(const EvoRelativeBias *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = rb_check(p)) return rc;
    if (!p->table || !p->out) return EVO_EINVAL;
    if (p->pair && (p->pair_stride_row < 0 || p->pair_stride_h < 0 || p->pair_stride_b < 0)) return EVO_EINVAL;
    const RbArgs a = rb_fwd_args(*p);
    const int64_t grid = (int64_t)a.strips * a.chunks * a.H * a.B;
    if (!grid_fits(grid, kRbWaves * 64)) return EVO_EOVERFLOW;
    const size_t lds = (2 * (size_t)p->reach + 1) * sizeof(float);
    return by_dtype(p->dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto pair, auto chain) {
            relative_bias_fwd<T, decltype(pair)::value, decltype(chain)::value><<<(unsigned)grid, kRbWaves * 64, lds, (hipStream_t)hip_stream>>>(a, (const T *)p->pair, (T *)p->out);
            return hip_rc();
        };
        const std::true_type yes;
        const std::false_type no;
        return p->pair ? p->chain_q ? go(yes, yes) : go(yes, no) : p->chain_q ? go(no, yes) : go(no, no);
    });
}

size_t evoattn_relative_bias_bwd_workspace_bytes(const EvoRelativeBias *p) {
    using namespace evo;
    if (rb_check(p)) return 0;
    const RbArgs a = rb_bwd_args(*p);
    if (!rb_bwd_fits(a)) return 0;
    return (size_t)rb_parts(a) * p->rows * p->H * sizeof(float);
}

int evoattn_relative_bias_bwd(const EvoRelativeBias *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = rb_check(p)) return rc;
    if (!p->dout || (!p->dtable && !p->dpair)) return EVO_EINVAL;
    hipStream_t st = (hipStream_t)hip_stream;
    // (before any launch)
    const int64_t n = (int64_t)p->H * p->Nq * p->Nk;
    const int v = p->dtype == EVO_F32 ? 4 : 8;
    if (p->dpair && !grid_fits((n + 256 * v - 1) / (256 * v), 256)) return EVO_EOVERFLOW;
    if (p->dtable) {
        const RbArgs a = rb_bwd_args(*p);
        if (!rb_bwd_fits(a)) return EVO_EOVERFLOW;
        const int64_t parts = rb_parts(a), grid = parts * a.heads, entries = (int64_t)a.rows * a.H;
        float *part = parts > 1 ? (float *)p->workspace : nullptr;
        if (parts > 1 && (!p->workspace || p->workspace_bytes < evoattn_relative_bias_bwd_workspace_bytes(p))) return EVO_EWORKSPACE;
        const int rc = by_dtype(p->dtype, [&](auto t) {
            typedef decltype(t) T;
            return p->chain_q ? rb_launch_bwd<T, true>(a, (unsigned)grid, (const T *)p->dout, part, p->dtable, st)
                              : rb_launch_bwd<T, false>(a, (unsigned)grid, (const T *)p->dout, part, p->dtable, st);
        });
        if (rc) return rc;
        if (part) {
            // (512 parts: 4 to 5 us, a launch and the way to memory)
            if (const int rc2 = launch_sum_parts(part, p->dtable, (int)entries, parts, p->table_dtype, st)) return rc2;
        }
    }
    if (p->dpair) {
        return by_dtype(p->dtype, [&](auto t) {
            typedef decltype(t) T;
            const int64_t groups = (n + 256 * RbVec<T>::V - 1) / (256 * RbVec<T>::V);
            relative_bias_batch_sum<T><<<(unsigned)groups, 256, 0, st>>>((const T *)p->dout, (T *)p->dpair, n, p->B);
            return hip_rc();
        });
    }
    return EVO_OK;
}

}  // extern "C"
