// The learned relative position bias of the attention: a number per head and bucket of the distance between two residues,
//   out[b,h,i,j] = table[bucket(b,i,j), h] (+ pair[b,h,i,j]),  bucket = lut[clamp(pos_q[b,i] - pos_k[b,j], -R, R) + R],
// or the table's last row where i and j lie in different chains; and the table's gradient, the sum of the output's over the pairs of
// each bucket.
#include <type_traits>

#include "common.h"
#include "bwd_common.h"
#include "kernels.h"

namespace evo {

constexpr int kRbWaves = 4;
constexpr int kRbMaxReach = 4096, kRbMaxRows = 256;
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

// What a lane holds of its V keys for all rows, and of a query; positions and chains of 4 or 8 bytes.
template <typename P, bool CHAIN>
struct RbSide {
    const P *pos, *chain;
    __device__ __forceinline__ int64_t at(int64_t i) const { return (int64_t)pos[i]; }
    __device__ __forceinline__ int64_t chain_at(int64_t i) const { return CHAIN ? (int64_t)chain[i] : 0; }
};

struct RbShape {
    int lanes;    // that a row's strip takes, a power of two up to 64
    int strips;   // of 64 lanes' elements, of a row
};

struct RbArgs {
    const void *pos_q, *pos_k, *chain_q, *chain_k;   // [B or 1, Nq], [B or 1, Nk]
    const uint8_t *lut;
    const void *table;
    int64_t pos_q_b, pos_k_b;     // from one batch to the next (0: the same)
    int64_t pair_b, pair_h, pair_row;
    int B, H, Nq, Nk, rows, reach, table_dtype;
    int lanes, strips, chunk, chunks;   // chunk: rows of a workgroup
};

__device__ __forceinline__ float rb_entry(const void *t, int64_t i, int dtype) {
    return dtype == EVO_F32 ? ((const float *)t)[i] : dtype == EVO_BF16 ? (float)((const bf16_t *)t)[i] : (float)((const f16_t *)t)[i];
}

__device__ __forceinline__ bool rb_near(int64_t p) { return p > -kRbNear && p < kRbNear; }

// The clipped distance from 0 on.  Positions near zero in 32 bits, any others in 64, where a difference may overflow.
__device__ __forceinline__ int rb_offset(int q, int k, int reach) { return min(max(q - k, -reach), reach) + reach; }
__device__ __forceinline__ int rb_offset(int64_t q, int64_t k, int reach) {
    const int64_t d = __builtin_elementwise_sub_sat(q, k);
    return (int)min(max(d, (int64_t)-reach), (int64_t)reach) + reach;
}

// Forward.
template <typename T, typename P, bool PAIR, bool CHAIN>
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
        val[o] = r < a.rows ? rb_entry(a.table, (int64_t)r * a.H + h, a.table_dtype) : 0.0f;
    }
    const float other = CHAIN ? rb_entry(a.table, (int64_t)(a.rows - 1) * a.H + h, a.table_dtype) : 0.0f;
    const RbSide<P, CHAIN> qs{(const P *)a.pos_q + b * a.pos_q_b, CHAIN ? (const P *)a.chain_q + b * a.pos_q_b : nullptr};
    const RbSide<P, CHAIN> ks{(const P *)a.pos_k + b * a.pos_k_b, CHAIN ? (const P *)a.chain_k + b * a.pos_k_b : nullptr};
    // The last lane of a row that is no whole number of pieces steps back: two lanes write the same values there.
    const int col = (strip * 64 + lane % a.lanes) * V, first = min(col, max(a.Nk - V, 0)), sub = lane / a.lanes, per = 64 / a.lanes;
    const bool mine = col < a.Nk;
    int64_t pk[V], ck[V];
    bool near = true;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t j = min(first + e, a.Nk - 1);
        pk[e] = ks.at(j);
        ck[e] = ks.chain_at(j);
        near = near && rb_near(pk[e]);
    }
    near = __all(near);
    __syncthreads();
    const int r0 = chunk * a.chunk, r1 = min(r0 + a.chunk, a.Nq);
    const int64_t plane = ((int64_t)b * a.H + h) * a.Nq;
    const bool whole = a.Nk >= V;
    for (int base = r0 + wave * per * U; base < r1; base += kRbWaves * per * U) {
        RbVec<T> in[U];
        int64_t pq[U], cq[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(base + u * per + sub, r1 - 1);
            pq[u] = qs.at(i);
            cq[u] = qs.chain_at(i);
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

// Sums over 64 lanes, the same in all.
__device__ __forceinline__ float rb_wave_sum(float s) {
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    return s;
}

// Backward: sums of dout over the pairs of each bucket, of a workgroup's rows.  A wave keeps COPIES sums of each bucket in LDS, lane l
// adding to copy l % COPIES; where there are fewer copies than lanes, the lanes take turns.  The LDS takes a wave's additions in their
// order, and lanes that add at once add to different copies: the order of a sum is fixed.
template <typename T, typename P, int COPIES, bool CHAIN>
__global__ void __launch_bounds__(kRbWaves * 64) relative_bias_bwd(RbArgs a, const T *dout, float *part, void *dtable) {
    constexpr int V = RbVec<T>::V, U = 4;
    extern __shared__ float sums[];   // [waves][rows + 1][COPIES], the last row for distances without a bucket; then uint16 [2 R + 1]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int held = (a.rows + 1) * COPIES;
    uint16_t *at = reinterpret_cast<uint16_t *>(sums + kRbWaves * held);
    unsigned id = blockIdx.x;
    const int strip = id % a.strips;
    id /= a.strips;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int b = id % a.B, h = id / a.B;
    for (int i = threadIdx.x; i < kRbWaves * held; i += kRbWaves * 64) sums[i] = 0.0f;
    for (int o = threadIdx.x; o <= 2 * a.reach; o += kRbWaves * 64) at[o] = (uint16_t)(min((int)a.lut[o], a.rows) * COPIES);
    const RbSide<P, CHAIN> qs{(const P *)a.pos_q + b * a.pos_q_b, CHAIN ? (const P *)a.chain_q + b * a.pos_q_b : nullptr};
    const RbSide<P, CHAIN> ks{(const P *)a.pos_k + b * a.pos_k_b, CHAIN ? (const P *)a.chain_k + b * a.pos_k_b : nullptr};
    const int col = (strip * 64 + lane % a.lanes) * V, first = min(col, max(a.Nk - V, 0)), sub = lane / a.lanes, per = 64 / a.lanes;
    const bool mine = col < a.Nk;
    int64_t pk[V], ck[V];
    bool near = true;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t j = min(first + e, a.Nk - 1);
        pk[e] = ks.at(j);
        ck[e] = ks.chain_at(j);
        near = near && rb_near(pk[e]);
    }
    near = __all(near);
    __syncthreads();
    float *own = sums + wave * held + lane % COPIES;
    const int r0 = chunk * a.chunk, r1 = min(r0 + a.chunk, a.Nq);
    const int64_t plane = ((int64_t)b * a.H + h) * a.Nq;
    const bool whole = a.Nk >= V;
    for (int base = r0 + wave * per * U; base < r1; base += kRbWaves * per * U) {
        RbVec<T> in[U];
        int64_t pq[U], cq[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(base + u * per + sub, r1 - 1);
            pq[u] = qs.at(i);
            cq[u] = qs.chain_at(i);
            const T *p = dout + (plane + i) * a.Nk;
            if (whole) {
                in[u] = RbVec<T>::load(p + first);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) in[u].e[e] = p[min(e, a.Nk - 1)];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = mine && base + u * per + sub < r1;
            int o[V];
            if (near && __all(rb_near(pq[u]))) {
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rb_offset((int)pq[u], (int)pk[e], a.reach);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rb_offset(pq[u], pk[e], a.reach);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                int r = at[o[e]];
                if (CHAIN) r = ck[e] == cq[u] ? r : (a.rows - 1) * COPIES;
                // (of a lane that stepped back, what the lane before it has; of a row shorter than a piece, what lies behind it)
                const bool counts = on && first + e >= col && first + e < a.Nk;
#pragma unroll
                for (int turn = 0; turn < 64 / COPIES; ++turn)
                    if (counts && lane / COPIES == turn) __builtin_amdgcn_ds_atomic_fadd_f32((__attribute__((address_space(3))) float *)(own + r), (float)in[u].e[e]);
            }
        }
    }
    __syncthreads();
    for (int r = wave; r < a.rows; r += kRbWaves) {
        float s = 0.0f;
        if (lane < COPIES) {
#pragma unroll
            for (int w = 0; w < kRbWaves; ++w) s += sums[w * held + r * COPIES + lane];
        }
        s = rb_wave_sum(s);
        if (lane == 0) {
            if (part) {
                part[((int64_t)r * a.H + h) * ((int64_t)a.B * a.chunks * a.strips) + ((int64_t)b * a.chunks + chunk) * a.strips + strip] = s;
            } else if (a.table_dtype == EVO_F32) {
                ((float *)dtable)[(int64_t)r * a.H + h] = s;
            } else if (a.table_dtype == EVO_BF16) {
                ((bf16_t *)dtable)[(int64_t)r * a.H + h] = (bf16_t)s;
            } else {
                ((f16_t *)dtable)[(int64_t)r * a.H + h] = (f16_t)s;
            }
        }
    }
}

// The workgroups' sums, a wave for each entry of the table.
__global__ void __launch_bounds__(256) relative_bias_sum(const float *part, void *dtable, int entries, int parts, int dtype) {
    const int e = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (e >= entries) return;
    float s = 0.0f;
#pragma unroll 4
    for (int i = lane; i < parts; i += 64) s += part[(int64_t)e * parts + i];
    s = rb_wave_sum(s);
    if (lane) return;
    if (dtype == EVO_F32) ((float *)dtable)[e] = s;
    else if (dtype == EVO_BF16) ((bf16_t *)dtable)[e] = (bf16_t)s;
    else ((f16_t *)dtable)[e] = (f16_t)s;
}

// The gradient of a pair bias that all batches share: the sum of the output's over them.
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

static int rb_rc() {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? EVO_OK : EVO_EHIP - (int)err;
}

static bool rb_dtype(int d) { return d == EVO_BF16 || d == EVO_F16 || d == EVO_F32; }

// How a row is dealt to lanes, and how many rows a workgroup takes so that `want` of them cover the call.
static void rb_shape(RbArgs &a, const EvoRelativeBias &p, int want) {
    const int v = p.dtype == EVO_F32 ? 4 : 8;
    const int64_t pieces = ((int64_t)p.Nk + v - 1) / v;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < pieces) a.lanes *= 2;
    a.strips = (int)((pieces + 63) / 64);
    const int step = kRbWaves * 64 / a.lanes;   // rows that a workgroup's waves take at once
    const int64_t rows = (int64_t)p.B * p.H * p.Nq * a.strips;
    int64_t chunk = (rows + want - 1) / want;
    chunk = (chunk + step - 1) / step * step;
    if (chunk > p.Nq) chunk = p.Nq;
    a.chunk = (int)chunk;
    a.chunks = (p.Nq + a.chunk - 1) / a.chunk;
}

static int rb_check(const EvoRelativeBias *p) {
    if (!p) return EVO_EINVAL;
    if (p->B <= 0 || p->H <= 0 || p->Nq <= 0 || p->Nk <= 0 || !rb_dtype(p->dtype) || !rb_dtype(p->table_dtype)) return EVO_EINVAL;
    if (!p->lut || !p->pos_q || !p->pos_k || (p->pos_bytes != 4 && p->pos_bytes != 8) || !p->chain_q != !p->chain_k) return EVO_EINVAL;
    if (p->reach < 0 || p->rows < 1) return EVO_EINVAL;
    if (p->reach > kRbMaxReach || p->rows > kRbMaxRows) return EVO_EUNSUPPORTED;
    if (p->pos_q_stride_b < 0 || p->pos_k_stride_b < 0) return EVO_EINVAL;
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
    return a;
}

template <typename F>
static int rb_by_dtype(int dtype, F &&f) {
    return dtype == EVO_BF16 ? f(bf16_t()) : dtype == EVO_F16 ? f(f16_t()) : f(float());
}
// positions' type and whether there are chains
template <typename F>
static int rb_by_side(const EvoRelativeBias &p, F &&f) {
    if (p.pos_bytes == 4) return p.chain_q ? f(int32_t(), std::true_type()) : f(int32_t(), std::false_type());
    return p.chain_q ? f(int64_t(), std::true_type()) : f(int64_t(), std::false_type());
}

constexpr int kRbFwdGroups = 2048, kRbBwdGroups = 1024;

static int rb_copies(int rows) { return rows <= 72 ? 64 : rows <= 144 ? 32 : 16; }
constexpr int kRbMaxLds = 96 << 10;
static_assert(kRbWaves * 73 * 64 * 4 + (2 * kRbMaxReach + 1) * 2 <= kRbMaxLds && 145 * 32 <= 73 * 64 && (kRbMaxRows + 1) * 16 <= 73 * 64, "what a workgroup keeps");

static RbArgs rb_bwd_args(const EvoRelativeBias &p) {
    RbArgs a = rb_args(p);
    rb_shape(a, p, kRbBwdGroups);
    return a;
}
static int64_t rb_parts(const RbArgs &a) { return (int64_t)a.B * a.chunks * a.strips; }

}  // namespace evo

extern "C" {

int evoattn_relative_bias_fwd(const EvoRelativeBias *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = rb_check(p)) return rc;
    if (!p->table || !p->out) return EVO_EINVAL;
    if (p->pair && (p->pair_stride_row < 0 || p->pair_stride_h < 0 || p->pair_stride_b < 0)) return EVO_EINVAL;
    RbArgs a = rb_args(*p);
    rb_shape(a, *p, kRbFwdGroups);
    const int64_t grid = (int64_t)a.strips * a.chunks * a.H * a.B;
    if (grid > INT32_MAX) return EVO_EOVERFLOW;
    const size_t lds = (2 * (size_t)p->reach + 1) * sizeof(float);
    return rb_by_dtype(p->dtype, [&](auto t) {
        typedef decltype(t) T;
        return rb_by_side(*p, [&](auto pos, auto chain) {
            typedef decltype(pos) P;
            constexpr bool C = decltype(chain)::value;
            if (p->pair) relative_bias_fwd<T, P, true, C><<<(unsigned)grid, kRbWaves * 64, lds, (hipStream_t)hip_stream>>>(a, (const T *)p->pair, (T *)p->out);
            else relative_bias_fwd<T, P, false, C><<<(unsigned)grid, kRbWaves * 64, lds, (hipStream_t)hip_stream>>>(a, nullptr, (T *)p->out);
            return rb_rc();
        });
    });
}

size_t evoattn_relative_bias_bwd_workspace_bytes(const EvoRelativeBias *p) {
    using namespace evo;
    if (rb_check(p)) return 0;
    const RbArgs a = rb_bwd_args(*p);
    return (size_t)rb_parts(a) * p->rows * p->H * sizeof(float);
}

int evoattn_relative_bias_bwd(const EvoRelativeBias *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = rb_check(p)) return rc;
    if (!p->dout || (!p->dtable && !p->dpair)) return EVO_EINVAL;
    hipStream_t st = (hipStream_t)hip_stream;
    if (p->dtable) {
        const RbArgs a = rb_bwd_args(*p);
        const int64_t parts = rb_parts(a), grid = parts * a.H, entries = (int64_t)a.rows * a.H;
        if (grid > INT32_MAX || entries > INT32_MAX || parts > INT32_MAX) return EVO_EOVERFLOW;
        float *part = parts > 1 ? (float *)p->workspace : nullptr;
        if (parts > 1 && (!p->workspace || p->workspace_bytes < evoattn_relative_bias_bwd_workspace_bytes(p))) return EVO_EWORKSPACE;
        const int copies = rb_copies(a.rows);
        const size_t lds = (size_t)kRbWaves * (a.rows + 1) * copies * sizeof(float) + (2 * (size_t)a.reach + 1) * sizeof(uint16_t);
        const int rc = rb_by_dtype(p->dtype, [&](auto t) {
            typedef decltype(t) T;
            return rb_by_side(*p, [&](auto pos, auto chain) {
                typedef decltype(pos) P;
                constexpr bool C = decltype(chain)::value;
                auto go = [&](auto n) {
                    constexpr auto kernel = relative_bias_bwd<T, P, decltype(n)::value, C>;
                    static PerDevice done;
                    if (const int rc = ensure_dynamic_lds((const void *)kernel, kRbMaxLds, done, nullptr)) return rc;
                    kernel<<<(unsigned)grid, kRbWaves * 64, lds, st>>>(a, (const T *)p->dout, part, p->dtable);
                    return rb_rc();
                };
                return copies == 64 ? go(std::integral_constant<int, 64>()) : copies == 32 ? go(std::integral_constant<int, 32>()) : go(std::integral_constant<int, 16>());
            });
        });
        if (rc) return rc;
        if (part) {
            relative_bias_sum<<<(unsigned)((entries + 3) / 4), 256, 0, st>>>(part, p->dtable, (int)entries, (int)parts, p->table_dtype);
            if (const int rc2 = rb_rc()) return rc2;
        }
    }
    if (p->dpair) {
        const int64_t n = (int64_t)p->H * p->Nq * p->Nk;
        return rb_by_dtype(p->dtype, [&](auto t) {
            typedef decltype(t) T;
            const int64_t groups = (n + 256 * RbVec<T>::V - 1) / (256 * RbVec<T>::V);
            if (groups > INT32_MAX) return (int)EVO_EOVERFLOW;
            relative_bias_batch_sum<T><<<(unsigned)groups, 256, 0, st>>>((const T *)p->dout, (T *)p->dpair, n, p->B);
            return rb_rc();
        });
    }
    return EVO_OK;
}

}  // extern "C"
