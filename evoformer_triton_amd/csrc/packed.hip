// Attention within packed sequences: its entry points, and a kernel of one row per wave.
//
// Forward: a wave keeps a query row and walks over the keys that it sees, 64 at a time, a key to a lane: scores, the running maximum m and sum l of 2^(score - m), then
// o += p_j v_j with the row's values in the lanes.  Backward with p_ij = 2^(score - lse_i) formed again, delta_i = sum do_i o_i: ds_ij = p_ij (do_i v_j - delta_i) scale,
// dq_i = sum_j ds_ij k_j by a wave per query, dk_j = sum_i ds_ij q_i and dv_j = sum_i p_ij do_i by a wave per key, over the heads that share it in their order.
#include "packed_common.h"

namespace evo {

template <typename T>
__global__ void __launch_bounds__(256) packed_rows_fwd(EvoPacked p, unsigned rows) {
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int i = row / (unsigned)p.H, h = row % (unsigned)p.H;
    row_forward<T>(p, segment_of_row<false>(p, i), i, h);
}
template <typename T>
__global__ void __launch_bounds__(256) packed_rows_dq(EvoPacked p, float *delta, unsigned rows) {
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int i = row / (unsigned)p.H, h = row % (unsigned)p.H;
    const float d = row_delta<T>(p, i, h);
    if ((threadIdx.x & 63) == 0) delta[(int64_t)h * p.Tq + i] = d;
    row_dq<T>(p, segment_of_row<false>(p, i), i, h, d);
}
template <typename T>
__global__ void __launch_bounds__(256) packed_rows_dkdv(EvoPacked p, const float *delta, unsigned rows) {
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= rows) return;
    const int j = row / (unsigned)p.Hk, hk = row % (unsigned)p.Hk;
    row_dkdv<T>(p, segment_of_row<true>(p, j), j, hk, delta);
}

static int packed_check(const EvoPacked *p) {
    if (!p || p->n < 0 || p->H < 1 || p->Hk < 1 || p->H % p->Hk || p->D < 1 || !known_dtype(p->dtype) || (p->offset_bytes != 4 && p->offset_bytes != 8) || p->Tq < 0 ||
        p->Tk < 0 || !(p->scale > 0.0f && p->scale <= FLT_MAX))
        return EVO_EINVAL;
    if (p->D > 128) return EVO_EUNSUPPORTED;
    // (row numbers and the positions of tiles are formed in 32 bits)
    if (p->Tq > INT32_MAX / 2 || p->Tk > INT32_MAX / 2 || p->n > INT32_MAX / 4 || (int64_t)p->H > 1 << 20) return EVO_EOVERFLOW;
    return EVO_OK;
}
static int packed_pointers(const EvoPacked &p, bool backward) {
    if (!p.offsets || !p.key_offsets) return EVO_EINVAL;
    if (p.Tq && (!p.q || !p.o || (backward && (!p.dout || !p.dq || !p.lse)))) return EVO_EINVAL;
    if (p.Tk && (!p.k || !p.v || (backward && !p.dk != !p.dv))) return EVO_EINVAL;
    if (backward && p.Tq && p.workspace_bytes < evoattn_packed_bwd_workspace_bytes(&p)) return EVO_EWORKSPACE;
    if (!backward && p.workspace_bytes < evoattn_packed_fwd_workspace_bytes(&p)) return EVO_EWORKSPACE;
    return EVO_OK;
}

}  // namespace evo

extern "C" {

size_t evoattn_packed_fwd_workspace_bytes(const EvoPacked *p) {
    using namespace evo;
    if (packed_check(p)) return 0;
    return 0;
}

int evoattn_packed_fwd(const EvoPacked *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = packed_check(p)) return rc;
    if (!p->Tq) return EVO_OK;
    if (const int rc = packed_pointers(*p, false)) return rc;
    const int64_t rows = p->Tq * p->H;
    if (rows > INT32_MAX || !grid_fits((rows + 3) / 4, 256)) return EVO_EOVERFLOW;
    return by_dtype(p->dtype, [&](auto t) {
        packed_rows_fwd<decltype(t)><<<(unsigned)((rows + 3) / 4), 256, 0, (hipStream_t)hip_stream>>>(*p, (unsigned)rows);
        return hip_rc();
    });
}

size_t evoattn_packed_bwd_workspace_bytes(const EvoPacked *p) {
    using namespace evo;
    if (packed_check(p)) return 0;
    return (size_t)p->H * p->Tq * sizeof(float);
}

int evoattn_packed_bwd(const EvoPacked *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = packed_check(p)) return rc;
    if (!p->Tq && !p->Tk) return EVO_OK;
    if (const int rc = packed_pointers(*p, true)) return rc;
    const int64_t rows = p->Tq * p->H, keys = p->Tk * p->Hk;
    if (rows > INT32_MAX || keys > INT32_MAX || !grid_fits((rows + 3) / 4, 256) || !grid_fits((keys + 3) / 4, 256)) return EVO_EOVERFLOW;
    const hipStream_t st = (hipStream_t)hip_stream;
    float *delta = (float *)p->workspace;
    return by_dtype(p->dtype, [&](auto t) {
        typedef decltype(t) T;
        if (rows) {
            packed_rows_dq<T><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(*p, delta, (unsigned)rows);
            if (const int rc = hip_rc()) return rc;
        }
        if (keys && p->dk) packed_rows_dkdv<T><<<(unsigned)((keys + 3) / 4), 256, 0, st>>>(*p, delta, (unsigned)keys);
        return hip_rc();
    });
}

}  // extern "C"
