// Attention within packed sequences: its entry points.
#include "packed_common.h"

namespace evo {

#define EVO_PACKED(D)                                                              \
    int launch_packed_fwd_d##D(const EvoPacked &, hipStream_t);                    \
    int launch_packed_dq_d##D(const EvoPacked &, const BackwardRows &, float *, hipStream_t);   \
    int launch_packed_dkdv_d##D(const EvoPacked &, const BackwardRows &, float *, hipStream_t); \
    size_t packed_dq_bytes_d##D(const EvoPacked &);                                \
    size_t packed_dkdv_bytes_d##D(const EvoPacked &);                              \
    size_t packed_fwd_bytes_d##D(const EvoPacked &);                               \
    size_t packed_few_bytes_d##D(const EvoPacked &);                               \
    int launch_packed_few_d##D(const EvoPacked &, hipStream_t);                    \
    size_t packed_f32_few_bytes_d##D(const EvoPacked &);                           \
    int launch_packed_f32_few_d##D(const EvoPacked &, hipStream_t);                \
    size_t packed_f32_fwd_bytes_d##D(const EvoPacked &);                           \
    int launch_packed_f32_fwd_d##D(const EvoPacked &, hipStream_t);                \
    size_t packed_f32_bwd_bytes_d##D(const EvoPacked &);                           \
    int launch_packed_f32_bwd_d##D(const EvoPacked &, const BackwardRows &, float *, hipStream_t);
EVO_PACKED(32)
EVO_PACKED(64)
EVO_PACKED(96)
EVO_PACKED(128)
#undef EVO_PACKED
// One of the four by the head dim
#define EVO_BY_HEAD_DIM(name, p, ...) \
    ((p).D <= 32 ? name##_d32(__VA_ARGS__) : (p).D <= 64 ? name##_d64(__VA_ARGS__) : (p).D <= 96 ? name##_d96(__VA_ARGS__) : name##_d128(__VA_ARGS__))

// Whether the kernels that split the keys of few queries serve the forward: by what an average sequence has of queries times the query heads that share a key head (`columns` there), of keys, and by sequences times key
// heads (`units`).  Measured with 1, 4, 16 and 256 sequences of 32 to 65536 keys (us; the tiled kernel in brackets):
//   16 bits, up to 32 columns; 17 to 32 are multiplied in two halves.  Fewer than 128 units, where tiles would leave most of the chip idle: 8 heads (8) of 64, 4 sequences of 1024 keys, 8 queries 13 (15), 32 queries 16 (16), of 256 keys 10.5 (9.1); 32 heads (8): one query, 16 of
//   1024 14 (28); least favourable, one sequence of 32 keys 8.1 (6.3).  Keys in one chunk: heads of their own cost the same both ways but for 17 to 32 columns of D = 128 (1000 of 32 keys 282 (226)); shared heads, which a tile reads again for each, 32 heads (8), 8 queries, 256 of 128
//   26 (66), 16 of 128 8.6 (8.5).  Keys in parts, whose results go to memory and back for every row: 32 heads (8) of 64, 32 sequences of 512 keys, 1 query 14 (20), 4 20 (21), 8 28 (21); 8 queries, of 1024 keys 34 (32), of 4096 82 (102); 8 heads (8): 1 query 13.6 (12.4), 8 16 (13), 16
//   19 (13); with 128 units 16 of 1024 keys, 1 query 14 (17), 8 14.5 (16), 16 17 (16), 32 22 (16.5).
//   fp32.  A second launch makes the results, a wave to each row.  8 heads (8) of 64, 8 queries: 1000 sequences of 8 keys 69 (84), 256 of 64 34 (39), of 1024 246 (365); 32 queries: 60 (44) and 287 (374); 64 queries: 100 (56) and 562 (538).  One sequence of 64 keys
//   14.3 (10.9), of 1024 14.7 (18.9).  32 heads (8) of 128, 16 queries: one of 1024 keys 34 (28), of 4096 43 (59), 4 of 1024 42 (65).
static bool few_queries(const EvoPacked &p) {
    const int64_t n = p.n, group = p.H / p.Hk, columns = p.Tq * group, units = n * p.Hk;   // (columns, and keys, of all sequences)
    if (!n) return false;
    if (p.dtype != EVO_F32) {
        if (columns > 32 * n) return false;
        const bool wide = columns > 16 * n;
        if (units < 128 && (!wide || p.Tk >= 1024 * n)) return true;
        if (!EVO_BY_HEAD_DIM(packed_few_bytes, p, p)) return !wide || (group > 1 && n * p.H >= 768);
        return (units < 256 && !wide ? 8192 : 24576) * p.Tq <= p.Tk * group * (p.D > 64 ? p.D : 64);
    }
    if (columns > 64 * n || 512 * p.Tq > (p.Tk > 64 * n ? p.Tk : 64 * n) * group * p.D) return false;   // (each row's way through memory, beside what its keys take)
    if (units < 512 && p.Tk < 128 * n) return false;
    if (units < 32 && columns > 32 * n && p.Tk < 4096 * n) return false;
    return row_waves_fit(p.Tq * p.H);
}

static int64_t align_rows(int64_t n) { return (n + 63) / 64 * 64; }   // (16-byte pieces behind them)

static int packed_check(const EvoPacked *p) {
    if (!p || p->n < 0 || p->H < 1 || p->Hk < 1 || p->H % p->Hk || p->D < 1 || !known_dtype(p->dtype) || (p->offset_bytes != 4 && p->offset_bytes != 8) || p->Tq < 0 ||
        p->Tk < 0 || !(p->scale >= 0x1p-64f && p->scale <= 0x1p64f))   // (the backward divides sums of exponents by it)
        return EVO_EINVAL;
    if (p->D > 128) return EVO_EUNSUPPORTED;
    // (row numbers and the positions of tiles are formed in 32 bits)
    if (p->Tq > INT32_MAX / 2 || p->Tk > INT32_MAX / 2 || p->n > INT32_MAX / 4 || (int64_t)p->H > 1 << 20) return EVO_EOVERFLOW;
    if (p->dtype != EVO_F32 && p->D % 8) return EVO_EALIGN;
    return EVO_OK;
}
// The matrix kernels move pieces of 16 bytes, address the rows of a stage by 32 bits, and take what is beyond a sequence for out of range, which rows have to lie apart for.
static bool packed_aligned(const EvoPacked &p, bool backward) {
    if (p.dtype == EVO_F32) return true;
    for (const void *x : {p.q, p.k, p.v, (const void *)p.o, (const void *)p.o_low, backward ? p.dout : nullptr, backward ? (const void *)p.dq : nullptr, backward ? (const void *)p.dk : nullptr,
                          backward ? (const void *)p.dv : nullptr})
        if ((uintptr_t)x % 16) return false;
    for (int64_t x : {p.q_stride_t, p.k_stride_t, p.v_stride_t, backward ? p.dout_stride_t : 0})
        if (x % 8 || x >= 1 << 23) return false;
    if ((p.Tq && p.q_stride_t < p.D) || (p.Tk && (p.k_stride_t < p.D || p.v_stride_t < p.D)) || (backward && p.Tq && p.dout_stride_t < p.D)) return false;
    for (int64_t x : {p.q_stride_h, p.k_stride_h, p.v_stride_h, backward ? p.dout_stride_h : 0})
        if (x % 8) return false;
    return true;
}
static int packed_pointers(const EvoPacked &p, bool backward) {
    if (!p.offsets || !p.key_offsets) return EVO_EINVAL;
    if (p.Tq && (!p.q || !p.o || (backward && (!p.dout || !p.dq || !p.lse)))) return EVO_EINVAL;
    if (p.Tk && (!p.k || !p.v || (backward && !p.dk != !p.dv))) return EVO_EINVAL;
    const size_t bytes = backward ? evoattn_packed_bwd_workspace_bytes(&p) : evoattn_packed_fwd_workspace_bytes(&p);
    if (p.workspace_bytes < bytes || (bytes && !p.workspace)) return EVO_EWORKSPACE;
    if (bytes && (uintptr_t)p.workspace % 16) return EVO_EALIGN;
    return packed_aligned(p, backward) ? EVO_OK : EVO_EALIGN;
}

}  // namespace evo

extern "C" {

size_t evoattn_packed_fwd_workspace_bytes(const EvoPacked *p) {
    using namespace evo;
    if (packed_check(p)) return 0;
    if (p->dtype == EVO_F32) return few_queries(*p) ? EVO_BY_HEAD_DIM(packed_f32_few_bytes, *p, *p) : EVO_BY_HEAD_DIM(packed_f32_fwd_bytes, *p, *p);
    return few_queries(*p) ? EVO_BY_HEAD_DIM(packed_few_bytes, *p, *p) : EVO_BY_HEAD_DIM(packed_fwd_bytes, *p, *p);
}

int evoattn_packed_fwd(const EvoPacked *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = packed_check(p)) return rc;
    if (!p->Tq) return EVO_OK;
    if (const int rc = packed_pointers(*p, false)) return rc;
    const hipStream_t st = (hipStream_t)hip_stream;
    if (few_queries(*p)) return p->dtype == EVO_F32 ? EVO_BY_HEAD_DIM(launch_packed_f32_few, *p, *p, st) : EVO_BY_HEAD_DIM(launch_packed_few, *p, *p, st);
    return p->dtype == EVO_F32 ? EVO_BY_HEAD_DIM(launch_packed_f32_fwd, *p, *p, st) : EVO_BY_HEAD_DIM(launch_packed_fwd, *p, *p, st);
}

size_t evoattn_packed_bwd_workspace_bytes(const EvoPacked *p) {
    using namespace evo;
    if (packed_check(p)) return 0;
    const size_t rows = (size_t)align_rows((int64_t)p->H * p->Tq) * sizeof(float);
    if (p->dtype == EVO_F32) return rows + EVO_BY_HEAD_DIM(packed_f32_bwd_bytes, *p, *p);
    const size_t dq = EVO_BY_HEAD_DIM(packed_dq_bytes, *p, *p), dkdv = EVO_BY_HEAD_DIM(packed_dkdv_bytes, *p, *p);
    return 2 * rows + (dq > dkdv ? dq : dkdv);
}

int evoattn_packed_bwd(const EvoPacked *p, void *hip_stream) {
    using namespace evo;
    if (const int rc = packed_check(p)) return rc;
    if (!p->Tq && !p->Tk) return EVO_OK;
    if (const int rc = packed_pointers(*p, true)) return rc;
    const hipStream_t st = (hipStream_t)hip_stream;
    const BackwardRows saved = {(float *)p->workspace, (float *)p->workspace + align_rows((int64_t)p->H * p->Tq)};
    if (p->dtype == EVO_F32) return EVO_BY_HEAD_DIM(launch_packed_f32_bwd, *p, *p, saved, saved.base, st);   // (`base` is 16 bits': sums begin there)
    float *const sums = saved.base + align_rows((int64_t)p->H * p->Tq);   // (dQ's parts, then dK's and dV's)
    if (p->Tq) {
        if (const int rc = EVO_BY_HEAD_DIM(launch_packed_dq, *p, *p, saved, sums, st)) return rc;
    }
    return p->Tk && p->dk ? EVO_BY_HEAD_DIM(launch_packed_dkdv, *p, *p, saved, sums, st) : EVO_OK;
}

}  // extern "C"
