// Packed attention in 16 bits: what its matrix kernels share.  Compiled once per head dim (-DEVO_D=32|64|96|128).
#pragma once

#include "packed_common.h"
#include "stream_common.h"

#ifndef EVO_D
#error "compile with -DEVO_D=<head dim>"
#endif

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {   // (one name for each head dim's kernels)

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

template <typename F>
static int by_half(int dtype, F &&f) {
    return dtype == EVO_BF16 ? f(bf16_t()) : f(f16_t());
}

}  // namespace
}  // namespace evo
