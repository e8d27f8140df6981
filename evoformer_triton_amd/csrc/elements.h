// Elements of a type that a call names at run time, and sums of parts: what the relative position bias and the 8-bit layers share.
#pragma once

#include "bwd_common.h"
#include "common.h"

namespace evo {

__device__ __forceinline__ float load_as(const void *p, int64_t i, int dtype) {
    return dtype == EVO_F32 ? ((const float *)p)[i] : dtype == EVO_BF16 ? (float)((const bf16_t *)p)[i] : (float)((const f16_t *)p)[i];
}
__device__ __forceinline__ void store_as(void *p, int64_t i, float v, int dtype) {
    if (dtype == EVO_F32) ((float *)p)[i] = v;
    else if (dtype == EVO_BF16) ((bf16_t *)p)[i] = (bf16_t)v;
    else ((f16_t *)p)[i] = (f16_t)v;
}

static inline bool known_dtype(int d) { return d == EVO_BF16 || d == EVO_F16 || d == EVO_F32; }
// f of a value of the type
template <typename F>
static int by_dtype(int dtype, F &&f) {
    return dtype == EVO_BF16 ? f(bf16_t()) : dtype == EVO_F16 ? f(f16_t()) : f(float());
}

// out[c] = sum of part[i][c], i < parts, in a fixed order: 32 columns to a workgroup by 32 slices of the parts, in their order.  THREADS: 32 of them, each with 32 / THREADS
// slices; the same additions.
template <int THREADS>
__device__ __forceinline__ void sum_parts(const float *part, void *out, int cols, int64_t parts, int dtype, unsigned id) {
    __shared__ float sums[32][33];
    const int c = id * 32 + (threadIdx.x & 31), first = threadIdx.x >> 5;
#pragma unroll
    for (int slice = first; slice < 32; slice += THREADS) {
        float s = 0.0f;
        if (c < cols) {
#pragma unroll 8
            for (int64_t i = slice; i < parts; i += 32) s += part[i * cols + c];
        }
        sums[slice][threadIdx.x & 31] = s;
    }
    __syncthreads();
    if (first || c >= cols) return;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sums[i][threadIdx.x];
    store_as(out, c, s, dtype);
}

}  // namespace evo
