// row_common.h — what the row operators share (layer_norm.hip, score_rows.hip): a row is the last dimension of a tensor whose
// leading dimensions are described by at most two strides; elements are float32, bfloat16 or float16, arithmetic is fp32.
#ifndef ARMNET_ROW_COMMON_H
#define ARMNET_ROW_COMMON_H

#include <float.h>

#include "armnet_common.h"

namespace armnet {

constexpr int WAVE = 64;

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// row r of a tensor: base + (r / inner) * outer_stride + (r % inner) * row_stride, in elements (inner = 0: one stride only)
struct RowView {
    const void* base;
    int64_t inner, outer_stride, row_stride;
};

template <typename T>
__device__ __forceinline__ const T* row_ptr(const RowView& v, int64_t r) {
    const T* p = (const T*)v.base;
    if (v.inner == 0) return p + r * v.row_stride;
    return p + (r / v.inner) * v.outer_stride + (r % v.inner) * v.row_stride;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }          // round to nearest even

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// sum / maximum over a block of NW waves, the same value in every thread; `scratch`: NW floats of LDS of its own
template <int NW>
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = wave_sum(v);
    if constexpr (NW == 1) return v;
    __syncthreads();
    if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += scratch[w];
    return s;
}

template <int NW>
__device__ __forceinline__ float block_max(float v, float* scratch) {
    v = wave_max(v);
    if constexpr (NW == 1) return v;
    __syncthreads();
    if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
    __syncthreads();
    float s = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) s = fmaxf(s, scratch[w]);
    return s;
}

// blocks of a launch with one row a block (the kernels stride over the rest: a launch holds fewer than 2^32 threads)
inline unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

inline bool row_type_ok(int t) { return t == ARMNET_F32 || t == ARMNET_BF16 || t == ARMNET_F16; }
inline size_t row_type_size(int t) { return t == ARMNET_F32 ? 4 : 2; }

}  // namespace armnet

// run `expr` with `T` bound to the element type of `type` (one of armnet_float_type)
#define ARMNET_ROW_TYPE(type, T, expr)                                   \
    do {                                                                 \
        if ((type) == ARMNET_F32) { using T = float; expr; }             \
        else if ((type) == ARMNET_BF16) { using T = bf16_t; expr; }      \
        else { using T = f16_t; expr; }                                  \
    } while (0)

#endif
