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

// 16 bytes of a row, at whatever address its elements have: one load / store instruction (the memory system takes any alignment;
// a wave's neighbouring pieces touch one cache line more than aligned ones)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
template <typename T>
struct Piece {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ u32x4 load(const T* p) {
        if constexpr (sizeof(T) == 4) return *(const u32x4_at4*)p;
        else return *(const u32x4_at2*)p;
    }
    static __device__ __forceinline__ void store(T* p, u32x4 v) {
        if constexpr (sizeof(T) == 4) *(u32x4_at4*)p = v;
        else *(u32x4_at2*)p = v;
    }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                f[i] = __uint_as_float(v[i]);
            } else if constexpr (__is_same(T, bf16_t)) {
                f[2 * i] = __uint_as_float(v[i] << 16);
                f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const uint32_t w = v[i];
                const h2 h = __builtin_bit_cast(h2, w);
                f[2 * i] = (float)h[0];
                f[2 * i + 1] = (float)h[1];
            }
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[N]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __float_as_uint(f[i]);
            } else {
                typedef T t2 __attribute__((ext_vector_type(2)));
                t2 h;
                h[0] = (T)f[2 * i];
                h[1] = (T)f[2 * i + 1];
                v[i] = __builtin_bit_cast(uint32_t, h);
            }
        }
        return v;
    }
};

// lane exchanges inside the vector unit: within rows of 16 lanes, then across them; the result ends in lane 63
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float old, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xf, false));
}

__device__ __forceinline__ float lane63(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0x111, 0xf>(0.f, v);      // from 1, 2, 4, 8 lanes below
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);      // lane 15 of a row to the next row
    v += dpp<0x143, 0xc>(0.f, v);      // lane 31 to the upper half
    return lane63(v);
}

// sum over aligned groups of LPR lanes, in each of them
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LPR >= 2) v += dpp<0xb1, 0xf>(0.f, v);       // lane ^ 1
    if constexpr (LPR >= 4) v += dpp<0x4e, 0xf>(0.f, v);       // lane ^ 2
    if constexpr (LPR >= 8) v += dpp<0x141, 0xf>(0.f, v);      // the other four of eight
    if constexpr (LPR >= 16) v += dpp<0x140, 0xf>(0.f, v);     // the other eight of sixteen
    if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
    return v;
}

template <int LPR>
__device__ __forceinline__ float lanes_max(float v) {
    if constexpr (LPR >= 2) v = fmaxf(v, dpp<0xb1, 0xf>(v, v));
    if constexpr (LPR >= 4) v = fmaxf(v, dpp<0x4e, 0xf>(v, v));
    if constexpr (LPR >= 8) v = fmaxf(v, dpp<0x141, 0xf>(v, v));
    if constexpr (LPR >= 16) v = fmaxf(v, dpp<0x140, 0xf>(v, v));
    if constexpr (LPR >= 32) v = fmaxf(v, __shfl_xor(v, 16));
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0x111, 0xf>(v, v));
    v = fmaxf(v, dpp<0x112, 0xf>(v, v));
    v = fmaxf(v, dpp<0x114, 0xf>(v, v));
    v = fmaxf(v, dpp<0x118, 0xf>(v, v));
    v = fmaxf(v, dpp<0x142, 0xa>(v, v));
    v = fmaxf(v, dpp<0x143, 0xc>(v, v));
    return lane63(v);
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

// a group of NW waves that works on one row; with NW = 1 the waves of a block go their own ways
template <int NW>
__device__ __forceinline__ void group_sync() {
    if constexpr (NW == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

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
