// layer_norm.hip — layer norm over the last dimension, forward and backward, gfx950.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd,  y = h w + b
//   g = dy w,  dx = rstd (g - sum g / D - h sum(g h) / D),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is taken from centred values (the exponential neurons have |mean| >> their spread: E[x^2] - E[x]^2 would
// cancel).  Sums, statistics and the parameter gradients are fp32; y and dx are rounded once, to x's type.
// Parameter gradients are reduced in a fixed order (partial sums per chunk of rows, then over the chunks): no atomics,
// the same bits on every run.
#include "row_common.h"

namespace armnet {

constexpr int LN_TPB = 256;

struct NormArgs {
    int64_t rows;
    int d;
    RowView x;
    const void* dy;        // backward: [rows, d]
    const void* weight;    // [d] or null
    const void* bias;      // [d] or null
    float eps;
    void* out;             // forward: y [rows, d] | backward: dx [rows, d] or null
    float* mean;           // [rows]
    float* rstd;           // [rows]
    float* partial;        // backward: [chunks, 2, d]
    int chunks;
};

template <typename T, typename W>
__global__ void __launch_bounds__(LN_TPB) norm_fwd_kernel(NormArgs a) {
    __shared__ float scratch[LN_TPB / WAVE];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = row_ptr<T>(a.x, r);
    float s = 0.f;
    for (int i = threadIdx.x; i < a.d; i += LN_TPB) s += to_f32(x[i]);
    const float mean = block_sum<LN_TPB / WAVE>(s, scratch) / (float)a.d;
    float q = 0.f;
    for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
        const float c = to_f32(x[i]) - mean;
        q = fmaf(c, c, q);
    }
    const float rstd = 1.f / sqrtf(block_sum<LN_TPB / WAVE>(q, scratch) / (float)a.d + a.eps);
    T* y = (T*)a.out + r * a.d;
    for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
        float v = (to_f32(x[i]) - mean) * rstd;
        if (a.weight) v *= to_f32(((const W*)a.weight)[i]);
        if (a.bias) v += to_f32(((const W*)a.bias)[i]);
        y[i] = from_f32<T>(v);
    }
    if (threadIdx.x == 0 && a.mean) {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
    }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_TPB) norm_dx_kernel(NormArgs a) {
    __shared__ float scratch[LN_TPB / WAVE];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = row_ptr<T>(a.x, r);
    const T* dy = (const T*)a.dy + r * a.d;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
        const float g = to_f32(dy[i]) * (a.weight ? to_f32(((const W*)a.weight)[i]) : 1.f);
        s1 += g;
        s2 = fmaf(g, (to_f32(x[i]) - mean) * rstd, s2);
    }
    const float m1 = block_sum<LN_TPB / WAVE>(s1, scratch) / (float)a.d;
    const float m2 = block_sum<LN_TPB / WAVE>(s2, scratch) / (float)a.d;
    T* dx = (T*)a.out + r * a.d;
    for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
        const float g = to_f32(dy[i]) * (a.weight ? to_f32(((const W*)a.weight)[i]) : 1.f);
        const float h = (to_f32(x[i]) - mean) * rstd;
        dx[i] = from_f32<T>(rstd * (g - m1 - h * m2));
    }
    }
}

// a thread owns one column of one chunk of rows
template <typename T>
__global__ void __launch_bounds__(LN_TPB) norm_param_partial_kernel(NormArgs a) {
    const int i = blockIdx.x * LN_TPB + threadIdx.x;
    if (i >= a.d) return;
    const int64_t per = (a.rows + a.chunks - 1) / a.chunks;
    const int64_t r0 = blockIdx.y * per;
    const int64_t r1 = r0 + per < a.rows ? r0 + per : a.rows;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = to_f32(((const T*)a.dy)[r * a.d + i]);
        sw = fmaf(g, (to_f32(row_ptr<T>(a.x, r)[i]) - a.mean[r]) * a.rstd[r], sw);
        sb += g;
    }
    a.partial[((int64_t)blockIdx.y * 2 + 0) * a.d + i] = sw;
    a.partial[((int64_t)blockIdx.y * 2 + 1) * a.d + i] = sb;
}

template <typename W>
__global__ void __launch_bounds__(LN_TPB) norm_param_sum_kernel(const float* partial, int chunks, int d, W* dw, W* db) {
    const int i = blockIdx.x * LN_TPB + threadIdx.x;
    if (i >= d) return;
    float sw = 0.f, sb = 0.f;
    for (int c = 0; c < chunks; ++c) {
        sw += partial[((int64_t)c * 2 + 0) * d + i];
        sb += partial[((int64_t)c * 2 + 1) * d + i];
    }
    if (dw) dw[i] = from_f32<W>(sw);
    if (db) db[i] = from_f32<W>(sb);
}

static int norm_chunks(int64_t rows) { return (int)(rows < 512 ? rows : 512); }

}  // namespace armnet

using namespace armnet;

extern "C" {

int armnet_layer_norm_fwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t d, int x_type,
                          const void* x, int w_type, const void* weight, const void* bias, float eps, void* y, float* mean,
                          float* rstd, void* stream) {
    if (rows < 0 || inner < 0 || d <= 0 || !row_type_ok(x_type) || !row_type_ok(w_type) || !(eps >= 0.f)) return ARMNET_ERR_BAD_ARG;
    if (rows >= ((int64_t)1 << 31) || d >= ((int64_t)1 << 31)) return ARMNET_ERR_UNSUPPORTED;
    if ((mean == nullptr) != (rstd == nullptr)) return ARMNET_ERR_BAD_ARG;
    if (rows == 0) return ARMNET_OK;
    if (!x || !y) return ARMNET_ERR_BAD_ARG;
    NormArgs a{};
    a.rows = rows; a.d = (int)d;
    a.x = RowView{x, inner, outer_stride, row_stride};
    a.weight = weight; a.bias = bias; a.eps = eps; a.out = y; a.mean = mean; a.rstd = rstd;
    ARMNET_ROW_TYPE(x_type, T, ARMNET_ROW_TYPE(w_type, W, (norm_fwd_kernel<T, W><<<row_grid(rows), LN_TPB, 0, (hipStream_t)stream>>>(a))));
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

int64_t armnet_layer_norm_bwd_ws_bytes(int64_t rows, int64_t d) {
    if (rows < 0 || d <= 0) return -1;
    return (int64_t)norm_chunks(rows) * 2 * d * 4;
}

int armnet_layer_norm_bwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t d, int x_type,
                          const void* x, const void* dy, int w_type, const void* weight, const float* mean, const float* rstd,
                          void* dx, void* dweight, void* dbias, void* workspace, int64_t ws_bytes, void* stream) {
    if (rows < 0 || inner < 0 || d <= 0 || !row_type_ok(x_type) || !row_type_ok(w_type)) return ARMNET_ERR_BAD_ARG;
    if (rows >= ((int64_t)1 << 31) || d >= ((int64_t)1 << 31)) return ARMNET_ERR_UNSUPPORTED;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return ARMNET_ERR_BAD_ARG;
    const bool params = dweight || dbias;
    if (params && rows > 0 && (!workspace || ws_bytes < armnet_layer_norm_bwd_ws_bytes(rows, d))) return ARMNET_ERR_BAD_ARG;
    hipStream_t st = (hipStream_t)stream;
    NormArgs a{};
    a.rows = rows; a.d = (int)d;
    a.x = RowView{x, inner, outer_stride, row_stride};
    a.dy = dy; a.weight = weight; a.out = dx; a.mean = (float*)mean; a.rstd = (float*)rstd;
    a.partial = (float*)workspace; a.chunks = norm_chunks(rows);
    if (dx && rows > 0) {
        ARMNET_ROW_TYPE(x_type, T, ARMNET_ROW_TYPE(w_type, W, (norm_dx_kernel<T, W><<<row_grid(rows), LN_TPB, 0, st>>>(a))));
        ARMNET_LAUNCH_CHECK();
    }
    if (params) {
        const unsigned gx = (unsigned)((d + LN_TPB - 1) / LN_TPB);
        if (rows > 0) {
            ARMNET_ROW_TYPE(x_type, T, (norm_param_partial_kernel<T><<<dim3(gx, a.chunks), LN_TPB, 0, st>>>(a)));
            ARMNET_LAUNCH_CHECK();
        }
        ARMNET_ROW_TYPE(w_type, W, (norm_param_sum_kernel<W><<<gx, LN_TPB, 0, st>>>(a.partial, a.chunks, a.d, (W*)dweight, (W*)dbias)));
        ARMNET_LAUNCH_CHECK();
    }
    return ARMNET_OK;
}

}  // extern "C"
