// layer_norm.hip — layer norm over the last dimension, forward and backward, gfx950.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd,  y = h w + b
//   g = dy w,  dx = rstd (g - sum g / D - h sum(g h) / D),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is taken from centred values (the exponential neurons have |mean| >> their spread: E[x^2] - E[x]^2 would
// cancel).  Sums, statistics and the parameter gradients are fp32; y and dx are rounded once, to x's type.
// Parameter gradients are reduced in a fixed order (a block's rows, its groups, then the blocks): no atomics, the same bits
// on every run.
//
// Both passes are bound by memory.  A row is read once and stays in registers: LPR lanes of a wave hold it (short rows: several
// rows a wave), or NW waves, NV pieces of 16 bytes a lane.  A lane keeps its columns for all its rows, so weight, bias and the
// sums of their gradients stay in registers too, and the next rows are on their way while a row is worked on.  Rows longer than
// 16384 values take a form that reads them again for each step.
#include "row_common.h"

namespace armnet {

constexpr int LN_TPB = 256;
constexpr int LN_MAX_D = 16384;            // longest row that is held in registers

struct NormArgs {
    int64_t rows;
    int d;
    RowView x;
    const void* dy;        // backward: [rows, d]
    int w_type;
    const void* weight;    // [d] or null
    const void* bias;      // [d] or null
    float eps;
    void* out;             // forward: y [rows, d] | backward: dx [rows, d] or null
    float* mean;           // [rows]
    float* rstd;           // [rows]
    // backward
    bool params;           // the parameters' gradients are wanted
    float* partial;        // [blocks, 2, d], for more than one block
    void* dweight;         // [d] or null
    void* dbias;
    int blocks;
};

__device__ __forceinline__ float load_param(const void* p, int type, int i) {
    if (type == ARMNET_F32) return ((const float*)p)[i];
    if (type == ARMNET_BF16) return (float)((const bf16_t*)p)[i];
    return (float)((const f16_t*)p)[i];
}

__device__ __forceinline__ void store_param(void* p, int type, int i, float v) {
    if (type == ARMNET_F32) ((float*)p)[i] = v;
    else if (type == ARMNET_BF16) ((bf16_t*)p)[i] = (bf16_t)v;
    else ((f16_t*)p)[i] = (f16_t)v;
}

// a piece of which only the first `n` elements are there; the others read as 0 and are not written
template <typename T>
__device__ __forceinline__ u32x4 load_some(const T* p, int n) {
    constexpr int V = Piece<T>::N;
    if (n >= V) return Piece<T>::load(p);
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < n ? to_f32(p[e]) : 0.f;
    return Piece<T>::pack(f);
}

template <typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&f)[Piece<T>::N]) {
    constexpr int V = Piece<T>::N;
    if (n >= V) {
        Piece<T>::store(p, Piece<T>::pack(f));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = from_f32<T>(f[e]);
    }
}

// sum over the lanes (and waves) that hold a row, in each of them; scratch: one float a wave, of this sum alone
template <int LPR, int NW>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    if constexpr (LPR < WAVE) {
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) v += __shfl_xor(v, d);
        return v;
    } else {
        v = wave_sum(v);
        if constexpr (NW == 1) return v;
        const int wave = threadIdx.x / WAVE;
        if ((threadIdx.x & (WAVE - 1)) == 0) scratch[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) v += scratch[wave / NW * NW + i];
        return v;
    }
}

// One row group: LPR lanes (NW = 1) or NW waves.  A block holds TPB / (LPR or NW * 64) of them.
template <typename T, int LPR, int NW, int NV, int TPB>
__global__ void __launch_bounds__(TPB) norm_fwd_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N, NT = LPR < WAVE ? LPR : NW * WAVE, GROUPS = TPB / NT;
    __shared__ float scratch[2][TPB / WAVE];
    const int group = threadIdx.x / NT, tid = threadIdx.x & (NT - 1);
    float w[NV][V], b[NV][V];
    int cnt[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * NT + tid) * V;
        cnt[i] = a.d - at < 0 ? 0 : a.d - at < V ? a.d - at : V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[i][e] = a.weight && e < cnt[i] ? load_param(a.weight, a.w_type, at + e) : 1.f;
            b[i][e] = a.bias && e < cnt[i] ? load_param(a.bias, a.w_type, at + e) : 0.f;
        }
    }
    const float rd = 1.f / (float)a.d;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int64_t rounds = (a.rows + step - 1) / step;
    auto load = [&](int64_t r, u32x4 (&raw)[NV]) {
        const T* x = row_ptr<T>(a.x, r < a.rows ? r : a.rows - 1);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (cnt[i]) raw[i] = load_some(x + (i * NT + tid) * V, cnt[i]);
    };
    u32x4 raw[NV] = {}, next[NV] = {};
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    load(r, raw);
    for (int64_t k = 0; k < rounds; ++k, r += step) {
        if (k + 1 < rounds) load(r + step, next);
        float f[NV][V];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Piece<T>::unpack(raw[i], f[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[i][e];
        }
        const float mean = row_sum<LPR, NW>(s, scratch[0]) / (float)a.d;     // a constant row is its own mean
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[i][e] = e < cnt[i] ? f[i][e] - mean : 0.f;
                q = fmaf(f[i][e], f[i][e], q);
            }
        const float rstd = 1.f / sqrtf(row_sum<LPR, NW>(q, scratch[1]) * rd + a.eps);
        if (r < a.rows) {
            T* y = (T*)a.out + r * a.d;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) f[i][e] = fmaf(f[i][e] * rstd, w[i][e], b[i][e]);
                if (cnt[i]) store_some(y + (i * NT + tid) * V, cnt[i], f[i]);
            }
            if (tid == 0 && a.mean) {
                a.mean[r] = mean;
                a.rstd[r] = rstd;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = next[i];
    }
}

// dx of a row, and the block's share of dw and db: in registers over its rows, then over its groups through LDS
template <typename T, int LPR, int NW, int NV, int TPB>
__global__ void __launch_bounds__(TPB) norm_bwd_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N, NT = LPR < WAVE ? LPR : NW * WAVE, GROUPS = TPB / NT;
    __shared__ float scratch[2][TPB / WAVE];
    constexpr int SHARES = LPR < WAVE ? TPB / WAVE : GROUPS;     // short rows: a wave's groups meet in registers
    __shared__ float sums[2][SHARES > 1 ? NV * NT * V : 1];
    const int group = threadIdx.x / NT, tid = threadIdx.x & (NT - 1);
    float w[NV][V], dw[NV][V] = {}, db[NV][V] = {};
    int cnt[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * NT + tid) * V;
        cnt[i] = a.d - at < 0 ? 0 : a.d - at < V ? a.d - at : V;
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = a.weight && e < cnt[i] ? load_param(a.weight, a.w_type, at + e) : 1.f;
    }
    const float rd = 1.f / (float)a.d;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int64_t rounds = (a.rows + step - 1) / step;
    struct Row {
        u32x4 x[NV], dy[NV];
        float mean, rstd;
    };
    auto load = [&](int64_t r, Row& o) {
        const bool in = r < a.rows;                    // a group without a row works on the last one's values and drops them
        const int64_t q = in ? r : a.rows - 1;
        const T* x = row_ptr<T>(a.x, q);
        const T* dy = (const T*)a.dy + q * a.d;
        o.mean = a.mean[q];
        o.rstd = a.rstd[q];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (cnt[i]) {
                o.x[i] = load_some(x + (i * NT + tid) * V, cnt[i]);
                o.dy[i] = load_some(dy + (i * NT + tid) * V, cnt[i]);
            }
    };
    Row cur = {}, next = {};
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    load(r, cur);
    for (int64_t k = 0; k < rounds; ++k, r += step) {
        if (k + 1 < rounds) load(r + step, next);
        const bool in = r < a.rows;
        float h[NV][V], g[NV][V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Piece<T>::unpack(cur.x[i], h[i]);
            Piece<T>::unpack(cur.dy[i], g[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[i][e] = e < cnt[i] ? (h[i][e] - cur.mean) * cur.rstd : 0.f;
                if (in) {
                    dw[i][e] = fmaf(g[i][e], h[i][e], dw[i][e]);
                    db[i][e] += g[i][e];
                }
                g[i][e] *= w[i][e];
                s1 += g[i][e];
                s2 = fmaf(g[i][e], h[i][e], s2);
            }
        }
        if (a.out) {
            const float m1 = row_sum<LPR, NW>(s1, scratch[0]) * rd;
            const float m2 = row_sum<LPR, NW>(s2, scratch[1]) * rd;
            if (in) {
                T* dx = (T*)a.out + r * a.d;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
#pragma unroll
                    for (int e = 0; e < V; ++e) g[i][e] = cur.rstd * (g[i][e] - m1 - h[i][e] * m2);
                    if (cnt[i]) store_some(dx + (i * NT + tid) * V, cnt[i], g[i]);
                }
            }
        }
        cur = next;
    }
    if (!a.params) return;
    int share = group;
    if constexpr (LPR < WAVE) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int d = LPR; d < WAVE; d <<= 1) {
                    dw[i][e] += __shfl_xor(dw[i][e], d);
                    db[i][e] += __shfl_xor(db[i][e], d);
                }
        share = (threadIdx.x & (WAVE - 1)) < LPR ? (int)threadIdx.x / WAVE : -1;
    }
    if constexpr (SHARES > 1) {
        for (int q = 0; q < SHARES; ++q) {             // one after the other; the last leaves with the sum
            if (share == q) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int at = (e * NV + i) * NT + tid;
                        if (q) {
                            dw[i][e] += sums[0][at];
                            db[i][e] += sums[1][at];
                        }
                        sums[0][at] = dw[i][e];
                        sums[1][at] = db[i][e];
                    }
            }
            __syncthreads();
        }
    }
    if (share == SHARES - 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int col = (i * NT + tid) * V + e;
                if (e >= cnt[i]) continue;
                if (a.blocks == 1) {
                    if (a.dweight) store_param(a.dweight, a.w_type, col, dw[i][e]);
                    if (a.dbias) store_param(a.dbias, a.w_type, col, db[i][e]);
                } else {
                    a.partial[((int64_t)blockIdx.x * 2 + 0) * a.d + col] = dw[i][e];
                    a.partial[((int64_t)blockIdx.x * 2 + 1) * a.d + col] = db[i][e];
                }
            }
    }
}

// the blocks' shares together: 64 columns a block, 16 waves that take the shares in turn
constexpr int LN_SUM_WAVES = 16;
__global__ void __launch_bounds__(LN_SUM_WAVES * WAVE) norm_param_kernel(const float* partial, int blocks, int d, int w_type, void* dweight,
                                                                         void* dbias) {
    __shared__ float part[LN_SUM_WAVES][WAVE];
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    const int col = blockIdx.x * WAVE + lane;
    void* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    float s = 0.f;
    if (col < d) {
        const float* p = partial + (int64_t)blockIdx.y * d + col;
#pragma unroll 8
        for (int k = wave; k < blocks; k += LN_SUM_WAVES) s += p[(int64_t)k * 2 * d];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < d) {
#pragma unroll
        for (int i = 1; i < LN_SUM_WAVES; ++i) s += part[i][lane];
        store_param(out, w_type, col, s);
    }
}

// ---- rows longer than LN_MAX_D: a block a row, read again for each step ---------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(LN_TPB) norm_long_fwd_kernel(NormArgs a) {
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
            const float w = a.weight ? load_param(a.weight, a.w_type, i) : 1.f, b = a.bias ? load_param(a.bias, a.w_type, i) : 0.f;
            y[i] = from_f32<T>(fmaf((to_f32(x[i]) - mean) * rstd, w, b));
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LN_TPB) norm_long_dx_kernel(NormArgs a) {
    __shared__ float scratch[LN_TPB / WAVE];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        const T* dy = (const T*)a.dy + r * a.d;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
            const float g = to_f32(dy[i]) * (a.weight ? load_param(a.weight, a.w_type, i) : 1.f);
            s1 += g;
            s2 = fmaf(g, (to_f32(x[i]) - mean) * rstd, s2);
        }
        const float m1 = block_sum<LN_TPB / WAVE>(s1, scratch) / (float)a.d;
        const float m2 = block_sum<LN_TPB / WAVE>(s2, scratch) / (float)a.d;
        T* dx = (T*)a.out + r * a.d;
        for (int i = threadIdx.x; i < a.d; i += LN_TPB) {
            const float g = to_f32(dy[i]) * (a.weight ? load_param(a.weight, a.w_type, i) : 1.f);
            const float h = (to_f32(x[i]) - mean) * rstd;
            dx[i] = from_f32<T>(rstd * (g - m1 - h * m2));
        }
    }
}

// a thread owns one column of one share of the rows
template <typename T>
__global__ void __launch_bounds__(LN_TPB) norm_long_param_kernel(NormArgs a) {
    const int i = blockIdx.x * LN_TPB + threadIdx.x;
    if (i >= a.d) return;
    const int64_t per = (a.rows + a.blocks - 1) / a.blocks;
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

// ---- launches ------------------------------------------------------------------------------------------------------------

constexpr int LN_BWD_TPB = 1024;

// how many rows a block of the backward works on at a time: the groups of 16 waves (see launch_norm)
static int norm_bwd_groups(int64_t d, int64_t v) {
    const int64_t np = (d + v - 1) / v;
    if (np <= WAVE) {
        int lpr = 1;
        while (lpr < np) lpr *= 2;
        return LN_BWD_TPB / lpr;
    }
    if (np <= 2 * WAVE) return 16;
    if (np <= 8 * WAVE) return 4;
    return 1;
}

// Blocks of the backward, one a unit: 16 waves with a row in work and one on its way each keep enough bytes in flight, and fewer
// blocks mean fewer shares of the parameters' gradients to add up.  (The 16-bit types' groups: never fewer rows than blocks need.)
static int norm_blocks(int64_t rows, int64_t d, int64_t v) {
    if (d > LN_MAX_D) return (int)(rows < 256 ? rows : 256);
    const int64_t groups = norm_bwd_groups(d, v);
    const int64_t n = (rows + groups - 1) / groups;
    return (int)(n < 256 ? n : 256);
}

template <typename T, int LPR, int NW, int NV, bool BWD>
static void launch_norm_one(const NormArgs& a, hipStream_t st) {
    if constexpr (BWD) {
        norm_bwd_kernel<T, LPR, NW, NV, LN_BWD_TPB><<<a.blocks, LN_BWD_TPB, 0, st>>>(a);
    } else {
        constexpr int TPB = NW == 16 ? 1024 : LN_TPB, GROUPS = TPB / (LPR < WAVE ? LPR : NW * WAVE);
        int64_t blocks = (a.rows + GROUPS - 1) / GROUPS;
        const int64_t most = (int64_t)device_cu_count() * (NW == 16 ? 2 : 8);
        if (blocks > most) blocks = most;
        norm_fwd_kernel<T, LPR, NW, NV, TPB><<<(unsigned)blocks, TPB, 0, st>>>(a);
    }
}

// who holds a row: by its number of 16-byte pieces
template <typename T, bool BWD>
static void launch_norm(const NormArgs& a, hipStream_t st) {
    const int np = (a.d + Piece<T>::N - 1) / Piece<T>::N;
    if (np <= 1) launch_norm_one<T, 1, 1, 1, BWD>(a, st);
    else if (np <= 2) launch_norm_one<T, 2, 1, 1, BWD>(a, st);
    else if (np <= 4) launch_norm_one<T, 4, 1, 1, BWD>(a, st);
    else if (np <= 8) launch_norm_one<T, 8, 1, 1, BWD>(a, st);
    else if (np <= 16) launch_norm_one<T, 16, 1, 1, BWD>(a, st);
    else if (np <= 32) launch_norm_one<T, 32, 1, 1, BWD>(a, st);
    else if (np <= 64) launch_norm_one<T, 64, 1, 1, BWD>(a, st);
    else if (np <= 128) launch_norm_one<T, 64, 1, 2, BWD>(a, st);
    else if (np <= 256) launch_norm_one<T, 64, 4, 1, BWD>(a, st);
    else if (np <= 512) launch_norm_one<T, 64, 4, 2, BWD>(a, st);
    else if (np <= 1024) launch_norm_one<T, 64, 16, 1, BWD>(a, st);
    else if (np <= 2048) launch_norm_one<T, 64, 16, 2, BWD>(a, st);
    else if constexpr (sizeof(T) == 4) launch_norm_one<T, 64, 16, 4, BWD>(a, st);
}

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
    a.w_type = w_type; a.weight = weight; a.bias = bias; a.eps = eps; a.out = y; a.mean = mean; a.rstd = rstd;
    hipStream_t st = (hipStream_t)stream;
    if (d <= LN_MAX_D) {
        ARMNET_ROW_TYPE(x_type, T, (launch_norm<T, false>(a, st)));
    } else {
        ARMNET_ROW_TYPE(x_type, T, (norm_long_fwd_kernel<T><<<row_grid(rows), LN_TPB, 0, st>>>(a)));
    }
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

int64_t armnet_layer_norm_bwd_ws_bytes(int64_t rows, int64_t d) {
    if (rows < 0 || d <= 0) return -1;
    const int n4 = norm_blocks(rows, d, 4), n8 = norm_blocks(rows, d, 8);
    const int64_t n = n4 > n8 ? n4 : n8;
    return n == 1 && d <= LN_MAX_D ? 0 : n * 2 * d * 4;              // one block writes the gradients by itself
}

int armnet_layer_norm_bwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t d, int x_type,
                          const void* x, const void* dy, int w_type, const void* weight, const float* mean, const float* rstd,
                          void* dx, void* dweight, void* dbias, void* workspace, int64_t ws_bytes, void* stream) {
    if (rows < 0 || inner < 0 || d <= 0 || !row_type_ok(x_type) || !row_type_ok(w_type)) return ARMNET_ERR_BAD_ARG;
    if (rows >= ((int64_t)1 << 31) || d >= ((int64_t)1 << 31)) return ARMNET_ERR_UNSUPPORTED;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return ARMNET_ERR_BAD_ARG;
    const bool params = dweight || dbias;
    if (params && rows > 0 && (ws_bytes < armnet_layer_norm_bwd_ws_bytes(rows, d) || (ws_bytes > 0 && !workspace))) return ARMNET_ERR_BAD_ARG;
    hipStream_t st = (hipStream_t)stream;
    NormArgs a{};
    a.rows = rows; a.d = (int)d;
    a.x = RowView{x, inner, outer_stride, row_stride};
    a.dy = dy; a.w_type = w_type; a.weight = weight; a.out = dx; a.mean = (float*)mean; a.rstd = (float*)rstd;
    a.params = params; a.partial = (float*)workspace;
    a.dweight = dweight; a.dbias = dbias;
    a.blocks = norm_blocks(rows, d, x_type == ARMNET_F32 ? 4 : 8);
    if (rows > 0 && (dx || params)) {
        if (d <= LN_MAX_D) {
            ARMNET_ROW_TYPE(x_type, T, (launch_norm<T, true>(a, st)));
            ARMNET_LAUNCH_CHECK();
            if (a.blocks == 1) return ARMNET_OK;                     // the one block has written the parameters' gradients
        } else {
            if (dx) {
                ARMNET_ROW_TYPE(x_type, T, (norm_long_dx_kernel<T><<<row_grid(rows), LN_TPB, 0, st>>>(a)));
                ARMNET_LAUNCH_CHECK();
            }
            if (params) {
                const dim3 grid((unsigned)((d + LN_TPB - 1) / LN_TPB), a.blocks);
                ARMNET_ROW_TYPE(x_type, T, (norm_long_param_kernel<T><<<grid, LN_TPB, 0, st>>>(a)));
                ARMNET_LAUNCH_CHECK();
            }
        }
    }
    if (params) {
        norm_param_kernel<<<dim3((unsigned)((d + WAVE - 1) / WAVE), 2), LN_SUM_WAVES * WAVE, 0, st>>>(a.partial, a.blocks, a.d, w_type,
                                                                                                      dweight, dbias);
        ARMNET_LAUNCH_CHECK();
    }
    return ARMNET_OK;
}

}  // extern "C"
