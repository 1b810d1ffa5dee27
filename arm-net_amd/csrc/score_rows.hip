// score_rows.hip — rows of scores as an answer and as a loss, gfx950: log probabilities of given ids with the entropy and the
// best alternatives (forward, backward), and the distillation loss from a teacher's listed scores (forward, backward).
//
//   m = max x,  z = (x - m) / T,  S = sum e^z,  p = e^z / S,  log p = z - log S,  H = -sum p log p = log S - sum e^z z / S
//   dx_j = (1/T) [ sum_k g_k 1(id_k = j) - p_j (G + g_H (log p_j + H)) ],   G = sum of the g_k whose id is inside the row
//
//   q = softmax over the listed teacher scores / T,  loss = T^2 sum_k q_k (log q_k - log p[id_k])
//   dx_j = g T (p_j - sum_k q_k 1(id_k = j))
//
// Sums are held in base 2 (z2 = z log2 e, exponentials by the hardware's exp2) and everything in fp32; log p is
// (x - m) / T - ln2 log2 S, as far as fp32 reaches.  Gradients are rounded once, to x's type.  m starts at the lowest finite number instead of -inf: a masked score (-inf) then has z = -inf and e^z = 0
// without a special case, a row of the lowest number has p = 1/C, and S = 0 says that nothing in the row is above -inf.
// (m, log2 S) go from the forward to the backward as two numbers: their sum would lose what m's magnitude takes.
#include "row_common.h"

namespace armnet {

constexpr int SC_TPB = 256;
constexpr int SC_NW = SC_TPB / WAVE;
constexpr int SC_MAX_IDS = 1024;        // ids of a row
constexpr int SC_MAX_TOP = 64;          // alternatives of a row
constexpr float Z_FLOOR = -1000.f;      // exp2 is 0 far above it; keeps 0 * (-inf) out of the entropy's sum
constexpr float LN2 = 0.6931471805599453f;

struct ScoreArgs {
    int64_t rows;
    int c;
    RowView x;
    float t;                   // temperature
    float rt;                  // 1 / T
    float c2;                  // log2(e) / T
    int n_ids;
    const void* ids;           // [rows, n_ids]
    int id_type;
    // log probabilities
    float* logp;               // [rows, n_ids]
    float* entropy;            // [rows] or null
    int top;
    float* top_logp;           // [rows, top]
    int64_t* top_ids;          // [rows, top]
    // distillation
    const void* teacher;       // [rows, n_ids]
    int t_type;
    float* loss;               // [rows]
    // forward out, backward in
    float* stats;              // [rows, 2]: m, log2 S (+inf: nothing above -inf); distillation [rows, 4]: also the teacher's
    // backward
    const float* g_logp;       // [rows, n_ids] or null | distillation: g_loss [rows]
    const float* g_entropy;    // [rows] or null
    void* dx;                  // [rows, c]
    int32_t* id_status;
};

__device__ __forceinline__ int64_t load_id(const void* ids, int id_type, int64_t i) {
    return id_type == ARMNET_ID_I64 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (type == ARMNET_F32) return ((const float*)p)[i];
    if (type == ARMNET_BF16) return (float)((const bf16_t*)p)[i];
    return (float)((const f16_t*)p)[i];
}

// unsigned keys in the order of (value, lowest id first); -0 and 0 are the same value.  0 is below every key.
__device__ __forceinline__ uint64_t score_key(float v, uint32_t id) {
    const uint32_t b = __float_as_uint(v + 0.f);
    const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((uint64_t)k << 32) | (uint32_t)~id;
}

template <int NW>
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* scratch) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const uint64_t o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
    __syncthreads();
    uint64_t s = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) s = scratch[w] > s ? scratch[w] : s;
    return s;
}

// (m, S, sum e z2) of a row, the same in every thread
template <typename T>
__device__ __forceinline__ void row_sums(const ScoreArgs& a, const T* x, float* scratch, float& m, float& S, float& W) {
    float mx = -FLT_MAX;
    for (int i = threadIdx.x; i < a.c; i += SC_TPB) mx = fmaxf(mx, to_f32(x[i]));
    m = block_max<SC_NW>(mx, scratch);
    float s = 0.f, w = 0.f;
    for (int i = threadIdx.x; i < a.c; i += SC_TPB) {
        const float z = (to_f32(x[i]) - m) * a.c2;
        const float e = exp2f(z);
        s += e;
        w = fmaf(e, fmaxf(z, Z_FLOOR), w);
    }
    S = block_sum<SC_NW>(s, scratch);
    W = block_sum<SC_NW>(w, scratch);
}

template <typename T>
__global__ void __launch_bounds__(SC_TPB) score_fwd_kernel(ScoreArgs a) {
    __shared__ float scratch[SC_NW];
    __shared__ uint64_t scratch64[SC_NW];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        float m, S, W;
        row_sums(a, x, scratch, m, S, W);
        const bool some = !(S == 0.f);
        const float l2 = some ? log2f(S) : INFINITY;
        if (threadIdx.x == 0) {
            if (a.entropy) a.entropy[r] = some ? LN2 * (l2 - W / S) : 0.f;
            if (a.stats) {
                a.stats[2 * r] = m;
                a.stats[2 * r + 1] = l2;
            }
        }
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
            float v = 0.f;
            if (id >= a.c) {
                v = NAN;
                if (a.id_status) flag_bad_id(a.id_status);
            } else if (id >= 0) {
                v = some ? (to_f32(x[id]) - m) * a.rt - LN2 * l2 : -INFINITY;
            }
            a.logp[r * a.n_ids + k] = v;
        }
        uint64_t last = ~(uint64_t)0;
        for (int k = 0; k < a.top; ++k) {              // the largest key below the last one
            uint64_t best = 0;
            for (int i = threadIdx.x; i < a.c; i += SC_TPB) {
                const float v = to_f32(x[i]);
                const uint64_t key = v > -INFINITY ? score_key(v, (uint32_t)i) : 0;
                if (key < last && key > best) best = key;
            }
            last = block_max_u64<SC_NW>(best, scratch64);
            if (threadIdx.x == 0) {
                const int64_t id = last ? (int64_t)(uint32_t)~(uint32_t)last : -1;
                const bool nan = S != S;
                a.top_ids[r * a.top + k] = nan ? -1 : id;
                a.top_logp[r * a.top + k] = nan ? NAN : id < 0 ? -INFINITY : (to_f32(x[id]) - m) * a.rt - LN2 * l2;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(SC_TPB) distill_fwd_kernel(ScoreArgs a) {
    __shared__ float scratch[SC_NW];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        float m, S, W;
        row_sums(a, x, scratch, m, S, W);
        const float l2 = S == 0.f ? INFINITY : log2f(S);
        float mt = -FLT_MAX;
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
            if (id >= 0) mt = fmaxf(mt, load_any(a.teacher, a.t_type, r * a.n_ids + k));
            if (id >= a.c && a.id_status) flag_bad_id(a.id_status);
        }
        mt = block_max<SC_NW>(mt, scratch);
        float st = 0.f;
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
            if (id >= 0) st += exp2f((load_any(a.teacher, a.t_type, r * a.n_ids + k) - mt) * a.c2);
        }
        st = block_sum<SC_NW>(st, scratch);
        const float lt = st == 0.f ? INFINITY : log2f(st);
        float loss = 0.f;
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
            if (id < 0) continue;
            const float zt = load_any(a.teacher, a.t_type, r * a.n_ids + k) - mt;
            const float q = exp2f(zt * a.c2 - lt);
            const float lp = id < a.c ? (to_f32(x[id]) - m) * a.rt - LN2 * l2 : NAN;
            if (!(q == 0.f)) loss = fmaf(q, (zt * a.rt - LN2 * lt) - lp, loss);
        }
        loss = block_sum<SC_NW>(loss, scratch) * (a.t * a.t);
        if (threadIdx.x == 0) {
            a.loss[r] = loss;
            if (a.stats) {
                a.stats[4 * r + 0] = m;
                a.stats[4 * r + 1] = l2;
                a.stats[4 * r + 2] = mt;
                a.stats[4 * r + 3] = lt;
            }
        }
    }
}

// one row: p and its part of the gradient everywhere, then the listed ids' values again with what they add
template <typename T, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB) score_bwd_kernel(ScoreArgs a) {
    __shared__ float scratch[SC_NW];
    __shared__ int32_t s_id[SC_MAX_IDS];
    __shared__ float s_g[SC_MAX_IDS];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        T* dx = (T*)a.dx + r * a.c;
        const float m = a.stats[(DISTILL ? 4 : 2) * r], l2 = a.stats[(DISTILL ? 4 : 2) * r + 1];
        const bool none = l2 == INFINITY;
        __syncthreads();                                // the row before is done with s_id, s_g
        float sum = 0.f;
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
            const bool in = id >= 0 && id < a.c && !none;
            float g = 0.f;
            if (DISTILL) {
                if (id >= 0) g = exp2f((load_any(a.teacher, a.t_type, r * a.n_ids + k) - a.stats[4 * r + 2]) * a.c2 - a.stats[4 * r + 3]);
            } else if (in && a.g_logp) {
                g = a.g_logp[r * a.n_ids + k];
                sum += g;
            }
            s_id[k] = in ? (int32_t)id : -1;
            s_g[k] = g;
        }
        // dx = A p + B p (log2 p + H2) + (the listed ids) * u
        float A, B = 0.f, H2 = 0.f, u;
        if (DISTILL) {
            u = -a.g_logp[r] * a.t;
            const float lt = a.stats[4 * r + 3];
            A = lt == INFINITY ? 0.f : -u + (lt - lt);     // a teacher without a distribution (NaN) has no gradient either
        } else {
            A = -block_sum<SC_NW>(sum, scratch) / a.t;
            u = 1.f / a.t;
            if (a.g_entropy) {
                B = -a.g_entropy[r] * LN2 / a.t;
                H2 = a.entropy[r] / LN2;
            }
        }
        __syncthreads();
        auto base = [&](float xv) {
            const float lp = (xv - m) * a.c2 - l2;
            return exp2f(lp) * fmaf(B, fmaxf(lp, Z_FLOOR) + H2, A);
        };
        for (int i = threadIdx.x; i < a.c; i += SC_TPB) dx[i] = from_f32<T>(base(to_f32(x[i])));
        __syncthreads();
        for (int k = threadIdx.x; k < a.n_ids; k += SC_TPB) {
            const int32_t id = s_id[k];
            if (id < 0) continue;
            float g = s_g[k];
            bool first = true;
            for (int j = 0; j < k; ++j) first = first && s_id[j] != id;
            if (!first) continue;                       // the first slot of an id adds up all of them, in order
            for (int j = k + 1; j < a.n_ids; ++j) g += s_id[j] == id ? s_g[j] : 0.f;
            dx[id] = from_f32<T>(fmaf(g, u, base(to_f32(x[id]))));
        }
    }
}

static int score_common(ScoreArgs& a, int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t c,
                        int x_type, const void* x, float t, int64_t n_ids, const void* ids, int id_type) {
    if (rows < 0 || inner < 0 || c <= 0 || n_ids < 0 || !row_type_ok(x_type)) return ARMNET_ERR_BAD_ARG;
    if (id_type != ARMNET_ID_I64 && id_type != ARMNET_ID_I32) return ARMNET_ERR_BAD_ARG;
    if (!(t >= 1e-6f && t <= 1e6f)) return ARMNET_ERR_BAD_ARG;
    if (rows >= ((int64_t)1 << 31) || c >= ((int64_t)1 << 31) || n_ids > SC_MAX_IDS) return ARMNET_ERR_UNSUPPORTED;
    if (rows > 0 && (!x || (n_ids > 0 && !ids))) return ARMNET_ERR_BAD_ARG;
    a.rows = rows; a.c = (int)c;
    a.x = RowView{x, inner, outer_stride, row_stride};
    a.t = t; a.rt = (float)(1.0 / (double)t); a.c2 = (float)(1.4426950408889634 / (double)t);
    a.n_ids = (int)n_ids; a.ids = ids; a.id_type = id_type;
    return ARMNET_OK;
}

}  // namespace armnet

using namespace armnet;

extern "C" {

int64_t armnet_score_ws_bytes(int64_t rows, int64_t c, int top) {
    if (rows < 0 || c <= 0 || top < 0) return -1;
    return 0;
}

int armnet_score_logprobs_fwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t c, int x_type,
                              const void* x, float temperature, int64_t n_ids, const void* ids, int id_type, int top,
                              float* logp, float* entropy, float* top_logp, int64_t* top_ids, float* stats, void* workspace,
                              int64_t ws_bytes, int32_t* id_status, void* stream) {
    ScoreArgs a{};
    const int rc = score_common(a, rows, inner, outer_stride, row_stride, c, x_type, x, temperature, n_ids, ids, id_type);
    if (rc != ARMNET_OK) return rc;
    if (top < 0 || top > c) return ARMNET_ERR_BAD_ARG;
    if (top > SC_MAX_TOP) return ARMNET_ERR_UNSUPPORTED;
    if (rows == 0) return ARMNET_OK;
    if ((n_ids > 0 && !logp) || (top > 0 && (!top_logp || !top_ids))) return ARMNET_ERR_BAD_ARG;
    a.logp = logp; a.entropy = entropy; a.top = top; a.top_logp = top_logp; a.top_ids = top_ids; a.stats = stats;
    a.id_status = id_status;
    ARMNET_ROW_TYPE(x_type, T, (score_fwd_kernel<T><<<row_grid(rows), SC_TPB, 0, (hipStream_t)stream>>>(a)));
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

int armnet_score_logprobs_bwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t c, int x_type,
                              const void* x, float temperature, int64_t n_ids, const void* ids, int id_type,
                              const float* stats, const float* entropy, const float* g_logp, const float* g_entropy, void* dx,
                              void* stream) {
    ScoreArgs a{};
    const int rc = score_common(a, rows, inner, outer_stride, row_stride, c, x_type, x, temperature, n_ids, ids, id_type);
    if (rc != ARMNET_OK) return rc;
    if (rows == 0) return ARMNET_OK;
    if (!stats || !dx || (g_entropy && !entropy)) return ARMNET_ERR_BAD_ARG;
    a.stats = (float*)stats; a.entropy = (float*)entropy; a.g_logp = g_logp; a.g_entropy = g_entropy; a.dx = dx;
    ARMNET_ROW_TYPE(x_type, T, (score_bwd_kernel<T, false><<<row_grid(rows), SC_TPB, 0, (hipStream_t)stream>>>(a)));
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

int armnet_distill_fwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t c, int x_type,
                       const void* x, float temperature, int64_t k, const void* ids, int id_type, int t_type,
                       const void* teacher, float* loss, float* stats, void* workspace, int64_t ws_bytes, int32_t* id_status,
                       void* stream) {
    ScoreArgs a{};
    const int rc = score_common(a, rows, inner, outer_stride, row_stride, c, x_type, x, temperature, k, ids, id_type);
    if (rc != ARMNET_OK) return rc;
    if (k < 1 || !row_type_ok(t_type)) return ARMNET_ERR_BAD_ARG;
    if (rows == 0) return ARMNET_OK;
    if (!teacher || !loss) return ARMNET_ERR_BAD_ARG;
    a.teacher = teacher; a.t_type = t_type; a.loss = loss; a.stats = stats; a.id_status = id_status;
    ARMNET_ROW_TYPE(x_type, T, (distill_fwd_kernel<T><<<row_grid(rows), SC_TPB, 0, (hipStream_t)stream>>>(a)));
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

int armnet_distill_bwd(int64_t rows, int64_t inner, int64_t outer_stride, int64_t row_stride, int64_t c, int x_type,
                       const void* x, float temperature, int64_t k, const void* ids, int id_type, int t_type,
                       const void* teacher, const float* stats, const float* g_loss, void* dx, void* stream) {
    ScoreArgs a{};
    const int rc = score_common(a, rows, inner, outer_stride, row_stride, c, x_type, x, temperature, k, ids, id_type);
    if (rc != ARMNET_OK) return rc;
    if (k < 1 || !row_type_ok(t_type)) return ARMNET_ERR_BAD_ARG;
    if (rows == 0) return ARMNET_OK;
    if (!teacher || !stats || !g_loss || !dx) return ARMNET_ERR_BAD_ARG;
    a.teacher = teacher; a.t_type = t_type; a.stats = (float*)stats; a.g_logp = g_loss; a.dx = dx;
    ARMNET_ROW_TYPE(x_type, T, (score_bwd_kernel<T, true><<<row_grid(rows), SC_TPB, 0, (hipStream_t)stream>>>(a)));
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
}

}  // extern "C"
