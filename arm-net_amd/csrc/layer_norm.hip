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

__device__ __forceinline__ void store_param(void* p, int type, int i, float v) {
    if (type == ARMNET_F32) ((float*)p)[i] = v;
    else if (type == ARMNET_BF16) ((bf16_t*)p)[i] = (bf16_t)v;
    else ((f16_t*)p)[i] = (f16_t)v;
}

// The elements of a row that a lane holds: NV pieces of V.  Piece i is [at, at + V) with at = (i * NT + tid) * V; past the row's
// end it is pulled back to the row's last V elements, so that every load is a whole one inside the row, and only the elements from
// `lo` on are the lane's own (all: 0, none: V).  Rows shorter than V (one lane each) are read element by element.
template <typename T, int NT, int NV>
struct Columns {
    static constexpr int V = Piece<T>::N;
    int off[NV], lo[NV];
    bool tiny;
    int d;
    __device__ __forceinline__ Columns(int d_, int tid) : d(d_) {
        tiny = NT == 1 && d < V;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (i * NT + tid) * V;
            off[i] = at + V <= d ? at : (d < V ? 0 : d - V);
            lo[i] = at - off[i] < V ? at - off[i] : V;
        }
    }
    __device__ __forceinline__ void load(const T* row, u32x4 (&raw)[NV]) const {
        if (NT == 1 && tiny) {
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = e < d ? to_f32(row[e]) : 0.f;
            raw[0] = Piece<T>::pack(f);
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = Piece<T>::load(row + off[i]);
    }
    // what is not the lane's own counts as 0 in sums
    __device__ __forceinline__ void own(int i, float (&f)[V]) const {
        if (NT == 1) {
            if (tiny)
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] = e < d ? f[e] : 0.f;
        } else if (lo[i]) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = e >= lo[i] ? f[e] : 0.f;
        }
    }
    __device__ __forceinline__ bool whole(int i) const { return NT == 1 ? !tiny : lo[i] == 0; }
    __device__ __forceinline__ bool has(int i, int e) const { return NT == 1 ? !tiny || e < d : e >= lo[i]; }
    __device__ __forceinline__ void store(T* row, int i, const float (&f)[V]) const {
        if (whole(i)) {
            Piece<T>::store(row + off[i], Piece<T>::pack(f));
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (has(i, e)) row[off[i] + e] = from_f32<T>(f[e]);
        }
    }
    // a parameter's values, `fill` without one
    template <typename W>
    __device__ __forceinline__ void param_of(const W* p, float (&f)[NV][V]) const {
        if (NT == 1 && tiny) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[0][e] = e < d ? to_f32(p[e]) : 0.f;
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; e += Piece<W>::N) {
                if constexpr (Piece<W>::N <= V) {
                    Piece<W>::unpack(Piece<W>::load(p + off[i] + e), *(float(*)[Piece<W>::N])(f[i] + e));
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) f[i][k] = to_f32(p[off[i] + k]);
                }
            }
    }
    __device__ __forceinline__ void param(const void* p, int type, float fill, float (&f)[NV][V]) const {
        if (!p) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) f[i][e] = fill;
        } else if (type == ARMNET_F32) {
            param_of((const float*)p, f);
        } else if (type == ARMNET_BF16) {
            param_of((const bf16_t*)p, f);
        } else {
            param_of((const f16_t*)p, f);
        }
    }
};

// sum over the lanes (and waves) that hold a row, in each of them; scratch: one float a wave, of this sum alone
template <int LPR, int NW>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    if constexpr (LPR < WAVE) return lanes_sum<LPR>(v);
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

// One row group: LPR lanes (NW = 1) or NW waves.  A block holds TPB / (LPR or NW * 64) of them and goes on to further rows; the next
// row is asked for as soon as this one is unpacked, into the same registers.  Bound by memory: called again and again 65536 x 512 f32
// takes 50 us (5.4 TB/s), 16384 x 4096 bf16 47 (5.8), 8000 x 8192 bf16 44 (5.9; a large copy moves 5.2), behind a backward 55, 49 and
// 46; rows whose length is no multiple of 16 bytes are slower (10007 x 2049 f16, whose last piece keeps another half of the block busy:
// 22 us, 3.7 TB/s).
template <typename T, int LPR, int NW, int NV, int TPB>
__global__ void __launch_bounds__(TPB) norm_fwd_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N, NT = LPR < WAVE ? LPR : NW * WAVE, GROUPS = TPB / NT;
    __shared__ float scratch[2][TPB / WAVE];
    const int group = threadIdx.x / NT, tid = threadIdx.x & (NT - 1);
    const Columns<T, NT, NV> cols(a.d, tid);
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int64_t rounds = (a.rows + step - 1) / step;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    u32x4 raw[NV];
    cols.load(row_ptr<T>(a.x, r < a.rows ? r : a.rows - 1), raw);
    float w[NV][V], b[NV][V];
    cols.param(a.weight, a.w_type, 1.f, w);
    cols.param(a.bias, a.w_type, 0.f, b);
    for (int64_t k = 0; k < rounds; ++k, r += step) {
        float f[NV][V];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Piece<T>::unpack(raw[i], f[i]);
            cols.own(i, f[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[i][e];
        }
        if (k + 1 < rounds) cols.load(row_ptr<T>(a.x, r + step < a.rows ? r + step : a.rows - 1), raw);
        const float mean = row_sum<LPR, NW>(s, scratch[0]) / (float)a.d;     // a division: one rounding less
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[i][e] -= mean;
            cols.own(i, f[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) q = fmaf(f[i][e], f[i][e], q);
        }
        const float rstd = 1.f / sqrtf(row_sum<LPR, NW>(q, scratch[1]) / (float)a.d + a.eps);
        if (r < a.rows) {
            T* y = (T*)a.out + r * a.d;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) f[i][e] = fmaf(f[i][e] * rstd, w[i][e], b[i][e]);
                cols.store(y, i, f[i]);
            }
            if (tid == 0 && a.mean) {
                a.mean[r] = mean;
                a.rstd[r] = rstd;
            }
        }
    }
}

// A lane's own values between the rows, in LDS instead of registers: [NV][V] floats as 16-byte cells, nobody else's.
template <int NV, int V, int TPB>
struct LaneCells {
    static constexpr int N = NV * V / 4;
    static __device__ __forceinline__ void put(float4 (*cells)[TPB], int i, const float (&f)[V]) {
#pragma unroll
        for (int e = 0; e < V; e += 4) cells[(i * V + e) / 4][threadIdx.x] = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
    static __device__ __forceinline__ void put(float4 (*cells)[TPB], const float (&f)[NV][V]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) put(cells, i, f[i]);
    }
    static __device__ __forceinline__ void get(const float4 (*cells)[TPB], int i, float (&f)[V]) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 q = cells[(i * V + e) / 4][threadIdx.x];
            f[e] = q.x, f[e + 1] = q.y, f[e + 2] = q.z, f[e + 3] = q.w;
        }
    }
};

// dx of a row, and the block's share of dw and db: in registers over its rows, then over its groups through LDS.  x and dy are read
// once for all three.  Bound by memory: behind its forward 65536 x 512 f32 takes 79 us (5.1 TB/s), 16384 x 4096 bf16 80 (5.0), 8000 x 8192
// bf16 77 (5.1), and norm_param_kernel 5 more; of more than 8192 values less (1500 x 16384 f32 68 + 7, 4.4 TB/s): one row a CU is in
// work, one on its way.  A few hundred long rows cost what the blocks' shares cost (1000 x 10000 bf16: 20 + 5 us where reading and writing
// the rows takes 12; 35 in all with the shares stored value by value).
// KEEP: what waits in LDS between the rows instead of in registers: 0 nothing, 1 the weights, 2 the sums for dw too.
template <typename T, int LPR, int NW, int NV, int TPB, int KEEP>
__global__ void __launch_bounds__(TPB) norm_bwd_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N, NT = LPR < WAVE ? LPR : NW * WAVE, GROUPS = TPB / NT;
    __shared__ float scratch[2][2][TPB / WAVE];
    constexpr int SHARES = LPR < WAVE ? TPB / WAVE : GROUPS;     // short rows: a wave's groups meet in registers
    __shared__ float sums[2][SHARES > 1 ? NV * NT * V : 1];
    using Cells = LaneCells<NV, V, TPB>;
    __shared__ float4 w_cells[KEEP >= 1 ? Cells::N : 1][KEEP >= 1 ? TPB : 1], dw_cells[KEEP >= 2 ? Cells::N : 1][KEEP >= 2 ? TPB : 1];
    const int group = threadIdx.x / NT, tid = threadIdx.x & (NT - 1);
    const Columns<T, NT, NV> cols(a.d, tid);
    const float rd = 1.f / (float)a.d;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const int64_t rounds = (a.rows + step - 1) / step;
    u32x4 rx[NV], ry[NV];
    float mean, rstd;
    auto load = [&](int64_t r) {                       // a group without a row works on the last one's values and drops them
        const int64_t q = r < a.rows ? r : a.rows - 1;
        cols.load(row_ptr<T>(a.x, q), rx);
        cols.load((const T*)a.dy + q * a.d, ry);
        mean = a.mean[q];
        rstd = a.rstd[q];
    };
    // the forward's last rows first: some are still in the last-level cache
    int64_t r = (rounds - 1) * step + (int64_t)blockIdx.x * GROUPS + group;
    load(r);
    float w[NV][V], dw[NV][V] = {}, db[NV][V] = {};
    cols.param(a.weight, a.w_type, 1.f, w);
    if constexpr (KEEP >= 1) Cells::put(w_cells, w);
    if constexpr (KEEP >= 2) Cells::put(dw_cells, dw);
    for (int64_t k = 0; k < rounds; ++k, r -= step) {
        const bool in = r < a.rows;
        const float rs = rstd;
        float h[NV][V], g[NV][V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Piece<T>::unpack(rx[i], h[i]);
            Piece<T>::unpack(ry[i], g[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) h[i][e] = (h[i][e] - mean) * rs;
            cols.own(i, g[i]);                         // 0 in g makes 0 of everything below
        }
        if (k + 1 < rounds) load(r - step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (KEEP >= 1) Cells::get(w_cells, i, w[i]);
            if constexpr (KEEP >= 2) Cells::get(dw_cells, i, dw[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (in) {
                    dw[i][e] = fmaf(g[i][e], h[i][e], dw[i][e]);
                    db[i][e] += g[i][e];
                }
                g[i][e] *= w[i][e];
                s1 += g[i][e];
                s2 = fmaf(g[i][e], h[i][e], s2);
            }
            if constexpr (KEEP >= 2) Cells::put(dw_cells, i, dw[i]);
        }
        if (a.out) {
            float m1, m2;
            if constexpr (NW == 1) {
                m1 = row_sum<LPR, NW>(s1, nullptr) * rd;
                m2 = row_sum<LPR, NW>(s2, nullptr) * rd;
            } else {                                   // both through one barrier; the next row takes the other scratch
                float(*sc)[TPB / WAVE] = scratch[k & 1];
                const int wave = threadIdx.x / WAVE;
                s1 = wave_sum(s1);
                s2 = wave_sum(s2);
                if ((threadIdx.x & (WAVE - 1)) == 0) {
                    sc[0][wave] = s1;
                    sc[1][wave] = s2;
                }
                __syncthreads();
                m1 = m2 = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    m1 += sc[0][wave / NW * NW + i];
                    m2 += sc[1][wave / NW * NW + i];
                }
                m1 *= rd;
                m2 *= rd;
            }
            if (in) {
                T* dx = (T*)a.out + r * a.d;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
#pragma unroll
                    for (int e = 0; e < V; ++e) g[i][e] = rs * (g[i][e] - m1 - h[i][e] * m2);
                    cols.store(dx, i, g[i]);
                }
            }
        }
    }
    if (!a.params) return;
    if constexpr (KEEP >= 2)
#pragma unroll
        for (int i = 0; i < NV; ++i) Cells::get(dw_cells, i, dw[i]);
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
        for (int i = 0; i < NV; ++i) {
            float* part = a.partial + (int64_t)blockIdx.x * 2 * a.d + cols.off[i];
            if (a.blocks > 1 && cols.whole(i)) {
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    Piece<float>::store(part + e, Piece<float>::pack(*(float(*)[4])(dw[i] + e)));
                    Piece<float>::store(part + a.d + e, Piece<float>::pack(*(float(*)[4])(db[i] + e)));
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (!cols.has(i, e)) continue;
                if (a.blocks == 1) {
                    if (a.dweight) store_param(a.dweight, a.w_type, cols.off[i] + e, dw[i][e]);
                    if (a.dbias) store_param(a.dbias, a.w_type, cols.off[i] + e, db[i][e]);
                } else {
                    part[e] = dw[i][e];
                    part[a.d + e] = db[i][e];
                }
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
//
// Bound by reading a row three times (of which the caches serve a part): 1000 x 20000 f32 forward in 45 us, 3.5 TB/s of what it cannot
// do without (52 behind a backward); backward, with the parameters' gradients in a pass of their own, 61 + 29 + 7 us, 2.5 TB/s.

constexpr int LN_LONG_TPB = 1024, LN_LONG_NW = LN_LONG_TPB / WAVE;

// n elements of a piece, 0 for the others
template <typename T>
__device__ __forceinline__ void load_n(const T* p, int n, float (&f)[Piece<T>::N]) {
    if (n == Piece<T>::N) {
        Piece<T>::unpack(Piece<T>::load(p), f);
    } else {
#pragma unroll
        for (int e = 0; e < Piece<T>::N; ++e) f[e] = e < n ? to_f32(p[e]) : 0.f;
    }
}

// f(elements, first column, how many of them) for the pieces of a row of d elements that this thread owns
template <typename T, typename F>
__device__ __forceinline__ void for_pieces(const T* x, int d, F f) {
    constexpr int V = Piece<T>::N;
    const int nvec = d / V;
    int j = threadIdx.x;
    for (; j + 3 * LN_LONG_TPB < nvec; j += 4 * LN_LONG_TPB) {
        u32x4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = Piece<T>::load(x + (int64_t)(j + u * LN_LONG_TPB) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float v[V];
            Piece<T>::unpack(raw[u], v);
            f(v, (j + u * LN_LONG_TPB) * V, V);
        }
    }
    for (; j <= nvec; j += LN_LONG_TPB) {
        const int n = j < nvec ? V : d - nvec * V;
        if (n == 0) break;
        float v[V];
        load_n(x + (int64_t)j * V, n, v);
        f(v, j * V, n);
    }
}

template <typename T>
__device__ __forceinline__ void store_n(T* p, int n, const float (&f)[Piece<T>::N]) {
    if (n == Piece<T>::N) {
        Piece<T>::store(p, Piece<T>::pack(f));
    } else {
#pragma unroll
        for (int e = 0; e < Piece<T>::N; ++e)
            if (e < n) p[e] = from_f32<T>(f[e]);
    }
}

// n of a parameter's values from column `at` on, `fill` without one
template <int V>
__device__ __forceinline__ void load_params(const void* p, int type, int at, int n, float fill, float (&f)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = fill;
    if (!p) return;
    if (type == ARMNET_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = ((const float*)p)[at + (e < n ? e : 0)];
    } else if (type == ARMNET_BF16) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = to_f32(((const bf16_t*)p)[at + (e < n ? e : 0)]);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = to_f32(((const f16_t*)p)[at + (e < n ? e : 0)]);
    }
}

template <typename T>
__global__ void __launch_bounds__(LN_LONG_TPB) norm_long_fwd_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N;
    __shared__ float scratch[LN_LONG_NW];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        T* y = (T*)a.out + r * a.d;
        float s = 0.f;
        for_pieces(x, a.d, [&](const float (&v)[V], int, int) {
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[e];
        });
        const float mean = block_sum<LN_LONG_NW>(s, scratch) / (float)a.d;
        float q = 0.f;
        for_pieces(x, a.d, [&](const float (&v)[V], int, int n) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float c = e < n ? v[e] - mean : 0.f;
                q = fmaf(c, c, q);
            }
        });
        const float rstd = 1.f / sqrtf(block_sum<LN_LONG_NW>(q, scratch) / (float)a.d + a.eps);
        for_pieces(x, a.d, [&](const float (&v)[V], int at, int n) {
            float o[V], w[V], b[V];
            load_params(a.weight, a.w_type, at, n, 1.f, w);
            load_params(a.bias, a.w_type, at, n, 0.f, b);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf((v[e] - mean) * rstd, w[e], b[e]);
            store_n(y + at, n, o);
        });
        if (threadIdx.x == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LN_LONG_TPB) norm_long_dx_kernel(NormArgs a) {
    constexpr int V = Piece<T>::N;
    __shared__ float scratch[LN_LONG_NW];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        const T* dy = (const T*)a.dy + r * a.d;
        T* dx = (T*)a.out + r * a.d;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        auto both = [&](const float (&v)[V], int at, int n, float (&g)[V], float (&h)[V]) {
            float w[V];
            load_n(dy + at, n, g);                     // 0 past the end
            load_params(a.weight, a.w_type, at, n, 1.f, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                g[e] *= w[e];
                h[e] = (v[e] - mean) * rstd;
            }
        };
        for_pieces(x, a.d, [&](const float (&v)[V], int at, int n) {
            float g[V], h[V];
            both(v, at, n, g, h);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s1 += g[e];
                s2 = fmaf(g[e], h[e], s2);
            }
        });
        const float m1 = block_sum<LN_LONG_NW>(s1, scratch) / (float)a.d;
        const float m2 = block_sum<LN_LONG_NW>(s2, scratch) / (float)a.d;
        for_pieces(x, a.d, [&](const float (&v)[V], int at, int n) {
            float g[V], h[V];
            both(v, at, n, g, h);
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = rstd * (g[e] - m1 - h[e] * m2);
            store_n(dx + at, n, g);
        });
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
#pragma unroll 4
    for (int64_t r = r0; r < r1; ++r) {
        const float g = to_f32(((const T*)a.dy)[r * a.d + i]);
        sw = fmaf(g, (to_f32(row_ptr<T>(a.x, r)[i]) - a.mean[r]) * a.rstd[r], sw);
        sb += g;
    }
    a.partial[((int64_t)blockIdx.y * 2 + 0) * a.d + i] = sw;
    a.partial[((int64_t)blockIdx.y * 2 + 1) * a.d + i] = sb;
}

// ---- launches ------------------------------------------------------------------------------------------------------------

// Who holds a row of `np` 16-byte pieces: lpr lanes of a wave or nw waves, nv pieces a lane; tpb threads a block.
struct NormShape {
    int lpr, nw, nv, tpb;
};

// Few pieces a lane keep everything in registers.  A barrier's cost grows with the waves that meet at it.
static NormShape norm_fwd_shape(int64_t np) {
    if (np <= WAVE) {
        int lpr = 1;
        while (lpr < np) lpr *= 2;
        return {lpr, 1, 1, LN_TPB};
    }
    if (np <= 128) return {WAVE, 1, 2, LN_TPB};
    if (np <= 256) return {WAVE, 4, 1, LN_TPB};
    if (np <= 512) return {WAVE, 4, 2, LN_TPB};        // (16384 x 4096 bf16: 47 us; eight waves with one piece a lane 55)
    if (np <= 1024) return {WAVE, 8, 2, 512};          // (8000 x 8192 bf16: 44 us; sixteen waves with one piece a lane 65)
    if (np <= 2048) return {WAVE, 16, 2, 1024};
    return {WAVE, 16, 4, 1024};
}

// The backward keeps five values of a column (w, h, g and two sums): one piece a lane, then more registers a lane in smaller blocks.
static NormShape norm_bwd_shape(int64_t np, int v) {
    if (np <= WAVE) {
        int lpr = 1;
        while (lpr < np) lpr *= 2;
        return {lpr, 1, 1, 1024};
    }
    if (np <= 128) return v == 4 ? NormShape{WAVE, 1, 2, 1024} : NormShape{WAVE, 2, 1, 1024};
    if (np <= 256) return {WAVE, 4, 1, 1024};
    if (np <= 512) return {WAVE, 8, 1, 1024};
    if (np <= 1024) return {WAVE, 16, 1, 1024};
    if (np <= 2048) return v == 4 ? NormShape{WAVE, 16, 2, 1024} : NormShape{WAVE, 8, 4, 512};
    return {WAVE, 8, 8, 512};
}

static int64_t norm_groups(const NormShape& s) { return s.tpb / (s.lpr < WAVE ? s.lpr : s.nw * WAVE); }

// Blocks of the backward, one a unit: its waves with a row in work and one on its way each keep enough bytes in flight, and fewer
// blocks mean fewer shares of the parameters' gradients to add up.
static int norm_blocks(int64_t rows, int64_t d, int v) {
    if (d > LN_MAX_D) return (int)(rows < 256 ? rows : 256);
    const int64_t groups = norm_groups(norm_bwd_shape((d + v - 1) / v, v));
    const int64_t n = (rows + groups - 1) / groups;
    return (int)(n < 256 ? n : 256);
}

template <typename T, int LPR, int NW, int NV, int TPB>
static bool try_norm_fwd(const NormShape& s, const NormArgs& a, hipStream_t st) {
    if (s.lpr != LPR || s.nw != NW || s.nv != NV || s.tpb != TPB) return false;
    const int64_t groups = norm_groups(s), most = (int64_t)device_cu_count() * (2048 / TPB);
    int64_t blocks = (a.rows + groups - 1) / groups;
    if (blocks > most) blocks = most;
    norm_fwd_kernel<T, LPR, NW, NV, TPB><<<(unsigned)blocks, TPB, 0, st>>>(a);
    return true;
}

template <typename T, int LPR, int NW, int NV, int TPB>
static bool try_norm_bwd(const NormShape& s, const NormArgs& a, hipStream_t st) {
    if (s.lpr != LPR || s.nw != NW || s.nv != NV || s.tpb != TPB) return false;
    // 32 values a lane do not fit its registers, least of all in float32, whose row on its way is as large as the one in work
    // (1500 x 16384 f32: the weights in LDS take 24 us off, dw another 26; 4000 x 12288 bf16: 7 and 0)
    constexpr int KEEP = NV * Piece<T>::N < 32 ? 0 : Piece<T>::N == 4 ? 2 : 1;
    norm_bwd_kernel<T, LPR, NW, NV, TPB, KEEP><<<a.blocks, TPB, 0, st>>>(a);
    return true;
}

template <typename T>
static bool launch_norm_fwd(const NormArgs& a, hipStream_t st) {
    const NormShape s = norm_fwd_shape((a.d + Piece<T>::N - 1) / Piece<T>::N);
    if (try_norm_fwd<T, 1, 1, 1, 256>(s, a, st) || try_norm_fwd<T, 2, 1, 1, 256>(s, a, st) || try_norm_fwd<T, 4, 1, 1, 256>(s, a, st) ||
        try_norm_fwd<T, 8, 1, 1, 256>(s, a, st) || try_norm_fwd<T, 16, 1, 1, 256>(s, a, st) || try_norm_fwd<T, 32, 1, 1, 256>(s, a, st) ||
        try_norm_fwd<T, 64, 1, 1, 256>(s, a, st) || try_norm_fwd<T, 64, 1, 2, 256>(s, a, st) || try_norm_fwd<T, 64, 4, 1, 256>(s, a, st) ||
        try_norm_fwd<T, 64, 4, 2, 256>(s, a, st) || try_norm_fwd<T, 64, 8, 2, 512>(s, a, st) ||
        try_norm_fwd<T, 64, 16, 2, 1024>(s, a, st))
        return true;
    if constexpr (sizeof(T) == 4) return try_norm_fwd<T, 64, 16, 4, 1024>(s, a, st);
    return false;
}

template <typename T>
static bool launch_norm_bwd(const NormArgs& a, hipStream_t st) {
    constexpr int V = Piece<T>::N;
    const NormShape s = norm_bwd_shape((a.d + V - 1) / V, V);
    if (try_norm_bwd<T, 1, 1, 1, 1024>(s, a, st) || try_norm_bwd<T, 2, 1, 1, 1024>(s, a, st) || try_norm_bwd<T, 4, 1, 1, 1024>(s, a, st) ||
        try_norm_bwd<T, 8, 1, 1, 1024>(s, a, st) || try_norm_bwd<T, 16, 1, 1, 1024>(s, a, st) || try_norm_bwd<T, 32, 1, 1, 1024>(s, a, st) ||
        try_norm_bwd<T, 64, 1, 1, 1024>(s, a, st) || try_norm_bwd<T, 64, 4, 1, 1024>(s, a, st) || try_norm_bwd<T, 64, 8, 1, 1024>(s, a, st) ||
        try_norm_bwd<T, 64, 16, 1, 1024>(s, a, st))
        return true;
    if constexpr (sizeof(T) == 4)
        return try_norm_bwd<T, 64, 1, 2, 1024>(s, a, st) || try_norm_bwd<T, 64, 16, 2, 1024>(s, a, st) || try_norm_bwd<T, 64, 8, 8, 512>(s, a, st);
    else
        return try_norm_bwd<T, 64, 2, 1, 1024>(s, a, st) || try_norm_bwd<T, 64, 8, 4, 512>(s, a, st);
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
        bool there = false;
        ARMNET_ROW_TYPE(x_type, T, there = launch_norm_fwd<T>(a, st));
        if (!there) return ARMNET_ERR_UNSUPPORTED;
    } else {
        ARMNET_ROW_TYPE(x_type, T, (norm_long_fwd_kernel<T><<<row_grid(rows), LN_LONG_TPB, 0, st>>>(a)));
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
            bool there = false;
            ARMNET_ROW_TYPE(x_type, T, there = launch_norm_bwd<T>(a, st));
            if (!there) return ARMNET_ERR_UNSUPPORTED;
            ARMNET_LAUNCH_CHECK();
            if (a.blocks == 1) return ARMNET_OK;                     // the one block has written the parameters' gradients
        } else {
            if (dx) {
                ARMNET_ROW_TYPE(x_type, T, (norm_long_dx_kernel<T><<<row_grid(rows), LN_LONG_TPB, 0, st>>>(a)));
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
