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
// (x - m) / T - ln2 log2 S, as far as fp32 reaches.  Gradients are rounded once, to x's type.  m starts at the lowest finite
// number instead of -inf: a masked score (-inf) then has z = -inf and e^z = 0 without a special case, a row of the lowest number
// has p = 1/C, and S = 0 says that nothing in the row is above -inf.  (m, log2 S) go from the forward to the backward as two
// numbers: their sum would lose what m's magnitude takes.
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
    // a row in several slices
    int splits;
    int64_t per;               // scores of a slice
    int slots;                 // of a long list's table
    float4* part;              // [rows, splits]: m, S, W
    uint64_t* keys;            // [rows, splits, top], best first; 0: none
};

__device__ __forceinline__ int64_t load_id(const void* ids, int id_type, int64_t i) {
    return id_type == ARMNET_ID_I64 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (type == ARMNET_F32) return ((const float*)p)[i];
    if (type == ARMNET_BF16) return (float)((const bf16_t*)p)[i];
    return (float)((const f16_t*)p)[i];
}

// unsigned keys in the order of the values; -0 and 0 are the same value.  0 is below every key.
__device__ __forceinline__ uint32_t value_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// ... of (value, lowest id first)
__device__ __forceinline__ uint64_t score_key(float v, uint32_t id) { return ((uint64_t)value_key(v) << 32) | (uint32_t)~id; }

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }   // results below 2^-126 are 0

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

struct Sums {
    float m, S, W;             // largest score, sum of e^z, sum of e^z z2
};

// moves sums to another reference
template <bool ENT>
__device__ __forceinline__ void rebase(Sums& s, float m, float c2) {
    const float d = fmaxf((s.m - m) * c2, Z_FLOOR);
    const float f = exp2_raw(d);
    if constexpr (ENT) s.W = f * fmaf(d, s.S, s.W);
    s.S *= f;
    s.m = m;
}

// The largest score so far is the reference.  Returns the largest of these.
template <bool ENT, int N>
__device__ __forceinline__ float add_scores(Sums& s, const float (&v)[N], float c2) {
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, v[i]);
    rebase<ENT>(s, fmaxf(s.m, mx), c2);
    float e0 = 0.f, w0 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float z = (v[i] - s.m) * c2;
        const float e = exp2_raw(z);
        e0 += e;
        if constexpr (ENT) w0 = fmaf(e, fmaxf(z, Z_FLOOR), w0);
    }
    s.S += e0;
    if constexpr (ENT) s.W += w0;
    return mx;
}

// the largest score of a thread, the batch of pieces it is in (by its first piece; -1: behind the last piece) and the largest score
// of all other batches
struct Peak {
    float m1, m2;
    int at;
    __device__ __forceinline__ void add(float mx, int batch) {
        at = mx > m1 ? batch : at;
        m2 = __builtin_amdgcn_fmed3f(m1, m2, mx);
        m1 = fmaxf(m1, mx);
    }
};

// all threads' sums of a group, in every thread; scratch: 3 * NW floats of the group's own
template <int NW, bool ENT>
__device__ __forceinline__ Sums group_sums(Sums s, float c2, float* scratch) {
    rebase<ENT>(s, wave_max(s.m), c2);
    s.S = wave_sum(s.S);
    if constexpr (ENT) s.W = wave_sum(s.W);
    if constexpr (NW > 1) {
        const int w = threadIdx.x / WAVE;
        if ((threadIdx.x & (WAVE - 1)) == 0) {
            scratch[w] = s.m;
            scratch[NW + w] = s.S;
            scratch[2 * NW + w] = s.W;
        }
        __syncthreads();
        float m = scratch[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) m = fmaxf(m, scratch[i]);
        Sums t{m, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            Sums p{scratch[i], scratch[NW + i], scratch[2 * NW + i]};
            rebase<ENT>(p, m, c2);
            t.S += p.S;
            t.W += p.W;
        }
        return t;
    }
    return s;
}

constexpr int SC_UNROLL = 2;             // pieces of 16 bytes in flight a thread (2048 x 131072 bf16: 96 us; four 106)
constexpr int SC_BWD_UNROLL = 4;         // ... in the backward, which computes less and has no state to keep
constexpr int SC_BUF = 512;              // candidates for the alternatives
// So few scores are all candidates (4618 x 73 with 48 alternatives: f32 11.4 us, by their bound 31.9; bf16 11.6 and 15.0)
constexpr int SC_FEW = 128;

template <int NW>
struct TopScratch {
    uint64_t key[SC_BUF + 8];
    int n, threads, first;
    uint32_t cut;
    int count[NW];
    uint8_t who[NW * WAVE];
};

template <int NW>
__device__ __forceinline__ void push(TopScratch<NW>& ts, float v, uint32_t id) {
    const int at = atomicAdd(&ts.n, 1);
    if (at < SC_BUF) ts.key[at] = score_key(v, id);
}

// how many of a slice's scores are at least `cut`
template <typename T, int NW>
__device__ int count_from(const T* x, int n, float cut, int tid, TopScratch<NW>& ts) {
    int mine = 0;
    for (int i = tid; i < n; i += NW * WAVE) mine += to_f32(x[i]) >= cut ? 1 : 0;
    if (tid == 0) ts.first = 0;
    group_sync<NW>();
    atomicAdd(&ts.first, mine);
    group_sync<NW>();
    const int all = ts.first;
    group_sync<NW>();
    return all;
}

// The `top` best scores of a slice of n scores that begins at id `id0`, as keys in ts.key[0 .. result), unordered; the result is at
// most SC_BUF and covers the best ones.  pk: the peak of this thread, which owns the pieces tid, tid + NT, ...
//
// The top-th largest of the threads' largest scores is a bound: at least `top` scores reach it, and few more do (for scores in no
// particular order about top + top^2 / 2 NT).  A thread whose largest score reaches it reads the batch that holds it again; the few
// that have a second batch with such a score read all of theirs.  Where more than SC_BUF scores reach the bound (ties, or large
// scores that recur at a fixed distance), it is raised by halving until they fit; if ties remain, the ones with the lowest ids are
// taken.
template <typename T, int NW>
__device__ int best_scores(const T* x, int n, uint32_t id0, const Peak& pk, int top, int tid, TopScratch<NW>& ts) {
    constexpr int NT = NW * WAVE, V = Piece<T>::N, U = SC_UNROLL;
    const float m = pk.m1;
    const int lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int nvec = n / V, rem = n - nvec * V;
    if (n <= SC_FEW) {                   // all of them; a masked one is below every other and has no value
        for (int i = tid; i < n; i += NT) {
            const float v = to_f32(x[i]);
            ts.key[i] = v > -INFINITY ? score_key(v, id0 + i) : (uint64_t)~(id0 + i);
        }
        group_sync<NW>();
        return n;
    }
    float* maxima = (float*)ts.key;
    if constexpr (NW > 1) maxima[tid] = m;
    if (tid == 0) ts.n = ts.threads = 0;
    group_sync<NW>();
    constexpr int SPARE = sizeof(T) == 2 ? 13 : 0;                // of a 16-bit score's key the lower 13 bits say nothing
    if (wave == 0) {                     // between lo (reached by >= top threads) and hi (by fewer), until lo is close
        uint32_t k[NW];
        float mn = m, mx = m;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float v = NW > 1 ? maxima[i * WAVE + lane] : m;
            k[i] = value_key(v) >> SPARE;
            mn = fminf(mn, v);
            mx = fmaxf(mx, v);
        }
        uint32_t lo = value_key(-wave_max(-mn)) >> SPARE, hi = (value_key(wave_max(mx)) >> SPARE) + 1;
        int reach = NT;
        uint32_t mid = lo + 1;           // first: are there `top` threads at all above the least (those without a score)?
        while (hi - lo > 1 && reach > top + 8) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < NW; ++i) c += __popcll(__ballot(k[i] >= mid));
            if (c >= top) { lo = mid; reach = c; } else hi = mid;
            mid = lo + (hi - lo) / 2;
        }
        lo <<= SPARE;                    // a negative score's key ends in ones
        if (lane == 0) ts.cut = lo & 0x80000000u ? lo : lo | ((1u << SPARE) - 1);
    }
    group_sync<NW>();
    const uint32_t cut = ts.cut;
    const float cutv = key_value(cut);
    const int pieces = (nvec + NT - 1) / NT;
    auto candidates = [&](int at) {
        float f[V];
        Piece<T>::unpack(Piece<T>::load(x + (int64_t)at * V), f);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (f[e] >= cutv) push(ts, f[e], id0 + at * V + e);
    };
    if (m >= cutv) {
        if (pk.m2 < cutv) {
            if (pk.at >= 0)
                for (int u = 0; u < U; ++u)
                    if (pk.at + u * NT < nvec) candidates(pk.at + u * NT);
        } else {
            ts.who[atomicAdd(&ts.threads, 1)] = (uint8_t)tid;
        }
    }
    group_sync<NW>();
    const int threads = ts.threads;      // a wave reads what such a thread owns
    for (int w = wave; w < threads; w += NW)
        for (int j = lane; j < pieces; j += WAVE) {
            const int at = j * NT + ts.who[w];
            if (at < nvec) candidates(at);
        }
    if (tid < rem) {
        const float v = to_f32(x[nvec * V + tid]);
        if (v >= cutv) push(ts, v, id0 + nvec * V + tid);
    }
    group_sync<NW>();
    int got = ts.n;
    group_sync<NW>();
    if (got <= SC_BUF) return got;

    // too many: lo is reached by more than SC_BUF scores, hi by fewer than `top`
    uint32_t lo = cut, hi = 0xff800001u, mid = cut + 1;            // hi: above +inf
    bool fits = false;
    while (hi - lo > 1) {
        const int c = count_from<T, NW>(x, n, key_value(mid), tid, ts);
        if (c >= top) {
            lo = mid;
            if (c <= SC_BUF) { fits = true; break; }
        } else {
            hi = mid;
        }
        mid = lo + (hi - lo) / 2;
    }
    if (tid == 0) ts.n = 0;
    group_sync<NW>();
    const float from = key_value(fits ? lo : hi);
    for (int i = tid; i < n; i += NT) {
        const float v = to_f32(x[i]);
        if (v >= from) push(ts, v, id0 + i);
    }
    group_sync<NW>();
    got = ts.n;
    group_sync<NW>();
    if (!fits) {                                                   // ties at lo: the lowest ids, in order
        const float tie = key_value(lo);
        int need = top - got;
        for (int i0 = 0; i0 < n && need > 0; i0 += NT) {
            const int i = i0 + tid;
            const bool is = i < n && to_f32(x[i]) == tie;
            const uint64_t b = __ballot(is);
            int before = __popcll(b & ((1ull << lane) - 1)), all = __popcll(b);
            if constexpr (NW > 1) {
                if (lane == 0) ts.count[wave] = all;
                __syncthreads();
                all = 0;
                for (int w = 0; w < NW; ++w) {
                    if (w < wave) before += ts.count[w];
                    all += ts.count[w];
                }
                __syncthreads();
            }
            if (is && before < need) ts.key[got + before] = score_key(tie, id0 + i);
            const int took = all < need ? all : need;
            got += took;
            need -= took;
        }
        group_sync<NW>();
    }
    return got;
}

// What a row says, from its sums: log p of the ids, the entropy; or the distillation loss.  id, teacher, given: the thread's first
// slot (NT or, for the loss, 64 slots are held by the threads), the teacher's score of it and the row's
template <typename T, int NT, bool DISTILL>
__device__ __forceinline__ void row_answer(const ScoreArgs& a, int64_t r, const T* x, const Sums& s, int tid, int64_t id,
                                           float teacher, float given) {
    const bool some = !(s.S == 0.f);
    const float l2 = some ? log2f(s.S) : INFINITY;
    if constexpr (!DISTILL) {
        if (tid == 0) {
            if (a.entropy) a.entropy[r] = some ? LN2 * (l2 - s.W / s.S) : 0.f;
            if (a.stats) {
                a.stats[2 * r] = s.m;
                a.stats[2 * r + 1] = l2;
            }
        }
        for (int k = tid; k < a.n_ids; k += NT) {
            if (k != tid) {
                id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                if (id >= 0 && id < a.c) given = to_f32(x[id]);
            }
            float v = 0.f;
            if (id >= a.c) {
                v = NAN;
                if (a.id_status) flag_bad_id(a.id_status);
            } else if (id >= 0) {
                v = some ? (given - s.m) * a.rt - LN2 * l2 : -INFINITY;
            }
            a.logp[r * a.n_ids + k] = v;
        }
    } else if (tid < WAVE) {                          // the list is short: one wave reads it three times
        const int64_t id0 = id;
        const float t0 = teacher, x0 = given;
        auto slot = [&](int k) {
            if (k == tid) {
                id = id0;
                teacher = t0;
                given = x0;
            } else {
                id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                teacher = load_any(a.teacher, a.t_type, r * a.n_ids + k);
                given = id >= 0 && id < a.c ? to_f32(x[id]) : 0.f;
            }
        };
        float mt = -FLT_MAX;
        for (int k = tid; k < a.n_ids; k += WAVE) {
            slot(k);
            if (id >= 0) mt = fmaxf(mt, teacher);
            if (id >= a.c && a.id_status) flag_bad_id(a.id_status);
        }
        mt = wave_max(mt);
        float st = 0.f;
        for (int k = tid; k < a.n_ids; k += WAVE) {
            slot(k);
            if (id >= 0) st += exp2_raw((teacher - mt) * a.c2);
        }
        st = wave_sum(st);
        const float lt = st == 0.f ? INFINITY : log2f(st);
        float loss = 0.f;
        for (int k = tid; k < a.n_ids; k += WAVE) {
            slot(k);
            if (id < 0) continue;
            const float zt = teacher - mt;
            const float q = exp2_raw(zt * a.c2 - lt);
            const float lp = id < a.c ? (given - s.m) * a.rt - LN2 * l2 : NAN;
            if (!(q == 0.f)) loss = fmaf(q, (zt * a.rt - LN2 * lt) - lp, loss);
        }
        loss = wave_sum(loss) * (a.t * a.t);
        if (tid == 0) {
            a.loss[r] = loss;
            if (a.stats) {
                a.stats[4 * r + 0] = s.m;
                a.stats[4 * r + 1] = l2;
                a.stats[4 * r + 2] = mt;
                a.stats[4 * r + 3] = lt;
            }
        }
    }
}

// Orders `got` unordered keys and writes the best `top`: as a row's alternatives, or (keys != null) as keys.  buf has room for
// `got` rounded up to whole eights.
template <typename T, int NW>
__device__ __forceinline__ void write_best(const ScoreArgs& a, int64_t r, const T* x, const Sums& s, uint64_t* buf, int got,
                                           uint64_t* keys, int tid) {
    constexpr int NT = NW * WAVE;
    const float ll = LN2 * log2f(s.S);
    const bool nan = s.S != s.S;
    const int g8 = (got + 7) & ~7;
    if (tid < g8 - got) buf[got + tid] = 0;
    group_sync<NW>();
    for (int i = tid; i < got; i += NT) {
        const uint64_t mine = buf[i];
        int rank = 0;
        for (int j = 0; j < g8; j += 8)
#pragma unroll
            for (int e = 0; e < 8; ++e) rank += buf[j + e] > mine ? 1 : 0;
        if (rank >= a.top) continue;
        if (keys) {
            keys[rank] = mine >> 32 ? mine : 0;
        } else {
            const uint32_t id = ~(uint32_t)mine;
            const bool some = !nan && mine >> 32;
            a.top_ids[r * a.top + rank] = some ? (int64_t)id : -1;
            a.top_logp[r * a.top + rank] = nan ? NAN : some ? (to_f32(x[id]) - s.m) * a.rt - ll : -INFINITY;
        }
    }
    for (int i = got + tid; i < a.top; i += NT) {
        if (keys) {
            keys[i] = 0;
        } else {
            a.top_ids[r * a.top + i] = -1;
            a.top_logp[r * a.top + i] = nan ? NAN : -INFINITY;
        }
    }
}

// blocks of 256 threads that a unit holds at once
constexpr int score_fwd_blocks(bool top) { return top ? 6 : 8; }

// One pass over a slice of a row: each thread keeps the largest score and the two sums of its pieces against it, a group's threads
// meet at the end.  NW waves a slice; with NW = 1 a block holds four rows.  splits = 1: the answer; else the slice's sums and best
// keys.
//
// Bound by reading: called again and again 2048 x 131072 bf16 takes 96 us, 5.6 TB/s (a large copy moves 5.2), 65536 x 1001 f32, a wave
// a row, 55 us, 4.8 TB/s; behind a backward 130 and 70.  A score takes nine instructions
// (unpack, half a max3, subtract, multiply, exp2 as four, add; the entropy two more), which is 60 % of the vector unit at that rate: the
// maximum is taken over two pieces at once so that moving the sums to it costs a sixteenth, and nothing else is done per score.  Short of
// that: what a row costs beside its scores (8191 x 5382 f16 19 us, 4.6 TB/s; behind a backward 27) and, with 50 alternatives of
// 256 x 1e6 bf16, 120 us for 99, and 9 for 5 in score_join_kernel: the slices' searches come at the same time, at their ends, and their
// second reads are a fifth of the first.
template <typename T, int NW, bool ENT, bool TOP, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB, score_fwd_blocks(TOP)) score_fwd_kernel(ScoreArgs a) {
    constexpr int NT = NW * WAVE, GROUPS = SC_TPB / NT, V = Piece<T>::N, U = SC_UNROLL;
    __shared__ float scratch[GROUPS][3 * NW];
    __shared__ TopScratch<NW> top_scratch[TOP ? GROUPS : 1];
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x & (NT - 1);
    const int64_t units = a.rows * a.splits;
    for (int64_t unit = (int64_t)blockIdx.x * GROUPS + group; unit < units; unit += (int64_t)gridDim.x * GROUPS) {
        const int64_t r = a.splits == 1 ? unit : unit / a.splits;
        const int from = (int)((unit - r * a.splits) * a.per);
        const int n = (int)(a.per < a.c - from ? a.per : a.c - from);
        const int nvec = n / V, rem = n - nvec * V;
        const T* row = row_ptr<T>(a.x, r);
        const T* x = row + from;
        // the first id of this thread, and further down what the row says about it: both are back before they are needed
        int64_t id = -1;
        float teacher = 0.f, given = 0.f;
        if (a.splits == 1 && tid < a.n_ids && (!DISTILL || tid < WAVE)) {
            id = load_id(a.ids, a.id_type, r * a.n_ids + tid);
            if constexpr (DISTILL) teacher = load_any(a.teacher, a.t_type, r * a.n_ids + tid);
        }
        Sums s{-FLT_MAX, 0.f, 0.f};
        Peak pk{-FLT_MAX, -FLT_MAX, -1};
        int j = 0;
        const T* p = x + tid * V;
        for (; j + U * NT <= nvec; j += U * NT, p += U * NT * V) {
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = Piece<T>::load(p + u * NT * V);
            float v[U * V];
#pragma unroll
            for (int u = 0; u < U; ++u) Piece<T>::unpack(raw[u], *(float(*)[V])(v + u * V));
            const float mx = add_scores<ENT>(s, v, a.c2);
            if constexpr (TOP) pk.add(mx, j + tid);
        }
        if (id >= 0 && id < a.c) given = to_f32(row[id]);
        if (j < nvec) {                               // the last pieces: past the end the last one again, masked
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = j + tid + u * NT;
                if (j + u * NT < nvec) raw[u] = Piece<T>::load(x + (int64_t)(at < nvec ? at : nvec - 1) * V);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j + u * NT < nvec) {
                    float v[V];
                    Piece<T>::unpack(raw[u], v);
                    const bool in = j + tid + u * NT < nvec;
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = in ? v[e] : -INFINITY;
                    const float mx = add_scores<ENT>(s, v, a.c2);
                    if constexpr (TOP) pk.add(mx, j + tid);
                }
            }
        }
        if (rem) {
            const float v[1] = {tid < rem ? to_f32(x[nvec * V + tid]) : -INFINITY};
            const float mx = add_scores<ENT>(s, v, a.c2);
            if constexpr (TOP) pk.add(mx, -1);
        }
        s = group_sums<NW, ENT>(s, a.c2, scratch[group]);
        if (a.splits == 1) {
            row_answer<T, NT, DISTILL>(a, r, row, s, tid, id, teacher, given);
        } else if (tid == 0) {
            a.part[unit] = make_float4(s.m, s.S, s.W, 0.f);
        }
        if constexpr (TOP) {
            const int got = best_scores<T, NW>(x, n, (uint32_t)from, pk, a.top, tid, top_scratch[group]);
            write_best<T, NW>(a, r, row, s, top_scratch[group].key, got, a.splits == 1 ? nullptr : a.keys + unit * a.top, tid);
        }
        group_sync<NW>();                             // the scratch is free again
    }
}

// A row's slices together: thread t holds slice t, its keys are in order.  A chain of latencies: two loads, the cut, two more loads
// and the ordering, 7 us for 244 slices with 20 keys each, 2.5 us without alternatives.
template <typename T, bool ENT, bool TOP, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB) score_join_kernel(ScoreArgs a) {
    __shared__ float scratch[3 * SC_NW];
    __shared__ uint64_t scratch64[SC_NW];
    __shared__ uint64_t buf[TOP ? SC_MAX_TOP * SC_MAX_TOP + 8 : 1];
    __shared__ uint64_t heads[TOP ? SC_TPB + 8 : 1];
    __shared__ uint64_t cut;
    __shared__ int n, lists;
    __shared__ uint8_t who[SC_TPB];
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = row_ptr<T>(a.x, r);
        int64_t id = -1;
        float teacher = 0.f, given = 0.f;
        if (tid < a.n_ids && (!DISTILL || tid < WAVE)) {
            id = load_id(a.ids, a.id_type, r * a.n_ids + tid);
            if constexpr (DISTILL) teacher = load_any(a.teacher, a.t_type, r * a.n_ids + tid);
        }
        // Every slice's q-th best key, q = top / slices rounded up: the m-th largest of them, m q >= top, bounds the row's best
        const int q = TOP ? (a.top + a.splits - 1) / a.splits : 1, m = TOP ? (a.top + q - 1) / q : 1;
        uint64_t head = 0;
        Sums s{-FLT_MAX, 0.f, 0.f};
        if (tid < a.splits) {
            const float4 p = a.part[r * a.splits + tid];
            s = Sums{p.x, p.y, p.z};
            if constexpr (TOP) head = a.keys[(r * a.splits + tid) * a.top + q - 1];
        }
        if (id >= 0 && id < a.c) given = to_f32(x[id]);
        if constexpr (TOP) {
            heads[tid] = head;
            if (tid < 8) heads[SC_TPB + tid] = 0;
            if (tid == 0) {
                cut = 1;
                n = lists = 0;
            }
        }
        s = group_sums<SC_NW, ENT>(s, a.c2, scratch);             // (its barrier is the one that `heads` needs)
        row_answer<T, SC_TPB, DISTILL>(a, r, x, s, tid, id, teacher, given);
        if constexpr (TOP) {
            if (head) {
                int rank = 0;
                for (int i = 0; i < a.splits; i += 8)
#pragma unroll
                    for (int e = 0; e < 8; ++e) rank += heads[i + e] > head ? 1 : 0;
                if (rank == m - 1) cut = head;
            }
            __syncthreads();
            // the slices that can have keys that good: with q = 1 those whose best is, else (fewer than top) all
            if (tid < a.splits && (q > 1 || head >= cut)) who[atomicAdd(&lists, 1)] = (uint8_t)tid;
            __syncthreads();
            const uint64_t* all = a.keys + r * a.splits * a.top;
            const int items = lists * a.top;
            for (int i0 = tid; i0 < items; i0 += 4 * SC_TPB) {
                uint64_t k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = i0 + u * SC_TPB, w = i / a.top;
                    k[u] = i < items ? all[who[w] * a.top + i - w * a.top] : 0;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (k[u] >= cut) buf[atomicAdd(&n, 1)] = k[u];
            }
            __syncthreads();
            int got = n;
            if (got > SC_BUF) {                       // ties in many slices: one after the other, into the place of the heads
                uint64_t last = ~(uint64_t)0;
                for (int k = 0; k < a.top; ++k) {
                    uint64_t best = 0;
                    for (int i = tid; i < got; i += SC_TPB)
                        if (buf[i] < last && buf[i] > best) best = buf[i];
                    last = block_max_u64<SC_NW>(best, scratch64);
                    if (tid == 0) heads[k] = last;
                }
                __syncthreads();
                write_best<T, SC_NW>(a, r, x, s, heads, a.top, nullptr, tid);
            } else {
                write_best<T, SC_NW>(a, r, x, s, buf, got, nullptr, tid);
            }
        }
        __syncthreads();
    }
}

// ---- short rows: LPR lanes of a wave a row -------------------------------------------------------------------------------
//
// What a row costs beside reading it — maxima and sums across lanes, the ids, the writes — is the same instructions for one row or
// for the 64 / LPR rows that a wave holds side by side.  A lane keeps P pieces; the piece that crosses the row's end is pulled
// back into it, as in layer_norm.hip.  Bound by those instructions: 131072 x 64 f32 forward in 12 us (2.8 TB/s), backward in 20
// (3.4 TB/s; with the entropy 21); 50000 x 10 f32 in 3.4 and 4 us, which is little more than an empty launch.

template <typename T, int LPR, int P>
struct ShortRow {
    static constexpr int V = Piece<T>::N;
    float v[P][V];
    int off[P], lo[P];                    // the lane's own: columns off + e for e in [lo, V)
    __device__ __forceinline__ void load(const T* x, int c, int tid) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int at = (i * LPR + tid) * V;
            if (c >= V) {
                off[i] = at + V <= c ? at : c - V;
                lo[i] = at - off[i] < V ? at - off[i] : V;
                Piece<T>::unpack(Piece<T>::load(x + off[i]), v[i]);
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = e >= lo[i] ? v[i][e] : -INFINITY;
            } else {                      // the first lane holds all: columns c - V .. c - 1, of which the negative are not there
                off[i] = c - V;
                lo[i] = at ? V : V - c;
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = e >= lo[i] ? to_f32(x[off[i] + e]) : -INFINITY;
            }
        }
    }
};

// keys of (value, lowest column first) of a short row.  A 16-bit score is exact in the upper 19 bits of its fp32 form, which leaves 13
// for the column and halves what a comparison costs.  Of a masked score only the column remains.
template <typename T>
struct ShortKey {
    typedef uint64_t type;
    static __device__ __forceinline__ type of(float v, uint32_t col) { return v > -INFINITY ? score_key(v, col) : (type)~col; }
    static __device__ __forceinline__ bool live(type k) { return k >> 32; }
};
struct ShortKey16 {
    typedef uint32_t type;
    static __device__ __forceinline__ type of(float v, uint32_t col) {
        return (v > -INFINITY ? value_key(v) & ~0x1fffu : 0u) | (0x1fffu - col);
    }
    static __device__ __forceinline__ bool live(type k) { return k >> 13; }
};
template <>
struct ShortKey<bf16_t> : ShortKey16 {};
template <>
struct ShortKey<f16_t> : ShortKey16 {};

// the largest key of aligned groups of LPR lanes, in each of them
template <int LPR, typename K>
__device__ __forceinline__ K lanes_max_key(K k) {
    auto step = [&](auto exchange) {
        K o;
        if constexpr (sizeof(K) == 4) o = exchange((uint32_t)k);
        else o = ((K)exchange((uint32_t)(k >> 32)) << 32) | exchange((uint32_t)k);
        k = o > k ? o : k;
    };
    if constexpr (LPR >= 2) step([](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xb1, 0xf, 0xf, false); });
    if constexpr (LPR >= 4) step([](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4e, 0xf, 0xf, false); });
    if constexpr (LPR >= 8) step([](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, false); });
    if constexpr (LPR >= 16) step([](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, false); });
    static_assert(LPR <= 16, "within a row of 16 lanes");
    return k;
}

// TOP: 0 no alternatives, 1 a few, 2 any number of them
template <typename T, int LPR, int P, bool ENT, int TOP, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB) score_short_fwd_kernel(ScoreArgs a) {
    typedef ShortKey<T> Key;
    constexpr int V = Piece<T>::N, ROWS = SC_TPB / LPR, W = TOP == 2 ? LPR * P * V + 1 : 1;
    __shared__ typename Key::type keys[TOP == 2 ? ROWS * W : 1];
    const int tid = threadIdx.x & (LPR - 1), slot = threadIdx.x / LPR;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const bool in = r0 + slot < a.rows;            // lanes without a row work on the last one's and write nothing
        const int64_t r = in ? r0 + slot : a.rows - 1;
        const T* x = row_ptr<T>(a.x, r);
        int64_t id = -1;
        if (tid < a.n_ids) id = load_id(a.ids, a.id_type, r * a.n_ids + tid);
        ShortRow<T, LPR, P> row;
        row.load(x, a.c, tid);
        Sums s{-FLT_MAX, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s.m = fmaxf(s.m, row.v[i][e]);
        s.m = lanes_max<LPR>(s.m);
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float z = (row.v[i][e] - s.m) * a.c2, p = exp2_raw(z);
                s.S += p;
                if constexpr (ENT) s.W = fmaf(p, fmaxf(z, Z_FLOOR), s.W);
            }
        s.S = lanes_sum<LPR>(s.S);
        if constexpr (ENT) s.W = lanes_sum<LPR>(s.W);
        const bool some = !(s.S == 0.f);
        const float l2 = some ? log2f(s.S) : INFINITY;
        if constexpr (!DISTILL) {
            if (in && tid == 0) {
                if (ENT) a.entropy[r] = some ? LN2 * (l2 - s.W / s.S) : 0.f;
                if (a.stats) {
                    a.stats[2 * r] = s.m;
                    a.stats[2 * r + 1] = l2;
                }
            }
            for (int k = tid; k < a.n_ids; k += LPR) {
                if (k != tid) id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                float v = 0.f;
                if (id >= a.c) {
                    v = NAN;
                    if (a.id_status) flag_bad_id(a.id_status);
                } else if (id >= 0) {
                    v = some ? (to_f32(x[id]) - s.m) * a.rt - LN2 * l2 : -INFINITY;
                }
                if (in) a.logp[r * a.n_ids + k] = v;
            }
        } else {
            float mt = -FLT_MAX, st = 0.f, loss = 0.f;
            for (int k = tid; k < a.n_ids; k += LPR) {
                id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                if (id >= 0) mt = fmaxf(mt, load_any(a.teacher, a.t_type, r * a.n_ids + k));
                if (id >= a.c && a.id_status) flag_bad_id(a.id_status);
            }
            mt = lanes_max<LPR>(mt);
            for (int k = tid; k < a.n_ids; k += LPR)
                if (load_id(a.ids, a.id_type, r * a.n_ids + k) >= 0)
                    st += exp2_raw((load_any(a.teacher, a.t_type, r * a.n_ids + k) - mt) * a.c2);
            st = lanes_sum<LPR>(st);
            const float lt = st == 0.f ? INFINITY : log2f(st);
            for (int k = tid; k < a.n_ids; k += LPR) {
                id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                if (id < 0) continue;
                const float zt = load_any(a.teacher, a.t_type, r * a.n_ids + k) - mt;
                const float q = exp2_raw(zt * a.c2 - lt);
                const float lp = id < a.c ? (to_f32(x[id]) - s.m) * a.rt - LN2 * l2 : NAN;
                if (!(q == 0.f)) loss = fmaf(q, (zt * a.rt - LN2 * lt) - lp, loss);
            }
            loss = lanes_sum<LPR>(loss) * (a.t * a.t);
            if (in && tid == 0) {
                a.loss[r] = loss;
                if (a.stats) {
                    a.stats[4 * r + 0] = s.m;
                    a.stats[4 * r + 1] = l2;
                    a.stats[4 * r + 2] = mt;
                    a.stats[4 * r + 3] = lt;
                }
            }
        }
        if constexpr (TOP) {
            const bool nan = s.S != s.S;
            typename Key::type key[P][V];
            auto write = [&](int i, int e, int rank) {
                const bool live = !nan && Key::live(key[i][e]);
                a.top_ids[r * a.top + rank] = live ? row.off[i] + e : -1;
                a.top_logp[r * a.top + rank] = nan ? NAN : live ? (row.v[i][e] - s.m) * a.rt - LN2 * l2 : -INFINITY;
            };
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) key[i][e] = e >= row.lo[i] ? Key::of(row.v[i][e], row.off[i] + e) : 0;
            // few: the largest key below the last one, again and again; by ranks any number costs the same.  131072 x 64 bf16, 8 of
            // them 32 us and by ranks 42, but 16 of them 57 and 43, 21 71 and 43; f32 8 of 64 40 and 47, 16 of 64 68 and 47; of 30
            // scores 5 15 and 15, 10 26 and 16: the two meet at about a sixth of the row
            if (TOP == 1 || 3 * a.top <= a.c) {
                typename Key::type last = ~(typename Key::type)0;
                for (int k = 0; k < a.top; ++k) {
                    typename Key::type most = 0;
#pragma unroll
                    for (int i = 0; i < P; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) most = key[i][e] < last && key[i][e] > most ? key[i][e] : most;
                    last = lanes_max_key<LPR>(most);
#pragma unroll
                    for (int i = 0; i < P; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (in && key[i][e] == last) write(i, e, k);
                }
            } else if constexpr (TOP == 2) {           // many: a score's rank is how many of the row are better
                typename Key::type* mine = keys + slot * W;
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e >= row.lo[i]) mine[row.off[i] + e] = key[i][e];
                group_sync<1>();
                int rank[P][V] = {};
                for (int j = 0; j < a.c; ++j) {
                    const typename Key::type other = mine[j];
#pragma unroll
                    for (int i = 0; i < P; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) rank[i][e] += other > key[i][e] ? 1 : 0;
                }
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (in && e >= row.lo[i] && rank[i][e] < a.top) write(i, e, rank[i][e]);
                group_sync<1>();
            }
        }
    }
}

// the gradient; what the listed ids add is summed per column in LDS, slot after slot
template <typename T, int LPR, int P, bool ENT, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB) score_short_bwd_kernel(ScoreArgs a) {
    constexpr int V = Piece<T>::N, ROWS = SC_TPB / LPR;
    extern __shared__ float added[];                   // [ROWS, c]
    const int tid = threadIdx.x & (LPR - 1), slot = threadIdx.x / LPR;
    float* mine = added + slot * a.c;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.rows; r0 += (int64_t)gridDim.x * ROWS) {
        const bool in = r0 + slot < a.rows;
        const int64_t r = in ? r0 + slot : a.rows - 1;
        const T* x = row_ptr<T>(a.x, r);
        ShortRow<T, LPR, P> row;
        row.load(x, a.c, tid);
        const float m = a.stats[(DISTILL ? 4 : 2) * r], l2 = a.stats[(DISTILL ? 4 : 2) * r + 1];
        const float mt = DISTILL ? a.stats[4 * r + 2] : 0.f, lt = DISTILL ? a.stats[4 * r + 3] : 0.f;
        const bool none = l2 == INFINITY;
        for (int i = tid; i < a.c; i += LPR) mine[i] = 0.f;
        group_sync<1>();
        float sum = 0.f;
        float used = 0.f;
        for (int k0 = 0; k0 < a.n_ids; k0 += LPR) {
            int at = -1;
            float g = 0.f;
            if (k0 + tid < a.n_ids) {
                const int64_t k = r * a.n_ids + k0 + tid, id = load_id(a.ids, a.id_type, k);
                const float given = DISTILL ? load_any(a.teacher, a.t_type, k) : a.g_logp ? a.g_logp[k] : 0.f;     // beside the id
                if (id >= 0 && id < a.c && !none) {
                    at = (int)id;
                    used = 1.f;
                    g = DISTILL ? exp2_raw((given - mt) * a.c2 - lt) : given;
                    sum += g;
                }
            }
            const int slots = a.n_ids - k0 < LPR ? a.n_ids - k0 : LPR;
            for (int t = 0; t < slots; ++t) {
                if (tid == t && at >= 0) mine[at] += g;
                group_sync<1>();
            }
        }
        group_sync<1>();
        float A, B = 0.f, H2 = 0.f, u;
        if (DISTILL) {
            u = -a.g_logp[r] * a.t;
            A = -u + (lt - lt);
        } else {
            A = -lanes_sum<LPR>(sum) * a.rt;
            u = a.rt;
            if (ENT) {
                B = -a.g_entropy[r] * LN2 * a.rt;
                H2 = a.entropy[r] / LN2;
            }
        }
        const bool dead = DISTILL ? lt == INFINITY : lanes_max<LPR>(used) == 0.f && (!ENT || B == 0.f);
        T* dx = (T*)a.dx + r * a.c;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float lp = fmaf(row.v[i][e] - m, a.c2, -l2);
                const float p = exp2_raw(lp);
                const float d = ENT ? p * fmaf(B, fmaxf(lp, Z_FLOOR) + H2, A) : p * A;
                o[e] = e >= row.lo[i] && !dead ? fmaf(mine[row.off[i] + e], u, d) : 0.f;
            }
            if (!in) continue;
            if (row.lo[i] == 0) {
                Piece<T>::store(dx + row.off[i], Piece<T>::pack(o));
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e >= row.lo[i]) dx[row.off[i] + e] = from_f32<T>(o[e]);
            }
        }
        group_sync<1>();
    }
}

static unsigned short_grid(int64_t rows, int lpr) {
    const int64_t blocks = (rows * lpr + SC_TPB - 1) / SC_TPB, most = (int64_t)device_cu_count() * 8;
    return (unsigned)(blocks < most ? blocks : most);
}

// Rows of up to 64 pieces go several to a wave: 4 lanes with one piece each, or 16 with up to four (131072 x 64 f32: 12 us, with a
// wave a row 42; 100000 x 250 f32: 28 and 38).  Alternatives: of up to 64 scores any number; of more by repeated maxima, as long as
// that beats a wave a row.  20000 x 100 f32 with 5 / 24 / 40 / 48 of them 10 / 24 / 37 / 42 us, a wave a row 40; bf16 8 / 21 / 33 / 38, a
// wave a row 41.  Of 250 scores with 1 / 5 / 8 of them, in brackets a wave a row: 8192 rows bf16 5.9 / 8.6 / 10.7 (11.7 / 12.3 / 12.4),
// f32 7.2 / 10.9 / 13.5 (10.8 / 11.0 / 11.1); 4096 rows bf16 5.5 / 8.0 / 9.9 (8.9 / 9.2 / 9.4), f32 6.3 / 9.5 / 11.8 (8.0 / 8.1 / 8.4); 2048
// rows bf16 5.4 / 7.9 / 9.8 (7.5 / 7.8 / 8.0), f32 5.8 / 9.1 / 11.6 (6.7 / 6.9 / 7.0).  One rule for all types: it gives bf16 its due and
// costs f32 up to 3 us with five to eight.
template <typename T, bool ENT, bool TOP, bool DISTILL>
static bool launch_short_fwd(const ScoreArgs& a, hipStream_t st) {
    constexpr int V = Piece<T>::N;
    if (DISTILL && a.n_ids > 64) return false;
    if constexpr (TOP) {
        constexpr int P = sizeof(T) == 4 ? 2 : 1;     // 4 lanes: 32 scores, 16 lanes: 128
        if (a.c <= 4 * P * V) score_short_fwd_kernel<T, 4, P, ENT, 2, false><<<short_grid(a.rows, 4), SC_TPB, 0, st>>>(a);
        else if (a.c <= 64) score_short_fwd_kernel<T, 64 / V, 1, ENT, 2, false><<<short_grid(a.rows, 64 / V), SC_TPB, 0, st>>>(a);
        else if (a.c <= 128 && a.top <= 40) score_short_fwd_kernel<T, 16, P, ENT, 1, false><<<short_grid(a.rows, 16), SC_TPB, 0, st>>>(a);
        else if (a.c <= 256 && a.top <= 8 && a.rows >= 4096) score_short_fwd_kernel<T, 16, 2 * P, ENT, 1, false><<<short_grid(a.rows, 16), SC_TPB, 0, st>>>(a);
        else return false;
    } else {
        if (a.c <= 4 * V) score_short_fwd_kernel<T, 4, 1, ENT, 0, DISTILL><<<short_grid(a.rows, 4), SC_TPB, 0, st>>>(a);
        else if (a.c <= 16 * V) score_short_fwd_kernel<T, 16, 1, ENT, 0, DISTILL><<<short_grid(a.rows, 16), SC_TPB, 0, st>>>(a);
        else if (a.c <= 64 * V) score_short_fwd_kernel<T, 16, 4, ENT, 0, DISTILL><<<short_grid(a.rows, 16), SC_TPB, 0, st>>>(a);
        else return false;
    }
    return true;
}

template <typename T, bool ENT, bool DISTILL>
static bool launch_short_bwd(const ScoreArgs& a, hipStream_t st) {
    constexpr int V = Piece<T>::N;
    if (a.n_ids > 64) return false;
    const size_t row = (size_t)a.c * sizeof(float);
    if (a.c <= 4 * V) score_short_bwd_kernel<T, 4, 1, ENT, DISTILL><<<short_grid(a.rows, 4), SC_TPB, SC_TPB / 4 * row, st>>>(a);
    else if (a.c <= 16 * V) score_short_bwd_kernel<T, 16, 1, ENT, DISTILL><<<short_grid(a.rows, 16), SC_TPB, SC_TPB / 16 * row, st>>>(a);
    else if (a.c <= 64 * V) score_short_bwd_kernel<T, 16, 4, ENT, DISTILL><<<short_grid(a.rows, 16), SC_TPB, SC_TPB / 16 * row, st>>>(a);
    else return false;
    return true;
}

// Slices of a row: what makes rounds(slices) * (a slice's length + what a slice costs beside reading it) + the joining kernel
// smallest.  The costs are in scores that a block of a full chip reads meanwhile (2.7 KB/us of 16-bit scores): about 2 us a slice,
// 5 us with alternatives, 5 us for the second kernel.  No slice is below 4096 scores; the joining kernel has a thread for each.
static int score_splits(int64_t rows, int64_t c, int top) {
    if (c < 8192) return 1;
    const int64_t slots = (int64_t)device_cu_count() * score_fwd_blocks(top > 0), own = top ? 6700 : 2700;
    int64_t most = c / 4096 < SC_TPB ? c / 4096 : SC_TPB, best = 0;
    int n = 1;
    for (int64_t k = 1; k <= most; ++k) {
        const int64_t cost = (rows * k + slots - 1) / slots * (c / k + own) + (k > 1 ? 6700 : 0);
        if (k == 1 || cost < best) {
            best = cost;
            n = (int)k;
        }
    }
    return n;
}

// blocks that take slice after slice: at most what the chip holds at once
static unsigned score_grid(int64_t blocks, int per_unit) {
    const int64_t most = (int64_t)device_cu_count() * per_unit;
    return (unsigned)(blocks < most ? blocks : most);
}

static int64_t score_ws(int64_t rows, int64_t c, int top) {
    const int64_t splits = score_splits(rows, c, top);
    return splits == 1 ? 0 : rows * splits * (16 + (int64_t)top * 8);
}

template <typename T, bool ENT, bool TOP, bool DISTILL>
static int launch_score_fwd(ScoreArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
    if (launch_short_fwd<T, ENT, TOP, DISTILL>(a, st)) {
        ARMNET_LAUNCH_CHECK();
        return ARMNET_OK;
    }
    a.splits = score_splits(a.rows, a.c, a.top);
    a.per = a.splits == 1 ? a.c : ((a.c + a.splits - 1) / a.splits + 63) / 64 * 64;
    if (a.splits > 1) {
        if (!ws || ws_bytes < score_ws(a.rows, a.c, a.top)) return ARMNET_ERR_BAD_ARG;
        a.splits = (int)((a.c + a.per - 1) / a.per);                 // rounding up may leave the last slices empty
        a.part = (float4*)ws;
        a.keys = (uint64_t*)(a.part + a.rows * a.splits);
    }
    // A wave a row: what a row costs beside reading it is paid once instead of by four waves.  For short rows always, for longer ones
    // where rows alone fill the chip.  x 5382 f16, a wave and a block a row: 8191 rows 20 and 26 us, 4096 11.8 and 14.4, 2048 8.0 and
    // 9.2, 1000 7.0 and 6.3; f32 4096 rows 17.4 and 18.9, 2048 10.4 and 11.5; 4096 x 20001 f16 38 and 44.  The border lies above the
    // crossing, so a wave is taken only where it wins
    const int64_t one_go = WAVE * Piece<T>::N * 4;
    if (a.c <= one_go || (a.splits == 1 && a.rows >= 4096 && a.c <= 16 * one_go))
        score_fwd_kernel<T, 1, ENT, TOP, DISTILL><<<score_grid((a.rows + 3) / 4, score_fwd_blocks(TOP)), SC_TPB, 0, st>>>(a);
    else
        score_fwd_kernel<T, SC_NW, ENT, TOP, DISTILL><<<score_grid(a.rows * a.splits, score_fwd_blocks(TOP)), SC_TPB, 0, st>>>(a);
    ARMNET_LAUNCH_CHECK();
    if (a.splits > 1) {
        score_join_kernel<T, ENT, TOP, DISTILL><<<row_grid(a.rows), SC_TPB, 0, st>>>(a);
        ARMNET_LAUNCH_CHECK();
    }
    return ARMNET_OK;
}

template <typename T>
static int launch_scores(ScoreArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
    if (a.entropy) return a.top ? launch_score_fwd<T, true, true, false>(a, ws, ws_bytes, st) : launch_score_fwd<T, true, false, false>(a, ws, ws_bytes, st);
    return a.top ? launch_score_fwd<T, false, true, false>(a, ws, ws_bytes, st) : launch_score_fwd<T, false, false, false>(a, ws, ws_bytes, st);
}

// A long list, each of its ids once: add(id, sum of its addends), from one lane of the group.  The slots' numbers go into an open
// table by their ids (a power of two, a fifth larger than the list at least, -1 where empty); the slot that is there keeps the id and
// is marked if another one comes.  Which one that is may differ from run to run; the sum does not: a wave adds up a marked id's
// addends from the whole list, in an order that their places fix.
constexpr int32_t MORE = 1 << 30;

template <int NW, typename F>
__device__ __forceinline__ void add_listed(const int32_t* s_id, const float* s_g, int n, int32_t* table, int slots, int tid, F add) {
    constexpr int NT = NW * WAVE;
    const int lane = tid & (WAVE - 1);
    for (int k = tid; k < n; k += NT) {
        const int32_t id = s_id[k];
        if (id < 0) continue;
        uint32_t h = (uint32_t)id * 2654435769u >> 16;            // Knuth's multiplicative hash
        for (;;) {                                                // ends: the table has empty places
            h &= (uint32_t)slots - 1;
            const int32_t there = atomicCAS(table + h, -1, k);
            if (there == -1) break;
            if (s_id[there & ~MORE] == id) {
                atomicOr(table + h, MORE);
                break;
            }
            ++h;
        }
    }
    group_sync<NW>();
    for (int h = tid; h < slots; h += NT) {                       // whole waves
        const int32_t k = table[h];
        const int32_t id = k == -1 ? -1 : s_id[k & ~MORE];
        float g = k == -1 ? 0.f : s_g[k & ~MORE];
        for (uint64_t more = __ballot(k != -1 && (k & MORE)); more; more &= more - 1) {
            const int l = __builtin_ctzll(more);
            const int32_t its = __builtin_amdgcn_readlane(id, l);
            float part = 0.f;
            for (int i = lane; i < n; i += WAVE) part += s_id[i] == its ? s_g[i] : 0.f;
            part = wave_sum(part);
            if (lane == l) g = part;
        }
        if (id >= 0) add(id, g);
    }
}

// The gradient of a slice of a row: p's part of it everywhere, then the listed ids' values again with what they add.  Of a
// list of up to 64 every slot looks at all others, and the first one of an id adds them up in order; a longer one has a table.  NW
// waves a slice; NW = 1: four rows a block.  List of a group in LDS: n16 ids (padded with -1 to whole sixteens), n16 addends, the
// table.  The first pieces and the list are on their way at the same time.
//
// Bound by reading and writing: behind its forward 2048 x 131072 bf16 takes 181 us, 5.9 TB/s, 65536 x 1001 f32 with the entropy's part
// 95 us, 5.5 TB/s (again and again 194 and 111; an addend's load behind its id's instead of beside it costs 4 %).
// 4096 x 5382 bf16 19 us with one id a row, 24 with 64, 26 with 100, 48 with 200, 167 with 1024 (the last three with the ids compared
// with each other 34, 67 and 979): what is left is the ids that come twice.
template <typename T, int NW, bool ENT, bool DISTILL>
__global__ void __launch_bounds__(SC_TPB) score_bwd_kernel(ScoreArgs a) {
    constexpr int NT = NW * WAVE, GROUPS = SC_TPB / NT, V = Piece<T>::N, U = SC_BWD_UNROLL;
    extern __shared__ int4 lists[];
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x & (NT - 1), lane = tid & (WAVE - 1);
    const int n16 = (a.n_ids + 15) & ~15;
    int32_t* s_id = (int32_t*)lists + group * (2 * n16 + a.slots);
    float* s_g = (float*)(s_id + n16);
    int32_t* table = s_id + 2 * n16;                    // [slots], none for a short list
    const int64_t units = a.rows * a.splits;
    for (int64_t unit = (int64_t)blockIdx.x * GROUPS + group; unit < units; unit += (int64_t)gridDim.x * GROUPS) {
        const int64_t back = units - 1 - unit;          // the forward's last rows first: some are still in the last-level cache
        const int64_t r = a.splits == 1 ? back : back / a.splits;
        const int from = (int)((back - r * a.splits) * a.per);
        const int n = (int)(a.per < a.c - from ? a.per : a.c - from);
        const int nvec = n / V, rem = n - nvec * V;
        const T* x = row_ptr<T>(a.x, r) + from;
        T* dx = (T*)a.dx + r * a.c + from;
        u32x4 raw[U];
        auto load = [&](int j) {                        // past the end: the last piece again
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int at = j + tid + i * NT;
                if (j + i * NT < nvec) raw[i] = Piece<T>::load(x + (int64_t)(at < nvec ? at : nvec - 1) * V);
            }
        };
        load(0);
        const float m = a.stats[(DISTILL ? 4 : 2) * r], l2 = a.stats[(DISTILL ? 4 : 2) * r + 1];
        const float mt = DISTILL ? a.stats[4 * r + 2] : 0.f, lt = DISTILL ? a.stats[4 * r + 3] : 0.f;
        const bool none = l2 == INFINITY;
        group_sync<NW>();                               // the slice before is done with the list
        float sum = 0.f;
        bool used = false;
        int32_t first = -1;                             // this thread's slot of the list (k = tid), its addend and the row's score
        float first_g = 0.f, first_x = 0.f;
        for (int h = tid; h < a.slots; h += NT) table[h] = -1;
        for (int k0 = 0; k0 < n16; k0 += WAVE) {        // every wave adds up the whole list, each keeps its share of it
            const int k = k0 + lane;
            int32_t at = -1;
            float g = 0.f;
            if (k < a.n_ids) {
                const int64_t id = load_id(a.ids, a.id_type, r * a.n_ids + k);
                if (DISTILL) g = load_any(a.teacher, a.t_type, r * a.n_ids + k);          // beside the id
                else if (a.g_logp) g = a.g_logp[r * a.n_ids + k];
                const bool in = id >= 0 && id < a.c && !none;
                used = used || in;
                if (DISTILL) g = exp2_raw((g - mt) * a.c2 - lt);
                g = in ? g : 0.f;
                sum += g;
                if (in && id >= from && id < from + n) at = (int32_t)id - from;
            }
            if (k < n16 && (k0 / WAVE) % NW == tid / WAVE) {
                s_id[k] = at;
                s_g[k] = g;
                if (k == tid) {
                    first = at;
                    first_g = g;
                    if (at >= 0) first_x = to_f32(x[at]);
                }
            }
        }
        // dx = p (A + B (log2 p + H2)) + u * (what the listed ids add)
        float A, B = 0.f, H2 = 0.f, u;
        if (DISTILL) {
            u = -a.g_logp[r] * a.t;
            A = -u + (lt - lt);                         // a teacher without a distribution (NaN) has no gradient either
        } else {
            A = -wave_sum(sum) * a.rt;
            u = a.rt;
            if (ENT) {
                B = -a.g_entropy[r] * LN2 * a.rt;
                H2 = a.entropy[r] / LN2;
            }
        }
        // a row that nothing is asked of has gradient 0, whatever it holds (the padding of a batch)
        const bool dead = __builtin_amdgcn_readfirstlane(DISTILL ? lt == INFINITY : !__any(used) && (!ENT || B == 0.f));
        auto base = [&](float xv) {
            const float lp = fmaf(xv - m, a.c2, -l2);
            const float p = exp2_raw(lp);
            return ENT ? p * fmaf(B, fmaxf(lp, Z_FLOOR) + H2, A) : p * A;
        };
        for (int j = 0; j < nvec; j += U * NT) {
            if (j) load(j);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (j + tid + i * NT < nvec) {
                    float v[V];
                    Piece<T>::unpack(raw[i], v);
                    if (dead) {
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] = 0.f;
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] = base(v[e]);
                    }
                    Piece<T>::store(dx + (int64_t)(j + tid + i * NT) * V, Piece<T>::pack(v));
                }
            }
        }
        if (tid < rem) dx[nvec * V + tid] = from_f32<T>(dead ? 0.f : base(to_f32(x[nvec * V + tid])));
        if (a.n_ids == 0 || dead) continue;
        // the list is complete, and the stores above come before the ones below
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        group_sync<NW>();
        if (a.slots) {
            add_listed<NW>(s_id, s_g, n16, table, a.slots, tid, [&](int32_t id, float g) {
                dx[id] = from_f32<T>(fmaf(g, u, base(to_f32(x[id]))));
            });
            continue;
        }
        if (tid < a.n_ids && first >= 0) {
            const int32_t id = first;
            float g = first_g;
            int same = 0;
            for (int i = 0; i < n16; i += 16)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int4 o = *(const int4*)(s_id + i + 4 * q);
                    same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
                }
            if (same > 1) {                             // the first of them adds them all up, in order
                int lead = tid;
                g = 0.f;
                for (int i = 0; i < n16; i += 16)
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        const bool is = s_id[i + q] == id;
                        lead = is && i + q < lead ? i + q : lead;
                        g += is ? s_g[i + q] : 0.f;
                    }
                if (lead != tid) continue;
            }
            dx[id] = from_f32<T>(fmaf(g, u, base(first_x)));
        }
    }
}

template <typename T, bool ENT, bool DISTILL>
static int launch_score_bwd(ScoreArgs& a, hipStream_t st) {
    if (launch_short_bwd<T, ENT, DISTILL>(a, st)) {
        ARMNET_LAUNCH_CHECK();
        return ARMNET_OK;
    }
    const bool narrow = a.c <= WAVE * Piece<T>::N * 4;               // a wave a row: its lanes hold it in one go
    // slices of 16384 scores (2048 x 131072 bf16, again and again: 8192 220 us, 16384 194, 32768 211, 65536 222); few rows: down to what a block's
    // threads load at once
    const int64_t at_once = SC_TPB * Piece<T>::N * SC_BWD_UNROLL;
    int64_t splits = (a.c + 16383) / 16384;
    if (a.rows < 2048) {
        int64_t want = (2048 + a.rows - 1) / a.rows;
        if (want > (a.c + at_once - 1) / at_once) want = (a.c + at_once - 1) / at_once;
        if (want > splits) splits = want;
    }
    if (narrow) splits = 1;
    a.per = splits == 1 ? a.c : ((a.c + splits - 1) / splits + 63) / 64 * 64;
    a.splits = (int)((a.c + a.per - 1) / a.per);
    const int n16 = (a.n_ids + 15) & ~15;
    a.slots = 0;
    if (a.n_ids > WAVE)
        for (a.slots = 128; a.slots < n16 + n16 / 5;) a.slots *= 2;
    const size_t list = (size_t)(2 * n16 + a.slots) * 4;          // four of them: at most 64 KiB
    if (narrow)
        score_bwd_kernel<T, 1, ENT, DISTILL><<<row_grid((a.rows + 3) / 4), SC_TPB, 4 * list, st>>>(a);
    else
        score_bwd_kernel<T, SC_NW, ENT, DISTILL><<<row_grid(a.rows * a.splits), SC_TPB, list, st>>>(a);
    ARMNET_LAUNCH_CHECK();
    return ARMNET_OK;
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
    return score_ws(rows, c, top);
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
    ARMNET_ROW_TYPE(x_type, T, return launch_scores<T>(a, workspace, ws_bytes, (hipStream_t)stream));
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
    hipStream_t st = (hipStream_t)stream;
    ARMNET_ROW_TYPE(x_type, T, return g_entropy ? (launch_score_bwd<T, true, false>(a, st)) : (launch_score_bwd<T, false, false>(a, st)));
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
    ARMNET_ROW_TYPE(x_type, T, return (launch_score_fwd<T, false, false, true>(a, workspace, ws_bytes, (hipStream_t)stream)));
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
    ARMNET_ROW_TYPE(x_type, T, return (launch_score_bwd<T, false, true>(a, (hipStream_t)stream)));
}

}  // extern "C"
