// token_logprobs.cu -- what a model's logits say about given tokens, and the gradient.
//
// For a row of logits x, temperature T, m = max x:
//   y_v = (x_v - m) / T,  s = sum e^y_v,  ln p_v = y_v - ln s
//   log probability of the given token t: ln p_t
//   entropy:                              H = ln s - (sum e^y_v y_v) / s
//   alternatives:                         the `top` largest logits, ties to the lowest token
//   gradient:  dx_v = [ -p_v (gl + sum gk + gH (ln p_v + H)) + gl [v = t] + sum gk [v = id_k] ] / T
//
// logprobs_kernel reads the logits once: running maximum, sum and weighted sum per thread
// (rescaled when the maximum grows), and the alternatives by a threshold that a first look at
// the row sets, so that the few elements above it go to a buffer in shared memory.  A row is
// one block's, or a cluster's when there are few rows: each block of the cluster then takes a
// share of the columns and the first one joins them over distributed shared memory.
//
// neighbours_kernel mixes in the tokens of a search's neighbours:
//   w = softmax(-distance / tau),  p_v = (1 - l) q_v + l sum of w_j over neighbours j with token v
// It needs the statistics of q and its alternatives only: a token that is no neighbour's keeps
// its order among those, so the mixture's alternatives are among q's and the neighbours' tokens,
// and the entropy differs from q's in the neighbours' terms and the factor (1 - l).
#include <cooperative_groups.h>

#include <cmath>
#include <limits>

#include "operators.cuh"

namespace hanns {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxThreads = 256;
constexpr int kUnroll = 4;
constexpr int kMaxTop = 32;
constexpr int kCap = 1024;       // buffered candidates of a block
constexpr int kMaxCluster = 8;
constexpr int kMaxNeighbours = 1024;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;
// 2^y is zero in f32 below this; also what a masked element's -inf becomes, so that
// 2^y y is 0 and not NaN
constexpr float kLowest = -200.0f;
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // total_order_key(-inf)

struct ProbArgs {
    const void* logits;
    int64_t ld;
    int32_t vocab;
    const int64_t* tokens;
    float c, inv_t;  // log2(e) / T, 1 / T
    int top;
    float *logprobs, *entropy;
    int64_t* top_tokens;
    float* top_logprobs;
    float4* stats;  // {m, s, H, state: 1, 0 for an empty row, NaN for an undefined one}
};

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// (x - m) / T - ln s.  Halves, because x - m may pass f32's range where (x - m) / T does not.
__device__ __forceinline__ float log_prob(float x, float m, float inv_t, float log_s) {
    return fmaf(fmaf(0.5f, x, -0.5f * m), 2.0f * inv_t, -log_s);
}

// Order of the alternatives: larger logit first, then lower token; 0 is "none".  -0 and +0
// are the same logit.
__device__ __forceinline__ uint64_t cand_key(float x, int32_t col) {
    return ((uint64_t)total_order_key(x + 0.0f) << 32) | (0xffffffffu - (uint32_t)col);
}
__device__ __forceinline__ float key_logit(uint64_t k) { return key_to_float((uint32_t)(k >> 32)); }
__device__ __forceinline__ int32_t key_col(uint64_t k) { return (int32_t)(0xffffffffu - (uint32_t)k); }

// A row's elements as 16-byte vectors from the 16-byte boundary at or before its first one;
// the vectors that the row does not fill are read element by element, -inf outside the row.
template <class T>
struct RowView {
    static constexpr int VE = 16 / sizeof(T);
    const T* row;
    int lead, vocab;
    __device__ __forceinline__ RowView(const T* r, int v)
        : row(r), lead((int)(((uintptr_t)r & 15) / sizeof(T))), vocab(v) {}
    __device__ __forceinline__ int vectors() const { return (int)(((int64_t)lead + vocab + VE - 1) / VE); }
    __device__ __forceinline__ int64_t first(int i) const { return (int64_t)i * VE - lead; }
    __device__ __forceinline__ Pack<T, VE> load(int i) const {
        const int64_t e = first(i);
        if (e >= 0 && e + VE <= vocab) return load_pack<T, VE>(row + e);
        Pack<T, VE> p;
#pragma unroll
        for (int k = 0; k < VE; ++k)
            p.v[k] = e + k >= 0 && e + k < vocab ? row[e + k] : from_f32<T>(-INFINITY);
        return p;
    }
};

// Sum of 2^y and of 2^y y, y = (x - m) c.
struct Running {
    float m = -INFINITY, s = 0.0f, u = 0.0f;
    __device__ __forceinline__ void grow(float nm, float c) {
        const float d = fmaxf((m - nm) * c, kLowest), f = ex2(d);
        u = f * fmaf(d, s, u);
        s *= f;
        m = nm;
    }
};

template <class T>
__device__ __forceinline__ float pack_max(const Pack<T, RowView<T>::VE>& p) {
    float v = to_f32(p.v[0]);
#pragma unroll
    for (int k = 1; k < RowView<T>::VE; ++k) v = max_nan(v, to_f32(p.v[k]));
    return v;
}

struct Shared {
    uint64_t buf[kCap];
    uint64_t best[kMaxTop];  // this block's alternatives, best first
    uint32_t hist[256];
    float red[3][kMaxThreads / 32];
    uint32_t warp_key[kMaxThreads / 32];
    int count;      // candidates offered (may pass kCap: then some were dropped)
    int dropped;
    uint64_t low;   // fallback: every key from here on is collected
    float m, s, u;  // of this block's columns
};

__device__ __forceinline__ void offer(Shared& sh, uint64_t key) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kCap) sh.buf[at] = key;
}

// best[0 .. top) = the largest of the first n buffered keys (all different), 0 behind them.
__device__ void rank_select(Shared& sh, int n, int top) {
    for (int i = threadIdx.x; i < top; i += blockDim.x) sh.best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t k = sh.buf[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.buf[j] > k;
        if (rank < top) sh.best[rank] = k;
    }
    __syncthreads();
}

// Lower bound of the row's `top`-th logit from each thread's first maximum: the smallest over
// the warps of the warp's ceil(top / warps)-th largest maximum.
__device__ float first_threshold(Shared& sh, float vm, int top) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    uint32_t key = vm != vm ? 0xffffffffu : total_order_key(vm), found = 0;
    for (int r = (top + warps - 1) / warps; r > 0; --r) {
        found = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == found);
        if (lane == __ffs(who) - 1) key = 0;
    }
    if (lane == 0) sh.warp_key[threadIdx.x >> 5] = found;
    __syncthreads();
    uint32_t low = sh.warp_key[0];
    for (int w = 1; w < warps; ++w) low = min(low, sh.warp_key[w]);
    return low <= kKeyMinusInf ? -INFINITY : key_to_float(low);
}

// Keeps the best of the buffer when it has grown and returns the new threshold.
__device__ float refine(Shared& sh, int top, float thr) {
    __syncthreads();
    const int offered = sh.count, n = min(offered, kCap);
    __syncthreads();  // every thread has read the count before the first new candidate
    if (n <= 2 * top + 32) return thr;
    rank_select(sh, n, top);
    for (int i = threadIdx.x; i < top; i += blockDim.x) sh.buf[i] = sh.best[i];
    if (threadIdx.x == 0) {
        if (offered > kCap) sh.dropped = 1;
        sh.count = top;
    }
    __syncthreads();
    return fmaxf(thr, key_logit(sh.buf[top - 1]));
}

// Candidates were dropped (a row that climbs, or ties by the thousand): find by counting key
// bytes, highest first, a bound that at least `top` and at most kCap keys reach, and collect
// those.  Reads the columns up to nine times.
template <class T>
__device__ void collect_again(Shared& sh, const RowView<T>& view, int v0, int v1, int top) {
    const int64_t e0 = max((int64_t)0, view.first(v0)), e1 = min((int64_t)view.vocab, view.first(v1));
    uint64_t prefix = 0;
    int need = top;
    for (int byte = 7; byte >= 0; --byte) {
        __syncthreads();
        for (int b = threadIdx.x; b < 256; b += blockDim.x) sh.hist[b] = 0;
        __syncthreads();
        for (int64_t e = e0 + threadIdx.x; e < e1; e += blockDim.x) {
            const float x = to_f32(view.row[e]);
            if (!(x > -INFINITY)) continue;
            const uint64_t k = cand_key(x, (int32_t)e);
            if (byte == 7 || (k >> (8 * byte + 8)) == prefix) atomicAdd(&sh.hist[(k >> (8 * byte)) & 255], 1u);
        }
        __syncthreads();
        // every thread walks the counts alike
        int above = 0, b = 255;
        while (b > 0 && above + (int)sh.hist[b] < need) above += sh.hist[b--];
        const int reach = top - need + above + (int)sh.hist[b];
        prefix = (prefix << 8) | (uint64_t)b;
        if (threadIdx.x == 0) sh.low = prefix << (8 * byte);
        if (reach <= kCap) break;
        need -= above;
    }
    __syncthreads();
    const uint64_t low = sh.low;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int64_t e = e0 + threadIdx.x; e < e1; e += blockDim.x) {
        const float x = to_f32(view.row[e]);
        if (!(x > -INFINITY)) continue;
        const uint64_t k = cand_key(x, (int32_t)e);
        if (k >= low) offer(sh, k);
    }
}

__device__ __forceinline__ float block_reduce(Shared& sh, int slot, float v, bool is_max) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, d);
        v = is_max ? max_nan(v, o) : v + o;
    }
    if ((threadIdx.x & 31) == 0) sh.red[slot][threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.red[slot][0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = is_max ? max_nan(v, sh.red[slot][w]) : v + sh.red[slot][w];
    return v;
}

// What the columns' sums become against another maximum (an empty or undefined one: nothing).
__device__ __forceinline__ void rescale(float m, float& s, float& u, float to, float c) {
    const float d = fmaxf((m - to) * c, kLowest), f = ex2(d);
    u = f * fmaf(d, s, u);
    s *= f;
}

template <class T, bool Top>
__global__ void __launch_bounds__(kMaxThreads) logprobs_kernel(ProbArgs a) {
    constexpr int VE = RowView<T>::VE;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int64_t r = blockIdx.x / parts;
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    const RowView<T> view(row, a.vocab);
    const int nvec = view.vectors(), per = (nvec + parts - 1) / parts;
    const int v0 = min(nvec, part * per), v1 = min(nvec, v0 + per);
    int64_t token = -1;
    float x_t = 0.0f;
    if (part == 0 && threadIdx.x == 0) {
        token = a.tokens[r];
        if ((uint64_t)token < (uint64_t)a.vocab) x_t = to_f32(row[token]);
    }
    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.dropped = 0;
    }
    __syncthreads();

    Running run;
    float thr = -INFINITY;
    const int step = blockDim.x * kUnroll;
    int round = 0, look = 2;
    for (int base = v0; base < v1; base += step, ++round) {
        Pack<T, VE> p[kUnroll];
        float vm[kUnroll];
#pragma unroll
        for (int q = 0; q < kUnroll; ++q) {
            const int i = base + q * blockDim.x + threadIdx.x;
            if (i < v1) {
                p[q] = view.load(i);
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k) p[q].v[k] = from_f32<T>(-INFINITY);
            }
        }
#pragma unroll
        for (int q = 0; q < kUnroll; ++q) vm[q] = pack_max<T>(p[q]);
        if (Top) {
            if (round == 0) {
                float t = vm[0];
#pragma unroll
                for (int q = 1; q < kUnroll; ++q) t = max_nan(t, vm[q]);
                thr = first_threshold(sh, t, a.top);
            } else if (round == look) {
                thr = refine(sh, a.top, thr);
                look = 2 * look;
            }
        }
#pragma unroll
        for (int q = 0; q < kUnroll; ++q) {
            if (!(vm[q] <= run.m)) run.grow(max_nan(vm[q], run.m), a.c);
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const float y = fmaxf((to_f32(p[q].v[k]) - run.m) * a.c, kLowest), e = ex2(y);
                run.s += e;
                run.u = fmaf(e, y, run.u);
            }
            if (Top && vm[q] >= thr) {
                const int64_t e0 = view.first(base + q * blockDim.x + threadIdx.x);
#pragma unroll
                for (int k = 0; k < VE; ++k) {
                    const float x = to_f32(p[q].v[k]);
                    if (x >= thr && x > -INFINITY) offer(sh, cand_key(x, (int32_t)(e0 + k)));
                }
            }
        }
    }

    const float m = block_reduce(sh, 0, run.m, true);
    rescale(run.m, run.s, run.u, m, a.c);
    const float s = block_reduce(sh, 1, run.s, false);
    const float u = block_reduce(sh, 2, run.u, false);
    if (threadIdx.x == 0) {
        sh.m = m;
        sh.s = s;
        sh.u = u;
    }
    if (Top) {
        __syncthreads();
        if (sh.dropped || sh.count > kCap) collect_again(sh, view, v0, v1, a.top);
        __syncthreads();
        rank_select(sh, min(sh.count, kCap), a.top);
    }
    if (parts > 1) cluster.sync();
    if (part == 0) {
        float M = m, S = s, U = u;
        if (parts > 1) {
            for (int q = 1; q < parts; ++q) M = max_nan(M, cluster.map_shared_rank(&sh, q)->m);
            S = U = 0.0f;
            for (int q = 0; q < parts; ++q) {
                const Shared* o = cluster.map_shared_rank(&sh, q);
                float ps = o->s, pu = o->u;
                rescale(o->m, ps, pu, M, a.c);
                S += ps;
                U += pu;
            }
            if (Top) {
                if (threadIdx.x == 0) sh.count = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < parts * a.top; i += blockDim.x) {
                    const uint64_t k = cluster.map_shared_rank(&sh, i / a.top)->best[i % a.top];
                    if (k) offer(sh, k);
                }
                __syncthreads();
                rank_select(sh, sh.count, a.top);
            }
        }
        const bool empty = M == -INFINITY, undefined = !(M < INFINITY);
        const float log_s = logf(S);
        if (threadIdx.x == 0) {
            float lp = 0.0f, h = 0.0f;
            if (undefined) {
                lp = h = NAN;
            } else {
                if (!empty) h = fmaxf(log_s - __fdiv_rn(U, S) * kLn2, 0.0f);
                if ((uint64_t)token < (uint64_t)a.vocab) lp = empty ? -INFINITY : log_prob(x_t, M, a.inv_t, log_s);
            }
            a.logprobs[r] = lp;
            a.entropy[r] = h;
            if (a.stats)
                a.stats[r] = make_float4(empty ? 0.0f : M, empty ? 1.0f : S, h, undefined ? NAN : empty ? 0.0f : 1.0f);
        }
        if (Top) {
            for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
                const uint64_t k = undefined ? 0 : sh.best[i];
                a.top_tokens[r * a.top + i] = k ? key_col(k) : -1;
                a.top_logprobs[r * a.top + i] =
                    undefined ? NAN : k ? log_prob(key_logit(k), M, a.inv_t, log_s) : -INFINITY;
            }
        }
    }
    if (parts > 1) cluster.sync();  // the others' shared memory stays until it has been read
}

// ---------------------------------------------------------------- gradient
struct GradArgs {
    const void* logits;
    int64_t ld, out_ld;
    int32_t vocab;
    const int64_t* tokens;
    float c, inv_t;
    int top;
    const int64_t* top_tokens;
    const float4* stats;
    const float *g_logprobs, *g_entropy, *g_top;
    void* out;
    int blocks_per_row;
};

struct RowGrad {
    float m, inv_s, log_s, h, g, gh, c, inv_t;
    // -p (G + gH (ln p + H)) before 1 / T
    __device__ __forceinline__ float dense(float x) const {
        const float y = fmaxf((x - m) * c, kLowest), p = ex2(y) * inv_s;
        return -p * fmaf(gh, fmaf(y, kLn2, h - log_s), g);
    }
};

template <class T, bool Wide>
__global__ void __launch_bounds__(kMaxThreads) logprobs_grad_kernel(GradArgs a) {
    constexpr int VE = RowView<T>::VE;
    const int64_t r = blockIdx.x / (unsigned)a.blocks_per_row;
    const int chunk = (int)(blockIdx.x - r * a.blocks_per_row);
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    T* out = static_cast<T*>(a.out) + r * a.out_ld;
    const float4 st = a.stats[r];
    const bool live = st.w == 1.0f;
    const int64_t token = a.tokens[r];
    const bool given = (uint64_t)token < (uint64_t)a.vocab;
    const float gl = a.g_logprobs && given ? a.g_logprobs[r] : 0.0f;
    RowGrad rg;
    rg.m = st.x;
    rg.inv_s = __fdiv_rn(1.0f, st.y);
    rg.log_s = logf(st.y);
    rg.h = st.z;
    rg.g = gl;
    rg.gh = a.g_entropy ? a.g_entropy[r] : 0.0f;
    rg.c = a.c;
    rg.inv_t = a.inv_t;
    if (a.g_top)
        for (int k = 0; k < a.top; ++k)
            if (a.top_tokens[r * a.top + k] >= 0) rg.g += a.g_top[r * a.top + k];
    if (!(st.w == st.w)) rg.g = NAN;

    const RowView<T> view(row, a.vocab);
    const int nvec = view.vectors(), per = kMaxThreads * kUnroll;
    const int v0 = chunk * per, v1 = min(nvec, v0 + per);
    Pack<T, VE> p[kUnroll];
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
        const int i = v0 + q * kMaxThreads + threadIdx.x;
        if (i < v1) p[q] = view.load(i);
    }
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
        const int i = v0 + q * kMaxThreads + threadIdx.x;
        if (i >= v1) continue;
        Pack<T, VE> d;
#pragma unroll
        for (int k = 0; k < VE; ++k) d.v[k] = from_f32<T>(rg.dense(to_f32(p[q].v[k])) * a.inv_t);
        const int64_t e = view.first(i);
        if (Wide && e >= 0 && e + VE <= a.vocab) {
            *reinterpret_cast<Pack<T, VE>*>(out + e) = d;
        } else {
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (e + k >= 0 && e + k < a.vocab) out[e + k] = d.v[k];
        }
    }
    // the given token and the alternatives have terms of their own
    if (!live) return;
    __syncthreads();
    const int64_t e0 = view.first(v0), e1 = view.first(v1);
    for (int i = threadIdx.x; i <= a.top; i += kMaxThreads) {
        if (i > 0 && !a.g_top) break;
        const int64_t v = i == 0 ? token : a.top_tokens[r * a.top + i - 1];
        if ((uint64_t)v >= (uint64_t)a.vocab || v < e0 || v >= e1) continue;
        float own = v == token ? gl : 0.0f;
        if (a.g_top)
            for (int k = 0; k < a.top; ++k)
                if (a.top_tokens[r * a.top + k] == v) own += a.g_top[r * a.top + k];
        out[v] = from_f32<T>((own + rg.dense(to_f32(row[v]))) * a.inv_t);
    }
}

// ---------------------------------------------------------------- neighbours
struct NearArgs {
    const void* logits;
    int64_t ld;
    int32_t vocab;
    const int64_t* tokens;
    double inv_t;
    int top;
    const float4* stats;
    const int64_t* ids;
    const float* distances;
    const int64_t* values;
    int64_t n_values;
    int k;
    double weight, inv_tau;
    float *logprobs, *entropy;
    int64_t* top_tokens;
    float* top_logprobs;
};

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += red[w];
    return v;
}

// One block per row.  Everything here is f64: there are at most k + top values per row, and
// the alternatives are ordered by sums of two sources, which f32 would tie or swap.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) neighbours_kernel(NearArgs a) {
    __shared__ int32_t tok[kMaxNeighbours];    // a neighbour's token, -1 where it does not count
    __shared__ double wgt[kMaxNeighbours];     // its weight
    __shared__ double cp[kMaxNeighbours + kMaxTop];    // candidates: log probability, token
    __shared__ int32_t ct[kMaxNeighbours + kMaxTop];
    __shared__ double red[kMaxThreads / 32];
    __shared__ int n_cand;
    __shared__ double lp_token;  // of the given token; NaN: no neighbour's
    const int64_t r = blockIdx.x;
    const float4 st = a.stats[r];
    if (st.w != 1.0f) return;  // empty and undefined rows stay as they are
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    const double m = st.x, log_s = log((double)st.y);
    const int64_t given = a.tokens[r];
    if (threadIdx.x == 0) {
        n_cand = 0;
        lp_token = NAN;
    }
    // which neighbours count, and the nearest of them
    float near = INFINITY;
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        const int64_t id = a.ids[r * a.k + j];
        const float d = a.distances[r * a.k + j];
        int64_t t = -1;
        if ((uint64_t)id < (uint64_t)a.n_values && fabsf(d) < INFINITY) t = a.values[id];
        if ((uint64_t)t >= (uint64_t)a.vocab || !(to_f32(row[t]) > -INFINITY)) t = -1;
        tok[j] = (int32_t)t;
        if (t >= 0) near = fminf(near, d);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) near = fminf(near, __shfl_xor_sync(0xffffffffu, near, d));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = near;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) near = fminf(near, (float)red[w]);
    if (near == INFINITY) return;  // no neighbour: the model's distribution alone
    double sum = 0.0;
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        double w = 0.0;
        if (tok[j] >= 0) w = exp(((double)near - (double)a.distances[r * a.k + j]) * a.inv_tau);
        wgt[j] = w;
        sum += w;
    }
    const double scale = a.weight / block_sum(sum, red);
    const double keep = 1.0 - a.weight, log_keep = log(keep);
    // the first neighbour with a token carries the token
    double mass = 0.0, q_log_q = 0.0, h = 0.0;
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        const int32_t t = tok[j];
        if (t < 0) continue;
        bool first = true;
        for (int i = 0; i < j; ++i) first = first && tok[i] != t;
        if (!first) continue;
        double w = wgt[j];
        for (int i = j + 1; i < a.k; ++i)
            if (tok[i] == t) w += wgt[i];
        const double log_q = ((double)to_f32(row[t]) - m) * a.inv_t - log_s, q = exp(log_q);
        const double p = keep * q + w * scale;
        mass += q;
        if (q > 0.0) q_log_q += q * log_q;
        // a probability below f64's range keeps its logarithm
        const double lp = p > 0.0 ? log(p) : log_keep + log_q;
        if (p > 0.0) h -= p * lp;
        if (t == given) lp_token = lp;
        const int at = atomicAdd(&n_cand, 1);
        cp[at] = lp;
        ct[at] = t;
    }
    mass = block_sum(mass, red);
    q_log_q = block_sum(q_log_q, red);
    h = block_sum(h, red);
    if (threadIdx.x == 0) {
        const double rest = fmax(1.0 - mass, 0.0);
        if (keep > 0.0) h -= keep * (log_keep * rest - (double)st.z - q_log_q);
        a.entropy[r] = (float)fmax(h, 0.0);
        if ((uint64_t)given < (uint64_t)a.vocab) {
            double lp = lp_token;
            if (lp != lp) lp = log_keep + ((double)to_f32(row[given]) - m) * a.inv_t - log_s;
            a.logprobs[r] = (float)lp;
        }
    }
    if (a.top == 0) return;
    const int n_near = n_cand;
    __syncthreads();
    // the model's alternatives that are no neighbour's token
    for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
        const int64_t t = a.top_tokens[r * a.top + i];
        if (t < 0) continue;
        bool mine = true;
        for (int j = 0; j < n_near; ++j) mine = mine && ct[j] != t;
        if (!mine) continue;
        const int at = atomicAdd(&n_cand, 1);
        cp[at] = log_keep + ((double)to_f32(row[t]) - m) * a.inv_t - log_s;
        ct[at] = (int32_t)t;
    }
    __syncthreads();
    const int n = n_cand;
    for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
        a.top_tokens[r * a.top + i] = -1;
        a.top_logprobs[r * a.top + i] = -INFINITY;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const double lp = cp[i];
        if (!(lp > -INFINITY)) continue;
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += cp[j] > lp || (cp[j] == lp && ct[j] < ct[i]);
        if (rank < a.top) {
            a.top_tokens[r * a.top + rank] = ct[i];
            a.top_logprobs[r * a.top + rank] = (float)lp;
        }
    }
}

// ---------------------------------------------------------------- host
void check_probs(const hanns_token_logprobs_t* t) {
    require(t, "token_logprobs: null arguments");
    require(dtype_known(t->dtype), "token_logprobs: unknown element type");
    require(t->n >= 0 && t->n < 0x7fffffff, "token_logprobs: n must be in [0, 2^31 - 1)");
    require(t->vocab >= 1 && t->vocab < 0x7fffffff - 64, "token_logprobs: vocab must be in [1, 2^31 - 65)");
    require(t->top >= 0 && t->top <= kMaxTop, "token_logprobs: top must be in [0, 32]");
    require(t->temperature > 1e-30f && t->temperature < 1e30f, "token_logprobs: temperature must be positive and finite");
    if (t->n == 0) return;
    require(t->logits && t->tokens && t->logprobs && t->entropy, "token_logprobs: null logits, tokens or output");
    require((uintptr_t)t->logits % dtype_bytes(t->dtype) == 0, "token_logprobs: misaligned logits");
    require(t->top == 0 || (t->top_tokens && t->top_logprobs), "token_logprobs: null output of the alternatives");
    require((uintptr_t)t->stats % 16 == 0, "token_logprobs: stats must be 16-byte aligned");
}

int sm_count() {
    int dev = 0, n = 0;
    HANNS_CUDA_OK(cudaGetDevice(&dev));
    HANNS_CUDA_OK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    return n;
}

template <class T, bool Top>
void launch_probs(const hanns_token_logprobs_t* t, const ProbArgs& a, cudaStream_t s) {
    const int64_t vectors = (t->vocab + RowView<T>::VE - 1) / RowView<T>::VE + 1;
    // A cluster's blocks share a row when the rows alone do not give every SM two blocks,
    // as long as each block still has two rounds of full loads.
    int parts = 1;
    const int64_t want = 2 * sm_count();
    while (parts < kMaxCluster && t->n * parts * 2 <= want && vectors / (parts * 2) >= 2 * kMaxThreads) parts *= 2;
    int threads = 32;
    while (threads < kMaxThreads && vectors / parts > (int64_t)threads * kUnroll) threads *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(t->n * parts));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    HANNS_CUDA_OK(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, Top>, a));
}

template <class T>
void launch_grad(const hanns_token_logprobs_t* t, GradArgs a, cudaStream_t s) {
    const int64_t vectors = (t->vocab + RowView<T>::VE - 1) / RowView<T>::VE + 1;  // one more where a row starts inside a vector
    a.blocks_per_row = (int)((vectors + kMaxThreads * kUnroll - 1) / (kMaxThreads * kUnroll));
    require(t->n * a.blocks_per_row < 0x7fffffff, "token_logprobs: too many elements for one gradient call");
    // wide stores where each output row starts as its logits do within 16 bytes
    const bool wide = ((uintptr_t)a.logits - (uintptr_t)a.out) % 16 == 0 && ((a.ld - a.out_ld) * (int64_t)sizeof(T)) % 16 == 0;
    const unsigned grid = (unsigned)(t->n * a.blocks_per_row);
    if (wide) logprobs_grad_kernel<T, true><<<grid, kMaxThreads, 0, s>>>(a);
    else logprobs_grad_kernel<T, false><<<grid, kMaxThreads, 0, s>>>(a);
    HANNS_CUDA_OK(cudaGetLastError());
}

template <class T>
void launch_probs_typed(const hanns_token_logprobs_t* t, const ProbArgs& a, cudaStream_t s) {
    if (t->top) launch_probs<T, true>(t, a, s);
    else launch_probs<T, false>(t, a, s);
}

}  // namespace
}  // namespace hanns

// Declared in include/hanns_gpu.h.
extern "C" int32_t hanns_gpu_token_logprobs_device(const hanns_token_logprobs_t* t, void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_probs(t);
        if (t->n == 0) return;
        ProbArgs a{};
        a.logits = t->logits;
        a.ld = t->ld;
        a.vocab = (int32_t)t->vocab;
        a.tokens = t->tokens;
        a.c = (float)((double)kLog2e / t->temperature);
        a.inv_t = (float)(1.0 / t->temperature);
        a.top = t->top;
        a.logprobs = t->logprobs;
        a.entropy = t->entropy;
        a.top_tokens = t->top_tokens;
        a.top_logprobs = t->top_logprobs;
        a.stats = reinterpret_cast<float4*>(t->stats);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (t->dtype == HANNS_DTYPE_F32) launch_probs_typed<float>(t, a, s);
        else if (t->dtype == HANNS_DTYPE_F16) launch_probs_typed<__half>(t, a, s);
        else launch_probs_typed<__nv_bfloat16>(t, a, s);
    });
}

extern "C" int32_t hanns_gpu_token_logprobs_grad_device(const hanns_token_logprobs_t* t, const float* g_logprobs,
                                                        const float* g_entropy, const float* g_top, void* d_logits,
                                                        int64_t d_ld, void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_probs(t);
        if (t->n == 0) return;
        require(t->stats && d_logits, "token_logprobs: the gradient needs stats and an output");
        require((uintptr_t)d_logits % dtype_bytes(t->dtype) == 0, "token_logprobs: misaligned gradient");
        GradArgs a{};
        a.logits = t->logits;
        a.ld = t->ld;
        a.out_ld = d_ld;
        a.vocab = (int32_t)t->vocab;
        a.tokens = t->tokens;
        a.c = (float)((double)kLog2e / t->temperature);
        a.inv_t = (float)(1.0 / t->temperature);
        a.top = t->top;
        a.top_tokens = t->top_tokens;
        a.stats = reinterpret_cast<const float4*>(t->stats);
        a.g_logprobs = g_logprobs;
        a.g_entropy = g_entropy;
        a.g_top = t->top ? g_top : nullptr;
        a.out = d_logits;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (t->dtype == HANNS_DTYPE_F32) launch_grad<float>(t, a, s);
        else if (t->dtype == HANNS_DTYPE_F16) launch_grad<__half>(t, a, s);
        else launch_grad<__nv_bfloat16>(t, a, s);
    });
}

extern "C" int32_t hanns_gpu_neighbour_logprobs_device(const hanns_token_logprobs_t* t, const int64_t* d_ids,
                                                       const float* d_distances, int32_t k, const int64_t* d_values,
                                                       int64_t n_values, float weight, float knn_temperature,
                                                       void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_probs(t);
        require(k >= 0 && k <= kMaxNeighbours, "neighbour_logprobs: k must be in [0, 1024]");
        require(weight >= 0.0f && weight <= 1.0f, "neighbour_logprobs: weight must be in [0, 1]");
        require(knn_temperature > 1e-30f && knn_temperature < 1e30f,
                "neighbour_logprobs: temperature must be positive and finite");
        if (t->n == 0 || k == 0 || n_values <= 0 || weight == 0.0f) return;
        require(t->stats, "neighbour_logprobs: the model's statistics (stats) are needed");
        require(d_ids && d_distances && d_values, "neighbour_logprobs: null ids, distances or values");
        NearArgs a{};
        a.logits = t->logits;
        a.ld = t->ld;
        a.vocab = (int32_t)t->vocab;
        a.tokens = t->tokens;
        a.inv_t = 1.0 / t->temperature;
        a.top = t->top;
        a.stats = reinterpret_cast<const float4*>(t->stats);
        a.ids = d_ids;
        a.distances = d_distances;
        a.values = d_values;
        a.n_values = n_values;
        a.k = k;
        a.weight = weight;
        a.inv_tau = 1.0 / knn_temperature;
        a.logprobs = t->logprobs;
        a.entropy = t->entropy;
        a.top_tokens = t->top_tokens;
        a.top_logprobs = t->top_logprobs;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const unsigned threads = k <= 32 ? 32 : k <= 128 ? 128 : kMaxThreads;
        if (t->dtype == HANNS_DTYPE_F32) neighbours_kernel<float><<<(unsigned)t->n, threads, 0, s>>>(a);
        else if (t->dtype == HANNS_DTYPE_F16) neighbours_kernel<__half><<<(unsigned)t->n, threads, 0, s>>>(a);
        else neighbours_kernel<__nv_bfloat16><<<(unsigned)t->n, threads, 0, s>>>(a);
        HANNS_CUDA_OK(cudaGetLastError());
    });
}
