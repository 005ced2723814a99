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
// (rescaled when the maximum grows).  Exponents are in powers of two, y = x c - R with
// c = log2(e) / T and the reference R = m c as f32 rounds it: any R near m c serves, since the same
// one is taken off again, and y then has a single rounding.  Logits so far from 0 that R's rounding
// is many powers of two are summed from their differences (kNoRef).  For the alternatives each thread keeps
// the maxima of its two largest rounds of loads; the `top`-th of the threads' maxima bounds the
// row's `top`-th logit, and the few rounds that reach the bound are read again, from the L2.  A row
// is one block's, or a cluster's when there are few rows: each block of the cluster then takes a
// share of the columns and the first one joins them over distributed shared memory.
//
// neighbours_kernel mixes in the tokens of a search's neighbours:
//   w = softmax(-distance / tau),  p_v = (1 - l) q_v + l sum of w_j over neighbours j with token v
// It needs the statistics of q and its alternatives only: a token that is no neighbour's keeps
// its order among those, so the mixture's alternatives are among q's and the neighbours' tokens,
// and the entropy differs from q's in the neighbours' terms and the factor (1 - l).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "operators.cuh"

namespace hanns {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxThreads = 128;
constexpr int kUnroll = 4;
constexpr int kGradThreads = 128, kGradUnroll = 2;
constexpr int kGradRounds = 8;  // of a block, where there are blocks enough
constexpr int kMaxTop = 32;
constexpr int kCap = 1024;       // buffered candidate vectors of a block
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

// A row's elements as 16-byte vectors, numbered from the 16-byte boundary at or before its first
// one.  Those that the row fills are body[0 .. n); the vector before them and the one behind
// them may be filled in part and are read element by element, -inf outside the row.
template <class T>
struct RowView {
    static constexpr int VE = 16 / sizeof(T);
    const T* row;
    const Pack<T, VE>* body;
    int lead, vocab, n;
    __device__ __forceinline__ RowView(const T* r, int v)
        : row(r), lead((int)(((uintptr_t)r & 15) / sizeof(T))), vocab(v) {
        const int head = lead ? min(VE - lead, vocab) : 0;
        body = reinterpret_cast<const Pack<T, VE>*>(row + head);
        n = (vocab - head) / VE;
    }
    __device__ __forceinline__ int skipped() const { return lead ? 1 : 0; }  // vectors before the body
    __device__ __forceinline__ int64_t first(int64_t i) const { return i * VE - lead; }
    __device__ __forceinline__ Pack<T, VE> edge(int64_t i) const {
        const int64_t e = first(i);
        Pack<T, VE> p;
#pragma unroll
        for (int k = 0; k < VE; ++k)
            p.v[k] = e + k >= 0 && e + k < vocab ? row[e + k] : from_f32<T>(-INFINITY);
        return p;
    }
    __device__ __forceinline__ Pack<T, VE> load(int64_t i) const {
        const int64_t j = i - skipped();
        return j >= 0 && j < n ? body[j] : edge(i);
    }
    // all vectors, the partial ones among them
    __device__ __forceinline__ int vectors() const { return (int)(((int64_t)lead + vocab + VE - 1) / VE); }
};

// The larger of two words' 16-bit elements, two by two (`max_pairs` keeps a NaN, `raise_pairs`
// drops it).
template <class T> __device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max_pairs<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <> __device__ __forceinline__ uint32_t max_pairs<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <class T> __device__ __forceinline__ uint32_t raise_pairs(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t raise_pairs<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <> __device__ __forceinline__ uint32_t raise_pairs<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <class T> __device__ __forceinline__ uint32_t pack_pair(float2 v);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ uint4 words(const Pack<T, 8>& p) {
    return *reinterpret_cast<const uint4*>(&p);
}

// 16-bit elements are raised to `floor` before their exponent, two per instruction, so that a
// masked -inf has a finite y (2^y y is then 0 and not NaN).  A row whose maximum is not well
// above the floor is summed again from its differences (see row_needs_differences).
template <class T> __device__ __forceinline__ float floor_of();
template <> __device__ __forceinline__ float floor_of<float>() { return -INFINITY; }
template <> __device__ __forceinline__ float floor_of<__half>() { return -65504.0f; }
template <> __device__ __forceinline__ float floor_of<__nv_bfloat16>() { return -0x1p100f; }
template <class T> __device__ __forceinline__ uint32_t floor_pair();  // the same, twice in a word
template <> __device__ __forceinline__ uint32_t floor_pair<__half>() { return 0xfbfffbffu; }
template <> __device__ __forceinline__ uint32_t floor_pair<__nv_bfloat16>() { return 0xf180f180u; }

// y of a vector's elements against the reference R, as pairs.
template <class T>
__device__ __forceinline__ void exponents(const Pack<T, 8>& p, float c, float ref, float2 (&y)[4]) {
    const uint4 w = words(p);
    const float2 c2 = make_float2(c, c), r2 = make_float2(-ref, -ref);
    y[0] = fma2_rn(pair_f32<T>(raise_pairs<T>(w.x, floor_pair<T>())), c2, r2);
    y[1] = fma2_rn(pair_f32<T>(raise_pairs<T>(w.y, floor_pair<T>())), c2, r2);
    y[2] = fma2_rn(pair_f32<T>(raise_pairs<T>(w.z, floor_pair<T>())), c2, r2);
    y[3] = fma2_rn(pair_f32<T>(raise_pairs<T>(w.w, floor_pair<T>())), c2, r2);
}
__device__ __forceinline__ void exponents(const Pack<float, 4>& p, float c, float ref, float2 (&y)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        y[i] = fma2_rn(make_float2(p.v[2 * i], p.v[2 * i + 1]), make_float2(c, c), make_float2(-ref, -ref));
        y[i].x = fmaxf(y[i].x, kLowest);
        y[i].y = fmaxf(y[i].y, kLowest);
    }
}

// References are kept to 2^27 in magnitude, where R's rounding moves y by 4 at most (at 1e10 it would
// be 512 and 2^512 no f32).  A thread whose logits all lie below takes -2^27 itself: against that
// they are 2^-200, which is right unless the whole row lies there.
constexpr float kNoRef = -0x1p27f;

// Largest element, NaN if there is one.
__device__ __forceinline__ float pack_max(const Pack<float, 4>& p) {
    return max_nan(max_nan(p.v[0], p.v[1]), max_nan(p.v[2], p.v[3]));
}
template <class T>
__device__ __forceinline__ uint32_t pair_max(const Pack<T, 8>& p) {
    const uint4 w = words(p);
    return max_pairs<T>(max_pairs<T>(w.x, w.y), max_pairs<T>(w.z, w.w));
}
template <class T>
__device__ __forceinline__ float pack_max(const Pack<T, 8>& p) {
    const float2 v = pair_f32<T>(pair_max(p));
    return max_nan(v.x, v.y);
}
// Of several vectors.
template <int N>
__device__ __forceinline__ float packs_max(const Pack<float, 4> (&p)[N]) {
    float v = pack_max(p[0]);
#pragma unroll
    for (int q = 1; q < N; ++q) v = max_nan(v, pack_max(p[q]));
    return v;
}
template <class T, int N>
__device__ __forceinline__ float packs_max(const Pack<T, 8> (&p)[N]) {
    uint32_t w = pair_max(p[0]);
#pragma unroll
    for (int q = 1; q < N; ++q) w = max_pairs<T>(w, pair_max(p[q]));
    const float2 v = pair_f32<T>(w);
    return max_nan(v.x, v.y);
}

// f (u + d s), f s for the factor f = 2^d that moves sums from one reference to another.
__device__ __forceinline__ void rescale(float d, float& s, float& u) {
    d = fmaxf(d, kLowest);
    const float f = ex2(d);
    u = f * fmaf(d, s, u);
    s *= f;
}

// Sums of 2^y and of 2^y y of one thread, two of each so that pairs add up in one instruction.
template <class T>
struct Running {
    float m = -INFINITY, ref;
    float2 s = make_float2(0.0f, 0.0f), u = make_float2(0.0f, 0.0f);
    // masked elements before the first live one may count as 2^0 against the floor, which a row's
    // maximum far above it makes nothing of
    __device__ __forceinline__ explicit Running(float c)
        : ref(sizeof(T) == 2 ? fmaxf(floor_of<T>() * c, kNoRef) : kNoRef) {}
    // before elements of maximum vm are added
    __device__ __forceinline__ void reach(float vm, float c) {
        if (!(vm <= m)) {
            m = max_nan(vm, m);
            const float to = fmaxf((sizeof(T) == 2 ? fmaxf(m, floor_of<T>()) : m) * c, kNoRef), d = ref - to;
            rescale(d, s.x, u.x);
            rescale(d, s.y, u.y);
            ref = to;
        }
    }
    __device__ __forceinline__ void add(const Pack<T, RowView<T>::VE>& p, float c) {
        constexpr int N = RowView<T>::VE / 2;
        float2 y[N];
        exponents(p, c, ref, y);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 e = make_float2(ex2(y[i].x), ex2(y[i].y));
            s = add2_rn(s, e);
            u = fma2_rn(e, y[i], u);
        }
    }
};

// Rows for which y = x c - R is not good enough: the maximum is too far from 0 for a reference, the
// floor overflows, or masked elements at the floor would count (a maximum near the type's lowest
// value, a very high or low temperature).  They are read again and summed from (x - m) c.
template <class T>
__device__ __forceinline__ bool row_needs_differences(float m, float c) {
    bool bad = !(fabsf(m * c) < -kNoRef);
    if (sizeof(T) == 2) bad = bad || !(floor_of<T>() * c > -1e37f) || !((floor_of<T>() - m) * c < -150.0f);
    return bad;
}

// Buffers in shared memory from which the threads of a group (a block, or a warp) choose.
struct Choice {
    uint64_t* buf;   // candidate vectors: order of the maximum, then the lower vector
    int cap;         // a warp's holds every vector of its row; a block's may drop some
    uint64_t* elem;  // elements of the best vectors, kMaxTop * 8
    uint64_t* best;  // the alternatives, best first, kMaxTop
    int* count;      // candidates offered (may pass cap: then some were dropped)
    __device__ __forceinline__ void offer(uint64_t key) const {
        const int at = atomicAdd(count, 1);
        if (at < cap) buf[at] = key;
    }
};
struct BlockGroup {
    static __device__ __forceinline__ int rank() { return threadIdx.x; }
    static __device__ __forceinline__ int size() { return blockDim.x; }
    static __device__ __forceinline__ void sync() { __syncthreads(); }
};
struct WarpGroup {
    static __device__ __forceinline__ int rank() { return threadIdx.x & 31; }
    static __device__ __forceinline__ int size() { return 32; }
    static __device__ __forceinline__ void sync() { __syncwarp(); }
};

// out[0 .. top) = the largest of n different keys, 0 behind them.  Needs a barrier before,
// ends with one.
template <class Group>
__device__ __forceinline__ void rank_select(const uint64_t* keys, int n, uint64_t* out, int top) {
    for (int i = Group::rank(); i < n; i += Group::size()) {
        const uint64_t k = keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += keys[j] > k;
        if (rank < top) out[rank] = k;
    }
    for (int i = n + Group::rank(); i < top; i += Group::size()) out[i] = 0;
    Group::sync();
}

// This lane's key's place among the warp's (ties by lane).
__device__ __forceinline__ int warp_rank(uint32_t key) {
    const int lane = threadIdx.x & 31;
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const uint32_t o = __shfl_sync(0xffffffffu, key, j);
        rank += o > key || (o == key && j < lane);
    }
    return rank;
}
__device__ __forceinline__ uint32_t max_key(float vm) { return vm != vm ? 0xffffffffu : total_order_key(vm); }
// The `top`-th largest of the lanes' keys, as a logit.
__device__ __forceinline__ float warp_threshold(uint32_t key, int top) {
    const int at = __ffs(__ballot_sync(0xffffffffu, warp_rank(key) == top - 1)) - 1;
    const uint32_t low = __shfl_sync(0xffffffffu, key, at);
    return low <= kKeyMinusInf ? -INFINITY : key_to_float(low);
}

// best[] from the buffered vectors: the `top` best vectors hold the `top` best elements (each
// vector before an element's own has an element before it).  Needs a barrier before, ends
// with one.
template <class Group, class T>
__device__ void select_elements(const Choice& ch, const RowView<T>& view, int top) {
    constexpr int VE = RowView<T>::VE;
    rank_select<Group>(ch.buf, min(*ch.count, ch.cap), ch.best, top);
    const uint64_t least = ch.best[top - 1];  // as many elements as this vector's maximum are no worse
    const float bound = least ? key_logit(least) : -INFINITY;
    if (Group::rank() == 0) *ch.count = 0;
    Group::sync();
    for (int i = Group::rank(); i < top * VE; i += Group::size()) {
        const uint64_t v = ch.best[i / VE];
        const int64_t e = v ? view.first(key_col(v)) + i % VE : -1;
        if (e < 0 || e >= view.vocab) continue;
        const float x = to_f32(view.row[e]);
        if (x > -INFINITY && x >= bound) ch.elem[atomicAdd(ch.count, 1)] = cand_key(x, (int32_t)e);
    }
    Group::sync();
    rank_select<Group>(ch.elem, *ch.count, ch.best, top);
}

struct Shared {
    uint64_t buf[kCap], elem[kMaxTop * 8], best[kMaxTop];
    uint32_t hist[256];
    float wm[kMaxThreads / 32], wr[kMaxThreads / 32], ws[kMaxThreads / 32], wu[kMaxThreads / 32];
    uint32_t lead[32];       // maxima of groups of threads
    float thr;
    int count;
    float m, ref, s, u;      // of this block's columns
    __device__ __forceinline__ Choice choice() { return Choice{buf, kCap, elem, best, &count}; }
};

// Lower bound of the row's `top`-th logit: the `top`-th of the 32 maxima that groups of threads
// have in their columns.
__device__ float block_threshold(Shared& sh, float vm, int top) {
    constexpr int kGroup = kMaxThreads / 32;
    uint32_t key = max_key(vm);
#pragma unroll
    for (int d = 1; d < kGroup; d <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, d));
    if (threadIdx.x % kGroup == 0) sh.lead[threadIdx.x / kGroup] = key;
    __syncthreads();
    if (threadIdx.x < 32) {
        const float thr = warp_threshold(sh.lead[threadIdx.x], top);
        if (threadIdx.x == 0) sh.thr = thr;
    }
    __syncthreads();
    return sh.thr;
}

// Candidates were dropped (ties by the thousand): find by counting key
// bytes, highest first, a bound that at least `top` and at most kCap elements reach, collect
// those and take the best.  Reads the columns up to nine times.
template <class T>
__device__ void select_again(Shared& sh, const RowView<T>& view, int v0, int v1, int top) {
    const int64_t e0 = max((int64_t)0, view.first(v0)), e1 = min((int64_t)view.vocab, view.first(v1));
    uint64_t prefix = 0, low = 0;
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
        low = prefix << (8 * byte);
        if (reach <= kCap) break;
        need -= above;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int64_t e = e0 + threadIdx.x; e < e1; e += blockDim.x) {
        const float x = to_f32(view.row[e]);
        if (!(x > -INFINITY)) continue;
        const uint64_t k = cand_key(x, (int32_t)e);
        if (k >= low) sh.choice().offer(k);
    }
    __syncthreads();
    rank_select<BlockGroup>(sh.buf, min(sh.count, kCap), sh.best, top);
}

// A row's outputs from its maximum, reference and sums.
template <class Group>
__device__ __forceinline__ void write_row(const ProbArgs& a, int64_t r, int64_t token, float x_t, float m, float ref,
                                          float s, float u, bool differences, const uint64_t* best) {
    const bool empty = m == -INFINITY, undefined = !(m < INFINITY);
    // the sum of e^((x - m) / T): the reference is m c but for f32's rounding of it
    const float s_m = differences ? s : s * exp2f(-fmaf(m, a.c, -ref)), log_s = logf(s_m);
    if (Group::rank() == 0) {
        float lp = 0.0f, h = 0.0f;
        if (undefined) {
            lp = h = NAN;
        } else {
            if (!empty) h = fmaxf(logf(s) - __fdiv_rn(u, s) * kLn2, 0.0f);
            if ((uint64_t)token < (uint64_t)a.vocab) lp = empty ? -INFINITY : log_prob(x_t, m, a.inv_t, log_s);
        }
        a.logprobs[r] = lp;
        a.entropy[r] = h;
        if (a.stats)
            a.stats[r] = make_float4(empty ? 0.0f : m, empty ? 1.0f : s_m, h, undefined ? NAN : empty ? 0.0f : 1.0f);
    }
    for (int i = Group::rank(); i < a.top; i += Group::size()) {
        const uint64_t k = undefined ? 0 : best[i];
        a.top_tokens[r * a.top + i] = k ? key_col(k) : -1;
        a.top_logprobs[r * a.top + i] = undefined ? NAN : k ? log_prob(key_logit(k), m, a.inv_t, log_s) : -INFINITY;
    }
}

// A block's share of a row: vectors [v0, v1), of them [b0, b1) of the body.
template <class T>
struct Columns {
    RowView<T> view;
    int v0, v1, b0, b1;
    __device__ __forceinline__ Columns(const ProbArgs& a, int64_t r, int part, int parts)
        : view(static_cast<const T*>(a.logits) + r * a.ld, a.vocab) {
        const int nvec = view.vectors(), per = (nvec + parts - 1) / parts;
        v0 = min(nvec, part * per);
        v1 = min(nvec, v0 + per);
        b0 = max(0, v0 - view.skipped());
        b1 = min(view.n, v1 - view.skipped());
    }
    // a round of kUnroll vectors per thread, -inf behind the last
    __device__ __forceinline__ void fetch(int base, Pack<T, RowView<T>::VE> (&p)[kUnroll]) const {
        const Pack<T, RowView<T>::VE>* src = view.body + base + threadIdx.x;
        if (base + (int)blockDim.x * kUnroll <= b1) {
#pragma unroll
            for (int q = 0; q < kUnroll; ++q) p[q] = src[q * blockDim.x];
        } else {
#pragma unroll
            for (int q = 0; q < kUnroll; ++q) {
                if (base + q * (int)blockDim.x + (int)threadIdx.x < b1) {
                    p[q] = src[q * blockDim.x];
                } else {
#pragma unroll
                    for (int k = 0; k < RowView<T>::VE; ++k) p[q].v[k] = from_f32<T>(-INFINITY);
                }
            }
        }
    }
};

// Without alternatives a block takes a row after the other, and the first round of the next one is
// on the way while a row is brought to its end (4096 x 128,000 bf16: 176 -> 174 us, 4099 x 50,257:
// 80 -> 77).  With them it takes one: their second look at the row would wait behind that round
// (with 5 alternatives: 93 -> 107 us).
template <class T, bool Top>
__global__ void __launch_bounds__(kMaxThreads, 8) logprobs_kernel(ProbArgs a, int64_t n) {
    wait_for_previous();
    constexpr int VE = RowView<T>::VE;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    int64_t r = blockIdx.x / parts;
    Columns<T> c(a, r, part, parts);
    Pack<T, VE> p[kUnroll];
    c.fetch(c.b0, p);
    while (true) {
        const RowView<T>& view = c.view;
        const T* row = view.row;
        const int v0 = c.v0, v1 = c.v1, b0 = c.b0, b1 = c.b1;
        int64_t token = -1;
        float x_t = 0.0f;
        if (part == 0 && threadIdx.x == 0) {
            token = a.tokens[r];
            if ((uint64_t)token < (uint64_t)a.vocab) x_t = to_f32(row[token]);
        }
        if (threadIdx.x == 0) sh.count = 0;

        Running<T> run(a.c);
        float best = -INFINITY, second = -INFINITY, third = -INFINITY;  // largest maxima of this thread's rounds
        int best_round = 0, second_round = 0;
        const int step = blockDim.x * kUnroll;
        int round = 0;
        for (int base = b0; base < b1; base += step, ++round) {
            if (round) c.fetch(base, p);
            const float vm = packs_max(p);
            if (Top) {
                third = fmaxf(third, fminf(second, vm));
                if (vm > second) {
                    const bool first = vm > best;
                    second = first ? best : vm;
                    second_round = first ? best_round : round;
                    best = first ? vm : best;
                    best_round = first ? round : best_round;
                }
            }
            run.reach(vm, a.c);
#pragma unroll
            for (int q = 0; q < kUnroll; ++q) run.add(p[q], a.c);
        }
        const int64_t next_r = r + gridDim.x / parts;
        const Columns<T> next(a, min(next_r, n - 1), part, parts);
        if (!Top && next_r < n) next.fetch(next.b0, p);
        // the alternatives' candidates: a thread whose maxima reach the threshold reads those rounds
        // again; where a third one does, its warp reads all of that thread's rounds
        float thr = -INFINITY;
        if (Top) {
            thr = block_threshold(sh, best, a.top);
            auto offer_vector = [&](int j) {
                const float pm = pack_max(view.body[j]);
                if (pm >= thr && pm > -INFINITY) sh.choice().offer(cand_key(pm, view.skipped() + j));
            };
            const bool many = third >= thr && third > -INFINITY;
            if (!many) {
                for (int k = 0; k < 2; ++k) {
                    if ((k ? second : best) < thr || (k ? second : best) == -INFINITY) break;
                    const int j = b0 + (k ? second_round : best_round) * step + (int)threadIdx.x;
#pragma unroll
                    for (int q = 0; q < kUnroll; ++q)
                        if (j + q * (int)blockDim.x < b1) offer_vector(j + q * (int)blockDim.x);
                }
            }
            for (uint32_t who = __ballot_sync(0xffffffffu, many); who; who &= who - 1) {
                const int j0 = b0 + (int)(threadIdx.x & ~31u) + __ffs(who) - 1;
                for (int j = j0 + (int)(threadIdx.x & 31) * (int)blockDim.x; j < b1; j += 32 * (int)blockDim.x)
                    offer_vector(j);
            }
        }
        // the partial vectors at the row's ends
        if (threadIdx.x < 2) {
            const int i = threadIdx.x ? view.skipped() + view.n : 0;
            if ((threadIdx.x || view.skipped()) && i >= v0 && i < v1) {
                const Pack<T, VE> p = view.edge(i);
                const float vm = pack_max(p);
                if (Top && vm >= thr && vm > -INFINITY) sh.choice().offer(cand_key(vm, i));
                run.reach(vm, a.c);
                run.add(p, a.c);
            }
        }

        // the warp's sums against its largest reference, then the block's
        float m = run.m, ref = run.ref, s = run.s.x + run.s.y, u = run.u.x + run.u.y;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
            ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, d));
        }
        rescale(run.ref - ref, s, u);
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, d);
            u += __shfl_xor_sync(0xffffffffu, u, d);
        }
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            sh.wm[warp] = m;
            sh.wr[warp] = ref;
            sh.ws[warp] = s;
            sh.wu[warp] = u;
        }
        __syncthreads();
        m = sh.wm[0];
        ref = sh.wr[0];
        for (int w = 1; w < warps; ++w) {
            m = max_nan(m, sh.wm[w]);
            ref = fmaxf(ref, sh.wr[w]);
        }
        s = u = 0.0f;
        for (int w = 0; w < warps; ++w) {
            float ps = sh.ws[w], pu = sh.wu[w];
            rescale(sh.wr[w] - ref, ps, pu);
            s += ps;
            u += pu;
        }
        if (threadIdx.x == 0) {
            sh.m = m;
            sh.ref = ref;
            sh.s = s;
            sh.u = u;
        }
        if (Top) {
            if (sh.count > kCap) select_again(sh, view, v0, v1, a.top);
            else select_elements<BlockGroup>(sh.choice(), view, a.top);
        }
        if (parts > 1) {
            cluster.sync();
            for (int q = 0; q < parts; ++q) {
                const Shared* o = cluster.map_shared_rank(&sh, q);
                m = q ? max_nan(m, o->m) : o->m;
                ref = q ? fmaxf(ref, o->ref) : o->ref;
            }
        }
        const bool empty = m == -INFINITY, undefined = !(m < INFINITY);
        const bool differences = !empty && !undefined && row_needs_differences<T>(m, a.c);
        if (differences) {
            s = u = 0.0f;
            const int64_t e1 = min((int64_t)a.vocab, view.first(v1));
            for (int64_t e = max((int64_t)0, view.first(v0)) + threadIdx.x; e < e1; e += blockDim.x) {
                const float y = fmaxf((to_f32(row[e]) - m) * a.c, kLowest), f = ex2(y);
                s += f;
                u = fmaf(f, y, u);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, d);
                u += __shfl_xor_sync(0xffffffffu, u, d);
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 0) {
                sh.ws[warp] = s;
                sh.wu[warp] = u;
            }
            __syncthreads();
            s = u = 0.0f;
            for (int w = 0; w < warps; ++w) {
                s += sh.ws[w];
                u += sh.wu[w];
            }
            if (threadIdx.x == 0) {
                sh.s = s;
                sh.u = u;
            }
            if (parts > 1) cluster.sync();
        }
        if (part == 0) {
            if (parts > 1) {
                s = u = 0.0f;
                for (int q = 0; q < parts; ++q) {
                    const Shared* o = cluster.map_shared_rank(&sh, q);
                    float ps = o->s, pu = o->u;
                    if (!differences) rescale(o->ref - ref, ps, pu);
                    s += ps;
                    u += pu;
                }
                if (Top) {
                    if (threadIdx.x == 0) sh.count = 0;
                    __syncthreads();
                    for (int i = threadIdx.x; i < parts * a.top; i += blockDim.x) {
                        const uint64_t k = cluster.map_shared_rank(&sh, i / a.top)->best[i % a.top];
                        if (k) sh.elem[atomicAdd(&sh.count, 1)] = k;
                    }
                    __syncthreads();
                    rank_select<BlockGroup>(sh.elem, sh.count, sh.best, a.top);
                }
            }
            write_row<BlockGroup>(a, r, token, x_t, m, ref, s, u, differences, sh.best);
        }
        if (parts > 1) cluster.sync();  // the others' shared memory stays until it has been read
        if (Top || next_r >= n) break;
        __syncthreads();
        r = next_r;
        c = next;
    }
}

// Short rows (8192 x 1000 bf16: 7.9 us, with 5 alternatives 14.3): a warp takes a row whose vectors
// (the partial ones among them) fit in its registers, U a lane, and goes on to another.
template <class T, bool Top, int U>
__global__ void __launch_bounds__(kMaxThreads, U > kUnroll ? 6 : 8) logprobs_rows_kernel(ProbArgs a, int64_t n) {
    wait_for_previous();
    constexpr int VE = RowView<T>::VE, kWarps = kMaxThreads / 32, kRowVectors = 32 * U;
    __shared__ uint64_t buf[kWarps][Top ? kRowVectors : 1], elem[kWarps][Top ? kMaxTop * 8 : 1];
    __shared__ uint64_t top_keys[kWarps][kMaxTop];
    __shared__ int count[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Choice ch{buf[warp], kRowVectors, elem[warp], top_keys[warp], &count[warp]};
    for (int64_t r = (int64_t)blockIdx.x * kWarps + warp; r < n; r += (int64_t)gridDim.x * kWarps) {
        const T* row = static_cast<const T*>(a.logits) + r * a.ld;
        const RowView<T> view(row, a.vocab);
        const int nvec = view.vectors();
        Pack<T, VE> p[U];
#pragma unroll
        for (int q = 0; q < U; ++q) {
            if (q * 32 + lane < nvec) {
                p[q] = view.load(q * 32 + lane);
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k) p[q].v[k] = from_f32<T>(-INFINITY);
            }
        }
        const int64_t token = a.tokens[r];
        const float x_t = (uint64_t)token < (uint64_t)a.vocab ? to_f32(row[token]) : 0.0f;
        const float vm = packs_max(p);
        float m = vm;
#pragma unroll
        for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
        const bool differences = m > -INFINITY && m < INFINITY && row_needs_differences<T>(m, a.c);
        Running<T> run(a.c);
        float s, u;
        if (!differences) {
            run.reach(m, a.c);  // nothing added yet: this sets the reference
#pragma unroll
            for (int q = 0; q < U; ++q)
                if (q * 32 < nvec) run.add(p[q], a.c);
            s = run.s.x + run.s.y;
            u = run.u.x + run.u.y;
        } else {
            s = u = 0.0f;
            for (int e = lane; e < a.vocab; e += 32) {
                const float y = fmaxf((to_f32(row[e]) - m) * a.c, kLowest), f = ex2(y);
                s += f;
                u = fmaf(f, y, u);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, d);
            u += __shfl_xor_sync(0xffffffffu, u, d);
        }
        if (Top) {
            if (lane == 0) count[warp] = 0;
            __syncwarp();
            const float thr = warp_threshold(max_key(vm), a.top);
            if (vm >= thr) {
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const float pm = pack_max(p[q]);
                    if (pm >= thr && pm > -INFINITY) ch.offer(cand_key(pm, q * 32 + lane));
                }
            }
            __syncwarp();
            select_elements<WarpGroup>(ch, view, a.top);
        }
        write_row<WarpGroup>(a, r, token, x_t, m, run.ref, s, u, differences, top_keys[warp]);
        __syncwarp();
    }
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
    int blocks_per_row, span;
};

// dx_v before its own terms: -p_v (G + gH (ln p_v + H)) / T = 2^y_v (base + slope y_v), where
// 2^y / s = p and ln p = y ln 2 - ln s.
struct RowGrad {
    float m, c, ref, base, slope;
    // from (x - m) c
    __device__ __forceinline__ float dense(float x) const {
        const float y = fmaxf((x - m) * c, kLowest);
        return ex2(y) * fmaf(slope, y, base);
    }
};

// Of a vector; the reference here is m c itself, so y is off by its rounding, which `base` and
// `slope` take back (they are of the sum against that reference).
template <class T>
__device__ __forceinline__ void dense_vector(const RowGrad& g, const Pack<T, 8>& p, Pack<T, 8>& d) {
    float2 y[4];
    exponents(p, g.c, g.ref, y);
    uint32_t* out = reinterpret_cast<uint32_t*>(&d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = fma2_rn(y[i], make_float2(g.slope, g.slope), make_float2(g.base, g.base));
        const float2 v = mul2_rn(make_float2(ex2(y[i].x), ex2(y[i].y)), f);
        out[i] = pack_pair<T>(v);
    }
}
__device__ __forceinline__ void dense_vector(const RowGrad& g, const Pack<float, 4>& p, Pack<float, 4>& d) {
    float2 y[2];
    exponents(p, g.c, g.ref, y);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = fma2_rn(y[i], make_float2(g.slope, g.slope), make_float2(g.base, g.base));
        d.v[2 * i] = ex2(y[i].x) * f.x;
        d.v[2 * i + 1] = ex2(y[i].y) * f.y;
    }
}

// Blocks take `span` vectors of a row each; its first block takes the partial ones at its ends.
// Bound by memory: 4096 x 128,000 bf16 take 318 us, 6.6 TB/s (313 behind the forward call, whose last
// logits are still in the L2).
template <class T, bool Wide>
__global__ void __launch_bounds__(kGradThreads, 12) logprobs_grad_kernel(GradArgs a) {
    wait_for_previous();
    constexpr int VE = RowView<T>::VE;
    const int64_t r = blockIdx.x / (unsigned)a.blocks_per_row;
    const int part = (int)(blockIdx.x - r * a.blocks_per_row);
    const T* row = static_cast<const T*>(a.logits) + r * a.ld;
    T* out = static_cast<T*>(a.out) + r * a.out_ld;
    const RowView<T> view(row, a.vocab);
    const int b0 = min(view.n, part * a.span), b1 = min(view.n, b0 + a.span);
    const float4 st = a.stats[r];
    const bool live = st.w == 1.0f, undefined = !(st.w == st.w);
    const int64_t token = a.tokens[r];
    const bool given = (uint64_t)token < (uint64_t)a.vocab;
    const float gl = a.g_logprobs && given ? a.g_logprobs[r] : 0.0f;
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.0f;
    float g = gl;
    if (a.g_top)
        for (int k = 0; k < a.top; ++k)
            if (a.top_tokens[r * a.top + k] >= 0) g += a.g_top[r * a.top + k];
    RowGrad rg;
    rg.m = st.x;
    rg.c = a.c;
    rg.ref = st.x * a.c;
    const float scale = -__fdiv_rn(a.inv_t, st.y);
    rg.base = scale * (g + gh * (st.z - logf(st.y)));
    rg.slope = scale * gh * kLn2;
    if (undefined) rg.base = NAN;
    if (!live) rg.m = rg.c = 0.0f;  // 2^0 base: NaN, or the zeros of an empty row
    if (!live && !undefined) rg.base = rg.slope = 0.0f;
    Pack<T, VE>* wide_out = reinterpret_cast<Pack<T, VE>*>(out + (view.skipped() ? view.first(1) : 0));
    auto store = [&](int j, const Pack<T, VE>& d) {
        if (Wide) {
            wide_out[j] = d;
        } else {
            const int64_t e = view.first(j + view.skipped());
#pragma unroll
            for (int k = 0; k < VE; ++k) out[e + k] = d.v[k];
        }
    };
    // a 16-bit element at the floor has 2^y = 0, which slope y must not turn into NaN (a large gradient of
    // the entropy, a low temperature); exponents of f32 logits and those from differences are clamped
    const bool steep = sizeof(T) == 2 && !(fabsf(floor_of<T>() * rg.c * rg.slope) < 1e37f);
    if (!live || steep || row_needs_differences<T>(st.x, a.c)) {
        for (int j = b0 + threadIdx.x; j < b1; j += kGradThreads) {
            const Pack<T, VE> p = view.body[j];
            Pack<T, VE> d;
#pragma unroll
            for (int k = 0; k < VE; ++k) d.v[k] = from_f32<T>(live ? rg.dense(to_f32(p.v[k])) : rg.base);
            store(j, d);
        }
    } else {
        RowGrad near = rg;  // against the rounded reference: 2^y is larger by 2^rest
        const float rest = fmaf(rg.m, rg.c, -rg.ref), f = exp2f(-rest);
        near.base = f * fmaf(-rest, rg.slope, rg.base);
        near.slope = f * rg.slope;
        for (int base = b0; base < b1; base += kGradThreads * kGradUnroll) {
            Pack<T, VE> p[kGradUnroll];
            const int j = base + threadIdx.x;
            if (base + kGradThreads * kGradUnroll <= b1) {
#pragma unroll
                for (int q = 0; q < kGradUnroll; ++q) p[q] = view.body[j + q * kGradThreads];
#pragma unroll
                for (int q = 0; q < kGradUnroll; ++q) {
                    Pack<T, VE> d;
                    dense_vector(near, p[q], d);
                    store(j + q * kGradThreads, d);
                }
            } else {
                for (int i = j; i < b1; i += kGradThreads) {
                    const Pack<T, VE> v = view.body[i];
                    Pack<T, VE> d;
                    dense_vector(near, v, d);
                    store(i, d);
                }
            }
        }
    }
    const int64_t head = view.skipped() ? min((int64_t)a.vocab, view.first(1)) : 0;
    const int64_t tail = head + (int64_t)view.n * VE;
    if (part == 0 && threadIdx.x < 2 * VE) {
        const int64_t e = (int)threadIdx.x < VE ? (int64_t)threadIdx.x : tail + threadIdx.x - VE;
        if ((int)threadIdx.x < VE ? e < head : e < a.vocab)
            out[e] = from_f32<T>(live ? rg.dense(to_f32(row[e])) : rg.base);
    }
    // the given token and the alternatives have terms of their own
    if (!live) return;
    __syncthreads();
    const int64_t e0 = head + (int64_t)b0 * VE, e1 = head + (int64_t)b1 * VE;
    for (int i = threadIdx.x; i <= a.top; i += kGradThreads) {
        if (i > 0 && !a.g_top) break;
        const int64_t v = i == 0 ? token : a.top_tokens[r * a.top + i - 1];
        if ((uint64_t)v >= (uint64_t)a.vocab) continue;
        if (v < head || v >= tail ? part != 0 : v < e0 || v >= e1) continue;
        float own = v == token ? gl : 0.0f;
        if (a.g_top)
            for (int k = 0; k < a.top; ++k)
                if (a.top_tokens[r * a.top + k] == v) own += a.g_top[r * a.top + k];
        out[v] = from_f32<T>(fmaf(own, a.inv_t, rg.dense(to_f32(row[v]))));
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

// Sums over the block, N at a time; `red` has N values for each warp.
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* red) {
#pragma unroll
    for (int d = 16; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    if (blockDim.x == 32) return;
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) red[(threadIdx.x >> 5) * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0;
        for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v[i] += red[w * N + i];
    }
}

// One block per row; 2048 rows with k = 100 take 26 us, the chain ids - values - logits and the f64
// functions.  Everything here is f64: there are at most k + top values per row, and
// the alternatives are ordered by sums of two sources, which f32 would tie or swap.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) neighbours_kernel(NearArgs a) {
    wait_for_previous();
    // candidates (log probability, token), neighbours (weight; token, -1 where one does not count)
    extern __shared__ double space[];
    double* cp = space;
    double* wgt = cp + a.k + a.top;
    int32_t* ct = reinterpret_cast<int32_t*>(wgt + a.k);
    int32_t* tok = ct + a.k + a.top;
    __shared__ double red[3 * kMaxThreads / 32];
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
    double sum[1] = {};
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        double w = 0.0;
        if (tok[j] >= 0) w = exp(((double)near - (double)a.distances[r * a.k + j]) * a.inv_tau);
        wgt[j] = w;
        sum[0] += w;
    }
    block_sums(sum, red);
    const double scale = a.weight / sum[0];
    const double keep = 1.0 - a.weight, log_keep = log(keep);
    // the first neighbour with a token carries the token
    __syncthreads();
    double part[3] = {};  // sums of q, q ln q, -p ln p over the neighbours' tokens
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        const int32_t t = tok[j];
        if (t < 0) continue;
        bool first = true;
        double w = 0.0;
#pragma unroll 8
        for (int i = 0; i < a.k; ++i) {
            const bool same = tok[i] == t;
            first = first & !(same & (i < j));
            if (same) w += wgt[i];
        }
        if (!first) continue;
        const double log_q = ((double)to_f32(row[t]) - m) * a.inv_t - log_s, q = exp(log_q);
        const double p = keep * q + w * scale;
        part[0] += q;
        if (q > 0.0) part[1] += q * log_q;
        // a probability below f64's range keeps its logarithm
        const double lp = p > 0.0 ? log(p) : log_keep + log_q;
        if (p > 0.0) part[2] -= p * lp;
        if (t == given) lp_token = lp;
        const int at = atomicAdd(&n_cand, 1);
        cp[at] = lp;
        ct[at] = t;
    }
    block_sums(part, red);
    __syncthreads();
    if (threadIdx.x == 0) {
        double h = part[2];
        const double rest = fmax(1.0 - part[0], 0.0);
        if (keep > 0.0) h -= keep * (log_keep * rest - (double)st.z - part[1]);
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
#pragma unroll 8
        for (int j = 0; j < n_near; ++j) mine = mine & (ct[j] != t);
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
        const int32_t t = ct[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += (cp[j] > lp) | ((cp[j] == lp) & (ct[j] < t));
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
    require(aligned(t->logits, dtype_bytes(t->dtype)), "token_logprobs: misaligned logits");
    require(t->ld >= 0, "token_logprobs: rows must not run backwards");
    require(aligned(t->tokens, 8) && (t->top == 0 || aligned(t->top_tokens, 8)), "token_logprobs: misaligned tokens");
    require(t->top == 0 || (t->top_tokens && t->top_logprobs), "token_logprobs: null output of the alternatives");
    require(aligned(t->stats, 16), "token_logprobs: stats must be 16-byte aligned");
}
// Of the calls that write them.
void check_outputs(const hanns_token_logprobs_t* t) {
    require(t->n == 0 || (aligned(t->logprobs, 4) && aligned(t->entropy, 4) && (t->top == 0 || aligned(t->top_logprobs, 4))),
            "token_logprobs: misaligned output");
}

// The launch rules count the SMs of a B200 (a launch is right on any number).
constexpr int sm_count() { return 148; }

template <class T, bool Top>
void launch_probs(const hanns_token_logprobs_t* t, const ProbArgs& a, cudaStream_t s) {
    // one more where a row starts inside a vector
    const int64_t vectors = (t->vocab + RowView<T>::VE - 1) / RowView<T>::VE + 1;
    // A warp for a row that fits in its registers, 4 or 8 vectors a lane: 8192 rows of 100 f32 with 5
    // alternatives take 10.5 us (a block each: 36.8), of 2,000 bf16 21.9 us (43.1).
    if (vectors <= 32 * 2 * kUnroll) {
        constexpr int warps = kMaxThreads / 32;
        const unsigned blocks = (unsigned)std::min<int64_t>((t->n + warps - 1) / warps, 8 * sm_count());
        auto* kernel = vectors <= 32 * kUnroll ? logprobs_rows_kernel<T, Top, kUnroll>
                                               : logprobs_rows_kernel<T, Top, 2 * kUnroll>;
        launch_early(kernel, blocks, kMaxThreads, 0, s, a, t->n);
        return;
    }
    // A cluster's blocks share a row when the rows alone are few for the SMs, as long as each block
    // still has a round of full loads: one row of 128,000 bf16 takes 8 us on eight blocks (one:
    // 18.6), 222 rows 17.4 on four (two: 21.5), 300 rows 23.5 on two (one: 33.5).  Up to six blocks an
    // SM: clusters do not fill the eight places of every SM, and those left over wait (296 rows on
    // four blocks 26.2, on two 23.1).  The alternatives of all blocks have a thread each to join
    // them (100 rows of 50,257 with 20: 13.4 us on four blocks, 17.2 on eight).
    int parts = 1;
    const int64_t want = 6 * sm_count();
    while (parts < kMaxCluster && t->n * parts * 2 <= want && vectors / (parts * 2) >= kMaxThreads * kUnroll &&
           parts * 2 * t->top <= kMaxThreads)
        parts *= 2;
    const int threads = kMaxThreads;
    cudaLaunchConfig_t cfg{};
    // blocks that take several rows: as many as are resident
    cfg.gridDim = dim3((unsigned)(Top || parts > 1 ? t->n * parts : std::min<int64_t>(t->n, 8 * sm_count())));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 2;
    HANNS_CUDA_OK(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, Top>, a, t->n));
}

template <class T>
void launch_grad(const hanns_token_logprobs_t* t, GradArgs a, cudaStream_t s) {
    const int64_t vectors = (t->vocab + RowView<T>::VE - 1) / RowView<T>::VE;
    // several rounds to a block, for what a block works out once, unless that leaves SMs idle (600
    // rows of 32,000 f32: 21.7 us, one round each 28.1)
    const int64_t round = kGradThreads * kGradUnroll;
    int64_t rounds = kGradRounds;
    while (rounds > 1 && t->n * ((vectors + rounds * round - 1) / (rounds * round)) < 16 * sm_count())
        rounds /= 2;
    a.span = (int)(rounds * round);
    a.blocks_per_row = (int)((vectors + a.span - 1) / a.span);
    require(t->n * a.blocks_per_row < 0x7fffffff, "token_logprobs: too many elements for one gradient call");
    // wide stores where each output row starts as its logits do within 16 bytes
    const bool wide = ((uintptr_t)a.logits - (uintptr_t)a.out) % 16 == 0 &&
                      ((a.ld - a.out_ld) * (int64_t)sizeof(T)) % 16 == 0;
    const unsigned grid = (unsigned)(t->n * a.blocks_per_row);
    if (wide) launch_early(logprobs_grad_kernel<T, true>, grid, kGradThreads, 0, s, a);
    else launch_early(logprobs_grad_kernel<T, false>, grid, kGradThreads, 0, s, a);
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
        check_outputs(t);
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
        require(aligned(d_logits, dtype_bytes(t->dtype)), "token_logprobs: misaligned gradient");
        require(aligned(g_logprobs, 4) && aligned(g_entropy, 4) && aligned(g_top, 4),
                "token_logprobs: misaligned gradients of the outputs");
        require(t->n <= 1 || d_ld >= t->vocab, "token_logprobs: the gradient's rows overlap");
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
        check_outputs(t);
        require(k >= 0 && k <= kMaxNeighbours, "neighbour_logprobs: k must be in [0, 1024]");
        require(weight >= 0.0f && weight <= 1.0f, "neighbour_logprobs: weight must be in [0, 1]");
        require(knn_temperature > 1e-30f && knn_temperature < 1e30f,
                "neighbour_logprobs: temperature must be positive and finite");
        if (t->n == 0 || k == 0 || n_values <= 0 || weight == 0.0f) return;
        require(t->stats, "neighbour_logprobs: the model's statistics (stats) are needed");
        require(d_ids && d_distances && d_values, "neighbour_logprobs: null ids, distances or values");
        require(aligned(d_ids, 8) && aligned(d_distances, 4) && aligned(d_values, 8),
                "neighbour_logprobs: misaligned ids, distances or values");
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
        const unsigned threads = k <= 32 ? 32 : k <= 64 ? 64 : kMaxThreads, n = (unsigned)t->n;
        const size_t shared = (2 * (size_t)k + a.top) * sizeof(double) + (2 * (size_t)k + a.top) * sizeof(int32_t);
        if (t->dtype == HANNS_DTYPE_F32) launch_early(neighbours_kernel<float>, n, threads, shared, s, a);
        else if (t->dtype == HANNS_DTYPE_F16) launch_early(neighbours_kernel<__half>, n, threads, shared, s, a);
        else launch_early(neighbours_kernel<__nv_bfloat16>, n, threads, shared, s, a);
    });
}
