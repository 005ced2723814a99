// embed_bags.cu -- token ids to the vectors the index searches, and the gradient.
//
//   out_i  = (scale / c_i) * sum over the tokens t_j of bag i of  w_j E[t_j]
//   dE[v]  = sum over the positions j with t_j = v of  (scale w_j / c_bag(j)) g_bag(j)
//   dw_j   = (scale / c_bag(j)) <E[t_j], g_bag(j)>
//
// c_i is the number of counted tokens of bag i for a mean and 1 for a sum; a token outside
// [0, rows) is not counted.  Both sums are one operation: entries (row of a matrix, factor)
// in a fixed order, cut into segments, one output row per segment.  Forward, the segments
// are the bags and the matrix is the table.  Backward, the positions are sorted by token
// (stable, so that a token's terms are added in the order of their positions and the result
// does not change from run to run), the segments are the tokens and the matrix is the
// incoming gradient.  Sums are f32, rounded once to the output's type.
//
// A segment of at most `limit` entries is summed by one warp per column tile
// (segments_kernel).  Longer ones are cut at the multiples of `limit` positions
// (pieces_kernel writes f32 partial rows) and joined in order (join_kernel), so that one
// document, or the most frequent token of a batch, does not run on a single warp.
#include <algorithm>

#include "operators.cuh"

namespace hanns {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnroll = 4;
constexpr int kMaxBinBits = 9, kMaxBins = 1 << kMaxBinBits;
constexpr int kSortItems = 4, kSortTile = kThreads * kSortItems;

// ---------------------------------------------------------------- entries and segments
// Position j of the tokens as the caller gave them.
struct TokenEntries {
    const int64_t* tokens;
    const float* weights;
    int64_t rows;
    __device__ __forceinline__ void get(int64_t j, int& row, float& coef) const {
        const int64_t t = tokens[j];
        row = (uint64_t)t < (uint64_t)rows ? (int)t : -1;
        coef = weights ? weights[j] : 1.0f;
    }
};
// Entry j of the positions sorted by token.
struct SortedEntries {
    const int32_t* src;
    const float* coef;
    __device__ __forceinline__ void get(int64_t j, int& row, float& c) const {
        row = src[j];
        c = coef[j];
    }
};

__device__ __forceinline__ int64_t clamp_pos(int64_t p, int64_t lo, int64_t hi) {
    return p < lo ? lo : p > hi ? hi : p;
}

// Bags: [offsets[i], offsets[i+1]), kept inside [0, n_tokens] whatever the offsets hold.
struct BagSegments {
    const int64_t* offsets;  // null: bag i is position i
    int64_t n_bags, n_tokens;
    __device__ __forceinline__ void bounds(int64_t i, int64_t& lo, int64_t& hi) const {
        if (!offsets) {
            lo = i;
            hi = i + 1;
            return;
        }
        lo = clamp_pos(offsets[i], 0, n_tokens);
        hi = clamp_pos(offsets[i + 1], lo, n_tokens);
    }
    // The bag that holds position p, or -1.
    __device__ __forceinline__ int64_t at(int64_t p) const {
        if (!offsets) return p;
        int64_t a = 0, b = n_bags + 1;  // first index whose offset is > p
        while (a < b) {
            const int64_t m = (a + b) >> 1;
            if (offsets[m] <= p) a = m + 1;
            else b = m;
        }
        return a >= 1 && a <= n_bags ? a - 1 : -1;
    }
};
// Tokens: runs of equal keys in the sorted order.
struct TokenSegments {
    const int32_t *start, *stop;
    const uint32_t* key;
    int64_t rows;
    __device__ __forceinline__ void bounds(int64_t v, int64_t& lo, int64_t& hi) const {
        lo = start[v];
        hi = stop[v];
    }
    __device__ __forceinline__ int64_t at(int64_t p) const {
        const uint32_t k = key[p];
        return k < rows ? (int64_t)k : -1;
    }
};

struct SumArgs {
    const void* base;  // matrix of the summed rows
    int64_t ld;
    void* out;
    int64_t out_ld;
    int64_t n_segments, n_entries;
    int dim, lanes_log2, tiles;  // lanes that share a row's tile, column tiles
    int limit;                   // longest segment of one warp; pieces are this long
    float scale;
    int mean;
    float* inv_counts;
    float* partial;              // [chunks][2][tiles * lanes * VE]
    int32_t* partial_count;      // [chunks][2]
};

template <class T, int VE>
__device__ __forceinline__ void add_pack(float (&acc)[VE], const Pack<T, VE>& p, float c) {
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = fmaf(c, to_f32(p.v[e]), acc[e]);
}

// Stores VE results in accesses of at most 16 bytes.
template <class TO, int VE>
__device__ __forceinline__ void store_row(TO* p, const float (&acc)[VE], float factor) {
    constexpr int N = VE * sizeof(TO) > 16 ? 16 / sizeof(TO) : VE;
#pragma unroll
    for (int o = 0; o < VE; o += N) {
        Pack<TO, N> q;
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = from_f32<TO>(acc[o + e] * factor);
        *reinterpret_cast<Pack<TO, N>*>(p + o) = q;
    }
}

// The sum of entries [lo, hi) over this warp's column tile.  A row's tile is read by
// 2^lanes_log2 lanes; the warp's 32 >> lanes_log2 lane groups take entries in turn and are
// added at the end (every lane then holds the sum of its columns).  Returns the number of
// counted entries.
template <class T, int VE, class Entries>
__device__ __forceinline__ int sum_entries(const Entries& entries, const SumArgs& a, int col, int64_t lo,
                                           int64_t hi, float (&acc)[VE]) {
    const int lane = threadIdx.x & 31, groups = 32 >> a.lanes_log2, group = lane >> a.lanes_log2;
    const bool col_ok = col < a.dim;
    const T* base = static_cast<const T*>(a.base) + col;
    int count = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    for (int64_t b = lo; b < hi; b += 32) {
        const int n = (int)min((int64_t)32, hi - b);
        int row = -1;
        float coef = 0.0f;
        if (lane < n) entries.get(b + lane, row, coef);
        count += __popc(__ballot_sync(0xffffffffu, row >= 0));
        for (int q = 0; q < n; q += kUnroll * groups) {
            Pack<T, VE> p[kUnroll];
            int r[kUnroll];
            float c[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = q + u * groups + group;
                r[u] = __shfl_sync(0xffffffffu, row, i & 31);
                c[u] = __shfl_sync(0xffffffffu, coef, i & 31);
                if (i >= n || !col_ok) r[u] = -1;
                if (r[u] >= 0) p[u] = load_pack<T, VE>(base + (int64_t)r[u] * a.ld);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (r[u] >= 0) add_pack<T, VE>(acc, p[u], c[u]);
        }
    }
    for (int m = 16; m >= 1 << a.lanes_log2; m >>= 1)
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], m);
    return count;
}

// What a finished sum is multiplied by.
__device__ __forceinline__ float finish_factor(const SumArgs& a, int64_t seg, int64_t count, bool write) {
    float inv = 1.0f;
    if (a.mean) {
        inv = __fdiv_rn(1.0f, (float)(count > 0 ? count : 1));
        if (a.inv_counts && write) a.inv_counts[seg] = inv;
    }
    return a.scale * inv;
}

// One warp per (segment, column tile); segments longer than the limit are left to the
// pieces.  Every other segment's row is written here, zeros for an empty one.
template <class T, class TO, int VE, class Entries, class Segments>
__global__ void __launch_bounds__(kThreads) segments_kernel(SumArgs a, Entries entries, Segments segs) {
    const uint32_t w = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const uint32_t seg = w / (uint32_t)a.tiles, tile = w - seg * (uint32_t)a.tiles;
    if (seg >= a.n_segments) return;
    int64_t lo, hi;
    segs.bounds(seg, lo, hi);
    if (hi - lo > a.limit) return;
    const int lane = threadIdx.x & 31, lanes = 1 << a.lanes_log2;
    const int col = ((tile << a.lanes_log2) + (lane & (lanes - 1))) * VE;
    float acc[VE];
    const int count = sum_entries<T, VE>(entries, a, col, lo, hi, acc);
    const float f = finish_factor(a, seg, count, tile == 0 && lane == 0);
    if (lane < lanes && col < a.dim)
        store_row<TO, VE>(static_cast<TO*>(a.out) + (int64_t)seg * a.out_ld + col, acc, f);
}

// One warp per (chunk of `limit` positions, column tile).  A segment longer than a chunk that
// reaches into one holds its first position (slot 0) or its last (slot 1).
template <class T, int VE, class Entries, class Segments>
__global__ void __launch_bounds__(kThreads) pieces_kernel(SumArgs a, Entries entries, Segments segs) {
    const uint32_t w = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const uint32_t chunk = w / (uint32_t)a.tiles, tile = w - chunk * (uint32_t)a.tiles;
    const int64_t first = (int64_t)chunk * a.limit;
    if (first >= a.n_entries) return;
    const int64_t end = min(first + a.limit, a.n_entries);
    const int lane = threadIdx.x & 31, lanes = 1 << a.lanes_log2;
    const int col = ((tile << a.lanes_log2) + (lane & (lanes - 1))) * VE;
    const int width = (a.tiles << a.lanes_log2) * VE;
    const int64_t head = segs.at(first), tail = segs.at(end - 1);
    for (int slot = 0; slot < 2; ++slot) {
        const int64_t seg = slot ? tail : head;
        if (seg < 0 || (slot && tail == head)) continue;
        int64_t lo, hi;
        segs.bounds(seg, lo, hi);
        if (hi - lo <= a.limit) continue;
        float acc[VE];
        const int count = sum_entries<T, VE>(entries, a, col, max(lo, first), min(hi, end), acc);
        if (lane < lanes) store_row<float, VE>(a.partial + ((int64_t)chunk * 2 + slot) * width + col, acc, 1.0f);
        if (tile == 0 && lane == 0) a.partial_count[(int64_t)chunk * 2 + slot] = count;
    }
}

// One block per (chunk, column tile): the long segment that starts in this chunk, if one
// does, is the sum of its pieces.  The warps take pieces in turn and are added in order.
template <class TO, int VE, class Segments>
__global__ void __launch_bounds__(kThreads) join_kernel(SumArgs a, Segments segs) {
    const uint32_t chunk = blockIdx.x / (uint32_t)a.tiles, tile = blockIdx.x - chunk * (uint32_t)a.tiles;
    const int64_t first = (int64_t)chunk * a.limit, end = min(first + a.limit, a.n_entries);
    const int64_t seg = segs.at(end - 1);
    if (seg < 0) return;
    int64_t lo, hi;
    segs.bounds(seg, lo, hi);
    if (hi - lo <= a.limit || lo < first || lo >= end) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = 1 << a.lanes_log2;
    const int groups = 32 >> a.lanes_log2, group = lane >> a.lanes_log2;
    const int col = ((tile << a.lanes_log2) + (lane & (lanes - 1))) * VE;
    const int width = (a.tiles << a.lanes_log2) * VE;
    const int64_t last = (hi - 1) / a.limit, pieces = last - chunk + 1;
    float acc[VE];
    int64_t count = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    for (int64_t p = warp * groups + group; p < pieces; p += kWarps * groups) {
        const int64_t at = (chunk + p) * 2 + (p == 0 && lo > first ? 1 : 0);
        count += a.partial_count[at];
        const float* src = a.partial + at * width + col;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] += src[e];
    }
    for (int m = 16; m >= lanes; m >>= 1) {
        count += __shfl_xor_sync(0xffffffffu, count, m);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], m);
    }
    __shared__ float s_acc[kWarps][32 * VE];
    __shared__ int64_t s_count[kWarps];
#pragma unroll
    for (int e = 0; e < VE; ++e) s_acc[warp][lane * VE + e] = acc[e];
    if (lane == 0) s_count[warp] = count;
    __syncthreads();
    if (warp) return;
    count = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
        count += s_count[w];
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] += s_acc[w][lane * VE + e];
    }
    const float f = finish_factor(a, seg, count, tile == 0 && lane == 0);
    if (lane < lanes && col < a.dim)
        store_row<TO, VE>(static_cast<TO*>(a.out) + seg * a.out_ld + col, acc, f);
}

// ---------------------------------------------------------------- sort by token
// Least significant digit first, each pass stable: digit counts per tile of positions,
// running sums per digit over the tiles, and the move.  The last pass writes the entries the
// sums read (bag and factor of the position) instead of the position.
struct SortArgs {
    BagSegments bags;
    const int64_t* tokens;
    const float* weights;
    const float* inv_counts;  // null: sums, not means
    int64_t rows;             // also the key of a position that counts nowhere
    int32_t n;
    int32_t tiles;
    float scale;
    int shift, bins;
    const uint32_t *key_in, *pos_in;
    uint32_t *key_out, *pos_out;
    int32_t* src;
    float* coef;
    int32_t* hist;   // [bins][tiles]
    int32_t* total;  // [bins]
};

template <bool First>
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t j) {
    if (!First) return a.key_in[j];
    const int64_t t = a.tokens[j];
    if ((uint64_t)t >= (uint64_t)a.rows) return (uint32_t)a.rows;
    if (a.bags.offsets && (j < a.bags.offsets[0] || j >= a.bags.offsets[a.bags.n_bags]))
        return (uint32_t)a.rows;
    return (uint32_t)t;
}

template <bool First>
__global__ void __launch_bounds__(kThreads) sort_count_kernel(SortArgs a) {
    __shared__ int32_t count[kMaxBins];
    for (int b = threadIdx.x; b < a.bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t j = base + i * kThreads + threadIdx.x;
        if (j < a.n) atomicAdd(&count[(sort_key<First>(a, j) >> a.shift) & (a.bins - 1)], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.bins; b += kThreads) a.hist[(int64_t)b * a.tiles + blockIdx.x] = count[b];
}

// One warp per digit: its counts become the number of its keys in earlier tiles.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(SortArgs a) {
    const int bin = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (bin >= a.bins) return;
    int32_t* h = a.hist + (int64_t)bin * a.tiles;
    int32_t run = 0;
    for (int t0 = 0; t0 < a.tiles; t0 += 32) {
        const int t = t0 + lane;
        const int32_t v = t < a.tiles ? h[t] : 0;
        int32_t s = v;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int32_t o = __shfl_up_sync(0xffffffffu, s, m);
            if (lane >= m) s += o;
        }
        if (t < a.tiles) h[t] = run + s - v;
        run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) a.total[bin] = run;
}

template <bool First, bool Last>
__global__ void __launch_bounds__(kThreads) sort_move_kernel(SortArgs a) {
    __shared__ int32_t seen[kWarps][kMaxBins];  // a warp's keys per digit, then its first place
    __shared__ int32_t warp_sum[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&seen[0][0])[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile + warp * (32 * kSortItems);
    uint32_t key[kSortItems];
    int32_t rank[kSortItems];
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t j = base + i * 32 + lane;
        const bool in = j < a.n;
        key[i] = in ? sort_key<First>(a, j) : 0;
        const int d = (key[i] >> a.shift) & (a.bins - 1);
        const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : -1);
        rank[i] = 0;
        if (in) rank[i] = seen[warp][d] + __popc(peers & ((1u << lane) - 1));
        __syncwarp();
        if (in && (peers >> lane) == 1) seen[warp][d] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    // digits before this one, in all tiles: two digits per thread (bins <= 2 * kThreads)
    int32_t t0 = 0, t1 = 0;
    const int b0 = threadIdx.x * 2;
    if (b0 < a.bins) t0 = a.total[b0];
    if (b0 + 1 < a.bins) t1 = a.total[b0 + 1];
    int32_t s = t0 + t1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int32_t o = __shfl_up_sync(0xffffffffu, s, m);
        if (lane >= m) s += o;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int32_t before = s - t0 - t1;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int b = b0 + q;
        if (b < a.bins) {
            int32_t at = before + (q ? t0 : 0) + a.hist[(int64_t)b * a.tiles + blockIdx.x];
            for (int w = 0; w < kWarps; ++w) {
                const int32_t c = seen[w][b];
                seen[w][b] = at;
                at += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t j = base + i * 32 + lane;
        if (j >= a.n) continue;
        const int32_t to = seen[warp][(key[i] >> a.shift) & (a.bins - 1)] + rank[i];
        a.key_out[to] = key[i];
        const uint32_t pos = First ? (uint32_t)j : a.pos_in[j];
        if (!Last) {
            a.pos_out[to] = pos;
            continue;
        }
        const int64_t bag = key[i] < a.rows ? a.bags.at(pos) : -1;
        float c = a.scale;
        if (a.weights) c *= a.weights[pos];
        if (a.inv_counts && bag >= 0) c *= a.inv_counts[bag];
        a.src[to] = (int32_t)bag;
        a.coef[to] = c;
    }
}

// Where each token's run begins and ends (both arrays start as zeros: tokens without a run).
__global__ void __launch_bounds__(kThreads) sort_runs_kernel(const uint32_t* key, int32_t n, int64_t rows,
                                                             int32_t* start, int32_t* stop) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const uint32_t k = key[i];
    if (k >= rows) return;
    if (i == 0 || key[i - 1] != k) start[k] = (int32_t)i;
    if (i == n - 1 || key[i + 1] != k) stop[k] = (int32_t)(i + 1);
}

// ---------------------------------------------------------------- gradient of the weights
// One warp per position: the inner product of its table row with its bag's gradient.
template <class T, class TG>
__global__ void __launch_bounds__(kThreads)
    weights_grad_kernel(BagSegments bags, const int64_t* tokens, int64_t rows, const T* table, int64_t ld, int dim,
                        const TG* grad, int64_t grad_ld, const float* inv_counts, float scale, float* d_weights) {
    const int64_t j = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (j >= bags.n_tokens) return;
    const int lane = threadIdx.x & 31;
    const int64_t t = tokens[j];
    const int64_t bag = (uint64_t)t < (uint64_t)rows ? bags.at(j) : -1;
    float dot = 0.0f;
    if (bag >= 0) {
        const T* e = table + t * ld;
        const TG* g = grad + bag * grad_ld;
        for (int c = lane; c < dim; c += 32) dot = fmaf(to_f32(e[c]), to_f32(g[c]), dot);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
    if (lane == 0) {
        float f = scale;
        if (inv_counts && bag >= 0) f *= inv_counts[bag];
        d_weights[j] = bag >= 0 ? dot * f : 0.0f;
    }
}

// ---------------------------------------------------------------- host
struct Plan {
    int lanes_log2, tiles, limit;
    int64_t chunks;
    int64_t width;  // floats of a partial row
};

// Widest access that every row of both matrices allows.
int vector_elems(const void* in, int64_t in_ld, int in_size, const void* out, int64_t out_ld, int out_size, int dim) {
    for (int ve = 16 / in_size; ve > 1; ve /= 2) {
        if (in_size == 2 && ve == 2) break;  // 16-bit rows: 8, 4 or 1 elements
        const int ib = ve * in_size, ob = std::min(16, ve * out_size);
        if (dim % ve == 0 && (uintptr_t)in % ib == 0 && (in_ld * in_size) % ib == 0 && (uintptr_t)out % ob == 0 &&
            (out_ld * out_size) % ob == 0)
            return ve;
    }
    return 1;
}

Plan make_plan(int dim, int ve, int64_t n_entries) {
    Plan p;
    const int packs = (dim + ve - 1) / ve;
    p.lanes_log2 = 0;
    while (p.lanes_log2 < 5 && (1 << p.lanes_log2) < packs) ++p.lanes_log2;
    p.tiles = (packs + (1 << p.lanes_log2) - 1) >> p.lanes_log2;
    // at least 64 entries per piece, and at most about 4,096 pieces
    p.limit = (int)std::max<int64_t>(64, (n_entries + 4095) / 4096);
    p.chunks = (n_entries + p.limit - 1) / p.limit;
    p.width = ((int64_t)p.tiles << p.lanes_log2) * ve;
    return p;
}

// Bytes of the partial rows for any vector width (a row is padded to whole tiles).
size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
size_t partial_bytes(int64_t n_entries, int dim) {
    const int64_t limit = std::max<int64_t>(64, (n_entries + 4095) / 4096);
    if (n_entries <= limit) return 0;
    const int64_t chunks = (n_entries + limit - 1) / limit;
    const size_t width = (size_t)dim + 32 * 8;
    return round256(chunks * 2 * width * sizeof(float)) + round256(chunks * 2 * sizeof(int32_t));
}

struct Carver {
    char* p;
    size_t used = 0;
    template <class T>
    T* take(size_t n) {
        T* r = reinterpret_cast<T*>(p + used);
        used += round256(n * sizeof(T));
        return r;
    }
};

template <class T, class TO, int VE, class Entries, class Segments>
void launch_sum(SumArgs a, const Entries& entries, const Segments& segs, const Plan& p, cudaStream_t s) {
    const int64_t warps = a.n_segments * p.tiles;
    require(warps < (int64_t)1 << 32, "embed_bags: too many output tiles");
    if (warps > 0) {
        segments_kernel<T, TO, VE><<<(unsigned)((warps + kWarps - 1) / kWarps), kThreads, 0, s>>>(a, entries, segs);
        HANNS_CUDA_OK(cudaGetLastError());
    }
    if (a.n_entries <= p.limit || warps == 0) return;
    const int64_t pw = p.chunks * p.tiles;
    pieces_kernel<T, VE><<<(unsigned)((pw + kWarps - 1) / kWarps), kThreads, 0, s>>>(a, entries, segs);
    HANNS_CUDA_OK(cudaGetLastError());
    join_kernel<TO, VE><<<(unsigned)pw, kThreads, 0, s>>>(a, segs);
    HANNS_CUDA_OK(cudaGetLastError());
}

template <class T, class TO, class Entries, class Segments>
void sum_segments(SumArgs a, const Entries& entries, const Segments& segs, Carver& ws, cudaStream_t s) {
    const int ve = vector_elems(a.base, a.ld, sizeof(T), a.out, a.out_ld, sizeof(TO), a.dim);
    const Plan p = make_plan(a.dim, ve, a.n_entries);
    a.lanes_log2 = p.lanes_log2;
    a.tiles = p.tiles;
    a.limit = p.limit;
    if (a.n_entries > p.limit) {
        a.partial = ws.take<float>(p.chunks * 2 * p.width);
        a.partial_count = ws.take<int32_t>(p.chunks * 2);
    }
    constexpr int wide = 16 / sizeof(T);
    if (ve == wide) launch_sum<T, TO, wide>(a, entries, segs, p, s);
    else if (ve == wide / 2) launch_sum<T, TO, wide / 2>(a, entries, segs, p, s);
    else launch_sum<T, TO, 1>(a, entries, segs, p, s);
}

template <class Entries, class Segments>
void sum_typed(int32_t in, int32_t out, const SumArgs& a, const Entries& e, const Segments& g, Carver& ws,
               cudaStream_t s) {
    if (in == HANNS_DTYPE_F32) {
        if (out == HANNS_DTYPE_F32) return sum_segments<float, float>(a, e, g, ws, s);
        if (out == HANNS_DTYPE_F16) return sum_segments<float, __half>(a, e, g, ws, s);
        return sum_segments<float, __nv_bfloat16>(a, e, g, ws, s);
    }
    if (in == HANNS_DTYPE_F16) {
        if (out == HANNS_DTYPE_F32) return sum_segments<__half, float>(a, e, g, ws, s);
        return sum_segments<__half, __half>(a, e, g, ws, s);
    }
    if (out == HANNS_DTYPE_F32) return sum_segments<__nv_bfloat16, float>(a, e, g, ws, s);
    return sum_segments<__nv_bfloat16, __nv_bfloat16>(a, e, g, ws, s);
}

void check_bags(const hanns_embed_bags_t* b) {
    require(b, "embed_bags: null arguments");
    require(dtype_known(b->dtype) && dtype_known(b->out_dtype), "embed_bags: unknown element type");
    require(b->out_dtype == b->dtype || b->out_dtype == HANNS_DTYPE_F32,
            "embed_bags: the output is f32 or of the table's type");
    require(b->dim >= 1 && b->dim <= 1 << 24, "embed_bags: dim must be in [1, 2^24]");
    require(b->rows >= 1 && b->rows < 0x7fffffff, "embed_bags: rows must be in [1, 2^31 - 1)");
    require(b->n_tokens >= 0 && b->n_tokens < 0x7fffffff, "embed_bags: n_tokens must be in [0, 2^31 - 1)");
    require(b->n_bags >= 0 && b->n_bags < 0x7fffffff, "embed_bags: n_bags must be in [0, 2^31 - 1)");
    require(b->offsets || b->n_bags == b->n_tokens, "embed_bags: without offsets each token is its own bag");
}

void check_workspace(size_t need, const void* p, int64_t have) {
    require(need == 0 || (p && (uintptr_t)p % 256 == 0), "embed_bags: the workspace must be 256-byte aligned");
    require(have >= 0 && (size_t)have >= need, "embed_bags: the workspace is too small");
}

struct SortPlan {
    int passes, bits;  // digits, bits of each
    int32_t tiles;
};
SortPlan sort_plan(int64_t rows, int64_t n) {
    int bits = 1;
    while (((int64_t)1 << bits) <= rows) ++bits;  // keys 0 .. rows
    SortPlan p;
    p.passes = (bits + kMaxBinBits - 1) / kMaxBinBits;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.tiles = (int32_t)((n + kSortTile - 1) / kSortTile);
    return p;
}

size_t grad_bytes(const hanns_embed_bags_t* b) {
    if (b->n_tokens == 0) return round256(b->rows * sizeof(int32_t)) * 2;
    const SortPlan sp = sort_plan(b->rows, b->n_tokens);
    size_t t = 6 * round256(b->n_tokens * 4);
    t += round256(((size_t)sp.tiles << sp.bits) * 4) + round256(((size_t)1 << sp.bits) * 4);
    t += 2 * round256(b->rows * sizeof(int32_t));
    return t + partial_bytes(b->n_tokens, b->dim);
}

template <bool First>
void sort_pass(const SortArgs& a, bool last, cudaStream_t s) {
    sort_count_kernel<First><<<a.tiles, kThreads, 0, s>>>(a);
    sort_scan_kernel<<<(a.bins + kWarps - 1) / kWarps, kThreads, 0, s>>>(a);
    if (last) sort_move_kernel<First, true><<<a.tiles, kThreads, 0, s>>>(a);
    else sort_move_kernel<First, false><<<a.tiles, kThreads, 0, s>>>(a);
    HANNS_CUDA_OK(cudaGetLastError());
}

template <class T, class TG>
void launch_weights_grad(const hanns_embed_bags_t* b, const BagSegments& bags, const void* grad, int64_t grad_ld,
                         float* d_weights, cudaStream_t s) {
    weights_grad_kernel<T, TG><<<(unsigned)((b->n_tokens + kWarps - 1) / kWarps), kThreads, 0, s>>>(
        bags, b->tokens, b->rows, static_cast<const T*>(b->table), b->ld, b->dim, static_cast<const TG*>(grad), grad_ld,
        b->mean ? b->inv_counts : nullptr, b->scale, d_weights);
    HANNS_CUDA_OK(cudaGetLastError());
}

}  // namespace
}  // namespace hanns

// Declared in include/hanns_gpu.h.
extern "C" int64_t hanns_gpu_embed_bags_workspace_bytes(const hanns_embed_bags_t* b) {
    int64_t n = -1;
    hanns::operator_entry([&] {
        hanns::check_bags(b);
        n = (int64_t)hanns::partial_bytes(b->n_tokens, b->dim);
    });
    return n;
}

extern "C" int32_t hanns_gpu_embed_bags_device(const hanns_embed_bags_t* b, void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        if (b->n_bags == 0) return;
        require(b->table && b->out && (b->tokens || b->n_tokens == 0), "embed_bags: null table, tokens or out");
        check_workspace(partial_bytes(b->n_tokens, b->dim), b->workspace, b->workspace_bytes);
        Carver ws{static_cast<char*>(b->workspace)};
        SumArgs a{};
        a.base = b->table;
        a.ld = b->ld;
        a.out = b->out;
        a.out_ld = b->out_ld;
        a.n_segments = b->n_bags;
        a.n_entries = b->n_tokens;
        a.dim = b->dim;
        a.scale = b->scale;
        a.mean = b->mean != 0;
        a.inv_counts = b->inv_counts;
        sum_typed(b->dtype, b->out_dtype, a, TokenEntries{b->tokens, b->weights, b->rows},
                  BagSegments{b->offsets, b->n_bags, b->n_tokens}, ws, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int64_t hanns_gpu_embed_bags_grad_workspace_bytes(const hanns_embed_bags_t* b) {
    int64_t n = -1;
    hanns::operator_entry([&] {
        hanns::check_bags(b);
        n = (int64_t)hanns::grad_bytes(b);
    });
    return n;
}

extern "C" int32_t hanns_gpu_embed_bags_grad_device(const hanns_embed_bags_t* b, const void* grad, int64_t grad_ld,
                                                    void* d_table, int64_t d_table_ld, float* d_weights,
                                                    void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        require(grad || b->n_bags == 0, "embed_bags: null gradient");
        require(b->tokens || b->n_tokens == 0, "embed_bags: null tokens");
        require(!b->mean || b->inv_counts || b->n_bags == 0, "embed_bags: a mean's gradient needs inv_counts");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const BagSegments bags{b->offsets, b->n_bags, b->n_tokens};
        if (d_weights && b->n_tokens > 0) {
            require(b->table, "embed_bags: the weights' gradient needs the table");
            const bool g32 = b->out_dtype == HANNS_DTYPE_F32;
            if (b->dtype == HANNS_DTYPE_F32) launch_weights_grad<float, float>(b, bags, grad, grad_ld, d_weights, s);
            else if (b->dtype == HANNS_DTYPE_F16) {
                if (g32) launch_weights_grad<__half, float>(b, bags, grad, grad_ld, d_weights, s);
                else launch_weights_grad<__half, __half>(b, bags, grad, grad_ld, d_weights, s);
            } else {
                if (g32) launch_weights_grad<__nv_bfloat16, float>(b, bags, grad, grad_ld, d_weights, s);
                else launch_weights_grad<__nv_bfloat16, __nv_bfloat16>(b, bags, grad, grad_ld, d_weights, s);
            }
        }
        if (!d_table) return;
        check_workspace(grad_bytes(b), b->workspace, b->workspace_bytes);
        Carver ws{static_cast<char*>(b->workspace)};
        int32_t* start = ws.take<int32_t>(b->rows);
        int32_t* stop = ws.take<int32_t>(b->rows);
        HANNS_CUDA_OK(cudaMemsetAsync(start, 0, (char*)stop - (char*)start + b->rows * sizeof(int32_t), s));
        const size_t n = (size_t)b->n_tokens;
        uint32_t* key[2] = {nullptr, nullptr};
        uint32_t* pos[2] = {nullptr, nullptr};
        int32_t* src = nullptr;
        float* coef = nullptr;
        uint32_t* sorted = nullptr;
        if (n > 0) {
            const SortPlan sp = sort_plan(b->rows, b->n_tokens);
            for (auto* k : {&key[0], &key[1], &pos[0], &pos[1]}) *k = ws.take<uint32_t>(n);
            src = ws.take<int32_t>(n);
            coef = ws.take<float>(n);
            SortArgs a{};
            a.bags = bags;
            a.tokens = b->tokens;
            a.weights = b->weights;
            a.inv_counts = b->mean ? b->inv_counts : nullptr;
            a.rows = b->rows;
            a.n = (int32_t)n;
            a.tiles = sp.tiles;
            a.scale = b->scale;
            a.bins = 1 << sp.bits;
            a.src = src;
            a.coef = coef;
            a.hist = ws.take<int32_t>((size_t)sp.tiles << sp.bits);
            a.total = ws.take<int32_t>((size_t)1 << sp.bits);
            for (int p = 0; p < sp.passes; ++p) {
                a.shift = p * sp.bits;
                a.key_in = key[(p + 1) & 1];
                a.pos_in = pos[(p + 1) & 1];
                a.key_out = key[p & 1];
                a.pos_out = pos[p & 1];
                if (p == 0) sort_pass<true>(a, sp.passes == 1, s);
                else sort_pass<false>(a, p == sp.passes - 1, s);
            }
            sorted = key[(sp.passes - 1) & 1];
            sort_runs_kernel<<<(unsigned)((n + kThreads - 1) / kThreads), kThreads, 0, s>>>(sorted, (int32_t)n, b->rows,
                                                                                           start, stop);
            HANNS_CUDA_OK(cudaGetLastError());
        }
        SumArgs a{};
        a.base = grad;
        a.ld = grad_ld;
        a.out = d_table;
        a.out_ld = d_table_ld;
        a.n_segments = b->rows;
        a.n_entries = b->n_tokens;
        a.dim = b->dim;
        a.scale = 1.0f;
        sum_typed(b->out_dtype, b->dtype, a, SortedEntries{src, coef}, TokenSegments{start, stop, sorted, b->rows}, ws,
                  s);
    });
}
