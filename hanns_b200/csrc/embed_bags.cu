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
// A warp sums a segment's rows over a column tile (segments_kernel): its lanes look 32 entries up,
// put the counted ones side by side in shared memory, and then read several rows at a time, up to
// four vectors of a row to a lane, without a branch between them.  What an entry, a segment and a
// warp cost besides is as much as a few vectors' sums, which is why the tiles are wide.  A segment
// longer than kLimit goes to a list of pieces, each a warp's (pieces_kernel); the last one of a
// segment to finish adds its pieces up in order, so that one document, or the most frequent token
// of a batch, does not run on a single warp.
//
// The weights' gradient falls out of the table's: the warp that sums token v's gradient rows has
// E[v]'s tile in registers and takes each row's inner product with it on the way.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "operators.cuh"

namespace hanns {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSegmentThreads = 64;   // two warps: a block ends with the longer of two segments
constexpr int kLimit = 32;            // longest segment of one warp
constexpr int kPiece = 64;            // least entries of a longer one's pieces
constexpr int kDots = 8;              // inner products that are reduced together
// Vectors of a row that a lane takes, rows that it has on the way then, and the blocks of an SM
// that its registers are kept to (more spill, fewer leave the memory idle).
constexpr int kMostPacks = 4;
__host__ __device__ constexpr int rows_ahead(int packs) { return packs == 1 ? 8 : packs == 2 ? 3 : 2; }
constexpr int blocks_of_sm(int packs, int ve, bool forward) {
    return packs == 1 ? 14 : ve == 1 ? 16 : forward ? (ve == 8 ? 16 : 18) : ve == 8 ? 10 : 14;
}
constexpr int kLookupPacks = 8;       // vectors of a lane in a lookup
constexpr int kMaxBinBits = 9, kMaxBins = 1 << kMaxBinBits;
constexpr int kSortItems = 4, kSortTile = kThreads * kSortItems;
// Up to so many tiles each adds up the counts of those before it itself, without a scan kernel between.
// The gradient of a lookup in 32,000 x 64 f32 (device time): 8 tiles of positions 29.8 us (with the scan
// 32.4), 16 tiles 32.6 (34.5), 24 36.1 (37.4), 32 39.8 (39.9), 64 45.4 (43.0).
constexpr int kFewTiles = 16;
// Offsets to a position of a tile from which the positions search among them: 3,000 positions and
// 70,000 bags sort in 20 us (marked 53), 16,000 bags 20 (23), 300 bags 16 (13.6 marked).
constexpr int kManyBags = 8;

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
    __device__ __forceinline__ int position(int64_t j) const { return (int)j; }
};
// Entry j of the positions sorted by token.
struct SortedEntries {
    const int32_t* src;
    const float* coef;
    const uint32_t* pos;
    __device__ __forceinline__ int position(int64_t j) const { return (int)pos[j]; }
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
    const int64_t* offsets;  // null: bag i is position i, and the functions here are not called
    int64_t n_bags, n_tokens;
    __device__ __forceinline__ void bounds(int64_t i, int64_t& lo, int64_t& hi) const {
        lo = clamp_pos(offsets[i], 0, n_tokens);
        hi = clamp_pos(offsets[i + 1], lo, n_tokens);
    }
    // The number of offsets that are at most p, found by a whole warp: a 32nd of the range a step.
    __device__ __forceinline__ int64_t starts_up_to_by_warp(int64_t p) const {
        const int lane = threadIdx.x & 31;
        int64_t a = 0, n = n_bags + 1;  // the answer is in [a, a + n]
        while (n > 0) {
            const int64_t step = (n + 31) / 32, at = a + lane * step;  // lane's part: [at, at + step)
            const bool below = at + step - 1 < a + n && offsets[at + step - 1] <= p;
            const int parts = __popc(__ballot_sync(0xffffffffu, below));
            a += parts * step;
            n = parts == 32 ? 0 : min(step - 1, n - parts * step);
            if (n < 0) n = 0;
        }
        return a;
    }
};
// A token's run of entries in the sorted order.
struct Run {
    int32_t token, lo, hi, reserved;
};

// A piece of a long segment: entries [lo, hi), piece `index` of `n`, the segment's first one at
// `first` in the list.
struct alignas(16) Piece {
    int32_t segment, lo, hi, index, first, n, reserved[2];
};
// Long segments of one piece and the pieces of longer ones are listed apart: only those need
// partial rows.  Rooms that ascending offsets stay within; what would pass them is dropped.
struct PieceLists {
    int32_t* count;              // of singles, of parts
    Piece *singles, *parts;
    int64_t most_singles, most_parts;
    int32_t length;              // least entries of a piece
    int32_t* arrived;            // [parts][piece tiles], used at a segment's first piece
    float* partial;              // [parts][piece tiles * lanes * VE]
    int32_t* partial_count;      // [parts][piece tiles]
};

struct SumArgs {
    const void* base;  // matrix of the summed rows
    int64_t ld;
    void* out;
    int64_t out_ld;
    int64_t n_segments, n_entries;
    int dim, lanes_log2;         // lanes that share a row's tile
    int tiles, piece_tiles;      // column tiles of a segment, and of a piece
    float scale;
    int mean;
    float* inv_counts;
    // inner products with the segment's row of a second matrix
    const void* dot_base;
    int64_t dot_ld;
    float* dot;                  // [tiles, or piece tiles of a long segment][n_entries], by position
    PieceLists lists;
};

// VE elements in accesses of at most 16 bytes.
template <class T, int VE>
__device__ __forceinline__ Pack<T, VE> load_wide(const T* p) {
    constexpr int N = VE * sizeof(T) > 16 ? 16 / sizeof(T) : VE;
    Pack<T, VE> r;
#pragma unroll
    for (int o = 0; o < VE; o += N) {
        const Pack<T, N> q = load_pack<T, N>(p + o);
#pragma unroll
        for (int k = 0; k < N; ++k) r.v[o + k] = q.v[k];
    }
    return r;
}

// Stores VE results in accesses of at most 16 bytes.
template <class TO, int VE>
__device__ __forceinline__ void store_row(TO* p, const float2 (&sum)[(VE + 1) / 2], float factor) {
    float acc[VE];
#pragma unroll
    for (int k = 0; k < VE; ++k) acc[k] = k & 1 ? sum[k / 2].y : sum[k / 2].x;
    constexpr int N = VE * sizeof(TO) > 16 ? 16 / sizeof(TO) : VE;
#pragma unroll
    for (int o = 0; o < VE; o += N) {
        Pack<TO, N> q;
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = from_f32<TO>(acc[o + e] * factor);
        *reinterpret_cast<Pack<TO, N>*>(p + o) = q;
    }
}

// The first column this lane works on (its vectors are 32 vectors apart), and the groups of lanes
// that take entries in turn where a row is narrower than a warp.
struct Lanes {
    int lane, count, groups, group, col;
    __device__ __forceinline__ Lanes(const SumArgs& a, int tile, int ve, int packs)
        : lane(threadIdx.x & 31), count(1 << a.lanes_log2), groups(32 >> a.lanes_log2), group(lane >> a.lanes_log2),
          col((((tile * packs) << a.lanes_log2) + (lane & (count - 1))) * ve) {}
};

// What a finished sum is multiplied by.
__device__ __forceinline__ float finish_factor(const SumArgs& a, int64_t seg, int64_t count, bool write) {
    float inv = 1.0f;
    if (a.mean) {
        inv = __fdiv_rn(1.0f, (float)(count > 0 ? count : 1));
        if (a.inv_counts && write) a.inv_counts[seg] = inv;
    }
    return a.scale * inv;
}

// Sums of v[u] over each group's lanes, kDots at a time: 4 + 2 + 1 exchanges and one for each
// remaining doubling.  The result is v[0], of the entry whose number is returned (the same in
// lanes that differ below the group's width / kDots).
__device__ __forceinline__ int reduce_dots(float (&v)[kDots], int lanes_log2, int lane) {
    int entry = 0;
#pragma unroll
    for (int half = kDots / 2; half; half >>= 1) {
        --lanes_log2;
        const int bit = 1 << lanes_log2;
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
        }
        entry += up ? half : 0;
    }
    for (int bit = 1 << lanes_log2 >> 1; bit; bit >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
    return entry;
}

// A warp's counted entries of a batch of 32.
struct Batch {
    int64_t at[32];  // byte offset of the row in the summed matrix
    float coef[32];
    int32_t pos[32];
};

// Entries q, q + groups, ... of a batch of n, N per group (all there when Full).  step[t]: column of
// vector t; vectors behind the row's end are the first one's again.
template <class T, int VE, int Packs, bool Dot, int N, bool Full>
__device__ __forceinline__ void add_rows(const SumArgs& a, const Lanes& ln, const Batch& bt, const char* base,
                                         const int (&step)[Packs], int q, int n,
                                         float2 (&acc)[Packs][(VE + 1) / 2],
                                         const float2 (&e)[Packs][(VE + 1) / 2], float* dot) {
    constexpr int H = (VE + 1) / 2;
    Pack<T, VE> p[N][Packs];
    float d[kDots] = {};
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = q + u * ln.groups + ln.group;
        if (Full || i < n) {
            const T* row = reinterpret_cast<const T*>(base + bt.at[i]);
#pragma unroll
            for (int t = 0; t < Packs; ++t) p[u][t] = load_pack<T, VE>(row + step[t]);
        }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = q + u * ln.groups + ln.group;
        if (!Full && i >= n) continue;
        const float c = bt.coef[i];
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int t = 0; t < Packs; ++t) {
            float2 x[H];
            unpack(p[u][t], x);
#pragma unroll
            for (int k = 0; k < H; ++k) {
                acc[t][k] = fma2_rn(x[k], make_float2(c, c), acc[t][k]);
                if (Dot) {
                    if (ln.col + t * 32 * VE < a.dim) sum = fma2_rn(x[k], e[t][k], sum);
                }
            }
        }
        if (Dot) d[u] = sum.x + sum.y;
    }
    if constexpr (Dot) {
        if (ln.count >= kDots) {
            const int i = q + reduce_dots(d, a.lanes_log2, ln.lane) * ln.groups + ln.group;
            if (i < n && i < q + N * ln.groups && (ln.lane & (ln.count / kDots - 1)) == 0) dot[bt.pos[i]] = d[0];
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = q + u * ln.groups + ln.group;
                for (int bit = ln.count >> 1; bit; bit >>= 1) d[u] += __shfl_xor_sync(0xffffffffu, d[u], bit);
                if (i < n && (ln.lane & (ln.count - 1)) == 0) dot[bt.pos[i]] = d[u];
            }
        }
    }
}

// The sum of entries [lo, hi) over this warp's column tile, in every lane for its columns (vectors
// behind the last column are another's and are not stored).  Returns the number of counted
// entries.
template <class T, class TE, int VE, int Packs, bool Dot, class Entries>
__device__ __forceinline__ int sum_entries(const SumArgs& a, const Lanes& ln, Batch& bt, const Entries& entries,
                                           int64_t lo, int64_t hi, const TE* dot_row, float* dot,
                                           float2 (&acc)[Packs][(VE + 1) / 2]) {
    constexpr int H = (VE + 1) / 2, N = rows_ahead(Packs), Tail = (N + 1) / 2;
    static_assert(N <= kDots, "reduce_dots takes a round's products");
    int step[Packs];
#pragma unroll
    for (int t = 0; t < Packs; ++t) step[t] = ln.col + t * 32 * VE < a.dim ? ln.col + t * 32 * VE : 0;
    const char* base = static_cast<const char*>(a.base);
    float2 e[Packs][H];
#pragma unroll
    for (int t = 0; t < Packs; ++t)
#pragma unroll
        for (int k = 0; k < H; ++k) acc[t][k] = e[t][k] = make_float2(0.0f, 0.0f);
    int row = -1, pos = 0, count = 0;
    float coef = 0.0f;
    auto look_up = [&](int64_t b) {
        row = -1;
        if (b + ln.lane < hi) {
            entries.get(b + ln.lane, row, coef);
            if (Dot) pos = entries.position(b + ln.lane);
        }
    };
    look_up(lo);
    if constexpr (Dot) {
#pragma unroll
        for (int t = 0; t < Packs; ++t) unpack(load_wide<TE, VE>(dot_row + step[t]), e[t]);
    }
    for (int64_t b = lo; b < hi; b += 32) {
        const uint32_t counted = __ballot_sync(0xffffffffu, row >= 0);
        const int n = __popc(counted);
        __syncwarp();
        if (row >= 0) {
            const int i = __popc(counted & ((1u << ln.lane) - 1));
            bt.at[i] = (int64_t)row * a.ld * (int)sizeof(T);
            bt.coef[i] = coef;
            if (Dot) bt.pos[i] = pos;
        }
        __syncwarp();
        if (b + 32 < hi) look_up(b + 32);
        count += n;
        int q = 0;
        for (; q + N * ln.groups <= n; q += N * ln.groups)
            add_rows<T, VE, Packs, Dot, N, true>(a, ln, bt, base, step, q, n, acc, e, dot);
        for (; q < n; q += Tail * ln.groups)
            add_rows<T, VE, Packs, Dot, Tail, false>(a, ln, bt, base, step, q, n, acc, e, dot);
    }
    for (int m = 16; m >= ln.count; m >>= 1)
#pragma unroll
        for (int k = 0; k < H; ++k) {  // a narrow row has one vector a lane
            acc[0][k].x += __shfl_xor_sync(0xffffffffu, acc[0][k].x, m);
            acc[0][k].y += __shfl_xor_sync(0xffffffffu, acc[0][k].y, m);
        }
    return count;
}

// Stores a lane's vectors of a row.
template <class TO, int VE, int Packs>
__device__ __forceinline__ void store_sums(const SumArgs& a, const Lanes& ln, TO* row,
                                           const float2 (&acc)[Packs][(VE + 1) / 2], float factor) {
    if (ln.lane >= ln.count) return;
#pragma unroll
    for (int t = 0; t < Packs; ++t)
        if (ln.col + t * 32 * VE < a.dim) store_row<TO, VE>(row + ln.col + t * 32 * VE, acc[t], factor);
}

// Lists a long segment's pieces (a whole warp's call).
__device__ __forceinline__ void list_pieces(const SumArgs& a, int lane, int32_t seg, int32_t lo, int32_t hi) {
    const PieceLists& l = a.lists;
    // the square root: one after the other come a piece's entries and then the pieces
    const int length = max(l.length, (int)sqrtf(1.5f * (float)(hi - lo)));
    const int n = (int)(((int64_t)(hi - lo) + length - 1) / length);
    int32_t first = 0;
    if (lane == 0) first = atomicAdd(l.count + (n > 1), n);
    first = __shfl_sync(0xffffffffu, first, 0);
    Piece* to = n > 1 ? l.parts : l.singles;
    const int64_t room = n > 1 ? l.most_parts : l.most_singles;
    if (first < 0) return;
    for (int i = lane; i < n && first + (int64_t)i < room; i += 32)
        to[first + (int64_t)i] = Piece{seg,   lo + i * length, (int32_t)min((int64_t)hi, lo + (i + 1) * (int64_t)length),
                                       i,     first,           n,
                                       {0, 0}};
    if (n > 1 && first < room)
        for (int t = lane; t < a.piece_tiles; t += 32) l.arrived[(int64_t)first * a.piece_tiles + t] = 0;
}

// A segment's row (of not more than kLimit entries) by one warp and column tile.
template <class T, class TO, int VE, int Packs, bool Dot, class Entries>
__device__ __forceinline__ void sum_segment(const SumArgs& a, const Lanes& ln, Batch& bt, const Entries& entries,
                                            int64_t seg, int64_t lo, int64_t hi, int tile) {
    float2 acc[Packs][(VE + 1) / 2];
    const TO* dot_row = static_cast<const TO*>(a.dot_base) + seg * a.dot_ld;
    float* dot = a.dot + (int64_t)tile * a.n_entries;
    const int count = sum_entries<T, TO, VE, Packs, Dot>(a, ln, bt, entries, lo, hi, dot_row, dot, acc);
    const float f = finish_factor(a, seg, count, tile == 0 && ln.lane == 0);
    store_sums<TO, VE, Packs>(a, ln, static_cast<TO*>(a.out) + seg * a.out_ld, acc, f);
}

// Forward: one warp per (bag, column tile).  Bound by the gather through the L2 and the chain offsets
// - tokens - rows: of 150,001 tokens in 10,000 bags of a 768-wide bf16 table this kernel's share
// (198 MB through the L2, rows and vectors) takes 25 us, 8 TB/s.  Longest bag here 32: 25 + 15 us
// with the pieces, 64: 37 + 14, 16: 21 + 30.
template <class T, class TO, int VE, int Packs>
__global__ void __launch_bounds__(kSegmentThreads, blocks_of_sm(Packs, VE, true))
    bags_kernel(SumArgs a, TokenEntries entries, BagSegments bags) {
    wait_for_previous();
    __shared__ Batch batch[kSegmentThreads / 32];
    const uint32_t w = blockIdx.x * (kSegmentThreads / 32) + (threadIdx.x >> 5);
    const uint32_t seg = w / (uint32_t)a.tiles, tile = w - seg * (uint32_t)a.tiles;
    if (seg >= a.n_segments) return;
    const Lanes ln(a, tile, VE, Packs);
    int64_t lo, hi;
    bags.bounds(seg, lo, hi);
    if (hi - lo > kLimit) {
        if (tile == 0) list_pieces(a, ln.lane, (int32_t)seg, (int32_t)lo, (int32_t)hi);
        return;
    }
    sum_segment<T, TO, VE, Packs, false>(a, ln, batch[threadIdx.x >> 5], entries, seg, lo, hi, tile);
}

// Backward: one warp per (run, column tile), and behind those one per 2^clear_log2 table rows for the
// rows of tokens without a run.  The same 150,001 tokens in f32, both gradients: 52 us, then 45 us for the
// pieces of tokens that occur more than 32 times (59 % of the positions).
template <class T, class TO, int VE, int Packs, bool Dot>
__global__ void __launch_bounds__(kSegmentThreads, blocks_of_sm(Packs, VE, false))
    runs_kernel(SumArgs a, SortedEntries entries, const Run* runs, const int32_t* n_runs, int64_t most_runs,
                const uint32_t* touched, int clear_log2) {
    wait_for_previous();
    __shared__ Batch batch[kSegmentThreads / 32];
    const int64_t w = (int64_t)blockIdx.x * (kSegmentThreads / 32) + (threadIdx.x >> 5);
    if (w < most_runs * a.tiles) {
        const uint32_t r = (uint32_t)w / (uint32_t)a.tiles, tile = (uint32_t)w - r * (uint32_t)a.tiles;
        if ((int)r >= *n_runs) return;
        const Run run = runs[r];
        const Lanes ln(a, tile, VE, Packs);
        if (run.hi - run.lo > kLimit) {
            if (tile == 0) list_pieces(a, ln.lane, run.token, run.lo, run.hi);
            return;
        }
        sum_segment<T, TO, VE, Packs, Dot>(a, ln, batch[threadIdx.x >> 5], entries, run.token, run.lo, run.hi, tile);
        return;
    }
    const int64_t first = (w - most_runs * a.tiles) << clear_log2;
    if (first >= a.n_segments) return;
    const int each = (int)min((int64_t)1 << clear_log2, a.n_segments - first);
    uint32_t rows = ~touched[first / 32] >> (first & 31);
    if (each < 32) rows &= (1u << each) - 1;
    const float2 zeros[Packs][(VE + 1) / 2] = {};
    for (; rows; rows &= rows - 1)
        for (int tile = 0; tile < a.tiles; ++tile)
            store_sums<TO, VE, Packs>(a, Lanes(a, tile, VE, Packs),
                                      static_cast<TO*>(a.out) + (first + __ffs(rows) - 1) * a.out_ld, zeros, 1.0f);
}

// One warp per (piece, column tile), one vector a lane: there may be few, and then a warp's time is
// what counts.  The segment's last warp to arrive adds the pieces, in order.
template <class T, class TO, int VE, bool Dot, class Entries>
__global__ void __launch_bounds__(kSegmentThreads, Dot ? 12 : 14) pieces_kernel(SumArgs a, Entries entries) {
    wait_for_previous();
    constexpr int Packs = 1;
    __shared__ Batch batch[kSegmentThreads / 32];
    const PieceLists& l = a.lists;
    const int64_t n_parts = min((int64_t)max(l.count[1], 0), l.most_parts);
    const int64_t n_singles = min((int64_t)max(l.count[0], 0), l.most_singles);
    const int64_t items = (n_parts + n_singles) * a.piece_tiles;
    const int width = (a.piece_tiles << a.lanes_log2) * VE;
    constexpr int of_block = kSegmentThreads / 32;
    for (int64_t item = (int64_t)blockIdx.x * of_block + (threadIdx.x >> 5); item < items;
         item += (int64_t)gridDim.x * of_block) {
        const int64_t at = item / a.piece_tiles;
        const int tile = (int)(item - at * a.piece_tiles);
        const Lanes ln(a, tile, VE, Packs);
        const Piece pc = at < n_parts ? l.parts[at] : l.singles[at - n_parts];
        float2 acc[Packs][(VE + 1) / 2];
        int count = sum_entries<T, TO, VE, Packs, Dot>(a, ln, batch[threadIdx.x >> 5], entries, pc.lo, pc.hi,
                                                       static_cast<const TO*>(a.dot_base) + pc.segment * a.dot_ld,
                                                       a.dot + (int64_t)tile * a.n_entries, acc);
        if (pc.n > 1) {
            if (ln.lane < ln.count) store_row<float, VE>(l.partial + at * width + ln.col, acc[0], 1.0f);
            if (ln.lane == 0) l.partial_count[item] = count;
            __threadfence();
            __syncwarp();
            int before = 0;
            if (ln.lane == 0) before = atomicAdd(&l.arrived[(int64_t)pc.first * a.piece_tiles + tile], 1);
            if (__shfl_sync(0xffffffffu, before, 0) != pc.n - 1) continue;
            __threadfence();
            count = 0;
            const int n = (int)min((int64_t)pc.n, l.most_parts - pc.first);
            if (a.mean) {
                for (int i = ln.lane; i < n; i += 32)
                    count += __ldcg(l.partial_count + (int64_t)(pc.first + i) * a.piece_tiles + tile);
                count = __reduce_add_sync(0xffffffffu, count);
            }
#pragma unroll
            for (int t = 0; t < Packs; ++t) {
#pragma unroll
                for (int k = 0; k < (VE + 1) / 2; ++k) acc[t][k] = make_float2(0.0f, 0.0f);
                constexpr int kJoin = VE >= 4 ? 48 / VE : 16;  // partial rows on the way
                for (int i0 = ln.group; i0 < n; i0 += kJoin * ln.groups) {
                    float x[kJoin][VE];
#pragma unroll
                    for (int u = 0; u < kJoin; ++u) {
                        const int i = i0 + u * ln.groups;
                        const float* p = l.partial + (int64_t)(pc.first + min(i, n - 1)) * width + ln.col + t * 32 * VE;
                        if constexpr (VE >= 4) {
#pragma unroll
                            for (int k = 0; k < VE; k += 4) {
                                const float4 v = __ldcg(reinterpret_cast<const float4*>(p + k));
                                x[u][k] = v.x, x[u][k + 1] = v.y, x[u][k + 2] = v.z, x[u][k + 3] = v.w;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < VE; ++k) x[u][k] = __ldcg(p + k);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kJoin; ++u)
#pragma unroll
                        for (int k = 0; k < VE; ++k)
                            if (i0 + u * ln.groups < n) (k & 1 ? acc[t][k / 2].y : acc[t][k / 2].x) += x[u][k];
                }
                for (int m = 16; m >= ln.count; m >>= 1)
#pragma unroll
                    for (int k = 0; k < (VE + 1) / 2; ++k) {
                        acc[t][k].x += __shfl_xor_sync(0xffffffffu, acc[t][k].x, m);
                        acc[t][k].y += __shfl_xor_sync(0xffffffffu, acc[t][k].y, m);
                    }
            }
        }
        const float f = finish_factor(a, pc.segment, count, tile == 0 && ln.lane == 0);
        store_sums<TO, VE, Packs>(a, ln, static_cast<TO*>(a.out) + (int64_t)pc.segment * a.out_ld, acc, f);
    }
}

// Bags of one token: a warp moves a column tile of several rows, kLookupPacks vectors a lane in all.
// Bound by memory: 16,384 rows of 768 bf16 take 8.3 us (50 MB).
template <class T, class TO, int VE, int Packs>
__global__ void __launch_bounds__(kSegmentThreads) lookup_kernel(SumArgs a, TokenEntries entries) {
    wait_for_previous();
    constexpr int kRows = kLookupPacks / Packs, H = (VE + 1) / 2;
    const uint32_t w = blockIdx.x * (kSegmentThreads / 32) + (threadIdx.x >> 5);
    const uint32_t batch = w / (uint32_t)a.tiles, tile = w - batch * (uint32_t)a.tiles;
    const Lanes ln(a, tile, VE, Packs);
    const int64_t first = (int64_t)batch * kRows * ln.groups;
    if (first >= a.n_segments) return;
    const T* base = static_cast<const T*>(a.base);
    Pack<T, VE> p[kRows][Packs];
    int row[kRows];
    float f[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
        const int64_t i = first + u * ln.groups + ln.group;
        row[u] = -1;
        f[u] = 0.0f;
        if (i < a.n_segments) entries.get(i, row[u], f[u]);
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u)
#pragma unroll
        for (int t = 0; t < Packs; ++t)
            if (row[u] >= 0 && ln.col + t * 32 * VE < a.dim)
                p[u][t] = load_pack<T, VE>(base + (int64_t)row[u] * a.ld + ln.col + t * 32 * VE);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
        const int64_t i = first + u * ln.groups + ln.group;
        if (i >= a.n_segments) continue;
        if (a.mean && a.inv_counts && tile == 0 && (ln.lane & (ln.count - 1)) == 0) a.inv_counts[i] = 1.0f;
#pragma unroll
        for (int t = 0; t < Packs; ++t) {
            const int col = ln.col + t * 32 * VE;
            if (col >= a.dim) continue;
            float2 acc[H] = {};
            if (row[u] >= 0) {
                unpack(p[u][t], acc);
#pragma unroll
                for (int k = 0; k < H; ++k) acc[k] = mul2_rn(acc[k], make_float2(f[u], f[u]));
            }
            store_row<TO, VE>(static_cast<TO*>(a.out) + i * a.out_ld + col, acc, a.scale);
        }
    }
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
    uint32_t *key_in, *pos_in;  // the first pass's count writes key_in, in position order
    uint32_t *key_out, *pos_out;
    int32_t* bag;    // [n] by position, from the first pass
    int32_t* src;
    float* coef;
    // zeroed by the first pass: bit maps of the tokens with a run, and with a long one; counts
    uint32_t *touched, *lengthy;
    int32_t *list_counts, *n_runs;
    Run* runs;
    int64_t most_runs;
    int32_t* hist;   // [bins][tiles]; few tiles: [tiles][bins]
    int32_t* total;  // [bins]
};

// The lanes of the warp that hold the same digit: a ballot a bit, whose time does not grow with the
// number of different digits as that of __match_any_sync does (one block's sort of 4,001 positions
// 16 us for 19, a pass over 150,001 keys 4.4 for 4.9).
template <int Bits>
__device__ __forceinline__ uint32_t lanes_with(int d) {
    uint32_t same = 0xffffffffu;
#pragma unroll
    for (int b = 0; b < Bits; ++b) {
        const bool one = d >> b & 1;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// The bags of a tile's positions, into bag[]: the offsets at or before its first and its last position
// are searched for, those between are marked at their positions (the last of equal ones counts),
// and the largest mark up to a position is its bag.  Where they are many (empty bags), each position
// searches among them instead.
template <int Threads>
__device__ void tile_bags(const BagSegments& bags, int64_t base, int32_t* bag, int32_t* warp_max) {
    constexpr int Tile = Threads * kSortItems;
    if (!bags.offsets) {
        for (int i = threadIdx.x; i < Tile; i += Threads) bag[i] = (int32_t)(base + i);
        __syncthreads();
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t last = min(base + Tile, bags.n_tokens) - 1;
    const int64_t starts = bags.starts_up_to_by_warp(warp & 1 ? last : base);
    if (warp < 2 && lane == 0) warp_max[warp] = (int32_t)starts;
    __syncthreads();
    const int32_t before = warp_max[0], after = warp_max[1];
    if (after - before > kManyBags * Tile) {
        int32_t a[kSortItems], n[kSortItems];  // the answer is in [a, a + n]; all items' steps together
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) a[i] = before, n[i] = after - before;
        for (int32_t left = after - before; left > 0; left >>= 1) {
#pragma unroll
            for (int i = 0; i < kSortItems; ++i) {
                if (n[i] <= 0) continue;
                const int32_t half = n[i] >> 1;
                if (bags.offsets[a[i] + half] <= base + i * Threads + threadIdx.x) {
                    a[i] += half + 1;
                    n[i] -= half + 1;
                } else {
                    n[i] = half;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) bag[i * Threads + threadIdx.x] = a[i] <= bags.n_bags ? a[i] - 1 : -1;
        __syncthreads();
        return;
    }
    for (int i = threadIdx.x; i < Tile; i += Threads) bag[i] = before;
    __syncthreads();
#pragma unroll 4
    // (unsigned: k may pass 2^31 in its last step)
    for (uint32_t k = (uint32_t)before + threadIdx.x; k < (uint32_t)after; k += Threads) {
        const int64_t o = bags.offsets[k] - base;
        if (o > 0 && o < Tile) atomicMax(&bag[o], (int32_t)k + 1);
    }
    __syncthreads();
    int32_t v[kSortItems];
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        v[i] = bag[threadIdx.x * kSortItems + i];
        if (i) v[i] = max(v[i], v[i - 1]);
    }
    int32_t top = v[kSortItems - 1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) top = max(top, __shfl_up_sync(0xffffffffu, top, d));
    if (lane == 31) warp_max[warp] = top;
    int32_t left = __shfl_up_sync(0xffffffffu, top, 1);
    __syncthreads();
    if (lane == 0) left = 0;
    for (int w = 0; w < warp; ++w) left = max(left, warp_max[w]);
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int32_t starts = max(v[i], left);  // offsets at or before the position
        bag[threadIdx.x * kSortItems + i] = starts <= bags.n_bags ? starts - 1 : -1;
    }
    __syncthreads();
}
__device__ __forceinline__ float entry_factor(const SortArgs& a, uint32_t pos, int32_t bag) {
    float c = a.scale;
    if (a.weights) c *= a.weights[pos];
    if (a.inv_counts && bag >= 0) c *= a.inv_counts[bag];
    return c;
}
__device__ __forceinline__ void clear_runs(const SortArgs& a) {  // every thread of the grid
    const int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i0 < 2) a.list_counts[i0] = 0;
    if (i0 == 2) *a.n_runs = 0;
    for (int64_t i = i0; i < (a.rows + 31) / 32; i += (int64_t)gridDim.x * blockDim.x)
        a.touched[i] = a.lengthy[i] = 0;
}

template <bool First>
__global__ void __launch_bounds__(kThreads) sort_count_kernel(SortArgs a) {
    wait_for_previous();
    __shared__ int32_t count[kMaxBins];
    __shared__ int32_t bag[First ? kSortTile : 1], warp_max[kWarps];
    for (int b = threadIdx.x; b < a.bins; b += kThreads) count[b] = 0;
    const int64_t base = (int64_t)blockIdx.x * kSortTile;
    int64_t token[kSortItems];  // or the keys of a later pass; all are read before any is used
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t j = base + i * kThreads + threadIdx.x;
        token[i] = -1;
        if (j < a.n) token[i] = First ? a.tokens[j] : (int64_t)a.key_in[j];
    }
    if constexpr (First) {
        clear_runs(a);
        tile_bags<kThreads>(a.bags, base, bag, warp_max);
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int at = i * kThreads + threadIdx.x;
        const int64_t j = base + at;
        if (j >= a.n) break;
        uint32_t key;
        if constexpr (First) {
            // a position that counts nowhere has the key `rows` and no bag
            const int32_t b = (uint64_t)token[i] < (uint64_t)a.rows ? bag[at] : -1;
            key = b >= 0 ? (uint32_t)token[i] : (uint32_t)a.rows;
            a.bag[j] = b;
            a.key_in[j] = key;
        } else {
            key = (uint32_t)token[i];
        }
        atomicAdd(&count[(key >> a.shift) & (a.bins - 1)], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.bins; b += kThreads) {
        const int64_t at = a.tiles > kFewTiles ? (int64_t)b * a.tiles + blockIdx.x : (int64_t)blockIdx.x * a.bins + b;
        a.hist[at] = count[b];
    }
}

// One warp per digit: its counts become the number of its keys in earlier tiles.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(SortArgs a) {
    wait_for_previous();
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
    wait_for_previous();
    __shared__ int32_t seen[kWarps][kMaxBins];  // a warp's keys per digit, then its first place
    __shared__ int32_t warp_sum[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&seen[0][0])[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile + warp * (32 * kSortItems);
    // all that is read, before it is used
    uint32_t key[kSortItems], pos[kSortItems];
    int32_t rank[kSortItems], bag[kSortItems];
    float coef[kSortItems];
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t j = base + i * 32 + lane;
        key[i] = j < a.n ? a.key_in[j] : 0;
        pos[i] = First ? (uint32_t)j : j < a.n ? a.pos_in[j] : 0;
    }
    // keys of digits b0 and b0 + 1 in all tiles and in those before this one
    // (two digits per thread: bins <= 2 * kThreads)
    const int b0 = threadIdx.x * 2;
    int32_t all[2] = {}, earlier[2] = {};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if (b0 + q >= a.bins) continue;
        if (a.tiles > kFewTiles) {
            all[q] = a.total[b0 + q];
            earlier[q] = a.hist[(int64_t)(b0 + q) * a.tiles + blockIdx.x];
        } else {
#pragma unroll 8
            for (int t = 0; t < a.tiles; ++t) {
                const int32_t c = a.hist[t * a.bins + b0 + q];
                all[q] += c;
                if (t < (int)blockIdx.x) earlier[q] += c;
            }
        }
    }
    if constexpr (Last) {
#pragma unroll
        for (int i = 0; i < kSortItems; ++i) bag[i] = base + i * 32 + lane < a.n ? a.bag[pos[i]] : -1;
#pragma unroll
        for (int i = 0; i < kSortItems; ++i)
            coef[i] = base + i * 32 + lane < a.n ? entry_factor(a, pos[i], bag[i]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const bool in = base + i * 32 + lane < a.n;
        const int d = (key[i] >> a.shift) & (a.bins - 1);
        const uint32_t peers = lanes_with<kMaxBinBits>(d) & __ballot_sync(0xffffffffu, in);
        rank[i] = 0;
        if (in) rank[i] = seen[warp][d] + __popc(peers & ((1u << lane) - 1));
        __syncwarp();
        if (in && (peers >> lane) == 1) seen[warp][d] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    int32_t s = all[0] + all[1];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int32_t o = __shfl_up_sync(0xffffffffu, s, m);
        if (lane >= m) s += o;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int32_t before = s - all[0] - all[1];  // keys of smaller digits
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int b = b0 + q;
        if (b < a.bins) {
            int32_t at = before + (q ? all[0] : 0) + earlier[q], of_warp[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) of_warp[w] = seen[w][b];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                seen[w][b] = at;
                at += of_warp[w];
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
        a.pos_out[to] = pos[i];
        if constexpr (Last) {
            a.src[to] = bag[i];
            a.coef[to] = coef[i];
        }
    }
}

// Lists each token's run; the thread at its first entry looks for its end, in steps that double.
__global__ void __launch_bounds__(kThreads) sort_runs_kernel(SortArgs a, const uint32_t* key) {
    wait_for_previous();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    uint32_t k = (uint32_t)a.rows;
    if (i < a.n) k = key[i];
    const bool begins = k < a.rows && (i == 0 || key[i - 1] != k);
    int64_t end = i + 1;
    if (begins) {
        int64_t in = i, step = 1;  // key[in] is k
        while (in + step < a.n && key[in + step] == k) {
            in += step;
            step *= 2;
        }
        for (; step; step >>= 1)
            if (in + step < a.n && key[in + step] == k) in += step;
        end = in + 1;
        atomicOr(a.touched + k / 32, 1u << (k & 31));
        if (end - i > kLimit) atomicOr(a.lengthy + k / 32, 1u << (k & 31));
    }
    const int lane = threadIdx.x & 31;
    const uint32_t who = __ballot_sync(0xffffffffu, begins);
    int32_t at = 0;
    if (lane == 0 && who) at = atomicAdd(a.n_runs, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
    if (begins) a.runs[at] = Run{(int32_t)k, (int32_t)i, (int32_t)end, 0};
}

// The whole sort and the list of runs for up to kSmallSort positions: one block, the keys in shared
// memory, instead of five launches.  3,001 positions in 257 bags: 13.5 us, the whole gradient 19.5 us
// on the device for 22 and 28 us of the host's for 37; at 4,001 positions the device takes 22.8 us
// either way, beyond that several blocks are faster.
constexpr int kSmallThreads = 1024, kSmallWarps = kSmallThreads / 32, kSmallItems = 4;
static_assert(kSmallItems == kSortItems);  // tile_bags
constexpr int kSmallSort = kSmallThreads * kSmallItems, kSmallBits = 8;
constexpr int64_t kSmallRows = 1 << 20;  // bit maps that one block clears quickly

__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(SortArgs a, int passes) {
    wait_for_previous();
    __shared__ uint32_t s_key[kSmallSort];
    __shared__ uint16_t s_pos[kSmallSort];
    __shared__ uint16_t seen[kSmallWarps][1 << kSmallBits];  // a warp's keys per digit, then its first place
    __shared__ int32_t warp_sum[(1 << kSmallBits) / 32];
    __shared__ int32_t n_runs;
    __shared__ int32_t warp_max[kSmallWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // places of this thread's items, in every pass
    auto place = [&](int i) { return warp * (32 * kSmallItems) + i * 32 + lane; };
    auto used = [&](int i) { return place(i) - lane < a.n; };  // alike in the warp; others take no part
    if (threadIdx.x < 2) a.list_counts[threadIdx.x] = 0;
    if (threadIdx.x == 0) n_runs = 0;
    for (int64_t i = threadIdx.x; i < (a.rows + 31) / 32; i += kSmallThreads) a.touched[i] = a.lengthy[i] = 0;
    // the bags of the positions; the keys come to lie there later
    int32_t* s_bag = reinterpret_cast<int32_t*>(s_key);
    int64_t token[kSmallItems];
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
        const int j = place(i);
        token[i] = j < a.n ? a.tokens[j] : -1;
    }
    tile_bags<kSmallThreads>(a.bags, 0, s_bag, warp_max);
    uint32_t key[kSmallItems];
    uint16_t pos[kSmallItems];
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
        const int j = place(i);
        pos[i] = (uint16_t)j;
        key[i] = 0xffffffffu;  // behind the last position
        if (j >= a.n) continue;
        const int32_t bag = (uint64_t)token[i] < (uint64_t)a.rows ? s_bag[j] : -1;
        a.bag[j] = bag;
        key[i] = bag >= 0 ? (uint32_t)token[i] : (uint32_t)a.rows;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * kSmallBits;
        uint32_t* words = reinterpret_cast<uint32_t*>(&seen[0][0]);
        for (int b = threadIdx.x; b < kSmallWarps << (kSmallBits - 1); b += kSmallThreads) words[b] = 0;
        __syncthreads();
        int rank[kSmallItems];
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            if (!used(i)) continue;
            const int d = (key[i] >> shift) & ((1 << kSmallBits) - 1);
            const uint32_t peers = lanes_with<kSmallBits>(d);
            rank[i] = seen[warp][d] + __popc(peers & ((1u << lane) - 1));
            __syncwarp();
            if ((peers >> lane) == 1) seen[warp][d] += (uint16_t)__popc(peers);
            __syncwarp();
        }
        __syncthreads();
        int32_t total = 0, upto = 0;
        uint16_t of_warp[kSmallWarps];  // this thread's digit
        if (threadIdx.x < 1 << kSmallBits) {
#pragma unroll
            for (int w = 0; w < kSmallWarps; ++w) of_warp[w] = seen[w][threadIdx.x];
#pragma unroll
            for (int w = 0; w < kSmallWarps; ++w) total += of_warp[w];
            upto = total;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int32_t o = __shfl_up_sync(0xffffffffu, upto, m);
                if (lane >= m) upto += o;
            }
            if (lane == 31) warp_sum[warp] = upto;
        }
        __syncthreads();
        if (threadIdx.x < 1 << kSmallBits) {
            int32_t before = upto - total;
            for (int w = 0; w < warp; ++w) before += warp_sum[w];
#pragma unroll
            for (int w = 0; w < kSmallWarps; ++w) {
                seen[w][threadIdx.x] = (uint16_t)before;
                before += of_warp[w];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            if (!used(i)) continue;
            const int to = seen[warp][(key[i] >> shift) & ((1 << kSmallBits) - 1)] + rank[i];
            s_key[to] = key[i];
            s_pos[to] = pos[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            if (!used(i)) continue;
            key[i] = s_key[place(i)];
            pos[i] = s_pos[place(i)];
        }
    }
    int32_t bag[kSmallItems];
    float coef[kSmallItems];
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) bag[i] = place(i) < a.n ? a.bag[pos[i]] : -1;
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) coef[i] = place(i) < a.n ? entry_factor(a, pos[i], bag[i]) : 0.0f;
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
        const int at = place(i);
        const uint32_t k = key[i];
        const bool begins = k < a.rows && (at == 0 || s_key[at - 1] != k);
        if (at < a.n) {
            a.pos_out[at] = pos[i];
            a.src[at] = bag[i];
            a.coef[at] = coef[i];
        }
        int end = at + 1;
        if (begins) {
            int in = at, step = 1;  // s_key[in] is k
            while (in + step < a.n && s_key[in + step] == k) {
                in += step;
                step *= 2;
            }
            for (; step; step >>= 1)
                if (in + step < a.n && s_key[in + step] == k) in += step;
            end = in + 1;
            atomicOr(a.touched + k / 32, 1u << (k & 31));
            if (end - at > kLimit) atomicOr(a.lengthy + k / 32, 1u << (k & 31));
        }
        const uint32_t who = __ballot_sync(0xffffffffu, begins);
        int32_t to = 0;
        if (lane == 0 && who) to = atomicAdd(&n_runs, __popc(who));
        to = __shfl_sync(0xffffffffu, to, 0) + __popc(who & ((1u << lane) - 1));
        if (begins) a.runs[to] = Run{(int32_t)k, at, end, 0};
    }
    __syncthreads();
    if (threadIdx.x == 0) *a.n_runs = n_runs;
}

// dw_j: the column tiles' inner products in order, times scale / c_bag; 0 where j does not count.
__global__ void __launch_bounds__(kThreads)
    weights_grad_kernel(const float* dot, int tiles, int piece_tiles, SortArgs a, float* d_weights) {
    wait_for_previous();
    const int64_t j = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (j >= a.n) return;
    const int32_t b = a.bag[j];
    float v = 0.0f;
    if (b >= 0) {
        const uint32_t t = (uint32_t)a.tokens[j];
        const int n = a.lengthy[t / 32] >> (t & 31) & 1 ? piece_tiles : tiles;
        for (int i = 0; i < n; ++i) v += dot[(int64_t)i * a.n + j];
        v *= a.inv_counts ? a.scale * a.inv_counts[b] : a.scale;
    }
    d_weights[j] = v;
}

// ---------------------------------------------------------------- host
struct Matrix {
    const void* p;
    int64_t ld;
    int size;  // of an element
};

// Elements per access that every row of the matrices allows: 16 bytes of the first one's, 8, 4, or
// one element.  Forward, 150,001 tokens in 10,000 bags, with these accesses and with single elements:
// 500 bf16 (4 at a time) 35 and 80 us, 502 bf16 (2) 46 and 80, 502 f32 (2) 52 and 87.  Both gradients of
// f32 rows of 502 (2 at a time) take 188 and 183: there the single elements' wider tiles make up for it.
int vector_elems(int dim, std::initializer_list<Matrix> all) {
    for (int ve = 16 / all.begin()->size; ve > 1; ve /= 2) {
        bool ok = dim % ve == 0;
        for (const Matrix& m : all) {
            const int bytes = std::min(16, ve * m.size);
            ok = ok && (uintptr_t)m.p % bytes == 0 && (m.ld * m.size) % bytes == 0;
        }
        if (ok) return ve;
    }
    return 1;
}

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

// Least entries of a long segment's pieces.
int64_t piece_length(int64_t n_entries) { return std::max<int64_t>(kPiece, n_entries >> 14); }

// Tiles of a row of dim elements: as many lanes as its vectors need, up to a warp, and then up to
// `most` vectors a lane, as evenly as whole tiles allow.
struct Tiling {
    int lanes_log2 = 0, packs, tiles;
    Tiling(int dim, int ve, int most) {
        const int all = (dim + ve - 1) / ve;
        while (lanes_log2 < 5 && (1 << lanes_log2) < all) ++lanes_log2;
        tiles = (all + 32 * most - 1) / (32 * most);
        packs = (all + 32 * tiles - 1) / (32 * tiles);
    }
};
// Bounds for every vector width.
int64_t most_tiles(int dim) { return (dim + 31) / 32; }
int64_t most_width(int dim) { return (int64_t)dim + dim / 4 + 32 * 8 * 2; }

// The workspace: taken piece by piece, or only counted (p null).
struct Carver {
    char* p = nullptr;
    size_t used = 0;
    template <class T>
    T* take(size_t n) {
        T* r = p ? reinterpret_cast<T*>(p + used) : nullptr;
        used += round256(n * sizeof(T));
        return r;
    }
};

// Lists and partial rows of long segments, for any tiling.
void take_lists(SumArgs& a, Carver& ws) {
    PieceLists& l = a.lists;
    l.length = (int32_t)piece_length(a.n_entries);
    l.most_singles = a.n_entries / kLimit;
    l.most_parts = 2 * (a.n_entries / l.length);  // n > length entries have at most 2 n / length pieces
    l.count = ws.take<int32_t>(2);
    l.singles = ws.take<Piece>(l.most_singles);
    l.parts = ws.take<Piece>(l.most_parts);
    l.arrived = ws.take<int32_t>(l.most_parts * most_tiles(a.dim));
    l.partial = ws.take<float>(l.most_parts * most_width(a.dim));
    l.partial_count = ws.take<int32_t>(l.most_parts * most_tiles(a.dim));
}

unsigned grid_of(int64_t warps) {
    require(warps < (int64_t)1 << 32, "embed_bags: too many output tiles");
    constexpr int of_block = kSegmentThreads / 32;
    return (unsigned)((warps + of_block - 1) / of_block);
}

// Warps that clear the rows of tokens without a run: a row each until that is more than the SMs hold,
// then up to 32 rows each.
constexpr int64_t kMostClearing = 148 * 64;

// Launches the kernels of the sums; `b` and `so` are the forward and the backward call's.
template <class T, class TO, int VE, bool Dot, class Entries>
void launch_sum(SumArgs& a, const Entries& entries, const BagSegments& bags, const SortArgs& so, cudaStream_t s) {
    constexpr bool forward = std::is_same_v<Entries, TokenEntries>;
    // several vectors a lane for the widest accesses, and for single elements, of which rows have
    // the most (in between tiles stay narrow: fewer kernels, for widths that are seldom)
    constexpr bool several = VE * sizeof(T) == 16 || VE == 1;
    const Tiling narrow(a.dim, VE, 1), t(a.dim, VE, several ? kMostPacks : 1);
    a.lanes_log2 = t.lanes_log2;
    a.tiles = t.tiles;
    a.piece_tiles = narrow.tiles;
    if (a.n_segments == 0) return;
    auto launch = [&](auto packs) {
        constexpr int Packs = decltype(packs)::value;
        if constexpr (forward) {
            if (bags.offsets) {
                launch_early(bags_kernel<T, TO, VE, Packs>, grid_of(a.n_segments * a.tiles), kSegmentThreads, 0, s, a,
                             entries, bags);
            } else {
                const int64_t each = (int64_t)(kLookupPacks / Packs) * (32 >> a.lanes_log2);
                const unsigned grid = grid_of((a.n_segments + each - 1) / each * a.tiles);
                launch_early(lookup_kernel<T, TO, VE, Packs>, grid, kSegmentThreads, 0, s, a, entries);
            }
        } else {
            int clear_log2 = 0;
            while (clear_log2 < 5 && a.n_segments >> clear_log2 > kMostClearing) ++clear_log2;
            const int64_t warps = so.most_runs * a.tiles + ((a.n_segments - 1) >> clear_log2) + 1;
            launch_early(runs_kernel<T, TO, VE, Packs, Dot>, grid_of(warps), kSegmentThreads, 0, s, a, entries, so.runs,
                         so.n_runs, so.most_runs, so.touched, clear_log2);
        }
    };
    if constexpr (several) {
        switch (t.packs) {
            case 1: launch(std::integral_constant<int, 1>()); break;
            case 2: launch(std::integral_constant<int, 2>()); break;
            case 3: launch(std::integral_constant<int, 3>()); break;
            default: launch(std::integral_constant<int, 4>());
        }
    } else {
        launch(std::integral_constant<int, 1>());
    }
    if (forward && !bags.offsets) return;
    if (a.n_entries <= kLimit) return;
    const int64_t most = (a.lists.most_singles + a.lists.most_parts) * a.piece_tiles;
    const unsigned blocks = (unsigned)std::min<int64_t>(grid_of(most), 16 * 148);
    launch_early(pieces_kernel<T, TO, VE, Dot, Entries>, blocks, kSegmentThreads, 0, s, a, entries);
}

// In: type of the summed rows, Out: of the result (and of the rows of the inner products).
template <class T, class TO, bool Dot, class Entries>
void sum_segments(SumArgs& a, const Entries& entries, const BagSegments& bags, const SortArgs& so, cudaStream_t s) {
    const Matrix in{a.base, a.ld, sizeof(T)}, out{a.out, a.out_ld, sizeof(TO)};
    const Matrix table = Dot ? Matrix{a.dot_base, a.dot_ld, sizeof(TO)} : out;
    const int ve = vector_elems(a.dim, {in, out, table});
    constexpr int wide = 16 / sizeof(T);
    if (ve == wide) return launch_sum<T, TO, wide, Dot>(a, entries, bags, so, s);
    if (ve == wide / 2) return launch_sum<T, TO, wide / 2, Dot>(a, entries, bags, so, s);
    if constexpr (wide == 8) {
        if (ve == 2) return launch_sum<T, TO, 2, Dot>(a, entries, bags, so, s);
    }
    launch_sum<T, TO, 1, Dot>(a, entries, bags, so, s);
}

// Forward: from a table's type to the same or f32; backward the other way.
void sum_bags(int32_t in, int32_t out, SumArgs& a, const TokenEntries& e, const BagSegments& bags, cudaStream_t s) {
    const SortArgs none{};
    if (in == HANNS_DTYPE_F32) return sum_segments<float, float, false>(a, e, bags, none, s);
    if (in == HANNS_DTYPE_F16) {
        if (out == HANNS_DTYPE_F32) return sum_segments<__half, float, false>(a, e, bags, none, s);
        return sum_segments<__half, __half, false>(a, e, bags, none, s);
    }
    if (out == HANNS_DTYPE_F32) return sum_segments<__nv_bfloat16, float, false>(a, e, bags, none, s);
    sum_segments<__nv_bfloat16, __nv_bfloat16, false>(a, e, bags, none, s);
}
template <bool Dot>
void sum_runs(int32_t in, int32_t out, SumArgs& a, const SortedEntries& e, const SortArgs& so, cudaStream_t s) {
    const BagSegments none{};
    if (in == HANNS_DTYPE_F16) return sum_segments<__half, __half, Dot>(a, e, none, so, s);
    if (in == HANNS_DTYPE_BF16) return sum_segments<__nv_bfloat16, __nv_bfloat16, Dot>(a, e, none, so, s);
    if (out == HANNS_DTYPE_F32) return sum_segments<float, float, Dot>(a, e, none, so, s);
    if (out == HANNS_DTYPE_F16) return sum_segments<float, __half, Dot>(a, e, none, so, s);
    sum_segments<float, __nv_bfloat16, Dot>(a, e, none, so, s);
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
    require(aligned(b->tokens, 8) && aligned(b->offsets, 8), "embed_bags: misaligned tokens or offsets");
    require(aligned(b->weights, 4) && aligned(b->inv_counts, 4), "embed_bags: misaligned weights or inv_counts");
    require(aligned(b->table, dtype_bytes(b->dtype)), "embed_bags: misaligned table");
}

// Rows that are read may overlap (a broadcast row is `ld` 0), rows that are written may not.
void check_read(int64_t ld) { require(ld >= 0, "embed_bags: rows must not run backwards"); }
void check_written(int64_t rows, int64_t ld, int dim) {
    require(rows <= 1 || ld >= dim, "embed_bags: output rows overlap");
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

template <bool First>
void sort_pass(const SortArgs& a, bool last, cudaStream_t s) {
    launch_early(sort_count_kernel<First>, a.tiles, kThreads, 0, s, a);
    if (a.tiles > kFewTiles) launch_early(sort_scan_kernel, (a.bins + kWarps - 1) / kWarps, kThreads, 0, s, a);
    if (last) launch_early(sort_move_kernel<First, true>, a.tiles, kThreads, 0, s, a);
    else launch_early(sort_move_kernel<First, false>, a.tiles, kThreads, 0, s, a);
}

// Workspace of a gradient call, carved alike when it is counted and when it is used.
struct GradSpace {
    SumArgs sum{};
    SortArgs sort{};
    uint32_t* key[2];
    uint32_t* pos[2];
    GradSpace(const hanns_embed_bags_t* b, const SortPlan& sp, Carver& ws) {
        const size_t n = (size_t)b->n_tokens;
        sort.touched = ws.take<uint32_t>((b->rows + 31) / 32);
        sort.lengthy = ws.take<uint32_t>((b->rows + 31) / 32);
        sort.n_runs = ws.take<int32_t>(1);
        sort.most_runs = std::min<int64_t>(b->rows, b->n_tokens);
        sort.runs = ws.take<Run>(sort.most_runs);
        for (auto* k : {&key[0], &key[1], &pos[0], &pos[1]}) *k = ws.take<uint32_t>(n);
        sort.bag = ws.take<int32_t>(n);
        sort.src = ws.take<int32_t>(n);
        sort.coef = ws.take<float>(n);
        sort.hist = ws.take<int32_t>((size_t)sp.tiles << sp.bits);
        sort.total = ws.take<int32_t>((size_t)1 << sp.bits);
        sum.dim = b->dim;
        sum.n_entries = b->n_tokens;
        take_lists(sum, ws);
        sort.list_counts = sum.lists.count;
        // inner products of the weights' gradient, which needs the table
        sum.dot = ws.take<float>(b->weights && b->table ? n * most_tiles(b->dim) : 0);
    }
};

}  // namespace
}  // namespace hanns

// Declared in include/hanns_gpu.h.
extern "C" int64_t hanns_gpu_embed_bags_workspace_bytes(const hanns_embed_bags_t* b) {
    int64_t n = -1;
    hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        n = 0;
        if (!b->offsets || b->n_tokens <= kLimit) return;  // no bag can be long
        Carver ws;
        SumArgs a{};
        a.dim = b->dim;
        a.n_entries = b->n_tokens;
        take_lists(a, ws);
        n = (int64_t)ws.used;
    });
    return n;
}

extern "C" int32_t hanns_gpu_embed_bags_device(const hanns_embed_bags_t* b, void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        if (b->n_bags == 0) return;
        require(b->table && b->out && (b->tokens || b->n_tokens == 0), "embed_bags: null table, tokens or out");
        require(aligned(b->out, dtype_bytes(b->out_dtype)), "embed_bags: misaligned out");
        check_read(b->ld);
        check_written(b->n_bags, b->out_ld, b->dim);
        check_workspace((size_t)hanns_gpu_embed_bags_workspace_bytes(b), b->workspace, b->workspace_bytes);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
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
        if (b->offsets && b->n_tokens > kLimit) {
            Carver ws{static_cast<char*>(b->workspace)};
            take_lists(a, ws);
            HANNS_CUDA_OK(cudaMemsetAsync(a.lists.count, 0, 2 * sizeof(int32_t), s));
        }
        sum_bags(b->dtype, b->out_dtype, a, TokenEntries{b->tokens, b->weights, b->rows},
                 BagSegments{b->offsets, b->n_bags, b->n_tokens}, s);
    });
}

extern "C" int64_t hanns_gpu_embed_bags_grad_workspace_bytes(const hanns_embed_bags_t* b) {
    int64_t n = -1;
    hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        Carver ws;
        GradSpace(b, sort_plan(b->rows, b->n_tokens), ws);
        n = (int64_t)ws.used;
    });
    return n;
}

extern "C" int32_t hanns_gpu_embed_bags_grad_device(const hanns_embed_bags_t* b, const void* grad, int64_t grad_ld,
                                                    void* d_table, int64_t d_table_ld, float* d_weights,
                                                    void* stream) {
    return hanns::operator_entry([&] {
        using namespace hanns;
        check_bags(b);
        if (!d_table && !d_weights) return;
        require(d_table, "embed_bags: the weights' gradient comes with the table's");
        require(grad || b->n_bags == 0, "embed_bags: null gradient");
        require(b->tokens || b->n_tokens == 0, "embed_bags: null tokens");
        require(!b->mean || b->inv_counts || b->n_bags == 0, "embed_bags: a mean's gradient needs inv_counts");
        require(!d_weights || (b->table && b->weights),
                "embed_bags: the weights' gradient needs the table and the weights");
        require(aligned(grad, dtype_bytes(b->out_dtype)) && aligned(d_table, dtype_bytes(b->dtype)) &&
                    aligned(d_weights, 4),
                "embed_bags: misaligned gradient");
        check_read(grad_ld);
        if (d_weights) check_read(b->ld);
        check_written(b->rows, d_table_ld, b->dim);
        check_workspace((size_t)hanns_gpu_embed_bags_grad_workspace_bytes(b), b->workspace, b->workspace_bytes);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const SortPlan sp = sort_plan(b->rows, b->n_tokens);
        Carver ws{static_cast<char*>(b->workspace)};
        GradSpace gs(b, sp, ws);
        SortArgs& so = gs.sort;
        const int32_t n = (int32_t)b->n_tokens;
        so.bags = BagSegments{b->offsets, b->n_bags, b->n_tokens};
        so.tokens = b->tokens;
        so.weights = b->weights;
        so.inv_counts = b->mean ? b->inv_counts : nullptr;
        so.rows = b->rows;
        so.n = n;
        so.tiles = sp.tiles;
        so.scale = b->scale;
        so.bins = 1 << sp.bits;
        const unsigned by_position = (unsigned)(((int64_t)n + kThreads - 1) / kThreads);
        const uint32_t *sorted = nullptr, *position = nullptr;
        if (n == 0) {
            HANNS_CUDA_OK(cudaMemsetAsync(so.touched, 0, (b->rows + 31) / 32 * sizeof(uint32_t), s));
            HANNS_CUDA_OK(cudaMemsetAsync(so.n_runs, 0, sizeof(int32_t), s));
        } else if (n <= kSmallSort && b->rows <= kSmallRows) {
            int passes = 1;
            while (b->rows >> (passes * kSmallBits)) ++passes;  // keys 0 .. rows
            so.pos_out = gs.pos[0];
            position = so.pos_out;
            launch_early(sort_small_kernel, 1, kSmallThreads, 0, s, so, passes);
        } else {
            for (int p = 0; p < sp.passes; ++p) {
                so.shift = p * sp.bits;
                so.key_in = gs.key[p & 1];
                so.pos_in = gs.pos[p & 1];
                so.key_out = gs.key[(p + 1) & 1];
                so.pos_out = gs.pos[(p + 1) & 1];
                if (p == 0) sort_pass<true>(so, sp.passes == 1, s);
                else sort_pass<false>(so, p == sp.passes - 1, s);
            }
            sorted = gs.key[sp.passes & 1];
            position = gs.pos[sp.passes & 1];
            launch_early(sort_runs_kernel, by_position, kThreads, 0, s, so, sorted);
        }
        SumArgs& a = gs.sum;
        a.base = grad;
        a.ld = grad_ld;
        a.out = d_table;
        a.out_ld = d_table_ld;
        a.n_segments = b->rows;
        a.scale = 1.0f;
        const SortedEntries entries{so.src, so.coef, position};
        if (!d_weights || n == 0) return sum_runs<false>(b->out_dtype, b->dtype, a, entries, so, s);
        a.dot_base = b->table;
        a.dot_ld = b->ld;
        sum_runs<true>(b->out_dtype, b->dtype, a, entries, so, s);
        launch_early(weights_grad_kernel, by_position, kThreads, 0, s, a.dot, a.tiles, a.piece_tiles, so, d_weights);
    });
}
