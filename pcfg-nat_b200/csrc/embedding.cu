// Rows of the vocabulary table for tokens, times a scale, and the table's gradient.
//
// Forward: out[i] = scale * w[token_i].  One read of the rows that occur and one write; a thread moves one vector.
// Gradient: dw[v] = scale * sum of g[i] over token_i = v, summed in float32 in an order that the input alone decides:
//   1. embed_group_kernel — every tile of 1 024 positions grouped by bucket, the token modulo 128, in the positions' order.
//   2. embed_sort_kernel  — a block per bucket gathers its groups of all tiles and sorts them by token; what the tiles hold of the
//      buckets before it says where its part of the list begins, so no block waits for another.
//   3. embed_sum_kernel   — the sorted list cut into pieces of equal length.  A run of one token inside a piece is written
//      to the table at once; the part of a run that crosses a piece's border goes to scratch memory.
//   4. embed_join_kernel  — adds up the parts of every run that crosses pieces, in an order that its pieces decide.
// A placeholder that fills most positions is thus spread over as many blocks as its share of the list.
#include <algorithm>

#include "row_vectors.cuh"

namespace pcfgnat {

namespace {

constexpr int kThreads = 256;

// ---- forward

// A row by a group of `lanes` lanes (a power of two, at most a warp).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    embed_rows_kernel(const T *__restrict__ weight, int64_t w_stride, int64_t V, int H, const int64_t *__restrict__ tokens,
                      int64_t n, int lanes, float scale, T *__restrict__ out, int *status) {
    using Raw = typename RawVec<VEC * sizeof(T)>::type;
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t r = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
    if (r >= n) return;
    const int64_t t = tokens[r];
    const bool bad = t < 0 || t >= V;
    if (bad && lane == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    const float factor = bad ? CUDART_NAN_F : scale;
    const Raw *from = reinterpret_cast<const Raw *>(weight + (bad ? 0 : t) * w_stride);
    Raw *to = reinterpret_cast<Raw *>(out + r * H);
    constexpr int kLoads = VEC * sizeof(T) >= 8 ? 4 : 8;  // of a lane in flight
    const int chunks = H / VEC;
    for (int c0 = lane; c0 < chunks; c0 += kLoads * lanes) {
        Raw raw[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; j++)
            if (c0 + j * lanes < chunks) raw[j] = __ldg(from + c0 + j * lanes);
#pragma unroll
        for (int j = 0; j < kLoads; j++) {
            if (c0 + j * lanes >= chunks) break;
            float x[VEC];
            unpack_vec<T, VEC>(raw[j], x);
#pragma unroll
            for (int k = 0; k < VEC; k++) x[k] *= factor;
            to[c0 + j * lanes] = pack_vec<T, VEC>(x);
        }
    }
}

// ---- gradient

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kTile = 1024;           // positions that one block of the first kernel groups
constexpr int kBucketBits = 7, kBuckets = 1 << kBucketBits;  // a bucket: the tokens v with the same v mod 128
constexpr int kGroups = kBuckets + 1;  // of a tile: the buckets, and the token that fills much of the list
constexpr int kChunk = kSortWarps * 32;  // tiles that a block of the second kernel goes over at a time
constexpr int kCopyBlocks = 16;       // of the second kernel, for that token's entries
constexpr int kMaxRange = 1024;       // tokens of a bucket that are sorted at a time
constexpr int kFrequent = 8;          // of 32 positions that a frequent token holds
constexpr int kManyTiles = 4;         // from here on a frequent token is looked for
constexpr int kBatch = 4;             // entries of a lane in flight
constexpr int kAhead = 7;             // rows that a warp has in flight

// Rows of the table set to zero by the blocks behind the sorting ones, which wait for their loads most of the time.
__device__ void zero_table(char *dw, int64_t rows, int64_t row_bytes, int64_t stride_bytes, int64_t block, int64_t blocks) {
    const int lane = threadIdx.x & 31;
    if (stride_bytes == row_bytes) row_bytes *= rows, stride_bytes = 0, rows = 1;  // one long row
    const bool wide = !((reinterpret_cast<uintptr_t>(dw) | row_bytes | stride_bytes) & 15);
    if (rows == 1) {
        const int64_t head = wide ? 0 : min((int64_t)(-reinterpret_cast<uintptr_t>(dw) & 15), row_bytes), vecs = (row_bytes - head) / 16;
        for (int64_t i = block * blockDim.x + threadIdx.x; i < vecs; i += blocks * blockDim.x)
            reinterpret_cast<uint4 *>(dw + head)[i] = make_uint4(0, 0, 0, 0);
        if (block == 0) {
            const int64_t loose = (row_bytes - vecs * 16) / 2, i = threadIdx.x;  // in units of two bytes
            if (i < loose) *reinterpret_cast<uint16_t *>(dw + (2 * i < head ? 2 * i : 2 * i + vecs * 16)) = 0;
        }
        return;
    }
    for (int64_t r = block * (blockDim.x / 32) + (threadIdx.x >> 5); r < rows; r += blocks * (blockDim.x / 32)) {
        char *p = dw + r * stride_bytes;
        if (wide) {
            for (int64_t i = lane; i < row_bytes / 16; i += 32) reinterpret_cast<uint4 *>(p)[i] = make_uint4(0, 0, 0, 0);
        } else {
            for (int64_t i = lane; i < row_bytes / 2; i += 32) reinterpret_cast<uint16_t *>(p)[i] = 0;
        }
    }
}

struct Sorted {
    int *token, *at;     // the tokens that count and their positions, equal tokens side by side
    int *row_end;        // [V] where the list's entries of a token end
    int *total;          // entries
    int *frequent;       // a token that fills much of the list, -1 where there is none
    uint2 *grouped;      // [tile][kTile] (token / kBuckets, position) by bucket
    int *bucket_begin;   // [tile][kGroups + 1] where a bucket's entries of the tile begin, the frequent token's behind them
};

struct Zeroed {  // rows [first, last) of the table that a launch's further blocks set to zero
    char *dw;
    int64_t first, last, row_bytes, stride_bytes;
    __device__ __forceinline__ void run(int block, int blocks) const {
        zero_table(dw + first * stride_bytes, last - first, row_bytes, stride_bytes, block, blocks);
    }
};

// The positions of a tile grouped by bucket, in their order within one.  A token that a quarter of 32 positions spread over the list
// hold (every block looks at the same) is left out of its bucket, which would be sorted by one SM while the others wait, and only
// copied by several: 28 980 tokens, half of them one, added onto a table of 512 float32 columns in 24.0 us; 36.2 while it was sorted.
__global__ void __launch_bounds__(kTile, 2)
    embed_group_kernel(const int64_t *__restrict__ tokens, int n, int V, uint32_t padding, int tiles, Sorted sorted, Zeroed zeroed,
                       int *status) {
    constexpr int kCells = (kGroups + 31) / 32 * 32;
    __shared__ int cell[kTile / 32][kCells];
    __shared__ int begin[kCells], warp_sum[kCells / 32];
    __shared__ uint32_t chosen;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the next kernel waits for this one's end all the same
    if ((int)blockIdx.x >= tiles) {
        zeroed.run(blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t i = (int64_t)blockIdx.x * kTile + tid;
    const uint2 t = i < n ? reinterpret_cast<const uint2 *>(tokens)[i] : make_uint2(padding, 0);
    uint32_t frequent = 0xffffffffu;
    if (tiles >= kManyTiles) {
        if (warp == 0) {
            uint2 sample = reinterpret_cast<const uint2 *>(tokens)[(int64_t)lane * n >> 5];
            if (sample.y != 0 || sample.x >= (uint32_t)V || sample.x == padding) sample.x = 0xffffffffu;
            const int held = __popc(__match_any_sync(0xffffffffu, sample.x));
            const int most = __reduce_max_sync(0xffffffffu, sample.x == 0xffffffffu ? 0 : held * 32 + lane);
            if (most >= kFrequent * 32) frequent = __shfl_sync(0xffffffffu, sample.x, most & 31);
            if (lane == 0) chosen = frequent;
        }
        __syncthreads();
        frequent = chosen;
    }
    if (blockIdx.x == 0 && tid == 0) *sorted.frequent = (int)frequent;
    const bool inside = t.y == 0 && t.x < (uint32_t)V, counts = inside && t.x != padding;
    if (i < n && !inside) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    const int bucket = t.x == frequent ? kBuckets : t.x & (kBuckets - 1);
    uint32_t same = __ballot_sync(0xffffffffu, counts);  // the lanes with the same bucket
#pragma unroll
    for (int k = 0; k <= kBucketBits; k++) {
        const uint32_t set = __ballot_sync(0xffffffffu, bucket >> k & 1);
        same &= bucket >> k & 1 ? set : ~set;
    }
#pragma unroll
    for (int k = 0; k < kCells / 32; k++) cell[warp][k * 32 + lane] = 0;
    __syncwarp();
    const int rank = __popc(same & ((1u << lane) - 1));
    if (counts && rank == 0) cell[warp][bucket] = __popc(same);
    __syncthreads();
    if (tid < kCells) {
        int held[kTile / 32], sum = 0;
#pragma unroll
        for (int w = 0; w < kTile / 32; w++) held[w] = cell[w][tid];
#pragma unroll
        for (int w = 0; w < kTile / 32; w++) cell[w][tid] = sum, sum += held[w];
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += x;
        }
        if (lane == 31) warp_sum[warp] = scan;
        begin[tid] = scan - sum;
    }
    __syncthreads();
    if (tid < kCells) {
        int before = begin[tid];
        for (int w = 0; w < warp; w++) before += warp_sum[w];
        begin[tid] = before;
        if (tid <= kGroups) sorted.bucket_begin[(int64_t)blockIdx.x * (kGroups + 1) + tid] = before;
    }
    __syncthreads();
    if (counts)
        sorted.grouped[(int64_t)blockIdx.x * kTile + begin[bucket] + cell[warp][bucket] + rank] = make_uint2(t.x >> kBucketBits, (uint32_t)i);
}

// The tiles that one warp goes over of up to 1 024: side by side, at most 32; where there are fewer tiles than warps, warps share one.
struct Share {
    int tile0, tiles, part, parts_log;
    __device__ __forceinline__ Share(int chunk, int there, int warp) {
        const int each = (there + kSortWarps - 1) / kSortWarps;
        parts_log = there > 1 ? max(0, __clz(there - 1) - __clz(kSortWarps - 1)) : 31 - __clz(kSortWarps);
        part = warp & ((1 << parts_log) - 1);
        const int first = min((warp >> parts_log) * each, there);
        tile0 = chunk + first, tiles = min(each, there - first);
    }
};

// The entries of a bucket in them, at most one tile per lane, numbered through.
struct Span {
    int begin, count, shift;  // of the lane's tile: its first number, its entries, and from a number to the place in the tiles' list
    int n, tile0, tiles;
    __device__ __forceinline__ Span(const Sorted &s, int bucket, const Share &share, int lane) : tile0(share.tile0), tiles(share.tiles) {
        int from = 0;
        count = 0;
        if (lane < tiles) {
            const int *b = s.bucket_begin + (int64_t)(tile0 + lane) * (kGroups + 1) + bucket;
            from = b[0], count = b[1] - from;
        }
        const int first = count * share.part >> share.parts_log;
        count = (count * (share.part + 1) >> share.parts_log) - first;
        from += first;
        begin = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, begin, o);
            if (lane >= o) begin += x;
        }
        n = __shfl_sync(0xffffffffu, begin, 31);
        begin -= count;
        shift = lane * kTile + from - begin;
    }
    // Entry e of them; e may differ from lane to lane, but all lanes call.
    __device__ __forceinline__ uint2 entry(const Sorted &s, int e, uint2 none) const {
        int of = 0;
        if (tiles > 1) {
#pragma unroll
            for (int step = 16; step > 0; step /= 2)
                if (__shfl_sync(0xffffffffu, begin, of + step) <= e) of += step;
        }
        const int at = __shfl_sync(0xffffffffu, shift, of) + e;
        return e < n ? s.grouped[(int64_t)tile0 * kTile + at] : none;
    }
};

// The frequent token's entries behind all others, by one of several blocks, each for tiles that lie side by side.
__device__ void copy_frequent(const Sorted &s, int tiles, int block, int *base, int *all) {
    const int tid = threadIdx.x, lane = tid & 31;
    const int each = (tiles + kCopyBlocks - 1) / kCopyBlocks, first = min(block * each, tiles), last = min(first + each, tiles);
    const auto range_of = [&](int tile) { return s.bucket_begin + (int64_t)tile * (kGroups + 1) + kBuckets; };
    if (tid == 0) *all = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int before = 0, sum = 0;
    for (int t = tid; t < tiles; t += kSortThreads) {
        const int *r = range_of(t);
        before += t < first ? r[1] : r[0], sum += r[1];
    }
    before = __reduce_add_sync(0xffffffffu, before), sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0 && sum) atomicAdd(base, before), atomicAdd(all, sum);
    __syncthreads();
    const int token = *s.frequent;
    if (block == 0 && tid == 0) {
        *s.total = *all;
        if (token >= 0) s.row_end[token] = *all;
    }
    if (token < 0) return;
    int place = *base;
    for (int t0 = first; t0 < last; t0 += 32) {
        int from = 0, count = 0;
        if (t0 + lane < last) {
            const int *r = range_of(t0 + lane);
            from = r[0], count = r[1] - r[0];
        }
#pragma unroll 4
        for (int j = 0; j < min(32, last - t0); j++) {
            const int entries = __shfl_sync(0xffffffffu, count, j), at = __shfl_sync(0xffffffffu, from, j) + tid;
            if (tid < entries) s.token[place + tid] = token, s.at[place + tid] = (int)s.grouped[(int64_t)(t0 + j) * kTile + at].y;
            place += entries;
        }
    }
}

// A block sorts a bucket by token: counted per warp and token, numbered, placed.  There are fewer buckets than SMs, so
// that a second block per SM would only take registers away: forward and backward of 14 400 tokens on a table of 41 MB
// took 37.6 us in all with two blocks per SM, 35.1 with one.
__global__ void __launch_bounds__(kSortThreads, 1)
    embed_sort_kernel(int V, int tiles, int range, Sorted sorted, Zeroed zeroed) {
    extern __shared__ int cell[];  // [warp][token of the bucket]: entries of the warp's span, then where the next one goes
    __shared__ int warp_sum[kSortWarps], base;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x >= kBuckets + kCopyBlocks) {
        zeroed.run(blockIdx.x - (kBuckets + kCopyBlocks), gridDim.x - (kBuckets + kCopyBlocks));
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bucket = blockIdx.x;
    const Share share(0, min(kChunk, tiles), warp);
    if (tid == 0) base = 0;
    if (blockIdx.x >= kBuckets) {
        copy_frequent(sorted, tiles, blockIdx.x - kBuckets, &base, warp_sum);
        return;
    }
    for (int i = tid; i < kSortWarps * range; i += kSortThreads) cell[i] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int frequent = *sorted.frequent;
    const int tokens = (V - bucket + kBuckets - 1) >> kBucketBits;  // of the bucket (0 where V is smaller than its number)
    const uint2 none = make_uint2(0xffffffffu, 0);
    // The first entries stay in registers from the count to the placing; lists of more than 1 024 tiles are gone over by as many at a time.
    const Span head(sorted, bucket, share, lane);
    uint2 ahead[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; k++) ahead[k] = head.entry(sorted, k * 32 + lane, none);
    const auto rest = [&](const Span &span, int g0, auto visit) {
        for (; g0 < span.n; g0 += 32 * kBatch) {
            uint2 entry[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++) entry[k] = span.entry(sorted, g0 + k * 32 + lane, none);
#pragma unroll
            for (int k = 0; k < kBatch; k++)
                if (g0 + k * 32 < span.n) visit(entry[k]);
        }
    };
    const auto over = [&](auto visit) {
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (k * 32 < head.n) visit(ahead[k]);
        rest(head, 32 * kBatch, visit);
        for (int chunk = kChunk; chunk < tiles; chunk += kChunk)
            rest(Span(sorted, bucket, Share(chunk, min(kChunk, tiles - chunk), warp), lane), 0, visit);
    };
    int below = 0;  // what the tiles hold of the buckets before this one
    for (int t = tid; t < tiles; t += kSortThreads) below += sorted.bucket_begin[(int64_t)t * (kGroups + 1) + bucket];
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0 && below) atomicAdd(&base, below);
    int *mine = cell + warp * range;
    int begin_of_window = 0;
    for (int r0 = 0; r0 < tokens || r0 == 0; r0 += range) {  // most tables: one window of the bucket's tokens
        const int rows = min(range, tokens - r0);
        if (r0) {
            for (int i = tid; i < kSortWarps * range; i += kSortThreads) cell[i] = 0;
            __syncthreads();
        }
        const auto row_of = [&](uint2 entry) {  // of the window, -1 where it is of none
            const int row = (int)entry.x - r0;
            return entry.x != none.x && row >= 0 && row < rows ? row : -1;
        };
        over([&](uint2 entry) {
            const int row = row_of(entry);
            const uint32_t in = __ballot_sync(0xffffffffu, row >= 0);
            const int one = __shfl_sync(0xffffffffu, row, __ffs(in) - 1);
            const uint32_t same = __ballot_sync(0xffffffffu, row == one);  // a frequent token fills whole groups
            if (row >= 0 && (row != one || lane == __ffs(in) - 1)) atomicAdd(mine + row, row == one ? __popc(same) : 1);
        });
        __syncthreads();
        if (r0 == 0) begin_of_window = base;
        // where every token begins, and within it every warp
        int held[kSortWarps], sum = 0;
        if (tid < rows)
#pragma unroll
            for (int w = 0; w < kSortWarps; w++) held[w] = cell[w * range + tid], sum += held[w];
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += x;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        int next = begin_of_window + scan - sum + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
        if (tid < rows) {
#pragma unroll
            for (int w = 0; w < kSortWarps; w++) cell[w * range + tid] = next, next += held[w];
            const int token = ((r0 + tid) << kBucketBits) + bucket;
            if (token != frequent) sorted.row_end[token] = next;
        }
        begin_of_window += __reduce_add_sync(0xffffffffu, warp_sum[lane]);
        __syncthreads();
        over([&](uint2 entry) {
            const int row = row_of(entry);
            const uint32_t in = __ballot_sync(0xffffffffu, row >= 0);
            if (!in) return;
            const int one = __shfl_sync(0xffffffffu, row, __ffs(in) - 1);
            uint32_t same = __ballot_sync(0xffffffffu, row == one);  // a frequent token fills whole groups
            if (same != in) same = __match_any_sync(0xffffffffu, row);
            int from = 0;
            if (row >= 0) from = mine[row];
            __syncwarp();
            if (row >= 0) {
                const int rank = __popc(same & ((1u << lane) - 1)), at = from + rank;
                if (rank == 0) mine[row] = from + __popc(same);
                sorted.token[at] = ((row + r0) << kBucketBits) + bucket, sorted.at[at] = (int)entry.y;
            }
            __syncwarp();
        });
        __syncthreads();
    }
}

// A finished sum into the table.  Every number of the table gets at most one sum per call, so adding to a float32 table by a
// reduction (which needs not wait for what is there) has one order only.  A reduction takes operands and results below the least normal
// number, 2^-126, for 0.  Reading, adding and writing instead, which keeps them, takes 36.7 us where 28 980 halves of 512 columns take 31.3 by
// reductions (four tables in turn, so that none is in L2), 68 where 60 000 take 49; with the table's row read ahead 35.5 and 58.
template <typename T, int VEC>
__device__ __forceinline__ void write_row(T *p, const float (&acc)[VEC], float scale, int accumulate) {
    if constexpr (sizeof(T) == 4) {
        if (accumulate) {
            if constexpr (VEC % 4 == 0) {
#pragma unroll
                for (int k = 0; k < VEC; k += 4)
                    atomicAdd(reinterpret_cast<float4 *>(p + k),
                              make_float4(acc[k] * scale, acc[k + 1] * scale, acc[k + 2] * scale, acc[k + 3] * scale));
            } else {
#pragma unroll
                for (int k = 0; k < VEC; k++) atomicAdd(p + k, acc[k] * scale);
            }
            return;
        }
    }
    constexpr int kStep = VEC * sizeof(T) > 16 ? 16 / sizeof(T) : VEC;  // numbers of one store
    using Raw = typename RawVec<kStep * sizeof(T)>::type;
#pragma unroll
    for (int j = 0; j < VEC; j += kStep) {
        float x[kStep] = {};
        if (accumulate) unpack_vec<T, kStep>(*reinterpret_cast<const Raw *>(p + j), x);
#pragma unroll
        for (int k = 0; k < kStep; k++) x[k] += acc[j + k] * scale;
        *reinterpret_cast<Raw *>(p + j) = pack_vec<T, kStep>(x);
    }
}

constexpr int kSumWarps = 8;

struct Pieces {
    Sorted sorted;
    float *parts;  // [piece][2][H]: what a piece holds of a run that began before it, and of one that goes on behind it
    int length;    // entries of a warp, kSumWarps warps to a piece
};

// Columns of a block: 512 bytes of a gradient's row.
template <typename G>
constexpr int kColumns = 512 / (int)sizeof(G);

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(to)), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_address(to)), "l"(from) : "memory");
}

// A tile's columns of a gradient's row into shared memory, by a warp.  ALIGNED: in 16-byte vectors, all of them there.
template <typename G, bool ALIGNED>
__device__ __forceinline__ void stage_row(G *to, const G *from, int columns, int lane) {
    if constexpr (ALIGNED) {
        constexpr int kVec = 16 / sizeof(G);
        if (lane * kVec < columns) copy_async<16>(to + lane * kVec, from + lane * kVec);
    } else {
#pragma unroll
        for (int k = 0; k < kColumns<G> / 32; k++) {
            const int c = k * 32 + lane;
            if (c >= columns) continue;
            if constexpr (sizeof(G) == 4) copy_async<4>(to + c, from + c);
            else to[c] = from[c];
        }
    }
}

// A block adds up a piece of the list for a tile of columns, a warp an equal share of it: seven rows on their way to shared memory
// while one is added.  A warp's runs that cross its borders are joined in shared memory, in the list's order, and so are given on only
// where they cross the piece's.  A lane's columns lie side by side where rows of table and gradient allow vectors, else 32 apart.
template <typename G, typename W, bool ALIGNED>
__global__ void __launch_bounds__(32 * kSumWarps)
    embed_sum_kernel(const G *__restrict__ grad, int64_t g_stride, int H, Pieces p, W *dw, int64_t dw_stride, float scale,
                     int accumulate) {
    constexpr int kCols = kColumns<G>, kMine = kCols / 32;
    constexpr int kUnit = 16 / sizeof(W) < kMine ? 16 / sizeof(W) : kMine;  // columns side by side: one store of the table's type
    const auto column = [](int k, int lane) { return ALIGNED ? k / kUnit * (32 * kUnit) + lane * kUnit + k % kUnit : k * 32 + lane; };
    __shared__ __align__(16) G staged[kSumWarps][kAhead][kCols];
    __shared__ float crossing[kSumWarps][2][kCols];
    __shared__ int4 ends[kSumWarps];  // of a warp's share: first and last token, whether those runs go on before and behind it
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.y * kCols, columns = H - tile;
    const int total = *p.sorted.total;
    const int64_t begin64 = ((int64_t)blockIdx.x * kSumWarps + warp) * p.length;
    const int *token = p.sorted.token;
    if ((int64_t)blockIdx.x * kSumWarps * p.length >= total) return;
    if (begin64 < total) {
        const int begin = (int)begin64, end = min(begin + p.length, total);
        const int before = begin > 0 ? token[begin - 1] : -1, after = end < total ? token[end] : -1;
        int my_token = begin + lane < end ? token[begin + lane] : -1, my_at = begin + lane < end ? p.sorted.at[begin + lane] : 0;
        int run = __shfl_sync(0xffffffffu, my_token, 0);
        bool began_before = run == before;
        if (lane == 0) ends[warp].x = run, ends[warp].z = run == before;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int at = __shfl_sync(0xffffffffu, my_at, j);
            if (begin + j < end) stage_row<G, ALIGNED>(staged[warp][j], grad + at * g_stride + tile, columns, lane);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        float acc[kMine] = {};
        int slot = 0;
        int ahead_at = my_at;  // positions of the 32 entries that hold the one kAhead further on
        int ahead_base = begin;
#pragma unroll 1
        for (int i = begin; i < end; i++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
            __syncwarp();
            const G *row = staged[warp][slot];
            if constexpr (ALIGNED) {
#pragma unroll
                for (int k = 0; k < kMine; k += kUnit) {
                    float x[kUnit];
                    unpack_vec<G, kUnit>(*reinterpret_cast<const typename RawVec<kUnit * sizeof(G)>::type *>(row + column(k, lane)), x);
#pragma unroll
                    for (int q = 0; q < kUnit; q++) acc[k + q] += x[q];
                }
            } else {
#pragma unroll
                for (int k = 0; k < kMine; k++) acc[k] += num_to_float<G>(row[column(k, lane)]);
            }
            __syncwarp();  // the row has been read
            const int ahead = i + kAhead;
            if (ahead - ahead_base >= 32) {
                ahead_base += 32;
                ahead_at = ahead_base + lane < end ? p.sorted.at[ahead_base + lane] : 0;
            }
            const int at = __shfl_sync(0xffffffffu, ahead_at, ahead - ahead_base);
            if (ahead < end) stage_row<G, ALIGNED>(staged[warp][slot], grad + at * g_stride + tile, columns, lane);
            asm volatile("cp.async.commit_group;" ::: "memory");
            slot = slot + 1 == kAhead ? 0 : slot + 1;
            // the next entry's token
            int next = -1;
            if ((i + 1 - begin) % 32 == 0) my_token = i + 1 + lane < end ? token[i + 1 + lane] : -1;
            next = __shfl_sync(0xffffffffu, my_token, (i + 1 - begin) & 31);
            if (i + 1 == end) next = -1;
            if (next == run) continue;
            const bool goes_on = next < 0 && run == after;
            if (began_before || goes_on) {
                float *to = crossing[warp][began_before ? 0 : 1];
#pragma unroll
                for (int k = 0; k < kMine; k++) to[column(k, lane)] = acc[k];
            } else {
                constexpr int kStore = ALIGNED ? kUnit : 1;
#pragma unroll
                for (int k = 0; k < kMine; k += kStore) {
                    float x[kStore];
#pragma unroll
                    for (int q = 0; q < kStore; q++) x[q] = acc[k + q];
                    if (column(k, lane) < columns) write_row<W, kStore>(dw + run * dw_stride + tile + column(k, lane), x, scale, accumulate);
                }
            }
#pragma unroll
            for (int k = 0; k < kMine; k++) acc[k] = 0.f;
            if (next < 0 && lane == 0) ends[warp].y = run, ends[warp].w = run == after;
            run = next;
            began_before = false;
        }
    }
    __syncthreads();
    // a thread per column: what the warps left, in the list's order
    const int col = threadIdx.x, cc = tile + col;
    if (col < kCols && cc < H) {
        float *give = p.parts + (int64_t)blockIdx.x * 2 * H + cc;
        float acc[1] = {0.f};
        bool from_outside = false, open = false;
        for (int w = 0; w < kSumWarps; w++) {
            if (((int64_t)blockIdx.x * kSumWarps + w) * p.length >= total) break;
            const int head = ends[w].x, tail = ends[w].y;
            const bool before = ends[w].z, behind = ends[w].w;
            if (before) {
                if (w == 0) from_outside = true;
                acc[0] += crossing[w][0][col];
                open = head == tail && behind;
                if (!open) {
                    if (from_outside) give[0] = acc[0];
                    else write_row<W, 1>(dw + head * dw_stride + cc, acc, scale, accumulate);
                    acc[0] = 0.f;
                    from_outside = false;
                }
            }
            if (behind && !(before && head == tail)) acc[0] = crossing[w][1][col], open = true;
        }
        if (open) give[from_outside ? 0 : H] = acc[0];
    }
}

constexpr int kJoinGroups = 16, kJoinColumns = 128;

// The runs that cross pieces: the first part and those of the pieces behind it, sixteen warps taking every sixteenth piece, a
// lane four columns.  Most blocks only find that no run begins in theirs, so they load all that tells it at once.  With eight warps
// 28 980 tokens, half of them one, take 26.1 us in all instead of 23.9; with a warp per piece 23.9, but 32 768 of 301 columns 49.4, not 45.3.
template <typename W>
__global__ void __launch_bounds__(32 * kJoinGroups)
    embed_join_kernel(int H, Pieces p, W *dw, int64_t dw_stride, float scale, int accumulate) {
    __shared__ float sums[kJoinGroups][kJoinColumns];
    chain_begin();
    if (blockIdx.x + 1 == gridDim.x) return;  // nothing behind the last piece
    const int length = p.length * kSumWarps, begin = blockIdx.x * length, end = begin + length;
    const int total = *p.sorted.total;
    const int token = p.sorted.token[end - 1], behind = p.sorted.token[end], before = begin > 0 ? p.sorted.token[begin - 1] : -1;
    if (end >= total || behind != token || before == token) return;
    const int last = (p.sorted.row_end[token] - 1) / length;  // the piece in which the run ends
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, tile = blockIdx.y * kJoinColumns;
    float acc[4] = {};
    const auto add = [&](int64_t piece, int which) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int c = tile + k * 32 + lane;
            if (c < H) acc[k] += p.parts[(piece * 2 + which) * H + c];
        }
    };
    if (group == 0) add(blockIdx.x, 1);
#pragma unroll 4
    for (int q = (int)blockIdx.x + 1 + group; q <= last; q += kJoinGroups) add(q, 0);
#pragma unroll
    for (int k = 0; k < 4; k++) sums[group][k * 32 + lane] = acc[k];
    __syncthreads();
    const int col = threadIdx.x, c = tile + col;
    if (col < kJoinColumns && c < H) {
        float sum[1] = {0.f};
#pragma unroll
        for (int g = 0; g < kJoinGroups; g++) sum[0] += sums[g][col];
        write_row<W, 1>(dw + token * dw_stride + c, sum, scale, accumulate);
    }
}

constexpr int kFew = 256;  // positions that one launch without a sorted list takes

// Few positions: a block owns every so many-th row of the table, sets its rows to zero, and looks through all positions for its
// tokens.  The rows of one token are summed by groups of `across` threads, which hold the columns; every group takes every so
// many-th row, and the groups' sums are added in their order.
template <typename G, typename W, int VEC>
__global__ void __launch_bounds__(kThreads)
    embed_few_kernel(const G *__restrict__ grad, int64_t g_stride, int H, int across, const int64_t *__restrict__ tokens, int n,
                     int64_t V, uint32_t padding, W *dw, int64_t dw_stride, float scale, int accumulate, int *status) {
    using Raw = typename RawVec<VEC * sizeof(G)>::type;
    constexpr int kWarps = kThreads / 32;
    __shared__ __align__(16) uint32_t token[kFew];
    __shared__ int at[kFew], same_at[kFew], count_of[kWarps];
    __shared__ float sums[kThreads * VEC];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // places for the threads that have something, in the threads' order, behind the `used` ones; has barriers
    const auto place = [&](bool has, int &used) {
        const uint32_t mask = __ballot_sync(0xffffffffu, has);
        if (lane == 0) count_of[warp] = __popc(mask);
        __syncthreads();
        int to = used + __popc(mask & ((1u << lane) - 1));
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) to += count_of[w];
            used += count_of[w];
        }
        __syncthreads();
        return to;
    };
    if (!accumulate) {
        const int64_t row_bytes = (int64_t)H * sizeof(W);
        const bool wide = !((reinterpret_cast<uintptr_t>(dw) | row_bytes | (dw_stride * sizeof(W))) & 15);
        for (int64_t r = blockIdx.x + (int64_t)warp * gridDim.x; r < V; r += (int64_t)kWarps * gridDim.x) {
            W *row = dw + r * dw_stride;
            if (wide) {
                for (int64_t i = lane; i < row_bytes / 16; i += 32) reinterpret_cast<uint4 *>(row)[i] = make_uint4(0, 0, 0, 0);
            } else {
                for (int c = lane; c < H; c += 32) row[c] = num_from_float<W>(0.f);
            }
        }
    }
    int mine = 0;  // positions with a token of this block
    for (int i0 = 0; i0 < n; i0 += kThreads) {
        const int i = i0 + tid;
        const uint2 t = i < n ? reinterpret_cast<const uint2 *>(tokens)[i] : make_uint2(padding, 0);
        const bool inside = t.y == 0 && t.x < (uint32_t)V;
        if (i < n && !inside && blockIdx.x == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
        const bool has = inside && t.x != padding && t.x % gridDim.x == blockIdx.x;
        const int to = place(has, mine);
        if (has) token[to] = t.x, at[to] = i;
    }
    __syncthreads();
    const int group = tid / across, groups = kThreads / across, chunks = H / VEC;
    for (int e = 0; e < mine;) {
        const uint4 four = reinterpret_cast<const uint4 *>(token)[e / 4];
        const uint32_t left[4] = {four.x, four.y, four.z, four.w};
        uint32_t v = 0xffffffffu;  // the next token that has not been summed; the same for the whole block
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (v == 0xffffffffu && e / 4 * 4 + k >= e && e / 4 * 4 + k < mine) v = left[k];
        if (v == 0xffffffffu) {
            e = e / 4 * 4 + 4;
            continue;
        }
        __syncthreads();
        int found = 0;
        for (int j0 = e; j0 < mine; j0 += kThreads) {
            const int j = j0 + tid;
            const bool same = j < mine && token[j] == v;
            const int to = place(same, found);
            if (same) same_at[to] = at[j], token[j] = 0xffffffffu;
        }
        __syncthreads();
        for (int c0 = 0; c0 < chunks; c0 += across) {
            const int c = c0 + tid % across;
            float acc[VEC] = {};
            if (c < chunks) {
                for (int k0 = group; k0 < found; k0 += 8 * groups) {  // eight rows in flight
                    Raw raw[8];
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k0 + k * groups < found)
                            raw[k] = __ldg(reinterpret_cast<const Raw *>(grad + same_at[k0 + k * groups] * g_stride) + c);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        if (k0 + k * groups >= found) break;
                        float x[VEC];
                        unpack_vec<G, VEC>(raw[k], x);
#pragma unroll
                        for (int q = 0; q < VEC; q++) acc[q] += x[q];
                    }
                }
            }
            if (groups > 1) {
#pragma unroll
                for (int q = 0; q < VEC; q++) sums[q * kThreads + tid] = acc[q];
                __syncthreads();
                if (group == 0)
                    for (int other = 1; other < groups; other++)
#pragma unroll
                        for (int q = 0; q < VEC; q++) acc[q] += sums[q * kThreads + other * across + tid];
                __syncthreads();
            }
            if (group == 0 && c < chunks) write_row<W, VEC>(dw + v * dw_stride + c * VEC, acc, scale, accumulate);
        }
    }
}

int widest(uintptr_t bits, int size) {  // bytes of the widest vector that addresses and strides allow, at least an element's
    for (int b = 16; b > size; b /= 2)
        if (!(bits & (uintptr_t)(b - 1))) return b;
    return size;
}

// Entries of a warp, for at most PCFGNAT_MAX_INDEX positions 131 008: a share's begin and its length, and the rows staged ahead, add up
// to less than 2^31.  The more of a short list's blocks there are, the more SMs add to the table; fewer and longer pieces leave less
// to join.  Added onto 512 float32 columns with 2, 4, 8 and 16 entries: 1 500 tokens 14.0, 15.9, 18.2 us, 5 000 15.4, 16.5, 20.3, 27.0,
// 10 000 19.9, 18.1, 20.8, 27.0, 20 000 29.6, 23.5, 22.2, 28.7, 60 000 56.3, 56.3, 47.8, 43.5.  More where that made over 2 048 pieces.
int warp_entries(int64_t n) {
    int share = 2;
    while (share < 16 && share * 4096 < n) share *= 2;
    const int64_t even = (n + 2048 * kSumWarps - 1) / (2048 * kSumWarps);
    return even <= share ? share : (int)((even + 7) / 8 * 8);
}
int64_t piece_count(int64_t n) {
    const int64_t length = (int64_t)warp_entries(n) * kSumWarps;
    return (n + length - 1) / length;
}

struct Scratch {
    Sorted sorted;
    float *parts;
    size_t bytes;
    Scratch(char *at, int64_t n, int64_t V, int H) {
        bytes = 0;
        const auto take = [&](size_t size) {
            char *p = at + bytes;
            bytes += (size + 15) / 16 * 16;
            return p;
        };
        const size_t tiles = (size_t)((n + kTile - 1) / kTile);
        sorted.total = reinterpret_cast<int *>(take(sizeof(int)));
        sorted.frequent = reinterpret_cast<int *>(take(sizeof(int)));
        sorted.token = reinterpret_cast<int *>(take((size_t)n * sizeof(int)));
        sorted.at = reinterpret_cast<int *>(take((size_t)n * sizeof(int)));
        sorted.row_end = reinterpret_cast<int *>(take((size_t)V * sizeof(int)));
        sorted.grouped = reinterpret_cast<uint2 *>(take(tiles * kTile * sizeof(uint2)));
        sorted.bucket_begin = reinterpret_cast<int *>(take(tiles * (kGroups + 1) * sizeof(int)));
        parts = reinterpret_cast<float *>(take((size_t)piece_count(n) * 2 * H * sizeof(float)));
    }
};

}  // namespace

size_t embed_workspace_bytes(int64_t n, int64_t V, int H) { return n <= kFew ? 0 : Scratch(nullptr, n, V, H).bytes; }

int launch_embed(const void *weight, int dtype, int64_t w_stride, int64_t V, int H, const int64_t *tokens, int64_t n, float scale,
                 void *out, int *status, cudaStream_t st) {
    if (n == 0) return PCFGNAT_OK;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const uintptr_t bits = reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out) |
                               (uintptr_t)(w_stride * sizeof(T)) | (uintptr_t)(H * sizeof(T));
        const auto run = [&](auto vec) {
            constexpr int VEC = decltype(vec)::value;
            int lanes = 1;
            while (lanes < 32 && lanes < H / VEC) lanes *= 2;
            const int64_t blocks = (n * lanes + kThreads - 1) / kThreads;
            if (blocks > INT32_MAX) return (int)PCFGNAT_ERR_TOO_LARGE;
            embed_rows_kernel<T, VEC><<<(unsigned)blocks, kThreads, 0, st>>>(static_cast<const T *>(weight), w_stride, V, H, tokens, n,
                                                                             lanes, scale, static_cast<T *>(out), status);
            return cuda_rc(cudaGetLastError());
        };
        switch (widest(bits, sizeof(T))) {
            case 16: return run(std::integral_constant<int, 16 / sizeof(T)>());
            case 8: return run(std::integral_constant<int, 8 / sizeof(T)>());
            case 4: return run(std::integral_constant<int, 4 / sizeof(T)>());
            default: return run(std::integral_constant<int, 1>());
        }
    });
}

int launch_embed_backward(const void *grad, int dtype, int64_t g_stride, const int64_t *tokens, int64_t n, int64_t V, int H, float scale,
                          int has_padding, int64_t padding, void *dw, int dw_dtype, int64_t dw_stride, int accumulate, void *workspace,
                          int *status, cudaStream_t st) {
    const uint32_t skip = has_padding && padding >= 0 && padding < V ? (uint32_t)padding : 0xffffffffu;
    const auto bits = [&](const void *a, int64_t stride, int64_t size) {  // of a matrix with H numbers of that size in a row
        return reinterpret_cast<uintptr_t>(a) | (uintptr_t)(stride * size) | (uintptr_t)(H * size);
    };
    // Up to 256 positions one launch.  Added onto a float32 table of 512 columns: 20, 140 and 256 positions 3.2, 5.5 and 6.6 us (11.7
    // where one token fills 70 % of 256); 257 by the sorted list 11.6 (12.7).
    if (n <= kFew)
        return with_dtype(dtype, [&](auto g) {
            using G = decltype(g);
            const auto run = [&](auto w) {
                using W = decltype(w);
                const bool aligned = widest(bits(grad, g_stride, sizeof(G)), sizeof(G)) == 16 && widest(bits(dw, dw_stride, sizeof(W)), sizeof(W)) == 16;
                const auto few = [&](auto vec) {
                    constexpr int VEC = decltype(vec)::value;
                    int across = 32;
                    while (across < kThreads && across < H / VEC) across *= 2;
                    embed_few_kernel<G, W, VEC><<<2 * (unsigned)sm_count(), kThreads, 0, st>>>(
                        static_cast<const G *>(grad), g_stride, H, across, tokens, (int)n, V, skip, static_cast<W *>(dw), dw_stride, scale,
                        accumulate, status);
                    return cuda_rc(cudaGetLastError());
                };
                return aligned ? few(std::integral_constant<int, 16 / sizeof(G)>()) : few(std::integral_constant<int, 1>());
            };
            return dw_dtype == PCFGNAT_DTYPE_F32 ? run(float()) : run(g);
        });
    const Scratch scratch(static_cast<char *>(workspace), n, V, H);
    const Sorted &sorted = scratch.sorted;
    const int64_t dw_size = dw_dtype == PCFGNAT_DTYPE_F32 ? 4 : 2;
    const int tiles = (int)((n + kTile - 1) / kTile), zeroing = accumulate ? 0 : sm_count();
    const int range = (int)std::min<int64_t>(kMaxRange, (V + kBuckets - 1) / kBuckets);
    const size_t smem = (size_t)kSortWarps * range * sizeof(int);
    cudaError_t e = ensure_dynamic_smem(embed_sort_kernel, smem);
    if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    // the table is set to zero beside the sorting, a third of it beside the first, shorter kernel
    const int64_t third = V / 3;
    const Zeroed first{static_cast<char *>(dw), 0, third, H * dw_size, dw_stride * dw_size};
    const Zeroed rest{static_cast<char *>(dw), third, V, H * dw_size, dw_stride * dw_size};
    embed_group_kernel<<<(unsigned)(tiles + zeroing), kTile, 0, st>>>(tokens, (int)n, (int)V, skip, tiles, sorted, first, status);
    e = cudaGetLastError();
    if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    // every further kernel waits for the one before it to end, but may be scheduled before that
    const auto launch = [&](auto kernel, dim3 grid, unsigned threads, size_t bytes, auto... args) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = bytes;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, args...);
    };
    e = launch(embed_sort_kernel, dim3(kBuckets + kCopyBlocks + zeroing), kSortThreads, smem, (int)V, tiles, range, sorted, rest);
    if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    const Pieces p{sorted, scratch.parts, warp_entries(n)};
    const unsigned pieces = (unsigned)piece_count(n);
    return with_dtype(dtype, [&](auto g) {
        using G = decltype(g);
        const auto run = [&](auto w) {
            using W = decltype(w);
            const bool aligned = widest(bits(grad, g_stride, sizeof(G)), sizeof(G)) == 16 && widest(bits(dw, dw_stride, sizeof(W)), sizeof(W)) == 16;
            const dim3 grid(pieces, (unsigned)((H + kColumns<G> - 1) / kColumns<G>));
            const auto sum = [&](auto kernel) {
                return launch(kernel, grid, 32 * kSumWarps, 0, static_cast<const G *>(grad), g_stride, H, p, static_cast<W *>(dw),
                              dw_stride, scale, accumulate);
            };
            cudaError_t rc = aligned ? sum(embed_sum_kernel<G, W, true>) : sum(embed_sum_kernel<G, W, false>);
            if (rc == cudaSuccess)
                rc = launch(embed_join_kernel<W>, dim3(pieces, (unsigned)((H + kJoinColumns - 1) / kJoinColumns)), 32 * kJoinGroups, 0, H, p,
                            static_cast<W *>(dw), dw_stride, scale, accumulate);
            return rc == cudaSuccess ? (int)PCFGNAT_OK : (int)PCFGNAT_ERR_CUDA;
        };
        return dw_dtype == PCFGNAT_DTYPE_F32 ? run(float()) : run(g);  // the caller's check leaves no other
    });
}

}  // namespace pcfgnat
