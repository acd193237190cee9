// Rows of the vocabulary table for tokens, times a scale, and the table's gradient.
//
// Forward: out[i] = scale * w[token_i].  One read of the rows that occur and one write; a thread moves one vector.
// Gradient: dw[v] = scale * sum of g[i] over token_i = v, summed in float32 in an order that the input alone decides:
//   1. embed_sort_kernel  — the positions grouped by token, equal tokens by position.  A block owns every 128th token of the
//      table and reads all positions: those of the blocks before it count where its entries begin, so no block waits for another.
//   2. embed_sum_kernel   — the sorted list cut into pieces of equal length.  A run of one token inside a piece is written
//      to the table at once; the part of a run that crosses a piece's border goes to scratch memory.
//   3. embed_join_kernel  — adds up the parts of every run that crosses pieces, in an order that its pieces decide.
// A placeholder that fills most positions is thus spread over as many blocks as its share of the list.
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
constexpr int kMaxRange = 512;   // tokens that one block may own
constexpr int kAhead = 8;        // loads of a lane in flight

struct Sorted {
    int *token, *at;  // the tokens that count and their positions, by token and then by position
    int *row_end;     // [V] where the list's entries of a token end
    int *total;       // entries
};

// The whole table set to zero by the blocks behind the sorting ones: those wait for their loads most of the time.
__device__ void zero_table(char *dw, int64_t rows, int64_t row_bytes, int64_t stride_bytes, int64_t block, int64_t blocks) {
    const int lane = threadIdx.x & 31;
    if (stride_bytes == row_bytes) row_bytes *= rows, stride_bytes = 0, rows = 1;  // one long row
    const bool wide = !((reinterpret_cast<uintptr_t>(dw) | row_bytes | stride_bytes) & 15);
    if (rows == 1) {
        const int64_t head = wide ? 0 : min((int64_t)(-reinterpret_cast<uintptr_t>(dw) & 15), row_bytes), vecs = (row_bytes - head) / 16;
        for (int64_t i = block * kSortThreads + threadIdx.x; i < vecs; i += blocks * kSortThreads)
            reinterpret_cast<uint4 *>(dw + head)[i] = make_uint4(0, 0, 0, 0);
        if (block == 0) {
            const int64_t loose = (row_bytes - vecs * 16) / 2, i = threadIdx.x;  // in units of two bytes
            if (i < loose) *reinterpret_cast<uint16_t *>(dw + (2 * i < head ? 2 * i : 2 * i + vecs * 16)) = 0;
        }
        return;
    }
    for (int64_t r = block * kSortWarps + (threadIdx.x >> 5); r < rows; r += blocks * kSortWarps) {
        char *p = dw + r * stride_bytes;
        if (wide) {
            for (int64_t i = lane; i < row_bytes / 16; i += 32) reinterpret_cast<uint4 *>(p)[i] = make_uint4(0, 0, 0, 0);
        } else {
            for (int64_t i = lane; i < row_bytes / 2; i += 32) reinterpret_cast<uint16_t *>(p)[i] = 0;
        }
    }
}

// Block b of 2^bits owns the tokens v with v mod 2^bits = b, so that neighbouring (frequent) words are dealt out.
__global__ void __launch_bounds__(kSortThreads, 2)
    embed_sort_kernel(const int64_t *__restrict__ tokens, int n, int V, uint32_t padding, int bits, int range, Sorted sorted,
                      char *dw, int row_bytes, int64_t dw_stride_bytes, int *status) {
    extern __shared__ int cell[];  // [warp][token of the block]: tokens of the warp's span, then where the next one goes
    __shared__ int warp_sum[kSortWarps], warp_below[kSortWarps];
    const int buckets = 1 << bits;
    if (blockIdx.x >= buckets) {
        zero_table(dw, V, row_bytes, dw_stride_bytes, blockIdx.x - buckets, gridDim.x - buckets);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bucket = blockIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the next kernel waits for this one's end all the same
    for (int i = tid; i < kSortWarps * range; i += kSortThreads) cell[i] = 0;
    __syncthreads();
    const int span = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
    const int first = (int)min((int64_t)warp * span, (int64_t)n), last = (int)min((int64_t)first + span, (int64_t)n);
    int *mine = cell + warp * range;
    const uint2 *words = reinterpret_cast<const uint2 *>(tokens);
    constexpr uint32_t kNone = 0xffffffffu;
    // the token of a position, kNone where it does not count
    const auto counted = [&](uint2 t) { return t.y == 0 && t.x < (uint32_t)V && t.x != padding ? t.x : kNone; };
    int below = 0;
    bool bad = false;
    uint64_t seen = 0;  // groups of 32 of the first 64 that hold tokens of the block; later groups are all looked at again
    int group = 0;
    for (int i0 = first; i0 < last; i0 += 32 * kAhead) {
        uint2 t[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + k * 32 + lane;
            t[k] = i < last ? words[i] : make_uint2(padding, 0);
            if (bucket == 0 && i < last) bad |= t[k].y != 0 || t[k].x >= (uint32_t)V;
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const uint32_t v = counted(t[k]);
            const int of = v == kNone ? buckets : (int)(v & (buckets - 1));
            below += of < bucket;
            if (of == bucket) atomicAdd(mine + (v >> bits), 1);
            if (__any_sync(0xffffffffu, of == bucket) && group < 64) seen |= 1ull << group;
            group++;
        }
    }
    if (bad) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) warp_below[warp] = below;
    __syncthreads();
    // where every token of the block begins, and within it every warp
    int mine_total = 0;
    if (tid < range)
        for (int w = 0; w < kSortWarps; w++) mine_total += cell[w * range + tid];
    int scan = mine_total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += x;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    if (tid < range) {
        int next = scan - mine_total;
        for (int w = 0; w < kSortWarps; w++) next += warp_below[w] + (w < warp ? warp_sum[w] : 0);
#pragma unroll 8
        for (int w = 0; w < kSortWarps; w++) {
            const int c = cell[w * range + tid];
            cell[w * range + tid] = next;
            next += c;
        }
        const int64_t v = ((int64_t)tid << bits) + bucket;
        if (v < V) sorted.row_end[v] = next;
        if (tid == range - 1 && bucket == buckets - 1) *sorted.total = next;
    }
    __syncthreads();
    group = 0;
    for (int i0 = first; i0 < last; i0 += 32 * kAhead, group += kAhead) {
        const uint32_t some = group < 64 ? (uint32_t)(seen >> group) & ((1u << kAhead) - 1) : (1u << kAhead) - 1;
        if (!some) continue;
        uint32_t v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + k * 32 + lane;
            v[k] = (some >> k & 1) && i < last ? counted(words[i]) : kNone;
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            // one token after the other, as few of them are the block's
            uint32_t todo = __ballot_sync(0xffffffffu, v[k] != kNone && (int)(v[k] & (buckets - 1)) == bucket);
            while (todo) {
                const uint32_t one = __shfl_sync(0xffffffffu, v[k], __ffs(todo) - 1);
                const uint32_t same = __ballot_sync(0xffffffffu, v[k] == one);
                const int row = (int)(one >> bits), from = mine[row];
                __syncwarp();
                if (v[k] == one) {
                    const int at = from + __popc(same & ((1u << lane) - 1));
                    sorted.token[at] = (int)one, sorted.at[at] = i0 + k * 32 + lane;
                }
                if (lane == 0) mine[row] = from + __popc(same);
                __syncwarp();
                todo &= ~same;
            }
        }
    }
}

// A finished sum into the table.  Every number of the table gets at most one sum per call, so adding to a float32 table by a
// reduction (which needs not wait for what is there) has one order only.
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

// A block adds up a piece of the list for a tile of columns, a warp an equal share of it, a lane REP times VEC columns (32 * VEC
// apart).  A warp's runs that cross its borders are joined in shared memory, in the list's order, and so are given on only where
// they cross the piece's.
template <typename G, typename W, int VEC, int REP>
__global__ void __launch_bounds__(32 * kSumWarps)
    embed_sum_kernel(const G *__restrict__ grad, int64_t g_stride, int H, Pieces p, W *dw, int64_t dw_stride, float scale,
                     int accumulate) {
    using Raw = typename RawVec<VEC * sizeof(G)>::type;
    constexpr int kTile = 32 * VEC * REP;
    __shared__ float crossing[kSumWarps][2][kTile];
    __shared__ int4 ends[kSumWarps];  // of a warp's share: first and last token, whether those runs go on before and behind it
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.y * kTile, c = tile + lane * VEC;  // of the lane's columns, the first
    const int total = *p.sorted.total;
    const int64_t begin64 = ((int64_t)blockIdx.x * kSumWarps + warp) * p.length;
    const int *token = p.sorted.token;
    if ((int64_t)blockIdx.x * kSumWarps * p.length >= total) return;
    if (begin64 < total) {
        const int begin = (int)begin64, end = min(begin + p.length, total);
        const int before = begin > 0 ? token[begin - 1] : -1, after = end < total ? token[end] : -1;
        float acc[REP][VEC] = {};
        int run = token[begin];
        bool began_before = run == before;
        if (lane == 0) {
            const int tail = token[end - 1];
            ends[warp] = make_int4(run, tail, run == before, tail == after);
        }
        for (int i0 = begin; i0 < end; i0 += 32) {
            const int count = min(32, end - i0);
            const int my_token = lane < count ? token[i0 + lane] : -1, my_at = lane < count ? p.sorted.at[i0 + lane] : 0;
            const int behind = i0 + count < end ? token[i0 + count] : -1;
            for (int j0 = 0; j0 < count; j0 += kAhead) {
                Raw raw[kAhead][REP];
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    const G *row = grad + __shfl_sync(0xffffffffu, my_at, (j0 + j) & 31) * g_stride;
#pragma unroll
                    for (int q = 0; q < REP; q++)
                        if (j0 + j < count && c + q * 32 * VEC < H) raw[j][q] = __ldg(reinterpret_cast<const Raw *>(row + c + q * 32 * VEC));
                }
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    const int next_of = __shfl_sync(0xffffffffu, my_token, (j0 + j + 1) & 31);
                    if (j0 + j >= count) continue;  // the same for the whole warp
#pragma unroll
                    for (int q = 0; q < REP; q++) {
                        float x[VEC];
                        unpack_vec<G, VEC>(raw[j][q], x);
#pragma unroll
                        for (int k = 0; k < VEC; k++) acc[q][k] += x[k];
                    }
                    const int next = j0 + j + 1 == count ? behind : next_of;
                    if (next == run) continue;
                    const bool goes_on = next < 0 && run == after;
#pragma unroll
                    for (int q = 0; q < REP; q++) {
                        if (began_before || goes_on) {
                            float *to = crossing[warp][began_before ? 0 : 1] + q * 32 * VEC + lane * VEC;
#pragma unroll
                            for (int k = 0; k < VEC; k++) to[k] = acc[q][k];
                        } else if (c + q * 32 * VEC < H) {
                            write_row<W, VEC>(dw + run * dw_stride + c + q * 32 * VEC, acc[q], scale, accumulate);
                        }
#pragma unroll
                        for (int k = 0; k < VEC; k++) acc[q][k] = 0.f;
                    }
                    run = next;
                    began_before = false;
                }
            }
        }
    }
    __syncthreads();
    // a thread per column: what the warps left, in the list's order
    for (int col = threadIdx.x; col < kTile; col += 32 * kSumWarps) {
        const int cc = tile + col;
        if (cc >= H) continue;
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
// lane four columns.
template <typename W>
__global__ void __launch_bounds__(32 * kJoinGroups)
    embed_join_kernel(int H, Pieces p, W *dw, int64_t dw_stride, float scale, int accumulate) {
    __shared__ float sums[kJoinGroups][kJoinColumns];
    chain_begin();
    const int total = *p.sorted.total, length = p.length * kSumWarps;
    const int64_t begin64 = (int64_t)blockIdx.x * length;
    if (begin64 + length >= total) return;
    const int begin = (int)begin64, end = begin + length;
    const int token = p.sorted.token[end - 1], behind = p.sorted.token[end], before = begin > 0 ? p.sorted.token[begin - 1] : -1;
    if (behind != token || before == token) return;
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

int widest(uintptr_t bits, int size) {  // bytes of the widest vector that addresses and strides allow, at least an element's
    for (int b = 16; b > size; b /= 2)
        if (!(bits & (uintptr_t)(b - 1))) return b;
    return size;
}

// Entries of a warp: eight loads of a lane in flight, more where that made over 2 048 pieces.
int warp_entries(int64_t n) {
    const int64_t even = (n + 2048 * kSumWarps - 1) / (2048 * kSumWarps);
    return (int)((even + kAhead - 1) / kAhead * kAhead) + (even == 0 ? kAhead : 0);
}
int64_t piece_count(int64_t n) {
    const int64_t length = (int64_t)warp_entries(n) * kSumWarps;
    return (n + length - 1) / length;
}

constexpr size_t round16(size_t x) { return (x + 15) / 16 * 16; }

}  // namespace

size_t embed_workspace_bytes(int64_t n, int64_t V, int H) {
    return 16 + 2 * round16((size_t)n * sizeof(int)) + round16((size_t)V * sizeof(int)) + (size_t)piece_count(n) * 2 * H * sizeof(float);
}

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
    char *ws = static_cast<char *>(workspace);
    const size_t list = round16((size_t)n * sizeof(int));
    const Sorted sorted{reinterpret_cast<int *>(ws + 16), reinterpret_cast<int *>(ws + 16 + list),
                        reinterpret_cast<int *>(ws + 16 + 2 * list), reinterpret_cast<int *>(ws)};
    float *parts = reinterpret_cast<float *>(ws + 16 + 2 * list + round16((size_t)V * sizeof(int)));
    const size_t dw_size = dw_dtype == PCFGNAT_DTYPE_F32 ? 4 : 2;
    int bits = 7;  // 128 blocks: as many as one of 1 024 threads each per SM gives
    while ((V + (1ll << bits) - 1) >> bits > kMaxRange) bits++;
    const int range = (int)((V + (1ll << bits) - 1) >> bits);
    const size_t smem = (size_t)kSortWarps * range * sizeof(int);
    cudaError_t e = ensure_dynamic_smem(embed_sort_kernel, smem);
    if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    const uint32_t skip = has_padding && padding >= 0 && padding < V ? (uint32_t)padding : 0xffffffffu;
    embed_sort_kernel<<<(1u << bits) + (accumulate ? 0u : (unsigned)sm_count()), kSortThreads, smem, st>>>(
        tokens, (int)n, (int)V, skip, bits, range, sorted, static_cast<char *>(dw), (int)(H * dw_size), (int64_t)(dw_stride * dw_size),
        status);
    e = cudaGetLastError();
    if (e != cudaSuccess || n == 0) return cuda_rc(e);
    const Pieces p{sorted, parts, warp_entries(n)};
    const unsigned pieces = (unsigned)piece_count(n);
    return with_dtype(dtype, [&](auto g) {
        using G = decltype(g);
        const auto run = [&](auto w) {
            using W = decltype(w);
            // a lane's columns: as many of the gradient's as 16 bytes hold, where both rows' addresses allow whole vectors
            const auto bits = [&](const void *a, int64_t stride, size_t size) {
                return reinterpret_cast<uintptr_t>(a) | (uintptr_t)(stride * size) | (uintptr_t)(H * size);
            };
            const int wide_g = widest(bits(grad, g_stride, sizeof(G)), sizeof(G)) / (int)sizeof(G);
            const int wide_w = widest(bits(dw, dw_stride, sizeof(W)), sizeof(W)) / (int)sizeof(W);
            // every kernel waits for the one before it to end, but may be scheduled before that
            const auto launch = [&](auto kernel, unsigned tiles, unsigned threads, auto... args) {
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = dim3(pieces, tiles);
                cfg.blockDim = dim3(threads);
                cfg.stream = st;
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
                attr[0].val.programmaticStreamSerializationAllowed = 1;
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                return cudaLaunchKernelEx(&cfg, kernel, args...);
            };
            const auto sum = [&](auto vec, auto rep) {
                constexpr int VEC = decltype(vec)::value, REP = decltype(rep)::value;
                return launch(embed_sum_kernel<G, W, VEC, REP>, (unsigned)((H + 32 * VEC * REP - 1) / (32 * VEC * REP)), 32 * kSumWarps,
                              static_cast<const G *>(grad), g_stride, H, p, static_cast<W *>(dw), dw_stride, scale, accumulate);
            };
            constexpr int kWide = 16 / sizeof(G), kWideW = 16 / sizeof(W) < kWide ? 16 / sizeof(W) : kWide;
            using std::integral_constant;
            cudaError_t rc;
            if (wide_g >= kWide && wide_w >= kWideW && H % kWide == 0) rc = sum(integral_constant<int, kWide>(), integral_constant<int, 1>());
            else if (wide_g >= 2 && wide_w >= 2) rc = sum(integral_constant<int, 2>(), integral_constant<int, 2>());
            else rc = sum(integral_constant<int, 1>(), integral_constant<int, 4>());
            if (rc != cudaSuccess) return (int)PCFGNAT_ERR_CUDA;
            if (pieces > 1)  // one piece has no border
                rc = launch(embed_join_kernel<W>, (unsigned)((H + kJoinColumns - 1) / kJoinColumns), 32 * kJoinGroups, H, p,
                            static_cast<W *>(dw), dw_stride, scale, accumulate);
            if (rc != cudaSuccess) return (int)PCFGNAT_ERR_CUDA;
            return cuda_rc(cudaGetLastError());
        };
        if (dw_dtype == PCFGNAT_DTYPE_F32) return run(float());
        if (dw_dtype == dtype) return run(g);
        return (int)PCFGNAT_ERR_UNSUPPORTED;
    });
}

}  // namespace pcfgnat
