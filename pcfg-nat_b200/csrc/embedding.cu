// Rows of the vocabulary table for tokens, times a scale, and the table's gradient.
//
// Forward: out[i] = scale * w[token_i].  One read of the rows that occur and one write; a thread moves one vector.
// Gradient: dw[v] = scale * sum of g[i] over token_i = v, summed in float32 in an order that the input alone decides:
//   1. embed_sort_kernel  — the positions sorted by token, equal tokens by position.  A block owns a range of the table's rows
//      and reads all tokens: those below its range count where its entries begin, so no block waits for another.
//   2. embed_sum_kernel   — the sorted list cut into pieces of equal length.  A run of one token inside a piece is written
//      to the table at once; the part of a run that crosses a piece's border goes to scratch memory.
//   3. embed_join_kernel  — adds up the parts of every run that crosses borders, in the order of the pieces.
// A placeholder that fills most positions is thus spread over as many blocks as its share of the list.
#include "row_vectors.cuh"

namespace pcfgnat {

namespace {

constexpr int kThreads = 256;

// ---- forward

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    embed_rows_kernel(const T *__restrict__ weight, int64_t w_stride, int64_t V, int H, const int64_t *__restrict__ tokens,
                      int64_t n, float scale, T *__restrict__ out, int *status) {
    using Raw = typename RawVec<VEC * sizeof(T)>::type;
    const int per_row = H / VEC;
    const int64_t total = n * per_row;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / per_row;
        const int c = (int)(i - r * per_row);
        const int64_t t = tokens[r];
        float x[VEC];
        if (t < 0 || t >= V) {
#pragma unroll
            for (int k = 0; k < VEC; k++) x[k] = CUDART_NAN_F;
            if (c == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
        } else {
            unpack_vec<T, VEC>(__ldg(reinterpret_cast<const Raw *>(weight + t * w_stride) + c), x);
#pragma unroll
            for (int k = 0; k < VEC; k++) x[k] *= scale;
        }
        reinterpret_cast<Raw *>(out + r * H)[c] = pack_vec<T, VEC>(x);
    }
}

// ---- gradient

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxRange = 512;   // rows of the table that one block may own

__device__ __forceinline__ void zero_row(char *p, int bytes, int lane) {
    if (!((reinterpret_cast<uintptr_t>(p) | (unsigned)bytes) & 15)) {
        for (int i = lane; i < bytes / 16; i += 32) reinterpret_cast<uint4 *>(p)[i] = make_uint4(0, 0, 0, 0);
    } else {
        for (int i = lane; i < bytes / 2; i += 32) reinterpret_cast<uint16_t *>(p)[i] = 0;
    }
}

// sorted_token / sorted_at: the tokens that count and their positions, sorted; *total their number.  Rows of dw without a
// token are set to zero where `zero`.
__global__ void __launch_bounds__(kSortThreads)
    embed_sort_kernel(const int64_t *__restrict__ tokens, int n, int64_t V, int has_padding, int64_t padding, int range,
                      int *sorted_token, int *sorted_at, int *total, char *dw, int64_t row_bytes, int64_t dw_stride_bytes,
                      int zero, int *status) {
    extern __shared__ int cell[];  // [warp][row of the range]: tokens of the warp's span, then where the next one goes
    __shared__ int warp_sum[kSortWarps], warp_below[kSortWarps];
    __shared__ int counts[kMaxRange];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t v0 = (int64_t)blockIdx.x * range, v1 = min(v0 + range, V);
    const int rows = (int)(v1 - v0);
    for (int i = tid; i < kSortWarps * range; i += kSortThreads) cell[i] = 0;
    __syncthreads();
    const int span = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
    const int first = min((int64_t)warp * span, (int64_t)n), last = min((int64_t)first + span, (int64_t)n);
    int *mine = cell + warp * range;
    int below = 0;
    bool bad = false;
    for (int i = first + lane; i < last; i += 32) {
        const int64_t t = tokens[i];
        if (t < 0 || t >= V) {
            bad = true;
            continue;
        }
        if (has_padding && t == padding) continue;
        if (t < v0) below++;
        else if (t < v1) atomicAdd(mine + (t - v0), 1);
    }
    if (bad && blockIdx.x == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) warp_below[warp] = below;
    __syncthreads();
    // where every row of the range begins, and within it every warp
    int mine_total = 0;
    if (tid < rows)
        for (int w = 0; w < kSortWarps; w++) mine_total += cell[w * range + tid];
    int scan = mine_total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += x;
    }
    if (lane == 31) warp_sum[warp] = scan;
    if (tid < kMaxRange) counts[tid] = mine_total;
    __syncthreads();
    int start = scan - mine_total;
    for (int w = 0; w < kSortWarps; w++) start += warp_below[w] + (w < warp ? warp_sum[w] : 0);
    if (tid < rows) {
        int next = start;
        for (int w = 0; w < kSortWarps; w++) {
            const int c = cell[w * range + tid];
            cell[w * range + tid] = next;
            next += c;
        }
        if (tid == rows - 1 && v1 == V) *total = next;
    }
    __syncthreads();
    if (zero)
        for (int r = warp; r < rows; r += kSortWarps)
            if (counts[r] == 0) zero_row(dw + (v0 + r) * dw_stride_bytes, (int)row_bytes, lane);
    for (int i0 = first; i0 < last; i0 += 32) {
        const int i = i0 + lane;
        const int64_t t = i < last ? tokens[i] : -1;
        const bool in = t >= v0 && t < v1 && !(has_padding && t == padding);
        const uint32_t any = __ballot_sync(0xffffffffu, in);
        if (any == 0) continue;
        const int row = in ? (int)(t - v0) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, row);
        int at = 0;
        if (in) at = mine[row] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (in && lane == __ffs(same) - 1) mine[row] += __popc(same);
        __syncwarp();
        if (in) sorted_token[at] = (int)t, sorted_at[at] = i;
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void write_row(T *p, const float (&acc)[VEC], float scale, int accumulate) {
    using Raw = typename RawVec<VEC * sizeof(T)>::type;
    float x[VEC];
    if (accumulate) {
        unpack_vec<T, VEC>(*reinterpret_cast<const Raw *>(p), x);
#pragma unroll
        for (int k = 0; k < VEC; k++) x[k] += acc[k] * scale;
    } else {
#pragma unroll
        for (int k = 0; k < VEC; k++) x[k] = acc[k] * scale;
    }
    *reinterpret_cast<Raw *>(p) = pack_vec<T, VEC>(x);
}

struct Pieces {
    const int *sorted_token, *sorted_at, *total;
    float *parts;  // [piece][2][H]: what a piece holds of a run that began before it, and of one that goes on behind it
    int length;    // entries of a piece
};

// VEC elements of the gradient per thread; a table of another type than the gradient's is written VEC at a time as well.
template <typename G, typename W, int VEC>
__global__ void __launch_bounds__(kThreads)
    embed_sum_kernel(const G *__restrict__ grad, int64_t g_stride, int H, Pieces p, W *dw, int64_t dw_stride, float scale,
                     int accumulate) {
    using Raw = typename RawVec<VEC * sizeof(G)>::type;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int total = *p.total;
    const int64_t begin64 = (int64_t)blockIdx.x * p.length;
    if (begin64 >= total || c >= H) return;
    const int begin = (int)begin64, end = min(begin + p.length, total);
    const int before = begin > 0 ? p.sorted_token[begin - 1] : -1, after = end < total ? p.sorted_token[end] : -1;
    float *head = p.parts + (int64_t)blockIdx.x * 2 * H + c, *tail = head + H;
    float acc[VEC] = {};
    int token = p.sorted_token[begin];
    bool began_before = token == before;
    for (int i = begin; i < end; i++) {
        const int at = p.sorted_at[i];
        float x[VEC];
        unpack_vec<G, VEC>(__ldg(reinterpret_cast<const Raw *>(grad + at * g_stride + c)), x);
#pragma unroll
        for (int k = 0; k < VEC; k++) acc[k] += x[k];
        const int next = i + 1 < end ? p.sorted_token[i + 1] : -1;
        if (next == token) continue;
        if (began_before || (i + 1 == end && token == after)) {
            float *to = began_before ? head : tail;
#pragma unroll
            for (int k = 0; k < VEC; k++) to[k] = acc[k];
        } else {
            write_row<W, VEC>(dw + token * dw_stride + c, acc, scale, accumulate);
        }
#pragma unroll
        for (int k = 0; k < VEC; k++) acc[k] = 0.f;
        token = next;
        began_before = false;
    }
}

template <typename W>
__global__ void __launch_bounds__(kThreads)
    embed_join_kernel(int H, Pieces p, W *dw, int64_t dw_stride, float scale, int accumulate) {
    const int total = *p.total;
    const int64_t begin64 = (int64_t)blockIdx.x * p.length;
    const int c = blockIdx.y * kThreads + threadIdx.x;
    if (begin64 + p.length >= total || c >= H) return;
    const int begin = (int)begin64, end = begin + p.length;
    const int token = p.sorted_token[end - 1];
    if (p.sorted_token[end] != token || (begin > 0 && p.sorted_token[begin - 1] == token)) return;
    float acc[1] = {p.parts[(int64_t)blockIdx.x * 2 * H + H + c]};
    for (int64_t q = blockIdx.x + 1; q * p.length < total && p.sorted_token[q * p.length] == token; q++)
        acc[0] += p.parts[q * 2 * H + c];
    write_row<W, 1>(dw + token * dw_stride + c, acc, scale, accumulate);
}

int widest(uintptr_t bits, int size) {  // bytes of the widest vector that addresses and strides allow, at least an element's
    for (int b = 16; b > size; b /= 2)
        if (!(bits & (uintptr_t)(b - 1))) return b;
    return size;
}

int piece_length(int64_t n) {
    const int64_t even = (n + 2047) / 2048;  // at most 2 048 pieces
    return (int)(even < 16 ? 16 : even);
}
int64_t piece_count(int64_t n) { return (n + piece_length(n) - 1) / piece_length(n); }

constexpr size_t round16(size_t x) { return (x + 15) / 16 * 16; }

}  // namespace

size_t embed_workspace_bytes(int64_t n, int H) {
    return 16 + 2 * round16((size_t)n * sizeof(int)) + (size_t)piece_count(n) * 2 * H * sizeof(float);
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
            const int64_t blocks = (n * (H / VEC) + kThreads - 1) / kThreads;
            const int64_t most = (int64_t)sm_count() * 32;
            embed_rows_kernel<T, VEC><<<(unsigned)(blocks < most ? blocks : most), kThreads, 0, st>>>(
                static_cast<const T *>(weight), w_stride, V, H, tokens, n, scale, static_cast<T *>(out), status);
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
    int *total = reinterpret_cast<int *>(ws);
    int *sorted_token = reinterpret_cast<int *>(ws + 16);
    int *sorted_at = reinterpret_cast<int *>(ws + 16 + round16((size_t)n * sizeof(int)));
    float *parts = reinterpret_cast<float *>(ws + 16 + 2 * round16((size_t)n * sizeof(int)));
    const size_t dw_size = dw_dtype == PCFGNAT_DTYPE_F32 ? 4 : 2;
    const int64_t per_sm = (V + sm_count() - 1) / sm_count();
    const int range = (int)(per_sm < kMaxRange ? per_sm : kMaxRange);
    const size_t smem = (size_t)kSortWarps * range * sizeof(int);
    cudaError_t e = ensure_dynamic_smem(embed_sort_kernel, smem);
    if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    embed_sort_kernel<<<(unsigned)((V + range - 1) / range), kSortThreads, smem, st>>>(
        tokens, (int)n, V, has_padding, padding, range, sorted_token, sorted_at, total, static_cast<char *>(dw), (int64_t)(H * dw_size),
        (int64_t)(dw_stride * dw_size), !accumulate, status);
    e = cudaGetLastError();
    if (e != cudaSuccess || n == 0) return cuda_rc(e);
    const Pieces p{sorted_token, sorted_at, total, parts, piece_length(n)};
    const unsigned pieces = (unsigned)piece_count(n);
    return with_dtype(dtype, [&](auto g) {
        using G = decltype(g);
        const auto run = [&](auto w) {
            using W = decltype(w);
            // one vector width for both: the gradient's rows in 16 bytes, the table's in as many elements
            const auto bits = [&](const void *a, int64_t stride, size_t size) {
                return reinterpret_cast<uintptr_t>(a) | (uintptr_t)(stride * size) | (uintptr_t)(H * size);
            };
            const int wide_g = widest(bits(grad, g_stride, sizeof(G)), sizeof(G)) / (int)sizeof(G);
            const int wide_w = widest(bits(dw, dw_stride, sizeof(W)), sizeof(W)) / (int)sizeof(W);
            const int wide = wide_g < wide_w ? wide_g : wide_w;
            const auto sum = [&](auto vec) {
                constexpr int VEC = decltype(vec)::value;
                const int chunks = H / VEC;
                const int threads = chunks >= kThreads ? kThreads : (chunks + 31) / 32 * 32;
                embed_sum_kernel<G, W, VEC><<<dim3(pieces, (unsigned)((chunks + threads - 1) / threads)), threads, 0, st>>>(
                    static_cast<const G *>(grad), g_stride, H, p, static_cast<W *>(dw), dw_stride, scale, accumulate);
            };
            if (wide >= 4) sum(std::integral_constant<int, 4>());
            else if (wide >= 2) sum(std::integral_constant<int, 2>());
            else sum(std::integral_constant<int, 1>());
            embed_join_kernel<W><<<dim3(pieces, (unsigned)((H + kThreads - 1) / kThreads)), kThreads, 0, st>>>(
                H, p, static_cast<W *>(dw), dw_stride, scale, accumulate);
            return cuda_rc(cudaGetLastError());
        };
        if (dw_dtype == PCFGNAT_DTYPE_F32) return run(float());
        if (dw_dtype == dtype) return run(g);
        return (int)PCFGNAT_ERR_UNSUPPORTED;
    });
}

}  // namespace pcfgnat
