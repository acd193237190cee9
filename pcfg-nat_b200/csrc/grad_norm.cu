// Global norm of many gradient tensors and clipping: n = |s| sqrt(sum g^2), c = min(1, limit / (n + 1e-6)), out = s c g.
//
// Two launches for up to kMaxTensors tensors, whose addresses and lengths travel as kernel parameters (copied at the launch, so
// that a captured graph holds them): squares summed per block into the caller's scratch memory, then every block adds up the
// blocks' sums in the same order, forms the factor, and scales its share.  Nothing is scaled where the factor is 1 and a tensor
// is its own output.  Squares and sums are held in 64 bits: the square of a float32 gradient beyond 1.8e19 or below 1e-19 has
// no float32.
#include "row_vectors.cuh"

namespace pcfgnat {

namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 4;
constexpr int kChunk = 8192;        // numbers that a block takes at a time
constexpr int kMaxTensors = 1024;   // of one launch: 29 bytes each of the 32 764 that parameters may have

struct Tensors {
    const void *src[kMaxTensors];
    void *dst[kMaxTensors];
    int64_t size[kMaxTensors];
    int first_chunk[kMaxTensors];  // chunks of the tensors before it
    uint8_t kind[kMaxTensors];     // type of src, and of dst times 4
    int count, chunks;
};

// The tensor that a chunk belongs to.
__device__ __forceinline__ int tensor_of(const Tensors &t, int chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first_chunk[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <class F>
__device__ __forceinline__ void with_type(int kind, F f) {
    if (kind == PCFGNAT_DTYPE_F32) f(float());
    else if (kind == PCFGNAT_DTYPE_F16) f(__half());
    else f(__nv_bfloat16());
}

__device__ __forceinline__ double block_sum(double v, double *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kThreads / 32; w++) v += part[w];
    return v;
}

__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Tensors t, double *sums) {
    __shared__ double part[kThreads / 32];
    const int tid = threadIdx.x;
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, t.size[k] - begin);
        with_type(t.kind[k] & 3, [&](auto type) {
            using T = decltype(type);
            constexpr int kVec = RowCut<T>::kVec;
            const T *src = static_cast<const T *>(t.src[k]) + begin;
            const RowCut<T> cut(src, n);
            const uint4 *vec = reinterpret_cast<const uint4 *>(src + cut.head);
#pragma unroll 4
            for (int i = tid; i < cut.vecs; i += kThreads) {
                float x[kVec];
                unpack_vec<T, kVec>(__ldg(vec + i), x);
#pragma unroll
                for (int j = 0; j < kVec; j++) sum += (double)x[j] * (double)x[j];
            }
            if (tid < cut.loose(n)) {
                const double x = num_to_float<T>(src[cut.loose_at(tid)]);
                sum += x * x;
            }
        });
    }
    sum = block_sum(sum, part);
    if (tid == 0) sums[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads)
    grad_scale_kernel(const __grid_constant__ Tensors t, const double *__restrict__ sums, int n_sums, float limit, float scale,
                      float *norm_out) {
    __shared__ double part[kThreads / 32];
    const int tid = threadIdx.x;
    double sum = 0.0;
    for (int i = tid; i < n_sums; i += kThreads) sum += sums[i];
    sum = block_sum(sum, part);
    const float norm = (float)(fabs((double)scale) * sqrt(sum));
    if (norm_out && blockIdx.x == 0 && tid == 0) *norm_out = norm;
    const float part_of = limit / (norm + 1e-6f);
    const float factor = (part_of >= 1.f ? 1.f : part_of) * scale;  // NaN stays NaN
    for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {  // what was read last is still in L2
        const int k = tensor_of(t, c);
        if (factor == 1.f && t.src[k] == t.dst[k]) continue;
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, t.size[k] - begin);
        with_type(t.kind[k] & 3, [&](auto type) {
            using T = decltype(type);
            const T *src = static_cast<const T *>(t.src[k]) + begin;
            const auto write = [&](auto other) {
                using D = decltype(other);
                constexpr int kVec = 16 / sizeof(T);
                D *dst = static_cast<D *>(t.dst[k]) + begin;
                const RowCut<T> cut(src, n);
                const uint4 *vec = reinterpret_cast<const uint4 *>(src + cut.head);
                if (!(reinterpret_cast<uintptr_t>(dst + cut.head) & 15)) {
                    for (int i = tid; i < cut.vecs; i += kThreads) {
                        float x[kVec];
                        unpack_vec<T, kVec>(vec[i], x);
#pragma unroll
                        for (int j = 0; j < kVec; j++) x[j] *= factor;
#pragma unroll
                        for (int j = 0; j < kVec; j += 16 / sizeof(D)) {
                            constexpr int kOut = 16 / sizeof(D) < kVec ? 16 / sizeof(D) : kVec;
                            float y[kOut];
#pragma unroll
                            for (int q = 0; q < kOut; q++) y[q] = x[j + q];
                            reinterpret_cast<uint4 *>(dst + cut.head + i * kVec + j)[0] = pack_vec<D, kOut>(y);
                        }
                    }
                    if (tid < cut.loose(n)) {
                        const int i = cut.loose_at(tid);
                        dst[i] = num_from_float<D>(num_to_float<T>(src[i]) * factor);
                    }
                } else {
                    for (int i = tid; i < n; i += kThreads) dst[i] = num_from_float<D>(num_to_float<T>(src[i]) * factor);
                }
            };
            if ((t.kind[k] >> 2) == PCFGNAT_DTYPE_F32) write(float());
            else if constexpr (sizeof(T) == 2) write(T());
        });
    }
}

}  // namespace

int clip_grad_norm_sums(int n) {  // doubles of scratch memory for n tensors
    return kBlocksPerSm * sm_count() * ((n + kMaxTensors - 1) / kMaxTensors);
}

int launch_clip_grad_norm(int n, const void *const *src, const int *src_dtype, void *const *dst, const int *dst_dtype,
                          const int64_t *size, float limit, float scale, double *sums, float *norm, cudaStream_t st) {
    const int blocks = kBlocksPerSm * sm_count();
    int n_sums = 0;
    Tensors t;
    for (int pass = 0; pass < 2; pass++) {
        bool norm_written = false;
        for (int first = 0; first < n || (pass == 1 && !norm_written); first += kMaxTensors) {
            int64_t chunks = 0;
            t.count = 0;
            for (int i = first; i < n && i < first + kMaxTensors; i++) {
                t.src[t.count] = src[i], t.dst[t.count] = dst[i], t.size[t.count] = size[i];
                t.kind[t.count] = (uint8_t)(src_dtype[i] | dst_dtype[i] << 2);
                t.first_chunk[t.count++] = (int)chunks;
                chunks += (size[i] + kChunk - 1) / kChunk;
                if (chunks > 0x3fffffff) return PCFGNAT_ERR_TOO_LARGE;
            }
            t.chunks = (int)chunks;
            const int grid = chunks < blocks ? (chunks > 0 ? (int)chunks : 1) : blocks;
            if (pass == 0) {
                grad_squares_kernel<<<grid, kThreads, 0, st>>>(t, sums + n_sums);
                n_sums += grid;
            } else {
                grad_scale_kernel<<<grid, kThreads, 0, st>>>(t, sums, n_sums, limit, scale, norm_written ? nullptr : norm);
                norm_written = true;
            }
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
        }
    }
    return PCFGNAT_OK;
}

}  // namespace pcfgnat
