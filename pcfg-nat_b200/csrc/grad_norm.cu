// Global norm of many gradient tensors and clipping: n = |s| sqrt(sum g^2), c = min(1, limit / (n + 1e-6)), out = s c g.
//
// Two launches for up to kMaxTensors tensors, whose addresses and lengths travel as kernel parameters (copied at the launch, so
// that a captured graph holds them): squares summed per block into the caller's scratch memory, then every block adds up the
// blocks' sums in the same order, forms the factor, and scales its share.  Nothing is scaled where the factor is 1 and a tensor
// is its own output.  Sums are held in 64 bits, and so are the squares of float32 gradients: beyond 1.8e19 or below 1e-19 they have
// no float32.  Of halves, eight squares are added in float32 before.
#include "row_vectors.cuh"

namespace pcfgnat {

namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 8;      // base model, halves to floats: 98 us, with four 115
constexpr int kChunk = 8192;        // numbers that a block takes at a time
constexpr int kUnroll = 4;           // loads of a thread in flight
constexpr int kMaxTensors = 1024;   // of one launch: 29 bytes each of the 32 764 that parameters may have

// N is a few sizes, so that a short list does not pay for the parameters of a long one.
template <int N>
struct Tensors {
    const void *src[N];
    void *dst[N];
    int64_t size[N];
    int first_chunk[N];  // chunks of the tensors before it
    uint8_t kind[N];     // type of src, and of dst times 4
    int count, chunks, all_in_place;
};

// Which tensor a chunk belongs to, by a search in shared memory.
template <int N>
struct ChunkMap {
    int first_chunk[N];
    __device__ __forceinline__ void fill(const Tensors<N> &t) {
        for (int i = threadIdx.x; i < t.count; i += kThreads) first_chunk[i] = t.first_chunk[i];
        __syncthreads();
    }
    __device__ __forceinline__ int tensor_of(int chunk, int count) const {
        int lo = 0, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first_chunk[mid] <= chunk) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};

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

// The squares of a vector's numbers.  Those of half-precision numbers have at most 22 bits: in float32 every product is exact, and
// the eight are added by pairs, so that each passes three roundings of 2^-24 (one after the other the sum could lose 7 of them); the
// sum is added in 64 bits.  The norm is then off by at most 1.5 * 2^-24 before its own rounding.  bfloat16 numbers have the range of
// float32, so sums that left float32's range, or come near its lower end, are formed again in 64 bits.
template <typename T>
__device__ __forceinline__ double squares(const uint4 &raw) {
    constexpr int kVec = RowCut<T>::kVec;
    float x[kVec];
    unpack_vec<T, kVec>(raw, x);
    if constexpr (sizeof(T) == 2) {
        float two[kVec / 2];
#pragma unroll
        for (int j = 0; j < kVec / 2; j++) two[j] = fmaf(x[2 * j], x[2 * j], x[2 * j + 1] * x[2 * j + 1]);
        const float s = (two[0] + two[1]) + (two[2] + two[3]);
        if (std::is_same_v<T, __half> || (s >= 1e-25f && s <= 1e37f)) return s;
        if (((raw.x | raw.y | raw.z | raw.w) & 0x7fff7fffu) == 0) return 0.0;
    }
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kVec; j++) sum += (double)x[j] * (double)x[j];
    return sum;
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Tensors<N> t, double *sums) {
    __shared__ double part[kThreads / 32];
    __shared__ ChunkMap<N> map;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the next kernel waits for this one's end all the same
    map.fill(t);
    const int tid = threadIdx.x;
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = map.tensor_of(c, t.count);
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, t.size[k] - begin);
        with_type(t.kind[k] & 3, [&](auto type) {
            using T = decltype(type);
            constexpr int kVec = RowCut<T>::kVec;
            const T *src = static_cast<const T *>(t.src[k]) + begin;
            const RowCut<T> cut(src, n);
            const uint4 *vec = reinterpret_cast<const uint4 *>(src + cut.head);
            int i = tid;
            for (; i + (kUnroll - 1) * kThreads < cut.vecs; i += kUnroll * kThreads) {
                uint4 raw[kUnroll];
#pragma unroll
                for (int j = 0; j < kUnroll; j++) raw[j] = __ldg(vec + i + j * kThreads);
#pragma unroll
                for (int j = 0; j < kUnroll; j++) sum += squares<T>(raw[j]);
            }
            for (; i < cut.vecs; i += kThreads) sum += squares<T>(__ldg(vec + i));
            if (tid < cut.loose(n)) {
                const double x = num_to_float<T>(src[cut.loose_at(tid)]);
                sum += x * x;
            }
        });
    }
    sum = block_sum(sum, part);
    if (tid == 0) sums[blockIdx.x] = sum;
}

template <int N>
__global__ void __launch_bounds__(kThreads)
    grad_scale_kernel(const __grid_constant__ Tensors<N> t, const double *sums, int n_sums, float limit, float scale, float *norm_out) {
    __shared__ double part[kThreads / 32];
    __shared__ ChunkMap<N> map;
    map.fill(t);
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the sums are still formed
    double sum = 0.0;
    for (int i = tid; i < n_sums; i += kThreads) sum += sums[i];
    sum = block_sum(sum, part);
    const float norm = (float)(fabs((double)scale) * sqrt(sum));
    if (norm_out && blockIdx.x == 0 && tid == 0) *norm_out = norm;
    const float part_of = limit == CUDART_INF_F ? 1.f : limit / (norm + 1e-6f);  // no limit: whatever the norm is
    const float factor = (part_of >= 1.f ? 1.f : part_of) * scale;  // NaN stays NaN
    if (factor == 1.f && t.all_in_place) return;
    for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {  // what was read last is still in L2
        const int k = map.tensor_of(c, t.count);
        if (factor == 1.f && t.src[k] == t.dst[k]) continue;
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * kChunk;
        const int n = (int)min((int64_t)kChunk, t.size[k] - begin);
        with_type(t.kind[k] & 3, [&](auto type) {
            using T = decltype(type);
            const T *src = static_cast<const T *>(t.src[k]) + begin;
            const auto write = [&](auto other) {
                using D = decltype(other);
                // whole 16-byte stores side by side: halves are read eight bytes at a time where floats are written
                constexpr int kNum = 16 / sizeof(D);
                using Raw = typename RawVec<kNum * sizeof(T)>::type;
                D *dst = static_cast<D *>(t.dst[k]) + begin;
                const RowCut<T> cut(src, n);
                const Raw *from = reinterpret_cast<const Raw *>(src + cut.head);
                if (!(reinterpret_cast<uintptr_t>(dst + cut.head) & 15)) {
                    const auto scale_vector = [&](const Raw &raw, int i) {
                        float x[kNum];
                        unpack_vec<T, kNum>(raw, x);
#pragma unroll
                        for (int j = 0; j < kNum; j++) x[j] *= factor;
                        // not read again here: it should not push out what is still to be read
                        __stcs(reinterpret_cast<uint4 *>(dst + cut.head) + i, pack_vec<D, kNum>(x));
                    };
                    const int units = cut.vecs * RowCut<T>::kVec / kNum;
                    int i = tid;
                    for (; i + (kUnroll - 1) * kThreads < units; i += kUnroll * kThreads) {
                        Raw raw[kUnroll];
#pragma unroll
                        for (int j = 0; j < kUnroll; j++) raw[j] = from[i + j * kThreads];
#pragma unroll
                        for (int j = 0; j < kUnroll; j++) scale_vector(raw[j], i + j * kThreads);
                    }
                    for (; i < units; i += kThreads) scale_vector(from[i], i);
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

namespace {

// Both launches' parameters for the tensors [first, first + count); false where a chunk's number does not fit.
template <int N>
bool describe(Tensors<N> &t, int first, int count, const void *const *src, const int *src_dtype, void *const *dst, const int *dst_dtype,
              const int64_t *size) {
    int64_t chunks = 0;
    t.count = count, t.all_in_place = 1;
    for (int i = 0; i < count; i++) {
        t.src[i] = src[first + i], t.dst[i] = dst[first + i], t.size[i] = size[first + i];
        t.kind[i] = (uint8_t)(src_dtype[first + i] | dst_dtype[first + i] << 2);
        t.first_chunk[i] = (int)chunks;
        if (t.src[i] != t.dst[i]) t.all_in_place = 0;
        chunks += (t.size[i] + kChunk - 1) / kChunk;
        if (chunks > 0x3fffffff) return false;
    }
    t.chunks = (int)chunks;
    return true;
}

template <int N>
int clip_all(int n, const void *const *src, const int *src_dtype, void *const *dst, const int *dst_dtype, const int64_t *size,
             float limit, float scale, double *sums, float *norm, cudaStream_t st) {
    const int blocks = kBlocksPerSm * sm_count();
    int n_sums = 0;
    Tensors<N> t;
    const auto next = [&](int first) {  // describes the tensors from `first` on; blocks of their launches, -1: too many chunks
        if (!describe(t, first, n - first < N ? n - first : N, src, src_dtype, dst, dst_dtype, size)) return -1;
        return t.chunks < 1 ? 1 : t.chunks < blocks ? t.chunks : blocks;
    };
    for (int first = 0; first < n; first += N) {
        const int grid = next(first);
        if (grid < 0) return PCFGNAT_ERR_TOO_LARGE;
        grad_squares_kernel<N><<<grid, kThreads, 0, st>>>(t, sums + n_sums);
        n_sums += grid;
        if (cudaGetLastError() != cudaSuccess) return PCFGNAT_ERR_CUDA;
    }
    for (int first = 0; first < n || first == 0; first += N) {
        const int grid = n > N || n == 0 ? next(first) : n_sums;  // what a single launch was told is still there
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, grad_scale_kernel<N>, t, (const double *)sums, n_sums, limit, scale,
                                                 first == 0 ? norm : (float *)nullptr);
        if (e != cudaSuccess) return PCFGNAT_ERR_CUDA;
    }
    return PCFGNAT_OK;
}

}  // namespace

int launch_clip_grad_norm(int n, const void *const *src, const int *src_dtype, void *const *dst, const int *dst_dtype,
                          const int64_t *size, float limit, float scale, double *sums, float *norm, cudaStream_t st) {
    if (n <= 64) return clip_all<64>(n, src, src_dtype, dst, dst_dtype, size, limit, scale, sums, norm, st);
    if (n <= 320) return clip_all<320>(n, src, src_dtype, dst, dst_dtype, size, limit, scale, sums, norm, st);
    return clip_all<kMaxTensors>(n, src, src_dtype, dst, dst_dtype, size, limit, scale, sums, norm, st);
}

}  // namespace pcfgnat
