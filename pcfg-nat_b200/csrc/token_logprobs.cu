// Log probabilities of given tokens from materialised logits, with the row's entropy and its best alternatives, and the
// gradient of the logits.
//
// With m = max x, S = sum e^(x-m), U = sum e^(x-m) (x-m):  log p_v = (x_v - m) - log S,  H = log S - U / S.
// All three come from one pass over the row: a thread keeps its own m, S and U and rescales them when its maximum grows
// (U' = r (U + S (m - m')), r = e^(m-m'), all terms of one sign), and the threads' triples are joined the same way.
// Entries of -inf (a masked vocabulary) have probability 0 and add nothing; the least finite number of a type is a number
// like any other.  A row with NaN or +inf in it is NaN throughout, a row of nothing but -inf has log p = -inf and H = 0.
//
// The `top` largest values (equal ones by rising index) need no second pass: the top-th largest of the threads' maxima is a
// lower bound of the top-th largest value, so only the few threads whose maximum reaches it look at their numbers again.
#include <cfloat>

#include "row_vectors.cuh"

namespace pcfgnat {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnroll = 4;            // 16-byte loads of a thread in flight
constexpr int kMaxTop = PCFGNAT_MAX_TOP;
constexpr int kCandidates = 512;      // values that reach the bound; more are handled one at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFarBelow = -1.0e4f;  // 2^x of anything smaller is 0, and 0 * x stays 0 (with -inf it would be NaN)

struct Stats {
    float m = -FLT_MAX, s = 0.f, u = 0.f;  // maximum of the finite entries, S, and U in units of log 2
};

// Moves the reference of (S, U) from its own maximum up to m.
__device__ __forceinline__ void rescale(Stats &a, float m) {
    const float d = max_nan((a.m - m) * kLog2e, kFarBelow), r = exp2_approx(d);
    a.u = r * (a.u + d * a.s);
    a.s *= r;
    a.m = m;
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float m = max_nan(a.m, b.m);
    rescale(a, m);
    rescale(b, m);
    a.s += b.s;
    a.u += b.u;
    return a;
}
template <int N>
__device__ __forceinline__ void take(Stats &a, const float (&x)[N]) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < N; k++) m = max_nan(m, x[k]);
    rescale(a, m);
#pragma unroll
    for (int k = 0; k < N; k++) {
        const float d = max_nan((x[k] - m) * kLog2e, kFarBelow), e = exp2_approx(d);
        a.s += e;
        a.u += e * d;
    }
}

// Order-preserving integers of floats (no NaN among them).
__device__ __forceinline__ uint32_t rank_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 equals +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// One key per entry: larger value first, then smaller index.
__device__ __forceinline__ uint64_t entry_key(float x, int index) {
    return (uint64_t)rank_bits(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

struct Rows {
    const void *logits;
    int64_t inner, stride_outer, stride_inner;  // row r lies at (r / inner) * stride_outer + (r % inner) * stride_inner
    int V;
    template <typename T>
    __device__ __forceinline__ const T *at(int64_t r) const {
        return static_cast<const T *>(logits) + (r / inner) * stride_outer + (r % inner) * stride_inner;
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
    token_logprobs_kernel(Rows rows, const int64_t *__restrict__ tokens, int has_ignore, int64_t ignore, int top,
                          float *logprob, float *entropy, float *top_logprob, int64_t *top_index, float *kept, int *status) {
    constexpr int kVec = RowCut<T>::kVec;
    __shared__ Stats part[kWarps];
    __shared__ uint32_t maxima[kThreads];
    __shared__ uint64_t found[kCandidates];
    __shared__ int n_found;
    __shared__ uint32_t bound;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r = blockIdx.x;
    const int V = rows.V;
    const int64_t token = tokens[r];
    if (has_ignore && token == ignore) {
        if (tid == 0) {
            logprob[r] = 0.f;
            if (entropy) entropy[r] = 0.f;
            if (kept) kept[2 * r] = kept[2 * r + 1] = 0.f;
        }
        if (tid < top) top_logprob[r * top + tid] = 0.f, top_index[r * top + tid] = -1;
        return;
    }
    const T *row = rows.at<T>(r);
    const RowCut<T> cut(row, V);
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + cut.head);
    Stats a;
    {
        int i = tid;
        for (; i + (kUnroll - 1) * kThreads < cut.vecs; i += kUnroll * kThreads) {
            uint4 raw[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; k++) raw[k] = __ldg(vec + i + k * kThreads);
#pragma unroll
            for (int k = 0; k < kUnroll; k++) {
                float x[kVec];
                unpack_vec<T, kVec>(raw[k], x);
                take(a, x);
            }
        }
        for (; i < cut.vecs; i += kThreads) {
            float x[kVec];
            unpack_vec<T, kVec>(__ldg(vec + i), x);
            take(a, x);
        }
        if (tid < cut.loose(V)) {
            float x[1] = {num_to_float<T>(row[cut.loose_at(tid)])};
            take(a, x);
        }
    }
    const float own_max = a.m;
    const bool own_any = a.s > 0.f;  // some entry that is not -inf
    if (tid == 0) n_found = 0;
    maxima[tid] = own_any ? rank_bits(own_max) : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stats b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.u = __shfl_xor_sync(0xffffffffu, a.u, o);
        a = join(a, b);
    }
    if (lane == 0) part[warp] = a;
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int w = 1; w < kWarps; w++) a = join(a, part[w]);
    const float log_s = logf(a.s);  // -inf for a row of nothing but -inf
    if (tid == 0) {
        float lp;
        if (token < 0 || token >= V) {
            lp = CUDART_NAN_F;
            flag(status, PCFGNAT_STATUS_BAD_INDEX);
        } else {
            const float x = num_to_float<T>(row[token]);
            lp = a.s == 0.f ? neg_inf() : (x - a.m) - log_s;
        }
        logprob[r] = lp;
        if (entropy) entropy[r] = a.s == 0.f ? 0.f : log_s - kLn2 * (a.u / a.s);
        if (kept) kept[2 * r] = a.m, kept[2 * r + 1] = log_s;
    }
    if (top == 0) return;
    if (!(a.s > 0.f)) {  // no distribution, or nothing in it
        if (tid < top) top_logprob[r * top + tid] = a.s == 0.f ? neg_inf() : a.s, top_index[r * top + tid] = -1;
        return;
    }
    if (warp == 0) {  // the top-th largest of the threads' maxima
        uint32_t v[kWarps];
        uint32_t best = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) v[w] = maxima[w * 32 + lane], best = max(best, v[w]);
        uint32_t at = 0;
        for (int k = 0; k < top; k++) {
            at = __reduce_max_sync(0xffffffffu, best);
            if (at == 0) break;  // fewer threads than that saw anything: every number is a candidate
            const uint32_t who = __ballot_sync(0xffffffffu, best == at);
            if (lane == __ffs(who) - 1) {
                bool gone = false;
                best = 0;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    if (!gone && v[w] == at) v[w] = 0, gone = true;
                    best = max(best, v[w]);
                }
            }
        }
        if (lane == 0) bound = at;
    }
    __syncthreads();
    const uint32_t least = bound;
    const uint32_t again = __ballot_sync(0xffffffffu, own_any && rank_bits(own_max) >= least);
    const auto offer = [&](float x, int index) {
        if (x == neg_inf() || rank_bits(x) < least) return;
        const int at = atomicAdd(&n_found, 1);
        if (at < kCandidates) found[at] = entry_key(x, index);
    };
    for (uint32_t todo = again; todo; todo &= todo - 1) {
        const int of = warp * 32 + __ffs(todo) - 1;
        for (int i = of + lane * kThreads; i < cut.vecs; i += 32 * kThreads) {
            float x[kVec];
            unpack_vec<T, kVec>(__ldg(vec + i), x);
#pragma unroll
            for (int k = 0; k < kVec; k++) offer(x[k], cut.head + i * kVec + k);
        }
        if (lane == 0 && of < cut.loose(V)) {
            const int i = cut.loose_at(of);
            offer(num_to_float<T>(row[i]), i);
        }
    }
    __syncthreads();
    const int n = n_found;
    if (n <= kCandidates) {
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t key = found[i];
            int better = 0;
            for (int j = 0; j < n; j++) better += found[j] > key;
            if (better < top) {
                top_logprob[r * top + better] = (key_value(key) - a.m) - log_s;
                top_index[r * top + better] = key_index(key);
            }
        }
        if (tid >= n && tid < top) top_logprob[r * top + tid] = neg_inf(), top_index[r * top + tid] = -1;
        return;
    }
    // Many equal values at the bound: one sweep over the row per alternative.
    uint64_t last = ~0ull;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        for (int i = tid; i < V; i += kThreads) {
            const float x = num_to_float<T>(row[i]);
            const uint64_t key = entry_key(x, i);
            if (x != neg_inf() && key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) found[warp] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; w++) best = found[w] > best ? found[w] : best;
        if (tid == 0) {
            top_logprob[r * top + k] = (key_value(best) - a.m) - log_s;
            top_index[r * top + k] = key_index(best);
        }
        last = best;
    }
}

// d x_v = p_v (-G - h (log p_v + H)) + sum of the gradients given to v, G their sum over the row, h the entropy's.
// The few entries that tokens and alternatives name are formed again, with what is added, before they are rounded.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    token_logprobs_grad_kernel(Rows rows, const int64_t *__restrict__ tokens, int has_ignore, int64_t ignore, int top,
                               const float *__restrict__ kept, const float *__restrict__ entropy,
                               const int64_t *__restrict__ top_index, const float *__restrict__ g_logprob,
                               const float *__restrict__ g_entropy, const float *__restrict__ g_top, T *dlogits, int64_t pitch,
                               int *status) {
    constexpr int kVec = RowCut<T>::kVec;
    __shared__ int at[kMaxTop + 1];
    __shared__ float add[kMaxTop + 1];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int V = rows.V;
    const T *row = rows.at<T>(r);
    T *out = dlogits + r * pitch;
    const int64_t token = tokens[r];
    const bool left_out = has_ignore && token == ignore;
    const float m = kept[2 * r], log_s = kept[2 * r + 1];
    const bool bad = !left_out && g_logprob && (token < 0 || token >= V);
    if (bad && tid == 0) flag(status, PCFGNAT_STATUS_BAD_INDEX);
    if (tid <= kMaxTop) {
        int64_t index = -1;
        float g = 0.f;
        if (tid == 0 && g_logprob) index = token, g = g_logprob[r];
        if (tid > 0 && tid <= top && g_top) index = top_index[r * top + tid - 1], g = index < 0 ? 0.f : g_top[r * top + tid - 1];
        at[tid] = (int)index;
        add[tid] = g;
    }
    __syncthreads();
    float G = 0.f;
    for (int k = 0; k <= top; k++) G += add[k];
    if (bad) G = CUDART_NAN_F;
    const float h = g_entropy ? g_entropy[r] : 0.f, H = g_entropy ? entropy[r] : 0.f;
    const bool zero = left_out || log_s == neg_inf();  // not asked for, or nothing in it
    const float base = -G - h * H;
    const auto grad = [&](float x) {
        const float lp = max_nan((x - m) - log_s, kFarBelow);
        return exp2_approx(lp * kLog2e) * (base - h * lp);
    };
    const RowCut<T> cut(out, V);
    const bool same = !((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15);
    if (zero || same) {
        const uint4 *vec = reinterpret_cast<const uint4 *>(row + cut.head);
        uint4 *to = reinterpret_cast<uint4 *>(out + cut.head);
        for (int i = tid; i < cut.vecs; i += kThreads) {
            float x[kVec] = {};
            if (!zero) {
                unpack_vec<T, kVec>(__ldg(vec + i), x);
#pragma unroll
                for (int k = 0; k < kVec; k++) x[k] = grad(x[k]);
            }
            to[i] = pack_vec<T, kVec>(x);
        }
        if (tid < cut.loose(V)) {
            const int i = cut.loose_at(tid);
            out[i] = num_from_float<T>(zero ? 0.f : grad(num_to_float<T>(row[i])));
        }
    } else {
        for (int i = tid; i < V; i += kThreads) out[i] = num_from_float<T>(grad(num_to_float<T>(row[i])));
    }
    if (zero) return;
    __syncthreads();
    if (tid <= top && at[tid] >= 0 && at[tid] < V) {
        float g = 0.f;
        for (int k = 0; k <= top; k++) g += at[k] == at[tid] ? add[k] : 0.f;
        out[at[tid]] = num_from_float<T>(grad(num_to_float<T>(row[at[tid]])) + g);
    }
}

}  // namespace

int launch_token_logprobs(const void *logits, int dtype, int64_t n, int64_t inner, int64_t stride_outer, int64_t stride_inner, int V,
                          const int64_t *tokens, int has_ignore, int64_t ignore, int top, float *logprob, float *entropy,
                          float *top_logprob, int64_t *top_index, float *kept, int *status, cudaStream_t st) {
    if (n == 0) return PCFGNAT_OK;
    const Rows rows{logits, inner, stride_outer, stride_inner, V};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        token_logprobs_kernel<T><<<(unsigned)n, kThreads, 0, st>>>(rows, tokens, has_ignore, ignore, top, logprob, entropy,
                                                                   top_logprob, top_index, kept, status);
        return cuda_rc(cudaGetLastError());
    });
}

int launch_token_logprobs_grad(const void *logits, int dtype, int64_t n, int64_t inner, int64_t stride_outer, int64_t stride_inner,
                               int V, const int64_t *tokens, int has_ignore, int64_t ignore, int top, const float *kept,
                               const float *entropy, const int64_t *top_index, const float *g_logprob, const float *g_entropy,
                               const float *g_top, void *dlogits, int64_t pitch, int *status, cudaStream_t st) {
    if (n == 0) return PCFGNAT_OK;
    const Rows rows{logits, inner, stride_outer, stride_inner, V};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        token_logprobs_grad_kernel<T><<<(unsigned)n, kThreads, 0, st>>>(rows, tokens, has_ignore, ignore, top, kept, entropy, top_index,
                                                                        g_logprob, g_entropy, g_top, static_cast<T *>(dlogits), pitch,
                                                                        status);
        return cuda_rc(cudaGetLastError());
    });
}

}  // namespace pcfgnat
