// Rows of float, half or bfloat16 numbers as 16-byte vectors, for the kernels over logits, the vocabulary table and gradients.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace pcfgnat {

template <typename T>
__device__ __forceinline__ float num_to_float(T v);
template <>
__device__ __forceinline__ float num_to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float num_to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float num_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T num_from_float(float v);
template <>
__device__ __forceinline__ float num_from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half num_from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 num_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// BYTES consecutive bytes of a row, held in registers.
template <int BYTES>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<2> { using type = uint16_t; };

template <typename T, int N>
__device__ __forceinline__ void unpack_vec(const typename RawVec<N * sizeof(T)>::type &raw, float (&x)[N]) {
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = num_to_float<T>(e[k]);
}
template <typename T, int N>
__device__ __forceinline__ typename RawVec<N * sizeof(T)>::type pack_vec(const float (&x)[N]) {
    typename RawVec<N * sizeof(T)>::type raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int k = 0; k < N; k++) e[k] = num_from_float<T>(x[k]);
    return raw;
}

// A row of n numbers cut into the numbers before the first 16-byte boundary, whole 16-byte vectors, and the rest.
template <typename T>
struct RowCut {
    static constexpr int kVec = 16 / sizeof(T);
    int head, vecs;
    __device__ __forceinline__ RowCut(const T *p, int n) {
        head = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
        head = head < n ? head : n;
        vecs = (n - head) / kVec;
    }
    __device__ __forceinline__ int loose(int n) const { return n - vecs * kVec; }              // numbers in no vector
    __device__ __forceinline__ int loose_at(int i) const { return i < head ? i : i + vecs * kVec; }  // where the i-th lies
};

// Maximum that keeps NaN, which fmaxf drops.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two floats for the packed instructions, each result rounded as by itself.
struct Packed {
    unsigned long long bits;
    __device__ __forceinline__ Packed(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(x), "f"(y)); }
    __device__ __forceinline__ Packed operator+(const Packed &o) const {
        Packed r = *this;
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(r.bits) : "l"(o.bits));
        return r;
    }
    __device__ __forceinline__ Packed operator*(const Packed &o) const {
        Packed r = *this;
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(r.bits) : "l"(o.bits));
        return r;
    }
    __device__ __forceinline__ float2 get() const {
        float2 v;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(bits));
        return v;
    }
};
__device__ __forceinline__ Packed fma(const Packed &a, const Packed &b, const Packed &c) {
    Packed r = a;
    asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(r.bits) : "l"(b.bits), "l"(c.bits));
    return r;
}

// The pair of numbers that begins at 32-bit word k: two halves of one word, or two words.
template <typename T>
__device__ __forceinline__ Packed pair_of_words(const uint32_t *word, int k) {
    if constexpr (sizeof(T) == 4) {
        return Packed(__uint_as_float(word[k]), __uint_as_float(word[k + 1]));
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        return Packed(__uint_as_float(word[k] << 16), __uint_as_float(word[k] & 0xffff0000u));
    } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(word + k));
        return Packed(v.x, v.y);
    }
}
// The largest number in N words; NaN if there is one.
template <typename T, int N>
__device__ __forceinline__ float max_of_words(const uint32_t *word) {
    uint32_t m = word[0];
#pragma unroll
    for (int k = 1; k < N; k++) {
        if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %0, %1;" : "+r"(m) : "r"(word[k]));
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(word[k]));
        else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(word[k]));
    }
    if constexpr (sizeof(T) == 4) return __uint_as_float(m);
    const float2 v = pair_of_words<T>(&m, 0).get();
    return max_nan(v.x, v.y);
}
template <typename T>
__device__ __forceinline__ uint32_t neg_inf_word() {
    return sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u : 0xfc00fc00u;
}

// Calls f with a value of the C++ type of a PCFGNAT_DTYPE_*.
template <class F>
inline int with_dtype(int dtype, F f) {
    switch (dtype) {
        case PCFGNAT_DTYPE_F32: return f(float());
        case PCFGNAT_DTYPE_F16: return f(__half());
        case PCFGNAT_DTYPE_BF16: return f(__nv_bfloat16());
    }
    return PCFGNAT_ERR_UNSUPPORTED;
}

}  // namespace pcfgnat
