// bssm_io.cuh -- element types and packed sequences of the operators that take
// float32, bfloat16 and float16 rows (causal convolution, selective scan,
// distillation).  Everything is widened to float32 on load and rounded once on
// store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "bayes_ssm_b200.h"

namespace bssm {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Elements of parameters (weights, biases) keep their own type: element i of
// an array whose type is a BSSM_* code.
__device__ __forceinline__ float load_as_float(const void *p, int dtype, long i) {
    if (dtype == BSSM_F32) return static_cast<const float *>(p)[i];
    if (dtype == BSSM_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void *p, int dtype, long i, float v) {
    if (dtype == BSSM_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == BSSM_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}

__host__ __device__ constexpr bool io_dtype_known(int dtype) {
    return dtype == BSSM_F32 || dtype == BSSM_BF16 || dtype == BSSM_F16;
}

// VEC consecutive elements as float32, in one access when VEC * sizeof(T) <= 16
// (the address must then be a multiple of that), else in 16-byte accesses.
template <typename T, int VEC> constexpr int packed_alignment() {
    constexpr int bytes = VEC * static_cast<int>(sizeof(T));
    return (VEC & (VEC - 1)) != 0 ? static_cast<int>(sizeof(T)) : bytes < 16 ? bytes : 16;
}
template <typename T, int VEC> struct alignas(packed_alignment<T, VEC>()) Packed {
    T e[VEC];
};
template <typename T, int VEC> __device__ __forceinline__ void widen(const Packed<T, VEC> &p, float (&o)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = to_float(p.e[i]);
}
template <typename T, int VEC> __device__ __forceinline__ Packed<T, VEC> load_packed(const T *p) {
    return *reinterpret_cast<const Packed<T, VEC> *>(p);
}
template <typename T, int VEC> __device__ __forceinline__ void store_packed(T *p, const float (&v)[VEC]) {
    Packed<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.e[i] = from_float<T>(v[i]);
    *reinterpret_cast<Packed<T, VEC> *>(p) = o;
}

// VEC elements between their load and their use, as whole 32-bit registers.
// (As 16-bit variables the compiler takes them apart right behind the load,
// which then waits there instead of running on under other work.)  VEC is a
// power of two and the address a multiple of min(16, VEC * sizeof(T)).
template <typename T, int VEC> struct RawVec {
    static constexpr int kWords = (VEC * static_cast<int>(sizeof(T)) + 3) / 4;
    unsigned w[kWords];

    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC * sizeof(T) == 2) {
            w[0] = *reinterpret_cast<const unsigned short *>(p);
        } else if constexpr (kWords == 1) {
            w[0] = *reinterpret_cast<const unsigned *>(p);
        } else if constexpr (kWords == 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x; w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned *>(p) + i);
                w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return __uint_as_float(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
        else {
            const unsigned bits = i % 2 == 0 ? w[i / 2] & 0xffffu : w[i / 2] >> 16;
            return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        }
    }
    __device__ __forceinline__ void values(float (&o)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = value(i);
    }
    // The largest (a NaN gives way to a number); 16-bit types two at a time.
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4 || VEC == 1) {
            float m = value(0);
#pragma unroll
            for (int i = 1; i < VEC; ++i) m = fmaxf(m, value(i));
            return m;
        } else {
            using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
            T2 m = *reinterpret_cast<const T2 *>(&w[0]);
#pragma unroll
            for (int i = 1; i < kWords; ++i) m = __hmax2(m, *reinterpret_cast<const T2 *>(&w[i]));
            return fmaxf(to_float(m.x), to_float(m.y));
        }
    }
};

// expf rather than __expf: the latter rounds x log2 e to float32 first, which
// costs |x| 2^-24 of the result.
__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.f, 1.f + expf(-x)); }

// The sequences in the token rows: `count` runs of `length` tokens each, or,
// with offsets (count + 1 int64 values from 0 to tokens, never decreasing),
// run s from offsets[s] to offsets[s + 1].  Bounds are clamped to the rows
// there are, so offsets outside the contract read nothing out of range.
struct Sequences {
    const long *offsets;
    long count, length, tokens;

    __device__ __forceinline__ long begin(long s) const {
        if (offsets == nullptr) return s * length;
        const long o = offsets[s];
        return o < 0 ? 0 : (o > tokens ? tokens : o);
    }
    __device__ __forceinline__ long end(long s) const { return offsets == nullptr ? (s + 1) * length : begin(s + 1); }
    // The sequence that holds token row g (g < tokens).
    __device__ __forceinline__ long find(long g) const {
        if (offsets == nullptr) return g / length;
        long lo = 0, hi = count;  // offsets[lo] <= g < offsets[hi]
        while (hi - lo > 1) {
            const long mid = (lo + hi) / 2;
            if (offsets[mid] <= g) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

}  // namespace bssm
