// Element types of the operators that take fp32, bf16 and fp16 tensors (RE_F32 / RE_BF16 / RE_F16): conversions and 16-byte vectors.
#pragma once
#include "re_common.h"

typedef __bf16 re_bf16;
typedef _Float16 re_f16;

template <class T, int N>
struct alignas(sizeof(T) * N) re_vec {
    T e[N];
};

template <class T>
struct re_type;
template <>
struct re_type<float> {
    static constexpr int32_t CODE = RE_F32;
    static constexpr int VEC = 4;      // elements of a 16-byte load
};
template <>
struct re_type<re_bf16> {
    static constexpr int32_t CODE = RE_BF16;
    static constexpr int VEC = 8;
};
template <>
struct re_type<re_f16> {
    static constexpr int32_t CODE = RE_F16;
    static constexpr int VEC = 8;
};

static inline size_t re_dtype_size(int32_t t) { return t == RE_F32 ? 4 : (t == RE_BF16 || t == RE_F16) ? 2 : 0; }

// one element of a tensor whose type is known at run time only (weights, tables: a few loads a workgroup)
__device__ __forceinline__ float re_load_as_float(const void* p, int64_t i, int32_t dtype) {
    if (dtype == RE_F32) return static_cast<const float*>(p)[i];
    if (dtype == RE_BF16) return (float)static_cast<const re_bf16*>(p)[i];
    return (float)static_cast<const re_f16*>(p)[i];
}
__device__ __forceinline__ void re_store_float(void* p, int64_t i, int32_t dtype, float v) {
    if (dtype == RE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == RE_BF16) static_cast<re_bf16*>(p)[i] = (re_bf16)v;
    else static_cast<re_f16*>(p)[i] = (re_f16)v;
}

// VEC consecutive elements as floats (p aligned to VEC elements)
template <class T, int VEC>
__device__ __forceinline__ void re_load_vec(const T* p, float* f) {
    const re_vec<T, VEC> v = *reinterpret_cast<const re_vec<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = (float)v.e[i];
}
template <class T, int VEC>
__device__ __forceinline__ void re_store_vec(T* p, const float* f) {
    re_vec<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.e[i] = (T)f[i];
    *reinterpret_cast<re_vec<T, VEC>*>(p) = v;
}

// VEC consecutive elements that start on any element (the hardware takes the address as it is), as far as they lie below `left` elements
template <class T, int VEC, bool ALIGNED>
__device__ __forceinline__ void re_load_some(const T* p, int left, float* f) {
    if constexpr (ALIGNED) {
        re_load_vec<T, VEC>(p, f);
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) any {
            T e[VEC];
        };
        if (left >= VEC) {
            const any v = *reinterpret_cast<const any*>(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = (float)v.e[i];
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = i < left ? (float)p[i] : 0.f;
        }
    }
}
template <class T, int VEC, bool ALIGNED>
__device__ __forceinline__ void re_store_some(T* p, int left, const float* f) {
    if constexpr (ALIGNED) {
        re_store_vec<T, VEC>(p, f);
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) any {
            T e[VEC];
        };
        if (left >= VEC) {
            any v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v.e[i] = (T)f[i];
            *reinterpret_cast<any*>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < left) p[i] = (T)f[i];
        }
    }
}
