// block_types.h -- element types of the trainable block operators (block_kernels.hip, ffn_kernels.hip): fp32, bf16 and fp16 storage, fp32
// arithmetic; conversions round to nearest even.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum { IFF_DT_F32 = 0, IFF_DT_BF16 = 1, IFF_DT_F16 = 2 };      // include/iffnerf_hip.h IFF_TYPE_*

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// V consecutive elements of T as fp32, one 16-byte access (V = 16 / sizeof(T)) or element by element (V = 1)
template <class T, int V> struct Pack;
template <class T> struct Pack<T, 1> {
    static __device__ __forceinline__ void load(const T* p, float v[1]) { v[0] = (float)*p; }
    static __device__ __forceinline__ void store(T* p, const float v[1]) { *p = (T)v[0]; }
};
template <> struct Pack<float, 4> {
    static __device__ __forceinline__ void load(const float* p, float v[4]) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p);
        v[0] = t[0]; v[1] = t[1]; v[2] = t[2]; v[3] = t[3];
    }
    static __device__ __forceinline__ void store(float* p, const float v[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]}; }
};
template <class T, class T8> struct Pack8 {
    static __device__ __forceinline__ void load(const T* p, float v[8]) {
        const T8 t = *reinterpret_cast<const T8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
    }
    static __device__ __forceinline__ void store(T* p, const float v[8]) {
        T8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
        *reinterpret_cast<T8*>(p) = t;
    }
};
template <> struct Pack<__bf16, 8> : Pack8<__bf16, bf16x8> {};
template <> struct Pack<_Float16, 8> : Pack8<_Float16, f16x8> {};

// the same V elements as they are in memory
template <class T, int V> struct Raw;
template <class T> struct Raw<T, 1> {
    typedef T t;
    static __device__ __forceinline__ void unpack(T r, float v[1]) { v[0] = (float)r; }
};
template <> struct Raw<float, 4> {
    typedef f32x4 t;
    static __device__ __forceinline__ void unpack(f32x4 r, float v[4]) { v[0] = r[0]; v[1] = r[1]; v[2] = r[2]; v[3] = r[3]; }
};
template <class T8> struct Raw8 {
    typedef T8 t;
    static __device__ __forceinline__ void unpack(T8 r, float v[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
    }
};
template <> struct Raw<__bf16, 8> : Raw8<bf16x8> {};
template <> struct Raw<_Float16, 8> : Raw8<f16x8> {};

inline size_t dt_size(int dt) { return dt == IFF_DT_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
