// Element types of maps, rows and their gradients, shared by the loss and norm kernels.
#pragma once
#include "od_common.h"

namespace od {

typedef float vec4f __attribute__((ext_vector_type(4)));

// Element types of the head outputs and of their gradients: fp32, or the 16-bit types a head produces under autocast
// (the reference trains with use_amp, reference object_detection/configs/config_all.py:16, train.py:61).  All
// arithmetic is fp32; a 16-bit gradient is rounded once, to nearest even.
struct bf16_t { unsigned short bits; };
template <typename T> struct Elem;
template <> struct Elem<float> {
    typedef vec4f V;
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
    static __device__ __forceinline__ float4 unpack(V v) { return make_float4(v.x, v.y, v.z, v.w); }
    static __device__ __forceinline__ V pack(float4 f) { V v; v.x = f.x; v.y = f.y; v.z = f.z; v.w = f.w; return v; }
};
template <> struct Elem<_Float16> {
    typedef _Float16 V __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 from_float(float v) { return (_Float16)v; }
    static __device__ __forceinline__ float4 unpack(V v) { return make_float4((float)v.x, (float)v.y, (float)v.z, (float)v.w); }
    static __device__ __forceinline__ V pack(float4 f) {
        V v; v.x = (_Float16)f.x; v.y = (_Float16)f.y; v.z = (_Float16)f.z; v.w = (_Float16)f.w; return v;
    }
};
template <> struct Elem<bf16_t> {
    typedef unsigned short V __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ float up(unsigned short h) { return u2f((uint32_t)h << 16); }
    static __device__ __forceinline__ unsigned short down(float f) {
        const uint32_t u = f2u(f);
        if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40u);      // NaN stays NaN
        return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
    static __device__ __forceinline__ float to_float(bf16_t v) { return up(v.bits); }
    static __device__ __forceinline__ bf16_t from_float(float v) { bf16_t r; r.bits = down(v); return r; }
    static __device__ __forceinline__ float4 unpack(V v) { return make_float4(up(v.x), up(v.y), up(v.z), up(v.w)); }
    static __device__ __forceinline__ V pack(float4 f) { V v; v.x = down(f.x); v.y = down(f.y); v.z = down(f.z); v.w = down(f.w); return v; }
};

// VEC consecutive elements from / to memory, as fp32 in registers.  The address is a multiple of VEC elements.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// two fp32 values to a pair of 16-bit ones, nearest even (one instruction on gfx950 for bf16)
__device__ __forceinline__ uint32_t pack2(float a, float b, const bf16_t*) {
    f32x2 f; f.x = a; f.y = b;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const _Float16*) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 h; h.x = (_Float16)a; h.y = (_Float16)b;
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, const bf16_t*) {
    a = u2f(w << 16);
    b = u2f(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, const _Float16*) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = __builtin_bit_cast(h2, w);
    a = (float)h.x;
    b = (float)h.y;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
    if constexpr (VEC == 1) {
        f[0] = Elem<T>::to_float(*p);
    } else if constexpr (sizeof(T) == 4) {
        static_assert(VEC == 4, "fp32 vectors hold four elements");
        const vec4f v = *reinterpret_cast<const vec4f*>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else if constexpr (VEC == 4) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(p);
        unpack2(v.x, f[0], f[1], (const T*)nullptr);
        unpack2(v.y, f[2], f[3], (const T*)nullptr);
    } else {
        static_assert(VEC == 8, "16-bit vectors hold eight or four elements");
        const u32x4 v = *reinterpret_cast<const u32x4*>(p);
        unpack2(v.x, f[0], f[1], (const T*)nullptr);
        unpack2(v.y, f[2], f[3], (const T*)nullptr);
        unpack2(v.z, f[4], f[5], (const T*)nullptr);
        unpack2(v.w, f[6], f[7], (const T*)nullptr);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
    if constexpr (VEC == 1) {
        *p = Elem<T>::from_float(f[0]);
    } else if constexpr (sizeof(T) == 4) {
        vec4f v; v.x = f[0]; v.y = f[1]; v.z = f[2]; v.w = f[3];
        *reinterpret_cast<vec4f*>(p) = v;
    } else if constexpr (VEC == 4) {
        u32x2 v;
        v.x = pack2(f[0], f[1], (const T*)nullptr);
        v.y = pack2(f[2], f[3], (const T*)nullptr);
        *reinterpret_cast<u32x2*>(p) = v;
    } else {
        u32x4 v;
        v.x = pack2(f[0], f[1], (const T*)nullptr);
        v.y = pack2(f[2], f[3], (const T*)nullptr);
        v.z = pack2(f[4], f[5], (const T*)nullptr);
        v.w = pack2(f[6], f[7], (const T*)nullptr);
        *reinterpret_cast<u32x4*>(p) = v;
    }
}

}  // namespace od
