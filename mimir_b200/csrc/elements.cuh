// Runs of F32 or BF16 elements as f32 values: VEC of them at once, 8 from 16-byte boundaries, or one. Ordinary loads (kernels of `launch_after`).
#pragma once

#include "common.cuh"

namespace mimk {

#ifdef __CUDACC__

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// What a load brings, before it is taken apart: loads of several runs can be under way in few registers.
template <class T, int VEC>
struct Run;
template <>
struct Run<float, 8> {
    uint4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4); }
    __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<uint4*>(p) = a, *reinterpret_cast<uint4*>(p + 4) = b; }
    __device__ __forceinline__ void clear() { a = b = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
    }
};
template <>
struct Run<__nv_bfloat16, 8> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = a; }
    __device__ __forceinline__ void clear() { a = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = bf16_low(a.x), v[1] = bf16_high(a.x), v[2] = bf16_low(a.y), v[3] = bf16_high(a.y);
        v[4] = bf16_low(a.z), v[5] = bf16_high(a.z), v[6] = bf16_low(a.w), v[7] = bf16_high(a.w);
    }
};
template <>
struct Run<float, 1> {
    float a;
    __device__ __forceinline__ void load(const float* p) { a = *p; }
    __device__ __forceinline__ void store(float* p) const { *p = a; }
    __device__ __forceinline__ void clear() { a = 0.f; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = a; }
};
template <>
struct Run<__nv_bfloat16, 1> {
    uint16_t a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint16_t*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint16_t*>(p) = a; }
    __device__ __forceinline__ void clear() { a = 0; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = __uint_as_float(uint32_t(a) << 16); }
};

__device__ __forceinline__ void put(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p)     = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void put(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void put(float* p, const float (&v)[1]) { *p = v[0]; }
__device__ __forceinline__ void put(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }

#endif

}  // namespace mimk
