// Vectors of V consecutive elements held in their stored type: 16 bytes where
// the row's alignment allows it, one element where it does not.
#pragma once

#include "common.cuh"

namespace tb {

template <typename T, int V>
struct RowVec;

template <>
struct RowVec<float, 4> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const float* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(w[i]); }
    static __device__ __forceinline__ void store(float* p, const float* v) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};

template <>
struct RowVec<__nv_bfloat16, 8> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ float get(int i) const { return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* v) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                  pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
};

template <>
struct RowVec<float, 1> {
    float f;
    __device__ __forceinline__ void load(const float* p) { f = *p; }
    __device__ __forceinline__ void zero() { f = 0.f; }
    __device__ __forceinline__ float get(int) const { return f; }
    static __device__ __forceinline__ void store(float* p, const float* v) { *p = v[0]; }
};

template <>
struct RowVec<__nv_bfloat16, 1> {
    uint16_t u;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint16_t*>(p); }
    __device__ __forceinline__ void zero() { u = 0; }
    __device__ __forceinline__ float get(int) const { return __uint_as_float((uint32_t)u << 16); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* v) { *p = __float2bfloat16_rn(v[0]); }
};

}  // namespace tb
