// self-corr-pose_amd/csrc/vec_io.h -- vector loads / stores of fp32 and bf16 rows as floats, at any element alignment.
// A chunk is 16 bytes (4 fp32 or 8 bf16).  Rows of an odd number of elements start at any 2- or 4-byte boundary; global memory takes
// 16-byte accesses at such addresses (unaligned access mode is on for every HSA process), so a chunk is one instruction either way.
#pragma once
#include <hip/hip_runtime.h>

namespace scp {

typedef unsigned u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T> struct VecIO;

template <> struct VecIO<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float rounded(float v) { return v; }
    static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
        const u32x4_a4 u = *reinterpret_cast<const u32x4_a4*>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __uint_as_float(u[i]);
    }
    static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
        u32x4_a4 u;
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __float_as_uint(v[i]);
        *reinterpret_cast<u32x4_a4*>(p) = u;
    }
};

template <> struct VecIO<__bf16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float one(const __bf16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(__bf16* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ float rounded(float v) { return (float)(__bf16)v; }      // round to nearest even
    static __device__ __forceinline__ void load(const __bf16* p, float (&v)[8]) {
        const u32x4_a2 u = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__bf16* p, const float (&v)[8]) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        u32x4_a2 u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bf16x2 w = {(__bf16)v[2 * i], (__bf16)v[2 * i + 1]};
            u[i] = __builtin_bit_cast(unsigned, w);
        }
        *reinterpret_cast<u32x4_a2*>(p) = u;
    }
};

// chunk c of a row of C elements: whole, or element by element where the row ends inside it (elements past the end read as zero)
template <typename T> __device__ __forceinline__ void load_chunk(const T* row, int c, int C, float (&v)[VecIO<T>::VEC]) {
    constexpr int VEC = VecIO<T>::VEC;
    const int c0 = c * VEC;
    if (c0 + VEC <= C) {
        VecIO<T>::load(row + c0, v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = c0 + i < C ? VecIO<T>::one(row + c0 + i) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store_chunk(T* row, int c, int C, const float (&v)[VecIO<T>::VEC]) {
    constexpr int VEC = VecIO<T>::VEC;
    const int c0 = c * VEC;
    if (c0 + VEC <= C) {
        VecIO<T>::store(row + c0, v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (c0 + i < C) VecIO<T>::put(row + c0 + i, v[i]);
    }
}

}  // namespace scp
