// self-corr-pose_amd/csrc/act8.hip -- activation checkpoints in 8 bits, and the GELU that uses one in its backward pass.
//
// Format: 32 neighbouring channels of a row share a power-of-two step 2^e with max|x| / 2^e in [64, 128); a code is x / 2^e rounded to the
// nearest integer (ties to even), clamped to +-127 (a value above 127.5 steps loses up to one step).  The step is at least 2^-126, so
// code * step is exact in fp32 and, the code having at most 7 bits, in bf16 too: what the backward pass multiplies with is exactly what
// the codes stand for.  Stored: one int8 per channel, and per group the step's exponent field (1..254); 0xFF marks a group that held an
// infinity or a NaN, and gives NaN back for all of it, so that a diverged activation still shows in the gradients.
//
//   gelu8:  y = x Phi(x);   gx = gy (Phi(x8) + x8 phi(x8)),  x8 = the checkpoint's value
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;
constexpr int GROUP = 32, THREADS = 256;

__device__ __forceinline__ int step_field(float amax) {                    // exponent field of the step; 255: not finite
    const int f = (int)(__float_as_uint(amax) >> 23);
    return f == 255 ? 255 : (f - 6 > 1 ? f - 6 : 1);
}
__device__ __forceinline__ float step_of(int field) { return __uint_as_float(field == 255 ? 0x7fc00000u : (unsigned)field << 23); }
__device__ __forceinline__ int code_of(float x, int field) {
    if (field == 255) return 0;
    // x / 2^(field - 127) = x 2^(127 - field): exact but for results below 2^-126, which round to code 0 either way
    const float q = rintf(ldexpf(x, 127 - field));
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ float gelu(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float gelu_slope(float x) {
    return 0.5f * (1.f + erff(x * 0.70710678118654752f)) + x * expf(-0.5f * x * x) * 0.39894228040143268f;
}

// a half-wavefront per group, a lane per channel
template <typename T, bool GELU> __global__ __launch_bounds__(THREADS) void pack8_kernel(const T* x, T* y, signed char* codes, unsigned char* exps,
                                                                                    long rows, int C, int groups) {
    const long total = rows * groups;
    const int l = threadIdx.x & 31;
    for (long g = (long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); g < total; g += (long)gridDim.x * (THREADS / 32)) {
        const long row = g / groups;
        const int gi = (int)(g - row * groups), c = gi * GROUP + l;
        const bool in = c < C;
        const float v = in ? VecIO<T>::one(x + row * C + c) : 0.f;
        unsigned m = __float_as_uint(fabsf(v));                            // integer order = magnitude order, NaN on top
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, k));
        const int field = step_field(__uint_as_float(m));
        if (codes && in) codes[row * C + c] = (signed char)code_of(v, field);
        if (exps && l == 0) exps[row * groups + gi] = (unsigned char)field;
        if constexpr (GELU)
            if (in) VecIO<T>::put(y + row * C + c, gelu(v));
    }
}
template <typename T, bool GELU> __global__ __launch_bounds__(THREADS) void unpack8_kernel(const signed char* codes, const unsigned char* exps, const T* gy,
                                                                                      T* out, long rows, int C, int groups) {
    const long total = rows * groups;
    const int l = threadIdx.x & 31;
    for (long g = (long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); g < total; g += (long)gridDim.x * (THREADS / 32)) {
        const long row = g / groups;
        const int gi = (int)(g - row * groups), c = gi * GROUP + l;
        if (c >= C) continue;
        const float v = (float)codes[row * C + c] * step_of(exps[row * groups + gi]);
        VecIO<T>::put(out + row * C + c, GELU ? VecIO<T>::one(gy + row * C + c) * gelu_slope(v) : v);
    }
}

unsigned grid_for(long rows, int groups) {
    const long need = (rows * groups + THREADS / 32 - 1) / (THREADS / 32);
    return (unsigned)(need < 16384 ? need : 16384);
}
const char* bad_problem(long rows, int C, int dtype) {
    if (rows <= 0 || C <= 0) return "act8: empty problem";
    if (C > (1 << 24)) return "act8: more than 2^24 channels";
    if (rows > (1ll << 62) / C) return "act8: problem too large";
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return "act8: unknown type";
    return nullptr;
}
template <typename T, bool GELU> void run_pack(const void* x, void* y, signed char* codes, unsigned char* exps, long rows, int C, hipStream_t st) {
    const int groups = (C + GROUP - 1) / GROUP;
    hipLaunchKernelGGL((pack8_kernel<T, GELU>), dim3(grid_for(rows, groups)), dim3(THREADS), 0, st, static_cast<const T*>(x), static_cast<T*>(y),
                       codes, exps, rows, C, groups);
}
template <typename T, bool GELU> void run_unpack(const signed char* codes, const unsigned char* exps, const void* gy, void* out, long rows, int C,
                                                 hipStream_t st) {
    const int groups = (C + GROUP - 1) / GROUP;
    hipLaunchKernelGGL((unpack8_kernel<T, GELU>), dim3(grid_for(rows, groups)), dim3(THREADS), 0, st, codes, exps, static_cast<const T*>(gy),
                       static_cast<T*>(out), rows, C, groups);
}

}  // namespace

extern "C" int scp_pack8(const void* x, long rows, int C, int dtype, signed char* codes, unsigned char* exps, void* stream) {
    if (const char* why = bad_problem(rows, C, dtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!x || !codes || !exps) return scp::fail(hipErrorInvalidValue, "pack8: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SCP_DTYPE_F32) run_pack<float, false>(x, nullptr, codes, exps, rows, C, st);
    else run_pack<__bf16, false>(x, nullptr, codes, exps, rows, C, st);
    return scp::check_launch("pack8");
}
extern "C" int scp_unpack8(const signed char* codes, const unsigned char* exps, long rows, int C, int dtype, void* x, void* stream) {
    if (const char* why = bad_problem(rows, C, dtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!x || !codes || !exps) return scp::fail(hipErrorInvalidValue, "unpack8: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SCP_DTYPE_F32) run_unpack<float, false>(codes, exps, nullptr, x, rows, C, st);
    else run_unpack<__bf16, false>(codes, exps, nullptr, x, rows, C, st);
    return scp::check_launch("unpack8");
}
extern "C" int scp_gelu8_forward(const void* x, long rows, int C, int dtype, void* y, signed char* codes, unsigned char* exps, void* stream) {
    if (const char* why = bad_problem(rows, C, dtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!x || !y || (codes != nullptr) != (exps != nullptr)) return scp::fail(hipErrorInvalidValue, "gelu8_forward: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SCP_DTYPE_F32) run_pack<float, true>(x, y, codes, exps, rows, C, st);
    else run_pack<__bf16, true>(x, y, codes, exps, rows, C, st);
    return scp::check_launch("gelu8_forward");
}
extern "C" int scp_gelu8_backward(const signed char* codes, const unsigned char* exps, const void* gy, long rows, int C, int dtype, void* gx,
                                  void* stream) {
    if (const char* why = bad_problem(rows, C, dtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!codes || !exps || !gy || !gx) return scp::fail(hipErrorInvalidValue, "gelu8_backward: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SCP_DTYPE_F32) run_unpack<float, true>(codes, exps, gy, gx, rows, C, st);
    else run_unpack<__bf16, true>(codes, exps, gy, gx, rows, C, st);
    return scp::check_launch("gelu8_backward");
}
