// self-corr-pose_amd/csrc/act8_wgrad.hip -- weight and bias gradient of a linear layer from the 8-bit checkpoint of its input.
//
//   gw[n][k] = sum_m gy[m][n] x8[m][k],   gb[n] = sum_m gy[m][n],   x8 = code * step (csrc/act8.hip)
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;

// a 16 x 16 tile of gw per workgroup, a thread per element; 16 rows of gy and x8 at a time through LDS
template <typename T> __global__ __launch_bounds__(256) void wgrad8_kernel(const T* gy, const signed char* codes, const unsigned char* exps, long M, int N,
                                                                          int K, float* gw, float* gb) {
    __shared__ float a[16][17], b[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int n0 = blockIdx.y * 16, k0 = blockIdx.x * 16, groups = (K + 31) / 32;
    float acc = 0.f, bias = 0.f;
    for (long m0 = 0; m0 < M; m0 += 16) {
        const long m = m0 + ty;
        const int n = n0 + tx, k = k0 + tx;
        a[ty][tx] = m < M && n < N ? VecIO<T>::one(gy + m * N + n) : 0.f;
        float v = 0.f;
        if (m < M && k < K) {
            const unsigned e = exps[m * groups + k / 32];
            v = (float)codes[m * K + k] * __uint_as_float(e == 255 ? 0x7fc00000u : e << 23);
        }
        b[ty][tx] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i++) {
            acc += a[i][ty] * b[i][tx];
            bias += a[i][ty];
        }
        __syncthreads();
    }
    const int n = n0 + ty, k = k0 + tx;
    if (n < N && k < K) gw[(size_t)n * K + k] = acc;
    if (gb && blockIdx.x == 0 && tx == 0 && n < N) gb[n] = bias;
}

}  // namespace

extern "C" size_t scp_weight_grad8_workspace(long M, int N, int K, int dtype) { return 0; }

extern "C" int scp_weight_grad8(const void* gy, const signed char* codes, const unsigned char* exps, long M, int N, int K, int dtype, float* gw,
                                float* gb, void* workspace, size_t workspace_bytes, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0) return scp::fail(hipErrorInvalidValue, "weight_grad8: empty problem");
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return scp::fail(hipErrorInvalidValue, "weight_grad8: unknown type");
    if (!gy || !codes || !exps || !gw) return scp::fail(hipErrorInvalidValue, "weight_grad8: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((K + 15) / 16, (N + 15) / 16);
    if (dtype == SCP_DTYPE_F32)
        hipLaunchKernelGGL(wgrad8_kernel<float>, grid, dim3(256), 0, st, static_cast<const float*>(gy), codes, exps, M, N, K, gw, gb);
    else
        hipLaunchKernelGGL(wgrad8_kernel<__bf16>, grid, dim3(256), 0, st, static_cast<const __bf16*>(gy), codes, exps, M, N, K, gw, gb);
    return scp::check_launch("weight_grad8");
}
