// self-corr-pose_amd/csrc/act8.hip -- activation checkpoints in 8 bits, and the GELU that uses one in its backward pass.
//
// Format: 32 neighbouring channels of a row share a power-of-two step 2^e with max|x| / 2^e in [64, 128); a code is x / 2^e rounded to the
// nearest integer (ties to even), clamped to +-127 (a value above 127.5 steps loses up to one step).  The step is at least 2^-126, so
// code * step is exact in fp32 and, the code having at most 7 bits, in bf16 too: what the backward pass multiplies with is exactly what
// the codes stand for.  Stored: one int8 per channel, and per group the step's exponent field (1..254); 0xFF marks a group that held an
// infinity or a NaN, and gives NaN back for all of it, so that a diverged activation still shows in the gradients.
//
//   gelu8:  y = x Phi(x);   gx = gy (Phi(x8) + x8 phi(x8)),  x8 = the checkpoint's value
//
// Bound by HBM (fp32 gelu8 forward: 4 + 4 + 1 1/32 bytes per value, backward the same).  A lane owns 8 channels, 4 lanes a group: the group's
// maximum is two cross-lane moves, everything else is per lane.  A thread has UNROLL independent pieces in flight.  Rows whose length is no
// multiple of 32 take the same kernel with a division per piece and a guarded last piece (FLAT = false); loads and stores need no
// alignment (vec_io.h).  Phi is Abramowitz & Stegun 7.1.26 (rational approximation of erf, |error| <= 1.5e-7): one reciprocal, one
// exponential -- shared with phi in the backward pass -- and 5 multiply-adds, so that bf16 streams too stay bound by memory.
// Measured: gelu8 of 32800 x 1536 fp32 87 us forward, 90 us backward (455 MB each, 5.1 TB/s: the rate of a copy); pack8 of the same 42 us.
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;
typedef unsigned u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));
constexpr int GROUP = 32, THREADS = 256, UNROLL = 2;

__device__ __forceinline__ int step_field(unsigned amax) {                 // exponent field of the step; 255: not finite
    const int f = (int)(amax >> 23);
    return f == 255 ? 255 : (f - 6 > 1 ? f - 6 : 1);
}
__device__ __forceinline__ float step_of(int field) { return __uint_as_float(field == 255 ? 0x7fc00000u : (unsigned)field << 23); }

// Phi(x) and exp(-x^2 / 2)
__device__ __forceinline__ float normal_cdf(float x, float& bell) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(x), 0.3275911f * 0.70710678118654752f, 1.f));
    bell = __builtin_amdgcn_exp2f(x * x * (-0.5f * 1.4426950408889634f));
    float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    q = __builtin_fmaf(t, q, 1.421413741f);
    q = __builtin_fmaf(t, q, -0.284496736f);
    q = __builtin_fmaf(t, q, 0.254829592f);
    q *= 0.5f * t * bell;                                                  // the tail beyond |x|
    return x > 0.f ? 1.f - q : q;
}
__device__ __forceinline__ float gelu(float x) {
    float bell;
    return x * normal_cdf(x, bell);
}
__device__ __forceinline__ float gelu_slope(float x) {
    float bell;
    const float c = normal_cdf(x, bell);
    return __builtin_fmaf(x * 0.39894228040143268f, bell, c);
}

// where 8-channel piece p lies: element offset, how many of its channels exist, group index; false past the end
struct Piece { long at, group; int n; };
template <bool FLAT> __device__ __forceinline__ bool piece_at(long p, long pieces, int C, int groups, Piece& o) {
    if (p >= pieces) return false;
    o.group = p >> 2;
    if (FLAT) {
        o.at = p * 8;
        o.n = 8;
        return true;
    }
    const long row = pieces <= 0x7fffffffl ? (long)((unsigned)o.group / (unsigned)groups) : o.group / groups;
    const int c = (int)(o.group - row * groups) * GROUP + 8 * (int)(p & 3);
    o.at = row * C + c;
    o.n = C - c < 8 ? (C - c > 0 ? C - c : 0) : 8;
    return true;
}
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if (n == 8) {
        if constexpr (sizeof(T) == 2) {
            VecIO<T>::load(p, v);
        } else {
            float lo[4], hi[4];
            VecIO<T>::load(p, lo);
            VecIO<T>::load(p + 4, hi);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = lo[i]; v[4 + i] = hi[i]; }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? VecIO<T>::one(p + i) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (n == 8) {
        if constexpr (sizeof(T) == 2) {
            VecIO<T>::store(p, v);
        } else {
            const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
            VecIO<T>::store(p, lo);
            VecIO<T>::store(p + 4, hi);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) VecIO<T>::put(p + i, v[i]);
    }
}

template <typename T, bool GELU, bool FLAT> __global__ __launch_bounds__(THREADS) void pack8_kernel(const T* x, T* y, signed char* codes, unsigned char* exps,
                                                                                               long pieces, int C, int groups) {
    const long stride = (long)gridDim.x * THREADS;
    for (long p0 = (long)blockIdx.x * THREADS + threadIdx.x; p0 < pieces; p0 += UNROLL * stride) {
        Piece at[UNROLL];
        bool in[UNROLL];
        float v[UNROLL][8];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            in[u] = piece_at<FLAT>(p0 + u * stride, pieces, C, groups, at[u]);
            if (in[u]) load8<T>(x + at[u].at, at[u].n, v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (!in[u]) continue;                                          // pieces of a group come and go together: `pieces` is a multiple of 4
            if (codes) {
                unsigned m = 0;                                            // integer order = magnitude order, NaN on top
#pragma unroll
                for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[u][i]) & 0x7fffffffu);
                m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));      // quad_perm [1,0,3,2]
                m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));      // quad_perm [2,3,0,1]
                const int field = step_field(m);
                // 1 / step is a normal power of two (field 1..248); x / step is exact but below 2^-126, where the code is 0 either way
                const float inv = __uint_as_float(field == 255 ? 0u : (unsigned)(254 - field) << 23);
                unsigned w[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    unsigned b[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // adding 1.5 2^23 leaves the nearest integer (ties to even) in the low bits, two's complement
                        const float c = fminf(fmaxf(v[u][4 * h + i] * inv, -127.f), 127.f);
                        b[i] = __float_as_uint(c + 12582912.f);
                    }
                    w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
                    if (field == 255) w[h] = 0;
                }
                if (at[u].n == 8) {
                    *reinterpret_cast<u32x2_a1*>(codes + at[u].at) = u32x2_a1{w[0], w[1]};
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (i < at[u].n) codes[at[u].at + i] = (signed char)(w[i >> 2] >> (8 * (i & 3)));
                }
                if (((p0 + u * stride) & 3) == 0) exps[at[u].group] = (unsigned char)field;
            }
            if constexpr (GELU) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] = gelu(v[u][i]);
                store8<T>(y + at[u].at, at[u].n, v[u]);
            }
        }
    }
}

template <typename T, bool GELU, bool FLAT> __global__ __launch_bounds__(THREADS) void unpack8_kernel(const signed char* codes, const unsigned char* exps,
                                                                                                 const T* gy, T* out, long pieces, int C, int groups) {
    const long stride = (long)gridDim.x * THREADS;
    for (long p0 = (long)blockIdx.x * THREADS + threadIdx.x; p0 < pieces; p0 += UNROLL * stride) {
        Piece at[UNROLL];
        bool in[UNROLL];
        float g[UNROLL][8];
        unsigned w[UNROLL][2];
        int field[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            in[u] = piece_at<FLAT>(p0 + u * stride, pieces, C, groups, at[u]);
            if (!in[u]) continue;
            w[u][0] = w[u][1] = 0;
            if (at[u].n == 8) {
                const u32x2_a1 c = *reinterpret_cast<const u32x2_a1*>(codes + at[u].at);
                w[u][0] = c[0];
                w[u][1] = c[1];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < at[u].n) w[u][i >> 2] |= (unsigned)(unsigned char)codes[at[u].at + i] << (8 * (i & 3));
            }
            field[u] = exps[at[u].group];
            if constexpr (GELU) load8<T>(gy + at[u].at, at[u].n, g[u]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (!in[u]) continue;
            const float step = step_of(field[u]);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = (float)(signed char)(w[u][i >> 2] >> (8 * (i & 3))) * step;
                if constexpr (GELU) v[i] = g[u][i] * gelu_slope(v[i]);
            }
            store8<T>(out + at[u].at, at[u].n, v);
        }
    }
}

const char* bad_problem(long rows, int C, int dtype) {
    if (rows <= 0 || C <= 0) return "act8: empty problem";
    if (C > (1 << 24)) return "act8: more than 2^24 channels";
    if (rows > (1ll << 62) / C) return "act8: problem too large";
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return "act8: unknown type";
    return nullptr;
}
// UNROLL pieces per thread, at most 32 workgroups per CU: beyond that a thread takes further pieces
unsigned grid_for(long pieces) {
    const long need = (pieces + THREADS * UNROLL - 1) / (THREADS * UNROLL);
    return (unsigned)(need < 8192 ? need : 8192);
}
template <typename T, bool GELU> void run_pack(const void* x, void* y, signed char* codes, unsigned char* exps, long rows, int C, hipStream_t st) {
    const int groups = (C + GROUP - 1) / GROUP;
    const long pieces = rows * groups * 4;
    const dim3 grid(grid_for(pieces));
    if (C % GROUP == 0)
        hipLaunchKernelGGL((pack8_kernel<T, GELU, true>), grid, dim3(THREADS), 0, st, static_cast<const T*>(x), static_cast<T*>(y), codes, exps, pieces, C, groups);
    else
        hipLaunchKernelGGL((pack8_kernel<T, GELU, false>), grid, dim3(THREADS), 0, st, static_cast<const T*>(x), static_cast<T*>(y), codes, exps, pieces, C, groups);
}
template <typename T, bool GELU> void run_unpack(const signed char* codes, const unsigned char* exps, const void* gy, void* out, long rows, int C,
                                                 hipStream_t st) {
    const int groups = (C + GROUP - 1) / GROUP;
    const long pieces = rows * groups * 4;
    const dim3 grid(grid_for(pieces));
    if (C % GROUP == 0)
        hipLaunchKernelGGL((unpack8_kernel<T, GELU, true>), grid, dim3(THREADS), 0, st, codes, exps, static_cast<const T*>(gy), static_cast<T*>(out), pieces, C, groups);
    else
        hipLaunchKernelGGL((unpack8_kernel<T, GELU, false>), grid, dim3(THREADS), 0, st, codes, exps, static_cast<const T*>(gy), static_cast<T*>(out), pieces, C, groups);
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
