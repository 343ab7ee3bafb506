// self-corr-pose_amd/csrc/layernorm_train.hip -- LayerNorm with gradients (ViT training), the residual add in front of it fused.
//
//   s = x + r (rounded to the storage type; s = x without a residual)      mu = mean_c s,  var = mean_c (s - mu)^2
//   y = (s - mu) rstd w + b,   rstd = 1 / sqrt(var + eps)
//   gx = rstd (g w - mean_c(g w) - xhat mean_c(g w xhat)) + gs,   xhat = (s - mu) rstd
//   gw = sum_rows g xhat,   gb = sum_rows g
//
// Bound by HBM: every row is read once per pass and stays in registers between the statistics and the output; the backward pass folds the
// column sums into the same pass.  A row belongs to TPR = 16, 64 or 256 lanes, the fewest that hold it with at most 32 elements per
// lane; sums over a row are butterflies inside the wavefront (plus 4 words of LDS for TPR = 256).  Mean and variance are two passes
// over the registers in 32 bits (no E[x^2] - E[x]^2 cancellation).
// Column sums: a workgroup strides over the rows with its gw / gb partials in registers, folds its row groups through LDS in a fixed
// order and writes one [2][C] partial; a second kernel adds the partials of all workgroups in order.  No atomics: bit-reproducible.
// Measured: 32800 x 384 fp32 with the residual add, forward 43 us and backward 45 + 4 us for 202 MB each (4.6 TB/s; a copy of that size 5.1);
// 8209 x 1001 bf16 14 and 22 + 4 us.
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;

constexpr int THREADS = 256;
constexpr int MAX_C = 8192;
constexpr int BWD_MAX_BLOCKS = 512;      // partials of the column sums: 2 workgroups per CU

template <int TPR> __device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
    for (int m = 1; m < (TPR < 64 ? TPR : 64); m <<= 1) v += __shfl_xor(v, m);
    if constexpr (TPR == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

// VEC weights from column c0 (NULL: all `fill`); columns past the end repeat the last one
template <typename W, int VEC> __device__ __forceinline__ void load_weights(const void* w, int c0, int C, float fill, float (&v)[VEC]) {
    constexpr int WV = VecIO<W>::VEC;
    const W* p = static_cast<const W*>(w);
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = fill;
    } else if (c0 + VEC <= C) {
        if constexpr (WV == VEC) {
            VecIO<W>::load(p + c0, v);
        } else {
#pragma unroll
            for (int h = 0; h < VEC / WV; h++) {
                float x[WV];
                VecIO<W>::load(p + c0 + h * WV, x);
#pragma unroll
                for (int i = 0; i < WV; i++) v[h * WV + i] = x[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = VecIO<W>::one(p + (c0 + i < C ? c0 + i : C - 1));
    }
}

struct NormArgs {
    const void *x, *resid, *gamma, *beta;
    void *sum, *y;
    float* stats;
    float eps;
    long rows;
    int C;
};

template <typename T, typename W, int TPR, int NCH> __global__ __launch_bounds__(THREADS) void layernorm_forward_kernel(const NormArgs a) {
    constexpr int VEC = VecIO<T>::VEC;
    __shared__ float lds[4];
    const int lane = threadIdx.x % TPR;
    const long row = (long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
    if (TPR < 256 && row >= a.rows) return;
    const int C = a.C;
    const T* xr = static_cast<const T*>(a.x) + (size_t)row * C;
    const T* rr = a.resid ? static_cast<const T*>(a.resid) + (size_t)row * C : nullptr;
    float v[NCH][VEC];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; j++) scp::load_chunk<T>(xr, lane + TPR * j, C, v[j]);
    if (rr) {
        T* so = static_cast<T*>(a.sum) + (size_t)row * C;
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            float r[VEC];
            scp::load_chunk<T>(rr, lane + TPR * j, C, r);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[j][i] = VecIO<T>::rounded(v[j][i] + r[i]);
            scp::store_chunk<T>(so, lane + TPR * j, C, v[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < NCH; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) s += v[j][i];
    const float mean = row_sum<TPR>(s, lds) / C;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float d = (lane + TPR * j) * VEC + i < C ? v[j][i] - mean : 0.f;
            q += d * d;
        }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, lds) / C + a.eps);
    if (a.stats && lane == 0) {
        a.stats[2 * row] = mean;
        a.stats[2 * row + 1] = rstd;
    }
    T* yr = static_cast<T*>(a.y) + (size_t)row * C;
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        float g[VEC], b[VEC];
        load_weights<W, VEC>(a.gamma, (lane + TPR * j) * VEC, C, 1.f, g);
        load_weights<W, VEC>(a.beta, (lane + TPR * j) * VEC, C, 0.f, b);
#pragma unroll
        for (int i = 0; i < VEC; i++) v[j][i] = (v[j][i] - mean) * rstd * g[i] + b[i];
        scp::store_chunk<T>(yr, lane + TPR * j, C, v[j]);
    }
}

struct NormGradArgs {
    const void *s, *gamma, *gy, *gsum;
    const float* stats;
    void* gx;            // may be NULL
    float *part_w, *part_b;      // column sums of each workgroup, `part_stride` floats apart (one workgroup: the results); NULL: not wanted
    long part_stride;
    long rows;
    int C;
};

template <typename T, typename W, int TPR, int NCH> __global__ __launch_bounds__(THREADS) void layernorm_backward_kernel(const NormGradArgs a) {
    constexpr int VEC = VecIO<T>::VEC, GROUPS = THREADS / TPR;
    constexpr int FOLD = TPR == 16 ? 4 : GROUPS;                    // row groups left after the in-wavefront fold of TPR = 16
    __shared__ float lds[4];
    __shared__ float fold[FOLD > 1 ? NCH * VEC * TPR : 1];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const int C = a.C;
    float w[NCH][VEC], gw[NCH][VEC], gb[NCH][VEC];
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        load_weights<W, VEC>(a.gamma, (lane + TPR * j) * VEC, C, 1.f, w[j]);
#pragma unroll
        for (int i = 0; i < VEC; i++) gw[j][i] = gb[j][i] = 0.f;
    }
    // the next row's x and gy are on their way while this one is worked on (a row past the end reads the last one again)
    const long stride = (long)gridDim.x * GROUPS;
    const T *sp = static_cast<const T*>(a.s), *gp = static_cast<const T*>(a.gy);
    float nx[NCH][VEC], ng[NCH][VEC], nmean, nrstd;
    auto fetch = [&](long row) {
        row = row < a.rows ? row : a.rows - 1;
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            scp::load_chunk<T>(sp + (size_t)row * C, lane + TPR * j, C, nx[j]);
            scp::load_chunk<T>(gp + (size_t)row * C, lane + TPR * j, C, ng[j]);
        }
        nmean = a.stats[2 * row];
        nrstd = a.stats[2 * row + 1];
    };
    fetch((long)blockIdx.x * GROUPS + group);
    for (long row0 = (long)blockIdx.x * GROUPS; row0 < a.rows; row0 += stride) {
        const long row = row0 + group;
        if (TPR < 256 && row >= a.rows) break;                     // the last row group(s) of the last stride; no barrier below for TPR < 256
        float x[NCH][VEC], g[NCH][VEC];
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                x[j][i] = nx[j][i];
                g[j][i] = ng[j][i];
            }
        const float mean = nmean, rstd = nrstd;
        fetch(row + stride);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                x[j][i] = (x[j][i] - mean) * rstd;                 // xhat; past the row's end g = 0 keeps every sum clean
                gb[j][i] += g[j][i];
                gw[j][i] += g[j][i] * x[j][i];
                g[j][i] *= w[j][i];
                s1 += g[j][i];
                s2 += g[j][i] * x[j][i];
            }
        if (a.gx) {
            s1 = row_sum<TPR>(s1, lds) / C;
            s2 = row_sum<TPR>(s2, lds) / C;
            T* gxr = static_cast<T*>(a.gx) + (size_t)row * C;
            const T* gs = a.gsum ? static_cast<const T*>(a.gsum) + (size_t)row * C : nullptr;
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                float e[VEC];
                if (gs) scp::load_chunk<T>(gs, lane + TPR * j, C, e);
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = rstd * (g[j][i] - s1 - x[j][i] * s2);
                    g[j][i] = gs ? d + e[i] : d;
                }
                scp::store_chunk<T>(gxr, lane + TPR * j, C, g[j]);
            }
        }
    }
    if (!a.part_w && !a.part_b) return;
    if constexpr (TPR == 16) {
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                gw[j][i] += __shfl_xor(gw[j][i], 16);
                gw[j][i] += __shfl_xor(gw[j][i], 32);
                gb[j][i] += __shfl_xor(gb[j][i], 16);
                gb[j][i] += __shfl_xor(gb[j][i], 32);
            }
    }
    const int folder = TPR == 16 ? threadIdx.x >> 6 : group;       // which of the FOLD partials this lane holds
    const bool mine = TPR != 16 || (threadIdx.x & 63) < 16;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* out = which ? a.part_b : a.part_w;
        if (!out) continue;
        out += blockIdx.x * a.part_stride;
        for (int f = 1; f < FOLD; f++) {                            // partial 0 += 1, 2, ...: a fixed order
            __syncthreads();
            if (folder == f && mine) {
#pragma unroll
                for (int j = 0; j < NCH; j++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) fold[(j * VEC + i) * TPR + lane] = which ? gb[j][i] : gw[j][i];
            }
            __syncthreads();
            if (folder == 0 && mine) {
#pragma unroll
                for (int j = 0; j < NCH; j++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) (which ? gb[j][i] : gw[j][i]) += fold[(j * VEC + i) * TPR + lane];
            }
        }
        if (folder == 0 && mine) {
#pragma unroll
            for (int j = 0; j < NCH; j++)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const int c = (lane + TPR * j) * VEC + i;
                    if (c < C) out[c] = which ? gb[j][i] : gw[j][i];
                }
        }
    }
}

// gw[c] = sum_b partial[b][0][c], gb[c] = sum_b partial[b][1][c]: 64 columns x 16 slices of the blocks per workgroup
constexpr int SLICES = 16;
__global__ __launch_bounds__(64 * SLICES) void layernorm_fold_kernel(const float* __restrict__ partial, int blocks, int C, float* gw, float* gb) {
    __shared__ float lds[SLICES][64];
    const int t = threadIdx.x & 63, col = blockIdx.x * 64 + t, slice = threadIdx.x >> 6;
    const int n = 2 * C;
    float s = 0.f;
    if (col < n) {
        const int per = (blocks + SLICES - 1) / SLICES, b0 = slice * per, b1 = min(blocks, b0 + per);
#pragma unroll 8
        for (int b = b0; b < b1; b++) s += partial[(size_t)b * n + col];
    }
    lds[slice][t] = s;
    __syncthreads();
    if (slice == 0 && col < n) {
        float r = 0.f;
#pragma unroll
        for (int i = 0; i < SLICES; i++) r += lds[i][t];
        if (col < C) { if (gw) gw[col] = r; } else { if (gb) gb[col - C] = r; }
    }
}

// One workgroup where it needs at most 5 rounds (of 16, 4 or 1 rows): no partials and no second launch, which cost an eager caller 6.5 us (85 x 384:
// forward + backward 58.5 us, with them 65).  A round is a memory round trip whatever the rows' width.  Kernels of forward + backward, 1 / 2 /
// 4 / 6 / 8 / 32 rounds, fp32, 64 channels: one workgroup 5.3 / 6.3 / 7.9 / 9.1 / 10.8 / 27 us, one per 16 rows 5.3 / 7.2 / 7.4 / 7.8 / 7.4 / 8.0;
// 384 channels 11.3 / 13.1 / 16.2 / 19.5 / 22.5 / 58 against 11.3 / 13.8 / 13.6 / 13.6 / 13.8 / 14.2.
int backward_blocks(long rows, int tpr) {
    const long groups = THREADS / tpr, need = (rows + groups - 1) / groups;
    if (need <= 5) return 1;
    return (int)(need < BWD_MAX_BLOCKS ? need : BWD_MAX_BLOCKS);
}
int lanes_per_row(int C) { return C <= 512 ? 16 : C <= 2048 ? 64 : 256; }

template <typename T, typename W, int TPR, int NCH> struct Launch {
    // a launch has fewer than 2^32 threads: more than 2^23 workgroups go out in several
    static void forward(const NormArgs& a, hipStream_t st) {
        constexpr long PER = THREADS / TPR, MOST = PER << 23;
        for (long row = 0; row < a.rows; row += MOST) {
            NormArgs part = a;
            const size_t at = (size_t)row * a.C;
            part.rows = a.rows - row < MOST ? a.rows - row : MOST;
            part.x = static_cast<const T*>(a.x) + at;
            if (a.resid) part.resid = static_cast<const T*>(a.resid) + at;
            if (a.sum) part.sum = static_cast<T*>(a.sum) + at;
            part.y = static_cast<T*>(a.y) + at;
            if (a.stats) part.stats = a.stats + 2 * row;
            hipLaunchKernelGGL((layernorm_forward_kernel<T, W, TPR, NCH>), dim3((unsigned)((part.rows + PER - 1) / PER)), dim3(THREADS), 0, st, part);
        }
    }
    static void backward(const NormGradArgs& a, hipStream_t st) {
        hipLaunchKernelGGL((layernorm_backward_kernel<T, W, TPR, NCH>), dim3(backward_blocks(a.rows, TPR)), dim3(THREADS), 0, st, a);
    }
};

// at most 32 elements per lane: NCH chunks of VEC; rounded up to the instantiated counts
template <typename T, typename W, int TPR, typename A> void by_chunks(int C, const A& a, hipStream_t st) {
    constexpr int VEC = VecIO<T>::VEC;
    const int n = (C + VEC * TPR - 1) / (VEC * TPR);
#define SCP_LN(NCH)                                                                                     \
    do {                                                                                                \
        if constexpr ((NCH) * VEC <= 32) {                                                              \
            if constexpr (__is_same(A, NormArgs)) Launch<T, W, TPR, NCH>::forward(a, st); \
            else Launch<T, W, TPR, NCH>::backward(a, st);                                               \
        }                                                                                               \
    } while (0)
    if (n <= 1) SCP_LN(1);
    else if (n <= 2) SCP_LN(2);
    else if (n <= 3) SCP_LN(3);
    else if (n <= 4) SCP_LN(4);
    else if (n <= 6) SCP_LN(6);
    else SCP_LN(8);
#undef SCP_LN
}
template <typename T, typename W, typename A> void by_lanes(int C, const A& a, hipStream_t st) {
    switch (lanes_per_row(C)) {
        case 16: by_chunks<T, W, 16>(C, a, st); break;
        case 64: by_chunks<T, W, 64>(C, a, st); break;
        default: by_chunks<T, W, 256>(C, a, st); break;
    }
}
template <typename A> void by_type(int dtype, int wdtype, int C, const A& a, hipStream_t st) {
    if (dtype == SCP_DTYPE_F32) by_lanes<float, float>(C, a, st);
    else if (wdtype == SCP_DTYPE_F32) by_lanes<__bf16, float>(C, a, st);
    else by_lanes<__bf16, __bf16>(C, a, st);
}

const char* bad_problem(long rows, int C, int dtype, int wdtype) {
    if (rows <= 0 || C <= 0) return "layernorm: empty problem";
    if (C > MAX_C) return "layernorm: more than 8192 channels";
    if (rows > (1ll << 31) - 1024) return "layernorm: more than 2^31 rows";
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return "layernorm: unknown type";
    if (wdtype != SCP_DTYPE_F32 && wdtype != dtype) return "layernorm: weight and bias must be fp32 or of the input's type";
    return nullptr;
}

}  // namespace

extern "C" int scp_layernorm_forward(const void* x, const void* resid, const void* gamma, const void* beta, float eps, long rows, int C,
                                     int dtype, int wdtype, void* sum_out, void* y, float* stats, void* stream) {
    if (const char* why = bad_problem(rows, C, dtype, wdtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!x || !y || (resid != nullptr) != (sum_out != nullptr))
        return scp::fail(hipErrorInvalidValue, "layernorm_forward: null argument, or residual without sum_out");
    const NormArgs a{x, resid, gamma, beta, sum_out, y, stats, eps, rows, C};
    by_type(dtype, wdtype, C, a, static_cast<hipStream_t>(stream));
    return scp::check_launch("layernorm_forward");
}

extern "C" size_t scp_layernorm_backward_workspace(long rows, int C) {
    if (rows <= 0 || C <= 0 || C > MAX_C) return 0;
    const int blocks = backward_blocks(rows, lanes_per_row(C));
    return blocks > 1 ? (size_t)blocks * 2 * C * sizeof(float) : 0;
}

extern "C" int scp_layernorm_backward(const void* s, const void* gamma, const void* gy, const void* gsum, const float* stats, long rows,
                                      int C, int dtype, int wdtype, void* gx, float* g_gamma, float* g_beta, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (const char* why = bad_problem(rows, C, dtype, wdtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!s || !gy || !stats) return scp::fail(hipErrorInvalidValue, "layernorm_backward: null argument");
    if (!gx && !g_gamma && !g_beta) return 0;
    const int blocks = backward_blocks(rows, lanes_per_row(C));
    const bool fold = blocks > 1 && (g_gamma || g_beta);
    if (fold && (!workspace || workspace_bytes < scp_layernorm_backward_workspace(rows, C)))
        return scp::fail(hipErrorInvalidValue, "layernorm_backward: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* part = static_cast<float*>(workspace);
    const NormGradArgs a{s, gamma, gy, gsum, stats, gx, fold ? part : g_gamma, fold ? part + C : g_beta, fold ? 2l * C : 0, rows, C};
    by_type(dtype, wdtype, C, a, st);
    if (const int e = scp::check_launch("layernorm_backward")) return e;
    if (fold) {
        hipLaunchKernelGGL(layernorm_fold_kernel, dim3((2 * C + 63) / 64), dim3(64 * SLICES), 0, st, part, blocks, C, g_gamma, g_beta);
        return scp::check_launch("layernorm_backward fold");
    }
    return 0;
}
