// self-corr-pose_amd/csrc/act8_wgrad.hip -- weight and bias gradient of a linear layer from the 8-bit checkpoint of its input.
//
//   gw[n][k] = sum_m gy[m][n] x8[m][k],   gb[n] = sum_m gy[m][n],   x8 = code * step (csrc/act8.hip)
//
// A matrix product whose reduction runs over the ROWS of both operands, on v_mfma_f32_32x32x16_bf16.  x8 is exact in bf16 and bf16 gy is what
// it is, so every product is exact and only the fp32 accumulation rounds; fp32 gy is cut into three bf16 parts of 8 bits each
// (gy = h + m + l exactly) and multiplied part by part: 3 matrix instructions for 1, still 5 times the rate of the fp32 cores.
//   * a workgroup owns a BN x 128 tile of gw over a range of rows and walks it 32 rows at a time: gy and the codes go global -> registers one
//     step ahead, are cut / dequantised there (once per tile, not per wavefront) and written to LDS row-major; ds_read_b64_tr_b16 turns
//     4 rows x 16 columns into operand order, the same row order for both operands, so no transposition is ever stored;
//   * LDS rows are swizzled in 16-byte chunks so that the 4 rows x 4 chunks of half a transposed read touch each bank once;
//   * a wavefront owns (BN / 2) x 64 of the tile.  BN = 256 for bf16 (12 KiB of LDS reads per 16 matrix instructions), 128 for fp32, where
//     the three parts share the x8 operand;
//   * a workgroup has two teams of four wavefronts, which take alternate steps of its rows and join their tiles through LDS at the end: two
//     wavefronts per SIMD at half the partial tiles that two workgroups per CU would write (33 MB for 1536 x 384, not 66);
//   * the rows are split so that about one workgroup per CU runs; each writes an fp32 partial tile and a second kernel adds the partials in
//     order (bit-reproducible).  gb falls out of the registers of the workgroups of the first column of tiles.
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

constexpr int BK = 128, STEP = 32, TEAM = 256, TEAMS = 2, THREADS = TEAM * TEAMS;

struct Wgrad8Args {
    const void* gy;
    const signed char* codes;
    const unsigned char* exps;
    float *gw, *gb;              // the results, or [splits] partials of them
    long M;
    int N, K, tiles_n, tiles_k, splits;
    long rows_per_split;         // a multiple of STEP
};

// element offset of (row, 16-byte chunk) in a [32][COLS] bf16 tile
template <int COLS> __device__ __forceinline__ int lds_at(int row, int chunk) {
    return row * COLS + 8 * (chunk ^ (((row & 3) << 2) | ((row >> 2) & 3)));
}
// columns c0 .. c0+31 (one per lane & 31), rows 16 s + {4 half + 0..3, 8 + 4 half + 0..3}
template <int COLS> __device__ __forceinline__ bf16x8 operand(const __bf16* t, int s, int c0) {
    const int lane = threadIdx.x & 63, i = lane & 15, half = lane >> 5, cg = (lane >> 4) & 1;
    bf16x4 h[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const __bf16* at = t + lds_at<COLS>(16 * s + 8 * u + 4 * half + (i >> 2), c0 / 8 + 2 * cg + ((i & 3) >> 1)) + 4 * (i & 1);
        h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)at);
    }
    return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// the 16 bytes of x from byte `shift` on (what follows them is of no account)
__device__ __forceinline__ u32x4 from_byte(u32x4 x, int shift) {
    const bool two = shift & 8, one = shift & 4;
    u32x4 y = {two ? x[2] : x[0], two ? x[3] : x[1], x[2], x[3]};
    u32x4 z = {one ? y[1] : y[0], one ? y[2] : y[1], one ? y[3] : y[2], y[3]};
#pragma unroll
    for (int i = 0; i < 3; i++) z[i] = __builtin_amdgcn_alignbyte(z[i + 1], z[i], shift & 3);
    z[3] >>= 8 * (shift & 3);
    return z;
}

template <typename T> struct Wgrad8Shape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BN = F32 ? 128 : 256, PARTS = F32 ? 3 : 1;
    static constexpr int E = 16 / sizeof(T);                              // gy elements per 16 bytes
    static constexpr int CPR = BN / E;                                    // 16-byte pieces of gy per row of the tile: 32 either way
    static constexpr int PIECES = STEP * CPR / TEAM;                   // 4 per thread
    static constexpr int NB = BN / 64;                                    // 32-column blocks of n per wavefront
};

// RAGGED: rows of gy or of the codes are no whole number of 16-byte pieces, or not aligned to them
template <typename T, bool RAGGED> __global__ __launch_bounds__(THREADS, 2) void wgrad8_kernel(const Wgrad8Args a) {
    typedef Wgrad8Shape<T> S;
    constexpr int BN = S::BN, PARTS = S::PARTS, NB = S::NB;
    struct Stage { __bf16 g[2][PARTS][STEP * BN], x[2][STEP * BK]; };
    __shared__ __attribute__((aligned(16))) Stage stage[TEAMS];

    // tiles of one range of rows next to each other on one XCD: they read the same rows of gy and of the codes
    const int tiles = a.tiles_n * a.tiles_k, total = tiles * a.splits, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= total || (blockIdx.x >> 3) >= (unsigned)per) return;
    const int split = id / tiles, tile = id - split * tiles, tn = tile / a.tiles_k, tk = tile - tn * a.tiles_k;
    const int n0 = tn * BN, k0 = tk * BK;
    const long m_beg = split * a.rows_per_split, m_end = m_beg + a.rows_per_split < a.M ? m_beg + a.rows_per_split : a.M;

    const int tid = threadIdx.x & (TEAM - 1), team = __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l31 = lane & 31;
    const int wn = (wave >> 1) * (BN / 2), wk = (wave & 1) * 64;
    auto& gbuf = stage[team].g;
    auto& xbuf = stage[team].x;
    const int groups = (a.K + 31) / 32;

    // loads: gy piece i of this thread = row tid / 32 + 8 i, elements E (tid % 32); codes = row tid / 8, 16 of them.  Pieces past a row's end
    // are read from its end instead and moved into place (RAGGED); what stands behind them, and in pieces past the matrix, goes into
    // products that nobody stores.  Rows past the range are read from its last row and stored as zeros.
    const char* gy = static_cast<const char*>(a.gy);
    const int g_row = tid / S::CPR, g_col = n0 + S::E * (tid % S::CPR);
    const int x_row = tid >> 3, x_col = k0 + 16 * (tid & 7);
    const int g_at = min(g_col, a.N - S::E), x_at = min(x_col, a.K - 16);
    const int g_shift = min(g_col - g_at, S::E - 1) * (int)sizeof(T), x_shift = min(x_col - x_at, 15);
    const int e_at = min(x_col >> 5, groups - 1);
    u32x4 graw[S::PIECES], xraw;
    unsigned xexp;
    auto load = [&](long m) {
        const int last = m_end - m < STEP ? (int)(m_end - m) - 1 : STEP - 1;
        const char* gbase = gy + m * a.N * (long)sizeof(T);
        const char* xbase = reinterpret_cast<const char*>(a.codes) + m * a.K;
        const char* ebase = reinterpret_cast<const char*>(a.exps) + m * groups;
#pragma unroll
        for (int i = 0; i < S::PIECES; i++) {
            const unsigned off = (unsigned)(min(g_row + (TEAM / S::CPR) * i, last) * a.N + g_at) * (unsigned)sizeof(T);
            if constexpr (RAGGED) graw[i] = *reinterpret_cast<const u32x4_a1*>(gbase + off);
            else graw[i] = *reinterpret_cast<const u32x4*>(gbase + off);
        }
        const int r = min(x_row, last);
        if constexpr (RAGGED) xraw = *reinterpret_cast<const u32x4_a1*>(xbase + (unsigned)(r * a.K + x_at));
        else xraw = *reinterpret_cast<const u32x4*>(xbase + (unsigned)(r * a.K + x_at));
        xexp = *reinterpret_cast<const unsigned char*>(ebase + (unsigned)(r * groups + e_at));
    };
    const bool bias = a.gb && tk == 0;
    float bsum[S::E];
#pragma unroll
    for (int i = 0; i < S::E; i++) bsum[i] = 0.f;
    auto store = [&](int buf, long m) {
        if constexpr (RAGGED) {
#pragma unroll
            for (int i = 0; i < S::PIECES; i++) graw[i] = from_byte(graw[i], g_shift);
            xraw = from_byte(xraw, x_shift);
        }
        if (m + STEP > m_end) {
            const int rows = (int)(m_end - m);
#pragma unroll
            for (int i = 0; i < S::PIECES; i++)
                if (g_row + (TEAM / S::CPR) * i >= rows) graw[i] = u32x4{};
            if (x_row >= rows) {
                xraw = u32x4{};
                xexp = 1;
            }
        }
#pragma unroll
        for (int i = 0; i < S::PIECES; i++) {
            const int row = g_row + (TEAM / S::CPR) * i, col = S::E * (tid % S::CPR);
            if constexpr (S::F32) {
                unsigned h[4], m[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {                            // 8 + 8 + 8 bits: h + m + l = gy exactly
                    const float x = __uint_as_float(graw[i][e]);
                    h[e] = graw[i][e] & 0xffff0000u;
                    const float rest = x - __uint_as_float(h[e]);
                    m[e] = __float_as_uint(rest) & 0xffff0000u;
                    l[e] = __float_as_uint(rest - __uint_as_float(m[e]));
                    if (bias) bsum[e] += x;
                }
                const int at = lds_at<BN>(row, col / 8) + (col & 7);
                *reinterpret_cast<u32x2*>(&gbuf[buf][0][at]) = u32x2{upper_halves(h[0], h[1]), upper_halves(h[2], h[3])};
                *reinterpret_cast<u32x2*>(&gbuf[buf][1 % PARTS][at]) = u32x2{upper_halves(m[0], m[1]), upper_halves(m[2], m[3])};
                *reinterpret_cast<u32x2*>(&gbuf[buf][2 % PARTS][at]) = u32x2{upper_halves(l[0], l[1]), upper_halves(l[2], l[3])};
            } else {
                *reinterpret_cast<u32x4*>(&gbuf[buf][0][lds_at<BN>(row, col / 8)]) = graw[i];
                if (bias) {
#pragma unroll
                    for (int e = 0; e < 8; e++) bsum[e % S::E] += __uint_as_float(e & 1 ? graw[i][e / 2] & 0xffff0000u : graw[i][e / 2] << 16);
                }
            }
        }
        const float step = __uint_as_float(xexp == 255 ? 0x7fc00000u : xexp << 23);
        u32x4 x[2];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (float)(signed char)(xraw[w] >> (8 * e)) * step;
            x[w >> 1][2 * (w & 1)] = upper_halves(__float_as_uint(v[0]), __float_as_uint(v[1]));
            x[w >> 1][2 * (w & 1) + 1] = upper_halves(__float_as_uint(v[2]), __float_as_uint(v[3]));
        }
#pragma unroll
        for (int w = 0; w < 2; w++) *reinterpret_cast<u32x4*>(&xbuf[buf][lds_at<BK>(x_row, 2 * (tid & 7) + w)]) = x[w];
    };

    f32x16 acc[NB][2];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f32x16{};

    // the teams' steps alternate; both pass every barrier, a team without a step left does nothing between them
    const int steps = (int)((m_end - m_beg + STEP - 1) / STEP);
    auto at = [&](int i) { return m_beg + (long)i * STEP; };
    if (team < steps) {
        load(at(team));
        store(0, at(team));
    }
    int buf = 0;
    for (int i0 = 0; i0 < steps; i0 += TEAMS, buf ^= 1) {
        const int i = i0 + team;
        __syncthreads();
        const bool more = i + TEAMS < steps;
        if (more) load(at(i + TEAMS));
        if (i < steps) {
#pragma unroll
            for (int s = 0; s < STEP / 16; s++) {
                bf16x8 x[2];
#pragma unroll
                for (int j = 0; j < 2; j++) x[j] = operand<BK>(xbuf[buf], s, wk + 32 * j);
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        const bf16x8 g = operand<BN>(gbuf[buf][p], s, wn + 32 * n);
#pragma unroll
                        for (int j = 0; j < 2; j++) acc[n][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(g, x[j], acc[n][j], 0, 0, 0);
                    }
            }
        }
        if (more) store(buf ^ 1, at(i + TEAMS));
    }

    // join: the second team's tile through LDS to the first, two 32-row blocks at a time; the bias sums of all rows with it
    float* join = reinterpret_cast<float*>(&stage[0]);
    static_assert(sizeof(stage) >= 2 * 2 * 16 * TEAM * sizeof(float), "two blocks of a team's tile fit the stages");
#pragma unroll
    for (int n0b = 0; n0b < NB; n0b += 2) {
        __syncthreads();
        if (team == 1) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) join[((n * 2 + j) * 16 + r) * TEAM + tid] = acc[n0b + n][j][r];
        }
        __syncthreads();
        if (team == 0) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[n0b + n][j][r] += join[((n * 2 + j) * 16 + r) * TEAM + tid];
        }
    }
    // accumulator: column k = lane & 31, row n = (reg & 3) + 8 (reg >> 2) + 4 half
    if (team == 0) {
        float* out = a.gw + (size_t)split * a.N * a.K;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int k = k0 + wk + 32 * j + l31;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int n = n0 + wn + 32 * i + (r & 3) + 8 * (r >> 2) + 4 * half;
                    if (n < a.N && k < a.K) out[(size_t)n * a.K + k] = acc[i][j][r];
                }
            }
    }
    if (bias) {
        constexpr int GROUPS = TEAM / S::CPR;                           // rows that a team loads side by side
        __syncthreads();
#pragma unroll
        for (int e = 0; e < S::E; e++) join[(team * GROUPS + g_row) * BN + S::E * (tid % S::CPR) + e] = bsum[e];
        __syncthreads();
        if (threadIdx.x < BN && n0 + threadIdx.x < a.N) {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < TEAMS * GROUPS; g++) s += join[g * BN + threadIdx.x];
            a.gb[(size_t)split * a.N + n0 + threadIdx.x] = s;
        }
    }
}

// gw[i] = sum over the splits of part[split][i], in order; gb the same from part_b: a thread per 4 values
__global__ __launch_bounds__(256) void wgrad8_fold_kernel(const float* __restrict__ part_w, const float* __restrict__ part_b, float* gw, float* gb, long n, int nb,
                                                         int splits, int blocks_w) {
    const bool second = blockIdx.x >= (unsigned)blocks_w;
    const long len = second ? nb : n, i = 4 * ((long)(blockIdx.x - (second ? blocks_w : 0)) * 256 + threadIdx.x);
    const float* part = second ? part_b : part_w;
    float* out = second ? gb : gw;
    if (i + 4 <= len && (len & 3) == 0) {
        f32x4 s = {};
#pragma unroll 8
        for (int p = 0; p < splits; p++) s += *reinterpret_cast<const f32x4*>(part + p * len + i);
        *reinterpret_cast<f32x4*>(out + i) = s;
    } else {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = 0; p < splits; p++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < len) s[j] += part[p * len + i + j];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < len) out[i + j] = s[j];
    }
}

struct Wgrad8Plan { int tiles_n, tiles_k, splits; long rows_per_split; };
// about one workgroup per CU, none with fewer than 4 steps of rows (a partial tile costs as much traffic as 2 to 4 steps)
Wgrad8Plan plan_of(long M, int N, int K, int dtype) {
    Wgrad8Plan p;
    const int BN = dtype == SCP_DTYPE_F32 ? 128 : 256;
    p.tiles_n = (N + BN - 1) / BN;
    p.tiles_k = (K + BK - 1) / BK;
    const long tiles = (long)p.tiles_n * p.tiles_k, steps = (M + STEP - 1) / STEP;
    long want = tiles >= 256 ? 1 : 256 / tiles;
    if (want > (steps + 3) / 4) want = (steps + 3) / 4;
    const long per = (steps + want - 1) / want;
    p.splits = (int)((steps + per - 1) / per);
    p.rows_per_split = per * STEP;
    return p;
}
const char* bad_problem(long M, int N, int K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return "weight_grad8: empty problem";
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return "weight_grad8: unknown type";
    if (N < (dtype == SCP_DTYPE_F32 ? 4 : 8) || K < 16) return "weight_grad8: fewer than 16 bytes in a row of gy or of the codes";
    if (N > (1 << 20) || K > (1 << 20) || (long)N * K > (1l << 34)) return "weight_grad8: more than 2^20 columns or 2^34 weights";
    return nullptr;
}

}  // namespace

extern "C" size_t scp_weight_grad8_workspace(long M, int N, int K, int dtype) {
    if (bad_problem(M, N, K, dtype)) return 0;
    const Wgrad8Plan p = plan_of(M, N, K, dtype);
    return p.splits > 1 ? (size_t)p.splits * ((size_t)N * K + N) * sizeof(float) : 0;
}

extern "C" int scp_weight_grad8(const void* gy, const signed char* codes, const unsigned char* exps, long M, int N, int K, int dtype, float* gw,
                                float* gb, void* workspace, size_t workspace_bytes, void* stream) {
    if (const char* why = bad_problem(M, N, K, dtype)) return scp::fail(hipErrorInvalidValue, why);
    if (!gy || !codes || !exps || !gw) return scp::fail(hipErrorInvalidValue, "weight_grad8: null argument");
    const Wgrad8Plan p = plan_of(M, N, K, dtype);
    const size_t n = (size_t)N * K;
    if (p.splits > 1 && (!workspace || workspace_bytes < p.splits * (n + N) * sizeof(float) || (reinterpret_cast<size_t>(workspace) & 15)))
        return scp::fail(hipErrorInvalidValue, "weight_grad8: workspace too small or not 16-byte aligned");
    if ((reinterpret_cast<size_t>(gw) | reinterpret_cast<size_t>(gb)) & 15)
        return scp::fail(hipErrorInvalidValue, "weight_grad8: gw and gb must be 16-byte aligned");
    float* part = static_cast<float*>(workspace);
    const Wgrad8Args a{gy, codes, exps, p.splits > 1 ? part : gw, !gb ? nullptr : p.splits > 1 ? part + p.splits * n : gb, M, N, K, p.tiles_n, p.tiles_k,
                       p.splits, p.rows_per_split};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const long total = (long)p.tiles_n * p.tiles_k * p.splits;
    const dim3 grid((unsigned)((total + 7) / 8 * 8));
    const size_t size = dtype == SCP_DTYPE_F32 ? 4 : 2;
    const bool ragged = ((reinterpret_cast<size_t>(gy) | reinterpret_cast<size_t>(codes) | N * size | K) & 15) != 0;
    if (dtype == SCP_DTYPE_F32) {
        if (ragged) hipLaunchKernelGGL((wgrad8_kernel<float, true>), grid, dim3(THREADS), 0, st, a);
        else hipLaunchKernelGGL((wgrad8_kernel<float, false>), grid, dim3(THREADS), 0, st, a);
    } else {
        if (ragged) hipLaunchKernelGGL((wgrad8_kernel<__bf16, true>), grid, dim3(THREADS), 0, st, a);
        else hipLaunchKernelGGL((wgrad8_kernel<__bf16, false>), grid, dim3(THREADS), 0, st, a);
    }
    if (const int e = scp::check_launch("weight_grad8")) return e;
    if (p.splits > 1) {
        const unsigned blocks_w = (unsigned)((n / 4 + 256) / 256), blocks_b = gb ? (unsigned)((N / 4 + 256) / 256) : 0;
        hipLaunchKernelGGL(wgrad8_fold_kernel, dim3(blocks_w + blocks_b), dim3(256), 0, st, part, part + p.splits * n, gw, gb, (long)n, N, p.splits, (int)blocks_w);
        return scp::check_launch("weight_grad8 fold");
    }
    return 0;
}
