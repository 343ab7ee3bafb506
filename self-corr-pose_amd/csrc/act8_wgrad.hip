// self-corr-pose_amd/csrc/act8_wgrad.hip -- weight and bias gradient of a linear layer from the 8-bit checkpoint of its input.
//
//   gw[n][k] = sum_m gy[m][n] x8[m][k],   gb[n] = sum_m gy[m][n],   x8 = code * step (csrc/act8.hip)
//
// A matrix product whose reduction runs over the ROWS of both operands, on v_mfma_f32_32x32x16_bf16.  x8 is exact in bf16 and bf16 gy is what
// it is, so every product is exact and only the fp32 accumulation rounds; fp32 gy is cut into three bf16 parts of 8 bits each
// (gy = h + m + l exactly; an infinity takes a second pass over its tile) and multiplied part by part: 3 matrix instructions for 1, still 5
// times the rate of the fp32 cores.
//   * a workgroup owns a BN x 128 tile of gw over a range of rows and walks it 64 rows at a time, with two kinds of wavefronts: eight FILL (gy and
//     the codes go global -> registers three steps ahead, are cut / dequantised there and written to LDS row-major one step ahead) and
//     eight MULTIPLY, so that the vector work of the one runs beside the matrix instructions of the other;
//   * ds_read_b64_tr_b16 turns 4 rows x 16 columns into operand order, the same row order for both operands, so no transposition is ever
//     stored; LDS rows are swizzled in 16-byte chunks so that the 4 rows x 4 chunks of half a transposed read touch each bank once;
//   * BN = 256 for bf16 (a multiplying wavefront owns 64 x 64), 128 for fp32 (32 x 64), where the three parts share the x8 operand;
//   * the rows are split so that about one workgroup per CU runs; each writes an fp32 partial tile and a second kernel adds the partials in
//     order (bit-reproducible).  gb falls out of the registers of the filling wavefronts of the first column of tiles.
// Bound by filling and multiplying together, not by memory: of 77 us for 32800 rows, 384 -> 1536, bf16 (with pack8 9 and the fold 6.5), 62 are
// left without the products, 55 without the filling, 28 without both; steps of 64 rows instead of 32 halve the barriers (69), addresses that
// are constants of the loop and rows past the end read as zeros: 64 to 68 us.  The kernel alone: 52 us, 740 TFLOP/s; 1536 -> 384, fp32 132 to
// 146 us, 3 x 265 to 290.
#include <hip/hip_runtime.h>

#include <type_traits>

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
typedef unsigned u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

constexpr int BK = 128, STEP = 64, FILL = 512, MULTIPLY = 512, THREADS = MULTIPLY + FILL;

struct Wgrad8Args {
    const void* gy;
    const signed char* codes;
    const unsigned char* exps;
    float *gw, *gb;              // the results, or [splits] partials of them
    long M;
    int N, K, tiles_n, tiles_k, splits;
    long rows_per_split;         // a multiple of STEP
};

// element offset of (row, 16-byte chunk) in a [STEP][COLS] bf16 tile
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

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes > 0 ? bytes : 0, 0x00020000);
}

// the bytes of x from byte `shift` on (what follows them is of no account)
__device__ __forceinline__ u32x2 from_byte(u32x2 x, int shift) {
    const u32x2 y = {shift & 4 ? x[1] : x[0], x[1]};
    return u32x2{__builtin_amdgcn_alignbyte(y[1], y[0], shift & 3), y[1] >> (8 * (shift & 3))};
}
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
    static constexpr int PIECES = STEP * CPR / FILL;                      // 4 per thread
    static constexpr int NB = BN / 128;                                   // 32-column blocks of n per multiplying wavefront (4 x 2 of them)
};

// RAGGED: rows of gy (of the codes) are no whole number of 16-byte (8-byte) pieces, or not aligned to them
template <typename T, bool RAGGED> __global__ __launch_bounds__(THREADS, 4) void wgrad8_kernel(const Wgrad8Args a) {
    typedef Wgrad8Shape<T> S;
    constexpr int BN = S::BN, PARTS = S::PARTS, NB = S::NB;
    __shared__ __attribute__((aligned(16))) __bf16 gbuf[2][PARTS][STEP * BN];
    __shared__ __attribute__((aligned(16))) __bf16 xbuf[2][STEP * BK];
    __shared__ float bias_sums[FILL / S::CPR][BN];
    __shared__ int again;

    // tiles of one range of rows next to each other on one XCD: they read the same rows of gy and of the codes
    const int tiles = a.tiles_n * a.tiles_k, total = tiles * a.splits, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= total || (blockIdx.x >> 3) >= (unsigned)per) return;
    const int split = id / tiles, tile = id - split * tiles, tn = tile / a.tiles_k, tk = tile - tn * a.tiles_k;
    const int n0 = tn * BN, k0 = tk * BK;
    const long m_beg = split * a.rows_per_split, m_end = m_beg + a.rows_per_split < a.M ? m_beg + a.rows_per_split : a.M;

    const bool fills = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= MULTIPLY / 64;
    const int tid = fills ? threadIdx.x - MULTIPLY : threadIdx.x;
    const int groups = (a.K + 31) / 32;
    const int steps = (int)((m_end - m_beg + STEP - 1) / STEP);
    auto at = [&](int i) { return m_beg + (long)(i < steps ? i : steps - 1) * STEP; };        // a step past the end repeats the last

    if (threadIdx.x == 0) again = 0;                                    // (read after the barrier that ends the first pass)
    if (!fills) {
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l31 = lane & 31;
        const int wn = (wave >> 1) * (BN / 4), wk = (wave & 1) * 64;
        f32x16 acc[NB][2];
        auto multiply = [&](int buf) {
            __syncthreads();
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
        };
        for (bool first = true;; first = false) {
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = f32x16{};
            int i = 0;
            for (; i + 1 < steps; i += 2) {                             // the buffers by name: every LDS address is a constant of the loop
                multiply(0);
                multiply(1);
            }
            if (i < steps) multiply(0);
            if (S::F32 && first) {                                      // a NaN: a second pass, see below
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NB; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int r = 0; r < 16; r++) sum += acc[i][j][r];
                if (sum != sum) again = 1;
            }
            __syncthreads();                                            // the filling wavefronts' last one of the pass
            if (!S::F32 || !first || !again) break;
        }
        // accumulator: column k = lane & 31, row n = (reg & 3) + 8 (reg >> 2) + 4 half
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
        if (a.gb && tk == 0 && tid < BN && n0 + tid < a.N) {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < FILL / S::CPR; g++) s += bias_sums[g][tid];
            a.gb[(size_t)split * a.N + n0 + tid] = s;
        }
        return;
    }

    auto fill = [&](const int tid, auto infinities) {
        // loads: gy piece i of this thread = row tid / 32 + 16 i, elements E (tid % 32); codes = rows tid / 16 and tid / 16 + 32, 8 of each.
        // Pieces past a row's end are read from its end instead and moved into place (RAGGED); what stands behind them, and in pieces past the
        // matrix, goes into products that nobody stores.  Rows past the range are read from its last row and stored as zeros (RAGGED), or read
        // as zeros from behind the end of a buffer: without minima and multiplications per piece, which cost as much as the dequantisation.
        const char* gy = static_cast<const char*>(a.gy);
        const int g_row = tid / S::CPR, g_col = n0 + S::E * (tid % S::CPR);
        const int x_row = tid >> 4, x_col = k0 + 8 * (tid & 15);
        const int g_at = min(g_col, a.N - S::E), x_at = min(x_col, a.K - 8);
        const int g_shift = min(g_col - g_at, S::E - 1) * (int)sizeof(T), x_shift = min(x_col - x_at, 7);
        const int e_at = min(x_col >> 5, groups - 1);
        // (Loads are never conditional: the wait for the older of the two register sets can then leave the younger in flight.)
        constexpr int XR = STEP * 16 / FILL;                                 // rows of codes per thread
        struct Raw { u32x4 g[S::PIECES]; u32x2 x[XR]; unsigned exp[XR]; };
        constexpr int XROWS = FILL / 16;
        const int g_off = (g_row * a.N + g_at) * (int)sizeof(T), g_next = FILL / S::CPR * a.N * (int)sizeof(T);
        const int x_off = x_row * a.K + x_at, x_next = XROWS * a.K, e_off = x_row * groups + e_at, e_next = XROWS * groups;
        auto load = [&](Raw& raw, long m) {
            const int rows = m_end - m < STEP ? (int)(m_end - m) : STEP;
            const char* gbase = gy + m * a.N * (long)sizeof(T);
            const char* xbase = reinterpret_cast<const char*>(a.codes) + m * a.K;
            const char* ebase = reinterpret_cast<const char*>(a.exps) + m * groups;
            if constexpr (RAGGED) {
#pragma unroll
                for (int i = 0; i < S::PIECES; i++)
                    raw.g[i] = *reinterpret_cast<const u32x4_a1*>(gbase + (unsigned)(min(g_row + (FILL / S::CPR) * i, rows - 1) * a.N + g_at) * (unsigned)sizeof(T));
#pragma unroll
                for (int i = 0; i < XR; i++) {
                    const int r = min(x_row + XROWS * i, rows - 1);
                    raw.x[i] = *reinterpret_cast<const u32x2_a1*>(xbase + (unsigned)(r * a.K + x_at));
                    raw.exp[i] = *reinterpret_cast<const unsigned char*>(ebase + (unsigned)(r * groups + e_at));
                }
            } else {                                                        // rows past the range are past the buffer's end: zeros
                const int g_bytes = rows * a.N * (int)sizeof(T), x_bytes = rows * a.K, e_bytes = rows * groups;
#pragma unroll
                for (int i = 0; i < S::PIECES; i++)
                    raw.g[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer(gbase + i * g_next, g_bytes - i * g_next), g_off, 0, 0));
#pragma unroll
                for (int i = 0; i < XR; i++) {
                    raw.x[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(buffer(xbase + i * x_next, x_bytes - i * x_next), x_off, 0, 0));
                    raw.exp[i] = __builtin_amdgcn_raw_buffer_load_b8(buffer(ebase + i * e_next, e_bytes - i * e_next), e_off, 0, 0);
                }
            }
        };
        const bool bias = a.gb && tk == 0;
        float bsum[S::E];
#pragma unroll
        for (int i = 0; i < S::E; i++) bsum[i] = 0.f;
        auto store = [&](Raw& raw, int buf, long m, bool counts) {
            if constexpr (RAGGED) {
#pragma unroll
                for (int i = 0; i < S::PIECES; i++) raw.g[i] = from_byte(raw.g[i], g_shift);
#pragma unroll
                for (int i = 0; i < XR; i++) raw.x[i] = from_byte(raw.x[i], x_shift);
            }
            if (RAGGED && m + STEP > m_end) {
                const int rows = (int)(m_end - m);
#pragma unroll
                for (int i = 0; i < S::PIECES; i++)
                    if (g_row + (FILL / S::CPR) * i >= rows) raw.g[i] = u32x4{};
#pragma unroll
                for (int i = 0; i < XR; i++)
                    if (x_row + XROWS * i >= rows) {
                        raw.x[i] = u32x2{};
                        raw.exp[i] = 1;
                    }
            }
#pragma unroll
            for (int i = 0; i < S::PIECES; i++) {
                const int row = g_row + (FILL / S::CPR) * i, col = S::E * (tid % S::CPR);
                if constexpr (S::F32) {
                    unsigned h[4], m[4], l[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {                            // 8 + 8 + 8 bits: h + m + l = gy exactly
                        const float x = __uint_as_float(raw.g[i][e]);
                        h[e] = raw.g[i][e] & 0xffff0000u;
                        float rest = x - __uint_as_float(h[e]);
                        if constexpr (infinities.value) rest = (raw.g[i][e] & 0x7fffffffu) == 0x7f800000u ? 0.f : rest;
                        m[e] = __float_as_uint(rest) & 0xffff0000u;
                        l[e] = __float_as_uint(rest - __uint_as_float(m[e]));
                        if (bias && counts) bsum[e] += x;
                    }
                    const int at = lds_at<BN>(row, col / 8) + (col & 7);
                    *reinterpret_cast<u32x2*>(&gbuf[buf][0][at]) = u32x2{upper_halves(h[0], h[1]), upper_halves(h[2], h[3])};
                    *reinterpret_cast<u32x2*>(&gbuf[buf][1 % PARTS][at]) = u32x2{upper_halves(m[0], m[1]), upper_halves(m[2], m[3])};
                    *reinterpret_cast<u32x2*>(&gbuf[buf][2 % PARTS][at]) = u32x2{upper_halves(l[0], l[1]), upper_halves(l[2], l[3])};
                } else {
                    *reinterpret_cast<u32x4*>(&gbuf[buf][0][lds_at<BN>(row, col / 8)]) = raw.g[i];
                    if (bias && counts) {
#pragma unroll
                        for (int e = 0; e < 8; e++) bsum[e % S::E] += __uint_as_float(e & 1 ? raw.g[i][e / 2] & 0xffff0000u : raw.g[i][e / 2] << 16);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < XR; i++) {
                const float unit = __uint_as_float(raw.exp[i] == 255 ? 0x7fc00000u : raw.exp[i] << 23);
                u32x4 x;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (float)(signed char)(raw.x[i][w] >> (8 * e)) * unit;
                    x[2 * w] = upper_halves(__float_as_uint(v[0]), __float_as_uint(v[1]));
                    x[2 * w + 1] = upper_halves(__float_as_uint(v[2]), __float_as_uint(v[3]));
                }
                *reinterpret_cast<u32x4*>(&xbuf[buf][lds_at<BK>(x_row + XROWS * i, tid & 15)]) = x;
            }
        };

        Raw even, odd;
        load(even, at(0));
        load(odd, at(1));
        store(even, 0, at(0), true);
        load(even, at(2));
        // step i is being multiplied: step i + 1 goes to the other buffer, the loads of step i + 3 start
        auto step = [&](int i, int buf, Raw& next) {
            __syncthreads();
            store(next, buf ^ 1, at(i + 1), i + 1 < steps);
            load(next, at(i + 3));
        };
        int i = 0;
        for (; i + 1 < steps; i += 2) {
            step(i, 0, odd);
            step(i + 1, 1, even);
        }
        if (i < steps) __syncthreads();                                     // the last of an odd number of steps: nothing left to fill
        if (bias) {
#pragma unroll
            for (int e = 0; e < S::E; e++) bias_sums[g_row][S::E * (tid % S::CPR) + e] = bsum[e];
        }
    };
    fill(tid, std::false_type{});
    __syncthreads();
    // The parts of an infinity are inf, inf - inf and so on: NaN where the sum of products is an infinity.  A tile that came out with a NaN is
    // computed again with infinities cut into themselves and zeros; looking at every element in the first pass cost 18 % (133 -> 157 us).
    if constexpr (S::F32) {
        if (again) {
            int same = tid;
            asm("" : "+v"(same));                                       // nothing of the first pass is kept in registers for the second
            fill(same, std::true_type{});
            __syncthreads();
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
// about one workgroup per CU, none with fewer than 2 steps of rows (a partial tile costs as much traffic as 1 to 2 steps)
Wgrad8Plan plan_of(long M, int N, int K, int dtype) {
    Wgrad8Plan p;
    const int BN = dtype == SCP_DTYPE_F32 ? 128 : 256;
    p.tiles_n = (N + BN - 1) / BN;
    p.tiles_k = (K + BK - 1) / BK;
    const long tiles = (long)p.tiles_n * p.tiles_k, steps = (M + STEP - 1) / STEP;
    long want = tiles >= 256 ? 1 : 256 / tiles;
    if (want > (steps + 1) / 2) want = (steps + 1) / 2;
    const long per = (steps + want - 1) / want;
    p.splits = (int)((steps + per - 1) / per);
    p.rows_per_split = per * STEP;
    return p;
}
const char* bad_problem(long M, int N, int K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return "weight_grad8: empty problem";
    if (dtype != SCP_DTYPE_F32 && dtype != SCP_DTYPE_BF16) return "weight_grad8: unknown type";
    if (N < (dtype == SCP_DTYPE_F32 ? 4 : 8) || K < 8) return "weight_grad8: fewer than 16 bytes in a row of gy or 8 codes in a row";
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
    const bool ragged = ((reinterpret_cast<size_t>(gy) | N * size) & 15) != 0 || ((reinterpret_cast<size_t>(codes) | K) & 7) != 0;
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
