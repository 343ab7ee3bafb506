// self-corr-pose_amd/csrc/attn_core.h -- matrix-core kernels of csrc/cross_attn.hip, shared by its fp32 and bf16 instantiations.
//
// One skeleton serves forward, query gradient and key / value gradient: a wavefront keeps 32 columns (queries, or keys) STATIONARY in
// registers, lane l31 = lane & 31 owning column l31, and streams 32-row blocks of the other side through LDS.
//   a dot product block   D[row][col] = X[row][:] . F[col][:]  comes out with the rows in the accumulator registers
//     (row = (reg & 3) + 8 (reg >> 2) + 4 half, half = lane >> 5), so softmax statistics of a column are lane-local;
//   a product over rows   Acc[d][col] += X[row][d] P[row][col]  takes P from exactly those registers: its row order inside a matrix
//     instruction is the order in which the accumulators already hold the rows, and X comes transposed out of LDS in that order
//     (ds_read_b64_tr_b16).
// forward:           stationary Q,     streamed K, V;   Acc = o^T  += V^T p
// query gradient:    stationary Q, gO, streamed K, V;   Acc = gq^T += K^T gs
// key/value gradient: stationary K, V, streamed Q, gO;  Acc = gk^T += Q^T gs,  Acc2 = gv^T += gO^T p
// Everything runs on v_mfma_f32_32x32x16_bf16.
// fp32: every operand is three bf16 parts of 8 bits each (x = h + m + l exactly), q, k, v and g_out cut once into a workspace by csrc/
// cross_attn.hip, p and gs in registers; a product is the six products of parts that reach 2^-24 of it, the small ones first.  That is 6 matrix
// instructions for 16 of v_mfma_f32_32x32x2_f32 and the same LDS reads (4 x 6 heads of 642 x 1025: forward + backward 193 -> 144 us).  An
// infinity that is not masked gives NaN: its parts are inf and NaN.
// bf16: p and gs are rounded to bf16 for their product: one operand of it has to be bf16, and the result is rounded to bf16 anyway (error of the
// results of 642 x 1025 in norm 2.3e-3 to 2.4e-3, their own rounding 1.7e-3; 16 bits of p would be 3 products for 2).  What
// that does to gs = p (gO . v - delta) where a few keys hold most of the softmax, and gO . v and delta cancel: the denominator is the sum of
// the ROUNDED p (v_dot2_f32_bf16, as fast as the 16 additions that it replaces), so o is a weighted mean of v whatever the rounding did
// and its error in delta is of the size of gs's own rounding; and the next 8 bits of o are kept for the backward pass (o_low), so delta sees
// o to 16 bits.  Error of gq, 300 queries x 300 keys with a softmax on 2 to 3 keys: 5.7e-3
// without the two, 3.0e-3 with them.
//
// Three ways to deal the work (Plan).  OWN: each of 4 wavefronts has 32 columns of its own and all read the same tile (64 rows in bf16, 32 in
// fp32).  SHARE: 4 (bf16) or 2 (fp32) wavefronts have the SAME 32 columns, each reads its 32 rows of a tile of 128 or 64, and their partial
// results are joined through LDS at the end; that divides the reuse of a tile by the number and multiplies the wavefronts by it: it is for
// problems that would leave SIMDs empty otherwise.  FEW: no tiles, see few_rows_kernel.  Tiles are double-buffered (the next one in flight
// during the products) where two fit 80 KB.
// Measured: bf16 forward of 2562 x 4097, 8 x 6 heads of 64 on 2, 156 us (830 TFLOP/s); forward + backward of 642 x 1025, 32 x 6 heads, a padded
// batch, 175 to 193 us; what bounds both is matrix and vector instructions, which overlap to about 70 % of their sum.
//
// LDS tiles are filled by buffer loads that write LDS directly, 16 bytes per lane.  A lane whose row is masked, past the end, or whose
// channel is past head_dim gets an out-of-range offset: the hardware writes zeros, so nothing stored there can reach a product.  The
// tile's image is swizzled through the SOURCE address (16-byte chunk `slot ^ f(row)`), such that both reads of it -- 16 consecutive rows at
// one chunk, 4 consecutive rows at four -- touch each bank once.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "scp_common.h"

namespace scp_attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const void *q, *k, *v, *go;           // what the matrix products read: the tensors (bf16), or their parts (fp32: Parts)
    const void* dgo;                      // g_out itself, for delta
    const unsigned char* mask;
    const void* o_in;
    const signed char* o_low_in;
    void *o, *gq, *gk, *gv;
    signed char* o_low;
    float *lse, *delta;
    float *part_o, *part_ml;              // split over the keys: [split][bh][R][D], [split][bh][R][2]
    long qs[3], ks[3], vs[3], gs[3], dgs[3];      // strides in elements: batch, token, head
    int BH, Nq, Nk, Hk, G, D;
    int nsplit, keys_per_split;           // keys_per_split: a multiple of the tile
    float scale;
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THR = 8.f;        // the accumulator is rescaled only when the maximum grows by more than 2^8
constexpr unsigned OUT_OF_RANGE = 0x80000000u;

__device__ __forceinline__ int acc_row(int reg, int half) { return (reg & 3) + 8 * (reg >> 2) + 4 * half; }
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return (threadIdx.x & 32) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}

// what a tensor's element becomes for the matrix cores: bf16 itself, or three bf16 parts of 8 bits each of an fp32 number
template <typename T> constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;

// rows of a [32 n][DP] bf16 tile in LDS, 16-byte chunks
template <int DP> struct Tile {
    static constexpr int CH = 8;                       // elements per chunk
    static constexpr int CPR = DP / CH;                // chunks per row
    static __device__ __forceinline__ int swizzle(int chunk, int row) {
        if constexpr (CPR == 4) return chunk ^ ((row >> 2) & 3);
        else if constexpr (CPR == 8) return chunk ^ (((row & 2) << 1) | ((row & 4) >> 1) | ((row >> 3) & 1));
        else if constexpr (CPR == 12) { const int s = chunk + ((row >> 2) & 3); return s >= 12 ? s - 12 : s; }
        else return chunk ^ (((row & 3) << 2) | ((row >> 2) & 3));
    }
    static __device__ __forceinline__ int unswizzle(int slot, int row) {
        if constexpr (CPR == 12) { const int s = slot - ((row >> 2) & 3); return s < 0 ? s + 12 : s; }
        else return swizzle(slot, row);
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return (row * CPR + swizzle(chunk, row)) * CH; }
};

// an fp32 number as h + m + l, each of 8 bits; the parts of two numbers packed
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ void three_parts(float x, float y, unsigned (&out)[3]) {
    const unsigned xh = __float_as_uint(x) & 0xffff0000u, yh = __float_as_uint(y) & 0xffff0000u;
    const float xr = x - __uint_as_float(xh), yr = y - __uint_as_float(yh);
    const unsigned xm = __float_as_uint(xr) & 0xffff0000u, ym = __float_as_uint(yr) & 0xffff0000u;
    out[0] = upper_halves(xh, yh);
    out[1] = upper_halves(xm, ym);
    out[2] = upper_halves(__float_as_uint(xr - __uint_as_float(xm)), __float_as_uint(yr - __uint_as_float(ym)));
}

template <typename T> struct Out;
template <> struct Out<__bf16> {
    typedef __bf16 T;
    static __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
        const bf16x4 v = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
        *reinterpret_cast<bf16x4*>(p) = v;
    }
    // channels 32 db .. 32 db + 31 of this lane's column, in accumulator order, to `row` where ok; `low` (or null): low_bits of them.
    // The halves of the wavefront trade accumulators, so that each lane stores 8 channels in a row.
    static __device__ __forceinline__ void store_column(T* row, signed char* low, int db, int D, bool ok, const f32x16& v) {
        const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int d = 32 * db + 16 * k + 8 * half;
            u32x4 hi = {};
#pragma unroll
            for (int w = 0; w < 2; w++) {
                unsigned h[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const bf16x2 pair = {(__bf16)v[8 * k + 4 * u + 2 * w], (__bf16)v[8 * k + 4 * u + 2 * w + 1]};
                    h[u] = __builtin_bit_cast(unsigned, pair);
                }
                const auto a = __builtin_amdgcn_permlane32_swap(h[0], h[1], false, false);
                hi[w] = a[0];
                hi[2 + w] = a[1];
            }
            if (ok && d < D) *reinterpret_cast<u32x4*>(row + d) = hi;
            if (low) {
                unsigned l[2];
#pragma unroll
                for (int u = 0; u < 2; u++) l[u] = low_bits(v[8 * k + 4 * u], v[8 * k + 4 * u + 1], v[8 * k + 4 * u + 2], v[8 * k + 4 * u + 3]);
                const auto a = __builtin_amdgcn_permlane32_swap(l[0], l[1], false, false);
                if (ok && d < D) *reinterpret_cast<u32x2*>(low + d) = u32x2{a[0], a[1]};
            }
        }
    }
    // The 8 bits of a number that follow its bf16 rounding, signed: (bits - rounded bits) >> 8, whole numbers both, is in -128 .. 128 (a tie
    // that rounds down to even is +128) and is kept as at most 127; with half a step of it added the number comes back to 2^-16 of itself.
    static __device__ __forceinline__ unsigned low_bits(float a, float b, float c, float d) {
        const float x[4] = {a, b, c, d};
        unsigned out = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float top = (float)(__bf16)x[i];
            const int rest = min((int)(__float_as_uint(x[i]) - __float_as_uint(top)), 0x7fff);
            out |= ((unsigned)(rest >> 8) & 0xffu) << (8 * i);
        }
        return out;
    }
    // (an infinity stays one; a NaN's rest is of no account)
    static __device__ __forceinline__ float with_low(float top, int code) {
        const unsigned bits = __float_as_uint(top);
        return __uint_as_float((bits & 0x7f800000u) == 0x7f800000u ? bits : bits + (unsigned)(code * 256 + 128));
    }
    static __device__ __forceinline__ void store_low(signed char* p, float a, float b, float c, float d) { *reinterpret_cast<unsigned*>(p) = low_bits(a, b, c, d); }
};
template <> struct Out<float> {
    typedef float T;
    static __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
        const f32x4 v = {a, b, c, d};
        *reinterpret_cast<f32x4*>(p) = v;
    }
    static __device__ __forceinline__ void store_column(T* row, signed char*, int db, int D, bool ok, const f32x16& v) {
        const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int d = 32 * db + 8 * g + 4 * half;
            if (ok && d < D) store4(row + d, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
    }
    static __device__ __forceinline__ void store_low(signed char*, float, float, float, float) {}
    static __device__ __forceinline__ float with_low(float top, int) { return top; }
};

// PS: elements between the planes of a tile (its parts, one [rows][DP] image each)
template <typename T, int DP, int PS> struct Mma {
    typedef Tile<DP> L;
    static constexpr int DB = DP / 32, NP = PARTS<T>;
    struct Frag { bf16x8 f[NP][DP / 16]; };
    // the parts' products that count, the small ones first: (part of x, part of y)
    static constexpr int PAIRS = NP == 1 ? 1 : 6;
    static constexpr int PX[6] = {NP == 1 ? 0 : 2, 1, 0, 1, 0, 0}, PY[6] = {0, 1, 2, 0, 1, 0};
    static __device__ __forceinline__ void load(Frag& x, const __bf16* row, bool valid, int D, float sign) {
        const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
            for (int i = 0; i < DP / 16; i++) {
                u32x4 v = {};
                if (valid && 16 * i + 8 * half < D) v = *reinterpret_cast<const u32x4*>(row + p * D + 16 * i + 8 * half);
                x.f[p][i] = __builtin_bit_cast(bf16x8, v ^ (sign < 0.f ? 0x80008000u : 0u));
            }
    }
    // acc[c] = rows r0 .. r0+31 of `t` times the stationary columns of block c
    template <int CB> static __device__ __forceinline__ void dots(f32x16 (&acc)[CB], const __bf16* t, int r0, const Frag (&x)[CB]) {
        const int half = (threadIdx.x >> 5) & 1, row = r0 + (threadIdx.x & 31);
#pragma unroll
        for (int c = 0; c < CB; c++) acc[c] = f32x16{};
#pragma unroll
        for (int i = 0; i < DP / 16; i++) {
            bf16x8 a[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) a[p] = *reinterpret_cast<const bf16x8*>(t + p * PS + L::at(row, 2 * i + half));
#pragma unroll
            for (int y = 0; y < PAIRS; y++)
#pragma unroll
                for (int c = 0; c < CB; c++) acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[PX[y]], x[c].f[PY[y]][i], acc[c], 0, 0, 0);
        }
    }
    // a[c][db][d][col] += sum_row t[r0 + row][32 db + d] p[c][row][col];  bf16: sums[c] (where given) += the p that were multiplied, half a
    // column each; LOW: what rounding p to bf16 drops is multiplied too
    template <int CB, bool LOW = false> static __device__ __forceinline__ void adds(f32x16 (&a)[CB][DB], const __bf16* t, int r0, const f32x16 (&p)[CB], float* sums = nullptr) {
        const int lane = threadIdx.x & 63, i = lane & 15, half = lane >> 5, cg = (lane >> 4) & 1;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            bf16x8 b[CB][NP], low[CB];
#pragma unroll
            for (int c = 0; c < CB; c++) {
                if constexpr (NP == 1) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        b[c][0][j] = (__bf16)p[c][8 * s + j];
                        if constexpr (LOW) low[c][j] = (__bf16)(p[c][8 * s + j] - (float)b[c][0][j]);
                    }
                } else {
                    u32x4 parts[3];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        unsigned w[3];
                        three_parts(p[c][8 * s + 2 * j], p[c][8 * s + 2 * j + 1], w);
#pragma unroll
                        for (int k = 0; k < 3; k++) parts[k][j] = w[k];
                    }
#pragma unroll
                    for (int k = 0; k < NP; k++) b[c][k] = __builtin_bit_cast(bf16x8, parts[k]);
                }
            }
            if (NP == 1 && sums) {
                const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
                for (int c = 0; c < CB; c++)
#pragma unroll
                    for (int j = 0; j < 4; j++) sums[c] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{b[c][0][2 * j], b[c][0][2 * j + 1]}, one, sums[c], false);
            }
#pragma unroll
            for (int db = 0; db < DB; db++) {
                bf16x8 w[NP];
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    bf16x4 h[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int row = r0 + 16 * s + 8 * u + 4 * half + (i >> 2);
                        const __bf16* at = t + k * PS + L::at(row, 4 * db + 2 * cg + ((i & 3) >> 1)) + 4 * (i & 1);
                        h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)at);
                    }
                    w[k] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
                }
                if constexpr (NP == 1 && LOW) {
#pragma unroll
                    for (int c = 0; c < CB; c++) a[c][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[0], low[c], a[c][db], 0, 0, 0);
                }
#pragma unroll
                for (int y = 0; y < PAIRS; y++)
#pragma unroll
                    for (int c = 0; c < CB; c++) a[c][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[PX[y]], b[c][PY[y]], a[c][db], 0, 0, 0);
            }
        }
    }
};

// rows of one head in global memory: row r is token r / G (of stride ts) and head r % G (of stride hs) behind `base`
struct Rows {
    const char* base;
    long ts, hs;          // bytes
    int G;
    __device__ __forceinline__ const char* row(int r) const {
        if (G == 1) return base + r * ts;
        const int n = r / G;
        return base + n * ts + (r - n * G) * hs;
    }
};
template <typename T> __device__ __forceinline__ Rows rows_of(const void* p, const long* st, int b, int h, int G) {
    return {reinterpret_cast<const char*>(static_cast<const T*>(p) + b * st[0] + h * st[2]), st[1] * (long)sizeof(T), st[2] * (long)sizeof(T), G};
}

__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p; }
// 16 (4) bytes per lane from rsrc + off to LDS at `lds` + 16 (4) lane.  Inline assembly: the compiler would take every later LDS read for one of
// the bytes in flight and wait for the NEXT tile before working on this one.  wait_tiles() is the wait.
__device__ __forceinline__ void to_lds16(unsigned off, __amdgpu_buffer_rsrc_t rsrc, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(rsrc), "s"(lds) : "memory");
}
__device__ __forceinline__ void to_lds4(unsigned off, __amdgpu_buffer_rsrc_t rsrc, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(rsrc), "s"(lds) : "memory");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)OUT_OF_RANGE, 0x00020000);
}

// moves rows r0 .. r0+N-1 of one head into an LDS tile; on[]: one bit per row, a clear one gives a row of zeros.  The lanes' offsets behind
// the tile's first row are the same for every tile (tokens of one head, or a tile of a whole number of tokens), so they are kept; the
// tile's own place is a 64-bit address.  The host has checked that a tile spans less than 2^31 bytes.
template <int DP, int N, int WAVES, int NPARTS> struct Loader {
    typedef Tile<DP> L;
    static constexpr int PIECES = N * L::CPR / 64, NP = (PIECES + WAVES - 1) / WAVES;
    Rows src;
    int D, wave;
    unsigned off[NP];
    static __device__ __forceinline__ int row_of(int wave, int i) { return ((wave + WAVES * i) * 64 + (int)(threadIdx.x & 63)) / L::CPR; }
    __device__ __forceinline__ void place_pieces(int r0) {
        const int n0 = src.G == 1 ? 0 : r0 / src.G;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int row = row_of(wave, i), chunk = L::unswizzle(((wave + WAVES * i) * 64 + (int)(threadIdx.x & 63)) % L::CPR, row);
            unsigned o;
            if (src.G == 1) o = (unsigned)row * (unsigned)src.ts;
            else {
                const int n = (r0 + row) / src.G;
                o = (unsigned)(n - n0) * (unsigned)src.ts + (unsigned)(r0 + row - n * src.G) * (unsigned)src.hs;
            }
            off[i] = chunk * L::CH < D ? o + 16u * chunk : OUT_OF_RANGE;
        }
    }
    __device__ __forceinline__ Loader(const Rows& rows, int head_dim) : src(rows), D(head_dim) {
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        place_pieces(0);
    }
    __device__ __forceinline__ void issue(__bf16* lds, int r0, const unsigned (&on)[N / 32]) {
        if (src.G > 1 && N % src.G) place_pieces(r0);
        const __amdgpu_buffer_rsrc_t rsrc = buffer(src.base + (src.G == 1 ? r0 : r0 / src.G) * src.ts);
        unsigned all = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < N / 32; j++) all &= on[j];
        const unsigned at = __builtin_amdgcn_readfirstlane(lds_address(lds));
        if (all == 0xffffffffu) {
#pragma unroll
            for (int p = 0; p < NPARTS; p++)
#pragma unroll
                for (int i = 0; i < NP; i++)
                    if (wave + WAVES * i < PIECES) to_lds16(off[i] + 2u * p * D, rsrc, at + 2u * p * N * DP + (wave + WAVES * i) * 1024u);
        } else {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int row = row_of(wave, i);
                unsigned word = on[0];
#pragma unroll
                for (int j = 1; j < N / 32; j++) word = (row >> 5) == j ? on[j] : word;
                const unsigned o = (word >> (row & 31)) & 1 ? off[i] : OUT_OF_RANGE;
#pragma unroll
                for (int p = 0; p < NPARTS; p++)
                    if (wave + WAVES * i < PIECES) to_lds16(o + 2u * p * D, rsrc, at + 2u * p * N * DP + (wave + WAVES * i) * 1024u);
            }
        }
    }
};
// every load of this wavefront has arrived (vmcnt 0; the builtin, so that the compiler knows it too and does not wait again later for
// registers it loaded before the loop), then everybody's
__device__ __forceinline__ void wait_tiles() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
    __syncthreads();
}

// which keys of the next 64 tiles of KT keys exist: one bit per key in `words`, and the tiles that hold any as a bit set
template <int KT, int WAVES> __device__ __forceinline__ unsigned long long key_window(unsigned* words, const unsigned char* mask, int key0, int key_end) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __syncthreads();
    static_assert(KT % WAVES == 0, "64 tiles of KT keys are KT groups of 64, dealt to the wavefronts");
    const int groups = min(KT, (key_end - key0 + 63) >> 6);  // groups that hold a key; the words of the others are not read
    if (mask) {
        constexpr int BATCH = 4;                             // loads in flight per lane
        for (int g0 = wave; g0 < groups; g0 += BATCH * WAVES) {
            unsigned char byte[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) byte[i] = mask[min(key0 + 64 * (g0 + WAVES * i) + lane, key_end - 1)];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int g = g0 + WAVES * i;
                const unsigned long long bits = __ballot(key0 + 64 * g + lane < key_end && byte[i]);
                if (g < groups && lane < 2) words[2 * g + lane] = (unsigned)(bits >> (32 * lane));
            }
        }
    } else {
        for (int w = threadIdx.x; w < 2 * groups; w += 64 * WAVES) {
            const int left = key_end - key0 - 32 * w;
            words[w] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
        }
    }
    __syncthreads();
    unsigned any = 0;
    if (lane * KT < 64 * groups) {
#pragma unroll
        for (int i = 0; i < KT / 32; i++)
            if (lane * (KT / 32) + i < 2 * groups) any |= words[lane * (KT / 32) + i];
    }
    return __ballot(any != 0);
}

// block index -> (head, block): blocks of one head on one XCD (its K and V then live in that XCD's L2), heads dealt to the 8 XCDs in turn
__device__ __forceinline__ bool place(int BH, int per_head, int& bh, int& blk) {
    const int lin = blockIdx.x;
    if (BH >= 16) {
        const int slot = lin >> 3;
        bh = (slot / per_head) * 8 + (lin & 7);
        blk = slot % per_head;
        return bh < BH;
    }
    bh = lin / per_head;
    blk = lin % per_head;
    return true;
}
inline unsigned placed_blocks(int BH, int per_head) { return (unsigned)((BH >= 16 ? (BH + 7) / 8 * 8 : BH) * per_head); }

// SH: wavefronts that share their columns (1: OWN); tile rows, buffers
template <typename T, int DP, int SH> struct Shape {
    static constexpr int WAVES = 4, THREADS = 256, NP = PARTS<T>;
    static constexpr int N = SH > 1 ? 32 * SH : NP == 1 ? 64 : 32;          // rows per tile
    static constexpr int COLS = 128 / SH;                                   // columns per workgroup (of one block per wavefront)
    static constexpr int BYTES = 2 * NP * N * DP * 2;                       // the two tiles
    static constexpr int NBUF = 2 * BYTES <= 81920 ? 2 : 1;
    // column blocks that a wavefront can take in the forward pass.  Two: every LDS read feeds two matrix instructions, and the products of one
    // block run beside the exponentials of the other (bf16, 64 channels: 173 -> 160 us for 7686 x 4097 x 16 heads); more would not fit
    // the registers.
    static constexpr int MAX_CB = SH == 1 && NP == 1 && DP <= 64 ? 2 : 1;
    // wavefronts per SIMD that the registers are bounded for
    static constexpr int FWD_OCC = NP == 1 && SH == 1 ? 2 : DP > 64 ? 1 : 2;
    static constexpr int GRAD_OCC = DP > 64 ? 1 : 2;
};
template <typename T> constexpr int SHARED = PARTS<T> == 1 ? 4 : 2;         // SH where the columns are too few for OWN

// walks the tiles of [key_beg, key_end) that hold a key: move(t, buf, on) starts the loads of the tile at key win + t N, work(buf, on) uses it
template <typename S, typename Move, typename Work>
__device__ __forceinline__ void walk_keys(unsigned* words, const unsigned char* mask, int key_beg, int key_end, Move move, Work work) {
    constexpr int W = S::N / 32;
    for (int win = key_beg; win < key_end; win += 64 * S::N) {
        unsigned long long active = key_window<S::N, S::WAVES>(words, mask, win, key_end);
        unsigned on[W], next[W];
        auto start = [&](int buf, unsigned (&w)[W]) {
            const int t = __builtin_ctzll(active);
            active &= active - 1;
#pragma unroll
            for (int j = 0; j < W; j++) w[j] = win + t * S::N + 32 * j < key_end ? __builtin_amdgcn_readfirstlane(words[t * W + j]) : 0u;
            move(win + t * S::N, buf, w);
        };
        if (!active) continue;
        if constexpr (S::NBUF == 2) {
            int buf = 0;
            start(0, on);
            for (;;) {
                wait_tiles();                                // this tile is in LDS, and nobody reads the other buffer any more
                const bool more = active != 0;
                if (more) start(buf ^ 1, next);
                work(buf, on);
                if (!more) break;
                buf ^= 1;
#pragma unroll
                for (int j = 0; j < W; j++) on[j] = next[j];
            }
        } else {
            for (;;) {
                start(0, on);
                wait_tiles();
                work(0, on);
                if (!active) break;
                __syncthreads();                             // everybody is done with the tile
            }
        }
    }
}

// (a loop over on[] would keep it in memory)
template <int SH> __device__ __forceinline__ unsigned one_of(const unsigned* on, int i) {
    if constexpr (SH == 2) return i == 0 ? on[0] : on[1];
    else return i == 0 ? on[0] : i == 1 ? on[1] : i == 2 ? on[2] : on[3];
}
// factor of a partial softmax with maximum m and sum l in one with maximum `top`.  m is -inf where there was no key (l is 0: nothing to add) or
// where every score was NaN (l is NaN, and so is the result).
__device__ __forceinline__ float share_of(float m, float l, float top) { return m == -INFINITY ? l : __builtin_amdgcn_exp2f(m - top); }

// joins SHARES wavefronts' partials jo [SHARES][ROWS][DP], jm [SHARES][ROWS][maximum, sum] of rows row0 .. into the result, or into this split's partial
template <typename T, int DP, int ROWS, int SHARES>
__device__ __forceinline__ void join_waves(const Args& a, const float* jo, const float* jm, int row0, int split, int bh) {
    const int R = a.Nq * a.G, H = a.Hk * a.G, b = bh / a.Hk, hk = bh - b * a.Hk;
    for (int idx = threadIdx.x; idx < ROWS * (DP / 4); idx += 256) {
        const int row = idx / (DP / 4), d = 4 * (idx % (DP / 4)), rr = row0 + row;
        if (rr >= R || d >= a.D) continue;
        float mt = -INFINITY, lt = 0.f;
#pragma unroll
        for (int i = 0; i < SHARES; i++) mt = fmaxf(mt, jm[(i * ROWS + row) * 2]);
        f32x4 sum = {};
#pragma unroll
        for (int i = 0; i < SHARES; i++) {
            const float* his = jm + (i * ROWS + row) * 2;
            const float f = share_of(his[0], his[1], mt);
            lt += f * his[1];
            if (f != 0.f) sum += f * *reinterpret_cast<const f32x4*>(jo + (i * ROWS + row) * DP + d);
        }
        if (a.nsplit > 1) {
            const long at = ((long)split * a.BH + bh) * R + rr;
            *reinterpret_cast<f32x4*>(a.part_o + at * a.D + d) = sum;
            if (d == 0) {
                a.part_ml[2 * at] = mt;
                a.part_ml[2 * at + 1] = lt;
            }
        } else {
            const int n = rr / a.G, h = hk * a.G + rr - n * a.G;
            sum *= lt == 0.f ? 0.f : 1.f / lt;
            const long at = (((long)b * a.Nq + n) * H + h) * a.D + d;
            Out<T>::store4(static_cast<T*>(a.o) + at, sum[0], sum[1], sum[2], sum[3]);
            if (a.o_low) Out<T>::store_low(a.o_low + at, sum[0], sum[1], sum[2], sum[3]);
            if (a.lse && d == 0) a.lse[(long)bh * R + rr] = lt == 0.f ? INFINITY : mt + __builtin_amdgcn_logf(lt);
        }
    }
}

template <typename T, int DP, int SH, int CB>
__global__ __launch_bounds__(256, (Shape<T, DP, SH>::FWD_OCC)) void forward_kernel(const Args a) {
    typedef Shape<T, DP, SH> S;
    typedef Mma<T, DP, S::N * DP> M;
    constexpr bool SHARE = SH > 1;
    constexpr int WAVES = S::WAVES, N = S::N, DB = M::DB, COLS = S::COLS * CB;
    __shared__ __attribute__((aligned(16))) __bf16 tile[S::NBUF][2][S::NP * N * DP];
    __shared__ unsigned words[2 * N];
    __shared__ float jm[SHARE ? 2 * SH * COLS : 1];

    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Nq * a.G, row_blocks = (R + COLS - 1) / COLS;
    int bh, blk;
    if (!place(a.BH, row_blocks * a.nsplit, bh, blk)) return;
    const int split = SHARE ? blk / row_blocks : 0, rb = blk - split * row_blocks;
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int r_wave = rb * COLS + 32 * CB * (wave / SH);
    const bool idle = r_wave >= R;                           // a wavefront without rows only moves tiles
    const Rows qr = rows_of<__bf16>(a.q, a.qs, b, hk * a.G, a.G);
    const unsigned char* mask = a.mask ? a.mask + (long)b * a.Nk : nullptr;
    const int key_beg = SHARE ? split * a.keys_per_split : 0, key_end = SHARE ? min(a.Nk, key_beg + a.keys_per_split) : a.Nk;
    // a negative scale goes into q's sign: the maximum of s is the maximum of c s; c > 0 keeps -inf * c = -inf for masked keys at scale 0
    const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f);

    typename M::Frag q[CB];
    f32x16 o[CB][DB];
    float m[CB], l[CB];                                      // maximum, sum of p as they are multiplied
#pragma unroll
    for (int x = 0; x < CB; x++) {
        const int r = r_wave + 32 * x + l31;
        M::load(q[x], reinterpret_cast<const __bf16*>(qr.row(r < R ? r : 0)), r < R, a.D, a.scale);
#pragma unroll
        for (int i = 0; i < DB; i++) o[x][i] = f32x16{};
        m[x] = -INFINITY;
        l[x] = 0.f;
    }
    Loader<DP, N, WAVES, S::NP> keys(rows_of<__bf16>(a.k, a.ks, b, hk, 1), a.D), values(rows_of<__bf16>(a.v, a.vs, b, hk, 1), a.D);

    // `blocks` 32-key blocks from row r0 of the tile
    auto products = [&](auto blocks, int buf, int r0, const unsigned* on) {
        constexpr int NKB = decltype(blocks)::value;
        f32x16 s[NKB][CB];
        unsigned all = 0xffffffffu;
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
            M::template dots<CB>(s[kb], tile[buf][0], r0 + 32 * kb, q);
            all &= on[kb];
        }
        if (all != 0xffffffffu) {
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!((on[kb] >> acc_row(i, half)) & 1)) {
#pragma unroll
                        for (int x = 0; x < CB; x++) s[kb][x][i] = -INFINITY;
                    }
        }
        float top[CB];
        bool grow = false;
#pragma unroll
        for (int x = 0; x < CB; x++) {
            top[x] = s[0][x][0];
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++) top[x] = fmaxf(top[x], s[kb][x][i]);
            top[x] = fmaxf(top[x], other_half(top[x])) * c;
            grow |= top[x] > m[x] + RESCALE_THR;
        }
        if (__any(grow)) {
#pragma unroll
            for (int x = 0; x < CB; x++) {
                const float mn = fmaxf(m[x], top[x]);
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[x] - mn);
                l[x] *= alpha;
                m[x] = mn;
#pragma unroll
                for (int i = 0; i < DB; i++)
#pragma unroll
                    for (int j = 0; j < 16; j++) o[x][i][j] *= alpha;
            }
        }
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
#pragma unroll
            for (int x = 0; x < CB; x++) {
                const float base = m[x] == -INFINITY ? 0.f : m[x];
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    s[kb][x][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][x][i], c, -base));
                    if (sizeof(T) == 4) part[i & 3] += s[kb][x][i];
                }
                if (sizeof(T) == 4) l[x] += (part[0] + part[1]) + (part[2] + part[3]);
            }
            M::template adds<CB>(o, tile[buf][1], r0 + 32 * kb, s[kb], l);
        }
    };
    walk_keys<S>(words, mask, key_beg, key_end,
                 [&](int key, int buf, const unsigned (&on)[N / 32]) {
                     keys.issue(tile[buf][0], key, on);
                     values.issue(tile[buf][1], key, on);
                 },
                 [&](int buf, const unsigned (&on)[N / 32]) {
                     if (idle) return;
                     if constexpr (SHARE) {
                         const unsigned mine = one_of<SH>(on, wave % SH);
                         if (mine) products(std::integral_constant<int, 1>{}, buf, 32 * (wave % SH), &mine);
                     } else {
                         products(std::integral_constant<int, N / 32>{}, buf, 0, on);
                     }
                 });
#pragma unroll
    for (int x = 0; x < CB; x++) l[x] += other_half(l[x]);

    const int H = a.Hk * a.G;
    if constexpr (SHARE) {                                   // join the wavefronts' shares of the keys
        float* jo = reinterpret_cast<float*>(&tile[0][0][0]);        // [SH][COLS rows][DP]
        const int share = wave % SH, mine = 32 * (wave / SH) + l31;
        static_assert(sizeof(tile) >= SH * COLS * DP * sizeof(float), "the joined partials fit the tiles");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<f32x4*>(jo + (share * COLS + mine) * DP + 32 * i + 8 * g + 4 * half) =
                    f32x4{o[0][i][4 * g], o[0][i][4 * g + 1], o[0][i][4 * g + 2], o[0][i][4 * g + 3]};
        if (half == 0) {
            jm[(share * COLS + mine) * 2] = m[0];
            jm[(share * COLS + mine) * 2 + 1] = l[0];
        }
        __syncthreads();
        join_waves<T, DP, COLS, SH>(a, jo, jm, rb * COLS, split, bh);
    } else {
#pragma unroll
        for (int x = 0; x < CB; x++) {
            const int r = r_wave + 32 * x + l31, n = r / a.G, h = hk * a.G + r - n * a.G;
            const long at = (((long)b * a.Nq + n) * H + h) * a.D;
            const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
            signed char* low = a.o_low ? a.o_low + at : nullptr;
#pragma unroll
            for (int i = 0; i < DB; i++) Out<T>::store_column(static_cast<T*>(a.o) + at, low, i, a.D, r < R, o[x][i] * inv);
            if (a.lse && half == 0 && r < R) a.lse[(long)bh * R + r] = l[x] == 0.f ? INFINITY : m[x] + __builtin_amdgcn_logf(l[x]);
        }
    }
}

// ---- few rows (single queries) -------------------------------------------------------------------------------------------------------
// With few rows per key / value head nothing is reused: the time is that of reading K and V once, and what counts is how much of them
// is in flight.  No LDS tiles: a group of LPR = DP / 8 lanes holds a key, 8 channels per lane; a wavefront loads UNROLL x 64 / LPR keys and
// their values straight into registers, all loads in flight together, and each group keeps its own softmax of the keys it has seen (fp32
// products and weights); groups, wavefronts and splits are joined at the end.
template <typename T, int DP> struct Few {
    static constexpr int LPR = DP <= 32 ? 4 : DP <= 64 ? 8 : 16, GROUPS = 64 / LPR;
    static constexpr int UNROLL = sizeof(T) == 2 ? 8 : 4, KEYS = UNROLL * GROUPS;       // keys of a wavefront at a time
    static constexpr int NV = 8 * sizeof(T) / 16;                                       // 16-byte pieces of 8 channels
};
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// sum over the LPR neighbouring lanes: lane ^ 1, lane ^ 2, the other quad of 8, the other half of 16
template <int LPR> __device__ __forceinline__ float group_sum(float x) {
    x += dpp<0xB1>(x);
    x += dpp<0x4E>(x);
    if constexpr (LPR >= 8) x += dpp<0x141>(x);
    if constexpr (LPR >= 16) x += dpp<0x140>(x);
    return x;
}
__device__ __forceinline__ float channel(const u32x4 (&x)[1], int i) { return __uint_as_float(i & 1 ? x[0][i / 2] & 0xffff0000u : x[0][i / 2] << 16); }
__device__ __forceinline__ float channel(const u32x4 (&x)[2], int i) { return __uint_as_float(x[i / 4][i & 3]); }
__device__ __forceinline__ float dot8(const u32x4 (&x)[1], const u32x4 (&y)[1]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned u = x[0][i], v = y[0][i];             // (bit_cast of the subscript itself takes element 0 every time)
        s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u), __builtin_bit_cast(bf16x2, v), s, false);
    }
    return s;
}
__device__ __forceinline__ float dot8(const u32x4 (&x)[2], const u32x4 (&y)[2]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s = __builtin_fmaf(channel(x, i), channel(y, i), s);
    return s;
}
template <typename T, int DP, int ROWS> __global__ __launch_bounds__(256, 2) void few_rows_kernel(const Args a) {
    typedef Few<T, DP> S;
    constexpr int UNROLL = S::UNROLL, GROUPS = S::GROUPS, LPR = S::LPR, NV = S::NV;
    __shared__ __attribute__((aligned(16))) float jo[4 * ROWS * DP];
    __shared__ float jm[4 * ROWS * 2];
    const int R = a.Nq * a.G, row_groups = (R + ROWS - 1) / ROWS;
    int bh, blk;
    if (!place(a.BH, a.nsplit * row_groups, bh, blk)) return;
    const int split = blk / row_groups, row0 = ROWS * (blk - split * row_groups);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane / LPR, d = 8 * (lane % LPR);
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const bool has = d < a.D;
    const Rows qr = rows_of<T>(a.q, a.qs, b, hk * a.G, a.G), kr = rows_of<T>(a.k, a.ks, b, hk, 1), vr = rows_of<T>(a.v, a.vs, b, hk, 1);
    const unsigned char* mask = a.mask ? a.mask + (long)b * a.Nk : nullptr;
    const int key_beg = split * a.keys_per_split, key_end = min(a.Nk, key_beg + a.keys_per_split);
    const float c = a.scale * LOG2E;

    u32x4 q[ROWS][NV];
    float m[ROWS], l[ROWS], acc[ROWS][8];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            q[r][i] = u32x4{};
            if (row0 + r < R && has) q[r][i] = *reinterpret_cast<const u32x4*>(qr.row(row0 + r) + d * sizeof(T) + 16 * i);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) acc[r][i] = 0.f;
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    for (int key0 = key_beg + wave * S::KEYS; key0 < key_end; key0 += 4 * S::KEYS) {
        bool on[UNROLL];
        unsigned char byte[UNROLL];
        if (mask) {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) byte[u] = mask[min(key0 + GROUPS * u + g, key_end - 1)];
        }
        bool any = false;
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            on[u] = key0 + GROUPS * u + g < key_end && (!mask || byte[u]);
            any |= on[u];
        }
        if (!__any(any)) continue;
        const __amdgpu_buffer_rsrc_t kb = buffer(kr.base + key0 * kr.ts), vb = buffer(vr.base + key0 * vr.ts);
        u32x4 kx[UNROLL][NV], vx[UNROLL][NV];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const unsigned off = on[u] && has ? (unsigned)(GROUPS * u + g) * (unsigned)kr.ts + d * sizeof(T) : OUT_OF_RANGE;
#pragma unroll
            for (int i = 0; i < NV; i++) kx[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kb, off + 16 * i, 0, 0));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const unsigned off = on[u] && has ? (unsigned)(GROUPS * u + g) * (unsigned)vr.ts + d * sizeof(T) : OUT_OF_RANGE;
#pragma unroll
            for (int i = 0; i < NV; i++) vx[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vb, off + 16 * i, 0, 0));
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            float s[UNROLL], top = m[r];
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                s[u] = on[u] ? c * group_sum<LPR>(dot8(q[r], kx[u])) : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float base = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m[r] - base);
            m[r] = top;
            l[r] *= alpha;
#pragma unroll
            for (int i = 0; i < 8; i++) acc[r][i] *= alpha;
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const float p = __builtin_amdgcn_exp2f(s[u] - base);
                l[r] += p;
#pragma unroll
                for (int i = 0; i < 8; i++) acc[r][i] = __builtin_fmaf(p, channel(vx[u], i), acc[r][i]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {                         // join the groups of the wavefront
        float top = m[r];
#pragma unroll
        for (int x = LPR; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float f = share_of(m[r], l[r], top);
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < 8; i++) acc[r][i] *= f;
#pragma unroll
        for (int x = LPR; x < 64; x <<= 1) {
            l[r] += __shfl_xor(l[r], x);
#pragma unroll
            for (int i = 0; i < 8; i++) acc[r][i] += __shfl_xor(acc[r][i], x);
        }
        if (g == 0 && d < DP) {
            float* to = jo + (wave * ROWS + r) * DP + d;
            *reinterpret_cast<f32x4*>(to) = f32x4{acc[r][0], acc[r][1], acc[r][2], acc[r][3]};
            *reinterpret_cast<f32x4*>(to + 4) = f32x4{acc[r][4], acc[r][5], acc[r][6], acc[r][7]};
        }
        if (lane == 0) {
            jm[(wave * ROWS + r) * 2] = top;
            jm[(wave * ROWS + r) * 2 + 1] = l[r];
        }
    }
    __syncthreads();
    join_waves<T, DP, ROWS, 4>(a, jo, jm, row0, split, bh);
}

// joins the splits: a thread per 4 channels of a row
template <typename T> __global__ __launch_bounds__(256) void join_kernel(const Args a) {
    const int R = a.Nq * a.G, H = a.Hk * a.G, q4 = a.D / 4;
    const long idx = (long)blockIdx.x * 256 + threadIdx.x, rows = (long)a.BH * R;
    const long row = idx / q4;
    if (row >= rows) return;
    const int d = 4 * (int)(idx - row * q4);
    float mt = -INFINITY, lt = 0.f;
    for (int s = 0; s < a.nsplit; s++) mt = fmaxf(mt, a.part_ml[2 * (s * rows + row)]);
    f32x4 sum = {};
    for (int s = 0; s < a.nsplit; s++) {
        const float* ml = a.part_ml + 2 * (s * rows + row);
        const float f = share_of(ml[0], ml[1], mt);
        lt += f * ml[1];
        if (f != 0.f) sum += f * *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * a.D + d);
    }
    const int bh = (int)(row / R), r = (int)(row - (long)bh * R), b = bh / a.Hk, hk = bh - b * a.Hk;
    const int n = r / a.G, h = hk * a.G + r - n * a.G;
    sum *= lt == 0.f ? 0.f : 1.f / lt;
    const long at = (((long)b * a.Nq + n) * H + h) * a.D + d;
    Out<T>::store4(static_cast<T*>(a.o) + at, sum[0], sum[1], sum[2], sum[3]);
    if (a.o_low) Out<T>::store_low(a.o_low + at, sum[0], sum[1], sum[2], sum[3]);
    if (a.lse && d == 0) a.lse[row] = lt == 0.f ? INFINITY : mt + __builtin_amdgcn_logf(lt);
}

// delta[row] = gO . o: DP / 8 lanes per row (rounded up to a power of two), 8 channels each, DELTA_ROWS rows per group of lanes with all their
// loads in flight at once (32 x 642 rows of 6 x 64, bf16: 16 lanes and one row each 10 us); rows in the order of o (a batch entry's tokens, then heads)
constexpr int DELTA_ROWS = 4;
constexpr int delta_lanes(int DP) { return DP <= 32 ? 4 : DP <= 64 ? 8 : 16; }
template <typename T, int DP> __global__ __launch_bounds__(256) void delta_kernel(const Args a, int blocks_per_batch) {
    constexpr int LANES = delta_lanes(DP), GROUPS = 256 / LANES;
    typedef T tx8 __attribute__((ext_vector_type(8)));
    const int H = a.Hk * a.G, R = a.Nq * a.G, l = threadIdx.x % LANES;
    const int b = blockIdx.x / blocks_per_batch;
    const unsigned first = (blockIdx.x - b * blocks_per_batch) * (GROUPS * DELTA_ROWS) + threadIdx.x / LANES, rows = a.Nq * H;
    const int d = 8 * l < a.D ? 8 * l : 0;                   // a lane past the last channel reads the first ones and leaves them out
    unsigned n[DELTA_ROWS], h[DELTA_ROWS];
    typedef signed char cx8 __attribute__((ext_vector_type(8)));
    tx8 x[DELTA_ROWS], y[DELTA_ROWS];
    cx8 z[DELTA_ROWS];
    const bool low = sizeof(T) == 2 && a.o_low_in;
#pragma unroll
    for (int i = 0; i < DELTA_ROWS; i++) {
        const unsigned row = min(first + GROUPS * i, rows - 1);
        n[i] = row / (unsigned)H;
        h[i] = row - n[i] * H;
        x[i] = *reinterpret_cast<const tx8*>(static_cast<const T*>(a.dgo) + b * a.dgs[0] + n[i] * a.dgs[1] + h[i] * a.dgs[2] + d);
        const long at = ((long)b * rows + row) * a.D + d;
        y[i] = *reinterpret_cast<const tx8*>(static_cast<const T*>(a.o_in) + at);
        if (low) z[i] = *reinterpret_cast<const cx8*>(a.o_low_in + at);
    }
#pragma unroll
    for (int i = 0; i < DELTA_ROWS; i++) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) s += (float)x[i][e] * (low ? Out<T>::with_low((float)y[i][e], z[i][e]) : (float)y[i][e]);
        if (8 * l >= a.D) s = 0.f;
#pragma unroll
        for (int k = 1; k < LANES; k <<= 1) s += __shfl_xor(s, k);
        if (l == 0 && first + GROUPS * i < rows) {
            const unsigned hk = h[i] / (unsigned)a.G;
            a.delta[((long)b * a.Hk + hk) * R + n[i] * a.G + (h[i] - hk * a.G)] = s;
        }
    }
}

template <typename T, int DP, int SH> struct GradLds {
    typedef Shape<T, DP, SH> S;
    __bf16 tile[S::NBUF][2][S::NP * S::N * DP];
    float rowstat[S::NBUF][2][S::N < 64 ? 64 : S::N];        // log-sum-exp and delta of the streamed rows
    unsigned words[2 * S::N];
};

// KV: stationary keys, streamed query rows (gk, gv); otherwise stationary query rows, streamed keys (gq)
template <typename T, int DP, bool KV, int SH, bool LOW>
__device__ __forceinline__ void gradient_columns(const Args& a, GradLds<T, DP, SH>& lds, int bh, int blk) {
    typedef Shape<T, DP, SH> S;
    typedef Mma<T, DP, S::N * DP> M;
    constexpr bool SHARE = SH > 1;
    constexpr int WAVES = S::WAVES, N = S::N, DB = M::DB, NRB = SHARE ? 1 : N / 32, W = N / 32;
    auto& tile = lds.tile;
    auto& rowstat = lds.rowstat;

    const int lane = threadIdx.x & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int R = a.Nq * a.G, C = KV ? a.Nk : R;
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int col_wave = blk * S::COLS + 32 * (wave / SH), col = col_wave + l31;
    const unsigned char* mask = a.mask ? a.mask + (long)b * a.Nk : nullptr;
    const bool valid = col < C && (!KV || !mask || mask[col]);
    const bool idle = !__any(valid);                         // a wavefront without columns only moves tiles
    const Rows qr = rows_of<__bf16>(a.q, a.qs, b, hk * a.G, a.G), gr = rows_of<__bf16>(a.go, a.gs, b, hk * a.G, a.G);
    const Rows kr = rows_of<__bf16>(a.k, a.ks, b, hk, 1), vr = rows_of<__bf16>(a.v, a.vs, b, hk, 1);
    const float* lse = a.lse + (long)bh * R;
    const float* delta = a.delta + (long)bh * R;
    const float c = a.scale * LOG2E;

    f32x16 acc1[1][DB], acc2[1][DB];
#pragma unroll
    for (int i = 0; i < DB; i++) acc1[0][i] = acc2[0][i] = f32x16{};
    typename M::Frag f1[1], f2[1];
    {
        const int at = valid ? col : 0;
        M::load(f1[0], reinterpret_cast<const __bf16*>((KV ? kr : qr).row(at)), valid, a.D, 1.f);
        M::load(f2[0], reinterpret_cast<const __bf16*>((KV ? vr : gr).row(at)), valid, a.D, 1.f);
    }
    const float col_lse = !KV && valid ? lse[col] : INFINITY, col_delta = !KV && valid ? delta[col] : 0.f;

    // one 32-row block: p, gs and the products over its rows
    auto block = [&](int buf, int r0, auto masked, unsigned on) {
        f32x16 pp[1], dd[1];
        M::template dots<1>(pp, tile[buf][0], r0, f1);
        M::template dots<1>(dd, tile[buf][1], r0, f2);
        f32x16 &p = pp[0], &ds = dd[0];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            f32x4 ls = {col_lse, col_lse, col_lse, col_lse}, dl = {col_delta, col_delta, col_delta, col_delta};
            if constexpr (KV) {
                ls = *reinterpret_cast<const f32x4*>(&rowstat[buf][0][r0 + 8 * g + 4 * half]);
                dl = *reinterpret_cast<const f32x4*>(&rowstat[buf][1][r0 + 8 * g + 4 * half]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = 4 * g + j;
                p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], c, -ls[j]));
                if constexpr (masked.value)
                    if (!((on >> acc_row(i, half)) & 1)) p[i] = 0.f;
                ds[i] = p[i] * (ds[i] - dl[j]);
            }
        }
        if constexpr (KV) M::template adds<1, LOW>(acc2, tile[buf][1], r0, pp);
        M::template adds<1, LOW>(acc1, tile[buf][0], r0, dd);
    };

    Loader<DP, N, WAVES, S::NP> first(KV ? qr : kr, a.D), second(KV ? gr : vr, a.D);
    if constexpr (KV) {
        if (__syncthreads_or(valid)) {
            auto issue = [&](int r0, int buf) {
                unsigned on[W];
#pragma unroll
                for (int j = 0; j < W; j++) {
                    const int left = R - r0 - 32 * j;
                    on[j] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                }
                first.issue(tile[buf][0], r0, on);
                second.issue(tile[buf][1], r0, on);
                // statistics of the tile's rows, 64 per instruction; 0 past the last row, where q and gO are 0
                constexpr int HALVES = N > 64 ? 2 : 1;
                if (wave < 2 * HALVES) {
                    const int which = wave & 1, part = 64 * (wave >> 1);
                    const unsigned off = part + lane < N && r0 + part + lane < R ? 4u * (part + lane) : OUT_OF_RANGE;
                    to_lds4(off, buffer((which ? delta : lse) + r0), __builtin_amdgcn_readfirstlane(lds_address(&rowstat[buf][which][part])));
                }
            };
            auto products = [&](int buf, int r0) {
                if (idle) return;
                if constexpr (SHARE) {
                    if (r0 + 32 * (wave % SH) < R) block(buf, 32 * (wave % SH), std::false_type{}, 0u);
                } else if (NRB == 1 || r0 + N - 32 < R) {
#pragma unroll
                    for (int rb = 0; rb < NRB; rb++) block(buf, 32 * rb, std::false_type{}, 0u);
                } else {                                     // the rows end in the tile's first half
                    block(buf, 0, std::false_type{}, 0u);
                }
            };
            if constexpr (S::NBUF == 2) {
                issue(0, 0);
                int buf = 0;
                for (int r0 = 0; r0 < R; r0 += N, buf ^= 1) {
                    wait_tiles();
                    if (r0 + N < R) issue(r0 + N, buf ^ 1);
                    products(buf, r0);
                }
            } else {
                for (int r0 = 0; r0 < R; r0 += N) {
                    issue(r0, 0);
                    wait_tiles();
                    products(0, r0);
                    __syncthreads();
                }
            }
        }
    } else {
        walk_keys<S>(lds.words, mask, 0, a.Nk,
                     [&](int key, int buf, const unsigned (&on)[W]) {
                         first.issue(tile[buf][0], key, on);
                         second.issue(tile[buf][1], key, on);
                     },
                     [&](int buf, const unsigned (&on)[W]) {
                         if (idle) return;
                         if constexpr (SHARE) {
                             const unsigned mine = one_of<SH>(on, wave % SH);
                             if (mine == 0xffffffffu) block(buf, 32 * (wave % SH), std::false_type{}, mine);
                             else if (mine) block(buf, 32 * (wave % SH), std::true_type{}, mine);
                         } else {
                             unsigned all = 0xffffffffu;
#pragma unroll
                             for (int j = 0; j < W; j++) all &= on[j];
                             if (all == 0xffffffffu) {
#pragma unroll
                                 for (int rb = 0; rb < NRB; rb++) block(buf, 32 * rb, std::false_type{}, 0u);
                             } else {
#pragma unroll
                                 for (int rb = 0; rb < NRB; rb++)
                                     if (on[rb]) block(buf, 32 * rb, std::true_type{}, on[rb]);
                             }
                         }
                     });
    }

    T* out1 = static_cast<T*>(KV ? a.gk : a.gq);
    T* out2 = static_cast<T*>(a.gv);
    if constexpr (SHARE) {                                   // add up the wavefronts' rows, in order
        float* join = reinterpret_cast<float*>(&tile[0][0][0]);      // [SH][COLS columns][DP]
        constexpr int COLS = S::COLS;
        const int share = wave % SH, at_col = 32 * (wave / SH) + l31;
        static_assert(sizeof(lds.tile) >= SH * COLS * DP * sizeof(float), "the joined partials fit the tiles");
#pragma unroll
        for (int which = 0; which < (KV ? 2 : 1); which++) {
            T* out = which ? out2 : out1;
            if (!out) continue;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < DB; i++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const f32x16& x = which ? acc2[0][i] : acc1[0][i];
                    *reinterpret_cast<f32x4*>(join + (share * COLS + at_col) * DP + 32 * i + 8 * g + 4 * half) = f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
                }
            __syncthreads();
            for (int idx = threadIdx.x; idx < COLS * (DP / 4); idx += 256) {
                const int row = idx / (DP / 4), d = 4 * (idx % (DP / 4)), cc = blk * COLS + row;
                if (cc >= C || d >= a.D) continue;
                f32x4 sum = {};
#pragma unroll
                for (int w = 0; w < SH; w++) sum += *reinterpret_cast<const f32x4*>(join + (w * COLS + row) * DP + d);
                const float f = which ? 1.f : a.scale;
                if (KV && mask && !mask[cc]) sum = f32x4{};
                long at;
                if (KV) at = (((long)b * a.Nk + cc) * a.Hk + hk) * a.D;
                else {
                    const int n = cc / a.G;
                    at = (((long)b * a.Nq + n) * (a.Hk * a.G) + hk * a.G + cc - n * a.G) * a.D;
                }
                Out<T>::store4(out + at + d, sum[0] * f, sum[1] * f, sum[2] * f, sum[3] * f);
            }
        }
        return;
    }
    long at;
    if (KV) at = (((long)b * a.Nk + col) * a.Hk + hk) * a.D;
    else {
        const int n = col / a.G;
        at = (((long)b * a.Nq + n) * (a.Hk * a.G) + hk * a.G + col - n * a.G) * a.D;
    }
#pragma unroll
    for (int which = 0; which < (KV ? 2 : 1); which++) {
        T* out = which ? out2 : out1;
        if (!out) continue;
        const float f = which ? 1.f : a.scale;
#pragma unroll
        for (int i = 0; i < DB; i++)                         // a masked key gets zeros, whatever went through its column
            Out<T>::store_column(out + at, nullptr, i, a.D, col < C, valid ? (which ? acc2[0][i] : acc1[0][i]) * f : f32x16{});
    }
}

// A backward pass over one query runs here too: its query gradient is one workgroup per head that walks the keys tile by tile, and that is its
// time (bf16, 32 x 6 heads of 1 x 1025 64 us, 6 heads of 1 x 4097 66 us in 33 tiles; fp32 189 and 184).
// Both gradients in one launch: the two kinds of workgroups of a head run next to each other, and the last, partly filled round of
// workgroups is paid once (32 x 6 heads of 642 x 1025, bf16: two launches 142 us).
// LOW (bf16): p and gs enter their products with 16 bits instead of 8, 10 products for 7: where there are few rows to sum over, so that single
// roundings show (gv of one query: 2.8e-3 off without it, 1.7e-3, the rounding of gv itself, with it).  32 x 6 heads of 1 x 1025: 65 us for
// 60; 8 x 6 heads of 2562 x 40 would be 112 for 87.
template <typename T, int DP, int SH, bool LOW>
__global__ __launch_bounds__(256, (Shape<T, DP, SH>::GRAD_OCC)) void backward_kernel(const Args a) {
    typedef Shape<T, DP, SH> S;
    __shared__ __attribute__((aligned(16))) GradLds<T, DP, SH> lds;
    const int nkv = a.gk || a.gv ? (a.Nk + S::COLS - 1) / S::COLS : 0, nq = a.gq ? (a.Nq * a.G + S::COLS - 1) / S::COLS : 0;
    int bh, blk;
    if (!place(a.BH, nkv + nq, bh, blk)) return;
    if (blk < nkv) gradient_columns<T, DP, true, SH, LOW>(a, lds, bh, blk);
    else gradient_columns<T, DP, false, SH, LOW>(a, lds, bh, blk - nkv);
}

// ---- launch plan --------------------------------------------------------------------------------------------------------------------
struct Plan { bool share, few, two_blocks; int nsplit, keys_per_split, row_blocks; };
// Rows per key / value head that few_rows_kernel takes, in groups of up to 8 that each read K and V.
// fp32, where the matrix kernels first write the tensors' parts (6 bytes an element) and read them again: 64 x 6 heads of 64 x 4097 keys,
// 1 / 8 / 32 / 64 rows: 144 / 163 / 388 / 742 us against 610 to 619; 32 x 6 x 1025 keys: 23 / 39 / 63 / 110 against 73 to 79.
// bf16, where they read the tensors: 64 x 6 x 4097 keys, 1 / 2 / 4 rows: 76 / 80 / 93 us against 74 to 75, but 32 x 6 x 1025 keys, 1 row:
// 13.5 against 18.5, 32 x 8 heads of 128: 27 against 41; so one row only.
constexpr int few_rows(int size) { return size == 4 ? 32 : 1; }
// Single queries: a workgroup walks its keys in trips of 4 x Few::KEYS, each a memory round trip of 1.5 us, and the join of a split is a second
// launch of 2 to 3 us that reads every part.  So fewer than 4 trips are not split (32 x 6 heads x 257 keys of 64, bf16: whole 7.9 us, split
// 10.5; 4 x 6 heads, fp32 5.8 and 7.6), parts keep 2 trips, there are at most 6 of them (4 x 6 x 4097, bf16, 1 / 4 / 6 / 12 / 16 parts: 33 / 17.7 /
// 16.9 / 19.3 / 23.3 us) and no more workgroups than CUs, beyond which the memory's rate counts (16 x 6 x 4097, bf16, 1 / 2 / 4 / 8: 33.6 /
// 27.3 / 24.4 / 26.3; fp32 40.1 / 36.7 / 37.7 / 38.9; 32 x 6 x 1025, 1 / 2 / 4, bf16 15.5 / 16.1 / 17.2, fp32 20.5 / 22.6 / 22.9).  Against the best
// number of parts that costs 2.5 % on average over 72 shapes of 6 to 384 heads, 257 to 4097 keys, 32 to 128 channels, both types.
inline int few_parts(long blocks, int keys, int few_keys) {
    const long trips = (keys + 4l * few_keys - 1) / (4l * few_keys);
    if (trips < 4) return 1;
    return (int)std::min(std::min((trips + 1) / 2, 6l), std::max(1l, 256 / blocks));
}
// SHARE below so many wavefronts of 32 columns; fewer leave SIMDs empty (256 CUs x 4).  8 x 6 heads of 642 x 1025, bf16: backward pass OWN 72 us,
// SHARE 97; fp32: forward OWN 92, SHARE 98, 4 x 6 heads backward OWN 130, SHARE 120; 512 to 4096 are within 10 % of each other there.
constexpr long SHARE_BELOW = 1024;
constexpr int LOW_ROWS = 16;
inline long wavefronts(const Args& a, int columns) { return (long)a.BH * ((columns + 31) / 32); }
// may_two: the OWN kernel can take two column blocks per wavefront (Shape::MAX_CB); shared: SHARED.
// Two blocks or one: a CU works through its workgroups, so the time goes by the largest number that one CU gets; a workgroup of 128 columns
// takes 0.54 of one of 256 (1025 keys, 64 channels: 12.2 and 22.5 us).  16 / 24 / 32 / 64 x 6 heads of 642 queries: two blocks 45 / 45 /
// 74 / 103 us, one 36 / 49 / 64 / 96; 8 x 6 heads of 2562: 67, 51; 7686 rows x 4097 keys x 16: 154, 172.
// split: where even SHARE has too few workgroups, the keys are divided as long as each part keeps two tiles
inline Plan forward_plan(const Args& a, bool may_two, int shared, int max_few, int few_keys) {
    Plan p;
    const int R = a.Nq * a.G;
    p.two_blocks = false;
    p.few = R <= max_few;
    if (p.few) {
        p.share = false;
        p.row_blocks = R <= 4 ? 1 : (R + 7) / 8;
        const long blocks = (long)a.BH * p.row_blocks;
        const int parts = few_parts(blocks, a.Nk, few_keys);
        p.keys_per_split = ((a.Nk + parts - 1) / parts + 15) / 16 * 16;
        p.nsplit = (a.Nk + p.keys_per_split - 1) / p.keys_per_split;
        return p;
    }
    p.share = wavefronts(a, R) < SHARE_BELOW;
    p.nsplit = 1;
    p.keys_per_split = a.Nk;
    if (may_two && !p.share) {
        const long one = ((long)a.BH * ((R + 127) / 128) + 255) / 256, two = ((long)a.BH * ((R + 255) / 256) + 255) / 256;
        p.two_blocks = 54 * one >= 100 * two;
    }
    const int cols = p.share ? 128 / shared : p.two_blocks ? 256 : 128, tile = 32 * shared;
    p.row_blocks = (R + cols - 1) / cols;
    if (p.share) {
        const int tiles = (a.Nk + tile - 1) / tile;
        const long blocks = (long)a.BH * p.row_blocks;
        // 256 / 512: bf16 4 x 6 heads of 64 x 4097 19 / 22 us, 16 x 6 of 40 x 1025 15 / 18 (the join is a second launch); fp32, whose workgroups take
        // longer, 16 x 6 of 40 x 1025 52 / 47, 4 x 6 of 64 x 4097 56 / 57
        const int target = shared == SHARED<__bf16> ? 256 : 512;
        int want = blocks >= target ? 1 : (int)(target / blocks);
        if (want > tiles / 2) want = tiles / 2 > 0 ? tiles / 2 : 1;
        const int per = (tiles + want - 1) / want;
        p.nsplit = (tiles + per - 1) / per;
        p.keys_per_split = per * tile;
    }
    return p;
}
inline int padded_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

template <typename T, int DP> void launch_forward(const Args& a, const Plan& p, hipStream_t st) {
    const dim3 grid(placed_blocks(a.BH, p.row_blocks * p.nsplit));
    if (p.few) {
        constexpr int DF = DP == 96 ? 128 : DP;              // lanes per key: a power of two
        const int R = a.Nq * a.G;
        if (R == 1) {
            hipLaunchKernelGGL((few_rows_kernel<T, DF, 1>), grid, dim3(256), 0, st, a);
        } else if constexpr (few_rows(sizeof(T)) > 1) {
            if (R == 2) hipLaunchKernelGGL((few_rows_kernel<T, DF, 2>), grid, dim3(256), 0, st, a);
            else if (R <= 4) hipLaunchKernelGGL((few_rows_kernel<T, DF, 4>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((few_rows_kernel<T, DF, 8>), grid, dim3(256), 0, st, a);
        }
    } else if (p.share) hipLaunchKernelGGL((forward_kernel<T, DP, SHARED<T>, 1>), grid, dim3(256), 0, st, a);
    else if (Shape<T, DP, 1>::MAX_CB == 1 || !p.two_blocks) hipLaunchKernelGGL((forward_kernel<T, DP, 1, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((forward_kernel<T, DP, 1, Shape<T, DP, 1>::MAX_CB>), grid, dim3(256), 0, st, a);
    if (p.nsplit > 1) {
        const long n = (long)a.BH * a.Nq * a.G * (a.D / 4);
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    }
}
template <typename T, int DP> void launch_backward(const Args& a, hipStream_t st) {
    const int R = a.Nq * a.G;
    constexpr int PER = 256 / delta_lanes(DP) * DELTA_ROWS;
    const int per_batch = (a.Nq * a.Hk * a.G + PER - 1) / PER;
    hipLaunchKernelGGL((delta_kernel<T, DP>), dim3((unsigned)(per_batch * (a.BH / a.Hk))), dim3(256), 0, st, a, per_batch);
    const int rows = a.gq ? R : 0, keys = a.gk || a.gv ? a.Nk : 0;
    const bool share = wavefronts(a, rows) + wavefronts(a, keys) < 2 * SHARE_BELOW;
    const int cols = share ? 128 / SHARED<T> : 128;
    const dim3 grid(placed_blocks(a.BH, (rows + cols - 1) / cols + (keys + cols - 1) / cols));
    constexpr bool CAN = PARTS<T> == 1;
    const bool low = CAN && (R <= LOW_ROWS || a.Nk <= LOW_ROWS);
    if (share && low) hipLaunchKernelGGL((backward_kernel<T, DP, SHARED<T>, CAN>), grid, dim3(256), 0, st, a);
    else if (share) hipLaunchKernelGGL((backward_kernel<T, DP, SHARED<T>, false>), grid, dim3(256), 0, st, a);
    else if (low) hipLaunchKernelGGL((backward_kernel<T, DP, 1, CAN>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((backward_kernel<T, DP, 1, false>), grid, dim3(256), 0, st, a);
}

// instantiated in csrc/cross_attn_f32.hip and csrc/cross_attn_bf16.hip
template <typename T> void run_forward(const Args& a, const Plan& p, hipStream_t st);
template <typename T> void run_backward(const Args& a, hipStream_t st);

#define SCP_ATTN_INSTANTIATE(T)                                                                  \
    namespace scp_attn {                                                                         \
    template <> void run_forward<T>(const Args& a, const Plan& p, hipStream_t st) {              \
        switch (padded_dim(a.D)) {                                                               \
            case 32: launch_forward<T, 32>(a, p, st); break;                                     \
            case 64: launch_forward<T, 64>(a, p, st); break;                                     \
            case 96: launch_forward<T, 96>(a, p, st); break;                                     \
            default: launch_forward<T, 128>(a, p, st); break;                                    \
        }                                                                                        \
    }                                                                                            \
    template <> void run_backward<T>(const Args& a, hipStream_t st) {                            \
        switch (padded_dim(a.D)) {                                                               \
            case 32: launch_backward<T, 32>(a, st); break;                                       \
            case 64: launch_backward<T, 64>(a, st); break;                                       \
            case 96: launch_backward<T, 96>(a, st); break;                                       \
            default: launch_backward<T, 128>(a, st); break;                                      \
        }                                                                                        \
    }                                                                                            \
    }

}  // namespace scp_attn
