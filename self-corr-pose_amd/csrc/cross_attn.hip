// self-corr-pose_amd/csrc/cross_attn.hip -- attention of a set of queries to another set of tokens, forward and backward.
//
//   s[r][j] = scale q_r . k_j  (-inf where key j is masked),  p = softmax_j(s),  o_r = sum_j p[r][j] v_j,  L_r = log2 sum_j 2^(s log2 e)
//   gv_j = sum_r p[r][j] go_r,   gs = p (go_r . v_j - go_r . o_r),   gq_r = scale sum_j gs k_j,   gk_j = scale sum_r gs q_r
// Query heads that share a key / value head are extra ROWS of it: row r of head hk is query r / G of query head hk G + r % G, so the sums
// of a shared head's gradient are ordinary sums over rows.  A batch entry whose keys are all masked gives zeros, and zero gradients.
// Masked keys are never read into a product: an infinity or NaN stored there does not reach any result.
// The kernels are in csrc/attn_core.h; this file checks the arguments and launches.
#include <hip/hip_runtime.h>

#include "attn_core.h"
#include "scp_common.h"
#include "scp_hip.h"

namespace scp_attn {
template <> void run_forward<float>(const Args&, const Plan&, hipStream_t);
template <> void run_forward<__bf16>(const Args&, const Plan&, hipStream_t);
template <> void run_backward<float>(const Args&, hipStream_t);
template <> void run_backward<__bf16>(const Args&, hipStream_t);
}  // namespace scp_attn

namespace {

using scp_attn::Args;
using scp_attn::Plan;

const char* bad_problem(const scp_cross_attn_params* p) {
    if (!p) return "cross_attention: null parameters";
    if (p->batch <= 0 || p->queries <= 0 || p->keys <= 0 || p->heads <= 0 || p->kv_heads <= 0) return "cross_attention: empty problem";
    if (p->heads % p->kv_heads) return "cross_attention: heads must be a multiple of kv_heads";
    if (p->dtype != SCP_DTYPE_F32 && p->dtype != SCP_DTYPE_BF16) return "cross_attention: unknown type";
    if (p->head_dim <= 0 || p->head_dim > 128 || p->head_dim % 8) return "cross_attention: head_dim must be a multiple of 8 up to 128";
    const int unit = p->dtype == SCP_DTYPE_F32 ? 4 : 8;
    for (int i = 0; i < 3; i++)
        if (p->q_stride[i] % unit || p->k_stride[i] % unit || p->v_stride[i] % unit || p->g_stride[i] % unit)
            return "cross_attention: strides must be multiples of 16 bytes";
    const long long lim = 1ll << 31, R = (long long)p->queries * (p->heads / p->kv_heads), bh = (long long)p->batch * p->kv_heads;
    if (R >= lim / 128 || p->keys >= lim / 128 || bh >= lim / 128 || bh * R >= lim || bh * p->keys >= lim)
        return "cross_attention: more than 2^31 rows or keys over all heads";
    return nullptr;
}
// a tile (at most 128 rows) is addressed with 31-bit byte offsets behind its first row; the tile's own place is a 64-bit address
bool tile_too_wide(const scp_cross_attn_params* p, bool backward) {
    const long long size = p->dtype == SCP_DTYPE_F32 ? 4 : 2, lim = 1ll << 31, G = p->heads / p->kv_heads;
    if (size == 4 && 130ll * p->heads * p->head_dim * 6 >= lim) return true;                 // a tile of the parts
    for (const long long* st : {p->k_stride, p->v_stride})
        if (st[1] < 0 || 128 * st[1] * size >= lim) return true;
    if (backward)
        for (const long long* st : {p->q_stride, p->g_stride})
            if (st[1] < 0 || st[2] < 0 || (129 * st[1] + G * st[2]) * size >= lim) return true;
    return false;
}
// a launch has fewer than 2^32 threads: fewer than 2^24 workgroups of 256
constexpr long long MOST_BLOCKS = (1ll << 24) - 1;
long long per_group(long long n, long long group) { return (n + group - 1) / group; }
int parts_rows(int D) { return 256 / (D <= 32 ? 4 : D <= 64 ? 8 : 16); }                     // rows per workgroup of parts_kernel
// workgroups of the kernel that cuts q (and g_out), k and v into parts; 0 in bf16
long long parts_blocks(const scp_cross_attn_params* p, bool backward) {
    if (p->dtype != SCP_DTYPE_F32) return 0;
    const long long rows = (long long)p->batch * p->queries * p->heads, keys = (long long)p->batch * p->keys * p->kv_heads;
    return (backward ? 2 : 1) * per_group(rows, parts_rows(p->head_dim)) + 2 * per_group(keys, parts_rows(p->head_dim));
}
bool too_many_blocks_forward(const scp_cross_attn_params* p, const Args& a, const Plan& plan) {
    const long long heads = a.BH >= 16 ? per_group(a.BH, 8) * 8 : a.BH;
    return heads * plan.row_blocks * plan.nsplit > MOST_BLOCKS || (!plan.few && parts_blocks(p, false) > MOST_BLOCKS) ||
           (plan.nsplit > 1 && per_group((long long)a.BH * a.Nq * a.G * (a.D / 4), 256) > MOST_BLOCKS);
}
// (for all three gradients in workgroups of 128 columns; narrower ones are taken for small problems only)
bool too_many_blocks_backward(const scp_cross_attn_params* p) {
    const long long R = (long long)p->queries * (p->heads / p->kv_heads), bh = (long long)p->batch * p->kv_heads, heads = bh >= 16 ? per_group(bh, 8) * 8 : bh;
    return heads * (per_group(R, 128) + per_group(p->keys, 128)) > MOST_BLOCKS || parts_blocks(p, true) > MOST_BLOCKS ||
           p->batch * per_group((long long)p->queries * p->heads, parts_rows(p->head_dim) * scp_attn::DELTA_ROWS) > MOST_BLOCKS;
}
bool misaligned(const void* p) { return (reinterpret_cast<size_t>(p) & 15) != 0; }

Args make_args(const scp_cross_attn_params* p) {
    Args a{};
    for (int i = 0; i < 3; i++) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.gs[i] = p->g_stride[i]; }
    a.Nq = p->queries;
    a.Nk = p->keys;
    a.Hk = p->kv_heads;
    a.G = p->heads / p->kv_heads;
    a.D = p->head_dim;
    a.scale = p->scale;
    a.BH = p->batch * a.Hk;
    a.nsplit = 1;
    return a;
}
Plan plan_of(const Args& a, int dtype) {
    const bool bf16 = dtype == SCP_DTYPE_BF16;
    const int few_keys = (bf16 ? 8 : 4) * 64 / (a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16);                          // Few::KEYS
    return scp_attn::forward_plan(a, bf16 && a.D <= 64, bf16 ? scp_attn::SHARED<__bf16> : scp_attn::SHARED<float>, scp_attn::few_rows(bf16 ? 2 : 4),
                                  few_keys);
}
size_t split_floats(const Args& a, const Plan& p) { return p.nsplit > 1 ? (size_t)p.nsplit * a.BH * a.Nq * a.G * (a.D + 2) : 0; }


// fp32 tensors as three bf16 parts: dst [batch][tokens][heads][3][D]; a thread per 8 channels, 256 / lanes rows per workgroup
struct Parts { const float* src[4]; __bf16* dst[4]; long st[4][3]; int tokens[4], heads[4]; unsigned first[5]; int batch, D; };
__global__ __launch_bounds__(256) void parts_kernel(const Parts a) {
    int t = 0;
#pragma unroll
    for (int i = 1; i < 4; i++) t += blockIdx.x >= a.first[i];
    const int lanes = a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16, d = 8 * (threadIdx.x % lanes);
    const unsigned heads = a.heads[t], per = (unsigned)a.tokens[t] * heads;
    const unsigned row = (blockIdx.x - a.first[t]) * (256 / lanes) + threadIdx.x / lanes;
    if (row >= per * (unsigned)a.batch || d >= a.D) return;
    const unsigned b = row / per, r = row - b * per, n = r / heads, h = r - n * heads;
    const float* x = a.src[t] + b * a.st[t][0] + n * a.st[t][1] + h * a.st[t][2] + d;
    const scp_attn::f32x4 lo = *reinterpret_cast<const scp_attn::f32x4*>(x), hi = *reinterpret_cast<const scp_attn::f32x4*>(x + 4);
    scp_attn::u32x4 parts[3];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        unsigned w[3];
        if (j < 2) scp_attn::three_parts(lo[2 * j], lo[2 * j + 1], w);
        else scp_attn::three_parts(hi[2 * j - 4], hi[2 * j - 3], w);
#pragma unroll
        for (int k = 0; k < 3; k++) parts[k][j] = w[k];
    }
    __bf16* to = a.dst[t] + (long)row * 3 * a.D + d;
#pragma unroll
    for (int k = 0; k < 3; k++) *reinterpret_cast<scp_attn::u32x4*>(to + k * a.D) = parts[k];
}
// bytes of the parts of q (and g_out), k and v
size_t parts_bytes(const scp_cross_attn_params* p, bool backward) {
    if (p->dtype != SCP_DTYPE_F32) return 0;
    return (size_t)p->batch * ((size_t)p->queries * p->heads * (backward ? 2 : 1) + 2 * (size_t)p->keys * p->kv_heads) * p->head_dim * 6;
}
// makes the parts at `to` and points the matrix kernels at them
void make_parts(Args& a, const scp_cross_attn_params* p, bool backward, void* to, hipStream_t st) {
    Parts c{};
    const void** view[4] = {&a.q, &a.k, &a.v, &a.go};
    long* strides[4] = {a.qs, a.ks, a.vs, a.gs};
    __bf16* at = static_cast<__bf16*>(to);
    c.batch = p->batch;
    c.D = p->head_dim;
    unsigned blocks = 0;
    for (int t = 0; t < 4; t++) {
        c.first[t] = t < 3 || backward ? blocks : ~0u;
        if (t == 3 && !backward) break;
        const bool keys = t == 1 || t == 2;
        c.tokens[t] = keys ? p->keys : p->queries;
        c.heads[t] = keys ? p->kv_heads : p->heads;
        c.src[t] = static_cast<const float*>(*view[t]);
        c.dst[t] = at;
        for (int i = 0; i < 3; i++) c.st[t][i] = strides[t][i];
        const long rows = (long)p->batch * c.tokens[t] * c.heads[t], row = 3l * p->head_dim;
        blocks += (unsigned)((rows + parts_rows(c.D) - 1) / parts_rows(c.D));
        *view[t] = at;
        strides[t][2] = row;
        strides[t][1] = row * c.heads[t];
        strides[t][0] = strides[t][1] * c.tokens[t];
        at += rows * row;
    }
    hipLaunchKernelGGL(parts_kernel, dim3(blocks), dim3(256), 0, st, c);
}

}  // namespace

extern "C" size_t scp_cross_attention_forward_workspace(const scp_cross_attn_params* p) {
    if (bad_problem(p)) return 0;
    const Args a = make_args(p);
    const Plan plan = plan_of(a, p->dtype);
    return (plan.few ? 0 : parts_bytes(p, false)) + split_floats(a, plan) * sizeof(float);
}

extern "C" int scp_cross_attention_forward(const void* q, const void* k, const void* v, const unsigned char* key_mask,
                                           const scp_cross_attn_params* p, void* out, signed char* out_low, float* lse, void* workspace,
                                           size_t workspace_bytes, void* stream) {
    if (const char* why = bad_problem(p)) return scp::fail(hipErrorInvalidValue, why);
    if (!q || !k || !v || !out) return scp::fail(hipErrorInvalidValue, "cross_attention_forward: null argument");
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(out_low) || misaligned(workspace))
        return scp::fail(hipErrorInvalidValue, "cross_attention_forward: tensors must be 16-byte aligned");
    if (tile_too_wide(p, false)) return scp::fail(hipErrorInvalidValue, "cross_attention_forward: token stride of k or v too large");
    Args a = make_args(p);
    const Plan plan = plan_of(a, p->dtype);
    if (too_many_blocks_forward(p, a, plan)) return scp::fail(hipErrorInvalidValue, "cross_attention_forward: more than 2^24 workgroups");
    const size_t parts = plan.few ? 0 : parts_bytes(p, false), need = parts + split_floats(a, plan) * sizeof(float);
    if (need && (!workspace || workspace_bytes < need))
        return scp::fail(hipErrorInvalidValue, "cross_attention_forward: workspace too small");
    a.q = q;
    a.k = k;
    a.v = v;
    a.mask = key_mask;
    a.o = out;
    a.o_low = p->dtype == SCP_DTYPE_F32 ? nullptr : out_low;
    a.lse = lse;
    a.nsplit = plan.nsplit;
    a.keys_per_split = plan.keys_per_split;
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + parts);
    a.part_ml = a.part_o + (size_t)plan.nsplit * a.BH * a.Nq * a.G * a.D;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (parts) {
        make_parts(a, p, false, workspace, st);
        if (const int e = scp::check_launch("cross_attention_forward parts")) return e;
    }
    if (p->dtype == SCP_DTYPE_F32) scp_attn::run_forward<float>(a, plan, st);
    else scp_attn::run_forward<__bf16>(a, plan, st);
    return scp::check_launch("cross_attention_forward");
}

extern "C" size_t scp_cross_attention_backward_workspace(const scp_cross_attn_params* p) {
    if (bad_problem(p) || tile_too_wide(p, true) || too_many_blocks_backward(p)) return 0;
    return parts_bytes(p, true) + (size_t)p->batch * p->heads * p->queries * sizeof(float);
}

extern "C" int scp_cross_attention_backward(const void* q, const void* k, const void* v, const unsigned char* key_mask, const void* out,
                                            const signed char* out_low, const float* lse, const void* g_out, const scp_cross_attn_params* p, void* g_q, void* g_k,
                                            void* g_v, void* workspace, size_t workspace_bytes, void* stream) {
    if (const char* why = bad_problem(p)) return scp::fail(hipErrorInvalidValue, why);
    if (!q || !k || !v || !out || !lse || !g_out) return scp::fail(hipErrorInvalidValue, "cross_attention_backward: null argument");
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(out_low) || misaligned(g_out) || misaligned(workspace) || misaligned(g_q) || misaligned(g_k) || misaligned(g_v))
        return scp::fail(hipErrorInvalidValue, "cross_attention_backward: tensors must be 16-byte aligned");
    if (tile_too_wide(p, true)) return scp::fail(hipErrorInvalidValue, "cross_attention_backward: token or head stride too large");
    if (too_many_blocks_backward(p)) return scp::fail(hipErrorInvalidValue, "cross_attention_backward: more than 2^24 workgroups");
    if (!g_q && !g_k && !g_v) return 0;
    if (!workspace || workspace_bytes < scp_cross_attention_backward_workspace(p))
        return scp::fail(hipErrorInvalidValue, "cross_attention_backward: workspace too small");
    Args a = make_args(p);
    a.q = q;
    a.k = k;
    a.v = v;
    a.mask = key_mask;
    a.o_in = out;
    a.o_low_in = out_low;
    a.lse = const_cast<float*>(lse);
    a.go = a.dgo = g_out;
    for (int i = 0; i < 3; i++) a.dgs[i] = a.gs[i];
    const size_t parts = parts_bytes(p, true);
    a.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + parts);
    a.gq = g_q;
    a.gk = g_k;
    a.gv = g_v;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (parts) {
        make_parts(a, p, true, workspace, st);
        if (const int e = scp::check_launch("cross_attention_backward parts")) return e;
    }
    if (p->dtype == SCP_DTYPE_F32) scp_attn::run_backward<float>(a, st);
    else scp_attn::run_backward<__bf16>(a, st);
    return scp::check_launch("cross_attention_backward");
}
