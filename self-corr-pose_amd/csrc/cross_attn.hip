// self-corr-pose_amd/csrc/cross_attn.hip -- attention of a set of queries to another set of tokens, forward and backward.
//
//   s[r][j] = scale q_r . k_j  (-inf where key j is masked),  p = softmax_j(s),  o_r = sum_j p[r][j] v_j,  L_r = log2 sum_j 2^(s log2 e)
//   gv_j = sum_r p[r][j] go_r,   gs = p (go_r . v_j - go_r . o_r),   gq_r = scale sum_j gs k_j,   gk_j = scale sum_r gs q_r
// Query heads that share a key / value head are extra ROWS of it: row r of head hk is query r / G of query head hk G + r % G, so the sums
// of a shared head's gradient are ordinary sums over rows.  A batch entry whose keys are all masked gives zeros, and zero gradients.
// Masked keys are never read into a product: an infinity or NaN stored there does not reach any result.
#include <hip/hip_runtime.h>

#include "scp_common.h"
#include "scp_hip.h"
#include "vec_io.h"

namespace {

using scp::VecIO;
constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
    const void *q, *k, *v, *go;
    const unsigned char* mask;
    const void* o_in;
    void *o, *gq, *gk, *gv;
    float *lse, *delta;
    long qs[3], ks[3], vs[3], gs[3];      // strides in elements: batch, token, head
    int Nq, Nk, Hk, G, D;
    float scale;
};

template <typename T> __device__ __forceinline__ const T* row_of(const void* base, const long* st, int b, int n, int h) {
    return static_cast<const T*>(base) + b * st[0] + n * st[1] + h * st[2];
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}
template <typename T> __device__ __forceinline__ float dot(const T* a, const T* b, int D) {
    float s = 0.f;
    for (int d = 0; d < D; d++) s += VecIO<T>::one(a + d) * VecIO<T>::one(b + d);
    return s;
}

// one wavefront per row: scores of 64 keys, a lane each; the products with v lane = channel (two channels per lane)
template <typename T> __global__ __launch_bounds__(64) void attn_forward_kernel(const AttnArgs a) {
    const int R = a.Nq * a.G, lane = threadIdx.x;
    const int r = blockIdx.x % R, bh = blockIdx.x / R, hk = bh % a.Hk, b = bh / a.Hk;
    const int n = r / a.G, h = hk * a.G + r % a.G, H = a.Hk * a.G;
    const T* q = row_of<T>(a.q, a.qs, b, n, h);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = 0; j0 < a.Nk; j0 += 64) {
        const int j = j0 + lane;
        const bool on = j < a.Nk && (!a.mask || a.mask[(long)b * a.Nk + j]);
        const float s = on ? dot<T>(q, row_of<T>(a.k, a.ks, b, j, hk), a.D) * a.scale * LOG2E : -INFINITY;
        const float mt = fmaxf(m, wave_max(s));
        if (!__any(on)) continue;
        const float alpha = exp2f(m - mt), p = on ? exp2f(s - mt) : 0.f;
        l = l * alpha + wave_sum(p);
        o0 *= alpha;
        o1 *= alpha;
        m = mt;
        const unsigned long long bits = __ballot(on);
        for (int t = 0; t < 64; t++) {
            const float pt = __shfl(p, t);
            if (!((bits >> t) & 1)) continue;
            const T* v = row_of<T>(a.v, a.vs, b, j0 + t, hk);
            if (lane < a.D) o0 += pt * VecIO<T>::one(v + lane);
            if (lane + 64 < a.D) o1 += pt * VecIO<T>::one(v + lane + 64);
        }
    }
    T* o = static_cast<T*>(a.o) + (((long)b * a.Nq + n) * H + h) * a.D;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    if (lane < a.D) VecIO<T>::put(o + lane, o0 * inv);
    if (lane + 64 < a.D) VecIO<T>::put(o + lane + 64, o1 * inv);
    if (a.lse && lane == 0) a.lse[(long)bh * R + r] = l == 0.f ? INFINITY : m + log2f(l);
}

// delta_r = go_r . o_r
template <typename T> __global__ __launch_bounds__(64) void attn_delta_kernel(const AttnArgs a) {
    const int R = a.Nq * a.G, lane = threadIdx.x;
    const int r = blockIdx.x % R, bh = blockIdx.x / R, hk = bh % a.Hk, b = bh / a.Hk;
    const int n = r / a.G, h = hk * a.G + r % a.G, H = a.Hk * a.G;
    const T* g = row_of<T>(a.go, a.gs, b, n, h);
    const T* o = static_cast<const T*>(a.o_in) + (((long)b * a.Nq + n) * H + h) * a.D;
    float s = 0.f;
    for (int d = lane; d < a.D; d += 64) s += VecIO<T>::one(g + d) * VecIO<T>::one(o + d);
    s = wave_sum(s);
    if (lane == 0) a.delta[(long)bh * R + r] = s;
}

template <typename T> __global__ __launch_bounds__(64) void attn_gq_kernel(const AttnArgs a) {
    const int R = a.Nq * a.G, lane = threadIdx.x;
    const int r = blockIdx.x % R, bh = blockIdx.x / R, hk = bh % a.Hk, b = bh / a.Hk;
    const int n = r / a.G, h = hk * a.G + r % a.G, H = a.Hk * a.G;
    const T* q = row_of<T>(a.q, a.qs, b, n, h);
    const T* g = row_of<T>(a.go, a.gs, b, n, h);
    const float lse = a.lse[(long)bh * R + r], delta = a.delta[(long)bh * R + r];
    float g0 = 0.f, g1 = 0.f;
    for (int j0 = 0; j0 < a.Nk; j0 += 64) {
        const int j = j0 + lane;
        const bool on = j < a.Nk && (!a.mask || a.mask[(long)b * a.Nk + j]);
        float ds = 0.f;
        if (on) {
            const float p = exp2f(dot<T>(q, row_of<T>(a.k, a.ks, b, j, hk), a.D) * a.scale * LOG2E - lse);
            ds = p * (dot<T>(g, row_of<T>(a.v, a.vs, b, j, hk), a.D) - delta) * a.scale;
        }
        const unsigned long long bits = __ballot(on);
        for (int t = 0; t < 64; t++) {
            const float dt = __shfl(ds, t);
            if (!((bits >> t) & 1)) continue;
            const T* k = row_of<T>(a.k, a.ks, b, j0 + t, hk);
            if (lane < a.D) g0 += dt * VecIO<T>::one(k + lane);
            if (lane + 64 < a.D) g1 += dt * VecIO<T>::one(k + lane + 64);
        }
    }
    T* o = static_cast<T*>(a.gq) + (((long)b * a.Nq + n) * H + h) * a.D;
    if (lane < a.D) VecIO<T>::put(o + lane, g0);
    if (lane + 64 < a.D) VecIO<T>::put(o + lane + 64, g1);
}

// one wavefront per key
template <typename T> __global__ __launch_bounds__(64) void attn_gkv_kernel(const AttnArgs a) {
    const int R = a.Nq * a.G, lane = threadIdx.x;
    const int j = blockIdx.x % a.Nk, bh = blockIdx.x / a.Nk, hk = bh % a.Hk, b = bh / a.Hk;
    const bool on = !a.mask || a.mask[(long)b * a.Nk + j];
    const T* k = row_of<T>(a.k, a.ks, b, j, hk);
    const T* v = row_of<T>(a.v, a.vs, b, j, hk);
    float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
    for (int r0 = 0; on && r0 < R; r0 += 64) {
        const int r = r0 + lane;
        float p = 0.f, ds = 0.f;
        if (r < R) {
            const int n = r / a.G, h = hk * a.G + r % a.G;
            p = exp2f(dot<T>(row_of<T>(a.q, a.qs, b, n, h), k, a.D) * a.scale * LOG2E - a.lse[(long)bh * R + r]);
            ds = p * (dot<T>(row_of<T>(a.go, a.gs, b, n, h), v, a.D) - a.delta[(long)bh * R + r]) * a.scale;
        }
        for (int t = 0; t < 64 && r0 + t < R; t++) {
            const float pt = __shfl(p, t), dt = __shfl(ds, t);
            const int n = (r0 + t) / a.G, h = hk * a.G + (r0 + t) % a.G;
            const T* q = row_of<T>(a.q, a.qs, b, n, h);
            const T* g = row_of<T>(a.go, a.gs, b, n, h);
            if (lane < a.D) { v0 += pt * VecIO<T>::one(g + lane); k0 += dt * VecIO<T>::one(q + lane); }
            if (lane + 64 < a.D) { v1 += pt * VecIO<T>::one(g + lane + 64); k1 += dt * VecIO<T>::one(q + lane + 64); }
        }
    }
    const long at = (((long)b * a.Nk + j) * a.Hk + hk) * a.D;
    T* gk = a.gk ? static_cast<T*>(a.gk) + at : nullptr;
    T* gv = a.gv ? static_cast<T*>(a.gv) + at : nullptr;
    if (gk && lane < a.D) VecIO<T>::put(gk + lane, k0);
    if (gk && lane + 64 < a.D) VecIO<T>::put(gk + lane + 64, k1);
    if (gv && lane < a.D) VecIO<T>::put(gv + lane, v0);
    if (gv && lane + 64 < a.D) VecIO<T>::put(gv + lane + 64, v1);
}

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
bool misaligned(const void* p) { return (reinterpret_cast<size_t>(p) & 15) != 0; }

AttnArgs make_args(const scp_cross_attn_params* p) {
    AttnArgs a{};
    for (int i = 0; i < 3; i++) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.gs[i] = p->g_stride[i]; }
    a.Nq = p->queries;
    a.Nk = p->keys;
    a.Hk = p->kv_heads;
    a.G = p->heads / p->kv_heads;
    a.D = p->head_dim;
    a.scale = p->scale;
    return a;
}

}  // namespace

extern "C" size_t scp_cross_attention_forward_workspace(const scp_cross_attn_params* p) { return 0; }

extern "C" int scp_cross_attention_forward(const void* q, const void* k, const void* v, const unsigned char* key_mask,
                                           const scp_cross_attn_params* p, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                           void* stream) {
    if (const char* why = bad_problem(p)) return scp::fail(hipErrorInvalidValue, why);
    if (!q || !k || !v || !out) return scp::fail(hipErrorInvalidValue, "cross_attention_forward: null argument");
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out))
        return scp::fail(hipErrorInvalidValue, "cross_attention_forward: tensors must be 16-byte aligned");
    AttnArgs a = make_args(p);
    a.q = q;
    a.k = k;
    a.v = v;
    a.mask = key_mask;
    a.o = out;
    a.lse = lse;
    const dim3 grid((unsigned)(p->batch * a.Hk * (a.Nq * a.G)));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->dtype == SCP_DTYPE_F32) hipLaunchKernelGGL(attn_forward_kernel<float>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(attn_forward_kernel<__bf16>, grid, dim3(64), 0, st, a);
    return scp::check_launch("cross_attention_forward");
}

extern "C" size_t scp_cross_attention_backward_workspace(const scp_cross_attn_params* p) {
    if (bad_problem(p)) return 0;
    return (size_t)p->batch * p->heads * p->queries * sizeof(float);
}

extern "C" int scp_cross_attention_backward(const void* q, const void* k, const void* v, const unsigned char* key_mask, const void* out,
                                            const float* lse, const void* g_out, const scp_cross_attn_params* p, void* g_q, void* g_k,
                                            void* g_v, void* workspace, size_t workspace_bytes, void* stream) {
    if (const char* why = bad_problem(p)) return scp::fail(hipErrorInvalidValue, why);
    if (!q || !k || !v || !out || !lse || !g_out) return scp::fail(hipErrorInvalidValue, "cross_attention_backward: null argument");
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(g_out) || misaligned(g_q) || misaligned(g_k) || misaligned(g_v))
        return scp::fail(hipErrorInvalidValue, "cross_attention_backward: tensors must be 16-byte aligned");
    if (!workspace || workspace_bytes < scp_cross_attention_backward_workspace(p))
        return scp::fail(hipErrorInvalidValue, "cross_attention_backward: workspace too small");
    AttnArgs a = make_args(p);
    a.q = q;
    a.k = k;
    a.v = v;
    a.mask = key_mask;
    a.o_in = out;
    a.lse = const_cast<float*>(lse);
    a.go = g_out;
    a.delta = static_cast<float*>(workspace);
    a.gq = g_q;
    a.gk = g_k;
    a.gv = g_v;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 rows((unsigned)(p->batch * a.Hk * (a.Nq * a.G))), keys((unsigned)(p->batch * a.Hk * a.Nk));
    const bool f32 = p->dtype == SCP_DTYPE_F32;
    if (f32) hipLaunchKernelGGL(attn_delta_kernel<float>, rows, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(attn_delta_kernel<__bf16>, rows, dim3(64), 0, st, a);
    if (g_q) {
        if (f32) hipLaunchKernelGGL(attn_gq_kernel<float>, rows, dim3(64), 0, st, a);
        else hipLaunchKernelGGL(attn_gq_kernel<__bf16>, rows, dim3(64), 0, st, a);
    }
    if (g_k || g_v) {
        if (f32) hipLaunchKernelGGL(attn_gkv_kernel<float>, keys, dim3(64), 0, st, a);
        else hipLaunchKernelGGL(attn_gkv_kernel<__bf16>, keys, dim3(64), 0, st, a);
    }
    return scp::check_launch("cross_attention_backward");
}
