// self-corr-pose_amd/csrc/vit_ops_binding.cpp -- the autograd nodes and argument checks of scp_amd/vit_ops.py.
//
// Many of these calls take less time on the GPU than Python needs to make them (LayerNorm of a class token: 4 us), and a backward pass runs
// on the engine's own thread, where every Python step costs two to three times what it does on the caller's.  So what stands between a
// caller and the C entry points of include/scp_hip.h -- checks, allocation from torch's caching allocator, autograd nodes -- is compiled:
// against the same in Python, a LayerNorm of 4 x 384 takes 7.7 us for 12, forward + backward of 8209 x 1001 bf16 65 us for 98, gelu8 of
// 1025 x 1536 48 us for 78; autograd's engine alone is about 44 of the last two.
// The entry points come from the library that scp_amd/capi.py has loaded (init()); nothing here is linked to it.
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <torch/version.h>

#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "scp_hip.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---- the library's entry points --------------------------------------------------------------------------------------------------------
#define SCP_ENTRIES(X)                                                                                                               \
    X(scp_last_error) X(scp_layernorm_forward) X(scp_layernorm_backward_workspace) X(scp_layernorm_backward)                         \
    X(scp_cross_attention_forward_workspace) X(scp_cross_attention_forward) X(scp_cross_attention_backward_workspace)                \
    X(scp_cross_attention_backward) X(scp_pack8) X(scp_unpack8) X(scp_gelu8_forward) X(scp_gelu8_backward) X(scp_weight_grad8_workspace) X(scp_weight_grad8)
struct Entries {
#define X(name) decltype(&::name) name##_;
    SCP_ENTRIES(X)
#undef X
} lib;

void init(const py::dict& addresses) {
#define X(name) lib.name##_ = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<size_t>());
    SCP_ENTRIES(X)
#undef X
}

// ---- checks ----------------------------------------------------------------------------------------------------------------------------
[[noreturn]] void refuse(const std::string& why) { throw std::runtime_error(why); }
void check(int code, const char* what) {
    if (code) refuse(std::string("scp_amd: ") + what + " failed (hip error " + std::to_string(code) + "): " + lib.scp_last_error_());
}
std::string text(at::ScalarType t) {
    const std::string s = at::toString(t);
    return t == at::kFloat ? "float32" : t == at::kBFloat16 ? "bfloat16" : t == at::kBool ? "bool" : t == at::kChar ? "int8" : t == at::kByte ? "uint8" : s;
}
std::string text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}
// the tensor behind a Python object: on the current device, of one of the types, and with nothing attached that would be lost
Tensor tensor(const py::handle& o, const char* name, std::initializer_list<at::ScalarType> types) {
    if (!THPVariable_Check(o.ptr())) refuse(std::string(name) + " must be a CUDA tensor (no CPU fallback)");
    const Tensor& t = THPVariable_Unpack(o.ptr());
    if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor (no CPU fallback)");
    bool ok = false;
    std::string want;
    for (auto type : types) ok |= t.scalar_type() == type;
    if (!ok) {
        for (auto type : types) want += (want.empty() ? "" : " or ") + text(type);
        refuse(std::string(name) + " must be " + want + ", not " + text(t.scalar_type()));
    }
    const int device = c10::hip::current_device();
    if (t.get_device() != device)
        refuse(std::string(name) + " lives on cuda:" + std::to_string(t.get_device()) + " but the current device is cuda:" + std::to_string(device) +
               " (torch.cuda.set_device first)");
    // a subclass that answers for its operations itself, a wrapper of torch.func, a zero tensor: a null pointer would pass for an operand that is
    // left out
    constexpr c10::DispatchKeySet others({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::ZeroTensor});
    if (t.key_set().has_any(others)) refuse(std::string(name) + " is a tensor without memory of its own");
    // autograd's nodes of this file know neither: without the refusal the tangent would be dropped, the traced result kept as a constant
    if (t._fw_grad(/*level=*/0).defined()) refuse(std::string(name) + " has a forward-mode tangent: the operators of scp_amd.vit_ops have no forward-mode derivative");
    if (torch::jit::tracer::isTracing()) refuse(std::string(name) + ": the operators of scp_amd.vit_ops cannot be traced (torch.jit.trace)");
    return t.is_neg() ? t.resolve_neg() : t;
}
Tensor operand(const py::handle& o, const char* name) { return tensor(o, name, {at::kFloat, at::kBFloat16}); }
Tensor operand_like(const py::handle& o, const char* name, const Tensor& like) { return tensor(o, name, {like.scalar_type()}); }

int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? SCP_DTYPE_F32 : SCP_DTYPE_BF16; }
void* stream() { return c10::hip::getCurrentHIPStream().stream(); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({(long)bytes}, like.options().dtype(at::kByte)) : Tensor(); }
bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// a tensor that may be missing, as Function::apply takes it: a missing one is no variable, and needs_input_grad() does not count it
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor plain(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
int64_t present(std::initializer_list<Tensor> ts) {
    int64_t bits = 0, i = 0;
    for (const Tensor& t : ts) bits |= (int64_t)t.defined() << i++;
    return bits;
}
struct Wanted {                                                      // asked for the tensors in order
    AutogradContext* ctx;
    int64_t bits;
    size_t next = 0;
    bool operator()() {
        const bool is = bits & 1;
        bits >>= 1;
        return is && ctx->needs_input_grad(next++);
    }
};
// an incoming gradient as its memory holds it: autograd hands on tensors whose negation is only a bit of theirs
Tensor resolved(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// A backward pass that is being captured must not reach a leaf whose gradient accumulator belongs to the default stream: one made by an eager
// graph of the same leaf that is still alive.  The engine would have the default stream wait for the capturing one, which ends the process.
void check_capture() {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream().stream(), &status) != hipSuccess) {
        (void)hipGetLastError();                                        // (the default stream while another thread captures: not this call's error)
        return;
    }
    if (status == hipStreamCaptureStatusNone) return;
    const auto self = torch::autograd::get_current_node();
    if (!self) return;
    const auto* plan = torch::autograd::get_current_graph_task_exec_info();     // empty: everything runs
    auto runs = [&](torch::autograd::Node* node) {
        if (!plan || plan->empty()) return true;
        const auto it = plan->find(node);
        return it != plan->end() && it->second.should_execute();
    };
    std::vector<torch::autograd::Node*> todo{self.get()};
    std::unordered_set<torch::autograd::Node*> seen{self.get()};
    while (!todo.empty()) {
        torch::autograd::Node* node = todo.back();
        todo.pop_back();
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node)) {
            const auto stream = node->stream();
            if (stream && stream->id() == 0)
                refuse("scp_amd.vit_ops: this backward pass is being captured, and a graph made on the default stream from the same leaf is alive: delete its "
                       "results first, or capture with leaves of their own (detach().requires_grad_())");
        }
        for (const auto& edge : node->next_edges())
            if (edge.function && runs(edge.function.get()) && seen.insert(edge.function.get()).second) todo.push_back(edge.function.get());
    }
}
// Gradients of a backward pass that is itself recorded (create_graph) cannot be differentiated again: they get a node that says so.
variable_list first_order(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    const auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice an operator of scp_amd.vit_ops: they are once differentiable",
                                                                      grads.size());
    return (*node)(std::move(grads));
}

// ---- layer norm ------------------------------------------------------------------------------------------------------------------------
struct NormOut { Tensor total, y, stats; };
NormOut norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, double eps, bool keep) {
    const int64_t c = x.size(-1), rows = x.numel() / c;
    const Tensor& w = weight.defined() ? weight : bias;
    NormOut r;
    r.y = at::empty_like(x);
    if (residual.defined()) r.total = at::empty_like(x);
    if (keep) r.stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    if (rows)
        check(lib.scp_layernorm_forward_(x.data_ptr(), ptr(residual), ptr(weight), ptr(bias), (float)eps, rows, (int)c, type_of(x), w.defined() ? type_of(w) : type_of(x),
                                         ptr(r.total), r.y.data_ptr(), ptr<float>(r.stats), stream()),
              "scp_layernorm_forward");
    return r;
}

struct LayerNorm : Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual_, const Maybe& weight_, const Maybe& bias_, double eps) {
        const Tensor residual = plain(residual_), weight = plain(weight_), bias = plain(bias_);
        NormOut r = norm_forward(x, residual, weight, bias, eps, true);
        ctx->save_for_backward({r.total.defined() ? r.total : x, weight, r.stats});
        ctx->saved_data["present"] = present({x, residual, weight, bias});
        ctx->saved_data["bias"] = bias.defined() ? (int64_t)bias.scalar_type() : (int64_t)-1;
        ctx->set_materialize_grads(false);
        if (r.total.defined()) return {r.total, r.y};
        return {r.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_capture();
        Wanted wanted{ctx, ctx->saved_data["present"].toInt()};
        const bool want_x = wanted(), want_r = wanted(), want_w = wanted(), want_b = wanted();
        const Tensor gsum = grads.size() == 2 ? resolved(grads[0]) : Tensor(), gy = resolved(grads.back());
        if (!gy.defined()) return {want_x ? gsum : Tensor(), want_r ? gsum : Tensor(), {}, {}, {}};            // only the sum was used
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &s = saved[0], &weight = saved[1], &stats = saved[2];
        const int64_t c = s.size(-1), rows = s.numel() / c, bias = ctx->saved_data["bias"].toInt();
        const int dtype = type_of(s), wdtype = weight.defined() ? type_of(weight) : dtype;
        Tensor gx, gw, gb;
        const auto sums = s.options().dtype(at::kFloat);
        if (want_x || want_r) gx = at::empty_like(s);
        if (want_w) gw = rows ? at::empty({c}, sums) : at::zeros({c}, sums);
        if (want_b) gb = rows ? at::empty({c}, sums) : at::zeros({c}, sums);
        if (rows) {
            const Tensor g = gy.contiguous(), gs = gsum.defined() ? gsum.contiguous() : Tensor();
            const size_t bytes = want_w || want_b ? lib.scp_layernorm_backward_workspace_(rows, (int)c) : 0;
            const Tensor ws = workspace(bytes, s);
            check(lib.scp_layernorm_backward_(s.data_ptr(), ptr(weight), g.data_ptr(), ptr(gs), ptr<const float>(stats), rows, (int)c, dtype, wdtype, ptr(gx), ptr<float>(gw),
                                              ptr<float>(gb), ptr(ws), bytes, stream()),
                  "scp_layernorm_backward");
        }
        if (want_w && weight.scalar_type() != at::kFloat) gw = gw.to(weight.scalar_type());
        if (want_b && bias != (int64_t)at::kFloat) gb = gb.to((at::ScalarType)bias);
        return first_order({want_x ? gx : Tensor(), want_r ? gx : Tensor(), gw, gb, {}});
    }
};

py::object layer_norm(const py::object& x_, const py::object& weight_, const py::object& bias_, double eps, const py::object& residual_) {
    Tensor x = operand(x_, "layer_norm: x"), weight, bias, residual;
    if (x.dim() < 1 || x.size(-1) < 1) refuse("layer_norm: x needs a last dimension of at least one channel");
    const int64_t c = x.size(-1);
    if (c > 8192) refuse("layer_norm: at most 8192 channels, got " + std::to_string(c));
    auto affine = [&](const py::object& o, const char* name) {
        Tensor t = tensor(o, (std::string("layer_norm: ") + name).c_str(), {at::kFloat, x.scalar_type()});
        if (t.dim() != 1 || t.size(0) != c) refuse(std::string("layer_norm: ") + name + " must have " + std::to_string(c) + " entries");
        return t.contiguous();
    };
    if (!weight_.is_none()) weight = affine(weight_, "weight");
    if (!bias_.is_none()) bias = affine(bias_, "bias");
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) refuse("layer_norm: weight and bias must have one type");
    if (!residual_.is_none()) {
        residual = operand_like(residual_, "layer_norm: residual", x);
        if (residual.sizes() != x.sizes()) refuse("layer_norm: residual must have x's shape " + text(x.sizes()) + ", not " + text(residual.sizes()));
        residual = residual.contiguous();
    }
    x = x.contiguous();
    Tensor total, y;
    {
        py::gil_scoped_release release;
        if (wants_grad({x, residual, weight, bias})) {
            const variable_list r = LayerNorm::apply(x, maybe(residual), maybe(weight), maybe(bias), eps);
            if (r.size() == 2) total = r[0];
            y = r.back();
        } else {
            const NormOut r = norm_forward(x, residual, weight, bias, eps, false);
            total = r.total;
            y = r.y;
        }
    }
    return residual.defined() ? py::object(py::make_tuple(total, y)) : py::cast(y);
}

// ---- cross attention -------------------------------------------------------------------------------------------------------------------
// t itself when the kernels can address it (channels contiguous, pointer and strides multiples of 16 bytes, 130 tokens of all heads within
// 2^31 bytes), else a contiguous copy (contiguous() would return a misaligned tensor as it is)
Tensor addressable(const Tensor& t) {
    const int64_t size = t.element_size(), sb = t.stride(0), sn = t.stride(1), sh = t.stride(2);
    if (t.stride(3) == 1 && !(((int64_t)(size_t)t.data_ptr() | sb * size | sn * size | sh * size) & 15) && (130 * sn + t.size(2) * sh) * size < 1l << 31) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}
void strides(const Tensor& t, long long* to) {
    for (int i = 0; i < 3; i++) to[i] = t.stride(i);
}
scp_cross_attn_params attention_params(const Tensor& q, const Tensor& k, const Tensor& v, double scale) {
    scp_cross_attn_params p{};
    p.batch = (int)q.size(0);
    p.queries = (int)q.size(1);
    p.keys = (int)k.size(1);
    p.heads = (int)q.size(2);
    p.kv_heads = (int)k.size(2);
    p.head_dim = (int)q.size(3);
    p.dtype = type_of(q);
    p.scale = (float)scale;
    strides(q, p.q_stride);
    strides(k, p.k_stride);
    strides(v, p.v_stride);
    return p;
}
struct AttnOut { Tensor out, low, lse; };
AttnOut attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, double scale, bool keep) {
    AttnOut r;
    r.out = at::empty(q.sizes(), q.options());
    if (r.out.numel() == 0) return r;
    if (k.size(1) == 0) {
        r.out.zero_();
        return r;
    }
    if (keep) r.lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    if (keep && q.scalar_type() == at::kBFloat16) r.low = at::empty(q.sizes(), q.options().dtype(at::kChar));
    const scp_cross_attn_params p = attention_params(q, k, v, scale);
    const size_t bytes = lib.scp_cross_attention_forward_workspace_(&p);
    const Tensor ws = workspace(bytes, q);
    check(lib.scp_cross_attention_forward_(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr<unsigned char>(mask), &p, r.out.data_ptr(), ptr<signed char>(r.low), ptr<float>(r.lse),
                                           ptr(ws), bytes, stream()),
          "scp_cross_attention_forward");
    return r;
}

struct CrossAttention : Function<CrossAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& mask_, double scale) {
        const Tensor mask = plain(mask_);
        if (q.numel() && k.size(1)) {                                   // the backward pass must be possible too (its gradient comes dense or is copied)
            scp_cross_attn_params p = attention_params(q, k, v, scale);
            p.g_stride[2] = q.size(3);
            p.g_stride[1] = q.size(2) * p.g_stride[2];
            p.g_stride[0] = q.size(1) * p.g_stride[1];
            if (!lib.scp_cross_attention_backward_workspace_(&p)) refuse("cross_attention: q " + text(q.sizes()) + " with k " + text(k.sizes()) + " is too large for the backward pass");
        }
        AttnOut r = attention_forward(q, k, v, mask, scale, true);
        ctx->save_for_backward({q, k, v, mask, r.out, r.low, r.lse});
        ctx->saved_data["scale"] = scale;
        return {r.out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_capture();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor q = addressable(saved[0]), k = addressable(saved[1]), v = addressable(saved[2]);             // a hook may have moved them
        const Tensor &mask = saved[3], &out = saved[4], &low = saved[5], &lse = saved[6];
        Tensor gq, gk, gv;
        if (ctx->needs_input_grad(0)) gq = at::empty(q.sizes(), q.options());
        if (ctx->needs_input_grad(1)) gk = at::empty(k.sizes(), k.options());
        if (ctx->needs_input_grad(2)) gv = at::empty(v.sizes(), v.options());
        if (!lse.defined()) {                                          // no query or no key: nothing depends on the other side
            for (Tensor* g : {&gq, &gk, &gv})
                if (g->defined()) g->zero_();
        } else {
            const Tensor g = addressable(resolved(grads[0]));
            scp_cross_attn_params p = attention_params(q, k, v, ctx->saved_data["scale"].toDouble());
            strides(g, p.g_stride);
            const size_t bytes = lib.scp_cross_attention_backward_workspace_(&p);
            const Tensor ws = workspace(bytes, q);
            check(lib.scp_cross_attention_backward_(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr<unsigned char>(mask), out.data_ptr(), ptr<signed char>(low), ptr<const float>(lse),
                                                    g.data_ptr(), &p, ptr(gq), ptr(gk), ptr(gv), ptr(ws), bytes, stream()),
                  "scp_cross_attention_backward");
        }
        return first_order({gq, gk, gv, {}, {}});
    }
};

Tensor cross_attention(const py::object& q_, const py::object& k_, const py::object& v_, const py::object& scale_, const py::object& mask_) {
    Tensor q = operand(q_, "cross_attention: q"), k = operand_like(k_, "cross_attention: k", q), v = operand_like(v_, "cross_attention: v", q), mask;
    if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) refuse("cross_attention: q, k and v must be [batch, tokens, heads, channels]");
    const int64_t b = q.size(0), h = q.size(2), d = q.size(3), nk = k.size(1), hk = k.size(2);
    if (k.sizes() != v.sizes() || k.size(0) != b || k.size(3) != d)
        refuse("cross_attention: q " + text(q.sizes()) + " does not go with k " + text(k.sizes()) + " and v " + text(v.sizes()));
    if (hk == 0 || h % hk) refuse("cross_attention: " + std::to_string(h) + " query heads are no multiple of " + std::to_string(hk) + " key heads");
    if (d < 8 || d > 128 || d % 8) refuse("cross_attention: head dimension " + std::to_string(d) + "; a multiple of 8 up to 128 is needed");
    for (int64_t n : {b, q.size(1), nk, h})
        if (n > INT32_MAX) refuse("cross_attention: more than 2^31 tokens, heads or batch entries");
    if (!mask_.is_none()) {
        mask = tensor(mask_, "cross_attention: key_mask", {at::kBool});
        if (mask.dim() != 2 || mask.size(0) != b || mask.size(1) != nk)
            refuse("cross_attention: key_mask must be [" + std::to_string(b) + ", " + std::to_string(nk) + "], not " + text(mask.sizes()));
        mask = mask.contiguous();
    }
    const double scale = scale_.is_none() ? 1.0 / std::sqrt((double)d) : scale_.cast<double>();
    py::gil_scoped_release release;
    q = addressable(q);
    k = addressable(k);
    v = addressable(v);
    if (wants_grad({q, k, v})) return CrossAttention::apply(q, k, v, maybe(mask), scale)[0];
    return attention_forward(q, k, v, mask, scale, false).out;
}

// ---- 8-bit activation checkpoints --------------------------------------------------------------------------------------------------------
struct Packed { Tensor codes, exps; };
Packed packed_like(const Tensor& x) {
    std::vector<int64_t> e = x.sizes().vec();
    e.back() = (e.back() + 31) / 32;
    return {at::empty(x.sizes(), x.options().dtype(at::kChar)), at::empty(e, x.options().dtype(at::kByte))};
}
Tensor rows_of(const py::handle& o, const char* name) {
    Tensor x = operand(o, name);
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 1 << 24) refuse(std::string(name) + " needs a last dimension of 1 to 2^24 channels");
    return x;
}
void check_packed(const Tensor& codes, const Tensor& exps, const std::string& what) {
    std::vector<int64_t> e = codes.sizes().vec();
    if (!e.empty()) e.back() = (e.back() + 31) / 32;
    if (codes.dim() < 1 || exps.sizes() != at::IntArrayRef(e))
        refuse(what + ": exps " + text(exps.sizes()) + " do not go with codes " + text(codes.sizes()));
    if (!codes.is_contiguous() || !exps.is_contiguous()) refuse(what + ": codes and exps must be contiguous");
}

Packed pack(const Tensor& x) {                                       // contiguous
    Packed p = packed_like(x);
    if (x.numel())
        check(lib.scp_pack8_(x.data_ptr(), x.numel() / x.size(-1), (int)x.size(-1), type_of(x), ptr<signed char>(p.codes), ptr<unsigned char>(p.exps), stream()), "scp_pack8");
    return p;
}
py::tuple pack8(const py::object& x_) {
    const Packed p = pack(rows_of(x_, "pack8: x").detach().contiguous());
    return py::make_tuple(p.codes, p.exps);
}
Tensor unpack8(const py::object& codes_, const py::object& exps_, bool bf16) {
    const Tensor codes = tensor(codes_, "Packed8.unpack: codes", {at::kChar}), exps = tensor(exps_, "Packed8.unpack: exps", {at::kByte});
    check_packed(codes, exps, "Packed8.unpack");
    const Tensor x = at::empty(codes.sizes(), codes.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
    if (x.numel())
        check(lib.scp_unpack8_(ptr<signed char>(codes), ptr<unsigned char>(exps), x.numel() / x.size(-1), (int)x.size(-1), type_of(x), x.data_ptr(), stream()), "scp_unpack8");
    return x;
}

Tensor gelu_forward(const Tensor& x, Packed* keep) {
    Tensor y = at::empty(x.sizes(), x.options());
    if (keep) *keep = packed_like(x);
    if (x.numel())
        check(lib.scp_gelu8_forward_(x.data_ptr(), x.numel() / x.size(-1), (int)x.size(-1), type_of(x), y.data_ptr(), keep ? ptr<signed char>(keep->codes) : nullptr,
                                     keep ? ptr<unsigned char>(keep->exps) : nullptr, stream()),
              "scp_gelu8_forward");
    return y;
}
struct Gelu8 : Function<Gelu8> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x) {
        Packed p;
        Tensor y = gelu_forward(x, &p);
        ctx->save_for_backward({p.codes, p.exps});
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_capture();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor gy = resolved(grads[0]).contiguous();
        Tensor gx = at::empty(gy.sizes(), gy.options());
        if (gy.numel())
            check(lib.scp_gelu8_backward_(ptr<signed char>(saved[0]), ptr<unsigned char>(saved[1]), gy.data_ptr(), gy.numel() / gy.size(-1), (int)gy.size(-1), type_of(gy),
                                          gx.data_ptr(), stream()),
                  "scp_gelu8_backward");
        return first_order({gx});
    }
};
Tensor gelu8(const py::object& x_) {
    Tensor x = rows_of(x_, "gelu8: x");
    py::gil_scoped_release release;
    x = x.contiguous();
    return wants_grad({x}) ? Gelu8::apply(x)[0] : gelu_forward(x, nullptr);
}

struct WeightGrad { Tensor gw, gb; };
WeightGrad weight_grad(Tensor grad, Tensor codes, const Tensor& exps, bool bias) {
    const int64_t n = grad.size(-1), k = codes.size(-1), rows = grad.numel() / n;
    const auto sums = grad.options().dtype(at::kFloat);
    if (rows == 0) return {at::zeros({n, k}, sums), bias ? at::zeros({n}, sums) : Tensor()};
    grad = grad.contiguous();
    // the kernel reads 16 bytes of grad and 8 codes of a row at a time: narrower rows are widened with zeros
    const int64_t pad_n = std::max<int64_t>(0, 16 / grad.element_size() - n), pad_k = std::max<int64_t>(0, 8 - k);
    if (pad_n) grad = at::constant_pad_nd(grad, {0, pad_n});
    if (pad_k) codes = at::constant_pad_nd(codes, {0, pad_k});
    const int N = (int)(n + pad_n), K = (int)(k + pad_k), dtype = type_of(grad);
    WeightGrad r{at::empty({N, K}, sums), bias ? at::empty({N}, sums) : Tensor()};
    const size_t bytes = lib.scp_weight_grad8_workspace_(rows, N, K, dtype);
    const Tensor ws = workspace(bytes, grad);
    check(lib.scp_weight_grad8_(grad.data_ptr(), ptr<signed char>(codes), ptr<unsigned char>(exps), rows, N, K, dtype, ptr<float>(r.gw), ptr<float>(r.gb), ptr(ws), bytes,
                                stream()),
          "scp_weight_grad8");
    if (pad_n || pad_k) {
        r.gw = r.gw.slice(0, 0, n).slice(1, 0, k).contiguous();
        if (bias) r.gb = r.gb.slice(0, 0, n).contiguous();
    }
    return r;
}
py::tuple weight_grad8(const py::object& grad_, const py::object& codes_, const py::object& exps_, bool bias) {
    const Tensor grad = operand(grad_, "weight_grad8: grad"), codes = tensor(codes_, "weight_grad8: packed: codes", {at::kChar}),
                 exps = tensor(exps_, "weight_grad8: packed: exps", {at::kByte});
    check_packed(codes, exps, "weight_grad8: packed");
    if (grad.dim() < 1 || grad.sizes().slice(0, grad.dim() - 1) != codes.sizes().slice(0, codes.dim() - 1) || grad.size(-1) < 1 || codes.size(-1) < 1 ||
        grad.size(-1) > 1 << 20 || codes.size(-1) > 1 << 20)
        refuse("weight_grad8: grad " + text(grad.sizes()) + " does not go with a packed input " + text(codes.sizes()));
    const WeightGrad r = weight_grad(grad.detach(), codes, exps, bias);
    return py::make_tuple(r.gw, r.gb.defined() ? py::cast(r.gb) : py::none());
}

// the library products run in their operands' type under autocast too
struct OwnType { c10::impl::ExcludeDispatchKeyGuard guard{c10::DispatchKey::AutocastCUDA}; };
// t [..., c] as a contiguous matrix.  The library products are two-dimensional: a strided tensor of more dimensions would become a batched
// product with a transposed view as its right operand, which has faulted the GPU in bf16.
Tensor as_matrix(const Tensor& t) {
    const int64_t c = t.size(-1);
    return t.contiguous().view({t.numel() / c, c});
}
std::vector<int64_t> with_last(const Tensor& like, int64_t c) {
    std::vector<int64_t> s = like.sizes().vec();
    s.back() = c;
    return s;
}
Tensor linear(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    const Tensor y = bias.defined() ? at::linear(as_matrix(x), weight, bias) : at::linear(as_matrix(x), weight);
    return at::_unsafe_view(y, with_last(x, weight.size(0)));                       // not a view of it: a caller may change the result in place
}

struct Linear8 : Function<Linear8> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias_, bool keep) {
        const Tensor bias = plain(bias_);
        Packed p;
        if (keep) p = pack(x.contiguous());
        ctx->save_for_backward({weight, p.codes, p.exps});
        ctx->saved_data["present"] = present({x, weight, bias});
        return {linear(x, weight, bias)};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_capture();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &weight = saved[0];
        Wanted wanted{ctx, ctx->saved_data["present"].toInt()};
        const bool want_x = wanted(), want_w = wanted(), want_b = wanted();
        Tensor gx, gw, gb;
        {
            at::NoGradGuard no;
            const OwnType own_type;
            const Tensor gy = as_matrix(resolved(grads[0]));
            if (want_x) gx = at::_unsafe_view(gy.mm(weight), with_last(grads[0], weight.size(1)));
            if (want_w || want_b) {
                Tensor codes = saved[1], exps = saved[2];
                if (!want_w) {                                          // a bias alone: its column sums beside the narrowest weight gradient
                    codes = at::zeros({gy.size(0), 8}, gy.options().dtype(at::kChar));
                    exps = at::zeros({gy.size(0), 1}, gy.options().dtype(at::kByte));
                }
                WeightGrad r = weight_grad(gy, codes, exps, want_b);
                if (want_w) gw = r.gw.to(weight.scalar_type());
                if (r.gb.defined()) gb = r.gb.to(weight.scalar_type());
            }
        }
        return first_order({gx, gw, gb, {}});
    }
};
Tensor linear8(const py::object& x_, const py::object& weight_, const py::object& bias_) {
    const Tensor x = rows_of(x_, "linear8: x"), weight = operand_like(weight_, "linear8: weight", x);
    Tensor bias;
    if (weight.dim() != 2 || weight.size(1) != x.size(-1) || weight.size(0) < 1)
        refuse("linear8: weight " + text(weight.sizes()) + " does not go with x " + text(x.sizes()));
    if (!bias_.is_none()) {
        bias = operand_like(bias_, "linear8: bias", x);
        if (bias.dim() != 1 || bias.size(0) != weight.size(0)) refuse("linear8: bias must have " + std::to_string(weight.size(0)) + " entries");
    }
    const bool sums = wants_grad({weight, bias});
    if (sums && (x.size(-1) > 1 << 20 || weight.size(0) > 1 << 20 || weight.numel() > 1l << 34))
        refuse("linear8: a gradient of weight " + text(weight.sizes()) + "; at most 2^20 rows and columns and 2^34 entries are possible");
    py::gil_scoped_release release;
    const OwnType own_type;
    if (sums || wants_grad({x})) return Linear8::apply(x, weight, maybe(bias), wants_grad({weight}))[0];
    return linear(x, weight, bias);
}

}  // namespace

PYBIND11_MODULE(scp_vit_ops, m) {
    py::list entries;
#define X(name) entries.append(#name);
    SCP_ENTRIES(X)
#undef X
    m.attr("entries") = entries;
    m.attr("torch_version") = TORCH_VERSION;                           // of the headers
    m.def("init", &init);
    m.def("layer_norm", &layer_norm);
    m.def("cross_attention", &cross_attention);
    m.def("pack8", &pack8);
    m.def("unpack8", &unpack8);
    m.def("gelu8", &gelu8);
    m.def("weight_grad8", &weight_grad8);
    m.def("linear8", &linear8);
}
