"""scp_amd/vit_ops.py -- the operators of a transformer block WITH gradients: what training a ViT, or a decoder that attends to its tokens,
needs next to the forward-only operators of scp_amd.dino (the reference's blocks, vision_transformer_flexible.py:54-132, are ordinary
modules; its pipeline keeps them frozen).

  layer_norm       LayerNorm, alone or with the residual add in front of it          (csrc/layernorm_train.hip)
  cross_attention  queries of one length against keys / values of another            (csrc/cross_attn.hip)
  gelu8            erf GELU whose input is kept for the backward pass in 8 bits       (csrc/act8.hip)
  linear8          linear layer whose input is kept for the backward pass in 8 bits   (csrc/act8_wgrad.hip)
  pack8, Packed8, weight_grad8: the 8-bit checkpoint by itself, and the weight gradient taken from it

float32 and bfloat16 GPU tensors on the current device only, anything else raises RuntimeError (no CPU fallback).  Statistics, softmax and
sums are fp32; results are rounded once to the type they are returned in.  No atomics: a call repeated gives the same bits.  Launches
go to the current stream; workspaces come from torch's allocator, so a call can be captured into a HIP graph.  Once differentiable."""
import ctypes

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import capi

_F32_BF16 = (torch.float32, torch.bfloat16)


def _tensor(t, name, dtypes=_F32_BF16):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor (no CPU fallback)" % name)
    if t.dtype not in dtypes:
        raise RuntimeError("%s must be %s, not %s" % (name, " or ".join(str(d)[6:] for d in dtypes), t.dtype))
    if t.get_device() != torch._C._cuda_getDevice():
        raise RuntimeError("%s lives on cuda:%d but the current device is cuda:%d (torch.cuda.set_device first)"
                           % (name, t.device.index, torch.cuda.current_device()))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    """capi.current_stream() without the Python stream object (3 us of a call whose kernel may take 4)"""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _first_order(f):
    """backward(ctx, *grads) that refuses to be differentiated again.  torch's once_differentiable does that for a pass that records a
    graph (create_graph=True); any other pass skips its bookkeeping.  A backward pass runs on the engine's thread, where every
    Python step costs two to three times what it does on the caller's, so these functions do little: what can be prepared is
    prepared in the forward pass."""
    guarded = once_differentiable(f)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else f(ctx, *grads)
    return backward


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
def _norm_forward(x, residual, weight, bias, eps, want_stats):
    c = x.shape[-1]
    rows = x.numel() // c
    dtype = capi.DTYPES[x.dtype]
    w = weight if weight is not None else bias
    wdtype = dtype if w is None else capi.DTYPES[w.dtype]
    y = torch.empty_like(x)
    total = None if residual is None else torch.empty_like(x)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if want_stats else None
    if rows:
        code = capi.lib().scp_layernorm_forward(x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias), eps, rows, c, dtype, wdtype, _ptr(total),
                                                y.data_ptr(), _ptr(stats), _stream())
        if code:
            capi.check(code, "scp_layernorm_forward")
    return total, y, stats, (rows, c, dtype, wdtype)


class _LayerNorm(Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        total, y, stats, ctx.sizes = _norm_forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(x if total is None else total, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        if residual is None:
            return y
        return total, y

    @staticmethod
    @_first_order
    def backward(ctx, *grads):
        s, weight, stats = ctx.saved_tensors
        want_x, want_r, want_w, want_b = ctx.needs_input_grad[:4]
        gsum, gy = grads if len(grads) == 2 else (None, grads[0])
        if gy is None:                                           # only the sum was used
            return gsum, gsum if want_r else None, None, None, None
        rows, c, dtype, wdtype = ctx.sizes
        dev = s.device
        gx = torch.empty_like(s) if want_x or want_r else None
        if rows == 0:
            zero = torch.zeros(c, dtype=torch.float32, device=dev)
            gw, gb = zero, zero.clone()
        else:
            gy = gy.contiguous()
            if gsum is not None:
                gsum = gsum.contiguous()
            gw = torch.empty(c, dtype=torch.float32, device=dev) if want_w else None
            gb = torch.empty(c, dtype=torch.float32, device=dev) if want_b else None
            L = capi.lib()
            ws, nbytes = None, 0
            if want_w or want_b:
                nbytes = L.scp_layernorm_backward_workspace(rows, c)
                if nbytes:
                    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            code = L.scp_layernorm_backward(s.data_ptr(), _ptr(weight), gy.data_ptr(), _ptr(gsum), stats.data_ptr(), rows, c, dtype, wdtype, _ptr(gx),
                                            _ptr(gw), _ptr(gb), _ptr(ws), nbytes, _stream())
            if code:
                capi.check(code, "scp_layernorm_backward")
        if wdtype:                                               # bf16 weights get bf16 gradients
            gw = None if not want_w else gw.to(weight.dtype)
            gb = None if not want_b else gb.to(ctx.bias_dtype)
        return gx if want_x else None, gx if want_r else None, gw if want_w else None, gb if want_b else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-6, residual=None):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance, at most 8192 channels).  weight / bias
    [C], float32 or of x's type, None = 1 / 0.  With `residual` (x's shape and type): s = x + residual is rounded to x's type and
    normalised, and (s, y) is returned -- the residual stream and its normalised copy in one pass, as scp_amd.dino.add_layernorm does
    for the frozen ViT.  Any strides; the results are contiguous."""
    _tensor(x, "layer_norm: x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("layer_norm: x needs a last dimension of at least one channel")
    c = x.shape[-1]
    if c > 8192:
        raise RuntimeError("layer_norm: at most 8192 channels, got %d" % c)
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _tensor(t, "layer_norm: " + name, (torch.float32, x.dtype))
            if t.dim() != 1 or t.shape[0] != c:
                raise RuntimeError("layer_norm: %s must have %d entries" % (name, c))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("layer_norm: weight and bias must have one type")
    if residual is not None:
        _tensor(residual, "layer_norm: residual", (x.dtype,))
        if residual.shape != x.shape:
            raise RuntimeError("layer_norm: residual must have x's shape %s, not %s" % (tuple(x.shape), tuple(residual.shape)))
        residual = residual.contiguous()
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _wants_grad(x, residual, weight, bias):
        return _LayerNorm.apply(x, residual, weight, bias, float(eps))
    total, y, _, _ = _norm_forward(x, residual, weight, bias, float(eps), False)
    return y if residual is None else (total, y)


# ---- cross attention ---------------------------------------------------------------------------------------------------------------------
def _addressable(t):
    """t itself when the kernels can address it (channels contiguous, pointer and strides multiples of 16 bytes, 128 tokens of all heads
    within 2^31 bytes), else a contiguous copy"""
    size = t.element_size()
    sb, sn, sh, sd = t.stride()
    if sd == 1 and not (t.data_ptr() | sb * size | sn * size | sh * size) & 15 and (128 * sn + t.shape[2] * sh) * size < 1 << 31:
        return t
    return t.clone(memory_format=torch.contiguous_format)      # contiguous() would return a misaligned tensor as it is


def _attn_forward(q, k, v, mask, scale, keep):
    """(out, the bits after its rounding to bfloat16 or None, log-sum-exp or None, C parameters); keep: for a backward pass"""
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if keep else None
    if out.numel() == 0:
        return out, None, lse, None
    if k.shape[1] == 0:
        return out.zero_(), None, lse, None
    low = torch.empty_like(out, dtype=torch.int8) if keep and out.dtype == torch.bfloat16 else None
    L = capi.lib()
    p = capi.CrossAttnParams(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], capi.DTYPES[q.dtype], scale, q.stride()[:3],
                             k.stride()[:3], v.stride()[:3])
    ref = ctypes.byref(p)
    nbytes = L.scp_cross_attention_forward_workspace(ref)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    code = L.scp_cross_attention_forward(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), ref, out.data_ptr(), _ptr(low), _ptr(lse),
                                         _ptr(ws), nbytes, _stream())
    if code:
        capi.check(code, "scp_cross_attention_forward")
    return out, low, lse, p


class _CrossAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, scale):
        out, low, lse, ctx.p = _attn_forward(q, k, v, mask, scale, True)
        ctx.save_for_backward(q, k, v, mask, out, low, lse)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, g):
        q, k, v, mask, out, low, lse = ctx.saved_tensors
        wq, wk, wv = ctx.needs_input_grad[:3]
        dev, dt = q.device, q.dtype
        gq = torch.empty(q.shape, dtype=dt, device=dev) if wq else None
        gk = torch.empty(k.shape, dtype=dt, device=dev) if wk else None
        gv = torch.empty(k.shape, dtype=dt, device=dev) if wv else None
        p = ctx.p
        if p is None:                                            # no query or no key: nothing depends on the other side
            return tuple(None if t is None else t.zero_() for t in (gq, gk, gv)) + (None, None)
        g = _addressable(g)
        p.g_stride = g.stride()[:3]
        L = capi.lib()
        ref = ctypes.byref(p)
        nbytes = L.scp_cross_attention_backward_workspace(ref)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        code = L.scp_cross_attention_backward(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), out.data_ptr(), _ptr(low), lse.data_ptr(),
                                              g.data_ptr(), ref, _ptr(gq), _ptr(gk), _ptr(gv), ws.data_ptr(), nbytes, _stream())
        if code:
            capi.check(code, "scp_cross_attention_backward")
        return gq, gk, gv, None, None


def cross_attention(q, k, v, scale=None, key_mask=None):
    """softmax(scale * q k^T) v per head: q [B, Nq, H, D] against an encoder's k, v [B, Nk, Hkv, D] of another length -> [B, Nq, H, D]
    (contiguous).  H a multiple of Hkv: query head h reads key / value head h // (H // Hkv).  D a multiple of 8, at most 128.  `scale`
    defaults to D ** -0.5.  `key_mask` (bool [B, Nk], True = attend): an image's padding; values stored at masked keys, NaN included,
    reach no result; a batch entry without a key gives zeros, and zero gradients.  Any strides (slices of a fused qkv projection, an
    expanded batch); gradients for q, k and v.  float32 is multiplied as three exact bfloat16 parts: an infinity that is not masked may come
    out as NaN."""
    _tensor(q, "cross_attention: q")
    for t, name in ((k, "k"), (v, "v")):
        _tensor(t, "cross_attention: " + name, (q.dtype,))
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise RuntimeError("cross_attention: q, k and v must be [batch, tokens, heads, channels]")
    b, nq, h, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise RuntimeError("cross_attention: q %s does not go with k %s and v %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if hk == 0 or h % hk:
        raise RuntimeError("cross_attention: %d query heads are no multiple of %d key heads" % (h, hk))
    if d < 8 or d > 128 or d % 8:
        raise RuntimeError("cross_attention: head dimension %d; a multiple of 8 up to 128 is needed" % d)
    mask = None
    if key_mask is not None:
        _tensor(key_mask, "cross_attention: key_mask", (torch.bool,))
        if key_mask.shape != (b, nk):
            raise RuntimeError("cross_attention: key_mask must be [%d, %d], not %s" % (b, nk, tuple(key_mask.shape)))
        mask = key_mask.contiguous()
    scale = float(d) ** -0.5 if scale is None else float(scale)
    q, k, v = _addressable(q), _addressable(k), _addressable(v)
    if _wants_grad(q, k, v):
        return _CrossAttention.apply(q, k, v, mask, scale)
    return _attn_forward(q, k, v, mask, scale, False)[0]


# ---- 8-bit activation checkpoints ----------------------------------------------------------------------------------------------------------
class Packed8:
    """An activation [..., C] held in 8 bits: `codes` int8 of its shape and `exps` uint8 [..., ceil(C / 32)]; 32 neighbouring channels share
    the step 2 ** (exps - 127), value = code * step (exact in float32 and bfloat16).  exps 255: the group held an infinity or a NaN."""

    def __init__(self, codes, exps, dtype):
        self.codes, self.exps, self.dtype = codes, exps, dtype

    @property
    def shape(self):
        return self.codes.shape

    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self, dtype=None):
        """the values the codes stand for, in `dtype` (default: the type that was packed)"""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in capi.DTYPES:
            raise RuntimeError("Packed8.unpack: float32 or bfloat16, not %s" % dtype)
        _check_packed(self, "Packed8.unpack")
        out = torch.empty(self.codes.shape, dtype=dtype, device=self.codes.device)
        if out.numel():
            c = out.shape[-1]
            capi.check(capi.lib().scp_unpack8(_ptr(self.codes), _ptr(self.exps), out.numel() // c, c, capi.DTYPES[dtype], _ptr(out),
                                              _stream()), "scp_unpack8")
        return out


def _packed_like(x):
    codes = torch.empty_like(x, dtype=torch.int8)
    exps = torch.empty(x.shape[:-1] + ((x.shape[-1] + 31) // 32,), dtype=torch.uint8, device=x.device)
    return codes, exps


def _check_packed(p, what):
    _tensor(p.codes, what + ": codes", (torch.int8,))
    _tensor(p.exps, what + ": exps", (torch.uint8,))
    if p.codes.dim() < 1 or tuple(p.exps.shape) != tuple(p.codes.shape[:-1]) + ((p.codes.shape[-1] + 31) // 32,):
        raise RuntimeError("%s: exps %s do not go with codes %s" % (what, tuple(p.exps.shape), tuple(p.codes.shape)))
    if not (p.codes.is_contiguous() and p.exps.is_contiguous()):
        raise RuntimeError("%s: codes and exps must be contiguous" % what)


def _check_rows(x, what):
    _tensor(x, what)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > 1 << 24:
        raise RuntimeError("%s needs a last dimension of 1 to 2^24 channels" % what)


def pack8(x):
    """x [..., C] -> Packed8: per 32 channels a power-of-two step with max|x| in [64, 128) steps, codes rounded to nearest (ties to
    even) and clamped to +-127.  1 + 1/32 bytes per value; not differentiable (it is what an autograd node keeps)."""
    _check_rows(x, "pack8: x")
    x = x.detach().contiguous()
    codes, exps = _packed_like(x)
    if x.numel():
        c = x.shape[-1]
        capi.check(capi.lib().scp_pack8(_ptr(x), x.numel() // c, c, capi.DTYPES[x.dtype], _ptr(codes), _ptr(exps), _stream()), "scp_pack8")
    return Packed8(codes, exps, x.dtype)


def _gelu_forward(x, keep):
    y = torch.empty_like(x)
    codes, exps = _packed_like(x) if keep else (None, None)
    if x.numel():
        c = x.shape[-1]
        capi.check(capi.lib().scp_gelu8_forward(_ptr(x), x.numel() // c, c, capi.DTYPES[x.dtype], _ptr(y), _ptr(codes), _ptr(exps),
                                                _stream()), "scp_gelu8_forward")
    return y, codes, exps


class _Gelu8(Function):
    @staticmethod
    def forward(ctx, x):
        y, codes, exps = _gelu_forward(x, True)
        ctx.save_for_backward(codes, exps)
        ctx.sizes = x.numel(), x.shape[-1], capi.DTYPES[x.dtype]
        return y

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        codes, exps = ctx.saved_tensors
        n, c, dtype = ctx.sizes
        gy = gy.contiguous()
        gx = torch.empty_like(gy)
        if n:
            code = capi.lib().scp_gelu8_backward(codes.data_ptr(), exps.data_ptr(), gy.data_ptr(), n // c, c, dtype, gx.data_ptr(), _stream())
            if code:
                capi.check(code, "scp_gelu8_backward")
        return gx


def gelu8(x):
    """erf GELU of x [..., C] (the MLP's activation, vision_transformer_flexible.py:54-70).  The backward pass takes the slope at the
    8-bit checkpoint of x instead of keeping x: 1 + 1/32 bytes per value held between the passes.  The forward value is exact."""
    _check_rows(x, "gelu8: x")
    x = x.contiguous()
    if _wants_grad(x):
        return _Gelu8.apply(x)
    return _gelu_forward(x, False)[0]


def weight_grad8(grad, packed, bias=True):
    """(gw [N, K], gb [N] or None) in float32 of a linear layer y = x w^T + b from grad = gy [..., N] and the 8-bit checkpoint of x
    [..., K]: gw = sum over rows gy[:, n] x8[:, k], gb = sum over rows gy."""
    _tensor(grad, "weight_grad8: grad")
    if not isinstance(packed, Packed8):
        raise RuntimeError("weight_grad8: packed must be a Packed8 (scp_amd.vit_ops.pack8)")
    _check_packed(packed, "weight_grad8: packed")
    if grad.dim() < 1 or grad.shape[:-1] != packed.shape[:-1] or grad.shape[-1] < 1 or packed.shape[-1] < 1:
        raise RuntimeError("weight_grad8: grad %s does not go with a packed input %s" % (tuple(grad.shape), tuple(packed.shape)))
    n, k = grad.shape[-1], packed.shape[-1]
    rows = grad.numel() // n
    if rows == 0:
        return torch.zeros(n, k, dtype=torch.float32, device=grad.device), torch.zeros(n, dtype=torch.float32, device=grad.device) if bias else None
    grad, codes, exps = grad.detach().contiguous(), packed.codes, packed.exps
    # the kernel reads 16 bytes of grad and 8 codes of a row at a time: narrower rows are widened with zeros
    pad_n, pad_k = max(0, 16 // grad.element_size() - n), max(0, 8 - k)
    if pad_n:
        grad = torch.nn.functional.pad(grad, (0, pad_n))
    if pad_k:
        codes = torch.nn.functional.pad(codes, (0, pad_k))
    gw = torch.empty(n + pad_n, k + pad_k, dtype=torch.float32, device=grad.device)
    gb = torch.empty(n + pad_n, dtype=torch.float32, device=grad.device) if bias else None
    L = capi.lib()
    dt = capi.DTYPES[grad.dtype]
    nbytes = L.scp_weight_grad8_workspace(rows, n + pad_n, k + pad_k, dt)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=grad.device) if nbytes else None
    code = L.scp_weight_grad8(grad.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows, n + pad_n, k + pad_k, dt, gw.data_ptr(), _ptr(gb), _ptr(ws),
                              nbytes, _stream())
    if code:
        capi.check(code, "scp_weight_grad8")
    if pad_n or pad_k:
        gw, gb = gw[:n, :k].contiguous(), None if gb is None else gb[:n].contiguous()
    return gw, gb


class _Linear8(Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        p = pack8(x) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else None
        ctx.save_for_backward(weight, None if p is None else p.codes, None if p is None else p.exps)
        ctx.x_dtype = x.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        weight, codes, exps = ctx.saved_tensors
        gx = gy.matmul(weight) if ctx.needs_input_grad[0] else None
        gw = gb = None
        if codes is not None:
            gw, gb = weight_grad8(gy, Packed8(codes, exps, ctx.x_dtype), bias=ctx.needs_input_grad[2])
            gw = gw.to(weight.dtype) if ctx.needs_input_grad[1] else None
            gb = None if gb is None else gb.to(ctx.bias_dtype)
        return gx, gw, gb


def linear8(x, weight, bias=None):
    """x [..., K] @ weight [N, K]^T + bias, with x kept for the weight gradient in 8 bits (weight_grad8).  One type for all three.  The
    forward product and the input's gradient are plain library products at full precision; nothing else is saved."""
    _check_rows(x, "linear8: x")
    _tensor(weight, "linear8: weight", (x.dtype,))
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise RuntimeError("linear8: weight %s does not go with x %s" % (tuple(weight.shape), tuple(x.shape)))
    if bias is not None:
        _tensor(bias, "linear8: bias", (x.dtype,))
        if bias.dim() != 1 or bias.shape[0] != weight.shape[0]:
            raise RuntimeError("linear8: bias must have %d entries" % weight.shape[0])
    if _wants_grad(x, weight, bias):
        return _Linear8.apply(x, weight, bias)
    return torch.nn.functional.linear(x, weight, bias)
