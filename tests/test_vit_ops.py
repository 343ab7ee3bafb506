"""scp_amd.vit_ops (LayerNorm, cross attention, GELU / linear with 8-bit checkpoints, all with gradients) against their definitions in
float64.

Tolerances are bounds per element, written down from the arithmetic before the first run: u = 2^-24 (half a step of fp32) times the number
of roundings a value goes through, half a step of the output's type (bf16: 2^-8) for the final rounding, and for bf16 attention half a
step for each operand of a product that is rounded on the way (the probabilities and the score gradients)."""
import math

import pytest
import torch

from scp_amd import vit_ops

gpu = pytest.mark.gpu
U = 2.0 ** -24
FP32, BF16 = torch.float32, torch.bfloat16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, ref, bound, what):
    """|got - ref| <= bound per element, the same places not finite"""
    got = got.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin), what + ": finite in other places"
    d = torch.where(fin, (got - ref).abs(), torch.zeros_like(ref))
    bound = bound + 1e-300
    worst = (d / bound).max().item() if d.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g of the bound, |d| up to %.3g" % (what, worst, d.max().item())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- refusals (no GPU needed) ----------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x = torch.rand(3, 8)
    q = torch.rand(1, 2, 1, 8)
    for call in (lambda: vit_ops.layer_norm(x), lambda: vit_ops.cross_attention(q, q, q), lambda: vit_ops.pack8(x), lambda: vit_ops.gelu8(x),
                 lambda: vit_ops.linear8(x, torch.rand(4, 8)), lambda: vit_ops.weight_grad8(x, None),
                 lambda: vit_ops.Packed8(torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3, 1, dtype=torch.uint8), FP32).unpack()):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def _abi_params(**kw):
    from scp_amd import capi
    p = capi.CrossAttnParams()
    p.batch, p.queries, p.keys, p.heads, p.kv_heads, p.head_dim, p.dtype, p.scale = 1, 2, 3, 4, 2, 64, 0, 1.0
    for f in ("q_stride", "k_stride", "v_stride", "g_stride"):
        getattr(p, f)[:] = (64 * 16, 64 * 4, 64)
    for name, v in kw.items():
        setattr(p, name, v)
    return p


def test_c_entries_refuse_bad_problems_before_any_launch():
    """every check of the C entry points is host code: it answers without a device, with the reason in scp_last_error()"""
    import ctypes
    from scp_amd import capi
    L = capi.lib()
    one = ctypes.c_void_p(4096)

    def attn(want, q=one, **kw):
        assert L.scp_cross_attention_forward(q, one, one, None, ctypes.byref(_abi_params(**kw)), one, None, None, None, 0, None) != 0
        assert want in L.scp_last_error().decode()

    attn("empty", batch=0)
    attn("empty", keys=-1)
    attn("multiple of kv_heads", heads=3)
    attn("multiple of 8", head_dim=136)
    attn("multiple of 8", head_dim=12)
    attn("unknown type", dtype=7)
    attn("2^31", queries=1 << 30)
    attn("2^31", batch=1 << 30)
    attn("16-byte", q=ctypes.c_void_p(4100))
    attn("null", q=None)
    p = _abi_params()
    p.k_stride[1] = 66
    assert L.scp_cross_attention_forward(one, one, one, None, ctypes.byref(p), one, None, None, None, 0, None) != 0
    assert "strides" in L.scp_last_error().decode()
    assert L.scp_cross_attention_backward(one, one, one, None, one, None, one, one, ctypes.byref(_abi_params()), one, one, one, None, 0, None) != 0
    assert "workspace" in L.scp_last_error().decode()
    assert L.scp_layernorm_forward(one, None, None, None, 1e-6, 4, 9000, 0, 0, None, one, None, None) != 0
    assert "8192" in L.scp_last_error().decode()
    assert L.scp_layernorm_forward(one, one, None, None, 1e-6, 4, 64, 0, 0, None, one, None, None) != 0
    assert L.scp_layernorm_forward(one, None, one, None, 1e-6, 4, 64, 0, 1, None, one, None, None) != 0
    assert L.scp_layernorm_backward(one, None, one, None, one, 400, 640, 0, 0, one, one, one, None, 0, None) != 0
    assert "workspace" in L.scp_last_error().decode()
    assert L.scp_pack8(one, 0, 64, 0, one, one, None) != 0 and L.scp_pack8(one, 1, 64, 2, one, one, None) != 0
    assert L.scp_gelu8_forward(one, 1, 64, 0, one, one, None, None) != 0
    assert L.scp_weight_grad8(one, one, one, 4, 0, 64, 0, one, None, None, 0, None) != 0
    assert L.scp_weight_grad8(one, one, None, 4, 8, 64, 0, one, None, None, 0, None) != 0
    assert L.scp_weight_grad8(one, one, one, 4, 7, 64, 1, one, None, None, 0, None) != 0 and L.scp_weight_grad8(one, one, one, 4, 8, 7, 0, one, None, None, 0, None) != 0


@gpu
def test_arguments_are_checked():
    f = lambda *s, dtype=FP32: torch.zeros(*s, device="cuda", dtype=dtype)
    x, q, k = f(3, 16), f(2, 3, 4, 16), f(2, 5, 2, 16)
    bad = [lambda: vit_ops.layer_norm(x, f(15)), lambda: vit_ops.layer_norm(x, f(16), f(16, dtype=BF16)), lambda: vit_ops.layer_norm(x.half()),
           lambda: vit_ops.layer_norm(x, f(16, dtype=BF16)), lambda: vit_ops.layer_norm(x, residual=f(16)), lambda: vit_ops.layer_norm(f(2, 8193)),
           lambda: vit_ops.layer_norm(x, residual=x.bfloat16()), lambda: vit_ops.cross_attention(q, k, f(2, 6, 2, 16)),
           lambda: vit_ops.cross_attention(q, k.bfloat16(), k.bfloat16()), lambda: vit_ops.cross_attention(q, f(2, 5, 3, 16), f(2, 5, 3, 16)),
           lambda: vit_ops.cross_attention(f(2, 3, 4, 20), f(2, 5, 2, 20), f(2, 5, 2, 20)), lambda: vit_ops.cross_attention(q[0], k[0], k[0]),
           lambda: vit_ops.cross_attention(q, k, k, key_mask=torch.ones(2, 4, dtype=torch.bool, device="cuda")),
           lambda: vit_ops.cross_attention(q, k, k, key_mask=f(2, 5)), lambda: vit_ops.cross_attention(q, f(1, 5, 2, 16), f(1, 5, 2, 16)),
           lambda: vit_ops.gelu8(x.double()), lambda: vit_ops.linear8(x, f(4, 15)), lambda: vit_ops.linear8(x, f(4, 16), f(5)),
           lambda: vit_ops.linear8(x, f(4, 16, dtype=BF16)), lambda: vit_ops.weight_grad8(f(4, 8), vit_ops.pack8(x)),
           lambda: vit_ops.weight_grad8(x, x), lambda: vit_ops.pack8(f(3, 0)), lambda: vit_ops.pack8(x).unpack(torch.float16),
           lambda: vit_ops.Packed8(f(3, 64, dtype=torch.int8), f(3, 1, dtype=torch.uint8), FP32).unpack()]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("call %d was not refused" % i)


# ---- layer norm --------------------------------------------------------------------------------------------------------------------------
def norm_reference(x, r, w, b, eps, gy, gsum, dtype):
    """values and their bounds.  Sums over a row: at most 32 elements per lane one after the other, 8 more additions -> 40 u sum|.|"""
    s = x.double() if r is None else (x.float() + r.float()).to(dtype).double()
    c = s.shape[1]
    w64 = torch.ones(c, dtype=torch.float64, device=s.device) if w is None else w.double()
    b64 = torch.zeros(c, dtype=torch.float64, device=s.device) if b is None else b.double()
    mean, var = s.mean(1, keepdim=True), s.var(1, unbiased=False, keepdim=True)
    rstd = (var + eps).rsqrt()
    xhat = (s - mean) * rstd
    y = xhat * w64 + b64
    d_mean = 42 * U * s.abs().mean(1, keepdim=True)
    d_diff = d_mean + U * (s - mean).abs()                                      # of s - mean
    # relative error of the variance: 2 |d| d_diff / var on average, 40 additions; half of it goes into rstd, plus sqrt, division
    d_rstd = ((s - mean).abs() * d_diff).mean(1, keepdim=True) * rstd ** 2 + 26 * U
    d_xhat = rstd * d_diff + xhat.abs() * (d_rstd + 2 * U)
    out = {"s": s, "y": (y, half_step(dtype) * y.abs() + (w64.abs() * d_xhat + 3 * U * (y.abs() + b64.abs())) * (1 + half_step(dtype)))}
    if gy is not None:
        g = gy.double()
        gw = g * w64
        m1, m2 = gw.mean(1, keepdim=True), (gw * xhat).mean(1, keepdim=True)
        a1, a2 = gw.abs().mean(1, keepdim=True), (gw * xhat).abs().mean(1, keepdim=True)
        gx = rstd * (gw - m1 - xhat * m2)
        d_m2 = (gw.abs() * d_xhat).mean(1, keepdim=True) + 44 * U * a2
        d_gx = rstd * (3 * U * gw.abs() + 44 * U * a1 + xhat.abs() * d_m2 + d_xhat * m2.abs() + 3 * U * xhat.abs() * a2) + gx.abs() * (d_rstd + 3 * U)
        if gsum is not None:
            gx = gx + gsum.double()
            d_gx = d_gx + U * gx.abs()
        out["gx"] = (gx, half_step(dtype) * gx.abs() + d_gx * (1 + half_step(dtype)))
        rows = s.shape[0]
        n_add = rows / 2 + 200                                                   # far more than any lane, fold or slice adds up
        out["gw"] = ((g * xhat).sum(0), (g.abs() * d_xhat).sum(0) + n_add * U * (g * xhat).abs().sum(0))
        out["gb"] = (g.sum(0), n_add * U * g.abs().sum(0))
    return out


NORM_SHAPES = [(1, 1), (1, 384), (3, 7), (5, 63), (64, 384), (130, 385), (1025, 384), (7, 512), (33, 513), (9, 1001), (66, 2048), (5, 2049), (19, 1536),
               (3, 8192), (2, 8191), (2100, 40)]


@gpu
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("dtype,wdtype", [(FP32, FP32), (BF16, FP32), (BF16, BF16)])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_matches_definition(shape, dtype, wdtype, residual):
    g = gen(shape[0] * 7919 + shape[1])
    rows, c = shape
    new = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale)
    x = (new(rows, c) * (1 + 3 * torch.rand(c, generator=g, device="cuda")) + 5 * new(rows, 1)).to(dtype).requires_grad_(True)
    r = new(rows, c).to(dtype).requires_grad_(True) if residual else None
    w, b = (1 + 0.3 * new(c)).to(wdtype).requires_grad_(True), new(c).to(wdtype).requires_grad_(True)
    gy = new(rows, c).to(dtype)
    gs = new(rows, c).to(dtype) if residual else None
    ref = norm_reference(x.detach(), None if r is None else r.detach(), w.detach(), b.detach(), 1e-6, gy, gs, dtype)
    if residual:
        total, y = vit_ops.layer_norm(x, w, b, residual=r)
        gx, gr, gw, gb = torch.autograd.grad((total, y), (x, r, w, b), (gs, gy))
        assert torch.equal(total.detach().double(), ref["s"])
        assert torch.equal(gx, gr)
    else:
        y = vit_ops.layer_norm(x, w, b)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    assert y.dtype == dtype and gx.dtype == dtype and gw.dtype == wdtype and gb.dtype == wdtype
    within(y.detach(), *ref["y"], "y")
    within(gx, *ref["gx"], "gx")
    for got, name in ((gw, "gw"), (gb, "gb")):
        v, bound = ref[name]
        within(got, v, bound + (half_step(BF16) * (v.abs() + bound) if wdtype == BF16 else 0), name)
    with torch.no_grad():                                                        # the inference form is the same computation
        again = vit_ops.layer_norm(x, w, b, residual=r)
        assert torch.equal(again[1] if residual else again, y)


@gpu
def test_layer_norm_without_affine_and_partial_gradients():
    g = gen(3)
    x = torch.randn(10, 96, generator=g, device="cuda").requires_grad_(True)
    w = torch.randn(96, generator=g, device="cuda").requires_grad_(True)
    b = torch.randn(96, generator=g, device="cuda").requires_grad_(True)
    gy = torch.randn(10, 96, generator=g, device="cuda")
    ref = norm_reference(x.detach(), None, None, None, 1e-6, gy, None, FP32)
    y = vit_ops.layer_norm(x)
    within(y.detach(), *ref["y"], "y")
    within(torch.autograd.grad(y, x, gy)[0], *ref["gx"], "gx")
    ref = norm_reference(x.detach(), None, w.detach(), b.detach(), 1e-6, gy, None, FP32)
    only_w = torch.autograd.grad(vit_ops.layer_norm(x.detach(), w, b), w, gy)[0]                  # neither x nor bias
    only_b = torch.autograd.grad(vit_ops.layer_norm(x.detach(), None, b), b, gy)[0]
    within(only_w, *ref["gw"], "gw")
    within(only_b, *ref["gb"], "gb")
    # sum only / y only of the residual form
    r = torch.randn(10, 96, generator=g, device="cuda").requires_grad_(True)
    total, y = vit_ops.layer_norm(x, w, b, residual=r)
    assert torch.equal(torch.autograd.grad(total, (x, r), gy, retain_graph=True)[1], gy)
    ref = norm_reference(x.detach(), r.detach(), w.detach(), b.detach(), 1e-6, gy, None, FP32)
    within(torch.autograd.grad(y, r, gy)[0], *ref["gx"], "gx of y alone")


@gpu
def test_layer_norm_layouts_and_edges():
    g = gen(4)
    base = torch.randn(6, 40, 5, generator=g, device="cuda")
    x = base.transpose(1, 2)                                                     # channels not contiguous
    ref = norm_reference(x.reshape(-1, 40).clone(), None, None, None, 1e-6, None, None, FP32)
    within(vit_ops.layer_norm(x).reshape(-1, 40), *ref["y"], "transposed")
    flat = torch.randn(7 * 33 + 1, generator=g, device="cuda").bfloat16()
    x = flat[1:].view(7, 33)                                                     # starts 2 bytes into its storage
    ref = norm_reference(x.clone(), None, None, None, 1e-6, None, None, BF16)
    within(vit_ops.layer_norm(x), *ref["y"], "odd address")
    e = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = vit_ops.layer_norm(e, w)
    assert y.shape == (0, 16)
    ge, gw = torch.autograd.grad(y, (e, w), torch.empty(0, 16, device="cuda"))
    assert ge.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device="cuda"))
    const = torch.full((2, 64), 1e4, device="cuda")                              # no variance: y = bias
    assert torch.equal(vit_ops.layer_norm(const, None, torch.full((64,), 2.0, device="cuda")), torch.full((2, 64), 2.0, device="cuda"))
    x = torch.randn(4, 64, generator=g, device="cuda")
    x[2, 5] = math.inf                                                           # stays in its own row
    y = vit_ops.layer_norm(x)
    assert torch.isfinite(y[[0, 1, 3]]).all() and not torch.isfinite(y[2]).any()


# ---- cross attention ---------------------------------------------------------------------------------------------------------------------
def attn_reference(q, k, v, mask, scale, go, dtype):
    b, nq, h, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    g = h // hk
    # rounding of a probability before its product with v (one row: fp32 all the way); and of a probability or a score gradient in the
    # backward pass, which keeps 16 bits of it where one side has at most 16 rows
    half = half_step(dtype) if dtype != FP32 else 0.0
    e, e_back = half if nq * g > 1 else 0.0, half ** 2 if min(nq * g, nk) <= 16 else half
    if mask is not None:                                                         # values at masked keys do not exist
        k = torch.where(mask[:, :, None, None], k, torch.zeros_like(k))
        v = torch.where(mask[:, :, None, None], v, torch.zeros_like(v))
    Q = q.double().permute(0, 2, 1, 3)
    K, V = (t.double().permute(0, 2, 1, 3).repeat_interleave(g, 1) for t in (k, v))
    s = scale * Q @ K.transpose(2, 3)
    # absolute error of a score in its exponent: d roundings of the products' sum, two of the scaling
    d_s = abs(scale) * (d + 4) * U * (Q.abs() @ K.abs().transpose(2, 3)) + 2 * U * s.abs()
    on = torch.ones(b, 1, 1, nk, dtype=torch.bool, device=q.device) if mask is None else mask[:, None, None, :]
    s = s.masked_fill(~on, -math.inf)
    top = s.amax(3, keepdim=True) if nk else s.sum(3, keepdim=True)
    p = torch.where(on, (s - torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp(), torch.zeros_like(s))
    den = p.sum(3, keepdim=True)
    p = torch.where(den > 0, p / den, torch.zeros_like(p))
    # relative error of a probability: exponent, two exponentials (2 steps each) and the subtraction of a maximum of up to max|s|, the sum
    top_s = (s.abs().masked_fill(~on, 0)).amax(3, keepdim=True) if nk else 0.0
    d_p = p * (2 * d_s + 2 * (p * d_s).sum(3, keepdim=True) + 4 * U * top_s + (nk / 4 + 24) * U)
    o = p @ V
    # o = sum_j w_j v_j / sum_j w_j with w = p rounded by up to e of itself: with w_j = p_j (1 + x_j), |x_j| <= e, and sum p = 1
    #   o - o_exact = sum_j p_j x_j (v_j - o) / (1 + sum p x), so at most e (1 + 2 e) (sum_j p_j |v_j| + |o|).
    e1 = e * (1 + 2 * e)
    d_sum = (d_p + (nk / 4 + 24) * U * p) @ V.abs()
    d_o = d_sum + e1 * (p @ V.abs() + o.abs())
    back = lambda t: t.permute(0, 2, 1, 3)
    out = {"o": (back(o), back(d_o + half_step(dtype) * (o.abs() + d_o)))}
    if go is not None:
        G = go.double().permute(0, 2, 1, 3)
        gp = G @ V.transpose(2, 3)
        delta = (G * o).sum(3, keepdim=True)
        gs = p * (gp - delta)
        # delta = G . o.  The rounding of the weights moves it by sum_j p_j x_j (gp_j - delta): at most e1 sum |gs|.  o is rounded to fp32, or
        # kept in two bf16 numbers: the second is off by half a step of something that is at most half a step of o.
        low = half_step(dtype) if dtype == FP32 else half_step(dtype) ** 2
        d_delta = (G.abs() * (d_sum + low * (o.abs() + d_o))).sum(3, keepdim=True) + e1 * gs.abs().sum(3, keepdim=True) \
            + (d + 2) * U * (G * o).abs().sum(3, keepdim=True)
        d_p = d_p + e1 * p                                                       # the backward pass divides the unrounded p by the sum of the w
        d_gs = d_p * (gp - delta).abs() + p * (d_delta + (d + 4) * U * (G.abs() @ V.abs().transpose(2, 3)))
        d_gs = d_gs + (e_back + 4 * U) * (gs.abs() + d_gs)
        n_q, n_r = (nk / 4 + 24) * U, (nq * g + 24) * U
        fold = lambda t: t.reshape(b, hk, g, nk, d).sum(2).permute(0, 2, 1, 3)
        for name, val, err in (("gq", back(scale * gs @ K), back(abs(scale) * (d_gs + n_q * gs.abs()) @ K.abs())),
                               ("gk", fold(scale * gs.transpose(2, 3) @ Q), fold(abs(scale) * (d_gs + n_r * gs.abs()).transpose(2, 3) @ Q.abs())),
                               ("gv", fold(p.transpose(2, 3) @ G), fold((d_p + (e_back + n_r) * p).transpose(2, 3) @ G.abs()))):
            out[name] = (val, err + half_step(dtype) * (val.abs() + err))
    return out


def attn_inputs(b, nq, nk, h, hk, d, dtype, seed, spread=1.0):
    g = gen(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return ((new(b, nq, h, d) * spread).to(dtype), new(b, nk, hk, d).to(dtype), new(b, nk, hk, d).to(dtype), new(b, nq, h, d).to(dtype), g)


def check_attn(q, k, v, go, mask=None, scale=None, what=""):
    d = q.shape[3]
    sc = d ** -0.5 if scale is None else scale
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = vit_ops.cross_attention(*leaves, scale=scale, key_mask=mask)
    grads = torch.autograd.grad(o, leaves, go)
    ref = attn_reference(q, k, v, mask, sc, go, q.dtype)
    within(o.detach(), *ref["o"], what + "o")
    for got, name, like in zip(grads, ("gq", "gk", "gv"), (q, k, v)):
        assert got.shape == like.shape and got.dtype == like.dtype
        within(got, *ref[name], what + name)
    with torch.no_grad():
        within(vit_ops.cross_attention(q, k, v, scale=scale, key_mask=mask), *ref["o"], what + "inference o")
    return o, grads


ATTN_SHAPES = [  # batch, queries, keys, heads, kv_heads, head_dim
    (1, 1, 1, 1, 1, 64), (2, 1, 77, 6, 6, 64), (1, 3, 64, 4, 1, 64), (2, 33, 65, 2, 2, 64), (1, 128, 128, 3, 1, 64), (2, 129, 31, 6, 2, 64), (1, 200, 1025, 2, 1, 64),
    (1, 70, 97, 2, 2, 32), (1, 45, 130, 2, 1, 96), (2, 40, 100, 2, 1, 128), (1, 37, 50, 3, 3, 8), (1, 65, 70, 2, 1, 40), (1, 50, 66, 1, 1, 120), (9, 5, 257, 2, 1, 64),
    (3, 2, 4, 8, 8, 16), (1, 642, 300, 1, 1, 64), (2, 1, 4097, 4, 2, 64), (1, 9, 2050, 1, 1, 128),
    (2, 3, 300, 2, 2, 64), (1, 1, 500, 4, 1, 96), (2, 2, 90, 4, 2, 128), (1, 1, 2050, 1, 1, 32), (20, 1, 130, 3, 3, 8), (2, 1, 700, 2, 2, 120), (1, 4, 1500, 1, 1, 40), (3, 20, 400, 2, 2, 40), (1, 17, 1100, 2, 1, 64), (1, 33, 300, 1, 1, 96),
    (16, 700, 40, 3, 3, 64), (24, 600, 33, 6, 6, 32)]


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=str)
def test_cross_attention_matches_definition(shape, dtype):
    b, nq, nk, h, hk, d = shape
    q, k, v, go, _ = attn_inputs(b, nq, nk, h, hk, d, dtype, sum(shape))
    check_attn(q, k, v, go)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nq", [1, 40, 150])
def test_cross_attention_masks(dtype, nq):
    """random holes, a padded tail, whole tiles off, one key, none; infinities and NaN stored at masked keys"""
    nk = 331
    q, k, v, go, g = attn_inputs(6, nq, nk, 4, 2, 64, dtype, nq)
    mask = torch.rand(6, nk, generator=g, device="cuda") < 0.5
    mask[1] = torch.arange(nk, device="cuda") < 100
    mask[2] = torch.arange(nk, device="cuda") >= 270
    mask[3] = torch.arange(nk, device="cuda") == 200
    mask[4] = False
    mask[5] = True
    for fill in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        k = torch.where(mask[:, :, None, None], k, torch.full_like(k, fill))
        v = torch.where(mask[:, :, None, None], v, torch.full_like(v, fill))
        o, (gq, gk, gv) = check_attn(q, k, v, go, mask, what="fill %s " % fill)
        assert not o[4].any() and not gq[4].any() and not gk[4].any() and not gv[4].any()
        off = ~mask[:, :, None, None].expand_as(gk)
        assert not gk[off].any() and not gv[off].any()


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(24, 642, 161, 6, 6, 32), (48, 66, 300, 8, 2, 64), (40, 130, 193, 8, 8, 64), (33, 320, 140, 4, 4, 40), (24, 257, 129, 6, 3, 128)], ids=str)
def test_cross_attention_many_columns(shape, dtype):
    """enough rows and keys for workgroups of 128 of them, with short last ones of 1 to 64, or more, on either side; masked keys among them"""
    b, nq, nk, h, hk, d = shape
    q, k, v, go, g = attn_inputs(b, nq, nk, h, hk, d, dtype, 77)
    mask = torch.rand(b, nk, generator=g, device="cuda") < 0.7
    mask[0, :128] = False
    mask[1, 128:] = False
    k = torch.where(mask[:, :, None, None], k, torch.full_like(k, math.nan))
    check_attn(q, k, v, go, mask)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_cross_attention_peaked_and_scaled(dtype):
    """scores of +-hundreds (the running maximum moves late), a negative and a zero scale"""
    q, k, v, go, _ = attn_inputs(1, 70, 260, 2, 1, 64, dtype, 5, spread=6.0)
    k[:, 200] *= 5
    check_attn(q, k, v, go, scale=0.5, what="peaked ")
    check_attn(q, k, v, go, scale=-0.05, what="negative ")
    check_attn(q, k, v, go, scale=0.0, what="zero ")
    # the largest score comes late and is less than 2^8 times the ones before it, so the maximum that is subtracted is not the row's;
    # nearly all of the softmax on one or two keys: gs is a difference of nearly equal numbers
    k[:, 250] = 1.02 * k[:, 200]
    check_attn(q, k, v, go, scale=0.1, what="on two keys ")
    check_attn(q, k[:, 190:260], v[:, 190:260], go, scale=0.05, what="few keys ")
    check_attn(q, k[:, 200:202], v[:, 200:202], go, scale=0.02, what="two keys ")


@gpu
@pytest.mark.parametrize("nq", [1, 3, 40, 2500])
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_cross_attention_shows_nan(dtype, nq):
    """a NaN in a query, or at a key that is not masked, is in the rows it belongs to and in no other; in every form of the forward pass"""
    q, k, v, go, _ = attn_inputs(2, nq, 700, 2, 2, 64, dtype, 31)
    q[0, nq - 1, 1, 5] = math.nan
    o = vit_ops.cross_attention(q, k, v)
    assert o[0, nq - 1, 1].isnan().all() and o.isnan().sum() == 64
    k[1, 650, 0, 7] = math.nan
    o = vit_ops.cross_attention(q, k, v)
    assert o[1, :, 0].isnan().all() and o.isnan().sum() == 64 + 64 * nq
    mask = torch.ones(2, 700, dtype=torch.bool, device="cuda")
    mask[1, 650] = False
    assert vit_ops.cross_attention(q, k, v, key_mask=mask).isnan().sum() == 64


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_cross_attention_layouts(dtype):
    g = gen(8)
    b, n, h, d = 2, 75, 3, 64
    qkv = torch.randn(b, n, 3, h, d, generator=g, device="cuda").to(dtype)                        # a fused projection
    go = torch.randn(b, n, h, d, generator=g, device="cuda").to(dtype)
    check_attn(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], go, what="fused qkv ")
    hf = torch.randn(3, b, h, n, d, generator=g, device="cuda").to(dtype).transpose(2, 3)         # head-major storage
    check_attn(hf[0], hf[1], hf[2], go.transpose(1, 2).contiguous().transpose(1, 2), what="head-major ")
    k = torch.randn(1, 50, h, d, generator=g, device="cuda").to(dtype)                            # one encoder state for the whole batch
    v = torch.randn(1, 50, h, d, generator=g, device="cuda").to(dtype)
    check_attn(qkv[:, :, 0], k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), go, what="broadcast ")
    leaf = k.clone().requires_grad_(True)                                                          # ... whose gradient is the batch's sum
    o = vit_ops.cross_attention(qkv[:, :, 0], leaf.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1))
    ref = attn_reference(qkv[:, :, 0], k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), None, d ** -0.5, go, dtype)
    val, bound = ref["gk"]
    within(torch.autograd.grad(o, leaf, go)[0], val.sum(0, keepdim=True), bound.sum(0, keepdim=True) * 1.02 + half_step(dtype) * val.sum(0, keepdim=True).abs(), "broadcast leaf")
    flat = torch.randn(b * n * h * d + 1, generator=g, device="cuda").to(dtype)                    # not 16-byte aligned
    odd = flat[1:].view(b, n, h, d)
    check_attn(odd, qkv[:, :, 1], qkv[:, :, 2], go, what="misaligned ")
    wide = torch.randn(b, n, h, d, 2, generator=g, device="cuda").to(dtype)[..., 0]                # channels not contiguous
    check_attn(wide, qkv[:, :, 1], wide, go, what="strided channels ")


@gpu
def test_cross_attention_empty_sides():
    q = torch.randn(2, 3, 4, 16, device="cuda", requires_grad=True)
    k = torch.randn(2, 0, 4, 16, device="cuda", requires_grad=True)
    o = vit_ops.cross_attention(q, k, k)
    assert torch.equal(o, torch.zeros_like(q))
    gq, gk = torch.autograd.grad(o, (q, k), torch.ones_like(o))
    assert torch.equal(gq, torch.zeros_like(q)) and gk.shape == k.shape
    none = torch.randn(2, 0, 4, 16, device="cuda", requires_grad=True)
    k = torch.randn(2, 5, 4, 16, device="cuda", requires_grad=True)
    o = vit_ops.cross_attention(none, k, k)
    assert o.shape == none.shape
    assert torch.equal(torch.autograd.grad(o, k, torch.empty_like(o))[0], torch.zeros_like(k))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("n,step", [(1100, 1 << 21), (66, 1 << 25)], ids=["addressed", "copied"])
def test_cross_attention_offsets_past_32_bits(dtype, n, step):
    """a cache whose last key is over 2^31 elements into the storage; at 2^25 elements per token a tile spans more than 2^31 bytes"""
    store = torch.empty(n * step, dtype=dtype, device="cuda")
    k = store.view(1, n, step)[:, :, :64].unflatten(2, (1, 64))
    v = store.view(1, n, step)[:, :, 64:128].unflatten(2, (1, 64))
    q, kk, vv, go, _ = attn_inputs(1, 5, n, 1, 1, 64, dtype, 9)
    k.copy_(kk)
    v.copy_(vv)
    check_attn(q, k, v, go)


# ---- 8-bit checkpoints ---------------------------------------------------------------------------------------------------------------------
def round8_reference(x):
    """the format's definition in float64 on the CPU: (value, code, exponent byte)"""
    rows, c = x.shape
    t = torch.nn.functional.pad(x.double().cpu(), (0, -c % 32)).view(rows, -1, 32)
    top = t.abs().amax(2, keepdim=True)
    bad = ~torch.isfinite(t).all(2, keepdim=True)
    mant, ex = torch.frexp(torch.where(bad, torch.ones_like(top), top))                          # top = mant 2^ex, mant in [0.5, 1)
    e = torch.where(top == 0, torch.full_like(ex, -126), (ex - 7).clamp(min=-126))
    step = torch.ldexp(torch.ones_like(top), e)
    code = (torch.where(bad, torch.zeros_like(t), t) / step).round().clamp(-127, 127)
    value = torch.where(bad, torch.full_like(t, math.nan), code * step)
    return value.view(rows, -1)[:, :c], code.view(rows, -1)[:, :c].to(torch.int8), torch.where(bad, torch.full_like(e, 255), e + 127)[..., 0].to(torch.uint8)


def spread_values(rows, c, dtype, seed):
    g = gen(seed)
    x = torch.randn(rows, c, generator=g, device="cuda") * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(dtype)


ACT_SHAPES = [(1, 1), (1, 31), (2, 32), (3, 33), (5, 384), (17, 1001), (130, 1536), (4100, 64), (3, 96), (1, 16), (7, 48)]


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", ACT_SHAPES, ids=str)
def test_pack8_is_the_format(shape, dtype):
    x = spread_values(*shape, dtype, shape[0] + shape[1])
    if x.numel() > 200:
        flat = x.view(-1)
        flat[3], flat[70], flat[71] = 0.0, 127.75 * 2.0 ** -7, -1.0                              # clamping: 127.75 steps and its neighbour
        flat[100:132] = 0.0
        flat[150] = 2.0 ** -133 if dtype == BF16 else 2.0 ** -140                                 # a denormal among normal values
    p = vit_ops.pack8(x)
    value, code, exps = round8_reference(x)
    assert torch.equal(p.codes.cpu(), code) and torch.equal(p.exps.cpu(), exps)
    assert torch.equal(p.unpack(FP32).double().cpu(), value)
    assert torch.equal(p.unpack(BF16).double().cpu(), value)                                      # exact in bf16 too
    assert p.unpack().dtype == dtype and p.shape == x.shape


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("c", [96, 90])
def test_pack8_extremes(dtype, c):
    x = torch.zeros(12, c, device="cuda", dtype=dtype)
    big, tiny = torch.finfo(dtype).max, 2.0 ** -126
    x[0, 5], x[1, 40], x[2, 70] = math.inf, -math.inf, math.nan
    x[3, :] = 1.0
    x[4, 0], x[4, 1] = big, -big
    x[5, :] = tiny
    x[6, :] = tiny / 4                                                                           # denormals
    x[7, 0:32:2], x[7, 1:32:2] = 1.0, 2.0 ** -8                                                   # half a step: a tie, to even
    x[8, 0], x[8, 1], x[8, 2] = 64.0, 0.5, 1.5
    x[9, 0], x[9, 1] = 2.0 - 2.0 ** -7, -(2.0 - 2.0 ** -7)
    x[10, :] = -0.0
    x[0, 60] = 3.0                                                                               # the neighbouring group is not touched by the infinity
    p = vit_ops.pack8(x)
    value, code, exps = round8_reference(x)
    assert torch.equal(p.codes.cpu(), code) and torch.equal(p.exps.cpu(), exps)
    got = p.unpack(FP32).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(value))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(value))
    x8 = torch.nan_to_num(value)
    gy = torch.ones(12, c, device="cuda", dtype=dtype)
    leaf = x.clone().requires_grad_(True)
    gx = torch.autograd.grad(vit_ops.gelu8(leaf), leaf, gy)[0].double().cpu()
    assert torch.equal(torch.isnan(gx), torch.isnan(value))
    assert (torch.nan_to_num(gx) - torch.where(torch.isnan(value), torch.zeros_like(x8), gelu_slope64(x8))).abs().max() <= half_step(dtype) * 1.2 + 1e-6


def gelu64(x):
    return x * torch.special.erfc(-x / math.sqrt(2.0)) / 2


def gelu_slope64(x):
    return torch.special.erfc(-x / math.sqrt(2.0)) / 2 + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", ACT_SHAPES, ids=str)
def test_gelu8_matches_definition(shape, dtype):
    """Phi and the slope are computed to 4e-7 absolute (error function to 1.5e-7, exponential and the roundings around them); y multiplies
    it by x"""
    x = (spread_values(*shape, FP32, 77 + shape[1]).clamp(-30, 30)).to(dtype).requires_grad_(True)
    gy = torch.randn(*shape, generator=gen(78), device="cuda").to(dtype)
    y = vit_ops.gelu8(x)
    gx = torch.autograd.grad(y, x, gy)[0]
    ref = gelu64(x.detach().double())
    err = 4e-7 * x.detach().double().abs() + 2 * U * ref.abs()
    within(y.detach(), ref, err + half_step(dtype) * (ref.abs() + err), "y")
    slope = gelu_slope64(round8_reference(x.detach())[0]).cuda()
    ref = gy.double() * slope
    err = gy.double().abs() * (4e-7 * (1 + slope.abs())) + 2 * U * ref.abs()
    within(gx, ref, err + half_step(dtype) * (ref.abs() + err), "gx")
    with torch.no_grad():
        assert torch.equal(vit_ops.gelu8(x), y)


WGRAD_SHAPES = [(1, 1, 1), (1, 8, 16), (3, 7, 5), (33, 64, 64), (100, 65, 96), (257, 128, 128), (1025, 40, 48), (70, 384, 384), (130, 333, 384), (2100, 130, 72), (64, 16, 1001),
                (515, 136, 160), (31, 17, 33), (32, 129, 131), (65, 257, 17), (200, 4, 16), (200, 8, 15), (200, 7, 7), (97, 261, 16), (1000, 255, 143)]


def wgrad_reference(gy, x8):
    g = gy.double()
    rows = g.shape[0]
    gw = g.t().contiguous() @ x8
    # products are exact in the kernel's operands (fp32: 24 x 7 bits over the split parts); every addition of a term rounds once
    n = (rows + 64) * U
    return (gw, n * (g.abs().t().contiguous() @ x8.abs())), (g.sum(0), n * g.abs().sum(0))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", WGRAD_SHAPES, ids=str)
def test_weight_grad8_matches_definition(shape, dtype):
    rows, n, k = shape
    x = spread_values(rows, k, dtype, rows + k).clamp(-50, 50)
    gy = torch.randn(rows, n, generator=gen(rows * n), device="cuda").to(dtype)
    x8 = round8_reference(x)[0].cuda()
    p = vit_ops.pack8(x)
    gw, gb = vit_ops.weight_grad8(gy, p)
    ref_w, ref_b = wgrad_reference(gy, x8)
    within(gw, *ref_w, "gw")
    within(gb, *ref_b, "gb")
    again, none = vit_ops.weight_grad8(gy, p, bias=False)
    assert none is None and torch.equal(again, gw)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_weight_grad8_layouts_and_edges(dtype):
    x = spread_values(60, 64, dtype, 1).view(3, 20, 64)
    flat = torch.randn(60 * 24 + 1, generator=gen(2), device="cuda").to(dtype)
    gy = flat[1:].view(3, 20, 24)                                                                 # off its storage's alignment
    x8 = round8_reference(x.view(60, 64))[0].cuda()
    ref_w, ref_b = wgrad_reference(gy.reshape(60, 24), x8)
    gw, gb = vit_ops.weight_grad8(gy, vit_ops.pack8(x))
    within(gw, *ref_w, "gw")
    within(gb, *ref_b, "gb")
    gw, gb = vit_ops.weight_grad8(gy.transpose(0, 1).contiguous().transpose(0, 1), vit_ops.pack8(x))
    within(gw, *ref_w, "gw of a transposed gradient")
    gw, gb = vit_ops.weight_grad8(torch.empty(0, 4, device="cuda", dtype=dtype), vit_ops.pack8(torch.empty(0, 6, device="cuda", dtype=dtype)))
    assert not gw.any() and gw.shape == (4, 6) and not gb.any()
    x = torch.zeros(5, 64, device="cuda", dtype=dtype)                                            # a group that was not finite shows in its columns only
    x[3, 33] = math.nan
    gw, _ = vit_ops.weight_grad8(torch.ones(5, 8, device="cuda", dtype=dtype), vit_ops.pack8(x))
    assert torch.isnan(gw[:, 32:]).all() and not gw[:, :32].any()


@gpu
def test_linear8_matches_definition():
    g = gen(11)
    x = torch.randn(4, 37, 96, generator=g, device="cuda").requires_grad_(True)
    w = (torch.randn(48, 96, generator=g, device="cuda") * 0.1).requires_grad_(True)
    b = torch.randn(48, generator=g, device="cuda").requires_grad_(True)
    gy = torch.randn(4, 37, 48, generator=g, device="cuda")
    y = vit_ops.linear8(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    x64, w64, g64 = x.detach().double().reshape(-1, 96), w.detach().double(), gy.double().reshape(-1, 48)
    n = 100 * U                                                                                   # library products: one rounding per term
    within(y.detach().reshape(-1, 48), x64 @ w64.t() + b.detach().double(), n * (x64.abs() @ w64.abs().t() + b.detach().double().abs()), "y")
    within(gx.reshape(-1, 96), g64 @ w64, n * (g64.abs() @ w64.abs()), "gx")
    ref_w, ref_b = wgrad_reference(gy.reshape(-1, 48), round8_reference(x.detach().reshape(-1, 96))[0].cuda())
    within(gw, *ref_w, "gw")
    within(gb, *ref_b, "gb")
    assert torch.equal(torch.autograd.grad(vit_ops.linear8(x, w), w, gy)[0], gw)                  # no bias
    assert torch.equal(torch.autograd.grad(vit_ops.linear8(x.detach(), w.detach(), b), b, gy)[0], gb)
    assert torch.equal(torch.autograd.grad(vit_ops.linear8(x, w.detach()), x, gy)[0], gx)         # frozen weight: nothing packed


# ---- as a user runs them -------------------------------------------------------------------------------------------------------------------
def _decoder_step(q_tok, enc, mask, P, dtype):
    """vertices attend to an image's tokens, then the MLP: a run of the operators together"""
    s, y = vit_ops.layer_norm(q_tok, P["n1w"], P["n1b"], residual=P["pos"].expand_as(q_tok))
    b, n, c = y.shape
    kv = vit_ops.linear8(enc, P["wkv"]).unflatten(2, (2, 2, 32))
    q = vit_ops.linear8(y, P["wq"], P["bq"]).unflatten(2, (4, 32))
    a = vit_ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_mask=mask).reshape(b, n, 128)
    s, y = vit_ops.layer_norm(s, P["n2w"], P["n2b"], residual=vit_ops.linear8(a, P["wo"], P["bo"]))
    return s + vit_ops.linear8(vit_ops.gelu8(vit_ops.linear8(y, P["w1"], P["b1"])), P["w2"], P["b2"])


class Keep8(torch.autograd.Function):                                                        # gelu whose slope is taken at the 8-bit value
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(round8_reference(x.reshape(-1, x.shape[-1]).float())[0].to(x.device).view_as(x))
        return gelu64(x)

    @staticmethod
    def backward(ctx, g):
        return g * gelu_slope64(ctx.saved_tensors[0])

class Lin8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(round8_reference(x.reshape(-1, x.shape[-1]).float())[0].to(x.device).view_as(x), w)
        return x @ w.t()

    @staticmethod
    def backward(ctx, g):
        x8, w = ctx.saved_tensors
        return g @ w, g.reshape(-1, g.shape[-1]).t() @ x8.reshape(-1, x8.shape[-1])


def _decoder_reference(q_tok, enc, mask, P):
    """the same in float64 with straight-through 8-bit checkpoints"""
    ln = lambda t, w, b: torch.nn.functional.layer_norm(t, t.shape[-1:], w, b, 1e-6)
    s = q_tok + P["pos"]
    y = ln(s, P["n1w"], P["n1b"])
    b, n, c = y.shape
    kv = Lin8.apply(enc, P["wkv"]).unflatten(2, (2, 2, 32))
    q = (Lin8.apply(y, P["wq"]) + P["bq"]).unflatten(2, (4, 32)).permute(0, 2, 1, 3)
    k, v = (t.permute(0, 2, 1, 3).repeat_interleave(2, 1) for t in (kv[:, :, 0], kv[:, :, 1]))
    sc = (q @ k.transpose(2, 3) * 32 ** -0.5).masked_fill(~mask[:, None, None, :], -math.inf)
    a = (sc.softmax(3) @ v).permute(0, 2, 1, 3).reshape(b, n, 128)
    s = s + (Lin8.apply(a, P["wo"]) + P["bo"])
    y = ln(s, P["n2w"], P["n2b"])
    return s + (Lin8.apply(Keep8.apply(Lin8.apply(y, P["w1"]) + P["b1"]), P["w2"]) + P["b2"])


def _decoder_setup(seed=21):
    g = gen(seed)
    new = lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale
    P = dict(n1w=1 + new(96, scale=0.1), n1b=new(96, scale=0.1), n2w=1 + new(96, scale=0.1), n2b=new(96, scale=0.1), pos=new(1, 50, 96, scale=0.3),
             wkv=new(128, 64, scale=0.12), wq=new(128, 96, scale=0.1), bq=new(128, scale=0.1), wo=new(96, 128, scale=0.09), bo=new(96, scale=0.1),
             w1=new(384, 96, scale=0.1), b1=new(384, scale=0.1), w2=new(96, 384, scale=0.05), b2=new(96, scale=0.1))
    q_tok, enc = new(3, 50, 96), new(3, 77, 64)
    mask = torch.arange(77, device="cuda")[None] < torch.tensor([[77], [40], [5]], device="cuda")
    return P, q_tok, enc, mask, new(3, 50, 96)


@gpu
def test_a_decoder_block_of_them_together():
    """forward and every gradient of the run against float64.  The codes of both sides agree but where an fp32 activation and its float64
    twin fall on different sides of a rounding border, which moves a value by one step of 2^-6 relative to its group's maximum; such
    flips are rarer than 1 in 10^4 (fp32 activations are off by ~1e-6, a step is ~1e-2), so gradients are compared in norm: 1e-3"""
    P, q_tok, enc, mask, go = _decoder_setup()
    leaves = {k: v.clone().requires_grad_(True) for k, v in dict(P, q_tok=q_tok, enc=enc).items()}
    names = sorted(leaves)
    out = _decoder_step(leaves["q_tok"], leaves["enc"], mask, leaves, FP32)
    grads = torch.autograd.grad(out, [leaves[n] for n in names], go)
    l64 = {k: v.double().requires_grad_(True) for k, v in dict(P, q_tok=q_tok, enc=enc).items()}
    ref = _decoder_reference(l64["q_tok"], l64["enc"], mask, l64)
    refs = torch.autograd.grad(ref, [l64[n] for n in names], go.double())
    assert (out.detach().double() - ref.detach()).norm() <= 1e-5 * ref.detach().norm()
    for n, a, b in zip(names, grads, refs):
        assert (a.double() - b).norm() <= 1e-3 * b.norm(), n


def _small_vit():
    from scp_amd import dino
    torch.manual_seed(3)
    vit = dino.VisionTransformer(patch_size=8, embed_dim=128, depth=3, num_heads=2)
    for p in vit.parameters():                                                                    # trunc_normal(0.02) weights would make every block a near-identity
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=0.08)
    return vit


def _vit_reference(vit, img, layer, act8):
    """key_tokens_grad in float64"""
    lin = (lambda m, t: Lin8.apply(t, m.weight) + m.bias) if act8 else (lambda m, t: torch.nn.functional.linear(t, m.weight, m.bias))
    act = Keep8.apply if act8 else gelu64
    x = vit.prepare_tokens(img)
    ln = lambda m, t: torch.nn.functional.layer_norm(t, t.shape[-1:], m.weight, m.bias, m.eps)
    for blk in vit.blocks[:layer]:
        b, n, c = x.shape
        q, k, v = (t.transpose(1, 2) for t in lin(blk.attn.qkv, ln(blk.norm1, x)).view(b, n, 3, blk.attn.num_heads, -1).unbind(2))
        y = ((q @ k.transpose(2, 3) * blk.attn.scale).softmax(3) @ v).transpose(1, 2).reshape(b, n, c)
        x = x + lin(blk.attn.proj, y)
        x = x + lin(blk.mlp.fc2, act(lin(blk.mlp.fc1, ln(blk.norm2, x))))
    c, blk = x.shape[2], vit.blocks[layer]
    y = ln(blk.norm1, x)
    w, bias = blk.attn.qkv.weight[c:2 * c], blk.attn.qkv.bias[c:2 * c]
    return (Lin8.apply(y, w) if act8 else y @ w.t()) + bias


@gpu
@pytest.mark.parametrize("act8", [True, False], ids=["act8", "plain"])
def test_vit_fine_tuning_path(act8):
    """VisionTransformer.key_tokens_grad: keys as the frozen path computes them, gradients against float64 (2 blocks deep; products of
    fp32 library kernels, ~10^3 roundings of 6e-8 in norm: 1e-4; with 8-bit checkpoints 2e-3 for the codes that fall on the other side
    of a rounding border, as in the decoder test, through two blocks)"""
    import copy
    vit = _small_vit()
    img = torch.rand(2, 3, 40, 40)
    ref = copy.deepcopy(vit).double()
    out64 = _vit_reference(ref, img.double(), 2, act8)
    go = torch.randn(out64.shape)
    out64.backward(go.double())
    vit = vit.cuda()
    out = vit.key_tokens_grad(img.cuda(), layer=2, act8=act8)
    out.backward(go.cuda())
    assert (out.detach().double().cpu() - out64.detach()).norm() <= 1e-5 * out64.detach().norm()
    with torch.no_grad():
        frozen = vit.key_tokens(img.cuda(), layer=2)
    assert (frozen.double().cpu() - out64.detach()).norm() <= 1e-5 * out64.detach().norm()
    checked = 0
    for (name, p), (_, q) in zip(vit.named_parameters(), ref.named_parameters()):
        if q.grad is None:
            assert p.grad is None, name
            continue
        checked += 1
        assert (p.grad.double().cpu() - q.grad).norm() <= (2e-3 if act8 else 1e-4) * q.grad.norm() + 1e-12, name
    assert checked == 2 * 12 + 4 + 3                                                              # two blocks, norm1 + qkv of the third, patch embedding + class token


@gpu
def test_vit_fine_tuning_path_in_bf16():
    """MIXED_BF16: the same keys and gradients to bf16's accuracy (every value passes some 30 roundings of 2^-8 of itself: 5 % in norm)"""
    from scp_amd import dino
    vit = _small_vit().cuda()
    img = torch.rand(2, 3, 40, 40, device="cuda")
    want = vit.key_tokens_grad(img, layer=2, act8=False)
    go = torch.randn_like(want)
    want_g = torch.autograd.grad(want, [vit.blocks[0].attn.qkv.weight, vit.blocks[1].mlp.fc1.weight], go)
    dino.MIXED_BF16 = True
    try:
        got = vit.key_tokens_grad(img, layer=2)
        got_g = torch.autograd.grad(got, [vit.blocks[0].attn.qkv.weight, vit.blocks[1].mlp.fc1.weight], go.bfloat16())
    finally:
        dino.MIXED_BF16 = False
    assert got.dtype == BF16
    assert (got.detach().float() - want.detach()).norm() <= 0.05 * want.detach().norm()
    for a, b in zip(got_g, want_g):
        assert a.dtype == FP32 and (a - b).norm() <= 0.05 * b.norm()


@gpu
@pytest.mark.parametrize("op", ["norm", "attention"])
def test_gradients_against_differences(op):
    """directional derivative of the float64 definition by central differences (h = 1e-4: truncation ~1e-8) against the kernels' gradient;
    fp32 gradients of ~10^4 terms: 1e-4 of the sum of absolute terms"""
    g = gen(31)
    if op == "norm":
        ins = [torch.randn(20, 48, generator=g, device="cuda"), torch.randn(48, generator=g, device="cuda"), torch.randn(48, generator=g, device="cuda")]
        f64 = lambda x, w, b: torch.nn.functional.layer_norm(x, (48,), w, b, 1e-6)
        f = lambda x, w, b: vit_ops.layer_norm(x, w, b)
    else:
        q, k, v, _, _ = attn_inputs(2, 20, 30, 2, 1, 32, FP32, 33)
        ins = [q, k, v]
        f = lambda q, k, v: vit_ops.cross_attention(q, k, v)

        def f64(q, k, v):
            q, k, v = (t.permute(0, 2, 1, 3) for t in (q, k, v))
            return ((q @ k.transpose(2, 3) * 32 ** -0.5).softmax(3) @ v).permute(0, 2, 1, 3)
    go = torch.randn(f(*ins).shape, generator=g, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in ins]
    grads = torch.autograd.grad(f(*leaves), leaves, go)
    for i, gr in enumerate(grads):
        d = torch.randn(ins[i].shape, generator=g, device="cuda").double()
        at = lambda h: (f64(*[t.double() + (h * d if j == i else 0) for j, t in enumerate(ins)]) * go.double()).sum()
        diff = (at(1e-4) - at(-1e-4)) / 2e-4
        assert (diff - (gr.double() * d).sum()).abs() <= 1e-4 * (gr.double() * d).abs().sum(), i


@gpu
def test_second_derivatives_are_refused():
    g = gen(51)
    x = torch.randn(5, 64, generator=g, device="cuda").requires_grad_(True)
    w = torch.randn(64, 64, generator=g, device="cuda").requires_grad_(True)
    q = torch.randn(1, 4, 2, 32, generator=g, device="cuda").requires_grad_(True)
    for y, leaf in ((vit_ops.layer_norm(x), x), (vit_ops.gelu8(x), x), (vit_ops.linear8(x, w), x), (vit_ops.cross_attention(q, q, q), q)):
        first, = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), leaf)
            pytest.fail("a second derivative was not refused")


@gpu
def test_backward_twice_over_one_forward():
    g = gen(52)
    x, gy, w = (torch.randn(40, 64, generator=g, device="cuda") for _ in range(3))
    q, go = (torch.randn(2, 7, 2, 64, generator=g, device="cuda") for _ in range(2))
    x, w, q = (t.requires_grad_(True) for t in (x, w, q))
    for y, leaves, up in ((vit_ops.layer_norm(x), (x,), gy), (vit_ops.gelu8(x), (x,), gy), (vit_ops.linear8(x, w), (x, w), gy[:, :40].contiguous()),
                          (vit_ops.cross_attention(q, q, q), (q,), go)):
        a = torch.autograd.grad(y, leaves, up, retain_graph=True)
        keep = [t.clone() for t in a]
        torch.autograd.grad(y, leaves, 2 * up, retain_graph=True)
        b = torch.autograd.grad(y, leaves, up.transpose(0, 1).contiguous().transpose(0, 1))
        assert all(torch.equal(s, k) for s, k in zip(a, keep))                                    # not written again by the second pass
        library = len(leaves) == 2                                                                # linear8's gx: a library product, whose kernel goes by the layout
        if library:                                                                               # two fp32 sums of 40 terms: 2 x 40 roundings of sum|terms|
            within(b[0], a[0].double(), 80 * U * (up.double().abs() @ w.detach().double().abs()), "gx")
        assert all(torch.equal(s, t) for s, t in list(zip(a, b))[library:])


def _all_operators(seed=41):
    """outputs and gradients of each operator"""
    g = gen(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").requires_grad_(True)
    x, r, w, b = new(40, 96), new(40, 96), new(96), new(96)
    q, kv, lw, lb = new(2, 9, 2, 32), new(2, 70, 2, 2, 32), new(48, 96), new(48)
    s, y = vit_ops.layer_norm(x, w, b, residual=r)
    outs = [s, y, vit_ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1]), vit_ops.gelu8(x), vit_ops.linear8(x, lw, lb)]
    go = [torch.randn(o.shape, generator=g, device="cuda") for o in outs]
    return outs + list(torch.autograd.grad(outs, (x, r, w, b, q, kv, lw, lb), go))


@gpu
def test_saved_tensors_kept_on_the_host():
    """what the operators keep for their backward passes can be moved away by saved-tensor hooks; strided views come back contiguous"""
    plain = _all_operators()
    with torch.autograd.graph.save_on_cpu():
        moved = _all_operators()
    for i, (a, b) in enumerate(zip(plain, moved)):
        assert torch.equal(a, b), i


@gpu
def test_autocast_leaves_the_types():
    plain = _all_operators()
    with torch.autocast("cuda", dtype=BF16):
        cast = _all_operators()
    for i, (a, b) in enumerate(zip(plain, cast)):
        assert a.dtype == b.dtype == FP32 and torch.equal(a, b), i


@gpu
def test_lazily_negated_input():
    x = torch.randn(5, 64, generator=gen(3), device="cuda")
    neg = torch._neg_view(x)
    assert neg.is_neg() and torch.equal(vit_ops.layer_norm(neg), vit_ops.layer_norm(-x)) and torch.equal(vit_ops.gelu8(neg), vit_ops.gelu8(-x))


@gpu
def test_two_threads_at_once():
    """callers on two threads and streams: each gets the bits it gets alone"""
    import threading
    want = [_all_operators(s) for s in (51, 52)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = _all_operators(51 + i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_repeated_calls_give_the_same_bits():
    P, q_tok, enc, mask, go = _decoder_setup(5)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (q_tok, enc, P["w1"], P["wkv"], P["n1w"])]
        out = _decoder_step(leaves[0], leaves[1], mask, dict(P, w1=leaves[2], wkv=leaves[3], n1w=leaves[4]), FP32)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, go))

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


@gpu
def test_another_stream():
    P, q_tok, enc, mask, go = _decoder_setup(6)
    with torch.no_grad():
        want = _decoder_step(q_tok, enc, mask, P, FP32)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _decoder_step(q_tok, enc, mask, P, FP32)
        side.synchronize()
    assert torch.equal(got, want)


@gpu
def test_captured_and_replayed():
    """forward and backward of every operator in one graph, replayed on new inputs between eager work; a second graph of the same
    calls does not disturb the first"""
    g = gen(41)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, b, gy = new(70, 96), new(96), new(96), new(70, 96)
    q, k, v, go = new(2, 3, 4, 64), new(2, 300, 2, 64), new(2, 300, 2, 64), new(2, 3, 4, 64)

    def run():
        xs, ws, bs = (t.detach().requires_grad_(True) for t in (x, w, b))
        y = vit_ops.layer_norm(xs, ws, bs)
        out = [y.detach()] + list(torch.autograd.grad(y, (xs, ws, bs), gy))
        ls = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = vit_ops.cross_attention(*ls)
        out += [o.detach()] + list(torch.autograd.grad(o, ls, go))
        xs = x.detach().requires_grad_(True)
        z = vit_ops.gelu8(xs)
        out += [z.detach(), torch.autograd.grad(z, xs, gy)[0]]
        out += list(vit_ops.weight_grad8(gy, vit_ops.pack8(x)))
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    for i in range(4):
        for t in (x, w, b, gy, q, k, v, go):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        want = run()
        torch.cuda.synchronize()
        for graph, outs in graphs if i % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, c) for a, c in zip(outs, want)), i
