"""scp_amd.vit_ops at calls that tests/test_vit_ops.py does not make: exact ties, lazily negated gradients, forward-mode derivatives and
tracing, problems past a launch's limits, infinities, many steps of the pipelines.  Tolerances are bounds per element as there."""
import ctypes
import math

import pytest
import torch

from scp_amd import vit_ops
from test_vit_ops import BF16, FP32, U, attn_inputs, attn_reference, check_attn, gelu64, gelu_slope64, gen, gpu, half_step, spread_values, wgrad_reference, within


# ---- cross attention: the bits of the output that its rounding drops ----------------------------------------------------------------------
TIES = [  # batch, queries, keys, heads, kv_heads, attended keys (None: all); the forms of the forward pass
    (3, 1, 2, 2, 2, None), (2, 40, 4, 2, 1, None), (24, 250, 4, 6, 6, None), (24, 700, 2, 6, 6, None), (1, 1, 2050, 1, 1, 4), (1, 40, 2050, 2, 2, 2)]


def _even_weights(shape, seed):
    b, nq, nk, h, hk, kept = shape
    g = gen(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF16)
    k, v = new(b, nk, hk, 64), new(b, nk, hk, 64)
    mask = None
    if kept is not None:
        mask = torch.zeros(b, nk, dtype=torch.bool, device="cuda")
        mask[:, torch.linspace(3, nk - 2, kept).long()] = True
    return torch.zeros(b, nq, h, 64, device="cuda", dtype=BF16), k, v, mask, g


@gpu
@pytest.mark.parametrize("shape", TIES, ids=str)
def test_attention_output_low_bits_at_ties(shape):
    """q = 0: the output is the mean of 2 or 4 values of 8 bits, half-way between two bf16 numbers for one element in ten.  The bf16 output
    and its low byte together are within half a step of the byte, 2^-16 of the value, and 4 roundings of the sum."""
    from scp_amd import capi
    b, nq, nk, h, hk, kept = shape
    q, k, v, mask, _ = _even_weights(shape, sum(shape[:5]))
    p = capi.CrossAttnParams()
    p.batch, p.queries, p.keys, p.heads, p.kv_heads, p.head_dim, p.dtype, p.scale = b, nq, nk, h, hk, 64, 1, 1.0
    for f, t in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
        getattr(p, f)[:] = t.stride()[:3]
    lib = capi.lib()
    ws = torch.empty(lib.scp_cross_attention_forward_workspace(ctypes.byref(p)) + 16, dtype=torch.uint8, device="cuda")
    out, low = torch.empty_like(q), torch.empty(q.shape, dtype=torch.int8, device="cuda")
    at = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
    m8 = None if mask is None else mask.to(torch.uint8)
    assert lib.scp_cross_attention_forward(at(q), at(k), at(v), at(m8), ctypes.byref(p), at(out), at(low), None, at(ws), ws.numel(), capi.current_stream()) == 0
    on = torch.ones(b, nk, dtype=torch.float64, device="cuda") if mask is None else mask.double()
    wide = v.double().repeat_interleave(h // hk, 2)
    w = on / on.sum(1, keepdim=True)
    ref = torch.einsum("bn,bnhd->bhd", w, wide)[:, None].expand(b, nq, h, 64)
    mean_abs = torch.einsum("bn,bnhd->bhd", w, wide.abs())[:, None].expand(b, nq, h, 64)
    ties = (ref != ref.to(BF16).double()) & (ref == 0.5 * (ref.to(BF16).double() + (2 * ref - ref.to(BF16).double()).to(BF16).double()))
    assert ties.double().mean() > 0.03
    restored = (out.float().view(torch.int32) + low.int() * 256 + 128).view(FP32)
    within(restored, ref, 2.0 ** -16 * ref.abs() + 4 * U * mean_abs, "output with its low bits")


@gpu
@pytest.mark.parametrize("shape", TIES[:4], ids=str)
def test_attention_gradient_at_ties(shape):
    """two values that are each other with neighbouring channels swapped, a gradient that is the same for both of a pair: gO . v = gO . o for
    every key, gs = 0 and gq = 0.  What may be left: 2^-16 of o in delta, the roundings of two sums of 64 products, of gs, and of gq itself."""
    b, nq, nk, h, hk, _ = shape
    q, k, v, _, g = _even_weights((b, nq, 2, h, hk, None), 5 + sum(shape[:5]))
    v[:, 1] = v[:, 0].unflatten(-1, (32, 2)).flip(-1).flatten(-2)
    go = torch.randn(b, nq, h, 32, 1, generator=g, device="cuda").expand(-1, -1, -1, -1, 2).flatten(-2).to(BF16)
    leaf = q.requires_grad_(True)
    gq, = torch.autograd.grad(vit_ops.cross_attention(leaf, k, v, scale=1.0), leaf, go)
    G, V, K = go.double(), v.double().repeat_interleave(h // hk, 2), k.double().repeat_interleave(h // hk, 2)
    o = V.mean(1, keepdim=True)
    d_delta = (G.abs() * (2.0 ** -16 * o.abs() + 8 * U * V.abs().mean(1, keepdim=True))).sum(-1) + 66 * U * (G * o).abs().sum(-1)
    d_gp = 66 * U * (G.abs()[:, :, None] * V.abs()[:, None]).sum(-1)                              # b, q, key, head
    d_gs = 0.5 * (d_gp + d_delta[:, :, None]) * (1 + 2.0 ** -8)
    bound = (d_gs[..., None] * K.abs()[:, None]).sum(2) * (1 + 2.0 ** -7)
    within(gq, torch.zeros_like(bound), bound, "gq")


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nq", [1, 40, 700])
def test_attention_gradients_asked_for_one_by_one(dtype, nq):
    """any of gq, gk, gv alone or in pairs"""
    q, k, v, go, _ = attn_inputs(2, nq, 150, 4, 2, 64, dtype, 13)
    ref = attn_reference(q, k, v, None, 64 ** -0.5, go, dtype)
    for bits in range(1, 7):
        ls = [t.detach().requires_grad_(bool(bits >> i & 1)) for i, t in enumerate((q, k, v))]
        wanted = [t for t in ls if t.requires_grad]
        got = torch.autograd.grad(vit_ops.cross_attention(*ls), wanted, go)
        for a, name in zip(got, [f for i, f in enumerate(("gq", "gk", "gv")) if bits >> i & 1]):
            within(a, *ref[name], "%s of %d" % (name, bits))


WINDOWS = [  # a wavefront looks at the mask 64 tiles at a time: more keys than that, in the forms with own and with shared columns
    (8, 700, 4500, 6, 6, BF16, 4096), (8, 700, 2300, 6, 3, FP32, 2048), (8, 1100, 9000, 1, 1, BF16, 8192), (8, 2000, 4300, 2, 2, FP32, 4096)]


@gpu
@pytest.mark.parametrize("case", WINDOWS, ids=lambda c: "%dx%dx%d-%s" % (c[0], c[1], c[2], "fp32" if c[5] == FP32 else "bf16"))
def test_attention_over_several_windows_of_keys(case):
    b, nq, nk, h, hk, dtype, window = case
    q, k, v, go, g = attn_inputs(b, nq, nk, h, hk, 64, dtype, 19)
    mask = torch.rand(b, nk, generator=g, device="cuda") < 0.8
    mask[0, :window] = False                                                     # nothing in the first window
    mask[1, window:] = False                                                     # nothing after it
    mask[2, window - 70:window + 70] = False
    mask[3] = torch.arange(nk, device="cuda") == nk - 1
    k = torch.where(mask[:, :, None, None], k, torch.full_like(k, math.nan))
    check_attn(q, k, v, go, mask)


def _limits(**kw):
    from scp_amd import capi
    p = capi.CrossAttnParams()
    p.batch, p.queries, p.keys, p.heads, p.kv_heads, p.head_dim, p.dtype, p.scale = 1, 1, 1, 1, 1, 8, 1, 1.0
    for name, v in kw.items():
        setattr(p, name, v)
    for f, n, h in (("q_stride", p.queries, p.heads), ("k_stride", p.keys, p.kv_heads), ("v_stride", p.keys, p.kv_heads), ("g_stride", p.queries, p.heads)):
        getattr(p, f)[:] = (n * h * p.head_dim, h * p.head_dim, p.head_dim)
    return p


def test_attention_refuses_what_a_launch_cannot_hold():
    """a launch has fewer than 2^32 threads, so fewer than 2^24 workgroups of 256; the entry points say so before anything is launched"""
    from scp_amd import capi
    L = capi.lib()
    one, ws = ctypes.c_void_p(4096), ctypes.c_size_t(1 << 60)
    forward = lambda p: L.scp_cross_attention_forward(one, one, one, None, ctypes.byref(p), one, None, None, one, ws, None)
    backward = lambda p: L.scp_cross_attention_backward(one, one, one, None, one, None, one, one, ctypes.byref(p), one, one, one, one, ws, None)
    p = _limits(batch=(1 << 24) - 3)                                             # a workgroup per head, rounded up to the 8 XCDs
    assert forward(p) != 0 and "workgroups" in L.scp_last_error().decode()
    assert L.scp_cross_attention_backward_workspace(ctypes.byref(p)) == 0
    p = _limits(batch=1 << 23, heads=2)                                          # two rows a head: a workgroup each in the forward pass ...
    assert backward(p) != 0 and "workgroups" in L.scp_last_error().decode()      # ... and one more for its key in the backward pass
    p = _limits(batch=1 << 20, queries=1 << 10, dtype=0)                         # 2^30 rows of q and of g_out to cut into parts, 64 a workgroup
    assert backward(p) != 0 and "workgroups" in L.scp_last_error().decode()
    assert L.scp_cross_attention_backward_workspace(ctypes.byref(_limits(batch=1 << 20, heads=4))) > 0


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_attention_takes_backward_what_it_takes_forward(dtype):
    """tokens so far apart that 128 of them are within 2^31 bytes and 130 are not"""
    step = (1 << 31) // (129 * torch.finfo(dtype).bits // 8) // 8 * 8 + 8
    q, k, v, go, _ = attn_inputs(1, 3, 3, 1, 1, 64, dtype, 10)
    far = []
    for t in (q, k, v):
        wide = torch.empty(3, step, dtype=dtype, device="cuda")[None, :, None, :64]
        far.append(wide.copy_(t))
    check_attn(*far, go)


def test_single_queries_are_split_where_that_saves_round_trips():
    """no workspace: the keys are not split.  The choice goes by the keys that a workgroup walks and by the number of workgroups, without a
    step between neighbouring batches"""
    from scp_amd import capi

    def split(batch, keys, dtype, dim=64):
        p = _limits(batch=batch, heads=6, kv_heads=6, keys=keys, dtype=dtype, head_dim=dim)
        return capi.lib().scp_cross_attention_forward_workspace(ctypes.byref(p)) // (batch * 6 * (dim + 2) * 4)
    for dtype in (0, 1):
        assert [split(b, 1025, dtype) for b in (30, 31, 32, 33, 64)] == [0] * 5
        assert [split(b, 257, dtype) for b in (1, 4, 16, 32)] == [0] * 4
        assert [split(b, 4097, dtype) for b in (1, 4, 8, 16, 31, 32)] == [6, 6, 5, 2, 0, 0]


# ---- incoming gradients and other kinds of derivatives --------------------------------------------------------------------------------------
def _calls(seed=71, dtype=FP32):
    """(name, output, leaves) of every operator with a gradient"""
    g = gen(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype).requires_grad_(True)
    x, r, w, b, q, kv, lw, lb = new(40, 96), new(40, 96), new(96), new(96), new(2, 9, 2, 32), new(2, 70, 2, 2, 32), new(48, 96), new(48)
    return [("norm", vit_ops.layer_norm(x, w, b), (x, w, b)), ("norm + residual", vit_ops.layer_norm(x, w, b, residual=r), (x, r, w, b)),
            ("attention", vit_ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1]), (q, kv)), ("gelu8", vit_ops.gelu8(x), (x,)), ("linear8", vit_ops.linear8(x, lw, lb), (x, lw, lb))]


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_lazily_negated_gradients(dtype):
    """autograd hands a gradient with the negative bit on as it is (the imaginary part of a conjugate is one)"""
    for name, out, leaves in _calls(dtype=dtype):
        outs = out if isinstance(out, tuple) else (out,)
        gs = [torch.randn(o.shape, generator=gen(72), device="cuda").to(dtype) for o in outs]
        want = torch.autograd.grad(outs, leaves, [-t for t in gs], retain_graph=True)
        neg = [torch._neg_view(t) for t in gs]
        assert all(t.is_neg() for t in neg)
        for a, c in zip(torch.autograd.grad(outs, leaves, neg), want):
            assert torch.equal(a, c), name
    x = torch.randn(30, 64, generator=gen(73), device="cuda").to(dtype)
    p = vit_ops.pack8(x)
    for a, c in zip(vit_ops.weight_grad8(torch._neg_view(x), p), vit_ops.weight_grad8(-x, p)):
        assert torch.equal(a, c)


@gpu
def test_a_conjugate_brings_a_negated_gradient():
    """the same through ordinary operations"""
    x = torch.randn(6, 64, generator=gen(74), device="cuda").requires_grad_(True)
    up = torch.randn(6, 64, generator=gen(75), device="cuda")
    through = lambda y: (torch.complex(torch.zeros_like(y), y).conj().imag * up).sum()            # = -(y up).sum()
    got, = torch.autograd.grad(through(vit_ops.gelu8(x)), x)
    want, = torch.autograd.grad(vit_ops.gelu8(x), x, -up)
    assert torch.equal(got, want)


def _entries():
    x, w, b, r = (torch.randn(*s, device="cuda") for s in ((4, 64), (64,), (64,), (4, 64)))
    q, k, lw, lb = (torch.randn(*s, device="cuda") for s in ((1, 3, 2, 32), (1, 5, 2, 32), (8, 64), (8,)))
    p = vit_ops.pack8(x)
    return [(lambda *a: vit_ops.layer_norm(a[0], a[1], a[2], residual=a[3]), [x, w, b, r]), (lambda *a: vit_ops.cross_attention(*a), [q, k, k.clone()]),
            (lambda *a: vit_ops.gelu8(*a), [x]), (lambda *a: vit_ops.linear8(*a), [x, lw, lb]), (lambda a: vit_ops.pack8(a).codes, [x]),
            (lambda a: vit_ops.weight_grad8(a, p)[0], [r])]


@gpu
def test_forward_mode_derivatives_are_refused():
    """a tangent on any operand: an error, not a result without it"""
    import torch.autograd.forward_ad as fwd
    for i, (call, args) in enumerate(_entries()):
        call(*args)
        for j in range(len(args)):
            with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*[fwd.make_dual(t, torch.ones_like(t)) if n == j else t for n, t in enumerate(args)])
                pytest.fail("operand %d of call %d was not refused" % (j, i))


@gpu
def test_tracing_is_refused():
    """torch.jit.trace would keep the result of the traced call as a constant"""
    for i, (call, args) in enumerate(_entries()):
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(call, tuple(args), check_trace=False)
            pytest.fail("call %d was traced" % i)


@gpu
@pytest.mark.child_process
def test_a_captured_backward_pass_beside_an_eager_graph_is_refused():
    """the eager graph's accumulator belongs to the default stream; torch's engine would end the process at it.  With the eager results gone the
    same capture runs, and replays what the eager pass computes"""
    for pick in range(5):
        name, eager, leaves = _calls()[pick]
        first = leaves[0]
        base = first.detach().clone().requires_grad_(True)                       # a leaf behind a view, too
        make = [lambda t: vit_ops.layer_norm(t, leaves[1], leaves[2]), lambda t: vit_ops.layer_norm(t, leaves[2], leaves[3], residual=leaves[1])[1],
                lambda t: vit_ops.cross_attention(t, leaves[1].detach()[:, :, 0], leaves[1].detach()[:, :, 1]), vit_ops.gelu8, lambda t: vit_ops.linear8(t, leaves[1], leaves[2])][pick]
        del eager
        go = torch.randn(first.shape if name != "linear8" else (40, 48), generator=gen(77), device="cuda")
        want, = torch.autograd.grad(make(base), base, go)
        torch.cuda.synchronize()
        for view in (False, True):
            alive = base * 1.0 if view else make(base)                           # an eager graph of the leaf
            graph = torch.cuda.CUDAGraph()
            with pytest.raises(RuntimeError, match="being captured"):
                with torch.cuda.graph(graph):
                    torch.autograd.grad(make(base[:] if view else base), base, go)
                    pytest.fail("%s was not refused" % name)
            torch.cuda.synchronize()
            del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(make(base), base, go)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


@gpu
def test_exceptions_keep_their_type():
    """what a saved-tensor hook raises, and torch's own errors, arrive as they are"""
    class Stop(Exception):
        pass

    def hook(t):
        raise Stop("stop")
    for i, (call, args) in enumerate(_entries()[:4]):
        with pytest.raises(Stop), torch.autograd.graph.saved_tensors_hooks(hook, lambda t: t):
            call(*[t.requires_grad_(True) for t in args])
    huge = torch.zeros(1, 8192, device="cuda").expand(1 << 26, 8192)             # 2 TiB as rows of their own
    with pytest.raises(torch.OutOfMemoryError):
        vit_ops.layer_norm(huge)
    with pytest.raises(TypeError):
        vit_ops.layer_norm(torch.zeros(2, 8, device="cuda"), eps="small")


@gpu
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("last", ["linear8", "gelu8", "attention", "norm"])
def test_inside_a_checkpointed_block(last, reentrant):
    """torch.utils.checkpoint ends the second forward pass by an exception of its own out of the last saved tensor"""
    from torch.utils.checkpoint import checkpoint
    g = gen(76)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").requires_grad_(True)
    x, n, w1, b1, w2 = new(2, 20, 64), new(64), new(96, 64), new(96), new(64, 96)

    def block(t):
        y = vit_ops.linear8(vit_ops.gelu8(vit_ops.linear8(vit_ops.layer_norm(t, n), w1, b1)), w2)
        if last == "linear8":
            return y
        if last == "gelu8":
            return vit_ops.gelu8(y)
        if last == "norm":
            return vit_ops.layer_norm(y, n, residual=t)[1]
        return vit_ops.cross_attention(*(y.unflatten(2, (2, 32)) for _ in range(3)))
    plain, kept = block(x), checkpoint(block, x, use_reentrant=reentrant)
    go = torch.randn(plain.shape, generator=g, device="cuda")
    grads = []
    for out in (plain, kept):
        for t in (x, n, w1, b1, w2):
            t.grad = None
        out.backward(go)
        grads.append([t.grad for t in (x, n, w1, b1, w2)])
    assert torch.equal(plain, kept)
    assert all(torch.equal(a, c) for a, c in zip(*grads))


@gpu
def test_tensors_without_memory_of_their_own_are_refused():
    """a subclass that answers for its operations itself (a distributed or a fake tensor), a zero tensor: nothing is there to be read"""
    class Answers(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
            return args[0]
    for i, (call, args) in enumerate(_entries()):
        with pytest.raises(RuntimeError, match="memory"):                        # torch.func's wrappers are no plain tensors either
            torch.func.vmap(call)(*[t[None] for t in args])
        with pytest.raises(RuntimeError, match="memory"):
            torch.func.grad(lambda *a: call(*a).sum())(*args)
        for j in range(len(args)):
            for odd in (Answers(args[j]), torch._efficientzerotensor(args[j].shape, device="cuda")):
                with pytest.raises(RuntimeError, match="memory"):
                    call(*[odd if n == j else t for n, t in enumerate(args)])
                    pytest.fail("operand %d of call %d was not refused" % (j, i))


@gpu
@pytest.mark.child_process
def test_a_captured_backward_pass_that_does_not_reach_the_eager_leaf():
    """gradients of x alone, while an eager graph of the weight is alive: nothing of that graph runs"""
    g = gen(79)
    x, w, gy = (torch.randn(*s, generator=g, device="cuda") for s in ((40, 96), (48, 96), (40, 48)))
    w.requires_grad_(True)
    alive = w * 1.0
    leaf = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(vit_ops.linear8(vit_ops.gelu8(leaf), w), leaf, gy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inner = x.detach().requires_grad_(True)
        got, = torch.autograd.grad(vit_ops.linear8(vit_ops.gelu8(inner), w), inner, gy)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert alive.requires_grad


# ---- sizes ---------------------------------------------------------------------------------------------------------------------------------------
@gpu
def test_linear8_refuses_at_once_what_its_backward_pass_cannot_take():
    c = (1 << 20) + 8
    x, w = torch.randn(2, c, device="cuda"), torch.randn(1, c, device="cuda")
    with pytest.raises(RuntimeError, match="2\\^20"):
        vit_ops.linear8(x, w.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="2\\^20"):
        vit_ops.linear8(x, w, torch.zeros(1, device="cuda", requires_grad=True))
    with pytest.raises(RuntimeError, match="2\\^20"):
        vit_ops.linear8(torch.randn(2, 8, device="cuda"), torch.randn(c, 8, device="cuda").requires_grad_(True))
    leaf = x.clone().requires_grad_(True)                                        # a frozen weight asks for no weight gradient
    gx, = torch.autograd.grad(vit_ops.linear8(leaf, w), leaf, torch.ones(2, 1, device="cuda"))
    assert torch.equal(gx, w.expand(2, c))


@gpu
@pytest.mark.parametrize("shape", [(20000, 1), (8192, 4), (32768, 1), (4096, 8), (1024, 32), (512, 64), (300, 96)], ids=str)
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_layer_norm_gradients_of_narrow_rows(shape, dtype):
    from test_vit_ops import norm_reference
    rows, c = shape
    g = gen(rows + c)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, gy, w, b = (3 * new(rows, c) + 1).to(dtype).requires_grad_(True), new(rows, c).to(dtype), (1 + 0.3 * new(c)).requires_grad_(True), new(c).requires_grad_(True)
    ref = norm_reference(x.detach(), None, w.detach(), b.detach(), 1e-3, gy, None, dtype)
    y = vit_ops.layer_norm(x, w, b, eps=1e-3)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    for got, name in ((y.detach(), "y"), (gx, "gx"), (gw, "gw"), (gb, "gb")):
        within(got, *ref[name], name)


def test_layer_norm_gives_narrow_rows_to_many_workgroups():
    """one workgroup holds 16 rows at a time: what it takes goes by the number of its rounds, whatever the rows' width.  A workspace is asked
    for where there is more than one workgroup."""
    from scp_amd import capi
    size = capi.lib().scp_layernorm_backward_workspace
    for rows, c in ((32768, 1), (4096, 8), (1024, 32), (512, 64)):
        assert size(rows, c) > 0, (rows, c)
    for rows, c in ((4, 384), (16, 64), (1, 8192), (3, 1001)):
        assert size(rows, c) == 0, (rows, c)


@gpu
def test_layer_norm_of_more_rows_than_one_launch_holds():
    """2^28 rows and some: 2^24 workgroups of 16 rows would have 2^32 threads.  y of two channels is +-1 scaled; both ends are compared"""
    from test_vit_ops import norm_reference
    rows = (1 << 28) + 37
    x = torch.empty(rows, 2, device="cuda", dtype=BF16).normal_(generator=gen(3))
    w, b = torch.tensor([1.5, -0.75], device="cuda"), torch.tensor([0.25, 3.0], device="cuda")
    x.requires_grad_(True)
    y = vit_ops.layer_norm(x, w, b, eps=1e-2)
    gx, = torch.autograd.grad(y, x, x.detach())
    for part in (slice(0, 3000), slice((1 << 27) - 1500, (1 << 27) + 1500), slice((1 << 28) - 1500, (1 << 28) + 37)):
        xs = x.detach()[part].contiguous()
        ref = norm_reference(xs, None, w, b, 1e-2, xs, None, BF16)
        within(y.detach()[part], *ref["y"], "y")
        within(gx[part], *ref["gx"], "gx")


# ---- more than 2^31 elements ---------------------------------------------------------------------------------------------------------------------
def _far(rows, c, seed):
    return torch.empty(rows, c, dtype=BF16, device="cuda").normal_(generator=gen(seed))


ENDS = (slice(0, 40), slice(-40, None))


@gpu
def test_layer_norm_past_32_bits():
    """rows are independent: both ends are what they are alone, bit for bit"""
    rows, c = (1 << 18) + 37, 8192
    x, w = _far(rows, c, 1).requires_grad_(True), torch.randn(c, generator=gen(2), device="cuda")
    total, y = vit_ops.layer_norm(x, w, residual=x.detach())
    gx, = torch.autograd.grad((total, y), x, (x.detach(), y.detach()))
    for part in ENDS:
        xs = x.detach()[part].clone().requires_grad_(True)
        ts, ys = vit_ops.layer_norm(xs, w, residual=xs.detach())
        gs, = torch.autograd.grad((ts, ys), xs, (xs.detach(), ys.detach()))
        assert torch.equal(total[part], ts) and torch.equal(y[part], ys) and torch.equal(gx[part], gs)


@gpu
@pytest.mark.parametrize("c", [32768, 32757])
def test_checkpoints_past_32_bits(c):
    rows = (1 << 31) // c + 50
    x = _far(rows, c, 3).requires_grad_(True)
    y = vit_ops.gelu8(x)
    gx, = torch.autograd.grad(y, x, x.detach())
    p = vit_ops.pack8(x)
    back = p.unpack()
    for part in ENDS:
        xs = x.detach()[part].clone().requires_grad_(True)
        ys, ps = vit_ops.gelu8(xs), vit_ops.pack8(xs)
        gs, = torch.autograd.grad(ys, xs, xs.detach())
        assert torch.equal(y[part], ys) and torch.equal(gx[part], gs) and torch.equal(p.codes[part], ps.codes) and torch.equal(p.exps[part], ps.exps) and torch.equal(back[part], ps.unpack())


@gpu
def test_weight_grad8_past_32_bits():
    """the last rows alone differ from zero: what they give is what they give alone, up to the order of the sums"""
    rows, n, k = (1 << 20) + 333, 2056, 40
    gy, x = torch.zeros(rows, n, dtype=BF16, device="cuda"), torch.zeros(rows, k, dtype=BF16, device="cuda")
    last = slice(rows - 300, rows)
    gy[last], x[last] = _far(300, n, 4), _far(300, k, 5)
    ref_w, ref_b = wgrad_reference(gy[last], vit_ops.pack8(x[last].contiguous()).unpack(FP32).double())
    gw, gb = vit_ops.weight_grad8(gy, vit_ops.pack8(x))
    within(gw, *ref_w, "gw")
    within(gb, *ref_b, "gb")


@gpu
@pytest.mark.parametrize("dtype,nq", [(BF16, 300007), (FP32, 150011)], ids=["bf16", "fp32"])
def test_attention_of_queries_past_32_bits(dtype, nq):
    """the results of rows past 2^31 elements (of the parts, in fp32) against the definition; gk and gv are those of a gradient of these rows alone"""
    h, d, nk, part = 120, 64, 40, slice(nq - 60, nq)
    k, v = (torch.randn(1, nk, h, d, generator=gen(6 + i), device="cuda").to(dtype).requires_grad_(True) for i in range(2))
    q = torch.empty(1, nq, h, d, dtype=dtype, device="cuda").normal_(generator=gen(8)).requires_grad_(True)
    o = vit_ops.cross_attention(q, k, v)
    go = torch.zeros_like(q, requires_grad=False)
    go[:, part] = torch.randn(1, 60, h, d, generator=gen(9), device="cuda").to(dtype)
    gq, gk, gv = torch.autograd.grad(o, (q, k, v), go)
    ref = attn_reference(q.detach()[:, part], k.detach(), v.detach(), None, d ** -0.5, go[:, part], dtype)
    within(o.detach()[:, part], *ref["o"], "o")
    within(gq[:, part], *ref["gq"], "gq")
    within(gk, *ref["gk"], "gk")                                                 # (every other term is 0)
    within(gv, *ref["gv"], "gv")
    assert not gq[:, :nq - 60].any()


# ---- 8-bit checkpoints --------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(200, 40, 48), (200, 37, 41), (1000, 333, 144), (9000, 1536, 384), (9001, 1535, 383)], ids=str)
def test_weight_grad8_of_infinities(shape, dtype):
    """an infinite gradient gives what the sum of products gives: an infinity where the input is not 0, NaN where it is, or where infinities
    of both signs meet; a NaN gives NaN; every other column is untouched"""
    rows, n, k = shape
    x = spread_values(rows, k, dtype, 3).clamp(-50, 50)
    gy = torch.randn(rows, n, generator=gen(4), device="cuda").to(dtype)
    gy[7, 3], gy[rows - 1, 5], gy[64, 9], gy[65, 9], gy[100, 11] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    x[7, 2] = 0.0
    p = vit_ops.pack8(x)
    x8 = p.unpack(FP32).double()
    gw, gb = vit_ops.weight_grad8(gy, p)
    hit = torch.tensor([3, 5, 9, 11], device="cuda")
    ref = (gy.double()[:, hit, None] * x8[:, None]).sum(0)
    assert torch.isinf(ref[0]).any() and torch.isnan(ref[0, 2])
    signs = lambda t: torch.nan_to_num(t.double(), 0.0, 1.0, -1.0)
    assert torch.equal(torch.isnan(gw[hit]), torch.isnan(ref)) and torch.equal(signs(gw[hit]), signs(ref))
    assert gb[3] == math.inf and gb[5] == -math.inf and gb[9].isnan() and gb[11].isnan()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[hit] = False
    ref_w, ref_b = wgrad_reference(gy[:, rest].contiguous(), x8)
    within(gw[rest], *ref_w, "gw")
    within(gb[rest], *ref_b, "gb")


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nk", [(1536, 384), (1535, 383)], ids=["aligned", "ragged"])
@pytest.mark.parametrize("steps", [3, 4, 5, 37, 38])
def test_weight_grad8_over_many_steps(steps, nk, dtype):
    """rows for `steps` steps of 64 in every workgroup (about one workgroup per CU), the last one short: registers and LDS buffers are used
    again and again from the third step on"""
    n, k = nk
    tiles = -(-n // (128 if dtype == FP32 else 256)) * -(-k // 128)
    rows = 256 // tiles * steps * 64 - 29
    x = spread_values(rows, k, dtype, steps).clamp(-50, 50)
    gy = torch.randn(rows, n, generator=gen(steps), device="cuda").to(dtype)
    p = vit_ops.pack8(x)
    gw, gb = vit_ops.weight_grad8(gy, p)
    ref_w, ref_b = wgrad_reference(gy, p.unpack(FP32).double())                  # (the codes themselves: test_pack8_is_the_format)
    # every term is rounded in at most 64 steps of a workgroup and once per workgroup when they are added up
    tight = (64 * steps + 64 + 256 // tiles) / (rows + 64)
    within(gw, ref_w[0], tight * ref_w[1], "gw")
    within(gb, ref_b[0], tight * ref_b[1], "gb")


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("c", [1536, 1500])
def test_checkpoints_of_more_values_than_threads(c, dtype):
    """over 33.5 million values every thread takes further pieces"""
    rows = 24001
    x = spread_values(rows, c, dtype, c).clamp(-30, 30)
    p = vit_ops.pack8(x)
    t = torch.nn.functional.pad(x.float(), (0, -c % 32)).view(rows, -1, 32)
    field = ((t.abs().amax(2, keepdim=True).view(torch.int32) >> 23) - 6).clamp(min=1)
    step = (field << 23).view(FP32)
    code = (t.double() / step.double()).round().clamp(-127, 127)
    assert torch.equal(p.exps.int(), field[..., 0])
    assert torch.equal(p.codes.double(), code.view(rows, -1)[:, :c])
    x8 = (code * step.double()).view(rows, -1)[:, :c]
    del code, step, t
    assert torch.equal(p.unpack(FP32).double(), x8)
    leaf, gy = x.requires_grad_(True), torch.randn(rows, c, generator=gen(78), device="cuda").to(dtype)
    y = vit_ops.gelu8(leaf)
    gx, = torch.autograd.grad(y, leaf, gy)
    ref = gelu64(x.detach().double())                                            # bounds as in test_gelu8_matches_definition
    err = 4e-7 * x.detach().double().abs() + 2 * U * ref.abs()
    within(y.detach(), ref, err + half_step(dtype) * (ref.abs() + err), "y")
    slope = gelu_slope64(x8)
    ref = gy.double() * slope
    err = gy.double().abs() * (4e-7 * (1 + slope.abs())) + 2 * U * ref.abs()
    within(gx, ref, err + half_step(dtype) * (ref.abs() + err), "gx")


# ---- linear8 ----------------------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("bias", [True, False])
def test_linear8_of_each_type_matches_definition(dtype, bias):
    """products of the operands' type with fp32 sums: one rounding per term, and one to the type"""
    g = gen(12)
    new = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)
    x, w, b, gy = new(3, 50, 96), new(80, 96, scale=0.1), new(80) if bias else None, new(3, 50, 80)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = vit_ops.linear8(x, w, b)
    got = torch.autograd.grad(y, leaves, gy)
    assert y.dtype == dtype and all(t.dtype == dtype for t in got)
    x64, w64, g64, b64 = x.detach().double().reshape(-1, 96), w.detach().double(), gy.double().reshape(-1, 80), b.detach().double() if bias else torch.zeros(80, device="cuda", dtype=torch.float64)
    rounded = lambda val, err: (val, err + (half_step(BF16) if dtype == BF16 else 0.0) * (val.abs() + err))
    within(y.detach().reshape(-1, 80), *rounded(x64 @ w64.t() + b64, 104 * U * (x64.abs() @ w64.abs().t() + b64.abs())), "y")
    within(got[0].reshape(-1, 96), *rounded(g64 @ w64, 88 * U * (g64.abs() @ w64.abs())), "gx")
    ref_w, ref_b = wgrad_reference(gy.reshape(-1, 80), vit_ops.pack8(x.detach()).unpack(FP32).double().reshape(-1, 96))
    within(got[1], *rounded(*ref_w), "gw")
    if bias:
        within(got[2], *rounded(*ref_b), "gb")


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_linear8_makes_no_batched_product(dtype):
    """strided inputs and gradients, weights frozen or not, transposed views as weights: every product is a two-dimensional one"""
    from torch.utils._python_dispatch import TorchDispatchMode

    class NoBatch(TorchDispatchMode):
        seen = 0

        def __torch_dispatch__(self, f, types, args=(), kwargs=None):
            assert "bmm" not in str(f), f
            NoBatch.seen += "mm" in str(f)
            return f(*args, **(kwargs or {}))
    g = gen(14)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    base, b = new(5, 4, 6, 32), new(24)
    xs = [base[0], base[:, 0].transpose(0, 1), base.permute(1, 0, 2, 3), new(4, 32, 5).transpose(1, 2), base[0, 0, 0], base[:, :, :, ::2].transpose(0, 1)]
    for i, x in enumerate(xs):
        k = x.shape[-1]
        for w in (new(24, k), new(k, 24).t()):
            gy = new(*x.shape[:-1][::-1], 24)
            gy = gy.permute(*reversed(range(gy.dim() - 1)), gy.dim() - 1)        # strided as well
            for frozen in (True, False):
                plain = x.contiguous().clone().requires_grad_(True), w.contiguous().clone().requires_grad_(not frozen)
                want_y = vit_ops.linear8(plain[0], plain[1], b)
                want = torch.autograd.grad(want_y, [t for t in plain if t.requires_grad], gy.contiguous())
                xs_, ws_ = x.detach().requires_grad_(True), w.detach().requires_grad_(not frozen)
                with NoBatch():
                    y = vit_ops.linear8(xs_, ws_, b)
                    got = torch.autograd.grad(y, [t for t in (xs_, ws_) if t.requires_grad], gy)
                    with torch.no_grad():
                        again = vit_ops.linear8(x, w.detach(), b)
                for a, c in ((y, want_y), (again, want_y)) + tuple(zip(got, want)):
                    assert a.shape == c.shape
                    # the library's kernel goes by the weight's layout: sums of at most 32 products in another order
                    scale = a.detach().double().abs().amax() + 1
                    assert (a.detach().double() - c.detach().double()).abs().max() <= (2 * half_step(dtype) + 200 * U) * scale, i
    assert NoBatch.seen > 0


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16], ids=["fp32", "bf16"])
def test_linear8_of_a_bias_alone_keeps_no_checkpoint(dtype):
    """a frozen weight: nothing of x's size is held for the backward pass"""
    g = gen(16)
    x, w, gy = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((3, 500, 640), (72, 640), (3, 500, 72)))
    b = torch.zeros(72, device="cuda", dtype=dtype, requires_grad=True)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t.numel()) or t, lambda t: t):
        y = vit_ops.linear8(x, w, b)
    assert max(held, default=0) <= w.numel() and w.numel() < x.numel()
    val, bound = wgrad_reference(gy.reshape(-1, 72), torch.zeros(1500, 1, dtype=torch.float64, device="cuda"))[1]
    got, = torch.autograd.grad(y, b, gy)
    within(got, val, bound + (half_step(BF16) * (val.abs() + bound) if dtype == BF16 else 0), "gb")
    full = torch.autograd.grad(vit_ops.linear8(x, w.clone().requires_grad_(True), b), b, gy)[0]      # asked for alone, the weight could have had one
    within(full, val, bound + (half_step(BF16) * (val.abs() + bound) if dtype == BF16 else 0), "gb beside a weight")


@gpu
def test_results_can_be_changed_in_place():
    x, w, b = (torch.randn(*s, generator=gen(15), device="cuda").requires_grad_(True) for s in ((2, 3, 32), (16, 32), (16,)))
    for call in (lambda t: vit_ops.linear8(t, w, b), lambda t: vit_ops.linear8(t, w), lambda t: vit_ops.linear8(t[0], w, b), lambda t: vit_ops.linear8(t[0, 0], w, b), vit_ops.gelu8,
                 vit_ops.layer_norm):
        want, = torch.autograd.grad(3 * call(x), x, torch.ones_like(call(x)))
        got, = torch.autograd.grad(call(x).mul_(3), x, torch.ones_like(call(x)))
        assert torch.equal(got, want)
    q = x[None]
    o = vit_ops.cross_attention(q, q, q).mul_(3)                                 # kept for its backward pass: changing it is noticed
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o, x, torch.ones_like(o))


# ---- build ------------------------------------------------------------------------------------------------------------------------------------------
def test_the_binding_is_built_again_for_another_torch(monkeypatch):
    """its sources may be older than it is: what it was compiled against counts too, and loading one of another version is an error"""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("scp_build_edges", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(vit_ops.__file__))), "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    build.build(verbose=False)
    assert not build.binding_stale() and not build.needs_build()
    monkeypatch.setattr(torch, "__version__", "2.99.0+rocm9.9")
    assert build.binding_stale() and build.needs_build()
    monkeypatch.setattr(vit_ops, "_binding", None)
    with pytest.raises(RuntimeError, match="built against torch"):
        vit_ops._load()
