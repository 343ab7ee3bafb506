"""scp_amd/vit_ops.py -- the operators of a transformer block WITH gradients: what training a ViT, or a decoder that attends to its tokens,
needs next to the forward-only operators of scp_amd.dino (the reference's blocks, vision_transformer_flexible.py:54-132, are ordinary
modules; its pipeline keeps them frozen).

  layer_norm       LayerNorm, alone or with the residual add in front of it          (csrc/layernorm_train.hip)
  cross_attention  queries of one length against keys / values of another            (csrc/cross_attn.hip)
  gelu8            erf GELU whose input is kept for the backward pass in 8 bits       (csrc/act8.hip)
  linear8          linear layer whose input is kept for the backward pass in 8 bits   (csrc/act8_wgrad.hip)
  pack8, Packed8, weight_grad8: the 8-bit checkpoint by itself, and the weight gradient taken from it
Argument checks, allocation and autograd nodes are compiled (csrc/vit_ops_binding.cpp).

float32 and bfloat16 GPU tensors on the current device only, anything else raises RuntimeError (no CPU fallback).  Statistics, softmax and
sums are fp32, and results are rounded to the type they are returned in.  In between bfloat16 attention rounds its probabilities and score
gradients to bfloat16 for the products they enter (not those of a single query, nor in a backward pass over at most 16 rows or keys): the
error of its results is 1.4 times that of their own rounding.  No atomics: a call repeated gives the same bits.  Launches
go to the current stream; workspaces come from torch's allocator, so a call can be captured into a HIP graph; a
captured backward pass is refused while an eager graph of the same leaves is alive, which would end the process.  Once differentiable,
in reverse mode: a forward-mode tangent is refused, and so is torch.jit.trace."""
import ctypes
import importlib.util
import os

import torch

from . import capi

BINDING_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib", "scp_vit_ops.so")
_binding = None


def _load():
    """csrc/vit_ops_binding.cpp on the library of scp_amd.capi: checks, allocation and autograd nodes"""
    global _binding
    if not os.path.exists(BINDING_PATH):
        raise RuntimeError("scp_amd: %s is missing -- build it with `python self-corr-pose_amd/build.py` (there is no fallback)" % BINDING_PATH)
    lib = capi.lib()
    spec = importlib.util.spec_from_file_location("scp_vit_ops", BINDING_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    if module.torch_version != torch.__version__.split("+")[0]:
        raise RuntimeError("scp_amd: %s was built against torch %s, this is torch %s -- build it again with `python self-corr-pose_amd/build.py`"
                           % (BINDING_PATH, module.torch_version, torch.__version__))
    module.init({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in module.entries})
    _binding = module
    return module


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-6, residual=None):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance, at most 8192 channels).  weight / bias
    [C], float32 or of x's type, None = 1 / 0.  With `residual` (x's shape and type): s = x + residual is rounded to x's type and
    normalised, and (s, y) is returned -- the residual stream and its normalised copy in one pass, as scp_amd.dino.add_layernorm does
    for the frozen ViT.  Any strides; the results are contiguous."""
    return (_binding or _load()).layer_norm(x, weight, bias, eps, residual)


# ---- cross attention ---------------------------------------------------------------------------------------------------------------------
def cross_attention(q, k, v, scale=None, key_mask=None):
    """softmax(scale * q k^T) v per head: q [B, Nq, H, D] against an encoder's k, v [B, Nk, Hkv, D] of another length -> [B, Nq, H, D]
    (contiguous).  H a multiple of Hkv: query head h reads key / value head h // (H // Hkv).  D a multiple of 8, at most 128.  `scale`
    defaults to D ** -0.5.  `key_mask` (bool [B, Nk], True = attend): an image's padding; values stored at masked keys, NaN included,
    reach no result; a batch entry without a key gives zeros, and zero gradients (so does a query whose every score is -inf).  Any strides (slices of a fused qkv projection, an
    expanded batch); gradients for q, k and v.  float32 is multiplied as three exact bfloat16 parts: an infinity that is not masked may come
    out as NaN."""
    return (_binding or _load()).cross_attention(q, k, v, scale, key_mask)


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
        return (_binding or _load()).unpack8(self.codes, self.exps, dtype == torch.bfloat16)


def pack8(x):
    """x [..., C] -> Packed8: per 32 channels a power-of-two step with max|x| in [64, 128) steps, codes rounded to nearest (ties to
    even) and clamped to +-127.  1 + 1/32 bytes per value; not differentiable (it is what an autograd node keeps)."""
    codes, exps = (_binding or _load()).pack8(x)
    return Packed8(codes, exps, x.dtype)


def gelu8(x):
    """erf GELU of x [..., C] (the MLP's activation, vision_transformer_flexible.py:54-70).  The backward pass takes the slope at the
    8-bit checkpoint of x instead of keeping x: 1 + 1/32 bytes per value held between the passes.  The forward value is that of x itself,
    within 4e-7 |x| before its rounding (the error function of Abramowitz & Stegun 7.1.26, which is good to 1.5e-7 absolute)."""
    return (_binding or _load()).gelu8(x)


def weight_grad8(grad, packed, bias=True):
    """(gw [N, K], gb [N] or None) in float32 of a linear layer y = x w^T + b from grad = gy [..., N] and the 8-bit checkpoint of x
    [..., K]: gw = sum over rows gy[:, n] x8[:, k], gb = sum over rows gy.  N and K at most 2^20, N K at most 2^34; not differentiable."""
    if isinstance(packed, Packed8):
        return (_binding or _load()).weight_grad8(grad, packed.codes, packed.exps, bias)
    if isinstance(grad, torch.Tensor) and not grad.is_cuda:
        raise RuntimeError("weight_grad8: grad must be a CUDA tensor (no CPU fallback)")
    raise RuntimeError("weight_grad8: packed must be a Packed8 (scp_amd.vit_ops.pack8)")


def linear8(x, weight, bias=None):
    """x [..., K] @ weight [N, K]^T + bias, with x kept for the weight gradient in 8 bits (weight_grad8).  One type for all three.  The
    forward product and the input's gradient are plain library products at full precision; nothing else is saved.  A weight or bias that
    takes a gradient may have 2^20 rows, 2^20 columns and 2^34 entries."""
    return (_binding or _load()).linear8(x, weight, bias)
