"""Operators of the AR head's layers on torch tensors, for training through the frozen LLM (train_emg_llm.py:145-181),
for prompts and scored candidates, and for beam steps over long prefixes.

    attention(q, k, v)                  whole sequences, differentiable                  nsd_attn_fwd, nsd_attn_bwd
    shared_prefix_attention(q, ...)     one new token per hypothesis of a beam           nsd_attn_prefix, nsd_attn_step
    add_rms_norm(x, delta, w)           residual add + RMSNorm, differentiable           nsd_add_rmsnorm, nsd_add_rmsnorm_bwd

Device tensors in float32 or bfloat16; there is no CPU fall-back.  Kernels run on the current stream of the tensors'
device; scratch comes from torch's allocator, call by call.  Same arguments, same bits; the order of sums, and with it the
last bits, follows from all sizes of a call, the batch's among them.  Arguments are checked and the
autograd nodes live in csrc/nsd_torch.cpp: ValueError and TypeError for arguments, NsdError for what the library
refuses.  Derivatives are reverse-mode only: a tensor with a forward-mode tangent (torch.autograd.forward_ad) is refused.
A backward pass is captured into a graph from leaves made inside the capture (x.detach().requires_grad_()).
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
from typing import Optional, Sequence

import torch

from . import lib as _lib

_torch_side = None
_ENTRIES = ("nsd_strerror", "nsd_attn_fwd_workspace", "nsd_attn_fwd", "nsd_attn_bwd_workspace", "nsd_attn_bwd",
            "nsd_attn_prefix_workspace", "nsd_attn_prefix", "nsd_attn_step", "nsd_add_rmsnorm",
            "nsd_add_rmsnorm_bwd_workspace", "nsd_add_rmsnorm_bwd")


def load():
    """The torch side, bound to the loaded library; raises NsdError when either has not been built."""
    global _torch_side
    if _torch_side is None:
        L = _lib.load()
        path = _lib.PKG / "_nsd_torch.so"
        if not path.exists():
            raise _lib.NsdError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        loader = importlib.machinery.ExtensionFileLoader("_nsd_torch", os.fspath(path))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_nsd_torch", loader))
        loader.exec_module(module)
        module.bind({n: C.cast(getattr(L, n), C.c_void_p).value for n in _ENTRIES}, _lib.NsdError)
        _torch_side = module
    return _torch_side


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
              key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v over the visible keys, differentiable in q, k and v (once).

    q [Z, Lq, heads, hd]; k, v [Z, Lk, kv_heads, hd], heads a multiple of kv_heads (query head i reads kv head
    i // (heads // kv_heads)); hd a multiple of 8 up to 128; any strides.  causal: query i sees keys j <= i + Lk - Lq.
    key_mask [Z, Lk] bool (or uint8): keys that are False are seen by no query, whatever they hold.  A query that sees
    no key gives zeros and has no part in any gradient, whatever it and its row of the output's gradient hold.  scale > 0,
    default 1 / sqrt(hd).  Returns [Z, Lq, heads, hd].

    bfloat16: softmax and sums are float32; probabilities and their gradients are rounded to bfloat16 where they enter a
    product, in small launches to 16 bits (a relative error of 1.9e-3 of a result and up to 2.4e-3 of a gradient, where
    their own rounding makes 1.7e-3)."""
    return (_torch_side or load()).attention(q, k, v, causal, key_mask, scale)


def shared_prefix_attention(q: torch.Tensor, prefixes: Sequence, kgen: torch.Tensor, vgen: torch.Tensor,
                            anc: Optional[torch.Tensor], t: int, beam: int, *, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token per hypothesis over [every prefix of its groups ; its ancestors' generated positions
    0..t-1 ; its own position t], each prefix read once for all hypotheses that share it.

    q [M, heads, hd] (rotated), M = utterances x beam.  prefixes: (k, v) or (k, v, lens) for each level, k and v
    [groups, kv_heads, P, hd] with any strides and any P; groups divides M, hypothesis m belongs to group
    m // (M // groups) - 1 group is a prompt that all utterances share, M // beam groups are the utterances' contexts;
    lens int32 [groups]: positions at and after it are not read (default P).  kgen, vgen [> t, M, kv_heads, hd] slabs of
    the generated positions and anc uint8 [>= t, M] as nsd_rope_kv_append and nsd_ancestors write them (contiguous).
    heads / kv_heads in {1, 2, 3, 4, 8}, hd a power of two from 8 to 128.  No gradient.  Returns [M, heads, hd]."""
    return (_torch_side or load()).shared_prefix_attention(q, prefixes, kgen, vgen, anc, t, beam, scale)


def add_rms_norm(x: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-5):
    """(x_out, h): x_out = x + delta (x itself where delta is None), h = w * x_out * rsqrt(mean(x_out^2) + eps) over
    the last axis, both in the tensors' type, differentiable (once) in x, delta and w.  In bfloat16 the normed row is
    rounded before w is applied, and the product again, as LlamaRMSNorm does.  The rows' mean squares have to be inside
    float32.

    x, delta [..., hidden], w [hidden]; hidden a multiple of 4 (float32) or 8 (bfloat16)."""
    return (_torch_side or load()).add_rms_norm(x, delta, w, eps)
