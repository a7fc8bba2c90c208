"""Operators of the AR head's layers on torch tensors, for training through the frozen LLM (train_emg_llm.py:145-181),
for prompts and scored candidates, and for beam steps over long prefixes.

    attention(q, k, v)                  whole sequences, differentiable                  nsd_attn_fwd, nsd_attn_bwd
    shared_prefix_attention(q, ...)     one new token per hypothesis of a beam           nsd_attn_prefix, nsd_attn_step
    add_rms_norm(x, delta, w)           residual add + RMSNorm, differentiable           nsd_add_rmsnorm, nsd_add_rmsnorm_bwd

Device tensors in float32 or bfloat16; there is no CPU fall-back.  Kernels run on the current stream of the tensors'
device; scratch comes from torch's allocator, call by call.  Same arguments, same bits.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import lib as _lib

_DT = {torch.float32: 0, torch.bfloat16: 1}


def _same_device(name: str, first: torch.Tensor, *more) -> None:
    if not first.is_cuda:
        raise _lib.NsdError(f"{name} needs device tensors (there is no CPU fall-back)")
    for t in more:
        if t is not None and t.device != first.device:
            raise ValueError(f"{name}: tensors on {first.device} and {t.device}")


def _same_type(name: str, first: torch.Tensor, *more) -> int:
    if first.dtype not in _DT:
        raise TypeError(f"{name} takes float32 or bfloat16, not {first.dtype}")
    for t in more:
        if t is not None and t.dtype != first.dtype:
            raise TypeError(f"{name}: {first.dtype} and {t.dtype} together")
    return _DT[first.dtype]


def _stream(device: torch.device) -> int:
    # (the stream's handle alone: building a torch.cuda.Stream object costs more than the launch)
    return torch._C._cuda_getCurrentRawStream(device.index)


class _on:
    """The tensors' device as the current one, as torch.cuda.device does, but for nothing where it is that already."""

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.prev = torch._C._cuda_getDevice()
        if self.prev != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch._C._cuda_setDevice(self.prev)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it, with consecutive elements in its rows and everything else in steps of 16 bytes."""
    a, b, c, d = x.stride()
    n = x.shape
    piece = 16 // x.element_size()
    ok = d == 1 and x.data_ptr() % 16 == 0 and (a % piece == 0 or n[0] == 1) and (b % piece == 0 or n[1] == 1) and (
        c % piece == 0 or n[2] == 1)
    return x if ok else x.clone(memory_format=torch.contiguous_format)


_I64x3 = C.c_int64 * 3


def _strides(x: torch.Tensor, i: int, j: int, k: int):
    s, n = x.stride(), x.shape                                  # (the stride of an axis of one element says nothing)
    return _I64x3(s[i] if n[i] > 1 else 0, s[j] if n[j] > 1 else 0, s[k] if n[k] > 1 else 0)


def _scratch(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(x: Optional[torch.Tensor]) -> Optional[int]:
    return None if x is None else x.data_ptr()


# ---------------------------------------------------------------------- attention of whole sequences
def _seq(q, k, v, mask, causal, scale):
    p = _lib.SeqAttn()
    p.batch, p.len_q, p.heads, p.hd = q.shape
    p.len_k, p.kv_heads = k.shape[1], k.shape[2]
    p.dtype, p.causal, p.scale = _DT[q.dtype], int(causal), scale
    p.q_stride, p.k_stride, p.v_stride = _strides(q, 0, 1, 2), _strides(k, 0, 1, 2), _strides(v, 0, 1, 2)
    p.key_mask = _ptr(mask)
    return p


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, causal, scale):
        q, k, v = _rows(q.detach()), _rows(k.detach()), _rows(v.detach())
        Z, Lq, H, D = q.shape
        L = _lib.load()
        with _on(q.device):
            p = _seq(q, k, v, mask, causal, scale)
            out = torch.empty((Z, Lq, H, D), dtype=q.dtype, device=q.device)
            lse = rest = None
            if any(ctx.needs_input_grad):
                lse = torch.empty((Z, k.shape[2], Lq, H // k.shape[2]), dtype=torch.float32, device=q.device)
                rest = torch.empty((Z, Lq, H, D), dtype=torch.uint8, device=q.device) if p.dtype else None
            n = L.nsd_attn_fwd_workspace(p)
            ws = _scratch(n, q.device)
            _lib.check(L.nsd_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), p, out.data_ptr(), _ptr(lse),
                                      _ptr(rest), _ptr(ws), n, _stream(q.device)), "nsd_attn_fwd")
        if lse is not None:
            ctx.save_for_backward(q, k, v, mask, out, lse, rest)
            ctx.shape = p                                       # (the tensors it points at are kept with it)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, mask, out, lse, rest = ctx.saved_tensors
        L, p = _lib.load(), ctx.shape
        with _on(q.device):
            dout = dout.contiguous()
            if dout.data_ptr() % 16:
                dout = dout.clone()
            dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
            dv = torch.empty(k.shape, dtype=q.dtype, device=q.device)
            n = L.nsd_attn_bwd_workspace(p)
            ws = _scratch(n, q.device)
            _lib.check(L.nsd_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(rest),
                                      dout.data_ptr(), p, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), n,
                                      _stream(q.device)), "nsd_attn_bwd")
        return dq, dk, dv, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
              key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v over the visible keys, differentiable in q, k and v (once).

    q [Z, Lq, heads, hd]; k, v [Z, Lk, kv_heads, hd], heads a multiple of kv_heads (query head i reads kv head
    i // (heads // kv_heads)); hd a multiple of 8 up to 128; any strides.  causal: query i sees keys j <= i + Lk - Lq.
    key_mask [Z, Lk] bool (or uint8): keys that are False are seen by no query, whatever they hold.  A query that sees
    no key gives zeros, and no gradient.  scale > 0, default 1 / sqrt(hd).  Returns [Z, Lq, heads, hd]."""
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError("attention takes q [Z, Lq, heads, hd] and k, v [Z, Lk, kv_heads, hd]")
    Z, Lq, H, D = q.shape
    KVH = k.shape[2]
    if k.shape[0] != Z or k.shape[3] != D or KVH < 1 or H < 1 or H % KVH:
        raise ValueError(f"attention: q {tuple(q.shape)} does not go with k {tuple(k.shape)}")
    if D < 8 or D > 128 or D % 8:
        raise ValueError(f"attention: head dimension {D} is not a multiple of 8 up to 128")
    _same_device("attention", q, k, v, key_mask)
    _same_type("attention", q, k, v)
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or tuple(key_mask.shape) != (Z, k.shape[1]):
            raise ValueError("attention: key_mask is [Z, Lk] of bool or uint8")
        key_mask = key_mask.detach().contiguous().view(torch.uint8)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("attention: scale is a positive number")
    return _Attention.apply(q, k, v, key_mask, bool(causal), scale)


# ---------------------------------------------------------------------- a beam step over shared prefixes
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
    if q.dim() != 3 or kgen.dim() != 4 or vgen.shape != kgen.shape:
        raise ValueError("shared_prefix_attention takes q [M, heads, hd] and kgen, vgen [T, M, kv_heads, hd]")
    M, H, D = q.shape
    T, KVH, t, beam = kgen.shape[0], kgen.shape[2], int(t), int(beam)
    if kgen.shape[1] != M or kgen.shape[3] != D or KVH < 1 or H % KVH or H // KVH not in (1, 2, 3, 4, 8):
        raise ValueError(f"shared_prefix_attention: q {tuple(q.shape)} does not go with kgen {tuple(kgen.shape)}")
    if D not in (8, 16, 32, 64, 128):
        raise ValueError(f"shared_prefix_attention: head dimension {D} is not a power of two from 8 to 128")
    if not 1 <= beam <= _lib.MAX_BEAM or M % beam or not 0 <= t < T:
        raise ValueError("shared_prefix_attention: beam divides M and is at most 64, and 0 <= t < len(kgen)")
    levels = [tuple(p) for p in prefixes]
    _same_device("shared_prefix_attention", q, kgen, vgen, anc, *(x for p in levels for x in p))
    dt = _same_type("shared_prefix_attention", q, kgen, vgen, *(x for p in levels for x in p[:2]))
    for x in (kgen, vgen) if anc is None else (kgen, vgen, anc):
        if not x.is_contiguous():
            raise ValueError("shared_prefix_attention: the generated cache and its ancestor table are contiguous")
    if t > 0 and (anc is None or anc.dtype != torch.uint8 or anc.dim() != 2 or anc.shape[0] < t or anc.shape[1] != M):
        raise ValueError("shared_prefix_attention: anc is uint8 [>= t, M]")
    for p in levels:
        if len(p) not in (2, 3) or p[0].dim() != 4 or p[1].shape != p[0].shape:
            raise ValueError("shared_prefix_attention: a prefix is (k, v) or (k, v, lens), k and v [groups, kv_heads, P, hd]")
        n = p[0].shape[0]
        if n < 1 or M % n or p[0].shape[1] != KVH or p[0].shape[3] != D:
            raise ValueError(f"shared_prefix_attention: a prefix {tuple(p[0].shape)} does not go with q {tuple(q.shape)}")
        if len(p) == 3 and (p[2].dtype != torch.int32 or tuple(p[2].shape) != (n,)):
            raise ValueError("shared_prefix_attention: lens is int32 [groups]")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, kgen, vgen, *(x for p in levels for x in p[:2]))):
        raise ValueError("shared_prefix_attention has no gradient: call it under torch.no_grad()")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("shared_prefix_attention: scale is a positive number")
    L, dev = _lib.load(), q.device
    with _on(dev):
        st = _stream(dev)
        q = q if q.is_contiguous() and q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
        out = torch.empty_like(q)
        state = None
        for i, p in enumerate(levels):
            k, v = _rows(p[0]), _rows(p[1])
            n = k.shape[0]
            if state is None:
                state = torch.empty(M * H * (D + 2), dtype=torch.float32, device=dev)
                po, pm, pl = (state[a * M * H:].data_ptr() for a in (0, D, D + 1))
            s = _lib.SeqAttn()
            s.batch, s.len_q, s.len_k, s.heads, s.kv_heads, s.hd, s.dtype = n, M // n, k.shape[2], H, KVH, D, dt
            s.scale = scale
            s.q_stride = _I64x3(M // n * H * D, H * D, D)
            s.k_stride, s.v_stride = _strides(k, 0, 2, 1), _strides(v, 0, 2, 1)
            lens = p[2].contiguous() if len(p) == 3 else None
            s.key_len = _ptr(lens)
            nb = L.nsd_attn_prefix_workspace(s)
            ws = _scratch(nb, dev)
            _lib.check(L.nsd_attn_prefix(q.data_ptr(), k.data_ptr(), v.data_ptr(), s, int(i > 0), po, pm, pl,
                                         _ptr(ws), nb, st), "nsd_attn_prefix")
        part = (po, pm, pl) if state is not None else (None, None, None)
        _lib.check(L.nsd_attn_step(q.data_ptr(), None, None, kgen.data_ptr(), vgen.data_ptr(), _ptr(anc), out.data_ptr(),
                                   M // beam, beam, H, KVH, D, 0, t, scale, dt, *part, st), "nsd_attn_step")
    return out


# ---------------------------------------------------------------------- residual add + RMSNorm
class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, w, eps):
        hidden = x.shape[-1]
        ctx.set_materialize_grads(False)
        xc, wc = _flat(x.detach()), _flat(w.detach())
        dc = None if delta is None else _flat(delta.detach())
        L = _lib.load()
        with _on(x.device):
            h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            x_out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if dc is not None else None
            _lib.check(L.nsd_add_rmsnorm(xc.data_ptr(), _ptr(dc), wc.data_ptr(), eps, x.numel() // hidden, hidden,
                                         _DT[x.dtype], _ptr(x_out), h.data_ptr(), _stream(x.device)), "nsd_add_rmsnorm")
        ctx.save_for_backward(x_out if x_out is not None else xc, wc)
        ctx.eps, ctx.has_delta = eps, dc is not None
        return (x_out if x_out is not None else x.view_as(x)), h

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_out, dh):
        x_out, w = ctx.saved_tensors
        hidden, rows = x_out.shape[-1], x_out.numel() // x_out.shape[-1]
        want_x = ctx.needs_input_grad[0] or (ctx.has_delta and ctx.needs_input_grad[1])
        want_w = ctx.needs_input_grad[2]
        if dh is None:                                          # h is not used: the sum's gradient passes through
            dx, dw = dx_out, torch.zeros_like(w) if want_w else None
        else:
            L = _lib.load()
            with _on(x_out.device):
                dh = _flat(dh)
                go = None if dx_out is None else _flat(dx_out)
                dx = torch.empty(x_out.shape, dtype=x_out.dtype, device=x_out.device)
                dw = torch.empty_like(w) if want_w else None
                n = L.nsd_add_rmsnorm_bwd_workspace(rows, hidden) if want_w else 0
                ws = _scratch(n, x_out.device)
                _lib.check(L.nsd_add_rmsnorm_bwd(x_out.data_ptr(), w.data_ptr(), dh.data_ptr(), _ptr(go), ctx.eps, rows,
                                                 hidden, _DT[x_out.dtype], dx.data_ptr(), _ptr(dw), _ptr(ws), n,
                                                 _stream(x_out.device)), "nsd_add_rmsnorm_bwd")
        return (dx if want_x and ctx.needs_input_grad[0] else None,
                dx if ctx.has_delta and ctx.needs_input_grad[1] else None, dw, None)


def _flat(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def add_rms_norm(x: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor, eps: float = 1e-5):
    """(x_out, h): x_out = x + delta (x itself where delta is None), h = w * x_out * rsqrt(mean(x_out^2) + eps) over
    the last axis, both in the tensors' type, differentiable (once) in x, delta and w.

    x, delta [..., hidden], w [hidden]; hidden a multiple of 4 (float32) or 8 (bfloat16)."""
    if x.dim() < 1 or tuple(w.shape) != (x.shape[-1],) or (delta is not None and delta.shape != x.shape):
        raise ValueError("add_rms_norm takes x and delta [..., hidden] and w [hidden]")
    _same_device("add_rms_norm", x, delta, w)
    dt = _same_type("add_rms_norm", x, delta, w)
    if x.numel() // max(1, x.shape[-1]) >= 2 ** 31:
        raise ValueError("add_rms_norm: at most 2^31 - 1 rows")
    if x.shape[-1] < 1 or x.shape[-1] % (8 if dt else 4):
        raise ValueError(f"add_rms_norm: hidden = {x.shape[-1]} is not a multiple of {8 if dt else 4}")
    return _AddRmsNorm.apply(x, delta, w, float(eps))
