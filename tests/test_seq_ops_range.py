"""The sequence operators over the range that they are documented for."""
import math
import re
from pathlib import Path

import pytest
import torch

from tests import seq_reference as R
from tests.test_seq_ops import _gen, _mask

BF, FP = torch.bfloat16, torch.float32
CUS = 256


# ---------------------------------------------------------------------- gradients of large and small rows of a norm
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,hidden", [(FP, 5, 100), (BF, 9, 1000), (FP, 3, 8196), (BF, 2, 16392)])
@pytest.mark.parametrize("size,eps", [(1e13, 1e-5), (1e15, 1e-5), (3e16, 1e-5), (1e-15, 1e-36)])
def test_norm_gradients_of_large_and_small_rows(dtype, rows, hidden, size, eps):
    """Rows whose rsqrt is far from 1, its cube outside fp32: the squares' sum and every factor of the definition are inside."""
    from silent_speech_amd import ops
    g = _gen(hidden + rows)
    x, dh = (torch.randn(rows, hidden, generator=g) * size).to(dtype), torch.randn(rows, hidden, generator=g).to(dtype)
    dh = (dh.float() + 2.0 * torch.sign(x.float())).to(dtype)  # a gradient along the row: the projection counts
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(dtype)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    x_out, h = ops.add_rms_norm(xd, None, wd, eps)
    want = R.add_rms_norm(x, None, w, eps, None, dh)
    R.within(h, want["h"], "h")
    dx, dw = torch.autograd.grad(h, (xd, wd), dh.cuda())
    R.within(dx, want["dx"], "dx")
    R.within(dw, want["dw"], "dw")


# ---------------------------------------------------------------------- derivatives that there are not
def _dual_calls(dev, grad):
    """(name, call with its arguments of which one is a dual tensor)"""
    from silent_speech_amd import ops
    z = lambda *s: torch.ones(*s, device=dev)                   # noqa: E731
    dual = lambda x: torch.autograd.forward_ad.make_dual(x.requires_grad_(grad), torch.ones_like(x))   # noqa: E731
    calls = []
    for i in range(3):
        def attention(i=i):
            a = [z(1, 4, h, 16) for h in (4, 2, 2)]
            a[i] = dual(a[i])
            return ops.attention(*a)
        def norm(i=i):                                           # noqa: E306
            a = [z(3, 16), z(3, 16), z(16)]
            a[i] = dual(a[i])
            return ops.add_rms_norm(*a)
        calls += [(f"attention {i}", attention), (f"add_rms_norm {i}", norm)]
    for i in range(5):
        def beam(i=i):
            a = [z(4, 4, 16), z(1, 2, 5, 16), z(1, 2, 5, 16), z(1, 4, 2, 16), z(1, 4, 2, 16)]
            a[i] = dual(a[i])
            with torch.no_grad():
                return ops.shared_prefix_attention(a[0], [(a[1], a[2])], a[3], a[4], None, 0, 2)
        calls.append((f"shared_prefix_attention {i}", beam))
    return calls


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    with torch.autograd.forward_ad.dual_level():
        for name, call in _dual_calls("cpu", grad):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused_on_the_device(grad):
    from silent_speech_amd import ops
    with torch.autograd.forward_ad.dual_level():
        for name, call in _dual_calls("cuda", grad):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        # a backward pass of a dual gradient: a derivative of the gradient
        q, k = (torch.randn(1, 4, 2, 16, device="cuda").requires_grad_() for _ in range(2))
        out = ops.attention(q, k, k)
        with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
            torch.autograd.grad(out, q, torch.autograd.forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
        x, w = torch.randn(3, 32, device="cuda").requires_grad_(), torch.ones(32, device="cuda")
        y = ops.add_rms_norm(x, None, w)
        for dual in range(2):
            one = torch.ones_like(x)
            go = [one, one]
            go[dual] = torch.autograd.forward_ad.make_dual(one, torch.ones_like(one))
            with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
                torch.autograd.grad(y, x, go, retain_graph=True)
    q = torch.randn(1, 4, 2, 16, device="cuda")                 # outside of a level nothing is dual
    assert ops.attention(q, q, q).shape == q.shape


@pytest.mark.gpu
def test_gradients_of_gradients_raise_whatever_they_are_taken_for():
    """Also where torch may leave out what a result does not depend on (allow_unused, its functional Hessian): a gradient is
    not independent of the arguments that it was computed from, nor of the gradient that came in."""
    from silent_speech_amd import ops
    g = _gen(4)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda().requires_grad_()   # noqa: E731
    def strided(x):                                                         # noqa: E306
        return torch.stack((x, x), -1)[..., 0]                             # (copied inside)
    for form in (lambda x: x, strided):
        q, k, v, do = rnd(1, 9, 4, 32), rnd(1, 9, 2, 32), rnd(1, 9, 2, 32), rnd(1, 9, 4, 32)
        out = ops.attention(*(form(x) for x in (q, k, v)))
        grads = torch.autograd.grad(out, (q, k, v), do, create_graph=True)
        for d in grads:
            for x in (q, k, v, do):
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(d.sum(), x, retain_graph=True, allow_unused=True)
        x, delta, w, go, dh = rnd(3, 32), rnd(3, 32), rnd(32), rnd(3, 32), rnd(3, 32)
        x_out, h = ops.add_rms_norm(form(x), form(delta), w)
        grads = torch.autograd.grad((x_out, h), (x, delta, w), (go, dh), create_graph=True)
        for d in grads:
            for y in (x, delta, w, go, dh):
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(d.sum(), y, retain_graph=True, allow_unused=True)
        (dx,) = torch.autograd.grad(ops.add_rms_norm(form(x), form(delta), w)[0], x, go, create_graph=True)
        (one,) = torch.autograd.grad(dx.sum(), go)                          # the sum's own: what came in
        assert torch.equal(dx, go) and torch.equal(one, torch.ones_like(go))
    w = torch.ones(32, device="cuda")
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.functional.hessian(lambda x: ops.add_rms_norm(x, None, w)[1].sum(), torch.randn(2, 32, device="cuda"))


# ---------------------------------------------------------------------- shapes that only the gradients refuse
def test_attention_refuses_before_the_forward_pass_what_its_gradients_refuse():
    from silent_speech_amd import lib, ops
    one = lambda *s: torch.zeros(1, dtype=BF).expand(*s)       # noqa: E731
    for lq in (1, 0):
        q, k = one(1 << 23, lq, 1, 8), one(1 << 23, 65, 1, 8).requires_grad_()
        with pytest.raises(lib.NsdError, match="nsd_attn_bwd"):
            ops.attention(q, k, k.detach())
        with pytest.raises(lib.NsdError, match="device"):       # without gradients the shape is fine
            ops.attention(q, k.detach(), k.detach())
    q, k = one(1 << 23, 1, 1, 8), one(1 << 23, 64, 1, 8).requires_grad_()
    with pytest.raises(lib.NsdError, match="device"):
        ops.attention(q, k, k.detach())


# ---------------------------------------------------------------------- every form of the backward kernels
def _plans(Z, KVH, R_, Lk):
    """Waves along the rows (dQ) and along the keys (dK, dV) of a workgroup, as bwd_q_plan and bwd_kv_plan choose them (the
    kernels' names in a trace of these shapes carry the same numbers)."""
    pairs, up = Z * KVH, lambda a, b: -(-a // b)                # noqa: E731
    q = 4 if R_ > 64 and pairs * up(R_, 128) >= CUS else 2 if R_ > 32 and pairs * up(R_, 64) >= CUS else 1
    return q, 2 if Lk > 32 and pairs * up(Lk, 64) >= CUS // 2 else 1


FORMS = [  # Z, Lq, Lk, kv heads, G, causal, mask, plans of dQ and of dK, dV
    (16, 67, 67, 8, 2, True, None, (4, 2)), (16, 67, 150, 8, 2, True, "random", (4, 2)), (43, 45, 71, 3, 3, False, "pad", (4, 2)),
    (16, 131, 67, 8, 1, True, "empty", (4, 2)), (86, 300, 300, 1, 1, True, "pad", (4, 2)), (32, 23, 45, 8, 2, True, "random", (2, 2)),
    (32, 47, 33, 8, 1, True, None, (2, 2)), (43, 11, 129, 6, 5, False, "empty", (2, 2)), (32, 40, 31, 8, 1, False, "pad", (2, 1)),
    # more pairs of an XCD than it works on together
    (64, 70, 140, 8, 4, True, "pad", (4, 2)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (BF, 72), (FP, 128), (FP, 64), (FP, 40)])
@pytest.mark.parametrize("Z,Lq,Lk,KVH,G,causal,kind,plans", FORMS)
def test_attention_gradients_in_every_form(dtype, D, Z, Lq, Lk, KVH, G, causal, kind, plans):
    from silent_speech_amd import ops
    assert _plans(Z, KVH, Lq * G, Lk) == plans
    g = _gen(Lq + 3 * Lk + D)
    q, k, v = (torch.randn(Z, n, h, D, generator=g).to(dtype) for n, h in ((Lq, KVH * G), (Lk, KVH), (Lk, KVH)))
    do = torch.randn(Z, Lq, KVH * G, D, generator=g).to(dtype)
    mask = _mask(kind, Z, Lk, g)
    if mask is not None:
        k = k.masked_fill(~mask[:, :, None, None], float("nan"))
        v = v.masked_fill(~mask[:, :, None, None], float("inf"))
    scale = 1.3 / math.sqrt(D)
    want = R.attention(q, k, v, causal, mask, scale, do)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    out = ops.attention(*leaves, causal=causal, key_mask=None if mask is None else mask.cuda(), scale=scale)
    R.within(out, want["out"], "out")
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do.cuda())):
        R.within(x, want[name], name)


# ---------------------------------------------------------------------- rows that see no key
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Z,L,KVH,G,D,pad", [
    (2, 50, 1, 2, 64, "left"), (2, 150, 2, 3, 128, "left"), (16, 67, 8, 2, 64, "left"), (16, 67, 8, 2, 128, "left"),
    (32, 23, 8, 2, 128, "left"), (2, 90, 1, 2, 64, "short"), (3, 40, 2, 1, 128, "none"), (1, 600, 1, 8, 64, "left")])
def test_what_rows_without_keys_hold_takes_no_part(dtype, Z, L, KVH, G, D, pad):
    """A batch padded on the left whose padding holds NaN everywhere (or fewer keys than queries under a causal mask, or a
    sequence that sees nothing): such a row gives zeros and has no part in any gradient, whatever its query and its
    gradient hold."""
    from silent_speech_amd import ops
    g = _gen(L + D)
    Lk = L // 2 if pad == "short" else L
    q, k, v = (torch.randn(Z, n, h, D, generator=g).to(dtype) for n, h in ((L, KVH * G), (Lk, KVH), (Lk, KVH)))
    do = torch.randn(Z, L, KVH * G, D, generator=g).to(dtype)
    mask = torch.ones(Z, Lk, dtype=torch.bool)
    rows = torch.zeros(Z, L, dtype=torch.bool)                  # that see no key
    if pad == "short":
        rows[:, :L - Lk] = True
    for z in range(Z):
        n = (5 * z + 3) % L if pad == "left" else L if pad == "none" and z == 1 else 0
        if n:
            mask[z, :n] = False
            rows[z, :n] = True
    at = rows[:, :, None, None]
    want = R.attention(q.masked_fill(at, 0.0), k, v, True, mask, 1 / math.sqrt(D), do.masked_fill(at, 0.0))
    k, v = (x.masked_fill(~mask[:, :, None, None], float("nan")) for x in (k, v))
    leaves = [x.cuda().requires_grad_() for x in (q.masked_fill(at, float("nan")), k, v)]
    out = ops.attention(*leaves, key_mask=None if pad == "short" else mask.cuda())
    R.within(out, want["out"], "out")
    grads = torch.autograd.grad(out, leaves, do.masked_fill(at, float("inf")).cuda())
    for name, x in zip(("dq", "dk", "dv"), grads):
        R.within(x, want[name], name)
    assert not bool(grads[0][rows.cuda()].any())


# ---------------------------------------------------------------------- signs that are not in memory yet
@pytest.mark.gpu
def test_views_with_a_sign_of_their_own():
    from silent_speech_amd import ops
    g = _gen(6)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()        # noqa: E731
    neg = torch._neg_view                                       # what x.conj().imag is, here with rows in steps of one
    assert neg(rnd(2)).is_neg() and rnd(2).to(torch.complex64).conj().imag.is_neg()
    x = [rnd(1, 9, h, 32) for h in (4, 2, 2)]
    do = rnd(1, 9, 4, 32)
    for i in range(4):
        got, want = ([f(y) if j == i else y for j, y in enumerate((*x, do))] for f in (neg, torch.neg))
        a, b = ([y.detach().requires_grad_() for y in z[:3]] for z in (got, want))
        oa, ob = ops.attention(*a), ops.attention(*b)
        assert torch.equal(oa, ob) and torch.equal(ops.attention(*got[:3]), ob)
        for da, db in zip(torch.autograd.grad(oa, a, got[3]), torch.autograd.grad(ob, b, want[3])):
            assert torch.equal(da, db)
    r = [rnd(3, 32), rnd(3, 32), rnd(32)]
    for i in range(3):
        got, want = (ops.add_rms_norm(*(f(y) if j == i else y for j, y in enumerate(r))) for f in (neg, torch.neg))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, k, v, kg = rnd(4, 4, 32), rnd(1, 2, 5, 32), rnd(1, 2, 5, 32), rnd(1, 4, 2, 32)
    for i in range(3):
        got, want = ([f(y) if j == i else y for j, y in enumerate((q, k, v))] for f in (neg, torch.neg))
        a, b = (ops.shared_prefix_attention(z[0], [tuple(z[1:])], kg, kg, None, 0, 2) for z in (got, want))
        assert torch.equal(a, b)
    for bad in ((neg(kg), kg), (kg, neg(kg))):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(q, [(k, v)], *bad, None, 0, 2)


# ---------------------------------------------------------------------- a shared prompt joined to many sequences
@pytest.mark.gpu
def test_sequences_that_share_a_prompt_are_joined_a_few_at_a_time():
    """Teacher-forced rows and contexts behind a prompt: the copies of the prompt's keys and values stay within
    JOIN_BYTES (and what one sequence needs), and the rows are the same bits whatever that is."""
    from tests.test_ar_head import _small_dims, _small_head
    g = _gen(21)
    dims = _small_dims(layers=1, heads=8, kv_heads=8, head_dim=64)
    seq, lens = torch.randint(0, 37, (9, 7), generator=g), torch.full((9,), 7)
    prefix, ctx = torch.randn(6, dims.hidden, generator=g), torch.randn(5, 9, dims.hidden, generator=g)
    got = []
    for room in (None, 1, 100_000):                             # all at once, one by one, four by four (22 positions of 4 KiB)
        head = _small_head("HipLlamaStep", dims, "cuda")
        head.JOIN_BYTES = room or head.JOIN_BYTES
        head.encode_context(ctx, 2, 3, prefix=prefix)
        got.append((head.teacher_logits(seq, lens), head.teacher_logits(seq, lens, torch.randint(0, 5, (9,), generator=_gen(1)))))
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(other, got[0]))
    assert not torch.equal(*got[0])
    # 64 sequences behind 8192 positions: 1 GiB of copies in bf16
    head = _small_head("HipLlamaStep", dims, "cuda", torch.bfloat16)
    head.JOIN_BYTES = 64 << 20
    seq, lens = torch.randint(0, 37, (64, 5), generator=g), torch.full((64,), 5)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    head.encode_context(torch.randn(64, 2, dims.hidden, generator=g), 2, 3, prefix=torch.randn(8192, dims.hidden, generator=g))
    head.teacher_logits(seq, lens)
    assert torch.cuda.max_memory_allocated() - before < 512 << 20


# ---------------------------------------------------------------------- assembly leaves m0 alone
def test_assembly_restores_m0():
    """m0 is the compiler's (it keeps the index of a register array there, for instance, and cannot be told that a statement
    overwrites it): a statement that needs it puts back what it found."""
    seen = 0
    for path in sorted((Path(__file__).parent.parent / "silent-speech_amd" / "csrc").iterdir()):
        for text in re.findall(r'\basm volatile\(((?:\s*"[^"]*")+)', path.read_text()):
            steps = [x.strip() for x in text.replace('"', "").replace("\\t", "").split("\\n")]
            if any(re.match(r"s_mov_b32 m0,", x) for x in steps):
                seen += 1
                saved = re.fullmatch(r"s_mov_b32 (%\d), m0", steps[0])
                assert saved and steps[-1] == f"s_mov_b32 m0, {saved[1]}", (path.name, text)
    assert seen
