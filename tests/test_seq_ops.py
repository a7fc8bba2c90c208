"""Attention of whole sequences with its gradients, a beam step over shared prefixes, and the gradients of
add + RMSNorm, against plain 64-bit forms within bounds derived there (seq_reference)."""
import ctypes as C
import math

import pytest
import torch

from tests import seq_reference as R

BF, FP = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _mask(kind, Z, Lk, g):
    if kind is None:
        return None
    if kind == "random":
        return torch.rand(Z, Lk, generator=g) < 0.6
    m = torch.arange(Lk)[None].expand(Z, Lk) < torch.tensor([(3 * i + 2) * Lk // (3 * Z + 1) for i in range(Z)])[:, None]
    m = m.clone()
    if kind == "empty":
        m[0] = False                                            # one sequence of the batch sees nothing at all
    return m


CASES = [  # dtype, Z, Lq, Lk, kv heads, G, hd, causal, mask
    (FP, 1, 1, 1, 1, 1, 8, True, None), (BF, 1, 1, 1, 1, 1, 64, True, None), (BF, 2, 5, 5, 2, 2, 64, True, None),
    (BF, 1, 31, 31, 1, 1, 128, True, None), (BF, 1, 33, 33, 1, 3, 128, True, None), (BF, 2, 64, 64, 2, 1, 64, True, "pad"),
    (BF, 1, 129, 129, 2, 3, 128, True, "random"), (BF, 3, 100, 100, 1, 8, 64, True, "empty"),
    (BF, 1, 300, 300, 1, 2, 96, True, None), (BF, 1, 65, 200, 2, 3, 128, True, "random"),
    (BF, 2, 1, 700, 2, 4, 128, True, None), (BF, 1, 7, 1000, 1, 3, 64, False, "pad"), (BF, 1, 40, 513, 1, 1, 128, True, "random"),
    (BF, 2, 90, 40, 1, 2, 64, True, None), (BF, 1, 257, 127, 2, 1, 128, False, None), (BF, 1, 20, 64, 1, 5, 24, False, None),
    (BF, 1, 600, 600, 2, 3, 128, True, "random"),
    # walks split over workgroups: keys of the forward pass and of dQ, rows of dK and dV
    (BF, 1, 3, 2100, 2, 2, 128, True, "random"), (BF, 1, 50, 3000, 1, 1, 64, False, "pad"), (BF, 1, 600, 600, 1, 8, 64, True, "pad"),
    (BF, 1, 400, 700, 1, 12, 128, True, "random"), (BF, 2, 9, 40, 1, 32, 64, True, None),
    (FP, 2, 37, 37, 2, 2, 16, True, "pad"), (FP, 1, 130, 130, 1, 3, 64, True, None), (FP, 1, 70, 150, 2, 2, 128, True, "random"),
    (FP, 3, 50, 50, 1, 3, 80, True, "empty"), (FP, 1, 3, 900, 2, 2, 128, False, None), (FP, 1, 33, 700, 1, 2, 64, True, "pad"),
    (FP, 1, 20, 300, 1, 3, 128, False, "random"), (FP, 2, 80, 33, 1, 4, 40, True, None), (FP, 1, 260, 260, 1, 1, 128, False, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,Z,Lq,Lk,KVH,G,D,causal,kind", CASES)
def test_attention_and_its_gradients(dtype, Z, Lq, Lk, KVH, G, D, causal, kind):
    from silent_speech_amd import ops
    g = _gen(Lq * 7 + Lk + D)
    q, k, v = (torch.randn(Z, n, h, D, generator=g).to(dtype) for n, h in ((Lq, KVH * G), (Lk, KVH), (Lk, KVH)))
    do = torch.randn(Z, Lq, KVH * G, D, generator=g).to(dtype)
    mask = _mask(kind, Z, Lk, g)
    if mask is not None:                                        # what lies at masked keys takes no part
        k = k.masked_fill(~mask[:, :, None, None], float("nan"))
        v = v.masked_fill(~mask[:, :, None, None], float("inf"))
    scale = 1.3 / math.sqrt(D)
    want = R.attention(q, k, v, causal, mask, scale, do)
    qd, kd, vd = (x.cuda().requires_grad_() for x in (q, k, v))
    md = None if mask is None else mask.cuda()
    out = ops.attention(qd, kd, vd, causal=causal, key_mask=md, scale=scale)
    R.within(out, want["out"], "out")
    grads = torch.autograd.grad(out, (qd, kd, vd), do.cuda())
    for name, x in zip(("dq", "dk", "dv"), grads):
        R.within(x, want[name], name)
    with torch.no_grad():                                       # without gradients: the same bits
        assert torch.equal(out, ops.attention(qd, kd, vd, causal=causal, key_mask=md, scale=scale))


@pytest.mark.gpu
def test_attention_takes_views():
    """One projection's split, heads before positions, a batch that is one sequence expanded, rows that start off a
    16-byte boundary, keys in an axis that runs with a stride; gradients arrive at the tensors behind the views."""
    from silent_speech_amd import ops
    g = _gen(3)
    Z, L, KVH, G, D = 2, 70, 2, 3, 64
    H = KVH * G
    qkv = torch.randn(Z, L, (H + 2 * KVH) * D, generator=g).to(BF).cuda().requires_grad_()
    split = lambda x: [y.unflatten(-1, (-1, D)) for y in x.split([H * D, KVH * D, KVH * D], -1)]     # noqa: E731
    do = torch.randn(Z, L, H, D, generator=g).to(BF).cuda()
    q, k, v = split(qkv)
    out = ops.attention(q, k, v)
    (dqkv,) = torch.autograd.grad(out, qkv, do)
    want = R.attention(q, k, v, True, None, 1 / math.sqrt(D), do)
    R.within(out, want["out"], "out")
    for name, x in zip(("dq", "dk", "dv"), split(dqkv)):
        R.within(x, want[name], name)
    base = [x.detach().clone() for x in (q, k, v)]
    def heads_first(x): return x.transpose(1, 2).contiguous().transpose(1, 2)                        # noqa: E704
    def shifted(x):                                                                                    # noqa: E306
        y = torch.zeros(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
        return y.copy_(x)
    def strided(x):                                                                                    # noqa: E306
        y = torch.zeros(*x.shape, 2, dtype=x.dtype, device=x.device)
        y[..., 0] = x
        return y[..., 0]
    for form in (heads_first, shifted, strided):
        assert torch.equal(ops.attention(*(form(x) for x in base)), out), form.__name__
    one = [x[:1].expand(3, -1, -1, -1).requires_grad_(False) for x in base]
    many = ops.attention(*one)
    assert all(torch.equal(many[i], out[0]) for i in range(3))
    leaves = [x[:1].clone().requires_grad_() for x in base]
    o = ops.attention(*(x.expand(3, -1, -1, -1) for x in leaves))
    grads = torch.autograd.grad(o, leaves, do[:1].expand(3, -1, -1, -1))                             # summed over the copies
    want1 = R.attention(*(x[:1] for x in base), True, None, 1 / math.sqrt(D), do[:1])
    for name, x in zip(("dq", "dk", "dv"), grads):
        value, bound = want1[name]
        R.within(x, (3 * value, 3 * bound + 4 * R.half_step(BF) * 3 * value.abs()), name)


@pytest.mark.gpu
def test_attention_gradient_against_differences():
    """Directional derivatives of the 64-bit form by central differences (step 1e-5: off by about 1e-9)."""
    from silent_speech_amd import ops
    g = _gen(11)
    Z, L, KVH, G, D = 1, 41, 2, 2, 32
    x = [torch.randn(Z, L, h, D, generator=g) for h in (KVH * G, KVH, KVH)]
    d = [torch.randn(*y.shape, generator=g) for y in x]
    do = torch.randn(Z, L, KVH * G, D, generator=g)
    mask = torch.rand(Z, L, generator=g) < 0.7
    scale = 1 / math.sqrt(D)

    def loss(e):
        y = [a.double() + e * b.double() for a, b in zip(x, d)]
        s = torch.einsum("zihd,zjhd->zhij", y[0], y[1].repeat_interleave(G, 2)) * scale
        vis = torch.ones(L, L, dtype=torch.bool).tril() & mask[:, None, None]
        p = torch.softmax(s.masked_fill(~vis, -math.inf), -1).masked_fill(~vis.any(-1, keepdim=True), 0.0)
        return float((torch.einsum("zhij,zjhd->zihd", p, y[2].repeat_interleave(G, 2)) * do.double()).sum())

    step = 1e-5
    diff = (loss(step) - loss(-step)) / (2 * step)
    leaves = [y.cuda().requires_grad_() for y in x]
    out = ops.attention(*leaves, key_mask=mask.cuda(), scale=scale)
    grads = torch.autograd.grad(out, leaves, do.cuda())
    got = sum(float((a.cpu().double() * b.double()).sum()) for a, b in zip(grads, d))
    want = R.attention(*x, True, mask, scale, do)
    slack = sum(float((want[n][1] * b.double().abs()).sum()) for n, b in zip(("dq", "dk", "dv"), d))
    assert abs(got - diff) <= slack + 1e-6 * max(1.0, abs(diff))


@pytest.mark.gpu
def test_attention_of_large_scores_and_no_sequences():
    from silent_speech_amd import ops
    g = _gen(5)
    q, k, v = (torch.randn(1, 70, 2, 64, generator=g) * s for s in (30.0, 30.0, 1.0))
    for dtype in (BF, FP):                                      # scores of some thousands: a row is nearly one key
        x = [y.to(dtype) for y in (q, k, v)]
        want = R.attention(*x, True, None, 1.0, torch.ones_like(x[0]))
        xd = [y.cuda().requires_grad_() for y in x]
        out = ops.attention(*xd, scale=1.0)
        R.within(out, want["out"], "out")
        for name, y in zip(("dq", "dk", "dv"), torch.autograd.grad(out, xd, torch.ones_like(out))):
            R.within(y, want[name], name)
    for Z, Lq, Lk in ((0, 4, 4), (2, 0, 5), (2, 5, 0), (1, 0, 0)):
        q, k, v = (torch.randn(Z, n, h, 64, device="cuda", dtype=BF).requires_grad_() for n, h in ((Lq, 4), (Lk, 2), (Lk, 2)))
        out = ops.attention(q, k, v)
        assert out.shape == (Z, Lq, 4, 64) and not bool(out.any())
        for x, d in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert d.shape == x.shape and not bool(d.any())


def _beam_case(dtype, N, B, KVH, G, D, levels, t, seed):
    """levels: (groups, P, lens or None) each."""
    g = _gen(seed)
    M = N * B
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)     # noqa: E731
    q, kgen, vgen = rnd(M, KVH * G, D), rnd(t + 2, M, KVH, D), rnd(t + 2, M, KVH, D)
    anc = torch.randint(0, B, (t + 1, M), generator=g).to(torch.uint8)
    ps = []
    for groups, P, lens in levels:
        k, v = rnd(groups, KVH, P, D), rnd(groups, KVH, P, D)
        if lens is not None:
            for i, n in enumerate(lens):
                k[i, :, max(n, 0):] = float("nan")              # behind a prefix: not read
                v[i, :, max(n, 0):] = float("inf")
            ps.append((k, v, torch.tensor(lens, dtype=torch.int32)))
        else:
            ps.append((k, v))
    return q, ps, kgen, vgen, anc


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,B,KVH,G,D,levels,t", [
    (BF, 1, 1, 1, 1, 64, [(1, 1, None)], 0), (BF, 1, 4, 2, 2, 64, [(1, 100, None)], 3), (BF, 2, 5, 2, 3, 128, [(1, 65, None)], 7),
    (BF, 3, 7, 1, 3, 128, [(1, 300, None), (3, 40, None)], 5), (BF, 4, 16, 2, 3, 128, [(1, 1500, None)], 2),
    (BF, 5, 3, 1, 8, 32, [(5, 90, [90, 0, 1, 64, 33])], 4), (BF, 2, 16, 1, 4, 128, [(2, 700, [700, 129])], 1),
    (BF, 3, 2, 1, 1, 8, [(3, 20, [0, 0, 0])], 0), (BF, 2, 3, 1, 3, 64, [(2, 90, [-3, 95])], 1), (BF, 2, 8, 1, 2, 64, [(1, 0, None), (2, 77, None)], 2), (BF, 2, 3, 1, 2, 64, [], 2),
    (BF, 6, 4, 1, 3, 64, [(1, 128, None), (2, 64, [64, 5]), (6, 33, None)], 3), (BF, 40, 4, 1, 1, 64, [(1, 70, None)], 2),
    (FP, 1, 4, 2, 2, 64, [(1, 100, None)], 3), (FP, 5, 7, 1, 2, 64, [(5, 150, [150, 3, 0, 149, 70])], 6),
    (FP, 2, 9, 1, 3, 128, [(1, 400, None), (2, 33, [33, 1])], 2), (FP, 2, 12, 1, 2, 128, [(1, 90, None)], 0), (FP, 12, 8, 1, 2, 16, [(1, 40, None)], 1),
])
def test_beam_step_over_shared_prefixes(dtype, N, B, KVH, G, D, levels, t):
    from silent_speech_amd import ops
    q, ps, kgen, vgen, anc = _beam_case(dtype, N, B, KVH, G, D, levels, t, 13 * D + t)
    scale = 1.2 / math.sqrt(D)
    want = R.beam_step(q, ps, kgen, vgen, anc, t, B, scale)
    dev = [tuple(x.cuda() for x in p) for p in ps]
    args = (kgen.cuda(), vgen.cuda(), anc.cuda() if t else None, t, B)
    got = ops.shared_prefix_attention(q.cuda(), dev, *args, scale=scale)
    R.within(got, want, "out")
    # positions before heads in the prefix, as a prompt's projection leaves them: the same bits
    other = [(p[0].transpose(1, 2).contiguous().transpose(1, 2), p[1].transpose(1, 2).contiguous().transpose(1, 2), *p[2:]) for p in dev]
    assert torch.equal(got, ops.shared_prefix_attention(q.cuda(), other, *args, scale=scale))


@pytest.mark.gpu
def test_prefix_state_continues_another():
    """nsd_attn_prefix over two halves of a prefix leaves the state of the whole, whatever the split."""
    from silent_speech_amd import ops
    q, ps, kgen, vgen, anc = _beam_case(FP, 2, 6, 2, 2, 64, [(1, 1000, None)], 4, 2)
    k, v = (x.cuda() for x in ps[0])
    args = (kgen.cuda(), vgen.cuda(), anc.cuda(), 4, 6)
    want = R.beam_step(q, ps, kgen, vgen, anc, 4, 6, 0.125)
    for cut in (1, 64, 500, 999):
        halves = [(k[:, :, :cut], v[:, :, :cut]), (k[:, :, cut:], v[:, :, cut:])]
        R.within(ops.shared_prefix_attention(q.cuda(), halves, *args), want, cut)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,hidden,delta", [
    (FP, 1, 4, False), (BF, 1, 8, True), (FP, 7, 100, True), (BF, 33, 1000, True), (BF, 600, 2048, False), (FP, 515, 260, True),
    (BF, 5, 16384, True), (BF, 9, 16392, True), (FP, 6, 8196, False), (BF, 1100, 64, True), (FP, 1030, 1180, True)])
def test_add_rms_norm_and_its_gradients(dtype, rows, hidden, delta):
    from silent_speech_amd import ops
    g = _gen(rows + hidden)
    rnd = lambda s: (torch.randn(rows, hidden, generator=g) * s).to(dtype)   # noqa: E731
    x, d = rnd(2.0), rnd(0.7) if delta else None
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(dtype)
    go, dh = rnd(1.0), rnd(1.0)
    leaves = [y.cuda().requires_grad_() if y is not None else None for y in (x, d, w)]
    for parts in ("both", "h", "sum"):
        x_out, h = ops.add_rms_norm(*leaves, 1e-5)
        want = R.add_rms_norm(x, d, w, 1e-5, go if parts != "h" else None, dh if parts != "sum" else torch.zeros_like(dh))
        if parts == "both":
            R.within(x_out, want["x_out"], "x_out")
            R.within(h, want["h"], "h")
        outs = {"both": ((x_out, h), (go, dh)), "h": ((h,), (dh,)), "sum": ((x_out,), (go,))}[parts]
        take = [y for y in leaves if y is not None]
        grads = torch.autograd.grad(outs[0], take, [y.cuda() for y in outs[1]], allow_unused=parts == "sum")
        R.within(grads[0], want["dx"], parts + " dx")
        if delta:
            assert torch.equal(grads[0], grads[1])
        if grads[-1] is not None:
            R.within(grads[-1], want["dw"], parts + " dw")
        else:
            assert parts == "sum"
    # a frozen weight, and rows with other axes in front
    xs = leaves[0].detach().view(1, rows, hidden).requires_grad_()
    x_out, h = ops.add_rms_norm(xs, None, leaves[2].detach(), 1e-5)
    (dx,) = torch.autograd.grad((x_out, h), xs, (go.cuda()[None], dh.cuda()[None]))
    R.within(dx[0], R.add_rms_norm(x, None, w, 1e-5, go, dh)["dx"], "frozen dx")


@pytest.mark.gpu
def test_add_rms_norm_of_no_rows_and_odd_views():
    from silent_speech_amd import ops
    x, w = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True), torch.ones(64, device="cuda", dtype=BF, requires_grad=True)
    x_out, h = ops.add_rms_norm(x, None, w)
    dx, dw = torch.autograd.grad(h, (x, w), torch.empty_like(h))
    assert dx.shape == (0, 64) and dw.shape == (64,) and not bool(dw.any())
    g = _gen(8)
    big = torch.randn(6, 130, generator=g).cuda()
    view = big[:, 1:129]                                        # rows that start off a 16-byte boundary
    wv = torch.ones(128, device="cuda")
    a, b = ops.add_rms_norm(view, None, wv), ops.add_rms_norm(view.contiguous(), None, wv)
    assert torch.equal(a[1], b[1])


# ---------------------------------------------------------------------- streams, graphs, threads
def _work(seed, L=150, dtype=BF):
    g = _gen(seed)
    KVH, G, D = 2, 3, 64
    x = [torch.randn(2, L, h, D, generator=g).to(dtype).cuda() for h in (KVH * G, KVH, KVH)]
    do = torch.randn(2, L, KVH * G, D, generator=g).to(dtype).cuda()
    r = [torch.randn(300, 256, generator=g).to(dtype).cuda() for _ in range(4)]
    w = torch.randn(256, generator=g).to(dtype).cuda()
    q, ps, kgen, vgen, anc = _beam_case(dtype, 2, 6, 2, 2, 64, [(1, 1300, None), (2, 50, [50, 7])], 3, seed)
    beam = (q.cuda(), [tuple(y.cuda() for y in p) for p in ps], kgen.cuda(), vgen.cuda(), anc.cuda(), 3, 6)
    return x, do, r, w, beam


def _all_ops(x, do, r, w, beam):
    """Every operator once, forward and backward, from leaves of its own."""
    from silent_speech_amd import ops
    leaves = [y.detach().requires_grad_() for y in x]
    out = ops.attention(*leaves)
    got = [out, *torch.autograd.grad(out, leaves, do)]
    ln = [y.detach().requires_grad_() for y in (r[0], r[1], w)]
    x_out, h = ops.add_rms_norm(*ln)
    got += [x_out, h, *torch.autograd.grad((x_out, h), ln, (r[2], r[3]))]
    got.append(ops.shared_prefix_attention(*beam))
    return [y.detach() for y in got]


@pytest.mark.gpu
def test_operators_give_the_same_bits_again_and_on_other_streams():
    case = _work(1)
    want = [y.clone() for y in _all_ops(*case)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_all_ops(*case), want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:                                          # two at once, their scratch apart
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([_all_ops(*case) for _ in range(5)])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for runs in got:
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, want))


@pytest.mark.gpu
def test_operators_in_two_captured_graphs():
    """Forward and backward passes captured into two graphs, replayed by turns with other inputs and the program's own
    eager work between: every replay equals the eager result."""
    cases = [_work(2, 150), _work(3, 90)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            _all_ops(*c)
    torch.cuda.current_stream().wait_stream(side)
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_ops(*c))
        graphs.append(g)
    for i in range(4):
        for c in cases:                                         # new inputs in the captured places
            for t in (*c[0], c[1], *c[2], c[4][0]):
                t.copy_(torch.randn(t.shape, generator=_gen(100 + i)).to(t.dtype))
        want = [[y.clone() for y in _all_ops(*c)] for c in cases]
        for k in (0, 1, 0):
            graphs[k].replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, e)), i


@pytest.mark.gpu
def test_operators_from_two_threads():
    import threading
    cases = [_work(5, 120), _work(6, 77)]
    want = [[y.clone() for y in _all_ops(*c)] for c in cases]
    bad = []

    def run(i):
        try:
            st = torch.cuda.Stream()
            st.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(st):
                runs = [_all_ops(*cases[i]) for _ in range(20)]
            st.synchronize()
            if not all(torch.equal(a, b) for r in runs for a, b in zip(r, want[i])):
                bad.append(i)
        except Exception as e:                                  # noqa: BLE001 - reported below
            bad.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
def test_gradients_are_differentiable_once():
    from silent_speech_amd import ops
    q, k, v = (torch.randn(1, 9, 2, 32, device="cuda").requires_grad_() for _ in range(3))
    (dq,) = torch.autograd.grad(ops.attention(q, k, v).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()
    x, w = torch.randn(3, 32, device="cuda").requires_grad_(), torch.ones(32, device="cuda")
    (dx,) = torch.autograd.grad(ops.add_rms_norm(x, None, w)[1].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    go = torch.ones(3, 32, device="cuda")                       # a gradient that only passes through is left as it was
    torch.autograd.grad(ops.add_rms_norm(x, None, w)[0], x, go, create_graph=True)
    assert not go.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(9, 512), (5, 16392)])
def test_add_rmsnorm_bwd_writes_over_dx_out(rows, hidden):
    lib, L = _lib()
    g = _gen(hidden)
    x, dh, go = (torch.randn(rows, hidden, generator=g).to(BF).cuda() for _ in range(3))
    w, dw = torch.randn(hidden, generator=g).to(BF).cuda(), torch.zeros(hidden, dtype=BF, device="cuda")
    n = L.nsd_add_rmsnorm_bwd_workspace(rows, hidden)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    want = R.add_rms_norm(x, None, w, 1e-5, go, dh)
    lib.check(L.nsd_add_rmsnorm_bwd(x.data_ptr(), w.data_ptr(), dh.data_ptr(), go.data_ptr(), 1e-5, rows, hidden, 1, go.data_ptr(),
                                    dw.data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream), "nsd_add_rmsnorm_bwd")
    R.within(go, want["dx"], "dx")
    R.within(dw, want["dw"], "dw")


@pytest.mark.gpu
def test_attention_over_an_offset_past_32_bits():
    """Keys and values more than 4 GiB apart within one call: the batch stride of a large cache."""
    from silent_speech_amd import ops
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB")
    g = _gen(4)
    L, D = 130, 64
    far = (1 << 31) + (1 << 20)                                 # elements: 4.3 GB
    base = torch.empty(far + L * D, dtype=BF, device="cuda")
    k = base.as_strided((2, L, 1, D), (far, D, D, 1))
    k.copy_(torch.randn(2, L, 1, D, generator=g).to(BF))
    q = torch.randn(2, L, 2, D, generator=g).to(BF).cuda()
    want = ops.attention(q, k.contiguous(), k.contiguous())
    assert torch.equal(ops.attention(q, k, k), want)
    tok = base.as_strided((1, 2, 1, D), (0, far, D, 1))         # the same as a position's stride
    ref = ops.attention(q[:1, :2], tok.contiguous(), tok.contiguous())
    assert torch.equal(ops.attention(q[:1, :2], tok, tok), ref)
    kgen = torch.zeros(1, 4, 1, D, dtype=BF, device="cuda")
    pre = base.as_strided((2, 1, L, D), (far, D, D, 1))
    qs = torch.randn(4, 2, D, generator=g).to(BF).cuda()
    a, b = (ops.shared_prefix_attention(qs, [(p, p)], kgen, kgen, None, 0, 2) for p in (pre, pre.contiguous()))
    assert torch.equal(a, b)


# ---------------------------------------------------------------------- refusals (no GPU needed)
def _lib():
    from silent_speech_amd import lib
    return lib, lib.load()


def _seq(**kw):
    lib, _ = _lib()
    p = lib.SeqAttn()
    base = dict(batch=1, len_q=4, len_k=4, heads=4, kv_heads=2, hd=64, dtype=1, causal=1, scale=0.125)
    base.update({k: v for k, v in kw.items() if not k.endswith("_stride")})
    for k, v in base.items():
        setattr(p, k, v)
    for n in ("q_stride", "k_stride", "v_stride"):
        setattr(p, n, (C.c_int64 * 3)(*kw.get(n, (1024, 256, 64))))
    return p


def test_c_entries_refuse_what_they_cannot_do():
    lib, L = _lib()
    A, SIZE, NULL = 4096, -7, -1                                 # an aligned address that no refused call reads
    fwd = lambda p, q=A, k=A, v=A, out=A, ws=None, n=0: L.nsd_attn_fwd(q, k, v, C.byref(p), out, None, None, ws, n, None)   # noqa: E731
    for bad in (dict(hd=4), dict(hd=136), dict(hd=60), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(dtype=2), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(batch=-1), dict(len_q=-1), dict(len_k=-2),
                dict(len_q=1 << 30, heads=8), dict(batch=1 << 30), dict(len_k=(1 << 30) + 1),
                dict(batch=(1 << 31) - 1, heads=1 << 20, kv_heads=1 << 20), dict(len_q=1 << 16, heads=512, kv_heads=1)):
        assert fwd(_seq(**bad)) == SIZE, bad
        assert L.nsd_attn_bwd(A, A, A, A, A, None, A, C.byref(_seq(**bad)), A, A, A, A, 1 << 40, None) == SIZE, bad
        assert L.nsd_attn_prefix(A, A, A, C.byref(_seq(**{"causal": 0, **bad})), 0, A, A, A, A, 1 << 40, None) == SIZE, bad
        assert L.nsd_attn_fwd_workspace(C.byref(_seq(**bad))) == 0 and L.nsd_attn_bwd_workspace(C.byref(_seq(**bad))) == 0
    assert fwd(_seq(), q=None) == NULL and fwd(_seq(), k=None) == NULL and fwd(_seq(), out=None) == NULL
    for bad in ("q_stride", "k_stride", "v_stride"):
        assert fwd(_seq(**{bad: (1024, 250, 64)})) == lib.E_ALIGN
    assert fwd(_seq(), q=A + 8) == lib.E_ALIGN and fwd(_seq(), out=A + 2) == lib.E_ALIGN
    assert fwd(_seq(batch=0)) == 0 and fwd(_seq(len_q=0)) == 0    # nothing to do
    long = _seq(len_q=1, len_k=50000)
    need = L.nsd_attn_fwd_workspace(C.byref(long))
    assert need > 0 and fwd(long) == NULL and fwd(long, ws=A, n=need - 1) == SIZE
    bwd = lambda p, ws=A, n=1 << 20, dq=A, dk=A: L.nsd_attn_bwd(A, A, A, A, A, None, A, C.byref(p), dq, dk, A, ws, n, None)   # noqa: E731
    assert bwd(_seq(), ws=None) == NULL and bwd(_seq(), n=8) == SIZE and bwd(_seq(), dq=None) == NULL and bwd(_seq(), dk=A + 4) == lib.E_ALIGN
    p = _seq()
    p.key_len = A
    assert bwd(p) == SIZE                                       # ragged keys have no gradient form
    assert L.nsd_attn_prefix(A, A, A, C.byref(_seq(causal=1)), 0, A, A, A, A, 1 << 30, None) == SIZE
    p = _seq(causal=0)
    p.key_mask = A
    assert L.nsd_attn_prefix(A, A, A, C.byref(p), 0, A, A, A, A, 1 << 30, None) == SIZE
    assert L.nsd_attn_prefix(A, A, A, C.byref(_seq(causal=0)), 0, A, None, A, A, 1 << 30, None) == NULL
    nb = lambda rows=4, hidden=64, dt=1, x=A, dw=A, ws=A, n=1 << 20: L.nsd_add_rmsnorm_bwd(x, A, A, None, 1e-5, rows, hidden, dt, A, dw, ws, n, None)   # noqa: E731
    assert nb(hidden=60) == SIZE and nb(rows=-1) == SIZE and nb(dt=3) == SIZE and nb(x=None) == NULL and nb(ws=None) == NULL
    assert nb(n=4) == SIZE and nb(x=A + 2) == lib.E_ALIGN and nb(rows=0, dw=None) == 0


def test_c_entries_refuse_launches_of_2_to_the_32_threads():
    lib, L = _lib()
    A, SIZE, many = 4096, -7, 1 << 24
    one = dict(heads=1, kv_heads=1, hd=8, len_q=1, len_k=1, causal=0)
    for p in (_seq(**{**one, "batch": many}), _seq(**{**one, "batch": many // 64, "len_q": 8192}),
              _seq(**{**one, "batch": many // 4, "kv_heads": 4, "heads": 4})):
        assert L.nsd_attn_fwd(A, A, A, C.byref(p), A, None, None, None, 0, None) == SIZE
        assert L.nsd_attn_prefix(A, A, A, C.byref(p), 0, A, A, A, None, 0, None) == SIZE
        assert L.nsd_attn_bwd(A, A, A, A, A, None, A, C.byref(p), A, A, A, A, 1 << 62, None) == SIZE
    p = _seq(**{**one, "batch": many // 2, "len_k": 65})          # two tiles of keys for each sequence
    assert L.nsd_attn_fwd_workspace(C.byref(p)) == 0 and L.nsd_attn_bwd_workspace(C.byref(p)) == 0
    assert L.nsd_attn_bwd(A, A, A, A, A, None, A, C.byref(p), A, A, A, A, 1 << 62, None) == SIZE
    p = _seq(**{**one, "batch": many // 2, "len_k": 64})
    assert L.nsd_attn_bwd_workspace(C.byref(p)) > 0
    norm = lambda rows, hidden: L.nsd_add_rmsnorm(A, None, A, 1e-5, rows, hidden, 1, None, A, None)   # noqa: E731
    assert norm(1 << 26, 8) == SIZE and norm(1 << 24, 4096) == SIZE and norm((1 << 31) - 1, 1 << 20) == SIZE
    back = lambda rows, hidden: L.nsd_add_rmsnorm_bwd(A, A, A, None, 1e-5, rows, hidden, 1, A, A, A, 1 << 62, None)   # noqa: E731
    assert back((1 << 31) - 1, 8) == SIZE and back(1 << 22, 1 << 15) == SIZE and back(0, 1 << 28) == SIZE and back(4, 1 << 28) == SIZE
    step = lambda N, B, kvh: L.nsd_attn_step(A, None, None, A, A, A, A, N, B, kvh, kvh, 8, 0, 1, 0.3, 1, None, None, None, None)   # noqa: E731
    assert step(1 << 26, 1, 1) == SIZE and step(1 << 20, 16, 4) == SIZE and step(1 << 30, 1, 1 << 10) == SIZE


@pytest.mark.gpu
def test_beam_step_holds_its_ancestors_to_the_beam():
    """A table entry past the beam reads the beam's last slot."""
    from silent_speech_amd import ops
    g = _gen(11)
    N, B, t, D = 3, 4, 5, 64
    kg, vg = (torch.randn(t + 1, N * B, 2, D, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.randn(N * B, 4, D, generator=g).to(BF).cuda()
    anc = torch.randint(0, 256, (t, N * B), generator=g).to(torch.uint8)
    a = ops.shared_prefix_attention(q, [], kg, vg, anc.cuda(), t, B)
    b = ops.shared_prefix_attention(q, [], kg, vg, anc.clamp(max=B - 1).cuda(), t, B)
    assert torch.equal(a, b)


def test_python_entries_refuse_what_they_cannot_do():
    from silent_speech_amd import lib, ops
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)             # noqa: E731
    q, k = z(1, 4, 4, 64), z(1, 4, 2, 64)
    with pytest.raises(lib.NsdError):
        ops.attention(q, k, k)
    for bad in ((z(4, 4, 64), k, k), (q, k, z(1, 5, 2, 64)), (q, z(2, 4, 2, 64), z(2, 4, 2, 64)), (q, z(1, 4, 3, 64), z(1, 4, 3, 64)),
                (z(1, 4, 4, 60), z(1, 4, 2, 60), z(1, 4, 2, 60)), (z(1, 4, 4, 256), z(1, 4, 2, 256), z(1, 4, 2, 256))):
        with pytest.raises(ValueError):
            ops.attention(*bad)
    kg, anc = z(3, 6, 2, 64), z(3, 6, dt=torch.uint8)
    qs, pre = z(6, 4, 64), (z(1, 2, 9, 64), z(1, 2, 9, 64))
    with pytest.raises(lib.NsdError):
        ops.shared_prefix_attention(qs, [pre], kg, kg, anc, 2, 3)
    for bad in (dict(t=3), dict(t=-1), dict(beam=4), dict(beam=0), dict(q=z(6, 10, 64)), dict(q=z(6, 4, 32)), dict(q=z(5, 4, 64))):
        a = dict(q=qs, t=2, beam=3)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(a["q"], [pre], kg, kg, anc, a["t"], a["beam"])
    x = z(4, 64)
    with pytest.raises(lib.NsdError):
        ops.add_rms_norm(x, None, z(64))
    for bad in ((x, None, z(32)), (x, z(4, 32), z(64)), (z(()), None, z(1))):
        with pytest.raises(ValueError):
            ops.add_rms_norm(*bad)


@pytest.mark.gpu
def test_python_entries_refuse_device_tensors_that_do_not_fit():
    from silent_speech_amd import ops
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device="cuda")   # noqa: E731
    q, k = z(1, 4, 4, 64), z(1, 4, 2, 64)
    with pytest.raises(TypeError):
        ops.attention(q.half(), k.half(), k.half())
    with pytest.raises(TypeError):
        ops.attention(q, k.float(), k.float())
    with pytest.raises(ValueError):
        ops.attention(q, k, k.cpu())
    for bad in (dict(key_mask=z(1, 5, dt=torch.bool)), dict(key_mask=z(1, 4, dt=FP)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf)):
        with pytest.raises(ValueError):
            ops.attention(q, k, k, **bad)
    kg, anc, qs = z(3, 6, 2, 64), z(3, 6, dt=torch.uint8), z(6, 4, 64)
    pre = (z(1, 2, 9, 64), z(1, 2, 9, 64))
    for bad in ([pre[:1]], [(pre[0], pre[1][:, :, :4])], [(z(4, 2, 9, 64), z(4, 2, 9, 64))], [(z(1, 1, 9, 64), z(1, 1, 9, 64))],
                [(*pre, z(1, dt=torch.int64))], [(*pre, z(2, dt=torch.int32))]):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(qs, bad, kg, kg, anc, 2, 3)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(qs, [pre], kg, kg, None, 2, 3)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(qs, [pre], kg.transpose(0, 1).contiguous().transpose(0, 1), kg, anc, 2, 3)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(qs.requires_grad_(), [pre], kg, kg, anc, 2, 3)
    with pytest.raises(ValueError):
        ops.add_rms_norm(z(4, 60), None, z(60))
    with pytest.raises(TypeError):
        ops.add_rms_norm(z(4, 64), None, z(64, dt=FP))
