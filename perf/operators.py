"""The AR head's operators for training and for long prompts, in plain form and as the framework's own calls.

attn    causal attention of whole sequences with a key mask, forward and (train) its gradients
prefix  one decode step of a beam: every hypothesis attends to prefixes that it shares with others, to the generated
        positions of its own ancestors, and to itself
norm    residual add + RMSNorm, forward and gradients, the weight's among them
"""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
_DT = {BF16: torch.bfloat16, F32: torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------- cases
def _attn(name, dtype, z, lq, lk, kvh, g, d, train, masked):
    return {"name": name, "op": "attn", "dtype": dtype, "z": z, "lq": lq, "lk": lk, "kvh": kvh, "g": g, "d": d,
            "train": train, "masked": masked}


def _prefix(name, dtype, n, b, kvh, g, d, shared, ctx, ragged, t):
    return {"name": name, "op": "prefix", "dtype": dtype, "n": n, "b": b, "kvh": kvh, "g": g, "d": d,
            "shared": shared, "ctx": ctx, "ragged": ragged, "t": t}


def _norm(name, dtype, rows, hidden, delta):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "hidden": hidden, "delta": delta}


def listed():
    return [
        # one short utterance in a small model: what a call costs when there is hardly any work
        _attn("train_tiny", BF16, 1, 24, 24, 2, 2, 64, True, False),
        # a training batch: 512 context frames, padded to the longest of the batch, and up to 128 characters
        _attn("train_batch", BF16, 8, 640, 640, 8, 3, 128, True, True),
        # one long recording
        _attn("train_long", BF16, 1, 8192, 8192, 8, 3, 128, True, False),
        # the same in fp32, as a check of gradients is run, at sizes that fit no tile
        _attn("train_f32_odd", F32, 3, 217, 217, 2, 3, 80, True, True),
        # contexts of a decode batch, prefill only
        _attn("prefill", BF16, 32, 768, 768, 8, 3, 128, False, True),
        # candidate transcripts scored against cached contexts: few new positions over many cached ones
        _attn("candidates", BF16, 96, 63, 320, 8, 3, 128, False, False),
        # one utterance, a small beam, a short prompt
        _prefix("beam_tiny", BF16, 1, 4, 2, 2, 64, 100, 0, False, 3),
        # a decode batch that shares a prompt, with a context of frames for each utterance
        _prefix("beam_batch", BF16, 64, 16, 8, 3, 128, 2048, 160, False, 20),
        # one utterance over a very long recording: the cache is all there is to read
        _prefix("beam_long", BF16, 1, 16, 8, 3, 128, 131072, 0, False, 9),
        # contexts of differing lengths, fp32, a beam that fills no tile
        _prefix("beam_f32_ragged", F32, 5, 7, 3, 2, 64, 0, 1537, True, 13),
        # the norm of a training batch's tokens
        _norm("norm_batch", BF16, 8192, 4096, True),
        # fp32, odd numbers of rows and columns
        _norm("norm_f32_odd", F32, 1037, 1180, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attn", "attn", "prefix", "prefix", "norm"))
    dtype = rng.choice((BF16, BF16, F32))
    if op == "norm":
        hidden = 8 * _log(rng, 8, 1024)
        rows = min(_log(rng, 1, 16384), 8192 * 4096 // hidden)
        return {"op": "norm", "dtype": dtype, "rows": rows, "hidden": hidden, "delta": rng.random() < 0.7}
    kvh, g = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8))
    if op == "attn":
        lk = _log(rng, 1, 4096)
        lq = lk if rng.random() < 0.7 else min(lk, _log(rng, 1, 512))
        d = rng.choice((32, 64, 80, 96, 128, 128))
        room = 8192 * 8192 * 24 * 128 // (8 if dtype == F32 else 2)
        z = max(1, min(_log(rng, 1, 32), room // (lq * lk * kvh * g * d)))
        return {"op": "attn", "dtype": dtype, "z": z, "lq": lq, "lk": lk, "kvh": kvh, "g": g, "d": d,
                "train": rng.random() < 0.7, "masked": rng.random() < 0.5}
    n, b = _log(rng, 1, 64), rng.randint(1, 24)
    shared = _log(rng, 16, 65536) if rng.random() < 0.7 else 0
    ctx = _log(rng, 16, 2048) if rng.random() < 0.5 or not shared else 0
    room = 30_000_000
    while n > 1 and n * b * kvh * g * (shared + ctx) > room:
        n //= 2
    return {"op": "prefix", "dtype": dtype, "n": n, "b": b, "kvh": kvh, "g": g, "d": rng.choice((64, 128)),
            "shared": shared, "ctx": ctx, "ragged": ctx > 0 and rng.random() < 0.5, "t": rng.randint(0, 40)}


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dt)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device=dev)

    s = {"case": case}
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        s["x"] = rnd(rows, hidden, scale=2.0).requires_grad_()
        s["delta"] = rnd(rows, hidden, scale=0.5).requires_grad_() if case["delta"] else None
        s["w"] = (1.0 + 0.2 * rnd(hidden).float()).to(dt).requires_grad_()
        s["dx_out"], s["dh"] = rnd(rows, hidden), rnd(rows, hidden)
        return s
    kvh, g, d = case["kvh"], case["g"], case["d"]
    h = kvh * g
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] == "attn":
        z, lq, lk = case["z"], case["lq"], case["lk"]
        # projections of one product, as a layer has them: q, k and v are views of it where all positions are new
        if lq == lk:
            qkv = rnd(z, lq, (h + 2 * kvh) * d, scale=1.3)
            s["q"], s["k"], s["v"] = (t.unflatten(-1, (-1, d)) for t in qkv.split([h * d, kvh * d, kvh * d], dim=-1))
        else:
            s["q"], s["k"], s["v"] = rnd(z, lq, h, d, scale=1.3), rnd(z, lk, kvh, d, scale=1.3), rnd(z, lk, kvh, d)
        s["mask"] = None
        if case["masked"]:
            # [context padded at its end ; characters padded at theirs]
            c = max(1, lk * 4 // 5)
            pos = torch.arange(lk, device=dev)[None]
            n_ctx, n_chr = whole(c // 2, c + 1, z)[:, None], whole(0, lk - c + 1, z)[:, None]
            s["mask"] = (pos < n_ctx) | ((pos >= c) & (pos < c + n_chr))
        if case["train"]:
            for n in "qkv":
                s[n] = s[n].detach().requires_grad_()
            s["dout"] = rnd(z, lq, h, d)
            if s["mask"] is not None:       # a loss gives no gradient to padded positions
                s["dout"] = s["dout"] * s["mask"][:, lk - lq:, None, None]
        return s
    n, b, t = case["n"], case["b"], case["t"]
    m = n * b
    s["q"] = rnd(m, h, d, scale=1.3)
    s["prefixes"] = []
    if case["shared"]:
        s["prefixes"].append((rnd(1, kvh, case["shared"], d, scale=1.3), rnd(1, kvh, case["shared"], d)))
    if case["ctx"]:
        k, v = rnd(n, kvh, case["ctx"], d, scale=1.3), rnd(n, kvh, case["ctx"], d)
        lens = whole(case["ctx"] // 2, case["ctx"] + 1, n).to(torch.int32) if case["ragged"] else None
        s["prefixes"].append((k, v) if lens is None else (k, v, lens))
    s["kgen"], s["vgen"] = rnd(t + 1, m, kvh, d, scale=1.3), rnd(t + 1, m, kvh, d)
    # ancestors[s, m]: the rank at position s of the hypothesis that m descends from
    anc = torch.zeros(max(t, 1), m, dtype=torch.uint8, device=dev)
    back = whole(0, b, max(t, 1), n, b)
    at = torch.arange(b, device=dev).expand(n, b)
    for i in range(t - 1, -1, -1):
        at = back[i].gather(1, at)
        anc[i] = at.reshape(-1)
    s["anc"] = anc
    return s


# ---------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"attn": _plain_attn, "prefix": _plain_prefix, "norm": _plain_norm}[s["case"]["op"]](s)


def _run_own(s):
    from silent_speech_amd import ops
    c = s["case"]
    if c["op"] == "prefix":
        return {"out": ops.shared_prefix_attention(s["q"], s["prefixes"], s["kgen"], s["vgen"], s["anc"], c["t"],
                                                   c["b"], scale=s["scale"])}
    if c["op"] == "attn":
        out = ops.attention(s["q"], s["k"], s["v"], causal=True, key_mask=s["mask"], scale=s["scale"])
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    x_out, h = ops.add_rms_norm(s["x"], s["delta"], s["w"], EPS)
    dx, dw = torch.autograd.grad((x_out, h), (s["x"], s["w"]), (s["dx_out"], s["dh"]))
    return {"x_out": x_out.detach(), "h": h.detach(), "dx": dx, "dw": dw}


def _visible(c, mask, dev):
    lq, lk = c["lq"], c["lk"]
    vis = torch.arange(lk, device=dev)[None] <= torch.arange(lq, device=dev)[:, None] + (lk - lq)
    return vis if mask is None else vis & mask[:, None, None, None, :]


def _softmax(x):
    """Over the last axis, in place; a row of -inf gives zeros."""
    x -= x.amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)
    x.exp_()
    x /= x.sum(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).tiny)
    return x


def _plain_attn(s):
    c = s["case"]
    z, lq, lk, kvh, g, d = (c[n] for n in ("z", "lq", "lk", "kvh", "g", "d"))
    dt = s["q"].dtype

    def rows(x):                                    # [z, lq, kvh * g, d] -> [z, kvh, g * lq, d]
        return x.float().view(z, lq, kvh, g, d).permute(0, 2, 3, 1, 4).reshape(z, kvh, g * lq, d)

    def back(x):
        return x.view(z, kvh, g, lq, d).permute(0, 3, 1, 2, 4).reshape(z, lq, kvh * g, d).to(dt)

    q, k, v = rows(s["q"]), s["k"].float().transpose(1, 2).contiguous(), s["v"].float().transpose(1, 2).contiguous()
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).view(z, kvh, g, lq, lk)
    p = _softmax(p.masked_fill_(~_visible(c, s["mask"], p.device), -math.inf)).view(z, kvh, g * lq, lk)
    out = torch.matmul(p, v)
    if not c["train"]:
        return {"out": back(out)}
    do = rows(s["dout"])
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (do * out).sum(-1, keepdim=True)
    ds *= p
    del p
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(-1, -2), q) * s["scale"]
    return {"out": back(out), "dq": back(dq), "dk": dk.transpose(1, 2).contiguous().to(dt),
            "dv": dv.transpose(1, 2).contiguous().to(dt)}


def _plain_prefix(s):
    c = s["case"]
    n, b, kvh, g, d, t = (c[x] for x in ("n", "b", "kvh", "g", "d", "t"))
    m, dev = n * b, s["q"].device
    q = s["q"].float().view(m, kvh, g, d)

    def groups(x, ng):                              # [m, kvh, g, *] -> [ng, kvh, (m / ng) * g, *]
        return x.reshape(ng, m // ng, kvh, g, -1).transpose(1, 2).reshape(ng, kvh, m // ng * g, -1)

    def members(x, ng):
        return x.reshape(ng, kvh, m // ng, g, -1).transpose(1, 2).reshape(m, kvh, g, -1)

    scores = []
    for p in s["prefixes"]:
        ng, length = p[0].shape[0], p[0].shape[2]
        x = torch.matmul(groups(q, ng), p[0].float().transpose(-1, -2))
        if len(p) == 3:
            x = x.masked_fill(torch.arange(length, device=dev) >= p[2][:, None, None, None], -math.inf)
        scores.append(members(x, ng))
    # the generated rows of m's ancestors, and its own
    slot = torch.cat([s["anc"][:t].long() + torch.arange(m, device=dev) // b * b, torch.arange(m, device=dev)[None]])
    at = torch.arange(t + 1, device=dev)[:, None]
    kg, vg = (s[x][at, slot].float().permute(1, 2, 0, 3).contiguous() for x in ("kgen", "vgen"))   # [m, kvh, t + 1, d]
    scores.append(torch.matmul(q, kg.transpose(-1, -2)))
    w = _softmax(torch.cat(scores, -1).mul_(s["scale"])).split([x.shape[-1] for x in scores], -1)
    out = torch.matmul(w[-1], vg)
    for p, x in zip(s["prefixes"], w):
        out = out + members(torch.matmul(groups(x, p[0].shape[0]), p[1].float()), p[0].shape[0])
    return {"out": out.reshape(m, kvh * g, d).to(s["q"].dtype)}


def _plain_norm(s):
    dt = s["x"].dtype
    # the residual stream is kept in its type: the norm is of the sum as it is stored
    x_out = s["x"] if s["delta"] is None else (s["x"].float() + s["delta"].float()).to(dt)
    x, w, dh = x_out.float(), s["w"].float(), s["dh"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh = x * r
    gw = dh * w
    dx = s["dx_out"].float() + r * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    return {"x_out": x_out.detach(), "h": (xh * w).to(dt), "dx": dx.to(dt), "dw": (dh * xh).sum(0).to(dt)}


# ---------------------------------------------------------------------- 64 bits, from the definition
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "prefix": _exact_prefix, "norm": _exact_norm}[case["op"]](s)


def _exact_attn(s):
    c = s["case"]
    g, off = c["g"], c["lk"] - c["lq"]
    got = {n: [] for n in ("out", "dq", "dk", "dv")}
    hidden = torch.ones(c["lq"], c["lk"], dtype=torch.bool, device=s["q"].device).triu(off + 1)
    for z in range(c["z"]):
        hide = hidden if s["mask"] is None else hidden | ~s["mask"][z]
        empty = hide.all(-1, keepdim=True)
        per = {n: [] for n in got}
        for j in range(c["kvh"]):
            k, v = (s[n][z, :, j].detach().double().requires_grad_(c["train"]) for n in "kv")
            for i in range(j * g, j * g + g):
                q = s["q"][z, :, i].detach().double().requires_grad_(c["train"])
                a = (q @ k.t() * s["scale"]).masked_fill(hide, -math.inf).masked_fill(empty, 0.0)
                o = (torch.softmax(a, -1) @ v).masked_fill(empty, 0.0)
                per["out"].append(o.detach())
                if c["train"]:
                    o.backward(s["dout"][z, :, i].double())
                    per["dq"].append(q.grad)
            if c["train"]:
                per["dk"].append(k.grad)
                per["dv"].append(v.grad)
        for n in got:
            if per[n]:
                got[n].append(torch.stack(per[n], 1))
    return {n: torch.stack(x) for n, x in got.items() if x}


def _exact_prefix(s):
    c = s["case"]
    m, b, g, t = c["n"] * c["b"], c["b"], c["g"], c["t"]
    q = s["q"].double()
    out = torch.empty_like(q)
    for i in range(m):
        gen = torch.tensor([int(a) for a in s["anc"][:t, i].tolist()], device=q.device).long() + i // b * b
        for j in range(c["kvh"]):
            ks, vs = [], []
            for p in s["prefixes"]:
                u = i * p[0].shape[0] // m
                n = int(p[2][u]) if len(p) == 3 else p[0].shape[2]
                ks.append(p[0][u, j, :n])
                vs.append(p[1][u, j, :n])
            steps = torch.arange(t, device=q.device)
            ks += [s["kgen"][steps, gen, j], s["kgen"][t, i, j][None]]
            vs += [s["vgen"][steps, gen, j], s["vgen"][t, i, j][None]]
            k, v = torch.cat(ks).double(), torch.cat(vs).double()
            a = q[i, j * g:j * g + g] @ k.t() * s["scale"]
            out[i, j * g:j * g + g] = torch.exp(a - torch.logsumexp(a, -1, keepdim=True)) @ v
    return {"out": out}


def _exact_norm(s):
    x64 = s["x"].detach().double() if s["delta"] is None else s["x"].detach().double() + s["delta"].detach().double()
    x = x64.to(s["x"].dtype).double().requires_grad_()
    w = s["w"].detach().double().requires_grad_()
    h = x / (x * x).mean(-1, keepdim=True).add(EPS).sqrt() * w
    dx, dw = torch.autograd.grad((x * 1.0, h), (x, w), (s["dx_out"].double(), s["dh"].double()))
    return {"x_out": x64, "h": h.detach(), "dx": dx, "dw": dw}


# ---------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        # x, delta, both gradients in; the sum (where there is one), the normed rows and the gradient out
        return {"bytes": e * (n * (7 if case["delta"] else 5) + 2 * case["hidden"]), "flops": 14 * n}
    kvh, g, d = case["kvh"], case["g"], case["d"]
    h = kvh * g
    if case["op"] == "attn":
        z, lq, lk = case["z"], case["lq"], case["lk"]
        seen = 0.7 if case["masked"] else 1.0       # the share of keys that a padded batch keeps, on average
        pairs = z * h * (lq * (lk - lq) + lq * (lq + 1) // 2) * seen
        q, kv = z * lq * h * d * e, z * lk * kvh * d * e * 2
        if case["train"]:
            return {"bytes": 4 * q + 2 * kv, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + kv, "flops": 4 * d * pairs}
    n, b, t = case["n"], case["b"], case["t"]
    m = n * b
    ctx = case["ctx"] * (0.75 if case["ragged"] else 1.0)
    # of a generated position, the rows that are some hypothesis's ancestor: at least one for each utterance
    kv = 2 * kvh * d * e * (case["shared"] + n * ctx + n * t + m)
    return {"bytes": kv + 2 * m * h * d * e, "flops": 4 * d * m * h * (case["shared"] + ctx + t + 1)}
