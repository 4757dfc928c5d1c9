"""Performance cases of the operators for fine-tuning on packed images and clips: LayerNorm, rotary positions with several axes, and attention over
packed sequences, each with its gradient.

A case is a dict of plain values; its "kind" says which operator a pass goes through:

    attention   q, k, v of several sequences (images, clips) behind one another -> output and log-sum-exp, with train also the gradients of q, k, v.
                Lengths are texts ("1605,261"); k_lens "" = the lengths of q.  causal: a token sees itself and what is before it, and the first
                `prefix` tokens of its sequence.  cap: scores go through cap * tanh(score / cap).  bias: every head takes its slope times the
                distance off the score.
    rope        queries and keys rotated by positions on `axes` axes, with train also the gradient
    norm        LayerNorm of rows, with train also the gradients of the rows, the weight and the bias

`own` chooses between the plain form (elementary torch operations in 32 bits) and the package's operators.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
D = 64                                                  # channels per head in attention


# ------------------------------------------------------------------------------------------------ the cases
def _attention(name, q_lens, *, k_lens="", heads=16, kv_heads=16, dtype="bf16", causal=False, prefix=0, cap=0.0, bias=False, train=False):
    return dict(name=name, kind="attention", q_lens=q_lens, k_lens=k_lens, heads=heads, kv_heads=kv_heads, dtype=dtype, causal=causal, prefix=prefix, cap=cap,
                bias=bias, train=train)


def listed():
    return [
        # one thumbnail through a small model: 256 patches and 5 further tokens, the smallest call, latency counts
        _attention("attention_thumbnail", "261", heads=12, kv_heads=12),
        # frames of several sizes behind one another in one batch, for features
        _attention("attention_packed_sizes", "1605,261,1029,4101,77,1605,1,1029"),
        # a clip as a sequence: its first tokens (queries, cls, registers) are seen by all, the others by what follows
        _attention("attention_clip_prefix", "8197", dtype="f16", heads=16, kv_heads=4, causal=True, prefix=205),
        # a training step on a batch of frames of one size
        _attention("attention_train_frames", "1605,1605,1605,1605,1605,1605,1605,1605", train=True),
        # a training step on ragged crops with capped scores and shared key heads
        _attention("attention_train_capped", "1029,261,517,2053,133,1,1605,711,64,129", dtype="f16", heads=12, kv_heads=4, causal=True, prefix=5, cap=30.0, train=True),
        # 200 queries per image that read the image's tokens, the score falling with the distance, with gradients
        _attention("attention_train_queries", "200,200,200,31", k_lens="1605,1605,1029,261", heads=12, kv_heads=12, bias=True, train=True),
        # queries and keys of one thumbnail, rows and columns as positions
        dict(name="rope_thumbnail", kind="rope", tokens=261, heads=24, head_dim=64, axes=2, dtype="bf16", interleaved=False, partial=False, far=False, train=False),
        # queries and keys of a batch of clips: time, row and column, forward and gradient
        dict(name="rope_clips", kind="rope", tokens=51205, heads=32, head_dim=64, axes=3, dtype="bf16", interleaved=False, partial=False, far=False, train=True),
        # 32-bit features, a part of the channels rotated in neighbouring pairs, positions far out on a long time line
        dict(name="rope_far_partial", kind="rope", tokens=5003, heads=9, head_dim=80, axes=3, dtype="f32", interleaved=True, partial=True, far=True, train=True),
        # the residual stream of one thumbnail in 32 bits to 16-bit rows
        dict(name="norm_thumbnail", kind="norm", rows=261, width=768, dtype="f32", out="bf16", residual=False, train=False),
        # the residual stream of 14 frames, forward and gradient, the gradient of the residual path joined
        dict(name="norm_train_frames", kind="norm", rows=1605 * 14, width=1024, dtype="f32", out="bf16", residual=True, train=True),
        # many rows of an odd width in 16 bits
        dict(name="norm_train_odd", kind="norm", rows=40009, width=333, dtype="bf16", out="bf16", residual=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "rope", "norm"])
    if kind == "attention":
        top = max(work(c)["flops"] for c in listed() if c["kind"] == "attention")
        while True:
            n = rng.randint(1, 12)
            q = [_log(rng, 1, 4200) for _ in range(n)]
            cross = rng.random() < 0.25
            k = [max(a, _log(rng, 1, 4200)) for a in q] if cross else []
            kv = rng.choice([1, 2, 3, 4, 8])
            heads = kv * rng.choice([1, 2, 4]) if rng.random() < 0.5 else kv
            c = _attention("", ",".join(map(str, q)), k_lens=",".join(map(str, k)), heads=heads, kv_heads=kv, dtype=rng.choice(["bf16", "f16"]),
                           causal=rng.random() < 0.5, prefix=rng.choice([0, 5, 205]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3,
                           train=rng.random() < 0.6)
            if work(c)["flops"] <= top:
                break
    elif kind == "rope":
        c = dict(kind="rope", tokens=_log(rng, 1, 40000), heads=rng.randint(1, 32), head_dim=rng.choice([32, 48, 64, 80, 96, 128]), axes=rng.randint(1, 3),
                 dtype=rng.choice(["bf16", "f16", "f32"]), interleaved=rng.random() < 0.5, partial=rng.random() < 0.5, far=rng.random() < 0.3,
                 train=rng.random() < 0.5)
        while work(c)["bytes"] > 400e6:
            c["tokens"] = max(1, c["tokens"] // 2)
    else:
        c = dict(kind="norm", rows=_log(rng, 1, 40000), width=rng.choice([_log(rng, 1, 4200), 8 * _log(rng, 16, 520)]), dtype=rng.choice(["f32", "bf16", "f16"]),
                 out=rng.choice(["f32", "bf16", "f16"]), residual=rng.random() < 0.3, train=rng.random() < 0.7)
        while work(c)["bytes"] > 400e6:
            c["rows"] = max(1, c["rows"] // 2)
    c.pop("name", None)
    return c


def _lengths(case):
    q = [int(n) for n in case["q_lens"].split(",")]
    k = [int(n) for n in case["k_lens"].split(",")] if case["k_lens"] else q
    return q, k


def _rotated(case):
    """channels per axis that are rotated: as equal as even numbers allow; with partial about half of the head's channels."""
    pairs = case["head_dim"] // 4 if case["partial"] else case["head_dim"] // 2
    each, more = divmod(pairs, case["axes"])
    return [2 * (each + (a < more)) for a in range(case["axes"])]


def _pairs(case):
    """(query, key) pairs that see one another, of one head"""
    total = 0
    for lq, lk in zip(*_lengths(case)):
        if not case["causal"]:
            total += lq * lk
            continue
        off, pre = lk - lq, min(case["prefix"], lk)
        edge = min(max(pre - off, 0), lq)                # queries in front of this one see the prefix and nothing more
        total += edge * pre + (lq - edge) * off + (lq * (lq + 1) - edge * (edge + 1)) // 2
    return total


def work(case):
    if case["kind"] == "attention":
        q, k = (sum(n) for n in _lengths(case))
        h, hk = case["heads"], case["kv_heads"]
        pairs = _pairs(case) * h
        moved = 2 * D * (2 * q * h + 2 * k * hk) + 4 * q * h
        flops = 4 * D * pairs
        if case["train"]:
            moved += 2 * D * (2 * q * h + 2 * k * hk)       # the gradient in, those of q, k and v out
            flops += 10 * D * pairs
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * case["head_dim"]
        turned = case["tokens"] * case["heads"] * sum(_rotated(case))
        times = 2 if case["train"] else 1
        return {"bytes": times * 2 * n * BYTES[case["dtype"]] + 4 * case["tokens"] * case["axes"], "flops": times * 3 * turned}
    n = case["rows"] * case["width"]
    b, bo = BYTES[case["dtype"]], BYTES[case["out"]]
    moved, flops = n * (b + bo) + 8 * case["width"], 8 * n
    if case["train"]:
        moved += n * (bo + b + (b if case["residual"] else 0)) + 8 * case["width"]    # x is one input, read once for both directions
        flops += 14 * n
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _rand(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "attention":
        dt = DTYPES[case["dtype"]]
        ql, kl = _lengths(case)
        h, hk = case["heads"], case["kv_heads"]
        if case["k_lens"]:
            q = _rand(g, sum(ql), h, D, scale=1.5, dtype=dt)
            kv = _rand(g, sum(kl), 2 * hk, D, dtype=dt)
            s["q"], s["k"], s["v"] = q, kv[:, :hk], kv[:, hk:]
        else:                                           # one projection's rows: query, key and value heads side by side
            qkv = _rand(g, sum(ql), h + 2 * hk, D, scale=1.2, dtype=dt)
            s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        if case["train"]:
            s["dout"] = _rand(g, sum(ql), h, D, dtype=dt)
        s["slopes"] = 2.0 ** (-4 - 4 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h) if case["bias"] else None
        s["scale"] = D ** -0.5
        s["lens"] = (ql, kl)
        if own:
            from lightly_trian_quant_b200 import ops

            s["plan"] = ops.AttnPlan(ql, kl, causal=case["causal"], prefix=[min(case["prefix"], n) for n in kl] if case["causal"] else None)
    elif case["kind"] == "rope":
        dt, T = DTYPES[case["dtype"]], case["tokens"]
        s["x"] = _rand(g, T, case["heads"], case["head_dim"], dtype=dt)
        if case["train"]:
            s["dy"] = _rand(g, T, case["heads"], case["head_dim"], dtype=dt)
        side = 40
        t = torch.arange(T, device="cuda")
        grid = [t % side, t // side % side, t // (side * side)][:case["axes"]]
        if case["far"]:
            first = int(torch.randint(100_000, 900_000, (1,), generator=g, device="cuda"))
            grid = [first + 997 * p if i == len(grid) - 1 else p for i, p in enumerate(grid)]
        s["pos"] = torch.stack(grid, 1).to(torch.int32)
        s["freqs"] = [[10000.0 ** (-2.0 * i / n) for i in range(n // 2)] for n in _rotated(case)]
        if own:
            from lightly_trian_quant_b200 import ops

            s["table"] = ops.RopeTable(s["freqs"], case["head_dim"], interleaved=case["interleaved"])
        else:
            s["freq"] = torch.tensor([f for fs in s["freqs"] for f in fs], dtype=torch.float64, device="cuda")
            s["axis"] = torch.tensor([a for a, fs in enumerate(s["freqs"]) for _ in fs], device="cuda")
    else:
        dt, R, w = DTYPES[case["dtype"]], case["rows"], case["width"]
        channel = torch.where(torch.rand(w, generator=g, device="cuda") < 0.01, 20.0, 1.0)     # a few channels of a residual stream are far larger
        s["x"] = (_rand(g, R, w) * channel + _rand(g, R, 1, scale=0.5)).to(dt)
        s["w"], s["b"] = 1.0 + _rand(g, w, scale=0.2), _rand(g, w, scale=0.1)
        s["eps"] = 1e-5
        if case["train"]:
            s["dy"] = _rand(g, R, w, dtype=DTYPES[case["out"]])
            s["dres"] = _rand(g, R, w, dtype=dt) if case["residual"] else None
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _visible(lq, lk, s, pre):
    """which keys (columns) each query (row) of a sequence sees, and how far they are from it"""
    at = torch.arange(lq, device="cuda")[:, None] + (lk - lq)
    key = torch.arange(lk, device="cuda")[None, :]
    seen = (key <= at) | (key < pre) if s["causal"] else torch.ones(lq, lk, dtype=torch.bool, device="cuda")
    return seen, (at - key).abs().float()


def _plain_attention(s):
    ql, kl = s["lens"]
    h, hk = s["heads"], s["kv_heads"]
    share = h // hk
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    lse = torch.empty(h, q.shape[0], device="cuda")
    if s["train"]:
        dq = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        dk, dv = torch.empty(k.shape, dtype=k.dtype, device="cuda"), torch.empty(v.shape, dtype=v.dtype, device="cuda")
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        seen, far = _visible(lq, lk, s, min(s["prefix"], lk))
        rq, rk = slice(q0, q0 + lq), slice(k0, k0 + lk)
        for g in range(hk):                              # a key head and the query heads that share it
            hs = slice(g * share, (g + 1) * share)
            qg = q[rq, hs].float().transpose(0, 1)       # [share, lq, 64]
            kg, vg = k[rk, g].float(), v[rk, g].float()
            score = qg @ kg.t() * s["scale"]
            if s["cap"]:
                bent = torch.tanh(score / s["cap"])
                score = bent * s["cap"]
            if s["slopes"] is not None:
                score = score - s["slopes"][hs, None, None] * far
            score = score.masked_fill(~seen, float("-inf"))
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - top)
            norm = p.sum(-1, keepdim=True)
            p = p / norm
            og = p @ vg
            out[rq, hs] = og.transpose(0, 1).to(out.dtype)
            lse[hs, rq] = (top + torch.log(norm))[..., 0]
            if s["train"]:
                dg = s["dout"][rq, hs].float().transpose(0, 1)
                dv[rk, g] = (p.transpose(1, 2) @ dg).sum(0).to(dv.dtype)
                ds = p * (dg @ vg.t() - (dg * og).sum(-1, keepdim=True))
                if s["cap"]:
                    ds = ds * (1 - bent * bent)
                ds = ds * s["scale"]
                dq[rq, hs] = (ds @ kg).transpose(0, 1).to(dq.dtype)
                dk[rk, g] = (ds.transpose(1, 2) @ qg).sum(0).to(dk.dtype)
        q0 += lq
        k0 += lk
    return (out, lse, dq, dk, dv) if s["train"] else (out, lse)


def _turn(x, cos, sin, interleaved):
    n = 2 * cos.shape[-1]
    y = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :n // 2], y[..., n // 2:n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., n:]), -1).to(x.dtype)


def _plain_rope(s):
    angle = s["pos"].double()[:, s["axis"]] * s["freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    y = _turn(s["x"], cos, sin, s["interleaved"])
    return (y, _turn(s["dy"], cos, -sin, s["interleaved"])) if s["train"] else (y,)


def _plain_norm(s):
    x = s["x"].float()
    mid = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((mid * mid).mean(-1, keepdim=True) + s["eps"])
    xh = mid * rstd
    y = (xh * s["w"] + s["b"]).to(DTYPES[s["out"]])
    if not s["train"]:
        return (y,)
    dy = s["dy"].float()
    g = dy * s["w"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return y, dx.to(s["x"].dtype), (dy * xh).double().sum(0).float(), dy.double().sum(0).float()


# ------------------------------------------------------------------------------------------------ the package's operators
def _own(s):
    from lightly_trian_quant_b200 import ops

    if s["kind"] == "attention":
        how = dict(scale=s["scale"], cap=s["cap"], slopes=s["slopes"])
        out, lse = ops.attn_packed(s["q"], s["k"], s["v"], s["plan"], **how)
        if not s["train"]:
            return out, lse
        return (out, lse, *ops.attn_packed_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, s["plan"], **how))
    if s["kind"] == "rope":
        y = ops.rope_axes(s["x"], s["pos"], s["table"])
        return (y, ops.rope_axes(s["dy"], s["pos"], s["table"], inverse=True)) if s["train"] else (y,)
    y, mean, rstd = ops.layer_norm_fwd(s["x"], s["w"], s["b"], s["eps"], DTYPES[s["out"]])
    return (y, *ops.layer_norm_bwd(s["dy"], s["x"], s["w"], mean, rstd, dres=s["dres"])) if s["train"] else (y,)


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "rope": _plain_rope, "norm": _plain_norm}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(s):
    """softmax over the visible keys head by head, its gradients by differentiation"""
    parts = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["heads"], s["q"].shape[0], dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for lq, lk in zip(*s["lens"]):
        rows, cols = torch.meshgrid(torch.arange(lk - lq, lk, device="cuda"), torch.arange(lk, device="cuda"), indexing="ij")
        hidden = (cols > rows) & (cols >= min(s["prefix"], lk)) if s["causal"] else None
        for h in range(s["heads"]):
            g = h * s["kv_heads"] // s["heads"]
            q = s["q"][q0:q0 + lq, h].double().requires_grad_(s["train"])
            k = s["k"][k0:k0 + lk, g].double().requires_grad_(s["train"])
            v = s["v"][k0:k0 + lk, g].double().requires_grad_(s["train"])
            score = torch.einsum("id,jd->ij", q, k) * s["scale"]
            if s["cap"]:
                score = s["cap"] * torch.tanh(score / s["cap"])
            if s["slopes"] is not None:
                score = score - s["slopes"][h].double() * (rows - cols).abs()
            if hidden is not None:
                score = torch.where(hidden, float("-inf"), score)
            z = torch.logsumexp(score, -1)
            o = torch.exp(score - z[:, None]) @ v
            out[q0:q0 + lq, h], lse[h, q0:q0 + lq] = o.detach(), z.detach()
            if s["train"]:
                grads = torch.autograd.grad(o, (q, k, v), s["dout"][q0:q0 + lq, h].double())
                parts["q"][q0:q0 + lq, h] += grads[0]
                parts["k"][k0:k0 + lk, g] += grads[1]
                parts["v"][k0:k0 + lk, g] += grads[2]
        q0 += lq
        k0 += lk
    return (out, lse, parts["q"], parts["k"], parts["v"]) if s["train"] else (out, lse)


def _exact_rope(s):
    """channel pairs as complex numbers, turned by a unit number"""
    pairs = sum(len(fs) for fs in s["freqs"])
    turn = torch.cat([torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                  s["pos"][:, a:a + 1].double() * torch.tensor(fs, dtype=torch.float64, device="cuda")) for a, fs in enumerate(s["freqs"]) if fs], -1)[:, None]

    def apply(x, unit):
        y = x.double()
        head = y[..., :2 * pairs]
        z = head.unflatten(-1, (pairs, 2)) if s["interleaved"] else head.unflatten(-1, (2, pairs)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * unit)
        return torch.cat(((z if s["interleaved"] else z.transpose(-1, -2)).flatten(-2), y[..., 2 * pairs:]), -1)

    y = apply(s["x"], turn)
    return (y, apply(s["dy"], turn.conj())) if s["train"] else (y,)


def _exact_norm(s):
    x = s["x"].double().requires_grad_(s["train"])
    w, b = s["w"].double().requires_grad_(s["train"]), s["b"].double().requires_grad_(s["train"])
    y = (x - x.mean(1, keepdim=True)) / (x.var(1, unbiased=False, keepdim=True) + s["eps"]).sqrt() * w + b
    if not s["train"]:
        return (y,)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return y.detach(), dx if s["dres"] is None else dx + s["dres"].double(), dw, db


@torch.enable_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rope": _exact_rope, "norm": _exact_norm}[case["kind"]](s)
