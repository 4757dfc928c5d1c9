"""Attention over packed sequences and its gradients against float64.

Tolerances.  u = eps / 2 of the 16-bit type.  The kernels round P and dS to 16 bits (the products' operand) and each result once; the rest is fp32.
A rounding is off by at most u |x|, with a standard deviation of at most u |x| / sqrt(3); sums of independent roundings add as squares, so
6 standard deviations of sum_j r_j x_j v_j are 6 / sqrt(3) u sqrt(sum x_j^2 v_j^2) < 3.5 u sqrt(...).  The fp32 part is bounded outright: the exponent of
a score is off by E = 2^-24 (72 sum_c |q_c k_c| scale + 8 |s| + 4 cap) + 4e-6 (accumulation, scaling, exponentials' 2.7e-6), and so P by the factor E.
delta = rowsum(dO * O) takes the rounded output: off by 3.5 u sqrt(sum (dO O)^2) for the whole row.  Numbers below the 16-bit type's normal range are
off by half its smallest step.  Below 2^-126 the exponential gives 0 (ex2.ftz) or stops falling (the polynomial's clamp), and products of fp32 numbers may
be flushed: P and dS are off by up to 2^-126 besides, which for a key 97 steps of slope 0.9 away from any query (P = e^-87.3 = 2^-126) is more than half a
step of bf16 below its normal range, 2^-134: with |dP - delta| about 15, |Q| 3 and 1/8 for the scale 2^-126 * 6 = 7e-38 where 3.5 * 2^-134 * sqrt(201) =
2.3e-39 was allowed."""
import math

import pytest
import torch

from oracle import train_oracle as to

gpu = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _ops():
    from lightly_trian_quant_b200 import ops

    return ops


def _rms(x, dim):
    return (x * x).sum(dim).sqrt()


def reference(q, k, v, do, q_lens, k_lens, causal, prefix, scale, cap, slopes, dtype):
    """-> {name: (value, bound)} in float64 on the operands' device, rows of no sequence left out of the comparison (NaN bound)"""
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    dev, share = q.device, q.shape[1] // k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    val = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    var = {n: torch.zeros_like(t) for n, t in val.items()}            # squares of the independent roundings, in units of (3.5)^2
    hard = {n: torch.full_like(t, float("nan")) for n, t in val.items()}
    val["lse"], hard["lse"] = torch.zeros(q.shape[1], q.shape[0], dtype=torch.float64, device=dev), torch.full((q.shape[1], q.shape[0]), float("nan"), dtype=torch.float64, device=dev)
    q0 = k0 = 0
    for d, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        rq, rk = slice(q0, q0 + lq), slice(k0, k0 + lk)
        for n, r in (("out", rq), ("dq", rq), ("dk", rk), ("dv", rk)):
            hard[n][r] = 0
        hard["lse"][:, rq] = 0
        sees = to.attn_sees(lq, lk, causal, prefix[d] if prefix else 0).to(dev)
        far = (torch.arange(lq, device=dev)[:, None] + (lk - lq) - torch.arange(lk, device=dev)[None]).abs()
        for h in range(q.shape[1]):
            g = h // share
            Q, K, V, dO = q[rq, h], k[rk, g], v[rk, g], do[rq, h]
            raw = Q @ K.t() * scale
            s = cap * torch.tanh(raw / cap) if cap else raw
            slope = (1 - (s / cap) ** 2) if cap else torch.ones_like(s)
            if slopes is not None:
                s = s - slopes[h].double() * far
            s = s.masked_fill(~sees, -math.inf)
            z = torch.logsumexp(s, -1, keepdim=True) if lk else s.new_full((lq, 1), -math.inf)
            p = torch.where(sees, torch.exp(s - z), 0.0)
            E = 2.0 ** -24 * (72 * (Q.abs() @ K.abs().t()) * scale + 8 * s.masked_fill(~sees, 0).abs() + 4 * cap) + 4e-6
            o = p @ V
            val["out"][rq, h], val["lse"][h, rq] = o, z[:, 0]
            pe = p * (E + (p * E).sum(-1, keepdim=True)) + 2.0 ** -126 * sees
            var["out"][rq, h] = u * u * ((p * p) @ (V * V) + o * o) + tiny ** 2 * (1 + (V * V).sum(0))
            hard["out"][rq, h] = pe @ V.abs()
            hard["lse"][h, rq] = (p * E).sum(-1) + 2.0 ** -22 * (1 + z[:, 0].abs().nan_to_num(posinf=0))
            delta = (dO * o).sum(-1, keepdim=True)
            dp = dO @ V.t()
            ds = p * (dp - delta) * slope
            dv, dq, dk = p.t() @ dO, ds @ K * scale, ds.t() @ Q * scale
            val["dv"][rk, g] += dv
            val["dq"][rq, h] = dq
            val["dk"][rk, g] += dk
            d_delta = u * _rms(dO * o, -1)[:, None]
            # fp32: P off by E, dp and delta by 64 steps of their sums of sizes, the cap's factor by 2^-20
            dse = pe * (dp - delta).abs() + p * 2.0 ** -24 * 72 * (dO.abs() @ V.abs().t() + (dO * o).abs().sum(-1, keepdim=True)) + (ds.abs() * 2.0 ** -20 + 2.0 ** -126) + pe * (dO.abs() * (pe @ V.abs())).sum(-1, keepdim=True)
            one = p * slope * d_delta                                  # the same error for the whole row: adds up along it
            var["dv"][rk, g] += u * u * (p * p).t() @ (dO * dO) + tiny ** 2 * (dO * dO).sum(0)
            hard["dv"][rk, g] += pe.t() @ dO.abs()
            var["dq"][rq, h] = scale ** 2 * (u * u * (ds * ds) @ (K * K) + (one @ K) ** 2 + tiny ** 2 * (K * K).sum(0)) + u * u * dq * dq + tiny ** 2
            hard["dq"][rq, h] = scale * (dse @ K.abs())
            var["dk"][rk, g] += scale ** 2 * (u * u * (ds * ds).t() @ (Q * Q) + (one * one).t() @ (Q * Q) + tiny ** 2 * (Q * Q).sum(0))
            hard["dk"][rk, g] += scale * (dse.t() @ Q.abs())
        q0, k0 = q0 + lq, k0 + lk
    for n in ("dk", "dv"):
        var[n] += u * u * val[n] ** 2 + tiny ** 2
    return {n: (val[n], 3.5 * (var[n].sqrt() if n in var else 0) + hard[n]) for n in val}


def close(got, ref, names):
    for name, t in zip(names, got):
        value, bound = ref[name]
        used = ~bound.isnan()
        t = t.double()
        none = used & value.isinf()
        assert torch.equal(t[none], value[none]), name
        m = used & ~none
        assert torch.isfinite(t[m]).all(), name
        if m.any():
            worst = ((t - value).abs()[m] / bound[m].clamp_min(1e-300)).max().item()
            assert worst <= 1, (name, worst)


def case(q_lens, k_lens, Hq, Hk, dtype, seed, sharp=1.3, rows_behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Tq, Tk = sum(q_lens) + rows_behind, sum(k_lens) + rows_behind
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (r(Tq, Hq, 64) * sharp).to(dtype), r(Tk, Hk, 64).to(dtype), r(Tk, Hk, 64).to(dtype), r(Tq, Hq, 64).to(dtype)


def run(q, k, v, do, plan, **how):
    ops = _ops()
    out, lse = ops.attn_packed(q, k, v, plan, **how)
    ops.check_device_error()
    grads = ops.attn_packed_bwd(do, q, k, v, out, lse, plan, **how)
    ops.check_device_error()
    return (out, lse, *grads)


NAMES = ("out", "lse", "dq", "dk", "dv")
LENS = [[1], [2, 1], [128], [127, 1, 0, 129, 128], [96, 97, 95, 33], [300, 77, 513], [64, 65, 191, 192, 193]]


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2)])
@pytest.mark.parametrize("lens", LENS, ids=lambda n: "-".join(map(str, n)))
def test_document_mask(lens, heads, dtype):
    ops = _ops()
    q, k, v, do = case(lens, lens, *heads, dtype, sum(lens))
    got = run(q, k, v, do, ops.AttnPlan(lens))
    close(got, reference(q, k, v, do, lens, lens, False, None, 0.125, 0.0, None, dtype), NAMES)


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("prefix", [None, 0, 5, 130])
@pytest.mark.parametrize("lens", LENS[1:], ids=lambda n: "-".join(map(str, n)))
def test_causal_and_prefix(lens, prefix, dtype):
    ops = _ops()
    pre = None if prefix is None else [min(prefix, n) for n in lens]
    q, k, v, do = case(lens, lens, 3, 3, dtype, sum(lens) + 1)
    got = run(q, k, v, do, ops.AttnPlan(lens, causal=True, prefix=pre))
    close(got, reference(q, k, v, do, lens, lens, True, pre, 0.125, 0.0, None, dtype), NAMES)


CROSS = [([5, 200, 1], [300, 96, 1]), ([130, 3, 40], [3, 130, 0]), ([0, 7, 0], [9, 0, 4]), ([257, 129], [129, 257]), ([0], [5]), ([5], [0])]


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("causal,prefix", [(False, 0), (True, 0), (True, 4)])
@pytest.mark.parametrize("lens", CROSS, ids=str)
def test_queries_and_keys_of_different_lengths(lens, causal, prefix, dtype):
    """more queries than keys (the first see nothing under a causal mask), sequences without queries or without keys"""
    ops = _ops()
    ql, kl = lens
    pre = [min(prefix, n) for n in kl] if prefix else None
    q, k, v, do = case(ql, kl, 4, 2, dtype, 7)
    got = run(q, k, v, do, ops.AttnPlan(ql, kl, causal=causal, prefix=pre))
    close(got, reference(q, k, v, do, ql, kl, causal, pre, 0.125, 0.0, None, dtype), NAMES)


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap,bias", [(20.0, False), (1.5, False), (0.0, True), (50.0, True)])
def test_cap_and_distance(cap, bias, causal, dtype):
    """capped scores (also where most of them reach the cap) and a bias by distance, steep and flat, with shared key heads and another scale"""
    ops = _ops()
    lens, pre = [261, 1, 97, 450], [5, 0, 97, 130]
    slopes = torch.tensor([0.5, 0.01, 0.0, 2.0, -0.02, 0.125], device="cuda") if bias else None
    q, k, v, do = case(lens, lens, 6, 2, dtype, 11, sharp=2.5)
    how = dict(scale=0.2, cap=cap, slopes=slopes)
    got = run(q, k, v, do, ops.AttnPlan(lens, causal=causal, prefix=pre if causal else None), **how)
    close(got, reference(q, k, v, do, lens, lens, causal, pre if causal else None, 0.2, cap, slopes, dtype), NAMES)


@gpu
@pytest.mark.parametrize("cap", [1e-12, 1e-3, 1e6])
def test_caps_at_the_ends_of_their_range(cap):
    """a cap that leaves no score (P is uniform over the keys a query sees, and q, k have next to no gradient), and one that changes none"""
    ops = _ops()
    lens = [130, 33]
    q, k, v, do = case(lens, lens, 2, 1, BF, 3)
    q[5] = 0
    out, lse, dq, dk, dv = run(q, k, v, do, ops.AttnPlan(lens), cap=cap)
    close((out, lse, dv), reference(q, k, v, do, lens, lens, False, None, 0.125, cap, None, BF), ("out", "lse", "dv"))
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
def test_images_of_several_sizes(dtype):
    """more items than CTAs, of one to many tiles"""
    ops = _ops()
    lens = [1605, 261, 77, 1029, 1, 1605, 517]
    q, k, v, do = case(lens, lens, 8, 4, dtype, 5)
    close(run(q, k, v, do, ops.AttnPlan(lens)), reference(q, k, v, do, lens, lens, False, None, 0.125, 0.0, None, dtype), NAMES)


@gpu
def test_many_short_sequences():
    ops = _ops()
    lens = [i % 7 for i in range(700)]
    q, k, v, do = case(lens, lens, 2, 1, BF, 6)
    close(run(q, k, v, do, ops.AttnPlan(lens, causal=True)), reference(q, k, v, do, lens, lens, True, None, 0.125, 0.0, None, BF), NAMES)


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lo", [64, 96, 288])
def test_scores_that_grow_along_the_keys(lo, dtype):
    """keys whose scores exceed the maximum of the first ones by far more than 2^15 in the exponent's domain, next to rows that stay flat"""
    ops = _ops()
    lens = [453, 300]
    q, k, v, do = case(lens, lens, 2, 2, dtype, 3)
    k[lo:lo + 32] *= 12
    q[::4] *= 0.05
    close(run(q, k, v, do, ops.AttnPlan(lens)), reference(q, k, v, do, lens, lens, False, None, 0.125, 0.0, None, dtype), NAMES)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("causal", [False, True])
def test_what_lies_outside_a_sequence_is_not_seen(causal, bad):
    """rows behind the last sequence, and whole other sequences, hold NaN or infinities: the finite sequences next to them come out as without them, and the rows
    of outputs given by the caller that belong to no sequence stay as they were"""
    ops = _ops()
    lens = [70, 131, 45, 200, 3]
    q, k, v, do = case(lens, lens, 2, 2, BF, 9, rows_behind=150)
    plan = ops.AttnPlan(lens, causal=causal)
    want = run(q, k, v, do, plan)
    ends = torch.tensor([0, *lens]).cumsum(0).tolist()
    used = [t.clone() for t in (q, k, v, do)]
    for t in used:
        t[ends[1]:ends[2]] = bad                                    # the second sequence
        t[ends[5]:] = bad
    outs = [torch.full_like(t, 7) for t in (q, q, k, v)]
    out, lse = ops.attn_packed(*used[:3], plan, out=outs[0])
    dq, dk, dv = ops.attn_packed_bwd(used[3], *used[:3], out, lse, plan, grads=tuple(outs[1:]))
    ops.check_device_error()
    assert out is outs[0] and dq is outs[1] and dk is outs[2] and dv is outs[3]
    rows = torch.ones(ends[5], dtype=torch.bool)
    rows[ends[1]:ends[2]] = False
    rows = rows.nonzero().flatten().cuda()
    for a, b in zip((out, dq, dk, dv), (want[0], *want[2:])):
        assert torch.equal(a[rows], b[rows])
        assert (a[ends[5]:] == 7).all() and not b[ends[5]:].any()
    assert torch.equal(lse[:, rows], want[1][:, rows]) and not want[1][:, ends[5]:].any()


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
def test_strides(dtype):
    """operands that are parts of one projection ([T, heads, 64] and [heads, T, 64] layouts), gradients written into the parts of one tensor"""
    ops = _ops()
    lens, Hq, Hk = [130, 261, 9], 4, 2
    T = sum(lens)
    q, k, v, do = case(lens, lens, Hq, Hk, dtype, 21)
    plan = ops.AttnPlan(lens, causal=True)
    want = run(q, k, v, do, plan)
    qkv = torch.cat((q, k, v), 1)
    parts = (qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:])
    out, lse = ops.attn_packed(*parts, plan)
    dqkv = torch.zeros_like(qkv)
    gparts = (dqkv[:, :Hq], dqkv[:, Hq:Hq + Hk], dqkv[:, Hq + Hk:])
    ops.attn_packed_bwd(do, *parts, out, lse, plan, grads=gparts)
    for a, b in zip((out, lse, *gparts), want):
        assert torch.equal(a, b)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]           # head-major
    o8 = torch.zeros(Hq * 64 * T + 8, dtype=dtype, device="cuda")[8:].view(T, Hq, 64)       # 16- but not 32-byte aligned
    out, lse = ops.attn_packed(*hm[:3], plan, out=o8)
    for a, b in zip((out, lse, *ops.attn_packed_bwd(hm[3], *hm[:3], out, lse, plan)), want):
        assert torch.equal(a, b)
    ops.check_device_error()


@gpu
def test_gradients_by_differences():
    """dq, dk, dv against central differences of the float64 oracle along random directions (the formulas, independent of the ones above)"""
    ops = _ops()
    lens, pre = [33, 150], [4, 20]
    q, k, v, do = case(lens, lens, 2, 1, F16, 33)
    slopes = torch.tensor([0.05, 0.3], device="cuda")
    got = run(q, k, v, do, ops.AttnPlan(lens, causal=True, prefix=pre), cap=8.0, slopes=slopes)
    f = lambda *t: (to.attn(*t, lens, lens, causal=True, prefix=pre, cap=8.0, slopes=slopes.cpu())[0] * do.double().cpu()).sum()  # noqa: E731
    ref = reference(q, k, v, do, lens, lens, True, pre, 0.125, 8.0, slopes, F16)
    ops64 = [t.double().cpu() for t in (q, k, v)]
    g = torch.Generator().manual_seed(1)
    for i, name in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            step = torch.randn(ops64[i].shape, generator=g, dtype=torch.float64)
            at = lambda e: f(*[t + e * step if n == i else t for n, t in enumerate(ops64)])  # noqa: E731
            slope = (at(1e-4) - at(-1e-4)) / 2e-4                      # third derivatives are of size 1: 1e-8 of the value's size
            here = (got[2 + i].double().cpu() * step).sum()
            bound = (ref[name][1].cpu() ** 2 * step ** 2).sum().sqrt() * 2 + 1e-6 * (step.abs() * ref[name][0].cpu().abs()).sum()
            assert (slope - here).abs() <= bound, (name, slope, here, bound)


@gpu
def test_the_same_bits_from_run_to_run_in_graphs_and_on_other_streams():
    ops = _ops()
    lens = [300, 77, 513]
    q, k, v, do = case(lens, lens, 4, 2, BF, 2)
    plan = ops.AttnPlan(lens, causal=True)
    want = run(q, k, v, do, plan, cap=15.0)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = run(q, k, v, do, plan, cap=15.0)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    graphs = []
    for _ in range(2):                                              # two graphs alive at once, replayed in turn and on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = ops.attn_packed(q, k, v, plan, cap=15.0)
            res = (out, lse, *ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=15.0))
        graphs.append((graph, res))
    for _ in range(3):
        for i, (graph, res) in enumerate(graphs):
            for t in res:
                t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for graph, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want))
    ops.check_device_error()


@gpu
def test_workspace_is_checked_by_the_call():
    from lightly_trian_quant_b200 import _lib

    L, p = _lib.lib(), _lib.AttnPackParams()
    p.dtype, p.Hq, p.Hk, p.n_q_tiles, p.n_k_tiles, p.scale, p.Tq, p.Tk = 1, 4, 2, 1, 1, 0.125, 40, 40
    p.q_tiles = p.k_tiles = p.lse = p.ws = 4096                     # never dereferenced: the calls end on the host
    for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        setattr(p, n, _lib.Heads(4096, 256, 64))
    need = L.kf_attn_pack_ws_bytes(4, 2, 1, 1)
    assert need >= 2 * 4 * 128 * 4
    for size, at in ((need - 1, 4096), (need, None), (need, 4112)):
        p.ws_bytes, p.ws = size, at
        assert L.kf_attn_pack_bwd(p, None) == -1 and "workspace" in L.kf_last_error_string().decode()


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("heads", [(3, 1), (8, 2), (2, 2)])
def test_shared_key_heads_with_few_and_many_items(heads, dtype):
    """an item per query head and their sums joined (few tiles), an item per key head (many tiles): both against the same reference"""
    ops = _ops()
    for lens in ([200, 37], [130] * 160):
        q, k, v, do = case(lens, lens, *heads, dtype, 77)
        close(run(q, k, v, do, ops.AttnPlan(lens, causal=True)), reference(q, k, v, do, lens, lens, True, None, 0.125, 0.0, None, dtype), NAMES)


@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True), (50.0, True)])
@pytest.mark.parametrize("q_lens,k_lens,causal,prefix", [([200], [1605], False, None), ([1], [4101], False, None), ([1], [97], True, None), ([261], [261], True, None), ([700], [700], True, [5]),
                                                         ([130, 1, 40], [96, 300, 0], False, None), ([500, 3], [200, 97], True, None), ([300], [193], True, [193]),
                                                         ([130, 1, 40], [960, 1300, 0], False, None), ([500, 3], [1200, 97], True, None), ([1300], [900], True, [7]), ([900], [901], True, None)], ids=str)
def test_few_queries_share_their_keys_among_ctas(q_lens, k_lens, causal, prefix, cap, bias, dtype):
    """items so few that each is split along its keys, and the same ones unsplit: parts of several tiles and of none, rows that see nothing of a part or at all"""
    ops = _ops()
    q, k, v, do = case(q_lens, k_lens, 4, 2, dtype, 31)
    slopes = torch.tensor([0.0, 0.01, 0.1, 0.9], device="cuda") if bias else None
    ref = reference(q, k, v, do, q_lens, k_lens, causal, prefix, 0.125, cap, slopes, dtype)
    plan = ops.AttnPlan(q_lens, k_lens, causal=causal, prefix=prefix)
    assert plan.longest == max(k_lens)
    close(run(q, k, v, do, plan, cap=cap, slopes=slopes), ref, NAMES)
    plan.longest = 0                                              # not known: no split
    close(run(q, k, v, do, plan, cap=cap, slopes=slopes), ref, NAMES)


@gpu
def test_refusals():
    ops = _ops()
    q, k, v, do = case([40], [40], 4, 2, BF, 1)
    plan = ops.AttnPlan([40])
    out, lse = ops.attn_packed(q, k, v, plan)
    f = lambda *a, **kw: (lambda: ops.attn_packed(*a, **kw))  # noqa: E731
    b = lambda *a, **kw: (lambda: ops.attn_packed_bwd(*a, **kw))  # noqa: E731
    odd = torch.zeros(40 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(40, 4, 64)
    narrow = torch.zeros(40, 4, 65, dtype=BF, device="cuda")[..., :64]
    for bad in (f(q.float(), k, v, plan), f(q.half(), k, v, plan), f(q.cpu(), k, v, plan), f(q, k.cpu(), v, plan), f(q[:, :3], k, v, plan), f(q[..., :32], k[..., :32], v[..., :32], plan),
                f(q[:39], k, v, plan), f(q, k[:39], v[:39], plan), f(q, k, v[:39], plan), f(q, k, v, plan, scale=0.0), f(q, k, v, plan, scale=-1.0), f(q, k, v, plan, scale=float("nan")),
                f(q, k, v, plan, cap=-1.0), f(q, k, v, plan, cap=float("inf")), f(q, k, v, plan, slopes=torch.zeros(3, device="cuda")), f(q, k, v, plan, slopes=torch.zeros(4, device="cuda").half()),
                f(q, k, v, ops.AttnPlan([40], device="cpu")), f(odd, k, v, plan), f(narrow, k, v, plan), f(q[:1].expand(40, 4, 64), k, v, plan), f(q, k, v, plan, out=out.float()),
                f(q, k, v, plan, out=out[:20]), f(q, k, v, plan, out=out[:1].expand(40, 4, 64)), f(q.transpose(0, 2), k, v, plan), b(do[:20], q, k, v, out, lse, plan),
                b(do.float(), q, k, v, out, lse, plan), b(do[:, :1].expand(40, 4, 64), q, k, v, out, lse, plan), b(do, q, k, v, out, lse[:2], plan), b(do, q, k, v, out, lse.double(), plan),
                b(do, q, k, v, out[:20], lse, plan), b(do, q, k, v, out, lse, plan, grads=(None, q, None))):
        with pytest.raises(ops.KfError):
            bad()
    ops.check_device_error()
    assert torch.equal(ops.attn_packed(q, k, v, plan)[0], out)


@gpu
def test_outputs_that_overlap_what_is_read():
    """refused, while parts of one buffer that lie between one another without a common byte are taken"""
    ops = _ops()
    q, k, v, do = case([40], [40], 4, 2, BF, 1)
    plan = ops.AttnPlan([40])
    out, lse = ops.attn_packed(q, k, v, plan)
    want = ops.attn_packed_bwd(do, q, k, v, out, lse, plan)
    flat, both = torch.zeros(45 * 8 * 64, dtype=BF, device="cuda"), torch.zeros(40, 8, 64, dtype=BF, device="cuda")
    both[:, :4], both[:, 4:6], both[:, 6:] = q, k, v
    bq, bk, bv = both[:, :4], both[:, 4:6], both[:, 6:]
    overlapping = flat.as_strided((40, 4, 64), (64, 64, 1))
    shifted = flat[32 * 64:].as_strided((40, 4, 64), (512, 64, 1))
    f = lambda o, q=q, k=k, v=v: (lambda: ops.attn_packed(q, k, v, plan, out=o))  # noqa: E731
    b = lambda *g: (lambda: ops.attn_packed_bwd(do, q, k, v, out, lse, plan, grads=g))  # noqa: E731
    for bad in (f(q), f(both[:, 3:7], bq, bk, bv), f(both[:, 4:], bq, bk, bv), f(overlapping), b(q, None, None), b(do, None, None), b(out, None, None),
                b(None, k, None), b(None, None, v), b(None, want[1], want[1]), b(flat.as_strided((40, 4, 64), (512, 64, 1)), both[:, :2], both[:, 1:3]),
                b(shifted, flat[33 * 64:].as_strided((40, 2, 64), (512, 64, 1)), None)):
        with pytest.raises(ops.KfError):
            bad()
    # heads of q, k and v in turn, gradients side by side, an output in the columns that the call does not read
    turn = torch.zeros(40, 4, 2, 64, dtype=BF, device="cuda")
    turn[:, :, 0] = q
    assert torch.equal(ops.attn_packed(turn[:, :, 0], k, v, plan, out=turn[:, :, 1])[0], out)
    side = torch.zeros(40, 8, 64, dtype=BF, device="cuda")
    got = ops.attn_packed_bwd(do, bq, bk, bv, out, lse, plan, grads=(side[:, :4], side[:, 4:6], side[:, 6:]))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # key rows of one tensor behind the query rows of another: extents side by side
    assert torch.equal(ops.attn_packed(q, k, v, plan, out=flat[:40 * 256].view(40, 4, 64))[0], out)
    ops.check_device_error()


def test_plan_says_who_sees_whom():
    """the tables of random batches, expanded to (query, key) pairs, are the masks; slots number the query tiles along the rows"""
    import random

    ops = _ops()
    r = random.Random(0)
    sizes = [0, 1, 5, 127, 128, 129, 300]
    for _ in range(60):
        n = r.randint(0, 5)
        lq = [r.choice(sizes) for _ in range(n)]
        lk = [r.choice(sizes) for _ in range(n)] if r.random() < 0.6 else None
        causal = r.random() < 0.7
        pre = [r.randint(0, a) for a in (lk or lq)] if causal and r.random() < 0.7 else None
        plan = ops.AttnPlan(lq, lk, causal=causal, prefix=pre, device="cpu")
        want = torch.zeros(sum(lq), sum(lk or lq), dtype=torch.bool)
        q0 = k0 = 0
        for d, (a, b) in enumerate(zip(lq, lk or lq)):
            want[q0:q0 + a, k0:k0 + b] = to.attn_sees(a, b, causal, pre[d] if pre else 0)
            q0, k0 = q0 + a, k0 + b
        seen, slots = torch.zeros_like(want), {}
        for row, rows, k_row, k_len, pos, prefix, slot, _ in plan.q_tiles.tolist():
            slots[slot] = (row, rows)
            for i in range(rows):
                seen[row + i, k_row:k_row + min(max(pos + i + 1, prefix, 0), k_len)] = True
        assert torch.equal(seen, want) and sorted(slots) == list(range(len(slots)))
        seen = torch.zeros_like(want)
        for row, rows, q_row, q_len, first, off, prefix, slot0 in plan.k_tiles.tolist():
            for t in range(-(-q_len // 128)):
                assert slots[slot0 + t] == (q_row + 128 * t, min(128, q_len - 128 * t))
            for i in range(rows):
                seen[q_row + (0 if first + i < prefix else min(max(first + i - off, 0), q_len)):q_row + q_len, row + i] = True
        assert torch.equal(seen, want)


def test_plan_refusals():
    ops = _ops()
    for bad in (lambda: ops.AttnPlan([1, -1], device="cpu"), lambda: ops.AttnPlan([1], [1, 2], device="cpu"), lambda: ops.AttnPlan([4], prefix=[2], device="cpu"),
                lambda: ops.AttnPlan([4], causal=True, prefix=[5], device="cpu"), lambda: ops.AttnPlan([4], causal=True, prefix=[1, 1], device="cpu"),
                lambda: ops.AttnPlan([2**31], device="cpu"), lambda: ops.AttnPlan([4], causal=True, prefix=[-1], device="cpu")):
        with pytest.raises(ops.KfError):
            bad()
    assert ops.AttnPlan([], device="cpu").q_tiles.shape == (0, 8)


def test_host_checks_of_the_packed_attention():
    """bad arguments end as a status with a message before any launch; the mirror of the parameter block is the header's"""
    from lightly_trian_quant_b200 import _lib

    L = _lib.lib()
    msg = lambda: L.kf_last_error_string().decode()  # noqa: E731

    def params(**kw):
        p = _lib.AttnPackParams()
        p.dtype, p.Hq, p.Hk, p.n_q_tiles, p.n_k_tiles, p.scale, p.Tq, p.Tk = 1, 4, 2, 1, 1, 0.125, 40, 40
        p.q_tiles = p.k_tiles = p.lse = p.ws = 4096
        p.ws_bytes = 1 << 20
        for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
            setattr(p, n, _lib.Heads(4096, 256, 64))
        for n, x in kw.items():
            setattr(p, n, x)
        return p

    H = _lib.Heads
    for kw, text in ((dict(dtype=0), "dtype"), (dict(Hk=3), "share"), (dict(Hk=0), "share"), (dict(scale=0.0), "scale"), (dict(cap=-1.0), "cap"), (dict(Tq=1 << 31), "rows"),
                     (dict(n_q_tiles=1 << 29), "items"), (dict(q_tiles=None), "null"), (dict(q=H(4098, 256, 64)), "aligned"), (dict(q=H(None, 256, 64)), "non-null"),
                     (dict(k=H(4096, 252, 64)), "strides of k"), (dict(v=H(4096, 0, 64)), "strides of v"), (dict(o=H(4096, 256, 8)), "strides of o")):
        for call in (L.kf_attn_pack_fwd, L.kf_attn_pack_bwd):
            assert call(params(**kw), None) == -1 and text in msg(), (kw, msg())
    assert L.kf_attn_pack_bwd(params(dk=H(4096, 256, 63)), None) == -1 and "strides of dk" in msg()
    assert L.kf_attn_pack_fwd(params(n_q_tiles=0), None) == 0 and L.kf_attn_pack_bwd(params(n_q_tiles=0, n_k_tiles=0), None) == 0
    assert L.kf_attn_pack_ws_bytes(0, 1, 3, 3) == -1 and L.kf_attn_pack_ws_bytes(4, 3, 3, 3) == -1 and L.kf_attn_pack_ws_bytes(4, 2, -1, 3) == -1


def test_mirrors_match_the_header(tmp_path):
    import ctypes as C
    import subprocess
    from pathlib import Path

    from lightly_trian_quant_b200 import _lib

    inc = Path(__file__).resolve().parents[1] / "include"
    types = {"kf_attn_pack_params": _lib.AttnPackParams, "kf_heads": _lib.Heads, "kf_rope_params": _lib.RopeParams}
    body = "".join(f'  printf("{t} %zu\\n", sizeof({t}));\n' + "".join(f'  printf("{t}.{f} %zu\\n", offsetof({t}, {f}));\n' for f, _ in m._fields_) for t, m in types.items())
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kf_b200.h"\nint main(void) {\n' + body + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", str(inc), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for t, m in types.items():
        assert int(out[t]) == C.sizeof(m)
        assert all(int(out[f"{t}.{f}"]) == getattr(m, f).offset for f, _ in m._fields_)
