"""Packed attention at the edges of its range: saturated caps, masked keys of any size, positions behind 2^24, probabilities below f16's normal range,
gradients that nobody asks for."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _ops():
    from lightly_trian_quant_b200 import ops

    return ops


# ------------------------------------------------------------------------------------------------ masked keys
@gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True), (50.0, True)])
@pytest.mark.parametrize("q_lens,k_lens,huge", [([264], [264], 256), ([130, 72, 5], [130, 72, 5], 126), ([72, 264], [72, 264], 330), ([8], [1208], 1205), ([300], [1400], 1399)], ids=str)
def test_masked_keys_have_no_part_in_a_row(q_lens, k_lens, huge, cap, bias, dtype):
    """values of keys from `huge` on are as large as the type allows: rows that do not see them come out with the bits that they have without them"""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = r(sum(q_lens), 2, 64), r(sum(k_lens), 2, 64), r(sum(k_lens), 2, 64)
    slopes = torch.tensor([0.02, 0.5], device="cuda") if bias else None
    plan = ops.AttnPlan(q_lens, k_lens, causal=True)
    large = v.clone()
    large[huge:huge + 8] = torch.finfo(dtype).max
    for longest in (plan.longest, 0):                                    # split along the keys where that is the rule, and whole
        plan.longest = longest
        want, lse = ops.attn_packed(q, k, v, plan, cap=cap, slopes=slopes)
        got, lse2 = ops.attn_packed(q, k, large, plan, cap=cap, slopes=slopes)
        ops.check_device_error()
        assert torch.equal(lse, lse2)
        q0 = k0 = rows = 0
        for lq, lk in zip(q_lens, k_lens):
            for i in range(lq):
                if k0 + i + lk - lq < huge or k0 >= huge + 8:
                    rows += 1
                    assert torch.equal(got[q0 + i], want[q0 + i]), (q0 + i, (got[q0 + i].float() - want[q0 + i].float()).abs().max())
            q0, k0 = q0 + lq, k0 + lk
        assert rows


# ------------------------------------------------------------------------------------------------ far positions
@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("split", [True, False])
def test_distances_behind_position_two_to_the_24(split, causal):
    """a sequence of more than 2^24 keys: the distance of neighbours is a small number there too.  Keys but the last 200 are zero, the slope is steep, so that a float64 sum
    over the last 2048 keys is all of it (e^-900 is left out).  Tolerance: scores up to 8 and slopes times distances in fp32, 1e-5 of a probability; u = 2^-8 of each
    term for P or dS and of the result, 3.5 standard deviations as everywhere in these tests."""
    ops = _ops()
    Lq, Lk, near, slope, u = 3, 2 ** 24 + 5, 2048, 0.5, 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)  # noqa: E731
    q, do = r(Lq, 1, 64), r(Lq, 1, 64)
    k, v = torch.zeros(Lk, 1, 64, dtype=BF, device="cuda"), torch.zeros(Lk, 1, 64, dtype=BF, device="cuda")
    k[-200:], v[-200:] = r(200, 1, 64), r(200, 1, 64)
    slopes = torch.tensor([slope], device="cuda")
    plan = ops.AttnPlan([Lq], [Lk], causal=causal)
    if not split:
        plan.longest = 0
    out, lse = ops.attn_packed(q, k, v, plan, slopes=slopes)
    dq, dk, dv = ops.attn_packed_bwd(do, q, k, v, out, lse, plan, slopes=slopes)
    ops.check_device_error()
    assert not dk[:-near].any() and not dv[:-near].any()
    Q, K, V, dO = q[:, 0].double(), k[-near:, 0].double(), v[-near:, 0].double(), do[:, 0].double()
    at, key = torch.arange(Lk - Lq, Lk, device="cuda")[:, None], torch.arange(Lk - near, Lk, device="cuda")[None]
    s = Q @ K.t() * 0.125 - slope * (at - key).abs()
    if causal:
        s = s.masked_fill(key > at, -math.inf)
    z = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - z)
    o = p @ V
    dp, delta = dO @ V.t(), (dO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = p * (dp.abs() + (dO * o).abs().sum(-1, keepdim=True))
    row = p * (u * (dO * o).square().sum(-1, keepdim=True).sqrt())
    assert (lse[0].double() - z[:, 0]).abs().max() <= 1e-5
    checks = {"out": (out, o, (u * p) ** 2 @ V ** 2, 1e-5 * p @ V.abs()),
              "dq": (dq, ds @ K / 8, (u / 8) ** 2 * (ds ** 2 @ K ** 2) + (row @ K / 8) ** 2, 2e-5 * (size @ K.abs()) / 8),
              "dk": (dk[-near:], ds.t() @ Q / 8, (u / 8) ** 2 * ((ds ** 2).t() @ Q ** 2) + (row ** 2).t() @ Q ** 2 / 64, 2e-5 * (size.t() @ Q.abs()) / 8),
              "dv": (dv[-near:], p.t() @ dO, (u * p.t()) ** 2 @ dO ** 2, 1e-5 * p.t() @ dO.abs())}
    for name, (got, want, var, hard) in checks.items():
        bound = 3.5 * (var + u * u * want ** 2).sqrt() + hard + 2.0 ** -118
        worst = ((got[:, 0].double() - want).abs() / bound).max().item()
        assert worst <= 1, (name, worst)


# ------------------------------------------------------------------------------------------------ small probabilities in f16
@gpu
@pytest.mark.parametrize("heads", [(1, 1), (2, 1)])
@pytest.mark.parametrize("Lk", [818401, 65537])
def test_f16_gradients_of_values_over_many_keys(Lk, heads):
    """q = 0: every probability is 1 / Lk, and dv the sum of dout over it.  Below 2^-14 an f16 probability would lose its digits (at 818 401 keys it is 20.5 steps of
    2^-24), the same ones in every row, so that they do not cancel.  Tolerance: P rounded once by u = 2^-11 in every row alike, the result once; 1e-5 for the exponent
    (log-sum-exp 13.6 in fp32 and its product with log2(e), 2^-21 each, and the exponentials' 4e-6)."""
    ops = _ops()
    Hq, Hk = heads
    Lq, u = 100, 2.0 ** -11
    q = torch.zeros(Lq, Hq, 64, dtype=F16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    k = torch.randn(Lk, Hk, 64, generator=g, device="cuda").to(F16)
    do = (1 + torch.rand(Lq, Hq, 64, generator=g, device="cuda")).to(F16)
    plan = ops.AttnPlan([Lq], [Lk])
    out, lse = ops.attn_packed(q, k, k, plan)
    dq, dk, dv = ops.attn_packed_bwd(do, q, k, k, out, lse, plan)
    ops.check_device_error()
    want = do.double().view(Lq, Hk, Hq // Hk, 64).sum((0, 2)) / Lk
    assert ((dv.double() - want).abs() <= (2 * u + 1e-5) * want + 2.0 ** -25).all(), ((dv.double() / want - 1).abs().max().item())
    assert not dk.any() and torch.isfinite(dq).all()


# ------------------------------------------------------------------------------------------------ caps that fp32 cannot hold
def test_caps_out_of_fp32s_range_are_refused_by_the_library():
    """a cap below fp32's normal range, or one whose scale leaves it, makes infinities of factors that meet zeros"""
    from lightly_trian_quant_b200 import _lib

    L, H = _lib.lib(), _lib.Heads
    for cap, scale in ((1e-40, 0.125), (1e-38, 0.125), (1e-20, 1e25), (1e-36, 1e3)):
        p = _lib.AttnPackParams()
        p.dtype, p.Hq, p.Hk, p.n_q_tiles, p.n_k_tiles, p.scale, p.cap, p.Tq, p.Tk = 1, 4, 2, 1, 1, scale, cap, 40, 40
        p.q_tiles = p.k_tiles = p.lse = p.ws = 4096                     # never dereferenced: the calls end on the host
        p.ws_bytes = 1 << 20
        for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
            setattr(p, n, H(4096, 256, 64))
        for call in (L.kf_attn_pack_fwd, L.kf_attn_pack_bwd):
            assert call(p, None) == -1 and "cap" in L.kf_last_error_string().decode(), (cap, scale, L.kf_last_error_string())


@gpu
def test_caps_that_vanish_in_fp32_are_refused():
    """1e-50 is 0 in fp32, which means no cap: the opposite of what was asked for"""
    ops = _ops()
    q = torch.randn(8, 1, 64, device="cuda").to(BF)
    plan = ops.AttnPlan([8])
    out, lse = ops.attn_packed(q, q, q, plan)
    for cap in (1e-50, 1e-300, 1e-40):
        with pytest.raises(ops.KfError, match="cap"):
            ops.attn_packed(q, q, q, plan, cap=cap)
        with pytest.raises(ops.KfError, match="cap"):
            ops.attn_packed_bwd(q, q, q, q, out, lse, plan, cap=cap)
    ops.check_device_error()


# ------------------------------------------------------------------------------------------------ saturated caps
@gpu
@pytest.mark.parametrize("heads", [(1, 1), (2, 1)])
@pytest.mark.parametrize("cap", [1.5, 30.0])
@pytest.mark.parametrize("lo,hi", [(7.0, 9.0), (0.4, 9.0)])
def test_gradients_at_saturated_scores(lo, hi, cap, heads):
    """queries and keys whose capped scores lie at lo to hi times the cap: their gradients are the small 1 - tanh^2 = 4 e / (1 + e)^2, e = exp(-2y), which has to
    come out with its own digits, not with those of 1.

    Scores are products of one channel with few digits each, so that they are exact; the other channels of q meet zeros of k and the other way round, and carry the
    gradients.  Tolerance in bf16, u = 2^-8: dS and the result are rounded once (standard deviation u / sqrt(3), six of them: 3.5 u sqrt(sum of squares)), delta
    takes the rounded output, for a whole row.  fp32: t = 2 y log2(e) <= 26 is off by two roundings, so e by 26 * 2^-23 * ln 2 = 2.2e-6 of itself; exponential 2^-22, reciprocal
    2^-23 twice, three products 2^-24; P from a capped score off by 2^-22 cap and its log-sum-exp the same, so 2 * 2^-22 * 30 = 1.4e-5 of itself at cap 30: 2e-5 of every term
    in all, with the sizes of dP and delta in place of their difference."""
    ops = _ops()
    Hq, Hk = heads
    n, scale, u = 96, 0.125, 2.0 ** -8
    g = torch.Generator().manual_seed(int(hi + 100 * lo))
    q, k = torch.zeros(n, Hq, 64), torch.zeros(n, Hk, 64)
    k[..., 0] = torch.where(torch.rand(n, Hk, generator=g) < 0.5, -1.0, 1.0)
    q[..., 0] = torch.empty(n, Hq).uniform_(lo, hi, generator=g) * cap / scale
    q[..., 1:32] = torch.randn(n, Hq, 31, generator=g)
    k[..., 32:] = torch.randn(n, Hk, 32, generator=g)
    q, k = q.to(BF), k.to(BF)
    v, do = torch.randn(n, Hk, 64, generator=g).to(BF), torch.randn(n, Hq, 64, generator=g).to(BF)
    plan = ops.AttnPlan([n])
    qc, kc, vc, dc = (t.cuda() for t in (q, k, v, do))
    out, lse = ops.attn_packed(qc, kc, vc, plan, scale=scale, cap=cap)
    dq, dk, dv = ops.attn_packed_bwd(dc, qc, kc, vc, out, lse, plan, scale=scale, cap=cap)
    ops.check_device_error()
    q, k, v, do = (t.double() for t in (q, k, v, do))
    dk_want, dk_var, dk_hard = torch.zeros_like(k), torch.zeros_like(k), torch.zeros_like(k)
    for h in range(Hq):
        gk = h * Hk // Hq
        Q, K, V, dO = q[:, h], k[:, gk], v[:, gk], do[:, h]
        y = Q @ K.t() * scale / cap
        e = torch.exp(-2 * y.abs())
        factor = 4 * e / (1 + e) ** 2
        p = torch.softmax(cap * torch.tanh(y), -1)
        o = p @ V
        dp, delta = dO @ V.t(), (dO * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * factor
        size = p * factor * (dp.abs() + (dO * o).abs().sum(-1, keepdim=True))
        row = p * factor * (u * (dO * o).square().sum(-1, keepdim=True).sqrt())
        value = ds @ K * scale
        bound = 3.5 * ((u * scale) ** 2 * (ds ** 2 @ K ** 2) + (scale * row @ K) ** 2 + u * u * value ** 2).sqrt() + 2e-5 * scale * (size @ K.abs()) + 2.0 ** -120
        worst = ((dq[:, h].cpu().double() - value).abs() / bound).max().item()
        assert worst <= 1, ("dq", h, worst)
        dk_want[:, gk] += ds.t() @ Q * scale
        dk_var[:, gk] += scale ** 2 * (u * u * (ds ** 2).t() @ Q ** 2 + (row ** 2).t() @ Q ** 2)
        dk_hard[:, gk] += 2e-5 * scale * (size.t() @ Q.abs())
    bound = 3.5 * (dk_var + u * u * dk_want ** 2).sqrt() + dk_hard + 2.0 ** -120
    worst = ((dk.cpu().double() - dk_want).abs() / bound).max().item()
    assert worst <= 1, ("dk", worst)
    assert torch.isfinite(dv).all()


# ------------------------------------------------------------------------------------------------ dependent launches
@gpu
@pytest.mark.parametrize("mode", [True, False, None])
def test_a_chain_of_the_operators_in_every_launch_mode(mode):
    """both directions of all operators behind one another, short ones, so that each is there while the one before it still runs: the same bits in every mode"""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(12)
    lens, H, Hk = [70, 1, 130], 6, 2
    T, d = sum(lens), (H + 2 * Hk) * 64
    x, w = torch.randn(T, d, generator=g, device="cuda"), 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    do = torch.randn(T, H, 64, generator=g, device="cuda").to(BF)
    pos, table = torch.arange(2 * T, device="cuda").view(T, 2).int(), ops.RopeTable([[1.0, 0.1], [0.5]], 64)
    plan = ops.AttnPlan(lens, causal=True)

    def step():
        y, mean, rstd = ops.layer_norm_fwd(x, w, w, 1e-5, BF)
        qkv = y.view(T, H + 2 * Hk, 64)
        turned = ops.rope_axes(qkv, pos, table)
        q, k, v = turned[:, :H], turned[:, H:H + Hk], qkv[:, H + Hk:]
        out, lse = ops.attn_packed(q, k, v, plan, cap=20.0)
        gq = torch.empty_like(qkv)
        ops.attn_packed_bwd(do, q, k, v, out, lse, plan, cap=20.0, grads=(gq[:, :H], gq[:, H:H + Hk], gq[:, H + Hk:]))
        ops.rope_axes(gq[:, :H + Hk], pos, table, inverse=True, out=gq[:, :H + Hk])
        return (out, lse, gq, *ops.layer_norm_bwd(gq.view(T, d), x, w, mean, rstd, dres=x))

    ops.set_pdl(False)
    want = step()
    ops.set_pdl(mode)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    ops.check_device_error()


# ------------------------------------------------------------------------------------------------ many small weights beside a large one in f16
@gpu
@pytest.mark.parametrize("cap,bias", [(0.0, False), (60.0, False), (0.0, True)])
@pytest.mark.parametrize("split", [True, False])
def test_f16_weights_far_below_the_largest(split, cap, bias):
    """the first key weighs about as much as 400 002 others together, each at 20.5 steps of 2^-24 of it: f16 weights relative to the largest would lose a fortieth of each, the same
    way.  Tolerance: weights and output rounded once by u = 2^-11, the exponents to 2e-5 (scores of 13.6, the cap's 60 * 2^-22).  The products are summed 16 keys at a time in fp32 without rounding to nearest: each of the n = 25 000 additions may cut
2^-23 of a sum that grows evenly, n / 2 * 2^-23 = 1.5e-3 in all (an eighth of it where eight CTAs share the keys).  The weights' own sum takes 96 keys at a time, rounded to nearest, with equal terms the same way over long
stretches: 4167 / 2 * 2^-24 = 1.2e-4 of the sum, and so of the log-sum-exp."""
    ops = _ops()
    Lq, Lk, u = 3, 400003, 2.0 ** -11
    q, k = torch.zeros(Lq, 1, 64, dtype=F16, device="cuda"), torch.zeros(Lk, 1, 64, dtype=F16, device="cuda")
    v = torch.ones(Lk, 1, 64, dtype=F16, device="cuda")
    q[..., 0], k[0, 0, 0], v[0] = 8, 13.615, 0
    if cap:
        k[0, 0, 0] = cap * math.atanh(13.615 / cap)
    slopes = torch.zeros(1, device="cuda") if bias else None
    plan = ops.AttnPlan([Lq], [Lk])
    if not split:
        plan.longest = 0
    out, lse = ops.attn_packed(q, k, v, plan, cap=cap, slopes=slopes)
    ops.check_device_error()
    s = k[0, 0, 0].double().item()
    s = cap * math.tanh(s / cap) if cap else s
    total = math.exp(s) + Lk - 1
    want = (Lk - 1) / total
    sums = Lk / 16 / 2 * 2.0 ** -23 / (8 if split else 1)
    assert (out.double() - want).abs().max() <= (2 * u + 2e-5 + sums) * want, (out.double() / want - 1).abs().max()
    assert (lse.double() - math.log(total)).abs().max() <= 2e-5 + Lk / 96 / 2 * 2.0 ** -24 / (8 if split else 1)
