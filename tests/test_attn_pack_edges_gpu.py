"""Packed attention at the edges of its range: saturated caps, masked keys of any size, positions behind 2^24, probabilities below f16's normal range,
gradients that nobody asks for."""
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
