"""The kernels of the operators for training: what the compiler made of them, and how they end behind a launch that failed."""
import re

import pytest
import torch

gpu = pytest.mark.gpu


@pytest.mark.parametrize("stem,kernels,registers", [("kf_attn_pack", 16, 128), ("kf_attn_pack_bwd", 16, 96)])
def test_register_splits_have_what_they_draw_on(stem, kernels, registers):
    """the packed attention's kernels hand registers from one role to another; the sum comes from what a block is launched with, and a build that
    allocates less would wait for the rest without end."""
    from lightly_trian_quant_b200 import build

    build.build()
    (path,) = (build.CSRC / "build").glob(f"{stem}.*.ptxas")
    used = [int(m) for block in path.read_text().split("Compiling entry function")[1:] if "attn_pack" in block.split("\n")[0] for m in re.findall(r"Used (\d+) registers", block)]
    assert used == [registers] * kernels


@gpu
def test_calls_behind_a_failed_launch_end_and_the_next_ones_work():
    """kernels that find the error word set compute nothing and return; what comes after the check is right again."""
    from lightly_trian_quant_b200 import _lib, ops

    q = torch.randn(300, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    plan = ops.AttnPlan([300], causal=True)
    out, lse = ops.attn_packed(q, q, q, plan)
    grads = ops.attn_packed_bwd(q, q, q, q, out, lse, plan)
    _lib.check(_lib.lib().kf_selftest_raise_error(0, torch.cuda.current_stream().cuda_stream), "kf_selftest_raise_error")
    bad, bad_lse = ops.attn_packed(q, q, q, plan)
    ops.attn_packed_bwd(q, q, q, q, bad, bad_lse, plan)
    with pytest.raises(ops.KfError, match="site 200"):
        ops.check_device_error()
    again, again_lse = ops.attn_packed(q, q, q, plan)
    assert torch.equal(again, out) and torch.equal(again_lse, lse)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.attn_packed_bwd(q, q, q, q, again, again_lse, plan)))
    ops.check_device_error()
