"""The operators for training from several threads at once, each on a stream of its own."""
import threading

import pytest
import torch

gpu = pytest.mark.gpu
BF = torch.bfloat16


@gpu
def test_threads_on_their_own_streams():
    """both directions of all operators, among them forwards that are split into clusters: the bits of a thread alone"""
    from lightly_trian_quant_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kinds = []
    for q_lens, k_lens, Hq, Hk, how in (([200, 31], [1605, 261], 4, 4, {}), ([300, 77], [300, 77], 6, 2, {"cap": 20.0}), ([1], [4101], 8, 1, {"slopes": torch.linspace(0, 0.5, 8, device="cuda")})):
        q, k, v, do = r(sum(q_lens), Hq, 64).to(BF), r(sum(k_lens), Hk, 64).to(BF), r(sum(k_lens), Hk, 64).to(BF), r(sum(q_lens), Hq, 64).to(BF)
        kinds.append((q, k, v, do, ops.AttnPlan(q_lens, k_lens), how))
    x, w, dy = r(3000, 333), 1 + 0.1 * r(333), r(3000, 333)
    pos, table = torch.arange(3000, device="cuda")[:, None], ops.RopeTable([[1.0 / (i + 1) for i in range(16)]], 37)

    def step(i):
        q, k, v, do, plan, how = kinds[i % 3]
        out, lse = ops.attn_packed(q, k, v, plan, **how)
        grads = ops.attn_packed_bwd(do, q, k, v, out, lse, plan, **how)
        y, mean, rstd = ops.layer_norm_fwd(x, w, w, 1e-5)
        return (out, lse, *grads, y, *ops.layer_norm_bwd(dy, x, w, mean, rstd), ops.rope_axes(x.view(3000, 9, 37), pos, table))

    want = [step(i) for i in range(3)]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for n in range(60):
                    i = (first + n) % 3
                    got = step(i)
                    same = torch.stack([(a == b).all() for a, b in zip(got, want[i])]).all()
                    stream.synchronize()
                    if not same.item():
                        wrong.append((first, n))
        except Exception as e:                                     # shown by the assertion below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ops.check_device_error()
    assert not wrong, wrong[:5]
