"""LayerNorm where a group of warps goes through many rows: ring slots and their barriers in turn, statistics fetched a row ahead, column sums over a group's rows.

Against float64, in units of 2^-24 of the sizes that enter a value.  y and dx as in test_train_rows_gpu.py (48 and 64 steps).  dw and db: the statistics in every term (48
steps), and a chain of additions of a group's rows (at one CTA per SM R / (148 * groups of a CTA), at most 41 here), the 8 groups of a CTA, the lines of a thread of the second
launch (148 / 32; four times as many where the rows of a group are a quarter) and 5 steps of a warp: 59 at most, 112 with the statistics and the products."""
import pytest
import torch

from oracle import train_oracle as to
from tests.test_train_rows_gpu import BF, F16, F32, _close, _norm_case, _ops

gpu = pytest.mark.gpu

# rows so many that on 148 SMs with at most 4 CTAs each every group of warps takes 5 rows or more (slots and phases come round twice), in every
# number of warps per row (forward 1 up to 1024 wide, 2 up to 2048, 4 up to 4096, 8; backward 1 up to 512, 2 up to 1024, 4 up to 2048, 8), both widths of access
CASES = [(40009, 333, BF, BF), (24001, 512, F16, F32), (23700, 77, F32, F32), (24003, 1024, F32, BF), (24005, 1000, F16, F16), (12001, 2048, F32, BF), (12003, 1999, BF, F32), (6007, 4096, BF, BF),
         (6007, 3001, F32, F16), (3001, 8192, BF, F32), (3003, 8191, BF, BF),
         (24007, 397, BF, BF), (24001, 603, F32, BF), (24007, 801, F16, F32), (12007, 1001, BF, BF), (12001, 1201, F32, F32), (12005, 1601, BF, F16), (6001, 3501, F16, F16), (3007, 5001, F32, BF)]


def _check_norm(x, w, b, ty, dy, dres, y, dx, dw, db):
    xd, wd, gd = x.double(), w.double(), dy.double()
    ry, rdx, rdw, rdb = to.layer_norm_grads(xd, wd, b, 1e-5, gd)
    mean = xd.mean(-1, keepdim=True)
    rstd = (((xd - mean) ** 2).mean(-1, keepdim=True) + 1e-5) ** -0.5
    size = (xd.abs().mean(-1, keepdim=True) + mean.abs()) * rstd
    at = (xd.abs() + mean.abs()) * rstd + ((xd - mean) * rstd).abs() * (1 + size)           # what enters xh
    _close(y, ry, ty, at * wd.abs() + b.double().abs(), 48)
    gsz = (gd * wd).abs()
    inner = gsz + gsz.mean(-1, keepdim=True) + at * (gsz * at).mean(-1, keepdim=True)
    res = torch.zeros(()).double() if dres is None else dres.double()
    _close(dx, rdx + res, x.dtype, rstd * inner * (1 + size) + res.abs(), 64)
    _close(dw, rdw, F32, (gd.abs() * at).sum(0), 112)
    _close(db, rdb, F32, gd.abs().sum(0), 112)


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("R,d,tx,ty", CASES, ids=str)
def test_many_rows_per_group(R, d, tx, ty, residual):
    ops = _ops()
    g, x, w, b = _norm_case(R, d, tx, 5)
    dy = torch.randn(R, d, generator=g).to(ty)
    dres = torch.randn(R, d, generator=g).to(tx) if residual else None
    xc, wc = x.cuda(), w.cuda()
    y, mean, rstd = ops.layer_norm_fwd(xc, wc, b.cuda(), 1e-5, ty)
    dx, dw, db = ops.layer_norm_bwd(dy.cuda(), xc, wc, mean, rstd, dres=None if dres is None else dres.cuda())
    ops.check_device_error()
    _check_norm(x, w, b, ty, dy, dres, y, dx, dw, db)


@gpu
def test_many_strided_rows():
    """rows of a wider tensor at addresses that change their place in 16 bytes from row to row"""
    ops = _ops()
    R, d = 24007, 333
    g, x, w, b = _norm_case(R, d, BF, 6)
    dy = torch.randn(R, d, generator=g).to(BF)
    wide, wide_dy = torch.full((R, d + 3), float("nan"), dtype=BF, device="cuda"), torch.full((R, d + 6), float("nan"), dtype=BF, device="cuda")
    wide[:, 1:1 + d], wide_dy[:, 5:5 + d] = x.cuda(), dy.cuda()
    xc, dyc = wide[:, 1:1 + d], wide_dy[:, 5:5 + d]
    y, mean, rstd = ops.layer_norm_fwd(xc, w.cuda(), b.cuda(), 1e-5)
    dx, dw, db = ops.layer_norm_bwd(dyc, xc, w.cuda(), mean, rstd)
    ops.check_device_error()
    _check_norm(x, w, b, BF, dy, None, y, dx, dw, db)
