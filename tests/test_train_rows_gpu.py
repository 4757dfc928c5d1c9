"""LayerNorm with its gradient and rotary positions with several axes, against float64 (oracle/train_oracle.py).

Tolerances count roundings.  u(t) = eps(t) / 2 is the relative error of one rounding to type t; fp32 intermediate steps are counted in units of
u(f32) = 2^-24 with a generous number of steps per value."""
import pytest
import torch

from oracle import train_oracle as to

gpu = pytest.mark.gpu
F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF, F16)}


def _ops():
    from lightly_trian_quant_b200 import ops

    return ops


def _close(got, want, dtype, scale, steps):
    """|got - want| <= u(dtype) |want| + steps * 2^-24 * scale, one half step of the smallest number of the type added"""
    got, want = got.detach().cpu().double(), want.double()
    assert torch.isfinite(got).all()
    bound = U[dtype] * want.abs() * (1 + 2 ** -10) + steps * 2.0 ** -24 * scale + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1, worst


def _norm_case(R, d, tx, seed=0):
    g = torch.Generator().manual_seed(seed + R * 8192 + d)
    x = (torch.randn(R, d, generator=g) * torch.where(torch.rand(d, generator=g) < 0.03, 15.0, 1.0) + 0.5 * torch.randn(R, 1, generator=g)).to(tx)
    return g, x, 1 + 0.2 * torch.randn(d, generator=g), 0.1 * torch.randn(d, generator=g)


def _check_norm(x, w, b, eps, ty, dy, dres, y, dx, dw, db):
    """y, dx: sums of d terms in fp32 through about log2(32) + 32 additions per thread and warp, at most 8 warps: 48 steps; the row's statistics
    enter every value, so the scale is that of the row.  dw, db: sums over the rows: R terms of size |dy xh|, relative to the sum of sizes."""
    xd, wd = x.double(), w.double()
    ry, rdx, rdw, rdb = to.layer_norm_grads(xd, wd, b, eps, torch.zeros_like(xd) if dy is None else dy)
    mean = xd.mean(-1, keepdim=True)
    rstd = (((xd - mean) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    xh = (xd - mean) * rstd
    # x - mean loses |x| + |mean| relative to itself
    size = (xd.abs().mean(-1, keepdim=True) + mean.abs()) * rstd
    at = (xd.abs() + mean.abs()) * rstd + xh.abs() * (1 + size)
    _close(y, ry, ty, at * wd.abs() + (0 if b is None else b.double().abs()), 48)
    if dy is None:
        return
    gsz = (dy.double() * wd).abs()
    inner = gsz + gsz.mean(-1, keepdim=True) + at * (gsz * at).mean(-1, keepdim=True)
    if dres is not None:
        rdx = rdx + dres.double()
    _close(dx, rdx, x.dtype, rstd * inner * (1 + size) + (0 if dres is None else dres.double().abs()), 64)
    _close(dw, rdw, F32, (dy.double().abs() * at).sum(0), 64)
    if db is not None:
        _close(db, rdb, F32, dy.double().abs().sum(0), 64)


@gpu
@pytest.mark.parametrize("tx,ty", [(F32, BF), (F32, F32), (F32, F16), (BF, BF), (F16, F16), (BF, F32), (F16, BF)])
@pytest.mark.parametrize("R,d", [(1, 1), (3, 7), (5, 64), (261, 768), (9, 1024), (33, 333), (2, 1032), (7, 2048), (4, 2047), (3, 4096), (2, 8192), (2, 8191), (700, 40)])
def test_layer_norm_and_its_gradient(tx, ty, R, d):
    ops = _ops()
    g, x, w, b = _norm_case(R, d, tx)
    dy, dres = torch.randn(R, d, generator=g).to(ty), torch.randn(R, d, generator=g).to(tx)
    xc, wc = x.cuda(), w.cuda()
    y, mean, rstd = ops.layer_norm_fwd(xc, wc, b.cuda(), 1e-5, ty)
    dx, dw, db = ops.layer_norm_bwd(dy.cuda(), xc, wc, mean, rstd, dres=dres.cuda())
    assert y.dtype == ty and dx.dtype == tx and dw.dtype == db.dtype == F32
    _check_norm(x, w, b, 1e-5, ty, dy, dres, y, dx, dw, db)


@gpu
@pytest.mark.parametrize("d", [768, 333, 2056])
def test_layer_norm_strided_rows_and_shapes(d):
    """rows of a wider tensor, a tensor of three dimensions, a gradient that is one row repeated, addresses that forbid wide accesses"""
    ops = _ops()
    R = 12
    g, x, w, b = _norm_case(R, d, BF, 1)
    wide = torch.zeros(R, d + 24, dtype=BF, device="cuda")
    wide[:, 8:8 + d] = x.cuda()
    view = wide[:, 8:8 + d]
    one = torch.randn(1, d, generator=g).to(BF)
    y, mean, rstd = ops.layer_norm_fwd(view, w.cuda(), b.cuda(), 1e-5)
    dx, dw, db = ops.layer_norm_bwd(one.cuda().expand(R, d), view, w.cuda(), mean, rstd)
    assert dx.is_contiguous()
    _check_norm(x, w, b, 1e-5, BF, one.expand(R, d), None, y, dx, dw, db)
    odd = torch.zeros(R * d + 1, dtype=BF, device="cuda")[1:].view(R, d)
    odd.copy_(x)
    y2, m2, r2 = ops.layer_norm_fwd(odd, w.cuda(), None, 1e-5)
    dx2, dw2, none = ops.layer_norm_bwd(one.cuda().expand(R, d), odd, w.cuda(), m2, r2, bias=False)
    assert none is None
    _check_norm(x, w, None, 1e-5, BF, one.expand(R, d), None, y2, dx2, dw2, None)
    cube = x.cuda().view(3, 4, d)
    y3, m3, r3 = ops.layer_norm_fwd(cube, w.cuda(), b.cuda(), 1e-5)
    assert y3.shape == cube.shape and m3.shape == (R,) and torch.equal(y3.view(R, d), ops.layer_norm_fwd(x.cuda(), w.cuda(), b.cuda(), 1e-5)[0])
    dx3 = ops.layer_norm_bwd(cube, cube, w.cuda(), m3, r3)[0]
    assert dx3.shape == cube.shape


@gpu
def test_layer_norm_no_rows_and_repeatable_gradients():
    ops = _ops()
    w = torch.ones(96, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(torch.zeros(0, 96, device="cuda"), w, w, 1e-5, BF)
    assert y.shape == (0, 96) and mean.numel() == 0
    dx, dw, db = ops.layer_norm_bwd(y, torch.zeros(0, 96, device="cuda"), w, mean, rstd)
    assert dx.shape == (0, 96) and not dw.any() and not db.any()
    g, x, w, b = _norm_case(5000, 768, F32)
    xc, dy = x.cuda(), torch.randn(5000, 768, generator=g).cuda()
    y, mean, rstd = ops.layer_norm_fwd(xc, w.cuda(), b.cuda(), 1e-5)
    first = ops.layer_norm_bwd(dy, xc, w.cuda(), mean, rstd)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, ops.layer_norm_bwd(dy, xc, w.cuda(), mean, rstd)))


@gpu
def test_layer_norm_rows_that_are_no_numbers_stay_alone():
    """a row with a NaN or an infinity makes NaN of itself (and of dw, db), not of its neighbours"""
    ops = _ops()
    g, x, w, b = _norm_case(40, 1024, BF, 2)
    x[7, 3], x[21, 1000] = float("nan"), float("inf")
    y, mean, rstd = ops.layer_norm_fwd(x.cuda(), w.cuda(), b.cuda(), 1e-5)
    bad = y.isnan().any(1).cpu()
    assert bad.nonzero().flatten().tolist() == [7, 21]
    dx, _, _ = ops.layer_norm_bwd(torch.ones_like(y), x.cuda(), w.cuda(), mean, rstd)
    assert dx.isnan().any(1).cpu().nonzero().flatten().tolist() == [7, 21]


@gpu
def test_layer_norm_refusals():
    ops = _ops()
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    y, m, r = ops.layer_norm_fwd(x, w, w, 1e-5)
    for bad in (lambda: ops.layer_norm_fwd(x.double(), w, w, 1e-5), lambda: ops.layer_norm_fwd(x, w[:32], w, 1e-5), lambda: ops.layer_norm_fwd(x, w.bfloat16(), w, 1e-5),
                lambda: ops.layer_norm_fwd(x.t(), torch.ones(4, device="cuda"), None, 1e-5), lambda: ops.layer_norm_fwd(torch.zeros(2, 8193, device="cuda"), w, w, 1e-5),
                lambda: ops.layer_norm_fwd(torch.zeros(2, 0, device="cuda"), w, w, 1e-5), lambda: ops.layer_norm_fwd(x.cpu(), w, w, 1e-5),
                lambda: ops.layer_norm_fwd(x, w.cpu(), w, 1e-5), lambda: ops.layer_norm_bwd(y[:2], x, w, m, r), lambda: ops.layer_norm_bwd(y, x, w, m[:2], r),
                lambda: ops.layer_norm_bwd(y, x, w, m, r, dres=x.bfloat16()), lambda: ops.layer_norm_bwd(y, x.view(2, 2, 64).transpose(0, 1), w, m, r)):
        with pytest.raises(ops.KfError):
            bad()
    with pytest.raises(KeyError):
        ops.layer_norm_fwd(x, w, w, 1e-5, torch.float64)


# ------------------------------------------------------------------------------------------------ rotary positions
FREQS = {64: [[100.0 ** -(i / 16) * 6.283 for i in range(16)]] * 2, 48: [[1.0, 0.3, 0.1, 0.03]] * 3, 80: [[1.0, 0.5, 0.25, 0.1, 0.01, 1e-3, 1e-4]] * 2 + [[1.0, 0.2, 0.04, 1e-2, 1e-3, 1e-4]],
         6: [[1.0], [0.5]], 256: [[10000 ** -(i / 128) for i in range(128)]], 34: [[0.7] * 8, [], [0.1] * 9], 8: [[]]}


def _check_rope(y, x, pos, freqs, dtype, interleaved=False, inverse=False):
    """two products and a sum in fp32, sine and cosine to 2 units in the last place: 8 steps of the pair's size"""
    want = to.rope(x, pos, freqs, interleaved, inverse)
    _close(y, want, dtype, x.double().abs().amax(-1, keepdim=True), 8)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D", [(1, 1, 64), (261, 24, 64), (9, 3, 48), (17, 5, 80), (5, 2, 6), (12, 2, 256), (40, 7, 34), (3, 300, 64), (2, 2, 8)])
def test_rope_axes_and_its_gradient(dtype, interleaved, T, H, D):
    ops = _ops()
    g = torch.Generator().manual_seed(T * 1000 + H)
    freqs = FREQS[D]
    x = torch.randn(T, H, D, generator=g).to(dtype)
    pos = torch.randint(-50, 3000, (T, len(freqs)), generator=g)
    table = ops.RopeTable(freqs, D, interleaved=interleaved)
    for p in (pos.int(), pos, pos.float() * 0.37 - 1):
        for inverse in (False, True):
            y = ops.rope_axes(x.cuda(), p.cuda(), table, inverse=inverse)
            _check_rope(y, x, p, freqs, dtype, interleaved, inverse)


@gpu
@pytest.mark.parametrize("pos", [1_000_003, 16_777_217, 2_147_483_647])
def test_rope_far_positions(pos):
    """the angle keeps all digits fp32 can show of its sine"""
    ops = _ops()
    x = torch.randn(4, 3, 48, generator=torch.Generator().manual_seed(1))
    p = torch.tensor([[pos - i, i, pos // (i + 1)] for i in range(4)], dtype=torch.int64)
    for cast in (torch.int32, torch.int64):
        _check_rope(ops.rope_axes(x.cuda(), p.to(cast).cuda(), ops.RopeTable(FREQS[48], 48)), x, p, FREQS[48], F32)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF])
def test_rope_strides_outer_dimension_and_in_place(dtype):
    """queries and keys of one projection as [2, T, H, D] with any strides, the result in place, next to tensors that stay as they are; strides that
    allow narrow accesses only"""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    T, H, D = 37, 4, 64
    table, pos = ops.RopeTable(FREQS[D], D), torch.randint(0, 40, (T, 2), generator=g)
    qkv = torch.randn(T, 3, H, D, generator=g).to(dtype)
    dev = qkv.cuda()
    qk = dev.permute(1, 0, 2, 3)[:2]                            # [2, T, H, D]
    same = ops.rope_axes(qk, pos.cuda(), table, out=qk)
    assert same is qk and torch.equal(dev[:, 2].cpu(), qkv[:, 2])
    for i in range(2):
        _check_rope(dev[:, i], qkv[:, i], pos, FREQS[D], dtype)
    for pad in (1, 2, 4):                                       # row strides of 1, 2 and 4 values beyond a multiple of 8
        x = torch.zeros(T, H, D + pad, dtype=dtype, device="cuda")[..., :D]
        x.copy_(qkv[:, 0])
        _check_rope(ops.rope_axes(x, pos.cuda(), table), qkv[:, 0], pos, FREQS[D], dtype)
    stretched = qkv[:, :1, 0].cuda().expand(T, H, D)            # an input head read by all
    _check_rope(ops.rope_axes(stretched, pos.cuda(), table), qkv[:, :1, 0].expand(T, H, D), pos, FREQS[D], dtype)
    wide = torch.zeros(T, 5, dtype=torch.int64)
    wide[:, 1], wide[:, 4] = pos[:, 0], pos[:, 1]
    _check_rope(ops.rope_axes(qkv[:, 1].cuda(), wide.cuda()[:, 1::3], table), qkv[:, 1], pos, FREQS[D], dtype)


@gpu
def test_rope_matches_the_backbones_tables():
    """the positions and frequencies of the backbone's own tables turn as its rope_apply does; prefix tokens with position 0 stay"""
    from lightly_trian_quant_b200 import modeldef

    ops = _ops()
    emb = modeldef.RopePositionEmbedding(64, 100.0)
    sin, cos = emb(H=6, W=9)
    f = (2 * torch.pi / emb.periods.double()).tolist()
    ch, cw = (torch.arange(0.5, 6) / 6 * 2 - 1), (torch.arange(0.5, 9) / 9 * 2 - 1)
    pos = torch.cat((torch.zeros(5, 2), torch.stack(torch.meshgrid(ch, cw, indexing="ij"), -1).flatten(0, 1)))
    x = torch.randn(59, 3, 64, generator=torch.Generator().manual_seed(4))
    y = ops.rope_axes(x.cuda(), pos.cuda(), ops.RopeTable([f, f], 64)).cpu()
    assert torch.equal(y[:5], x[:5])
    # the tables' angles are fp32 products of up to 2 pi: half a step of 2^-22 each for coordinate, product and division
    assert torch.allclose(y[5:], modeldef.rope_apply(x[5:].transpose(0, 1), sin, cos).transpose(0, 1), rtol=0, atol=2.0 ** -20 * x.abs().max().item())


@gpu
def test_rope_refusals():
    ops = _ops()
    x, pos, table = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), ops.RopeTable(FREQS[64], 64)
    inter = ops.RopeTable(FREQS[64], 64, interleaved=True)
    narrow = torch.zeros(4, 2, 65, device="cuda")[..., :64]
    for bad in (lambda: ops.rope_axes(x.double(), pos, table), lambda: ops.rope_axes(x[..., :48], pos, table), lambda: ops.rope_axes(x, pos[:3], table),
                lambda: ops.rope_axes(x, pos[:, :1], table), lambda: ops.rope_axes(x, pos.short(), table), lambda: ops.rope_axes(x.transpose(1, 2), pos, table),
                lambda: ops.rope_axes(x[0], pos, table), lambda: ops.rope_axes(x, pos.cpu(), table), lambda: ops.rope_axes(x.cpu(), pos, table),
                lambda: ops.rope_axes(x, pos, table, out=x.bfloat16()), lambda: ops.rope_axes(x, pos, table, out=x[:1].expand(4, 2, 64)),
                lambda: ops.rope_axes(narrow, pos, inter)):
        with pytest.raises(ops.KfError):
            bad()
    assert ops.rope_axes(x[:0], pos[:0], table).shape == (0, 2, 64)


@gpu
def test_rope_outputs_that_overlap_the_input():
    ops = _ops()
    pos, table = torch.arange(8, device="cuda").view(4, 2).int(), ops.RopeTable(FREQS[64], 64)
    buf = torch.randn(2, 4, 6, 64, device="cuda")
    x = buf[:, :, :3]
    want = ops.rope_axes(x, pos, table)
    for bad in (buf[:, :, 2:5], buf[:, :, 1:4], buf.flatten()[32:32 + 2 * 4 * 192].view(2, 4, 3, 64), buf.as_strided((2, 4, 3, 64), (64, 64, 64, 1)),
                torch.zeros(1024, device="cuda").as_strided((2, 4, 3, 64), (192, 64, 64, 1))):
        with pytest.raises(ops.KfError, match="overlap"):
            ops.rope_axes(x, pos, table, out=bad)
    assert torch.equal(ops.rope_axes(x, pos, table, out=buf[:, :, 3:]), want)        # the columns between
    assert torch.equal(ops.rope_axes(x, pos, table, out=x), want)
    ops.check_device_error()


def test_rope_table_refusals():
    ops = _ops()
    for bad in (lambda: ops.RopeTable([[1.0] * 33], 64, device="cpu"), lambda: ops.RopeTable([[1.0]], 258, device="cpu"), lambda: ops.RopeTable([[float("inf")]], 64, device="cpu"),
                lambda: ops.RopeTable.geometric([3], 64, device="cpu"), lambda: ops.RopeTable([[1.0]], 0, device="cpu")):
        with pytest.raises(ops.KfError):
            bad()
    t = ops.RopeTable.geometric([8, 4], 16, device="cpu")
    assert t.axis.tolist() == [0] * 4 + [1] * 2 and t.axes == 2 and torch.allclose(t.freq * torch.pi, torch.tensor([1, 0.1, 0.01, 0.001, 1, 0.01], dtype=torch.float64))


def test_training_operators_refuse_cpu_tensors():
    ops = _ops()
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(ops.KfError):
        ops.layer_norm_fwd(x, w, w, 1e-5)
    with pytest.raises(ops.KfError):
        ops.layer_norm_bwd(x, x, w, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ops.KfError):
        ops.rope_axes(x.view(4, 1, 64), torch.zeros(4, 2, dtype=torch.int32), ops.RopeTable(FREQS[64], 64, device="cpu"))


def test_host_checks_of_the_row_operators():
    """bad arguments end as a status with a message before any launch"""
    from lightly_trian_quant_b200 import _lib

    L = _lib.lib()
    msg = lambda: L.kf_last_error_string().decode()  # noqa: E731
    assert L.kf_layer_norm_fwd(7, 4096, 64, 4096, 4096, 1e-5, 4, 64, 0, 4096, 4096, 4096, None) == -1 and "types" in msg()
    assert L.kf_layer_norm_fwd(0, 4096, 64, 4096, 4096, 1e-5, 4, 8193, 0, 4096, 4096, 4096, None) == -1 and "8192" in msg()
    assert L.kf_layer_norm_fwd(0, None, 64, 4096, 4096, 1e-5, 4, 64, 0, 4096, 4096, 4096, None) == -1 and "null" in msg()
    assert L.kf_layer_norm_fwd(0, None, 64, None, None, 1e-5, 0, 64, 0, None, None, None, None) == 0
    assert L.kf_layer_norm_bwd(0, 4096, 64, 0, 4096, 64, None, 4096, 4096, None, 0, 4, 64, 4096, 4096, 4096, 4096, 0, None) == -1 and "null" in msg()
    assert L.kf_layer_norm_ws_bytes(-1, 64) == -1 and L.kf_layer_norm_ws_bytes(4, 0) == -1
    p = _lib.RopeParams()
    p.dtype, p.G, p.T, p.H, p.D, p.P = 0, 1, 4, 2, 64, 33
    p.x = p.y = p.pos = p.freq = p.axis = 4096
    assert L.kf_rope_axes(p, None) == -1 and "pairs" in msg()
    p.P, p.pos_kind = 32, 9
    assert L.kf_rope_axes(p, None) == -1 and "positions" in msg()
    p.pos_kind, p.x = 0, None
    assert L.kf_rope_axes(p, None) == -1 and "null" in msg()
