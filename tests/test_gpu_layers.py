"""The trainable-layer operators on the GPU against their definitions in float64 (tests/layers_ref.py), and a run of them together."""
import numpy as np
import pytest
import torch

import _pkg
import layers_ref as R

pytestmark = pytest.mark.gpu
L = _pkg.load().layers
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def same_checkpoint(kept, x, signed):
    """codes and scales of `kept` are those of the definition applied to x, bit for bit"""
    c, e = R.pack(x, signed)
    gc, ge = R.raw(kept)
    assert kept.signed == signed
    assert np.array_equal(ge, e) and np.array_equal(gc, c)


# ------------------------------------------------------------------------------------------------------------------------------------------- checkpoints
@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 32), (7, 33), (65, 63), (130, 8), (9, 257)])
def test_checkpoint_is_the_definition(n, k, dtype, signed):
    x = randn(gen(n * 1000 + k), n, k, dtype=dtype)
    x = x * torch.exp2(torch.randint(-12, 12, (n, 1), generator=gen(1)).float()).to(DEV).to(dtype)
    kept = L.checkpoint(x, signed=signed)
    same_checkpoint(kept, x, signed)
    for t in TYPES[:2]:                                     # exact in float32 and bfloat16
        assert torch.equal(kept.values(t).double().cpu(), R.stored(kept))
    if dtype == torch.float16:                              # ... and in float16 for what was float16
        assert torch.equal(kept.values(torch.float16).double().cpu(), R.stored(kept))


@pytest.mark.parametrize("signed", [True, False])
def test_checkpoint_borders_and_special_values(signed):
    q = 127.0 if signed else 255.0
    up = float(np.nextafter(np.float32(q), np.float32(1e9)))
    rows = [[0.0] * 33, [q, 0.5, 1.5, 2.5, -0.5], [up, 1.0], [q * 2.0 ** -126, 2.0 ** -126], [2.0 ** -149], [3.4e38, 1.0], [1.0, float("nan")], [float("inf"), 2.0], [-float("inf"), 2.0],
            [-3.0, -7.0], [0.25] * 32 + [float("nan")], [1e-3, 255.0, 254.5, 253.5], [1e-30, 1.0], [float("nan")] * 2]
    x = torch.zeros(len(rows), 33)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    kept = L.checkpoint(x.to(DEV), signed=signed)
    same_checkpoint(kept, x, signed)
    v = kept.values()
    assert torch.equal(torch.isnan(v.cpu()), torch.isnan(R.stored(kept)))
    if not signed:                                          # a positive entry never becomes zero, another one always does
        fin = torch.isfinite(v.cpu())
        assert torch.equal((v.cpu() > 0) & fin, (x > 0) & fin)


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpoint_of_strided_rows(dtype):
    wide = randn(gen(3), 50, 101, dtype=dtype)
    for view in (wide[:, 1:70], wide[::3, 2:3], wide[:, :40].t()):
        same_checkpoint(L.checkpoint(view), view, True)
    assert L.checkpoint(wide.view(5, 10, 101)).rows == 50


def test_no_rows():
    x = torch.zeros((0, 40), device=DEV)
    kept = L.checkpoint(x)
    assert kept.rows == 0 and kept.values().shape == (0, 40)
    y, ky = L.dense_forward(x, torch.ones(3, 40, device=DEV), relu=True)
    assert y.shape == (0, 3) and ky.rows == 0
    dx, dw, db = L.dense_backward(y, kept, torch.ones(3, 40, device=DEV), relu=ky)
    assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (3, 40)
    assert L.lookup(torch.ones(4, 6, device=DEV), torch.zeros(0, dtype=torch.long, device=DEV)).shape == (0, 6)
    assert not L.lookup_backward(torch.ones(0, 6, device=DEV), torch.zeros(0, dtype=torch.long, device=DEV), 70000).any()


# ------------------------------------------------------------------------------------------------------------------------------------------------- dense
SHAPES = [(1, 1, 1), (1, 512, 512), (2, 3, 7), (31, 27, 33), (33, 63, 64), (65, 64, 32), (127, 65, 129), (128, 128, 128), (129, 539, 130), (300, 32, 18), (257, 256, 1), (1000, 96, 260)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", SHAPES)
def test_dense_forward(n, k, o, dtype):
    g = gen(n + 7 * k + 31 * o)
    x, w, b = randn(g, n, k, dtype=dtype), randn(g, o, k, dtype=dtype, scale=k ** -0.5), randn(g, o, dtype=dtype)
    want = x.double() @ w.double().t() + b.double()
    size = x.double().abs() @ w.double().abs().t() + b.double().abs()
    for relu, bias in ((True, b), (False, b), (False, None)):
        y, kept = L.dense_forward(x, w, bias, relu=relu)
        ref = want if bias is not None else want - b.double()
        R.close(y, ref.clamp_min(0) if relu else ref, size, k, dtype)
        same_checkpoint(kept, y, not relu)
        y2, none = L.dense_forward(x, w, bias, relu=relu, keep=False)
        assert none is None and torch.equal(y, y2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", SHAPES)
def test_dense_backward(n, k, o, dtype):
    g = gen(5 + n + 7 * k + 31 * o)
    x, y, w = randn(g, n, k, dtype=dtype), randn(g, n, o, dtype=dtype).clamp_min(0), randn(g, o, k, dtype=dtype, scale=o ** -0.5)
    dy = randn(g, n, o, dtype=dtype) * torch.exp2(-torch.randint(0, 8, (n, 1), generator=g).float()).to(DEV).to(dtype)
    for signed, relu in ((True, False), (False, True)):
        kx, ky = L.checkpoint(x, signed=signed), (L.checkpoint(y, signed=False) if relu else None)
        if relu:                                            # what stands in a closed place does not matter
            dy_in = torch.where(y > 0, dy, torch.full_like(dy, float("nan")))
            dy_in[:, ::3] = torch.where(y[:, ::3] > 0, dy[:, ::3], torch.full_like(dy[:, ::3], float("inf")))
        else:
            dy_in = dy
        dx, dw, db = L.dense_backward(dy_in, kx, w, relu=ky)
        dz = torch.where(y > 0, dy, torch.zeros_like(dy)).double() if relu else dy.double()
        xv = R.stored(kx).to(DEV)
        R.close(dx, dz @ w.double(), dz.abs() @ w.double().abs(), o, dtype)
        R.close(dw, dz.t() @ xv, dz.abs().t() @ xv.abs(), n, dtype)
        R.close(db, dz.sum(0), dz.abs().sum(0), n, dtype)
        dx32, dw32, db32 = L.dense_backward(dy_in, kx, w, relu=ky, need_dx=False, grad_dtype=torch.float32)
        assert dx32 is None
        R.close(dw32, dz.t() @ xv, dz.abs().t() @ xv.abs(), n, torch.float32)
        R.close(db32, dz.sum(0), dz.abs().sum(0), n, torch.float32)
        again = L.dense_backward(dy_in, kx, w, relu=ky)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))      # the same bits every time
        only = L.dense_backward(dy_in, kx, w, relu=ky, need_dw=False, need_db=False)
        assert only[1] is None and only[2] is None and torch.equal(only[0], dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", [(33001, 70, 130), (32900, 40, 24), (40000, 3, 300), (33000, 200, 512)])
def test_dense_many_rows(n, k, o, dtype):
    """more row tiles than compute units: the forms for many rows, ragged in every size"""
    g = gen(n + k + o)
    x, w, b = randn(g, n, k, dtype=dtype), randn(g, o, k, dtype=dtype, scale=k ** -0.5), randn(g, o, dtype=dtype)
    y, kept = L.dense_forward(x, w, b, relu=True)
    R.close(y, (x.double() @ w.double().t() + b.double()).clamp_min(0), x.double().abs() @ w.double().abs().t() + b.double().abs(), k, dtype)
    again = L.checkpoint(y, signed=False)                   # (held to the definition above)
    assert torch.equal(kept.codes, again.codes) and torch.equal(kept.scales, again.scales)
    dy = randn(g, n, o, dtype=dtype)
    kx = L.checkpoint(x)
    dx, dw, db = L.dense_backward(torch.where(y > 0, dy, torch.full_like(dy, float("nan"))), kx, w, relu=kept)
    dz, xv = torch.where(y > 0, dy, torch.zeros_like(dy)).double(), kx.values().double()
    R.close(dx, dz @ w.double(), dz.abs() @ w.double().abs(), o, dtype)
    R.close(dw, dz.t() @ xv, dz.abs().t() @ xv.abs(), n // 4, dtype)
    R.close(db, dz.sum(0), dz.abs().sum(0), n // 4, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", [(4096, 32, 32), (4095, 32, 32), (5003, 5, 26), (4100, 33, 3), (9001, 280, 5), (6007, 31, 177), (4099, 1, 33), (33100, 26, 18), (33000, 8, 1), (33000, 160, 8), (8229, 26, 500), (8200, 511, 31), (8193, 4, 7), (33001, 511, 31), (32769, 32, 33), (700, 30, 7), (1500, 200, 20), (1025, 9, 140)])
def test_dense_narrow_layers(n, k, o, dtype):
    """many rows of a layer with at most 32 inputs or outputs, and its borders"""
    g = gen(n + 3 * k + 5 * o)
    x, w, b = randn(g, n, k, dtype=dtype), randn(g, o, k, dtype=dtype, scale=k ** -0.5), randn(g, o, dtype=dtype)
    for relu in (True, False):
        y, kept = L.dense_forward(x, w, b, relu=relu)
        want = x.double() @ w.double().t() + b.double()
        R.close(y, want.clamp_min(0) if relu else want, x.double().abs() @ w.double().abs().t() + b.double().abs(), k, dtype)
        again = L.checkpoint(y, signed=not relu)                   # (held to the definition above)
        assert torch.equal(kept.codes, again.codes) and torch.equal(kept.scales, again.scales)
        alone, none = L.dense_forward(x, w, b, relu=relu, keep=False)
        assert none is None and torch.equal(alone, y)
        dy = randn(g, n, o, dtype=dtype)
        kx = L.checkpoint(x)
        dx, dw, db = L.dense_backward(torch.where(y > 0, dy, torch.full_like(dy, float("nan"))) if relu else dy, kx, w, relu=kept if relu else None)
        dz, xv = (torch.where(y > 0, dy, torch.zeros_like(dy)) if relu else dy).double(), kx.values().double()
        R.close(dx, dz @ w.double(), dz.abs() @ w.double().abs(), o, dtype)
        R.close(dw, dz.t() @ xv, dz.abs().t() @ xv.abs(), n // 4, dtype)
        R.close(db, dz.sum(0), dz.abs().sum(0), n // 4, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_long_reduction(dtype):
    """many rows: the pieces of the weight gradient and their sum; 70 001 rows, more than one launch tile of each kind"""
    g = gen(11)
    n, k, o = 70001, 40, 24
    x, dy = randn(g, n, k, dtype=dtype).clamp_min(0), randn(g, n, o, dtype=dtype)
    w = randn(g, o, k, dtype=dtype)
    kx = L.checkpoint(x, signed=False)
    dx, dw, db = L.dense_backward(dy, kx, w)
    xv = R.stored(kx).to(DEV)
    R.close(dx, dy.double() @ w.double(), dy.double().abs() @ w.double().abs(), o, dtype)
    # (a piece adds at most n / splits terms in one chain and the pieces add up after that: the bound counts a quarter of the rows)
    R.close(dw, dy.double().t() @ xv, dy.double().abs().t() @ xv.abs(), n // 4, dtype)
    R.close(db, dy.double().sum(0), dy.double().abs().sum(0), n // 4, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_strided_and_odd_rows(dtype):
    g = gen(12)
    wide, ww, gy = randn(g, 70, 203, dtype=dtype), randn(g, 45, 121, dtype=dtype), randn(g, 70, 91, dtype=dtype)
    x, w, dy = wide[:, 3:104], ww[::2, 7:108], gy[:, 5:28]
    y, kept = L.dense_forward(x, w, None, relu=True)
    assert y.shape == (70, 23)
    R.close(y, (x.double() @ w.double().t()).clamp_min(0), x.double().abs() @ w.double().abs().t(), 101, dtype)
    yc, _ = L.dense_forward(x.contiguous(), w.contiguous(), None, relu=True)
    assert torch.equal(y, yc)
    kx = L.checkpoint(x)
    a = L.dense_backward(dy, kx, w, relu=kept)
    b = L.dense_backward(dy.contiguous(), kx, w.contiguous(), relu=kept)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y3, k3 = L.dense_forward(wide.view(7, 10, 203)[..., 3:104], w, None, relu=True)
    assert y3.shape == (7, 10, 23) and torch.equal(y3.reshape(70, 23), y) and torch.equal(k3.codes, kept.codes)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_non_finite(dtype):
    """a NaN passes the ReLU and shows; other rows are untouched; a NaN block of the output's checkpoint counts as open, of the input's poisons its columns' weight gradients"""
    g = gen(13)
    x, w, b = randn(g, 40, 50, dtype=dtype), randn(g, 36, 50, dtype=dtype), randn(g, 36, dtype=dtype)
    clean, kc = L.dense_forward(x, w, b, relu=True)
    x2 = x.clone()
    x2[7, 3] = float("nan")
    y, ky = L.dense_forward(x2, w, b, relu=True)
    assert torch.isnan(y[7]).all()
    rest = torch.arange(40, device=DEV) != 7
    assert torch.equal(y[rest], clean[rest]) and torch.equal(ky.codes[rest], kc.codes[rest])
    assert (ky.scales[7] == 255).all() and torch.isnan(ky.values()[7]).all()
    kx = L.checkpoint(x2)
    dy = randn(g, 40, 36, dtype=dtype)
    dx, dw, db = L.dense_backward(dy, kx, w, relu=ky)
    assert torch.isnan(dw[:, :32]).all() and torch.isfinite(dw[:, 32:]).all() and torch.isfinite(dx).all() and torch.isfinite(db).all()
    dz = torch.where((clean > 0) | ~rest[:, None], dy, torch.zeros_like(dy)).double()
    R.close(dx, dz @ w.double(), dz.abs() @ w.double().abs(), 36, dtype)


def test_dense_small_magnitudes_in_float16():
    """float16 subnormals are operands like any others (activations and their checkpoint's values)"""
    x = torch.full((33, 32), 2.0 ** -24, dtype=torch.float16, device=DEV)
    x[:, 1] = 2.0 ** -20
    w = torch.full((5, 32), 1024.0, dtype=torch.float16, device=DEV)
    y, _ = L.dense_forward(x, w)
    assert torch.equal(y, torch.full_like(y, (31 * 2.0 ** -24 + 2.0 ** -20) * 1024))
    kx = L.checkpoint(x, signed=False)
    assert torch.equal(kx.values(torch.float16), x)
    dy = torch.full((33, 5), 512.0, dtype=torch.float16, device=DEV)
    _, dw, _ = L.dense_backward(dy, kx, w, grad_dtype=torch.float32)
    assert torch.equal(dw[0], (x[0].double() * 512 * 33).float())


def test_dense_autograd_against_the_formula_and_differences():
    """small whole numbers: the checkpoint holds them exactly, so the gradient is the layer's own — float64 autograd's, and that of differences (y is linear in each weight while
    no ReLU changes sides: a step of 2^-4 on sums at least 1/2 away from zero, exact in float32)"""
    g = gen(21)
    x = torch.randint(-7, 8, (37, 20), generator=g).float().to(DEV)
    w = (torch.randint(-3, 4, (9, 20), generator=g).float()).to(DEV).requires_grad_(True)
    b = (torch.randint(-3, 4, (9,), generator=g).float() + 0.5).to(DEV).requires_grad_(True)
    up = torch.randint(-4, 5, (37, 9), generator=g).float().to(DEV)
    xr = x.clone().requires_grad_(True)
    y, kept = L.dense(xr, w, b, relu=True)
    (y * up).sum().backward()
    x6, w6, b6 = x.double().requires_grad_(True), w.detach().double().requires_grad_(True), b.detach().double().requires_grad_(True)
    (torch.relu(x6 @ w6.t() + b6) * up.double()).sum().backward()
    for got, want in ((xr.grad, x6.grad), (w.grad, w6.grad), (b.grad, b6.grad)):
        assert torch.equal(got.double(), want)              # every sum is a whole number below 2^24
    h = 2.0 ** -6
    for i, j in ((0, 0), (3, 7), (8, 19)):
        f = []
        for s in (h, -h):
            wp = w.detach().clone()
            wp[i, j] += s
            f.append(float((L.dense_forward(x, wp, b, relu=True, keep=False)[0].double() * up.double()).sum()))
        assert abs((f[0] - f[1]) / (2 * h) - float(w.grad[i, j])) <= 1e-9


def test_dense_autograd_mixed_types_and_chain():
    """float32 parameters beside bfloat16 activations; two layers, the second reading the checkpoint that the first wrote; leaves that need no gradient"""
    g = gen(22)
    x = randn(g, 90, 48, dtype=torch.bfloat16)
    w1, b1 = randn(g, 70, 48, scale=0.2).requires_grad_(True), randn(g, 70).requires_grad_(True)
    w2 = randn(g, 33, 70, scale=0.2).requires_grad_(True)
    y1, k1 = L.dense(x, w1, b1, relu=True)
    y2, k2 = L.dense(y1, w2, None, kept=k1)
    assert y2.dtype == torch.bfloat16 and k2.signed and not k1.signed
    up = randn(g, 90, 33, dtype=torch.bfloat16)
    (y2 * up).sum().backward()
    assert w1.grad.dtype == torch.float32 and x.grad is None
    dw2 = up.double().t() @ R.stored(k1).to(DEV)
    R.close(w2.grad, dw2, up.double().abs().t() @ R.stored(k1).to(DEV).abs(), 90, torch.float32)
    dy1 = (up.double() @ w2.detach().to(torch.bfloat16).double()).to(torch.bfloat16).double()     # (rounded to the activations' type between the layers)
    dz1 = torch.where(y1 > 0, dy1, torch.zeros_like(dy1))
    kx = L.checkpoint(x)
    want = dz1.t() @ R.stored(kx).to(DEV)
    # dy1 above is rounded from a float64 product, the layer's from a float32 one: where the two round apart the entry is off by a whole step (2^-8), counted on the sum of
    # magnitudes
    off = (w1.grad.double() - want).abs()
    assert (off <= 2.0 ** -8 * (dz1.abs().t() @ R.stored(kx).to(DEV).abs()) + 1e-6).all()
    assert float(off.norm() / want.norm()) < 2.0 ** -9      # ... but hardly any do


def test_dense_refuses():
    x = torch.zeros(4, 8, device=DEV)
    w = torch.zeros(3, 8, device=DEV)
    k = L.checkpoint(x)
    for bad in (lambda: L.dense_forward(x, torch.zeros(3, 7, device=DEV)), lambda: L.dense_forward(x, w, torch.zeros(4, device=DEV)), lambda: L.dense_forward(x, w[:0]),
                lambda: L.dense_forward(x, torch.zeros(3, 8)), lambda: L.dense_backward(torch.zeros(5, 3, device=DEV), k, w), lambda: L.dense_backward(torch.zeros(4, 2, device=DEV), k, w),
                lambda: L.dense_backward(torch.zeros(4, 3, device=DEV), k, w, relu=k), lambda: L.dense(x, w, kept=L.checkpoint(x[:2]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: L.dense_forward(x, w.half()), lambda: L.dense_forward(x, w, torch.zeros(3, device=DEV).half()),
                lambda: L.dense_backward(torch.zeros(4, 3, device=DEV).half(), k, w.half(), grad_dtype=torch.bfloat16)):
        with pytest.raises(TypeError):
            bad()


# ------------------------------------------------------------------------------------------------------------------------------------------------ lookup
@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,per,v,d", [(1, 1, 1, 1), (5, 3, 7, 9), (100, 1, 200, 48), (33, 64, 4, 32), (1000, 7, 70000, 3), (4097, 1, 50, 65), (9000, 2, 600, 8), (3, 1, 5, 520)])
def test_lookup_and_gradient(n, per, v, d, dtype, bits):
    g = gen(n + per + v + d)
    table = randn(g, v, d, dtype=dtype)
    index = torch.randint(-1, v, (n,), generator=g).to(bits).to(DEV)
    out = L.lookup(table, index, scale=0.37, rows_per_index=per)
    rows = index.long().repeat_interleave(per)
    s = float(np.float32(0.37))
    want = torch.where(rows[:, None] < 0, torch.zeros((), dtype=torch.float64, device=DEV), table.double()[rows.clamp_min(0)] * s)
    R.close(out, want, want.abs(), 0, dtype)
    dout = randn(g, n * per, d, dtype=dtype)
    got = L.lookup_backward(dout, index, v, scale=0.37, rows_per_index=per)
    ok = rows >= 0
    ref = torch.zeros((v, d), dtype=torch.float64, device=DEV).index_add_(0, rows[ok], dout.double()[ok]) * s
    size = torch.zeros((v, d), dtype=torch.float64, device=DEV).index_add_(0, rows[ok], dout.double()[ok].abs()) * s
    most = int(torch.bincount(rows[ok], minlength=1).max()) if ok.any() else 0
    R.close(got, ref, size, most, dtype)
    assert torch.equal(got, L.lookup_backward(dout, index, v, scale=0.37, rows_per_index=per))


@pytest.mark.parametrize("n,per", [(4096, 1), (4096, 192), (4097, 1), (50000, 3)])
def test_lookup_gradient_of_one_token(n, per):
    """every row has the same token: one run over all pieces (values of one size so that the bound is tight)"""
    dout = torch.randint(-8, 9, (n * per, 24), generator=gen(31)).float().to(DEV)
    index = torch.full((n,), 5, dtype=torch.long, device=DEV)
    got = L.lookup_backward(dout, index, 9, rows_per_index=per)
    want = torch.zeros((9, 24), dtype=torch.float64, device=DEV)
    want[5] = dout.double().sum(0)
    assert torch.equal(got.double(), want)                  # whole numbers below 2^24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,per,v,d", [(4096, 1, 1024, 24), (4096, 2, 1025, 24), (4095, 1, 5003, 3), (64, 128, 131072, 9), (64, 128, 131073, 9), (7, 1, 100000, 300), (1, 1, 2049, 1030),
                                       (2000, 4, 1500, 70), (4096, 1, 3, 2), (4096, 2, 1, 256), (90, 91, 2, 33), (5000, 1, 40, 2056), (16384, 1, 257, 5), (16384, 4, 70000, 31), (16385, 1, 300, 5), (341, 192, 3000, 20)])
def test_lookup_gradient_of_clustered_tokens(n, per, v, d, dtype):
    """most positions on few tokens that lie side by side (one workgroup's range), one of them with half of all: whole numbers, so that every sum is exact"""
    g = gen(n + per + v + d)
    index = torch.randint(0, min(v, 40), (n,), generator=g)
    index[torch.rand(n, generator=g) < 0.5] = min(v - 1, 17)
    index[torch.rand(n, generator=g) < 0.05] = v - 1
    index[torch.rand(n, generator=g) < 0.05] = -1
    index = index.to(DEV)
    dout = torch.randint(-2, 3, (n * per, d), generator=g).to(DEV)
    rows = index.repeat_interleave(per)
    want = torch.zeros((v, d), dtype=torch.float64, device=DEV).index_add_(0, rows.clamp_min(0), torch.where(rows[:, None] >= 0, dout, torch.zeros_like(dout)).double())
    assert float(want.abs().max()) < 2 ** 24
    got = L.lookup_backward(dout.to(dtype), index, v, rows_per_index=per)
    assert torch.equal(got, want.to(dtype))                  # (float64 holds the sums, and one rounding is what the operator does)


def test_lookup_indices_outside_the_table():
    table = randn(gen(32), 6, 10)
    index = torch.tensor([0, -1, 6, 5, -(1 << 40), 1 << 40, 2], device=DEV)
    out = L.lookup(table, index, scale=2.0)
    assert torch.equal(out[[0, 3, 6]], 2 * table[[0, 5, 2]]) and not out[[1, 4]].any() and torch.isnan(out[[2, 5]]).all()
    dout = randn(gen(33), 7, 10)
    dout[1] = float("nan")
    got = L.lookup_backward(dout, index, 6)
    want = torch.zeros_like(table)
    want[0], want[5], want[2] = dout[0], dout[3], dout[6]
    assert torch.equal(got, want)
    assert not L.lookup_backward(dout, torch.full((7,), -1, dtype=torch.long, device=DEV), 6).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_into_a_slice_and_from_strided_rows(dtype):
    """the codes written beside the direction encoding, the gradient read from there; the neighbours stay as they were"""
    wide = torch.full((60, 45), 7.0, dtype=dtype, device=DEV)
    table = randn(gen(34), 9, 31, dtype=dtype)[:, 2:15]
    index = torch.randint(0, 9, (20,), generator=gen(35)).to(DEV)
    out = L.lookup(table, index, scale=0.5, rows_per_index=3, out=wide[:, 27:40])
    assert torch.equal(out, L.lookup(table.contiguous(), index, scale=0.5, rows_per_index=3))
    assert (wide[:, :27] == 7).all() and (wide[:, 40:] == 7).all()
    a = L.lookup_backward(wide[:, 27:40], index, 9, rows_per_index=3)
    assert torch.equal(a, L.lookup_backward(wide[:, 27:40].contiguous(), index, 9, rows_per_index=3))


def test_lookup_autograd_against_differences():
    table = torch.randint(-5, 6, (7, 6), generator=gen(36)).float().to(DEV).requires_grad_(True)
    index = torch.tensor([[1, 1], [3, -1], [6, 1]], device=DEV)
    up = torch.randint(-5, 6, (3, 4, 6), generator=gen(37)).float().to(DEV)
    out = L.lookup(table, index, scale=0.5, rows_per_index=2)
    assert out.shape == (3, 4, 6)
    (out * up).sum().backward()
    for i, j in ((1, 0), (3, 5), (0, 2), (6, 1)):
        f = []
        for s in (1.0, -1.0):
            t = table.detach().clone()
            t[i, j] += s
            f.append(float((L.lookup(t, index, scale=0.5, rows_per_index=2) * up).sum()))
        assert (f[0] - f[1]) / 2 == float(table.grad[i, j])


def test_lookup_refuses():
    t, i = torch.zeros(4, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    for bad in (lambda: L.lookup(t[:0], i), lambda: L.lookup(t, i, rows_per_index=0), lambda: L.lookup(t, i.cpu()), lambda: L.lookup(t, i, out=torch.zeros(4, 8, device=DEV)),
                lambda: L.lookup_backward(torch.zeros(4, 8, device=DEV), i, 4), lambda: L.lookup_backward(torch.zeros(3, 8, device=DEV), i, 0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        L.lookup(t, i.float())
    with pytest.raises(TypeError):
        L.lookup(t, i, out=torch.zeros(3, 8, device=DEV).half())


# ------------------------------------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.parametrize("dtype,n,k,o", [(torch.bfloat16, 8400000, 520, 520), (torch.float32, 2200000, 500, 500), (torch.bfloat16, 150000000, 30, 20)])
def test_offsets_beyond_32_bits(dtype, n, k, o):
    """the last rows of tensors of more than 4 GB (more than 2^32 elements in 16 bits) are what a call on those rows alone gives, bit for bit (40 000: the same form of the kernels)"""
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    tail = 40000
    w, b = torch.randn(o, k, generator=g, device=DEV).to(dtype), torch.randn(o, generator=g, device=DEV).to(dtype)
    x = torch.zeros(n, k, dtype=dtype, device=DEV)
    x[-tail:] = torch.randn(tail, k, generator=g, device=DEV).to(dtype)
    y, kept = L.dense_forward(x, w, b, relu=True)
    y2, kept2 = L.dense_forward(x[-tail:].clone(), w, b, relu=True)
    assert torch.equal(y[-tail:], y2) and torch.equal(kept.codes[-tail:], kept2.codes) and torch.equal(kept.scales[-tail:], kept2.scales)
    assert torch.equal(y[0], b.clamp_min(0)) and torch.equal(y[n // 2], y[0])
    kx, kx2 = L.checkpoint(x), L.checkpoint(x[-tail:].clone())
    assert torch.equal(kx.codes[-tail:], kx2.codes) and torch.equal(kx.scales[-tail:], kx2.scales)
    del x, y2
    vals = kx.values(dtype)
    assert torch.equal(vals[-tail:], kx2.values(dtype)) and not vals[0].any()
    del vals
    dy = torch.zeros_like(y)
    del y
    dy[-tail:] = torch.randn(tail, o, generator=g, device=DEV).to(dtype)
    dx, dw, db = L.dense_backward(dy, kx, w, relu=kept, grad_dtype=torch.float32)
    dx2, dw2, db2 = L.dense_backward(dy[-tail:].clone(), kx2, w, relu=kept2, grad_dtype=torch.float32)
    assert torch.equal(dx[-tail:], dx2) and not dx[0].any()
    for p, q in ((dw, dw2), (db, db2)):          # (other pieces: float32 sums of 40 000 terms in another order, 200 of them in one chain at random)
        assert (p - q).abs().max() <= 2e-4 * q.abs().max()


def test_lookup_offsets_beyond_32_bits():
    n, per, d = 400000, 192, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    table, index = torch.randn(50, d, generator=g, device=DEV).half(), torch.randint(0, 50, (n,), generator=g, device=DEV)
    out = L.lookup(table, index, 1.0, per)
    assert torch.equal(out[-per * 1000:], table[index[-1000:].repeat_interleave(per)]) and torch.equal(out[0], table[index[0]])
    out.zero_()
    out[-per * 1000:] = torch.randint(-1, 2, (per * 1000, d), generator=g, device=DEV).half()
    got = L.lookup_backward(out, index, 50, 1.0, per)
    want = torch.zeros(50, d, dtype=torch.float64, device=DEV).index_add_(0, index[-1000:].repeat_interleave(per), out[-per * 1000:].double())
    assert torch.equal(got, want.half())          # (whole numbers)


# ------------------------------------------------------------------------------------------------------------------------------ the C boundary: strided rows, what lies around them
class Guarded:
    """rows x cols elements with a row stride, 64 KB of sentinel bytes before and behind, sentinels between the rows"""

    def __init__(self, rows, cols, dtype, ld=None, values=None, fill=0xA5):
        self.rows, self.cols, self.ld = rows, cols, ld or cols
        size = torch.empty((), dtype=dtype).element_size()
        n = ((rows - 1) * self.ld + cols if rows else 0) * size
        self.raw = torch.full((65536 + n + 65536,), fill, dtype=torch.uint8, device=DEV)
        self.view = self.raw[65536:65536 + n].view(dtype).as_strided((rows, cols), (self.ld, 1)) if n else torch.empty((0, cols), dtype=dtype, device=DEV)
        self.ptr = self.raw.data_ptr() + 65536
        self.fill = fill
        if values is not None:
            self.view.copy_(values)

    def intact(self):
        """are all bytes but the rows' own still the sentinel?"""
        mine = torch.zeros(self.raw.numel(), dtype=torch.bool, device=DEV)
        if self.rows:
            size = self.view.element_size()
            mine[65536:mine.numel() - 65536].as_strided((self.rows, self.cols * size), (self.ld * size, 1)).fill_(True)
        return bool((self.raw[~mine] == self.fill).all())


def call(name, *args):
    import _pkg
    B = _pkg.load().binding
    B.check_layers(getattr(B.load_library(), name)(torch.cuda.current_stream().cuda_stream, *args))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", [(3, 5, 7), (200, 70, 33), (1003, 539, 512), (8300, 65, 130), (8300, 65, 260), (33000, 70, 130), (33000, 26, 18), (40000, 130, 5), (33000, 64, 300)])
def test_nothing_else_is_read_or_written(n, k, o, dtype):
    """through the C boundary: rows with a stride, NaN between and behind the inputs' rows, sentinels around the outputs — the same bits as for contiguous rows, the sentinels untouched"""
    lib = _pkg.load().binding.load_library()
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    g = gen(n + k + o)
    x, w, b, dy = randn(g, n, k, dtype=dtype).clamp_min(0), randn(g, o, k, dtype=dtype, scale=k ** -0.5), randn(g, o, dtype=dtype), randn(g, n, o, dtype=dtype)
    gx, gw, gdy = (Guarded(*t.shape, dtype, t.shape[1] + pad, t, fill=0xFF) for t, pad in ((x, 3), (w, 5), (dy, 1)))       # (bytes 0xff: NaN in every type)
    ko, kk = (o + 31) // 32, (k + 31) // 32
    y, kept = L.dense_forward(x, w, b, relu=True)
    gy, gc, gs = Guarded(n, o, dtype, o + 9), Guarded(n, 32 * ko, torch.uint8), Guarded(n, ko, torch.uint8)
    need = lib.iblnerf_dense_forward_workspace(code, n, k, o)
    ws = Guarded(1, max(need, 1), torch.uint8)
    call("iblnerf_dense_forward", code, gx.ptr, k + 3, n, k, gw.ptr, k + 5, o, b.data_ptr(), 1, gy.ptr, o + 9, gc.ptr, gs.ptr, ws.ptr, need)
    assert torch.equal(gy.view, y) and torch.equal(gc.view, kept.codes) and torch.equal(gs.view, kept.scales)
    kx = L.checkpoint(x, signed=False)
    gxc, gxs, gyc = Guarded(n, 32 * kk, torch.uint8, values=kx.codes), Guarded(n, kk, torch.uint8, values=kx.scales), Guarded(n, 32 * ko, torch.uint8, values=kept.codes)
    cc, cs = Guarded(n, 32 * kk, torch.uint8), Guarded(n, kk, torch.uint8)
    call("iblnerf_checkpoint", code, gx.ptr, k + 3, n, k, 0, cc.ptr, cs.ptr)
    assert torch.equal(cc.view, kx.codes) and torch.equal(cs.view, kx.scales)
    dx, dw, db = L.dense_backward(dy, kx, w, relu=kept)
    gdx, gdw, gdb = Guarded(n, k, dtype, k + 2), Guarded(o, k, dtype), Guarded(1, o, dtype)
    need = lib.iblnerf_dense_backward_workspace(code, n, k, o)
    ws2 = Guarded(1, max(need, 1), torch.uint8)
    call("iblnerf_dense_backward", code, gdy.ptr, o + 1, n, k, o, gxc.ptr, gxs.ptr, 0, gyc.ptr, gw.ptr, k + 5, gdx.ptr, k + 2, code, gdw.ptr, gdb.ptr, ws2.ptr, need)
    assert torch.equal(gdx.view, dx) and torch.equal(gdw.view, dw) and torch.equal(gdb.view[0], db)
    vals = Guarded(n, k, dtype, k + 6)
    call("iblnerf_checkpoint_values", gxc.ptr, gxs.ptr, n, k, 0, code, vals.ptr, k + 6)
    assert torch.equal(vals.view, kx.values(dtype))
    for t in (gx, gw, gdy, gy, gc, gs, ws, cc, cs, gdx, gdw, gdb, ws2, gxc, gxs, gyc, vals):
        assert t.intact()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,per,v,d", [(5, 3, 7, 9), (4096, 1, 200, 48), (300, 7, 900, 13), (17000, 1, 5000, 21), (2000, 64, 300, 33), (20000, 2, 9, 3)])
def test_lookups_read_and_write_nothing_else(n, per, v, d, dtype):
    lib = _pkg.load().binding.load_library()
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    g = gen(n + per + v + d)
    table, dout, index = randn(g, v, d, dtype=dtype), randn(g, n * per, d, dtype=dtype), torch.randint(-1, v, (n,), generator=g).to(DEV)
    gt, gd = Guarded(v, d, dtype, d + 3, table, fill=0xFF), Guarded(n * per, d, dtype, d + 5, dout, fill=0xFF)
    out = Guarded(n * per, d, dtype, d + 7)
    call("iblnerf_lookup", code, gt.ptr, d + 3, v, d, index.data_ptr(), 64, n, per, 0.5, out.ptr, d + 7)
    assert torch.equal(out.view, L.lookup(table, index, 0.5, per))
    need = lib.iblnerf_lookup_backward_workspace(n, per, v, d)
    ws, grad = Guarded(1, max(need, 1), torch.uint8), Guarded(v, d, dtype)
    call("iblnerf_lookup_backward", code, gd.ptr, d + 5, index.data_ptr(), 64, n, per, v, d, 0.5, grad.ptr, ws.ptr, need)
    assert torch.equal(grad.view, L.lookup_backward(dout, index, v, 0.5, per))
    for t in (gt, gd, out, ws, grad):
        assert t.intact()


# ------------------------------------------------------------------------------------------------------------------------------ streams, graphs, together
def _step(table, index, x, w1, w2):
    """codes beside the input, two layers, their gradients: what a training step does with the operators together"""
    n, k, d = x.shape[0], x.shape[1], table.shape[1]
    wide = torch.empty((n, k + d), dtype=x.dtype, device=x.device)
    wide[:, :k].copy_(x)
    L.lookup(table, index, scale=0.25, rows_per_index=n // index.numel(), out=wide[:, k:])
    kx = L.checkpoint(wide)
    y1, k1 = L.dense_forward(wide, w1, relu=True)
    y2, _ = L.dense_forward(y1, w2)
    dy1, dw2, db2 = L.dense_backward(y2, k1, w2)
    dwide, dw1, db1 = L.dense_backward(dy1, kx, w1, relu=k1)
    return y2, dw2, db2, dw1, db1, L.lookup_backward(dwide[:, k:], index, table.shape[0], scale=0.25, rows_per_index=n // index.numel())


def _step_inputs(seed, dtype):
    g = gen(seed)
    return (randn(g, 30, 16, dtype=dtype), torch.randint(0, 30, (6000,), generator=g).to(DEV), randn(g, 12000, 50, dtype=dtype), randn(g, 96, 66, dtype=dtype, scale=0.1),
            randn(g, 40, 96, dtype=dtype, scale=0.1))


@pytest.mark.parametrize("dtype", TYPES)
def test_together(dtype):
    table, index, x, w1, w2 = _step_inputs(41, dtype)
    y2, dw2, db2, dw1, db1, dtable = _step(table, index, x, w1, w2)
    codes = (table.double() * 0.25).to(dtype)[index].repeat_interleave(2, 0)
    wide = torch.cat([x, codes], 1)
    y1 = torch.relu(wide.double() @ w1.double().t()).to(dtype).double()
    z2 = (y1 @ w2.double().t()).to(dtype).double()
    tol = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -9}[dtype]      # two roundings to the type in a row, norms
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())      # noqa: E731
    assert rel(y2, z2) <= tol
    # the backward pass reads the activations in 8 bits (a block's step is at most 2^-6 of its largest entry, an entry off by half of it, independently): 2^-6 on norms
    dy1 = z2 @ w2.double()
    dz1 = torch.where(y1 > 0, dy1, torch.zeros_like(dy1))
    assert rel(dw2, z2.t() @ y1) <= 2.0 ** -6 + tol and rel(dw1, dz1.t() @ wide.double()) <= 2.0 ** -6 + tol
    dc = (dz1 @ w1.double())[:, 50:].reshape(6000, 2, 16).sum(1)
    assert rel(dtable, torch.zeros((30, 16), dtype=torch.float64, device=DEV).index_add_(0, index, dc) * 0.25) <= 2.0 ** -6 + tol


def test_another_stream_and_two_at_once():
    a, b = _step_inputs(42, torch.bfloat16), _step_inputs(43, torch.float16)
    want_a, want_b = _step(*a), _step(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            got_a = _step(*a)
        with torch.cuda.stream(s2):
            got_b = _step(*b)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got_a, want_a)) and all(torch.equal(p, q) for p, q in zip(got_b, want_b))


def test_captured_and_replayed():
    """two graphs of the same calls, replayed in turn with new inputs and eager work between"""
    sets = [_step_inputs(s, torch.bfloat16) for s in (44, 45)]
    bufs = [tuple(t.clone() for t in s) for s in sets]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(*bufs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for b in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_step(*b))
        graphs.append(gr)
    for r in range(4):
        for i in (0, 1):
            src = sets[(i + r) % 2]
            for t, v in zip(bufs[i], src):
                t.copy_(v)
            graphs[i].replay()
            want = _step(*src)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs[i], want))
