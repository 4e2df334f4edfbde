"""Checkpoints at the upper end of their types' ranges: what a finite activation's codes stand for is finite, and the weight gradient reads just that."""
import pytest
import torch

import _pkg
import layers_ref as R

pytestmark = pytest.mark.gpu
L = _pkg.load().layers
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
MOST = {torch.float32: 255 * 2.0 ** 120, torch.bfloat16: 255 * 2.0 ** 120, torch.float16: 65504.0}


def read_as(kept, dtype):
    """The definition's values in `dtype`: one step beyond the type's range is the type's largest (bfloat16's for float32, whose products take a checkpoint's value as one)."""
    v = R.stored(kept)
    beyond = 65536.0 if dtype == torch.float16 else 2.0 ** 128
    return torch.where(v.abs() == beyond, v.sign() * MOST[dtype], v).to(dtype)


def large_rows(dtype, signed):
    """a block of small and large entries of both signs for each of these maxima"""
    top = torch.finfo(dtype).max
    tops = [top, top * (1 - 2.0 ** -7), 65280.0, 65296.0, 65504.0, 65024.0, 65056.0, 32512.0, 32768.0, 512.0]
    if dtype != torch.float16:
        tops += [1.8e38, 1.6e38, 127 * 2.0 ** 120, 128 * 2.0 ** 120, 127 * 2.0 ** 121, 254.5 * 2.0 ** 120, 255 * 2.0 ** 120, 2.0 ** 126, 1e38, 70000.0]
    g = torch.Generator().manual_seed(6)
    x = torch.empty((len(tops), 40), dtype=torch.float64)
    for i, m in enumerate(tops):
        x[i] = m * (torch.rand(40, generator=g, dtype=torch.float64) * 2 - 1)
        x[i, 3], x[i, 5], x[i, 7], x[i, 35] = m, -m, 0.0, m
    x = x.clamp(-top, top).to(dtype)
    return x if signed else x.clamp_min(0)


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_of_large_blocks(dtype, signed):
    x = large_rows(dtype, signed)
    kept = L.checkpoint(x.to(DEV), signed=signed)
    c, e = R.pack(x, signed)
    got_c, got_e = R.raw(kept)
    assert (got_c == c).all() and (got_e == e).all()
    for t in TYPES:
        got, want = kept.values(t).cpu(), read_as(kept, t)
        assert torch.equal(got, want)
        if t != torch.float16 or dtype == torch.float16:
            assert torch.isfinite(got).all()
    # half a step; a positive entry of an unsigned checkpoint that keeps code 1: a step
    step, one = torch.from_numpy(2.0 ** e).repeat_interleave(32, 1)[:, :40], torch.from_numpy(c == 1)[:, :40]
    assert ((kept.values(dtype).double().cpu() - x.double()).abs() <= torch.where(one & (not signed), step, step / 2)).all()


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,o", [(1, 1), (1, 40), (3, 200), (66000, 3), (66000, 200)])
def test_weight_gradient_of_large_blocks(n, o, dtype, signed):
    """one row of dY is 1, the others 0: dW is that row's values, with no rounding (a tile of every width; 66 000 rows of 216 or more columns: the widest)"""
    rows = large_rows(dtype, signed)
    wide = torch.cat([rows, torch.zeros(rows.shape[0], 24, dtype=dtype)], 1)                  # [., 64]
    for r0 in range(0, rows.shape[0], 4):
        x = wide[r0:r0 + 4].reshape(1, -1)                                                    # up to 256 columns
        k = x.shape[1]
        kept = L.checkpoint(x.to(DEV), signed=signed)
        codes, scales = torch.zeros(n, kept.codes.shape[1], dtype=torch.uint8, device=DEV), torch.full((n, kept.scales.shape[1]), 127, dtype=torch.uint8, device=DEV)
        codes[-1], scales[-1] = kept.codes[0], kept.scales[0]
        dy = torch.zeros(n, o, dtype=dtype, device=DEV)
        dy[-1] = 1
        _, dw, db = L.dense_backward(dy, L.Checkpoint(codes, scales, k, signed), torch.zeros(o, k, dtype=dtype, device=DEV), need_dx=False, grad_dtype=torch.float32)
        want = read_as(kept, dtype).float()
        assert torch.equal(dw.cpu(), want.expand(o, k)) and (db == 1).all()


def test_a_bad_block_is_nan_beside_large_ones():
    x = torch.full((2, 64), 3e38, device=DEV)
    x[1, 40] = float("inf")
    for signed in (True, False):
        v = L.checkpoint(x, signed=signed).values()
        assert torch.isfinite(v[0]).all() and torch.isfinite(v[1, :32]).all() and torch.isnan(v[1, 32:]).all()


def test_a_written_slice_is_an_in_place_write():
    """what an operation kept of a tensor for its backward pass is gone once codes are written into it: torch's own error, not the gradient of other numbers"""
    table, index = torch.randn(5, 6, device=DEV), torch.tensor([1, 4, 0], device=DEV)
    wide, w = torch.randn(3, 10, device=DEV), torch.randn(10, 4, device=DEV, requires_grad=True)
    y = (wide @ w).sum()
    L.lookup(table, index, out=wide[:, 4:])
    assert torch.equal(wide[:, 4:], table[index])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    (wide @ w).sum().backward()
    with pytest.raises(ValueError, match="require a gradient"):
        L.lookup(table, index, out=torch.ones(3, 6, device=DEV) * w[0, 0])
    with torch.no_grad():
        L.lookup(table, index, out=torch.ones(3, 6, device=DEV) * w[0, 0])
    with torch.inference_mode():
        assert torch.equal(L.lookup(table, index, out=torch.empty(3, 6, device=DEV)), table[index])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", [(70, 5, 3), (70, 40, 40), (130, 3, 200)])
def test_the_longest_strides(dtype, n, k, o):
    """rows 2^24 elements apart, the most that a call takes without a copy: a step's rows lie up to 4 GB apart"""
    ld = L.MAX_STRIDE
    room = torch.empty((n - 1) * ld + max(k, o), dtype=dtype, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(n + k)

    def far(rows, cols):
        t = torch.as_strided(room, (rows, cols), (ld, 1))
        t.copy_(torch.randint(-3, 4, (rows, cols), generator=g, device=DEV))
        return t, t.clone().contiguous()
    x, xc = far(n, k)
    w = torch.randint(-3, 4, (o, k), generator=g, device=DEV).to(dtype)
    kx = L.checkpoint(x)
    assert torch.equal(kx.values(dtype), xc)
    y, ky = L.dense_forward(x, w, relu=True)
    assert torch.equal(y, (xc.double() @ w.double().t()).clamp_min(0).to(dtype))
    index = torch.randint(0, n, (50,), generator=g, device=DEV)
    assert torch.equal(L.lookup(x, index), xc[index])
    far(n, k)                                    # (the room has been read)
    L.lookup(xc, torch.arange(n, device=DEV), out=x)
    assert torch.equal(x, xc)
    dy, dyc = far(n, o)
    dx, dw, db = L.dense_backward(dy, kx, w, relu=ky, grad_dtype=torch.float32)
    dz = torch.where(y > 0, dyc, torch.zeros_like(dyc)).double()
    assert torch.equal(dx, (dz @ w.double()).to(dtype)) and torch.equal(dw.double(), dz.t() @ xc.double()) and torch.equal(db.double(), dz.sum(0))
    want = torch.zeros(9, o, dtype=torch.float64, device=DEV).index_add_(0, torch.arange(n, device=DEV) % 9, dyc.double())
    assert torch.equal(L.lookup_backward(dy, torch.arange(n, device=DEV) % 9, 9), want.to(dtype))
    if o <= n:                                   # (the room holds a weight too)
        wf, wc = far(o, k)
        y2, _ = L.dense_forward(xc, wf)
        dx2, _, _ = L.dense_backward(dyc, kx, wf, need_dw=False, need_db=False)
        assert torch.equal(y2, (xc.double() @ wc.double().t()).to(dtype)) and torch.equal(dx2, (dyc.double() @ wc.double()).to(dtype))


@pytest.mark.parametrize("e", [-100, -110, -114, -120, -127, -135])
def test_small_float32_operands(e):
    """Of three bfloat16 parts the last is a multiple of 2^-133: an operand below 2^-110 is off by up to 2^-134, which its partners' magnitudes multiply; beside that the bound of any
    other size (half a step of the result, 2^-23 of the magnitudes summed for each addition and product).  Subnormal parts are operands like any others."""
    g = torch.Generator(device=DEV)
    g.manual_seed(-e)
    n, k, o = 70, 48, 40
    x, w = torch.randn(n, k, generator=g, device=DEV) * 2.0 ** e, torch.randn(o, k, generator=g, device=DEV)
    dy = torch.randn(n, o, generator=g, device=DEV) * 2.0 ** e
    kept = L.checkpoint(torch.randn(n, k, generator=g, device=DEV))
    y, _ = L.dense_forward(x, w, keep=False)
    dx, dw, db = L.dense_backward(dy, kept, w)
    xv = kept.values().double()
    for got, a, b in ((y, x.double(), w.double().t()), (dx, dy.double(), w.double()), (dw, dy.double().t(), xv), (db[:, None], dy.double().t(), torch.ones(n, 1, dtype=torch.float64, device=DEV))):
        want, size, lost = a @ b, a.abs() @ b.abs(), torch.ones_like(a) @ b.abs()
        bound = 2.0 ** -24 * want.abs() + 2.0 ** -149 + (n + 8) * 2.0 ** -23 * size + 2.0 ** -134 * lost
        assert ((got.double() - want).abs() <= bound * (1 + 2.0 ** -8)).all()
    assert y.any() and dx.any() and dw.any()
