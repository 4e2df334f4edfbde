"""Every row, column and product of the dense layers counts exactly once: small whole numbers, which a checkpoint holds exactly and whose sums stay below 2^24, so that outputs and gradients
are the float64 sums rounded once — bit for bit, in every form the sizes choose, at their seams."""
import pytest
import torch

import _pkg

pytestmark = pytest.mark.gpu
L = _pkg.load().layers
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


def whole(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV).double()


def inputs(n, k, o):
    """x -3..3, weights -3..3, dY -2..2, output signs; nothing in the first and the last row is zero"""
    g = torch.Generator(device=DEV)
    g.manual_seed(n + 3 * k + 5 * o)
    x, w, b, dy, y = whole(g, -3, 3, n, k), whole(g, -3, 3, o, k), whole(g, -3, 3, o), whole(g, -2, 2, n, o), whole(g, -1, 2, n, o).clamp_min(0)
    for r in (0, -1):
        x[r], dy[r], y[r] = 3, 2, 1
    return x, w, b, dy, y


# (columns in, columns out): weight tiles of 32 x 32, 32 x 128, 128 x 32, 128 x 128 (one and several)
SIDES = [(20, 10), (100, 20), (20, 100), (100, 100), (130, 260)]
# around the 32, 64 and 128 rows of a step, two steps and a piece
SEAMS = [1, 7, 31, 32, 33, 63, 64, 65, 71, 95, 97, 127, 128, 129, 135, 191, 193, 255, 257, 391, 1023, 1025, 2047, 2049, 2111]
# pieces and their sums: 1, 4, 16 and 64 groups of threads (with the sides above)
MANY = [4097, 5000, 8191, 12801, 20000, 32767, 40001, 65537]
# 256 x 256 tiles: one, and two of half the pieces
WIDE = [(65535, 256, 200), (65536, 250, 256), (65537, 256, 256), (66001, 199, 251), (33000, 512, 256), (33001, 450, 500), (65600, 512, 500), (70001, 240, 240)]


def gradients(n, k, o, dtype):
    x, w, _, dy, y = inputs(n, k, o)
    ky = L.checkpoint(y.to(dtype), signed=False)
    for relu in (None, ky):
        dz = dy if relu is None else torch.where(y > 0, dy, torch.zeros_like(dy))
        for signed in (True, False):
            xv = x if signed else x.clamp_min(0)
            kx = L.checkpoint(x.to(dtype), signed=signed)
            assert torch.equal(kx.values().double(), xv)
            dx, dw, db = L.dense_backward(dy.to(dtype), kx, w.to(dtype), relu=relu, grad_dtype=torch.float32)
            assert torch.equal(dw.double(), dz.t() @ xv) and torch.equal(db.double(), dz.sum(0))
            want = dz @ w
            assert float(want.abs().max()) < 2 ** 24 and torch.equal(dx, want.to(dtype))
            alone = L.dense_backward(dy.to(dtype), kx, w.to(dtype), relu=relu, need_dx=False)
            assert torch.equal(alone[1], dw.to(dtype)) and torch.equal(alone[2], db.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,o", SIDES)
def test_gradients_count_every_row_once(k, o, dtype):
    for n in SEAMS:
        gradients(n, k, o, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", MANY)
@pytest.mark.parametrize("k,o", SIDES)
def test_gradients_in_pieces_count_every_row_once(n, k, o, dtype):
    gradients(n, k, o, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", WIDE)
def test_gradients_in_wide_tiles_count_every_row_once(n, k, o, dtype):
    gradients(n, k, o, dtype)


# From 32 768 rows: rows in pieces of 64 (at most 64 columns) and 128 columns, one piece and several, the last one short; up to 8 passes of 256 outputs, and one output more than they hold
FORMS = [(32768, 64, 40), (32769, 65, 33), (33001, 130, 513), (33000, 72, 2048), (32900, 72, 2049), (33000, 2048, 72), (33003, 257, 255), (32895, 129, 128), (32768, 8, 300), (33000, 7, 300), (32767, 130, 257)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", FORMS)
def test_many_rows_forward_and_input_gradient(n, k, o, dtype):
    x, w, b, dy, y = inputs(n, k, o)
    z = x @ w.t() + b
    assert float(z.abs().max()) < 2 ** 24
    for relu in (True, False):
        want = (z.clamp_min(0) if relu else z).to(dtype)
        for keep in (True, False):
            got, kept = L.dense_forward(x.to(dtype), w.to(dtype), b.to(dtype), relu=relu, keep=keep)
            assert torch.equal(got, want) and (kept is None) == (not keep)
            if keep:
                again = L.checkpoint(want, signed=not relu)          # (held to the definition by test_gpu_layers.py)
                assert torch.equal(kept.codes, again.codes) and torch.equal(kept.scales, again.scales)
        assert torch.equal(L.dense_forward(x.to(dtype), w.to(dtype), None, relu=relu, keep=False)[0], ((z - b).clamp_min(0) if relu else z - b).to(dtype))
    ky, kx = L.checkpoint(y.to(dtype), signed=False), L.checkpoint(x.to(dtype))
    for relu in (None, ky):
        dz = dy if relu is None else torch.where(y > 0, dy, torch.zeros_like(dy))
        dx, none, db = L.dense_backward(dy.to(dtype), kx, w.to(dtype), relu=relu, need_dw=False, need_db=False)
        assert none is None and db is None and torch.equal(dx, (dz @ w).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,o", [(1, 4096, 4096), (100, 4096, 640), (100, 640, 4096), (3000, 1027, 2050), (9, 65536, 5), (9, 5, 65536)])
def test_wide_layers(n, k, o, dtype):
    """the widths that a network may have, and the widest there are"""
    x, w, b, dy, _ = inputs(n, k, o)
    z = x @ w.t() + b
    got, kept = L.dense_forward(x.to(dtype), w.to(dtype), b.to(dtype), relu=True)
    assert torch.equal(got, z.clamp_min(0).to(dtype))          # (what float16 cannot hold is infinite on both sides)
    again = L.checkpoint(got, signed=False)
    assert torch.equal(kept.codes, again.codes) and torch.equal(kept.scales, again.scales)
    gradients(n, k, o, dtype)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("wide", ["weight", "bias", "both", "neither"])
def test_gradients_of_wider_parameters_are_wide_sums(wide, dtype):
    """a float32 weight or bias beside 16-bit activations gets a sum that 16 bits do not hold; a 16-bit one that sum rounded once"""
    x, w, b, dy, _ = inputs(3001, 40, 33)
    x, dy = x.abs() + 1, dy.abs() + 1          # (sums of 6 000 and 20 000)
    w = w.to(torch.float32 if wide in ("weight", "both") else dtype).requires_grad_(True)
    b = b.to(torch.float32 if wide in ("bias", "both") else dtype).requires_grad_(True)
    y, _ = L.dense(x.to(dtype), w, b)
    y.backward(dy.to(dtype))
    for p, want in ((w, dy.t() @ x), (b, dy.sum(0))):
        assert p.grad.dtype == p.dtype and torch.equal(p.grad, want.to(p.dtype))
        assert not torch.equal(want, want.to(dtype).double())
