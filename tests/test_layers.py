"""The trainable-layer operators without a GPU: what the calls refuse, and the C entries' own argument checks (nothing is launched)."""
import ctypes as C

import pytest
import torch

import _pkg
from ibl_nerf_amd import binding as B

L = _pkg.load().layers


@pytest.fixture(scope="module")
def lib():
    return B.load_library()


def test_no_cpu_path():
    x = torch.zeros(2, 3)
    for call in (lambda: L.checkpoint(x), lambda: L.dense_forward(x, torch.zeros(4, 3)), lambda: L.lookup(x, torch.zeros(1, dtype=torch.long)),
                 lambda: L.lookup_backward(x, torch.zeros(2, dtype=torch.long), 5)):
        with pytest.raises(B.IblNerfError, match="no CPU path"):
            call()


def test_types_are_refused_by_name():
    for t in (torch.float64, torch.int32):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            L.checkpoint(torch.zeros(2, 3, dtype=t))
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            L.lookup(torch.zeros(2, 3, dtype=t), torch.zeros(1, dtype=torch.long))


def test_checkpoint_shapes():
    ok = L.Checkpoint(torch.zeros(5, 64, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.uint8), 33)
    assert ok.rows == 5 and ok.columns == 33 and not ok.signed
    for codes, scales, k in (((5, 33), (5, 2), 33), ((5, 64), (5, 1), 33), ((5, 64), (4, 2), 33), ((5, 64), (5, 2), 65), ((5, 0), (5, 0), 0)):
        with pytest.raises(ValueError):
            L.Checkpoint(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), k)
    with pytest.raises(TypeError):
        L.Checkpoint(torch.zeros(5, 64, dtype=torch.int8), torch.zeros(5, 2, dtype=torch.uint8), 33)


P = C.c_void_p(1 << 20)      # an address that no refused call looks at


def refused(lib, rc, word):
    assert rc == -1
    assert word in lib.iblnerf_layers_last_error().decode()


def test_c_checkpoint_refuses(lib):
    good = dict(dtype=0, x=P, ld=8, n=4, k=8, s=0, codes=P, scales=P)
    for bad in (dict(dtype=3), dict(dtype=-1), dict(x=None), dict(ld=7), dict(ld=(1 << 24) + 1), dict(n=-1), dict(n=1 << 31), dict(k=0), dict(k=65537), dict(codes=None), dict(scales=None),
                dict(codes=C.c_void_p((1 << 20) + 4)), dict(x=C.c_void_p((1 << 20) + 2))):
        a = dict(good, **bad)
        refused(lib, lib.iblnerf_checkpoint(None, a["dtype"], a["x"], a["ld"], a["n"], a["k"], a["s"], a["codes"], a["scales"]), "checkpoint")
        refused(lib, lib.iblnerf_checkpoint_values(None, a["codes"], a["scales"], a["n"], a["k"], a["s"], a["dtype"], a["x"], a["ld"]), "checkpoint_values")
    assert lib.iblnerf_checkpoint(None, 0, None, 8, 0, 8, 0, None, None) == 0      # no rows: nothing to do


def test_c_dense_refuses(lib):
    good = dict(dtype=1, x=P, ldx=8, n=4, k=8, w=P, ldw=8, o=5, b=P, y=P, ldy=5, codes=P, scales=P)
    for bad in (dict(dtype=9), dict(x=None), dict(ldx=7), dict(n=-1), dict(k=0), dict(o=0), dict(o=1 << 17), dict(w=None), dict(ldw=7), dict(y=None), dict(ldy=4), dict(codes=None),
                dict(scales=None), dict(b=C.c_void_p((1 << 20) + 1)), dict(codes=C.c_void_p((1 << 20) + 1)), dict(n=2147482000, o=65536, ldy=65536)):
        a = dict(good, **bad)
        refused(lib, lib.iblnerf_dense_forward(None, a["dtype"], a["x"], a["ldx"], a["n"], a["k"], a["w"], a["ldw"], a["o"], a["b"], 1, a["y"], a["ldy"], a["codes"], a["scales"], P, 1 << 40), "dense_forward")
    need = lib.iblnerf_dense_forward_workspace(1, 100000, 512, 512)
    assert need > 0
    refused(lib, lib.iblnerf_dense_forward(None, 1, P, 512, 100000, 512, P, 512, 512, P, 1, P, 512, P, P, P, need - 1), "workspace")
    good = dict(dtype=1, dy=P, ldy=5, n=400, k=8, o=5, xc=P, xs=P, yc=P, w=P, ldw=8, dx=P, ldx=8, gt=1, dw=P, db=P, ws=P, bytes=1 << 30)
    for bad in (dict(dtype=9), dict(dy=None), dict(ldy=4), dict(n=-1), dict(k=0), dict(o=0), dict(xc=None), dict(xs=None), dict(w=None), dict(ldw=7), dict(ldx=7), dict(gt=2), dict(dw=None),
                dict(yc=C.c_void_p((1 << 20) + 1)), dict(ws=None), dict(bytes=8), dict(db=C.c_void_p((1 << 20) + 1))):
        a = dict(good, **bad)
        refused(lib, lib.iblnerf_dense_backward(None, a["dtype"], a["dy"], a["ldy"], a["n"], a["k"], a["o"], a["xc"], a["xs"], 0, a["yc"], a["w"], a["ldw"], a["dx"], a["ldx"], a["gt"], a["dw"],
                                                a["db"], a["ws"], a["bytes"]), "dense_backward")
    assert lib.iblnerf_dense_backward_workspace(1, 400, 8, 5) >= 2 * (8 * 5 + 5) * 4
    assert lib.iblnerf_dense_backward_workspace(1, 400, 0, 5) == 0


def test_c_lookup_refuses(lib):
    good = dict(dtype=0, tab=P, ld=8, v=10, d=8, idx=P, bits=64, n=4, per=2, out=P, ldo=8)
    for bad in (dict(dtype=3), dict(tab=None), dict(ld=7), dict(v=0), dict(d=0), dict(idx=None), dict(bits=16), dict(n=-1), dict(per=0), dict(n=1 << 20, per=1 << 12), dict(out=None), dict(ldo=7),
                dict(idx=C.c_void_p((1 << 20) + 4))):
        a = dict(good, **bad)
        refused(lib, lib.iblnerf_lookup(None, a["dtype"], a["tab"], a["ld"], a["v"], a["d"], a["idx"], a["bits"], a["n"], a["per"], 1.0, a["out"], a["ldo"]), "lookup")
        if not set(bad) & {"ld"}:
            refused(lib, lib.iblnerf_lookup_backward(None, a["dtype"], a["out"], a["ldo"], a["idx"], a["bits"], a["n"], a["per"], a["v"], a["d"], 1.0, a["tab"], P, 1 << 40), "lookup_backward")
    need = lib.iblnerf_lookup_backward_workspace(20000, 2, 10, 8)          # (few positions need none)
    assert need > 0 and lib.iblnerf_lookup_backward_workspace(20000, 0, 10, 8) == 0 and lib.iblnerf_lookup_backward_workspace(4, 2, 10, 8) == 0
    refused(lib, lib.iblnerf_lookup_backward(None, 0, P, 8, P, 64, 20000, 2, 10, 8, 1.0, P, P, need - 1), "workspace")
