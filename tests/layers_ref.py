"""The layer operators from their definitions, in float64 on the CPU: what tests/test_gpu_layers.py holds the kernels to."""
import numpy as np
import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step of a rounding, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # the smallest step


def pack(x, signed):
    """codes (as integers) [n, 32 kb], exponents [n, kb] (scale byte - 127; 128: a block with a non-finite entry) of x, from the definition, one block at a time."""
    x = x.detach().double().cpu().numpy()
    n, k = x.shape
    kb = (k + 31) // 32
    v = np.zeros((n, 32 * kb))
    v[:, :k] = x
    v = v.reshape(n, kb, 32)
    codes, exps = np.zeros(v.shape, np.int64), np.zeros((n, kb), np.int64)
    most = 127 if signed else 255
    for i in range(n):
        for j in range(kb):
            b = v[i, j]
            if not np.isfinite(b).all():
                codes[i, j], exps[i, j] = 1, 128
                continue
            a = np.abs(b).max() if signed else max(b.max(), 0.0)
            e = -126
            if a > 0:
                e = max(-126, int(np.floor(np.log2(a))) - 9)
                while most * 2.0 ** e < a:
                    e += 1
            c = np.round(b / 2.0 ** e)      # (ties to even)
            if not signed:
                c = np.where(b > 0, np.maximum(c, 1), 0)
            codes[i, j], exps[i, j] = c, e
    return codes.reshape(n, 32 * kb), exps


def values(codes, exps, k):
    v = codes.reshape(exps.shape + (32,)) * np.exp2(exps.astype(np.float64))[..., None]
    v[exps == 128] = np.nan
    return torch.from_numpy(v.reshape(codes.shape)[:, :k])


def raw(kept):
    """A Checkpoint's codes as integers and its exponents."""
    c = kept.codes.cpu()
    c = c.view(torch.int8) if kept.signed else c
    return c.numpy().astype(np.int64), kept.scales.cpu().numpy().astype(np.int64) - 127


def stored(kept):
    """A Checkpoint's values in float64 from its bytes."""
    c, e = raw(kept)
    return values(c, e, kept.columns)


def close(got, want, size, terms, dtype):
    """got (rounded to dtype) against want in float64: half a step of the rounding, and for a sum of `terms` products of total magnitude `size` a float32 step (2^-23: matrix
    instructions may truncate) for each addition and each product."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin)
    off = (got - want).abs()
    bound = (EPS[dtype] * want.abs() + TINY[dtype] + (terms + 8) * 2.0 ** -23 * size.double().cpu()) * (1 + 2.0 ** -8)
    bad = fin & (off > bound)
    assert not bad.any(), "%d of %d beyond the bound: worst %.3g where %.3g is allowed" % (int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound[bad].min()))
