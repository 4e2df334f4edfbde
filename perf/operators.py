"""The trainable-layer operators (ibl_nerf_amd.layers) as timed cases: their plain forms in elementary torch, the calls a user makes of the kernels, and
the definitions in 64 bits.

Three operators and their directions (T = float32, bfloat16 or float16):

    checkpoint     an activation [n, k] held in 8 bits: per row and block of 32 columns one power of two 2^e and whole codes c, value c 2^e.  A signed checkpoint has
                   |c| <= 127, an unsigned one (what a ReLU leaves) 0 <= c <= 255; e is the smallest exponent >= -126 with max|x| <= 127 2^e (255 2^e), codes are rounded to
                   nearest, ties to even, and a positive entry of an unsigned checkpoint keeps at least code 1: the code says whether the ReLU was open
    dense          y = act(x W^T + b) rounded to T, and y's checkpoint
    dense backward from the checkpoints of the layer's input X and of its output Y:  dZ = dY where Y's code is positive (ReLU) or everywhere,
                   dX = dZ W,  dW = dZ^T X,  db = sum over rows of dZ
    lookup         out[p] = scale * table[index[p / rows_per_index]]; a negative index is a row without a code: zeros
    lookup gradient   d table[t] = scale * sum of dOut[p] over the rows p with index[p / rows_per_index] = t
"""
import math

import torch

own = False

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one sample of one ray through one layer of a 512-wide network: what an interactive probe of a point pays (no checkpoint: nothing is trained)
        dict(name="dense one point 512 bf16", op="dense", n=1, k=512, o=512, t="bf16", relu=True, keep=False),
        # a hidden layer of the 384-wide network on the coarse samples of 1 001 rays, in the precision of its parameters
        dict(name="dense 64064 x 384 f32", op="dense", n=64064, k=384, o=384, t="f32", relu=True, keep=True),
        # a hidden layer of a 512-wide network on a training step's fine pass: 4 096 rays of 64 + 128 samples
        dict(name="dense 786432 x 512 bf16", op="dense", n=786432, k=512, o=512, t="bf16", relu=True, keep=True),
        # the view layer (feature 512 + direction encoding 27 columns) on the live samples of a small step: rows that fill no tile, columns that fill no vector
        dict(name="dense backward 1003 x 539 bf16", op="dense_backward", n=1003, k=539, o=512, t="bf16", relu=True),
        # a hidden layer of the 384-wide network, coarse pass of 1 024 rays, in the precision of its parameters
        dict(name="dense backward 65536 x 384 f32", op="dense_backward", n=65536, k=384, o=384, t="f32", relu=True),
        # a hidden layer of a 512-wide network on a whole fine pass
        dict(name="dense backward 786432 x 512 f16", op="dense_backward", n=786432, k=512, o=512, t="f16", relu=True),
        # the encoded positions (63 columns) that the first and the skip layer read, coarse pass of 1 024 rays
        dict(name="checkpoint 65536 x 63 f32", op="checkpoint", n=65536, k=63, t="f32", signed=True),
        # the last trunk activation of a whole fine pass
        dict(name="checkpoint 786432 x 512 bf16", op="checkpoint", n=786432, k=512, t="bf16", signed=False),
        # a code of 48 numbers for the view of each ray of a training batch, 200 training views
        dict(name="lookup 4096 of 200 x 48 f32", op="lookup", n=4096, per=1, v=200, d=48, t="f32", hot=1.0),
        # ... the same for every sample of the rays, beside the direction encoding
        dict(name="lookup 4096 x 192 rows x 32 bf16", op="lookup", n=4096, per=192, v=200, d=32, t="bf16", hot=1.0),
        # the gradient of the batch's codes
        dict(name="lookup gradient 4096 of 200 x 48", op="lookup_backward", n=4096, per=1, v=200, d=48, t="f32", hot=1.0),
        # all pixels of an 800 x 800 frame over a large table (a code for each cell of a grid), a few cells taking most of the rays
        dict(name="lookup gradient 640000 of 65536 x 64", op="lookup_backward", n=640000, per=1, v=65536, d=64, t="f32", hot=3.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dense", "dense", "dense_backward", "dense_backward", "checkpoint", "lookup", "lookup_backward"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op in ("dense", "dense_backward"):
        k, o = _log(rng, 3, 640), _log(rng, 1, 640)
        n = _log(rng, 1, max(1, min(786432, 786432 * 512 * 512 // (2 * k * o))))
        c = dict(op=op, n=n, k=k, o=o, t=t, relu=rng.random() < 0.7)
        if op == "dense":
            c["keep"] = rng.random() < 0.7
        return c
    if op == "checkpoint":
        return dict(op=op, n=_log(rng, 1, 500000), k=_log(rng, 1, 640), t=t, signed=rng.random() < 0.5)
    per = rng.choice([1, 1, 64, 192, 7])
    d = _log(rng, 1, 256)
    rows = _log(rng, 1, max(1, min(786432, 786432 * 64 // d)))
    return dict(op=op, n=max(1, rows // per), per=per, v=_log(rng, 1, 100000), d=d, t=t, hot=rng.choice([1.0, 2.0, 3.0]))


# ---------------------------------------------------------------------------------------------------------------------------------------------- the inputs
def _activation(g, n, k, relu):
    """A network's activations: a scale of its own for each column, half of the entries closed by a ReLU where there is one."""
    x = torch.randn((n, k), generator=g, device=DEV) * (0.2 + 2.0 * torch.rand((1, k), generator=g, device=DEV))
    return x.clamp_min_(0.0) if relu else x


def _upstream(g, n, o):
    """dL/dy: samples in front of or behind a surface carry orders of magnitude less than those on it."""
    return torch.randn((n, o), generator=g, device=DEV) * torch.pow(10.0, -3.0 * torch.rand((n, 1), generator=g, device=DEV))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    c, op = dict(case), case["op"]
    t = T[c["t"]]
    s = {"case": c}
    if op == "checkpoint":
        s["x"] = _activation(g, c["n"], c["k"], not c["signed"]).to(t)
    elif op in ("dense", "dense_backward"):
        n, k, o = c["n"], c["k"], c["o"]
        s["w"] = ((2 * torch.rand((o, k), generator=g, device=DEV) - 1) / math.sqrt(k)).to(t)
        s["b"] = ((2 * torch.rand((o,), generator=g, device=DEV) - 1) / math.sqrt(k)).to(t)
        if op == "dense":
            s["x"] = _activation(g, n, k, True).to(t)
        else:      # what the forward pass left: the 8-bit checkpoints of the layer's input and (under a ReLU) of its output
            s["x_codes"], s["x_scales"] = _pack(_activation(g, n, k, True).to(t), False)
            if c["relu"]:
                s["y_codes"], s["y_scales"] = _pack(_activation(g, n, o, True).to(t), False)
            s["dy"] = _upstream(g, n, o).to(t)
    else:
        u = torch.rand((c["n"],), generator=g, device=DEV, dtype=torch.float64)
        s["index"] = (u ** c["hot"] * c["v"]).long().clamp_(0, c["v"] - 1)
        s["scale"] = 1.0 / math.sqrt(c["d"])
        if op == "lookup":
            s["table"] = torch.randn((c["v"], c["d"]), generator=g, device=DEV).to(t)
        else:
            s["dout"] = _upstream(g, c["n"] * c["per"], c["d"]).to(t)
    return s


# ---------------------------------------------------------------------------------------------------------------------------------------- the plain forms
def _pack(x, signed):
    """Codes (uint8, two's complement where signed) and scale bytes (e + 127; 255 marks a block with a non-finite entry, whose codes are 1) of an activation; padding columns are zero."""
    n, k = x.shape
    kb = (k + 31) // 32
    v = torch.zeros((n, 32 * kb), dtype=torch.float32, device=x.device)
    v[:, :k] = x
    v = v.view(n, kb, 32)
    a = v.abs().amax(-1) if signed else v.amax(-1).clamp_min(0.0)
    bad = ~torch.isfinite(v).all(-1)
    top, shift = (127.0 / 128.0, 7) if signed else (255.0 / 256.0, 8)
    m, e = torch.frexp(torch.where(bad, torch.zeros_like(a), a))
    e = torch.where(a > 0, (e - shift + (m > top).int()).clamp_min(-126), torch.full_like(e, -126))
    c = torch.round(torch.ldexp(v, -e[..., None]))
    c = c.clamp(-127, 127) if signed else torch.where(v > 0, c.clamp(1, 255), torch.zeros_like(c))
    c = torch.where(bad[..., None], torch.ones_like(c), c)
    codes = c.to(torch.int8).view(torch.uint8) if signed else c.to(torch.uint8)
    return codes.view(n, 32 * kb), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _restore(codes, scales, k, signed):
    """The values a checkpoint stands for, float32 (at most 8 significant bits each: exact in bfloat16 too)."""
    n, kb = scales.shape
    c = (codes.view(torch.int8) if signed else codes).float().view(n, kb, 32)
    e = scales.int()
    v = torch.ldexp(c, (e - 127)[..., None])
    v = torch.where((e == 255)[..., None], torch.full_like(v, float("nan")), v)
    return v.view(n, 32 * kb)[:, :k]


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    t = T[c["t"]]
    if op == "checkpoint":
        return {"kept": _restore(*_pack(s["x"], c["signed"]), c["k"], c["signed"]).to(torch.bfloat16)}
    if op == "dense":
        y = s["x"].float() @ s["w"].float().t() + s["b"].float()
        y = (torch.where(y < 0, torch.zeros_like(y), y) if c["relu"] else y).to(t)
        if not c["keep"]:
            return {"y": y}
        return {"y": y, "kept": _restore(*_pack(y, not c["relu"]), c["o"], not c["relu"]).to(torch.bfloat16)}
    if op == "dense_backward":
        dz = s["dy"].float()
        if c["relu"]:
            dz = torch.where(s["y_codes"][:, :c["o"]] > 0, dz, torch.zeros_like(dz))
        x = _restore(s["x_codes"], s["x_scales"], c["k"], False)
        return {"dx": (dz @ s["w"].float()).to(t), "dw": (dz.t() @ x).to(t), "db": dz.sum(0).to(t)}
    rows = s["index"].repeat_interleave(c["per"]) if c["per"] > 1 else s["index"]
    if op == "lookup":
        out = s["table"].float()[rows.clamp_min(0)] * s["scale"]
        return {"out": torch.where((rows >= 0)[:, None], out, torch.zeros_like(out)).to(t)}
    grad = torch.zeros((c["v"] + 1, c["d"]), dtype=torch.float32, device=DEV)
    grad.index_add_(0, torch.where(rows >= 0, rows, torch.full_like(rows, c["v"])), s["dout"].float())
    return {"dtable": (grad[:c["v"]] * s["scale"]).to(t)}


# ------------------------------------------------------------------------------------------------------------------------------------------ the two sides
def _kernels(s):
    import _pkg
    L = _pkg.load().layers
    c, op = s["case"], s["case"]["op"]
    if op == "checkpoint":
        return {"kept": L.checkpoint(s["x"], signed=c["signed"]).values(torch.bfloat16)}
    if op == "dense":
        y, kept = L.dense_forward(s["x"], s["w"], s["b"], relu=c["relu"], keep=c["keep"])
        return {"y": y, "kept": kept.values(torch.bfloat16)} if c["keep"] else {"y": y}
    if op == "dense_backward":
        x = L.Checkpoint(s["x_codes"], s["x_scales"], c["k"], signed=False)
        y = L.Checkpoint(s["y_codes"], s["y_scales"], c["o"], signed=False) if c["relu"] else None
        dx, dw, db = L.dense_backward(s["dy"], x, s["w"], relu=y)
        return {"dx": dx, "dw": dw, "db": db}
    if op == "lookup":
        return {"out": L.lookup(s["table"], s["index"], scale=s["scale"], rows_per_index=c["per"])}
    return {"dtable": L.lookup_backward(s["dout"], s["index"], c["v"], scale=s["scale"], rows_per_index=c["per"])}


def run(state):
    return _kernels(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, z = case, SIZE[case["t"]]
    kept = lambda n, k: n * 32 * ((k + 31) // 32) * 33 // 32      # noqa: E731  (codes and scale bytes)
    if c["op"] == "checkpoint":
        return {"bytes": c["n"] * c["k"] * (z + 2), "flops": c["n"] * c["k"]}
    if c["op"] == "dense":
        n, k, o = c["n"], c["k"], c["o"]
        return {"bytes": z * (n * k + o * k + o + n * o) + (2 * n * o if c["keep"] else 0), "flops": 2.0 * n * k * o}
    if c["op"] == "dense_backward":
        n, k, o = c["n"], c["k"], c["o"]
        return {"bytes": z * (n * o + o * k + n * k + o * k + o) + kept(n, k) + (kept(n, o) if c["relu"] else 0), "flops": 4.0 * n * k * o}
    rows = c["n"] * c["per"]
    if c["op"] == "lookup":
        return {"bytes": z * c["d"] * (rows + min(c["v"], c["n"])) + 8 * c["n"], "flops": rows * c["d"]}
    return {"bytes": z * c["d"] * (rows + c["v"]) + 8 * c["n"], "flops": rows * c["d"]}


# ------------------------------------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _values64(x, signed):
    """What the checkpoint of x stands for, from the definition: the block's exponent from a logarithm put right by two comparisons."""
    n, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).reshape(n, -1, 32)
    most = 127.0 if signed else 255.0
    a = v.abs().amax(-1, keepdim=True) if signed else v.amax(-1, keepdim=True).clamp_min(0)
    e = torch.ceil(torch.log2(a / most)).clamp_min(-126)
    e = torch.where(most * torch.exp2(e) < a, e + 1, e)
    e = torch.where((most * torch.exp2(e - 1) >= a) & (e > -126), e - 1, e)
    step = torch.exp2(e)
    c = torch.round(v / step)
    if not signed:
        c = torch.where(v > 0, torch.maximum(c, torch.ones_like(c)), torch.zeros_like(c))
    return (c * step).reshape(n, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], s["case"]["op"]
    if op == "checkpoint":
        return {"kept": _values64(s["x"], c["signed"])}
    if op == "dense":
        y = torch.addmm(s["b"].double(), s["x"].double(), s["w"].double().t())
        if c["relu"]:
            y = torch.relu(y)
        return {"y": y, "kept": None} if c["keep"] else {"y": y}      # (the checkpoint is one of the ROUNDED y: it has no value in 64 bits)
    if op == "dense_backward":
        dz = s["dy"].double()
        if c["relu"]:
            dz = dz * (s["y_codes"][:, :c["o"]] != 0)
        step = torch.exp2(s["x_scales"].double() - 127).repeat_interleave(32, dim=1)
        x = (s["x_codes"].double() * step)[:, :c["k"]]
        return {"dx": torch.mm(dz, s["w"].double()), "dw": torch.mm(dz.t(), x), "db": dz.sum(dim=0)}
    which = s["index"][torch.arange(c["n"] * c["per"], device=DEV) // c["per"]]
    if op == "lookup":
        return {"out": torch.where(which[:, None] < 0, 0.0, s["table"].double()[which.clamp_min(0)] * s["scale"])}
    order = torch.argsort(which)
    grad = torch.zeros((c["v"], c["d"]), dtype=torch.float64, device=DEV)
    order = order[which[order] >= 0]
    grad.index_put_((which[order],), s["dout"].double()[order], accumulate=True)
    return {"dtable": grad * s["scale"]}
