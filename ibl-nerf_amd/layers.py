"""Trainable layers on hand-written kernels: dense layers whose backward pass reads 8-bit checkpoints of their activations, and rows of a table by index (a code for the view
of each ray) with the table's gradient by sorted tokens.  include/iblnerf_layers.h is the C boundary; csrc/dense_kernel.hip and csrc/lookup_kernel.hip say what bounds
them.

They train what the fused backward (training.py) is not built for: networks outside the 8 x 256 shape, layer by layer (`network_query` below,
model.fused_network_query, training.render_rays_train).

    y, kept = dense(x, weight, bias, relu=True)        autograd; keeps 1.03 bytes an activation instead of x and y
    y, kept = dense(y, weight2, bias2, kept=kept)      the next layer reads the checkpoint that the first has written
    rows = lookup(codes, view, scale)                  autograd

Tensors are float32, bfloat16 or float16 on one GPU; rows may be strided, what lies along a row is contiguous (anything else is copied).  Calls run on the current stream of the
tensors' device and never synchronise."""
from __future__ import annotations

import contextlib

import torch

from . import binding as B
from . import checkpoint as ck

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_COLUMNS, MAX_STRIDE = 65536, 1 << 24
# the current stream's handle without a Stream object around it (these calls cost microseconds, and so do a small layer's kernels)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _type(t, what):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (what, t.dtype))
    return code


def _on(t):
    """(library, stream, what makes the tensor's device current for the call, or None where it is)."""
    if not t.is_cuda:
        raise B.IblNerfError("the layer operators have no CPU path: got a tensor on %s" % t.device)
    dev = t.get_device()
    return B.load_library(), _raw_stream(dev), None if dev == _current_device() else torch.cuda.device(dev)


def _call(guard, f, *args):
    if guard is None:
        rc = f(*args)
    else:
        with guard:
            rc = f(*args)
    if rc:
        B.check_layers(rc)


def _same(t, like, what, dtype=None):
    if t.device != like.device:
        raise ValueError("%s is on %s, the call's other tensors on %s" % (what, t.device, like.device))
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (what, dtype, t.dtype))


def _rows(t, what):
    """t [..., k] as [n, k] with unit stride along a row, and its row stride in elements."""
    shape = t.shape
    if len(shape) == 2 and 1 <= shape[1] <= MAX_COLUMNS and t.is_contiguous():
        return t, shape[1]
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_COLUMNS:
        raise ValueError("%s must be [..., k] with 1 <= k <= %d, got %s" % (what, MAX_COLUMNS, tuple(shape)))
    k = shape[-1]
    if len(shape) != 2:
        t = t.reshape(-1, k) if t.numel() else t.new_empty((0, k))
    if (k > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and not k <= t.stride(0) <= MAX_STRIDE):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else k)


def _workspace(size, like):
    """Scratch memory of one call from torch's allocator: reused in stream order, a captured graph's from the graph's own pool."""
    return (like.new_empty((size,), dtype=torch.uint8), size) if size else (None, 0)


def _address(t):
    return None if t is None else t.data_ptr()


class Checkpoint:
    """An activation [n, columns] in 8 bits: `codes` [n, 32 ceil(columns / 32)] uint8 and `scales` [n, ceil(columns / 32)] uint8 (include/iblnerf_layers.h has the format).
    `signed`: two's-complement codes; unsigned ones come from a ReLU."""

    __slots__ = ("codes", "scales", "columns", "signed")

    def __init__(self, codes, scales, columns, signed=False):
        blocks = (int(columns) + 31) // 32
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("a checkpoint's codes and scales are uint8, got %s and %s" % (codes.dtype, scales.dtype))
        if columns < 1 or codes.dim() != 2 or tuple(codes.shape) != (scales.shape[0], 32 * blocks) or tuple(scales.shape) != (codes.shape[0], blocks):
            raise ValueError("a checkpoint of %d columns has codes [n, %d] and scales [n, %d], got %s and %s" % (columns, 32 * blocks, blocks, tuple(codes.shape), tuple(scales.shape)))
        _same(scales, codes, "scales")
        self.codes, self.scales, self.columns, self.signed = codes.contiguous(), scales.contiguous(), int(columns), bool(signed)

    @property
    def rows(self):
        return self.codes.shape[0]

    def values(self, dtype=torch.float32):
        """The values the checkpoint stands for, [n, columns]: exact in float32 and bfloat16 (at most 8 significant bits; 2^128, which an entry beyond 3.37e38 may round up
        to, as 3.39e38, and 65536 in float16 as 65504)."""
        out = self.codes.new_empty((self.codes.shape[0], self.columns), dtype=dtype)
        t = _type(out, "the values")
        lib, stream, guard = _on(out)
        _call(guard, lib.iblnerf_checkpoint_values, stream, self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.columns, int(self.signed), t, out.data_ptr(), self.columns)
        return out


def _made(codes, scales, columns, signed):
    """A Checkpoint of buffers that a kernel has just written."""
    c = Checkpoint.__new__(Checkpoint)
    c.codes, c.scales, c.columns, c.signed = codes, scales, columns, bool(signed)
    return c


def _codes_like(x, n, columns):
    blocks = (columns + 31) // 32
    return x.new_empty((n, 32 * blocks), dtype=torch.uint8), x.new_empty((n, blocks), dtype=torch.uint8)


def checkpoint(x, signed=True):
    """The 8-bit checkpoint of x [..., k] (rows flattened).  signed=False: negative entries become zero."""
    t = _type(x, "x")
    lib, stream, guard = _on(x)
    x, ld = _rows(x, "x")
    n, k = x.shape
    codes, scales = _codes_like(x, n, k)
    _call(guard, lib.iblnerf_checkpoint, stream, t, x.data_ptr(), ld, n, k, int(bool(signed)), codes.data_ptr(), scales.data_ptr())
    return _made(codes, scales, k, signed)


def _weight(weight, k, like, dtype):
    if weight.dim() != 2 or weight.shape[1] != k:
        raise ValueError("a layer of %d inputs takes a weight [o, %d], got %s" % (k, k, tuple(weight.shape)))
    _same(weight, like, "weight", dtype)
    return _rows(weight, "weight")


def dense_forward(x, weight, bias=None, relu=False, keep=True):
    """y = x weight^T + bias (negative values to zero if relu), x [..., k], weight [o, k], bias [o] or None, all of one type -> (y [..., o], y's checkpoint or None).
    keep=False: no checkpoint (nothing will be trained)."""
    t = _type(x, "x")
    lib, stream, guard = _on(x)
    lead = x.shape[:-1]
    x, ld = _rows(x, "x")
    n, k = x.shape
    w, ldw = _weight(weight, k, x, x.dtype)
    o = w.shape[0]
    if not 1 <= o <= MAX_COLUMNS:
        raise ValueError("a layer has 1 to %d outputs, got %d" % (MAX_COLUMNS, o))
    if bias is not None:
        if tuple(bias.shape) != (o,):
            raise ValueError("the bias of a layer of %d outputs is [%d], got %s" % (o, o, tuple(bias.shape)))
        _same(bias, x, "bias", x.dtype)
        bias = bias.contiguous()
    y = x.new_empty((n, o))
    codes, scales = _codes_like(x, n, o) if keep else (None, None)
    ws, ws_bytes = _workspace(lib.iblnerf_dense_forward_workspace(t, n, k, o), x)
    _call(guard, lib.iblnerf_dense_forward, stream, t, x.data_ptr(), ld, n, k, w.data_ptr(), ldw, o, _address(bias), int(bool(relu)), y.data_ptr(), o, _address(codes), _address(scales),
          _address(ws), ws_bytes)
    return (y if len(lead) == 1 else y.reshape(lead + (o,))), (_made(codes, scales, o, not relu) if keep else None)


def dense_backward(dy, x, weight, relu=None, need_dx=True, need_dw=True, need_db=True, grad_dtype=None):
    """The gradients of dense_forward from checkpoints: dy [..., o], x the Checkpoint of the layer's input, relu the Checkpoint of its output (None: the layer has no ReLU)
    -> (dX [..., k], dW [o, k], db [o]), None where not asked for.  grad_dtype: dW's and db's type (dy's own by default, or float32)."""
    t = _type(dy, "dy")
    lib, stream, guard = _on(dy)
    lead = dy.shape[:-1]
    dy, ld = _rows(dy, "dy")
    n, o = dy.shape
    if not isinstance(x, Checkpoint) or x.rows != n:
        raise ValueError("x must be the Checkpoint of the layer's %d input rows" % n)
    k = x.columns
    w, ldw = _weight(weight, k, dy, dy.dtype)
    if w.shape[0] != o:
        raise ValueError("dy has %d columns, the weight %d rows" % (o, w.shape[0]))
    _same(x.codes, dy, "the input's checkpoint")
    if relu is not None:
        if not isinstance(relu, Checkpoint) or relu.rows != n or relu.columns != o or relu.signed:
            raise ValueError("relu must be the unsigned Checkpoint of the layer's output [%d, %d]" % (n, o))
        _same(relu.codes, dy, "the output's checkpoint")
    grad_dtype = grad_dtype or dy.dtype
    if grad_dtype not in (dy.dtype, torch.float32):
        raise TypeError("the parameters' gradients are %s or float32, not %s" % (dy.dtype, grad_dtype))
    dx = dy.new_empty((n, k)) if need_dx else None
    dw = dy.new_empty((o, k), dtype=grad_dtype) if need_dw or need_db else None
    db = dy.new_empty((o,), dtype=grad_dtype) if need_db else None
    ws, ws_bytes = _workspace(lib.iblnerf_dense_backward_workspace(t, n, k, o), dy)
    _call(guard, lib.iblnerf_dense_backward, stream, t, dy.data_ptr(), ld, n, k, o, x.codes.data_ptr(), x.scales.data_ptr(), int(x.signed),
          None if relu is None else relu.codes.data_ptr(), w.data_ptr(), ldw, _address(dx), k, _TYPES[grad_dtype], _address(dw), _address(db),
          _address(ws), ws_bytes)
    return (dx if dx is None or len(lead) == 1 else dx.reshape(lead + (k,))), (dw if need_dw else None), db


def _phase(like, capturing):
    """(is a graph being captured, does an eager result made now stand in a capture's way: is the current stream the default one)"""
    if capturing is None and like.is_cuda:
        with _on(like)[2] or contextlib.nullcontext():
            return torch.cuda.is_current_stream_capturing(), _raw_stream(like.get_device()) == 0
    return capturing, True


def _leaves(*tensors, capturing=None):
    """A leaf's gradient is accumulated on the stream of the first live graph that reads the leaf.  Under stream capture an EAGER graph of the default stream that still lives would
    pull that stream into the captured backward pass, where nothing can be reported and the process ends; so such graphs sign the accumulation node (it lives as long as
    they do, or as what else holds it: called behind the operator that holds it), and a capture that meets the sign is refused."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves:
        return
    capturing, default = _phase(leaves[0], capturing)
    if not (capturing or default):
        return
    for t in leaves:
        sign = t.view_as(t).grad_fn.next_functions[0][0].metadata
        if not capturing:
            sign["eager"] = True
        elif "eager" in sign:
            raise RuntimeError("a graph is being captured while an eager result of the same leaf (%s) is alive, or something else that holds the leaf's gradient accumulator of the default "
                               "stream (a hook on it, a distributed wrapper): delete that result (or its loss) first; make such a wrapper, and warm up, on a side stream" % (tuple(t.shape),))


def sign(result, capturing=None):
    """The same sign on the leaves that `result`, what an autograd Function has just given, was computed from (the framework's fused passes: their eager results stand in a captured
    backward pass's way as a layer's do)."""
    if result.grad_fn is None:
        return
    capturing, default = _phase(result, capturing)
    if default and not capturing:
        for node, _ in result.grad_fn.next_functions:
            if hasattr(node, "variable"):
                node.metadata["eager"] = True


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, relu, x_codes, x_scales, x_signed):
        w = weight.to(x.dtype)
        y, kept = dense_forward(x, w, None if bias is None else bias.to(x.dtype), relu)
        if x_codes is None:
            own = checkpoint(x)
            x_codes, x_scales, x_signed = own.codes, own.scales, True
        ctx.relu, ctx.x_signed, ctx.has_bias, ctx.type = relu, x_signed, bias is not None, x.dtype
        ctx.wide = any(t is not None and t.dtype not in (torch.bfloat16, torch.float16) for t in (weight, bias))      # (a gradient is cast to its parameter's type by autograd)
        ctx.save_for_backward(weight, x_codes, x_scales, *((kept.codes, kept.scales) if relu else ()))
        ctx.mark_non_differentiable(kept.codes, kept.scales)
        ctx.set_materialize_grads(False)                       # (or zeros of the codes' size would be written for them)
        return y, kept.codes, kept.scales

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _codes, _scales):
        if dy is None:
            return (None,) * 7
        weight, xc, xs, *out = ctx.saved_tensors
        k, o = weight.shape[1], weight.shape[0]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = dense_backward(dy.to(ctx.type), Checkpoint(xc, xs, k, ctx.x_signed), weight.to(ctx.type), Checkpoint(*out, o) if ctx.relu else None, need_x, need_w, need_b and ctx.has_bias,
                                    torch.float32 if ctx.wide else None)
        return dx, dw, db, None, None, None, None


def dense(x, weight, bias=None, relu=False, kept=None):
    """dense_forward with autograd -> (y, Checkpoint of y).  kept: the Checkpoint of x that an earlier layer has written (None: one is made here, signed) — the backward pass
    reads the checkpoints of x and, under a ReLU, of y, so neither tensor is held for it.  Parameters may be float32 beside 16-bit activations (either of them): they are cast for
    the products, and their gradients are float32 sums.  First derivatives only.
    A backward pass may be captured into a graph while no eager result of the same leaves is alive (RuntimeError otherwise; results of torch's own operations on them are not seen
    here, and end the process there)."""
    if kept is not None and (kept.columns != x.shape[-1] or kept.rows * kept.columns != x.numel()):
        raise ValueError("kept is a checkpoint of [%d, %d], x is %s" % (kept.rows, kept.columns, tuple(x.shape)))
    y, codes, scales = _Dense.apply(x, weight, bias, bool(relu), *((None, None, True) if kept is None else (kept.codes, kept.scales, kept.signed)))
    if y.requires_grad:
        _leaves(x, weight, bias)
    return y, Checkpoint(codes, scales, weight.shape[0], not relu)


def _index(index, like):
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError("index must be int32 or int64, got %s" % index.dtype)
    _same(index, like, "index")
    return index.contiguous(), 64 if index.dtype == torch.int64 else 32


def _lookup(table, index, scale, rows_per_index, out):
    t = _type(table, "table")
    lib, stream, guard = _on(table)
    if table.dim() != 2 or table.shape[0] < 1:
        raise ValueError("table must be [v, d] with at least one row, got %s" % (tuple(table.shape),))
    tab, ld = _rows(table, "table")
    v, d = tab.shape
    idx, bits = _index(index, table)
    n, per = idx.numel(), int(rows_per_index)
    if per < 1:
        raise ValueError("rows_per_index must be at least 1, got %d" % per)
    shape = tuple(index.shape[:-1]) + (index.shape[-1] * per, d) if index.dim() else (per, d)
    if out is None:
        out = table.new_empty(shape)
    else:
        _same(out, table, "out", table.dtype)
        if out.dim() != 2 or tuple(out.shape) != (n * per, d) or (d > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and not d <= out.stride(0) <= MAX_STRIDE):
            raise ValueError("out must be [%d, %d] with unit stride along a row, got %s strides %s" % (n * per, d, tuple(out.shape), tuple(out.stride())))
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out is written without autograd: it may not require a gradient")
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)          # (what an earlier operation has kept of it for its backward pass is no longer what it read)
    ld_out = out.stride(0) if out.dim() == 2 and out.shape[0] > 1 else d
    _call(guard, lib.iblnerf_lookup, stream, t, tab.data_ptr(), ld, v, d, idx.data_ptr(), bits, n, per, float(scale), out.data_ptr(), ld_out)
    return out


def lookup_backward(dout, index, v, scale=1.0, rows_per_index=1):
    """d table [v, d] = scale * the sums of dout [..., d] over each token's rows (rows in index's order, rows_per_index of them each).  Rows with an index outside [0, v)
    count nowhere.  The same inputs give the same bits."""
    t = _type(dout, "dout")
    lib, stream, guard = _on(dout)
    dout, ld = _rows(dout, "dout")
    idx, bits = _index(index, dout)
    n, per, d = idx.numel(), int(rows_per_index), dout.shape[1]
    if per < 1 or int(v) < 1 or n * per != dout.shape[0]:
        raise ValueError("%d indices with %d rows each over a table of %d rows do not fit %d gradient rows" % (n, per, int(v), dout.shape[0]))
    grad = dout.new_empty((int(v), d))
    ws, ws_bytes = _workspace(lib.iblnerf_lookup_backward_workspace(n, per, int(v), d), dout)
    _call(guard, lib.iblnerf_lookup_backward, stream, t, dout.data_ptr(), ld, idx.data_ptr(), bits, n, per, int(v), d, float(scale), grad.data_ptr(), _address(ws), ws_bytes)
    return grad


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, per):
        ctx.save_for_backward(index)
        ctx.v, ctx.scale, ctx.per = table.shape[0], scale, per
        return _lookup(table, index, scale, per, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (index,) = ctx.saved_tensors
        return lookup_backward(dout, index, ctx.v, ctx.scale, ctx.per), None, None, None


def lookup(table, index, scale=1.0, rows_per_index=1, out=None):
    """scale * table[index]: table [v, d], index [...] int32 or int64 -> [..., d]; rows_per_index > 1 repeats each row (a ray's code for each of its samples): the last axis of
    index grows by that factor.  A negative index is a row without a code (zeros, no gradient); one beyond the table reads NaN.  Differentiable in the table; `out`
    ([n, d], rows may be strided: a slice of a wider input) is written instead of a new tensor, without autograd (an in-place write like torch's own: a backward pass that kept the
    tensor before says so)."""
    if out is None and torch.is_grad_enabled() and table.requires_grad:
        rows = _Lookup.apply(table, index, float(scale), int(rows_per_index))
        _leaves(table)
        return rows
    return _lookup(table, index, scale, rows_per_index, out)


# ------------------------------------------------------------------------------------------------------------- a network layer by layer
def encode(x, freqs):
    """[x, sin(2^0 x), cos(2^0 x), ..., sin(2^(freqs-1) x), cos(2^(freqs-1) x)] of x [n, 3] (positional_embedder.py:21-34): the products with powers of two are exact, the angles of
    the high frequencies large — sine and cosine in 64 bits, rounded once (as csrc/generic_mlp.hip)."""
    if freqs == 0:
        return x
    a = (x[:, None, :] * torch.exp2(torch.arange(freqs, device=x.device, dtype=x.dtype))[None, :, None]).double()
    e = torch.stack([torch.sin(a), torch.cos(a)], 2).to(x.dtype)              # [n, freqs, 2, 3]
    return torch.cat([x, e.reshape(x.shape[0], 6 * freqs)], -1)


def _linear(params, name):
    return params[name + ".weight"], params[name + ".bias"]


def _network(params, n_code, whole):
    """(depth, width, frequencies of the points, of the directions) behind a network's parameters, n_code columns of views_linears.0 being a view's code; whole=False: the trunk and the
    density alone.  What no other path of the framework takes is refused here too: the module's own forward fails for 5 layers (the skip's concatenation is consumed by none),
    and layers beyond the reference's would not be run."""
    shapes = {k[:-len(".weight")]: tuple(w.shape) for k, w in params.items() if k.endswith(".weight")}
    width, ch = shapes["positions_linears.0"]
    depth = 1 + max(int(k.split(".")[1]) for k in shapes if k.startswith("positions_linears."))
    chv = 3
    if whole:
        columns = shapes["views_linears.0"][1]
        chv = columns - width - n_code
        if chv < 3 or (chv - 3) % 6:
            raise ValueError("views_linears.0 takes %d columns: %d features, %d code columns and no positional encoding's width beside them" % (columns, width, n_code))
    if ch < 3 or (ch - 3) % 6:
        raise ValueError("positions_linears.0 takes %d columns, no positional encoding's width" % ch)
    arch = (depth, width, (ch - 3) // 6, (chv - 3) // 6)
    if not (ck.is_member_of_built(arch) or ck.is_generic_arch(arch)):
        raise NotImplementedError("IBLNeRF%s is outside what is built (netdepth <= 32 and != 5, netwidth <= 256 or even and <= 4096, multires, multires_views <= 24)" % (arch,))
    want = {n: (o, i + (n_code if n == "views_linears.0" else 0)) for n, o, i in ck.arch_schema(*arch) if whole or n.startswith(("positions_linears.", "sigma_linear"))}
    lists = ("positions_linears.",) + (("views_linears.", "additional_radiance_feature_linear.", "additional_radiance_linear.") if whole else ())
    odd = sorted({n for n, s in want.items() if shapes.get(n) != s} | {n for n in shapes if n.startswith(lists) and n not in want})
    if odd:
        raise NotImplementedError("not the layers of IBLNeRF%s (skips = [4], coarse_radiance_number = 3): %s" % (arch, ", ".join("%s %s" % (n, shapes.get(n, "is missing")) for n in odd[:4])))
    return arch


def network_query(inputs, viewdirs, network_fn, codes=None, views=None, code_scale=1.0, dtype=None):
    """IBLNeRF.forward (ibl_nerf.py:154-208) of any network that the framework renders (netdepth <= 32 and != 5, netwidth <= 4096), with autograd, on `dense`: inputs [..., 3] points,
    viewdirs [n, 3] one direction for each row of points (or None: the density alone, :175-176), `network_fn` a torch module with the reference's parameter names -> raw
    [..., 18] float32 (or [..., 1]).  What is held for the backward pass is one 8-bit checkpoint of each activation.
    codes [v, c] and views [n] (int): a code for each training view (photographs differ in exposure and white balance), code_scale * codes[view], beside the direction's
    encoding of every sample of the ray: views_linears.0 then takes c more columns (checkpoint.bake_view_code makes the network of one view for rendering); the codes
    receive their gradient by sorted views.  c may be no multiple of 6 (ValueError): such a network's shapes would be those of one with more frequencies, and queried, loaded or
    rendered without its codes it would be taken for that one; any other width is refused there.
    dtype: the type of the layers between the encodings and the heads (float32, bfloat16, float16: the last for a scaled loss); parameters stay what they are, heads are float32.
    None: what the module's attribute `layer_dtype` says, or float32."""
    dtype = dtype or getattr(network_fn, "layer_dtype", None) or torch.float32
    params = dict(network_fn.named_parameters())
    if getattr(network_fn, "is_color_independent_to_direction", False):
        raise NotImplementedError("colour-independent networks run on the fused kernels only")
    if (codes is None) != (views is None):
        raise ValueError("codes and views come together")
    lead, flat = inputs.shape[:-1], inputs.reshape(-1, 3)
    n_code = 0 if codes is None else codes.shape[1]
    if codes is not None and n_code % 6 == 0:
        raise ValueError("codes of %d columns: a multiple of 6 looks like the encoding of %d more frequencies to whatever meets the network without its codes; take another width "
                         "(one more column)" % (n_code, n_code // 6))
    depth, _, freqs, freqs_views = _network(params, n_code, viewdirs is not None)
    e = encode(flat, freqs).to(dtype)
    h, kept = dense(e, *_linear(params, "positions_linears.0"), relu=True)
    for i in range(1, depth):
        if i == 5:                                                              # cat([x, h]) behind layer 4 (:168)
            h, kept = torch.cat([e, h], -1), None
        h, kept = dense(h, *_linear(params, "positions_linears.%d" % i), relu=True, kept=kept)

    def head(x, names, kept_x):                                                 # the narrow outputs of one activation, float32
        w = [params[n + ".weight"] for n in names]
        b = [params[n + ".bias"] for n in names]
        y = dense(x.float(), w[0] if len(w) == 1 else torch.cat(w), b[0] if len(b) == 1 else torch.cat(b), kept=kept_x)[0]
        if len(names) > 1 and y.requires_grad:
            _leaves(*w, *b)
        return y

    if viewdirs is None:
        sigma = head(h, ("sigma_linear",), kept).reshape(lead + (1,))
        if sigma.requires_grad:
            _leaves(inputs)
        return sigma
    sigma_rough = head(h, ("sigma_linear", "roughness_linear"), kept)

    def branch(x, kept_x, feature, out):
        f, k = dense(x, *_linear(params, feature), relu=True, kept=kept_x)
        return head(f, (out,), k)

    albedo = branch(h, kept, "albedo_feature_linear", "albedo_linear")
    irradiance = branch(h, kept, "irradiance_feature_linear", "irradiance_linear")
    feature, _ = dense(h, *_linear(params, "feature_linear"), kept=kept)
    rays, samples = viewdirs.shape[0], flat.shape[0] // max(viewdirs.shape[0], 1)
    if rays * samples != flat.shape[0]:
        raise ValueError("%d points do not divide among %d directions" % (flat.shape[0], rays))
    ev = encode(viewdirs.reshape(-1, 3).to(flat.dtype), freqs_views).to(dtype)
    parts = [feature, ev[:, None].expand(rays, samples, ev.shape[1]).reshape(-1, ev.shape[1])]
    if codes is not None:
        if views.numel() != rays:
            raise ValueError("views has %d entries for %d rays" % (views.numel(), rays))
        parts.append(lookup(codes, views.reshape(-1), code_scale, rows_per_index=samples).to(dtype) if samples else codes.new_zeros((0, n_code), dtype=dtype))
    h2, kept2 = dense(torch.cat(parts, -1), *_linear(params, "views_linears.0"), relu=True)
    out = [sigma_rough[:, :1], albedo, sigma_rough[:, 1:], irradiance, head(h2, ("radiance_linear",), kept2)]
    out += [branch(h2, kept2, "additional_radiance_feature_linear.%d" % k, "additional_radiance_linear.%d" % k) for k in range(3)]
    raw = torch.cat(out, -1).reshape(lead + (18,))
    if raw.requires_grad:
        _leaves(inputs, viewdirs)
    return raw


GRADIENT_BYTES = 24 << 30      # what a piece of network_gradients may take beside the batch (of the card's 288 GB)


def gradient_points(params):
    """Samples that network_gradients takes at a time, at most 2^20: a sample holds a checkpoint of each layer's output and of the three inputs that no layer wrote (33 / 32 bytes a
    column), and beside them at most six float32 rows of the widest layer are alive (an activation and its gradient, the sum of the branches' gradients and the term being
    added, a concatenation and its parts)."""
    sides = {k[:-len(".weight")]: tuple(w.shape) for k, w in params.items() if k.endswith(".weight")}
    made = [o for o, _ in sides.values()] + [sides[k][1] for k in ("positions_linears.0", "positions_linears.5", "views_linears.0") if k in sides]
    a_sample = sum((c + 31) // 32 * 33 for c in made) + 6 * 4 * max(max(s) for s in sides.values())
    return max(1, min(1 << 20, GRADIENT_BYTES // a_sample))


def network_gradients(inputs, viewdirs, draw, network_fn, dtype=None, points=None):
    """{parameter name: dL/d parameter} of network_query from dL/d raw (draw [n, S, 18]), `points` samples at a time (None: gradient_points, by the network's widths), whole rays."""
    dtype = dtype or getattr(network_fn, "layer_dtype", None)
    named = dict(network_fn.named_parameters())
    names, params = list(named), list(named.values())
    points = points or gradient_points(named)
    total = None
    step = max(1, points // max(1, inputs.shape[1]))
    for i in range(0, inputs.shape[0], step):
        with torch.enable_grad():
            held = [p.detach().requires_grad_(True) for p in params]
            raw = network_query(inputs[i:i + step], viewdirs[i:i + step], _Named(dict(zip(names, held))), dtype=dtype)
        grads = torch.autograd.grad(raw, held, draw[i:i + step].contiguous())
        total = list(grads) if total is None else [a.add_(b) for a, b in zip(total, grads)]
    return dict(zip(names, total if total is not None else [torch.zeros_like(p) for p in params]))


class _Named:
    """Parameters by name, as network_query asks a module for them."""

    def __init__(self, params):
        self._params = params

    def named_parameters(self):
        return self._params.items()
