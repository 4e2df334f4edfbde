"""A network layer by layer (layers.network_query) on the CPU: its wiring against the plain module, with plain products in the places of the kernels; the codes of the views; what it
refuses; the sign that an eager graph leaves on its leaves."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from ibl_nerf_amd import checkpoint as ck, layers  # noqa: E402
from torch_ref import RefShaped, embed  # noqa: E402


def plain_dense(x, weight, bias=None, relu=False, kept=None):
    y = x @ weight.to(x.dtype).T + bias.to(x.dtype)
    y = torch.relu(y) if relu else y
    assert kept is None or torch.equal(kept.to(x.dtype), x)          # (the checkpoint that is handed on is the one of this very input)
    return y, y.detach()


def plain_lookup(table, index, scale=1.0, rows_per_index=1):
    return (scale * table[index.long()]).repeat_interleave(rows_per_index, 0)


@pytest.fixture()
def plain(monkeypatch):
    monkeypatch.setattr(layers, "dense", plain_dense)
    monkeypatch.setattr(layers, "lookup", plain_lookup)


def with_codes(net, c, seed):
    """The module with c more columns in views_linears.0 and a table of 5 codes."""
    g = torch.Generator().manual_seed(seed)
    old = net.views_linears[0]
    new = torch.nn.Linear(old.in_features + c, old.out_features).to(old.weight.dtype)
    with torch.no_grad():
        new.weight.copy_(torch.cat([old.weight, 0.3 * torch.randn(old.out_features, c, generator=g, dtype=old.weight.dtype)], 1))
        new.bias.copy_(old.bias)
    net.views_linears[0] = new
    return torch.randn(5, c, generator=g, dtype=old.weight.dtype)


ARCHS = [(8, 256, 10, 4), (2, 6, 3, 0), (6, 32, 0, 2), (10, 48, 12, 5)]


@pytest.mark.parametrize("arch", ARCHS)
@pytest.mark.parametrize("coded", [False, True])
def test_wiring(plain, arch, coded):
    net = RefShaped(ck.synthetic_arch_state_dict(3, arch), arch).double()
    codes = with_codes(net, 7, 11) if coded else None
    g = torch.Generator().manual_seed(5)
    pts, dirs = torch.rand(4, 3, 3, generator=g, dtype=torch.float64) * 2 - 1, torch.randn(4, 3, generator=g, dtype=torch.float64)
    views = torch.tensor([2, 0, 4, 2])
    e, d = embed(pts.reshape(-1, 3), arch[2]), embed(dirs.repeat_interleave(3, 0), arch[3])
    if coded:
        d = torch.cat([d, 0.5 * codes[views].repeat_interleave(3, 0)], -1)
        got = layers.network_query(pts, dirs, net, codes=codes, views=views, code_scale=0.5, dtype=torch.float64)
    else:
        got = layers.network_query(pts, dirs, net, dtype=torch.float64)
    want = net(e, d).reshape(4, 3, 18).detach()
    # the heads run in float32: the feature layers' outputs rounded once (2^-24), products of up to 256 terms summed in float32
    assert (got - want).abs().max() <= 300 * 2.0 ** -23 * max(1.0, float(want.abs().max())) and got.dtype == torch.float32
    sigma = layers.network_query(pts, None, net, dtype=torch.float64)
    assert sigma.shape == (4, 3, 1) and (sigma[..., 0] - got[..., 0]).abs().max() <= 300 * 2.0 ** -23 * max(1.0, float(want.abs().max()))      # (another order of the same sum)


def test_encode():
    x = torch.rand(50, 3, dtype=torch.float64) * 4 - 2
    for k in (0, 1, 4, 24):
        assert layers.encode(x, k).shape == (50, 3 + 6 * k) and (layers.encode(x, k) - embed(x, k)).abs().max() <= 1e-15 * 2.0 ** k
    x32 = x.float()                # float32 points: one rounding of the true sine
    e = layers.encode(x32, 12)
    assert e.dtype == torch.float32 and (e.double() - embed(x32.double(), 12)).abs().max() <= 2.0 ** -24 + 1e-11


def test_bake_view_code():
    arch = (6, 32, 4, 2)
    net = RefShaped(ck.synthetic_arch_state_dict(3, arch), arch).double()
    codes = with_codes(net, 7, 2)
    e, d = torch.randn(9, 27, dtype=torch.float64), torch.randn(9, 15, dtype=torch.float64)
    want = net(e, torch.cat([d, 0.25 * codes[3].expand(9, 7)], -1))
    sd = ck.bake_view_code(net.state_dict(), 0.25 * codes[3])
    one = RefShaped(arch=arch).double()
    one.load_state_dict(sd)
    assert ck.arch_of(sd) == arch and (one(e, d) - want).abs().max() <= 1e-13
    sn = ck.bake_view_code({k: v.numpy() for k, v in net.state_dict().items()}, (0.25 * codes[3]).numpy())
    assert all(isinstance(v, np.ndarray) and np.allclose(v, sd[k].numpy(), rtol=0, atol=1e-14) for k, v in sn.items())
    for bad in (codes, torch.zeros(0), torch.zeros(54), codes[0, :5]):
        with pytest.raises(ValueError):
            ck.bake_view_code(net.state_dict(), bad)


def test_refuses(plain):
    arch = (2, 16, 2, 1)
    net = RefShaped(ck.synthetic_arch_state_dict(3, arch), arch)
    p, d, codes = torch.zeros(4, 3, 3), torch.zeros(4, 3), torch.zeros(5, 7)
    with pytest.raises(ValueError, match="together"):
        layers.network_query(p, d, net, codes=codes)
    with pytest.raises(ValueError, match="together"):
        layers.network_query(p, d, net, views=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="columns"):
        layers.network_query(p, d, net, codes=codes, views=torch.zeros(4, dtype=torch.int32))          # (the network has no columns for a code)
    with_codes(net, 7, 1)
    with pytest.raises(ValueError, match="columns"):
        layers.network_query(p, d, net)
    with pytest.raises(ValueError, match="entries"):
        layers.network_query(p, d, net, codes=codes, views=torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="divide"):
        layers.network_query(p, torch.zeros(5, 3), net, codes=codes, views=torch.zeros(5, dtype=torch.int32))
    net.is_color_independent_to_direction = True
    with pytest.raises(NotImplementedError):
        layers.network_query(p, d, net)


def test_an_eager_graph_signs_its_leaves():
    w, b = torch.nn.Parameter(torch.zeros(3)), torch.zeros(3)
    layers._leaves(w, b, None, capturing=True)                  # nothing alive
    layers._leaves(w, b, None, capturing=False)
    layers._leaves(w, capturing=True)                           # (the sign went with the node: no graph holds it)
    y = (w * 2).sum()
    layers._leaves(w, capturing=False)
    with pytest.raises(RuntimeError, match="alive"):
        layers._leaves(w, capturing=True)
    layers._leaves(b, capturing=True)
    del y
    layers._leaves(w, capturing=True)
    z = w * 2
    layers._leaves(w, capturing=True)                           # a graph made within the capture is no eager one
    del z


def test_pieces_of_the_gradients_go_by_the_widths():
    """the 512-wide network keeps its 2^20 samples a piece; the widest one that trains takes what fits the same memory"""
    def shapes(arch):
        return {n + ".weight": torch.empty(o, i, device="meta") for n, o, i in ck.arch_schema(*arch)}
    assert layers.gradient_points(shapes((8, 512, 10, 4))) == 1 << 20 and layers.gradient_points(shapes((9, 256, 10, 4))) == 1 << 20
    for arch in ((8, 1024, 10, 4), (32, 512, 10, 4), (32, 4096, 24, 24)):
        held = sum(33 / 32 * o for _, o, _ in ck.arch_schema(*arch))
        n = layers.gradient_points(shapes(arch))
        assert 1000 < n < 1 << 20 and n * (held + 4 * 4 * arch[1]) < layers.GRADIENT_BYTES
    assert layers.gradient_points(shapes((32, 4096, 24, 24))) > 80000


@pytest.mark.parametrize("arch", [(5, 64, 4, 2), (5, 512, 10, 4), (8, 513, 10, 4), (33, 64, 4, 2), (2, 4098, 1, 1), (2, 64, 25, 4), (2, 64, 4, 25)])
def test_refuses_what_no_other_path_takes(plain, arch):
    """5 layers (the module's own forward fails: the skip's concatenation is consumed by none), odd widths beyond the built one, more than 32 layers, more than 24 frequencies"""
    from ibl_nerf_amd import model as M
    net = RefShaped(arch=arch)
    p, d = torch.zeros(2, 3, 3), torch.ones(2, 3)
    for call in (lambda: M.fused_query(p, d, net), lambda: M.fused_network_query(p, d, net), lambda: layers.network_query(p, d, net), lambda: layers.network_gradients(p, d, torch.zeros(2, 3, 18), net)):
        with pytest.raises(NotImplementedError, match="outside"):
            call()
    if arch[3] <= 24:
        for call in (lambda: M.fused_query(p, None, net), lambda: M.fused_trunk_query(p, net)):
            with pytest.raises(NotImplementedError, match="outside"):
                call()


def test_refuses_layers_that_it_would_not_run(plain):
    """a fourth coarse radiance, a second view layer, a skip elsewhere: never 18 columns of another network"""
    p, d = torch.zeros(2, 3, 3), torch.ones(2, 3)

    def net(change, arch=(6, 64, 12, 5)):
        n = RefShaped(arch=arch)
        change(n)
        return n

    def fourth(n):
        n.additional_radiance_feature_linear.append(torch.nn.Linear(64, 32))
        n.additional_radiance_linear.append(torch.nn.Linear(32, 3))

    def skip(n):
        n.positions_linears[5], n.positions_linears[3] = torch.nn.Linear(64, 64), torch.nn.Linear(64 + 75, 64)

    for change, word in ((fourth, "additional_radiance"), (lambda n: n.views_linears.append(torch.nn.Linear(64, 64)), "views_linears.1"), (skip, "positions_linears"),
                         (lambda n: n.__delattr__("irradiance_linear"), "irradiance_linear")):
        with pytest.raises(NotImplementedError, match=word):
            layers.network_query(p, d, net(change))
    with pytest.raises(NotImplementedError, match="positions_linears"):
        layers.network_query(p, None, net(skip))
    assert layers.network_query(p, None, net(fourth)).shape == (2, 3, 1)                       # (the density has nothing to do with them)
    n = net(lambda n: n.register_parameter("my_codes", torch.nn.Parameter(torch.zeros(4, 5))))  # parameters that are no layer of the network stay out of its way
    assert layers.network_query(p, d, n).shape == (2, 3, 18)


@pytest.mark.parametrize("c", [6, 12, 48])
def test_a_codes_width_is_never_that_of_frequencies(plain, c):
    """a network trained with codes of 6 m columns would be read as one of m more direction frequencies wherever it is met without them: not trained; any other width is refused there"""
    arch = (6, 32, 4, 2)
    p, d, views = torch.zeros(4, 3, 3), torch.ones(4, 3), torch.zeros(4, dtype=torch.int32)
    net = RefShaped(arch=arch)
    codes = with_codes(net, c, 2)
    assert ck.arch_of(net.state_dict()) == (6, 32, 4, 2 + c // 6)
    with pytest.raises(ValueError, match="multiple of 6"):
        layers.network_query(p, d, net, codes=codes, views=views)
    net = RefShaped(arch=arch)
    codes = with_codes(net, c + 1, 2)
    assert layers.network_query(p, d, net, codes=codes, views=views).shape == (4, 3, 18)
    with pytest.raises(ValueError, match="columns"):
        layers.network_query(p, d, net)
    with pytest.raises(ValueError, match="encoding"):
        ck.arch_of(net.state_dict())


def test_a_functions_result_signs_its_leaves():
    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            return 2 * w, 3 * w

        @staticmethod
        def backward(ctx, a, b):
            return None, 2 * a + 3 * b

    w, b, x = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3)), torch.zeros(3)
    y = Twice.apply(x, w)
    layers.sign(y[0], capturing=True)                           # made within a capture: nothing stands in its way
    layers._leaves(w, capturing=True)
    layers.sign(y[0], capturing=False)
    with pytest.raises(RuntimeError, match="alive"):
        layers._leaves(b, w, capturing=True)
    layers._leaves(b, capturing=True)
    del y
    layers._leaves(w, capturing=True)
    layers.sign(Twice.apply(x, x)[0], capturing=False)          # (nothing to differentiate)


def test_what_holds_an_accumulator_is_named():
    """a distributed wrapper or a hook keeps the node, and the sign, with no result alive: the refusal says so"""
    w = torch.nn.Parameter(torch.zeros(3))
    held = w.view_as(w).grad_fn.next_functions[0][0]
    (w * 2).sum()
    layers._leaves(w, capturing=False)
    with pytest.raises(RuntimeError, match="wrapper.*side stream"):
        layers._leaves(w, capturing=True)
    del held
    layers._leaves(w, capturing=True)


def test_points_that_carry_a_gradient_are_signed(plain, monkeypatch):
    seen = []
    monkeypatch.setattr(layers, "_leaves", lambda *t, **k: seen.extend(t))
    net, p, d = RefShaped(arch=(6, 32, 4, 2)), torch.zeros(4, 3, 3, requires_grad=True), torch.ones(4, 3, requires_grad=True)
    layers.network_query(p, d, net)
    assert any(t is p for t in seen) and any(t is d for t in seen)
    seen.clear()
    layers.network_query(p, None, net)
    assert any(t is p for t in seen)
