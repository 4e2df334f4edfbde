"""Networks outside the built 8 x 256 shape, layer by layer with gradients (layers.network_query through model.fused_network_query, training.render_rays_train), and a code for each
view: against the plain module in float64, against the reference's own loss.backward(), against the fused kernels.

What the tolerances count.  A weight's gradient reads its layer's input from the 8-bit checkpoint: a code's step is at most m / 63.5 (signed) or m / 127.5 (ReLU outputs) for the largest
magnitude m of its block of 32 columns — twice the finest, since the step is a power of two — so an entry is off by at most m / 127 or m / 255, and dW by that times sum |dy|.  dy itself
comes from exact masks: biases and inputs see float32 sums alone."""
import os

import numpy as np
import pytest

from conftest import GOLDEN

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    from ibl_nerf_amd import checkpoint as ck, layers, model as M  # noqa: E402
from test_layer_network import with_codes  # noqa: E402
from torch_ref import RefShaped, embed  # noqa: E402


def oracle(net, pts, dirs, arch, tail, draw, margin=0.0):
    """{layer: (its input [n, k], dL/d its output before the ReLU [n, o], ReLU?)}, raw, and which rows keep every ReLU's argument `margin` away from zero (relative to the layer's
    rms), in float64."""
    got, far = {}, torch.ones(pts.shape[0], dtype=torch.bool)
    hooks = []

    def hook(name):
        def f(mod, inp, out):
            out.retain_grad()
            got[name] = (inp[0].detach(), out)
            if name.startswith(("positions_", "views_")) or ("_feature_linear" in name):
                far.logical_and_((out.detach().abs() > margin * out.detach().square().mean().sqrt()).all(-1))
        return f
    for name, mod in net.named_modules():
        if isinstance(mod, torch.nn.Linear):
            hooks.append(mod.register_forward_hook(hook(name)))
    raw = net(embed(pts, arch[2]), None if dirs is None else torch.cat([embed(dirs, arch[3])] + ([] if tail is None else [tail]), -1))
    for h in hooks:
        h.remove()
    if draw is not None:
        (raw * draw).sum().backward()
    return got, raw.detach(), far


def most(x):
    """the largest magnitude of each entry's block of 32 columns"""
    n, k = x.shape
    p = torch.nn.functional.pad(x.abs(), (0, -k % 32)).reshape(n, -1, 32).amax(-1)
    return p.repeat_interleave(32, 1)[:, :k]


@pytest.mark.parametrize("arch,coded", [((10, 384, 12, 5), False), ((8, 512, 10, 4), True), ((2, 258, 2, 0), True), ((8, 256, 10, 4), True)])
def test_gradients_against_the_formula(arch, coded):
    net = RefShaped(ck.synthetic_arch_state_dict(21, arch, 1.5), arch).double()
    codes = with_codes(net, 9, 4) if coded else None
    g = torch.Generator().manual_seed(8)
    n = 700
    pts = (torch.rand(n, 3, generator=g) * 1.6 - 0.8).double()
    dirs = torch.nn.functional.normalize(torch.randn(n, 3, generator=g), dim=-1).float().double()
    views = torch.randint(0, 4, (n,), generator=g)                              # (view 4 is never used)
    draw = torch.randn(n, 18, generator=g).double()
    # rows whose ReLU arguments all keep 2e-5 of the layer's rms from zero: float32's errors flip none of their masks (what one flip changes is no error of a formula)
    tail = None if codes is None else 0.5 * codes[views]
    far = oracle(net, pts, dirs, arch, tail, None, 2e-5)[2]
    pts, dirs, views, draw = pts[far], dirs[far], views[far], draw[far]
    n = pts.shape[0]
    assert n >= 200
    if codes is not None:
        codes = codes.float().double().requires_grad_(True)
        tail = 0.5 * codes[views]
    got, raw, _ = oracle(net, pts, dirs, arch, tail, draw)
    import copy
    dev = copy.deepcopy(net).float().cuda()
    for p in dev.parameters():
        p.grad = None
    points = pts.float().cuda().reshape(n, 1, 3)
    dcodes = None if codes is None else codes.detach().float().cuda().requires_grad_(True)
    out = M.fused_network_query(points, dirs.float().cuda(), dev, codes=dcodes, views=None if codes is None else views.cuda(), code_scale=0.5)
    # 20 layers in sequence, each a float32 sum of up to 600 terms: 20 * 600 * 2^-23 = 1.5e-3 of the magnitudes summed if every rounding were against us
    assert (out.detach().double().cpu().reshape(n, 18) - raw).abs().max() <= 1.5e-3 * max(1.0, float(raw.abs().max()))
    out.backward(draw.float().cuda().reshape(n, 1, 18))
    for name, mod in dev.named_modules():
        if not isinstance(mod, torch.nn.Linear):
            continue
        x, y = got[name]
        dy = y.grad
        ref = dict(net.named_parameters())
        assert (mod.bias.grad.double().cpu() - ref[name + ".bias"].grad).abs().max() <= 1.5e-3 * dy.abs().sum(0).max(), name
        size = dy.abs().T @ x.abs()
        bound = dy.abs().T @ (most(x) / 127) + 1.5e-3 * size.max()
        assert ((mod.weight.grad.double().cpu() - ref[name + ".weight"].grad).abs() <= bound).all(), name
    if codes is not None:
        size = torch.zeros_like(codes).index_add_(0, views, (0.5 * got["views_linears.0"][1].grad.abs() @ net.views_linears[0].weight.detach().abs())[:, -codes.shape[1]:])
        assert ((dcodes.grad.double().cpu() - codes.grad).abs() <= 1.5e-3 * size.max()).all() and not dcodes.grad[4].any()
        # the network of one view, as it renders: its bias holds the code's products
        one = int(views[0])
        sd = ck.bake_view_code({k: v.detach() for k, v in dev.state_dict().items()}, (0.5 * dcodes.detach())[one])
        rows = torch.nonzero(views == one)[:, 0].cuda()
        from ibl_nerf_amd import renderer as R
        r = R.Renderer(64, 128)
        r.load_weights(0, sd)
        q = r.network_query(points[rows], dirs.float().cuda()[rows], 0).reshape(-1, 18)
        assert (q - out.detach().reshape(n, 18)[rows]).abs().max() <= 1.5e-3 * max(1.0, float(raw.abs().max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sixteen_bits_between_the_encodings_and_the_heads(dtype):
    """The layers in 16 bits against the same module evaluated by torch in that type: both are off the float64 network by their roundings; ours by no more than twice as much, in
    its outputs and in its gradients (whose checkpoint adds half a code step, of the size of bfloat16's own rounding)."""
    arch = (8, 512, 10, 4)
    net = RefShaped(ck.synthetic_arch_state_dict(5, arch), arch).cuda()
    g = torch.Generator().manual_seed(3)
    pts, dirs = (torch.rand(64, 33, 3, generator=g) - 0.5).cuda(), torch.nn.functional.normalize(torch.randn(64, 3, generator=g), dim=-1).cuda()
    draw = torch.randn(64, 33, 18, generator=g).cuda()
    e, d = embed(pts.reshape(-1, 3).double(), 10), embed(dirs.double().repeat_interleave(33, 0), 4)

    def grads(raw, params, up):
        return [t.double() for t in torch.autograd.grad(raw, params, up)]
    import copy
    exact, low = copy.deepcopy(net).double(), copy.deepcopy(net).to(dtype)
    raw64 = exact(e, d)
    g64 = grads(raw64, list(exact.parameters()), draw.reshape(-1, 18).double())
    raw16 = low(e.to(dtype), d.to(dtype))
    g16 = grads(raw16, list(low.parameters()), draw.reshape(-1, 18).to(dtype))
    raw = M.fused_network_query(pts, dirs, net, layer_dtype=dtype)
    assert raw.dtype == torch.float32 and raw.shape == (64, 33, 18)
    ours = grads(raw, list(net.parameters()), draw)
    off = lambda a, b: float((a.detach().double() - b.detach()).norm())
    assert off(raw.reshape(-1, 18), raw64) <= 2 * off(raw16, raw64)
    # What half a code step adds to a weight's gradient at most is sum |dy| most(x) / 127 (the head of this file); the 16-bit activations' blocks have their largest within 2^-6 of the
    # exact ones'.  (In proportion to the gradient it is more than 2 * 2^-8 where the sum cancels: draws of both signs leave an entry sqrt(rows) rms(x), the step's share is
    # sqrt(rows) most(x) / (127.5 sqrt(12)), and most(x) of a block of 32 ReLU outputs is 3 to 5 rms(x): about 1 %.)
    got = oracle(copy.deepcopy(net).double().cpu(), pts.reshape(-1, 3).double().cpu(), dirs.double().repeat_interleave(33, 0).cpu(), arch, None, draw.reshape(-1, 18).double().cpu())[0]
    for (name, _), a, b, c in zip(net.named_parameters(), ours, g16, g64):
        more = 2 * 2.0 ** -8 * float(c.norm())
        if name.endswith("weight"):
            x, y = got[name[:-7]]
            more = max(more, float((y.grad.abs().T @ (most(x) / 127)).norm()) * (1 + 2.0 ** -6))
        assert off(a, c) <= 2 * off(b, c) + more, name


@pytest.mark.parametrize("phase", ["warmup", "full"])
def test_a_training_step_of_a_larger_network(lut, phase):
    """IBLNeRF(6, 320, multires 12 / 5), outside the built shape, that computes what the fixture's IBLNeRF(6, 128, 6 / 2) computes — zero units, zero frequency columns: the
    reference's own loss.backward() holds for the sub-blocks, and what feeds or leaves a zero unit gets what the formula gives it (zero into the units' incoming weights).  Bars: the
    smaller network's own, and for weights 1 / 127 more for their checkpoints (a sum without cancellation keeps that relative error at worst)."""
    import train_loss as TL
    from ibl_nerf_amd import renderer as R
    from test_gpu_training import _grads_against
    G = np.load(os.path.join(GOLDEN, "train_step_arch.npz"))
    small = tuple(int(v) for v in G["arch"])
    arch = (small[0], 320, 12, 5)

    def places(name, kind):
        """the small parameter's rows and columns within the large one"""
        w, W, cp, Cp, cv = small[1], arch[1], 3 + 6 * small[2], 3 + 6 * arch[2], 3 + 6 * small[3]
        out = {n: o for n, o, _ in ck.arch_schema(*small)}[name]
        rows = torch.arange(out)
        if kind == "bias":
            return rows, None
        if name == "positions_linears.0":
            cols = torch.arange(cp)
        elif name == "positions_linears.5":
            cols = torch.cat([torch.arange(cp), Cp + torch.arange(w)])
        elif name == "views_linears.0":
            cols = torch.cat([torch.arange(w), W + torch.arange(cv)])
        else:
            cols = torch.arange({n: i for n, _, i in ck.arch_schema(*small)}[name])
        return rows, cols

    def take(t, name):
        rows, cols = places(*name.rsplit(".", 1))
        return t[rows.to(t.device)] if cols is None else t[rows.to(t.device)][:, cols.to(t.device)]

    nets, smalls = [], []
    for seed in (8100, 8101):
        sd = ck.synthetic_arch_state_dict(seed, small, 1.5)
        big = {k: torch.zeros_like(v) for k, v in RefShaped(arch=arch).state_dict().items()}
        for k, v in sd.items():
            rows, cols = places(*k.rsplit(".", 1))
            if cols is None:
                big[k][rows] = torch.from_numpy(v)
            else:
                big[k][rows[:, None], cols[None, :]] = torch.from_numpy(v)
        net = RefShaped(arch=arch)
        net.load_state_dict(big)
        net.coarse_radiance_number = 3
        nets.append(net.cuda())
        smalls.append(RefShaped(sd, small))
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=64, N_importance=128, perturb=1.0, pytest=True, raw_noise_std=0.0,
              brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True, correct_depth_for_prefiltered_radiance_infer=True,
              epsilon=0.01, target_normal_map_for_radiance_calculation="normal_map_from_depth_gradient_epsilon", use_radiance_linear=False,
              lindisp=False, near=float(G["near"]), far=float(G["far"]))
    f_ = np.float32(0.5 * 800 / np.tan(0.5 * np.deg2rad(60.0)))
    K = np.array([[f_, 0, 400], [0, f_, 400], [0, 0, 1]], dtype=np.float32)
    rays = torch.from_numpy(np.stack([G["rays_o"], G["rays_d"]], 0)).cuda()
    approx = phase == "full"
    res = R.render_decomp(800, 800, K, chunk=int(G["chunk"]), rays=rays, gt_values={}, approximate_radiance=approx, **kw)
    loss = TL.total_loss(torch, res, {k[8:]: G[k] for k in G.files if k.startswith("target__")}, approx)
    assert abs(float(loss.detach()) - float(G[phase + "__loss"])) <= (3e-4 if approx else 2e-5) * float(G[phase + "__loss"])
    loss.backward()
    for net, sm in zip(nets, smalls):
        for (name, p), (_, q) in zip(net.named_parameters(), sm.named_parameters()):
            assert p.grad is not None and p.grad.shape == p.shape, name
            q.grad = take(p.grad, name).cpu().reshape(q.shape)
    for net in nets:          # a zero unit has no outgoing weight: nothing reaches what feeds it
        assert not net.positions_linears[1].weight.grad[small[1]:].any() and not net.positions_linears[3].bias.grad[small[1]:].any()
    worst, zero = _grads_against(G, phase, smalls)
    assert len(worst) == 2 * 2 * (6 + 15) and not zero, (len(worst), zero)
    lim = lambda k: (5e-3 if (approx and "roughness_linear" in k) else (1.5e-3 if (approx and k.startswith("f.")) else 1e-3)) + (1 / 127 if k.endswith("weight") else 0.0)
    bad = {k: v for k, v in worst.items() if v > lim(k)}
    assert not bad, bad


def test_steps_of_a_larger_network_learn(lut):
    """Some optimizer steps of an IBLNeRF(8, 512) render on the live samples run through, and every parameter that the loss depends on moves."""
    from ibl_nerf_amd import renderer as R
    arch = (8, 512, 10, 4)
    nets = [RefShaped(ck.synthetic_arch_state_dict(s, arch, 1.5, sigma_bias=1.0), arch).cuda() for s in (1, 2)]
    for net in nets:
        net.coarse_radiance_number = 3
    before = [p.detach().clone() for net in nets for p in net.parameters()]
    opt = torch.optim.Adam([p for net in nets for p in net.parameters()], 5e-4)
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=32, N_importance=32, perturb=0.0, brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True, use_radiance_linear=False, near=0.5, far=4.0)
    g = torch.Generator().manual_seed(1)
    rays = torch.stack([torch.zeros(96, 3), torch.nn.functional.normalize(torch.randn(96, 3, generator=g), dim=-1)]).cuda()
    for _ in range(3):
        opt.zero_grad()
        res = R.render_decomp(8, 12, np.eye(3, dtype=np.float32), rays=rays, gt_values={}, approximate_radiance=False, **kw)
        loss = sum((res[k + s] - 0.3).square().mean() for k in ("radiance_map", "albedo_map", "irradiance_map", "roughness_map", "radiance_map_1", "radiance_map_2", "radiance_map_3") for s in ("", "0"))
        loss.backward()
        opt.step()
    assert all(torch.isfinite(p).all() and not torch.equal(p, q) for p, q in zip((p for net in nets for p in net.parameters()), before))


@pytest.mark.parametrize("approx", [False, True])
def test_a_batch_and_its_halves(lut, approx):
    """2 304 rays (the backward on the live samples, where a route would be held for the built shape): the gradients of a summed loss are those of its two halves.  The same rows, the
    same codes: what differs is the order of float32 sums over up to 2 304 x 64 rows (their rounding averages out: 2^-24 sqrt(10^5) = 2e-5 of the magnitudes summed) and the
    rows below 1e-7 of a pass's largest."""
    from ibl_nerf_amd import renderer as R
    arch = (8, 288, 10, 4)
    nets = [RefShaped(ck.synthetic_arch_state_dict(s, arch, 1.5, sigma_bias=1.0), arch).cuda() for s in (1, 2)]
    for net in nets:
        net.coarse_radiance_number = 3
    params = [p for net in nets for p in net.parameters()]
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=32, N_importance=32, perturb=0.0, brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True,
              use_radiance_linear=False, near=0.5, far=4.0, epsilon=0.01, correct_depth_for_prefiltered_radiance_infer=True,
              target_normal_map_for_radiance_calculation="normal_map_from_depth_gradient_epsilon")
    g = torch.Generator().manual_seed(1)
    rays = torch.stack([torch.zeros(2304, 3), torch.nn.functional.normalize(torch.randn(2304, 3, generator=g), dim=-1)]).cuda()

    def grads(part):
        res = R.render_decomp(8, 12, np.eye(3, dtype=np.float32), rays=rays[:, part].contiguous(), gt_values={}, approximate_radiance=approx, **kw)
        loss = sum((res[k + s] - 0.3).square().sum() for k in ("radiance_map", "albedo_map", "irradiance_map", "radiance_map_1") for s in ("", "0"))
        return torch.autograd.grad(loss, params, allow_unused=True)
    whole, a, b = grads(slice(0, 2304)), grads(slice(0, 1152)), grads(slice(1152, 2304))
    names = [n for net in nets for n, _ in net.named_parameters()]
    assert sum(w is not None and bool(w.any()) for w in whole) >= 60
    for n, w, x, y in zip(names, whole, a, b):
        if w is not None:
            assert (w - (x + y)).abs().max() <= 1e-3 * max(float(x.abs().max() + y.abs().max()), 1e-6), n


def test_a_context_takes_a_built_network_behind_a_larger_one():
    """weights that live on the GPU (a training step's) leave a slot that held a larger network as a fresh context has it"""
    from ibl_nerf_amd import renderer as R
    built, larger = (8, 256, 10, 4), (8, 264, 10, 4)
    sds = [{k: torch.from_numpy(v).cuda() for k, v in ck.synthetic_arch_state_dict(s, a, 1.5).items()} for s, a in ((4, built), (5, larger), (6, built))]
    g = torch.Generator().manual_seed(2)
    pts, dirs = (torch.rand(50, 7, 3, generator=g) - 0.5).cuda(), torch.randn(50, 3, generator=g).cuda()
    used, fresh = R.Renderer(64, 128), R.Renderer(64, 128)
    used.load_weights(0, sds[0])
    used.load_weights(0, sds[1])
    big = used.network_query(pts, dirs, 0)
    used.load_weights(0, sds[2])
    fresh.load_weights(0, sds[2])
    assert torch.equal(used.network_query(pts, dirs, 0), fresh.network_query(pts, dirs, 0)) and not torch.equal(used.network_query(pts, dirs, 0), big)


def test_points_and_density_alone_against_differences():
    """The density's gradient in the points (the trunk-only query of the normal modes) against central differences of the float64 module, on points whose ReLU arguments keep 2e-5 of
    their layer's rms from zero: no step of 1e-8 and no float32 error crosses one.  The differences are right to 1e-16 / 1e-8; the float32 products to 22 * 270 * 2^-23 = 7e-4 of the
    magnitudes summed."""
    arch = (10, 264, 4, 1)
    net = RefShaped(ck.synthetic_arch_state_dict(9, arch, 1.5), arch)
    import copy
    exact = copy.deepcopy(net).double()
    x = (torch.rand(100, 3, generator=torch.Generator().manual_seed(2)) - 0.5).double()
    x = x[oracle(exact, x, None, arch, None, None, 2e-5)[2]]
    x = x[:x.shape[0] // 5 * 5]
    assert x.shape[0] >= 40
    pts = x.float().cuda().requires_grad_(True)
    net = net.cuda()
    sigma = M.fused_query(pts.reshape(-1, 5, 3), None, net)
    assert sigma.shape == (x.shape[0] // 5, 5, 1)
    (got,) = torch.autograd.grad(sigma, pts, torch.ones_like(sigma))
    want = torch.zeros_like(x)
    for i in range(3):
        h = torch.zeros(3, dtype=torch.float64)
        h[i] = 1e-8
        want[:, i] = ((exact(embed(x + h, 4)) - exact(embed(x - h, 4)))[:, 0] / 2e-8).detach()
    assert ((got.double().cpu() - want).abs() <= 7e-4 * max(1.0, float(want.abs().max()))).all()


def test_pieces_of_a_batch_and_its_whole():
    """network_gradients in pieces of the batch adds what the whole gives (float32 sums of two pieces: half a step each), points that repeat included."""
    arch = (2, 264, 4, 1)
    net = RefShaped(ck.synthetic_arch_state_dict(9, arch), arch).cuda()
    g = torch.Generator().manual_seed(2)
    pts, dirs, draw = torch.rand(40, 8, 3, generator=g).cuda(), torch.randn(40, 3, generator=g).cuda(), torch.randn(40, 8, 18, generator=g).cuda()
    whole, parts = layers.network_gradients(pts, dirs, draw, net), layers.network_gradients(pts, dirs, draw, net, points=100)
    for k in whole:          # 320 terms of the sums, in another order
        assert (whole[k] - parts[k]).abs().max() <= 330 * 2.0 ** -23 * 40 * max(1e-3, float(whole[k].abs().max())), k
    none = layers.network_gradients(pts[:0], dirs[:0], draw[:0], net)
    assert set(none) == set(whole) and not any(v.any() for v in none.values())
    empty = M.fused_network_query(pts[:0], dirs[:0], net)
    assert empty.shape == (0, 8, 18)


def test_the_type_of_the_layers_is_the_modules_attribute(lut):
    from ibl_nerf_amd import renderer as R
    arch = (2, 264, 4, 1)
    nets = [RefShaped(ck.synthetic_arch_state_dict(s, arch, 1.5, sigma_bias=1.0), arch).cuda() for s in (1, 2)]
    g = torch.Generator().manual_seed(2)
    pts, dirs, draw = torch.rand(40, 8, 3, generator=g).cuda(), torch.randn(40, 3, generator=g).cuda(), torch.randn(40, 8, 18, generator=g).cuda()
    rays = torch.stack([torch.zeros(40, 3), torch.nn.functional.normalize(torch.randn(40, 3, generator=g), dim=-1)]).cuda()
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=32, N_importance=32, perturb=0.0, brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True,
              use_radiance_linear=False, near=0.5, far=4.0)

    def step():
        res = R.render_decomp(8, 12, np.eye(3, dtype=np.float32), rays=rays, gt_values={}, approximate_radiance=False, **kw)
        w = nets[1].positions_linears[1].weight
        return torch.autograd.grad((res["radiance_map"] - 0.3).square().sum(), w)[0]
    single = layers.network_gradients(pts, dirs, draw, nets[0]), M.fused_network_query(pts, dirs, nets[0]).detach(), step()
    low = layers.network_gradients(pts, dirs, draw, nets[0], dtype=torch.bfloat16), M.fused_network_query(pts, dirs, nets[0], layer_dtype=torch.bfloat16).detach()
    for net in nets:
        net.coarse_radiance_number, net.layer_dtype = 3, torch.bfloat16
    got = layers.network_gradients(pts, dirs, draw, nets[0]), M.fused_network_query(pts, dirs, nets[0]).detach(), step()
    assert all(torch.equal(got[0][k], low[0][k]) and got[0][k].dtype == torch.float32 for k in low[0]) and torch.equal(got[1], low[1])
    assert not torch.equal(got[1], single[1]) and not torch.equal(got[2], single[2])
    # (the step's gradient in 16 bits: 2 + 3 layers forward and backward, 10 roundings of 2^-8 and half a code step: 0.08 of the magnitudes summed, which here cancel little)
    assert float((got[2] - single[2]).norm()) <= 0.08 * float(single[2].norm())


def test_captured_training_of_a_network():
    """forward and backward in a graph, replayed with new points between eager work; an eager result of the same leaves that is alive is refused."""
    arch = (2, 264, 4, 1)
    net = RefShaped(ck.synthetic_arch_state_dict(9, arch), arch).cuda()
    params = list(net.parameters())
    g = torch.Generator().manual_seed(2)
    sets = [(torch.rand(16, 8, 3, generator=g).cuda(), torch.randn(16, 3, generator=g).cuda(), torch.randn(16, 8, 18, generator=g).cuda()) for _ in range(3)]
    want = [torch.autograd.grad(M.fused_network_query(p, d, net), params, u) for p, d, u in sets]
    pts, dirs, draw = (t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(M.fused_network_query(pts, dirs, net), params, draw)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = torch.autograd.grad(M.fused_network_query(pts, dirs, net), params, draw)
    for i in (1, 2, 0, 1):
        for dst, src in zip((pts, dirs, draw), sets[i]):
            dst.copy_(src)
        gr.replay()
        torch.autograd.grad(M.fused_network_query(*sets[2][:2], net), params, sets[2][2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    alive = M.fused_network_query(pts, dirs, net)
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            M.fused_network_query(pts, dirs, net)
    del alive


def test_memory_of_a_wide_networks_gradients(monkeypatch):
    """a batch of several pieces takes a piece's memory (a sample's bytes: layers.gradient_points) and the parameters' gradients: two pieces' and the running total, and the weights in the products' type"""
    arch = (6, 1024, 10, 4)
    net = RefShaped(ck.synthetic_arch_state_dict(9, arch), arch).cuda()
    monkeypatch.setattr(layers, "GRADIENT_BYTES", 1 << 30)
    piece = layers.gradient_points(dict(net.named_parameters()))
    n = 4 * piece // 64
    g = torch.Generator(device="cuda").manual_seed(2)
    pts, dirs, draw = torch.rand(n, 64, 3, generator=g, device="cuda"), torch.randn(n, 3, generator=g, device="cuda"), torch.randn(n, 64, 18, generator=g, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    layers.network_gradients(pts, dirs, draw, net)
    parameters = sum(4 * p.numel() for p in net.parameters())
    workspaces = 64 << 20          # (the weight gradient's pieces: up to 512 / tiles of a layer's float32 weights, a few MB each)
    assert torch.cuda.max_memory_allocated() - before <= (1 << 30) + 4 * parameters + workspaces


@pytest.mark.parametrize("arch", [(8, 264, 10, 4), (10, 258, 4, 2)])
def test_queries_without_a_gradient_are_the_render_paths(arch):
    """exact fp32, bit for bit what a render evaluates (and what these queries gave before they could be trained); a gradient, a type or a capture takes the trained layers"""
    net = RefShaped(ck.synthetic_arch_state_dict(9, arch, 1.5), arch).cuda()
    g = torch.Generator().manual_seed(2)
    pts, dirs = (torch.rand(20, 8, 3, generator=g) - 0.5).cuda(), torch.randn(20, 3, generator=g).cuda()
    want, sigma = M.network_query_fn(pts, dirs, net), M.network_query_fn(pts, None, net)
    with torch.no_grad():
        assert torch.equal(M.fused_network_query(pts, dirs, net), want) and torch.equal(M.fused_query(pts, dirs, net), want)
        assert torch.equal(M.fused_trunk_query(pts, net), sigma) and torch.equal(M.fused_query(pts, None, net), sigma)
        assert torch.equal(M.fused_trunk_query(pts.reshape(160, 3), net), sigma.reshape(160, 1))
        assert torch.equal(M.fused_network_query(pts.reshape(160, 3), dirs, net), want.reshape(160, 18))
        assert M.fused_network_query(pts[:0], dirs[:0], net).shape == (0, 8, 18) and M.fused_trunk_query(pts[:0], net).shape == (0, 8, 1)
        with pytest.raises(ValueError, match="divide"):
            M.fused_network_query(pts, dirs[:7], net)
        low = M.fused_network_query(pts, dirs, net, layer_dtype=torch.bfloat16)
    trained = M.fused_network_query(pts, dirs, net)
    assert trained.requires_grad and not torch.equal(trained, want) and not torch.equal(low, want)
    for p in net.parameters():
        p.requires_grad_(False)
    assert torch.equal(M.fused_network_query(pts, dirs, net), want)
    assert M.fused_trunk_query(pts.clone().requires_grad_(True), net).requires_grad
    net.layer_dtype = torch.bfloat16
    assert torch.equal(M.fused_network_query(pts, dirs, net), low)


def test_a_capture_meets_the_frameworks_own_eager_results(lut):
    """A fused query's result and a training render's, eager and alive, stand in a captured training pass's way like a layer's: refused at the forward pass.  (No backward pass is
    captured here; without the refusal one would end the process.)"""
    from ibl_nerf_amd import renderer as R
    built, larger = (8, 256, 10, 4), (2, 264, 4, 1)
    net = RefShaped(ck.synthetic_arch_state_dict(9, built), built).cuda()
    g = torch.Generator().manual_seed(2)
    pts, dirs = torch.rand(16, 8, 3, generator=g).cuda(), torch.randn(16, 3, generator=g).cuda()

    def refused(query):
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                query()

    query = lambda: M.fused_network_query(pts, dirs, net, layer_dtype=torch.bfloat16)      # noqa: E731
    query()
    for eager in (lambda: M.fused_network_query(pts, dirs, net), lambda: M.fused_trunk_query(pts, net), lambda: M.fused_trunk_features(pts, net),
                  lambda: M.fused_trunk_features2(pts, dirs, net)[1], lambda: M.fused_query(pts, dirs, net)):
        alive = eager()
        refused(query)
        del alive
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            query()
    nets = [RefShaped(ck.synthetic_arch_state_dict(s, larger, 1.5, sigma_bias=1.0), larger).cuda() for s in (1, 2)]
    for n in nets:
        n.coarse_radiance_number = 3
    rays = torch.stack([torch.zeros(40, 3), torch.nn.functional.normalize(torch.randn(40, 3, generator=g), dim=-1)]).cuda()
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=32, N_importance=32, perturb=0.0, brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True,
              use_radiance_linear=False, near=0.5, far=4.0)
    query = lambda: M.fused_network_query(pts, dirs, nets[1])      # noqa: E731
    query()
    res = R.render_decomp(8, 12, np.eye(3, dtype=np.float32), rays=rays, gt_values={}, approximate_radiance=False, **kw)
    loss = res["radiance_map"].sum()
    del res
    refused(query)
    del loss
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        query()
    moving = pts.clone().requires_grad_(True)
    alive = M.fused_network_query(moving, dirs, nets[1])
    for p in nets[1].parameters():
        p.requires_grad_(False)
    del alive
    alive = M.fused_network_query(moving, dirs, nets[1])
    refused(lambda: M.fused_network_query(moving, dirs, nets[1]))
    del alive


def test_weights_changed_before_the_backward_pass_are_refused(lut):
    """The layers' gradients come from a second forward pass on the module's parameters: an optimizer step between a render and its backward pass is an error, as it is in torch"""
    from ibl_nerf_amd import renderer as R
    arch = (2, 264, 4, 1)
    nets = [RefShaped(ck.synthetic_arch_state_dict(s, arch, 1.5, sigma_bias=1.0), arch).cuda() for s in (1, 2)]
    for n in nets:
        n.coarse_radiance_number = 3
    g = torch.Generator().manual_seed(2)
    rays = torch.stack([torch.zeros(40, 3), torch.nn.functional.normalize(torch.randn(40, 3, generator=g), dim=-1)]).cuda()
    kw = dict(network_fn=nets[0], network_fine=nets[1], N_samples=32, N_importance=32, perturb=0.0, brdf_lut=torch.from_numpy(lut).cuda(), lut_coefficient="F", gamma_correct=True,
              use_radiance_linear=False, near=0.5, far=4.0)
    params = [p for n in nets for p in n.parameters()]

    def loss():
        return (R.render_decomp(8, 12, np.eye(3, dtype=np.float32), rays=rays, gt_values={}, approximate_radiance=False, **kw)["radiance_map"] - 0.3).square().sum()
    want = torch.autograd.grad(loss(), params, allow_unused=True)
    first, second = loss(), loss()
    got = torch.autograd.grad(first, params, allow_unused=True)
    assert all((a is None) == (b is None) and (a is None or torch.equal(a, b)) for a, b in zip(got, want))
    with torch.no_grad():
        nets[1].positions_linears[0].weight.mul_(1.5)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(second, params, allow_unused=True)
    torch.autograd.grad(loss(), params, allow_unused=True)
