"""A training step's render on the fused kernels, forward AND backward: ONE torch.autograd.Function around render_rays.

Replaces, for train.py:285-297 / :479-481, what torch autograd does through the reference's render_decomp -> batchify_rays -> render_rays ->
raw2outputs (nerf_models/ibl_nerf_renderer.py:759-813, :629-732, :153-527) when `network_fn` / `network_fine` are trainable nn.Modules:

    forward   approximate_radiance=True:  iblnerf_render_rays_tapped — the inference path itself, which also hands out both passes' z_vals
              and main raw rows; approximate_radiance=False (the first N_iter_ignore_approximated_radiance iterations, train.py:295) and
              is_depth_only (:366-374): the stages of render_rays strung together (iblnerf_coarse_z / _sample_points / _network_query /
              _composite_direct / _fine_z / _composite_sigma).
    backward  per pass: dL/d(output maps) -> dL/d(the 19 linear direct maps) by torch autograd over the RAY-sized part of raw2outputs
              (`_ray_outputs`: output lambdas, disparity, and under approximate_radiance the split-sum shading :412-474 — LUT fetch by
              F.grid_sample, Fresnel, mip interpolation, gamma — with everything the reference computes under no_grad / detached held
              constant: the normal :358-361, x_surface :263, the reflected-ray maps :442-448, depth in the mip level :455) ->
              iblnerf_composite_direct_backward (the reference's weights_detached stop-gradients, :246) -> dL/d raw [n, S, 18] ->
              iblnerf_network_backward -> the 46 parameter gradients of that pass's network.
Nothing of size [n_rays, n_samples] is computed by torch: such tensors exist only as buffers the kernels read and write.
`forward_freezed` (ibl_nerf.py:88-152; train.py:275-283): with network.freeze_radiance only the albedo / irradiance feature layers and heads
(and roughness_linear unless freeze_roughness) receive gradients — the upstream rows of the frozen outputs are zeroed and the gradients
of the frozen layers dropped.

Edit / insert overrides and the four *_from_gt substitutions are constants of the backward (override_rows, _gt_constants), under either value of
approximate_radiance; colour-independent networks run the same backward with the identity in place of their unused feature / view layers.
Auxiliary networks receive their columns' gradients (Renderer.aux_backward); use_gradient_for_incident_radiance carries dL/d(reflected-ray maps) through the
reflected query into the pass's network.  Not built here (raise): a trainable depth_mlp (infer_depth; the reference's own backward raises there), a trainable
normal_mlp as the target normal.  (raw_noise_std > 0 is: the step's noise rows are drawn once, added to the
density the compositing reads in both directions, and are constants of the backward.)
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import binding as B
from . import checkpoint as ck

ALL_PARAMS = tuple(n + s for n, _, _ in ck.SCHEMA for s in (".weight", ".bias"))
# network_backward_live: a pass of at least this many points is compacted to its live samples before the network's backward (below it the two extra launches and the one
# host synchronisation for the count cost more than the dead samples: a 512-ray step is launch-bound)
COMPACT_MIN_POINTS = 131072
# ... and a row counts as live when its largest entry exceeds this share of the pass's largest: a sample deep behind a surface (transmittance 1e-8 .. 1e-30) has a
# nonzero row of dL/d raw too — 70 % of the coarse pass's nonzero rows and 10 % of the fine pass's lie below 1e-8 of the largest (scratch/live_rows_hist.py) — and all of
# them together move no parameter gradient by 1e-7 of itself, four orders below what the backward's f16 operand stash resolves
LIVE_REL = 1e-7


def network_backward_live(r, pts, rays_d, draw, which, backward=None):
    """Renderer.network_backward on the samples that carry a gradient only.  A sample whose density is not positive has alpha = 0: its weight is exactly zero and the ReLU in
    front of the density is dead, so its whole row of dL/d raw is EXACTLY zero (iblnerf_composite_direct_backward) — nine in ten samples on a scene with surfaces — and a
    zero row adds exactly nothing to any parameter gradient.  Those rows — and the rows below LIVE_REL of the pass's largest — are dropped (one mask, one nonzero — the
    step's only host synchronisation — three gathers) and the
    fused backward runs on the rest as a batch of one-sample "rays": the same kernels, a third of the points (round 6: "training evaluates every
    sample").  Parameter gradients agree with the whole batch's to fp32 round-off of the weight-gradient sums (another grouping of the same terms); dL/d pts is not returned
    (a training step's rays are constants).  backward: another (pts, rays_d, draw) -> (dL/d pts or None, gradients) than the fused one (a network that runs layer by layer)."""
    torch = __import__("torch")
    backward = backward or (lambda p, d, u: r.network_backward(p, d, u, which))
    n, S = int(pts.shape[0]), int(pts.shape[1])
    if n * S < COMPACT_MIN_POINTS:
        return backward(pts, rays_d, draw)
    rows = draw.reshape(n * S, -1)
    mag = rows.abs().amax(-1)
    idx = (~(mag <= LIVE_REL * mag.max())).nonzero().reshape(-1)      # (an all-zero upstream gradient: every row is dropped; a NaN row is kept, so that it shows)
    if idx.numel() > 0.7 * n * S:                      # fog: (almost) everything is live
        return backward(pts, rays_d, draw)
    if idx.numel() == 0:
        idx = torch.zeros((1,), dtype=torch.long, device=rows.device)      # (an all-zero upstream gradient: one dead sample keeps the call's shape; its gradients are zeros)
    pts_c = pts.reshape(n * S, 3)[idx].reshape(-1, 1, 3).contiguous()
    rd_c = rays_d.reshape(n, 3)[idx // S].contiguous()
    return backward(pts_c, rd_c, rows[idx].reshape(-1, 1, rows.shape[-1]).contiguous())

# parameters that still receive gradients under forward_freezed (ibl_nerf.py:113-131)
UNFROZEN = ("albedo_feature_linear.", "albedo_linear.", "irradiance_feature_linear.", "irradiance_linear.", "roughness_linear.")
MAP3 = ("albedo_map", "radiance_map", "radiance_map_1", "radiance_map_2", "radiance_map_3")
# the ray-sized shading's backward: one fused launch (iblnerf_ray_outputs_backward) | torch autograd through _ray_outputs (False: the tests' reference)
FUSED_SHADING_BACKWARD = True
# output maps that carry a gradient into the linear direct maps (the others are computed under no_grad / detached in the reference)
SHADED_KEYS = ("color_map", "radiance_map", "radiance_map_1", "radiance_map_2", "radiance_map_3", "irradiance_map", "albedo_map", "roughness_map",
               "specular_map", "diffuse_map", "prefiltered_reflected_map", "disp_map", "acc_map", "depth_map", "target_depth_map")


# auxiliary networks (ibl_nerf_renderer.py:291-303): the raw columns their outputs replace; normal_mlp (:267-275) feeds inferred_normal_map instead
AUX_COLS = {"albedo_mlp": slice(1, 4), "roughness_mlp": slice(4, 5), "irradiance_mlp": slice(5, 6)}
AUX_PARAMS = tuple("positions_linears.%d.%s" % (i, t) for i in range(8) for t in ("weight", "bias")) + ("out_linears.weight", "out_linears.bias")


def _torch():
    import torch
    return torch


def is_training_call(kw):
    """render_decomp was called the way train.py calls it: autograd on and a network with trainable parameters."""
    torch = _torch()
    if not torch.is_grad_enabled():
        return False
    for net in (kw.get("network_fn"), kw.get("network_fine")) + tuple(kw.get(k) for k in AUX_COLS) + ((kw.get("normal_mlp"),) if kw.get("infer_normal") else ()):
        ps = getattr(net, "parameters", None)
        if ps is not None and any(getattr(p, "requires_grad", False) for p in ps()):
            return True
    return False


def _gamma(x, on):
    return (x + 1e-12) ** (1.0 / 2.2) if on else x            # rgb_to_srgb, ibl_nerf_renderer.py:26-27


def _ungamma(y, on):
    return (y ** 2.2 - 1e-12).clamp_min(0.0) if on else y


def _ray_outputs(x, consts, flags, gt=None):
    """The ray-sized part of raw2outputs as differentiable torch: x [n, 19] = the linear direct maps (Renderer.MAP_SLOTS order) -> the
    pass's output maps.  consts (approximate_radiance): n_dot_v [n], env [n, 4, 3] linear reflected-ray maps, lut [3, 512, 512],
    depth0 = (near + far) / 2.  gt: the target maps of the *_from_gt flags that are on (:251-252, :320-330), constants."""
    torch = _torch()
    import torch.nn.functional as F
    gt = gt or {}
    g, hdr = flags["gamma_correct"], flags["use_radiance_linear"]
    out_f = (lambda v: _gamma(v / (v + 1) if hdr else v, g))                         # output_f (:480-490)
    depth, acc = x[:, 0], x[:, 1]
    rough_net = x[:, 5]                                                             # roughness_map: the mip level reads it whatever the target is (:457-460)
    albedo = gt["albedo"] if gt.get("albedo") is not None else x[:, 2:5]
    rough = gt["roughness"] if gt.get("roughness") is not None else rough_net
    irr = gt["irradiance"] if gt.get("irradiance") is not None else x[:, 6:7]       # [n, 3] | [n, 1]
    res = {"radiance_map": out_f(x[:, 7:10])}
    for k in range(3):
        res["radiance_map_%d" % (k + 1)] = out_f(x[:, 10 + 3 * k:13 + 3 * k])
    res["irradiance_map"] = out_f(irr)                                              # target_irradiance_map = irradiance_map[..., None] (:326)
    res["albedo_map"] = _gamma(albedo, g)                                           # albedo_f (:491)
    res["roughness_map"] = rough
    q = depth / acc
    res["disp_map"] = 1.0 / torch.maximum(torch.full_like(q, 1e-10), q)             # :258
    res["acc_map"], res["depth_map"] = acc, depth
    res["target_depth_map"] = gt["depth"] if gt.get("depth") is not None else depth
    if consts is None:
        return res
    ndv, env, lut = consts["n_dot_v"], consts["env"], consts["lut"]
    uv = torch.stack([2 * ndv - 1, 2 * rough - 1], -1)                              # :418
    e = F.grid_sample(lut[None], uv[None, :, None, :], align_corners=True)[0, :, :, 0].t()      # [n, 3]  (:419-421)
    metallic = (1 - rough)[:, None]
    F0 = 0.04 * (1 - metallic) + albedo * metallic                                  # :424-427
    F1 = torch.maximum(1.0 - rough[:, None], F0) - F0                               # fresnel_schlick_roughness (microfacet.py:8-12)
    fres = F0 + F1 * torch.clip(1.0 - ndv[:, None], 0.0, 1.0) ** 5.0
    coef = (fres if flags["lut_coefficient"] == "F" else F0) * e[:, 0:1] + e[:, 1:2]             # :433-436
    if flags["correct_depth"]:
        level = torch.clip(rough_net * depth.detach() / consts["depth0"], 0, 1)     # :453-457
    else:
        level = rough_net
    i1 = torch.clip((level * 3).long(), 0, 3)
    i2 = torch.clip(i1 + 1, 0, 3)
    rem = (level * 3 - i1)[:, None]
    ar = torch.arange(env.shape[0], device=env.device)
    pref = (1 - rem) * env[ar, i1] + rem * env[ar, i2]                              # :461-467
    diffuse = (1 - fres) * (1 - metallic) * albedo * irr                            # :469
    spec = coef * pref
    res.update(color_map=out_f(diffuse + spec), specular_map=out_f(spec), diffuse_map=out_f(diffuse), prefiltered_reflected_map=out_f(pref))
    return res


def override_rows(r, n, gt_values, edit, approximate_radiance, chunk=None):
    """The edit / insert overrides of raw2outputs (ibl_nerf_renderer.py:218-238 masks; :253-256 depth; :378-410 albedo / roughness / irradiance — the latter three only
    inside `if approximate_radiance`) as RAY-sized rows: {"depth" | "albedo" | "roughness" | "irradiance": (mask [n] bool, values [n] or [n, 3])} in the order the
    reference assigns them.  In the reference they are in-place masked assignments on the target maps: the masked rows become constants of the step (no gradient
    reaches the network's own map there, neither through the output of that name nor through the shading), the other rows are untouched.  The forward applies
    them in pass A (iblnerf_overrides); a backward substitutes them into the linear maps it differentiates at and zeroes dL/d(those entries).
    (The normal overrides make n.v and the reflected ray constants of the backward already: both are computed under no_grad / detached, :358-361, :442.)"""
    torch = _torch()
    from .renderer import _dev_f32, _truthy, resolve_edit_roughness
    edit = edit or {}
    gv = gt_values or {}
    on = lambda k: _truthy(edit.get(k, False))
    ei, io = on("edit_intrinsic"), on("insert_object")
    if not ei and not io:
        return {}
    dev = r.device
    row = lambda key: _dev_f32(gv[key], dev).reshape(n, -1)
    mask_img = row("edit_intrinsic_mask" if ei else "object_insert_mask")[:, 0]
    nobj = int(edit.get("num_edit_objects" if ei else "num_insert_objects") or 0)
    assert nobj > 0, "num_edit_objects must be greater than 0" if ei else "num_insert_objects must be greater than 0"
    masks = [torch.logical_and(11 * (i + 1) / 255. > mask_img, mask_img > 9 * (i + 1) / 255.) for i in range(nobj)]        # :224-226, :234-236
    mask_all = mask_img > 0
    out = {}

    def per_object(values, width):
        """the objects' masks assigned in order (a later object wins where two masks overlap — they cannot: disjoint grey-level bands)"""
        m = torch.zeros((n,), dtype=torch.bool, device=dev)
        v = torch.zeros((n, width), dtype=torch.float32, device=dev)
        for i, val in enumerate(values):
            if val is None:
                continue
            m = m | masks[i]
            v[masks[i]] = torch.as_tensor(val, dtype=torch.float32, device=dev).reshape(1, width)
        return m, (v if width > 1 else v[:, 0])

    if ei:
        if on("edit_depth"):
            out["depth"] = (mask_all, row("edit_depth")[:, 0])
        if approximate_radiance:
            if on("edit_albedo"):
                if on("edit_albedo_by_img"):
                    out["albedo"] = (mask_all, row("edit_albedo")[:, :3])
                else:
                    alb = list(edit.get("editing_target_albedo_list") or [])
                    out["albedo"] = per_object([alb[3 * i:3 * i + 3] for i in range(nobj)], 3)
            if on("edit_roughness"):
                if on("edit_roughness_by_img"):
                    per_ray = (_dev_f32(gv["_edit_roughness_resolved"], dev).reshape(n) if "_edit_roughness_resolved" in gv
                               else resolve_edit_roughness(mask_img, row("edit_roughness")[:, 0], chunk))
                    out["roughness"] = (mask_all, per_ray)
                else:
                    out["roughness"] = per_object(list(edit.get("editing_target_roughness_list") or [])[:nobj], 1)
    else:
        out["depth"] = (mask_all, row("object_insert_depth")[:, 0])
        if approximate_radiance:
            rgh = list(edit.get("inserting_target_roughness_list") or [])
            alb = list(edit.get("inserting_target_albedo_list") or [])
            irr = list(edit.get("inserting_target_irradiance_list") or [])
            out["roughness"] = per_object(rgh[:nobj], 1)
            out["irradiance"] = per_object([v if v > 0 else None for v in irr[:nobj]], 1)                                    # :406-407
            out["albedo"] = per_object([alb[3 * i:3 * i + 3] for i in range(nobj)], 3)
    return out


# the columns of the linear direct maps (Renderer.MAP_SLOTS order) an override of that name replaces
_OVERRIDE_COLS = {"depth": slice(0, 1), "albedo": slice(2, 5), "roughness": slice(5, 6), "irradiance": slice(6, 7)}


def _apply_overrides(x, gt_const, rows):
    """(x', gt') with the override rows substituted where the reference's in-place assignments land: in the ground-truth map when a *_from_gt flag made that the
    target (:321-330: target_albedo_map = gt_values["albedo"], then target_albedo_map[mask] = ...), else in the network's own map."""
    torch = _torch()
    if not rows:
        return x, gt_const
    x = x.clone()
    gt_const = dict(gt_const or {})
    for name, (mask, vals) in rows.items():
        if gt_const.get(name) is not None:
            g = gt_const[name].clone()
            v = vals if vals.dim() == g.dim() else vals[:, None].expand_as(g)
            gt_const[name] = torch.where(mask[:, None] if g.dim() == 2 else mask, v, g).contiguous()
        else:
            cols = _OVERRIDE_COLS[name]
            v = vals if vals.dim() == 2 else vals[:, None]
            x[:, cols] = torch.where(mask[:, None], v, x[:, cols])
    return x, gt_const


def _zero_overridden(dx, gt_const, rows):
    """dL/d(linear maps) of the rows an override made constants"""
    for name, (mask, _) in (rows or {}).items():
        if (gt_const or {}).get(name) is None:
            dx[:, _OVERRIDE_COLS[name]] = dx[:, _OVERRIDE_COLS[name]].masked_fill(mask[:, None], 0.0)
    return dx


def _flags(r):
    o = r.opt
    return dict(gamma_correct=bool(o.gamma_correct), use_radiance_linear=bool(o.use_radiance_linear),
                lut_coefficient="F0" if o.lut_coefficient_f0 else "F", correct_depth=bool(o.correct_depth_for_prefiltered_radiance))


def _draws(r, n, perturb, pytest, chunk):
    """(t_rand [n, N_samples], u [n, N_importance]) of perturb > 0, or (None, None): torch's generator on the device, or — pytest — numpy's
    seed-0 stream re-seeded per chunk as batchify_rays / render_rays / sample_pdf do (ibl_nerf_renderer.py:686-690, nerf_renderer_helper.py:106-113)."""
    torch = _torch()
    from .renderer import _dev_f32, _pytest_uniform
    if not perturb or float(perturb) <= 0.:
        return None, None
    Sc, Ni = r.N_samples, max(r.N_importance, 1)
    if pytest:
        ch = int(chunk or n or 1)
        t = torch.cat([_pytest_uniform(min(ch, n - i), Sc) for i in range(0, n, ch)] or [torch.zeros((0, Sc))])
        u = torch.cat([_pytest_uniform(min(ch, n - i), Ni) for i in range(0, n, ch)] or [torch.zeros((0, Ni))])
        return _dev_f32(t, r.device), _dev_f32(u, r.device)
    return torch.rand((n, Sc), device=r.device), torch.rand((n, Ni), device=r.device)


class _Stages:
    """Thin callers of the stage entry points (include/iblnerf.h: iblnerf_coarse_z ...), device tensors in and out."""

    def __init__(self, r):
        self.r, self.lib, self.ctx = r, r.lib, r.ctx

    def _e(self, *sh):
        torch = _torch()
        return torch.empty(sh, dtype=torch.float32, device=self.r.device)

    def coarse_z(self, near, far, t_rand, n):
        """near / far: floats, or one plane per ray ([n] tensors: render_decomp's [n, 1] near / far, ibl_nerf_renderer.py:802-805)"""
        torch = _torch()
        z = self._e(n, self.r.N_samples)
        tr = None if t_rand is None else t_rand.data_ptr()
        if torch.is_tensor(near) or torch.is_tensor(far):
            from .renderer import _dev_f32
            nr, fr = (_dev_f32(v, self.r.device).reshape(-1).contiguous() if torch.is_tensor(v) else torch.full((n,), float(v), dtype=torch.float32, device=self.r.device)
                      for v in (near, far))
            if nr.numel() != n or fr.numel() != n:
                raise RuntimeError("near / far planes must have one entry per ray (%d), got %s" % (n, [int(nr.numel()), int(fr.numel())]))
            B.check(self.ctx, self.lib.iblnerf_coarse_z_rays(self.ctx, self.r._stream(), nr.data_ptr(), fr.data_ptr(), tr, n, z.data_ptr()))
            self._keep = (nr, fr)
        else:
            B.check(self.ctx, self.lib.iblnerf_coarse_z(self.ctx, self.r._stream(), float(near), float(far), tr, n, z.data_ptr()))
        return z

    def points(self, ro, rd, z):
        n, S = z.shape
        pts = self._e(n, S, 3)
        B.check(self.ctx, self.lib.iblnerf_sample_points(self.ctx, self.r._stream(), ro.data_ptr(), rd.data_ptr(), z.data_ptr(), n, S, pts.data_ptr()))
        return pts

    def fine_z(self, zc, wc, u):
        n = zc.shape[0]
        zf, zs = self._e(n, self.r.N_samples + self.r.N_importance), self._e(n)
        B.check(self.ctx, self.lib.iblnerf_fine_z(self.ctx, self.r._stream(), zc.data_ptr(), wc.data_ptr(), n, None if u is None else u.data_ptr(), zf.data_ptr(), zs.data_ptr()))
        return zf, zs

    def composite_sigma(self, sigma, z, rd):
        n, S = z.shape
        w, d, v = self._e(n, S), self._e(n), self._e(n)
        B.check(self.ctx, self.lib.iblnerf_composite_sigma(self.ctx, self.r._stream(), sigma.data_ptr(), z.data_ptr(), rd.data_ptr(), n, S, w.data_ptr(), d.data_ptr(), v.data_ptr()))
        return w, d, v


def render_rays_depth_only(r, rays_o, rays_d, near, far, perturb=0., pytest=False, chunk=None, raw_noise_std=0.):
    """is_depth_only (raw2outputs_depth, ibl_nerf_renderer.py:118-152, through render_rays :693-718): trunk-only queries, the keys
    depth_map / weights / visibility (+ '0') and z_std.  Forward only (train.py:374 detaches the one map it reads)."""
    torch = _torch()
    from .renderer import _dev_f32
    ro, rd = _dev_f32(rays_o, r.device), _dev_f32(rays_d, r.device)
    n = ro.shape[0]
    st = _Stages(r)
    t_rand, u = _draws(r, n, perturb, pytest, chunk)
    noise = r.noise_rows(n, raw_noise_std, False, chunk) if raw_noise_std > 0. else (None, None)       # raw2outputs_depth (:131-133): torch.randn, no pytest hook there
    zc = st.coarse_z(near, far, t_rand, n)
    sig = r.network_query(st.points(ro, rd, zc), None, 0)[..., 0].contiguous()
    wc, dc, vc = st.composite_sigma(sig if noise[0] is None else (sig + noise[0]).contiguous(), zc, rd)
    if r.N_importance <= 0:
        return {"depth_map": dc, "weights": wc, "visibility": vc}
    zf, zstd = st.fine_z(zc, wc, u)
    sig = r.network_query(st.points(ro, rd, zf), None, 1 if r.has_fine else 0)[..., 0].contiguous()      # run_fn = network_fn if network_fine is None (:705)
    wf, df, vf = st.composite_sigma(sig if noise[1] is None else (sig + noise[1]).contiguous(), zf, rd)
    return {"depth_map": df, "weights": wf, "visibility": vf, "depth_map0": dc, "weights0": wc, "visibility0": vc, "z_std": zstd}


def _aux_names(r):
    """the auxiliary networks loaded on the context, as raw2outputs consults them"""
    return [k for k in ("albedo_mlp", "roughness_mlp", "irradiance_mlp", "normal_mlp") if r._aux.get(k) is not None]


def _aux_columns(r, raw, pts):
    """raw rows with the albedo / roughness / irradiance columns replaced by the auxiliary networks' outputs (:291-303), as the render path's workspace holds them"""
    names = [k for k in _aux_names(r) if k in AUX_COLS]
    if not names:
        return raw
    if "irradiance_mlp" in names and r.opt.use_radiance_linear:
        raise NotImplementedError("an irradiance_mlp under use_radiance_linear outside the inference render: its samples take a sigmoid where the compositing stage "
                                  "applies radiance_f (ibl_nerf_renderer.py:300-303)")
    raw = raw.clone()
    for k in names:
        raw[..., AUX_COLS[k]] = r.aux_query(k, pts)
    return raw


def _inferred_normal(r, pts, weights, ro, rd, target_depth):
    """inferred_normal_map (:266-275) and what its backward needs: normal_mlp at every sample, composited with the detached weights — or, infer_normal_at_surface,
    once per ray at x_surface = rays_o + rays_d * target_depth_map (detached, :262-263).  -> (map [n, 3], query points, d map / d raw as a factor [.., 3] of the upstream)"""
    torch = _torch()
    if r.opt.infer_normal_at_surface:
        xs = (ro + rd * target_depth.detach()[:, None]).contiguous()
        s_ = torch.sigmoid(r.aux_query("normal_mlp", xs))                       # [n, 3]
        return 2 * s_ - 1, xs, 2 * s_ * (1 - s_)
    s_ = torch.sigmoid(r.aux_query("normal_mlp", pts))                          # [n, S, 3]
    return torch.sum(weights[..., None] * (2 * s_ - 1), -2), pts, weights[..., None] * (2 * s_ * (1 - s_))


BASE_KEYS = ["radiance_map", "radiance_map_1", "radiance_map_2", "radiance_map_3", "irradiance_map", "albedo_map", "roughness_map", "disp_map",
             "acc_map", "depth_map", "target_depth_map", "weights"]          # raw2outputs' non-None entries without approximate_radiance, in its order (:494-525)


def _with_noise(raw, noise):
    """raw rows whose density column carries the pass's noise (raw[..., 0] + noise, ibl_nerf_renderer.py:242): what the compositing reads; the noise is a
    constant of the step, so dL/d raw is unchanged by it"""
    if noise is None:
        return raw
    out = raw.clone()
    out[..., 0] += noise
    return out


def _forward_direct(r, st, ro, rd, near, far, t_rand, u, flags, noise=(None, None), gt_const=None, rows=None):
    """render_rays with approximate_radiance=False from its stages: (result dict, what a backward needs).  gt_const: the target maps of the *_from_gt flags that are
    on (raw2outputs substitutes them whatever approximate_radiance is, :251-252, :320-330); rows: override_rows(approximate_radiance=False) — the depth overrides,
    the only ones outside `if approximate_radiance` (:253-256)."""
    torch = _torch()
    n = ro.shape[0]
    zc = st.coarse_z(near, far, t_rand, n)
    pc = st.points(ro, rd, zc)
    rawc = _with_noise(_aux_columns(r, r.network_query(pc, rd, 0), pc), noise[0])
    mc, wc = r.composite_direct(rawc, zc, rd)
    zf, zstd = st.fine_z(zc, wc, u)
    pf = st.points(ro, rd, zf)
    rawf = _with_noise(_aux_columns(r, r.network_query(pf, rd, 1 if r.has_fine else 0), pf), noise[1])
    mf, wf = r.composite_direct(rawf, zf, rd)
    res = {}
    normal_on = "normal_mlp" in _aux_names(r)
    for sfx, m, w, p in (("", mf, wf, pf), ("0", mc, wc, pc)):
        m_eff, gt_eff = _apply_overrides(m, gt_const, rows)
        o = _ray_outputs(m_eff, None, flags, gt_eff)
        o["weights"] = w
        res.update({k + sfx: o[k] for k in BASE_KEYS})
        if normal_on:
            res["inferred_normal_map" + sfx] = _inferred_normal(r, p, w, ro, rd, o["target_depth_map"])[0]
    res["z_std"] = zstd       # (no synchronisation: every launch is on torch's current stream, whose allocator reuses freed blocks in stream order)
    return res, dict(zc=zc, zf=zf, rawc=rawc, rawf=rawf)


def _gt_constants(r, n, gt_values, from_gt):
    """{"albedo" [n, 3], "roughness" [n], "irradiance" [n, 3], "depth" [n]} of the *_from_gt flags that are on (:251-252, :320-330)"""
    from .renderer import _dev_f32
    gt_const, gv = {}, gt_values or {}
    for flag, key, ch in (("calculate_albedo_from_gt", "albedo", 3), ("calculate_roughness_from_gt", "roughness", 1),
                          ("calculate_irradiance_from_gt", "irradiance", 3), ("depth_map_from_ground_truth", "depth", 1)):
        if (from_gt or {}).get(flag):
            t = _dev_f32(gv[key], r.device).reshape(n, -1)
            gt_const[key] = (t[:, :3] if ch == 3 else t[:, 0]).contiguous()      # gt_values["roughness"][..., 0] (:326), gt_values["depth"][..., 0] (:252)
    return gt_const


def render_rays_direct(r, rays_o, rays_d, near, far, perturb=0., pytest=False, chunk=None, raw_noise_std=0., gt_values=None, from_gt=None, edit=None):
    """approximate_radiance=False without autograd (e.g. a validation render during the warm-up iterations): the reference's result dict."""
    from .renderer import _dev_f32
    torch = _torch()
    ro, rd = _dev_f32(rays_o, r.device), _dev_f32(rays_d, r.device)
    if r.N_importance <= 0:
        raise NotImplementedError("approximate_radiance=False is built for N_importance > 0 (every shipped config)")
    t_rand, u = _draws(r, ro.shape[0], perturb, pytest, chunk)
    noise = r.noise_rows(ro.shape[0], raw_noise_std, pytest, chunk) if raw_noise_std > 0. else (None, None)
    n = ro.shape[0]
    with torch.no_grad():
        res, _ = _forward_direct(r, _Stages(r), ro, rd, near, far, t_rand, u, _flags(r), noise, _gt_constants(r, n, gt_values, from_gt),
                                 override_rows(r, n, gt_values, edit, False, chunk))
    return res


def render_rays_train(r, rays_o, rays_d, near, far, net_c, net_f, lut, *, approximate_radiance, perturb=0., pytest=False, chunk=None, teacher_maps=None,
                      raw_noise_std=0., gt_values=None, from_gt=None, edit=None, aux_nets=None, incident_gradient=False):
    """render_rays + raw2outputs for a training step: the reference's result dict whose tensors carry a grad_fn into the parameters of
    `net_c` (network_fn) and `net_f` (network_fine).  `r`: the Renderer holding both networks' current weights (renderer_for).
    incident_gradient (use_gradient_for_incident_radiance, ibl_nerf_renderer.py:442-453): the reflected-ray query carries a gradient — dL/d(the four reflected-ray maps)
    from the shading backward goes through raw2outputs_simple (every map on the live weights, :38-66) into the pass's own network at the reflected rays' points
    (x_surface and the reflected direction are detached / no-grad quantities: nothing but the network's parameters receives it).
    aux_nets: {'albedo_mlp' | 'roughness_mlp' | 'irradiance_mlp' | 'normal_mlp': module} — the auxiliary networks loaded on `r` (ibl_nerf.py:305-323 registers
    them with the optimizer): their outputs replace the main network's albedo / roughness / irradiance columns in both passes (the main network gets no gradient
    there), normal_mlp feeds inferred_normal_map; a module with trainable parameters receives its gradients (Renderer.aux_backward), summed over the passes.
    teacher_maps (parity tests; the backward's counterpart of iblnerf_composite_pass): {n_dot_v_map[0], reflected_radiance_map[0],
    reflected_coarse_radiance_map_k[0]} taken as the shading backward's constants instead of this forward's own — the reflected-ray maps are
    ill-conditioned in the reference itself, and d color / d roughness is proportional to them."""
    torch = _torch()
    from .renderer import RESULT_ORDER, Renderer, _dev_f32
    ro, rd = _dev_f32(rays_o, r.device), _dev_f32(rays_d, r.device)
    n = ro.shape[0]
    if r.N_importance <= 0 or net_f is None:
        raise NotImplementedError("a training step on the fused path needs N_importance > 0 and a network_fine (every shipped config)")
    if not r.coarse_outputs:
        raise NotImplementedError("a training step reads the coarse pass's maps: coarse_outputs=True")
    flags = _flags(r)
    named = [dict(net.named_parameters()) for net in (net_c, net_f)]
    # smaller architectures run inside the built one (checkpoint.embed_architecture at upload): their gradients are the sub-blocks their parameters were written to
    try:
        archs = [ck.arch_of(nm) for nm in named]
    except (KeyError, ValueError):
        archs = [None, None]
    pnames = []
    for nm, arch in zip(named, archs):
        want = None if arch is None else [n + t for n, _, _ in ck.arch_schema(*arch) for t in (".weight", ".bias")]
        if want is None or set(nm) != set(want) or not (ck.is_member_of_built(arch) or ck.is_generic_arch(arch)):
            raise NotImplementedError("the backward is built for the IBLNeRF architecture (46 parameters per network at netdepth 8): fused for netdepth <= 8 and != 5, netwidth <= 256, "
                                      "multires <= 10, multires_views <= 4, layer by layer for larger networks (netdepth <= 32, even netwidth <= 4096, multires, multires_views <= 24)")
        # (a network outside the built shape: its forward on the layer-by-layer render path, its gradients from 8-bit checkpoints of a second forward, layers.network_gradients)
        pnames.append([k for k in ALL_PARAMS if k in nm] if ck.is_member_of_built(arch) else want)
    params = [nm[k] for nm, ks in zip(named, pnames) for k in ks]
    ci = bool(r.opt.color_independent_to_direction)      # (the context's streams carry the identity in place of the unused layers: iblnerf_network_backward)
    frozen = [bool(getattr(net, "freeze_radiance", False)) for net in (net_c, net_f)]
    frozen_rough = [bool(getattr(net, "freeze_roughness", False)) for net in (net_c, net_f)]
    st = _Stages(r)
    if torch.is_tensor(near) or torch.is_tensor(far):      # per-ray planes: a mip-level depth_0 per ray (:455-457)
        as_t = lambda v: _dev_f32(v, r.device).reshape(-1) if torch.is_tensor(v) else torch.full((n,), float(v), dtype=torch.float32, device=r.device)
        depth0 = ((as_t(far) + as_t(near)) * 0.5).contiguous()
    else:
        depth0 = 0.5 * (float(near) + float(far))
    lut_t = _dev_f32(lut, r.device)
    # calculate_*_from_gt / depth_map_from_ground_truth (render kwargs of a step; :251-252, :320-330): the forward substitutes the target maps (pass A), the backward
    # takes them as constants — no gradient reaches the network's own map through the shading or through the output of the same name
    from_gt = {k: True for k, v in (from_gt or {}).items() if v}
    gt_const = _gt_constants(r, n, gt_values, from_gt)
    # edit / insert overrides (:218-256, :378-410): masked rows of the target maps become constants of the step — substituted into the linear maps the backward
    # differentiates at, their dL/d(entries) zeroed (override_rows); the forward applies them in pass A as the inference path does
    edit = {k: v for k, v in (edit or {}).items() if k not in from_gt}
    rows = override_rows(r, n, gt_values, edit, approximate_radiance, chunk)

    aux = _aux_names(r)
    normal_on = "normal_mlp" in aux
    aux_named = {}
    for name in aux:
        mod = (aux_nets or {}).get(name)
        nm = dict(mod.named_parameters()) if hasattr(mod, "named_parameters") else {}
        if nm and any(p_.requires_grad for p_ in nm.values()):
            shapes = {k: tuple(v.shape) for k, v in nm.items()}
            if set(nm) != set(AUX_PARAMS) or shapes.get("positions_linears.0.weight") != (256, 63) or any(shapes["positions_linears.%d.weight" % l][0] != 256 for l in range(8)):
                # (load_aux embeds SMALLER PositionMLPs for rendering; their gradients would come back in the built shape and have no unembed — refuse by name, not with a
                # size mismatch deep inside the backward)
                raise NotImplementedError("a TRAINABLE auxiliary network's backward is built for PositionMLP(D=8, W=256, multires=10) (networks/MLP.py:6-30): positions_linears.0-7 "
                                          "[256, ...], out_linears — got %s: %s; freeze it (requires_grad_(False)) to render with it, or train it at the built shape"
                                          % (name, {k: v for k, v in sorted(shapes.items())[:3]}))
            aux_named[name] = nm
    if "normal_mlp" in aux_named and r.normal_mode == "inferred_normal_map":
        raise NotImplementedError("a trainable normal_mlp as the target normal (target_normal_map_for_radiance_calculation='inferred_normal_map') in a gradient-carrying "
                                  "render: the shading's n.v would carry a gradient, and the fused shading backward holds it constant")
    if "irradiance_mlp" in aux and r.opt.use_radiance_linear:
        raise NotImplementedError("an irradiance_mlp under use_radiance_linear in a gradient-carrying render (its samples take a sigmoid, ibl_nerf_renderer.py:300-303)")
    aux_params = [aux_named[name][k] for name in aux_named for k in AUX_PARAMS]
    order = list(RESULT_ORDER if approximate_radiance else BASE_KEYS)
    if normal_on:      # results["inferred_normal_map"] sits before target_normal_map / disp_map (:517-518)
        i_n = 16 if approximate_radiance else order.index("disp_map")
        order = order[:i_n] + ["inferred_normal_map"] + order[i_n:]
    keys = [k + s for s in ("", "0") for k in order] + ["z_std"]

    again = [nm[k] for nm, ks, arch in zip(named, pnames, archs) if not ck.is_member_of_built(arch) for k in ks]      # parameters that the backward pass reads once more
    versions = lambda: [0 if p_.is_inference() else p_._version for p_ in again]      # noqa: E731

    class _Fn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, ro_, rd_, *ps):
            t_rand, u = _draws(r, n, perturb, pytest, chunk)
            # raw_noise_std > 0 (train.py's option; :208-216, :242): the step's density noise, drawn once and shared by forward and backward
            noise = r.noise_rows(n, raw_noise_std, pytest, chunk) if raw_noise_std > 0. else (None, None)
            Sc, Sf = r.N_samples, r.N_samples + r.N_importance
            if approximate_radiance:
                taps = B.Taps()
                sv = dict(zc=st._e(n, Sc), zf=st._e(n, Sf), rawc=st._e(n, Sc, 18), rawf=st._e(n, Sf, 18), envc=st._e(n, 4, 3), envf=st._e(n, 4, 3))
                taps.d_z_coarse, taps.d_z_fine, taps.d_raw_coarse, taps.d_raw_fine = (sv[k].data_ptr() for k in ("zc", "zf", "rawc", "rawf"))
                taps.d_env_coarse, taps.d_env_fine = sv["envc"].data_ptr(), sv["envf"].data_ptr()    # the linear reflected-ray maps, exact (no gamma round trip)
                r._training_route(ro_, rd_, near, far)      # (Renderer.training_lists: the step's forward under a route — estimates + lists — or, off, every sample)
                res = r.render_rays(ro_, rd_, near, far, gt_values if (from_gt or rows) else None, draws=(t_rand, u), taps=taps, raw_noise_std=raw_noise_std,
                                    noise=None if noise[0] is None else noise, chunk=chunk, **from_gt, **(edit if rows else {}))
                sv["rawc"], sv["rawf"] = _with_noise(sv["rawc"], noise[0]), _with_noise(sv["rawf"], noise[1])     # (the taps are the network's rows: the noise is added in pass A)
            else:
                res, sv = _forward_direct(r, st, ro_, rd_, near, far, t_rand, u, flags, noise, gt_const, rows)
            ctx.saved = dict(sv, ro=ro_, rd=rd_)
            ctx.versions = versions()
            if normal_on or (incident_gradient and approximate_radiance):
                ctx.saved.update(tdepth=res["target_depth_map"].detach().clone(), tdepth0=res["target_depth_map0"].detach().clone())
            if incident_gradient and approximate_radiance:
                tm = {k: _dev_f32(v, r.device).reshape(res[k].shape) for k, v in (teacher_maps or {}).items() if k.startswith(("target_normal_map", "target_depth_map"))}
                ctx.saved.update(tnormal=tm.get("target_normal_map", res["target_normal_map"]).detach().clone(),
                                 tnormal0=tm.get("target_normal_map0", res["target_normal_map0"]).detach().clone())
                if "target_depth_map" in tm:      # (parity tests: the reflected rays' origin and direction as the reference had them — x_surface :262, the normal :358-361)
                    ctx.saved.update(tdepth=tm["target_depth_map"].clone(), tdepth0=tm["target_depth_map0"].clone())
            if approximate_radiance:
                src = dict(res, **{k: _dev_f32(v, r.device).reshape(res[k].shape) for k, v in (teacher_maps or {}).items() if k in res})
                for sfx, tap in (("", "envf"), ("0", "envc")):
                    if teacher_maps:                                 # parity tests: the reference's own (gamma-corrected) maps, inverted
                        env = torch.stack([_ungamma(src[k + sfx], flags["gamma_correct"]) for k in
                                           ("reflected_radiance_map", "reflected_coarse_radiance_map_1", "reflected_coarse_radiance_map_2", "reflected_coarse_radiance_map_3")], 1)
                        if flags["use_radiance_linear"]:
                            env = env / (1 - env)                    # inverse of tonemap_reinherd
                    else:
                        env = sv[tap]
                    ctx.saved["consts" + sfx] = dict(n_dot_v=src["n_dot_v_map" + sfx].clone(), env=env, lut=lut_t, depth0=depth0)   # (a copy: the map itself goes to the caller)
            outs = tuple(res[k] for k in keys)
            const_maps = tuple({"albedo": "albedo_map", "roughness": "roughness_map", "irradiance": "irradiance_map", "depth": "target_depth_map"}[k] for k in gt_const)
            ctx.mark_non_differentiable(*[res[k] for k in keys if k.startswith(("target_normal_map", "n_dot_v_map", "reflected_", "z_std") + const_maps)])
            return outs

        @staticmethod
        def backward(ctx, *gouts):
            sv = ctx.saved
            gout = dict(zip(keys, gouts))
            if ctx.versions != versions():
                # (layer by layer the backward pass evaluates the network on the module's parameters as they are now: gradients at other weights than the render's)
                raise RuntimeError("a parameter of a network outside the built shape was modified in place between this render and its backward pass")
            grads_all, oks = [], []
            aux_grads = {name: None for name in aux_named}

            def aux_add(name, g):
                if getattr(r, "last_backward_ok", None) is not None:
                    oks.append(r.last_backward_ok)
                aux_grads[name] = g if aux_grads[name] is None else {k: aux_grads[name][k] + g[k] for k in g}

            r.last_backward_ok = None
            for which, sfx, z, raw in ((0, "0", sv["zc"], sv["rawc"]), (1, "", sv["zf"], sv["rawf"])):
                lin, w_pass = r.composite_direct(raw, z, sv["rd"], want_weights="normal_mlp" in aux_named)
                lin, gt_eff = _apply_overrides(lin, gt_const, rows)
                consts = sv.get("consts" + sfx)
                if FUSED_SHADING_BACKWARD:                           # one launch (iblnerf_ray_outputs_backward) instead of ~160 ray-sized ones
                    ups = {k: gout.get(k + sfx) for k in SHADED_KEYS if (consts is not None or k in BASE_KEYS)}
                    for name in ("albedo", "roughness", "irradiance"):          # (an output map that IS the ground truth carries no gradient; the irradiance one is [n, 3] then)
                        if name in gt_const:
                            ups.pop(name + "_map", None)
                    denv = None
                    if incident_gradient and consts is not None:
                        dx, denv = r.ray_outputs_backward(lin, ups, consts["n_dot_v"], consts["env"], depth0, gt=gt_eff or None, want_denv=True)
                    else:
                        dx = r.ray_outputs_backward(lin, ups, None if consts is None else consts["n_dot_v"], None if consts is None else consts["env"],
                                                    depth0, gt=gt_eff or None)
                else:                                                # the same by torch autograd (the tests' reference for the kernel above)
                    with torch.enable_grad():
                        x = lin.detach().requires_grad_(True)
                        outs = _ray_outputs(x, consts, flags, gt_eff)
                        pairs = [(outs[k], gout[k + sfx]) for k in outs if gout.get(k + sfx) is not None and outs[k].requires_grad]     # (a *_from_gt output is a constant)
                        if pairs:
                            (dx,) = torch.autograd.grad([o for o, _ in pairs], x, [g.reshape(o.shape).to(o.dtype) for o, g in pairs], allow_unused=True)
                            dx = torch.zeros_like(lin) if dx is None else dx
                        else:
                            dx = torch.zeros_like(lin)
                dx = _zero_overridden(dx, gt_const, rows)
                gw = gout.get("weights" + sfx)
                draw = r.composite_direct_backward(raw, z, sv["rd"], dx.contiguous(), None if gw is None else gw.contiguous())
                if frozen[which]:                                     # forward_freezed: sigma, radiance and the coarse radiances are computed under no_grad
                    draw[..., 0] = 0
                    draw[..., 6:] = 0
                    if frozen_rough[which]:
                        draw[..., 4] = 0
                pts = st.points(sv["ro"], sv["rd"], z)
                for name in aux:      # the auxiliary networks' columns (:291-303): their gradient goes to them, none of it to the main network
                    if name in AUX_COLS:
                        if name in aux_named:
                            aux_add(name, r.aux_backward(name, pts, draw[..., AUX_COLS[name]].contiguous()))
                        draw[..., AUX_COLS[name]] = 0
                gn = gout.get("inferred_normal_map" + sfx)
                if "normal_mlp" in aux_named and gn is not None:
                    _, qpts, fac = _inferred_normal(r, pts, w_pass, sv["ro"], sv["rd"], sv["tdepth" + sfx])
                    gn = gn.reshape(n, 3)
                    aux_add("normal_mlp", r.aux_backward("normal_mlp", qpts, (gn * fac) if fac.dim() == 2 else (gn[:, None, :] * fac)))
                r.last_backward_ok = None
                layered = None
                if not ck.is_member_of_built(archs[which]):
                    from . import layers
                    layered = lambda p, d, u, net=(net_c, net_f)[which]: (None, layers.network_gradients(p, d, u, net))      # noqa: E731
                _, grads = network_backward_live(r, pts, sv["rd"], draw, which, layered)
                if incident_gradient and consts is not None and not frozen[which]:      # (forward_freezed computes sigma and every radiance under no_grad: nothing to carry)
                    # the reflected ray of this pass (:438-440): x_surface + reflected_dir * z_vals_constant (the coarse grid, jitter included, :694), queried on the
                    # pass's own network (:451); raw2outputs_simple composites radiance and the three coarse radiances on the live weights
                    if not FUSED_SHADING_BACKWARD:
                        raise NotImplementedError("use_gradient_for_incident_radiance needs the fused shading backward (dL/d env)")
                    if getattr(r, "last_backward_ok", None) is not None:
                        oks.append(r.last_backward_ok)
                    nrm, xs = sv["tnormal" + sfx], (sv["ro"] + sv["rd"] * sv["tdepth" + sfx][:, None]).contiguous()
                    rdir = (sv["rd"] - 2 * torch.sum(nrm * sv["rd"], -1, keepdim=True) * nrm).contiguous()
                    rpts = st.points(xs, rdir, sv["zc"])
                    rraw = r.network_query(rpts, rdir, which)
                    dm = torch.zeros((n, 19), dtype=torch.float32, device=r.device)
                    dm[:, 7:19] = denv.reshape(n, 12)
                    rdraw = r.composite_direct_backward(rraw, sv["zc"], rdir, dm, None, full=True)
                    r.last_backward_ok = None
                    _, g2 = (layered or (lambda p, d, u: r.network_backward(p, d, u, which)))(rpts, rdir, rdraw)
                    grads = {k: grads[k] + g2[k] for k in grads}
                if getattr(r, "last_backward_ok", None) is not None:
                    oks.append(r.last_backward_ok)
                if archs[which] != ck.SHIPPED_ARCH and layered is None:
                    grads = ck.unembed_gradients(grads, archs[which])
                for k in pnames[which]:
                    gk = grads[k]
                    if frozen[which] and not (k.startswith(UNFROZEN) and not (frozen_rough[which] and k.startswith("roughness_linear."))):
                        gk = None                                        # h is computed under no_grad: nothing reaches the trunk / view layers
                    if ci and k.startswith(("feature_linear.", "views_linears.")):
                        gk = None                                        # is_color_independent_to_direction (ibl_nerf.py:192): unused parameters, no gradient
                    grads_all.append(gk)
            for name in aux_named:
                for k in AUX_PARAMS:
                    grads_all.append(None if aux_grads[name] is None else aux_grads[name][k])
            if r.range_check == "lazy" and len(oks) >= 2:
                # one decision for the step: an overflow in any network's backward skips EVERY network's gradients (the range flag is sticky on
                # the device until the next call settles it, so a later call's view already includes an earlier overflow; this also zeroes the
                # first network's gradients when only a later one overflowed)
                both = torch.stack([o.reshape(()) for o in oks]).all()
                skip = ~both
                # (the per-parameter gradients are views of a few blobs — one per backward call: the blobs are zeroed in place, one launch each instead of one per tensor)
                bases = {}
                for gk in grads_all:
                    if gk is not None:
                        base = gk._base if gk._base is not None else gk
                        bases[base.data_ptr()] = base
                for base in bases.values():
                    base.masked_fill_(skip, 0.0)
            out = []
            for i, (p, gk) in enumerate(zip(params + aux_params, grads_all)):
                # (views of the call's own gradient blob, a fresh tensor per network_backward: no copy — 92 launches less per step)
                out.append(gk.reshape(p.shape).to(p.device) if (gk is not None and ctx.needs_input_grad[2 + i]) else None)
            return (None, None) + tuple(out)

    outs = _Fn.apply(ro, rd, *params, *aux_params)
    from . import layers
    layers.sign(next((o for o in outs if o.requires_grad), outs[0]))
    return dict(zip(keys, outs))
