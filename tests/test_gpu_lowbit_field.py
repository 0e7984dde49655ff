"""The deformation field with its 8-bit rows: activations kept in 8 bits for the backward (activation_bits = 8) and frames from
frozen planes (freeze_planes).

What is exact is compared for equality or with the tolerances of the float32 path (plane gradients: float atomics).  A weight
gradient is sum over rows of dy * x with x off by at most half a step of its group, so it is off by at most
sum |dy| * step / 2; its relative 2-norm error is checked against 1 / 127 (random signs make it far smaller)."""
import copy
import types

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import deformation_ref as R
from oracle import lowbit_ref as Q
from test_gpu_deformation import make_args

pytestmark = pytest.mark.gpu


def field(bits, depth=0, channels=32, multires=(1, 2), seed=0, **kw):
    cfg = R.DeformConfig(plane_channels=channels, resolution=[24, 20, 16, 9], multires=list(multires), defor_depth=depth, **kw)
    a = make_args(cfg)
    a.activation_bits = bits
    torch.manual_seed(seed)
    net = pkg("scene.deformation").deform_network(a)
    g = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():                                             # no zero-initialised heads: every gradient is alive
        for n, p in net.named_parameters():
            if "deform" in n:
                p.add_(0.05 * torch.randn(p.shape, generator=g))
    return net.cuda()


def inputs(P, seed=3):
    g = torch.Generator().manual_seed(seed)
    x = dict(points=torch.rand(P, 3, generator=g) * 3 - 1.5, scales=torch.randn(P, 3, generator=g) * 0.5 - 3,
             rotations=torch.randn(P, 4, generator=g), opacity=torch.randn(P, 1, generator=g), shs=torch.randn(P, 16, 3, generator=g) * 0.3)
    ws = [torch.randn(s, generator=g).cuda() for s in ((P, 3), (P, 3), (P, 4), (P, 1), (P, 16, 3))]
    return {k: v.cuda() for k, v in x.items()}, torch.full((P, 1), 0.61).cuda(), torch.full((P, 1), -0.3).cuda(), ws


def step(net, x, t, f, ws):
    leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
    net.zero_grad(set_to_none=True)
    out = net.forward_dynamic(*(leaves[k] for k in ("points", "scales", "rotations", "opacity", "shs")), t, f, None)
    sum((o * w).sum() for o, w in zip(out, ws)).backward()
    return [o.detach() for o in out], {k: v.grad for k, v in leaves.items()}, {n: p.grad for n, p in net.named_parameters() if p.grad is not None}


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


@pytest.mark.parametrize("P", [1, 31, 500, 3001])
@pytest.mark.parametrize("depth,channels,multires", [(0, 32, (1, 2)), (5, 16, (1, 2)), (2, 128, (1, 2)), (1, 4, (1, 2)), (3, 8, (1, 2, 4))])
def test_step_with_kept_activations(P, depth, channels, multires, monkeypatch):
    monkeypatch.setattr(pkg("scene.deformation"), "CHECKPOINT_ROWS", 1024)           # 3001 rows: three chunks
    a, b = field(32, depth, channels, multires), field(8, depth, channels, multires)
    x, t, f, ws = inputs(P)
    out32, in32, p32 = step(a, x, t, f, ws)
    out8, in8, p8 = step(b, x, t, f, ws)
    assert all(torch.equal(u, v) for u, v in zip(out32, out8))                       # the forward is the same
    for k in ("scales", "rotations", "opacity", "shs"):
        assert torch.equal(in32[k], in8[k]), k                                       # masks are exact
    assert rel(in8["points"], in32["points"]) <= 1e-5
    assert p32.keys() == p8.keys()
    for n in p32:
        if "grid" in n or "force_time" in n:
            assert rel(p8[n], p32[n]) <= 1e-4, n
        elif n.endswith("bias"):
            assert rel(p8[n], p32[n]) <= 1e-5, n
        else:
            assert rel(p8[n], p32[n]) <= 1 / 127, (n, rel(p8[n], p32[n]))
    again = step(b, x, t, f, ws)
    for n in p8:
        if "grid" not in n and "force_time" not in n:
            assert rel(again[2][n], p8[n]) <= 1e-6, n


@pytest.mark.parametrize("depth,channels,P", [(0, 32, 700), (3, 128, 65), (2, 4, 1)])
def test_checkpoint_holds_what_the_definition_says(depth, channels, P):
    """A forward's workspace (tprime | features | inner trunk layers | Z | H1 | O | sign words, each 256-byte aligned), packed and
    unpacked: the encodings and signs bit for bit, the rest as the 8-bit rows of the definition."""
    import ctypes as C
    D, net = pkg("scene.deformation"), field(8, depth, channels)
    L = D._lib()
    x, t, f, _ = inputs(P)
    _, cfg = net.deformation_net.cached_plan()
    d = cfg["plan"].desc
    d.no_grad = 0
    nb = int(L.gs4d_deform_workspace_bytes(C.byref(d), C.c_int(P)))
    ws, ws2 = (torch.full((nb,), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
    kept = torch.empty(int(L.gs4d_deform_checkpoint_bytes(C.byref(d), C.c_int(P))), dtype=torch.uint8, device="cuda")
    p, st = lambda v: C.c_void_p(v.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    out = [torch.empty_like(x[k]) for k in ("points", "scales", "rotations", "shs")]
    ins = [p(x["points"]), p(x["scales"]), p(x["rotations"])]
    assert L.gs4d_deform_forward(C.byref(d), C.c_int(P), *ins, p(x["shs"]), p(t), p(f), *(p(o) for o in out), p(ws), st) == 0
    assert L.gs4d_deform_checkpoint_pack(C.byref(d), C.c_int(P), p(ws), p(kept), st) == 0
    assert L.gs4d_deform_checkpoint_unpack(C.byref(d), C.c_int(P), *ins, p(t), p(f), p(kept), p(ws2), st) == 0
    F, n_trunk, a = 2 * channels, max(depth, 1), net.deformation_net.args
    pad8 = lambda v: (v + 7) // 8 * 8
    ldz = pad8(64 + pad8(6 * a.posebase_pe) + pad8(6 * a.scale_rotation_pe) + pad8(8 * a.scale_rotation_pe) + 2 + 2 * a.time_pe + 2 * a.force_pe)
    off, views = 0, []
    for words in [1, F] + [64] * (n_trunk - 1) + [ldz, 256, 72, 10]:
        views.append([w[off:off + 4 * P * words].view(torch.float32).view(P, words) for w in (ws, ws2)])
        off = (off + 4 * P * words + 255) // 256 * 256
    tp, feat, *trunk, Z, H1, O, hm = views
    same = lambda u, v: torch.equal(u.contiguous().view(torch.int32), v.contiguous().view(torch.int32))
    assert same(*tp) and same(O[0][:, 16:20], O[1][:, 16:20]) and same(*hm)
    assert same(Z[0][:, 64:], Z[1][:, 64:])
    n64 = lambda v: v.cpu().double().numpy()
    assert torch.equal(feat[1].cpu(), torch.from_numpy(Q.quantise(n64(feat[0]), "int8", 64)[0]).float())
    for old, new in trunk + [[Z[0][:, :64], Z[1][:, :64]], H1]:
        want = Q.quantise(np.maximum(n64(old), 0), "uint8", 64)[0].astype(np.float32)
        want = np.where(n64(old) > 0, np.maximum(want, np.float32(2.0 ** -126)), 0)   # a positive number stays positive
        assert torch.equal(new.cpu(), torch.from_numpy(want))
    assert L.gs4d_deform_checkpoint_pack(C.byref(d), C.c_int(P), p(ws[1:]), p(kept), st) == -1
    assert L.gs4d_deform_checkpoint_unpack(C.byref(d), C.c_int(P), *ins, p(t), None, p(kept), p(ws2), st) == -1
    d.no_grad = 1
    assert L.gs4d_deform_checkpoint_pack(C.byref(d), C.c_int(P), p(ws), p(kept), st) == -1
    d.no_grad = 0


def test_memory_per_row():
    L, net = pkg("_cabi").lib(), field(8)
    import ctypes as C
    D = pkg("scene.deformation")
    D._lib()
    _, cfg = net.deformation_net.cached_plan()
    d = cfg["plan"].desc
    ws, kept = (f(C.byref(d), C.c_int(100_000)) / 100_000 for f in (L.gs4d_deform_workspace_bytes, L.gs4d_deform_checkpoint_bytes))
    assert ws > 2000 and kept < 500, (ws, kept)
    # what a training query holds until its backward
    x, t, f, ws_ = inputs(60_000)
    held = {}
    for bits in (32, 8):
        n = field(bits)
        leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = n.forward_dynamic(*(leaves[k] for k in ("points", "scales", "rotations", "opacity", "shs")), t, f, None)
        held[bits] = (torch.cuda.memory_allocated() - before) / 60_000
        del out
    assert held[8] < 0.4 * held[32], held


def test_layered_heads_and_unsupported_bits():
    """A field whose encodings do not fit the fused heads keeps the signs through the values themselves."""
    kw = dict(posebase_pe=10, scale_rotation_pe=5)
    a, b = field(32, **kw), field(8, **kw)
    x, t, f, ws = inputs(900)
    out32, in32, p32 = step(a, x, t, f, ws)
    out8, in8, p8 = step(b, x, t, f, ws)
    assert all(torch.equal(u, v) for u, v in zip(out32, out8))
    for k in ("scales", "rotations", "shs"):
        assert torch.equal(in32[k], in8[k]), k
    for n in p32:
        assert rel(p8[n], p32[n]) <= 1 / 127, n
    with pytest.raises(NotImplementedError, match="activation_bits"):
        field(4).forward_dynamic(*(x[k] for k in ("points", "scales", "rotations", "opacity", "shs")), t, f, None)


def test_data_parallel_hook_sees_final_gradients(monkeypatch):
    monkeypatch.setattr(pkg("scene.deformation"), "CHECKPOINT_ROWS", 256)
    net = field(8, 2)
    x, t, f, ws = inputs(1000)
    want_in, want_p = step(net, x, t, f, ws)[1:]
    seen = {}
    net.deformation_net.data_grad_hook = lambda dp, ds, dr, planes, ftw, ftb: seen.update(points=dp.clone(), scales=ds.clone(), plane=planes[3].clone())
    got_p = step(net, x, t, f, ws)[2]
    assert rel(seen["points"], want_in["points"]) <= 1e-5 and torch.equal(seen["scales"], want_in["scales"])
    planes = [n for n in want_p if "grid.grids" in n]
    assert rel(seen["plane"], want_p[planes[3]]) <= 1e-4
    for n in want_p:
        assert rel(got_p[n], want_p[n]) <= 1e-4, n


# ------------------------------------------------------------------------------------------ frozen planes
@pytest.mark.parametrize("channels,multires,P", [(32, (1, 2), 3000), (128, (1, 2), 700), (4, (1, 2), 33), (16, (1, 2, 4, 8), 1), (64, (2,), 5000)])
@pytest.mark.parametrize("fmt,group", [("int8", 64), ("int8", 32), ("e4m3", 128)])
def test_frozen_planes_query(channels, multires, P, fmt, group, monkeypatch):
    """The cache holds the spatial product within half a step; a query then is the oracle's network on exactly those values (the
    float32 path's forward tolerance, 1e-5 of max(1, |x|); a rotation is divided by the norm of what the head gives, so there
    what float32 loses is measured on the query of six planes, whose roundings are the same kind and number)."""
    net = field(32, 2, channels, multires)
    x, t, f, _ = inputs(P)
    args = [x[k] for k in ("points", "scales", "rotations", "opacity", "shs")]
    sd = {k: v.detach().cpu().double() for k, v in net.state_dict().items()}
    cfg = R.DeformConfig(plane_channels=channels, resolution=[24, 20, 16, 9], multires=list(multires), defor_depth=2)
    with torch.no_grad():
        want6 = net.forward_dynamic(*args, t, f, None)
        cache = net.freeze_planes(x["points"], fmt, group)
        assert cache.capacity == P and cache.width == channels * len(multires)
        held = cache.read().cpu().double().numpy()
        each = net.forward_dynamic(*args, t, f, None)                                 # a time per row
        one = net.forward_dynamic(*args, t[:1].expand(P, 1), f[:1].expand(P, 1), None)     # one time
        mixed = torch.linspace(0, 1, 2 * P, device="cuda")[:, None]
        twice = net.forward_dynamic(*(torch.cat([a, a]) for a in args), mixed, torch.cat([f, f]), None)
        net.thaw_planes()
        back = net.forward_dynamic(*args, t, f, None)
    assert all(torch.equal(u, v) for u, v in zip(want6, back))
    # the cache against the planes
    G = "deformation_net.grid."
    box, pts = sd[G + "aabb"], x["points"].cpu().double()
    u = (pts - box[0]) * (2.0 / (box[1] - box[0])) - 1.0
    static = torch.cat([torch.stack([R.bilinear_border(sd[f"{G}grids.{lv}.{i}"], u[:, a], u[:, b]) for i, a, b in ((0, 0, 1), (1, 0, 2), (3, 1, 2))]).prod(0)
                        for lv in range(len(multires))], 1).numpy()
    step_ = Q.quantise(static, fmt, group)[1]
    # coordinates of at most 2 in float32, up to 192 texels an axis, values in [0.5, 1.5]: 6 coordinates, 8 roundings each
    assert (np.abs(held - static) <= 0.5 * step_ * (1 + 2 ** -10) + np.abs(static) * 6 * 8 * 2 * 192 * 2.0 ** -24).all()
    six = [float((g.cpu().double() - w).abs().max()) for g, w in zip(want6, R.forward_dynamic(sd, cfg, *(a.cpu().double() for a in args), t.cpu().double(), f.cpu().double()))]
    # the query against the network on what the cache holds
    times = [sd[f"{G}grids.{lv}.{i}"][0].numpy() for lv in range(len(multires)) for i in (2, 4, 5)]

    def expect(n, tt, ff):
        tile = lambda v: v.cpu().double().repeat(n, *[1] * (v.dim() - 1))
        monkeypatch.setattr(R, "hexplane_features", lambda sd_, cfg_, xyz, tp: torch.from_numpy(
            Q.frame_features(np.tile(held, (n, 1)), times, box.numpy(), xyz.numpy(), tp[:, 0].numpy())))
        return R.forward_dynamic(sd, cfg, *(tile(a) for a in args), tt.cpu().double(), ff.cpu().double())

    for got, want in ((each, expect(1, t, f)), (one, expect(1, t, f)), (twice, expect(2, mixed, torch.cat([f, f])))):
        for k, (g, w) in enumerate(zip(got, want)):
            err = float((g.cpu().double() - w).abs().max())
            assert err <= 1e-5 * max(1.0, float(w.abs().max())) + (2 * six[2] if k == 2 else 0), (k, err)


def test_frozen_planes_lifetime():
    net = field(32)
    x, t, f, ws = inputs(400)
    args = [x[k] for k in ("points", "scales", "rotations", "opacity", "shs")]
    q = lambda n=net: n.forward_dynamic(*args, t, f, None)
    dn = net.deformation_net
    for bad in (x["points"][:, :2], x["points"].cpu(), x["points"].double(), x["points"][:0]):
        with pytest.raises(RuntimeError):
            net.freeze_planes(bad)
    with torch.no_grad():
        net.freeze_planes(x["points"])
        with pytest.raises(RuntimeError, match="frozen planes"):                      # other points
            net.forward_dynamic(*(a[:399] for a in args), t[:399], f[:399], None)
        q()
        other = copy.deepcopy(net)                                                    # a copy is not frozen
        assert "_frozen" not in other.deformation_net.__dict__ and "_frozen" in dn.__dict__
        dn.grid.grids[0][0].mul_(1.01)
        with pytest.raises(RuntimeError, match="modified after freeze_planes"):
            q()
        net.freeze_planes(x["points"])
        q()
        net.deformation_net.set_aabb([1.3, 1.3, 1.3], [-1.3, -1.3, -1.3])
        net.cuda()
        assert "_frozen" not in dn.__dict__
        net.freeze_planes(x["points"])
    out32 = step(copy.deepcopy(net), x, t, f, ws)
    got = step(net, x, t, f, ws)                                                      # training thaws, and is unchanged
    assert "_frozen" not in dn.__dict__ and all(torch.equal(u, v) for u, v in zip(out32[0], got[0]))


def test_frames_and_training_of_one_scene_together():
    """As they would be used: train steps with kept activations, then frames from frozen planes, one view and several, the one-call
    path and the staged one."""
    wl, rd = pkg("workload"), pkg("renderer")
    sc = wl.build_scene("C1", torch.device("cuda"), P=3000)
    net, pc, cam, bg = sc["deform"], sc["pc"], sc["cam"], sc["bg"]
    dn = net.deformation_net
    ref = copy.deepcopy(net)
    dn.activation_bits = 8
    losses = []
    for n in (ref, net):
        pc.zero_grad(set_to_none=True)
        out = rd.render_with_l1(cam, pc, n, bg, sc["target"])
        out[0].backward()
        losses.append((out[0].detach(), out[1].detach(), pc._scaling.grad.clone()))
    assert torch.equal(losses[0][1], losses[1][1])                                    # the same image
    assert rel(losses[1][2], losses[0][2]) <= 1e-4
    for (n, p), (_, r) in zip(net.named_parameters(), ref.named_parameters()):
        assert (p.grad is None) == (r.grad is None), n
        if p.grad is not None and float(r.grad.norm()) > 0:
            assert rel(p.grad, r.grad) <= 1 / 127, (n, rel(p.grad, r.grad))
    loss, image, *_ = rd.render_l1_step(cam, pc, net, bg, sc["target"])
    assert torch.equal(image, losses[0][1])
    with torch.no_grad():
        exact = rd.render_for_image(cam, pc, net, bg)
        net.freeze_planes(pc._xyz)
        frozen = rd.render_for_image(cam, pc, net, bg)
        views = rd.render_batch([cam, cam], pc, net, bg)
        assert "_frozen" in dn.__dict__ and not torch.equal(frozen, exact)

        def by_stages(t, f):                                          # the field's query, then a scene without a field
            q = net.forward_dynamic(pc._xyz, pc._scaling, pc._rotation, pc._opacity, pc._features, t, f, None)
            still = types.SimpleNamespace(**dict(zip(("_xyz", "_scaling", "_rotation", "_opacity", "_features"), q)), active_sh_degree=pc.active_sh_degree)
            return rd.render_for_image(cam, still, None, bg)
        t, f = cam.time_force_columns(3000, pc._xyz.device)
        assert torch.equal(frozen, by_stages(t[:1].expand(3000, 1), f[:1].expand(3000, 1)))
        assert all(torch.equal(v[0], by_stages(t, f)) for v in views)                 # a time per row
    rd.render_l1_step(cam, pc, net, bg, sc["target"])
    assert "_frozen" not in dn.__dict__
