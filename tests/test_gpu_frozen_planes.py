"""Frozen planes (freeze_planes) beside training, other streams, other cameras and many points."""
import copy

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import deformation_ref as R
from oracle import lowbit_ref as Q
from test_gpu_lowbit_field import field, inputs, step

pytestmark = pytest.mark.gpu
NAMES = ("points", "scales", "rotations", "opacity", "shs")


@pytest.mark.parametrize("fused", [True, False])
def test_an_optimizer_step_makes_frozen_planes_stale(fused):
    """backward, an evaluation that freezes, then the step: a frame must not mix the old spatial product with the new planes."""
    net = field(32)
    x, t, f, ws = inputs(300)
    args = [x[k] for k in NAMES]
    opt = (pkg("optim").FusedAdamW if fused else torch.optim.AdamW)(net.parameters(), lr=1e-2)
    step(net, x, t, f, ws)
    with torch.no_grad():
        net.freeze_planes(x["points"])
        net.forward_dynamic(*args, t, f, None)
        opt.step()
        with pytest.raises(RuntimeError, match="modified after freeze_planes"):
            net.forward_dynamic(*args, t, f, None)
        net.freeze_planes(x["points"])
        frozen = net.forward_dynamic(*args, t, f, None)
        net.thaw_planes()
        exact = net.forward_dynamic(*args, t, f, None)
    assert float((frozen[0] - exact[0]).abs().max()) <= 1e-2 * float(exact[0].abs().max())


def test_the_fused_optimizer_changes_versions():
    """As torch's does: a backward through parameters that were stepped since its forward is refused."""
    opt_mod = pkg("optim")
    a, b = (torch.nn.Parameter(torch.randn(8, 4, device="cuda")) for _ in range(2))
    opt = opt_mod.FusedAdamW([a, b], lr=1e-2)
    a.grad = torch.ones_like(a)
    va, vb = a._version, b._version
    opt.step()
    assert a._version > va and b._version == vb                       # b had no gradient
    net = field(32)
    x, t, f, ws = inputs(50)
    opt = opt_mod.FusedAdamW(net.parameters(), lr=1e-2)
    step(net, x, t, f, ws)
    out = net.forward_dynamic(*(x[k] for k in NAMES), t, f, None)
    opt.step()
    with pytest.raises(RuntimeError, match="modified in place"):
        out[0].sum().backward()


def test_frozen_frame_of_a_camera_with_a_time_per_row():
    """Which frames have one time is read off the columns themselves, not off the camera's class."""
    wl, rd = pkg("workload"), pkg("renderer")
    sc = wl.build_scene("C1", torch.device("cuda"), P=3000)
    net, pc, cam, bg = sc["deform"], sc["pc"], sc["cam"], sc["bg"]
    g = torch.Generator().manual_seed(0)
    times = torch.rand(3000, 1, generator=g).cuda()
    one = torch.full((3000, 1), cam.time, device="cuda"), torch.full((3000, 1), cam.force, device="cuda")

    class Rolling(type(cam)):
        def time_force_columns(self, n, device):
            return times, one[1]

    def frame(c, t, f):
        """(the frame, the same from a query of the field and a scene without one)"""
        q = net.forward_dynamic(pc._xyz, pc._scaling, pc._rotation, pc._opacity, pc._features, t, f, None)
        still = type("Still", (), dict(zip(("_xyz", "_scaling", "_rotation", "_opacity", "_features"), q), active_sh_degree=pc.active_sh_degree))
        return rd.render_for_image(c, pc, net, bg), rd.render_for_image(c, still, None, bg)
    rolling = copy.copy(cam)
    rolling.__class__ = Rolling
    with torch.no_grad():
        net.freeze_planes(pc._xyz)
        got, want = frame(rolling, times, one[1])
        assert torch.equal(got, want)
        plain, want1 = frame(cam, *one)
        assert torch.equal(plain, want1) and not torch.equal(plain, got)
        cam.time_force_columns(3000, pc._xyz.device)[0].copy_(times)  # the camera's own columns, written to
        assert torch.equal(rd.render_for_image(cam, pc, net, bg), want)
        cam._columns.clear()
    with torch.inference_mode():
        assert torch.equal(rd.render_for_image(cam, pc, net, bg), plain)
        t, f = cam.time_force_columns(3000, pc._xyz.device)
        assert not t.is_inference() and t.one_value_version == t._version


def test_frozen_frame_of_columns_made_in_inference_mode():
    """Tensors without a version are columns like any others."""
    wl, rd = pkg("workload"), pkg("renderer")
    sc = wl.build_scene("C1", torch.device("cuda"), P=500)
    net, pc, cam, bg = sc["deform"], sc["pc"], sc["cam"], sc["bg"]

    class Own(type(cam)):
        def time_force_columns(self, n, device):
            return torch.full((n, 1), self.time, device=device), torch.full((n, 1), self.force, device=device)
    own = copy.copy(cam)
    own.__class__ = Own
    with torch.inference_mode():
        net.freeze_planes(pc._xyz)
        assert torch.equal(rd.render_for_image(own, pc, net, bg), rd.render_for_image(cam, pc, net, bg))


def test_thawing_does_not_take_the_cache_from_a_frame_on_another_stream():
    net = field(32)
    x, t, f, ws = inputs(4000)
    args = [x[k] for k in NAMES]
    side = torch.cuda.Stream()
    with torch.no_grad():
        cache = net.freeze_planes(x["points"])
        sizes = [cache.codes.shape, cache.scales.shape]
        del cache
        want = [o.clone() for o in net.forward_dynamic(*args, t, f, None)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)                            # some 50 ms before the frame's turn
            got = net.forward_dynamic(*args, t, f, None)
    step(net, x, t, f, ws)                                            # thaws by itself
    assert "_frozen" not in net.deformation_net.__dict__
    others = [torch.full(s, 77, dtype=d, device="cuda") for s, d in zip(sizes, (torch.uint8, torch.float32)) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del others


def test_a_captured_frame_keeps_its_cache():
    net = field(32)
    x, t, f, ws = inputs(700)
    args = [x[k] for k in NAMES]
    with torch.no_grad():
        cache = net.freeze_planes(x["points"])
        sizes = [cache.codes.shape, cache.scales.shape]
        del cache
        want = [o.clone() for o in net.forward_dynamic(*args, t, f, None)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = net.forward_dynamic(*args, t, f, None)
    step(net, x, t, f, ws)
    others = [torch.full(s, 77, dtype=d, device="cuda") for s, d in zip(sizes, (torch.uint8, torch.float32)) for _ in range(8)]
    for _ in range(3):
        for o in (got[0], got[1], got[2], got[4]):                    # (the opacity is the caller's own tensor)
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        step(net, x, t, f, ws)
    assert copy.deepcopy(net).deformation_net.__dict__.get("_captured") is None
    del others


@pytest.mark.parametrize("channels,P,copies", [(32, 65_600, 1), (64, 32_800, 1), (16, 70_001, 2)])
@pytest.mark.parametrize("use_time,use_force", [(True, False), (True, True), (False, True), (False, False)])
def test_frozen_frames_of_so_many_points_that_lines_are_blended(channels, P, copies, use_time, use_force, monkeypatch):
    """One time and one force for all rows, of one view and of several, against the network on what the cache holds at some rows, and
    against the query with a time per row at all of them."""
    kw = dict(use_time=use_time, use_force=use_force)
    net = field(32, 1, channels, (1, 2), **kw)
    x, t, f, _ = inputs(P)
    many = [torch.cat([x[k]] * copies) for k in NAMES]
    n = P * copies
    with torch.no_grad():
        cache = net.freeze_planes(x["points"])
        one = net.forward_dynamic(*many, t[:1].expand(n, 1), f[:1].expand(n, 1), None)
        each = net.forward_dynamic(*many, t[:1].repeat(n, 1), f[:1].repeat(n, 1), None)
    at = torch.cat([torch.arange(400), torch.arange(n - 400, n), torch.randint(0, n, (700,), generator=torch.Generator().manual_seed(P))])
    held = cache.read(at.cuda() % P).cpu().double().numpy()
    sd = {k: v.detach().cpu().double() for k, v in net.state_dict().items()}
    cfg = R.DeformConfig(plane_channels=channels, resolution=[24, 20, 16, 9], multires=[1, 2], defor_depth=1, **kw)
    G = "deformation_net.grid."
    times = [sd[f"{G}grids.{lv}.{i}"][0].numpy() for lv in range(2) for i in (2, 4, 5)]
    monkeypatch.setattr(R, "hexplane_features", lambda sd_, cfg_, xyz, tp: torch.from_numpy(
        Q.frame_features(held, times, sd[G + "aabb"].numpy(), xyz.numpy(), tp[:, 0].numpy())))
    sub = [a.cpu()[at].double() for a in many]
    want = R.forward_dynamic(sd, cfg, *sub, torch.full((len(at), 1), float(t[0])).double(), torch.full((len(at), 1), float(f[0])).double())
    for k, (a, e, w) in enumerate(zip(one, each, want)):
        tol = 1e-5 * max(1.0, float(w.abs().max()))                   # the float32 path's forward tolerance
        if k == 2:                                                    # a rotation is divided by the norm of what the head gives
            tol *= 20
        assert float((a.cpu()[at].double() - w).abs().max()) <= tol, k
        assert float((a - e).abs().max()) <= 2 * tol, k
