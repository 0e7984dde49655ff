"""Frozen planes (freeze_planes) beside training, other streams, other cameras and many points."""
import copy

import numpy as np
import pytest
import torch

from conftest import pkg
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
