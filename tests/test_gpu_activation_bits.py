"""The field's activations in 8 bits (activation_bits = 8): what happens between a forward and its backward."""
import pytest
import torch

from conftest import pkg
from test_gpu_lowbit_field import field, inputs, rel

pytestmark = pytest.mark.gpu
NAMES = ("points", "scales", "rotations", "opacity", "shs")


@pytest.mark.parametrize("before,after", [(256, 1024), (1024, 256), (700, 256)])
def test_the_backward_reads_the_checkpoint_where_its_forward_put_it(before, after, monkeypatch):
    D, net = pkg("scene.deformation"), field(8, 2)
    x, t, f, ws = inputs(900)

    def run(rows_forward, rows_backward):
        leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
        net.zero_grad(set_to_none=True)
        monkeypatch.setattr(D, "CHECKPOINT_ROWS", rows_forward)
        out = net.forward_dynamic(*(leaves[k] for k in NAMES), t, f, None)
        monkeypatch.setattr(D, "CHECKPOINT_ROWS", rows_backward)
        sum((o * w).sum() for o, w in zip(out, ws)).backward()
        return {k: v.grad for k, v in leaves.items()}, {n: p.grad.clone() for n, p in net.named_parameters() if p.grad is not None}
    want, got = run(before, before), run(before, after)
    for k in ("scales", "rotations", "shs"):
        assert torch.equal(want[0][k], got[0][k]), k
    assert rel(got[0]["points"], want[0]["points"]) <= 1e-5
    for n in want[1]:
        assert rel(got[1][n], want[1][n]) <= 1e-4, n


def both(kw, P, x=None, depth=2, t=None, f=None):
    """The same step with activations in 32 and in 8 bits -> two (outputs, input gradients, parameter gradients)."""
    res = []
    inp, t0, f0, ws = inputs(P)
    t, f = t0 if t is None else t, f0 if f is None else f
    for bits in (32, 8):
        net = field(bits, depth, **kw)
        leaves = {k: v.clone().requires_grad_(True) for k, v in (x or inp).items()}
        out = net.forward_dynamic(*(leaves[k] for k in NAMES), t, f, None)
        loss = sum((o * w).sum() for o, w in zip(out, ws))
        loss.backward(retain_graph=True)
        loss.backward()                                               # the checkpoint is read twice: gradients double
        res.append(([o.detach() for o in out], {k: v.grad for k, v in leaves.items()},
                    {n: p.grad for n, p in net.named_parameters() if p.grad is not None}))
    return res


def alike(res):
    (o32, i32, p32), (o8, i8, p8) = res
    assert all(torch.equal(a, b) for a, b in zip(o32, o8))
    for k in i32:
        assert (i32[k] is None) == (i8[k] is None), k
        if i32[k] is not None:
            assert torch.equal(i32[k], i8[k]) if k != "points" else rel(i8[k], i32[k]) <= 1e-5, k
    assert p32.keys() == p8.keys()
    for n in p32:
        # a weight gradient is sum_r dy_r x_r with x_r off by e_r, |e_r| <= max / 254 in each of at most 64 columns of a group, whose own
        # norm is at least max: |e_r| <= 8 / 254 |x_r|, and the signs of dy (of random weights on the outputs) are those of no x or e
        tol = 1e-4 if "grid" in n or "force_time" in n else 1e-5 if n.endswith("bias") else 8 / 254
        assert rel(p8[n], p32[n]) <= tol or float(p32[n].norm()) == 0 == float(p8[n].norm()), (n, rel(p8[n], p32[n]))


@pytest.mark.parametrize("kw", [dict(no_dx=True), dict(no_ds=True, no_dr=True, no_dshs=True), dict(no_dr=True), dict(no_dshs=True, apply_rotation=False),
                                dict(use_time=False, use_force=True), dict(use_force=True), dict(posebase_pe=10, scale_rotation_pe=5, no_ds=True)])
@pytest.mark.parametrize("depth", [0, 3])
def test_heads_that_are_off_and_a_backward_twice(kw, depth, monkeypatch):
    monkeypatch.setattr(pkg("scene.deformation"), "CHECKPOINT_ROWS", 256)
    alike(both(kw, 700, depth=depth))


def test_no_rows_and_strided_inputs():
    alike(both({}, 0))
    x, _, _, _ = inputs(300)
    wide = torch.randn(300, 9).cuda()
    wide[:, 2:5] = x["points"]
    odd = {**x, "points": wide[:, 2:5], "rotations": x["rotations"].t().contiguous().t()}
    alike(both({}, 300, x=odd, t=torch.tensor([[0.3]]).cuda().expand(300, 1), f=torch.rand(300, 2).cuda()[:, 1:]))


def test_a_captured_step_repeats():
    """Forward and backward with 8-bit activations in a graph, replayed with other points between eager steps."""
    x, t, f, ws = inputs(600)
    net = field(8, 2)

    def step(leaves):
        out = net.forward_dynamic(*(leaves[k] for k in NAMES), t, f, None)
        loss = sum((o * w).sum() for o, w in zip(out, ws))
        need = [leaves[k] for k in NAMES] + [net.deformation_net.pos_deform[1].weight, net.deformation_net.shs_deform[3].weight]
        return [o.detach() for o in out[:3]], torch.autograd.grad(loss, need)
    def fresh():
        return {k: v.detach().requires_grad_(True) for k, v in x.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, grads = step(fresh())
    for k in range(3):
        g = torch.Generator().manual_seed(50 + k)
        x["points"].copy_(torch.rand(600, 3, generator=g) * 3 - 1.5)
        x["scales"].copy_(torch.randn(600, 3, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want_o, want_g = step(fresh())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want_o))
        for a, b in zip(grads, want_g):
            assert rel(a, b) <= 1e-5
