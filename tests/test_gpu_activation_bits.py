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
