"""What the 8-bit operators compute where rounding, infinities or the order of a sum decide, on the GPU.

Tolerances count roundings of float32, 2^-24 of the sum of the products' magnitudes each.  A weight gradient is summed over at most
`steps` matrix instructions of 16 rows and one of three exact terms in a wave (17 roundings each), 3 joins of a workgroup's waves,
chunks / 8 + 8 sums of the chunks, and dy * scale is rounded once."""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import lowbit_ref as R
from test_gpu_lowbit import DTYPES, leaf, lb, np64, rows

pytestmark = pytest.mark.gpu


def weight_gradient_roundings(n, k, m):
    """The summation depth of linear's weight gradient: rows in about 256 chunks of at least 128, 8 / min(8, groups) waves each."""
    groups, tiles = -(-k // 64), -(-m // 64)
    gw = 8 if groups >= 8 else 4 if groups >= 4 else 2 if groups >= 2 else 1
    chunks = max(1, min(256 // (tiles * -(-groups // gw)), -(-n // 128)))
    per = -(-(-(-n // chunks)) // 128) * 128
    steps = -(-per // (16 * (8 // gw)))
    return 51 * steps + 1 + 3 + -(-chunks // 8) + 8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1023, 1025, 3001])
def test_weight_gradient_of_rows_that_cancel(n, dtype):
    """Every other row has a scale whose last eight bits are (nearly) ones and dy = 1, the rest the scale 1 and dy = -1, and the last
    row takes what is left: the sum is near 0, so what it loses of each product shows, whatever the type of the result."""
    tops = torch.arange(100, 160, 1 / 16).to(dtype).float().unique().numpy()
    tops = tops[(tops > 100) & ((tops / np.float32(127)).view(np.uint32) >> 15 & 1 > 0)]      # 16 bits end 8 above the last
    top = tops[np.argmax((tops / np.float32(127)).view(np.uint32) & 255)]
    scale = np.float32(top / np.float32(127))
    assert (scale.view(np.uint32) & 255) >= 0xe0
    codes = torch.arange(127, 63, -1) * 1.0                            # the first is the group's largest
    x = codes.repeat(n, 1)
    x[:-1:2] = (codes * float(scale)).to(dtype).float()
    x[:-1:2, 0] = float(top)
    x = x.to(dtype)
    dy = torch.ones(n, 64)
    dy[1::2] = -1
    dy[-1] = -float(len(dy[:-1:2]) * scale - len(dy[1::2]))
    dy = dy.to(dtype)
    kept = R.quantise(np64(x), "int8", 64)[0]
    assert (kept[0] == codes.double().numpy() * float(scale)).all() and (kept[1] == codes.double().numpy()).all()
    ws = leaf(torch.zeros(64, 64, dtype=dtype))
    dw, = torch.autograd.grad(lb().linear(x.cuda(), ws), ws, dy.cuda())
    want = np64(dy).T @ kept
    tol = weight_gradient_roundings(n, 64, 64) * 2.0 ** -24 * (np.abs(np64(dy)).T @ np.abs(kept)) + np.abs(want) * torch.finfo(dtype).eps / 2
    # with each product cut to 16 of its 24 bits the sum would be off by more than the tolerance
    lost = (len(dy[:-1:2]) * (float(scale) - float((scale.view(np.uint32) & np.uint32(0xffffff00)).view(np.float32)))) * codes.double().numpy()
    assert (lost > 1.2 * tol).all(), (lost / tol).min()
    assert (np.abs(np64(dw) - want) <= tol).all(), (np.abs(np64(dw) - want) / tol).max()
