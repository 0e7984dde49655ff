"""Calls of the 8-bit operators that only some sizes, streams or modes reach, on the GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import lowbit_ref as R
from test_gpu_lowbit import DTYPES, check_linear, f32, leaf, lb, make, near, np64, rows, same

pytestmark = pytest.mark.gpu


def raw_frame(cache, capacity, planes, aabb, pts, t):
    """gs4d_frame_features with a cache that says it has `capacity` rows; the call reads the first len(pts) of them."""
    n, ch = pts.shape[0], planes[0].shape[1]
    d = type(cache._desc).from_buffer_copy(cache._desc)
    d.capacity = capacity
    out = torch.empty(n, cache.width, device="cuda")
    rc = pkg("_cabi").lib().gs4d_frame_features(
        C.addressof(d), len(planes) // 3, ch, (C.c_void_p * len(planes))(*[p.data_ptr() for p in planes]),
        (C.c_int * len(planes))(*[p.shape[3] for p in planes]), (C.c_int * len(planes))(*[p.shape[2] for p in planes]),
        aabb.data_ptr(), pts.data_ptr(), t.data_ptr(), 0 if t.numel() == 1 else 1, n, out.data_ptr(), cache.width,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


@pytest.mark.parametrize("n,ch", [(9, 4), (8200, 256)])               # the general kernel, and lines blended first
def test_frame_features_of_a_cache_of_more_than_32_bits_of_rows(n, ch):
    g = torch.Generator().manual_seed(n)
    c = lb().RowCache(n, ch)
    c.write((0.1 + torch.rand(n, ch, generator=g)).cuda())
    planes = [(0.5 + torch.rand(1, 5, 7, ch, generator=g)).permute(0, 3, 1, 2).cuda() for _ in range(3)]
    aabb = torch.tensor([[1.3, 1.2, 1.1], [-1.3, -1.2, -1.0]]).cuda()
    pts, t = (torch.rand(n, 3, generator=g) * 2 - 1).cuda(), torch.tensor([0.25], device="cuda")
    want = lb().frame_features(c, planes, aabb, pts, t)
    assert len(want.unique(dim=0)) > 5
    for capacity in (n, 2 ** 31 + 5, 2 ** 32, 2 ** 32 + 5):
        assert torch.equal(raw_frame(c, capacity, planes, aabb, pts, t), want), capacity


def test_a_write_on_another_stream_outlives_its_cache_object():
    """The caller keeps codes and scales; the helper array of many scattered rows goes with the object, but not before the write."""
    codes, scales = torch.zeros(5000, 64, dtype=torch.uint8, device="cuda"), torch.zeros(5000, 1, device="cuda")
    x = rows(3000, 64).cuda()
    slots = torch.randint(0, 5000, (3000,), generator=torch.Generator().manual_seed(1)).cuda()
    want = f32(R.write(np.zeros((5000, 64)), np64(x), slots.tolist(), "int8", 64))
    c = lb().RowCache.from_buffers(codes, scales, 64)
    c.write(torch.zeros_like(x), slots)                               # the helper array comes from this stream
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        c.write(x, slots)
    del c
    others = [torch.full((5000,), 2 ** 30, dtype=torch.int32, device="cuda") for _ in range(16)]       # who may have the memory now
    torch.cuda.synchronize()
    same(lb().RowCache.from_buffers(codes, scales, 64).read(), want)
    assert all((o == 2 ** 30).all().item() for o in others)


@pytest.mark.parametrize("needs_grad", [False, True])
def test_linear_refuses_operands_with_tangents(needs_grad):
    from torch.autograd import forward_ad
    x, w, b = (t.cuda().requires_grad_(needs_grad) for t in make(6, 8, 4, torch.float32)[:3])
    y = lb().linear(x, w, b)
    with forward_ad.dual_level():
        for i in range(3):
            args = [x, w, b]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                lb().linear(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                lb().linear(*args)
        assert torch.equal(lb().linear(x, w, b), y)                   # without a tangent: as ever


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
def test_linear_under_autocast(low):
    x, w, b, dy = make(70, 40, 20, torch.float32)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    cast = [t.detach().to(low).requires_grad_(True) for t in (xs, ws, bs)]
    y0 = lb().linear(*cast, relu=True)
    want = torch.autograd.grad(y0, cast, dy.cuda().to(low))
    with torch.autocast("cuda", low):
        for args in ((cast[0], ws, bs), (xs, cast[1], bs), (xs, cast[1], cast[2]), (cast[0], cast[1], bs)):
            y = lb().linear(*args, relu=True)
            assert y.dtype is low and torch.equal(y, y0)
            got = torch.autograd.grad(y, args, dy.cuda().to(low))
            assert all(g.dtype is a.dtype and torch.equal(g.to(low), v) for g, a, v in zip(got, args, want))
        assert lb().linear(xs, ws, bs).dtype is torch.float32         # one type: as it is
        for bad in ((xs.double(), ws, bs), (xs, ws.double(), bs), (xs, ws, bs.double())):
            with pytest.raises(RuntimeError):
                lb().linear(*bad)
    for args in ((cast[0], ws, bs), (xs, ws, cast[2])):
        with pytest.raises(RuntimeError):
            lb().linear(*args)


@pytest.mark.parametrize("levels,ch,res,res_t,n", [(1, 4, 1, 1, 524_289), (2, 128, 1, 5, 16_385), (1, 256, 1, 1, 8200), (1, 64, 5000, 3, 32_769),
                                                   (4, 4, 6000, 2, 524_300), (1, 32, 2500, 4, 65_540)])
def test_frame_features_of_axes_of_one_and_of_lines_that_do_not_fit(levels, ch, res, res_t, n):
    """Enough points for blended lines: axes of one texel, lines that leave few channels at once, and lines too long for any."""
    g = torch.Generator().manual_seed(n)
    static = 0.1 + torch.rand(n, levels * ch, generator=g) * 2
    c = lb().RowCache(n, levels * ch, "int8", 64)
    c.write(static.cuda())
    planes = [(0.5 + torch.rand(1, res_t, res, ch, generator=g)).permute(0, 3, 1, 2) for _ in range(3 * levels)]
    aabb = torch.tensor([[1.3, 1.2, 1.1], [-1.3, -1.2, -1.0]])
    pts = (torch.rand(n, 3, generator=g) * 2 - 1) * 1.6
    args = [p.cuda() for p in planes], aabb.cuda(), pts.cuda()
    at = torch.cat([torch.arange(300), torch.arange(n - 300, n), torch.randint(0, n, (400,), generator=g)])
    held = R.quantise(np64(static[at]), "int8", 64)[0]
    # a coordinate of at most 4 in units of the axis is off by 8 roundings; a plane of values in [0.5, 1.5] turns an error of d texels
    # into at most 2 d relative, three planes, two coordinates each; 20 roundings in the products
    tol = (12 * 8 * 4 * max(res, res_t) + 20) * 2.0 ** -24
    for t in (torch.tensor([0.3721]), torch.tensor([-2.0])):
        got = lb().frame_features(c, *args, t.cuda())
        want = R.frame_features(held, [p[0].numpy() for p in planes], aabb.numpy(), pts[at].numpy(), t.expand(len(at)).numpy())
        assert np.abs(np64(got.cpu()[at]) / want - 1).max() <= tol
        each = lb().frame_features(c, *args, t.expand(n).contiguous().cuda())
        assert (got / each - 1).abs().max().item() <= 2 * tol


@pytest.mark.parametrize("n", [1, 7, 8, 9, 23, 24, 25, 64])
@pytest.mark.parametrize("k,m", [(70, 16_500), (16_500, 70), (2100, 2000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_few_rows_and_a_large_weight(n, k, m, dtype):
    """On both sides of what the large dimension leaves to the kernels for few rows."""
    check_linear(*make(n, k, m, dtype), True, "int8")


def test_few_rows_of_a_large_weight_take_no_longer_than_many():
    """200 rows of 8192 -> 8192 against 512 of them: the time of the kernels for few rows grows with the rows (they took four times
    as long; a factor of two leaves room for clocks)."""
    w = torch.randn(8192, 8192, device="cuda")

    def time(n):
        x = torch.randn(n, 8192, device="cuda")
        with torch.no_grad():
            for _ in range(2):
                lb().linear(x, w)
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                lb().linear(x, w)
            b.record()
            torch.cuda.synchronize()
        return a.elapsed_time(b)
    assert time(200) <= 2 * time(512)
