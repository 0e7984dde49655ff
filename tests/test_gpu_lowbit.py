"""8-bit rows on the GPU against their definition in 64 bits (oracle/lowbit_ref.py).

Tolerances.  What the cache holds is defined bit for bit: values are compared for equality (float32: the product s * code
rounded once; 16-bit reads: that number rounded again).  A sum of n products in float32, in any order and with operands held to
24 bits, is off by at most (n + 8) 2^-24 times the sum of the products' magnitudes; a result in a 16-bit type by half a step of
that type more."""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import lowbit_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FMTS = ["int8", "e4m3", "e5m2"]


def lb():
    return pkg("lowbit")


def rows(n, width, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    return x.to(dtype)


def np64(t):
    return t.detach().cpu().double().numpy()


def f32(values):
    return torch.from_numpy(values).float()


def same(got, want):
    """Equal numbers, NaN where NaN is wanted."""
    got = got.detach().cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("width", [1, 7, 8, 16, 64, 100, 257, 2100, 4104])
def test_write_and_read_in_order(fmt, group, width):
    for dtype in DTYPES:
        x = rows(37, width, dtype, seed=width)
        c = lb().RowCache(41, width, fmt, group)
        c.write(x.cuda(), start=3)
        want = np.zeros((41, width))
        want[3:40] = R.quantise(np64(x), fmt, group)[0]
        same(c.read(), f32(want))
        for dt in DTYPES:
            same(c.read(start=2, count=5, dtype=dt), f32(want[2:7]).to(dt))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 5000])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_scattered_rows_last_one_wins_and_padding(n, idx):
    cap = max(3, n // 2)                                              # many slots are named twice or more
    g = torch.Generator().manual_seed(n)
    slots = torch.randint(-2, cap + 2, (n,), generator=g)            # -2, -1, cap and cap + 1 are padding
    x = rows(n, 70, seed=n)
    c = lb().RowCache(cap, 70, "int8", 32)
    before = rows(cap, 70, seed=1)
    c.write(before.cuda())
    table = R.write(R.quantise(np64(before), "int8", 32)[0], np64(x), slots.tolist(), "int8", 32)
    for _ in range(3):                                                # again: the helper array is as it was
        c.write(x.cuda(), slots.to(idx).cuda())
        same(c.read(), f32(table))
    got = c.read(slots.to(idx).cuda())
    inside = (slots >= 0) & (slots < cap)
    want = torch.where(inside[:, None], f32(table)[slots.clamp(0, cap - 1)], torch.zeros(()))
    same(got, want)


def test_every_row_to_one_slot_and_far_slots():
    c = lb().RowCache(4, 16)
    x = rows(3000, 16)
    c.write(x.cuda(), torch.full((3000,), 2, dtype=torch.int64, device="cuda"))
    want = np.zeros((4, 16))
    want[2] = R.quantise(np64(x[-1:]), "int8", 64)[0]
    same(c.read(), f32(want))
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 2, 2], device="cuda")     # no slot is taken modulo 2^32
    c.write(x[:4].cuda(), far)
    want[2] = R.quantise(np64(x[3:4]), "int8", 64)[0]
    same(c.read(), f32(want))
    assert (c.read(far[:3]) == 0).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_groups_of_zeros_tiny_huge_and_nonfinite_numbers(fmt):
    x = rows(12, 128)
    x[0] = 0
    x[1, :64] = 0
    x[2] *= 1e-38                                                     # subnormal scale: stored as zero
    x[3] = 1e-45
    x[4] = x[4].sign() * 3.4e38
    x[5, 3], x[6, 70], x[7, 127] = float("inf"), float("-inf"), float("nan")
    x[8] = -x[8].abs()
    x[9] = torch.where(torch.arange(128) % 2 == 0, 1e-20, 1.0)
    x[10] = torch.finfo(torch.float32).min                            # the type's lowest number
    x[11, 5] = -0.0
    c = lb().RowCache(12, 128, fmt, 64)
    c.write(x.cuda())
    want = R.quantise(np64(x), fmt, 64)[0]
    got = c.read().cpu()
    same(got, f32(want))
    assert torch.isnan(got[5, :64]).all() and not torch.isnan(got[5, 64:]).any() and torch.isnan(got[7, 64:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_rows(dtype):
    base = rows(50, 200, dtype).cuda()
    flat = rows(1, 20 * 33 + 1, dtype).cuda().flatten()
    views = [base[:, 3:67], base[::2, :64], base.t()[:64], base[:1, 1:65].expand(9, 64), base[5:6, 8:72], base[:, 1::3][:, :64],
             flat[1:].view(20, 33), flat[1:1 + 64].view(1, 64)]
    for v in views:
        n, w = v.shape
        c = lb().RowCache(n, w)
        c.write(v)
        same(c.read(), f32(R.quantise(np64(v), "int8", 64)[0]))


def test_offsets_past_32_bits():
    cap = 17_000_000                                                  # 4.35 GB of codes
    c = lb().RowCache(cap, 256)
    x = rows(4, 256)
    slots = torch.tensor([cap - 1, 16_777_216, 16_777_215, 0], device="cuda")
    c.write(x.cuda(), slots)
    want = f32(R.quantise(np64(x), "int8", 64)[0])
    same(c.read(slots), want)
    same(c.read(start=cap - 1), want[:1])
    c.write(x[1:3].cuda(), start=cap - 2)
    same(c.read(start=cap - 2, count=2), want[1:3])


def test_zero_rows_and_refusals():
    c = lb().RowCache(8, 20)
    c.write(torch.zeros(0, 20, device="cuda"))
    assert c.read(torch.zeros(0, dtype=torch.int64, device="cuda")).shape == (0, 20)
    assert c.read(start=8).shape == (0, 20)
    x = torch.zeros(4, 20, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: c.write(x[:, :19]), lambda: c.write(x.double()), lambda: c.write(x.cpu()), lambda: c.write(x, start=5),
                 lambda: c.write(x, start=-1), lambda: c.write(x, slots[:3]), lambda: c.write(x, slots.float()),
                 lambda: c.write(x, slots.cpu()), lambda: c.write(x, slots.view(2, 2)), lambda: c.write(x, slots, start=1),
                 lambda: c.read(start=9), lambda: c.read(count=9), lambda: c.read(count=-1), lambda: c.read(dtype=torch.float64),
                 lambda: c.read(slots, count=3), lambda: c.read(slots.short())):
        with pytest.raises(RuntimeError):
            call()
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt, device="cuda")
    for codes, scales, width in ((z(4, 24), z(4, 1, dt=torch.float32), 20), (z(4, 16), z(4, 1, dt=torch.float32), 20),
                                 (z(4, 32), z(4, 2, dt=torch.float32), 20), (z(4, 32), z(4, 1, dt=torch.float64), 20),
                                 (z(4, 32, dt=torch.int8), z(4, 1, dt=torch.float32), 20), (z(4, 64)[:, ::2], z(4, 1, dt=torch.float32), 20)):
        with pytest.raises(RuntimeError):
            lb().RowCache.from_buffers(codes, scales, width)


def test_cache_calls_follow_the_current_stream_and_replay():
    c = lb().RowCache(600, 96, "e4m3", 32)
    x = rows(600, 96).cuda()
    slots = torch.arange(600, device="cuda").flip(0)
    want = f32(R.quantise(np64(x), "e4m3", 32)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            x2 = x * 2
            c.write(x2, slots)
        c.write(x, slots)
        got = c.read(slots)
    torch.cuda.current_stream().wait_stream(side)
    same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(x, slots)
        out = c.read(slots)
    for k in range(4):
        x.copy_(rows(600, 96, seed=10 + k))
        c.write(torch.zeros_like(x))                                  # the program's own eager work between replays
        graph.replay()
        torch.cuda.synchronize()
        same(out, f32(R.quantise(np64(x), "e4m3", 32)[0]))


def test_a_cache_captured_before_its_first_write():
    """The helper array of many scattered rows must not be one whose zeros only a replay writes."""
    c = lb().RowCache(500, 64)
    x = rows(1000, 64).cuda()
    slots = torch.randint(0, 500, (1000,), generator=torch.Generator().manual_seed(0)).cuda()
    want = f32(R.write(np.zeros((500, 64)), np64(x), slots.tolist(), "int8", 64))
    filler = torch.full((4096,), 2 ** 30, dtype=torch.int32, device="cuda")           # what uninitialised memory may hold
    del filler
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(x, slots)
    c.write(x, slots)                                                 # eager, before any replay
    same(c.read(), want)
    for _ in range(3):
        c.write(torch.zeros(500, 64, device="cuda"))
        graph.replay()
        same(c.read(), want)
        c.write(x, slots)
        same(c.read(), want)


def test_a_captured_write_outlives_its_cache_object():
    """The caller keeps codes and scales; the graph must not use an array that goes with the cache object."""
    codes, scales = torch.zeros(500, 64, dtype=torch.uint8, device="cuda"), torch.zeros(500, 1, device="cuda")
    x = rows(1000, 64).cuda()
    slots = torch.randint(0, 500, (1000,), generator=torch.Generator().manual_seed(1)).cuda()
    want = f32(R.write(np.zeros((500, 64)), np64(x), slots.tolist(), "int8", 64))
    c = lb().RowCache.from_buffers(codes, scales, 64)
    c.write(x, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(x, slots)
    torch.cuda.synchronize()
    del c
    others = [torch.full((500,), 2 ** 30, dtype=torch.int32, device="cuda") for _ in range(64)]       # who may have the memory now
    for _ in range(3):
        codes.zero_()
        graph.replay()
        same(lb().RowCache.from_buffers(codes, scales, 64).read(), want)
        assert all((o == 2 ** 30).all().item() for o in others)


@pytest.mark.parametrize("size", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [2, 63, 255, 256, 257, 511, 513])
def test_the_last_of_several_rows_for_one_slot(n, size):
    for capacity in (1, 5, n):
        x = rows(n, 40, seed=n)
        slots = torch.randint(-1, capacity + 1, (n,), generator=torch.Generator().manual_seed(n), dtype=size)
        c = lb().RowCache(capacity, 40, group=32)
        c.write(torch.zeros(capacity, 40, device="cuda"))
        for _ in range(2):
            c.write(x.cuda(), slots.cuda())
            same(c.read(), f32(R.write(np.zeros((capacity, 40)), np64(x), slots.tolist(), "int8", 32)))


# ------------------------------------------------------------------------------------------ frame features
@pytest.mark.parametrize("levels,ch,res,res_t,n", [(1, 4, 5, 2, 1), (2, 32, 9, 7, 300), (1, 16, 1, 1, 65), (4, 8, 6, 3, 77), (2, 128, 12, 5, 130),
                                                   (1, 256, 4, 4, 9)])
@pytest.mark.parametrize("fmt", FMTS)
def test_frame_features(levels, ch, res, res_t, n, fmt):
    g = torch.Generator().manual_seed(n)
    static = 0.1 + torch.rand(n + 2, levels * ch, generator=g) * 2
    c = lb().RowCache(n + 2, levels * ch, fmt, 32)
    c.write(static.cuda())
    held = R.quantise(np64(static), fmt, 32)[0][:n]
    planes = [(0.5 + torch.rand(1, res_t + lv, res + lv, ch, generator=g)).permute(0, 3, 1, 2) for lv in range(levels) for _ in range(3)]
    aabb = torch.tensor([[1.3, 1.2, 1.1], [-1.3, -1.2, -1.0]])
    pts = (torch.rand(n, 3, generator=g) * 2 - 1) * 1.6
    pts[0] = torch.tensor([1.3, -1.2, 5.0])                           # on and far beyond the border
    for t in (torch.rand(1, generator=g) * 2 - 1, torch.rand(n, generator=g) * 3 - 1.5, torch.tensor([-1.0])):
        got = lb().frame_features(c, [p.cuda() for p in planes], aabb.cuda(), pts.cuda(), t.cuda())
        want = R.frame_features(held, [p[0].numpy() for p in planes], aabb.numpy(), pts.numpy(), t.expand(n).numpy())
        # a coordinate of at most 4 in units of the axis is off by 8 roundings; a plane of values in [0.5, 1.5] turns an error
        # of d texels into at most 2 d relative, three planes, two coordinates each; 20 roundings in the products
        tol = (12 * 8 * 4 * max(res + levels, res_t + levels) + 20) * 2.0 ** -24
        assert np.abs(np64(got) / want - 1).max() <= tol
        again = lb().frame_features(c, [p.cuda().contiguous() for p in planes], aabb.cuda(), pts.cuda(), t.cuda())
        assert torch.equal(got, again)                                # planes of another memory format


@pytest.mark.parametrize("levels,ch,res,res_t,n", [(2, 32, 20, 7, 4099), (2, 128, 64, 5, 1031), (1, 256, 9, 3, 700), (3, 4, 5, 4, 20_000),
                                                   (4, 16, 30, 9, 5000), (1, 64, 900, 3, 2000), (1, 8, 4000, 2, 9000), (1, 4, 1, 1, 17_000)])
@pytest.mark.parametrize("fmt", FMTS)
def test_frame_features_of_many_points(levels, ch, res, res_t, n, fmt):
    """One t for enough points that the planes are blended to lines first; long axes among them."""
    g = torch.Generator().manual_seed(n)
    static = 0.1 + torch.rand(n, levels * ch, generator=g) * 2
    c = lb().RowCache(n, levels * ch, fmt, 128)
    c.write(static.cuda())
    held = R.quantise(np64(static), fmt, 128)[0]
    planes = [(0.5 + torch.rand(1, res_t, res << (lv % 2), ch, generator=g)).permute(0, 3, 1, 2) for lv in range(levels) for _ in range(3)]
    aabb = torch.tensor([[1.3, 1.2, 1.1], [-1.3, -1.2, -1.0]])
    pts = (torch.rand(n, 3, generator=g) * 2 - 1) * 1.6
    args = [p.cuda() for p in planes], aabb.cuda(), pts.cuda()
    for t in (torch.tensor([0.3721]), torch.tensor([1.0]), torch.tensor([-2.0])):
        got = lb().frame_features(c, *args, t.cuda())
        want = R.frame_features(held, [p[0].numpy() for p in planes], aabb.numpy(), pts.numpy(), t.expand(n).numpy())
        tol = (12 * 8 * 4 * max(2 * res, res_t) + 20) * 2.0 ** -24    # as above
        assert np.abs(np64(got) / want - 1).max() <= tol
        each = lb().frame_features(c, *args, t.expand(n).contiguous().cuda())
        assert np.abs(np64(each) / want - 1).max() <= tol             # a value per point: the other kernel


@pytest.mark.parametrize("levels,ch,res,res_t,n", [(2, 32, 64, 75, 65_537), (2, 128, 128, 25, 16_385), (1, 256, 9, 3, 8192),
                                                   (1, 256, 1500, 2, 8200), (3, 64, 300, 6, 32_771), (4, 16, 30, 9, 131_100), (1, 4, 3, 1, 524_289)])
@pytest.mark.parametrize("fmt", FMTS)
def test_frame_features_from_blended_lines(levels, ch, res, res_t, n, fmt):
    """A frame of so many points that the lines of its one t are blended first; against the kernel for a t per point and, at some
    points, the definition."""
    g = torch.Generator().manual_seed(n)
    static = 0.1 + torch.rand(n, levels * ch, generator=g) * 2
    c = lb().RowCache(n, levels * ch, fmt, 64)
    c.write(static.cuda())
    planes = [(0.5 + torch.rand(1, res_t, res << (lv % 2), ch, generator=g)).permute(0, 3, 1, 2) for lv in range(levels) for _ in range(3)]
    aabb = torch.tensor([[1.3, 1.2, 1.1], [-1.3, -1.2, -1.0]])
    pts = (torch.rand(n, 3, generator=g) * 2 - 1) * 1.6
    args = [p.cuda() for p in planes], aabb.cuda(), pts.cuda()
    at = torch.cat([torch.arange(600), torch.arange(n - 600, n), torch.randint(0, n, (800,), generator=g)])
    held = R.quantise(np64(static[at]), fmt, 64)[0]
    tol = (12 * 8 * 4 * max(2 * res, res_t) + 20) * 2.0 ** -24        # as above
    for t in (torch.tensor([0.3721]), torch.tensor([1.0]), torch.tensor([-2.0])):
        got = lb().frame_features(c, *args, t.cuda())
        want = R.frame_features(held, [p[0].numpy() for p in planes], aabb.numpy(), pts[at].numpy(), t.expand(len(at)).numpy())
        assert np.abs(np64(got.cpu()[at]) / want - 1).max() <= tol
        each = lb().frame_features(c, *args, t.expand(n).contiguous().cuda())
        assert (got / each - 1).abs().max().item() <= 2 * tol         # every point: two results within tol of one number


def test_frame_features_refuses():
    c = lb().RowCache(10, 16)
    z = lambda *s: torch.zeros(*s, device="cuda")
    p, box, pts, t = [z(1, 16, 3, 3)] * 3, z(2, 3), z(10, 3), z(1)
    assert lb().frame_features(c, p, box, z(0, 3), t).shape == (0, 16)
    for args in ((c, p[:2], box, pts, t), (c, p * 5, box, pts, t), (c, p * 2, box, pts, t), (c, [z(1, 8, 3, 3)] * 3, box, pts, t),
                 (c, p, box, z(11, 3), t), (c, p, box, z(10, 2), t), (c, p, z(3, 2), pts, t), (c, p, box, pts, z(3)), (c, p, box, pts.double(), t),
                 (c, p, box, pts.cpu(), t), (None, p, box, pts, t), (c, [z(1, 16, 3, 3).half()] * 3, box, pts, t)):
        with pytest.raises(RuntimeError):
            lb().frame_features(*args)


def test_frame_features_refuses_a_single_number_for_points():
    c = lb().RowCache(10, 16)
    z = lambda *s: torch.zeros(*s, device="cuda")
    with pytest.raises(RuntimeError, match="points"):
        lb().frame_features(c, [z(1, 16, 3, 3)] * 3, z(2, 3), z(1)[0], z(1))


# ------------------------------------------------------------------------------------------ linear
def leaf(t):
    return t.cuda().requires_grad_(True)


def make(n, k, m, dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * n + 3 * k + m)
    x = rows(n, k, dtype, seed=seed + n)
    w = (torch.randn(m, k, generator=g) / k ** 0.5).to(dtype)
    b = (0.1 * torch.randn(m, generator=g)).to(dtype) if bias else None
    dy = (1e-2 * torch.randn(n, m, generator=g)).to(dtype)
    return x, w, b, dy


def near(got, want, magnitude, terms):
    """magnitude: the sum of the products' magnitudes, elementwise."""
    got = got.detach()
    tol = (terms + 8) * 2.0 ** -24 * magnitude
    if got.dtype != torch.float32:
        tol = tol + np.abs(want) * torch.finfo(got.dtype).eps / 2 + float(torch.finfo(got.dtype).smallest_normal) * torch.finfo(got.dtype).eps
    err = np.abs(np64(got) - want)
    assert got.shape == want.shape and (err <= tol).all(), (float((err - tol).max()), float(err.max()))


def check_linear(x, w, b, dy, relu, fmt):
    xs, ws, bs = leaf(x), leaf(w), None if b is None else leaf(b)
    y = lb().linear(xs, ws, bs, relu=relu, fmt=fmt)
    grads = torch.autograd.grad(y, [xs, ws] + ([] if b is None else [bs]), dy.cuda())
    X, W, D = np64(x), np64(w), np64(dy)
    wy, wdx, wdw, wdb, kept = R.linear(X, W, None if b is None else np64(b), relu, fmt, D)
    near(y, wy, np.abs(np.maximum(X, 0) if relu else X) @ np.abs(W).T + (0 if b is None else np.abs(np64(b))), x.shape[1])
    near(grads[0], wdx, np.abs(D) @ np.abs(W), w.shape[0])
    near(grads[1], wdw, np.abs(D).T @ np.abs(kept), x.shape[0])
    if b is not None:
        near(grads[2], wdb, np.abs(D).sum(axis=0), x.shape[0])
    assert not (grads[0].cpu()[(x <= 0)] != 0).any() if relu else True
    with torch.no_grad():
        assert torch.equal(lb().linear(xs, ws, bs, relu=relu, fmt=fmt), y)       # nothing kept, the same numbers
    return y, grads


SHAPES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (3, 300, 1), (31, 64, 64), (33, 65, 63), (128, 64, 48), (129, 128, 64), (500, 31, 200),
          (1000, 333, 129), (2049, 64, 64), (7, 1000, 70), (70, 7, 1000)]


@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_step(n, k, m, dtype):
    for relu in (False, True):
        check_linear(*make(n, k, m, dtype, bias=relu), relu, "int8")


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_step_in_8_bit_floats(fmt, dtype):
    for relu in (False, True):
        check_linear(*make(700, 130, 70, dtype), relu, fmt)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_many_rows(dtype):
    check_linear(*make(70_001, 64, 64, dtype), True, "int8")


def test_linear_shapes_strides_and_partial_gradients():
    x, w, b, dy = make(24, 40, 20, torch.float32)
    y0 = lb().linear(x.cuda(), w.cuda(), b.cuda())
    wide = torch.randn(24, 90).cuda()
    wide[:, 5:45] = x.cuda()
    turned = x.cuda().t().contiguous().t()
    for v in (wide[:, 5:45], turned, x.cuda().view(2, 3, 4, 40)):
        assert torch.equal(lb().linear(v, w.cuda(), b.cuda()).reshape(24, 20), y0)
    assert lb().linear(x[0].cuda(), w.cuda(), b.cuda()).shape == (20,)
    one = leaf(x[:1])
    lb().linear(one.expand(24, 40), w.cuda(), relu=True).backward(dy.cuda())
    near(one.grad, R.linear(np64(x[:1].expand(24, 40)), np64(w), None, True, "int8", np64(dy))[1].sum(0, keepdims=True),
         (np.abs(np64(dy)) @ np.abs(np64(w))).sum(0, keepdims=True), 20 + 24)
    # an upstream gradient that is a broadcast view
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    lb().linear(xs, ws, bs, relu=True).sum().backward()
    want = R.linear(np64(x), np64(w), np64(b), True, "int8", np.ones((24, 20)))
    near(xs.grad, want[1], np.abs(np.ones((24, 20))) @ np.abs(np64(w)), 20)
    near(ws.grad, want[2], np.abs(want[4]).sum(0)[None].repeat(20, 0), 24)
    near(bs.grad, want[3], np.full(20, 24.0), 24)
    # only some of the three
    full = torch.autograd.grad(lb().linear(xs, ws, bs, relu=True), (xs, ws, bs), dy.cuda())
    for i, leaves in enumerate(((xs, w.cuda(), b.cuda()), (x.cuda(), ws, b.cuda()), (x.cuda(), w.cuda(), bs))):
        g, = torch.autograd.grad(lb().linear(*leaves, relu=True), leaves[i], dy.cuda())
        assert torch.equal(g, full[i])


def test_linear_keeps_nothing_without_gradients():
    x, w, b, _ = make(4096, 256, 64, torch.float32)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    sizes = []
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            y = lb().linear(xs, ws, bs, relu=True)
            sizes.append(torch.cuda.memory_allocated() - before - y.numel() * 4)
            del y
    # 256 codes, 4 scales and 32 bytes of signs a row (the allocator may add up to 1 MiB to a block), not 1024 bytes
    assert sizes[0] < 4096 and 4096 * 304 <= sizes[1] <= 4096 * 305 + (1 << 20), sizes


def test_linear_without_rows():
    xs, ws, bs = leaf(torch.zeros(0, 8)), leaf(torch.zeros(5, 8)), leaf(torch.zeros(5))
    y = lb().linear(xs, ws, bs, relu=True)
    assert y.shape == (0, 5)
    y.sum().backward()
    assert (ws.grad == 0).all() and (bs.grad == 0).all() and xs.grad.shape == (0, 8)


def test_linear_does_not_need_its_input_again():
    x, w, b, dy = make(300, 64, 64, torch.float32)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    want = torch.autograd.grad(lb().linear(xs, ws, bs, relu=True), (xs, ws, bs), dy.cuda())
    h = xs * 1.0
    y = lb().linear(h, ws, bs, relu=True)
    with torch.no_grad():
        h.fill_(float("nan"))                                         # the input may be overwritten
    got = torch.autograd.grad(y, (ws, bs), dy.cuda(), retain_graph=True)
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, (xs, ws, bs), dy.cuda()), want))     # twice the same
    y = lb().linear(xs, ws, bs)
    with torch.no_grad():
        ws.add_(1)                                                    # the weight may not
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, xs, dy.cuda())


def test_linear_nonfinite_numbers_stay_where_they_are():
    x, w, b, dy = make(130, 70, 40, torch.float32)
    x[5, 3], x[77, 66], x[100, 1] = float("-inf"), float("nan"), float("inf")
    xs, ws = leaf(x), leaf(w)
    y = lb().linear(xs, ws, relu=True)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy.cuda())
    fine = torch.ones(130, dtype=torch.bool)
    fine[77] = fine[100] = False
    assert torch.isfinite(y.cpu()[fine]).all()                        # relu(-inf) is 0
    assert torch.isnan(y.cpu()[77]).all() and not torch.isfinite(y.cpu()[100]).any()
    assert torch.isfinite(dx).all()
    want = np64(x.clone())
    want[[77, 100]] = 1
    near(y[fine.cuda()], R.linear(want, np64(w), None, True, "int8")[fine.numpy()], (np.maximum(np.nan_to_num(want, neginf=0), 0) @ np.abs(np64(w)).T)[fine.numpy()], 70)


def test_linear_gradients_against_differences():
    """y is linear in w and b and piecewise linear in x: differences are exact up to rounding, except that the weight gradient is
    taken with the kept values, each within half a step."""
    x, w, b, dy = make(200, 96, 33, torch.float32)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    dx, dw, db = (np64(t) for t in torch.autograd.grad(lb().linear(xs, ws, bs, relu=True), (xs, ws, bs), dy.cuda()))
    g = np.random.default_rng(0)
    f = lambda X, W, B: (R.linear(X, W, B, True, "int8") * np64(dy)).sum()
    X, W, B = np64(x), np64(w), np64(b)
    v = g.standard_normal(X.shape) * np.minimum(np.abs(X), 1)         # no sign changes at h = 1e-3
    h = 1e-3
    d = (f(X + h * v, W, B) - f(X - h * v, W, B)) / (2 * h)
    assert abs(d - (dx * v).sum()) <= 1e-5 * np.abs(dx * v).sum()
    u = g.standard_normal(W.shape)
    d = (f(X, W + h * u, B) - f(X, W - h * u, B)) / (2 * h)
    step = R.quantise(np.maximum(X, 0), "uint8", 64)[1]
    assert abs(d - (dw * u).sum()) <= (np.abs(np64(dy) @ u) * 0.5 * step).sum() + 1e-5 * np.abs(dw * u).sum()
    z = g.standard_normal(B.shape)
    d = (f(X, W, B + h * z) - f(X, W, B - h * z)) / (2 * h)
    assert abs(d - (db * z).sum()) <= 1e-5 * np.abs(db * z).sum()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_runs_are_equal_bit_for_bit(dtype):
    x, w, b, dy = make(30_000, 100, 72, dtype)
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    first = None
    for _ in range(3):
        y = lb().linear(xs, ws, bs, relu=True)
        out = (y.detach(), *torch.autograd.grad(y, (xs, ws, bs), dy.cuda()))
        first = first or out
        assert all(torch.equal(a, c) for a, c in zip(first, out))


def test_linear_step_replays_and_follows_the_stream():
    x, w, b, dy = make(3000, 64, 64, torch.float32)
    X, W, B, D = x.cuda(), w.cuda(), b.cuda(), dy.cuda()

    def step():
        xs, ws, bs = X.detach().requires_grad_(True), W.detach().requires_grad_(True), B.detach().requires_grad_(True)
        y = lb().linear(xs, ws, bs, relu=True)
        return (y.detach(), *torch.autograd.grad(y, (xs, ws, bs), D))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        aside = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(aside, step()))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for k in range(3):
        X.copy_(rows(3000, 64, seed=50 + k))
        for g, out in zip(graphs, outs):
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


@pytest.mark.parametrize("n,k,m,dtype", [(3000, 256, 300, torch.float32), (5000, 500, 70, torch.float16), (4000, 40, 600, torch.float32),
                                         (6, 33, 17, torch.bfloat16)])
def test_linear_replays_in_every_form(n, k, m, dtype):
    """Several groups, a wide result, few rows: captured, replayed with other numbers, against the eager call."""
    x, w, b, dy = make(n, k, m, dtype)
    X, W, B, D = x.cuda(), w.cuda(), b.cuda(), dy.cuda()

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (X, W, B)]
        y = lb().linear(*leaves, relu=True)
        return (y.detach(), *torch.autograd.grad(y, leaves, D))
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        X.copy_(rows(n, k, dtype, seed=90 + i))
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


@pytest.mark.parametrize("n,k,m", [(4, 64, 64), (5, 64, 64), (2048, 64, 64), (2049, 64, 64), (600, 512, 500), (1100, 512, 512), (3000, 7, 200),
                                   (2500, 9, 3), (2500, 1, 1), (2304, 100, 400), (2304, 576, 130)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_on_both_sides_of_every_rule(n, k, m, dtype):
    check_linear(*make(n, k, m, dtype), True, "int8")


@pytest.mark.parametrize("n,k,m", [(4096, 64, 64), (4097, 64, 64), (1524, 256, 256), (1525, 256, 256), (712, 256, 256), (713, 256, 256),
                                   (712, 512, 512), (713, 512, 512), (1224, 512, 512), (1225, 512, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_on_both_sides_of_the_rules_for_few_rows(n, k, m, dtype):
    check_linear(*make(n, k, m, dtype), True, "int8")


@pytest.mark.parametrize("n,k,m", [(4097, 333, 129), (5000, 128, 64), (4100, 320, 40), (3000, 70, 257), (8000, 384, 128), (16384, 65, 64),
                                   (16385, 65, 64), (4321, 600, 30), (2333, 77, 500), (6000, 130, 130)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_several_groups_and_few_tiles(n, k, m, dtype):
    """The waves of a workgroup share a tile of rows, each a part of the contraction; and the sizes next to that."""
    check_linear(*make(n, k, m, dtype), True, "int8")
    check_linear(*make(n, k, m, dtype, bias=False), False, "e4m3")


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_at_any_alignment(dtype):
    """Rows, weights and gradients whose first element is not on 16 bytes, pitches that are no multiple of anything."""
    for n, k, m in ((70, 48, 33), (2500, 72, 66), (2500, 61, 5)):
        x, w, b, dy = make(n, k, m, dtype)
        pool = torch.empty(n * (k + 3) + 5, dtype=dtype, device="cuda")
        xv = pool[1:1 + n * (k + 3)].view(n, k + 3)[:, 1:k + 1]
        xv.copy_(x)
        odd = lambda t: torch.cat([torch.zeros(1, dtype=dtype), t.flatten()]).cuda()[1:].view(t.shape)
        leaves = [xv.detach().requires_grad_(True), odd(w).requires_grad_(True), odd(b).requires_grad_(True)]
        y = lb().linear(*leaves, relu=True)
        grads = torch.autograd.grad(y, leaves, odd(dy))
        yy, gg = check_linear(x, w, b, dy, True, "int8")
        assert torch.equal(y, yy) and all(torch.equal(a, c) for a, c in zip(grads, gg))


def test_linear_refusals():
    x, w, b = (t.cuda() for t in make(4, 8, 6, torch.float32)[:3])
    for call in (lambda: lb().linear(x, w[:, :7]), lambda: lb().linear(x, w[0]), lambda: lb().linear(x.double(), w.double()),
                 lambda: lb().linear(x.half(), w), lambda: lb().linear(x, w, b[:5]), lambda: lb().linear(x, w, b.half()),
                 lambda: lb().linear(x, w, b, fmt="int4"), lambda: lb().linear(x, w.cpu()), lambda: lb().linear(x, w, b.cpu()),
                 lambda: lb().linear(x, w[:0]), lambda: lb().linear(x.sum(), w)):
        with pytest.raises(RuntimeError):
            call()
