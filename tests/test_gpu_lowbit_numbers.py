"""What the 8-bit operators compute where rounding, infinities or the order of a sum decide, on the GPU.

Tolerances count roundings of float32, 2^-24 of the sum of the products' magnitudes each.  A weight gradient is summed over at most
`steps` matrix instructions of 16 rows and one of three exact terms in a wave (17 roundings each), 3 joins of a workgroup's waves,
chunks / 8 + 8 sums of the chunks, and dy * scale is rounded once."""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import lowbit_ref as R
from test_gpu_lowbit import DTYPES, leaf, lb, make, near, np64, rows

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


# (rows, contraction, features) of each way to walk the products over the rows: one group of columns and one block of features, with
# and without a multiple of 8 columns; several blocks; several groups with few and with many rows; a weight that does not fit LDS
WALKS = [(5000, 64, 64), (4100, 64, 20), (4500, 61, 64), (4500, 64, 200), (5000, 256, 64), (4300, 333, 129), (70_000, 128, 32), (70_000, 100, 64),
         (20_000, 450, 66), (20_000, 512, 66)]
LOW_NAN = 0x7f800001                                                  # a NaN whose upper half is an infinity's


def products(x, w):
    """sum_c x[r, c] w[f, c] as it is defined, infinities and NaNs among them, a few rows at a time."""
    with np.errstate(invalid="ignore"):
        return np.concatenate([(r[:, None, :] * w[None]).sum(-1) for r in np.array_split(x, max(1, len(x) // 64))])


def _plain(x, w):
    with torch.no_grad():
        return lb().linear(x.cuda(), w.cuda())


@np.errstate(invalid="ignore")
def magnitude(x, w):
    return np.abs(x) @ np.abs(w).T


def same_specials(got, want, most, terms):
    got = np64(got)
    assert (np.isnan(got) == np.isnan(want)).all()
    assert ((got == np.inf) == (want == np.inf)).all() and ((got == -np.inf) == (want == -np.inf)).all()
    f = np.isfinite(want)
    assert (np.abs(got[f] - want[f]) <= (terms + 8) * 2.0 ** -24 * most[f]).all()


def special_operands(n, c, f, seed):
    """A few rows and features with infinities and NaNs, weights of few significant bits and zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x, w = rows(n, c, seed=seed), torch.randn(f, c, generator=g)
    w[::3] = w[::3].bfloat16().float()
    w[1::3, ::2], w[1::3, 1::2] = 0.5, -1.0
    w[2, ::5] = 0
    at = torch.randperm(n, generator=g)[:40]
    col = torch.randint(0, c, (40,), generator=g)
    inf = float("inf")
    for i, v in enumerate([inf, -inf, float("nan"), 0.0, 0.0] * 8):
        x[at[i], col[i]] = v
    x[at[5:10], (col[5:10] + 7) % c] = inf                            # two in a row: the same or opposite ones
    x[at[10], :] = inf
    x[n - 1, c - 1] = -inf
    bits = x.view(torch.int32)
    bits[at[13], col[13]], bits[at[14], col[14]] = LOW_NAN, LOW_NAN - 2 ** 31
    hit = torch.zeros(n, dtype=torch.bool)
    hit[at] = hit[n - 1] = True
    return x, w, hit, torch.cat([at, torch.tensor([n - 1]), torch.randint(0, n, (60,), generator=g)])


@pytest.mark.parametrize("n,c,f", WALKS)
def test_infinities_and_nans_of_the_rows(n, c, f):
    x, w, hit, look = special_operands(n, c, f, n + c)
    X, W = np64(x), np64(w)
    for relu in (False, True):
        with torch.no_grad():
            y = lb().linear(x.cuda(), w.cuda(), relu=relu)
            clean = lb().linear(torch.where(hit[:, None], 0, x).cuda(), w.cuda(), relu=relu)
        A = np.maximum(X, 0) if relu else X                           # (keeps NaNs)
        same_specials(y.cpu()[look], products(A[look], W), magnitude(A[look], W), c)
        assert torch.equal(y.cpu()[~hit], clean.cpu()[~hit])          # the other rows: not another bit
        leaf_x = leaf(x)
        kept = lb().linear(leaf_x, leaf(w), relu=relu)
        assert torch.equal(torch.nan_to_num(kept), torch.nan_to_num(y)) and torch.equal(kept.isnan(), y.isnan())
    # the same numbers as an upstream gradient: dx = dy W over the features of dy
    xs = leaf(torch.ones(n, f))
    for relu in (False, True):
        dx, = torch.autograd.grad(lb().linear(xs, w.t().contiguous().cuda(), relu=relu), xs, x.cuda())
        same_specials(dx.cpu()[look], products(X[look], W), magnitude(X[look], W), c)


@pytest.mark.parametrize("n,c,f", WALKS)
def test_infinities_and_nans_of_the_weight(n, c, f):
    x, w, hit, look = special_operands(n, c, f, n + f)
    x = torch.where(torch.isfinite(x), x, 1.0)
    x[5, :] = 0
    inf = float("inf")
    w2 = w.clone()
    for i, v in enumerate([inf, -inf, float("nan")]):
        w2[(7 * i) % f, (5 + 11 * i) % c] = v
    w2.view(torch.int32)[11 % f, 3] = LOW_NAN
    w2[f - 1, c - 1], w2[f - 2, :] = -inf, inf
    look = torch.cat([look, torch.tensor([5])])
    y = _plain(x, w2).cpu()
    same_specials(y[look], products(np64(x[look]), np64(w2)), magnitude(np64(x[look]), np64(w2)), c)
    fine = torch.isfinite(w2).all(dim=1)
    assert torch.equal(y[:, fine], _plain(x, w).cpu()[:, fine])
    # both at once: where they meet and where they do not
    x2 = x.clone()
    x2[:4, 5 % c], x2[4, 0], x2[6, c - 1] = torch.tensor([inf, -inf, float("nan"), inf]), inf, -inf
    at = torch.arange(8)
    same_specials(_plain(x2, w2).cpu()[at], products(np64(x2[at]), np64(w2)), magnitude(np64(x2[at]), np64(w2)), c)


@pytest.mark.parametrize("n,k,m", [(300, 64, 64), (3000, 100, 65), (129, 5, 1), (5001, 600, 70), (40_000, 64, 3)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nans_of_the_gradient(n, k, m, fmt, dtype):
    """Weight and bias gradients: the columns of dy that hold them get what the sum is, the other columns keep their bits."""
    g = torch.Generator().manual_seed(n + k)
    x, dy = rows(n, k, dtype, seed=n), (1e-2 * torch.randn(n, m, generator=g)).to(dtype)
    x[7, :] = 0                                                       # an infinity times 0
    clean, bad = dy.clone(), sorted({0, m // 2, m - 1})
    inf = float("inf")
    dy[n // 3, bad[0]] = inf
    dy[n - 1, bad[-1]] = -inf
    dy[torch.randint(8, n, (5,), generator=g), bad[len(bad) // 2]] = inf
    if m > 64:
        dy[5, 33], dy[9, 34], dy[11, 34], dy[7, 35] = float("nan"), inf, -inf, inf
        bad += [33, 34, 35]
    ws, bs = leaf(torch.zeros(m, k, dtype=dtype)), leaf(torch.zeros(m, dtype=dtype))
    run = lambda d: [t.cpu() for t in torch.autograd.grad(lb().linear(x.cuda(), ws, bs, relu=True, fmt=fmt), (ws, bs), d.cuda())]
    got, fine = run(dy), run(clean)
    others = [c for c in range(m) if c not in bad]
    assert all(torch.equal(a[others], b[others]) for a, b in zip(got, fine))
    kept = R.quantise(np.maximum(np64(x), 0), "uint8" if fmt == "int8" else fmt, 64)[0]
    with np.errstate(invalid="ignore"):
        want = np.stack([(np64(dy[:, c, None]) * kept).sum(0) for c in bad])
        wdb = np64(dy[:, bad]).sum(0)
    for a, b in ((got[0][bad], want), (got[1][bad], wdb)):
        a = np64(a)
        assert (np.isnan(a) == np.isnan(b)).all() and (a[~np.isnan(b)] == b[~np.isnan(b)]).all()      # nothing finite is left
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(run(dy), got))


@pytest.mark.parametrize("n,c,f", [(5000, 1, 64), (4100, 1, 20), (4500, 1, 200), (5000, 65, 64), (70_000, 129, 32), (20_000, 513, 66)])
def test_a_product_of_two_float32_numbers_is_rounded_like_one(n, c, f):
    """One product per result (the other columns of x are zeros), of numbers with all 24 bits set or drawn.  At most 2^-24 (1 + 2^-8)
    of it is left out and the sums of the terms' products are rounded: five below 2^-6 of the product, then one that may be half a
    step or, cut off, a step of 2^-23 off."""
    g = torch.Generator().manual_seed(n + c)
    at = torch.randint(0, c, (n,), generator=g)
    v = (1 + torch.rand(n, generator=g)) * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0) * torch.exp(4 * torch.randn(n, generator=g))
    v[:500] = 1 + 2.0 ** -7 - 2.0 ** -23
    v[500:1000] = -(1 + 2.0 ** -8 + 2.0 ** -9 - 2.0 ** -23)
    x = torch.zeros(n, c)
    x[torch.arange(n), at] = v
    w = (1 + torch.rand(f, c, generator=g)) * torch.where(torch.rand(f, c, generator=g) < 0.5, -1.0, 1.0)
    w[::4] = 1 + 2.0 ** -7 - 2.0 ** -23
    w[1::4] = 1 + 2.0 ** -8 + 2.0 ** -9 - 2.0 ** -23
    want = np64(v)[:, None] * np64(w).T[at.numpy()]
    y = np64(_plain(x, w))
    bound = (1.01 + 5 * 2.0 ** -6 + 2) * 2.0 ** -24
    assert (np.abs(y - want) <= bound * np.abs(want)).all(), (np.abs(y - want) / np.abs(want)).max() * 2.0 ** 24
    xs = leaf(torch.ones(n, f))
    dx, = torch.autograd.grad(lb().linear(xs, w.t().contiguous().cuda()), xs, x.cuda())
    dx = np64(dx)
    assert (np.abs(dx - want) <= bound * np.abs(want)).all()


@pytest.mark.parametrize("n,c,f", WALKS)
def test_numbers_next_to_the_largest(n, c, f):
    """Rows and weights that rounding to 8 bits would make infinite, the type's lowest number among them, against small ones."""
    g = torch.Generator().manual_seed(n + c + f)
    x, w = rows(n, c, seed=n), torch.randn(f, c, generator=g) * 1e-3
    big = torch.finfo(torch.float32)
    at, col = torch.randperm(n, generator=g)[:30], torch.randint(0, c, (30,), generator=g)
    x[at, col] = torch.tensor([big.max, big.min, 3.3961e38, -3.399e38, 3.3960e38] * 6)
    w2 = w.clone()
    for i, v in enumerate([big.max, big.min, 3.397e38]):
        w2[(5 * i) % f, (3 + 7 * i) % c] = v
    look = torch.cat([at, torch.randint(0, n, (50,), generator=g)])
    small = torch.where(x.abs() > 1e38, 1e-3 * torch.ones(()), x.clamp(-0.4, 0.4))
    for a, b in ((x, w), (small, w2)):
        want = products(np64(a[look]), np64(b))
        assert np.isfinite(want.astype(np.float32)).all()
        same_specials(_plain(a, b).cpu()[look], want, magnitude(np64(a[look]), np64(b)), c)
        xs = leaf(torch.ones(n, f))
        dx, = torch.autograd.grad(lb().linear(xs, b.t().contiguous().cuda()), xs, a.cuda())
        same_specials(dx.cpu()[look], want, magnitude(np64(a[look]), np64(b)), c)
    # both: a row's largest number meets an infinite weight, a weight's an infinite number
    x3, w3 = x.clone(), w2.clone()
    x3[0, :], w3[1 % f, :] = big.max, float("inf")
    x3[1, :] = float("-inf")
    assert (_plain(x3, w3).cpu()[0, 1 % f] == float("inf")) and (_plain(x3, w3).cpu()[1, 1 % f] == float("-inf"))


def chunk_rows(n, k, m):
    groups, tiles = -(-k // 64), -(-m // 64)
    gw = 8 if groups >= 8 else 4 if groups >= 4 else 2 if groups >= 2 else 1
    chunks = max(1, min(256 // (tiles * -(-groups // gw)), -(-n // 128)))
    return -(-(-(-n // chunks)) // 128) * 128


SUMS = [(70_001, 64, 64), (40_007, 200, 70), (33_000, 520, 20), (5000, 64, 64), (129, 70, 33), (17, 64, 64), (16, 64, 5), (15, 64, 2), (1, 64, 1)]


@pytest.mark.parametrize("n,k,m", SUMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_row_is_in_the_weight_gradient_once(n, k, m, dtype):
    """Whole numbers: scales of 1, codes of at most 127, dy of -1, 0 and 1.  Every partial sum is below 2^24 (70 001 x 127), so the
    result does not depend on the order and is compared for equality, in the 16-bit types after its one rounding."""
    g = torch.Generator().manual_seed(n + k + m)
    x = torch.randint(-127, 128, (n, k), generator=g).float()
    x[:, ::64] = 127                                                  # every group's largest: a scale of 1
    dy = torch.randint(-1, 2, (n, m), generator=g).float()
    dy[-1] = 1
    ws, bs = leaf(torch.zeros(m, k, dtype=dtype)), leaf(torch.zeros(m, dtype=dtype))
    dw, db = torch.autograd.grad(lb().linear(x.to(dtype).cuda(), ws, bs), (ws, bs), dy.to(dtype).cuda())
    assert torch.equal(dw.cpu(), (dy.double().T @ x.double()).to(dtype)) and torch.equal(db.cpu(), dy.double().sum(0).to(dtype))
    db1, = torch.autograd.grad(lb().linear(x.to(dtype).cuda(), ws.detach(), bs), bs, dy.to(dtype).cuda())
    assert torch.equal(db1, db)


@pytest.mark.parametrize("n,k,m", SUMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_rows_at_every_border_are_whole(n, k, m, dtype):
    """One row per column of dy is not zero -- the first and last of steps of 16 and of chunks, and of all -- with a number of all the
    type's bits; codes are powers of two, so the sum is exact: a lost row, or a lost term of dy, is all of the result or its last bits."""
    per = chunk_rows(n, k, m)
    at = {0, n - 1, n - 2, n - 15, n - 16, n - 17, 15, 16}
    for b in range(per, n + per, per):
        at |= {b - 17, b - 16, b - 1, b, b + 15, b + 16}
    at = sorted(r for r in at if 0 <= r < n)
    bits = {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}[dtype]
    x = 2.0 ** ((torch.arange(n)[:, None] * 5 + torch.arange(k)) % 7).float()
    x[:, ::64] = 127
    for i in range(0, len(at), m):
        dy, want = torch.zeros(n, m), torch.zeros(m, k, dtype=torch.float64)
        for c, r in enumerate(at[i:i + m]):
            dy[r, c] = (2 ** bits - 1 - 2 * (c % 50)) * 2.0 ** (-bits)
            want[c] = dy[r, c].double() * x[r].double()
        ws, bs = leaf(torch.zeros(m, k, dtype=dtype)), leaf(torch.zeros(m, dtype=dtype))
        dw, db = torch.autograd.grad(lb().linear(x.to(dtype).cuda(), ws, bs), (ws, bs), dy.to(dtype).cuda())
        exact = torch.ones(k, dtype=torch.bool)
        exact[::64] = False                                           # times 127: rounded
        assert torch.equal(dw.cpu()[:, exact], want[:, exact].to(dtype)) and torch.equal(db.cpu(), dy.sum(0).to(dtype))


@pytest.mark.parametrize("n,k,m", [(70_001, 64, 64), (40_007, 200, 70), (33_000, 520, 20)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_of_many_rows(n, k, m, dtype):
    g = torch.Generator().manual_seed(n)
    x, dy = rows(n, k, dtype, seed=n), (1e-2 * torch.randn(n, m, generator=g)).to(dtype)
    ws, bs = leaf(torch.zeros(m, k, dtype=dtype)), leaf(torch.zeros(m, dtype=dtype))
    dw, db = torch.autograd.grad(lb().linear(x.cuda(), ws, bs, relu=True), (ws, bs), dy.cuda())
    kept, D = R.quantise(np.maximum(np64(x), 0), "uint8", 64)[0], np64(dy)
    depth = weight_gradient_roundings(n, k, m)
    for got, want, most in ((dw, D.T @ kept, np.abs(D).T @ kept), (db, D.sum(0), np.abs(D).sum(0))):
        tol = depth * 2.0 ** -24 * most
        if dtype is not torch.float32:
            tol = tol + np.abs(want) * torch.finfo(dtype).eps / 2 + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
        assert (np.abs(np64(got) - want) <= tol).all(), (np.abs(np64(got) - want) / tol).max()
        if dtype is torch.float32:                                    # what a lost step of 16 rows would be is well above the tolerance
            assert (np.abs(D[-17:-1].T @ kept[-17:-1]) > 3 * tol).mean() > 0.5 if got is dw else True


@pytest.mark.parametrize("n,k,m,dtype", [(20_000, 450, 450, torch.float32), (70_000, 512, 66, torch.float32), (70_000, 66, 450, torch.float32),
                                         (45_000, 700, 300, torch.bfloat16), (45_000, 300, 700, torch.float16)])
def test_a_weight_that_does_not_fit_over_several_rounds(n, k, m, dtype):
    """The contraction's groups pass through LDS in portions, again for each round of rows: every one of forward and input gradient."""
    x, w, b, dy = make(n, k, m, dtype)
    xs = leaf(x)
    y = lb().linear(xs, w.cuda(), b.cuda(), relu=True)
    dx, = torch.autograd.grad(y, xs, dy.cuda())
    X, W, D = np.maximum(np64(x), 0), np64(w), np64(dy)
    near(y, X @ W.T + np64(b), X @ np.abs(W).T + np.abs(np64(b)), k)
    near(dx, np.where(X > 0, D @ W, 0), np.abs(D) @ np.abs(W), m)
