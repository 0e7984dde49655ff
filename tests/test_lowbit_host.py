"""8-bit rows without a GPU: what the entry points refuse, the sizes they ask for, and the oracle's own arithmetic."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import lowbit_ref as R


@pytest.fixture(scope="module")
def lb():
    return pkg("lowbit")


def test_no_cpu_path(lb):
    with pytest.raises(RuntimeError, match="no CPU path"):
        lb.RowCache(4, 8, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        lb.RowCache.from_buffers(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1), 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        lb.linear(torch.zeros(2, 4), torch.zeros(3, 4))


@pytest.mark.parametrize("kw", [dict(capacity=0, width=8), dict(capacity=4, width=0), dict(capacity=4, width=8, group=48),
                                dict(capacity=4, width=8, fmt="int4")])
def test_cache_refuses(lb, kw):
    with pytest.raises(RuntimeError):
        lb.RowCache(device="cpu", **kw)


def desc(lb, **kw):
    d = dict(codes=1 << 20, scales=1 << 16, owner=0, capacity=10, width=20, pitch=32, group=64, fmt=0)
    d.update(kw)
    return lb.Rows8(*[d[n] for n, _ in lb.Rows8._fields_])


BAD_CACHE = [dict(codes=0), dict(scales=0), dict(codes=(1 << 20) + 8), dict(capacity=0), dict(width=0), dict(width=33),
             dict(pitch=24), dict(group=16), dict(group=0), dict(fmt=3), dict(fmt=-1)]
# n, ld, dtype, slots, slot_bytes, start
BAD_ROWS = [(-1, 20, 0, 0, 0, 0), (11, 20, 0, 0, 0, 0), (5, 20, 0, 0, 0, 6), (5, 20, 0, 0, 0, -1), (5, 19, 0, 0, 0, 0), (5, 20, 3, 0, 0, 0),
            (5, 20, -1, 0, 0, 0), (5, 20, 0, 4096, 2, 0), (1 << 31, 20, 0, 4096, 8, 0)]


@pytest.mark.parametrize("name", ["gs4d_rows8_write", "gs4d_rows8_read"])
def test_entry_points_refuse_bad_caches_and_rows(lb, name):
    f = getattr(pkg("_cabi").lib(), name)
    call = lambda d, rows=4096, n=5, ld=20, dtype=0, slots=0, size=0, start=0: f(
        C.byref(d), C.c_void_p(rows), C.c_int(dtype), C.c_longlong(ld), C.c_longlong(n), C.c_void_p(slots), C.c_int(size),
        C.c_longlong(start), C.c_void_p(0))
    for kw in BAD_CACHE:
        assert call(desc(lb, **kw)) == -1, kw
    for n, ld, dtype, slots, size, start in BAD_ROWS:
        assert call(desc(lb), n=n, ld=ld, dtype=dtype, slots=slots, size=size, start=start) == -1, (n, ld, dtype, slots, size, start)
    assert call(desc(lb), rows=0) == -1
    assert call(desc(lb, capacity=1 << 25, width=4096, pitch=4096), n=1 << 24, ld=4096) == -1
    assert call(desc(lb), n=0) == 0                                   # nothing to do, nothing launched
    if name == "gs4d_rows8_write":                                    # many rows at given slots need the owner array
        assert call(desc(lb), n=lb.SCAN + 1, slots=4096, size=8) == -1
        assert "owner" in pkg("_cabi").lib().gs4d_last_error().decode()


def test_linear_refuses(lb):
    L = pkg("_cabi").lib()
    fwd = lambda dtype=0, N=4, K=8, M=8, x=4096, ldx=8, w=4096, b=0, relu=0, fmt=0, y=4096, keep=0, what=0: L.gs4d_linear8_forward(
        C.c_int(dtype), C.c_longlong(N), C.c_int(K), C.c_int(M), C.c_void_p(x), C.c_longlong(ldx), C.c_void_p(w), C.c_void_p(b),
        C.c_int(relu), C.c_int(fmt), C.c_void_p(y), C.c_void_p(keep), C.c_int(what), C.c_void_p(0))
    for kw in (dict(dtype=3), dict(N=-1), dict(K=0), dict(M=0), dict(x=0), dict(w=0), dict(y=0), dict(ldx=7), dict(fmt=3), dict(what=1),
               dict(what=1, keep=64), dict(what=2, keep=4096), dict(N=1 << 31), dict(K=1 << 15, M=1 << 14, ldx=1 << 15)):
        assert fwd(**kw) == -1, kw
    assert fwd(N=0, x=0, y=0) == 0
    bwd = lambda dtype=0, N=4, K=8, M=8, dy=4096, w=4096, relu=0, fmt=0, keep=4096, what=3, dx=4096, dw=4096, db=0, scratch=4096: \
        L.gs4d_linear8_backward(C.c_int(dtype), C.c_longlong(N), C.c_int(K), C.c_int(M), C.c_void_p(dy), C.c_void_p(w), C.c_int(relu),
                                C.c_int(fmt), C.c_void_p(keep), C.c_int(what), C.c_void_p(dx), C.c_void_p(dw), C.c_void_p(db),
                                C.c_void_p(scratch), C.c_void_p(0))
    for kw in (dict(dy=0), dict(w=0), dict(keep=0), dict(keep=64), dict(scratch=0), dict(scratch=64), dict(what=2), dict(what=1, relu=1),
               dict(fmt=4), dict(M=0), dict(dtype=-1)):
        assert bwd(**kw) == -1, kw


def test_sizes(lb):
    L = pkg("_cabi").lib()
    keep = lambda n, k, what: L.gs4d_linear8_keep_bytes(C.c_longlong(n), C.c_int(k), C.c_int(what))
    assert keep(100_000, 64, 1) < 100_000 * 68 + 1024                 # 64 codes and a scale per row, not 256 bytes
    assert keep(100_000, 64, 3) < 100_000 * 76 + 1024
    assert keep(1 << 26, 64, 1) > (1 << 26) * 68                      # past 32 bits
    assert keep(0, 64, 3) > 0 and keep(5, 64, 0) > 0


def test_frame_refuses(lb):
    L = pkg("_cabi").lib()
    planes, ones = (C.c_void_p * 3)(4096, 4096, 4096), (C.c_int * 3)(4, 4, 4)

    def call(levels=1, ch=16, P=4, cache=None, planes=planes, w=ones, out=4096, ld=16, stride=0, points=4096, **kw):
        d = cache if cache is not None else desc(lb, width=16, **kw)
        return L.gs4d_frame_features(C.byref(d), C.c_int(levels), C.c_int(ch), planes, w, ones, C.c_void_p(4096), C.c_void_p(points),
                                     C.c_void_p(4096), C.c_int(stride), C.c_longlong(P), C.c_void_p(out), C.c_longlong(ld), C.c_void_p(0))
    assert call(P=0) == 0
    for kw in (dict(levels=0), dict(levels=5), dict(ch=12), dict(ch=8), dict(P=11), dict(P=-1), dict(out=0), dict(out=4100), dict(ld=12),
               dict(ld=18), dict(stride=2), dict(points=0), dict(planes=(C.c_void_p * 3)(4096, 0, 4096)),
               dict(planes=(C.c_void_p * 3)(4096, 4100, 4096)), dict(w=(C.c_int * 3)(4, 0, 4)), dict(codes=0), dict(group=8), dict(fmt=3)):
        assert call(**kw) == -1, kw


@pytest.mark.parametrize("fmt", ["int8", "uint8", "e4m3", "e5m2"])
def test_oracle_is_within_half_a_step_and_idempotent(fmt):
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 150)) * np.exp(3 * rng.standard_normal((50, 1)))).astype(np.float32)
    x[3, :64] = 0
    if fmt == "uint8":
        x = np.abs(x)
    v, step = R.quantise(x, fmt, 64)
    # the quotient and the product each add a relative 2^-24 of at most Q steps
    assert (np.abs(v - x) <= 0.5 * step + np.abs(x) * 2.0 ** -22).all()
    assert (v[3, :64] == 0).all()
    if fmt in ("e4m3", "e5m2"):
        t = torch.from_numpy(x[:, :64] * (R.TOP[fmt] / np.abs(x[:, :64]).max(axis=1, keepdims=True).clip(min=1e-30)).astype(np.float32))
        q = t.to(torch.float8_e4m3fn if fmt == "e4m3" else torch.float8_e5m2).double().numpy()
        s = (np.abs(x[:, :64]).max(axis=1, keepdims=True) / np.float32(R.TOP[fmt])).astype(np.float64)
        assert (q * s == v[:, :64]).all()


@pytest.mark.parametrize("k, m", [(1, (1 << 20) + 1), ((1 << 20) + 1, 1), (1, 1 << 28), (1 << 28, 1)])
def test_linear_refuses_one_very_long_dimension(lb, k, m):
    """Few weights, but eight rows of M or K elements no longer have 32-bit offsets."""
    L = pkg("_cabi").lib()
    p, z = C.c_void_p(4096), C.c_void_p(0)
    assert L.gs4d_linear8_forward(C.c_int(0), C.c_longlong(4), C.c_int(k), C.c_int(m), p, C.c_longlong(k), p, z, C.c_int(0), C.c_int(0),
                                  p, z, C.c_int(0), z) == -1
    assert L.gs4d_linear8_backward(C.c_int(0), C.c_longlong(4), C.c_int(k), C.c_int(m), p, p, C.c_int(0), C.c_int(0), p, C.c_int(1),
                                   z, p, z, p, z) == -1
