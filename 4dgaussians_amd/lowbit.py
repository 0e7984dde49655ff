"""Rows of numbers kept in 8 bits, over libgs4d.so (csrc/lowbit.hip, csrc/hexplane.hip):

  RowCache(capacity, width, fmt, group)
      a table of rows that are quantised as they are written (`write`) and read back as numbers (`read`), at consecutive or at
      given slots: what a renderer keeps per Gaussian between frames;
  frame_features(cache, planes, aabb, points, t)
      the plane features of one frame, the spatial planes' product read from such a cache;
  linear(x, weight, bias, relu, fmt)
      a linear layer that keeps its input in 8 bits, not the input itself, for the backward.

The format: columns in groups, one float32 scale per group and row,

    a = max |x| over the group     s = a / Q     code = round_half_even(x * (Q / a))     value = s * code

with Q = 127 for "int8", 448 for "e4m3", 57344 for "e5m2" (the quotients and the product rounded to float32).  A group whose s
is below 2^-126 is stored as zero; a group that holds an infinity or a NaN reads as NaN.  The value is off by at most half a
step: s / 2 for int8, a relative 2^-4 (e4m3) or 2^-3 (e5m2) above the format's subnormals.

Host plumbing only; there is no CPU path (CPU tensors and a missing library raise).
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _cabi

FORMATS = {"int8": 0, "e4m3": 1, "e5m2": 2}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GROUPS = (32, 64, 128)
KEEP_CODES, KEEP_SIGNS = 1, 2          # GS4D_KEEP_* of include/gs4d.h
SCAN = 256                             # GS4D_ROWS8_SCAN


class Rows8(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("scales", C.c_void_p), ("owner", C.c_void_p), ("capacity", C.c_longlong),
                ("width", C.c_int), ("pitch", C.c_int), ("group", C.c_int), ("fmt", C.c_int)]


def _format(fmt):
    if fmt not in FORMATS:
        raise RuntimeError(f"unknown 8-bit format {fmt!r}: one of {', '.join(FORMATS)}")
    return FORMATS[fmt]


def _on_device(name, t, dev=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on a HIP device; there is no CPU path")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, expected {dev}")


def _dtype(name, t):
    if t.dtype not in DTYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return DTYPES[t.dtype]


class RowCache:
    """`capacity` rows of `width` numbers in 8 bits.  codes: uint8 [capacity, pitch], pitch = width rounded up to 16; scales:
    float32 [capacity, ceil(width / group)].  Both start as zeros, i.e. as rows of zeros.

    Calls run on the current stream of the cache's device; calls on one cache from several streams are ordered by the caller."""

    def __init__(self, capacity, width, fmt="int8", group=64, device="cuda"):
        if int(capacity) < 1 or not 1 <= int(width) <= 65536:
            raise RuntimeError(f"RowCache: at least one row of 1 to 65536 columns, got {capacity} and {width}")
        if group not in GROUPS:
            raise RuntimeError(f"RowCache: group must be 32, 64 or 128, got {group}")
        _format(fmt)
        codes = torch.zeros(int(capacity), (int(width) + 15) // 16 * 16, dtype=torch.uint8, device=device)
        scales = torch.zeros(int(capacity), -(-int(width) // group), dtype=torch.float32, device=device)
        self._set(codes, scales, int(width), fmt, group)

    @classmethod
    def from_buffers(cls, codes, scales, width, fmt="int8", group=64):
        """A cache over existing arrays (no copy): codes uint8 [capacity, pitch], scales float32 [capacity, ceil(width / group)]."""
        self = cls.__new__(cls)
        self._set(codes, scales, int(width), fmt, group)
        return self

    def _set(self, codes, scales, width, fmt, group):
        if group not in GROUPS:
            raise RuntimeError(f"RowCache: group must be 32, 64 or 128, got {group}")
        f = _format(fmt)
        _on_device("codes", codes)
        _on_device("scales", scales, codes.device)
        if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_contiguous() or codes.shape[0] < 1 or not 1 <= width <= 65536 \
                or codes.shape[1] < width or codes.shape[1] % 16 or codes.data_ptr() % 16:
            raise RuntimeError("RowCache: codes must be a contiguous uint8 tensor [capacity, pitch], 16-byte aligned, pitch a "
                               "multiple of 16 and at least width")
        if scales.dtype != torch.float32 or not scales.is_contiguous() or tuple(scales.shape) != (codes.shape[0], -(-width // group)):
            raise RuntimeError("RowCache: scales must be a contiguous float32 tensor [capacity, ceil(width / group)]")
        self.codes, self.scales, self.width, self.fmt, self.group = codes, scales, width, fmt, group
        self.capacity, self.device = codes.shape[0], codes.device
        self._owner = None
        self._desc = Rows8(codes.data_ptr(), scales.data_ptr(), None, self.capacity, width, codes.shape[1], group, f)
        self._ref = C.addressof(self._desc)

    def _at(self, slots, start, n):
        """-> (address, bytes per slot, tensor to keep alive); checks what the host can see."""
        if slots is None:
            if start < 0 or start + n > self.capacity:
                raise RuntimeError(f"RowCache: rows {start} .. {start + n} do not fit {self.capacity} slots")
            return None, 0, None
        if start != 0:
            raise RuntimeError("RowCache: give either slots or start")
        _on_device("slots", slots, self.device)
        if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
            raise RuntimeError("RowCache: slots must be a vector of int32 or int64")
        slots = slots.contiguous()
        return slots.data_ptr(), 8 if slots.dtype is torch.int64 else 4, slots

    def write(self, rows, slots=None, start=0):
        """rows [n, width] (float32, bfloat16 or float16, any row stride) to the slots start, start + 1, ... or to slots [n]
        (int32 / int64).  A slot outside the cache is padding: its row is not stored.  Of several rows for one slot the last is
        kept.  No gradient flows into the cache."""
        _on_device("rows", rows, self.device)
        if rows.dim() != 2 or rows.shape[1] != self.width:
            raise RuntimeError(f"RowCache.write: rows must have the shape [n, {self.width}], got {tuple(rows.shape)}")
        rows = rows.detach()
        dt, n = _dtype("rows", rows), rows.shape[0]
        if slots is not None and isinstance(slots, torch.Tensor) and slots.numel() != n:
            raise RuntimeError(f"RowCache.write: {n} rows and {slots.numel()} slots")
        p, size, keep = self._at(slots, int(start), n)
        if n == 0:
            return
        if (self.width > 1 and rows.stride(1) != 1) or (n > 1 and rows.stride(0) < self.width):
            rows = rows.contiguous()
        ref = self._ref
        with _cabi.on_device(self.device):
            stream = _cabi.stream_of(self.device)
            if slots is not None and n > SCAN:
                if torch.cuda.is_current_stream_capturing():
                    # an array of the graph's own: its zeros are written when the graph runs, and it lives as long as the graph
                    owner = torch.zeros(self.capacity, dtype=torch.int32, device=self.device)
                    d = Rows8.from_buffer_copy(self._desc)
                    d.owner, ref = owner.data_ptr(), C.addressof(d)
                elif self._owner is None:
                    self._owner, self._owner_stream = torch.zeros(self.capacity, dtype=torch.int32, device=self.device), stream
                    self._desc.owner = self._owner.data_ptr()
                elif stream != self._owner_stream:
                    self._owner.record_stream(torch.cuda.current_stream(self.device))      # the caller cannot, and may drop the cache
            rc = _cabi.lib().gs4d_rows8_write(ref, rows.data_ptr(), dt, rows.stride(0) if n > 1 else self.width, n, p, size,
                                              int(start), stream)
        if rc:
            _cabi.check(rc, "gs4d_rows8_write")

    def read(self, slots=None, start=0, count=None, dtype=torch.float32):
        """-> [n, width] of `dtype`: the rows at slots [n] (zeros where a slot lies outside the cache), or `count` rows (all
        that follow, by default) from `start` on."""
        if dtype not in DTYPES:
            raise RuntimeError(f"RowCache.read: dtype must be float32, bfloat16 or float16, got {dtype}")
        if slots is None:
            n = self.capacity - int(start) if count is None else int(count)
            if n < 0:
                raise RuntimeError("RowCache.read: count must not be negative")
        else:
            _on_device("slots", slots, self.device)
            n = slots.numel()
            if count is not None and int(count) != n:
                raise RuntimeError(f"RowCache.read: count is {count}, but there are {n} slots")
        p, size, keep = self._at(slots, int(start), n)
        out = torch.empty(n, self.width, dtype=dtype, device=self.device)
        if n == 0:
            return out
        with _cabi.on_device(self.device):
            rc = _cabi.lib().gs4d_rows8_read(self._ref, out.data_ptr(), DTYPES[dtype], self.width, n, p, size, int(start),
                                             _cabi.stream_of(self.device))
        if rc:
            _cabi.check(rc, "gs4d_rows8_read")
        return out


def frame_features(cache, planes, aabb, points, t):
    """The features [P, L * C] (float32) of points [P, 3] in the frame at the normalised time t (a tensor of one or of P values):
    row p of the cache -- the product of a level's three spatial planes, levels side by side -- times the bilinear samples of
    the level's three planes over (axis, t).  planes: 3 per level in the order x, y, z, each [1, C, T, axis] float32, C a power of
    two from 4 to 256 (channels last in memory, or it is copied so); aabb [2, 3] as HexPlaneField keeps it.  Rendering only: no gradient."""
    if not isinstance(cache, RowCache):
        raise RuntimeError("frame_features: cache must be a RowCache")
    dev = cache.device
    planes = list(planes)
    if not planes or len(planes) % 3 or len(planes) > 12:
        raise RuntimeError(f"frame_features: three planes for each of 1 to 4 levels, got {len(planes)} planes")
    shapes, data = [], []
    for p in planes:
        _on_device("planes", p, dev)
        shape = p.shape
        if p.dtype is not torch.float32 or len(shape) != 4 or shape[0] != 1 or (shapes and shape[1] != shapes[0][1]):
            raise RuntimeError("frame_features: planes must be float32 [1, C, T, axis] with one C")
        shapes.append(shape)
        data.append(p if p.is_contiguous(memory_format=torch.channels_last) else p.detach().contiguous(memory_format=torch.channels_last))
    for name, v in (("aabb", aabb), ("points", points), ("t", t)):
        _on_device(name, v, dev)
        if v.dtype is not torch.float32:
            raise RuntimeError(f"frame_features: {name} must be float32, got {v.dtype}")
    if points.dim() != 2 or points.shape[1] != 3 or tuple(aabb.shape) != (2, 3) or t.numel() not in (1, points.shape[0]):
        raise RuntimeError("frame_features: points [P, 3], aabb [2, 3] and one or P values of t")
    P, ch, levels = points.shape[0], shapes[0][1], len(planes) // 3
    if cache.width != levels * ch or P > cache.capacity:
        raise RuntimeError(f"frame_features: the cache holds {cache.capacity} rows of {cache.width}, expected at least {P} of {levels * ch}")
    aabb, points, t = aabb.detach().contiguous(), points.detach().contiguous(), t.detach().reshape(-1).contiguous()
    out = torch.empty(P, cache.width, dtype=torch.float32, device=dev)
    n = len(planes)
    with _cabi.on_device(dev):
        rc = _cabi.lib().gs4d_frame_features(
            cache._ref, levels, ch, (C.c_void_p * n)(*[p.data_ptr() for p in data]), (C.c_int * n)(*[q[3] for q in shapes]),
            (C.c_int * n)(*[q[2] for q in shapes]), aabb.data_ptr(), points.data_ptr(), t.data_ptr(),
            0 if t.numel() == 1 else 1, P, out.data_ptr(), cache.width, _cabi.stream_of(dev))
    if rc:
        _cabi.check(rc, "gs4d_frame_features")
    return out


def _linear_forward(x, weight, bias, relu, fmt, what):
    """-> y, the kept block (or None), rows; x, weight and bias detached."""
    L = _cabi.lib()
    dev = x.device
    M, K = weight.shape
    rows = x.reshape(-1, K)
    N = rows.shape[0]
    if N and ((K > 1 and rows.stride(1) != 1) or (N > 1 and rows.stride(0) < K)):
        rows = rows.contiguous()
    weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
    y = torch.empty(*x.shape[:-1], M, dtype=x.dtype, device=dev)
    keep = torch.empty(L.gs4d_linear8_keep_bytes(N, K, what), dtype=torch.uint8, device=dev) if what else None
    with _cabi.on_device(dev):
        rc = L.gs4d_linear8_forward(DTYPES[x.dtype], N, K, M, rows.data_ptr(), rows.stride(0) if N > 1 else K, weight.data_ptr(),
                                    _cabi.address(bias), relu, fmt, y.data_ptr(), _cabi.address(keep), what, _cabi.stream_of(dev))
    if rc:
        _cabi.check(rc, "gs4d_linear8_forward")
    return y, keep, N


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, relu, fmt):
        need_x, need_w = ctx.needs_input_grad[:2]
        what = (KEEP_CODES if need_w else 0) | (KEEP_SIGNS if relu and need_x else 0)
        y, keep, N = _linear_forward(x.detach(), weight.detach(), None if bias is None else bias.detach(), relu, fmt, what)
        ctx.save_for_backward(weight, keep)
        ctx.args = (DTYPES[x.dtype], N, weight.shape[1], weight.shape[0], relu, fmt, what, x.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        L = _cabi.lib()
        weight, keep = ctx.saved_tensors
        dt, N, K, M, relu, fmt, what, x_shape = ctx.args
        dev = g.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy, w = g.reshape(N, M).contiguous(), weight.detach().contiguous()
        dx = torch.empty(N, K, dtype=g.dtype, device=dev) if need_x else None
        dw = torch.empty(M, K, dtype=g.dtype, device=dev) if need_w else None
        db = torch.empty(M, dtype=g.dtype, device=dev) if need_b else None
        scratch = torch.empty(L.gs4d_linear8_scratch_bytes(N, K, M), dtype=torch.uint8, device=dev) if need_w or need_b else None
        with _cabi.on_device(dev):
            rc = L.gs4d_linear8_backward(dt, N, K, M, dy.data_ptr() if N else None, w.data_ptr(), relu, fmt, _cabi.address(keep), what,
                                         _cabi.address(dx), _cabi.address(dw), _cabi.address(db), _cabi.address(scratch),
                                         _cabi.stream_of(dev))
        if rc:
            _cabi.check(rc, "gs4d_linear8_backward")
        return None if dx is None else dx.view(x_shape), dw, db, None, None


def linear(x, weight, bias=None, relu=False, fmt="int8"):
    """act(x) @ weight.T + bias with act = relu or nothing: x [..., K], weight [M, K], bias [M], all of one dtype (float32,
    bfloat16 or float16; sums in float32).  For the backward it keeps act(x) in 8 bits in groups of 64 columns ("int8": 255
    levels of a rectified input, 127 each way of a signed one) and, with relu, the signs of x, instead of x: per row and group 64
    bytes and a scale of 4, with relu 8 more, the last group in full -- about a quarter of a float32 input of 64 columns, but more
    than the input itself below 19 columns (38 of a 16-bit type).  The input gradient is exact; the weight gradient is taken
    with the kept values.  Operands of several types are cast to autocast's under autocast
    and refused outside of it; operands of one type are taken as they are.  No forward-mode derivative.  At most 2^28 weights, K
    and M at most 2^20."""
    f = _format(fmt)
    _on_device("x", x)
    _on_device("weight", weight, x.device)
    _dtype("x", x)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"linear: x [..., K] and weight [M, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if (weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype)) and torch.is_autocast_enabled("cuda") \
            and all(v is None or v.dtype in DTYPES for v in (weight, bias)):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
    if weight.dtype != x.dtype:
        raise RuntimeError(f"linear: x is {x.dtype}, weight {weight.dtype}")
    if bias is not None:
        _on_device("bias", bias, x.device)
        if bias.dtype != x.dtype or tuple(bias.shape) != (weight.shape[0],):
            raise RuntimeError(f"linear: bias must be {x.dtype} [{weight.shape[0]}], got {bias.dtype} {tuple(bias.shape)}")
    if forward_ad._current_level >= 0 and any(v is not None and forward_ad.unpack_dual(v).tangent is not None for v in (x, weight, bias)):
        raise RuntimeError("linear has no forward-mode derivative; an operand has a tangent")
    relu = int(bool(relu))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _Linear.apply(x, weight, bias, relu, f)
    return _linear_forward(x, weight, bias, relu, f, 0)[0]
