"""Plain restatement of the 8-bit row operators on the CPU in 64 bits (numpy): test infrastructure only.

Definition (include/gs4d.h): columns in groups, a = max |x|, s = fl32(a / Q), code = round_half_even(fl32(x * fl32(Q / a))) in
the format, value = s * code; s below 2^-126: zero; a group with an infinity or a NaN: NaN.  A quotient or a product of two
float32 numbers taken in 64 bits and rounded to 32 is the float32 operation's result (53 >= 2 * 24 + 2)."""
import numpy as np

TOP = {"int8": 127.0, "uint8": 255.0, "e4m3": 448.0, "e5m2": 57344.0}
STEPS = {"e4m3": (3, -6), "e5m2": (2, -14)}          # mantissa bits, least exponent
TINY = 2.0 ** -126


def _f32(x):
    with np.errstate(over="ignore"):
        return x.astype(np.float32).astype(np.float64)


def quantise(x, fmt, group):
    """x [n, width] -> (values [n, width], step at the value [n, width]), float64; the value is within half a step of x."""
    x = np.asarray(x, np.float64)
    out, step = np.empty_like(x), np.empty_like(x)
    for g0 in range(0, x.shape[1], group):
        v = x[:, g0:g0 + group]
        bad = ~np.isfinite(v).all(axis=1, keepdims=True)
        a = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(axis=1, keepdims=True))
        s = _f32(a / TOP[fmt])
        live = s >= TINY
        with np.errstate(divide="ignore", invalid="ignore"):
            inv = np.where(live, _f32(TOP[fmt] / np.where(live, a, 1.0)), 0.0)
            q = _f32(np.where(bad, 0.0, v) * inv)
        if fmt in STEPS:
            bits, least = STEPS[fmt]
            one = np.ldexp(1.0, np.maximum(np.frexp(q)[1] - 1, least) - bits)
            q = np.clip(np.round(q / one) * one, -TOP[fmt], TOP[fmt])
        else:
            one = np.ones_like(q)
            q = np.round(q)
        out[:, g0:g0 + group] = np.where(bad, np.nan, q * np.where(live, s, 0.0))
        step[:, g0:g0 + group] = np.where(live, one * s, 2 * a)
    return out, step


def write(table, rows, slots, fmt, group):
    """table [capacity, width] float64 after the rows were written to `slots`, one after the other."""
    table = table.copy()
    held = quantise(rows, fmt, group)[0]
    for i, s in enumerate(slots):
        if 0 <= s < table.shape[0]:
            table[s] = held[i]
    return table


def frame_features(static, planes, aabb, points, t):
    """static [P, L C] (values of the cache), planes: 3 L arrays [C, T, X], aabb [2, 3], points [P, 3], t [P] -> [P, L C]."""
    out = np.array(static, np.float64)
    ch = planes[0].shape[0]
    box, pts = np.asarray(aabb, np.float64), np.asarray(points, np.float64)
    for i, plane in enumerate(planes):
        p = np.asarray(plane, np.float64)
        u = (pts[:, i % 3] - box[0, i % 3]) * 2 / (box[1, i % 3] - box[0, i % 3]) - 1
        x = np.clip((u + 1) / 2 * (p.shape[2] - 1), 0, p.shape[2] - 1)
        y = np.clip((np.asarray(t, np.float64) + 1) / 2 * (p.shape[1] - 1), 0, p.shape[1] - 1)
        x0, y0 = np.floor(x).astype(int), np.floor(y).astype(int)
        x1, y1 = np.minimum(x0 + 1, p.shape[2] - 1), np.minimum(y0 + 1, p.shape[1] - 1)
        fx, fy = x - x0, y - y0
        v = ((p[:, y0, x0] * (1 - fx) + p[:, y0, x1] * fx) * (1 - fy) + (p[:, y1, x0] * (1 - fx) + p[:, y1, x1] * fx) * fy).T
        out[:, (i // 3) * ch:(i // 3 + 1) * ch] *= v
    return out


def linear(x, w, b, relu, fmt, dy=None):
    """-> y, or (y, dx, dw, db, kept) with the upstream gradient dy."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    a = np.maximum(x, 0) if relu else x
    y = a @ w.T + (0 if b is None else np.asarray(b, np.float64))
    if dy is None:
        return y
    dy = np.asarray(dy, np.float64)
    kept = quantise(a, "uint8" if relu and fmt == "int8" else fmt, 64)[0]
    dx = dy @ w
    return y, np.where(x > 0, dx, 0.0) if relu else dx, dy.T @ kept, dy.sum(axis=0), kept
