"""64-bit definitions of the adapter and checkpoint operators, element by element in numpy (test infrastructure only)."""
import numpy as np

BLOCK = 32


def forward(x, w, b, down, up, groups, scale, slope):
    """(u, y) in float64."""
    x, w, down, up = (np.asarray(t, np.float64) for t in (x, w, down, up))
    u = np.zeros((len(x), down.shape[1]))
    z = x @ w.T + (0 if b is None else np.asarray(b, np.float64))
    for r, g in enumerate(groups):
        if 0 <= g < len(down):
            u[r] = down[g] @ x[r]
            z[r] += scale * (up[g] @ u[r])
    return u, (z if slope is None else np.where(z > 0, z, slope * z))


def backward(dy, x, y, u, w, down, up, groups, scale, slope):
    """(dx, ddown, dup, dw, db); y: what the derivative is read from (None without an activation)."""
    dy, x, u, w, down, up = (np.asarray(t, np.float64) for t in (dy, x, u, w, down, up))
    p = dy if slope is None else np.where(np.asarray(y, np.float64) > 0, dy, slope * dy)
    dx, ddown, dup = p @ w, np.zeros_like(down), np.zeros_like(up)
    for r, g in enumerate(groups):
        if 0 <= g < len(down):
            v = scale * (p[r] @ up[g])
            dx[r] += v @ down[g]
            ddown[g] += np.outer(v, x[r])
            dup[g] += scale * np.outer(p[r], u[r])
    return dx, ddown, dup, p.T @ x, p.sum(0)


def e4m3_table():
    """The 256 values of the format, from its definition."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        s = -1.0 if c & 128 else 1.0
        v[c] = np.nan if (c & 127) == 127 else s * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return v


def encode(x):
    """(codes, exponents) of the checkpoint of x, by a search among the format's values."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    mags = e4m3_table()[:127]
    codes = np.full((rows, blocks * BLOCK), 0x80, np.uint8)
    exps = np.empty((rows, blocks), np.uint8)
    for r in range(rows):
        for b in range(blocks):
            v = x[r, b * BLOCK:(b + 1) * BLOCK]
            amax = max([abs(t) for t in v if np.isfinite(t)], default=0.0)
            k = -117
            while amax > 448 * 2.0 ** k:
                k += 1
            k = min(k, 120)
            exps[r, b] = k + 127
            for i, t in enumerate(v):
                if not np.isfinite(t):
                    codes[r, b * BLOCK + i] = 0xff
                    continue
                d = np.abs(mags - abs(t) * 2.0 ** -k)
                near = np.flatnonzero(d == d.min())
                c = int(near[0] if len(near) == 1 or near[0] % 2 == 0 else near[1])   # ties to the even mantissa
                if k == 120:
                    c = min(c, 0x77)   # 240: the next value, 256 * 2^120, is beyond float32 and bf16
                codes[r, b * BLOCK + i] = c if t > 0 else c | 0x80
    return codes, exps


def decode(codes, exps, cols):
    """The values as float32 has them: exact, except that codes of 256 and above at e = 120 (none that an encoder writes) stand for
    2^128 and more, past the largest float32 (2 - 2^-23) 2^127: infinities."""
    with np.errstate(over="ignore"):
        return _decode64(codes, exps, cols).astype(np.float32).astype(np.float64)


def _decode64(codes, exps, cols):
    return (e4m3_table()[codes] * np.repeat(2.0 ** (exps.astype(np.float64) - 127), BLOCK, axis=1))[:, :cols]
