"""The adapters' operators through every tile of the projection and both forms of the gradients, at sizes that end inside tiles, against the 64-bit
definition (tests/adapter_oracle.py) on some of the rows and groups.  Which kernels a size takes is asserted, so that a changed rule cannot
leave one of them without a test.

Tolerances, of the sum of the magnitudes S: a float32 sum of m products m 2^-24; float32 operands' dropped cuts 2^-21; p of bf16 tensors 2^-16 where
the slope applies; and half a step of the result's type (2^-8 or 2^-24 of the value)."""
import ctypes

import numpy as np
import pytest
import torch

import adapter_oracle as ao

pytestmark = pytest.mark.gpu
SLOPE, SCALE = 0.01, 0.5
F32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NARROW, MID, WIDE = 0, 1, 2


@pytest.fixture(scope="module")
def ad():
    from vamb_amd import _lib, adapters
    _lib.require_gpu()
    return adapters


def choice(rows, groups, n, k, rank, dtype):
    from vamb_amd import _lib
    out = [ctypes.c_int() for _ in range(3)]
    _lib.check(_lib.load().vh_debug_adapt_choice(rows, groups, n, k, rank, 0 if dtype == torch.float32 else 1, *out))
    return tuple(o.value for o in out)


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, tol, what):
    bad = ~(np.abs(f64(got) - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(f64(got) - want) / np.maximum(tol, 1e-300)):.3g} times the tolerance"


# rows, k, n, rank, groups, dtype, forward tile, backward tile, waves of the gradients
CASES = [
    (3000, 154, 512, 20, 30, torch.bfloat16, MID, NARROW, 4),
    (9001, 304, 200, 24, 60, torch.bfloat16, MID, MID, 4),
    (9001, 200, 304, 40, 60, torch.bfloat16, MID, MID, 1),
    (40001, 264, 264, 9, 20, torch.bfloat16, WIDE, WIDE, 4),
    (70001, 300, 520, 24, 300, torch.bfloat16, WIDE, WIDE, 1),
    (70001, 520, 300, 40, 300, torch.bfloat16, WIDE, WIDE, 1),
    (70001, 304, 512, 16, 700, torch.bfloat16, WIDE, WIDE, 1),
    (65537, 300, 520, 32, 900, torch.bfloat16, WIDE, WIDE, 1),
    (66000, 136, 264, 64, 1500, torch.bfloat16, WIDE, WIDE, 1),
    (3000, 154, 512, 20, 30, torch.float32, MID, NARROW, 4),
    (9001, 300, 200, 32, 60, torch.float32, MID, MID, 4),
    (20001, 300, 520, 24, 200, torch.float32, MID, MID, 4),
    (20001, 520, 300, 64, 200, torch.float32, MID, MID, 1),
    (30001, 300, 520, 33, 900, torch.float32, MID, MID, 1),
]


@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_every_tile(ad, case, held):
    rows, k, n, rank, groups, dtype, *kernels = case
    assert choice(rows, groups, n, k, rank, dtype) == tuple(kernels)
    gen = torch.Generator(device="cuda").manual_seed(rows + rank)
    t = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    x, w, b, dy = t(rows, k), t(n, k) * k ** -0.5, t(n), t(rows, n)
    down, up = t(groups, rank, k) * k ** -0.5, t(groups, n, rank) * rank ** -0.5
    of = torch.randint(-1, groups, (rows,), generator=gen, device="cuda").to(torch.int32)
    of[::7][:1300] = 5                      # one group of several items (512 rows each; with fewer groups than 128, of 128)
    of[of == 9] = 8                         # and one without rows
    shared, plan = ad.SharedProjection(w, b), ad.group_rows(of, groups)
    y, low, y8 = ad.adapted_linear_train(x, shared, down, up, plan, SCALE, SLOPE)
    x8 = ad.checkpoint8(x)
    dx, ddown, dup = ad.adapted_linear_backward(dy, x8 if held else x, y8 if held else y, low, shared, down, up, plan, SCALE, SLOPE)
    without = ad.adapted_linear_backward(dy, x8 if held else x, y8 if held else y, low, shared, down, up, plan, SCALE, SLOPE, need_dx=False)
    assert without[0] is None and torch.equal(without[1], ddown) and torch.equal(without[2], dup)
    xv = x8.restore(dtype) if held else x   # (a checkpoint's values are exact in either type)

    # rows: the first and last tiles' and some between
    at = np.unique(np.concatenate([np.arange(20), np.random.default_rng(1).integers(0, rows, 160), np.arange(rows - 20, rows)]))
    it, g = torch.from_numpy(at).cuda(), of.cpu().numpy()[at]
    cut = 2.0 ** -21 if dtype == torch.float32 else 0.0
    pcut = 0.0 if dtype == torch.float32 else 2.0 ** -16
    args = [f64(z) for z in (x[it], w, b, down, up)]
    u, want = ao.forward(*args, g, SCALE, SLOPE)
    su, s = ao.forward(*(np.abs(z) for z in args), g, SCALE, None)
    close(low[it], u, (k + 8) * F32 * su + cut * su, "u")
    tol = ((2 * k + rank + 16) * F32 + cut) * s
    close(y[it], want, tol + HALF[dtype] * (np.abs(want) + tol), "y")
    p = np.where(f64(y[it]) > 0, f64(dy[it]), np.float64(np.float32(SLOPE)) * f64(dy[it]))
    wn, dn, un = args[1], args[3], args[4]
    want, s = p @ wn, np.abs(p) @ np.abs(wn)
    for i, q in enumerate(g):
        if 0 <= q:
            want[i] += SCALE * (p[i] @ un[q]) @ dn[q]
            s[i] += SCALE * (np.abs(p[i]) @ np.abs(un[q])) @ np.abs(dn[q])
    tol = ((2 * n + rank + 16) * F32 + cut + pcut) * s
    close(dx[it], want, tol + HALF[dtype] * (np.abs(want) + tol), "dx")

    # groups: the large one, the empty one, the first, the last and two more
    of = of.cpu().numpy()
    for q in (5, 9, 0, groups - 1, 8, groups // 2):
        mine = torch.from_numpy(np.flatnonzero(of == q)).cuda()
        if len(mine) == 0:
            assert not ddown[q].any() and not dup[q].any()
            continue
        assert q != 5 or len(mine) > (512 if groups >= 128 else 128)
        p = np.where(f64(y[mine]) > 0, f64(dy[mine]), np.float64(np.float32(SLOPE)) * f64(dy[mine]))
        xm, um, b_, m = f64(xv[mine]), f64(low[mine]), f64(up[q]), len(mine)
        v, sv = SCALE * p @ b_, SCALE * np.abs(p) @ np.abs(b_)
        want, s = v.T @ xm, sv.T @ np.abs(xm)
        tol = ((n + m + 16) * F32 + cut + pcut) * s
        close(ddown[q], want, tol + HALF[dtype] * (np.abs(want) + tol), f"ddown of {q}")
        want, s = SCALE * p.T @ um, SCALE * np.abs(p).T @ np.abs(um)
        tol = ((m + 16) * F32 + pcut) * s
        close(dup[q], want, tol + HALF[dtype] * (np.abs(want) + tol), f"dup of {q}")
    assert 9 not in of
