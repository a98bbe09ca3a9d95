"""The adapter and checkpoint operators on small exact cases: what a part is held in, infinities and NaN, refusals on the GPU.

Inputs are chosen so that the formulas' results are known without a rounding (or with one that is named), and so that a part which was held
in fewer bits, or met a zero that the formula does not have, is seen."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
SCALE = 0.5
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ad():
    from vamb_amd import _lib, adapters
    _lib.require_gpu()
    return adapters


def test_low_products_keep_all_their_bits(ad):
    """u = (1 + 2^-8 + 2^-20, 1 + 2^-8), B = (1, -1): y = scale 2^-20, and the same of v in the backward pass; nothing in it is rounded (bf16
    tensors).  (1 + 2^-20 alone would not do: its parts are 8 bits each.)"""
    rows, n, k = 20, 40, 72
    bf = lambda t: t.to("cuda", torch.bfloat16)  # noqa: E731
    x, dy = torch.zeros(rows, k), torch.zeros(rows, n)
    for t in (x, dy):
        t[:, 0], t[:, 1], t[:, 2] = 1.0, 2.0 ** -8, 2.0 ** -20
    down, up = torch.zeros(1, 2, k), torch.zeros(1, n, 2)
    down[0, :, :2], down[0, 0, 2] = 1.0, 1.0      # u as above
    up[0, :, 0], up[0, :, 1] = 1.0, -1.0
    shared = ad.SharedProjection(bf(torch.zeros(n, k)))
    groups = torch.zeros(rows, dtype=torch.int32, device="cuda")
    plan = ad.group_rows(groups, 1)
    want = SCALE * 2.0 ** -20
    for g in (groups, plan):
        assert (ad.adapted_linear(bf(x), shared, bf(down), bf(up), g, SCALE) == want).all()
    up[0] = 0.0
    up[0, :2, :], up[0, 2, 0] = 1.0, 1.0          # v = scale u
    down[0, 0], down[0, 1] = 1.0, -1.0
    dx, _, _ = ad.adapted_linear_backward(bf(dy), bf(x), None, torch.zeros(rows, 2, device="cuda"), shared, bf(down), bf(up), plan, SCALE)
    assert (dx == want).all()


def slope_case(ad, dtype, slope):
    """Pairs of rows: p is (slope, 1, ...) in the first of a pair (the slope applies to its first column) and (t, 0, ...) in the second, t the
    slope in the tensors' type; with these, sums that leave slope - t, which is below half a step of that type."""
    pairs, n, k = 20, 40, 72
    dy, y = torch.zeros(pairs, 2, n), torch.ones(pairs, 2, n)
    t = float(torch.tensor(slope).to(dtype))
    dy[:, 0, :2], dy[:, 1, 0] = 1.0, t
    y[:, 0, 0] = -1.0
    x = torch.zeros(pairs, 2, k)
    x[:, 0], x[:, 1] = 1.0, -1.0
    to = lambda z: z.reshape(2 * pairs, -1).to("cuda", dtype)  # noqa: E731
    return pairs, n, k, to(dy), to(y), to(x), t, float(np.float32(slope)) - t


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("slope", [0.01, 0.3])
def test_a_slope_leaves_dy_more_bits_than_it_had(ad, slope, held):
    """p = dy slope of bf16 tensors is held to 2^-16 of its size in every product of the backward pass (rounded to bf16 it would be 2^-8,
    and the sums below nothing)."""
    dtype = torch.bfloat16
    pairs, n, k, dy, y, x, t, rest = slope_case(ad, dtype, slope)
    rows = 2 * pairs
    plan = ad.group_rows(torch.zeros(rows, dtype=torch.int32, device="cuda"), 1)
    low = torch.ones(rows, 1, device="cuda")
    low[1::2] = -1.0
    w, down, up = torch.zeros(n, k), torch.zeros(1, 1, k), torch.zeros(1, n, 1)
    w[0], w[1] = 1.0, -t                              # p w: slope - t in a pair's first row, t in its second
    up[0, 0], up[0, 1] = 1.0, -t                      # v: the same, times the scale
    to = lambda z: z.to("cuda", dtype)  # noqa: E731
    shared, down, up = ad.SharedProjection(to(w)), to(down), to(up)
    ys, xs = (ad.checkpoint8(y), ad.checkpoint8(x)) if held else (y, x)
    dx, ddown, dup = ad.adapted_linear_backward(dy, xs, ys, low, shared, down, up, plan, SCALE, slope)
    tol = 2.0 ** -16 * slope + 2.0 ** -8 * abs(rest)  # p's bits, and the result's rounding
    assert ((dx[0::2].double() - rest).abs() <= tol).all() and (dx[1::2] == t).all()
    # dA = sum v x = scale pairs ((slope - t) - t)
    want = SCALE * pairs * (rest - t)
    assert ((ddown.double() - want).abs() <= SCALE * pairs * 2.0 ** -16 * slope + 2.0 ** -8 * abs(want)).all()
    # dB of the first column = scale sum p u = scale pairs (slope - t)
    assert ((dup[0, 0].double() - SCALE * pairs * rest).abs() <= SCALE * pairs * tol).all()
    assert (dup[0, 1] == SCALE * pairs).all() and not dup[0, 2:].any()


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("slope", [0.01, 0.3])
def test_weight_gradient_of_a_slope(ad, slope, held):
    pairs, n, k, dy, y, x, t, rest = slope_case(ad, torch.bfloat16, slope)
    dw, db = ad.checkpoint_weight_grad(dy, ad.checkpoint8(x), ad.checkpoint8(y) if held else y, slope)
    tol = 2.0 ** -16 * slope + 2.0 ** -8 * abs(rest)
    assert ((dw[0].double() - pairs * rest).abs() <= pairs * tol).all() and (dw[1] == pairs).all() and not dw[2:].any()
    total = pairs * (float(np.float32(slope)) + t)      # the sum of p itself is of float32 values
    assert abs(float(db[0]) - total) <= 2.0 ** -8 * total + 2 * pairs * 2.0 ** -24 * total and db[1] == pairs
