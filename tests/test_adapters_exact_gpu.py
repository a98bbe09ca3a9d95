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


INF = float("inf")


def positive(dtype, exact, rows=70, k=72, n=40, rank=3, groups=6):
    """A layer all of whose numbers are positive (so that an infinity stays one in every sum that it enters) and, with `exact`, powers of two
    (whose parts behind the first eight bits are zero).  Rows 10 and 11 are of group 2, rows 12 and 13 have no adapter."""
    g = torch.Generator().manual_seed(5)

    def t(*s):
        z = torch.exp2(torch.randint(-3, 3, s, generator=g).float()) if exact else torch.rand(s, generator=g) + 0.25
        return z.to("cuda", dtype)
    of = torch.randint(0, groups, (rows,), generator=g, dtype=torch.int32)
    of[10:12], of[12:14] = 2, -1
    y = t(rows, n) * torch.where(torch.rand((rows, n), generator=g) < 0.5, -1.0, 1.0).to("cuda", dtype)
    return dict(x=t(rows, k), w=t(n, k), b=t(n), down=t(groups, rank, k), up=t(groups, n, rank), dy=t(rows, n), y=y, low=t(rows, rank).float(), of=of.cuda())


def forward_of(ad, c):
    shared = ad.SharedProjection(c["w"], c["b"])
    plan = ad.group_rows(c["of"], len(c["down"]))
    y, low, _ = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, 0.01)
    few = ad.adapted_linear(c["x"][8:24], shared, c["down"], c["up"], c["of"][8:24].contiguous(), SCALE, 0.01)     # (without a plan)
    return {"y": y, "few": few, "low": low}


def backward_of(ad, c, slope=0.01):
    shared = ad.SharedProjection(c["w"], c["b"])
    plan = ad.group_rows(c["of"], len(c["down"]))
    out = ad.adapted_linear_backward(c["dy"], c["x"], c["y"], c["low"], shared, c["down"], c["up"], plan, SCALE, slope)
    dw, db = ad.checkpoint_weight_grad(c["dy"], ad.checkpoint8(torch.ones_like(c["x"])), c["y"] if slope is not None else None, slope)
    return dict(zip(("dx", "ddown", "dup"), out), dw=dw, db=db)


def check(got, clean, want):
    """Every result is the clean one, bit for bit, but for what `want` says: {name: index of the elements that are +infinity}."""
    for name, z in clean.items():
        z = z.clone()
        for at in want.get(name, ()):
            z[at] = INF
        bad = ~((got[name] == z) | (torch.isnan(got[name]) & torch.isnan(z)))
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, such as {got[name][bad][:3].tolist()} for {z[bad][:3].tolist()}"


def run_infinities(ad, dtype, exact, places, slope=0.01):
    """Infinities at `places`, {tensor: index}: what they reach is infinite in the formulas, and nothing else is touched."""
    c = positive(dtype, exact)
    forward, backward = forward_of(ad, c), backward_of(ad, c, slope)
    c = {k: v.clone() for k, v in c.items()}
    of = c["of"].cpu()
    fw, bw = {k: [] for k in forward}, {k: [] for k in backward}

    def reach(rows, cols):      # of y
        fw["y"].append((rows, cols))
        few = [int(r) - 8 for r in torch.arange(len(of))[rows].tolist() if 8 <= r < 24]
        fw["few"].append((few, cols))
    every = slice(None)
    for name, at in places.items():
        c[name][at] = INF
        if name == "x":
            r, k = at
            reach([r], every)
            if of[r] >= 0:
                fw["low"].append((r,))
                bw["ddown"].append((int(of[r]), every, k))
        elif name == "w":
            reach(slice(0, len(of)), at[0])
            bw["dx"].append((every, at[1]))
        elif name == "b":
            reach(slice(0, len(of)), at[0])
        elif name == "down":
            rows = torch.nonzero(of == at[0])[:, 0]
            fw["low"].append((rows, at[1]))
            reach(rows, every)
            bw["dx"].append((rows, at[2]))
        elif name == "up":
            rows = torch.nonzero(of == at[0])[:, 0]
            reach(rows, at[1])
            bw["dx"].append((rows, every))
            bw["ddown"].append((at[0], at[2]))
        elif name == "dy":
            bw["dx"].append((at[0], every))
            bw["dw"].append((at[1], every))
            bw["db"].append((at[1],))
            if of[at[0]] >= 0:
                bw["ddown"].append((int(of[at[0]]),))
                bw["dup"].append((int(of[at[0]]), at[1]))
        elif name == "low":
            if of[at[0]] >= 0:
                bw["dup"].append((int(of[at[0]]), every, at[1]))
    check(forward_of(ad, c), forward, fw)
    check(backward_of(ad, c, slope), backward, bw)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("slope", [0.01, None])
@pytest.mark.parametrize("places", [{"x": (10, 3)}, {"x": (13, 3)}, {"dy": (10, 3)}, {"dy": (12, 5)}, {"b": (5,)}, {"low": (11, 2)}], ids=str)
def test_an_infinity_of_a_bf16_row(ad, places, slope, exact):
    """Ranks that end inside a tile, and rows without an adapter: the zeros that stand there do not meet the row's infinity."""
    run_infinities(ad, torch.bfloat16, exact, places, slope)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_an_adapter_have_no_low_product(ad, dtype):
    c = positive(dtype, False)
    c["x"][12, 3], c["x"][13, 5] = INF, float("nan")
    assert not forward_of(ad, c)["low"][12:14].any()


PLACES = [{"x": (10, 3)}, {"x": (13, 3)}, {"dy": (10, 3)}, {"dy": (12, 5)}, {"w": (5, 3)}, {"b": (5,)}, {"down": (2, 1, 3)}, {"up": (2, 5, 1)}, {"low": (11, 2)},
          {"x": (10, 3), "w": (5, 3)}, {"x": (10, 3), "down": (2, 1, 3)}, {"dy": (10, 3), "w": (3, 5)}, {"dy": (10, 3), "up": (2, 3, 1)}, {"down": (2, 1, 3), "up": (2, 5, 1)}]


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("slope", [0.01, None])
@pytest.mark.parametrize("places", PLACES, ids=str)
def test_an_infinity_of_float32(ad, places, slope, exact):
    """An infinity in any tensor, and two that meet: infinities where the formulas have them, no NaN; numbers whose later cuts are zero too."""
    run_infinities(ad, torch.float32, exact, places, slope)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("slope", [0.01, 0.5, None])
@pytest.mark.parametrize("places", PLACES, ids=str)
def test_an_infinity_of_bf16(ad, places, slope, exact):
    """bf16 weights and adapters are one plane, u, v and a masked p several, whose later ones are often zero."""
    run_infinities(ad, torch.bfloat16, exact, places, slope)


@pytest.mark.parametrize("dtype", TYPES)
def test_signs_and_zeros_beside_an_infinity(ad, dtype):
    """-inf, an infinity times zero (NaN in the formula) and two infinities of unlike sign (NaN)."""
    c = positive(dtype, True)
    rows = [10, 12]
    c["x"][rows, 3], c["w"][7, 3] = -INF, 0.0
    c["b"][:] = 0.0
    got = forward_of(ad, c)
    assert torch.isnan(got["y"][rows, 7]).all()
    rest = [i for i in range(40) if i != 7]
    assert (got["y"][rows][:, rest] == -INF).all() and (got["low"][10] == -INF).all()
    c["x"][rows, 9] = INF
    assert torch.isnan(forward_of(ad, c)["y"][rows]).all()


def test_encoding_with_adapters_that_require_a_gradient(ad):
    """(a user's own optimiser may have set that): encoding gives none, and is not refused."""
    from vamb_amd import encode
    rng = np.random.default_rng(4)
    loader = encode.make_dataloader(rng.random((40, 4)).astype(np.float32) + 0.1, rng.standard_normal((40, 103)).astype(np.float32),
                                    rng.integers(2000, 9000, 40), batchsize=32, destroy=False)
    a = encode.VAE(4, nhiddens=[32], nlatent=8, seed=1).adapters(3, rank=2)
    want = a.encode(loader, np.arange(40) % 3)
    for t in (*a.down, *a.up):
        t.requires_grad_()
    assert np.array_equal(a.encode(loader, np.arange(40) % 3), want)
