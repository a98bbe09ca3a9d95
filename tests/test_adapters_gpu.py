"""The adapter and checkpoint operators (vamb_amd.adapters) against their 64-bit definitions (tests/adapter_oracle.py).

Tolerances, element by element.  H = 2^-8 (bf16) or 2^-24 (float32): one rounding of the result.  A sum of m products in float32 is off by
at most m 2^-24 of the sum of the magnitudes; three cuts of a float32 drop products below 2^-22 of theirs; two cuts of u (bf16
tensors) keep it to 2^-15; a masked p of a bf16 backward pass is rounded to bf16 (2^-8).  `S` is the sum of the magnitudes, from the
oracle run on absolute values."""
import numpy as np
import pytest
import torch

import adapter_oracle as ao

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SLOPE, SCALE = 0.01, 0.5
TYPES = [torch.float32, torch.bfloat16]

# rows, k, n, rank, groups
SHAPES = [
    (1, 1, 1, 1, 1), (1, 304, 512, 8, 200), (5, 107, 33, 3, 2), (16, 64, 128, 16, 4), (17, 8, 16, 1, 20), (63, 154, 130, 64, 7),
    (257, 512, 32, 17, 50), (300, 65, 257, 16, 1), (1000, 40, 256, 5, 300), (700, 33, 36, 4, 3000), (2049, 96, 64, 33, 3),
    (17000, 24, 40, 4, 5), (3000, 31, 20, 2, 16384),
]


@pytest.fixture(scope="module")
def ad():
    from vamb_amd import _lib, adapters
    _lib.require_gpu()
    return adapters


def f64(t):
    return t.detach().double().cpu().numpy()


def groups_for(rng, rows, groups, order):
    g = rng.integers(-1, groups, rows)
    if rows > 3:
        g[rng.integers(0, rows)] = groups + 5      # outside: no adapter
        g[rng.integers(0, rows)] = -(2 ** 31)
    if order == "sorted":
        g = np.sort(g)
    return g.astype(np.int32)


def make(seed, dtype, rows, k, n, rank, groups, order="shuffled", bias=True):
    rng = np.random.default_rng(seed)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to("cuda", dtype)  # noqa: E731
    c = dict(x=t(rows, k), w=t(n, k) * k ** -0.5, b=t(n) if bias else None, down=t(groups, rank, k) * k ** -0.5, up=t(groups, n, rank) * rank ** -0.5,
             dy=t(rows, n), g=groups_for(rng, rows, groups, order))
    c["groups"] = torch.from_numpy(c["g"]).cuda()
    return c


def close(got, want, tol, what):
    got = f64(got)
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} times the tolerance"


def forward_bounds(c, dtype, slope):
    """(u, y, tolerance of u, tolerance of y)."""
    a = [np.abs(f64(c[i])) if c[i] is not None else None for i in ("x", "w", "b", "down", "up")]
    u, y = ao.forward(f64(c["x"]), f64(c["w"]), None if c["b"] is None else f64(c["b"]), f64(c["down"]), f64(c["up"]), c["g"], SCALE, slope)
    su, sy = ao.forward(*a, c["g"], SCALE, None)
    k, rank = c["x"].shape[1], c["down"].shape[1]
    tu = (k + 8) * F32 * su + 2.0 ** -22 * su
    cut = 2.0 ** -15 if dtype == torch.bfloat16 else 0
    ty = ((2 * k + rank + 16) * F32 + 2.0 ** -21 + cut) * sy
    return u, y, tu, ty + HALF[dtype] * (np.abs(y) + ty)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(ad, shape, dtype):
    rows, k, n, rank, groups = shape
    for seed, (order, slope, bias) in enumerate([("shuffled", SLOPE, True), ("sorted", None, False)]):
        c = make(seed + 7, dtype, *shape, order=order, bias=bias)
        u, y, tu, ty = forward_bounds(c, dtype, slope)
        shared = ad.SharedProjection(c["w"], c["b"])
        got = ad.adapted_linear(c["x"], shared, c["down"], c["up"], c["groups"], SCALE, slope)
        close(got, y, ty, "y")
        plan = ad.group_rows(c["groups"], groups)
        got, low, held = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, slope)
        close(got, y, ty, "y with a plan")
        close(low, u, tu, "u")
        again = ad.checkpoint8(got)     # the checkpoint that the launch wrote is that of the rounded y
        assert torch.equal(held.codes, again.codes) and torch.equal(held.exponents, again.exponents)
        assert torch.equal(ad.adapted_linear(c["x"], shared, c["down"], c["up"], plan, SCALE, slope), got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 512, 40, 64, 3), (2, 1104, 33, 16, 9), (3, 100, 512, 30, 2), (16, 65, 17, 8, 200), (33, 32, 16, 1, 1000), (60, 304, 512, 8, 4)])
def test_few_rows(ad, shape, dtype, monkeypatch):
    """The launch without a plan, whatever the number of rows; and that both ways give the same layer."""
    monkeypatch.setattr(ad, "_FEW", {t: 10 ** 12 for t in TYPES})
    c = make(80, dtype, *shape)
    u, y, tu, ty = forward_bounds(c, dtype, SLOPE)
    shared = ad.SharedProjection(c["w"], c["b"])
    got = ad.adapted_linear(c["x"], shared, c["down"], c["up"], c["groups"], SCALE, SLOPE)
    close(got, y, ty, "y")
    monkeypatch.setattr(ad, "_FEW", {t: 0 for t in TYPES})
    close(ad.adapted_linear(c["x"], shared, c["down"], c["up"], c["groups"], SCALE, SLOPE), y, ty, "y with a plan")


@pytest.mark.parametrize("dtype", TYPES)
def test_plan_sorts_stably_and_covers_every_row(ad, dtype):
    if dtype != torch.float32:
        pytest.skip("the plan has no type")
    rng = np.random.default_rng(3)
    for rows, groups in [(1, 1), (15, 3), (16, 1), (1024, 7), (16384, 1000), (16385, 1000), (5000, 5000), (40001, 1), (70000, 16384), (300000, 33)]:
        g = groups_for(rng, rows, groups, "sorted" if rows % 3 == 1 else "shuffled")
        plan = ad.group_rows(torch.from_numpy(g).cuda(), groups).plan.cpu().numpy()
        n_sub = int(plan[0])
        o_sub = 16 + 16 * (rows // 16 + min(groups + 1, rows))
        slots, subs = plan[16:16 + 16 * n_sub], plan[o_sub:o_sub + n_sub]
        key = np.where((g >= 0) & (g < groups), g, groups)
        counts = np.bincount(key, minlength=groups + 1)
        want = np.full(16 * n_sub, -1)
        order, at = np.argsort(key, kind="stable"), 0
        starts = np.cumsum(counts) - counts
        for q in np.flatnonzero(counts):
            want[at:at + counts[q]] = order[starts[q]:starts[q] + counts[q]]
            assert (subs[at // 16:(at + counts[q] + 15) // 16] == (q if q < groups else -1)).all()
            at += -(-counts[q] // 16) * 16
        assert at == 16 * n_sub
        assert np.array_equal(slots, want), (rows, groups)
        o_item = (o_sub + rows // 16 + min(groups + 1, rows) + 3) // 4 * 4
        items = plan[o_item:o_item + 4 * int(plan[1])].reshape(-1, 4)
        assert np.array_equal(np.bincount(items[:, 0], weights=items[:, 2], minlength=groups), counts[:groups])
        assert set(items[:, 0]) == set(range(groups))


def backward_bounds(c, x, y, u, dtype, slope):
    w, down, up, dy = (f64(c[i]) for i in ("w", "down", "up", "dy"))
    args = lambda f: (f(dy), f(x), y, f(u), f(w), f(down), f(up), c["g"], SCALE, slope)  # noqa: E731
    want = ao.backward(*args(lambda t: t))
    mag = ao.backward(*args(np.abs))
    rows, n = dy.shape
    rank = down.shape[1]
    # p rounded to bf16 where the slope was applied: at most 2^-8 of its magnitude in every product that has it
    p = 2.0 ** -8 if dtype == torch.bfloat16 and slope is not None else 0.0
    cut = 2.0 ** -15 if dtype == torch.bfloat16 else 0.0
    rel = {"dx": (2 * n + rank + 16) * F32 + 2.0 ** -21 + cut + p, "ddown": (n + rows + 16) * F32 + 2.0 ** -21 + p, "dup": (rows + 16) * F32 + p,
           "dw": (rows + 16) * F32 + 2.0 ** -21 + p, "db": (rows + 16) * F32}
    out = {}
    for name, v, m in zip(("dx", "ddown", "dup", "dw", "db"), want, mag):
        t = rel[name] * m
        out[name] = (v, t + HALF[dtype] * (np.abs(v) + t))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(ad, shape, dtype):
    rows, k, n, rank, groups = shape
    for seed, (order, slope, held) in enumerate([("shuffled", SLOPE, True), ("sorted", None, True), ("shuffled", SLOPE, False)]):
        c = make(seed + 70, dtype, *shape, order=order)
        shared = ad.SharedProjection(c["w"], c["b"])
        plan = ad.group_rows(c["groups"], groups)
        y, low, y8 = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, slope)
        x8 = ad.checkpoint8(c["x"])
        xs, ys = (x8, y8) if held else (c["x"], y)
        xv = f64(x8.restore()) if held else f64(c["x"])
        want = backward_bounds(c, xv, f64(y), f64(low), dtype, slope)
        dx, ddown, dup = ad.adapted_linear_backward(c["dy"], xs, ys, low, shared, c["down"], c["up"], plan, SCALE, slope)
        close(dx, *want["dx"], "dx")
        close(ddown, *want["ddown"], "ddown")
        close(dup, *want["dup"], "dup")
        none, d2, u2 = ad.adapted_linear_backward(c["dy"], xs, ys, low, shared, c["down"], c["up"], plan, SCALE, slope, need_dx=False)
        assert none is None and torch.equal(d2, ddown) and torch.equal(u2, dup)
        if held:
            dw, db = ad.checkpoint_weight_grad(c["dy"], x8, y8 if slope is not None else None, slope)
            close(dw, *want["dw"], "dw")
            close(db, *want["db"], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 8, 1), (63, 40, 33), (129, 33, 130), (700, 136, 300), (257, 257, 31), (320, 128, 128)])
def test_weight_gradient_of_every_kind_of_mask(ad, dtype, rows, n, k):
    """Masks as elements and as codes are the same mask, bit for bit; what stands beside the rows of dy and y enters nothing."""
    c = make(90, dtype, rows, k, n, 1, 1)
    x8 = ad.checkpoint8(c["x"])
    y = make(91, dtype, rows, k, n, 1, 1)["dy"]
    beside = [torch.full((rows, n + 8), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    dy, ys = (b[:, :n].copy_(t) for b, t in zip(beside, (c["dy"], y)))
    got = ad.checkpoint_weight_grad(dy, x8, ys, SLOPE)
    held = ad.checkpoint_weight_grad(c["dy"], x8, ad.checkpoint8(y), SLOPE)
    assert all(torch.equal(a, b) for a, b in zip(got, held))
    for slope, (dw, db) in ((SLOPE, got), (None, ad.checkpoint_weight_grad(dy, x8))):
        want = backward_bounds(c, f64(x8.restore()), f64(y), np.zeros((rows, 1)), dtype, slope)
        close(dw, *want["dw"], "dw")
        close(db, *want["db"], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (7, 32), (5, 33), (64, 154), (9, 512), (2, 1104)])
def test_checkpoint(ad, rows, cols, dtype):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = torch.from_numpy((rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-30, 30, (rows, 1)))).astype(np.float32)).to("cuda", dtype)
    x[0, 0] = 0.0
    x[rows - 1, cols - 1] = -0.0
    held = ad.checkpoint8(x)
    codes, exps = ao.encode(f64(x))
    assert np.array_equal(held.codes.cpu().numpy(), codes) and np.array_equal(held.exponents.cpu().numpy(), exps)
    for t in TYPES:
        assert np.array_equal(f64(held.restore(t)), ao.decode(codes, exps, cols))


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpoint_of_extreme_values(ad, dtype):
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    rows = [[0.0] * 40, [top, -top, 1.0, 0.0] * 10, [tiny, -tiny, tiny / 4, 0.0] * 10, [float("inf"), 1.0, -2.0, float("nan")] * 10, [float("nan")] * 40,
            [448.0, 449.0, 1.75, -1e-30] * 10, [2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133] * 40, [1.0, 2.0 ** -9, 2.0 ** -10, -2.0 ** -11] * 10,
            [448.0, 2.0 ** -10, 3 * 2.0 ** -10, -2.0 ** -10] * 10, [240.0, 248.0, 232.0, 17.0] * 10]
    x = torch.tensor(rows, dtype=torch.float32).to("cuda", dtype)
    held = ad.checkpoint8(x)
    codes, exps = ao.encode(f64(x))
    assert np.array_equal(held.exponents.cpu().numpy(), exps)
    assert np.array_equal(held.codes.cpu().numpy(), codes)
    for t in TYPES:
        got, want = f64(held.restore(t)), ao.decode(codes, exps, 40)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


def test_all_codes_restore_exactly(ad):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(1, 256).repeat(3, 1).contiguous()
    for byte in (10, 127, 247):
        held = ad.Checkpoint8(codes, torch.full((3, 8), byte, dtype=torch.uint8, device="cuda"), 256)
        want = ao.decode(codes.cpu().numpy(), held.exponents.cpu().numpy(), 256)
        for t in TYPES:
            got = f64(held.restore(t))
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_tensors(ad, dtype):
    rows, k, n, rank, groups = 130, 48, 64, 8, 5
    c = make(5, dtype, rows, k, n, rank, groups)
    shared = ad.SharedProjection(c["w"], c["b"])
    plan = ad.group_rows(c["groups"], groups)
    want = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, SLOPE)
    x8, y8 = ad.checkpoint8(c["x"]), want[2]
    grads = ad.adapted_linear_backward(c["dy"], x8, y8, want[1], shared, c["down"], c["up"], plan, SCALE, SLOPE)
    wgrads = ad.checkpoint_weight_grad(c["dy"], x8, y8, SLOPE)
    for pad, off in [(16, 8), (3, 1), (1, 0), (8, 5)]:
        def view(t):
            big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=dtype, device="cuda")
            v = big[:, off:off + t.shape[1]] if off + t.shape[1] <= big.shape[1] else big[:, :t.shape[1]]
            v.copy_(t)
            return v
        x, dy, y = view(c["x"]), view(c["dy"]), view(want[0])
        got = ad.adapted_linear_train(x, ad.SharedProjection(view(c["w"]), c["b"]), c["down"], c["up"], plan, SCALE, SLOPE)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        few = ad.adapted_linear(x[:40], shared, c["down"], c["up"], c["groups"][:40], SCALE, SLOPE)
        assert torch.equal(few, ad.adapted_linear(c["x"][:40], shared, c["down"], c["up"], c["groups"][:40], SCALE, SLOPE))
        xx = ad.checkpoint8(x)
        assert torch.equal(xx.codes, x8.codes)
        for a, b in zip(ad.adapted_linear_backward(dy, xx, y, want[1], shared, c["down"], c["up"], plan, SCALE, SLOPE), grads):
            assert torch.equal(a, b)
        for a, b in zip(ad.checkpoint_weight_grad(dy, xx, y, SLOPE), wgrads):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_values_stay_in_their_row(ad, dtype):
    rows, k, n, rank, groups = 100, 64, 64, 4, 6
    c = make(6, dtype, rows, k, n, rank, groups)
    c["groups"][10] = 2
    shared = ad.SharedProjection(c["w"], c["b"])
    for take in (slice(0, rows), slice(0, 50)):
        g = c["groups"][take].contiguous()
        clean = ad.adapted_linear(c["x"][take], shared, c["down"], c["up"], g, SCALE)
        x = c["x"][take].clone()
        x[10, 3] = float("nan")
        x[11, 5] = float("inf")
        got = ad.adapted_linear(x, shared, c["down"], c["up"], g, SCALE)
        rest = [i for i in range(len(x)) if i not in (10, 11)]
        assert torch.equal(got[rest], clean[rest])
        assert torch.isnan(got[10]).all() and not torch.isfinite(got[11]).any()
    # an adapter that no row asks for is not touched
    down = c["down"].clone()
    used = c["groups"].clone()
    used[used == 4] = 1
    down[4] = float("nan")
    assert torch.isfinite(ad.adapted_linear(c["x"], shared, down, c["up"], used, SCALE)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(ad, dtype):
    c = make(1, dtype, 4, 40, 36, 3, 5)
    shared = ad.SharedProjection(c["w"])
    empty = c["x"][:0]
    plan = ad.group_rows(c["groups"][:0], 5)
    assert ad.adapted_linear(empty, shared, c["down"], c["up"], c["groups"][:0]).shape == (0, 36)
    y, low, held = ad.adapted_linear_train(empty, shared, c["down"], c["up"], plan)
    assert y.shape == (0, 36) and low.shape == (0, 3) and held.shape == (0, 36)
    assert held.restore().shape == (0, 36)
    dx, ddown, dup = ad.adapted_linear_backward(y, ad.checkpoint8(empty), None, low, shared, c["down"], c["up"], plan)
    assert dx.shape == (0, 40) and not ddown.any() and not dup.any()
    dw, db = ad.checkpoint_weight_grad(y, ad.checkpoint8(empty))
    assert dw.shape == (36, 40) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_adapters_are_the_plain_layer(ad, dtype):
    c = make(2, dtype, 90, 40, 72, 3, 5)
    none = torch.full((90,), -1, dtype=torch.int32, device="cuda")
    shared = ad.SharedProjection(c["w"], c["b"])
    c["g"] = none.cpu().numpy()
    plan = ad.group_rows(none, 5)
    u, y, tu, ty = forward_bounds(c, dtype, SLOPE)
    got, low, y8 = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, SLOPE)
    close(got, y, ty, "y")
    assert not low.any()
    dx, ddown, dup = ad.adapted_linear_backward(c["dy"], c["x"], y8, low, shared, c["down"], c["up"], plan, SCALE, SLOPE)
    assert not ddown.any() and not dup.any() and dx.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_inputs_give_equal_bits(ad, dtype):
    c = make(9, dtype, 5000, 200, 130, 12, 3)
    shared = ad.SharedProjection(c["w"], c["b"])

    def once():
        plan = ad.group_rows(c["groups"], 3)
        y, low, y8 = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, SLOPE)
        x8 = ad.checkpoint8(c["x"])
        return (y, low, y8.codes, *ad.adapted_linear_backward(c["dy"], x8, y8, low, shared, c["down"], c["up"], plan, SCALE, SLOPE),
                *ad.checkpoint_weight_grad(c["dy"], x8, y8, SLOPE))
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_gradients_against_differences(ad):
    """The backward pass against central differences of the forward pass (float32, a smooth region of the loss)."""
    rows, k, n, rank, groups = 40, 24, 20, 3, 4
    c = make(12, torch.float32, rows, k, n, rank, groups)
    shared = ad.SharedProjection(c["w"], c["b"])
    plan = ad.group_rows(c["groups"], groups)
    y, low, _ = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, None)
    dx, ddown, dup = ad.adapted_linear_backward(c["dy"], c["x"], None, low, shared, c["down"], c["up"], plan, SCALE, None)
    rng = np.random.default_rng(0)
    for name, grad in (("x", dx), ("down", ddown), ("up", dup)):
        way = torch.from_numpy(rng.standard_normal(tuple(c[name].shape)).astype(np.float32)).cuda()
        h = 2.0 ** -6
        args = lambda s: [c[i] + s * h * way if i == name else c[i] for i in ("x", "down", "up")]  # noqa: E731
        f = [float((ad.adapted_linear(a[0], shared, a[1], a[2], plan, SCALE).double() * c["dy"].double()).sum()) for a in (args(1), args(-1))]
        want, got = (f[0] - f[1]) / (2 * h), float((grad.double() * way.double()).sum())
        # the loss is linear in each of the three: no truncation term, only the roundings of y (K 2^-24 of about |dy| |y| sqrt(rows n)) over h
        size = float((y.double().abs() * c["dy"].double().abs()).sum())
        assert abs(got - want) <= 64 * F32 * size / h + 1e-4 * abs(want), name


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(ad, dtype):
    c = make(21, dtype, 600, 64, 96, 8, 40)
    shared = ad.SharedProjection(c["w"], c["b"])

    def step():
        plan = ad.group_rows(c["groups"], 40)
        x8 = ad.checkpoint8(c["x"])
        y, low, y8 = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, SLOPE)
        few = ad.adapted_linear(c["x"][:20], shared, c["down"], c["up"], c["groups"][:20], SCALE, SLOPE)
        return (y, few, y8.restore(dtype), *ad.adapted_linear_backward(c["dy"], x8, y8, low, shared, c["down"], c["up"], plan, SCALE, SLOPE),
                *ad.checkpoint_weight_grad(c["dy"], x8, y8, SLOPE))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    rng = np.random.default_rng(2)
    for _ in range(3):
        c["x"].copy_(torch.from_numpy(rng.standard_normal((600, 64)).astype(np.float32)))
        c["groups"].copy_(torch.from_numpy(groups_for(rng, 600, 40, "shuffled")))
        for graph, out in zip(graphs, outs):
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(300, 96), (129, 130), (640, 200)])
def test_large_batches_take_the_wide_tiles(ad, dtype, n, k):
    """Enough rows for the widest tiles, and widths that end inside one, in both directions."""
    rows, rank, groups = 70000, 20 if n == 300 else 9, 300
    c = make(50, dtype, rows, k, n, rank, groups, order="sorted")
    shared = ad.SharedProjection(c["w"], c["b"])
    plan = ad.group_rows(c["groups"], groups)
    y, low, y8 = ad.adapted_linear_train(c["x"], shared, c["down"], c["up"], plan, SCALE, SLOPE)
    dx, _, _ = ad.adapted_linear_backward(c["dy"], c["x"], y, low, shared, c["down"], c["up"], plan, SCALE, SLOPE)
    rng = np.random.default_rng(0)
    at = np.concatenate([np.arange(40), rng.integers(0, rows, 200), np.arange(rows - 40, rows)])
    t = torch.from_numpy(at).cuda()
    part = dict(c, x=c["x"][t], dy=c["dy"][t], g=c["g"][at])
    u, want, tu, ty = forward_bounds(part, dtype, SLOPE)
    close(y[t], want, ty, "y")
    close(low[t], u, tu, "u")
    value, tol = backward_bounds(part, f64(part["x"]), f64(y[t]), f64(low[t]), dtype, SLOPE)["dx"]
    close(dx[t], value, tol, "dx")
    again = ad.checkpoint8(y)
    assert torch.equal(y8.codes, again.codes) and torch.equal(y8.exponents, again.exponents)


def test_two_streams_at_once(ad):
    c = [make(30 + i, torch.bfloat16, 4000, 128, 128, 16, 60) for i in range(2)]
    shared = [ad.SharedProjection(d["w"], d["b"]) for d in c]

    def step(i):
        d = c[i]
        plan = ad.group_rows(d["groups"], 60)
        y, low, y8 = ad.adapted_linear_train(d["x"], shared[i], d["down"], d["up"], plan, SCALE, SLOPE)
        return (y, *ad.adapted_linear_backward(d["dy"], ad.checkpoint8(d["x"]), y8, low, shared[i], d["down"], d["up"], plan, SCALE, SLOPE))
    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for o in got[i] for a, b in zip(o, want[i]))


def test_row_offsets_beyond_32_bits(ad):
    """x of more than 2^31 elements: rows at the end of it are read and written where they are."""
    rows, k, n = 2_200_000, 1024, 16     # 2.25e9 elements of bf16: 4.5 GB
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    g = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(1)
    x[-3:] = torch.from_numpy(rng.standard_normal((3, k)).astype(np.float32)).to("cuda", torch.bfloat16)
    g[-2:] = 1
    c = make(40, torch.bfloat16, 3, k, n, 4, 2)
    shared = ad.SharedProjection(c["w"], None)
    y = ad.adapted_linear(x, shared, c["down"], c["up"], g, SCALE)
    want = ad.adapted_linear(x[-3:], shared, c["down"], c["up"], ad.group_rows(g[-3:].contiguous(), 2), SCALE)
    assert torch.equal(y[-3:], want) and not y[:-3].any()
    held = ad.checkpoint8(x)
    assert torch.equal(held.codes[-3:], ad.checkpoint8(x[-3:]).codes)
    plan = ad.group_rows(g, 2)
    dy = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    dy[-3:] = c["dy"]
    low = torch.zeros((rows, 4), device="cuda")
    low[-3:] = 1.0
    dx, ddown, dup = ad.adapted_linear_backward(dy, held, None, low, shared, c["down"], c["up"], plan, SCALE)
    small = ad.adapted_linear_backward(c["dy"], ad.checkpoint8(x[-3:]), None, low[-3:].contiguous(), shared, c["down"], c["up"],
                                       ad.group_rows(g[-3:].contiguous(), 2), SCALE)
    assert torch.equal(dx[-3:], small[0]) and torch.equal(ddown[1], small[1][1]) and torch.equal(dup[1], small[2][1])
    assert not dx[:-3].any() and not ddown[0].any()
