"""What vamb_amd.adapters and its C entries refuse: checked before any device work, so on any machine."""
import ctypes

import numpy as np
import pytest
import torch

import adapter_oracle as ao
from vamb_amd import _lib, adapters as ad

ROWS, K, N, RANK, GROUPS = 6, 40, 36, 3, 5


class _Shared(ad.SharedProjection):
    """A projection that was never packed (no GPU here)."""

    def __init__(self, dtype=torch.float32):
        self.n, self.k, self.dtype, self.device = N, K, dtype, torch.device("cpu")
        self.packed = torch.zeros(16, dtype=torch.uint8)


def args(**kw):
    a = dict(x=torch.zeros(ROWS, K), shared=_Shared(), down=torch.zeros(GROUPS, RANK, K), up=torch.zeros(GROUPS, N, RANK),
             groups=torch.zeros(ROWS, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,why", [
    (dict(x=torch.zeros(ROWS, K + 1)), "x must be"),
    (dict(x=torch.zeros(K)), "two-dimensional"),
    (dict(x=torch.zeros(K, ROWS).t()), "contiguous"),
    (dict(x=torch.zeros(1, K).expand(ROWS, K)), "overlap"),
    (dict(x=torch.zeros(ROWS, K, dtype=torch.float16)), "type"),
    (dict(x=torch.zeros(ROWS, K, dtype=torch.bfloat16)), "type"),
    (dict(shared="W"), "SharedProjection"),
    (dict(down=torch.zeros(GROUPS, RANK, K + 1)), "down must be"),
    (dict(down=torch.zeros(GROUPS, K, RANK).transpose(1, 2)), "contiguous"),
    (dict(down=torch.zeros(GROUPS, 0, K)), "rank"),
    (dict(down=torch.zeros(GROUPS, 65, K), up=torch.zeros(GROUPS, N, 65)), "rank"),
    (dict(down=torch.zeros(RANK, K)), "groups, rank, k"),
    (dict(up=torch.zeros(GROUPS, N, RANK + 1)), "up must be"),
    (dict(up=torch.zeros(GROUPS, N, RANK, dtype=torch.bfloat16)), "type"),
    (dict(groups=torch.zeros(ROWS, dtype=torch.int64)), "int32"),
    (dict(groups=torch.zeros(ROWS + 1, dtype=torch.int32)), "rows"),
    (dict(groups=torch.zeros(2 * ROWS, dtype=torch.int32)[::2]), "contiguous"),
    (dict(groups=ad.RowGroups(ROWS, GROUPS + 1, None)), "adapters"),
    (dict(groups=ad.RowGroups(ROWS + 1, GROUPS, None)), "rows"),
    (dict(scale=float("nan")), "scale"),
    (dict(negative_slope=-0.1), "negative_slope"),
    (dict(negative_slope=float("inf")), "negative_slope"),
    (dict(), "on a GPU"),
])
def test_forward_refuses(change, why):
    with pytest.raises(ValueError, match=why):
        ad.adapted_linear(**args(**change))


def test_training_forward_wants_a_plan():
    with pytest.raises(ValueError, match="group_rows"):
        ad.adapted_linear_train(**args())


def held(rows=ROWS, cols=K):
    b = -(-cols // 32)
    return ad.Checkpoint8(torch.zeros(rows, 32 * b, dtype=torch.uint8), torch.zeros(rows, b, dtype=torch.uint8), cols)


def backward_args(**kw):
    a = dict(dy=torch.zeros(ROWS, N), x=held(), y=held(ROWS, N), low=torch.zeros(ROWS, RANK), shared=_Shared(), down=torch.zeros(GROUPS, RANK, K),
             up=torch.zeros(GROUPS, N, RANK), groups=ad.RowGroups(ROWS, GROUPS, torch.zeros(64, dtype=torch.int32)), negative_slope=0.01)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,why", [
    (dict(dy=torch.zeros(ROWS, N + 1)), "dy must be"),
    (dict(dy=torch.zeros(ROWS, N, dtype=torch.bfloat16)), "dy must have"),
    (dict(x=held(ROWS, K + 1)), "checkpoint x"),
    (dict(x=held(ROWS + 1, K)), "checkpoint x"),
    (dict(x=torch.zeros(ROWS, K, dtype=torch.bfloat16)), "x must be"),
    (dict(y=None), "derivative"),
    (dict(y=torch.zeros(ROWS, K)), "y must be"),
    (dict(low=torch.zeros(ROWS, RANK + 1)), "low must be"),
    (dict(low=torch.zeros(ROWS, RANK, dtype=torch.bfloat16)), "float32"),
    (dict(groups=torch.zeros(ROWS, dtype=torch.int32)), "group_rows"),
    (dict(), "on a GPU"),
])
def test_backward_refuses(change, why):
    with pytest.raises(ValueError, match=why):
        ad.adapted_linear_backward(**backward_args(**change))


def test_others_refuse():
    for call, why in [
        (lambda: ad.group_rows(torch.zeros(3), 2), "int32"),
        (lambda: ad.group_rows(torch.zeros(3, dtype=torch.int32), 0), "number of groups"),
        (lambda: ad.group_rows(torch.zeros(3, dtype=torch.int32), 16385), "number of groups"),
        (lambda: ad.group_rows(torch.zeros(3, dtype=torch.int32), 2), "on a GPU"),
        (lambda: ad.SharedProjection(torch.zeros(0, 3)), "empty"),
        (lambda: ad.SharedProjection(torch.zeros(3, 3, dtype=torch.float64)), "float32 or bfloat16"),
        (lambda: ad.SharedProjection(torch.zeros(3, 4), torch.zeros(4)), "bias"),
        (lambda: ad.SharedProjection(torch.zeros(3, 4), torch.zeros(3, dtype=torch.bfloat16)), "bias"),
        (lambda: ad.checkpoint8(torch.zeros(3, 4, dtype=torch.int32)), "float32 or bfloat16"),
        (lambda: ad.checkpoint8(torch.zeros(3, 0)), "one column"),
        (lambda: ad.checkpoint8(torch.zeros(3, 4)), "on a GPU"),
        (lambda: ad.Checkpoint8(torch.zeros(3, 40, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8), 40), "codes must be"),
        (lambda: ad.Checkpoint8(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 40), "exponents must be"),
        (lambda: ad.Checkpoint8(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 2), 40), "uint8"),
        (lambda: ad.Checkpoint8(torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 0), "one column"),
        (lambda: held().restore(torch.float16), "float32 or bfloat16"),
        (lambda: held().restore(), "on a GPU"),
        (lambda: ad.checkpoint_weight_grad(torch.zeros(ROWS, N), torch.zeros(ROWS, K)), "Checkpoint8"),
        (lambda: ad.checkpoint_weight_grad(torch.zeros(ROWS + 1, N), held()), "dy must be"),
        (lambda: ad.checkpoint_weight_grad(torch.zeros(ROWS, N), held(), None, 0.01), "derivative"),
        (lambda: ad.checkpoint_weight_grad(torch.zeros(ROWS, N), held(), held(ROWS, N), -1.0), "negative_slope"),
        (lambda: ad.checkpoint_weight_grad(torch.zeros(ROWS, N), held()), "on a GPU"),
    ]:
        with pytest.raises(ValueError, match=why):
            call()


def test_c_entries_refuse():
    """The library's own checks (a caller may bind it without this package)."""
    lib = _lib.load()
    layer = _lib.AdaptLayer(0, 0, N, K, RANK, GROUPS, 4096, 4096, 4096, 1.0, 0.0)
    some = 4096
    a, b = ctypes.c_int64(), ctypes.c_int64()

    def changed(**kw):
        new = _lib.AdaptLayer.from_buffer_copy(layer)
        for k, v in kw.items():
            setattr(new, k, v)
        return new
    for call in [
        lambda: lib.vh_rows_plan_size(0, 5, a, b),
        lambda: lib.vh_rows_plan_size(5, 16385, a, b),
        lambda: lib.vh_rows_plan_size(5, 5, None, b),
        lambda: lib.vh_rows_plan(None, 5, 5, some, None, None),
        lambda: lib.vh_rows_plan(some, 5, 5, some + 4, None, None),
        lambda: lib.vh_rows_plan(some, 20000, 5, some, None, None),          # needs scratch
        lambda: lib.vh_adapt_weight_size(0, 5, 0, a),
        lambda: lib.vh_adapt_weight_size(5, 5, 2, a),
        lambda: lib.vh_adapt_weight_pack(some, 4, None, 5, 5, 0, some, None),
        lambda: lib.vh_adapt_weight_pack(some, 5, None, 5, 5, 0, some + 8, None),
        lambda: lib.vh_adapt_forward(None, some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(rank=65), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(groups=0), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(dtype=7), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(down=None), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(activation=1, negative_slope=-1.0), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(changed(scale=float("inf")), some, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(layer, None, K, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(layer, some, K - 1, 5, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward(layer, some, K, 5, some, some, N, None, some, None, None),     # codes without exponents
        lambda: lib.vh_adapt_forward(layer, some, K, 2 ** 31, some, some, N, None, None, None, None),
        lambda: lib.vh_adapt_forward_few(layer, some, K, 5, None, some, N, None),
        lambda: lib.vh_adapt_backward_size(5, 5, N, K, 0, 0, a),
        lambda: lib.vh_adapt_backward(layer, some, N, _lib.Held(None, 0, None, None), None, some, 5, some, some, K, some, some, some, None),
        lambda: lib.vh_adapt_backward(layer, some, N, _lib.Held(some, K, some, some), None, some, 5, some, some, K, some, some, some, None),
        lambda: lib.vh_adapt_backward(layer, some, N, _lib.Held(some, K - 1, None, None), None, some, 5, some, some, K, some, some, some, None),
        lambda: lib.vh_adapt_backward(changed(activation=1), some, N, _lib.Held(some, K, None, None), None, some, 5, some, some, K, some, some, some, None),
        lambda: lib.vh_checkpoint8(some, 3, 5, 4, 0, some, some, None),
        lambda: lib.vh_checkpoint8(some, 4, 5, 4, 0, some + 4, some, None),
        lambda: lib.vh_checkpoint8(some, 4, 5, 4, 0, some, None, None),
        lambda: lib.vh_checkpoint8_restore(some, some, 5, 4, 0, None, None),
        lambda: lib.vh_checkpoint8_weight_grad_size(5, 0, 4, a),
        lambda: lib.vh_checkpoint8_weight_grad(some, N, _lib.Held(some, K, None, None), None, 0.0, 5, N, K, 0, some, some, some, None),
        lambda: lib.vh_checkpoint8_weight_grad(some, N - 1, _lib.Held(None, 0, some, some), None, 0.0, 5, N, K, 0, some, some, some, None),
    ]:
        with pytest.raises(ValueError):
            _lib.check(call())


def test_oracle_encoding():
    """The oracle's codes against torch's own e4m3 type, and its exponents against the definition."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((20, 70)) * np.exp2(rng.integers(-20, 20, (20, 1)))).astype(np.float32)
    codes, exps = ao.encode(x)
    k = exps.astype(int) - 127
    amax = np.abs(np.pad(x, ((0, 0), (0, 26)))).reshape(20, 3, 32).max(2)
    assert (amax <= 448 * np.exp2(k)).all() and (amax > 448 * np.exp2(k - 1)).all()
    scaled = torch.from_numpy(np.pad(x, ((0, 0), (0, 26))) * np.repeat(np.exp2(-k), 32, 1).astype(np.float32)).float()
    want = scaled.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes & 127, want & 127)
    assert np.array_equal(codes >= 128, ~(scaled.numpy() > 0))
    assert np.abs(ao.decode(codes, exps, 70) - x).max() <= (2.0 ** -4 * np.abs(x)).max()


@pytest.mark.parametrize("rows,groups", [(1, 1), (1, 2), (1, 200), (3, 4), (7, 9), (15, 16), (15, 200), (16, 40), (17, 3), (300, 5), (2000, 2)])
def test_gradient_items_read_slots_that_exist(rows, groups):
    """A plan laid out as adapt_common.hpp describes it: whatever groups the rows are of, groups without rows behind them too, no item's rows are
    looked for at or behind the plan's last slot (behind it, in the last plane of p, the caller's scratch ends)."""
    lib = _lib.load()
    rng = np.random.default_rng(rows * 1000 + groups)
    highest, slots = ctypes.c_int64(), ctypes.c_int64()
    for of in (np.arange(rows) % groups, np.zeros(rows, int), rng.integers(0, groups, rows), np.full(rows, -1), np.full(rows, groups - 1)):
        first = 0
        for g in range(groups):
            count = int((of == g).sum())
            for at in range(0, max(count, 1), 128):
                piece = min(128, count - at)
                _lib.check(lib.vh_debug_adapt_item_reads(rows, groups, first + at, piece, highest, slots))
                assert 0 <= highest.value < slots.value, (g, first + at, piece)
                if piece:
                    assert highest.value == first + at + piece - 1
            first += -(-count // 16) * 16


@pytest.mark.parametrize("which", ["x", "down", "up"])
def test_forward_refuses_what_asks_for_a_gradient(which):
    """Its result would be cut off from autograd without a word."""
    a = args()
    a[which].requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        ad.adapted_linear(**a)
    with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):      # (past that check)
        ad.adapted_linear(**a)
    a[which] = a[which].detach()
    with pytest.raises(ValueError, match="on a GPU"):
        ad.adapted_linear(**a)


def test_c_entries_refuse_what_no_launch_holds():
    """Sizes within the documented limits whose launch would have 2^32 threads or more: an argument error, before any device work."""
    lib = _lib.load()
    some = 4096
    for call, why in [
        (lambda: lib.vh_adapt_forward(_lib.AdaptLayer(1, 0, 32, 8, 4, 1, some, some, some, 1.0, 0.0), some, 8, 2 ** 29, some, some, 32, None, None, None, None),
         "rows"),
        (lambda: lib.vh_adapt_forward(_lib.AdaptLayer(0, 0, 4096, 8, 40, 1, some, some, some, 1.0, 0.0), some, 8, 2 ** 28, some, some, 4096, None, None, None,
                                      None), "rows"),
        (lambda: lib.vh_adapt_backward(_lib.AdaptLayer(1, 0, 4096, 8, 4, 1, some, some, some, 1.0, 0.0), some, 4096, _lib.Held(some, 8, None, None), None,
                                       some, 2 ** 26, some, some, 8, some, some, some, None), "rows"),
        (lambda: lib.vh_checkpoint8_weight_grad(some, 2 ** 16, _lib.Held(None, 0, some, some), None, 0.0, 5, 2 ** 16, 2 ** 16, 1, some, None, some, None),
         "gradient"),
    ]:
        with pytest.raises(ValueError, match=why + ".*one launch"):
            _lib.check(call())


@pytest.mark.parametrize("dtype,rows,k,n,rank,groups,few", [
    (torch.bfloat16, 64, 304, 512, 8, 4, True), (torch.bfloat16, 5000, 32, 512, 1, 200, False), (torch.bfloat16, 16, 1104, 512, 16, 200, False),
    (torch.bfloat16, 14, 304, 512, 8, 200, True), (torch.float32, 17, 512, 512, 1, 200, False), (torch.float32, 3, 304, 512, 8, 200, True),
    (torch.bfloat16, 312, 512, 512, 1, 200, False), (torch.bfloat16, 2500, 64, 1104, 1, 1, False)])
def test_calls_that_go_without_a_plan(dtype, rows, k, n, rank, groups, few):
    """The measured side of each (adapters.py): what a workgroup reads counts, not the rows' elements alone."""
    assert (ad._few_cost(rows, n, k, rank, groups) <= ad._FEW[dtype]) == few
