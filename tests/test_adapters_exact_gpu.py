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
