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
    """u = (1 + 2^-20, 1), B = (1, -1): y = scale 2^-20, and the same of v in the backward pass; nothing in it is rounded (bf16 tensors)."""
    rows, n, k = 20, 40, 72
    bf = lambda t: t.to("cuda", torch.bfloat16)  # noqa: E731
    x, dy = torch.zeros(rows, k), torch.zeros(rows, n)
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -20
    dy[:, 0], dy[:, 1] = 1.0, 2.0 ** -20
    down, up = torch.zeros(1, 2, k), torch.zeros(1, n, 2)
    down[0, :, 0], down[0, 0, 1] = 1.0, 1.0       # u as above
    up[0, :, 0], up[0, :, 1] = 1.0, -1.0
    shared = ad.SharedProjection(bf(torch.zeros(n, k)))
    groups = torch.zeros(rows, dtype=torch.int32, device="cuda")
    plan = ad.group_rows(groups, 1)
    want = SCALE * 2.0 ** -20
    for g in (groups, plan):
        assert (ad.adapted_linear(bf(x), shared, bf(down), bf(up), g, SCALE) == want).all()
    up[0] = 0.0
    up[0, 0, :], up[0, 1, 0] = 1.0, 1.0           # v = scale (1 + 2^-20, 1)
    down[0, 0], down[0, 1] = 1.0, -1.0
    dx, _, _ = ad.adapted_linear_backward(bf(dy), bf(x), None, torch.zeros(rows, 2, device="cuda"), shared, bf(down), bf(up), plan, SCALE)
    assert (dx == want).all()
