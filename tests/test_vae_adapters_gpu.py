"""vamb_amd.adapters.VAEAdapters on a VAE: the operators of adapters.py as they are used together."""
import io

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup():
    from vamb_amd import encode
    rng = np.random.default_rng(4)
    n, samples = 1500, 7
    depths = rng.random((n, samples)).astype(np.float32) * 20 + 0.1
    tnf = rng.standard_normal((n, 103)).astype(np.float32)
    loader = encode.make_dataloader(depths, tnf, rng.integers(2000, 9000, n), batchsize=128, destroy=False)
    vae = encode.VAE(samples, nhiddens=[48, 40], nlatent=8, seed=1)
    vae.trainmodel(loader, nepochs=3, batchsteps=None)
    return vae, loader, rng.integers(-1, 5, n)


def test_new_adapters_change_nothing(setup):
    vae, loader, groups = setup
    want = vae.encode(loader)
    got = vae.adapters(5, rank=3, dtype=torch.float32).encode(loader, groups, batchsize=700)
    assert got.shape == want.shape and got.dtype == np.float32
    # two float32 evaluations (BatchNorm applied, or folded into the weights) of sums of at most 110 terms over three layers, whose
    # terms are of the size of the result times a few; then 12 mantissa bits are cut off: 2^-11 of the value
    size = np.abs(want).max()
    assert np.abs(got - want).max() <= 2.0 ** -11 * size + 3 * 128 * 2.0 ** -24 * 8 * size


def oracle_loss(a, x, w, groups, noise, down, up):
    """The loss in 64 bits from the folded layers."""
    f = lambda t: t.double().cpu()  # noqa: E731
    h = f(x)
    for i, (shared, d, u) in enumerate(zip(a._test_encoder, down, up)):
        weight, bias = (f(t) for t in shared)
        z = h @ weight.t() + bias
        for r, g in enumerate(groups.tolist()):
            if 0 <= g < a.n_groups:
                z[r] += a.scale * (f(u)[g] @ (f(d)[g] @ h[r]))
        h = z if i == len(down) - 1 else torch.where(z > 0, z, 0.01 * z)
    mu, h = h, h + f(noise)
    for i, (weight, bias) in enumerate(a._test_decoder):
        h = h @ f(weight).t() + f(bias)
        if i < len(a._test_decoder) - 1:
            h = torch.where(h > 0, h, 0.01 * h)
    s, x = a.nsamples, f(x)
    p = torch.softmax(h[:, :s], 1)
    ce = -((p + 1e-9).log() * x[:, :s]).sum(1) * (1 - a.alpha) * (s - 1) / (s * np.log(s))
    sse = (h[:, s:s + 103] - x[:, s:s + 103]).square().sum(1) * a.alpha / 103
    ab = (h[:, s + 103:] - x[:, s + 103:]).square().sum(1) * (1 - a.alpha) / s
    kld = 0.5 * mu.square().sum(1) / (a.nlatent * a.beta)
    return float((ce + sse + ab + kld).mean() * f(w).mean())


def test_loss_and_gradients(setup, monkeypatch):
    from vamb_amd import adapters as ad
    vae, loader, groups = setup
    seen = []
    init = ad.SharedProjection.__init__

    def spy(self, weight, bias=None):
        seen.append((weight.clone(), bias.clone()))
        init(self, weight, bias)
    monkeypatch.setattr(ad.SharedProjection, "__init__", spy)
    a = vae.adapters(5, rank=3, scale=0.5, dtype=torch.float32, seed=3)
    a._test_encoder, a._test_decoder = seen[:3], seen[3:6]
    g = torch.Generator(device="cuda").manual_seed(0)
    for u in a.up:
        u.copy_(0.3 * torch.randn(u.shape, generator=g, device="cuda"))
    x, w = a._features(loader)
    of = a._groups(groups, len(x))
    x, w, of = x[:60], w[:60], of[:60]
    noise = torch.randn((60, 8), generator=g, device="cuda")
    loss, downs, ups, (dw, db) = a.gradients(x, w, of, noise, mu_too=True)
    want = oracle_loss(a, x, w, of.cpu(), noise, a.down, a.up)
    assert abs(float(loss) - want) <= 1e-5 * abs(want)
    # differences of the 64-bit loss along one direction per parameter.  h = 1e-4: a truncation error of h^2 and a kink of LeakyReLU crossed by few
    # of the 60 x 88 units weigh 1e-3 at most.  up's gradient has no rounding but float32's; down's reads its input as a checkpoint, each
    # element of which is off by up to 2^-4 with either sign: the sum of the magnitudes of the row terms, 2^-4, bounds it
    rng = torch.Generator(device="cuda").manual_seed(9)
    for kind, grads in (("up", ups), ("down", downs)):
        for i in range(3):
            p = getattr(a, kind)[i]
            way = torch.randn(p.shape, generator=rng, device="cuda")
            h = 1e-4
            ends = []
            for s in (h, -h):
                moved = [t + s * way if j == i else t for j, t in enumerate(getattr(a, kind))]
                ends.append(oracle_loss(a, x, w, of.cpu(), noise, moved if kind == "down" else a.down, moved if kind == "up" else a.up))
            want = (ends[0] - ends[1]) / (2 * h)
            got = float((grads[i].double() * way.double()).sum())
            size = float((grads[i].double().abs() * way.double().abs()).sum())
            assert abs(got - want) <= (1e-3 if kind == "up" else 2.0 ** -4) * size, (kind, i, got, want, size)
    assert dw.shape == a._mu_weight.shape and db.shape == a._mu_bias.shape
    assert torch.isfinite(dw).all() and db.abs().sum() > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_runs_and_is_reproducible(setup, dtype):
    vae, loader, groups = setup
    runs = []
    for _ in range(2):
        a = vae.adapters(5, rank=4, dtype=dtype, seed=2)
        losses = a.train(loader, groups, nepochs=2, batchsize=256, mu_too=True)
        assert len(losses) == 2 and np.isfinite(losses).all()
        runs.append((losses, a.encode(loader, groups), a))
    assert runs[0][0] == runs[1][0] and np.array_equal(runs[0][1], runs[1][1])
    assert all(u.abs().sum() > 0 for u in runs[0][2].up)
    # a contig without an adapter is encoded by the shared layers alone
    alone = runs[0][2].encode(loader, np.full(len(groups), -1))
    assert np.array_equal(alone[groups < 0], runs[0][1][groups < 0]) and not np.array_equal(alone, runs[0][1])
    from vamb_amd.adapters import VAEAdapters
    f = io.BytesIO()
    runs[0][2].save(f)
    f.seek(0)
    again = VAEAdapters.load(f, vae, dtype=dtype)
    assert np.array_equal(again.encode(loader, groups), runs[0][1])


def test_refusals(setup):
    from vamb_amd import adapters as ad
    vae, loader, groups = setup
    for call in [lambda: vae.adapters(0), lambda: vae.adapters(5, rank=65), lambda: vae.adapters(5, dtype=torch.float16),
                 lambda: vae.adapters(5, scale=float("inf")), lambda: ad.VAEAdapters("vae", 5)]:
        with pytest.raises(ValueError):
            call()
    a = vae.adapters(5)
    for call in [lambda: a.encode(loader, groups[:-1]), lambda: a.encode(loader, groups.astype(np.float32)), lambda: a.encode(loader, groups, batchsize=0),
                 lambda: a.train(loader, groups, nepochs=0), lambda: a.train(loader, groups, lrate=0.0), lambda: a.train(loader, groups, batchsize=0)]:
        with pytest.raises(ValueError):
            call()
