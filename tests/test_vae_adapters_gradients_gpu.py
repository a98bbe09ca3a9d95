"""VAEAdapters.gradients, tensor by tensor, against the chain rule in 64 bits.

The reference computes the forward pass for itself; what the product holds for its backward pass (the checkpoints' values and signs) it reads from
the product, so that the checkpoints' own rounding, tested elsewhere, does not blur the comparison.  Tolerances are of a tensor's norm (an
unrelated gradient, a wrong sign or a factor of two is off by 1 or more).  float32: a layer's sums of up to 110 terms are within (2 * 110 + 20) 2^-24
+ 2^-21 < 2^-15 of their magnitudes, eight layers one behind the other, magnitudes up to sqrt(110) times the result: 2^-9.  bf16: 13 roundings of half
a step (2^-9 of a tensor's norm each, two ways through the layer) that add up at worst: 2^-4."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
SLOPE = 0.01
TOL = {torch.float32: 2.0 ** -9, torch.bfloat16: 2.0 ** -4}


def trained(samples, seed):
    from vamb_amd import encode
    rng = np.random.default_rng(seed)
    n = 600
    loader = encode.make_dataloader(rng.random((n, samples)).astype(np.float32) * 20 + 0.1, rng.standard_normal((n, 103)).astype(np.float32),
                                    rng.integers(2000, 9000, n), batchsize=128, destroy=False)
    vae = encode.VAE(samples, nhiddens=[48, 40], nlatent=8, seed=1)
    vae.trainmodel(loader, nepochs=2, batchsteps=None)
    return vae, loader, rng.integers(-1, 5, n)


def expected(a, weights, x, w, groups, noise, down, up, signs, held):
    """(loss, ddown, dup, dmu weight, dmu bias): weights [(W, b)] of encoder and decoder, signs [layer] what y > 0 was read as, held the
    encoder layers' inputs as they were kept (None: as they are)."""
    d = lambda t: t.detach().double().cpu()  # noqa: E731
    x, w, noise, groups = d(x), d(w), d(noise), groups.cpu().long()
    n_enc, rows, s = len(down), len(x), a.nsamples
    with_adapter = ((groups >= 0) & (groups < a.n_groups)).double()[:, None]
    at = groups.clamp(0, a.n_groups - 1)
    h, us, ins = x, [], []
    for i, (W, b) in enumerate(weights):
        z = h @ d(W).t() + d(b)
        if i < n_enc:
            A, B = d(down[i])[at], d(up[i])[at]
            u = torch.einsum("rjk,rk->rj", A, h) * with_adapter
            z = z + a.scale * torch.einsum("rnj,rj->rn", B, u)
            us.append(u)
            ins.append(h)
        last = i in (n_enc - 1, len(weights) - 1)
        h = z if last else torch.where(signs[i], z, SLOPE * z)
        if i == n_enc - 1:
            mu = h
            h = h + noise
    held, out = held or ins, h
    p = torch.softmax(out[:, :s], 1)
    wm = float(w.mean())
    ab, sse, kld = (1 - a.alpha) / s, a.alpha / 103, 1 / (a.nlatent * a.beta)
    diff = out[:, s:] - x[:, s:]
    loss = diff[:, :103].square().sum(1) * sse + diff[:, 103:].square().sum(1) * ab + 0.5 * mu.square().sum(1) * kld
    g = torch.zeros_like(out)
    g[:, s:s + 103], g[:, s + 103:] = 2 * sse * diff[:, :103], 2 * ab * diff[:, 103:]
    if s > 1:
        ce = (1 - a.alpha) * (s - 1) / (s * np.log(s))
        loss = loss - ((p + 1e-9).log() * x[:, :s]).sum(1) * ce
        dp = -ce * x[:, :s] / (p + 1e-9)
        g[:, :s] = p * (dp - (dp * p).sum(1, keepdim=True))
    g = g * wm / rows
    ddown, dup, dmu = [None] * n_enc, [None] * n_enc, None
    for i in range(len(weights) - 1, -1, -1):
        W = d(weights[i][0])
        if i == n_enc - 1:
            g = g + mu * kld * wm / rows
            dmu = g.t() @ held[i], g.sum(0)
        elif i != len(weights) - 1:
            g = torch.where(signs[i], g, SLOPE * g)
        nxt = g @ W
        if i < n_enc:
            A, B = d(down[i])[at], d(up[i])[at]
            v = a.scale * torch.einsum("rn,rnj->rj", g, B) * with_adapter
            nxt = nxt + torch.einsum("rj,rjk->rk", v, A)
            ddown[i], dup[i] = torch.zeros_like(d(down[i])), torch.zeros_like(d(up[i]))
            for q in range(a.n_groups):
                m = groups == q
                ddown[i][q] = v[m].t() @ held[i][m]
                dup[i][q] = a.scale * g[m].t() @ us[i][m]
        g = nxt
    return float(loss.mean() * wm), ddown, dup, dmu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("samples,checkpoints", [(7, True), (1, True), (7, False)])
def test_gradients_tensor_by_tensor(samples, checkpoints, dtype, monkeypatch):
    from vamb_amd import adapters as ad
    vae, loader, groups = trained(samples, 11)
    weights, held = [], []
    init, keep, train = ad.SharedProjection.__init__, ad.checkpoint8, ad.adapted_linear_train

    def spy_init(self, weight, bias=None):
        weights.append((weight.clone(), bias.clone()))
        init(self, weight, bias)

    def spy_keep(x):
        held.append(keep(x))
        return held[-1]

    def spy_train(*args, **kw):
        out = train(*args, **kw)
        held.append(out[2])
        return out
    monkeypatch.setattr(ad.SharedProjection, "__init__", spy_init)
    a = vae.adapters(5, rank=3, scale=0.5, dtype=dtype, seed=3, **({} if checkpoints else {"checkpoints": False}))
    gen = torch.Generator(device="cuda").manual_seed(0)
    for u in a.up:
        u.copy_(0.3 * torch.randn(u.shape, generator=gen, device="cuda"))
    if dtype == torch.bfloat16:      # parameters that bf16 holds: their rounding is not what is looked at
        for i in range(2):
            for t in (a.down[i], a.up[i]):
                t.copy_(t.to(dtype))
    x, w = a._features(loader)
    x, w, of = x[:200].to(dtype).float(), w[:200], a._groups(groups, len(x))[:200]
    noise = torch.randn((200, 8), generator=gen, device="cuda")
    monkeypatch.setattr(ad, "checkpoint8", spy_keep)
    monkeypatch.setattr(ad, "adapted_linear_train", spy_train)
    loss, downs, ups, (dw, db) = a.gradients(x, w, of, noise, mu_too=True)
    assert len(weights) == 6
    if checkpoints:     # the input, three layers of the encoder, the latent, three of the decoder
        assert len(held) == 8
        values, held = [h.restore().double().cpu() for h in held[:3]], held[1:4] + held[5:8]
    else:               # (the checkpoints that the layers' launches wrote, whose signs are those of the tensors that were kept)
        assert len(held) == 6
        values = None
    signs = [(h.codes[:, :h.columns] < 128).cpu() for h in held]
    want_loss, ddown, dup, (mw, mb) = expected(a, weights, x, w, of, noise, a.down, a.up, signs, values)
    assert abs(float(loss) - want_loss) <= (1e-5 if dtype == torch.float32 else 2.0 ** -6) * abs(want_loss)
    found = {f"down {i}": (downs[i], ddown[i]) for i in range(3)} | {f"up {i}": (ups[i], dup[i]) for i in range(3)} | {"mu weight": (dw, mw), "mu bias": (db, mb)}
    off = {k: float((got.double().cpu() - want).norm() / want.norm()) for k, (got, want) in found.items()}
    assert all(want.norm() > 0 for _, want in found.values())
    assert max(off.values()) <= TOL[dtype], off


def test_training_without_checkpoints():
    from vamb_amd.adapters import VAEAdapters
    import io
    vae, loader, groups = trained(7, 12)
    runs = []
    for _ in range(2):
        a = vae.adapters(5, rank=4, seed=2, checkpoints=False)
        losses = a.train(loader, groups, nepochs=2, batchsize=256, mu_too=True)
        runs.append((losses, a.encode(loader, groups), a))
    assert np.isfinite(runs[0][0]).all() and runs[0][0] == runs[1][0] and np.array_equal(runs[0][1], runs[1][1])
    f = io.BytesIO()
    runs[0][2].save(f)
    f.seek(0)
    again = VAEAdapters.load(f, vae, checkpoints=False)
    assert not again.checkpoints and np.array_equal(again.encode(loader, groups), runs[0][1])
