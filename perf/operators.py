"""What is measured of the adapter and checkpoint operators of ``vamb_amd.adapters``.

    u = x A_g^T,   y = f(x W^T + b + s u B_g^T)                 one shared projection W, one low-rank pair (A, B) per group g of rows
    p = dy f'(y),  v = s p B_g,  dx = p W + v A_g,  dA_g = sum v^T x,  dB_g = s sum p^T u,  dW = p^T x,  db = sum p

x is [rows, k], W [n, k], A = down [groups, rank, k], B = up [groups, n, rank]; a row whose group is -1 has no adapter.  Activations
that wait for the backward pass are held as e4m3 codes with a power-of-two scale for every 32 columns of a row: the scale 2^e is
the least that brings the block's largest magnitude to 448 or below (e in [-117, 120]), and a code's sign bit is set where x > 0 does not hold.
"""
import math

import torch

own = False

SLOPE = 0.01      # torch.nn.LeakyReLU's default, the one that the VAE uses
SCALE = 0.5       # of the adapters' part
BLOCK = 32        # columns that share a scale


def listed():
    return [
        # one contig's latent layer asked for by itself: the latency of a single row
        {"name": "encode_one_contig", "op": "forward", "type": "bfloat16", "rows": 1, "k": 304, "n": 512, "rank": 8, "groups": 200, "order": "shuffled", "act": True},
        # the `mu` layer for a ragged set of contigs of 50 samples, in the framework's default type, no activation
        {"name": "encode_mu_fp32", "op": "forward", "type": "float32", "rows": 4099, "k": 512, "n": 32, "rank": 4, "groups": 50, "order": "sorted", "act": False},
        # the first layer of an encode pass over a large cohort: 1000 samples, contigs in the order of the samples
        {"name": "encode_cohort", "op": "forward", "type": "bfloat16", "rows": 524288, "k": 1104, "n": 512, "rank": 16, "groups": 1000, "order": "sorted", "act": True},
        # the first layer of the smallest training batch (256 contigs of 50 samples: 50 + 104 columns, an odd width for vectors)
        {"name": "train_batch256_fp32", "op": "train", "type": "float32", "rows": 256, "k": 154, "n": 512, "rank": 8, "groups": 50, "order": "shuffled", "act": True},
        # a hidden layer in the largest training batch
        {"name": "train_batch8192", "op": "train", "type": "bfloat16", "rows": 8192, "k": 512, "n": 512, "rank": 16, "groups": 200, "order": "shuffled", "act": True},
        # the backward passes of both
        {"name": "backward_batch256_fp32", "op": "backward", "type": "float32", "rows": 256, "k": 512, "n": 512, "rank": 8, "groups": 50, "order": "shuffled", "act": True},
        {"name": "backward_batch8192", "op": "backward", "type": "bfloat16", "rows": 8192, "k": 512, "n": 512, "rank": 16, "groups": 200, "order": "shuffled", "act": True},
        # ... and of a pass over a cohort's contigs in one batch, wide input, a higher rank, an odd number of rows
        {"name": "backward_cohort", "op": "backward", "type": "bfloat16", "rows": 65537, "k": 1104, "n": 512, "rank": 32, "groups": 1000, "order": "shuffled", "act": True},
        # the checkpoint of a small batch's input, odd width; and of a hidden layer over a million contigs
        {"name": "checkpoint_batch256_fp32", "op": "checkpoint", "type": "float32", "rows": 256, "k": 154},
        {"name": "checkpoint_million", "op": "checkpoint", "type": "bfloat16", "rows": 1000003, "k": 512},
        # the shared projection's own gradient from the checkpoints: a hidden layer, and the wide first layer in the default type
        {"name": "weight_grad_batch8192", "op": "weight_grad", "type": "bfloat16", "rows": 8192, "k": 512, "n": 512, "act": True},
        {"name": "weight_grad_wide_fp32", "op": "weight_grad", "type": "float32", "rows": 4096, "k": 1104, "n": 512, "act": True},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["forward", "forward", "train", "backward", "backward", "checkpoint", "weight_grad"])
    case = {"op": op, "type": rng.choice(["bfloat16", "float32"]),
            "rows": _spread(rng, 1, {"forward": 262144, "train": 65536, "backward": 40000, "checkpoint": 500000, "weight_grad": 40000}[op])}
    case["k"] = rng.choice([104 + _spread(rng, 2, 1000), _spread(rng, 32, 512), 512])
    if op != "checkpoint":
        case["n"] = rng.choice([_spread(rng, 16, 512), 512, 32])
        case["act"] = rng.random() < 0.75
    if op in ("forward", "train", "backward"):
        case["rank"] = _spread(rng, 1, 64 if case["rows"] <= 40000 else 16)
        case["groups"] = _spread(rng, 1, 1000)
        case["order"] = rng.choice(["shuffled", "sorted"])
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _leaky(z):
    return torch.where(z > 0, z, SLOPE * z)


def _codes_of(x):
    """e4m3 values (as float32) and exponents [rows, blocks] of the checkpoint of x."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    z = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    size = torch.where(torch.isfinite(z), z.abs(), 0.0).amax(2)
    m, e = torch.frexp(size)
    k = torch.where(size > 0, e - 9 + (m > 0.875).int(), -117).clamp(-117, 120)
    z = torch.ldexp(z, -k.unsqueeze(2))
    step = torch.exp2((torch.frexp(z)[1] - 1).clamp(min=-6).float() - 3)
    return torch.where(torch.isfinite(z), torch.round(z / step) * step, torch.nan), k


def _held(x):
    """The checkpoint of x as a program holds it: codes [rows, a multiple of 32] and exponents [rows, blocks], both bytes."""
    q, k = _codes_of(x)
    codes = q.view(len(x), q.shape[1] * BLOCK).to(torch.float8_e4m3fn).view(torch.uint8)
    above = torch.nn.functional.pad(x.float(), (0, codes.shape[1] - x.shape[1])) > 0
    return torch.where(above, codes & 127, codes | 128).contiguous(), (k + 127).to(torch.uint8).contiguous()


def _values(codes, exponents, cols):
    """float32 values of a held checkpoint."""
    q = codes.view(torch.float8_e4m3fn).float().view(len(codes), -1, BLOCK)
    return torch.ldexp(q, exponents.int().unsqueeze(2) - 127).view(len(codes), -1)[:, :cols]


def prepare(case, seed):
    g = _generator(seed)
    t = getattr(torch, case["type"])
    rows, k = case["rows"], case["k"]
    state = {"case": dict(case)}
    x = _leaky(_normal(g, rows, k)).to(t)     # what a hidden layer hands on
    if case["op"] == "checkpoint":
        state["x"] = x
        return state
    n = case["n"]
    weight = (_normal(g, n, k) / math.sqrt(k)).to(t)
    bias = (0.1 * _normal(g, n)).to(t)
    if case["op"] in ("backward", "weight_grad"):
        state["dy"] = (_normal(g, rows, n) / 64).to(t)
        state["x_codes"], state["x_exponents"] = _held(x)
        state["y_codes"], state["y_exponents"] = _held(_leaky(_normal(g, rows, n)).to(t))
    else:
        state["x"] = x
    if case["op"] == "weight_grad":
        if own:
            _wrap(state)
        return state
    groups, rank = case["groups"], case["rank"]
    share = torch.exp(0.5 * _normal(g, groups))   # samples have unlike numbers of contigs
    of = torch.searchsorted((share.cumsum(0) / share.sum()).contiguous(), torch.rand(rows, generator=g, device="cuda")).clamp(max=groups - 1)
    of = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.01, -1, of)   # a few contigs of no known sample
    if case["order"] == "sorted":
        of = of.sort().values
    state["groups"] = of.to(torch.int32)
    state["most"] = max(1, int(torch.bincount(of[of >= 0], minlength=1).max()))   # the largest group, which the plain form pads to
    state["weight"], state["bias"] = weight, bias
    state["down"] = (_normal(g, groups, rank, k) / math.sqrt(k)).to(t)
    state["up"] = (_normal(g, groups, n, rank) / math.sqrt(rank)).to(t)
    if case["op"] == "backward":
        state["low"] = torch.where(of[:, None] >= 0, _normal(g, rows, rank), 0.0)
    if own:
        _wrap(state)
    return state


def _wrap(state):
    """The framework's objects that a program keeps: the projection laid out once, the checkpoints that the forward pass left."""
    from vamb_amd import adapters
    if "weight" in state:
        state["shared"] = adapters.SharedProjection(state["weight"], state["bias"])
    case = state["case"]
    if "x_codes" in state:
        state["x8"] = adapters.Checkpoint8(state["x_codes"], state["x_exponents"], case["k"])
        state["y8"] = adapters.Checkpoint8(state["y_codes"], state["y_exponents"], case["n"])


def _slots(of, most, groups):
    """Where each row stands when the rows of every group are laid out in `most` places; rows without a group share the last place."""
    rows = len(of)
    order = torch.argsort(of, stable=True)
    counts = torch.zeros(groups + 1, dtype=torch.int64, device=of.device).scatter_add_(0, of + 1, torch.ones_like(of))
    starts = counts.cumsum(0) - counts
    rank = torch.empty_like(of)
    rank[order] = torch.arange(rows, device=of.device) - starts[of[order] + 1]
    return torch.where(of >= 0, of * most + rank, groups * most)


def _laid(z, slots, most, groups):
    out = torch.zeros(groups * most + 1, z.shape[1], device=z.device)
    out[slots] = z
    return out[:-1].view(groups, most, z.shape[1])


def _back(z, slots):
    flat = z.reshape(-1, z.shape[2])
    return torch.cat([flat, torch.zeros_like(flat[:1])])[slots]


def _slope_of(case):
    return SLOPE if case["act"] else None


def _plain_forward(s):
    c = s["case"]
    of = s["groups"].long()
    slots = _slots(of, s["most"], c["groups"])
    x = s["x"].float()
    low = torch.bmm(_laid(x, slots, s["most"], c["groups"]), s["down"].float().transpose(1, 2).contiguous())
    part = _back(torch.bmm(low, s["up"].float().transpose(1, 2).contiguous()), slots)
    y = x @ s["weight"].float().t() + s["bias"].float() + SCALE * part
    return (_leaky(y) if c["act"] else y).to(s["x"].dtype), _back(low, slots)


def _plain_p(s):
    p = s["dy"].float()
    return p * torch.where(s["y_codes"][:, :p.shape[1]] < 128, 1.0, SLOPE) if s["case"]["act"] else p


def _plain_backward(s):
    c, t = s["case"], s["dy"].dtype
    groups, most = c["groups"], s["most"]
    slots = _slots(s["groups"].long(), most, groups)
    x, p = _values(s["x_codes"], s["x_exponents"], c["k"]), _plain_p(s)
    laid_p = _laid(p, slots, most, groups)
    v = SCALE * torch.bmm(laid_p, s["up"].float())
    dx = p @ s["weight"].float() + _back(torch.bmm(v, s["down"].float()), slots)
    ddown = torch.bmm(v.transpose(1, 2).contiguous(), _laid(x, slots, most, groups))
    dup = SCALE * torch.bmm(laid_p.transpose(1, 2).contiguous(), _laid(s["low"], slots, most, groups))
    return dx.to(t), ddown.to(t), dup.to(t)


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"] == "forward":
        return _plain_forward(s)[0]
    if c["op"] == "train":
        y, low = _plain_forward(s)
        q, k = _codes_of(y)
        return {"y": y, "low": low, "held": torch.ldexp(q, k.unsqueeze(2)).view(len(y), -1)[:, :c["n"]].to(torch.bfloat16)}
    if c["op"] == "backward":
        return dict(zip(("dx", "ddown", "dup"), _plain_backward(s)))
    if c["op"] == "checkpoint":
        q, k = _codes_of(s["x"])
        return torch.ldexp(q, k.unsqueeze(2)).view(c["rows"], -1)[:, :c["k"]].to(torch.bfloat16)
    p = _plain_p(s)
    return {"dweight": (p.t().contiguous() @ _values(s["x_codes"], s["x_exponents"], c["k"])).to(s["dy"].dtype), "dbias": p.sum(0).to(s["dy"].dtype)}


def _own(s, c):
    from vamb_amd import adapters
    if c["op"] == "forward":
        return adapters.adapted_linear(s["x"], s["shared"], s["down"], s["up"], s["groups"], scale=SCALE, negative_slope=_slope_of(c))
    if c["op"] == "train":
        rows = adapters.group_rows(s["groups"], c["groups"])
        y, low, held = adapters.adapted_linear_train(s["x"], s["shared"], s["down"], s["up"], rows, scale=SCALE, negative_slope=_slope_of(c))
        return {"y": y, "low": low, "held": held.restore(torch.bfloat16)}
    if c["op"] == "backward":
        rows = adapters.group_rows(s["groups"], c["groups"])
        dx, ddown, dup = adapters.adapted_linear_backward(s["dy"], s["x8"], s["y8"], s["low"], s["shared"], s["down"], s["up"], rows,
                                                          scale=SCALE, negative_slope=_slope_of(c))
        return {"dx": dx, "ddown": ddown, "dup": dup}
    if c["op"] == "checkpoint":
        return adapters.checkpoint8(s["x"]).restore(torch.bfloat16)
    dweight, dbias = adapters.checkpoint_weight_grad(s["dy"], s["x8"], s["y8"], negative_slope=_slope_of(c))
    return {"dweight": dweight, "dbias": dbias}


def work(case):
    size = 2 if case["type"] == "bfloat16" else 4
    rows, k, op = case["rows"], case["k"], case["op"]
    held = lambda cols: rows * (cols + -(-cols // BLOCK))  # noqa: E731
    if op == "checkpoint":   # read x, write the codes, read them, write their values
        return {"bytes": rows * k * (size + 2) + 2 * held(k), "flops": 2 * rows * k}
    n = case["n"]
    if op == "weight_grad":
        return {"bytes": rows * n * size + held(n) + held(k) + (n * k + n) * size, "flops": 2 * rows * n * k}
    rank = case["rank"]
    used = min(rows, case["groups"])      # adapters that some row asks for
    pairs = used * rank * (n + k) * size
    if op == "backward":
        return {"bytes": rows * (n * size + 4 + 4 * rank) + held(n) + held(k) + n * k * size + pairs + rows * k * size + case["groups"] * rank * (n + k) * size,
                "flops": 2 * rows * (n * k + 2 * rank * (n + k))}
    moved = rows * (k * size + 4 + n * size) + (n * k + n) * size + pairs
    if op == "train":
        moved += rows * 4 * rank + held(n) * 2 + rows * n * 2
    return {"bytes": moved, "flops": 2 * rows * (n * k + rank * (n + k))}


def _exact_held(x):
    """64-bit values of the checkpoint of x, block by block from the definition."""
    z = x.double()
    out = torch.empty_like(z)
    for at in range(0, z.shape[1], BLOCK):
        b = z[:, at:at + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448))
        for step in (-1, 1):   # log2's own rounding: the least k that holds
            k = torch.where(top <= 448 * torch.exp2(k - 1), k - 1, k) if step < 0 else torch.where(top > 448 * torch.exp2(k), k + 1, k)
        k = k.clamp(-117, 120)
        q = b / torch.exp2(k)
        e = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
        e = torch.where(q.abs() < torch.exp2(e), e - 1, torch.where(q.abs() >= torch.exp2(e + 1), e + 1, e)).clamp(min=-6)
        unit = torch.exp2(e - 3)
        out[:, at:at + BLOCK] = torch.round(q / unit) * unit * torch.exp2(k)
    return out


def _exact_read(codes, exponents, cols):
    """64-bit values of held bytes: sign, 4 bits of exponent, 3 of mantissa."""
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    size = torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0 ** -9)
    value = torch.where(c >= 128, -size, size) * torch.exp2(exponents.double() - 127).repeat_interleave(BLOCK, 1)
    return value[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        return _exact_held(s["x"])
    act = case["act"]
    if op in ("backward", "weight_grad"):
        x = _exact_read(s["x_codes"], s["x_exponents"], case["k"])
        p = s["dy"].double()
        if act:
            p = torch.where(s["y_codes"][:, :case["n"]] >= 128, SLOPE * p, p)
        if op == "weight_grad":
            return {"dweight": p.t() @ x, "dbias": p.sum(0)}
        dx = p @ s["weight"].double()
        ddown, dup = torch.zeros_like(s["down"], dtype=torch.float64), torch.zeros_like(s["up"], dtype=torch.float64)
        for g in range(case["groups"]):
            rows = torch.nonzero(s["groups"] == g)[:, 0]
            v = SCALE * p[rows] @ s["up"][g].double()
            dx[rows] += v @ s["down"][g].double()
            ddown[g] = v.t() @ x[rows]
            dup[g] = SCALE * p[rows].t() @ s["low"][rows].double()
        return {"dx": dx, "ddown": ddown, "dup": dup}
    x = s["x"].double()
    y = x @ s["weight"].double().t() + s["bias"].double()
    low = torch.zeros(case["rows"], case["rank"], dtype=torch.float64, device="cuda")
    for g in range(case["groups"]):
        rows = torch.nonzero(s["groups"] == g)[:, 0]
        low[rows] = x[rows] @ s["down"][g].double().t()
        y[rows] += SCALE * low[rows] @ s["up"][g].double().t()
    if act:
        y = torch.where(y > 0, y, SLOPE * y)
    if op == "forward":
        return y
    return {"y": y, "low": low, "held": None}   # what a rounded y is held as depends on its rounding
