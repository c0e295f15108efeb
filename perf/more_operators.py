"""What joins the blocks of a layer: the norms with their gate and residual
scale, rows in 8 bits, and the product in 8-bit integers that reads them.

  linear     matmul_q8(x, weight, weight_scales, bias=...)      float rows in
  shared     quantize_q8(x), then two matmul_q8 of its rows     gate and up projections
  gated      gated_norm(x, weight, z, ...)                      the norm after a scan
  residual   residual_norm(x, residual, weight, ...)            a block's end and the next one's start
  block      residual_norm(..., quantize=True), then matmul_q8  a block's end and the next one's first projection

Inputs are drawn on the GPU from the seed.  Activations have channels of unequal
size, as they do in earnest.  8-bit weights are kept in rows that start every
16 bytes, as quantize_q8 lays them out.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _package():
    """The package lies in a folder of the repository's root."""
    path = os.path.abspath("pto-einsum_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pto_einsum

    return pto_einsum


def listed():
    return [
        # The largest square product of the benchmark, from 16-bit activations.
        dict(name="linear_large", op="linear", m=8192, n=8192, k=8192, bias=False, dtype="bfloat16"),
        # The input projection of 64 heads of 64 for a prompt of 4096 tokens:
        # gate, convolved channels, step sizes (no whole tile along n).
        dict(name="linear_prompt", op="linear", m=4096, n=8512, k=2048, bias=False, dtype="float16"),
        # A projection of one token, where latency counts.
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, bias=False, dtype="float16"),
        # An up projection of a batch of 16 tokens: the weights are read.
        dict(name="linear_batch", op="linear", m=16, n=16384, k=8192, bias=False, dtype="bfloat16"),
        # Gate and up projections of 64 sequences' tokens from one set of rows.
        dict(name="shared_tokens", op="shared", m=64, n=8192, k=4096, bias=False, dtype="float16"),
        # The same of a packed prompt in float32, sizes that are no whole tiles or
        # vectors, with a bias.
        dict(name="shared_odd", op="shared", m=1203, n=5001, k=2500, bias=True, dtype="float32"),
        # Behind the scan of 2 x 4096 tokens, 64 heads of 64: the gate is a
        # slice of the input projection, one norm for each of 8 groups.
        dict(name="gated_large", op="gated", b=2, t=4096, d=4096, groups=8, slice=True, norm_first=False,
             dtype="float16"),
        # One token of 64 sequences, odd channels, the gate behind the norm.
        dict(name="gated_tokens", op="gated", b=64, t=1, d=1283, groups=1, slice=False, norm_first=True,
             dtype="float32"),
        # Between two blocks of four prompts: a norm of the block's output, a
        # gate for each sequence, the residual kept in float32.
        dict(name="residual_large", op="residual", b=4, t=4096, d=4096, post=True, gate="sequence", scale=0.5,
             wide=True, dtype="bfloat16"),
        # Packed prompts, odd channels, a gate for each channel.
        dict(name="residual_odd", op="residual", b=1, t=3993, d=2500, post=False, gate="channel", scale=1.0,
             wide=False, dtype="float16"),
        # One token between two blocks, and the next block's input projection.
        dict(name="block_token", op="block", b=1, t=1, d=2048, post=False, gate="none", scale=1.0, wide=True, n=8512,
             dtype="float16"),
        # A prompt between two blocks, up to the next input projection.
        dict(name="block_prompt", op="block", b=1, t=2051, d=2048, post=True, gate="channel", scale=0.7, wide=False,
             n=8512, dtype="bfloat16"),
    ]


# ------------------------------------------------------------------ drawing --

def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], as it falls or rounded to a
    multiple of 8 or 64."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    step = rng.choice([1, 1, 8, 64])
    return min(hi, max(lo, n // step * step))


def _between(rng, most):
    """A place between two blocks, ``most`` values at most."""
    d = _size(rng, 16, 16384)
    b = _size(rng, 1, max(1, min(64, most // d)))
    return dict(b=b, t=_size(rng, 1, max(1, min(8192, most // d // b))), d=d)


def draw(rng):
    op = rng.choice(["linear", "linear", "shared", "gated", "residual", "block"])
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    if op in ("linear", "shared"):
        n, k = _size(rng, 64, 16384), _size(rng, 64, 16384)
        return dict(op=op, m=_size(rng, 1, min(8192, (1 << 38) // (n * k))), n=n, k=k, bias=rng.random() < 0.3,
                    dtype=dtype)
    if op == "gated":
        case = _between(rng, 1 << 26)
        groups = rng.choice([1, 1, 2, 4, 8])
        case["d"] = max(groups, case["d"] // groups * groups)
        return dict(op=op, **case, groups=groups, slice=rng.random() < 0.5, norm_first=rng.random() < 0.4, dtype=dtype)
    case = dict(op=op, **_between(rng, 1 << (26 if op == "residual" else 23)), post=rng.random() < 0.5,
                gate=rng.choice(["none", "channel", "sequence", "token", "full"]), scale=rng.choice([1.0, 0.5, 0.7]),
                wide=rng.random() < 0.5, dtype=dtype)
    if op == "block":
        # (rows in 8 bits of values that are themselves computed: an output of
        # 16 bits)
        case.update(n=_size(rng, 64, min(16384, (1 << 27) // (case["b"] * case["t"]))),
                    dtype=rng.choice(["float16", "bfloat16"]))
    return case


# ------------------------------------------------------------------- inputs --

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 97)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV) * scale

    def channels(d):
        """Sizes of channels: most alike, a few much larger."""
        return torch.exp(0.5 * normal(d)) * torch.where(torch.rand(d, generator=g, device=DEV) < 0.002, 10.0, 1.0)

    def weights(n, k):
        """[n, k] in 8 bits, rows every 16 bytes, and the scales of its rows."""
        rows = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device=DEV)
        rows[:, :k] = (normal(n, k) * 32).round_().clamp_(-127, 127)
        return rows[:, :k], (torch.rand(n, generator=g, device=DEV) + 0.5) / (32 * math.sqrt(k))

    s = dict(case=case, dtype=dt)
    if op in ("linear", "shared"):
        s["x"] = (normal(case["m"], case["k"]) * channels(case["k"])).to(dt)
        s["w"], s["ws"] = weights(case["n"], case["k"])
        s["bias"] = normal(case["n"], scale=0.1) if case["bias"] else None
        if op == "shared":
            s["w2"], s["ws2"] = weights(case["n"], case["k"])
        return s
    b, t, d = case["b"], case["t"], case["d"]
    s["x"] = (normal(b, t, d) * channels(d)).to(dt)
    s["weight"] = (1 + normal(d, scale=0.1)).to(dt)
    if op == "gated":
        z = normal(b, t, 2 * d + 64 if case["slice"] else d).to(dt)
        s["z"] = z[..., :d]
        return s
    s["residual"] = normal(b, t, d, scale=2.0).to(torch.float32 if case["wide"] else dt)
    s["post_weight"] = (1 + normal(d, scale=0.1)).to(dt) if case["post"] else None
    shape = dict(none=None, channel=(d,), sequence=(b, 1, d), token=(b, t, 1), full=(b, t, d))[case["gate"]]
    s["gate"] = None if shape is None else normal(*shape).to(dt)
    if op == "block":
        s["w"], s["ws"] = weights(case["n"], d)
        s["bias"] = None
    return s


# --------------------------------------------------------------- plain forms --

def _rows(x):
    """Rows of x in 8 bits (as float32 whole numbers) and their scales.  Which
    whole number is nearest is decided in 64 bits: half-way values are common
    (half the largest value of a row is one)."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.where(most > 0, torch.round(x.double() * 127 / most.double()), 0.0).float()
    return q, most / torch.full_like(most, 127.0)


def _product(q, scale, w, ws, bias, dt):
    y = torch.matmul(q, w.float().t()) * scale * ws
    return (y if bias is None else y + bias).to(dt)


def _rsqrt_mean(u, eps=1e-5):
    return torch.rsqrt((u * u).mean(-1, keepdim=True) + eps)


def _gated(s):
    c = s["case"]
    x, z, w = s["x"].float(), s["z"].float(), s["weight"].float()
    gate = z * torch.sigmoid(z)
    u = (x if c["norm_first"] else x * gate).unflatten(-1, (c["groups"], -1))
    y = (u * _rsqrt_mean(u)).flatten(-2) * w
    return (y * gate if c["norm_first"] else y).to(s["dtype"])


def _residual(s):
    c, u = s["case"], s["x"].float()
    if c["post"]:
        u = u * _rsqrt_mean(u) * s["post_weight"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    r = s["residual"].float() + c["scale"] * u
    return r * _rsqrt_mean(r) * s["weight"].float(), r.to(s["residual"].dtype)


def run(s):
    op, dt = s["case"]["op"], s["dtype"]
    if not own:
        if op == "gated":
            return _gated(s)
        if op in ("residual", "block"):
            y, r = _residual(s)
            return (_product(*_rows(y), s["w"], s["ws"], None, dt) if op == "block" else y.to(dt)), r
        rows = _rows(s["x"])
        y = _product(*rows, s["w"], s["ws"], s["bias"], dt)
        return (y, _product(*rows, s["w2"], s["ws2"], s["bias"], dt)) if op == "shared" else y
    pe, c = _package(), s["case"]
    if op == "linear":
        return pe.matmul_q8(s["x"], s["w"], s["ws"], bias=s["bias"])
    if op == "shared":
        q, scales = pe.quantize_q8(s["x"])
        return (pe.matmul_q8(q, s["w"], s["ws"], scales=scales, bias=s["bias"], dtype=dt),
                pe.matmul_q8(q, s["w2"], s["ws2"], scales=scales, bias=s["bias"], dtype=dt))
    if op == "gated":
        return pe.gated_norm(s["x"], s["weight"], s["z"], groups=c["groups"], norm_first=c["norm_first"])
    more = dict(post_weight=s["post_weight"], gate=s["gate"], scale=c["scale"])
    if op == "residual":
        return pe.residual_norm(s["x"], s["residual"], s["weight"], **more)
    (q, scales), r = pe.residual_norm(s["x"], s["residual"], s["weight"], quantize=True, **more)
    return pe.matmul_q8(q, s["w"], s["ws"], scales=scales, dtype=dt), r


# ------------------------------------------------------------ work and truth --

def work(case):
    e, op = 4 if case["dtype"] == "float32" else 2, case["op"]
    if op in ("linear", "shared"):
        m, n, k = case["m"], case["n"], case["k"]
        times = 2 if op == "shared" else 1
        return dict(bytes=e * m * k + times * (n * k + 4 * n + e * m * n) + (4 * n if case["bias"] else 0),
                    flops=times * 2 * m * n * k)
    rows, d = case["b"] * case["t"], case["d"]
    if op == "gated":
        return dict(bytes=e * (3 * rows * d + d), flops=12 * rows * d)
    r = 4 if case["wide"] else e
    gate = dict(none=0, channel=d, sequence=case["b"] * d, token=rows, full=rows * d)[case["gate"]]
    into = rows * d * (e + 2 * r) + e * (gate + d + (d if case["post"] else 0))
    if op == "residual":
        return dict(bytes=into + e * rows * d, flops=12 * rows * d)
    n = case["n"]
    return dict(bytes=into + n * d + 4 * n + e * rows * n, flops=12 * rows * d + 2 * rows * n * d)


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}

    def linear(x, names):
        top = torch.linalg.vector_norm(x, math.inf, -1)
        level = torch.where(top > 0, top, 1.0)[..., None]
        q = torch.round(127 * x / level)                     # (ties to even)
        out = []
        for w, ws in names:
            y = (q @ f[w].t().contiguous()) * f[ws]
            y *= (top / 127)[..., None]
            out.append(y + f["bias"] if s["bias"] is not None else y)
        return out

    if op == "linear":
        return linear(f["x"], [("w", "ws")])[0]
    if op == "shared":
        return tuple(linear(f["x"], [("w", "ws"), ("w2", "ws2")]))

    def norm(u, parts=1):
        shape = u.shape
        u = u.reshape(*shape[:-1], parts, shape[-1] // parts)
        return (u / torch.sqrt(u.square().sum(-1, keepdim=True) / u.shape[-1] + 1e-5)).reshape(shape)

    if op == "gated":
        gate = f["z"] / (1 + torch.exp(-f["z"]))
        if case["norm_first"]:
            return norm(f["x"], case["groups"]) * f["weight"] * gate
        return norm(f["x"] * gate, case["groups"]) * f["weight"]
    u = norm(f["x"]) * f["post_weight"] if case["post"] else f["x"]
    r = f["residual"] + case["scale"] * (u if s["gate"] is None else u * f["gate"])
    y = norm(r) * f["weight"]
    return (linear(y, [("w", "ws")])[0] if op == "block" else y), r
