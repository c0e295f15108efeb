"""The serving operators of a state-space layer: the short causal convolution,
the selective scan (both for prompts and for single tokens) and the
matrix-vector product with 4-bit weights that projects one token.

  conv       causal_conv(x, weight, bias, ...)                 a prompt
  conv_step  causal_conv_step(x, weight, state, bias, ...)     a token
  scan       selective_scan(x, dt, A, B, C, ...)               a prompt
  scan_step  selective_scan_step(x, dt, A, B, C, state, ...)   a token
  q4         matvec_q4(x, packed, scales, zeros, ...)          few tokens

Inputs are drawn on the GPU from the seed.  A prompt is either a dense batch
(``lens`` empty) or several sequences packed one after another (``lens`` gives
their lengths).  As in a layer, x, B and C of the scan are slices of the
convolution's output and so lie at a token stride of their sum.
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
        # Four prompts of 4096 tokens, the channels of 64 heads of 64 and of B
        # and C: the largest convolution.
        dict(name="conv_large", op="conv", b=4, t=4096, lens="", d=4352, w=4, silu=True, state=False, dtype="float16"),
        # A packed batch of unequal prompts that continue earlier ones (a
        # chunked prefill), channels and lengths odd.
        dict(name="conv_ragged", op="conv", b=6, t=0, lens="1 700 33 2051 5 1203", d=1283, w=3, silu=True, state=True,
             dtype="bfloat16"),
        # One token of each of 64 sequences.
        dict(name="conv_token", op="conv_step", b=64, slots=96, d=4352, w=4, silu=True, dtype="bfloat16"),
        # Two prompts of 4096 tokens with gate and skip: the largest scan in
        # the type that the contractions take.
        dict(name="scan_large", op="scan", b=2, t=4096, lens="", h=64, p=64, g=1, n=128, gate=True, state=False,
             dtype="float16"),
        # One long prompt and few heads: little parallel work but along time.
        dict(name="scan_long", op="scan", b=1, t=16384, lens="", h=24, p=64, g=8, n=128, gate=True, state=False,
             dtype="bfloat16"),
        # Unequal packed prompts that continue, with odd head sizes.
        dict(name="scan_ragged", op="scan", b=6, t=0, lens="1 700 33 2051 5 1203", h=10, p=80, g=2, n=100, gate=False,
             state=True, dtype="bfloat16"),
        # A short prompt in float32: a small call.
        dict(name="scan_float32", op="scan", b=2, t=500, lens="", h=16, p=32, g=1, n=16, gate=True, state=True,
             dtype="float32"),
        # One token of one sequence, where latency counts.
        dict(name="scan_token", op="scan_step", b=1, slots=4, h=32, p=64, g=1, n=128, gate=True, dtype="float16"),
        # One token of each of 128 sequences: the states are read and written.
        dict(name="scan_tokens", op="scan_step", b=128, slots=160, h=64, p=64, g=8, n=128, gate=True, dtype="bfloat16"),
        # A projection of one token.
        dict(name="q4_token", op="q4", m=1, n=4096, k=4096, group=128, zeros=False, dtype="float16"),
        # An up projection of a batch of 16 tokens, with zero points.
        dict(name="q4_batch", op="q4", m=16, n=16384, k=8192, group=64, zeros=True, dtype="bfloat16"),
        # Sizes that are no whole tiles or groups, float32 activations.
        dict(name="q4_odd", op="q4", m=5, n=1001, k=2500, group=32, zeros=True, dtype="float32"),
    ]


# ------------------------------------------------------------------ drawing --

def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], as it falls or rounded to a
    multiple of 8 or 64."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    step = rng.choice([1, 1, 8, 64])
    return min(hi, max(lo, n // step * step))


def _prompts(rng, most):
    """Either b prompts of t tokens or packed lengths, most tokens in all."""
    b = _size(rng, 1, 16)
    if rng.random() < 0.5:
        return dict(b=b, t=_size(rng, 1, max(1, min(16384, most // b))), lens="")
    lens = [_size(rng, 1, max(1, min(4096, most // b))) for _ in range(b)]
    return dict(b=b, t=0, lens=" ".join(map(str, lens)))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan_step", "q4", "q4"])
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    if op == "conv":
        d = _size(rng, 32, 8192)
        return dict(op=op, **_prompts(rng, (1 << 25) // d), d=d, w=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.7,
                    state=rng.random() < 0.5, dtype=dtype)
    if op == "conv_step":
        b = _size(rng, 1, 256)
        return dict(op=op, b=b, slots=b + rng.randint(0, 32), d=_size(rng, 32, 8192), w=rng.choice([2, 3, 4, 4]),
                    silu=rng.random() < 0.7, dtype=dtype)
    if op == "q4":
        n = _size(rng, 64, 16384)
        return dict(op=op, m=_size(rng, 1, 32), n=n, k=_size(rng, 64, 8192), group=rng.choice([32, 64, 128]),
                    zeros=rng.random() < 0.5, dtype=dtype)
    g = rng.choice([1, 1, 2, 4, 8])
    h = g * rng.randint(1, 64 // g)
    p = rng.choice([16, 32, 64, 64, 80, 128, rng.randint(8, 128)])
    n = rng.choice([16, 32, 64, 128, 128, 256, rng.randint(8, 256)])
    if op == "scan":
        return dict(op=op, **_prompts(rng, min(16384, (1 << 32) // (h * p * max(n, 64)))), h=h, p=p, g=g, n=n,
                    gate=rng.random() < 0.6, state=rng.random() < 0.5, dtype=dtype)
    b = _size(rng, 1, max(1, min(256, (1 << 26) // (h * p * n))))
    return dict(op=op, b=b, slots=b + rng.randint(0, 8), h=h, p=p, g=g, n=n, gate=rng.random() < 0.6, dtype=dtype)


# ------------------------------------------------------------------- inputs --

def _lens(case):
    return [int(x) for x in case["lens"].split()]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 41)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo

    s = dict(case=case, dtype=dt)
    if op == "q4":
        m, n, k, grp = case["m"], case["n"], case["k"], case["group"]
        ng = -(-k // grp)
        s.update(x=normal(m, k),
                 packed=torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8),
                 # weights of about 1 / sqrt(k): the 16 levels span some five
                 # standard deviations
                 scales=(uniform(0.7, 1.3, n, ng) * (0.3 / math.sqrt(k))).to(dt),
                 zeros=torch.randint(4, 12, (n, ng), generator=g, device=DEV).to(dt) if case["zeros"] else None)
        return s
    lens = _lens(case) if "lens" in case else []
    seqs = case["b"]
    if lens:
        s["lens"] = lens
        s["cu_seqlens"] = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)
    # leading axes of a prompt's, or of a token's, tensors
    lead = (sum(lens),) if lens else (seqs, case["t"]) if "t" in case else (seqs,)
    if "slots" in case:
        s["slots"] = torch.randperm(case["slots"], generator=g, device=DEV)[:seqs].to(torch.int32)
    if op in ("conv", "conv_step"):
        d, w = case["d"], case["w"]
        s.update(x=normal(*lead, d), weight=normal(d, w, scale=w ** -0.5), bias=normal(d, scale=0.1))
        if op == "conv_step":
            s["state"] = normal(case["slots"], w - 1, d)
        else:
            s["initial_state"] = normal(seqs, w - 1, d) if case["state"] else None
        return s
    h, p, gr, n = case["h"], case["p"], case["g"], case["n"]
    xbc = normal(*lead, h * p + 2 * gr * n)
    s["x"] = xbc[..., :h * p].unflatten(-1, (h, p))
    s["B"] = xbc[..., h * p:h * p + gr * n].unflatten(-1, (gr, n))
    s["C"] = xbc[..., h * p + gr * n:].unflatten(-1, (gr, n))
    s["z"] = normal(*lead, h, p) if case["gate"] else None
    s["dt"] = normal(*lead, h)
    # step sizes of 0.001 to 0.1 around dt = 0, decay rates of 1 to 16
    step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), h))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["A"] = -uniform(1.0, 16.0, h)
    s["D"] = uniform(0.5, 1.5, h)
    if op == "scan_step":
        s["state"] = torch.randn((case["slots"], h, p, n), generator=g, device=DEV)
    else:
        s["initial_state"] = torch.randn((seqs, h, p, n), generator=g, device=DEV) if case["state"] else None
    return s


# --------------------------------------------------------------- plain forms --

def _silu(x):
    return x * torch.sigmoid(x)


def _padded_index(s):
    """Packed sequences as rows of equal length: the token at each place, and
    whether there is one."""
    start = s["cu_seqlens"][:-1].long()
    n = s["cu_seqlens"][1:].long() - start
    at = torch.arange(max(s["lens"]), device=DEV)
    return start[:, None] + torch.minimum(at[None], (n - 1)[:, None]), at[None] < n[:, None], n


def _conv(s):
    x, w = s["x"], s["case"]["w"]
    if "lens" in s:
        index, there, n = _padded_index(s)
        x = x[index] * there[..., None]
    else:
        n = torch.full((x.shape[0],), x.shape[1], device=DEV)
    first = s["initial_state"]
    before = torch.zeros((x.shape[0], w - 1, x.shape[2]), dtype=x.dtype, device=DEV) if first is None else first
    line = torch.cat([before, x], 1)
    y = (line.float().unfold(1, w, 1) * s["weight"].float()).sum(-1) + s["bias"].float()
    y = (_silu(y) if s["case"]["silu"] else y).to(x.dtype)
    last = n[:, None] + torch.arange(w - 1, device=DEV)
    state = line[torch.arange(x.shape[0], device=DEV)[:, None], last]
    return (y[there] if "lens" in s else y), state


def _conv_step(s):
    slots = s["slots"].long()
    line = torch.cat([s["state"][slots], s["x"][:, None]], 1)
    y = (line.float() * s["weight"].float().t()).sum(1) + s["bias"].float()
    s["state"][slots] = line[:, 1:]
    return (_silu(y) if s["case"]["silu"] else y).to(s["x"].dtype), s["state"]


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan(s):
    """The scan in chunks of q tokens: products within a chunk, the chunks'
    states, and the states at the chunks' starts as products over chunks."""
    c = s["case"]
    x, dt, bm, cm, z = s["x"], s["dt"], s["B"], s["C"], s["z"]
    if "lens" in s:
        index, there, _ = _padded_index(s)
        x, bm, cm = x[index], bm[index], cm[index]
        z = None if z is None else z[index]
        step = _softplus(dt[index].float() + s["dt_bias"]) * there[..., None]
    else:
        step = _softplus(dt.float() + s["dt_bias"])
    b, t, h, p, n, q = x.shape[0], x.shape[1], c["h"], c["p"], c["n"], 64
    nc = -(-t // q)
    rep = h // c["g"]

    def chunks(v):
        """[b, t, heads, k] -> [b, heads, chunks, q, k], zero past the end."""
        v = torch.cat([v.float(), torch.zeros((b, nc * q - t, *v.shape[2:]), device=DEV)], 1)
        return v.unflatten(1, (nc, q)).permute(0, 3, 1, 2, 4)

    xs, bs, cs = chunks(x), chunks(bm), chunks(cm)
    ds = chunks(step[..., None])[..., 0]                               # [b, h, nc, q]
    # sums of the exponents in 64 bits: their differences are what counts
    run_sum = torch.cumsum(ds.double() * s["A"].double()[:, None, None], -1)
    total = run_sum[..., -1]                                           # [b, h, nc]
    lower = torch.tril(torch.ones(q, q, dtype=torch.bool, device=DEV))
    decay = torch.where(lower, run_sum[..., :, None] - run_sum[..., None, :], -math.inf).float().exp()
    score = torch.matmul(cs, bs.transpose(-1, -2).contiguous()).repeat_interleave(rep, 1)
    y = torch.matmul(score * decay * ds[..., None, :], xs)
    # what each chunk adds to the state, and the states at the chunks' starts
    left = (total[..., None] - run_sum).float().exp() * ds
    add = torch.matmul((xs * left[..., None]).transpose(-1, -2).contiguous(), bs.repeat_interleave(rep, 1))
    upto = torch.cumsum(total, -1)
    from0 = torch.zeros((b, h, 1), dtype=torch.float64, device=DEV)
    edges = torch.cat([from0, upto], -1)                               # [b, h, nc + 1]
    earlier = torch.tril(torch.ones(nc + 1, nc, dtype=torch.bool, device=DEV), -1)
    carry = torch.where(earlier, edges[..., :, None] - upto[..., None, :], -math.inf).float().exp()
    states = torch.matmul(carry, add.flatten(-2)).unflatten(-1, (p, n))  # [b, h, nc + 1, p, n]
    if s["initial_state"] is not None:
        states = states + edges.float().exp()[..., None, None] * s["initial_state"][:, :, None]
    read = torch.matmul(cs.repeat_interleave(rep, 1), states[:, :, :-1].transpose(-1, -2).contiguous())
    y = (y + read * run_sum.float().exp()[..., None]).permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :t]
    y = y + x.float() * s["D"][:, None]
    if z is not None:
        y = y * _silu(z.float())
    y = y.to(x.dtype)
    return (y[there] if "lens" in s else y), states[:, :, -1].contiguous()


def _scan_step(s):
    c, slots = s["case"], s["slots"].long()
    rep = c["h"] // c["g"]
    step = _softplus(s["dt"].float() + s["dt_bias"])
    bm, cm = (s[k].float().repeat_interleave(rep, 1) for k in ("B", "C"))
    x = s["x"].float()
    h = s["state"][slots] * (step * s["A"]).exp()[..., None, None] + (step[..., None] * x)[..., None] * bm[:, :, None]
    s["state"][slots] = h
    y = (h * cm[:, :, None]).sum(-1) + x * s["D"][:, None]
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(s["dtype"]), s["state"]


def _q4(s):
    k, grp = s["case"]["k"], s["case"]["group"]
    q = torch.stack([s["packed"] & 15, s["packed"] >> 4], -1).flatten(1)[:, :k].float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(grp, 1)[:, :k]
    w = (q - zero) * s["scales"].float().repeat_interleave(grp, 1)[:, :k]
    return torch.matmul(s["x"].float(), w.t()).to(s["dtype"])


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "q4": _q4}[op](s)
    pe = _package()
    if op == "q4":
        return pe.matvec_q4(s["x"], s["packed"], s["scales"], s["zeros"], group=s["case"]["group"])
    if op in ("conv", "conv_step"):
        act = "silu" if s["case"]["silu"] else None
        if op == "conv":
            return pe.causal_conv(s["x"], s["weight"], s["bias"], activation=act, initial_state=s["initial_state"],
                                  cu_seqlens=s.get("cu_seqlens"))
        return pe.causal_conv_step(s["x"], s["weight"], s["state"], s["bias"], activation=act,
                                   slots=s["slots"]), s["state"]
    more = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
    if op == "scan":
        return pe.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], initial_state=s["initial_state"],
                                 cu_seqlens=s.get("cu_seqlens"), **more)
    return pe.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], slots=s["slots"],
                                  **more), s["state"]


# ------------------------------------------------------------ work and truth --

def work(case):
    e, op = 4 if case["dtype"] == "float32" else 2, case["op"]
    if op == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = n * -(-k // case["group"]) * (2 if case["zeros"] else 1)
        return dict(bytes=n * ((k + 1) // 2) + e * (groups + m * (k + n)), flops=2 * m * n * k)
    tokens = sum(_lens(case)) or case["b"] * case["t"] if "lens" in case else case["b"]
    if op in ("conv", "conv_step"):
        d, w = case["d"], case["w"]
        rows = case["b"] * (w - 1) * (2 if op == "conv_step" or case["state"] else 1)
        return dict(bytes=e * d * (2 * tokens + rows + w + 1), flops=2 * tokens * d * w)
    h, p, n = case["h"], case["p"], case["n"]
    states = 2 if op == "scan_step" or case["state"] else 1
    return dict(bytes=e * tokens * (h * p * (3 if case["gate"] else 2) + 2 * case["g"] * n + h)
                + 4 * case["b"] * h * p * n * states + 12 * h,
                flops=tokens * h * (5 * p * n + 2 * p))


def exact(case, seed):
    """The definitions, token by token, in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op == "q4":
        n, k = case["n"], case["k"]
        q = torch.empty((n, 2 * s["packed"].shape[1]), dtype=torch.float64, device=DEV)
        q[:, 0::2], q[:, 1::2] = s["packed"].bitwise_and(15), s["packed"].div(16, rounding_mode="floor")
        group_of = torch.arange(k, device=DEV) // case["group"]
        q = q[:, :k] - (f["zeros"][:, group_of] if case["zeros"] else 8)
        return f["x"] @ (q * f["scales"][:, group_of]).t().contiguous()
    if op in ("conv", "conv_step"):
        w = case["w"]

        def conv(line):
            """Outputs of the rows from w - 1 on."""
            y = sum(f["weight"][:, j] * line[j:line.shape[0] - w + 1 + j] for j in range(w)) + f["bias"]
            return y / (1 + torch.exp(-y)) if case["silu"] else y

        if op == "conv_step":
            got = [conv(torch.cat([f["state"][slot], x[None]])) for slot, x in zip(s["slots"].tolist(), f["x"])]
            for slot, x in zip(s["slots"].tolist(), f["x"]):
                f["state"][slot] = torch.cat([f["state"][slot, 1:], x[None]])
            return torch.cat(got), f["state"]
        parts = torch.split(f["x"], s["lens"]) if "lens" in s else f["x"]
        zero = torch.zeros((w - 1, case["d"]), dtype=torch.float64, device=DEV)
        lines = [torch.cat([f["initial_state"][i] if case["state"] else zero, x]) for i, x in enumerate(parts)]
        ys = [conv(line) for line in lines]
        return torch.cat(ys) if "lens" in s else torch.stack(ys), torch.stack([v[len(v) - w + 1:] for v in lines])
    h, p, n = case["h"], case["p"], case["n"]
    rep = h // case["g"]
    step = f["dt"] + f["dt_bias"]
    step = torch.where(step > 30, step, torch.log(1 + torch.exp(step)))
    fade = torch.exp(step * f["A"])
    heads = torch.arange(h, device=DEV) // rep

    def token(state, at):
        """One token of some sequences: the new states and the outputs."""
        x = f["x"][at]
        state = state * fade[at][..., None, None] + (x * step[at][..., None])[..., None] * f["B"][at][..., heads, None, :]
        y = (state @ f["C"][at][..., heads, :, None])[..., 0] + x * f["D"][:, None]
        if case["gate"]:
            y = y * f["z"][at] / (1 + torch.exp(-f["z"][at]))
        return state, y

    if op == "scan_step":
        new, y = token(f["state"][s["slots"].long()], slice(None))
        f["state"][s["slots"].long()] = new
        return y, f["state"]
    y = torch.empty(f["x"].shape, dtype=torch.float64, device=DEV)
    zero = torch.zeros((case["b"], h, p, n), dtype=torch.float64, device=DEV)
    state = f["initial_state"] if case["state"] else zero
    if "lens" not in s:
        for t in range(case["t"]):
            state, y[:, t] = token(state, (slice(None), t))
        return y, state
    # packed sequences in step, the longest first
    order = sorted(range(case["b"]), key=lambda i: -s["lens"][i])
    starts = s["cu_seqlens"].long()[:-1][torch.tensor(order, device=DEV)]
    state = state[torch.tensor(order, device=DEV)].clone()
    for t in range(max(s["lens"])):
        live = sum(1 for v in s["lens"] if v > t)
        at = starts[:live] + t
        state[:live], y[at] = token(state[:live], at)
    back = torch.empty_like(state)
    back[torch.tensor(order, device=DEV)] = state
    return y, back
