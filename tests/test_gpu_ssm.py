"""Short causal convolution and selective scan on the GPU against their
definitions in 64 bits, token by token."""
import pytest
import torch

import ssm_util as u

pytestmark = pytest.mark.gpu


def _within(got, ref, bound, what):
    err = (got.double().cpu() - ref).abs()
    assert bool(torch.isfinite(got).all()), what
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


# --------------------------------------------------------------- convolution --

def _conv_case(dtype, lens, D, W, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    x = torch.randn(T, D, generator=g).to(dtype)
    w = torch.randn(D, W, generator=g).to(dtype)
    b = torch.randn(D, generator=g).to(dtype)
    st = torch.randn(len(lens), W - 1, D, generator=g).to(dtype)
    return x, w, b, st


def _check_conv(y, state, x, w, b, act, st, lens, dtype):
    at = 0
    for i, n in enumerate(lens):
        ref, last, size = u.conv(x[at:at + n], w, b, act, st[i])
        _within(y[at:at + n], ref, u.conv_bound(ref, size, dtype), f"sequence {i} of {n}")
        assert torch.equal(state[i].cpu().double(), last), f"state {i}"
        at += n


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("W", [2, 3, 4, 8])
@pytest.mark.parametrize("lens,D", [([1, 0, 5, 40, 0, 2, 33], 50), ([70], 7), ([0], 8), ([3, 3, 64, 31, 0], 64)])
def test_conv_packed(dtype, W, lens, D):
    from pto_einsum import causal_conv

    x, w, b, st = _conv_case(dtype, lens, D, W)
    print(f"causal_conv {dtype} lens {lens} D {D} W {W}", flush=True)
    y, state = causal_conv(x.cuda(), w.cuda(), b.cuda(), activation="silu", initial_state=st.cuda(),
                           cu_seqlens=_cu(lens))
    _check_conv(y, state, x, w, b, True, st, lens, dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("b,T,D,act,bias", [(3, 37, 40, True, True), (2, 1, 9, False, False), (1, 200, 513, True, False),
                                            (2, 2, 16, False, True)])
def test_conv_dense(dtype, b, T, D, act, bias):
    from pto_einsum import causal_conv

    lens = [T] * b
    x, w, bb, _ = _conv_case(dtype, lens, D, 4, seed=b)
    st = torch.zeros(b, 3, D, dtype=dtype)
    bb = bb if bias else None
    print(f"causal_conv {dtype} dense {b} x {T} x {D}", flush=True)
    y, state = causal_conv(x.reshape(b, T, D).cuda(), w.cuda(), None if bb is None else bb.cuda(),
                           activation="silu" if act else None)
    _check_conv(y.reshape(b * T, D), state, x, w, bb, act, st, lens, dtype)


def test_conv_empty_and_tail():
    """No tokens keep the state; tokens past the last offset give zeros and are
    in nobody's state; offsets past the buffer end at it."""
    from pto_einsum import causal_conv

    x, w, b, st = _conv_case(torch.float16, [20], 24, 4)
    xc, wc, sc = x.cuda(), w.cuda(), st.cuda()
    y, state = causal_conv(xc.reshape(1, 20, 24)[:, :0], wc, initial_state=sc)
    assert y.shape == (1, 0, 24) and torch.equal(state, sc)
    y, state = causal_conv(xc, wc, initial_state=torch.cat([sc, sc]), cu_seqlens=_cu([5, 7]))
    _check_conv(y[:12], state, x[:12], w, None, False, torch.cat([st, st]), [5, 7], torch.float16)
    assert bool((y[12:] == 0).all())
    y, state = causal_conv(xc, wc, initial_state=sc, cu_seqlens=torch.tensor([0, 99], dtype=torch.int32).cuda())
    _check_conv(y, state, x, w, None, False, st, [20], torch.float16)


def test_conv_strides_and_alignment():
    """Channels sliced from a wider tensor at an odd offset."""
    from pto_einsum import causal_conv, causal_conv_step

    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 50, 101, generator=g).half()
    w = torch.randn(60, 4, generator=g).half()
    zero = torch.zeros(2, 3, 60).half()
    part = wide.cuda()[:, :, 3:63]
    y, state = causal_conv(part, w.cuda())
    _check_conv(y.reshape(100, 60), state, wide[:, :, 3:63].reshape(100, 60), w, None, False, zero, [50, 50],
                torch.float16)
    st = state.clone()
    y1 = causal_conv_step(part[:, 7], w.cuda(), st)
    y2, st2 = causal_conv(part[:, 7:8], w.cuda(), initial_state=state)
    assert torch.equal(y1, y2[:, 0]) and torch.equal(st, st2)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("W", [2, 4, 5])
def test_conv_step(dtype, W):
    """Tokens one by one give a prompt's outputs and states; other slots stay, a
    slot outside the cache is a row without a sequence."""
    from pto_einsum import causal_conv, causal_conv_step

    g = torch.Generator().manual_seed(W)
    B, S, D, T = 3, 6, 37, 5
    x = torch.randn(B, T, D, generator=g).to(dtype).cuda()
    w = torch.randn(D, W, generator=g).to(dtype).cuda()
    b = torch.randn(D, generator=g).to(dtype).cuda()
    cache = torch.randn(S, W - 1, D, generator=g).to(dtype).cuda()
    before = cache.clone()
    slots = torch.tensor([4, -1, 2], dtype=torch.int32).cuda()
    y, state = causal_conv(x, w, b, activation="silu", initial_state=cache[[4, 0, 2]])
    for t in range(T):
        got = causal_conv_step(x[:, t], w, cache, b, activation="silu", slots=slots)
        assert torch.equal(got[[0, 2]], y[[0, 2], t]) and bool((got[1] == 0).all())
    assert torch.equal(cache[[4, 2]], state[[0, 2]])
    assert torch.equal(cache[[0, 1, 3, 5]], before[[0, 1, 3, 5]])
    slots[1] = S
    assert bool((causal_conv_step(x[:, 0], w, cache, b, slots=slots)[1] == 0).all())
    assert causal_conv_step(x[:0, 0], w, cache, b).shape == (0, D)


def test_conv_non_finite_stays():
    """A non-finite input reaches width - 1 later tokens of its channel alone."""
    from pto_einsum import causal_conv

    x, w, b, st = _conv_case(torch.bfloat16, [30, 30], 16, 4)
    x[10, 3], x[29, 5] = float("nan"), float("inf")
    y, _ = causal_conv(x.cuda(), w.cuda(), b.cuda(), initial_state=st.cuda(), cu_seqlens=_cu([30, 30]))
    bad = torch.zeros(60, 16, dtype=torch.bool)
    bad[10:14, 3] = True
    bad[29, 5] = True
    assert torch.equal(~torch.isfinite(y.cpu()), bad)


# --------------------------------------------------------------------- scan --

def _scan_case(dtype, lens, H, P, G, N, seed=0, gate=True, dt32=False, rate=(1.0, 16.0), step=(1e-3, 1e-1)):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    x = torch.randn(T, H, P, generator=g).to(dtype)
    B = torch.randn(T, G, N, generator=g).to(dtype)
    C = torch.randn(T, G, N, generator=g).to(dtype)
    z = torch.randn(T, H, P, generator=g).to(dtype) if gate else None
    dt = torch.randn(T, H, generator=g).to(torch.float32 if dt32 else dtype)
    d0 = torch.empty(H).uniform_(step[0], step[1], generator=g)
    bias = d0 + torch.log(-torch.expm1(-d0))
    A = -torch.empty(H).uniform_(rate[0], rate[1], generator=g)
    D = torch.rand(H, generator=g)
    st = torch.randn(len(lens), H, P, N, generator=g)
    return dict(x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=bias, st=st)


def _cuda(v):
    return None if v is None else v.cuda()


def _call(c, lens=None, dense=None, state=True):
    from pto_einsum import selective_scan

    t = {k: _cuda(v) for k, v in c.items()}
    if dense is not None:
        for k in ("x", "dt", "B", "C", "z"):
            t[k] = None if t[k] is None else t[k].unflatten(0, (dense, -1))
    return selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                          dt_softplus=True, initial_state=t["st"] if state else None,
                          cu_seqlens=None if lens is None else _cu(lens))


def _check_scan(y, state, c, lens, dtype, have_state=True):
    at = 0
    N = c["B"].shape[-1]
    for i, n in enumerate(lens):
        cut = slice(at, at + n)
        st = c["st"][i] if have_state else torch.zeros_like(c["st"][i])
        ry, rs, ya, sa = u.scan(c["x"][cut], c["dt"][cut], c["A"], c["B"][cut], c["C"][cut], c["D"],
                                None if c["z"] is None else c["z"][cut], c["dt_bias"], True, st)
        rel = u.scan_bound(n, N, 0, 0)
        _within(y[cut], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], f"y of sequence {i} ({n})")
        _within(state[i], rs, rel * sa + 1e-37, f"state of sequence {i} ({n})")
        if n >= 16:
            # Roundings of random sign: a surviving term makes some 4 sqrt(T) of
            # them, sums as many; and one to dtype for y.
            far = float((state[i].cpu().double() - rs).norm() / rs.norm())
            assert far <= 2.0 ** -24 * 8 * max(n, 16) ** 0.5, f"state of sequence {i}: {far:.3g}"
            far = float((y[cut].cpu().double() - ry).norm() / ry.norm())
            assert far <= 1.2 * u.HALF[dtype] + 2.0 ** -24 * 16 * max(n, 16) ** 0.5, f"y of sequence {i}: {far:.3g}"
        at += n


SHAPES = [
    # lens, H, P, G, N
    ([1, 0, 5, 64, 65, 0, 130], 4, 16, 2, 16),
    ([200], 2, 64, 1, 128),
    ([63, 129], 6, 33, 3, 20),        # nothing a whole tile
    ([300, 40], 3, 80, 1, 100),
    ([70], 5, 128, 5, 64),            # a group for every head
    ([100, 28], 1, 7, 1, 256),
    ([90], 2, 40, 2, 200),
    ([50], 9, 64, 1, 32),             # more heads than a block's, odd
    ([17], 2, 1, 1, 1),
]


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("lens,H,P,G,N", SHAPES)
def test_scan_packed(dtype, lens, H, P, G, N):
    c = _scan_case(dtype, lens, H, P, G, N, seed=P)
    print(f"selective_scan {dtype} lens {lens} H {H} P {P} G {G} N {N}", flush=True)
    y, state = _call(c, lens)
    _check_scan(y, state, c, lens, dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("b,T,H,P,G,N,gate,state", [
    (2, 1, 4, 64, 1, 128, True, True), (3, 64, 4, 32, 2, 64, False, False), (2, 70, 8, 64, 2, 128, True, False),
    (1, 700, 4, 64, 1, 64, False, True), (1, 1500, 2, 48, 1, 128, True, True), (5, 2, 3, 5, 1, 3, False, True)])
def test_scan_dense(dtype, b, T, H, P, G, N, gate, state):
    c = _scan_case(dtype, [T] * b, H, P, G, N, seed=T, gate=gate, dt32=True)
    print(f"selective_scan {dtype} dense {b} x {T} H {H} P {P} G {G} N {N}", flush=True)
    y, st = _call(c, dense=b, state=state)
    _check_scan(y.flatten(0, 1), st, c, [T] * b, dtype, state)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
def test_scan_decay_extremes(dtype):
    """Decays from none (steps of 0) to complete within a token, in one chunk and
    over chunks."""
    T, H = 260, 6
    c = _scan_case(dtype, [T], H, 32, 1, 64, seed=1, dt32=True, gate=False)
    c["dt_bias"], c["dt"] = None, c["dt"].abs() * 0.05
    c["A"] = torch.tensor([-0.0, -1e-3, -1.0, -30.0, -1000.0, -1.0])
    c["dt"][100:160] = 0.0
    c["dt"][:, 5] *= 20.0
    from pto_einsum import selective_scan

    t = {k: _cuda(v) for k, v in c.items()}
    y, st = selective_scan(t["x"][None], t["dt"][None], t["A"], t["B"][None], t["C"][None], D=t["D"],
                           initial_state=t["st"])
    ry, rs, ya, sa = u.scan(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], None, None, False, c["st"][0])
    # An exponent A d summed to s is off by at most 2^-23 s, which counts while
    # exp(s) does: s exp(s) <= 0.37 of a term.
    rel = u.scan_bound(T, 64, 0, 0)
    _within(y[0], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], "y")
    _within(st[0], rs, rel * sa + 1e-37, "state")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("scale_x,scale_b,scale_c", [(1e-3, 1.0, 1.0), (1.0, 1e-3, 1e-3), (100.0, 30.0, 1e-2),
                                                     (1e-4, 1e-4, 100.0)])
def test_scan_magnitudes(dtype, scale_x, scale_b, scale_c):
    """Small and large operands keep float32 states (float16's range is narrow)."""
    c = _scan_case(dtype, [150], 4, 32, 1, 64, seed=2, gate=False)
    c["x"], c["B"], c["C"] = (c["x"].float() * scale_x).to(dtype), (c["B"].float() * scale_b).to(dtype), \
        (c["C"].float() * scale_c).to(dtype)
    c["st"] *= scale_x * scale_b
    y, state = _call(c, dense=1)
    _check_scan(y[0], state, c, [150], dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
def test_scan_non_finite_stays(dtype, value):
    """A non-finite x at token 70 reaches tokens from 70 on of its own channel
    alone; non-finite B and C their tokens and those after; other sequences
    nothing."""
    lens, H, P, N = [100, 100], 3, 40, 32
    c = _scan_case(dtype, lens, H, P, 1, N, seed=5)
    clean, cstate = _call(c, lens)
    x = c["x"].clone()
    x[70, 1, 7] = value
    y, state = _call({**c, "x": x}, lens)
    bad = torch.zeros(200, H, P, dtype=torch.bool)
    bad[70:100, 1, 7] = True
    assert bool((~torch.isfinite(y.cpu()[70, 1, 7])).all()) and bool((~torch.isfinite(state.cpu()[0, 1, 7])).all())
    assert bool(torch.isfinite(y.cpu()[~bad]).all())
    _check_scan(torch.where(bad, clean.cpu(), y.cpu()), cstate, c, lens, dtype)
    assert bool(torch.isfinite(state.cpu()[1]).all())
    C = c["C"].clone()
    C[70, 0, 3] = value
    y, state = _call({**c, "C": C}, lens)
    _check_scan(torch.cat([y[:70], clean[70:71], y[71:]]), state, c, lens, dtype)
    assert bool((~torch.isfinite(y[70])).all())
    B = c["B"].clone()
    B[70, 0, 3] = value
    y, state = _call({**c, "B": B}, lens)
    assert bool((~torch.isfinite(y[70:100])).any()) and bool(torch.isfinite(y[100:]).all())
    _check_scan(torch.cat([y[:70], clean[70:100], y[100:]]), cstate, c, lens, dtype)


def test_scan_empty_and_tail():
    from pto_einsum import selective_scan

    c = _scan_case(torch.bfloat16, [100], 2, 32, 1, 64, seed=6)
    t = {k: _cuda(v) for k, v in c.items()}
    more = dict(D=t["D"], dt_bias=t["dt_bias"], dt_softplus=True)
    y, st = selective_scan(t["x"][None, :0], t["dt"][None, :0], t["A"], t["B"][None, :0], t["C"][None, :0],
                           initial_state=t["st"], **more)
    assert y.shape == (1, 0, 2, 32) and torch.equal(st, t["st"])
    y, st = selective_scan(t["x"][None, :0], t["dt"][None, :0], t["A"], t["B"][None, :0], t["C"][None, :0], **more)
    assert bool((st == 0).all())
    # tokens past the last offset, and an offset past the buffer
    two = torch.cat([t["st"], t["st"]])
    y, st = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], z=t["z"], initial_state=two, cu_seqlens=_cu([5, 20]),
                           **more)
    c2 = {**c, "st": torch.cat([c["st"], c["st"]])}
    _check_scan(y[:25], st, c2, [5, 20], torch.bfloat16)
    assert bool((y[25:] == 0).all())
    y, st = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], z=t["z"], initial_state=t["st"],
                           cu_seqlens=torch.tensor([0, 1000], dtype=torch.int32).cuda(), **more)
    _check_scan(y, st, c, [100], torch.bfloat16)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
def test_scan_strides(dtype):
    """x, B, C as slices of one tensor at odd offsets, heads in another order, z
    and dt strided; the same values laid out give the same results."""
    from pto_einsum import selective_scan

    g = torch.Generator().manual_seed(8)
    H, P, G, N, T = 4, 24, 2, 40, 90
    wide = torch.randn(2, T, 1 + H * P + 2 * G * N, generator=g).to(dtype).cuda()
    x = wide[..., 1:1 + H * P].unflatten(-1, (H, P))
    B = wide[..., 1 + H * P:1 + H * P + G * N].unflatten(-1, (G, N))
    C = wide[..., 1 + H * P + G * N:].unflatten(-1, (G, N))
    z = torch.randn(2, H, T, P, generator=g).to(dtype).cuda().transpose(1, 2)
    dt = torch.rand(2, H, T, generator=g).to(dtype).cuda().transpose(1, 2) * 0.1
    A = -torch.rand(2 * H, generator=g).cuda()[::2] * 4
    y, st = selective_scan(x, dt, A, B, C, z=z)
    y2, st2 = selective_scan(*(v.contiguous() for v in (x, dt, A, B, C)), z=z.contiguous())
    for i in range(2):
        ry, rs, ya, sa = u.scan(x[i].cpu(), dt[i].cpu(), A.cpu(), B[i].cpu(), C[i].cpu(), None, z[i].cpu(), None,
                                False, torch.zeros(H, P, N))
        rel = u.scan_bound(T, N, 0, 0)
        for yy, ss in ((y, st), (y2, st2)):
            _within(yy[i], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], "y")
            _within(ss[i], rs, rel * sa + 1e-37, "state")


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("H,P,G,N", [(4, 64, 1, 128), (6, 33, 3, 20), (2, 5, 1, 256), (3, 16, 3, 16), (2, 80, 2, 63)])
def test_scan_step(dtype, H, P, G, N):
    """Single tokens against the definition; other slots stay."""
    from pto_einsum import selective_scan_step

    n, S = 3, 5
    c = _scan_case(dtype, [n], H, P, G, N, seed=N)
    t = {k: _cuda(v) for k, v in c.items()}
    cache = torch.randn(S, H, P, N, generator=torch.Generator().manual_seed(1))
    state = cache.cuda()
    slots = torch.tensor([3, -5, 0], dtype=torch.int32).cuda()
    print(f"selective_scan_step {dtype} H {H} P {P} G {G} N {N}", flush=True)
    y = selective_scan_step(t["x"], t["dt"], t["A"], t["B"], t["C"], state, D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                            dt_softplus=True, slots=slots)
    assert bool((y[1] == 0).all()) and torch.equal(state[[1, 2, 4]].cpu(), cache[[1, 2, 4]])
    rel = u.scan_bound(1, N, 0, 0)
    for row, slot in ((0, 3), (2, 0)):
        cut = slice(row, row + 1)
        ry, rs, ya, sa = u.scan(c["x"][cut], c["dt"][cut], c["A"], c["B"][cut], c["C"][cut], c["D"], c["z"][cut],
                                c["dt_bias"], True, cache[slot])
        _within(y[cut], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], "y")
        _within(state[slot], rs, rel * sa + 1e-37, "state")


def test_scan_step_continues_a_prompt():
    """A prompt in two parts, and its tokens one by one, give the whole one's."""
    from pto_einsum import selective_scan, selective_scan_step

    c = _scan_case(torch.float32, [140], 4, 32, 2, 64, seed=9)
    t = {k: _cuda(v) for k, v in c.items()}
    more = dict(D=t["D"], dt_bias=t["dt_bias"], dt_softplus=True)

    def part(a, b, st):
        return selective_scan(*(t[k][None, a:b] if k != "A" else t[k] for k in ("x", "dt", "A", "B", "C")),
                              z=t["z"][None, a:b], initial_state=st, **more)

    y, st = part(0, 140, t["st"])
    y1, s1 = part(0, 77, t["st"])
    y2, s2 = part(77, 130, s1)
    state = s2.clone()
    ys = [selective_scan_step(*(t[k][i:i + 1] if k != "A" else t[k] for k in ("x", "dt", "A", "B", "C")), state,
                              z=t["z"][i:i + 1], **more) for i in range(130, 140)]
    _check_scan(torch.cat([y1[0], y2[0], *ys]), state, c, [140], torch.float32)
    _check_scan(y[0], st, c, [140], torch.float32)


def test_scan_is_deterministic_and_captured():
    """Replays of a captured layer step and prompt are bit-identical to eager
    calls, on inputs that change between replays and on another stream."""
    from pto_einsum import StageGraph, causal_conv, causal_conv_step, selective_scan, selective_scan_step

    H, P, G, N, T, Bn = 8, 64, 2, 128, 300, 2
    g = torch.Generator().manual_seed(4)
    width = H * P + 2 * G * N
    u_in = torch.randn(Bn, T, width, generator=g).half().cuda()
    w = (torch.randn(width, 4, generator=g) * 0.5).half().cuda()
    dt = torch.randn(Bn, T, H, generator=g).half().cuda()
    A = -torch.rand(H, generator=g).cuda() * 8
    bias = torch.full((H,), -3.0).cuda()
    tok, tok_dt = u_in[:, 0].clone(), dt[:, 0].clone()
    cs, ss = torch.zeros(Bn, 3, width).half().cuda(), torch.zeros(Bn, H, P, N).cuda()

    def cut(v):
        return (v[..., :H * P].unflatten(-1, (H, P)), v[..., H * P:H * P + G * N].unflatten(-1, (G, N)),
                v[..., H * P + G * N:].unflatten(-1, (G, N)))

    def stage():
        v, conv_state = causal_conv(u_in, w, activation="silu")
        x, B, C = cut(v)
        y, state = selective_scan(x, dt, A, B, C, dt_bias=bias, dt_softplus=True)
        cs.copy_(conv_state)
        ss.copy_(state)
        x, B, C = cut(causal_conv_step(tok, w, cs, activation="silu"))
        y1 = selective_scan_step(x, tok_dt, A, B, C, ss, dt_bias=bias, dt_softplus=True)
        return y, y1, cs, ss

    graph = StageGraph(stage)
    side = torch.cuda.Stream()
    for i in range(3):
        u_in.copy_(torch.randn(Bn, T, width, generator=g).half())
        tok.copy_(torch.randn(Bn, width, generator=g).half())
        got = [v.clone() for v in graph.replay()]
        torch.cuda.synchronize()
        want = [v.clone() for v in stage()]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [v.clone() for v in stage()]
        side.synchronize()
        for a, b in zip(again, want):
            assert torch.equal(a, b)
