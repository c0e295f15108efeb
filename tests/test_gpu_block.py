"""The norms, the 8-bit product and the state-space operators as a block of a layer
uses them: prompts, then single tokens, eager, captured and on another stream."""
import pytest
import torch

import rows_util as ru
import ssm_util

pytestmark = pytest.mark.gpu

HEADS, P, GROUPS, N, WIDTH, MODEL = 4, 32, 2, 16, 4, 96
INNER, BC = HEADS * P, GROUPS * N


class Block:
    """norm -> projection -> convolution -> scan -> norm with gate -> projection,
    twice, with a residual kept in float32."""

    def __init__(self, dtype):
        g = torch.Generator().manual_seed(11)

        def normal(*shape, scale=1.0):
            return torch.randn(shape, generator=g) * scale

        self.dtype = dtype
        self.host = [dict(norm=(1 + normal(MODEL, scale=0.1)).to(dtype), gate=normal(MODEL).to(dtype),
                          w_in=normal(INNER + INNER + 2 * BC + HEADS, MODEL, scale=MODEL ** -0.5).to(dtype),
                          w_out=normal(MODEL, INNER, scale=INNER ** -0.5).to(dtype),
                          conv=normal(INNER + 2 * BC, WIDTH, scale=0.5).to(dtype),
                          inner_norm=(1 + normal(INNER, scale=0.1)).to(dtype), dt_bias=normal(HEADS) - 3,
                          A=-torch.rand(HEADS, generator=g) * 8 - 1, D=normal(HEADS)) for _ in range(2)]
        from pto_einsum import quantize_q8

        self.gpu = []
        for p in self.host:
            q = {k: t.cuda() for k, t in p.items()}
            q["w_in"], q["w_out"] = quantize_q8(q["w_in"]), quantize_q8(q["w_out"])
            self.gpu.append(q)

    def caches(self, b):
        return [(torch.zeros(b, WIDTH - 1, INNER + 2 * BC, dtype=self.dtype, device="cuda"),
                 torch.zeros(b, HEADS, P, N, device="cuda")) for _ in self.gpu]

    def __call__(self, u, residual, caches, token):
        from pto_einsum import (causal_conv, causal_conv_step, gated_norm, matmul_q8, residual_norm, selective_scan,
                                selective_scan_step)

        states = []
        for p, (conv_state, state) in zip(self.gpu, caches):
            rows, residual = residual_norm(u, residual, p["norm"], gate=p["gate"], scale=0.5, quantize=True)
            z, xbc, dt = matmul_q8(rows[0], *p["w_in"], scales=rows[1], dtype=self.dtype).split(
                (INNER, INNER + 2 * BC, HEADS), -1)
            if token:
                xbc = causal_conv_step(xbc, p["conv"], conv_state, activation="silu")
            else:
                xbc, conv_state = causal_conv(xbc, p["conv"], activation="silu")
            x, B, C = xbc.split((INNER, BC, BC), -1)
            x, B, C = x.unflatten(-1, (HEADS, P)), B.unflatten(-1, (GROUPS, N)), C.unflatten(-1, (GROUPS, N))
            more = dict(D=p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
            if token:
                y = selective_scan_step(x, dt, p["A"], B, C, state, **more)
            else:
                y, state = selective_scan(x, dt, p["A"], B, C, **more)
            q, s = gated_norm(y.flatten(-2), p["inner_norm"], z, groups=GROUPS, quantize=True)
            u = matmul_q8(q, *p["w_out"], scales=s, dtype=self.dtype)
            states.append((conv_state, state))
        return residual_norm(u, residual, scale=0.5) + (states,)

    def reference(self, u, residual):
        """The same of whole prompts in 64 bits, every tensor between two operators
        rounded to its type."""
        def rounded(t):
            return t.to(self.dtype).double()

        for p in self.host:
            y, residual, _, _ = ru.residual(u, residual, p["norm"], None, p["gate"], 0.5, 1e-5)
            residual = residual.float()
            w_in, w_out = ru.quantize(p["w_in"]), ru.quantize(p["w_out"])
            h = rounded(ru.product(*ru.quantize(y.float()), *w_in, None)[0])
            z, xbc, dt = h.split((INNER, INNER + 2 * BC, HEADS), -1)
            out = []
            for i in range(u.shape[0]):
                state = torch.zeros(WIDTH - 1, INNER + 2 * BC)
                c = rounded(ssm_util.conv(xbc[i], p["conv"], None, True, state)[0])
                x, B, C = c.split((INNER, BC, BC), -1)
                s = ssm_util.scan(x.unflatten(-1, (HEADS, P)), dt[i], p["A"], B.unflatten(-1, (GROUPS, N)),
                                  C.unflatten(-1, (GROUPS, N)), p["D"], None, p["dt_bias"], True,
                                  torch.zeros(HEADS, P, N))[0]
                out.append(rounded(s.flatten(-2)))
            y = ru.gated(torch.stack(out), p["inner_norm"], z, 1e-5, GROUPS, False)[0]
            u = rounded(ru.product(*ru.quantize(y.float()), *w_out, None)[0])
        return ru.residual(u, residual, None, None, None, 0.5, 1e-5)[:2]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
def test_block_runs_as_defined(dtype):
    """What differs: roundings of the type between the operators, and values next to
    a half that go to the other of two whole numbers, a 1/254 of the row's largest
    value each.  Two of 96 or 128 terms of a product gone the other way, through
    two blocks, stay below 2 % of the largest output; a wrong index does not."""
    block = Block(dtype)
    g = torch.Generator().manual_seed(1)
    u = torch.randn(2, 37, MODEL, generator=g).to(dtype)
    residual = torch.randn(2, 37, MODEL, generator=g)
    with torch.no_grad():
        y, r, _ = block(u.cuda(), residual.cuda(), block.caches(2), False)
    want_y, want_r = block.reference(u, residual)
    for got, want in ((y, want_y), (r, want_r)):
        assert float((got.cpu().double() - want).abs().max() / want.abs().max()) < 0.02


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_tokens_continue_prompts_in_a_graph(dtype):
    """A captured step of both blocks, replayed with eager work between, answers what
    the eager step answers, bit for bit."""
    from pto_einsum import StageGraph

    block = Block(dtype)
    g = torch.Generator().manual_seed(2)
    tokens = [(torch.randn(3, MODEL, generator=g).to(dtype).cuda(), torch.randn(3, MODEL, generator=g).cuda())
              for _ in range(4)]
    with torch.no_grad():
        eager_caches = block.caches(3)
        eager = [block(u, r, eager_caches, True)[:2] for u, r in tokens]
        caches = block.caches(3)
        u, r = (t.clone() for t in tokens[0])
        graph = StageGraph(lambda: block(u, r, caches, True)[:2])
        for pair, new in zip(caches, block.caches(3)):
            for old, zero in zip(pair, new):
                old.copy_(zero)
        for (a, b), want in zip(tokens, eager):
            u.copy_(a), r.copy_(b)
            got = graph.replay()
            torch.randn(1000, device="cuda").sum()
            block(a, b, block.caches(3), True)
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for old, new in zip(eager_caches, caches):
            assert torch.equal(old[0], new[0]) and torch.equal(old[1], new[1])


def test_streams_and_threads():
    """The same calls on several streams and threads at once."""
    import threading

    from pto_einsum import matmul_q8, quantize_q8, residual_norm

    g = torch.Generator().manual_seed(4)
    x = [torch.randn(200, 1500, generator=g).cuda().half() for _ in range(4)]
    w, ws = quantize_q8(torch.randn(700, 1500, generator=g).cuda())
    want = [(matmul_q8(t, w, ws), *residual_norm(t, t)) for t in x]
    torch.cuda.synchronize()
    bad = []

    def work(t, ref):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = (matmul_q8(t, w, ws), *residual_norm(t, t))
                s.synchronize()
                bad.extend(i for i, (a, b) in enumerate(zip(got, ref)) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=a) for a in zip(x, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_graphs_share_nothing():
    """Two captured products of float rows, replayed in turn: each has its own workspace."""
    from pto_einsum import StageGraph, matmul_q8, quantize_q8

    g = torch.Generator().manual_seed(5)
    w, ws = quantize_q8(torch.randn(300, 1024, generator=g).cuda())
    x = [torch.randn(m, 1024, generator=g).cuda() for m in (3, 150)]
    graphs = [StageGraph(lambda t=t: matmul_q8(t, w, ws)) for t in x]
    for _ in range(3):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g))
        got = [graph.replay() for graph in graphs]
        torch.cuda.synchronize()
        for t, y in zip(x, got):
            assert torch.equal(y, matmul_q8(t, w, ws))
