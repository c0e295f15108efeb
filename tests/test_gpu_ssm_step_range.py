"""The scan's recurrence (single tokens and short prompts) on infinite and NaN
operands, for states whose rows end inside a lane's or a wave's share."""
import pytest
import torch

import ssm_util as u
from test_gpu_ssm import _call, _cuda, _scan_case

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
PLACES = [("x", 3, INF), ("x", 3, -INF), ("x", 3, NAN), ("B", 1, INF), ("C", 2, -INF), ("st", 5, INF), ("dt", 0, INF)]


def same(got, ref, bound, what):
    """NaN where the definition has NaN, its infinities, the rest within bounds."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(torch.where(torch.isinf(got), got, 0.0), torch.where(torch.isinf(ref), ref, 0.0)), what
    ok = torch.isfinite(ref)
    assert bool(((got - ref)[ok].abs() <= bound[ok]).all()), what


def _case(dtype, T, P, N, name, at, value):
    """Signs alike, so that infinite states give infinite outputs."""
    c = _scan_case(dtype, [T], 2, P, 1, N, seed=N + T)
    c["B"], c["C"] = c["B"].abs(), c["C"].abs()
    index = {"x": (T // 2, 1, at), "B": (T // 2, 0, at), "C": (T // 2, 0, at), "dt": (T // 2, 1),
             "st": (0, 1, 2, at)}[name]
    c[name][index] = value
    return c


def _ref(c, n, cut=slice(None)):
    ry, rs, ya, sa = u.scan(c["x"][cut], c["dt"][cut], c["A"], c["B"][cut], c["C"][cut], c["D"], c["z"][cut], c["dt_bias"],
                            True, c["st"][0])
    rel = u.scan_bound(n, c["B"].shape[-1], 0, 0)
    dtype = c["x"].dtype
    return (ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype]), (rs, rel * sa + 1e-37)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("N", [6, 16, 24, 63, 100, 130, 256])
@pytest.mark.parametrize("name,at,value", PLACES)
def test_short_prompts(dtype, N, name, at, value):
    c = _case(dtype, 12, 20, N, name, at, value)
    print(f"selective_scan {dtype} N {N} {name} {value}", flush=True)
    y, state = _call(c, dense=1)
    for got, (ref, bound), what in zip((y[0], state[0]), _ref(c, 12), ("y", "state")):
        same(got, ref, bound, what)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("N", [6, 24, 63, 130])
@pytest.mark.parametrize("name,at,value", PLACES)
def test_tokens(dtype, N, name, at, value):
    from pto_einsum import selective_scan_step

    c = _case(dtype, 1, 20, N, name, at, value)
    t = {k: _cuda(v) for k, v in c.items()}
    state = t["st"].clone()
    y = selective_scan_step(t["x"], t["dt"], t["A"], t["B"], t["C"], state, D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                            dt_softplus=True)
    for got, (ref, bound), what in zip((y, state[0]), _ref(c, 1), ("y", "state")):
        same(got, ref, bound, what)


@pytest.mark.parametrize("N", [24, 63])
def test_growth_past_float32(N):
    """A rate above 0 and a long step: an infinite growth of the state is its own,
    not that of lanes past N."""
    c = _case(torch.float32, 12, 20, N, "x", 3, 1.0)
    c["A"], c["z"] = -c["A"], torch.ones_like(c["z"])
    c["dt"][6] = 1000.0
    y, state = _call(c, dense=1)
    grown = torch.isinf(state[0].cpu())
    assert bool(grown.all()) and not bool(torch.isnan(state).any())
    assert bool(torch.isfinite(y[0, :6]).all())
