"""Selective scans of infinite, NaN and very large operands: prompts of any length
give what the recurrence gives, element by element."""
import pytest
import torch

import ssm_util as u
from test_gpu_ssm import _call, _scan_case

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _agree(got, ref, size, rel, half, tiny, what):
    """NaN where the definition has NaN, its infinities, and the rest within the
    bounds of finite operands."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(torch.isinf(got), torch.isinf(ref)), what
    assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)]), what
    ok = torch.isfinite(ref)
    assert bool(((got - ref)[ok].abs() <= (half * ref.abs() + rel * size + tiny)[ok]).all()), what


def _check(y, state, c, lens, dtype):
    at, N = 0, c["B"].shape[-1]
    for i, n in enumerate(lens):
        cut = slice(at, at + n)
        ry, rs, ya, sa = u.scan(c["x"][cut], c["dt"][cut], c["A"], c["B"][cut], c["C"][cut], c["D"],
                                None if c["z"] is None else c["z"][cut], c["dt_bias"], True, c["st"][i])
        rel = u.scan_bound(n, N, 0, 0)
        _agree(y[cut], ry, ya, rel, u.HALF[dtype], u.TINY[dtype], f"y of sequence {i} ({n})")
        _agree(state[i], rs, sa, rel, 0.0, 1e-37, f"state of sequence {i} ({n})")
        at += n


# where a value goes: (tensor, index from the token axis on)
PLACES = {
    "x": [("x", (70, 1, 7), INF)],
    "x_minus": [("x", (70, 1, 7), -INF)],
    "x_twice": [("x", (70, 1, 7), INF), ("x", (90, 1, 7), -INF)],
    "x_nan": [("x", (70, 1, 7), NAN)],
    "first": [("x", (0, 0, 0), INF)],
    "B": [("B", (70, 0, 3), INF)],
    "C": [("C", (70, 0, 3), -INF)],
    "C_nan": [("C", (33, 0, 5), NAN)],
    "dt": [("dt", (70, 1), INF)],
    "dt_nan": [("dt", (65, 0), NAN)],
    "state": [("st", (0, 1, 7, 3), INF)],
    "state_minus": [("st", (0, 0, 2, 0), -INF)],
}


def _put(c, place):
    c = {k: (None if v is None else v.clone()) for k, v in c.items()}
    for name, index, value in PLACES[place]:
        c[name][index] = value
    return c


def _signs(c, alike):
    """B and C of one sign: infinite states then give infinite outputs, not NaN."""
    return {**c, "B": c["B"].abs(), "C": c["C"].abs()} if alike else c


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("place", sorted(PLACES))
@pytest.mark.parametrize("alike", [False, True], ids=["mixed", "alike"])
def test_packed(dtype, place, alike):
    """Two sequences of 100 tokens; a head of 40 rows."""
    lens, H, P, N = [100, 100], 3, 40, 32
    c = _put(_signs(_scan_case(dtype, lens, H, P, 1, N, seed=5), alike), place)
    print(f"selective_scan {dtype} {place} packed", flush=True)
    y, state = _call(c, lens)
    _check(y, state, c, lens, dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("place", sorted(PLACES))
@pytest.mark.parametrize("P,G,N,T", [(80, 2, 100, 700), (130, 1, 200, 150), (16, 2, 16, 1300), (64, 1, 128, 333)])
def test_pieces(dtype, place, P, G, N, T):
    """One sequence in pieces: contributions, the states at their starts and
    outputs; decays of a piece that are 0 in float32."""
    c = _put(_signs(_scan_case(dtype, [T], 2, P, G, N, seed=T, step=(1e-2, 2e-1)), True), place)
    print(f"selective_scan {dtype} {place} {T} tokens P {P} N {N}", flush=True)
    y, state = _call(c, dense=1)
    _check(y[0], state, c, [T], dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("T", [15, 16, 17, 33])
@pytest.mark.parametrize("name,index", [("x", (9, 1, 3)), ("B", (9, 0, 3)), ("st", (0, 1, 3, 3)), ("dt", (9, 1))])
def test_any_length(dtype, T, name, index):
    """What up to 16 tokens give by the recurrence, 17 give by chunks."""
    c = _signs(_scan_case(dtype, [T], 2, 24, 1, 24, seed=T), True)
    c[name][index] = INF
    y, state = _call(c, dense=1)
    _check(y[0], state, c, [T], dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("ex,eb,ec", [(-60, 70, 70), (-100, 100, 0), (70, -60, 0), (100, -110, -60), (0, 57, 60)])
@pytest.mark.parametrize("T", [16, 70, 400])
def test_magnitudes_of_float32(dtype, ex, eb, ec, T):
    """Operands whose products pass float32's range while the outputs do not."""
    c = _scan_case(dtype, [T], 2, 32, 1, 32, seed=2, gate=False)
    for k, e in (("x", ex), ("B", eb), ("C", ec)):
        c[k] = (c[k].double() * 2.0 ** e).to(dtype)
    c["st"] = (c["st"].double() * 2.0 ** (ex + eb)).float()
    y, state = _call(c, dense=1)
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(state).all())
    _check(y[0], state, c, [T], dtype)
