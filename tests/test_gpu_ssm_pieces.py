"""Selective scan where a prompt is cut into tiles and pieces: rows P past one
tile, tiles of fewer than eight rows, many pieces, packed sequences that end at
and around the pieces' ends, and what is left to the token-by-token kernel."""
import pytest
import torch

import ssm_util as u
from test_gpu_ssm import _call, _check_scan, _cu, _cuda, _scan_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("P,N", [(48, 8), (65, 16), (130, 24), (193, 40), (8, 65), (100, 129)])
def test_tiles_of_rows(dtype, P, N):
    """Two to four waves a block, one to four tiles, the last of one row."""
    lens = [70, 33]
    c = _scan_case(dtype, lens, 2, P, 1, N, seed=P + N)
    print(f"selective_scan {dtype} P {P} N {N}", flush=True)
    y, state = _call(c, lens)
    _check_scan(y, state, c, lens, dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("lens", [[64, 64, 128], [1, 63, 65, 127, 129], [32, 0, 96, 0, 0, 31, 1, 300], [513], [17]])
def test_ends_of_pieces(dtype, lens):
    c = _scan_case(dtype, lens, 2, 32, 1, 32, seed=len(lens))
    print(f"selective_scan {dtype} lens {lens}", flush=True)
    y, state = _call(c, lens)
    _check_scan(y, state, c, lens, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_many_pieces(dtype):
    """One head of one sequence: as many pieces as a sequence is cut into."""
    lens = [6500]
    c = _scan_case(dtype, lens, 1, 16, 1, 16, seed=3, rate=(0.01, 0.1))
    y, state = _call(c, dense=1)
    _check_scan(y[0], state, c, lens, dtype)


def test_offsets_out_of_order_stay_inside():
    """Offsets that fall, or lie outside the buffer, are clamped: the outputs mean
    nothing then, but nothing outside the buffers is touched."""
    from pto_einsum import causal_conv, selective_scan

    c = _scan_case(torch.float16, [200], 2, 32, 1, 64, seed=4)
    t = {k: _cuda(v) for k, v in c.items()}
    for cu in ([0, 150, 20, 200], [-5, 90, 1 << 30, 7], [200, 200, 0, 0]):
        cu = torch.tensor(cu, dtype=torch.int32).cuda()
        first = t["st"].repeat(3, 1, 1, 1)
        y, st = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], dt_bias=t["dt_bias"], dt_softplus=True,
                               initial_state=first, cu_seqlens=cu)
        z, cs = causal_conv(t["x"].flatten(1), torch.ones(64, 4).half().cuda(), cu_seqlens=cu)
        torch.cuda.synchronize()
        assert y.shape == c["x"].shape and st.shape == first.shape and z.shape == (200, 64) and cs.shape == (3, 3, 64)
    again, st2 = _call(c, dense=1)
    _check_scan(again[0], st2, c, [200], torch.float16)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
def test_strides_past_a_chunk_s_offsets(dtype):
    """A token stride of 2^24 elements: token by token, the same results."""
    from pto_einsum import selective_scan

    T, H, P, N = 18, 1, 8, 8
    c = _scan_case(dtype, [T], H, P, 1, N, seed=6, gate=False)
    wide = torch.zeros(1 + (T - 1) * (1 << 24) + H * P, dtype=dtype, device="cuda")
    x = wide[1:].as_strided((1, T, H, P), (0, 1 << 24, P, 1))
    x.copy_(c["x"][None])
    t = {k: _cuda(v) for k, v in c.items()}
    y, st = selective_scan(x, t["dt"][None], t["A"], t["B"][None], t["C"][None], D=t["D"], dt_bias=t["dt_bias"],
                           dt_softplus=True, initial_state=t["st"])
    _check_scan(y[0], st, c, [T], dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
def test_not_a_number_in_steps_and_gates(dtype):
    """A NaN step size reaches its own and later tokens of its head; a NaN gate its
    own output."""
    lens, H, P, N = [100, 60], 2, 40, 32
    c = _scan_case(dtype, lens, H, P, 1, N, seed=7)
    clean, cstate = _call(c, lens)
    dt, z = c["dt"].clone(), c["z"].clone()
    dt[70, 1] = float("nan")
    z[20, 0, 5] = float("nan")
    y, state = _call({**c, "dt": dt, "z": z}, lens)
    bad = torch.zeros(160, H, P, dtype=torch.bool)
    bad[70:100, 1] = True
    bad[20, 0, 5] = True
    assert torch.equal(torch.isnan(y.cpu()), bad)
    assert bool(torch.isnan(state[0, 1]).all()) and bool(torch.isfinite(state[1]).all())
    _check_scan(torch.where(bad, clean.cpu(), y.cpu()), cstate, c, lens, dtype)


def test_layouts_share_plans_not_data():
    """Calls of one layout after another, on other data and on operands that have
    to be laid out first."""
    from pto_einsum import matvec_q4, selective_scan_step

    for seed in (1, 2):
        c = _scan_case(torch.float16, [3], 2, 16, 1, 16, seed=seed)
        t = {k: _cuda(v) for k, v in c.items()}
        s1, s2 = t["st"].repeat(3, 1, 1, 1), t["st"].repeat(3, 1, 1, 1)
        odd = t["x"].transpose(1, 2).contiguous().transpose(1, 2)
        more = dict(D=t["D"], z=t["z"], dt_bias=t["dt_bias"], dt_softplus=True)
        a = selective_scan_step(t["x"], t["dt"], t["A"], t["B"], t["C"], s1, **more)
        b = selective_scan_step(odd, t["dt"], t["A"], t["B"], t["C"], s2, **more)
        assert torch.equal(a, b) and torch.equal(s1, s2)
        x = torch.randn(64, 5, generator=torch.Generator().manual_seed(seed)).half().cuda()
        packed = torch.full((3, 32), 0x9A, dtype=torch.uint8).cuda()
        scales = torch.ones(3, 2).half().cuda()
        assert torch.equal(matvec_q4(x.t(), packed, scales, group=32), matvec_q4(x.t().contiguous(), packed, scales, group=32))
