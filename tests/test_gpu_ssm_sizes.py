"""Kernels that are chosen at the sizes of real calls: 4-bit products with several
weight tiles a wave, token steps whose states pass the caches, convolutions with
long runs of tokens."""
import pytest
import torch

import ssm_util as u
from pto_einsum.ssm import DTYPES
from test_gpu_ssm import _check_conv, _cu, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,zeros", [(1, 8203, True), (16, 16411, False), (20, 8203, True)],
                         ids=["two", "four", "two_by_two"])
@pytest.mark.parametrize("K", [97, 4635])
def test_q4_weight_tiles(dtype, group, M, N, zeros, K):
    """Two and four tiles of 16 weight rows for each of x (256 blocks are left
    then), under one step and over what is loaded ahead, with odd ends."""
    from pto_einsum import matvec_q4

    g = torch.Generator(device="cuda").manual_seed(K + M)
    ng = -(-K // group)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    packed = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(N, ng, generator=g, device="cuda") * 0.02 + 0.01).to(dtype)
    z = (torch.rand(N, ng, generator=g, device="cuda") * 15).to(dtype) if zeros else None
    print(f"matvec_q4 {dtype} M {M} N {N} K {K} group {group}", flush=True)
    y = matvec_q4(x, packed, scales, z, group=group)
    # every place in a tile, and the rows at both ends
    rows = torch.cat([torch.arange(0, 70), torch.arange(70, N - 70, 37), torch.arange(N - 70, N)]).cuda()
    ref, size = u.q4(x.cpu(), packed[rows].cpu(), scales[rows].cpu(), None if z is None else z[rows].cpu(), group, K)
    err = (y[:, rows].double().cpu() - ref).abs()
    assert bool((err <= u.q4_bound(ref, size, K, dtype)).all())
    far = float((y[:, rows].double().cpu() - ref).norm() / ref.norm())
    assert far <= 1.2 * u.HALF[dtype] + 2.0 ** -24 * 8 * max(1.0, K ** 0.5 / 4), far


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("P,N,H", [(64, 128, 16), (80, 100, 17), (33, 256, 16), (64, 16, 130)])
def test_step_of_many_states(dtype, P, N, H):
    """States of 32 MB and more pass the caches by; slots in any order, the others
    stay."""
    from pto_einsum import selective_scan_step

    n, S, G = 64, 70, 1
    assert 4 * n * H * P * N >= 32 << 20
    g = torch.Generator(device="cuda").manual_seed(P)
    x, z = (torch.randn(n, H, P, generator=g, device="cuda").to(dtype) for _ in range(2))
    B, C = (torch.randn(n, G, N, generator=g, device="cuda").to(dtype) for _ in range(2))
    dt = torch.randn(n, H, generator=g, device="cuda").to(dtype)
    A, D = -(1 + 15 * torch.rand(H, generator=g, device="cuda")), torch.rand(H, generator=g, device="cuda")
    bias = torch.linspace(-6.9, -2.2, H, device="cuda")
    state = torch.randn(S, H, P, N, generator=g, device="cuda")
    before = state.clone()
    slots = torch.randperm(S, generator=g, device="cuda")[:n].to(torch.int32)
    slots[5], slots[40] = -1, S
    print(f"selective_scan_step {dtype} {n} x {H} x {P} x {N}", flush=True)
    y = selective_scan_step(x, dt, A, B, C, state, D=D, z=z, dt_bias=bias, dt_softplus=True, slots=slots)
    rel = u.scan_bound(1, N, 0, 0)
    used = set()
    for row, slot in enumerate(slots.tolist()):
        if not 0 <= slot < S:
            assert bool((y[row] == 0).all())
            continue
        used.add(slot)
        cut = slice(row, row + 1)
        ry, rs, ya, sa = u.scan(x[cut].cpu(), dt[cut].cpu(), A.cpu(), B[cut].cpu(), C[cut].cpu(), D.cpu(), z[cut].cpu(),
                                bias.cpu(), True, before[slot].cpu())
        _within(y[cut], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], f"y of row {row}")
        _within(state[slot], rs, rel * sa + 1e-37, f"state of row {row}")
    rest = [s for s in range(S) if s not in used]
    assert len(rest) >= 8 and torch.equal(state[rest], before[rest])


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("packed", [False, True], ids=["dense", "packed"])
@pytest.mark.parametrize("run", [16, 32])
@pytest.mark.parametrize("W", [3, 4])
def test_conv_runs(dtype, packed, run, W):
    """Runs of 16 and 32 tokens a thread (2^18 threads take them), lengths that are
    no whole runs."""
    from pto_einsum import causal_conv

    V = 4 if dtype is torch.float32 else 8
    D = 2051
    lens = [8611, 1, 0, 4099, 45] if packed else [4305] * 3
    if run == 32:
        lens = [2 * n + 1 for n in lens]
    if V == 8:
        lens = [2 * n + 1 for n in lens]
    T = sum(lens)
    threads = [-(-n // run) for n in ([T] if packed else lens)]
    vecs = -(-D // V)
    assert sum(threads) * vecs >= 1 << 18 and (run == 32 or sum(-(-n // 32) for n in ([T] if packed else lens)) * vecs < 1 << 18)
    g = torch.Generator(device="cuda").manual_seed(run + W)
    x = torch.randn(T, D, generator=g, device="cuda").to(dtype)
    w = torch.randn(D, W, generator=g, device="cuda").to(dtype)
    b = torch.randn(D, generator=g, device="cuda").to(dtype)
    st = torch.randn(len(lens), W - 1, D, generator=g, device="cuda").to(dtype)
    print(f"causal_conv {dtype} lens {lens} D {D} W {W}", flush=True)
    if packed:
        y, state = causal_conv(x, w, b, activation="silu", initial_state=st, cu_seqlens=_cu(lens))
    else:
        y, state = causal_conv(x.unflatten(0, (len(lens), -1)), w, b, activation="silu", initial_state=st)
        y = y.flatten(0, 1)
    some = torch.tensor([0, 1, 7, 8, 1000, 1023, D - 9, D - 8, D - 2, D - 1]).cuda()
    _check_conv(y[:, some], state[:, :, some], x[:, some].cpu(), w[some].cpu(), b[some].cpu(), True, st[:, :, some].cpu(),
                lens, dtype)
