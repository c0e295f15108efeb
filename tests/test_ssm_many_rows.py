"""Prompts of so many sequences and heads that a launch of chunks would not hold
them run token by token: no workspace, no refusal."""
import pytest
import torch

import ssm_util as u
from test_ssm_plan import _bytes


def test_what_passes_a_launch_needs_no_workspace():
    # 64 x 128 a head: 8 blocks of 256 threads carry its states
    assert _bytes(packed=1, nseq=16384, T=300000, H=128) == 0
    assert _bytes(packed=1, nseq=16383, T=300000, H=128) > 0
    assert _bytes(packed=1, nseq=131080, T=131100, H=128, P=8, N=8) == 0
    assert _bytes(packed=1, nseq=100000, T=131100, H=128, P=8, N=8) > 0


@pytest.mark.gpu
def test_many_sequences():
    """131080 sequences, most of one token, of 128 heads of 8 x 8."""
    from pto_einsum import selective_scan

    nseq, H, P, N = 131080, 128, 8, 8
    lens = torch.ones(nseq, dtype=torch.int64)
    lens[0], lens[70000], lens[nseq - 2], lens[nseq - 1] = 20, 0, 7, 3
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    T = int(cu[-1])
    g = torch.Generator(device="cuda").manual_seed(0)
    x, B, C = (torch.randn(T, h, n, generator=g, device="cuda").half() for h, n in ((H, P), (1, N), (1, N)))
    dt, A = torch.rand(T, H, generator=g, device="cuda") * 0.1, -torch.rand(H, generator=g, device="cuda") * 8
    print(f"selective_scan {nseq} sequences", flush=True)
    y, st = selective_scan(x, dt, A, B, C, cu_seqlens=cu.to(torch.int32).cuda())
    for i in (0, 1, 69999, 70000, 70001, nseq - 2, nseq - 1):
        cut = slice(int(cu[i]), int(cu[i + 1]))
        ry, rs, ya, sa = u.scan(x[cut].cpu(), dt[cut].cpu(), A.cpu(), B[cut].cpu(), C[cut].cpu(), None, None, None, False,
                                torch.zeros(H, P, N))
        rel = u.scan_bound(int(lens[i]), N, 0, 0)
        assert bool(((y[cut].double().cpu() - ry).abs() <= u.HALF[torch.float16] * ry.abs() + rel * ya + 2.0 ** -25).all())
        assert bool(((st[i].double().cpu() - rs).abs() <= rel * sa + 1e-37).all())
    assert bool(torch.isfinite(st).all()) and bool((st[70000] == 0).all())
