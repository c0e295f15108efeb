"""Pieces longer than the 256 step sizes that a block of the chunked scan prepares
at a time: a prompt with enough sequences and heads is not cut, or into few
pieces.  That the pieces are so long is read off the workspace's size."""
import pytest
import torch

import ssm_util as u
from pto_einsum.ssm import DTYPES
from test_gpu_ssm import _cu, _within
from test_ssm_plan import _bytes

pytestmark = pytest.mark.gpu


def _pieces(size, H, P, N):
    """The pieces in a workspace of that size."""
    tiles = -(-P // 64)
    nt = 32 if N <= 32 else 64 if N <= 64 else 128 if N <= 128 else 256
    waves = max(3 if nt == 256 else 2, -(-(-(-P // 16)) // tiles))
    each = H * (1 + tiles * waves * nt // 16 * 256)
    assert H % 4 == 0 and size % (4 * each) == 0
    return size // (4 * each)


def _operands(dtype, dt_dtype, lead, H, P, G, N, nseq, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    return dict(x=normal(*lead, H, P).to(dtype), B=normal(*lead, G, N).to(dtype), C=normal(*lead, G, N).to(dtype),
                z=normal(*lead, H, P).to(dtype), dt=normal(*lead, H).to(dt_dtype),
                A=-(1 + 15 * torch.rand(H, generator=g, device="cuda")), D=torch.rand(H, generator=g, device="cuda"),
                dt_bias=torch.linspace(-6.9, -2.2, H, device="cuda"), st=normal(nseq, H, P, N))


def _check(y, state, t, seq, cut, heads, dtype):
    """Some heads of one sequence: t's tensors from the token axis on."""
    H = t["x"].shape[-2]
    G = t["B"].shape[-2]
    groups = [h // (H // G) for h in heads]
    x, dt, z = (t[k][cut][:, heads].cpu() for k in ("x", "dt", "z"))
    B, C = (t[k][cut][:, groups].cpu() for k in ("B", "C"))
    n, N = x.shape[0], B.shape[-1]
    ry, rs, ya, sa = u.scan(x, dt, t["A"][heads].cpu(), B, C, t["D"][heads].cpu(), z, t["dt_bias"][heads].cpu(), True,
                            t["st"][seq, heads].cpu())
    rel = u.scan_bound(n, N, 0, 0)
    _within(y[cut][:, heads], ry, u.HALF[dtype] * ry.abs() + rel * ya + u.TINY[dtype], f"y of sequence {seq} ({n})")
    _within(state[seq, heads], rs, rel * sa + 1e-37, f"state of sequence {seq} ({n})")
    if n >= 16:
        # roundings of random sign, as in the tests of short pieces
        far = float((state[seq, heads].cpu().double() - rs).norm() / rs.norm())
        assert far <= 2.0 ** -24 * 8 * n ** 0.5, f"state of sequence {seq}: {far:.3g}"
        far = float((y[cut][:, heads].cpu().double() - ry).norm() / ry.norm())
        assert far <= 1.2 * u.HALF[dtype] + 2.0 ** -24 * 16 * n ** 0.5, f"y of sequence {seq}: {far:.3g}"


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("dt32", [False, True], ids=["dt", "dt32"])
@pytest.mark.parametrize("T", [257, 561])
@pytest.mark.parametrize("P,N,G", [(16, 16, 1), (48, 30, 4), (64, 16, 64), (64, 100, 2)],
                         ids=["two", "three", "four", "wide"])
def test_dense(dtype, dt32, T, P, N, G):
    """One piece a sequence, two to four waves a block."""
    from pto_einsum import selective_scan

    nseq, H = 24, 64
    dt_dtype = torch.float32 if dt32 else dtype
    assert _bytes(nseq=nseq, T=T, H=H, P=P, N=N, G=G, dtype=DTYPES[dtype], dt_dtype=DTYPES[dt_dtype]) == 0
    t = _operands(dtype, dt_dtype, (nseq, T), H, P, G, N, nseq, seed=T + P)
    print(f"selective_scan {dtype} {nseq} x {T} P {P} N {N} G {G}", flush=True)
    y, state = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                              dt_softplus=True, initial_state=t["st"])
    for seq in (0, nseq - 1):
        one = {k: (v[seq] if k in ("x", "B", "C", "z", "dt") else v) for k, v in t.items()}
        _check(y[seq], state, one, seq, slice(None), [0, 33, H - 1], dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("dt32", [False, True], ids=["dt", "dt32"])
@pytest.mark.parametrize("P,H", [(16, 768), (48, 512), (64, 384)], ids=["two", "three", "four"])
@pytest.mark.parametrize("lens", [[5, 0, 1300, 615], [1921], [257, 255, 600, 801]], ids=["mixed", "one", "even"])
def test_packed(dtype, dt32, P, H, lens):
    """Pieces of over 512 tokens, their contributions and their outputs."""
    from pto_einsum import selective_scan

    T, N, G = sum(lens), 16, 1
    if dtype is torch.float32:
        H = {768: 512, 512: 256, 384: 256}[H]
    dt_dtype = torch.float32 if dt32 else dtype
    size = _bytes(packed=1, nseq=len(lens), T=T, H=H, P=P, N=N, G=G, dtype=DTYPES[dtype], dt_dtype=DTYPES[dt_dtype])
    per = _pieces(size, H, P, N) - len(lens)
    assert per >= 1 and T / per > 512
    t = _operands(dtype, dt_dtype, (T,), H, P, G, N, len(lens), seed=T + P)
    print(f"selective_scan {dtype} lens {lens} P {P} H {H}, {per} stretches", flush=True)
    y, state = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                              dt_softplus=True, initial_state=t["st"], cu_seqlens=_cu(lens))
    at = 0
    for seq, n in enumerate(lens):
        _check(y, state, t, seq, slice(at, at + n), [0, H // 2, H - 1], dtype)
        at += n
