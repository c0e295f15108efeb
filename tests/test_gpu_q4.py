"""Products with 4-bit weights on the GPU against 64 bits."""
import pytest
import torch

import ssm_util as u

pytestmark = pytest.mark.gpu


def _case(dtype, M, N, K, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    ng = -(-K // group)
    return (torch.randn(M, K, generator=g).to(dtype),
            torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8),
            (torch.rand(N, ng, generator=g) * 0.02 + 0.01).to(dtype),
            (torch.rand(N, ng, generator=g) * 15).to(dtype) if zeros else None)


def _run(x, packed, scales, zeros, group):
    from pto_einsum import matvec_q4

    return matvec_q4(x.cuda(), packed.cuda(), scales.cuda(), None if zeros is None else zeros.cuda(), group=group)


def _check(y, x, packed, scales, zeros, group, dtype):
    K = x.shape[-1]
    ref, size = u.q4(x, packed, scales, zeros, group, K)
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= u.q4_bound(ref, size, K, dtype)).all())
    if ref.numel() > 64:
        # Sums of roundings of random sign: sqrt(K) of them rather than K.
        far = float((y.double().cpu() - ref).norm() / ref.norm())
        assert far <= 1.2 * u.HALF[dtype] + 2.0 ** -24 * 8 * max(1.0, K ** 0.5 / 4), far


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
@pytest.mark.parametrize("M,N,K,group", [
    (1, 256, 1024, 128), (1, 1, 1, 32), (3, 17, 33, 32), (16, 100, 500, 64), (5, 48, 1000, 32), (17, 33, 129, 128),
    (40, 70, 255, 64), (65, 16, 256, 128), (130, 20, 300, 32), (2, 5000, 96, 64), (1, 40, 9001, 128)])
def test_shapes(dtype, zeros, M, N, K, group):
    case = _case(dtype, M, N, K, group, zeros, seed=K)
    print(f"matvec_q4 {dtype} M {M} N {N} K {K} group {group}", flush=True)
    _check(_run(*case, group), *case, group, dtype)


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
def test_every_weight_value_and_position(dtype):
    """x with one 1 picks out each weight exactly."""
    K, N = 64, 16
    packed = torch.arange(N * K // 2, dtype=torch.int64).mul(37).remainder(256).to(torch.uint8).reshape(N, K // 2)
    scales = torch.ones(N, 2).to(dtype)
    y = _run(torch.eye(K).to(dtype), packed, scales, None, 32).float().cpu()
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(1).float()
    assert torch.equal(y, (q - 8).t())


def test_axes_strides_and_alignment():
    from pto_einsum import matvec_q4

    x, packed, scales, zeros = _case(torch.float16, 6, 40, 101, 32, True)
    wide = torch.zeros(2, 3, 105).half().cuda()
    wide[..., 3:104] = x.cuda().reshape(2, 3, 101)
    y = matvec_q4(wide[..., 3:104], packed.cuda(), scales.cuda(), zeros.cuda(), group=32)
    assert y.shape == (2, 3, 40)
    _check(y.reshape(6, 40), x, packed, scales, zeros, 32, torch.float16)
    one = matvec_q4(wide[0, 1, 3:104], packed.cuda(), scales.cuda(), zeros.cuda(), group=32)
    assert torch.equal(one, y[0, 1])
    # weights that start at an odd byte
    buf = torch.zeros(packed.numel() + 1, dtype=torch.uint8).cuda()
    buf[1:] = packed.cuda().flatten()
    assert torch.equal(matvec_q4(wide[..., 3:104], buf[1:].view(40, 51), scales.cuda(), zeros.cuda(), group=32), y)


def test_empty_and_non_finite_rows():
    from pto_einsum import matvec_q4

    x, packed, scales, _ = _case(torch.bfloat16, 3, 20, 96, 32, False)
    s = scales.cuda()
    assert matvec_q4(x.cuda()[:0], packed.cuda(), s, group=32).shape == (0, 20)
    assert matvec_q4(x.cuda(), packed.cuda()[:0], s[:0], group=32).shape == (3, 0)
    none = matvec_q4(x.cuda()[:, :0], packed.cuda()[:, :0], s[:, :0], group=32)
    assert none.shape == (3, 20) and bool((none == 0).all())
    x[1, 5] = float("nan")
    y = matvec_q4(x.cuda(), packed.cuda(), s, group=32)
    assert bool(torch.isnan(y[1]).all())
    _check(y[[0, 2]], x[[0, 2]], packed, scales, None, 32, torch.bfloat16)


def test_captured():
    from pto_einsum import StageGraph, matvec_q4

    x, packed, scales, zeros = (None if v is None else v.cuda() for v in _case(torch.float16, 4, 200, 700, 64, True))
    graph = StageGraph(lambda: matvec_q4(x, packed, scales, zeros, group=64))
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).half())
        got = graph.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, matvec_q4(x, packed, scales, zeros, group=64))
