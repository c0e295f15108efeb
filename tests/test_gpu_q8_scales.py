"""Scales near both ends of float32: a row's and a channel's may each take a sum out of
its range where their product does not."""
import ctypes

import pytest
import torch

import rows_util as ru

pytestmark = pytest.mark.gpu

ROWS = [2.0 ** -149, 1e-40, 1e-38, 1e-20, 1.0, 1e28, 2.0 ** 96, 1e30, 1e36, 3e38]
COLS = [2.0 ** -149, 3e-41, 1e-38, 1e-33, 1e-30, 1e-10, 1.0, 1e5, 1e30, 3e38, -1e-31]


def operands(m, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    q[:, -1], w[:, -1] = 127, 127
    s = torch.tensor(ROWS)[torch.arange(m) * 7 % len(ROWS)]
    ws = torch.tensor(COLS)[torch.arange(n) * 5 % len(COLS)]
    w[n // 2] = 0                   # sums of 0
    return q, w, s, ws


def within(y, ref, size, dtype):
    """Where the result itself is within float32: 3e38 and a rounding of bfloat16 are."""
    y = y.cpu().double()
    keep = ref.abs() <= 3e38
    assert keep.any(1).all()
    zero = torch.zeros_like(ref)
    ru.assert_within(torch.where(keep, y, zero), torch.where(keep, ref, zero),
                     ru.product_bound(ref, size, dtype).nan_to_num(posinf=0.0), "y")
    beyond = ref.abs() > 3.5e38
    assert torch.equal(y[beyond], torch.sign(ref[beyond]) * float("inf"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 60, 100), (10, 77, 300), (30, 50, 1000), (60, 300, 64), (300, 520, 1000), (2000, 1500, 192)])
def test_scales(m, n, k, dtype):
    from pto_einsum import matmul_q8

    q, w, s, ws = operands(m, n, k, m)
    for start in range(len(ROWS) if m < len(ROWS) else 1):
        s = torch.roll(s, 1) if m > 1 else torch.tensor([ROWS[start]])
        ref, size = ru.product(q, s, w, ws, None)
        within(matmul_q8(q.cuda(), w.cuda(), ws.cuda(), scales=s.cuda(), dtype=dtype), ref, size, dtype)
    bias = torch.linspace(-1, 1, n) * 1e37
    ref, size = ru.product(q, s, w, ws, bias)
    within(matmul_q8(q.cuda(), w.cuda(), ws.cuda(), scales=s.cuda(), bias=bias.cuda(), dtype=dtype), ref, size, dtype)


@pytest.mark.parametrize("m,k", [(1, 64), (3, 1000), (16, 200), (50, 4096), (400, 700)])
def test_rows_of_large_values(m, k):
    """Float rows up to float32's end, which the call takes to 8 bits itself."""
    from pto_einsum import matmul_q8

    g = torch.Generator().manual_seed(k)
    x = torch.randn(m, k, generator=g)
    x = x / x.abs().amax(-1, keepdim=True) * torch.tensor([3.4e38, 1.0])[torch.arange(m) % 2][:, None]
    w = torch.randint(-127, 128, (70, k), generator=g, dtype=torch.int8)
    ws = torch.rand(70, generator=g) * 1e-6 + 1e-7
    q, s = ru.quantize(x)
    ref, size = ru.product(q, s, w, ws, None)
    within(matmul_q8(x.cuda(), w.cuda(), ws.cuda()), ref, size, torch.float32)


@pytest.mark.parametrize("kernel", range(1, 9))
def test_every_kernel(kernel):
    from pto_einsum import abi, launch

    m, n, k = 70, 140, 192
    q, w, s, ws = (t.cuda() for t in operands(m, n, k, 3))
    ref, size = ru.product(q.cpu(), s.cpu(), w.cpu(), ws.cpu(), None)
    y = torch.empty(m, n, device="cuda")
    d = abi.Q8Desc(launch.DT_I8, launch.DT_F32, launch.DT_F32, kernel, m, n, k, k, k, m * k, n * k)
    assert abi.bind().pe_matmul_q8(ctypes.byref(d), q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), None,
                                   y.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    within(y, ref, size, torch.float32)


def test_scales_that_are_no_numbers():
    """NaN stays in its row or column; an infinite scale makes what it meets infinite or NaN."""
    from pto_einsum import matmul_q8

    for m in (2, 40, 300):
        q, w, s, ws = operands(m, 90, 128, 1)
        s, ws = torch.full((m,), 1e30), torch.full((90,), 1e-30)
        s[1], ws[7] = float("nan"), float("nan")
        s[0] = float("inf")
        y = matmul_q8(q.cuda(), w.cuda(), ws.cuda(), scales=s.cuda()).cpu()
        assert torch.isnan(y[1]).all() and torch.isnan(y[:, 7]).all()
        assert not torch.isfinite(y[0]).any()
        rest = torch.ones(m, 90, dtype=torch.bool)
        rest[:2], rest[:, 7] = False, False
        assert torch.isfinite(y[rest]).all()
