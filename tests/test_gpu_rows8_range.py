"""Tensors whose offsets pass 32 bits."""
import pytest
import torch

import rows_util as ru

pytestmark = pytest.mark.gpu


def test_products_past_32_bits():
    """y of 2.4e9 elements, by the tiles; 5.1e9 with one row for each of many weights,
    by the kernel for few rows."""
    from pto_einsum import matmul_q8

    g = torch.Generator(device="cuda").manual_seed(1)

    def whole(*shape):
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)

    for m, n, k in ((40_000, 60_000, 64), (64, 80_000_000, 16)):
        q, w = whole(m, k), whole(n, k)
        s, ws = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        y = matmul_q8(q, w, ws, scales=s, dtype=torch.float16 if n < 1 << 20 else torch.bfloat16)
        rows = torch.tensor([0, m // 2, m - 2, m - 1], device="cuda")
        cols = torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
        ref, size = ru.product(q[rows].cpu(), s[rows].cpu(), w[cols].cpu(), ws[cols].cpu(), None)
        ru.assert_within(y[rows][:, cols] * 1, ref, ru.product_bound(ref, size, y.dtype))
        del y, q, w
        torch.cuda.empty_cache()


def test_weights_past_32_bits():
    """5.2e9 bytes of weights: their last rows."""
    from pto_einsum import matmul_q8

    n, k = 80_000, 65_536
    w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    w[-3:] = torch.randint(-127, 128, (3, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(n, generator=g, device="cuda")
    for m in (2, 200):
        q = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        s = torch.rand(m, generator=g, device="cuda")
        y = matmul_q8(q, w, ws, scales=s)
        ref, size = ru.product(q.cpu(), s.cpu(), w[-3:].cpu(), ws[-3:].cpu(), None)
        ru.assert_within(y[:, -3:], ref, ru.product_bound(ref, size, torch.float32))
        assert not y[:, :-3].any()


@pytest.mark.parametrize("rows,d", [(300_000, 16_384), (60_000, 80_000)])
def test_rows_past_32_bits(rows, d):
    """4.8e9 elements and more: the last rows of a norm, of rows in 8 bits and of the
    residual, in registers and read again."""
    from pto_einsum import gated_norm, quantize_q8, residual_norm

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, d, generator=g, device="cuda").bfloat16()
    last = x[-2:].cpu()
    ref, units = ru.gated(last, None, None, 1e-5, 1, False)
    y = gated_norm(x)
    ru.assert_within(y[-2:], ref, ru.gated_bound(ref, units, torch.bfloat16))
    assert not y[:-2].any()
    del y
    q, s = quantize_q8(x)
    want, scale = ru.quantize(last)
    assert torch.equal(q[-2:].cpu().double(), want) and torch.equal(s[-2:].cpu(), scale.float())
    assert not s[:-2].any()
    del q, s
    y, r = residual_norm(x, x)
    y_ref, r_ref, y_err, r_err = ru.residual(last, last, None, None, None, 1.0, 1e-5)
    ru.assert_within(y[-2:], y_ref, ru.bound(y_ref, y_err, torch.bfloat16))
    ru.assert_within(r[-2:], r_ref, ru.bound(r_ref, r_err, torch.bfloat16))
    del x, y, r
    torch.cuda.empty_cache()
