"""residual_norm's y is formed from the sum before it is rounded to the residual's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 700, 3000, 20000])
@pytest.mark.parametrize("dtype,res,x", [(torch.bfloat16, 256.0, 0.25), (torch.float16, 2048.0, 0.25)], ids=["bf16", "f16"])
def test_rows_of_a_swallowed_sum(dtype, res, x, d):
    """Residuals of plus and minus 2^k and x less than half a step: r is the residual.
    The sums' sizes are 2^k + x and 2^k - x, so the row's largest y is
    (2^k + x) / sqrt(4^k + x^2) and its scale 1 / 127 of that; from the rounded r it
    would be 1 / 127.  (x / 2^k is 2^-10 or 2^-13, and 2^-20 of float32 is far less.)"""
    from pto_einsum import residual_norm

    r0 = torch.full((1, d), res, dtype=dtype)
    r0[0, ::2] = -res
    (q, s), r = residual_norm(torch.full((1, d), x, dtype=dtype).cuda(), r0.cuda(), eps=0.0, quantize=True)
    assert torch.equal(r.cpu(), r0)
    want = (res + x) / (res * res + x * x) ** 0.5 / 127
    assert abs(float(s) - want) <= 2.0 ** -20 * want
    assert want > (1 + 2.0 ** -14) / 127
    # the sizes' quotient is 1 - 2 x / 2^k: both round to 127
    assert torch.equal(q.cpu().abs(), torch.full((1, d), 127, dtype=torch.int8))
