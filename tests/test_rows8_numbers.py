"""Numbers that float32 does not hold are refused, not taken for infinity or zero."""
import pytest
import torch

from pto_einsum import gated_norm, residual_norm

x = torch.zeros(2, 8)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1e39, -4e38, 1e-60, -1e-50])
def test_scale(scale):
    with pytest.raises(ValueError, match="scale"):
        residual_norm(x, x, scale=scale)


@pytest.mark.parametrize("eps", [1e-60, 1e-46, 1e39, float("nan"), -1e-60])
@pytest.mark.parametrize("f", [lambda **kw: gated_norm(x, **kw), lambda **kw: residual_norm(x, x, **kw)], ids=["gated", "residual"])
def test_eps(f, eps):
    with pytest.raises(ValueError, match="eps"):
        f(eps=eps)


@pytest.mark.parametrize("more", [dict(scale=0), dict(scale=-0.0), dict(scale=3.4e38), dict(scale=-2.0 ** -149), dict(scale=3),
                                  dict(eps=0), dict(eps=2.0 ** -149), dict(eps=3.4e38)])
def test_numbers_that_it_holds(more):
    with pytest.raises(ValueError, match="GPU"):
        residual_norm(x, x, **more)
