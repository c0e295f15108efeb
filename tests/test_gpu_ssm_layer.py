"""The example of a served state-space layer: its operators together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture()
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pto-einsum_amd", "examples",
                        "state_space_layer.py")
    spec = importlib.util.spec_from_file_location("state_space_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    grad = torch.is_grad_enabled()
    yield module
    torch.set_grad_enabled(grad)


def test_tokens_continue_prompts(example):
    """Prompts and tokens round at the same places but for the order of float32
    sums, which moves some of a layer's bfloat16 values (convolution, scan and two
    projections) by one step of 2^-8: a few of the last projection's 512 terms, each
    some 1 / sqrt(512) of an output."""
    assert example.main() <= 2.0 ** -6


def test_quantize_keeps_levels(example):
    """Weights that lie on 16 levels come back exactly, whatever the length."""
    from pto_einsum import matvec_q4

    g = torch.Generator().manual_seed(0)
    q = torch.randint(0, 16, (12, 75), generator=g)
    q[:, 0::32], q[:, 1::32] = 0, 15
    w = (q.float() - 4) * 0.25
    packed, scales, zeros = example.quantize(w, 32)
    y = matvec_q4(torch.eye(75).cuda(), packed.cuda(), scales.cuda(), zeros.cuda(), group=32)
    assert torch.equal(y.cpu(), w.t())
