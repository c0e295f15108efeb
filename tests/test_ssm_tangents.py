"""Operands with forward-mode tangents, which the state-space operators and the
4-bit product would drop, are refused; on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

from pto_einsum import causal_conv, causal_conv_step, matvec_q4, selective_scan, selective_scan_step
from test_ssm_refusals import conv_args, f16, scan_args

CALLS = [
    (causal_conv, conv_args(), ("x", "weight", "bias")),
    (causal_conv_step, conv_args(x=torch.zeros(2, 8, dtype=f16), state=torch.zeros(2, 3, 8, dtype=f16)),
     ("x", "weight", "state", "bias")),
    (selective_scan, scan_args(D=torch.zeros(4), z=torch.zeros(2, 5, 4, 8, dtype=f16), dt_bias=torch.zeros(4),
                               initial_state=torch.zeros(2, 4, 8, 16)),
     ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")),
    (selective_scan_step, scan_args(lead=(2,), state=torch.zeros(2, 4, 8, 16)), ("x", "dt", "A", "B", "C", "state")),
    (matvec_q4, dict(x=torch.zeros(2, 50, dtype=f16), packed=torch.zeros(3, 25, dtype=torch.uint8),
                     scales=torch.zeros(3, 2, dtype=f16), zeros=torch.zeros(3, 2, dtype=f16), group=32),
     ("x", "scales", "zeros")),
]


@pytest.mark.parametrize("f,args,name", [(f, a, n) for f, a, names in CALLS for n in names],
                         ids=[f"{f.__name__}-{n}" for f, _, names in CALLS for n in names])
def test_tangents_are_refused(f, args, name):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(**{**args, name: dual})
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            f(**{**args, name: dual})
        # no tangent, or none any more: as far as without a level
        for plain in (args[name], dual.detach()):
            with pytest.raises(ValueError, match="GPU"):
                f(**{**args, name: plain})
