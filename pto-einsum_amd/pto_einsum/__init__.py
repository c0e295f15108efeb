"""pto_einsum for AMD Instinct MI355X (gfx950).

Public API, unchanged from the reference (src/pto_einsum/__init__.py:12-15):

    einsum(equation, a, b, device="cuda")   -> float32 result tensor
    EinsumBuilder(equation, shapes, dtype)  -> reusable compiled runner
    INCLUDE_DIR                             -> headers the JIT sources compile against

Beyond the reference's surface:

    einsum(eq, a, b, reduce_solo_axes=True) -> also sums indices found in one operand
                                               only (e.g. "ij,jk->k"), which the
                                               reference rejects
    linear_attention(q, k, v, m)            -> fused einsum("tn,sn,sp,ts->tp"), float32
    causal_conv(x, weight, ...)             -> short causal convolution of each channel, and
    causal_conv_step(x, weight, state, ...)    the same for one token, its state in place
    selective_scan(x, dt, A, B, C, ...)     -> state-space scan of prompts, and
    selective_scan_step(x, ..., state)         the same for one token, its state in place
    matvec_q4(x, packed, scales, ...)       -> product of few rows with 4-bit weights
    StageGraph(fn)                          -> fn's launches captured into one HIP graph

Example:
    >>> from pto_einsum import einsum
    >>> c = einsum("ij, jk -> ik", a, b)    # a, b are tensors on the GPU
"""

from .builder import EinsumBuilder, INCLUDE_DIR, einsum
from .graph import StageGraph
from .linattn import linear_attention
from .quant import matvec_q4
from .ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

__all__ = ["einsum", "EinsumBuilder", "INCLUDE_DIR", "linear_attention", "StageGraph", "causal_conv",
           "causal_conv_step", "selective_scan", "selective_scan_step", "matvec_q4"]
__version__ = "0.2.0"
