"""A state-space layer served with 4-bit weights.

    python pto-einsum_amd/examples/state_space_layer.py

Prompts of unequal lengths run packed (projection, causal convolution, selective
scan, projection) and leave their states in two caches; single tokens then
continue from the caches, a step captured once into a StageGraph and replayed.
The tokens' outputs are compared with those of the prompts run to their ends.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))
from pto_einsum import (StageGraph, causal_conv, causal_conv_step, matvec_q4, selective_scan,  # noqa: E402
                        selective_scan_step)


def quantize(w: torch.Tensor, group: int):
    """(packed, scales, zeros) of a weight [N, K] for matvec_q4: 16 levels from the
    least to the largest value of each group along K."""
    n, k = w.shape
    pad = -k % group
    g = torch.nn.functional.pad(w.float(), (0, pad), mode="replicate" if pad else "constant").unflatten(1, (-1, group))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).clamp(min=1e-8)
    q = torch.round((g - low) / scale).clamp(0, 15).to(torch.uint8).flatten(1)[:, :k]
    q = torch.nn.functional.pad(q, (0, k % 2))
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale[..., 0].to(w.dtype), (-low / scale)[..., 0].to(w.dtype)


class Layer:
    def __init__(self, d_model=256, heads=8, head_dim=64, groups=2, d_state=64, width=4, group=64,
                 dtype=torch.bfloat16, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        self.h, self.p, self.g, self.n, self.group = heads, head_dim, groups, d_state, group
        inner, bc = heads * head_dim, groups * d_state
        self.split = (inner, inner + 2 * bc, heads)          # gate; x, B, C; step sizes

        def put(t):
            return t.to(dtype).to(device)

        self.w_in = [t.to(device) for t in quantize((torch.randn(sum(self.split), d_model, generator=g)
                                                     / d_model ** 0.5).to(dtype), group)]
        self.w_out = [t.to(device) for t in quantize((torch.randn(d_model, inner, generator=g)
                                                      / inner ** 0.5).to(dtype), group)]
        self.conv_w = put(torch.randn(inner + 2 * bc, width, generator=g) * width ** -0.5)
        self.conv_b = put(torch.zeros(inner + 2 * bc))
        step = torch.exp(torch.empty(heads).uniform_(-6.9, -2.3, generator=g))
        self.dt_bias = (step + torch.log(-torch.expm1(-step))).to(device)
        self.A = -torch.empty(heads).uniform_(1, 16, generator=g).to(device)
        self.D = torch.ones(heads, device=device)
        self.dtype, self.device, self.width = dtype, device, width

    def caches(self, slots: int):
        inner = self.h * self.p + 2 * self.g * self.n
        return (torch.zeros(slots, self.width - 1, inner, dtype=self.dtype, device=self.device),
                torch.zeros(slots, self.h, self.p, self.n, device=self.device))

    def _project(self, u):
        return matvec_q4(u, *self.w_in, group=self.group).split(self.split, -1)

    def _operands(self, xbc):
        x, B, C = xbc.split((self.h * self.p, self.g * self.n, self.g * self.n), -1)
        return x.unflatten(-1, (self.h, self.p)), B.unflatten(-1, (self.g, self.n)), C.unflatten(-1, (self.g, self.n))

    def prompts(self, u, cu_seqlens):
        """u [tokens, d_model] of packed prompts: outputs and the states after each."""
        z, xbc, dt = self._project(u)
        xbc, conv_state = causal_conv(xbc, self.conv_w, self.conv_b, activation="silu", cu_seqlens=cu_seqlens)
        x, B, C = self._operands(xbc)
        y, state = selective_scan(x, dt, self.A, B, C, D=self.D, z=z.unflatten(-1, (self.h, self.p)),
                                  dt_bias=self.dt_bias, dt_softplus=True, cu_seqlens=cu_seqlens)
        return matvec_q4(y.flatten(-2), *self.w_out, group=self.group), conv_state, state

    def tokens(self, u, conv_state, state, slots):
        """One token u [B, d_model] of each sequence, its states in the caches' slots."""
        z, xbc, dt = self._project(u)
        x, B, C = self._operands(causal_conv_step(xbc, self.conv_w, conv_state, self.conv_b, activation="silu",
                                                  slots=slots))
        y = selective_scan_step(x, dt, self.A, B, C, state, D=self.D, z=z.unflatten(-1, (self.h, self.p)),
                                dt_bias=self.dt_bias, dt_softplus=True, slots=slots)
        return matvec_q4(y.flatten(-2), *self.w_out, group=self.group)


def main(lens=(37, 5, 150), more=6) -> float:
    """The largest difference, relative to the largest output."""
    torch.set_grad_enabled(False)
    layer, g = Layer(), torch.Generator().manual_seed(1)
    seqs = [torch.randn(n + more, 256, generator=g).to(layer.dtype).cuda() for n in lens]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)

    def cu(step):
        return torch.tensor([o + i * step for i, o in enumerate(offsets)], dtype=torch.int32).cuda()

    whole, _, _ = layer.prompts(torch.cat(seqs), cu(more))
    _, conv_state, state = layer.prompts(torch.cat([s[:n] for s, n in zip(seqs, lens)]), cu(0))
    conv_cache, cache = layer.caches(8)
    slots = torch.tensor([6, 1, 4], dtype=torch.int32).cuda()
    conv_cache[slots.long()], cache[slots.long()] = conv_state, state
    u = torch.zeros(len(lens), 256, dtype=layer.dtype).cuda()
    kept = conv_cache.clone(), cache.clone()
    step = StageGraph(lambda: layer.tokens(u, conv_cache, cache, slots))
    conv_cache.copy_(kept[0]), cache.copy_(kept[1])          # capturing ran the step
    worst = 0.0
    for t in range(more):
        u.copy_(torch.stack([s[n + t] for s, n in zip(seqs, lens)]))
        got = step.replay().float()
        want = torch.stack([whole[o + i * more + n + t] for i, (o, n) in enumerate(zip(offsets, lens))]).float()
        worst = max(worst, float((got - want).abs().max() / want.abs().max()))
    return worst


if __name__ == "__main__":
    print(f"state-space layer: tokens against whole prompts, largest difference {main():.2e} of the largest output")
