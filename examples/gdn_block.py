"""One Gated DeltaNet block end to end: ragged prompts into 8-bit recurrent states, then decode from them.

    python examples/gdn_block.py [--lens 4096,1000,3,517] [--steps 64]

    x, h -> in_proj(h) = q | k | v | z | b | a;  y = out_proj(gated_norm(rule(conv(q | k | v)), z));  x, h = add_norm(x, y)

The prompts take the operators for whole sequences (`leapquant_amd.seq`: the ragged conv, the chunked gated delta rule) through
`LeapQuantState.prefill`, which leaves the layer's 8-bit checkpoint; each decode token then takes one `decode_conv` call on it.
The weights are random, in bf16.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from leapquant_amd import seq                                       # noqa: E402
from leapquant_amd.state import LeapQuantState                      # noqa: E402

BF16 = torch.bfloat16


class GDNBlock:
    """Weights, conv cache and state cache of a block with `slots` sequences (slot 0 pads)."""

    def __init__(self, hidden, H, HV, D, slots, device="cuda:0", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device=device)                 # noqa: E731
        self.hidden, self.H, self.HV, self.D = hidden, H, HV, D
        self.C = C = 2 * H * D + HV * D
        self.w_in = (rn(hidden, C + HV * D + 2 * HV) * hidden ** -0.5).to(BF16)
        self.w_out = (rn(HV * D, hidden) * (HV * D) ** -0.5).to(BF16)
        self.w_conv, self.norm_core, self.norm_next = (0.5 * rn(C, 4)).to(BF16), torch.ones(D, device=device), torch.ones(hidden, device=device)
        # rates 1 to 16 a head, time steps 1e-3 to 0.1
        u = torch.rand(2, HV, generator=g, device=device)
        self.A_log = torch.log(1 + 15 * u[0])
        self.dt_bias = torch.log(torch.expm1(1e-3 * 100 ** u[1]))
        self.conv = torch.zeros(slots + 1, C, 3, device=device, dtype=BF16)
        self.ssm = torch.zeros(slots + 1, HV, D, D, device=device)
        self.state = LeapQuantState(self.ssm, H)

    def _project(self, h):
        return torch.matmul(h, self.w_in).split([self.C, self.HV * self.D, self.HV, self.HV], -1)

    def _close(self, x, o, z):
        """Gated norm, output projection, residual and the norm before the next block: (x, h)."""
        seq.gated_norm(o, z.unflatten(-1, (self.HV, self.D)), self.norm_core, o)
        y, h = torch.matmul(o.flatten(1), self.w_out), torch.empty_like(x)
        seq.add_norm(x, y, self.norm_next, y, h)
        return y, h

    def prefill(self, x, h, idx, loc, has_state=None, longest=None):
        """x, h [T, hidden]: the residual stream and its norm, the packed tokens of the sequences in slots idx, at most `longest` each."""
        mixed, z, b, a = self._project(h)
        src = torch.zeros_like(idx) if has_state is None else idx * has_state
        m = torch.empty(x.shape[0], self.C, device=x.device, dtype=BF16)
        seq.conv_prefill(mixed, self.conv, self.w_conv, None, idx, loc, m, src=src)
        o = torch.empty(x.shape[0], self.HV, self.D, device=x.device, dtype=BF16)
        self.state.prefill(self.ssm, m, a, b, self.A_log, self.dt_bias, idx, loc, o, has_state=has_state, longest=longest)
        return self._close(x, o, z)

    def decode(self, x, h, idx):
        """One token of each slot in idx."""
        mixed, z, b, a = self._project(h)
        o = torch.empty(x.shape[0], self.HV, self.D, device=x.device, dtype=BF16)
        self.state.decode_conv(self.ssm, mixed.contiguous(), self.conv, self.w_conv, None, True, a.contiguous(), b.contiguous(),
                               self.A_log, self.dt_bias, idx, o)
        return self._close(x, o, z)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--lens", default="4096,1000,3,517")
    p.add_argument("--steps", type=int, default=64)
    a = p.parse_args()
    lens = [int(n) for n in a.lens.split(",")]
    dev, hidden = "cuda:0", 2048
    block = GDNBlock(hidden, 16, 32, 128, len(lens))
    g = torch.Generator(device=dev).manual_seed(1)
    idx = torch.arange(1, len(lens) + 1, dtype=torch.int32, device=dev)
    loc = torch.tensor([sum(lens[:n]) for n in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    x = torch.randn(sum(lens), hidden, generator=g, device=dev).to(BF16)
    ev = lambda: torch.cuda.Event(enable_timing=True)               # noqa: E731
    for timed in (False, True):
        t0, t1, t2 = ev(), ev(), ev()
        t0.record()
        y, h = block.prefill(x, x, idx, loc, longest=max(lens))
        t1.record()
        last = (loc[1:] - 1).long()
        y, h = y[last], h[last]
        for _ in range(a.steps):
            y, h = block.decode(y, h, idx)
        t2.record()
        torch.cuda.synchronize()
    print("prefill of %d tokens in %d sequences: %.3f ms; %d decode steps: %.1f us each; |h| %.4f"
          % (x.shape[0], len(lens), t0.elapsed_time(t1), a.steps, 1e3 * t1.elapsed_time(t2) / a.steps, float(h.float().norm())))


if __name__ == "__main__":
    main()
