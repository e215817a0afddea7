"""A CCQ gated-delta-rule block on this framework's kernels: norm with the residual stream, projections, l2norm +
cleaning read + gated delta rule, gated norm, output projection.  It takes training steps, then generates from a
prompt with the cache and checks the generated outputs against one pass over the whole sequence.

    python examples/gdn_block.py            # needs a B200 and the built library
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ccq_b200  # noqa: E402


class GDNBlock(torch.nn.Module):
    def __init__(self, width, heads, value_heads=None, head_size=128, value_size=128, dtype=torch.bfloat16):
        super().__init__()
        self.H, self.HV, self.K, self.V = heads, value_heads or heads, head_size, value_size
        self.norm_weight = torch.nn.Parameter(torch.ones(width))
        self.head_weight = torch.nn.Parameter(torch.ones(value_size))
        sizes = [heads * head_size] * 2 + [self.HV * value_size] * 2 + [self.HV] * 2 + [heads]
        self.sizes = sizes
        self.proj = torch.nn.Linear(width, sum(sizes), bias=False, dtype=dtype)
        self.out = torch.nn.Linear(self.HV * value_size, width, bias=False, dtype=dtype)
        # decay -A softplus(a + bias), A in 1..16 and steps of 0.001..0.1 by head
        self.log_a = torch.nn.Parameter(torch.log(torch.linspace(1.0, 16.0, self.HV)))
        step = torch.exp(torch.linspace(math.log(0.001), math.log(0.1), self.HV))
        self.step_bias = torch.nn.Parameter(torch.log(torch.expm1(step)))

    def forward(self, x, stream, cache=None, output_cache=False, cu_seqlens=None):
        """x: the last block's output [B, T, width]; stream: the residual stream it is added to.
        Returns (this block's output, the stream, the cache or None)."""
        B, T, _ = x.shape
        x, stream = ccq_b200.rms_norm(x, self.norm_weight, residual=stream)
        q, k, v, gate, a, b, lam = self.proj(x).split(self.sizes, -1)
        q, k = (t.reshape(B, T, self.H, self.K) for t in (q, k))
        v, gate = (t.reshape(B, T, self.HV, self.V) for t in (v, gate))
        g = -torch.exp(self.log_a) * torch.nn.functional.softplus(a.float() + self.step_bias)
        beta, lam = torch.sigmoid(b), torch.sigmoid(lam)
        if self.H != self.HV and self.HV % self.H:
            raise ValueError('value_heads must be a multiple of heads')
        if cache is not None and T <= 64 and not torch.is_grad_enabled() and cu_seqlens is None:
            o, cache = ccq_b200.ccq_gated_delta_step(q, k, v, lam, g, beta, cache)
        else:
            o, cache = ccq_b200.ccq_gated_delta_rule(q, k, v, lam, g, beta, cache=cache, output_cache=output_cache,
                                                     cu_seqlens=cu_seqlens)
        o = ccq_b200.gated_rms_norm(o, gate, self.head_weight)
        return self.out(o.reshape(B, T, -1)), stream, cache


def train(block, steps=5, B=2, T=512, width=512, device='cuda', seed=0):
    """Fits the block to a fixed target; returns the losses."""
    gen = torch.Generator(device=device).manual_seed(seed)
    x, s, y = (torch.randn(B, T, width, generator=gen, device=device).bfloat16() for _ in range(3))
    opt = torch.optim.SGD(block.parameters(), lr=0.5)
    losses = []
    for _ in range(steps):
        o, _, _ = block(x, s)
        loss = (o.float() - y.float()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def generate(block, prompt=200, tokens=8, B=2, width=512, device='cuda', seed=1):
    """Prefill, then one token at a time over the cache; returns how far the generated outputs are (2-norm) from
    those of one pass over everything."""
    gen = torch.Generator(device=device).manual_seed(seed)
    x, s = (torch.randn(B, prompt + tokens, width, generator=gen, device=device).bfloat16() for _ in range(2))
    whole, _, _ = block(x, s)
    _, _, cache = block(x[:, :prompt], s[:, :prompt], output_cache=True)
    off = 0.0
    for t in range(prompt, prompt + tokens):
        o, _, cache = block(x[:, t:t + 1], s[:, t:t + 1], cache)
        want = whole[:, t:t + 1].float()
        off = max(off, ((o.float() - want).norm() / want.norm()).item())
    return off


if __name__ == '__main__':
    torch.manual_seed(0)
    block = GDNBlock(512, 4, 8).cuda()
    print('losses:', ' '.join(f'{v:.4f}' for v in train(block)))
    print(f'generation against one pass: {generate(block):.2e}')
