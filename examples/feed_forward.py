"""Trains a gated feed-forward block twice, as msamp.nn.FeedForward and as FP8 linear layers with torch's operators between them:
loss, time of a step, memory held between the forward and the backward pass and the most that a step takes.

    python examples/feed_forward.py [--tokens 16384] [--width 4096] [--hidden 11008] [--steps 20]
"""

import argparse
import gc
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'ms-amp_amd'))

import msamp    # noqa: E402
from msamp.nn import FeedForward, model_state, saved_in_8_bits    # noqa: E402


class Plain(torch.nn.Module):
    """The same block with operators of its own for activation, gate and residual."""

    def __init__(self, up, down, gate):
        super().__init__()
        self.up, self.down, self.gate = up, down, gate

    def forward(self, x, residual):
        return self.down(torch.nn.functional.silu(self.gate(x)) * self.up(x)) + residual


class Block(torch.nn.Module):
    """x + feed_forward(norm(x))"""

    def __init__(self, feed_forward, width):
        super().__init__()
        self.norm = torch.nn.RMSNorm(width)
        self.feed_forward = feed_forward

    def forward(self, x):
        with saved_in_8_bits():    # what the norm saves
            y = self.norm(x)
        return self.feed_forward(y, residual=x)


def train(fused, args):
    model_state.clear()
    torch.manual_seed(0)
    up, down, gate = (torch.nn.Linear(a, b, bias=False) for a, b in ((args.width, args.hidden), (args.hidden, args.width), (args.width, args.hidden)))
    block = FeedForward(up, down, gate=gate, activation='silu') if fused else Plain(up, down, gate)
    model, optimizer = msamp.initialize(Block(block, args.width).bfloat16().cuda(), opt_level='O2')
    for group in optimizer.param_groups:
        group['lr'] = 2e-4
    x = torch.randn(args.tokens, args.width, device='cuda', dtype=torch.bfloat16)
    target = torch.roll(x, 1, dims=1)
    held = 0
    for step in range(args.steps):
        if step == args.steps // 2 - 5:
            gc.collect()    # (a collection of all generations takes some 80 ms: not in the steps that are timed, nor right before them)
        if step == args.steps // 2:
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            began = time.perf_counter()
        optimizer.zero_grad()
        if step == 1:    # the model, the optimizer's state and the data, without the last step's loss and what hangs on it
            y = loss = None
            stands = torch.cuda.memory_allocated()
        before = torch.cuda.memory_allocated()
        y = model(x)
        held = torch.cuda.memory_allocated() - before
        loss = (y - target).float().square().mean()
        loss.backward()
        optimizer.step()
    torch.cuda.synchronize()
    most = torch.cuda.max_memory_allocated() - stands
    ms = (time.perf_counter() - began) / (args.steps - args.steps // 2) * 1e3
    print(f'{"fused" if fused else "plain"}: loss {float(loss.detach()):.4f}, {ms:.2f} ms a step, {held / 2**20:.0f} MiB held after the forward pass, '
          f'{most / 2**20:.0f} MiB at most beside model and optimizer', flush=True)


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (('tokens', 16384), ('width', 4096), ('hidden', 11008), ('steps', 20)):
        parser.add_argument('--' + name, type=int, default=default)
    args = parser.parse_args()
    for fused in (False, True):
        train(fused, args)
