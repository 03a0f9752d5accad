"""Trains a small attention block over image or video tokens, every operator forward and backward by this library.

    tokens -> norm -> q, k, v -> rotary positions (one axis per dimension of the grid) -> attention -> projection
           -> gate, residual sum, norm -> two linear layers with SiLU -> gate, residual sum

torch keeps the tape, the optimizer, the memory and the SiLU; the rest of the block's arithmetic is ``tracea_amd.ops``:
``norm_gate_residual``, ``rotary``, ``attention_forward`` / ``attention_backward`` and ``gemm`` for the linear layers and their
two gradients.  Gradients of gradients are not offered: torch's tape says so where one is asked for.

    python examples/train_attention_block.py [--grid 4 8 8] [--steps 20]
"""
import argparse
import os
import sys

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tracea_amd import capi, ops  # noqa: E402


def in_rows(t):
    """A gradient as the tape brings it: one that was expanded (that of a sum has only strides of zero) is written out, because rotary
    and the norms read contiguous rows of channels."""
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


class Linear(torch.autograd.Function):
    """y = x w^T for tokens x [..., K] and w [N, K]."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return ops.gemm(x.reshape(-1, x.shape[-1]), w.t()).view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dy = dy.reshape(-1, dy.shape[-1])
        return ops.gemm(dy, w).view(x.shape), ops.gemm(dy.t(), x.reshape(-1, x.shape[-1]))


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections):
        ctx.save_for_backward(positions, inv_freq)
        ctx.sections = sections
        return ops.rotary(q, k, positions, inv_freq, sections)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        return (*ops.rotary(in_rows(dq), in_rows(dk), positions, inv_freq, ctx.sections, inverse=True), None, None, None)


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths):
        o, lse = ops.attention_forward(q, k, v, q_lengths=lengths, k_lengths=lengths)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.lengths = lengths
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        return (*ops.attention_backward(*ctx.saved_tensors, d_o, q_lengths=ctx.lengths, k_lengths=ctx.lengths), None)


class NormGateResidual(torch.autograd.Function):
    """(x_out, y): the sum between two blocks and the norm in front of the second; h None: the first norm, w_pre None: the last sum."""

    @staticmethod
    def forward(ctx, x, h, w_post, gate, w_pre):
        x_out, y = ops.norm_gate_residual(x, h, w_post, gate, w_pre)
        ctx.save_for_backward(x_out, h, w_post, gate, w_pre)
        ctx.set_materialize_grads(False)
        return (x_out.view_as(x) if h is None else x_out), y

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_out, dy):
        x_out, h, w_post, gate, w_pre = ctx.saved_tensors
        if w_pre is not None and dy is None:
            dy = torch.zeros_like(x_out)
        return ops.norm_gate_residual_backward(in_rows(dx_out), in_rows(dy), x_out, h, w_post, gate, w_pre)


class Block(torch.nn.Module):
    def __init__(self, channels, heads, kv_heads, head_dim, axes, dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        c, d = channels, head_dim
        matrix = lambda n, k: torch.nn.Parameter(torch.randn(n, k) * k ** -0.5)  # noqa: E731
        self.w_qkv = matrix((heads + 2 * kv_heads) * d, c)
        self.w_o, self.w_up, self.w_down = matrix(c, heads * d), matrix(4 * c, c), matrix(c, 4 * c)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(c)) for _ in range(4)])
        self.gates = torch.nn.ParameterList([torch.nn.Parameter(torch.full((1, c), 0.5)) for _ in range(2)])
        pairs = d // 2
        self.sections = [pairs // axes + (a < pairs % axes) for a in range(axes)]
        self.register_buffer("inv_freq", torch.cat([100.0 ** (-torch.arange(n, dtype=torch.float32) / n) for n in self.sections]))

    def forward(self, x, positions, lengths=None):
        b, t, _ = x.shape
        d, h, g = self.head_dim, self.heads, self.kv_heads
        half = lambda w: w.to(self.dtype)  # noqa: E731
        heads = lambda y: y.unflatten(-1, (-1, d)).transpose(1, 2)  # noqa: E731
        x, y = NormGateResidual.apply(x, None, None, None, self.norms[0])
        q, k, v = Linear.apply(y, half(self.w_qkv)).split([h * d, g * d, g * d], dim=-1)
        q, k = Rotary.apply(heads(q), heads(k), positions, self.inv_freq, self.sections)
        o = Attention.apply(q, k, heads(v), lengths).transpose(1, 2).reshape(b, t, h * d)
        o = Linear.apply(o, half(self.w_o))
        x, y = NormGateResidual.apply(x, o, self.norms[1], self.gates[0], self.norms[2])
        y = Linear.apply(torch.nn.functional.silu(Linear.apply(y, half(self.w_up))), half(self.w_down))
        return NormGateResidual.apply(x, y, self.norms[3], self.gates[1], None)[0]


def grid_positions(sizes, device):
    axes = torch.meshgrid(*[torch.arange(n, dtype=torch.int32, device=device) for n in sizes], indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], dim=-1)[None].contiguous()


def train(grid=(4, 8, 8), batch=2, channels=256, heads=8, kv_heads=2, head_dim=64, steps=20, seed=0, lr=2e-3, report=None):
    """Losses of `steps` steps at undoing a fixed mixing of the tokens (synthetic data)."""
    capi.init()
    torch.manual_seed(seed)
    dev = torch.device("cuda:0")
    block = Block(channels, heads, kv_heads, head_dim, len(grid)).to(dev)
    positions = grid_positions(grid, dev)
    tokens = positions.shape[1]
    x = torch.randn(batch, tokens, channels, device=dev)
    target = 0.5 * (x.roll(1, dims=1) + x.mean(1, keepdim=True))
    optimizer = torch.optim.AdamW(block.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        loss = (block(x.to(block.dtype), positions).float() - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if report:
            report("step %2d  loss %.4f" % (step, losses[-1]))
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--grid", type=int, nargs="+", default=[4, 8, 8], help="extents of the token grid, 1 to 4 axes")
    ap.add_argument("--batch", type=int, default=2)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    train(tuple(a.grid), a.batch, steps=a.steps, report=lambda s: print(s, flush=True))
