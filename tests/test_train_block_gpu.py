"""The example block: its gradients against plain torch on the same 16-bit weights, and that it learns."""
import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def plain(block, x, positions, lengths=None):
    """The block in 64 bits on the CPU."""
    p = {n: v.detach().cpu().to(torch.bfloat16).double() if v.dim() == 2 and "gates" not in n else v.detach().cpu().double()
         for n, v in block.named_parameters()}
    for v in p.values():
        v.requires_grad_(True)
    d, h, g = block.head_dim, block.heads, block.kv_heads

    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def heads(t):
        return t.unflatten(-1, (-1, d)).transpose(1, 2)
    pos, freq = positions.cpu().double(), block.inv_freq.cpu().double()
    axis = torch.repeat_interleave(torch.arange(pos.shape[-1]), torch.tensor(block.sections))
    angle = (pos[..., axis] * freq)[:, None]

    def turn(t):
        u, v = t.chunk(2, -1)
        return torch.cat([u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()], -1)
    y = norm(x, p["norms.0"])
    q, k, v = (y @ p["w_qkv"].t()).split([h * d, g * d, g * d], -1)
    q, k, v = turn(heads(q)), turn(heads(k)).repeat_interleave(h // g, 1), heads(v).repeat_interleave(h // g, 1)
    s = q @ k.transpose(-1, -2) / math.sqrt(d)
    if lengths is not None:
        n = torch.arange(x.shape[1])
        s = s.masked_fill((n[None] >= lengths.cpu()[:, None])[:, None, None], -math.inf)
    o = torch.softmax(s, -1) @ v
    if lengths is not None:
        o = o * (n[None] < lengths.cpu()[:, None])[:, None, :, None]
    o = o.transpose(1, 2).flatten(2) @ p["w_o"].t()
    x = x + p["gates.0"] * norm(o, p["norms.1"])
    y = norm(x, p["norms.2"])
    y = torch.nn.functional.silu(y @ p["w_up"].t()) @ p["w_down"].t()
    return x + p["gates.1"] * norm(y, p["norms.3"]), p


@pytest.mark.parametrize("grid,heads,kv,lengths", [((3, 4, 5), 4, 2, None), ((37,), 4, 4, [37, 20]), ((6, 11), 6, 1, None)])
def test_gradients_of_the_block(tracea_gpu, grid, heads, kv, lengths):
    import train_attention_block as ex
    torch.manual_seed(1)
    block = ex.Block(128, heads, kv, 64, len(grid)).to("cuda")
    positions = ex.grid_positions(grid, "cuda")
    x = torch.randn(2, positions.shape[1], 128, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(2, positions.shape[1], 128, device="cuda").bfloat16()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = block(x, positions, n)
    out.backward(dy)
    ref_x = x.detach().cpu().double().requires_grad_(True)
    ref, params = plain(block, ref_x, positions, n)
    ref.backward(dy.cpu().double())

    def off(a, b):
        return float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    # some ten 16-bit roundings one behind the other, each a relative 2^-9.8 (rms): 3.2 of them in 2-norm; four times that, and the
    # ReLU's few switched signs, is the bound
    assert off(out, ref) <= 0.015
    assert off(x.grad, ref_x.grad) <= 0.03
    for name, p in block.named_parameters():
        assert off(p.grad, params[name].grad) <= 0.04, name


def test_it_learns(tracea_gpu):
    import train_attention_block as ex
    losses = ex.train(grid=(2, 6, 6), steps=15)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.6 * losses[0], losses
