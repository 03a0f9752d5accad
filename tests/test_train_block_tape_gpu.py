"""The example block under torch's tape: gradients as the tape brings them, and what it does not offer."""
import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def make(grid=(5, 7), heads=4, kv=2, seed=1, batch=2):
    import train_attention_block as ex
    torch.manual_seed(seed)
    block = ex.Block(128, heads, kv, 64, len(grid)).to("cuda")
    positions = ex.grid_positions(grid, "cuda")
    x = torch.randn(batch, positions.shape[1], 128, device="cuda").bfloat16().requires_grad_(True)
    return block, x, positions


def gradients(block, x, out, d_out):
    block.zero_grad(set_to_none=True)
    x.grad = None
    out.backward(d_out)
    return [x.grad] + [p.grad for p in block.parameters()]


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 1), (1, 35, 1), (1, 1, 128)], ids=str)
def test_expanded_gradients(tracea_gpu, shape):
    """The gradient of a sum, and others whose strides are zero: as if they were written out."""
    block, x, positions = make()
    d = torch.randn(shape, device="cuda").bfloat16().expand(x.shape)
    want = gradients(block, x, block(x, positions), d.contiguous())
    for a, b in zip(gradients(block, x, block(x, positions), d), want):
        assert torch.equal(a, b)


def test_the_sum_of_the_results(tracea_gpu):
    import train_attention_block as ex
    block, x, positions = make()
    block(x, positions).sum().backward()
    assert torch.isfinite(x.grad).all()
    # each operator that a gradient may meet first
    q, k = (torch.randn(1, h, 35, 64, device="cuda").bfloat16().requires_grad_(True) for h in (4, 2))
    for result in (ex.Rotary.apply(q, k, positions, block.inv_freq, block.sections)[0], ex.Attention.apply(q, k, k, None),
                   ex.Linear.apply(q, block.w_o.detach()[:, :64].bfloat16()), ex.NormGateResidual.apply(x, None, None, None, block.norms[0])[1]):
        result.sum().backward()
    assert torch.isfinite(q.grad).all() and torch.isfinite(k.grad).all()


def test_second_derivatives_are_refused_with_the_reason(tracea_gpu):
    block, x, positions = make()
    g, = torch.autograd.grad(block(x, positions).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().square().sum().backward()
