"""Operands whose elements lie more than 2^32 bytes apart: the operators for training give what they give for dense ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS = 300


class Spread:
    """Tensors [1,H,S,D] side by side in rows `pitch` elements apart."""

    def __init__(self, pitch, dtype):
        self.pitch, self.at = pitch, 0
        self.buffer = torch.empty(ROWS * pitch, dtype=dtype, device="cuda")

    def like(self, t, copy=True):
        _, h, s, d = t.shape
        v = self.buffer.as_strided((1, h, s, d), (s * self.pitch, d, self.pitch, 1), self.at)
        self.at += h * d
        if copy:
            v.copy_(t)
        return v


# (64 rows of the first pitch fit the 32-bit offsets inside a tile, of the second they do not: copies)
@pytest.mark.parametrize("pitch", [16_000_000, 18_000_000])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(tracea_gpu, pitch, causal):
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(1, h, ROWS, 64, generator=g).cuda().bfloat16() for h in (4, 2, 2, 4))
    o, lse = tracea_gpu.attention_forward(q, k, v, causal=causal)
    dense = tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=causal)
    far = Spread(pitch, torch.bfloat16)
    out = Spread(pitch, torch.bfloat16)
    fq, fk, fv, fdo = far.like(q), far.like(k), far.like(v), far.like(do)
    fo, flse = tracea_gpu.attention_forward(fq, fk, fv, causal=causal, out=out.like(o, False))
    assert torch.equal(fo, o) and torch.equal(flse, lse)
    got = tracea_gpu.attention_backward(fq, fk, fv, fo, flse, fdo, causal=causal, dq=out.like(q, False), dk=out.like(k, False),
                                        dv=out.like(v, False))
    for a, b in zip(got, dense):
        assert torch.equal(a, b)


def test_rotary(tracea_gpu):
    g = torch.Generator().manual_seed(6)
    q, k = (torch.randn(1, h, ROWS, 64, generator=g).cuda().bfloat16() for h in (12, 3))
    pos = torch.arange(ROWS, dtype=torch.int32, device="cuda").view(1, ROWS, 1)
    freq = torch.logspace(0, -3, 32, device="cuda")
    dense = tracea_gpu.rotary(q, k, pos, freq)
    far = Spread(16_000_000, torch.bfloat16)
    fq, fk = far.like(q), far.like(k)
    got = tracea_gpu.rotary(fq, fk, pos, freq, q_out=fq, k_out=fk)
    for a, b in zip(got, dense):
        assert torch.equal(a, b)


@pytest.mark.parametrize("c", [512, 501])
def test_norm_gate_residual(tracea_gpu, c):
    g = torch.Generator().manual_seed(7)
    x, h, dx, dy = (torch.randn(1, ROWS, c, generator=g).cuda().bfloat16() for _ in range(4))
    w, gate = torch.randn(c, generator=g).cuda(), torch.randn(1, c, generator=g).cuda()
    x_out, y = tracea_gpu.norm_gate_residual(x, h, w, gate, w)
    dense = tracea_gpu.norm_gate_residual_backward(dx, dy, x_out, h, w, gate, w)
    far = Spread(16_000_000, torch.bfloat16)

    def rows(t):
        return far.like(t.unsqueeze(1)).squeeze(1)
    fx, fh, fdx, fdy = rows(x), rows(h), rows(dx), rows(dy)
    fo, fy = tracea_gpu.norm_gate_residual(fx, fh, w, gate, w, x_out=rows(x), y=rows(x))
    assert torch.equal(fo, x_out) and torch.equal(fy, y)
    got = tracea_gpu.norm_gate_residual_backward(fdx, fdy, fo, fh, w, gate, w, dx=fdx, dh=fh)
    for a, b in zip(got, dense):
        assert torch.equal(a, b)
