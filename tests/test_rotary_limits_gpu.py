"""Rotations of more threads than one dimension of a launch has."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("s", [1 << 29, (1 << 29) + 1, 1431655777])
def test_more_than_2_to_the_32_threads(tracea_gpu, s):
    """One pair a head: a thread per token, three batch entries (up to 4.3e9 tokens); every entry turned by a quarter."""
    q = torch.empty(3, 1, s, 2, device="cuda", dtype=torch.float16)
    q[..., 0], q[..., 1] = 1.0, 2.0
    pos = torch.ones(1, s, 1, device="cuda", dtype=torch.int32)
    out = torch.zeros_like(q)
    tracea_gpu.rotary(q, None, pos, torch.full((1,), 1.5707963267948966, device="cuda"), q_out=out)
    for i in range(3):  # (cos of the fp32 quarter is 4.4e-8)
        assert (out[i, ..., 0] == -2.0).all() and (out[i, ..., 1] == 1.0).all()
