"""Numbers of rows at the limit of tracea_norm_gate_residual's 32-bit row counter."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 2 ** 20


@pytest.mark.parametrize("t", [MOST + 1, 2 ** 31 - 1])
def test_more_rows_are_refused(tracea_gpu, t):
    from tracea_amd import capi
    w = torch.ones(1, device="cuda")
    x = torch.empty(1, t, 1, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: tracea_gpu.norm_gate_residual(x, w_pre=w, y=x), lambda: tracea_gpu.norm_gate_residual_backward(x, x, x, w_pre=w, dx=x)):
        with pytest.raises(capi.TraceaError) as e:
            call()
        assert e.value.status == capi.UNSUPPORTED_CONFIG


def test_the_most_rows(tracea_gpu):
    w = torch.full((1,), 2.0, device="cuda")
    x = torch.empty(1, MOST, 1, device="cuda", dtype=torch.bfloat16)
    x.fill_(3.0)
    x[0, ::7] = -0.5
    y = torch.zeros_like(x)
    tracea_gpu.norm_gate_residual(x, w_pre=w, y=y)
    step = 1 << 28  # (a row of one channel: its sign times the weight, to within eps)
    for i in range(0, MOST, step):
        assert torch.equal(y[0, i:i + step], x[0, i:i + step].sign() * 2)
