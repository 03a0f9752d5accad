"""Results of attention over the vectors of lengths that the same call reads: refused."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q_lengths", "k_lengths"])
def test_results_over_the_lengths_are_refused(tracea_gpu, which):
    from tracea_amd import capi
    q = torch.randn(4, 2, 6, 64, device="cuda").half()
    memory = torch.full((4 * 2 * 6 * 64 // 2,), 6, device="cuda", dtype=torch.int32)
    as_half = memory.view(torch.float16).view(4, 2, 6, 64)
    as_lse = memory.view(torch.float32)[:48].view(4, 2, 6)
    n = {which: memory[:4]}
    o, lse = tracea_gpu.attention_forward(q, q, q, **n)

    def refused(call, **kw):
        with pytest.raises(capi.TraceaError) as e:
            call(**kw)
        assert e.value.status == capi.INVALID_PARAMS, e.value
    refused(lambda **kw: tracea_gpu.attention_forward(q, q, q, **n, **kw), out=as_half)
    refused(lambda **kw: tracea_gpu.attention_forward(q, q, q, **n, **kw), lse=as_lse)
    for name in ("dq", "dk", "dv"):
        refused(lambda **kw: tracea_gpu.attention_backward(q, q, q, o, lse, q, **n, **kw), **{name: as_half})
    assert (memory == 6).all()
    tracea_gpu.attention_backward(q, q, q, o, lse, q, **n)


def test_rotary_over_the_end_of_its_positions_is_refused(tracea_gpu):
    from tracea_amd import capi
    memory = torch.zeros(64 + 64 * 64, device="cuda", dtype=torch.int32)
    pos = memory[:64].view(1, 64, 1)
    out = memory[63:63 + 64 * 64].view(torch.float32).view(1, 1, 64, 64)  # (over the last position alone)
    with pytest.raises(capi.TraceaError) as e:
        tracea_gpu.rotary(torch.randn(1, 1, 64, 64, device="cuda"), None, pos, torch.ones(32, device="cuda"), q_out=out)
    assert e.value.status == capi.INVALID_PARAMS and "positions" in str(e.value)
