"""Sizes, strides and overlaps at the limits of the operators for training: what is taken gives the formulas' results, the rest is refused."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk", [(16, 16), (32, 16)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_more_than_65535_problems(tracea_gpu, hq, hk, dtype):
    # windows of an image: 4100 of them with 16 key/value heads each
    from test_attention_train_gpu import check
    check(tracea_gpu, 4100, hq, hk, 3, 5, 8, dtype)
    check(tracea_gpu, 4100, hq, hk, 3, 3, 16, dtype, True)


def test_gradients_side_by_side_within_a_head(tracea_gpu):
    """Operands and gradients as [B,S,H,3,D]: the three share the range of a head's row and no element."""
    g = torch.Generator(device="cuda").manual_seed(11)
    qkv = torch.randn(2, 70, 4, 3, 64, device="cuda", generator=g).bfloat16()
    do = torch.randn(2, 4, 70, 64, device="cuda", generator=g).bfloat16()
    q, k, v = (qkv[:, :, :, i].transpose(1, 2) for i in range(3))
    o, lse = tracea_gpu.attention_forward(q, k, v, causal=True)
    want = tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True)
    grad = torch.zeros_like(qkv)
    part = {n: grad[:, :, :, i].transpose(1, 2) for i, n in enumerate(("dq", "dk", "dv"))}
    for a, b in zip(tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True, **part), want):
        assert torch.equal(a, b)
    # rotary over them, in place
    pos = torch.arange(70, dtype=torch.int32, device="cuda").view(1, 70, 1)
    freq = torch.logspace(0, -3, 32, device="cuda")
    want = tracea_gpu.rotary(q.contiguous(), k.contiguous(), pos, freq)
    for a, b in zip(tracea_gpu.rotary(q, k, pos, freq, q_out=q, k_out=k), want):
        assert torch.equal(a, b)


def test_results_that_share_elements_are_refused(tracea_gpu):
    from tracea_amd import capi
    q = torch.randn(2, 4, 10, 64, device="cuda").half()
    lse = torch.zeros(2, 4, 10, device="cuda")
    wide = torch.empty(2, 10, 4, 160, device="cuda").half()
    dq, dk, dv = (wide[..., i:i + 64].transpose(1, 2) for i in (0, 56, 96))
    with pytest.raises(capi.TraceaError) as e:
        tracea_gpu.attention_backward(q, q, q, q, lse, q, dq=dq, dk=dk, dv=torch.empty_like(q))
    assert e.value.status == capi.INVALID_PARAMS
    with pytest.raises(capi.TraceaError) as e:
        tracea_gpu.attention_backward(q, q, q, q, lse, q, dq=dq, dk=torch.empty_like(q), dv=wide[:, :, :, 1:65].transpose(1, 2))
    assert e.value.status == capi.INVALID_PARAMS


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_as_many_workgroups_as_a_launch_has(tracea_gpu, dtype):
    """Up to 2^24 - 1 workgroups of 256 threads (a launch of 2^32 threads and more drops some of them without an error)."""
    from tracea_amd import capi
    x = torch.randn(1 << 20, 16, 1, 8, device="cuda").to(dtype)
    lse = torch.empty(1 << 20, 16, 1, device="cuda")
    with pytest.raises(capi.TraceaError) as e:
        tracea_gpu.attention_forward(x, x, x, out=torch.empty_like(x), lse=lse)
    assert e.value.status == capi.UNSUPPORTED_CONFIG
    some = x[1:]
    o, lse = tracea_gpu.attention_forward(some, some, some)  # (one key: o is its value)
    assert torch.equal(o, some) and torch.isfinite(lse).all()
    with pytest.raises(capi.TraceaError) as e:
        tracea_gpu.attention_backward(some, some, some, o, lse, some)
    assert e.value.status == capi.UNSUPPORTED_CONFIG
    some, o, lse = some[: (1 << 19) - 1], o[: (1 << 19) - 1], lse[: (1 << 19) - 1]
    dq, dk, dv = tracea_gpu.attention_backward(some, some, some, o, lse, some)
    assert (dq == 0).all() and (dk == 0).all() and torch.equal(dv, some)


def test_padded_copies_of_the_next_multiple_of_8(tracea_gpu):
    """Head dimension 90 off 16 bytes: copies of 96 columns, which fit their buffer where 128 would not; the bits of a call with zeros behind
    the 90."""
    g = torch.Generator(device="cuda").manual_seed(21)
    wide = [torch.randn(4, 32, 4100, 96, device="cuda", generator=g).bfloat16() for _ in range(4)]
    for t in wide:
        t[..., 90:] = 0
    q, k, v, do = (torch.empty(4, 32, 4100, 91, device="cuda", dtype=torch.bfloat16)[..., 1:].copy_(t[..., :90]) for t in wide)
    o, lse = tracea_gpu.attention_forward(q, k, v, scale=0.1)
    got = (o, lse) + tracea_gpu.attention_backward(q, k, v, o, lse, do, scale=0.1)
    o, lse = tracea_gpu.attention_forward(*wide[:3], scale=0.1)
    want = (o, lse) + tracea_gpu.attention_backward(*wide[:3], o, lse, wide[3], scale=0.1)
    for a, b in zip(got, want):
        assert torch.equal(a, b if a.dim() == 3 else b[..., :90])
