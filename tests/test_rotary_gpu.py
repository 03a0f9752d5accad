"""tracea_rotary against rotations in 64 bits.

Bound per element: the result's rounding (u |x|; fp32: u = 2^-24), and for the sine, the cosine and the two products 2^-21 of |u| + |v|."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SIN = 2.0 ** -21


def reference(x, pos, freq, sections, adjacent, inverse):
    x = x.cpu().double()
    b, h, s, d = x.shape
    p = freq.numel()
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = (pos.cpu().double()[..., axis] * freq.cpu().double()).expand(b, s, p)[:, None]
    if inverse:
        angle = -angle
    u_at = torch.arange(p) * 2 if adjacent else torch.arange(p)
    v_at = u_at + 1 if adjacent else u_at + p
    u, v = x[..., u_at], x[..., v_at]
    y, err = x.clone(), torch.zeros_like(x)
    y[..., u_at], y[..., v_at] = u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()
    err[..., u_at] = err[..., v_at] = SIN * (u.abs() + v.abs())
    return y, err


def within(got, want, dtype):
    ref, err = want
    far = (got.double().cpu() - ref).abs() - (U[dtype] * ref.abs() + 1.01 * err + 2.0 ** -25 * (dtype == torch.float16))
    assert far.max() <= 0, far.max()


def make(shape, dtype, layout, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, h, s, d = shape
    if layout == "bshd":
        return torch.randn(b, s, h, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
    if layout == "odd":
        return torch.randn(b, h, s, d + 3, device="cuda", generator=g).to(dtype)[..., 1:1 + d]
    return torch.randn(b, h, s, d, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", list(U), ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "adjacent"])
@pytest.mark.parametrize("d,sections", [(64, [32]), (128, [22, 21, 21]), (128, [16, 24, 24]), (64, [8, 16]), (40, [20]), (40, [5, 4]), (7, [3]),
                                        (2, [1]), (96, [12, 12, 12, 12]), (64, [0, 32]), (72, [36])])
def test_types_axes_and_widths(tracea_gpu, dtype, adjacent, d, sections):
    for layout, b, hq, hk, s, shared in (("bhsd", 2, 4, 2, 37, True), ("bshd", 3, 3, 1, 1, False), ("odd", 1, 2, 2, 65, False)):
        q, k = make((b, hq, s, d), dtype, layout, 1), make((b, hk, s, d), dtype, layout, 2)
        g = torch.Generator(device="cuda").manual_seed(3)
        pos = torch.randint(-50, 3000, (1 if shared else b, s, len(sections)), device="cuda", generator=g, dtype=torch.int32)
        freq = 10000.0 ** (-torch.rand(sum(sections), device="cuda", generator=g))
        for inverse in (False, True):
            got = tracea_gpu.rotary(q, k, pos, freq, sections, adjacent, inverse)
            for x, y in zip((q, k), got):
                within(y, reference(x, pos, freq, sections, adjacent, inverse), dtype)


def test_long_positions_lose_nothing(tracea_gpu):
    q = make((1, 2, 64, 64), torch.float32, "bhsd", 1)
    pos = (2 ** 31 - 1 - 7919 * torch.arange(64, device="cuda", dtype=torch.int64)).to(torch.int32).view(1, 64, 1)
    freq = 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float32) / 32)
    got, none = tracea_gpu.rotary(q, None, pos, freq)
    assert none is None
    within(got, reference(q, pos, freq, [32], False, False), torch.float32)


def test_many_heads_and_tokens(tracea_gpu):
    q, k = make((2, 40, 3000, 64), torch.bfloat16, "bshd", 1), make((2, 8, 3000, 64), torch.bfloat16, "bshd", 2)
    pos = torch.arange(6000, device="cuda", dtype=torch.int32).view(2, 3000)  # one axis, no axis dimension
    freq = 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float32) / 32)
    for x, y in zip((q, k), tracea_gpu.rotary(q, k, pos, freq)):
        within(y, reference(x, pos.unsqueeze(-1), freq, [32], False, False), torch.bfloat16)


@pytest.mark.parametrize("d,p", [(64, 32), (64, 24), (10, 3)])
def test_in_place_and_back(tracea_gpu, d, p):
    q, k = make((2, 4, 50, d), torch.float32, "bhsd", 1), make((2, 2, 50, d), torch.float32, "bhsd", 2)
    pos = torch.arange(50, device="cuda", dtype=torch.int32).view(1, 50, 1)
    freq = 100.0 ** (-torch.arange(p, device="cuda", dtype=torch.float32) / p)
    want = reference(q, pos, freq, [p], False, False)
    q0 = q.clone()
    assert tracea_gpu.rotary(q, k, pos, freq, q_out=q, k_out=k)[0] is q
    within(q, want, torch.float32)
    assert torch.equal(q[..., 2 * p:], q0[..., 2 * p:])
    tracea_gpu.rotary(q, k, pos, freq, inverse=True, q_out=q, k_out=k)
    assert (q - q0).abs().max() <= 4 * 2.0 ** -20 * q0.abs().max()
    # the gradient of a rotation is the rotation back: <turn(x), y> = <x, back(y)>
    x, y = make((1, 2, 50, d), torch.float32, "bhsd", 4), make((1, 2, 50, d), torch.float32, "bhsd", 5)
    a = (tracea_gpu.rotary(x, None, pos, freq)[0].double() * y.double()).sum()
    b = (x.double() * tracea_gpu.rotary(y, None, pos, freq, inverse=True)[0].double()).sum()
    assert abs(a - b) <= 2.0 ** -20 * (x.double().abs() * y.double().abs()).sum() * 4


def test_nothing_to_turn(tracea_gpu):
    q = torch.randn(2, 0, 5, 64, device="cuda")
    pos, freq = torch.zeros(1, 5, 1, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    assert tracea_gpu.rotary(q, None, pos, freq)[0].shape == q.shape
    q = torch.randn(2, 2, 0, 64, device="cuda")
    assert tracea_gpu.rotary(q, None, pos[:, :0], freq)[0].shape == q.shape
    q = torch.randn(2, 2, 5, 64, device="cuda")  # no pairs: a copy
    assert torch.equal(tracea_gpu.rotary(q, None, pos, freq[:0], sections=[0])[0], q)


def test_refusals(tracea_gpu):
    from tracea_amd import capi
    q = torch.randn(2, 4, 5, 64, device="cuda")
    pos, freq = torch.zeros(1, 5, 2, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")

    def refused(status, *args, **kw):
        with pytest.raises(capi.TraceaError) as e:
            tracea_gpu.rotary(*args, **kw)
        assert e.value.status == status, e.value
    refused(capi.INVALID_PARAMS, q, None, pos, freq)                                # two axes, one section
    refused(capi.INVALID_PARAMS, q, None, pos, freq, sections=[16, 15])
    refused(capi.INVALID_PARAMS, q, None, pos, torch.ones(33, device="cuda"), sections=[16, 17])
    refused(capi.INVALID_PARAMS, q, None, pos[:, :4], freq, sections=[16, 16])
    refused(capi.INVALID_PARAMS, q, None, pos.float(), freq, sections=[16, 16])
    refused(capi.INVALID_PARAMS, q, None, pos, freq.half(), sections=[16, 16])
    refused(capi.INVALID_PARAMS, q, q[:1], pos, freq, sections=[16, 16])
    refused(capi.UNSUPPORTED_CONFIG, q, q.half(), pos, freq, sections=[16, 16])
    refused(capi.UNSUPPORTED_CONFIG, q.transpose(2, 3).contiguous().transpose(2, 3), None, pos, freq, sections=[16, 16])
    refused(capi.CPU_ERROR, q.cpu(), None, pos, freq, sections=[16, 16])
    refused(capi.INVALID_PARAMS, q, None, pos.cpu(), freq, sections=[16, 16])
    refused(capi.INVALID_PARAMS, q[:, :2], None, pos, freq, sections=[16, 16], q_out=q[:, 1:3])   # over its operand in part
    refused(capi.INVALID_PARAMS, q, q, pos, freq, sections=[16, 16], q_out=q)                     # q is also k's operand
    with pytest.raises(ValueError):
        tracea_gpu.rotary(q, None, pos, freq, sections=[8] * 5)
