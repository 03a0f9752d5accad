"""Norms of heads with rotary positions, and their gradients, against the formulas in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
from cache_oracle import U32, angles, half_step, heads, rotated  # noqa: E402

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6


def setup(seed, b, hq, hk, s, d, rot, sections, dtype, layout, far=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = heads(g, b, hq, s, d, dtype, layout, 3.0), heads(g, b, hk, s, d, dtype, layout, 0.3)
    wq, wk = (1 + 0.3 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(far, far + 5000, (b, s, len(sections)), device="cuda", generator=g, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float32) / max(rot // 2, 1))
    return g, q, k, wq, wk, pos, freq


def normed(x, w):
    x = x.double()
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()


def check_forward(out, x, w, pos, freq, rot, sections, adjacent):
    y, made_of = rotated(normed(x, w), angles(pos, freq, sections) if rot else None, rot, adjacent)
    # the sum of squares is off by up to 22 roundings and its root by half of them, the angle and its sine by 4, the products by 6
    off = (out.double() - y).abs()
    assert (off <= half_step(out.dtype) * y.abs() * (1 + 1e-6) + 32 * U32 * made_of + (2.0 ** -25 if out.dtype == torch.float16 else 0)).all()


CASES = [  # b, hq, hk, s, d, rot, sections, adjacent, layout
    (1, 1, 1, 1, 8, 0, [], False, "bhsd"), (2, 4, 2, 1, 128, 128, [64], False, "bshd"), (2, 6, 3, 37, 64, 48, [8, 16], True, "bhsd"),
    (3, 5, 1, 19, 96, 96, [16, 0, 32], False, "bshd"), (1, 12, 12, 197, 64, 64, [32], True, "bshd"), (2, 3, 2, 33, 80, 40, [20], False, "bhsd"),
    (2, 2, 1, 11, 40, 40, [20], True, "bhsd"), (1, 3, 2, 50, 128, 64, [32], False, "odd"), (1, 2, 2, 9, 33, 20, [5, 5], True, "odd"),
    (1, 2, 1, 21, 512, 256, [128], False, "bshd"), (1, 2, 1, 5, 511, 511 // 2 * 2, [255], False, "bhsd"), (1, 1, 1, 3, 1, 0, [], False, "bhsd"),
    (1, 4, 4, 700, 256, 256, [128], True, "bshd"),
    # pairs in fours and twos
    (2, 3, 1, 17, 40, 20, [10], False, "bshd"), (1, 3, 1, 70, 40, 20, [4, 6], True, "bhsd"), (2, 2, 2, 9, 88, 24, [12], True, "bhsd"),
    (2, 2, 2, 9, 88, 24, [12], False, "bshd"), (1, 2, 1, 9, 12, 4, [2], False, "bhsd"), (1, 40, 8, 300, 80, 40, [20], True, "bshd")]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(tracea_gpu, case, dtype):
    b, hq, hk, s, d, rot, sections, adjacent, layout = case
    _, q, k, wq, wk, pos, freq = setup(3, b, hq, hk, s, d, rot, sections, dtype, layout)
    turn = dict(positions=pos, inv_freq=freq, sections=sections) if rot else {}
    qo, ko = tracea_gpu.qk_norm_rotary(q, k, wq, wk, adjacent=adjacent, eps=EPS, **turn)
    check_forward(qo, q, wq, pos, freq, rot, sections, adjacent)
    check_forward(ko, k, wk, pos, freq, rot, sections, adjacent)
    # in place, queries alone, without weights, one set of positions for the batch
    q2 = q.clone() if layout != "odd" else q
    want, none = tracea_gpu.qk_norm_rotary(q2, None, adjacent=adjacent, eps=EPS, **(dict(turn, positions=pos[:1]) if rot else {}))
    assert none is None
    check_forward(want, q2, torch.ones_like(wq), pos[:1], freq, rot, sections, adjacent)
    got, _ = tracea_gpu.qk_norm_rotary(q2, None, adjacent=adjacent, eps=EPS, q_out=q2, **(dict(turn, positions=pos[:1]) if rot else {}))
    assert got.data_ptr() == q2.data_ptr() and torch.equal(got, want)


def exact_backward(dy, x, w, angle, rot, adjacent):
    x, w = x.double().requires_grad_(True), w.double().requires_grad_(True)
    dn, made_of = rotated(dy, angle, rot, adjacent, -1.0)
    r = 1 / torch.sqrt(x.detach().square().mean(-1, keepdim=True) + EPS)
    dx, dw = torch.autograd.grad(x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w, (x, w), dn)
    xn, g = (x.detach() * r).abs(), made_of * w.detach().abs()
    dx_made_of = r * (g + xn * (g * xn).mean(-1, keepdim=True))
    return dx, dw, dx_made_of, (made_of * xn).sum((0, 1, 2))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward(tracea_gpu, case, dtype):
    b, hq, hk, s, d, rot, sections, adjacent, layout = case
    g, q, k, wq, wk, pos, freq = setup(4, b, hq, hk, s, d, rot, sections, dtype, layout)
    dqo, dko = heads(g, b, hq, s, d, dtype, layout), heads(g, b, hk, s, d, dtype, layout)
    turn = dict(positions=pos, inv_freq=freq, sections=sections) if rot else {}
    got = tracea_gpu.qk_norm_rotary_backward(dqo, dko, q, k, wq, wk, adjacent=adjacent, eps=EPS, **turn)
    angle = angles(pos, freq, sections) if rot else None
    for i, (dy, x, w) in enumerate(((dqo, q, wq), (dko, k, wk))):
        dx, dw, dx_of, dw_of = exact_backward(dy, x, w, angle, rot, adjacent)
        # as forward, both sums of a row and twice as many products; D = 1 cancels to nothing, of what it is made of
        assert ((got[i].double() - dx).abs() <= half_step(dtype) * dx.abs() * (1 + 1e-6) + 80 * U32 * dx_of + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
        # a column's terms are summed in chains of at most 400 here: rows of a lane group, groups, workgroups
        assert ((got[2 + i].double() - dw).abs() <= 480 * U32 * dw_of).all()
    again = tracea_gpu.qk_norm_rotary_backward(dqo, dko, q, k, wq, wk, adjacent=adjacent, eps=EPS, **turn)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    # over the operands, queries alone, without weights
    want = tracea_gpu.qk_norm_rotary_backward(dqo, None, q, None, adjacent=adjacent, eps=EPS, **turn)
    assert want[1:] == (None, None, None)
    for over in ("q", "dqo"):
        q2, dqo2 = (q.clone(), dqo.clone()) if layout != "odd" else (q, dqo)
        if layout == "odd" and over == "dqo":
            break
        r = tracea_gpu.qk_norm_rotary_backward(dqo2, None, q2, None, adjacent=adjacent, eps=EPS, dq=q2 if over == "q" else dqo2, **turn)
        assert torch.equal(r[0], want[0])


def test_gradients_are_those_of_differences(tracea_gpu):
    """A direction in x and in w, by central differences of the operator's own forward pass in fp32."""
    g, q, k, wq, wk, pos, freq = setup(5, 2, 4, 2, 17, 64, 64, [20, 12], torch.float32, "bhsd")
    dq, dk = heads(g, 2, 4, 17, 64, torch.float32), heads(g, 2, 2, 17, 64, torch.float32)
    turn = dict(positions=pos, inv_freq=freq, sections=[20, 12], eps=EPS)
    got = tracea_gpu.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, **turn)
    step = 2.0 ** -7
    for i in range(4):
        base = [q, k, wq, wk]
        direction = torch.randn(base[i].shape, device="cuda", generator=g)
        ends = []
        for sign in (1, -1):
            at = [t + sign * step * direction if j == i else t for j, t in enumerate(base)]
            a, b = tracea_gpu.qk_norm_rotary(*at, **turn)
            ends.append((a.double() * dq.double()).sum() + (b.double() * dk.double()).sum())
        slope = (got[i].double() * direction.double()).sum()
        # truncation: step^2 / 6 times a third derivative that is a few tens of the first; k has entries of 0.3
        scale = (got[i].double().abs() * direction.double().abs()).sum()
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 2e-2 * scale


def test_far_positions(tracea_gpu):
    _, q, k, wq, wk, pos, freq = setup(6, 1, 2, 1, 40, 64, 64, [32], torch.float32, "bhsd", far=2 ** 31 - 6000)
    qo, _ = tracea_gpu.qk_norm_rotary(q, k, wq, wk, pos, freq, eps=EPS)
    check_forward(qo, q, wq, pos, freq, 64, [32], False)


def test_no_rows(tracea_gpu):
    q, w = torch.zeros(2, 3, 0, 64, device="cuda"), torch.ones(64, device="cuda")
    assert tracea_gpu.qk_norm_rotary(q, None, w)[0].shape == q.shape
    dq, _, dw, _ = tracea_gpu.qk_norm_rotary_backward(q, None, q, None, w)
    assert dq.shape == q.shape and (dw == 0).all()
    k = torch.randn(2, 1, 0, 64, device="cuda")
    assert (tracea_gpu.qk_norm_rotary_backward(q, k, q, k, w, w)[3] == 0).all()


def test_zeros_and_infinities(tracea_gpu):
    q = torch.randn(1, 2, 5, 64, device="cuda").bfloat16()
    q[0, 0, 1] = 0
    q[0, 0, 2, 7] = float("inf")
    q[0, 1, 3, 9] = float("nan")
    want, _ = tracea_gpu.qk_norm_rotary(torch.nan_to_num(q, 1.0, 1.0), None)
    got, _ = tracea_gpu.qk_norm_rotary(q, None)
    assert (got[0, 0, 1] == 0).all() and torch.isnan(got[0, 0, 2, 7]) and torch.isnan(got[0, 1, 3]).all()
    for h, s in ((0, 0), (0, 3), (1, 0), (1, 2), (1, 4)):  # other rows do not see it
        assert torch.equal(got[0, h, s], want[0, h, s])


def test_graph_and_other_stream(tracea_gpu):
    g, q, k, wq, wk, pos, freq = setup(7, 2, 8, 2, 64, 128, 128, [64], torch.bfloat16, "bshd")
    dq, dk = heads(g, 2, 8, 64, 128, torch.bfloat16), heads(g, 2, 2, 64, 128, torch.bfloat16)
    turn = dict(positions=pos, inv_freq=freq, eps=EPS)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tracea_gpu.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, **turn)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = tracea_gpu.qk_norm_rotary(q, k, wq, wk, **turn) + tracea_gpu.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, **turn)
        for i in range(3):
            q.normal_(generator=g)
            dk.normal_(generator=g)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            want = tracea_gpu.qk_norm_rotary(q, k, wq, wk, **turn) + tracea_gpu.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, **turn)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
