"""tracea_attention_forward and tracea_attention_backward against the formulas in 64 bits.

Error bounds are worked out next to the reference, per element, from where the kernels round: with u the unit roundoff
of the operand type (2^-8 bf16, 2^-11 f16), results are rounded once (u |x|), probabilities and dS once before
they enter a matrix product (u times the product of the magnitudes), o once before delta is taken from it; scores,
statistics and sums are fp32, for which 2^-17 of the magnitudes is allowed (128 products and up to some hundred exponents
of a few units)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -17


def visible(b, sq, sk, causal, lq, lk):
    i, j = torch.arange(sq)[None, :, None], torch.arange(sk)[None, None]
    lq = torch.full((b,), sq) if lq is None else lq.cpu().long().clamp(0, sq)
    lk = torch.full((b,), sk) if lk is None else lk.cpu().long().clamp(0, sk)
    lq, lk = lq.view(-1, 1, 1), lk.view(-1, 1, 1)
    seen = (i < lq) & (j < lk)
    return (seen & (j <= i + lk - lq)) if causal else seen


def reference(q, k, v, do, causal, scale, lq=None, lk=None):
    """o, lse, dq, dk, dv in 64 bits, each with the bound of its error."""
    u = U[q.dtype]
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    seen = visible(b, sq, sk, causal, lq, lk)[:, None]
    rep = lambda t: t.cpu().double().repeat_interleave(hq // hk, dim=1)  # noqa: E731
    qd, kd, vd, dod = q.cpu().double(), rep(k), rep(v), do.cpu().double()
    rows = seen.any(-1)          # what nobody sees or is nobody's may hold anything
    cols = seen.any(-2)
    qd, dod = (torch.where(rows[..., None], t, torch.zeros(())) for t in (qd, dod))
    kd, vd = (torch.where(cols[..., None], t, torch.zeros(())) for t in (kd, vd))
    scale = scale or 1.0 / math.sqrt(d)
    s = torch.where(seen, scale * qd @ kd.transpose(-1, -2), torch.tensor(-math.inf))
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, (s - torch.where(lse > -math.inf, lse, torch.zeros(()))[..., None]).exp(), torch.zeros(()))
    o = p @ vd
    dp = dod @ vd.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # per score: fp32 error relative to the magnitudes that went into it
    s_mag = abs(scale) * qd.abs() @ kd.abs().transpose(-1, -2) + torch.where(lse > -math.inf, lse.abs(), torch.zeros(()))[..., None] + 1
    p_err = p * F32 * s_mag
    dp_mag = dod.abs() @ vd.abs().transpose(-1, -2)
    one = (seen.sum(-1, keepdim=True) == 1)  # a row with one key: P = 1, dS = 0 exactly
    o_err = u * o.abs() + (u * p + p_err) @ vd.abs()
    delta_err = (dod.abs() * o_err).sum(-1, keepdim=True) + F32 * (dod.abs() * o.abs()).sum(-1, keepdim=True)
    ds_err = u * ds.abs() + p * (delta_err + F32 * dp_mag) + p_err * (dp - delta).abs()
    if q.dtype == torch.float16:  # below the smallest normal operand
        big = 2 * dod.norm(dim=-1).amax() * vd.norm(dim=-1).amax()
        ds_err = ds_err + torch.where(seen, big * 2.0 ** -37, torch.zeros((), dtype=torch.float64))
    ds_err = torch.where(one, torch.zeros((), dtype=torch.float64), ds_err)
    fold = lambda t: t.reshape(b, hk, hq // hk, sk, d).sum(2)  # noqa: E731
    dq, dk, dv = scale * ds @ kd, fold(scale * ds.transpose(-1, -2) @ qd), fold(p.transpose(-1, -2) @ dod)
    tiny = 2.0 ** -25  # half a step of the smallest f16
    e_dq = u * dq.abs() + abs(scale) * ds_err @ kd.abs() + F32 * abs(scale) * ds.abs() @ kd.abs() + tiny
    e_dk = u * dk.abs() + fold(abs(scale) * (ds_err + F32 * ds.abs()).transpose(-1, -2) @ qd.abs()) + tiny
    e_dv = u * dv.abs() + fold(((u + F32) * p + p_err).transpose(-1, -2) @ dod.abs()) + tiny
    e_lse = F32 * (1 + s_mag.amax(-1)) / 4
    return {"o": (o, o_err + tiny), "lse": (lse, e_lse), "dq": (dq, e_dq), "dk": (dk, e_dk), "dv": (dv, e_dv)}


def within(name, got, want):
    ref, err = want
    got = got.double().cpu()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin), name + ": not finite in other places than the reference"
    assert torch.equal(got[~fin], ref[~fin]), name
    worst = ((got - ref).abs() - 1.02 * err)[fin]
    assert worst.numel() == 0 or worst.max() <= 0, "%s: %.3g beyond the bound" % (name, worst.max())


def heads(shape, layout, dtype, gen, scale=1.0):
    b, h, n, d = shape
    if layout == "bhsd":
        return (torch.randn(b, h, n, d, device="cuda", generator=gen) * scale).to(dtype)
    if layout == "bshd":
        return (torch.randn(b, n, h, d, device="cuda", generator=gen) * scale).to(dtype).transpose(1, 2)
    if layout == "pitch":  # rows wider than the head, in a larger buffer
        return (torch.randn(b, h, n, d + 24, device="cuda", generator=gen) * scale).to(dtype)[..., 8:8 + d]
    if layout == "odd":  # bases and rows on any element: the copies' road
        return (torch.randn(b, h, n, d + 3, device="cuda", generator=gen) * scale).to(dtype)[..., 1:1 + d]
    raise ValueError(layout)


def check(ops, b, hq, hk, sq, sk, d, dtype=torch.bfloat16, causal=False, layout="bhsd", scale=0.0, lq=None, lk=None, spoil=False,
          q_scale=1.0, do_scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = heads((b, hq, sq, d), layout, dtype, g, q_scale)
    k, v = heads((b, hk, sk, d), layout, dtype, g), heads((b, hk, sk, d), layout, dtype, g)
    do = heads((b, hq, sq, d), layout, dtype, g, do_scale)
    lq = None if lq is None else torch.tensor(lq, dtype=torch.int32, device="cuda")
    lk = None if lk is None else torch.tensor(lk, dtype=torch.int32, device="cuda")
    want = reference(q, k, v, do, causal, scale, lq, lk)
    if spoil:  # what lies behind the lengths
        for i in range(b):
            for t, n in ((q, lq), (do, lq), (k, lk), (v, lk)):
                if n is not None:
                    t[i, :, max(0, int(n[i])):] = float("nan") if i % 2 else float("inf")
    kw = dict(causal=causal, scale=scale, q_lengths=lq, k_lengths=lk)
    o, lse = ops.attention_forward(q, k, v, **kw)
    within("o", o, want["o"])
    within("lse", lse, want["lse"])
    dq, dk, dv = ops.attention_backward(q, k, v, o, lse, do, **kw)
    for name, t in (("dv", dv), ("dk", dk), ("dq", dq)):
        within(name, t, want[name])
    again = ops.attention_backward(q, k, v, o, lse, do, **kw)
    for x, y in zip((dq, dk, dv), again):
        assert torch.equal(x, y), "two calls on the same inputs differ"
    return q, k, v, do, o, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("causal", [False, True], ids=["dense", "causal"])
def test_head_dimensions(tracea_gpu, d, dtype, causal):
    check(tracea_gpu, 2, 4, 2, 150, 150, d, dtype, causal)


@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 64), (1, 500), (2, 3), (3, 2), (63, 64), (64, 65), (65, 63), (128, 128), (129, 257),
                                   (300, 40), (40, 300), (257, 1), (31, 1000)])
@pytest.mark.parametrize("causal", [False, True], ids=["dense", "causal"])
def test_lengths(tracea_gpu, sq, sk, causal):
    # more queries than keys under a causal mask: the first sq - sk rows see nothing
    check(tracea_gpu, 2, 3, 3, sq, sk, 64, torch.bfloat16, causal)
    check(tracea_gpu, 1, 2, 2, sq, sk, 128, torch.float16, causal)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (8, 2), (6, 2), (7, 1), (10, 2), (64, 1)])
@pytest.mark.parametrize("causal", [False, True], ids=["dense", "causal"])
def test_shared_heads(tracea_gpu, hq, hk, causal):
    check(tracea_gpu, 2, hq, hk, 70, 90, 64, torch.bfloat16, causal)
    check(tracea_gpu, 1, hq, hk, 33, 33, 128, torch.bfloat16, causal)


@pytest.mark.parametrize("layout", ["bshd", "pitch", "odd"])
@pytest.mark.parametrize("d", [64, 96, 50, 33, 1])
def test_strides(tracea_gpu, layout, d):
    check(tracea_gpu, 2, 6, 3, 77, 77, d, torch.bfloat16, True, layout)
    check(tracea_gpu, 2, 2, 2, 20, 130, d, torch.float16, False, layout)


@pytest.mark.parametrize("causal", [False, True], ids=["dense", "causal"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_padded_batches(tracea_gpu, causal, dtype):
    # lengths of zero and one, lengths beyond the tensors, and rubbish behind every length
    n = [0, 1, 65, 130, 200, 64, 128]
    check(tracea_gpu, 7, 4, 2, 130, 130, 64, dtype, causal, lq=n, lk=n, spoil=True)
    check(tracea_gpu, 4, 4, 4, 100, 140, 128, dtype, causal, lk=[140, 0, 1, 77], spoil=True)
    check(tracea_gpu, 4, 2, 1, 100, 140, 96, dtype, causal, lq=[0, 1, 99, 100], spoil=True)
    check(tracea_gpu, 3, 8, 2, 1, 700, 128, dtype, causal, lk=[700, 0, 333], spoil=True)


def test_no_keys_and_no_queries(tracea_gpu):
    q, k = torch.randn(2, 2, 5, 64, device="cuda").half(), torch.empty(2, 2, 0, 64, device="cuda").half()
    o, lse = tracea_gpu.attention_forward(q, k, k)
    assert (o == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = tracea_gpu.attention_backward(q, k, k, o, lse, q)
    assert (dq == 0).all() and dk.shape == k.shape
    o, lse = tracea_gpu.attention_forward(k, q, q)
    assert o.shape == k.shape
    dq, dk, dv = tracea_gpu.attention_backward(k, q, q, o, lse, k, dk=torch.full_like(q, 7), dv=torch.full_like(q, 7))
    assert (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("scale", [1.0, -0.2, 0.01])
def test_scales(tracea_gpu, scale):
    check(tracea_gpu, 1, 2, 2, 100, 100, 64, torch.bfloat16, False, scale=scale, q_scale=0.5)
    check(tracea_gpu, 1, 2, 1, 100, 100, 128, torch.float16, True, scale=scale, q_scale=0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_scores_far_from_zero(tracea_gpu, dtype):
    # scores of some tens: peaked rows, reference maxima that move from tile to tile
    check(tracea_gpu, 1, 2, 2, 200, 300, 64, dtype, False, q_scale=10.0)
    check(tracea_gpu, 1, 2, 2, 200, 300, 128, dtype, True, q_scale=10.0)


@pytest.mark.parametrize("do_scale", [1e-4, 1.0, 200.0])
def test_gradients_of_any_size_in_f16(tracea_gpu, do_scale):
    # operands of the second products leave f16's range on either side unless they are scaled
    check(tracea_gpu, 1, 2, 2, 64, 1500, 64, torch.float16, False, do_scale=do_scale)
    check(tracea_gpu, 1, 2, 1, 130, 130, 128, torch.float16, True, do_scale=do_scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_a_row_that_sees_one_key_has_no_gradient(tracea_gpu, dtype):
    _, _, _, _, _, _, dq, dk, _ = check(tracea_gpu, 2, 4, 4, 33, 1, 64, dtype)
    assert (dq == 0).all() and (dk == 0).all()
    dq = check(tracea_gpu, 1, 4, 2, 70, 70, 128, dtype, True)[6]
    assert (dq[:, :, 0] == 0).all()


@pytest.mark.parametrize("b,hq,hk,sq,sk,d", [(1, 2, 2, 1, 5000, 128), (2, 8, 2, 3, 4100, 64), (1, 16, 1, 1, 3000, 96)])
def test_few_rows_over_many_keys(tracea_gpu, b, hq, hk, sq, sk, d):
    check(tracea_gpu, b, hq, hk, sq, sk, d, torch.bfloat16, True)
    check(tracea_gpu, b, hq, hk, sq, sk, d, torch.float16, False, lk=[sk - 100 * i for i in range(b)], spoil=True)


def test_gradients_against_differences(tracea_gpu):
    """d/dt of sum(o * do) along a direction, in 64 bits around the 16-bit operands, equals the gradients' product with it."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, do = (heads((1, 2, 40, 64), "bhsd", torch.bfloat16, g) for _ in range(4))
    o, lse = tracea_gpu.attention_forward(q, k, v, causal=True)
    grads = tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True)

    def loss(q, k, v):
        s = (q @ k.transpose(-1, -2)) / 8.0
        s = s.masked_fill(~visible(1, 40, 40, True, None, None)[:, None], -math.inf)
        return (torch.softmax(s, -1) @ v * do.cpu().double()).sum()
    base = [t.cpu().double() for t in (q, k, v)]
    want = reference(q, k, v, do, True, 0.0)
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(q.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        at = lambda t: [x + t * way if j == i else x for j, x in enumerate(base)]  # noqa: E731
        slope = (loss(*at(1e-5)) - loss(*at(-1e-5))) / 2e-5
        got = (grads[i].cpu().double() * way).sum()
        assert abs(got - slope) <= (want[name][1] * way.abs()).sum() + 1e-6 * abs(slope)


def test_results_over_operands_and_in_packed_rows(tracea_gpu):
    """dq, dk, dv side by side in one [B,S,3,H,D] buffer, and o over q."""
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(2, 50, 3, 4, 64, device="cuda", generator=g).bfloat16()
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    do = heads((2, 4, 50, 64), "bshd", torch.bfloat16, g)
    want = reference(q, k, v, do, True, 0.0)
    o, lse = tracea_gpu.attention_forward(q, k, v, causal=True)
    grad = torch.zeros_like(qkv)
    tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True, **{n: grad[:, :, i].transpose(1, 2) for i, n in enumerate(("dq", "dk", "dv"))})
    for i, n in enumerate(("dq", "dk", "dv")):
        within(n, grad[:, :, i].transpose(1, 2), want[n])
    own = q.clone()
    tracea_gpu.attention_forward(own, k, v, causal=True, out=own)
    within("o", own, want["o"])


def test_streams_and_graphs(tracea_gpu):
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v, do = (heads((2, 4, 150, 64), "bhsd", torch.float16, g) for _ in range(4))
    want = reference(q, k, v, do, True, 0.0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out = [torch.empty_like(q) for _ in range(4)] + [torch.empty(2, 4, 150, device="cuda")]

    def step():
        tracea_gpu.attention_forward(q, k, v, causal=True, out=out[0], lse=out[4])
        tracea_gpu.attention_backward(q, k, v, out[0], out[4], do, causal=True, dq=out[1], dk=out[2], dv=out[3])
    with torch.cuda.stream(stream):
        step()  # (its workspace is there from here on)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(3):
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for t, n in zip(out, ("o", "dq", "dk", "dv", "lse")):
                within(n, t, want[n])
            tracea_gpu.attention_forward(k, q, v)  # eager work of another shape in between
            torch.cuda.synchronize()


def test_refusals(tracea_gpu):
    from tracea_amd import capi
    q = torch.randn(2, 4, 10, 64, device="cuda").half()
    k = torch.randn(2, 2, 12, 64, device="cuda").half()
    lse = torch.zeros(2, 4, 10, device="cuda")
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    fwd, bwd = tracea_gpu.attention_forward, tracea_gpu.attention_backward

    def refused(status, call, *args, **kw):
        with pytest.raises(capi.TraceaError) as e:
            call(*args, **kw)
        assert e.value.status == status, e.value
    refused(capi.UNSUPPORTED_CONFIG, fwd, q.float(), k.float(), k.float())
    refused(capi.UNSUPPORTED_CONFIG, fwd, q, k.bfloat16(), k)
    refused(capi.INVALID_PARAMS, fwd, q, k[:, :, :5], k)
    refused(capi.INVALID_PARAMS, fwd, q[:, :3], k, k)                   # 3 heads over 2
    refused(capi.INVALID_PARAMS, fwd, q[:1], k, k)
    refused(capi.INVALID_PARAMS, fwd, q[..., :32], k, k)
    refused(capi.INVALID_PARAMS, fwd, q[0], k, k)                       # rank
    refused(capi.CPU_ERROR, fwd, q.cpu(), k.cpu(), k.cpu())
    refused(capi.INVALID_PARAMS, fwd, q, k.cpu(), k)
    refused(capi.INVALID_PARAMS, fwd, q, k, k, k_lengths=n.long().int().cpu())
    refused(capi.INVALID_PARAMS, fwd, q, k, k, k_lengths=n[:1])
    refused(capi.INVALID_PARAMS, fwd, q, k, k, q_lengths=lse[0, 0, :2])  # not i32
    refused(capi.INVALID_PARAMS, fwd, q, k, k, scale=float("inf"))
    refused(capi.INVALID_PARAMS, fwd, q, k, k, lse=lse.half())
    refused(capi.INVALID_PARAMS, fwd, q, k, k, lse=lse[:, :, :9])
    refused(capi.INVALID_PARAMS, fwd, q, k, k, out=torch.empty(2, 1, 10, 64, device="cuda").half().expand(2, 4, 10, 64))
    wide = torch.randn(1, 1, 4, 129, device="cuda").half()
    refused(capi.UNSUPPORTED_CONFIG, fwd, wide, wide, wide)
    refused(capi.INVALID_PARAMS, bwd, q, k, k, q, lse, q[:, :, :9])
    refused(capi.INVALID_PARAMS, bwd, q, k, k, q, lse[:1], q)
    both = torch.empty_like(k)
    refused(capi.INVALID_PARAMS, bwd, q, k, k, q, lse, q, dk=both, dv=both)
    with pytest.raises(TypeError):
        fwd(q.long(), k, k)


def test_the_road_a_call_takes(tracea_gpu):
    """Launches of a call: the forward pass alone, or with the join of a split key axis; backward the row statistics and the gradients,
    or with the sums of dK and dV from parts of the rows.  Either road against the formulas."""
    from helpers import launches
    for b, hq, hk, sq, sk, d, fwd, bwd in ((1, 2, 1, 1, 4000, 128, 2, 2), (1, 12, 12, 256, 256, 64, 1, 2), (1, 16, 1, 500, 500, 64, 1, 3),
                                           (1, 20, 1, 300, 300, 128, 1, 3)):
        q, k, v, do, o, lse, dq, dk, dv = check(tracea_gpu, b, hq, hk, sq, sk, d)
        assert launches(lambda: tracea_gpu.attention_forward(q, k, v, out=o, lse=lse)) == fwd, (hq, hk, sq, sk, d)
        assert launches(lambda: tracea_gpu.attention_backward(q, k, v, o, lse, do, dq=dq, dk=dk, dv=dv)) == bwd, (hq, hk, sq, sk, d)
