"""tracea_norm_gate_residual and its backward pass against the formulas in 64 bits.

Bounds: a result's rounding (u |x|) and, for the fp32 arithmetic, 2^-19 of the magnitudes that are added up in it (sums over up to
8192 channels, each thread's in order, then across threads: errors of some ten roundings); column sums 2^-16 of the
magnitudes they add (up to a thousand rows in order)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F, COL = 2.0 ** -19, 2.0 ** -16


def rms(t, eps):
    return torch.rsqrt((t * t).mean(-1, keepdim=True) + eps)


def forward64(x, h, w_post, gate, w_pre, scale, eps):
    """{name: (value, magnitude of its terms)}"""
    out = {}
    x = x.cpu().double()
    mag = x.abs()
    if h is not None:
        h = h.cpu().double()
        n = h * rms(h, eps) * w_post.cpu().double()
        if gate is not None:
            n = n * gate.cpu().double()[:, None]
        x, mag = scale * x + n, abs(scale) * x.abs() + n.abs()
        out["x_out"] = (x, mag)
    if w_pre is not None:
        r = rms(x, eps)
        w = w_pre.cpu().double()
        # (an error of x shows in y directly and through the norm)
        out["y"] = (x * r * w, (mag + x.abs() * ((x.abs() * mag).mean(-1, keepdim=True) * r * r)) * r * w.abs() * 2)
    return out


def backward64(dx_out, dy, x, h, w_post, gate, w_pre, scale, eps):
    out = {}
    x = x.cpu().double()
    dt = torch.zeros_like(x) if dx_out is None else dx_out.cpu().double()
    mag = dt.abs()
    if dy is not None:
        dy, w = dy.cpu().double(), w_pre.cpu().double()
        r = rms(x, eps)
        xn, g = x * r, dy * w
        through = r * (g - xn * (g * xn).mean(-1, keepdim=True))
        mag = mag + r * (g.abs() + xn.abs() * (g * xn).abs().mean(-1, keepdim=True))
        dt = dt + through
        out["dw_pre"] = ((dy * xn).sum((0, 1)), (dy * xn).abs().sum((0, 1)))
    out["dx"] = (dt, mag) if h is None else (scale * dt, abs(scale) * mag)
    if h is not None:
        h, w = h.cpu().double(), w_post.cpu().double()
        gt = torch.ones(1, 1, x.shape[-1], dtype=torch.float64) if gate is None else gate.cpu().double()[:, None]
        r = rms(h, eps)
        hn, a, am = h * r, dt * gt * w, mag * gt.abs() * w.abs()
        out["dh"] = (r * (a - hn * (a * hn).mean(-1, keepdim=True)), r * (am + hn.abs() * (am * hn.abs()).mean(-1, keepdim=True)))
        each, em = dt * hn, mag * hn.abs()
        out["dw_post"] = ((each * gt).sum((0, 1)), (em * gt.abs()).sum((0, 1)))
        if gate is not None:
            by, bm = (each.sum(1) * w, em.sum(1) * w.abs())
            out["dgate"] = (by, bm) if gate.shape[0] == x.shape[0] else (by.sum(0, keepdim=True), bm.sum(0, keepdim=True))
    return out


def within(name, got, want, u, f):
    ref, mag = want
    far = (got.cpu().double() - ref).abs() - (1.01 * u * ref.abs() + f * mag + 2.0 ** -25 * (u == 2.0 ** -11))
    assert torch.isfinite(got).all() and far.max() <= 0, "%s: %.3g beyond the bound" % (name, far.max())


def make(b, t, c, dtype, gates, layout="plain", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(scale=1.0):
        x = (torch.randn(b, t, c + (layout != "plain") * 5, device="cuda", generator=g) * scale).to(dtype)
        return x if layout == "plain" else x[..., 3:3 + c]
    vec = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return dict(x=rows(2.0), h=rows(0.3), dx=rows(), dy=rows(), w_post=1 + 0.1 * vec(c), w_pre=1 + 0.1 * vec(c),
                gate=None if gates is None else vec(b if gates == "each" else 1, c))


def check(ops, b, t, c, dtype, gates="each", layout="plain", scale=1.0, eps=1e-6, post=True, pre=True, dx_out=True):
    m = make(b, t, c, dtype, gates if post else None, layout)
    u = U[dtype]
    fkw = dict(residual_scale=scale, eps=eps)
    w = dict(w_post=m["w_post"] if post else None, gate=m["gate"], w_pre=m["w_pre"] if pre else None)
    h = m["h"] if post else None
    want = forward64(m["x"], h, w["w_post"], w["gate"], w["w_pre"], scale, eps)
    x_out, y = ops.norm_gate_residual(m["x"], h, **w, **fkw)
    if post:
        within("x_out", x_out, want["x_out"], u, F)
    else:
        assert x_out is m["x"]
    if pre:
        within("y", y, want["y"], u, F)
    else:
        assert y is None
    dx, dy = m["dx"] if dx_out else None, m["dy"] if pre else None
    want = backward64(dx, dy, x_out, h, w["w_post"], w["gate"], w["w_pre"], scale, eps)
    names = ("dx", "dh", "dw_post", "dgate", "dw_pre")
    got = dict(zip(names, ops.norm_gate_residual_backward(dx, dy, x_out, h, **w, **fkw)))
    for n in names:
        assert (got[n] is None) == (n not in want), n
        if n in want:
            whole = n in ("dx", "dh")
            within(n, got[n], want[n], u if whole else 2.0 ** -24, F if whole else COL)
    again = dict(zip(names, ops.norm_gate_residual_backward(dx, dy, x_out, h, **w, **fkw)))
    for n in want:
        assert torch.equal(got[n], again[n]), n + ": two calls on the same inputs differ"


@pytest.mark.parametrize("dtype", list(U), ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", [1, 3, 8, 31, 64, 100, 256, 257, 264, 512, 768, 1000, 1001, 1152, 2048, 4096, 5000, 8192])
def test_widths_and_types(tracea_gpu, c, dtype):
    check(tracea_gpu, 2, 7, c, dtype)


@pytest.mark.parametrize("b,t", [(1, 1), (1, 2), (16, 1), (3, 333), (1, 5000), (300, 2), (5, 129)])
@pytest.mark.parametrize("c", [64, 768])
def test_rows(tracea_gpu, b, t, c):
    check(tracea_gpu, b, t, c, torch.bfloat16, "each")
    check(tracea_gpu, b, t, c, torch.float32, "one")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("c", [72, 640])
@pytest.mark.parametrize("kw", [dict(gates=None), dict(gates="one"), dict(scale=0.5), dict(scale=-1.25), dict(scale=0.0), dict(eps=0.5), dict(post=False),
                                dict(pre=False), dict(dx_out=False), dict(post=False, dx_out=False), dict(pre=False, gates=None),
                                dict(layout="odd"), dict(layout="odd", post=False)],
                         ids=lambda k: "-".join("%s=%s" % i for i in k.items()))
def test_forms(tracea_gpu, dtype, c, kw):
    check(tracea_gpu, 3, 40, c, dtype, **kw)


def test_rows_of_zeros(tracea_gpu):
    x = torch.zeros(1, 3, 128, device="cuda")
    w = torch.ones(128, device="cuda")
    x_out, y = tracea_gpu.norm_gate_residual(x, x.clone(), w, None, w)
    assert (x_out == 0).all() and (y == 0).all()
    for t in tracea_gpu.norm_gate_residual_backward(x + 1, x + 1, x_out, x, w, None, w):
        assert t is None or torch.isfinite(t).all()


def test_gradients_against_differences(tracea_gpu):
    b, t, c = 2, 5, 48
    m = make(b, t, c, torch.float32, "each")
    x_out, y = tracea_gpu.norm_gate_residual(m["x"], m["h"], m["w_post"], m["gate"], m["w_pre"], residual_scale=0.7)
    got = tracea_gpu.norm_gate_residual_backward(m["dx"], m["dy"], x_out, m["h"], m["w_post"], m["gate"], m["w_pre"], residual_scale=0.7)
    base = [m[n].cpu().double() for n in ("x", "h", "w_post", "gate", "w_pre")]
    dxo, dy = m["dx"].cpu().double(), m["dy"].cpu().double()

    def loss(x, h, wp, g, wq):
        s = 0.7 * x + g[:, None] * (h * rms(h, 1e-6) * wp)
        return (s * dxo).sum() + (s * rms(s, 1e-6) * wq * dy).sum()
    for i in range(5):
        way = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        at = lambda e: [v + e * way if j == i else v for j, v in enumerate(base)]  # noqa: E731
        slope = (loss(*at(1e-5)) - loss(*at(-1e-5))) / 2e-5
        dot = (got[i].cpu().double() * way).sum()
        assert abs(dot - slope) <= 1e-5 * (got[i].cpu().double() * way).abs().sum()


def test_in_place(tracea_gpu):
    m = make(2, 50, 320, torch.bfloat16, "each")
    args = (m["w_post"], m["gate"], m["w_pre"])
    want = tracea_gpu.norm_gate_residual(m["x"], m["h"], *args)
    x, h = m["x"].clone(), m["h"].clone()
    tracea_gpu.norm_gate_residual(x, h, *args, x_out=x, y=h)
    assert torch.equal(x, want[0]) and torch.equal(h, want[1])
    want_b = tracea_gpu.norm_gate_residual_backward(m["dx"], m["dy"], x, m["h"], *args)
    dx, hh = m["dx"].clone(), m["h"].clone()
    got = tracea_gpu.norm_gate_residual_backward(dx, m["dy"], x, hh, *args, dx=dx, dh=hh)
    for a, b in zip(got, want_b):
        assert torch.equal(a, b)


def test_graph(tracea_gpu):
    m = make(2, 60, 512, torch.bfloat16, "each")
    args = (m["w_post"], m["gate"], m["w_pre"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        a, y = tracea_gpu.norm_gate_residual(m["x"], m["h"], *args)
        return (a, y) + tracea_gpu.norm_gate_residual_backward(m["dx"], m["dy"], a, m["h"], *args)
    with torch.cuda.stream(stream):
        want = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            step()
            torch.cuda.synchronize()


def test_empty(tracea_gpu):
    w = torch.ones(64, device="cuda")
    x = torch.empty(2, 0, 64, device="cuda")
    x_out, y = tracea_gpu.norm_gate_residual(x, x, w, None, w)
    assert y.shape == x.shape
    dx, dh, dw_post, dgate, dw_pre = tracea_gpu.norm_gate_residual_backward(x, x, x, x, w, None, w)
    assert (dw_post == 0).all() and (dw_pre == 0).all() and dgate is None


@pytest.mark.parametrize("gates", [None, 0, 1])
def test_a_batch_without_entries_has_zero_weight_gradients(tracea_gpu, gates):
    w = torch.ones(72, device="cuda")
    x = torch.empty(0, 3, 72, device="cuda", dtype=torch.bfloat16)
    gate = None if gates is None else torch.ones(gates, 72, device="cuda")
    dx, dh, dw_post, dgate, dw_pre = tracea_gpu.norm_gate_residual_backward(x, x, x, x, w, gate, w)
    assert dx.shape == dh.shape == x.shape
    assert (dw_post == 0).all() and (dw_pre == 0).all()
    assert (dgate is None) == (gates is None) and (gates is None or (dgate.shape == gate.shape and (dgate == 0).all()))


def test_refusals(tracea_gpu):
    from tracea_amd import capi
    x = torch.randn(2, 5, 64, device="cuda")
    w, g = torch.ones(64, device="cuda"), torch.ones(2, 64, device="cuda")
    fwd, bwd = tracea_gpu.norm_gate_residual, tracea_gpu.norm_gate_residual_backward

    def refused(status, call, *args, **kw):
        with pytest.raises(capi.TraceaError) as e:
            call(*args, **kw)
        assert e.value.status == status, e.value
    refused(capi.INVALID_PARAMS, fwd, x, x.clone())                       # h without w_post
    refused(capi.INVALID_PARAMS, fwd, x)                                  # nothing to do
    refused(capi.INVALID_PARAMS, fwd, x, None, None, g, w)                # gate without h
    refused(capi.INVALID_PARAMS, fwd, x, x[:, :4], w)
    refused(capi.UNSUPPORTED_CONFIG, fwd, x, x.half(), w)
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w[:63])
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w.half())
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w, torch.ones(3, 64, device="cuda"))
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w, g, w, eps=-1.0)
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w, g, w, eps=float("nan"))
    refused(capi.UNSUPPORTED_CONFIG, fwd, torch.randn(1, 1, 8193, device="cuda"), w_pre=torch.ones(8193, device="cuda"))
    refused(capi.UNSUPPORTED_CONFIG, fwd, x.transpose(1, 2).contiguous().transpose(1, 2), w_pre=w)
    refused(capi.CPU_ERROR, fwd, x.cpu(), w_pre=w)
    refused(capi.INVALID_PARAMS, fwd, x, w_pre=w.cpu())
    same = torch.empty_like(x)
    refused(capi.INVALID_PARAMS, fwd, x, x.clone(), w, g, w, x_out=same, y=same)
    refused(capi.INVALID_PARAMS, fwd, x[:, :4], w_pre=w, y=x[:, 1:])
    refused(capi.INVALID_PARAMS, bwd, x, x, x)                            # dy without w_pre
    refused(capi.INVALID_PARAMS, bwd, None, None, x)
    refused(capi.INVALID_PARAMS, bwd, x, x[:1], x, w_pre=w)
