"""A sequence's life with a cache, as a program that samples from a model has it: a prompt in pieces, then tokens one by one, some of them drafted and
taken back; every step's attention against dense attention over everything so far."""
import pytest

torch = pytest.importorskip("torch")
from cache_oracle import E4M3, U32, Pool, attention, check_attention, half_step, rotated  # noqa: E402
from tracea_amd.capi import TraceaError  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Caches:
    """What a program keeps: pools, a table, the lengths so far; pages are handed out as sequences grow."""

    def __init__(self, b, hk, d, page, m, dtype, e4m3):
        n = b * m
        kind = E4M3 if e4m3 else dtype
        self.k, self.v = (torch.full((n, hk, page, d), 0x7f if e4m3 else 0, dtype=torch.uint8 if e4m3 else dtype, device="cuda") for _ in range(2))
        if e4m3:
            self.k, self.v = self.k.view(kind), self.v.view(kind)
        else:
            self.k.fill_(float("nan"))
            self.v.fill_(float("nan"))
        self.scales = {s: torch.full((n, hk), float("nan"), device="cuda") for s in ("k_scale", "v_scale")} if e4m3 else {}
        order = torch.randperm(n, generator=torch.Generator().manual_seed(4)).to(torch.int32)
        self.table = order.view(b, m).cuda()
        self.lengths = torch.zeros(b, dtype=torch.int32, device="cuda")

    def pool(self, page, e4m3):
        p = object.__new__(Pool)
        p.page, p.e4m3, p.k, p.v = page, e4m3, self.k, self.v
        p.k_scale, p.v_scale = self.scales.get("k_scale"), self.scales.get("v_scale")
        return p


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype,d,rot,page,adjacent", [(torch.bfloat16, 128, 128, 64, False), (torch.float16, 80, 40, 16, True)], ids=["bf16", "f16"])
def test_prompt_then_tokens(tracea_gpu, dtype, d, rot, page, adjacent, e4m3):
    g = torch.Generator(device="cuda").manual_seed(41)
    b, hq, hk, m = 3, 8, 2, 400 // page + 1
    caches = Caches(b, hk, d, page, m, dtype, e4m3)
    freq = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float32) / (rot // 2))
    wq, wk = (1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    kept = [[torch.zeros(hk, 0, d, device="cuda", dtype=torch.float64) for _ in range(2)] for _ in range(b)]  # exact keys and values

    def step(new, counts=None, back=0):
        """`new` tokens a sequence (counts: of each), of which the last `back` are taken back afterwards."""
        q, k, v = (torch.randn(b, new, h, d, device="cuda", generator=g).to(dtype).transpose(1, 2) for h in (hq, hk, hk))
        n = torch.full((b,), new, dtype=torch.int32, device="cuda") if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
        qn, kn = tracea_gpu.qk_norm_rotary(q, k, wq, wk, eps=EPS)
        qt = tracea_gpu.cache_append(kn, v, caches.k, caches.v, caches.table, caches.lengths, lengths=None if counts is None else n, q=qn, inv_freq=freq,
                                     adjacent=adjacent, **caches.scales)
        now = caches.lengths + n
        lse = torch.empty(b, hq, new, device="cuda")
        o = tracea_gpu.attention_cached(qt, caches.k, caches.v, caches.table, now, q_lengths=None if counts is None else n, lse=lse, **caches.scales)
        # against what the caches hold
        want, want_lse, allowed, lse_off = attention(qt, caches.pool(page, e4m3), caches.table, now.tolist(), n.tolist())
        check_attention(o, lse, want, want_lse, allowed, lse_off)
        # and what they hold against what was put in
        for i in range(b):
            c, start = int(n[i]), int(caches.lengths[i])
            if start + c == 0:
                continue
            angle = torch.arange(start, start + c, device="cuda", dtype=torch.float64)[None, :, None] * freq.double()
            kept[i][0] = torch.cat([kept[i][0], rotated(kn[i:i + 1, :, :c], angle, rot, adjacent)[0][0]], 1)
            kept[i][1] = torch.cat([kept[i][1], v[i, :, :c].double()], 1)
            for j, name in enumerate("kv"):
                pool = caches.pool(page, e4m3).values(name)
                slots = torch.arange(start + c, device="cuda")
                held = pool[caches.table[i].long()[slots // page], :, slots % page].transpose(0, 1)
                x = kept[i][j]
                off = half_step(dtype) * x.abs() + 32 * U32 * x.abs().amax()
                if e4m3:  # half a step of a code, and what rescaling rounds below the normal codes
                    s = caches.scales[name + "_scale"].double()[caches.table[i].long()[slots // page]].t()[..., None]
                    off = torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -9 * s) + 32 * U32 * x.abs().amax()
                assert ((held - x).abs() <= off).all()
        caches.lengths = now - back
        for i in range(b):
            if back:
                kept[i] = [x[:, :x.shape[1] - back] for x in kept[i]]
        return o

    step(70, counts=[70, 33, 0])
    step(100, counts=[1, 100, 64])
    for _ in range(3):
        step(1)
    step(5, back=3)
    step(1)
    step(5, back=5)
    step(17)


def test_decoding_in_a_graph(tracea_gpu):
    """The three calls of a step captured once and replayed for every token, lengths counted on the device, against the same calls one by one."""
    g = torch.Generator(device="cuda").manual_seed(42)
    b, hq, hk, d, page, m = 4, 16, 4, 128, 16, 40
    one, two = Caches(b, hk, d, page, m, torch.bfloat16, True), Caches(b, hk, d, page, m, torch.bfloat16, True)
    freq = torch.logspace(0, -4, 64, device="cuda")
    w = torch.ones(d, device="cuda")
    q, k, v = (torch.randn(b, 1, h, d, device="cuda", generator=g).bfloat16().transpose(1, 2) for h in (hq, hk, hk))

    def step(c):
        qn, kn = tracea_gpu.qk_norm_rotary(q, k, w, w)
        tracea_gpu.cache_append(kn, v, c.k, c.v, c.table, c.lengths, q=qn, q_out=qn, inv_freq=freq, **c.scales)
        c.lengths += 1
        return tracea_gpu.attention_cached(qn, c.k, c.v, c.table, c.lengths, **c.scales)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c in (one, two):  # (also makes the workspaces)
            x = torch.randn(b, 500, hk, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16().transpose(1, 2)
            tracea_gpu.cache_append(x, x, c.k, c.v, c.table, c.lengths, inv_freq=freq, **c.scales)
            c.lengths += torch.tensor([500, 1, 255, 256], dtype=torch.int32, device="cuda")
            step(c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(one)
        for _ in range(6):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device="cuda", generator=g))
            graph.replay()
            want = step(two)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(one.lengths, two.lengths)


def test_calls_from_two_threads_on_one_stream(tracea_gpu):
    """Both split their keys in the stream's workspace: launches of a call stay together."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(43)
    pool = Pool(g, 1100, 2, 16, 128, torch.bfloat16, True)
    table = torch.randperm(1100, device="cuda", generator=g)[:1000].int().view(1, 1000)
    qs = [torch.randn(1, 8, n, 128, device="cuda", generator=g).bfloat16() for n in (1, 40)]
    lengths = torch.tensor([16000], dtype=torch.int32, device="cuda")
    call = lambda q: tracea_gpu.attention_cached(q, pool.k, pool.v, table, lengths, **pool.scales())  # noqa: E731
    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    wrong, stream = [], torch.cuda.Stream()

    def many(i):
        with torch.cuda.stream(stream):
            got = [call(qs[i]) for _ in range(40)]
        stream.synchronize()
        wrong.extend(x for x in got if not torch.equal(x, want[i]))

    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_training_step_through_norms_and_attention(tracea_gpu):
    """Gradients of queries, keys and weights through norm, rotation and attention, against differentiating the formulas in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(44)
    b, hq, hk, s, d = 2, 4, 2, 48, 64
    q, k, v, do = (torch.randn(b, h, s, d, device="cuda", generator=g).half() for h in (hq, hk, hk, hq))
    wq, wk = (1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    pos = torch.arange(s, dtype=torch.int32, device="cuda").view(1, s, 1)
    freq = torch.logspace(0, -3, 32, device="cuda")
    qn, kn = tracea_gpu.qk_norm_rotary(q, k, wq, wk, pos, freq)
    o, lse = tracea_gpu.attention_forward(qn, kn, v, causal=True)
    dqn, dkn, dv = tracea_gpu.attention_backward(qn, kn, v, o, lse, do, causal=True)
    got = tracea_gpu.qk_norm_rotary_backward(dqn, dkn, q, k, wq, wk, pos, freq) + (dv,)
    leaves = [t.double().requires_grad_(True) for t in (q, k, wq, wk, v)]
    angle = pos.double() * freq.double()
    norm = lambda x, w: rotated(x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w, angle, 64, False)[0]  # noqa: E731
    qq, kk, vv = norm(leaves[0], leaves[2]), norm(leaves[1], leaves[3]).repeat_interleave(2, 1), leaves[4].repeat_interleave(2, 1)
    x = (qq @ kk.transpose(-1, -2)) / 8
    x = x.masked_fill(torch.arange(s, device="cuda")[None] > torch.arange(s, device="cuda")[:, None], float("-inf"))
    want = torch.autograd.grad(torch.softmax(x, -1) @ vv, leaves, do.double())
    for a, w in zip(got, want):
        # some ten roundings to 11 bits one after another, of gradients of a few times the result's size; in 2-norm
        assert (a.double() - w).norm() <= 40 * 2.0 ** -11 * w.norm()


def test_other_operators_refuse_codes(tracea_gpu):
    """Codes of 8 bits are a type of caches only."""
    x = torch.randn(2, 4, 16, 64, device="cuda").to(E4M3)
    a, pos, freq = x[0, 0], torch.zeros(2, 16, 1, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    w = torch.ones(64, device="cuda")
    for call in (lambda: tracea_gpu.gemm(a, a.t()), lambda: tracea_gpu.attention(x, x, x), lambda: tracea_gpu.softmax(a),
                 lambda: tracea_gpu.attention_forward(x, x, x), lambda: tracea_gpu.rotary(x, x, pos, freq),
                 lambda: tracea_gpu.qk_norm_rotary(x, x, w, w, pos, freq), lambda: tracea_gpu.norm_gate_residual(x[0], x[0], w, None, w)):
        with pytest.raises((TraceaError, TypeError)):
            call()
