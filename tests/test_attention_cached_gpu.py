"""Attention over a key/value cache in pages against the formula in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
from cache_oracle import E4M3, Pool, attention, check_attention, heads, table  # noqa: E402

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


def run(ops, seed, b, hq, hk, sq, k_lengths, d, page, dtype, e4m3, causal=True, q_lengths=None, layout="bhsd", order="nhpd", scale=None, extra=0, spoil=None,
        garbage=True, rounded=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = max(1, -(-max(k_lengths) // page)) + extra
    pool = Pool(g, b * per + 1, hk, page, d, dtype, e4m3, order)
    pt = table(g, b, per, b * per + 1)
    q = heads(g, b, hq, sq, d, dtype, layout)
    kl = torch.tensor(k_lengths, dtype=torch.int32, device="cuda")
    ql = None if q_lengths is None else torch.tensor(q_lengths, dtype=torch.int32, device="cuda")
    if spoil is not None:
        spoil(pt, pool)
    want, want_lse, allowed, lse_off = attention(q, pool, pt, k_lengths, q_lengths, causal, scale, rounded)
    if garbage and e4m3:  # pages in no table, the first of the pool too
        used = torch.zeros(b * per + 1, dtype=torch.bool, device="cuda")
        used[pt[(pt >= 0) & (pt <= b * per)].long()] = True
        pool.k_scale[~used], pool.v_scale[~used] = float("inf"), float("nan")
    if garbage:  # what lies behind the lengths may be anything
        for i in range(b):
            for slot in range(per):
                page_id = int(pt[i, slot])
                if 0 <= page_id < pool.k.shape[0]:
                    first = max(0, min(page, k_lengths[i] - slot * page))
                    for t in (pool.k, pool.v):
                        if e4m3:
                            Pool._u8(t)[page_id, :, first:] = 0x7f
                            if first == 0:  # (a page that nobody uses)
                                pool.k_scale[page_id] = float("nan")
                                pool.v_scale[page_id] = float("inf")
                        else:
                            t[page_id, :, first:] = float("nan")
    lse = torch.full((b, hq, sq), 7.0, device="cuda")
    out = torch.full_like(q, 9.0) if layout != "odd" else heads(g, b, hq, sq, d, dtype, "odd")
    got = ops.attention_cached(q, pool.k, pool.v, pt, kl, q_lengths=ql, causal=causal, scale=scale or 0.0, out=out, lse=lse, **pool.scales())
    check_attention(got, lse, want, want_lse, allowed, lse_off)
    again = ops.attention_cached(q, pool.k, pool.v, pt, kl, q_lengths=ql, causal=causal, scale=scale or 0.0, **pool.scales())
    assert torch.equal(again, got)
    return got


CASES = [  # b, hq, hk, sq, k_lengths, d, page, causal, q_lengths, layout, order
    (1, 1, 1, 1, [1], 8, 16, True, None, "bhsd", "nhpd"), (1, 12, 12, 1, [197], 64, 16, True, None, "bshd", "nhpd"),
    (3, 8, 2, 1, [0, 1, 129], 128, 64, True, None, "bshd", "npHd"), (2, 16, 4, 5, [5, 333], 96, 16, True, None, "bshd", "both"),
    (2, 10, 1, 3, [2, 700], 80, 48, True, None, "bhsd", "nhpd"), (4, 6, 2, 9, [30, 9, 4, 0], 40, 32, True, [9, 9, 9, 9], "bhsd", "npHd"),
    (2, 4, 4, 70, [300, 70], 64, 128, True, [70, 33], "bshd", "nhpd"), (2, 4, 2, 33, [100, 64], 72, 16, False, [0, 33], "bhsd", "nhpd"),
    (1, 32, 8, 1, [5000], 128, 256, True, None, "bhsd", "nhpd"), (3, 20, 4, 4, [1025, 31, 640], 128, 16, True, None, "odd", "nhpd"),
    (2, 28, 4, 40, [1000, 90], 112, 64, True, [40, 40], "odd", "both"), (1, 40, 1, 2, [2050], 32, 16, False, None, "bshd", "nhpd"),
    (5, 2, 1, 130, [130, 7, 500, 129, 128], 128, 32, True, [130, 130, 2, 1, 128], "bshd", "npHd")]


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(tracea_gpu, case, dtype, e4m3):
    b, hq, hk, sq, k_lengths, d, page, causal, q_lengths, layout, order = case
    run(tracea_gpu, 21, b, hq, hk, sq, k_lengths, d, page, dtype, e4m3, causal, q_lengths, layout, order)


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("sq, long", [(1, 20000), (6, 20000), (40, 20000), (1, 100000), (6, 100000)])
def test_long_and_short_sequences_together(tracea_gpu, sq, long, e4m3):
    """70 sequences, most of them short, cut one by one (20000 keys) or as one line of steps, parts of which begin and end anywhere."""
    lengths = [(i * 37) % 90 for i in range(70)]
    lengths[3], lengths[66] = long, 3001
    run(tracea_gpu, 22, 70, 4, 2, sq, lengths, 64, 32 if long < 50000 else 1024, torch.bfloat16, e4m3)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
def test_a_table_far_wider_than_the_sequences(tracea_gpu, dtype):
    run(tracea_gpu, 23, 2, 8, 2, 1, [40, 300], 128, 16, dtype, True, extra=600)


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("sq", [1, 50, 100])
def test_pages_that_are_not_there(tracea_gpu, sq, e4m3):
    def spoil(pt, pool):
        pt[0, 1], pt[0, 3], pt[1, 0], pt[1, 1], pt[2] = -1, 10 ** 6, 2 ** 31 - 1, -(2 ** 31), -7
    run(tracea_gpu, 24, 3, 4, 2, sq, [100, 90, 64], 64, 16, torch.float16, e4m3, spoil=spoil)


def test_no_pages_at_all(tracea_gpu):
    for e4m3 in (False, True):
        pool = Pool(torch.Generator(device="cuda").manual_seed(1), 0, 2, 16, 64, torch.float16, e4m3)
        q = torch.randn(2, 4, 3, 64, device="cuda").half()
        lse = torch.zeros(2, 4, 3, device="cuda")
        for m in (0, 4):
            o = tracea_gpu.attention_cached(q, pool.k, pool.v, torch.zeros(2, m, dtype=torch.int32, device="cuda"),
                                            torch.tensor([3, 50], dtype=torch.int32, device="cuda"), lse=lse, **pool.scales())
            assert (o == 0).all() and (lse == -math.inf).all()


def test_lengths_beyond_what_there_is(tracea_gpu):
    g = torch.Generator(device="cuda").manual_seed(25)
    pool = Pool(g, 8, 2, 16, 64, torch.float16, False)
    pt = table(g, 2, 4, 8)
    q = heads(g, 2, 4, 3, 64, torch.float16)
    as_is = dict(device="cuda", dtype=torch.int32)
    got = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, torch.tensor([2 ** 31 - 1, -5], **as_is), q_lengths=torch.tensor([99, -1], **as_is))
    want = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, torch.tensor([64, 0], **as_is), q_lengths=torch.tensor([3, 0], **as_is))
    assert torch.equal(got, want) and (got[1] == 0).all() and (got[0] != 0).any()


@pytest.mark.parametrize("scale", [-0.2, 3.0])
@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
def test_scales_of_scores(tracea_gpu, scale, e4m3):
    run(tracea_gpu, 26, 2, 4, 2, 3, [150, 77], 64, 16, torch.bfloat16, e4m3, scale=scale)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
def test_pages_of_very_different_scales(tracea_gpu, dtype):
    """Values of one page 2^20 times another's, in any order, and a page of zeros with the least scale."""
    def spoil(pt, pool):
        n, h = pool.v_scale.shape
        pool.v_scale.copy_(torch.exp2(torch.randint(-28, -7, (n, h), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).float()))
        pool.v_scale[pt[0, 2].long()] = 2.0 ** -126
        pool.k_scale[pt[0, 4].long()] = 2.0 ** -126
    run(tracea_gpu, 27, 2, 4, 2, 2, [3000, 555], 128, 16, dtype, True, spoil=spoil, garbage=False)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("sq", [1, 9, 70])
def test_scales_that_are_no_powers_of_two(tracea_gpu, sq, dtype):
    def spoil(pt, pool):
        g = torch.Generator(device="cuda").manual_seed(6)
        for t in (pool.k_scale, pool.v_scale):
            t.copy_(0.002 + 0.01 * torch.rand(t.shape, device="cuda", generator=g))
    run(tracea_gpu, 34, 2, 4, 2, sq, [1100, 333], 128, 16, dtype, True, spoil=spoil, rounded=True)
    run(tracea_gpu, 35, 2, 4, 2, sq, [1100, 333], 64, 64, dtype, True, spoil=spoil, rounded=True)


@pytest.mark.parametrize("sq", [1, 40])
def test_f16_values_at_the_ends_of_the_type(tracea_gpu, sq):
    """Codes times scales beyond f16's largest number and below its smallest: only the results have to fit."""
    def spoil(pt, pool):
        pool.k_scale.fill_(2.0 ** -8)
        pool.k_scale[pt[0, :2].long()] = 2.0 ** -26
        pool.v_scale.fill_(2.0 ** -22)
        pool.v_scale[pt[1].long()] = 2.0 ** 5
    run(tracea_gpu, 36, 2, 4, 2, sq, [200, 200], 64, 16, torch.float16, True, spoil=spoil, garbage=False)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
def test_a_dominant_key_wherever_it_is(tracea_gpu, dtype, e4m3):
    """One key scores far above all others: its value comes back, whichever lane, wave or part meets it."""
    for at in (0, 5, 17, 30, 33, 100, 127, 128, 1000, 2999):
        def spoil(pt, pool):
            page, place = int(pt[0, at // 16]), at % 16
            for h in range(2):
                pool.k[page, h, place] = (torch.full((64,), 200.0, device="cuda") if e4m3 else torch.full((64,), 60.0, device="cuda")).to(pool.k.dtype)
                if e4m3:
                    pool.k_scale[page, h] = 0.25
        g = torch.Generator(device="cuda").manual_seed(28)
        pool = Pool(g, 188, 2, 16, 64, dtype, e4m3)
        pt = table(g, 1, 188, 188)
        spoil(pt, pool)
        q = torch.full((1, 4, 1, 64), 2.0, device="cuda").to(dtype)
        o = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, torch.tensor([3000], dtype=torch.int32, device="cuda"), **pool.scales())
        want = pool.values("v")[int(pt[0, at // 16]), :, at % 16].repeat_interleave(2, 0)
        assert ((o[0, :, 0].double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-6).all(), at


def test_every_code(tracea_gpu):
    """One visible key: o is its value, for all finite codes and their sign."""
    codes = torch.tensor([c for c in range(256) if c & 0x7f != 0x7f] + [0, 0], dtype=torch.uint8, device="cuda").view(2, 128)
    for dtype in HALVES:
        for i in range(2):
            k = torch.zeros(1, 1, 16, 128, dtype=torch.uint8, device="cuda")
            v = torch.full((1, 1, 16, 128), 0x7f, dtype=torch.uint8, device="cuda")  # (NaN behind the only key)
            v[0, 0, 0] = codes[i]
            one = torch.ones(1, 1, device="cuda")
            zero = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
            o = tracea_gpu.attention_cached(torch.ones(1, 1, 1, 128, device="cuda", dtype=dtype), k.view(E4M3), v.view(E4M3), zero, zero[0] + 1,
                                            k_scale=one, v_scale=one)
            assert torch.equal(o.flatten().float(), codes[i].view(E4M3).float())


def test_nan_among_the_keys_shows(tracea_gpu):
    g = torch.Generator(device="cuda").manual_seed(29)
    pool = Pool(g, 8, 2, 16, 128, torch.bfloat16, True)
    pt = table(g, 2, 4, 8)
    pool.k.view(torch.uint8)[pt[0, 1].long(), 0, 3, 9] = 0x7f
    q = heads(g, 2, 4, 1, 128, torch.bfloat16)
    o = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, torch.tensor([50, 50], dtype=torch.int32, device="cuda"), **pool.scales())
    assert torch.isnan(o[0, :2]).all() and torch.isfinite(o[0, 2:]).all() and torch.isfinite(o[1]).all()


def test_offsets_past_32_bits(tracea_gpu):
    """Pages of a cache of more than 2^32 bytes, from both its ends."""
    n, hk, page, d = 70000, 4, 64, 128
    k = torch.zeros(n, hk, page, d, device="cuda", dtype=E4M3)
    v = torch.zeros_like(k)
    scale = torch.full((n, hk), 2.0 ** -7, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(30)
    pt = torch.tensor([[0, n - 1, n // 2 + 3, n - 2], [n - 3, 1, 2, n - 4]], dtype=torch.int32, device="cuda")
    small = Pool(g, 8, hk, page, d, torch.bfloat16, True)
    for i in range(8):
        at = int(pt.flatten()[i])
        for big, part, ps in ((k, small.k, small.k_scale), (v, small.v, small.v_scale)):
            big.view(torch.uint8)[at] = part.view(torch.uint8)[i]
    small.k_scale.fill_(2.0 ** -7)
    small.v_scale.fill_(2.0 ** -7)
    near = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lengths = torch.tensor([256, 199], dtype=torch.int32, device="cuda")
    q = heads(g, 2, 8, 1, d, torch.bfloat16)
    o = tracea_gpu.attention_cached(q, k, v, pt, lengths, k_scale=scale, v_scale=scale)
    assert torch.equal(o, tracea_gpu.attention_cached(q, small.k, small.v, near, lengths, **small.scales()))
    x = heads(g, 2, hk, 3, d, torch.bfloat16)
    starts = torch.tensor([250, 196], dtype=torch.int32, device="cuda")
    tracea_gpu.cache_append(x, x, k, v, pt, starts, k_scale=scale, v_scale=scale.clone())
    tracea_gpu.cache_append(x, x, small.k, small.v, near, starts, **small.scales())
    for i in range(8):
        assert torch.equal(k.view(torch.uint8)[int(pt.flatten()[i])], small.k.view(torch.uint8)[i])


@pytest.mark.parametrize("sq", [1, 4, 60])
def test_captured_and_replayed(tracea_gpu, sq):
    g = torch.Generator(device="cuda").manual_seed(31)
    pool = Pool(g, 520, 2, 16, 128, torch.bfloat16, True)
    pt = table(g, 2, 256, 520)
    q = heads(g, 2, 8, sq, 128, torch.bfloat16)
    lengths = torch.tensor([4000, 100], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tracea_gpu.attention_cached(q, pool.k, pool.v, pt, lengths, **pool.scales())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, lengths, **pool.scales())
        for n in ([4000, 100], [1, 4096], [0, 0], [2222, 3333]):
            lengths.copy_(torch.tensor(n))
            q.normal_(generator=g)
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            want = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, lengths, **pool.scales())
            torch.cuda.synchronize()
            assert torch.equal(got, want), n


def test_capture_without_a_workspace_runs_unsplit(tracea_gpu):
    g = torch.Generator(device="cuda").manual_seed(32)
    pool = Pool(g, 256, 2, 16, 64, torch.float16, False)
    pt = table(g, 1, 256, 256)
    q = heads(g, 1, 4, 1, 64, torch.float16)
    lengths = torch.tensor([4096], dtype=torch.int32, device="cuda")
    want = attention(q, pool, pt, [4096])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = tracea_gpu.attention_cached(q, pool.k, pool.v, pt, lengths)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            check_attention(out, None, want[0], want[1], want[2], want[3])


def test_agrees_with_the_attention_over_dense_keys(tracea_gpu):
    """A cache of one page per sequence is a dense tensor."""
    g = torch.Generator(device="cuda").manual_seed(33)
    q, k, v = heads(g, 2, 8, 64, 128, torch.bfloat16), heads(g, 2, 2, 208, 128, torch.bfloat16), heads(g, 2, 2, 208, 128, torch.bfloat16)
    lengths = torch.tensor([208, 99], dtype=torch.int32, device="cuda")
    ql = torch.tensor([64, 50], dtype=torch.int32, device="cuda")
    lse = torch.empty(2, 8, 64, device="cuda")
    got = tracea_gpu.attention_cached(q, k, v, torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), lengths, q_lengths=ql, lse=lse)
    want, want_lse = tracea_gpu.attention_forward(q, k, v, causal=True, q_lengths=ql, k_lengths=lengths)
    assert ((got.double() - want.double()).abs() <= 2 * 2.0 ** -8 * want.double().abs() + 2 * 2.0 ** -8 * v.abs().max()).all()
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    fine = lse > -math.inf
    assert ((lse - want_lse).abs()[fine] <= 1e-5 * lse[fine].abs() + 1e-5).all()


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("hq, hk, sq", [(33, 1, 1), (8, 1, 5), (16, 2, 6), (64, 1, 1), (32, 2, 4)])  # 33, 40, 48, 64, 64 rows a key/value head
@pytest.mark.parametrize("k_lengths, page", [([70, 6, 256], 16), ([3000, 5, 700], 64), ([20000, 1030, 6], 64)])
def test_two_blocks_of_32_rows(tracea_gpu, k_lengths, page, hq, hk, sq, dtype, e4m3):
    """Heads that share keys, times drafted tokens, beyond one block: keys uncut, cut problem by problem, and cut as one line."""
    run(tracea_gpu, 37, 3, hq, hk, sq, k_lengths, 128 if sq < 6 else 96, page, dtype, e4m3, True, [sq, max(1, sq - 2), sq])


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("hq, sq", [(8, 1), (8, 5), (8, 10), (8, 100)])  # rows a key/value head: 4, 20, 40, 400
def test_tables_far_wider_than_the_sequences(tracea_gpu, hq, sq, e4m3):
    """The plan is that of the longest sequences that the table could hold: parts of one step, shares of nothing."""
    run(tracea_gpu, 38, 3, hq, 2, sq, [197, 0, 700], 128, 16, torch.bfloat16, e4m3, extra=2000, q_lengths=[sq, 0, max(1, sq - 1)], layout="bshd")
