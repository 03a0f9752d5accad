"""Appending to a key/value cache in pages against the definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
from cache_oracle import E4M3, U32, Pool, angles, append, half_step, heads, rotated, table  # noqa: E402

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


def run(ops, seed, b, hq, hk, t, d, rot, page, dtype, e4m3, starts, lengths=None, adjacent=False, layout="bhsd", order="nhpd", positions=None,
        spoil=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    per = max(1, -(-(max(0, int(starts.max())) + t) // page))
    pool = Pool(g, b * per + 2, hk, page, d, dtype, e4m3, order)
    pt = table(g, b, per, b * per + 2)
    q = heads(g, b, hq, t, d, dtype, layout) if hq else None
    k, v = heads(g, b, hk, t, d, dtype, layout, 2.0), heads(g, b, hk, t, d, dtype, layout, 0.5)
    if spoil is not None:
        spoil(pt, k, v)
    freq = 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float32) / max(rot // 2, 1)) if rot else None
    if positions is None:
        angle = (starts.clamp(min=0).double()[:, None] + torch.arange(t, device="cuda"))[..., None] * freq.double() if rot else None
    else:
        angle = positions.double() * freq.double()
    want = append(pool, pt, k, v, starts, lengths, rot, angle, adjacent)
    before = {n: Pool._u8(getattr(pool, n)).clone() for n in "kv"}
    turn = dict(inv_freq=freq, positions=positions, adjacent=adjacent) if rot else {}
    q_out = ops.cache_append(k, v, pool.k, pool.v, pt, starts, lengths=lengths, q=q, **pool.scales(), **turn)
    for n in "kv":
        values, allowed, scale, changed = want[n]
        got = pool.values(n)
        if e4m3:
            now = getattr(pool, n + "_scale").double()
            assert torch.equal(now, scale), n
        nan = torch.isnan(values) | torch.isinf(values) & e4m3
        assert torch.equal(torch.isnan(got), nan)
        fine = torch.isfinite(values)
        assert ((got - values).abs()[fine] <= allowed[fine] * (1 + 1e-9)).all(), n
        # nothing else is touched, to the bit: what is neither a new token nor in a page whose scale has grown
        same = ~changed
        assert torch.equal(Pool._u8(getattr(pool, n))[same], before[n][same])
    if q is not None:
        y, made_of = rotated(q, angle, rot, adjacent) if rot else (q.double(), q.double().abs())
        for i in range(b):
            n = t if lengths is None else max(0, min(int(lengths[i]), t))
            off = (q_out[i, :, :n].double() - y[i, :, :n]).abs()
            assert (off <= half_step(dtype) * y[i, :, :n].abs() * (1 + 1e-6) + 16 * U32 * made_of[i, :, :n] + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
            assert (q_out[i, :, n:] == 0).all()
    return pool, q_out


CASES = [  # b, hq, hk, t, d, rot, page, starts, lengths, adjacent, layout, order
    (1, 0, 1, 1, 8, 0, 16, [0], None, False, "bhsd", "nhpd"), (3, 8, 2, 1, 128, 128, 64, [0, 63, 64], None, False, "bshd", "nhpd"),
    (2, 4, 4, 5, 64, 64, 16, [14, 3], None, False, "bshd", "npHd"), (3, 10, 2, 77, 80, 48, 16, [0, 33, 100], [77, 1, 40], True, "bhsd", "both"),
    (2, 3, 1, 130, 96, 96, 48, [47, 5], [0, 130], False, "bhsd", "npHd"), (1, 2, 2, 300, 40, 20, 256, [100], None, False, "odd", "nhpd"),
    (2, 5, 3, 33, 128, 128, 32, [0, 31], None, True, "odd", "both"), (1, 0, 8, 64, 128, 128, 64, [64], None, False, "bshd", "nhpd"),
    (2, 6, 2, 20, 72, 0, 32, [9, 40], [20, 7], False, "bhsd", "nhpd"), (1, 1, 1, 40, 512, 512, 16, [7], None, False, "bhsd", "nhpd"),
    (2, 4, 70, 3, 16, 16, 16, [15, 0], None, False, "bhsd", "nhpd"), (1, 2, 1, 600, 64, 64, 512, [500], None, False, "bhsd", "nhpd"),
    (2, 5, 3, 300, 128, 128, 256, [200, 0], [300, 131], True, "bshd", "npHd"), (1, 3, 3, 300, 128, 64, 256, [131], None, False, "bhsd", "both"),
    (1, 2, 2, 270, 128, 128, 512, [300], None, False, "bhsd", "nhpd"),
    # pairs in fours and twos
    (2, 5, 2, 70, 80, 40, 16, [0, 33], [70, 9], False, "bhsd", "npHd"), (2, 5, 2, 70, 80, 40, 64, [0, 33], [70, 9], True, "bshd", "npHd"),
    (2, 3, 3, 130, 40, 40, 64, [5, 64], None, False, "bshd", "nhpd"), (2, 3, 3, 130, 40, 40, 256, [5, 64], None, True, "bhsd", "nhpd"),
    (1, 2, 2, 50, 40, 20, 32, [3], None, False, "bhsd", "nhpd"), (1, 2, 2, 50, 40, 20, 32, [3], None, True, "bhsd", "nhpd"),
    (1, 4, 1, 33, 88, 24, 48, [7], None, False, "bshd", "nhpd"), (2, 1, 1, 9, 72, 8, 16, [0, 9], None, True, "bhsd", "nhpd"),
    (1, 2, 2, 300, 80, 40, 512, [9], None, False, "bhsd", "nhpd"), (1, 2, 2, 300, 80, 40, 512, [9], None, True, "bhsd", "nhpd")]


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_append(tracea_gpu, case, dtype, e4m3):
    b, hq, hk, t, d, rot, page, starts, lengths, adjacent, layout, order = case
    run(tracea_gpu, 11, b, hq, hk, t, d, rot, page, dtype, e4m3, starts, lengths, adjacent, layout, order)


def test_positions_of_the_caller(tracea_gpu):
    pos = torch.randint(0, 2 ** 31 - 1, (2, 9, 1), dtype=torch.int32, device="cuda")
    run(tracea_gpu, 12, 2, 4, 2, 9, 64, 64, 16, torch.bfloat16, True, [3, 20], positions=pos)


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
def test_tokens_without_a_place(tracea_gpu, e4m3):
    def spoil(pt, k, v):
        pt[0, 1], pt[1, 0], pt[1, 2] = -1, 10 ** 6, -(2 ** 31)
    run(tracea_gpu, 13, 2, 4, 2, 60, 64, 64, 16, torch.float16, e4m3, [5, -9], spoil=spoil)
    # behind the table, and beyond 32 bits
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = Pool(g, 4, 2, 16, 64, torch.float16, e4m3)
    before = {n: Pool._u8(getattr(pool, n)).clone() for n in "kv"}
    pt = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    k = torch.randn(1, 2, 40, 64, device="cuda").half()
    for start in (64, 2 ** 31 - 1, 2 ** 31 - 20):
        tracea_gpu.cache_append(k, k, pool.k, pool.v, pt, torch.tensor([start], dtype=torch.int32, device="cuda"), **pool.scales())
    assert all(torch.equal(Pool._u8(getattr(pool, n)), before[n]) for n in "kv")
    tracea_gpu.cache_append(k, k, pool.k, pool.v, pt, torch.tensor([60], dtype=torch.int32, device="cuda"), **pool.scales())
    assert torch.equal(Pool._u8(pool.k)[:3], before["k"][:3]) and not torch.equal(Pool._u8(pool.k)[3], before["k"][3])


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
def test_infinities_and_nan(tracea_gpu, dtype):
    def spoil(pt, k, v):
        k[0, 0, 3, 5], v[0, 1, 4, 6], v[1, 0, 0, 0], k[1, 1] = float("inf"), float("nan"), -float("inf"), 0
    for e4m3 in (False, True):
        run(tracea_gpu, 14, 2, 0, 2, 20, 64, 0, 16, dtype, e4m3, [4, 0], spoil=spoil)


def test_extreme_values(tracea_gpu):
    """The largest and smallest bf16 numbers: scales from 2^-126 to the type's end."""
    def spoil(pt, k, v):
        k[0, 0] = torch.finfo(torch.bfloat16).max
        k[0, 1] = 2.0 ** -133
        v[0, 0] = 448 * 2.0 ** -20
        v[0, 1] = 450 * 2.0 ** -20  # (above 448: the next power of two)
    run(tracea_gpu, 15, 1, 0, 2, 16, 64, 0, 16, torch.bfloat16, True, [0], spoil=spoil)


def test_codes_are_those_of_a_rounding_to_nearest_even(tracea_gpu):
    """Values that are not turned: every f16 number up to 448 that a code or the middle of two is, and its neighbours."""
    codes = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
    mids = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mids, mids * (1 + 2.0 ** -9), mids * (1 - 2.0 ** -9)]).half()
    x = torch.cat([x, -x])
    x = torch.cat([x, torch.full((16 * 64 - x.numel(),), 448.0, dtype=torch.float16)]).view(1, 1, 16, 64).cuda()
    pool = Pool(torch.Generator(device="cuda").manual_seed(1), 1, 1, 16, 64, torch.float16, True)
    zero = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    tracea_gpu.cache_append(x, x, pool.k, pool.v, zero, zero[0], **pool.scales())
    assert pool.k_scale.item() == 1.0 and pool.v_scale.item() == 1.0
    want = x[0].float().to(E4M3).view(torch.uint8)
    assert torch.equal(pool.k.view(torch.uint8)[0], want) and torch.equal(pool.v.view(torch.uint8)[0], want)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
def test_a_cache_is_the_same_however_its_tokens_were_cut(tracea_gpu, dtype):
    g = torch.Generator(device="cuda").manual_seed(16)
    b, hk, t, d, page = 2, 3, 50, 64, 32
    k, v = (heads(g, b, hk, t, d, dtype) * torch.exp2(torch.randint(-3, 4, (t, 1), device="cuda", generator=g).float()).to(dtype) for _ in range(2))
    freq = torch.logspace(0, -3, 32, device="cuda")
    pt = table(g, b, 2, 5)
    whole, cut = (Pool(torch.Generator(device="cuda").manual_seed(2), 5, hk, page, d, dtype, True) for _ in range(2))
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    tracea_gpu.cache_append(k, v, whole.k, whole.v, pt, zero, inv_freq=freq, **whole.scales())
    at = 0
    for n in (1, 1, 7, 20, 1, 3, 17):
        tracea_gpu.cache_append(k[:, :, at:at + n], v[:, :, at:at + n], cut.k, cut.v, pt, zero + at, inv_freq=freq, **cut.scales())
        at += n
    assert at == t and torch.equal(whole.k_scale, cut.k_scale) and torch.equal(whole.v_scale, cut.v_scale)
    for n in "kv":
        # the tokens' places (what lies behind them is no token's, and moves with the scale as often as it grows)
        of = pt.long()
        x, y = (p.values(n)[of].transpose(2, 3).flatten(1, 2)[:, :t] for p in (whole, cut))  # [B,T,Hk,D]
        scale = getattr(whole, n + "_scale").double()[of].repeat_interleave(page, 1)[:, :t, :, None]
        # codes below the normal ones (2^-6) may have been rounded at up to six scales, each half a step of the last or less
        assert torch.equal(torch.where(x.abs() >= 2.0 ** -6 * scale, x, y), torch.where(y.abs() > 2.0 ** -6 * scale, y, torch.where(x.abs() >= 2.0 ** -6 * scale, x, y)))
        assert ((x - y).abs() <= 2.0 ** -9 * scale).all()


def test_graph_and_in_place_queries(tracea_gpu):
    g = torch.Generator(device="cuda").manual_seed(17)
    b, hq, hk, d, page = 4, 8, 2, 128, 16
    pool, eager = (Pool(torch.Generator(device="cuda").manual_seed(3), 12, hk, page, d, torch.bfloat16, True) for _ in range(2))
    pt = table(g, b, 3, 12)
    q, k, v = heads(g, b, hq, 1, d, torch.bfloat16), heads(g, b, hk, 1, d, torch.bfloat16), heads(g, b, hk, 1, d, torch.bfloat16)
    starts = torch.tensor([0, 3, 15, 30], dtype=torch.int32, device="cuda")
    freq = torch.logspace(0, -3, 64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            tracea_gpu.cache_append(k, v, pool.k, pool.v, pt, starts, q=q, q_out=q, inv_freq=freq, **pool.scales())
            starts += 1
        for i in range(5):
            for x in (q, k, v):
                x.normal_(generator=g)
            want = tracea_gpu.cache_append(k, v, eager.k, eager.v, pt, starts, q=q, inv_freq=freq, **eager.scales())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(q, want) and starts.tolist() == [i + 1, i + 4, i + 16, i + 31]
            for n in "kv":
                assert torch.equal(getattr(pool, n).view(torch.uint8), getattr(eager, n).view(torch.uint8))
                assert torch.equal(getattr(pool, n + "_scale"), getattr(eager, n + "_scale"))


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "side"])
@pytest.mark.parametrize("t, page", [(20, 16), (70, 64), (300, 256)])
@pytest.mark.parametrize("d", [8, 24, 40, 72, 88, 104])
def test_scales_are_those_of_turned_keys(tracea_gpu, d, t, page, adjacent, dtype):
    """Heads that are turned as a whole and end in half a couple of pieces: the last pair of some tokens is (450, 0), turned by 45 degrees or so.  What
    is written stays below 448, what was given does not."""
    def spoil(pt, k, v):
        k *= 2.0 ** -6
        k[:, :, ::7, d - 2 if adjacent else d // 2 - 1] = 450
        k[:, :, ::7, d - 1] = 0
    slowest = 10000.0 ** (-(d // 2 - 1) / (d // 2))
    pos = torch.full((2, t, 1), round(0.785 / slowest), dtype=torch.int32, device="cuda")
    run(tracea_gpu, 18, 2, 3, 2, t, d, d, page, dtype, True, [0, 33], None, adjacent, "bshd", positions=pos, spoil=spoil)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "side"])
@pytest.mark.parametrize("d, rot, page", [(40, 40, 64), (72, 72, 32), (24, 24, 256), (128, 128, 64), (80, 40, 48), (64, 32, 16)])
def test_every_layout_of_keys_gives_the_same_cache(tracea_gpu, d, rot, page, adjacent, dtype):
    """Rows on 16 bytes and rows that begin anywhere are taken by different kernels: the same scales and codes.  (Queries in 16 bits may be rounded
    once or, behind fp32, twice.)"""
    b, hq, hk, t = 2, 3, 2, 300
    freq = torch.logspace(0, -3, rot // 2, device="cuda")
    starts = torch.tensor([5, 1000], dtype=torch.int32, device="cuda")
    got = []
    for layout in ("bshd", "odd"):
        g = torch.Generator(device="cuda").manual_seed(19)
        pool = Pool(g, 2 * (1300 // page + 1), hk, page, d, dtype, True)
        pt = table(g, b, 1300 // page + 1, 2 * (1300 // page + 1))
        q, k, v = (heads(g, b, h, t, d, dtype, layout) for h in (hq, hk, hk))
        tracea_gpu.cache_append(k, v, pool.k, pool.v, pt, starts, q=q, inv_freq=freq, adjacent=adjacent, **pool.scales())
        got.append([pool.k_scale, pool.v_scale, pool.k.view(torch.uint8), pool.v.view(torch.uint8)])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", HALVES, ids=["f16", "bf16"])
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "side"])
@pytest.mark.parametrize("d, page", [(40, 64), (72, 64), (24, 512), (128, 512)])
def test_heads_of_any_width_are_the_same_however_their_tokens_were_cut(tracea_gpu, d, page, adjacent, dtype):
    """The scales of pages that a call, or several (whose pages the other kernel may take), have written; codes up to what was rounded more than once."""
    g = torch.Generator(device="cuda").manual_seed(20)
    b, hk, t = 4, 4, 600
    k, v = (heads(g, b, hk, t, d, dtype, "bshd") for _ in range(2))
    freq = torch.logspace(0, -3, d // 2, device="cuda")
    per = -(-t // page)
    pt = table(g, b, per, b * per)
    whole, cut = (Pool(torch.Generator(device="cuda").manual_seed(2), b * per, hk, page, d, dtype, True) for _ in range(2))
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    turn = dict(inv_freq=freq, adjacent=adjacent)
    tracea_gpu.cache_append(k, v, whole.k, whole.v, pt, zero, **whole.scales(), **turn)
    at = 0
    for n in (1, 1, 7, 300, 1, 3, 20, 267):
        tracea_gpu.cache_append(k[:, :, at:at + n], v[:, :, at:at + n], cut.k, cut.v, pt, zero + at, **cut.scales(), **turn)
        at += n
    assert at == t and torch.equal(whole.k_scale, cut.k_scale) and torch.equal(whole.v_scale, cut.v_scale)
    for n in "kv":
        of = pt.long()
        x, y = (p.values(n)[of].transpose(2, 3).flatten(1, 2)[:, :t] for p in (whole, cut))
        scale = getattr(whole, n + "_scale").double()[of].repeat_interleave(page, 1)[:, :t, :, None]
        normal = torch.maximum(x.abs(), y.abs()) > 2.0 ** -6 * scale
        assert torch.equal(x[normal], y[normal]) and ((x - y).abs() <= 2.0 ** -9 * scale).all()


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("layout", ["bshd", "odd"])
@pytest.mark.parametrize("batches", [1, 3])
def test_positions_along_several_axes(tracea_gpu, batches, layout, e4m3):
    """Positions [1,T,A] and [B,T,A], sections of unlike length, one of them empty."""
    g = torch.Generator(device="cuda").manual_seed(21)
    b, hq, hk, t, d, page, sections = 3, 4, 2, 50, 96, 32, [20, 0, 17, 7]
    pos = torch.randint(0, 5000, (batches, t, 4), dtype=torch.int32, device="cuda", generator=g)
    freq = torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float32) / max(n, 1)) for n in sections])
    angle = angles(pos, freq, sections).expand(b, -1, -1)
    starts = torch.tensor([0, 40, 7], dtype=torch.int32, device="cuda")
    pool = Pool(g, 12, hk, page, d, torch.bfloat16, e4m3)
    pt = table(g, b, 3, 12)
    q, k, v = (heads(g, b, h, t, d, torch.bfloat16, layout) for h in (hq, hk, hk))
    want = append(pool, pt, k, v, starts, None, 88, angle, False)
    q_out = tracea_gpu.cache_append(k, v, pool.k, pool.v, pt, starts, q=q, positions=pos, inv_freq=freq, sections=sections, **pool.scales())
    for n in "kv":
        values, allowed, scale, _ = want[n]
        assert ((pool.values(n) - values).abs() <= allowed * (1 + 1e-9)).all(), n
        assert not e4m3 or torch.equal(getattr(pool, n + "_scale").double(), scale), n
    y, made_of = rotated(q, angle, 88, False)
    assert ((q_out.double() - y).abs() <= half_step(torch.bfloat16) * y.abs() * (1 + 1e-6) + 16 * U32 * made_of).all()


@pytest.mark.parametrize("layout", ["bshd", "odd"])
def test_queries_at_places_beyond_31_bits(tracea_gpu, layout):
    """starts + t reaches 2^31: such tokens have no place, their queries are turned like all others."""
    g = torch.Generator(device="cuda").manual_seed(22)
    t, d = 40, 64
    starts = torch.tensor([2 ** 31 - 1, 2 ** 31 - 20, 3], dtype=torch.int32, device="cuda")
    freq = torch.logspace(0, -3, 32, device="cuda")
    pool = Pool(g, 9, 2, 16, d, torch.bfloat16, False)
    q, k, v = (heads(g, 3, h, t, d, torch.bfloat16, layout) for h in (4, 2, 2))
    q_out = tracea_gpu.cache_append(k, v, pool.k, pool.v, table(g, 3, 3, 9), starts, q=q, inv_freq=freq)
    y, made_of = rotated(q, (starts.double()[:, None] + torch.arange(t, device="cuda"))[..., None] * freq.double(), d, False)
    assert ((q_out.double() - y).abs() <= half_step(torch.bfloat16) * y.abs() * (1 + 1e-6) + 16 * U32 * made_of).all()


@pytest.mark.parametrize("e4m3", [False, True], ids=["16", "e4m3"])
def test_more_query_heads_than_are_taken_at_once(tracea_gpu, e4m3):
    run(tracea_gpu, 23, 2, 1100, 1, 5, 24, 16, 16, torch.float16, e4m3, [0, 14], [5, 3], layout="odd")


def test_long_pages_without_a_rotation(tracea_gpu):
    """More tokens of a page than a workgroup takes at once."""
    run(tracea_gpu, 24, 1, 3, 2, 9000, 40, 0, 16384, torch.bfloat16, True, [100], layout="odd")
    run(tracea_gpu, 25, 1, 3, 2, 9000, 40, 0, 16384, torch.bfloat16, False, [100], [8195])


def test_more_than_31_bits_of_pieces_in_a_page(tracea_gpu):
    """131072 tokens of 128 heads and 128 columns in one page, rows that begin anywhere: 2^31 pieces, all of them one workgroup's (5 s)."""
    t, h, d = 131072, 128, 128
    g = torch.Generator(device="cuda").manual_seed(26)
    at = lambda n: torch.randn(1, n, t, d + 1, device="cuda", dtype=torch.bfloat16, generator=g)[..., 1:]  # noqa: E731
    q, k, v = at(h), at(1), at(1)
    out = torch.full((1, h, t, d + 1), 7.0, device="cuda", dtype=torch.bfloat16)[..., 1:]
    k_cache, v_cache = (torch.zeros(1, 1, t, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    zero = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    tracea_gpu.cache_append(k, v, k_cache, v_cache, zero, zero[0], q=q, q_out=out)
    assert torch.equal(k_cache, k) and torch.equal(v_cache, v) and all(torch.equal(q[0, i], out[0, i]) for i in range(h))
