"""Attention whose rows have one large probability and a long tail of small ones: the tail counts in o as it counts in lse.

The other keys lie exp(17.375) = 2^25.07 below the row's peak: each alone is nothing to a 16-bit operand, 131072 of them together are 0.4 % of
the row.  Bounds: those of the formulas, per element, from where the kernels round (see the reference)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_attention_train_gpu import reference, within  # noqa: E402

KEYS = 131072


def operands(rows, d, peak, dtype):
    g = torch.Generator().manual_seed(peak + rows)
    q, k = torch.zeros(1, 1, rows, d), torch.zeros(1, 1, KEYS, d)
    q[..., 0] = 1 + (torch.arange(rows) % 3) / 16  # gaps of 17.375, 18.46 and 19.55
    k[:, :, peak, 0] = 17.375
    v, do = torch.rand(1, 1, KEYS, d, generator=g) + 0.5, torch.randn(1, 1, rows, d, generator=g)  # (values of one sign: nothing cancels)
    return [t.to(dtype).cuda() for t in (q, k, v, do)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("peak", [0, KEYS // 2 + 5, KEYS - 1])
@pytest.mark.parametrize("rows,d", [(1, 64), (3, 128), (40, 64)])
def test_few_rows_over_parts_of_the_keys(tracea_gpu, rows, d, peak, dtype):
    from helpers import launches
    q, k, v, do = operands(rows, d, peak, dtype)
    want = reference(q, k, v, do, False, 1.0)
    o, lse = tracea_gpu.attention_forward(q, k, v, scale=1.0)
    within("o", o, want["o"])
    within("lse", lse, want["lse"])
    for name, t in zip(("dq", "dk", "dv"), tracea_gpu.attention_backward(q, k, v, o, lse, do, scale=1.0)):
        within(name, t, want[name])
    assert launches(lambda: tracea_gpu.attention_forward(q, k, v, scale=1.0, out=o, lse=lse)) == 2


@pytest.fixture(scope="module", params=[(dtype, peak) for dtype in (torch.float16, torch.bfloat16) for peak in (0, KEYS - 1)],
                ids=lambda p: "%s-%d" % ({torch.float16: "f16", torch.bfloat16: "bf16"}[p[0]], p[1]))
def one_walk(request):
    """(o, lse, what they should be) of 512 heads over the operands of one: enough workgroups that the keys stay in one piece."""
    from helpers import launches
    from tracea_amd import capi, ops
    capi.init()
    dtype, peak = request.param
    heads = 512
    q, k, v, do = operands(128, 64, peak, dtype)
    want = reference(q[:, :, :3], k, v, do[:, :, :3], False, 1.0)
    q, k, v = (t.expand(1, heads, -1, -1) for t in (q, k, v))
    o, lse = torch.empty(1, heads, 128, 64, device="cuda", dtype=dtype), torch.empty(1, heads, 128, device="cuda")
    assert launches(lambda: ops.attention_forward(q, k, v, scale=1.0, out=o, lse=lse)) == 1
    return o, lse, want


def test_one_walk_over_the_keys_lse(one_walk):
    """(2048 tiles are added to a number near 1, one after another)"""
    _, lse, want = one_walk
    for h in (0, 200, 511):
        for i in range(0, 126, 3):
            within("lse", lse[:, h:h + 1, i:i + 3], want["lse"])


def test_one_walk_over_the_keys_o(one_walk):
    o, _, want = one_walk
    for h in (0, 200, 511):
        for i in range(0, 126, 3):
            within("o", o[:, h:h + 1, i:i + 3], want["o"])


@pytest.mark.parametrize("shape", [(8, 32, 8, 1, 8192, 128), (2, 8, 2, 1000, 1000, 64), (1, 4, 4, 40, 6000, 96)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_the_forward_pass_repeats_itself(tracea_gpu, shape, dtype):
    b, hq, hk, sq, sk, d = shape
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(b, h, s, d, device="cuda", generator=g).to(dtype) for h, s in ((hq, sq), (hk, sk), (hk, sk)))
    o, lse = tracea_gpu.attention_forward(q, k, v, causal=True)
    for _ in range(5):
        again = tracea_gpu.attention_forward(q, k, v, causal=True)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
