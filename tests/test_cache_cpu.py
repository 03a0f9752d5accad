"""What the operators over a key/value cache refuse and how they plan their launches, without a device: the dispatch code built for the host with
launches that write down what they were asked for."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from tracea_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16, I32, I8, E4M3 = capi.F32, capi.F16, capi.BF16, capi.I32, capi.I8, capi.E4M3
SIZES = {F32: 4, F16: 2, BF16: 2, I32: 4, I8: 1, E4M3: 1}
OK, INVALID, UNSUPPORTED, HOST = capi.SUCCESS, capi.INVALID_PARAMS, capi.UNSUPPORTED_CONFIG, 4


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    cxx = shutil.which("g++")
    rocm = "/opt/rocm/include"
    if cxx is None or not os.path.isdir(rocm):
        pytest.skip("no g++ or no HIP headers")
    so = str(tmp_path_factory.mktemp("cache") / "stub.so")
    csrc = os.path.join(ROOT, "tracea_amd", "csrc")
    subprocess.check_call([cxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", csrc, "-I",
                           os.path.join(csrc, "host"), "-isystem", rocm, "-shared", "-fPIC", os.path.join(ROOT, "tests", "cpp_cache_stub.cpp"), "-o", so])
    lib = C.CDLL(so)
    for name in ("tracea_qk_norm_rotary", "tracea_qk_norm_rotary_backward", "tracea_cache_append", "tracea_attention_cached"):
        getattr(lib, name).restype, getattr(lib, name).argtypes = capi.SIGNATURES[name]
    lib.stub_message.restype = lib.stub_launch.restype = C.c_char_p
    lib.stub_value.restype, lib.stub_value.argtypes = C.c_longlong, [C.c_char_p]
    lib.stub_page_of.argtypes = [C.c_void_p, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int, C.c_longlong]
    return lib


class T:
    """A tensor that is nowhere: a view at an address of its own, or at another's."""
    next = 1 << 32

    def __init__(self, shape, dtype=BF16, stride=None, ptr=None, device=0):
        if stride is None:
            stride, n = [], 1
            for e in reversed(shape):
                stride.insert(0, n)
                n *= max(e, 1)
        if ptr is None:
            ptr = T.next
            T.next += (sum((max(e, 1) - 1) * abs(s) for e, s in zip(shape, stride)) + 1) * SIZES[dtype] + 4096 & ~255
        self.shape, self.stride, self.dtype, self.ptr, self.device = list(shape), list(stride), dtype, ptr, device
        self.view = capi.View(ptr, self.shape, self.stride, dtype, device)

    def but(self, **kw):
        a = dict(shape=self.shape, stride=self.stride, dtype=self.dtype, ptr=self.ptr, device=self.device)
        if "shape" in kw and "stride" not in kw:
            a["stride"] = None
        if ("shape" in kw or "dtype" in kw) and "ptr" not in kw:
            a["ptr"] = None
        a.update(kw)
        return T(**a)

    def at(self, offset):
        return self.but(ptr=self.ptr + offset)


def val(t):
    return t.view.c


def ref(t):
    return None if t is None else C.byref(t.view.c)


def norm_args(b=2, hq=4, hk=2, s=10, d=64, p=32, axes=1, dtype=BF16):
    return dict(q=T([b, hq, s, d], dtype), k=T([b, hk, s, d], dtype), qw=T([d], F32), kw=T([d], F32), pos=T([b, s, axes], I32), freq=T([p], F32),
                qo=T([b, hq, s, d], dtype), ko=T([b, hk, s, d], dtype), sections=[p], axes=axes, eps=1e-6, adjacent=0)


def norm(stub, a):
    stub.stub_reset(0)
    params = capi.QkNormParams(a["axes"], (C.c_uint32 * 4)(*a["sections"]), a["adjacent"], a["eps"], None)
    return stub.tracea_qk_norm_rotary(val(a["q"]), ref(a["k"]), ref(a["qw"]), ref(a["kw"]), ref(a["pos"]), ref(a["freq"]), ref(a["qo"]), ref(a["ko"]), params)


def norm_backward(stub, a, no_workspace=0):
    stub.stub_reset(no_workspace)
    params = capi.QkNormParams(a["axes"], (C.c_uint32 * 4)(*a["sections"]), a["adjacent"], a["eps"], None)
    return stub.tracea_qk_norm_rotary_backward(val(a["dqo"]), ref(a["dko"]), val(a["q"]), ref(a["k"]), ref(a["qw"]), ref(a["kw"]), ref(a["pos"]),
                                               ref(a["freq"]), ref(a["qo"]), ref(a["ko"]), ref(a["dqw"]), ref(a["dkw"]), params)


def backward_args(**kw):
    a = norm_args(**kw)
    a.update(dqo=a["q"].but(ptr=None), dko=a["k"].but(ptr=None), dqw=T([a["q"].shape[3]], F32), dkw=T([a["q"].shape[3]], F32))
    return a


def append_args(b=2, hq=4, hk=2, t=5, d=64, p=32, pages=9, page=16, m=4, dtype=BF16, cache=E4M3):
    return dict(k=T([b, hk, t, d], dtype), v=T([b, hk, t, d], dtype), q=T([b, hq, t, d], dtype), kc=T([pages, hk, page, d], cache),
                vc=T([pages, hk, page, d], cache), ks=T([pages, hk], F32) if cache == E4M3 else None, vs=T([pages, hk], F32) if cache == E4M3 else None,
                pt=T([b, m], I32), starts=T([b], I32), lengths=T([b], I32), pos=T([b, t, 1], I32), freq=T([p], F32), qo=T([b, hq, t, d], dtype),
                sections=[p], axes=1)


def append(stub, a):
    stub.stub_reset(0)
    params = capi.CacheAppendParams(a["axes"], (C.c_uint32 * 4)(*a["sections"]), 0, None)
    return stub.tracea_cache_append(val(a["k"]), val(a["v"]), ref(a["q"]), ref(a["kc"]), ref(a["vc"]), ref(a["ks"]), ref(a["vs"]), val(a["pt"]),
                                    val(a["starts"]), ref(a["lengths"]), ref(a["pos"]), ref(a["freq"]), ref(a["qo"]), params)


def attention_args(b=2, hq=4, hk=2, sq=1, d=64, pages=9, page=16, m=4, dtype=BF16, cache=E4M3):
    return dict(q=T([b, hq, sq, d], dtype), kc=T([pages, hk, page, d], cache), vc=T([pages, hk, page, d], cache),
                ks=T([pages, hk], F32) if cache == E4M3 else None, vs=T([pages, hk], F32) if cache == E4M3 else None, pt=T([b, m], I32), ql=T([b], I32),
                kl=T([b], I32), o=T([b, hq, sq, d], dtype), lse=T([b, hq, sq], F32), scale=0.0, causal=1)


def attention(stub, a, no_workspace=0):
    stub.stub_reset(no_workspace)
    return stub.tracea_attention_cached(val(a["q"]), val(a["kc"]), val(a["vc"]), ref(a["ks"]), ref(a["vs"]), val(a["pt"]), ref(a["ql"]), val(a["kl"]),
                                        ref(a["o"]), ref(a["lse"]), capi.AttentionParams(a["causal"], 0, a["scale"], None))


CALLS = {"norm": (norm, norm_args), "norm_backward": (norm_backward, backward_args), "append": (append, append_args), "attention": (attention, attention_args)}
FOLDED = lambda t: t.but(stride=[0] + t.stride[1:])  # noqa: E731
SIDEWAYS = lambda t: t.but(stride=t.stride[:2] + [1, max(t.shape[2], 2)])  # noqa: E731


@pytest.mark.parametrize("call", sorted(CALLS))
def test_good_calls_are_launched(stub, call):
    run, args = CALLS[call]
    assert run(stub, args()) == OK, stub.stub_message()
    assert stub.stub_launch() != b""


REFUSALS = [  # call, name, what becomes of the operand (or a value), status, part of the message
    ("norm", "q", lambda t: t.but(dtype=I8), UNSUPPORTED, "f32, f16 or bf16"), ("norm", "k", lambda t: t.but(dtype=F16), UNSUPPORTED, "one type"),
    ("norm", "k", lambda t: t.but(shape=[2, 2, 11, 64]), INVALID, "k"), ("norm", "qo", lambda t: t.but(shape=[2, 3, 10, 64]), INVALID, "q_out"),
    ("norm", "qo", lambda t: None, INVALID, "result"), ("norm", "ko", lambda t: None, INVALID, "result"), ("norm", "k", lambda t: None, INVALID, "operand"),
    ("norm", "q", SIDEWAYS, UNSUPPORTED, "contiguous"), ("norm", "ko", SIDEWAYS, UNSUPPORTED, "contiguous"), ("norm", "qo", FOLDED, INVALID, "share an address"),
    ("norm", "qw", lambda t: t.but(shape=[63]), INVALID, "q_weight"), ("norm", "kw", lambda t: t.but(dtype=BF16), INVALID, "k_weight"),
    ("norm", "kw", lambda t: t.but(stride=[2]), INVALID, "k_weight"), ("norm", "pos", lambda t: None, INVALID, "positions"),
    ("norm", "freq", lambda t: None, INVALID, "inv_freq"), ("norm", "freq", lambda t: t.but(shape=[33]), INVALID, "sections"),
    ("norm", "sections", lambda s: [31], INVALID, "sections"), ("norm", "sections", lambda s: [2 ** 32 - 1], INVALID, "sections"),
    ("norm", "axes", lambda n: 5, INVALID, "axes"), ("norm", "axes", lambda n: 0, INVALID, "axes"), ("norm", "axes", lambda n: 2, INVALID, "positions"),
    ("norm", "pos", lambda t: t.but(dtype=F32), INVALID, "positions"), ("norm", "eps", lambda e: -1.0, INVALID, "eps"),
    ("norm", "eps", lambda e: float("nan"), INVALID, "eps"), ("norm", "q", lambda t: t.but(device=-1), HOST, "host memory"),
    ("norm", "q", lambda t: t.but(device=7), INVALID, "out of range"), ("norm", "k", lambda t: t.but(device=1), INVALID, "devices"),
    ("norm", "qw", lambda t: t.but(device=1), INVALID, "devices"), ("norm", "pos", lambda t: t.but(device=1), INVALID, "devices"),
    ("norm", "q", lambda t: t.but(shape=[2, 4, 10]), INVALID, "rank"), ("norm", "q", lambda t: t.but(ptr=0), INVALID, "NULL"),
    ("norm_backward", "dqw", lambda t: t.but(dtype=BF16), INVALID, "dq_weight"), ("norm_backward", "qw", lambda t: None, INVALID, "needs the weight"),
    ("norm_backward", "dko", lambda t: None, INVALID, "go together"), ("norm_backward", "dqo", lambda t: t.but(shape=[2, 4, 9, 64]), INVALID, "dq_out"),
    ("norm_backward", "qo", FOLDED, INVALID, "share an address"), ("norm_backward", "dqo", SIDEWAYS, UNSUPPORTED, "contiguous"),
    ("append", "k", lambda t: t.but(dtype=F32), UNSUPPORTED, "f16 or bf16"), ("append", "v", lambda t: t.but(dtype=F16), UNSUPPORTED, "one type"),
    ("append", "v", lambda t: t.but(shape=[2, 2, 6, 64]), INVALID, "k and v"), ("append", "q", lambda t: None, INVALID, "go together"),
    ("append", "qo", lambda t: None, INVALID, "go together"), ("append", "kc", lambda t: t.but(dtype=I8), UNSUPPORTED, "e4m3"),
    ("append", "vc", lambda t: t.but(dtype=BF16), UNSUPPORTED, "caches"), ("append", "ks", lambda t: None, INVALID, "k_scale"),
    ("append", "vs", lambda t: t.but(dtype=BF16), INVALID, "v_scale"), ("append", "vs", lambda t: t.but(shape=[9, 3]), INVALID, "v_scale"),
    ("append", "kc", lambda t: t.but(shape=[9, 3, 16, 64]), INVALID, "heads"), ("append", "vc", lambda t: t.but(shape=[8, 2, 16, 64]), INVALID, "k_cache and v_cache"),
    ("append", "kc", SIDEWAYS, UNSUPPORTED, "contiguous"), ("append", "kc", lambda t: t.but(stride=[2048, 1024, 68, 1]), UNSUPPORTED, "multiples of 8"),
    ("append", "kc", lambda t: t.but(stride=[-2048, 1024, 64, 1]), UNSUPPORTED, "not negative"), ("append", "kc", lambda t: t.at(4), UNSUPPORTED, "begin on"),
    ("append", "kc", lambda t: t.but(stride=[1 << 31, 1 << 30, 1 << 27, 1]), UNSUPPORTED, "apart"),
    ("append", "pt", lambda t: t.but(dtype=F32), INVALID, "page_table"), ("append", "pt", lambda t: t.but(shape=[3, 4]), INVALID, "page_table"),
    ("append", "pt", lambda t: t.but(stride=[8, 2]), INVALID, "page_table"), ("append", "pt", lambda t: t.but(shape=[2, 1 << 28], stride=[1 << 28, 1]), UNSUPPORTED, "pages of"),
    ("append", "starts", lambda t: t.but(shape=[3]), INVALID, "starts"), ("append", "lengths", lambda t: t.but(dtype=F32), INVALID, "lengths"),
    ("append", "starts", lambda t: t.but(device=1), INVALID, "devices"), ("append", "kc", lambda t: t.but(device=1), INVALID, "devices"),
    ("append", "vs", lambda t: t.but(device=1), INVALID, "devices"), ("append", "kc", FOLDED, INVALID, "share an address"),
    ("append", "ks", FOLDED, INVALID, "share an address"), ("append", "kc", lambda t: None, INVALID, "NULL"), ("append", "freq", lambda t: None, INVALID, "inv_freq"),
    ("attention", "q", lambda t: t.but(dtype=F32), UNSUPPORTED, "f16 or bf16"), ("attention", "o", lambda t: t.but(dtype=F16), UNSUPPORTED, "one type"),
    ("attention", "o", lambda t: t.but(shape=[2, 4, 2, 64]), INVALID, "q and o"), ("attention", "o", lambda t: None, INVALID, "NULL"),
    ("attention", "lse", lambda t: t.but(dtype=BF16), INVALID, "lse"), ("attention", "lse", lambda t: t.but(shape=[2, 4, 2]), INVALID, "lse"),
    ("attention", "kc", lambda t: t.but(dtype=F16), UNSUPPORTED, "caches"), ("attention", "ks", lambda t: None, INVALID, "k_scale"),
    ("attention", "kl", lambda t: t.but(shape=[1]), INVALID, "k_lengths"), ("attention", "ql", lambda t: t.but(dtype=F32), INVALID, "q_lengths"),
    ("attention", "q", SIDEWAYS, UNSUPPORTED, "contiguous"), ("attention", "o", SIDEWAYS, UNSUPPORTED, "contiguous"), ("attention", "o", FOLDED, INVALID, "share an address"),
    ("attention", "scale", lambda s: float("inf"), INVALID, "scale"), ("attention", "q", lambda t: t.but(device=-1), HOST, "host memory"),
    ("attention", "kl", lambda t: t.but(device=1), INVALID, "devices"), ("attention", "lse", lambda t: t.but(device=1), INVALID, "devices")]


@pytest.mark.parametrize("call,name,change,status,message", REFUSALS, ids=["%s-%s-%d" % (r[0], r[1], i) for i, r in enumerate(REFUSALS)])
def test_refusals(stub, call, name, change, status, message):
    run, args = CALLS[call]
    a = args()
    a[name] = change(a[name])
    got = run(stub, a)
    assert got == status, (got, stub.stub_message())
    assert message.encode() in stub.stub_message() and stub.stub_launch() == b""


def test_shapes_that_are_too_large(stub):
    assert norm(stub, norm_args(d=514, p=32)) == UNSUPPORTED
    assert append(stub, append_args(d=520)) == UNSUPPORTED
    assert append(stub, append_args(d=60, p=30)) == UNSUPPORTED
    assert append(stub, append_args(page=24)) == UNSUPPORTED and append(stub, append_args(page=0)) == UNSUPPORTED
    assert append(stub, append_args(b=65536, t=1)) == UNSUPPORTED
    assert attention(stub, attention_args(d=136)) == UNSUPPORTED and attention(stub, attention_args(d=60)) == UNSUPPORTED
    assert attention(stub, attention_args(hq=5)) == INVALID
    assert attention(stub, attention_args(hq=1 << 14, hk=1, sq=16)) == UNSUPPORTED
    assert attention(stub, attention_args(b=1 << 20, hk=16, hq=16)) == UNSUPPORTED
    big = attention_args()
    big["pt"] = T([2, (1 << 31) // 16], I32)
    assert attention(stub, big) == UNSUPPORTED
    assert attention(stub, attention_args(page=1 << 16, m=256)) == UNSUPPORTED  # M P P = 2^40


def test_overlaps(stub):
    a = norm_args()
    assert norm(stub, dict(a, qo=a["q"], ko=a["k"])) == OK
    for name, other, shift in (("qo", "q", 128), ("qo", "k", 0), ("ko", "q", 64), ("qo", "qw", 0), ("ko", "pos", 0), ("qo", "freq", 0)):
        assert norm(stub, dict(a, **{name: a[name].but(ptr=a[other].ptr + shift)})) == INVALID, (name, other)
    assert norm(stub, dict(a, ko=a["ko"].but(ptr=a["qo"].ptr))) == INVALID
    a = backward_args()
    assert norm_backward(stub, dict(a, qo=a["q"], ko=a["dko"])) == OK
    for name, other in (("qo", "k"), ("qo", "dko"), ("qo", "qw"), ("dqw", "qw"), ("dqw", "q"), ("dkw", "dqw"), ("ko", "qo"), ("dqw", "pos")):
        assert norm_backward(stub, dict(a, **{name: a[name].but(ptr=a[other].ptr)})) == INVALID, (name, other)
    a = append_args()
    assert append(stub, dict(a, qo=a["q"])) == OK
    for name, other, shift in (("qo", "q", 16), ("qo", "k", 0), ("kc", "vc", 0), ("kc", "k", 0), ("vc", "v", 0), ("ks", "vs", 0), ("ks", "kc", 0), ("kc", "pt", 0),
                               ("vs", "starts", 0), ("kc", "lengths", 0), ("qo", "pos", 0), ("vc", "freq", 0), ("qo", "kc", 0)):
        assert append(stub, dict(a, **{name: a[name].but(ptr=a[other].ptr + shift)})) == INVALID, (name, other)
    a = attention_args()
    for name, other in (("o", "q"), ("o", "kc"), ("o", "vc"), ("o", "ks"), ("o", "pt"), ("o", "kl"), ("o", "ql"), ("lse", "q"), ("lse", "vs"), ("lse", "o")):
        assert attention(stub, dict(a, **{name: a[name].but(ptr=a[other].ptr)})) == INVALID, (name, other)
    # keys and values of one buffer
    both = T([9, 2, 2, 16, 64], E4M3)
    fused = dict(kc=both.but(shape=[9, 2, 16, 64], stride=[4096, 1024, 64, 1], ptr=both.ptr), vc=both.but(shape=[9, 2, 16, 64], stride=[4096, 1024, 64, 1], ptr=both.ptr + 2048))
    assert append(stub, dict(append_args(), **fused)) == OK and attention(stub, dict(a, **fused)) == OK


def test_calls_with_nothing_to_do(stub):
    assert norm(stub, norm_args(b=0)) == OK and stub.stub_launch() == b""
    assert norm(stub, norm_args(s=0)) == OK and stub.stub_launch() == b""
    assert norm_backward(stub, backward_args(s=0)) == OK and stub.stub_launch() == b"qk_norm_backward"  # (gradients of the weights: zeros)
    assert append(stub, append_args(t=0)) == OK and stub.stub_launch() == b""
    assert append(stub, append_args(b=0)) == OK and stub.stub_launch() == b""
    assert attention(stub, attention_args(sq=0)) == OK and stub.stub_launch() == b""
    a = attention_args(pages=0)
    for n in ("kc", "vc", "ks", "vs"):
        a[n] = a[n].but(ptr=0)
    assert attention(stub, a) == OK and stub.stub_launch() == b"attention" and stub.stub_value(b"M") == 0


def test_optional_operands(stub):
    a = norm_args()
    assert norm(stub, dict(a, k=None, ko=None, kw=None)) == OK and norm(stub, dict(a, qw=None, kw=None)) == OK
    assert norm(stub, dict(a, pos=None, freq=None, axes=0, sections=[])) == OK
    a = append_args()
    assert append(stub, dict(a, q=None, qo=None)) == OK and append(stub, dict(a, lengths=None, pos=None)) == OK
    assert append(stub, dict(a, pos=None, freq=None, axes=0, sections=[])) == OK
    assert append(stub, dict(a, pos=None, axes=2, sections=[16, 16])) == INVALID
    assert attention(stub, dict(attention_args(), ql=None, lse=None)) == OK
    assert norm_backward(stub, dict(backward_args(), dqw=None, dkw=None)) == OK and stub.stub_value(b"workspace") == 0


def test_no_workspace(stub):
    assert norm_backward(stub, backward_args(), no_workspace=1) == UNSUPPORTED and b"workspace" in stub.stub_message()
    assert norm_backward(stub, dict(backward_args(), dqw=None, dkw=None), no_workspace=1) == OK
    for a in (attention_args(b=1, m=4096, pages=4096, d=128), attention_args(b=1, sq=200, m=4096, pages=4096, d=128)):
        assert attention(stub, a, no_workspace=1) == OK
        assert stub.stub_value(b"workgroups") == 0 and stub.stub_value(b"splits") == 1 and stub.stub_value(b"meta") == 0


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("d", [40, 64, 128])
def test_workspaces_hold_what_the_kernels_write(stub, d, cache):
    for b in (1, 3, 16, 64, 300):
        for hq, hk in ((1, 1), (8, 2), (40, 8), (32, 1)):
            for sq in (1, 3, 5, 17, 200, 1500):
                for m in (1, 8, 100, 2048):
                    assert attention(stub, attention_args(b=b, hq=hq, hk=hk, sq=sq, d=d, m=m, page=64, cache=cache)) == OK
                    v = lambda n: stub.stub_value(n.encode())  # noqa: E731
                    rows, blocks, problems = v("rows"), v("row_blocks"), b * hk * v("row_blocks")
                    assert rows in (16, 32, 128) and blocks * rows >= hq // hk * sq > (blocks - 1) * rows
                    slots = problems * v("splits") if rows == 128 else 2 * v("workgroups")
                    if rows == 128 and v("splits") == 1 or rows < 128 and v("workgroups") == 0:
                        assert v("meta") == 0 and v("workspace") == 0
                        continue
                    width = 64 if d <= 64 else 128
                    assert v("part_ml") - v("part_o") == slots * rows * width * 4 and v("meta") - v("part_ml") == slots * rows * 8
                    assert v("workspace") == v("meta") - v("part_o") + problems * 8 and v("part_o") % 16 == 0
                    assert v("workspace") <= 80 << 20
                    assert problems <= 65535 and problems * -(-m * 64 // v("step")) < 1 << 30
                    if rows < 128:  # a line's shares have workgroups, as parts for one a share and a last one for each problem have
                        assert v("workgroups") >= v("line") and (v("apart") == 0 or v("workgroups") >= v("shares") + problems)
    a = backward_args(b=4, hq=32, hk=8, s=2048, d=128, p=64)
    assert norm_backward(stub, a) == OK and stub.stub_value(b"workspace") == 2 * stub.stub_value(b"qk.blocks") * 128 * 4 <= 4 << 20


def test_heads_of_appending_workgroups(stub):
    for hk in (1, 2, 7, 8, 65, 200):
        for hq in (0, 1, 8, 33, 256):
            for b, t, page in ((1, 1, 16), (16, 1, 64), (2, 4096, 64), (64, 300, 128)):
                a = append_args(b=b, hq=max(hq, 1), hk=hk, t=t, page=page, m=100)
                if hq == 0:
                    a["q"] = a["qo"] = None
                assert append(stub, a) == OK
                v = lambda n: stub.stub_value(n.encode())  # noqa: E731
                assert v("append.heads") <= 64 and v("append.heads") * v("append.groups") >= hk and (v("append.groups") - 1) * v("append.heads") < hk
                assert v("append.queries") * v("append.groups") >= hq
                assert v("append.pages") == (t + page - 2) // page + 1


def test_pieces_of_appending_are_counted_in_32_bits(stub):
    """Whatever pages, heads and rotations a call has, what a workgroup takes at once (heads x tokens x pieces of single columns) stays below 2^31."""
    for t, page in ((1, 16), (4096, 64), (131072, 131072), (1 << 20, (1 << 20) - 16), (1 << 22, 16), ((1 << 31) - (1 << 16), (1 << 20) - 16)):
        for hq, hk in ((1, 1), (128, 1), (200, 65), (1 << 20, 1)):
            for d, p in ((128, 0), (512, 0), (512, 1), (128, 5), (512, 256), (512, 255)):
                if hq * t > 1 << 42:
                    continue
                a = append_args(b=1, hq=1, hk=1, t=t, d=d, p=max(p, 1), page=page, m=1)
                for n, h in (("q", hq), ("qo", hq), ("k", hk), ("v", hk)):  # (rows that begin anywhere)
                    a[n] = T([1, h, t, d], BF16, stride=[0, (d + 1) * t, d + 1, 1]).at(2)
                for n in ("kc", "vc"):
                    a[n] = T([9, hk, page, d], E4M3)
                for n in ("ks", "vs"):
                    a[n] = T([9, hk], F32)
                if p == 0:
                    a.update(pos=None, freq=None, axes=0, sections=[])
                v = lambda n: stub.stub_value(n.encode())  # noqa: E731
                assert append(stub, a) == OK and v("append.vec") == 1, stub.stub_message()
                tokens = min(t, page, v("append.tokens_at_once"))
                assert tokens > 0 and tokens * p <= 4096
                for heads in (v("append.heads"), min(v("append.queries"), v("append.queries_at_once"))):
                    assert heads > 0 and heads * tokens * d < (1 << 31) - 256


def test_more_new_tokens_than_are_counted(stub):
    a = append_args(b=1, t=(1 << 31) - (1 << 16) + 1, page=1 << 19, m=1)
    assert append(stub, a) == UNSUPPORTED and b"new tokens" in stub.stub_message()


def test_pieces_are_taken_where_rows_allow_them(stub):
    a = norm_args()
    assert norm(stub, a) == OK and stub.stub_value(b"qk.vec") == 8 and stub.stub_value(b"qk.lanes") == 4
    assert norm(stub, dict(a, q=a["q"].at(2))) == OK and stub.stub_value(b"qk.vec") == 0 and stub.stub_value(b"qk.lanes") == 64
    assert norm(stub, dict(a, q=a["q"].but(stride=[2604, 651, 65, 1]))) == OK and stub.stub_value(b"qk.vec") == 0
    assert norm(stub, dict(a, q=a["q"].at(4))) == OK and stub.stub_value(b"qk.vec") == 2 and stub.stub_value(b"qk.lanes") == 16
    assert norm(stub, dict(a, q=a["q"].at(8))) == OK and stub.stub_value(b"qk.vec") == 4 and stub.stub_value(b"qk.lanes") == 8
    for p, pieces in ((32, 8), (30, 2), (28, 4), (16, 8), (15, 0), (0, 8)):
        assert norm(stub, norm_args(p=p)) == OK and stub.stub_value(b"qk.vec") == pieces, p
    a = append_args()
    assert append(stub, a) == OK and stub.stub_value(b"append.vec") == 8 and stub.stub_value(b"append.held") == 1
    assert append(stub, dict(a, k=a["k"].at(2))) == OK and stub.stub_value(b"append.vec") == 1 and stub.stub_value(b"append.held") == 0
    assert append(stub, dict(a, q=a["q"].at(8))) == OK and stub.stub_value(b"append.vec") == 4 and stub.stub_value(b"append.held") == 0
    for p, pieces in ((32, 8), (30, 2), (28, 4), (15, 1), (0, 8)):
        assert append(stub, append_args(p=p)) == OK and stub.stub_value(b"append.vec") == pieces and stub.stub_value(b"append.held") == (p % 4 == 0), p
    flipped = a["v"].but(stride=[640, 320, -64, 1], ptr=1 << 50)
    assert append(stub, dict(a, v=flipped)) == OK and stub.stub_value(b"append.held") == 0
    far = a["v"].but(stride=[1 << 33, 1 << 32, 1 << 28, 1], ptr=1 << 50)
    assert append(stub, dict(a, v=far)) == OK and stub.stub_value(b"append.held") == 0


def test_pages_outside_a_table_or_a_cache(stub):
    table = (C.c_int * 8)(3, -1, 9, 0, 8, 2 ** 31 - 1, -2 ** 31, 7)
    at = lambda b, slot, n=9, m=4: stub.stub_page_of(C.addressof(table), 4, m, n, 16, b, slot)  # noqa: E731
    assert [at(0, s) for s in (-1, 0, 1, 2, 3, 4, 2 ** 40)] == [-1, 3, -1, -1, 0, -1, -1]
    assert [at(1, s) for s in range(4)] == [8, -1, -1, 7]
    assert [at(0, s, n=0) for s in range(4)] == [-1] * 4 and at(0, 0, m=0) == -1


@pytest.mark.parametrize("page", [16, 32, 48, 80, 256, 4096, 65520])
def test_page_of_a_group_by_a_product(stub, page):
    """slot = group / (page / 16) by a 32-bit product, for all groups that a table can have."""
    m = min(((1 << 40) - 1) // page // page, ((1 << 31) - (1 << 16)) // page)
    a = attention_args(page=page, m=m)
    assert attention(stub, a) == OK
    magic, per = stub.stub_value(b"page_magic"), page // 16
    groups = m * per
    for g in {0, 1, per - 1, per, per + 1, groups // 2, groups - 1, groups - per, (groups - 1) // per * per, 12345 % groups}:
        if 0 <= g < groups:
            assert (g if magic == 0 else g * magic >> 32) == g // per, (g, per)


def test_sizes_of_parameter_blocks():
    assert C.sizeof(capi.QkNormParams) == 40 and (capi.QkNormParams.adjacent.offset, capi.QkNormParams.eps.offset, capi.QkNormParams.stream.offset) == (20, 24, 32)
    assert C.sizeof(capi.CacheAppendParams) == 32 and (capi.CacheAppendParams.adjacent.offset, capi.CacheAppendParams.stream.offset) == (20, 24)


def test_before_initialisation():
    lib = capi.lib()
    lib.tracea_shutdown()
    a = attention_args()
    st = lib.tracea_attention_cached(val(a["q"]), val(a["kc"]), val(a["vc"]), ref(a["ks"]), ref(a["vs"]), val(a["pt"]), None, val(a["kl"]), ref(a["o"]), None,
                                     capi.AttentionParams())
    assert st == capi.UNKNOWN_ERROR and "tracea_init" in capi.last_error()


def test_sections_are_checked_in_python():
    import torch
    from tracea_amd import ops
    q, freq, pos = torch.zeros(1, 1, 1, 8), torch.ones(4), torch.zeros(1, 1, 5, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, None, None, None, pos, freq, sections=[1, 1, 1, 1, 0])
    with pytest.raises(ValueError):
        ops.cache_append(q, q, q, q, pos, pos, inv_freq=freq, sections=[5, -1])
