"""Buffers that the operators for training keep per stream: whose they are, what two threads see, what a stream under capture gets."""
import ctypes as C
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def new_stream():
    """A stream that no call has been made on."""
    from tracea_amd import capi
    handle = C.c_void_p()
    assert capi.lib().hipStreamCreate(C.byref(handle)) == 0
    return torch.cuda.ExternalStream(handle.value)


def make(*shapes, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, device="cuda", generator=g).to(dtype) for s in shapes]


def under_capture(stream, call):
    """What `call` returns or raises on `stream` under capture, and the graph."""
    from tracea_amd import capi
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    result = None
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            try:
                result = call()
            except capi.TraceaError as e:
                result = e
    return result, graph


def test_copies_are_not_in_the_buffer_of_other_operators(tracea_gpu):
    """A stream on which a GEMM has made its padded copies has no buffer for those of attention yet: under capture, where none can be
    allocated, the call is refused instead of writing over the GEMM's."""
    from tracea_amd import capi
    a, b = make((333, 4099), (4099, 65))
    q, k, v = make((2, 2, 40, 50), (2, 2, 40, 50), (2, 2, 40, 50))
    out, lse = torch.empty_like(q), torch.empty(2, 2, 40, device="cuda")
    stream = new_stream()
    with torch.cuda.stream(stream):
        tracea_gpu.gemm(a.t().contiguous().t(), b)  # strided along K: from copies
        torch.cuda.synchronize()
    result, _ = under_capture(stream, lambda: tracea_gpu.attention_forward(q, k, v, out=out, lse=lse))
    assert isinstance(result, capi.TraceaError) and result.status == capi.UNSUPPORTED_CONFIG, result


def test_two_threads_on_one_stream(tracea_gpu):
    """Attention and a GEMM, both from copies of their operands, in two threads on the default stream."""
    a, b = make((333, 1031), (1031, 265), seed=1)
    a = a.t().contiguous().t()
    q, k, v, do = make(*[(2, 4, 130, 50)] * 4, seed=2)

    def attend():
        o, lse = tracea_gpu.attention_forward(q, k, v, causal=True)
        return (o, lse) + tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True)

    def multiply():
        return (tracea_gpu.gemm(a, b),)
    want = {f: f() for f in (attend, multiply)}
    torch.cuda.synchronize()
    got, errors = {attend: [], multiply: []}, []

    def run(f):
        try:
            for _ in range(100):
                got[f].append(f())
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)
    threads = [threading.Thread(target=run, args=(f,)) for f in got]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for f in got:
        for results in got[f]:
            for x, y in zip(results, want[f]):
                assert torch.equal(x, y)


def test_the_parts_of_one_query_take_its_rows(tracea_gpu):
    """One query of 40 heads (8 key heads) over 32768 keys: the partial results of 32 parts at most are 32 x 40 rows of 130 numbers, not of
    as many as a tile has."""
    from helpers import launches
    q, k, v = make((1, 40, 1, 128), (1, 8, 32768, 128), (1, 8, 32768, 128), seed=3)
    out, lse = torch.empty_like(q), torch.empty(1, 40, 1, device="cuda")

    def call():
        tracea_gpu.attention_forward(q, k, v, out=out, lse=lse)
    assert launches(call) == 2  # (the kernels are loaded, too)
    stream = new_stream()
    with torch.cuda.stream(stream):
        out.zero_()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] <= 2 << 20  # (at least 1 MiB by the rule of these buffers, in the device's pieces of 2)


def test_under_capture_without_a_workspace(tracea_gpu):
    """On a stream that has made no such call: the forward pass runs unsplit, the backward passes, which cannot do without, are refused."""
    from helpers import launches
    from test_attention_train_gpu import reference, within
    from tracea_amd import capi
    q, k, v, do = make((1, 8, 2, 64), (1, 2, 5000, 64), (1, 2, 5000, 64), (1, 8, 2, 64), seed=4)
    want = reference(q, k, v, do, True, 0.0)
    o, lse = torch.empty_like(q), torch.empty(1, 8, 2, device="cuda")
    assert launches(lambda: tracea_gpu.attention_forward(q, k, v, causal=True, out=o, lse=lse)) == 2  # split where there is a workspace
    stream = new_stream()
    _, graph = under_capture(stream, lambda: tracea_gpu.attention_forward(q, k, v, causal=True, out=o, lse=lse))
    for _ in range(3):
        o.fill_(float("nan"))
        lse.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        within("o", o, want["o"])
        within("lse", lse, want["lse"])
    grads = [torch.empty_like(t) for t in (q, k, v)]
    result, _ = under_capture(stream, lambda: tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True, dq=grads[0], dk=grads[1],
                                                                            dv=grads[2]))
    assert isinstance(result, capi.TraceaError) and result.status == capi.UNSUPPORTED_CONFIG, result
    x, h, dx, dy = make(*[(2, 9, 64)] * 4, dtype=torch.float32, seed=5)
    w = torch.ones(64, device="cuda")
    result, _ = under_capture(stream, lambda: tracea_gpu.norm_gate_residual_backward(dx, dy, x, h, w, None, w, dx=torch.empty_like(x),
                                                                                     dh=torch.empty_like(x)))
    assert isinstance(result, capi.TraceaError) and result.status == capi.UNSUPPORTED_CONFIG, result
    with torch.cuda.stream(stream):  # and eagerly they have one
        tracea_gpu.attention_backward(q, k, v, o, lse, do, causal=True, dq=grads[0], dk=grads[1], dv=grads[2])
        torch.cuda.synchronize()
    for name, t in zip(("dq", "dk", "dv"), grads):
        within(name, t, want[name])
