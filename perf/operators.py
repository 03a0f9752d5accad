"""Timed cases of the operators that a trainable attention block over image, video or text tokens is made of.

``attention_forward`` keeps the statistics that ``attention_backward`` recomputes the probabilities from, ``rotary`` turns
queries and keys by their positions on several axes (and turns gradients back), ``norm_gate_residual`` joins two blocks:
norm of a block's result, gate, residual sum, norm of what the next block reads.  ``run`` computes one pass, in plain torch
or, with ``own`` set, by ``tracea_amd.ops``.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one new token for each of eight sequences over what they have kept so far: sampling from a model in training.
        # Heads shared four ways; bound by reading keys and values once.
        {"name": "attn_fwd_one_token", "kind": "attn_fwd", "b": 8, "hq": 32, "hk": 8, "sq": 1, "sk": 8192, "d": 128, "causal": True,
         "ragged": True, "dtype": "bf16", "layout": "bhsd"},
        # the forward half of a training step on text: shared heads, heads interleaved as a projection leaves them
        {"name": "attn_fwd_causal", "kind": "attn_fwd", "b": 2, "hq": 32, "hk": 8, "sq": 2048, "sk": 2048, "d": 128, "causal": True,
         "ragged": False, "dtype": "bf16", "layout": "bshd"},
        # one image of 14x14 patches and its class token: latency
        {"name": "attn_bwd_197", "kind": "attn_bwd", "b": 1, "hq": 12, "hk": 12, "sq": 197, "sk": 197, "d": 64, "causal": False,
         "ragged": False, "dtype": "f16", "layout": "bshd"},
        # the benchmark's short causal attention, one sequence: few workgroups
        {"name": "attn_bwd_s1024_causal", "kind": "attn_bwd", "b": 1, "hq": 12, "hk": 12, "sq": 1024, "sk": 1024, "d": 64, "causal": True,
         "ragged": False, "dtype": "f16", "layout": "bhsd"},
        # a padded batch of sequences of several lengths, shared heads, a head dimension between the kernels' two
        {"name": "attn_bwd_ragged_d96", "kind": "attn_bwd", "b": 4, "hq": 16, "hk": 4, "sq": 1500, "sk": 1500, "d": 96, "causal": True,
         "ragged": True, "dtype": "bf16", "layout": "bshd"},
        # the benchmark's attention, the largest case here
        {"name": "attn_bwd_s4096", "kind": "attn_bwd", "b": 4, "hq": 32, "hk": 32, "sq": 4096, "sk": 4096, "d": 128, "causal": False,
         "ragged": False, "dtype": "bf16", "layout": "bhsd"},
        # queries and keys of a video of 16 frames of 30x52 patches
        {"name": "rotary_video", "kind": "rotary", "b": 1, "hq": 32, "hk": 8, "axes": 3, "n0": 16, "n1": 30, "n2": 52, "d": 128, "rot": 128,
         "adjacent": False, "inverse": False, "dtype": "bf16", "layout": "bshd"},
        # gradients of the queries and keys of eight images of 32x32 patches, in 32 bits, pairs side by side, a quarter of a head not turned
        {"name": "rotary_image_grad_f32", "kind": "rotary", "b": 8, "hq": 12, "hk": 12, "axes": 2, "n0": 32, "n1": 32, "n2": 1, "d": 64, "rot": 48,
         "adjacent": True, "inverse": True, "dtype": "f32", "layout": "bhsd"},
        # one new token for each of sixteen sequences: latency
        {"name": "norm_fwd_one_token", "kind": "norm_fwd", "b": 16, "t": 1, "c": 4096, "gates": 1, "scale": 1.0, "dtype": "bf16"},
        # eight images of 1024 patches, each with a gate of its own (the image's condition sets it)
        {"name": "norm_fwd_image", "kind": "norm_fwd", "b": 8, "t": 1024, "c": 1152, "gates": 8, "scale": 1.0, "dtype": "f16"},
        # an odd width and an odd number of rows in 32 bits, one gate for all, residual scaled down
        {"name": "norm_bwd_odd_f32", "kind": "norm_bwd", "b": 3, "t": 333, "c": 1001, "gates": 1, "scale": 0.7, "dtype": "f32"},
        # the tokens of that video, four times as many channels as the convolutions' widest: bound by memory
        {"name": "norm_bwd_video", "kind": "norm_bwd", "b": 1, "t": 24960, "c": 2048, "gates": 1, "scale": 1.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_PAIRS = 4 * 32 * 4096 * 4096 * 128  # batch * heads * queries * keys * head dimension of the largest listed case


def draw(rng):
    kind = rng.choice(["attn_fwd", "attn_fwd", "attn_bwd", "attn_bwd", "attn_bwd", "rotary", "rotary", "norm_fwd", "norm_bwd", "norm_bwd"])
    half = rng.choice(["f16", "bf16", "bf16"])
    any_type = rng.choice(["f16", "bf16", "bf16", "f32"])
    layout = rng.choice(["bhsd", "bshd"])
    if kind in ("attn_fwd", "attn_bwd"):
        hq, hk = rng.choice([(4, 4), (12, 12), (32, 32), (32, 8), (16, 2), (6, 2), (10, 1), (28, 4)])
        b, d = _log(rng, 1, 8), rng.choice([64, 64, 128, 128, 128, 96, 80, 32, 40, 72, 112])
        if kind == "attn_fwd" and rng.random() < 0.4:
            sq, sk = rng.choice([1, 1, 2, 5]), _log(rng, 64, 32768)
        else:
            sq = _log(rng, 16, 4096)
            sk = sq if rng.random() < 0.7 else _log(rng, 16, 4096)
        while b > 1 and b * hq * sq * sk * d > _MOST_PAIRS:
            b -= 1
        return {"kind": kind, "b": b, "hq": hq, "hk": hk, "sq": sq, "sk": sk, "d": d, "causal": rng.random() < 0.5,
                "ragged": rng.random() < 0.4, "dtype": half, "layout": layout}
    if kind == "rotary":
        axes = rng.choice([1, 2, 3])
        n = [_log(rng, 1, 4096), 1, 1] if axes == 1 else [_log(rng, 4, 96), _log(rng, 4, 96), 1] if axes == 2 else [_log(rng, 2, 16), _log(rng, 4, 48), _log(rng, 4, 48)]
        hq, hk = rng.choice([(12, 12), (32, 32), (32, 8), (16, 2), (10, 1)])
        d = rng.choice([64, 128, 96, 80, 40])
        rot = d if rng.random() < 0.7 else d // 4 * 2
        b = _log(rng, 1, 8)
        while b > 1 and b * n[0] * n[1] * n[2] * (hq + hk) * d > 1 << 28:
            b -= 1
        return {"kind": "rotary", "b": b, "hq": hq, "hk": hk, "axes": axes, "n0": n[0], "n1": n[1], "n2": n[2], "d": d, "rot": rot,
                "adjacent": rng.random() < 0.5, "inverse": rng.random() < 0.5, "dtype": any_type, "layout": layout}
    c = _log(rng, 64, 8192)
    c = c if rng.random() < 0.3 else max(64, c // 64 * 64)
    b, t = _log(rng, 1, 16), _log(rng, 1, 8192)
    while b > 1 and b * t * c > 1 << 27:
        b -= 1
    while b * t * c > 1 << 27:
        t //= 2
    return {"kind": kind, "b": b, "t": t, "c": c, "gates": rng.choice([1, b]), "scale": rng.choice([1.0, 0.5]), "dtype": any_type}


def _lengths(case, rows, g):
    """Lengths of the sequences of a padded batch: the first fills its rows, the others between a quarter of them and all."""
    part = 0.25 + 0.75 * torch.rand(case["b"], generator=g)
    n = (part * rows).ceil().clamp(1, rows).to(torch.int32)
    n[0] = rows
    return n


def prepare(case, seed):
    c = case
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dt = _TYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dt)

    def heads(h, n):
        return normal(c["b"], h, n, c["d"]) if c["layout"] == "bhsd" else normal(c["b"], n, h, c["d"]).transpose(1, 2)

    s = {"case": c}
    if c["kind"] in ("attn_fwd", "attn_bwd"):
        s["q"], s["k"], s["v"] = heads(c["hq"], c["sq"]), heads(c["hk"], c["sk"]), heads(c["hk"], c["sk"])
        lk = _lengths(c, c["sk"], host) if c["ragged"] else None
        # self-attention: one length for both; else the queries are all there
        lq = lk if c["ragged"] and c["sq"] == c["sk"] else None
        s["q_lengths"] = None if lq is None else lq.to(dev)
        s["k_lengths"] = None if lk is None else lk.to(dev)
        if c["kind"] == "attn_bwd":
            s["do"] = heads(c["hq"], c["sq"])
            s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty(c["b"], c["hq"], c["sq"], device=dev)
            for i in range(c["b"]):  # what the forward pass left, sequence by sequence: a batch's scores would fill much of the card
                one = {n: t if t is None else t[i:i + 1] for n, t in s.items() if n in ("q", "k", "v", "q_lengths", "k_lengths")}
                o, s["lse"][i:i + 1] = _attn_fwd({**one, "case": {**c, "b": 1}})
                s["o"][i:i + 1] = o
    elif c["kind"] == "rotary":
        n = c["n0"] * c["n1"] * c["n2"]
        s["q"], s["k"] = heads(c["hq"], n), heads(c["hk"], n)
        grid = torch.meshgrid(*[torch.arange(c["n%d" % a], device=dev, dtype=torch.int32) for a in range(c["axes"])], indexing="ij")
        first = torch.randint(0, 64, (c["b"], 1, c["axes"]), generator=host, dtype=torch.int32).to(dev)  # where a crop begins
        s["positions"] = (torch.stack([p.reshape(-1) for p in grid], dim=-1)[None] + first).contiguous()
        pairs = c["rot"] // 2
        s["sections"] = [pairs // c["axes"] + (a < pairs % c["axes"]) for a in range(c["axes"])]
        s["axis"] = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(s["sections"])).to(dev)  # of each pair
        s["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(m, device=dev, dtype=torch.float32) / m) for m in s["sections"]])
    else:
        b, t, ch = c["b"], c["t"], c["c"]
        s["h"], s["x"] = normal(b, t, ch, scale=0.5), normal(b, t, ch, scale=2.0)
        s["w_post"] = 1.0 + 0.1 * torch.randn(ch, device=dev, generator=g)
        s["w_pre"] = 1.0 + 0.1 * torch.randn(ch, device=dev, generator=g)
        s["gate"] = 0.3 * torch.randn(c["gates"], ch, device=dev, generator=g)
        if c["kind"] == "norm_bwd":
            s["x_out"] = s.pop("x")
            s["dx_out"], s["dy"] = normal(b, t, ch), normal(b, t, ch)
    return s


def _visible(c, lq, lk, dev):
    """[B,1,1,Sq,Sk]: which keys a query sees."""
    i, j = torch.arange(c["sq"], device=dev)[:, None], torch.arange(c["sk"], device=dev)[None]
    lq = torch.full((c["b"],), c["sq"], device=dev) if lq is None else lq
    lk = torch.full((c["b"],), c["sk"], device=dev) if lk is None else lk
    lq, lk = lq.view(-1, 1, 1), lk.view(-1, 1, 1)
    seen = (i < lq) & (j < lk)
    if c["causal"]:
        seen = seen & (j <= i + lk - lq)
    return seen[:, None, None]


def _scores(s):
    """Scaled scores [B,Hk,G,Sq,Sk], -inf where a key is not seen, and the inputs in 32 bits with the heads that share keys in one axis."""
    c = s["case"]
    b, hk, gr, sq, sk, d = c["b"], c["hk"], c["hq"] // c["hk"], c["sq"], c["sk"], c["d"]
    q = s["q"].float().reshape(b, hk, gr * sq, d)
    k, v = s["k"].float(), s["v"].float()
    x = torch.matmul(q, k.transpose(-1, -2)).view(b, hk, gr, sq, sk) * d ** -0.5
    x = x.masked_fill(~_visible(c, s["q_lengths"], s["k_lengths"], x.device), -math.inf)
    return x, q, k, v


def _softmax(x):
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total)), top + total.log()


def _attn_fwd(s):
    c = s["case"]
    x, _, _, v = _scores(s)
    p, lse = _softmax(x)
    o = torch.matmul(p.view(c["b"], c["hk"], -1, c["sk"]), v).view(c["b"], c["hq"], c["sq"], c["d"])
    return o.to(s["q"].dtype), lse.view(c["b"], c["hq"], c["sq"])


def _attn_bwd(s):
    c = s["case"]
    dt = s["q"].dtype
    x, q, k, v = _scores(s)
    p, _ = _softmax(x)
    del x
    p = p.view(c["b"], c["hk"], -1, c["sk"])
    do = s["do"].float().reshape(q.shape)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * c["d"] ** -0.5
    dk = torch.matmul(ds.transpose(-1, -2), q) * c["d"] ** -0.5
    return dq.view(s["q"].shape).to(dt), dk.to(dt), dv.to(dt)


def _rotary_one(x, cos, sin, rot, adjacent):
    y = x.float()
    u, v = (y[..., 0:rot:2], y[..., 1:rot:2]) if adjacent else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = u * cos - v * sin, v * cos + u * sin
    turned = torch.stack([a, b], -1).flatten(-2) if adjacent else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    angle = s["positions"].float()[..., s["axis"]] * s["inv_freq"]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None] * (-1.0 if c["inverse"] else 1.0)
    return tuple(_rotary_one(t, cos, sin, c["rot"], c["adjacent"]) for t in (s["q"], s["k"]))


_EPS = 1e-6


def _norm_fwd(s):
    c = s["case"]
    dt = s["x"].dtype
    h, x = s["h"].float(), s["x"].float()
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * s["w_post"]
    x = c["scale"] * x + s["gate"][:, None] * n
    return x.to(dt), (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * s["w_pre"]).to(dt)


def _norm_bwd(s):
    c = s["case"]
    dt = s["h"].dtype
    h, x, dx_out, dy = s["h"].float(), s["x_out"].float(), s["dx_out"].float(), s["dy"].float()
    w, gate = s["w_post"], s["gate"][:, None]
    r2 = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xn, g = x * r2, dy * s["w_pre"]
    dt_x = dx_out + r2 * (g - xn * (g * xn).mean(-1, keepdim=True))
    r1 = torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
    hn = h * r1
    a = dt_x * gate * w
    dh = r1 * (a - hn * (a * hn).mean(-1, keepdim=True))
    by_batch = (dt_x * hn).sum(1)
    dgate = by_batch if c["gates"] == c["b"] else by_batch.sum(0, keepdim=True)
    return ((c["scale"] * dt_x).to(dt), dh.to(dt), (by_batch * s["gate"]).sum(0), dgate * w, (dy * xn).sum((0, 1)))


def _run_own(s):
    from tracea_amd import capi, ops
    capi.init()
    c = s["case"]
    if c["kind"] == "attn_fwd":
        return ops.attention_forward(s["q"], s["k"], s["v"], causal=c["causal"], q_lengths=s["q_lengths"], k_lengths=s["k_lengths"])
    if c["kind"] == "attn_bwd":
        return ops.attention_backward(s["q"], s["k"], s["v"], s["o"], s["lse"], s["do"], causal=c["causal"],
                                      q_lengths=s["q_lengths"], k_lengths=s["k_lengths"])
    if c["kind"] == "rotary":
        return ops.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], sections=s["sections"], adjacent=c["adjacent"], inverse=c["inverse"])
    if c["kind"] == "norm_fwd":
        return ops.norm_gate_residual(s["x"], s["h"], s["w_post"], s["gate"], s["w_pre"], residual_scale=c["scale"], eps=_EPS)
    return ops.norm_gate_residual_backward(s["dx_out"], s["dy"], s["x_out"], s["h"], s["w_post"], s["gate"], s["w_pre"],
                                           residual_scale=c["scale"], eps=_EPS)


_PLAIN = {"attn_fwd": _attn_fwd, "attn_bwd": _attn_bwd, "rotary": _rotary, "norm_fwd": _norm_fwd, "norm_bwd": _norm_bwd}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state)


def _pairs(c):
    """Visible (query, key) pairs of one head over the batch, as the listed lengths have them on average."""
    def of(lq, lk):
        if not c["causal"]:
            return float(lq) * lk
        rows = min(lq, lk)  # the last `rows` queries see lk - rows + 1 .. lk keys
        return rows * (2.0 * lk - rows + 1) / 2
    whole = of(c["sq"], c["sk"])
    if not c["ragged"]:
        return c["b"] * whole
    part = 0.625
    return whole + (c["b"] - 1) * of(c["sq"] * part if c["sq"] == c["sk"] else c["sq"], c["sk"] * part)


def work(case):
    c = case
    e = _BYTES[c["dtype"]]
    if c["kind"] in ("attn_fwd", "attn_bwd"):
        fill = (1 + (c["b"] - 1) * 0.625) / c["b"] if c["ragged"] else 1.0  # of the rows, those that a sequence has
        rows_q = c["b"] * c["hq"] * c["sq"] * (fill if c["sq"] == c["sk"] else 1.0)
        rows_k = c["b"] * c["hk"] * c["sk"] * fill
        out_q, out_k = c["b"] * c["hq"] * c["sq"], c["b"] * c["hk"] * c["sk"]
        flops = c["hq"] * c["d"] * _pairs(c)
        if c["kind"] == "attn_fwd":
            return {"bytes": e * c["d"] * (rows_q + 2 * rows_k + out_q) + 4 * out_q, "flops": 4 * flops}
        return {"bytes": e * c["d"] * (3 * rows_q + 2 * rows_k + out_q + 2 * out_k) + 4 * rows_q, "flops": 10 * flops}
    if c["kind"] == "rotary":
        n = c["b"] * c["n0"] * c["n1"] * c["n2"]
        return {"bytes": 2 * e * n * (c["hq"] + c["hk"]) * c["d"] + 4 * n * c["axes"] + 2 * c["rot"], "flops": 3.0 * n * (c["hq"] + c["hk"]) * c["rot"]}
    n = c["b"] * c["t"] * c["c"]
    if c["kind"] == "norm_fwd":
        return {"bytes": 4 * e * n + 4 * c["c"] * (2 + c["gates"]), "flops": 10.0 * n}
    return {"bytes": 6 * e * n + 8 * c["c"] * (2 + c["gates"]), "flops": 24.0 * n}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------------------------

def _exact_attention(s, backward):
    """Sequence by sequence and head by head on the rows and keys that there are; gradients by differentiating the definition."""
    c = s["case"]
    dev, per = s["q"].device, c["hq"] // c["hk"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device=dev)
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device=dev) for n in "qkv")
    for b in range(c["b"]):
        lq = c["sq"] if s["q_lengths"] is None else int(s["q_lengths"][b])
        lk = c["sk"] if s["k_lengths"] is None else int(s["k_lengths"][b])
        first = max(0, lq - lk) if c["causal"] else 0  # the first query that sees a key
        hidden = torch.arange(lk, device=dev)[None] > torch.arange(first, lq, device=dev)[:, None] + (lk - lq) if c["causal"] else None
        for h in range(c["hq"]):
            q, k, v = (t.double().requires_grad_(backward) for t in (s["q"][b, h, first:lq], s["k"][b, h // per, :lk], s["v"][b, h // per, :lk]))
            x = (q @ k.t()) / math.sqrt(c["d"])
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            if not backward:
                o[b, h, first:lq], lse[b, h, first:lq] = torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)
                continue
            grads = torch.autograd.grad(torch.softmax(x, -1) @ v, (q, k, v), s["do"][b, h, first:lq].double())
            dq[b, h, first:lq] = grads[0]
            dk[b, h // per, :lk] += grads[1]
            dv[b, h // per, :lk] += grads[2]
    return (dq, dk, dv) if backward else (o, lse)


def _exact_rotary(s):
    c = s["case"]
    outs = []
    freq, pos = s["inv_freq"].double(), s["positions"].double()
    start = [sum(s["sections"][:a]) for a in range(c["axes"] + 1)]
    angle = torch.cat([pos[..., a:a + 1] * freq[start[a]:start[a + 1]] for a in range(c["axes"])], -1)
    turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)[:, None]
    for t in (s["q"], s["k"]):
        y = t.double().clone()
        re, im = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["adjacent"] else (slice(0, c["rot"] // 2), slice(c["rot"] // 2, c["rot"]))
        z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * turn
        y[..., re], y[..., im] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_norm(s, backward):
    c = s["case"]

    def rms_norm(t, w):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + _EPS) * w

    w_post, w_pre, gate, h = (s[n].double().requires_grad_(backward) for n in ("w_post", "w_pre", "gate", "h"))
    added = gate[:, None] * rms_norm(h, w_post)
    if not backward:
        x = c["scale"] * s["x"].double() + added
        return x, rms_norm(x, w_pre)
    x = s["x_out"].double().requires_grad_(True)  # the sum as the forward pass stored it
    through, dw_pre = torch.autograd.grad(rms_norm(x, w_pre), (x, w_pre), s["dy"].double())
    total = s["dx_out"].double() + through
    dh, dw_post, dgate = torch.autograd.grad(added, (h, w_post, gate), total)
    return c["scale"] * total, dh, dw_post, dgate, dw_pre


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attn_fwd", "attn_bwd"):
        return _exact_attention(s, kind == "attn_bwd")
    if kind == "rotary":
        return _exact_rotary(s)
    return _exact_norm(s, kind == "norm_bwd")
