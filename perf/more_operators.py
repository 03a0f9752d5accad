"""Timed cases of the operators that attention with a key/value cache is made of.

``qk_norm_rotary`` norms every head of queries and keys and turns it by its position in one pass (and takes gradients back through
both), ``cache_append`` turns new keys and writes them and their values into the pages of a cache, in 16 bits or in 8 with a
scale for each page and head, ``attention_cached`` reads such a cache for one query of a sequence or for many.  ``run`` computes one
pass, in plain torch or, with ``own`` set, by ``tracea_amd.ops``.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_E4M3 = torch.float8_e4m3fn
_EPS = 1e-6


def listed():
    return [
        # one image's class token over its 14x14 patches, a cache of 16 bits: latency
        {"name": "cached_one_token_197", "kind": "attn", "b": 1, "hq": 12, "hk": 12, "sq": 1, "sk": 197, "d": 64, "page": 16, "causal": True,
         "ragged": False, "dtype": "f16", "cache": "16", "layout": "bshd"},
        # one new token for each of eight sequences over what they have kept so far in 8 bits: bound by reading the cache
        {"name": "cached_one_token_8bit", "kind": "attn", "b": 8, "hq": 32, "hk": 8, "sq": 1, "sk": 8192, "d": 128, "page": 64, "causal": True,
         "ragged": True, "dtype": "bf16", "cache": "e4m3", "layout": "bshd"},
        # one sequence with a very long cache: the keys have to be split
        {"name": "cached_long_8bit", "kind": "attn", "b": 1, "hq": 40, "hk": 8, "sq": 1, "sk": 131072, "d": 128, "page": 128, "causal": True,
         "ragged": False, "dtype": "bf16", "cache": "e4m3", "layout": "bhsd"},
        # five drafted tokens for each of sixteen sequences, a cache of 16 bits, a head dimension between the powers of two
        {"name": "cached_five_tokens", "kind": "attn", "b": 16, "hq": 16, "hk": 4, "sq": 5, "sk": 2000, "d": 96, "page": 16, "causal": True,
         "ragged": True, "dtype": "f16", "cache": "16", "layout": "bshd"},
        # a piece of a long prompt for two sequences behind what the cache holds of them: bound by the products
        {"name": "cached_prompt_8bit", "kind": "attn", "b": 2, "hq": 32, "hk": 8, "sq": 1024, "sk": 8192, "d": 128, "page": 64, "causal": True,
         "ragged": True, "dtype": "bf16", "cache": "e4m3", "layout": "bshd"},
        # the new token's queries, keys and values of sixteen sequences: latency
        {"name": "append_one_token", "kind": "append", "b": 16, "hq": 32, "hk": 8, "t": 1, "start": 1000, "d": 128, "rot": 128, "page": 64,
         "adjacent": False, "ragged": True, "dtype": "bf16", "cache": "e4m3", "layout": "bshd"},
        # two whole prompts: bound by memory
        {"name": "append_prompt_8bit", "kind": "append", "b": 2, "hq": 32, "hk": 8, "t": 4096, "start": 0, "d": 128, "rot": 128, "page": 64,
         "adjacent": False, "ragged": False, "dtype": "bf16", "cache": "e4m3", "layout": "bshd"},
        # pieces of odd lengths that begin inside a page, a cache of 16 bits, pairs side by side, part of a head not turned
        {"name": "append_odd_16bit", "kind": "append", "b": 3, "hq": 10, "hk": 2, "t": 777, "start": 300, "d": 80, "rot": 48, "page": 16,
         "adjacent": True, "ragged": True, "dtype": "f16", "cache": "16", "layout": "bhsd"},
        # one new token for each of sixteen sequences: latency
        {"name": "qk_fwd_one_token", "kind": "qk_fwd", "b": 16, "hq": 32, "hk": 8, "axes": 1, "n0": 1, "n1": 1, "n2": 1, "d": 128, "rot": 128,
         "adjacent": False, "dtype": "bf16", "layout": "bshd"},
        # queries and keys of a video of 16 frames of 30x52 patches: bound by memory
        {"name": "qk_fwd_video", "kind": "qk_fwd", "b": 1, "hq": 32, "hk": 8, "axes": 3, "n0": 16, "n1": 30, "n2": 52, "d": 128, "rot": 128,
         "adjacent": False, "dtype": "bf16", "layout": "bshd"},
        # the gradients of a training step on text
        {"name": "qk_bwd_text", "kind": "qk_bwd", "b": 4, "hq": 32, "hk": 8, "axes": 1, "n0": 2048, "n1": 1, "n2": 1, "d": 128, "rot": 128,
         "adjacent": False, "dtype": "bf16", "layout": "bshd"},
        # the gradients of images of an odd number of patches, in 32 bits, pairs side by side, part of a head not turned
        {"name": "qk_bwd_image_f32", "kind": "qk_bwd", "b": 3, "hq": 12, "hk": 12, "axes": 2, "n0": 19, "n1": 27, "n2": 1, "d": 64, "rot": 48,
         "adjacent": True, "dtype": "f32", "layout": "bhsd"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_PAIRS = 2 * 32 * 1024 * 8192 * 128   # batch * heads * queries * keys * head dimension of the largest listed case
_MOST_CACHE = 131072 * 8 * 128             # values of one cache of the largest
_MOST_ROWS = 24960 * 40 * 128              # values of queries and keys of the largest


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "append", "append", "append", "qk_fwd", "qk_fwd", "qk_bwd", "qk_bwd"])
    half = rng.choice(["f16", "bf16", "bf16"])
    layout = rng.choice(["bhsd", "bshd"])
    hq, hk = rng.choice([(4, 4), (12, 12), (32, 32), (32, 8), (16, 2), (6, 2), (10, 1), (28, 4)])
    if kind == "attn":
        d = rng.choice([64, 64, 128, 128, 128, 96, 80, 32, 40, 72, 112])
        b = _log(rng, 1, 32)
        sq = rng.choice([1, 1, 1, 1, 2, 5, 8]) if rng.random() < 0.65 else _log(rng, 9, 1500)
        sk = max(sq, _log(rng, 16, 65536))
        while b > 1 and (b * hq * sq * sk * d > _MOST_PAIRS or b * sk * hk * d > _MOST_CACHE):
            b = (b + 1) // 2
        while sk > sq and (b * hq * sq * sk * d > _MOST_PAIRS or b * sk * hk * d > _MOST_CACHE):
            sk = max(sq, sk // 2)
        return {"kind": kind, "b": b, "hq": hq, "hk": hk, "sq": sq, "sk": sk, "d": d, "page": rng.choice([16, 16, 32, 48, 64, 64, 128, 256]),
                "causal": rng.random() < 0.8, "ragged": rng.random() < 0.6, "dtype": half, "cache": rng.choice(["16", "e4m3"]), "layout": layout}
    if kind == "append":
        d = rng.choice([64, 128, 128, 128, 96, 80, 40])
        b, start = _log(rng, 1, 32), rng.choice([0, _log(rng, 1, 2000)])
        t = rng.choice([1, 1, 2, 5]) if rng.random() < 0.5 else _log(rng, 6, 4096)
        while b > 1 and b * (t + start) * (hq + 2 * hk) * d > _MOST_ROWS:
            b = (b + 1) // 2
        return {"kind": kind, "b": b, "hq": rng.choice([0, hq, hq]), "hk": hk, "t": t, "start": start, "d": d, "rot": d if rng.random() < 0.7 else d // 4 * 2,
                "page": rng.choice([16, 16, 32, 48, 64, 64, 128, 256]), "adjacent": rng.random() < 0.4, "ragged": rng.random() < 0.6, "dtype": half,
                "cache": rng.choice(["16", "e4m3", "e4m3"]), "layout": layout}
    axes = rng.choice([1, 1, 2, 3])
    n = [_log(rng, 1, 4096), 1, 1] if axes == 1 else [_log(rng, 4, 96), _log(rng, 4, 96), 1] if axes == 2 else [_log(rng, 2, 16), _log(rng, 4, 48), _log(rng, 4, 48)]
    d = rng.choice([64, 128, 128, 96, 80, 40])
    b = _log(rng, 1, 8)
    while b > 1 and b * n[0] * n[1] * n[2] * (hq + hk) * d > _MOST_ROWS:
        b -= 1
    while b * n[0] * n[1] * n[2] * (hq + hk) * d > _MOST_ROWS:
        n[0] = (n[0] + 1) // 2
    return {"kind": kind, "b": b, "hq": hq, "hk": hk, "axes": axes, "n0": n[0], "n1": n[1], "n2": n[2], "d": d,
            "rot": d if rng.random() < 0.7 else d // 4 * 2, "adjacent": rng.random() < 0.5, "dtype": rng.choice(["f16", "bf16", "bf16", "f32"]), "layout": layout}


def _part(case, most, g):
    """Lengths of the sequences of a batch: the first has all there can be, the others between a quarter of it and all."""
    n = torch.full((case["b"],), most, dtype=torch.int32)
    if case["ragged"]:
        n = ((0.25 + 0.75 * torch.rand(case["b"], generator=g)) * most).ceil().clamp(min(1, most), most).to(torch.int32)
        n[0] = most
    return n


def _power_of_two_scale(largest):
    """The least power of two by which `largest` is at most 448, the largest e4m3 value (at least 2^-126)."""
    m, e = torch.frexp(largest)
    return torch.ldexp(torch.ones_like(largest), (e - 9 + (m > 0.875)).clamp(min=-126))


def _pages(s, rows, normal):
    """A pool of caches with pages enough for `rows` tokens of each sequence, in no order, all of them written."""
    c = s["case"]
    per = -(-rows // c["page"])
    s["page_table"] = torch.randperm(c["b"] * per + 3, generator=s["host"])[:c["b"] * per].to(torch.int32).view(c["b"], per).cuda()
    spread = torch.exp2(2.0 * normal(c["hk"], 1, c["d"]).float()).clamp(0.1, 6.0)  # some channels of the keys are far larger than others
    for name, by in (("k", spread), ("v", 1.0)):
        pool = normal(c["b"] * per + 3, c["hk"], c["page"], c["d"])
        pool = (pool * by).to(pool.dtype)
        s[name + "_scale"] = None
        if c["cache"] == "e4m3":
            scale = _power_of_two_scale(pool.abs().amax((2, 3)).float())
            s[name + "_scale"] = scale
            pool = (pool.float() / scale[:, :, None, None]).to(_E4M3)
        s[name + "_cache"] = pool


def prepare(case, seed):
    c = case
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dt = _TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=dt)

    def heads(h, n):
        return normal(c["b"], h, n, c["d"]) if c["layout"] == "bhsd" else normal(c["b"], n, h, c["d"]).transpose(1, 2)

    s = {"case": c, "host": host}
    if c["kind"] == "attn":
        s["q"] = heads(c["hq"], c["sq"])
        _pages(s, c["sk"], normal)
        s["k_lengths"] = _part(c, c["sk"], host).to(dev)
        s["q_lengths"] = _part(c, c["sq"], host).to(dev) if c["ragged"] and c["sq"] > 8 else None  # (a piece of a prompt; drafts are as long as each other)
        return s
    pairs = c["rot"] // 2
    if c["kind"] == "append":
        s["q"] = heads(c["hq"], c["t"]) if c["hq"] else None
        s["k"], s["v"] = heads(c["hk"], c["t"]), heads(c["hk"], c["t"])
        _pages(s, c["start"] + c["t"], normal)
        s["starts"] = _part(c, c["start"], host).to(dev)
        s["lengths"] = _part(c, c["t"], host).to(dev) if c["ragged"] and c["t"] > 8 else None
        s["inv_freq"] = 10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float32) / pairs)
        return s
    n = c["n0"] * c["n1"] * c["n2"]
    s["q"], s["k"] = heads(c["hq"], n), heads(c["hk"], n)
    s["q_weight"] = 1.0 + 0.2 * torch.randn(c["d"], device=dev, generator=g)
    s["k_weight"] = 1.0 + 0.2 * torch.randn(c["d"], device=dev, generator=g)
    grid = torch.meshgrid(*[torch.arange(c["n%d" % a], device=dev, dtype=torch.int32) for a in range(c["axes"])], indexing="ij")
    first = torch.randint(0, 64 if c["axes"] > 1 else 8192, (c["b"], 1, c["axes"]), generator=host, dtype=torch.int32).to(dev)
    s["positions"] = (torch.stack([p.reshape(-1) for p in grid], dim=-1)[None] + first).contiguous()
    s["sections"] = [pairs // c["axes"] + (a < pairs % c["axes"]) for a in range(c["axes"])]
    s["axis"] = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(s["sections"])).to(dev)  # of each pair
    s["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(m, device=dev, dtype=torch.float32) / m) for m in s["sections"]])
    if c["kind"] == "qk_bwd":
        s["dq_out"], s["dk_out"] = heads(c["hq"], n), heads(c["hk"], n)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _gathered(s, name):
    """[B,Hk,M*page,D] of a cache in 32 bits: every page that the table names, in its order."""
    pool, scale = s[name + "_cache"], s[name + "_scale"]
    table = s["page_table"].long()
    if scale is None:
        x = pool[table].float()
    else:
        x = pool.view(torch.uint8)[table].view(_E4M3).float() * scale[table][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attn(s):
    c = s["case"]
    b, hk, gr, sq, d = c["b"], c["hk"], c["hq"] // c["hk"], c["sq"], c["d"]
    k = _gathered(s, "k")
    x = torch.matmul(s["q"].float().reshape(b, hk, gr * sq, d), k.transpose(-1, -2)).view(b, hk, gr, sq, -1) * d ** -0.5
    del k
    i, j = torch.arange(sq, device=x.device)[:, None], torch.arange(x.shape[-1], device=x.device)[None]
    lk = s["k_lengths"].view(-1, 1, 1)
    lq = lk * 0 + sq if s["q_lengths"] is None else s["q_lengths"].view(-1, 1, 1)
    seen = (i < lq) & (j < lk)
    if c["causal"]:
        seen = seen & (j <= i + lk - lq)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = (x - torch.where(top > -math.inf, top, torch.zeros_like(top))).exp()
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(x.view(b, hk, gr * sq, -1), _gathered(s, "v"))
    return o.view(b, c["hq"], sq, d).to(s["q"].dtype)


def _turned(x, angle, rot, adjacent, sign=1.0):
    """x in 32 bits, [B,H,S,D], with its pairs turned by the angles [B,S,pairs] (in 64 bits)."""
    angle = torch.remainder(angle, 2.0 * math.pi)[:, None]
    cos, sin = angle.cos().float(), angle.sin().float() * sign
    u, v = (x[..., 0:rot:2], x[..., 1:rot:2]) if adjacent else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = u * cos - v * sin, v * cos + u * sin
    turned = torch.stack([a, b], -1).flatten(-2) if adjacent else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _append(s):
    c = s["case"]
    b, t, page = c["b"], c["t"], c["page"]
    start = s["starts"].long()
    n = torch.full_like(start, t) if s["lengths"] is None else s["lengths"].long()
    token = torch.arange(t, device=start.device)
    angle = (start[:, None] + token).double()[..., None] * s["inv_freq"].double()
    q = None
    if s["q"] is not None:
        q = _turned(s["q"].float(), angle, c["rot"], c["adjacent"])
        q = torch.where((token < n[:, None])[:, None, :, None], q, torch.zeros_like(q)).to(s["q"].dtype)
    # the pages that get tokens, [B,J] (the last of a sequence again where it has fewer), and the token of each of their places
    first, last = start // page, (start + n.clamp(min=1) - 1) // page
    at = torch.minimum(first[:, None] + torch.arange((t + page - 2) // page + 1, device=start.device), last[:, None])
    pages = s["page_table"].long().gather(1, at)
    here = at[..., None] * page + torch.arange(page, device=start.device) - start[:, None, None]  # [B,J,page]
    new = ((here >= 0) & (here < n[:, None, None]))[:, :, None, :, None]
    rows = here.clamp(0, t - 1).flatten(1)[:, None, :, None].expand(-1, c["hk"], -1, c["d"])
    for name, x in (("k", _turned(s["k"].float(), angle, c["rot"], c["adjacent"])), ("v", s["v"].float())):
        x = x.gather(2, rows).view(b, c["hk"], -1, page, c["d"]).transpose(1, 2)  # [B,J,Hk,page,D]
        pool, scale = s[name + "_cache"], s[name + "_scale"]
        if scale is None:
            pool[pages] = torch.where(new, x.to(pool.dtype), pool[pages])
            continue
        need = _power_of_two_scale(torch.where(new, x, torch.zeros_like(x)).abs().amax((3, 4)))
        old = torch.where((at * page >= start[:, None])[..., None], torch.zeros_like(need), scale[pages])  # (nothing in it before)
        now = torch.where(new.any(3).any(-1), torch.maximum(old, need), scale[pages])
        held = pool.view(torch.uint8)[pages].view(_E4M3).float()
        held = torch.where((now == scale[pages])[..., None, None] | (old == 0)[..., None, None], held, held * (old / now)[..., None, None])
        whole = torch.where(new, x / now[..., None, None], held).to(_E4M3)
        pool.view(torch.uint8)[pages] = whole.view(torch.uint8)
        scale[pages] = now
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], q


def _angles(s):
    return s["positions"].double()[..., s["axis"]] * s["inv_freq"].double()


def _qk_fwd(s):
    c, out = s["case"], []
    for name in ("q", "k"):
        x = s[name].float()
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * s[name + "_weight"]
        out.append(_turned(n, _angles(s), c["rot"], c["adjacent"]).to(s[name].dtype))
    return tuple(out)


def _qk_bwd(s):
    c, out, sums = s["case"], [], []
    for name in ("q", "k"):
        x = s[name].float()
        dn = _turned(s["d%s_out" % name].float(), _angles(s), c["rot"], c["adjacent"], -1.0)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        xn, g = x * r, dn * s[name + "_weight"]
        out.append((r * (g - xn * (g * xn).mean(-1, keepdim=True))).to(s[name].dtype))
        sums.append((dn * xn).sum((0, 1, 2)))
    return tuple(out + sums)


def _run_own(s):
    from tracea_amd import capi, ops
    capi.init()
    c = s["case"]
    if c["kind"] == "attn":
        return ops.attention_cached(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["k_lengths"], q_lengths=s["q_lengths"],
                                    causal=c["causal"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if c["kind"] == "append":
        q = ops.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["starts"], lengths=s["lengths"], k_scale=s["k_scale"],
                             v_scale=s["v_scale"], q=s["q"], inv_freq=s["inv_freq"], adjacent=c["adjacent"])
        # a cache of 8 bits as its own float8 values, in units of the scales beside it
        return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], q
    if c["kind"] == "qk_fwd":
        return ops.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], sections=s["sections"],
                                  adjacent=c["adjacent"], eps=_EPS)
    return ops.qk_norm_rotary_backward(s["dq_out"], s["dk_out"], s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"],
                                       sections=s["sections"], adjacent=c["adjacent"], eps=_EPS)


_PLAIN = {"attn": _attn, "append": _append, "qk_fwd": _qk_fwd, "qk_bwd": _qk_bwd}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    c = case
    e = _BYTES[c["dtype"]]
    fill = (1 + (c["b"] - 1) * 0.625) / c["b"] if c.get("ragged") else 1.0  # of the longest sequence, what a sequence has on average
    if c["kind"] == "attn":
        per_key = 1 if c["cache"] == "e4m3" else 2
        keys = c["sk"] * fill
        queries = c["sq"] * (fill if c["sq"] > 8 else 1.0)
        rows = min(queries, keys)
        pairs = rows * (2.0 * keys - rows + 1) / 2 if c["causal"] else queries * keys
        scales = 2 * 4 * c["b"] * c["hk"] * keys / c["page"] if per_key == 1 else 0
        return {"bytes": 2 * per_key * c["b"] * keys * c["hk"] * c["d"] + scales + 4 * c["b"] * keys / c["page"] + e * c["b"] * c["hq"] * c["d"] * (queries + c["sq"]),
                "flops": 4.0 * c["b"] * c["hq"] * c["d"] * pairs}
    if c["kind"] == "append":
        tokens = c["b"] * c["t"] * (fill if c["t"] > 8 else 1.0)
        per_value = 1 if c["cache"] == "e4m3" else 2
        return {"bytes": tokens * c["d"] * (2 * c["hk"] * (e + per_value) + c["hq"] * e) + c["b"] * c["t"] * c["hq"] * c["d"] * e + 2 * c["rot"],
                "flops": 3.0 * tokens * (c["hq"] + c["hk"]) * c["rot"] + (4.0 * tokens * c["hk"] * c["d"] if per_value == 1 else 0)}
    n = c["b"] * c["n0"] * c["n1"] * c["n2"]
    rows = n * (c["hq"] + c["hk"])
    if c["kind"] == "qk_fwd":
        return {"bytes": 2 * e * rows * c["d"] + 4 * n * c["axes"] + 2 * c["rot"] + 8 * c["d"], "flops": rows * (4.0 * c["d"] + 3.0 * c["rot"])}
    return {"bytes": 3 * e * rows * c["d"] + 4 * n * c["axes"] + 2 * c["rot"] + 16 * c["d"], "flops": rows * (12.0 * c["d"] + 3.0 * c["rot"])}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------------------------

def _exact_attn(s):
    """Sequence by sequence and head by head, on the queries and keys that there are, read page by page."""
    c = s["case"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(c["b"]):
        lk = int(s["k_lengths"][b])
        lq = c["sq"] if s["q_lengths"] is None else int(s["q_lengths"][b])
        pages = s["page_table"][b, :-(-lk // c["page"])].tolist()
        first = max(0, lq - lk) if c["causal"] else 0  # the first query that sees a key
        hidden = torch.arange(lk)[None] > torch.arange(first, lq)[:, None] + (lk - lq) if c["causal"] else torch.zeros(lq, lk, dtype=torch.bool)
        hidden = hidden.to(o.device)
        for h in range(c["hk"]):
            kv = []
            for name in ("k", "v"):
                scale = s[name + "_scale"]
                kv.append(torch.cat([s[name + "_cache"][p, h].double() * (1.0 if scale is None else scale[p, h].double()) for p in pages])[:lk])
            for u in range(h * (c["hq"] // c["hk"]), (h + 1) * (c["hq"] // c["hk"])):
                x = (s["q"][b, u, first:lq].double() @ kv[0].t() / math.sqrt(c["d"])).masked_fill(hidden, -math.inf)
                o[b, u, first:lq] = torch.softmax(x, -1) @ kv[1]
    return o


def _exact_turn(x, angle, rot, adjacent, sign=1.0):
    """As a product with a complex number of length 1."""
    y = x.double().clone()
    re, im = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * torch.polar(torch.ones_like(angle), sign * angle)
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_append(s):
    c = s["case"]
    pools = {n: s[n + "_cache"].double() for n in "kv"}
    scales = {n: None if s[n + "_scale"] is None else s[n + "_scale"].double() for n in "kv"}
    q = None if s["q"] is None else torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(c["b"]):
        start, n = int(s["starts"][b]), c["t"] if s["lengths"] is None else int(s["lengths"][b])
        angle = torch.arange(start, start + n, device=s["k"].device, dtype=torch.float64)[:, None] * s["inv_freq"].double()
        if q is not None:
            q[b, :, :n] = _exact_turn(s["q"][b, :, :n], angle, c["rot"], c["adjacent"])
        rows = {"k": _exact_turn(s["k"][b, :, :n], angle, c["rot"], c["adjacent"]), "v": s["v"][b, :, :n].double()}
        for i in range(start // c["page"], (start + n - 1) // c["page"] + 1):
            p = int(s["page_table"][b, i])
            lo, hi = max(start, i * c["page"]), min(start + n, (i + 1) * c["page"])
            for name in "kv":
                x = rows[name][:, lo - start:hi - start]
                if scales[name] is None:
                    pools[name][p, :, lo - i * c["page"]:hi - i * c["page"]] = x
                    continue
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448.0)))  # (inputs are not all zero)
                before = scales[name][p]
                now = need if lo == i * c["page"] else torch.maximum(before, need)
                if lo > i * c["page"]:
                    pools[name][p] *= (before / now)[:, None, None]
                pools[name][p, :, lo - i * c["page"]:hi - i * c["page"]] = x / now[:, None, None]
                scales[name][p] = now
    return pools["k"], pools["v"], scales["k"], scales["v"], q


def _exact_qk(s, backward):
    c = s["case"]
    dev = s["q"].device
    start = [sum(s["sections"][:a]) for a in range(c["axes"] + 1)]
    angle = torch.cat([s["positions"][..., a:a + 1].double() * s["inv_freq"][start[a]:start[a + 1]].double() for a in range(c["axes"])], -1)
    out, sums = [], []
    for name in ("q", "k"):
        full = torch.empty(s[name].shape, dtype=torch.float64, device=dev)
        total = torch.zeros(c["d"], dtype=torch.float64, device=dev)
        for b in range(c["b"]):
            x, w = s[name][b].double().requires_grad_(backward), s[name + "_weight"].double().requires_grad_(backward)
            n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * w
            if not backward:
                full[b] = _exact_turn(n, angle[b], c["rot"], c["adjacent"])
                continue
            back = _exact_turn(s["d%s_out" % name][b], angle[b], c["rot"], c["adjacent"], -1.0)  # the turn's transpose
            full[b], dw = torch.autograd.grad(n, (x, w), back)
            total += dw
        out.append(full)
        sums.append(total)
    return tuple(out + sums) if backward else tuple(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(s)
    return _exact_append(s) if case["kind"] == "append" else _exact_qk(s, case["kind"] == "qk_bwd")
