"""Plain implementations in 64 bits of the operators over a key/value cache, and tensors for their tests.

Tolerances count roundings: a value rounded to a type is off by half a step, ``finfo.eps / 2`` of it; sums and products in fp32 are off by
2^-24 each of what they add up."""
import math

import torch

U32 = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


def half_step(dtype):
    return 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2


def heads(g, b, h, s, d, dtype, layout="bhsd", scale=1.0):
    x = torch.randn(b, h, s, d, device="cuda", generator=g) * scale
    x = x.to(dtype)
    if layout == "bshd":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":  # rows of an odd number of elements, the base off 16 bytes
        wide = torch.zeros(b, h, s, d + 3, device="cuda", dtype=dtype)
        wide[..., 1:d + 1] = x
        return wide[..., 1:d + 1]
    return x


def rotated(x, angle, rot, adjacent, sign=1.0):
    """(x turned, the sum of the magnitudes that each element is made of) in 64 bits: x [B,H,S,D], angle [B or 1,S,rot/2]."""
    x = x.double()
    if rot == 0:
        return x, x.abs()
    u, v = (x[..., 0:rot:2], x[..., 1:rot:2]) if adjacent else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = angle.cos()[:, None], sign * angle.sin()[:, None]
    a, b, m = u * c - v * s, v * c + u * s, u.abs() + v.abs()
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if adjacent else (lambda p, q: torch.cat([p, q], -1))
    return torch.cat([join(a, b), x[..., rot:]], -1), torch.cat([join(m, m), x[..., rot:].abs()], -1)


def angles(positions, inv_freq, sections):
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(positions.device)
    return positions.double()[..., axis] * inv_freq.double()


class Pool:
    """Caches of `pages` pages, all filled with what a user may find there, and a table of pages in no order."""

    def __init__(self, g, pages, hk, page, d, dtype, e4m3, order="nhpd", fill=1.0):
        self.page, self.e4m3 = page, e4m3
        shape = (pages, hk, page, d)
        self.k, self.v = (torch.randn(shape, device="cuda", generator=g).mul(fill).to(dtype) for _ in range(2))
        self.k_scale = self.v_scale = None
        if e4m3:
            self.k_scale, self.v_scale = (torch.exp2(torch.randint(-9, -5, (pages, hk), device="cuda", generator=g).float()) for _ in range(2))
            self.k, self.v = ((t.float() / s[..., None, None]).clamp(-448, 448).to(E4M3) for t, s in ((self.k, self.k_scale), (self.v, self.v_scale)))
        if order == "npHd":  # tokens in front of heads
            self.k, self.v = (self._u8(t).transpose(1, 2).contiguous().transpose(1, 2) for t in (self.k, self.v))
        elif order == "both":  # one buffer for keys and values
            both = torch.stack([self._u8(self.k), self._u8(self.v)], 1)
            self.k, self.v = both[:, 0], both[:, 1]
        if e4m3:
            self.k, self.v = (t.view(E4M3) for t in (self.k, self.v))

    @staticmethod
    def _u8(t):
        return t.view(torch.uint8) if t.dtype == E4M3 else t

    def values(self, name):
        t, s = getattr(self, name), getattr(self, name + "_scale")
        return t.double() if s is None else t.double() * s.double()[..., None, None]

    def scales(self):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale}


def table(g, b, per, pages):
    return torch.randperm(pages, device="cuda", generator=g)[:b * per].to(torch.int32).view(b, per)


def gathered(pool, name, page_table, length):
    """([length, Hk, D] values, [length] whether there is a page) of one sequence."""
    values = pool.values(name)
    n, p = values.shape[0], pool.page
    t = torch.arange(length, device=values.device)
    slot = t // p
    inside = slot < page_table.shape[0]
    entry = page_table.long()[slot.clamp(max=max(page_table.shape[0] - 1, 0))] if page_table.shape[0] else torch.full_like(t, -1)
    there = inside & (entry >= 0) & (entry < n)
    x = values[entry.clamp(0, max(n - 1, 0)), :, t % p] if n else torch.zeros(length, values.shape[1], values.shape[3], device=values.device).double()
    return torch.where(there[:, None, None], x, torch.zeros_like(x)), there


def attention(q, pool, page_table, k_lengths, q_lengths=None, causal=True, scale=None, rounded=False):
    """(o, lse, allowed, lse_off) in 64 bits; allowed: how far a kernel's o may be off, without its last rounding.  rounded: keys and values are
    rounded to the type of q (scales that are no powers of two)."""
    b, hq, sq, d = q.shape
    hk = pool.k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(b, hq, sq, d, device=q.device, dtype=torch.float64)
    allowed = torch.zeros_like(o)
    lse = torch.full((b, hq, sq), -math.inf, device=q.device, dtype=torch.float64)
    lse_off = torch.zeros_like(lse)
    for i in range(b):
        lk = max(0, min(int(k_lengths[i]), page_table.shape[1] * pool.page))
        lq = sq if q_lengths is None else max(0, min(int(q_lengths[i]), sq))
        k, there = gathered(pool, "k", page_table[i], lk)
        v, _ = gathered(pool, "v", page_table[i], lk)
        for h in range(hq):
            kk, vv = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
            x = scale * (q[i, h, :lq].double() @ kk.t())
            seen = there[None].expand(lq, lk)
            if causal:
                seen = seen & (torch.arange(lk, device=q.device)[None] <= torch.arange(lq, device=q.device)[:, None] + (lk - lq))
            x = x.masked_fill(~seen, -math.inf)
            some = seen.any(-1)
            lse[i, h, :lq] = torch.logsumexp(x, -1) if lk else -math.inf
            p = torch.where(some[:, None], torch.softmax(x, -1), torch.zeros_like(x)) if lk else x
            o[i, h, :lq] = p @ vv
            # a score is a sum of D products in fp32, its exponent and the scales some roundings more
            made_of = abs(scale) * (q[i, h, :lq].double().abs() @ kk.abs().t())
            off = U32 * ((d + 8) * torch.where(seen, made_of, torch.zeros_like(x)).amax(-1) + 40 if lk else torch.zeros(lq, device=q.device))
            if rounded and lk:
                off = off + half_step(q.dtype) * torch.where(seen, made_of, torch.zeros_like(x)).amax(-1)
            weight = p @ vv.abs()
            # a probability is rounded to the operand type; f16 loses what is 2^36 below a row's largest
            lost = (2.0 ** -36) * vv.abs().sum(0) if q.dtype == torch.float16 and lk else 0.0
            allowed[i, h, :lq] = (half_step(q.dtype) * (2 if rounded else 1) + 2 * off[:, None] + 64 * U32) * weight + lost
            lse_off[i, h, :lq] = off + 8 * U32 * torch.where(some, lse[i, h, :lq].abs(), torch.zeros_like(off))
    return o, lse, allowed, lse_off


def check_attention(got, lse, want, want_lse, allowed, lse_off):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    bad = err > allowed + half_step(got.dtype) * want.abs() + 1e-30 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)  # (f16: below its normal numbers)
    assert not bad.any(), "%d of %d, the worst off by %.3g where %.3g is allowed" % (bad.sum(), bad.numel(), err[bad].max(), allowed[bad].max())
    if lse is not None:
        assert torch.equal(lse == -math.inf, want_lse == -math.inf)
        fine = want_lse > -math.inf
        assert ((lse.double() - want_lse).abs()[fine] <= lse_off[fine] + 1e-6).all()


def append(pool, page_table, k, v, starts, lengths=None, rot=0, angle=None, adjacent=False):
    """What the caches hold afterwards: {name: (values [N,Hk,P,D], allowed, scales or None, changed)} in 64 bits.  Sequence by sequence.
    changed [N,Hk,P]: the new tokens' places, and all others of a page and head whose scale has grown."""
    out = {}
    for name, x in (("k", k), ("v", v)):
        y, made_of = rotated(x, angle, rot, adjacent) if name == "k" and rot else (x.double(), x.double().abs())
        fp32 = 16 * U32 * made_of if name == "k" and rot else torch.zeros_like(y)
        values = pool.values(name).clone()
        scale = None if not pool.e4m3 else getattr(pool, name + "_scale").double().clone()
        allowed, written = torch.zeros_like(values), torch.zeros(values.shape[:3], dtype=torch.bool, device=values.device)
        n_pages, p = values.shape[0], pool.page
        for i in range(k.shape[0]):
            start = max(0, int(starts[i]))
            n = k.shape[2] if lengths is None else max(0, min(int(lengths[i]), k.shape[2]))
            for slot in range(start // p, (start + n - 1) // p + 1 if n else 0):
                page = int(page_table[i, slot]) if slot < page_table.shape[1] else -1
                if not 0 <= page < n_pages:
                    continue
                lo, hi = max(start, slot * p), min(start + n, (slot + 1) * p)
                at, new = slice(lo - slot * p, hi - slot * p), slice(lo - start, hi - start)
                values[page, :, at] = y[i, :, new]
                allowed[page, :, at] = fp32[i, :, new]
                written[page, :, at] = True
                if scale is None:
                    allowed[page, :, at] += half_step(pool.k.dtype) * y[i, :, new].abs()
                    continue
                z = y[i, :, new]
                top = torch.where(torch.isfinite(z), z.abs(), torch.zeros_like(z)).amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-126))
                old = torch.zeros_like(need) if lo == slot * p else scale[page]
                now = torch.maximum(old, need)
                grown = (now > old) & (old > 0)
                written[page] |= grown[:, None]
                rows = torch.ones(p, dtype=torch.bool, device=values.device)  # (the other places)
                rows[at] = False
                if lo == slot * p:  # (begun anew: what its other codes stand for is nobody's)
                    allowed[page, :, rows] = math.inf
                step = torch.maximum(2.0 ** -10 * now[:, None, None].expand_as(values[page, :, rows]), torch.zeros(1, device=values.device).double())
                allowed[page, :, rows] += torch.where(grown[:, None, None], step, torch.zeros_like(step))  # (below the normal codes)
                scale[page] = now
                allowed[page, :, at] += torch.maximum(2.0 ** -4 * z.abs(), 2.0 ** -10 * now[:, None, None].expand_as(z))
        out[name] = (values, allowed, scale, written)
    return out
