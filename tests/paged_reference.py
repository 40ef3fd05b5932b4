"""A paged KV cache on the CPU in 64 bits, for the tests of ops.paged_*.

Everything is written from the definitions: a pool of pages as [pages, page
size, heads, head_dim] codes and [pages, heads, page size] scales, sequences as
(new tokens, tokens in all) pairs, and loops over tokens.
"""

from __future__ import annotations

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
NAN = float("nan")


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """Codes and fp32 scales of fp16 rows [..., hd]: the nearest code to x / scale
    in exact arithmetic (doubles hold x and the borders' products exactly), ties
    to even; zeros: scale 0, rows that are not finite: scale NaN, codes 0."""
    xd = x.double()
    amax = xd.abs().amax(-1)
    scale = (amax / TOP[dtype]).float()
    fine = torch.isfinite(xd).all(-1)
    safe = torch.where(fine & (amax > 0), scale, torch.ones_like(scale)).double()
    y = torch.where(fine[..., None], xd, 0.0) / safe[..., None]
    if dtype == torch.int8:
        code = y.round().clamp(-127, 127).to(torch.int8)
    else:
        grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
        hi = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 126)
        lo = hi - 1
        down, up = y.abs() - grid[lo], grid[hi] - y.abs()
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        # values that round to zero keep their sign, rows of zeros do not
        code = torch.copysign(grid[pick], torch.where(amax[..., None] > 0, y, 0.0))
        code = code.float().to(dtype)
    return code, torch.where(fine, scale, torch.tensor(NAN))


class Pool:
    """Pages for sequences [(new, total), ...], in a shuffled order, with spare
    pages; slots that hold no token are filled with `stale`."""

    def __init__(self, lens, page, heads, hd, dtype, seed, order="head", spare=2, stale=NAN,
                 extra_width=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.heads, self.hd, self.dtype = lens, page, heads, hd, dtype
        need = [-(-kv // page) for _, kv in lens]
        self.pages = sum(need) + spare
        perm = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1]) + extra_width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.start = torch.tensor([sum(n for n, _ in lens[:b]) for b in range(len(lens) + 1)],
                                  dtype=torch.int32)
        self.kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32)
        self.tokens = int(self.start[-1])
        gain = 0.5 + torch.rand(heads, hd, generator=g)
        self.data = []  # fp16 rows of every sequence: k, v [kv, heads, hd]
        for _, kv in lens:
            k = (torch.randn(kv, heads, hd, generator=g) * gain).half()
            v = torch.randn(kv, heads, hd, generator=g).half()
            self.data.append([k, v])
        self.q_gen = g
        self.order, self.stale = order, stale

    def rows(self, which):
        """The new tokens of every sequence, packed."""
        return torch.cat([d[which][kv - n:] for d, (n, kv) in zip(self.data, self.lens)])

    def place(self, b, pos):
        return int(self.table[b, pos // self.page]), pos % self.page

    def empty(self, stale=None):
        """(k, v, k_scale, v_scale) without tokens: codes of a NaN or of `stale`."""
        stale = self.stale if stale is None else stale
        shape = (self.pages, self.page, self.heads, self.hd)
        if self.dtype == torch.float16:
            return [torch.full(shape, stale, dtype=torch.float16) for _ in range(2)] + [None, None]
        if self.dtype == torch.int8:
            code = [torch.full(shape, 101, dtype=torch.int8) for _ in range(2)]
        else:
            code = [torch.full(shape, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    for _ in range(2)]
        return code + [torch.full((self.pages, self.heads, self.page), stale) for _ in range(2)]

    def filled(self, upto=None):
        """The pool with every token (or only the first upto[b] of sequence b)."""
        t = self.empty()
        for b, (_, kv) in enumerate(self.lens):
            for which in (0, 1):
                x = self.data[b][which][:kv if upto is None else upto[b]]
                pos = torch.arange(x.shape[0])
                pages, slots = self.table[b, pos // self.page].long(), pos % self.page
                if self.dtype == torch.float16:
                    t[which][pages, slots] = x
                else:
                    code, scale = quantise(x, self.dtype)
                    t[which].view(torch.uint8)[pages, slots] = code.view(torch.uint8)
                    t[2 + which][pages, :, slots] = scale
        return t

    def values(self, b, which):
        """What the cache holds of sequence b, in doubles [kv, heads, hd]."""
        x = self.data[b][which]
        if self.dtype == torch.float16:
            return x.double()
        code, scale = quantise(x, self.dtype)
        return code.float().double() * scale[..., None].double()

    def on(self, dev, tensors):
        """Tensors of the cache on `dev`, in the pool's memory order."""
        out = []
        for t in tensors[:2]:
            u = t.view(torch.uint8) if t.dtype != torch.float16 else t
            if self.order == "head":
                u = u.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
            elif self.order == "gap":  # token by token, rows and pages apart
                big = torch.zeros(self.pages + 1, self.page, self.heads + 1, self.hd + 16,
                                  dtype=u.dtype, device=dev)
                view = big[1:, :, :self.heads, 16:]
                view.copy_(u.to(dev))
                u = view
            else:
                u = u.to(dev)
            out.append(u if t.dtype == torch.float16 else u.view(t.dtype))
        return out + [None if s is None else s.to(dev) for s in tensors[2:]]


def attention(pool, q, group, causal=True, scale=None, absent=()):
    """(out, A): fp64 result [T, heads * group * hd], and A = sum of weight * |value|
    with a bound on the weights' exponents, from which tolerances are made.
    absent: (b, page index) pairs whose keys are masked."""
    hd = pool.hd
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(pool.tokens, pool.heads * group, hd, dtype=torch.float64)
    mag, expo = torch.zeros_like(out), torch.zeros(pool.tokens, pool.heads * group, 1).double()
    for b, (n, kv) in enumerate(pool.lens):
        if n == 0 or kv == 0:
            continue
        k, v = pool.values(b, 0), pool.values(b, 1)
        pos = torch.arange(kv)
        held = torch.ones(kv, dtype=torch.bool)
        for ab, page in absent:
            if ab == b:
                held &= pos // pool.page != page
        last = torch.arange(kv - n, kv) if causal else torch.full((n,), kv - 1)
        seen = (pos[None] <= last[:, None]) & held[None]
        lo = int(pool.start[b])
        for h in range(pool.heads * group):
            x = q[lo:lo + n, h].double()
            kk, vv = k[:, h // group], v[:, h // group]
            s = torch.where(seen, x @ kk.T * scale, -torch.inf)
            m = s.amax(-1, keepdim=True)
            w = torch.where(seen, torch.exp(s - torch.where(m == -torch.inf, 0.0, m)), 0.0)
            l = w.sum(-1, keepdim=True)
            w = torch.where(l > 0, w / l, 0.0)
            # a weight of a key that is not seen takes no part, whatever the value
            fine = torch.where(torch.isfinite(vv), vv, 0.0)
            o = w @ fine
            for j in (~torch.isfinite(vv)).any(-1).nonzero().flatten().tolist():
                bad = torch.where(torch.isfinite(vv[j]), 0.0, vv[j])
                o = o + torch.where(seen[:, j:j + 1], bad[None], 0.0)
            out[lo:lo + n, h] = o
            mag[lo:lo + n, h] = w @ fine.abs()
            reach = torch.where(seen, (x.abs() @ torch.nan_to_num(kk).abs().T) * scale, 0.0)
            expo[lo:lo + n, h] = reach.amax(-1, keepdim=True)
    return out.flatten(1), mag.flatten(1), expo.expand(-1, -1, hd).flatten(1)


def tolerance(pool, ref, mag, expo):
    """How far fp16 results may be off the 64-bit ones, element by element.

    Half a step of the result (2^-11 of it; 2^-25 where it is subnormal), and of
    each weight (2^-11), on A = sum w|v|; weights below 2^-14 are rounded by at most
    2^-25 (of the largest value, a row's largest weight being 1). Exponentials are
    within 2^-13 of themselves (7.5e-5, the polynomial's). Sums over hd
    products and over the keys in fp32 whose steps may truncate (2^-23 each): on
    the exponent hd + 8 steps of its largest sum, on the result one step for each
    16 keys and 8 more."""
    n = max([kv for _, kv in pool.lens] + [1])
    most = max([float(torch.nan_to_num(pool.values(b, 1), 0, 0, 0).abs().max()) if kv else 0.0
                for b, (_, kv) in enumerate(pool.lens)] + [0.0])
    on_exp = (pool.hd + 8) * 2.0 ** -23 * expo + 2.0 ** -21
    per = 2.0 ** -11 + 2.0 ** -13 + (n / 16 + 8) * 2.0 ** -23
    # an error d of the exponents moves weights by at most exp(2d) - 1 of themselves
    return 2.0 ** -11 * ref.abs() + 2.0 ** -25 + (per + torch.expm1(2 * on_exp)) * mag + \
        n * 2.0 ** -25 * most


def attention_own(pool, q, group, causal=True, scale=None, absent=()):
    """(out, tol): fp64 result [T, heads * group * hd], and how far fp16 results may be off
    it, element by element, from the keys that the element's own row sees and nothing else.

    With weights w_j (sum 1), values v_j = s_j c_j (s a value's scale in 8 bits, else 1) and
    A = sum w_j |v_j| >= |out|:
      the result is rounded: 2^-11 |out|, 2^-25 where it is subnormal;
      w_j s_j is rounded to fp16, relative to its largest, R = max w_j s_j, which the kernels'
      reference does not exceed: 2^-11 of itself, and below 2^-14 R by 2^-25 R, but never by
      more than itself: 2^-11 A + sum min(w_j s_j, 2^-25 R) |c_j|;
      the weights' sum may take them as rounded: (2^-11 + n 2^-25 max w) |out|;
      exponentials are within 2^-13 (the polynomial's 7.5e-5), in both sums;
      an exponent is off by d_j: hd products summed in fp32 in steps that may truncate (2^-23
      of the largest sum each) and 8 more steps; 8 bits add log2(s_j), within 2^-22 of itself,
      40 at most, and a step of exponents up to 40 larger: w_j is off by expm1(d_j) of itself,
      in both sums;
      both sums are in fp32, one step of 2^-23 for each 16 keys and 8 more."""
    hd, quant = pool.hd, pool.dtype != torch.float16
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(pool.tokens, pool.heads * group, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b, (n, kv) in enumerate(pool.lens):
        if n == 0 or kv == 0:
            continue
        k, v = pool.values(b, 0), pool.values(b, 1)
        s = torch.ones(kv, pool.heads, dtype=torch.float64)
        if quant:
            s = quantise(pool.data[b][1], pool.dtype)[1].double()
        pos = torch.arange(kv)
        held = torch.ones(kv, dtype=torch.bool)
        for ab, page in absent:
            if ab == b:
                held &= pos // pool.page != page
        last = torch.arange(kv - n, kv) if causal else torch.full((n,), kv - 1)
        seen = (pos[None] <= last[:, None]) & held[None]
        lo = int(pool.start[b])
        for h in range(pool.heads * group):
            x = q[lo:lo + n, h].double()
            kk, vv, ss = k[:, h // group], v[:, h // group], s[:, h // group]
            cc = torch.where(ss[:, None] > 0, vv.abs() / ss[:, None], 0.0)
            e = torch.where(seen, x @ kk.T * scale, -torch.inf)
            m = e.amax(-1, keepdim=True)
            w = torch.where(seen, torch.exp(e - torch.where(m == -torch.inf, 0.0, m)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            o, mag = w @ vv, w @ vv.abs()
            reach = (x.abs() @ kk.abs().T) * scale
            d = torch.expm1((hd + 8) * 2.0 ** -23 * reach + 2.0 ** -21 +
                            (40 * (2.0 ** -22 + 2.0 ** -23) if quant else 0.0)) * w
            y = w * ss[None]
            lost = torch.minimum(y, 2.0 ** -25 * y.amax(-1, keepdim=True)) @ cc
            count = seen.sum(-1, keepdim=True)
            both = 2.0 ** -11 + 2.0 ** -13 + (count / 16 + 8) * 2.0 ** -23
            out[lo:lo + n, h] = o
            tol[lo:lo + n, h] = (2.0 ** -11 * o.abs() + 2.0 ** -25 + both * (mag + o.abs()) + lost +
                                 d @ vv.abs() + d.sum(-1, keepdim=True) * o.abs() +
                                 count * 2.0 ** -25 * w.amax(-1, keepdim=True) * o.abs())
    return out.flatten(1), tol.flatten(1)
