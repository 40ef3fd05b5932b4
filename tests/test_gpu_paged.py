"""The paged KV cache on a B200: ops.paged_append, paged_read and
paged_attention against the 64-bit model in paged_reference.py."""

from __future__ import annotations

import pytest
import torch

import paged_reference as pr

pytestmark = pytest.mark.gpu

F16, I8, E4 = torch.float16, torch.int8, torch.float8_e4m3fn
NAMES = {F16: "fp16", I8: "int8", E4: "e4m3"}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _batch(pkg, dev, pool, tokens=None, **kw):
    return pkg.PagedBatch(pool.table.to(dev), pool.start.to(dev), pool.kv.to(dev),
                          pool.tokens if tokens is None else tokens, **kw)


def _hints(pool):
    return {"max_query_len": max(n for n, _ in pool.lens), "max_kv_len": int(pool.kv.max())}


def _cpu(t):
    return t.view(torch.uint8).cpu() if t.dtype in (I8, E4) else t.cpu()


def _same(got, want):
    """Equal bit for bit, NaN included."""
    got, want = got.cpu(), want.cpu()
    if got.is_floating_point() and got.element_size() > 1:
        nan = torch.isnan(want)
        return torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
    return torch.equal(got, want)


# sequences (new, total): single tokens, whole prompts, no new token, a first
# token, page ends at, before and behind a length
LENS = [(1, 33), (16, 16), (0, 20), (17, 64), (1, 1), (65, 65), (5, 130)]
COPY = [(F16, 8, 3, 16, "head"), (F16, 64, 2, 32, "token"), (F16, 256, 1, 16, "gap")]
COPY += [(t, hd, h, page, order) for t in (I8, E4) for hd, h, page, order in
         ((16, 3, 16, "head"), (32, 4, 64, "token"), (64, 5, 32, "gap"), (128, 2, 128, "head"),
          (256, 1, 256, "token"))]


@pytest.mark.parametrize("dtype,hd,heads,page,order", COPY,
                         ids=lambda v: NAMES.get(v, str(v)) if not isinstance(v, (int, str)) else str(v))
def test_append_then_read(pkg, dev, dtype, hd, heads, page, order):
    """Codes and scales bit for bit, slots of other tokens untouched; the values
    read back are code * scale rounded once."""
    pool = pr.Pool(LENS, page, heads, hd, dtype, hd + page, order)
    # rows of every size: tiny, huge, zeros, one outlier
    for b, d in enumerate(pool.data):
        for x in d:
            if x.shape[0] > 2:
                x[0] *= 1e-4
                x[1] *= 2000
                x[-1, 0] = 0
                x[-2, -1, -1] = 50000.0
    before = pool.filled(upto=[kv - n for n, kv in LENS])
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, before))
    batch = _batch(pkg, dev, pool)
    new = torch.stack((pool.rows(0), pool.rows(1)), 1).to(dev)  # packed projection
    pkg.ops.paged_append(new[:, 0], new[:, 1], cache, batch)
    want = pool.filled()
    for got, ref in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if ref is not None:
            assert _same(_cpu(got), _cpu(ref))
    k, v = pkg.ops.paged_read(cache, batch)
    for which, got in enumerate((k, v)):
        ref = torch.cat([pool.values(b, which)[kv - n:] for b, (n, kv) in enumerate(LENS)])
        assert torch.equal(got.cpu(), ref.float().half())
    # whole sequences
    full = pr.Pool([(kv, kv) for _, kv in LENS], page, heads, hd, dtype, hd + page, order)
    whole = pkg.PagedBatch(batch.page_table, full.start.to(dev), batch.kv_len, full.tokens)
    k, v = pkg.ops.paged_read(cache, whole)
    for which, got in enumerate((k, v)):
        ref = torch.cat([pool.values(b, which) for b in range(len(LENS))])
        assert torch.equal(got.cpu(), ref.float().half())


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
def test_codes_next_to_borders(pkg, dev, dtype):
    """Every fp16 magnitude against many row maxima: quotients on and beside the
    borders of two codes, ties, subnormals of fp16 and of e4m3."""
    mags = torch.arange(0, 0x7c00, dtype=torch.int32).to(torch.int16).view(F16)
    tops = torch.cat([torch.tensor([65504.0, 127.0, 448.0, 254.0, 1.0, 3.5, 6e-8, 2e-5]).half(),
                      (torch.rand(24, generator=torch.Generator().manual_seed(5)) * 4).half()])
    hd, rows = 64, []
    for top in tops:
        x = mags[mags <= top]
        x = torch.cat([x, x.new_zeros(-x.numel() % (hd - 1))]).view(-1, hd - 1)
        x[::2, ::3] *= -1
        rows.append(torch.cat([x, top.expand(x.shape[0], 1)], 1))
    x = torch.cat(rows)[:, None]  # [T, 1, hd]
    n = x.shape[0]
    page, pages = 64, -(-n // 64)
    cache = pkg.PagedKVCache(pages, page, 1, hd, dtype, dev)
    batch = pkg.PagedBatch(torch.arange(pages, dtype=torch.int32, device=dev)[None],
                           torch.tensor([0, n], dtype=torch.int32, device=dev),
                           torch.tensor([n], dtype=torch.int32, device=dev), n)
    pkg.ops.paged_append(x.to(dev), (-x).to(dev), cache, batch)
    for sign, codes, scales in ((1, cache.k, cache.k_scale), (-1, cache.v, cache.v_scale)):
        code, scale = pr.quantise(sign * x, dtype)
        got = codes.reshape(-1, 1, hd).view(torch.uint8).cpu()[:n]
        assert torch.equal(got, code.view(torch.uint8))
        assert torch.equal(scales.transpose(1, 2).reshape(-1, 1).cpu()[:n], scale)


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
def test_copies_leave_everything_else(pkg, dev, dtype):
    """Tokens without a page are dropped and read as zeros, rows behind the last
    sequence keep what they held, infinities and NaN poison their own row."""
    lens = [(40, 40), (3, 50), (2, 2)]
    pool = pr.Pool(lens, 16, 2, 64, dtype, 9)
    pool.data[0][0][7, 1, 3] = float("inf")
    pool.data[1][1][48, 0, 0] = float("nan")
    table = pool.table.clone()
    table[0, 1] = -1
    table[1, 3] = pool.pages          # one past the pool
    table[2, 0] = -2 ** 31
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.empty(stale=7.0)))
    rows = pool.tokens + 5
    batch = pkg.PagedBatch(table.to(dev), pool.start.to(dev), pool.kv.to(dev), rows)
    new = torch.zeros(rows, 2, 2, 64, dtype=F16)
    new[:pool.tokens] = torch.stack((pool.rows(0), pool.rows(1)), 1)
    new = new.to(dev)
    pkg.ops.paged_append(new[:, 0], new[:, 1], cache, batch)
    want = pool.empty(stale=7.0)
    for b, (n, kv) in enumerate(lens):
        for pos in range(kv - n, kv):
            page = int(table[b, pos // 16])
            if not 0 <= page < pool.pages:
                continue
            for which in (0, 1):
                x = pool.data[b][which][pos]
                if dtype == F16:
                    want[which][page, pos % 16] = x
                else:
                    code, scale = pr.quantise(x, dtype)
                    want[which].view(torch.uint8)[page, pos % 16] = code.view(torch.uint8)
                    want[2 + which][page, :, pos % 16] = scale
    for got, ref in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if ref is not None:
            assert _same(_cpu(got), _cpu(ref))
    out = tuple(torch.full((rows, 2, 64), -3.0, dtype=F16, device=dev) for _ in range(2))
    k, v = pkg.ops.paged_read(cache, batch, out=out)
    assert k is out[0] and v is out[1]
    for which, got in enumerate((k.cpu(), v.cpu())):
        assert bool((got[pool.tokens:] == -3).all())
        for b, (n, kv) in enumerate(lens):
            for i, pos in enumerate(range(kv - n, kv)):
                row = got[int(pool.start[b]) + i]
                if not 0 <= int(table[b, pos // 16]) < pool.pages:
                    assert bool((row == 0).all())
                elif dtype == F16:
                    assert _same(row, pool.data[b][which][pos])
                else:
                    code, scale = pr.quantise(pool.data[b][which][pos], dtype)
                    assert _same(row, (code.float() * scale[..., None]).half())


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
def test_the_same_slot_twice(pkg, dev, dtype):
    """Tokens that share a slot, which is not allowed, leave every other slot right."""
    heads, hd, page = 3, 64, 16
    gen = torch.Generator().manual_seed(77)
    x = torch.randn(40, 2, heads, hd, generator=gen).half()
    cache = pkg.PagedKVCache(4, page, heads, hd, dtype, dev)
    # sequence 0 has page 2 twice (positions 0-15 and 16-31), sequence 1 page 0
    batch = pkg.PagedBatch(torch.tensor([[2, 2], [0, 1]], dtype=torch.int32, device=dev),
                           torch.tensor([0, 20, 40], dtype=torch.int32, device=dev),
                           torch.tensor([20, 20], dtype=torch.int32, device=dev), 40)
    pkg.ops.paged_append(x[:, 0].to(dev), x[:, 1].to(dev), cache, batch)
    k, v = pkg.ops.paged_read(cache, batch)
    for which, got in enumerate((k.cpu(), v.cpu())):
        for row in [*range(4, 16), *range(20, 40)]:  # slots 0-3 of page 2 are written twice
            want = x[row, which]
            if dtype != F16:
                code, scale = pr.quantise(want, dtype)
                want = (code.float() * scale[..., None]).half()
            assert _same(got[row], want)


def _attend(pkg, dev, pool, group, causal=True, scale=None, hints=True, q=None, gain=1.5):
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    batch = _batch(pkg, dev, pool, **(_hints(pool) if hints else {}))
    if q is None:
        q = (gain * torch.randn(pool.tokens, pool.heads * group, pool.hd,
                                generator=pool.q_gen)).half()
    got = pkg.ops.paged_attention(q.to(dev), cache, batch, is_causal=causal, scale=scale)
    return q, got.double().cpu()


def _check(pool, got, q, group, causal=True, scale=None, absent=()):
    ref, mag, expo = pr.attention(pool, q, group, causal, scale, absent)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    ok = torch.isfinite(ref)
    err = (got - ref).abs()[ok]
    tol = pr.tolerance(pool, ref, mag, expo)[ok]
    assert bool((err <= tol).all()), float((err / tol).max())


DECODE = [(1, 1), (1, 700), (1, 16), (0, 40), (1, 257), (1, 513), (1, 1300)]
DRAFT = [(4, 300), (1, 64), (7, 7), (3, 1025), (0, 0), (2, 31)]
CHUNK = [(130, 400), (1, 77), (64, 64), (257, 300), (31, 1000)]
# (10 heads of CHUNK are enough work for the tcgen05 kernel, 2 are not)


@pytest.mark.parametrize("dtype,hd", [(F16, hd) for hd in (8, 16, 32, 64, 128, 256)] +
                         [(t, hd) for t in (I8, E4) for hd in (16, 32, 64, 128, 256)],
                         ids=lambda v: NAMES.get(v, str(v)) if not isinstance(v, int) else str(v))
@pytest.mark.parametrize("what", ["decode", "draft", "chunk", "prompt"])
def test_attention(pkg, dev, dtype, hd, what):
    lens = {"decode": DECODE, "draft": DRAFT, "chunk": CHUNK, "prompt": CHUNK}[what]
    heads, group, page, order = {"decode": (3, 1, 16, "head"), "draft": (2, 4, 64, "token"),
                                 "chunk": (2, 2, 128, "head"), "prompt": (10, 2, 32, "token")}[what]
    pool = pr.Pool(lens, page, heads, hd, dtype, hd, order)
    q, got = _attend(pkg, dev, pool, group)
    _check(pool, got, q, group)


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("hd,heads,group,page,order,lens", [
    (64, 2, 3, 32, "gap", [(43, 43), (1, 90), (50, 177)]),     # groups that do not divide a tile
    (64, 2, 5, 16, "head", [(7, 400), (3, 3)]),
    (64, 2, 16, 64, "head", [(1, 2000)]),
    (128, 2, 33, 64, "head", [(5, 70)]),                        # more heads in a group than rows of a block
    (64, 1, 130, 64, "head", [(2, 70), (1, 5)]),
    # the tcgen05 kernel
    (64, 16, 3, 32, "gap", [(43, 1043), (1, 90), (50, 1177), (90, 90)]),
    (64, 32, 5, 16, "head", [(37, 1400), (3, 3)]),
    (128, 16, 7, 256, "head", [(40, 1300), (1, 256), (22, 1257)]),
    (128, 40, 33, 64, "gap", [(9, 1070)]),
    (128, 48, 1, 128, "token", [(300, 1111)]),
    (256, 12, 2, 16, "head", [(133, 1333), (65, 65)]),
    (256, 16, 128, 64, "gap", [(2, 900), (1, 300)]),
    (256, 16, 3, 128, "token", [(90, 700), (30, 500)]),
])
def test_attention_heads_and_orders(pkg, dev, dtype, hd, heads, group, page, order, lens):
    pool = pr.Pool(lens, page, heads, hd, dtype, group, order)
    q, got = _attend(pkg, dev, pool, group)
    _check(pool, got, q, group)
    # without the optional bounds: more splits and blocks than needed
    _, again = _attend(pkg, dev, pool, group, hints=False, q=q)
    _check(pool, again, q, group)


@pytest.mark.parametrize("dtype", [F16, I8], ids=["fp16", "int8"])
@pytest.mark.parametrize("hd,heads", [(32, 2), (64, 2), (64, 10), (128, 10), (256, 10)])
def test_attention_not_causal_and_scaled(pkg, dev, dtype, hd, heads):
    pool = pr.Pool(CHUNK, 32, heads, hd, dtype, 3)
    q, got = _attend(pkg, dev, pool, 1, causal=False)
    _check(pool, got, q, 1, causal=False)
    q, got = _attend(pkg, dev, pool, 1, scale=0.3)
    _check(pool, got, q, 1, scale=0.3)


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,heads", [(DRAFT, 2), (CHUNK, 2), (CHUNK, 10)],
                         ids=["draft", "chunk", "prompt"])
def test_attention_hides_what_a_row_does_not_see(pkg, dev, dtype, hd, lens, heads):
    """NaN, infinities and huge values at positions that a row does not see (later
    tokens; slots behind the sequence are NaN in every test here) leave it as
    it is; the rows that see them get them."""
    pool = pr.Pool(lens, 16, heads, hd, dtype, 11)
    n, kv = lens[0]
    pool.data[0][1][kv - 2, 0, 1] = float("inf")     # value
    pool.data[0][1][kv - 1, 1, 5] = float("nan")
    pool.data[0][0][kv - 1, 0, 0] = float("nan")     # key
    pool.data[2][1][5, 1, :] = 60000.0
    q, got = _attend(pkg, dev, pool, 2)
    assert torch.isfinite(got[:n - 2]).all() and not torch.isfinite(got[n - 1]).all()
    ref, mag, expo = pr.attention(pool, q, 2)
    rows = torch.ones(pool.tokens, dtype=torch.bool)
    rows[n - 2:n] = False  # these see a value or key that is not finite
    tol = pr.tolerance(pool, ref, mag, expo)
    err = (got - ref).abs()
    assert bool((err <= tol)[rows].all()), float((err / tol)[rows].max())
    # row n - 2 sees the infinity of head 0 (8 bits: its whole scale is NaN), not the last token
    row = got[n - 2].view(2 * heads, hd)
    assert not torch.isfinite(row[:2, 1]).any() and torch.isfinite(row[2:]).all()
    if dtype == F16:
        assert int((~torch.isfinite(row)).sum()) == 2 and bool((row[:2, 1] == float("inf")).all())
    last = got[n - 1].view(2 * heads, hd)  # a NaN key of head 0, a NaN value of head 1
    assert not torch.isfinite(last[:2]).any() and not torch.isfinite(last[2:4, 5]).any()
    assert torch.isfinite(last[4:]).all()


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("hd,heads,lens", [
    (32, 2, [(20, 300), (3, 40), (2, 10), (90, 200)]), (64, 2, [(20, 300), (3, 40), (2, 10), (90, 200)]),
    (64, 12, [(20, 3000), (3, 40), (2, 10), (200, 2000)]),
    (128, 12, [(20, 2000), (3, 40), (2, 10), (200, 1500)]),
    (256, 8, [(20, 2000), (3, 40), (2, 10), (100, 1500)])])
def test_attention_pages_outside_the_pool(pkg, dev, dtype, hd, heads, lens):
    """Their keys are masked; a row that sees no key at all is zero; rows behind the
    last sequence are left as they were."""
    pool = pr.Pool(lens, 16, heads, hd, dtype, 4)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    table = pool.table.clone()
    absent = [(0, 0), (0, 7), (0, 18), (2, 0), (3, 9), (3, 8)]
    for i, (b, page) in enumerate(absent):
        table[b, page] = [-1, pool.pages, 2 ** 31 - 1, -2 ** 31][i % 4]
    rows = pool.tokens + 3
    batch = pkg.PagedBatch(table.to(dev), pool.start.to(dev), pool.kv.to(dev), rows, **_hints(pool))
    q = torch.randn(rows, 2 * heads, hd, generator=pool.q_gen).half()
    out = torch.full((rows, 2 * heads * hd), -3.0, dtype=F16, device=dev)
    got = pkg.ops.paged_attention(q.to(dev), cache, batch, out=out)
    assert got is out
    got = got.double().cpu()
    assert bool((got[pool.tokens:] == -3).all())
    assert bool((got[int(pool.start[2]):int(pool.start[3])] == 0).all())
    _check(pool, got[:pool.tokens], q[:pool.tokens], 2, absent=absent)


def test_lengths_and_starts_out_of_range(pkg, dev):
    """Lengths beyond the table or below the new tokens, and starts beyond the rows,
    are clamped: every access stays inside, what is well-formed is right."""
    pool = pr.Pool([(4, 64), (2, 30), (5, 48)], 16, 2, 64, F16, 2, extra_width=0)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    q = torch.randn(pool.tokens, 2, 64, generator=pool.q_gen).half()
    ref = pr.attention(pool, q, 1)[0]
    kv = pool.kv.clone()
    kv[1] = 2 ** 31 - 1           # far more than its pages
    start = pool.start.clone()
    start[3] = 2 ** 31 - 1        # clamped to the 11 rows
    batch = pkg.PagedBatch(pool.table.to(dev), start.to(dev), kv.to(dev), pool.tokens)
    got = pkg.ops.paged_attention(q.to(dev), cache, batch).double().cpu()
    assert (got - ref)[:4].abs().max() < 4e-3 and (got - ref)[6:].abs().max() < 4e-3
    kv[1], kv[0] = -5, 2          # fewer tokens than new ones: the first two have no position
    batch = pkg.PagedBatch(pool.table.to(dev), start.to(dev), kv.to(dev), pool.tokens)
    got = pkg.ops.paged_attention(q.to(dev), cache, batch).double().cpu()
    assert bool((got[:2] == 0).all()) and bool((got[4:6] == 0).all())
    k, _ = pkg.ops.paged_read(cache, batch)
    assert bool((k[:2] == 0).all()) and torch.equal(k[2:4].cpu(), pool.data[0][0][:2])
    before = cache.k.clone()
    pkg.ops.paged_append(torch.ones_like(k), torch.ones_like(k), cache, batch)
    bits = lambda t: t.view(torch.int16)  # noqa: E731  (slots without a token are NaN)
    changed = (bits(cache.k) != bits(before)).flatten(2).any(-1)
    assert int(changed.sum()) <= 2 + 5  # two of sequence 0, none of 1, five of 2


def test_no_new_tokens(pkg, dev):
    pool = pr.Pool([(0, 5), (0, 0)], 16, 2, 64, I8, 2)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    q = torch.zeros(0, 2, 64, dtype=F16, device=dev)
    for rows in (0, 3):  # none at all; rows of no sequence
        batch = _batch(pkg, dev, pool, rows)
        out = torch.full((rows, 128), 2.0, dtype=F16, device=dev)
        x = torch.zeros(rows, 2, 64, dtype=F16, device=dev)
        before = _cpu(cache.k).clone()
        pkg.ops.paged_append(x, x, cache, batch)
        assert torch.equal(_cpu(cache.k), before)
        got = pkg.ops.paged_attention(x, cache, batch, out=out)
        assert bool((got == 2).all())
        assert pkg.ops.paged_read(cache, batch)[0].shape == (rows, 2, 64)
    assert q.shape[0] == 0


@pytest.mark.parametrize("dtype", [F16, I8], ids=["fp16", "int8"])
@pytest.mark.parametrize("lens,hint", [([(1, 5000), (1, 300)], 700), ([(1, 9000)], 2000),
                                       ([(90, 9000), (1, 4000)], 4096), ([(200, 7000)], 1)])
def test_sequences_longer_than_the_hint(pkg, dev, dtype, lens, hint):
    """max_kv_len only sizes the split over keys: longer sequences are attended whole."""
    pool = pr.Pool(lens, 64, 1, 64, dtype, 13)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    batch = _batch(pkg, dev, pool, max_query_len=max(n for n, _ in lens), max_kv_len=hint)
    q = torch.randn(pool.tokens, 2, 64, generator=pool.q_gen).half()
    got = pkg.ops.paged_attention(q.to(dev), cache, batch).double().cpu()
    _check(pool, got, q, 2)


@pytest.mark.parametrize("dtype", [F16, I8], ids=["fp16", "int8"])
@pytest.mark.parametrize("hd,heads,lens,most", [
    (64, 2, [(5, 3000), (1, 40), (2, 700)], 2),         # keys split over CTAs, and joined
    (32, 3, [(40, 50), (9, 9), (1, 1)], 11),            # more than a block of rows
    (128, 10, [(300, 900), (1, 500), (190, 190)], 150),  # the tcgen05 kernel, and few rows
    (64, 1, [(400, 9000)], 130),
])
def test_more_new_tokens_than_the_bound(pkg, dev, dtype, hd, heads, lens, most):
    """The first max_query_len tokens of a sequence attend as ever, further rows stay as
    they were."""
    pool, group = pr.Pool(lens, 64, heads, hd, dtype, 14), 2
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    batch = _batch(pkg, dev, pool, max_query_len=most, max_kv_len=int(pool.kv.max()))
    q = torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen).half()
    out = torch.full((pool.tokens, heads * group * hd), -3.0, dtype=F16, device=dev)
    got = pkg.ops.paged_attention(q.to(dev), cache, batch, out=out).double().cpu()
    ref, mag, expo = pr.attention(pool, q, group, True, None, ())
    ok = (got - ref).abs() <= pr.tolerance(pool, ref, mag, expo)
    for b, (n, _) in enumerate(lens):
        rows = int(pool.start[b]) + torch.arange(n)
        assert bool(ok[rows[:most]].all())
        assert bool((got[rows[most:]] == -3).all())


@pytest.mark.parametrize("dtype", [F16, E4], ids=["fp16", "e4m3"])
def test_shared_pages_and_packed_slices(pkg, dev, dtype):
    """Two sequences share the pages of a common prefix; q, k, v are slices of one
    packed projection and the results slices of one packed buffer."""
    hd, heads, page = 64, 2, 16
    pool = pr.Pool([(3, 67), (3, 70)], page, heads, hd, dtype, 3)
    for which in (0, 1):  # the first 48 tokens are the same
        pool.data[1][which][:48] = pool.data[0][which][:48]
    pool.table[1, :3] = pool.table[0, :3]
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled(upto=[64, 67])))
    batch = _batch(pkg, dev, pool)
    q = torch.randn(pool.tokens, heads, hd, generator=pool.q_gen).half()
    packed = torch.stack((q, pool.rows(0), pool.rows(1)), 1).to(dev)  # [T, 3, heads, hd]
    pkg.ops.paged_append(packed[:, 1], packed[:, 2], cache, batch)
    both = torch.zeros(pool.tokens, 2, heads, hd, dtype=F16, device=dev)
    pkg.ops.paged_read(cache, batch, out=(both[:, 0], both[:, 1]))
    for which in (0, 1):
        want = torch.cat([pool.values(b, which)[kv - 3:] for b, (_, kv) in enumerate(pool.lens)])
        assert torch.equal(both[:, which].cpu(), want.float().half())
    out = torch.zeros(pool.tokens, 3 * heads * hd, dtype=F16, device=dev)[:, heads * hd:2 * heads * hd]
    got = pkg.ops.paged_attention(packed[:, 0], cache, batch, out=out)
    _check(pool, got.double().cpu(), q, 1)


def test_two_streams_at_once(pkg, dev):
    """Split decodes on two streams of one cache at the same time, many times over."""
    pool = pr.Pool([(1, 6000), (1, 5000)], 64, 1, 128, I8, 5)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    batch = _batch(pkg, dev, pool, **_hints(pool))
    qs = [torch.randn(2, 8, 128, generator=pool.q_gen).half().to(dev) for _ in range(2)]
    alone = [pkg.ops.paged_attention(q, cache, batch) for q in qs]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(pkg.ops.paged_attention(qs[i], cache, batch))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
def test_running_sequences(pkg, dev, dtype):
    """Prompts written whole, then single tokens and drafts, as a server runs:
    write, attend, step by step; also captured once and replayed with other
    lengths in the same tensors, on another stream."""
    hd, heads, group, page = 64, 2, 3, 16
    steps = [[(40, 40), (5, 5)], [(1, 41), (1, 6)], [(4, 45), (1, 7)], [(0, 45), (30, 37)]]
    pool = pr.Pool(steps[-1], page, heads, hd, dtype, 21)
    cache = pkg.PagedKVCache(pool.pages, page, heads, hd, dtype, dev)
    tables = pool.table.to(dev)
    for lens in steps:
        pool.lens = lens
        pool.start = torch.tensor([0, lens[0][0], lens[0][0] + lens[1][0]], dtype=torch.int32)
        pool.kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32)
        pool.tokens = int(pool.start[-1])
        part = pr.Pool.__new__(pr.Pool)
        part.__dict__.update(pool.__dict__)
        part.data = [[x[:kv] for x in d] for d, (_, kv) in zip(pool.data, lens)]
        batch = pkg.PagedBatch(tables, part.start.to(dev), part.kv.to(dev), part.tokens)
        q = torch.randn(part.tokens, heads * group, hd, generator=pool.q_gen).half()
        pkg.ops.paged_append(part.rows(0).to(dev), part.rows(1).to(dev), cache, batch)
        got = pkg.ops.paged_attention(q.to(dev), cache, batch).double().cpu()
        _check(part, got, q, group)


def test_captured_steps_follow_the_tensors(pkg, dev):
    """A decode step captured once: replays take what query_start, kv_len, the
    page table and the inputs hold then. Two graphs and an eager call on other
    streams keep apart."""
    hd, heads, page = 64, 4, 16
    lens = [(1, 600), (1, 900), (1, 3)]
    pool = pr.Pool(lens, page, heads, hd, I8, 8)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    q = torch.randn(3, heads, hd, generator=pool.q_gen).half()
    kv, qd = pool.kv.to(dev), q.to(dev)
    batch = pkg.PagedBatch(pool.table.to(dev), pool.start.to(dev), kv, 3, max_query_len=1)
    graphs, outs = [], []
    warm = pkg.ops.paged_attention(qd, cache, batch)
    side = torch.cuda.Stream()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.ops.paged_attention(qd, cache, batch))
        graphs.append(g)
    for cut in ((600, 900, 3), (17, 258, 1), (599, 1, 2)):
        kv.copy_(torch.tensor(cut, dtype=torch.int32))
        part = pr.Pool.__new__(pr.Pool)
        part.__dict__.update(pool.__dict__)
        part.lens = [(1, c) for c in cut]
        part.data = [[x[:c] for x in d] for d, c in zip(pool.data, cut)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
            eager = pkg.ops.paged_attention(qd, cache, batch)
        graphs[1].replay()
        torch.cuda.synchronize()
        for got in (outs[0], outs[1], eager):
            _check(part, got.double().cpu(), q, 1)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], eager)
    assert warm.shape == (3, heads * hd)


@pytest.mark.parametrize("dtype,hd,heads", [(F16, 64, 16), (F16, 128, 10), (I8, 128, 10),
                                            (E4, 256, 8)],
                         ids=lambda v: NAMES.get(v, str(v)) if not isinstance(v, int) else str(v))
def test_chained_steps_of_prompts_and_single_tokens(pkg, dev, dtype, hd, heads):
    """Both attention kernels of a mixed batch run at the same time; what follows
    finds both done: each step writes its tokens from the step before and attends,
    with nothing between the calls, against the same steps one at a time."""
    lens, group = [(1, 900), (190, 1100), (1, 3000), (17, 30), (140, 140), (1, 1), (6, 2000)], 2
    pool = pr.Pool(lens, 64, heads, hd, dtype, 31)
    batch = _batch(pkg, dev, pool, **_hints(pool))
    q = torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen).half().to(dev)
    filled = pool.on(dev, pool.filled())

    def steps(cache, pause):
        outs, x = [], q
        for _ in range(6):
            pkg.ops.paged_append(x[:, :heads], x[:, heads:], cache, batch)
            pause()
            out = pkg.ops.paged_attention(x, cache, batch)
            pause()
            outs.append(out)
            x = out.view(pool.tokens, heads * group, hd)
        return outs

    def fresh():
        return pkg.PagedKVCache.from_tensors(*[None if t is None else t.clone() for t in filled])

    alone = steps(fresh(), torch.cuda.synchronize)
    for _ in range(5):
        got = steps(fresh(), lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))
    cache = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = steps(cache, lambda: None)
    for _ in range(3):
        for new, old in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), filled):
            if old is not None:
                new.copy_(old)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_offsets_past_32_bits(pkg, dev):
    """Pages whose offset passes 2^32 elements (8-bit codes: 4.3 GB of K and of V)."""
    heads, hd, page = 16, 128, 256
    pages = 2 ** 32 // (heads * hd * page) + 3
    k = torch.empty(pages, heads, page, hd, dtype=I8, device=dev).transpose(1, 2)
    v = torch.empty_like(k)
    s = [torch.empty(pages, heads, page, device=dev) for _ in range(2)]
    cache = pkg.PagedKVCache.from_tensors(k, v, *s)
    pool = pr.Pool([(300, 300)], page, heads, hd, I8, 6)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    batch = pkg.PagedBatch(table, pool.start.to(dev), pool.kv.to(dev), 300)
    pkg.ops.paged_append(pool.rows(0).to(dev), pool.rows(1).to(dev), cache, batch)
    got, _ = pkg.ops.paged_read(cache, batch)
    assert torch.equal(got.cpu(), pool.values(0, 0).float().half())
    last = pkg.PagedBatch(table, torch.tensor([0, 1], dtype=torch.int32, device=dev), batch.kv_len, 1)
    pool.lens, pool.start, pool.tokens = [(1, 300)], torch.tensor([0, 1]), 1
    q = torch.randn(1, heads, hd, generator=pool.q_gen).half()
    _check(pool, pkg.ops.paged_attention(q.to(dev), cache, last).double().cpu(), q, 1)


def test_no_device_timeout(pkg, dev):
    torch.cuda.synchronize()
    assert pkg._lib.read_device_error() == 0
