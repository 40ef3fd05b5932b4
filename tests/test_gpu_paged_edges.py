"""The paged KV cache on a B200 where it is most likely to go wrong: against the 64-bit
model with tolerances from the keys that a row sees itself."""

from __future__ import annotations

import pytest
import torch

import paged_reference as pr
from test_gpu_paged import CHUNK, DRAFT, E4, F16, I8, NAMES, _batch, _hints, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _ids(v):
    return NAMES.get(v, str(v)) if not isinstance(v, (int, str)) else str(v)


@pytest.mark.parametrize("hd,heads,lens", [(64, 4, [(300, 20000)]), (64, 20, [(129, 3000), (700, 5000)]),
                                           (128, 4, [(300, 20000)]), (128, 20, [(129, 3000), (700, 5000)]),
                                           (256, 8, [(140, 9000), (65, 4000)])])
def test_prompt_parts_behind_long_prefixes(pkg, dev, hd, heads, lens):  # noqa: F811
    """Many tiles that every row sees all of before the ones that some do not, several to each
    stage of the ring: every pass ends and gives the same, whoever in a CTA is late."""
    pool = pr.Pool(lens, 16, heads, hd, F16, 41)
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    batch = _batch(pkg, dev, pool, **_hints(pool))
    q = torch.randn(pool.tokens, heads, hd, generator=pool.q_gen).half()
    outs = [pkg.ops.paged_attention(q.to(dev), cache, batch) for _ in range(20)]
    torch.cuda.synchronize()
    assert pkg._lib.read_device_error() == 0
    assert all(torch.equal(o, outs[0]) for o in outs)
    few = torch.cat([torch.arange(n - 3, n) + int(s) for (n, _), s in zip(lens, pool.start)])
    last = pr.Pool.__new__(pr.Pool)  # the last three tokens of each sequence
    last.__dict__.update(pool.__dict__)
    last.lens = [(3, kv) for _, kv in lens]
    last.start, last.tokens = torch.arange(len(lens) + 1, dtype=torch.int32) * 3, 3 * len(lens)
    ref, tol = pr.attention_own(last, q[few], 1)
    err = (outs[0].double().cpu()[few] - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _attend_own(pkg, dev, pool, group, q, tensors=None):  # noqa: F811
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled() if tensors is None else tensors))
    return pkg.ops.paged_attention(q.to(dev), cache, _batch(pkg, dev, pool, **_hints(pool))).double().cpu()


def _check_own(pool, got, q, group, rows=slice(None)):
    ref, tol = pr.attention_own(pool, q, group)
    err = (got - ref).abs()[rows]
    assert bool((err <= tol[rows]).all()), float((err / tol[rows]).max())


SHAPES = {"draft": ([(6, 300), (1, 64), (7, 7), (3, 1025), (2, 31)], 2, 2), "prompt": (CHUNK, 10, 2),
          "long": ([(2, 9000), (1, 5000)], 1, 4)}


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=_ids)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("kind", ["later", "earlier", "mixed", "zeros"])
def test_values_of_very_different_sizes(pkg, dev, dtype, hd, shape, kind):  # noqa: F811
    """The largest value there is, in a token that a row does not see or gives no weight,
    beside small ones; tokens of every size; values of zero with nearly all the weight."""
    lens, heads, group = SHAPES[shape]
    for small in (1.0, 1e-2, 1e-3) if kind in ("later", "earlier") else (1.0,):
        pool = pr.Pool(lens, 16, heads, hd, dtype, 51)
        q = (1.5 * torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen)).half()
        q[:, :, 0] = 4.0
        for (k, v), (n, kv) in zip(pool.data, lens):
            v *= small
            if kind == "later" and n > 1:
                v[-1] = 65504.0
            if kind == "earlier" and kv > n:
                v[kv // 3 if kv // 3 < kv - n else 0] = 65504.0
            if kind == "mixed":
                size = 10.0 ** (8 * torch.rand(kv, heads, 1, generator=pool.q_gen) - 4)
                v.copy_((v.float() * size).clamp(-65504, 65504))
            at = kv // 3 if kv // 3 < kv - n else 0
            if kind in ("earlier", "zeros") and kv > n:
                k[at] = 0
                k[at, :, 0] = (-15.0 if kind == "earlier" else 5.0) * hd ** 0.5  # 60 less, 20 more
            if kind == "zeros":
                v[::3] = 0
                v[at] = 0
        tensors = pool.filled()
        if kind == "zeros" and dtype != F16:  # a scale of zero makes any code zero
            codes, scale = tensors[1].view(torch.uint8), tensors[3].transpose(1, 2)
            codes[scale == 0] = 0x55
        got = _attend_own(pkg, dev, pool, group, q, tensors)
        _check_own(pool, got, q, group)


@pytest.mark.parametrize("dtype", [I8, E4], ids=_ids)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("scale", [-0.01, float("inf"), float("nan")])
def test_scales_that_are_none(pkg, dev, dtype, hd, shape, scale):  # noqa: F811
    """A value's scale that is negative, infinite or NaN makes the rows that see it NaN, in its
    head, and no other."""
    lens, heads, group = SHAPES[shape]
    pool = pr.Pool(lens, 16, heads, hd, dtype, 52)
    q = torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen).half()
    tensors, hit = pool.filled(), torch.zeros(pool.tokens, heads * group, dtype=torch.bool)
    for b, pos in ((0, lens[0][1] - 2), (2 % len(lens), 0)):  # not seen by all; seen by all
        page, slot = pool.place(b, pos)
        tensors[3][page, 0, slot] = scale
        n, kv = lens[b]
        first = int(pool.start[b]) + max(0, pos - (kv - n))
        hit[first:int(pool.start[b]) + n, :group] = True
    got = _attend_own(pkg, dev, pool, group, q, tensors).view(pool.tokens, heads * group, hd)
    ref, tol = pr.attention_own(pool, q, group)
    ref, tol = ref.view_as(got), tol.view_as(got)
    assert bool(torch.isnan(got[hit]).all())
    err = (got - ref).abs()[~hit]
    assert bool((err <= tol[~hit]).all()), float((err / tol[~hit]).max())


def test_more_row_blocks_than_a_grid_has(pkg, dev):  # noqa: F811
    """65600 new tokens in groups of 65 at head_dim 256, one to a CTA of the tcgen05 kernel.
    (All but the last 40 have no position, and so see nothing.)"""
    pool, group, many = pr.Pool([(40, 40), (3, 500)], 16, 1, 256, F16, 61), 65, 65600
    cache = pkg.PagedKVCache.from_tensors(*pool.on(dev, pool.filled()))
    table = torch.full((2, 64), -1, dtype=torch.int32)
    table[:, :pool.table.shape[1]] = pool.table
    q = torch.randn(pool.tokens, group, 256, generator=pool.q_gen).half()
    rows = torch.zeros(many + 3, group, 256, dtype=F16, device=dev)
    rows[many - 40:] = q.to(dev)
    start = torch.tensor([0, many, many + 3], dtype=torch.int32, device=dev)
    got = pkg.ops.paged_attention(rows, cache, pkg.PagedBatch(table.to(dev), start, pool.kv.to(dev),
                                                              many + 3))
    assert bool((got[:many - 40] == 0).all())
    _check_own(pool, got[many - 40:].double().cpu(), q, group)


@pytest.mark.parametrize("dtype,hd,heads", [(F16, 32, 3), (F16, 64, 16), (F16, 128, 10), (I8, 64, 16),
                                            (I8, 128, 10), (E4, 256, 8)], ids=_ids)
def test_one_capture_for_every_batch(pkg, dev, dtype, hd, heads):  # noqa: F811
    """Write, attend and read back, captured once: replays on another stream take the lengths,
    starts, pages and rows that the tensors hold then, whether prompts, running sequences or
    both; rows of no sequence stay as they were."""
    group, page, rows, width, pages = 2, 16, 310, 80, 160
    index = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    table, start, kv = index(3, width), index(4), index(3)
    cache = pkg.PagedKVCache(pages, page, heads, hd, dtype, dev)
    batch = pkg.PagedBatch(table, start, kv, rows, max_query_len=300)
    new = torch.zeros(rows, 2, heads, hd, dtype=F16, device=dev)
    q = torch.zeros(rows, heads * group, hd, dtype=F16, device=dev)
    out = torch.zeros(rows, heads * group * hd, dtype=F16, device=dev)
    back = tuple(torch.zeros(rows, heads, hd, dtype=F16, device=dev) for _ in range(2))

    def step():
        pkg.ops.paged_append(new[:, 0], new[:, 1], cache, batch)
        pkg.ops.paged_attention(q, cache, batch, out=out)
        pkg.ops.paged_read(cache, batch, out=back)

    step()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        step()
    batches = [[(250, 900), (1, 500), (49, 49)], [(1, 700), (1, 1), (200, 1100)],
               [(0, 64), (300, 300), (0, 0)], [(1, 33), (1, 1279), (1, 800)], [(8, 40), (0, 7), (3, 1200)]]
    for seed, lens in enumerate(batches):
        pool = pr.Pool(lens, page, heads, hd, dtype, 70 + seed)
        assert pool.pages <= pages
        torch.cuda.synchronize()
        for mine, there in zip((cache.k, cache.v, cache.k_scale, cache.v_scale),
                               pool.on(dev, pool.filled(upto=[m - n for n, m in lens]))):
            if mine is not None:
                bits = (lambda t: t.view(torch.uint8)) if mine.dtype in (I8, E4) else (lambda t: t)
                bits(mine)[:pool.pages].copy_(bits(there))
        table.fill_(-1)
        table[:, :min(width, pool.table.shape[1])] = pool.table[:, :width].to(dev)
        start.copy_(pool.start)
        kv.copy_(pool.kv)
        new.zero_()
        new[:pool.tokens] = torch.stack((pool.rows(0), pool.rows(1)), 1).to(dev)
        qs = torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen).half()
        q[:pool.tokens] = qs.to(dev)
        for t in (out, *back):
            t.fill_(-3)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        for t in (out, *back):
            assert bool((t[pool.tokens:] == -3).all())
        _check_own(pool, out[:pool.tokens].double().cpu(), qs, group)
        for which in (0, 1):
            want = torch.cat([pool.values(b, which)[m - n:] for b, (n, m) in enumerate(lens)])
            assert torch.equal(back[which][:pool.tokens].cpu(), want.float().half())


@pytest.mark.parametrize("hd", [8, 32, 64, 128, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_infinite_scores(pkg, dev, hd, shape):  # noqa: F811
    """A key whose score is -inf has no weight; a row that sees no other key is zero, as one that
    sees none. A score of +inf makes its row NaN."""
    lens, heads, group = SHAPES[shape]
    pool = pr.Pool(lens, 16, heads, hd, F16, 81)
    q = torch.randn(pool.tokens, heads * group, hd, generator=pool.q_gen).half()
    q[:, :, 0] = 2.0
    tensors = pool.filled()
    hidden = {0: [0, lens[0][1] // 2, lens[0][1] - 1], len(lens) - 1: range(lens[-1][1])}
    for b, positions in hidden.items():
        for pos in positions:
            page, slot = pool.place(b, pos)
            tensors[0][page, slot, :, 0] = -float("inf")
            pool.data[b][0][pos] = 0
            pool.data[b][0][pos, :, 0] = -60000.0  # no weight left either
    if len(lens) > 2:  # the first key of a sequence in between
        page, slot = pool.place(1, 0)
        tensors[0][page, slot, 0, 0] = float("inf")
    got = _attend_own(pkg, dev, pool, group, q, tensors).view(pool.tokens, heads * group, hd)
    ref, tol = (x.view_as(got) for x in pr.attention_own(pool, q, group))
    fine = torch.ones(pool.tokens, heads * group, dtype=torch.bool)
    if len(lens) > 2:
        row = slice(int(pool.start[1]), int(pool.start[2]))
        assert bool(torch.isnan(got[row, :group]).all())
        fine[row, :group] = False
    last = slice(int(pool.start[-2]), pool.tokens)
    assert bool((got[last] == 0).all())
    fine[last] = False
    err = (got - ref).abs()[fine]
    assert bool((err <= tol[fine]).all()), float((err / tol[fine]).max())
