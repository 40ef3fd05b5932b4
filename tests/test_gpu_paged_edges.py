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
