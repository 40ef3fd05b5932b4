"""The paged KV cache on the host, where it is most likely to go wrong: no GPU is needed."""

from __future__ import annotations

import ctypes
import importlib
import threading

import pytest
import torch

import paged_reference as pr
from conftest import load_package

F16, I8, E4 = torch.float16, torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [F16, I8, E4], ids=["fp16", "int8", "e4m3"])
@pytest.mark.parametrize("lens", [[(4, 300), (1, 64), (7, 7), (3, 1025), (0, 0), (2, 31)],
                                  [(130, 400), (1, 77), (64, 64), (257, 300), (31, 1000)]],
                         ids=["draft", "chunk"])
def test_the_tolerance_can_fail(dtype, lens):
    """A value of 60000 in one token: results of zero, and results that a token leaks into which
    the row does not see, are far outside the tolerance of the rows that do not see it."""
    pool, group = pr.Pool(lens, 16, 2, 64, dtype, 11), 2
    pool.data[2][1][5, 1, :] = 60000.0
    q = (1.5 * torch.randn(pool.tokens, 4, 64, generator=pool.q_gen)).half()
    ref, tol = (x.view(pool.tokens, 4, 64) for x in pr.attention_own(pool, q, group))
    plain = pr.attention(pool, q, group)[0].view_as(ref)
    assert bool(((ref - plain).abs() <= 1e-13 * (1 + ref.abs())).all())
    blind = torch.ones(pool.tokens, 4, dtype=torch.bool)  # (row, head) that do not see it
    first, n = int(pool.start[2]), lens[2][0]
    blind[first + 5:first + n, 2:] = False
    zero = (ref.abs() > tol)[blind]
    assert float(zero.double().mean()) > 0.97 and bool(zero.any(-1).all())
    leaky = pr.attention_own(pool, q, group, causal=False)[0].view_as(ref)
    leaked = ((leaky - ref).abs() > tol)[first:first + 5, 2:]
    assert bool(leaked.all())


def test_sizes_past_32_bits():
    """Sizes are ints in the C structures: a longer one is refused, never cut to what is left of
    it; a bound above num_tokens says as much as num_tokens does."""
    pkg = load_package()
    i = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")  # noqa: E731
    batch = pkg.PagedBatch(i(1, 4), i(2), i(1), 7, max_query_len=2 ** 32)
    assert batch.max_query_len == 2 ** 32 and batch._struct.max_query_len == 7
    assert pkg.PagedBatch(i(1, 4), i(2), i(1), 7, max_query_len=3)._struct.max_query_len == 3
    assert pkg.PagedBatch(i(1, 4), i(2), i(1), 7, max_kv_len=2 ** 33)._struct.max_kv_len == 2 ** 30
    for args in ((i(1, 4), i(2), i(1), 2 ** 32 + 7), (i(1, 2 ** 32 + 4), i(2), i(1), 7),
                 (i(2 ** 31, 1), i(2 ** 31 + 1), i(2 ** 31), 7)):
        with pytest.raises(ValueError, match="2\\^31"):
            pkg.PagedBatch(*args)
    pool = torch.empty(2 ** 31, 16, 1, 8, dtype=F16, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        pkg.PagedKVCache.from_tensors(pool, pool)
    cache = pkg.PagedKVCache(3, 16, 1, 8, F16, "meta")
    one = pkg.PagedBatch(i(1, 4), i(2), i(1), 1)
    q = torch.empty(1, 2 ** 32 + 1, 8, dtype=F16, device="meta")
    for handle in (cache, one):
        handle.__dict__["_index"] = q.get_device()  # as if they were on a GPU
    with pytest.raises(ValueError, match="2\\^31"):
        pkg.ops.paged_attention(q, cache, one)


def test_geometries_made_at_once(monkeypatch):
    """Two threads that make caches of different sizes at the same moment get different numbers
    (a batch keeps the workspace sizes of its calls under them)."""
    pkg = load_package()
    paged = importlib.import_module(pkg.__name__ + ".paged")

    class Late(dict):  # both have looked before either has written
        def __init__(self):
            super().__init__()
            self.looked = threading.Barrier(2)

        def setdefault(self, key, value):
            self.looked.wait(20)
            return super().setdefault(key, value)

    monkeypatch.setattr(paged, "_GEOMETRIES", Late())
    caches = {}

    def make(hd):
        caches[hd] = pkg.PagedKVCache(2, 16, 1, hd, F16, "cpu")

    threads = [threading.Thread(target=make, args=(hd,)) for hd in (8, 256)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert caches[8]._geometry != caches[256]._geometry


def test_workspace_is_planned_on_the_cache_s_device(monkeypatch):
    """The plan depends on the device's SM count: it is made where the call will run, whichever
    device is current."""
    pkg = load_package()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    current, planned = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Lib:
        @staticmethod
        def tfx_paged_attention_workspace_bytes(cache, batch, heads):
            planned.append((current[-1], heads))
            return 512

    monkeypatch.setattr(torch.cuda, "device", Device)
    cache, batch = pkg.PagedKVCache(2, 16, 1, 8, F16, "cpu"), pkg.PagedBatch(i(1, 2), i(2), i(1), 1)
    batch.__dict__["_index"] = 3
    assert [batch._workspace_bytes(Lib, cache, h) for h in (4, 4, 8)] == [512] * 3
    assert planned == [(3, 4), (3, 8)]


def test_append_refuses_one_memory_for_keys_and_values():
    """Every slot would hold parts of both."""
    pkg = load_package()
    importlib.import_module(pkg.__name__ + ".build").build()
    L = pkg._lib
    lib = L.load()
    batch = ctypes.byref(L.TfxPagedBatch(256, 6, 6, 320, 384, 3, 0, 4, 80))  # no token: no launch
    for k, v, ks, vs, want in ((4096, 8192, 512, 1024, 0), (4096, 4096, 512, 1024, L.TFX_ERR_INVALID_ARGUMENT),
                               (4096, 8192, 512, 512, L.TFX_ERR_INVALID_ARGUMENT)):
        cache = ctypes.byref(L.TfxPagedCache(k, v, ks, vs, L.TFX_CACHE_INT8, 10, 16, 2, 64, 2048, 64, 1024))
        assert lib.tfx_paged_append(4096, 128, 8192, 128, cache, batch, None) == want
        assert lib.tfx_paged_read(cache, batch, 4096, 128, 8192, 128, None) == 0  # reading is fine
