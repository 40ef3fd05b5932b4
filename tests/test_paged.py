"""What the paged KV cache refuses, on the host: no GPU is needed. And the
64-bit model of the GPU tests against itself."""

from __future__ import annotations

import ctypes

import pytest
import torch

import paged_reference as pr
from conftest import load_package

F16, I8, E4 = torch.float16, torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    pkg = load_package()
    __import__("importlib").import_module(pkg.__name__ + ".build").build()
    return pkg._lib.load()


def _structs(L, **kw):
    """A well-formed cache and batch over fake addresses; kw changes fields."""
    c = L.TfxPagedCache(4096, 8192, 512, 1024, L.TFX_CACHE_INT8, 10, 16, 2, 64, 2048, 64, 1024)
    b = L.TfxPagedBatch(256, 6, 6, 320, 384, 3, 7, 4, 80)
    for name, value in kw.items():
        setattr(c if hasattr(c, name) else b, name, value)
    return ctypes.byref(c), ctypes.byref(b)


BAD = [
    ({"k": None}, "INVALID_ARGUMENT"), ({"v": None}, "INVALID_ARGUMENT"),
    ({"k_scale": None}, "INVALID_ARGUMENT"), ({"page_table": None}, "INVALID_ARGUMENT"),
    ({"query_start": None}, "INVALID_ARGUMENT"), ({"kv_len": None}, "INVALID_ARGUMENT"),
    ({"dtype": 3}, "INVALID_ARGUMENT"), ({"dtype": -1}, "INVALID_ARGUMENT"),
    ({"num_pages": 0}, "INVALID_ARGUMENT"), ({"kv_heads": 0}, "INVALID_ARGUMENT"),
    ({"batch": 0}, "INVALID_ARGUMENT"), ({"max_pages": 0}, "INVALID_ARGUMENT"),
    ({"num_tokens": -1}, "INVALID_ARGUMENT"), ({"max_query_len": -1}, "INVALID_ARGUMENT"),
    ({"max_kv_len": -1}, "INVALID_ARGUMENT"), ({"table_stride": 5}, "INVALID_ARGUMENT"),
    ({"page_stride": 63}, "INVALID_ARGUMENT"), ({"token_stride": -64}, "INVALID_ARGUMENT"),
    ({"head_stride": 0}, "INVALID_ARGUMENT"),
    ({"head_dim": 48}, "UNSUPPORTED"), ({"head_dim": 8}, "UNSUPPORTED"),
    ({"page_size": 8}, "UNSUPPORTED"), ({"page_size": 48}, "UNSUPPORTED"),
    ({"page_size": 512}, "UNSUPPORTED"), ({"batch": 65536}, "UNSUPPORTED"),
    ({"kv_heads": 65536}, "UNSUPPORTED"), ({"num_tokens": 1 << 30}, "UNSUPPORTED"),
    ({"max_pages": (1 << 26) + 1, "table_stride": 1 << 27}, "UNSUPPORTED"),
    ({"k": 4104}, "MISALIGNED"), ({"token_stride": 72}, "MISALIGNED"),
    ({"page_stride": 2056}, "MISALIGNED"), ({"head_stride": 1032}, "MISALIGNED"),
    ({"k_scale": 514}, "MISALIGNED"), ({"page_table": 258}, "MISALIGNED"),
    ({"kv_len": 386}, "MISALIGNED"), ({"query_start": 321}, "MISALIGNED"),
]


@pytest.mark.parametrize("change,status", BAD, ids=lambda v: str(v))
def test_bad_caches_and_batches(lib, change, status):
    L = load_package()._lib
    want = getattr(L, "TFX_ERR_" + status)
    c, b = _structs(L, **change)
    heads = change.get("kv_heads", 2) or 2
    ld = 65536 * 64
    assert lib.tfx_paged_append(4096, ld, 8192, ld, c, b, None) == want
    assert b"tfx_paged_append" in lib.tfx_last_error_message()
    assert lib.tfx_paged_read(c, b, 4096, ld, 8192, ld, None) == want
    assert lib.tfx_paged_attention(4096, ld, c, b, 8192, ld, heads, 0.1, 1, 4096, 1 << 40,
                                   None) == want
    assert lib.tfx_paged_attention_workspace_bytes(c, b, heads) == -1


def test_bad_calls(lib):
    L = load_package()._lib
    c, b = _structs(L)
    inv, mis = L.TFX_ERR_INVALID_ARGUMENT, L.TFX_ERR_MISALIGNED
    copy = [(None, 128, 8192, 128, inv), (4096, 128, None, 128, inv), (4096, 120, 8192, 128, inv),
            (4096, 128, 8192, 127, inv), (4096, 132, 8192, 128, mis), (4098, 128, 8192, 128, mis)]
    for k, ld_k, v, ld_v, want in copy:
        assert lib.tfx_paged_append(k, ld_k, v, ld_v, c, b, None) == want
        assert lib.tfx_paged_read(c, b, k, ld_k, v, ld_v, None) == want
    assert lib.tfx_paged_append(4096, 128, 8192, 128, None, b, None) == inv
    assert lib.tfx_paged_read(c, None, 4096, 128, 8192, 128, None) == inv
    need = lib.tfx_paged_attention_workspace_bytes(c, b, 4)
    assert need >= 0 and need % 256 == 0
    attend = lambda q=4096, ld_q=256, out=8192, ld_out=256, heads=4, scale=0.1, ws=4096, n=1 << 40: (  # noqa: E731
        lib.tfx_paged_attention(q, ld_q, c, b, out, ld_out, heads, scale, 1, ws, n, None))
    for kw, want in (({"q": None}, inv), ({"out": None}, inv), ({"heads": 3}, inv),
                     ({"heads": 0}, inv), ({"heads": -2}, inv), ({"ld_q": 248}, inv),
                     ({"ld_out": 255}, inv), ({"scale": 0.0}, inv), ({"scale": -1.0}, inv),
                     ({"scale": float("nan")}, inv), ({"scale": float("inf")}, inv),
                     ({"scale": 3e38}, inv), ({"q": 4100}, mis), ({"out": 8200}, mis),
                     ({"ld_q": 260}, mis), ({"ld_out": 260}, mis)):
        assert attend(**kw) == want, kw
    # outputs over inputs, K over V; slices of one packed row are fine
    assert attend(out=4096) == inv and b"overlap" in lib.tfx_last_error_message()
    assert attend(out=4096 + 512 * 3) == inv  # 7 rows of 512 bytes
    assert attend(out=4096 + 128, ld_q=264) == inv
    assert lib.tfx_paged_read(c, b, 4096, 128, 4096 + 256, 128, None) == inv
    assert lib.tfx_paged_read(c, b, 4096, 256, 4096 + 128, 256, None) == inv
    # keys long enough to be split: the workspace is checked
    c, b = _structs(L, max_pages=4096, table_stride=4096, max_kv_len=65536)
    need = lib.tfx_paged_attention_workspace_bytes(c, b, 4)
    assert need > 0
    assert attend(ws=None) == inv
    assert attend(ws=4096 + 16) == mis
    assert attend(n=need - 1) == L.TFX_ERR_WORKSPACE
    assert lib.tfx_paged_attention_workspace_bytes(c, b, 3) == -1
    # nothing to do: nothing is enqueued
    c, b = _structs(L, num_tokens=0)
    assert lib.tfx_paged_append(4096, 128, 8192, 128, c, b, None) == 0
    assert lib.tfx_paged_read(c, b, 4096, 128, 8192, 128, None) == 0
    assert lib.tfx_paged_attention(4096, 256, c, b, 8192, 256, 4, 0.1, 1, None, 0, None) == 0


def _cpu_cache(pkg, dtype=I8, pages=3, page=16, heads=2, hd=64):
    return pkg.PagedKVCache(pages, page, heads, hd, dtype, "cpu")


def test_cache_objects():
    pkg = load_package()
    c = _cpu_cache(pkg)
    assert c.k.shape == (3, 16, 2, 64) and c.k_scale.shape == (3, 2, 16)
    assert (c.num_pages, c.page_size, c.kv_heads, c.head_dim, c.dtype) == (3, 16, 2, 64, I8)
    assert _cpu_cache(pkg, F16).k_scale is None
    x = lambda *s, t=F16: torch.zeros(s, dtype=t)  # noqa: E731
    make = pkg.PagedKVCache.from_tensors
    good = make(x(3, 16, 1, 64), x(3, 16, 1, 64))  # a dimension of size 1: any stride
    assert good._struct.head_stride == 64 and good._struct.token_stride == 64
    s = torch.zeros(3, 2, 16)
    for args in ((x(3, 16, 2, 64), x(3, 16, 2, 32)), (x(3, 16, 2, 64), x(3, 16, 2, 64, t=I8)),
                 (x(3, 16, 64), x(3, 16, 64)), (x(3, 16, 2, 64, t=torch.bfloat16),) * 2,
                 (x(3, 16, 2, 64), x(3, 2, 16, 64).transpose(1, 2)),
                 (x(3, 16, 64, 2).transpose(2, 3),) * 2,
                 (x(3, 16, 2, 64), x(3, 16, 2, 64), s, s), (x(3, 16, 2, 64, t=I8),) * 2,
                 (x(3, 16, 2, 64, t=I8), x(3, 16, 2, 64, t=I8), s, s[:2]),
                 (x(3, 16, 2, 64, t=I8), x(3, 16, 2, 64, t=I8), s, s.half()),
                 (x(3, 16, 2, 64, t=I8), x(3, 16, 2, 64, t=I8), s,
                  torch.zeros(3, 16, 2).transpose(1, 2))):
        with pytest.raises(ValueError):
            make(*args)


def test_batch_objects():
    pkg = load_package()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    b = pkg.PagedBatch(i(3, 4), i(4), i(3), 9)
    assert b.max_query_len == 9 and b.num_tokens == 9
    assert pkg.PagedBatch(i(3, 8)[:, :4], i(4), i(3), 9)._struct.table_stride == 8
    for args in ((i(3), i(4), i(3), 1), (i(3, 4), i(3), i(3), 1), (i(3, 4), i(4), i(4), 1),
                 (i(0, 4), i(1), i(0), 1), (i(3, 0), i(4), i(3), 1),
                 (i(3, 4).long(), i(4), i(3), 1), (i(3, 4), i(4).float(), i(3), 1),
                 (i(4, 3).t(), i(4), i(3), 1), (i(3, 4), i(8)[::2], i(3), 1),
                 (i(3, 4), i(4), i(3), -1), (i(3, 4), i(4), i(3), 1, -1),
                 (i(3, 4), i(4), i(3), 1, 1, -1)):
        with pytest.raises(ValueError):
            pkg.PagedBatch(*args)


def test_ops_refuse_cpu_tensors():
    pkg = load_package()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cache, batch = _cpu_cache(pkg), pkg.PagedBatch(i(1, 2), i(2), i(1), 4)
    x = torch.zeros(4, 2, 64, dtype=F16)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.ops.paged_append(x, x, cache, batch)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.ops.paged_read(cache, batch)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.ops.paged_attention(x, cache, batch)


def test_the_model_of_the_cache():
    """quantise() picks the nearest of all codes; attention() is a plain softmax."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(40, 16, generator=g) * torch.logspace(-6, 4, 40)[:, None]).half()
    for dtype in (I8, E4):
        code, scale = pr.quantise(x, dtype)
        every = torch.arange(256, dtype=torch.uint8).view(dtype).float().double()
        every = every[torch.isfinite(every) & (every.abs() <= pr.TOP[dtype])]
        y = x.double() / scale[:, None].double()
        best = (y[..., None] - every).abs().amin(-1)
        assert torch.equal((y - code.float().double()).abs(), best)
    pool = pr.Pool([(5, 9), (3, 3)], 16, 2, 16, F16, 0)
    q = torch.randn(8, 4, 16, generator=g).half()
    out, _, _ = pr.attention(pool, q, 2)
    k, v = pool.values(0, 0), pool.values(0, 1)
    w = torch.softmax(q[4, 3].double() @ k[:, 1].T / 4, -1)
    assert torch.allclose(out[4].view(4, 16)[3], w @ v[:, 1], atol=1e-14)


def test_handles_are_fixed():
    """The C structures hold the tensors' addresses: replacing one would leave them behind."""
    pkg = load_package()
    cache = pkg.PagedKVCache(3, 16, 2, 32, I8, "cpu")
    batch = pkg.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32),
                           torch.zeros(2, dtype=torch.int32), 4)
    for obj, name, value in ((cache, "k", cache.k.clone()), (cache, "k_scale", None),
                             (cache, "head_dim", 16), (batch, "num_tokens", 2),
                             (batch, "kv_len", torch.ones(2, dtype=torch.int32)),
                             (batch, "max_query_len", 1)):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(obj, name, value)
    batch.kv_len.fill_(5)
