"""Tensor-level wrappers over the C ABI, mirroring the reference's op layer.

Same names, argument meaning and error behaviour as the reference's Python
kernels where one exists (``layer_norm`` / ``fused_residual_layer_norm`` of
triton_fused_norm.py:140-215), plus the ops the reference took from PyTorch
(``F.linear``, ``torch._addmm_activation``, ``F.scaled_dot_product_attention``;
torch_transformer_benchmark.py:741, 767-818, 875-896). All work runs on the
current CUDA stream through ``lib/libtfx_b200.so``; there is no fallback.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .paged import PagedBatch, PagedKVCache


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA tensors")


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.float16:
        return _lib.TFX_DTYPE_F16
    if dtype == torch.float32:
        return _lib.TFX_DTYPE_F32
    raise ValueError(f"output dtype must be float16 or float32, got {dtype}")


def layer_norm(
    inputs: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    eps: float,
    output_dtype: torch.dtype,
    apply_affine: bool = True,
) -> torch.Tensor:
    """LayerNorm whose output is stored directly in the next GEMM's dtype.

    Mirrors triton_fused_norm.py:140-170: fp32 ``inputs`` [..., D], fp32
    statistics, output in ``output_dtype`` (float16 or float32).
    """
    _require_cuda(inputs, "the fused LayerNorm kernel")
    n_cols = inputs.shape[-1]
    if n_cols != weight.numel() or weight.shape != bias.shape:
        raise ValueError("LayerNorm parameters do not match the input width")
    if inputs.dtype != torch.float32:
        raise ValueError("layer_norm expects float32 inputs")
    x = inputs.contiguous()
    w = weight.detach().float().contiguous()
    b = bias.detach().float().contiguous()
    out = torch.empty(x.shape, device=x.device, dtype=output_dtype)
    rows = x.numel() // n_cols
    _lib.check(
        _lib.load().tfx_layer_norm(
            x.data_ptr(), w.data_ptr(), b.data_ptr(), out.data_ptr(), _dtype_code(output_dtype),
            rows, n_cols, float(eps), int(apply_affine), _stream(x.device),
        ),
        "tfx_layer_norm",
    )
    return out


def fused_residual_layer_norm(
    residual: torch.Tensor,
    update: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    eps: float,
    norm_dtype: torch.dtype,
    store_residual: bool = True,
    apply_affine: bool = True,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Return the fp32 residual sum and the normalised output in ``norm_dtype``.

    Mirrors triton_fused_norm.py:173-215 (``store_residual=False`` returns the
    input residual object, as the reference does).
    """
    _require_cuda(residual, "the fused LayerNorm kernel")
    if residual.shape != update.shape:
        raise ValueError("residual and update must have identical shapes")
    if residual.shape[-1] != weight.numel() or weight.shape != bias.shape:
        raise ValueError("LayerNorm parameters do not match the input width")
    if residual.dtype != torch.float32:
        raise ValueError("residual must be float32")
    n_cols = residual.shape[-1]
    r = residual.contiguous()
    u = update.to(torch.float16).contiguous()
    w = weight.detach().float().contiguous()
    b = bias.detach().float().contiguous()
    r_out = torch.empty_like(r) if store_residual else r
    out = torch.empty(r.shape, device=r.device, dtype=norm_dtype)
    rows = r.numel() // n_cols
    _lib.check(
        _lib.load().tfx_residual_layer_norm(
            r.data_ptr(), u.data_ptr(), w.data_ptr(), b.data_ptr(),
            r_out.data_ptr() if store_residual else None, out.data_ptr(),
            _dtype_code(norm_dtype), rows, n_cols, float(eps), int(apply_affine),
            _stream(r.device),
        ),
        "tfx_residual_layer_norm",
    )
    return r_out, out


def _linear(x, weight, bias, residual, epilogue, out_dtype, what):
    _require_cuda(x, what)
    if weight.ndim != 2 or bias.ndim != 1:
        raise ValueError("weight must be 2-D and bias must be 1-D")
    n, k = weight.shape
    if x.shape[-1] != k or bias.numel() != n:
        raise ValueError("weight does not match the input")
    lead = x.shape[:-1]
    a = x.reshape(-1, k).to(torch.float16).contiguous()
    w = weight.detach().to(torch.float16).contiguous()
    b = bias.detach().float().contiguous()
    m = a.shape[0]
    res_ptr = None
    if residual is not None:
        if residual.shape[:-1] != lead or residual.shape[-1] != n:
            raise ValueError("residual does not match the output shape")
        residual = residual.float().contiguous()
        res_ptr = residual.data_ptr()
    out = torch.empty((m, n), device=x.device, dtype=out_dtype)
    _lib.check(
        _lib.load().tfx_linear(
            a.data_ptr(), w.data_ptr(), b.data_ptr(), res_ptr, out.data_ptr(), m, n, k,
            epilogue, _stream(x.device),
        ),
        what,
    )
    return out.view(*lead, n)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """fp16 tensor-core ``F.linear(x, weight, bias)`` (fp32 accumulate, fp16 out).

    ``weight`` is nn.Linear's [out, in]. Replaces the cached-fp16 ``F.linear``
    of torch_transformer_benchmark.py:675-685 / :741.
    """
    return _linear(x, weight, bias, None, _lib.TFX_EPI_BIAS, torch.float16, "tfx_linear")


def linear_gelu(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """``gelu_erf(x @ weight.T + bias)`` in one tensor-core kernel, fp16 out.

    Replaces ``triton_ffn_gelu`` (triton_fused_ffn.py:224-261), which takes the
    weight transposed ([K, N]) and applies the tanh GELU; this takes
    nn.Linear's [N, K] weight and applies the exact erf GELU the baseline
    uses (torch_transformer_benchmark.py:286).
    """
    return _linear(x, weight, bias, None, _lib.TFX_EPI_BIAS_GELU, torch.float16,
                   "tfx_linear(gelu)")


def linear_residual(
    x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, residual: torch.Tensor
) -> torch.Tensor:
    """``residual + x @ weight.T + bias`` with the add done in fp32 (fp32 out)."""
    return _linear(x, weight, bias, residual, _lib.TFX_EPI_BIAS_RESIDUAL, torch.float32,
                   "tfx_linear(residual)")


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    is_causal: bool = True,
    scale: Optional[float] = None,
    valid_lengths: Optional[torch.Tensor] = None,
    key_mask: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Flash attention on [B, S, H, hd] views (e.g. slices of the packed QKV).

    Key padding: ``valid_lengths`` (int [B], keys >= length masked) or
    ``key_mask`` (bool [B, S], False = masked key, any pattern), not both.

    q, k, v: fp16 tensors indexed (b, s, h, e) whose last two dims are
    contiguous and which share the same row stride (the packed projection's
    [B, S, 3, H, hd] layout qualifies). Returns ctx [B, S, H*hd] fp16.
    Replaces F.scaled_dot_product_attention in
    torch_transformer_benchmark.py:767-808 (which takes [B, H, S, hd] views of
    the same memory).
    """
    _require_cuda(q, "tfx_attention")
    if q.dtype != torch.float16 or k.dtype != torch.float16 or v.dtype != torch.float16:
        raise ValueError("q, k and v must be float16")
    if q.ndim != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must be [B, S, H, hd] with identical shapes")
    bsz, seq, heads, hd = q.shape
    for t in (q, k, v):
        if t.stride(3) != 1 or t.stride(2) != hd or t.stride(1) != q.stride(1) or \
                t.stride(0) != seq * q.stride(1):
            raise ValueError("q, k, v must share a [B, S, *] row layout with contiguous heads")
    if scale is None:
        scale = hd ** -0.5
    out = torch.empty((bsz, seq, heads * hd), device=q.device, dtype=torch.float16)
    if key_mask is not None:
        if valid_lengths is not None:
            raise ValueError("pass valid_lengths or key_mask, not both")
        if key_mask.shape != (bsz, seq) or key_mask.dtype != torch.bool:
            raise ValueError("key_mask must be a [B, S] bool tensor")
        from .model import key_bitmask

        words = key_bitmask(key_mask.to(q.device))
        _lib.check(
            _lib.load().tfx_attention_masked(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(1), out.data_ptr(),
                heads * hd, bsz, heads, seq, hd, float(scale), int(is_causal), words.data_ptr(),
                _stream(q.device),
            ),
            "tfx_attention_masked",
        )
        return out
    vl_ptr = None
    if valid_lengths is not None:
        valid_lengths = valid_lengths.to(device=q.device, dtype=torch.int32).contiguous()
        if valid_lengths.numel() != bsz:
            raise ValueError("valid_lengths must have one entry per batch element")
        vl_ptr = valid_lengths.data_ptr()
    _lib.check(
        _lib.load().tfx_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(1), out.data_ptr(), heads * hd,
            bsz, heads, seq, hd, float(scale), int(is_causal), vl_ptr, _stream(q.device),
        ),
        "tfx_attention",
    )
    return out


def _packed_rows(t: torch.Tensor, what: str, tokens: int, heads: int, hd: int, index: int) -> int:
    """Checks a packed [T, heads, head_dim] fp16 tensor; its row stride in elements."""
    if t.dtype != torch.float16 or t.shape != (tokens, heads, hd):
        raise ValueError(f"{what} must be float16 [{tokens}, {heads}, {hd}]")
    if t.get_device() != index:
        raise ValueError(f"{what} must be on the cache's device")
    st = t.stride()
    if st[2] != 1 or (heads > 1 and st[1] != hd):
        raise ValueError(f"{what} must have contiguous heads (any row stride)")
    return st[0] if tokens > 1 else heads * hd


def _paged_device(cache: PagedKVCache, batch: PagedBatch) -> int:
    """Index of the device that both live on."""
    index = cache._index
    if index is None:
        raise ValueError("the paged cache requires CUDA tensors")
    if batch._index != index:
        raise ValueError("batch and cache must be on one device")
    return index


def _call_on(index: int, what: str, fn, *args) -> None:
    """fn(*args, stream) on device ``index`` and its current stream. (The raw
    handle: a decode step's calls are short, and a Stream object costs 2 us.)"""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream)
    if status:
        _lib.check(status, what)


def paged_append(k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, batch: PagedBatch) -> None:
    """Write the batch's new keys and values into their pages.

    k, v: fp16 [num_tokens, kv_heads, head_dim] with contiguous heads (slices of
    the packed projection qualify). 8-bit caches quantise here, one scale per
    token and head (max|x| / 127 or / 448): codes are those of exact
    arithmetic, ties to even; a row of zeros gets scale 0, a row with an
    infinity or NaN gets scale NaN and reads back as NaN. Tokens whose page is
    outside the pool are dropped. Two tokens of a batch must not share a slot (it
    would hold parts of both; other slots are not affected); a cache whose k and v
    are one tensor is refused, and k and v must not lie in it. The paged form of the
    reference's ``_append_kv_cache`` (torch_transformer_benchmark.py:426-462).
    """
    index = _paged_device(cache, batch)
    n, heads, hd = batch.num_tokens, cache.kv_heads, cache.head_dim
    ld_k = _packed_rows(k, "k", n, heads, hd, index)
    ld_v = _packed_rows(v, "v", n, heads, hd, index)
    if n:
        _call_on(index, "tfx_paged_append", _lib.load().tfx_paged_append, k.data_ptr(), ld_k,
                 v.data_ptr(), ld_v, cache._ref, batch._ref)


def paged_read(
    cache: PagedKVCache,
    batch: PagedBatch,
    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of the batch's tokens, fp16 [num_tokens, kv_heads, head_dim].

    The same tokens that ``paged_append`` writes: the last ones of each
    sequence, all of it where query_start counts kv_len tokens. 8-bit caches
    give code * scale in fp32, rounded to fp16. Tokens without a page read as zeros; rows
    that belong to no sequence are not written. ``out``: write into these two.
    """
    index = _paged_device(cache, batch)
    n, heads, hd = batch.num_tokens, cache.kv_heads, cache.head_dim
    if out is None:
        k, v = cache._half.new_empty(n, heads, hd), cache._half.new_empty(n, heads, hd)
        ld_k = ld_v = heads * hd
    else:
        k, v = out
        ld_k = _packed_rows(k, "out[0]", n, heads, hd, index)
        ld_v = _packed_rows(v, "out[1]", n, heads, hd, index)
    if n:
        _call_on(index, "tfx_paged_read", _lib.load().tfx_paged_read, cache._ref, batch._ref,
                 k.data_ptr(), ld_k, v.data_ptr(), ld_v)
    return k, v


def paged_attention(
    q: torch.Tensor,
    cache: PagedKVCache,
    batch: PagedBatch,
    is_causal: bool = True,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of the batch's new tokens over their sequences' cached ones.

    q: fp16 [num_tokens, q_heads, head_dim] with contiguous heads; q_heads a
    multiple of the cache's kv_heads (query head h reads key/value head
    h // (q_heads // kv_heads)). The new tokens' own keys and values are in the
    cache already (``paged_append``). ``is_causal``: a token sees the positions up
    to its own; otherwise all of its sequence. ``scale`` (default
    head_dim ** -0.5) is positive. Returns ctx [num_tokens, q_heads * head_dim]
    fp16 (``out`` if given); a row that sees no key, or only keys whose scores
    are -inf, is zero, rows that belong to no sequence are not written. Single tokens, drafts of a few and chunks of a
    prompt may share a batch. The paged form of the cached attention of
    torch_transformer_benchmark.py:747-765.
    """
    index = _paged_device(cache, batch)
    n, hd = batch.num_tokens, cache.head_dim
    if q.ndim != 3:
        raise ValueError("q must be [num_tokens, q_heads, head_dim]")
    heads = q.shape[1]
    ld_q = _packed_rows(q, "q", n, heads, hd, index)
    if heads == 0 or heads % cache.kv_heads or heads >= 2 ** 31:
        raise ValueError(f"q_heads ({heads}) must be a multiple of kv_heads ({cache.kv_heads}), "
                         "below 2^31")
    ld_out = heads * hd
    if out is None:
        out = q.new_empty(n, ld_out)
    elif out.shape != (n, ld_out) or out.dtype != torch.float16 or out.get_device() != index or \
            (n > 0 and out.stride(1) != 1):
        raise ValueError("out must be float16 [num_tokens, q_heads * head_dim] with contiguous rows")
    elif n > 1:
        ld_out = out.stride(0)
    if n == 0:
        return out
    lib = _lib.load()
    need = batch._workspace_bytes(lib, cache, heads)
    ws = None
    if need > 0:
        # A workspace of its own for each call, from the stream's allocator: calls
        # on different streams, and graphs captured apart, never share one.
        ws = cache._half.new_empty(need // 2)
    _call_on(index, "tfx_paged_attention", lib.tfx_paged_attention, q.data_ptr(), ld_q, cache._ref,
             batch._ref, out.data_ptr(), ld_out, heads, cache._scale if scale is None else float(scale),
             int(is_causal), None if ws is None else ws.data_ptr(), max(need, 0))
    return out


def math_scale(head_dim: int) -> float:
    """Softmax scale head_dim**-0.5 (torch_transformer_benchmark.py:215)."""
    return 1.0 / math.sqrt(head_dim)
