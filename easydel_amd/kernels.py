"""Tensor-level entry points: thin, checked wrappers over the C ABI.

PyTorch appears here only as the owner of device memory and streams (``data_ptr()`` and the
current HIP stream); all arithmetic happens in librpa_hip.so.  Every function raises if the
library is missing, if a tensor is not on a GPU, or if the C ABI reports an error.
"""

from __future__ import annotations

import math

import torch

from . import _lib

_DTYPE_TAG = {
    torch.float32: _lib.RPA_F32,
    torch.bfloat16: _lib.RPA_BF16,
    torch.float8_e4m3fn: _lib.RPA_FP8_E4M3,
    torch.int8: _lib.RPA_INT8,
    torch.float16: _lib.RPA_F16,
}

_workspaces: dict[tuple, torch.Tensor] = {}


def dtype_tag(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_TAG[dtype]
    except KeyError:
        raise NotImplementedError(f"dtype {dtype} is not supported by the ROCm ragged-page kernels") from None


def _dev(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor holding device memory, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}; the ROCm ragged-page kernels need GPU memory (no CPU fallback)")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _i32(t: torch.Tensor, name: str) -> int:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    return _dev(t, name)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def page_geometry(kv_pages: torch.Tensor, head_dim: int) -> tuple[int, int, int, int]:
    """(P, page_size, C, Dp) of a v2 ``[P, pg, 2*Hkv, D]`` or v3 ``[P, pg, groups, packing, Dp]`` page buffer.

    Both have token rows of ``C`` combined heads of ``Dp`` stored elements, K at even and V at odd
    combined heads.  The v3 shape for ``head_dim == 64`` packs K_h|V_h into one 128-wide row, which
    is the same bytes as rows of 64 (``Dp = 64``); any other head size is stored padded to a multiple
    of 128 (easydel/caching/ragged_page/cache.py:640-647), ``Dp > head_dim`` with zeros in the padding.
    """
    if kv_pages.ndim not in (4, 5):
        raise ValueError(f"kv_pages must be 4-D (v2) or 5-D (v3), got shape {tuple(kv_pages.shape)}")
    stored = kv_pages.shape[-1]
    if stored < head_dim:
        raise ValueError(f"kv_pages rows hold {stored} elements, fewer than head_dim {head_dim}")
    if head_dim == 64 and stored == 128 and kv_pages.ndim == 5:
        stored = 64  # K_h | V_h share one 128-wide row
    per_token = math.prod(kv_pages.shape[2:])
    return kv_pages.shape[0], kv_pages.shape[1], per_token // stored, stored


def workspace_bytes(T, S, M, page_size, Hq, Hkv, D, q_dtype: torch.dtype, kv_dtype: torch.dtype) -> int:
    return int(_lib.load().rpa_attention_workspace_bytes(T, S, M, page_size, Hq, Hkv, D, dtype_tag(q_dtype), dtype_tag(kv_dtype)))


def _workspace(device, nbytes: int) -> torch.Tensor:
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def page_scatter_slices(new_kv, slice_indices, num_slices, kv_cache_pages, *, page_size: int, page_shard_index: int = 0):
    """In-place v2 scatter: ``kv_cache_pages [N, C, D]`` (flat positions) <- ``new_kv [T, C, D]`` by slices."""
    lib = _lib.load()
    if new_kv.dtype != kv_cache_pages.dtype:
        raise TypeError(f"new_kv dtype {new_kv.dtype} != cache dtype {kv_cache_pages.dtype}")
    if slice_indices.ndim != 2 or slice_indices.shape[0] != 3:
        raise ValueError(f"slice_indices must be [3, N], got {tuple(slice_indices.shape)}")
    if tuple(new_kv.shape[1:]) != tuple(kv_cache_pages.shape[1:]):
        raise ValueError(f"token row shapes differ: {tuple(new_kv.shape[1:])} vs {tuple(kv_cache_pages.shape[1:])}")
    T, N, n_pos = new_kv.shape[0], slice_indices.shape[1], kv_cache_pages.shape[0]
    if T == 0 or N == 0 or n_pos == 0:
        return kv_cache_pages
    row_bytes = math.prod(new_kv.shape[1:]) * new_kv.element_size()
    _dev(kv_cache_pages, "kv_cache_pages")
    with torch.cuda.device(kv_cache_pages.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_page_scatter_slices(
            _stream(kv_cache_pages), _dev(new_kv, "new_kv"), _i32(slice_indices, "slice_indices"),
            _i32(num_slices, "num_slices"), _dev(kv_cache_pages, "kv_cache_pages"), T, N, n_pos, int(page_size), row_bytes,
            int(page_shard_index)))
    return kv_cache_pages


def page_scatter_ragged(key, value, kv_pages, context_lens, block_tables, query_start_loc, num_seqs):
    """In-place v3 write: tokens of sequence i land at positions ``[ctx_i - q_len_i, ctx_i)`` of its pages."""
    lib = _lib.load()
    if key.dtype != kv_pages.dtype or value.dtype != kv_pages.dtype:
        raise TypeError(f"key/value dtype {key.dtype}/{value.dtype} must equal the cache dtype {kv_pages.dtype}")
    T, Hkv, D = key.shape
    P, pg, C, Dp = page_geometry(kv_pages, D)
    S = context_lens.shape[0]
    M = block_tables.numel() // S
    if T == 0:
        return kv_pages
    _dev(kv_pages, "kv_pages")
    with torch.cuda.device(kv_pages.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_page_scatter_ragged(
            _stream(kv_pages), _dev(key, "key"), _dev(value, "value"), _dev(kv_pages, "kv_pages"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(num_seqs, "num_seqs"), T, S, M, P, pg, Hkv, D, Dp, C, key.element_size()))
    return kv_pages


def page_scatter_ragged_quantised(key, value, kv_pages, kv_scales, context_lens, block_tables, query_start_loc, num_seqs):
    """In-place quantising v3 write into scaled fp8 / int8 pages: per (page, combined head) the scale only grows
    (``max(old, amax / qmax)``), tokens already in the page are re-coded when it does."""
    lib = _lib.load()
    if key.dtype != value.dtype or key.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"key/value must both be float32 or bfloat16, got {key.dtype}/{value.dtype}")
    if kv_pages.dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError(f"kv_pages must be float8_e4m3fn or int8 for the quantising write, got {kv_pages.dtype}")
    T, Hkv, D = key.shape
    P, pg, C, Dp = page_geometry(kv_pages, D)
    if kv_scales.dtype != torch.float32 or kv_scales.numel() != P * C:
        raise ValueError(f"kv_scales must be float32 [P={P}, C={C}]")
    S = context_lens.shape[0]
    M = block_tables.numel() // S
    if T == 0:
        return kv_pages, kv_scales
    _dev(kv_pages, "kv_pages")
    with torch.cuda.device(kv_pages.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_page_scatter_ragged_quantised(
            _stream(kv_pages), _dev(key, "key"), _dev(value, "value"), _dev(kv_pages, "kv_pages"), _dev(kv_scales, "kv_scales"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(num_seqs, "num_seqs"), T, S, M, P, pg, Hkv, D, Dp, C, dtype_tag(key.dtype), dtype_tag(kv_pages.dtype)))
    return kv_pages, kv_scales


def _sinks(softmax_aux, num_q_heads: int, device):
    """Attention-sink logits as the library takes them: float32 ``[Hq]`` on the query's device (the reference
    casts them to float32 and shards them by head, easydel/operations/kernels/ragged_page_attention.py:469-471).
    Returns ``(tensor kept alive by the caller, pointer)``; ``(None, None)`` without sinks."""
    if softmax_aux is None:
        return None, None
    if softmax_aux.ndim != 1 or softmax_aux.shape[0] != num_q_heads:
        raise NotImplementedError(f"softmax_aux must hold one sink logit per query head, shape [{num_q_heads}]; "
                                  f"got {tuple(softmax_aux.shape)}")
    if softmax_aux.device != device:
        raise ValueError(f"softmax_aux is on {softmax_aux.device}, the query on {device}")
    aux = softmax_aux.detach().to(torch.float32).contiguous()
    return aux, _dev(aux, "softmax_aux")


def _attn_common(query, kv_pages, context_lens, block_tables, num_kv_heads, softmax_scale, sliding_window, logits_soft_cap):
    T, Hq, D = query.shape
    P, pg, C, Dp = page_geometry(kv_pages, D)
    S = context_lens.shape[0]
    if block_tables.numel() % S:
        raise ValueError("block_tables size is not a multiple of the number of sequence rows")
    M = block_tables.numel() // S
    Hkv = int(num_kv_heads) if num_kv_heads is not None else C // 2
    scale = float(D) ** -0.5 if softmax_scale is None else float(softmax_scale)
    window = int(sliding_window) if sliding_window else 0
    cap = float(logits_soft_cap) if logits_soft_cap else 0.0
    return T, Hq, D, Dp, P, pg, C, S, M, Hkv, scale, window, cap


def ragged_paged_attention(query, kv_pages, context_lens, block_tables, query_start_loc, num_seqs, *,
                           softmax_scale=None, sliding_window=None, logits_soft_cap=None, kv_scales=None,
                           num_kv_heads=None, softmax_aux=None, out=None):
    """Read-only ragged paged attention; returns ``[T, Hq, D]`` in the query dtype."""
    lib = _lib.load()
    T, Hq, D, Dp, P, pg, C, S, M, Hkv, scale, window, cap = _attn_common(
        query, kv_pages, context_lens, block_tables, num_kv_heads, softmax_scale, sliding_window, logits_soft_cap)
    if out is None:
        out = torch.empty_like(query)
    if T == 0:
        return out
    qd, kd = dtype_tag(query.dtype), dtype_tag(kv_pages.dtype)
    for name, t in (("query", query), ("kv_pages", kv_pages), ("out", out)):
        _dev(t, name)
    aux, aux_ptr = _sinks(softmax_aux, Hq, query.device)
    ws = _workspace(query.device, int(lib.rpa_attention_workspace_bytes(T, S, M, pg, Hq, Hkv, Dp, qd, kd)))
    scales_ptr = None
    if kv_scales is not None:
        if kv_scales.dtype != torch.float32 or kv_scales.numel() != P * C:
            raise ValueError(f"kv_scales must be float32 [P={P}, C={C}]")
        scales_ptr = _dev(kv_scales, "kv_scales")
    with torch.cuda.device(query.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_ragged_paged_attention(
            _stream(query), _dev(query, "query"), _dev(kv_pages, "kv_pages"), scales_ptr,
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(num_seqs, "num_seqs"), _dev(out, "out"), ws.data_ptr(), ws.numel(),
            T, S, M, P, pg, Hq, Hkv, D, Dp, C, qd, kd, scale, window, cap, aux_ptr))
    return out


def unified_attention(query, key_cache, value_cache, context_lens, block_tables, query_start_loc, num_seqs=None, *,
                      softmax_scale=None, sliding_window=None, logits_soft_cap=None, kv_scales=None, softmax_aux=None,
                      out=None):
    """Ragged paged attention over separate K and V pools ``[P, page_size, Hkv, D]`` (the reference's
    unified-attention layout).  ``num_seqs`` is optional: without it every row of ``context_lens`` is live."""
    lib = _lib.load()
    if key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise ValueError(f"key_cache {tuple(key_cache.shape)} {key_cache.dtype} and value_cache "
                         f"{tuple(value_cache.shape)} {value_cache.dtype} must match")
    if key_cache.ndim != 4:
        raise ValueError(f"key_cache must be [P, page_size, Hkv, D], got {tuple(key_cache.shape)}")
    T, Hq, D = query.shape
    P, pg, Hkv, Dk = key_cache.shape
    if Dk != D:
        raise NotImplementedError(f"cache head_dim {Dk} != query head_dim {D}")
    S = context_lens.shape[0]
    if block_tables.numel() % S:
        raise ValueError("block_tables size is not a multiple of the number of sequence rows")
    M = block_tables.numel() // S
    scale = float(D) ** -0.5 if softmax_scale is None else float(softmax_scale)
    window = int(sliding_window) if sliding_window else 0
    cap = float(logits_soft_cap) if logits_soft_cap else 0.0
    if out is None:
        out = torch.empty_like(query)
    if T == 0:
        return out
    qd, kd = dtype_tag(query.dtype), dtype_tag(key_cache.dtype)
    for name, t in (("query", query), ("key_cache", key_cache), ("value_cache", value_cache), ("out", out)):
        _dev(t, name)
    aux, aux_ptr = _sinks(softmax_aux, Hq, query.device)
    ws = _workspace(query.device, int(lib.rpa_attention_workspace_bytes(T, S, M, pg, Hq, Hkv, D, qd, kd)))
    scales_ptr = None
    if kv_scales is not None:
        if kv_scales.dtype != torch.float32 or kv_scales.numel() != P * 2 * Hkv:
            raise ValueError(f"kv_scales must be float32 [P={P}, 2*Hkv={2 * Hkv}]")
        scales_ptr = _dev(kv_scales, "kv_scales")
    with torch.cuda.device(query.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_unified_attention(
            _stream(query), _dev(query, "query"), _dev(key_cache, "key_cache"), _dev(value_cache, "value_cache"), scales_ptr,
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            None if num_seqs is None else _i32(num_seqs, "num_seqs"), _dev(out, "out"), ws.data_ptr(), ws.numel(),
            T, S, M, P, pg, Hq, Hkv, D, qd, kd, scale, window, cap, aux_ptr))
    return out


def ragged_paged_attention_v3(query, key, value, kv_pages, context_lens, block_tables, query_start_loc, distribution, *,
                              softmax_scale=None, sliding_window=None, logits_soft_cap=None, num_kv_heads=None,
                              softmax_aux=None, out=None):
    """Fused scatter + attention; updates ``kv_pages`` in place and returns ``(out, kv_pages)``."""
    lib = _lib.load()
    if key.dtype != kv_pages.dtype or value.dtype != kv_pages.dtype:
        raise TypeError(f"key/value dtype {key.dtype}/{value.dtype} must equal the cache dtype {kv_pages.dtype}")
    T, Hq, D, Dp, P, pg, C, S, M, Hkv, scale, window, cap = _attn_common(
        query, kv_pages, context_lens, block_tables, key.shape[1] if num_kv_heads is None else num_kv_heads,
        softmax_scale, sliding_window, logits_soft_cap)
    if out is None:
        out = torch.empty_like(query)
    if T == 0:
        return out, kv_pages
    qd, kd = dtype_tag(query.dtype), dtype_tag(kv_pages.dtype)
    for name, t in (("query", query), ("key", key), ("value", value), ("kv_pages", kv_pages), ("out", out)):
        _dev(t, name)
    aux, aux_ptr = _sinks(softmax_aux, Hq, query.device)
    ws = _workspace(query.device, int(lib.rpa_attention_workspace_bytes(T, S, M, pg, Hq, Hkv, Dp, qd, kd)))
    with torch.cuda.device(query.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_ragged_paged_attention_v3(
            _stream(query), _dev(query, "query"), _dev(key, "key"), _dev(value, "value"), _dev(kv_pages, "kv_pages"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(distribution, "distribution"), _dev(out, "out"), ws.data_ptr(), ws.numel(),
            T, S, M, P, pg, Hq, Hkv, D, Dp, C, qd, kd, scale, window, cap, aux_ptr))
    return out, kv_pages


def ragged_paged_attention_v3_static(query, key, value, kv_pages, context_lens, block_tables, query_start_loc, distribution, *,
                                     softmax_scale=None, sliding_window=None, logits_soft_cap=None, num_kv_heads=None,
                                     softmax_aux=None, out):
    """``ragged_paged_attention_v3`` through the entry point that allocates nothing: the caller passes ``out``, the
    scratch memory is the library's built-in per-GPU array (64 MiB; larger needs raise ``RpaError``).  Calls that
    overlap on one GPU share that array and race."""
    lib = _lib.load()
    if key.dtype != kv_pages.dtype or value.dtype != kv_pages.dtype:
        raise TypeError(f"key/value dtype {key.dtype}/{value.dtype} must equal the cache dtype {kv_pages.dtype}")
    T, Hq, D, Dp, P, pg, C, S, M, Hkv, scale, window, cap = _attn_common(
        query, kv_pages, context_lens, block_tables, key.shape[1] if num_kv_heads is None else num_kv_heads,
        softmax_scale, sliding_window, logits_soft_cap)
    if T == 0:
        return out, kv_pages
    qd, kd = dtype_tag(query.dtype), dtype_tag(kv_pages.dtype)
    aux_ptr = None
    if softmax_aux is not None:  # no conversion here: that would allocate
        if softmax_aux.dtype != torch.float32 or tuple(softmax_aux.shape) != (Hq,):
            raise ValueError(f"softmax_aux must be float32 [{Hq}] for the call that allocates nothing")
        aux_ptr = _dev(softmax_aux, "softmax_aux")
    with torch.cuda.device(query.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_ragged_paged_attention_v3_static(
            _stream(query), _dev(query, "query"), _dev(key, "key"), _dev(value, "value"), _dev(kv_pages, "kv_pages"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(distribution, "distribution"), _dev(out, "out"), T, S, M, P, pg, Hq, Hkv, D, Dp, C, qd, kd, scale, window, cap,
            aux_ptr))
    return out, kv_pages


def ragged_paged_attention_v3_quantised(query, key, value, kv_pages, kv_scales, context_lens, block_tables,
                                        query_start_loc, distribution, *, softmax_scale=None, sliding_window=None,
                                        logits_soft_cap=None, num_kv_heads=None, softmax_aux=None, out=None):
    """Fused quantising write + attention over scaled 8-bit pages; updates ``kv_pages`` and ``kv_scales`` in place
    and returns ``(out, kv_pages, kv_scales)``.  ``key`` / ``value`` are float32 or bfloat16."""
    lib = _lib.load()
    if key.dtype != value.dtype or key.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"key/value must both be float32 or bfloat16, got {key.dtype}/{value.dtype}")
    T, Hq, D, Dp, P, pg, C, S, M, Hkv, scale, window, cap = _attn_common(
        query, kv_pages, context_lens, block_tables, key.shape[1] if num_kv_heads is None else num_kv_heads,
        softmax_scale, sliding_window, logits_soft_cap)
    if kv_scales.dtype != torch.float32 or kv_scales.numel() != P * C:
        raise ValueError(f"kv_scales must be float32 [P={P}, C={C}]")
    if out is None:
        out = torch.empty_like(query)
    if T == 0:
        return out, kv_pages, kv_scales
    qd, kd = dtype_tag(query.dtype), dtype_tag(kv_pages.dtype)
    for name, t in (("query", query), ("key", key), ("value", value), ("kv_pages", kv_pages), ("kv_scales", kv_scales), ("out", out)):
        _dev(t, name)
    aux, aux_ptr = _sinks(softmax_aux, Hq, query.device)
    ws = _workspace(query.device, int(lib.rpa_attention_workspace_bytes(T, S, M, pg, Hq, Hkv, Dp, qd, kd)))
    with torch.cuda.device(query.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_ragged_paged_attention_v3_quantised(
            _stream(query), _dev(query, "query"), _dev(key, "key"), _dev(value, "value"), _dev(kv_pages, "kv_pages"),
            _dev(kv_scales, "kv_scales"), _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"),
            _i32(query_start_loc, "query_start_loc"), _i32(distribution, "distribution"), _dev(out, "out"), ws.data_ptr(),
            ws.numel(), T, S, M, P, pg, Hq, Hkv, D, Dp, C, qd, dtype_tag(key.dtype), kd, scale, window, cap, aux_ptr))
    return out, kv_pages, kv_scales


def mla_row_geometry(kv_pages: torch.Tensor) -> tuple[int, int, int]:
    """(P, page_size, row_elems) of a latent page pool: ``[P, pg, row]`` or the reference's
    ``[P, pg / packing, packing, row]`` (easydel/caching/mla_ragged_page/cache.py:270-287), the same bytes."""
    if kv_pages.ndim == 3:
        return kv_pages.shape[0], kv_pages.shape[1], kv_pages.shape[2]
    if kv_pages.ndim == 4:
        return kv_pages.shape[0], kv_pages.shape[1] * kv_pages.shape[2], kv_pages.shape[3]
    raise ValueError(f"latent kv_pages must be 3-D or 4-D, got shape {tuple(kv_pages.shape)}")


def _mla_shapes(queries_nope, queries_pe, kv_pages, context_lens, block_tables):
    if queries_nope.ndim != 3 or queries_pe.ndim != 3 or queries_nope.shape[:2] != queries_pe.shape[:2]:
        raise ValueError("`queries_nope` and `queries_pe` must share [total_tokens, num_q_heads]. "
                         f"Got {tuple(queries_nope.shape)} vs {tuple(queries_pe.shape)}.")
    T, Hq, lkv = queries_nope.shape
    rope = queries_pe.shape[2]
    P, pg, row = mla_row_geometry(kv_pages)
    S = context_lens.shape[0]
    if block_tables.numel() % S:
        raise ValueError("block_tables size is not a multiple of the number of sequence rows")
    return T, Hq, lkv, rope, P, pg, row, S, block_tables.numel() // S


def mla_page_scatter(keys_values, keys_pe, kv_pages, context_lens, block_tables, query_start_loc, num_seqs):
    """In-place write of latent rows and rope keys: tokens of sequence i land at positions
    ``[ctx_i - q_len_i, ctx_i)`` of its pages (latent at 0, rope key at the padded latent width, padding zeroed)."""
    lib = _lib.load()
    if keys_values.dtype != kv_pages.dtype or keys_pe.dtype != kv_pages.dtype:
        raise TypeError(f"keys_values/keys_pe dtype {keys_values.dtype}/{keys_pe.dtype} must equal the cache dtype {kv_pages.dtype}")
    if keys_values.ndim != 2 or keys_pe.ndim != 2 or keys_values.shape[0] != keys_pe.shape[0]:
        raise ValueError(f"keys_values [T, kv_lora_rank] and keys_pe [T, rope] expected, got {tuple(keys_values.shape)}, {tuple(keys_pe.shape)}")
    T, lkv = keys_values.shape
    rope = keys_pe.shape[1]
    P, pg, row = mla_row_geometry(kv_pages)
    S = context_lens.shape[0]
    M = block_tables.numel() // S
    if T == 0:
        return kv_pages
    _dev(kv_pages, "kv_pages")
    with torch.cuda.device(kv_pages.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_mla_page_scatter(
            _stream(kv_pages), _dev(keys_values, "keys_values"), _dev(keys_pe, "keys_pe"), _dev(kv_pages, "kv_pages"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(num_seqs, "num_seqs"), T, S, M, P, pg, lkv, rope, row, keys_values.element_size()))
    return kv_pages


def mla_ragged_paged_attention(queries_nope, queries_pe, keys_values, keys_pe, kv_pages, context_lens, block_tables,
                               query_start_loc, distribution, *, softmax_scale=None, sliding_window=None,
                               logits_soft_cap=None, softmax_aux=None, out=None):
    """Multi-latent attention over latent pages, fused with the write of the new rows (``keys_values`` may be None:
    the pages are then read as they are).  Returns ``(out [T, Hq, kv_lora_rank], kv_pages)``."""
    lib = _lib.load()
    T, Hq, lkv, rope, P, pg, row, S, M = _mla_shapes(queries_nope, queries_pe, kv_pages, context_lens, block_tables)
    if queries_pe.dtype != queries_nope.dtype:
        raise TypeError(f"queries_pe dtype {queries_pe.dtype} != queries_nope dtype {queries_nope.dtype}")
    if keys_values is not None:
        if keys_pe is None:
            raise ValueError("multi_latent_ragged_page_attention requires `keys_pe`. Pass it as `keys_pe=` (or `k_pe=`).")
        if keys_values.dtype != kv_pages.dtype or keys_pe.dtype != kv_pages.dtype:
            raise TypeError(f"keys_values/keys_pe dtype {keys_values.dtype}/{keys_pe.dtype} must equal the cache dtype {kv_pages.dtype}")
        if tuple(keys_values.shape) != (T, lkv) or tuple(keys_pe.shape) != (T, rope):
            raise ValueError(f"keys_values {tuple(keys_values.shape)} / keys_pe {tuple(keys_pe.shape)} must be [{T}, {lkv}] / [{T}, {rope}]")
    if out is None:
        out = torch.empty_like(queries_nope)
    if T == 0:
        return out, kv_pages
    qd, kd = dtype_tag(queries_nope.dtype), dtype_tag(kv_pages.dtype)
    for name, t in (("queries_nope", queries_nope), ("queries_pe", queries_pe), ("kv_pages", kv_pages), ("out", out)):
        _dev(t, name)
    scale = float(lkv + rope) ** -0.5 if softmax_scale is None else float(softmax_scale)
    window = int(sliding_window) if sliding_window else 0
    cap = float(logits_soft_cap) if logits_soft_cap else 0.0
    aux, aux_ptr = _sinks(softmax_aux, Hq, queries_nope.device)
    ws = _workspace(queries_nope.device, int(lib.rpa_mla_workspace_bytes(T, S, M, pg, Hq, lkv, qd, kd)))
    with torch.cuda.device(queries_nope.device):  # the library queries and launches on HIP's current device
        _lib.check(lib.rpa_mla_ragged_paged_attention(
            _stream(queries_nope), _dev(queries_nope, "queries_nope"), _dev(queries_pe, "queries_pe"),
            None if keys_values is None else _dev(keys_values, "keys_values"),
            None if keys_values is None else _dev(keys_pe, "keys_pe"), _dev(kv_pages, "kv_pages"),
            _i32(context_lens, "context_lens"), _i32(block_tables, "block_tables"), _i32(query_start_loc, "query_start_loc"),
            _i32(distribution, "distribution"), _dev(out, "out"), ws.data_ptr(), ws.numel(),
            T, S, M, P, pg, Hq, lkv, rope, row, qd, kd, scale, window, cap, aux_ptr))
    return out, kv_pages


def _rows(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, device) -> tuple[int, int]:
    """(pointer, elements between token rows) of a ``[T, heads, dim]`` or ``[T, dim]`` operand whose token rows are
    contiguous and may lie apart, as views of one projection's output do."""
    # what a good call looks like first, in few steps: a decode step's launch waits for them
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device.index and t.shape == shape:
        if t.is_contiguous():
            return t.data_ptr(), shape[1] * shape[2] if len(shape) == 3 else shape[1]
        st = t.stride()
        if len(st) == 3 and st[2] == 1 and st[1] == shape[2] and shape[0] > 1:
            return t.data_ptr(), st[0]
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor holding device memory, got {type(t).__name__}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}; the ROCm ragged-page kernels need GPU memory (no CPU fallback)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the query on {device}")
    row, want = math.prod(shape[1:]), 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != want:
            raise ValueError(f"{name}: the elements of a token row must be contiguous, got strides {t.stride()}")
        want *= size
    return t.data_ptr(), row if t.shape[0] <= 1 else t.stride(0)


def _launch(device, fn, *args) -> None:
    """``fn(stream, *args)`` on ``device``, its current stream, with HIP's current device set to it (the library queries and
    launches on that)."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:  # a tensor of the device exists: the runtime is initialised
        code = fn(stream, *args)
    else:
        with torch.cuda.device(device):
            code = fn(stream, *args)
    if code != 0:
        _lib.check(code)


def _on(t: torch.Tensor, name: str, dtype: torch.dtype, device) -> int:
    if t.dtype is dtype and t.is_contiguous() and t.get_device() == device.index:  # a good call, in few steps
        return t.data_ptr()
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    ptr = _dev(t, name)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the query on {device}")
    return ptr


def _span(t: torch.Tensor) -> tuple[int, int]:
    if t.is_contiguous():
        start = t.data_ptr()
        return start, start + t.nbytes
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _turned_out(query, query_out, others, name: str):
    """The tensor the turned queries go to: a new one, the queries themselves, or one that overlaps no operand (``others``: all of them but
    the queries; None: not given)."""
    if query_out is None:
        return torch.empty_like(query) if query.is_contiguous() else query.new_empty(query.shape)
    if query_out.shape != query.shape or query_out.dtype != query.dtype or query_out.device != query.device:
        raise ValueError(f"{name} must be {list(query.shape)} {query.dtype} on {query.device}, got {list(query_out.shape)} "
                         f"{query_out.dtype} on {query_out.device}")
    if not query_out.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    a, b = _span(query_out)
    in_place = query_out.data_ptr() == query.data_ptr() and query.is_contiguous()
    for t in others if in_place else (query, *others):
        if t is None:
            continue
        c, d = _span(t)
        if a < d and c < b:
            raise ValueError(f"{name} overlaps another operand (only the contiguous queries themselves may be given)")
    return query_out


def _table(cos_sin, rope_dim: int | None, dim: int, device) -> tuple[int, int, int]:
    """(pointer, rotated elements, rows) of a float32 ``[rows, rope_dim]`` table: cosines, then sines."""
    if cos_sin.ndim != 2:
        raise ValueError(f"cos_sin must be [positions, rope_dim], got {list(cos_sin.shape)}")
    rows, width = cos_sin.shape
    if rows == 0 or width == 0 or width % 2 or width > dim:
        raise ValueError(f"cos_sin [positions, rope_dim] must hold a row and an even rope_dim of at most {dim}, got {list(cos_sin.shape)}")
    if rope_dim is not None and width != rope_dim:
        raise ValueError(f"cos_sin has rows of {width}, the rope part is {rope_dim} wide")
    return _on(cos_sin, "cos_sin", torch.float32, device), width, rows


def _ragged(context_lens, block_tables, query_start_loc, num_seqs, positions, T: int, device):
    """(S, M, pointers of context_lens, block_tables, query_start_loc, num_seqs, positions), checked against each other."""
    S = context_lens.shape[0]
    if S == 0 or block_tables.numel() == 0 or block_tables.numel() % S:
        raise ValueError("block_tables size is not a multiple of the number of sequence rows")
    if query_start_loc.numel() != S + 1:
        raise ValueError(f"query_start_loc must hold {S + 1} entries, got {query_start_loc.numel()}")
    if num_seqs is not None and num_seqs.numel() < 1:
        raise ValueError("num_seqs is empty")
    if positions is not None and tuple(positions.shape) != (T,):
        raise ValueError(f"positions must be [{T}], got {list(positions.shape)}")
    i32 = torch.int32
    return (S, block_tables.numel() // S, _on(context_lens, "context_lens", i32, device), _on(block_tables, "block_tables", i32, device),
            _on(query_start_loc, "query_start_loc", i32, device), None if num_seqs is None else _on(num_seqs, "num_seqs", i32, device),
            None if positions is None else _on(positions, "positions", i32, device))


def _rope_operands(query, key, value):
    if query.ndim != 3 or key.ndim != 3 or value.shape != key.shape:
        raise ValueError(f"query [T, Hq, D] and key, value [T, Hkv, D] expected, got {list(query.shape)}, {list(key.shape)}, {list(value.shape)}")
    T, Hq, D = query.shape
    Hkv = key.shape[1]
    dev, dt = query.device, query.dtype
    if dt not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"query must be float32, bfloat16 or float16, got {dt}")
    return (T, Hq, Hkv, D, _rows(query, "query", (T, Hq, D), dt, dev), _rows(key, "key", (T, Hkv, D), dt, dev),
            _rows(value, "value", (T, Hkv, D), dt, dev))


def rope_page_scatter_ragged(query, key, value, kv_pages, cos_sin, context_lens, block_tables, query_start_loc, num_seqs, *,
                             kv_scales=None, positions=None, is_neox_style: bool = True, query_out=None):
    """Rotary position embedding and page write in one launch: ``query [T, Hq, D]`` and ``key [T, Hkv, D]`` turn by the
    angles of their positions, the keys and ``value`` go to the pages as :func:`page_scatter_ragged` places them (scaled
    8-bit pages: coded from the turned float32 keys as :func:`page_scatter_ragged_quantised` codes them, with the scale
    ``amax * (1 / qmax)`` in the place of ``amax / qmax``).

    ``cos_sin [rows, rope_dim]`` float32 holds the cosines, then the sines, of a position's angles; a token's row is its
    cache position, or ``positions [T]``, clamped into the table.  The first ``rope_dim`` elements of a head turn, in
    pairs ``(d, d + rope_dim / 2)`` (``is_neox_style``) or ``(2 d, 2 d + 1)``.  The token rows of query, key and value may lie
    apart (views of one projection).  Returns ``(turned query, kv_pages)``, with scales ``(..., kv_scales)``; rows of
    padded tokens of the turned query are zeros (``query_out=query`` turns it in place and leaves them)."""
    lib = _lib.load()
    T, Hq, Hkv, D, (q, qs), (k, ks), (v, vs) = _rope_operands(query, key, value)
    P, pg, C, Dp = page_geometry(kv_pages, D)
    kd = dtype_tag(kv_pages.dtype)
    if kv_scales is not None and (kv_scales.dtype != torch.float32 or kv_scales.numel() != P * C):
        raise ValueError(f"kv_scales must be float32 [P={P}, C={C}]")
    dev = query.device
    table, rope, rows = _table(cos_sin, None, D, dev)
    S, M, ctx, bt, qsl, ns, pos = _ragged(context_lens, block_tables, query_start_loc, num_seqs, positions, T, dev)
    out = _turned_out(query, query_out, (key, value, kv_pages, kv_scales, cos_sin, positions, context_lens, block_tables, query_start_loc, num_seqs), "query_out")
    pages = _on(kv_pages, "kv_pages", kv_pages.dtype, dev)
    scales = None if kv_scales is None else _on(kv_scales, "kv_scales", torch.float32, dev)
    if T > 0:
        _launch(dev, lib.rpa_rope_page_scatter_ragged, q, k, v, out.data_ptr(), pages, scales, table, pos, ctx, bt, qsl, ns, T, S, M, P, pg, Hq, Hkv, D, Dp, C,
                rope, rows, 1 if is_neox_style else 0, qs, ks, vs, _DTYPE_TAG[query.dtype], kd)
    return (out, kv_pages) if kv_scales is None else (out, kv_pages, kv_scales)


def rope_unified_page_scatter(query, key, value, key_cache, value_cache, cos_sin, context_lens, block_tables, query_start_loc,
                              num_seqs=None, *, positions=None, is_neox_style: bool = True, query_out=None):
    """:func:`rope_page_scatter_ragged` into separate K and V pools ``[P, page_size, Hkv, D]`` (without scales).  Without
    ``num_seqs`` every row of ``context_lens`` is live.  Returns ``(turned query, key_cache, value_cache)``."""
    lib = _lib.load()
    T, Hq, Hkv, D, (q, qs), (k, ks), (v, vs) = _rope_operands(query, key, value)
    if key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise ValueError(f"key_cache {tuple(key_cache.shape)} {key_cache.dtype} and value_cache "
                         f"{tuple(value_cache.shape)} {value_cache.dtype} must match")
    if key_cache.ndim != 4 or tuple(key_cache.shape[2:]) != (Hkv, D):
        raise ValueError(f"key_cache must be [P, page_size, {Hkv}, {D}], got {tuple(key_cache.shape)}")
    P, pg = key_cache.shape[:2]
    kd, dev = dtype_tag(key_cache.dtype), query.device
    table, rope, rows = _table(cos_sin, None, D, dev)
    S, M, ctx, bt, qsl, ns, pos = _ragged(context_lens, block_tables, query_start_loc, num_seqs, positions, T, dev)
    out = _turned_out(query, query_out, (key, value, key_cache, value_cache, cos_sin, positions, context_lens, block_tables, query_start_loc, num_seqs), "query_out")
    kc, vc = _on(key_cache, "key_cache", key_cache.dtype, dev), _on(value_cache, "value_cache", key_cache.dtype, dev)
    if T > 0:
        _launch(dev, lib.rpa_rope_unified_page_scatter, q, k, v, out.data_ptr(), kc, vc, table, pos, ctx, bt, qsl, ns, T, S, M, P, pg, Hq, Hkv, D, rope, rows,
                1 if is_neox_style else 0, qs, ks, vs, _DTYPE_TAG[query.dtype], kd)
    return out, key_cache, value_cache


def rope_mla_page_scatter(queries_pe, keys_values, keys_pe, kv_pages, cos_sin, context_lens, block_tables, query_start_loc, num_seqs, *,
                          positions=None, is_neox_style: bool = True, query_out=None):
    """The rotation of multi-latent attention and its page write in one launch: ``queries_pe [T, Hq, rope]`` turn,
    ``keys_pe [T, rope]`` turn into the latent rows, ``keys_values [T, kv_lora_rank]`` (already in the pages' element type) are
    copied beside them as :func:`mla_page_scatter` places them.  Table, positions, styles and padded rows as for
    :func:`rope_page_scatter_ragged`, over the whole rope part.  Returns ``(turned queries_pe, kv_pages)``."""
    lib = _lib.load()
    if queries_pe.ndim != 3 or keys_pe.ndim != 2 or keys_values.ndim != 2:
        raise ValueError(f"queries_pe [T, Hq, rope], keys_pe [T, rope] and keys_values [T, kv_lora_rank] expected, got "
                         f"{list(queries_pe.shape)}, {list(keys_pe.shape)}, {list(keys_values.shape)}")
    T, Hq, rope = queries_pe.shape
    dev, dt = queries_pe.device, queries_pe.dtype
    if dt not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"queries_pe must be float32, bfloat16 or float16, got {dt}")
    q, qs = _rows(queries_pe, "queries_pe", (T, Hq, rope), dt, dev)
    k, ks = _rows(keys_pe, "keys_pe", (T, rope), dt, dev)
    if keys_values.shape[0] != T:
        raise ValueError(f"keys_values must hold {T} rows, got {keys_values.shape[0]}")
    lkv = keys_values.shape[1]
    P, pg, row = mla_row_geometry(kv_pages)
    kd = dtype_tag(kv_pages.dtype)
    latent = _on(keys_values, "keys_values", kv_pages.dtype, dev)
    table, _, rows = _table(cos_sin, rope, rope, dev)
    S, M, ctx, bt, qsl, ns, pos = _ragged(context_lens, block_tables, query_start_loc, num_seqs, positions, T, dev)
    out = _turned_out(queries_pe, query_out, (keys_pe, keys_values, kv_pages, cos_sin, positions, context_lens, block_tables, query_start_loc, num_seqs),
                      "query_out")
    pages = _on(kv_pages, "kv_pages", kv_pages.dtype, dev)
    if T > 0:
        _launch(dev, lib.rpa_rope_mla_page_scatter, q, latent, k, out.data_ptr(), pages, table, pos, ctx, bt, qsl, ns, T, S, M, P, pg, Hq, lkv, rope, row, rows,
                1 if is_neox_style else 0, qs, ks, _DTYPE_TAG[dt], kd)
    return out, kv_pages


_DECAY_WHOLE = 256  # kDecayWhole of rpa_decay.h: calls of up to this many tokens need no scratch


def decay_linear_attention(query, key, value, log_decay, state, state_indices, query_start_loc, num_seqs, *, context_lens=None,
                           state_out_indices=None, scale: float | None = None, out=None):
    """Linear attention with one decay per KV head over a ragged batch; the states live in the slots of a pool.

    For the tokens of a sequence in order, ``S <- exp(log_decay[h]) S + k v^T`` and ``out = scale * q S``, with ``query
    [T, Hq, Dk]``, ``key [T, Hkv, Dk]``, ``value [T, Hkv, Dv]`` of one dtype (float32, bfloat16, float16; token rows may lie
    apart) and ``state [slots, Hkv, Dk, Dv]`` float32, one state to ``Hq / Hkv`` query heads.  Sequence ``i`` goes on from slot
    ``state_indices[i]``, or from zero where ``context_lens[i]`` says that it has no tokens before these, and leaves its
    state in ``state_out_indices[i]`` (default: the same slot); slots written must differ from each other and from those that other
    sequences of the call read.  ``scale`` defaults to ``Dk ** -0.5``.  States and sums are float32; in sequences of more than 16
    tokens bfloat16 rows aligned to 16 bytes round the scores inside a chunk, and the state where it meets a query, to bfloat16 on
    their way to the outputs.  Returns ``(out [T, Hq, Dv], state)``: the pool updated in place, rows of padded tokens zeros."""
    lib = _lib.load()
    if query.ndim != 3 or key.ndim != 3 or value.ndim != 3:
        raise ValueError(f"query [T, Hq, Dk], key [T, Hkv, Dk] and value [T, Hkv, Dv] expected, got {list(query.shape)}, "
                         f"{list(key.shape)}, {list(value.shape)}")
    T, Hq, Dk = query.shape
    Hkv, Dv = key.shape[1], value.shape[2]
    dev, dt = query.device, query.dtype
    if dt not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"query must be float32, bfloat16 or float16, got {dt}")
    q, qs = _rows(query, "query", (T, Hq, Dk), dt, dev)
    k, ks = _rows(key, "key", (T, Hkv, Dk), dt, dev)
    v, vs = _rows(value, "value", (T, Hkv, Dv), dt, dev)
    if state.ndim != 4 or tuple(state.shape[1:]) != (Hkv, Dk, Dv):
        raise ValueError(f"state must be [slots, {Hkv}, {Dk}, {Dv}], got {list(state.shape)}")
    if tuple(log_decay.shape) != (Hkv,):
        raise ValueError(f"log_decay must be [{Hkv}], got {list(log_decay.shape)}")
    S = state_indices.shape[0]
    for name, t, n in (("query_start_loc", query_start_loc, S + 1), ("context_lens", context_lens, S), ("state_out_indices", state_out_indices, S)):
        if t is not None and t.shape != (n,):
            raise ValueError(f"{name} must be [{n}], got {list(t.shape)}")
    if S == 0 or num_seqs.numel() < 1:
        raise ValueError("no sequence rows")
    i32 = torch.int32
    ptrs = (_on(log_decay, "log_decay", torch.float32, dev), _on(state, "state", torch.float32, dev),
            _on(state_indices, "state_indices", i32, dev),
            None if state_out_indices is None else _on(state_out_indices, "state_out_indices", i32, dev),
            None if context_lens is None else _on(context_lens, "context_lens", i32, dev),
            _on(query_start_loc, "query_start_loc", i32, dev), _on(num_seqs, "num_seqs", i32, dev))
    if out is None:
        out = query.new_empty((T, Hq, Dv))
    elif tuple(out.shape) != (T, Hq, Dv):
        raise ValueError(f"out must be [{T}, {Hq}, {Dv}], got {list(out.shape)}")
    else:
        a, b = _span(out)
        for name, t in (("query", query), ("key", key), ("value", value), ("state", state), ("log_decay", log_decay), ("state_indices", state_indices),
                        ("state_out_indices", state_out_indices), ("context_lens", context_lens), ("query_start_loc", query_start_loc),
                        ("num_seqs", num_seqs)):
            if t is None:
                continue
            c, d = _span(t)
            if a < d and c < b:
                raise ValueError(f"out overlaps {name}")
    o = _on(out, "out", dt, dev)
    if T > 0:
        tag = _DTYPE_TAG[dt]
        # scratch of its own for every call: the caching allocator orders its reuse by stream, and a captured graph keeps its own
        need = 0
        if T > _DECAY_WHOLE:
            with torch.cuda.device(dev):  # the size goes by the current device's compute units
                need = lib.rpa_decay_attention_workspace_bytes(T, S, Hq, Hkv, Dk, Dv, tag)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _launch(dev, lib.rpa_decay_linear_attention, q, k, v, *ptrs, o, None if ws is None else ws.data_ptr(), need, T, S, state.shape[0],
                Hq, Hkv, Dk, Dv, qs, ks, vs, tag, float(Dk) ** -0.5 if scale is None else float(scale))
    return out, state
