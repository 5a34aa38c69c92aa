"""The reference's attention-math kernel API, served by the HIP library.

Same names, arguments and errors as model/kernels.py of the reference:
``paired_qk_norm_rope_paged_cache_`` (:94-160), ``paired_qk_norm_rope_``
(:275-332), ``paired_qk_norm_rope_dense_cache_`` (:335-405) and
``decode_attn_nhd_short_cache`` (:466-520).  All inputs must live on the GPU;
there is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib


def _require_bf16(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.bfloat16:
            raise TypeError("HIP attention kernels take bf16 tensors")


def paired_qk_norm_rope_paged_cache_(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    query_weight: torch.Tensor,
    key_weight: torch.Tensor,
    position_ids: torch.Tensor,
    epsilon: float,
    rope_theta: float,
    layer_cache: torch.Tensor,
    write_pages: torch.Tensor,
    write_offsets: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalize/rotate QK in place and stage K/V into the paged cache once."""

    if query.ndim != 3 or key.ndim != 3 or value.ndim != 3:
        raise ValueError("Qwen3-TTS QKV tensors must have rank three")
    tokens, query_heads, head_dim = query.shape
    if key.shape != value.shape or key.shape[0] != tokens or key.shape[2] != head_dim:
        raise ValueError("Qwen3-TTS QKV shapes are incompatible")
    key_heads = key.shape[1]
    _lib.require_device(query, key, value, layer_cache, position_ids, write_pages, write_offsets)
    if not (query.dtype == key.dtype == value.dtype == layer_cache.dtype):
        raise TypeError("paired QKV paged staging requires one dtype")
    _require_bf16(query, query_weight, key_weight)
    if head_dim % 2 or query_weight.shape != (head_dim,) or key_weight.shape != (head_dim,):
        raise ValueError("QK norm weights must match an even head dimension")
    if position_ids.shape != (tokens,) or write_pages.shape != (tokens,) or write_offsets.shape != (tokens,):
        raise ValueError("paged QKV metadata must contain one entry per token")
    if layer_cache.ndim != 5 or layer_cache.shape[1] != 2 or layer_cache.shape[3:] != (key_heads, head_dim):
        raise ValueError("paged QKV cache has an invalid layout")
    if not all(t.stride(-1) == 1 for t in (query, key, value, layer_cache)):
        raise ValueError("QKV and paged cache must be contiguous per head")
    for t in (position_ids, write_pages, write_offsets):
        if t.dtype != torch.long:
            raise TypeError("paged QKV metadata must be int64")
    _lib.call(
        "nq_qk_norm_rope_kv_write",
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1),
        value.data_ptr(), value.stride(0), value.stride(1),
        query_weight.data_ptr(), key_weight.data_ptr(),
        position_ids.data_ptr(), position_ids.stride(0), tokens, query_heads, key_heads, head_dim,
        float(epsilon), float(rope_theta), 1,
        layer_cache.data_ptr(), layer_cache.stride(0), layer_cache.stride(1), layer_cache.stride(2),
        layer_cache.stride(3), write_pages.data_ptr(), write_offsets.data_ptr(), 0,
        _lib.stream(query.device),
    )
    return query, key


def _validate_qk(query, key, query_weight, key_weight, positions):
    if query.ndim != 3 or key.ndim != 3:
        raise ValueError("QK tensors must have shape [tokens, heads, head_dim]")
    tokens, query_heads, head_dim = query.shape
    if key.shape[0] != tokens or key.shape[2] != head_dim or head_dim % 2:
        raise ValueError("QK shapes are incompatible")
    _lib.require_device(query, key, positions)
    if key.device != query.device or query.dtype != key.dtype:
        raise ValueError("paired QK transform requires one dtype/device")
    _require_bf16(query, query_weight, key_weight)
    if query.stride(-1) != 1 or key.stride(-1) != 1:
        raise ValueError("QK tensors must be contiguous per head")
    if positions.shape != (tokens,) or positions.device != query.device:
        raise ValueError("positions must contain one device value per token")
    if positions.dtype != torch.long:
        raise TypeError("positions must be int64")
    if query_weight.shape != (head_dim,) or key_weight.shape != (head_dim,):
        raise ValueError("QK norm weights must match head_dim")
    return tokens, query_heads, key.shape[1], head_dim


def paired_qk_norm_rope_(query, key, query_weight, key_weight, positions, epsilon, rope_theta):
    """Apply the paired QK transform with its bf16 rounding boundary (no cache write)."""

    tokens, hq, hk, d = _validate_qk(query, key, query_weight, key_weight, positions)
    _lib.call(
        "nq_qk_norm_rope_kv_write",
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1),
        None, 0, 0, query_weight.data_ptr(), key_weight.data_ptr(),
        positions.data_ptr(), positions.stride(0), tokens, hq, hk, d, float(epsilon), float(rope_theta), 1,
        None, 0, 0, 0, 0, None, None, 0, _lib.stream(query.device),
    )
    return query, key


def paired_qk_norm_rope_dense_cache_(
    query, key, value, query_weight, key_weight, positions, epsilon, rope_theta, key_cache, value_cache,
    cache_position: int,
):
    """Transform one-token QK and stage K/V into the fixed code-predictor cache."""

    tokens, hq, hk, d = _validate_qk(query, key, query_weight, key_weight, positions)
    expected = (tokens, key_cache.shape[1], hk, d)
    if value.shape != (tokens, hk, d) or key_cache.shape != expected or value_cache.shape != expected:
        raise ValueError("dense CP QKV cache shape mismatch")
    if not 0 <= cache_position < key_cache.shape[1]:
        raise ValueError("dense CP cache position is invalid")
    if not (value.device == key_cache.device == value_cache.device == query.device):
        raise ValueError("dense CP QKV cache requires one device")
    if not (value.dtype == key_cache.dtype == value_cache.dtype == query.dtype):
        raise TypeError("dense CP QKV cache requires one dtype")
    if key_cache.stride() != value_cache.stride() or key_cache.stride(-1) != 1 or value.stride(-1) != 1:
        raise ValueError("dense CP K and V caches must share one layout")
    delta = value_cache.data_ptr() - key_cache.data_ptr()
    if delta % key_cache.element_size():
        raise ValueError("dense CP K and V caches are misaligned")
    c_kind = delta // key_cache.element_size()
    _lib.call(
        "nq_qk_norm_rope_kv_write",
        query.data_ptr(), query.stride(0), query.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1),
        value.data_ptr(), value.stride(0), value.stride(1),
        query_weight.data_ptr(), key_weight.data_ptr(),
        positions.data_ptr(), positions.stride(0), tokens, hq, hk, d, float(epsilon), float(rope_theta), 0,
        key_cache.data_ptr(), key_cache.stride(0), c_kind, key_cache.stride(1), key_cache.stride(2),
        None, None, int(cache_position), _lib.stream(query.device),
    )
    return query, key


def qkv_partials_norm_rope_dense_cache_(
    partials, splits: int, q_out, query_weight, key_weight, positions, epsilon, rope_theta, key_cache, value_cache,
    cache_position: int,
):
    """paired_qk_norm_rope_dense_cache_ fed by the packed QKV projection's fp32 split-K planes
    [splits, tokens, (Hq + 2 Hkv) * D] (``layers.linear_partials`` leaves them at the start of its
    workspace): each value is the plane-order sum rounded to bf16, the bf16 projection output, so
    the rotated q (into ``q_out`` [tokens, Hq, D]) and the cache rows are those of the projection
    followed by paired_qk_norm_rope_dense_cache_, without the projection's reduction launch."""

    _require_bf16(q_out, query_weight, key_weight, key_cache, value_cache)
    tokens, hq, d = q_out.shape
    hk = key_cache.shape[2]
    if key_cache.shape != (tokens, key_cache.shape[1], hk, d) or value_cache.shape != key_cache.shape:
        raise ValueError("dense CP cache shape mismatch")
    if not 0 <= cache_position < key_cache.shape[1]:
        raise ValueError("dense CP cache position is invalid")
    if key_cache.stride() != value_cache.stride() or key_cache.stride(-1) != 1 or q_out.stride(-1) != 1:
        raise ValueError("dense CP K and V caches must share one layout")
    if positions.dtype != torch.long or positions.shape[0] != tokens:
        raise ValueError("positions must be int64 with one entry per token")
    if partials.numel() * partials.element_size() < splits * tokens * (hq + 2 * hk) * d * 4:
        raise ValueError("partials hold fewer planes than splits")
    delta = value_cache.data_ptr() - key_cache.data_ptr()
    if delta % key_cache.element_size():
        raise ValueError("dense CP K and V caches are misaligned")
    _lib.require_device(partials, q_out, query_weight, key_weight, positions, key_cache, value_cache)
    _lib.call(
        "nq_qkv_partials_norm_rope_kv_write", partials.data_ptr(), int(splits), tokens,
        q_out.data_ptr(), q_out.stride(0), q_out.stride(1), None, 0, 0,
        query_weight.data_ptr(), key_weight.data_ptr(), positions.data_ptr(), positions.stride(0), hq, hk, d,
        float(epsilon), float(rope_theta), 0,
        key_cache.data_ptr(), key_cache.stride(0), delta // key_cache.element_size(), key_cache.stride(1),
        key_cache.stride(2), None, None, int(cache_position), _lib.stream(q_out.device),
    )
    return q_out


def qkv_partials_rope_short_attention_(
    partials, splits: int, q_out, query_weight, key_weight, positions, epsilon, rope_theta, key_cache, value_cache,
    cache_position: int, out,
):
    """qkv_partials_norm_rope_dense_cache_ followed by decode_attn_nhd_short_cache(q_out, key_cache,
    value_cache, cache_position + 1, out=out), the pair the code predictor's decode layer runs
    (model/components.py:294-345), in one launch with the same bits: q_out receives the rotated q,
    the caches position ``cache_position``'s K and V, ``out`` [tokens, Hq, D] the attention."""

    _require_bf16(q_out, query_weight, key_weight, key_cache, value_cache, out)
    tokens, hq, d = q_out.shape
    if key_cache.ndim != 4:
        raise ValueError("dense CP cache shape mismatch")
    hk = key_cache.shape[2]
    if key_cache.shape != (tokens, key_cache.shape[1], hk, d) or value_cache.shape != key_cache.shape:
        raise ValueError("dense CP cache shape mismatch")
    if not isinstance(cache_position, int) or isinstance(cache_position, bool) or not 0 <= cache_position < min(
            key_cache.shape[1], 16):
        raise ValueError("dense CP cache position is invalid (short-cache attention covers at most 16)")
    if key_cache.stride() != value_cache.stride() or key_cache.stride(-1) != 1 or q_out.stride(-1) != 1:
        raise ValueError("dense CP K and V caches must share one layout")
    if out.shape != q_out.shape or out.stride(-1) != 1:
        raise ValueError("out must be [tokens, Hq, D] like q_out")
    if hq % hk:
        raise ValueError("short-cache attention requires compatible heads")
    if positions.dtype != torch.long or positions.shape[0] != tokens:
        raise ValueError("positions must be int64 with one entry per token")
    if partials.numel() * partials.element_size() < splits * tokens * (hq + 2 * hk) * d * 4:
        raise ValueError("partials hold fewer planes than splits")
    delta = value_cache.data_ptr() - key_cache.data_ptr()
    if delta % key_cache.element_size():
        raise ValueError("dense CP K and V caches are misaligned")
    _lib.require_device(partials, q_out, query_weight, key_weight, positions, key_cache, value_cache, out)
    _lib.call(
        "nq_cp_rope_short_attention", partials.data_ptr(), int(splits), tokens,
        query_weight.data_ptr(), key_weight.data_ptr(), positions.data_ptr(), positions.stride(0),
        float(epsilon), float(rope_theta), 0, q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
        key_cache.data_ptr(), key_cache.stride(0), delta // key_cache.element_size(), key_cache.stride(1),
        key_cache.stride(2), int(cache_position), hq, hk, d, float(d) ** -0.5,
        out.data_ptr(), out.stride(0), out.stride(1), _lib.stream(q_out.device),
    )
    return out


def rope_short_linear_splits(tokens: int, qo_heads: int, kv_heads: int, head_dim: int, out_features: int) -> int:
    """The planes ``qkv_partials_rope_short_linear_`` leaves for a shape; -1 where it does not take it."""

    return int(_lib.load().nq_cp_rope_short_linear_splits(tokens, qo_heads, kv_heads, head_dim, out_features))


def qkv_partials_rope_short_linear_(
    partials, splits: int, query_weight, key_weight, positions, epsilon, rope_theta, key_cache, value_cache,
    cache_position: int, weight, planes,
) -> int:
    """qkv_partials_rope_short_attention_ and the projection of its output by ``weight`` [out, Hq * D] in one
    launch, for at most 8 tokens: the caches receive position ``cache_position``'s K and V, ``planes`` the
    projection as fp32 split-K planes (their number is returned)."""

    _require_bf16(query_weight, key_weight, key_cache, value_cache, weight)
    tokens, limit, hk, d = key_cache.shape
    if value_cache.shape != key_cache.shape or value_cache.stride() != key_cache.stride() or key_cache.stride(-1) != 1:
        raise ValueError("dense CP K and V caches must share one layout")
    out_features, hq = weight.shape[0], weight.shape[1] // d
    if weight.ndim != 2 or hq * d != weight.shape[1] or weight.stride(1) != 1 or query_weight.shape != (d,) \
            or key_weight.shape != (d,):
        raise ValueError("the weight must be [out, Hq * D] and the norm weights [D]")
    if not isinstance(cache_position, int) or isinstance(cache_position, bool) or not 0 <= cache_position < min(limit, 16):
        raise ValueError("dense CP cache position is invalid (short-cache attention covers at most 16)")
    if positions.dtype != torch.long or positions.shape[0] != tokens:
        raise ValueError("positions must be int64 with one entry per token")
    if partials.numel() * partials.element_size() < splits * tokens * (hq + 2 * hk) * d * 4:
        raise ValueError("partials hold fewer planes than splits")
    delta = value_cache.data_ptr() - key_cache.data_ptr()
    if delta % key_cache.element_size():
        raise ValueError("dense CP K and V caches are misaligned")
    _lib.require_device(partials, query_weight, key_weight, positions, key_cache, value_cache, weight, planes)
    _lib.call(
        "nq_cp_rope_short_linear", partials.data_ptr(), int(splits), tokens, query_weight.data_ptr(),
        key_weight.data_ptr(), positions.data_ptr(), positions.stride(0), float(epsilon), float(rope_theta), 0,
        key_cache.data_ptr(), key_cache.stride(0), delta // key_cache.element_size(), key_cache.stride(1),
        key_cache.stride(2), int(cache_position), hq, hk, d, float(d) ** -0.5, weight.data_ptr(), weight.stride(0),
        out_features, planes.data_ptr(), planes.numel() * planes.element_size(), _lib.stream(key_cache.device),
    )
    return rope_short_linear_splits(tokens, hq, hk, d, out_features)


def decode_attn_nhd_short_cache(query, key_cache, value_cache, cache_length: int, out=None):
    """Fixed 16-position code-predictor attention (one query per row)."""

    if not isinstance(cache_length, int) or isinstance(cache_length, bool) or not 1 <= cache_length <= 16:
        raise ValueError("short-cache attention requires cache_length in [1, 16]")
    squeeze = query.ndim == 4
    if squeeze:
        if query.shape[1] != 1:
            raise ValueError("short-cache attention supports one query token")
        query = query.squeeze(1)
    if query.ndim != 3 or key_cache.ndim != 4 or key_cache.shape != value_cache.shape:
        raise ValueError("short-cache QKV ranks are invalid")
    rows, hq, d = query.shape
    cache_rows, capacity, hk, cd = key_cache.shape
    if (cache_rows, cd) != (rows, d) or cache_length > capacity:
        raise ValueError("short-cache QKV shapes are incompatible")
    if hq % hk:
        raise ValueError("short-cache attention requires compatible heads")
    _lib.require_device(query, key_cache, value_cache)
    _require_bf16(query, key_cache, value_cache)
    if key_cache.stride() != value_cache.stride():
        raise ValueError("short-cache K and V caches must share one layout")
    delta = value_cache.data_ptr() - key_cache.data_ptr()
    if delta % 2:
        raise ValueError("short-cache K and V caches are misaligned")
    output = torch.empty_like(query) if out is None else out
    _lib.call(
        "nq_cp_short_attention",
        query.data_ptr(), query.stride(0), query.stride(1),
        key_cache.data_ptr(), key_cache.stride(0), delta // 2, key_cache.stride(1), key_cache.stride(2),
        rows, cache_length, hq, hk, d, float(d) ** -0.5,
        output.data_ptr(), output.stride(0), output.stride(1), _lib.stream(query.device),
    )
    return output.unsqueeze(1) if squeeze else output


def paged_attention_noalloc(query: torch.Tensor, layer_cache: torch.Tensor, metadata, *, max_pages: int,
                            sm_scale: float | None = None, parts: int = _lib.NQ_ATTN_DECODE | _lib.NQ_ATTN_PREFILL,
                            status: torch.Tensor | None = None, out: torch.Tensor) -> torch.Tensor:
    """Paged attention of ``query`` [tokens, Hq, D] over one layer ``[pages, 2, ps, Hkv, D]`` of the
    cache with ``metadata`` (a TalkerAttentionMetadata), planned and run with the library's static
    scratch (``nq_paged_attention_noalloc``): no device allocation, no workspace argument.  ``out``
    is required for the same reason.  Calls that overlap on one GPU share the scratch and race."""

    _require_bf16(query, layer_cache, out)
    if query.ndim != 3 or layer_cache.ndim != 5 or layer_cache.shape[1] != 2:
        raise ValueError("query must be [tokens, Hq, D] and the cache [pages, 2, page_size, Hkv, D]")
    tokens, hq, d = query.shape
    pages, _, page_size, hkv, d_cache = layer_cache.shape
    if d_cache != d or out.shape != query.shape or out.stride(-1) != 1 or query.stride(-1) != 1:
        raise ValueError("query, cache and out disagree on the head layout")
    rows = metadata.paged_kv_indptr.numel() - 1
    need = int(_lib.load().nq_attention_workspace_bytes(tokens, int(max_pages), page_size, hq, hkv, d))
    _lib.check(min(need, 0), "nq_attention_workspace_bytes")
    if need > _lib.NQ_NOALLOC_SCRATCH_BYTES:
        raise ValueError(f"this batch needs {need} bytes of attention scratch; the no-allocation entry point "
                         f"holds {_lib.NQ_NOALLOC_SCRATCH_BYTES} per GPU (use the workspace path)")
    for t in (metadata.paged_kv_indptr, metadata.paged_kv_last_page_len, metadata.paged_kv_indices):
        if t.dtype != torch.int32:
            raise TypeError("paged metadata must be int32")
    _lib.require_device(query, layer_cache, out, metadata.paged_kv_indptr, status)
    scale = float(d) ** -0.5 if sm_scale is None else float(sm_scale)
    _lib.call(
        "nq_paged_attention_noalloc",
        _lib.ptr(metadata.qo_indptr), metadata.paged_kv_indptr.data_ptr(),
        metadata.paged_kv_last_page_len.data_ptr(), metadata.paged_kv_indices.data_ptr(), rows,
        query.data_ptr(), query.stride(0), query.stride(1), layer_cache.data_ptr(), layer_cache.stride(0),
        layer_cache.stride(1), layer_cache.stride(2), layer_cache.stride(3), pages, page_size, hq, hkv, d, scale,
        out.data_ptr(), out.stride(0), out.stride(1), tokens, int(max_pages), int(parts), _lib.ptr(status),
        _lib.stream(query.device),
    )
    return out


INT8_BLOCK = 16  # cache slots that share a scale
_INT8_SLOTS = 0x7FFF0000  # slots that a call's page list may name
_INT8_SM_SCALE = 2.3e38  # times log2(e) still a float32


def _int8_cache(layer_cache: torch.Tensor, layer_scales: torch.Tensor) -> tuple:
    """Heads, head size and the C ABI's cache arguments after checks: codes and strides, scales and strides, pages,
    page size."""

    if layer_cache.dtype is not torch.int8 or layer_scales.dtype is not torch.float32:
        raise TypeError("the 8-bit cache is int8 codes with float32 scales")
    shape, strides = layer_cache.shape, layer_cache.stride()
    if len(shape) != 5 or shape[1] != 2 or shape[0] < 1 or strides[4] != 1:
        raise ValueError("the 8-bit cache must be [pages, 2, page_size, Hkv, D], contiguous per head")
    pages, _, page_size, heads, d = shape
    if page_size < INT8_BLOCK or page_size & (page_size - 1):
        raise TypeError(f"the 8-bit cache needs a page size that is a power of two of at least {INT8_BLOCK}")
    if layer_scales.shape != (pages, 2, page_size // INT8_BLOCK, heads):
        raise ValueError("the scales must be [pages, 2, page_size // 16, Hkv]")
    return heads, d, (layer_cache.data_ptr(), *strides[:4], layer_scales.data_ptr(), *layer_scales.stride(), pages,
                      page_size)


def _int8_slots(pages: torch.Tensor, offsets: torch.Tensor) -> int:
    if pages.dtype is not torch.long or offsets.dtype is not torch.long:
        raise TypeError("cache slots must be int64")
    shape = pages.shape
    if len(shape) != 1 or offsets.shape != shape or not pages.is_contiguous() or not offsets.is_contiguous():
        raise ValueError("cache slots must be contiguous vectors with one entry per token")
    return shape[0]


def _int8_heads(t: torch.Tensor, shape: tuple) -> tuple:
    """Pointer, token and head stride of key or value."""

    if t.dtype is not torch.bfloat16:
        raise TypeError("HIP attention kernels take bf16 tensors")
    strides = t.stride()
    if t.shape != shape or strides[2] != 1:
        raise ValueError("key and value must be [tokens, Hkv, D] with the cache's heads, contiguous per head")
    return t.data_ptr(), strides[0], strides[1]


def _int8_status(status: torch.Tensor | None) -> int | None:
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.numel() < 1:
        raise TypeError("status must be an int32 tensor")
    return status.data_ptr()


def paged_cache_write_int8_(key: torch.Tensor, value: torch.Tensor, layer_cache: torch.Tensor,
                            layer_scales: torch.Tensor, write_pages: torch.Tensor, write_offsets: torch.Tensor,
                            status: torch.Tensor | None = None) -> None:
    """Quantize ``key`` and ``value`` [tokens, Hkv, D] (bf16, rotated) into one layer of the 8-bit cache:
    codes int8 [pages, 2, page_size, Hkv, D], scales float32 [pages, 2, page_size // 16, Hkv], a value
    being code * scale.

    Tokens go to the slots (``write_pages[t]``, ``write_offsets[t]``).  A block of 16 slots has one scale per
    kind and head, the least power of two s (at least 2^-126) with max |x| / s <= 127 over the tokens in it; when
    a later token makes it grow, the codes of the block's earlier slots are rescaled (rounded to the nearest,
    ties to even), which adds less than one step to any value.  A write at a block's first slot starts the block anew; a write further
    on takes the slots before it as held and those behind the written ones as empty.  Tokens that
    share a block stand next to each other in slot order (as a request's do); two separate runs into one block in
    one call leave that block unspecified.  A NaN or infinity makes its block's scale NaN.  A slot may be
    written again where its token was discarded, but scales do not shrink: the block's other tokens keep the coarser
    step that a discarded outlier brought, and a discarded NaN leaves the block NaN, until the block is written from
    its first slot again.  A slot outside the pool is skipped and
    ``status`` (int32, optional) set to NQ_ERR_INVALID_ARGUMENT.  No counterpart in the reference."""

    heads, d, cache = _int8_cache(layer_cache, layer_scales)
    tokens = _int8_slots(write_pages, write_offsets)
    shape = (tokens, heads, d)
    source = _int8_heads(key, shape) + _int8_heads(value, shape)
    _lib.launch(
        _lib.one_device(key, value, layer_cache, layer_scales, write_pages, write_offsets, status), "nq_kv_int8_write",
        *source, tokens, heads, d, *cache, write_pages.data_ptr(), write_offsets.data_ptr(), _int8_status(status),
    )


def paged_cache_read_int8(layer_cache: torch.Tensor, layer_scales: torch.Tensor, pages: torch.Tensor,
                          offsets: torch.Tensor, key: torch.Tensor | None = None, value: torch.Tensor | None = None,
                          status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V [tokens, Hkv, D] of the slots (``pages[t]``, ``offsets[t]``) of the 8-bit cache as bf16 (to move a
    request to a bf16 pool, or off the device): code * scale, which bf16 holds exactly for the scales that
    ``paged_cache_write_int8_`` makes.  A slot outside the pool gives zeros and sets ``status``."""

    heads, d, cache = _int8_cache(layer_cache, layer_scales)
    tokens = _int8_slots(pages, offsets)
    shape = (tokens, heads, d)
    target = []
    for given in (key, value):
        if given is None:  # sizes as numbers parse faster than as a tuple
            t = torch.empty(tokens, heads, d, dtype=torch.bfloat16, device=layer_cache.device)
            target.append((t, (t.data_ptr(), heads * d, d)))
        else:
            target.append((given, _int8_heads(given, shape)))
    (key, key_args), (value, value_args) = target
    _lib.launch(
        _lib.one_device(layer_cache, layer_scales, pages, offsets, key, value, status), "nq_kv_int8_read", *cache,
        pages.data_ptr(), offsets.data_ptr(), tokens, heads, d, *key_args, *value_args, _int8_status(status),
    )
    return key, value


def paged_attention_int8_workspace_bytes(tokens: int, rows: int, qo_heads: int, kv_heads: int, head_dim: int,
                                         parts: int = _lib.NQ_ATTN_DECODE | _lib.NQ_ATTN_PREFILL) -> int:
    """The workspace ``paged_attention_int8`` needs; raises for shapes it does not cover."""

    n = int(_lib.load().nq_paged_attention_int8_workspace_bytes(tokens, rows, qo_heads, kv_heads, head_dim, parts))
    if n < 0:
        raise TypeError(f"no 8-bit paged attention for {tokens} tokens, {rows} rows, {qo_heads} / {kv_heads} heads of "
                        f"{head_dim}")
    return n


def paged_attention_int8(query: torch.Tensor, layer_cache: torch.Tensor, layer_scales: torch.Tensor, metadata, *,
                         sm_scale: float | None = None, parts: int | None = None,
                         status: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged attention of ``query`` [tokens, Hq, D] (bf16) over one layer of the 8-bit cache (see
    ``paged_cache_write_int8_``) with ``metadata`` (a TalkerAttentionMetadata; its qo_indptr, paged_kv_indptr,
    paged_kv_indices and paged_kv_last_page_len are read), without a plan.  A captured call may be replayed with whatever
    the planner has written since: a paged_kv_indices that is the first part of a buffer stands for the whole buffer.

    ``parts`` as ``paged_attention_noalloc`` takes them: NQ_ATTN_DECODE for the rows with one query,
    NQ_ATTN_PREFILL for those with several (alone: for all of them); both by default, NQ_ATTN_DECODE where the
    metadata has no qo_indptr.  A query that sees no key gets zeros; tokens of no row keep what ``out`` held.
    A block whose K or V scale is negative or not finite makes the queries that see it NaN.
    ``workspace`` (``paged_attention_int8_workspace_bytes``; allocated if None) belongs to one call at a
    time.  The same inputs give the same bits.  No counterpart in the reference."""

    hkv, d, cache = _int8_cache(layer_cache, layer_scales)
    shape, strides = query.shape, query.stride()
    if len(shape) != 3 or strides[2] != 1:
        raise ValueError("query must be [tokens, Hq, D], contiguous per head")
    tokens, hq, q_dim = shape
    if q_dim != d or hq < hkv or hq % hkv:
        raise ValueError("query and cache disagree on the heads")
    if query.dtype is not torch.bfloat16 or (out is not None and out.dtype is not torch.bfloat16):
        raise TypeError("HIP attention kernels take bf16 tensors")
    if out is not None and (out.shape != shape or out.stride(2) != 1):
        raise ValueError("out must be [tokens, Hq, D] like the query")
    qo, kv, ids, last = (metadata.qo_indptr, metadata.paged_kv_indptr, metadata.paged_kv_indices,
                         metadata.paged_kv_last_page_len)
    for t in (qo, kv, ids, last):
        if t is not None:
            if t.dtype is not torch.int32:
                raise TypeError("paged metadata must be int32")
            if t.ndim != 1 or not t.is_contiguous():
                raise ValueError("paged metadata must be contiguous vectors")
    rows = kv.shape[0] - 1
    if rows < 0 or last.shape[0] < rows or (qo is not None and qo.shape[0] != rows + 1):
        raise ValueError("paged metadata must describe one set of rows")
    if parts is None:
        parts = _lib.NQ_ATTN_DECODE if qo is None else _lib.NQ_ATTN_DECODE | _lib.NQ_ATTN_PREFILL
    if qo is None and (parts != _lib.NQ_ATTN_DECODE or rows > tokens):
        raise ValueError("without qo_indptr every row has one query and only NQ_ATTN_DECODE runs")
    sm_scale = float(d) ** -0.5 if sm_scale is None else float(sm_scale)
    if not -_INT8_SM_SCALE < sm_scale < _INT8_SM_SCALE:
        raise ValueError("sm_scale must be finite, also times log2(e) in float32")
    index = _lib.one_device(query, layer_cache, layer_scales, out, qo, kv, ids, last, status, workspace)
    # paged_kv_indptr says which entries count.  A planner's paged_kv_indices is the part of its buffer that one step fills:
    # a captured call reads the lists of later steps from the same buffer, so the bound is what the buffer holds.
    entries = ids.shape[0]
    room = ids.untyped_storage().nbytes() // 4 - ids.storage_offset()
    if room > entries:
        entries = max(entries, min(room, _INT8_SLOTS // cache[-1]))
    o_strides = (hq * d, d) if out is None else out.stride()
    out = torch.empty(tokens, hq, d, dtype=torch.bfloat16, device=query.device) if out is None else out
    if tokens == 0 or rows == 0:
        return out
    need = paged_attention_int8_workspace_bytes(tokens, rows, hq, hkv, d, parts)
    if workspace is None:
        workspace, size = torch.empty(need, dtype=torch.uint8, device=query.device), need
    else:
        size = workspace.numel() * workspace.element_size()
        if size < need or not workspace.is_contiguous():
            raise ValueError(f"8-bit paged attention needs a contiguous workspace of {need} bytes")
    _lib.launch(
        index, "nq_paged_attention_int8", None if qo is None else qo.data_ptr(), kv.data_ptr(), last.data_ptr(),
        ids.data_ptr(), rows, entries, query.data_ptr(), strides[0], strides[1], tokens, *cache, hq, hkv, d,
        sm_scale, out.data_ptr(), o_strides[0], o_strides[1], int(parts), workspace.data_ptr(), size,
        _int8_status(status),
    )
    return out


__all__ = [
    "INT8_BLOCK",
    "paged_attention_int8",
    "paged_attention_int8_workspace_bytes",
    "paged_cache_read_int8",
    "paged_cache_write_int8_",
    "paged_attention_noalloc",
    "decode_attn_nhd_short_cache",
    "paired_qk_norm_rope_",
    "paired_qk_norm_rope_dense_cache_",
    "qkv_partials_norm_rope_dense_cache_",
    "qkv_partials_rope_short_attention_",
    "paired_qk_norm_rope_paged_cache_",
]
