"""Paged KV-cache append, mirroring ``flashinfer.page.append_paged_kv_cache`` as called at
miniagentserve/models/devstral2/devstral2.py:170-173, plus the equivalent slot-mapping store.

Cache layout (miniagentserve/engine/model_runner.py:83-85): per layer ``[num_pages, page_size,
kv_heads, head_dim]`` for "NHD", ``[num_pages, kv_heads, page_size, head_dim]`` for "HND". The
model runner keeps one extra page as a sink for padding rows (model_runner.py:82), so duplicate
destinations within one call are legal; the kernel lets one writer win.

The same store into a cache held in 4 bits (``Fp4KVCache``, ``fp4_kv_cache``): ``append_paged_kv_cache_fp4`` and
``store_kv_slots_fp4`` quantize the rows on the way, ``load_kv_slots_fp4`` reads rows back as bf16. Keys and
values are microscaling fp4: a head's row is cut into blocks of 32 elements, each 32 e2m1 codes under one power of
two, 4.25 bits an element against 16. The attention over it is ``attention.batch_decode_with_fp4_kv_cache`` and
``attention.batch_context_with_fp4_kv_cache``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._tensors import error_word, require_dtype, require_gpu, require_same_device

__all__ = ["append_paged_kv_cache", "store_kv_slots", "slot_mapping_from_block_tables", "Fp4KVCache", "fp4_kv_cache",
           "append_paged_kv_cache_fp4", "store_kv_slots_fp4", "load_kv_slots_fp4"]

FP4_BLOCK = 32        # elements of a head's row that share a power of two
FP4_MIN_PAGE = 16     # slots per page, at least


def _cache_geometry(paged_kv_cache, kv_layout: str):
    """(k_cache, v_cache, page_stride, entry_stride, head_stride, num_pages, page_size, heads, dim)."""
    if kv_layout not in ("NHD", "HND"):
        raise ValueError(f"kv_layout must be 'NHD' or 'HND', got {kv_layout!r}")
    if isinstance(paged_kv_cache, (tuple, list)):
        if len(paged_kv_cache) != 2:
            raise ValueError("paged_kv_cache tuple must be (k_cache, v_cache)")
        k_cache, v_cache = paged_kv_cache
    else:
        t = paged_kv_cache
        if t.dim() != 5 or t.shape[1] != 2:
            raise ValueError("a single paged_kv_cache tensor must be [num_pages, 2, ...] (k at index 0, v at 1)")
        k_cache, v_cache = t[:, 0], t[:, 1]
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        require_gpu(c, name)
        require_dtype(c, name, torch.bfloat16)
        if c.dim() != 4:
            raise ValueError(f"{name} must be 4-D, got shape {tuple(c.shape)}")
        if c.shape[3] > 1 and c.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    if kv_layout == "NHD":
        num_pages, page_size, heads, dim = k_cache.shape
        page_stride, entry_stride, head_stride = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    else:
        num_pages, heads, page_size, dim = k_cache.shape
        page_stride, entry_stride, head_stride = k_cache.stride(0), k_cache.stride(2), k_cache.stride(1)
    return k_cache, v_cache, page_stride, entry_stride, head_stride, num_pages, page_size, heads, dim


def _source_view(t: torch.Tensor, name: str, heads: int, dim: int) -> tuple[int, int, int]:
    """(rows, row_stride, head_stride) of [nnz, heads, dim] or [nnz, heads * dim] k/v rows."""
    require_gpu(t, name)
    require_dtype(t, name, torch.bfloat16)
    if t.dim() == 3:
        if tuple(t.shape[1:]) != (heads, dim):
            raise ValueError(f"{name} shape {tuple(t.shape)} does not match the cache's ({heads}, {dim}) heads")
        if dim > 1 and t.stride(2) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
        return t.shape[0], t.stride(0), t.stride(1)
    if t.dim() == 2:
        if t.shape[1] != heads * dim:
            raise ValueError(f"{name} width {t.shape[1]} != kv_heads * head_dim = {heads * dim}")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        return t.shape[0], t.stride(0), dim
    raise ValueError(f"{name} must be [nnz, kv_heads, head_dim] or [nnz, kv_heads * head_dim]")


def _index_vector(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    require_gpu(t, name)
    require_dtype(t, name, dtype)
    if t.dim() != 1 or (t.numel() > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous 1-D tensor")


def _append(append_key, append_value, batch_indices, positions, paged_kv_cache, kv_indices, kv_indptr,
            kv_layout: str, error_flags: torch.Tensor | None) -> None:
    k_cache, v_cache, pstride, estride, hstride, pages, page_size, heads, dim = _cache_geometry(paged_kv_cache,
                                                                                                kv_layout)
    rows, ks, khs = _source_view(append_key, "append_key", heads, dim)
    vrows, vs, vhs = _source_view(append_value, "append_value", heads, dim)
    for name, t in (("batch_indices", batch_indices), ("positions", positions), ("kv_indices", kv_indices),
                    ("kv_indptr", kv_indptr)):
        _index_vector(t, name, torch.int32)
    device = require_same_device(("append_key", append_key), ("append_value", append_value), ("k_cache", k_cache),
                                 ("batch_indices", batch_indices), ("positions", positions),
                                 ("kv_indices", kv_indices), ("kv_indptr", kv_indptr))
    if not (vrows == rows == batch_indices.shape[0] == positions.shape[0]):
        raise ValueError("append_key, append_value, batch_indices and positions must have the same length")
    if kv_indptr.shape[0] < 1:
        raise ValueError("kv_indptr needs batch + 1 entries")
    st = _lib.load().mas_append_paged_kv_cache_bf16(
        k_cache.data_ptr(), v_cache.data_ptr(), pstride, estride, hstride, pages, page_size, append_key.data_ptr(),
        ks, khs, append_value.data_ptr(), vs, vhs, batch_indices.data_ptr(), positions.data_ptr(),
        kv_indices.data_ptr(), kv_indices.shape[0], kv_indptr.data_ptr(), kv_indptr.shape[0] - 1, rows, heads, dim,
        error_word(error_flags, device), _lib.stream_handle(device))
    _lib.check(st, "append_paged_kv_cache")


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                          positions: torch.Tensor, paged_kv_cache, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor | None = None,
                          kv_layout: str = "NHD", *, error_flags: torch.Tensor | None = None) -> None:
    """Writes token t's k/v rows to page ``kv_indices[kv_indptr[b] + p // page_size]``, entry
    ``p % page_size``, where ``b = batch_indices[t]`` and ``p = positions[t]``.

    append_key/append_value: bf16 ``[nnz, kv_heads, head_dim]`` (any row stride, e.g. views of a
    fused qkv output); paged_kv_cache: ``(k_cache, v_cache)`` or one ``[num_pages, 2, ...]``
    tensor; index tensors int32. ``kv_last_page_len`` is accepted for signature compatibility
    and not needed by the store. Tokens whose destination is out of range are skipped; with
    ``error_flags`` (a 1-element int32 device tensor) the kernel records why (bits 2/4/8).
    """
    if torch.compiler.is_compiling():
        k_cache, v_cache = (paged_kv_cache if isinstance(paged_kv_cache, (tuple, list)) else (paged_kv_cache, None))
        torch.ops.mas.append_paged_kv_cache(append_key, append_value, batch_indices, positions, k_cache, v_cache,
                                            kv_indices, kv_indptr, kv_layout, error_flags)
        return
    _append(append_key, append_value, batch_indices, positions, paged_kv_cache, kv_indices, kv_indptr, kv_layout,
            error_flags)


def _store_slots(key, value, k_cache, v_cache, slot_mapping, kv_layout: str, error_flags) -> None:
    k_cache, v_cache, pstride, estride, hstride, pages, page_size, heads, dim = _cache_geometry((k_cache, v_cache),
                                                                                                kv_layout)
    rows, ks, khs = _source_view(key, "key", heads, dim)
    vrows, vs, vhs = _source_view(value, "value", heads, dim)
    _index_vector(slot_mapping, "slot_mapping", torch.int64)
    device = require_same_device(("key", key), ("value", value), ("k_cache", k_cache), ("slot_mapping", slot_mapping))
    if not (vrows == rows == slot_mapping.shape[0]):
        raise ValueError("key, value and slot_mapping must have the same length")
    st = _lib.load().mas_store_kv_slots_bf16(
        k_cache.data_ptr(), v_cache.data_ptr(), pstride, estride, hstride, pages, page_size, key.data_ptr(), ks, khs,
        value.data_ptr(), vs, vhs, slot_mapping.data_ptr(), rows, heads, dim, error_word(error_flags, device),
        _lib.stream_handle(device))
    _lib.check(st, "store_kv_slots")


def store_kv_slots(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slot_mapping: torch.Tensor, kv_layout: str = "NHD", *,
                   error_flags: torch.Tensor | None = None) -> None:
    """Slot-mapping form of the store: token t goes to page ``slot // page_size``, entry
    ``slot % page_size`` with ``slot = slot_mapping[t]`` (int64); a negative slot is skipped."""
    if torch.compiler.is_compiling():
        torch.ops.mas.store_kv_slots(key, value, k_cache, v_cache, slot_mapping, kv_layout, error_flags)
        return
    _store_slots(key, value, k_cache, v_cache, slot_mapping, kv_layout, error_flags)


def slot_mapping_from_block_tables(block_tables: torch.Tensor, batch_indices: torch.Tensor, positions: torch.Tensor,
                                   page_size: int) -> torch.Tensor:
    """``slot[t] = block_tables[b, p // page_size] * page_size + p % page_size`` (int64), the slot
    that the block-table form of the store resolves for token t (devstral2.py:170-173,289)."""
    b = batch_indices.long()
    p = positions.long()
    return block_tables[b, p // page_size].long() * page_size + p % page_size


# ---- the cache in 4 bits -------------------------------------------------------------------------------

class Fp4KVCache(NamedTuple):
    """One layer's KV cache in microscaling fp4, all uint8.

    k, v: two e2m1 codes a byte (the even element in the low half), ``[num_pages, page_size, kv_heads, head_dim / 2]``
    ("NHD") or ``[num_pages, kv_heads, page_size, head_dim / 2]`` ("HND"); k_scale, v_scale: for each block of 32
    elements its power of two's exponent + 127 (255: NaN), ``[num_pages, kv_heads, head_dim / 32, page_size]`` for both.
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def fp4_kv_cache(num_pages: int, page_size: int, kv_heads: int, head_dim: int, device,
                 kv_layout: str = "HND") -> Fp4KVCache:
    """A zeroed 4-bit cache. In "HND" order a head's page is one run of memory (1 KiB of codes at 16 slots of 128),
    which is what attention reads at a time; in "NHD" order a token's heads are."""
    if kv_layout not in ("NHD", "HND"):
        raise ValueError(f"kv_layout must be 'NHD' or 'HND', got {kv_layout!r}")
    if page_size < FP4_MIN_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two of at least {FP4_MIN_PAGE}, got {page_size}")
    if head_dim <= 0 or head_dim % FP4_BLOCK:
        raise ValueError(f"head_dim must be a multiple of {FP4_BLOCK}, got {head_dim}")
    shape = (num_pages, page_size, kv_heads) if kv_layout == "NHD" else (num_pages, kv_heads, page_size)
    powers = (num_pages, kv_heads, head_dim // FP4_BLOCK, page_size)
    return Fp4KVCache(*(torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=device) for _ in range(2)),
                      *(torch.zeros(powers, dtype=torch.uint8, device=device) for _ in range(2)))


def _fp4_geometry(kv_cache, kv_layout: str):
    """(code strides (page, entry, head), (power strides (page, head), pages, page_size), heads, dim) of an Fp4KVCache
    or an equal tuple, checked."""
    if kv_layout not in ("NHD", "HND"):
        raise ValueError(f"kv_layout must be 'NHD' or 'HND', got {kv_layout!r}")
    if not isinstance(kv_cache, (tuple, list)) or len(kv_cache) != 4:
        raise ValueError("a 4-bit cache is an Fp4KVCache (k, v, k_scale, v_scale)")
    k, v, ks, vs = kv_cache
    for name, t in (("k", k), ("v", v), ("k_scale", ks), ("v_scale", vs)):
        require_gpu(t, name)
        require_dtype(t, name, torch.uint8)
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D, got shape {tuple(t.shape)}")
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
    # (a dimension of one has no stride of its own)
    def strides(t):
        return tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride()))

    k_strides, ks_strides = strides(k), strides(ks)
    if k.shape != v.shape or k_strides != strides(v) or ks.shape != vs.shape or ks_strides != strides(vs):
        raise ValueError("k and v, and k_scale and v_scale, must have the same shape and strides")
    if kv_layout == "NHD":
        num_pages, page_size, heads, half = k.shape
        page, entry, head = k_strides[:3]
    else:
        num_pages, heads, page_size, half = k.shape
        page, head, entry = k_strides[:3]
    dim = 2 * half
    if page_size < FP4_MIN_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two of at least {FP4_MIN_PAGE}, got {page_size}")
    if dim == 0 or dim % FP4_BLOCK:
        raise ValueError(f"head_dim must be a multiple of {FP4_BLOCK}, got {dim}")
    if tuple(ks.shape) != (num_pages, heads, dim // FP4_BLOCK, page_size):
        raise ValueError(f"k_scale and v_scale must be {(num_pages, heads, dim // FP4_BLOCK, page_size)}, "
                         f"got {tuple(ks.shape)}")
    if dim > FP4_BLOCK and ks.stride(2) != page_size:
        raise ValueError("k_scale and v_scale must be contiguous in their last two dimensions")
    require_same_device(("k", k), ("v", v), ("k_scale", ks), ("v_scale", vs))
    return (page, entry, head), (*ks_strides[:2], num_pages, page_size), heads, dim


def _fp4_args(kv_cache, code_strides, rest) -> tuple:
    """The C entry points' cache arguments."""
    k, v, ks, vs = kv_cache
    return (k.data_ptr(), v.data_ptr(), *code_strides, ks.data_ptr(), vs.data_ptr(), *rest)


def _append_fp4(append_key, append_value, batch_indices, positions, kv_cache, kv_indices, kv_indptr, kv_layout: str,
                error_flags: torch.Tensor | None) -> None:
    strides, rest, heads, dim = _fp4_geometry(kv_cache, kv_layout)
    rows, ks, khs = _source_view(append_key, "append_key", heads, dim)
    vrows, vs, vhs = _source_view(append_value, "append_value", heads, dim)
    for name, t in (("batch_indices", batch_indices), ("positions", positions), ("kv_indices", kv_indices),
                    ("kv_indptr", kv_indptr)):
        _index_vector(t, name, torch.int32)
    device = require_same_device(("append_key", append_key), ("append_value", append_value), ("k", kv_cache[0]),
                                 ("batch_indices", batch_indices), ("positions", positions),
                                 ("kv_indices", kv_indices), ("kv_indptr", kv_indptr))
    if not (vrows == rows == batch_indices.shape[0] == positions.shape[0]):
        raise ValueError("append_key, append_value, batch_indices and positions must have the same length")
    if kv_indptr.shape[0] < 1:
        raise ValueError("kv_indptr needs batch + 1 entries")
    err = error_word(error_flags, device)
    with _lib.on_device(device):
        st = _lib.load().mas_append_paged_kv_cache_fp4(
            *_fp4_args(kv_cache, strides, rest), append_key.data_ptr(), ks, khs, append_value.data_ptr(), vs, vhs, batch_indices.data_ptr(),
            positions.data_ptr(), kv_indices.data_ptr(), kv_indices.shape[0], kv_indptr.data_ptr(),
            kv_indptr.shape[0] - 1, rows, heads, dim, err, _lib.stream_handle(device))
    _lib.check(st, "append_paged_kv_cache_fp4")


def append_paged_kv_cache_fp4(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                              positions: torch.Tensor, kv_cache, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                              kv_last_page_len: torch.Tensor | None = None, kv_layout: str = "NHD", *,
                              error_flags: torch.Tensor | None = None) -> None:
    """``append_paged_kv_cache`` into a 4-bit cache: token t's k/v rows (bf16), quantized, to the same destination.

    Each block of 32 elements gets the smallest power of two (of at least 2^-127) under which its largest element
    lies below 7, and each element the nearest e2m1 code, ties to the even one: the bits follow from the row
    alone. A block that holds a NaN or an infinity stands for NaN throughout. Two tokens of one call must not share a
    destination: a block could keep the codes of one and the power of the other.
    """
    if torch.compiler.is_compiling():
        torch.ops.mas.append_paged_kv_cache_fp4(append_key, append_value, batch_indices, positions, *kv_cache,
                                                kv_indices, kv_indptr, kv_layout, error_flags)
        return
    if _lib.direct is not None and (st := _lib.direct.append_fp4(append_key, append_value, batch_indices, positions, kv_cache,
                                                                 kv_indices, kv_indptr, kv_layout, error_flags)) is not None:
        if st:
            _lib.check(st, "append_paged_kv_cache_fp4")
        return
    _append_fp4(append_key, append_value, batch_indices, positions, kv_cache, kv_indices, kv_indptr, kv_layout,
                error_flags)


def _slots_fp4(entry: str, key, value, kv_cache, slot_mapping, kv_layout: str, error_flags) -> None:
    strides, rest, heads, dim = _fp4_geometry(kv_cache, kv_layout)
    rows, ks, khs = _source_view(key, "key", heads, dim)
    vrows, vs, vhs = _source_view(value, "value", heads, dim)
    _index_vector(slot_mapping, "slot_mapping", torch.int64)
    device = require_same_device(("key", key), ("value", value), ("k", kv_cache[0]), ("slot_mapping", slot_mapping))
    if not (vrows == rows == slot_mapping.shape[0]):
        raise ValueError("key, value and slot_mapping must have the same length")
    err, cache = error_word(error_flags, device), _fp4_args(kv_cache, strides, rest)
    rows_args = (key.data_ptr(), ks, khs, value.data_ptr(), vs, vhs)
    first, then = (cache, rows_args) if entry == "store" else (rows_args, cache)
    lib = _lib.load()
    fn = lib.mas_store_kv_slots_fp4 if entry == "store" else lib.mas_load_kv_slots_fp4
    with _lib.on_device(device):
        st = fn(*first, *then, slot_mapping.data_ptr(), rows, heads, dim, err, _lib.stream_handle(device))
    _lib.check(st, f"{entry}_kv_slots_fp4")


def store_kv_slots_fp4(key: torch.Tensor, value: torch.Tensor, kv_cache, slot_mapping: torch.Tensor,
                       kv_layout: str = "NHD", *, error_flags: torch.Tensor | None = None) -> None:
    """Slot-mapping form of ``append_paged_kv_cache_fp4``: token t goes to page ``slot // page_size``, entry
    ``slot % page_size`` with ``slot = slot_mapping[t]`` (int64); a negative slot is skipped, and no
    slot is named twice."""
    if torch.compiler.is_compiling():
        torch.ops.mas.store_kv_slots_fp4(key, value, *kv_cache, slot_mapping, kv_layout, error_flags)
        return
    if _lib.direct is not None and (st := _lib.direct.store_slots_fp4(key, value, kv_cache, slot_mapping, kv_layout,
                                                                      error_flags)) is not None:
        if st:
            _lib.check(st, "store_kv_slots_fp4")
        return
    _slots_fp4("store", key, value, kv_cache, slot_mapping, kv_layout, error_flags)


def load_kv_slots_fp4(kv_cache, slot_mapping: torch.Tensor, kv_layout: str = "NHD", *, key: torch.Tensor | None = None,
                      value: torch.Tensor | None = None, error_flags: torch.Tensor | None = None):
    """The rows at ``slot_mapping`` (int64) as bf16 ``(key, value)``, each ``[nnz, kv_heads, head_dim]`` (allocated
    when not given): exactly the values the codes stand for, for moving rows to a bf16 cache or to another pool. A
    negative slot gives zeros; one past the cache too, and sets bit 16 of ``error_flags``."""
    if key is None or value is None:
        heads = kv_cache[2].shape[1]
        shape = (slot_mapping.shape[0], heads, 2 * kv_cache[0].shape[3])
        key = torch.empty(shape, dtype=torch.bfloat16, device=slot_mapping.device) if key is None else key
        value = torch.empty(shape, dtype=torch.bfloat16, device=slot_mapping.device) if value is None else value
    if torch.compiler.is_compiling():
        torch.ops.mas.load_kv_slots_fp4(key, value, *kv_cache, slot_mapping, kv_layout, error_flags)
        return key, value
    if _lib.direct is not None and (st := _lib.direct.load_slots_fp4(key, value, kv_cache, slot_mapping, kv_layout,
                                                                     error_flags)) is not None:
        if st:
            _lib.check(st, "load_kv_slots_fp4")
        return key, value
    _slots_fp4("load", key, value, kv_cache, slot_mapping, kv_layout, error_flags)
    return key, value
