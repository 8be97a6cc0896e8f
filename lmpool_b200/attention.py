"""Drop-in ``store_kvcache`` (src/lmpool/layers/attention.py:67-108) on B200.

The reference launches a Triton program per (token, kv head) that copies
``head_dim`` elements of K and V into ``cache[slot // bs, slot % bs, h]``
(attention.py:7-64). Here one sm_100a kernel moves a token's whole row
(all heads: ``kv_heads * head_dim`` contiguous elements, e.g. 2 KiB) per warp
with 16-byte vectors, K and V on neighbouring warps. ``store_kvcache_layers``
writes every layer of a step in one launch.

Both run on the current CUDA stream, never synchronise and never allocate,
so they can be captured in a CUDA graph (model_runner.py:630-683). Slots
outside ``[-1, num_blocks * block_size)`` are skipped and recorded in a
per-device status word (``kv_transfer.check_device_status``); the reference
kernel would write out of bounds for them.

Beside them stand a 4-bit form of the cache (``store_kvcache_q4``,
``load_kvcache_q4``) and the attention that reads either cache
(``paged_attention``, ``paged_attention_q4``): what LMPool's
``Attention.forward`` does right after the store (attention.py:490-507), with
an optional sliding window and sinks.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _capi
from .kv_transfer import _STATUS, _status_word


def _cache_strides(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int]:
    if k_cache.dim() != 4:
        raise RuntimeError("k_cache must be [num_blocks, block_size, num_kv_heads, head_dim]")
    st = k_cache.stride()
    if st != v_cache.stride():
        raise RuntimeError("k_cache and v_cache must have the same strides")
    H, D = k_cache.shape[2], k_cache.shape[3]
    if st[3] != 1 or (H > 1 and st[2] != D):
        raise RuntimeError("each cache slot [num_kv_heads, head_dim] must be contiguous")
    e = k_cache.element_size()
    return st[0] * e, st[1] * e


def _device_of(*tensors: torch.Tensor) -> int:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError("store_kvcache needs CUDA tensors: the B200 path has no CPU implementation")
    for t in tensors[1:]:
        if t.device != dev:
            raise RuntimeError(f"all tensors must be on {dev}, got {t.device}")
    return dev.index if dev.index is not None else torch.cuda.current_device()


def _raw_stream(device: int) -> int:
    """cudaStream_t of the current stream (cheap path; capture streams included)."""
    try:
        return torch._C._cuda_getCurrentRawStream(device)
    except AttributeError:
        return torch.cuda.current_stream(device).cuda_stream


def store_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
) -> None:
    """attention.py:67-108: ``cache[slot // bs, slot % bs] = key[t]`` for every slot != -1."""
    num_tokens, num_kv_heads, head_dim = key.shape
    if not key.is_contiguous():
        key = key.contiguous()
    if not value.is_contiguous():
        value = value.contiguous()
    assert k_cache.shape == v_cache.shape, "K and V cache shapes must match"
    assert slot_mapping.numel() == num_tokens, "Slot mapping size must match number of tokens"
    if slot_mapping.dtype != torch.int64:
        raise TypeError(f"slot_mapping must be int64, got {slot_mapping.dtype}")
    if key.dtype != k_cache.dtype or value.dtype != v_cache.dtype:
        raise TypeError("key/value and cache dtypes must match (the copy is bit-exact)")
    kshape = k_cache.shape
    if kshape[2] != num_kv_heads or kshape[3] != head_dim or value.shape != key.shape:
        raise RuntimeError("key/value [T, H, D] must match the cache's [H, D]")
    device = _device_of(key, value, k_cache, v_cache, slot_mapping)
    if num_tokens == 0:
        return
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    block_stride, slot_stride = _cache_strides(k_cache, v_cache)
    e = key.element_size()
    rc = _capi.lib().kvx_store_kvcache(
        device, key.data_ptr(), value.data_ptr(), key.stride(0) * e, value.stride(0) * e, k_cache.data_ptr(),
        v_cache.data_ptr(), block_stride, slot_stride, slot_mapping.data_ptr(), num_tokens, kshape[0],
        int(block_size), num_kv_heads * head_dim * e, _status_word(device).data_ptr(), _raw_stream(device))
    if rc:
        _capi.check(rc, "kvx_store_kvcache")


def store_kvcache_layers(
    keys: torch.Tensor,
    values: torch.Tensor,
    kv_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
) -> None:
    """Every layer in one launch.

    ``keys``/``values``: ``[L, T, H, D]`` (each layer's token rows contiguous);
    ``kv_cache``: the ``[2, L, N, bs, H, D]`` tensor of model_runner.py:397-400.
    Equivalent to ``store_kvcache(keys[l], values[l], kv_cache[0, l],
    kv_cache[1, l], slot_mapping, block_size)`` for every l.
    """
    if kv_cache.dim() != 6:
        raise RuntimeError("kv_cache must be [2, L, N, block_size, H, D]")
    L, T, H, D = keys.shape
    if values.shape != keys.shape:
        raise RuntimeError("keys and values must have the same shape")
    if tuple(kv_cache.shape[1:2]) != (L,) or tuple(kv_cache.shape[4:]) != (H, D):
        raise RuntimeError("keys [L, T, H, D] do not match kv_cache [2, L, N, bs, H, D]")
    assert slot_mapping.numel() == T, "Slot mapping size must match number of tokens"
    if slot_mapping.dtype != torch.int64:
        raise TypeError(f"slot_mapping must be int64, got {slot_mapping.dtype}")
    if keys.dtype != kv_cache.dtype or values.dtype != kv_cache.dtype:
        raise TypeError("key/value and cache dtypes must match (the copy is bit-exact)")
    for name, t in (("keys", keys), ("values", values)):
        if t.stride(3) != 1 or (H > 1 and t.stride(2) != D):
            raise RuntimeError(f"{name}: each token row [H, D] must be contiguous")
    device = _device_of(keys, values, kv_cache, slot_mapping)
    if T == 0:
        return
    slot_mapping = slot_mapping.contiguous()
    k0, v0 = kv_cache[0, 0], kv_cache[1, 0]
    block_stride, slot_stride = _cache_strides(k0, v0)
    e = keys.element_size()
    rc = _capi.lib().kvx_store_kvcache_layers(
        device, L, keys.data_ptr(), values.data_ptr(), keys.stride(0) * e, values.stride(0) * e, keys.stride(1) * e,
        values.stride(1) * e, k0.data_ptr(), v0.data_ptr(), kv_cache.stride(1) * e, kv_cache.stride(1) * e,
        block_stride, slot_stride, slot_mapping.data_ptr(), T, kv_cache.shape[2], int(block_size), H * D * e,
        _status_word(device).data_ptr(), _raw_stream(device))
    if rc:
        _capi.check(rc, "kvx_store_kvcache_layers")


# ---------------------------------------------------------------------------
# 4-bit cache
# ---------------------------------------------------------------------------

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1}


def _status(device: int) -> int:
    """Address of the device's status word. Its first use allocates it, which a graph's capture must not record."""
    word = _STATUS.get(device)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make the first call on a device before capturing a graph")
        word = _status_word(device)
    return word.data_ptr()


def q4_row_bytes(head_dim: int) -> int:
    """Bytes of one token's row of one kv head in a 4-bit cache: ``head_dim / 2`` of codes and ``head_dim / 16``
    of scales. A 4-bit cache is a ``uint8`` tensor ``[..., N, block_size, H, q4_row_bytes(D)]``; inside a page the
    bytes are laid out head by head, codes before scales (include/kvx.h), so only whole pages are meaningful. The
    block mover (``kv_transfer``) takes such a cache as it takes any other."""
    if head_dim <= 0 or head_dim % 16:
        raise ValueError(f"head_dim must be a multiple of 16, got {head_dim}")
    return head_dim // 2 + head_dim // 16


def _q4_check(k_cache: torch.Tensor, v_cache: torch.Tensor, block_size: int, head_dim: int) -> int:
    """Checks a 4-bit cache; its block stride in bytes."""
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise TypeError("a 4-bit cache holds bytes: k_cache and v_cache must be uint8")
    shape, st = k_cache.shape, k_cache.stride()
    if shape != v_cache.shape or st != v_cache.stride():
        raise RuntimeError("k_cache and v_cache must have the same shape and strides")
    if len(shape) != 4:
        raise RuntimeError("k_cache must be [num_blocks, block_size, num_kv_heads, head_dim / 2 + head_dim / 16]")
    N, bs, H, row = shape
    if bs != block_size or row * 16 != head_dim * 9 or head_dim % 16:
        raise RuntimeError(f"a 4-bit cache for block_size {block_size} and head_dim {head_dim} is [num_blocks, "
                           f"{block_size}, num_kv_heads, head_dim / 2 + head_dim / 16], got {list(shape)}")
    if st[3] != 1 or (H > 1 and st[2] != row) or (bs > 1 and st[1] != H * row):
        raise RuntimeError("each page [block_size, num_kv_heads, row] of a 4-bit cache must be contiguous")
    return st[0] if N > 1 else bs * H * row


def _same_device(first: torch.Tensor, *others: torch.Tensor) -> int:
    """The CUDA device of all of them (raises as ``_device_of``, at less cost a call)."""
    device = first.get_device()
    if device < 0:
        return _device_of(first, *others)
    for t in others:
        if t.get_device() != device:
            return _device_of(first, *others)
    return device


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """16-bit x [T, H, D] with contiguous, 16-byte aligned token rows (a copy where it has none). The stride of a
    dimension of one entry is not used and may be anything."""
    T, H, D = x.shape
    st = x.stride()
    if st[2] == 1 and (H == 1 or st[1] == D) and (T == 1 or st[0] % 8 == 0) and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _token_stride(x: torch.Tensor) -> int:
    """Bytes from a token's row of 16-bit x [T, H, D] to the next one's; a single token's is that of its row."""
    return 2 * x.stride(0) if x.shape[0] > 1 else 2 * x.shape[1] * x.shape[2]


def _check_slots(slot_mapping: torch.Tensor) -> torch.Tensor:
    if slot_mapping.dtype != torch.int64:
        raise TypeError(f"slot_mapping must be int64, got {slot_mapping.dtype}")
    return slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()


def store_kvcache_q4(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> None:
    """:func:`store_kvcache` into a 4-bit cache: rows are rounded to 4 bits on the way.

    ``key``/``value``: bf16 or fp16 ``[T, H, D]``, ``D`` a multiple of 16 up to 256; caches: ``uint8`` ``[N,
    block_size, H, q4_row_bytes(D)]``, ``block_size`` a multiple of 16. Every 16 elements of a row share an e4m3 scale
    ``amax / 6`` and become e2m1 codes (4.5 bits an element), all rounded to the nearest, ties to even. A group with an
    infinity or a NaN reads back as NaN. The scales reach from 2^-9 to 448 (elements up to 2688); ``k_scale`` and
    ``v_scale``, powers of two, divide what is stored where rows lie outside that, and every reader of the cache takes
    the same two numbers. Slots as in :func:`store_kvcache`; two tokens of a call must not share one.
    """
    T, H, D = key.shape
    if value.shape != key.shape:
        raise RuntimeError("key and value must have the same shape")
    if key.dtype not in _DTYPE_CODE or value.dtype != key.dtype:
        raise TypeError(f"key and value must both be bfloat16 or float16, got {key.dtype} and {value.dtype}")
    assert slot_mapping.numel() == T, "Slot mapping size must match number of tokens"
    block_stride = _q4_check(k_cache, v_cache, block_size, D)
    num_blocks, _, kv_heads, _ = k_cache.shape
    if kv_heads != H:
        raise RuntimeError("key/value [T, H, D] must match the cache's kv heads")
    slot_mapping = _check_slots(slot_mapping)
    device = _same_device(key, value, k_cache, v_cache, slot_mapping)
    if T == 0:
        return
    key, value = _rows_of(key), _rows_of(value)
    rc = _capi.lib().kvx_store_kvcache_q4(
        device, _DTYPE_CODE[key.dtype], key.data_ptr(), value.data_ptr(), _token_stride(key), _token_stride(value),
        k_cache.data_ptr(), v_cache.data_ptr(), block_stride, slot_mapping.data_ptr(), T, num_blocks, block_size, H, D,
        k_scale, v_scale, _status(device), _raw_stream(device))
    if rc:
        _capi.check(rc, "kvx_store_kvcache_q4")


def load_kvcache_q4(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
    dtype: torch.dtype = torch.bfloat16,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of a 4-bit cache as ``dtype`` (bf16 or fp16) ``key, value [T, H, D]``: what :func:`store_kvcache_q4` kept
    of them. With ``k_scale`` and ``v_scale`` of 1 every value is exact in either type. Rows of slot -1 are zero. To
    turn pages of a 4-bit cache into pages of a 16-bit one, pass the result to :func:`store_kvcache`."""
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    if k_cache.dim() != 4 or k_cache.shape[3] % 9:
        raise RuntimeError("k_cache must be [num_blocks, block_size, num_kv_heads, head_dim / 2 + head_dim / 16]")
    D = k_cache.shape[3] // 9 * 16
    block_stride = _q4_check(k_cache, v_cache, block_size, D)
    slot_mapping = _check_slots(slot_mapping)
    device = _same_device(k_cache, v_cache, slot_mapping)
    T, H = slot_mapping.numel(), k_cache.shape[2]
    key = torch.empty((T, H, D), dtype=dtype, device=k_cache.device)
    value = torch.empty_like(key)
    if T == 0:
        return key, value
    rc = _capi.lib().kvx_load_kvcache_q4(
        device, _DTYPE_CODE[dtype], key.data_ptr(), value.data_ptr(), H * D * 2, H * D * 2, k_cache.data_ptr(),
        v_cache.data_ptr(), block_stride, slot_mapping.data_ptr(), T, k_cache.shape[0], block_size, H, D,
        k_scale, v_scale, _status(device), _raw_stream(device))
    if rc:
        _capi.check(rc, "kvx_load_kvcache_q4")
    return key, value


# ---------------------------------------------------------------------------
# Attention over the paged cache
# ---------------------------------------------------------------------------

def _rows_overlap(tokens: int, token_stride: int, heads: int, head_stride: int, size: int) -> bool:
    """Whether two of the rows of ``size`` elements at ``t * token_stride + h * head_stride`` share one."""
    if tokens == 0 or heads == 0:
        return False
    if tokens == 1 or heads == 1:
        return tokens * heads > 1 and (token_stride if tokens > 1 else head_stride) < size
    (small, n), (large, m) = sorted(((token_stride, tokens), (head_stride, heads)))
    if small < size:
        return True
    span = (n - 1) * small + size
    if large >= span:
        return False
    # Crossed: a step along the large stride ends between two rows of the small one.
    for far in range(large, min(m * large, span), large):
        rest = far % small
        if rest < size or (small - rest < size and far + small - rest < span):
            return True
    return False


@functools.lru_cache(maxsize=1024)
def _attention_workspace(device: int, ragged: bool, sizes: tuple) -> int:
    """Bytes of scratch that a call needs: its sizes alone decide."""
    out = ctypes.c_uint64(0)
    args = _capi.pack_attention(0, 0, 0, 0, 0, 0, int(ragged), *(0,) * 8, 1, *sizes)
    _capi.check(_capi.lib().kvx_attention_workspace(device, args, ctypes.byref(out)), "kvx_attention_workspace")
    return out.value


def _paged_attention(query, k_cache, v_cache, block_tables, context_lens, block_size, cu_seqlens_q, scale, window, sinks,
                     out, bits, k_scale, v_scale):
    # This runs once a layer and step: what follows is written for few interpreter steps.
    if query.dim() != 3:
        raise RuntimeError("query must be [num_tokens, num_heads, head_dim]")
    T, heads, D = query.shape
    dtype = query.dtype
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"query must be bfloat16 or float16, got {dtype}")
    if D != 64 and D != 128:
        raise RuntimeError(f"head_dim must be 64 or 128, got {D}")
    st = k_cache.stride()
    if bits == 4:
        block_stride, slot_stride, head_stride = _q4_check(k_cache, v_cache, block_size, D), 0, 0
    else:
        if k_cache.dtype != dtype or v_cache.dtype != dtype:
            raise TypeError("query and cache dtypes must match")
        shape = k_cache.shape
        if len(shape) != 4 or shape != v_cache.shape:
            raise RuntimeError("k_cache and v_cache must both be [num_blocks, block_size, num_kv_heads, head_dim]")
        if st != v_cache.stride():
            raise RuntimeError("k_cache and v_cache must have the same strides")
        if shape[1] != block_size or shape[3] != D:
            raise RuntimeError(f"the cache's pages [block_size, num_kv_heads, head_dim] do not match block_size "
                               f"{block_size} and head_dim {D}")
        if st[3] != 1:
            raise RuntimeError("the cache's head_dim must be contiguous")
        # The stride of a dimension of one entry is not used and may be anything.
        block_stride = 2 * st[0] if shape[0] > 1 else 2 * D * block_size * shape[2]
        slot_stride = 2 * st[1] if block_size > 1 else 2 * D * shape[2]
        head_stride = 2 * st[2] if shape[2] > 1 else 2 * D
    num_blocks, _, kv_heads, _ = k_cache.shape
    if kv_heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{heads} query heads are no multiple of {kv_heads} kv heads")
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise TypeError("block_tables and context_lens must be int32")
    if block_tables.dim() != 2 or context_lens.dim() != 1 or block_tables.shape[0] != context_lens.shape[0]:
        raise RuntimeError("block_tables must be [num_seqs, width] and context_lens [num_seqs]")
    S, width = block_tables.shape
    table_stride, step = block_tables.stride()
    if width > 1 and step != 1:
        block_tables = block_tables.contiguous()
        table_stride = width
    if S > 1 and context_lens.stride(0) != 1:
        context_lens = context_lens.contiguous()
    device = _same_device(query, k_cache, v_cache, block_tables, context_lens)
    cu = 0
    if cu_seqlens_q is None:
        if T != S:
            raise RuntimeError(f"without cu_seqlens_q every sequence has one token: {T} tokens, {S} sequences")
    else:
        if cu_seqlens_q.dtype != torch.int32:
            raise TypeError(f"cu_seqlens_q must be int32, got {cu_seqlens_q.dtype}")
        if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] != S + 1:
            raise RuntimeError(f"cu_seqlens_q must hold num_seqs + 1 = {S + 1} entries")
        if S > 0 and cu_seqlens_q.stride(0) != 1:
            cu_seqlens_q = cu_seqlens_q.contiguous()
        _same_device(query, cu_seqlens_q)
        cu = cu_seqlens_q.data_ptr()
    if window is None:
        window = 0
    elif window <= 0:
        raise ValueError(f"window must be positive (None: every key), got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    # The stride of a dimension of one entry is not used and may be anything.
    qs = query.stride()
    q_step, q_head = qs[0] if T > 1 else heads * D, qs[1] if heads > 1 else D
    if qs[2] != 1 or q_step % 8 or q_head % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)
        q_step, q_head = heads * D, D
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        o_step, o_head = heads * D, D
    else:
        if out.shape != query.shape or out.dtype != dtype:
            raise RuntimeError("out must have query's shape and dtype")
        _same_device(query, out)
        os = out.stride()
        o_step, o_head = os[0] if T > 1 else heads * D, os[1] if heads > 1 else D
        if os[2] != 1 or o_step % 8 or o_head % 8 or out.data_ptr() % 16:
            raise RuntimeError("out must have contiguous, 16-byte aligned rows of head_dim")
        if _rows_overlap(T, o_step, heads, o_head, D):
            raise RuntimeError("out's rows must not overlap")
        if out.data_ptr() == query.data_ptr() and T:
            raise RuntimeError("out must not be the query")
    if T == 0 or S == 0:
        return out
    # Positions are 32-bit: a window or sinks beyond them are all the same.
    sizes = (T, S, heads, kv_heads, D, block_size, width, code, bits, min(window, _INT_MAX), min(sinks, _INT_MAX),
             D ** -0.5 if scale is None else scale, k_scale, v_scale, 0, 0)
    need = _attention_workspace(device, cu != 0, sizes)
    workspace = None
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=query.device)
        workspace = scratch.data_ptr()
    rc = _capi.lib().kvx_paged_attention(
        device,
        _capi.pack_attention(query.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                             block_tables.data_ptr(), context_lens.data_ptr(), cu, 2 * q_step, 2 * q_head, 2 * o_step,
                             2 * o_head, block_stride, slot_stride, head_stride, table_stride, num_blocks, *sizes),
        workspace, need, _status(device), _raw_stream(device))
    if rc:
        _capi.check(rc, "kvx_paged_attention")
    return out


_INT_MAX = 2 ** 31 - 1


def paged_attention(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    *,
    cu_seqlens_q: torch.Tensor | None = None,
    scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of new tokens over the paged cache they were stored in, optionally with a sliding window and
    a few first tokens that stay visible (sinks).

    ``query``: bf16 or fp16 ``[T, Hq, D]``, ``D`` 64 or 128; caches ``[N, block_size, H, D]`` of the same type, as
    :func:`store_kvcache` fills them (any strides over blocks, slots and heads that are multiples of 16 bytes);
    ``block_tables`` int32 ``[S, width]`` page ids; ``context_lens`` int32 ``[S]``: tokens of each sequence in the
    cache, the new ones among them. Query head ``h`` reads kv head ``h // (Hq // H)``.

    Without ``cu_seqlens_q`` each sequence has one new token (``T == S``, decode). With it (int32 ``[S + 1]``, rising
    from 0) sequence ``s`` has the tokens ``cu_seqlens_q[s]`` to ``cu_seqlens_q[s + 1]``, the last of its context:
    prompts, chunks of prompts, drafted tokens. (They may be mixed, but a call is planned for the average of new tokens a
    sequence: single tokens and long prompts are quicker as two calls.) Token at position ``p`` sees key ``j <= p`` if ``window`` is None, if
    ``p - j < window`` or if ``j < sinks``. A token that sees no key gets zeros. Rows behind the last sequence are left
    as they were. ``out`` takes the result and must not overlap the inputs. ``scale`` (default ``D ** -0.5``) must be
    positive. No gradient is recorded: this reads a serving cache. A value that is infinite or NaN decides its element of
    the tokens that see it and reaches no other.

    Runs on the current stream without synchronising; lengths and tables are read on the device, so a captured call
    can be replayed with others. Bad page ids (their keys read as zeros) and lengths are recorded in the device's
    status word (``kv_transfer.check_device_status``).
    """
    return _paged_attention(query, k_cache, v_cache, block_tables, context_lens, block_size, cu_seqlens_q, scale, window,
                            sinks, out, 16, 1.0, 1.0)


def paged_attention_q4(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    *,
    cu_seqlens_q: torch.Tensor | None = None,
    scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_attention` over a 4-bit cache (``uint8`` ``[N, block_size, H, q4_row_bytes(D)]``, filled by
    :func:`store_kvcache_q4` with the same ``k_scale`` and ``v_scale``). The cache is read as 4.5 bits an element and
    widened, exactly, next to the products."""
    return _paged_attention(query, k_cache, v_cache, block_tables, context_lens, block_size, cu_seqlens_q, scale, window,
                            sinks, out, 4, k_scale, v_scale)
