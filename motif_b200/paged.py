"""A paged Chord key / value cache held in 4 bits, for serving requests of unequal lengths.

The reference keeps one contiguous 16-bit buffer per layer with one length for the whole batch
(`motif/model/cache.py:73-252`); these operators have no counterpart there.  A pool of pages is
shared by all requests, every request has a row of a block table, and a stored row of 64 dims
takes 36 bytes instead of 128, so a decode step reads 3.6 times fewer cache bytes.

    pool = kv4_pool(num_pages, num_kv_heads, head_dim)             # one per Chord layer
    slots, lens, count = paged_reserve(lens, new_lens, table, free, count, page_size, total_new)
    kv4_append(k, v, slots, pool)                                  # quantise and store the new tokens
    o = kv4_chord_attention(q, pool, table, lens, alpha, beta, mu, ssmax)   # newest tokens of each
    k, v = kv4_gather(pool, table, lens, max_len)                  # cached prefixes, for a prompt chunk
    paged_release(done, lens, table, free, count, page_size)       # finished requests give pages back

Every call launches on the current stream of its tensors' device and returns without waiting;
lengths, tables and the free list stay on the device, so a captured CUDA graph replays at any
lengths.  A stored value is `m + s (c - 8)` with a 4-bit code c and, per group of min(D, 64) dims
of one token, s = bf16((max - min) / 15), m = bf16(min + 8 s), c - 8 = the nearest whole number to
(x - m) / s within -8 .. 7 (ties to even).  A group with a NaN or an infinity (or whose range
exceeds the largest float) is stored as NaN.
"""

import functools
from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ['kv4_pool', 'paged_reserve', 'paged_release', 'kv4_append', 'kv4_gather', 'kv4_chord_attention']

UNIT = 16  # tokens of one storage unit: page sizes are multiples of it
_UNIT_BYTES = {32: 640, 64: 1152, 128: 2304}  # motif_b200_kv4_unit_bytes
_DIMS = {v: k for k, v in _UNIT_BYTES.items()}


def kv4_pool(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, device='cuda') -> torch.Tensor:
    """An empty pool `[num_pages, num_kv_heads, page_size / 16, unit bytes]` (uint8): its shape
    carries the page size and the head dim (32, 64 or 128) for the calls below."""
    if head_dim not in _UNIT_BYTES:
        raise NotImplementedError(f'head_dim must be 32, 64 or 128, got {head_dim}')
    if page_size < UNIT or page_size % UNIT or page_size > 1024:
        raise ValueError(f'page_size must be a multiple of {UNIT} up to 1024, got {page_size}')
    if num_pages < 1 or num_kv_heads < 1:
        raise ValueError(f'num_pages and num_kv_heads must be positive, got {num_pages}, {num_kv_heads}')
    return torch.zeros((num_pages, num_kv_heads, page_size // UNIT, _UNIT_BYTES[head_dim]), dtype=torch.uint8,
                       device=device)


@functools.lru_cache(maxsize=256)
def _shape_dims(shape):
    pages, kv, units, nbytes = shape
    return pages, kv, units * UNIT, _DIMS[nbytes]


def _pool_dims(pool) -> Tuple[int, int, int, int]:
    """(pages, kv heads, page size, head dim) of a pool."""
    if not isinstance(pool, torch.Tensor) or not pool.is_cuda:
        raise ValueError('pool must live on CUDA')
    shape = pool.shape
    if pool.dtype is not torch.uint8 or len(shape) != 4 or shape[3] not in _DIMS or not pool.is_contiguous():
        raise ValueError(f'pool must be a contiguous uint8 tensor from kv4_pool, got {pool.dtype} {tuple(shape)}')
    return _shape_dims(shape)


def _vector(name, t, n, dev, dtype=torch.int32):
    """t is a contiguous [n] tensor of dtype on dev."""
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f'{name} must live on {dev}')
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous {dtype} tensor [{n}], got {t.dtype} {tuple(t.shape)}')


def _table(t, dev, batch=None):
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f'block_table must live on {dev}')
    if t.dtype is not torch.int32 or t.dim() != 2 or t.stride(1) != 1 or (batch is not None and t.shape[0] != batch):
        raise ValueError(f'block_table must be an int32 [B, max_pages] tensor with contiguous rows, got {t.dtype} '
                         f'{tuple(t.shape)}')


@functools.lru_cache(maxsize=256)
def _attention_workspace(index, H, kv, T, D) -> int:
    with torch.cuda.device(index):
        return _lib.load().motif_b200_kv4_attention_workspace_bytes(H, kv, T, D)


def paged_reserve(lens, new_lens, block_table, free_pages, free_count, page_size: int, total_new: int,
                  lens_out: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None,
                  slots: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Reserve cache slots for `new_lens[b]` more tokens of every request; all on the device.

    `lens` / `new_lens` [B] int32: cached and new tokens; `block_table` [B, max_pages] int32, its
    first ceil(lens / page_size) columns in use; `free_pages[:free_count]` int32: the free pages,
    taken from the end.  Returns `(slots, lens_out, free_count_out)`: `slots` [total_new] int32
    holds `page * page_size + offset` of every new token, request after request (the tokens past
    `sum(new_lens)` and those of a request that was not served get -1); `block_table` gets the
    fresh pages in place.  Requests are served in order: one that does not fit its table row, the
    `total_new` slots or the pages left gets nothing and keeps its length, and so does every later
    one that needs a page once the pages have run out.  The outputs may be given, and `lens_out`
    and `free_count_out` may be `lens` and `free_count` themselves (a captured step updates them in
    place).
    """
    if not isinstance(lens, torch.Tensor) or not lens.is_cuda or lens.dim() != 1:
        raise ValueError('lens must be a CUDA tensor [B]')
    dev, B = lens.device, lens.shape[0]
    _vector('lens', lens, B, dev)
    _vector('new_lens', new_lens, B, dev)
    _table(block_table, dev, B)
    _vector('free_pages', free_pages, free_pages.numel(), dev)
    _vector('free_count', free_count, 1, dev)
    if total_new < 0:
        raise ValueError(f'total_new must not be negative, got {total_new}')
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    else:
        _vector('lens_out', lens_out, B, dev)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    else:
        _vector('free_count_out', free_count_out, 1, dev)
    if slots is None:
        slots = lens.new_empty((total_new,))
    else:
        _vector('slots', slots, total_new, dev)
    _lib.call('motif_b200_paged_reserve', lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(),
              block_table.stride(0), free_pages.data_ptr(), free_count.data_ptr(), lens_out.data_ptr(),
              free_count_out.data_ptr(), slots.data_ptr(), total_new, B, block_table.shape[1], free_pages.numel(),
              page_size, _lib.stream_ptr(dev))
    return slots, lens_out, free_count_out


def paged_release(done, lens, block_table, free_pages, free_count, page_size: int) -> None:
    """Return the pages of the requests with `done[b]` (bool [B]) to the free list, in place: their
    table entries become -1 and their lengths 0; pages go onto the end of `free_pages` request after
    request (those past its size are dropped)."""
    if not isinstance(lens, torch.Tensor) or not lens.is_cuda or lens.dim() != 1:
        raise ValueError('lens must be a CUDA tensor [B]')
    dev, B = lens.device, lens.shape[0]
    _vector('lens', lens, B, dev)
    _vector('done', done, B, dev, torch.bool)
    _table(block_table, dev, B)
    _vector('free_pages', free_pages, free_pages.numel(), dev)
    _vector('free_count', free_count, 1, dev)
    _lib.call('motif_b200_paged_release', done.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
              block_table.stride(0), free_pages.data_ptr(), free_count.data_ptr(), B, block_table.shape[1],
              free_pages.numel(), page_size, _lib.stream_ptr(dev))


def _rows16(t):
    """t with rows that the kernel can read as 16-byte vectors (a copy where they are not)."""
    *outer, last = t.stride()
    step = 16 // t.element_size()
    if last == 1 and t.data_ptr() % 16 == 0 and not any(s % step for s in outer):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _token_strides(t):
    """Element strides (batch, head, token) of [N, Hkv, D] or [B, Hkv, T, D]."""
    s = t.stride()
    return (0, s[1], s[0]) if t.dim() == 3 else s[:3]


def kv4_append(k, v, slots, pool, values: bool = False):
    """Quantise new keys and values to 4 bits and store them at their slots.

    `k` / `v`: [N, Hkv, D], or [B, Hkv, T, D] with N = B T tokens in (b, t) order; `slots` [N] int32
    from `paged_reserve` (tokens with a slot outside the pool are not stored; two tokens must not
    share one).  With `values`, returns `(k, v)` as the stored bits stand for them, in the inputs'
    shape and dtype: a prompt chunk that attends to these sees what later steps will see.
    """
    pages, kv, page_size, D = _pool_dims(pool)
    dev = pool.device
    for name, t in (('k', k), ('v', v)):
        if not isinstance(t, torch.Tensor) or t.device != dev:
            raise ValueError(f'{name} must live on {dev}')
    if k.dim() not in (3, 4) or k.shape != v.shape or k.shape[1] != kv or k.shape[-1] != D:
        raise ValueError(f'k / v must be [N, {kv}, {D}] or [B, {kv}, T, {D}], got {tuple(k.shape)}, {tuple(v.shape)}')
    if k.dtype != v.dtype:
        raise ValueError('k / v must share one dtype')
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError('the 4-bit cache is forward-only (no autograd)')
    B, T = (1, k.shape[0]) if k.dim() == 3 else (k.shape[0], k.shape[2])
    _vector('slots', slots, B * T, dev)
    dc = _lib.dtype_code(k.dtype)
    k, v = _rows16(k), _rows16(v)
    if not values:
        strides = _lib.i64_const(*_token_strides(k), *_token_strides(v), 0, 0, 0, 0, 0, 0)
        _lib.call('motif_b200_kv4_append', k.data_ptr(), v.data_ptr(), slots.data_ptr(), pool.data_ptr(), None, None,
                  strides, B, T, kv, D, pages, page_size, dc, _lib.stream_ptr(dev))
        return None
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    vo = torch.empty_like(ko)
    to = _token_strides(ko)
    strides = _lib.i64_const(*_token_strides(k), *_token_strides(v), *to, *to)
    _lib.call('motif_b200_kv4_append', k.data_ptr(), v.data_ptr(), slots.data_ptr(), pool.data_ptr(), ko.data_ptr(),
              vo.data_ptr(), strides, B, T, kv, D, pages, page_size, dc, _lib.stream_ptr(dev))
    return ko, vo


def kv4_gather(pool, block_table, lens, max_len: int, dtype=torch.bfloat16):
    """The cached keys and values of every request as two `[B, Hkv, max_len, D]` tensors of `dtype`,
    zeros at and past `lens[b]` (and where a table entry is no page of the pool)."""
    pages, kv, page_size, D = _pool_dims(pool)
    dev = pool.device
    _table(block_table, dev)
    B = block_table.shape[0]
    _vector('lens', lens, B, dev)
    if max_len < 0:
        raise ValueError(f'max_len must not be negative, got {max_len}')
    dc = _lib.dtype_code(dtype)
    k = torch.empty((B, kv, max_len, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _lib.call('motif_b200_kv4_gather', pool.data_ptr(), block_table.data_ptr(), block_table.stride(0), lens.data_ptr(),
              k.data_ptr(), v.data_ptr(), B, kv, max_len, D, pages, page_size, block_table.shape[1], dc,
              _lib.stream_ptr(dev))
    return k, v


def kv4_chord_attention(q, pool, block_table, lens, alpha, beta, mu, ssmax, q_lens: Optional[torch.Tensor] = None,
                        softmax_scale: Optional[float] = None, eps: float = 1e-5) -> torch.Tensor:
    """Chord attention of each request's newest tokens over its 4-bit cache
    (`apply_chord_attention`'s mathematics, `motif/ops/chord_attention.py:1557-1625`, with
    log_n = log(position + 1)).

    `q` [B, H, T, D] (any strides, last dim contiguous): token t of request b sits at position
    `lens[b] - T + t` (`lens[b] - q_lens[b] + t` with `q_lens` [B] int32, rows t >= q_lens[b] being
    padding) and sees the cached keys up to its own position, which must have been appended before.
    Rows that see no key (padding, positions below 0) are zeros; keys whose table entry is no page
    of the pool are left out.  Head h reads kv head h / (H / Hkv).  Returns [B, H, T, D] in q's dtype.
    """
    pages, kv, page_size, D = _pool_dims(pool)
    dev = pool.device
    if not isinstance(q, torch.Tensor) or q.device != dev:
        raise ValueError(f'q must live on {dev}')
    if q.dim() != 4 or q.shape[3] != D:
        raise ValueError(f'q must be [B, H, T, {D}], got {tuple(q.shape)}')
    B, H, T, _ = q.shape
    if H % kv:
        raise ValueError(f'num_heads {H} must be divisible by num_kv_heads {kv}')
    if q.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError('the 4-bit cache is forward-only (no autograd)')
    dc = _lib.dtype_code(q.dtype)
    _table(block_table, dev, B)
    _vector('lens', lens, B, dev)
    if q_lens is not None:
        _vector('q_lens', q_lens, B, dev)
    _vector('alpha', alpha, H, dev, torch.float32)
    _vector('beta', beta, H, dev, torch.float32)
    _vector('mu', mu, H, dev, torch.float32)
    _vector('ssmax', ssmax, H, dev, torch.float32)
    q = _rows16(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ws_bytes = _attention_workspace(dev.index, H, kv, T, D)
    ws = pool.new_empty((ws_bytes,))
    strides = _lib.i64_const(*q.stride()[:3], *out.stride()[:3])
    _lib.call('motif_b200_kv4_chord_attention', q.data_ptr(), pool.data_ptr(), block_table.data_ptr(),
              block_table.stride(0), lens.data_ptr(), _lib.ptr(q_lens), alpha.data_ptr(), beta.data_ptr(),
              mu.data_ptr(), ssmax.data_ptr(), out.data_ptr(), strides, B, H, kv, T, D, pages, page_size,
              block_table.shape[1], D ** -0.5 if softmax_scale is None else float(softmax_scale), float(eps),
              ws.data_ptr(), ws_bytes, dc, _lib.stream_ptr(dev))
    return out
