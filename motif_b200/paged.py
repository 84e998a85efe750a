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
exceeds the largest float) is stored as NaN, and reaches the rows that see its token only.  A centre
beyond bf16's largest number is infinite.  White noise comes back 9 % of its deviation off.
"""

from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ['kv4_pool', 'paged_reserve', 'paged_release', 'kv4_append', 'kv4_gather', 'kv4_chord_attention']

UNIT = 16  # tokens of one storage unit: page sizes are multiples of it
_UNIT_BYTES = {32: 640, 64: 1152, 128: 2304}  # motif_b200_kv4_unit_bytes


def check_head_dim(head_dim: int) -> None:
    if head_dim not in _UNIT_BYTES:
        raise NotImplementedError(f'head_dim must be 32, 64 or 128, got {head_dim}')


def check_page_size(page_size: int) -> None:
    if page_size < UNIT or page_size % UNIT or page_size > 1024:
        raise ValueError(f'page_size must be a multiple of {UNIT} up to 1024, got {page_size}')


def kv4_pool(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, device='cuda') -> torch.Tensor:
    """An empty pool `[num_pages, num_kv_heads, page_size / 16, unit bytes]` (uint8): its shape
    carries the page size and the head dim (32, 64 or 128) for the calls below."""
    check_head_dim(head_dim)
    check_page_size(page_size)
    if num_pages < 1 or num_kv_heads < 1:
        raise ValueError(f'num_pages and num_kv_heads must be positive, got {num_pages}, {num_kv_heads}')
    return torch.zeros((num_pages, num_kv_heads, page_size // UNIT, _UNIT_BYTES[head_dim]), dtype=torch.uint8,
                       device=device)


def _host():
    """The compiled entry points (checks, output allocation and the C ABI call in one step)."""
    global _module
    if _module is None:
        _lib.load()
        try:
            from . import _paged_host
        except ImportError as e:
            raise RuntimeError('motif_b200/_paged_host.so is missing or was built for another torch: build it with '
                               f'`python -m motif_b200.build` ({e})') from e
        _module = _paged_host
    return _module


_module = None


def _call(name, *args):
    """One call, counted and timed by a launch tracker like `_lib.call`'s."""
    tr = _lib._tracker
    if tr is None:
        return getattr(_module or _host(), name)(*args)
    ev = tr.start('motif_b200_' + name)
    out = getattr(_host(), name)(*args)
    tr.stop('motif_b200_' + name, ev)
    return out


def paged_reserve(lens, new_lens, block_table, free_pages, free_count, page_size: int, total_new: int,
                  lens_out: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None,
                  slots: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Reserve cache slots for `new_lens[b]` more tokens of every request; all on the device.

    `lens` / `new_lens` [B] int32: cached and new tokens; `block_table` [B, max_pages] int32, its
    first ceil(lens / page_size) columns in use; `free_pages[:free_count]` int32: the free pages,
    taken from the end.  Returns `(slots, lens_out, free_count_out)`: `slots` [total_new] int32
    holds `page * page_size + offset` of every new token, request after request (the tokens past
    `sum(new_lens)` and those of a request that was not served get -1; at most 2^31 - 2^20); `block_table` gets the
    fresh pages in place.  Requests are served in order: one that does not fit its table row, the
    `total_new` slots or the pages left gets nothing and keeps its length, and so does every later
    one that needs a page once the pages have run out.  The outputs may be given, and `lens_out`
    and `free_count_out` may be `lens` and `free_count` themselves (a captured step updates them in
    place), but overlap nothing else.
    """
    return _call('paged_reserve', lens, new_lens, block_table, free_pages, free_count, page_size, total_new, lens_out,
                 free_count_out, slots)


def paged_release(done, lens, block_table, free_pages, free_count, page_size: int) -> None:
    """Return the pages of the requests with `done[b]` (bool [B]) to the free list, in place: their
    table entries become -1 and their lengths 0; pages go onto the end of `free_pages` request after
    request (those past its size are dropped)."""
    _call('paged_release', done, lens, block_table, free_pages, free_count, page_size)


def kv4_append(k, v, slots, pool, values: bool = False):
    """Quantise new keys and values to 4 bits and store them at their slots.

    `k` / `v`: [N, Hkv, D], or [B, Hkv, T, D] with N = B T tokens in (b, t) order; `slots` [N] int32
    from `paged_reserve` (tokens with a slot outside the pool are not stored; two tokens must not
    share one).  With `values`, returns `(k, v)` as the stored bits stand for them, in the inputs'
    shape and dtype: a prompt chunk that attends to these sees what later steps will see.
    """
    return _call('kv4_append', k, v, slots, pool, values)


def kv4_gather(pool, block_table, lens, max_len: int, dtype=torch.bfloat16):
    """The cached keys and values of every request as two `[B, Hkv, max_len, D]` tensors of `dtype`,
    zeros at and past `lens[b]` (and where a table entry is no page of the pool)."""
    return _call('kv4_gather', pool, block_table, lens, max_len, dtype)


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
    Rows whose copies from the pool did not arrive in time (never expected) are NaN and counted in
    `_lib.wait_timeouts()`.
    """
    return _call('kv4_chord_attention', q, pool, block_table, lens, alpha, beta, mu, ssmax, q_lens, softmax_scale, eps)
