"""The paged 4-bit Chord cache's operators where they can go wrong: inputs at the edges of what the
calls take, each against the definition in 64 bits (or a plain loop).

Bars are those of `test_paged_gpu.py` unless a test derives its own.
"""

import threading
import time

import pytest
import torch

from motif_b200 import _lib, ops
from test_paged_gpu import attention_64, close, gen, params, random_cache

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ sums of 16-bit tensors
def attention_32(q, pool, table, lens, alpha, beta, mu, ssmax, scale=None):
    """Elementary operations in 32 bits, rounded once at the end."""
    most = int(lens.max())
    k, v = ops.kv4_gather(pool, table, lens, most, dtype=torch.float32)
    B, H, T, D = q.shape
    x = (q.float().view(B, k.shape[1], -1, D) @ k.transpose(-1, -2) * (scale or D ** -0.5)).view(B, H, T, most)
    pos = (lens[:, None] - T + torch.arange(T, device='cuda')).view(B, 1, T, 1)
    key = torch.arange(most, device='cuda')
    alpha, beta, mu, ssmax = (p.view(1, H, 1, 1) for p in (alpha, beta, mu, ssmax))
    x = (x - alpha * ((key - pos - mu).abs() + 1e-5) ** beta) * (ssmax * torch.log(pos + 1.0))
    w = x.masked_fill(key > pos, float('-inf')).softmax(-1)
    return (w.view(B, k.shape[1], -1, most) @ v).view(B, H, T, D).to(q.dtype)


@pytest.mark.parametrize('H,kv,D,T', [(12, 3, 64, 1), (12, 3, 64, 4), (8, 4, 128, 1), (8, 2, 128, 2), (12, 3, 32, 1),
                                      (8, 2, 32, 2)])
def test_sums_of_16_bit_tensors_keep_their_bits(H, kv, D, T):
    """An error e of a sum crosses a midpoint between two neighbours of the output's type, s apart, with
    probability e / s, so the outputs that are not the correctly rounded ones count the bits of the sums:
    sums of 21 bits give at most 8 times as many as sums of 24.  (fp16; bf16 differs in nothing but the
    last rounding, which sums of 24 bits of these few thousand outputs hardly ever get wrong.)"""
    lens = [4000, 3001, 2500, 3777] * 2
    pool, table, ln = random_cache(lens, kv, D, 64, 60 + D)
    g = gen(61)
    q = torch.randn(len(lens), H, T, D, device='cuda', generator=g).half()
    alpha, beta, mu, ssmax = (torch.rand(H, device='cuda', generator=g) for _ in range(4))
    p = 0.3 + 1.2 * alpha, 0.6 * beta, 3 * mu - 1, 0.3 + 0.6 * ssmax
    want = attention_64(q, pool, table, ln, *p).half()
    wrong = (ops.kv4_chord_attention(q, pool, table, ln, *p) != want).sum()
    assert wrong <= 8 * (attention_32(q, pool, table, ln, *p) != want).sum()
    # logits ten times as large: an error of the first product's sums grows with them
    scale = 10 * D ** -0.5
    want = attention_64(q, pool, table, ln, *p, scale=scale).half()
    wrong = (ops.kv4_chord_attention(q, pool, table, ln, *p, softmax_scale=scale) != want).sum()
    assert wrong <= 8 * (attention_32(q, pool, table, ln, *p, scale) != want).sum()


# ------------------------------------------------------------------ waits that run out
@pytest.mark.parametrize('H,kv,D,T', [(12, 3, 64, 1), (16, 1, 64, 3), (8, 2, 128, 2), (4, 4, 32, 1)])
def test_rows_of_a_failed_wait_are_nan_and_counted(H, kv, D, T):
    """A CTA whose copy wait runs out (here at once, in every third CTA) leaves NaN in the rows that
    needed it, the right values in all others, and is counted; the next call is as ever."""
    lens = [(91 * i) % 700 + 1 for i in range(90)] + [9000, 0, 2, 4001]
    pool, table, ln = random_cache(lens, kv, D, 64, 62)
    q = torch.randn(len(lens), H, T, D, device='cuda', generator=gen(63)).bfloat16()
    pr = params(H, 10)
    want = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    assert _lib.wait_timeouts() == 0 and not want.isnan().any()
    with _lib.forced(_lib.FORCE_KV4_WAIT_FAILS):
        got = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    ctas = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.wait_timeouts() == len(range(1, ctas, 3))
    lost = got.isnan()
    assert torch.equal(lost.any(-1), lost.all(-1))             # whole rows
    assert torch.equal(got[~lost], want[~lost])
    assert lost[90].all() and not lost[91].any()               # over many CTAs; without keys
    assert 0.2 < lost.double().mean() < 0.8
    assert torch.equal(ops.kv4_chord_attention(q, pool, table, ln, *pr), want) and _lib.wait_timeouts() == 0


# ------------------------------------------------------------------ values far larger than those of weight
def slots_of(table, lens, P):
    """Slot of every cached token, request after request."""
    out = []
    for b, n in enumerate(lens):
        pos = torch.arange(n, device='cuda')
        out.append(table[b, (pos // P).long()] * P + pos % P)
    return torch.cat(out).to(torch.int32)


LAYOUTS = [(2, 2, 64, 2), (8, 2, 64, 2), (16, 2, 64, 2), (4, 2, 128, 2), (8, 4, 32, 2)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,kv,D,T', LAYOUTS)
@pytest.mark.parametrize('exponent', [14, 30, 60])
def test_large_values_that_a_row_does_not_see(dtype, H, kv, D, T, exponent):
    """The newest token's values are 2^exponent times as large as the others: the rows before it do not
    see them, and keep the bar against their own largest output."""
    lens, P = [80, 200, 64, 3], 16
    pool, table, ln = random_cache(lens, kv, D, P, 19)
    newest = slots_of(table, lens, P)[torch.tensor(lens, device='cuda').cumsum(0) - 1].contiguous()
    g = gen(20)
    k, v = (torch.randn(4, kv, D, device='cuda', generator=g) for _ in range(2))
    ops.kv4_append(k, 2.0 ** exponent * v, newest, pool)
    q = torch.randn(4, H, T, D, device='cuda', generator=g).to(dtype)
    pr = params(H, 9)
    out, ref = ops.kv4_chord_attention(q, pool, table, ln, *pr), attention_64(q, pool, table, ln, *pr)
    for b in range(4):
        for t in range(T - 1):
            for h in range(H):
                close(out[b, h, t], ref[b, h, t], dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,kv,D,T', LAYOUTS)
@pytest.mark.parametrize('at', ['first', 'middle'])
def test_large_values_without_weight(dtype, H, kv, D, T, at):
    """One key per request has values 2^30 times as large and, by the decay, a weight of 2^-200 at most.
    Its neighbours (and their weights) change by steps of 2^-40 a key, so the reference moves on with
    every tile."""
    lens, P = [300, 200, 90, 131], 16
    pool, table, ln = random_cache(lens, kv, D, P, 19)
    starts = torch.tensor([0] + lens[:-1], device='cuda').cumsum(0)
    which = slots_of(table, lens, P)[starts + (0 if at == 'first' else 70)].contiguous()
    g = gen(21)
    k, v = (torch.randn(4, kv, D, device='cuda', generator=g) for _ in range(2))
    ops.kv4_append(k, 2.0 ** 30 * v, which, pool)
    q = torch.randn(4, H, T, D, device='cuda', generator=g).to(dtype)
    alpha, beta, mu, ssmax = (torch.full((H,), c, device='cuda') for c in (10.0, 1.0, 0.0, 0.7))
    out = ops.kv4_chord_attention(q, pool, table, ln, alpha, beta, mu, ssmax)
    ref = attention_64(q, pool, table, ln, alpha, beta, mu, ssmax)
    for b in range(4):
        for t in range(T):
            for h in range(H):
                close(out[b, h, t], ref[b, h, t], dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('H,kv,D,T', LAYOUTS)
def test_values_that_shrink_and_grow_along_the_cache(dtype, H, kv, D, T):
    """Values of 2^-60 to 2^60 in turn, tile by tile, under no decay and under one that leaves the last keys
    alone with a weight: every row keeps the bar against its own largest output."""
    lens, P = [640, 300], 16
    pool, table, ln = random_cache(lens, kv, D, P, 22)
    g = gen(23)
    n = sum(lens)
    size = 2.0 ** (60.0 * torch.tensor([1.0, -1.0, 0.0, 0.9, -0.3, 0.4], device='cuda'))
    where = torch.cat([torch.arange(x, device='cuda') for x in lens])
    v = torch.randn(n, kv, D, device='cuda', generator=g) * size[(where // 50) % 6].view(n, 1, 1)
    k = torch.randn(n, kv, D, device='cuda', generator=g)
    ops.kv4_append(k, v, slots_of(table, lens, P), pool)
    q = torch.randn(2, H, T, D, device='cuda', generator=g).to(dtype)
    for a in (0.0, 20.0):
        alpha, beta, mu, ssmax = (torch.full((H,), c, device='cuda') for c in (a, 1.0, 0.0, 0.5))
        out = ops.kv4_chord_attention(q, pool, table, ln, alpha, beta, mu, ssmax)
        ref = attention_64(q, pool, table, ln, alpha, beta, mu, ssmax)
        for b in range(2):
            for t in range(T):
                for h in range(H):
                    close(out[b, h, t], ref[b, h, t], dtype)


# ------------------------------------------------------------------ values that are no numbers
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,kv,D,T', [(2, 2, 64, 3), (8, 2, 64, 3), (16, 2, 64, 3), (4, 2, 128, 3), (8, 4, 32, 3)])
@pytest.mark.parametrize('what', [float('nan'), float('inf')])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(dtype, H, kv, D, T, what):
    """The newest token holds a NaN or an infinity in its first group of dims: NaN in that group's outputs of
    its own row, nothing in its other group's values, nothing in the rows before it."""
    lens, P = [80, 17, 64, 3], 16
    pool, table, ln = random_cache(lens, kv, D, P, 16)
    clean = pool.clone()
    newest = slots_of(table, lens, P)[torch.tensor(lens, device='cuda').cumsum(0) - 1].contiguous()
    k, v = (torch.randn(4, kv, D, device='cuda', generator=gen(17)) for _ in range(2))
    ops.kv4_append(k, v, newest, clean)
    v[..., 5] = what
    ops.kv4_append(k, v, newest, pool)
    q = torch.randn(4, H, T, D, device='cuda', generator=gen(18)).to(dtype)
    pr = params(H, 9)
    out, ref = ops.kv4_chord_attention(q, pool, table, ln, *pr), attention_64(q, clean, table, ln, *pr)
    first = min(D, 64)
    close(out[:, :, :T - 1], ref[:, :, :T - 1], dtype)
    assert out[:, :, T - 1, :first].isnan().all()
    if D > first:
        close(out[:, :, T - 1, first:], ref[:, :, T - 1, first:], dtype)
    # a key that is no number is NaN in the row that sees it, and in no other
    k[..., 5] = what
    ops.kv4_append(k, torch.ones_like(k), newest, pool)
    out = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    close(out[:, :, :T - 1], ref[:, :, :T - 1], dtype)
    assert out[:, :, T - 1].isnan().all()


# ------------------------------------------------------------------ the decay at distance 0
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('D', [32, 64, 128])
def test_decay_of_a_key_at_distance_0(dtype, D):
    """No eps and a whole mu: 0^beta is 0 however small beta is, and infinite for a negative one (its key
    then weighs nothing)."""
    H, kv, P = 8, 2, 16
    pool, table, ln = random_cache([300, 40, 2], kv, D, P, 14)
    q = torch.randn(3, H, 1, D, device='cuda', generator=gen(15)).to(dtype)
    beta = torch.tensor([0.01, 0.02, 0.05, 0.1, 0.01, 0.05, -0.05, -0.5], device='cuda')
    mu = torch.tensor([0.0, 0.0, 0.0, 0.0, -1.0, -3.0, 0.0, -1.0], device='cuda')
    alpha, ssmax = torch.full((H,), 1.5, device='cuda'), torch.full((H,), 0.7, device='cuda')
    out = ops.kv4_chord_attention(q, pool, table, ln, alpha, beta, mu, ssmax, eps=0.0)
    close(out, attention_64(q, pool, table, ln, alpha, beta, mu, ssmax, eps=0.0), dtype)


# ------------------------------------------------------------------ refusals
def test_pools_without_pages_heads_or_units_are_refused():
    pool, table, ln = random_cache([20, 3], 2, 64, 16, 30)
    q, p = torch.zeros(2, 4, 1, 64, device='cuda'), torch.zeros(4, device='cuda')
    x, slots = torch.zeros(3, 2, 64, device='cuda'), torch.zeros(3, dtype=torch.int32, device='cuda')
    for bad in (pool[:0], pool[:, :0], pool[:, :, :0]):
        with pytest.raises(ValueError, match='pool must be'):
            ops.kv4_chord_attention(q, bad, table, ln, p, p, p, p)
        with pytest.raises(ValueError, match='pool must be'):
            ops.kv4_append(x, x, slots, bad)
        with pytest.raises(ValueError, match='pool must be'):
            ops.kv4_gather(bad, table, ln, 20)


def test_gradients_are_refused_and_not_dropped():
    """Forward-only: an argument that asks for a gradient, or carries a forward-mode tangent, raises."""
    pool, table, ln = random_cache([20, 3], 2, 64, 16, 30)
    q, p = torch.zeros(2, 4, 1, 64, device='cuda'), torch.zeros(4, device='cuda')
    x, slots = torch.zeros(3, 2, 64, device='cuda'), torch.full((3,), -1, dtype=torch.int32, device='cuda')
    fwd = torch.autograd.forward_ad
    for i in range(5):
        a = [q, p, p, p, p]
        a[i] = a[i].clone().requires_grad_()
        with pytest.raises(NotImplementedError, match='forward-only'):
            ops.kv4_chord_attention(a[0], pool, table, ln, *a[1:])
        with torch.no_grad():
            assert not ops.kv4_chord_attention(a[0], pool, table, ln, *a[1:]).requires_grad
        with fwd.dual_level():
            a[i] = fwd.make_dual(a[i].detach(), torch.ones_like(a[i]))
            with pytest.raises(NotImplementedError, match='forward-only'):
                ops.kv4_chord_attention(a[0], pool, table, ln, *a[1:])
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for k, v in ((dual, x), (x, dual)):
            with pytest.raises(NotImplementedError, match='forward-only'):
                ops.kv4_append(k, v, slots, pool)


# ------------------------------------------------------------------ batches without requests
def test_a_batch_of_no_requests():
    i32 = dict(dtype=torch.int32, device='cuda')
    none, table = torch.empty(0, **i32), torch.empty((0, 4), **i32)
    free, count = torch.arange(5, **i32), torch.tensor([5], **i32)
    for total in (0, 3, 5000):
        slots, lens, left = ops.paged_reserve(none, none, table, free, count, 16, total)
        assert slots.tolist() == [-1] * total and lens.shape == (0,) and left.tolist() == [5]
        slots, lens, left = ops.paged_reserve(none, none, table, free, count, 16, total, lens_out=none,
                                              free_count_out=count)
        assert slots.tolist() == [-1] * total and count.tolist() == [5]
    ops.paged_release(torch.empty(0, dtype=torch.bool, device='cuda'), none, table, free, count, 16)
    assert count.tolist() == [5] and free.tolist() == list(range(5))


# ------------------------------------------------------------------ other threads
def test_other_python_threads_run_while_a_launch_waits():
    """The GPU is kept busy for about a second and the launch queue (some thousand launches) filled
    behind it: a call then waits in its launch, and meanwhile another Python thread goes on."""
    pool, table, ln = random_cache([20, 3], 2, 64, 16, 30)
    x = torch.randn(3, 2, 64, device='cuda', generator=gen(31))
    slots = torch.full((3,), -1, dtype=torch.int32, device='cuda')
    ops.kv4_append(x, x, slots, pool)
    torch.cuda.synchronize()
    longest, stop = [0.0], threading.Event()

    def watch():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            longest[0], last = max(longest[0], now - last), now

    thread = threading.Thread(target=watch)
    thread.start()
    try:
        torch.cuda._sleep(2_000_000_000)  # cycles of at most 1.965 GHz
        begin = time.perf_counter()
        for _ in range(6000):
            ops.kv4_append(x, x, slots, pool)
        waited = time.perf_counter() - begin
    finally:
        stop.set()
        thread.join()
        torch.cuda.synchronize()
    assert waited > 0.7, 'the launches did not fill the queue'
    assert longest[0] < 0.35


def test_reservations_into_their_own_inputs_are_refused():
    """lens_out may be lens, free_count_out free_count; anything else that overlaps would be read by one CTA
    after another has written it."""
    i32 = dict(dtype=torch.int32, device='cuda')
    both = torch.tensor([3, 4, 5, 1, 1, 1], **i32)
    lens, new = both[:3], both[3:]
    free, count = torch.arange(20, **i32), torch.tensor([20], **i32)
    table = torch.tensor([[15, -1], [16, -1], [17, -1]], **i32)

    def reserve(**kw):
        return ops.paged_reserve(lens, new, table, free, count, 16, 3, **kw)

    for kw in (dict(lens_out=new), dict(lens_out=both[1:4]), dict(lens_out=both[2:5]), dict(slots=lens), dict(slots=new),
               dict(slots=both[2:5]), dict(free_count_out=both[:1]), dict(free_count_out=both[5:])):
        with pytest.raises(ValueError, match='overlap'):
            reserve(**kw)
    assert both.tolist() == [3, 4, 5, 1, 1, 1] and count.tolist() == [20]
    slots, out, left = reserve(lens_out=lens, free_count_out=count)
    assert slots.tolist() == [15 * 16 + 3, 16 * 16 + 4, 17 * 16 + 5] and out.tolist() == [4, 5, 6] and left is count
