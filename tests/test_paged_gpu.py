"""The paged 4-bit Chord cache (`motif_b200.paged`) against plain implementations.

Slot reservation is compared with a sequential Python loop (whole numbers: equal).  Stored pairs and
codes are checked against their definition in 64 bits, read-back values are exact (one fp32 rounding
of an exact product and sum, then the output type's), and attention is compared with the formula in
64 bits over the values that the stored bits stand for.

Attention tolerance: logits up to 64 in magnitude carry up to eight fp32 roundings of 2^-24 each, an
error of 64 * 8 * 2^-24 = 3e-5 in the exponent and so in every weight; the result is then rounded
once to its type (2^-24, 2^-12, 2^-9 relative).
"""

import math

import pytest
import torch

from motif_b200 import ops
from motif_b200.paged import UNIT, _UNIT_BYTES

pytestmark = pytest.mark.gpu

_DIMS = {v: k for k, v in _UNIT_BYTES.items()}

ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LOGIT = 3e-5


# ------------------------------------------------------------------ plain implementations
def reserve_loop(lens, new, table, free, count, P, total):
    """One request after the other."""
    lens, new, free = lens.tolist(), new.tolist(), free.tolist()
    table = [r[:] for r in table.tolist()]
    slots, out, at, used, taken = [-1] * total, [], 0, 0, 0
    for b, (n, m) in enumerate(zip(lens, new)):
        have, want = -(-n // P), -(-(n + m) // P)
        possible = want <= len(table[b]) and at + m <= total
        need = want - have if possible else 0
        used += need
        ok = possible and (need == 0 or used <= count)
        if ok:
            for j in range(need):
                table[b][have + j] = free[count - 1 - (used - need + j)]
            taken += need
            for t in range(m):
                slots[at + t] = table[b][(n + t) // P] * P + (n + t) % P
        out.append(n + m if ok else n)
        at += m
    return slots, out, count - taken, table


def stored(pool):
    """(codes [pages, Hkv, P, D], scale, centre [pages, Hkv, P, groups]) of K and of V, in 64 bits."""
    pages, kv, units, nbytes = pool.shape
    D = _DIMS[nbytes]
    half, ng = D // 2, D // min(D, 64)
    found = []
    for c0, p0 in ((0, 2 * UNIT * half), (UNIT * half, 2 * UNIT * half + 4 * UNIT * ng)):
        byte = pool[..., c0:c0 + UNIT * half].reshape(pages, kv, units * UNIT, half)
        code = torch.stack([byte % 16, byte // 16], -1).reshape(pages, kv, units * UNIT, D)
        pair = pool[..., p0:p0 + 4 * UNIT * ng].contiguous().view(torch.bfloat16).reshape(pages, kv, units, ng, UNIT, 2)
        pair = pair.permute(0, 1, 2, 4, 3, 5).reshape(pages, kv, units * UNIT, ng, 2).double()
        found.append((code.double(), pair[..., 0], pair[..., 1]))
    return found


def values(code, scale, centre):
    g = code.shape[-1] // scale.shape[-1]
    s, m = scale.repeat_interleave(g, -1), centre.repeat_interleave(g, -1)
    return m + s * (code - 8)


def cached(pool, table, b, n):
    """K, V [Hkv, n, D] of request b in 64 bits."""
    P = pool.shape[2] * UNIT
    out = []
    for code, s, m in stored(pool[table[b, :-(-n // P)].long()] if n else pool[:1]):
        x = values(code, s, m)                       # [pages of b, Hkv, P, D]
        out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n])
    return out


def attention_64(q, pool, table, lens, alpha, beta, mu, ssmax, q_lens=None, scale=None, eps=1e-5, drop=None):
    """The definition, row by row; `drop` [B, keys] marks keys that are left out."""
    B, H, T, D = q.shape
    kv = pool.shape[1]
    q, alpha, beta, mu, ssmax = (x.double() for x in (q, alpha, beta, mu, ssmax))
    out = torch.zeros_like(q)
    for b in range(B):
        n = int(lens[b])
        k, v = cached(pool, table, b, n)
        k, v = (x.repeat_interleave(H // kv, 0) for x in (k, v))
        nq = T if q_lens is None else int(q_lens[b])
        for t in range(nq):
            pos = n - nq + t
            if pos < 0:
                continue
            j = torch.arange(pos + 1, device=q.device, dtype=torch.float64)
            bias = -alpha[:, None] * ((j - pos - mu[:, None]).abs() + eps) ** beta[:, None]
            x = torch.einsum('hd,hsd->hs', q[b, :, t], k[:, :pos + 1]) * (D ** -0.5 if scale is None else scale)
            x = (x + bias) * ssmax[:, None] * math.log(pos + 1)
            if drop is not None:
                x = x.masked_fill(drop[b, None, :pos + 1], float('-inf'))
                if bool(drop[b, :pos + 1].all()):
                    continue
            out[b, :, t] = torch.einsum('hs,hsd->hd', x.softmax(-1), v[:, :pos + 1])
    return out


def close(got, ref, dtype):
    err = (got.double() - ref).abs()
    bar = ROUND[dtype] * ref.abs() + LOGIT * ref.abs().max()
    assert got.dtype == dtype and bool((err <= bar).all()), (err - bar).max().item()


# ------------------------------------------------------------------ inputs
def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def random_cache(lens, kv, D, P, seed, fill=0xff):
    """A pool filled through kv4_append; every byte outside the requests' tokens is `fill` (a scale of
    0xffff is a NaN: an unused token that is read shows)."""
    g = gen(seed)
    counts = [-(-n // P) for n in lens]
    pages = sum(counts) + 3
    pool = ops.kv4_pool(pages, kv, D, P)
    pool.fill_(fill)
    order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(counts)) + 1), -1, dtype=torch.int32, device='cuda')
    at, slots = 0, []
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
        pos = torch.arange(lens[b], device='cuda')
        slots.append(table[b, (pos // P).long()] * P + pos % P)
    slots = torch.cat(slots).to(torch.int32)
    n = slots.numel()
    k = torch.randn(n, kv, D, device='cuda', generator=g)
    v = torch.randn(n, kv, D, device='cuda', generator=g) + 0.3
    ops.kv4_append(k, v, slots, pool)
    return pool, table, torch.tensor(lens, dtype=torch.int32, device='cuda')


def params(H, seed):
    g = gen(seed)
    r = [torch.rand(H, device='cuda', generator=g) for _ in range(4)]
    p = [0.2 + r[0], 0.8 * r[1], 3 * r[2] - 1, 0.3 + 0.7 * r[3]]
    p[3][0] = -p[3][0]  # a negative logit scale
    return p


# ------------------------------------------------------------------ reservation
def check_reserve(lens, new, table, free, count, P, total):
    ref = reserve_loop(lens, new, table, free, count, P, total)
    c = torch.tensor([count], dtype=torch.int32).cuda()
    t, ln, f = table.cuda(), lens.cuda(), free.cuda()
    slots, out, left = ops.paged_reserve(ln, new.cuda(), t, f, c, P, total)
    assert slots.tolist() == ref[0] and out.tolist() == ref[1] and left.tolist() == [ref[2]] and t.tolist() == ref[3]
    assert ln.tolist() == lens.tolist() and c.tolist() == [count] and f.tolist() == free.tolist()
    # in place, on another stream
    t = table.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slots, out, left = ops.paged_reserve(ln, new.cuda(), t, f, c, P, total, lens_out=ln, free_count_out=c)
    side.synchronize()
    assert out is ln and left is c
    assert slots.tolist() == ref[0] and ln.tolist() == ref[1] and c.tolist() == [ref[2]] and t.tolist() == ref[3]


def reserve_state(B, P, most, new_most, seed, spare=0, columns=None):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, most + 1, (B,), generator=g).to(torch.int32)
    new = torch.randint(0, new_most + 1, (B,), generator=g).to(torch.int32)
    held = [-(-n // P) for n in lens.tolist()]
    want = [-(-n // P) for n in (lens + new).tolist()]
    columns = columns or max(1, max(want))
    pages = sum(want) + 5
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((B, columns), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(held):
        table[b, :c] = order[at:at + min(c, columns)]
        at += c
    free = torch.zeros(pages, dtype=torch.int32)
    free[:pages - at] = order[at:]
    return lens, new, table, free, pages - at + spare


@pytest.mark.parametrize('B,P,most,new_most', [(1, 16, 0, 1), (3, 64, 100, 1), (64, 64, 900, 1), (33, 128, 700, 300),
                                               (517, 16, 90, 40), (1025, 32, 60, 3), (2100, 16, 20, 9), (5, 48, 0, 0)])
def test_reserve_matches_loop(B, P, most, new_most):
    lens, new, table, free, count = reserve_state(B, P, most, new_most, B + P)
    total = int(new.sum())
    check_reserve(lens, new, table, free, count, P, total)
    check_reserve(lens, new, table, free, count, P, total + 7)  # room left over: -1


@pytest.mark.parametrize('B', [9, 1500])
def test_reserve_when_pages_tables_or_slots_run_out(B):
    lens, new, table, free, count = reserve_state(B, 16, 70, 50, B)
    total = int(new.sum())
    check_reserve(lens, new, table, free, count // 3, 16, total)
    check_reserve(lens, new, table, free, 0, 16, total)
    check_reserve(lens, new, table, free, count, 16, total // 2)
    check_reserve(lens, new, table, free, count, 16, 0)
    # a table too narrow for some requests
    wide = table.shape[1]
    narrow = table[:, :wide - 2].contiguous()
    check_reserve(torch.minimum(lens, torch.tensor(16 * (wide - 2), dtype=torch.int32)), new, narrow, free, count, 16,
                  total)


def test_reserve_with_strided_table_and_long_requests():
    P = 64
    lens = torch.tensor([0, 8191, 130000], dtype=torch.int32)
    new = torch.tensor([70000, 1, 64], dtype=torch.int32)
    columns = 2040
    want = [-(-int(n) // P) for n in lens + new]
    order = torch.randperm(4000, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((3, columns), -1, dtype=torch.int32)
    at = 0
    for b in range(3):
        c = -(-int(lens[b]) // P)
        table[b, :c] = order[at:at + c]
        at += c
    free = order[at:].contiguous()
    ref = reserve_loop(lens, new, table, free, free.numel(), P, 70065)
    wide = torch.zeros(3, columns + 9, dtype=torch.int32).cuda()
    view = wide[:, :columns]
    view.copy_(table)
    slots, out, left = ops.paged_reserve(lens.cuda(), new.cuda(), view, free.cuda(),
                                         torch.tensor([free.numel()], dtype=torch.int32).cuda(), P, 70065)
    assert slots.tolist() == ref[0] and out.tolist() == ref[1] and left.tolist() == [ref[2]]
    assert view.tolist() == ref[3] and not wide[:, columns:].any() and sum(want) <= 4000


@pytest.mark.parametrize('B', [1, 40, 1300])
def test_release_returns_every_page(B):
    P = 32
    g = torch.Generator().manual_seed(B)
    new = torch.randint(0, 200, (B,), generator=g).to(torch.int32).cuda()
    lens = torch.zeros(B, dtype=torch.int32).cuda()
    pages = int(((new + P - 1) // P).sum()) + 2
    free = torch.arange(pages, dtype=torch.int32).cuda()
    count = torch.tensor([pages], dtype=torch.int32).cuda()
    table = torch.full((B, 8), -1, dtype=torch.int32).cuda()
    slots, lens, count = ops.paged_reserve(lens, new, table, free, count, P, int(new.sum()), lens_out=lens,
                                           free_count_out=count)
    assert (slots >= 0).all() and slots.unique().numel() == slots.numel() and lens.tolist() == new.tolist()
    left, before, held = int(count), table.tolist(), lens.tolist()
    done = (torch.rand(B, generator=g) < 0.5).cuda()
    ops.paged_release(done, lens, table, free, count, P)
    expect = free[:left].tolist()
    for b in range(B):
        c = -(-held[b] // P)
        if done[b]:
            expect += before[b][:c]
            assert table[b].tolist() == [-1] * 8 and int(lens[b]) == 0
        else:
            assert table[b].tolist() == before[b] and int(lens[b]) == held[b]
    assert int(count) == len(expect) and free[:len(expect)].tolist() == expect
    ops.paged_release(~done, lens, table, free, count, P)
    assert int(count) == pages and sorted(free.tolist()) == list(range(pages)) and not lens.any()


# ------------------------------------------------------------------ append / gather
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('N,kv,D,P', [(1, 1, 64, 64), (37, 3, 64, 16), (130, 2, 32, 128), (65, 8, 128, 48),
                                      (1000, 3, 64, 64)])
def test_append_stores_the_nearest_codes(dtype, N, kv, D, P):
    g = gen(N * D)
    k = (torch.randn(N, kv, D, device='cuda', generator=g) * torch.rand(N, kv, 1, device='cuda', generator=g) * 4)
    v = torch.randn(N, kv, D, device='cuda', generator=g) * 0.01 + torch.randn(N, kv, 1, device='cuda', generator=g)
    k[0, 0] = 1.75                       # a constant row
    k, v = k.to(dtype), v.to(dtype)
    pages = -(-N // P) + 2
    slots = torch.randperm(pages * P, device='cuda', generator=g)[:N].to(torch.int32)
    pool = ops.kv4_pool(pages, kv, D, P)
    assert ops.kv4_append(k, v, slots, pool) is None
    again = ops.kv4_pool(pages, kv, D, P)
    ko, vo = ops.kv4_append(k, v, slots, again, values=True)
    assert torch.equal(pool, again)
    page, off = slots.long() // P, slots.long() % P
    for x, back, (code, s, m) in zip((k, v), (ko, vo), stored(pool)):
        code, s, m = (t[page, :, off] for t in (code, s, m))     # [N, Hkv, ...]
        y = x.double().view(N, kv, -1, min(D, 64))
        lo, hi = y.amin(-1), y.amax(-1)
        # the quotient's fp32 rounding and bf16's (2^-9 relative)
        assert bool(((s - (hi - lo) / 15).abs() <= 2.0 ** -8 * s).all())
        assert bool(((m - (lo + 8 * s)).abs() <= 2.0 ** -8 * (lo.abs() + 8 * s)).all())
        ratio = torch.where(s[..., None] > 0, (y - m[..., None]) / s[..., None], torch.zeros_like(y))
        want = ratio.round().clamp(-8, 7) + 8
        got = code.view(N, kv, -1, min(D, 64))
        # a quotient is rounded to fp32 (and its dividend may be): near a half either neighbour is right
        tie = ((ratio - ratio.floor()) - 0.5).abs() < 4e-6 * ratio.abs().clamp_min(1.0)
        assert bool(((got == want) | (tie & ((got - want).abs() <= 1))).all())
        exact = values(code, s, m)
        assert torch.equal(back, exact.float().to(dtype)) and back.shape == x.shape


def test_append_ties_go_to_the_even_code():
    x = torch.tensor([-8.0, 7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5] + [0.0] * 24, device='cuda').view(1, 1, 32)
    pool = ops.kv4_pool(1, 1, 32, 16)
    ko, _ = ops.kv4_append(x, x, torch.zeros(1, dtype=torch.int32, device='cuda'), pool, values=True)
    (code, s, m), _ = stored(pool)
    assert s[0, 0, 0, 0] == 1.0 and m[0, 0, 0, 0] == 0.0
    assert ko[0, 0, :8].tolist() == [-8.0, 7.0, 0.0, 2.0, 2.0, 0.0, -2.0, -2.0]


def test_append_non_finite_and_extreme_groups():
    pool = ops.kv4_pool(1, 1, 128, 16)
    x = torch.randn(7, 1, 128, device='cuda')
    x[0, 0, 3] = float('nan')
    x[1, 0, 70] = float('inf')
    x[2, 0, 127] = float('-inf')
    x[3, 0, :64] = 1e30 * x[3, 0, :64]
    x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38            # the range is no float
    x[5, 0, :64] = 0.0
    x[6, 0, :64] = 1e-40
    slots = torch.arange(7, dtype=torch.int32, device='cuda')
    ko, vo = ops.kv4_append(x, x, slots, pool, values=True)
    assert torch.equal(ko.isnan(), vo.isnan())
    nan = ko.isnan().view(7, 2, 64)
    bad = [(0, 0), (1, 1), (2, 1), (4, 0)]
    for n in range(7):
        for grp in range(2):
            assert bool(nan[n, grp].all()) == ((n, grp) in bad) and bool(nan[n, grp].any()) == ((n, grp) in bad)
    assert bool((ko[5, 0, :64] == 0).all())
    span = x[3, 0, :64].max() - x[3, 0, :64].min()
    assert bool(((ko[3, 0, :64] - x[3, 0, :64]).abs() <= span / 15).all())
    # below bf16's normal numbers: half of its smallest step, 2^-133
    assert bool((ko[6, 0, :64].double() - x[6, 0, :64].double()).abs().max() <= 2.0 ** -134)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_append_layouts_strides_and_skipped_slots(dtype):
    g = gen(5)
    B, kv, T, D, P = 3, 2, 17, 64, 32
    base = torch.randn(B, T, 3, kv, D, device='cuda', generator=g).to(dtype)
    k, v = base[:, :, 0].transpose(1, 2), base[:, :, 2].transpose(1, 2)          # [B, kv, T, D] views
    pages = 4
    slots = torch.randperm(pages * P, device='cuda', generator=g)[:B * T].to(torch.int32)
    slots[4], slots[9] = -1, pages * P + 3
    pool, flat = ops.kv4_pool(pages, kv, D, P), ops.kv4_pool(pages, kv, D, P)
    ko, vo = ops.kv4_append(k, v, slots, pool, values=True)
    fk, fv = ops.kv4_append(base[:, :, 0].reshape(B * T, kv, D).contiguous(),
                            base[:, :, 2].reshape(B * T, kv, D).contiguous(), slots, flat, values=True)
    assert torch.equal(pool, flat)
    assert torch.equal(ko, fk.view(B, T, kv, D).transpose(1, 2)) and torch.equal(vo, fv.view(B, T, kv, D).transpose(1, 2))
    # rows that do not start on 16 bytes are copied first
    odd = torch.randn(B * T * kv * D + 1, device='cuda', generator=g).to(dtype)[1:].view(B * T, kv, D)
    p1, p2 = ops.kv4_pool(pages, kv, D, P), ops.kv4_pool(pages, kv, D, P)
    ops.kv4_append(odd, odd, slots, p1)
    ops.kv4_append(odd.clone(), odd.clone(), slots, p2)
    assert torch.equal(p1, p2) and p1.any()
    # nothing to do
    empty = torch.empty(0, kv, D, device='cuda', dtype=dtype)
    a, b = ops.kv4_append(empty, empty, slots[:0].contiguous(), p2, values=True)
    assert a.shape == (0, kv, D) and torch.equal(p1, p2)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('N,kv,D,P', [(10007, 4, 32, 64), (5001, 3, 64, 48), (1027, 8, 128, 16)])
def test_append_of_many_tokens_equals_small_calls(dtype, N, kv, D, P):
    g = gen(N + D)
    base = torch.randn(N, 2, kv, D, device='cuda', generator=g) * torch.rand(N, 2, kv, 1, device='cuda', generator=g)
    base = base + torch.randint(-3, 4, (N, 2, kv, 1), device='cuda', generator=g)
    base[5, 0, 0, D - 1], base[N - 1, 1, kv - 1, 8], base[7, 0, 0, 0] = float('nan'), float('inf'), float('-inf')
    base[11, 0, 0], base[12, 1, 0] = 1e-6 * base[11, 0, 0], 0.0
    base = base.to(dtype)
    k, v = base[:, 0], base[:, 1]
    pages = -(-N // P)
    slots = torch.randperm(pages * P, device='cuda', generator=g)[:N].to(torch.int32)
    slots[3], slots[N - 2] = -1, pages * P
    pool, parts = ops.kv4_pool(pages, kv, D, P), ops.kv4_pool(pages, kv, D, P)
    ko, vo = ops.kv4_append(k, v, slots, pool, values=True)
    for i in range(0, N, 128):
        pk, pv = ops.kv4_append(k[i:i + 128], v[i:i + 128], slots[i:i + 128].contiguous(), parts, values=True)
        assert torch.equal(ko[i:i + 128].isnan(), pk.isnan()) and torch.equal(vo[i:i + 128].isnan(), pv.isnan())
        assert torch.equal(ko[i:i + 128].nan_to_num(), pk.nan_to_num())
        assert torch.equal(vo[i:i + 128].nan_to_num(), pv.nan_to_num())
    assert torch.equal(pool, parts)
    # [1, Hkv, N, D] views whose batch stride needs 64 bits (it is never taken a step of)
    far = [x.transpose(0, 1).as_strided((1, kv, N, D), (2 ** 33, D, 2 * kv * D, 1), x.storage_offset()) for x in (k, v)]
    again = ops.kv4_pool(pages, kv, D, P)
    ops.kv4_append(*far, slots, again)
    assert torch.equal(pool, again)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('kv,D,P', [(1, 32, 16), (3, 64, 64), (2, 128, 48)])
def test_gather_is_exact(dtype, kv, D, P):
    lens = [0, 1, 47, 48, 49, 200]
    pool, table, ln = random_cache(lens, kv, D, P, D + P)
    for most in (200, 130, 1, 260):
        k, v = ops.kv4_gather(pool, table, ln, most, dtype=dtype)
        for b, n in enumerate(lens):
            n = min(n, most)
            rk, rv = cached(pool, table, b, n)
            assert torch.equal(k[b, :, :n], rk.float().to(dtype)) and torch.equal(v[b, :, :n], rv.float().to(dtype))
            assert not k[b, :, n:].any() and not v[b, :, n:].any()
    table[5, 1] = pool.shape[0]          # no page of the pool: zeros there
    k, v = ops.kv4_gather(pool, table, ln, 200, dtype=dtype)
    rk, _ = cached(pool, table.clamp(0, pool.shape[0] - 1), 5, 200)
    assert not k[5, :, P:2 * P].any() and not v[5, :, P:2 * P].any()
    assert torch.equal(k[5, :, 2 * P:], rk[:, 2 * P:].float().to(dtype))
    assert ops.kv4_gather(pool, table, ln, 0, dtype=dtype)[0].shape == (6, kv, 0, D)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('kv,D,P', [(4, 32, 16), (3, 64, 48), (8, 128, 64)])
def test_gather_of_many_tokens_equals_small_calls(dtype, kv, D, P):
    lens = [3001, 0, 2600, 1, 1777, 3000, 2999, 16]
    pool, table, ln = random_cache(lens, kv, D, P, D)
    table[2, 5] = -1
    step = 10 * P
    k, v = ops.kv4_gather(pool, table, ln, 3001, dtype=dtype)
    for b in range(len(lens)):
        for i in range(0, 3001, step):
            row, left = table[b:b + 1, i // P:], (ln[b:b + 1] - i).clamp_min(0)
            if row.shape[1] == 0:
                continue
            sk, sv = ops.kv4_gather(pool, row, left, min(step, 3001 - i), dtype=dtype)
            assert torch.equal(k[b, :, i:i + step], sk[0]) and torch.equal(v[b, :, i:i + step], sv[0])
    assert not k[2, :, 5 * P:6 * P].any() and k[2, :, 6 * P:2600].any() and not k[2, :, 2600:].any()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,kv,D,P,T', [(12, 3, 64, 64, 1), (4, 4, 64, 16, 1), (6, 2, 32, 32, 3), (8, 1, 128, 128, 1),
                                        (10, 2, 64, 48, 2), (16, 4, 128, 32, 4), (3, 3, 32, 16, 5), (16, 1, 64, 64, 7),
                                        (2, 2, 64, 64, 33)])
def test_attention_matches_64_bits(dtype, H, kv, D, P, T):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 129, 700]
    pool, table, ln = random_cache(lens, kv, D, P, H * D + P)
    q = torch.randn(len(lens), H, T, D, device='cuda', generator=gen(T)).to(dtype)
    pr = params(H, H)
    out = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    close(out, attention_64(q, pool, table, ln, *pr), dtype)
    assert not out[8].any()
    assert torch.equal(out, ops.kv4_chord_attention(q, pool, table, ln, *pr))


@pytest.mark.parametrize('dtype,H,kv,D', [(torch.bfloat16, 12, 3, 64), (torch.float32, 4, 2, 32),
                                          (torch.float16, 8, 2, 128)])
def test_attention_long_and_many_requests(dtype, H, kv, D):
    lens = [20011]
    pool, table, ln = random_cache(lens, kv, D, 64, 3)
    q = torch.randn(1, H, 1, D, device='cuda', generator=gen(1)).to(dtype)
    pr = params(H, 1)
    close(ops.kv4_chord_attention(q, pool, table, ln, *pr), attention_64(q, pool, table, ln, *pr), dtype)
    lens = [(37 * i) % 301 for i in range(300)]
    pool, table, ln = random_cache(lens, kv, D, 16, 4)
    q = torch.randn(300, H, 1, D, device='cuda', generator=gen(2)).to(dtype)
    close(ops.kv4_chord_attention(q, pool, table, ln, *pr), attention_64(q, pool, table, ln, *pr), dtype)


def test_attention_query_lengths_scale_eps_and_strides():
    H, kv, D, P, T = 12, 3, 64, 32, 4
    lens = [300, 3, 1, 0, 64, 65]
    pool, table, ln = random_cache(lens, kv, D, P, 9)
    base = torch.randn(len(lens), T, H, D + 8, device='cuda', generator=gen(3)).bfloat16()
    q = base[..., 3:3 + D].transpose(1, 2)            # token-major rows at odd offsets
    ql = torch.tensor([4, 1, 3, 2, 0, 2], dtype=torch.int32, device='cuda')
    pr = params(H, 2)
    out = ops.kv4_chord_attention(q, pool, table, ln, *pr, q_lens=ql, softmax_scale=0.2, eps=1e-3)
    ref = attention_64(q, pool, table, ln, *pr, q_lens=ql, scale=0.2, eps=1e-3)
    close(out, ref, torch.bfloat16)
    for b in range(len(lens)):
        assert not out[b, :, int(ql[b]):].any()
    assert not out[2, :, :2].any() and not out[3].any()    # positions below 0
    # transposed storage of q (last dim not contiguous)
    qt = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(out, ops.kv4_chord_attention(qt, pool, table, ln, *pr, q_lens=ql, softmax_scale=0.2, eps=1e-3))
    assert ops.kv4_chord_attention(q[:, :, :0], pool, table, ln, *pr).shape == (len(lens), H, 0, D)
    assert ops.kv4_chord_attention(q[:0], pool, table[:0], ln[:0], *pr).shape == (0, H, T, D)


def test_attention_leaves_out_pages_that_are_none():
    H, kv, D, P = 8, 2, 64, 32
    lens = [200, 90, 32]
    pool, table, ln = random_cache(lens, kv, D, P, 11, fill=0)
    good = table.clone()
    drop = torch.zeros(3, 200, dtype=torch.bool, device='cuda')
    table[0, 2], table[1, 0], table[2, 0] = -1, pool.shape[0], -7
    drop[0, 64:96], drop[1, :32], drop[2, :32] = True, True, True
    q = torch.randn(3, H, 1, D, device='cuda', generator=gen(4)).bfloat16()
    pr = params(H, 3)
    out = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    close(out, attention_64(q, pool, good, ln, *pr, drop=drop), torch.bfloat16)
    assert not out[2].any()
    # lengths past the table's columns read what the table holds; negative ones nothing
    ln2 = torch.tensor([10 ** 9, -5, 32], dtype=torch.int32, device='cuda')
    out = ops.kv4_chord_attention(q, pool, good, ln2, *pr)
    assert not out[1].any() and not out[0].isnan().any()


def test_attention_of_large_and_tiny_values():
    """Keys and values far from 1 (a range of 2^60), and queries that scale against them."""
    H, kv, D, P = 4, 2, 64, 16
    pool, table, ln = random_cache([100, 33], kv, D, P, 12)
    g = gen(6)
    n = 133
    slots = torch.cat([table[b, (torch.arange(x, device='cuda') // P).long()] * P + torch.arange(x, device='cuda') % P
                       for b, x in ((0, 100), (1, 33))]).to(torch.int32)
    big = 2.0 ** (40 * torch.rand(n, kv, 1, device='cuda', generator=g) - 20)
    k = torch.randn(n, kv, D, device='cuda', generator=g) * 1e-12
    v = torch.randn(n, kv, D, device='cuda', generator=g) * big
    ops.kv4_append(k, v, slots, pool)
    q = torch.randn(2, H, 1, D, device='cuda', generator=g) * 1e12
    pr = params(H, 4)
    for dtype in (torch.float32, torch.bfloat16):
        close(ops.kv4_chord_attention(q.to(dtype), pool, table, ln, *pr),
              attention_64(q.to(dtype), pool, table, ln, *pr), dtype)
    zero = torch.zeros_like(q)
    close(ops.kv4_chord_attention(zero, pool, table, ln, *pr), attention_64(zero, pool, table, ln, *pr),
          torch.float32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_attention_decay_at_its_edges(dtype):
    """No decay (beta = 0: x^0 is 1 at x = 0 too), eps = 0 at a key that lies at mu, a steep decay whose
    far keys weigh nothing, and a negative exponent."""
    H, kv, D, P = 8, 2, 32, 16
    pool, table, ln = random_cache([300, 40, 1], kv, D, P, 13)
    q = torch.randn(3, H, 1, D, device='cuda', generator=gen(7)).to(dtype)
    alpha = torch.tensor([1.0, 0.5, 1.0, 2.0, 0.3, 40.0, 0.5, 0.0], device='cuda')
    beta = torch.tensor([0.0, 0.7, 1.0, 0.0, 2.5, 3.0, -0.5, 1.0], device='cuda')
    mu = torch.tensor([0.0, -3.0, 0.0, -5.0, -1.0, 0.0, 0.5, 0.0], device='cuda')
    ssmax = torch.full((H,), 0.7, device='cuda')
    for eps in (0.0, 1e-5):
        out = ops.kv4_chord_attention(q, pool, table, ln, alpha, beta, mu, ssmax, eps=eps)
        close(out, attention_64(q, pool, table, ln, alpha, beta, mu, ssmax, eps=eps), dtype)


def test_offsets_past_32_bits():
    """Pages whose bytes lie past 4 GiB."""
    kv, D, P = 4, 128, 128
    page = kv * (P // UNIT) * 2304
    pages = (5 << 30) // page
    pool = torch.empty((pages, kv, P // UNIT, 2304), dtype=torch.uint8, device='cuda')
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device='cuda')
    n = 300
    pos = torch.arange(n, device='cuda')
    slots = (table[0, pos // P] * P + pos % P).to(torch.int32)
    k = torch.randn(n, kv, D, device='cuda', generator=gen(8)).bfloat16()
    v = torch.randn(n, kv, D, device='cuda', generator=gen(9)).bfloat16()
    ko, vo = ops.kv4_append(k, v, slots, pool, values=True)
    ln = torch.tensor([n], dtype=torch.int32, device='cuda')
    gk, gv = ops.kv4_gather(pool, table, ln, n)
    assert torch.equal(gk[0].transpose(0, 1), ko) and torch.equal(gv[0].transpose(0, 1), vo)
    q = torch.randn(1, 8, 1, D, device='cuda', generator=gen(10)).bfloat16()
    pr = params(8, 5)
    close(ops.kv4_chord_attention(q, pool, table, ln, *pr), attention_64(q, pool, table, ln, *pr), torch.bfloat16)


def test_step_in_a_cuda_graph_follows_the_lengths():
    """Reserve, append and attention captured once and replayed: lengths advance on the device."""
    B, H, kv, D, P, steps = 3, 8, 2, 64, 16, 40
    g = gen(20)
    ks, vs, qs = (torch.randn(steps, B, h, 1, D, device='cuda', generator=g).bfloat16() for h in (kv, kv, H))
    pr = params(H, 6)
    pool = ops.kv4_pool(16, kv, D, P)
    free = torch.arange(16, dtype=torch.int32, device='cuda')
    count = torch.tensor([16], dtype=torch.int32, device='cuda')
    table = torch.full((B, 4), -1, dtype=torch.int32, device='cuda')
    lens = torch.tensor([0, 0, 0], dtype=torch.int32, device='cuda')
    new = torch.tensor([1, 1, 0], dtype=torch.int32, device='cuda')
    slots = torch.empty(B, dtype=torch.int32, device='cuda')
    k, v, q = torch.empty_like(ks[0]), torch.empty_like(vs[0]), torch.empty_like(qs[0])
    order = torch.tensor([0, 1, 2], device='cuda')

    def step():
        ops.paged_reserve(lens, new, table, free, count, P, B, lens_out=lens, free_count_out=count, slots=slots)
        ops.kv4_append(k[order], v[order], slots, pool)
        return ops.kv4_chord_attention(q, pool, table, lens, *pr)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lens.zero_()
    count.fill_(16)
    table.fill_(-1)
    pool.zero_()
    free.copy_(torch.arange(16))
    for i in range(steps):
        k.copy_(ks[i])
        v.copy_(vs[i])
        q.copy_(qs[i])
        graph.replay()
    torch.cuda.synchronize()
    assert lens.tolist() == [steps, steps, 0] and int(count) == 16 - 2 * -(-steps // P)
    close(out, attention_64(qs[-1], pool, table, lens, *pr), torch.bfloat16)
    gk, _ = ops.kv4_gather(pool, table, lens, steps)
    fake = ops.kv4_pool(8, kv, D, P)
    ko, _ = ops.kv4_append(ks[:, 0, :, 0].contiguous(), vs[:, 0, :, 0].contiguous(),
                           torch.arange(steps, dtype=torch.int32, device='cuda'), fake, values=True)
    assert torch.equal(gk[0].transpose(0, 1), ko)


def test_refusals_on_device_tensors():
    """Shapes, types and places that the calls refuse before anything is launched."""
    pool, table, ln = random_cache([20, 3], 2, 64, 16, 30)
    q, p = torch.zeros(2, 4, 1, 64, device='cuda'), torch.zeros(4, device='cuda')
    x, slots = torch.zeros(3, 2, 64, device='cuda'), torch.zeros(3, dtype=torch.int32, device='cuda')
    free, one = torch.zeros(4, dtype=torch.int32, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')

    def bad(match, call, *a, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            call(*a, **kw)

    att = ops.kv4_chord_attention
    bad('q must be', att, q[..., :32], pool, table, ln, p, p, p, p)
    bad('divisible', att, q[:, :3], pool, table, ln, p[:3], p[:3], p[:3], p[:3])
    bad('alpha must be', att, q, pool, table, ln, p.double(), p, p, p)
    bad('mu must be', att, q, pool, table, ln, p, p, p[:3], p)
    bad('beta must live', att, q, pool, table, ln, p, p.cpu(), p, p)
    bad('lens must be', att, q, pool, table, ln.long(), p, p, p, p)
    bad('q_lens must be', att, q, pool, table, ln, p, p, p, p, q_lens=ln[:1])
    bad('block_table', att, q, pool, table[:1], ln, p, p, p, p)
    bad('block_table', att, q, pool, table.t(), ln, p, p, p, p)
    bad('dtype', att, q.double(), pool, table, ln, p, p, p, p)
    bad('pool must be', att, q, pool[..., :100], table, ln, p, p, p, p)
    bad('forward-only', att, q.clone().requires_grad_(), pool, table, ln, p, p, p, p, error=NotImplementedError)
    bad('k / v must be', ops.kv4_append, x[:, :1], x[:, :1], slots, pool)
    bad('k / v must be', ops.kv4_append, x, x[:2], slots, pool)
    bad('share one dtype', ops.kv4_append, x, x.half(), slots, pool)
    bad('slots must be', ops.kv4_append, x, x, slots[:2], pool)
    bad('slots must be', ops.kv4_append, x, x, slots.long(), pool)
    bad('forward-only', ops.kv4_append, x.clone().requires_grad_(), x, slots, pool, error=NotImplementedError)
    bad('max_len', ops.kv4_gather, pool, table, ln, -1)
    bad('dtype', ops.kv4_gather, pool, table, ln, 3, dtype=torch.int32)
    bad('new_lens', ops.paged_reserve, ln, ln[:1], table, free, one, 16, 3)
    bad('free_count', ops.paged_reserve, ln, ln, table, free, free, 16, 3)
    bad('total_new', ops.paged_reserve, ln, ln, table, free, one, 16, -3)
    bad('page size', ops.paged_reserve, ln, ln, table, free, one, 20, 3)
    bad('slots must be', ops.paged_reserve, ln, ln, table, free, one, 16, 3, slots=slots[:2])
    bad('lens_out', ops.paged_reserve, ln, ln, table, free, one, 16, 3, lens_out=slots)
    bad('done must be', ops.paged_release, ln, ln, table, free, one, 16)
    with torch.no_grad():
        ops.kv4_append(x.clone().requires_grad_(), x, torch.full_like(slots, -1), pool)


def test_a_chain_of_calls_sees_what_was_just_written():
    """Every call of a step starts while the one before it ends: lengths, slots, pool and queries are all
    written by the kernels right before.  The chain without waits equals the one with a wait after
    every call."""
    B, H, kv, D, P = 40, 12, 3, 64, 16
    g = gen(40)
    base = torch.randint(0, 400, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    pr = params(H, 8)
    ks, vs = (torch.randn(8, B * 16, kv, D, device='cuda', generator=g).bfloat16() for _ in range(2))
    qs = torch.randn(8, B, H, 1, D, device='cuda', generator=g).bfloat16()

    def chain(wait):
        pause = torch.cuda.synchronize if wait else (lambda: None)
        pool = ops.kv4_pool(2200, kv, D, P)
        table = torch.full((B, 64), -1, dtype=torch.int32, device='cuda')
        free = torch.arange(2200, dtype=torch.int32, device='cuda')
        count = torch.full((1,), 2200, dtype=torch.int32, device='cuda')
        lens = torch.zeros(B, dtype=torch.int32, device='cuda')
        new = torch.empty_like(lens)
        outs = []
        pause()
        for i in range(8):
            new.copy_((base * (i + 3)) % 16 + (0 if i else 1))
            pause()
            slots, lens, count = ops.paged_reserve(lens, new, table, free, count, P, B * 16)
            pause()
            ops.kv4_append(ks[i], vs[i], slots, pool)
            pause()
            q = qs[i] * 1.0
            pause()
            outs.append(ops.kv4_chord_attention(q, pool, table, lens, *pr))
            pause()
            outs += list(ops.kv4_gather(pool, table, lens, 130))
            pause()
            done = lens > 100
            pause()
            ops.paged_release(done, lens, table, free, count, P)
            pause()
        return outs + [lens, count, table]

    want = chain(True)
    for _ in range(5):
        got = chain(False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """Calls on two streams share nothing but what they read."""
    H, kv, D, P = 8, 2, 64, 32
    pool, table, ln = random_cache([3000, 17, 900], kv, D, P, 41)
    pr = params(H, 9)
    qs = [torch.randn(3, H, 2, D, device='cuda', generator=gen(50 + i)).half() for i in range(2)]
    want = [ops.kv4_chord_attention(q, pool, table, ln, *pr) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(ops.kv4_chord_attention(q, pool, table, ln, *pr))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
