"""The operators of a paged Chord key / value cache held in 4 bits, as a serving program calls them.

    reserve    block tables and slot maps built on the GPU from request lengths
    append     new keys and values quantised to 4 bits and stored at their slots, with the values
               that the stored bits stand for given back for the chunk's own attention
    gather     the cached keys and values of a batch read back as contiguous [B, Hkv, S, D] tensors
               (a later prompt chunk attends to them with the prefill kernel)
    attention  Chord attention of the newest tokens of every request over the 4-bit cache

The cache is one uint8 tensor [pages, Hkv, page_size / 16, bytes]: 16 tokens of one kv head make a
unit of K codes [16][D / 2] | V codes [16][D / 2] | K pairs [groups][16] | V pairs [groups][16].  A
group is min(D, 64) neighbouring dims of one token; its pair is (scale, centre) in bf16, scale in the
low half of a 32-bit word, and a code c in 0..15 (dim 2i in the low half of byte i) stands for
centre + scale * (c - 8).

`listed` and `draw` give cases, `prepare` the inputs of one, `run` one pass (elementary torch
operations in 32 bits, or the framework's calls where `own` is set), `work` what a pass cannot do
without, and `exact` the results in 64 bits.
"""

import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
UNIT = 16          # tokens of one storage unit
EPS = 1e-5         # the decay bias's epsilon


# ---------------------------------------------------------------------------------- cases
def listed():
    """The 172M model's shapes (12 query heads, 3 kv heads of 64, context 8192, prompts of 4096) and
    generic ones around them."""
    return [
        # one decode step's bookkeeping: every request of a full batch gets one more token
        _reserve('reserve_decode_64', 64, 1, 8192, 64, 160),
        # a wave of long prompts admitted at once
        _reserve('reserve_prompts_32x4096', 32, 4096, 0, 64, 128),
        # a large mixed batch, chunks of ragged lengths, small pages
        _reserve('reserve_mixed_517', 517, 97, 3001, 16, 256),
        # one layer's new keys and values of a decode step
        _append('append_decode_64', 64, 3, 64, 'bf16', 64),
        # one layer of a prefill of 32 prompts of 4096 tokens
        _append('append_prefill_131072', 131072, 3, 64, 'bf16', 64),
        # the parity mode's type, wide heads, an odd token count
        _append('append_fp32_d128_5003', 5003, 8, 128, 'fp32', 32),
        # a short cached prefix read back for one request's next chunk
        _gather('gather_1x777', 1, 777, 4, 64, 'fp16', 64, False),
        # a batch of cached prefixes of unequal lengths read back for its next chunk
        _gather('gather_32x4096', 32, 4096, 3, 64, 'bf16', 64, True),
        # interactive use: one request, a short context, the parity mode's type
        _attention('attention_1x300_fp32', 1, 300, 1, 4, 4, 64, 'fp32', 64, False),
        # a few requests at the benchmark's context length
        _attention('attention_8x8192', 8, 8192, 1, 12, 3, 64, 'bf16', 64, False),
        # the benchmark's decode batch
        _attention('attention_64x8192', 64, 8192, 1, 12, 3, 64, 'bf16', 64, False),
        # ragged lengths, several tokens per request (drafted tokens to verify), wide heads, small pages
        _attention('attention_ragged_48x5000_t4', 48, 5000, 4, 16, 4, 128, 'fp16', 32, True),
    ]


def _reserve(name, batch, new, cached, page, columns):
    return {'name': name, 'op': 'reserve', 'batch': batch, 'new': new, 'cached': cached, 'page': page,
            'columns': columns}


def _append(name, tokens, kv_heads, dim, dtype, page):
    return {'name': name, 'op': 'append', 'tokens': tokens, 'kv_heads': kv_heads, 'dim': dim, 'dtype': dtype,
            'page': page}


def _gather(name, batch, length, kv_heads, dim, dtype, page, ragged):
    return {'name': name, 'op': 'gather', 'batch': batch, 'length': length, 'kv_heads': kv_heads, 'dim': dim,
            'dtype': dtype, 'page': page, 'ragged': ragged}


def _attention(name, batch, length, new, heads, kv_heads, dim, dtype, page, ragged):
    return {'name': name, 'op': 'attention', 'batch': batch, 'length': length, 'new': new, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'dtype': dtype, 'page': page, 'ragged': ragged}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges: batches 1 to 64 (the bookkeeping: to 1024), contexts 1 to 8192
    tokens, every head dim, type and page size."""
    op = rng.choice(['reserve', 'append', 'gather', 'attention', 'attention'])
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([32, 64, 64, 128])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op == 'reserve':
        batch = _log_int(rng, 1, 1024)
        new = _log_int(rng, 1, min(4096, max(1, 131072 // batch)))
        cached = rng.choice([0, _log_int(rng, 1, 8192)])
        case = _reserve('', batch, new, cached, page, -(-(cached + new) // page) + rng.randrange(0, 9))
    elif op == 'append':
        kv = rng.choice([1, 2, 3, 4, 8])
        tokens = _log_int(rng, 1, 131072 * 3 * 64 // (kv * dim) // (2 if dtype == 'fp32' else 1))
        case = _append('', tokens, kv, dim, dtype, page)
    else:
        kv = rng.choice([1, 2, 3, 4, 8])
        batch = _log_int(rng, 1, 64)
        most = 64 * 8192 * 3 * 64 if op == 'attention' else 16 * 4096 * 3 * 64 // (2 if dtype == 'fp32' else 1)
        length = _log_int(rng, 1, max(1, min(8192, most // (batch * kv * dim))))
        ragged = batch > 1 and rng.random() < 0.5
        if op == 'gather':
            case = _gather('', batch, length, kv, dim, dtype, page, ragged)
        else:
            new = min(length, rng.choice([1, 1, 1, 2, 3, 4]))
            heads = kv * rng.choice([1, 2, 3, 4, 8])
            case = _attention('', batch, length, new, heads, kv, dim, dtype, page, ragged)
    del case['name']
    return case


def _lengths(case):
    """Cached lengths of the requests, by the case alone: equal, or spread over 0 .. length (one
    request empty, one at the full length)."""
    batch, length = case['batch'], case['length']
    if not case['ragged']:
        return [length] * batch
    spread = [(i * 2654435761 + 12345) % (length + 1) for i in range(batch)]
    spread[0], spread[-1] = length, 0
    return spread


def _group(dim):
    return min(dim, 64)


def _unit_bytes(dim):
    return UNIT * dim + 2 * 4 * UNIT * (dim // _group(dim))


# ---------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def _random_pool(pages, kv_heads, dim, page, g):
    """Filled pages: codes of normal values (a row's 64 values span about 4.7 standard deviations, so
    the codes lie about 8 with a deviation of about 3.2), scales and centres as quantised rows have them."""
    units = pages * kv_heads * (page // UNIT)
    ng = dim // _group(dim)

    def codes():
        x = torch.empty((units, UNIT * dim), device='cuda', dtype=torch.float16).normal_(7.5, 3.2, generator=g)
        c = x.round_().clamp_(0, 15).to(torch.uint8)
        return c[:, 0::2] | (c[:, 1::2] << 4)

    def pairs(sigma):
        scale = torch.empty((units, ng * UNIT), device='cuda').uniform_(0.26 * sigma, 0.36 * sigma, generator=g)
        centre = torch.empty((units, ng * UNIT), device='cuda').normal_(0.0, 0.2 * sigma, generator=g)
        both = torch.stack([scale, centre], -1).to(torch.bfloat16)
        return both.view(torch.uint8).reshape(units, -1)

    pool = torch.cat([codes(), codes(), pairs(1.0), pairs(0.5)], 1)
    return pool.reshape(pages, kv_heads, page // UNIT, _unit_bytes(dim))


def _cached_batch(case, g):
    """A pool, block tables (pages in no order, the unused columns -1) and lengths."""
    lens = _lengths(case)
    page = case['page']
    counts = [-(-n // page) for n in lens]
    columns, used = max(1, max(counts)), sum(counts)
    pages = used + 1 + case['batch'] % 7
    order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32)
    count = torch.tensor(counts, device='cuda')
    start = count.cumsum(0) - count
    col = torch.arange(columns, device='cuda')
    held = col[None, :] < count[:, None]
    table = torch.where(held, order[(start[:, None] + col[None, :]).clamp_max(pages - 1)], -1).to(torch.int32)
    return {'pool': _random_pool(pages, case['kv_heads'], case['dim'], page, g), 'table': table.contiguous(),
            'lens': torch.tensor(lens, dtype=torch.int32, device='cuda'), 'max_len': max(lens)}


def prepare(case, seed):
    g = _generator(seed)
    state = {'case': case}
    if case['op'] == 'reserve':
        batch, page, columns = case['batch'], case['page'], case['columns']
        # lengths and chunks spread around the case's figures; about one request in 16 has nothing new
        lens = (case['cached'] * (0.5 + 0.5 * torch.rand(batch, device='cuda', generator=g))).int()
        new = (case['new'] * (0.5 + 0.5 * torch.rand(batch, device='cuda', generator=g))).ceil().int()
        if case['new'] == 1 and batch > 1:
            new[torch.rand(batch, device='cuda', generator=g) < 0.06] = 0
        held = ((lens + page - 1) // page).long()
        needed = int(((lens + new + page - 1) // page).sum())
        pages = needed + 8
        order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32)
        used = int(held.sum())
        col = torch.arange(columns, device='cuda')
        start = held.cumsum(0) - held
        table = torch.where(col[None, :] < held[:, None],
                            order[(start[:, None] + col[None, :]).clamp_max(pages - 1)], -1).to(torch.int32)
        free = torch.zeros(pages, dtype=torch.int32, device='cuda')
        free[:pages - used] = order[used:]
        state.update(lens=lens, new=new, table=table.contiguous(), free=free,
                     count=torch.tensor([pages - used], dtype=torch.int32, device='cuda'),
                     total=batch * case['new'])
    elif case['op'] == 'append':
        n, kv, dim, page = case['tokens'], case['kv_heads'], case['dim'], case['page']
        # keys are unit root-mean-square rows (as after the key norm) with learned per-channel weights,
        # values are normal with a few large channels
        chan = 1.0 + 0.3 * torch.randn(dim, device='cuda', generator=g)
        k = torch.randn((n, kv, dim), device='cuda', generator=g) * chan
        v = 0.5 * torch.randn((n, kv, dim), device='cuda', generator=g)
        v[..., ::17] *= 3.0
        pages = -(-n // page) + 3
        slots = (torch.randperm(pages, device='cuda', generator=g)[:, None] * page
                 + torch.arange(page, device='cuda')[None, :]).reshape(-1)[:n]
        state.update(k=k.to(DTYPES[case['dtype']]), v=v.to(DTYPES[case['dtype']]), slots=slots.to(torch.int32),
                     pool=torch.zeros((pages, kv, page // UNIT, _unit_bytes(dim)), dtype=torch.uint8, device='cuda'))
    else:
        state.update(_cached_batch(case, g))
        if case['op'] == 'attention':
            heads = case['heads']
            q = torch.randn((case['batch'], heads, case['new'], case['dim']), device='cuda', generator=g)

            def uniform(lo, hi):
                return lo + (hi - lo) * torch.rand(heads, device='cuda', generator=g)

            state.update(q=q.to(DTYPES[case['dtype']]), alpha=uniform(0.3, 1.5), beta=uniform(0.0, 0.6),
                         mu=uniform(-1.0, 2.0), ssmax=uniform(0.3, 0.9))
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    op = state['case']['op']
    if own:
        from motif_b200 import ops
        if op == 'reserve':
            slots, lens, count = ops.paged_reserve(state['lens'], state['new'], state['table'], state['free'],
                                                   state['count'], state['case']['page'], state['total'])
            return {'slots': slots, 'lens': lens, 'count': count, 'table': state['table']}
        if op == 'append':
            k, v = ops.kv4_append(state['k'], state['v'], state['slots'], state['pool'], values=True)
            return {'k': k, 'v': v}
        if op == 'gather':
            k, v = ops.kv4_gather(state['pool'], state['table'], state['lens'], state['max_len'],
                                  dtype=DTYPES[state['case']['dtype']])
            return {'k': k, 'v': v}
        return ops.kv4_chord_attention(state['q'], state['pool'], state['table'], state['lens'], state['alpha'],
                                       state['beta'], state['mu'], state['ssmax'])
    if op == 'reserve':
        return _plain_reserve(state)
    if op == 'append':
        return _plain_append(state)
    if op == 'gather':
        dtype = DTYPES[state['case']['dtype']]
        k, v = _plain_cached(state)
        return {'k': k.to(dtype), 'v': v.to(dtype)}
    return _plain_attention(state)


def _plain_reserve(state):
    """Requests are served in order until one does not fit; table columns are filled from the top of
    the free list, and every new token gets page * page_size + offset (-1 where its request got none)."""
    page, total = state['case']['page'], state['total']
    lens, new, table, free = state['lens'].long(), state['new'].long(), state['table'], state['free']
    columns, count = table.shape[1], state['count'].long()
    old_pages, all_pages = (lens + page - 1) // page, (lens + new + page - 1) // page
    ends = new.cumsum(0)
    possible = (all_pages <= columns) & (ends <= total)
    need = torch.where(possible, all_pages - old_pages, 0)
    upto = need.cumsum(0)
    served = possible & ((need == 0) | (upto <= count))
    taken = torch.where(served, need, 0)
    j = torch.arange(columns, device=lens.device)[None, :] - old_pages[:, None]
    source = count - 1 - ((upto - need)[:, None] + j)
    fresh = (j >= 0) & (j < taken[:, None])
    table.copy_(torch.where(fresh, free[source.clamp(0, free.numel() - 1)], table))
    token = torch.arange(total, device=lens.device)
    row = torch.searchsorted(ends, token, right=True).clamp_max(lens.numel() - 1)
    pos = lens[row] + token - (ends - new)[row]
    there = (token < ends[-1]) & served[row]
    slots = torch.where(there, table[row, (pos // page).clamp_max(columns - 1)].long() * page + pos % page, -1)
    return {'slots': slots.to(torch.int32), 'lens': torch.where(served, lens + new, lens).to(torch.int32),
            'count': (count - taken.sum()).to(torch.int32), 'table': table}


def _plain_quantise(x):
    """x [N, Hkv, D] in 32 bits -> codes (uint8), scale and centre (bf16), and the values they stand for."""
    n, kv, dim = x.shape
    y = x.reshape(n, kv, dim // _group(dim), _group(dim))
    lo = y.amin(-1, keepdim=True)
    steps = torch.full_like(lo, 15.0)  # a tensor: dividing by a number may multiply by its rounded reciprocal
    scale = ((y.amax(-1, keepdim=True) - lo) / steps).to(torch.bfloat16)
    s = scale.float()
    centre = (lo + 8.0 * s).to(torch.bfloat16)
    m = centre.float()
    code = torch.where(s > 0.0, (y - m) / s, torch.zeros_like(y))
    code = (code.round() + 8.0).clamp(0.0, 15.0)
    return code.to(torch.uint8).view(n, kv, dim), scale, centre, (m + s * (code - 8.0)).view(n, kv, dim)


def _plain_append(state):
    case, pool, slots = state['case'], state['pool'], state['slots'].long()
    dim, page = case['dim'], case['page']
    half, ng = dim // 2, dim // _group(dim)
    where = (slots // page, slice(None), slots % page // UNIT)
    inside = slots % UNIT
    values = []
    kinds = [(state['k'], 0, 2 * UNIT * half), (state['v'], UNIT * half, 2 * UNIT * half + 4 * ng * UNIT)]
    heads = torch.arange(pool.shape[1], device=pool.device)[None, :, None]
    pages, subs, rows = where[0][:, None, None], where[2][:, None, None], inside[:, None, None]
    byte = torch.arange(half, device=pool.device)[None, None, :]
    four = torch.arange(4 * ng, device=pool.device)[None, None, :]
    for x, code_at, pair_at in kinds:
        code, scale, centre, value = _plain_quantise(x.float())
        pool[pages, heads, subs, code_at + rows * half + byte] = code[..., 0::2] | (code[..., 1::2] << 4)
        pair = torch.stack([scale[..., 0], centre[..., 0]], -1).view(torch.uint8)
        pool[pages, heads, subs, pair_at + (four // 4) * 4 * UNIT + rows * 4 + four % 4] = pair.reshape(
            *code.shape[:2], 4 * ng)
        values.append(value.to(x.dtype))
    return {'k': values[0], 'v': values[1]}


def _plain_cached(state):
    """The cached keys and values in 32 bits, [B, Hkv, max_len, D], zeros past each length."""
    case, pool, table, most = state['case'], state['pool'], state['table'], state['max_len']
    dim, page, kv = case['dim'], case['page'], case['kv_heads']
    half, group = dim // 2, _group(dim)
    ng, batch, columns = dim // group, table.shape[0], table.shape[1]
    got = pool[table.clamp_min(0).long()]                       # [B, columns, Hkv, page / 16, bytes]
    got = got.transpose(1, 2).reshape(batch, kv, columns * page // UNIT, -1)
    seen = torch.arange(columns * page, device=pool.device)[None, :] < state['lens'][:, None]
    both = []
    for code_at, pair_at in ((0, 2 * UNIT * half), (UNIT * half, 2 * UNIT * half + 4 * ng * UNIT)):
        byte = got[..., code_at:code_at + UNIT * half].reshape(batch, kv, -1, half)
        code = torch.stack([byte & 15, byte >> 4], -1).reshape(batch, kv, -1, ng, group).float()
        pair = got[..., pair_at:pair_at + 4 * ng * UNIT].contiguous().view(torch.bfloat16)
        pair = pair.reshape(batch, kv, -1, ng, UNIT, 2).transpose(3, 4).reshape(batch, kv, -1, ng, 2).float()
        x = (pair[..., 1:] + pair[..., :1] * (code - 8.0)).reshape(batch, kv, -1, dim)
        both.append(torch.where(seen[:, None, :, None], x, torch.zeros_like(x))[:, :, :most])
    return both


def _plain_attention(state):
    q, lens = state['q'].float(), state['lens']
    batch, heads, new, dim = q.shape
    kv, most = state['case']['kv_heads'], state['max_len']
    k, v = _plain_cached(state)
    scores = q.reshape(batch, kv, heads // kv * new, dim) @ k.transpose(-1, -2) * dim ** -0.5
    scores = scores.view(batch, heads, new, most)
    pos = lens[:, None] - new + torch.arange(new, device=q.device)                       # [B, T]
    key = torch.arange(most, device=q.device)
    gap = (key[None, None, :] - pos[:, :, None]).float()[:, None]                        # [B, 1, T, S]
    per_head = [p.view(1, heads, 1, 1) for p in (state['alpha'], state['beta'], state['mu'], state['ssmax'])]
    alpha, beta, mu, ssmax = per_head
    bias = -alpha * ((gap - mu).abs() + EPS) ** beta
    logits = (scores + bias) * (ssmax * torch.log(pos.clamp_min(0).float() + 1.0)[:, None, :, None])
    logits = logits.masked_fill(key[None, None, None, :] > pos[:, None, :, None], float('-inf'))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == float('-inf'), torch.zeros_like(top), top))
    out = p.view(batch, kv, -1, most) @ v / p.sum(-1).clamp_min(1e-20).view(batch, kv, -1, 1)
    return out.view(batch, heads, new, dim).to(state['q'].dtype)


# ---------------------------------------------------------------------------------- what it needs
def work(case):
    if case['op'] == 'reserve':
        # lengths in and out, the slot of every new token, the fresh table entries and their pages
        tokens = case['batch'] * case['new']
        fresh = case['batch'] * -(-case['new'] // case['page'])
        return {'bytes': 12 * case['batch'] + 4 * tokens + 8 * fresh, 'flops': 0}
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'append':
        rows = 2 * case['tokens'] * case['kv_heads']
        held = case['dim'] // 2 + 4 * (case['dim'] // _group(case['dim']))
        # keys and values in, the stored bits and the values they stand for out
        return {'bytes': rows * (2 * size * case['dim'] + held) + 4 * case['tokens'], 'flops': 6 * rows * case['dim']}
    lens = _lengths(case)
    held = sum(lens) * case['kv_heads'] * (_unit_bytes(case['dim']) // UNIT)
    if case['op'] == 'gather':
        out = 2 * case['batch'] * max(lens) * case['kv_heads'] * case['dim'] * size
        return {'bytes': held + out, 'flops': 4 * sum(lens) * case['kv_heads'] * case['dim']}
    rows = case['heads'] * case['new']
    ends = 2 * case['batch'] * rows * case['dim'] * size
    return {'bytes': held + ends, 'flops': 4 * sum(lens) * rows * case['dim']}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The operator's definition in float64, request by request (the bookkeeping has whole numbers only)."""
    if case['op'] == 'reserve':
        return None
    state = prepare(case, seed)
    if case['op'] == 'append':
        return {'k': _exact_rounded(state['k']), 'v': _exact_rounded(state['v'])}
    dim, kv, page = case['dim'], case['kv_heads'], case['page']
    lens = state['lens'].tolist()
    if case['op'] == 'gather':
        k = torch.zeros((case['batch'], kv, state['max_len'], dim), dtype=torch.float64, device='cuda')
        v = torch.zeros_like(k)
        for b, n in enumerate(lens):
            if n:
                k[b, :, :n], v[b, :, :n] = _exact_request(state['pool'], state['table'][b], n, dim, page)
        return {'k': k, 'v': v}
    q, heads, new = state['q'].double(), case['heads'], case['new']
    out = torch.zeros_like(q)
    share = heads // kv
    alpha, beta, mu, ssmax = (state[x].double() for x in ('alpha', 'beta', 'mu', 'ssmax'))
    for b, n in enumerate(lens):
        if not n:
            continue
        k, v = _exact_request(state['pool'], state['table'][b], n, dim, page)
        key = torch.arange(n, device='cuda', dtype=torch.float64)
        for t in range(new):
            at = n - new + t
            if at < 0:
                continue
            dist = (key[None, :at + 1] - at - mu[:, None]).abs() + EPS
            dots = torch.einsum('kgd,ksd->kgs', q[b, :, t].view(kv, share, dim), k[:, :at + 1]).reshape(heads, -1)
            x = (dots / math.sqrt(dim) - alpha[:, None] * dist.pow(beta[:, None])) * ssmax[:, None] * math.log(at + 1.0)
            w = torch.softmax(x, -1).view(kv, share, -1)
            out[b, :, t] = torch.einsum('kgs,ksd->kgd', w, v[:, :at + 1]).reshape(heads, dim)
    return out


def _exact_rounded(x):
    """The nearest values of each group's 16 steps: scale (max - min) / 15 and centre min + 8 scale are
    numbers of 8 bits, the codes are whole."""
    d = x.double()
    d = d.view(*x.shape[:2], -1, _group(x.shape[-1]))
    low = d.min(-1, keepdim=True).values
    step = ((d.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
    mid = (low + 8 * step).bfloat16().double()
    code = torch.clamp(torch.round((d - mid) / step), -8, 7)
    return torch.where(step > 0, mid + step * code, mid).reshape(x.shape)


def _exact_request(pool, table, n, dim, page):
    """K and V of one request, [Hkv, n, D] in float64, read token by token out of the pages."""
    token = torch.arange(n, device=pool.device)
    unit = pool[table[token // page].long(), :, token % page // UNIT].transpose(0, 1)      # [Hkv, n, bytes]
    row, ng = token % UNIT, dim // _group(dim)
    found = []
    for start, after in ((0, UNIT * dim), (UNIT * dim // 2, UNIT * dim + 4 * UNIT * ng)):
        at = start + row[:, None] * (dim // 2) + torch.arange(dim, device=pool.device)[None, :] // 2
        byte = unit.gather(2, at.expand(unit.shape[0], -1, -1)).int()
        odd = torch.arange(dim, device=pool.device) % 2
        code = (byte >> (4 * odd)) % 16 - 8
        at = after + 4 * row[:, None] + 4 * UNIT * (torch.arange(dim, device=pool.device) // _group(dim))[None, :]

        def half(first):
            low = unit.gather(2, (at + first).expand(unit.shape[0], -1, -1)).int()
            high = unit.gather(2, (at + first + 1).expand(unit.shape[0], -1, -1)).int()
            return ((low + 256 * high) << 16).view(torch.float32).double()

        found.append(half(2) + half(0) * code)
    return found
