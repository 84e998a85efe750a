"""The model's 4-bit cache in the states that a program can bring it into: other dtypes, stopped and refused
forwards, resets, unequal lengths, every head dim.

Models, the cache of rounded values and the bar are those of `test_paged_model_gpu.py`.
"""

import pytest
import torch

from motif_b200 import model as engine
from motif_b200.cache import KV4LayerCache
from motif_b200.config import MotifChordConfig
from motif_b200.decode import GraphDecoder
from motif_b200.model import MotifChordModel
from test_paged_model_gpu import close, model_of, rounded_cache

pytestmark = pytest.mark.gpu


def ids_of(B, T, seed):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize('other', [torch.bfloat16, torch.float64])
def test_cache_of_another_dtype_is_read_back_in_the_models(other):
    """`cache.to(dtype=...)` changes what `k` and `v` are given as, not what the kernels read (a buffer of
    16-bit values read as 32-bit ones would end halfway)."""
    m = model_of(torch.float32)
    ids = ids_of(2, 30, 2)
    mask = torch.ones(2, 30, dtype=torch.bool)
    mask[0, :4] = False
    cache, ref = m.create_cache(kv_bits=4, kv_capacity=64), rounded_cache(m)
    for c in (cache, ref):
        m(ids[:, :20], cache=c, mask=mask[:, :20])
    for bc in cache:
        for lc in bc.attn:
            if hasattr(lc, 'pages'):
                lc.to(dtype=other)
    close(m(ids[:, 20:], cache=cache, mask=mask).logits, m(ids[:, 20:], cache=ref, mask=mask).logits)


@pytest.mark.parametrize('stopped,chunks', [(2, [1, 1, 1]), (1, [2, 1, 3]), (5, [1, 1, 8, 1]), (3, [3, 1])])
def test_layers_of_unequal_length_attend_to_their_own_tokens(monkeypatch, stopped, chunks):
    """A forward that stops between two Chord layers leaves the first one ahead; what follows is what two
    layers of separate caches give."""
    m = model_of(torch.float32, block=('chord', 'gdn', 'chord'))
    ids = ids_of(2, 60, 5)
    cache, ref = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16), rounded_cache(m)

    def stop(*a):
        raise RuntimeError('stopped')

    for c in (cache, ref):
        m(ids[:, :20], cache=c)
        with monkeypatch.context() as p, pytest.raises(RuntimeError, match='stopped'):
            p.setattr(engine, '_gdn_decoder', stop)
            m(ids[:, 20:20 + stopped], cache=c)
        c[0].attn_res.seq_len = 20
    first, last = cache[0].attn[0], cache[0].attn[2]
    assert (first.length, last.length, first.pages.length) == (20 + stopped, 20, 20 + stopped)
    with pytest.raises(ValueError, match='shared pages|disagree'):
        GraphDecoder(m, cache, max_steps=2)
    at = 20
    for n in chunks:
        close(m(ids[:, at:at + n], cache=cache).logits, m(ids[:, at:at + n], cache=ref).logits)
        at += n
    assert (first.length, last.length) == (at + stopped, at) and torch.equal(last.k, ref[0].attn[2].k[:, ::2])


def test_a_refused_forward_leaves_the_cache_as_it_was():
    """Capacity and batch are checked before any layer advances (the recurrent layers before the first
    Chord layer could not be taken back)."""
    m = model_of(torch.float32, block=('gdn', 'chord'), block_n=2)
    ids = ids_of(2, 40, 6)
    cache, whole = (m.create_cache(kv_bits=4, kv_capacity=n, page_size=16) for n in (32, 64))
    for c in (cache, whole):
        m(ids[:, :30], cache=c)
    for bad, match in ((ids[:, 30:33], 'capacity'), (ids[:1, 30:31], '2 requests'), (ids[:, :33], 'capacity')):
        with pytest.raises(ValueError, match=match):
            m(bad, cache=cache)
    assert cache.seq_len == 30
    assert torch.equal(m(ids[:, 30:32], cache=cache).logits, m(ids[:, 30:32], cache=whole).logits)
    with pytest.raises(ValueError, match='capacity'):
        m(ids[:, 32:33], cache=cache)
    assert cache.seq_len == 32 and all(lc.length == 32 for bc in cache for lc in bc.attn)


def test_reset_keeps_the_cache_in_4_bits():
    """After `ModelCache.reset` the layers are 4-bit ones of the same capacity, and empty."""
    m = model_of(torch.float32, block=('gdn', 'chord', 'chord'), block_n=2)
    ids = ids_of(2, 40, 5)
    cache = m.create_cache(kv_bits=4, kv_capacity=40, page_size=16)
    want = m(ids, cache=cache).logits
    for other in (ids, ids_of(3, 40, 5)):      # the batch may change
        cache.reset()
        assert cache.seq_len == 0 and cache[0].attn[1].pages.batch == 0
        out = m(other, cache=cache)
        for bc, block in zip(cache, m.blocks):
            assert [isinstance(lc, KV4LayerCache) for lc in bc.attn] == [d.attn_type == 'chord' for d in block.features]
        assert torch.equal(out.logits, m(other, cache=m.create_cache(kv_bits=4, kv_capacity=40, page_size=16)).logits)
        with pytest.raises(ValueError, match='capacity'):
            m(other[:, :9], cache=cache)
        if other is ids:
            assert torch.equal(out.logits, want)
    out.reset_caches()
    assert torch.equal(m(ids, cache=cache).logits, want)
    # caches of the model dtype are rebuilt from the decoders' types, as ever
    plain = m.create_cache()
    m(ids, cache=plain)
    plain.reset()
    assert all(len(bc.attn) == 0 for bc in plain)


def test_reset_of_one_layer_leaves_the_others():
    m = model_of(torch.float32, block=('chord', 'gdn', 'chord'))
    cache = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
    m(ids_of(2, 40, 5), cache=cache)
    a, b = cache[0].attn[0], cache[0].attn[2]
    k, v = b.k, b.v
    a.reset()
    assert (a.length, b.length, a.k) == (0, 40, None) and torch.equal(b.k, k) and torch.equal(b.v, v)
    x = torch.randn(2, 2, 50, 64, device='cuda')
    ka, va = a.append(x, x + 1, values=True)   # ahead of the other layer, on its pages and ten more tokens
    assert torch.equal(a.k, ka) and torch.equal(a.v, va) and torch.equal(b.k, k) and torch.equal(b.v, v)
    a.reset()
    b.reset()
    assert a.pages.batch == 0 and a.pages.table is None


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('D', [32, 64, 128])
def test_every_head_dim_decodes_as_a_graph(dtype, D):
    """The captured step runs the 4-bit attention alone, which takes head dims of 128 too; prefill and
    decode in fp32 are held against a cache of rounded values."""
    torch.manual_seed(1)
    cfg = MotifChordConfig(vocab_size=512, model_dim=4 * D, num_heads=4, num_kv_heads=2, head_k_dim=64,
                           block=('gdn', 'chord'), block_n=1)
    m = MotifChordModel(cfg).to('cuda', dtype).eval()
    ids = ids_of(2, 40, 7)
    runs = []
    for graph in (False, True):
        cache = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
        g = m.generate(ids[:, :30], max_new_tokens=20, cache=cache, graph=graph).run()
        assert g.graph_steps == (19 if graph else 0)
        runs.append(g.generated)
    assert torch.equal(*runs)
    if dtype == torch.float32:
        cache, ref = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16), rounded_cache(m)
        for a, b in ((0, 25), (25, 26), (26, 40)):
            close(m(ids[:, a:b], cache=cache).logits, m(ids[:, a:b], cache=ref).logits)


def test_captured_step_follows_lengths_that_differ_on_the_device():
    """Two requests of 24 and 10 tokens on one cache, crossing page boundaries at different steps: each decodes
    as it does alone."""
    m = model_of(torch.float32, block=('chord', 'chord'), seed=8)
    ids, lens = ids_of(2, 24, 9), (24, 10)
    cache = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
    m(ids, cache=cache)
    pages = cache[0].attn[0].pages
    pages.lens.copy_(torch.tensor(lens))   # the second request's later tokens are forgotten
    fed = torch.tensor([[7], [11]], device='cuda')
    dec = GraphDecoder(m, cache, max_steps=12)
    got = dec.run(fed, 12)
    assert pages.lens.tolist() == [n + 12 for n in lens]
    for b, n in enumerate(lens):
        alone = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
        m(ids[b:b + 1, :n], cache=alone)
        one = GraphDecoder(m, alone, max_steps=12)
        assert torch.equal(one.run(fed[b:b + 1], 12)[0], got[b])
        close(dec.logits[b:b + 1], one.logits)


@pytest.mark.parametrize('how', ['model cache', 'one layer', 'moved'])
def test_a_decoder_whose_cache_was_reset_refuses_to_run(how):
    """The graph writes to the pool and the lengths it was captured on; they stay its own."""
    m = model_of(torch.float32)
    ids = ids_of(2, 20, 10)
    cache = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
    first = m(ids, cache=cache).next_token()
    dec = GraphDecoder(m, cache, max_steps=8)
    dec.run(first, 2)
    saved = dec.save()
    if how == 'moved':
        lc = cache[0].attn[1]
        lc.pool = lc.pool.clone()
    else:
        (cache if how == 'model cache' else cache[0].attn[1]).reset()
    for call in (lambda: dec.run(first, 2), lambda: dec.load(saved), lambda: dec.breakdown(first, 1)):
        with pytest.raises(RuntimeError, match='reset or moved'):
            call()
    dec.release()
