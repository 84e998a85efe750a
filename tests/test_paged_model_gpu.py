"""The model on a 4-bit Chord cache (`create_cache(kv_bits=4)`).

The reference run is the same model on a 16 / 32-bit cache whose keys and values were rounded to what
the stored bits stand for, through the attention kernels that read such caches.  With one Chord layer,
the last one, both runs quantise the same numbers, so fp32 logits differ by the attention's own
rounding: 3e-5 in a weight (64 * 8 * 2^-24, see the operator tests), which the output projections and
the residual carry to the logits at the same relative size; the bar is 1e-4 of the largest logit.
"""

import pytest
import torch

from motif_b200 import ops
from motif_b200.cache import KV4LayerCache, KVLayerCache
from motif_b200.config import MotifChordConfig
from motif_b200.decode import GraphDecoder, fill_cache_random
from motif_b200.model import MotifChordModel

pytestmark = pytest.mark.gpu


class RoundedCache(KVLayerCache):
    """A cache of the model dtype that holds the values of the 4-bit codes."""

    def update(self, k_new, v_new, dim=2):
        B, kv, T, D = k_new.shape
        pool = ops.kv4_pool(-(-B * T // 16), kv, D, 16)
        k, v = ops.kv4_append(k_new, v_new, torch.arange(B * T, dtype=torch.int32, device='cuda'), pool, values=True)
        return super().update(k, v)


def model_of(dtype, block=('gdn', 'chord'), block_n=1, heads=4, kv=2, seed=0):
    torch.manual_seed(seed)
    cfg = MotifChordConfig(vocab_size=512, model_dim=256, num_heads=heads, num_kv_heads=kv, head_k_dim=64, block=block,
                           block_n=block_n)
    m = MotifChordModel(cfg).to('cuda', dtype).eval()
    with torch.no_grad():
        for n, p in m.named_parameters():
            if 'theta_beta' in n:
                p.copy_(0.5 * torch.rand_like(p))
            elif 'theta_alpha' in n:
                p.copy_(-1.0 - torch.rand_like(p))
    m.invalidate_packed()
    return m


def rounded_cache(m):
    c = m.create_cache()
    for bc in c:
        for i, lc in enumerate(bc.attn):
            if isinstance(lc, KVLayerCache):
                bc.attn[i] = RoundedCache(num_heads=m.config.num_heads)
    return c


def close(a, b, rel=1e-4):
    assert (a.double() - b.double()).abs().max() <= rel * b.double().abs().max()


@pytest.mark.parametrize('chunks', [[70, 1, 1, 1], [1, 1, 5], [40, 33, 1, 90, 2], [130, 1], [30, 350, 2]])
def test_logits_match_a_cache_of_rounded_values(chunks):
    m = model_of(torch.float32)
    B, total = 3, sum(chunks)
    ids = torch.randint(0, 512, (B, total), generator=torch.Generator().manual_seed(1)).cuda()
    cache, ref = m.create_cache(kv_bits=4, kv_capacity=total, page_size=16), rounded_cache(m)
    at = 0
    for n in chunks:
        x = ids[:, at:at + n]
        close(m(x, cache=cache).logits, m(x, cache=ref).logits)
        at += n
    lc = cache[0].attn[1]
    assert isinstance(lc, KV4LayerCache) and lc.length == total and lc.pages.lens.tolist() == [total] * B
    assert int(lc.pages.count) == B * (-(-total // 16)) - B * -(-total // 16)
    rc = ref[0].attn[1]
    assert torch.equal(lc.k, rc.k[:, ::2]) and torch.equal(lc.v, rc.v[:, ::2])   # two query heads per kv head


def test_mask_and_position_read_the_cache_back():
    m = model_of(torch.float32)
    ids = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(2)).cuda()
    mask = torch.ones(2, 30, dtype=torch.bool)
    mask[0, :4] = False
    cache, ref = m.create_cache(kv_bits=4, kv_capacity=64), rounded_cache(m)
    close(m(ids[:, :20], cache=cache, mask=mask[:, :20]).logits, m(ids[:, :20], cache=ref, mask=mask[:, :20]).logits)
    close(m(ids[:, 20:], cache=cache, mask=mask).logits, m(ids[:, 20:], cache=ref, mask=mask).logits)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_graph_decode_equals_eager_decode(dtype):
    m = model_of(dtype, block=('gdn', 'chord', 'chord'), block_n=2, heads=4, kv=1, seed=3)
    ids = torch.randint(0, 512, (2, 50), generator=torch.Generator().manual_seed(3)).cuda()
    runs = []
    for graph in (False, True):
        cache = m.create_cache(kv_bits=4, kv_capacity=50 + 40, page_size=32)
        g = m.generate(ids, max_new_tokens=40, cache=cache, graph=graph).run()
        assert g.graph_steps == (39 if graph else 0)
        runs.append((g.generated, cache))
    assert torch.equal(runs[0][0], runs[1][0])
    for bc0, bc1 in zip(runs[0][1], runs[1][1]):
        for a, b in zip(bc0.attn, bc1.attn):
            if isinstance(a, KV4LayerCache):
                assert a.length == b.length == 89 and a.pages.lens.tolist() == b.pages.lens.tolist() == [89, 89]
                assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_graph_decoder_rewinds_and_follows_unequal_lengths():
    """save / load puts the pages back; requests of unequal lengths decode as they do alone."""
    m = model_of(torch.float32, seed=4)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 512, (2, 24), generator=g).cuda()
    cache = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
    first = m(ids, cache=cache).next_token()
    dec = GraphDecoder(m, cache, max_steps=12)
    saved = dec.save()
    a = dec.run(first, 6).clone()
    left = int(dec.pages.count)
    dec.load(saved)
    assert dec.pages.lens.tolist() == [24, 24]
    assert torch.equal(a, dec.run(first, 6)) and int(dec.pages.count) == left
    dec.release()
    # one request alone, and the same one beside a longer one whose lengths differ on the device
    alone = m.create_cache(kv_bits=4, kv_capacity=64, page_size=16)
    f1 = m(ids[:1], cache=alone).next_token()
    want = GraphDecoder(m, alone, max_steps=6).run(f1, 6)
    assert torch.equal(want, a[:1])


def test_refusals_and_reset():
    m = model_of(torch.float32)
    ids = torch.zeros(1, 20, dtype=torch.int64, device='cuda')
    with pytest.raises(NotImplementedError, match='kv_bits'):
        m.create_cache(kv_bits=8, kv_capacity=10)
    with pytest.raises(ValueError, match='kv_capacity'):
        m.create_cache(kv_bits=4)
    with pytest.raises(ValueError, match='neither'):
        m.create_cache(kv_bits=4, kv_capacity=10, wide_kv=True)
    cache = m.create_cache(kv_bits=4, kv_capacity=16, page_size=16)
    with pytest.raises(ValueError, match='capacity'):
        m(ids, cache=cache)
    cache = m.create_cache(kv_bits=4, kv_capacity=32, page_size=16)
    m(ids, cache=cache)
    with pytest.raises(ValueError, match='capacity'):
        GraphDecoder(m, cache, max_steps=13)
    lc = cache[0].attn[1]
    assert lc.capacity == 32 and lc.seq_length == 20 and 'KV4' in repr(lc)
    lc.reset()
    assert lc.k is None and lc.pages.length == 0


def test_random_fill_stands_for_a_prefill():
    m = model_of(torch.bfloat16, block=('chord', 'gdn', 'chord'))
    cache = fill_cache_random(m, m.create_cache(kv_bits=4, kv_capacity=1200), 2, 1100, 1200)
    dec = GraphDecoder(m, cache, max_steps=8)
    toks = dec.run(torch.zeros(2, 1, dtype=torch.int64, device='cuda'), 8)
    a, b = cache[0].attn[0], cache[0].attn[2]
    assert a.k.shape == b.v.shape == (2, 2, 1108, 64) and not torch.equal(a.k, b.k)
    assert toks.shape == (2, 8) and dec.pages.lens.tolist() == [1108, 1108] and torch.isfinite(dec.logits).all()
