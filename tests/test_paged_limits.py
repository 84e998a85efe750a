"""Limits of the paged cache's calls (no GPU: nothing is launched)."""

import pytest

from motif_b200 import _lib
from motif_b200.config import MotifChordConfig
from motif_b200.model import MotifChordModel

ADDR = 4096  # a non-null, aligned stand-in: these calls fail before any use of it


@pytest.mark.parametrize('total', [2 ** 31 - 1, 2 ** 31 - 2 ** 20 + 1, 2 ** 31, -1])
def test_new_tokens_that_pass_32_bits_are_refused(total):
    """The kernel's 32-bit counts run a page ahead of the last token."""
    with pytest.raises(ValueError, match='new tokens'):
        _lib.call('motif_b200_paged_reserve', ADDR, ADDR, ADDR, 4, ADDR, ADDR, ADDR, ADDR, ADDR, total, 2, 4, 8, 16,
                  None)


@pytest.mark.parametrize('page,columns', [(16, 2 ** 27 - 1), (16, 2 ** 27), (512, 2 ** 22 - 1), (16, 2 ** 62)])
def test_tables_whose_tokens_pass_32_bits_are_refused(page, columns):
    """A key tile that begins in the last page ends past it."""
    for name, args in (('motif_b200_kv4_gather', (ADDR, ADDR, columns, ADDR, ADDR, ADDR, 2, 2, 5, 64, 4, page, columns,
                                                  _lib.MB_BF16, None)),
                       ('motif_b200_paged_release', (ADDR, ADDR, ADDR, columns, ADDR, ADDR, 2, columns, 8, page, None))):
        with pytest.raises(ValueError, match='fewer than 2'):
            _lib.call(name, *args)


def test_a_cache_that_cannot_be_kept_is_refused_when_it_is_made():
    """Page size, capacity and head dim, not at the first Chord layer of a forward."""
    def model(heads, block=('gdn', 'chord')):
        return MotifChordModel(MotifChordConfig(vocab_size=64, model_dim=128, num_heads=heads, num_kv_heads=1, head_k_dim=64,
                                                block=block, block_n=1))

    m = model(2)
    for page in (0, 8, 24, 40, 2048, -16):
        with pytest.raises(ValueError, match='page_size'):
            m.create_cache(kv_bits=4, kv_capacity=100, page_size=page)
    with pytest.raises(ValueError, match='capacity'):
        m.create_cache(kv_bits=4, kv_capacity=0)
    with pytest.raises(NotImplementedError, match='head_dim'):
        model(8).create_cache(kv_bits=4, kv_capacity=100)
    model(8, ('gdn',)).create_cache(kv_bits=4, kv_capacity=100)   # no Chord layer, nothing to keep
    assert m.create_cache(kv_bits=4, kv_capacity=100, page_size=48)[0].attn[1].capacity == 144
