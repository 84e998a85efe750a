"""Limits of the paged cache's calls (no GPU: nothing is launched)."""

import pytest

from motif_b200 import _lib

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
