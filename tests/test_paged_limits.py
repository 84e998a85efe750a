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
