"""The state that the vocabulary loss's forward pass leaves: the backward pass takes it as it was laid out then (no GPU:
nothing is launched)."""

import pytest

from motif_b200 import _lib

ADDR = 4096  # a non-null, aligned stand-in: these calls fail, or end, before any use of it
N, V, D = 40, 300, 96


def sizes(w, stride, dtype, n=N):
    out = _lib.i64_array((0, 0, 0))
    _lib.call('motif_b200_linear_cross_entropy_bytes', w, stride, n, V, D, dtype, out)
    return list(out)


def backward(w, stride, dtype, state_bytes, n=N):
    """Without a gradient to compute, the call ends after its checks."""
    _lib.call('motif_b200_linear_cross_entropy_backward', w, stride, ADDR, 1, 0, None, None, n, V, D, ADDR, state_bytes, ADDR,
              1 << 40, dtype, None)


@pytest.mark.parametrize('dtype', [_lib.MB_BF16, _lib.MB_F16])
def test_the_size_of_the_state_tells_its_layout(dtype):
    plain, packed = sizes(ADDR, D, dtype), sizes(ADDR + 2, D, dtype)
    assert sizes(ADDR, 97, dtype) == packed and sizes(ADDR, 104, dtype) == plain
    # 300 words are 512 packed rows
    assert packed[0] - plain[0] == 512 * D * 2 and packed[1:] == plain[1:]
    for w, stride in ((ADDR, D), (ADDR + 2, D), (ADDR, 97)):  # a copy in the state: w may be anywhere by now
        backward(w, stride, dtype, packed[0])
    backward(ADDR, D, dtype, plain[0])
    backward(ADDR + 16, 104, dtype, plain[0])
    for w, stride in ((ADDR + 2, D), (ADDR, 97)):
        with pytest.raises(ValueError, match='16-byte boundaries'):
            backward(w, stride, dtype, plain[0])
    for other in (0, 1, plain[0] - 256, plain[0] + 256, packed[0] - 256, packed[0] + 256):
        with pytest.raises(ValueError, match='none that a forward pass'):
            backward(ADDR, D, dtype, other)


def test_fp32_has_one_layout():
    for n in (N, 9):  # more tokens than the kernels for few take, and those
        need = sizes(ADDR, D, _lib.MB_F32, n)
        assert sizes(ADDR + 4, 97, _lib.MB_F32, n) == need
        backward(ADDR + 4, 97, _lib.MB_F32, need[0], n)
        backward(ADDR, D, _lib.MB_F32, need[0] + 4096, n)
        with pytest.raises(ValueError, match='bytes of state and workspace needed'):
            backward(ADDR, D, _lib.MB_F32, need[0] - 256, n)
