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


def up_to(n, m):
    return -(-n // m) * m


@pytest.mark.parametrize('dtype', [_lib.MB_BF16, _lib.MB_F16, _lib.MB_F32])
@pytest.mark.parametrize('shift', [0, 2])
def test_workspaces_are_within_their_documented_bounds(dtype, shift):
    """Over the range of sizes: up to 2 million words, 32768 features and tokens (sizes are asked for only)."""
    lib = _lib.load()
    parts = 3 if dtype == _lib.MB_F32 else 1
    for n in (17, 1000, 4097, 8192, 8193, 32768, 131072, 200000):
        for v in (100, 4096, 10753, 16385, 32000, 65537, 131072, 349000, 1000000, 2000000):
            for d in (1, 64, 767, 2048, 32768):
                rows, words, d8, d4 = up_to(n, 256), up_to(v, 256), up_to(d, 8), up_to(d, 4)
                x, w = 2 * parts * rows * d8, 2 * parts * words * d8 if parts == 3 or shift else 0
                at_once = _lib.i64_array((0, 0, 0))
                _lib.call('motif_b200_linear_cross_entropy_bytes', ADDR + shift, d8, n, v, d, dtype, at_once)
                state, forward, backward = at_once
                assert state <= x + w + 64 * rows + 4096 and forward <= 64 * rows + (1 << 20)
                run = 8192 // (2 if parts == 3 else 1)
                most = 0.34e9 + (4 * v * d4 if n > run else 0)
                if v > (10752 if parts == 3 else 16384):
                    most += 4 * min(rows, run) * d4
                assert backward <= most, (n, v, d, backward, most)
                if dtype == _lib.MB_F16:
                    continue
                train = lib.motif_b200_linear_cross_entropy_train_workspace_bytes(ADDR + shift, d8, n, v, d, dtype)
                r = min(rows, 65536, max(256, up_to((1 << 28) // parts // words - 255, 256)))
                most = x + w + 64 * rows + max(0.54e9, 512 * parts * words) + 2 * parts * r * d8 + 0.06e9
                most += (4 * v * d4 if n > r else 0) + (4 * r * d4 if parts == 1 and v > 65536 else 0)
                assert 0 < train <= most, (n, v, d, train, most)
