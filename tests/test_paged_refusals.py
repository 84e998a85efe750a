"""What the paged 4-bit cache operators refuse, and how (no GPU: nothing is launched)."""

import pytest
import torch

from motif_b200 import _lib, ops, paged


def test_pool_arguments():
    pool = ops.kv4_pool(3, 2, 64, 32, device='cpu')
    assert pool.shape == (3, 2, 2, 1152) and pool.dtype == torch.uint8
    for dim, nbytes in paged._UNIT_BYTES.items():
        assert _lib.load().motif_b200_kv4_unit_bytes(dim) == nbytes
    assert _lib.load().motif_b200_kv4_unit_bytes(48) == 0
    with pytest.raises(NotImplementedError, match='head_dim'):
        ops.kv4_pool(3, 2, 48, device='cpu')
    for page in (0, 8, 40, 1040):
        with pytest.raises(ValueError, match='page_size'):
            ops.kv4_pool(3, 2, 64, page, device='cpu')
    with pytest.raises(ValueError, match='positive'):
        ops.kv4_pool(0, 2, 64, device='cpu')


def test_host_tensors_are_refused():
    pool = ops.kv4_pool(3, 2, 64, 32, device='cpu')
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    x, p = torch.zeros(2, 2, 64), torch.zeros(4)
    with pytest.raises(ValueError, match='CUDA'):
        ops.paged_reserve(i32, i32, table, i32, i32[:1], 32, 2)
    with pytest.raises(ValueError, match='CUDA'):
        ops.paged_release(i32.bool(), i32, table, i32, i32[:1], 32)
    with pytest.raises(ValueError, match='CUDA'):
        ops.kv4_append(x, x, i32, pool)
    with pytest.raises(ValueError, match='CUDA'):
        ops.kv4_gather(pool, table, i32, 5)
    with pytest.raises(ValueError, match='CUDA'):
        ops.kv4_chord_attention(x.view(2, 2, 1, 64), pool, table, i32, p, p, p, p)


ADDR = 4096  # a non-null, aligned stand-in: these calls fail before any use of it


def reserve(B=2, columns=4, stride=4, cap=8, page=16, total=3, slots=ADDR, lens=ADDR):
    _lib.call('motif_b200_paged_reserve', lens, ADDR, ADDR, stride, ADDR, ADDR, ADDR, ADDR, slots, total, B, columns,
              cap, page, None)


def append(dtype=_lib.MB_BF16, D=64, k=ADDR, pool=ADDR, stride=64, pages=4, page=16, ko=None, vo=None, B=1, T=2):
    _lib.call('motif_b200_kv4_append', k, ADDR, ADDR, pool, ko, vo, _lib.i64_array([0, 64, stride] * 4), B, T, 2, D,
              pages, page, dtype, None)


def gather(dtype=_lib.MB_BF16, D=64, out=ADDR, S=5, pages=4, page=16, columns=3):
    _lib.call('motif_b200_kv4_gather', ADDR, ADDR, columns, ADDR, out, ADDR, 2, 2, S, D, pages, page, columns, dtype,
              None)


def attention(dtype=_lib.MB_BF16, D=64, q=ADDR, H=4, T=1, pool=ADDR, pages=4, page=16, columns=3, ws=ADDR, nbytes=1 << 40):
    _lib.call('motif_b200_kv4_chord_attention', q, pool, ADDR, columns, ADDR, None, ADDR, ADDR, ADDR, ADDR, ADDR,
              _lib.i64_array([0] * 6), 2, H, 2, T, D, pages, page, columns, 0.125, 1e-5, ws, nbytes, dtype, None)


@pytest.mark.parametrize('call,kw,error,match', [
    (reserve, dict(lens=None), ValueError, 'null pointer'),
    (reserve, dict(slots=None), ValueError, 'null pointer'),
    (reserve, dict(page=24), ValueError, 'page size'),
    (reserve, dict(stride=3), ValueError, 'row stride'),
    (reserve, dict(columns=0), ValueError, 'columns'),
    (reserve, dict(columns=1 << 28, stride=1 << 28), ValueError, 'fewer than 2'),
    (reserve, dict(total=-1), ValueError, 'new tokens'),
    (reserve, dict(cap=0), ValueError, 'free list'),
    (reserve, dict(B=-1), ValueError, 'requests'),
    (append, dict(k=None), ValueError, 'null pointer'),
    (append, dict(ko=ADDR), ValueError, 'together'),
    (append, dict(D=48), NotImplementedError, 'head dim'),
    (append, dict(dtype=9), ValueError, 'dtype'),
    (append, dict(k=ADDR + 8), ValueError, '16-byte'),
    (append, dict(stride=66), ValueError, '16-byte'),
    (append, dict(pool=ADDR + 4), ValueError, 'aligned'),
    (append, dict(pages=0), ValueError, 'pages'),
    (append, dict(pages=1 << 27), ValueError, 'slots'),
    (append, dict(page=2048), ValueError, 'page size'),
    (gather, dict(D=16), NotImplementedError, 'head dim'),
    (gather, dict(out=ADDR + 2), ValueError, '16-byte'),
    (gather, dict(S=-1), ValueError, 'length'),
    (gather, dict(dtype=-1), ValueError, 'dtype'),
    (attention, dict(q=None), ValueError, 'null pointer'),
    (attention, dict(H=5), ValueError, 'divisible'),
    (attention, dict(D=80), NotImplementedError, 'head dim'),
    (attention, dict(T=-1), ValueError, 'T -1'),
    (attention, dict(page=0), ValueError, 'page size'),
])
def test_calls_refused(call, kw, error, match):
    with pytest.raises(error, match=match):
        call(**kw)


def test_empty_calls_launch_nothing():
    append(T=0)
    gather(S=0)
    attention(T=0)


def test_host_entries_check_their_arguments():
    host = paged._host()
    with pytest.raises(TypeError, match='10 arguments'):
        host.paged_reserve(1, 2)
    with pytest.raises(ValueError, match='must be a tensor'):
        host.kv4_gather(1, 2, 3, 4, 5)
    with pytest.raises(ValueError, match='must be a tensor'):
        ops.kv4_append(None, None, None, None)
