"""The paged 4-bit Chord cache's operators where they can go wrong: inputs at the edges of what the
calls take, each against the definition in 64 bits (or a plain loop).

Bars are those of `test_paged_gpu.py` unless a test derives its own.
"""

import pytest
import torch

from motif_b200 import _lib, ops
from test_paged_gpu import attention_64, close, gen, params, random_cache

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ sums of 16-bit tensors
def attention_32(q, pool, table, lens, alpha, beta, mu, ssmax):
    """Elementary operations in 32 bits, rounded once at the end."""
    most = int(lens.max())
    k, v = ops.kv4_gather(pool, table, lens, most, dtype=torch.float32)
    B, H, T, D = q.shape
    x = (q.float().view(B, k.shape[1], -1, D) @ k.transpose(-1, -2) * D ** -0.5).view(B, H, T, most)
    pos = (lens[:, None] - T + torch.arange(T, device='cuda')).view(B, 1, T, 1)
    key = torch.arange(most, device='cuda')
    alpha, beta, mu, ssmax = (p.view(1, H, 1, 1) for p in (alpha, beta, mu, ssmax))
    x = (x - alpha * ((key - pos - mu).abs() + 1e-5) ** beta) * (ssmax * torch.log(pos + 1.0))
    w = x.masked_fill(key > pos, float('-inf')).softmax(-1)
    return (w.view(B, k.shape[1], -1, most) @ v).view(B, H, T, D).to(q.dtype)


@pytest.mark.parametrize('H,kv,D,T', [(12, 3, 64, 1), (12, 3, 64, 4), (8, 4, 128, 1), (8, 2, 128, 2), (12, 3, 32, 1),
                                      (8, 2, 32, 2)])
def test_sums_of_16_bit_tensors_keep_their_bits(H, kv, D, T):
    """An error e of a sum crosses a midpoint between two neighbours of the output's type, s apart, with
    probability e / s, so the outputs that are not the correctly rounded ones count the bits of the sums:
    sums of 21 bits give at most 8 times as many as sums of 24.  (fp16; bf16 differs in nothing but the
    last rounding, which sums of 24 bits of these few thousand outputs hardly ever get wrong.)"""
    lens = [4000, 3001, 2500, 3777] * 2
    pool, table, ln = random_cache(lens, kv, D, 64, 60 + D)
    g = gen(61)
    q = torch.randn(len(lens), H, T, D, device='cuda', generator=g).half()
    alpha, beta, mu, ssmax = (torch.rand(H, device='cuda', generator=g) for _ in range(4))
    p = 0.3 + 1.2 * alpha, 0.6 * beta, 3 * mu - 1, 0.3 + 0.6 * ssmax
    want = attention_64(q, pool, table, ln, *p).half()
    wrong = (ops.kv4_chord_attention(q, pool, table, ln, *p) != want).sum()
    assert wrong <= 8 * (attention_32(q, pool, table, ln, *p) != want).sum()


# ------------------------------------------------------------------ waits that run out
@pytest.mark.parametrize('H,kv,D,T', [(12, 3, 64, 1), (16, 1, 64, 3), (8, 2, 128, 2), (4, 4, 32, 1)])
def test_rows_of_a_failed_wait_are_nan_and_counted(H, kv, D, T):
    """A CTA whose copy wait runs out (here at once, in every third CTA) leaves NaN in the rows that
    needed it, the right values in all others, and is counted; the next call is as ever."""
    lens = [(91 * i) % 700 + 1 for i in range(90)] + [9000, 0, 2, 4001]
    pool, table, ln = random_cache(lens, kv, D, 64, 62)
    q = torch.randn(len(lens), H, T, D, device='cuda', generator=gen(63)).bfloat16()
    pr = params(H, 10)
    want = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    assert _lib.wait_timeouts() == 0 and not want.isnan().any()
    with _lib.forced(_lib.FORCE_KV4_WAIT_FAILS):
        got = ops.kv4_chord_attention(q, pool, table, ln, *pr)
    ctas = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.wait_timeouts() == len(range(1, ctas, 3))
    lost = got.isnan()
    assert torch.equal(lost.any(-1), lost.all(-1))             # whole rows
    assert torch.equal(got[~lost], want[~lost])
    assert lost[90].all() and not lost[91].any()               # over many CTAs; without keys
    assert 0.2 < lost.double().mean() < 0.8
    assert torch.equal(ops.kv4_chord_attention(q, pool, table, ln, *pr), want) and _lib.wait_timeouts() == 0
