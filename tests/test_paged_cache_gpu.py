"""The model's 4-bit cache in the states that a program can bring it into: other dtypes, stopped and refused
forwards, resets, unequal lengths, every head dim.

Models, the cache of rounded values and the bar are those of `test_paged_model_gpu.py`.
"""

import pytest
import torch

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
