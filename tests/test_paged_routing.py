"""Which chunks attend to a 4-bit cache directly (no GPU: the rule alone; times are in its comment)."""

import pytest
import torch

from motif_b200.model import _kv4_direct


@pytest.mark.parametrize('B,H,Hkv,T,D,direct', [
    (1, 12, 3, 512, 64, True), (4, 12, 3, 256, 64, False), (64, 12, 3, 16, 64, True), (64, 12, 3, 32, 64, False),
    # the number of kv heads counts
    (4, 8, 8, 256, 64, True), (4, 8, 8, 512, 64, False), (1, 32, 8, 256, 64, True), (1, 32, 8, 512, 64, False),
    (16, 32, 8, 16, 64, True), (16, 32, 8, 32, 64, False), (1, 16, 1, 512, 64, True), (16, 16, 1, 32, 64, True),
    # and the head dim
    (4, 12, 3, 256, 32, True), (4, 12, 3, 512, 32, False), (64, 32, 8, 16, 32, False), (64, 32, 8, 8, 32, True),
])
def test_16_bit_chunks_go_the_faster_way(B, H, Hkv, T, D, direct):
    for dt in (torch.float16, torch.bfloat16):
        assert _kv4_direct(B, H, Hkv, T, D, dt) == direct


@pytest.mark.parametrize('T', [1, 256, 4096])
def test_chunks_without_a_tensor_core_prefill_kernel_are_never_read_back(T):
    for D in (32, 64, 128):
        assert _kv4_direct(64, 32, 8, T, D, torch.float32)
    assert _kv4_direct(64, 32, 8, T, 128, torch.bfloat16)


def test_chunks_that_the_direct_kernel_cannot_count_are_read_back():
    assert _kv4_direct(64, 32, 8, 4096, 128, torch.bfloat16, 32768)
    assert not _kv4_direct(64, 32, 8, 4096, 128, torch.bfloat16, 131072)
    assert not _kv4_direct(1, 32, 8, 1 << 19, 64, torch.float32, 1 << 20)
