"""Sizes at the end of what the kernels of a cache in 4 bits count in 32 bits, without a GPU (arrays without memory)."""
import pytest
import torch

from mini_sglang_b200 import ops


def meta_cache(pages, n_kv, page, d):
    return ops.kv4_cache(pages, n_kv, page, d, device="meta")


def test_pages_of_more_words_than_a_block_counts():
    """(They came back unwritten: a page of 2^27 tokens of 128 elements has 2^31 words.)"""
    one = torch.zeros(1, dtype=torch.int32)
    for page, d in ((1 << 27, 128), (1 << 28, 64), (1 << 26, 512), (1 << 30, 8)):
        if page * d < 1 << 33:
            with pytest.raises(ops.KernelError, match="CUDA device"):          # (nothing else is wrong)
                ops.kv4_restore(meta_cache(1, 1, page, d), one, torch.bfloat16)
        else:
            with pytest.raises(ops.KernelError, match="a page and kv head"):
                ops.kv4_restore(meta_cache(1, 1, page, d), one, torch.bfloat16)
