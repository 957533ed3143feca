"""The page operations through ctypes: what they check of tensors before the library sees an address."""
import pytest
import torch

from vllm_xpu_kernels import cabi


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("pages", [7, 9])
def test_ref_counts_have_one_entry_per_page(pages):
    """The library takes the number of pages from ref_counts: with more counts than pages the copies would leave the caches."""
    caches = [torch.zeros(8, 32), torch.zeros(8, 32)]
    mapping = torch.zeros(2, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="one entry per page"):
        cabi.fork_blocks(ints(4, 4), ints(4), ints(pages), ints(2), ints(2), caches, 16, mapping, ints(2))
    with pytest.raises(RuntimeError, match="one entry per page"):
        cabi.compact_blocks(ints(4, 4), ints(pages), caches, mapping)
