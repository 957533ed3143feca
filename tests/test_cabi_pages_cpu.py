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


def test_caches_without_pages_and_caches_that_differ():
    """An empty pool is a list like any other (it was an IndexError); pages that are not dense or not alike are refused."""
    _, n, pages, _, rows, nbytes, _ = cabi._cache_list([torch.zeros(0, 4, 8), torch.zeros(0, 4, 8)], ints(0))
    assert (n, pages, rows, nbytes) == (2, 0, 1, 128)
    _, n, pages, stride, rows, nbytes, _ = cabi._cache_list([torch.zeros(6, 2, 4, 8)[:, 1]], ints(6))
    assert (n, pages, stride, rows, nbytes) == (1, 6, 256, 1, 128)
    for caches in ([torch.zeros(6, 8, 4).transpose(1, 2)], [torch.zeros(6, 8), torch.zeros(6, 4)], [torch.zeros(6, 8), torch.zeros(5, 8)],
                   [torch.zeros(6, 8), torch.zeros(6, 16)[:, :8]]):
        with pytest.raises(RuntimeError, match="dense pages of the same size"):
            cabi._cache_list(caches)
