"""The plan of the block-scaled product (host only): which kernel a size uses, and that the GPU tests reach all of them."""
import ctypes

import pytest

from tests.test_gpu_block_mm_variants import SOME, VARIANTS
from vllm_xpu_kernels import cabi


@pytest.mark.parametrize("shape", VARIANTS, ids=str)
def test_the_sizes_of_the_gpu_tests_use_the_kernels_they_name(shape):
    assert cabi.fp8_block_scaled_mm_plan(*shape) == VARIANTS[shape]


def test_the_gpu_tests_reach_every_kernel():
    assert {t for t, _ in VARIANTS.values()} == {16, 32, 64, 128, 256}
    for tokens in (16, 32, 64, 128):
        splits = {s for t, s in VARIANTS.values() if t == tokens}
        assert 1 in splits and len(splits) >= 3, (tokens, splits)
    assert {VARIANTS[s][0] for s in SOME} == {16, 32, 64, 128, 256}
    # shares of the groups that are not all the same, and a short last group
    assert any(s > 1 and (-(-k // 128)) % s for (_, _, k), (_, s) in VARIANTS.items())
    assert any(k % 128 for _, _, k in VARIANTS)


def test_a_plan_is_always_one_that_can_be_launched():
    for m in (1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 700, 5000, 100000, 1 << 29):
        for n in (1, 127, 128, 129, 4096, 10240, 151936, 1 << 29):
            for k in (1, 128, 129, 1024, 8192, 1 << 29):
                tokens, splits = cabi.fp8_block_scaled_mm_plan(m, n, k)
                groups = -(-k // 128)
                assert tokens in (16, 32, 64, 128, 256) and 1 <= splits <= min(8, groups)
                share = -(-groups // splits)
                assert (splits - 1) * share < groups  # the last CTA of a cluster has work
                if tokens < 256:
                    assert -(-m // tokens) <= 65535 and -(-n // 128) * splits < 1 << 31
                assert tokens < 256 or splits == 1


def test_refusals():
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (-1, 4, 4), (1 << 31, 1, 1)):
        with pytest.raises(RuntimeError, match="out of range"):
            cabi.fp8_block_scaled_mm_plan(*sizes)
    assert cabi.lib().kvc_fp8_block_scaled_mm_plan(1, 1, 1, ctypes.POINTER(ctypes.c_int32)(), None) == 0
