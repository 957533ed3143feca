"""The block-scaled product's bounded waits: one that runs out is seen in the status word, and the next product is right."""
import time

import pytest
import torch

from vllm_xpu_kernels import cabi
from vllm_xpu_kernels.fp8_quant import block_scaled_mm

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_a_bounded_wait_that_runs_out(cuda_device):
    """The self-test's CTA waits about a millisecond for an arrival that never comes and ends as the product's kernels would.
    Products of both kernels before it and behind it, on the same stream, have the same bits."""
    g = torch.Generator(device=DEV).manual_seed(1)

    def operands(m, n, k):
        fp8 = lambda rows: torch.randn(rows, k, generator=g, device=DEV).to(torch.float8_e4m3fn)  # noqa: E731
        groups = -(-k // 128)
        return fp8(m), torch.rand(m, groups, generator=g, device=DEV), fp8(n), torch.rand(-(-n // 128), groups, generator=g, device=DEV)

    cases = [operands(5, 400, 640), operands(64, 10240, 2048), operands(2100, 4100, 272)]
    want = [block_scaled_mm(a, sa, b, sb) for a, sa, b, sb in cases]
    assert all(bool(w.isfinite().all()) for w in want)
    assert cabi.fp8_block_scaled_mm_device_status() == 0
    try:
        t0 = time.perf_counter()
        cabi.fp8_block_scaled_mm_selftest_gives_up(50)
        got = [block_scaled_mm(a, sa, b, sb) for a, sa, b, sb in cases]
        assert cabi.fp8_block_scaled_mm_device_status() == 1  # waits for the device; the word stays raised
        assert time.perf_counter() - t0 < 5
        assert cabi.fp8_block_scaled_mm_device_status() == 1
    finally:
        cabi.fp8_block_scaled_mm_clear_device_status()
    assert cabi.fp8_block_scaled_mm_device_status() == 0
    assert cabi.paged_attention_device_status() == 0  # another library word
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("tries", [0, -1, 5001])
def test_limits(tries, cuda_device):
    with pytest.raises(RuntimeError, match="tries"):
        cabi.fp8_block_scaled_mm_selftest_gives_up(tries)
