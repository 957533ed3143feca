"""Every kernel of the block-scaled product, by the plan's word: each token tile, alone and with its groups divided over clusters
of several sizes (the last share shorter than the others), and the pairs of CTAs, in both fp8 types, with padded operands, scales
stored column by column, odd result rows, NaN and infinities, on two streams and in a graph.  Tolerances: test_gpu_block_mm."""
import pytest
import torch

from tests.test_gpu_block_mm import DEV, check, no_wait_gave_up, operands  # noqa: F401  (a fixture for every test here)
from vllm_xpu_kernels import cabi, ops
from vllm_xpu_kernels.fp8_quant import block_scaled_mm, scaled_fp8_group_quant

pytestmark = pytest.mark.gpu

# (m, n, k): (rows of a per tile, CTAs that divide a tile's groups)
VARIANTS = {
    (3, 700, 1104): (16, 5), (1, 130, 8208): (16, 8), (16, 6144, 2064): (16, 2), (33, 6144, 1040): (16, 1),
    (24, 8192, 4112): (32, 2), (64, 8192, 1168): (32, 1), (17, 3443, 4112): (32, 4), (100, 130, 4112): (32, 7),
    (64, 10240, 2064): (64, 3), (40, 10239, 2176): (64, 3), (48, 8192, 8208): (64, 4), (63, 3443, 14464): (64, 5),
    (63, 4096, 14464): (64, 8), (50, 5574, 8336): (64, 6), (37, 14336, 1040): (64, 1), (60, 14330, 4112): (64, 2),
    (96, 4096, 2064): (128, 4), (100, 8192, 2064): (128, 2), (65, 10240, 1168): (128, 1), (120, 10240, 8208): (128, 3),
    (100, 1000, 8208): (128, 8),
    (2101, 4100, 144): (256, 1), (2180, 4355, 1104): (256, 1), (300, 20000, 656): (256, 1), (2049, 5000, 48): (256, 1),
}
SOME = [(3, 700, 1104), (17, 3443, 4112), (40, 10239, 2176), (63, 3443, 14464), (96, 4096, 2064), (2101, 4100, 144), (2180, 4355, 1104)]


@pytest.mark.parametrize("shape", VARIANTS, ids=str)
@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_values(shape, kind, cuda_device):
    m, n, k = shape
    assert cabi.fp8_block_scaled_mm_plan(m, n, k) == VARIANTS[shape]
    a, b, sa, sb = operands(m, n, k, kind=kind, seed=k)
    if kind == "e5m2":
        sa = sa * 1e-4
    for out in (torch.float32, torch.bfloat16):
        result = torch.full((m, n), float("nan"), dtype=out, device=DEV)
        ops.fp8_block_scaled_mm(result, a, b, sa, sb)
        check(result, a, b, sa, sb)
        again = torch.full_like(result, float("nan"))
        ops.fp8_block_scaled_mm(again, a, b, sa, sb)
        assert torch.equal(result, again)


@pytest.mark.parametrize("shape", SOME, ids=str)
@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_strides_and_untouched_memory(shape, kind, cuda_device):
    m, n, k = shape
    a, b, sa, sb = operands(m, n, k, kind=kind, a_pad=16, b_pad=48)
    if kind == "e5m2":
        sa = sa * 1e-4
    columns = sa.t().contiguous().t()
    wide = torch.zeros(m + 3, 2 * sa.shape[1], device=DEV)[3:, ::2]  # neither rows nor columns next to each other
    wide.copy_(sa)
    for scales in (columns, wide):
        for left, extra, dtype in ((8, 24, torch.bfloat16), (3, 20, torch.bfloat16), (1, 21, torch.float16), (1, 24, torch.float32)):
            x = scales * 1e-3 if dtype == torch.float16 else scales
            store = torch.full((m + 2, n + extra), 5.0, dtype=dtype, device=DEV)
            result = store[1:m + 1, left:left + n]
            ops.fp8_block_scaled_mm(result, a, b, x, sb.t().contiguous().t())
            check(result, a, b, x, sb)
            result.fill_(5.0)
            assert bool((store == 5.0).all())


@pytest.mark.parametrize("shape", SOME, ids=str)
def test_rows_do_not_mix(shape, cuda_device):
    """NaN and infinite values and scales stay in their row of a, column of b, or block of 128 columns."""
    m, n, k = shape
    a, b, sa, sb = operands(m, n, k)
    clean, got = torch.empty(m, n, device=DEV), torch.empty(m, n, device=DEV)
    ops.fp8_block_scaled_mm(clean, a, b, sa, sb)
    rows, columns = torch.arange(m, device=DEV), torch.arange(n, device=DEV)
    for row in (0, m // 2, m - 1):
        a_bad = a.clone()
        a_bad.view(torch.uint8)[row, k - 1] = 0x7F
        ops.fp8_block_scaled_mm(got, a_bad, b, sa, sb)
        assert bool(got[row].isnan().all()) and torch.equal(got[rows != row], clean[rows != row])
        sa_bad = sa.clone()
        sa_bad[row, -1] = float("inf")
        ops.fp8_block_scaled_mm(got, a, b, sa_bad, sb)
        assert not bool(got[row].isfinite().any()) and torch.equal(got[rows != row], clean[rows != row])
    for column in (0, n // 2, n - 1):
        b_bad = b.clone()
        b_bad.view(torch.uint8)[column, 0] = 0xFF
        ops.fp8_block_scaled_mm(got, a, b_bad, sa, sb)
        assert bool(got[:, column].isnan().all()) and torch.equal(got[:, columns != column], clean[:, columns != column])
    sb_bad = sb.clone()
    sb_bad[-1, 0] = float("nan")
    ops.fp8_block_scaled_mm(got, a, b, sa, sb_bad)
    last = columns // 128 == (n - 1) // 128
    assert bool(got[:, last].isnan().all()) and torch.equal(got[:, ~last], clean[:, ~last])


def test_every_kernel_on_two_streams(cuda_device):
    """All variants at the same time on two streams, in opposite order: the same bits as one after the other."""
    cases = [operands(m, n, k, seed=i) for i, (m, n, k) in enumerate(VARIANTS)]
    alone = [block_scaled_mm(a, sa, b, sb) for a, b, sa, sb in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[i].append([block_scaled_mm(a, sa, b, sb) for a, b, sa, sb in (cases if i == 0 else cases[::-1])])
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in results[i]:
            assert all(torch.equal(x, y) for x, y in zip(r, alone if i == 0 else alone[::-1]))


@pytest.mark.parametrize("shape", SOME, ids=str)
def test_quantise_and_multiply_in_a_graph(shape, cuda_device):
    """The pair as a projection runs it (scales column by column), captured once and replayed on new activations; and against
    the definition on the quantised values."""
    m, n, k = shape
    _, b, _, sb = operands(m, n, k, seed=2)
    x = torch.randn(m, k, device=DEV).bfloat16()
    scaled_fp8_group_quant(x)
    block_scaled_mm(*scaled_fp8_group_quant(x), b, sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = scaled_fp8_group_quant(x)
        out = block_scaled_mm(q, s, b, sb)
    for i in range(3):
        x.copy_(torch.randn(m, k, device=DEV) * 3**i)
        graph.replay()
        check(out, q, b, s, sb)
        q2, s2 = scaled_fp8_group_quant(x)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
        assert torch.equal(out, block_scaled_mm(q2, s2, b, sb))
