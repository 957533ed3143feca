"""The table of the multi-axis rotation at any address: the same bits, and the same accesses to the tensors."""
import pytest
import torch

from vllm_xpu_kernels import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def case(tokens, heads, d, dtype, neox, shift):
    g = torch.Generator(device=DEV).manual_seed(3)
    query = torch.randn(tokens, heads, d, generator=g, device=DEV).to(dtype)
    positions = torch.randint(0, 100, (3, tokens), generator=g, device=DEV)
    angle = torch.rand(100, d // 2, generator=g, device=DEV) * 6
    table = torch.cat([angle.cos(), angle.sin()], 1).to(dtype)
    moved = torch.empty(100 * d + 8, dtype=dtype, device=DEV)[shift:shift + 100 * d].view(100, d)
    moved.copy_(table)
    out = torch.empty_like(query)
    sections = (d // 4, d // 8, d // 8)
    return out, lambda t: ops.multi_axis_rotary_embedding(positions, query, None, d, t, neox, sections, True, out), table, moved


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shift", [1, 2, 3, 4])
def test_same_bits_at_every_address(dtype, neox, shift, cuda_device):
    for d in (8, 64, 128):
        out, rotate, table, moved = case(37, 3, d, dtype, neox, shift)
        rotate(table)
        want = out.clone()
        out.fill_(7.0)
        rotate(moved)
        assert torch.equal(out, want)


def test_the_tensors_are_still_read_in_wide_pieces(cuda_device):
    """Single elements instead of 16 bytes take several times as long; the table's address must not choose them."""
    _, rotate, table, moved = case(8192, 64, 128, torch.bfloat16, True, 1)
    took = {}
    for name, t in (("even", table), ("odd", moved)) * 4:
        rotate(t)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(5):
            rotate(t)
        end.record()
        end.synchronize()
        took[name] = min(took.get(name, 1e9), start.elapsed_time(end))
    assert took["odd"] < 1.5 * took["even"], took
