"""Tensors whose elements lie more than 2^31 apart, and calls that go out in several launches, for the ops without a counterpart
in the reference.  Sampled rows are compared with the same rows computed alone, which the other tests compare with definitions."""
import pytest
import torch

from vllm_xpu_kernels import ops
from vllm_xpu_kernels.fp8_quant import block_scaled_mm, scaled_fp8_group_quant

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def give_memory_back(cuda_device):
    yield
    torch.cuda.empty_cache()


def fp8(rows, columns, pad=0):
    return torch.randint(0, 0x78, (rows, columns + pad), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[:, :columns]


@pytest.mark.parametrize("m,n,k,pad", [
    (140000, 16384, 128, 0),         # the result: 2.3e9 elements
    (270000, 256, 8192, 0),          # a: 2.2e9 bytes
    (40, 270000, 8192, 0),           # b: 2.2e9 bytes, few rows of a
    (65535 * 64 + 100, 40, 48, 5),   # more row tiles than a grid has, rows of a at odd addresses
], ids=str)
def test_product(m, n, k, pad, cuda_device):
    a, b = fp8(m, k, pad), fp8(n, k)
    groups = -(-k // 128)
    sa, sb = torch.rand(m, groups, device=DEV), torch.rand(-(-n // 128), groups, device=DEV)
    out = block_scaled_mm(a, sa, b, sb)
    rows = torch.cat([torch.arange(0, min(m, 40)), torch.arange(m // 2, min(m, m // 2 + 40)), torch.arange(max(0, m - 140), m)]).unique()
    rows = rows.to(DEV)
    w = 512 if n > 512 else n
    for c0 in {0, (n // 2) // 128 * 128, (n - w) // 128 * 128}:
        some = block_scaled_mm(a[rows].contiguous(), sa[rows], b[c0:c0 + w], sb[c0 // 128:-(-(c0 + w) // 128)])
        want = out[rows, c0:c0 + w]
        # Values and scales are all positive, so the sum of absolute values is the value: both fp32 sums are within
        # (130 + G) 2^-23 of the definition.  bf16 has 8 bits: a step is 2^-7 of the power of two below, each rounding is off by
        # at most half of it, finfo.eps / 2 = 2^-8 of the value.
        half = torch.finfo(torch.bfloat16).eps / 2
        far = (some.double() - want.double()).abs() / want.double().abs()
        assert float(far.max()) <= 2 * half * 1.01 + 2 * (130 + groups) * 2.0**-23, float(far.max())


def test_quantiser(cuda_device):
    tokens, hidden = 300000, 8192
    x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device=DEV).normal_()
    q, s = scaled_fp8_group_quant(x)
    for r0 in (0, tokens // 2, tokens - 300):
        q2, s2 = scaled_fp8_group_quant(x[r0:r0 + 300].clone())
        assert torch.equal(q[r0:r0 + 300].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[r0:r0 + 300], s2)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("neox", [True, False])
def test_rotation_and_cache_write(shift, neox, cuda_device):
    """2.3e9 elements of q; one element off a boundary every pair of elements is an item of its own, so that the call goes out
    in two launches (of at most 2^31 items)."""
    tokens, hq, d = 270000, 64, 128
    if shift:
        tokens = 540000
    store = torch.empty(tokens * hq * d + 8, dtype=torch.bfloat16, device=DEV)
    query = store[shift:shift + tokens * hq * d].view(tokens, hq, d)
    query.normal_()
    key, value = torch.randn(2, tokens, 1, d, device=DEV).bfloat16()
    positions = torch.randint(0, 4000, (3, tokens), device=DEV)
    table = torch.randn(4000, d, device=DEV).bfloat16()
    pages = tokens // 16 + 1
    caches = torch.zeros(2, pages, 16, 1, d, dtype=torch.bfloat16, device=DEV)
    slots = torch.randperm(tokens, device=DEV)
    one = torch.tensor(1.0, device=DEV)
    samples = [slice(t, t + 200) for t in (0, tokens // 2, tokens - 200)]
    if shift:
        step = (2**31 - 128) // ((hq + 1) * (d // 2) + d)  # about where the second launch begins; both sides of it
        samples += [slice(t, t + 40) for t in range(step - 4000, min(step + 4000, tokens - 40), 500)]
    before = [(query[s].clone(), key[s].clone()) for s in samples]
    ops.multi_axis_rotary_embedding_and_cache_flash(positions, query, key, value, d, table, neox, (24, 20, 20), True, caches[0],
                                                    caches[1], slots, "auto", one, one, True)
    flat = caches.view(2, -1, 1, d)
    for s, (q, k) in zip(samples, before):
        ops.multi_axis_rotary_embedding(positions[:, s].contiguous(), q, k, d, table, neox, (24, 20, 20), True)
        assert torch.equal(query[s], q) and torch.equal(key[s], k)
        assert torch.equal(flat[0][slots[s]], k) and torch.equal(flat[1][slots[s]], value[s])


def test_page_copies_in_several_launches(cuda_device):
    """256 caches and more rows of the mapping than one launch has units for: rows on both sides of the border are copied."""
    caches = [torch.randint(0, 256, (64, 16), dtype=torch.uint8, device=DEV) for _ in range(256)]
    rows = 8_400_000  # times 256 caches: 2.15e9 units, a launch takes 2^31 - 2^20
    mapping = torch.full((rows, 2), -1, dtype=torch.int64, device=DEV)
    border = (2**31 - 2**20) // 256
    pairs = {0: (0, 32), 5: (1, 33), border - 1: (2, 34), border: (3, 35), border + 1: (4, 36), rows - 1: (5, 37)}
    for r, p in pairs.items():
        mapping[r] = torch.tensor(p, device=DEV)
    want = [c.clone() for c in caches]
    for w in want:
        for src, dst in pairs.values():
            w[dst] = w[src]
    ops.copy_blocks(caches[:128], caches[128:], mapping)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_pages_of_a_pool_beyond_4_gb(cuda_device):
    """Pages of 128 KB, 40000 of them: byte offsets past 2^32, by copy, fork and compaction."""
    pages, page = 40000, 128 * 1024
    cache = torch.zeros(pages, page, dtype=torch.uint8, device=DEV)
    marks = torch.randint(1, 255, (pages,), dtype=torch.uint8, device=DEV)
    cache[:, 0] = marks
    cache[:, -1] = marks
    mapping = torch.tensor([[pages - 1, 3], [7, pages - 2]], device=DEV)
    ops.copy_blocks([cache], [], mapping)
    assert cache[3, 0] == marks[-1] and cache[3, -1] == marks[-1] and cache[pages - 2, -1] == marks[7]
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    table, lens = torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints(20, 0)
    table[0, :2] = ints(pages - 5, pages - 6)
    counts = torch.zeros(pages, dtype=torch.int32, device=DEV)
    counts[[pages - 5, pages - 6]] = 1
    out, made = torch.zeros(1, 2, dtype=torch.int64, device=DEV), ints(0)
    ops.fork_blocks(table, lens, counts, ints(0), ints(1), [cache], [], 16, out, made)
    assert out.tolist() == [[pages - 6, 0]] and cache[0, 0] == marks[pages - 6] and cache[0, -1] == marks[pages - 6]
    moves = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    ops.compact_blocks(table, counts, [cache], [], moves)
    assert moves.tolist() == [[pages - 5, 1], [pages - 6, 2], [-1, -1], [-1, -1]]
    assert table[:, :2].tolist() == [[1, 2], [1, 0]] and cache[1, -1] == marks[pages - 5] and cache[2, -1] == marks[pages - 6]
