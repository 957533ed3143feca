"""What the tensor-core kernels of the block-scaled product promise about clusters and about waits that give up, and what no run
shows: read off their source, in the order of its statements."""
import os
import re

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = os.path.join(REPO, "vllm-xpu-kernels_b200", "csrc", "fp8_block_mm_umma.cuh")


def kernel(name):
    """The kernel's body without comments."""
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("{", text.index(")", text.index(f" {name}(")))
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(name)


def test_no_cta_is_written_before_it_has_begun():
    """Distributed shared memory exists once every CTA of the cluster has begun: a cluster barrier comes before the first store
    to another CTA, and each thread that arrives on the early one also waits on it, whatever its role."""
    thin = kernel("block_mm_thin_kernel")
    first_store = min(m.start() for m in re.finditer(r"\bst_cluster4?\(", thin))
    arrive, wait = thin.index("cluster_begun_arrive()"), thin.rindex("cluster_begun_wait()", 0, first_store)
    assert arrive < wait < first_store and thin.count("cluster_begun_arrive()") == 1
    roles = re.split(r"\n  \} else (?:if \(warp >= kMmaWarp\) )?\{\n", thin[thin.index("if (warp >= kLoadWarp)"):])
    assert len(roles) >= 3 and all(r.count("cluster_begun_wait()") == 1 for r in roles[:3])
    wide = kernel("block_mm_wide_kernel")
    assert wide.index("cluster_sync()") < min(wide.index("cluster_addr("), wide.index("wide_tma_load("))


def test_nothing_is_in_flight_when_memory_is_given_back():
    """A wait can give up in any warp until the last barrier, so only behind it is it known whether copies and MMAs may still be
    under way; they are waited for there, before the tensor memory is freed and the CTA ends."""
    for name, barriers, free in (("block_mm_thin_kernel", ("__syncthreads()", "__syncthreads()"), "tmem_dealloc("),
                                 ("block_mm_wide_kernel", ("cluster_sync()", "mm_wait_limited(drained"), "tmem_dealloc_pair(")):
        body = kernel(name)
        drain, end = body.rindex("if (*abort_word) {"), body.index(free)
        # behind the last wait that can give up and a barrier of everyone; and everyone who frees memory or ends last waits for it
        last_wait = max(m.end() for m in re.finditer(r"\b(mm_wait|mbar_wait_bounded)\(", body))
        assert last_wait < body.rindex(barriers[0], 0, drain) < drain < body.rindex(barriers[1], 0, end) < end
        drains = [m.start() for m in re.finditer(r"\bmm_wait_limited\(", body)]
        assert len(drains) == 2 and all(drain < d < end for d in drains)
        commit = re.search(r"mma_commit(_pair)?\(drained\)", body)
        assert drain < commit.start() < drains[1]
    # whoever waits for the pair's drain has more patience than the drain's own waits, one per stage, can take together
    assert "mm_wait_limited(drained, 0, Cfg::kStages + 2)" in kernel("block_mm_wide_kernel")
    # the pair: one arrival for the copies and one of each issuing warp
    assert "mbar_init(drained, 3)" in kernel("block_mm_wide_kernel") and "mbar_init(drained, Cfg::kIssuers)" in kernel("block_mm_thin_kernel")


def test_lanes_leave_a_loop_together():
    """A warp that breaks out of its loop when a wait gives up does so as a whole: elect.sync and the barriers behind the loop
    need all of its lanes."""
    for name in ("block_mm_thin_kernel", "block_mm_wide_kernel"):
        body = kernel(name)
        assert re.search(r"\bmm_wait\(", body)
        for m in re.finditer(r"\bmbar_wait_bounded\(", body):  # these are statements of their own: the warp goes on
            assert re.search(r"[;{})]\s*$", body[:m.start()]) and not re.search(r"if \(!?$", body[:m.start()])


def test_results_that_could_not_be_computed_are_nan():
    """Whoever writes results looks at the abort word first, behind the last wait that they depend on: in the kernel for few rows
    after every CTA of the cluster has told the others, in the other one once per tile."""
    thin = kernel("block_mm_thin_kernel")
    tell = thin.index("st_cluster(cluster_addr(smem_addr(tmem_slot + 1), r), 1)")
    look = thin.index("const bool lost = *abort_word")
    assert tell < thin.index("cluster_sync()", tell) < look
    last_wait = max(m.end() for m in re.finditer(r"\b(mm_wait|mbar_wait_bounded)\(", thin))
    assert last_wait < tell
    stores = [m.group(0) for m in re.finditer(r"from_f32<Tout>\([^;]*;|store_words<Tout, 32>\([^;]*;", thin[look:])]
    assert len(stores) == 2 and all("lost ? " in s for s in stores)
    wide = kernel("block_mm_wide_kernel")
    additions = wide[wide.index("if (warp < 8) {"):wide.index("setmaxnreg.dec")]
    look = additions.index("if (*abort_word) {")
    waits = [m.end() for m in re.finditer(r"\b(mm_wait|mbar_wait_bounded)\(", additions)]
    assert len(waits) == 2 and max(waits) < look < additions.index("store_chunk(") < additions.index("st_if(")
