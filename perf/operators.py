"""The operators that are measured: their cases, their inputs, their plain forms and their definitions in 64 bits.

  product   fp8 matrix product with one fp32 scale per row and 128 columns of the activations and one per 128 x 128
            block of the weights
  quantise  the activations' side of it: fp8 values and one scale per row and group of 128 columns
  rotate    rotary positions with several axes, alone or together with the write into the paged cache
  fork      new sequences that share their parent's full pages and get a copy of its last, partly filled one
  compact   finished sequences give their pages back, then the highest pages in use move into the lowest free ones
"""
import math

import torch

own = False

FP8_MAX = 448.0
BLOCK = 128
MIN_SCALE = 1.0 / (FP8_MAX * 512.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one new token through the q/k/v projection of 32 query and 8 kv heads of 128
        {"name": "product-1-token", "op": "product", "m": 1, "n": 6144, "k": 4096, "out": "bf16"},
        # a decode batch of 64 sequences, 64 query and 8 kv heads of 128
        {"name": "product-64-tokens", "op": "product", "m": 64, "n": 10240, "k": 8192, "out": "bf16"},
        # a ragged batch and a weight whose sizes are no multiples of the blocks
        {"name": "product-ragged", "op": "product", "m": 333, "n": 2200, "k": 4240, "out": "fp16"},
        # a prefill batch of 16384 tokens through the same projection
        {"name": "product-prefill", "op": "product", "m": 16384, "n": 10240, "k": 8192, "out": "bf16"},
        # the activations of a small decode batch
        {"name": "quantise-decode", "op": "quantise", "tokens": 7, "hidden": 4096, "dtype": "bf16"},
        # the activations of a prefill batch
        {"name": "quantise-prefill", "op": "quantise", "tokens": 16384, "hidden": 8192, "dtype": "bf16"},
        # a decode step of 64 sequences: rotate q and k, write k and v into the fp8 cache
        {"name": "rotate-decode-cache", "op": "rotate", "tokens": 64, "q_heads": 64, "kv_heads": 8, "head": 128,
         "rot": 128, "axes": 3, "neox": True, "interleaved": False, "dtype": "bf16", "cache": "fp8", "block": 16},
        # a prefill batch with images: rotate q and k
        {"name": "rotate-prefill", "op": "rotate", "tokens": 16384, "q_heads": 64, "kv_heads": 8, "head": 128,
         "rot": 128, "axes": 3, "neox": True, "interleaved": True, "dtype": "bf16", "cache": "none", "block": 16},
        # one prompt, four samples
        {"name": "fork-4", "op": "fork", "layers": 16, "blocks": 1024, "block": 16, "kv_heads": 8, "head": 128,
         "dtype": "bf16", "sequences": 8, "tokens": 1021, "parents": 1, "each": 4},
        # a batch of 64 prompts, four samples each
        {"name": "fork-256", "op": "fork", "layers": 8, "blocks": 4096, "block": 16, "kv_heads": 8, "head": 128,
         "dtype": "bf16", "sequences": 512, "tokens": 333, "parents": 64, "each": 4},
        # a cache with a few holes, between two steps; "room" is the largest number of pages one step may move
        {"name": "compact-16", "op": "compact", "layers": 16, "blocks": 1024, "block": 16, "kv_heads": 8, "head": 128,
         "dtype": "bf16", "sequences": 32, "pages": 20, "finished": 4, "moves": 16, "room": 64},
        # a cache whose pages in use have scattered over its whole range
        {"name": "compact-800", "op": "compact", "layers": 8, "blocks": 8192, "block": 16, "kv_heads": 8, "head": 128,
         "dtype": "fp8", "sequences": 256, "pages": 20, "finished": 64, "moves": 800, "room": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "quantise", "rotate", "rotate", "fork", "compact"])
    if op == "product":
        return {"op": op, "m": _log(rng, 1, 16384), "n": _log(rng, 128, 10240), "k": 16 * _log(rng, 8, 512),
                "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "quantise":
        return {"op": op, "tokens": _log(rng, 1, 16384), "hidden": 8 * _log(rng, 16, 1024),
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "rotate":
        head = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, 16384), "q_heads": kv * rng.choice([1, 4, 8]), "kv_heads": kv,
                "head": head, "rot": rng.choice([head, head // 2]), "axes": rng.choice([2, 3, 3, 4]),
                "neox": rng.random() < 0.7, "interleaved": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"]),
                "cache": rng.choice(["none", "auto", "fp8"]), "block": rng.choice([8, 16, 64])}
    common = {"op": op, "layers": rng.randint(1, 16), "blocks": _log(rng, 600, 4000), "block": rng.choice([8, 16, 32]),
              "kv_heads": rng.choice([1, 2, 4]), "head": rng.choice([64, 128]), "dtype": rng.choice(["bf16", "fp8"])}
    if op == "fork":
        parents = rng.randint(1, 16)
        each = rng.randint(1, 8)
        bs = common["block"]
        return {**common, "sequences": parents * (each + 1) + rng.randint(0, 9),
                "tokens": bs * rng.randint(0, 28) + rng.randint(1, bs - 1), "parents": parents, "each": each}
    sequences, pages = rng.randint(4, 24), rng.randint(1, 12)
    finished = rng.randint(1, sequences // 2)
    live = (sequences - finished) * pages
    moves = rng.randint(1, live)  # the room for them bounds what one step moves
    return {**common, "sequences": sequences, "pages": pages, "finished": finished, "moves": moves,
            "room": rng.choice([64, 300, max(1, moves // 2)])}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _groups(x, size):
    """[rows, columns] as [rows, groups, size], the last group filled with zeros."""
    rows, columns = x.shape
    groups = -(-columns // size)
    if groups * size != columns:
        x = torch.nn.functional.pad(x, (0, groups * size - columns))
    return x.reshape(rows, groups, size)


def _activations(tokens, hidden, g):
    """Rows of different size and a few loud channels, as a norm layer leaves them."""
    x = torch.randn(tokens, hidden, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(tokens, 1, generator=g, device="cuda"))
    loud = torch.randint(0, hidden, (max(1, hidden // 256),), generator=g, device="cuda")
    x[:, loud] *= 12.0
    return x


def _prepare_product(c, g):
    m, n, k = c["m"], c["n"], c["k"]
    x = _groups(_activations(m, k, g), BLOCK)
    a_scales = (x.abs().amax(2) / FP8_MAX).clamp(min=MIN_SCALE)
    a = (x / a_scales[:, :, None]).clamp(-FP8_MAX, FP8_MAX).reshape(m, -1)[:, :k].contiguous().to(torch.float8_e4m3fn)
    w = torch.randn(n, k, generator=g, device="cuda") * k**-0.5
    rows = -(-n // BLOCK)
    w = torch.nn.functional.pad(w, (0, 0, 0, rows * BLOCK - n))
    blocks = _groups(w, BLOCK).reshape(rows, BLOCK, -1, BLOCK)
    b_scales = (blocks.abs().amax((1, 3)) / FP8_MAX).clamp(min=MIN_SCALE)
    w = (blocks / b_scales[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).reshape(rows * BLOCK, -1)
    b = w[:n, :k].contiguous().to(torch.float8_e4m3fn)
    out = torch.empty(m, n, dtype=DTYPES[c["out"]], device="cuda")
    return {"a": a, "b": b, "a_scales": a_scales.contiguous(), "b_scales": b_scales.contiguous(), "out": out}


def _prepare_quantise(c, g):
    x = _activations(c["tokens"], c["hidden"], g).to(DTYPES[c["dtype"]])
    groups = -(-c["hidden"] // BLOCK)
    return {"x": x, "q": torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda"),
            "scales": torch.empty(x.shape[0], groups, device="cuda")}


def _sections(c):
    """How many frequencies each axis turns: about a quarter for the first one where there are three."""
    half, axes = c["rot"] // 2, c["axes"]
    if axes == 2:
        rest = [half // 2]
    elif axes == 3:
        rest = [half * 3 // 8] * 2 if not c["interleaved"] else [half * 5 // 16] * 2
    else:
        rest = [half // 5] * 3
    return [half - sum(rest)] + rest


def _axis_of(c):
    """The axis that turns each frequency."""
    s = _sections(c)
    if not c["interleaved"]:
        return [a for a, count in enumerate(s) for _ in range(count)]
    axes = len(s)
    return [i % axes if i < axes * s[i % axes] else 0 for i in range(sum(s))]


def _prepare_rotate(c, g):
    dt = DTYPES[c["dtype"]]
    t, hq, hk, d, axes = c["tokens"], c["q_heads"], c["kv_heads"], c["head"], c["axes"]
    qkv = torch.randn(t, hq + 2 * hk, d, generator=g, device="cuda").to(dt)  # as one projection leaves them
    limit = 32768
    # text runs with equal positions on all axes, and image patches whose rows and columns count from the run's start
    start = torch.randint(0, limit - 256, (t,), generator=g, device="cuda")
    steps = torch.randint(0, 256, (axes, t), generator=g, device="cuda")
    image = torch.rand(t, generator=g, device="cuda") < 0.6
    positions = torch.where(image, start + steps, start).contiguous()
    half = c["rot"] // 2
    angle = (torch.arange(limit, device="cuda", dtype=torch.float64)[:, None]
             * (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)))
    table = torch.cat([angle.cos(), angle.sin()], 1).to(dt)
    state = {"qkv": qkv, "query": qkv[:, :hq], "key": qkv[:, hq:hq + hk], "value": qkv[:, hq + hk:],
             "positions": positions, "table": table, "query_out": torch.empty(t, hq, d, dtype=dt, device="cuda"),
             "key_out": torch.empty(t, hk, d, dtype=dt, device="cuda"), "sections": _sections(c), "case": dict(c),
             "axis": torch.tensor(_axis_of(c), device="cuda")}
    if c["cache"] != "none":
        bs = c["block"]
        blocks = -(-t // bs) + 3
        kind = torch.float8_e4m3fn if c["cache"] == "fp8" else dt
        state["caches"] = torch.zeros(2, blocks, bs, hk, d, device="cuda").to(kind)
        state["slots"] = torch.randperm(blocks * bs, generator=g, device="cuda")[:t].contiguous()
        state["k_scale"] = torch.tensor(0.013, device="cuda")
        state["v_scale"] = torch.tensor(0.011, device="cuda")
    return state


def _cache_of(c, g):
    shape = (c["layers"], 2, c["blocks"], c["block"], c["kv_heads"], c["head"])
    kind = torch.bfloat16 if c["dtype"] == "bf16" else torch.uint8
    cache = torch.empty(shape, dtype=kind, device="cuda")
    for layer in cache:
        if kind is torch.uint8:  # fp8 caches are bytes
            layer.copy_(torch.randint(0, 120, layer.shape, generator=g, device="cuda", dtype=torch.uint8))
        else:
            layer.normal_(generator=g)
    return cache


def _prepare_fork(c, g):
    cache = _cache_of(c, g)
    pages = -(-c["tokens"] // c["block"])
    parents, each, rows = c["parents"], c["each"], c["sequences"]
    width = pages + 8
    order = torch.randperm(c["blocks"], generator=g, device="cuda").to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    usable = min(parents, c["blocks"] // (2 * pages))  # prompts that leave half of the pages free
    table[:usable, :pages] = order[:usable * pages].reshape(usable, pages)
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens[:usable] = c["tokens"]
    counts = torch.zeros(c["blocks"], dtype=torch.int32, device="cuda")
    counts[order[:usable * pages].long()] = 1
    n = parents * each
    first = torch.arange(n, device="cuda") // each
    return {"cache": cache, "table": table, "lens": lens, "counts": counts,
            "parents": first.clamp(max=usable - 1).to(torch.int32),
            "children": (parents + torch.arange(n, device="cuda")).to(torch.int32),
            "mapping": torch.empty(n, 2, dtype=torch.int64, device="cuda"),
            "made": torch.empty(n, dtype=torch.int32, device="cuda"), "block": c["block"]}


def _prepare_compact(c, g):
    cache = _cache_of(c, g)
    rows, pages, done, moves = c["sequences"], c["pages"], c["finished"], c["moves"]
    live = (rows - done) * pages
    blocks = c["blocks"]
    moves = min(moves, live, blocks - rows * pages)
    # `moves` of the live pages lie above the border that the live pages would fill, the others below it
    low = torch.randperm(live, generator=g, device="cuda")
    high = live + torch.randperm(blocks - live, generator=g, device="cuda")
    in_use = torch.cat([low[:live - moves], high[:moves]])
    in_use = in_use[torch.randperm(live, generator=g, device="cuda")]
    other = torch.cat([low[live - moves:], high[moves:]])[:done * pages]
    table = torch.full((rows, pages + 4), -1, dtype=torch.int32, device="cuda")
    seat = torch.randperm(rows, generator=g, device="cuda")
    table[seat[:rows - done], :pages] = in_use.reshape(rows - done, pages).to(torch.int32)
    table[seat[rows - done:], :pages] = other.reshape(done, pages).to(torch.int32)
    lens = torch.randint((pages - 1) * c["block"] + 1, pages * c["block"] + 1, (rows,), generator=g, device="cuda")
    counts = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    counts[in_use] = 1
    counts[other] = 1
    return {"cache": cache, "table": table, "lens": lens.to(torch.int32), "counts": counts,
            "finished": seat[rows - done:].to(torch.int32),
            "mapping": torch.empty(c["room"], 2, dtype=torch.int64, device="cuda"), "block": c["block"]}


def prepare(case, seed):
    make = {"product": _prepare_product, "quantise": _prepare_quantise, "rotate": _prepare_rotate,
            "fork": _prepare_fork, "compact": _prepare_compact}[case["op"]]
    state = make(case, _gen(seed))
    state["op"] = case["op"]
    return state


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _ops():
    try:
        from vllm_xpu_kernels import ops
    except ModuleNotFoundError:  # the package's folder lies beside this file's, wherever the program was started
        import os
        import sys
        sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-xpu-kernels_b200"))
        from vllm_xpu_kernels import ops
    return ops


def _own(s):
    ops = _ops()
    if s["op"] == "product":
        ops.fp8_block_scaled_mm(s["out"], s["a"], s["b"], s["a_scales"], s["b_scales"])
        return s["out"]
    if s["op"] == "quantise":
        ops.dynamic_per_token_group_scaled_fp8_quant(s["q"], s["x"], s["scales"], BLOCK)
        return s["q"], s["scales"]
    if s["op"] == "rotate":
        c = s["case"]
        if c["cache"] == "none":
            ops.multi_axis_rotary_embedding(s["positions"], s["query"], s["key"], c["head"], s["table"], c["neox"],
                                            s["sections"], c["interleaved"], s["query_out"], s["key_out"])
            return s["query_out"], s["key_out"]
        ops.multi_axis_rotary_embedding_and_cache_flash(
            s["positions"], s["query"], s["key"], s["value"], c["head"], s["table"], c["neox"], s["sections"],
            c["interleaved"], s["caches"][0], s["caches"][1], s["slots"], c["cache"], s["k_scale"], s["v_scale"],
            write_back_key=False, query_out=s["query_out"])
        return s["query_out"], s["caches"]
    keys, values = [layer[0] for layer in s["cache"]], [layer[1] for layer in s["cache"]]
    table, lens, counts = s["table"].clone(), s["lens"].clone(), s["counts"].clone()  # the step's own copies
    if s["op"] == "fork":
        ops.fork_blocks(table, lens, counts, s["parents"], s["children"], keys, values, s["block"], s["mapping"],
                        s["made"])
        return table, lens, counts, s["mapping"], s["made"], s["cache"]
    ops.free_blocks(table, lens, counts, s["finished"], s["block"])
    ops.compact_blocks(table, counts, keys, values, s["mapping"])
    return table, lens, counts, s["mapping"], s["cache"]


# ---- plain forms -------------------------------------------------------------------------------------------------
def _plain_product(s):
    k, n = s["a"].shape[1], s["b"].shape[0]
    a = s["a"].float() * s["a_scales"].repeat_interleave(BLOCK, 1)[:, :k]
    b = s["b"].float() * s["b_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    s["out"].copy_(a @ b.T)
    return s["out"]


def _plain_quantise(s):
    x = s["x"].float()
    scales = (_groups(x, BLOCK).abs().amax(2) / FP8_MAX).clamp(min=MIN_SCALE)
    inverse = (1.0 / scales).repeat_interleave(BLOCK, 1)[:, :x.shape[1]]
    s["q"].copy_((x * inverse).clamp(-FP8_MAX, FP8_MAX))
    s["scales"].copy_(scales)
    return s["q"], s["scales"]


def _turned(x, cos, sin, neox):
    half = cos.shape[-1]
    x = x.float()
    out = x.clone()
    if neox:
        first, second = x[..., :half], x[..., half:2 * half]
        out[..., :half] = first * cos - second * sin
        out[..., half:2 * half] = second * cos + first * sin
    else:
        first, second = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2] = first * cos - second * sin
        out[..., 1:2 * half:2] = second * cos + first * sin
    return out


def _plain_rotate(s):
    c = s["case"]
    half = c["rot"] // 2
    rows = s["positions"][s["axis"]].T  # the position that each frequency of each token goes by
    at = torch.arange(half, device=rows.device)
    cos, sin = s["table"][rows, at].float()[:, None], s["table"][rows, half + at].float()[:, None]
    s["query_out"].copy_(_turned(s["query"], cos, sin, c["neox"]))
    s["key_out"].copy_(_turned(s["key"], cos, sin, c["neox"]))
    if c["cache"] == "none":
        return s["query_out"], s["key_out"]
    for i, (new, scale) in enumerate(((s["key_out"], s["k_scale"]), (s["value"], s["v_scale"]))):
        page, offset = s["slots"] // c["block"], s["slots"] % c["block"]
        if c["cache"] == "fp8":
            new = (new.float() / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            s["caches"][i].view(torch.uint8)[page, offset] = new
        else:
            s["caches"][i][page, offset] = new
    return s["query_out"], s["caches"]


def _plain_fork(s):
    table, lens, counts = s["table"].clone(), s["lens"].clone(), s["counts"].clone()
    parents, children, size = s["parents"].long(), s["children"].long(), s["block"]
    n, width = parents.numel(), table.shape[1]
    length = lens[parents].long()
    full, needs = length // size, length % size != 0
    free = torch.argsort((counts > 0).to(torch.int8), stable=True)  # the free pages first, the lowest first
    rank = needs.long().cumsum(0) - needs.long()
    made = ~needs | (rank < (counts == 0).sum())
    page = free[rank.clamp(max=free.numel() - 1)]
    copies = needs & made
    column = torch.arange(width, device=table.device)[None]
    rows = table[parents].long()
    last = rows.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    shared = (column < full[:, None]) & made[:, None]
    now = torch.where(shared, rows, table[children].long())
    now = torch.where((column == full[:, None]) & copies[:, None], page[:, None], now)
    table[children] = now.to(torch.int32)
    counts.index_add_(0, rows.clamp(min=0).reshape(-1), shared.reshape(-1).to(torch.int32))
    counts.index_add_(0, page, copies.to(torch.int32))
    lens[children] = torch.where(made, length, 0).to(torch.int32)
    s["made"].copy_(torch.where(made, length, -1))
    s["mapping"].copy_(torch.where(copies[:, None], torch.stack([last, page], 1), -1))
    source, target = last.clamp(min=0), torch.where(copies, page, last.clamp(min=0))
    for layer in s["cache"]:
        layer[:, target] = layer[:, source]
    return table, lens, counts, s["mapping"], s["made"], s["cache"]


def _plain_compact(s):
    table, lens, counts = s["table"].clone(), s["lens"].clone(), s["counts"].clone()
    size, done, blocks, width = s["block"], s["finished"].long(), counts.numel(), table.shape[1]
    column = torch.arange(width, device=table.device)[None]
    pages = (lens.long() + size - 1) // size
    gone = column < pages[done][:, None]
    counts.index_add_(0, table[done].long().clamp(min=0).reshape(-1), -gone.reshape(-1).to(torch.int32))
    table[done] = torch.where(gone, -1, table[done])
    lens[done] = 0
    number = torch.arange(blocks, device=table.device)
    used = counts > 0
    border = used.sum()
    holes = torch.argsort((used | (number >= border)).to(torch.int8), stable=True)  # the lowest first
    high = used & (number >= border)
    strays = torch.argsort(high.to(torch.int8).flip(0), descending=True, stable=True)
    strays = blocks - 1 - strays  # the highest first
    moves = high.sum()
    rows = s["mapping"].shape[0]
    k = torch.arange(rows, device=table.device)
    real = k < moves
    source, target = strays[:rows], holes[:rows]
    s["mapping"].copy_(torch.where(real[:, None], torch.stack([source, target], 1), -1))
    target = torch.where(real, target, source)
    for layer in s["cache"]:
        layer[:, target] = layer[:, source]
    goes_to = number.clone()
    goes_to[source] = target
    table = torch.where(table >= 0, goes_to[table.long().clamp(min=0)].to(torch.int32), table)
    moved = counts[source].clone()
    counts[source] = torch.where(real, 0, moved)
    counts[target] = moved
    return table, lens, counts, s["mapping"], s["cache"]


def run(state):
    if own:
        return _own(state)
    return {"product": _plain_product, "quantise": _plain_quantise, "rotate": _plain_rotate, "fork": _plain_fork,
            "compact": _plain_compact}[state["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        groups = -(-k // BLOCK)
        size = 4 if c["out"] == "fp32" else 2
        return {"bytes": m * k + n * k + 4 * groups * (m + -(-n // BLOCK)) + size * m * n, "flops": 2 * m * n * k}
    if c["op"] == "quantise":
        t, h = c["tokens"], c["hidden"]
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": t * h * (size + 1) + 4 * t * -(-h // BLOCK), "flops": 3 * t * h}
    if c["op"] == "rotate":
        t, d, hq, hk = c["tokens"], c["head"], c["q_heads"], c["kv_heads"]
        moved = 2 * 2 * t * hq * d + 8 * c["axes"] * t  # q in and out, the positions
        if c["cache"] == "none":
            moved += 2 * 2 * t * hk * d
        else:
            moved += 2 * t * hk * d * (2 + (1 if c["cache"] == "fp8" else 2)) + 8 * t
        moved += 2 * c["rot"] * min(t * c["axes"], 32768)  # the table's rows, each once
        return {"bytes": moved, "flops": 3 * t * (hq + hk) * c["rot"]}
    page = 2 * c["layers"] * c["block"] * c["kv_heads"] * c["head"] * (2 if c["dtype"] == "bf16" else 1)
    if c["op"] == "fork":
        n, pages = c["parents"] * c["each"], -(-c["tokens"] // c["block"])
        usable = min(c["parents"], c["blocks"] // (2 * pages))
        free = c["blocks"] - usable * pages
        return {"bytes": 2 * page * min(n, free) + 8 * n * pages + 4 * c["blocks"] + 32 * n, "flops": 0}
    live = (c["sequences"] - c["finished"]) * c["pages"]
    moves = min(c["moves"], live, c["blocks"] - c["sequences"] * c["pages"], c["room"])
    return {"bytes": 2 * page * moves + 8 * c["blocks"] + 8 * c["sequences"] * c["pages"] + 16 * moves, "flops": 0}


# ---- definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_product(s):
    total = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    row = torch.arange(s["b"].shape[0], device="cuda") // BLOCK
    for j in range(s["a_scales"].shape[1]):
        part = slice(j * BLOCK, (j + 1) * BLOCK)
        product = s["a"][:, part].double() @ s["b"][:, part].double().T
        product *= s["a_scales"][:, j, None].double()
        product *= s["b_scales"][row, j].double()
        total += product
    return total


def _exact_quantise(s):
    x = s["x"]
    q = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    scales = torch.empty(s["scales"].shape, dtype=torch.float64, device="cuda")
    for j in range(scales.shape[1]):
        part = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        scale = torch.clamp(part.abs().max(1).values / FP8_MAX, min=1.0 / (512 * 448))
        value = torch.clamp(part / scale[:, None], -FP8_MAX, FP8_MAX)
        # e4m3: three bits behind the leading one, exponents from -6 on
        step = torch.exp2(torch.floor(torch.log2(value.abs().clamp(min=2.0**-6))) - 3)
        q[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(value / step) * step
        scales[:, j] = scale
    return q, scales


def _exact_rotate(s):
    c = s["case"]
    half, table = c["rot"] // 2, s["table"].double()
    outs = []
    for x in (s["query"], s["key"]):
        out = x.double().clone()
        for i in range(half):
            position = s["positions"][int(_axis_of(c)[i])]
            cos, sin = table[position, i][:, None], table[position, half + i][:, None]
            one, two = (i, half + i) if c["neox"] else (2 * i, 2 * i + 1)
            u, v = x[..., one].double(), x[..., two].double()
            out[..., one] = u * cos - v * sin
            out[..., two] = v * cos + u * sin
        outs.append(out)
    if c["cache"] == "none":
        return outs[0], outs[1]
    caches = s["caches"].float().double()
    flat = caches.reshape(2, -1, c["kv_heads"], c["head"])
    for i, (new, scale) in enumerate(((outs[1], s["k_scale"]), (s["value"].double(), s["v_scale"]))):
        if c["cache"] == "fp8":
            new = torch.clamp(new / scale.double(), -FP8_MAX, FP8_MAX)
            step = torch.exp2(torch.floor(torch.log2(new.abs().clamp(min=2.0**-6))) - 3)
            new = torch.round(new / step) * step
        flat[i][s["slots"]] = new
    return outs[0], flat.reshape(caches.shape)


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers and copies: nothing is computed
    state = prepare(case, seed)
    return {"product": _exact_product, "quantise": _exact_quantise, "rotate": _exact_rotate}[case["op"]](state)
