"""Cases of the paged cache's operators: block tables and slot maps, writing new tokens, attention of single tokens.

A paged cache holds planes ``[blocks, block_size, heads, head_dim]`` (keys and values, or one latent plane); a
request owns the blocks that its row of a block table names, and slot ``s`` is row ``s % block_size`` of block
``s // block_size``. Operators:

* ``tables``   requests' lengths change: blocks are taken from a ring of free ones and given back to it, the new
               tokens' slots are listed
* ``append``   new tokens' keys and values -> the slots of one layer
* ``attend``   one new token a request over its tokens of one layer: softmax(scale q k) v and the log of the sum
* ``step``     the three in turn, as a decoding step calls them

Where ``own`` is false, ``run`` computes with elementary torch operations, attention in 32 bits; where it is true
it makes the framework's calls.
"""

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _tables(name, requests, held, new, block, width, finish=0.0, scarce=False):
    return {"name": name, "op": "tables", "requests": requests, "held": held, "new": new, "block": block, "width": width,
            "finish": finish, "scarce": scarce}


def _append(name, dtype, planes, heads, head_dim, tokens, block, order="NHD"):
    return {"name": name, "op": "append", "dtype": dtype, "planes": planes, "heads": heads, "head_dim": head_dim,
            "tokens": tokens, "block": block, "order": order}


def _attend(name, dtype, planes, heads, head_dim, group, requests, longest, block, order="NHD", ragged=True, empty=False,
            window=0, value_dim=0, op="attend"):
    return {"name": name, "op": op, "dtype": dtype, "planes": planes, "heads": heads, "head_dim": head_dim, "group": group,
            "requests": requests, "longest": longest, "block": block, "order": order, "ragged": ragged, "empty": empty,
            "window": window, "value_dim": value_dim or head_dim}


def listed():
    return [
        # a decoding step of 256 requests: one token each, one in sixteen needs a block
        _tables("tables decode 256", 256, 4000, 1, 16, 512),
        # a batch of prompts arrives while other requests end
        _tables("tables prompts 48", 48, 2000, 4096, 16, 512, finish=0.25),
        # a long queue is let in at once, until the free blocks run out
        _tables("tables queue 2000", 2000, 60, 1000, 32, 64, finish=0.1, scarce=True),
        # the key and value vectors of one new token of one layer of a [2, 32, T, 8, 128] cache
        _append("append one token", "bf16", 2, 8, 128, 1, 16),
        # a long prompt's vectors of that layer, pages that hold each head's tokens together
        _append("append prompt 8191", "bf16", 2, 8, 128, 8191, 64, "HND"),
        # one request over one stored chunk of 256 tokens, four query heads a key head: latency
        _attend("attend one chunk", "bf16", 2, 8, 128, 4, 1, 256, 16, ragged=False),
        # a batch being served
        _attend("attend batch 64", "bf16", 2, 8, 128, 4, 64, 4096, 16),
        # one long context: few rows, the work has to be split over its length
        _attend("attend long 131072", "bf16", 2, 8, 128, 4, 1, 131072, 16, ragged=False),
        # one rank's head of an 80-layer model in half precision, a batch padded with empty rows
        _attend("attend shard fp16", "fp16", 2, 1, 128, 8, 128, 8192, 64, "HND", empty=True),
        # a float32 cache whose vectors are no power of two long
        _attend("attend fp32 odd head", "fp32", 2, 3, 100, 2, 17, 3001, 16),
        # one shared latent vector a token in place of keys and values for each head
        _attend("attend latent 320", "bf16", 1, 1, 320, 16, 32, 4000, 64, value_dim=256),
        # a small model's decoding step, attention to the last 1024 tokens
        _attend("step small window", "bf16", 2, 8, 64, 1, 96, 2048, 16, window=1024, op="step", empty=True),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(lo * (hi / lo) ** rng.random() + rng.random()))

    op = rng.choice(["tables", "append", "attend", "attend", "attend", "step"])
    block = rng.choice([5, 8, 16, 16, 32, 48, 64])
    if op == "tables":
        new = rng.choice([1, 1, log(2, 2000)])
        requests, held = log(1, 2000), log(1, 4000)
        requests = max(1, min(requests, 1000 * 2000 // new))
        case = _tables("", requests, held, new, block, -(-(held + new) // block) + rng.randrange(0, 9),
                       rng.choice([0.0, 0.2]), rng.random() < 0.25)
    else:
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        order = rng.choice(["NHD", "HND"])
        planes = rng.choice([1, 2, 2, 2])
        heads = rng.choice([1, 2, 3, 4, 8, 8, 16]) if planes == 2 else 1
        sizes = [64, 80, 96, 112, 128, 128, 192, 256, rng.randrange(17, 257)] if planes == 2 else [128, 192, 256, 320, 576]
        head_dim = rng.choice(sizes)
        if op == "append":
            case = _append("", dtype, planes, heads, head_dim, log(1, (1 << 23) // (heads * head_dim)), block, order)
        else:
            group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 12, 16])
            requests = log(1, 256)
            most = (1 << 26) // (requests * heads * head_dim)   # half the longest case, with every row padded to the longest
            case = _attend("", dtype, planes, heads, head_dim, group, requests, log(1, max(2, min(65536, most))), block, order,
                           rng.random() < 0.8, rng.random() < 0.3, rng.choice([0, 0, 0, log(16, 2048)]),
                           rng.randrange(head_dim // 2, head_dim + 1) if planes == 1 else 0, op)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs


def _spread(lo, hi, count, salt):
    """`count` whole numbers spread over the logarithm of lo..hi: the case's own, whatever the seed."""
    rng = random.Random(salt * 1000003 + count * 31 + hi)
    return [min(hi, int(lo * (hi / lo) ** rng.random() + rng.random())) for _ in range(count)]


def _lengths(case):
    """Tokens that each request attends to; in a step the new one among them."""
    n, longest = case["requests"], case["longest"]
    lengths = _spread(1, longest, n, 1) if case["ragged"] else [longest] * n
    lengths[0] = longest
    if case["empty"]:
        lengths[n - n // 8:] = [0] * (n // 8)
    return lengths


def _changes(case):
    """(held, length) of each request of a ``tables`` case."""
    n = case["requests"]
    held = _spread(1, case["held"], n, 2)
    new = _spread(1, case["new"], n, 3)
    ends = random.Random(4 * n + case["held"])
    return [(h, 0 if ends.random() < case["finish"] else h + t) for h, t in zip(held, new)]


def _ceil(a, b):
    return -(-a // b)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _paged(state, case, held, lengths, g):
    """Tables of the blocks that requests hold, and the ring of the free ones, at some place of the ring."""
    block, width = case["block"], state["width"]
    n = len(held)
    need = sum(max(0, _ceil(x, block) - _ceil(h, block)) for h, x in zip(held, lengths))
    owned = sum(_ceil(h, block) for h in held)
    free = need * 3 // 4 if case.get("scarce") else need + 9
    blocks = owned + free
    state["blocks"] = blocks
    names = torch.randperm(blocks, generator=g, device="cuda").int()
    h = _ints([_ceil(x, block) for x in held])
    col = torch.arange(width, device="cuda")
    start = h.cumsum(0) - h
    at = (start.unsqueeze(1) + col).clamp(max=max(0, blocks - 1))
    # what lies behind a request's blocks is left over from other requests
    state["tables"] = torch.where(col < h.unsqueeze(1), names[at], names.flip(0)[at]).contiguous()
    first = blocks // 3
    ring = torch.full((blocks,), -7, dtype=torch.int32, device="cuda")
    ring[(first + torch.arange(free, device="cuda")) % blocks] = names[owned:]
    state["free"], state["cursor"] = ring, _ints([first, free])
    state["held"], state["lengths"] = _ints(held), _ints(lengths)
    state["kept"], state["cursor_after"] = torch.zeros(n, dtype=torch.int32, device="cuda"), _ints([0, 0])
    state["starts"] = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    state["slots"] = torch.zeros(state["capacity"], dtype=torch.int64, device="cuda")


def _cache(case, blocks, g):
    """One layer [planes, blocks, block, heads, head_dim] of random values."""
    shape = (case["planes"], blocks, case["block"], case["heads"], case["head_dim"])
    # channels of keys differ in size by an order of magnitude
    channel = torch.exp(0.7 * torch.randn((case["planes"], 1, 1, case["heads"], case["head_dim"]), generator=g, device="cuda"))
    if case["order"] == "HND":
        layer = torch.empty((shape[0], blocks, case["heads"], case["block"], case["head_dim"]), dtype=DTYPES[case["dtype"]],
                            device="cuda").transpose(2, 3)
    else:
        layer = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda")
    for k in range(case["planes"]):
        layer[k] = torch.randn(shape[1:], generator=g, device="cuda") * channel[k]
    return layer


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    state = {"case": case}
    op = case["op"]
    if op == "tables":
        changes = _changes(case)
        order.shuffle(changes)
        held, lengths = [h for h, _ in changes], [x for _, x in changes]
        state["width"] = max(case["width"], _ceil(case["held"] + case["new"], case["block"]))
        state["capacity"] = sum(max(0, x - h) for h, x in changes) + 7
        _paged(state, case, held, lengths, g)
    elif op == "append":
        tokens, block = case["tokens"], case["block"]
        blocks = _ceil(tokens, block) * 5 // 4 + 2
        state["layer"] = _cache(case, blocks, g)
        pages = torch.randperm(blocks, generator=g, device="cuda")[:_ceil(tokens, block)]
        state["slots"] = (pages.unsqueeze(1) * block + torch.arange(block, device="cuda")).flatten()[:tokens]
    else:
        lengths = _lengths(case)
        real = lengths[:len(lengths) - len(lengths) // 8] if case["empty"] else lengths
        order.shuffle(real)
        lengths = real + lengths[len(real):]
        held = [max(0, x - 1) for x in lengths] if op == "step" else lengths
        state["width"] = _ceil(case["longest"], case["block"]) + 3
        state["capacity"] = case["requests"]
        _paged(state, case, held, lengths, g)
        state["layer"] = _cache(case, state["blocks"], g)
        dtype, q = DTYPES[case["dtype"]], case["heads"] * case["group"]
        state["query"] = torch.randn((case["requests"], q, case["head_dim"]), generator=g, device="cuda").to(dtype)
        state["out"] = torch.zeros((case["requests"], q, case["value_dim"]), dtype=dtype, device="cuda")
        state["lse"] = torch.zeros((case["requests"], q), dtype=torch.float32, device="cuda")
        if op == "attend":
            # rows of a request's last block behind its tokens hold whatever was there before
            ends = [(r, x) for r, x in enumerate(lengths) if x % case["block"]]
            if ends:
                rows = _ints([r for r, _ in ends], torch.int64)
                last = state["tables"][rows, _ints([x // case["block"] for _, x in ends], torch.int64)].long()
                row = torch.arange(case["block"], device="cuda")
                stale = row >= _ints([x % case["block"] for _, x in ends]).unsqueeze(1)
                there = state["layer"][:, last]
                state["layer"][:, last] = torch.where(stale[None, :, :, None, None], float("nan"), there)
    if op in ("append", "step"):
        shape = (len(state["slots"]), case["heads"], case["head_dim"])
        parts = [torch.randn(shape, generator=g, device="cuda").to(DTYPES[case["dtype"]]) for _ in range(case["planes"])]
        state["keys"], state["values"] = parts[0], parts[-1] if case["planes"] == 2 else None
    if own:
        from confkv_b200.gpu_aesgcm import GpuAesGcmLibrary
        from confkv_b200.kv_codec import KvCodec, PagedKvCache
        from confkv_b200.kv_paged import KvAttention, KvBlockTables

        lib, device = GpuAesGcmLibrary(), torch.cuda.current_device()
        if "tables" in state:
            state["block_tables"] = KvBlockTables(lib, blocks=state["blocks"], block_size=case["block"], device=device)
        if "layer" in state:
            codec = KvCodec(lib, "int8", DTYPES[case["dtype"]], planes=case["planes"], layers=1, heads=case["heads"],
                            head_dim=case["head_dim"], device=device)
            state["attention"] = KvAttention(lib, PagedKvCache(codec, [state["layer"]]),
                                             query_heads=case["heads"] * case.get("group", 1),
                                             value_dim=case.get("value_dim"), window=case.get("window", 0))
            state["workspace"] = state["attention"].workspace()
    return state


# ------------------------------------------------------------------ one pass


def _resize(state, block):
    """The tables, the ring, what requests hold, the cursor, the slots and where each request's start."""
    held, lengths, tables, ring = (state[k].long() for k in ("held", "lengths", "tables", "free"))
    first, count = state["cursor"].long().unbind()
    cap, width, capacity = len(ring), tables.shape[1], len(state["slots"])
    before, after = (held + block - 1) // block, (lengths + block - 1) // block
    take, tokens = (after - before).clamp(min=0), (lengths - held).clamp(min=0)
    refused = ((take.cumsum(0) > count) | (tokens.cumsum(0) > capacity)).cumsum(0) > 0
    refused &= lengths > held
    kept = torch.where(refused, held, lengths)
    take, tokens = torch.where(refused, 0, take), torch.where(refused, 0, tokens)
    give = (before - after).clamp(min=0)
    col = torch.arange(width, device="cuda")
    old, new = before.unsqueeze(1), after.unsqueeze(1)
    # given back: a place behind the ring's end, in turn; all others go to a place of their own that is cut off
    place = (first + count + (give.cumsum(0) - give).unsqueeze(1) + col - new) % max(1, cap)
    place = torch.where((col >= new) & (col < old), place, cap)
    ring_after = torch.cat((ring, ring[:1])).scatter(0, place.flatten(), tables.flatten())[:cap]
    source = ring[(first + (take.cumsum(0) - take).unsqueeze(1) + col - old) % max(1, cap)]
    taken = (col >= old) & (col < old + take.unsqueeze(1))
    tables = torch.where(taken, source, tables)
    starts = torch.cat((tokens.new_zeros(1), tokens.cumsum(0)))
    i = torch.arange(capacity, device="cuda")
    r = torch.searchsorted(starts[1:], i, right=True).clamp(max=len(held) - 1)
    at = (held[r] + i - starts[r]).clamp(max=width * block - 1)
    slots = torch.where(i < starts[-1], tables[r, at // block] * block + at % block, -1)
    cursor = torch.stack(((first + take.sum()) % max(1, cap), count - take.sum() + give.sum()))
    return {"tables": tables.int(), "free": ring_after.int(), "kept": kept.int(), "cursor": cursor.int(), "slots": slots,
            "starts": starts}


def _write(state, slots, block):
    """The new vectors in their slots; a slot below 0 is none."""
    layer = state["layer"]
    keep = slots >= 0
    # where there is no slot, the first slot's vector is written once more
    at = torch.where(keep, slots, slots[0])
    keep = keep[:, None, None]
    layer[0][at // block, at % block] = torch.where(keep, state["keys"], state["keys"][:1])
    if state["values"] is not None:
        layer[1][at // block, at % block] = torch.where(keep, state["values"], state["values"][:1])
    return layer


def _attention(state, tables, lengths):
    case = state["case"]
    block, group, dim = case["block"], case["group"], case["head_dim"]
    pos = torch.arange(case["longest"], device="cuda")
    low = (lengths - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(lengths)
    there = (pos < lengths.unsqueeze(1)) & (pos >= low.unsqueeze(1))                  # [n, L]
    page = torch.where(there, tables.long()[:, pos // block], 0)
    row = (pos % block).expand_as(page)
    mask = there[:, :, None, None]
    k = torch.where(mask, state["layer"][0][page, row], 0).float()                   # [n, L, heads, d]
    v = torch.where(mask, state["layer"][-1][page, row], 0).float()[..., :case["value_dim"]]
    q = state["query"].float().unflatten(1, (case["heads"], group))                  # [n, heads, group, d]
    s = torch.einsum("nhgd,nlhd->nhgl", q, k) * dim ** -0.5
    s = torch.where(there[:, None, None, :], s, -torch.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0, m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("nhgl,nlhd->nhgd", p, v) / torch.where(total == 0, 1, total)
    lse = (m + torch.log(total)).squeeze(-1)
    return {"out": out.flatten(1, 2).to(DTYPES[case["dtype"]]), "lse": lse.flatten(1, 2)}


def _run_own(case, state):
    attention = state.get("attention")
    if case["op"] in ("tables", "step"):
        state["block_tables"].resize(state["tables"], state["held"], state["lengths"], state["free"], state["cursor"],
                                     kept=state["kept"], cursor_after=state["cursor_after"], slots=state["slots"],
                                     starts=state["starts"])
        tables = {"tables": state["tables"], "free": state["free"], "kept": state["kept"], "cursor": state["cursor_after"],
                  "slots": state["slots"], "starts": state["starts"]}
        if case["op"] == "tables":
            return tables
    if case["op"] in ("append", "step"):
        attention.append(0, state["slots"], state["keys"], state["values"])
        if case["op"] == "append":
            return state["layer"]
    attention.attend(0, state["query"], state["tables"], state["kept"] if case["op"] == "step" else state["lengths"],
                     state["out"], lse=state["lse"], workspace=state["workspace"])
    out = {"out": state["out"], "lse": state["lse"]}
    return {**tables, "layer": state["layer"], **out} if case["op"] == "step" else out


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "tables":
        return _resize(state, case["block"])
    if case["op"] == "append":
        return _write(state, state["slots"], case["block"])
    if case["op"] == "attend":
        return _attention(state, state["tables"], state["lengths"])
    tables = _resize(state, case["block"])
    layer = _write(state, tables["slots"], case["block"])
    return {**tables, "layer": layer, **_attention(state, tables["tables"], tables["kept"])}


def work(case):
    op = case["op"]
    moved = flops = 0
    if op in ("tables", "step"):
        if op == "tables":
            changes = _changes(case)
        else:
            changes = [(max(0, x - 1), x) for x in _lengths(case)]
        blocks = sum(abs(_ceil(x, case["block"]) - _ceil(h, case["block"])) for h, x in changes)
        tokens = sum(max(0, x - h) for h, x in changes)
        # held and length in, kept and start out; a block's name in and out; a slot out
        moved += 20 * len(changes) + 8 * blocks + 8 * tokens
        flops += 4 * len(changes) + 2 * tokens
    if op == "tables":
        return {"bytes": moved, "flops": flops}
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    vectors = case["planes"] * case["heads"] * case["head_dim"] * size
    if op in ("append", "step"):
        tokens = case["tokens"] if op == "append" else sum(x > 0 for x in _lengths(case))
        moved += tokens * (2 * vectors + 8)
    if op == "append":
        return {"bytes": moved, "flops": 1}
    seen = [min(x, case["window"]) if case["window"] else x for x in _lengths(case)]
    heads, values = case["heads"] * case["group"], case["value_dim"]
    moved += sum(seen) * vectors + 4 * sum(_ceil(x, case["block"]) for x in seen)
    moved += case["requests"] * (heads * (case["head_dim"] + values) * size + 4 * heads + 4)
    flops += 2 * sum(seen) * heads * (case["head_dim"] + values)
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    if case["op"] == "tables":
        return None                                     # whole numbers
    state = prepare(case, seed)
    block = case["block"]
    layer, result = state["layer"].double(), {}
    if case["op"] == "append":
        slots = state["slots"].tolist()
    else:
        tables, lengths = state["tables"].tolist(), state["lengths"].tolist()
    if case["op"] == "step":
        ring, (first, _) = state["free"].tolist(), state["cursor"].tolist()
        slots = []
        for r, x in enumerate(lengths):
            if x and (x - 1) % block == 0:
                tables[r][(x - 1) // block] = ring[first % len(ring)]
                first += 1
            if x:
                slots.append(tables[r][(x - 1) // block] * block + (x - 1) % block)
        result = dict.fromkeys(("tables", "free", "kept", "cursor", "slots", "starts"))
    if case["op"] in ("append", "step"):
        for i, s in enumerate(slots):
            layer[0, s // block, s % block] = state["keys"][i].double()
            if case["planes"] == 2:
                layer[1, s // block, s % block] = state["values"][i].double()
        if case["op"] == "append":
            return layer
        result["layer"] = layer
    n, heads, group = case["requests"], case["heads"], case["group"]
    out = torch.zeros((n, heads * group, case["value_dim"]), dtype=torch.float64, device="cuda")
    lse = torch.full((n, heads * group), -torch.inf, dtype=torch.float64, device="cuda")
    for r in range(n):
        low = max(0, lengths[r] - case["window"]) if case["window"] else 0
        if lengths[r] == 0:
            continue
        pages = _ints(tables[r][low // block:_ceil(lengths[r], block)], torch.int64)
        cut = slice(low - low // block * block, lengths[r] - low // block * block)
        k = layer[0][pages].flatten(0, 1)[cut]
        v = layer[-1][pages].flatten(0, 1)[cut]
        for h in range(heads):
            mine = slice(h * group, (h + 1) * group)
            s = state["query"][r, mine].double() @ k[:, h].T / case["head_dim"] ** 0.5
            lse[r, mine] = torch.logsumexp(s, -1)
            out[r, mine] = torch.softmax(s, -1) @ v[:, h, :case["value_dim"]]
    return {**result, "out": out, "lse": lse}
