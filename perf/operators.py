"""Cases of the KV-cache codec: quantising KV objects as they are stored, and reading them back.

A stored object is a record of codes and scales in one of three formats:

* ``int8``   one float32 scale a vector of ``head_dim`` values: s = amax / 127, code = round(x * 127 / amax)
* ``fp8``    the same with e4m3 codes: s = amax / 448, code = e4m3(x * 448 / amax)
* ``mxfp4``  e2m1 codes with one power of two a block of 32 values: e = floor(log2 amax) - 2, code = e2m1(x / 2^e)

A request's tokens are cut into chunks (the last one may be short) and every chunk becomes one
object ``[planes, layers, tokens, heads, head_dim]``. Operators:

* ``write``      objects -> records
* ``read``       records -> objects
* ``page_out``   tokens of a paged cache, found through their slots -> records
* ``page_in``    records -> the slots of a paged cache; the other slots keep their values
* ``roundtrip``  ``write`` and then ``read``: how 4-bit codes are seen as the values they stand for

Where ``own`` is false, ``run`` computes with elementary torch operations (in 64 bits up to the
rounding to a code: values may lie next to a border); where it is true it makes the framework's calls.
"""

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADER = 32
BLOCK = 32  # values that share one mxfp4 scale


def _case(name, op, fmt, dtype, planes, layers, heads, head_dim, tokens, chunk=256, block=16, order="NHD", skip=0):
    return {"name": name, "op": op, "fmt": fmt, "dtype": dtype, "planes": planes, "layers": layers, "heads": heads,
            "head_dim": head_dim, "tokens": tokens, "chunk": chunk, "block": block, "order": order, "skip": skip}


def listed():
    return [
        # the key and value vectors of one new token of an [2, 32, T, 8, 128] cache: launch latency
        _case("write int8 one token", "write", "int8", "bf16", 2, 32, 8, 128, 1),
        # the benchmarked batch, 32 chunks of 256 tokens, 1 GiB: a long prompt or a flush of the cache
        _case("write int8 32 chunks", "write", "int8", "bf16", 2, 32, 8, 128, 8192),
        # one rank's head of an 80-layer cache, three whole chunks and a short one, in half precision
        _case("write fp8 ragged fp16", "write", "fp8", "fp16", 2, 80, 1, 128, 1000),
        # a cache in float32 whose vectors are no power of two long
        _case("write int8 fp32 odd head", "write", "int8", "fp32", 2, 4, 3, 100, 1777),
        # a prefix hit on one chunk
        _case("read int8 one chunk", "read", "int8", "bf16", 2, 32, 8, 128, 256),
        # a prefix hit on a long prompt, stored in 4 bits
        _case("read mxfp4 16 chunks", "read", "mxfp4", "bf16", 2, 32, 8, 128, 4096),
        # a small model's 2 MiB objects, stored in 4 bits and read back
        _case("roundtrip mxfp4 small", "roundtrip", "mxfp4", "bf16", 2, 4, 8, 64, 4096),
        # one shared latent vector a token in place of keys and values for each head
        _case("roundtrip fp8 latent", "roundtrip", "fp8", "bf16", 1, 32, 1, 320, 3001),
        # a finished prompt goes from the paged cache to the store, pages of 16 tokens
        _case("page out int8 prompt", "page_out", "int8", "bf16", 2, 32, 8, 128, 4096),
        # one token out of a paged cache whose pages hold each head's tokens together
        _case("page out fp8 one token", "page_out", "fp8", "bf16", 2, 32, 8, 128, 1, 256, 64, "HND"),
        # a stored prompt comes back into pages of 64 tokens; its first tokens are there already
        _case("page in fp8 prompt", "page_in", "fp8", "fp16", 2, 32, 8, 128, 2051, 256, 64, "HND", 130),
        # 4-bit records with a head size between two powers of two into pages of 16 tokens
        _case("page in mxfp4 prompt", "page_in", "mxfp4", "bf16", 2, 16, 8, 96, 1024),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, int(lo * (hi / lo) ** rng.random() + rng.random()))

    op = rng.choice(["write", "read", "roundtrip", "page_out", "page_in"])
    # a write returns its codes as numbers, which 4-bit codes are not: they are seen through a round trip
    fmt = rng.choice(["int8", "fp8"] if op in ("write", "page_out") else ["int8", "fp8", "mxfp4", "mxfp4"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    head_dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256, 320, rng.randrange(17, 257)])
    planes = rng.choice([1, 2, 2, 2])
    layers, heads = log(1, 80), rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    chunk = rng.choice([16, 64, 100, 256, 256, 256])
    # from one token up to 2^26 values, a quarter of a GiB in float32
    most = max(1, min(chunk * 200, (1 << 26) // (planes * layers * heads * head_dim)))
    tokens = log(1, most)
    block = rng.choice([8, 16, 16, 32, 64, 48])
    skip = rng.choice([0, 0, rng.randrange(0, tokens)]) if op in ("page_out", "page_in") else 0
    case = _case("", op, fmt, dtype, planes, layers, heads, head_dim, tokens, chunk, block, rng.choice(["NHD", "HND"]), skip)
    del case["name"]
    return case


# ------------------------------------------------------------------ records


def _record(case, tokens):
    """(vectors, code bytes a vector, where the scales start, scale bytes, record bytes)."""
    d = case["head_dim"]
    vectors = case["planes"] * case["layers"] * tokens * case["heads"]
    code = (d + 1) // 2 if case["fmt"] == "mxfp4" else d
    scale = vectors * (-(-d // BLOCK) if case["fmt"] == "mxfp4" else 4)
    at = HEADER + -(-vectors * code // 16) * 16
    return vectors, code, at, scale, at + -(-scale // 16) * 16


def _parts(case):
    """(objects, tokens each) of the whole chunks and of the short last one."""
    full, rest = divmod(case["tokens"], case["chunk"])
    return [(n, t) for n, t in ((full, case["chunk"]), (1, rest)) if n and t]


def _code_view(case, record, tokens):
    vectors, code, _, _, _ = _record(case, tokens)
    raw = record[:, HEADER:HEADER + vectors * code]
    raw = raw if case["fmt"] == "mxfp4" else raw.view(torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn)
    shape = (case["planes"], case["layers"], tokens, case["heads"], code)
    return raw.unflatten(1, shape)


def _scale_view(case, record, tokens):
    _, _, at, scale, _ = _record(case, tokens)
    raw = record[:, at:at + scale]
    per = () if case["fmt"] != "mxfp4" else (-(-case["head_dim"] // BLOCK),)
    raw = raw if case["fmt"] == "mxfp4" else raw.view(torch.float32)
    return raw.unflatten(1, (case["planes"], case["layers"], tokens, case["heads"], *per))


def _blocks(x, d):
    """[..., d] -> [..., blocks of 32], zeros behind the last value."""
    return torch.nn.functional.pad(x, (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))


def _to_minifloat(y, mantissa, lowest, top):
    """The nearest value with `mantissa` bits after the leading one and exponents from `lowest`, ties to even, at most `top`."""
    exponent = torch.frexp(y)[1] - 1
    step = torch.ldexp(torch.ones_like(y), exponent.clamp(min=lowest) - mantissa)
    return (torch.round(y / step) * step).clamp(-top, top)


def _quantise(case, x):
    """Codes and scales of x [..., head_dim] in the plain form."""
    x = x.double()
    if case["fmt"] == "mxfp4":
        b = _blocks(x, case["head_dim"])
        amax = b.abs().amax(-1)
        e = torch.where(amax > 0, (torch.frexp(amax)[1] - 1 - 2).clamp(min=-127), torch.full_like(amax, -127)).int()
        v = _to_minifloat(torch.ldexp(b, -e.unsqueeze(-1)), 1, 0, 6.0).flatten(-2)[..., :case["head_dim"]]
        code = torch.round(torch.where(v.abs() < 2, v.abs() * 2, torch.where(v.abs() < 4, v.abs() + 2, v.abs() / 2 + 4)))
        code = code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
        code = torch.nn.functional.pad(code, (0, -case["head_dim"] % 2))
        return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)
    top = 127.0 if case["fmt"] == "int8" else 448.0
    amax = x.abs().amax(-1)
    scale = (amax / top).float()
    q = x * top / torch.where(amax > 0, amax, torch.ones_like(amax)).unsqueeze(-1)
    if case["fmt"] == "int8":
        return torch.round(q).to(torch.int8), scale
    return _to_minifloat(q, 3, -6, top).float().to(torch.float8_e4m3fn), scale


def _values(case, codes, scales):
    """The values that codes and scales stand for, in the cache's type."""
    if case["fmt"] == "mxfp4":
        c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :case["head_dim"]]
        m = (c & 7).float()
        v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, m * 2 - 8)) * torch.where(c >= 8, -1.0, 1.0)
        b = torch.ldexp(_blocks(v, case["head_dim"]), scales.int().unsqueeze(-1) - 127)
        return b.flatten(-2)[..., :case["head_dim"]].to(DTYPES[case["dtype"]])
    return (codes.float() * scales.unsqueeze(-1)).to(DTYPES[case["dtype"]])


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]
    lay = (case["planes"], case["layers"])
    # channels of keys differ in size by an order of magnitude
    channel = torch.exp(0.7 * torch.randn((*lay, 1, case["heads"], d), generator=g, device="cuda"))
    objects = []
    for n, t in _parts(case) if case["op"] != "page_out" else ():
        o = torch.empty((n, *lay, t, case["heads"], d), dtype=dtype, device="cuda")
        for k in range(n):
            o[k] = torch.randn((*lay, t, case["heads"], d), generator=g, device="cuda") * channel
        objects.append(o)
    state = {"case": case, "parts": _parts(case)}
    records = [torch.zeros((n, _record(case, t)[4]), dtype=torch.uint8, device="cuda") for n, t in _parts(case)]
    if case["op"] in ("read", "page_in"):
        for (n, t), o, r in zip(_parts(case), objects, records):
            words = [int.from_bytes(b"KVQ1", "little"), t, case["layers"] | case["heads"] << 16,
                     d | ["int8", "fp8", "mxfp4"].index(case["fmt"]) << 16 | list(DTYPES).index(case["dtype"]) << 20
                     | case["planes"] << 24]
            r[:, :16] = torch.tensor(words, dtype=torch.int32, device="cuda").view(torch.uint8)
            for k in range(n):
                codes, scales = _quantise(case, o[k])
                _code_view(case, r, t)[k] = codes
                _scale_view(case, r, t)[k] = scales
    state["records"] = records
    if case["op"] in ("page_out", "page_in"):
        block, tokens = case["block"], case["tokens"]
        blocks = -(-tokens // block) * 5 // 4 + 2
        shape = (case["layers"], case["planes"], blocks, block, case["heads"], d)
        if case["order"] == "HND":
            pool = torch.empty((*shape[:3], case["heads"], block, d), dtype=dtype, device="cuda").transpose(3, 4)
        else:
            pool = torch.empty(shape, dtype=dtype, device="cuda")
        for layer in range(case["layers"]):
            pool[layer] = torch.randn(shape[1:], generator=g, device="cuda") * channel[:, layer].unsqueeze(1)
        pages = torch.randperm(blocks, generator=g, device="cuda")[:-(-tokens // block)]
        slots = (pages.unsqueeze(1) * block + torch.arange(block, device="cuda")).flatten()[:tokens]
        slots[:case["skip"]] = -1
        state["pool"] = pool
        at, cut = 0, []
        for n, t in _parts(case):
            cut.append(slots[at:at + n * t].view(n, t))
            at += n * t
        state["slots"] = cut
    else:
        state["objects"] = objects if case["op"] in ("write", "roundtrip") else [torch.zeros_like(o) for o in objects]
        if case["op"] == "roundtrip":
            state["restored"] = [torch.zeros_like(o) for o in objects]
    if own:
        from confkv_b200.gpu_aesgcm import GpuAesGcmLibrary
        from confkv_b200.kv_codec import KvCodec, PagedKvCache

        state["codec"] = KvCodec(GpuAesGcmLibrary(), case["fmt"], dtype, planes=case["planes"], layers=case["layers"],
                                 heads=case["heads"], head_dim=d, device=torch.cuda.current_device())
        if "pool" in state:
            state["cache"] = PagedKvCache(state["codec"], list(state["pool"].unbind(0)))
        state["ok"] = [torch.zeros(n, dtype=torch.int32, device="cuda") for n, _ in _parts(case)]
    return state


# ------------------------------------------------------------------ one pass


def _pages(case, pool, slots):
    """[layers, planes, blocks, block, heads, d] seen by slots [n, t], and which of them are there."""
    n, t = slots.shape
    at = slots.clamp(min=0)
    return at // case["block"], at % case["block"], (slots >= 0).view(n, 1, 1, t, 1, 1)


def _codes_and_scales(case, state):
    return {"codes": [_code_view(case, r, t) for (_, t), r in zip(state["parts"], state["records"])],
            "scales": [_scale_view(case, r, t) for (_, t), r in zip(state["parts"], state["records"])]}


def _run_own(case, state):
    codec, records = state["codec"], state["records"]
    if case["op"] == "write":
        codec.quantise(state["objects"], records)
        return _codes_and_scales(case, state)
    if case["op"] == "read":
        codec.dequantise(records, state["objects"], ok=state["ok"])
        return state["objects"]
    if case["op"] == "roundtrip":
        codec.quantise(state["objects"], records)
        codec.dequantise(records, state["restored"], ok=state["ok"])
        return state["restored"]
    if case["op"] == "page_out":
        codec.quantise_paged(state["cache"], state["slots"], records)
        return _codes_and_scales(case, state)
    codec.dequantise_paged(records, state["cache"], state["slots"], ok=state["ok"])
    return state["pool"]


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "page_in":
        pool = state["pool"]
        for (_, t), record, slots in zip(state["parts"], state["records"], state["slots"]):
            values = _values(case, _code_view(case, record, t), _scale_view(case, record, t))
            keep = slots.flatten() >= 0
            at = slots.flatten()[keep]
            # [n, planes, layers, t, heads, d] -> [tokens, layers, planes, heads, d]
            values = values.permute(0, 3, 2, 1, 4, 5).flatten(0, 1)[keep]
            pool.permute(2, 3, 0, 1, 4, 5)[at // case["block"], at % case["block"]] = values
        return pool
    if case["op"] == "read":
        return [_values(case, _code_view(case, r, t), _scale_view(case, r, t))
                for (_, t), r in zip(state["parts"], state["records"])]
    if case["op"] == "page_out":
        objects = []
        for slots in state["slots"]:
            page, row, there = _pages(case, state["pool"], slots)
            x = state["pool"].permute(2, 3, 1, 0, 4, 5)[page, row]      # [n, t, planes, layers, heads, d]
            objects.append(torch.where(there, x.permute(0, 2, 3, 1, 4, 5), torch.zeros((), dtype=x.dtype, device="cuda")))
    else:
        objects = state["objects"]
    got = [_quantise(case, o) for o in objects]
    if case["op"] == "roundtrip":
        return [_values(case, c, s) for c, s in got]
    return {"codes": [c for c, _ in got], "scales": [s for _, s in got]}


def work(case):
    values = stored = 0
    for n, t in _parts(case):
        vectors, _, _, _, size = _record(case, t)
        values += n * vectors * case["head_dim"]
        stored += n * size
    there = 1 - case["skip"] / case["tokens"]
    size = values * torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    moved = {"write": size + stored, "read": size + stored, "roundtrip": 2 * size + stored,
             "page_out": size * there + stored, "page_in": (size + stored) * there}[case["op"]]
    if case["op"] in ("page_out", "page_in"):
        moved += 8 * case["tokens"]
    # a comparison, a product and a rounding a value on the way in, a product on the way out
    flops = {"write": 3, "page_out": 3, "read": 1, "page_in": 1, "roundtrip": 4}[case["op"]] * values
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ in 64 bits


def _nearest(y, levels):
    """y rounded to the nearest of +-levels (sorted, from 0), a tie to the level of even number."""
    a = y.abs().contiguous()
    middle = (levels[1:] + levels[:-1]) / 2
    at = torch.searchsorted(middle, a)                                   # middle[at - 1] < a <= middle[at]
    tie = (at < len(middle)) & (a == middle[at.clamp(max=len(middle) - 1)]) & (at % 2 == 1)
    return torch.copysign(levels[at + tie], y)


def _levels(fmt):
    if fmt == "int8":
        v = list(range(128))
    elif fmt == "fp8":
        v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]
    else:
        v = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _exact_codes(fmt, x):
    """Codes as numbers and one scale a value's vector or block, in 64 bits; x [..., d]."""
    levels = _levels(fmt)
    if fmt != "mxfp4":
        amax = x.abs().amax(-1, keepdim=True)
        unit = amax / levels[-1]
        return _nearest(torch.nan_to_num(levels[-1] * x / amax), levels), unit
    codes, unit = torch.empty_like(x), torch.empty_like(x)
    for at in range(0, x.shape[-1], BLOCK):
        part = x[..., at:at + BLOCK]
        amax = part.abs().amax(-1, keepdim=True)
        powers = 2.0 ** torch.arange(-127, 128, dtype=torch.float64, device="cuda")
        # the largest power of two that is not above amax / 4
        p = powers[(torch.searchsorted(powers, amax / 4, right=True) - 1).clamp(min=0)]
        codes[..., at:at + BLOCK] = _nearest(part / p, levels)
        unit[..., at:at + BLOCK] = p
    return codes, unit


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("read", "page_in"):
        restored = []
        for (_, t), r in zip(state["parts"], state["records"]):
            codes, scales = _code_view(case, r, t), _scale_view(case, r, t)
            if case["fmt"] == "mxfp4":
                nibble = torch.stack((codes % 16, codes // 16), -1).flatten(-2)[..., :case["head_dim"]].long()
                levels = _levels("mxfp4")
                v = torch.cat((levels, -levels))[nibble]
                unit = (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, -1)[..., :case["head_dim"]]
                restored.append(v * unit)
            else:
                restored.append(codes.double() * scales.double()[..., None])
        if case["op"] == "read":
            return restored
        pool = state["pool"].double()
        flat = pool.flatten(2, 3) if case["order"] == "NHD" else pool.reshape(*pool.shape[:2], -1, *pool.shape[4:])
        for v, slots in zip(restored, state["slots"]):
            for k in range(v.shape[0]):
                keep = (slots[k] >= 0).nonzero().flatten()
                flat.index_copy_(2, slots[k][keep], v[k].transpose(0, 1).index_select(2, keep))
        return flat.view(pool.shape)
    if case["op"] == "page_out":
        pool = state["pool"].double()
        flat = pool.reshape(*pool.shape[:2], -1, *pool.shape[4:])
        objects = []
        for slots in state["slots"]:
            x = torch.stack([flat.index_select(2, s.clamp(min=0)).transpose(0, 1) for s in slots])
            objects.append(x * (slots >= 0).double()[:, None, None, :, None, None])
    else:
        objects = [o.double() for o in state["objects"]]
    got = [_exact_codes(case["fmt"], o) for o in objects]
    if case["op"] == "roundtrip":
        return [c * u for c, u in got]
    codes = [None if case["fmt"] == "int8" else c for c, _ in got]      # whole numbers have no error to speak of
    return {"codes": codes, "scales": [u.squeeze(-1) for _, u in got]}
