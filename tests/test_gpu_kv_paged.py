"""Block tables, writing new tokens and attention of a paged cache against plain Python and numpy (paged_ref)."""

import random
import threading

import numpy as np
import paged_ref
import pytest
import torch

from confkv_b200.kv_codec import KvCodec, PagedKvCache
from confkv_b200.kv_paged import KvAttention, KvBlockTables

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
I32, I64 = torch.int32, torch.int64


def ints(values, dtype=I32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ------------------------------------------------------------------ block tables

def guarded(count, dtype, fill=-77):
    raw = torch.full((count + 32,), fill, dtype=dtype, device="cuda")
    return raw, raw[16:16 + count]


def unguarded(raw):
    assert bool((raw[:16] == -77).all()) and bool((raw[-16:] == -77).all()), "wrote outside an output"


def check_resize(lib, tables, held, lengths, ring, cursor, *, blocks, block_size, capacity, starts=True, stride=None):
    n, width = len(held), len(tables[0]) if tables else 0
    want = paged_ref.resize(tables, held, lengths, ring, cursor, blocks=blocks, block_size=block_size, capacity=capacity)
    stride = stride or max(width, 1)
    raw_tables, flat = guarded(max(n, 1) * stride, I32)
    rows = flat.view(-1, stride)[:n, :width]
    if n and width:
        rows.copy_(ints(tables))
    raw_ring, free = guarded(len(ring), I32)
    free.copy_(ints(ring))
    raw_kept, kept = guarded(n, I32)
    raw_after, after = guarded(2, I32)
    raw_slots, slots = guarded(capacity or 0, I64)
    raw_starts, at = guarded(n + 1, I64)
    k = KvBlockTables(lib, blocks=blocks, block_size=block_size)
    before = raw_tables.clone()
    k.resize(rows, ints(held), ints(lengths), free, ints(cursor), kept=kept, cursor_after=after,
             slots=slots if capacity is not None else None, starts=at if starts and capacity is not None else None)
    torch.cuda.synchronize()
    assert kept.tolist() == want["kept"]
    assert after.tolist() == want["cursor"]
    assert rows.tolist() == want["tables"] if width else True
    assert free.tolist() == want["free"]
    if capacity is not None:
        assert slots.tolist() == want["slots"]
        if starts:
            assert at.tolist() == want["starts"]
        else:
            unguarded(torch.cat((at, at))[:32] if n > 32 else raw_starts)
    for raw in (raw_tables, raw_ring, raw_kept, raw_after, raw_slots, raw_starts):
        unguarded(raw)
    if stride > width:
        gaps = torch.ones(max(n, 1) * stride, dtype=torch.bool, device="cuda").view(-1, stride)
        gaps[:n, :width] = False
        assert torch.equal(flat[gaps.flatten()], before[16:-16][gaps.flatten()]), "wrote between the rows"
    return want


def world(rng, n, width, block_size, most_new, finish, spare):
    """Requests with blocks of their own, a ring of the others, and lengths to come."""
    limit = width * block_size
    held = [rng.choice([0, 1, block_size, rng.randrange(0, limit + 1)]) for _ in range(n)]
    lengths = []
    for h in held:
        x = rng.random()
        lengths.append(0 if x < finish else rng.randrange(0, h + 1) if x < 1.5 * finish else min(limit, h + rng.randrange(0, most_new + 1)))
    owned = sum(paged_ref.ceil(h, block_size) for h in held)
    need = sum(max(0, paged_ref.ceil(x, block_size) - paged_ref.ceil(h, block_size)) for h, x in zip(held, lengths))
    free = max(0, int(need * spare))
    blocks = owned + free + rng.randrange(0, 3)
    names = list(range(blocks))
    rng.shuffle(names)
    tables, at = [], 0
    for h in held:
        c = paged_ref.ceil(h, block_size)
        tables.append(names[at:at + c] + [rng.randrange(-5, blocks + 5) for _ in range(width - c)])
        at += c
    ring = [rng.randrange(-5, blocks + 5) for _ in range(blocks)]
    first = rng.randrange(0, blocks) if blocks else 0
    for k in range(free):
        ring[(first + k) % blocks] = names[at + k]
    new = sum(max(0, x - h) for h, x in zip(held, lengths))
    return dict(tables=tables, held=held, lengths=lengths, ring=ring, cursor=[first, free], blocks=blocks, block_size=block_size), new


@pytest.mark.parametrize("n", [1, 2, 31, 33, 100, 511, 512, 513, 1100, 3000])
@pytest.mark.parametrize("block_size", [1, 5, 16])
def test_resize(gpu_lib, n, block_size):
    rng = random.Random(n * 100 + block_size)
    for width, most_new, finish, spare, room in ((9, 1, 0.0, 1.0, 1.0), (40, 300, 0.2, 1.1, 1.2), (40, 300, 0.2, 0.6, 1.0),
                                                 (40, 300, 0.3, 1.0, 0.7), (3, 2, 0.9, 0.0, 1.0)):
        w, new = world(rng, n, width, block_size, most_new, finish, spare)
        check_resize(gpu_lib, **w, capacity=int(new * room), stride=width + rng.choice([0, 3]))
        check_resize(gpu_lib, **w, capacity=int(new * room), starts=False)
        check_resize(gpu_lib, **w, capacity=None)


def test_resize_of_nothing(gpu_lib):
    check_resize(gpu_lib, [], [], [], [3, 4, 5], [1, 2], blocks=8, block_size=16, capacity=5)
    check_resize(gpu_lib, [[1, 2]] * 3, [0, 0, 0], [0, 0, 0], [], [0, 0], blocks=8, block_size=16, capacity=0)
    check_resize(gpu_lib, [[1, 2]] * 3, [0, 7, 32], [5, 12, 20], [], [3, 4], blocks=8, block_size=16, capacity=50)
    check_resize(gpu_lib, [[]] * 3, [0, 0, 0], [0, 1, 0], [3, 4, 5], [1, 2], blocks=8, block_size=16, capacity=5)
    check_resize(gpu_lib, [[1, 2]] * 2, [32, 31], [32, 32], [0], [0, 0], blocks=3, block_size=16, capacity=1)


def test_resize_of_bad_values(gpu_lib):
    """Lengths and cursors out of their ranges, names that are not the cache's, a ring without room."""
    rng = random.Random(5)
    w, _ = world(rng, 40, 12, 16, 100, 0.2, 2.0)
    for k, bad in enumerate((-1, 12 * 16 + 1, -(1 << 31), (1 << 31) - 1)):
        w["held"][3 + k], w["lengths"][13 + k], w["lengths"][3 + k] = bad, bad, 5
    check_resize(gpu_lib, **w, capacity=4000)
    for cursor in ([-3, 20], [1 << 30, 20], [-(1 << 31), 9], [5, -1], [5, (1 << 31) - 1], [5, -(1 << 31)]):
        check_resize(gpu_lib, **{**w, "cursor": cursor}, capacity=4000)
    # a ring that is full drops what it is given
    w["cursor"] = [4, w["blocks"] - 2]
    check_resize(gpu_lib, **w, capacity=4000)
    w["ring"] = [-(1 << 31), -1, (1 << 31) - 1, w["blocks"]] * (len(w["ring"]) // 4)
    w["cursor"] = [1, 30]
    want = check_resize(gpu_lib, **w, capacity=4000)
    assert -1 in want["slots"][:want["starts"][-1]]


def test_resize_of_a_few_hundred_thousand_tokens(gpu_lib):
    """More slots and blocks than one pass of the grid's threads."""
    rng = random.Random(6)
    w, new = world(rng, 40, 2000, 16, 30000, 0.3, 1.0)
    assert new > 148 * 512 * 2
    check_resize(gpu_lib, **w, capacity=new + 1000)
    w, new = world(rng, 700, 300, 1, 250, 0.4, 1.0)
    check_resize(gpu_lib, **w, capacity=new)


def test_a_row_that_counts_2_31_tokens(gpu_lib):
    """Slots near 2^31, and lengths near a row's 2^31 - 1 tokens."""
    size = 1 << 20
    blocks = 2047
    table = list(range(2047))[::-1]
    check_resize(gpu_lib, [table], [2047 * size - 10], [2047 * size], [0], [0, 0], blocks=blocks, block_size=size, capacity=11)
    check_resize(gpu_lib, [table + [0] * 10], [(1 << 31) - 5], [(1 << 31) - 1], [0], [0, 0], blocks=blocks, block_size=size, capacity=11)


# ------------------------------------------------------------------ writing new tokens

def plane_of(shape, dtype, order, offset=0, gap=0):
    """[blocks, size, heads, d] zeros: by tokens or by heads, `offset` elements behind an allocation, `gap` values behind each vector."""
    blocks, size, heads, d = shape
    inner = (size, heads) if order == "NHD" else (heads, size)
    raw = torch.full((offset + blocks * size * heads * (d + gap),), 3.0, dtype=dtype, device="cuda")
    t = raw[offset:].view(blocks, *inner, d + gap)[..., :d]
    return t if order == "NHD" else t.transpose(1, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("order", ["NHD", "HND"])
@pytest.mark.parametrize("d,offset,gap", [(128, 0, 0), (128, 4, 0), (128, 1, 0), (64, 0, 8), (65, 0, 0), (2, 0, 0), (1, 0, 0), (100, 2, 2), (1025, 0, 0)])
def test_append(gpu_lib, dtype, planes, order, d, offset, gap):
    t = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(d + offset)
    for tokens, heads, size in ((1, 8, 16), (37, 3, 5), (1000 if d < 1000 else 40, 2, 64)):
        blocks = tokens // size + 3
        layers = [[plane_of((blocks, size, heads, d), t, order, offset, gap) for _ in range(planes)] for _ in range(3)]
        codec = KvCodec(gpu_lib, "int8", t, planes=planes, layers=3, heads=heads, head_dim=d)
        attention = KvAttention(gpu_lib, PagedKvCache(codec, [tuple(x) for x in layers]), query_heads=heads) if d <= 1024 else None
        if attention is None:
            with pytest.raises(ValueError):
                KvAttention(gpu_lib, PagedKvCache(codec, [tuple(x) for x in layers]), query_heads=heads)
            continue
        slots = torch.randperm(blocks * size, generator=g, device="cuda")[:tokens]
        # some that are none
        slots[3::7] = ints([-1, blocks * size, -(1 << 62), 1 << 40], I64).repeat(tokens)[:len(slots[3::7])]
        wide = torch.randn((tokens, heads + 1, d + 3), generator=g, device="cuda").to(t)
        keys, values = wide[:, 1:, :d], torch.randn((heads, tokens, d), generator=g, device="cuda").to(t).transpose(0, 1)
        before = [[x._base.clone() if x._base is not None else x.clone() for x in layer] for layer in layers]
        want = [x.clone() for x in layers[1]]
        for k, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * size:
                for plane, source in zip(want, (keys, values)):
                    plane[s // size, s % size] = source[k]
        attention.append(1, slots, keys, values if planes == 2 else None)
        torch.cuda.synchronize()
        for got, x in zip(layers[1], want):
            assert torch.equal(got, x)
        for k in (0, 2):
            for got, x in zip(layers[k], before[k]):
                assert torch.equal(got._base if got._base is not None else got, x), "wrote to another layer"
        if gap:
            raw = layers[1][0]._base[offset:].view(-1, d + gap)
            assert bool((raw[:, d:] == 3).all()), "wrote between vectors"


def test_append_nothing(gpu_lib):
    codec = KvCodec(gpu_lib, "int8", torch.bfloat16, planes=2, layers=1, heads=2, head_dim=64)
    layer = torch.full((2, 4, 16, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    a = KvAttention(gpu_lib, PagedKvCache(codec, [layer]), query_heads=2)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    a.append(0, ints([], I64), none, none)
    one = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    a.append(0, ints([-1, 64, -5], I64), one, one)
    torch.cuda.synchronize()
    assert bool((layer == 3).all())
    empty = KvAttention(gpu_lib, PagedKvCache(codec, [torch.empty((2, 0, 16, 2, 64), dtype=torch.bfloat16, device="cuda")]), query_heads=2)
    empty.append(0, ints([0, 1, 2], I64), one, one)
    out = torch.full((2, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    empty.attend(0, one[:2], ints([[0, 1], [2, 3]]), ints([20, 0]), out)
    torch.cuda.synchronize()
    assert not out.any()


# ------------------------------------------------------------------ attention

class Case:
    """A cache of random values with requests' tokens in pages of it, and NaN everywhere else."""

    def __init__(self, lib, dtype, planes, heads, d, group, lengths, size, *, order="NHD", value_dim=None, window=0, scale=None,
                 seed=0, offset=0, gap=0, spare=3, layers=1, layer=0, extra=2, spread=1.0):
        t = DTYPES[dtype]
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [paged_ref.ceil(max(x, 0), size) for x in lengths]
        width = max(need) + extra
        blocks = sum(need) + spare
        names = list(range(blocks))
        rng.shuffle(names)
        self.tables, at = [], 0
        for c in need:
            # behind a request's blocks: anything
            self.tables.append(names[at:at + c] + [rng.choice([-1, blocks, (1 << 31) - 1, -(1 << 31), rng.randrange(blocks)]) for _ in range(width - c)])
            at += c
        self.planes = [plane_of((blocks, size, heads, d), t, order, offset, gap) for _ in range(planes)]
        channel = torch.exp(0.5 * torch.randn((heads, d), generator=g, device="cuda"))
        there = torch.zeros((blocks, size), dtype=torch.bool, device="cuda")
        for table, x in zip(self.tables, lengths):
            if x > 0:
                i = torch.arange(x, device="cuda")
                there[ints(table)[i // size].long(), i % size] = True
        for plane in self.planes:
            values = torch.randn(plane.shape, generator=g, device="cuda") * channel
            plane.copy_(torch.where(there[:, :, None, None], values, float("nan")))
        n = len(lengths)
        self.query = (spread * torch.randn((n, heads * group, d), generator=g, device="cuda")).to(t)
        self.lengths, self.size, self.window = lengths, size, window
        self.value_dim = d if value_dim is None else value_dim
        self.scale = d ** -0.5 if scale is None else scale
        codec = KvCodec(lib, "int8", t, planes=planes, layers=layers, heads=heads, head_dim=d)
        others = [tuple(torch.full_like(x, float("nan")) for x in self.planes) for _ in range(layers)] if layers > 1 else [None]
        if layers > 1:
            others = [tuple(plane_of(x.shape, t, order, offset, gap).fill_(float("nan")) for x in self.planes) for _ in range(layers)]
        others[layer] = tuple(self.planes)
        self.layer = layer
        self.cache = PagedKvCache(codec, others)
        self.attention = KvAttention(lib, self.cache, query_heads=heads * group, value_dim=value_dim, scale=scale, window=window)
        self.out = torch.full((n, heads * group, self.value_dim), 7.0, dtype=t, device="cuda")
        self.lse = torch.full((n, heads * group), 7.0, device="cuda")

    def run(self, **more):
        self.attention.attend(self.layer, self.query, ints(self.tables), ints(self.lengths), self.out, lse=self.lse, **more)
        torch.cuda.synchronize()
        return self

    def want(self):
        return paged_ref.attend([p.cpu() for p in self.planes], self.query.cpu(), self.tables, self.lengths, block_size=self.size,
                                value_dim=self.value_dim, scale=self.scale, window=self.window)

    def check(self, out=None, lse=None):
        assert_near(self.out if out is None else out, self.lse if lse is None else lse, *self.want())


def assert_near(out, lse, want, want_lse, far, lse_far):
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(out).all()
    off = np.abs(out - want) - far
    at = np.unravel_index(np.argmax(off), off.shape)
    assert off.max() <= 0, (at, out[at], want[at], far[at])
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(lse), empty)
    assert (np.abs(lse[~empty] - want_lse[~empty]) <= lse_far[~empty]).all()


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 500]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 7, 8, 16, 24, 33, 40, 64, 65, 72, 80, 96, 100, 112, 120, 127, 128, 130, 136, 160, 192, 200, 248, 255, 256, 257, 264, 320, 576,
                               1000, 1024])
def test_head_sizes(gpu_lib, dtype, d):
    Case(gpu_lib, dtype, 2, 2, d, 3, LENGTHS, 16, seed=d).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,value_dim", [(16, 16), (64, 64), (128, 100), (192, 128), (256, 1), (320, 256), (320, 319), (320, 320), (576, 512), (576, 576), (100, 99), (600, 512)])
def test_latent_vectors(gpu_lib, dtype, d, value_dim):
    for group in (1, 5, 16, 40):
        Case(gpu_lib, dtype, 1, 1, d, group, LENGTHS + [3000, 0, 64], 16, value_dim=value_dim, seed=d + group).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 9, 12, 15, 16, 17, 31, 32, 33, 71])
def test_groups(gpu_lib, dtype, d, group):
    for heads in (1, 3):
        Case(gpu_lib, dtype, 2, heads, d, group, [0, 1, 40, 64, 130], 16, seed=group).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [260, 320, 384, 388, 576, 640, 644])
def test_groups_of_long_vectors(gpu_lib, dtype, d):
    for group in (1, 2, 3, 4, 5, 9):
        Case(gpu_lib, dtype, 2, 2, d, group, [0, 1, 40, 130, 1000], 16, seed=group).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["NHD", "HND"])
@pytest.mark.parametrize("size", [1, 3, 5, 8, 16, 48, 64, 100, 256])
def test_block_sizes(gpu_lib, dtype, order, size):
    for d in (64, 100, 128):
        Case(gpu_lib, dtype, 2, 4, d, 2, LENGTHS, size, order=order, seed=size).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 65, 100, 499, 500, (1 << 32) - 1])
def test_windows(gpu_lib, dtype, window):
    for d, group in ((64, 4), (100, 4), (128, 4), (128, 9)):
        Case(gpu_lib, dtype, 2, 2, d, group, LENGTHS, 16, window=window, seed=window % 1000).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,gap", [(1, 0), (2, 0), (4, 0), (8, 0), (0, 8), (0, 4), (0, 1), (8, 8)])
def test_alignments_of_the_cache(gpu_lib, dtype, offset, gap):
    for d in (64, 128):
        Case(gpu_lib, dtype, 2, 2, d, 4, LENGTHS, 16, offset=offset, gap=gap, seed=offset).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 4), (100, 4), (128, 4), (256, 4), (64, 12), (128, 12), (128, 20)])
def test_strides_of_queries_and_results(gpu_lib, dtype, d, group):
    c = Case(gpu_lib, dtype, 2, 2, d, group, LENGTHS, 16, layers=3, layer=2)
    want = c.want()
    t, n, heads = c.query.dtype, len(c.lengths), 2 * group
    for off in (1, 2, 8):
        for by_heads in (False, True):
            shape = (heads, n, d + 16) if by_heads else (n, heads, d + 16)
            q, o = (torch.full(shape, 7.0, dtype=t, device="cuda") for _ in range(2))
            q_view, o_view = (x.transpose(0, 1)[..., off:off + d] if by_heads else x[..., off:off + d] for x in (q, o))
            q_view.copy_(c.query)
            lse = torch.full((n, heads + 5), 7.0, device="cuda")
            wide = torch.zeros((n, len(c.tables[0]) + 3), dtype=I32, device="cuda")
            wide[:, 2:-1] = ints(c.tables)
            c.attention.attend(2, q_view, wide[:, 2:-1], ints(c.lengths), o_view, lse=lse[:, 3:-2])
            torch.cuda.synchronize()
            assert_near(o_view, lse[:, 3:-2], *want)
            mask = torch.ones_like(o, dtype=torch.bool)
            (mask.transpose(0, 1) if by_heads else mask)[..., off:off + d] = False
            assert bool((o[mask] == 7).all()) and bool((lse[:, :3] == 7).all()) and bool((lse[:, -2:] == 7).all()), "wrote beside the results"
    # one query for all requests, and no lse
    shared = c.query[:1].expand(n, heads, d)
    c.attention.attend(2, shared, ints(c.tables), ints(c.lengths), c.out)
    c.query = shared.contiguous()
    again = c.want()
    torch.cuda.synchronize()
    assert_near(c.out, torch.from_numpy(again[1]), *again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 4), (100, 4), (128, 4), (128, 13), (64, 20)])
@pytest.mark.parametrize("lengths", [[20000], [1, 30000, 0, 5], [4000] * 9, [0] * 50 + [9000], list(range(0, 700, 3)), [1] * 700, [0] * 300], ids=lambda x: f"{len(x)}x{max(x)}")
def test_parts_of_rows(gpu_lib, dtype, d, group, lengths):
    """Few long rows, which many workers share, and many short ones; more requests than one pass of a block's threads."""
    c = Case(gpu_lib, dtype, 2, 2, d, group, lengths, 16, seed=len(lengths)).run()
    c.check()
    first = c.out.clone(), c.lse.clone()
    c.run()
    assert torch.equal(c.out, first[0]) and torch.equal(c.lse, first[1])            # equal calls, equal bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,planes,window", [(64, 2, 0), (72, 2, 100), (128, 2, 0), (256, 2, 0), (128, 1, 0), (320, 1, 70)])
def test_many_requests(gpu_lib, dtype, d, planes, window):
    """Rows enough that whole ones go to a warp each, empty and long ones among them."""
    rng = random.Random(d)
    lengths = [rng.choice([0, 1, 5, 16, 70, 130, 400]) if k % 300 else rng.choice([600, 5000]) for k in range(3000 if d < 256 else 1500)]
    Case(gpu_lib, dtype, planes, 1, d, 2, lengths, 16, window=window, value_dim=d - 3 if planes == 1 else None).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 4), (100, 4), (64, 12)])
def test_blocks_that_are_none(gpu_lib, dtype, d, group):
    """Tokens in blocks that are not the cache's are left out, whole rows and whole tiles of them too."""
    c = Case(gpu_lib, dtype, 2, 2, d, group, LENGTHS, 16, seed=9)
    blocks = c.planes[0].shape[0]
    bad = [-1, blocks, (1 << 31) - 1, -(1 << 31)]
    for r, table in enumerate(c.tables):
        for b in range(paged_ref.ceil(c.lengths[r], 16)):
            if r == 15 and b not in (0, 30) or r == 14 or r % 2 and b % 3 == 1:
                table[b] = bad[(r + b) % 4]
    c.run().check()
    assert bool(torch.isneginf(c.lse[14]).all()) and not c.out[14].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 100])
def test_lengths_out_of_range(gpu_lib, dtype, d):
    c = Case(gpu_lib, dtype, 2, 1, d, 4, [64, 64, 64, 64], 16, extra=0)
    c.lengths = [65, (1 << 31) - 1, -1, -(1 << 31)]
    c.run().check()
    assert not c.out[2:].any()
    c.attention.attend(0, c.query, torch.zeros((4, 0), dtype=I32, device="cuda"), ints([5, 0, 1, 9]), c.out, lse=c.lse)
    torch.cuda.synchronize()
    assert not c.out.any() and bool(torch.isneginf(c.lse).all())
    c.attention.attend(0, c.query[:0], ints(c.tables)[:0], ints([]), c.out[:0], lse=c.lse[:0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 4), (100, 4), (64, 12)])
@pytest.mark.parametrize("spread", [1e-3, 1.0, 60.0])
def test_scores_of_all_sizes(gpu_lib, dtype, d, group, spread):
    """From nearly equal weights to one token that outweighs all others, at the end, the beginning and in the middle."""
    Case(gpu_lib, dtype, 2, 2, d, group, [700, 64, 65, 3, 1], 16, spread=spread, seed=1).run().check()
    for at in (0, 350, 699):
        c = Case(gpu_lib, dtype, 2, 2, d, group, [700], 16, seed=2)
        c.planes[0][c.tables[0][at // 16], at % 16] = (c.query[0, ::group] * 8).to(c.query.dtype)
        c.run().check()
    for scale in (0.0, -0.3, 4.0):
        Case(gpu_lib, dtype, 2, 2, d, group, [700, 64, 3], 16, scale=scale, seed=3).run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 2), (128, 2), (64, 12)])
def test_many_small_weights_beside_a_large_one(gpu_lib, dtype, d, group):
    """One token with weight 1, and 40000 with 2^-17 each, which together weigh a third of it; half's least normal number is 2^-14."""
    c = Case(gpu_lib, dtype, 2, 1, d, group, [40000], 16, seed=4, scale=1.0)
    c.query.zero_()
    c.query[..., 0] = 1
    c.planes[0].zero_()
    c.planes[0][c.tables[0][700], 3] = 0
    c.planes[0][c.tables[0][700], 3, 0, 0] = 17 * 0.6931471805599453
    c.run().check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 2), (100, 2), (64, 10)])
def test_values_that_are_not_finite(gpu_lib, dtype, d, group):
    """What is not finite among a request's own tokens shows in its rows as the formula has it, and in no other's."""
    inf = float("inf")
    c = Case(gpu_lib, dtype, 2, 1, d, group, [200] * 8, 16, seed=5)
    clean = c.run().out.clone()
    q, (k, v) = c.query, c.planes
    q[:, :, 0] = 1
    clean = c.run().out.clone()

    def row(r, i):
        return c.tables[r][i // 16], i % 16

    k[(*row(1, 30), 0, 0)] = -inf                   # weight 0: the others remain
    k[(*row(2, 30), 0, 0)] = inf                    # inf - inf
    k[(*row(3, 30), 0, 3)] = float("nan")
    v[(*row(4, 30), 0, 3)] = float("nan")
    v[(*row(5, 130), 0, 3)] = inf
    for i in range(200):
        k[(*row(6, i), 0, 0)] = -inf                # all weights 0 / 0
    c.run()
    assert torch.equal(c.out[[0, 7]], clean[[0, 7]])
    assert bool(torch.isfinite(c.out[1]).all()) and bool(torch.isfinite(c.lse[1]).all())
    assert bool(torch.isnan(c.out[2]).all()) and bool(torch.isnan(c.out[3]).all()) and bool(torch.isnan(c.out[6]).all())
    assert bool(torch.isnan(c.lse[[2, 3, 6]]).all())
    assert bool(torch.isnan(c.out[4, :, 3]).all()) and bool((c.out[5, :, 3] == inf).all())
    rest = [x for x in range(d) if x != 3]
    assert bool(torch.isfinite(c.out[4:6][:, :, rest]).all())
    # the first row again, without the token of weight 0
    e = Case(gpu_lib, dtype, 2, 1, d, group, [200] * 8, 16, seed=5)
    e.query.copy_(q)
    e.planes[0][row(1, 30)] = 0
    want = paged_ref.attend([torch.where(torch.isfinite(p), p, 0).cpu() for p in e.planes], q.cpu(), e.tables, e.lengths, block_size=16,
                            value_dim=d, scale=e.scale)
    s = e.scale * (q[1].double() @ torch.stack([k[(*row(1, i), 0)].double() for i in range(200)]).T)
    p = torch.softmax(s, -1)
    vs = torch.stack([v[(*row(1, i), 0)].double() for i in range(200)])
    assert bool(((c.out[1].double() - p @ vs).abs().cpu().numpy() <= want[2][1] + want[2][0].max()).all())


def test_a_cache_of_more_than_4_gib(gpu_lib):
    """Blocks whose offsets pass 32 bits, in elements too."""
    size, heads, d, blocks = 16, 8, 128, 150_000                # 2.4 G values a plane
    planes = [torch.empty((blocks, size, heads, d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    codec = KvCodec(gpu_lib, "int8", torch.bfloat16, planes=2, layers=1, heads=heads, head_dim=d)
    a = KvAttention(gpu_lib, PagedKvCache(codec, [tuple(planes)]), query_heads=16)
    table = [149_999, 3, 131_072, 65_536, 140_000]
    tokens = 70
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((tokens, heads, d), generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = ints([table[i // size] * size + i % size for i in range(tokens)], I64)
    a.append(0, slots, k, v)
    q = torch.randn((1, 16, d), generator=g, device="cuda").bfloat16()
    out, lse = torch.empty_like(q), torch.empty((1, 16), device="cuda")
    a.attend(0, q, ints([table]), ints([tokens]), out, lse=lse)
    torch.cuda.synchronize()
    small = [torch.zeros((5, size, heads, d), dtype=torch.bfloat16) for _ in range(2)]
    for x, source in zip(small, (k, v)):
        x.view(80, heads, d)[:tokens] = source.cpu()
    for plane, x in zip(planes, small):
        for j, name in enumerate(table):
            there = min(size, tokens - j * size)
            assert torch.equal(plane[name, :there].cpu(), x[j, :there])
    assert_near(out, lse, *paged_ref.attend(small, q.cpu(), [list(range(5))], [tokens], block_size=size, value_dim=d, scale=d ** -0.5))


# ------------------------------------------------------------------ streams, graphs, threads

@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp32", 100)])
def test_streams_and_workspaces(gpu_lib, dtype, d):
    """Calls on streams of their own, with workspaces of their own, at once; the default one is the call's own too."""
    cases = [Case(gpu_lib, dtype, 2, 2, d, 4, [3000 + 100 * k, 0, 17], 16, seed=k) for k in range(6)]
    want = [c.want() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    at = [(ints(c.tables), ints(c.lengths)) for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, (tables, lengths) in zip(cases, streams, at):
            c.attention.attend(0, c.query, tables, lengths, c.out, lse=c.lse, stream=s)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert_near(c.out, c.lse, *w)
        c.out.fill_(7)
    own = [c.attention.workspace().fill_(255) for c in cases]
    torch.cuda.synchronize()

    def call(k):
        c = cases[k]
        for _ in range(20):
            c.attention.attend(0, c.query, *at[k], c.out, lse=c.lse, workspace=own[k], stream=streams[k])

    threads = [threading.Thread(target=call, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert_near(c.out, c.lse, *w)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp32", 100)])
def test_a_captured_step(gpu_lib, dtype, d):
    """resize, append and attend captured once and replayed while lengths grow on the device: a decoding loop, against
    the same steps in plain Python; requests end and others begin between replays."""
    t, heads, group, size, n, blocks = DTYPES[dtype], 2, 4, 4, 5, 60
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = torch.full((2, blocks, size, heads, d), float("nan"), dtype=t, device="cuda")
    codec = KvCodec(gpu_lib, "int8", t, planes=2, layers=1, heads=heads, head_dim=d)
    a = KvAttention(gpu_lib, PagedKvCache(codec, [layer]), query_heads=heads * group)
    k = KvBlockTables(gpu_lib, blocks=blocks, block_size=size)
    width = 12
    tables, held, lengths, kept = torch.full((n, width), -9, dtype=I32, device="cuda"), ints([0] * n), ints([0] * n), ints([0] * n)
    free, cursor, after = ints(list(range(blocks))[::-1]), ints([0, blocks]), ints([0, 0])
    slots, starts = torch.zeros(n, dtype=I64, device="cuda"), torch.zeros(n + 1, dtype=I64, device="cuda")
    keys, values, query = (torch.zeros((n, h, d), dtype=t, device="cuda") for h in (heads, heads, heads * group))
    out, lse = torch.zeros_like(query), torch.zeros((n, heads * group), device="cuda")

    def step():
        k.resize(tables, held, lengths, free, cursor, kept=kept, cursor_after=after, slots=slots, starts=starts)
        a.append(0, slots, keys, values)
        a.attend(0, query, tables, kept, out, lse=lse)
        cursor.copy_(after)
        held.copy_(kept)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()                                      # nothing to do: all lengths are 0
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    model = dict(tables=tables.tolist(), held=[0] * n, ring=free.tolist(), cursor=[0, blocks])
    mirror = layer.cpu()
    rng = random.Random(0)
    for turn in range(30):
        x = [h + 1 if rng.random() < 0.95 else 0 for h in model["held"]]
        lengths.copy_(ints(x))
        for b in (keys, values, query):
            b.copy_(torch.randn(b.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = paged_ref.resize(model["tables"], model["held"], x, model["ring"], model["cursor"], blocks=blocks, block_size=size, capacity=n)
        assert kept.tolist() == want["kept"] and tables.tolist() == want["tables"] and cursor.tolist() == want["cursor"]
        assert free.tolist() == want["free"] and slots.tolist() == want["slots"]
        for i, s in enumerate(want["slots"]):
            if s >= 0:
                mirror[0, s // size, s % size], mirror[1, s // size, s % size] = keys[i].cpu(), values[i].cpu()
        assert torch.equal(torch.nan_to_num(layer.cpu(), 99), torch.nan_to_num(mirror, 99))
        assert_near(out, lse, *paged_ref.attend(list(mirror), query.cpu(), want["tables"], want["kept"], block_size=size, value_dim=d,
                                                scale=d ** -0.5))
        model = dict(tables=want["tables"], held=want["kept"], ring=want["free"], cursor=want["cursor"])
    del graph


FIRST_CALL = """
import sys
sys.path[:0] = {paths!r}
import torch
from confkv_b200.gpu_aesgcm import GpuAesGcmLibrary
from test_gpu_kv_paged import Case, assert_near, ints
c = Case(GpuAesGcmLibrary(), {dtype!r}, 2, 2, {d}, {group}, [3000, 0, 17], 16)
tables, lengths = ints(c.tables), ints(c.lengths)
workspace = c.attention.workspace() if {own} else None
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c.attention.attend(0, c.query, tables, lengths, c.out, lse=c.lse, workspace=workspace)
c.out.zero_()
g.replay()
torch.cuda.synchronize()
c.check()
"""


@pytest.mark.parametrize("dtype,d,group,own", [("bf16", 128, 4, True), ("fp16", 64, 12, False), ("fp32", 100, 2, False)])
def test_a_process_whose_first_call_is_captured(gpu_lib, dtype, d, group, own):
    import subprocess
    import sys
    from pathlib import Path

    tests = Path(__file__).resolve().parent
    code = FIRST_CALL.format(paths=[str(tests), str(tests.parent)], dtype=dtype, d=d, group=group, own=own)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_graphs_with_one_workspace(gpu_lib):
    """Replayed in turns on one stream."""
    cases = [Case(gpu_lib, dtype, 2, 2, d, group, [5000, 70, 0, 400], 16, seed=d) for dtype, d, group in (("bf16", 128, 4), ("fp16", 64, 12), ("fp32", 100, 2))]
    want = [c.want() for c in cases]
    shared = torch.empty(max(c.attention.workspace().numel() for c in cases), dtype=torch.uint8, device="cuda")
    at = [(ints(c.tables), ints(c.lengths)) for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c, (tables, lengths) in zip(cases, at):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attention.attend(0, c.query, tables, lengths, c.out, lse=c.lse, workspace=shared)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert_near(c.out, c.lse, *w)
    del graphs


@pytest.mark.parametrize("fmt", ["int8", "mxfp4"])
def test_records_read_back_are_attended_to(gpu_lib, fmt):
    """A stored prompt: blocks for its tokens, its records read back into their slots, one more token, attention."""
    heads, d, size, tokens, chunk, layers, blocks = 2, 64, 16, 96, 32, 2, 20
    g = torch.Generator(device="cuda").manual_seed(3)
    codec = KvCodec(gpu_lib, fmt, torch.bfloat16, planes=2, layers=layers, heads=heads, head_dim=d)
    objects = torch.randn((tokens // chunk, 2, layers, chunk, heads, d), generator=g, device="cuda").bfloat16()
    records = torch.zeros((tokens // chunk, codec.record_bytes(chunk)), dtype=torch.uint8, device="cuda")
    codec.quantise(objects, records)
    restored = torch.empty_like(objects)
    codec.dequantise(records, restored)
    cache = PagedKvCache(codec, [torch.full((2, blocks, size, heads, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(layers)])
    k, a = KvBlockTables(gpu_lib, blocks=cache.blocks, block_size=size), KvAttention(gpu_lib, cache, query_heads=4)
    tables, free = torch.zeros((1, 10), dtype=I32, device="cuda"), torch.randperm(blocks, generator=g, device="cuda").int()
    kept, after, slots = ints([0]), ints([0, 0]), torch.zeros(tokens, dtype=I64, device="cuda")
    k.resize(tables, ints([0]), ints([tokens]), free, ints([7, 13]), kept=kept, cursor_after=after, slots=slots)
    ok = torch.zeros(tokens // chunk, dtype=I32, device="cuda")
    codec.dequantise_paged(records, cache, slots.view(-1, chunk), ok=ok)
    one, again, later = ints([0]), ints([0, 0]), torch.zeros(1, dtype=I64, device="cuda")
    k.resize(tables, kept, kept + 1, free, after, kept=one, cursor_after=again, slots=later)
    new = torch.randn((2, 1, heads, d), generator=g, device="cuda").bfloat16()
    for layer in range(layers):
        a.append(layer, later, new[0], new[1])
        q = torch.randn((1, 4, d), generator=g, device="cuda").bfloat16()
        out, lse = torch.empty_like(q), torch.empty((1, 4), device="cuda")
        a.attend(layer, q, tables, one, out, lse=lse)
        torch.cuda.synchronize()
        assert bool((ok == 1).all()) and one.tolist() == [tokens + 1]
        planes = []
        for p in range(2):
            x = torch.cat((restored[:, p, layer].flatten(0, 1), new[p])).cpu()
            planes.append(torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 15)).view(-1, size, heads, d))
        assert_near(out, lse, *paged_ref.attend(planes, q.cpu(), [list(range(7))], [tokens + 1], block_size=size, value_dim=d, scale=d ** -0.5))


def test_refusals_leave_everything_as_it_was(gpu_lib):
    c = Case(gpu_lib, "bf16", 2, 2, 64, 4, [20, 30], 16)
    for bad in (dict(workspace=c.attention.workspace()[16:]), dict(workspace=c.attention.workspace()[8:])):
        with pytest.raises(Exception):
            c.run(**bad)
    with pytest.raises(ValueError):
        c.attention.attend(0, c.query.float(), ints(c.tables), ints(c.lengths), c.out)
    with pytest.raises(ValueError):
        c.attention.attend(0, c.query.cpu(), ints(c.tables), ints(c.lengths), c.out)
    torch.cuda.synchronize()
    assert bool((c.out == 7).all()) and bool((c.lse == 7).all())
    c.run().check()


def test_another_current_device(gpu_lib):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    c = Case(gpu_lib, "bf16", 2, 2, 64, 4, [20, 3000], 16)
    tables, lengths = ints(c.tables), ints(c.lengths)
    torch.cuda.synchronize()
    with torch.cuda.device(1):
        c.attention.attend(0, c.query, tables, lengths, c.out, lse=c.lse)
    torch.cuda.synchronize(0)
    c.check()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,value_dim,group", [(260, 1, 2), (300, 16, 4), (320, 64, 4), (320, 128, 8), (260, 16, 9), (320, 320, 3), (576, 64, 4)])
def test_a_query_less_aligned_than_the_cache(gpu_lib, dtype, d, value_dim, group):
    """Queries at an odd element over an aligned cache of latent vectors, with a workspace of exactly the bytes asked for."""
    c = Case(gpu_lib, dtype, 1, 1, d, group, [20000, 0, 3000, 70], 16, value_dim=value_dim, seed=d + group)
    raw = torch.zeros(c.query.numel() + 1, dtype=c.query.dtype, device="cuda")
    query = raw[1:].view(c.query.shape)
    query.copy_(c.query)
    c.query = query
    size = c.attention.workspace().numel()
    space = torch.full((size + 8192,), 0x5a, dtype=torch.uint8, device="cuda")
    c.run(workspace=space[:size]).check()
    assert bool((space[size:] == 0x5a).all()), "wrote behind the workspace"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("planes,d,group", [(2, 64, 4), (2, 64, 12), (2, 128, 12), (2, 100, 2), (1, 128, 4), (1, 320, 16), (1, 576, 20)])
@pytest.mark.parametrize("size", [12000.0, 16384.0, 24000.0, 40000.0, 65504.0])
def test_scores_of_millions(gpu_lib, dtype, planes, d, group, size):
    """One channel of queries and keys so large that floats lie 2 to 32 apart at the scores. It alone makes the scores, so that they
    are equal or far apart: a mean of the values of the tokens that have it, which errs by the rounding of its n sums, 2^-23 n of the values'
    sizes, and its own to the type; and the score itself, rounded a few times."""
    c = Case(gpu_lib, dtype, planes, 1, d, group, [200, 1, 64, 5000, 0], 16, seed=8)
    channel = c.query.new_tensor(size)
    c.query.zero_()
    c.query[..., 0] = channel
    tops = [[7], [0], list(range(64)), list(range(0, 5000, 3)), []]
    for plane in c.planes:
        plane.copy_(torch.nan_to_num(plane))
    for table, x, top in zip(c.tables, c.lengths, tops):
        for i in range(x):
            c.planes[0][table[i // 16], i % 16, 0, 0] = channel if i in top else 0
    c.run()
    score = float(channel) ** 2 * c.scale
    values = c.planes[-1].double().cpu()
    for r, top in enumerate(tops):
        if not top:
            assert not c.out[r].any() and bool(torch.isneginf(c.lse[r]).all())
            continue
        v = torch.stack([values[c.tables[r][i // 16], i % 16, 0] for i in top])
        want, n = v.mean(0), len(top)
        got = c.out[r].double().cpu()
        far = v.abs().mean(0) * (n + 8) * 2.0 ** -23 + want.abs() * torch.finfo(c.out.dtype).eps / 2 * 1.001 + 2.0 ** -25
        assert bool(torch.isfinite(got).all()) and bool(((got - want).abs() <= far).all()), (r, (got - want).abs().max())
        lse = score + float(np.log(n))
        assert bool(((c.lse[r].double() - lse).abs() <= lse * 2.0 ** -21).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("planes,d,group", [(2, 64, 2), (2, 64, 12), (2, 100, 4), (2, 128, 4), (2, 128, 12), (2, 192, 20), (1, 128, 4), (1, 320, 16), (1, 576, 20)])
def test_weights_have_more_bits_than_the_type(gpu_lib, dtype, planes, d, group):
    """Values that cancel: what is left shows the weights' own roundings. Scores are of one product, exact, and times the scale; they err by
    3 2^-24 of their size, their difference from the maximum and its power by 2^-22; weights enter the products with 2^-15 (bfloat16) or
    2^-20 (half) of theirs; sums of n by n 2^-23. The result's own rounding is that of a small number."""
    lengths = [2, 3, 5, 9, 16, 17, 40] * 3
    c = Case(gpu_lib, dtype, planes, 1, d, group, lengths, 16, seed=11, scale=0.7)
    t = c.query.dtype
    g = torch.Generator(device="cuda").manual_seed(12)
    c.query.zero_()
    c.query[..., 0] = 1
    for plane in c.planes:
        plane.copy_(torch.nan_to_num(plane))
    step = {"bf16": 2.0 ** -15, "fp16": 2.0 ** -20}[dtype]
    for r, x in enumerate(lengths):
        at = [(c.tables[r][i // 16], i % 16) for i in range(x)]
        s = -4 * torch.rand(x, generator=g, device="cuda")
        s[int(torch.randint(x, (1,), generator=g, device="cuda"))] = 0
        for (b, row), y in zip(at, s.to(t)):
            c.planes[0][b, row, 0, 0] = y
        keys = torch.stack([c.planes[0][b, row, 0, 0] for b, row in at]).double()
        v = torch.stack([c.planes[-1][b, row, 0] for b, row in at]).double()
        p = torch.softmax(0.7 * keys, 0)
        last = (-(p[:-1, None] * v[:-1]).sum(0) / p[-1]).clamp(-60000, 60000)
        if planes == 1:
            last[0] = keys[-1]
        c.planes[-1][at[-1]] = last[None].to(t)
    c.run()
    got = c.out.double()
    worst = 0.0
    for r, x in enumerate(lengths):
        at = [(c.tables[r][i // 16], i % 16) for i in range(x)]
        keys = torch.stack([c.planes[0][b, row, 0, 0] for b, row in at]).double()
        v = torch.stack([c.planes[-1][b, row, 0] for b, row in at]).double()
        p = torch.softmax(0.7 * keys, 0)
        want, sizes = p @ v, p @ v.abs()
        far = sizes * (step + 4 * 0.7 * 4 * 2.0 ** -24 + 2.0 ** -22 + (x + 4) * 2.0 ** -23) + want.abs() * torch.finfo(t).eps / 2 * 1.01 + 2.0 ** -24
        off = (got[r] - want).abs() / far
        worst = max(worst, float(off.max()))
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 2), (64, 12), (100, 4), (128, 12), (192, 20), (256, 3)])
def test_infinite_values_of_small_weights(gpu_lib, dtype, d, group):
    """A value's infinity stays one as far down as floats have the weight, and a thousand finite values beside it are as they were."""
    c = Case(gpu_lib, dtype, 2, 1, d, group, [3, 100, 1000, 5000], 16, seed=13, scale=1.0)
    c.query.zero_()
    c.query[..., 0] = 1
    for plane in c.planes:
        plane.copy_(torch.nan_to_num(plane))
    for k, score in enumerate((-8.0, -20.0, -31.0, -60.0)):
        for r, x in enumerate(c.lengths):
            for i in range(x):
                c.planes[0][c.tables[r][i // 16], i % 16, 0, 0] = score if i else 0
        c.run().check()
        clean = c.out.clone()
        at = [(c.tables[r][(x - 1) // 16], (x - 1) % 16, 0, 5 + k) for r, x in enumerate(c.lengths)]
        for r, place in enumerate(at):
            c.planes[-1][place] = float("inf") if r % 2 else float("-inf")
        c.run()
        for r, place in enumerate(at):
            assert bool((c.out[r, :, 5 + k] == (float("inf") if r % 2 else float("-inf"))).all())
            c.planes[-1][place] = 0.5
        rest = [i for i in range(d) if i != 5 + k]
        assert torch.equal(c.out[:, :, rest], clean[:, :, rest])


def test_resize_of_arrays_between_the_rows(gpu_lib):
    """Whatever the call reads and writes beside the tables lies between their rows."""
    rng = random.Random(14)
    w, new = world(rng, 12, 9, 16, 40, 0.2, 1.2)
    want = paged_ref.resize(**w, capacity=20)
    gap, width = 64, 9
    big = torch.full((12, width + gap), -77, dtype=I32, device="cuda")
    rows = big[:, :width]
    rows.copy_(ints(w["tables"]))
    names = {"held": w["held"], "lengths": w["lengths"], "cursor": w["cursor"], "kept": [0] * 12, "cursor_after": [0, 0]}
    at = {}
    for k, (name, values) in enumerate(names.items()):
        at[name] = big[2 * k, width + 3:width + 3 + len(values)]
        at[name].copy_(ints(values))
    free = ints(w["ring"])
    slots = big.view(-1)[width + (width + gap) + 10:][:40].view(I64)        # 8-byte aligned: (9 + 73 + 10) names
    KvBlockTables(gpu_lib, blocks=w["blocks"], block_size=16).resize(rows, at["held"], at["lengths"], free, at["cursor"], kept=at["kept"],
                                                                     cursor_after=at["cursor_after"], slots=slots)
    torch.cuda.synchronize()
    assert rows.tolist() == want["tables"] and at["kept"].tolist() == want["kept"] and at["cursor_after"].tolist() == want["cursor"]
    assert slots.tolist() == want["slots"] and free.tolist() == want["free"]
    assert at["held"].tolist() == w["held"] and at["lengths"].tolist() == w["lengths"] and at["cursor"].tolist() == w["cursor"]


@pytest.mark.parametrize("n,new", [(100_003, 20), ((1 << 20) + 3, 1), ((1 << 22) + 1, 2)])
def test_resize_of_very_many_requests(gpu_lib, n, new):
    """Thousands of requests a thread: every one grows, the odd thousandth ends, and all that is written is compared."""
    size, width = 16, 4
    g = torch.Generator(device="cuda").manual_seed(n)
    held = torch.randint(0, 33, (n,), generator=g, device="cuda", dtype=I32)
    lengths = torch.where(torch.arange(n, device="cuda") % 1000 == 999, 0, held + new).to(I32)
    before, behind = (held + size - 1) // size, (lengths + size - 1) // size
    take, give = (behind - before).clamp(min=0), (before - behind).clamp(min=0)
    taken, given = int(take.sum()), int(give.sum())
    owned = int(before.sum())
    blocks = owned + taken + 7
    names = torch.randperm(blocks, generator=g, device="cuda").to(I32)
    col = torch.arange(width, device="cuda")
    first = before.cumsum(0) - before
    tables = torch.where(col < before[:, None], names[(first[:, None] + col).clamp(max=blocks - 1)], -9).to(I32).contiguous()
    ring = torch.full((blocks,), -7, dtype=I32, device="cuda")
    start = blocks - 5                                                  # the free names go over the ring's end
    ring[(start + torch.arange(taken + 7, device="cuda")) % blocks] = names[owned:]
    was, was_ring = tables.clone(), ring.clone()
    tokens = torch.where(lengths > held, lengths - held, 0)
    total = int(tokens.sum())
    kept, after = torch.full_like(held, -1), ints([0, 0])
    slots, starts = torch.zeros(total + 5, dtype=I64, device="cuda"), torch.zeros(n + 1, dtype=I64, device="cuda")
    KvBlockTables(gpu_lib, blocks=blocks, block_size=size).resize(tables, held, lengths, ring, ints([start, taken + 7]), kept=kept, cursor_after=after,
                                                                  slots=slots, starts=starts)
    torch.cuda.synchronize()
    assert torch.equal(kept, lengths) and after.tolist() == [(start + taken) % blocks, 7 + given]
    assert torch.equal(starts[1:], tokens.cumsum(0)) and int(starts[0]) == 0
    at = ((take.cumsum(0) - take)[:, None] + col - before[:, None]).clamp(0, blocks - 1)
    grown = (col >= before[:, None]) & (col < (before + take)[:, None])
    assert torch.equal(tables, torch.where(grown, was_ring[(start + at) % blocks], was))
    returned = was[(col >= behind[:, None]) & (col < before[:, None])]
    want = was_ring.clone()
    want[(start + taken + 7 + torch.arange(given, device="cuda")) % blocks] = returned
    assert torch.equal(ring, want)
    r = torch.repeat_interleave(torch.arange(n, device="cuda"), tokens.long())
    token = held[r] + torch.arange(total, device="cuda") - starts[r]
    assert torch.equal(slots[:total], tables[r, token // size].long() * size + token % size) and bool((slots[total:] == -1).all())
