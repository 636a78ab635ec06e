"""KV codec kernels against records and values in plain numpy (kv_ref: 64 bits up to the rounding to a code).

Codes, scales and record bytes are the definition's, so records are compared byte for byte, and values
read back bit for bit (one product in float32 and one rounding to the type on both sides): no tolerance but the sign
of an fp8 zero, which test_zeros_keep_their_sign alone compares."""

import threading

import kv_ref
import numpy as np
import pytest
import torch

from confkv_b200.kv_codec import KvCodec, PagedKvCache

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GUARD = 0xA5


@pytest.fixture
def make(gpu_lib):
    def make(fmt, dtype, planes, layers, heads, head_dim):
        return KvCodec(gpu_lib, fmt, DTYPES.get(dtype, dtype), planes=planes, layers=layers, heads=heads, head_dim=head_dim)
    return make


def values(shape, dtype, seed):
    """Vectors of very different sizes, with exact ties (halves of the largest), zeros and a zero vector among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn((*shape[:-1], 1), generator=g))
    x = x.to(dtype)
    flat = x.view(-1, shape[-1]) if x.numel() else x.reshape(0, shape[-1])
    for k in range(0, len(flat), 3):
        amax = flat[k].abs().max()
        flat[k, -1] = -amax / 2
        flat[k, 0] = amax
    if len(flat) > 4:
        flat[4] = 0
    return x


def guarded(n, count=1):
    """[count, n] records at a stride with guard bytes around them, and a check that the guards still stand."""
    stride = n + 48
    raw = torch.full((64 + count * stride,), GUARD, dtype=torch.uint8, device="cuda")
    view = raw[64 - 16:64 - 16 + count * stride].view(count, stride)[:, 16:16 + n]
    mask = torch.zeros_like(raw, dtype=torch.bool)
    mask[64 - 16:64 - 16 + count * stride].view(count, stride)[:, 16:16 + n] = True

    def check():
        assert bool((raw[~mask] == GUARD).all()), "wrote outside the record"
    return view, check


def bits(t):
    """Bit patterns, any NaN as one."""
    t = t.detach().cpu().contiguous()
    t = torch.where(torch.isnan(t), torch.full_like(t, float("nan")), t)
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


def assert_record(got, x, fmt):
    n = x.shape[:4].numel()
    want = kv_ref.record(x, fmt)
    got = got.cpu().numpy()[:len(want)]
    assert kv_ref.same_record(got, want, fmt, x.shape[-1], n), np.nonzero(got != want)[0][:8]


def round_trip(codec, x, device_view=None):
    """Write x's record, check it, read it back into a guarded copy and check that."""
    fmt, dtype = codec.format, codec.dtype
    src = x.cuda() if device_view is None else device_view
    size = codec.record_bytes(x.shape[2])
    rec, check = guarded(size)
    codec.quantise(src, rec[0])
    torch.cuda.synchronize()
    check()
    assert_record(rec[0], x, fmt)
    pad = torch.full((x.numel() + 64,), 7.0, dtype=dtype, device="cuda")
    out = pad[32:32 + x.numel()].view(x.shape)
    ok = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    codec.dequantise(rec[0], out, ok=ok)
    torch.cuda.synchronize()
    assert int(ok) == 1
    assert bool((pad[:32] == 7).all()) and bool((pad[32 + x.numel():] == 7).all()), "wrote outside the object"
    assert torch.equal(bits(out), bits(kv_ref.read(rec[0].cpu().numpy(), fmt, dtype, x.shape)))
    return out


# head sizes: one value, around a block, a chunk and a warp, odd ones, several chunks a lane, the largest group, beyond it
HEAD_DIMS = [1, 2, 3, 7, 8, 15, 16, 17, 24, 31, 32, 33, 40, 48, 63, 64, 65, 72, 80, 96, 100, 112, 127, 128, 129, 160, 192, 200, 256,
             272, 320, 500, 512, 520, 576, 768, 1000, 1024, 1040, 1536, 1552, 2050, 5000,
             # every number of granules a lane, for granules of 1, 2, 4 and 8 values
             34, 36, 50, 56, 60, 66, 68, 77, 88, 104, 108, 120, 126, 136, 201, 202, 204, 264, 400, 700, 1200, 1600, 2000, 2560, 2576,
             # the largest groups of small granules, and what they no longer hold
             44, 94, 140, 145, 172, 191, 257, 258, 260, 301, 386, 511, 513, 514, 516, 770, 772, 777, 1026, 1028]


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_head_sizes(make, fmt, dtype, d):
    x = values((2, 3, 5, 3, d), DTYPES[dtype], seed=d)
    round_trip(make(fmt, dtype, 2, 3, 3, d), x)


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 0, 1, 64), (2, 2, 0, 3, 33), (1, 1, 1, 1, 1), (1, 1, 1, 1, 128), (2, 32, 1, 8, 128), (2, 4, 256, 8, 64),
                                   (1, 1, 1031, 1, 320), (2, 80, 17, 1, 128), (1, 3, 257, 5, 96)], ids=str)
def test_shapes(make, fmt, dtype, shape):
    round_trip(make(fmt, dtype, *shape[:2], *shape[3:]), values(shape, DTYPES[dtype], seed=11))


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [33, 64, 128])
def test_values_that_are_not_finite_and_extremes(make, fmt, dtype, d):
    t = DTYPES[dtype]
    x = values((1, 2, 6, 4, d), t, seed=3)
    f = torch.finfo(t)
    flat = x.view(-1, d)
    flat[0, 5] = float("nan")
    flat[1, d - 1] = float("inf")
    flat[2, 0] = -float("inf")
    flat[3, :] = float("nan")
    flat[5, 7] = f.max
    flat[6, 7] = -f.max
    flat[7, :] = f.max
    flat[8, :] = f.smallest_normal
    flat[9, :] = 0
    flat[9, 3] = f.smallest_normal * f.eps          # the least subnormal
    flat[10] = torch.linspace(-1, 1, d).to(t) * f.smallest_normal
    flat[11] = -0.0
    flat[12] = 0
    flat[12, 1] = -0.0
    flat[13, 2] = -float("nan")
    out = round_trip(make(fmt, dtype, 1, 2, 4, d), x).view(-1, d).cpu()
    lost = torch.isnan(out).any(-1)
    assert lost[[0, 1, 2, 3, 13]].all() and not lost[4:13].any()
    if fmt != "mxfp4":
        assert torch.isnan(out[:4]).all()
        # code 127 (448) times its scale is the largest value again, not infinity; in float32 the scale, rounded
        # down, loses less than 2^-23 of its size and the product 2^-24
        assert bool((out[7].double() >= flat[7].double() * (1 - (2.0 ** -22 if dtype == "fp32" else 0))).all())
        assert bool((out[7] <= flat[7]).all())
    assert torch.isfinite(out[5:8]).all()
    assert not out[11].any() and not out[4].any()


def test_ties_go_to_even(make):
    """A = 127 makes codes of the values themselves; A = 448 e4m3 ones; A = 6 (e = 0) e2m1 ones."""
    def one(fmt, vals, d):
        x = torch.zeros(1, 1, 1, 1, d, dtype=torch.float32)
        x[..., :len(vals)] = torch.tensor(vals)
        return round_trip(make(fmt, "fp32", 1, 1, 1, d), x).view(-1)[:len(vals)].cpu().tolist()

    assert one("int8", [127, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, 62.5, 126.5], 16) == [127, 0, 2, 2, 0, -2, 64, 62, 126]
    assert one("fp8", [448, 1.0625, 1.1875, 17, 19, -17, 2 ** -10, 3 * 2 ** -10, 432], 16) == \
        [448, 1, 1.25, 16, 20, -16, 0, 2 * 2 ** -9, 448]
    assert one("mxfp4", [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 0.2500001, 7.9], 32) == \
        [6, 0, 1, 1, 2, 2, 4, 4, -4, 0.5, 6]


def quotients(dtype, firsts, gaps, exponent):
    """Vectors of 64: a largest value (every one of `firsts`, whole numbers of the type's bits, times 2^exponent) and all
    values of the type below it in `gaps` binades, of both signs in turns."""
    bits_ = {torch.bfloat16: 8, torch.float16: 11}[dtype]
    m = torch.arange(1 << (bits_ - 1), 1 << bits_, dtype=torch.float64)
    rows = []
    for a in firsts:
        x = torch.cat([m[m <= a]] + [m * 2.0 ** -g for g in range(1, gaps)])
        x = torch.nn.functional.pad(x, (0, -len(x) % 63)).view(-1, 63)
        x[:, 1::2] *= -1
        rows.append(torch.cat([torch.full((len(x), 1), float(a), dtype=torch.float64), x], 1))
    return (torch.cat(rows) * 2.0 ** exponent).to(dtype)


@pytest.mark.parametrize("fmt,gaps", [("int8", 10), ("fp8", 20)])
@pytest.mark.parametrize("exponent", [-7, 110, -110])
def test_every_code_of_bfloat16(make, fmt, gaps, exponent):
    x = quotients(torch.bfloat16, range(128, 256), gaps, exponent).view(1, 1, -1, 1, 64)
    round_trip(make(fmt, "bf16", 1, 1, 1, 64), x)


@pytest.mark.parametrize("fmt,gaps", [("int8", 10), ("fp8", 10)])
def test_codes_of_half(make, fmt, gaps):
    """All multiples of 127 and of 7 times a power of two among the largest values, their neighbours, and some others."""
    firsts = {k * 127 + o for k in range(9, 17) for o in (-1, 0, 1)} | {1024, 1025, 1120, 1344, 1568, 1792, 1793, 2047} | set(range(1030, 2048, 97))
    x = quotients(torch.float16, sorted(f for f in firsts if 1024 <= f < 2048), gaps, -10).view(1, 1, -1, 1, 64)
    round_trip(make(fmt, "fp16", 1, 1, 1, 64), x)


def test_errors_are_within_half_a_step(make):
    """Against the source itself, with bounds from the formats: A / 254; 2^-4 of the value or half of e4m3's least
    step; a quarter of the value, half of e2m1's least step, or what saturates (A < 8 2^e, the largest code 6 2^e). To
    these 2^-9 of the value for its rounding to bfloat16 and 2^-22 for the scale's and the product's."""
    x = values((2, 4, 64, 8, 128), torch.bfloat16, seed=8)
    for fmt in kv_ref.FORMATS:
        y = round_trip(make(fmt, "bf16", 2, 4, 8, 128), x).cpu().double()
        v, a = x.double().abs(), x.double().abs().amax(-1, keepdim=True)
        err = (x.double() - y).abs()
        if fmt == "mxfp4":
            blocks = v.unflatten(-1, (4, 32))
            unit = torch.where(blocks.amax(-1, keepdim=True) > 0, 2.0 ** (torch.floor(torch.log2(blocks.amax(-1, keepdim=True))) - 2), 0)
            unit = unit.expand_as(blocks).flatten(-2)
            bound = torch.maximum(torch.maximum(v / 4, unit / 4), torch.where(v > 6 * unit, 2 * unit, 0 * unit))
        else:
            bound = a / 254 if fmt == "int8" else torch.maximum(v / 16, a / 448 * 2.0 ** -10)
        assert bool((err <= bound + y.abs() * (2.0 ** -8 + 2.0 ** -22)).all())


# ------------------------------------------------------------ strides and batches

def views(x):
    """The same values with other strides: [name, device view]."""
    planes, layers, tokens, heads, d = x.shape
    yield "tokens first", x.permute(2, 0, 1, 3, 4).contiguous().cuda().permute(1, 2, 0, 3, 4)
    yield "heads before tokens", x.transpose(2, 3).contiguous().cuda().transpose(2, 3)
    for off in (1, 4, 8):
        wide = torch.full((*x.shape[:-1], d + 24), float("nan"), dtype=x.dtype, device="cuda")
        wide[..., off:off + d] = x.cuda()
        yield f"inside wider vectors at {off}", wide[..., off:off + d]
    raw = torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")
    raw[3:].copy_(x.reshape(-1))
    yield "three elements behind the allocation", raw[3:].view(x.shape)


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 40, 33])
def test_strided_objects(make, fmt, dtype, d):
    x = values((2, 3, 9, 4, d), DTYPES[dtype], seed=d)
    codec = make(fmt, dtype, 2, 3, 4, d)
    for name, view in views(x):
        assert torch.equal(bits(view), bits(x)), name
        size = codec.record_bytes(9)
        rec, check = guarded(size)
        codec.quantise(view, rec[0])
        check()
        assert_record(rec[0], x, fmt)
        # and back through the same strides, over other values
        whole = view._base if view._base is not None else view
        before = whole.clone()
        view.fill_(5)
        codec.dequantise(rec[0], view)
        want = kv_ref.read(rec[0].cpu().numpy(), fmt, DTYPES[dtype], x.shape)
        assert torch.equal(bits(view), bits(want)), name
        view.copy_(x)
        assert torch.equal(bits(whole), bits(before)), f"{name}: wrote beside the object"


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_objects_of_unequal_alignment_in_one_call(make, fmt):
    """Aligned and misaligned objects in turns, each to its own record."""
    d = 64
    codec = make(fmt, "bf16", 1, 2, 3, d)
    xs = [values((1, 2, 20 + k, 3, d), torch.bfloat16, seed=k) for k in range(9)]
    held, views_, recs, outs = [], [], [], []
    for k, x in enumerate(xs):
        for into in (views_, outs):
            raw = torch.full((x.numel() + 64,), 2.0, dtype=torch.bfloat16, device="cuda")
            held.append(raw)
            into.append(raw[(0, 1, 8, 16)[k % 4]:][:x.numel()].view(x.shape))
        views_[k].copy_(x)
        recs.append(torch.zeros(codec.record_bytes(20 + k), dtype=torch.uint8, device="cuda"))
    codec.quantise(views_, recs)
    codec.dequantise(recs, outs)
    for x, r, o in zip(xs, recs, outs):
        assert_record(r, x, fmt)
        assert torch.equal(bits(o), bits(kv_ref.read(r.cpu().numpy(), fmt, torch.bfloat16, x.shape)))
    for raw in held:
        inside = raw.numel() - 64
        assert int((raw == 2.0).sum()) >= raw.numel() - inside


def test_broadcast_source(make):
    """A source may share memory with itself (stride 0): one key head for all."""
    x = values((1, 2, 7, 1, 128), torch.bfloat16, seed=1)
    codec = make("int8", "bf16", 1, 2, 4, 128)
    rec = torch.empty(codec.record_bytes(7), dtype=torch.uint8, device="cuda")
    codec.quantise(x.cuda().expand(1, 2, 7, 4, 128), rec)
    assert_record(rec, x.expand(1, 2, 7, 4, 128), "int8")


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("d", [64, 100])
def test_many_objects_of_mixed_sizes_in_one_call(make, fmt, d):
    """Rows of objects and single ones, more than a launch's parameters hold, empty ones among them."""
    codec = make(fmt, "bf16", 2, 2, 3, d)
    counts = [(None, 5), (4, 16), (None, 0), (3, 0), (1, 1), (7, 33), (None, 256)] * 3 + [(0, 4), (None, 2)] * 8
    xs = [values((2, 2, t, 3, d) if n is None else (n, 2, 2, t, 3, d), torch.bfloat16, seed=i) for i, (n, t) in enumerate(counts)]
    recs, checks, oks, outs = [], [], [], []
    for (n, t), x in zip(counts, xs):
        r, check = guarded(codec.record_bytes(t), 1 if n is None else n)
        recs.append(r[0] if n is None else r)
        checks.append(check)
        oks.append(torch.full((1 if n is None else n,), 9, dtype=torch.int32, device="cuda"))
        outs.append(torch.full(x.shape, 3.0, dtype=torch.bfloat16, device="cuda"))
    codec.quantise([x.cuda() for x in xs], recs)
    codec.dequantise(recs, outs, ok=oks)
    torch.cuda.synchronize()
    for (n, t), x, r, check, ok, out in zip(counts, xs, recs, checks, oks, outs):
        check()
        assert bool((ok == 1).all())
        for k in range(1 if n is None else n):
            xk, rk, ok_ = (x, r, out) if n is None else (x[k], r[k], out[k])
            assert_record(rk, xk, fmt)
            assert torch.equal(bits(ok_), bits(kv_ref.read(rk.cpu().numpy(), fmt, torch.bfloat16, xk.shape)))


# ------------------------------------------------------------ records that are not the reader's

@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("d", [64, 33])
def test_foreign_records_read_as_zeros(make, fmt, d):
    codec = make(fmt, "bf16", 2, 2, 3, d)
    x = values((6, 2, 2, 7, 3, d), torch.bfloat16, seed=2)
    rec = torch.empty(6, codec.record_bytes(7), dtype=torch.uint8, device="cuda")
    codec.quantise(x.cuda(), rec)
    rec[1] = 0                                      # a rejected frame's plaintext
    rec[2, 0] ^= 1                                  # another magic word
    rec[3, 4] = 8                                   # another number of tokens
    rec[4, 14] ^= 1                                 # another format
    ok = torch.full((6,), 9, dtype=torch.int32, device="cuda")
    out = torch.full((6, 2, 2, 7, 3, d), 3.0, dtype=torch.bfloat16, device="cuda")
    codec.dequantise(rec, out, ok=ok)
    assert ok.tolist() == [1, 0, 0, 0, 0, 1]
    assert not out[1:5].any()
    for k in (0, 5):
        assert torch.equal(bits(out[k]), bits(kv_ref.read(rec[k].cpu().numpy(), fmt, torch.bfloat16, x.shape[1:])))
    # a codec of another type or head count refuses the same bytes, even where the sizes agree
    for other in (make(fmt, "fp16", 2, 2, 3, d), make(fmt, "bf16", 2, 3, 2, d), make(fmt, "bf16", 1, 4, 3, d)):
        out = torch.full((other.planes, other.layers, 7, other.heads, d), 3.0, dtype=other.dtype, device="cuda")
        verdict = torch.full((1,), 9, dtype=torch.int32, device="cuda")
        other.dequantise(rec[0], out, ok=verdict)
        assert int(verdict) == 0 and not out.any()


# ------------------------------------------------------------ paged caches

def paged(layers, planes, blocks, size, heads, d, dtype, order, seed):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, planes, blocks, size, heads, d)
    pool = torch.randn(shape, generator=g).to(dtype)
    if order == "HND":
        return pool, pool.transpose(3, 4).contiguous().cuda().transpose(3, 4)
    return pool, pool.cuda()


def by_slots(pool, slots):
    """The object of a host pool's slots, zeros for those that are not there: [planes, layers, tokens, heads, d]."""
    layers, planes, blocks, size, heads, d = pool.shape
    flat = pool.reshape(layers, planes, blocks * size, heads, d)
    there = (slots >= 0) & (slots < blocks * size)
    x = flat[:, :, slots.clamp(0, blocks * size - 1)] * there[:, None, None].to(pool.dtype)
    return torch.where(there[:, None, None], x, torch.zeros((), dtype=pool.dtype)).transpose(0, 1).contiguous()


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["NHD", "HND"])
@pytest.mark.parametrize("size,heads,d", [(16, 8, 128), (1, 1, 64), (7, 3, 33), (48, 2, 96), (64, 1, 320)])
def test_paged_round_trip(make, fmt, dtype, order, size, heads, d):
    t = DTYPES[dtype]
    layers, planes, blocks = 3, 2, 11
    codec = make(fmt, dtype, planes, layers, heads, d)
    host, pool = paged(layers, planes, blocks, size, heads, d, t, order, seed=size)
    cache = PagedKvCache(codec, list(pool.unbind(0)))
    total = blocks * size
    slots = torch.randperm(total, generator=torch.Generator().manual_seed(d))[:max(1, total - 5)]
    slots[::4] = -1                                 # padding
    if len(slots) > 2:
        slots[1], slots[2] = total, 1 << 40         # outside the cache
    rec, check = guarded(codec.record_bytes(len(slots)))
    codec.quantise_paged(cache, slots.cuda(), rec[0])
    torch.cuda.synchronize()
    check()
    x = by_slots(host, slots)
    assert_record(rec[0], x, fmt)

    # into another cache, whose other slots keep their bits
    before, dst = paged(layers, planes, blocks, size, heads, d, t, order, seed=99)
    ok = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    codec.dequantise_paged(rec[0], PagedKvCache(codec, [tuple(l.unbind(0)) for l in dst.unbind(0)]), slots.cuda(), ok=ok)
    assert int(ok) == 1
    want = before.reshape(layers, planes, total, heads, d).clone()
    read = kv_ref.read(rec[0].cpu().numpy(), fmt, t, x.shape).transpose(0, 1)
    there = ((slots >= 0) & (slots < total)).nonzero().flatten()
    want[:, :, slots[there]] = read[:, :, there]
    assert torch.equal(bits(dst), bits(want.view(before.shape)))


def test_paged_batches_and_foreign_records(make):
    """A request's chunks in one call (whole ones as a row, the short last one), one of them foreign: its slots are zeroed,
    those of the others restored, the rest left alone."""
    layers, planes, blocks, size, heads, d = 2, 2, 20, 16, 4, 64
    codec = make("int8", "bf16", planes, layers, heads, d)
    host, pool = paged(layers, planes, blocks, size, heads, d, torch.bfloat16, "NHD", seed=1)
    order = torch.randperm(blocks * size, generator=torch.Generator().manual_seed(2))
    rows, tail = order[:192].view(3, 64), order[192:205]
    recs = [torch.empty(3, codec.record_bytes(64), dtype=torch.uint8, device="cuda"),
            torch.empty(codec.record_bytes(13), dtype=torch.uint8, device="cuda")]
    cache = PagedKvCache(codec, list(pool.unbind(0)))
    codec.quantise_paged(cache, [rows.cuda(), tail.cuda()], recs)
    for k in range(3):
        assert_record(recs[0][k], by_slots(host, rows[k]), "int8")
    assert_record(recs[1], by_slots(host, tail), "int8")
    recs[0][1] = 0
    ok = [torch.full((3,), 9, dtype=torch.int32, device="cuda"), torch.full((1,), 9, dtype=torch.int32, device="cuda")]
    pool.fill_(3)
    codec.dequantise_paged(recs, cache, [rows.cuda(), tail.cuda()], ok=ok)
    assert ok[0].tolist() == [1, 0, 1] and ok[1].tolist() == [1]
    want = torch.full((layers, planes, blocks * size, heads, d), 3.0, dtype=torch.bfloat16)
    for s, r in ((rows[0], recs[0][0]), (rows[1], None), (rows[2], recs[0][2]), (tail, recs[1])):
        shape = (planes, layers, len(s), heads, d)
        want[:, :, s] = 0 if r is None else kv_ref.read(r.cpu().numpy(), "int8", torch.bfloat16, shape).transpose(0, 1)
    assert torch.equal(bits(pool), bits(want.view(pool.shape)))


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_blocks_that_hold_keys_and_values(make, fmt):
    """[blocks, 2, block_size, heads, head_dim] seen as [2, blocks, ...], out and back into another such cache."""
    codec = make(fmt, "bf16", 2, 3, 2, 80)
    host = torch.randn(3, 2, 7, 16, 2, 80, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    pool = host.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    slots = torch.randperm(7 * 16, generator=torch.Generator().manual_seed(4))[:50]
    rec = torch.empty(codec.record_bytes(50), dtype=torch.uint8, device="cuda")
    codec.quantise_paged(PagedKvCache(codec, list(pool.unbind(0))), slots.cuda(), rec)
    x = by_slots(host, slots)
    assert_record(rec, x, fmt)
    dst = torch.full((3, 7, 2, 16, 2, 80), 3.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    codec.dequantise_paged(rec, PagedKvCache(codec, list(dst.unbind(0))), slots.cuda())
    want = torch.full((3, 2, 7 * 16, 2, 80), 3.0, dtype=torch.bfloat16)
    want[:, :, slots] = kv_ref.read(rec.cpu().numpy(), fmt, torch.bfloat16, x.shape).transpose(0, 1)
    assert torch.equal(bits(dst), bits(want.view(3, 2, 7, 16, 2, 80)))


def test_slots_of_rows_at_a_distance(make):
    """A request table's rows: slots [n, tokens] inside a wider matrix."""
    codec = make("fp8", "bf16", 1, 2, 2, 64)
    host, pool = paged(2, 1, 8, 16, 2, 64, torch.bfloat16, "NHD", seed=4)
    table = torch.randperm(128, generator=torch.Generator().manual_seed(5)).view(4, 32).cuda()
    rec = torch.empty(4, codec.record_bytes(9), dtype=torch.uint8, device="cuda")
    codec.quantise_paged(PagedKvCache(codec, [l[0] for l in pool.unbind(0)]), table[:, 3:12], rec)
    for k in range(4):
        assert_record(rec[k], by_slots(host, table[k, 3:12].cpu()), "fp8")


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_no_tokens_and_no_pages(make, fmt):
    """Empty slots, and a cache without blocks, whose every slot is outside it."""
    codec = make(fmt, "bf16", 2, 3, 2, 64)
    _, pool = paged(3, 2, 4, 16, 2, 64, torch.bfloat16, "NHD", seed=1)
    before = pool.clone()
    cache = PagedKvCache(codec, list(pool.unbind(0)))
    nothing = PagedKvCache(codec, list(pool[:, :, :0].unbind(0)))
    slots = torch.empty(0, dtype=torch.int64, device="cuda")
    some = torch.tensor([0, 5, -1], device="cuda")
    rec = torch.full((codec.record_bytes(0),), 7, dtype=torch.uint8, device="cuda")
    codec.quantise_paged(cache, slots, rec)
    assert rec.cpu().numpy().tobytes() == kv_ref.header(fmt, torch.bfloat16, 2, 3, 0, 2, 64).tobytes()
    ok = torch.zeros(1, dtype=torch.int32, device="cuda")
    codec.dequantise_paged(rec, cache, slots, ok=ok)
    assert int(ok) == 1
    big = torch.full((codec.record_bytes(3),), 7, dtype=torch.uint8, device="cuda")
    codec.quantise_paged(nothing, some, big)
    assert_record(big, torch.zeros(2, 3, 3, 2, 64, dtype=torch.bfloat16), fmt)
    ok.zero_()
    codec.dequantise_paged(big, nothing, some, ok=ok)
    assert int(ok) == 1 and torch.equal(pool, before)
    # and rows of no objects
    codec.quantise(torch.empty(0, 2, 3, 4, 2, 64, dtype=torch.bfloat16, device="cuda"),
                   torch.empty(0, codec.record_bytes(4), dtype=torch.uint8, device="cuda"))
    codec.quantise([], [])


def test_a_nan_in_a_slot_that_is_not_named_stays_out(make):
    codec = make("int8", "bf16", 1, 1, 1, 64)
    pool = torch.full((1, 1, 4, 16, 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool[0, 0, 2, 3] = 1.0
    slots = torch.tensor([-1, 2 * 16 + 3, 64], device="cuda")
    rec = torch.empty(codec.record_bytes(3), dtype=torch.uint8, device="cuda")
    codec.quantise_paged(PagedKvCache(codec, list(pool.unbind(0))), slots, rec)
    _, scales = codec.split(rec, 3)
    assert scales.flatten().tolist() == [0.0, float(np.float32(1) / np.float32(127)), 0.0]


def test_offsets_beyond_32_bits(make):
    """Slots and objects that start more than 2^32 bytes behind their cache's or tensor's first element."""
    heads, d, size = 8, 128, 16
    codec = make("int8", "bf16", 1, 1, heads, d)
    blocks = (6 << 30) // (size * heads * d * 2)
    plane = torch.empty(blocks, size, heads, d, dtype=torch.bfloat16, device="cuda")
    total = blocks * size
    slots = torch.tensor([0, total - 1, total // 2, (1 << 32) // (heads * d * 2), (1 << 31) // (heads * d), total - 17])
    x = values((1, 1, len(slots), heads, d), torch.bfloat16, seed=6)
    flat = plane.view(total, heads, d)
    flat[slots.cuda()] = x[0, 0].cuda()
    x = flat[slots.cuda()].cpu()[None, None]        # two of the slots are the same one
    rec = torch.empty(codec.record_bytes(len(slots)), dtype=torch.uint8, device="cuda")
    cache = PagedKvCache(codec, [plane])
    codec.quantise_paged(cache, slots.cuda(), rec)
    assert_record(rec, x, "int8")
    flat[slots.cuda()] = 3
    codec.dequantise_paged(rec, cache, slots.cuda())
    want = kv_ref.read(rec.cpu().numpy(), "int8", torch.bfloat16, x.shape)
    assert torch.equal(bits(flat[slots.cuda()]), bits(want[0, 0]))
    # strided: two objects 5 GiB apart
    row = flat.as_strided((2, 1, 1, 3, heads, d), ((5 << 30) // 2, 1, 1, heads * d, d, 1))
    row.copy_(x[None, :, :, :3].expand(2, 1, 1, 3, heads, d))
    recs = torch.empty(2, codec.record_bytes(3), dtype=torch.uint8, device="cuda")
    codec.quantise(row, recs)
    for k in range(2):
        assert_record(recs[k], x[:, :, :3], "int8")
    row.fill_(2)
    codec.dequantise(recs, row)
    assert torch.equal(bits(row[1]), bits(kv_ref.read(recs[1].cpu().numpy(), "int8", torch.bfloat16, (1, 1, 3, heads, d))))


def test_more_vectors_than_a_launch_numbers(make):
    """Three objects of 2^30 vectors each in one row: 2^31 and more vectors are cut into several launches."""
    tokens, heads = 1 << 20, 1 << 10
    codec = make("int8", "bf16", 1, 1, heads, 1)
    source = torch.tensor([2.0, -3.0, 5.0], dtype=torch.bfloat16, device="cuda").view(3, 1, 1, 1, 1, 1)
    recs = torch.empty(3, codec.record_bytes(tokens), dtype=torch.uint8, device="cuda")
    codec.quantise(source.expand(3, 1, 1, tokens, heads, 1), recs)
    codes, scales = codec.split(recs, tokens)
    for k, (code, amax) in enumerate(((127, 2.0), (-127, 3.0), (127, 5.0))):
        assert kv_ref.HEADER == 32 and recs[k, :16].cpu().numpy().tobytes() == \
            kv_ref.header("int8", torch.bfloat16, 1, 1, tokens, heads, 1)[:16].tobytes()
        assert bool((codes[k] == code).all())
        assert bool((scales[k] == float(np.float32(amax) / np.float32(127))).all())
    # read back the last object alone, into every second place of a tensor
    out = torch.full((1, 1, tokens, heads, 2), 9.0, dtype=torch.bfloat16, device="cuda")
    codec.dequantise(recs[2], out[..., :1])
    assert bool((out[..., 0] == 5).all()) and bool((out[..., 1] == 9).all())


# ------------------------------------------------------------ streams, graphs, threads

def test_calls_follow_their_stream(make):
    """Write, read and the producer of the source on one side stream, behind a long kernel, without a wait between."""
    codec = make("fp8", "bf16", 2, 8, 8, 128)
    x = values((2, 8, 64, 8, 128), torch.bfloat16, seed=7)
    src, out = torch.zeros(x.shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(x.shape, dtype=torch.bfloat16, device="cuda")
    xd = x.cuda()
    rec = torch.zeros(codec.record_bytes(64), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)
        src.copy_(xd)
        codec.quantise(src, rec)                    # the current stream
    codec.dequantise(rec, out, stream=s)
    s.synchronize()
    assert_record(rec, x, "fp8")
    assert torch.equal(bits(out), bits(kv_ref.read(rec.cpu().numpy(), "fp8", torch.bfloat16, x.shape)))


def test_graph_replays_take_new_values(make):
    """Paged write and read captured together; each replay takes what the cache and the slots then hold."""
    layers, planes, blocks, size, heads, d = 4, 2, 12, 16, 4, 128
    codec = make("int8", "fp16", planes, layers, heads, d)
    _, pool = paged(layers, planes, blocks, size, heads, d, torch.float16, "NHD", seed=1)
    _, dst = paged(layers, planes, blocks, size, heads, d, torch.float16, "HND", seed=2)
    a, b = PagedKvCache(codec, list(pool.unbind(0))), PagedKvCache(codec, list(dst.unbind(0)))
    slots = torch.arange(40, device="cuda")
    rec = torch.zeros(codec.record_bytes(40), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        codec.quantise_paged(a, slots, rec)
        codec.dequantise_paged(rec, b, slots)
    del a, b                                        # the graph keeps the addresses, not the bindings
    for seed in range(3):
        host = torch.randn(pool.shape, generator=torch.Generator().manual_seed(seed)).half()
        new = torch.randperm(blocks * size, generator=torch.Generator().manual_seed(seed))[:40]
        pool.copy_(host)
        slots.copy_(new)
        dst.fill_(1)
        g.replay()
        torch.cuda.synchronize()
        x = by_slots(host, new)
        assert_record(rec, x, "int8")
        want = torch.ones(layers, planes, blocks * size, heads, d, dtype=torch.float16)
        want[:, :, new] = kv_ref.read(rec.cpu().numpy(), "int8", torch.float16, x.shape).transpose(0, 1)
        assert torch.equal(bits(dst), bits(want.view(dst.shape)))


def test_threads_share_a_codec(make):
    codec = make("mxfp4", "bf16", 2, 4, 8, 64)
    xs = [values((2, 4, 100 + k, 8, 64), torch.bfloat16, seed=k) for k in range(4)]
    device = [x.cuda() for x in xs]
    recs = [torch.zeros(codec.record_bytes(x.shape[2]), dtype=torch.uint8, device="cuda") for x in xs]
    outs = [torch.zeros_like(x) for x in device]
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            s = torch.cuda.Stream()
            for _ in range(50):
                codec.quantise(device[k], recs[k], stream=s)
                codec.dequantise(recs[k], outs[k], stream=s)
            s.synchronize()
        except Exception as e:  # pragma: no cover - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for x, r, o in zip(xs, recs, outs):
        assert_record(r, x, "mxfp4")
        assert torch.equal(bits(o), bits(kv_ref.read(r.cpu().numpy(), "mxfp4", torch.bfloat16, x.shape)))


def test_same_calls_give_the_same_bytes(make):
    codec = make("fp8", "bf16", 2, 8, 8, 128)
    x = values((2, 8, 333, 8, 128), torch.bfloat16, seed=9).cuda()
    recs = torch.zeros(4, codec.record_bytes(333), dtype=torch.uint8, device="cuda")
    for k in range(4):
        recs[k].fill_(k)                            # stale bytes do not show
        codec.quantise(x, recs[k])
    assert all(torch.equal(recs[0], recs[k]) for k in range(1, 4))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(gpu_lib):
    codec = KvCodec(gpu_lib, "int8", torch.bfloat16, planes=2, layers=2, heads=4, head_dim=64, device=1)
    x = values((2, 2, 33, 4, 64), torch.bfloat16, seed=1)
    with torch.cuda.device(0):
        rec = torch.zeros(codec.record_bytes(33), dtype=torch.uint8, device="cuda:1")
        out = torch.zeros(x.shape, dtype=torch.bfloat16, device="cuda:1")
        src = x.to("cuda:1")
        codec.quantise(src, rec)                    # cuda:1's current stream
        codec.dequantise(rec, out)
        torch.cuda.synchronize(1)
        assert torch.cuda.current_device() == 0
    assert_record(rec, x, "int8")
    assert torch.equal(bits(out), bits(kv_ref.read(rec.cpu().numpy(), "int8", torch.bfloat16, x.shape)))


def test_codec_and_seal_in_one_graph(make, gpu_lib):
    """Quantise, seal, open and read back captured together: no call waits for the host between them, and a replay
    takes the object's new values."""
    from confkv_b200.gpu_aesgcm import GpuAes128GcmKey

    codec = make("mxfp4", "bf16", 2, 4, 8, 64)
    x = torch.zeros(2, 4, 100, 8, 64, dtype=torch.bfloat16, device="cuda")
    size = codec.record_bytes(100)
    rec, opened = (torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    frame = torch.zeros(size + 29, dtype=torch.uint8, device="cuda")
    auth, ok = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.zeros_like(x)
    s = torch.cuda.Stream()

    def body():
        codec.quantise(x, rec, stream=s)
        key.seal_async(src_ptr=rec.data_ptr(), plaintext_len=size, dst_ptr=frame.data_ptr(), dst_capacity=size + 29,
                       iv=bytes(12), stream_ptr=s.cuda_stream)
        key.open_async(src_ptr=frame.data_ptr(), frame_len=size + 29, dst_ptr=opened.data_ptr(), plaintext_len=size,
                       auth_ok_ptr=auth.data_ptr(), stream_ptr=s.cuda_stream)
        codec.dequantise(opened, out, ok=ok, stream=s)

    with GpuAes128GcmKey(gpu_lib, bytes(range(16))) as key:
        torch.cuda.synchronize()
        body()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            body()
        for seed in range(3):
            host = values(x.shape, torch.bfloat16, seed=seed)
            x.copy_(host)
            for t in (opened, frame, auth, ok, out):
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert int(auth) == 1 and int(ok) == 1
            assert_record(opened, host, "mxfp4")
            assert torch.equal(bits(out), bits(kv_ref.read(opened.cpu().numpy(), "mxfp4", torch.bfloat16, host.shape)))
        del g


# every kernel's way to a code: granules of 16, 8, 4, 2 and 1 values, whole warps, a lane, several vectors a warp
@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 16, 33, 36, 40, 66, 100, 127, 128, 320, 514, 1030, 2576])
def test_zeros_keep_their_sign(make, fmt, dtype, d):
    """Records equal to the reference's in every byte: zeros of both signs, values that round to zero, vectors of nothing
    else."""
    t = DTYPES[dtype]
    x = values((1, 2, 8, 2, d), t, seed=d)
    flat = x.view(-1, d)
    flat[:, d // 2] = -0.0
    flat[8:16] *= torch.where(torch.arange(d) % 3 == 1, 2.0 ** -12, 1.0).to(t)      # below half of the least code
    flat[16] = -0.0
    flat[17] = 0.0
    flat[18] = torch.where(torch.arange(d) % 2 == 0, 0.0, -0.0).to(t)
    flat[19] = -torch.finfo(t).smallest_normal * torch.finfo(t).eps
    flat[20, 0], flat[20, 1:] = torch.finfo(t).max, -torch.finfo(t).smallest_normal
    codec = make(fmt, dtype, 1, 2, 2, d)
    rec = torch.full((codec.record_bytes(8),), GUARD, dtype=torch.uint8, device="cuda")
    codec.quantise(x.cuda(), rec)
    want = kv_ref.record(x, fmt)
    got = rec.cpu().numpy()
    assert np.array_equal(got, want), np.nonzero(got != want)[0][:8]
    if fmt != "int8":
        out = torch.empty_like(x, device="cuda")
        codec.dequantise(rec, out)
        assert bool((torch.signbit(out.cpu()) == torch.signbit(x)).all())


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_neighbours_of_objects_of_unequal_alignment(make, fmt):
    """What lies before and behind each object of a call, aligned or not, keeps its values."""
    d = 64
    codec = make(fmt, "bf16", 1, 2, 3, d)
    xs = [values((1, 2, 20 + k, 3, d), torch.bfloat16, seed=k) for k in range(9)]
    raws, outs, recs, starts = [], [], [], [(0, 1, 8, 16)[k % 4] for k in range(9)]
    for x, at in zip(xs, starts):
        raws.append(torch.full((x.numel() + 64,), 2.0, dtype=torch.bfloat16, device="cuda"))
        outs.append(raws[-1][at:at + x.numel()].view(x.shape))
        recs.append(torch.from_numpy(kv_ref.record(x, fmt)).cuda())
    codec.dequantise(recs, outs)
    for x, r, raw, o, at in zip(xs, recs, raws, outs, starts):
        assert torch.equal(bits(o), bits(kv_ref.read(r.cpu().numpy(), fmt, torch.bfloat16, x.shape)))
        assert bool((raw[:at] == 2).all()) and bool((raw[at + x.numel():] == 2).all())
    # and quantising leaves the sources and their neighbours alone
    before = [raw.clone() for raw in raws]
    codec.quantise(outs, recs)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(before, raws))


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("d", [64, 33, 5000])
def test_a_slot_named_twice_holds_values_of_either_token(make, fmt, d):
    """And no other slot changes; named twice on the way out it is two equal tokens."""
    codec = make(fmt, "bf16", 1, 2, 3, d)
    _, pool = paged(2, 1, 4, 16, 3, d, torch.bfloat16, "NHD", seed=5)
    before = pool.clone()
    cache = PagedKvCache(codec, list(pool.unbind(0)))
    x = values((1, 2, 40, 3, d), torch.bfloat16, seed=6)
    rec = torch.from_numpy(kv_ref.record(x, fmt)).cuda()
    slots = torch.arange(40, device="cuda") // 2 + 7            # pairs of neighbouring tokens
    codec.dequantise_paged(rec, cache, slots)
    want = kv_ref.read(rec.cpu().numpy(), fmt, torch.bfloat16, x.shape)
    got = pool.view(2, 64, 3, d).cpu()
    here = bits(got[:, 7:27])
    a, b = (bits(want[0, :, k::2]) for k in (0, 1))
    assert bool(((here == a) | (here == b)).all())
    rest = torch.ones(64, dtype=torch.bool)
    rest[7:27] = False
    assert torch.equal(bits(got[:, rest]), bits(before.view(2, 64, 3, d).cpu()[:, rest]))
    out = torch.empty(codec.record_bytes(40), dtype=torch.uint8, device="cuda")
    codec.quantise_paged(cache, slots, out)
    assert_record(out, pool.view(2, 64, 3, d)[:, 7:27].repeat_interleave(2, 1).cpu()[None], fmt)
