"""The KV codec's C-ABI and binding without a GPU: symbols, structures, sizes and refusals, all of which come
before any device access."""

import ctypes
import re
from pathlib import Path

import kv_ref
import pytest
import torch

from confkv_b200 import kv_codec
from confkv_b200.gpu_aesgcm import GpuAesGcmError
from confkv_b200.kv_codec import KvCodec, KvLayout, KvPages, PagedKvCache

HEADER = Path(__file__).resolve().parents[1] / "include" / "gpu_kv_codec_api.h"
OK, ERR_ARG = 0, -1


def header_functions():
    return set(re.findall(r"^\s*(?:size_t|int)\s+(lmcache_\w+)\s*\(", HEADER.read_text(), re.M))


@pytest.fixture
def lib(cpu_lib):
    kv_codec._declare(cpu_lib.lib)
    return cpu_lib.lib


def test_header_and_library_agree(cpu_lib):
    assert header_functions() == set(kv_codec.CODEC_SYMBOLS)
    for name in header_functions():
        assert hasattr(cpu_lib.lib, name), name


def test_structures_are_the_headers(tmp_path):
    import subprocess

    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "gpu_kv_codec_api.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n",'
                   "sizeof(lmcache_gpu_kv_layout), sizeof(lmcache_gpu_kv_pages), sizeof(lmcache_gpu_kv_run),"
                   "offsetof(lmcache_gpu_kv_run, slots), offsetof(lmcache_gpu_kv_run, record), offsetof(lmcache_gpu_kv_run, tokens));"
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", "-I", str(HEADER.parent), str(src), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(n) for n in got] == [ctypes.sizeof(KvLayout), ctypes.sizeof(KvPages), kv_codec.RUN.size, 48, 64, 96]


def layout(fmt=0, dtype=0, planes=2, layers=4, heads=8, head_dim=64):
    return KvLayout(fmt, dtype, planes, layers, heads, head_dim)


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_record_size(lib, fmt):
    for planes, layers, heads, d, tokens in ((2, 32, 8, 128, 256), (1, 1, 1, 1, 1), (2, 3, 5, 33, 7), (2, 4, 8, 64, 0)):
        n = planes * layers * heads * tokens
        size = lib.lmcache_gpu_kv_record_size(ctypes.byref(layout(kv_ref.FORMATS.index(fmt), 0, planes, layers, heads, d)), tokens)
        assert size == kv_ref.record_bytes(fmt, d, n)[1]


BAD_LAYOUTS = [dict(fmt=-1), dict(fmt=3), dict(dtype=-1), dict(dtype=3), dict(planes=0), dict(planes=3), dict(layers=0),
               dict(layers=65536), dict(heads=0), dict(heads=65536), dict(head_dim=0), dict(head_dim=65536)]


@pytest.mark.parametrize("bad", BAD_LAYOUTS, ids=str)
def test_bad_layouts(lib, bad):
    b = layout(**bad)
    assert lib.lmcache_gpu_kv_record_size(ctypes.byref(b), 1) == 0
    for f in (lib.lmcache_gpu_kv_quantise_async, lib.lmcache_gpu_kv_dequantise_async):
        assert f(ctypes.byref(b), None, b"", 0, 0, None) == ERR_ARG


def run(obj=0x100000, strides=(0, 1024, 512, 512, 64), slots=0, slots_stride=0, record=0x200000, record_stride=1 << 20,
        record_bytes=1 << 20, ok=0, tokens=1, count=1):
    return kv_codec.RUN.pack(obj, *strides, slots, slots_stride, record, record_stride, record_bytes, ok, tokens, count)


SIZE = kv_ref.record_bytes("int8", 64, 2 * 4 * 8)[1]
BAD_RUNS = [
    dict(obj=0), dict(obj=0x100001), dict(record=0), dict(record=0x200008), dict(record_bytes=SIZE - 1), dict(ok=2),
    dict(strides=(-1, 0, 0, 0, 0)), dict(strides=(0, -1, 0, 0, 0)), dict(strides=(0, 0, -1, 0, 0)),
    dict(strides=(0, 0, 0, -1, 0)), dict(strides=(0, 0, 0, 0, -1)), dict(count=2, record_stride=SIZE - 16),
    dict(count=2, record_stride=-(1 << 20)), dict(count=2, record_stride=(1 << 20) + 8), dict(tokens=1 << 25, record_bytes=1 << 62),
    dict(tokens=(1 << 32) - 1, record_bytes=1 << 62),
]


@pytest.mark.parametrize("bad", BAD_RUNS, ids=str)
def test_bad_runs(lib, bad):
    for f in (lib.lmcache_gpu_kv_quantise_async, lib.lmcache_gpu_kv_dequantise_async):
        # also behind a good run
        assert f(ctypes.byref(layout()), None, run(**bad), 1, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), None, run() + run(**bad), 2, 0, None) == ERR_ARG


def pages(**more):
    bases = (ctypes.c_void_p * 8)(*more.pop("bases", [0x100000 + 0x10000 * k for k in range(8)]))
    p = KvPages(ctypes.addressof(bases), 64, 16, 0, 16 * 512, 512, 64)
    for k, v in more.items():
        setattr(p, k, v)
    p.keep = bases
    return p


BAD_PAGES = [dict(bases=[0x100000] * 7 + [0]), dict(bases=[0x100000] * 7 + [0x100001]), dict(block_size=0),
             dict(blocks=1 << 31), dict(blocks=1 << 28), dict(block_stride=-1), dict(row_stride=-1), dict(head_stride=-1)]


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_bad_pages(lib, bad):
    for f in (lib.lmcache_gpu_kv_quantise_async, lib.lmcache_gpu_kv_dequantise_async):
        assert f(ctypes.byref(layout()), ctypes.byref(pages(**bad)), run(slots=0x300000), 1, 0, None) == ERR_ARG


def test_bad_slots_and_arrays(lib):
    for f in (lib.lmcache_gpu_kv_quantise_async, lib.lmcache_gpu_kv_dequantise_async):
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), run(slots=0), 1, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), run(slots=0x300004), 1, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), run(slots=0x300000, slots_stride=-1), 1, 0, None) == ERR_ARG
        none = KvPages(None, 64, 16, 0, 0, 0, 0)
        assert f(ctypes.byref(layout()), ctypes.byref(none), run(slots=0x300000), 1, 0, None) == ERR_ARG
        # 600 planes do not fit a call
        assert f(ctypes.byref(layout(layers=300)), ctypes.byref(pages()), b"", 0, 0, None) == ERR_ARG
        assert f(None, None, run(), 1, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), None, None, 1, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), None, run(), 1, -1, None) == ERR_ARG
        assert f(ctypes.byref(layout()), None, None, 0, 0, None) == OK                  # nothing to do


class Fake:
    """A tensor's shape, type and place without its memory."""

    def __init__(self, shape, dtype=torch.bfloat16, device="cuda:0", strides=None, ptr=1 << 20):
        self.shape, self.dtype, self.device, self._ptr = torch.Size(shape), dtype, torch.device(device), ptr
        self._strides = tuple(strides) if strides is not None else torch.empty(shape, device="meta").stride()

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, k=None):
        return self._strides if k is None else self._strides[k]

    def data_ptr(self):
        return self._ptr

    def get_device(self):
        return self.device.index if self.device.type == "cuda" else -1

    def is_contiguous(self):
        return self._strides == torch.empty(self.shape, device="meta").stride()


@pytest.fixture
def codec(cpu_lib):
    return KvCodec(cpu_lib, "int8", torch.bfloat16, planes=2, layers=4, heads=8, head_dim=64, device=0)


def test_codec_refuses_bad_configurations(cpu_lib):
    good = dict(planes=2, layers=4, heads=8, head_dim=64)
    for bad in (dict(planes=0), dict(planes=3), dict(layers=0), dict(heads=65536), dict(head_dim=0)):
        with pytest.raises(ValueError):
            KvCodec(cpu_lib, "int8", torch.bfloat16, **{**good, **bad})
    for fmt, dtype, device in (("int4", torch.bfloat16, 0), ("int8", torch.float64, 0), ("fp8", torch.uint8, 0),
                               ("mxfp4", torch.bfloat16, "cpu"), ("mxfp4", torch.bfloat16, "cuda")):
        with pytest.raises(ValueError):
            KvCodec(cpu_lib, fmt, dtype, **good, device=device)


U8, I32, I64 = torch.uint8, torch.int32, torch.int64
SHAPE = (2, 4, 3, 8, 64)
R = kv_ref.record_bytes("int8", 64, 2 * 4 * 3 * 8)[1]
BAD_CALLS = {
    "type": (Fake(SHAPE, torch.float16), Fake((R,), U8), None),
    "device": (Fake(SHAPE, device="cuda:1"), Fake((R,), U8), None),
    "host": (Fake(SHAPE, device="cpu"), Fake((R,), U8), None),
    "dimensions": (Fake((4, 3, 8, 64)), Fake((R,), U8), None),
    "shape": (Fake((2, 4, 3, 8, 32)), Fake((R,), U8), None),
    "vector stride": (Fake(SHAPE, strides=(4 * 3 * 8 * 128, 3 * 8 * 128, 8 * 128, 128, 2)), Fake((R,), U8), None),
    "record type": (Fake(SHAPE), Fake((R,), torch.int8), None),
    "record device": (Fake(SHAPE), Fake((R,), U8, "cuda:1"), None),
    "record room": (Fake(SHAPE), Fake((R - 1,), U8), None),
    "record address": (Fake(SHAPE), Fake((R,), U8, ptr=(1 << 20) + 8), None),
    "record stride": (Fake(SHAPE), Fake((R,), U8, strides=(2,)), None),
    "records": (Fake((3, *SHAPE)), Fake((2, R), U8), None),
    "records overlap": (Fake((2, *SHAPE)), Fake((2, R), U8, strides=(16, 1)), None),
    "records' distance": (Fake((2, *SHAPE)), Fake((2, R), U8, strides=(R + 8, 1)), None),
    "one record for a row": (Fake((2, *SHAPE)), Fake((R,), U8), None),
}
BAD_VERDICTS = {
    "verdict type": (Fake(SHAPE), Fake((R,), U8), Fake((1,), I64)),
    "verdict device": (Fake(SHAPE), Fake((R,), U8), Fake((1,), I32, "cpu")),
    "verdicts": (Fake((2, *SHAPE)), Fake((2, R), U8), Fake((3,), I32)),
    "verdict stride": (Fake((2, *SHAPE)), Fake((2, R), U8), Fake((2,), I32, strides=(2,))),
    "overlapping object": (Fake(SHAPE, strides=(0, 3 * 512, 512, 64, 1)), Fake((R,), U8), None),
}


@pytest.mark.parametrize("name", BAD_CALLS | BAD_VERDICTS)
def test_binding_refuses_bad_objects(codec, name):
    obj, record, ok = (BAD_CALLS | BAD_VERDICTS)[name]
    with pytest.raises(ValueError, match="kv codec"):
        codec.dequantise([record], [obj], ok=None if ok is None else [ok])
    if name in BAD_CALLS:
        with pytest.raises(ValueError, match="kv codec"):
            codec.quantise([obj], [record])


def test_binding_refuses_unequal_lists(codec):
    with pytest.raises(ValueError):
        codec.quantise([Fake(SHAPE)] * 2, [Fake((R,), U8)])
    with pytest.raises(ValueError):
        codec.dequantise([Fake((R,), U8)], [Fake(SHAPE)], ok=[None, None])
    with pytest.raises(ValueError):
        codec.record_bytes(-1)
    with pytest.raises(ValueError):
        codec.record_bytes(1 << 26)                  # 2^32 vectors


PLANE = (2, 9, 16, 8, 64)


def test_binding_refuses_bad_caches(codec, cpu_lib):
    def layers(n=4, **more):
        return [(Fake(PLANE[1:], **more), Fake(PLANE[1:], **more)) for _ in range(n)]

    cache = PagedKvCache(codec, layers())
    for bad in (layers(3), layers(dtype=torch.float16), layers(device="cuda:1"),
                layers(strides=(16 * 8 * 64 * 2, 8 * 64 * 2, 128, 2)),
                layers(3) + [(Fake((9, 32, 8, 64)), Fake((9, 32, 8, 64)))], layers(3) + [(Fake((9, 16, 8, 64)),)],
                [(Fake((9, 16, 4, 64)),) * 2] * 4, [(Fake((9, 16, 8, 32)),) * 2] * 4, [(Fake((1 << 27, 16, 8, 64)),) * 2] * 4):
        with pytest.raises(ValueError, match="kv codec"):
            PagedKvCache(codec, bad)
    many = KvCodec(cpu_lib, "int8", torch.bfloat16, planes=2, layers=300, heads=8, head_dim=64)
    with pytest.raises(ValueError, match="512"):
        PagedKvCache(many, layers(300))
    with pytest.raises(ValueError, match="overlap"):
        shared = PagedKvCache(codec, layers(strides=(8 * 64, 8 * 64, 64, 1)))
        codec.dequantise_paged([Fake((R,), U8)], shared, [Fake((3,), I64)])
    other = KvCodec(cpu_lib, "int8", torch.float16, planes=2, layers=4, heads=8, head_dim=64)
    for call in (lambda c: c.quantise_paged(cache, [Fake((3,), I64)], [Fake((R,), U8)]),
                 lambda c: c.dequantise_paged([Fake((R,), U8)], cache, [Fake((3,), I64)])):
        with pytest.raises(ValueError, match="paged cache"):
            call(other)
    for slots in (Fake((3,), I32), Fake((3,), I64, "cpu"), Fake((1, 1, 3), I64), Fake((3,), I64, strides=(2,))):
        with pytest.raises(ValueError, match="kv codec"):
            codec.quantise_paged(cache, [slots], [Fake((R,), U8)])
        with pytest.raises(ValueError, match="kv codec"):
            codec.dequantise_paged([Fake((R,), U8)], cache, [slots])


def test_caches_of_joint_and_separate_planes(codec, cpu_lib):
    """[planes, ...] tensors, transposed ones, and pairs give the same addresses; a plane that lies on another is not
    written to."""
    block = 16 * 8 * 64
    joint = [Fake((2, 9, 16, 8, 64), ptr=(1 << 20) + (k << 16)) for k in range(4)]
    pairs = [(Fake(PLANE[1:], ptr=(1 << 20) + (k << 16)), Fake(PLANE[1:], ptr=(1 << 20) + (k << 16) + 9 * block * 2)) for k in range(4)]
    a, b = PagedKvCache(codec, joint), PagedKvCache(codec, pairs)
    assert list(a._bases) == list(b._bases) and len(a._bases) == 8
    assert (a._pages.blocks, a._pages.block_size, a._pages.block_stride, a._pages.row_stride, a._pages.head_stride) == \
        (b._pages.blocks, b._pages.block_size, b._pages.block_stride, b._pages.row_stride, b._pages.head_stride) == \
        (9, 16, block, 512, 64)
    mixed = PagedKvCache(codec, joint[:2] + pairs[2:])
    assert list(mixed._bases) == list(a._bases)
    # blocks that hold keys and values, [blocks, 2, ...], seen as [2, blocks, ...]
    inside = [Fake((2, 9, 16, 8, 64), strides=(block, 2 * block, 512, 64, 1), ptr=1 << 20) for _ in range(4)]
    c = PagedKvCache(codec, inside)
    assert c.writable() is c and c._bases[4] - c._bases[0] == block * 2 and c._pages.block_stride == 2 * block
    same = PagedKvCache(codec, [Fake((2, 9, 16, 8, 64), strides=(0, block, 512, 64, 1)) for _ in range(4)])
    with pytest.raises(ValueError, match="overlap"):
        same.writable()
    one = KvCodec(cpu_lib, "int8", torch.bfloat16, planes=1, layers=2, heads=8, head_dim=64)
    assert list(PagedKvCache(one, [Fake(PLANE[1:]), Fake((1, *PLANE[1:]))])._bases) == [1 << 20] * 2
    for bad in ([Fake((3, 9, 16, 8, 64))] * 4, [Fake(PLANE[1:])] * 4, [Fake((2, 9, 16, 512))] * 4, [Fake((2, 1, 9, 16, 8, 64))] * 4):
        with pytest.raises(ValueError, match="kv codec"):
            PagedKvCache(codec, bad)


def test_native_errors_reach_the_caller(codec):
    # what the binding lets through and the library refuses: an object at half an element
    class Stream:
        device, cuda_stream = torch.device("cuda", 0), 0

    with pytest.raises(GpuAesGcmError, match="kv_quantise.*invalid argument"):
        codec.quantise([Fake(SHAPE, ptr=(1 << 20) + 1)], [Fake((R,), U8)], stream=Stream())
    Stream.device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="stream"):
        codec.quantise([Fake(SHAPE)], [Fake((R,), U8)], stream=Stream())


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_split_finds_codes_and_scales(cpu_lib, fmt):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 3, 5, 2, 37, generator=g).to(torch.float16)
    codec = KvCodec(cpu_lib, fmt, torch.float16, planes=2, layers=3, heads=2, head_dim=37)
    rec = torch.from_numpy(kv_ref.record(x, fmt))
    assert rec.numel() == codec.record_bytes(5)
    for r in (rec, torch.stack([rec, rec])):
        codes, scales = codec.split(r, 5)
        lead = r.shape[:-1]
        if fmt == "mxfp4":
            assert codes.shape == (*lead, 2, 3, 5, 2, 19) and scales.shape == (*lead, 2, 3, 5, 2, 2)
            continue
        assert codes.shape == (*lead, *x.shape) and scales.shape == (*lead, 2, 3, 5, 2)
        assert torch.equal((codes.float() * scales[..., None]).half().expand(*lead, *x.shape),
                           kv_ref.read(rec.numpy(), fmt, torch.float16, x.shape).expand(*lead, *x.shape))


def reached(fake, itemsize=2):
    """The bytes of a tensor's elements, from all of its indices."""
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(fake.shape, fake.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return set((at[:, None] * itemsize + torch.arange(itemsize) + fake.data_ptr()).flatten().tolist())


def write_to(codec, layers):
    codec.dequantise_paged([Fake((R,), U8)], PagedKvCache(codec, layers), [Fake((3,), I64, "cpu")])


def test_caches_with_shared_memory_are_not_written_to(codec):
    """Whichever layer, or pair of planes, shares memory. Slots on the host are refused behind that check: their error
    says that a cache is taken."""
    block = 16 * 8 * 64
    size = 2 * 9 * block * 2

    def joint(k, strides=None):
        return Fake((2, 9, 16, 8, 64), strides=strides, ptr=(1 << 20) + k * size)

    def pair(a, b):
        return tuple(Fake(PLANE[1:], ptr=(1 << 20) + p * (size // 2)) for p in (a, b))

    aliasing = {"a later layer's planes": [joint(0), joint(1, (0, block, 512, 64, 1)), joint(2), joint(3)],
                "planes half a block apart": [joint(0), joint(1), joint(2), joint(3, (block // 2, block, 512, 64, 1))],
                "a pair of one tensor": [pair(0, 1), pair(2, 3), pair(4, 4), pair(6, 7)],
                "pairs of one tensor": [pair(k, k) for k in range(4)],
                "one layer twice": [joint(0), joint(1), joint(2), joint(1)],
                "keys of one layer, values of another": [pair(0, 1), pair(2, 3), pair(4, 0), pair(6, 7)]}
    for name, layers in aliasing.items():
        with pytest.raises(ValueError, match="overlap"):
            write_to(codec, layers)
        # such a cache can be read
        with pytest.raises(ValueError, match="slots"):
            codec.quantise_paged(PagedKvCache(codec, layers), [Fake((3,), I64, "cpu")], [Fake((R,), U8)])
    # all layers of a block side by side, [blocks, layers, planes, ...], or of a row, [blocks, block_size, layers, planes, ...]
    whole = (4 * 2 * block, 512, 64, 1)
    rows = (16 * 4 * 2 * 512, 4 * 2 * 512, 64, 1)
    apart = {"in turn": [joint(k) for k in range(4)], "pairs": [pair(2 * k, 2 * k + 1) for k in range(4)],
             "by block": [Fake(PLANE, strides=(block, *whole), ptr=(1 << 20) + 4 * k * block) for k in range(4)],
             "by row": [Fake(PLANE, strides=(512, *rows), ptr=(1 << 20) + 4 * k * 512) for k in range(4)]}
    for name, layers in apart.items():
        with pytest.raises(ValueError, match="slots"):
            write_to(codec, layers)
    writable = PagedKvCache(codec, apart["in turn"])
    assert writable.writable() is writable
    for name in ("a later layer's planes", "planes half a block apart", "a pair of one tensor"):
        with pytest.raises(ValueError, match="overlap"):
            PagedKvCache(codec, aliasing[name]).writable()


def test_shared_memory_is_what_the_indices_say(cpu_lib):
    """Two layers at every distance, of tensors with and without gaps between vectors, rows and blocks, against the sets of
    their bytes."""
    codec = KvCodec(cpu_lib, "int8", torch.bfloat16, planes=1, layers=2, heads=2, head_dim=3)
    seen = set()
    for strides in ((12, 6, 3, 1), (24, 6, 3, 1), (40, 14, 4, 1), (30, 3, 9, 1), (100, 40, 16, 1)):
        first = Fake((3, 2, 2, 3), strides=strides, ptr=1 << 20)
        mine = reached(first)
        for elements in range(0, 300):
            second = Fake((3, 2, 2, 3), strides=strides, ptr=(1 << 20) + 2 * elements)
            meet = bool(mine & reached(second))
            seen.add(meet)
            for layers in ([first, second], [second, first]):
                with pytest.raises(ValueError, match="overlap" if meet else "slots"):
                    codec.dequantise_paged([Fake((64,), U8)], PagedKvCache(codec, layers), [Fake((1,), I64, "cpu")])
    assert seen == {True, False}


def test_a_cache_keeps_its_tensors(codec):
    """Whatever its caller does with the lists that it was made of."""
    import gc
    import weakref

    layers = [[Fake(PLANE[1:], ptr=(1 << 20) + (2 * k << 20)), Fake(PLANE[1:], ptr=(1 << 20) + (2 * k + 1 << 20))] for k in range(4)]
    held = [weakref.ref(t) for pair in layers for t in pair]
    cache = PagedKvCache(codec, layers)
    for pair in layers:
        pair.clear()
    layers.clear()
    gc.collect()
    assert all(r() is not None for r in held)
    del cache
    gc.collect()
    assert all(r() is None for r in held)
