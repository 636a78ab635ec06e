"""The C-ABI and binding of a paged cache's requests without a GPU: symbols, structures, sizes and refusals, all of which
come before any device access."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from confkv_b200 import kv_codec, kv_paged
from confkv_b200.gpu_aesgcm import GpuAesGcmError
from confkv_b200.kv_codec import KvCodec, KvLayout, KvPages, PagedKvCache
from confkv_b200.kv_paged import ATTENTION, TABLES, VECTORS, KvAttention, KvBlockTables
from test_kv_codec_api import Fake

HEADER = Path(__file__).resolve().parents[1] / "include" / "gpu_kv_paged_api.h"
OK, ERR_ARG = 0, -1
BF16, I32, I64, U8, F32 = torch.bfloat16, torch.int32, torch.int64, torch.uint8, torch.float32


@pytest.fixture
def lib(cpu_lib):
    kv_paged._declare(cpu_lib.lib)
    return cpu_lib.lib


def test_header_and_library_agree(cpu_lib):
    names = set(re.findall(r"^\s*(?:size_t|int)\s+(lmcache_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(kv_paged.PAGED_SYMBOLS)
    for name in names:
        assert hasattr(cpu_lib.lib, name), name


def test_structures_are_the_headers(tmp_path):
    fields = {"tables": (TABLES, ["tables", "table_stride", "held", "lengths", "free", "cursor", "kept", "cursor_after", "slots",
                                  "starts", "capacity", "requests", "width", "blocks", "block_size", "ring", "reserved"]),
              "vectors": (VECTORS, ["keys", "key_stride", "key_head_stride", "values", "value_stride", "value_head_stride",
                                    "slots", "tokens"]),
              "attention": (ATTENTION, ["query", "query_stride", "query_head_stride", "out", "out_stride", "out_head_stride",
                                        "lse", "lse_stride", "tables", "table_stride", "lengths", "workspace",
                                        "workspace_bytes", "requests", "query_heads", "value_dim", "width", "window", "scale"])}
    lines, want = [], []
    for name, (packed, names) in fields.items():
        struct = f"lmcache_gpu_kv_{name}"
        lines.append(f'printf("%zu\\n", sizeof({struct}));')
        want.append(packed.size)
        at = 0
        for field, code in zip(names, re.sub(r"(\d+)(\w)", lambda m: m[2] * int(m[1]), packed.format.lstrip("<"))):
            lines.append(f'printf("%zu\\n", offsetof({struct}, {field}));')
            want.append(at)
            at += 8 if code in "Qq" else 4
        assert at == packed.size
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "gpu_kv_paged_api.h"\nint main(void){' + "\n".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-std=c11", "-I", str(HEADER.parent), str(src), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(n) for n in got] == want


# ------------------------------------------------------------------ resize

P = {name: 0x100000 + 0x100000 * k for k, name in
     enumerate(("tables", "held", "lengths", "free", "cursor", "kept", "cursor_after", "slots", "starts"))}


def tables(**more):
    f = {**P, "table_stride": 64, "capacity": 100, "requests": 8, "width": 64, "blocks": 512, "block_size": 16, "ring": 512, **more}
    return TABLES.pack(f["tables"], f["table_stride"], f["held"], f["lengths"], f["free"], f["cursor"], f["kept"],
                       f["cursor_after"], f["slots"], f["starts"], f["capacity"], f["requests"], f["width"], f["blocks"],
                       f["block_size"], f["ring"], 0)


BAD_TABLES = [
    *({name: 0} for name in ("tables", "held", "lengths", "free", "cursor", "kept", "cursor_after")),
    *({name: P[name] + 2} for name in ("tables", "held", "lengths", "free", "cursor", "kept", "cursor_after")),
    dict(slots=P["slots"] + 4), dict(starts=P["starts"] + 4), dict(slots=0),
    dict(table_stride=63), dict(table_stride=-64), dict(table_stride=1 << 62), dict(requests=1 << 24), dict(block_size=0),
    dict(blocks=1 << 31), dict(blocks=1 << 27), dict(ring=(1 << 31) - 1), dict(ring=1 << 31), dict(width=(1 << 31) - 1),
    dict(capacity=(1 << 31) - 1), dict(capacity=1 << 63),
    # memory shared: outputs with inputs, outputs with one another
    dict(kept=P["held"]), dict(kept=P["lengths"] + 28), dict(cursor_after=P["cursor"]), dict(cursor_after=P["cursor"] + 4),
    dict(kept=P["cursor_after"]), dict(starts=P["slots"] + 8 * 99), dict(free=P["held"]), dict(free=P["tables"]),
    dict(tables=P["free"] + 4), dict(held=P["tables"] + 4 * (7 * 64 + 63)),
]


@pytest.mark.parametrize("bad", BAD_TABLES, ids=str)
def test_bad_tables(lib, bad):
    assert lib.lmcache_gpu_kv_resize_async(tables(**bad), 0, None) == ERR_ARG


def test_bad_devices_and_structures(lib):
    assert lib.lmcache_gpu_kv_resize_async(tables(), -1, None) == ERR_ARG
    assert lib.lmcache_gpu_kv_resize_async(None, 0, None) == ERR_ARG


# ------------------------------------------------------------------ a layer

def layout(dtype=0, planes=2, layers=4, heads=8, head_dim=64):
    return KvLayout(0, dtype, planes, layers, heads, head_dim)


def pages(**more):
    bases = (ctypes.c_void_p * 8)(*more.pop("bases", [0x100000 + 0x10000 * k for k in range(8)]))
    p = KvPages(ctypes.addressof(bases), 64, 16, 0, 16 * 512, 512, 64)
    for k, v in more.items():
        setattr(p, k, v)
    p.keep = bases
    return p


def vectors(**more):
    f = {"keys": 0x800000, "key_stride": 512, "key_head_stride": 64, "values": 0x900000, "value_stride": 512,
         "value_head_stride": 64, "slots": 0xa00000, "tokens": 5, **more}
    return VECTORS.pack(*f.values())


def attention(**more):
    f = {"query": 0x800000, "query_stride": 2048, "query_head_stride": 64, "out": 0x900000, "out_stride": 2048,
         "out_head_stride": 64, "lse": 0xa00000, "lse_stride": 32, "tables": 0xb00000, "table_stride": 64,
         "lengths": 0xc00000, "workspace": 0x10000000, "workspace_bytes": 1 << 40, "requests": 3, "query_heads": 32,
         "value_dim": 64, "width": 64, "window": 0, "scale": 0.125, **more}
    return ATTENTION.pack(*f.values())


BAD_LAYOUTS = [dict(dtype=-1), dict(dtype=3), dict(planes=0), dict(planes=3), dict(layers=0), dict(layers=65536), dict(heads=0),
               dict(heads=65536), dict(head_dim=0), dict(head_dim=65536)]
# layer 1's bases are the second and the sixth
BAD_PAGES = [dict(bases=[1 << 20] * 5 + [0, 1 << 20, 1 << 20]), dict(bases=[1 << 20, (1 << 20) + 1] + [1 << 20] * 6), dict(block_size=0),
             dict(blocks=1 << 31), dict(blocks=1 << 28), dict(block_stride=-1), dict(row_stride=-1), dict(head_stride=-1)]


@pytest.mark.parametrize("bad", BAD_LAYOUTS, ids=str)
def test_bad_layouts(lib, bad):
    b = layout(**bad)
    assert lib.lmcache_gpu_kv_append_async(ctypes.byref(b), ctypes.byref(pages()), 0, vectors(), 0, None) == ERR_ARG
    assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(b), ctypes.byref(pages()), 0, attention(), 0, None) == ERR_ARG
    if bad != dict(layers=0) and bad != dict(layers=65536):
        assert lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(b), 32, 64) == 0


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_bad_pages(lib, bad):
    for f, what in ((lib.lmcache_gpu_kv_append_async, vectors()), (lib.lmcache_gpu_kv_attend_async, attention())):
        assert f(ctypes.byref(layout()), ctypes.byref(pages(**bad)), 1, what, 0, None) == ERR_ARG


def test_bad_layers_and_structures(lib):
    for f, what in ((lib.lmcache_gpu_kv_append_async, vectors()), (lib.lmcache_gpu_kv_attend_async, attention())):
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), 4, what, 0, None) == ERR_ARG
        assert f(None, ctypes.byref(pages()), 0, what, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), None, 0, what, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), 0, None, 0, None) == ERR_ARG
        assert f(ctypes.byref(layout()), ctypes.byref(pages()), 0, what, -1, None) == ERR_ARG
        none = KvPages(None, 64, 16, 0, 0, 0, 0)
        assert f(ctypes.byref(layout()), ctypes.byref(none), 0, what, 0, None) == ERR_ARG


BAD_VECTORS = [dict(keys=0), dict(values=0), dict(slots=0), dict(keys=0x800001), dict(values=0x900001), dict(slots=0xa00004),
               dict(key_stride=-1), dict(key_head_stride=-1), dict(value_stride=-1), dict(value_head_stride=-1), dict(tokens=1 << 31)]


@pytest.mark.parametrize("bad", BAD_VECTORS, ids=str)
def test_bad_vectors(lib, bad):
    assert lib.lmcache_gpu_kv_append_async(ctypes.byref(layout()), ctypes.byref(pages()), 1, vectors(**bad), 0, None) == ERR_ARG


def test_vectors_too_large_for_a_launch(lib):
    b = layout(heads=65535, head_dim=65535)
    assert lib.lmcache_gpu_kv_append_async(ctypes.byref(b), ctypes.byref(pages()), 1, vectors(), 0, None) == ERR_ARG


def test_nothing_to_do(lib):
    none = vectors(keys=0, values=0, slots=0, tokens=0)
    assert lib.lmcache_gpu_kv_append_async(ctypes.byref(layout()), ctypes.byref(pages()), 1, none, 0, None) == OK
    empty = attention(query=0, out=0, lse=0, tables=0, lengths=0, requests=0)
    assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(layout()), ctypes.byref(pages()), 1, empty, 0, None) == OK


BAD_ATTENTION = [
    dict(query=0), dict(out=0), dict(tables=0), dict(lengths=0), dict(workspace=0), dict(query=0x800001), dict(out=0x900001),
    dict(lse=0xa00002), dict(tables=0xb00002), dict(lengths=0xc00002), dict(workspace=0x10000008), dict(workspace_bytes=64),
    dict(query_stride=-1), dict(query_head_stride=-1), dict(out_stride=-1), dict(out_head_stride=-1), dict(lse_stride=-1),
    dict(table_stride=-1), dict(requests=1 << 24), dict(query_heads=0), dict(query_heads=12), dict(query_heads=1 << 17),
    dict(value_dim=0), dict(value_dim=63), dict(value_dim=65), dict(width=(1 << 31) - 1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(scale=3e38), dict(requests=100, width=1 << 27), dict(requests=1 << 23, width=1024),
    # 2^24 requests of 32 heads of 2^31 tokens: more tiles than are counted
    dict(requests=(1 << 24) - 1, query_heads=65528, width=1 << 27),
]


@pytest.mark.parametrize("bad", BAD_ATTENTION, ids=str)
def test_bad_attention(lib, bad):
    assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(layout()), ctypes.byref(pages()), 1, attention(**bad), 0, None) == ERR_ARG


def test_workspace_size_is_what_the_call_takes(lib):
    for dtype in range(3):
        for planes, d, v in ((2, 1, 1), (2, 64, 64), (2, 100, 100), (2, 128, 128), (2, 256, 256), (1, 320, 256), (1, 576, 512), (2, 1024, 1024)):
            for heads, query_heads in ((1, 1), (1, 7), (2, 8), (8, 64), (1, 128)):
                b = layout(dtype, planes, 4, heads, d)
                size = lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(b), query_heads, v)
                assert 0 < size < 1 << 27
                for room in (size - 1, 0):
                    # too small before anything else is looked at
                    what = attention(workspace_bytes=room, query_heads=query_heads, value_dim=v, requests=0)
                    assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(b), ctypes.byref(pages()), 1, what, 0, None) == ERR_ARG
                what = attention(workspace_bytes=size, query_heads=query_heads, value_dim=v, requests=0)
                assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(b), ctypes.byref(pages()), 1, what, 0, None) == OK
    for bad in ((12, 64), (0, 64), (32, 0), (32, 63), (65536, 64)):
        assert lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(layout()), *bad) == 0
    assert lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(layout(head_dim=1025)), 32, 1025) == 0
    assert lib.lmcache_gpu_kv_attend_workspace_size(None, 32, 64) == 0

@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d", range(260, 321, 4))
def test_workspace_size_counts_a_query_less_aligned_than_the_cache(lib, dtype, d):
    """16-bit latent vectors that only the kernel of any type takes with a query at an odd element: 2 blocks on each of 148 SMs, 4 query
    heads in a row. A block has 16 bytes for its cut, and 2 places of 4 heads of 8 bytes and of value_dim floats, in fours."""
    for group in range(2, 9):
        for v in (1, 16, 64, 128, d):
            b = layout(dtype, 1, 4, 1, d)
            need = 296 * (16 + 2 * 4 * (8 + 4 * -(-v // 4) * 4))
            assert lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(b), group, v) >= need


@pytest.mark.parametrize("dtype", range(3))
@pytest.mark.parametrize("planes,d", [(2, 6), (2, 64), (2, 66), (2, 100), (2, 128), (2, 192), (2, 260), (2, 321), (2, 576), (2, 644), (1, 64), (1, 65), (1, 100),
                                      (1, 128), (1, 256), (1, 260), (1, 300), (1, 320), (1, 384), (1, 576), (1, 640), (1, 1024)])
def test_workspace_size_is_enough_for_every_alignment(lib, dtype, planes, d):
    """A call refuses less than its own kernel takes, whatever the size function says."""
    element = 4 if dtype == 2 else 2
    for group in (1, 2, 4, 5, 8, 9, 16, 17, 64):
        b = layout(dtype, planes, 4, 1, d)
        v = d if planes == 2 else max(1, d - 3)
        size = lib.lmcache_gpu_kv_attend_workspace_size(ctypes.byref(b), group, v)
        for at in (element, 2 * element, 4 * element, 8 * element):
            # one block of one token of one head: no stride counts, the addresses alone
            p = pages(bases=[0x100000 + 0x10000 * k + at for k in range(8)], blocks=1, block_size=1)
            for off in (element, 2 * element, 4 * element, 8 * element):
                what = attention(workspace_bytes=size, query=0x800000 + off, query_heads=group, value_dim=v, requests=0)
                assert lib.lmcache_gpu_kv_attend_async(ctypes.byref(b), ctypes.byref(p), 1, what, 0, None) == OK, (group, at, off)


NO_DEVICE = 1 << 20         # what passes all checks gets as far as this device, and no further


@pytest.mark.parametrize("width", [1024, 1025, 5000, 1 << 20])
def test_the_most_requests_for_a_width(lib, width):
    """As many as the header says: requests * (width * block_size / 64 + 4) below 2^31."""
    most = ((1 << 31) - 1) // (width * 16 // 64 + 4)
    for requests, refused in ((most, False), (most + 1, True)):
        what = attention(requests=requests, width=width, table_stride=width)
        rc = lib.lmcache_gpu_kv_attend_async(ctypes.byref(layout()), ctypes.byref(pages()), 1, what, NO_DEVICE, None)
        assert (rc == ERR_ARG) == refused and rc != OK


@pytest.mark.parametrize("name,size", [("held", 32), ("lengths", 32), ("kept", 32), ("cursor", 8), ("cursor_after", 8), ("starts", 72), ("free", 40)])
def test_what_lies_between_the_rows_of_tables(lib, name, size):
    """8 rows of 64 names, 100 apart: other arrays may lie between two of them and behind the last, and nowhere in one."""
    at, row, stride = P["tables"], 4 * 64, 4 * 100
    between = [(k, o) for k in (0, 3, 6) for o in (row, row + (stride - row - size) // 16 * 8, stride - size)] + [(7, row), (7, row + 200), (0, -size)]
    within = [(k, o) for k in (0, 3, 7) for o in (0, 8, row - 8, 8 - size)]
    for refused, places in ((False, between), (True, within)):
        for k, o in places:
            what = tables(**{name: at + k * stride + o, "table_stride": 100, "ring": 10})
            rc = lib.lmcache_gpu_kv_resize_async(what, NO_DEVICE, None)
            assert (rc == ERR_ARG) == refused and rc != OK, (k, o)


# ------------------------------------------------------------------ the binding

def cache(cpu_lib, planes=2, head_dim=64, dtype=BF16, layers=2, overlap=False):
    codec = KvCodec(cpu_lib, "int8", dtype, planes=planes, layers=layers, heads=8, head_dim=head_dim, device=0)
    strides = (0, 16 * 512, 512, 64, 1) if overlap else None
    return PagedKvCache(codec, [Fake((planes, 32, 16, 8, head_dim), dtype, strides=strides, ptr=(1 + k) << 28) for k in range(layers)])


def refused(call, *args, **kwargs):
    with pytest.raises((ValueError, GpuAesGcmError)) as e:
        call(*args, **kwargs)
    assert e.type is ValueError or "rc=-1 " in str(e.value)         # not a call that got as far as the device


def test_block_tables_refuse(cpu_lib):
    for bad in (dict(blocks=-1, block_size=16), dict(blocks=4, block_size=0), dict(blocks=1 << 27, block_size=16),
                dict(blocks=4, block_size=16, device="cpu"), dict(blocks=4, block_size=16, device="cuda")):
        refused(KvBlockTables, cpu_lib, **bad)
    b = KvBlockTables(cpu_lib, blocks=512, block_size=16)
    good = {"tables": Fake((8, 64), I32, ptr=1 << 20), "held": Fake((8,), I32, ptr=2 << 20), "lengths": Fake((8,), I32, ptr=3 << 20),
            "free": Fake((512,), I32, ptr=4 << 20), "cursor": Fake((2,), I32, ptr=5 << 20), "kept": Fake((8,), I32, ptr=6 << 20),
            "cursor_after": Fake((2,), I32, ptr=7 << 20), "slots": Fake((100,), I64, ptr=8 << 20), "starts": Fake((9,), I64, ptr=9 << 20)}
    bad = [("tables", Fake((7, 64), I32)), ("tables", Fake((8, 64), I64)), ("tables", Fake((8, 64), I32, "cuda:1")),
           ("tables", Fake((8,), I32)), ("tables", Fake((8, 64), I32, strides=(128, 2))), ("tables", Fake((8, 64), I32, strides=(32, 1))),
           ("held", Fake((8,), I64)), ("held", Fake((8,), I32, "cpu")), ("lengths", Fake((9,), I32)),
           ("lengths", Fake((8,), I32, strides=(2,))), ("free", Fake((512,), I64)), ("free", Fake((2, 256), I32)),
           ("free", Fake((512,), I32, strides=(2,))), ("cursor", Fake((3,), I32)), ("kept", Fake((8,), I32, strides=(0,))),
           ("kept", good["held"]), ("cursor_after", good["cursor"]), ("cursor_after", Fake((2,), F32)), ("slots", Fake((100,), I32)),
           ("slots", Fake((100,), I64, strides=(2,))), ("slots", None), ("starts", Fake((8,), I64)), ("starts", Fake((9,), I32))]
    for name, value in bad:
        refused(b.resize, **{**good, name: value}, stream=FakeStream())
    refused(b.resize, **good, stream=FakeStream("cuda:1"))


class FakeStream:
    def __init__(self, device="cuda:0"):
        self.device, self.cuda_stream = torch.device(device), 0


def test_attention_refuses_bad_configurations(cpu_lib):
    for bad in (dict(query_heads=0), dict(query_heads=12), dict(query_heads=1 << 16), dict(query_heads=8, value_dim=32),
                dict(query_heads=8, scale=float("nan")), dict(query_heads=8, scale=-3e38), dict(query_heads=8, scale=float("inf")), dict(query_heads=8, window=-1), dict(query_heads=8, window=1 << 32)):
        refused(KvAttention, cpu_lib, cache(cpu_lib), **bad)
    for v in (0, 65):
        refused(KvAttention, cpu_lib, cache(cpu_lib, planes=1), query_heads=8, value_dim=v)
    refused(KvAttention, cpu_lib, cache(cpu_lib, head_dim=1025), query_heads=8)


def test_append_refuses(cpu_lib):
    a = KvAttention(cpu_lib, cache(cpu_lib), query_heads=32)
    k, s = Fake((5, 8, 64)), Fake((5,), I64)
    for layer, slots, keys, values in (
            (2, s, k, k), (-1, s, k, k), (0, Fake((4,), I64), k, k), (0, Fake((5,), I32), k, k), (0, Fake((5,), I64, "cpu"), k, k),
            (0, Fake((5,), I64, strides=(2,)), k, k), (0, s, k, None), (0, s, Fake((5, 8, 32)), k), (0, s, k, Fake((4, 8, 64))),
            (0, s, Fake((5, 8, 64), F32), k), (0, s, k, Fake((5, 8, 64), device="cuda:1")),
            (0, s, k, Fake((5, 8, 64), strides=(1024, 128, 2))), (0, s, Fake((5, 8, 64), strides=(-512, 64, 1)), k)):
        refused(a.append, layer, slots, keys, values, stream=FakeStream())
    refused(a.append, 0, s, k, k, stream=FakeStream("cuda:1"))
    refused(KvAttention(cpu_lib, cache(cpu_lib, planes=1), query_heads=8).append, 0, s, k, k, stream=FakeStream())
    refused(KvAttention(cpu_lib, cache(cpu_lib, overlap=True), query_heads=8).append, 0, s, k, k, stream=FakeStream())


def test_attend_refuses(cpu_lib):
    a = KvAttention(cpu_lib, cache(cpu_lib), query_heads=32)
    good = {"layer": 0, "query": Fake((3, 32, 64)), "tables": Fake((3, 16), I32), "lengths": Fake((3,), I32), "out": Fake((3, 32, 64)),
            "lse": Fake((3, 32), F32), "workspace": Fake((a._workspace,), U8)}
    bad = [("layer", 2), ("layer", -1), ("query", Fake((4, 32, 64))), ("query", Fake((3, 8, 64))), ("query", Fake((3, 32, 64), F32)),
           ("query", Fake((3, 32, 64), strides=(4096, 128, 2))), ("query", Fake((3, 32, 64), device="cuda:1")),
           ("out", Fake((3, 32, 32))), ("out", Fake((3, 32, 64), torch.float16)), ("out", Fake((3, 32, 64), strides=(0, 64, 1))),
           ("out", Fake((3, 32, 64), strides=(64, 64, 1))), ("tables", Fake((2, 16), I32)), ("tables", Fake((3, 16), I64)),
           ("tables", Fake((3, 16), I32, strides=(32, 2))), ("lengths", Fake((3,), I64)), ("lengths", Fake((3,), I32, strides=(2,))),
           ("lse", Fake((3, 32), BF16)), ("lse", Fake((3, 31), F32)), ("lse", Fake((3, 32), F32, strides=(16, 1))),
           ("lse", Fake((3, 32), F32, strides=(64, 2))), ("workspace", Fake((a._workspace - 1,), U8)),
           ("workspace", Fake((a._workspace,), torch.int8)), ("workspace", Fake((a._workspace,), U8, "cuda:1")),
           ("workspace", Fake((a._workspace,), U8, ptr=(1 << 20) + 8)), ("workspace", Fake((a._workspace,), U8, strides=(2,)))]
    for name, value in bad:
        refused(a.attend, **{**good, name: value}, stream=FakeStream())
    refused(a.attend, **good, stream=FakeStream("cuda:1"))
