"""Index arithmetic of the paged cache's operators, compiled for the host and checked against Python's whole numbers."""

import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
MOST = (1 << 31) - 1


@pytest.fixture(scope="module")
def native(tmp_path_factory):
    so = tmp_path_factory.mktemp("paged") / "kv_paged_check.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", str(ROOT / "confkv_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "kv_paged_check.cpp"), "-o", str(so)], check=True)
    return ctypes.CDLL(str(so))


def pointer(a):
    return a.ctypes.data_as(ctypes.c_void_p)


def i32(values):
    return np.array(values, dtype=np.int64).astype(np.int32)


@pytest.mark.parametrize("block_size", [1, 2, 3, 5, 16, 48, 64, 1000, MOST])
@pytest.mark.parametrize("width", [0, 1, 7, 512, 1 << 27, MOST - 1])
def test_changes(native, block_size, width):
    limit = min(width * block_size, MOST)
    rng = random.Random(block_size * 7 + width)
    near = {0, 1, 2, 15, 16, 17, block_size - 1, block_size, block_size + 1, limit - 1, limit, limit + 1, limit // 2, -1, MOST, -MOST - 1}
    near |= {rng.randrange(0, limit + 1) for _ in range(20)}
    near = sorted(x for x in near if -MOST - 1 <= x <= MOST)
    pairs = [(h, x) for h in near for x in near]
    held, length = i32([h for h, _ in pairs]), i32([x for _, x in pairs])
    out = np.zeros((len(pairs), 5), dtype=np.uint32)
    native.changes(pointer(held), pointer(length), len(pairs), ctypes.c_uint32(width), ctypes.c_uint32(block_size), pointer(out))
    for (h, x), got in zip(pairs, out.tolist()):
        if not 0 <= h <= limit:
            assert got == [0] * 5, (h, x)
            continue
        before = -(-h // block_size)
        if not 0 <= x <= limit:
            assert got == [h, before, 0, 0, 0], (h, x)
            continue
        after = -(-x // block_size)
        assert got == [x, before, max(after - before, 0), max(before - after, 0), max(x - h, 0)], (h, x)


@pytest.mark.parametrize("ring", [0, 1, 2, 7, 1000, MOST - 1])
def test_cursors(native, ring):
    values = [-MOST - 1, -8, -7, -1, 0, 1, 6, 7, 8, 999, 1000, MOST - 2, MOST - 1, MOST]
    pairs = [(a, b) for a in values for b in values]
    first, count = i32([a for a, _ in pairs]), i32([b for _, b in pairs])
    out = np.zeros((len(pairs), 2), dtype=np.uint32)
    native.cursors(pointer(first), pointer(count), len(pairs), ctypes.c_uint32(ring), pointer(out))
    for (a, b), got in zip(pairs, out.tolist()):
        assert got == ([a % ring, min(max(b, 0), ring)] if ring else [0, 0]), (a, b)


@pytest.mark.parametrize("limit", [0, 1, 63, 64, 65, 100000, MOST])
@pytest.mark.parametrize("window", [0, 1, 64, 1000, MOST, (1 << 32) - 1])
@pytest.mark.parametrize("tile", [16, 64])
def test_spans(native, limit, window, tile):
    lengths = sorted({x for x in (-MOST - 1, -1, 0, 1, 63, 64, 65, 999, 1000, 1001, limit - 1, limit, limit + 1, MOST) if x <= MOST})
    out = np.zeros((len(lengths), 3), dtype=np.uint32)
    a = i32(lengths)
    native.spans(pointer(a), len(lengths), ctypes.c_uint32(limit), ctypes.c_uint32(window), ctypes.c_uint32(tile), pointer(out))
    for x, got in zip(lengths, out.tolist()):
        end = max(0, min(x, limit))
        first = max(0, end - window) if window else 0
        assert got == [first, end, max(1, -(-(end - first) // tile))], x


def test_parts(native):
    native.check_parts.argtypes = [ctypes.c_uint64, ctypes.c_uint32]
    rng = random.Random(1)
    totals = set(range(1, 200)) | {rng.randrange(1, 5000) for _ in range(200)}
    totals |= {(1 << 52) - 1 - k for k in range(3)} | {1 << k for k in range(52)} | {rng.randrange(1, 1 << 51) for _ in range(200)}
    for total in totals:
        for workers in (1, 2, 147, 148, 296, 592, 2047):
            assert native.check_parts(total, min(workers, total)) == 0, (total, workers)


def test_rows(native):
    rng = random.Random(2)
    rows = [[1], [2], [3], [1000], [1] * 7, [1] * 2000, [40000, 1, 1, 1, 70000], [5] * 300]
    rows += [[max(1, int(2 ** rng.uniform(0, top))) for _ in range(rng.randrange(1, 400))] for top in (2, 5, 8, 11) for _ in range(12)]
    for tiles in rows:
        a = np.array(tiles, dtype=np.uint32)
        for workers in (1, 2, 7, 148, 296, 592):
            for whole, least in ((1, 0), (2, 1), (4, 1), (8, 2), (16, 0)):
                got = native.check_rows(pointer(a), len(tiles), *map(ctypes.c_uint32, (workers, whole, least)))
                assert got == 0, (tiles, workers, whole, least)
