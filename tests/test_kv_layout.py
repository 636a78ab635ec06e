"""The KV codec's index arithmetic, record layout and quotients (csrc/kv_layout.h, csrc/kv_math.h, which the
kernels compile too) on the CPU, and the reference records' own consistency."""

import ctypes
import math
import subprocess
from pathlib import Path

import kv_ref
import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("kv") / "libkv_check.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-mfma", "-fPIC", "-shared", "-Wall", "-Wextra", "-I",
                    str(ROOT / "confkv_b200" / "csrc"), str(ROOT / "tests" / "native" / "kv_check.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    u32, u64, i32 = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int
    lib.kv_check_fast_div.argtypes = [u32, ctypes.c_void_p, ctypes.c_size_t]
    lib.kv_check_fast_div.restype = ctypes.c_int64
    lib.kv_check_vectors.argtypes = [u32] * 5
    lib.kv_check_vectors.restype = u64
    lib.kv_check_record_size.argtypes = [i32, u32, u64]
    lib.kv_check_record_size.restype = u64
    lib.kv_check_quotients.argtypes = [i32] * 5
    lib.kv_check_quotients.restype = u64
    lib.kv_check_int8.argtypes = [i32, i32, i32, ctypes.POINTER(u64)]
    lib.kv_check_int8.restype = u64
    lib.kv_check_mx_byte.argtypes = [u32]
    lib.kv_check_mx_byte.restype = u32
    lib.kv_check_mx_inverse.argtypes = [u32]
    lib.kv_check_mx_inverse.restype = ctypes.c_float
    lib.kv_check_scales.argtypes = [i32, i32]
    lib.kv_check_scales.restype = u64
    lib.kv_check_scale.argtypes = [i32, ctypes.c_float]
    lib.kv_check_scale.restype = ctypes.c_float
    return lib


def test_fast_division(lib):
    rng = np.random.default_rng(1)
    divisors = [*range(1, 600), 1023, 1024, 1025, 65535, 65536, 65537, (1 << 30) - 1, 1 << 30, (1 << 31) - 1,
                *rng.integers(1, 1 << 31, 200)]
    for d in divisors:
        d = int(d)
        near = np.array([k * d + o for k in (0, 1, 2, 7, (1 << 31) // d - 1, (1 << 31) // d) for o in (-1, 0, 1)])
        n = np.concatenate([near[(near >= 0) & (near < 1 << 31)], rng.integers(0, 1 << 31, 500), [0, (1 << 31) - 1]])
        n = np.ascontiguousarray(n.astype(np.uint32))
        assert lib.kv_check_fast_div(d, n.ctypes.data, len(n)) == -1, d


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 2, 5, 7, 3), (2, 1, 80, 33, 1), (5, 2, 32, 1, 8), (1, 2, 3, 256, 8)])
def test_vectors_in_the_objects_order(lib, shape):
    assert lib.kv_check_vectors(*shape) == 0


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
def test_record_size(lib, fmt):
    for d in (1, 2, 15, 16, 31, 32, 33, 64, 100, 128, 576, 65535):
        for n in (0, 1, 3, 512, 131072, (1 << 31) - 1):
            assert lib.kv_check_record_size(kv_ref.FORMATS.index(fmt), d, n) == kv_ref.record_bytes(fmt, d, n)[1]


# int8 codes end at gap 8 (127 / 2^8 < 1/2), e4m3's at 18 (448 / 2^18 < 2^-9 / 2)
@pytest.mark.parametrize("fmt,gap", [(0, 9), (1, 20)])
def test_every_bfloat16_quotient_is_on_its_side_of_the_borders(lib, fmt, gap):
    for exponent in (-7, 100, -120):
        assert lib.kv_check_quotients(fmt, 8, gap, 1, exponent) == 0


@pytest.mark.parametrize("fmt,gap", [(0, 9), (1, 20)])
def test_every_half_quotient_is_on_its_side_of_the_borders(lib, fmt, gap):
    assert lib.kv_check_quotients(fmt, 11, gap, 1, -10) == 0


@pytest.mark.parametrize("fmt,gap", [(0, 9), (1, 20)])
def test_float32_quotients_are_on_their_sides_of_the_borders(lib, fmt, gap):
    assert lib.kv_check_quotients(fmt, 24, gap, 15000, -23) == 0


@pytest.mark.parametrize("bits,exponent", [(8, -7), (8, 120), (8, -126), (11, -10), (11, 5), (11, -24)])
def test_every_int8_code_by_one_product(lib, bits, exponent):
    """Of every bfloat16 and half vector that does not take the divider: of half those whose A is a multiple of 127."""
    slow = ctypes.c_uint64()
    assert lib.kv_check_int8(bits, 9, exponent, ctypes.byref(slow)) == 0
    assert slow.value == (0 if bits == 8 else 8)


def test_int8_vectors_too_small_for_one_product(lib):
    slow = ctypes.c_uint64()
    assert lib.kv_check_int8(8, 9, -127, ctypes.byref(slow)) == 0 and slow.value == 128


def test_microscale_bytes(lib):
    rng = np.random.default_rng(2)
    bits = np.concatenate([rng.integers(0, 0x7f800000, 4000), np.arange(0, 300) << 23 & 0x7f000000, [0, 1, 0x7f7fffff]])
    for b in bits:
        a = float(np.array(b, dtype=np.uint32).view(np.float32))
        e = max(math.floor(math.log2(a)) - 2 if a > 0 else -127, -127)
        if a > 0:                                   # log2 of a value next to a power of two may be rounded onto it
            e = max(math.frexp(a)[1] - 3, -127)
        byte = lib.kv_check_mx_byte(int(b))
        assert byte == e + 127
        assert lib.kv_check_mx_inverse(byte) == 2.0 ** -e
    for b in (0x7f800000, 0x7f800001, 0x7fffffff):
        assert lib.kv_check_mx_byte(b) == 255


@pytest.mark.parametrize("fmt,top", [(0, 127), (1, 448)])
def test_scales(lib, fmt, top):
    for a in (0.0, 1e-45, 1e-38, 0.1, 1.0, 65504.0, 3e38, float(kv_ref.FLT_MAX)):
        s = lib.kv_check_scale(fmt, a)
        want = min(np.float32(a) / np.float32(top), kv_ref.MOST_SCALE[top])
        assert np.float32(s) == want
        assert np.isfinite(np.float32(s) * np.float32(top))


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("exponent", [0, -100, -101, 120])
def test_every_scale_is_the_rounded_quotient(lib, fmt, exponent):
    assert lib.kv_check_scales(fmt, exponent) == 0


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", kv_ref.DTYPES)
def test_reference_errors_are_within_half_a_step(fmt, dtype):
    """The reference reads back every value to half a step of its code: A / 254 (int8), 2^-4 of the value or half of
    e4m3's least step (fp8), 2^-2 of the value, half of e2m1's least step or what saturates (mxfp4: A < 8 2^e against 6 2^e)."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(2, 3, 5, 4, 100, generator=g) * torch.exp(2 * torch.randn(100, generator=g))).to(dtype)
    y = kv_ref.read(kv_ref.record(x, fmt), fmt, dtype, x.shape).double()
    x = x.double()
    rounding = torch.finfo(dtype).eps / 2 * x.abs() * 1.01 + 2.0 ** -22 * x.abs() + 1e-7   # to the type; of the scale and the product
    err = (x - y).abs() - rounding
    if fmt == "mxfp4":
        pad = torch.nn.functional.pad(x, (0, 28)).view(2, 3, 5, 4, 4, 32)
        e = torch.floor(torch.log2(pad.abs().amax(-1, keepdim=True))) - 2
        unit = (2.0 ** e).expand_as(pad).flatten(-2)[..., :100]
        bound = torch.maximum(torch.maximum(x.abs() / 4, unit / 4), torch.where(x.abs() > 6 * unit, 2 * unit, 0 * unit))
    else:
        a = x.abs().amax(-1, keepdim=True)
        bound = a / 254 if fmt == "int8" else torch.maximum(x.abs() / 16, a / 448 * 2.0 ** -10)
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("wide", [0, 1])
@pytest.mark.parametrize("exponent", [-140, -133, -7, 0, 100, 119])
def test_quotients_of_zero_keep_their_sign(lib, fmt, wide, exponent):
    lib.kv_check_signs.argtypes = [ctypes.c_int] * 3
    lib.kv_check_signs.restype = ctypes.c_uint64
    assert lib.kv_check_signs(fmt, exponent, wide) == 0
