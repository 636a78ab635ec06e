"""The KV codec's records in plain numpy, 64 bits up to the rounding to a code: quotients of whole numbers
below 2^31 by ones below 2^24 are at least 2^-32 of their size away from a border unless they are on it, and
float64 division is right to 2^-53, so these codes are the definition's."""

import numpy as np
import torch

FORMATS = ("int8", "fp8", "mxfp4")
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
HEADER = 32
BLOCK = 32
FLT_MAX = np.float32(3.4028234663852886e38)
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
# FLT_MAX / 127 and / 448, rounded down to float32
MOST_SCALE = {127: np.float32(float.fromhex("0x1.020406p+121")), 448: np.float32(float.fromhex("0x1.249248p+119"))}


def code_bytes(fmt, d):
    return (d + 1) // 2 if fmt == "mxfp4" else d


def record_bytes(fmt, d, vectors):
    at = HEADER + -(-vectors * code_bytes(fmt, d) // 16) * 16
    scales = vectors * (-(-d // BLOCK) if fmt == "mxfp4" else 4)
    return at, at + -(-scales // 16) * 16


def _minifloat(y, mantissa, lowest, top):
    step = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 1, lowest) - mantissa)
    return np.clip(np.round(y / step) * step, -top, top)


def quantise(x, fmt):
    """Codes and scales of x [vectors, d] (float64 of the cache's values), as bytes."""
    d = x.shape[-1]
    if fmt == "mxfp4":
        blocks = -(-d // BLOCK)
        b = np.zeros((len(x), blocks * BLOCK))
        b[:, :d] = x
        b = b.reshape(len(x), blocks, BLOCK)
        with np.errstate(invalid="ignore"):
            amax = np.abs(b).max(-1)
        bad = ~np.isfinite(amax)
        b = np.where(bad[..., None], 0.0, b)
        amax = np.where(bad, 0.0, amax)
        e = np.where(amax > 0, np.maximum(np.frexp(amax)[1] - 1 - 2, -127), -127)
        v = _minifloat(np.ldexp(b, -e[..., None]), 1, 0, 6.0).reshape(len(x), -1)[:, :d]
        code = np.abs(v)[..., None] == E2M1[:8]
        code = (code.argmax(-1) | (np.signbit(v) * 8)).astype(np.uint8)
        code = np.pad(code, ((0, 0), (0, d % 2)))
        return code[:, 0::2] | (code[:, 1::2] << 4), np.where(bad, 255, e + 127).astype(np.uint8)
    top = 127 if fmt == "int8" else 448
    amax = np.abs(x).max(-1)                       # NaN where one is
    bad = ~np.isfinite(amax)
    x = np.where(bad[:, None], 0.0, x)
    amax = np.where(bad, 0.0, amax)
    scale = np.minimum(amax.astype(np.float32) / np.float32(top), MOST_SCALE[top])
    scale = np.where(bad, np.float32(np.nan), scale).astype(np.float32)
    q = x * top / np.where(amax > 0, amax, 1.0)[:, None]
    if fmt == "int8":
        code = np.round(q).astype(np.int8).view(np.uint8)
    else:
        v = torch.from_numpy(_minifloat(q, 3, -6, 448.0).astype(np.float32))
        code = v.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return code, scale


def header(fmt, dtype, planes, layers, tokens, heads, d):
    words = [int.from_bytes(b"KVQ1", "little"), tokens, layers | heads << 16,
             d | FORMATS.index(fmt) << 16 | DTYPES.index(dtype) << 20 | planes << 24, 0, 0, 0, 0]
    return np.array(words, dtype=np.uint32).view(np.uint8)


def record(x, fmt):
    """The record of a [planes, layers, tokens, heads, d] tensor, as uint8."""
    planes, layers, tokens, heads, d = x.shape
    n = planes * layers * tokens * heads
    at, size = record_bytes(fmt, d, n)
    out = np.zeros(size, dtype=np.uint8)
    out[:HEADER] = header(fmt, x.dtype, planes, layers, tokens, heads, d)
    if n:
        codes, scales = quantise(x.detach().cpu().double().numpy().reshape(n, d), fmt)
        out[HEADER:HEADER + codes.size] = codes.reshape(-1)
        scales = np.ascontiguousarray(scales).reshape(-1).view(np.uint8)
        out[at:at + scales.size] = scales
    return out


def read(rec, fmt, dtype, shape):
    """The tensor that a record's bytes stand for: one product in float32, then one rounding to the type."""
    planes, layers, tokens, heads, d = shape
    n = planes * layers * tokens * heads
    if n == 0:
        return torch.empty(shape, dtype=dtype)
    at, _ = record_bytes(fmt, d, n)
    codes = rec[HEADER:HEADER + n * code_bytes(fmt, d)].reshape(n, -1)
    if fmt == "mxfp4":
        nibbles = np.stack((codes & 15, codes >> 4), -1).reshape(n, -1)[:, :d]
        blocks = -(-d // BLOCK)
        e = rec[at:at + n * blocks].reshape(n, blocks).astype(np.int64)
        s = np.where(e == 255, np.nan, np.ldexp(1.0, e - 127))
        v = E2M1[nibbles] * np.repeat(s, BLOCK, -1)[:, :d]
        f = v.astype(np.float32)
    else:
        s = rec[at:at + 4 * n].view(np.float32)
        if fmt == "int8":
            c = codes.view(np.int8).astype(np.float32)
        else:
            c = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).float().numpy()
        with np.errstate(invalid="ignore"):
            f = c * s[:, None]
    return torch.from_numpy(np.ascontiguousarray(f.astype(np.float32))).to(dtype).view(shape)


def same_record(got, want, fmt, d, vectors):
    """Equal bytes, but for the sign of an fp8 code of zero, which a test of its own compares."""
    got, want = np.array(got), np.array(want)
    if fmt == "fp8":
        for r in (got, want):
            codes = r[HEADER:HEADER + vectors * d]
            codes[codes == 0x80] = 0
        at, _ = record_bytes(fmt, d, vectors)
        for r in (got, want):                      # any NaN for any other
            s = r[at:at + 4 * vectors].view(np.float32)
            s[np.isnan(s)] = np.nan
    elif fmt == "int8":
        at, _ = record_bytes(fmt, d, vectors)
        for r in (got, want):
            s = r[at:at + 4 * vectors].view(np.float32)
            s[np.isnan(s)] = np.nan
    return np.array_equal(got, want)
