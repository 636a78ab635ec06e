"""The config runner's verdict on records: what was read back lies as close to the source objects as the format allows."""

import kv_ref
import pytest
import torch

from confkv_b200 import configs

SHAPE = (2, 3, 7, 2, 80)


def objects(dtype, n=2):
    g = torch.Generator().manual_seed(4)
    return (torch.randn(n, *SHAPE, generator=g) * torch.exp(2 * torch.randn(n, *SHAPE[:-1], 1, generator=g))).to(dtype)


def read_back(x, fmt):
    return torch.stack([kv_ref.read(kv_ref.record(o, fmt), fmt, x.dtype, o.shape) for o in x])


def work(x, restored, ok=None):
    """A QuantisedWork without a device, whose codec reads the same values out of the records each time."""
    w = object.__new__(configs.QuantisedWork)
    w.lens, w.records = [], None
    w.objects, w.restored = x, restored
    w.ok = torch.ones(len(x), dtype=torch.int32) if ok is None else ok

    class Codec:
        format = None

        def dequantise(self, records, out):
            out.copy_(restored)

    w.codec = Codec()
    return w


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", kv_ref.DTYPES)
def test_right_values_pass_and_wrong_ones_do_not(fmt, dtype):
    x = objects(dtype)
    y = read_back(x, fmt)

    def verdict(restored, ok=None):
        w = work(x, restored, ok)
        w.codec.format = fmt
        return w.round_trip_ok()

    assert verdict(y)
    assert not verdict(y, torch.tensor([1, 0], dtype=torch.int32))
    assert not verdict(torch.zeros_like(y))
    assert not verdict(y.roll(1, -2))                               # another head's vector
    assert not verdict((y.float() * 2).to(dtype))                   # a scale one power of two off
    assert not verdict(-y)
    assert not verdict(y.flip(0))                                   # the other object
    for at in ((0, 0, 0, 0, 0, 0), (1, 1, 2, 6, 1, 79)):            # one value, by two steps of the largest code
        z = y.clone()
        z[at] += 2 * x[at[:-1]].abs().max().double() / {"int8": 127, "fp8": 14, "mxfp4": 3}[fmt]
        assert not verdict(z)
    z = y.clone()
    z[1, 0, 1, 3, 0, 7] = float("nan")
    assert not verdict(z)


@pytest.mark.parametrize("fmt", kv_ref.FORMATS)
@pytest.mark.parametrize("dtype", kv_ref.DTYPES)
def test_values_at_the_ends_of_the_type(fmt, dtype):
    """The largest, the least, zeros, and vectors that are not finite and read back as NaN."""
    x = objects(dtype, 1)
    f = torch.finfo(dtype)
    v = x.view(-1, SHAPE[-1])
    v[0], v[1], v[2] = f.max, f.smallest_normal * f.eps, 0
    v[3] = torch.linspace(-1, 1, SHAPE[-1]).to(dtype) * f.smallest_normal
    v[4, 3], v[5, 70] = float("inf"), float("nan")
    y = read_back(x, fmt)
    w = work(x, y)
    w.codec.format = fmt
    assert w.round_trip_ok()
    y[torch.isnan(y)] = 0                                           # what is lost has to show
    assert not w.round_trip_ok()
