"""The config runner's verdict on attention, and its arguments."""

import contextlib
import subprocess
import sys
import types

import pytest
import torch

from confkv_b200 import configs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_right_results_pass_and_wrong_ones_do_not(dtype):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g).to(dtype) for s in ((8, 64), (50, 2, 64), (50, 2, 64)))
    scale = 64 ** -0.5
    kk, vv = (x.double().repeat_interleave(4, 1) for x in (k, v))
    p = torch.softmax(scale * torch.einsum("hd,thd->ht", q.double(), kk), -1)
    out = torch.einsum("ht,thd->hd", p, vv).to(dtype)
    assert configs.attended_within(out, q, k, v, scale)
    assert not configs.attended_within(torch.zeros_like(out), q, k, v, scale)
    assert not configs.attended_within(out.roll(1, 0), q, k, v, scale)
    assert not configs.attended_within(out, q, k, v, scale * 1.1)
    assert not configs.attended_within(out, q, k[:-1], v[:-1], scale)
    out[3, 5] = float("nan")
    assert not configs.attended_within(out, q, k, v, scale)


@pytest.mark.parametrize("more", [["--decode", "3"], ["--decode", "-1", "--kv-format", "int8"]])
def test_arguments(more):
    r = subprocess.run([sys.executable, "-m", "confkv_b200.configs", "--config", "kv_small", *more], capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "--decode" in r.stderr


class Order:
    """A stream that notes what waits for it or uses it, in turn."""

    device = torch.device("cuda", 0)

    def __init__(self):
        self.notes = []

    def wait_stream(self, other):
        self.notes.append(("wait", other))


class Stop(Exception):
    pass


def test_decoding_waits_for_the_stream_that_filled_its_tensors(monkeypatch):
    stream = Order()
    d = object.__new__(configs.DecodeWork)
    d.work = types.SimpleNamespace(stream=stream)

    def restore():
        stream.notes.append("restore")
        raise Stop

    d.restore = restore
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: f"current of {device}")
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    with pytest.raises(Stop):
        d.run()
    assert stream.notes == [("wait", "current of cuda:0"), "restore"]


def test_sealing_waits_for_the_stream_that_filled_its_buffers(monkeypatch):
    stream = Order()

    class Batch:
        def __init__(self, lib, count, device):
            self.workspace_bytes = 0

        def seal(self, key, entries, stream):
            stream.notes.append("seal")

        def open(self, key, entries, stream):
            stream.notes.append("open")

    monkeypatch.setattr(configs, "DeviceBatch", Batch)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: f"current of {device}")
    plain = torch.zeros(64, dtype=torch.uint8)
    configs.RankWork(None, None, [5, 20], plain, [0, 16], stream, [b"0" * 12] * 2)
    assert stream.notes == [("wait", "current of cpu"), "seal", "open"]
