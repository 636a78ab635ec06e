"""The config runner's verdict on attention, and its arguments."""

import contextlib
import datetime
import multiprocessing
import socket
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


def _decoding_rank(rank, world, port, q):
    import os

    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    try:
        def result(ms, ok):
            return {"requests": 4, "restore_ms": ms, "decode_ms_per_step": 10 - ms, "decode_ok": ok}

        q.put((rank, [configs.decoded_by_all(result(1.0 + rank, True), None), configs.decoded_by_all(result(1.0 + rank, rank == 0), None),
                      configs.decoded_by_all(result(2.0, True) if rank == 0 else None, None)]))
    finally:
        dist.destroy_process_group()


def test_the_verdict_on_decoding_is_that_of_all_ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = multiprocessing.get_context("spawn")
    q = ctx.Queue()
    ranks = [ctx.Process(target=_decoding_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in ranks:
        p.start()
    got = dict(q.get(timeout=120) for _ in ranks)
    for p in ranks:
        p.join(timeout=60)
        assert p.exitcode == 0
    right = {"requests": 4, "restore_ms": 2.0, "decode_ms_per_step": 9.0, "decode_ok": True}
    for rank in range(2):
        assert got[rank][:2] == [right, {**right, "decode_ok": False}]
    assert got[0][2] == {**right, "decode_ms_per_step": 8.0} and got[1][2] is None


def test_the_verdict_on_decoding_of_one_process():
    result = {"requests": 4, "restore_ms": 1.5, "decode_ms_per_step": 2.5, "decode_ok": False}
    assert configs.decoded_by_all(result, None) == result
    assert configs.decoded_by_all(None, None) is None
