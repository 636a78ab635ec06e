"""The config runner's decoding over records that were sealed, opened and read back into a paged cache."""

import pytest
import torch

from confkv_b200 import configs, workloads
from confkv_b200.gpu_aesgcm import GpuAes128GcmKey

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "fp8", "mxfp4"])
@pytest.mark.parametrize("shape,count", [((2, 4, 256, 8, 64), 9), ((2, 3, 32, 1, 128), 1), ((1, 2, 64, 1, 320), 6), ((2, 2, 48, 2, 40), 4)], ids=str)
def test_decode(gpu_lib, fmt, shape, count):
    objects = workloads.bf16_batch(shape, count, seed=3, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with GpuAes128GcmKey(gpu_lib, workloads.make_key(1)) as key:
        work = configs.QuantisedWork(gpu_lib, key, objects, fmt, stream, workloads.make_ivs(2, count))
        work.seal_batched()
        work.open_batched()
        d = configs.DecodeWork(gpu_lib, work, 20)
        torch.cuda.synchronize()
        got = d.run()
        torch.cuda.synchronize()
        assert work.round_trip_ok()
        assert got["decode_ok"] and got["decode_steps"] == 20 and got["requests"] == min(4, count)
        # what came out wrong does not pass
        good = d.out.clone()
        d.out[-1, -1, 0] += d.out.abs().max()
        assert not d.check()
        d.out.copy_(good.roll(1, -1))
        assert not d.check()
        d.out.copy_(good)
        assert d.check()
        del d, work


def test_the_command(gpu_lib):
    import json
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-m", "confkv_b200.configs", "--config", "kv_small", "--kv-format", "int8", "--decode", "5", "--api",
                        "batched", "--warmup", "1", "--iters", "2"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [json.loads(x) for x in r.stdout.splitlines()]
    assert lines[0]["round_trip_ok"] and lines[1]["decode_ok"] and lines[1]["decode_ms_per_step"] > 0


def test_decode_behind_a_busy_stream(gpu_lib):
    """The constructors' fills still wait behind other work of the current stream when the work's own stream starts."""
    objects = workloads.bf16_batch((2, 2, 48, 2, 40), 8, seed=4, device="cuda")
    stream = torch.cuda.Stream()
    with GpuAes128GcmKey(gpu_lib, workloads.make_key(1)) as key:
        torch.cuda.synchronize()
        torch.cuda._sleep(200_000_000)          # a tenth of a second
        work = configs.QuantisedWork(gpu_lib, key, objects, "int8", stream, workloads.make_ivs(2, 8))
        work.seal_batched()
        work.open_batched()
        torch.cuda._sleep(200_000_000)
        got = configs.DecodeWork(gpu_lib, work, 6).run()
        torch.cuda.synchronize()
        assert got["decode_ok"] and work.round_trip_ok()
        del work
