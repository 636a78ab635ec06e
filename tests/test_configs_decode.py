"""The config runner's verdict on attention, and its arguments."""

import subprocess
import sys

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
