"""The serde backend with `kv_format`: what is sealed is the object's record (kv_codec) in the place of its bytes.

Frames open on the CPU to exactly the record that the plain reference (kv_ref) makes of the object, in both
directions; what the GPU reads back is the reference's, bit for bit; rejected and foreign frames leave zeros."""

import ctypes
import sys
from pathlib import Path

import kv_ref
import numpy as np
import pytest
import torch
from cryptography.hazmat.primitives.ciphers.aead import AESGCM

FAKE = Path(__file__).resolve().parent / "fake_lmcache"
if str(FAKE) not in sys.path:
    sys.path.insert(0, str(FAKE))

from lmcache.v1.distributed.api import MemoryLayoutDesc  # noqa: E402

import confkv_b200.serde as gpu_serde  # noqa: E402
from test_serde import KEY, OTHER_TENANT, Buf, DevObj, key_path, processor, run_de, run_de_many, run_ser, run_ser_many  # noqa: E402,F401

FORMATS = kv_ref.FORMATS
IV = bytes(range(12))


def kv(shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * 3).to(dtype)


def row(t, d=None):
    """An object as the serde sees it: one row of vectors."""
    d = d or t.shape[-1]
    return t.reshape(1, 1, -1, 1, d)


def as_read(t, fmt, d=None):
    """What the object reads back as."""
    r = row(t, d)
    return kv_ref.read(kv_ref.record(r, fmt), fmt, t.dtype, r.shape).view(t.shape)


def dek(proc, key):
    return proc._ctx.keys.get_key(key.cache_salt)


def same(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


# ------------------------------------------------------------ CPU

@pytest.mark.parametrize("fmt", FORMATS)
def test_estimate_is_the_records_size(fmt):
    ctx = gpu_serde.GpuSerdeContext(key_provider=None, kv_format=fmt)
    ser = gpu_serde.GpuAesGcmSerializer(ctx)
    layout = MemoryLayoutDesc([torch.Size((2, 4, 256, 8, 64))], [torch.bfloat16])
    assert ser.estimate_serialized_size(layout) == kv_ref.record_bytes(fmt, 64, 2 * 4 * 256 * 8)[1] + 29
    # heads merged into the last dimension
    ctx = gpu_serde.GpuSerdeContext(key_provider=None, kv_format=fmt, kv_head_dim=64)
    merged = MemoryLayoutDesc([torch.Size((2, 4, 256, 512))], [torch.float16])
    assert gpu_serde.GpuAesGcmSerializer(ctx).estimate_serialized_size(merged) == \
        kv_ref.record_bytes(fmt, 64, 2 * 4 * 256 * 8)[1] + 29


def test_refused_configurations_and_objects(tmp_path):
    key = tmp_path / "k"
    key.write_bytes(b"k" * 32)
    for bad in ({"kv_format": "int4"}, {"kv_format": "int8", "kv_head_dim": 0}, {"kv_format": "int8", "kv_head_dim": 65536}):
        with pytest.raises(ValueError):
            gpu_serde.create_gpu_aesgcm_serde({"master_key_path": str(key), **bad})
    gpu_serde.create_gpu_aesgcm_serde({"master_key_path": str(key), "kv_format": ""}).close()     # off
    ctx = gpu_serde.GpuSerdeContext(key_provider=None, kv_format="int8", kv_head_dim=64)
    ser = gpu_serde.GpuAesGcmSerializer(ctx)
    for shape, dtype in (((4, 64), torch.uint8), ((4, 96), torch.bfloat16), ((4, 32), torch.bfloat16), ((3, 64), torch.float64)):
        with pytest.raises(ValueError):
            ser.estimate_serialized_size(MemoryLayoutDesc([torch.Size(shape)], [dtype]))
    with pytest.raises(ValueError):
        ser.estimate_serialized_size(MemoryLayoutDesc([torch.Size((4, 64))] * 2, [torch.bfloat16] * 2))
    for obj in (Buf(128), DevObj(torch.zeros(4, 128, dtype=torch.bfloat16)[:, :64])):
        with pytest.raises(ValueError):
            ser.serialize(obj, Buf(4096), KEY)
        with pytest.raises(ValueError):
            gpu_serde.GpuAesGcmDeserializer(ctx).deserialize(Buf(4096), obj, KEY)
    with pytest.raises(ValueError):
        ser.serialize(DevObj(torch.zeros(4, 64, dtype=torch.bfloat16)), Buf(16), KEY)        # destination too small


def test_a_short_frames_object_is_zeroed():
    """A frame that cannot hold the object's record is refused before any device access, and a host object is zeroed."""
    de = gpu_serde.GpuAesGcmDeserializer(gpu_serde.GpuSerdeContext(key_provider=None, kv_format="int8"))
    out = torch.full((4, 64), 5.0, dtype=torch.bfloat16)
    size = kv_ref.record_bytes("int8", 64, 4)[1] + 29
    for n in (0, 28, size - 1):
        out.fill_(5)
        with pytest.raises(ValueError, match="malformed"):
            de.deserialize(Buf(n), DevObj(out), KEY)
        assert not out.any()


# ------------------------------------------------------------ GPU

@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 4, 256, 8, 64), (2, 3, 7, 1, 40), (1, 5, 33)], ids=str)
def test_frames_hold_the_reference_records(key_path, fmt, dtype, shape):
    x = kv(shape, dtype)
    want = kv_ref.record(row(x), fmt)
    proc = processor("gpu", key_path, kv_format=fmt)
    try:
        size = proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [dtype]))
        assert size == len(want) + 29
        for src in (DevObj(x.cuda()), DevObj(x)):                 # in HBM and on the host
            frame = Buf(size)
            assert run_ser(proc, src, frame) is True
            raw = frame.bytes()
            assert raw[0] == 1
            plain = AESGCM(dek(proc, KEY)).decrypt(raw[1:13], raw[13:], None)
            assert kv_ref.same_record(np.frombuffer(plain, np.uint8), want, fmt, shape[-1], x.numel() // shape[-1])
            for out in (torch.full(shape, 5.0, dtype=dtype, device="cuda"), torch.full(shape, 5.0, dtype=dtype)):
                assert run_de(proc, frame, DevObj(out)) is True
                assert same(out, as_read(x, fmt))
        # a frame sealed on the CPU from the reference's record
        sealed = b"\x01" + IV + AESGCM(dek(proc, KEY)).encrypt(IV, want.tobytes(), None)
        dframe = torch.frombuffer(bytearray(sealed), dtype=torch.uint8).cuda()
        out = torch.full(shape, 5.0, dtype=dtype, device="cuda")
        assert run_de(proc, DevObj(dframe), DevObj(out)) is True
        assert same(out, as_read(x, fmt))
    finally:
        proc.close()


@pytest.mark.gpu
def test_merged_heads(key_path):
    x = kv((2, 4, 19, 8 * 64))
    proc = processor("gpu", key_path, kv_format="int8", kv_head_dim=64)
    try:
        frame, out = Buf(kv_ref.record_bytes("int8", 64, x.numel() // 64)[1] + 29), torch.zeros_like(x, device="cuda")
        assert run_ser(proc, DevObj(x.cuda()), frame) is True
        assert run_de(proc, frame, DevObj(out)) is True
        assert same(out, as_read(x, "int8", 64))
    finally:
        proc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["ciphertext", "tag", "iv", "version", "tenant"])
@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_rejected_frames_leave_zeros(key_path, case, where):
    x = kv((2, 4, 64, 8, 64))
    proc = processor("gpu", key_path, kv_format="mxfp4")
    try:
        frame = Buf(proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype])))
        assert run_ser(proc, DevObj(x.cuda()), frame) is True
        at = {"ciphertext": 13 + 1000, "tag": len(frame.bytes()) - 1, "iv": 3, "version": 0, "tenant": None}[case]
        if at is not None:
            memoryview(frame._arr).cast("B")[at] ^= 2
        out = torch.full(x.shape, 5.0, dtype=x.dtype, device=where)
        assert run_de(proc, frame, DevObj(out), OTHER_TENANT if case == "tenant" else KEY) is False
        assert not out.any()
        with pytest.raises(gpu_serde.InvalidTag):
            proc.deserializer.deserialize(frame, DevObj(out), OTHER_TENANT if case == "tenant" else KEY)
    finally:
        proc.close()


@pytest.mark.gpu
def test_another_formats_frames_are_refused(key_path):
    """An authentic frame of the same length that holds another format's record, or another head size's."""
    x = kv((2, 4, 64, 8, 64))
    one, other = (processor("gpu", key_path, kv_format=f) for f in ("int8", "fp8"))
    try:
        frame = Buf(one.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype])))
        assert run_ser(one, DevObj(x.cuda()), frame) is True
        out = torch.full(x.shape, 5.0, dtype=x.dtype, device="cuda")
        assert run_de(other, frame, DevObj(out)) is False
        assert not out.any()
        with pytest.raises(ValueError, match="fp8 record"):
            other.deserializer.deserialize(frame, DevObj(out), KEY)
        out = torch.full(x.shape, 5.0, dtype=torch.float16, device="cuda")
        assert run_de(one, frame, DevObj(out)) is False and not out.any()
        # too short for a record of that object
        assert run_de(one, frame, DevObj(torch.zeros(4, 4, 64, 8, 64, dtype=x.dtype, device="cuda"))) is False
    finally:
        one.close()
        other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_batches_of_two_tenants_types_and_sizes(key_path, fmt):
    """A multi-object submit: one quantise call a codec, one batched seal a key; then one tampered frame, which
    zeroes its object and no other."""
    shapes = [(2, 4, 256, 8, 64), (2, 4, 13, 8, 64), (2, 2, 5, 33), (1, 64), (3, 2, 9, 2, 128), (2, 4, 100, 8, 64)]
    dtypes = [torch.bfloat16, torch.float16, torch.bfloat16, torch.bfloat16, torch.float16, torch.bfloat16]
    keys = [KEY if i % 2 == 0 else OTHER_TENANT for i in range(len(shapes))]
    xs = [kv(s, t, seed=i) for i, (s, t) in enumerate(zip(shapes, dtypes))]
    proc = processor("gpu", key_path, kv_format=fmt)
    try:
        frames = [Buf(proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype]))) for x in xs]
        srcs = [DevObj(x.cuda() if i % 3 else x) for i, x in enumerate(xs)]
        assert run_ser_many(proc, srcs, frames, keys) is True
        for x, f, k in zip(xs, frames, keys):
            raw = f.bytes()
            plain = np.frombuffer(AESGCM(dek(proc, k)).decrypt(raw[1:13], raw[13:], None), np.uint8)
            assert kv_ref.same_record(plain, kv_ref.record(row(x), fmt), fmt, x.shape[-1], x.numel() // x.shape[-1])

        def outs():
            return [torch.full(x.shape, 5.0, dtype=x.dtype, device="cuda" if i % 2 else "cpu") for i, x in enumerate(xs)]

        got = outs()
        assert run_de_many(proc, frames, [DevObj(o) for o in got], keys) is True
        for x, o in zip(xs, got):
            assert same(o, as_read(x, fmt))
        memoryview(frames[2]._arr).cast("B")[13 + 40] ^= 1
        got = outs()
        assert run_de_many(proc, frames, [DevObj(o) for o in got], keys) is False
        for i, (x, o) in enumerate(zip(xs, got)):
            assert not o.any() if i == 2 else same(o, as_read(x, fmt))
    finally:
        proc.close()


@pytest.mark.gpu
def test_workers_share_a_processor(key_path):
    xs = [kv((2, 4, 50 + k, 8, 64), seed=k) for k in range(8)]
    proc = processor("gpu", key_path, kv_format="fp8", max_workers=4)
    try:
        device = [x.cuda() for x in xs]
        torch.cuda.synchronize()
        frames = [Buf(proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype]))) for x in xs]
        tasks = [proc.submit_serialize([DevObj(d)], [f], [KEY]) for d, f in zip(device, frames)]
        from test_serde import wait

        assert all(wait(proc.query_serialize_result, t) for t in tasks)
        outs = [torch.zeros_like(d) for d in device]
        torch.cuda.synchronize()
        tasks = [proc.submit_deserialize([f], [DevObj(o)], [KEY]) for f, o in zip(frames, outs)]
        assert all(wait(proc.query_deserialize_result, t) for t in tasks)
        for x, o in zip(xs, outs):
            assert same(o, as_read(x, "fp8"))
    finally:
        proc.close()


@pytest.mark.gpu
def test_without_a_format_frames_hold_the_objects_bytes(key_path):
    x = kv((2, 4, 64, 8, 64))
    proc = processor("gpu", key_path)
    try:
        P = x.numel() * 2
        frame = Buf(P + 29)
        assert run_ser(proc, DevObj(x.cuda()), frame) is True
        raw = frame.bytes()
        assert AESGCM(dek(proc, KEY)).decrypt(raw[1:13], raw[13:], None) == x.view(torch.uint8).numpy().tobytes()
        assert ctypes.sizeof(frame._arr) == P + 29
    finally:
        proc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_an_object_that_is_not_opened_reads_as_zeros(key_path, where, monkeypatch):
    """A descriptor that the device rejects leaves its record's buffer as it was: here an earlier record of the same
    layout, another tenant's. None of it may reach the object."""
    from confkv_b200.batch import DeviceBatch

    xs = [kv((2, 4, 32, 8, 64), seed=k) for k in range(3)]
    stale = torch.from_numpy(kv_ref.record(row(kv((2, 4, 32, 8, 64), seed=9)), "int8")).cuda()
    proc = processor("gpu", key_path, kv_format="int8")
    try:
        frames = [Buf(stale.numel() + 29) for _ in xs]
        assert run_ser_many(proc, [DevObj(x.cuda()) for x in xs], frames, [KEY] * 3) is True
        outs = [torch.full(x.shape, 5.0, dtype=x.dtype, device=where) for x in xs]
        empty, open_ = torch.empty, DeviceBatch.open

        def recycled(*size, **more):
            t = empty(*size, **more)
            return t.copy_(stale) if t.is_cuda and t.dtype == torch.uint8 and t.numel() == stale.numel() else t

        def one_rejected(self, key, entries, stream=None):
            f, d, p, n, a = entries[1]
            return open_(self, key, [entries[0], (f, d, p, n - 1, a), entries[2]], stream)

        torch.cuda.synchronize()
        monkeypatch.setattr(torch, "empty", recycled)
        monkeypatch.setattr(DeviceBatch, "open", one_rejected)
        with pytest.raises(ValueError, match="descriptor"):
            proc._open_many(frames, [DevObj(o) for o in outs], [KEY] * 3)
        monkeypatch.undo()
        assert not outs[1].any()
        for k in (0, 2):
            assert same(outs[k], as_read(xs[k], "int8"))
    finally:
        proc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_frames_of_other_lengths_leave_zeros(key_path, where):
    """Another format's frame, shorter or longer than the reader's, and a frame of whole bytes: refused, one or several at
    once, and the objects are zeros afterwards."""
    x = kv((2, 4, 64, 8, 64))
    names = ("int8", "mxfp4", None)
    procs = {f: processor("gpu", key_path, **({} if f is None else {"kv_format": f})) for f in names}
    try:
        frames = {}
        for f in names:
            frames[f] = Buf(procs[f].estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype])))
            assert run_ser(procs[f], DevObj(x.cuda()), frames[f]) is True
        cut = Buf(len(frames["int8"].bytes()) - 1)
        ctypes.memmove(cut.address, frames["int8"].address, len(cut.bytes()))
        for reader, frame, error in (("int8", frames["mxfp4"], ValueError), ("int8", cut, ValueError), ("int8", Buf(3), ValueError),
                                     ("mxfp4", frames["int8"], gpu_serde.InvalidTag),
                                     ("int8", frames[None], gpu_serde.InvalidTag), ("mxfp4", frames[None], gpu_serde.InvalidTag)):
            def out():
                return torch.full(x.shape, 5.0, dtype=x.dtype, device=where)

            o = out()
            assert run_de(procs[reader], frame, DevObj(o)) is False and not o.any()
            o = out()
            with pytest.raises(error):
                procs[reader].deserializer.deserialize(frame, DevObj(o), KEY)
            assert not o.any()
            # among frames that are its own, of the same and of another tenant: the whole task fails, and none of its
            # objects keeps what it held before
            o = [out() for _ in range(3)]
            assert run_de_many(procs[reader], [frames[reader], frame, frames[reader]], [DevObj(t) for t in o],
                               [KEY, KEY, OTHER_TENANT]) is False
            assert not o[1].any()
            if error is not ValueError:
                assert same(o[0], as_read(x, reader)) and not o[2].any()
    finally:
        for p in procs.values():
            p.close()


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_objects_on_another_device(key_path):
    """Objects of another GPU than the backend's are copied to it and back, one or several at once."""
    xs = [kv((2, 4, 33, 8, 64), seed=k) for k in range(3)]
    proc = processor("gpu", key_path, kv_format="int8", device=0)
    try:
        frames = [Buf(proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype]))) for x in xs]
        srcs = [DevObj(x.to("cuda:1")) for x in xs]
        torch.cuda.synchronize(1)
        assert run_ser_many(proc, srcs, frames, [KEY] * 3) is True and run_ser(proc, srcs[0], frames[0]) is True
        outs = [torch.full(x.shape, 5.0, dtype=x.dtype, device="cuda:1") for x in xs]
        torch.cuda.synchronize(1)
        assert run_de_many(proc, frames, [DevObj(o) for o in outs], [KEY] * 3) is True
        for x, o in zip(xs, outs):
            assert same(o, as_read(x, "int8"))
        outs[0].fill_(5)
        torch.cuda.synchronize(1)
        assert run_de(proc, frames[0], DevObj(outs[0])) is True and same(outs[0], as_read(xs[0], "int8"))
    finally:
        proc.close()


@pytest.mark.gpu
def test_objects_on_the_backends_device_are_read_back_in_place(key_path, monkeypatch):
    """And those on the host through a copy."""
    x = kv((2, 4, 33, 8, 64))
    proc = processor("gpu", key_path, kv_format="int8")
    seen = []
    try:
        frame = Buf(proc.estimate_serialized_size(MemoryLayoutDesc([x.shape], [x.dtype])))
        assert run_ser(proc, DevObj(x.cuda()), frame) is True
        from confkv_b200.kv_codec import KvCodec

        call = KvCodec.dequantise
        monkeypatch.setattr(KvCodec, "dequantise", lambda self, records, objects, **more: (
            seen.extend(o.data_ptr() for o in objects), call(self, records, objects, **more))[1])
        for where in ("cuda", "cpu"):
            out = torch.full(x.shape, 5.0, dtype=x.dtype, device=where)
            assert run_de(proc, frame, DevObj(out)) is True and same(out, as_read(x, "int8"))
            assert (seen.pop() == out.data_ptr()) == (where == "cuda") and not seen
    finally:
        proc.close()
