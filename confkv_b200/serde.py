"""LMCache serde backend on the B200 AES-128-GCM engine.

Drop-in counterpart of ConfKV's CPU serde plugins
(experiments/gpu_kv_seal/integration/native_aesgcm_serde.py:104-298): the same
Serializer / Deserializer interface, the same HKDF key lookup per object
(info prefix b"lmcache-l2-aesgcm-v1", key = provider.get_key(key.cache_salt)),
a fresh os.urandom IV per frame, the same frame [1 | IV | C | T] and P + 29
size estimate, InvalidTag on authentication failure with the destination
zeroed. What changes is where the work runs:

    GPU plaintext KV (MemoryObj.tensor on cuda)
      -> seal on the GPU -> device frame -> (if the destination is host memory)
         D2H copy on the same stream -> storage

and the reverse for deserialize (host frame -> H2D -> authenticated open ->
plaintext written to the device tensor only after the tag verified).

Objects are duck-typed like LMCache's MemoryObj: `.tensor` (a contiguous
torch tensor on a CUDA device or on the host) if present, else `.byte_array`
(a host buffer). Registered as serde type "gpu_aesgcm"; ConfKV's
LMCACHE_AESGCM_BACKEND switch selects it with the value "gpu".

With `kv_format` ("int8", "fp8" or "mxfp4") what is sealed is the object's
record (kv_codec: codes and scales, a half to a quarter of a 16-bit cache) in
the place of its bytes: quantise -> seal, and open -> dequantise. Objects then
need a `.tensor` of bfloat16, float16 or float32 whose vectors are its last
dimension, or `kv_head_dim` values where that dimension holds several heads.
"""

from __future__ import annotations

import itertools
import os
import threading
from collections import defaultdict
from concurrent.futures import ThreadPoolExecutor

from cryptography.exceptions import InvalidTag
from lmcache.v1.distributed.serde.async_processor import AsyncSerdeProcessor
from lmcache.v1.distributed.serde.base import Deserializer, Serializer
from lmcache.v1.distributed.serde.factory import register_serde_factory
from lmcache.v1.distributed.serde.key_provider import HkdfKeyProvider

from .gpu_aesgcm import FRAME_OVERHEAD, GpuAes128GcmKey, GpuAesGcmLibrary
from .kv_codec import DTYPES, FORMATS, HEADER_BYTES, KvCodec, record_size

HKDF_INFO_PREFIX = b"lmcache-l2-aesgcm-v1"
SERDE_TYPE = "gpu_aesgcm"


def _bytes_view(obj):
    """uint8 torch view of a MemoryObj-like object (no copy)."""
    import torch

    t = getattr(obj, "tensor", None)
    if t is not None:
        if not t.is_contiguous():
            raise ValueError("gpu aesgcm: tensor must be contiguous")
        return t.reshape(-1).view(torch.uint8)
    mv = memoryview(obj.byte_array).cast("B")
    if len(mv) == 0:
        return torch.empty(0, dtype=torch.uint8)
    return torch.frombuffer(mv, dtype=torch.uint8)


def _plaintext_bytes(layout_desc) -> int:
    import torch

    total = 0
    for shape, dtype in zip(layout_desc.shapes, layout_desc.dtypes, strict=True):
        n = 1
        for d in shape:
            n *= int(d)
        total += n * torch.empty((), dtype=dtype).element_size()
    return total


class GpuSerdeContext:
    """State shared by a serializer/deserializer pair: the device, one key
    handle per data-encryption key, and one CUDA stream per worker thread."""

    def __init__(self, key_provider, device: int | None = None, library: GpuAesGcmLibrary | None = None,
                 kv_format: str | None = None, kv_head_dim: int | None = None):
        if kv_format is not None and kv_format not in FORMATS:
            raise ValueError(f"gpu aesgcm: kv_format must be one of {', '.join(FORMATS)}")
        if kv_head_dim is not None and not 1 <= kv_head_dim <= 65535:
            raise ValueError("gpu aesgcm: kv_head_dim must be 1 to 65535")
        self.keys = key_provider
        self.kv_format = kv_format
        self._kv_head_dim = kv_head_dim
        self._codecs: dict[tuple, KvCodec] = {}
        self._device = device
        self._library = library
        self._handles: dict[bytes, GpuAes128GcmKey] = {}
        self._lock = threading.Lock()
        self._local = threading.local()

    @property
    def device(self) -> int:
        if self._device is None:
            import torch

            self._device = torch.cuda.current_device()
        return self._device

    def handle(self, dek: bytes) -> GpuAes128GcmKey:
        if len(dek) != 16:
            raise ValueError("gpu aesgcm supports AES-128 only")
        with self._lock:
            h = self._handles.get(dek)
            if h is None:
                if self._library is None:
                    self._library = GpuAesGcmLibrary()
                h = GpuAes128GcmKey(self._library, dek, device=self.device)
                self._handles[dek] = h
            return h

    def stream(self):
        import torch

        s = getattr(self._local, "stream", None)
        if s is None:
            s = torch.cuda.Stream(device=self.device)
            self._local.stream = s
        return s

    def batch(self, count: int):
        """This thread's DeviceBatch with room for `count` objects (grown by
        doubling; the descriptor array and workspace are reused)."""
        from .batch import DeviceBatch

        b = getattr(self._local, "batch", None)
        if b is None or b.capacity < count:
            cap = max(count, 2 * b.capacity if b is not None else 64)
            if self._library is None:
                self._library = GpuAesGcmLibrary()
            b = DeviceBatch(self._library, cap, self.device)
            self._local.batch = b
        return b

    def close(self) -> None:
        with self._lock:
            for h in self._handles.values():
                h.close()
            self._handles.clear()

    # ---- records in the place of the objects' bytes (kv_format)
    def vectors(self, shape, dtype) -> tuple[int, int]:
        """(vectors, head_dim) of an object of this shape and type."""
        if dtype not in DTYPES:
            raise ValueError("gpu aesgcm: kv_format needs bfloat16, float16 or float32 objects")
        numel = 1
        for n in shape:
            numel *= int(n)
        d = self._kv_head_dim or (int(shape[-1]) if len(shape) else 0)
        if d < 1 or d > 65535 or numel % d or len(shape) and int(shape[-1]) % d:
            raise ValueError(f"gpu aesgcm: an object of shape {tuple(shape)} is not made of vectors of {d} values")
        return numel // d, d

    def plaintext_bytes(self, obj) -> int:
        """Bytes that are sealed for an object: its own, or its record's."""
        if self.kv_format is None:
            return _bytes_view(obj).numel()
        t = _kv_tensor(obj)
        vectors, d = self.vectors(t.shape, t.dtype)
        return record_size(self.kv_format, d, vectors)

    def codec(self, t) -> tuple[KvCodec, tuple]:
        """The codec for an object's tensor, and the shape in which it sees it: one row of vectors."""
        vectors, d = self.vectors(t.shape, t.dtype)
        with self._lock:
            c = self._codecs.get((t.dtype, d))
            if c is None:
                if self._library is None:
                    self._library = GpuAesGcmLibrary()
                c = KvCodec(self._library, self.kv_format, t.dtype, planes=1, layers=1, heads=1, head_dim=d,
                            device=self.device)
                self._codecs[(t.dtype, d)] = c
        return c, (1, 1, vectors, 1, d)

    def quantise(self, objs, stream) -> list:
        """Device records of objects, written on `stream` (the current one), with one call a codec."""
        import torch

        dev = torch.device("cuda", self.device)
        records, calls = [], defaultdict(lambda: ([], []))
        for obj in objs:
            t = _kv_tensor(obj)
            codec, shape = self.codec(t)
            record = torch.empty(codec.record_bytes(shape[2]), dtype=torch.uint8, device=dev)
            sources, into = calls[codec]
            sources.append(t.to(dev, non_blocking=True).view(shape))
            into.append(record)
            records.append(record)
        for codec, (sources, into) in calls.items():
            codec.quantise(sources, into, stream=stream)
        return records

    def zero(self, objs) -> None:
        """Zero objects whose frames are too short for their records, and wait for it."""
        import torch

        for t in map(_kv_tensor, objs):
            t.zero_()
            if t.is_cuda:
                torch.cuda.current_stream(t.device).synchronize()

    def forget(self, records) -> None:
        """Clear the headers of record buffers on the current stream, before frames are opened into them: memory that a
        rejected descriptor leaves unwritten may hold an earlier record, which must not pass for this object's."""
        import torch

        torch._foreach_zero_([r[:HEADER_BYTES] for r in records])

    def dequantise(self, records, objs, stream):
        """Read device records back into objects on `stream` (the current one); the verdicts as a device tensor."""
        import torch

        dev = torch.device("cuda", self.device)
        ok = torch.zeros(len(objs), dtype=torch.int32, device=dev)
        calls, copies = defaultdict(lambda: ([], [], [])), []
        for k, (record, obj) in enumerate(zip(records, objs)):
            t = _kv_tensor(obj)
            codec, shape = self.codec(t)
            out = t if t.device == dev else torch.empty(t.shape, dtype=t.dtype, device=dev)
            if out is not t:                    # on the host, or on another device
                copies.append((t, out))
            sources, into, oks = calls[codec]
            sources.append(record)
            into.append(out.view(shape))
            oks.append(ok[k:k + 1])
        for codec, (sources, into, oks) in calls.items():
            codec.dequantise(sources, into, ok=oks, stream=stream)
        for t, out in copies:
            t.copy_(out, non_blocking=True)
        return ok


def _kv_tensor(obj):
    t = getattr(obj, "tensor", None)
    if t is None:
        raise ValueError("gpu aesgcm: kv_format needs objects with a tensor")
    if not t.is_contiguous():
        raise ValueError("gpu aesgcm: tensor must be contiguous")
    return t


class GpuAesGcmSerializer(Serializer):
    def __init__(self, ctx: GpuSerdeContext):
        self._ctx = ctx

    def serialize(self, src, dst, key) -> int:
        import torch

        ctx = self._ctx
        dst_t = _bytes_view(dst)
        plaintext_len = ctx.plaintext_bytes(src)
        frame_len = plaintext_len + FRAME_OVERHEAD
        if dst_t.numel() < frame_len:
            raise ValueError("gpu aesgcm: destination too small")
        gkey = ctx.handle(ctx.keys.get_key(key.cache_salt))
        iv = os.urandom(12)
        stream = ctx.stream()
        dev = torch.device("cuda", ctx.device)
        with torch.cuda.stream(stream):
            if ctx.kv_format is not None:
                src_d, = ctx.quantise([src], stream)
            else:
                src_d = _device_view(_bytes_view(src), dev, plaintext_len)
            frame_d = dst_t if dst_t.is_cuda else torch.empty(frame_len, dtype=torch.uint8, device=dev)
            gkey.seal_async(src_ptr=src_d.data_ptr(), plaintext_len=plaintext_len, dst_ptr=frame_d.data_ptr(),
                            dst_capacity=frame_d.numel(), iv=iv, stream_ptr=stream.cuda_stream)
            if not dst_t.is_cuda:
                dst_t[:frame_len].copy_(frame_d[:frame_len], non_blocking=True)
        stream.synchronize()
        return frame_len

    def estimate_serialized_size(self, layout_desc) -> int:
        ctx = self._ctx
        if ctx.kv_format is not None:
            if len(layout_desc.shapes) != 1 or len(layout_desc.dtypes) != 1:
                raise ValueError("gpu aesgcm: kv_format takes objects of one tensor")
            vectors, d = ctx.vectors(layout_desc.shapes[0], layout_desc.dtypes[0])
            return record_size(ctx.kv_format, d, vectors) + FRAME_OVERHEAD
        return _plaintext_bytes(layout_desc) + FRAME_OVERHEAD


class GpuAesGcmDeserializer(Deserializer):
    def __init__(self, ctx: GpuSerdeContext):
        self._ctx = ctx

    def deserialize(self, src, dst, key) -> None:
        import torch

        ctx = self._ctx
        src_t, dst_t = _bytes_view(src), _bytes_view(dst)
        plaintext_len = ctx.plaintext_bytes(dst)
        frame_len = plaintext_len + FRAME_OVERHEAD
        if src_t.numel() < frame_len:
            if ctx.kv_format is not None:
                ctx.zero([dst])
            raise ValueError("gpu aesgcm: malformed frame")
        direct = ctx.kv_format is None and dst_t.is_cuda and plaintext_len
        gkey = ctx.handle(ctx.keys.get_key(key.cache_salt))
        stream = ctx.stream()
        dev = torch.device("cuda", ctx.device)
        with torch.cuda.stream(stream):
            frame_d = src_t if src_t.is_cuda else src_t[:frame_len].to(dev, non_blocking=True)
            out_d = dst_t if direct else torch.empty(max(plaintext_len, 1), dtype=torch.uint8, device=dev)
            auth = torch.zeros(1, dtype=torch.int32, device=dev)
            if ctx.kv_format is not None:
                ctx.forget([out_d])
            gkey.open_async(src_ptr=frame_d.data_ptr(), frame_len=frame_len, dst_ptr=out_d.data_ptr(),
                            plaintext_len=plaintext_len, auth_ok_ptr=auth.data_ptr(), stream_ptr=stream.cuda_stream)
            if ctx.kv_format is not None:
                # a rejected frame leaves a zeroed record, which reads back as zeros
                ok_h = ctx.dequantise([out_d], [dst], stream).to("cpu", non_blocking=True)
            elif plaintext_len and not dst_t.is_cuda:
                dst_t.copy_(out_d[:plaintext_len], non_blocking=True)
            auth_h = auth.to("cpu", non_blocking=True)
        stream.synchronize()
        if int(auth_h.item()) != 1:
            # the kernels zero-filled the plaintext destination
            raise InvalidTag("gpu aesgcm authentication failed")
        if ctx.kv_format is not None and int(ok_h.item()) != 1:
            raise ValueError(f"gpu aesgcm: the frame does not hold a {ctx.kv_format} record of this object")


def _device_view(t, dev, n: int):
    """`t` itself when it is on the device, else a device copy of its first n
    bytes (a 1-byte placeholder when n == 0)."""
    import torch

    if n == 0:
        return torch.empty(1, dtype=torch.uint8, device=dev)
    return t if t.is_cuda else t[:n].to(dev, non_blocking=True)


class GpuAesGcmSerdeProcessor(AsyncSerdeProcessor):
    """AsyncSerdeProcessor whose multi-object submits run as one batched
    seal / open call per data-encryption key (lmcache_gpu_aes128gcm_*_batch_async)
    instead of one call per object; single-object submits take the
    per-object path. A batched deserialize reports False when any object
    fails authentication; every failed object's destination is zeroed and the
    authentic ones are written. Also releases the GPU key handles on close."""

    def __init__(self, ctx: GpuSerdeContext, max_workers: int = 1):
        super().__init__(GpuAesGcmSerializer(ctx), GpuAesGcmDeserializer(ctx), max_workers=max_workers)
        self._ctx = ctx
        self._bpool = ThreadPoolExecutor(max_workers=max(1, int(max_workers)))
        self._bids = itertools.count(1 << 40)   # disjoint from the base class's task ids
        self._btasks = {}
        self._block = threading.Lock()

    # ---- batched tasks
    def _bsubmit(self, fn, srcs, dsts, keys):
        tid = next(self._bids)
        with self._block:
            self._btasks[tid] = self._bpool.submit(fn, list(srcs), list(dsts), list(keys))
        return tid

    def _bquery(self, tid):
        with self._block:
            fut = self._btasks.get(tid)
        if fut is None or not fut.done():
            return None
        with self._block:
            self._btasks.pop(tid, None)
        return fut.exception() is None

    def _groups(self, keys):
        groups = defaultdict(list)
        for i, k in enumerate(keys):
            groups[self._ctx.keys.get_key(k.cache_salt)].append(i)
        return groups

    def _seal_many(self, srcs, dsts, keys):
        import torch

        ctx = self._ctx
        dev = torch.device("cuda", ctx.device)
        stream = ctx.stream()
        for dek, idx in self._groups(keys).items():
            handle = ctx.handle(dek)
            keep, copies, entries = [], [], []
            with torch.cuda.stream(stream):
                sizes = [ctx.plaintext_bytes(srcs[i]) for i in idx]
                if any(_bytes_view(dsts[i]).numel() < P + FRAME_OVERHEAD for i, P in zip(idx, sizes)):
                    raise ValueError("gpu aesgcm: destination too small")
                records = ctx.quantise([srcs[i] for i in idx], stream) if ctx.kv_format is not None else None
                for j, (i, P) in enumerate(zip(idx, sizes)):
                    dst_t = _bytes_view(dsts[i])
                    F = P + FRAME_OVERHEAD
                    src_d = records[j] if records is not None else _device_view(_bytes_view(srcs[i]), dev, P)
                    frame_d = dst_t if dst_t.is_cuda else torch.empty(F, dtype=torch.uint8, device=dev)
                    entries.append((src_d.data_ptr(), frame_d.data_ptr(), P, frame_d.numel(), os.urandom(12)))
                    keep += [src_d, frame_d]
                    if not dst_t.is_cuda:
                        copies.append((dst_t, frame_d, F))
                batch = ctx.batch(len(entries))
                batch.seal(handle, entries, stream)
                for dst_t, frame_d, F in copies:
                    dst_t[:F].copy_(frame_d[:F], non_blocking=True)
                status = batch.statuses().to("cpu", non_blocking=True)
            stream.synchronize()
            if bool(status.any()):
                raise ValueError("gpu aesgcm: an object descriptor was rejected")
        return True

    def _open_many(self, srcs, dsts, keys):
        import torch

        ctx = self._ctx
        dev = torch.device("cuda", ctx.device)
        stream = ctx.stream()
        failed = foreign = False
        if ctx.kv_format is not None:
            short = [d for s, d in zip(srcs, dsts) if _bytes_view(s).numel() < ctx.plaintext_bytes(d) + FRAME_OVERHEAD]
            if short:
                # another format's frames, say; nothing is opened
                ctx.zero(short)
                raise ValueError("gpu aesgcm: malformed frame")
        for dek, idx in self._groups(keys).items():
            handle = ctx.handle(dek)
            keep, copies, entries, records = [], [], [], []
            with torch.cuda.stream(stream):
                auth = torch.zeros(len(idx), dtype=torch.int32, device=dev)
                for j, i in enumerate(idx):
                    src_t, dst_t = _bytes_view(srcs[i]), _bytes_view(dsts[i])
                    P = ctx.plaintext_bytes(dsts[i])
                    F = P + FRAME_OVERHEAD
                    if src_t.numel() < F:
                        raise ValueError("gpu aesgcm: malformed frame")
                    frame_d = _device_view(src_t, dev, F)
                    direct = ctx.kv_format is None and dst_t.is_cuda and P
                    out_d = dst_t if direct else torch.empty(max(P, 1), dtype=torch.uint8, device=dev)
                    records.append(out_d)
                    entries.append((frame_d.data_ptr(), out_d.data_ptr(), P, F, auth.data_ptr() + 4 * j))
                    keep += [frame_d, out_d]
                    if ctx.kv_format is None and P and not dst_t.is_cuda:
                        copies.append((dst_t, out_d, P))
                if ctx.kv_format is not None:
                    ctx.forget(records)
                batch = ctx.batch(len(entries))
                batch.open(handle, entries, stream)
                ok_h = None
                if ctx.kv_format is not None:
                    ok_h = ctx.dequantise(records, [dsts[i] for i in idx], stream).to("cpu", non_blocking=True)
                for dst_t, out_d, P in copies:
                    dst_t.copy_(out_d[:P], non_blocking=True)
                auth_h = auth.to("cpu", non_blocking=True)
                status = batch.statuses().to("cpu", non_blocking=True)
            stream.synchronize()
            if bool(status.any()):
                raise ValueError("gpu aesgcm: an object descriptor was rejected")
            failed = failed or bool((auth_h != 1).any())
            foreign = foreign or ok_h is not None and bool((ok_h != 1).any())
        if failed:
            # the kernels zero-filled every rejected object's plaintext
            raise InvalidTag("gpu aesgcm authentication failed")
        if foreign:
            raise ValueError(f"gpu aesgcm: a frame does not hold a {ctx.kv_format} record of its object")
        return True

    # ---- SerdeProcessor interface
    def submit_serialize(self, srcs, dsts, keys):
        if len(srcs) < 2:
            return super().submit_serialize(srcs, dsts, keys)
        return self._bsubmit(self._seal_many, srcs, dsts, keys)

    def submit_deserialize(self, srcs, dsts, keys):
        if len(srcs) < 2:
            return super().submit_deserialize(srcs, dsts, keys)
        return self._bsubmit(self._open_many, srcs, dsts, keys)

    def query_serialize_result(self, tid):
        if tid in self._btasks:
            return self._bquery(tid)
        return super().query_serialize_result(tid)

    def query_deserialize_result(self, tid):
        if tid in self._btasks:
            return self._bquery(tid)
        return super().query_deserialize_result(tid)

    def close(self):
        self._bpool.shutdown(wait=True)
        super().close()
        self._ctx.close()


def create_gpu_aesgcm_serde(kwargs: dict) -> GpuAesGcmSerdeProcessor:
    """Factory with the kwargs of native_aesgcm_serde.py:236-292 plus
    `device` (CUDA ordinal; default the current device), `kv_format` (seal
    int8, fp8 or mxfp4 records; default the objects' own bytes) and
    `kv_head_dim` (values of a vector; default the objects' last dimension)."""
    if int(kwargs.get("aes_bits", 128)) != 128:
        raise ValueError("gpu aesgcm supports aes_bits=128 only")
    master_key_path = str(kwargs.get("master_key_path", ""))
    if not master_key_path:
        raise ValueError("gpu_aesgcm requires master_key_path")
    with open(master_key_path, "rb") as f:
        master_key = f.read()
    provider = HkdfKeyProvider(master_key, key_len=16, info_prefix=HKDF_INFO_PREFIX)
    device = kwargs.get("device")
    kv_format, kv_head_dim = kwargs.get("kv_format"), kwargs.get("kv_head_dim")
    ctx = GpuSerdeContext(provider, device=None if device is None else int(device), kv_format=kv_format or None,
                          kv_head_dim=None if kv_head_dim is None else int(kv_head_dim))
    return GpuAesGcmSerdeProcessor(ctx, max_workers=int(kwargs.get("max_workers", 1)))


register_serde_factory(SERDE_TYPE, create_gpu_aesgcm_serde)
