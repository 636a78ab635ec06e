"""KV-cache codec: 8- and 4-bit records of KV objects, on the GPU.

Wraps lmcache_gpu_kv_{quantise,dequantise}_async (include/gpu_kv_codec_api.h, which states the
formats and the record layout; an extension, ConfKV has no counterpart). A record is what is sealed in the
place of the object, so that frames, host copies and storage shrink to a half (int8, fp8) or a quarter
(mxfp4) of a 16-bit cache.

    codec = KvCodec(lib, "int8", torch.bfloat16, planes=2, layers=32, heads=8, head_dim=128, device=0)
    records = torch.empty(n, codec.record_bytes(256), dtype=torch.uint8, device="cuda:0")
    codec.quantise(objects, records)                  # objects [n, 2, 32, 256, 8, 128]
    codec.dequantise(records, restored, ok=ok)        # ok: int32 [n], 1 where the record was this codec's

    cache = PagedKvCache(codec, layers)               # one [2, blocks, block_size, 8, 128] tensor a layer
    codec.quantise_paged(cache, slots, records)       # slots [n, 256] int64: tokens that become n objects
    codec.dequantise_paged(records, cache, slots, ok=ok)

Every call enqueues on `stream` (default: the device's current one) and returns; as with seal_async the
caller keeps the buffers alive and synchronises.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .gpu_aesgcm import GpuAesGcmLibrary

FORMATS = ("int8", "fp8", "mxfp4")
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
HEADER_BYTES = 32
MX_BLOCK = 32
RECORD_ALIGN = 16
MAX_BASES = 512


class KvLayout(ctypes.Structure):
    """lmcache_gpu_kv_layout."""

    _fields_ = [("format", ctypes.c_int32), ("dtype", ctypes.c_int32), ("planes", ctypes.c_uint32),
                ("layers", ctypes.c_uint32), ("heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32)]


class KvPages(ctypes.Structure):
    """lmcache_gpu_kv_pages."""

    _fields_ = [("bases", ctypes.c_void_p), ("blocks", ctypes.c_uint64), ("block_size", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("block_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]


# lmcache_gpu_kv_run: object and its five strides, slots and their stride, record, record_stride,
# record_bytes, ok, tokens, count
RUN = struct.Struct("<Q5qQqQqQQII")

assert ctypes.sizeof(KvLayout) == 24 and ctypes.sizeof(KvPages) == 48 and RUN.size == 104

CODEC_SYMBOLS = (
    "lmcache_gpu_kv_record_size",
    "lmcache_gpu_kv_quantise_async",
    "lmcache_gpu_kv_dequantise_async",
)


def record_size(format: str, head_dim: int, vectors: int) -> int:
    """Bytes of a record of `vectors` vectors: lmcache_gpu_kv_record_size without the library."""
    mx = format == "mxfp4"
    codes = vectors * ((head_dim + 1) // 2 if mx else head_dim)
    scales = vectors * (-(-head_dim // MX_BLOCK) if mx else 4)
    return HEADER_BYTES + -(-codes // 16) * 16 + -(-scales // 16) * 16


def _declare(lib) -> None:
    if getattr(lib, "_kv_codec_declared", False):
        return
    vp = ctypes.c_void_p
    lib.lmcache_gpu_kv_record_size.argtypes = [vp, ctypes.c_uint32]
    lib.lmcache_gpu_kv_record_size.restype = ctypes.c_size_t
    for name in ("lmcache_gpu_kv_quantise_async", "lmcache_gpu_kv_dequantise_async"):
        fn = getattr(lib, name)
        fn.argtypes = [vp, vp, ctypes.c_char_p, ctypes.c_size_t, ctypes.c_int, vp]
        fn.restype = ctypes.c_int
    lib._kv_codec_declared = True


def _as_list(x):
    return [x] if isinstance(x, torch.Tensor) else list(x)


def _overlaps(shape, strides) -> bool:
    """Whether two indices of a tensor may share memory: in the order of the strides, each has to pass
    over all that the smaller ones reach."""
    reach = 0
    for stride, size in sorted((s, n) for n, s in zip(shape, strides) if n > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


def _meet(distance, dims) -> bool:
    """Whether two planes of the same shape and strides, `distance` bytes apart, share memory: whether whole numbers
    |a| < n give the distance as the sum of a * stride over `dims`, (stride, n) in falling order, of which each stride passes over
    all that the smaller ones reach. So only the two multiples of a stride next to the distance come into question."""
    if not dims:
        return distance == 0
    stride, n = dims[0]
    a = distance // stride
    return any(abs(k) < n and _meet(distance - k * stride, dims[1:]) for k in (a, a + 1))


class KvCodec:
    """A format for the objects of one cache: [planes, layers, tokens, heads, head_dim] of `dtype`."""

    def __init__(self, library: GpuAesGcmLibrary, format: str, dtype: torch.dtype, *, planes: int, layers: int,
                 heads: int, head_dim: int, device: int | torch.device = 0):
        if format not in FORMATS:
            raise ValueError(f"kv codec: format must be one of {', '.join(FORMATS)}")
        if dtype not in DTYPES:
            raise ValueError("kv codec: dtype must be bfloat16, float16 or float32")
        self.library = library
        self.format, self.dtype = format, dtype
        self.planes, self.layers, self.heads, self.head_dim = int(planes), int(layers), int(heads), int(head_dim)
        if not (1 <= self.planes <= 2 and all(1 <= n <= 65535 for n in (self.layers, self.heads, self.head_dim))):
            raise ValueError("kv codec: planes must be 1 or 2; layers, heads and head_dim 1 to 65535")
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type != "cuda" or self.device.index is None:
            raise ValueError("kv codec: device must be a CUDA device with its index")
        self._index = self.device.index
        _declare(library.lib)
        self._layout = KvLayout(FORMATS.index(format), DTYPES.index(dtype), self.planes, self.layers, self.heads,
                                self.head_dim)
        self._layout_ptr = ctypes.addressof(self._layout)
        self._sizes: dict[int, int] = {}
        self._quantise = library.lib.lmcache_gpu_kv_quantise_async
        self._dequantise = library.lib.lmcache_gpu_kv_dequantise_async
        self._shape = (self.planes, self.layers, self.heads, self.head_dim)
        self.signature = (self.dtype, *self._shape, self.device)

    # ---- records
    def record_bytes(self, tokens: int) -> int:
        """Bytes of the record of an object of `tokens` tokens."""
        size = self._sizes.get(tokens)
        if size is None:
            if not 0 <= tokens < 1 << 32:
                raise ValueError("kv codec: bad number of tokens")
            size = int(self.library.lib.lmcache_gpu_kv_record_size(self._layout_ptr, tokens))
            if size == 0:
                raise ValueError("kv codec: an object has to have fewer than 2^31 vectors")
            if len(self._sizes) < 4096:
                self._sizes[tokens] = size
        return size

    def split(self, record: torch.Tensor, tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Views of a record's (or of [n, R] records') codes and scales: codes [..., planes, layers, tokens,
        heads, head_dim] int8 or float8_e4m3fn (mxfp4: uint8, two values a byte), scales [..., planes, layers, tokens,
        heads] float32 (mxfp4: uint8, one a block of 32 values as their last dimension)."""
        vectors = self.planes * self.layers * tokens * self.heads
        mx = self.format == "mxfp4"
        size = (self.head_dim + 1) // 2 if mx else self.head_dim
        at = HEADER_BYTES + (vectors * size + 15) // 16 * 16
        per = -(-self.head_dim // MX_BLOCK)
        lead, index = record.shape[:-1], (self.planes, self.layers, tokens, self.heads)
        codes = record[..., HEADER_BYTES:HEADER_BYTES + vectors * size]
        scales = record[..., at:at + vectors * (per if mx else 4)]
        if mx:
            return codes.reshape(*lead, *index, size), scales.reshape(*lead, *index, per)
        codes = codes.view(torch.int8 if self.format == "int8" else torch.float8_e4m3fn)
        return codes.view(*lead, *index, size), scales.view(torch.float32).view(*lead, *index)

    # ---- arguments
    def _run(self, record, tokens, count, object_args, slots_args, ok) -> bytes:
        size = self._sizes.get(tokens) or self.record_bytes(tokens)
        if record.dtype is not torch.uint8 or record.get_device() != self._index:
            raise ValueError(f"kv codec: records are uint8 tensors on {self.device}")
        shape, strides = record.shape, record.stride()
        if len(shape) == 1 and count == 1:
            stride, room = 0, shape[0]
        elif len(shape) == 2 and shape[0] == count:
            stride, room = strides[0], shape[1]
        else:
            raise ValueError("kv codec: one record, or a row of records, for every object")
        if room < size:
            raise ValueError(f"kv codec: a record of {tokens} tokens takes {size} bytes")
        ptr = record.data_ptr()
        if strides[-1] != 1 or ptr % RECORD_ALIGN or count > 1 and (stride % RECORD_ALIGN or stride < size):
            raise ValueError("kv codec: records are contiguous, at multiples of 16 bytes, and do not overlap")
        ok_ptr = 0
        if ok is not None:
            if ok.dtype is not torch.int32 or ok.get_device() != self._index or ok.numel() != count or not ok.is_contiguous():
                raise ValueError(f"kv codec: ok is an int32 tensor of one value an object on {self.device}")
            ok_ptr = ok.data_ptr()
        return RUN.pack(*object_args, *slots_args, ptr, stride, size, ok_ptr, tokens, count)

    def _read_run(self, obj, record, ok) -> bytes:
        if obj.dtype is not self.dtype or obj.get_device() != self._index:
            raise ValueError(f"kv codec: objects are {self.dtype} tensors on {self.device}")
        shape, strides = obj.shape, obj.stride()
        if len(shape) == 5:
            count, stride = 1, 0
        elif len(shape) == 6:
            count, stride = shape[0], strides[0]
        else:
            raise ValueError("kv codec: objects are [planes, layers, tokens, heads, head_dim], or a row of them")
        planes, layers, tokens, heads, dim = shape[-5:]
        if (planes, layers, heads, dim) != self._shape:
            raise ValueError(f"kv codec: an object of shape {tuple(shape)} is not one of this codec's")
        if strides[-1] != 1 and dim > 1:
            raise ValueError("kv codec: the values of a vector have to follow one another")
        return self._run(record, tokens, count, (obj.data_ptr(), stride, *strides[-5:-1]), (0, 0), ok)

    def _written_run(self, obj, record, ok) -> bytes:
        if not obj.is_contiguous() and _overlaps(obj.shape, obj.stride()):
            raise ValueError("kv codec: an object that is written to may not overlap itself")
        return self._read_run(obj, record, ok)

    def _slots_run(self, slots, record, ok) -> bytes:
        if slots.dtype is not torch.int64 or slots.get_device() != self._index:
            raise ValueError(f"kv codec: slots are int64 tensors on {self.device}")
        shape, strides = slots.shape, slots.stride()
        if len(shape) == 1:
            count, stride = 1, 0
        elif len(shape) == 2:
            count, stride = shape[0], strides[0]
        else:
            raise ValueError("kv codec: slots are [tokens], or a row of them")
        tokens = shape[-1]
        if strides[-1] != 1 and tokens > 1:
            raise ValueError("kv codec: the slots of an object have to follow one another")
        return self._run(record, tokens, count, (0,) * 6, (slots.data_ptr(), stride), ok)

    def _call(self, fn, make, sources, records, ok, cache, stream) -> None:
        if isinstance(sources, torch.Tensor):
            sources, records = (sources,), _as_list(records)
            ok = ok if ok is None else _as_list(ok)
        if len(sources) != len(records) or ok is not None and len(ok) != len(sources):
            raise ValueError("kv codec: one tensor of records (and of verdicts) for every tensor of objects or slots")
        if len(sources) == 1:
            raw = make(sources[0], records[0], None if ok is None else ok[0])
        elif ok is None:
            raw = b"".join([make(s, r, None) for s, r in zip(sources, records)])
        else:
            raw = b"".join([make(s, r, k) for s, r, k in zip(sources, records, ok)])
        if stream is None:
            handle = torch._C._cuda_getCurrentRawStream(self._index)
        else:
            if stream.device != self.device:
                raise ValueError(f"kv codec: the stream is not one of {self.device}")
            handle = stream.cuda_stream
        rc = fn(self._layout_ptr, cache, raw, len(sources), self._index, handle)
        if rc != 0:
            self.library.check(rc, fn.__name__.removeprefix("lmcache_gpu_").removesuffix("_async"))

    def _cache(self, cache) -> "PagedKvCache":
        if cache.signature != self.signature:
            raise ValueError("kv codec: the paged cache is not one of this codec's shape, type or device")
        return cache

    # ---- calls
    def quantise(self, objects, records, stream: torch.cuda.Stream | None = None) -> None:
        """Write the records of objects. `objects`: a [planes, layers, tokens, heads, head_dim] tensor of any
        strides with contiguous vectors, a row of them [n, ...], or a sequence of either; `records`: for each a uint8
        tensor [>= R], or [n, >= R]; they may share memory with nothing else in the call."""
        self._call(self._quantise, self._read_run, objects, records, None, None, stream)

    def dequantise(self, records, objects, ok=None, stream: torch.cuda.Stream | None = None) -> None:
        """Read records back into objects. `ok`: for each tensor of objects an int32 tensor of one verdict an object:
        1, or 0 where the record is not one of this codec's for so many tokens; such an object is zero-filled. The objects of a
        call may not share memory."""
        self._call(self._dequantise, self._written_run, objects, records, ok, None, stream)

    def quantise_paged(self, cache: "PagedKvCache", slots, records, stream: torch.cuda.Stream | None = None) -> None:
        """Write the records of tokens of a paged cache. `slots`: an int64 tensor [tokens] on the device, a row of
        them [n, tokens], or a sequence of either; a slot below 0 or outside the cache is a token of zeros."""
        self._call(self._quantise, self._slots_run, slots, records, None, self._cache(cache)._pages_ptr, stream)

    def dequantise_paged(self, records, cache: "PagedKvCache", slots, ok=None,
                         stream: torch.cuda.Stream | None = None) -> None:
        """Read records back into slots of a paged cache, and write to no other slot. Slots below 0 or outside the
        cache are passed over; the others have to differ from one another (of a slot named twice each value is one of the two
        tokens'). A cache whose planes share memory is
        refused."""
        self._call(self._dequantise, self._slots_run, slots, records, ok, self._cache(cache).apart()._pages_ptr, stream)


class PagedKvCache:
    """The layers of a paged cache as a codec's calls take them: for each layer a tensor [planes, blocks, block_size,
    heads, head_dim] (any strides with contiguous vectors, equal in all layers: pages that hold each head's tokens
    together are a transposed view), or a (keys, values) pair of [blocks, block_size, heads, head_dim]. Slot s is row
    s % block_size of block s // block_size. Keeps the tensors alive."""

    def __init__(self, codec: KvCodec, layers):
        self.signature = codec.signature
        # pairs as tuples of their own: the addresses below are good only while their tensors live
        self.layers = [layer if hasattr(layer, "data_ptr") else tuple(layer) for layer in layers]
        if len(self.layers) != codec.layers or codec.layers * codec.planes > MAX_BASES:
            raise ValueError(f"kv codec: a paged cache has the codec's {codec.layers} layers, and {MAX_BASES} planes at most")
        # every plane is [blocks, block_size, heads, head_dim], all of one shape and with one set of strides
        shape = strides = None
        bases = [[] for _ in range(codec.planes)]
        for layer in self.layers:
            joint = hasattr(layer, "data_ptr")              # one tensor a layer
            parts = (layer,) if joint else layer            # or keys and values apart
            joint = joint and len(layer.shape) == 5
            if (layer.shape[0] if joint else len(parts)) != codec.planes:
                raise ValueError(f"kv codec: a layer has {codec.planes} planes")
            for k, t in enumerate(parts):
                if t.dtype is not codec.dtype or t.get_device() != codec._index:
                    raise ValueError(f"kv codec: the layers are {codec.dtype} tensors on {codec.device}")
                mine, by, ptr = t.shape, t.stride(), t.data_ptr()
                if joint:
                    step = by[0] * codec.dtype.itemsize
                    for plane in range(codec.planes):
                        bases[plane].append(ptr + plane * step)
                    mine, by = mine[1:], by[1:]
                else:
                    bases[k].append(ptr)
                if shape is None:
                    shape, strides = mine, by
                elif mine != shape or by != strides:
                    raise ValueError("kv codec: all planes have the same shape and strides")
        if len(shape) != 4:
            raise ValueError("kv codec: a plane is [blocks, block_size, heads, head_dim]")
        blocks, size, heads, dim = shape
        if (heads, dim) != (codec.heads, codec.head_dim) or size < 1 or blocks * size >= 1 << 31:
            raise ValueError(f"kv codec: a plane of shape {tuple(shape)} is not one of this codec's")
        if strides[-1] != 1 and dim > 1:
            raise ValueError("kv codec: the values of a vector have to follow one another")
        self.blocks, self.block_size = blocks, size
        self._starts, self._itemsize, self._within, self._between = bases, codec.dtype.itemsize, None, None
        self._shape, self._strides = shape, strides
        self._bases = (ctypes.c_void_p * (codec.planes * codec.layers))(*[p for plane in bases for p in plane])
        self._pages = KvPages(ctypes.addressof(self._bases), blocks, size, 0, *strides[:3])
        self._pages_ptr = ctypes.addressof(self._pages)

    def _meet_any(self, distances) -> bool:
        dims = sorted(((s * self._itemsize, n) for n, s in zip(self._shape, self._strides) if n > 1), reverse=True)
        return any(_meet(d, dims) for d in distances)

    def writable(self) -> "PagedKvCache":
        """The cache, if no plane shares memory with itself or with its layer's other plane."""
        if self._within is None:
            self._within = self.blocks > 0 and (
                _overlaps(self._shape, self._strides) or
                len(self._starts) == 2 and self._meet_any({v - k for k, v in zip(*self._starts)}))
        if self._within:
            raise ValueError("kv codec: a cache that is written to may not overlap itself")
        return self

    def apart(self) -> "PagedKvCache":
        """The cache, if it is writable and no plane shares memory with another layer's either."""
        if self._between is None:
            self.writable()
            starts = sorted(p for plane in self._starts for p in plane)
            reach = sum(s * (n - 1) for n, s in zip(self._shape, self._strides)) * self._itemsize
            distances = set()
            for i, a in enumerate(starts if self.blocks > 0 else ()):
                for b in starts[i + 1:]:
                    if b - a > reach:
                        break
                    distances.add(b - a)
            self._between = self._meet_any(distances)
        if self._between:
            raise ValueError("kv codec: the layers of a cache that is written to may not overlap one another")
        return self
