"""A paged cache's requests on the GPU: block tables and slot maps, writing new tokens, attention of single new tokens.

Wraps lmcache_gpu_kv_{resize,append,attend}_async (include/gpu_kv_paged_api.h, which states what each does; an
extension, ConfKV has no counterpart). The cache is the codec's PagedKvCache: records read back into its slots are
attended to here, and the slots that a resize lists are those that KvCodec's paged calls and append take.

    blocks = KvBlockTables(lib, blocks=cache.blocks, block_size=cache.block_size, device=0)
    blocks.resize(tables, held, lengths, free, cursor, kept=kept, cursor_after=after, slots=slots, starts=starts)

    attention = KvAttention(lib, cache, query_heads=32)
    attention.append(layer, slots, keys, values)              # keys, values [tokens, heads, head_dim]
    attention.attend(layer, query, tables, kept, out)         # query, out [requests, query_heads, head_dim]

Every call enqueues on `stream` (default: the device's current one) and returns; the caller keeps the buffers alive
and synchronises.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .gpu_aesgcm import GpuAesGcmLibrary
from .kv_codec import DTYPES, KvLayout, PagedKvCache, _overlaps

# lmcache_gpu_kv_tables: tables and their stride, held, lengths, free, cursor, kept, cursor_after, slots, starts,
# capacity, requests, width, blocks, block_size, ring, reserved
TABLES = struct.Struct("<QqQQQQQQQQQ6I")
# lmcache_gpu_kv_vectors: keys and their two strides, values and theirs, slots, tokens
VECTORS = struct.Struct("<QqqQqqQQ")
# lmcache_gpu_kv_attention: query and its two strides, out and its, lse and its stride, tables and theirs, lengths,
# workspace and its bytes, requests, query_heads, value_dim, width, window, scale
ATTENTION = struct.Struct("<QqqQqqQqQqQQQ5If")

assert TABLES.size == 112 and VECTORS.size == 64 and ATTENTION.size == 128

PAGED_SYMBOLS = (
    "lmcache_gpu_kv_resize_async",
    "lmcache_gpu_kv_append_async",
    "lmcache_gpu_kv_attend_workspace_size",
    "lmcache_gpu_kv_attend_async",
)


def _declare(lib) -> None:
    if getattr(lib, "_kv_paged_declared", False):
        return
    vp, u32 = ctypes.c_void_p, ctypes.c_uint32
    lib.lmcache_gpu_kv_resize_async.argtypes = [ctypes.c_char_p, ctypes.c_int, vp]
    lib.lmcache_gpu_kv_append_async.argtypes = [vp, vp, u32, ctypes.c_char_p, ctypes.c_int, vp]
    lib.lmcache_gpu_kv_attend_async.argtypes = [vp, vp, u32, ctypes.c_char_p, ctypes.c_int, vp]
    for name in PAGED_SYMBOLS:
        getattr(lib, name).restype = ctypes.c_int
    lib.lmcache_gpu_kv_attend_workspace_size.argtypes = [vp, u32, u32]
    lib.lmcache_gpu_kv_attend_workspace_size.restype = ctypes.c_size_t
    lib._kv_paged_declared = True


class _Calls:
    """What both classes have in common: the device, its stream, checks of whole-number tensors."""

    def __init__(self, library: GpuAesGcmLibrary, device: int | torch.device):
        self.library = library
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type != "cuda" or self.device.index is None:
            raise ValueError("kv paged: device must be a CUDA device with its index")
        self._index = self.device.index
        _declare(library.lib)

    def _stream(self, stream) -> int:
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self._index)
        if stream.device != self.device:
            raise ValueError(f"kv paged: the stream is not one of {self.device}")
        return stream.cuda_stream

    def _row(self, name, t, dtype, count) -> int:
        """The address of a contiguous [count] tensor."""
        if t.dtype is not dtype or t.get_device() != self._index or t.shape != (count,):
            raise ValueError(f"kv paged: {name} is a {dtype} tensor of {count} values on {self.device}")
        if not t.is_contiguous():
            raise ValueError(f"kv paged: the values of {name} have to follow one another")
        return t.data_ptr()

    def _rows(self, tables, requests) -> tuple[int, int, int]:
        """Address, stride and width of block tables [requests, width]."""
        shape = tables.shape
        if tables.dtype is not torch.int32 or tables.get_device() != self._index or len(shape) != 2 or shape[0] != requests:
            raise ValueError(f"kv paged: tables are an int32 tensor [{requests}, width] on {self.device}")
        stride, step = tables.stride()
        if step != 1 and shape[1] > 1:
            raise ValueError("kv paged: the names of a table's row have to follow one another")
        return tables.data_ptr(), stride, shape[1]


class KvBlockTables(_Calls):
    """Block tables of requests in a cache of `blocks` blocks of `block_size` tokens."""

    def __init__(self, library: GpuAesGcmLibrary, *, blocks: int, block_size: int, device: int | torch.device = 0):
        super().__init__(library, device)
        self.blocks, self.block_size = int(blocks), int(block_size)
        if self.blocks < 0 or self.block_size < 1 or max(self.blocks, 1) * self.block_size >= 1 << 31:
            raise ValueError("kv paged: a cache has blocks of one token at least, and fewer than 2^31 slots")
        self._resize = library.lib.lmcache_gpu_kv_resize_async

    def resize(self, tables, held, lengths, free, cursor, *, kept, cursor_after, slots=None, starts=None,
               stream: torch.cuda.Stream | None = None) -> None:
        """Take requests from `held` to `lengths` tokens (int32 [requests]; 0 ends one): take blocks for those that grow
        from the ring `free` (int32; `cursor` int32 [2]: the place of its first free name, and how many there are) into
        their rows of `tables` (int32 [requests, width]), give those of the others back behind the ring's end.
        `kept` (int32 [requests]): what each holds then, `held` where it grows and there was no room; `cursor_after`: the
        cursor of the next call; `slots` (int64): the slots of all new tokens, -1 behind the last; `starts`
        (int64 [requests + 1]): where in it each request's begin. Outputs share no memory with inputs."""
        shape = held.shape
        n = shape[0]
        handle = self._stream(stream)
        ptr, stride, width = self._rows(tables, n)
        ring, i32, index = free.numel(), torch.int32, self._index
        # all at once; where something is wrong, one by one to say what
        good = len(shape) == 1 and lengths.shape == shape and kept.shape == shape and cursor.shape == cursor_after.shape == (2,)
        for t in (held, lengths, kept, cursor, cursor_after):
            good = good and t.dtype is i32 and t.get_device() == index and t.is_contiguous()
        if not good:
            for name, t, count in (("held", held, n), ("lengths", lengths, n), ("kept", kept, n), ("cursor", cursor, 2), ("cursor_after", cursor_after, 2)):
                self._row(name, t, i32, count)
        slots_ptr = starts_ptr = capacity = 0
        if slots is not None:
            capacity = slots.numel()
            # an empty tensor has no address; any other than null says that there is a list, of no places
            slots_ptr = self._row("slots", slots, torch.int64, capacity) or 8
            if starts is not None:
                starts_ptr = self._row("starts", starts, torch.int64, n + 1)
        elif starts is not None:
            raise ValueError("kv paged: starts are places in slots")
        raw = TABLES.pack(ptr, stride, held.data_ptr(), lengths.data_ptr(), self._row("free", free, i32, ring), cursor.data_ptr(),
                          kept.data_ptr(), cursor_after.data_ptr(), slots_ptr, starts_ptr, capacity, n, width, self.blocks,
                          self.block_size, ring, 0)
        rc = self._resize(raw, self._index, handle)
        if rc != 0:
            self.library.check(rc, "kv_resize")


class KvAttention(_Calls):
    """Writing new tokens to a paged cache, and attention of one new token a request to it. `query_heads`: a multiple of the
    cache's heads; `value_dim`: with one plane, how many values of a vector are its value (default all); `scale`: of the
    products (default head_dim ** -0.5); `window`: how many of the last tokens are attended to (0: all)."""

    def __init__(self, library: GpuAesGcmLibrary, cache: PagedKvCache, *, query_heads: int, value_dim: int | None = None,
                 scale: float | None = None, window: int = 0):
        self.dtype, self.planes, self.layers, self.heads, self.head_dim, device = cache.signature
        super().__init__(library, device)
        self.cache = cache
        self.query_heads, self.window = int(query_heads), int(window)
        self.value_dim = self.head_dim if value_dim is None else int(value_dim)
        self.scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not 1 <= self.query_heads <= 65535 or self.query_heads % self.heads:
            raise ValueError(f"kv paged: query_heads is a multiple of the cache's {self.heads} heads, 65535 at most")
        if self.head_dim > 1024:
            raise ValueError("kv paged: attention takes vectors of 1024 values at most")
        if not 1 <= self.value_dim <= self.head_dim or self.planes == 2 and self.value_dim != self.head_dim:
            raise ValueError("kv paged: value_dim is head_dim, or with one plane 1 to head_dim")
        if not abs(self.scale) < 2.0 ** 127 or not 0 <= self.window < 1 << 32:
            raise ValueError("kv paged: scale has to be finite and below 2^127, window 0 to 2^32 - 1")
        self._layout = KvLayout(0, DTYPES.index(self.dtype), self.planes, self.layers, self.heads, self.head_dim)
        self._layout_ptr = ctypes.addressof(self._layout)
        lib = library.lib
        self._append, self._attend = lib.lmcache_gpu_kv_append_async, lib.lmcache_gpu_kv_attend_async
        self._workspace = int(lib.lmcache_gpu_kv_attend_workspace_size(self._layout_ptr, self.query_heads, self.value_dim))

    def _vectors(self, name, t, shape) -> tuple[int, int, int]:
        if t.dtype is not self.dtype or t.get_device() != self._index or t.shape != shape:
            raise ValueError(f"kv paged: {name} are a {self.dtype} tensor {list(shape)} on {self.device}")
        strides = t.stride()
        if strides[2] != 1 and shape[2] > 1:
            raise ValueError("kv paged: the values of a vector have to follow one another")
        return t.data_ptr(), strides[0], strides[1]

    def _layer(self, layer) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"kv paged: layer is one of the cache's {self.layers}")
        return layer

    def append(self, layer: int, slots, keys, values=None, stream: torch.cuda.Stream | None = None) -> None:
        """Write tokens' vectors [tokens, heads, head_dim] into their slots (int64 [tokens]) of a layer. Slots below 0 or
        outside the cache are passed over; the others have to differ from one another. A cache whose planes share memory
        is refused."""
        if (values is None) != (self.planes == 1):
            raise ValueError(f"kv paged: the cache has {self.planes} planes")
        tokens = slots.shape[0]
        shape = (tokens, self.heads, self.head_dim)
        places = self._vectors("keys", keys, shape)
        more = (0, 0, 0) if values is None else self._vectors("values", values, shape)
        raw = VECTORS.pack(*places, *more, self._row("slots", slots, torch.int64, tokens), tokens)
        rc = self._append(self._layout_ptr, self.cache.writable()._pages_ptr, self._layer(layer), raw, self._index, self._stream(stream))
        if rc != 0:
            self.library.check(rc, "kv_append")

    def workspace(self) -> torch.Tensor:
        """A workspace for attend: calls that use the same one have to follow one another on the device."""
        return torch.empty(self._workspace, dtype=torch.uint8, device=self.device)

    def attend(self, layer: int, query, tables, lengths, out, lse=None, workspace=None,
               stream: torch.cuda.Stream | None = None) -> None:
        """out[r] = softmax(scale query[r] keys) values over the `lengths[r]` tokens (int32) that row r of `tables` (int32 [requests,
        width]) names, the last `window` of them; zeros where there are none. query [requests, query_heads, head_dim], out
        [requests, query_heads, value_dim]; lse (float32 [requests, query_heads]): the log of the sum of exponents.
        Without a workspace the call takes one of its own from torch's allocator. out, lse and the workspace share no memory with
        one another or with what is read."""
        n = lengths.shape[0]
        query_at = self._vectors("query", query, (n, self.query_heads, self.head_dim))
        out_at = self._vectors("out", out, (n, self.query_heads, self.value_dim))
        if not out.is_contiguous() and _overlaps(out.shape, out.stride()):
            raise ValueError("kv paged: out may not overlap itself")
        lse_at = (0, 0)
        if lse is not None:
            if lse.dtype is not torch.float32 or lse.get_device() != self._index or lse.shape != (n, self.query_heads):
                raise ValueError(f"kv paged: lse is a float32 tensor [{n}, {self.query_heads}] on {self.device}")
            lse_at = lse.data_ptr(), lse.stride(0)
            if self.query_heads > 1 and lse.stride(1) != 1 or n > 1 and lse_at[1] < self.query_heads:
                raise ValueError("kv paged: the values of a row of lse have to follow one another, and rows may not overlap")
        handle = self._stream(stream)
        if workspace is None:
            if stream is None:
                workspace = self.workspace()
            else:
                with torch.cuda.stream(stream):
                    workspace = self.workspace()
        elif workspace.dtype is not torch.uint8 or workspace.get_device() != self._index or not workspace.is_contiguous():
            raise ValueError(f"kv paged: a workspace is a contiguous uint8 tensor on {self.device}")
        rows = self._rows(tables, n)
        raw = ATTENTION.pack(*query_at, *out_at, *lse_at, rows[0], rows[1], self._row("lengths", lengths, torch.int32, n),
                             workspace.data_ptr(), workspace.numel(), n, self.query_heads, self.value_dim, rows[2],
                             self.window, self.scale)
        rc = self._attend(self._layout_ptr, self.cache._pages_ptr, self._layer(layer), raw, self._index, handle)
        if rc != 0:
            self.library.check(rc, "kv_attend")
