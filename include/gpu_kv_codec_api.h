/*
 * KV-cache codec: 8- and 4-bit records of KV objects, written on the GPU before they are sealed
 * and read back after they are opened. An extension; ConfKV has no counterpart.
 *
 * A KV object holds vectors of head_dim values, [planes][layers][tokens][heads][head_dim]: planes
 * is 2 for keys and values, 1 for a cache with one latent vector a token. quantise writes an
 * object as a record; dequantise reads a record back. Both take strided objects, or the tokens
 * of a paged cache named by their slots.
 *
 * Formats (x a value; A the largest |x| of its vector, or of its block):
 *   INT8   s = fp32(A / 127),  code = 127 x / A rounded to a whole number, ties to even
 *   FP8    s = fp32(A / 448),  code = 448 x / A rounded to e4m3, ties to even
 *   MXFP4  blocks of 32 values along the vector (the last may be short),
 *          e = max(floor(log2 A) - 2, -127), code = x / 2^e rounded to e2m1, ties to even, |code| <= 6
 * The quotient is not rounded before the code is. s is a float of the vector (in INT8 and FP8 at most
 * FLT_MAX / 127 and FLT_MAX / 448, rounded down, so that no code times s overflows); 2^e is a byte
 * e + 127 of the block. A value read back is code * s rounded to float and then to the object's type
 * (code * 2^e is exact in float). FP8 and MXFP4 codes of zero have the sign of their x, a zero or a value that
 * rounds to one; INT8 has one zero. The scale of a zero vector is 0 (its block's byte 0). A vector (block) with a
 * value that is not finite has codes 0 and scale NaN (byte 255): all of it reads back as NaN.
 *
 * Record, R = lmcache_gpu_kv_record_size bytes, little endian; V = planes * layers * tokens * heads
 * vectors in the object's order, C code bytes each (head_dim; MXFP4: ceil(head_dim / 2), value 2i in
 * the low half of byte i, the last high half of an odd head_dim 0):
 *   0   uint32 "KVQ1", tokens, layers | heads << 16, head_dim | format << 16 | dtype << 20 | planes << 24
 *   16  16 zero bytes
 *   32  codes, V * C bytes, then zero bytes to a multiple of 16
 *   ..  scales: V floats, or MXFP4: V * ceil(head_dim / 32) bytes; then zero bytes to a multiple of 16
 * Every byte of a record is written, so a sealed record holds no stale memory.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { LMCACHE_GPU_KV_INT8 = 0, LMCACHE_GPU_KV_FP8 = 1, LMCACHE_GPU_KV_MXFP4 = 2 };
enum { LMCACHE_GPU_KV_BF16 = 0, LMCACHE_GPU_KV_FP16 = 1, LMCACHE_GPU_KV_FP32 = 2 };

/* What all objects of a call have in common. planes 1..2, layers, heads
 * and head_dim 1..65535. */
typedef struct lmcache_gpu_kv_layout {
    int32_t format;
    int32_t dtype;
    uint32_t planes;
    uint32_t layers;
    uint32_t heads;
    uint32_t head_dim;
} lmcache_gpu_kv_layout;

/* A paged cache. Slot s is row s % block_size of block s / block_size; the vector of (plane, layer,
 * slot, head) starts block * block_stride + row * row_stride + head * head_stride elements behind
 * bases[plane * layers + layer]. The values of a vector follow one another. */
typedef struct lmcache_gpu_kv_pages {
    void* const* bases;     /* HOST array of planes * layers DEVICE pointers (512 at most), copied before return */
    uint64_t blocks;        /* blocks * block_size < 2^31 */
    uint32_t block_size;
    uint32_t reserved;      /* set to 0 */
    int64_t block_stride;   /* elements, not negative */
    int64_t row_stride;
    int64_t head_stride;
} lmcache_gpu_kv_pages;

/* `count` objects of `tokens` tokens each, at equal distances. Strides in elements, not negative. */
typedef struct lmcache_gpu_kv_run {
    void* object;           /* DEVICE, strided calls: the first object; paged calls: unused */
    int64_t object_stride;
    int64_t plane_stride;
    int64_t layer_stride;
    int64_t token_stride;
    int64_t head_stride;
    const int64_t* slots;   /* DEVICE, paged calls: the first object's `tokens` slots; strided calls: unused */
    int64_t slots_stride;   /* from one object's slots to the next's */
    void* record;           /* DEVICE, 16-byte aligned: the first object's record */
    int64_t record_stride;  /* bytes, a multiple of 16, R at least */
    uint64_t record_bytes;  /* bytes of the last object's record, R at least */
    int32_t* ok;            /* DEVICE, dequantise: `count` verdicts, or null; quantise: unused */
    uint32_t tokens;
    uint32_t count;
} lmcache_gpu_kv_run;

/* R for an object of `tokens` tokens; 0 for a layout or a size that the calls refuse. Needs no GPU. */
size_t lmcache_gpu_kv_record_size(const lmcache_gpu_kv_layout* layout, uint32_t tokens);

/*
 * Enqueue the records of all objects of `count` runs on `stream` (a cudaStream_t of `device`, null =
 * legacy default stream). layout, pages and runs are HOST memory, read before return; pages null =
 * strided objects. Nothing is allocated and nothing is kept; the calls can be captured.
 *
 * Paged: a slot below 0 (padding) or outside the cache has zero vectors in the record.
 *
 * ERR_ARGUMENT before any launch: a null or misaligned pointer (objects and bases: to their element;
 * records: 16 bytes), values out of the ranges above, an object of 2^31 vectors or more, a
 * record stride or size below R. Sources are not written to; a record must not overlap
 * any source or other record.
 */
int lmcache_gpu_kv_quantise_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages,
                                  const lmcache_gpu_kv_run* runs, size_t count, int device, void* stream);

/*
 * Enqueue the reading back of all records. A record whose header is not that of the layout and of
 * the run's `tokens` (a rejected frame's zeroed plaintext, say) has ok = 0 and its object, or
 * the slots that it names, are zero-filled; else ok = 1.
 *
 * Paged: slots below 0 or outside the cache are passed over, and no other slot than the named ones is
 * written to. The slots of one call have to differ from one another: of a slot named twice, each
 * value is one of the two tokens', and one vector may hold values of both.
 *
 * Destinations (objects, or the planes behind `bases`) must not share memory with one another or with any record:
 * what is written twice is undefined.
 */
int lmcache_gpu_kv_dequantise_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages,
                                    const lmcache_gpu_kv_run* runs, size_t count, int device, void* stream);

#ifdef __cplusplus
}
#endif
