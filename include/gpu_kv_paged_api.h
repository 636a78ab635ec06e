/*
 * A paged cache's requests: block tables and slot maps, writing new tokens, attention of one new token a
 * request. An extension; ConfKV has no counterpart. The cache is the one that the KV-cache codec reads and
 * writes (gpu_kv_codec_api.h: lmcache_gpu_kv_layout, whose format these calls do not look at, and
 * lmcache_gpu_kv_pages): records that are read back into its slots are attended to here, and the slots that
 * resize lists are what the codec's paged calls and append take.
 *
 * All structures are HOST memory, read before return; the pointers in them are DEVICE memory. Nothing is
 * allocated and nothing is kept; every call can be captured. Calls that write the same memory, a shared
 * workspace among it, have to follow one another on the device.
 */
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "gpu_kv_codec_api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Requests whose lengths change. Row r of `tables` names the blocks of request r in turn: token i lies in row
 * i % block_size of block tables[r][i / block_size]. `free` is a ring of block names: the free ones are the
 * cursor[1] names from place cursor[0] on, past the ring's end at its beginning. */
typedef struct lmcache_gpu_kv_tables {
    int32_t* tables;         /* `requests` rows of `width` names */
    int64_t table_stride;    /* from row to row, `width` at least */
    const int32_t* held;     /* tokens that each request holds, whose blocks its row names */
    const int32_t* lengths;  /* tokens that it is to hold */
    int32_t* free;           /* ring of `ring` names */
    const int32_t* cursor;   /* place of the first free name, number of free names */
    int32_t* kept;           /* out: tokens that each request holds now */
    int32_t* cursor_after;   /* out: the cursor after the call */
    int64_t* slots;          /* out, or null: the slots of all new tokens */
    int64_t* starts;         /* out, or null: requests + 1 places in `slots`, where each request's begin */
    uint64_t capacity;       /* places of `slots`, below 2^31 - 1 */
    uint32_t requests;       /* below 2^24 */
    uint32_t width;          /* below 2^31 - 1 */
    uint32_t blocks;         /* of the cache; blocks * block_size < 2^31 */
    uint32_t block_size;
    uint32_t ring;           /* below 2^31 - 1 */
    uint32_t reserved;       /* set to 0 */
} lmcache_gpu_kv_tables;

/*
 * Enqueue the change of all requests from `held` to `lengths`.
 *
 * A request that grows takes names from the front of the ring, in the order of the requests; they become the
 * next names of its row. A request that shrinks (length 0: ends) gives its last names back behind the ring's
 * end, in the order of the requests and of its row; those can be taken from the next call on. kept[r] is then
 * lengths[r]. From the first request on for which names or places in `slots` run out, no request
 * grows: kept[r] is held[r], and its row stays. So it is for a request whose length is below 0 or
 * over width * block_size. Where held is that, kept is 0 and nothing of the request is read or written.
 *
 * slots: for each request that grew the slots of its tokens held .. lengths - 1, in the order of the
 * requests; -1 behind the last (the codec's calls and append pass over it), and for a token whose block is
 * not one of the cache's. Names that a row has behind its blocks stay as they are.
 *
 * A cursor that is no place or number of the ring's is brought into its range. Names that the ring has no room for are dropped.
 *
 * ERR_ARGUMENT before any launch: a null pointer (but slots and starts; free where ring is 0; any but
 * cursor and cursor_after where requests is 0), pointers that are not aligned to their
 * element, starts without slots, values out of the ranges above; kept, cursor_after, slots, starts, the ring or the rows sharing
 * memory with one another or with an input.
 */
int lmcache_gpu_kv_resize_async(const lmcache_gpu_kv_tables* tables, int device, void* stream);

/* New tokens' vectors of one layer. Strides in elements, not negative; the values of a vector follow one another. */
typedef struct lmcache_gpu_kv_vectors {
    const void* keys;        /* [tokens][heads][head_dim] of the cache's type */
    int64_t key_stride;      /* from token to token */
    int64_t key_head_stride;
    const void* values;      /* likewise; unused with one plane */
    int64_t value_stride;
    int64_t value_head_stride;
    const int64_t* slots;    /* one a token */
    uint64_t tokens;         /* below 2^31 */
} lmcache_gpu_kv_vectors;

/*
 * Enqueue the writing of tokens into their slots of a layer. Slots below 0 or outside the cache are passed over,
 * and no other slot than the named ones is written to. The slots have to differ from one another: of a slot
 * named twice, each value is one of the two tokens'. The planes must not share memory with each other or
 * with the vectors.
 *
 * ERR_ARGUMENT before any launch: null or misaligned pointers (vectors and bases to their element), a layer that is none, values
 * out of the ranges above or of the codec's.
 */
int lmcache_gpu_kv_append_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages, uint32_t layer,
                                const lmcache_gpu_kv_vectors* vectors, int device, void* stream);

/* One new token's query heads a request. Strides in elements, not negative; the values of a vector follow one another. */
typedef struct lmcache_gpu_kv_attention {
    const void* query;       /* [requests][query_heads][head_dim] of the cache's type */
    int64_t query_stride;    /* from request to request */
    int64_t query_head_stride;
    void* out;               /* [requests][query_heads][value_dim] of the cache's type */
    int64_t out_stride;
    int64_t out_head_stride;
    float* lse;              /* [requests][query_heads], or null */
    int64_t lse_stride;
    const int32_t* tables;   /* `requests` rows of `width` names, as above */
    int64_t table_stride;
    const int32_t* lengths;  /* tokens of each request */
    void* workspace;         /* 16-byte aligned, any contents */
    uint64_t workspace_bytes;
    uint32_t requests;       /* below 2^24 */
    uint32_t query_heads;    /* a multiple of the cache's heads; query head j reads head j / (query_heads / heads) */
    uint32_t value_dim;      /* two planes: head_dim; one: 1 .. head_dim */
    uint32_t width;          /* below 2^31 - 1 */
    uint32_t window;         /* 0: all tokens; else the last `window` */
    float scale;
} lmcache_gpu_kv_attention;

/* Bytes of workspace that attend takes, whatever the requests; 0 for values that it refuses. Needs no GPU. */
size_t lmcache_gpu_kv_attend_workspace_size(const lmcache_gpu_kv_layout* layout, uint32_t query_heads, uint32_t value_dim);

/*
 * Enqueue out = sum_i exp(s_i - lse) v_i with s_i = scale q k_i and lse = log sum_i exp(s_i) for every request and query head, i
 * over the request's tokens (the last `window` of them). k is the layer's first plane, v its second; with one plane
 * v_i is the first value_dim values of k_i. Tokens whose block is not one of the cache's are left out, lengths below 0 are 0,
 * and lengths over width * block_size are that. Where no token is left, out is 0 and lse -infinity. What lies in the cache
 * beside the tokens is not read. Scores, sums and products are held in 32 bits; with 16-bit types the weights exp(s_i - m), m the
 * largest score, may enter the products as the sum of two values of that type (off by 2^-15 of a weight in bfloat16; by 2^-20
 * of it in half, or by 2^-38 where that is more).
 * The order of the sums depends on the lengths, the shapes and the alignment alone: equal calls give equal bits.
 * out, lse and the workspace share no memory with one another or with anything that is read, and the rows of out and lse not with one another.
 *
 * ERR_ARGUMENT before any launch: null or misaligned pointers, a layer that is none, head_dim above 1024, query_heads above 65535, a workspace
 * that is too small, a scale that is not finite (times log2 e, in 32 bits), requests * (width * block_size / 64 + 4) of 2^31 or more (width *
 * block_size up to 2^31 - 1, which is all that a length counts), values out of the ranges above or of the codec's.
 */
int lmcache_gpu_kv_attend_async(const lmcache_gpu_kv_layout* layout, const lmcache_gpu_kv_pages* pages, uint32_t layer,
                                const lmcache_gpu_kv_attention* attention, int device, void* stream);

#ifdef __cplusplus
}
#endif
