/* A plan of packed requests (h3_hip_sdpa_packed_plan, hk_packed.hip), for the
 * attention kernels that run it: over bf16 keys and values (hk_packed.hip) and
 * over a cache in 8 bits (hk_kv8.hip). */
#ifndef HK_PACKED_H
#define HK_PACKED_H

#include "hk_common.h"
#include "hk_internal.h"

#define HK_PACKED_MAX_DIM 256u
#define HK_PACKED_MAX_KEYS 0xffffff00u /* of a request */
#define HK_PACKED_WAVES 4u
#define HK_PACKED_QB (HK_PACKED_WAVES * 32u) /* virtual rows of an item */

/* a request with query rows, in device memory */
struct hk_packed_request {
    uint32_t q_first, q_rows, kv_first, kv_rows;
    uint32_t before; /* query rows of the requests before it in the plan */
};

/* A work item: virtual rows [row, rows) of a request, at most HK_PACKED_QB, of
 * one key head, over key tiles [tile, tile_end) of the request's keys.  Whole
 * items store their rows; a piece leaves its sums in part `part`.  An item of
 * no rows fills a place in the launch. */
struct hk_packed_item {
    uint32_t q_first, rows, row, kv_head;
    uint32_t kv_first, kv_rows, tile, tile_end;
    uint32_t part;
};
#define HK_PACKED_WHOLE 0xffffffffu

/* The pieces [part, + pieces) of one item's rows. */
struct hk_packed_join {
    uint32_t q_first, rows, row, kv_head;
    uint32_t part, pieces;
};

/* hk_record.n of a plan */
enum { HK_PACKED_HEADS, HK_PACKED_KV_HEADS, HK_PACKED_DIM,
       HK_PACKED_REQUESTS, /* those with query rows */
       HK_PACKED_ROWS,     /* query rows of all requests */
       HK_PACKED_Q_END,    /* rows that the query and output tensors hold */
       HK_PACKED_KV_END,
       HK_PACKED_ITEMS,    /* entries of each list, which follow each other: */
       HK_PACKED_JOINS,    /* requests, items, joins */
       HK_PACKED_JOIN_ROWS, /* the most virtual rows of a join */
       HK_PACKED_PARTS,
       HK_PACKED_OFF_BLOCKS, /* a request's keys begin inside 64 rows */
       HK_PACKED_FEW, HK_PACKED_MANY, /* has items of up to 32 rows, over */
       HK_PACKED_SPANS, HK_PACKED_SPAN_BLOCKS };
#define HK_PACKED_TOO_MANY UINT32_MAX /* blocks of spans: they have no list */

/* For a cache in blocks of 64 rows that is unpacked into rows for the items of
 * many rows: blocks [block, + blocks) of it, which those items read, go to
 * blocks [at, + blocks) of the rows.  If any request has such items and all
 * begin at whole blocks, the spans follow a plan's lists, in the order of block
 * and blocks, one for each pair that a request has. */
struct hk_packed_span {
    uint32_t block, at, blocks;
};

/* What the codes of a block's keys are multiplied by before the products, and
 * the products after them: over 256 dims a raw score, the query's product with
 * the codes, would be up to 2^15 times the query's largest element, past F32's
 * range where the score, of keys of a scale under 1, is not.  A block of zeros (a
 * scale of 0) has zeros, whatever its codes, and what multiplies them leaves the
 * -inf of keys past the end. */
__device__ __forceinline__ float hk_packed_code_unit(float scale) {
    return scale == 0.0f ? 0.0f : scale < 1.0f ? 0x1p-15f : 1.0f;
}

__device__ __forceinline__ float hk_packed_code_scale(float scale) {
    return scale == 0.0f ? 1.0f : scale < 1.0f ? scale * 0x1p15f : scale;
}

struct hk_packed_args {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    uint64_t q_stride, kv_stride; /* elements from a row to the next */
    uint32_t heads, kv_heads, dim, group;
    float scale, scale_log2;
    const hk_packed_request *requests;
    uint32_t request_count, rows;
    const hk_packed_item *items;
    const hk_packed_join *joins;
    /* pieces' sums: F32 O [part][HK_PACKED_QB][padded dim], not divided, and
     * (reference, sum) [part][HK_PACKED_QB] */
    float *part_o;
    float2 *part_ml;
    /* keys that are codes times a unit (hk_packed_codes): where they lie among
     * the rows, their scales, [block][key head][2], and what the values are
     * divided by, of a span's first block [block among the spans'][key head] */
    const hk_packed_span *spans;
    uint32_t span_count;
    const float *key_scales, *value_units;
};

/* The last request that begins at or before the plan's nth query row. */
__device__ __forceinline__ uint32_t hk_packed_request_of(
    const hk_packed_request *requests, uint32_t count, uint32_t nth) {
    uint32_t low = 0, high = count;
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (requests[mid].before <= nth) low = mid;
        else high = mid;
    }
    return low;
}

/* Sets what a plan says in the arguments of a launch. */
static inline void hk_packed_of_plan(hk_packed_args &a,
                                     const h3_gpu_tensor *plan, float scale) {
    const uint32_t *n = plan->record.n;
    a.heads = n[HK_PACKED_HEADS];
    a.kv_heads = n[HK_PACKED_KV_HEADS];
    a.dim = n[HK_PACKED_DIM];
    a.scale = scale;
    a.group = a.heads / a.kv_heads;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.requests = (const hk_packed_request *)plan->data;
    a.request_count = n[HK_PACKED_REQUESTS];
    a.rows = n[HK_PACKED_ROWS];
    a.items = (const hk_packed_item *)(a.requests + a.request_count);
    a.joins = (const hk_packed_join *)(a.items + n[HK_PACKED_ITEMS]);
    a.spans = (const hk_packed_span *)(a.joins + n[HK_PACKED_JOINS]);
    a.span_count = n[HK_PACKED_SPANS];
}

/* Elements that a tensor needs for `rows` rows from `offset` on; sizes past
 * what an address can hold come out as the largest. */
static inline size_t hk_packed_extent(size_t offset, uint64_t stride,
                                      uint64_t rows, uint64_t width) {
    const uint64_t need = rows ? (rows - 1) * stride + width : 0;
    return offset > SIZE_MAX - need ? SIZE_MAX : offset + need;
}

/* Whether the matrix-core kernel takes these rows. */
bool hk_packed_takes(const struct h3_gpu *gpu, const hk_packed_args &a);
/* Launches it on the items of many rows, over codes. */
void hk_packed_many_scaled(struct h3_gpu *gpu, const hk_packed_args &a,
                           const uint32_t *n);
/* Launches the join of pieces' sums in rows of `padded` (64 or 128) dims. */
void hk_packed_join_pieces(struct h3_gpu *gpu, const hk_packed_args &a,
                           const uint32_t *n, uint32_t padded);

#endif
