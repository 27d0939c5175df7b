/* Keys and values cached in 8 bits (h3_hip_kv_int8_new, _store, _read in
 * h3_hip.h), and attention over them (h3_hip_sdpa_packed_int8_bf16): blocks of
 * 64 rows, each with one scale for its keys and one for its values a head.
 *
 * The codes lie in the order in which the matrix cores take them: a lane's 16
 * bytes are 16 dims of one key (the A operand of S^T = K . Q^T), or 16 keys of
 * one dim (of O^T = V^T . P^T), the keys in the order in which a lane of S^T
 * holds its scores.  So a wave reads 1 KiB at a time, whole lines, and V needs
 * no transposing reads.  A code is held as code + 128: one byte permutation
 * makes the f16 number 1024 + byte of it, one packed subtraction the code
 * (f16 holds whole numbers up to 2048).
 */
#include "hk_attn.h"
#include "hk_int8.h"
#include "hk_packed.h"

#include <math.h>

#include <algorithm>
#include <vector>

typedef _Float16 hk_f16x8 __attribute__((ext_vector_type(8)));

#define HK_KV8_BLOCK 64u
#define HK_KV8_RANGES 64u /* of a launch of the store */

/* hk_record.n of a cache */
enum { HK_KV8_BLOCKS, HK_KV8_HEADS, HK_KV8_DIM };

/* Dims of a block's rows, in whole groups of 32. */
__host__ __device__ __forceinline__ uint32_t hk_kv8_padded(uint32_t dim) {
    return (dim + 31u) & ~31u;
}

/* Where the code of a block's row and dim lies among the block's keys ... */
__device__ __forceinline__ uint32_t hk_kv8_key_at(uint32_t row, uint32_t dim,
                                                  uint32_t padded) {
    return (row >> 5) * padded * 32u + (dim >> 5) * 1024u +
           ((row & 31u) + ((dim >> 4) & 1u) * 32u) * 16u + (dim & 15u);
}

/* ... and its values, which follow them: byte b of lane l of 32 rows and 32
 * dims is dim l % 32 of row 16 (b / 8) + 8 (b / 4 % 2) + 4 (l / 32) + b % 4,
 * the order of a lane's scores in S^T. */
__device__ __forceinline__ uint32_t hk_kv8_value_at(uint32_t row, uint32_t dim,
                                                    uint32_t padded) {
    const uint32_t byte =
        ((row >> 4) & 1u) * 8u + ((row >> 3) & 1u) * 4u + (row & 3u);
    return (row >> 5) * padded * 32u + (dim >> 5) * 1024u +
           ((dim & 31u) + ((row >> 2) & 1u) * 32u) * 16u + byte;
}

struct hk_kv8_cache {
    uint8_t *codes; /* [block][head][keys, values][64 padded] */
    float2 *scales; /* [block][head]: of the keys, of the values */
    uint32_t blocks, heads, dim, padded;
};

static hk_kv8_cache hk_kv8_of(const h3_gpu_tensor *t) {
    hk_kv8_cache c = {(uint8_t *)t->data, NULL, t->record.n[HK_KV8_BLOCKS],
                      t->record.n[HK_KV8_HEADS], t->record.n[HK_KV8_DIM], 0};
    c.padded = hk_kv8_padded(c.dim);
    c.scales = (float2 *)(c.codes + (size_t)c.blocks * c.heads * 2u *
                                        HK_KV8_BLOCK * c.padded);
    return c;
}

/* A new cache's scales: 0, whatever its codes. */
__global__ void __launch_bounds__(256) hk_kv8_clear(float2 *scales, size_t n) {
    const size_t i = (size_t)blockIdx.x * 256u + threadIdx.x;
    if (i < n) scales[i] = make_float2(0.0f, 0.0f);
}

/* ------------------------------------------------------------ the store */

/* Rows [source, + rows) of the keys and values go to rows [cache, + rows) of
 * the cache, whose blocks are `before` and on of the launch. */
struct hk_kv8_range {
    uint32_t cache, source, rows, before;
};

struct hk_kv8_store_args {
    hk_kv8_cache cache;
    const uint16_t *key, *value;
    uint64_t stride;
    uint32_t count;
    hk_kv8_range ranges[HK_KV8_RANGES];
};

/* A thread's piece of a block's keys or values: eight dims, from `dim` on, of
 * four rows, from `row` on.  Its codes are whole words of either order: four
 * dims of a row, four rows of a dim. */
struct hk_kv8_piece {
    uint32_t row, dim;
    __device__ __forceinline__ hk_kv8_piece(uint32_t at, uint32_t padded) {
        row = at / (padded >> 3) * 4u;
        dim = at % (padded >> 3) * 8u;
    }
};

/* The image of a block's keys or values in LDS, as the cache has it, but that
 * 16-byte piece p lies at p ^ (p / 8 % 8): the words that threads write and
 * read at a time lie 16 bytes apart, over few banks. */
__device__ __forceinline__ uint32_t hk_kv8_image(uint32_t byte) {
    return byte ^ ((byte >> 3) & 0x70u);
}

/* One workgroup per block, head and one of keys and values: the new rows into
 * registers, their largest magnitude, the codes by way of the block's image in
 * LDS, whole lines to the cache.  A block whose first row is new takes its
 * scale from the new rows and zeros in the others; in any other its rows keep
 * their codes unless the scale grows, and where it does not, the new rows'
 * bytes alone are written.  PIECES of the block are a thread's, and ALIGNED rows
 * are read 16 bytes at a time.  889 rows of 40 heads of 128 take 9.0 us (3.0
 * TB/s; 13.2 with branches between the loads): 1200 workgroups, each a chain of
 * loads, maximum, codes and stores.  A row each of 16 requests, 8 heads: 5.2. */
template <int PIECES, bool ALIGNED>
__global__ void __launch_bounds__(256) hk_kv8_store(hk_kv8_store_args a) {
    __shared__ uint32_t tops[16];
    extern __shared__ __attribute__((aligned(16))) uint8_t image[];
    const hk_kv8_cache &c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    /* the last range that begins at or before the launch's block, a lane for
     * each (64 of them): scalar loads one after the other took 3 us */
    const hk_kv8_range mine = a.ranges[lane];
    const uint64_t begun = __builtin_amdgcn_ballot_w64(
        lane < a.count && mine.before <= blockIdx.x);
    const int last = __popcll(begun) - 1;
    const hk_kv8_range r = {
        (uint32_t)__builtin_amdgcn_readlane((int)mine.cache, last),
        (uint32_t)__builtin_amdgcn_readlane((int)mine.source, last),
        (uint32_t)__builtin_amdgcn_readlane((int)mine.rows, last),
        (uint32_t)__builtin_amdgcn_readlane((int)mine.before, last)};
    const uint32_t head = blockIdx.y, which = blockIdx.z;
    const uint32_t block = r.cache / HK_KV8_BLOCK + (blockIdx.x - r.before);
    /* rows [r0, r1) of the block are new, from row `from` on */
    const uint64_t row0 = (uint64_t)block * HK_KV8_BLOCK;
    const uint32_t r0 = r.cache > row0 ? (uint32_t)(r.cache - row0) : 0u;
    const uint64_t end = (uint64_t)r.cache + r.rows - row0;
    const uint32_t r1 = end < HK_KV8_BLOCK ? (uint32_t)end : HK_KV8_BLOCK;
    const uint64_t from = (uint64_t)r.source + (row0 + r0 - r.cache);
    const uint32_t part = HK_KV8_BLOCK * c.padded;
    const uint32_t pieces = part / 32u;
    const size_t at = (size_t)block * c.heads + head;
    const uint16_t *x = (which ? a.value : a.key) + from * a.stride +
                        (uint64_t)head * c.dim;
    float *scale = (float *)(c.scales + at) + which;
    const float old = r0 ? *scale : 0.0f;
    uint4 rows[PIECES][4];
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
        const hk_kv8_piece p(tid + k * 256u, c.padded);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t row = p.row + e;
            const bool has = row >= r0 && row < r1 && p.dim < c.dim;
            uint32_t w[4] = {};
            if (ALIGNED) {
                /* some new row's where it has none: no branch, behind which
                 * the loads would wait for each other */
                const uint4 v = *(const uint4 *)(
                    x + (min(max(row, r0), r1 - 1u) - r0) * a.stride +
                    min(p.dim, c.dim - 8u));
                w[0] = has ? v.x : 0u;
                w[1] = has ? v.y : 0u;
                w[2] = has ? v.z : 0u;
                w[3] = has ? v.w : 0u;
            } else if (has) {
                const uint16_t *y = x + (row - r0) * a.stride + p.dim;
#pragma unroll
                for (int d = 0; d < 8; d++)
                    if (p.dim + d < c.dim)
                        w[d >> 1] |= (uint32_t)y[d] << (16 * (d & 1));
            }
            rows[k][e] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < PIECES; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float f[8];
            hk_unpack8(rows[k][e], f);
#pragma unroll
            for (int d = 0; d < 8; d++) most = max(most, hk_magnitude(f[d]));
        }
    most = hk_block_umax(most, tops, 4u); /* (all have the old scale) */
    hk_int8_quantizer code(most);
    float keep = 1.0f;
    if (r0 && !(old < code.scale)) {
        /* the block's scale holds (also where it is NaN) */
        if (!isnan(code.scale))
            code = hk_int8_quantizer(hk_magnitude(127.0f * old));
        if (isnan(old)) code = hk_int8_quantizer(HK_NOT_FINITE);
        if (!isnan(code.scale)) code.scale = old;
    } else if (r0) {
        keep = old / code.scale;
    }
    if (tid == 0) *scale = code.scale;
    uint8_t *out = c.codes + (at * 2u + which) * part;
    /* (the same for the whole workgroup) */
    const bool few = r0 && !(keep < 1.0f);
    if (r0 && !few) {
        for (uint32_t u = tid; u < part / 16u; u += 256u) {
            const uint4 had = *(const uint4 *)(out + u * 16u);
            uint32_t w[4] = {had.x, had.y, had.z, had.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float f[4];
#pragma unroll
                for (int b = 0; b < 4; b++)
                    f[b] = rintf((float)((int)((w[j] >> (8 * b)) & 255u) -
                                         128) * keep) + 128.0f;
                w[j] = hk_int8_pack4(f[0], f[1], f[2], f[3]);
            }
            *(uint4 *)(image + hk_kv8_image(u * 16u)) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
    }
    auto put = [&](auto place) {
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            const hk_kv8_piece p(tid + k * 256u, c.padded);
            /* none of its rows are new, nor to be cleared */
            if (tid + k * 256u >= pieces ||
                (r0 && (p.row + 4u <= r0 || p.row >= r1)))
                continue;
            float f[4][8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                hk_unpack8(rows[k][e], f[e]);
#pragma unroll
                for (int d = 0; d < 8; d++) f[e][d] = code(f[e][d]) + 128.0f;
            }
            const bool all = !r0 || (p.row >= r0 && p.row + 4u <= r1);
            if (which == 0) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (all || (p.row + e >= r0 && p.row + e < r1))
                        *(uint2 *)place(
                            hk_kv8_key_at(p.row + e, p.dim, c.padded)) =
                            make_uint2(hk_int8_pack4(f[e][0], f[e][1], f[e][2],
                                                     f[e][3]),
                                       hk_int8_pack4(f[e][4], f[e][5], f[e][6],
                                                     f[e][7]));
                continue;
            }
#pragma unroll
            for (int d = 0; d < 8; d++) {
                uint8_t *word =
                    place(hk_kv8_value_at(p.row, p.dim + d, c.padded));
                const uint32_t w =
                    hk_int8_pack4(f[0][d], f[1][d], f[2][d], f[3][d]);
                if (all) {
                    *(uint32_t *)word = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (p.row + e >= r0 && p.row + e < r1)
                            word[e] = (uint8_t)(w >> (8 * e));
                }
            }
        }
    };
    if (few) {
        put([&](uint32_t byte) { return out + byte; });
        return;
    }
    put([&](uint32_t byte) { return image + hk_kv8_image(byte); });
    __syncthreads();
    for (uint32_t u = tid; u < part / 16u; u += 256u)
        *(uint4 *)(out + u * 16u) =
            *(const uint4 *)(image + hk_kv8_image(u * 16u));
}

/* Values of a block's keys or values (blockIdx.z) of a head, by way of the
 * block's image in LDS: the codes times `scale`, element d of row r at row(r) +
 * d, where row() is not NULL. */
template <bool F16, typename ROW>
__device__ __forceinline__ void hk_kv8_rows(const hk_kv8_cache &c, size_t at,
                                            uint32_t which, float scale,
                                            uint8_t *image, ROW row_of) {
    const uint32_t tid = threadIdx.x;
    const uint32_t part = HK_KV8_BLOCK * c.padded;
    const uint8_t *codes = c.codes + (at * 2u + which) * part;
    for (uint32_t u = tid; u < part / 16u; u += 256u)
        *(uint4 *)(image + hk_kv8_image(u * 16u)) =
            *(const uint4 *)(codes + u * 16u);
    __syncthreads();
    for (uint32_t k = tid; k < part / 32u; k += 256u) {
        const hk_kv8_piece p(k, c.padded);
        float f[4][8];
        auto value_of = [&](uint32_t word, int byte) {
            return ((float)((word >> (8 * byte)) & 255u) - 128.0f) * scale;
        };
        if (which == 0) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint2 w = *(const uint2 *)(
                    image +
                    hk_kv8_image(hk_kv8_key_at(p.row + e, p.dim, c.padded)));
#pragma unroll
                for (int d = 0; d < 8; d++)
                    f[e][d] = value_of(d < 4 ? w.x : w.y, d & 3);
            }
        } else {
#pragma unroll
            for (int d = 0; d < 8; d++) {
                const uint32_t w = *(const uint32_t *)(
                    image +
                    hk_kv8_image(hk_kv8_value_at(p.row, p.dim + d, c.padded)));
#pragma unroll
                for (int e = 0; e < 4; e++) f[e][d] = value_of(w, e);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint16_t *to = p.dim < c.dim ? row_of(p.row + e) : NULL;
            if (!to) continue;
            to += p.dim;
            if (F16 && which) { /* (dims in whole eights) */
                hk_f16x8 v;
#pragma unroll
                for (int d = 0; d < 8; d++) v[d] = (_Float16)f[e][d];
                *(hk_f16x8 *)to = v;
            } else if (c.dim % 8u == 0) {
                *(uint4 *)to = hk_pack8(f[e]);
            } else {
#pragma unroll
                for (int d = 0; d < 8; d++)
                    if (p.dim + d < c.dim) to[d] = hk_f2bf(f[e][d]);
            }
        }
    }
}

/* The values of rows [first, + rows): 889 of 40 heads of 128 in 7.0 us (3.9
 * TB/s). */
__global__ void __launch_bounds__(256)
hk_kv8_read(hk_kv8_cache c, uint16_t *key, uint16_t *value, uint32_t first,
            uint32_t rows) {
    extern __shared__ __attribute__((aligned(16))) uint8_t image[];
    const uint32_t block = first / HK_KV8_BLOCK + blockIdx.x;
    const uint32_t head = blockIdx.y, which = blockIdx.z;
    const size_t at = (size_t)block * c.heads + head;
    const uint64_t row0 = (uint64_t)block * HK_KV8_BLOCK;
    hk_kv8_rows<false>(c, at, which, ((const float *)(c.scales + at))[which],
                image, [&](uint32_t r) -> uint16_t * {
                    const uint64_t row = row0 + r;
                    if (row < first || row >= (uint64_t)first + rows)
                        return NULL;
                    return (which ? value : key) +
                           ((row - first) * c.heads + head) * c.dim;
                });
}

/* A plan's spans of blocks as rows, [block][64][keys, values][head][dim]: the
 * keys' codes, times their unit, as bf16, which holds them, and the values as
 * f16, divided by a power of two that leaves the span's largest in f16's range,
 * 2^15 at most, and rounded to 11 bits (those under 2^-29 of it to fewer).  889
 * rows of 40 heads of 128 in 9.4 us. */
__global__ void __launch_bounds__(256)
hk_kv8_unpack(hk_kv8_cache c, const hk_packed_span *spans, uint32_t count,
              uint16_t *out, float *units, uint32_t first) {
    __shared__ uint32_t tops[16];
    extern __shared__ __attribute__((aligned(16))) uint8_t image[];
    const uint32_t to = first + blockIdx.x;
    uint32_t low = 0, high = count; /* the last span that begins by then */
    while (high - low > 1u) {
        const uint32_t mid = (low + high) / 2u;
        if (spans[mid].at <= to) low = mid;
        else high = mid;
    }
    const hk_packed_span span = spans[low];
    const uint32_t block = span.block + (to - span.at);
    const uint32_t head = blockIdx.y, which = blockIdx.z;
    const uint64_t row0 = (uint64_t)to * HK_KV8_BLOCK;
    const size_t at = (size_t)block * c.heads + head;
    float scale;
    if (which == 0) {
        scale = hk_packed_code_unit(c.scales[at].x);
    } else {
        uint32_t most = 0;
        for (uint32_t i = threadIdx.x; i < span.blocks; i += 256u) {
            const uint32_t s = hk_magnitude(
                c.scales[((size_t)span.block + i) * c.heads + head].y);
            if (s < HK_NOT_FINITE) most = max(most, s);
        }
        most = hk_block_umax(most, tops, 4u);
        /* 127 scales over the unit are below 2^15 */
        const uint32_t exponent = max(most >> 23, 8u) - 7u;
        if (to == span.at && threadIdx.x == 0)
            units[(size_t)to * c.heads + head] =
                __uint_as_float(exponent << 23);
        scale = c.scales[at].y * __uint_as_float((254u - exponent) << 23);
    }
    hk_kv8_rows<true>(c, at, which, scale, image,
                      [&](uint32_t r) -> uint16_t * {
                          return out + (((row0 + r) * 2u + which) * c.heads +
                                        head) * c.dim;
                      });
}

/* ---------------------------------------------------------- the attention */

__device__ __forceinline__ float hk_kv8_key(const hk_kv8_cache &c,
                                            const uint8_t *codes, uint32_t row,
                                            uint32_t dim) {
    return (float)((int)codes[hk_kv8_key_at(row, dim, c.padded)] - 128);
}

__device__ __forceinline__ float hk_kv8_value(const hk_kv8_cache &c,
                                              const uint8_t *codes,
                                              uint32_t row, uint32_t dim) {
    return (float)((int)codes[HK_KV8_BLOCK * c.padded +
                              hk_kv8_value_at(row, dim, c.padded)] -
                   128);
}

struct hk_kv8_args {
    hk_packed_args p;
    hk_kv8_cache cache;
};

/* One wave per query row and head, 64 keys (a block) a turn, as
 * hk_packed_simple: H3_HIP_REFERENCE=1 and heads over 128. */
__device__ void hk_kv8_simple_row(const hk_kv8_args &g, uint32_t nth,
                                  uint32_t head) {
    const hk_packed_args &a = g.p;
    const hk_kv8_cache &c = g.cache;
    const uint32_t lane = threadIdx.x & 63u;
    const hk_packed_request r =
        a.requests[hk_packed_request_of(a.requests, a.request_count, nth)];
    const uint32_t row = r.q_first + (nth - r.before);
    const uint32_t kv_head = head / a.group;
    const uint16_t *q = a.q + row * a.q_stride + (uint64_t)head * a.dim;
    float top = -INFINITY, sum = 0.0f;
    float o[HK_PACKED_MAX_DIM / 64];
    for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++) o[d] = 0.0f;
    for (uint32_t j0 = 0; j0 < r.kv_rows; j0 += HK_KV8_BLOCK) {
        const uint32_t left = min(HK_KV8_BLOCK, r.kv_rows - j0);
        const size_t at =
            (size_t)((r.kv_first + j0) / HK_KV8_BLOCK) * c.heads + kv_head;
        const uint8_t *codes = c.codes + at * 2u * HK_KV8_BLOCK * c.padded;
        const float2 scale = c.scales[at];
        const float unit = hk_packed_code_unit(scale.x);
        float s = -INFINITY;
        if (lane < left) {
            s = 0.0f;
            for (uint32_t d = 0; d < a.dim; d++)
                s = fmaf(hk_bf2f(q[d]),
                         unit * hk_kv8_key(c, codes, lane, d), s);
            s *= hk_packed_code_scale(scale.x);
        }
        const float most = fmaxf(top, hk_wave_max(s));
        /* every score so far -inf: no weights yet */
        const float ref = most == -INFINITY ? 0.0f : most;
        const float keep =
            top == -INFINITY ? 0.0f : expf((top - ref) * a.scale);
        const float p = lane < left ? expf((s - ref) * a.scale) : 0.0f;
        top = most;
        sum = sum * keep + hk_wave_sum(p);
        for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++) o[d] *= keep;
        for (uint32_t j = 0; j < left; j++) {
            const float pj = __shfl(p, j, 64) * scale.y;
            for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++)
                if (d * 64u + lane < a.dim)
                    o[d] = fmaf(
                        pj, hk_kv8_value(c, codes, j, d * 64u + lane), o[d]);
        }
    }
    uint16_t *out = a.o + ((uint64_t)row * a.heads + head) * a.dim;
    for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++)
        if (d * 64u + lane < a.dim)
            out[d * 64u + lane] = hk_f2bf(sum == 0.0f ? 0.0f : o[d] / sum);
}

__global__ void __launch_bounds__(256) hk_kv8_simple(hk_kv8_args g) {
    for (uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
         i < (uint64_t)g.p.rows * g.p.heads; i += (uint64_t)gridDim.x * 4u) {
        const uint32_t nth = (uint32_t)(i / g.p.heads);
        hk_kv8_simple_row(g, nth,
                          (uint32_t)(i - (uint64_t)nth * g.p.heads));
    }
}

/* -------------------------------------------- few rows on the matrix cores
 *
 * The plan's items of at most 32 rows (hk_packed.h), 32 keys a step: S^T = K .
 * Q^T, the softmax in the lanes that hold a query's scores, O^T = V^T . P^T.
 * Codes and P are f16, which holds codes exactly and is made of them in two
 * instructions a pair.  A query row is scaled by a power of two of its own to
 * f16's range, which loses nothing of a bf16 within 2^27 of the row's largest;
 * that and the block's key scale go into the factor of the exponent.  The
 * product with the values is multiplied by their scale as it is added to O.
 *
 * P = 2^((s - m) L + 7) against a reference m (a score, L = scale log2(e)) that
 * moves when a lane's sum of P passes 2^15: so f16 holds every P, to 11 bits
 * those over 2^-21 of the largest; the factor 2^7 is in the sums too. */
typedef _Float16 hk_f16x2 __attribute__((ext_vector_type(2)));

#define HK_KV8_LIFT 7.0f
#define HK_KV8_MOST 0x1p15f

/* Four codes (+ 128) as f16: byte b is the low byte of 1024 + b. */
__device__ __forceinline__ uint2 hk_kv8_f16(uint32_t codes) {
    const hk_f16x2 less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const hk_f16x2 low =
        __builtin_bit_cast(hk_f16x2, __builtin_amdgcn_perm(
                                         0x64646464u, codes, 0x04010400u)) +
        less;
    const hk_f16x2 high =
        __builtin_bit_cast(hk_f16x2, __builtin_amdgcn_perm(
                                         0x64646464u, codes, 0x04030402u)) +
        less;
    return make_uint2(__builtin_bit_cast(uint32_t, low),
                      __builtin_bit_cast(uint32_t, high));
}

/* A lane's 16 bytes as two fragments of 8. */
__device__ __forceinline__ void hk_kv8_fragments(uint4 codes, uint4 (&f)[2]) {
    const uint2 a = hk_kv8_f16(codes.x), b = hk_kv8_f16(codes.y);
    const uint2 c = hk_kv8_f16(codes.z), d = hk_kv8_f16(codes.w);
    f[0] = make_uint4(a.x, a.y, b.x, b.y);
    f[1] = make_uint4(c.x, c.y, d.x, d.y);
}

__device__ __forceinline__ hk_f32x16 hk_kv8_mfma(uint4 a, hk_f16x8 b,
                                                 hk_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(hk_f16x8, a), b, c, 0, 0, 0);
}

/* Whether -(m L) is far from zero, infinite or NaN (hk_packed.hip). */
__device__ __forceinline__ bool hk_kv8_far(float neg) {
    return !(fabsf(neg) < 0x1p10f);
}

/* A wave's 32 virtual rows, lane % 32, and what it has of their sums. */
template <int DIMS> struct hk_kv8_wave {
    static constexpr int NK = DIMS / 16, ND = DIMS / 32;
    hk_f16x8 q[NK];   /* dims 32 (k / 2) + 16 half + 8 (k % 2) .. + 8 */
    float q_scale;    /* of the row */
    hk_f32x16 o[ND];
    float m, neg;     /* the reference, -(m L); unset: -+ infinity */
    float l;

    /* Its query row, zeros where there is none.  Whole pieces are loaded
     * without a branch, behind which each would wait for the one before. */
    __device__ __forceinline__ void load(const hk_packed_args &a,
                                         const hk_packed_item &it,
                                         uint32_t vrow, uint4 (&raw)[NK]) {
        const uint32_t half = (threadIdx.x & 63u) >> 5;
        const uint32_t of = min(vrow, it.rows - 1u);
        const uint32_t r = of / a.group, g = of - r * a.group;
        const uint16_t *row =
            a.q + ((uint64_t)it.q_first + r) * a.q_stride +
            (uint64_t)(it.kv_head * a.group + g) * a.dim;
        if (a.dim % 8u == 0 && a.q_stride % 8u == 0 &&
            ((uintptr_t)a.q & 15u) == 0) {
#pragma unroll
            for (int k = 0; k < NK; k++)
                raw[k] = *(const uint4 *)(
                    row + min((k >> 1) * 32u + half * 16u + (k & 1) * 8u,
                              a.dim - 8u));
        } else {
#pragma unroll
            for (int k = 0; k < NK; k++) {
                uint32_t w[4] = {};
#pragma unroll
                for (uint32_t e = 0; e < 8u; e++) {
                    const uint32_t d =
                        (k >> 1) * 32u + half * 16u + (k & 1) * 8u + e;
                    if (d < a.dim) w[e >> 1] |= (uint32_t)row[d] << (16 * (e & 1));
                }
                raw[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }

    __device__ __forceinline__ void start(const hk_packed_args &a,
                                          const hk_packed_item &it,
                                          uint32_t vrow,
                                          const uint4 (&raw)[NK]) {
        const uint32_t half = (threadIdx.x & 63u) >> 5;
        float x[NK][8];
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const uint32_t d = (k >> 1) * 32u + half * 16u + (k & 1) * 8u;
            const bool has = vrow < it.rows && d < a.dim;
            hk_unpack8(raw[k], x[k]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[k][e] = has ? x[k][e] : 0.0f;
                most = max(most, hk_magnitude(x[k][e]));
            }
        }
        most = max(most, (uint32_t)__shfl_xor(most, 32, 64));
        /* to [2^13, 2^14) */
        const int by = 13 + 127 - (int)(most >> 23);
        q_scale = ldexpf(1.0f, -by);
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                q[k][e] = (_Float16)ldexpf(x[k][e], by);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
        m = -INFINITY;
        neg = INFINITY;
        l = 0.0f;
    }

    /* Raw scores (products with the codes) to P; `keys` of the step's count. */
    __device__ __forceinline__ void softmax(hk_f32x16 &s, hk_f16x8 (&p)[2],
                                            float scale, uint32_t keys,
                                            float L) {
        const uint32_t half = (threadIdx.x & 63u) >> 5;
        /* a row or block of zeros: scores of 0, whatever multiplies them, and
         * -inf stays -inf */
        float by = q_scale * scale;
        if (by == 0.0f) by = 0x1p-100f;
        float own = by * L;
        if (own == 0.0f) own = 0x1p-126f;
        if (keys < 32u) {
            asm volatile(""); /* a branch, not 16 selects in every step */
#pragma unroll
            for (int r = 0; r < 16; r++)
                if ((r >> 2) * 8u + half * 4u + (r & 3) >= keys)
                    s[r] = -INFINITY;
        }
        auto exps = [&](float less) -> float {
            float sum = 0.0f;
            less += HK_KV8_LIFT;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float e = __builtin_amdgcn_exp2f(
                    __builtin_fmaf(s[r], own, less));
                sum += e;
                p[r >> 3][r & 7] = (_Float16)e;
            }
            return sum;
        };
        const bool far = hk_kv8_far(neg); /* or unset */
        float sum = far ? 0.0f : exps(neg);
        /* (a NaN sum stays) */
        uint32_t move = far || sum > HK_KV8_MOST;
        if (__builtin_amdgcn_ballot_w64(move)) {
            /* a row's other half's too, but no other row's */
            const auto both =
                __builtin_amdgcn_permlane32_swap(move, move, false, false);
            move = both[0] | both[1];
            float mx = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[r]);
            mx *= by;
            const auto sw = __builtin_amdgcn_permlane32_swap(
                __float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            const float now = move ? fmaxf(m, mx) : m;
            const float ref = now == -INFINITY ? 0.0f : now;
            const float c =
                move ? __builtin_amdgcn_exp2f((m - ref) * L) : 1.0f;
            m = now; /* unset while every score is -inf */
            neg = -(now * L);
            float less = -(ref * L);
            if (__builtin_amdgcn_ballot_w64(hk_kv8_far(less))) {
                /* this row's scores as they are, rounded as the reference was,
                 * and the reference off them first, which is exact near it */
                const bool apart = hk_kv8_far(less);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float x = s[r] * by;
                    asm volatile("" : "+v"(x)); /* no fused add */
                    s[r] = apart ? x - ref : s[r];
                }
                if (apart) {
                    own = L;
                    less = 0.0f;
                }
            }
            l *= c;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= c;
            sum = exps(less);
        }
        l += sum;
    }

    /* o += scale * the step's product, two groups of 32 dims at a time */
    __device__ __forceinline__ void values(const hk_f16x8 (&p)[2], float scale,
                                           const uint4 (&codes)[ND]) {
#pragma unroll
        for (int d0 = 0; d0 < ND; d0 += 2) {
            hk_f32x16 t[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (d0 + i >= ND) continue;
#pragma unroll
                for (int r = 0; r < 16; r++) t[i][r] = 0.0f;
                uint4 f[2];
                hk_kv8_fragments(codes[d0 + i], f);
                t[i] = hk_kv8_mfma(f[0], p[0], t[i]);
                t[i] = hk_kv8_mfma(f[1], p[1], t[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (d0 + i < ND)
                        o[d0 + i][r] = __builtin_fmaf(t[i][r], scale,
                                                      o[d0 + i][r]);
        }
    }
};

/* Eight dims of an output row. */
__device__ __forceinline__ void hk_kv8_put(const hk_packed_args &a,
                                           const hk_packed_item &it,
                                           uint32_t vrow, uint32_t dim,
                                           const float *v, bool whole) {
    const uint32_t r = vrow / a.group, g = vrow - r * a.group;
    uint16_t *to = a.o + (((uint64_t)it.q_first + r) * a.heads +
                          it.kv_head * a.group + g) * a.dim + dim;
    if (whole) {
        if (dim < a.dim) *(uint4 *)to = hk_pack8(v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (dim + e < a.dim) to[e] = hk_f2bf(v[e]);
}

/* The waves share the item's rows and split its keys, wave w every fourth 32 of
 * them from the wth on, straight from the cache into its registers; then their
 * sums are joined, 64 dims at a time.  Long contexts are bound by the cache's
 * bytes (8 rows of 64 heads over 8, 4096 to 9720 keys: 21 us, 5.5 TB/s), short
 * ones by the chain of item, keys, scores and join (16 rows of 40 heads, 20 to
 * 512 keys: 11 us).  32 keys a step and 32 KB of LDS let three workgroups share a
 * CU: 640 items of 300 keys 14.0 us; 64 a step leave room for two, 21. */
template <int DIMS>
__global__ void __launch_bounds__(256, 3) hk_kv8_few(hk_kv8_args g) {
    constexpr int ND = DIMS / 32;
    constexpr int DP = DIMS <= 64 ? 64 : 128;
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_lds[];
    float *lds = (float *)hk_lds;
    const hk_packed_args &a = g.p;
    hk_packed_item it = a.items[blockIdx.x];
    if (it.row >= it.rows || it.rows - it.row > 32u) return;
    if (!a.part_o && it.part != HK_PACKED_WHOLE) {
        /* no room for pieces' sums: the first one takes all keys */
        if (it.tile) return;
        it.tile_end = (it.kv_rows + HK_KV8_BLOCK - 1u) / HK_KV8_BLOCK;
        it.part = HK_PACKED_WHOLE;
    }
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 31u, half = lane >> 5;
    const uint32_t vrow = it.row + col;
    const uint32_t first = it.kv_first / HK_KV8_BLOCK;
    /* steps of 32 keys, two a block */
    auto block_at = [&](uint32_t step) {
        return (size_t)(first + (step >> 1)) * g.cache.heads + it.kv_head;
    };
    uint4 k[ND], v[ND];
    auto load = [&](uint32_t step, int which, uint4 (&to)[ND]) {
        const uint4 *from =
            (const uint4 *)(g.cache.codes +
                            ((block_at(step) * 2u + which) * 2u + (step & 1u)) *
                                (32u * DIMS)) +
            lane;
#pragma unroll
        for (int u = 0; u < ND; u++) to[u] = from[u * 64];
    };
    const uint32_t last =
        min(it.tile_end * 2u, (it.kv_rows + 31u) / 32u); /* (below 2^28) */
    uint32_t step = it.tile * 2u + wave;
    float2 ahead = make_float2(0.0f, 0.0f);
    hk_kv8_wave<DIMS> w;
    uint4 raw[DIMS / 16];
    w.load(a, it, vrow, raw);
    if (step < last) {
        ahead = g.cache.scales[block_at(step)];
        load(step, 0, k);
        load(step, 1, v);
    }
    w.start(a, it, vrow, raw);
    /* the queries, the same for all waves, wait in LDS */
    hk_f16x8 *queries = (hk_f16x8 *)lds + lane;
    if (wave == 0) {
#pragma unroll
        for (int i = 0; i < DIMS / 16; i++) queries[i * 64] = w.q[i];
    }
    __syncthreads();
    for (; step < last; step += HK_PACKED_WAVES) {
        const float2 scale = ahead;
        /* past the last step, that one again, which no one uses */
        const uint32_t next =
            step + HK_PACKED_WAVES < last ? step + HK_PACKED_WAVES : step;
        hk_f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < ND; j++) {
            uint4 f[2];
            hk_kv8_fragments(k[j], f);
            s = hk_kv8_mfma(f[0], queries[2 * j * 64], s);
            s = hk_kv8_mfma(f[1], queries[(2 * j + 1) * 64], s);
        }
        ahead = g.cache.scales[block_at(next)];
        load(next, 0, k);
        hk_f16x8 p[2];
        w.softmax(s, p, scale.x, it.kv_rows - step * 32u, a.scale_log2);
        w.values(p, scale.y, v);
        load(next, 1, v);
    }
    /* references and sums of each row, then O scaled to the common reference
     * (and by 1 / L for a whole item) */
    __syncthreads();
    float2 *ml = (float2 *)lds;
    const float own = w.l + __shfl_xor(w.l, 32, 64);
    if (half == 0) ml[wave * 32u + col] = make_float2(w.m, own);
    __syncthreads();
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < HK_PACKED_WAVES; i++)
        top = fmaxf(top, ml[i * 32u + col].x);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (uint32_t i = 0; i < HK_PACKED_WAVES; i++) {
        const float2 x = ml[i * 32u + col];
        l += __builtin_amdgcn_exp2f((x.x - ref) * a.scale_log2) * x.y;
    }
    const bool all = it.part == HK_PACKED_WHOLE;
    float weight = __builtin_amdgcn_exp2f((w.m - ref) * a.scale_log2);
    if (all) weight *= l == 0.0f ? 0.0f : 1.0f / l;
    else if (wave == 0 && half == 0 && vrow < it.rows)
        a.part_ml[(size_t)it.part * HK_PACKED_QB + col] = make_float2(top, l);
    const bool whole = a.dim % 8u == 0;
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += 2) {
        /* rows of 64 F32 a wave, 16-byte chunk c of row r at c ^ (r % 16) */
        __syncthreads();
#pragma unroll
        for (int d = 0; d < 2; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (d0 + d >= ND) continue;
                const uint32_t c = d * 8u + i * 2u + half;
                const hk_f32x16 &o = w.o[d0 + d];
                *(float4 *)(lds + wave * 2048u + col * 64u +
                            ((c ^ (col & 15u)) << 2)) =
                    make_float4(o[i * 4] * weight, o[i * 4 + 1] * weight,
                                o[i * 4 + 2] * weight, o[i * 4 + 3] * weight);
            }
        __syncthreads();
        const uint32_t r = tid >> 3, c = (tid & 7u) * 2u;
        const uint32_t dim = d0 * 32u + c * 4u;
        if (it.row + r >= it.rows || dim >= DIMS) continue;
        hk_f32x4 sum[2] = {};
#pragma unroll
        for (uint32_t i = 0; i < HK_PACKED_WAVES; i++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                sum[e] += *(const hk_f32x4 *)(lds + i * 2048u + r * 64u +
                                              (((c + e) ^ (r & 15u)) << 2));
        if (all) {
            const float y[8] = {sum[0][0], sum[0][1], sum[0][2], sum[0][3],
                                sum[1][0], sum[1][1], sum[1][2], sum[1][3]};
            hk_kv8_put(a, it, it.row + r, dim, y, whole);
            continue;
        }
        float *part =
            a.part_o + ((size_t)it.part * HK_PACKED_QB + r) * DP + dim;
        *(hk_f32x4 *)part = sum[0];
        *(hk_f32x4 *)(part + 4) = sum[1];
    }
}

template <int DIMS>
static void hk_kv8_launch_few(struct h3_gpu *gpu, const hk_kv8_args &g,
                              const uint32_t *n) {
    const uint32_t lds = 4u * 32u * 64u * 4u; /* 64 dims of the waves' O */
    const uint32_t most = 1u << 23; /* below 2^32 threads, turns of the XCDs */
    for (uint32_t first = 0; first < n[HK_PACKED_ITEMS]; first += most) {
        hk_kv8_args part = g;
        part.p.items += first;
        hipLaunchKernelGGL(hk_kv8_few<DIMS>,
                           dim3(std::min(n[HK_PACKED_ITEMS] - first, most)),
                           dim3(256), lds, gpu->stream, part);
    }
}

/* Unpacks the blocks that items of many rows read, for the kernel over rows
 * (hk_packed_codes): once a call, where each item would do it again.  The
 * kernel over rows is bound by the sum of its products and its vector
 * instructions, and making f16 of codes and scaling each block's product added
 * an eighth to those.  The values' scales are in the rows: on P they would round
 * alike for all keys of a block, on the sums cost the multiplications. */
static void hk_kv8_many(struct h3_gpu *gpu, const hk_kv8_args &g,
                        const uint32_t *n, uint16_t *rows, float *units) {
    const hk_kv8_cache &c = g.cache;
    const size_t width = (size_t)c.heads * c.dim;
    const uint32_t blocks = n[HK_PACKED_SPAN_BLOCKS];
    hk_packed_args a = g.p;
    if (blocks) {
        const uint32_t most = std::max(1u, (1u << 22) / c.heads);
        for (uint32_t first = 0; first < blocks; first += most)
            hipLaunchKernelGGL(
                hk_kv8_unpack, dim3(std::min(blocks - first, most), c.heads, 2),
                dim3(256), HK_KV8_BLOCK * c.padded, gpu->stream, c, a.spans,
                n[HK_PACKED_SPANS], rows, units, first);
        a.k = rows;
        a.v = rows + width;
    }
    a.kv_stride = 2u * width;
    a.key_scales = (const float *)c.scales;
    a.value_units = units;
    hk_packed_many_scaled(gpu, a, n);
}

/* ================================================================ ops */

static int hk_kv8_require(struct h3_gpu *gpu, const h3_gpu_tensor *t) {
    if (!t || t->record.kind != HK_RECORD_KV8)
        return hk_fail(gpu, "the cache was not made by h3_hip_kv_int8_new");
    return 1;
}

extern "C" {

h3_gpu_tensor *h3_hip_kv_int8_new(h3_gpu *gpu, uint32_t rows,
                                  uint32_t kv_heads, uint32_t head_dim) {
    if (!gpu) return NULL;
    if (!rows || rows > UINT32_MAX - HK_KV8_BLOCK || !kv_heads ||
        kv_heads > 65535u || !head_dim || head_dim > HK_PACKED_MAX_DIM) {
        hk_fail(gpu, "8-bit cache of %u rows, %u heads of %u (1 to 2^32 - 65 "
                     "rows, 1 to 65535 heads of 1 to %u)", rows, kv_heads,
                head_dim, HK_PACKED_MAX_DIM);
        return NULL;
    }
    const uint32_t blocks = (rows + HK_KV8_BLOCK - 1u) / HK_KV8_BLOCK;
    /* at most 2^26 blocks x 2^16 heads x 2^15 bytes */
    const size_t pairs = (size_t)blocks * kv_heads;
    h3_gpu_tensor *t = h3_gpu_tensor_new_i8(
        gpu, pairs * (2u * HK_KV8_BLOCK * hk_kv8_padded(head_dim) +
                      sizeof(float2)));
    if (!t) return NULL;
    t->record.kind = HK_RECORD_KV8;
    t->record.n[HK_KV8_BLOCKS] = blocks;
    t->record.n[HK_KV8_HEADS] = kv_heads;
    t->record.n[HK_KV8_DIM] = head_dim;
    /* launches of up to 2^31 threads */
    float2 *scales = hk_kv8_of(t).scales;
    for (size_t first = 0; first < pairs; first += (size_t)1 << 31) {
        const size_t n = std::min(pairs - first, (size_t)1 << 31);
        hipLaunchKernelGGL(hk_kv8_clear, dim3((unsigned)((n + 255u) / 256u)),
                           dim3(256), 0, gpu->stream, scales + first, n);
    }
    const hipError_t status = hipGetLastError();
    if (status != hipSuccess) {
        hk_fail_hip(gpu, "8-bit cache", status);
        h3_gpu_tensor_free(t);
        return NULL;
    }
    return t;
}

int h3_hip_kv_int8_store(h3_gpu *gpu, h3_gpu_tensor *cache,
                         const uint32_t *cache_first,
                         const uint32_t *source_first, const uint32_t *rows,
                         uint32_t count, const h3_gpu_tensor *key,
                         size_t key_offset, const h3_gpu_tensor *value,
                         size_t value_offset, uint32_t kv_stride) {
    if (!hk_kv8_require(gpu, cache)) return 0;
    if (count && (!cache_first || !source_first || !rows))
        return hk_fail(gpu, "cache store: no ranges");
    const hk_kv8_cache c = hk_kv8_of(cache);
    const uint64_t width = (uint64_t)c.heads * c.dim;
    if (kv_stride < width)
        return hk_fail(gpu, "cache store: a row stride of %u is under the "
                            "rows' %llu elements", kv_stride,
                       (unsigned long long)width);
    std::vector<hk_kv8_range> ranges;
    uint64_t source_end = 0;
    try {
        std::vector<std::pair<uint32_t, uint32_t>> blocks;
        for (uint32_t i = 0; i < count; i++) {
            if (!rows[i]) continue;
            const uint64_t end = (uint64_t)cache_first[i] + rows[i];
            if (end > (uint64_t)c.blocks * HK_KV8_BLOCK)
                return hk_fail(gpu, "cache store: range %u ends behind the "
                                    "cache's %u blocks of 64 rows", i,
                               c.blocks);
            source_end = std::max(source_end,
                                  (uint64_t)source_first[i] + rows[i]);
            ranges.push_back({cache_first[i], source_first[i], rows[i], 0});
            blocks.push_back({cache_first[i] / HK_KV8_BLOCK,
                              (uint32_t)((end - 1) / HK_KV8_BLOCK)});
        }
        std::sort(blocks.begin(), blocks.end());
        for (size_t i = 1; i < blocks.size(); i++)
            if (blocks[i].first <= blocks[i - 1].second)
                return hk_fail(gpu, "cache store: two ranges write rows of "
                                    "block %u", blocks[i].first);
    } catch (const std::bad_alloc &) {
        return hk_fail(gpu, "out of host memory");
    }
    if (!hk_require(gpu, key, hk_packed_extent(key_offset, kv_stride,
                                               source_end, width),
                    H3_GPU_BF16, "cache store key") ||
        !hk_require(gpu, value, hk_packed_extent(value_offset, kv_stride,
                                                 source_end, width),
                    H3_GPU_BF16, "cache store value") ||
        !hk_require_active(gpu))
        return 0;
    if (ranges.empty()) return 1;
    hk_op_begin(gpu, "kv_int8_store");
    hk_kv8_store_args a = {};
    a.cache = c;
    a.key = HK_CBF16(key) + key_offset;
    a.value = HK_CBF16(value) + value_offset;
    a.stride = kv_stride;
    /* launches of up to 64 ranges and 2^22 / heads blocks */
    const uint32_t most = std::max(1u, (1u << 22) / c.heads);
    uint32_t total = 0;
    const bool aligned = c.dim % 8u == 0 && kv_stride % 8u == 0 &&
                         (((uintptr_t)a.key | (uintptr_t)a.value) & 15u) == 0;
    auto kernel = c.padded > 128u
                      ? aligned ? hk_kv8_store<2, true> : hk_kv8_store<2, false>
                  : aligned ? hk_kv8_store<1, true>
                            : hk_kv8_store<1, false>;
    auto launch = [&]() {
        if (a.count)
            hipLaunchKernelGGL(kernel, dim3(total, c.heads, 2), dim3(256),
                               HK_KV8_BLOCK * c.padded, gpu->stream, a);
        a.count = total = 0;
    };
    for (hk_kv8_range r : ranges) {
        while (r.rows) {
            if (a.count == HK_KV8_RANGES || total == most) launch();
            /* as many of its rows as end with the launch's last block */
            const uint32_t begun = r.cache % HK_KV8_BLOCK;
            const uint64_t room =
                (uint64_t)(most - total) * HK_KV8_BLOCK - begun;
            const uint32_t n = (uint32_t)std::min<uint64_t>(r.rows, room);
            a.ranges[a.count++] = {r.cache, r.source, n, total};
            total += (begun + n + HK_KV8_BLOCK - 1u) / HK_KV8_BLOCK;
            r.cache += n;
            r.source += n;
            r.rows -= n;
        }
    }
    launch();
    return hk_op_end(gpu, "kv_int8_store", HK_KIND_DIRECT);
}

int h3_hip_kv_int8_read(h3_gpu *gpu, h3_gpu_tensor *key, h3_gpu_tensor *value,
                        const h3_gpu_tensor *cache, uint32_t first_row,
                        uint32_t rows) {
    if (!hk_kv8_require(gpu, cache)) return 0;
    const hk_kv8_cache c = hk_kv8_of(cache);
    if ((uint64_t)first_row + rows > (uint64_t)c.blocks * HK_KV8_BLOCK)
        return hk_fail(gpu, "cache read: the rows end behind the cache's %u "
                            "blocks of 64", c.blocks);
    const size_t width = (size_t)c.heads * c.dim;
    if (!hk_require(gpu, key, rows * width, H3_GPU_BF16, "cache read key") ||
        !hk_require(gpu, value, rows * width, H3_GPU_BF16,
                    "cache read value") ||
        !hk_require_active(gpu))
        return 0;
    if (key == value)
        return hk_fail(gpu, "cache read: keys and values need a tensor each");
    if (!rows) return 1;
    hk_op_begin(gpu, "kv_int8_read");
    const size_t most = std::max(1u, (1u << 22) / c.heads) * HK_KV8_BLOCK;
    for (uint64_t done = 0; done < rows;) {
        const uint32_t at = (uint32_t)(first_row + done);
        const uint32_t n = (uint32_t)std::min<uint64_t>(
            rows - done, most - at % HK_KV8_BLOCK);
        hipLaunchKernelGGL(
            hk_kv8_read,
            dim3((at % HK_KV8_BLOCK + n + HK_KV8_BLOCK - 1u) / HK_KV8_BLOCK,
                 c.heads, 2),
            dim3(256), HK_KV8_BLOCK * c.padded, gpu->stream, c,
            HK_BF16(key) + done * width,
            HK_BF16(value) + done * width, at, n);
        done += n;
    }
    return hk_op_end(gpu, "kv_int8_read", HK_KIND_DIRECT);
}

int h3_hip_sdpa_packed_int8_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                                 const h3_gpu_tensor *query,
                                 size_t query_offset, uint32_t query_stride,
                                 const h3_gpu_tensor *cache,
                                 const h3_gpu_tensor *plan, float scale) {
    if (!hk_kv8_require(gpu, cache)) return 0;
    if (!plan || plan->record.kind != HK_RECORD_PACKED)
        return hk_fail(gpu, "packed attention: the plan was not built by "
                            "h3_hip_sdpa_packed_plan");
    const uint32_t *n = plan->record.n;
    hk_kv8_args a = {};
    a.cache = hk_kv8_of(cache);
    hk_packed_of_plan(a.p, plan, scale);
    if (a.p.kv_heads != a.cache.heads || a.p.dim != a.cache.dim)
        return hk_fail(gpu, "packed attention: %u key heads of %u in the plan, "
                            "%u of %u in the cache", a.p.kv_heads, a.p.dim,
                       a.cache.heads, a.cache.dim);
    if (n[HK_PACKED_OFF_BLOCKS])
        return hk_fail(gpu, "packed attention: a request's rows of the cache "
                            "do not begin at a multiple of 64");
    if (n[HK_PACKED_SPAN_BLOCKS] == HK_PACKED_TOO_MANY)
        return hk_fail(gpu, "packed attention: over 2^32 rows of the cache to "
                            "unpack");
    if (n[HK_PACKED_KV_END] > (uint64_t)a.cache.blocks * HK_KV8_BLOCK)
        return hk_fail(gpu, "packed attention: the plan's %u key rows end "
                            "behind the cache's %u blocks of 64",
                       n[HK_PACKED_KV_END], a.cache.blocks);
    const uint64_t q_width = (uint64_t)a.p.heads * a.p.dim;
    if (query_stride < q_width)
        return hk_fail(gpu, "packed attention: a row stride of %u is under "
                            "the rows' %llu elements", query_stride,
                       (unsigned long long)q_width);
    if (!isfinite(scale) || scale < 0.0f)
        return hk_fail(gpu, "packed attention: the scale must be finite and "
                            "not negative");
    if (!hk_require(gpu, query,
                    hk_packed_extent(query_offset, query_stride,
                                     n[HK_PACKED_Q_END], q_width),
                    H3_GPU_BF16, "packed query") ||
        !hk_require(gpu, output, n[HK_PACKED_Q_END] * q_width, H3_GPU_BF16,
                    "packed output") ||
        !hk_require_active(gpu))
        return 0;
    if (output == query)
        return hk_fail(gpu, "packed attention: the output must be a tensor "
                            "of its own");
    if (!n[HK_PACKED_ROWS]) return 1;
    a.p.q = HK_CBF16(query) + query_offset;
    a.p.o = HK_BF16(output);
    a.p.q_stride = query_stride;
    /* few rows: any head of up to 128; many: what the kernel over rows takes.
     * (A scale of 0 times -inf, what keys past the end are set to, is no
     * -inf.) */
    a.p.kv_stride = 2u * (uint64_t)a.cache.heads * a.cache.dim;
    const bool fast = !gpu->reference_kernels && a.p.dim <= 128u &&
                      a.p.scale_log2 > 0x1p-100f && isfinite(a.p.scale_log2) &&
                      (!n[HK_PACKED_MANY] || hk_packed_takes(gpu, a.p));
    uint16_t *unpacked = NULL;
    float *units = NULL;
    if (fast && n[HK_PACKED_SPAN_BLOCKS]) {
        const size_t heads = (size_t)n[HK_PACKED_SPAN_BLOCKS] * a.cache.heads;
        const size_t elements = heads * HK_KV8_BLOCK * 2u * a.cache.dim;
        unpacked = (uint16_t *)hk_workspace(
            gpu, elements * sizeof(uint16_t) + heads * sizeof(float));
        if (!unpacked) return 0;
        units = (float *)(unpacked + elements);
    }
    hk_op_begin(gpu, "attention_packed_int8");
    if (fast) {
        const uint32_t padded = a.p.dim <= 64u ? 64u : 128u;
        const size_t rows = (size_t)n[HK_PACKED_PARTS] * HK_PACKED_QB;
        if (rows)
            a.p.part_o = (float *)hk_splitk_try(
                gpu, rows * (padded * sizeof(float) + sizeof(float2)));
        /* without scratch, items run whole */
        if (a.p.part_o) a.p.part_ml = (float2 *)(a.p.part_o + rows * padded);
        if (n[HK_PACKED_MANY]) hk_kv8_many(gpu, a, n, unpacked, units);
        if (n[HK_PACKED_FEW]) switch (a.cache.padded) {
            case 32: hk_kv8_launch_few<32>(gpu, a, n); break;
            case 64: hk_kv8_launch_few<64>(gpu, a, n); break;
            case 96: hk_kv8_launch_few<96>(gpu, a, n); break;
            default: hk_kv8_launch_few<128>(gpu, a, n);
            }
        if (a.p.part_o) hk_packed_join_pieces(gpu, a.p, n, padded);
        return hk_op_end(gpu, "attention_packed_int8", HK_KIND_SDPA);
    }
    const uint64_t blocks = ((uint64_t)a.p.rows * a.p.heads + 3) / 4;
    hipLaunchKernelGGL(
        hk_kv8_simple,
        dim3((unsigned)(blocks < 1u << 20 ? blocks : 1u << 20)), dim3(256), 0,
        gpu->stream, a);
    return hk_op_end(gpu, "attention_packed_int8", HK_KIND_SDPA);
}

} /* extern "C" */
