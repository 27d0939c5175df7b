/* Attention of several requests packed in one call (h3_hip_sdpa_packed_plan /
 * _bf16 in h3_hip.h): query row r of request i, head h,
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j),
 * over request i's key rows j and key head h / (heads / kv_heads).
 *
 * The plan is laid out on the host, once for a set of requests, and uploaded:
 * work items of 128 or 32 query rows of one request and key head, over all
 * of its key tiles or a piece of them.
 *
 * The query heads that share a key head are rows of one item: "virtual row"
 * r * group + g is head g of the group of the request's row r, so single rows
 * with shared heads fill an item's columns and K and V are read once for the
 * group.
 *
 * The simple kernel here (one wave per query row and head) serves
 * H3_HIP_REFERENCE=1 and the head sizes, offsets and strides that the
 * matrix-core kernel does not take.
 */
#include "hk_attn.h"
#include "hk_common.h"
#include "hk_internal.h"

#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <type_traits>
#include <vector>

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
       HK_PACKED_PARTS };

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
};

/* One wave per (query row, head) at a time, 64 keys a turn: lane j scores key
 * j of the turn, then lane l adds up dims l, l + 64, ... of the turn's values.
 * Running maximum and sum in F32; P stays F32.  The scale multiplies the
 * distance from the maximum, which F32 holds however far the scores lie from
 * zero. */
__device__ void hk_packed_simple_row(const hk_packed_args &a, uint32_t nth,
                                     uint32_t head) {
    const uint32_t lane = threadIdx.x & 63u;
    /* the last request that begins at or before the nth query row */
    uint32_t low = 0, high = a.request_count;
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (a.requests[mid].before <= nth) low = mid;
        else high = mid;
    }
    const hk_packed_request r = a.requests[low];
    const uint32_t row = r.q_first + (nth - r.before);
    const uint32_t kv_head = head / (a.heads / a.kv_heads);
    const uint16_t *q = a.q + row * a.q_stride + (uint64_t)head * a.dim;
    const uint16_t *k =
        a.k + r.kv_first * a.kv_stride + (uint64_t)kv_head * a.dim;
    const uint16_t *v =
        a.v + r.kv_first * a.kv_stride + (uint64_t)kv_head * a.dim;
    float top = -INFINITY, sum = 0.0f;
    float o[HK_PACKED_MAX_DIM / 64];
    for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++) o[d] = 0.0f;
    for (uint32_t j0 = 0; j0 < r.kv_rows; j0 += 64u) {
        const uint32_t left = min(64u, r.kv_rows - j0);
        float s = -INFINITY;
        if (lane < left) {
            const uint16_t *key = k + (j0 + lane) * a.kv_stride;
            s = 0.0f;
            for (uint32_t d = 0; d < a.dim; d++)
                s = fmaf(hk_bf2f(q[d]), hk_bf2f(key[d]), s);
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
            const float pj = __shfl(p, j, 64);
            const uint16_t *value = v + (j0 + j) * a.kv_stride;
            for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++)
                if (d * 64u + lane < a.dim)
                    o[d] = fmaf(pj, hk_bf2f(value[d * 64u + lane]), o[d]);
        }
    }
    uint16_t *out = a.o + ((uint64_t)row * a.heads + head) * a.dim;
    for (uint32_t d = 0; d < HK_PACKED_MAX_DIM / 64; d++)
        if (d * 64u + lane < a.dim)
            out[d * 64u + lane] = hk_f2bf(sum == 0.0f ? 0.0f : o[d] / sum);
}

__global__ void __launch_bounds__(256) hk_packed_simple(hk_packed_args a) {
    for (uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
         i < (uint64_t)a.rows * a.heads; i += (uint64_t)gridDim.x * 4u) {
        const uint32_t nth = (uint32_t)(i / a.heads);
        hk_packed_simple_row(a, nth, (uint32_t)(i - (uint64_t)nth * a.heads));
    }
}

/* ------------------------------------------------- the matrix-core kernel
 *
 * The scheme of hk_flash_fwd (hk_attn.hip) on a list of items: S^T = K . Q^T
 * with the Q fragments in registers, the softmax in the lanes that hold a
 * query's scores, O^T = V^T . P^T with P straight from the score accumulators
 * and V^T from transposing LDS reads, and two LDS stages of 64 keys filled by
 * direct-to-LDS loads.  What differs:
 *   - rows of K and V come through buffer resources that end with the
 *     request's keys, so what lies behind them (other requests' rows) reads
 *     as zeros and P = 0 meets no infinity or NaN there;
 *   - DIMS = 64, 96 or 128 dims in LDS rows of 64 or 128 (4000 rows, 24 heads
 *     of 96 over 4: 160 us, computed as 128 dims 184), smaller heads padded: a
 *     lane whose piece lies past the head's dims loads from beyond the
 *     resource, zeros;
 *   - tile addresses are 64-bit, so a context may pass 4 GiB;
 *   - NaN scores stay NaN (this file is compiled without the flag that lets
 *     hk_attn.hip assume none).
 *
 * What bounds it, measured (cards differ by up to 5%): self-attention products
 * and exponentials (778, 1536 and 2378 rows x 56 heads 252 to 264 us, 950
 * TFLOP/s; 6144 rows x 40 heads 705, 1.1 PFLOP/s), near the package's power
 * limit though not by that alone, as the figures beside hk_flash_fwd below
 * show; with heads of 64 also a step's barrier and its wait for all loads, as
 * long for half the products (four query heads a key head, 52 to 55 us, 840
 * TFLOP/s); cross-attention to a text an item's start and end around eight
 * tiles, and that items bound by products and items bound by bytes do not
 * overlap (four clips of 6144 rows 176 to 187 us, the sum of its bytes' 106 and
 * its products' 73); single rows the bytes of K and V (eight rows over contexts
 * of 4096 to 9720 49 us, 5 of them the join's: 5.1 TB/s, where a stream of
 * weights reads 6.4) or, with short contexts, the chain item, tiles, joining,
 * store (sixteen rows 13 us, 3.8 TB/s).
 *
 * Four waves of 32 rows and two workgroups a CU.  Beside hk_flash_fwd, whose
 * eight waves share a tile (one request, us here and there): 2378 rows x 56
 * heads 172 and 194, 4096 x 40 324 and 334, 6144 x 40 707 and 686.  Eight waves
 * here, before items were cut: 6144 rows 720 for 754, but 4096 rows 344 for
 * 335, 2378 rows x 56 heads 201 for 190 and 6144 rows x 512 keys 96 for 89.  64
 * rows a wave, which would halve the LDS reads, spill 300 registers at head
 * size 128. */

/* The swizzles of LDS tiles with rows of DP bf16: 16-byte chunk c of row r
 * lies at chunk c ^ key(r).  K's fragment reads take one chunk of 16
 * consecutive rows per 16 lanes, V's transposing reads 64 bytes of 4
 * consecutive rows per 32 lanes; with 256-byte rows each row fills all banks
 * once (keys as in hk_attn.h), 128-byte rows lie two to a turn of the
 * banks. */
template <int DP>
__device__ __forceinline__ uint32_t hk_packed_k_key(uint32_t row) {
    return DP == 128 ? row & 15u : (row >> 1) & 7u;
}

template <int DP>
__device__ __forceinline__ uint32_t hk_packed_v_key(uint32_t row) {
    return DP == 128 ? (row & 3u) << 2 : ((row >> 1) & 1u) << 2;
}

/* hk_vt_read and hk_vt_wait (hk_attn.h) for ND blocks of 32 dims and rows of
 * ROW bytes. */
template <int ND, uint32_t ROW>
__device__ __forceinline__ void hk_packed_vt_read(hk_v2i (&vt)[ND][2],
                                                  const uint32_t (&frag)[ND],
                                                  uint32_t off) {
#pragma unroll
    for (int d = 0; d < ND; d++)
        asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\t"
                     "ds_read_b64_tr_b16 %1, %2 offset:%4"
                     : "=&v"(vt[d][0]), "=&v"(vt[d][1])
                     : "v"(frag[d]), "i"(off), "i"(off + 8u * ROW));
}

template <int N>
__device__ __forceinline__ void hk_packed_vt_wait(hk_v2i (&vt)[4][2]) {
    hk_vt_wait<N>(vt);
}

template <int N>
__device__ __forceinline__ void hk_packed_vt_wait(hk_v2i (&vt)[3][2]) {
    asm volatile("s_waitcnt lgkmcnt(%6)"
                 : "+v"(vt[0][0]), "+v"(vt[0][1]), "+v"(vt[1][0]),
                   "+v"(vt[1][1]), "+v"(vt[2][0]), "+v"(vt[2][1])
                 : "i"(N));
}

template <int N>
__device__ __forceinline__ void hk_packed_vt_wait(hk_v2i (&vt)[2][2]) {
    asm volatile("s_waitcnt lgkmcnt(%4)"
                 : "+v"(vt[0][0]), "+v"(vt[0][1]), "+v"(vt[1][0]),
                   "+v"(vt[1][1])
                 : "i"(N));
}

/* P = exp2((s - m) L), L = scale log2(e), against a reference m, a score
 * itself (not yet times L): maxima, references between tiles and the pieces'
 * are compared as (m - m') L.  Near zero, |m L| < HK_PACKED_FAR, one fused
 * multiply-add a score does it, fma(s, L, -(m L)): what rounding m L moves the
 * reference by, up to 2^-15, is less than the rounding of a score there.  The
 * rounding grows with the score (at 2^33 it is 2^9, and P of every key would be
 * 0 or infinite), so that beyond it m is subtracted from the scores first,
 * which is exact near the maximum. */
#define HK_PACKED_FAR 0x1p10f

/* Whether -(m L) is: also if it is infinite or NaN. */
__device__ __forceinline__ bool hk_packed_far(float neg) {
    return !(fabsf(neg) < HK_PACKED_FAR);
}

/* A wave's direct-to-LDS load of 16 bytes per lane.  A function of its own:
 * in a lambda of a kernel template, the cast to LDS keeps the host pass from
 * emitting the kernel's launch stub when it depends on the template's
 * parameters. */
__device__ __forceinline__ void hk_packed_dma16(__amdgpu_buffer_rsrc_t r,
                                                uint8_t *lds,
                                                uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (hk_lds_void *)lds, 16, offset,
                                             0, 0, 0);
}

/* An item of at most 32 rows: the waves share its rows and split its keys, 32
 * at a time, wave w every fourth from the wth on.  A wave's tiles are its own,
 * so no wave waits for another before the end: K of its next one loads once S
 * is computed, V once P . V is.  Bound by the chain of a step (scores, maximum,
 * exponentials, product: about 1 us, whatever the loads do), of which there
 * are a quarter as many as with the waves on rows: three rows, the longest
 * context 473 keys, 64 heads over 8, 7.4 us instead of 12.9; sixteen rows x 40
 * heads 13.1 and 14.5; one row, 2566 keys, 24 heads of 96 over 4, 9.8 and 11.8.
 * Long contexts, bound by K's and V's bytes, are level.  A request's last few
 * rows beside many full items lose by it: 2185 rows x 40 heads, the last 9 of
 * each 119 us and 109. */
template <int DIMS>
__device__ __forceinline__ void hk_packed_few(const hk_packed_args &a,
                                              const hk_packed_item &it,
                                              uint8_t *lds) {
    constexpr int DP = DIMS <= 64 ? 64 : 128;
    constexpr int NK = DIMS / 16, ND = DIMS / 32, CHUNKS = DP / 8;
    constexpr uint32_t KEYS = 32, ROW = DP * 2u, TILE = KEYS * ROW;
    constexpr int LOADS = TILE / 1024; /* of K or V of a tile */
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 31u, half = lane >> 5;
    const uint32_t dim_chunks = a.dim >> 3;
    const uint32_t stride = (uint32_t)a.kv_stride * 2u;
    uint8_t *own = lds + wave * (2u * TILE);
    uint32_t k_off[LOADS], v_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const uint32_t row = i * (64u / CHUNKS) + lane / CHUNKS;
        const uint32_t kc = (lane % CHUNKS) ^ hk_packed_k_key<DP>(row);
        const uint32_t vc = (lane % CHUNKS) ^ hk_packed_v_key<DP>(row);
        k_off[i] = kc < dim_chunks ? row * stride + kc * 16u : 0x80000000u;
        v_off[i] = vc < dim_chunks ? row * stride + vc * 16u : 0x80000000u;
    }
    const uint64_t kv_base =
        (uint64_t)it.kv_first * a.kv_stride + (uint64_t)it.kv_head * a.dim;
    const uint32_t last =
        min(it.tile_end * (HK_KT / KEYS), (it.kv_rows + KEYS - 1u) / KEYS);
    /* K or V of a tile; past the last one, loads that touch no memory, so that
     * the waits below count right */
    auto load = [&](const uint16_t *from, uint32_t tile, uint8_t *to,
                    const uint32_t (&off)[LOADS]) {
        const uint32_t kv0 = tile * KEYS;
        const uint32_t rows = min(it.kv_rows - kv0, KEYS);
        const __amdgpu_buffer_rsrc_t r = hk_attn_rsrc(
            from + kv_base + kv0 * a.kv_stride,
            tile < last ? (rows - 1u) * stride + a.dim * 2u : 0u);
#pragma unroll
        for (int i = 0; i < LOADS; i++)
            hk_packed_dma16(r, to + i * 1024u, off[i]);
    };
    uint32_t tile = it.tile * (HK_KT / KEYS) + wave;
    load(a.k, tile, own, k_off);

    const uint32_t vrow = it.row + col, r0 = it.row / a.group;
    hk_bf16x8 qf[NK];
    {
        const uint32_t r = vrow / a.group, g = vrow - r * a.group;
        const __amdgpu_buffer_rsrc_t qr = hk_attn_rsrc(
            a.q + ((uint64_t)it.q_first + r0) * a.q_stride +
                (uint64_t)it.kv_head * a.group * a.dim,
            0x7ffffff0u);
        const uint32_t off = vrow < it.rows
                                 ? (r - r0) * (uint32_t)a.q_stride * 2u +
                                       g * a.dim * 2u + half * 16u
                                 : 0x80000000u;
#pragma unroll
        for (int ks = 0; ks < NK; ks++)
            qf[ks] = __builtin_bit_cast(
                hk_bf16x8,
                __builtin_amdgcn_raw_buffer_load_b128(
                    qr,
                    2u * ks + half < dim_chunks ? off + ks * 32u : 0x80000000u,
                    0, 0));
    }
    load(a.v, tile, own + TILE, v_off);

    const uint32_t own_at =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)own;
    uint32_t v_frag[ND];
    {
        const uint32_t j = lane & 15u, g1 = (lane >> 4) & 1u;
        const uint32_t row = 4u * half + (j >> 2);
        const uint32_t low = 2u * g1 + ((j & 3u) >> 1);
#pragma unroll
        for (int d = 0; d < ND; d++)
            v_frag[d] = own_at + TILE + row * ROW +
                        (((d * 4u + low) ^ hk_packed_v_key<DP>(row)) << 4) +
                        8u * (j & 1u);
    }
    hk_f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float m_run = -INFINITY, l_part = 0.0f;
    for (; tile < last; tile += HK_PACKED_WAVES) {
        /* K has landed; V, issued behind it, may be on its way */
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(LOADS) : "memory");
        hk_f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < NK; kk++) {
            const hk_bf16x8 kf = *(const hk_bf16x8 *)(
                own + col * ROW +
                (((kk * 2u + half) ^ hk_packed_k_key<DP>(col)) << 4));
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[kk], s, 0, 0,
                                                        0);
        }
        /* this tile's K has been read */
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        load(a.k, tile + HK_PACKED_WAVES, own, k_off);
        const uint32_t kv0 = tile * KEYS;
        if (it.kv_rows - kv0 < KEYS) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const uint32_t key = kv0 + (r >> 2) * 8u + half * 4u + (r & 3);
                if (key >= it.kv_rows) s[r] = -INFINITY;
            }
        }
        /* the softmax of hk_packed_flash, with the maximum itself */
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[r]);
        const auto sw = __builtin_amdgcn_permlane32_swap(
            __float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        const float m_new = fmaxf(m_run, mx);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float c = __builtin_amdgcn_exp2f((m_run - ref) * a.scale_log2);
        float neg = -(ref * a.scale_log2);
        if (__builtin_amdgcn_ballot_w64(hk_packed_far(neg))) {
            const float less = hk_packed_far(neg) ? ref : 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] -= less;
            if (hk_packed_far(neg)) neg = 0.0f;
        }
        m_run = m_new;
        float sum = 0.0f;
        hk_bf16x8 pf[2];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const float p = __builtin_amdgcn_exp2f(
                __builtin_fmaf(s[r], a.scale_log2, neg));
            sum += p;
            pf[r >> 3][r & 7] = (__bf16)p;
        }
        l_part = l_part * c + sum;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= c;
        /* V has landed; the next K may be on its way */
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(LOADS) : "memory");
        hk_v2i vt[2][ND][2];
        hk_packed_vt_read<ND, ROW>(vt[0], v_frag, 0);
        hk_packed_vt_read<ND, ROW>(vt[1], v_frag, 16u * ROW);
        hk_packed_vt_wait<2 * ND>(vt[0]);
#pragma unroll
        for (int st = 0; st < 2; st++) {
            if (st) hk_packed_vt_wait<0>(vt[1]);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const hk_v4i both = {vt[st][d][0][0], vt[st][d][0][1],
                                     vt[st][d][1][0], vt[st][d][1][1]};
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    __builtin_bit_cast(hk_bf16x8, both), pf[st], o[d], 0, 0,
                    0);
            }
        }
        asm volatile("" ::: "memory");
        load(a.v, tile + HK_PACKED_WAVES, own + TILE, v_off);
    }
    /* The waves' sums: M and L of each row over LDS, then O, scaled to M (and
     * by 1 / L for a whole item), 32 dims at a time in rows of 128 bytes. */
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    float2 *ml = (float2 *)lds;
    const float l_own = l_part + __shfl_xor(l_part, 32, 64);
    if (half == 0) ml[wave * 32u + col] = make_float2(m_run, l_own);
    __syncthreads();
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < HK_PACKED_WAVES; w++)
        top = fmaxf(top, ml[w * 32u + col].x);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (uint32_t w = 0; w < HK_PACKED_WAVES; w++) {
        const float2 v = ml[w * 32u + col];
        l += __builtin_amdgcn_exp2f((v.x - ref) * a.scale_log2) * v.y;
    }
    const bool whole = it.part == HK_PACKED_WHOLE;
    float weight = __builtin_amdgcn_exp2f((m_run - ref) * a.scale_log2);
    if (whole) weight *= l == 0.0f ? 0.0f : 1.0f / l;
    else if (wave == 0 && half == 0 && vrow < it.rows)
        a.part_ml[(size_t)it.part * HK_PACKED_QB + col] = make_float2(top, l);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int blk = 0; blk < 4; blk++) {
            const uint32_t c = blk * 2u + half;
            *(float4 *)(own + d * 4096u + col * 128u +
                        ((c ^ (col & 7u)) << 4)) =
                make_float4(o[d][blk * 4 + 0] * weight,
                            o[d][blk * 4 + 1] * weight,
                            o[d][blk * 4 + 2] * weight,
                            o[d][blk * 4 + 3] * weight);
        }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 32u * DIMS / 4u / (HK_PACKED_WAVES * 64u); i++) {
        const uint32_t at = i * (HK_PACKED_WAVES * 64u) + tid;
        const uint32_t r = at / (DIMS / 4u), dim4 = at % (DIMS / 4u);
        const uint32_t c = dim4 & 7u;
        hk_f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t w = 0; w < HK_PACKED_WAVES; w++)
            sum += *(const hk_f32x4 *)(lds + w * (2u * TILE) +
                                       (dim4 >> 3) * 4096u + r * 128u +
                                       ((c ^ (r & 7u)) << 4));
        const uint32_t vr = it.row + r;
        if (vr >= it.rows || dim4 * 4u >= a.dim) continue;
        if (!whole) {
            *(hk_f32x4 *)(a.part_o +
                          ((size_t)it.part * HK_PACKED_QB + r) * DP +
                          dim4 * 4u) = sum;
            continue;
        }
        const uint32_t qr = vr / a.group, g = vr - qr * a.group;
        *(uint2 *)(a.o +
                   (((uint64_t)it.q_first + qr) * a.heads +
                    it.kv_head * a.group + g) * a.dim +
                   dim4 * 4u) =
            make_uint2(hk_pack2(sum[0], sum[1]), hk_pack2(sum[2], sum[3]));
    }
}

template <int DIMS>
__global__ void __launch_bounds__(HK_PACKED_WAVES * 64, 2)
hk_packed_flash(hk_packed_args a) {
    constexpr int DP = DIMS <= 64 ? 64 : 128;
    constexpr int NK = DIMS / 16, ND = DIMS / 32, CHUNKS = DP / 8;
    constexpr uint32_t ROW = DP * 2u, TILE = HK_KT * ROW, STAGE = 2u * TILE;
    /* 1-KiB loads per wave, tile and operand */
    constexpr int DMA = TILE / 1024 / HK_PACKED_WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 31u, half = lane >> 5;

    hk_packed_item it = a.items[blockIdx.x];
    if (it.row >= it.rows) return;
    if (!a.part_o && it.part != HK_PACKED_WHOLE) {
        /* no room for pieces' sums: the first one takes all keys */
        if (it.tile) return;
        it.tile_end = (it.kv_rows + HK_KT - 1u) / HK_KT;
        it.part = HK_PACKED_WHOLE;
    }
    if (it.rows - it.row <= 32u) {
        hk_packed_few<DIMS>(a, it, hk_lds);
        return;
    }
    const uint32_t dim_chunks = a.dim >> 3;

    /* wave w fills rows of a tile with DMA loads of 64 / CHUNKS rows each,
     * lane l physical chunk l % CHUNKS of row l / CHUNKS; the swizzle is
     * applied on the global side */
    const uint32_t stride = (uint32_t)a.kv_stride * 2u; /* bytes */
    uint32_t k_off[DMA], v_off[DMA];
#pragma unroll
    for (int i = 0; i < DMA; i++) {
        const uint32_t row =
            (wave * DMA + i) * (64u / CHUNKS) + lane / CHUNKS;
        const uint32_t kc = (lane % CHUNKS) ^ hk_packed_k_key<DP>(row);
        const uint32_t vc = (lane % CHUNKS) ^ hk_packed_v_key<DP>(row);
        k_off[i] = kc < dim_chunks ? row * stride + kc * 16u : 0x80000000u;
        v_off[i] = vc < dim_chunks ? row * stride + vc * 16u : 0x80000000u;
    }
    const uint64_t kv_base =
        (uint64_t)it.kv_first * a.kv_stride + (uint64_t)it.kv_head * a.dim;
    auto issue_tile = [&](uint32_t tile, uint32_t stage) {
        const uint32_t kv0 = tile * HK_KT;
        const uint64_t base = kv_base + kv0 * a.kv_stride;
        /* the rows of this tile that the request has end the resource: 64
         * rows stay below 2^31 bytes (hk_packed_takes) */
        const uint32_t rows = min(it.kv_rows - kv0, (uint32_t)HK_KT);
        const uint32_t bytes = (rows - 1u) * stride + a.dim * 2u;
        const __amdgpu_buffer_rsrc_t vr = hk_attn_rsrc(a.v + base, bytes);
        const __amdgpu_buffer_rsrc_t kr = hk_attn_rsrc(a.k + base, bytes);
        uint8_t *st = hk_lds + stage * STAGE;
#pragma unroll
        for (int i = 0; i < DMA; i++)
            hk_packed_dma16(vr, st + TILE + (wave * DMA + i) * 1024u,
                            v_off[i]);
#pragma unroll
        for (int i = 0; i < DMA; i++)
            hk_packed_dma16(kr, st + (wave * DMA + i) * 1024u, k_off[i]);
    };
    const uint32_t n = it.tile_end - it.tile;
    if (n) issue_tile(it.tile, 0);

    /* Q fragments, the B operand of S^T = K . Q^T: k-step ks of this lane's
     * virtual row, dims 16 ks + 8 half .. + 8.  Offsets from the item's first
     * row (hk_packed_takes); rows past the request's and dims past the head's
     * load from beyond the resource, zeros. */
    const uint32_t vrow0 = it.row + wave * 32u, vrow = vrow0 + col;
    const uint32_t r0 = it.row / a.group;
    hk_bf16x8 qf[NK];
    {
        const uint32_t r = vrow / a.group, g = vrow - r * a.group;
        const __amdgpu_buffer_rsrc_t qr = hk_attn_rsrc(
            a.q + ((uint64_t)it.q_first + r0) * a.q_stride +
                (uint64_t)it.kv_head * a.group * a.dim,
            0x7ffffff0u);
        const uint32_t off =
            n && vrow < it.rows ? (r - r0) * (uint32_t)a.q_stride * 2u +
                                      g * a.dim * 2u + half * 16u
                                : 0x80000000u;
#pragma unroll
        for (int ks = 0; ks < NK; ks++)
            qf[ks] = __builtin_bit_cast(
                hk_bf16x8,
                __builtin_amdgcn_raw_buffer_load_b128(
                    qr,
                    2u * ks + half < dim_chunks ? off + ks * 32u : 0x80000000u,
                    0, 0));
    }

    const uint32_t lds_base =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)
            hk_lds;
    uint32_t k_frag[NK];
#pragma unroll
    for (int kk = 0; kk < NK; kk++)
        k_frag[kk] =
            lds_base + col * ROW +
            (((kk * 2u + half) ^ hk_packed_k_key<DP>(col)) << 4);
    /* the transposing reads' source lanes, as in hk_flash_fwd */
    uint32_t v_frag[ND];
    {
        const uint32_t j = lane & 15u, g1 = (lane >> 4) & 1u;
        const uint32_t row = 4u * half + (j >> 2);
        const uint32_t low = 2u * g1 + ((j & 3u) >> 1);
#pragma unroll
        for (int d = 0; d < ND; d++)
            v_frag[d] =
                lds_base + TILE + row * ROW +
                (((d * 4u + low) ^ hk_packed_v_key<DP>(row)) << 4) +
                8u * (j & 1u);
    }

    hk_f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    /* the reference m and -(m L); unset (-infinity) until a score has weight */
    float m_run = -INFINITY, neg = INFINITY, l_part = 0.0f;
    /* a wave whose rows all lie past the request's stages its share of every
     * tile and meets every barrier, and computes nothing */
    const bool live = vrow0 < it.rows;

    auto tile_step = [&](auto stage_tag, uint32_t tile, bool more,
                         auto tail_tag) {
        constexpr uint32_t stage = decltype(stage_tag)::value;
        constexpr bool tail = decltype(tail_tag)::value;
        if (more) issue_tile(tile + 1u, stage ^ 1u);
        if (live) {
        hk_f32x16 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[kt][r] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < NK; kk++)
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const hk_bf16x8 kf = *(const hk_bf16x8 *)(
                    (__attribute__((address_space(3))) uint8_t *)(uintptr_t)
                        (k_frag[kk] + stage * STAGE + kt * 32u * ROW));
                s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    kf, qf[kk], s[kt], 0, 0, 0);
            }
        const uint32_t kv0 = tile * HK_KT;
        if (tail && it.kv_rows - kv0 < HK_KT) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const uint32_t key = kv0 + kt * 32u + (r >> 2) * 8u +
                                         half * 4u + (r & 3);
                    if (key >= it.kv_rows) s[kt][r] = -INFINITY;
                }
        }
        /* The softmax of hk_flash_fwd: P against the running maximum as it
         * stands, which moves (O and l rescaled) only when it is unset or far
         * or one of its P sums passes 2^32.  P <= 2^32 keeps O and l far from
         * overflow.  P rounds to bf16, which the matrix cores take (two halves
         * as of the adapters would be half as many products again), l sums the
         * unrounded P: the result is off by 2^-8 of a weight at most where F32
         * weights would leave it at the rounding of the output, 0.0023 and
         * 0.0017 of its norm for 1500 keys. */
        hk_bf16x8 pf[2][2];
        auto exps = [&](float less) -> float {
            float sum = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                float p[16];
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    p[r] = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(s[kt][r], a.scale_log2, less));
                    sum += p[r];
                }
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    hk_bf16x8 v;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = (__bf16)p[st * 8 + e];
                    pf[kt][st] = v;
                }
            }
            return sum;
        };
        const bool far = hk_packed_far(neg); /* or unset */
        float sum = far ? 0.0f : exps(neg);
        uint32_t move = far || sum > 0x1p32f;
        if (__builtin_amdgcn_ballot_w64(move)) {
            /* a row's other half's too, but no other row's: what a row comes
             * to does not depend on the rows beside it */
            const auto mv =
                __builtin_amdgcn_permlane32_swap(move, move, false, false);
            move = mv[0] | mv[1];
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[kt][r]);
            const auto sw = __builtin_amdgcn_permlane32_swap(
                __float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            const float m_new = move ? fmaxf(m_run, mx) : m_run;
            const float ref = m_new == -INFINITY ? 0.0f : m_new;
            const float c =
                move ? __builtin_amdgcn_exp2f((m_run - ref) * a.scale_log2)
                     : 1.0f;
            /* every score so far -inf: the maximum stays unset */
            m_run = m_new;
            neg = -(m_new * a.scale_log2);
            float less = -(ref * a.scale_log2);
            if (__builtin_amdgcn_ballot_w64(hk_packed_far(less))) {
                const float by = hk_packed_far(less) ? ref : 0.0f;
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[kt][r] -= by;
                if (hk_packed_far(less)) less = 0.0f;
            }
            l_part *= c;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= c;
            sum = exps(less);
        }
        l_part += sum;

        hk_v2i vt[2][ND][2];
        hk_packed_vt_read<ND, ROW>(vt[0], v_frag, stage * STAGE);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int kt = i >> 1, st = i & 1;
            if (i < 3) {
                hk_packed_vt_read<ND, ROW>(vt[(i + 1) & 1], v_frag,
                                           stage * STAGE +
                                               (i + 1) * 16u * ROW);
                hk_packed_vt_wait<2 * ND>(vt[i & 1]);
            } else {
                hk_packed_vt_wait<0>(vt[i & 1]);
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const hk_v4i both = {vt[i & 1][d][0][0], vt[i & 1][d][0][1],
                                     vt[i & 1][d][1][0], vt[i & 1][d][1][1]};
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    __builtin_bit_cast(hk_bf16x8, both), pf[kt][st], o[d], 0,
                    0, 0);
            }
        }
        } /* live */
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    using S0 = std::integral_constant<uint32_t, 0>;
    using S1 = std::integral_constant<uint32_t, 1>;
    using NT = std::integral_constant<bool, false>;
    using TT = std::integral_constant<bool, true>;
    if (n) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t i = 0;
        for (; i + 2 < n; i += 2) {
            tile_step(S0(), it.tile + i, true, NT());
            tile_step(S1(), it.tile + i + 1, true, NT());
        }
        if (i + 2 == n) {
            tile_step(S0(), it.tile + i, true, NT());
            tile_step(S1(), it.tile + i + 1, false, TT());
        } else {
            tile_step(S0(), it.tile + i, false, TT());
        }
    }

    /* The lane holds query column `col`, dims 32 d + 8 (r / 4) + 4 half +
     * r % 4.  The wave's rows go through LDS of its own (free after the last
     * barrier), 16-byte chunk c of row r at c ^ key, and leave as whole
     * rows. */
    const float l = l_part + __shfl_xor(l_part, 32, 64);
    if (it.part != HK_PACKED_WHOLE) {
        /* 32 dims at a time, rows of 128 bytes */
        float *pw = (float *)(hk_lds + wave * (32u * 32u * 4u));
        float *part = a.part_o + (size_t)it.part * HK_PACKED_QB * DP;
#pragma unroll
        for (int d = 0; d < ND; d++) {
#pragma unroll
            for (int blk = 0; blk < 4; blk++) {
                const uint32_t c = blk * 2u + half;
                *(float4 *)(pw + col * 32u + ((c ^ (col & 7u)) << 2)) =
                    make_float4(o[d][blk * 4 + 0], o[d][blk * 4 + 1],
                                o[d][blk * 4 + 2], o[d][blk * 4 + 3]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t r = i * 8u + (lane >> 3), c = lane & 7u;
                const float4 v =
                    *(const float4 *)(pw + r * 32u + ((c ^ (r & 7u)) << 2));
                if (vrow0 + r < it.rows)
                    *(float4 *)(part + (size_t)(wave * 32u + r) * DP +
                                d * 32u + c * 4u) = v;
            }
        }
        if (half == 0 && vrow < it.rows)
            a.part_ml[(size_t)it.part * HK_PACKED_QB + wave * 32u + col] =
                make_float2(m_run, l);
        return;
    }
    /* no keys, or none with weight: zeros (a NaN sum gives NaN) */
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t *ow = hk_lds + wave * (32u * ROW);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int blk = 0; blk < 4; blk++) {
            const uint32_t chunk = d * 4u + blk;
            *(uint2 *)(ow + col * ROW +
                       ((chunk ^ hk_packed_k_key<DP>(col)) << 4) + half * 8u) =
                make_uint2(hk_pack2(o[d][blk * 4 + 0] * inv,
                                    o[d][blk * 4 + 1] * inv),
                           hk_pack2(o[d][blk * 4 + 2] * inv,
                                    o[d][blk * 4 + 3] * inv));
        }
    const __amdgpu_buffer_rsrc_t outr =
        hk_attn_rsrc(a.o + (((uint64_t)it.q_first + r0) * a.heads +
                            it.kv_head * a.group) * a.dim,
                     0x7ffffff0u);
#pragma unroll
    for (int i = 0; i < 32 * CHUNKS / 64; i++) {
        const uint32_t r = i * (64u / CHUNKS) + lane / CHUNKS;
        const uint32_t c = lane % CHUNKS, vr = vrow0 + r;
        const hk_v4i v = *(const hk_v4i *)(
            ow + r * ROW + ((c ^ hk_packed_k_key<DP>(r)) << 4));
        const uint32_t qr = vr / a.group, g = vr - qr * a.group;
        __builtin_amdgcn_raw_buffer_store_b128(
            v, outr,
            vr < it.rows && c < dim_chunks
                ? (((qr - r0) * a.heads + g) * a.dim + c * 8u) * 2u
                : 0x80000000u,
            0, 0);
    }
}

/* Joins the pieces of an item's rows: with the pieces' references m_p, sums
 * l_p and undivided O_p, O = sum_p w_p O_p / sum_p w_p l_p with w_p =
 * 2^((m_p - M) L), M = max_p m_p, in piece order.  A wave per row; a lane
 * holds DP / 64 dims and has four pieces on their way.  Bound by the launch and
 * two loads in sequence: 64 joins of 8 rows take 4.8 us. */
template <int DP>
__global__ void __launch_bounds__(256) hk_packed_joined(hk_packed_args a) {
    const hk_packed_join j = a.joins[blockIdx.x];
    const uint32_t ql = blockIdx.y * 4u + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, vr = j.row + ql;
    if (vr >= j.rows) return;
    constexpr int PER = DP / 64;
    typedef float per __attribute__((ext_vector_type(PER)));
    const float2 *ml = a.part_ml + (size_t)j.part * HK_PACKED_QB + ql;
    const float *po = a.part_o + ((size_t)j.part * HK_PACKED_QB + ql) * DP +
                      lane * PER;
    /* the maximum over all pieces, 64 at a time */
    float top = -INFINITY;
    for (uint32_t p = lane; p < j.pieces; p += 64u)
        top = fmaxf(top, ml[(size_t)p * HK_PACKED_QB].x);
    top = hk_wave_max(top);
    if (top == -INFINITY) top = 0.0f; /* no piece has a weight */
    per sum = {};
    float l = 0.0f;
    for (uint32_t first = 0; first < j.pieces; first += 4u) {
        float2 mine[4];
        per op[4];
#pragma unroll
        for (uint32_t p = 0; p < 4; p++) {
            const size_t at =
                (size_t)min(first + p, j.pieces - 1u) * HK_PACKED_QB;
            mine[p] = ml[at];
            op[p] = *(const per *)(po + at * DP);
        }
#pragma unroll
        for (uint32_t p = 0; p < 4; p++) {
            const float w = first + p < j.pieces
                                ? __builtin_amdgcn_exp2f((mine[p].x - top) *
                                                         a.scale_log2)
                                : 0.0f;
            l += first + p < j.pieces ? w * mine[p].y : 0.0f;
            sum += first + p < j.pieces ? op[p] * w : per{};
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint32_t qr = vr / a.group, g = vr - qr * a.group;
    uint16_t *out = a.o + (((uint64_t)j.q_first + qr) * a.heads +
                           j.kv_head * a.group + g) * a.dim;
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (lane * PER + e < a.dim) out[lane * PER + e] = hk_f2bf(sum[e] * inv);
}

template <int DIMS>
static void hk_packed_launch(struct h3_gpu *gpu, const hk_packed_args &a,
                             const uint32_t *n) {
    constexpr int DP = DIMS <= 64 ? 64 : 128;
    constexpr uint32_t lds = 2u * 2u * HK_KT * DP * 2u;
    /* a launch has fewer than 2^32 threads; whole turns of the XCDs */
    const uint32_t most = 1u << 23;
    for (uint32_t first = 0; first < n[HK_PACKED_ITEMS]; first += most) {
        hk_packed_args part = a;
        part.items = a.items + first;
        hipLaunchKernelGGL(hk_packed_flash<DIMS>,
                           dim3(std::min(n[HK_PACKED_ITEMS] - first, most)),
                           dim3(HK_PACKED_WAVES * 64u), lds, gpu->stream,
                           part);
    }
    if (a.part_o)
        hipLaunchKernelGGL(hk_packed_joined<DP>,
                           dim3(n[HK_PACKED_JOINS],
                                (n[HK_PACKED_JOIN_ROWS] + 3u) / 4u),
                           dim3(256), 0, gpu->stream, a);
}

/* Whether the matrix-core kernel takes these rows: whole 16-byte pieces, 64
 * key rows and 128 query and output rows below 2^31 bytes (the reach of lane
 * offsets), and a scale that -inf times it is -inf, what keys past the end are
 * set to, and 0 times it 0. */
static bool hk_packed_takes(const struct h3_gpu *gpu,
                            const hk_packed_args &a) {
    return !gpu->reference_kernels && a.dim % 8u == 0 && a.dim <= 128u &&
           a.q_stride % 8u == 0 && a.kv_stride % 8u == 0 &&
           a.kv_stride < (1u << 24) && a.q_stride < (1u << 23) &&
           (uint64_t)a.heads * a.dim < (1u << 23) && a.scale_log2 > 0x1p-100f &&
           isfinite(a.scale_log2) &&
           (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v |
             (uintptr_t)a.o) & 15u) == 0;
}

/* How a plan's items are dealt out.  An item costs its key tiles and, for its
 * start and end, about three tiles' time (`own`).
 *
 * Workgroups go to the 8 XCDs in turn.  A request's items, head by head, go to
 * the XCDs' queues in 8 even runs, so that items that share K and V mostly
 * share an L2 and every XCD has its part of the long and of the short ones (a
 * run to the least filled queue each time: 512 items of equal length dealt out
 * less evenly took a second round, 50 us for 43).  Longest first; items of no
 * rows fill the shorter queues.
 *
 * Items are cut into pieces by when the last of the places that take one after
 * the other would end, the join's time included:
 * - all items, where they are few and long (the longest over a place's share of
 *   the work), so that two workgroups a CU keep its loads going;
 * - those behind the last full round of one item a CU, where that promises 5%
 *   (two workgroups of matrix products share what one alone would get, so a
 *   CU is one place; self-attention in us, uncut and cut: 1200 rows x 56
 *   heads, 2.2 rounds, 62.4 and 54.7; 2378 x 56, 4.2, 187 and 167; 2560 x 40,
 *   3.1, 150 and 137; 6144 x 40, 7.5, 733 and 705; counted as two places a CU,
 *   2185 x 40, 2.8 rounds, was cut and took 129 for 113 then).
 *
 * Where 128 rows make few items, items of 32 rows fill the CUs and have a
 * quarter of the steps (hk_packed_few), at the price of K and V four times
 * from L2: up to one a CU, and up to two if they are mostly full (measured with
 * 128 and 32 rows, us: 700 rows of self-attention x 8 heads, 176 small items,
 * 17.7 and 10.3; 537 x 16 over 2, 272, 15.7 and 12.4; 1200 x 12 of 64, 456,
 * 18.0 and 12.1; 300 rows x 24 heads of 96, 512 keys, 240, 12.0 and 7.9; but
 * 300 rows x 40, 400 and 5 tiles, 11.3 and 12.4; four times 50 rows x 40, 320
 * half empty ones, 13.7 and 15.2). */
struct hk_packed_work {
    std::vector<hk_packed_item> items;
    std::vector<hk_packed_join> joins;
    uint32_t parts, join_rows;
};

/* Items [first, first + count) of a request: kv_head * blocks + block of its
 * rows. */
struct hk_packed_run {
    uint32_t request, tiles, rows, blocks;
    uint64_t first, count;
    uint32_t pieces, per; /* of each item, in tiles */
};

static const float hk_packed_own = 3.0f, hk_packed_join_time = 8.0f;

/* Cuts the run's items into pieces of at most `most` tiles. */
static void hk_packed_cut(hk_packed_run &r, uint32_t most) {
    r.pieces = r.tiles > most ? (r.tiles + most - 1) / most : 1;
    r.per = r.pieces > 1 ? (r.tiles + r.pieces - 1) / r.pieces : r.tiles;
    r.pieces = r.pieces > 1 ? (r.tiles + r.per - 1) / r.per : 1;
}

/* When the last place ends, in tiles.  `end` is sorted: the places before the
 * first one's end after an item of length t take one each, in order, before
 * any takes its second. */
static float hk_packed_end(const std::vector<hk_packed_run> &runs,
                           uint32_t places) {
    std::vector<float> end(places, 0.0f);
    bool cut = false;
    for (size_t i = 0; i < runs.size();) {
        const float t = (float)runs[i].per + hk_packed_own;
        uint64_t left = 0;
        for (const uint32_t per = runs[i].per;
             i < runs.size() && runs[i].per == per; i++) {
            cut |= runs[i].pieces > 1;
            left += runs[i].count * runs[i].pieces;
        }
        while (left) {
            const auto until = std::upper_bound(end.begin(), end.end(),
                                                end.front() + t);
            const uint64_t n =
                std::min<uint64_t>(left, (uint64_t)(until - end.begin()));
            for (uint64_t j = 0; j < n; j++) end[j] += t;
            std::inplace_merge(end.begin(), end.begin() + (ptrdiff_t)n,
                               end.end());
            left -= n;
        }
    }
    return end.back() + (cut ? hk_packed_join_time : 0.0f);
}

/* The requests' items of `qb` rows, whole, those with the most tiles first;
 * their number in `items`. */
static std::vector<hk_packed_run> hk_packed_whole(
    const std::vector<hk_packed_request> &list, uint32_t group,
    uint32_t kv_heads, uint32_t qb, uint64_t &items) {
    std::vector<hk_packed_run> runs;
    items = 0;
    for (uint32_t i = 0; i < list.size(); i++) {
        const uint32_t rows = list[i].q_rows * group;
        const uint32_t tiles =
            (uint32_t)(((uint64_t)list[i].kv_rows + HK_KT - 1) / HK_KT);
        const uint32_t blocks = (uint32_t)(((uint64_t)rows + qb - 1) / qb);
        const uint64_t count = (uint64_t)blocks * kv_heads;
        runs.push_back({i, tiles, rows, blocks, 0, count, 1, tiles});
        items += count;
    }
    std::stable_sort(runs.begin(), runs.end(),
                     [](const hk_packed_run &x, const hk_packed_run &y) {
                         return x.tiles > y.tiles;
                     });
    return runs;
}

static void hk_packed_lay_out(const std::vector<hk_packed_request> &list,
                              uint32_t group, uint32_t kv_heads,
                              uint32_t dims, uint32_t cus,
                              hk_packed_work &work) {
    const uint32_t places = cus * 2u;
    uint32_t qb = HK_PACKED_QB;
    uint64_t items, small;
    std::vector<hk_packed_run> runs =
        hk_packed_whole(list, group, kv_heads, qb, items);
    const std::vector<hk_packed_run> low =
        hk_packed_whole(list, group, kv_heads, 32, small);
    double total = 0.0;
    for (const hk_packed_run &r : runs)
        total += (double)r.count * (r.tiles + hk_packed_own);
    /* (many items come out level whole) */
    if (!runs.empty() && items <= 16ull * places) {
        std::vector<hk_packed_run> chosen = runs;
        const uint32_t share = (uint32_t)(total / places) + 1u;
        float best = hk_packed_end(runs, places);
        if (runs[0].tiles >= share) { /* few and long */
            uint32_t tried = 0;
            for (uint32_t i = 4; i <= 24; i++) { /* half to three shares */
                const uint32_t length = std::max(4u, share * i / 8u);
                if (length == tried || length >= runs[0].tiles) continue;
                tried = length;
                std::vector<hk_packed_run> cut = runs;
                double bytes = 0.0; /* of the pieces' sums, both ways */
                for (hk_packed_run &r : cut) {
                    hk_packed_cut(r, length);
                    if (r.pieces > 1)
                        bytes += (double)r.rows * kv_heads * r.pieces * dims *
                                 8.0;
                }
                const float end = hk_packed_end(cut, places) +
                                  (float)(bytes / 4.5e6);
                if (end < best) {
                    best = end;
                    chosen = cut;
                }
            }
        } else if (items % cus) {
            std::vector<hk_packed_run> head, tail;
            uint64_t whole = items - items % cus;
            double rest = 0.0;
            for (const hk_packed_run &r : runs) {
                hk_packed_run h = r, t = r;
                h.count = std::min(whole, r.count);
                t.first = h.count;
                t.count = r.count - h.count;
                whole -= h.count;
                rest += (double)t.count * t.tiles;
                if (h.count) head.push_back(h);
                if (t.count) tail.push_back(t);
            }
            float least = 0.95f * hk_packed_end(runs, cus);
            for (uint32_t i = 4; i <= 8; i++) { /* one to two shares */
                const uint32_t length =
                    std::max(4u, (uint32_t)(rest / cus * i / 4) + 1u);
                std::vector<hk_packed_run> cut = head;
                for (hk_packed_run r : tail) {
                    hk_packed_cut(r, length);
                    cut.push_back(r);
                }
                const float end = hk_packed_end(cut, cus);
                if (end < least) {
                    least = end;
                    chosen = cut;
                }
            }
        }
        const float step = small <= cus ? 0.6f : 0.85f;
        if (small > items && small <= places &&
            (small <= cus || small >= 3 * items) &&
            hk_packed_own + 1.0f + step * (float)runs[0].tiles < best) {
            qb = 32;
            chosen = low;
        }
        runs = chosen;
    }
    std::vector<hk_packed_item> queue[8];
    double load[8] = {};
    work.parts = work.join_rows = 0;
    for (const hk_packed_run &s : runs) {
        const hk_packed_request &r = list[s.request];
        for (uint64_t run = 0; run < 8; run++) {
            /* the longer runs are the last ones */
            const uint64_t end = s.first + s.count * (run + 1) / 8;
            uint64_t i = s.first + s.count * run / 8;
            auto &q = *std::min_element(
                queue, queue + 8, [&](const auto &x, const auto &y) {
                    return load[&x - queue] < load[&y - queue];
                });
            load[&q - queue] +=
                (double)(end - i) * (s.tiles + hk_packed_own * s.pieces);
            for (; i < end; i++) {
                const uint32_t row = (uint32_t)(i % s.blocks) * qb;
                hk_packed_item item = {r.q_first, std::min(s.rows, row + qb),
                                       row,
                                       (uint32_t)(i / s.blocks), r.kv_first,
                                       r.kv_rows, 0, s.tiles,
                                       HK_PACKED_WHOLE};
                if (s.pieces > 1) {
                    work.joins.push_back({r.q_first, item.rows, row,
                                          item.kv_head, work.parts,
                                          s.pieces});
                    work.join_rows = std::max(
                        work.join_rows, item.rows - row);
                }
                for (uint32_t p = 0; p < s.pieces; p++) {
                    item.tile = p * s.per;
                    item.tile_end = std::min(s.tiles, item.tile + s.per);
                    if (s.pieces > 1) item.part = work.parts++;
                    q.push_back(item);
                }
            }
        }
    }
    size_t longest = 0;
    for (const auto &q : queue) longest = std::max(longest, q.size());
    for (size_t j = 0; j < longest; j++)
        for (const auto &q : queue)
            work.items.push_back(j < q.size() ? q[j] : hk_packed_item{});
}

extern "C" {

h3_gpu_tensor *h3_hip_sdpa_packed_plan(h3_gpu *gpu, const uint32_t *q_first,
                                       const uint32_t *q_rows,
                                       const uint32_t *kv_first,
                                       const uint32_t *kv_rows,
                                       uint32_t requests, uint32_t heads,
                                       uint32_t kv_heads, uint32_t head_dim) {
    if (!gpu) return NULL;
    if (!requests || !q_first || !q_rows || !kv_first || !kv_rows) {
        hk_fail(gpu, "attention plan needs at least one request");
        return NULL;
    }
    if (!heads || !kv_heads || heads % kv_heads || !head_dim ||
        head_dim > HK_PACKED_MAX_DIM ||
        (uint64_t)heads * head_dim > UINT32_MAX) {
        hk_fail(gpu, "attention plan: %u heads of %u over %u key heads "
                     "(heads a multiple of key heads, head_dim 1 to %u)",
                heads, head_dim, kv_heads, HK_PACKED_MAX_DIM);
        return NULL;
    }
    try {
        std::vector<hk_packed_request> list;
        uint64_t rows = 0, q_end = 0, kv_end = 0;
        for (uint32_t i = 0; i < requests; i++) {
            const uint64_t qe = (uint64_t)q_first[i] + q_rows[i];
            const uint64_t ke = (uint64_t)kv_first[i] + kv_rows[i];
            if (qe > UINT32_MAX || ke > UINT32_MAX) {
                hk_fail(gpu, "attention plan: the rows of request %u pass "
                             "2^32", i);
                return NULL;
            }
            /* the kernels count keys in 32 bits, up to the end of the last
             * tile and a turn past it */
            if (kv_rows[i] > HK_PACKED_MAX_KEYS) {
                hk_fail(gpu, "attention plan: request %u has %u key rows, over "
                             "%u", i, kv_rows[i], HK_PACKED_MAX_KEYS);
                return NULL;
            }
            if (!q_rows[i]) continue;
            list.push_back({q_first[i], q_rows[i], kv_first[i], kv_rows[i],
                            (uint32_t)rows});
            rows += q_rows[i];
            q_end = std::max(q_end, qe);
            if (kv_rows[i]) kv_end = std::max(kv_end, ke);
        }
        std::vector<std::pair<uint32_t, uint32_t>> ranges;
        for (const auto &r : list) ranges.push_back({r.q_first, r.q_rows});
        std::sort(ranges.begin(), ranges.end());
        for (size_t i = 1; i < ranges.size(); i++)
            if ((uint64_t)ranges[i - 1].first + ranges[i - 1].second >
                ranges[i].first) {
                hk_fail(gpu, "attention plan: query rows of two requests "
                             "overlap at row %u", ranges[i].first);
                return NULL;
            }
        /* (an item for every 128 of them, or, of single rows, each) */
        if (rows * heads >= 1ull << 29) {
            hk_fail(gpu, "attention plan: too many query rows and heads");
            return NULL;
        }
        hk_packed_work work;
        hk_packed_lay_out(list, heads / kv_heads, kv_heads, head_dim,
                          gpu->num_cus > 0 ? (uint32_t)gpu->num_cus : 256u,
                          work);
        std::vector<uint32_t> words;
        auto add = [&](const void *data, size_t bytes) {
            const uint32_t *w = (const uint32_t *)data;
            words.insert(words.end(), w, w + bytes / 4);
        };
        add(list.data(), list.size() * sizeof(list[0]));
        add(work.items.data(), work.items.size() * sizeof(work.items[0]));
        add(work.joins.data(), work.joins.size() * sizeof(work.joins[0]));
        if (words.empty()) words.push_back(0);
        h3_gpu_tensor *plan =
            h3_gpu_tensor_from_u32(gpu, words.data(), words.size());
        if (!plan) return NULL;
        plan->record.kind = HK_RECORD_PACKED;
        plan->record.n[HK_PACKED_HEADS] = heads;
        plan->record.n[HK_PACKED_KV_HEADS] = kv_heads;
        plan->record.n[HK_PACKED_DIM] = head_dim;
        plan->record.n[HK_PACKED_REQUESTS] = (uint32_t)list.size();
        plan->record.n[HK_PACKED_ROWS] = (uint32_t)rows;
        plan->record.n[HK_PACKED_Q_END] = (uint32_t)q_end;
        plan->record.n[HK_PACKED_KV_END] = (uint32_t)kv_end;
        plan->record.n[HK_PACKED_ITEMS] = (uint32_t)work.items.size();
        plan->record.n[HK_PACKED_JOINS] = (uint32_t)work.joins.size();
        plan->record.n[HK_PACKED_JOIN_ROWS] = work.join_rows;
        plan->record.n[HK_PACKED_PARTS] = work.parts;
        return plan;
    } catch (const std::bad_alloc &) {
        hk_fail(gpu, "out of host memory");
        return NULL;
    }
}

int h3_hip_sdpa_packed_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                            const h3_gpu_tensor *query, size_t query_offset,
                            uint32_t query_stride, const h3_gpu_tensor *key,
                            size_t key_offset, const h3_gpu_tensor *value,
                            size_t value_offset, uint32_t kv_stride,
                            const h3_gpu_tensor *plan, float scale) {
    if (!plan || plan->record.kind != HK_RECORD_PACKED)
        return hk_fail(gpu, "packed attention: the plan was not built by "
                            "h3_hip_sdpa_packed_plan");
    const uint32_t *n = plan->record.n;
    const uint32_t heads = n[HK_PACKED_HEADS], dim = n[HK_PACKED_DIM];
    const uint32_t kv_heads = n[HK_PACKED_KV_HEADS];
    const uint64_t q_width = (uint64_t)heads * dim;
    const uint64_t kv_width = (uint64_t)kv_heads * dim;
    /* elements that a tensor needs for `rows` rows from `offset` on; sizes
     * past what an address can hold come out as the largest */
    auto extent = [](size_t offset, uint64_t stride, uint64_t rows,
                     uint64_t width) -> size_t {
        const uint64_t need = rows ? (rows - 1) * stride + width : 0;
        return offset > SIZE_MAX - need ? SIZE_MAX : offset + need;
    };
    if (query_stride < q_width || kv_stride < kv_width)
        return hk_fail(gpu, "packed attention: row strides %u and %u are "
                            "under the rows' %llu and %llu elements",
                       query_stride, kv_stride, (unsigned long long)q_width,
                       (unsigned long long)kv_width);
    if (!isfinite(scale) || scale < 0.0f)
        return hk_fail(gpu, "packed attention: the scale must be finite and "
                            "not negative");
    if (!hk_require(gpu, query,
                    extent(query_offset, query_stride, n[HK_PACKED_Q_END],
                           q_width), H3_GPU_BF16, "packed query") ||
        !hk_require(gpu, key,
                    extent(key_offset, kv_stride, n[HK_PACKED_KV_END],
                           kv_width), H3_GPU_BF16, "packed key") ||
        !hk_require(gpu, value,
                    extent(value_offset, kv_stride, n[HK_PACKED_KV_END],
                           kv_width), H3_GPU_BF16, "packed value") ||
        !hk_require(gpu, output, n[HK_PACKED_Q_END] * q_width, H3_GPU_BF16,
                    "packed output") ||
        !hk_require_active(gpu))
        return 0;
    if (output == query || output == key || output == value)
        return hk_fail(gpu, "packed attention: the output must be a tensor "
                            "of its own");
    if (!n[HK_PACKED_ROWS]) return 1;
    hk_packed_args a = {};
    a.q = HK_CBF16(query) + query_offset;
    a.k = HK_CBF16(key) + key_offset;
    a.v = HK_CBF16(value) + value_offset;
    a.o = HK_BF16(output);
    a.q_stride = query_stride;
    a.kv_stride = kv_stride;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.dim = dim;
    a.scale = scale;
    a.group = heads / kv_heads;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.requests = (const hk_packed_request *)plan->data;
    a.request_count = n[HK_PACKED_REQUESTS];
    a.rows = n[HK_PACKED_ROWS];
    a.items = (const hk_packed_item *)(a.requests + a.request_count);
    a.joins = (const hk_packed_join *)(a.items + n[HK_PACKED_ITEMS]);
    hk_op_begin(gpu, "attention_packed");
    if (hk_packed_takes(gpu, a)) {
        const size_t padded = dim <= 64 ? 64 : 128;
        const size_t rows = (size_t)n[HK_PACKED_PARTS] * HK_PACKED_QB;
        if (rows)
            a.part_o = (float *)hk_splitk_try(
                gpu, rows * (padded * sizeof(float) + sizeof(float2)));
        /* without scratch, items run whole */
        if (a.part_o) a.part_ml = (float2 *)(a.part_o + rows * padded);
        if (dim <= 64)
            hk_packed_launch<64>(gpu, a, n);
        else if (dim <= 96)
            hk_packed_launch<96>(gpu, a, n);
        else
            hk_packed_launch<128>(gpu, a, n);
        return hk_op_end(gpu, "attention_packed", HK_KIND_SDPA);
    }
    const uint64_t blocks = ((uint64_t)a.rows * heads + 3) / 4;
    hipLaunchKernelGGL(
        hk_packed_simple,
        dim3((unsigned)(blocks < 1u << 20 ? blocks : 1u << 20)), dim3(256), 0,
        gpu->stream, a);
    return hk_op_end(gpu, "attention_packed", HK_KIND_SDPA);
}

} /* extern "C" */
