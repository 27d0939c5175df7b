/* Attention of several requests packed in one call (h3_hip_sdpa_packed_plan /
 * _bf16 in h3_hip.h): query row r of request i, head h,
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j),
 * over request i's key rows j and key head h / (heads / kv_heads).
 *
 * The plan is laid out on the host, once for a set of requests, and uploaded.
 *
 * The simple kernel here (one wave per query row and head) serves
 * H3_HIP_REFERENCE=1 and the head sizes, offsets and strides that the
 * matrix-core kernel does not take.
 */
#include "hk_common.h"
#include "hk_internal.h"

#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <new>
#include <vector>

#define HK_PACKED_MAX_DIM 256u

/* a request with query rows, in device memory */
struct hk_packed_request {
    uint32_t q_first, q_rows, kv_first, kv_rows;
    uint32_t before; /* query rows of the requests before it in the plan */
};

/* hk_record.n of a plan */
enum { HK_PACKED_HEADS, HK_PACKED_KV_HEADS, HK_PACKED_DIM,
       HK_PACKED_REQUESTS, /* those with query rows */
       HK_PACKED_ROWS,     /* query rows of all requests */
       HK_PACKED_Q_END,    /* rows that the query and output tensors hold */
       HK_PACKED_KV_END };

struct hk_packed_args {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    uint64_t q_stride, kv_stride; /* elements from a row to the next */
    uint32_t heads, kv_heads, dim;
    float scale;
    const hk_packed_request *requests;
    uint32_t request_count, rows;
};

/* One wave per (query row, head), 64 keys at a time: lane j scores key j of
 * the turn, then lane l adds up dims l, l + 64, ... of the turn's values.
 * Running maximum and sum in F32; P stays F32. */
__global__ void __launch_bounds__(256) hk_packed_simple(hk_packed_args a) {
    const uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t nth = (uint32_t)(i / a.heads);
    const uint32_t head = (uint32_t)(i - (uint64_t)nth * a.heads);
    if (nth >= a.rows) return;
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
            s *= a.scale;
        }
        const float most = fmaxf(top, hk_wave_max(s));
        /* every score so far -inf: no weights yet */
        const float ref = most == -INFINITY ? 0.0f : most;
        const float keep = expf(top - ref), p = expf(s - ref);
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
        if (rows * heads > 0x7fffffffull) {
            hk_fail(gpu, "attention plan: too many query rows and heads");
            return NULL;
        }
        const size_t count = list.size();
        if (list.empty()) list.push_back({0, 0, 0, 0, 0});
        h3_gpu_tensor *plan = h3_gpu_tensor_from_u32(
            gpu, (const uint32_t *)list.data(),
            list.size() * sizeof(hk_packed_request) / 4);
        if (!plan) return NULL;
        plan->record.kind = HK_RECORD_PACKED;
        plan->record.n[HK_PACKED_HEADS] = heads;
        plan->record.n[HK_PACKED_KV_HEADS] = kv_heads;
        plan->record.n[HK_PACKED_DIM] = head_dim;
        plan->record.n[HK_PACKED_REQUESTS] = (uint32_t)count;
        plan->record.n[HK_PACKED_ROWS] = (uint32_t)rows;
        plan->record.n[HK_PACKED_Q_END] = (uint32_t)q_end;
        plan->record.n[HK_PACKED_KV_END] = (uint32_t)kv_end;
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
    a.requests = (const hk_packed_request *)plan->data;
    a.request_count = n[HK_PACKED_REQUESTS];
    a.rows = n[HK_PACKED_ROWS];
    hk_op_begin(gpu, "attention_packed");
    const uint64_t waves = (uint64_t)a.rows * heads;
    hipLaunchKernelGGL(hk_packed_simple, dim3((unsigned)((waves + 3) / 4)),
                       dim3(256), 0, gpu->stream, a);
    return hk_op_end(gpu, "attention_packed", HK_KIND_SDPA);
}

} /* extern "C" */
