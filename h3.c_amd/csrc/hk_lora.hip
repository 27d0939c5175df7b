/* Low-rank adapters of several requests beside one projection:
 *   y[r] = act(x[r] . W^T + b + s_a (x[r] . A_a^T) . B_a^T),  a = map[r]
 * (h3_hip_linear_lora_bf16 and its GELU form in h3_hip.h).
 *
 * The adapters live in a table built once: per adapter one entry, then its A
 * (the down projection, [rank][K]) and B (the up projection, [N][rank]), with
 * the rank padded by zeros to a multiple of 8, so that B's rows are whole
 * 16-byte pieces for any rank.
 *
 * The simple kernels here (one wave per element of x . A^T, one thread per
 * output, sums in sequence) serve H3_HIP_REFERENCE=1 and the shapes that the
 * matrix-core kernels do not take.
 */
#include "hk_common.h"
#include "hk_gemm.h"
#include "hk_internal.h"

#include <math.h>
#include <stdlib.h>

/* one adapter of a table, in device memory */
struct hk_lora_entry {
    const uint16_t *down; /* [padded][K] */
    const uint16_t *up;   /* [N][padded] */
    uint32_t rank, padded;
    float scale;
    uint32_t bad; /* set by hk_lora_pack: an element is not finite */
};

#define HK_LORA_MAX_RANK 1024u

/* hk_record.n of a table */
enum { HK_LORA_IN, HK_LORA_OUT, HK_LORA_COUNT, HK_LORA_PADDED /* largest */ };

struct hk_lora_args {
    const uint16_t *x, *w, *bias;
    uint16_t *c;
    uint32_t m, n, k;
    const hk_lora_entry *entries;
    uint32_t count;
    const uint32_t *map;
    /* s_a x . A_a^T: F32 [rows][pitch] for the simple kernels */
    float *low;
    uint32_t pitch;
    int gelu;
};

/* Copies a [rows][cols] matrix into [rows][pitch] with zeros behind each row,
 * and rows of zeros behind the last, up to `count` elements. */
__global__ void __launch_bounds__(256)
hk_lora_pack(const uint16_t *src, uint16_t *dst, uint32_t rows, uint32_t cols,
             uint32_t pitch, uint64_t count, hk_lora_entry *entry) {
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= count) return;
    const uint64_t r = i / pitch;
    const uint32_t c = (uint32_t)(i - r * pitch);
    const uint16_t v = r < rows && c < cols ? src[r * cols + c] : (uint16_t)0;
    dst[i] = v;
    if ((v & 0x7f80u) == 0x7f80u) entry->bad = 1; /* every writer writes 1 */
}

/* low[r][j] = s_a x[r] . A_a[j]: one wave an element. */
__global__ void __launch_bounds__(256) hk_lora_low_simple(hk_lora_args g) {
    const uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(i / g.pitch);
    const uint32_t j = (uint32_t)(i - (uint64_t)row * g.pitch);
    if (row >= g.m) return;
    const uint32_t a = g.map[row];
    if (a >= g.count) return;
    const hk_lora_entry e = g.entries[a];
    if (j >= e.rank) return;
    const uint16_t *x = g.x + (size_t)row * g.k;
    const uint16_t *down = e.down + (size_t)j * g.k;
    float sum = 0.0f;
    for (uint32_t k = threadIdx.x & 63u; k < g.k; k += 64u)
        sum = fmaf(hk_bf2f(x[k]), hk_bf2f(down[k]), sum);
    sum = hk_wave_sum(sum);
    if ((threadIdx.x & 63u) == 0) g.low[i] = e.scale * sum;
}

/* One thread an output: the shared product, then the adapter's. */
__global__ void __launch_bounds__(256) hk_lora_simple(hk_lora_args g) {
    const uint32_t col = blockIdx.x * 256u + threadIdx.x;
    const uint32_t row = blockIdx.y + blockIdx.z * 65535u;
    if (row >= g.m || col >= g.n) return;
    float sum = g.bias ? hk_bf2f(g.bias[col]) : 0.0f;
    const uint16_t *x = g.x + (size_t)row * g.k;
    const uint16_t *w = g.w + (size_t)col * g.k;
    for (uint32_t k = 0; k < g.k; k++)
        sum = fmaf(hk_bf2f(x[k]), hk_bf2f(w[k]), sum);
    const uint32_t a = g.map[row];
    if (a < g.count) {
        const hk_lora_entry e = g.entries[a];
        const float *low = g.low + (size_t)row * g.pitch;
        const uint16_t *up = e.up + (size_t)col * e.padded;
        for (uint32_t j = 0; j < e.rank; j++)
            sum = fmaf(low[j], hk_bf2f(up[j]), sum);
    }
    if (g.gelu) sum = hk_gelu_tanh_f(hk_bf2f(hk_f2bf(sum)));
    g.c[(size_t)row * g.n + col] = hk_f2bf(sum);
}

static int hk_lora_run_simple(struct h3_gpu *gpu, hk_lora_args &g) {
    if (g.pitch) {
        g.low = (float *)hk_workspace(gpu, (size_t)g.m * g.pitch * 4);
        if (!g.low) return 0;
        const uint64_t waves = (uint64_t)g.m * g.pitch;
        if ((waves + 3) / 4 > 0x7fffffffull)
            return hk_fail(gpu, "linear with adapters: too many rows");
        hipLaunchKernelGGL(hk_lora_low_simple, dim3((waves + 3) / 4),
                           dim3(256), 0, gpu->stream, g);
    }
    hipLaunchKernelGGL(hk_lora_simple,
                       dim3((g.n + 255) / 256, g.m < 65535u ? g.m : 65535u,
                            (g.m + 65534u) / 65535u),
                       dim3(256), 0, gpu->stream, g);
    return 1;
}

extern "C" {

h3_gpu_tensor *h3_hip_lora_table(h3_gpu *gpu,
                                 const h3_gpu_tensor *const *down,
                                 const h3_gpu_tensor *const *up,
                                 const uint32_t *ranks, const float *scales,
                                 uint32_t count, uint32_t input_dim,
                                 uint32_t output_dim) {
    if (!gpu) return NULL;
    if (!count || !down || !up || !ranks || !scales || !input_dim ||
        !output_dim) {
        hk_fail(gpu, "adapter table needs at least one adapter and its sizes");
        return NULL;
    }
    /* entries, then each adapter's A and B from a 256-byte boundary on */
    const size_t head = ((size_t)count * sizeof(hk_lora_entry) + 255) &
                        ~(size_t)255;
    size_t bytes = head;
    uint32_t largest = 0;
    for (uint32_t a = 0; a < count; a++) {
        if (ranks[a] > HK_LORA_MAX_RANK) {
            hk_fail(gpu, "adapter %u: rank %u is over %u", a, ranks[a],
                    HK_LORA_MAX_RANK);
            return NULL;
        }
        if (!isfinite(scales[a])) {
            hk_fail(gpu, "adapter %u: the scale is not finite", a);
            return NULL;
        }
        if (ranks[a] &&
            (!hk_require(gpu, down[a], (size_t)ranks[a] * input_dim,
                         H3_GPU_BF16, "adapter down") ||
             !hk_require(gpu, up[a], (size_t)ranks[a] * output_dim,
                         H3_GPU_BF16, "adapter up")))
            return NULL;
        const uint32_t padded = (ranks[a] + 7u) & ~7u;
        if (padded > largest) largest = padded;
        bytes += ((size_t)padded * input_dim * 2 + 255) & ~(size_t)255;
        bytes += ((size_t)padded * output_dim * 2 + 255) & ~(size_t)255;
    }
    hk_lora_entry *entries =
        (hk_lora_entry *)calloc(count, sizeof(hk_lora_entry));
    if (!entries) {
        hk_fail(gpu, "out of host memory");
        return NULL;
    }
    h3_gpu_tensor *table = h3_gpu_tensor_from_u32(gpu, NULL, bytes / 4);
    if (!table) {
        free(entries);
        return NULL;
    }
    hk_lora_entry *device = (hk_lora_entry *)table->data;
    uint8_t *at = (uint8_t *)table->data + head;
    for (uint32_t a = 0; a < count; a++) {
        hk_lora_entry &e = entries[a];
        e.rank = ranks[a];
        e.padded = (ranks[a] + 7u) & ~7u;
        e.scale = scales[a];
        if (!e.rank) continue;
        e.down = (const uint16_t *)at;
        at += ((size_t)e.padded * input_dim * 2 + 255) & ~(size_t)255;
        e.up = (const uint16_t *)at;
        at += ((size_t)e.padded * output_dim * 2 + 255) & ~(size_t)255;
    }
    const size_t entry_bytes = (size_t)count * sizeof(hk_lora_entry);
    hipError_t status = hipMemcpyAsync(device, entries, entry_bytes,
                                       hipMemcpyHostToDevice, gpu->stream);
    for (uint32_t a = 0; a < count && status == hipSuccess; a++) {
        const hk_lora_entry &e = entries[a];
        if (!e.rank) continue;
        const uint64_t d = (uint64_t)e.padded * input_dim;
        const uint64_t u = (uint64_t)e.padded * output_dim;
        hipLaunchKernelGGL(hk_lora_pack, dim3((unsigned)((d + 255) / 256)),
                           dim3(256), 0, gpu->stream, HK_CBF16(down[a]),
                           (uint16_t *)e.down, e.rank, input_dim, input_dim,
                           d, device + a);
        hipLaunchKernelGGL(hk_lora_pack, dim3((unsigned)((u + 255) / 256)),
                           dim3(256), 0, gpu->stream, HK_CBF16(up[a]),
                           (uint16_t *)e.up, output_dim, e.rank, e.padded, u,
                           device + a);
        status = hipGetLastError();
    }
    if (status == hipSuccess)
        status = hipMemcpyAsync(entries, device, entry_bytes,
                                hipMemcpyDeviceToHost, gpu->stream);
    /* the adapters may be freed once this returns */
    const hipError_t done = hipStreamSynchronize(gpu->stream);
    if (status == hipSuccess) status = done;
    uint32_t bad = count;
    for (uint32_t a = count; a-- > 0;)
        if (entries[a].bad) bad = a;
    free(entries);
    if (status != hipSuccess || bad < count) {
        if (status != hipSuccess)
            hk_fail_hip(gpu, "adapter table", status);
        else
            hk_fail(gpu, "adapter %u holds values that are not finite", bad);
        h3_gpu_tensor_free(table);
        return NULL;
    }
    table->record.kind = HK_RECORD_LORA;
    table->record.n[HK_LORA_IN] = input_dim;
    table->record.n[HK_LORA_OUT] = output_dim;
    table->record.n[HK_LORA_COUNT] = count;
    table->record.n[HK_LORA_PADDED] = largest;
    return table;
}

static int hk_linear_lora(h3_gpu *gpu, h3_gpu_tensor *output,
                          const h3_gpu_tensor *input,
                          const h3_gpu_tensor *weight,
                          const h3_gpu_tensor *bias,
                          const h3_gpu_tensor *table,
                          const h3_gpu_tensor *adapter_map, uint32_t rows,
                          uint32_t input_dim, uint32_t output_dim, int gelu) {
    if (!hk_require(gpu, input, (size_t)rows * input_dim, H3_GPU_BF16,
                    "linear input") ||
        !hk_require(gpu, weight, (size_t)output_dim * input_dim, H3_GPU_BF16,
                    "linear weight") ||
        !hk_require(gpu, output, (size_t)rows * output_dim, H3_GPU_BF16,
                    "linear output") ||
        (bias && !hk_require(gpu, bias, output_dim, H3_GPU_BF16,
                             "linear bias")) ||
        !hk_require(gpu, adapter_map, rows, H3_GPU_U32, "adapter map") ||
        !hk_require_active(gpu))
        return 0;
    if (!table || table->record.kind != HK_RECORD_LORA)
        return hk_fail(gpu, "linear with adapters: the table was not built "
                            "by h3_hip_lora_table");
    if (input_dim != table->record.n[HK_LORA_IN] ||
        output_dim != table->record.n[HK_LORA_OUT])
        return hk_fail(gpu, "linear with adapters: %u to %u differs from the "
                            "table's %u to %u", input_dim, output_dim,
                       table->record.n[HK_LORA_IN],
                       table->record.n[HK_LORA_OUT]);
    if (output == input || output == weight || output == bias ||
        output == adapter_map || output == table)
        return hk_fail(gpu, "linear with adapters: the output must be a "
                            "tensor of its own");
    if (!rows) return 1;
    hk_lora_args g = {};
    g.x = HK_CBF16(input);
    g.w = HK_CBF16(weight);
    g.bias = bias ? HK_CBF16(bias) : NULL;
    g.c = HK_BF16(output);
    g.m = rows; g.n = output_dim; g.k = input_dim;
    g.entries = (const hk_lora_entry *)table->data;
    g.count = table->record.n[HK_LORA_COUNT];
    g.pitch = table->record.n[HK_LORA_PADDED];
    g.map = HK_CU32(adapter_map);
    g.gelu = gelu;
    const char *name = gelu ? "gemm_lora_gelu" : "gemm_lora";
    hk_op_begin(gpu, name);
    if (!hk_lora_run_simple(gpu, g)) return 0;
    return hk_op_end(gpu, name, HK_KIND_LINEAR);
}

int h3_hip_linear_lora_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                            const h3_gpu_tensor *input,
                            const h3_gpu_tensor *weight,
                            const h3_gpu_tensor *bias,
                            const h3_gpu_tensor *table,
                            const h3_gpu_tensor *adapter_map, uint32_t rows,
                            uint32_t input_dim, uint32_t output_dim) {
    return hk_linear_lora(gpu, output, input, weight, bias, table,
                          adapter_map, rows, input_dim, output_dim, 0);
}

int h3_hip_linear_lora_gelu_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                                 const h3_gpu_tensor *input,
                                 const h3_gpu_tensor *weight,
                                 const h3_gpu_tensor *bias,
                                 const h3_gpu_tensor *table,
                                 const h3_gpu_tensor *adapter_map,
                                 uint32_t rows, uint32_t input_dim,
                                 uint32_t output_dim) {
    return hk_linear_lora(gpu, output, input, weight, bias, table,
                          adapter_map, rows, input_dim, output_dim, 1);
}

} /* extern "C" */
