/* Products of 8-bit integers with a scale for each token and output channel
 * (h3_hip_quantize_int8, _linear_int8_bf16, _mlp_int8_bf16 in h3_hip.h):
 *   y[m][n] = act(sx[m] sw[n] sum_k cx[m][k] cw[n][k] + bias[n]).
 * The sum is exact in 32 bits, so neither tiles nor pieces of K change it; what
 * rounds is its conversion to F32, the scales' product and the result.
 */
#include "hk_int8.h"
#include "hk_gemm.h"

#include <math.h>

#include <algorithm>

#define HK_INT8_THREADS 256u

/* --------------------------------------------------------- rows in 8 bits */

/* Where a row's values come from. */
enum {
    HK_ROWS_BF16,   /* the input */
    HK_ROWS_RMS,    /* RMS norm of it, weight, modulation */
    HK_ROWS_LAYER,  /* LayerNorm of it, weight and bias, modulation */
    HK_ROWS_F32,    /* F32 rows of `pitch` elements */
    HK_ROWS_SWIGLU, /* silu(g) u of F32 rows [g | u] */
};

struct hk_int8_rows_args {
    const uint16_t *input, *weight, *bias, *modulation;
    const float *wide;
    const uint32_t *row_map;
    int8_t *codes;
    float *scales;
    uint32_t rows, width, pitch, wide_pitch, slots, shift_slot, scale_slot;
    float epsilon;
};

/* silu(g) u in F32: the activation's own rounding is a few ulps, far below a
 * step of 8 bits.  Where 1 + e^-g overflows the quotient is 0, as it should
 * be. */
__device__ __forceinline__ float hk_swiglu_f(float g, float u) {
    return hk_silu_f(g) * u;
}

/* One workgroup a row, any width: the row is read again for each pass, which
 * the caches serve. */
template <int SOURCE>
__global__ void __launch_bounds__(HK_INT8_THREADS)
hk_int8_rows_any(hk_int8_rows_args a, uint32_t first) {
    __shared__ float sums[16];
    __shared__ uint32_t tops[16];
    const uint32_t row = first + blockIdx.x;
    constexpr bool norm = SOURCE == HK_ROWS_RMS || SOURCE == HK_ROWS_LAYER;
    const uint16_t *x = a.input + (size_t)row * a.width;
    const float *wide = a.wide + (size_t)row * a.wide_pitch;
    float mean = 0.0f, inverse = 1.0f;
    if (norm) {
        float sum = 0.0f;
        if (SOURCE == HK_ROWS_LAYER) {
            for (uint32_t c = threadIdx.x; c < a.width; c += HK_INT8_THREADS)
                sum += hk_bf2f(x[c]);
            mean = hk_block_sum(sum, sums) / (float)a.width;
            sum = 0.0f;
        }
        for (uint32_t c = threadIdx.x; c < a.width; c += HK_INT8_THREADS) {
            const float v = hk_bf2f(x[c]) - mean;
            sum = fmaf(v, v, sum);
        }
        inverse = 1.0f / sqrtf(hk_block_sum(sum, sums) / (float)a.width +
                               a.epsilon);
    }
    const uint16_t *shift = NULL, *scale = NULL;
    if (norm && a.modulation) {
        const size_t base = (size_t)a.row_map[row] * a.slots;
        shift = a.modulation + (base + a.shift_slot) * a.width;
        scale = a.modulation + (base + a.scale_slot) * a.width;
    }
    auto value = [&](uint32_t c) -> float {
        if (SOURCE == HK_ROWS_F32) return wide[c];
        if (SOURCE == HK_ROWS_SWIGLU)
            return hk_swiglu_f(wide[c], wide[a.width + c]);
        float v = hk_bf2f(x[c]);
        if (!norm) return v;
        v = (v - mean) * inverse;
        if (a.weight) v *= hk_bf2f(a.weight[c]);
        if (a.bias) v += hk_bf2f(a.bias[c]);
        if (shift) v = v * (1.0f + hk_bf2f(scale[c])) + hk_bf2f(shift[c]);
        return v;
    };
    uint32_t most = 0;
    for (uint32_t c = threadIdx.x; c < a.width; c += HK_INT8_THREADS)
        most = max(most, hk_magnitude(value(c)));
    const hk_int8_quantizer code(hk_block_umax(most, tops));
    int8_t *out = a.codes + (size_t)row * a.pitch;
    for (uint32_t c = threadIdx.x; c < a.pitch; c += HK_INT8_THREADS)
        out[c] = c < a.width ? (int8_t)(int)code(value(c)) : (int8_t)0;
    if (threadIdx.x == 0) a.scales[row] = code.scale;
}

__global__ void __launch_bounds__(HK_INT8_THREADS)
hk_int8_values(const int8_t *codes, const float *scales, uint16_t *out,
               uint32_t width, uint32_t pitch, uint32_t first) {
    const uint32_t row = first + blockIdx.x;
    const float scale = scales[row];
    for (uint32_t c = threadIdx.x; c < width; c += HK_INT8_THREADS)
        out[(size_t)row * width + c] =
            hk_f2bf((float)codes[(size_t)row * pitch + c] * scale);
}

/* A launch has fewer than 2^32 threads. */
template <typename F>
static void hk_int8_each_rows(uint32_t rows, F launch) {
    const uint32_t most = 1u << 23;
    for (uint32_t first = 0; first < rows; first += std::min(rows - first, most))
        launch(first, std::min(rows - first, most));
}

template <int SOURCE>
static void hk_int8_rows(struct h3_gpu *gpu, const hk_int8_rows_args &a) {
    hk_int8_each_rows(a.rows, [&](uint32_t first, uint32_t rows) {
        hipLaunchKernelGGL(hk_int8_rows_any<SOURCE>, dim3(rows),
                           dim3(HK_INT8_THREADS), 0, gpu->stream, a, first);
    });
}

/* ------------------------------------------------------------ the products */

/* What is made of the sums: act(acc sx sw + bias).  The scales are multiplied
 * first: their product with the sum passes F32's range only where the result
 * does. */
__device__ __forceinline__ float hk_int8_value(int acc, float sx, float sw) {
    return (float)acc * (sx * sw);
}

/* One thread per output: H3_HIP_REFERENCE=1.  `wide` or `out`. */
__global__ void __launch_bounds__(256)
hk_int8_simple(const int8_t *x, const float *xs, const int8_t *w,
               const float *ws, const uint16_t *bias, uint16_t *out,
               float *wide, uint32_t n, uint32_t pitch, int gelu,
               uint32_t first) {
    const uint32_t col = blockIdx.x * 256u + threadIdx.x;
    const size_t row = (size_t)first + blockIdx.y;
    if (col >= n) return;
    const int4 *xr = (const int4 *)(x + row * pitch);
    const int4 *wr = (const int4 *)(w + (size_t)col * pitch);
    int sum = 0;
    for (uint32_t i = 0; i < pitch / 16u; i++) {
        const int4 a = xr[i], b = wr[i];
        sum = __builtin_amdgcn_sdot4(a.x, b.x, sum, false);
        sum = __builtin_amdgcn_sdot4(a.y, b.y, sum, false);
        sum = __builtin_amdgcn_sdot4(a.z, b.z, sum, false);
        sum = __builtin_amdgcn_sdot4(a.w, b.w, sum, false);
    }
    float y = hk_int8_value(sum, xs[row], ws[col]);
    if (bias) y += hk_bf2f(bias[col]);
    if (gelu) y = hk_gelu_tanh_f(y);
    if (wide) wide[row * n + col] = y;
    else out[row * n + col] = hk_f2bf(y);
}

/* Rows in 8 bits. */
struct hk_int8_matrix {
    const int8_t *codes;
    const float *scales;
    uint32_t rows, pitch;
};

static hk_int8_matrix hk_int8_of(const h3_gpu_tensor *t, uint32_t rows) {
    return {hk_int8_codes(t), hk_int8_scales(t), rows,
            t->record.n[HK_INT8_PITCH]};
}

static void hk_int8_simple_run(struct h3_gpu *gpu, const hk_int8_matrix &x,
                               const hk_int8_matrix &w, const uint16_t *bias,
                               uint16_t *out, float *wide, int gelu) {
    for (uint32_t first = 0; first < x.rows; first += 32768u)
        hipLaunchKernelGGL(hk_int8_simple,
                           dim3((w.rows + 255u) / 256u,
                                std::min(x.rows - first, 32768u)),
                           dim3(256), 0, gpu->stream, x.codes, x.scales,
                           w.codes, w.scales, bias, out, wide, w.rows,
                           x.pitch, gelu, first);
}

/* bf16 rows of x . w^T. */
static int hk_int8_linear(struct h3_gpu *gpu, const hk_int8_matrix &x,
                          const hk_int8_matrix &w, const uint16_t *bias,
                          uint16_t *out, int gelu) {
    hk_int8_simple_run(gpu, x, w, bias, out, NULL, gelu);
    return 1;
}

/* ================================================================ ops */

extern "C" {

h3_gpu_tensor *h3_hip_int8_new(h3_gpu *gpu, uint32_t rows, uint32_t columns) {
    if (!gpu) return NULL;
    if (!rows || !columns || columns > HK_INT8_MOST_COLUMNS) {
        hk_fail(gpu, "8-bit matrix of %u rows and %u columns (1 row at least, "
                     "1 to %u columns)", rows, columns, HK_INT8_MOST_COLUMNS);
        return NULL;
    }
    const uint32_t pitch =
        (columns + HK_INT8_LINE - 1u) / HK_INT8_LINE * HK_INT8_LINE;
    h3_gpu_tensor *t = h3_gpu_tensor_new_i8(
        gpu, (size_t)rows * pitch + ((size_t)rows + 255u) / 256u * 1024u);
    if (!t) return NULL;
    t->record.kind = HK_RECORD_INT8;
    t->record.n[HK_INT8_ROWS] = rows;
    t->record.n[HK_INT8_COLUMNS] = columns;
    t->record.n[HK_INT8_PITCH] = pitch;
    return t;
}

int h3_hip_quantize_int8(h3_gpu *gpu, h3_gpu_tensor *output,
                         const h3_gpu_tensor *input, uint32_t rows,
                         uint32_t columns) {
    if (!hk_int8_require(gpu, output, rows, columns, "quantize output") ||
        !hk_require(gpu, input, (size_t)rows * columns, H3_GPU_BF16,
                    "quantize input") ||
        !hk_require_active(gpu))
        return 0;
    if (!rows) return 1;
    hk_op_begin(gpu, "quantize_int8");
    hk_int8_rows_args a = {};
    a.input = HK_CBF16(input);
    a.codes = (int8_t *)output->data;
    a.scales = hk_int8_scales(output);
    a.rows = rows;
    a.width = columns;
    a.pitch = output->record.n[HK_INT8_PITCH];
    hk_int8_rows<HK_ROWS_BF16>(gpu, a);
    return hk_op_end(gpu, "quantize_int8", HK_KIND_DIRECT);
}

static int hk_int8_adaln(h3_gpu *gpu, h3_gpu_tensor *output,
                         const h3_gpu_tensor *input,
                         const h3_gpu_tensor *norm_weight,
                         const h3_gpu_tensor *norm_bias,
                         const h3_gpu_tensor *modulation,
                         const h3_gpu_tensor *row_map, uint32_t rows,
                         uint32_t width, uint32_t slots, uint32_t shift_slot,
                         uint32_t scale_slot, float epsilon, bool layer) {
    /* as of h3_gpu_adaln_bf16 and h3_gpu_layer_adaln_bf16, the row map's
     * entries are the caller's to keep within the modulation */
    if (!hk_int8_require(gpu, output, rows, width, "adaLN output") ||
        !hk_require(gpu, input, (size_t)rows * width, H3_GPU_BF16,
                    "adaLN input") ||
        ((norm_weight || !layer) &&
         !hk_require(gpu, norm_weight, width, H3_GPU_BF16,
                     "adaLN weight")) ||
        (norm_bias && !hk_require(gpu, norm_bias, width, H3_GPU_BF16,
                                  "adaLN bias")) ||
        ((modulation || !layer) &&
         (!hk_require(gpu, modulation, (size_t)slots * width, H3_GPU_BF16,
                      "adaLN modulation") ||
          !hk_require(gpu, row_map, rows, H3_GPU_U32, "adaLN row map"))) ||
        !hk_require_active(gpu))
        return 0;
    if (modulation && (shift_slot >= slots || scale_slot >= slots))
        return hk_fail(gpu, "adaLN modulation slot out of range");
    if (!rows) return 1;
    const char *name = layer ? "layer_adaln_int8" : "adaln_int8";
    hk_op_begin(gpu, name);
    hk_int8_rows_args a = {};
    a.input = HK_CBF16(input);
    a.weight = norm_weight ? HK_CBF16(norm_weight) : NULL;
    a.bias = norm_bias ? HK_CBF16(norm_bias) : NULL;
    a.modulation = modulation ? HK_CBF16(modulation) : NULL;
    a.row_map = modulation ? HK_CU32(row_map) : NULL;
    a.codes = (int8_t *)output->data;
    a.scales = hk_int8_scales(output);
    a.rows = rows;
    a.width = width;
    a.pitch = output->record.n[HK_INT8_PITCH];
    a.slots = slots;
    a.shift_slot = shift_slot;
    a.scale_slot = scale_slot;
    a.epsilon = epsilon;
    if (layer) hk_int8_rows<HK_ROWS_LAYER>(gpu, a);
    else hk_int8_rows<HK_ROWS_RMS>(gpu, a);
    return hk_op_end(gpu, name, HK_KIND_DIRECT);
}

int h3_hip_adaln_int8(h3_gpu *gpu, h3_gpu_tensor *output,
                      const h3_gpu_tensor *input,
                      const h3_gpu_tensor *norm_weight,
                      const h3_gpu_tensor *modulation,
                      const h3_gpu_tensor *row_map, uint32_t rows,
                      uint32_t width, uint32_t slots, uint32_t shift_slot,
                      uint32_t scale_slot, float epsilon) {
    return hk_int8_adaln(gpu, output, input, norm_weight, NULL, modulation,
                         row_map, rows, width, slots, shift_slot, scale_slot,
                         epsilon, false);
}

int h3_hip_layer_adaln_int8(h3_gpu *gpu, h3_gpu_tensor *output,
                            const h3_gpu_tensor *input,
                            const h3_gpu_tensor *norm_weight,
                            const h3_gpu_tensor *norm_bias,
                            const h3_gpu_tensor *modulation,
                            const h3_gpu_tensor *row_map, uint32_t rows,
                            uint32_t width, uint32_t slots,
                            uint32_t shift_slot, uint32_t scale_slot,
                            float epsilon) {
    return hk_int8_adaln(gpu, output, input, norm_weight, norm_bias,
                         modulation, row_map, rows, width, slots, shift_slot,
                         scale_slot, epsilon, true);
}

int h3_hip_dequantize_int8(h3_gpu *gpu, h3_gpu_tensor *output,
                           const h3_gpu_tensor *input, uint32_t rows,
                           uint32_t columns) {
    if (!hk_int8_require(gpu, input, rows, columns, "dequantize input") ||
        !hk_require(gpu, output, (size_t)rows * columns, H3_GPU_BF16,
                    "dequantize output") ||
        !hk_require_active(gpu))
        return 0;
    if (!rows) return 1;
    hk_op_begin(gpu, "dequantize_int8");
    hk_int8_each_rows(rows, [&](uint32_t first, uint32_t count) {
        hipLaunchKernelGGL(hk_int8_values, dim3(count), dim3(HK_INT8_THREADS),
                           0, gpu->stream, hk_int8_codes(input),
                           hk_int8_scales(input), HK_BF16(output), columns,
                           input->record.n[HK_INT8_PITCH], first);
    });
    return hk_op_end(gpu, "dequantize_int8", HK_KIND_DIRECT);
}

static int hk_int8_linear_op(h3_gpu *gpu, h3_gpu_tensor *output,
                             const h3_gpu_tensor *input,
                             const h3_gpu_tensor *weight,
                             const h3_gpu_tensor *bias, uint32_t rows,
                             uint32_t input_dim, uint32_t output_dim,
                             int gelu) {
    if (!hk_int8_require(gpu, input, rows, input_dim, "8-bit linear input") ||
        !hk_int8_require(gpu, weight, output_dim, input_dim,
                         "8-bit linear weight") ||
        !hk_require(gpu, output, (size_t)rows * output_dim, H3_GPU_BF16,
                    "8-bit linear output") ||
        (bias && !hk_require(gpu, bias, output_dim, H3_GPU_BF16,
                             "8-bit linear bias")) ||
        !hk_require_active(gpu))
        return 0;
    if (output == bias)
        return hk_fail(gpu, "8-bit linear: the output must be a tensor of its "
                            "own");
    if (!rows || !output_dim) return 1;
    const char *name = gelu ? "gemm_int8_gelu" : "gemm_int8";
    hk_op_begin(gpu, name);
    if (!hk_int8_linear(gpu, hk_int8_of(input, rows),
                        hk_int8_of(weight, output_dim),
                        bias ? HK_CBF16(bias) : NULL, HK_BF16(output), gelu))
        return 0;
    return hk_op_end(gpu, name, HK_KIND_LINEAR);
}

int h3_hip_linear_int8_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                            const h3_gpu_tensor *input,
                            const h3_gpu_tensor *weight,
                            const h3_gpu_tensor *bias, uint32_t rows,
                            uint32_t input_dim, uint32_t output_dim) {
    return hk_int8_linear_op(gpu, output, input, weight, bias, rows, input_dim,
                             output_dim, 0);
}

int h3_hip_linear_gelu_int8_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                                 const h3_gpu_tensor *input,
                                 const h3_gpu_tensor *weight,
                                 const h3_gpu_tensor *bias, uint32_t rows,
                                 uint32_t input_dim, uint32_t output_dim) {
    return hk_int8_linear_op(gpu, output, input, weight, bias, rows, input_dim,
                             output_dim, 1);
}

int h3_hip_mlp_int8_bf16(h3_gpu *gpu, h3_gpu_tensor *output,
                         const h3_gpu_tensor *input,
                         const h3_gpu_tensor *fc1_weight,
                         const h3_gpu_tensor *fc2_weight, uint32_t rows,
                         uint32_t input_dim, uint32_t hidden_dim,
                         uint32_t output_dim) {
    if (!hidden_dim || hidden_dim > HK_INT8_MOST_COLUMNS)
        return hk_fail(gpu, "8-bit MLP: %u hidden columns (1 to %u)",
                       hidden_dim, HK_INT8_MOST_COLUMNS);
    if (!hk_int8_require(gpu, input, rows, input_dim, "8-bit MLP input") ||
        !hk_int8_require(gpu, fc1_weight, 2 * hidden_dim, input_dim,
                         "8-bit MLP fc1 weight") ||
        !hk_int8_require(gpu, fc2_weight, output_dim, hidden_dim,
                         "8-bit MLP fc2 weight") ||
        !hk_require(gpu, output, (size_t)rows * output_dim, H3_GPU_BF16,
                    "8-bit MLP output") ||
        !hk_require_active(gpu))
        return 0;
    if (!rows || !output_dim) return 1;
    /* F32 rows of the first product, then h in 8 bits */
    const uint32_t pitch = fc2_weight->record.n[HK_INT8_PITCH];
    const size_t wide_bytes =
        ((size_t)rows * 2 * hidden_dim * 4 + 255) & ~(size_t)255;
    const size_t code_bytes = (size_t)rows * pitch;
    uint8_t *space = (uint8_t *)hk_workspace(
        gpu, wide_bytes + code_bytes + ((size_t)rows + 255u) / 256u * 1024u);
    if (!space) return 0;
    hk_int8_matrix h = {(int8_t *)(space + wide_bytes),
                        (float *)(space + wide_bytes + code_bytes), rows,
                        pitch};
    hk_op_begin(gpu, "gemm_int8_swiglu");
    hk_int8_rows_args a = {};
    a.wide = (float *)space;
    a.codes = (int8_t *)h.codes;
    a.scales = (float *)h.scales;
    a.rows = rows;
    a.width = hidden_dim;
    a.pitch = pitch;
    a.wide_pitch = 2 * hidden_dim;
    hk_int8_simple_run(gpu, hk_int8_of(input, rows),
                       hk_int8_of(fc1_weight, 2 * hidden_dim), NULL, NULL,
                       (float *)space, 0);
    hk_int8_rows<HK_ROWS_SWIGLU>(gpu, a);
    if (!hk_op_end(gpu, "gemm_int8_swiglu", HK_KIND_LINEAR)) return 0;
    hk_op_begin(gpu, "gemm_int8");
    if (!hk_int8_linear(gpu, h, hk_int8_of(fc2_weight, output_dim), NULL,
                        HK_BF16(output), 0))
        return 0;
    return hk_op_end(gpu, "gemm_int8", HK_KIND_LINEAR);
}

} /* extern "C" */
