/* Products of 8-bit integers with a scale for each token and output channel
 * (h3_hip_quantize_int8, _linear_int8_bf16, _mlp_int8_bf16 in h3_hip.h):
 *   y[m][n] = act(sx[m] sw[n] sum_k cx[m][k] cw[n][k] + bias[n]).
 * The sum is exact in 32 bits, so neither tiles nor pieces of K change it; what
 * rounds is its conversion to F32, the scales' product and the result.
 */
#include "hk_int8.h"
#include "hk_gemm.h"
#include "hk_skinny.h"
#include "hk_skinny_tile.h"

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
    HK_ROWS_SWIGLU, /* silu(g) u of F32 rows [g | u], of the simple kernel */
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
    const hk_int8_quantizer code(
        hk_block_umax(most, tops, HK_INT8_THREADS / 64u));
    int8_t *out = a.codes + (size_t)row * a.pitch;
    for (uint32_t c = threadIdx.x; c < a.pitch; c += HK_INT8_THREADS)
        out[c] = c < a.width ? (int8_t)(int)code(value(c)) : (int8_t)0;
    if (threadIdx.x == 0) a.scales[row] = code.scale;
}

/* Elements [col, + 8) of a row, zeros behind its end.  EIGHTS: the width is a
 * multiple of 8, and behind the end stands whatever else the row has.  There is
 * no branch then, behind which a load would wait for those before (4756 x 14336
 * in bf16 31 us for 35, behind an RMS norm 45 for 64). */
template <bool EIGHTS>
__device__ __forceinline__ uint4 hk_int8_piece(const uint16_t *row,
                                               uint32_t col, uint32_t width) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (EIGHTS || col + 8u <= width) {
        __builtin_memcpy(&v, row + (EIGHTS ? min(col, width - 8u) : col),
                         16); /* rows of odd widths: not aligned */
    } else if (col < width) {
        uint32_t w[4] = {};
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++)
            if (col + i < width)
                w[i >> 1] |= (uint32_t)row[col + i] << (16u * (i & 1u));
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

template <bool EIGHTS>
__device__ __forceinline__ void hk_int8_piece(const float *row, uint32_t col,
                                              uint32_t width, float *to) {
    if (EIGHTS || col + 8u <= width) {
        __builtin_memcpy(to, row + (EIGHTS ? min(col, width - 8u) : col), 32);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++)
            to[i] = col + i < width ? row[col + i] : 0.0f;
    }
}

/* The same with the row in registers, 8 columns a thread and chunk: at most
 * CHUNKS * THREADS * 8 columns.  One pass over the row, bound by HBM: 4756 rows
 * of 14336 in F32 67 us (5.1 TB/s), 6144 x 5120 in bf16 16 us (5.9 TB/s); a row
 * alone by its chain of loads, maximum and codes, 2.1 us. */
template <int SOURCE, int CHUNKS, int THREADS, bool EIGHTS>
__global__ void __launch_bounds__(THREADS)
hk_int8_rows_vec(hk_int8_rows_args a, uint32_t first) {
    __shared__ float sums[16];
    __shared__ uint32_t tops[16];
    const uint32_t row = first + blockIdx.x;
    constexpr bool norm = SOURCE == HK_ROWS_RMS || SOURCE == HK_ROWS_LAYER;
    constexpr bool layer = SOURCE == HK_ROWS_LAYER;
    auto column = [](int c) {
        return (threadIdx.x + (uint32_t)c * THREADS) * 8u;
    };
    float v[CHUNKS][8];
    if (SOURCE == HK_ROWS_F32) {
        const float *from = a.wide + (size_t)row * a.wide_pitch;
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
            hk_int8_piece<EIGHTS>(from, column(c), a.width, v[c]);
        if (EIGHTS) {
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
                if (column(c) >= a.width) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[c][i] = 0.0f;
                }
        }
    } else {
        const uint16_t *from = a.input + (size_t)row * a.width;
        uint4 raw[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
            raw[c] = hk_int8_piece<EIGHTS>(from, column(c), a.width);
        const uint16_t *shift = NULL, *scale = NULL;
        if (norm && a.modulation) {
            const size_t base = (size_t)a.row_map[row] * a.slots;
            shift = a.modulation + (base + a.shift_slot) * a.width;
            scale = a.modulation + (base + a.scale_slot) * a.width;
        }
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            hk_unpack8(raw[c], v[c]);
            if (EIGHTS && column(c) >= a.width) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[c][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
                sum += layer ? v[c][i] : v[c][i] * v[c][i];
        }
        if (norm) {
            const float mean =
                layer ? hk_block_sum(sum, sums) / (float)a.width : 0.0f;
            if (layer) {
                sum = 0.0f;
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        v[c][i] -= mean;
                        if (column(c) + (EIGHTS ? 0 : i) < a.width)
                            sum = fmaf(v[c][i], v[c][i], sum);
                    }
            }
            const float inverse =
                1.0f / sqrtf(hk_block_sum(sum, sums) / (float)a.width +
                             a.epsilon);
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                float w[8], b[8];
                uint4 weight, bias, scales, shifts; /* on their way at once */
                auto load = [&](uint4 &to, const uint16_t *from) {
                    to = hk_int8_piece<EIGHTS>(from, column(c), a.width);
                };
                if (a.weight) load(weight, a.weight);
                if (layer && a.bias) load(bias, a.bias);
                if (shift) {
                    load(scales, scale);
                    load(shifts, shift);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) v[c][i] *= inverse;
                if (a.weight) {
                    hk_unpack8(weight, w);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[c][i] *= w[i];
                }
                if (layer && a.bias) {
                    hk_unpack8(bias, b);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[c][i] += b[i];
                }
                if (shift) {
                    hk_unpack8(scales, w);
                    hk_unpack8(shifts, b);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        v[c][i] = v[c][i] * (1.0f + w[i]) + b[i];
                }
                /* past the row's end, whatever came of it */
                if (column(c) + 8u > a.width) {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++)
                        if (EIGHTS || column(c) + i >= a.width)
                            v[c][i] = 0.0f;
                }
            }
        }
    }
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, hk_magnitude(v[c][i]));
    const hk_int8_quantizer code(hk_block_umax(most, tops, THREADS / 64u));
    int8_t *out = a.codes + (size_t)row * a.pitch;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
        /* zeros from the row's end to that of its last line */
        const uint32_t col = column(c);
        if (col < a.pitch)
            *(uint2 *)(out + col) = make_uint2(
                hk_int8_pack4(code(v[c][0]), code(v[c][1]), code(v[c][2]),
                              code(v[c][3])),
                hk_int8_pack4(code(v[c][4]), code(v[c][5]), code(v[c][6]),
                              code(v[c][7])));
    }
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

typedef void (*hk_int8_rows_kernel)(hk_int8_rows_args, uint32_t);

template <int SOURCE, bool EIGHTS>
static hk_int8_rows_kernel hk_int8_rows_pick(bool few, uint32_t pitch) {
    if (few)
        return pitch <= 8192u ? hk_int8_rows_vec<SOURCE, 1, 1024, EIGHTS>
                              : hk_int8_rows_vec<SOURCE, 2, 1024, EIGHTS>;
    return pitch <= 2048u   ? hk_int8_rows_vec<SOURCE, 1, 256, EIGHTS>
           : pitch <= 6144u ? hk_int8_rows_vec<SOURCE, 3, 256, EIGHTS>
                            : hk_int8_rows_vec<SOURCE, 8, 256, EIGHTS>;
}

/* A row's threads: where there are few rows, more of them, as there is nothing
 * else to hide a row's latency (one row of 14336: 6.4 us with 256). */
template <int SOURCE>
static void hk_int8_rows(struct h3_gpu *gpu, const hk_int8_rows_args &a) {
    const bool few = a.rows <= 512u && a.pitch > 2048u;
    const bool any = SOURCE == HK_ROWS_SWIGLU || a.pitch > 16384u ||
                     gpu->reference_kernels;
    hk_int8_rows_kernel kernel = hk_int8_rows_any<SOURCE>;
    if constexpr (SOURCE != HK_ROWS_SWIGLU) {
        if (!any)
            kernel = a.width % 8u == 0u
                         ? hk_int8_rows_pick<SOURCE, true>(few, a.pitch)
                         : hk_int8_rows_pick<SOURCE, false>(few, a.pitch);
    }
    const uint32_t threads = few && !any ? 1024u : 256u;
    hk_int8_each_rows(a.rows, [&](uint32_t first, uint32_t rows) {
        hipLaunchKernelGGL(kernel, dim3(rows), dim3(threads), 0, gpu->stream,
                           a, first);
    });
}

/* ------------------------------------------------------------ the products */

/* What is made of the sums: acc sx sw + bias, in every kernel with the same
 * roundings.  The scales are multiplied first: their product with the sum
 * passes F32's range only where the result does.  -0 is no bias: x + -0 is
 * x. */
__device__ __forceinline__ float hk_int8_value(int acc, float sx, float sw,
                                               float bias = -0.0f) {
    return __builtin_fmaf((float)acc, sx * sw, bias);
}

/* The elements of an F32 row of n, padded to whole 16-byte pieces. */
__host__ __device__ __forceinline__ uint32_t hk_int8_fours(uint32_t n) {
    return (n + 3u) & ~3u;
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
    float y = hk_int8_value(sum, xs[row], ws[col],
                            bias ? hk_bf2f(bias[col]) : -0.0f);
    if (gelu) y = hk_gelu_tanh_f(y);
    if (wide) wide[row * hk_int8_fours(n) + col] = y;
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

/* ------------------------------------- the products on the matrix cores */

/* Operands of a launch beside hk_gemm_args: the rows' scales, and where the
 * gated block's activation goes in F32. */
struct hk_int8_ext {
    const float *xs, *ws;
    float *wide;
    uint32_t wide_pitch;
};

/* The tiles: the bf16 GEMM's loop over bytes, 2.2 to 2.4 PFLOP/s where 16x16x64
 * MFMAs reach 4.3 from registers (2378 x 5376 -> 21504 241 us, 6144 x 5120 ->
 * 13824 375).  At the package's power: 1400 W and a clock of 1.9 to 2.1 GHz, 0.64
 * pJ an operation for the MFMA's own 0.31.  MFMAs are busy 56% of the cycles: a
 * tile's start and end take 7 us of 58, in which all CUs write, and the loop's
 * LDS reads and loads issue between them. */
#define HK_TRACE(p) ((void)0)
#define HK_TRACE_CLOCK(p) ((void)0)
#define HK_TRACE_VALUE(p, v) ((void)0)
#define HK_KERNEL_INT8
#define HK_KERNEL_NAME hk_int8_gemm
#define HK_KERNEL_TEMPLATE template <int EPI, bool GROUP, int ROW_BLOCKS>
#define HK_KERNEL_JB ROW_BLOCKS
#include "hk_gemm_kernel.inc"

/* Four columns of a row from their sums. */
struct hk_int8_out {
    const float *xs, *ws;
    const uint16_t *bias;
    uint16_t *out;
    float *wide; /* of the gated block: silu(g) u in F32, padded rows */
    uint32_t n;
    int gelu;
};

/* The scales and bias of columns [col, + 4). */
struct hk_int8_columns {
    float scale[4], bias[4];
    __device__ __forceinline__ void load(const hk_int8_out &o, uint32_t col) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            scale[e] = o.ws[col + e];
            bias[e] = o.bias && col + e < o.n ? hk_bf2f(o.bias[col + e])
                                              : -0.0f;
        }
    }
};

__device__ __forceinline__ float hk_int8_made(const hk_int8_out &o, float sx,
                                             float sw, float bias, int sum) {
    const float y = hk_int8_value(sum, sx, sw, bias);
    return o.gelu ? hk_gelu_tanh_f(y) : y;
}

__device__ __forceinline__ void hk_int8_finish(const hk_int8_out &o,
                                               uint32_t row, uint32_t col,
                                               float sx,
                                               const hk_int8_columns &c,
                                               hk_v4i sums) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        y[e] = hk_int8_made(o, sx, c.scale[e], c.bias[e], sums[e]);
    uint16_t *to = o.out + (size_t)row * o.n + col;
    if (o.n % 4u == 0) {
        *(uint2 *)to = make_uint2(hk_pack2(y[0], y[1]), hk_pack2(y[2], y[3]));
    } else if (o.n % 2u == 0) {
        *(uint32_t *)to = hk_pack2(y[0], y[1]);
        if (col + 2u < o.n) *(uint32_t *)(to + 2) = hk_pack2(y[2], y[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (col + e < o.n) to[e] = hk_f2bf(y[e]);
    }
}

/* The same, or of the gated block of a gate's sums and an up row's, whose scales
 * stand in the place of the bias. */
template <bool GATED>
__device__ __forceinline__ void hk_int8_columns_load(hk_int8_columns &c,
                                                     const hk_int8_out &o,
                                                     uint32_t col) {
    c.load(o, col);
    if (GATED) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            c.bias[e] = col + e < o.n ? o.ws[o.n + col + e] : 0.0f;
    }
}

template <bool GATED>
__device__ __forceinline__ void hk_int8_leave(const hk_int8_out &o,
                                              uint32_t row, uint32_t col,
                                              float sx,
                                              const hk_int8_columns &c,
                                              hk_v4i sums, hk_v4i up) {
    if (!GATED) {
        hk_int8_finish(o, row, col, sx, c, sums);
        return;
    }
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        y[e] = hk_swiglu_f(hk_int8_value(sums[e], sx, c.scale[e]),
                           hk_int8_value(up[e], sx, c.bias[e]));
    *(float4 *)(o.wide + (size_t)row * hk_int8_fours(o.n) + col) =
        make_float4(y[0], y[1], y[2], y[3]);
}

/* One row, on the vector units: a wave takes COLUMNS rows of W, each lane 16
 * bytes of every 1024, against X's row in LDS, and adds up its lanes.  W
 * streams from HBM once, in loads of whole KiB, with no pieces of K to join in
 * a second launch: 5120 -> 5120 7.3 us, 14336 -> 5376 14.8, 1024 -> 2048 3.5,
 * as MFMA tiles 9.7, 16.9 and 6.4; 5376 -> 28672 is level (25.4, 6.1 TB/s).  Of
 * more rows the reads of X from LDS are too many (two rows 5120 -> 5120 9.2 and
 * 9.7, 14336 -> 5376 21 and 17). */
template <int COLUMNS, bool GATED>
__global__ void __launch_bounds__(256)
hk_int8_dot(hk_skinny_args g, hk_int8_out o, uint32_t pitch) {
    extern __shared__ __attribute__((aligned(16))) uint8_t xs[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t chunks = pitch / 16u;
    const uint32_t col0 = (blockIdx.x * 4u + wave) * (GATED ? 1u : COLUMNS);
    constexpr int AHEAD = 4; /* loads of a row of W on their way */
    const hk_v4i *w[COLUMNS];
#pragma unroll
    for (int c = 0; c < COLUMNS; c++)
        w[c] = (const hk_v4i *)((const uint8_t *)g.w +
                                (size_t)min(GATED ? col0 + c * o.n : col0 + c,
                                            g.n - 1u) * pitch);
    hk_v4i next[AHEAD][COLUMNS];
    auto load = [&](uint32_t at, hk_v4i (&to)[COLUMNS]) {
#pragma unroll
        for (int c = 0; c < COLUMNS; c++)
            to[c] = at < chunks ? __builtin_nontemporal_load(w[c] + at)
                                : hk_v4i{0, 0, 0, 0};
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(i * 64u + lane, next[i]);
    for (uint32_t i = tid; i < chunks; i += 256u)
        *(hk_v4i *)(xs + i * 16u) = ((const hk_v4i *)g.x)[i];
    __syncthreads();
    int sum[COLUMNS] = {};
    for (uint32_t first = 0; first < chunks; first += AHEAD * 64u) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const uint32_t at = first + i * 64u + lane;
            hk_v4i now[COLUMNS];
#pragma unroll
            for (int c = 0; c < COLUMNS; c++) now[c] = next[i][c];
            load(at + AHEAD * 64u, next[i]);
            /* past the end W is zeros, and X any bytes of it */
            const hk_v4i x =
                *(const hk_v4i *)(xs + min(at, chunks - 1u) * 16u);
#pragma unroll
            for (int c = 0; c < COLUMNS; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    sum[c] = __builtin_amdgcn_sdot4(now[c][e], x[e], sum[c],
                                                    false);
        }
    }
#pragma unroll
    for (int c = 0; c < COLUMNS; c++)
#pragma unroll
        for (int off = 32; off; off >>= 1)
            sum[c] += __shfl_xor(sum[c], off, 64);
    if constexpr (GATED) {
        if (lane || col0 >= o.n) return;
        o.wide[col0] = hk_swiglu_f(
            hk_int8_value(sum[0], o.xs[0], o.ws[col0]),
            hk_int8_value(sum[1], o.xs[0], o.ws[o.n + col0]));
        return;
    }
#pragma unroll
    for (int c = 0; c < COLUMNS; c++) {
        const uint32_t col = col0 + c;
        if (lane != (uint32_t)c || col >= g.n) continue;
        o.out[col] = hk_f2bf(hk_int8_made(
            o, o.xs[0], o.ws[col], o.bias ? hk_bf2f(o.bias[col]) : -0.0f,
            sum[c]));
    }
}

/* How few rows run: groups of 32 mbs rows, and K in pieces where one workgroup
 * per 128 columns and group leaves CUs idle (hk_gemm_skinny_run). */
struct hk_int8_few_plan {
    uint32_t groups, mbs, columns, splits, steps;
    uint32_t narrow; /* waves of hk_int8_narrow, else 0 */
};

/* Few rows: the skinny GEMM's loop (hk_skinny_tile.h) over bytes, a workgroup
 * per 128 columns, piece of K and group of rows.  The groups of the same columns
 * follow each other on the same XCD, which has W's lines in its L2 after the
 * first (workgroup i runs on XCD i % 8): with the groups last in the grid 300 x
 * 1001 -> 5350 took 9.8 us, now 8.8, 256 x 5120 -> 13824 39.3 and 35.4.  A lone
 * group keeps the grid's order (128 x 5376 -> 28672: 37 us, dealt so 40). */
template <int MB, bool GATED>
__global__ void __launch_bounds__(256)
hk_int8_skinny(hk_skinny_args g, hk_int8_out o, hk_int8_few_plan plan) {
    uint32_t at = blockIdx.x;
    if (plan.groups > 1u)
        at = at % 8u * (gridDim.x / 8u) + at / 8u;
    const uint32_t unit = at / plan.groups, z = at - unit * plan.groups;
    const uint32_t y = unit / plan.columns, x = unit - y * plan.columns;
    if (y >= plan.splits) return;
    const uint32_t rows = plan.mbs * 32u, row0 = z * rows;
    g.x += (size_t)row0 * g.k;
    g.m = min(g.m - row0, rows);
    g.x_bytes = g.m * g.k * 2u;
    /* a lane's four columns of each eighth row, and the scales of rows lane and
     * lane + 64: on their way during the loop */
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr uint32_t COLS = GATED ? 16u : 32u, EACH = COLS / 4u;
    const uint32_t col = (x * 4u + wave) * COLS + lane % EACH * 4u;
    hk_int8_columns columns;
    float sx[(MB + 1) / 2];
    if (!g.partial) {
        hk_int8_columns_load<GATED>(columns, o, col);
#pragma unroll
        for (uint32_t i = 0; i < (MB + 1) / 2; i++)
            sx[i] = o.xs[row0 + min(i * 64u + lane, g.m - 1u)];
    }
    const auto use = [&](const hk_i32x16(&acc)[MB], uint32_t n0, uint32_t row,
                         uint32_t half, uint8_t *wbuf) {
        if (n0 >= g.n) return;
        if (g.partial) {
            hk_skinny_partial<MB>((hk_v4i *)g.partial,
                                  ((size_t)z * plan.splits + y) *
                                          plan.columns * 4u + n0 / 32u,
                                  g.m, acc);
            return;
        }
        /* all loads are in before the first store: behind one, a wait for them
         * would be one for the stores as well */
#pragma unroll
        for (int e = 0; e < 4; e++)
            asm volatile("" : "+v"(columns.scale[e]), "+v"(columns.bias[e]));
#pragma unroll
        for (int i = 0; i < (MB + 1) / 2; i++) asm volatile("" : "+v"(sx[i]));
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            /* through the wave's LDS, so that eight lanes write a row's 32
             * columns: rows of 128 bytes, 16-byte chunk c of row r at c ^ r % 8 */
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                *(hk_v4i *)(wbuf + row * 128u +
                            (((q * 2u + half) ^ (row & 7u)) << 4)) =
                    hk_v4i{acc[mb][q * 4], acc[mb][q * 4 + 1],
                           acc[mb][q * 4 + 2], acc[mb][q * 4 + 3]};
#pragma unroll 1
            for (uint32_t i = 0; i < EACH / 2u; i++) {
                const uint32_t r = i * (64u / EACH) + lane / EACH;
                auto of = [&](uint32_t chunk) {
                    return *(const hk_v4i *)(wbuf + r * 128u +
                                             ((chunk ^ (r & 7u)) << 4));
                };
                const hk_v4i sums = of(lane % EACH);
                const hk_v4i up = of(lane % EACH + (GATED ? EACH : 0u));
                const float s = __shfl(sx[mb / 2], (mb & 1) * 32 + r, 64);
                if (mb * 32u + r < g.m && col < o.n)
                    hk_int8_leave<GATED>(o, row0 + mb * 32u + r, col, s,
                                         columns, sums, up);
            }
        }
    };
    hk_skinny_sums<MB, 3, HK_LOAD_ONCE, hk_i32x16, GATED>(g, g.w, x, y, use);
}

/* Narrow products: a workgroup per 32 columns and 32 rows, whose waves take a
 * part of K each and join their sums in LDS, so that there are workgroups enough
 * and no second launch.  W takes its turn through LDS as there, X comes as
 * fragments, which costs more the more rows there are: bound by the steps'
 * latency, or by W's and X's bytes (8 rows 5120 -> 5120 7.7 us, 10.5 with pieces
 * of K; 8 x 3004 -> 5842 5.6 and 9.0; 2 x 5120 -> 13824 13.2 and 16.3; but 32 x
 * 13824 -> 5120 24 and 18.7). */
template <int WAVES, bool GATED>
__global__ void __launch_bounds__(WAVES * 64)
hk_int8_narrow(hk_skinny_args g, hk_int8_out o, uint32_t groups) {
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_lds[];
    constexpr int D = HK_SKINNY_RING;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row = lane & 31u, half = lane >> 5;
    uint32_t at = blockIdx.x;
    if (groups > 1u) at = at % 8u * (gridDim.x / 8u) + at / 8u;
    const uint32_t n0 = at / groups * 32u, row0 = at % groups * 32u;
    const uint32_t n = g.n, k = g.k;
    if (n0 >= n) return;
    const uint32_t m = min(g.m - row0, 32u), k_steps = k / 64u;
    const uint32_t per = (k_steps + WAVES - 1u) / WAVES, base = wave * per;
    const uint32_t steps = base < k_steps ? min(per, k_steps - base) : 0u;
    const __amdgpu_buffer_rsrc_t xr =
        hk_rsrc(g.x + (size_t)row0 * k, m * k * 2u);
    const __amdgpu_buffer_rsrc_t wr = hk_rsrc(g.w, g.w_bytes);
    uint32_t wo[4];
#pragma unroll
    for (int q = 0; q < 4; q++)
        wo[q] = ((GATED ? hk_skinny_gated(n0 + 8u * q + (lane >> 3), n)
                        : min(n0 + 8u * q + (lane >> 3), n)) * k +
                 (lane & 7u) * 8u) * 2u;
    const uint32_t xo = min(row, m) * k * 2u + half * 16u;
    hk_v4i wf[D][4], xf[D][4];
    auto load = [&](int slot, uint32_t step) {
        const uint32_t kb = hk_skinny_k_bytes(base + step, k_steps);
#pragma unroll
        for (int q = 0; q < 4; q++)
            wf[slot][q] = __builtin_amdgcn_raw_buffer_load_b128(
                wr, hk_skinny_lane(wo[q], step, steps), kb, HK_LOAD_ONCE);
#pragma unroll
        for (int q = 0; q < 4; q++)
            xf[slot][q] = __builtin_amdgcn_raw_buffer_load_b128(
                xr, hk_skinny_lane(xo + q * 32u, step, steps), kb, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    /* a thread makes four columns of every so many rows */
    constexpr uint32_t COLS = GATED ? 16u : 32u, EACH = COLS / 4u;
    constexpr uint32_t AT_ONCE = 64u * WAVES / EACH, TURNS = 32u / AT_ONCE;
    const uint32_t col = n0 / 32u * COLS + tid % EACH * 4u;
    hk_int8_columns columns;
    hk_int8_columns_load<GATED>(columns, o, col);
    float sx[TURNS];
#pragma unroll
    for (uint32_t i = 0; i < TURNS; i++)
        sx[i] = o.xs[row0 + min(i * AT_ONCE + tid / EACH, m - 1u)];
#pragma unroll
    for (int d = 0; d + 1 < D; d++) load(d, d);
    hk_i32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0;
    uint8_t *own = hk_lds + wave * 4096u;
    /* (steps past the end add zeros) */
    for (uint32_t s0 = 0; s0 < steps; s0 += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            load((d + 3) % D, s0 + d + 3u);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint32_t wrow = 8u * q + (lane >> 3);
                *(hk_v4i *)(own + wrow * 128u +
                            (((lane & 7u) ^ hk_swz_key(wrow)) << 4)) =
                    wf[d][q];
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
                hk_skinny_mfma(acc,
                               *(const hk_v4i *)(
                                   own + row * 128u +
                                   (((2u * q + half) ^ hk_swz_key(row)) << 4)),
                               xf[d][q]);
        }
    }
    /* rows of 128 bytes, 16-byte chunk c of row r at c ^ r % 8 */
#pragma unroll
    for (uint32_t q = 0; q < 4; q++)
        *(hk_v4i *)(own + row * 128u + (((q * 2u + half) ^ (row & 7u)) << 4)) =
            hk_v4i{acc[q * 4], acc[q * 4 + 1], acc[q * 4 + 2], acc[q * 4 + 3]};
    __syncthreads();
    if (col >= o.n) return;
#pragma unroll
    for (uint32_t i = 0; i < TURNS; i++) {
        const uint32_t r = i * AT_ONCE + tid / EACH;
        auto of = [&](uint32_t chunk) {
            hk_v4i sum = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t j = 0; j < WAVES; j++)
                sum += *(const hk_v4i *)(hk_lds + j * 4096u + r * 128u +
                                         ((chunk ^ (r & 7u)) << 4));
            return sum;
        };
        const hk_v4i sums = of(tid % EACH);
        const hk_v4i up = GATED ? of(tid % EACH + EACH) : sums;
        if (r < m)
            hk_int8_leave<GATED>(o, row0 + r, col, sx[i], columns, sums, up);
    }
}

/* Adds the pieces, as hk_skinny_reduce. */
template <bool GATED>
__global__ void __launch_bounds__(256)
hk_int8_skinny_reduce(hk_skinny_args g, hk_int8_out o, uint32_t mbs,
                      uint32_t tiles, uint32_t splits, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63u, q = threadIdx.x >> 6;
    const uint32_t tile = blockIdx.x / mbs, mb = blockIdx.x % mbs;
    const uint32_t row = mb * 32u + (lane & 31u);
    const uint32_t col =
        tile * (GATED ? 16u : 32u) + q * 8u + (lane >> 5) * 4u;
    const uint32_t row0 = blockIdx.y * rows;
    if (row >= min(g.m - row0, rows) || col >= o.n || (GATED && q >= 2u))
        return;
    const size_t stride = (size_t)tiles * mbs * 256u;
    const hk_v4i *p = (const hk_v4i *)g.partial +
                      blockIdx.y * splits * stride +
                      (size_t)blockIdx.x * 256u + threadIdx.x;
    hk_int8_columns columns;
    hk_int8_columns_load<GATED>(columns, o, col);
    const float sx = o.xs[row0 + row];
    constexpr uint32_t to_up = GATED ? 128u : 0u; /* two quarters further */
    hk_v4i sum = *p, up = p[to_up];
    for (uint32_t s = 1; s < splits; s++) {
        sum += p[s * stride];
        up += p[s * stride + to_up];
    }
    hk_int8_leave<GATED>(o, row0 + row, col, sx, columns, sum, up);
}

/* Adds the pieces of tiles, as hk_splitk_reduce: 4 columns a thread. */
__global__ void __launch_bounds__(256)
hk_int8_tile_reduce(hk_gemm_args g, hk_int8_out o, uint32_t splits) {
    const uint32_t blocks = g.tile_rows / 4u;
    const uint32_t part = blockIdx.x / blocks;
    const uint32_t row = (blockIdx.x - part * blocks) * 4u + (threadIdx.x >> 6);
    const uint32_t tcol = (threadIdx.x & 63u) * 4u;
    uint32_t tile_m, tile_n;
    hk_tile_coords(g.tile_base + part, g.tiles_m, g.tiles_n, tile_m, tile_n);
    const uint32_t m = tile_m * g.tile_rows + row, n = tile_n * HK_BN + tcol;
    if (m >= g.m || n >= g.n) return;
    const size_t tile = (size_t)g.tile_rows * HK_BN;
    const size_t stride = g.part_tiles * tile / 4u;
    const hk_v4i *p = (const hk_v4i *)((const int *)g.partial + part * tile +
                                       row * HK_BN + tcol);
    hk_int8_columns columns;
    columns.load(o, n);
    const float sx = o.xs[m];
    hk_v4i sum = *p;
    for (uint32_t s = 1; s < splits; s++) sum += p[s * stride];
    hk_int8_finish(o, m, n, sx, columns, sum);
}

/* The same of the gated block: F32 rows of its activation. */
__global__ void __launch_bounds__(256)
hk_int8_gated_reduce(hk_gemm_args g, hk_int8_ext scaled, uint32_t splits) {
    const uint32_t blocks = g.tile_rows / 8u;
    const uint32_t part = blockIdx.x / blocks;
    const uint32_t row = (blockIdx.x - part * blocks) * 8u + (threadIdx.x >> 5);
    const uint32_t c4 = (threadIdx.x & 31u) * 4u;
    uint32_t tile_m, tile_n;
    hk_tile_coords(g.tile_base + part, g.tiles_m, g.tiles_n, tile_m, tile_n);
    const uint32_t m = tile_m * g.tile_rows + row, n = tile_n * 128u + c4;
    if (m >= g.m || n >= g.n) return;
    const size_t tile = (size_t)g.tile_rows * HK_BN;
    const size_t stride = g.part_tiles * tile / 4u;
    /* 64 gate columns, then their 64 up ones */
    const hk_v4i *p =
        (const hk_v4i *)((const int *)g.partial + part * tile + row * HK_BN +
                         (c4 >> 6) * 128u + (c4 & 63u));
    hk_v4i gate = p[0], up = p[16];
    for (uint32_t s = 1; s < splits; s++) {
        gate += p[s * stride];
        up += p[s * stride + 16u];
    }
    const float sx = scaled.xs[m];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        y[e] = hk_swiglu_f(
            hk_int8_value(gate[e], sx, scaled.ws[n + e]),
            hk_int8_value(up[e], sx, scaled.ws[g.n + n + e]));
    /* (rows are padded to whole pieces) */
    *(float4 *)(scaled.wide + (size_t)m * scaled.wide_pitch + n) =
        make_float4(y[0], y[1], y[2], y[3]);
}

typedef void (*hk_int8_kernel)(hk_gemm_args, hk_int8_ext);

template <int EPI>
static hk_int8_kernel hk_int8_pick(uint32_t jb) {
    switch (jb) {
    case 4: return hk_int8_gemm<EPI, false, 4>;
    case 5: return hk_int8_gemm<EPI, false, 5>;
    case 6: return hk_int8_gemm<EPI, false, 6>;
    case 7: return hk_int8_gemm<EPI, false, 7>;
    default: return hk_int8_gemm<EPI, false, 8>;
    }
}

static hk_int8_kernel hk_int8_pick_epi(int epilogue, uint32_t jb) {
    switch (epilogue) {
    case HK_EPI_SWIGLU: return hk_int8_pick<HK_EPI_SWIGLU>(jb);
    case HK_EPI_GELU_F32: return hk_int8_pick<HK_EPI_GELU_F32>(jb);
    case HK_EPI_PARTIAL: return hk_int8_pick<HK_EPI_PARTIAL>(jb);
    case HK_EPI_PARTIAL_SWIGLU: return hk_int8_pick<HK_EPI_PARTIAL_SWIGLU>(jb);
    default: return hk_int8_pick<HK_EPI_STORE>(jb);
    }
}

/* beside the tiles: scales and bias */
static uint32_t hk_int8_lds(uint32_t jb) {
    return hk_gemm_lds(jb) + 768u * sizeof(float);
}

static void hk_int8_launch(struct h3_gpu *gpu, int epilogue, uint32_t jb,
                           uint32_t workgroups, const hk_gemm_args &g,
                           const hk_int8_ext &e) {
    static uint64_t ready = 0; /* devices, as in hk_gemm_lds_setup */
    const uint64_t bit = 1ull << (gpu->device & 63);
    if (!(ready & bit)) {
        for (uint32_t j = 4; j <= 8; j++)
            for (int epi : {HK_EPI_STORE, HK_EPI_GELU_F32, HK_EPI_SWIGLU,
                            HK_EPI_PARTIAL, HK_EPI_PARTIAL_SWIGLU})
                (void)hipFuncSetAttribute(
                    (const void *)hk_int8_pick_epi(epi, j),
                    hipFuncAttributeMaxDynamicSharedMemorySize,
                    (int)hk_int8_lds(j));
        ready |= bit;
    }
    hipLaunchKernelGGL(hk_int8_pick_epi(epilogue, jb), dim3(workgroups),
                       dim3(HK_GEMM_THREADS), hk_int8_lds(jb), gpu->stream, g,
                       e);
}

static uint32_t hk_int8_cus(const struct h3_gpu *gpu) {
    return gpu->num_cus > 0 ? (uint32_t)gpu->num_cus : 256u;
}

/* Rows whose bytes, and a K offset behind them, end below 2^32. */
static uint32_t hk_int8_reach(uint32_t pitch) {
    return (0xffffffffu - pitch - 4096u) / pitch;
}

/* x . w^T over tiles, in the plan of the bf16 GEMM: a K step is 128 bytes of
 * a row on both, and takes as long.  `gated`: the activation of n columns, of
 * 2 n rows of w, into e.wide; else o's rows. */
static void hk_int8_tiles(struct h3_gpu *gpu, const hk_int8_matrix &x,
                          const hk_int8_matrix &w, uint32_t n, bool gated,
                          const hk_int8_out &o, hk_int8_ext e) {
    const uint32_t cus = hk_int8_cus(gpu), k_steps = x.pitch / HK_INT8_LINE;
    hk_gemm_args g = {};
    g.x = (const uint16_t *)x.codes;
    g.w = (const uint16_t *)w.codes;
    g.bias = o.bias;
    g.c = o.out;
    g.m = x.rows;
    g.n = n;
    g.k = x.pitch / 2u;
    g.tiles_n = (n + (gated ? 127u : HK_BN - 1u)) / (gated ? 128u : HK_BN);
    const uint32_t jb =
        hk_gemm_row_blocks(g.m, g.tiles_n, k_steps, cus, true);
    g.tile_rows = 32u * jb;
    g.tiles_m = (g.m + g.tile_rows - 1u) / g.tile_rows;
    g.x_bytes = x.rows * x.pitch;
    g.w_bytes = w.rows * w.pitch;
    g.tile_count = g.tiles_m * g.tiles_n;
    const int epilogue = gated    ? HK_EPI_SWIGLU
                         : o.gelu ? HK_EPI_GELU_F32
                                  : HK_EPI_STORE;
    const hk_gemm_rounds r =
        hk_gemm_rounds_of(g.tile_count, k_steps, cus, true);
    float *partial = NULL;
    if (r.splits > 1)
        partial = (float *)hk_splitk_try(
            gpu, (size_t)r.splits * r.tail * g.tile_rows * HK_BN * 4);
    if (!partial) { /* or, without scratch, one more round */
        hk_int8_launch(gpu, epilogue, jb, hk_gemm_grid(g.tile_count, cus), g,
                       e);
        return;
    }
    if (r.full) {
        g.tile_count = r.full;
        hk_int8_launch(gpu, epilogue, jb, hk_gemm_grid(r.full, cus), g, e);
    }
    g.partial = partial;
    g.split_steps = r.steps;
    g.tile_base = r.full;
    g.part_tiles = r.tail;
    hk_int8_launch(gpu, gated ? HK_EPI_PARTIAL_SWIGLU : HK_EPI_PARTIAL, jb,
                   r.tail * r.splits, g, e);
    if (gated)
        hipLaunchKernelGGL(hk_int8_gated_reduce,
                           dim3(r.tail * (g.tile_rows / 8u)), dim3(256), 0,
                           gpu->stream, g, e, r.splits);
    else
        hipLaunchKernelGGL(hk_int8_tile_reduce,
                           dim3(r.tail * (g.tile_rows / 4u)), dim3(256), 0,
                           gpu->stream, g, o, r.splits);
}

/* The plan of the least estimated time, which it returns (us): a step of K takes
 * 0.18 and 0.11 per 32 rows, what comes before and after the steps 2.4 and 0.95,
 * joining pieces 4.6; more workgroups than CUs share them, four at once, and the
 * groups' reads of W end at 6.5 TB/s.  (us by rows of a group, 32 / 64 / 96 / 128:
 * 512 x 1024 -> 1024 5.9 / 7.6 / 9.3 / 11.3, 300 x 2675 -> 1001 10.3 / 11.3 / 12.6
 * / 14.4, 197 x 5120 -> 5120 33 / 24.1 / 20.5 / 22.5, 256 x 5120 -> 13824 70 / 46 /
 * 53 / 35.)  Narrow: 2.5, and a step of a wave 0.2 and as much for 32 rows, or W
 * at 6.2 TB/s and of X, for each workgroup, the part that L1 does not have; two
 * waves where they leave no second turn of the CUs.  (us, narrow and not: 16 x
 * 5120 -> 5120 9.0 and 10.9, 16 x 5120 -> 13824 15.9 and 16.9, 32 x 5120 -> 13824
 * 20.1 and 18.2, 2 x 5376 -> 28672 26.9 and 24.5.) */
static hk_int8_few_plan hk_int8_few_planned(uint32_t cus, uint32_t m,
                                            uint32_t n, uint32_t k_steps,
                                            float *us) {
    hk_int8_few_plan best = {};
    best.groups = (m + 31u) / 32u;
    best.columns = (n + 31u) / 32u;
    best.narrow = best.groups * best.columns <= cus ? 2u : 1u;
    const float lines = (float)best.groups * (float)k_steps *
                        ((float)HK_INT8_LINE / 6.2e6f);
    const float rows = (float)std::min(m, 32u);
    *us = 2.5f + std::max((float)((k_steps + best.narrow - 1u) / best.narrow) *
                              (0.2f + 0.2f / 32.0f * rows),
                          lines * ((float)n + (0.25f + 0.0125f * rows) * rows *
                                                  (float)best.columns));
    for (uint32_t most = 1; most <= 4; most++) {
        hk_int8_few_plan p = {};
        p.groups = (m + 32u * most - 1u) / (32u * most);
        p.mbs = ((m + p.groups - 1u) / p.groups + 31u) / 32u;
        if (p.mbs < most) continue; /* (that many groups have been tried) */
        p.columns = (n + 127u) / 128u;
        p.splits = std::max(
            1u, std::min(cus / (p.columns * p.groups), k_steps / 8u));
        p.steps = k_steps;
        if (p.splits > 1) {
            /* whole turns of the kernel's ring of 4 */
            p.steps = ((k_steps + p.splits - 1u) / p.splits + 3u) & ~3u;
            p.splits = (k_steps + p.steps - 1u) / p.steps;
        }
        const uint32_t workgroups = p.columns * p.groups * p.splits;
        const float rounds =
            workgroups <= cus
                ? 1.0f
                : 0.9f * (float)((workgroups + cus - 1u) / cus);
        const float step = 0.18f + 0.11f * (float)p.mbs;
        const float t =
            std::max((2.4f + 0.95f * (float)p.mbs + step * (float)p.steps) *
                         rounds,
                     (float)p.groups * (float)n * (float)k_steps *
                         ((float)HK_INT8_LINE / 6.5e6f)) +
            (p.splits > 1 ? 4.6f : 0.0f);
        if (t < *us) {
            best = p;
            *us = t;
        }
    }
    return best;
}

template <bool GATED>
static void hk_int8_few(struct h3_gpu *gpu, const hk_int8_matrix &x,
                        const hk_int8_matrix &w, const hk_int8_out &o) {
    hk_skinny_args g = {};
    g.x = (const uint16_t *)x.codes;
    g.w = (const uint16_t *)w.codes;
    g.m = x.rows;
    g.n = w.rows;
    g.k = x.pitch / 2u;
    g.w_bytes = w.rows * w.pitch;
    static uint64_t ready = 0;
    const uint64_t bit = 1ull << (gpu->device & 63);
    if (!(ready & bit)) {
        (void)hipFuncSetAttribute((const void *)hk_int8_skinny<4, GATED>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize,
                                  4 * 4096 * 4 + 16384);
        for (auto dot : {hk_int8_dot<GATED ? 2 : 1, GATED>,
                         hk_int8_dot<2, GATED>})
            (void)hipFuncSetAttribute(
                (const void *)dot, hipFuncAttributeMaxDynamicSharedMemorySize,
                HK_INT8_MOST_COLUMNS);
        ready |= bit;
    }
    if (x.rows == 1) {
        /* two columns a wave where that leaves it eight turns of the CUs, or a
         * gate and its up row */
        const bool two = GATED || g.n > 16384u;
        const uint32_t waves = two ? (g.n + 1u) / 2u : g.n;
        const auto dot = two ? hk_int8_dot<2, GATED>
                             : hk_int8_dot<GATED ? 2 : 1, GATED>;
        hipLaunchKernelGGL(dot, dim3((waves + 3u) / 4u), dim3(256), x.pitch,
                           gpu->stream, g, o, x.pitch);
        return;
    }
    float us;
    hk_int8_few_plan p = hk_int8_few_planned(hk_int8_cus(gpu), x.rows, g.n,
                                             x.pitch / HK_INT8_LINE, &us);
    if (p.narrow) {
        const uint32_t workgroups = p.columns * p.groups;
        const auto narrow = p.narrow == 2u ? hk_int8_narrow<2, GATED>
                                           : hk_int8_narrow<1, GATED>;
        hipLaunchKernelGGL(
            narrow,
            dim3(p.groups > 1u ? (workgroups + 7u) & ~7u : workgroups),
            dim3(p.narrow * 64u), p.narrow * 4096u, gpu->stream, g, o,
            p.groups);
        return;
    }
    g.split_steps = p.steps;
    if (p.splits > 1)
        g.partial = (float *)hk_splitk_try(
            gpu, (size_t)p.groups * p.splits * p.columns * 4 * p.mbs * 4096);
    if (!g.partial) p.splits = 1; /* no scratch: in one piece */
    void (*kernel)(hk_skinny_args, hk_int8_out, hk_int8_few_plan) =
        p.mbs == 1   ? hk_int8_skinny<1, GATED>
        : p.mbs == 2 ? hk_int8_skinny<2, GATED>
        : p.mbs == 3 ? hk_int8_skinny<3, GATED>
                     : hk_int8_skinny<4, GATED>;
    const uint32_t workgroups = p.columns * p.splits * p.groups;
    hipLaunchKernelGGL(kernel,
                       dim3(p.groups > 1u ? (workgroups + 7u) & ~7u
                                          : workgroups),
                       dim3(256), p.mbs * 4096 * 4 + 16384, gpu->stream, g, o,
                       p);
    if (p.splits > 1)
        hipLaunchKernelGGL(hk_int8_skinny_reduce<GATED>,
                           dim3((g.n + 31u) / 32u * p.mbs, p.groups),
                           dim3(256), 0, gpu->stream, g, o, p.mbs,
                           p.columns * 4u, p.splits, 32u * p.mbs);
}

/* Whether m rows run there rather than over tiles: up to 128 always, more of
 * them where the estimates say so (the tiles' is the bf16 GEMM's, a little above
 * what these take), held against both ways at 110 sizes of 160 to 6144 rows (320
 * to 13824 -> 320 to 28672 columns) and 36 of the gated block: the pick is
 * within 12% of the faster one.  Us, here and over tiles: 300 x 5120 -> 2560 17.6
 * and 23.5, 512 x 512 -> 1024 4.8 and 15, 1024 x 1024 -> 4096 12.8 and 33, 2378 x
 * 5120 -> 640 21.5 and 32; 1024 x 5120 -> 13824 112 and 63, 2378 x 1024 -> 4096
 * 26.7 and 17.4.  Few tiles are cut along K, and their pieces' sums cost as much
 * as the products. */
static bool hk_int8_takes_few(const struct h3_gpu *gpu, uint32_t m, uint32_t n,
                              uint32_t pitch) {
    if (m <= 128u) return true;
    float us;
    (void)hk_int8_few_planned(hk_int8_cus(gpu), m, n, pitch / HK_INT8_LINE,
                              &us);
    float tiles;
    (void)hk_gemm_tile_rows(gpu, m, n, pitch / 2u, &tiles);
    return us < 0.95f * tiles;
}

/* Whether x . w^T runs on the matrix cores: everything but weights of 4 GiB
 * and more, whose rows the buffer offsets do not reach. */
static bool hk_int8_fast(const struct h3_gpu *gpu, const hk_int8_matrix &w) {
    return !gpu->reference_kernels && w.rows <= hk_int8_reach(w.pitch);
}

/* bf16 rows of x . w^T. */
static void hk_int8_linear(struct h3_gpu *gpu, hk_int8_matrix x,
                           const hk_int8_matrix &w, const uint16_t *bias,
                           uint16_t *out, int gelu) {
    if (!hk_int8_fast(gpu, w)) {
        hk_int8_simple_run(gpu, x, w, bias, out, NULL, gelu);
        return;
    }
    hk_int8_out o = {x.scales, w.scales, bias, out, NULL, w.rows, gelu};
    const uint32_t most = hk_int8_reach(x.pitch);
    for (uint32_t left = x.rows; left; left -= x.rows) {
        x.rows = std::min(left, most);
        if (hk_int8_takes_few(gpu, x.rows, w.rows, x.pitch))
            hk_int8_few<false>(gpu, x, w, o);
        else
            hk_int8_tiles(gpu, x, w, w.rows, false, o,
                          {o.xs, o.ws, NULL, 0});
        x.codes += (size_t)x.rows * x.pitch;
        o.xs += x.rows;
        o.out += (size_t)x.rows * o.n;
    }
}

/* h = silu(x . gate^T) (x . up^T) in 8 bits, by way of padded F32 rows of it in
 * `wide`, or of both projections from the simple kernel. */
static void hk_int8_gated(struct h3_gpu *gpu, hk_int8_matrix x,
                          const hk_int8_matrix &w, uint32_t hidden,
                          float *wide, const hk_int8_matrix &h) {
    hk_int8_rows_args a = {};
    a.wide = wide;
    a.codes = (int8_t *)h.codes;
    a.scales = (float *)h.scales;
    a.rows = x.rows;
    a.width = hidden;
    a.pitch = h.pitch;
    if (!hk_int8_fast(gpu, w)) {
        a.wide_pitch = hk_int8_fours(2 * hidden);
        hk_int8_simple_run(gpu, x, w, NULL, NULL, wide, 0);
        hk_int8_rows<HK_ROWS_SWIGLU>(gpu, a);
        return;
    }
    a.wide_pitch = hk_int8_fours(hidden);
    const uint32_t most = hk_int8_reach(x.pitch);
    hk_int8_ext e = {x.scales, w.scales, wide, a.wide_pitch};
    for (uint32_t left = x.rows; left; left -= x.rows) {
        x.rows = std::min(left, most);
        if (hk_int8_takes_few(gpu, x.rows, w.rows, x.pitch))
            hk_int8_few<true>(gpu, x, w,
                              {e.xs, e.ws, NULL, NULL, e.wide, hidden, 0});
        else
            hk_int8_tiles(gpu, x, w, hidden, true, {}, e);
        x.codes += (size_t)x.rows * x.pitch;
        e.xs += x.rows;
        e.wide += (size_t)x.rows * e.wide_pitch;
    }
    hk_int8_rows<HK_ROWS_F32>(gpu, a);
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
    hk_int8_linear(gpu, hk_int8_of(input, rows),
                   hk_int8_of(weight, output_dim),
                   bias ? HK_CBF16(bias) : NULL, HK_BF16(output), gelu);
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
    /* F32 rows of the activation or, from the simple kernel, of both
     * projections, then h in 8 bits */
    const hk_int8_matrix x = hk_int8_of(input, rows);
    const hk_int8_matrix w1 = hk_int8_of(fc1_weight, 2 * hidden_dim);
    const uint32_t pitch = fc2_weight->record.n[HK_INT8_PITCH];
    const size_t wide = hk_int8_fours(
        hk_int8_fast(gpu, w1) ? hidden_dim : 2 * hidden_dim);
    const size_t wide_bytes = (rows * wide * 4 + 255) & ~(size_t)255;
    const size_t code_bytes = (size_t)rows * pitch;
    uint8_t *space = (uint8_t *)hk_workspace(
        gpu, wide_bytes + code_bytes + ((size_t)rows + 255u) / 256u * 1024u);
    if (!space) return 0;
    const hk_int8_matrix h = {(int8_t *)(space + wide_bytes),
                              (float *)(space + wide_bytes + code_bytes), rows,
                              pitch};
    hk_op_begin(gpu, "gemm_int8_swiglu");
    hk_int8_gated(gpu, x, w1, hidden_dim, (float *)space, h);
    if (!hk_op_end(gpu, "gemm_int8_swiglu", HK_KIND_LINEAR)) return 0;
    hk_op_begin(gpu, "gemm_int8");
    hk_int8_linear(gpu, h, hk_int8_of(fc2_weight, output_dim), NULL,
                   HK_BF16(output), 0);
    return hk_op_end(gpu, "gemm_int8", HK_KIND_LINEAR);
}

} /* extern "C" */
