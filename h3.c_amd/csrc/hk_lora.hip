/* Low-rank adapters of several requests beside one projection:
 *   y[r] = act(x[r] . W^T + b + s_a (x[r] . A_a^T) . B_a^T),  a = map[r]
 * (h3_hip_linear_lora_bf16 and its GELU form in h3_hip.h).
 *
 * The adapters live in a table built once: per adapter one entry, then its A
 * (the down projection, [rank][K]) and B (the up projection) as [N][2 padded],
 * with the rank padded by zeros to a multiple of 32 and each row twice, so
 * that a row against the two halves below is whole 64-deep steps of the GEMM
 * for any rank.
 *
 * The products run in two parts.  s_a x . A_a^T goes to scratch as two bf16
 * halves (hk_lora_low); then the projection's own GEMM takes it as a few more
 * steps of K against B_a.  Two halves because the matrix cores take bf16: one
 * would round the adapters' part to 8 bits before it is added, two keep 16,
 * below what F32 sums of that length keep.
 *
 * The simple kernels here (one wave per element of x . A^T, one thread per
 * output, sums in sequence) serve H3_HIP_REFERENCE=1 and the shapes that the
 * matrix-core kernels do not take.
 */
#include "hk_common.h"
#include "hk_gemm.h"
#include "hk_internal.h"
#include "hk_skinny_tile.h"

#include <math.h>
#include <stdlib.h>

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

/* The matrix-core kernels' first product and the joining of the second. */
struct hk_lora_low_args {
    const uint16_t *x;
    uint32_t m, k, x_bytes;
    hk_lora_ext ext;
    uint32_t row_groups; /* of 32 rows */
    uint32_t chunks;     /* of ranks, each a workgroup's */
    uint32_t slots;      /* workgroups that share a row group's adapters */
};

/* Copies a [rows][cols] matrix, `count` elements with zeros behind each row up
 * to `pitch`, with each row `times` over. */
__global__ void __launch_bounds__(256)
hk_lora_pack(const uint16_t *src, uint16_t *dst, uint32_t cols, uint32_t pitch,
             uint32_t times, uint64_t count, hk_lora_entry *entry) {
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= count) return;
    const uint64_t r = i / pitch;
    const uint32_t c = (uint32_t)(i - r * pitch);
    const uint16_t v = c < cols ? src[r * cols + c] : (uint16_t)0;
    for (uint32_t t = 0; t < times; t++)
        dst[(r * times + t) * pitch + c] = v;
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
        const uint16_t *up = e.up + (size_t)col * 2u * e.padded;
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

/* --------------------------------------------- the matrix-core kernels */

/* The least of the workgroup's 256 `ids` over `last` (any, where `last` is
 * none), the same for its four waves; `words` is 4 words of LDS. */
__device__ __forceinline__ uint32_t hk_lora_next(const uint32_t *ids,
                                                 uint32_t last,
                                                 uint32_t *words) {
    __syncthreads(); /* ids written, the words of the call before read */
    uint32_t value = ids[threadIdx.x];
    if (last != HK_LORA_NONE && value <= last) value = HK_LORA_NONE;
#pragma unroll
    for (int offset = 32; offset; offset >>= 1)
        value = min(value, (uint32_t)__shfl_xor((int)value, offset, 64));
    if ((threadIdx.x & 63u) == 0) words[threadIdx.x >> 6] = value;
    __syncthreads();
    value = min(min(words[0], words[1]), min(words[2], words[3]));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)value);
}

/* hk_lora_low's workgroup: rows [32 group, + 32), ranks [16 RB chunk, + 16 RB)
 * of the row group's adapters slot, slot + slots, ... (in rising order).
 *
 * v_mfma_f32_16x16x32_bf16 with A's rows against X's: RB blocks of 16 ranks,
 * two of 16 rows.  The four waves split K (64-deep steps w, w + 4, ...) and
 * add their sums in LDS.  Fragments come straight from global memory, two
 * 32-deep halves of a step so that every 128-byte line is used whole, and two
 * turns of two steps are in flight.  The kernel is bound by reading X once;
 * A is read by every row group, from L2. */
#define HK_LORA_LOW_LDS(RB) (4u * 2u * (RB) * 1024u)

template <int RB>
__device__ __forceinline__ void hk_lora_low_unit(const hk_lora_low_args &g,
                                                 uint32_t group,
                                                 uint32_t chunk,
                                                 uint32_t slot,
                                                 uint8_t *lds) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t r16 = lane & 15u, quad = lane >> 4;
    const uint32_t row0 = group * 32u, rank0 = chunk * (16u * RB);
    const uint32_t steps = g.k / HK_BK;
    /* lane l of every wave has row l % 32's adapter */
    uint32_t mine = HK_LORA_NONE;
    if (row0 + (lane & 31u) < g.m) mine = g.ext.map[row0 + (lane & 31u)];
    if (mine >= g.ext.count) mine = HK_LORA_NONE;

    const __amdgpu_buffer_rsrc_t xr = hk_rsrc(g.x, g.x_bytes);
    uint32_t x_off[2];
#pragma unroll
    for (int j = 0; j < 2; j++)
        x_off[j] = min(row0 + j * 16u + r16, g.m) * g.k * 2u + quad * 16u;

    uint32_t turn = 0;
    uint32_t left = mine;
    for (;;) {
        uint32_t adapter = left;
#pragma unroll
        for (int offset = 16; offset; offset >>= 1)
            adapter = min(adapter,
                          (uint32_t)__shfl_xor((int)adapter, offset, 64));
        adapter = (uint32_t)__builtin_amdgcn_readfirstlane((int)adapter);
        if (adapter == HK_LORA_NONE) break;
        left = left > adapter ? left : HK_LORA_NONE;
        const bool taken = turn++ % g.slots == slot;
        if (!taken) continue;
        const uint64_t *entry = (const uint64_t *)(g.ext.entries + adapter);
        const uint16_t *down = (const uint16_t *)hk_group_word(entry, 0);
        const uint64_t sizes = hk_group_word(entry, 2);
        const uint32_t rank = (uint32_t)sizes;
        const uint32_t padded = (uint32_t)(sizes >> 32);
        const float scale =
            __uint_as_float((uint32_t)hk_group_word(entry, 3));
        if (rank0 >= padded) continue;
        /* ranks past the last load, and come out, as zeros */
        const __amdgpu_buffer_rsrc_t ar = hk_rsrc(down, rank * g.k * 2u);
        uint32_t a_off[RB];
#pragma unroll
        for (int i = 0; i < RB; i++)
            a_off[i] = min(rank0 + i * 16u + r16, rank) * g.k * 2u +
                       quad * 16u;

        hk_f32x4 acc[RB][2];
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = hk_f32x4{0, 0, 0, 0};
        /* a turn: steps 8 t + wave and 8 t + 4 + wave; past the end of K the
         * lane offset lies beyond the buffers and loads zeros */
        hk_v4i fx[2][2][2][2], fa[2][2][2][RB];
        auto load = [&](int buf, uint32_t t) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t step = t * 8u + u * 4u + wave;
                const bool live = step < steps;
                const uint32_t kb = live ? step * (HK_BK * 2u) : 0u;
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        fx[buf][u][h][j] = __builtin_amdgcn_raw_buffer_load_b128(
                            xr, live ? x_off[j] + h * 64u : 0xfffff000u, kb,
                            0);
#pragma unroll
                    for (int i = 0; i < RB; i++)
                        fa[buf][u][h][i] = __builtin_amdgcn_raw_buffer_load_b128(
                            ar, live ? a_off[i] + h * 64u : 0xfffff000u, kb,
                            0);
                }
            }
        };
        auto compute = [&](int buf) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < RB; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(hk_bf16x8,
                                                   fa[buf][u][h][i]),
                                __builtin_bit_cast(hk_bf16x8,
                                                   fx[buf][u][h][j]),
                                acc[i][j], 0, 0, 0);
        };
        const uint32_t turns = (steps + 7u) / 8u;
        load(0, 0);
        for (uint32_t t = 0; t < turns; t += 2u) {
            load(1, t + 1u);
            compute(0);
            load(0, t + 2u);
            compute(1);
        }
        /* acc[i][j][e]: rank rank0 + 16 i + 4 quad + e, row row0 + 16 j + r16.
         * The waves' sums meet in LDS, [wave][row][rank]; a thread adds up 8
         * ranks of a row. */
        float *sums = (float *)lds;
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                *(hk_f32x4 *)(sums + ((wave * 32u + j * 16u + r16) * RB + i) *
                                         16u + quad * 4u) = acc[i][j];
        __syncthreads();
        if (tid < 64u * RB) {
            const uint32_t row = tid / (2u * RB), part = tid % (2u * RB);
            float u[8] = {};
#pragma unroll
            for (int w = 0; w < 4; w++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    u[e] += sums[(w * 32u + row) * (RB * 16u) + part * 8u + e];
            float low[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                u[e] *= scale;
                const float high = hk_bf2f(hk_f2bf(u[e]));
                /* past bf16's range the first half is infinite and stays so */
                low[e] = fabsf(high) == INFINITY ? 0.0f : u[e] - high;
            }
            const uint32_t first = rank0 + part * 8u;
            if (row0 + row < g.m && g.ext.map[row0 + row] == adapter &&
                first < padded) {
                uint16_t *out = (uint16_t *)g.ext.low +
                                (size_t)(row0 + row) * g.ext.pitch + first;
                *(uint4 *)out = hk_pack8(u);
                *(uint4 *)(out + padded) = hk_pack8(low);
            }
        }
        __syncthreads();
    }
}

/* Over 128 rows: a workgroup per (row group, rank chunk).  The chunks of a row
 * group read the same X, so they go to one XCD: workgroups are dealt to the 8
 * XCDs in turn. */
template <int RB>
__global__ void __launch_bounds__(256, 2) hk_lora_low(hk_lora_low_args g) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[HK_LORA_LOW_LDS(RB)];
    const uint32_t eight = blockIdx.x / (8u * g.chunks);
    const uint32_t in = blockIdx.x - eight * 8u * g.chunks;
    const uint32_t group = eight * 8u + (in & 7u);
    if (group < g.row_groups)
        hk_lora_low_unit<RB>(g, group, in >> 3, 0, lds);
}

/* The GEMM with adapters; trace points are hk_gemm.hip's alone. */
#undef HK_GEMM_TRACE_STALLS
#define HK_TRACE(p) ((void)0)
#define HK_TRACE_CLOCK(p) ((void)0)
#define HK_TRACE_VALUE(p, v) ((void)0)
#define HK_KERNEL_LORA
#define HK_KERNEL_NAME hk_gemm_lora
#define HK_KERNEL_TEMPLATE template <int EPI, bool GROUP, int ROW_BLOCKS>
#define HK_KERNEL_JB ROW_BLOCKS
#include "hk_gemm_kernel.inc"

typedef void (*hk_gemm_lora_kernel)(hk_gemm_args, hk_lora_ext);

template <int EPI>
static hk_gemm_lora_kernel hk_gemm_lora_pick(uint32_t jb) {
    switch (jb) {
    case 4: return hk_gemm_lora<EPI, false, 4>;
    case 5: return hk_gemm_lora<EPI, false, 5>;
    case 6: return hk_gemm_lora<EPI, false, 6>;
    case 7:
        /* no plan cuts 224-row tiles along K */
        if constexpr (EPI == HK_EPI_PARTIAL)
            return NULL;
        else
            return hk_gemm_lora<EPI, false, 7>;
    default: return hk_gemm_lora<EPI, false, 8>;
    }
}

static hk_gemm_lora_kernel hk_gemm_lora_pick_epi(int epilogue, uint32_t jb) {
    return epilogue == HK_EPI_PARTIAL ? hk_gemm_lora_pick<HK_EPI_PARTIAL>(jb)
           : epilogue == HK_EPI_GELU  ? hk_gemm_lora_pick<HK_EPI_GELU>(jb)
                                      : hk_gemm_lora_pick<HK_EPI_STORE>(jb);
}

/* the GEMM's LDS, then the rows' adapters and hk_lora_least's words */
static uint32_t hk_gemm_lora_lds(uint32_t jb) {
    return hk_gemm_lds(jb) + 1024u + 32u;
}

void hk_gemm_lora_launch(struct h3_gpu *gpu, int epilogue, uint32_t jb,
                         uint32_t workgroups, const hk_gemm_args &g,
                         const hk_lora_ext &lora) {
    /* devices (bit = ordinal) whose kernels have their LDS limit raised */
    static uint64_t ready = 0;
    const uint64_t bit = 1ull << (gpu->device & 63);
    if (!(ready & bit)) {
        for (uint32_t j = 4; j <= 8; j++)
            for (int epi : {HK_EPI_STORE, HK_EPI_GELU, HK_EPI_PARTIAL})
                if (const hk_gemm_lora_kernel kernel =
                        hk_gemm_lora_pick_epi(epi, j))
                    (void)hipFuncSetAttribute(
                        (const void *)kernel,
                        hipFuncAttributeMaxDynamicSharedMemorySize,
                        (int)hk_gemm_lora_lds(j));
        ready |= bit;
    }
    hipLaunchKernelGGL(hk_gemm_lora_pick_epi(epilogue, jb), dim3(workgroups),
                       dim3(HK_GEMM_THREADS), hk_gemm_lora_lds(jb),
                       gpu->stream, g, lora);
}

/* Up to 128 rows.  The skinny GEMM's workgroups and those of the adapters'
 * first product share one launch: the former stream W for the whole launch,
 * the latter end under them.  The former always leave F32 pieces, which
 * hk_lora_join adds up with the adapters' second product. */
template <int MB, int XA>
__global__ void __launch_bounds__(256)
hk_lora_skinny(hk_skinny_args s, hk_lora_low_args g, uint32_t columns,
               uint32_t pieces, uint32_t units) {
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_xs[];
    if (blockIdx.x < units) {
        uint32_t unit = blockIdx.x;
        const uint32_t chunk = unit % g.chunks;
        unit /= g.chunks;
        hk_lora_low_unit<1>(g, unit % g.row_groups, chunk,
                            unit / g.row_groups, hk_xs);
    } else {
        const uint32_t at = blockIdx.x - units;
        hk_skinny_tile<MB, XA>(s, at % columns, at / columns, 0, columns,
                               pieces);
    }
}

/* C = act(pieces' sums + bias + low . B^T) for 32 columns and 32 rows: wave w
 * takes pieces w, w + 4, ... and the rows' adapters w, w + 4, ..., so that
 * their loads overlap, and the four waves' sums meet in LDS.  32x32x16 MFMAs
 * with B's rows against the rows of `low`, in the layout of the pieces
 * (hk_gemm_skinny). */
__global__ void __launch_bounds__(256)
hk_lora_join(hk_skinny_args g, hk_lora_ext lora, uint32_t mbs, uint32_t tiles,
             uint32_t pieces, int gelu) {
    __shared__ hk_f32x4 lds[4][4][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t tile = blockIdx.x / mbs, mb = blockIdx.x % mbs;
    const uint32_t row = mb * 32u + (lane & 31u), half = lane >> 5;
    const uint32_t n0 = tile * 32u;
    hk_f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] = 0.0f;
    const size_t stride = (size_t)tiles * mbs * 256u;
    const hk_f32x4 *p =
        (const hk_f32x4 *)g.partial + (size_t)blockIdx.x * 256u + lane;
    if (row < g.m && n0 < g.n)
        for (uint32_t s = wave; s < pieces; s += 4u)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const hk_f32x4 v = p[s * stride + q * 64u];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[q * 4 + e] += v[e];
            }
    uint32_t left = HK_LORA_NONE;
    if (row < g.m) left = lora.map[row];
    if (left >= lora.count) left = HK_LORA_NONE;
    const uint32_t mine = left;
    for (uint32_t turn = 0;; turn++) {
        uint32_t adapter = left;
#pragma unroll
        for (int offset = 16; offset; offset >>= 1)
            adapter = min(adapter,
                          (uint32_t)__shfl_xor((int)adapter, offset, 64));
        adapter = (uint32_t)__builtin_amdgcn_readfirstlane((int)adapter);
        if (adapter == HK_LORA_NONE) break;
        left = left > adapter ? left : HK_LORA_NONE;
        if ((turn & 3u) != wave) continue;
        const uint64_t *entry = (const uint64_t *)(lora.entries + adapter);
        const uint16_t *up = (const uint16_t *)hk_group_word(entry, 1);
        const uint64_t sizes = hk_group_word(entry, 2);
        const uint32_t rank = (uint32_t)sizes;
        const uint32_t padded = (uint32_t)(sizes >> 32);
        const uint32_t col = n0 + (lane & 31u);
        const uint16_t *low = lora.low + (size_t)row * lora.pitch;
        for (uint32_t k = half * 8u; k - half * 8u < rank; k += 16u) {
            hk_v4i b = {0, 0, 0, 0}, high = {0, 0, 0, 0}, rest = {0, 0, 0, 0};
            if (col < g.n)
                b = *(const hk_v4i *)(up + (size_t)col * 2u * padded + k);
            if (mine == adapter) {
                high = *(const hk_v4i *)(low + k);
                rest = *(const hk_v4i *)(low + padded + k);
            }
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(hk_bf16x8, b),
                __builtin_bit_cast(hk_bf16x8, high), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(hk_bf16x8, b),
                __builtin_bit_cast(hk_bf16x8, rest), acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
        lds[wave][q][lane] = hk_f32x4{acc[q * 4], acc[q * 4 + 1],
                                      acc[q * 4 + 2], acc[q * 4 + 3]};
    __syncthreads();
    /* thread (q, lane): row as above, columns 8 q + 4 half .. + 4 */
    const uint32_t q = wave, col = n0 + q * 8u + half * 4u;
    if (row >= g.m || col >= g.n) return;
    hk_f32x4 sum = lds[0][q][lane];
#pragma unroll
    for (int w = 1; w < 4; w++) sum += lds[w][q][lane];
    if (g.bias) {
        const uint2 b = *(const uint2 *)(g.bias + col);
        sum[0] += hk_bf2f(b.x & 0xffffu);
        sum[1] += hk_bf2f(b.x >> 16);
        sum[2] += hk_bf2f(b.y & 0xffffu);
        sum[3] += hk_bf2f(b.y >> 16);
    }
    if (gelu)
#pragma unroll
        for (int e = 0; e < 4; e++)
            sum[e] = hk_gelu_tanh_f(hk_bf2f(hk_f2bf(sum[e])));
    *(uint2 *)(g.c + (size_t)row * g.n + col) =
        make_uint2(hk_pack2(sum[0], sum[1]), hk_pack2(sum[2], sum[3]));
}

/* Whether the matrix-core kernels take the call: what the GEMM takes, and the
 * table's largest A and B and the rows' halves within a buffer resource. */
static bool hk_lora_takes(const struct h3_gpu *gpu, const hk_lora_args &g) {
    const uint64_t a = (uint64_t)g.pitch * g.k * 2;
    const uint64_t b = (uint64_t)g.pitch * g.n * 4;
    const uint64_t low = (uint64_t)g.m * g.pitch * 4;
    const uint64_t most = 0xfffff000ull - 4096;
    return hk_gemm_mfma_ok(gpu, g.x, g.w, g.bias, g.c, g.m, g.n, g.k,
                           HK_EPI_STORE) &&
           a + 2ull * g.k < most && b < most && low < most;
}

static int hk_lora_run(struct h3_gpu *gpu, const hk_lora_args &a) {
    hk_lora_low_args g = {};
    g.x = a.x;
    g.m = a.m; g.k = a.k;
    g.x_bytes = (uint32_t)((uint64_t)a.m * a.k * 2);
    g.ext.entries = a.entries;
    g.ext.count = a.count;
    g.ext.map = a.map;
    g.ext.pitch = 2u * a.pitch;
    g.ext.low_bytes = (uint32_t)((uint64_t)a.m * a.pitch * 4);
    uint16_t *low = (uint16_t *)hk_workspace(gpu, g.ext.low_bytes);
    if (!low) return 0;
    g.ext.low = low;
    g.row_groups = (a.m + 31u) / 32u;
    g.slots = 1;
    if (a.m > 128u) {
        const uint32_t rb = a.pitch <= 16 ? 1 : a.pitch <= 32 ? 2 : 4;
        g.chunks = (a.pitch + 16u * rb - 1) / (16u * rb);
        if (a.pitch) {
            const uint32_t grid = (g.row_groups + 7u) / 8u * 8u * g.chunks;
            hipLaunchKernelGGL(rb == 1   ? hk_lora_low<1>
                               : rb == 2 ? hk_lora_low<2>
                                         : hk_lora_low<4>,
                               dim3(grid), dim3(256), 0, gpu->stream, g);
        }
        return hk_gemm_bf16(gpu, a.x, a.w, a.bias, a.c, a.m, a.n, a.k,
                            a.gelu ? HK_EPI_GELU : HK_EPI_STORE, NULL, 0,
                            &g.ext);
    }
    const uint32_t mbs = g.row_groups, columns = (a.n + 127u) / 128u;
    const uint32_t k_steps = a.k / HK_BK;
    const uint32_t cus = gpu->num_cus > 0 ? (uint32_t)gpu->num_cus : 256u;
    hk_skinny_args s = {};
    s.x = a.x; s.w = a.w; s.bias = a.bias; s.c = a.c;
    s.m = a.m; s.n = a.n; s.k = a.k;
    s.x_bytes = g.x_bytes;
    s.w_bytes = (uint32_t)((uint64_t)a.n * a.k * 2);
    /* pieces as the plain skinny GEMM cuts them */
    uint32_t pieces = min(cus / columns, k_steps / 8u);
    s.split_steps = k_steps;
    if (pieces > 1) {
        s.split_steps = ((k_steps + pieces - 1) / pieces + 3u) & ~3u;
        pieces = (k_steps + s.split_steps - 1) / s.split_steps;
    } else {
        pieces = 1;
    }
    s.partial = (float *)hk_splitk_space(
        gpu, (size_t)pieces * columns * 4 * mbs * 4096);
    if (!s.partial) return 0;
    g.chunks = (a.pitch + 15u) / 16u;
    /* a row group has at most 32 adapters */
    g.slots = a.count < 32u ? a.count : 32u;
    const uint32_t units = g.row_groups * g.chunks * g.slots;
    const size_t lds = mbs * 4096 * 4 + 16384;
    void (*kernel)(hk_skinny_args, hk_lora_low_args, uint32_t, uint32_t,
                   uint32_t) = mbs == 1   ? hk_lora_skinny<1, 3>
                               : mbs == 2 ? hk_lora_skinny<2, 3>
                               : mbs == 3 ? hk_lora_skinny<3, 3>
                                          : hk_lora_skinny<4, 3>;
    static uint64_t ready = 0;
    const uint64_t bit = 1ull << (gpu->device & 63);
    if (mbs == 4 && !(ready & bit)) {
        (void)hipFuncSetAttribute((const void *)hk_lora_skinny<4, 3>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)lds);
        ready |= bit;
    }
    hipLaunchKernelGGL(kernel, dim3(units + columns * pieces), dim3(256), lds,
                       gpu->stream, s, g, columns, pieces, units);
    hipLaunchKernelGGL(hk_lora_join, dim3((a.n + 31) / 32 * mbs), dim3(256), 0,
                       gpu->stream, s, g.ext, mbs, columns * 4, pieces,
                       a.gelu);
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
        const uint32_t padded = (ranks[a] + 31u) & ~31u;
        if (padded > largest) largest = padded;
        bytes += ((size_t)ranks[a] * input_dim * 2 + 255) & ~(size_t)255;
        bytes += (size_t)padded * output_dim * 4;
        bytes = (bytes + 255) & ~(size_t)255;
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
        e.padded = (ranks[a] + 31u) & ~31u;
        e.scale = scales[a];
        if (!e.rank) continue;
        e.down = (const uint16_t *)at;
        at += ((size_t)e.rank * input_dim * 2 + 255) & ~(size_t)255;
        e.up = (const uint16_t *)at;
        at += ((size_t)e.padded * output_dim * 4 + 255) & ~(size_t)255;
    }
    const size_t entry_bytes = (size_t)count * sizeof(hk_lora_entry);
    hipError_t status = hipMemcpyAsync(device, entries, entry_bytes,
                                       hipMemcpyHostToDevice, gpu->stream);
    for (uint32_t a = 0; a < count && status == hipSuccess; a++) {
        const hk_lora_entry &e = entries[a];
        if (!e.rank) continue;
        const uint64_t d = (uint64_t)e.rank * input_dim;
        const uint64_t u = (uint64_t)e.padded * output_dim;
        hipLaunchKernelGGL(hk_lora_pack, dim3((unsigned)((d + 255) / 256)),
                           dim3(256), 0, gpu->stream, HK_CBF16(down[a]),
                           (uint16_t *)e.down, input_dim, input_dim, 1u, d,
                           device + a);
        hipLaunchKernelGGL(hk_lora_pack, dim3((unsigned)((u + 255) / 256)),
                           dim3(256), 0, gpu->stream, HK_CBF16(up[a]),
                           (uint16_t *)e.up, e.rank, e.padded, 2u, u,
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
    if (!(hk_lora_takes(gpu, g) ? hk_lora_run(gpu, g)
                                : hk_lora_run_simple(gpu, g)))
        return 0;
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
