/* Low-rank adapters of several requests beside one projection:
 *   y[r] = act(x[r] . W^T + b + s_a (x[r] . A_a^T) . B_a^T),  a = map[r]
 * (h3_hip_linear_lora_bf16 and its GELU form in h3_hip.h).
 *
 * The adapters live in a table built once: per adapter one entry, then its A
 * (the down projection, [rank][K]) and B (the up projection) as [N][2 padded],
 * with the rank padded by zeros to a multiple of 32 and each row twice, so
 * that a row against the two halves below is whole 64-deep steps of the GEMM
 * for any rank; and B once more in the order in which the sum of few rows
 * takes it (as rows of 128 bytes it read four times the lines at rank 16).
 *
 * The products run in two parts.  x . A_a^T goes to scratch in F32, in pieces
 * of K (hk_lora_low_unit).  Their sum times s_a, as two bf16 halves, meets
 * B_a: up to 128 rows, and where the projection has few tiles or steps of K,
 * in the sum of the skinny GEMM's pieces (hk_lora_skinny, hk_lora_join), else
 * as a few more steps of K of the projection's own GEMM (hk_lora_halves,
 * hk_gemm_lora).  Two halves because the matrix cores take bf16: one would
 * round the adapters' part to 8 bits before it is added, two keep 16, below
 * what F32 sums of that length keep.  The activation takes the F32 sum.
 *
 * Measured, in brackets the projection alone in the same run (us; cards differ
 * by up to 5%): 8 rows x 5120 -> 5120, eight adapters of rank 16, 16.8 (13.7);
 * 39 x 2688 -> 96768 101 (87), 5.3 TB/s; 197 x 5120 -> 5376 32 (36); 778 x 7168
 * -> 5376 89 (85); 4756 x 5376 -> 21504, ranks 64 and 4, 828 to 855 (805), 1.3
 * PFLOP/s; 6144 x 5120 -> 13824 with GELU, ranks up to 128, 684 to 724 (667).
 * W's bytes bound the first two, launches and the chains of dependent loads in
 * them beside that; the third its steps of K, in which one wave a SIMD waits
 * for X and W, turns them through LDS and multiplies in sequence; the fourth
 * the cut GEMM and, 13.5 us, the two launches before it; the last two the
 * matrix cores at the package's power limit.
 *
 * What a launch is made of follows the table, not the rows' map, which is only
 * read on the device: workgroups for every rank chunk of the largest adapter
 * and, up to their rows' number, for every adapter.  Those that find nothing
 * leave, but are rounds of launches where there are many: 5120 -> 5120, rows of
 * one adapter of rank 16 out of a table of one, of 64, and of 63 and one of
 * rank 512: 8 rows 15.2, 15.2 and 17.8 us, 128 rows 26.1, 26.2 and 64.6.  And
 * rows of many adapters in any order meet all of them in each tile or 32 rows:
 * 400 x 5120 -> 13824 at rank 128 106 us with one, 114 with two, 218 with 16 and
 * 336 with 64; 4756 x 5376 -> 21504, 16 of rank 64, in order 865, mixed 1341.
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

#include <algorithm>

#define HK_LORA_MAX_RANK 1024u

/* hk_record.n of a table */
enum { HK_LORA_IN, HK_LORA_OUT, HK_LORA_COUNT,
       HK_LORA_RANK, HK_LORA_PADDED /* the largest */ };

struct hk_lora_args {
    const uint16_t *x, *w, *bias;
    uint16_t *c;
    uint32_t m, n, k;
    const hk_lora_entry *entries;
    uint32_t count;
    const uint32_t *map;
    /* s_a x . A_a^T: F32 [rows][pitch] for the simple kernels */
    float *low;
    uint32_t pitch; /* largest padded rank */
    uint32_t rank;  /* largest rank */
    int gelu;
};

/* The matrix-core kernels' first product. */
struct hk_lora_low_args {
    const uint16_t *x;
    uint32_t m, k, x_bytes;
    hk_lora_ext ext;
    /* x . A^T of K's pieces: F32 [piece][row][sum_pitch] */
    float *sums;
    uint32_t sum_pitch;
    uint32_t pieces, piece_steps; /* of K, in 64-deep steps */
    uint32_t row_groups;          /* of 16 J rows */
    uint32_t chunks;              /* of 16 RB ranks */
    uint32_t slots; /* workgroups that share a row group's adapters */
    uint32_t units; /* workgroups in all of them */
    struct hk_lora_row *rows; /* for hk_lora_join: each row's adapter */
};

/* A row's adapter, found once for all of hk_lora_join's waves; rank 0 without
 * one. */
struct hk_lora_row {
    const uint16_t *fragments;
    uint32_t rank;
    float scale;
    uint32_t adapter, unused[3];
};

/* Workgroups of the kernels below, each thread an element at a time: a launch
 * has fewer than 2^32 threads. */
static dim3 hk_lora_pack_grid(uint64_t count) {
    return dim3((unsigned)std::min<uint64_t>((count + 255) / 256, 1u << 22));
}

/* Copies a [rows][cols] matrix, `count` elements with zeros behind each row up
 * to `pitch`, with each row `times` over. */
__global__ void __launch_bounds__(256)
hk_lora_pack(const uint16_t *src, uint16_t *dst, uint32_t cols, uint32_t pitch,
             uint32_t times, uint64_t count, hk_lora_entry *entry) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < count;
         i += (uint64_t)gridDim.x * 256u) {
        const uint64_t r = i / pitch;
        const uint32_t c = (uint32_t)(i - r * pitch);
        const uint16_t v = c < cols ? src[r * cols + c] : (uint16_t)0;
        for (uint32_t t = 0; t < times; t++)
            dst[(r * times + t) * pitch + c] = v;
        /* every writer writes 1 */
        if ((v & 0x7f80u) == 0x7f80u) entry->bad = 1;
    }
}

/* B ([N][rank]) as hk_lora_entry's fragments. */
__global__ void __launch_bounds__(256)
hk_lora_pack_fragments(const uint16_t *src, uint16_t *dst, uint32_t n,
                       uint32_t rank, uint64_t count) {
    const uint32_t chunks = (rank + 15u) / 16u;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < count;
         i += (uint64_t)gridDim.x * 256u) {
        const uint32_t at = (uint32_t)(i % 512u), lane = at >> 3;
        const uint64_t block = i / 512u;
        const uint64_t col = block / chunks * 32u + (lane & 31u);
        const uint32_t k =
            (uint32_t)(block % chunks) * 16u + (lane >> 5) * 8u + (at & 7u);
        dst[i] = col < n && k < rank ? src[col * rank + k] : (uint16_t)0;
    }
}

/* low[r][j] = s_a x[r] . A_a[j]: one wave an element at a time. */
__global__ void __launch_bounds__(256) hk_lora_low_simple(hk_lora_args g) {
    const uint64_t count = (uint64_t)g.m * g.pitch;
    for (uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
         i < count; i += (uint64_t)gridDim.x * 4u) {
        const uint32_t row = (uint32_t)(i / g.pitch);
        const uint32_t j = (uint32_t)(i - (uint64_t)row * g.pitch);
        const uint32_t a = g.map[row];
        if (a >= g.count) continue;
        const hk_lora_entry e = g.entries[a];
        if (j >= e.rank) continue;
        const uint16_t *x = g.x + (size_t)row * g.k;
        const uint16_t *down = e.down + (size_t)j * g.k;
        float sum = 0.0f;
        for (uint32_t k = threadIdx.x & 63u; k < g.k; k += 64u)
            sum = fmaf(hk_bf2f(x[k]), hk_bf2f(down[k]), sum);
        sum = hk_wave_sum(sum);
        if ((threadIdx.x & 63u) == 0) g.low[i] = e.scale * sum;
    }
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
    if (g.gelu) sum = hk_gelu_tanh_f(sum);
    g.c[(size_t)row * g.n + col] = hk_f2bf(sum);
}

static int hk_lora_run_simple(struct h3_gpu *gpu, hk_lora_args &g) {
    if (g.pitch) {
        g.low = (float *)hk_workspace(gpu, (size_t)g.m * g.pitch * 4);
        if (!g.low) return 0;
        const uint64_t blocks = ((uint64_t)g.m * g.pitch + 3) / 4;
        hipLaunchKernelGGL(
            hk_lora_low_simple,
            dim3((unsigned)(blocks < 1u << 20 ? blocks : 1u << 20)),
            dim3(256), 0, gpu->stream, g);
    }
    hipLaunchKernelGGL(hk_lora_simple,
                       dim3((g.n + 255) / 256, g.m < 65535u ? g.m : 65535u,
                            (g.m + 65534u) / 65535u),
                       dim3(256), 0, gpu->stream, g);
    return 1;
}

/* --------------------------------------------- the matrix-core kernels */

/* A workgroup of the first product: 16 J rows from row0 on, ranks [16 RB chunk,
 * + 16 RB) of the rows' adapters slot, slot + slots, ... (in rising order),
 * piece `piece` of K.
 *
 * v_mfma_f32_16x16x32_bf16 with A's rows against X's: RB blocks of 16 ranks,
 * J of 16 rows.  The waves split K (64-deep steps wave, wave + WAVES, ...) and
 * add their sums in LDS.  A workgroup is bound by the latency of its loads and
 * by how fast a CU takes them, so two turns of DEEP steps are in flight (about
 * 190 registers), and a load takes 8 whole 128-byte lines: loaded as fragments
 * (16 half lines each), 197 rows x 5120 took 13.0 us for 16 ranks and 27 for
 * 64, and 6144 rows 34 for 64; as whole lines 6.9, 12.3 and 18.5 (one adapter,
 * one piece, by itself).  The lines
 * turn into fragments in LDS of the wave's own, with the GEMM's swizzle; a
 * wave's LDS operations run in order, so one step's room is enough. */
#define HK_LORA_WAVES 4

template <int RB, int J>
struct hk_lora_low_shape {
    static constexpr int DEEP = 24 / (2 * (RB + J)); /* steps of a turn */
    static constexpr uint32_t STEP = (RB + J) * 16u * 128u; /* bytes */
    /* the waves' lines, or their sums and the rows' adapters */
    static constexpr uint32_t SUMS = HK_LORA_WAVES * J * RB * 1024u;
    static constexpr uint32_t LDS =
        HK_LORA_WAVES * STEP > SUMS + 64u * J ? HK_LORA_WAVES * STEP
                                              : SUMS + 64u * J;
};

template <int RB, int J>
__device__ __forceinline__ void hk_lora_low_unit(const hk_lora_low_args &g,
                                                 uint32_t row0,
                                                 uint32_t chunk,
                                                 uint32_t slot,
                                                 uint32_t piece,
                                                 uint8_t *lds) {
    constexpr int DEEP = hk_lora_low_shape<RB, J>::DEEP;
    constexpr uint32_t STEP = hk_lora_low_shape<RB, J>::STEP;
    constexpr uint32_t WAVES = HK_LORA_WAVES;
    constexpr uint32_t ROWS = 16u * J;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t r16 = lane & 15u, quad = lane >> 4;
    const uint32_t rank0 = chunk * (16u * RB);
    const uint32_t first_step = piece * g.piece_steps;
    const uint32_t steps = min(g.piece_steps, g.k / HK_BK - first_step);
    /* lane l of every wave has row l % ROWS's adapter, and of the first 64
     * adapters the entry of number l: not one more wait for each */
    uint32_t left = HK_LORA_NONE;
    if (row0 + (lane & (ROWS - 1u)) < g.m)
        left = g.ext.map[row0 + (lane & (ROWS - 1u))];
    uint64_t down_of = 0;
    uint32_t rank_of = 0;
    if (lane < g.ext.count) {
        down_of = (uint64_t)(uintptr_t)g.ext.entries[lane].down;
        rank_of = g.ext.entries[lane].rank;
    }

    /* lane l loads chunk l % 8 of row l / 8 of every 8 */
    const uint32_t line = lane >> 3, chunk_off = (lane & 7u) * 16u;
    const __amdgpu_buffer_rsrc_t xr = hk_rsrc(g.x, g.x_bytes);
    uint32_t x_off[2 * J];
#pragma unroll
    for (int j = 0; j < 2 * J; j++)
        x_off[j] = min(row0 + j * 8u + line, g.m) * g.k * 2u + chunk_off;
    /* and puts it into the wave's LDS at the swizzled place: A's rows, then
     * X's; the key of 8 q + line depends on the parity of q */
    uint8_t *own = lds + wave * STEP;
    uint32_t put[2], get[2];
#pragma unroll
    for (int p = 0; p < 2; p++)
        put[p] = line * 128u + (((lane & 7u) ^ hk_swz_key(p * 8u + line)) << 4);
#pragma unroll
    for (int h = 0; h < 2; h++)
        get[h] = r16 * 128u + (((h * 4u + quad) ^ hk_swz_key(r16)) << 4);

    /* turn t of K: steps (DEEP t + u) WAVES + wave, u < DEEP; past the end of
     * K the lane offset lies beyond the buffers and loads zeros */
    hk_v4i lx[2][DEEP][2 * J];
    auto step_of = [&](uint32_t t, int u) {
        return (t * DEEP + u) * WAVES + wave;
    };
    auto load_x = [&](int buf, uint32_t t) {
#pragma unroll
        for (int u = 0; u < DEEP; u++) {
            const uint32_t step = step_of(t, u);
            const bool live = step < steps;
            const uint32_t kb = live ? (first_step + step) * (HK_BK * 2u) : 0u;
#pragma unroll
            for (int j = 0; j < 2 * J; j++)
                lx[buf][u][j] = __builtin_amdgcn_raw_buffer_load_b128(
                    xr, live ? x_off[j] : 0xfffff000u, kb, 0);
        }
    };
    /* X does not wait for the adapter, where there will mostly be one */
    bool have_x = slot == 0 && chunk == 0;
    if (have_x) load_x(0, 0);
    if (left >= g.ext.count) left = HK_LORA_NONE;
    const uint32_t mine = left;

    for (uint32_t turn = 0;; turn++) {
        uint32_t adapter = left;
#pragma unroll
        for (int offset = (int)ROWS / 2; offset; offset >>= 1)
            adapter = min(adapter,
                          (uint32_t)__shfl_xor((int)adapter, offset, 64));
        adapter = (uint32_t)__builtin_amdgcn_readfirstlane((int)adapter);
        if (adapter == HK_LORA_NONE) break;
        left = left > adapter ? left : HK_LORA_NONE;
        if (turn % g.slots != slot) continue;
        uint64_t down;
        uint32_t rank;
        if (adapter < 64u) {
            auto of = [&](uint32_t v) {
                return (uint32_t)__builtin_amdgcn_readlane((int)v,
                                                           (int)adapter);
            };
            down = (uint64_t)of((uint32_t)down_of) |
                   ((uint64_t)of((uint32_t)(down_of >> 32)) << 32);
            rank = of(rank_of);
        } else {
            const uint64_t *entry =
                (const uint64_t *)(g.ext.entries + adapter);
            down = hk_group_word(entry, 0);
            rank = (uint32_t)hk_group_word(entry, 2);
        }
        if (rank0 >= rank) continue;
        /* ranks past the last load, and come out, as zeros */
        const __amdgpu_buffer_rsrc_t ar =
            hk_rsrc((const uint16_t *)down, rank * g.k * 2u);
        uint32_t a_off[2 * RB];
#pragma unroll
        for (int i = 0; i < 2 * RB; i++)
            a_off[i] = min(rank0 + i * 8u + line, rank) * g.k * 2u + chunk_off;

        hk_f32x4 acc[RB][J];
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < J; j++) acc[i][j] = hk_f32x4{0, 0, 0, 0};
        hk_v4i la[2][DEEP][2 * RB];
        auto load_a = [&](int buf, uint32_t t) {
#pragma unroll
            for (int u = 0; u < DEEP; u++) {
                const uint32_t step = step_of(t, u);
                const bool live = step < steps;
                const uint32_t kb =
                    live ? (first_step + step) * (HK_BK * 2u) : 0u;
#pragma unroll
                for (int i = 0; i < 2 * RB; i++)
                    la[buf][u][i] = __builtin_amdgcn_raw_buffer_load_b128(
                        ar, live ? a_off[i] : 0xfffff000u, kb, 0);
            }
        };
        auto compute = [&](int buf) {
#pragma unroll
            for (int u = 0; u < DEEP; u++) {
#pragma unroll
                for (int i = 0; i < 2 * RB; i++)
                    *(hk_v4i *)(own + i * 1024 + put[i & 1]) = la[buf][u][i];
#pragma unroll
                for (int j = 0; j < 2 * J; j++)
                    *(hk_v4i *)(own + (2 * RB + j) * 1024 + put[j & 1]) =
                        lx[buf][u][j];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    hk_v4i fa[RB], fx[J];
#pragma unroll
                    for (int i = 0; i < RB; i++)
                        fa[i] = *(const hk_v4i *)(own + i * 2048 + get[h]);
#pragma unroll
                    for (int j = 0; j < J; j++)
                        fx[j] = *(const hk_v4i *)(own + (RB + j) * 2048 +
                                                  get[h]);
#pragma unroll
                    for (int i = 0; i < RB; i++)
#pragma unroll
                        for (int j = 0; j < J; j++)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(hk_bf16x8, fa[i]),
                                __builtin_bit_cast(hk_bf16x8, fx[j]),
                                acc[i][j], 0, 0, 0);
                }
            }
        };
        const uint32_t turns = (steps + DEEP * WAVES - 1u) / (DEEP * WAVES);
        if (!have_x) load_x(0, 0);
        have_x = false;
        load_a(0, 0);
        for (uint32_t t = 0; t < turns; t += 2u) {
            load_x(1, t + 1u);
            load_a(1, t + 1u);
            compute(0);
            load_x(0, t + 2u);
            load_a(0, t + 2u);
            compute(1);
        }
        /* acc[i][j][e]: rank rank0 + 16 i + 4 quad + e, row row0 + 16 j + r16.
         * The waves' sums meet in LDS, [wave][row][rank]; a thread adds up 8
         * ranks of a row. */
        float *sums = (float *)lds;
        uint32_t *has_of =
            (uint32_t *)(lds + hk_lora_low_shape<RB, J>::SUMS);
        __syncthreads(); /* the sums lie where other waves had their lines */
        if (tid < ROWS) has_of[tid] = mine; /* rows' adapters, none past m */
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < J; j++)
                *(hk_f32x4 *)(sums + ((wave * ROWS + j * 16u + r16) * RB + i) *
                                         16u + quad * 4u) = acc[i][j];
        __syncthreads();
        for (uint32_t at = tid; at < ROWS * 2u * RB; at += WAVES * 64u) {
            const uint32_t row = at / (2u * RB), part = at % (2u * RB);
            if (has_of[row] != adapter) continue;
            hk_f32x4 u[2] = {};
#pragma unroll
            for (int w = 0; w < (int)WAVES; w++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    u[e] += *(const hk_f32x4 *)(
                        sums + (w * ROWS + row) * (RB * 16u) + part * 8u +
                        e * 4u);
            const uint32_t first = rank0 + part * 8u;
            if (first >= g.sum_pitch) continue;
            /* an infinity in the row has met A's padding: zeros there */
            if (first + 8u > rank)
#pragma unroll
                for (uint32_t e = 0; e < 8; e++)
                    if (first + e >= rank) u[e >> 2][e & 3] = 0.0f;
            hk_f32x4 *out = (hk_f32x4 *)(
                g.sums + ((size_t)piece * g.m + row0 + row) * g.sum_pitch +
                first);
            out[0] = u[0];
            out[1] = u[1];
        }
        __syncthreads();
    }
}

/* A row's adapter, for hk_lora_second. */
__device__ __forceinline__ void hk_lora_find_row(const hk_lora_low_args &g,
                                                 uint32_t row) {
    if (row >= g.m) return;
    const uint32_t a = g.ext.map[row];
    hk_lora_row r = {};
    r.adapter = HK_LORA_NONE;
    if (a < g.ext.count) {
        const hk_lora_entry e = g.ext.entries[a];
        r.fragments = e.fragments;
        r.rank = e.rank;
        r.scale = e.scale;
        r.adapter = a;
    }
    g.rows[row] = r;
}

/* The first product by itself: a workgroup per (row group, rank chunk, piece
 * of K, slot).  The chunks of a row group read the same X, so they go to one
 * XCD: workgroups are dealt to the 8 XCDs in turn. */
template <int RB, int J>
__global__ void __launch_bounds__(HK_LORA_WAVES * 64, 2)
hk_lora_low(hk_lora_low_args g) {
    __shared__ __attribute__((aligned(16)))
    uint8_t lds[hk_lora_low_shape<RB, J>::LDS];
    const uint32_t eight = blockIdx.x / (8u * g.chunks);
    const uint32_t in = blockIdx.x - eight * 8u * g.chunks;
    const uint32_t at = eight * 8u + (in & 7u);
    const uint32_t group = at % g.row_groups, rest = at / g.row_groups;
    if (rest < g.pieces * g.slots)
        hk_lora_low_unit<RB, J>(g, group * 16u * J, in >> 3, rest / g.pieces,
                                rest % g.pieces, lds);
}

/* 8 ranks of a row: the sums of K's pieces, four on their way at a time.  (One
 * piece, as with a short K, is its own sum: with the general way's zeros and
 * additions at every 16 ranks of every 32 columns, the join of 573 rows x 3420
 * at rank 128 took 16.0 us for 12.8.) */
__device__ __forceinline__ void hk_lora_add_up(const float *sums,
                                               size_t stride, uint32_t pieces,
                                               hk_f32x4 (&u)[2]) {
    if (pieces == 1u) {
        u[0] = *(const hk_f32x4 *)sums;
        u[1] = *(const hk_f32x4 *)(sums + 4);
        return;
    }
    u[0] = u[1] = hk_f32x4{0, 0, 0, 0};
    for (uint32_t first = 0; first < pieces; first += 4u) {
        hk_f32x4 v[4][2] = {};
#pragma unroll
        for (uint32_t p = 0; p < 4; p++)
            if (first + p < pieces) {
                v[p][0] = *(const hk_f32x4 *)(sums + (first + p) * stride);
                v[p][1] = *(const hk_f32x4 *)(sums + (first + p) * stride + 4);
            }
#pragma unroll
        for (uint32_t p = 0; p < 4; p++) {
            u[0] += v[p][0];
            u[1] += v[p][1];
        }
    }
}

/* The sums times the scale, as bf16 halves. */
__device__ __forceinline__ void hk_lora_split(const hk_f32x4 (&u)[2],
                                              float scale, uint4 &high,
                                              uint4 &rest) {
    float v[8], low[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) {
        v[e] = scale * u[e >> 2][e & 3];
        const float h = hk_bf2f(hk_f2bf(v[e]));
        /* past bf16's range the first half is infinite and stays so */
        low[e] = fabsf(h) == INFINITY ? 0.0f : v[e] - h;
    }
    high = hk_pack8(v);
    rest = hk_pack8(low);
}

/* The halves that the GEMM takes (hk_lora_ext), zeros up to the padded rank:
 * workgroups [0, units) of 256 threads, a thread 8 ranks of a row.  The others
 * list the adapters of a row tile each: the least that is left, over and over.
 * 5 us, whatever the rows: the launch and three loads in sequence. */
__global__ void __launch_bounds__(256)
hk_lora_halves(hk_lora_low_args g, uint32_t units, uint32_t tile_rows) {
    const hk_lora_ext &x = g.ext;
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < units) {
        const uint32_t eights = x.pitch / 16u;
        const uint64_t at = (uint64_t)blockIdx.x * 256u + tid;
        const uint32_t row = (uint32_t)(at / eights);
        const uint32_t first = (uint32_t)(at - (uint64_t)row * eights) * 8u;
        if (row >= g.m) return;
        const uint32_t a = x.map[row];
        if (a >= x.count) return;
        const hk_lora_entry e = x.entries[a];
        if (first >= e.padded) return;
        uint4 high = make_uint4(0, 0, 0, 0), rest = high;
        if (first < e.rank) {
            hk_f32x4 u[2];
            hk_lora_add_up(g.sums + (size_t)row * g.sum_pitch + first,
                           (size_t)g.m * g.sum_pitch, g.pieces, u);
            hk_lora_split(u, e.scale, high, rest);
        }
        uint16_t *out = (uint16_t *)x.low + (size_t)row * x.pitch + first;
        *(uint4 *)out = high;
        *(uint4 *)(out + e.padded) = rest;
        return;
    }
    __shared__ uint32_t words[4];
    const uint32_t tile = blockIdx.x - units, row = tile * tile_rows + tid;
    uint32_t left = HK_LORA_NONE;
    if (tid < tile_rows && row < g.m) left = x.map[row];
    if (left >= x.count) left = HK_LORA_NONE;
    uint32_t count = 0, listed = HK_LORA_NONE;
    for (;;) {
        uint32_t value = left;
#pragma unroll
        for (int offset = 32; offset; offset >>= 1)
            value = min(value, (uint32_t)__shfl_xor((int)value, offset, 64));
        __syncthreads(); /* the words of the turn before have been read */
        if ((tid & 63u) == 0) words[tid >> 6] = value;
        __syncthreads();
        value = min(min(words[0], words[1]), min(words[2], words[3]));
        if (value == HK_LORA_NONE) break;
        if (tid == count) listed = value;
        count++;
        if (left == value) left = HK_LORA_NONE;
    }
    uint4 entry = make_uint4(listed, 0, 0, 0);
    if (listed != HK_LORA_NONE) {
        const hk_lora_entry e = x.entries[listed];
        const uint64_t up = (uint64_t)(uintptr_t)e.up;
        entry = make_uint4(listed, 2u * e.padded, (uint32_t)up,
                           (uint32_t)(up >> 32));
    }
    x.lists[(size_t)tile * 256u + tid] = entry;
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
           : epilogue == HK_EPI_GELU_F32
               ? hk_gemm_lora_pick<HK_EPI_GELU_F32>(jb)
               : hk_gemm_lora_pick<HK_EPI_STORE>(jb);
}

/* the GEMM's LDS, then a tile's adapters by row and its list */
static uint32_t hk_gemm_lora_lds(uint32_t jb) {
    return hk_gemm_lds(jb) + 1024u + 4096u;
}

void hk_gemm_lora_launch(struct h3_gpu *gpu, int epilogue, uint32_t jb,
                         uint32_t workgroups, const hk_gemm_args &g,
                         const hk_lora_ext &lora) {
    /* devices (bit = ordinal) whose kernels have their LDS limit raised */
    static uint64_t ready = 0;
    const uint64_t bit = 1ull << (gpu->device & 63);
    if (!(ready & bit)) {
        for (uint32_t j = 4; j <= 8; j++)
            for (int epi : {HK_EPI_STORE, HK_EPI_GELU_F32, HK_EPI_PARTIAL})
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

/* Adds s_a (x . A^T) . B^T to acc, the sums of 32 columns and 32 rows of a
 * wave in the layout of hk_skinny_tile: lane l has row l % 32 and its adapter
 * `mine` (rank 0 without one), so that what an adapter takes in turn is B
 * alone: 32x32x16 MFMAs of B's rows against the rows' halves, zeros in rows of
 * others.  16 ranks at a time: `u` holds the lane's 8 of the first (add_up of
 * `low`), the next load beside B.  Each B is a wait, but where the rows have
 * several adapters four of them are one. */
__device__ __forceinline__ void hk_lora_second(const hk_lora_low_args &g,
                                               const hk_lora_row &mine,
                                               const float *low,
                                               hk_f32x4 (&u)[2], uint32_t tile,
                                               hk_f32x16 &acc) {
    const uint32_t lane = threadIdx.x & 63u, half = lane >> 5;
    for (uint32_t k = 0;; k += 16u) {
        /* rows with ranks from k on */
        bool left = k < mine.rank;
        uint64_t with = __builtin_amdgcn_ballot_w64(left);
        if (!with) return;
        uint4 high, rest;
        hk_lora_split(u, mine.scale, high, rest);
        /* the next adapter of the rows that are left (of none: the last one
         * again, for no rows), and its B */
        int lead = 0;
        bool its = false;
        auto take = [&]() {
            if (with) lead = __builtin_ctzll(with);
            auto of = [&](uint32_t v) {
                return (uint32_t)__builtin_amdgcn_readlane((int)v, lead);
            };
            const uint64_t at = (uint64_t)(uintptr_t)mine.fragments;
            const hk_v4i *fragments =
                (const hk_v4i *)((uint64_t)of((uint32_t)at) |
                                 ((uint64_t)of((uint32_t)(at >> 32)) << 32));
            const uint32_t chunks = (of(mine.rank) + 15u) / 16u;
            its = left && mine.adapter == of(mine.adapter);
            left = left && !its;
            with = __builtin_amdgcn_ballot_w64(left);
            return fragments[((size_t)tile * chunks + k / 16u) * 64u + lane];
        };
        auto multiply = [&](const hk_v4i &b, bool rows) {
            const hk_v4i none = {0, 0, 0, 0};
            const hk_v4i h = rows ? __builtin_bit_cast(hk_v4i, high) : none;
            const hk_v4i r = rows ? __builtin_bit_cast(hk_v4i, rest) : none;
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(hk_bf16x8, b),
                __builtin_bit_cast(hk_bf16x8, h), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(hk_bf16x8, b),
                __builtin_bit_cast(hk_bf16x8, r), acc, 0, 0, 0);
        };
        const hk_v4i first = take();
        const bool firsts = its;
        /* beside B's wait, the rows' next 16 ranks */
        if (k + 16u < mine.rank)
            hk_lora_add_up(low + k + 16u, (size_t)g.m * g.sum_pitch, g.pieces,
                           u);
        if (!with) {
            multiply(first, firsts);
            continue;
        }
        hk_v4i b[3];
        bool rows[3];
        auto three = [&]() {
#pragma unroll
            for (int i = 0; i < 3; i++) {
                b[i] = take();
                rows[i] = its;
            }
        };
        three();
        multiply(first, firsts);
        for (;;) {
#pragma unroll
            for (int i = 0; i < 3; i++) multiply(b[i], rows[i]);
            if (!with) break;
            three();
        }
    }
}

/* C = act(acc + bias) for the lane's columns of `row`. */
__device__ __forceinline__ void hk_lora_store(const hk_skinny_args &s,
                                              const hk_f32x16 &acc,
                                              uint32_t row, uint32_t n0,
                                              int gelu) {
    const uint32_t half = (threadIdx.x & 63u) >> 5;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint32_t c = n0 + q * 8u + half * 4u;
        if (c >= s.n) continue;
        float out[4] = {acc[q * 4], acc[q * 4 + 1], acc[q * 4 + 2],
                        acc[q * 4 + 3]};
        if (s.bias) {
            const uint2 bias = *(const uint2 *)(s.bias + c);
            out[0] += hk_bf2f(bias.x & 0xffffu);
            out[1] += hk_bf2f(bias.x >> 16);
            out[2] += hk_bf2f(bias.y & 0xffffu);
            out[3] += hk_bf2f(bias.y >> 16);
        }
        if (gelu)
#pragma unroll
            for (int i = 0; i < 4; i++) out[i] = hk_gelu_tanh_f(out[i]);
        *(uint2 *)(s.c + (size_t)row * s.n + c) =
            make_uint2(hk_pack2(out[0], out[1]), hk_pack2(out[2], out[3]));
    }
}

/* The skinny GEMM and the adapters' first product in one launch: `tiles`
 * workgroups of the former, which stream W and leave F32 sums, in one piece
 * of K or more, and the latter's units (32 rows, 16 ranks).  hk_lora_join adds
 * both up.  Tiles that are all resident at once go first and the units beside
 * them (the other order kept CUs from W's stream: 160 rows x 5120 -> 5120 with
 * ranks up to 64 took 34 us against 29), several rounds of tiles behind the
 * units.
 *
 * Over 128 rows there are `groups` of 32 MB rows.  Those of one part of W
 * (column and piece) follow each other on one XCD and find it in its L2:
 * workgroups go to the 8 XCDs in turn, each XCD takes a run of (part, group). */
template <int MB, int J, bool GROUPS>
__global__ void __launch_bounds__(256, MB > 4 ? 1 : 2)
hk_lora_skinny(hk_skinny_args s, hk_lora_low_args g, uint32_t columns,
               uint32_t pieces, uint32_t groups, uint32_t first_tile,
               uint32_t tiles) {
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_xs[];
    const uint32_t at = blockIdx.x - first_tile;
    if (at < tiles) {
        const uint32_t turn =
            GROUPS ? at % 8u * (tiles / 8u) + at / 8u : at;
        const uint32_t part = GROUPS ? turn / groups : turn;
        if (part >= columns * pieces) return;
        hk_skinny_args own = s;
        if constexpr (GROUPS) {
            const uint32_t group = turn - part * groups;
            own.x += (size_t)group * 32u * MB * s.k;
            own.m = min(s.m - group * 32u * MB, 32u * MB);
            own.x_bytes = own.m * s.k * 2u;
            own.partial += (size_t)group * pieces * columns * 4u * MB * 1024u;
        }
        hk_skinny_tile<MB, 3, GROUPS ? HK_LOAD_SHARED : HK_LOAD_ONCE>(
            own, part % columns, part / columns, 0, columns, pieces);
        return;
    }
    uint32_t unit = blockIdx.x < first_tile ? blockIdx.x
                                            : blockIdx.x - tiles;
    if (unit >= g.units) {
        hk_lora_find_row(g, (unit - g.units) * 256u + threadIdx.x);
        return;
    }
    const uint32_t piece = unit % g.pieces;
    unit /= g.pieces;
    const uint32_t chunk = unit % g.chunks;
    unit /= g.chunks;
    const uint32_t group = unit % g.row_groups;
    hk_lora_low_unit<1, J>(g, group * 16u * J, chunk, unit / g.row_groups,
                           piece, hk_xs);
}

/* C = act(pieces' sums + bias + s_a (x . A^T) . B^T) for 32 columns and 32
 * rows, a wave; blockIdx.y is the row group.  Bound by its chain of loads (the
 * row, its first ranks and the pieces; B; 7 us at 8 rows x 5120), at higher
 * ranks by the halves' arithmetic, made anew for every 32 columns, and by how
 * many waves a CU holds: five workgroups (994 rows x 5120 took 16.3 us with
 * four, 14.4 with five; 39 rows x 96768 13.8).  Tried and slower: 32 ranks at
 * a time, all ranks of an adapter in sequence (8 rows with an adapter each 15
 * us), and the same in the skinny workgroups behind whole sums, where the
 * chain has one wave to hide in (160 rows x 320 -> 5120 32 us against 15 with
 * four adapters of up to 64). */
__global__ void __launch_bounds__(256, 5)
hk_lora_join(hk_skinny_args s, hk_lora_low_args g, uint32_t mbs,
             uint32_t tiles, uint32_t pieces, int gelu) {
    const uint32_t lane = threadIdx.x & 63u, half = lane >> 5;
    const uint32_t at =
        blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = at / mbs;
    const uint32_t mb = blockIdx.y * mbs + at % mbs;
    if (tile * 32u >= s.n) return;
    const uint32_t row = mb * 32u + (lane & 31u);
    const bool live = row < s.m;
    const float *low = g.sums + (size_t)row * g.sum_pitch + half * 8u;
    hk_lora_row mine = {};
    hk_f32x4 u[2] = {};
    hk_f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] = 0.0f;
    if (live) {
        mine = g.rows[row];
        /* (what a row without an adapter reads here is not used) */
        if (g.sum_pitch)
            hk_lora_add_up(low, (size_t)s.m * g.sum_pitch, g.pieces, u);
        const size_t stride = (size_t)tiles * mbs * 256u;
        const hk_f32x4 *p = (const hk_f32x4 *)s.partial +
                            blockIdx.y * pieces * stride +
                            (size_t)at * 256u + lane;
        for (uint32_t i = 0; i < pieces; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const hk_f32x4 v = p[i * stride + q * 64u];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[q * 4 + e] += v[e];
            }
    }
    hk_lora_second(g, mine, low, u, tile, acc);
    if (live) hk_lora_store(s, acc, row, tile * 32u, gelu);
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

/* The projection's own GEMM, with the halves as more steps of its K.
 *
 * The first product by itself: 16 RB ranks and 16 J rows a workgroup, K in
 * pieces, the adapters of a row group over slots (of several requests' rows
 * some groups have two or three).  A turn takes about 4 us and 20 KB a us of
 * X's and A's rows, a piece 0.35 us for its sums; two workgroups share a CU.
 * Within a third of the best of 14 shapes of launch: 778 rows x 7168, rank 16,
 * 8.4 us (in one piece 20), 4756 x 5376, ranks up to 64, 25 (44), 6144 x 5120,
 * up to 128, 36 (34 to 55). */
static int hk_lora_run_tiles(struct h3_gpu *gpu, const hk_lora_args &a,
                             hk_lora_low_args &g, uint32_t cus) {
    const uint32_t k_steps = a.k / HK_BK;
    float us;
    const uint32_t tile_rows = hk_gemm_tile_rows(gpu, a.m, a.n, a.k, &us);
    const uint32_t rb = a.rank <= 16 ? 1 : a.rank <= 32 ? 2 : 4;
    const uint32_t turns = std::min(a.count, 3u);
    g.chunks = (a.rank + 16u * rb - 1) / (16u * rb);
    uint32_t rows = 2;
    float least = INFINITY;
    for (uint32_t j = 2; j <= 4; j += 2)
        for (uint32_t slots = 1; slots <= turns; slots++)
            for (uint32_t p = 1; p <= 16 && p <= k_steps; p++) {
                const uint32_t steps = (k_steps + p - 1) / p;
                const uint32_t pieces = (k_steps + steps - 1) / steps;
                const uint32_t groups = (a.m + 16 * j - 1) / (16 * j);
                /* four workgroups that find no adapter in a turn's time; a
                 * group's further turns come once, at the end */
                const uint32_t wgs =
                    groups * g.chunks * pieces * (3 + slots) / 4;
                const float kb = (float)(steps * (j + rb)) * 2.0f;
                const float us = (float)((wgs + 2 * cus - 1) / (2 * cus) +
                                         (turns + slots - 1) / slots - 1) *
                                     (4.0f + kb / 20.0f) +
                                 0.35f * (float)pieces;
                if (us < least) {
                    least = us;
                    rows = j;
                    g.pieces = pieces;
                    g.piece_steps = steps;
                    g.slots = slots;
                    g.row_groups = groups;
                }
            }
    /* the tiles' lists (at most one for every 128 rows), the halves, the sums
     * of K's pieces */
    g.ext.low_bytes = (uint32_t)((uint64_t)a.m * a.pitch * 4);
    const size_t list_bytes = ((size_t)a.m + 127) / 128 * 256 * sizeof(uint4);
    const size_t low_bytes = ((size_t)g.ext.low_bytes + 255) & ~(size_t)255;
    uint8_t *space = (uint8_t *)hk_workspace(
        gpu, list_bytes + low_bytes +
                 (size_t)g.pieces * a.m * g.sum_pitch * sizeof(float));
    if (!space) return 0;
    g.ext.lists = (uint4 *)space;
    g.ext.low = (const uint16_t *)(space + list_bytes);
    g.sums = (float *)(space + list_bytes + low_bytes);
    void (*kernel)(hk_lora_low_args) =
        rb == 1   ? (rows == 2 ? hk_lora_low<1, 2> : hk_lora_low<1, 4>)
        : rb == 2 ? (rows == 2 ? hk_lora_low<2, 2> : hk_lora_low<2, 4>)
                  : (rows == 2 ? hk_lora_low<4, 2> : hk_lora_low<4, 4>);
    if (g.chunks)
        hipLaunchKernelGGL(kernel,
                           dim3((g.row_groups * g.pieces * g.slots + 7u) / 8u *
                                8u * g.chunks),
                           dim3(HK_LORA_WAVES * 64), 0, gpu->stream, g);
    const uint32_t units =
        (uint32_t)(((uint64_t)a.m * (a.pitch / 8u) + 255) / 256);
    hipLaunchKernelGGL(hk_lora_halves,
                       dim3(units + (a.m + tile_rows - 1) / tile_rows),
                       dim3(256), 0, gpu->stream, g, units, tile_rows);
    return hk_gemm_bf16(gpu, a.x, a.w, a.bias, a.c, a.m, a.n, a.k,
                        a.gelu ? HK_EPI_GELU_F32 : HK_EPI_STORE, NULL, 0,
                        &g.ext);
}

/* How the skinny GEMM's workgroups run: groups of 32 mbs rows, K in pieces of
 * `steps` 64-deep steps as the plain skinny GEMM cuts it, while there is one
 * workgroup a CU. */
struct hk_lora_cut {
    uint32_t groups, mbs, columns, pieces, steps, tiles;
};

static hk_lora_cut hk_lora_cut_of(uint32_t m, uint32_t n, uint32_t k_steps,
                                  uint32_t cus, uint32_t most) {
    hk_lora_cut c;
    const uint32_t blocks = (m + 31u) / 32u;
    c.groups = (blocks + most - 1u) / most;
    c.mbs = (blocks + c.groups - 1u) / c.groups;
    c.columns = (n + 127u) / 128u;
    c.pieces = std::min(cus / (c.columns * c.groups), k_steps / 8u);
    c.steps = k_steps;
    if (c.pieces > 1) {
        c.steps = ((k_steps + c.pieces - 1) / c.pieces + 3u) & ~3u;
        c.pieces = (k_steps + c.steps - 1) / c.steps;
    } else {
        c.pieces = 1;
    }
    c.tiles = c.columns * c.pieces * c.groups;
    if (c.groups > 1) c.tiles = (c.tiles + 7u) & ~7u;
    return c;
}

typedef void (*hk_lora_skinny_kernel)(hk_skinny_args, hk_lora_low_args,
                                      uint32_t, uint32_t, uint32_t, uint32_t,
                                      uint32_t);

static hk_lora_skinny_kernel hk_lora_skinny_pick(uint32_t m,
                                                 const hk_lora_cut &c) {
    if (c.groups > 1)
        return c.mbs == 3 ? hk_lora_skinny<3, 2, true>
                          : hk_lora_skinny<4, 2, true>;
    switch (c.mbs) {
    case 1:
        return m <= 16 ? hk_lora_skinny<1, 1, false>
                       : hk_lora_skinny<1, 2, false>;
    case 2: return hk_lora_skinny<2, 2, false>;
    case 3: return hk_lora_skinny<3, 2, false>;
    case 4: return hk_lora_skinny<4, 2, false>;
    case 5: return hk_lora_skinny<5, 2, false>;
    case 6: return hk_lora_skinny<6, 2, false>;
    default: return hk_lora_skinny<7, 2, false>;
    }
}

/* The skinny GEMM's workgroups over groups of at most 128 rows, or one of at
 * most 224. */
static int hk_lora_run_skinny(struct h3_gpu *gpu, const hk_lora_args &a,
                              hk_lora_low_args &g, uint32_t cus,
                              const hk_lora_cut &cut) {
    const uint32_t k_steps = a.k / HK_BK;
    g.chunks = g.sum_pitch / 16u;
    const uint32_t unit_rows = a.m <= 16u ? 16u : 32u;
    g.row_groups = (a.m + unit_rows - 1u) / unit_rows;
    /* the adapters of some rows side by side, and a quarter of K each (more
     * pieces the join would read for every 32 columns).  Over 128 rows there
     * are no more units than the CUs have places beside W's stream, and pieces
     * only of a long K: the join of 573 rows x 1280 -> 3420 with ranks of 128
     * took 25 us with four, 16 with one. */
    const uint32_t room =
        a.m <= 128u ? UINT32_MAX
                        : 3u * cus / (g.row_groups * std::max(1u, g.chunks));
    g.slots = std::max(1u, std::min({a.count, unit_rows, room}));
    const uint32_t most =
        a.m <= 128u ? 4u : std::min({4u, room / g.slots, k_steps / 16u});
    const uint32_t quarters = std::max(1u, most);
    g.piece_steps = (k_steps + quarters - 1u) / quarters;
    g.pieces = (k_steps + g.piece_steps - 1) / g.piece_steps;
    g.units = g.row_groups * g.chunks * g.slots * g.pieces;
    uint32_t others = g.units + (a.m + 255u) / 256u;
    if (cut.groups > 1) others = (others + 7u) & ~7u;
    /* the rows' adapters, the sums of K's pieces */
    const size_t row_bytes = (size_t)a.m * sizeof(hk_lora_row);
    uint8_t *space = (uint8_t *)hk_workspace(
        gpu, row_bytes +
                 (size_t)g.pieces * a.m * g.sum_pitch * sizeof(float));
    if (!space) return 0;
    g.rows = (hk_lora_row *)space;
    g.sums = (float *)(space + row_bytes);

    hk_skinny_args s = {};
    s.x = a.x; s.w = a.w; s.bias = a.bias; s.c = a.c;
    s.m = a.m; s.n = a.n; s.k = a.k;
    s.x_bytes = g.x_bytes;
    s.w_bytes = (uint32_t)((uint64_t)a.n * a.k * 2);
    s.split_steps = cut.steps;
    s.partial = (float *)hk_splitk_try(
        gpu, (size_t)cut.groups * cut.pieces * cut.columns * 4 * cut.mbs *
                 4096);
    /* the tiles need no sums of the whole output */
    if (!s.partial) return hk_lora_run_tiles(gpu, a, g, cus);
    const size_t lds = cut.mbs * 4096 * 4 + 16384;
    const hk_lora_skinny_kernel kernel = hk_lora_skinny_pick(a.m, cut);
    if (cut.mbs >= 4) {
        /* the limit raised, once per device (bit = ordinal) and kernel */
        static uint64_t ready[2][8];
        const uint64_t bit = 1ull << (gpu->device & 63);
        uint64_t &done = ready[cut.groups > 1][cut.mbs];
        if (!(done & bit))
            (void)hipFuncSetAttribute(
                (const void *)kernel,
                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        done |= bit;
    }
    /* tiles that are all resident at once start first */
    const bool tiles_first = cut.tiles <= (cut.mbs > 4 ? cus : 2u * cus);
    hipLaunchKernelGGL(kernel, dim3(cut.tiles + others), dim3(256), lds,
                       gpu->stream, s, g, cut.columns, cut.pieces, cut.groups,
                       tiles_first ? 0u : others, cut.tiles);
    hipLaunchKernelGGL(hk_lora_join,
                       dim3(((a.n + 31) / 32 * cut.mbs + 3) / 4, cut.groups),
                       dim3(256), 0, gpu->stream, s, g, cut.mbs,
                       cut.columns * 4, cut.pieces, a.gelu);
    return 1;
}

/* Estimated microseconds over 128 rows: a step takes 0.65 us with one
 * workgroup of up to 128 rows on a CU and 1.1 with two, more with more rows,
 * the pieces' sums go both ways at 4.5 TB/s; with more rows the first
 * product's units find no room on the CUs that have a workgroup, which a short
 * piece does not hide.  Groups of 128 rows and tiles, measured with one adapter of rank 16 (us): 160
 * x 320 -> 5120 12.5 and 24.6, 1200 rows 28.3 and 26.2; 512 x 512 -> 1536 14.2
 * and 31.1, 4000 rows 32.4 and 43.5; 160 x 5120 -> 5120 25.6 and 39.1, 384 38.4
 * and 46.0, 512 58.8 and 54.2; 384 x 5120 -> 13824 109 and 84.  Those and one
 * group: 133 x 5120 -> 13824 69 and 45, 197 rows 63 and 56; 133 x 5376 -> 21504
 * 95 (tiles) and 72; 197 x 5120 -> 5120 30.4 and 31.5. */
static float hk_lora_skinny_us(const hk_lora_cut &c, uint32_t m, uint32_t n,
                               uint32_t cus) {
    static const float step_us[8] = {0.65f, 0.65f, 0.65f, 0.65f,
                                     0.65f, 0.75f, 0.78f, 0.95f};
    const uint32_t places = c.mbs > 4 || c.tiles <= cus ? cus : 2 * cus;
    const float step = places > cus ? 1.1f : step_us[c.mbs];
    const uint32_t rounds = (c.tiles + places - 1) / places;
    const float start = c.mbs <= 4 ? 6.0f : c.pieces > 1 ? 14.0f : 8.0f;
    return (float)rounds * (float)c.steps * step + start +
           (float)m * (float)n * (float)(8 * c.pieces + 2) / 4.5e6f;
}

/* The adapters that `rows` rows next to each other have, where the table's
 * follow each other over the call's rows, as those of packed requests do: the
 * map itself is on the device. */
static float hk_lora_adapters(const hk_lora_args &a, uint32_t rows) {
    return std::min((float)a.count,
                    1.0f + (float)(a.count - 1u) * (float)rows / (float)a.m);
}

/* What the two estimates, made for one adapter of rank 16, leave out.  An
 * adapter of a tile is a change of operands and, at padded / 32, steps of 64:
 * 1 and 1.7 us a round of tiles. */
static float hk_lora_tiles_more_us(const hk_lora_args &a, uint32_t tile_rows,
                                   uint32_t cus) {
    const float rounds =
        std::max(1.0f, (float)((a.m + tile_rows - 1u) / tile_rows) *
                           (float)((a.n + HK_BN - 1u) / HK_BN) / (float)cus);
    return rounds * (hk_lora_adapters(a, tile_rows) *
                         (1.0f + 1.7f * (float)a.pitch / 32.0f) -
                     2.7f);
}

/* An adapter of the join's 32 rows is a B to wait for at every 16 ranks, with
 * 20 waves on a CU. */
static float hk_lora_join_more_us(const hk_lora_args &a, uint32_t cus) {
    const float waves = (float)((a.m + 31u) / 32u) * (float)((a.n + 31u) / 32u);
    return (hk_lora_adapters(a, 32u) * (float)((a.rank + 15u) / 16u) - 1.0f) *
           (0.5f + 1.3f * waves / (20.0f * (float)cus));
}

static int hk_lora_run(struct h3_gpu *gpu, const hk_lora_args &a) {
    const uint32_t cus = gpu->num_cus > 0 ? (uint32_t)gpu->num_cus : 256u;
    hk_lora_low_args g = {};
    g.x = a.x;
    g.m = a.m; g.k = a.k;
    g.x_bytes = (uint32_t)((uint64_t)a.m * a.k * 2);
    g.ext.entries = a.entries;
    g.ext.count = a.count;
    g.ext.map = a.map;
    g.ext.pitch = 2u * a.pitch;
    g.sum_pitch = (a.rank + 15u) & ~15u;
    hk_lora_cut cut = hk_lora_cut_of(a.m, a.n, a.k / HK_BK, cus, 4);
    if (cut.groups == 1) return hk_lora_run_skinny(gpu, a, g, cus, cut);
    float skinny = cut.groups <= 65535u /* a grid's second dimension */
                       ? hk_lora_skinny_us(cut, a.m, a.n, cus)
                       : INFINITY;
    if (a.m <= 224u) {
        const hk_lora_cut one = hk_lora_cut_of(a.m, a.n, a.k / HK_BK, cus, 7);
        const float us = hk_lora_skinny_us(one, a.m, a.n, cus);
        if (us < skinny) {
            skinny = us;
            cut = one;
        }
    }
    float tiles;
    const uint32_t tile_rows = hk_gemm_tile_rows(gpu, a.m, a.n, a.k, &tiles);
    /* Over tiles W streams at 3 TB/s at most, the first product and the halves
     * come before the GEMM.  The tiles are the safer side of the border.  Timed
     * both ways, the rule takes the faster one or one within 5% in 87 of 92
     * calls with one or two adapters (133 to 4000 rows of eight K x N; 12% at
     * worst) and in 62 of 63 with 4 to 64 whose rows follow each other (6%).
     * Rows in any order are not known here: 51 of 59, and up to 1.8 times (1536
     * x 7168 -> 5376, 64 of rank 16: 387 us over tiles, 219). */
    tiles = std::max(tiles, (float)a.n * (float)a.k * 2.0f / 3e6f) + 14.0f +
            hk_lora_tiles_more_us(a, tile_rows, cus);
    return skinny + hk_lora_join_more_us(a, cus) < 0.95f * tiles
               ? hk_lora_run_skinny(gpu, a, g, cus, cut)
               : hk_lora_run_tiles(gpu, a, g, cus);
}

/* elements of an adapter's fragments, a multiple of 512 */
static size_t hk_lora_fragment_count(uint32_t n, uint32_t rank) {
    return ((size_t)n + 31) / 32 * ((rank + 15) / 16) * 512;
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
    uint32_t largest = 0, largest_rank = 0;
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
        if (ranks[a] > largest_rank) largest_rank = ranks[a];
        bytes += ((size_t)ranks[a] * input_dim * 2 + 255) & ~(size_t)255;
        bytes += (size_t)padded * output_dim * 4;
        bytes = (bytes + 255) & ~(size_t)255;
        bytes += hk_lora_fragment_count(output_dim, ranks[a]) * 2;
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
        e.fragments = (const uint16_t *)at;
        at += hk_lora_fragment_count(output_dim, e.rank) * 2;
    }
    const size_t entry_bytes = (size_t)count * sizeof(hk_lora_entry);
    hipError_t status = hipMemcpyAsync(device, entries, entry_bytes,
                                       hipMemcpyHostToDevice, gpu->stream);
    for (uint32_t a = 0; a < count && status == hipSuccess; a++) {
        const hk_lora_entry &e = entries[a];
        if (!e.rank) continue;
        const uint64_t d = (uint64_t)e.rank * input_dim;
        const uint64_t u = (uint64_t)e.padded * output_dim;
        hipLaunchKernelGGL(hk_lora_pack, hk_lora_pack_grid(d), dim3(256), 0,
                           gpu->stream, HK_CBF16(down[a]),
                           (uint16_t *)e.down, input_dim, input_dim, 1u, d,
                           device + a);
        hipLaunchKernelGGL(hk_lora_pack, hk_lora_pack_grid(u), dim3(256), 0,
                           gpu->stream, HK_CBF16(up[a]),
                           (uint16_t *)e.up, e.rank, e.padded, 2u, u,
                           device + a);
        const uint64_t f = hk_lora_fragment_count(output_dim, e.rank);
        hipLaunchKernelGGL(hk_lora_pack_fragments, hk_lora_pack_grid(f),
                           dim3(256), 0,
                           gpu->stream, HK_CBF16(up[a]),
                           (uint16_t *)e.fragments, output_dim, e.rank, f);
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
    table->record.n[HK_LORA_RANK] = largest_rank;
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
    g.rank = table->record.n[HK_LORA_RANK];
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
