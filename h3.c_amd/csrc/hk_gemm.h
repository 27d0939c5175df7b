/* Shared by the kernels built on the BF16 GEMM (hk_gemm.hip) and the one with
 * low-rank adapters (hk_lora.hip): tile sizes, buffer resources and
 * direct-to-LDS loads, the LDS swizzle, the epilogue activations, the launch
 * arguments and the tile order. */
#ifndef HK_GEMM_H
#define HK_GEMM_H

#include "hk_common.h"

#define HK_BM 256
#define HK_BN 256
#define HK_BK 64
#define HK_STAGES 2
#define HK_GEMM_THREADS 256
#define HK_TILE_BYTES (HK_BM * HK_BK * 2)       /* 32 KiB per operand */
#define HK_STAGE_BYTES (2 * HK_TILE_BYTES)      /* X tile then W tile */
/* L2 prefetch distance of the 16x16x32 kernel's K loop, in 64-deep
 * stages past the stage loads' k step */
#define HK_GEMM_PF 2
/* + 256 bytes that the L2 prefetch loads write and nothing reads */
#define HK_GEMM_LDS (HK_STAGES * HK_STAGE_BYTES + 256) /* 128 KiB + 256 */
#define HK_GROUP_M 8

typedef int hk_v4i __attribute__((ext_vector_type(4)));
typedef int hk_v2i __attribute__((ext_vector_type(2)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t hk_rsrc(const void *base,
                                                          uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base),
                                             (short)0, (int)bytes,
                                             0x00020000);
}

/* A wave's direct-to-LDS loads of 16 or 4 bytes per lane: lane i's bytes go
 * to lds + 16 i (4 i).  Functions of their own: in a lambda of a kernel
 * template, the cast to LDS keeps the host pass from emitting the kernel's
 * launch stub when it depends on the template's parameters. */
__device__ __forceinline__ void hk_dma16(__amdgpu_buffer_rsrc_t r,
                                         uint8_t *lds, uint32_t offset,
                                         uint32_t scalar_offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void *)lds, 16, offset,
        scalar_offset, 0, 0);
}

__device__ __forceinline__ void hk_dma4(__amdgpu_buffer_rsrc_t r,
                                        uint8_t *lds, uint32_t offset,
                                        uint32_t scalar_offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void *)lds, 4, offset,
        scalar_offset, 0, 0);
}

/* LDS rows are 128 B (64 bf16 = 8 chunks of 16 B); logical chunk c of row
 * r lives at physical chunk c ^ key(r).  Any 8 consecutive rows get
 * distinct keys (32-bank view, 128 B per cycle) and any 16 consecutive rows
 * distinct (r & 1, key) pairs (64-bank view, 256 B per cycle), so the
 * 32-row fragment reads are conflict-free under either bank model. */
__device__ __forceinline__ uint32_t hk_swz_key(uint32_t row) {
    return (row & 7u) ^ ((row >> 3) & 1u);
}

/* Epilogue activations from the hardware exp2/rcp (v_exp_f32, v_rcp_f32,
 * about 1 ulp each), far below half a bf16 ulp, the rounding applied right
 * after.  silu(x) = x / (1 + e^-x).  The reference's tanh-form GELU
 * (h3_cuda_core.cu:139-158), 0.5 x (1 + tanh u) with
 * u = sqrt(2/pi) (x + 0.044715 x^3), is evaluated as x - x r with
 * r = 1 / (e^(2u) + 1) and e^(2u) = 2^(x (A + B x^2)): five VALU ops and
 * two transcendentals.  Its +-10 saturation needs no branch for finite x
 * (u <= -10 gives 1 + e^(2u) == 1, so r == 1 and x - x r == 0; u >= 10
 * gives |x r| below half an ulp of x); the clamps keep +-inf exact. */
__device__ __forceinline__ float hk_exp_fast(float x) {
    return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}

__device__ __forceinline__ float hk_silu_f(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + hk_exp_fast(-x));
}

__device__ __forceinline__ float hk_gelu_tanh_f(float x) {
    /* A = 2 log2(e) sqrt(2/pi), B = 0.044715 A; v = 2 u log2(e) */
    const float A = 2.302208198144325f, B = 0.1029432395800235f;
    const float v = x * __builtin_fmaf(x * x, B, A);
    const float r =
        __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(v) + 1.0f);
    const float g = __builtin_fmaf(-x, r, x);
    /* u = +-10 */
    return v <= -28.853900817779268f ? 0.0f
         : v >= 28.853900817779268f  ? x
                                     : g;
}

struct hk_gemm_args {
    const uint16_t *x;     /* [M, K] */
    const uint16_t *w;     /* [W rows, K] */
    const uint16_t *bias;  /* [N] or null */
    uint16_t *c;           /* [M, N] */
    uint32_t m, n, k;      /* n = output columns */
    uint32_t tiles_m, tiles_n;
    uint32_t tile_rows;    /* X rows of a tile: 256, or 32 JB */
    uint32_t x_bytes, w_bytes;
    /* split-K (EPI == HK_EPI_PARTIAL only): workgroup pid covers tile
     * tile_base + pid % part_tiles over K steps [split * split_steps,
     * +split_steps), split = pid / part_tiles, and writes the F32 tile to
     * partial[split][pid % part_tiles][tile_rows][256] */
    float *partial;
    uint32_t split_steps, tile_base, part_tiles;
    /* tiles [0, tile_count) of the launch, dealt to the workgroups in
     * rounds of gridDim.x (one round when the grid covers them all) */
    uint32_t tile_count;
    /* split-K over two problems of one shape and one X (EPI_PARTIAL):
     * parts [pair_tiles, 2 pair_tiles) use w1 / bias1 / c1; 0 = one
     * problem */
    uint32_t pair_tiles;
    const uint16_t *w1, *bias1;
    uint16_t *c1;
    /* a group of problems of one shape and one X (the GROUP kernel): tile
     * t is tile t % group_tiles of problem t / group_tiles, whose W, bias
     * and C are group[3 p], group[3 p + 1], group[3 p + 2] */
    uint32_t group_tiles;
    const uint64_t *group;
};

/* A word of the GROUP kernel's problem table, read with a uniform index:
 * marked uniform so that the buffer resources built from it stay in
 * scalar registers (a table load otherwise counts as divergent, and every
 * buffer load would become a loop over the lanes' descriptors). */
__device__ __forceinline__ uint64_t hk_group_word(const uint64_t *table,
                                                  uint32_t index) {
    const uint64_t v = table[index];
    /* readfirstlane returns int: widen through uint32_t, not sign-extend */
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi =
        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (uint64_t)lo | ((uint64_t)hi << 32);
}

/* Tile index -> (tile_m, tile_n): column bands of HK_GROUP_M row tiles, so
 * consecutive tiles share W rows (and, band by band, X rows). */
__device__ __forceinline__ void hk_tile_coords(uint32_t tile, uint32_t tiles_m,
                                               uint32_t tiles_n,
                                               uint32_t &tile_m,
                                               uint32_t &tile_n) {
    const uint32_t band = HK_GROUP_M * tiles_n;
    const uint32_t first_m = (tile / band) * HK_GROUP_M;
    const uint32_t band_rows = min(tiles_m - first_m, (uint32_t)HK_GROUP_M);
    const uint32_t in_band = tile % band;
    tile_m = first_m + in_band % band_rows;
    tile_n = in_band / band_rows;
}

/* Dynamic LDS of a kernel with 32 jb rows per tile. */
static inline uint32_t hk_gemm_lds(uint32_t jb) {
    return HK_STAGES * (32u * jb * HK_BK * 2u + HK_TILE_BYTES) + 256u;
}

/* ------------------------------------------------ low-rank adapters */

/* one adapter of a table (hk_lora.hip), in device memory; the kernels read
 * its first words as 8-byte ones */
struct hk_lora_entry {
    const uint16_t *down; /* A: [rank][K] */
    const uint16_t *up;   /* B twice: [N][2 padded], zeros past the rank */
    uint32_t rank, padded; /* the rank, and as a multiple of 32 */
    float scale;
    uint32_t bad; /* set by hk_lora_pack: an element is not finite */
    /* B as MFMA fragments: lane l of 32 columns and 16 ranks has column l % 32,
     * ranks 8 (l / 32) .. + 8: [N / 32][rank / 16][64][8], rounded up */
    const uint16_t *fragments;
};

#define HK_LORA_NONE 0xffffffffu

/* What the GEMM with adapters adds to its K loop: for row r of adapter a =
 * map[r] < count, s_a x[r] . A_a^T as bf16 halves low[r][0, padded) and
 * [padded, 2 padded) (their sum is the F32 value to 16 bits), against the row
 * of B twice. */
struct hk_lora_ext {
    const hk_lora_entry *entries;
    uint32_t count;
    const uint32_t *map;
    const uint16_t *low;
    uint32_t pitch; /* elements of a row of `low`: twice the largest padded */
    uint32_t low_bytes;
    /* the adapters of each row tile's rows, in rising order: 256 entries a
     * tile, (adapter, 2 padded, address of B), HK_LORA_NONE behind the last */
    uint4 *lists;
};

struct h3_gpu;
/* Launches hk_gemm_lora with 32 jb rows per tile on g; epilogue HK_EPI_STORE,
 * HK_EPI_GELU_F32 or HK_EPI_PARTIAL. */
void hk_gemm_lora_launch(struct h3_gpu *gpu, int epilogue, uint32_t jb,
                         uint32_t workgroups, const hk_gemm_args &g,
                         const hk_lora_ext &lora);

#endif
