/* The skinny GEMM's workgroup, for the kernel of its own (hk_gemm.hip) and the
 * one that shares its launch with adapters (hk_lora.hip). */
#ifndef HK_SKINNY_TILE_H
#define HK_SKINNY_TILE_H

#include "hk_gemm.h"
#include "hk_skinny.h"

/* Skinny GEMM for M <= 128 rows (the per-block modulation projections: time
 * rows x 2688 against 96768 x 2688 weights; the text refiner's projections of
 * a short prompt).  Bound by streaming W from HBM once, and W is never
 * re-read: each wave owns 32 W rows (output columns) and loads them into
 * registers D - 1 64-wide k steps ahead of the MFMAs, as whole 128-byte lines
 * (a load gives lane l chunk l % 8 of row 8 q + l / 8: eight rows per load,
 * where loading the MFMA fragments directly touches 32 partial rows per load
 * and runs into the cache-line request rate, 27% slower).  The lines go
 * through the wave's own 4-KiB LDS buffer (row-major, the big GEMM's chunk
 * swizzle) and come back out as MFMA fragments.  X (MB x 32 rows) is shared
 * by the workgroup's four waves: MB DMA loads per thread and step stage it
 * into LDS, XA steps ahead in a ring of XA + 1 stages (128-byte rows with the
 * 16-byte-chunk swizzle of the big GEMM), so L2 serves it once per workgroup
 * instead of once per wave.  The step's k offset goes in the buffer's scalar
 * offset; rows past M or N keep a lane offset beyond the buffer and read
 * zeros.
 *
 * W's loads are marked non-temporal: read once, W would push X and the sums
 * out of L2 (39 rows x 2688 -> 96768: 84 us against 97, 6.2 TB/s; 8 x 14336
 * -> 5376: 28.6 against 32.4; 120 x 5376 -> 21504: 68 against 73).  Loading
 * W as 16x16x32 fragments without the LDS turn took 85 for that last one.
 *
 * XA = 3 hides X's L2 latency behind two steps: with one stage ahead every
 * step waited for it where a CU has only one or two workgroups (40 rows x
 * 5376 -> 21504, 168 workgroups: 46.7 us against 52.8).  With several rounds
 * of workgroups, 33 to 64 rows and K from 1024 on, XA = 1 is level or up to 2%
 * ahead (64 rows x 2688 -> 96768: 89.6 us against 91.4): its smaller LDS lets
 * more workgroups share a CU.  With up to 32 rows and a shorter K it is behind
 * (8 x 2688 -> 96768 78.1 and 75.9; 40 x 320 18.8 and 16.1).
 *
 * Where one workgroup per 128 columns leaves CUs idle, K is split into as
 * many pieces as there are CUs for (blockIdx.y), which write F32 sums that
 * hk_skinny_reduce adds: 8 x 14336 -> 5376 takes 28.6 us instead of 146, 120
 * rows 41 instead of 231.  Two workgroups a CU were slower on all but one
 * shape (34 us, 45-53 us): each piece pays its own start and its sums.
 *
 * Ordering: a step waits until X(s) has landed (loads retire in order; W(s)
 * is a register result the compiler waits for), synchronises, stages
 * X(s + XA) into the buffer every wave finished reading in step s - 1, issues
 * W(s + 3) and computes. */
/* cache policies of W's loads: non-temporal (streaming), and as usual */
enum { HK_LOAD_ONCE = 2, HK_LOAD_SHARED = 0 };

struct hk_skinny_args {
    const uint16_t *x, *w, *bias;
    uint16_t *c;
    uint32_t m, n, k, x_bytes, w_bytes;
    /* split-K: workgroup (.., y) takes k steps [y split_steps, + split_steps)
     * and writes F32 sums to partial[y][32-column tile][MB][4][64 lanes] */
    float *partial;
    uint32_t split_steps;
    /* problem blockIdx.z's W, bias and C (a grouped launch), or null */
    const uint64_t *group;
    /* problem 1's W, bias and C of a paired launch (w1 null: one problem);
     * its pieces' sums follow those of problem 0 */
    const uint16_t *w1, *bias1;
    uint16_t *c1;
};

typedef int hk_i32x16 __attribute__((ext_vector_type(16)));

/* One product of a k step: 16 bf16 a row, or (whole-number sums) 32 bytes. */
__device__ __forceinline__ void hk_skinny_mfma(hk_f32x16 &acc, hk_v4i w,
                                               hk_v4i x) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(hk_bf16x8, w), __builtin_bit_cast(hk_bf16x8, x),
        acc, 0, 0, 0);
}

__device__ __forceinline__ void hk_skinny_mfma(hk_i32x16 &acc, hk_v4i w,
                                               hk_v4i x) {
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(w, x, acc, 0, 0, 0);
}

/* The W row of column `at` where each 32 are 16 columns' gates and then their up
 * rows, of n rows in all, gates first; n where there is none. */
__device__ __forceinline__ uint32_t hk_skinny_gated(uint32_t at, uint32_t n) {
    const uint32_t column = at / 32u * 16u + at % 16u;
    return column < n / 2u ? (at & 16u ? n / 2u : 0u) + column : n;
}

/* use(acc, n0, row, half, wbuf) with the sums of piece y of workgroup x's
 * columns: acc[mb][r] = C[mb*32 + row][n0 + (r/4)*8 + half*4 + r%4], n0 = (4 x +
 * wave) 32, row and half of the lane, wbuf 4 KiB of LDS that are the wave's own.
 * Rows of bytes count K in pairs.  GATED: columns as in hk_skinny_gated.  (With
 * sums that a caller holds, the compiler moves them about: 39 x 256 -> 10240, 5.0
 * us for 4.8.) */
template <int MB, int XA, int W_POLICY, typename SUMS, bool GATED = false,
          typename USE>
__device__ __forceinline__ void hk_skinny_sums(const hk_skinny_args &g,
                                               const uint16_t *w, uint32_t x,
                                               uint32_t y, const USE &use) {
    const uint32_t n = g.n, m = g.m, k = g.k;
    /* k steps of this split; its byte offset goes in the scalar offsets */
    const uint32_t base = g.partial ? y * g.split_steps : 0u;
    const uint32_t steps =
        g.partial ? min(g.split_steps, k / 64u - base) : k / 64u;
    constexpr int D = HK_SKINNY_RING;
    constexpr uint32_t XSTAGE = MB * 32u * 128u; /* bytes of X per k step */
    /* XA + 1 X stages, then the four waves' 4-KiB W buffers */
    extern __shared__ __attribute__((aligned(16))) uint8_t hk_xs[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row = lane & 31u, half = lane >> 5;
    const uint32_t n0 = (x * 4u + wave) * 32u;
    const __amdgpu_buffer_rsrc_t xr = hk_rsrc(g.x, g.x_bytes);
    const __amdgpu_buffer_rsrc_t wr = hk_rsrc(w, g.w_bytes);
    uint32_t wo[4];
#pragma unroll
    for (int q = 0; q < 4; q++)
        wo[q] = ((GATED ? hk_skinny_gated(n0 + 8u * q + (lane >> 3), n)
                        : min(n0 + 8u * q + (lane >> 3), n)) * k +
                 (lane & 7u) * 8u) * 2u;
    /* the wave's W buffer, after the X stages */
    uint8_t *wbuf = hk_xs + (XA + 1) * XSTAGE + wave * 4096u;
    /* X staging: slot p = 256 i + tid holds row p / 8, physical chunk p % 8
     * = logical chunk (p % 8) ^ key(row) */
    uint32_t xo[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const uint32_t p = 256u * i + tid, r = p >> 3;
        const uint32_t chunk = (p & 7u) ^ hk_swz_key(r);
        xo[i] = (min(r, m) * k + chunk * 8u) * 2u;
    }
    auto stage_x = [&](int buf, uint32_t step) {
#pragma unroll
        for (int i = 0; i < MB; i++)
            hk_dma16(xr, hk_xs + buf * XSTAGE + (256u * i + wave * 64u) * 16u,
                     hk_skinny_lane(xo[i], step, steps),
                     hk_skinny_k_bytes(base + step, k / 64u));
    };
    hk_v4i wf[D][4];
    auto load_w = [&](int slot, uint32_t step) {
#pragma unroll
        for (int q = 0; q < 4; q++)
            wf[slot][q] = __builtin_amdgcn_raw_buffer_load_b128(
                wr, hk_skinny_lane(wo[q], step, steps),
                hk_skinny_k_bytes(base + step, k / 64u), W_POLICY);
    };
    /* fragment of X rows mb*32 + row, logical chunk 2q + half */
    auto read_x = [&](int buf, int mb, int q) {
        const uint32_t r = mb * 32u + row;
        return *(const hk_v4i *)(
            hk_xs + buf * XSTAGE + r * 128u +
            (((2u * q + half) ^ hk_swz_key(r)) << 4));
    };
    SUMS acc[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[mb][r] = 0;
    /* The waits below count loads: a step's X loads must leave before its W
     * loads, and steps in order.  Nothing else orders them (they write LDS
     * and registers) up to the next step's barrier, which they do not
     * cross. */
    auto in_order = [] { __builtin_amdgcn_sched_barrier(0); };
    /* Steps past the end load zeros (lane offsets beyond the buffers, no
     * memory touched), so a turn of the ring has no branch: behind one, the
     * compiler drains every load in flight. */
#pragma unroll
    for (uint32_t d = 0; d + 1 < D; d++) {
        if (d < XA) stage_x(d, d);
        in_order();
        load_w(d, d);
        in_order();
    }
    /* the barrier as inline assembly: __syncthreads() would also wait for
     * every load in flight (vmcnt(0)), the loads of the steps ahead
     * included */
    auto barrier = [] {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    /* W of ring slot d: its lines into the wave's buffer and back out as
     * fragments (a wave's LDS operations run in order: no barrier), times X
     * of stage d % (XA + 1) */
    auto compute = [&](int d) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t r = 8u * q + (lane >> 3);
            *(hk_v4i *)(wbuf + r * 128u +
                        (((lane & 7u) ^ hk_swz_key(r)) << 4)) = wf[d][q];
        }
        hk_v4i wfrag[4];
#pragma unroll
        for (int q = 0; q < 4; q++)
            wfrag[q] = *(const hk_v4i *)(
                wbuf + row * 128u +
                (((2u * q + half) ^ hk_swz_key(row)) << 4));
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
                hk_skinny_mfma(acc[mb], wfrag[q],
                               read_x(d % (XA + 1), mb, q));
    };
    uint32_t s0 = 0;
    for (; XA == 1 ? s0 < steps : s0 + D <= steps; s0 += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const uint32_t s = s0 + d;
            /* X(s) has landed: after it, step s - XA issued one W step and
             * the XA - 1 steps since then MB + 4 loads each */
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(
                             4 + (XA - 1) * (MB + 4))
                         : "memory");
            barrier();
            stage_x((d + XA) % (XA + 1), s + XA);
            in_order();
            load_w((d + 3) % D, s + 3);
            compute(d);
        }
    }
    /* The steps of a last, partial turn, all of them on their way: run as a
     * whole turn, K = 64 took 4.7 us against 3.9 (32 rows -> 5376 columns).
     * With XA = 1 it stays a whole turn, whose dead steps add nothing: as
     * here it took 60 registers more. */
#pragma unroll
    for (int d = 0; XA > 1 && d + 1 < D; d++) {
        if (s0 + d >= steps) break;
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(
                         4 + (XA - 1 - d) * (MB + 4))
                     : "memory");
        barrier();
        compute(d);
    }
    /* no load to LDS outlives the workgroup */
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    use(acc, n0, row, half, wbuf);
}

/* A piece's sums, [32-column tile][MB][4][64 lanes] of four, `tile` counted
 * over the pieces: whole lines, each (mb, q) is a wave's 64 16-byte ones. */
template <int MB, typename SUMS, typename FOUR>
__device__ __forceinline__ void hk_skinny_partial(FOUR *partial, size_t tile,
                                                  uint32_t m,
                                                  const SUMS (&acc)[MB]) {
    const uint32_t lane = threadIdx.x & 63u, row = lane & 31u;
    FOUR *part = partial + tile * (MB * 256u);
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        if (mb * 32u + row >= m) continue;
#pragma unroll
        for (int q = 0; q < 4; q++)
            part[(mb * 4u + q) * 64u + lane] =
                FOUR{acc[mb][q * 4], acc[mb][q * 4 + 1], acc[mb][q * 4 + 2],
                     acc[mb][q * 4 + 3]};
    }
}

/* Addresses out of a table could be LDS for all the compiler knows, which
 * waits for the loads to LDS before each of them (39 x 256 -> 10240: 0.4 us of
 * 4.7). */
typedef uint32_t hk_v2u __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) hk_v2u hk_global_v2u;

/* Workgroup (x, y, z) of `columns` x `pieces` ones a problem. */
template <int MB, int XA, int W_POLICY = HK_LOAD_ONCE>
__device__ __forceinline__ void hk_skinny_tile(const hk_skinny_args &g,
                                               uint32_t x, uint32_t y,
                                               uint32_t z, uint32_t columns,
                                               uint32_t pieces) {
    const uint32_t n = g.n, m = g.m;
    const uint16_t *w = g.w, *bias = g.bias;
    uint16_t *c = g.c;
    if (g.group) {
        w = (const uint16_t *)hk_group_word(g.group, 3 * z);
        bias = (const uint16_t *)hk_group_word(g.group, 3 * z + 1);
        c = (uint16_t *)hk_group_word(g.group, 3 * z + 2);
    } else if (z) {
        w = g.w1;
        bias = g.bias1;
        c = g.c1;
    }
    const auto use = [&](const hk_f32x16(&acc)[MB], uint32_t n0, uint32_t row,
                         uint32_t half, uint8_t *) {
        if (g.partial) {
            if (n0 >= n) return;
            hk_skinny_partial<MB>(
                (hk_f32x4 *)g.partial,
                ((size_t)z * pieces + y) * columns * 4u + n0 / 32u, m, acc);
            return;
        }
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const uint32_t mm = mb * 32u + row;
            if (mm >= m) continue;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint32_t col = n0 + q * 8u + half * 4u;
                if (col >= n) continue;
                float out[4];
#pragma unroll
                for (int e = 0; e < 4; e++) out[e] = acc[mb][q * 4 + e];
                if (bias) {
                    const hk_v2u b = *(const hk_global_v2u *)(bias + col);
                    out[0] += hk_bf2f(b.x & 0xffffu);
                    out[1] += hk_bf2f(b.x >> 16);
                    out[2] += hk_bf2f(b.y & 0xffffu);
                    out[3] += hk_bf2f(b.y >> 16);
                }
                *(hk_global_v2u *)(c + (size_t)mm * n + col) =
                    hk_v2u{hk_pack2(out[0], out[1]), hk_pack2(out[2], out[3])};
            }
        }
    };
    hk_skinny_sums<MB, XA, W_POLICY, hk_f32x16>(g, w, x, y, use);
}

#endif
