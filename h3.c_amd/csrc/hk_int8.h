/* Rows of 8-bit integers with a scale each, as the products (hk_int8.hip) and
 * the cache of keys and values (hk_kv8.hip) hold them: value = code * scale,
 * scale = max|x| / 127, code = rint(127 x / max|x|). */
#ifndef HK_INT8_H
#define HK_INT8_H

#include "hk_common.h"
#include "hk_internal.h"

/* An 8-bit matrix (h3_hip_int8_new) is one tensor: codes [rows][pitch], the
 * rows padded with zeros to whole 128-byte lines (a K step of the matrix
 * kernels), then the rows' F32 scales, of which whole tiles of 256 may be
 * read. */
enum { HK_INT8_ROWS, HK_INT8_COLUMNS, HK_INT8_PITCH }; /* hk_record.n */
#define HK_INT8_LINE 128u
#define HK_INT8_MOST_COLUMNS 131072u /* 127^2 times as many stay below 2^31 */

static inline const int8_t *hk_int8_codes(const h3_gpu_tensor *t) {
    return (const int8_t *)t->data;
}

static inline float *hk_int8_scales(const h3_gpu_tensor *t) {
    return (float *)((uint8_t *)t->data +
                     (size_t)t->record.n[HK_INT8_ROWS] *
                         t->record.n[HK_INT8_PITCH]);
}

/* Magnitudes as the bits of |v|: in the order of the values, with infinities
 * and NaN above all of them. */
#define HK_NOT_FINITE 0x7f800000u

__device__ __forceinline__ uint32_t hk_magnitude(float v) {
    return __float_as_uint(v) & 0x7fffffffu;
}

/* (in registers; six turns through LDS took 0.3 us of a row's 2.6) */
__device__ __forceinline__ uint32_t hk_wave_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 15, 15, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 15, 15, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 15, 15, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 15, 15, true));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}

/* Over the workgroup; scratch as in hk_block_sum. */
__device__ __forceinline__ uint32_t hk_block_umax(uint32_t v,
                                                  uint32_t *scratch,
                                                  uint32_t waves) {
    v = hk_wave_umax(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < waves; w++) v = max(v, scratch[w]);
    return v;
}

/* Codes of values whose largest magnitude is `a` (bits).  The quotient 127 x /
 * a is that of a correctly rounded division, so that ties come out as defined:
 * x = a / 2 gives exactly 63.5.  With r about 1 / a, q = t r is off by an ulp
 * or two, what it leaves, t - q a, is exact, and adding that times r rounds
 * the sum of the two, in the place of a dozen instructions of a division.  For
 * bf16 values t = 127 x is exact too: no other quotient of two lies closer to
 * a border than 2^-17 of its size.
 * Row maxima near the ends of F32's range are first scaled by a power of two:
 * 127 a must not overflow nor 1 / a. */
struct hk_int8_quantizer {
    float scale; /* NaN if the values are not all finite; 0 if all are 0 */
    float times, top, inverse;

    __device__ __forceinline__ explicit hk_int8_quantizer(uint32_t a) {
        const float most = __uint_as_float(a);
        const bool good = a < HK_NOT_FINITE;
        scale = good ? most / 127.0f : __uint_as_float(0x7fc00000u);
        const float pre = most > 0x1p100f   ? 0x1p-64f
                          : most < 0x1p-60f ? 0x1p64f
                                            : 1.0f;
        /* all codes 0 where there is nothing to tell apart */
        times = good && a ? 127.0f * pre : 0.0f;
        top = good && a ? most * pre : 1.0f;
        inverse = __builtin_amdgcn_rcpf(top);
    }

    /* the code as a whole F32 number */
    __device__ __forceinline__ float operator()(float v) const {
        const float t = times == 0.0f ? 0.0f : v * times;
        const float q = t * inverse;
        return __builtin_rintf(
            __builtin_fmaf(__builtin_fmaf(-q, top, t), inverse, q));
    }
};

/* The low bytes of four whole numbers. */
__device__ __forceinline__ uint32_t hk_int8_pack4(float a, float b, float c,
                                                  float d) {
    const uint32_t low = __builtin_amdgcn_perm((uint32_t)(int)b,
                                               (uint32_t)(int)a, 0x0c0c0400u);
    const uint32_t high = __builtin_amdgcn_perm((uint32_t)(int)d,
                                                (uint32_t)(int)c, 0x04000c0cu);
    return low | high;
}

/* Checks an 8-bit matrix argument. */
static inline int hk_int8_require(struct h3_gpu *gpu, const h3_gpu_tensor *t,
                                  uint32_t rows, uint32_t columns,
                                  const char *label) {
    if (!t || t->record.kind != HK_RECORD_INT8)
        return hk_fail(gpu, "%s was not made by h3_hip_int8_new", label);
    if (t->record.n[HK_INT8_COLUMNS] != columns)
        return hk_fail(gpu, "%s has %u columns, not %u", label,
                       t->record.n[HK_INT8_COLUMNS], columns);
    if (t->record.n[HK_INT8_ROWS] < rows)
        return hk_fail(gpu, "%s has %u rows, under %u", label,
                       t->record.n[HK_INT8_ROWS], rows);
    return 1;
}

#endif
