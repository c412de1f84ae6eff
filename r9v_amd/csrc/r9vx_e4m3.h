/*
 * r9vx_e4m3.h -- shared parts of the block-scaled e4m3 path: how a value is
 * rounded to e4m3, the MFMA tile, and the internal launchers.
 *
 * Numbers: OCP e4m3 (largest 448, smallest 2^-9, NaN 0x7F, no infinity).  A
 * row of activations carries one f32 scale per 128 columns, a weight one per
 * 128 x 128 block.  Scaled sums are f32; what a block's 128 products keep
 * before that is the matrix instruction's matter (fp8_mma).
 */
#ifndef R9VX_E4M3_H
#define R9VX_E4M3_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "r9vx_device.h"
#include "r9vx_internal.h"
#include "r9vx_fp8.h"

constexpr uint32_t kFp8Block = 128; /* columns of one scale */

__host__ __device__ inline uint32_t r9vx_fp8_kb(uint32_t k) { return k / kFp8Block + (k % kFp8Block ? 1u : 0u); }

#ifdef __HIPCC__
namespace r9vx {

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int CTRL>
__device__ __forceinline__ uint32_t fp8_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
/* Largest of 8, 16 and 32 neighbouring lanes. */
__device__ __forceinline__ uint32_t fp8_max8(uint32_t x) {
    x = max(x, fp8_dpp<0xB1>(x));  /* quad_perm 1 0 3 2 */
    x = max(x, fp8_dpp<0x4E>(x));  /* quad_perm 2 3 0 1 */
    return max(x, fp8_dpp<0x141>(x)); /* row_half_mirror */
}
__device__ __forceinline__ uint32_t fp8_max16(uint32_t x) {
    x = fp8_max8(x);
    return max(x, fp8_dpp<0x140>(x)); /* row_mirror */
}

__device__ __forceinline__ uint32_t fp8_max32(uint32_t x) {
    x = fp8_max16(x);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

/* The scale of a block whose largest |x| has the bit pattern `amax`:
 * max(amax / 448, 2^-126), so that an empty or all-zero block has a scale
 * too.  A NaN or an infinity (patterns from 0x7F800000 on, which an
 * unsigned maximum carries through) makes the scale and every code NaN. */
struct Fp8Scale {
    float s, sp, inv, pre;
    bool bad;
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t amax) {
    Fp8Scale q;
    q.bad = amax >= 0x7F800000u;
    q.s = fmaxf(__builtin_bit_cast(float, amax) / 448.0f, 0x1p-126f);
    /* small blocks are lifted by an exact power of two, so that the residuals
     * below stay normal numbers */
    q.pre = q.s < 0x1p-64f ? 0x1p+64f : 1.0f;
    q.sp = q.s * q.pre;
    q.inv = 1.0f / q.sp;
    if (q.bad) q.s = __builtin_nanf("");
    return q;
}

/* x / s for a rounding to fewer bits: the nearest f32 towards which the exact
 * quotient lies, with its last bit set wherever the quotient is not exact
 * (rounding to odd), so that rounding it to e4m3 gives what rounding the
 * exact quotient gives.  x / s rounded to f32 alone would not: bf16
 * activations stand in ratios of few bits, and one quotient in some hundreds
 * of a block lies within 2^-24 of the middle between two codes.  q1 is within
 * one step of the quotient, the sign of its residual (exact in one fma) says
 * on which side. */
__device__ __forceinline__ float fp8_quotient(float x, const Fp8Scale &q) {
    const float xp = x * q.pre;
    const float q0 = xp * q.inv;
    const float q1 = fmaf(fmaf(-q0, q.sp, xp), q.inv, q0);
    const float r = fmaf(-q1, q.sp, xp);
    uint32_t b = __builtin_bit_cast(uint32_t, q1);
    const uint32_t odd = (b + (uint32_t)((int32_t)(__builtin_bit_cast(uint32_t, r) ^ b) >> 31)) | 1u;
    return __builtin_bit_cast(float, r != 0.0f ? odd : b);
}

/* Four quotients' codes in one word. */
__device__ __forceinline__ uint32_t fp8_code4(float a, float b, float c, float d, const Fp8Scale &q) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(a, q), fp8_quotient(b, q), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(c, q), fp8_quotient(d, q), w, true);
    return q.bad ? 0x7F7F7F7Fu : (uint32_t)w;
}

/* The same for values that carry f32 roundings themselves (h of the experts):
 * x times 1 / s, within 2^-23 of the quotient. */
__device__ __forceinline__ uint32_t fp8_near4(float a, float b, float c, float d, const Fp8Scale &q, float inv) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
    return q.bad ? 0x7F7F7F7Fu : (uint32_t)w;
}

__device__ __forceinline__ uint32_t fp8_absbits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

/* Eight lanes' share of one block to quantize: lane `part` holds groups of G
 * consecutive columns, the lanes' groups side by side, so that each load
 * instruction reads whole 128-byte lines. */
template <bool F32>
struct Fp8Block {
    static constexpr int G = F32 ? 4 : 8, N = 16 / G;
    r9vx_u32x4 w[N];

    static __device__ __forceinline__ uint32_t column(int j, uint32_t part) { return (j * 8 + part) * G; }
    /* x: the block's first value; `left` columns from there, zeros behind them */
    __device__ __forceinline__ void load(const uint8_t *x, uint32_t left, uint32_t part) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t c = column(j, part);
            w[j] = r9vx_u32x4{0u, 0u, 0u, 0u};
            if (c < left) w[j] = __builtin_nontemporal_load(reinterpret_cast<const r9vx_u32x4 *>(x + c * (F32 ? 4 : 2)));
        }
    }
    /* code: G / 4 words of each group; returns the block's scale */
    __device__ __forceinline__ float codes(uint32_t (&code)[4]) const {
        float v[16];
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            const uint32_t u = w[i / 4][i % 4]; /* a copy: bit_cast of a vector's element takes its first one */
            if constexpr (F32) {
                v[i] = __builtin_bit_cast(float, u);
            } else {
                v[2 * i] = __builtin_bit_cast(float, u << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, u & 0xFFFF0000u);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = max(amax, fp8_absbits(v[i]));
        const Fp8Scale s = fp8_scale(fp8_max8(amax));
#pragma unroll
        for (int i = 0; i < 4; ++i) code[i] = fp8_code4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s);
        return s.s;
    }
};

typedef _Float16 fp8_half2 __attribute__((ext_vector_type(2)));
typedef _Float16 fp8_half8 __attribute__((ext_vector_type(8)));

/* Eight codes as f16 (exact, NaN kept). */
__device__ __forceinline__ fp8_half8 fp8_widen(int lo, int hi) {
    const fp8_half2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)lo, 1.0f, false);
    const fp8_half2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)lo, 1.0f, true);
    const fp8_half2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)hi, 1.0f, false);
    const fp8_half2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)hi, 1.0f, true);
    return fp8_half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

/* One 16 x 16 tile over 128 columns, from zero: lane l gives 32 bytes of row
 * l % 16 of each operand and gets the products of column-operand row l % 16
 * with row-operand rows 4 (l / 16) .. + 3.  128 columns are one scale block,
 * so a step's sum leaves the matrix unit before the next block's scales.
 *
 * The 8-bit instruction adds each group of 8 neighbouring products in a window
 * of about 14 bits below the largest of them and only the groups' sums in f32
 * (measured: next to a product p, one of 2^-14 p in the same group is dropped,
 * in another group none is; 1.4e-5 of the result on normally distributed
 * codes).  EXACT widens the codes to f16, which holds every one of them, and
 * takes the f16 instruction, whose sums keep f32 throughout (1e-8 measured),
 * at half the rate. */
template <bool EXACT>
__device__ __forceinline__ r9vx_f32x4 fp8_mma(i32x8 rows, i32x8 cols) {
    if constexpr (!EXACT)
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(rows, cols, r9vx_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
    r9vx_f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 8; s += 2)
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp8_widen(rows[s], rows[s + 1]), fp8_widen(cols[s], cols[s + 1]), d, 0, 0, 0);
    return d;
}

__device__ __forceinline__ i32x8 fp8_frag(r9vx_u32x4 lo, r9vx_u32x4 hi) {
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

}  // namespace r9vx
#endif

/* Internal launchers (return hipError_t as int). */
/* ldq: columns of a row of codes, k or (zeros behind k) whole blocks. */
int r9vx_launch_quantize_fp8(const void *x, uint32_t x_dtype, uint64_t m, uint32_t k, uint32_t ldq, uint8_t *q, float *scales,
                             hipStream_t stream);
int r9vx_launch_pad_fp8(const uint8_t *x, uint32_t m, uint32_t k, uint8_t *q, hipStream_t stream);

struct r9vx_fp8_problem {
    const uint8_t *w;
    const float *w_scales;
    const void *x;
    const float *x_scales;
    const float *bias;
    const float *residual;
    void *y;
    uint8_t *workspace;
    uint32_t m, m_bucket, n, k, x_dtype, y_dtype, epilogue;
};
size_t r9vx_fp8_workspace_bytes(uint32_t m_bucket, uint32_t k, uint32_t x_dtype);
int r9vx_launch_matmul_fp8(const r9vx_fp8_problem &p, hipStream_t stream);

struct r9vx_moe_fp8_problem {
    const uint16_t *x;
    const uint32_t *ids;
    const float *weights;
    const uint8_t *w_gu, *w_dn;
    const float *s_gu, *s_dn;
    void *y;
    uint8_t *ws;
    uint32_t t, t_bucket, e, k, dm, dff, shared, y_dtype;
    uint32_t *status;     /* a refused call's bits are or-ed into it; NULL: none kept */
    uint32_t nan_refused; /* a refused call's y: NaN, otherwise left */
};
size_t r9vx_moe_fp8_workspace_bytes(const r9vx_moe_fp8_problem &p);
/* Whether t_bucket tokens' launches have no more threads than 32 bits count. */
bool r9vx_moe_fp8_launchable(const r9vx_moe_fp8_problem &p);
int r9vx_launch_moe_fp8(const r9vx_moe_fp8_problem &p, hipStream_t stream);
/* Device address of the status word in a workspace. */
const uint32_t *r9vx_moe_fp8_status_word(const r9vx_moe_fp8_problem &p);

#endif
