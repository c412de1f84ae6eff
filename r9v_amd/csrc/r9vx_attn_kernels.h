/*
 * r9vx_attn_kernels.h -- what the attention kernels share: the problem as the
 * launchers take it, the two element types, the score and its mask.
 */
#ifndef R9VX_ATTN_KERNELS_H
#define R9VX_ATTN_KERNELS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "r9vx_attn.h"
#include "r9vx_attn_index.h"
#include "r9vx_device.h"
#include "r9vx_internal.h"

struct r9vx_rope_problem {
    const void *q, *k, *v;
    const int32_t *positions;
    const double *freqs;
    void *q_out, *k_cache, *v_cache;
    const int64_t *slots;
    uint32_t *status;
    uint64_t q_stride[2], k_stride[2], v_stride[2], q_out_stride[2], k_cache_stride[3], v_cache_stride[3];
    uint32_t pages, t, heads, kv_heads, head_dim, rot, interleaved, page_shift, in_dtype, out_dtype;
    float amplitude;
};
int r9vx_launch_rope_kv(const r9vx_rope_problem &p, hipStream_t stream);

struct r9vx_attn_problem {
    const uint16_t *q, *k, *v;
    const int32_t *table, *lengths, *offsets, *starts, *prefix;
    const float *slopes;
    uint16_t *out;
    float *partial;   /* f32 [rows][splits][head_dim], then (m, l) [rows][splits] */
    uint32_t *status;
    uint64_t q_stride[3], out_stride[3], k_stride[3], v_stride[3], table_stride;
    uint32_t pages, b, t, b_bucket, t_bucket, len_bucket, heads, kv_heads, group, group_magic, head_dim, page_shift, dtype, causal, window;
    uint32_t splits, parts, part_blocks; /* parts of a row's keys in the grid; those a row is cut into, of at most part_blocks blocks (attn_part) */
    uint32_t halves; /* prefill: of a part's keys, for four waves each */
    float scale, softcap;
};
/* Sets splits, parts, part_blocks and halves: by the static alone. */
void r9vx_attn_decode_plan(r9vx_attn_problem &p);
void r9vx_attn_prefill_plan(r9vx_attn_problem &p);
int r9vx_launch_attn_decode(const r9vx_attn_problem &p, hipStream_t stream);
int r9vx_launch_attn_prefill(const r9vx_attn_problem &p, hipStream_t stream);
/* out from the parts of rows [0, rows): row r is token r / heads, head r % heads. */
int r9vx_launch_attn_join(const r9vx_attn_problem &p, uint64_t rows, hipStream_t stream);
uint64_t r9vx_attn_join_groups(const r9vx_attn_problem &p, uint64_t rows);
/* Workgroups a launch of these sizes has (the API refuses more than 32 bits of threads). */
uint64_t r9vx_attn_decode_groups(const r9vx_attn_problem &p);
uint64_t r9vx_attn_prefill_groups(const r9vx_attn_problem &p);

/* A part that saw nothing has the maximum -infinity and the sum 0; one that saw
 * scores of -infinity alone the sum NaN, which the join gives out where no part
 * saw more. */
#ifdef __HIPCC__
namespace r9vx {

typedef _Float16 attn_f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t attn_u32x3 __attribute__((ext_vector_type(3)));

constexpr float kLog2e = 1.4426950408889634f;

/* How far (in powers of two) a row's largest score may be above its reference. */
constexpr float kAttnSlack = 8.0f;

/* The largest cap whose scores take the short form: 5 * 2^-23 of it, the form's error,
 * moves a probability by 8e-5 at most (half an f16 step is 24e-5).  8192 causal tokens of
 * 32 heads of 128 columns take 727 us at a cap of 50 and 830 at one of 1000. */
constexpr float kAttnShortCap = 128.0f;

/* The two element types.  kTop is the exponent that the largest probability of a row is
 * given at most: f16 holds 2^-24 at the least, so 15 there (the largest is 2^7 to 2^15 where
 * the reference lags by kAttnSlack); bf16 has f32's exponents, and -32 keeps the sums of
 * 2^30 values of any size finite. */
struct AttnBf16 {
    typedef r9vx_bf16x8 x8;
    typedef __bf16 elem;
    static constexpr bool kWide = true; /* f32's exponents */
    static constexpr float kTop = -32.0f;
    static constexpr uint32_t kNan = 0x7FC07FC0u, kOnes = 0x3F803F80u;
    /* c and the eight elements, in f32 */
    static __device__ __forceinline__ float add8(x8 x, float c) {
        const r9vx_u32x4 w = __builtin_bit_cast(r9vx_u32x4, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = r9vx_dot2_bf16(w[i], kOnes, c);
        return c;
    }
    static __device__ __forceinline__ r9vx_f32x4 mma16(x8 a, x8 b, r9vx_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ r9vx_f32x16 mma32(x8 a, x8 b, r9vx_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
struct AttnF16 {
    typedef attn_f16x8 x8;
    typedef _Float16 elem;
    static constexpr bool kWide = false;
    static constexpr float kTop = 15.0f;
    static constexpr uint32_t kNan = 0x7E007E00u, kOnes = 0x3C003C00u;
    static __device__ __forceinline__ float add8(x8 x, float c) {
        const r9vx_u32x4 w = __builtin_bit_cast(r9vx_u32x4, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = r9vx_dot2_f16(w[i], kOnes, c);
        return c;
    }
    static __device__ __forceinline__ r9vx_f32x4 mma16(x8 a, x8 b, r9vx_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ r9vx_f32x16 mma32(x8 a, x8 b, r9vx_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

/* A key's row where there is none (zeros: a value nobody sees must not be a NaN
 * beside a probability of zero), and that of a page outside the cache (NaN: a
 * score that sees it is one). */
static __device__ const uint32_t kAttnZeroRow[128] = {};
template <class T>
__device__ __forceinline__ const uint16_t *attn_nan_row();
#define R9VX_ROW16(x) x, x, x, x, x, x, x, x, x, x, x, x, x, x, x, x
#define R9VX_ROW128(x) R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x), R9VX_ROW16(x)
static __device__ const uint32_t kAttnNanBf16[128] = {R9VX_ROW128(AttnBf16::kNan)};
static __device__ const uint32_t kAttnNanF16[128] = {R9VX_ROW128(AttnF16::kNan)};
template <>
__device__ __forceinline__ const uint16_t *attn_nan_row<AttnBf16>() { return reinterpret_cast<const uint16_t *>(kAttnNanBf16); }
template <>
__device__ __forceinline__ const uint16_t *attn_nan_row<AttnF16>() { return reinterpret_cast<const uint16_t *>(kAttnNanF16); }

/* What turns products into exponents of two, x = score * log2(e).  The query's sign
 * is the scale's (attn_signed), so that the largest product is the largest score;
 * a scale of zero makes it zeros.  A cap and a bias are applied to the
 * products first and leave them in units of 1 / log2(e): factor 1. */
struct AttnScore {
    float factor; /* of what is left of a product */
    float before; /* of a product before a bias */
    float inner;  /* 2 log2(e) scale / cap */
    float cap;    /* cap * log2(e) */
    __device__ __forceinline__ explicit AttnScore(const r9vx_attn_problem &a) {
        const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
        const bool capped = a.softcap > 0.0f, bias = a.slopes != nullptr;
        cap = a.softcap * kLog2e;
        inner = capped ? 2.0f * kLog2e * scale / a.softcap : 0.0f;
        before = capped ? 1.0f : scale * kLog2e;
        factor = capped || bias ? 1.0f : scale * kLog2e;
    }
    /* cap tanh(y), up to kAttnShortCap: 1 - 2 / (e^2y + 1), whose error of a few 2^-23 is
     * absolute, times the cap.  e^2y = infinity gives the cap. */
    __device__ __forceinline__ float capped(float product) const {
        const float e = __builtin_amdgcn_exp2f(product * inner);
        return fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(e + 1.0f), cap);
    }
    /* Above it: for |y| below 1/4 the score times the series of tanh(y) / y (the first term
     * left out is 1e-8 of it), beyond, where the cap is at most 4.1 times what comes out, the short
     * form.  In x = 2 log2(e) y, with ln(2) / 2 = 0.34657: no factors beside the short form's. */
    __device__ __forceinline__ float capped_far(float product) const {
        constexpr double k = 0.34657359027997265471, k2 = k * k;
        const float x = product * inner, t = x * x;
        const float series = fmaf(t, fmaf(t, fmaf(t, fmaf(t, (float)(k * k2 * k2 * k2 * k2 * 62 / 2835), (float)(-k * k2 * k2 * k2 * 17 / 315)), (float)(k * k2 * k2 * 2 / 15)),
                                          (float)(-k * k2 / 3)), (float)k);
        return fabsf(x) < (float)(0.25 / k) ? x * series * cap : capped(product);
    }
};

/* Eight elements of a query, with a scale's sign (zeros for one of zero). */
template <class T>
__device__ __forceinline__ typename T::x8 attn_signed(const r9vx_attn_problem &a, typename T::x8 q) {
    r9vx_u32x4 w = __builtin_bit_cast(r9vx_u32x4, q);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale == 0.0f ? 0u : ~0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ flip) & keep;
    return __builtin_bit_cast(typename T::x8, w);
}

/* A key's row of keys or values. */
template <class T>
__device__ __forceinline__ const uint16_t *attn_row(AttnPlace where, const uint16_t *base, const uint64_t *stride, uint32_t page, uint32_t place) {
    const uint16_t *p = base + page * stride[0] + place * stride[1];
    return where == kAttnKept ? p : where == kAttnBad ? attn_nan_row<T>() : reinterpret_cast<const uint16_t *>(kAttnZeroRow);
}

/* Bits of a pair of elements whose exponent is that of an infinity or a NaN. */
template <class T>
__device__ __forceinline__ uint32_t attn_odd(uint32_t w) {
    constexpr uint32_t e = T::kWide ? 0x7F80u : 0x7C00u;
    return ((w & e) == e ? 0xFFFFu : 0u) | ((w >> 16 & e) == e ? 0xFFFF0000u : 0u);
}

/* A weight of a sum that may hold an infinity: 0 times it would be none.  (Times a
 * finite sum the least number adds nothing that counts.) */
__device__ __forceinline__ float attn_some(float f) { return f < 0x1p-149f ? 0x1p-149f : f; }

typedef __attribute__((address_space(4))) const r9vx_attn_problem attn_kernel_args; /* a kernel's first argument, read again */

/* The larger of the two half waves' values. */
__device__ __forceinline__ float attn_max32(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

/* The other half wave's value. */
__device__ __forceinline__ float attn_swap32(float x) { return __shfl_xor(x, 32, R9VX_WAVE); }

}  // namespace r9vx
#endif
#endif
