/*
 * attn_rope.hip -- rotary positions, and keys and values into the paged cache.
 *
 *   a = position * freq[i];  (x, y) -> amplitude * (x cos a - y sin a, x sin a + y cos a)
 *
 * The angle is taken in turns in f64 and reduced there (a position of 2^20 times
 * a 24-bit frequency would be off by a sixteenth of a radian); cosine and sine of
 * what is left in f32.  A workgroup takes one token, or a part of its heads where
 * the tokens are few: rot / 2 of its threads make the token's cosines and sines
 * once, into LDS, and each thread turns 8 or 2 x 8 columns of a head by 16-byte
 * accesses, whose loads go out before the angles are worked on.
 *
 * Bound by memory where the tokens are many: 8192 tokens of 32 + 2 x 8 heads of
 * 128 columns, 201 MB read and written, 38 us (5.2 TB/s; a large copy reaches
 * 5.4); by the launch and two loads in turn where they are few: one token of 16 + 2 x 2
 * heads of 256 columns 3.6 us in a graph.
 */
#include "r9vx_attn_kernels.h"

using namespace r9vx;

namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 256; /* head_dim 512 */

struct RopeArgs {
    r9vx_rope_problem p;
    uint32_t per_head, per_copy, items, parts; /* work items of a turned head, of a copied one, of a token; workgroups of a token */
};

/* Eight elements as f32, and back. */
template <class E>
__device__ __forceinline__ void load8(const E *p, float (&x)[8]) {
    typedef E vec __attribute__((ext_vector_type(8)));
    const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
template <class E>
__device__ __forceinline__ void store8(E *p, const float (&x)[8]) {
    typedef E vec __attribute__((ext_vector_type(8)));
    vec v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (E)x[i];
    *reinterpret_cast<vec *>(p) = v;
}

template <class I, class O>
__global__ __launch_bounds__(kThreads) void rope_kv_kernel(RopeArgs a) {
    const r9vx_rope_problem &p = a.p;
    __shared__ float cs[kMostPairs], sn[kMostPairs];
    const uint32_t t = blockIdx.x / a.parts, part = blockIdx.x - t * a.parts;
    const uint32_t half = p.rot / 2;

    const int64_t slot = p.kv_heads ? p.slots[t] : -1;
    const int64_t slots = (int64_t)p.pages << p.page_shift;
    const bool kept = slot >= 0 && slot < slots;
    if (!kept && slot != -1 && threadIdx.x == 0 && part == 0 && p.status) atomicOr(p.status, R9VX_STATUS_BAD_SLOT);
    const uint64_t page = kept ? (uint64_t)slot >> p.page_shift : 0, place = kept ? (uint64_t)slot & ((1u << p.page_shift) - 1) : 0;

    for (uint32_t i = threadIdx.x; i < half; i += kThreads) {
        const double turns = (double)p.positions[t] * p.freqs[i] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cs[i] = p.amplitude * c;
        sn[i] = p.amplitude * s;
    }
    __syncthreads();

    const uint32_t turned = (p.heads + p.kv_heads) * a.per_head, step = a.parts * kThreads;
    const uint32_t pairs = p.interleaved ? p.rot / 8 : p.rot / 16; /* items of a head that turn; the others copy */
    for (uint32_t item = part * kThreads + threadIdx.x; item < a.items; item += step) {
        if (item < turned) {
            const uint32_t h = item / a.per_head, i = item - h * a.per_head;
            const bool key = h >= p.heads;
            const uint32_t kh = h - p.heads;
            if (key && !kept) continue;
            const I *x = key ? static_cast<const I *>(p.k) + t * p.k_stride[0] + kh * p.k_stride[1]
                             : static_cast<const I *>(p.q) + t * p.q_stride[0] + h * p.q_stride[1];
            O *y = key ? static_cast<O *>(p.k_cache) + page * p.k_cache_stride[0] + place * p.k_cache_stride[1] + kh * p.k_cache_stride[2]
                       : static_cast<O *>(p.q_out) + t * p.q_out_stride[0] + h * p.q_out_stride[1];
            float u[8], w[8];
            if (i >= pairs) {
                const uint32_t c = p.rot + 8 * (i - pairs);
                load8(x + c, u);
                store8(y + c, u);
            } else if (p.interleaved) {
                load8(x + 8 * i, u);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float c = cs[4 * i + j], s = sn[4 * i + j], x0 = u[2 * j], x1 = u[2 * j + 1];
                    u[2 * j] = fmaf(x0, c, -(x1 * s));
                    u[2 * j + 1] = fmaf(x0, s, x1 * c);
                }
                store8(y + 8 * i, u);
            } else {
                load8(x + 8 * i, u);
                load8(x + half + 8 * i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float c = cs[8 * i + j], s = sn[8 * i + j], x0 = u[j], x1 = w[j];
                    u[j] = fmaf(x0, c, -(x1 * s));
                    w[j] = fmaf(x0, s, x1 * c);
                }
                store8(y + 8 * i, u);
                store8(y + half + 8 * i, w);
            }
        } else if (kept) {
            const uint32_t h = (item - turned) / a.per_copy, c = 8 * (item - turned - h * a.per_copy);
            float u[8];
            load8(static_cast<const I *>(p.v) + t * p.v_stride[0] + h * p.v_stride[1] + c, u);
            store8(static_cast<O *>(p.v_cache) + page * p.v_cache_stride[0] + place * p.v_cache_stride[1] + h * p.v_cache_stride[2] + c, u);
        }
    }
}

template <class I, class O>
int launch(const RopeArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL((rope_kv_kernel<I, O>), dim3(a.p.t * a.parts), dim3(kThreads), 0, stream, a);
    return (int)hipGetLastError();
}

}  // namespace

int r9vx_launch_rope_kv(const r9vx_rope_problem &p, hipStream_t stream) {
    RopeArgs a{};
    a.p = p;
    a.per_head = (p.interleaved ? p.rot / 8 : p.rot / 16) + (p.head_dim - p.rot) / 8;
    a.per_copy = p.head_dim / 8;
    a.items = (p.heads + p.kv_heads) * a.per_head + p.kv_heads * a.per_copy;
    /* one round of items a workgroup where the tokens alone do not fill the card */
    const uint32_t most = (a.items + kThreads - 1) / kThreads;
    const uint32_t fill = 4 * r9vx_device_cus();
    a.parts = p.t >= fill ? 1 : (fill + p.t - 1) / p.t;
    if (a.parts > most) a.parts = most;
    const bool f32 = p.in_dtype == R9VX_DTYPE_F32;
    switch (p.out_dtype) {
    case R9VX_DTYPE_BF16: return f32 ? launch<float, __bf16>(a, stream) : launch<__bf16, __bf16>(a, stream);
    case R9VX_DTYPE_F16: return f32 ? launch<float, _Float16>(a, stream) : launch<_Float16, _Float16>(a, stream);
    default: return launch<float, float>(a, stream);
    }
}
