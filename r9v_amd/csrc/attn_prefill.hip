/*
 * attn_prefill.hip -- attention of packed prompts, or prompt chunks, over the
 * paged cache.
 *
 * A workgroup of four waves takes a sequence, a kv head and 128 of the rows that
 * share it (row = token * group + query head, so that a tile of few tokens still
 * fills the matrix unit and what a causal tile masks is a few tokens wide), and
 * runs over the keys that some of them sees, a tile at a time: keys and values
 * through registers into LDS, two buffers, one barrier a tile.  Scores are taken
 * transposed by 32 x 32 x 16 products, S^T = K Q^T: a lane then holds 16 keys
 * of one row in the order that the second product O^T = V^T P^T takes, so that
 * probabilities stay in registers; V^T comes from LDS by the transposing read.
 * Where the rows are too few to fill the card the keys are cut into parts,
 * joined by a further launch.
 */
#include "r9vx_attn_kernels.h"

using namespace r9vx;

namespace {

constexpr int kRows = 128;  /* of a workgroup */
constexpr int kWaves = 4;

typedef short attn_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) attn_s4 attn_lds_s4;

template <int D>
struct PrefillShape {
    static constexpr int KT = D > 128 ? 32 : 64;  /* keys of a tile */
    static constexpr int KP = D + 8;              /* a key's elements in LDS: 16 bytes more, so that rows start in other banks */
    static constexpr int VP = D + 32;
    static constexpr int N = KT * D / 8 / 256;    /* 16-byte pieces of a tile each thread moves */
};

template <class T, int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attn_prefill_kernel(r9vx_attn_problem a, uint32_t tiles) {
    using S = PrefillShape<D>;
    typedef typename T::x8 x8;
    constexpr int KT = S::KT, NK = KT / 32;
    __shared__ __attribute__((aligned(16))) uint16_t ks[2][KT * S::KP], vs[2][KT * S::VP];
    __shared__ int bounds[kWaves][4];
    __shared__ uint32_t redo;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c32 = lane & 31, h2 = lane >> 5;
    uint32_t id = blockIdx.x;
    const uint32_t kvh = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t split = id % a.splits;
    const uint32_t tile = tiles - 1 - id / a.splits; /* the longest of a causal sequence first */

    if (tile == 0 && kvh == 0 && split == 0 && a.status) {
        bool odd = false;
        for (uint32_t i = threadIdx.x; i < a.b; i += 256) odd |= a.offsets[i] < 0 || a.offsets[i] > a.offsets[i + 1] || (int64_t)a.offsets[i + 1] > a.t;
        if (odd) atomicOr(a.status, R9VX_STATUS_BAD_LENGTH);
    }
    AttnTile part;
    if (!attn_tile(a.offsets, a.b, a.t, a.group, kRows, tile, part)) return;
    const uint32_t b = part.b, r0 = part.row;
    const int off = part.offset, n = part.n;
    const int length = a.lengths[b];
    const bool bad_length = length < 0 || length > (int)a.len_bucket;
    if (bad_length && threadIdx.x == 0 && a.status) atomicOr(a.status, R9VX_STATUS_BAD_LENGTH);

    /* this lane's row */
    const uint32_t row = r0 + wave * 32 + c32;
    const bool there = row < (uint64_t)n * a.group;
    const int token = there ? (int)(row / a.group) : 0;
    const uint32_t head = kvh * a.group + (there ? row - token * a.group : 0);
    const uint64_t at = (uint64_t)off + token;
    const int pos = length - n + token;
    int lo, hi;
    attn_seen(a.window, a.causal, pos, length, a.starts ? a.starts[at] : 0, a.prefix ? a.prefix[b] : 0, lo, hi);
    if (!there || bad_length) lo = hi = 0;
    const bool some = lo < hi;
    x8 q[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        q[s] = x8{};
        if (there) q[s] = *reinterpret_cast<const x8 *>(a.q + at * a.q_stride[1] + head * a.q_stride[2] + s * 16 + h2 * 8);
    }
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    /* keys that some row of the wave (of the workgroup) sees, and those that all of them do */
    int wlo = some ? lo : INT32_MAX, whi = some ? hi : 0, wfl = there ? (some ? lo : INT32_MAX) : 0, wfh = there ? hi : INT32_MAX;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        wlo = min(wlo, __shfl_xor(wlo, s, R9VX_WAVE)), whi = max(whi, __shfl_xor(whi, s, R9VX_WAVE));
        wfl = max(wfl, __shfl_xor(wfl, s, R9VX_WAVE)), wfh = min(wfh, __shfl_xor(wfh, s, R9VX_WAVE));
    }
    wlo = __builtin_amdgcn_readfirstlane(wlo), whi = __builtin_amdgcn_readfirstlane(whi);
    wfl = __builtin_amdgcn_readfirstlane(wfl), wfh = __builtin_amdgcn_readfirstlane(wfh);
    if (lane == 0) bounds[wave][0] = wlo, bounds[wave][1] = whi;
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    const int ulo = min(min(bounds[0][0], bounds[1][0]), min(bounds[2][0], bounds[3][0]));
    const int uhi = max(max(bounds[0][1], bounds[1][1]), max(bounds[2][1], bounds[3][1]));

    /* this part's tiles */
    const int t0 = ulo < uhi ? ulo / KT : 0, t1 = ulo < uhi ? (uhi + KT - 1) / KT : 0;
    int begin, end;
    attn_part(t0, t1, 1, (int)a.splits, (int)split, begin, end);

    const AttnScore score(a);
    const uint16_t *kbase = a.k + kvh * a.k_stride[2], *vbase = a.v + kvh * a.v_stride[2];
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t mask = (1u << a.page_shift) - 1;

    float m, l;
    r9vx_f32x16 o[D / 32];
    r9vx_u32x4 kr[S::N], vr[S::N];
    uint32_t pages[S::N];

    auto look_up = [&](int t) {
#pragma unroll
        for (int i = 0; i < S::N; ++i) {
            const int key = t * KT + (int)(threadIdx.x + 256 * i) / (D / 8);
            pages[i] = key >= ulo && key < uhi ? (uint32_t)table[key >> a.page_shift] : 0u;
        }
    };
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < S::N; ++i) {
            const int c = (int)threadIdx.x + 256 * i, key = t * KT + c / (D / 8), e = c % (D / 8) * 8;
            const AttnPlace where = attn_place(pages[i], a.pages, key, ulo, uhi);
            const uint16_t *kp = attn_row<T>(where, kbase, a.k_stride, pages[i], (uint32_t)key & mask);
            const uint16_t *vp = attn_row<T>(where, vbase, a.v_stride, pages[i], (uint32_t)key & mask);
            kr[i] = *reinterpret_cast<const r9vx_u32x4 *>(kp + e);
            vr[i] = *reinterpret_cast<const r9vx_u32x4 *>(vp + e);
            if (where == kAttnBad && a.status) atomicOr(a.status, R9VX_STATUS_BAD_PAGE);
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < S::N; ++i) {
            const int c = (int)threadIdx.x + 256 * i, key = c / (D / 8), e = c % (D / 8) * 8;
            *reinterpret_cast<r9vx_u32x4 *>(&ks[buf][key * S::KP + e]) = kr[i];
            *reinterpret_cast<r9vx_u32x4 *>(&vs[buf][key * S::VP + e]) = vr[i];
        }
    };

    /* A first pass; a second one follows only where it gave a NaN or an infinity,
     * which a value that a row does not see may have brought into it through a
     * probability of zero.  The second pass then leaves out, token by token, the
     * values of each tile that not all rows see. */
    for (int pass = 0; pass < 2; ++pass) {
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
        if (begin < end) {
            look_up(begin);
            load(begin);
            if (begin + 1 < end) look_up(begin + 1);
            store(0);
        }
        __syncthreads();
        for (int t = begin; t < end; ++t) {
            const int buf = (t - begin) & 1;
            const int key0 = t * KT;
            if (t + 1 < end) {
                load(t + 1);
                if (t + 2 < end) look_up(t + 2);
            }
            if (key0 < whi && key0 + KT > wlo) {
                r9vx_f32x16 sc[NK];
#pragma unroll
                for (int k = 0; k < NK; ++k) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[k][e] = 0.0f;
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const x8 kf = *reinterpret_cast<const x8 *>(&ks[buf][(32 * k + c32) * S::KP + s * 16 + h2 * 8]);
                        sc[k] = T::mma32(kf, q[s], sc[k]);
                    }
                }
                const bool edge = key0 < wfl || key0 + KT > wfh;
                if (a.softcap > 0.0f) {
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[k][e] = score.capped(sc[k][e]);
                } else {
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[k][e] *= score.factor;
                }
                if (a.slopes) {
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int d = pos - (key0 + 32 * k + 8 * (e >> 2) + 4 * h2 + (e & 3));
                            sc[k][e] = fmaf(-slope, (float)(d < 0 ? -d : d), sc[k][e]);
                        }
                }
                if (edge) {
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int key = key0 + 32 * k + 8 * (e >> 2) + 4 * h2 + (e & 3);
                            if (key < lo || key >= hi) sc[k][e] = -INFINITY;
                        }
                }
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[k][e]);
                top = fmaxf(top, attn_swap32(top));
                if (__any(top > m)) {
                    const float now = fmaxf(m, top);
                    const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
                    m = now;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= f;
                }
                const float ref = (m == -INFINITY ? 0.0f : m) - T::kBits;
                x8 p[KT / 16];
#pragma unroll
                for (int s = 0; s < KT / 16; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = __builtin_amdgcn_exp2f(sc[s >> 1][8 * (s & 1) + e] - ref);
                        l += x;
                        p[s][e] = (typename T::elem)x;
                    }
                auto value = [&](int s, int d) -> x8 { /* 8 keys of column 32 d + c32: 16 s + 4 h2 .. + 3 and 8 further */
                    const uint16_t *v = &vs[buf][(16 * s + 4 * h2 + (lane & 15) / 4) * S::VP + 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
                    const attn_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)v);
                    const attn_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)(v + 8 * S::VP));
                    return __builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                if (pass == 0 || !edge) {
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
#pragma unroll
                        for (int s = 0; s < KT / 16; ++s) o[d] = T::mma32(value(s, d), p[s], o[d]);
                } else {
                    int done = -1;
                    for (int r = 0; r < 32; ++r) {
                        const int tok = __shfl(there ? token : -1, r, R9VX_WAVE);
                        if (tok == done || tok < 0) continue;
                        done = tok;
                        const int from = __shfl(lo, r, R9VX_WAVE), to = __shfl(hi, r, R9VX_WAVE);
#pragma unroll
                        for (int d = 0; d < D / 32; ++d) {
                            r9vx_f32x16 sum = o[d]; /* the same sum as the first pass's, for the rows whose keys these are */
#pragma unroll
                            for (int s = 0; s < KT / 16; ++s) {
                                typedef short s8 __attribute__((ext_vector_type(8)));
                                s8 v = __builtin_bit_cast(s8, value(s, d));
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const int key = key0 + 16 * s + 8 * (e >> 2) + 4 * h2 + (e & 3);
                                    v[e] = key >= from && key < to ? v[e] : (short)0;
                                }
                                sum = T::mma32(__builtin_bit_cast(x8, v), p[s], sum);
                            }
                            if (there && token == tok) o[d] = sum;
                        }
                    }
                }
            }
            if (t + 1 < end) store(buf ^ 1);
            __syncthreads();
        }
        l += attn_swap32(l);
        bool odd = !(fabsf(l) < INFINITY);
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) odd |= !(fabsf(o[d][e]) < INFINITY);
        if (pass == 0) {
            if (__any(odd && there) && lane == 0) redo = 1;
            __syncthreads();
            if (!redo) break;
        }
    }
    if (!there) return;
    float sum = l, top = m;
    if (bad_length || (sum != sum && top == -INFINITY)) top = 0.0f; /* a NaN that counts beside any other part */
    if (bad_length || (sum == 0.0f && top == -INFINITY && max(lo, begin * KT) < min(hi, end * KT))) sum = __builtin_nanf("");
    if (a.splits == 1) {
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t *y = a.out + at * a.out_stride[1] + head * a.out_stride[2];
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                typedef typename T::elem four __attribute__((ext_vector_type(4)));
                const four w = {(typename T::elem)(o[d][e] * f), (typename T::elem)(o[d][e + 1] * f), (typename T::elem)(o[d][e + 2] * f), (typename T::elem)(o[d][e + 3] * f)};
                *reinterpret_cast<four *>(y + 32 * d + 2 * e + 4 * h2) = w;
            }
    } else {
        const uint64_t r = (at * a.heads + head) * a.splits + split;
        float *y = a.partial + r * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) *reinterpret_cast<r9vx_f32x4 *>(y + 32 * d + 2 * e + 4 * h2) = r9vx_f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
        if (h2 == 0) {
            float2 *ml = reinterpret_cast<float2 *>(a.partial + (uint64_t)a.t_bucket * a.heads * a.splits * D);
            ml[r] = make_float2(top, sum);
        }
    }
}

template <class T>
int launch_prefill(const r9vx_attn_problem &p, hipStream_t stream) {
    const uint32_t tiles = attn_tiles(p.t, p.b, p.group, kRows);
    const dim3 grid((unsigned)r9vx_attn_prefill_groups(p)), block(256);
    switch (p.head_dim) {
    case 64: hipLaunchKernelGGL((attn_prefill_kernel<T, 64>), grid, block, 0, stream, p, tiles); break;
    case 96: hipLaunchKernelGGL((attn_prefill_kernel<T, 96>), grid, block, 0, stream, p, tiles); break;
    case 128: hipLaunchKernelGGL((attn_prefill_kernel<T, 128>), grid, block, 0, stream, p, tiles); break;
    case 192: hipLaunchKernelGGL((attn_prefill_kernel<T, 192>), grid, block, 0, stream, p, tiles); break;
    default: hipLaunchKernelGGL((attn_prefill_kernel<T, 256>), grid, block, 0, stream, p, tiles); break;
    }
    return (int)hipGetLastError();
}

}  // namespace

uint64_t r9vx_attn_prefill_groups(const r9vx_attn_problem &p) { return (uint64_t)attn_tiles(p.t, p.b, p.group, kRows) * p.kv_heads * p.splits; }

uint32_t r9vx_attn_prefill_splits(const r9vx_attn_problem &p) {
    const uint64_t groups = (uint64_t)attn_tiles(p.t_bucket, p.b_bucket, p.group, kRows) * p.kv_heads;
    const uint64_t fill = 2ull * r9vx_device_cus();
    const uint64_t most = ((uint64_t)p.len_bucket + 255) / 256; /* keys of a part: 256 or more */
    uint64_t s = groups ? fill / groups : 1;
    if (s > most) s = most;
    if (s > 64) s = 64;
    return s > 1 ? (uint32_t)s : 1u;
}

int r9vx_launch_attn_prefill(const r9vx_attn_problem &p, hipStream_t stream) {
    const int rc = p.dtype == R9VX_DTYPE_BF16 ? launch_prefill<AttnBf16>(p, stream) : launch_prefill<AttnF16>(p, stream);
    if (rc || p.splits == 1) return rc;
    return r9vx_launch_attn_join(p, (uint64_t)p.t * p.heads, stream);
}
