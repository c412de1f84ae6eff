/*
 * attn_prefill.hip -- attention of packed prompts, or prompt chunks, over the
 * paged cache.
 *
 * A workgroup of four waves takes a sequence, a kv head and 128 of the rows that
 * share it (row = token * group + query head, so that a tile of few tokens still
 * fills the matrix unit and what a causal tile masks is a few tokens wide), and
 * runs over the keys that some of them sees, a tile at a time: keys and values go
 * from the pages straight into LDS, the next tile's while this one is worked on,
 * one barrier a tile.  Scores are taken transposed by 32 x 32 x 16 products,
 * S^T = K Q^T: a lane then holds 16 keys of one row in the order that the second
 * product O^T = V^T P^T takes, so that probabilities stay in registers; V^T
 * comes from LDS by the transposing read.  Where the rows are too few to fill the
 * card the keys are cut into parts, joined by a further launch.
 */
#include "r9vx_attn_kernels.h"

using namespace r9vx;

namespace {

constexpr int kRows = 128; /* of a workgroup */
constexpr int kWaves = 4;

typedef short attn_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) attn_s4 attn_lds_s4;

template <int D>
struct PrefillShape {
    static constexpr int KT = D > 128 ? 32 : 64;             /* keys of a tile */
    static constexpr int CH = D / 8;                         /* 16-byte pieces of a key's row */
    static constexpr int R = CH <= 8 ? 8 : CH <= 16 ? 4 : 2; /* rows a wave copies at once, into 1 KiB: neighbours in one page */
    static constexpr int LANES = R * CH;                     /* of 64: all, or 48 for 96 and 192 columns */
    static constexpr int N = KT / R / kWaves;                /* copies of a tile's keys each wave makes */
    static constexpr int TILE = KT / R * 512;                /* elements of a tile's keys (of its values) in LDS */
    /* A row stands in LDS with its pieces' numbers xor-ed by swizzle(row), so that
     * both a score's reads (16 rows, the same piece) and the transposing ones (4
     * rows, 4 neighbouring pieces) meet each of the 64 banks once: rows of 256
     * bytes and their multiples start in one bank, of 128 and 384 in two, of 192
     * in four. */
    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (D == 96) return (r >> 2) & 3;
        else if constexpr (D % 128) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
        else return (r & 3) << 2 | ((r >> 2) & 3);
    }
    static __device__ __forceinline__ constexpr int row(int r) { return r / R * 512 + r % R * D; } /* its first element in LDS */
};

/* 16 bytes a lane from `base` + `off` (bytes) in global memory to LDS at `at` + 16 * lane. */
__device__ __forceinline__ void attn_copy16(uint32_t at, const uint16_t *base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory", "m0");
}

/* Bits of a pair of elements whose exponent is that of an infinity or a NaN. */
template <class T>
__device__ __forceinline__ uint32_t attn_odd(uint32_t w) {
    constexpr uint32_t e = T::kBits == 0.0f ? 0x7F80u : 0x7C00u;
    return ((w & e) == e ? 0xFFFFu : 0u) | ((w >> 16 & e) == e ? 0xFFFF0000u : 0u);
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void attn_prefill_kernel(r9vx_attn_problem a, uint32_t tiles) {
    using S = PrefillShape<D>;
    typedef typename T::x8 x8;
    constexpr int KT = S::KT, NK = KT / 32;
    __shared__ __attribute__((aligned(1024))) uint16_t kv[2][2][S::TILE]; /* buffer, keys and values */
    __shared__ int bounds[kWaves][2];
    __shared__ uint32_t redo, odds[2]; /* odds: keys of a tile with values that are not finite */

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31, h2 = lane >> 5;
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
        if (there) q[s] = attn_query<T>(a, a.q + at * a.q_stride[1] + head * a.q_stride[2] + s * 16 + h2 * 8);
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
    attn_part(t0, t1, 1, a.parts, a.part_blocks, split, begin, end);

    const AttnScore score(a);
    const uint16_t *kbase = a.k + kvh * a.k_stride[2], *vbase = a.v + kvh * a.v_stride[2];
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t mask = (1u << a.page_shift) - 1;

    float m, l;
    r9vx_f32x16 o[D / 32];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)kv;

    /* Lane j of every wave has the page of the tile's j-th eight keys (page 0 where
     * nothing of them is seen or the cache has no such page: something has to be
     * copied, and is replaced in LDS).  Copy i of a wave has rows R (wave + 4 i) ..
     * of the tile, all in one eight and at the same place in it for every i. */
    uint32_t page = 0, lacking = 0; /* lacking: eights of the next tile whose page the cache does not have */
    const int lrow = lane / S::CH, lpiece = lane % S::CH; /* (beyond the rows for lanes that copy nothing) */
    const int inside = S::R * wave % 8 + lrow;
    const uint32_t kstep = (uint32_t)(inside * a.k_stride[1] * 2), vstep = (uint32_t)(inside * a.v_stride[1] * 2);
    auto look_up = [&](int t) {
        const int key = t * KT + 8 * lane;
        if (lane < KT / 8) page = key < uhi && key + 8 > ulo ? (uint32_t)table[key >> a.page_shift] : 0u;
    };
    auto load = [&](int t, int buf) {
        const bool there = page < a.pages;
        const uint32_t place = (uint32_t)(t * KT + 8 * lane) & mask, from = there ? page : 0u;
        lacking = (uint32_t)__ballot(!there);
        const uint64_t kp = (uint64_t)(kbase + from * a.k_stride[0] + place * a.k_stride[1]), vp = (uint64_t)(vbase + from * a.v_stride[0] + place * a.v_stride[1]);
#pragma unroll
        for (int i = 0; i < S::N; ++i) {
            const int c = wave + kWaves * i, eight = S::R * c / 8;
            const uint32_t e = 16 * (lpiece ^ S::swizzle(S::R * c + lrow)), to = lds + (uint32_t)(buf * 4 * S::TILE + c * 1024);
            const uint64_t k8 = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(kp >> 32), eight) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)kp, eight);
            const uint64_t v8 = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(vp >> 32), eight) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)vp, eight);
            if (S::LANES == 64 || lane < S::LANES) {
                attn_copy16(to, (const uint16_t *)k8, kstep + e);
                attn_copy16(to + 2 * S::TILE, (const uint16_t *)v8, vstep + e);
            }
        }
        if (lacking && threadIdx.x == 0 && a.status) atomicOr(a.status, R9VX_STATUS_BAD_PAGE);
    };

    /* where this lane's pieces are: of key c32 for a score, of keys 4 h2 + lane / 4 % 4 for the values */
    const int krow = S::row(c32), kpiece = h2 ^ S::swizzle(c32);
    const int vkey = 4 * h2 + (lane & 15) / 4, vpiece = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ S::swizzle(vkey);
    const int vrow = S::row(vkey) + 4 * (lane & 1);

    /* A first pass; a second one follows only where it gave a NaN or an infinity,
     * which a value that a row does not see may have brought into it through a
     * probability of zero.  The second pass takes such values out of LDS, and
     * adds each to the rows that see its key (times a probability, a NaN or an
     * infinity is itself). */
    for (int pass = 0; pass < 2; ++pass) {
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
        if (begin < end) {
            look_up(begin);
            load(begin, 0);
            if (begin + 1 < end) look_up(begin + 1);
        }
        for (int t = begin; t < end; ++t) {
            const int buf = (t - begin) & 1;
            const int key0 = t * KT;
            /* this tile has landed, and every wave is done with the other buffer */
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const uint32_t gone = lacking;
            if (t + 1 < end) {
                load(t + 1, buf ^ 1);
                if (t + 2 < end) look_up(t + 2);
            }
            uint16_t *ks = kv[buf][0], *vs = kv[buf][1];
            if (pass || gone || key0 < ulo || key0 + KT > uhi) { /* what stands beside the keys that are seen is no value */
                if (threadIdx.x == 0) odds[0] = odds[1] = 0;
                __syncthreads();
                if (S::LANES == 64 || lane < S::LANES) {
#pragma unroll 1
                    for (int i = 0; i < S::N; ++i) {
                        const int r = S::R * (wave + kWaves * i) + lrow;
                        r9vx_u32x4 *at = reinterpret_cast<r9vx_u32x4 *>(vs + (wave + kWaves * i) * 512 + 8 * lane);
                        const bool lost = gone >> (r / 8) & 1u; /* a key that makes NaN of the scores that see it */
                        if (lost) at[-S::TILE / 8] = r9vx_u32x4{T::kNan, T::kNan, T::kNan, T::kNan};
                        if (lost || key0 + r < ulo || key0 + r >= uhi) {
                            *at = r9vx_u32x4{0u, 0u, 0u, 0u};
                        } else if (pass) {
                            r9vx_u32x4 w = *at;
                            uint32_t any = 0;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t x = attn_odd<T>(w[j]);
                                any |= x;
                                w[j] &= ~x;
                            }
                            if (any) {
                                *at = w;
                                atomicOr(&odds[r / 32], 1u << (r % 32));
                            }
                        }
                    }
                }
                __syncthreads();
            }
            if (key0 < whi && key0 + KT > wlo) {
                r9vx_f32x16 sc[NK];
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[k][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int k = 0; k < NK; ++k)
                        sc[k] = T::mma32(*reinterpret_cast<const x8 *>(ks + S::row(32 * k) + krow + 8 * (kpiece ^ (2 * s))), q[s], sc[k]);
                if (a.softcap > 0.0f) {
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[k][e] = score.capped(sc[k][e]);
                }
                if (a.slopes) {
                    const float far = (float)(pos - key0 - 4 * h2);
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            sc[k][e] = fmaf(-slope, fabsf(far - (float)(32 * k + 8 * (e >> 2) + (e & 3))), sc[k][e] * score.before);
                }
                if (key0 < wfl || key0 + KT > wfh) {
                    const int from = lo - key0 - 4 * h2, to = hi - key0 - 4 * h2;
#pragma unroll
                    for (int k = 0; k < NK; ++k)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int key = 32 * k + 8 * (e >> 2) + (e & 3);
                            if (key < from || key >= to) sc[k][e] = -INFINITY;
                        }
                }
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[k][e]);
                top = fmaxf(top, attn_swap32(top)) * score.factor;
                /* a row's reference moves only where its largest score has grown by 2^8:
                 * probabilities are then up to 2^8, and sums are rescaled seldom */
                const bool grown = top > m + kAttnSlack;
                if (__any(grown)) {
                    const float f = grown ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
                    m = grown ? top : m;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= f;
                }
                const float ref = (m == -INFINITY ? 0.0f : m) - T::kBits;
                x8 p[KT / 16];
#pragma unroll
                for (int s = 0; s < KT / 16; ++s) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        p[s][e] = (typename T::elem)__builtin_amdgcn_exp2f(fmaf(sc[s >> 1][8 * (s & 1) + e], score.factor, -ref));
                    l = T::add8(p[s], l); /* of what is multiplied, in f32 */
                }
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int s = 0; s < KT / 16; ++s) { /* 8 keys of column 32 d + c32: 16 s + 4 h2 .. + 3 and 8 further */
                        uint16_t *v = vs + S::row(16 * s) + vrow + 8 * (vpiece ^ (4 * d)), *w = vs + S::row(16 * s + 8) + vrow + 8 * (vpiece ^ (4 * d) ^ 2);
                        const attn_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)v), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)w);
                        o[d] = T::mma32(__builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), p[s], o[d]);
                    }
                if (pass) {
                    for (int r = 0; r < KT; ++r) {
                        const int key = key0 + r;
                        if (!(odds[r / 32] >> (r % 32) & 1u) || key < lo || key >= hi) continue;
                        const uint32_t own = (uint32_t)table[key >> a.page_shift];
                        const uint16_t *v = attn_row<T>(attn_place(own, a.pages, key, ulo, uhi), vbase, a.v_stride, own, (uint32_t)key & mask);
#pragma unroll
                        for (int d = 0; d < D / 32; ++d)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const uint16_t x = v[32 * d + 8 * (e >> 2) + 4 * h2 + (e & 3)];
                                if (attn_odd<T>(x)) o[d][e] += (float)__builtin_bit_cast(typename T::elem, x);
                            }
                    }
                }
            }
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

void r9vx_attn_prefill_plan(r9vx_attn_problem &p) {
    const uint64_t groups = (uint64_t)attn_tiles(p.t_bucket, p.b_bucket, p.group, kRows) * p.kv_heads;
    const uint64_t fill = 2ull * r9vx_device_cus();
    const uint64_t most = ((uint64_t)p.len_bucket + 255) / 256; /* keys of a part: 256 or more */
    uint64_t s = groups ? fill / groups : 1;
    if (s > most) s = most;
    if (s > 64) s = 64;
    p.splits = p.parts = s > 1 ? (uint32_t)s : 1u;
    p.part_blocks = 1u << 27; /* no limit */
}

int r9vx_launch_attn_prefill(const r9vx_attn_problem &p, hipStream_t stream) {
    const int rc = p.dtype == R9VX_DTYPE_BF16 ? launch_prefill<AttnBf16>(p, stream) : launch_prefill<AttnF16>(p, stream);
    if (rc || p.splits == 1) return rc;
    return r9vx_launch_attn_join(p, (uint64_t)p.t * p.heads, stream);
}
