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
 * card the keys are cut into parts, joined by a further launch, or into halves of
 * parts for two times four waves, joined through LDS.
 *
 * A tile's 1024 cycles of matrix instructions and its 700 or so of exponentials,
 * maxima and conversions overlap only where the two workgroups of a CU are at different
 * phases: 8192 causal tokens of 32 heads of 128 columns 532 to 583 us, 0.94 to 1.03 of
 * the matrix unit's 2.5 PFLOP/s (a large product reaches 1.47).
 * Eight waves at opposite phases behind shared barriers took 568 when this form
 * took 561, a tile's products in halves around the softmax no less: registers spilt.
 * A workgroup takes 5 us before its first tile is done: 17 tokens 12 us.  Heads of 256
 * columns fill the 256 registers and spill some; the other widths spill none.
 */
#include "r9vx_attn_kernels.h"

using namespace r9vx;

namespace {

constexpr int kRows = 128; /* of a workgroup */
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves; /* times the halves */

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

/* 16 bytes of each lane of `lanes` from `base` + `off` (bytes) in global memory to LDS at
 * `at` + 16 * lane.  Within straight-line code: a branch around it would cut the
 * schedule in pieces.  (No "memory": it writes a buffer that is read behind the next
 * barrier alone, and may stand among reads of the other.)  `base` comes from v_readlane:
 * a scalar register that a vector instruction wrote is a memory instruction's to read
 * five wait states later, which neither the hardware nor, in here, the compiler sees
 * to.  Two are the instructions before the load, three s_nop's. */
__device__ __forceinline__ void attn_copy16(uint32_t at, const uint16_t *base, uint32_t off, uint64_t lanes) {
    uint64_t all;
    asm volatile("s_mov_b32 m0, %3\n\ts_and_saveexec_b64 %0, %4\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, %0"
                 : "=&s"(all) : "v"(off), "s"(base), "s"(at), "s"(lanes) : "m0", "scc");
}

/* `lanes` or none, as attn_copy16 takes them: in scalar registers. */
__device__ __forceinline__ uint64_t attn_lanes(bool on, uint64_t lanes) {
    uint32_t lo = __builtin_amdgcn_readfirstlane(on ? (uint32_t)lanes : 0u), hi = __builtin_amdgcn_readfirstlane(on ? (uint32_t)(lanes >> 32) : 0u);
    asm volatile("" : "+s"(lo), "+s"(hi));
    return (uint64_t)hi << 32 | lo;
}

/* A wave at its products goes before one at its softmax (8192 causal tokens, 96
 * columns 262 -> 238 us, 192 457 -> 419, 64 353 -> 350; 128 and 256 took 562 and 572
 * without it, 570 and 579 with it). */
template <int D, int P>
__device__ __forceinline__ void attn_priority() {
    if constexpr (D % 128) __builtin_amdgcn_s_setprio(P);
}

template <int D, int H>
struct PrefillShared {
    __attribute__((aligned(1024))) uint16_t kv[H][4][PrefillShape<D>::TILE]; /* keys of two tiles, values of two; in the end the second half's sums */
    int bounds[kWaves];
    uint32_t redo, odds[H][2]; /* odds: keys of a tile with values that are not finite */
    float tops[H - 1 ? kThreads : 1], sums[H - 1 ? kThreads : 1];
};

/* A workgroup's rows.  CAREFUL: the second way through, which a workgroup takes where
 * the first one gave a NaN or an infinity: a value that a row does not see may have
 * brought it in through a probability of zero.  It takes such values out of LDS, and
 * adds each to the rows that see its key (times a probability, a NaN or an infinity is
 * itself).  Returns whether the second way has to be taken (nothing is written then).
 * FAR: of a cap above kAttnShortCap (both formulas in one loop cost calls without a cap 3
 * to 13 %: 8192 causal tokens 544 -> 559 us, a 300-token chunk onto 4096 47.6 -> 53.7). */
template <class T, int D, int H, bool FAR, bool CAREFUL>
__device__ __forceinline__ bool attn_prefill_rows(const r9vx_attn_problem &a, uint32_t tiles, PrefillShared<D, H> &sh) {
    using S = PrefillShape<D>;
    typedef typename T::x8 x8;
    constexpr int KT = S::KT, NK = KT / 32;
    uint32_t thread = threadIdx.x, id = blockIdx.x;
    if (CAREFUL) asm volatile("" : "+v"(thread), "+s"(id)); /* worked out anew: nothing is kept for this way through the first one's loop */
    const int lane = thread & 63, wave8 = __builtin_amdgcn_readfirstlane(thread >> 6), c32 = lane & 31, h2 = lane >> 5;
    const int half = H == 1 ? 0 : wave8 / kWaves, wave = H == 1 ? wave8 : wave8 % kWaves;
    auto &kv = sh.kv[half];
    auto &bounds = sh.bounds;
    auto &odds = sh.odds[half];
    const uint32_t kvh = id % a.kv_heads;
    id /= a.kv_heads;
    const uint32_t split = id % a.splits;
    const uint32_t tile = tiles - 1 - id / a.splits; /* the longest of a causal sequence first */

    if (tile == 0 && kvh == 0 && split == 0 && a.status) {
        bool odd = false;
        for (uint32_t i = thread; i < a.b; i += H * kThreads) odd |= a.offsets[i] < 0 || a.offsets[i] > a.offsets[i + 1] || (int64_t)a.offsets[i + 1] > a.t;
        if (odd) atomicOr(a.status, R9VX_STATUS_BAD_LENGTH);
    }
    AttnTile part;
    if (!attn_tile(a.offsets, a.b, a.t, a.group, kRows, tile, part)) return false;
    const uint32_t b = part.b, r0 = part.row;
    const int off = part.offset, news = part.n;
    const int length = a.lengths[b], prefix = a.prefix ? a.prefix[b] : 0;
    const bool bad_length = length < 0 || length > (int)a.len_bucket;
    if (bad_length && thread == 0 && a.status) atomicOr(a.status, R9VX_STATUS_BAD_LENGTH);

    /* this lane's row: the token and the head that row r0 + i is */
    const uint32_t rows = (uint32_t)news * a.group, i0 = wave * 32, t0 = r0 / a.group, h0 = r0 - t0 * a.group;
    auto token_of = [&](uint32_t i) { return (int)t0 + attn_token(h0 + i, a.group_magic); };
    const bool there = r0 + i0 + c32 < rows;
    const int token = there ? token_of(i0 + c32) : 0;
    const uint32_t head = kvh * a.group + (there ? h0 + i0 + c32 - (token - t0) * a.group : 0);
    const uint64_t at = (uint64_t)off + token;
    const int pos = length - news + token;
    int lo, hi;
    attn_seen(a.window, a.causal, pos, length, a.starts ? a.starts[at] : 0, prefix, lo, hi);
    if (!there || bad_length) lo = hi = 0;
    const bool some = lo < hi;
    x8 q[D / 16];
    const uint16_t *qrow = (there ? a.q + at * a.q_stride[1] + head * a.q_stride[2] : reinterpret_cast<const uint16_t *>(kAttnZeroRow)) + h2 * 8;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) q[s] = *(const __attribute__((address_space(1))) x8 *)(qrow + s * 16);
    if (a.scale <= 0.0f) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) q[s] = attn_signed<T>(a, q[s]);
    }
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    /* keys that all rows of the wave see, and those that some of the workgroup do: where
     * they begin and end grows with the token, but for the tokens' own starts */
    const uint32_t n0 = rows - r0 < (uint32_t)kRows ? rows - r0 : (uint32_t)kRows, n1 = i0 + 32 < n0 ? i0 + 32 : n0; /* rows of the workgroup; up to this wave's last (i0 >= n0: none is there) */
    int ulo, uhi, wfl, wfh, any;
    auto seen_by = [&](uint32_t i, int &from, int &to) { attn_seen(a.window, a.causal, length - news + token_of(i), length, 0, prefix, from, to); };
    seen_by(0, ulo, any);
    seen_by(n0 - 1, any, uhi);
    seen_by(i0 < n0 ? i0 : 0, any, wfh);
    seen_by(i0 < n0 ? n1 - 1 : 0, wfl, any);
    if (!CAREFUL && thread == 0) sh.redo = 0; /* (the second way is on while other waves read it) */
    if (a.starts) {
        int most = there ? lo : 0, least = some ? lo : INT32_MAX;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) most = max(most, __shfl_xor(most, s, R9VX_WAVE)), least = min(least, __shfl_xor(least, s, R9VX_WAVE));
        wfl = max(wfl, __builtin_amdgcn_readfirstlane(most));
        if (lane == 0) bounds[wave] = least;
        __syncthreads();
        least = min(min(bounds[0], bounds[1]), min(bounds[2], bounds[3]));
        ulo = max(ulo, __builtin_amdgcn_readfirstlane(least));
    }
    if (bad_length) ulo = uhi = 0;

    /* this part's tiles */
    const int k0 = ulo < uhi ? ulo / KT : 0, k1 = ulo < uhi ? (uhi + KT - 1) / KT : 0;
    int first, last; /* of the workgroup; then of this half */
    attn_part(k0, k1, 1, a.parts, a.part_blocks, split, first, last);
    const int steps = (last - first + H - 1) / H, begin = first + half * steps, end = H == 1 ? last : min(begin + steps, last);

    const AttnScore score(a);
    const uint16_t *kbase = a.k + kvh * a.k_stride[2], *vbase = a.v + kvh * a.v_stride[2];
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t mask = (1u << a.page_shift) - 1;

    float m, l;
    r9vx_f32x16 o[D / 32];
    constexpr uint32_t kTileBytes = 2 * S::TILE;
    constexpr uint64_t kLanes = ~0ull >> (64 - S::LANES);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)kv;

    /* Lane j of every wave has the page of the tile's j-th eight keys (page 0 where
     * nothing of them is seen or the cache has no such page: something has to be
     * copied, and is replaced in LDS); of two halves lane 32 + j the other half's.  Copy i
     * of a wave has rows R (wave + 4 i) .. of the tile, all in one eight and at the same
     * place in it for every i. */
    const int lrow = lane / S::CH, lpiece = lane % S::CH; /* (beyond the rows for lanes that copy nothing) */
    const int inside = S::R * wave % 8 + lrow;
    const uint32_t kstep = (uint32_t)(inside * a.k_stride[1] * 2), vstep = (uint32_t)(inside * a.v_stride[1] * 2);
    /* (nothing is done with what is loaded until the tile is copied: a wait here would be
     * one for the copies under way) */
    const int place8 = H == 1 ? 8 * lane : 8 * c32 + (h2 ? (half ? -steps : steps) * KT : 0);
    const int bound = H == 1 ? uhi : min(uhi, ((half ^ h2) ? last : first + steps) * KT);
    auto in_tile = [&](int key) { return (H == 1 ? lane : c32) < KT / 8 && key < bound && key + 8 > ulo; };
    auto page_of = [&](int t) -> uint32_t {
        const int key = t * KT + place8;
        return (uint32_t)table[(in_tile(key) ? key : ulo) >> a.page_shift];
    };
    auto no_page = [&](int t, uint32_t page) -> uint64_t { return __ballot(in_tile(t * KT + place8) && page >= a.pages); };
    /* where tile t's eights begin, in lane j's registers; copy i of them into a buffer */
    auto source = [&](int t, uint32_t page, const uint16_t *base, const uint64_t *stride) -> uint64_t {
        const uint32_t place = (uint32_t)(t * KT + place8) & mask, from = page < a.pages ? page : 0u;
        return (uint64_t)(base + from * stride[0] + place * stride[1]);
    };
    auto copy = [&](int i, uint64_t p, uint32_t step, uint32_t at, uint64_t on) {
        const int c = wave + kWaves * i, eight = S::R * c / 8;
        const uint64_t p8 = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), eight) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)p, eight);
        attn_copy16(__builtin_amdgcn_readfirstlane(lds + at + c * 1024), (const uint16_t *)p8, step + 16 * (lpiece ^ S::swizzle(S::R * c + lrow)), on);
    };

    /* where this lane's pieces are: of key c32 for a score, of keys 4 h2 + lane / 4 % 4 for the values */
    const int krow = S::row(c32), kpiece = h2 ^ S::swizzle(c32);
    const int vkey = 4 * h2 + (lane & 15) / 4, vpiece = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ S::swizzle(vkey);
    const int vrow = S::row(vkey) + 4 * (lane & 1);

    const int n = end - begin; /* (of the second half steps or one less) */
    constexpr int kEach = (2 * S::N + D / 16 - 1) / (D / 16); /* copies beside a score's step */
    static_assert(kEach * (D / 16) >= 2 * S::N);

    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
    r9vx_f32x16 sc[NK];
    x8 p[KT / 16];

    /* Tile t (of n) has landed.  What stands beside the keys that are seen is no value, a
     * key of a page that is not there makes NaN of the scores that see it. */
    auto landed = [&](int t, uint64_t nos) {
        const int key0 = (begin + t) * KT;
        const uint32_t no = (uint32_t)nos;
        /* (both halves come here or none: there are barriers) */
        if (!(CAREFUL || nos || (first + t) * KT < ulo || (H == 1 ? key0 : (first + steps + t) * KT) + KT > uhi)) return;
        if (CAREFUL && wave == 0 && lane == 0) odds[0] = odds[1] = 0;
        if (no && wave == 0 && lane == 0 && a.status) atomicOr(a.status, R9VX_STATUS_BAD_PAGE);
        if (CAREFUL) __syncthreads();
        if ((S::LANES == 64 || lane < S::LANES) && (H == 1 || t < n)) {
#pragma unroll 1
            for (int i = 0; i < S::N; ++i) {
                const int c = wave + kWaves * i, r = S::R * c + lrow;
                r9vx_u32x4 *at = reinterpret_cast<r9vx_u32x4 *>(kv[2 + (t & 1)] + c * 512 + 8 * lane);
                const bool lost = no >> (r / 8) & 1u;
                if (lost) *reinterpret_cast<r9vx_u32x4 *>(kv[t & 1] + c * 512 + 8 * lane) = r9vx_u32x4{T::kNan, T::kNan, T::kNan, T::kNan};
                if (lost || key0 + r < ulo || key0 + r >= uhi) {
                    *at = r9vx_u32x4{0u, 0u, 0u, 0u};
                } else if (CAREFUL) {
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
    };

    if (steps > 0) {
        uint32_t page = page_of(begin);
        uint64_t kp = source(begin, page, kbase, a.k_stride), vp = source(begin, page, vbase, a.v_stride);
        uint64_t no = no_page(begin, page);
        const uint64_t lanes0 = attn_lanes(H == 1 || n > 0, kLanes);
#pragma unroll
        for (int i = 0; i < S::N; ++i) copy(i, kp, kstep, 0, lanes0), copy(i, vp, vstep, 2 * kTileBytes, lanes0);
        page = page_of(begin + 1);
        for (int t = 0; t < steps; ++t) {
            const int buf = t & 1, key0 = (begin + t) * KT;
            /* this tile has landed, and every wave is done with the other buffers */
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("" : "+v"(page)); /* used before the copies go out: a wait for it behind would be one for the copies */
            __syncthreads();
            landed(t, no);
            const bool more = t + 1 < n;
            no = H == 2 || more ? no_page(begin + t + 1, page) : 0u;
            const uint32_t to = (buf ^ 1) * kTileBytes;
            const uint64_t lanes = attn_lanes(more, kLanes);
            kp = source(begin + t + 1, page, kbase, a.k_stride), vp = source(begin + t + 1, page, vbase, a.v_stride);
            page = page_of(begin + t + 2);
            if (H == 2 && t >= n) break; /* (the last step) */
            const uint16_t *ks = kv[buf];
            uint16_t *vs = kv[2 + buf];
            attn_priority<D, 1>();
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[k][e] = 0.0f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
#pragma unroll
                for (int k = 0; k < NK; ++k)
                    sc[k] = T::mma32(*reinterpret_cast<const x8 *>(ks + S::row(32 * k) + krow + 8 * (kpiece ^ (2 * s))), q[s], sc[k]);
#pragma unroll
                for (int i = s * kEach; i < (s + 1) * kEach && i < 2 * S::N; ++i)
                    if (i < S::N) copy(i, kp, kstep, to, lanes);
                    else copy(i - S::N, vp, vstep, to + 2 * kTileBytes, lanes);
            }
            /* two steps' keys are on their way while a step's are multiplied */
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NK, 0);
#pragma unroll
            for (int s = 0; s < D / 16 - 2; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x8, NK, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, NK, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 2 * NK, 0);
            attn_priority<D, 0>();
            if (a.softcap > 0.0f) {
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[k][e] = FAR ? score.capped_far(sc[k][e]) : score.capped(sc[k][e]);
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
            top = attn_max32(top) * score.factor;
            /* a row's reference moves only where its largest score has grown by 2^8:
             * probabilities are then up to 2^8 times the reference's, and sums are rescaled seldom */
            const bool grown = top > m + kAttnSlack;
            if (__any(grown)) {
                float f = grown && m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 1.0f; /* (sums before the first score: zeros, or what is no number) */
                if (CAREFUL) f = attn_some(f);
                m = grown ? top : m;
                l *= f;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= f;
            }
            const float ref = (m == -INFINITY ? 0.0f : m) - (T::kTop - kAttnSlack);
            /* One number each: second halves would make half as many products again of a tile's, for
             * 1.6e-3 from the definition instead of 2.1e-3 (bf16, 8192 tokens). */
#pragma unroll
            for (int s = 0; s < KT / 16; ++s) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    p[s][e] = (typename T::elem)__builtin_amdgcn_exp2f(fmaf(sc[s >> 1][8 * (s & 1) + e], score.factor, -ref));
                l = T::add8(p[s], l); /* of what is multiplied, in f32: a rounding moves the weights among each other alone */
            }
            attn_priority<D, 1>();
#pragma unroll
            for (int s = 0; s < KT / 16; ++s)
#pragma unroll
                for (int d = 0; d < D / 32; ++d) { /* 8 keys of column 32 d + c32: 16 s + 4 h2 .. + 3 and 8 further */
                    uint16_t *v = vs + S::row(16 * s) + vrow + 8 * (vpiece ^ (4 * d)), *w = vs + S::row(16 * s + 8) + vrow + 8 * (vpiece ^ (4 * d) ^ 2);
                    const attn_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)v), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn_lds_s4 *)w);
                    o[d] = T::mma32(__builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), p[s], o[d]);
                }
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * 4, 0);
#pragma unroll
            for (int s = 0; s < KT / 16 * (D / 32) - 4; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
            attn_priority<D, 0>();
            if (CAREFUL) {
#pragma unroll 1
                for (int r = 0; r < KT; ++r) {
                    const int key = key0 + r;
                    if (!(odds[r / 32] >> (r % 32) & 1u) || key < lo || key >= hi) continue;
                    const uint32_t own = (uint32_t)table[key >> a.page_shift];
                    const uint16_t *v = vbase + own * a.v_stride[0] + ((uint32_t)key & mask) * a.v_stride[1]; /* (a page that is not there has no odd value) */
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
    if constexpr (H == 2) { /* the second half's sums through LDS to the first */
        r9vx_f32x4 *far = reinterpret_cast<r9vx_f32x4 *>(sh.kv[0][0]) + wave * (D / 8 * 64) + lane;
        static_assert(kWaves * (D / 8) * 64 * 16 <= (int)sizeof(sh.kv));
        __syncthreads(); /* the last tiles have been read */
        if (half) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; e += 4) far[(4 * d + e / 4) * 64] = r9vx_f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            sh.tops[wave * 64 + lane] = m, sh.sums[wave * 64 + lane] = l;
        }
        __syncthreads();
        if (!half) {
            const float m1 = sh.tops[wave * 64 + lane], top = fmaxf(m, m1);
            /* a half that saw nothing (or scores of -infinity alone) has zeros, or a NaN of NaN scores */
            float f0 = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top), f1 = m1 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m1 - top);
            if (CAREFUL) f0 = attn_some(f0), f1 = attn_some(f1);
            l = l * f0 + sh.sums[wave * 64 + lane] * f1;
            m = top;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const r9vx_f32x4 y = far[(4 * d + e / 4) * 64];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][e + i] = o[d][e + i] * f0 + y[i] * f1;
                }
        }
    }
    if (!CAREFUL) {
        float zero = l * 0.0f; /* or a NaN where something is not finite */
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) zero = fmaf(o[d][e], 0.0f, zero);
        if (!half && __any(zero != 0.0f && there) && lane == 0) sh.redo = 1;
        __syncthreads();
        if (sh.redo) return true;
    }
    if (!there || half) return false;
    float sum = l, top = m;
    if (bad_length || (sum != sum && top == -INFINITY)) top = 0.0f; /* a NaN that counts beside any other part */
    if (bad_length || (sum == 0.0f && top == -INFINITY && max(lo, first * KT) < min(hi, last * KT))) sum = __builtin_nanf("");
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
    return false;
}

template <class T, int D, int H, bool FAR>
__global__ __launch_bounds__(H * kThreads, 2) void attn_prefill_kernel(r9vx_attn_problem a, uint32_t tiles) {
    __shared__ PrefillShared<D, H> sh;
    if (!attn_prefill_rows<T, D, H, FAR, false>(a, tiles, sh)) return;
    /* (in line: as a function it took 300 to 790 bytes of scratch a lane, 390 MB of a card's memory, and
     * registers that left 64 columns two waves a SIMD instead of three: 8192 tokens 375 us, 355 so) */
    uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args), "+s"(tiles));
    const r9vx_attn_problem again = *(const r9vx_attn_problem *)(attn_kernel_args *)args;
    attn_prefill_rows<T, D, H, FAR, true>(again, tiles, sh);
}

template <class T, int D, bool FAR>
void launch_halves(const r9vx_attn_problem &p, hipStream_t stream) {
    const uint32_t tiles = attn_tiles(p.t, p.b, p.group, kRows);
    const dim3 grid((unsigned)r9vx_attn_prefill_groups(p));
    if (p.halves == 2) hipLaunchKernelGGL((attn_prefill_kernel<T, D, 2, FAR>), grid, dim3(2 * kThreads), 0, stream, p, tiles);
    else hipLaunchKernelGGL((attn_prefill_kernel<T, D, 1, FAR>), grid, dim3(kThreads), 0, stream, p, tiles);
}

template <class T, int D>
void launch_columns(const r9vx_attn_problem &p, hipStream_t stream) {
    if (p.softcap > kAttnShortCap) launch_halves<T, D, true>(p, stream);
    else launch_halves<T, D, false>(p, stream);
}

template <class T>
int launch_prefill(const r9vx_attn_problem &p, hipStream_t stream) {
    switch (p.head_dim) {
    case 64: launch_columns<T, 64>(p, stream); break;
    case 96: launch_columns<T, 96>(p, stream); break;
    case 128: launch_columns<T, 128>(p, stream); break;
    case 192: launch_columns<T, 192>(p, stream); break;
    default: launch_columns<T, 256>(p, stream); break;
    }
    return (int)hipGetLastError();
}

}  // namespace

uint64_t r9vx_attn_prefill_groups(const r9vx_attn_problem &p) { return (uint64_t)attn_tiles(p.t, p.b, p.group, kRows) * p.kv_heads * p.splits; }

void r9vx_attn_prefill_plan(r9vx_attn_problem &p) {
    const uint64_t groups = (uint64_t)attn_tiles(p.t_bucket, p.b_bucket, p.group, kRows) * p.kv_heads;
    /* Where the rows are few: parts of 256 keys or more, so that there are two workgroups a
     * CU; or half as many parts for workgroups of two halves, one a CU, which join two in LDS:
     * half the sums to write and to join.  (us by parts and by halves: 300 tokens of 16 heads
     * of 256 columns onto 4096, 13 or 6 parts, 60 and 52; 700 tokens of 32 heads of 128, 2 or
     * 1, 31 and 22.)  Not where that leaves more CUs idle (512 tokens of 32 heads of 128 onto
     * 16384, 3 or 1: 183 and 244), nor where all parts are under way at once and are joined by
     * a launch in any case (4 x 40 tokens of 16 heads of 64 onto 2000, 8 or 4: 16.6 and 18). */
    const uint64_t fill = r9vx_device_cus(), keys = p.len_bucket;
    auto parts = [&](uint64_t places, uint64_t least) {
        const uint64_t s = groups ? places / groups : 1, most = (keys + least - 1) / least;
        return s < most ? (s < 64 ? s : 64) : most < 64 ? most : 64;
    };
    const uint64_t whole = parts(2 * fill, 256), halved = parts(fill, 512);
    p.halves = whole > 1 && 20 * halved >= 9 * whole && (halved == 1 || groups * whole > fill) ? 2 : 1;
    const uint64_t s = p.halves == 2 ? halved : whole;
    p.splits = p.parts = s > 1 ? (uint32_t)s : 1u;
    p.part_blocks = 1u << 27; /* no limit */
}

int r9vx_launch_attn_prefill(const r9vx_attn_problem &p, hipStream_t stream) {
    const int rc = p.dtype == R9VX_DTYPE_BF16 ? launch_prefill<AttnBf16>(p, stream) : launch_prefill<AttnF16>(p, stream);
    if (rc || p.splits == 1) return rc;
    return r9vx_launch_attn_join(p, (uint64_t)p.t * p.heads, stream);
}
