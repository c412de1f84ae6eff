/*
 * attn_decode.hip -- attention of the next 1 to 8 tokens of each sequence over
 * the paged cache.
 *
 * A workgroup of four waves takes a sequence, a kv head, 16 or 32 of the rows
 * that share it (tokens x query heads of the group) and a part of the keys; the
 * waves take blocks of 32 keys in turn, each with a softmax of its own (running
 * maximum and sum), and are joined through LDS; parts are joined by a further
 * launch (r9vx_launch_attn_join).  A part is one of len_bucket's: those of a short
 * sequence that have no key write their zeros all the same (64 sequences of 500 keys 26 us,
 * 194 in a table for 131072).
 *
 * Scores are taken transposed, S^T = K Q^T by 16 x 16 x 32 products, with a
 * block's keys dealt to the two tiles so that what a lane holds of S^T, 8
 * neighbouring keys of one row, is what the second product O^T = V^T P^T
 * takes from it: probabilities never leave their lane.  Keys and values are loaded
 * by whole lines, a lane head_dim / 16 columns of 8 neighbouring keys; keys are
 * dealt out through a part of LDS that is the wave's own (loaded in the operand's
 * order, 16 rows at once, the same bytes took 116 us instead of 107 at 131072 keys
 * and 136 instead of 106 for 48 ragged sequences), values are turned in registers
 * (half a v_perm an element).
 *
 * Bound by the keys' and values' bytes: a wave keeps a block's keys or values on
 * their way while it works on the others.  131072 keys of 8 kv heads of 128 columns,
 * 537 MB, 86 us (6.2 TB/s: part of them is still in the last cache) and 5 for the
 * join; 45 sequences of 100 to 8192 keys, 348 MB, 80 us, since the parts of the
 * longest end late.  Few keys cost 7 us from the launch on: a table's page, a block
 * and the waves' join, one after another (517 keys of 2 kv heads of 256 columns).
 */
#include "r9vx_attn_kernels.h"

using namespace r9vx;

namespace {

constexpr int kBlock = 32; /* keys of a wave's step */
constexpr int kWaves = 4;

template <int D>
struct DecodeShape {
    static constexpr int VC = D > 128 ? 2 : 1;   /* column pieces of a value row */
    static constexpr int CW = D / VC;            /* columns of a piece */
    static constexpr int DL = CW / 16;           /* of them a lane's: 4, 6 or 8 */
    static constexpr int DW = DL / 2;            /* in words */
    static constexpr int KS = D / 32;            /* steps of a score's product */
    /* A key's (or query's) elements in LDS, 16 bytes more than it has: the 16 rows
     * whose same piece an operand's read takes start in different banks. */
    static constexpr int KP = D + 8;
    static constexpr int kArea = kBlock * KP * 2; /* bytes of a wave: a block's keys, or after them its sums of 16 rows */
    static_assert(16 * (D + 4) * 4 <= kArea);
    /* waves a SIMD that the registers are to leave room for (256 columns: 366 of 512 for one) */
    static constexpr int kWavesASimd(int rt) { return D > 192 ? 1 : D * rt > 96 ? 2 : 3; }
};

/* DW words in LDS. */
template <int DW>
__device__ __forceinline__ void store_words(uint16_t *p, const uint32_t (&w)[DW]) {
    if constexpr (DW == 2) *reinterpret_cast<r9vx_u32x2 *>(p) = r9vx_u32x2{w[0], w[1]};
    else if constexpr (DW == 3) {
        typedef attn_u32x3 vec __attribute__((aligned(4)));
        *reinterpret_cast<vec *>(p) = attn_u32x3{w[0], w[1], w[2]};
    } else *reinterpret_cast<r9vx_u32x4 *>(p) = r9vx_u32x4{w[0], w[1], w[2], w[3]};
}

/* DW words of global memory.  Said so: a pointer that may be a row of zeros is loaded
 * through otherwise as one that may be LDS, whose waits are then those for these loads. */
template <int DW>
__device__ __forceinline__ void load_words(const uint16_t *p, uint32_t (&w)[DW]) {
    static_assert(DW >= 2 && DW <= 4);
    if constexpr (DW == 2) {
        const r9vx_u32x2 v = __builtin_nontemporal_load((const __attribute__((address_space(1))) r9vx_u32x2 *)p);
        w[0] = v.x, w[1] = v.y;
    } else if constexpr (DW == 3) { /* 12 bytes: dword alignment */
        typedef attn_u32x3 vec __attribute__((aligned(4)));
        const attn_u32x3 v = *(const __attribute__((address_space(1))) vec *)p;
        w[0] = v.x, w[1] = v.y, w[2] = v.z;
    } else {
        const r9vx_u32x4 v = __builtin_nontemporal_load((const __attribute__((address_space(1))) r9vx_u32x4 *)p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
}

template <int D>
struct DecodeShared {
    float jm[kWaves][16], jl[kWaves][16];
    __attribute__((aligned(16))) uint8_t area[kWaves][DecodeShape<D>::kArea];
    uint32_t redo;
};

/* A workgroup's rows.  FAR: of a cap above kAttnShortCap (both formulas in one loop took
 * 19.2 us for a token and four drafts at 8191 keys, without a cap, where one takes 18.7).
 * CAREFUL: the second way, which a workgroup takes where the first one gave a NaN or an
 * infinity: a key that another token alone sees may have brought it in through a
 * probability of zero, and one that is seen makes a NaN of a probability's second half of
 * zero.  It goes through the keys once for each token, and adds values that are not
 * finite by a product of their own, with ones.  Returns whether the second way has to be taken. */
template <class T, int D, int RT, bool FAR, bool CAREFUL>
__device__ __forceinline__ bool attn_decode_rows(const r9vx_attn_problem &a, uint32_t row_tiles, DecodeShared<D> &sh) {
    using S = DecodeShape<D>;
    typedef typename T::x8 x8;
    auto &jm = sh.jm;
    auto &jl = sh.jl;
    auto &area = sh.area;

    uint32_t thread = threadIdx.x, bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
    if (CAREFUL) /* worked out anew: what the first way's loop would keep for this one is reloaded in it */
        asm volatile("" : "+v"(thread), "+s"(bx), "+s"(by), "+s"(bz));
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    /* Consecutive workgroups go to the eight dies in turn.  Heads, then sequences,
     * then parts, so that it is not always the same dies whose sequences have ended;
     * and with each part the sequences move on, so that a long one's parts are not all
     * on one die (24 of 300 to 16384 keys, 2 kv heads of 256 columns: 73 us, 86 without it). */
    uint32_t split = bz, b = by, kvh = bx, tile = 0;
    if (row_tiles > 1) { /* the tiles of the same keys one after another on one die (40 rows, 4 x 8192 keys of 256 columns: 34 us; beside each other on several 44) */
        const uint32_t slot = bx / 8, turn = slot / row_tiles, group = turn * 8 + bx % 8, seqs = group / a.kv_heads;
        tile = slot - turn * row_tiles, kvh = group - seqs * a.kv_heads, split = seqs / a.b, b = seqs - split * a.b;
        if (split >= a.splits) return false;
    }
    if (split) b = (b + (a.b - 1) % 8 * split) % a.b;
    const int rows = (int)(a.t_bucket * a.group);
    const int row0 = (int)tile * RT * 16;
    const int length = a.lengths[b];
    const bool bad_length = length < 0 || length > (int)a.len_bucket;
    if (bad_length && thread == 0 && a.status) atomicOr(a.status, R9VX_STATUS_BAD_LENGTH);
    const int start = a.starts ? a.starts[b] : 0;
    const int p0 = length - (int)a.t_bucket; /* of token 0 */

    /* tokens of the rows; keys that some row sees, and those that all of them do */
    const int first = attn_token(row0, a.group_magic), last = attn_token((row0 + RT * 16 < rows ? row0 + RT * 16 : rows) - 1, a.group_magic);
    int ulo, uhi, flo, fhi;
    attn_seen(a.window, 1, p0 + first, length, start, 0, ulo, fhi);
    attn_seen(a.window, 1, p0 + last, length, start, 0, flo, uhi);
    if (bad_length) uhi = ulo = 0;

    /* this part's blocks */
    const int b0 = ulo / kBlock, b1 = uhi > ulo ? (uhi + kBlock - 1) / kBlock : b0;
    int begin, end;
    attn_part(b0, b1, kWaves, a.parts, a.part_blocks, split, begin, end);

    const uint16_t *kbase = a.k + kvh * a.k_stride[2], *vbase = a.v + kvh * a.v_stride[2];
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t mask = (1u << a.page_shift) - 1;

    /* A lane loads columns DL col .. of eight neighbouring keys, which stand in one
     * page: whole lines are read.  Keys go through the wave's part of LDS into the
     * operand's order, values are turned in registers.  A group of eight of which
     * nothing is seen has no page. */
    auto page_of = [&](int key) -> uint32_t { return key < uhi && key + 8 > ulo ? (uint32_t)table[key >> a.page_shift] : 0u; };
    auto load = [&](uint32_t (&w)[8][S::VC][S::DW], const uint16_t *base, const uint64_t *stride, uint32_t page, int key) {
        const bool seen = key < uhi && key + 8 > ulo;
        const AttnPlace where = attn_place(page, a.pages, seen ? ulo : -1, ulo, uhi);
        const uint16_t *p = attn_row<T>(where, base, stride, page, (uint32_t)key & mask) + S::DL * col;
        const uint64_t step = where == kAttnKept ? stride[1] : 0; /* zeros and NaN: one row for all */
#pragma unroll
        for (int i = 0; i < 8; ++i, p += step)
#pragma unroll
            for (int c = 0; c < S::VC; ++c) load_words<S::DW>(p + c * S::CW, w[i][c]);
    };
    uint16_t *mine = reinterpret_cast<uint16_t *>(area[wave]);
    uint32_t k[8][S::VC][S::DW], v[8][S::VC][S::DW];
    /* The first block's page, the queries' rows, then the block: each load goes out
     * before anything waits for the one before it. */
    uint32_t page = 0, after = 0; /* of the next block, and of the one after it */
    auto first_page = [&]() {
        if (begin + wave < end) page = page_of((begin + wave) * kBlock + 8 * g4);
    };
    auto first_block = [&]() {
        const int blk = begin + wave;
        if (blk >= end) return;
        load(k, kbase, a.k_stride, page, blk * kBlock + 8 * g4);
        load(v, vbase, a.v_stride, page, blk * kBlock + 8 * g4);
        if (page >= a.pages && a.status) atomicOr(a.status, R9VX_STATUS_BAD_PAGE);
        if (blk + kWaves < end) page = page_of((blk + kWaves) * kBlock + 8 * g4);
    };
    first_page();

    /* the queries: 16 rows at a time through LDS; a lane's row of each tile */
    uint32_t qw[RT][4][S::VC][S::DW];
    int lo[RT], hi[RT], pos[RT];
    float slope[RT];
    x8 q[RT][S::KS];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = row0 + r * 16 + 4 * g4 + i, tok = attn_token(row, a.group_magic);
            const uint32_t h = kvh * a.group + (row - tok * (int)a.group);
            const uint16_t *p = row < rows ? a.q + b * a.q_stride[0] + tok * a.q_stride[1] + h * a.q_stride[2] : reinterpret_cast<const uint16_t *>(kAttnZeroRow);
#pragma unroll
            for (int c = 0; c < S::VC; ++c) load_words<S::DW>(p + c * S::CW + S::DL * col, qw[r][i][c]);
        }
    first_block();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < S::VC; ++c) store_words<S::DW>(mine + (4 * g4 + i) * S::KP + c * S::CW + S::DL * col, qw[r][i][c]);
        const int row = row0 + r * 16 + col, tok = attn_token(row, a.group_magic);
        pos[r] = p0 + tok;
        attn_seen(a.window, 1, pos[r], length, start, 0, lo[r], hi[r]);
        if (row >= rows || bad_length) lo[r] = hi[r] = 0;
        slope[r] = a.slopes && row < rows ? a.slopes[kvh * a.group + (row - tok * (int)a.group)] * kLog2e : 0.0f;
#pragma unroll
        for (int s = 0; s < S::KS; ++s) q[r][s] = *reinterpret_cast<const x8 *>(mine + col * S::KP + s * 32 + g4 * 8);
        if (a.scale <= 0.0f) {
#pragma unroll
            for (int s = 0; s < S::KS; ++s) q[r][s] = attn_signed<T>(a, q[r][s]);
        }
    }
    const AttnScore score(a);

    float m[RT], l[RT];
    r9vx_f32x4 o[RT][S::VC][S::DL];

    /* keys [vlo, vhi) have values: those that some row sees, or of the second way those that its token does */
    int vlo = ulo, vhi = uhi;
    if (!CAREFUL && thread == 0) sh.redo = 0;
    for (int pass = CAREFUL ? first : last; pass <= last; ++pass) {
        if (CAREFUL) {
            attn_seen(a.window, 1, p0 + pass, length, start, 0, vlo, vhi);
            if (pass > first) {
                __syncthreads(); /* the sums of the pass before have been read */
                first_page();
                first_block();
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < S::VC; ++c)
#pragma unroll
                for (int j = 0; j < S::DL; ++j) o[r][c][j] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int blk = begin + wave; blk < end; blk += kWaves) {
            const int key0 = blk * kBlock, next = key0 + kWaves * kBlock;
            const bool more = blk + kWaves < end;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < S::VC; ++c) store_words<S::DW>(mine + (8 * g4 + i) * S::KP + c * S::CW + S::DL * col, k[i][c]);
            if (more) {
                load(k, kbase, a.k_stride, page, next + 8 * g4);
                if (page >= a.pages && a.status) atomicOr(a.status, R9VX_STATUS_BAD_PAGE);
                if (blk + 2 * kWaves < end) after = page_of(next + kWaves * kBlock + 8 * g4);
            }
            /* tile t has keys 4 t .. 4 t + 3 of each eight: what a lane gets of both is its own eight */
            r9vx_f32x4 sc[RT][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < RT; ++r) sc[r][t] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < S::KS; ++s) {
                    const x8 kf = *reinterpret_cast<const x8 *>(mine + (8 * (col >> 2) + 4 * t + (col & 3)) * S::KP + s * 32 + g4 * 8);
#pragma unroll
                    for (int r = 0; r < RT; ++r) sc[r][t] = T::mma16(kf, q[r][s], sc[r][t]);
                }
            }
            const int k8 = key0 + 8 * g4; /* of this lane's scores and values */
            x8 ph[RT], pl[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = sc[r][e >> 2][e & 3];
                if (a.softcap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = FAR ? score.capped_far(x[e]) : score.capped(x[e]);
                }
                if (a.slopes) {
                    const float far = (float)(pos[r] - k8);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = fmaf(-slope[r], fabsf(far - (float)e), x[e] * score.before);
                }
                if (key0 < flo || key0 + kBlock > fhi) {
                    const int from = lo[r] - k8, to = hi[r] - k8;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < from || e >= to) x[e] = -INFINITY;
                }
                float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                top = fmaxf(top, __shfl_xor(top, 16, R9VX_WAVE));
                top = fmaxf(top, __shfl_xor(top, 32, R9VX_WAVE)) * score.factor;
                if (__any(top > m[r])) {
                    const float now = fmaxf(m[r], top);
                    float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - now);
                    if (CAREFUL) f = attn_some(f);
                    m[r] = now;
                    l[r] *= f;
#pragma unroll
                    for (int c = 0; c < S::VC; ++c)
#pragma unroll
                        for (int j = 0; j < S::DL; ++j) o[r][c][j] *= f;
                }
                const float ref = (m[r] == -INFINITY ? 0.0f : m[r]) - T::kTop;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float pe = __builtin_amdgcn_exp2f(fmaf(x[e], score.factor, -ref));
                    l[r] += pe;
                    /* a bf16 probability as two numbers; one f16 number is off by 2^-11 as the output is,
                     * and two took 1 to 5 % longer (300 keys 7.5 -> 7.9 us, 5 tokens at 8 x 8192 keys of 256 columns 48.7 -> 51) */
                    ph[r][e] = (typename T::elem)pe;
                    if constexpr (T::kWide) pl[r][e] = (typename T::elem)(pe - (float)ph[r][e]);
                }
            }
            if (key0 < vlo || key0 + kBlock > vhi) { /* what stands behind the last key, or is not to be seen */
                const int from = vlo - k8, to = vhi - k8;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int c = 0; c < S::VC; ++c)
#pragma unroll
                        for (int w = 0; w < S::DW; ++w) v[i][c][w] = i >= from && i < to ? v[i][c][w] : 0u;
            }
#pragma unroll
            for (int c = 0; c < S::VC; ++c)
#pragma unroll
                for (int j = 0; j < S::DL; ++j) {
                    r9vx_u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = __builtin_amdgcn_perm(v[2 * i + 1][c][j >> 1], v[2 * i][c][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
                    if (CAREFUL) { /* what is not finite apart from what is */
                        const r9vx_u32x4 ones = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
                        r9vx_u32x4 not_finite;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t bits = attn_odd<T>(w[i]);
                            not_finite[i] = w[i] & bits;
                            w[i] &= ~bits;
                        }
#pragma unroll
                        for (int r = 0; r < RT; ++r) o[r][c][j] = T::mma16(__builtin_bit_cast(x8, not_finite), __builtin_bit_cast(x8, ones), o[r][c][j]);
                    }
                    const x8 vt = __builtin_bit_cast(x8, w);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        o[r][c][j] = T::mma16(vt, ph[r], o[r][c][j]);
                        if constexpr (T::kWide) o[r][c][j] = T::mma16(vt, pl[r], o[r][c][j]);
                    }
                }
            if (more) {
                load(v, vbase, a.v_stride, page, next + 8 * g4);
                page = after;
            }
        }

        /* the waves' sums, through LDS; then a thread has four columns of a row at a time */
        bool odd = false; /* a value that is not finite */
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            l[r] += __shfl_xor(l[r], 16, R9VX_WAVE);
            l[r] += __shfl_xor(l[r], 32, R9VX_WAVE);
            if (r > 0) __syncthreads();
            float *sums = reinterpret_cast<float *>(mine);
            if (lane < 16) jm[wave][col] = m[r], jl[wave][col] = l[r];
#pragma unroll
            for (int c = 0; c < S::VC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < S::DL; j += 2)
                        *reinterpret_cast<float2 *>(sums + col * (D + 4) + c * S::CW + S::DL * (4 * g4 + e) + j) = make_float2(o[r][c][j][e], o[r][c][j + 1][e]);
            __syncthreads();
            for (int i = thread; i < 16 * D / 4; i += 64 * kWaves) {
                const int in = i / (D / 4), c = i % (D / 4) * 4, row = row0 + r * 16 + in;
                const int tok = attn_token(row, a.group_magic);
                if (row >= rows || (CAREFUL && tok != pass)) continue;
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) top = fmaxf(top, jm[w][in]);
                r9vx_f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    /* a wave that saw nothing (or scores of -infinity alone) has zeros, or a NaN of NaN scores */
                    float f = jm[w][in] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(jm[w][in] - top);
                    if (CAREFUL) f = attn_some(f);
                    sum += jl[w][in] * f;
                    y += *reinterpret_cast<const r9vx_f32x4 *>(reinterpret_cast<const float *>(area[w]) + in * (D + 4) + c) * f;
                }
                odd |= !(fabsf(sum) < INFINITY) || !(fabsf(y[0]) < INFINITY) || !(fabsf(y[1]) < INFINITY) || !(fabsf(y[2]) < INFINITY) || !(fabsf(y[3]) < INFINITY);
                if (bad_length || (sum != sum && top == -INFINITY)) top = 0.0f; /* a NaN that counts beside any other part */
                if (bad_length) sum = __builtin_nanf("");
                if (sum == 0.0f && top == -INFINITY) { /* scores of -infinity alone are no softmax; no score at all is zeros */
                    int from, to;
                    attn_seen(a.window, 1, p0 + tok, length, start, 0, from, to);
                    if ((from > begin * kBlock ? from : begin * kBlock) < (to < end * kBlock ? to : end * kBlock)) sum = __builtin_nanf("");
                }
                const uint32_t h = kvh * a.group + (row - tok * (int)a.group);
                if (a.splits == 1) {
                    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                    typedef typename T::elem four __attribute__((ext_vector_type(4)));
                    const four w = {(typename T::elem)(y[0] * f), (typename T::elem)(y[1] * f), (typename T::elem)(y[2] * f), (typename T::elem)(y[3] * f)};
                    *reinterpret_cast<four *>(a.out + b * a.out_stride[0] + tok * a.out_stride[1] + h * a.out_stride[2] + c) = w;
                } else {
                    const uint64_t at = (((uint64_t)b * a.t_bucket + tok) * a.heads + h) * a.splits + split;
                    *reinterpret_cast<r9vx_f32x4 *>(a.partial + at * D + c) = y;
                    if (c == 0) reinterpret_cast<float2 *>(a.partial + (uint64_t)a.b_bucket * a.t_bucket * a.heads * a.splits * D)[at] = make_float2(top, sum);
                }
            }
        }
        if (!CAREFUL) {
            if (odd) sh.redo = 1;
            __syncthreads();
        }
    }
    return !CAREFUL && sh.redo;
}

template <class T, int D, int RT, bool FAR>
__global__ __launch_bounds__(64 * kWaves, DecodeShape<D>::kWavesASimd(RT)) void attn_decode_kernel(r9vx_attn_problem a, uint32_t row_tiles) {
    __shared__ DecodeShared<D> sh;
    if (!attn_decode_rows<T, D, RT, FAR, false>(a, row_tiles, sh)) return;
    /* (in line: as a function it takes 0.3 to 1 KB of scratch a lane, 480 MB of a card's memory) */
    uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args), "+s"(row_tiles));
    const r9vx_attn_problem again = *(const r9vx_attn_problem *)(attn_kernel_args *)args;
    attn_decode_rows<T, D, RT, FAR, true>(again, row_tiles, sh);
}

constexpr uint32_t kMostParts = 256;
constexpr int kFewParts = 16;
constexpr uint32_t kPartBlocks = 64; /* a part's blocks at most */

/* Where a row (token times heads + head) of the output stands; null for one of no
 * sequence, which is left. */
__device__ __forceinline__ uint16_t *join_out(const r9vx_attn_problem &a, uint64_t row) {
    const uint64_t tok = row / a.heads;
    const uint32_t h = (uint32_t)(row - tok * a.heads);
    uint64_t seq = 0, t = tok;
    if (a.offsets) { /* prefill */
        if ((int64_t)tok < a.offsets[0] || (int64_t)tok >= a.offsets[a.b]) return nullptr;
    } else {
        seq = tok / a.t_bucket;
        t = tok - seq * a.t_bucket;
    }
    return a.out + seq * a.out_stride[0] + t * a.out_stride[1] + h * a.out_stride[2];
}

/* A row's parts, by a workgroup for each 32 columns:
 * each wave takes the parts' maxima and sums, then four columns a thread are added
 * up, several parts side by side, and those through LDS.  Bound by a launch and
 * two loads in turn: 64 parts of 32 rows of 128 columns 5.1 us. */
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(r9vx_attn_problem a, const float2 *ml) {
    __shared__ float weight[kMostParts];
    __shared__ r9vx_f32x4 sums[256];
    const uint64_t row = blockIdx.x, at = row * a.splits;
    uint16_t *y = join_out(a, row);
    if (!y) return;
    const uint32_t lane = threadIdx.x & 63;
    constexpr int N = kMostParts / 64;
    float2 x[N];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = make_float2(-INFINITY, 0.0f);
        if (lane + 64 * i < a.splits) x[i] = ml[at + lane + 64 * i];
        m = fmaxf(m, x[i].x);
    }
    for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, R9VX_WAVE));
    /* a part that saw nothing, or scores of -infinity alone, has no weight beside
     * others; where no part saw more, one with a sum (a NaN) makes the row NaN */
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float w = x[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[i].x - m);
        if (x[i].x != -INFINITY || m == -INFINITY) sum += x[i].y * (m == -INFINITY ? 1.0f : w);
        if (threadIdx.x < 64) weight[lane + 64 * i] = x[i].x == -INFINITY ? 0.0f : attn_some(w);
    }
    for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, R9VX_WAVE);
    __syncthreads();
    const uint32_t width = a.head_dim / 4 / gridDim.y, side = 256 / width;
    const uint32_t part = threadIdx.x / width, c = threadIdx.x - part * width, column = 4 * (blockIdx.y * width + c);
    r9vx_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (part < side) {
        const float *p = a.partial + at * a.head_dim + column;
#pragma unroll 4
        for (uint32_t s = part; s < a.splits; s += side) {
            const r9vx_f32x4 v = *reinterpret_cast<const r9vx_f32x4 *>(p + (uint64_t)s * a.head_dim);
            const float w = weight[s];
            if (w != 0.0f || w != w) o += v * w; /* not 0 times what a part without weight left */
        }
    }
    sums[threadIdx.x] = o;
    __syncthreads();
    if (threadIdx.x < width) {
        for (uint32_t s = 1; s < side; ++s) o += sums[s * width + c];
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        typedef typename T::elem four __attribute__((ext_vector_type(4)));
        const four w = {(typename T::elem)(o[0] * f), (typename T::elem)(o[1] * f), (typename T::elem)(o[2] * f), (typename T::elem)(o[3] * f)};
        *reinterpret_cast<four *>(y + column) = w;
    }
}

/* The same of at most kFewParts parts, by a wave, which has all its loads on their way
 * at once: lane i % 16 part i's maximum and sum, and every lane four columns of
 * the parts lane / (D / 4), one in 256 / D.  13 parts of 4800 rows of 256 columns,
 * 64 MB, take 12 us (15.5 by a workgroup a row). */
template <class T, int D>
__global__ __launch_bounds__(256) void attn_join_few_kernel(r9vx_attn_problem a, const float2 *ml, uint64_t rows) {
    constexpr int kWidth = D / 4, kSide = 64 / kWidth, kMost = (kFewParts + kSide - 1) / kSide;
    const int lane = threadIdx.x & 63, side = lane / kWidth, c = 4 * (lane - side * kWidth);
    const uint64_t row = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = row * a.splits;
    if (row >= rows) return;
    uint16_t *y = join_out(a, row);
    if (!y) return;
    const int i = lane % kFewParts;
    const float2 x = i < (int)a.splits ? ml[at + i] : make_float2(-INFINITY, 0.0f);
    const int last = (int)a.splits - 1;
    r9vx_f32x4 v[kMost];
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int part = side + j * kSide; /* (one that is not there has no weight) */
        v[j] = *reinterpret_cast<const r9vx_f32x4 *>(a.partial + (at + (part < last ? part : last)) * D + c);
    }
    float m = x.x;
#pragma unroll
    for (int off = 1; off < kFewParts; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, R9VX_WAVE));
    const float w = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - m), some = x.x == -INFINITY ? 0.0f : attn_some(w);
    float sum = x.x != -INFINITY || m == -INFINITY ? x.y * (m == -INFINITY ? 1.0f : w) : 0.0f;
#pragma unroll
    for (int off = 1; off < kFewParts; off <<= 1) sum += __shfl_xor(sum, off, R9VX_WAVE);
    r9vx_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const float f = __shfl(some, (side + j * kSide) % kFewParts, R9VX_WAVE);
        if (f != 0.0f || f != f) o += v[j] * f; /* not 0 times what a part without weight left */
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float own = o[e];
#pragma unroll
        for (int j = 1; j < kSide; ++j) o[e] += __shfl(own, (lane + j * kWidth) % 64, R9VX_WAVE);
    }
    if (side > 0) return;
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef typename T::elem four __attribute__((ext_vector_type(4)));
    *reinterpret_cast<four *>(y + c) = four{(typename T::elem)(o[0] * f), (typename T::elem)(o[1] * f), (typename T::elem)(o[2] * f), (typename T::elem)(o[3] * f)};
}

/* 32 rows a workgroup work on each block of keys half as often (64 rows of 64 columns, 16 x 4096
 * keys: 32 us against 38; 32 of 128, 8 x 8192: 37 against 40).  Beyond 128 columns they take
 * all registers of a SIMD: slower (8 x 8192 keys of 256 columns, 32 rows: 50 us against 40). */
uint32_t decode_row_tiles(const r9vx_attn_problem &p, uint32_t &rt) {
    const uint32_t rows = p.t_bucket * p.group;
    rt = rows > 16 && p.head_dim <= 128 ? 2 : 1;
    return (rows + 16 * rt - 1) / (16 * rt);
}

template <class T>
int launch_join(const r9vx_attn_problem &p, const float2 *ml, uint64_t rows, hipStream_t stream) {
    const dim3 few((unsigned)((rows + 3) / 4)), many((unsigned)rows, p.head_dim / 32), block(256);
    if (p.splits > (uint32_t)kFewParts) hipLaunchKernelGGL(attn_join_kernel<T>, many, block, 0, stream, p, ml);
    else if (p.head_dim == 64) hipLaunchKernelGGL((attn_join_few_kernel<T, 64>), few, block, 0, stream, p, ml, rows);
    else if (p.head_dim == 96) hipLaunchKernelGGL((attn_join_few_kernel<T, 96>), few, block, 0, stream, p, ml, rows);
    else if (p.head_dim == 128) hipLaunchKernelGGL((attn_join_few_kernel<T, 128>), few, block, 0, stream, p, ml, rows);
    else if (p.head_dim == 192) hipLaunchKernelGGL((attn_join_few_kernel<T, 192>), few, block, 0, stream, p, ml, rows);
    else hipLaunchKernelGGL((attn_join_few_kernel<T, 256>), few, block, 0, stream, p, ml, rows);
    return (int)hipGetLastError();
}

template <class T, int D, int RT>
int launch_decode_rows(const r9vx_attn_problem &p, dim3 grid, uint32_t tiles, hipStream_t stream) {
    if (p.softcap > kAttnShortCap) hipLaunchKernelGGL((attn_decode_kernel<T, D, RT, true>), grid, dim3(64 * kWaves), 0, stream, p, tiles);
    else hipLaunchKernelGGL((attn_decode_kernel<T, D, RT, false>), grid, dim3(64 * kWaves), 0, stream, p, tiles);
    return (int)hipGetLastError();
}

template <class T, int D>
int launch_decode(const r9vx_attn_problem &p, hipStream_t stream) {
    uint32_t rt;
    const uint32_t tiles = decode_row_tiles(p, rt);
    const uint64_t groups = r9vx_attn_decode_groups(p);
    const dim3 grid = tiles > 1 ? dim3((unsigned)groups) : dim3(p.kv_heads, p.b, p.splits);
    if constexpr (D <= 128) {
        if (rt == 2) return launch_decode_rows<T, D, 2>(p, grid, tiles, stream);
    }
    return launch_decode_rows<T, D, 1>(p, grid, tiles, stream);
}

template <class T>
int launch_decode_type(const r9vx_attn_problem &p, hipStream_t stream) {
    switch (p.head_dim) {
    case 64: return launch_decode<T, 64>(p, stream);
    case 96: return launch_decode<T, 96>(p, stream);
    case 128: return launch_decode<T, 128>(p, stream);
    case 192: return launch_decode<T, 192>(p, stream);
    default: return launch_decode<T, 256>(p, stream);
    }
}

}  // namespace

uint64_t r9vx_attn_decode_groups(const r9vx_attn_problem &p) {
    uint32_t rt;
    const uint64_t tiles = decode_row_tiles(p, rt), groups = (uint64_t)p.b * p.kv_heads * p.splits;
    return tiles > 1 ? (groups + 7) / 8 * 8 * tiles : groups;
}

void r9vx_attn_decode_plan(r9vx_attn_problem &p) {
    uint32_t rt;
    const uint64_t groups = (uint64_t)p.b_bucket * p.kv_heads * decode_row_tiles(p, rt);
    const uint64_t fill = (p.head_dim > 192 ? 1ull : p.head_dim * rt > 96 ? 2ull : 3ull) * r9vx_device_cus();
    /* blocks of the longest row */
    const uint32_t whole = (p.len_bucket + kBlock - 1) / kBlock, seen = (p.window + p.t_bucket - 1) / kBlock + 2;
    const uint32_t most = seen < whole ? seen : whole > 0 ? whole : 1;
    uint64_t parts = groups ? fill / groups : 1;
    if (parts > (most + kWaves - 1) / kWaves) parts = (most + kWaves - 1) / kWaves;
    /* two or three blocks a wave cost what the launch of a join does (one part or one for
     * each four blocks, in a graph and in calls from Python: 200 keys of 128 columns 7.4 us
     * against 8.7 and 9.2 against 13.6, 350 9.0 against 9.0 and 9.1 against 13.8; 200 of
     * 256 columns 10.2 against 11.5, 350 12.7 against 11.6, 517 of 128 11.7 against 9.0) */
    if (most <= (p.head_dim > 128 ? 2u : 3u) * kWaves) parts = 1;
    if (parts > kMostParts) parts = kMostParts;
    if (parts < 1) parts = 1;
    uint32_t per = (uint32_t)((most + parts - 1) / parts);
    /* a long sequence among short ones ends late in one piece; the more workgroups
     * there are, the longer its pieces may be */
    const uint64_t piece = kPartBlocks * (groups > 4 * fill ? groups / (4 * fill) : 1);
    if (per > piece) per = (uint32_t)piece;
    if (per < (most + kMostParts - 1) / kMostParts) per = (most + kMostParts - 1) / kMostParts;
    per = (per + kWaves - 1) / kWaves * kWaves;
    p.parts = (uint32_t)parts;
    p.part_blocks = per;
    p.splits = (most + per - 1) / per;
    if (p.splits < p.parts) p.splits = p.parts;
}

uint64_t r9vx_attn_join_groups(const r9vx_attn_problem &p, uint64_t rows) { return p.splits > (uint32_t)kFewParts ? rows * (p.head_dim / 32) : (rows + 3) / 4; }

int r9vx_launch_attn_join(const r9vx_attn_problem &p, uint64_t rows, hipStream_t stream) {
    const float2 *ml = reinterpret_cast<const float2 *>(p.partial + (p.offsets ? (uint64_t)p.t_bucket : (uint64_t)p.b_bucket * p.t_bucket) * p.heads * p.splits * p.head_dim);
    return p.dtype == R9VX_DTYPE_BF16 ? launch_join<AttnBf16>(p, ml, rows, stream) : launch_join<AttnF16>(p, ml, rows, stream);
}

int r9vx_launch_attn_decode(const r9vx_attn_problem &p, hipStream_t stream) {
    const int rc = p.dtype == R9VX_DTYPE_BF16 ? launch_decode_type<AttnBf16>(p, stream) : launch_decode_type<AttnF16>(p, stream);
    if (rc || p.splits == 1) return rc;
    return r9vx_launch_attn_join(p, (uint64_t)p.b * p.t_bucket * p.heads, stream);
}
