/*
 * fp8_moe.hip -- moe_ffn over block-scaled e4m3 experts.
 *
 *   quantize x -> permute (the stable counting sort of moe.hip) -> per expert
 *   gate / up product, silu(g) * u, quantize h -> down product -> weighted
 *   sum per token.
 *
 * Rows of h and o stand in sorted order (the pairs of an expert together,
 * then the shared experts' rows), so an expert's rows are one run.  The sort
 * leaves a list of tiles of up to 256 rows of one expert; both products walk
 * it: few rows per expert through the streaming loop, many through the tiles
 * of r9vx_e4m3_gemm.h.  The streaming loop and f32 outputs' tiles keep every
 * product (EXACT, r9vx_e4m3.h), bf16 outputs' tiles take the 8-bit instruction.
 *
 * 48 tokens, 64 experts of 2 x 1408 x 2048: gate / up 65 to 75 us and down 35 to
 * 39 by the clock, 4.8 to 5.5 TB/s of weights (a 4 GiB copy: 4.7, reading alone
 * up to 7).  8192 tokens, 10 of 512 experts of 2 x 512 x 2048 (160 rows each),
 * bf16 outputs: gate / up 377 us (0.91 PFLOP/s, 2.9 TB/s of weights; of a tile's
 * 68 thousand cycles 55 are products, 10 the drain), down 317 us, whose K of four
 * steps is as long as its drain, combine 62 us (5.9 TB/s); f32 outputs 671, 505
 * and 127.
 */
#include "r9vx_e4m3_gemm.h"
#include "r9vx_moe.h"

using namespace r9vx;

namespace {

struct Fp8MoeLayout {
    MoeLayout sort; /* the sort's regions */
    uint64_t xq, xs, h, hq, hs, o, os, total;
    bool stream; /* few rows per expert */
    bool half;   /* o in f16, a power of two per kOutBlock columns beside it */
};

constexpr uint32_t kOutBlock = 128; /* columns that share a weight scale */

/* Few rows an expert: the streaming form.  us of a call in it / in tiles, rows an
 * expert in brackets, shared experts counted with the others; bf16 outputs:
 *   6 of 64 experts of 2 x 1408 x 2048    64 tokens (6) 120 / 142, 96 (9) 149 / 147, 150 (14) 172 / 150
 *   10 of 512, 512 x 2048                 64 (1) 165 / 228, 256 (5) 275 / 332, 384 (8) 337 / 354, 512 (10) 385 / 375
 *   2 of 16, 4096 x 2048                  64 (8) 104 / 125, 96 (12) 132 / 126
 *   8 of 256, 512 x 4096                  64 (2) 208 / 257, 200 (6) 327 / 359, 256 (8) 353 / 345
 * a shared expert has every token, 16 at a time through each workgroup:
 *   10 of 512 and one                     128 (3) 260 / 296, 256 (5) 358 / 350
 *   8 of 256 and one                      128 (5) 322 / 331, 256 (9) 482 / 380
 *   6 of 64 and two                       64 (8) 157 / 148, 128 (16) 231 / 157
 * f32 outputs, whose tiles are the slower exact ones:
 *   6 of 64                               150 (14) 172 / 246, 256 (24) 250 / 280, 512 (48) 424 / 301
 *   10 of 512                             64 (1) 164 / 349, 512 (10) 386 / 614
 *   2 of 16                               150 (19) 162 / 174, 256 (32) 272 / 206
 *   10 of 512 and one                     768 (16) 584 / 675, 1000 (21) 691 / 714
 *   8 of 256 and one                      384 (13) 576 / 649, 512 (18) 677 / 669
 * Up to 64 tokens always, whatever the experts' number, so that such calls' sums
 * are exact for every type. */
bool moe_streams(const r9vx_moe_fp8_problem &p) {
    const uint64_t rows = (uint64_t)p.t_bucket * (p.k + p.shared), experts = p.e + p.shared;
    if (p.t_bucket <= 64) return true;
    if (p.y_dtype == R9VX_DTYPE_F32) return rows <= 16 * experts;
    return rows <= 8 * experts && (p.shared == 0 || p.t_bucket <= 128);
}

Fp8MoeLayout moe_layout(const r9vx_moe_fp8_problem &p) {
    Fp8MoeLayout L{};
    const uint64_t pairs = (uint64_t)p.t_bucket * p.k, rows = pairs + (uint64_t)p.shared * p.t_bucket;
    const uint64_t nchunk = (pairs + 255) / 256;
    uint64_t off = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t at = off;
        off += (bytes + 255) & ~255ull;
        return at;
    };
    MoeLayout &s = L.sort;
    s.max_tiles3 = (uint32_t)(rows / kMoeTileM3 + (pairs < p.e ? pairs : p.e) + p.shared);
    s.status = take(64);
    s.counts = take(4ull * p.e);
    s.offsets = take(4ull * (p.e + 1));
    s.sorted = take(4 * pairs);
    s.inv = take(4 * pairs);
    s.rank = take(4 * pairs);
    s.ccount = take(4ull * p.e * nchunk);
    s.cbase = take(4ull * p.e * nchunk);
    s.cbad = take(4 * nchunk);
    s.tiles3 = take(16ull * s.max_tiles3 + 16);
    L.stream = moe_streams(p);
    L.xq = take((uint64_t)p.t_bucket * p.dm);
    L.xs = take(4ull * p.t_bucket * (p.dm / kFp8Block));
    L.h = take(L.stream ? 4 * rows * p.dff : 0);
    L.hq = take(rows * p.dff);
    L.hs = take(4 * rows * (p.dff / kFp8Block));
    /* o is written and read once each, in prompts by far the most bytes of all.
     * For bf16 outputs the tiles keep it in f16: a row's 128 columns of one
     * weight scale times the power of two that brings the largest into [1, 2)
     * (under 4 at f32's upper end), so that nothing overflows and an addend is
     * off by half a step, 2^-11 of itself or 2^-25 of the block's largest: an
     * eighth of the output's own rounding where the addends do not cancel.
     * 8192 tokens of 10 of 512 experts: 778 us a call against 832 with an f32 o,
     * and 2.516e-3 against 2.507e-3 from the exact outputs. */
    L.half = !L.stream && p.y_dtype == R9VX_DTYPE_BF16;
    L.o = take((L.half ? 2 : 4) * rows * p.dm);
    L.os = take(L.half ? 4 * rows * (p.dm / kOutBlock) : 0);
    L.total = off;
    return L;
}

struct Fp8MoeArgs {
    Fp8Args g;      /* n, k, kb, nb, xq, xs of this product; w, ws of expert 0 */
    uint8_t *ws;
    Fp8MoeLayout L;
    uint32_t p, t, topk;
    float *out;     /* f32 rows of h (streaming gate / up) or o (f16: Fp8MoeLayout::half) */
    float *os;
    uint8_t *hq;
    float *hs;
};

/* Tile `at` of the list: the rows of one expert. */
__device__ __forceinline__ r9vx_u32x4 moe_tile(const Fp8MoeArgs &a, uint32_t at) {
    return reinterpret_cast<const r9vx_u32x4 *>(a.ws + a.L.sort.tiles3)[at];
}
__device__ __forceinline__ uint32_t moe_word(const Fp8MoeArgs &a, uint32_t i) {
    return reinterpret_cast<const uint32_t *>(a.ws + a.L.sort.status)[i];
}
/* The token of row i of a tile that starts at sorted position `first`. */
__device__ __forceinline__ uint32_t moe_token(const Fp8MoeArgs &a, uint32_t pos) {
    if (pos >= a.p) return (pos - a.p) % a.t; /* a shared expert's row */
    return reinterpret_cast<const uint32_t *>(a.ws + a.L.sort.sorted)[pos] / a.topk;
}

/* UP: gate / up, rows gathered by token, h stored; else down on h's rows.
 * 128 registers, so that sixteen waves share a CU, in workgroups of four, whose
 * ends overlap more than those of eight: 5 tokens of 512 experts, gate / up and
 * down 20.8 + 12.5 us (eight: 23.0 + 15.9, and 31 at 133 registers).
 * The rows' codes come from launches of their own: quantized here, in
 * registers or in LDS, they cost the occupancy that keeps the weights
 * flowing (5 tokens of 512 experts: 56 us a call, 97 and 89 so). */
template <int MT, int NT, int W, bool UP>
__global__ __launch_bounds__(W * 64, 4) void fp8_moe_stream_kernel(Fp8MoeArgs a) {
    __shared__ __attribute__((aligned(16))) r9vx_f32x4 part[W * NT * MT * 64];
    __shared__ uint32_t token[256];
    if (moe_word(a, 0) != 0u || blockIdx.y >= moe_word(a, 4)) return;
    const r9vx_u32x4 tile = moe_tile(a, blockIdx.y);
    Fp8Rows r{};
    r.w = a.g.w + (uint64_t)tile.x * (UP ? 2u : 1u) * a.g.n * a.g.k;
    r.ws = a.g.ws + (uint64_t)tile.x * (UP ? 2u : 1u) * a.g.nb * a.g.kb;
    if (UP) r.list = token;
    for (uint32_t m0 = 0; m0 < tile.z; m0 += MT * 16) {
        r.m0 = (UP ? 0u : tile.y) + m0;
        r.rows = tile.z - m0 < MT * 16u ? tile.z - m0 : MT * 16u;
        auto tokens = [&] {
            if (!UP || m0 != 0) return;
            if (threadIdx.x < tile.z) token[threadIdx.x] = moe_token(a, tile.y + threadIdx.x); /* at most 256 */
            __syncthreads();
        };
        static_assert(W * 64 >= 256, "");
        fp8_stream<MT, NT, W, kFp8Codes, UP>(a.g, r, blockIdx.x, part, nullptr, tokens, [&](uint32_t row, uint32_t n, r9vx_f32x4 v) {
            *reinterpret_cast<r9vx_f32x4 *>(a.out + (uint64_t)(tile.y + m0 + row) * a.g.n + n) = v;
        });
        __syncthreads(); /* the partial sums have been read */
    }
}

/* BM rows of a list entry, 256 / BM workgroups for each.  EXACT as in the dense
 * products: f32 outputs keep their sums in f32 throughout (128 rows: the
 * widened codes leave no registers for 256).  bf16 outputs take the 8-bit
 * instruction for both products, 8192 tokens of 10 of 512 experts 778 us a call
 * against 1280: what it drops moves some codes of h, and the outputs are 2.5e-3
 * from the exact ones instead of the 1.7e-3 of their own rounding. */
template <bool UP, int BM, bool EXACT>
__global__ __launch_bounds__(512) void fp8_moe_tile_kernel(Fp8MoeArgs a) {
    typedef Fp8Tile<BM, 256, 2, UP, EXACT> T;
    constexpr uint32_t kParts = kMoeTileM3 / BM;
    static_assert(kParts * BM == kMoeTileM3, "");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLds];
    __shared__ uint32_t token[BM];
    if (moe_word(a, 0) != 0u) return;
    /* each XCD takes one run of the list, a tile's column blocks side by side */
    const uint32_t cols = (a.g.n + T::kCols - 1) / T::kCols, tiles = moe_word(a, 4) * cols * kParts;
    const uint32_t x = blockIdx.x & 7u, i = blockIdx.x >> 3, q = tiles >> 3, rem = tiles & 7u;
    if (i >= q + (x < rem ? 1u : 0u)) return;
    const uint32_t at = x * q + (x < rem ? x : rem) + i, nt = at / kParts % cols, r0 = at % kParts * BM;
    const r9vx_u32x4 tile = moe_tile(a, at / (kParts * cols));
    if (r0 >= tile.z) return;
    const uint32_t first = tile.y + r0; /* this workgroup's first sorted position */
    Fp8Rows r{};
    r.w = a.g.w + (uint64_t)tile.x * (UP ? 2u : 1u) * a.g.n * a.g.k;
    r.ws = a.g.ws + (uint64_t)tile.x * (UP ? 2u : 1u) * a.g.nb * a.g.kb;
    r.rows = tile.z - r0 < BM ? tile.z - r0 : (uint32_t)BM;
    r.m0 = UP ? 0u : first;
    if (UP) {
        for (uint32_t j = threadIdx.x; j < r.rows; j += 512) token[j] = moe_token(a, first + j);
        __syncthreads();
        r.list = token;
    }
    T t;
    t.run(a.g, r, nt, lds);
    t.drain(r.rows, lds, [&](uint32_t t0) {
        if constexpr (UP) {
            /* a row's 128 columns are one block of h: eight lanes, sixteen values each */
            const uint32_t part = threadIdx.x & 7u;
            for (uint32_t row = threadIdx.x >> 3; row < T::kPass && t0 + row < r.rows; row += 64) {
                r9vx_f32x4 v[4];
                uint32_t amax = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = *reinterpret_cast<const r9vx_f32x4 *>(lds + T::at(row, part * 4 + j));
                    amax = max(max(amax, max(fp8_absbits(v[j].x), fp8_absbits(v[j].y))), max(fp8_absbits(v[j].z), fp8_absbits(v[j].w)));
                }
                const Fp8Scale s = fp8_scale(fp8_max8(amax));
                r9vx_u32x4 c;
                const float inv = 1.0f / s.s;
                c.x = fp8_near4(v[0].x, v[0].y, v[0].z, v[0].w, s, inv);
                c.y = fp8_near4(v[1].x, v[1].y, v[1].z, v[1].w, s, inv);
                c.z = fp8_near4(v[2].x, v[2].y, v[2].z, v[2].w, s, inv);
                c.w = fp8_near4(v[3].x, v[3].y, v[3].z, v[3].w, s, inv);
                const uint64_t pos = (uint64_t)first + t0 + row;
                *reinterpret_cast<r9vx_u32x4 *>(a.hq + pos * a.g.n + nt * 128 + part * 16) = c;
                if (part == 0) a.hs[pos * a.g.nb + nt] = s.s;
            }
        } else {
            static_assert(T::kCols == 256 && kOutBlock == 128, "a wave's 64 quads are two blocks of a row");
            const uint32_t quad = threadIdx.x & 63u, n = nt * T::kCols + quad * 4;
            for (uint32_t row = threadIdx.x >> 6; row < T::kPass && t0 + row < r.rows; row += 8) {
                const r9vx_f32x4 v = *reinterpret_cast<const r9vx_f32x4 *>(lds + T::at(row, quad));
                const uint64_t pos = (uint64_t)first + t0 + row;
                if (a.L.half) {
                    auto finite = [](float f) { return fp8_absbits(f) < 0x7F800000u ? fp8_absbits(f) : 0u; };
                    uint32_t top = n < a.g.n ? max(max(finite(v.x), finite(v.y)), max(finite(v.z), finite(v.w))) : 0u;
                    top = fp8_max32(top) >> 23;
                    top = top < 27u ? 27u : top > 253u ? 253u : top; /* both powers stay normal numbers */
                    const float f = __builtin_bit_cast(float, (254u - top) << 23);
                    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
                    const half4 h = {(_Float16)(v.x * f), (_Float16)(v.y * f), (_Float16)(v.z * f), (_Float16)(v.w * f)};
                    if (n < a.g.n) *reinterpret_cast<half4 *>(reinterpret_cast<_Float16 *>(a.out) + pos * a.g.n + n) = h;
                    if (quad % 32 == 0 && n < a.g.n) a.os[pos * (a.g.n / kOutBlock) + n / kOutBlock] = __builtin_bit_cast(float, top << 23);
                } else if (n < a.g.n) {
                    *reinterpret_cast<r9vx_f32x4 *>(a.out + pos * a.g.n + n) = v;
                }
            }
        }
    });
}

struct Fp8CombineArgs {
    const float *weights;
    const float *o, *os;
    void *y;
    const uint8_t *ws;
    Fp8MoeLayout L;
    uint32_t t, k, dm, shared, p, y_bf16;
    const uint32_t *ids;
    uint32_t *status; /* the caller's word, or NULL */
    uint32_t nan_refused;
};

/* Four outputs of y. */
__device__ __forceinline__ void moe_store(const Fp8CombineArgs &a, uint64_t at, r9vx_f32x4 v) {
    if (a.y_bf16)
        *reinterpret_cast<r9vx_u32x2 *>(static_cast<uint16_t *>(a.y) + at) =
            r9vx_u32x2{(uint32_t)r9vx_f32_to_bf16(v.x) | ((uint32_t)r9vx_f32_to_bf16(v.y) << 16),
                       (uint32_t)r9vx_f32_to_bf16(v.z) | ((uint32_t)r9vx_f32_to_bf16(v.w) << 16)};
    else
        *reinterpret_cast<r9vx_f32x4 *>(static_cast<float *>(a.y) + at) = v;
}

/* y[t] = sum over the token's rows in ascending sorted position (= ascending
 * (expert, slot)) of w * o, then the shared experts' rows.  A workgroup takes
 * 256 pieces of one token: 4 columns each, or 8 of an f16 o. */
template <bool HALF>
__global__ __launch_bounds__(256) void fp8_moe_combine_kernel(Fp8CombineArgs a) {
    __shared__ uint32_t spos[kMoeMaxK], opos[kMoeMaxK];
    __shared__ float sw[kMoeMaxK], ow[kMoeMaxK];
    constexpr uint32_t kQuads = HALF ? 2 : 1;
    const uint32_t t = blockIdx.x, kk = a.k, d = (blockIdx.y * 256 + threadIdx.x) * 4 * kQuads;
    const uint32_t refused = reinterpret_cast<const uint32_t *>(a.ws + a.L.sort.status)[0];
    const bool row = a.ids[(uint64_t)t * kk] == 0xFFFFFFFFu; /* the call was not refused: a row that was */
    if (refused != 0u || row) { /* no y, or NaN */
        if (refused != 0u && a.status && (t | blockIdx.y | threadIdx.x) == 0u) atomicOr(a.status, refused);
        const float nan = __builtin_nanf("");
        for (uint32_t i = 0; i < kQuads; ++i)
            if ((refused == 0u || a.nan_refused) && d < a.dm) moe_store(a, (uint64_t)t * a.dm + d + i * 4, r9vx_f32x4{nan, nan, nan, nan});
        return;
    }
    if (threadIdx.x < kk) {
        spos[threadIdx.x] = reinterpret_cast<const uint32_t *>(a.ws + a.L.sort.inv)[(uint64_t)t * kk + threadIdx.x];
        sw[threadIdx.x] = a.weights[(uint64_t)t * kk + threadIdx.x];
    }
    __syncthreads();
    if (threadIdx.x < kk) {
        const uint32_t p = spos[threadIdx.x];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < kk; ++j) rank += spos[j] < p ? 1u : 0u;
        opos[rank] = p;
        ow[rank] = sw[threadIdx.x];
    }
    __syncthreads();
    if (d >= a.dm) return;
    r9vx_f32x4 acc[kQuads];
#pragma unroll
    for (uint32_t i = 0; i < kQuads; ++i) acc[i] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](float w, uint64_t row) {
        if constexpr (HALF) {
            typedef _Float16 half8 __attribute__((ext_vector_type(8)));
            const half8 h = __builtin_bit_cast(half8, __builtin_nontemporal_load(
                reinterpret_cast<const r9vx_u32x4 *>(reinterpret_cast<const _Float16 *>(a.o) + row * a.dm + d)));
            const float f = a.os[row * (a.dm / kOutBlock) + d / kOutBlock];
            acc[0] = acc[0] + w * (f * r9vx_f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]});
            acc[1] = acc[1] + w * (f * r9vx_f32x4{(float)h[4], (float)h[5], (float)h[6], (float)h[7]});
        } else {
            acc[0] = acc[0] + w * __builtin_nontemporal_load(reinterpret_cast<const r9vx_f32x4 *>(a.o + row * a.dm + d));
        }
    };
#pragma unroll 4
    for (uint32_t j = 0; j < kk; ++j) add(ow[j], opos[j]);
    for (uint32_t s = 0; s < a.shared; ++s) add(1.0f, (uint64_t)a.p + (uint64_t)s * a.t + t);
#pragma unroll
    for (uint32_t i = 0; i < kQuads; ++i) moe_store(a, (uint64_t)t * a.dm + d + i * 4, acc[i]);
}

/* The launch's list entries are at most this many (their own count is on the device). */
uint64_t moe_tiles(const r9vx_moe_fp8_problem &p, uint32_t t) {
    const uint64_t pairs = (uint64_t)t * p.k;
    return (pairs + (uint64_t)p.shared * t) / kMoeTileM3 + (pairs < p.e ? pairs : p.e) + p.shared;
}
/* f32 outputs: the exact tiles of 128 rows */
uint32_t moe_tile_rows(const r9vx_moe_fp8_problem &p) { return p.y_dtype == R9VX_DTYPE_F32 ? 128 : 256; }
/* Workgroups of the tiles' launches; seven more, for an even share to each XCD. */
uint64_t moe_up_tiles(const r9vx_moe_fp8_problem &p, uint64_t tiles) { return tiles * (kMoeTileM3 / moe_tile_rows(p)) * ((p.dff + 127) / 128) + 7; }
uint64_t moe_down_tiles(const r9vx_moe_fp8_problem &p, uint64_t tiles) { return tiles * (kMoeTileM3 / moe_tile_rows(p)) * ((p.dm + 255) / 256) + 7; }

template <int BM, bool EXACT>
int launch_tiles(const r9vx_moe_fp8_problem &p, const Fp8MoeArgs &up, const Fp8MoeArgs &dn, uint64_t tiles, hipStream_t s) {
    hipLaunchKernelGGL((fp8_moe_tile_kernel<true, BM, EXACT>), dim3((uint32_t)moe_up_tiles(p, tiles)), dim3(512), 0, s, up);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL((fp8_moe_tile_kernel<false, BM, EXACT>), dim3((uint32_t)moe_down_tiles(p, tiles)), dim3(512), 0, s, dn);
    return (int)hipGetLastError();
}

}  // namespace

size_t r9vx_moe_fp8_workspace_bytes(const r9vx_moe_fp8_problem &p) { return moe_layout(p).total; }

bool r9vx_moe_fp8_launchable(const r9vx_moe_fp8_problem &p) {
    const uint64_t tiles = moe_tiles(p, p.t_bucket), up = moe_up_tiles(p, tiles), down = moe_down_tiles(p, tiles);
    return moe_streams(p) || (up > down ? up : down) * 512 < 1ull << 32;
}

const uint32_t *r9vx_moe_fp8_status_word(const r9vx_moe_fp8_problem &p) {
    return reinterpret_cast<const uint32_t *>(p.ws + moe_layout(p).sort.status);
}

int r9vx_launch_moe_fp8(const r9vx_moe_fp8_problem &p, hipStream_t stream) {
    const Fp8MoeLayout L = moe_layout(p);
    uint8_t *const xq = p.ws + L.xq, *const hq = p.ws + L.hq;
    float *const xs = reinterpret_cast<float *>(p.ws + L.xs), *const hs = reinterpret_cast<float *>(p.ws + L.hs);
    float *const h = reinterpret_cast<float *>(p.ws + L.h), *const o = reinterpret_cast<float *>(p.ws + L.o);
    int rc = r9vx_launch_quantize_fp8(p.x, R9VX_DTYPE_BF16, p.t, p.dm, p.dm, xq, xs, stream);
    if (rc) return rc;
    r9vx_moe_problem sp{};
    sp.ids = p.ids;
    sp.ws = p.ws;
    sp.t = p.t;
    sp.e = p.e;
    sp.k = p.k;
    sp.shared = p.shared;
    sp.skip_refused = 1;
    rc = r9vx_moe_sort_stage(sp, L.sort, stream, false);
    if (rc) return rc;
    const uint32_t pairs = p.t * p.k, rows = pairs + p.shared * p.t;
    Fp8MoeArgs up{}, dn{};
    up.ws = dn.ws = p.ws;
    up.L = dn.L = L;
    up.p = dn.p = pairs;
    up.t = dn.t = p.t;
    up.topk = dn.topk = p.k;
    up.g.w = p.w_gu;
    up.g.ws = p.s_gu;
    up.g.xq = xq;
    up.g.xs = xs;
    up.g.n = p.dff;
    up.g.k = p.dm;
    up.g.nb = p.dff / kFp8Block;
    up.g.kb = p.dm / kFp8Block;
    up.out = h;
    up.hq = hq;
    up.hs = hs;
    dn.g.w = p.w_dn;
    dn.g.ws = p.s_dn;
    dn.g.xq = hq;
    dn.g.xs = hs;
    dn.g.n = p.dm;
    dn.g.k = p.dff;
    dn.g.nb = p.dm / kFp8Block;
    dn.g.kb = p.dff / kFp8Block;
    dn.out = o;
    dn.os = reinterpret_cast<float *>(p.ws + L.os);
    const uint32_t tiles = (uint32_t)moe_tiles(p, p.t);
    if (L.stream) {
        hipLaunchKernelGGL((fp8_moe_stream_kernel<1, 2, 4, true>), dim3(p.dff / 16, tiles), dim3(256), 0, stream, up);
        rc = (int)hipGetLastError();
        if (!rc) rc = r9vx_launch_quantize_fp8(h, R9VX_DTYPE_F32, rows, p.dff, p.dff, hq, hs, stream);
        if (rc) return rc;
        hipLaunchKernelGGL((fp8_moe_stream_kernel<1, 2, 4, false>), dim3(p.dm / 32, tiles), dim3(256), 0, stream, dn);
        rc = (int)hipGetLastError();
        if (rc) return rc;
    } else {
        rc = moe_tile_rows(p) == 128 ? launch_tiles<128, true>(p, up, dn, tiles, stream) : launch_tiles<256, false>(p, up, dn, tiles, stream);
        if (rc) return rc;
    }
    const Fp8CombineArgs c{p.weights, o, dn.os, p.y, p.ws, L, p.t, p.k, p.dm, p.shared, pairs, p.y_dtype == R9VX_DTYPE_BF16, p.ids,
                           p.status, p.nan_refused};
    if (L.half)
        hipLaunchKernelGGL(fp8_moe_combine_kernel<true>, dim3(p.t, (p.dm / 8 + 255) / 256), dim3(256), 0, stream, c);
    else
        hipLaunchKernelGGL(fp8_moe_combine_kernel<false>, dim3(p.t, (p.dm / 4 + 255) / 256), dim3(256), 0, stream, c);
    return (int)hipGetLastError();
}
