/*
 * r9vx_e4m3_gemm.h -- the two main loops of the block-scaled e4m3 products,
 * shared by the dense matmul and the grouped expert GEMMs.
 */
#ifndef R9VX_E4M3_GEMM_H
#define R9VX_E4M3_GEMM_H

#include "r9vx_e4m3.h"

struct Fp8Args {
    const uint8_t *w;      /* e4m3 [n or 2n, k] */
    const float *ws;       /* [nb or 2 nb, kb] */
    const void *x;         /* activations as given (in-kernel quantization) */
    const uint8_t *xq;     /* e4m3 [rows, k] */
    const float *xs;       /* [rows, kb] */
    const float *bias;
    const float *residual;
    void *y;
    uint32_t m, n, k, kb, nb;
    uint32_t y_bf16, epilogue;
    uint32_t m_tiles, n_tiles;
};

/* The weights and activation rows of one workgroup: rows m0 .. m0 + rows - 1,
 * or, with an index list, rows list[m0] .. list[m0 + rows - 1]. */
struct Fp8Rows {
    const uint8_t *w;
    const float *ws;
    uint32_t m0, rows;
    const uint32_t *list; /* NULL: none */
};

#ifdef __HIPCC__
namespace r9vx {

/* Four consecutive outputs of one row with the dense epilogues. */
__device__ __forceinline__ void fp8_store_dense(const Fp8Args &a, uint32_t m, uint32_t n, r9vx_f32x4 v) {
    const uint64_t at = (uint64_t)m * a.n + n;
    if ((a.n & 3u) == 0) { /* whole quads, 16- and 8-byte aligned */
        if (a.epilogue == R9VX_EPILOGUE_BIAS) {
            const r9vx_f32x4 b = *reinterpret_cast<const r9vx_f32x4 *>(a.bias + n);
            v = v + b;
        } else if (a.epilogue == R9VX_EPILOGUE_RESIDUAL) {
            const r9vx_f32x4 b = *reinterpret_cast<const r9vx_f32x4 *>(a.residual + at);
            v = v + b;
        }
        if (a.y_bf16)
            *reinterpret_cast<r9vx_u32x2 *>(static_cast<uint16_t *>(a.y) + at) =
                r9vx_u32x2{(uint32_t)r9vx_f32_to_bf16(v.x) | ((uint32_t)r9vx_f32_to_bf16(v.y) << 16),
                           (uint32_t)r9vx_f32_to_bf16(v.z) | ((uint32_t)r9vx_f32_to_bf16(v.w) << 16)};
        else
            *reinterpret_cast<r9vx_f32x4 *>(static_cast<float *>(a.y) + at) = v;
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (n + i >= a.n) return;
        float s = v[i];
        if (a.epilogue == R9VX_EPILOGUE_BIAS) s = s + a.bias[n + i];
        if (a.epilogue == R9VX_EPILOGUE_RESIDUAL) s = s + a.residual[at + i];
        if (a.y_bf16)
            static_cast<uint16_t *>(a.y)[at + i] = r9vx_f32_to_bf16(s);
        else
            static_cast<float *>(a.y)[at + i] = s;
    }
}

__device__ __forceinline__ float fp8_silu(float g) { return g / (1.0f + expf(-g)); }

__device__ __forceinline__ r9vx_f32x4 fp8_swiglu(r9vx_f32x4 g, r9vx_f32x4 u) {
    return r9vx_f32x4{fp8_silu(g.x) * u.x, fp8_silu(g.y) * u.y, fp8_silu(g.z) * u.z, fp8_silu(g.w) * u.w};
}

/* ------------------------------------------------------------------ stream */

/* One operand's 32 bytes of a lane for one 128-column block: 16-byte chunks g
 * and g + 4 of its row (the four lanes of a row read 64 contiguous bytes per
 * load); chunks past the row's end are zero. */
__device__ __forceinline__ i32x8 fp8_load_frag(const uint8_t *row, uint32_t g, uint32_t left) {
    r9vx_u32x4 lo = {0u, 0u, 0u, 0u}, hi = {0u, 0u, 0u, 0u};
    if (g * 16 < left) lo = *reinterpret_cast<const r9vx_u32x4 *>(row + g * 16);
    if (g * 16 + 64 < left) hi = *reinterpret_cast<const r9vx_u32x4 *>(row + g * 16 + 64);
    return fp8_frag(lo, hi);
}

template <int MT, int NT>
struct Fp8StreamRegs {
    i32x8 w[NT], x[MT];
    float sx[MT], sw[2];
};

/* Weight strip `strip` (NT tiles of 16 weight rows; GATED: NT / 2 of gate rows
 * and the NT / 2 of up rows beside them) times MT tiles of 16 activation rows.
 * Wave v takes the K blocks v, v + W, ...; the W partial sums are joined in
 * wave order in LDS.  store(row, n, four sums) gets each quad once. */
template <int MT, int NT, int W, int XT, bool GATED, typename Store>
__device__ __forceinline__ void fp8_stream(const Fp8Args &a, const Fp8Rows &r, uint32_t strip, r9vx_f32x4 *part, Store store) {
    constexpr int NC = GATED ? NT / 2 : NT; /* output tiles */
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15u;
    const uint32_t n0 = strip * (NC * 16);
    const uint8_t *wrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        uint32_t n = n0 + (uint32_t)(j % NC) * 16 + c;
        n = n < a.n ? n : a.n - 1;
        wrow[j] = r.w + ((uint64_t)n + (GATED && j >= NC ? a.n : 0u)) * a.k;
    }
    const uint8_t *xrow[MT];
    const float *srow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        uint32_t m = i * 16 + c;
        m = r.m0 + (m < r.rows ? m : r.rows - 1);
        if (r.list) m = r.list[m];
        xrow[i] = a.xq + (uint64_t)m * a.k;
        srow[i] = a.xs + (uint64_t)m * a.kb;
    }
    /* a strip lies in one 128-row block of the weight scales: 128 is a multiple of its 16 NC rows */
    const float *wsg = r.ws + (uint64_t)(n0 / kFp8Block) * a.kb, *wsu = wsg + (uint64_t)a.nb * a.kb;
    auto load = [&](Fp8StreamRegs<MT, NT> &q, uint32_t kb) {
        const uint32_t k0 = kb * kFp8Block, left = a.k - k0;
#pragma unroll
        for (int j = 0; j < NT; ++j) q.w[j] = fp8_load_frag(wrow[j] + k0, g, left);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            q.x[i] = fp8_load_frag(xrow[i] + k0, g, left);
            q.sx[i] = srow[i][kb];
        }
        q.sw[0] = wsg[kb];
        if constexpr (GATED) q.sw[1] = wsu[kb];
    };
    r9vx_f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](const Fp8StreamRegs<MT, NT> &q) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const r9vx_f32x4 d = fp8_mma<true>(q.w[j], q.x[i]);
                const float s = q.sx[i] * q.sw[GATED && j >= NC ? 1 : 0];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
            }
    };
    Fp8StreamRegs<MT, NT> q0, q1;
    uint32_t kb = wave;
    if (kb < a.kb) load(q0, kb);
    for (; kb < a.kb; kb += 2 * W) {
        if (kb + W < a.kb) load(q1, kb + W);
        add(q0);
        if (kb + W >= a.kb) break;
        if (kb + 2 * W < a.kb) load(q0, kb + 2 * W);
        add(q1);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < MT * NC * 64; o += W * 64) {
        const uint32_t l = o & 63u, i = (o >> 6) / NC, j = (o >> 6) % NC;
        r9vx_f32x4 v = part[(i * NT + j) * 64 + l], u = {0.f, 0.f, 0.f, 0.f};
        if constexpr (GATED) u = part[(i * NT + j + NC) * 64 + l];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            v = v + part[((w * MT + i) * NT + j) * 64 + l];
            if constexpr (GATED) u = u + part[((w * MT + i) * NT + j + NC) * 64 + l];
        }
        if constexpr (GATED) v = fp8_swiglu(v, u);
        const uint32_t row = i * 16 + (l & 15u), n = n0 + j * 16 + (l >> 4) * 4;
        if (row < r.rows && n < a.n) store(row, n, v);
    }
}

/* ------------------------------------------------------------------ tile */

/* BM activation rows x BN weight rows, K steps of 128, 8 waves as WM x 8 / WM:
 * wave (wm, wn) owns the 16-row tiles wm, wm + WM, ... of the activations and
 * BN / WN weight rows (GATED: half of them gate rows, half the up rows beside
 * them).  Both operands and the rows' scales of a step are copied straight
 * into LDS one step ahead; rows are 128 bytes of eight 16-byte chunks, chunk
 * c of row r at slot c ^ (r / 2 % 8), which the 16 rows of one LDS read spread
 * over all banks. */
template <int BM, int BN, int WM, bool GATED, bool EXACT>
struct Fp8Tile {
    static constexpr int WN = 8 / WM, TM = BM / 16 / WM, TN = BN / 16 / WN, NC = GATED ? TN / 2 : TN;
    static constexpr uint32_t kX = BM * 128, kW = BN * 128, kS = BM * 4, kStage = kX + kW + kS, kLds = 2 * kStage;
    static constexpr int IX = BM / 64, IW = BN / 64; /* copies of 8 rows per wave and step */
    static_assert(BM % 64 == 0 && BN % 128 == 0 && TM * 16 * WM == BM && TN * 16 * WN == BN, "");
    static_assert(GATED ? BN / 2 <= 128 : BN / WN <= 128, "a wave's rows share one block of weight scales");
    static_assert(kStage % 16 == 0 && kLds <= 160 * 1024, "");

    r9vx_f32x4 acc[TM][TN];

    static __device__ __forceinline__ void copy16(uint32_t lds_at, const uint8_t *base, uint32_t off) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_at)
                     : "memory", "m0");
    }
    static __device__ __forceinline__ void copy4(uint32_t lds_at, const float *base, uint32_t off) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds_at)
                     : "memory", "m0");
    }

    /* ALL: every row tile of the workgroup holds rows. */
    template <bool ALL>
    __device__ __forceinline__ void run(const Fp8Args &a, const Fp8Rows &r, uint32_t nt, uint8_t *lds) {
        const uint32_t lane = threadIdx.x & 63u;
        const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        const uint32_t wm = wave / WN, wn = wave % WN;
        const uint32_t n0 = nt * (GATED ? BN / 2 : BN);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
        const uint32_t tail = a.k % kFp8Block; /* columns of a last, ragged block */
        const uint32_t act = (r.rows + 15) / 16;

        /* sources of this lane's copies, from the tile's first row */
        uint32_t xo[IX], wo[IW];
        const uint8_t *xbase = r.list ? a.xq : a.xq + (uint64_t)r.m0 * a.k;
        const uint8_t *wg = r.w + (uint64_t)n0 * a.k, *wu = wg + (uint64_t)a.n * a.k;
#pragma unroll
        for (int i = 0; i < IX; ++i) {
            const uint32_t row = (wave * IX + i) * 8 + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u); /* the chunk at this lane's slot */
            const uint32_t in = row < r.rows ? row : r.rows - 1;
            xo[i] = (r.list ? r.list[r.m0 + in] : in) * a.k + c * 16;
        }
#pragma unroll
        for (int i = 0; i < IW; ++i) {
            const uint32_t row = (wave * IW + i) * 8 + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u);
            uint32_t j = GATED && row >= BN / 2 ? row - BN / 2 : row;
            j = n0 + j < a.n ? j : a.n - 1 - n0;
            wo[i] = j * a.k + c * 16;
        }
        uint32_t so = 0;
        const float *sbase = r.list ? a.xs : a.xs + (uint64_t)r.m0 * a.kb;
        if (wave < IX) {
            const uint32_t row = wave * 64 + lane, in = row < r.rows ? row : r.rows - 1;
            so = (r.list ? r.list[r.m0 + in] : in) * a.kb * 4;
        }
        /* this lane's chunk of an even and of an odd copy's row, in bytes */
        const uint32_t ce = ((lane & 7u) ^ (lane >> 4)) * 16, co = ce ^ 64u;
        auto issue = [&](uint32_t kb, uint32_t st) {
            const uint32_t k0 = kb * kFp8Block, at = lds0 + st * kStage;
            const uint32_t cut = tail && kb + 1 == a.kb ? tail : kFp8Block;
            const uint32_t de = ce >= cut ? ce : 0u, dd = co >= cut ? co : 0u; /* past the last column: the row's first chunk */
#pragma unroll
            for (int i = 0; i < IX; ++i) {
                const uint32_t r8 = (wave * IX + i) * 8;
                if (!ALL && r8 >= act * 16) break;
                copy16(at + r8 * 128, xbase + k0, xo[i] - ((wave * IX + i) & 1u ? dd : de));
            }
#pragma unroll
            for (int i = 0; i < IW; ++i) {
                const uint32_t r8 = (wave * IW + i) * 8;
                copy16(at + kX + r8 * 128, (GATED && r8 >= BN / 2 ? wu : wg) + k0, wo[i] - ((wave * IW + i) & 1u ? dd : de));
            }
            if (wave < IX) copy4(at + kX + kW + wave * 256, sbase + kb, so);
        };
        /* chunks past the last column were filled from the row's start: zeros instead */
        auto clear = [&](uint32_t st) {
#pragma unroll
            for (int i = 0; i < IX; ++i) {
                const uint32_t r8 = (wave * IX + i) * 8;
                if (((wave * IX + i) & 1u ? co : ce) >= tail)
                    *reinterpret_cast<r9vx_u32x4 *>(lds + st * kStage + r8 * 128 + lane * 16) = r9vx_u32x4{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < IW; ++i) {
                const uint32_t r8 = (wave * IW + i) * 8;
                if (((wave * IW + i) & 1u ? co : ce) >= tail)
                    *reinterpret_cast<r9vx_u32x4 *>(lds + st * kStage + kX + r8 * 128 + lane * 16) = r9vx_u32x4{0u, 0u, 0u, 0u};
            }
        };
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};

        const uint32_t frag = (lane & 15u) * 128 + (((lane >> 4) ^ ((lane >> 1) & 7u)) << 4);
        const float *wsg = r.ws + (uint64_t)((n0 + (GATED ? 0u : wn * (BN / WN))) / kFp8Block) * a.kb;
        const float *wsu = wsg + (uint64_t)a.nb * a.kb;
        const bool in_n = GATED || n0 + wn * (BN / WN) < a.n; /* else no such scale row; the sums are not stored */
        float swg = 0.f, swu = 0.f; /* lane i: the scale of block 64 (kb / 64) + i */

        issue(0, 0);
        for (uint32_t kb = 0; kb < a.kb; ++kb) {
            const uint32_t st = kb & 1u;
            if ((kb & 63u) == 0) {
                const uint32_t at = kb + lane < a.kb ? kb + lane : a.kb - 1;
                swg = in_n ? wsg[at] : 0.f;
                if constexpr (GATED) swu = wsu[at];
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (tail && kb + 1 == a.kb) clear(st);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (kb + 1 < a.kb) issue(kb + 1, st ^ 1u);
            const uint8_t *xs = lds + st * kStage, *wl = xs + kX;
            const float *sl = reinterpret_cast<const float *>(wl + kW);
            const float sg = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swg), (int)(kb & 63u)));
            const float su = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swu), (int)(kb & 63u)));
            step<ALL>(xs, wl, sl, sg, su, frag, wm, wn, act, lane);
        }
    }

    static __device__ __forceinline__ i32x8 read_frag(const uint8_t *p, uint32_t frag) {
        return fp8_frag(*reinterpret_cast<const r9vx_u32x4 *>(p + frag), *reinterpret_cast<const r9vx_u32x4 *>(p + (frag ^ 64u)));
    }
    __device__ __forceinline__ void fold(r9vx_f32x4 (&o)[TN], const r9vx_f32x4 (&d)[TN], float s0, float s1, int j) {
        const float s = GATED && j >= NC ? s1 : s0;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = fmaf(d[j][e], s, o[j][e]);
    }

    /* One K step: a row tile's products leave the matrix unit while the row
     * tile before it is scaled and added, so neither waits for the other. */
    template <bool ALL>
    __device__ __forceinline__ void step(const uint8_t *xs, const uint8_t *wl, const float *sl, float sg, float su, uint32_t frag,
                                         uint32_t wm, uint32_t wn, uint32_t act, uint32_t lane) {
        i32x8 w[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const uint32_t row = GATED ? (j >= NC ? BN / 2 : 0u) + (wn * NC + j % NC) * 16 : (wn * TN + j) * 16;
            w[j] = read_frag(wl + row * 128, frag);
        }
        xs += wm * 2048;
        sl += wm * 16 + (lane & 15u);
        if constexpr (ALL) {
            i32x8 x = read_frag(xs, frag);
            float sx = *sl;
            r9vx_f32x4 d[2][TN];
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                i32x8 xn = x;
                float sn = sx;
                if (i + 1 < TM) {
                    xn = read_frag(xs + (i + 1) * WM * 2048, frag);
                    sn = sl[(i + 1) * WM * 16];
                }
                const float t0 = sx * sg, t1 = GATED ? sx * su : 0.f;
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    d[i & 1][j] = fp8_mma<EXACT>(w[j], x);
                    if (i > 0) fold(acc[i > 0 ? i - 1 : 0], d[(i & 1) ^ 1], s0, s1, j);
                }
                s0 = t0;
                s1 = t1;
                x = xn;
                sx = sn;
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) fold(acc[TM - 1], d[(TM - 1) & 1], s0, s1, j);
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (i * WM + wm < act) {
                    const i32x8 x = read_frag(xs + i * WM * 2048, frag);
                    const float sx = sl[i * WM * 16], t0 = sx * sg, t1 = GATED ? sx * su : 0.f;
                    r9vx_f32x4 d[TN];
#pragma unroll
                    for (int j = 0; j < TN; ++j) d[j] = fp8_mma<EXACT>(w[j], x);
#pragma unroll
                    for (int j = 0; j < TN; ++j) fold(acc[i], d, t0, t1, j);
                }
            }
        }
    }

    /* Output columns of a tile, rows that go through LDS at once. */
    static constexpr uint32_t kCols = GATED ? BN / 2 : BN;
    static constexpr uint32_t kPass = (uint32_t)BM * kCols * 4 > kLds ? BM / 2 : BM;
    static_assert(kPass * kCols * 4 <= kLds && BM % kPass == 0 && kPass % (WM * 16) == 0, "");

    /* The tile through LDS as f32 rows, kPass at a time, so that it leaves in
     * whole rows: emit(first tile row) finds quad q of row t of the pass at
     * at(t, q).  The quads of a row are swizzled by it, so that the 16 rows
     * that a wave writes at a time lie in different banks. */
    static __device__ __forceinline__ uint32_t at(uint32_t t, uint32_t quad) { return (t * (kCols / 4) + (quad ^ (t & 15u))) * 16; }
    template <typename Emit>
    __device__ __forceinline__ void drain(uint8_t *lds, Emit emit) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
        constexpr int TP = kPass / (WM * 16);
#pragma unroll
        for (int p = 0; p < TM / TP; ++p) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    r9vx_f32x4 v = acc[p * TP + i][j];
                    if constexpr (GATED) v = fp8_swiglu(v, acc[p * TP + i][j + NC]);
                    *reinterpret_cast<r9vx_f32x4 *>(lds + at((i * WM + wm) * 16 + (lane & 15u), (wn * NC + j) * 4 + (lane >> 4))) = v;
                }
            __syncthreads();
            emit(p * kPass);
        }
    }
};

}  // namespace r9vx
#endif
#endif
