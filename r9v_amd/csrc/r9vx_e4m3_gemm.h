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
    const void *x;         /* activations as given, where a workgroup quantizes them itself */
    const uint8_t *xq;     /* e4m3 rows of kb whole blocks, zeros past column k */
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

/* f(0), f(1), ... f(N - 1) with the index a constant expression. */
template <int I>
struct Fp8Int {
    static constexpr int v = I;
};
template <int N, int I = 0, typename F>
__device__ __forceinline__ void fp8_for(F &&f) {
    if constexpr (I < N) {
        f(Fp8Int<I>{});
        fp8_for<N, I + 1>(f);
    }
}

/* o + s d */
__device__ __forceinline__ r9vx_f32x4 fp8_add_scaled(r9vx_f32x4 o, r9vx_f32x4 d, float s) {
    return r9vx_f32x4{fmaf(d.x, s, o.x), fmaf(d.y, s, o.y), fmaf(d.z, s, o.z), fmaf(d.w, s, o.w)};
}

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

/* g / (1 + exp(-g)) by the hardware's exponential and reciprocal, a step each (of a
 * tile's epilogue the library's exponential and divide took a third of the time
 * of its products).  e = exp(-|g| / 2) neither overflows nor underflows where the
 * result is a normal number: silu = g / (1 + e^2) for g >= 0, g e^2 / (1 + e^2)
 * below.  e is off by 2^-22 of itself (the exponential's step, its correction by
 * the low half of |g| log2(e) / 2 and their product), its square by 2^-21, and
 * the other roundings add 6 x 2^-24: under 2^-20 of the value, or 2^-149 where it
 * is denormal.  From |g| = 256 on e is 0.  -infinity gives NaN, as the formula. */
__device__ __forceinline__ float fp8_silu(float g) {
    const float c = fminf(fabsf(g), 256.0f);
    const float t = c * -0x1.715476p-1f;
    const float low = fmaf(c, -0x1.4ae0cp-27f, fmaf(c, -0x1.715476p-1f, -t));
    const float e = __builtin_amdgcn_exp2f(t) * fmaf(low, 0x1.62e43p-1f, 1.0f);
    return (g < 0.0f ? g * e * e : g) * __builtin_amdgcn_rcpf(fmaf(e, e, 1.0f));
}

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

/* How the activations of a streaming product come. */
enum Fp8X { kFp8Codes, /* e4m3 rows of whole blocks, and their scales */
            kFp8F32,   /* rows of K values, which each workgroup quantizes into its LDS */
            kFp8Bf16 };

/* Quantized rows in LDS: a row's codes, whole blocks with zeros past column k,
 * 16 bytes between rows so that a chunk of 16 rows lies in all banks; then the
 * rows' scales. */
__host__ __device__ inline uint32_t fp8_lds_row(uint32_t kb) { return kb * kFp8Block + 16; }
__host__ __device__ inline uint32_t fp8_lds_rows_bytes(uint32_t rows, uint32_t kb) { return rows * (fp8_lds_row(kb) + kb * 4); }

/* Whether `rows` of them leave room for two workgroups on a CU. */
inline bool fp8_fits_lds(uint32_t rows, uint32_t kb) { return fp8_lds_rows_bytes(rows, kb) <= 48 * 1024; }

template <int W, bool F32>
__device__ __forceinline__ void fp8_quantize_rows(const Fp8Args &a, const Fp8Rows &r, uint8_t *lds) {
    const uint32_t part = threadIdx.x & 7u, blocks = r.rows * a.kb;
    float *const scales = reinterpret_cast<float *>(lds + r.rows * fp8_lds_row(a.kb));
    for (uint32_t i = threadIdx.x >> 3; i < blocks; i += W * 8) {
        const uint32_t row = i / a.kb, b = i - row * a.kb, left = a.k - b * kFp8Block, m = r.m0 + row;
        Fp8Block<F32> block;
        block.load(static_cast<const uint8_t *>(a.x) + ((uint64_t)m * a.k + b * kFp8Block) * (F32 ? 4 : 2), left, part);
        uint32_t code[4];
        const float s = block.codes(code);
        uint8_t *const to = lds + row * fp8_lds_row(a.kb) + b * kFp8Block;
#pragma unroll
        for (int j = 0; j < block.N; ++j) {
            const uint32_t c = block.column(j, part);
            if constexpr (F32)
                *reinterpret_cast<uint32_t *>(to + c) = c < left ? code[j] : 0u;
            else
                *reinterpret_cast<r9vx_u32x2 *>(to + c) = c < left ? r9vx_u32x2{code[2 * j], code[2 * j + 1]} : r9vx_u32x2{0u, 0u};
        }
        if (part == 0) scales[i] = s;
    }
}

template <int MT, int NT>
struct Fp8StreamRegs {
    i32x8 w[NT], x[MT];
    float sx[MT], sw[2];
};

/* Weight strip `strip` (NT tiles of 16 weight rows; GATED: NT / 2 of gate rows
 * and the NT / 2 of up rows beside them) times MT tiles of 16 activation rows.
 * Wave v takes the K blocks v, v + W, ...; the W partial sums are joined in
 * wave order in LDS.  prepare() makes the rows' list, store(row, n, four sums)
 * gets each quad once.
 * Weights are read once and used for 16 rows: what bounds it is how many loads
 * are in flight, so every wave has two blocks' worth, nothing passes through
 * LDS on the way, and the strips are narrow (32 weight rows) to have many
 * workgroups.  64 experts' gate and up rows of 2 x 1408 x 2048: 65 to 75 us, 5.7 to
 * 4.9 TB/s. */
template <int MT, int NT, int W, int XT, bool GATED, typename Prepare, typename Store>
__device__ __forceinline__ void fp8_stream(const Fp8Args &a, const Fp8Rows &r, uint32_t strip, r9vx_f32x4 *part, uint8_t *rows, Prepare prepare,
                                           Store store) {
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
    /* a strip lies in one 128-row block of the weight scales: 128 is a multiple of its 16 NC rows */
    const float *wsg = r.ws + (uint64_t)(n0 / kFp8Block) * a.kb, *wsu = wsg + (uint64_t)a.nb * a.kb;
    auto load_w = [&](Fp8StreamRegs<MT, NT> &q, uint32_t kb) {
        const uint32_t k0 = kb * kFp8Block, left = a.k - k0;
#pragma unroll
        for (int j = 0; j < NT; ++j) q.w[j] = fp8_load_frag(wrow[j] + k0, g, left);
        q.sw[0] = wsg[kb];
        if constexpr (GATED) q.sw[1] = wsu[kb];
    };
    Fp8StreamRegs<MT, NT> q0, q1;
    uint32_t kb = wave;
    if (kb < a.kb) load_w(q0, kb); /* on their way while the rows are found, or quantized */
    prepare();
    const uint8_t *xrow[MT];
    const float *srow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        uint32_t m = i * 16 + c;
        if constexpr (XT != kFp8Codes) {
            m = m < r.rows ? m : r.rows - 1;
            xrow[i] = rows + m * fp8_lds_row(a.kb);
            srow[i] = reinterpret_cast<const float *>(rows + r.rows * fp8_lds_row(a.kb)) + m * a.kb;
            continue;
        }
        m = r.m0 + (m < r.rows ? m : r.rows - 1);
        if (r.list) m = r.list[m];
        xrow[i] = a.xq + (uint64_t)m * (a.kb * kFp8Block);
        srow[i] = a.xs + (uint64_t)m * a.kb;
    }
    auto load_x = [&](Fp8StreamRegs<MT, NT> &q, uint32_t kb) {
        const uint32_t k0 = kb * kFp8Block;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            q.x[i] = fp8_load_frag(xrow[i] + k0, g, kFp8Block);
            q.sx[i] = srow[i][kb];
        }
    };
    auto load = [&](Fp8StreamRegs<MT, NT> &q, uint32_t kb) {
        load_w(q, kb);
        load_x(q, kb);
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
                acc[i][j] = fp8_add_scaled(acc[i][j], d, s);
            }
    };
    if constexpr (XT != kFp8Codes) {
        fp8_quantize_rows<W, XT == kFp8F32>(a, r, rows);
        __syncthreads();
    }
    if (kb < a.kb) load_x(q0, kb);
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

/* Copies by the lanes of `mask` (all or none: a branch around them would
 * cut the step's schedule in pieces). */
__device__ __forceinline__ void fp8_copy16(uint32_t lds_at, const uint8_t *base, uint32_t off, uint32_t mask) {
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1" ::"v"(off),
                 "s"(base), "s"(lds_at), "s"(mask)
                 : "memory", "m0");
}
__device__ __forceinline__ void fp8_copy4(uint32_t lds_at, const float *base, uint32_t off, uint32_t mask) {
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dword %0, %1\n\ts_mov_b64 exec, -1" ::"v"(off),
                 "s"(base), "s"(lds_at), "s"(mask)
                 : "memory", "m0");
}

/* The mask of a copy: all lanes where a < b.  In a scalar register whatever the
 * compiler makes of the comparison (the value is hidden from it, or it would
 * take the vector register it knows to be uniform). */
__device__ __forceinline__ uint32_t fp8_copy_mask(uint32_t a, uint32_t b) {
    int32_t v = (int32_t)(a - b) >> 31;
    asm("" : "+v"(v));
    return (uint32_t)__builtin_amdgcn_readfirstlane(v);
}
/* A fragment from LDS rows of 128 bytes whose chunk c stands at slot c ^ (row / 2 % 8). */
__device__ __forceinline__ i32x8 fp8_read_frag(const uint8_t *p, uint32_t frag) {
    return fp8_frag(*reinterpret_cast<const r9vx_u32x4 *>(p + frag), *reinterpret_cast<const r9vx_u32x4 *>(p + (frag ^ 64u)));
}


/* BM activation rows x BN weight rows, K steps of 128, 8 waves as WM x 8 / WM:
 * wave (wm, wn) owns the 16-row tiles wm, wm + WM, ... of the activations and
 * BN / WN weight rows (GATED: half of them gate rows, half the up rows beside
 * them).  Both operands and the rows' scales of a step are copied straight
 * into LDS one step ahead; rows are 128 bytes of eight 16-byte chunks, chunk
 * c of row r at slot c ^ (r / 2 % 8), which the 16 rows of one LDS read spread
 * over all banks.
 * A 256 x 256 step takes 1.8 us: its matrix instructions alone need 0.86 at the
 * full clock, its LDS reads and copies as much, and under random codes the
 * clock falls to about 1.6 GHz (all zeros: a tenth faster).  Three to five
 * stages, a persistent workgroup and lines touched ahead brought nothing. */
template <int BM, int BN, int WM, bool GATED, bool EXACT>
struct Fp8Tile {
    static constexpr int WN = 8 / WM, TM = BM / 16 / WM, TN = BN / 16 / WN, NC = GATED ? TN / 2 : TN;
    static constexpr uint32_t kX = BM * 128, kW = BN * 128, kS = BM * 4, kStage = kX + kW + kS, kLds = 2 * kStage;
    static constexpr int IW = BN / 64; /* copies of 8 weight rows per wave and step */
    static_assert(BM % 64 == 0 && BN % 64 == 0 && TM * 16 * WM == BM && TN * 16 * WN == BN, "");
    static_assert(GATED ? BN / 2 <= 128 : BN / WN <= 128, "a wave's rows share one block of weight scales");
    static_assert(kStage % 16 == 0 && kLds <= 160 * 1024, "");

    r9vx_f32x4 acc[TM][TN];

    /* The products of the tile's rows: of all its row tiles, of three, two or
     * one quarter of them, whatever holds the rows (tiles of 128 rows have no
     * three quarters, smaller ones only the whole). */
    __device__ __forceinline__ void run(const Fp8Args &a, const Fp8Rows &r, uint32_t nt, uint8_t *lds) {
        if (TM % 4 != 0 || r.rows > BM / 4 * 3)
            run_rows<TM>(a, r, nt, lds);
        else if (r.rows > BM / 2)
            run_rows<BM % 256 ? TM : TM / 4 * 3>(a, r, nt, lds);
        else if (r.rows > BM / 4)
            run_rows<TM % 4 ? TM : TM / 2>(a, r, nt, lds);
        else
            run_rows<TM % 4 ? TM : TM / 4>(a, r, nt, lds);
    }

    /* NI row tiles of each wave. */
    template <int NI>
    __device__ __forceinline__ void run_rows(const Fp8Args &a, const Fp8Rows &r, uint32_t nt, uint8_t *lds) {
        const uint32_t lane = threadIdx.x & 63u;
        const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        const uint32_t wm = wave / WN, wn = wave % WN;
        const uint32_t n0 = nt * (GATED ? BN / 2 : BN);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
        const uint32_t tail = a.k % kFp8Block; /* columns of a last, ragged block */

        /* sources of this lane's copies, from the tile's first row */
        constexpr int RX = NI * WM * 16, IX = RX >= 64 ? RX / 64 : 1; /* activation rows, copies of 8 per wave and step */
        static_assert(RX % 64 == 0 || 64 % RX == 0, "");
        uint32_t xo[IX], wo[IW];
        /* the 8 rows of copy i (fewer than 64 rows: several waves copy the same ones, so that every wave's count of copies is the same) */
        auto xr8 = [&](int i) { return RX >= 64 ? (wave * IX + i) * 8 : wave % (RX / 8) * 8; };
        const uint32_t xk = a.kb * kFp8Block;
        const uint8_t *xbase = r.list ? a.xq : a.xq + (uint64_t)r.m0 * xk;
        const uint8_t *wg = r.w + (uint64_t)n0 * a.k, *wu = wg + (uint64_t)a.n * a.k;
#pragma unroll
        for (int i = 0; i < IX; ++i) {
            const uint32_t row = xr8(i) + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u); /* the chunk at this lane's slot */
            const uint32_t in = row < r.rows ? row : r.rows - 1;
            xo[i] = (r.list ? r.list[r.m0 + in] : in) * xk + c * 16;
        }
#pragma unroll
        for (int i = 0; i < IW; ++i) {
            const uint32_t row = (wave * IW + i) * 8 + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u);
            uint32_t j = GATED && row >= BN / 2 ? row - BN / 2 : row;
            j = n0 + j < a.n ? j : a.n - 1 - n0;
            wo[i] = j * a.k + c * 16;
        }
        const float *sbase = r.list ? a.xs : a.xs + (uint64_t)r.m0 * a.kb;
        const uint32_t s64 = wave % (BM / 64) * 64, srow = s64 + lane, sin = srow < r.rows ? srow : r.rows - 1;
        const uint32_t so = (r.list ? r.list[r.m0 + sin] : sin) * a.kb * 4;
        /* this lane's chunk of an even and of an odd copy's row, in bytes.  Weight
         * chunks past the last column are filled from the block's first one of the
         * same row: they meet zeros of the activations, and where they hold a NaN
         * the row's outputs are NaN already. */
        const uint32_t ce = ((lane & 7u) ^ (lane >> 4)) * 16, co = ce ^ 64u;
        constexpr int kCopies = IX + IW + 1; /* of one wave and step */
        /* copies [C0, C1) of step kb into stage kb % 2 */
        auto issue = [&](uint32_t kb, auto C0, auto C1) {
            const uint32_t mask = fp8_copy_mask(kb, a.kb);
            const uint32_t k0 = kb * kFp8Block, at = lds0 + (kb & 1u) * kStage;
            const uint32_t cut = tail && kb + 1 == a.kb ? tail : kFp8Block;
            const uint32_t de = ce >= cut ? ce : 0u, dd = co >= cut ? co : 0u;
            fp8_for<C1.v - C0.v>([&](auto I) {
                constexpr int c = C0.v + I.v;
                if constexpr (c < IW) {
                    const uint32_t r8 = (wave * IW + c) * 8;
                    fp8_copy16(at + kX + r8 * 128, (GATED && r8 >= BN / 2 ? wu : wg) + k0, wo[c] - ((wave * IW + c) & 1u ? dd : de), mask);
                } else if constexpr (c < IW + IX) {
                    const uint32_t r8 = xr8(c - IW);
                    fp8_copy16(at + r8 * 128, xbase + k0, xo[c - IW], mask);
                } else {
                    fp8_copy4(at + kX + kW + s64 * 4, sbase + kb, so, mask);
                }
            });
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

        /* A step's copies go out a few with each row tile's products, from the
         * barrier that frees their stage on: all at once they would hold the
         * wave until the address unit has taken them (16 cycles each).  The
         * barrier stands before a step's last row tile, whose operands are in
         * registers by then: the next step's first operands are read while its
         * products run. */
        constexpr int kPer = (8 * kCopies + 5 * NI - 1) / (5 * NI);
        auto slot = [&](uint32_t kb, auto I) {
            constexpr int c0 = I.v * kPer < kCopies ? I.v * kPer : kCopies, c1 = c0 + kPer < kCopies ? c0 + kPer : kCopies;
            issue(kb, Fp8Int<c0>{}, Fp8Int<c1>{});
        };
        issue(0, Fp8Int<0>{}, Fp8Int<kCopies>{});
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        slot(1, Fp8Int<0>{});

        i32x8 w[TN];
        auto read_w = [&](const uint8_t *stage) {
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const uint32_t row = GATED ? (j >= NC ? BN / 2 : 0u) + (wn * NC + j % NC) * 16 : (wn * TN + j) * 16;
                w[j] = fp8_read_frag(stage + kX + row * 128, frag);
            }
        };
        const uint32_t xat = wm * 2048, sat = kX + kW + (wm * 16 + (lane & 15u)) * 4;
        read_w(lds);
        i32x8 x = fp8_read_frag(lds + xat, frag);
        float sx = *reinterpret_cast<const float *>(lds + sat);
        constexpr bool kCarry = NI % 2 == 0; /* the last row tile's sums are added in the next step */
        r9vx_f32x4 d[2][TN];
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < TN; ++j) d[1][j] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t kb = 0; kb < a.kb; ++kb) {
            if ((kb & 63u) == 0) {
                const uint32_t at = kb + lane < a.kb ? kb + lane : a.kb - 1;
                swg = in_n ? wsg[at] : 0.f;
                if constexpr (GATED) swu = wsu[at];
                /* waited for here: a wait in the step would be one for the copies too */
                asm volatile("" : "+v"(swg), "+v"(swu));
            }
            const uint8_t *here = lds + (kb & 1u) * kStage, *there = lds + ((kb & 1u) ^ 1u) * kStage;
            const float sg = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swg), (int)(kb & 63u)));
            const float su = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swu), (int)(kb & 63u)));
            fp8_for<NI>([&](auto Tile) {
                constexpr int i = Tile.v;
                i32x8 xn;
                float sn;
                if constexpr (i + 1 < NI) {
                    xn = fp8_read_frag(here + xat + (i + 1) * WM * 2048, frag);
                    sn = *reinterpret_cast<const float *>(here + sat + (i + 1) * WM * 64);
                    slot(kb + 1, Fp8Int<i + 1>{});
                } else {
                    /* the other stage has its data, and nobody reads this one any more */
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    xn = fp8_read_frag(there + xat, frag); /* after the last step: stale LDS, unused */
                    sn = *reinterpret_cast<const float *>(there + sat);
                    slot(kb + 2, Fp8Int<0>{});
                }
                const float t0 = sx * sg, t1 = GATED ? sx * su : 0.f;
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    d[i & 1][j] = fp8_mma<EXACT>(w[j], x);
                    if constexpr (kCarry || i > 0) fold(acc[i > 0 ? i - 1 : NI - 1], d[(i & 1) ^ 1], s0, s1, j);
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) { /* one product, four additions */
                    __builtin_amdgcn_sched_group_barrier(0x8, EXACT ? 4 : 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
                }
                s0 = t0;
                s1 = t1;
                x = xn;
                sx = sn;
                if constexpr (i + 1 == NI) {
                    __builtin_amdgcn_sched_barrier(0);
                    read_w(there);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (!kCarry) {
#pragma unroll
                for (int j = 0; j < TN; ++j) fold(acc[NI - 1], d[(NI - 1) & 1], s0, s1, j);
            }
        }
        if constexpr (kCarry) {
#pragma unroll
            for (int j = 0; j < TN; ++j) fold(acc[NI - 1], d[1], s0, s1, j);
        }
    }

    __device__ __forceinline__ void fold(r9vx_f32x4 (&o)[TN], const r9vx_f32x4 (&d)[TN], float s0, float s1, int j) {
        o[j] = fp8_add_scaled(o[j], d[j], GATED && j >= NC ? s1 : s0);
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
    __device__ __forceinline__ void drain(uint32_t rows, uint8_t *lds, Emit emit) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
        constexpr int TP = kPass / (WM * 16);
#pragma unroll
        for (int p = 0; p < TM / TP; ++p) {
            if (p * kPass >= rows) return;
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

/* ------------------------------------------------------------------ small tiles */

/* The same product for grids that do not fill the chip with large tiles: there
 * a step lasts as long as its barrier, LDS reads and copies take, whatever it
 * computes, so the steps are made fewer.  KS groups of WM x WN waves take one
 * K block each per step; their sums are joined in group order in LDS. */
template <int BM, int BN, int WM, int WN, int KS, bool GATED, bool EXACT>
struct Fp8Thin {
    static constexpr int TM = BM / 16 / WM, TN = BN / 16 / WN, NC = GATED ? TN / 2 : TN;
    static constexpr uint32_t kX = BM * 128, kW = BN * 128, kSub = kX + kW + BM * 4, kStage = KS * kSub, kLds = 2 * kStage;
    static constexpr int RX = BM / 64, RW = BN / 64, RS = KS * BM / 64; /* copies of a wave per block; scale copies of a step */
    static constexpr uint32_t kCols = GATED ? BN / 2 : BN;
    static_assert(WM * WN * KS == 8 && BM % 64 == 0 && BN % 64 == 0 && TM * 16 * WM == BM && TN * 16 * WN == BN, "");
    static_assert(128 % (GATED ? BN / 2 : BN) == 0 && kLds <= 160 * 1024 && KS * BM * BN * 4 <= (int)kLds && RS <= 8, "");

    r9vx_f32x4 acc[TM][TN];

    __device__ __forceinline__ void run(const Fp8Args &a, const Fp8Rows &r, uint32_t nt, uint8_t *lds) {
        const uint32_t lane = threadIdx.x & 63u;
        const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        const uint32_t kg = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
        const uint32_t n0 = nt * kCols;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
        const uint32_t tail = a.k % kFp8Block, xk = a.kb * kFp8Block;
        uint32_t xo[RX], wo[RW];
        const uint8_t *xbase = r.list ? a.xq : a.xq + (uint64_t)r.m0 * xk;
        const uint8_t *wg = r.w + (uint64_t)n0 * a.k, *wu = wg + (uint64_t)a.n * a.k;
        const uint32_t at8 = wave * 8 + (lane >> 3);       /* this lane's row of a copy round of 64 rows */
        const uint32_t c = (lane & 7u) ^ ((at8 >> 1) & 7u); /* and its chunk */
#pragma unroll
        for (int i = 0; i < RX; ++i) {
            const uint32_t row = i * 64 + at8, in = row < r.rows ? row : r.rows - 1;
            xo[i] = (r.list ? r.list[r.m0 + in] : in) * xk + c * 16;
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const uint32_t row = i * 64 + at8;
            uint32_t j = GATED && row >= BN / 2 ? row - BN / 2 : row;
            j = n0 + j < a.n ? j : a.n - 1 - n0;
            wo[i] = j * a.k + c * 16;
        }
        const float *sbase = r.list ? a.xs : a.xs + (uint64_t)r.m0 * a.kb;
        const uint32_t sq = wave % RS / RX, s64 = wave % RX * 64, srow = s64 + lane, sin = srow < r.rows ? srow : r.rows - 1;
        const uint32_t so = (r.list ? r.list[r.m0 + sin] : sin) * a.kb * 4;
        const uint32_t steps = (a.kb + KS - 1) / KS;
        auto issue = [&](uint32_t step, uint32_t st) {
            const uint32_t mask = fp8_copy_mask(step, steps);
            fp8_for<KS>([&](auto Q) {
                uint32_t kb = step * KS + Q.v;
                kb = kb < a.kb ? kb : a.kb - 1; /* blocks past the last: the last one, not added */
                const uint32_t k0 = kb * kFp8Block, at = lds0 + st * kStage + Q.v * kSub + wave * 1024;
                /* weight chunks past the last column: the block's first one of the row (it meets zeros) */
                const uint32_t back = tail && kb + 1 == a.kb && c * 16 >= tail ? c * 16 : 0u;
#pragma unroll
                for (int i = 0; i < RW; ++i) {
                    const bool up = GATED && (i * 64 + wave * 8) >= BN / 2;
                    fp8_copy16(at + kX + i * 8192, (up ? wu : wg) + k0, wo[i] - back, mask);
                }
#pragma unroll
                for (int i = 0; i < RX; ++i) fp8_copy16(at + i * 8192, xbase + k0, xo[i], mask);
            });
            uint32_t kb = step * KS + sq;
            kb = kb < a.kb ? kb : a.kb - 1;
            fp8_copy4(lds0 + st * kStage + sq * kSub + kX + kW + s64 * 4, sbase, so + kb * 4, mask);
        };
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = r9vx_f32x4{0.f, 0.f, 0.f, 0.f};
        const uint32_t frag = (lane & 15u) * 128 + (((lane >> 4) ^ ((lane >> 1) & 7u)) << 4);
        const float *wsg = r.ws + (uint64_t)(n0 / kFp8Block) * a.kb, *wsu = wsg + (uint64_t)a.nb * a.kb;
        float swg = 0.f, swu = 0.f; /* lane i: the scales of this group's block in step 64 (step / 64) + i */
        issue(0, 0);
        for (uint32_t step = 0; step < steps; ++step) {
            if ((step & 63u) == 0) {
                const uint32_t kb = (step + lane) * KS + kg;
                swg = wsg[kb < a.kb ? kb : a.kb - 1];
                if constexpr (GATED) swu = wsu[kb < a.kb ? kb : a.kb - 1];
                asm volatile("" : "+v"(swg), "+v"(swu));
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const uint8_t *sub = lds + (step & 1u) * kStage + kg * kSub;
            const float sg = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swg), (int)(step & 63u)));
            const float su = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, swu), (int)(step & 63u)));
            const bool mine = step * KS + kg < a.kb;
            i32x8 w[TN], x[TM];
            float sx[TM];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const uint32_t row = GATED ? (j >= NC ? BN / 2 : 0u) + (wn * NC + j % NC) * 16 : (wn * TN + j) * 16;
                w[j] = fp8_read_frag(sub + kX + row * 128, frag);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                x[i] = fp8_read_frag(sub + (wm * TM + i) * 2048, frag);
                sx[i] = *reinterpret_cast<const float *>(sub + kX + kW + ((wm * TM + i) * 16 + (lane & 15u)) * 4);
            }
            __builtin_amdgcn_sched_barrier(0);
            issue(step + 1, (step & 1u) ^ 1u);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                r9vx_f32x4 d[TN];
                const float t0 = mine ? sx[i] * sg : 0.f, t1 = mine ? sx[i] * su : 0.f;
#pragma unroll
                for (int j = 0; j < TN; ++j) d[j] = fp8_mma<EXACT>(w[j], x[i]);
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = fp8_add_scaled(acc[i][j], d[j], GATED && j >= NC ? t1 : t0);
            }
        }
    }

    /* The groups' sums through LDS: store(tile row, n, four outputs) for every
     * quad inside the problem. */
    template <typename Store>
    __device__ __forceinline__ void drain(const Fp8Args &a, const Fp8Rows &r, uint32_t nt, uint8_t *lds, Store store) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, kg = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
        constexpr uint32_t kQuads = BN / 4, kTile = BM * BN * 4;
        auto at = [](uint32_t t, uint32_t quad) { return (t * kQuads + (quad ^ (t & 15u))) * 16; };
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const uint32_t col = GATED ? (j >= NC ? BN / 2 : 0u) + (wn * NC + j % NC) * 16 : (wn * TN + j) * 16;
                *reinterpret_cast<r9vx_f32x4 *>(lds + kg * kTile + at((wm * TM + i) * 16 + (lane & 15u), col / 4 + (lane >> 4))) = acc[i][j];
            }
        __syncthreads();
        auto sum = [&](uint32_t t, uint32_t quad) {
            r9vx_f32x4 v = *reinterpret_cast<const r9vx_f32x4 *>(lds + at(t, quad));
#pragma unroll
            for (int q = 1; q < KS; ++q) v = v + *reinterpret_cast<const r9vx_f32x4 *>(lds + q * kTile + at(t, quad));
            return v;
        };
        for (uint32_t o = threadIdx.x; o < BM * (kCols / 4); o += 512) {
            const uint32_t t = o / (kCols / 4), quad = o % (kCols / 4), n = nt * kCols + quad * 4;
            if (t >= r.rows || n >= a.n) continue;
            r9vx_f32x4 v = sum(t, quad);
            if constexpr (GATED) v = fp8_swiglu(v, sum(t, quad + BN / 8));
            store(t, n, v);
        }
    }
};

}  // namespace r9vx
#endif
#endif
