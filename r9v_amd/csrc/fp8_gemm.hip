/*
 * fp8_gemm.hip -- matrix products of e4m3 activations (one f32 scale per row
 * and 128 columns) with e4m3 weights (one per 128 x 128 block):
 *
 *   a[m, n] = sum_b xs[m, b] * ws[n / 128, b] * sum_{k in b} xq[m, k] * wq[n, k]
 *
 * A block's inner sum is one v_mfma_f32_16x16x128_f8f6f4 from zero; four FMAs
 * then add it, scaled, to the f32 accumulators.  The weights are the rows of
 * the matrix unit's tile and the activations its columns, so that a lane holds
 * four consecutive outputs n of one row m and one scale serves all four.
 *
 * Three kernels, chosen by the variant's bucket and sizes, never by the launch's m:
 *   stream  up to 32 rows: every wave streams weight rows straight into
 *           registers, the waves of a workgroup split K and join their sums in
 *           LDS.  Bound by the weights' way from memory, n / 32 workgroups of
 *           it: 1 x 4096 x 4096 f32 7.7 us (2.2 TB/s, 128 workgroups on 256 CUs),
 *           5 x 5120 x 2048 4.8 us, of which the launch is 2 (160 workgroups).
 *   thin    64-row tiles whose waves split K, for grids that do not fill the
 *           chip with large ones: 48 x (2 x 1408) x 2048 8.2 us (44 workgroups),
 *           517 x 2112 x 4096 f32 26 us (153)
 *   tile    256 x 256 tiles staged through LDS: 2048 x 14336 x 4096 bf16
 *           144 us, 1.67 PFLOP/s (448 tiles on 256 CUs: two rounds, of which an
 *           eighth is idle); the library's 8-bit product without block scales
 *           reaches 2.6 PFLOP/s at 8192 x 8192 x 8192.
 */
#include "r9vx_e4m3.h"
#include "r9vx_e4m3_gemm.h"

using namespace r9vx;

namespace {

template <int MT, int NT, int W, int XT, bool GATED>
__global__ __launch_bounds__(W * 64) void fp8_stream_kernel(Fp8Args a) {
    __shared__ __attribute__((aligned(16))) r9vx_f32x4 part[W * NT * MT * 64];
    extern __shared__ __attribute__((aligned(16))) uint8_t quantized[];
    const uint32_t strip = blockIdx.x, m0 = blockIdx.y * (MT * 16);
    Fp8Rows r{};
    r.w = a.w;
    r.ws = a.ws;
    r.m0 = m0;
    r.rows = a.m - m0 < MT * 16u ? a.m - m0 : MT * 16u;
    fp8_stream<MT, NT, W, XT, GATED>(a, r, strip, part, quantized, [] {}, [&](uint32_t row, uint32_t n, r9vx_f32x4 v) {
        fp8_store_dense(a, m0 + row, n, v);
    });
}

template <int BM, int BN, int WM, bool GATED, bool EXACT>
__global__ __launch_bounds__(512) void fp8_tile_kernel(Fp8Args a) {
    typedef Fp8Tile<BM, BN, WM, GATED, EXACT> T;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLds];
    /* consecutive workgroups go to the 8 XCDs in turn: each XCD takes one run
     * of the tile list, row tiles of one column tile first, so that a column
     * tile's weights are read into one L2 */
    const uint32_t tiles = a.m_tiles * a.n_tiles, x = blockIdx.x & 7u, i = blockIdx.x >> 3;
    const uint32_t q = tiles >> 3, rem = tiles & 7u;
    const uint32_t at = x * q + (x < rem ? x : rem) + i;
    const uint32_t nt = at / a.m_tiles, mt = at - nt * a.m_tiles;
    Fp8Rows r{};
    r.w = a.w;
    r.ws = a.ws;
    r.m0 = mt * BM;
    r.rows = a.m - r.m0 < (uint32_t)BM ? a.m - r.m0 : (uint32_t)BM;
    T t;
    t.run(a, r, nt, lds);
    t.drain(r.rows, lds, [&](uint32_t t0) {
        for (uint32_t o = threadIdx.x; o < T::kPass * (T::kCols / 4); o += 512) {
            const uint32_t row = o / (T::kCols / 4), quad = o % (T::kCols / 4), n = nt * T::kCols + quad * 4;
            if (t0 + row < r.rows && n < a.n) fp8_store_dense(a, r.m0 + t0 + row, n, *reinterpret_cast<const r9vx_f32x4 *>(lds + T::at(row, quad)));
        }
    });
}

template <int BM, int BN, int WM, int WN, int KS, bool GATED, bool EXACT>
__global__ __launch_bounds__(512) void fp8_thin_kernel(Fp8Args a) {
    typedef Fp8Thin<BM, BN, WM, WN, KS, GATED, EXACT> T;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLds];
    const uint32_t tiles = a.m_tiles * a.n_tiles, x = blockIdx.x & 7u, i = blockIdx.x >> 3, q = tiles >> 3, rem = tiles & 7u;
    const uint32_t at = x * q + (x < rem ? x : rem) + i, nt = at / a.m_tiles, mt = at - nt * a.m_tiles;
    Fp8Rows r{};
    r.w = a.w;
    r.ws = a.ws;
    r.m0 = mt * BM;
    r.rows = a.m - r.m0 < (uint32_t)BM ? a.m - r.m0 : (uint32_t)BM;
    T t;
    t.run(a, r, nt, lds);
    t.drain(a, r, nt, lds, [&](uint32_t row, uint32_t n, r9vx_f32x4 v) { fp8_store_dense(a, r.m0 + row, n, v); });
}

Fp8Args fp8_args(const r9vx_fp8_problem &p, const uint8_t *xq, const float *xs) {
    Fp8Args a{};
    a.w = p.w;
    a.ws = p.w_scales;
    a.x = p.x;
    a.xq = xq;
    a.xs = xs;
    a.bias = p.bias;
    a.residual = p.residual;
    a.y = p.y;
    a.m = p.m;
    a.n = p.n;
    a.k = p.k;
    a.kb = r9vx_fp8_kb(p.k);
    a.nb = r9vx_fp8_kb(p.n);
    a.y_bf16 = p.y_dtype == R9VX_DTYPE_BF16;
    a.epilogue = p.epilogue;
    return a;
}

template <int MT, int NT, int W, int XT>
int launch_stream(const Fp8Args &a, bool gated, hipStream_t s) {
    const uint32_t cols = gated ? NT * 8 : NT * 16;
    const dim3 grid((a.n + cols - 1) / cols, (a.m + MT * 16 - 1) / (MT * 16));
    const uint32_t lds = XT == kFp8Codes ? 0 : fp8_lds_rows_bytes(a.m < MT * 16 ? a.m : MT * 16, a.kb);
    if (gated)
        hipLaunchKernelGGL((fp8_stream_kernel<MT, NT, W, XT, true>), grid, dim3(W * 64), lds, s, a);
    else
        hipLaunchKernelGGL((fp8_stream_kernel<MT, NT, W, XT, false>), grid, dim3(W * 64), lds, s, a);
    return (int)hipGetLastError();
}

template <int BM, int BN, int WM, bool EXACT>
int launch_tile(Fp8Args a, bool gated, hipStream_t s) {
    const uint32_t cols = gated ? BN / 2 : BN;
    a.m_tiles = (a.m + BM - 1) / BM;
    a.n_tiles = (a.n + cols - 1) / cols;
    const dim3 grid(a.m_tiles * a.n_tiles);
    if (gated)
        hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, true, EXACT>), grid, dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, false, EXACT>), grid, dim3(512), 0, s, a);
    return (int)hipGetLastError();
}

template <int BM, int BN, int WM, int WN, int KS, bool EXACT>
int launch_thin(Fp8Args a, bool gated, hipStream_t s) {
    const uint32_t cols = gated ? BN / 2 : BN;
    a.m_tiles = (a.m + BM - 1) / BM;
    a.n_tiles = (a.n + cols - 1) / cols;
    const dim3 grid(a.m_tiles * a.n_tiles);
    if (gated)
        hipLaunchKernelGGL((fp8_thin_kernel<BM, BN, WM, WN, KS, true, EXACT>), grid, dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((fp8_thin_kernel<BM, BN, WM, WN, KS, false, EXACT>), grid, dim3(512), 0, s, a);
    return (int)hipGetLastError();
}

/* The kernels for more than 32 rows, each with its time in ns as measured
 * (n = 2112 .. 14336, K = 2048 .. 8192): a workgroup's start and end, and per K
 * block; `slots` workgroups run beside each other before a round is full.
 * EXACT = false / true:
 *   256 x 256 (EXACT 128 x 256)  4096 x 4096 x 4096  75 / 132 us
 *   64 x 128                     1024 x 4096 x 4096  33 / 44
 *   64 x 128, 2 blocks a step     517 x 2112 x 4096  19 / 23
 *   64 x 64, 4 blocks a step      256 x 4096 x 4096  12 / 15 */
template <bool EXACT>
int launch_many(const Fp8Args &a, uint32_t m_bucket, bool gated, hipStream_t s) {
    static constexpr struct {
        uint32_t bm, bn, slots, start, block, start_x, block_x;
    } kShapes[4] = {{EXACT ? 128 : 256, 256, 256, 17000, 1790, 12000, 1900},
                    {64, 128, 512, 4000, 900, 4000, 1250},
                    {64, 128, 256, 4000, 440, 4000, 590},
                    {64, 64, 256, 4000, 260, 4000, 330}};
    const uint64_t n = gated ? 2ull * a.n : a.n;
    uint32_t best = 0;
    uint64_t least = ~0ull;
    for (uint32_t i = 0; i < 4; ++i) {
        const auto &k = kShapes[i];
        const uint64_t tiles = ((m_bucket + k.bm - 1) / k.bm) * ((n + k.bn - 1) / k.bn);
        if (tiles * 512 >> 32) continue; /* a launch's threads: 32 bits; the large tiles' outputs would not fit the card first */
        const uint64_t block = EXACT ? k.block_x : k.block, start = EXACT ? k.start_x : k.start;
        /* half a round of the 64 x 128 tiles, which share a CU, is two thirds as long as a whole one */
        const uint64_t rounds = (tiles + k.slots - 1) / k.slots;
        const uint64_t ns = rounds * start + (i == 1 && tiles <= k.slots / 2 ? block * 2 / 3 : rounds * block) * a.kb;
        if (ns < least) least = ns, best = i;
    }
    switch (best) {
    case 0: return launch_tile<EXACT ? 128 : 256, 256, 2, EXACT>(a, gated, s);
    case 1: return launch_tile<64, 128, 2, EXACT>(a, gated, s);
    case 2: return launch_thin<64, 128, 2, 2, 2, EXACT>(a, gated, s);
    default: return launch_thin<64, 64, 2, 1, 4, EXACT>(a, gated, s);
    }
}

}  // namespace

/* The activations' codes in rows of whole blocks, then (in-call quantization)
 * their scales.  Codes that come in such rows are read where they are. */
static size_t fp8_codes_bytes(uint32_t m_bucket, uint32_t k) {
    return ((size_t)m_bucket * r9vx_fp8_kb(k) * kFp8Block + 255) & ~(size_t)255;
}
/* Few activations: each workgroup quantizes them into its LDS beside its first
 * weights' way from memory, which costs less than a launch of its own for them
 * (and a workspace): 1 x 4096 x 4096, from Python, 13.0 / 8.7 us. */
static bool fp8_in_lds(uint32_t m_bucket, uint32_t k, uint32_t x_dtype) {
    return x_dtype != R9VX_DTYPE_E4M3 && m_bucket <= 16 && fp8_fits_lds(m_bucket, r9vx_fp8_kb(k));
}
size_t r9vx_fp8_workspace_bytes(uint32_t m_bucket, uint32_t k, uint32_t x_dtype) {
    if (fp8_in_lds(m_bucket, k, x_dtype)) return 0;
    if (x_dtype == R9VX_DTYPE_E4M3) return k % kFp8Block ? fp8_codes_bytes(m_bucket, k) : 0;
    return fp8_codes_bytes(m_bucket, k) + (size_t)m_bucket * r9vx_fp8_kb(k) * 4;
}

int r9vx_launch_matmul_fp8(const r9vx_fp8_problem &p, hipStream_t stream) {
    const uint8_t *xq = static_cast<const uint8_t *>(p.x);
    const float *xs = p.x_scales;
    const bool gated = p.epilogue == R9VX_EPILOGUE_SWIGLU;
    if (fp8_in_lds(p.m_bucket, p.k, p.x_dtype)) {
        const Fp8Args a = fp8_args(p, nullptr, nullptr);
        return p.x_dtype == R9VX_DTYPE_F32 ? launch_stream<1, 2, 8, kFp8F32>(a, gated, stream) : launch_stream<1, 2, 8, kFp8Bf16>(a, gated, stream);
    }
    if (p.x_dtype != R9VX_DTYPE_E4M3) {
        float *s = reinterpret_cast<float *>(p.workspace + fp8_codes_bytes(p.m_bucket, p.k));
        const int rc = r9vx_launch_quantize_fp8(p.x, p.x_dtype, p.m, p.k, r9vx_fp8_kb(p.k) * kFp8Block, p.workspace, s, stream);
        if (rc) return rc;
        xq = p.workspace;
        xs = s;
    } else if (p.k % kFp8Block) {
        const int rc = r9vx_launch_pad_fp8(xq, p.m, p.k, p.workspace, stream);
        if (rc) return rc;
        xq = p.workspace;
    }
    const Fp8Args a = fp8_args(p, xq, xs);
    /* Four tiles of 16 rows in the streaming kernel against 64 x 64 tiles, 48 rows,
     * weights from HBM: 2 x 1408 x 2048 9.8 / 8.0 us, 2112 x 4096 16.8 / 12.8,
     * 14336 x 4096 34.2 / 20.5, 7168 x 7168 27.0 / 30.1; two tiles, 32 rows:
     * 7.7 / 7.8, 11.9 / 11.9, 24.9 / 18.8, 20.6 / 27.3; 17 rows: 6.7 / 7.4,
     * 9.7 / 11.0, 21.0 / 18.8, 16.7 / 25.3.  The line is drawn by rows alone, where
     * most of these sizes cross; of them it costs 24.9 instead of 18.8 us (32 rows of
     * the widest) and 30.1 instead of 27.0 (48 of the square one). */
    if (p.m_bucket <= 16) return launch_stream<1, 2, 8, kFp8Codes>(a, gated, stream);
    if (p.m_bucket <= 32) return launch_stream<2, 2, 8, kFp8Codes>(a, gated, stream);
    return p.y_dtype == R9VX_DTYPE_F32 ? launch_many<true>(a, p.m_bucket, gated, stream) : launch_many<false>(a, p.m_bucket, gated, stream);
}
