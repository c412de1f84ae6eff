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
 * Two kernels, chosen by the variant's bucket and sizes, never by the launch's m:
 *   stream  few rows: every wave streams weight rows straight into registers,
 *           the waves of a workgroup split K and join their sums in LDS
 *   tile    many rows: 256-column tiles staged through LDS
 */
#include "r9vx_e4m3.h"
#include "r9vx_e4m3_gemm.h"

using namespace r9vx;

namespace {

template <int MT, int NT, int W, int XT, bool GATED>
__global__ __launch_bounds__(W * 64) void fp8_stream_kernel(Fp8Args a) {
    __shared__ __attribute__((aligned(16))) r9vx_f32x4 part[W * NT * MT * 64];
    const uint32_t strip = blockIdx.x, m0 = blockIdx.y * (MT * 16);
    Fp8Rows r{};
    r.w = a.w;
    r.ws = a.ws;
    r.m0 = m0;
    r.rows = a.m - m0 < MT * 16u ? a.m - m0 : MT * 16u;
    fp8_stream<MT, NT, W, XT, GATED>(a, r, strip, part, [&](uint32_t row, uint32_t n, r9vx_f32x4 v) {
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
    if (r.rows > BM - 16)
        t.template run<true>(a, r, nt, lds);
    else
        t.template run<false>(a, r, nt, lds);
    t.drain(lds, [&](uint32_t t0) {
        for (uint32_t o = threadIdx.x; o < T::kPass * (T::kCols / 4); o += 512) {
            const uint32_t row = o / (T::kCols / 4), quad = o % (T::kCols / 4), n = nt * T::kCols + quad * 4;
            if (t0 + row < r.rows && n < a.n) fp8_store_dense(a, r.m0 + t0 + row, n, *reinterpret_cast<const r9vx_f32x4 *>(lds + T::at(row, quad)));
        }
    });
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

template <int MT, int NT, int W>
int launch_stream(const Fp8Args &a, bool gated, hipStream_t s) {
    const uint32_t cols = gated ? NT * 8 : NT * 16;
    const dim3 grid((a.n + cols - 1) / cols, (a.m + MT * 16 - 1) / (MT * 16));
    if (gated)
        hipLaunchKernelGGL((fp8_stream_kernel<MT, NT, W, 0, true>), grid, dim3(W * 64), 0, s, a);
    else
        hipLaunchKernelGGL((fp8_stream_kernel<MT, NT, W, 0, false>), grid, dim3(W * 64), 0, s, a);
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

}  // namespace

/* The codes, then the scales, of in-call quantization. */
size_t r9vx_fp8_workspace_bytes(uint32_t m_bucket, uint32_t k, uint32_t n, uint32_t x_dtype, uint32_t epilogue) {
    if (x_dtype == R9VX_DTYPE_E4M3) return 0;
    return (((size_t)m_bucket * k + 255) & ~(size_t)255) + (size_t)m_bucket * r9vx_fp8_kb(k) * 4;
}

int r9vx_launch_matmul_fp8(const r9vx_fp8_problem &p, hipStream_t stream) {
    const uint8_t *xq = static_cast<const uint8_t *>(p.x);
    const float *xs = p.x_scales;
    if (p.x_dtype != R9VX_DTYPE_E4M3) {
        float *s = reinterpret_cast<float *>(p.workspace + (((size_t)p.m_bucket * p.k + 255) & ~(size_t)255));
        const int rc = r9vx_launch_quantize_fp8(p.x, p.x_dtype, p.m, p.k, p.workspace, s, stream);
        if (rc) return rc;
        xq = p.workspace;
        xs = s;
    }
    const Fp8Args a = fp8_args(p, xq, xs);
    const bool gated = p.epilogue == R9VX_EPILOGUE_SWIGLU;
    if (p.m_bucket <= 16) return launch_stream<1, 2, 8>(a, gated, stream);
    if (p.m_bucket <= 32) return launch_stream<2, 2, 8>(a, gated, stream);
    if (p.m_bucket <= 64) return launch_stream<4, 2, 8>(a, gated, stream);
    if (p.y_dtype == R9VX_DTYPE_F32) return launch_tile<128, 256, 2, true>(a, gated, stream);
    return launch_tile<256, 256, 2, false>(a, gated, stream);
}
