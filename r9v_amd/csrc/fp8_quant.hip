/*
 * fp8_quant.hip -- activations to e4m3 with one f32 scale per row and 128
 * columns.
 *
 *   s[m, b] = max(max |x[m, 128 b ..]| / 448, 2^-126)      (f32)
 *   q[m, k] = e4m3, nearest-even, of the exact x[m, k] / s[m, k / 128]
 *
 * One pass: eight lanes hold a block in registers, sixteen values each, take
 * its maximum by three cross-lane steps and write codes and scale.  Bound by
 * memory: 3 bytes (bf16) or 5 (f32) per value.  8192 x 4096 bf16: 21 us, 4.9
 * TB/s (a 4 GiB copy reaches 4.7); 5 x 2048: 2.4 us, a launch.
 */
#include "r9vx_e4m3.h"

using namespace r9vx;

namespace {

template <bool F32>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const void *__restrict__ x, uint32_t blocks, uint32_t k, uint32_t kb,
                                                           uint32_t ldq, uint8_t *__restrict__ q, float *__restrict__ scales) {
    const uint32_t blk = blockIdx.x * 32 + (threadIdx.x >> 3);
    if (blk >= blocks) return; /* whole groups of eight lanes */
    const uint32_t part = threadIdx.x & 7u;
    const uint32_t row = blk / kb, b = blk - row * kb;
    const uint32_t left = k - b * kFp8Block; /* columns from the block's first; k is a multiple of 16 */
    const uint64_t at = (uint64_t)row * k + b * kFp8Block, to = (uint64_t)row * ldq + b * kFp8Block;
    const uint32_t room = ldq - b * kFp8Block; /* code columns: k's, or with zeros behind them to the end of the block */
    Fp8Block<F32> block;
    block.load(static_cast<const uint8_t *>(x) + at * (F32 ? 4 : 2), left, part);
    uint32_t code[4];
    const float s = block.codes(code);
#pragma unroll
    for (int j = 0; j < block.N; ++j) {
        const uint32_t c = block.column(j, part);
        if constexpr (F32) {
            if (c < room) *reinterpret_cast<uint32_t *>(q + to + c) = c < left ? code[j] : 0u;
        } else {
            if (c < room) *reinterpret_cast<r9vx_u32x2 *>(q + to + c) = c < left ? r9vx_u32x2{code[2 * j], code[2 * j + 1]} : r9vx_u32x2{0u, 0u};
        }
    }
    if (part == 0) scales[blk] = s;
}

/* Rows of k codes to rows of whole blocks, zeros behind them. */
__global__ __launch_bounds__(256) void pad_fp8_kernel(const r9vx_u32x4 *__restrict__ x, uint64_t n, uint32_t k16, uint32_t ld16,
                                                      r9vx_u32x4 *__restrict__ q) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint64_t row = i / ld16;
    const uint32_t c = (uint32_t)(i - row * ld16);
    q[i] = c < k16 ? x[row * k16 + c] : r9vx_u32x4{0u, 0u, 0u, 0u};
}

}  // namespace

/* A launch's threads are counted in 32 bits: rows beyond this many go through
 * a further one. */
static constexpr uint32_t kLaunchThreads = 1u << 31;

int r9vx_launch_pad_fp8(const uint8_t *x, uint32_t m, uint32_t k, uint8_t *q, hipStream_t stream) {
    const uint32_t ld16 = r9vx_fp8_kb(k) * (kFp8Block / 16);
    const uint32_t rows = kLaunchThreads / ld16;
    for (uint32_t r0 = 0; r0 < m; r0 += rows) {
        const uint64_t n = (uint64_t)(m - r0 < rows ? m - r0 : rows) * ld16;
        hipLaunchKernelGGL(pad_fp8_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream,
                           reinterpret_cast<const r9vx_u32x4 *>(x) + (uint64_t)r0 * (k / 16), n, k / 16, ld16,
                           reinterpret_cast<r9vx_u32x4 *>(q) + (uint64_t)r0 * ld16);
        const int e = (int)hipGetLastError();
        if (e) return e;
    }
    return 0;
}

int r9vx_launch_quantize_fp8(const void *x, uint32_t x_dtype, uint64_t m, uint32_t k, uint32_t ldq, uint8_t *q, float *scales,
                             hipStream_t stream) {
    const uint32_t kb = r9vx_fp8_kb(k);
    const uint64_t rows = kLaunchThreads / 8 / kb; /* eight threads a block */
    for (uint64_t r0 = 0; r0 < m; r0 += rows) {
        const uint32_t n = (uint32_t)((m - r0 < rows ? m - r0 : rows) * kb);
        const dim3 grid((n + 31) / 32);
        if (x_dtype == R9VX_DTYPE_F32)
            hipLaunchKernelGGL(quantize_fp8_kernel<true>, grid, dim3(256), 0, stream, static_cast<const float *>(x) + r0 * k, n, k, kb, ldq,
                               q + r0 * ldq, scales + r0 * kb);
        else
            hipLaunchKernelGGL(quantize_fp8_kernel<false>, grid, dim3(256), 0, stream, static_cast<const uint16_t *>(x) + r0 * k, n, k, kb, ldq,
                               q + r0 * ldq, scales + r0 * kb);
        const int e = (int)hipGetLastError();
        if (e) return e;
    }
    return 0;
}
