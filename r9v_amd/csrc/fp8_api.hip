/*
 * fp8_api.hip -- the C ABI of include/r9vx_fp8.h: every problem of a call is
 * reported and nothing is enqueued when any is found.
 */
#include "r9vx_e4m3.h"
#include "r9vx_host.h"

namespace {

bool float_dtype(uint32_t d) { return d == R9VX_DTYPE_F32 || d == R9VX_DTYPE_BF16; }

void check_k(uint32_t k, Problems &pr) {
    if (k == 0 || k % 16) pr.add(R9VX_ERR_INVALID, "k=%u must be a positive multiple of 16", k);
    else if (k > (1u << 20)) pr.add(R9VX_ERR_UNSUPPORTED, "k=%u exceeds 2^20", k); /* 256 rows are addressed by 32 bits */
}

uint64_t scale_blocks(uint32_t n, uint32_t k) { return (uint64_t)r9vx_fp8_kb(n) * r9vx_fp8_kb(k); }

uint64_t float_bytes(uint32_t d) { return d == R9VX_DTYPE_F32 ? 4 : 2; }

}  // namespace

extern "C" {

int r9vx_quantize_fp8_launch(const r9vx_quantize_fp8_args *a, r9vx_stream_t stream) {
    Problems pr;
    if (!a) {
        pr.add(R9VX_ERR_NULL, "args must be non-NULL");
        return pr.finish("quantize_fp8");
    }
    check_k(a->k, pr);
    if (!float_dtype(a->in_dtype)) pr.add(R9VX_ERR_UNSUPPORTED, "in_dtype %u: only f32 and bf16 are quantized", a->in_dtype);
    if (a->m > (1ull << 40)) pr.add(R9VX_ERR_INVALID, "m=%llu exceeds 2^40", (unsigned long long)a->m);
    if (a->m && (!a->x || !a->q || !a->scales)) pr.add(R9VX_ERR_NULL, "x, q and scales are required");
    if (!aligned16(a->x) || !aligned16(a->q)) pr.add(R9VX_ERR_ALIGN, "x and q must be 16-byte aligned");
    if ((uintptr_t)a->scales & 3u) pr.add(R9VX_ERR_ALIGN, "scales must be 4-byte aligned");
    if (pr.code == R9VX_OK && a->m) {
        const uint64_t nx = a->m * a->k * (a->in_dtype == R9VX_DTYPE_F32 ? 4 : 2), nq = a->m * a->k,
                       ns = a->m * r9vx_fp8_kb(a->k) * 4;
        if (overlap(a->x, nx, a->q, nq) || overlap(a->x, nx, a->scales, ns) || overlap(a->q, nq, a->scales, ns))
            pr.add(R9VX_ERR_INVALID, "x, q and scales must not overlap");
    }
    const int rc = pr.finish("quantize_fp8");
    if (rc || a->m == 0) return rc;
    return hip_status("quantize_fp8", r9vx_launch_quantize_fp8(a->x, a->in_dtype, a->m, a->k, a->k, a->q, a->scales,
                                                               reinterpret_cast<hipStream_t>(stream)));
}

static void check_matmul_fp8_static(const r9vx_matmul_fp8_static *st, Problems &pr) {
    check_k(st->k, pr);
    if (st->n == 0) pr.add(R9VX_ERR_INVALID, "n must be positive");
    if (st->n > (1u << 26)) pr.add(R9VX_ERR_UNSUPPORTED, "n=%u exceeds 2^26", st->n); /* a launch's threads: 32 bits */
    if (st->m_bucket > (1u << 24)) pr.add(R9VX_ERR_UNSUPPORTED, "m_bucket=%u exceeds 2^24", st->m_bucket);
    if (!float_dtype(st->in_dtype) && st->in_dtype != R9VX_DTYPE_E4M3)
        pr.add(R9VX_ERR_UNSUPPORTED, "in_dtype %u: only f32, bf16 and e4m3 activations", st->in_dtype);
    if (!float_dtype(st->out_dtype)) pr.add(R9VX_ERR_UNSUPPORTED, "out_dtype %u: only f32 and bf16 outputs", st->out_dtype);
    if (st->epilogue > R9VX_EPILOGUE_SWIGLU)
        pr.add(R9VX_ERR_UNSUPPORTED, "epilogue %u: only none/bias/residual/swiglu", st->epilogue);
}

static bool matmul_fp8_static_ok(const r9vx_matmul_fp8_static *st) {
    if (!st) return false;
    Problems pr;
    check_matmul_fp8_static(st, pr);
    return pr.code == R9VX_OK;
}

size_t r9vx_matmul_fp8_workspace_bytes(const r9vx_matmul_fp8_static *st) {
    return matmul_fp8_static_ok(st) ? r9vx_fp8_workspace_bytes(st->m_bucket, st->k, st->in_dtype) : 0;
}

uint64_t r9vx_matmul_fp8_static_bytes(const r9vx_matmul_fp8_static *st, uint32_t m) {
    if (!matmul_fp8_static_ok(st)) return 0;
    const uint64_t pair = st->epilogue == R9VX_EPILOGUE_SWIGLU ? 2 : 1;
    const uint64_t x = st->in_dtype == R9VX_DTYPE_E4M3 ? (uint64_t)m * (st->k + 4ull * r9vx_fp8_kb(st->k))
                                                       : (uint64_t)m * st->k * (st->in_dtype == R9VX_DTYPE_F32 ? 4 : 2);
    return pair * ((uint64_t)st->n * st->k + 4 * scale_blocks(st->n, st->k)) + x +
           (uint64_t)m * st->n * (st->out_dtype == R9VX_DTYPE_F32 ? 4 : 2);
}

uint64_t r9vx_matmul_fp8_static_flops(const r9vx_matmul_fp8_static *st, uint32_t m) {
    if (!matmul_fp8_static_ok(st)) return 0;
    return (st->epilogue == R9VX_EPILOGUE_SWIGLU ? 4ull : 2ull) * m * st->n * st->k;
}

int r9vx_matmul_fp8_launch(const r9vx_matmul_fp8_static *st, const r9vx_matmul_fp8_args *a, r9vx_stream_t stream) {
    Problems pr;
    if (!st || !a) {
        pr.add(R9VX_ERR_NULL, "static and args must be non-NULL");
        return pr.finish("matmul_fp8");
    }
    check_matmul_fp8_static(st, pr);
    if (a->m > st->m_bucket) pr.add(R9VX_ERR_INVALID, "m=%u exceeds m_bucket=%u", a->m, st->m_bucket);
    const bool codes = st->in_dtype == R9VX_DTYPE_E4M3;
    if (a->m > 0) {
        if (!a->w || !a->w_scales) pr.add(R9VX_ERR_NULL, "w and w_scales are required");
        if (!a->x) pr.add(R9VX_ERR_NULL, "x is NULL");
        if (!a->y) pr.add(R9VX_ERR_NULL, "y is NULL");
        if (codes && !a->x_scales) pr.add(R9VX_ERR_NULL, "e4m3 activations without x_scales");
    }
    if (!codes && a->x_scales) pr.add(R9VX_ERR_INVALID, "x_scales given with activations that are quantized within the launch");
    if (st->epilogue == R9VX_EPILOGUE_BIAS && a->m > 0 && !a->bias) pr.add(R9VX_ERR_NULL, "bias epilogue without bias");
    if (st->epilogue != R9VX_EPILOGUE_BIAS && a->bias) pr.add(R9VX_ERR_INVALID, "bias given without bias epilogue");
    if (st->epilogue == R9VX_EPILOGUE_RESIDUAL && a->m > 0 && !a->residual)
        pr.add(R9VX_ERR_NULL, "residual epilogue without residual");
    if (st->epilogue != R9VX_EPILOGUE_RESIDUAL && a->residual)
        pr.add(R9VX_ERR_INVALID, "residual given without residual epilogue");
    if (!aligned16(a->w) || !aligned16(a->x) || !aligned16(a->y) || !aligned16(a->bias) || !aligned16(a->residual))
        pr.add(R9VX_ERR_ALIGN, "w, x, y, bias and residual must be 16-byte aligned");
    if (((uintptr_t)a->w_scales | (uintptr_t)a->x_scales) & 3u) pr.add(R9VX_ERR_ALIGN, "scales must be 4-byte aligned");
    const size_t ws = r9vx_matmul_fp8_workspace_bytes(st);
    if (ws && a->m > 0 && !a->workspace)
        pr.add(R9VX_ERR_WORKSPACE, "workspace of r9vx_matmul_fp8_workspace_bytes (%zu) required", ws);
    if ((uintptr_t)a->workspace & 255u) pr.add(R9VX_ERR_ALIGN, "workspace must be 256-byte aligned");
    if (pr.code == R9VX_OK && a->m) {
        /* workgroups read operands while others store their outputs */
        const uint64_t m = a->m, ny = m * st->n * float_bytes(st->out_dtype), nx = m * st->k * (codes ? 1 : float_bytes(st->in_dtype)),
                       nxs = m * r9vx_fp8_kb(st->k) * 4, pair = st->epilogue == R9VX_EPILOGUE_SWIGLU ? 2 : 1;
        const bool in_place = a->residual == a->y && st->out_dtype == R9VX_DTYPE_F32;
        if (overlap(a->y, ny, a->x, nx) || overlap(a->y, ny, a->x_scales, nxs) || overlap(a->y, ny, a->w, pair * st->n * st->k) ||
            overlap(a->y, ny, a->w_scales, pair * scale_blocks(st->n, st->k) * 4) || overlap(a->y, ny, a->bias, 4ull * st->n) ||
            (!in_place && overlap(a->y, ny, a->residual, m * st->n * 4)))
            pr.add(R9VX_ERR_INVALID, "y must not overlap an operand (an f32 y may be the residual)");
        if (overlap(a->workspace, ws, a->x, nx) || overlap(a->workspace, ws, a->x_scales, nxs) || overlap(a->workspace, ws, a->y, ny))
            pr.add(R9VX_ERR_INVALID, "the workspace must not overlap x, x_scales or y");
    }
    const int rc = pr.finish("matmul_fp8");
    if (rc || a->m == 0) return rc;
    r9vx_fp8_problem p{};
    p.w = a->w;
    p.w_scales = a->w_scales;
    p.x = a->x;
    p.x_scales = a->x_scales;
    p.bias = a->bias;
    p.residual = a->residual;
    p.y = a->y;
    p.workspace = a->workspace;
    p.m = a->m;
    p.m_bucket = st->m_bucket;
    p.n = st->n;
    p.k = st->k;
    p.x_dtype = st->in_dtype;
    p.y_dtype = st->out_dtype;
    p.epilogue = st->epilogue;
    return hip_status("matmul_fp8", r9vx_launch_matmul_fp8(p, reinterpret_cast<hipStream_t>(stream)));
}

static r9vx_moe_fp8_problem moe_fp8_problem(const r9vx_moe_ffn_fp8_static *st) {
    r9vx_moe_fp8_problem p{};
    p.t_bucket = st->t_bucket;
    p.e = st->e_local;
    p.k = st->k_topk;
    p.dm = st->dm;
    p.dff = st->dff;
    p.shared = st->shared_experts;
    p.y_dtype = st->out_dtype;
    return p;
}

static void check_moe_fp8_static(const r9vx_moe_ffn_fp8_static *st, Problems &pr) {
    if (st->e_local == 0) pr.add(R9VX_ERR_INVALID, "E must be > 0");
    if (st->e_local > 1024) pr.add(R9VX_ERR_UNSUPPORTED, "E=%u exceeds 1024", st->e_local);
    if (st->k_topk == 0) pr.add(R9VX_ERR_INVALID, "top-k must be > 0");
    if (st->k_topk > 32) pr.add(R9VX_ERR_UNSUPPORTED, "top-k %u exceeds 32", st->k_topk);
    if (st->dm == 0 || st->dm % kFp8Block) pr.add(R9VX_ERR_INVALID, "dm=%u must be a positive multiple of 128", st->dm);
    if (st->dff == 0 || st->dff % kFp8Block) pr.add(R9VX_ERR_INVALID, "dff=%u must be a positive multiple of 128", st->dff);
    if (st->dm > (1u << 16) || st->dff > (1u << 16)) pr.add(R9VX_ERR_UNSUPPORTED, "dm=%u or dff=%u exceeds 2^16", st->dm, st->dff);
    if (st->t_bucket > (1u << 23)) pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u exceeds 2^23", st->t_bucket); /* a launch's threads: 32 bits */
    if (st->shared_experts > 64) pr.add(R9VX_ERR_UNSUPPORTED, "%u shared experts exceed 64", st->shared_experts);
    /* rows are addressed by 32 bits */
    if ((uint64_t)st->t_bucket * st->dm >= (1ull << 32))
        pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u times dm=%u reaches 2^32", st->t_bucket, st->dm);
    if ((uint64_t)st->t_bucket * (st->k_topk + (uint64_t)st->shared_experts) >= (1ull << 26))
        pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u rows of %u experts reach 2^26", st->t_bucket, st->k_topk + st->shared_experts);
    if (!float_dtype(st->out_dtype)) pr.add(R9VX_ERR_UNSUPPORTED, "out_dtype %u: only f32 and bf16 outputs", st->out_dtype);
    if (pr.code == R9VX_OK && !r9vx_moe_fp8_launchable(moe_fp8_problem(st)))
        pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u rows of %u experts and dff=%u have more tiles than a launch", st->t_bucket,
               st->k_topk + st->shared_experts, st->dff);
}

static bool moe_fp8_static_ok(const r9vx_moe_ffn_fp8_static *st) {
    if (!st) return false;
    Problems pr;
    check_moe_fp8_static(st, pr);
    return pr.code == R9VX_OK;
}

size_t r9vx_moe_ffn_fp8_workspace_bytes(const r9vx_moe_ffn_fp8_static *st) {
    return moe_fp8_static_ok(st) ? r9vx_moe_fp8_workspace_bytes(moe_fp8_problem(st)) : 0;
}

uint64_t r9vx_moe_ffn_fp8_expert_bytes(const r9vx_moe_ffn_fp8_static *st) {
    if (!moe_fp8_static_ok(st)) return 0;
    return 3ull * st->dm * st->dff + 12ull * (st->dm / kFp8Block) * (st->dff / kFp8Block);
}

uint64_t r9vx_moe_ffn_fp8_static_bytes(const r9vx_moe_ffn_fp8_static *st, uint32_t t) {
    if (!moe_fp8_static_ok(st)) return 0;
    const uint64_t pairs = (uint64_t)t * st->k_topk;
    const uint64_t experts = (pairs < st->e_local ? pairs : st->e_local) + st->shared_experts;
    return experts * r9vx_moe_ffn_fp8_expert_bytes(st) + (uint64_t)t * st->dm * (2 + (st->out_dtype == R9VX_DTYPE_F32 ? 4 : 2)) + pairs * 8;
}

uint64_t r9vx_moe_ffn_fp8_static_flops(const r9vx_moe_ffn_fp8_static *st, uint32_t t) {
    if (!moe_fp8_static_ok(st)) return 0;
    return 6ull * t * (st->k_topk + st->shared_experts) * st->dm * st->dff;
}

int r9vx_moe_ffn_fp8_launch(const r9vx_moe_ffn_fp8_static *st, const r9vx_moe_ffn_fp8_args *a, r9vx_stream_t stream) {
    return r9vx_moe_ffn_fp8_launch_ex(st, a, nullptr, 0, stream);
}

int r9vx_moe_ffn_fp8_launch_ex(const r9vx_moe_ffn_fp8_static *st, const r9vx_moe_ffn_fp8_args *a, uint32_t *status, uint32_t nan_refused,
                               r9vx_stream_t stream) {
    Problems pr;
    if (!st || !a) {
        pr.add(R9VX_ERR_NULL, "static and args must be non-NULL");
        return pr.finish("moe_ffn_fp8");
    }
    check_moe_fp8_static(st, pr);
    if (a->t > st->t_bucket) pr.add(R9VX_ERR_INVALID, "t=%u exceeds t_bucket=%u", a->t, st->t_bucket);
    if (a->t > 0) {
        if (!a->x || !a->expert_ids || !a->weights || !a->y) pr.add(R9VX_ERR_NULL, "x, expert_ids, weights and y are required");
        if (!a->w_gate_up || !a->w_gate_up_scales || !a->w_down || !a->w_down_scales)
            pr.add(R9VX_ERR_NULL, "w_gate_up, w_down and their scales are required");
        if (!a->workspace) pr.add(R9VX_ERR_WORKSPACE, "workspace of r9vx_moe_ffn_fp8_workspace_bytes required");
    }
    if (!aligned16(a->x) || !aligned16(a->w_gate_up) || !aligned16(a->w_down) || !aligned16(a->y))
        pr.add(R9VX_ERR_ALIGN, "x, w_gate_up, w_down and y must be 16-byte aligned");
    if (((uintptr_t)a->expert_ids | (uintptr_t)a->weights | (uintptr_t)a->w_gate_up_scales | (uintptr_t)a->w_down_scales) & 3u)
        pr.add(R9VX_ERR_ALIGN, "expert_ids, weights and scales must be 4-byte aligned");
    if ((uintptr_t)a->workspace & 255u) pr.add(R9VX_ERR_ALIGN, "workspace must be 256-byte aligned");
    if ((uintptr_t)status & 3u) pr.add(R9VX_ERR_ALIGN, "the status word must be 4-byte aligned");
    if (pr.code == R9VX_OK && a->t) { /* x is read before y is written, the rest beside it */
        const uint64_t t = a->t, ny = t * st->dm * float_bytes(st->out_dtype), pairs = t * st->k_topk * 4, ws = r9vx_moe_ffn_fp8_workspace_bytes(st);
        if (overlap(a->y, ny, a->expert_ids, pairs) || overlap(a->y, ny, a->weights, pairs))
            pr.add(R9VX_ERR_INVALID, "y must not overlap expert_ids or weights");
        if (overlap(a->workspace, ws, a->y, ny) || overlap(a->workspace, ws, a->x, t * st->dm * 2) ||
            overlap(a->workspace, ws, a->expert_ids, pairs) || overlap(a->workspace, ws, a->weights, pairs))
            pr.add(R9VX_ERR_INVALID, "the workspace must not overlap x, expert_ids, weights or y");
    }
    const int rc = pr.finish("moe_ffn_fp8");
    if (rc || a->t == 0) return rc;
    r9vx_moe_fp8_problem p = moe_fp8_problem(st);
    p.x = reinterpret_cast<const uint16_t *>(a->x);
    p.ids = a->expert_ids;
    p.weights = a->weights;
    p.w_gu = a->w_gate_up;
    p.w_dn = a->w_down;
    p.s_gu = a->w_gate_up_scales;
    p.s_dn = a->w_down_scales;
    p.y = a->y;
    p.ws = a->workspace;
    p.t = a->t;
    p.status = status;
    p.nan_refused = nan_refused;
    return hip_status("moe_ffn_fp8", r9vx_launch_moe_fp8(p, reinterpret_cast<hipStream_t>(stream)));
}

int r9vx_moe_ffn_fp8_status(const r9vx_moe_ffn_fp8_static *st, const uint8_t *workspace, uint32_t *status, r9vx_stream_t stream) {
    Problems pr;
    if (!st || !workspace || !status) {
        pr.add(R9VX_ERR_NULL, "static, workspace and status are required");
        return pr.finish("moe_ffn_fp8_status");
    }
    check_moe_fp8_static(st, pr);
    const int rc = pr.finish("moe_ffn_fp8_status");
    if (rc) return rc;
    r9vx_moe_fp8_problem p = moe_fp8_problem(st);
    p.ws = const_cast<uint8_t *>(workspace);
    return r9vx_status_read(r9vx_moe_fp8_status_word(p), status, stream);
}

}  // extern "C"
