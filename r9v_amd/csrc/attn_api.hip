/*
 * attn_api.hip -- the C ABI of include/r9vx_attn.h: every problem of a call is
 * reported and nothing is enqueued when any is found.
 */
#include <math.h>
#include <string.h>

#include "r9vx_attn_kernels.h"
#include "r9vx_host.h"

using namespace r9vx;

namespace {

float as_float(uint32_t bits) {
    float f;
    memcpy(&f, &bits, 4);
    return f;
}

bool half_dtype(uint32_t d) { return d == R9VX_DTYPE_BF16 || d == R9VX_DTYPE_F16; }
uint64_t dtype_bytes(uint32_t d) { return d == R9VX_DTYPE_F32 ? 4 : 2; }

uint32_t log2_of(uint32_t x) { return 31u - (uint32_t)__builtin_clz(x); }

bool power_of_two(uint32_t x) { return x && !(x & (x - 1)); }

/* Bytes from a strided operand's first element to behind its last one. */
template <int N>
uint64_t span(const uint64_t (&stride)[N], const uint64_t (&size)[N], uint64_t columns, uint64_t bytes) {
    uint64_t last = 0;
    for (int i = 0; i < N; ++i) {
        if (!size[i]) return 0;
        last += (size[i] - 1) * stride[i];
    }
    return (last + columns) * bytes;
}

/* Whether an output's rows stand apart: by ascending strides, each row behind the last one's end. */
template <int N>
bool rows_apart(const uint64_t (&stride)[N], const uint64_t (&size)[N], uint64_t columns) {
    bool done[N] = {};
    for (int n = 0; n < N; ++n) {
        int least = -1;
        for (int i = 0; i < N; ++i)
            if (!done[i] && size[i] > 1 && (least < 0 || stride[i] < stride[least])) least = i;
        if (least < 0) return true;
        if (stride[least] < columns) return false;
        columns += (size[least] - 1) * stride[least];
        done[least] = true;
    }
    return true;
}

/* A strided operand's rows: of `columns` elements, `size` of them `stride` apart on each axis. */
template <int N>
struct Rows {
    uintptr_t at;
    uint64_t stride[N], size[N], columns, bytes;
    __int128 extent(int axis) const { /* from an element to behind the last of the axes from `axis` on */
        __int128 last = 0;
        for (int i = axis; i < N; ++i) last += (__int128)(size[i] - 1) * stride[i];
        return (last + columns) * bytes;
    }
};

/* Whether no row of x meets one of y, whose first element is `d` bytes behind x's.  Axes
 * go from the widest stride on.  Where both have the same stride, longer than what is
 * inside it, y's inner rows are between two of x's, the distance modulo the stride apart:
 * those are looked at in turn.  (Rows that may be apart and are not of this kind
 * count as meeting.) */
template <int N>
bool apart(const Rows<N> &x, const Rows<N> &y, __int128 d, int axis = 0) {
    if (d >= x.extent(axis) || -d >= y.extent(axis)) return true;
    if (axis == N) return false;
    const bool many = x.size[axis] > 1, also = y.size[axis] > 1;
    if (!many && !also) return apart(x, y, d, axis + 1);
    const __int128 stride = (__int128)(many ? x.stride[axis] : y.stride[axis]) * x.bytes;
    if ((many && also && x.stride[axis] != y.stride[axis]) || stride < x.extent(axis + 1) || stride < y.extent(axis + 1)) return false;
    const __int128 r = (d % stride + stride) % stride;
    return apart(x, y, r, axis + 1) && apart(x, y, r - stride, axis + 1);
}

template <int N>
bool apart(const void *px, const uint64_t (&sx)[N], const uint64_t (&nx)[N], const void *py, const uint64_t (&sy)[N], const uint64_t (&ny)[N], uint64_t columns,
           uint64_t bytes) {
    Rows<N> x{(uintptr_t)px, {}, {}, columns, bytes}, y{(uintptr_t)py, {}, {}, columns, bytes};
    bool done[N] = {};
    for (int n = 0; n < N; ++n) {
        int widest = -1;
        uint64_t most = 0;
        for (int i = 0; i < N; ++i) {
            if (!nx[i] || !ny[i]) return true;
            const uint64_t s = nx[i] > 1 ? sx[i] : ny[i] > 1 ? sy[i] : 0;
            if (!done[i] && (widest < 0 || s > most)) widest = i, most = s;
        }
        done[widest] = true;
        x.stride[n] = sx[widest], x.size[n] = nx[widest], y.stride[n] = sy[widest], y.size[n] = ny[widest];
    }
    return apart(x, y, (__int128)y.at - (__int128)x.at);
}

template <int N>
void check_strides(const char *name, const uint64_t (&stride)[N], uint64_t bytes, Problems &pr) {
    for (int i = 0; i < N; ++i) {
        if (stride[i] * bytes % 16) pr.add(R9VX_ERR_ALIGN, "%s: a stride of %llu elements is no multiple of 16 bytes", name, (unsigned long long)stride[i]);
        if (stride[i] >> 40) pr.add(R9VX_ERR_INVALID, "%s: a stride of %llu elements exceeds 2^40", name, (unsigned long long)stride[i]);
    }
}

void check_rope_static(const r9vx_rope_kv_static *st, Problems &pr) {
    if (st->heads == 0 || st->heads > 1024 || st->kv_heads > 1024)
        pr.add(R9VX_ERR_INVALID, "heads=%u must be 1 .. 1024, kv_heads=%u at most 1024", st->heads, st->kv_heads);
    if (st->head_dim == 0 || st->head_dim % 8 || st->head_dim > 512)
        pr.add(R9VX_ERR_UNSUPPORTED, "head_dim=%u must be a multiple of 8, at most 512", st->head_dim);
    if (st->rot == 0 || st->rot % 16 || st->rot > st->head_dim)
        pr.add(R9VX_ERR_INVALID, "rot=%u must be a positive multiple of 16, at most head_dim=%u", st->rot, st->head_dim);
    if (st->interleaved > 1) pr.add(R9VX_ERR_INVALID, "interleaved=%u must be 0 or 1", st->interleaved);
    if (st->kv_heads && !power_of_two(st->page_size)) pr.add(R9VX_ERR_UNSUPPORTED, "page_size=%u must be a power of two", st->page_size);
    if (st->in_dtype != R9VX_DTYPE_F32 && !half_dtype(st->in_dtype))
        pr.add(R9VX_ERR_UNSUPPORTED, "in_dtype %u: only f32, bf16 and f16", st->in_dtype);
    if (st->out_dtype != st->in_dtype && !(st->in_dtype == R9VX_DTYPE_F32 && half_dtype(st->out_dtype)))
        pr.add(R9VX_ERR_UNSUPPORTED, "out_dtype %u of in_dtype %u: only its own, or bf16 or f16 of f32", st->out_dtype, st->in_dtype);
    if (!isfinite(as_float(st->amplitude_bits))) pr.add(R9VX_ERR_INVALID, "the amplitude must be finite");
}

/* Strides alone tell an exact in-place call from one that would read what it has written. */
bool same_rows(const r9vx_rope_kv_args *a) {
    return a->q == a->q_out && a->q_stride[0] == a->q_out_stride[0] && a->q_stride[1] == a->q_out_stride[1];
}

void check_attn_static(const r9vx_attn_static *st, bool decode, Problems &pr) {
    if (st->heads == 0 || st->kv_heads == 0 || st->heads % (st->kv_heads ? st->kv_heads : 1))
        pr.add(R9VX_ERR_INVALID, "heads=%u must be a positive multiple of kv_heads=%u", st->heads, st->kv_heads);
    if (st->heads > 1024) pr.add(R9VX_ERR_UNSUPPORTED, "heads=%u exceeds 1024", st->heads);
    if (st->head_dim != 64 && st->head_dim != 96 && st->head_dim != 128 && st->head_dim != 192 && st->head_dim != 256)
        pr.add(R9VX_ERR_UNSUPPORTED, "head_dim=%u: only 64, 96, 128, 192 and 256", st->head_dim);
    if (!power_of_two(st->page_size) || st->page_size < 8)
        pr.add(R9VX_ERR_UNSUPPORTED, "page_size=%u must be a power of two, at least 8", st->page_size);
    if (!half_dtype(st->dtype)) pr.add(R9VX_ERR_UNSUPPORTED, "dtype %u: only bf16 and f16", st->dtype);
    if (st->causal > 1 || (decode && st->causal != 1)) pr.add(R9VX_ERR_INVALID, "causal=%u: 1, or for prefill 0 or 1", st->causal);
    if (!isfinite(as_float(st->scale_bits))) pr.add(R9VX_ERR_INVALID, "the scale must be finite");
    const float cap = as_float(st->softcap_bits);
    if (!(cap >= 0.0f && cap < INFINITY)) pr.add(R9VX_ERR_INVALID, "the softcap must be finite and not negative");
    else if (cap > 0.0f && !isfinite(as_float(st->scale_bits) / cap * 2.885390f)) pr.add(R9VX_ERR_INVALID, "scale / softcap must be finite");
    if (st->len_bucket > (1u << 30)) pr.add(R9VX_ERR_UNSUPPORTED, "len_bucket=%u exceeds 2^30", st->len_bucket);
    if (st->b_bucket >= (1u << 16)) pr.add(R9VX_ERR_UNSUPPORTED, "b_bucket=%u reaches 2^16", st->b_bucket); /* a grid's third extent */
    if (decode && (st->t_bucket == 0 || st->t_bucket > 8)) pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u: 1 to 8 new tokens a sequence", st->t_bucket);
    if (!decode && st->t_bucket > (1u << 24)) pr.add(R9VX_ERR_UNSUPPORTED, "t_bucket=%u exceeds 2^24", st->t_bucket);
}

r9vx_attn_problem attn_problem(const r9vx_attn_static *st, bool decode) {
    r9vx_attn_problem p{};
    p.b_bucket = st->b_bucket;
    p.t_bucket = st->t_bucket;
    p.len_bucket = st->len_bucket;
    p.heads = st->heads;
    p.kv_heads = st->kv_heads;
    p.group = st->heads / st->kv_heads;
    p.group_magic = attn_group_magic(p.group);
    p.head_dim = st->head_dim;
    p.page_shift = log2_of(st->page_size);
    p.dtype = st->dtype;
    p.causal = st->causal;
    p.window = st->window && st->window < kAttnNoWindow ? st->window : kAttnNoWindow;
    p.scale = as_float(st->scale_bits);
    /* (a cap of 2^100 leaves scores up to 2^88 as they are, and scale / cap a normal number) */
    p.softcap = fminf(as_float(st->softcap_bits), 0x1p100f);
    p.b = st->b_bucket;
    p.t = st->t_bucket;
    if (decode) r9vx_attn_decode_plan(p);
    else r9vx_attn_prefill_plan(p);
    return p;
}

/* A launch's threads are counted in 32 bits. */
void check_groups(const r9vx_attn_static *st, bool decode, Problems &pr) {
    const r9vx_attn_problem p = attn_problem(st, decode);
    const uint64_t groups = decode ? r9vx_attn_decode_groups(p) : r9vx_attn_prefill_groups(p);
    if (groups >= (1u << 24) || (!decode && (uint64_t)st->t_bucket * p.group >= (1u << 31)))
        pr.add(R9VX_ERR_UNSUPPORTED, "b_bucket=%u, t_bucket=%u of %u heads have more tiles than a launch", st->b_bucket, st->t_bucket, st->heads);
    const uint64_t rows = (decode ? (uint64_t)st->b_bucket : 1ull) * st->t_bucket * st->heads;
    if (p.splits > 1 && r9vx_attn_join_groups(p, rows) >= (1u << 24))
        pr.add(R9VX_ERR_UNSUPPORTED, "b_bucket=%u, t_bucket=%u of %u heads and len_bucket=%u: more rows to join than a launch has", st->b_bucket, st->t_bucket, st->heads, st->len_bucket);
}

size_t attn_workspace_bytes(const r9vx_attn_static *st, bool decode) {
    if (!st) return 0;
    Problems pr;
    check_attn_static(st, decode, pr);
    if (pr.code == R9VX_OK) check_groups(st, decode, pr);
    if (pr.code != R9VX_OK) return 0;
    const r9vx_attn_problem p = attn_problem(st, decode);
    if (p.splits == 1) return 0;
    const uint64_t rows = (decode ? (uint64_t)st->b_bucket : 1ull) * st->t_bucket * st->heads;
    return rows * p.splits * (4ull * st->head_dim + 8);
}

int attn_launch(const char *op, bool decode, const r9vx_attn_static *st, const r9vx_attn_args *a, r9vx_stream_t stream) {
    Problems pr;
    if (!st || !a) {
        pr.add(R9VX_ERR_NULL, "static and args must be non-NULL");
        return pr.finish(op);
    }
    check_attn_static(st, decode, pr);
    if (pr.code == R9VX_OK) check_groups(st, decode, pr);
    const uint32_t t = decode ? st->t_bucket : a->t;
    const bool work = a->b > 0 && t > 0;
    if (a->b > st->b_bucket) pr.add(R9VX_ERR_INVALID, "b=%u exceeds b_bucket=%u", a->b, st->b_bucket);
    if (decode && a->t) pr.add(R9VX_ERR_INVALID, "t=%u: a decode launch has its static's t_bucket", a->t);
    if (!decode && a->t > st->t_bucket) pr.add(R9VX_ERR_INVALID, "t=%u exceeds t_bucket=%u", a->t, st->t_bucket);
    if (work) {
        if (!a->q || !a->k_cache || !a->v_cache || !a->out) pr.add(R9VX_ERR_NULL, "q, k_cache, v_cache and out are required");
        if (!a->table || !a->lengths) pr.add(R9VX_ERR_NULL, "table and lengths are required");
        if (!decode && !a->offsets) pr.add(R9VX_ERR_NULL, "offsets are required");
        if (a->pages == 0) pr.add(R9VX_ERR_INVALID, "the cache has no page");
    }
    if (a->pages > (1u << 31)) pr.add(R9VX_ERR_UNSUPPORTED, "pages=%u exceeds 2^31", a->pages);
    if (decode && (a->offsets || a->prefix)) pr.add(R9VX_ERR_INVALID, "offsets and prefix are prefill's");
    if (!st->causal && a->prefix) pr.add(R9VX_ERR_INVALID, "a prefix without a causal mask");
    if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out))
        pr.add(R9VX_ERR_ALIGN, "q, k_cache, v_cache and out must be 16-byte aligned");
    if (((uintptr_t)a->table | (uintptr_t)a->lengths | (uintptr_t)a->offsets | (uintptr_t)a->starts | (uintptr_t)a->prefix |
         (uintptr_t)a->slopes | (uintptr_t)a->status) & 3u)
        pr.add(R9VX_ERR_ALIGN, "table, lengths, offsets, starts, prefix, slopes and status must be 4-byte aligned");
    check_strides("q", a->q_stride, 2, pr);
    check_strides("out", a->out_stride, 2, pr);
    check_strides("k_cache", a->k_stride, 2, pr);
    check_strides("v_cache", a->v_stride, 2, pr);
    if (a->k_stride[1] >> 27 || a->v_stride[1] >> 27) pr.add(R9VX_ERR_UNSUPPORTED, "a cache's tokens are 2^27 elements or more apart"); /* 8 rows: 32 bits */
    const size_t ws = pr.code == R9VX_OK ? attn_workspace_bytes(st, decode) : 0;
    if (ws && work && !a->workspace) pr.add(R9VX_ERR_WORKSPACE, "workspace of r9vx_attn_%s_workspace_bytes (%zu) required", decode ? "decode" : "prefill", ws);
    if ((uintptr_t)a->workspace & 255u) pr.add(R9VX_ERR_ALIGN, "workspace must be 256-byte aligned");
    if (pr.code == R9VX_OK && work) {
        if (a->b > 1 && a->table_stride < (st->len_bucket + (uint64_t)st->page_size - 1) / st->page_size)
            pr.add(R9VX_ERR_INVALID, "rows of the table are %llu columns apart, fewer than len_bucket=%u has pages", (unsigned long long)a->table_stride, st->len_bucket);
        const uint64_t rows[3] = {decode ? a->b : 1, t, st->heads}, cache[3] = {a->pages, st->page_size, st->kv_heads};
        const uint64_t nq = span(a->q_stride, rows, st->head_dim, 2), ny = span(a->out_stride, rows, st->head_dim, 2);
        const uint64_t nk = span(a->k_stride, cache, st->head_dim, 2), nv = span(a->v_stride, cache, st->head_dim, 2);
        const uint64_t tokens = decode ? a->b : t;
        const uint64_t nt = ((uint64_t)(a->b - 1) * a->table_stride + (st->len_bucket + (uint64_t)st->page_size - 1) / st->page_size) * 4;
        if (overlap(a->out, ny, a->q, nq) || overlap(a->out, ny, a->k_cache, nk) || overlap(a->out, ny, a->v_cache, nv) ||
            overlap(a->out, ny, a->table, nt) || overlap(a->out, ny, a->lengths, 4ull * a->b) || overlap(a->out, ny, a->offsets, 4ull * a->b + 4) ||
            overlap(a->out, ny, a->starts, 4 * tokens) || overlap(a->out, ny, a->prefix, 4ull * a->b) || overlap(a->out, ny, a->slopes, 4ull * st->heads))
            pr.add(R9VX_ERR_INVALID, "out must not overlap an operand");
        if (!rows_apart(a->out_stride, rows, st->head_dim)) pr.add(R9VX_ERR_INVALID, "rows of out overlap each other");
        if (overlap(a->workspace, ws, a->q, nq) || overlap(a->workspace, ws, a->out, ny) || overlap(a->workspace, ws, a->k_cache, nk) ||
            overlap(a->workspace, ws, a->v_cache, nv) || overlap(a->workspace, ws, a->table, nt) || overlap(a->workspace, ws, a->lengths, 4ull * a->b) ||
            overlap(a->workspace, ws, a->offsets, 4ull * a->b + 4) || overlap(a->workspace, ws, a->starts, 4 * tokens) ||
            overlap(a->workspace, ws, a->prefix, 4ull * a->b) || overlap(a->workspace, ws, a->slopes, 4ull * st->heads))
            pr.add(R9VX_ERR_INVALID, "the workspace must not overlap an operand or out");
    }
    const int rc = pr.finish(op);
    if (rc || !work) return rc;
    r9vx_attn_problem p = attn_problem(st, decode);
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k_cache);
    p.v = static_cast<const uint16_t *>(a->v_cache);
    p.table = a->table;
    p.lengths = a->lengths;
    p.offsets = a->offsets;
    p.starts = a->starts;
    p.prefix = a->prefix;
    p.slopes = a->slopes;
    p.out = static_cast<uint16_t *>(a->out);
    p.partial = reinterpret_cast<float *>(a->workspace);
    p.status = a->status;
    memcpy(p.q_stride, a->q_stride, sizeof p.q_stride);
    memcpy(p.out_stride, a->out_stride, sizeof p.out_stride);
    memcpy(p.k_stride, a->k_stride, sizeof p.k_stride);
    memcpy(p.v_stride, a->v_stride, sizeof p.v_stride);
    p.table_stride = a->table_stride;
    p.pages = a->pages;
    p.b = a->b;
    p.t = a->t;
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return hip_status(op, decode ? r9vx_launch_attn_decode(p, s) : r9vx_launch_attn_prefill(p, s));
}

}  // namespace

extern "C" {

int r9vx_rope_kv_launch(const r9vx_rope_kv_static *st, const r9vx_rope_kv_args *a, r9vx_stream_t stream) {
    Problems pr;
    if (!st || !a) {
        pr.add(R9VX_ERR_NULL, "static and args must be non-NULL");
        return pr.finish("rope_kv");
    }
    check_rope_static(st, pr);
    const bool cache = st->kv_heads > 0;
    const uint64_t in = dtype_bytes(st->in_dtype), out = dtype_bytes(st->out_dtype);
    if (a->t > (1u << 23)) pr.add(R9VX_ERR_UNSUPPORTED, "t=%u exceeds 2^23", a->t); /* a launch's threads: 32 bits */
    if (a->t) {
        if (!a->q || !a->q_out || !a->positions || !a->freqs) pr.add(R9VX_ERR_NULL, "q, q_out, positions and freqs are required");
        if (cache && (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slots)) pr.add(R9VX_ERR_NULL, "k, v, k_cache, v_cache and slots are required");
    }
    if (!cache && (a->k || a->v || a->k_cache || a->v_cache || a->slots)) pr.add(R9VX_ERR_INVALID, "k, v, a cache or slots without kv_heads");
    if (a->pages > (1u << 31)) pr.add(R9VX_ERR_UNSUPPORTED, "pages=%u exceeds 2^31", a->pages);
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
        pr.add(R9VX_ERR_ALIGN, "q, k, v, q_out, k_cache and v_cache must be 16-byte aligned");
    if (((uintptr_t)a->freqs | (uintptr_t)a->slots) & 7u) pr.add(R9VX_ERR_ALIGN, "freqs and slots must be 8-byte aligned");
    if (((uintptr_t)a->positions | (uintptr_t)a->status) & 3u) pr.add(R9VX_ERR_ALIGN, "positions and status must be 4-byte aligned");
    check_strides("q", a->q_stride, in, pr);
    check_strides("q_out", a->q_out_stride, out, pr);
    if (cache) {
        check_strides("k", a->k_stride, in, pr);
        check_strides("v", a->v_stride, in, pr);
        check_strides("k_cache", a->k_cache_stride, out, pr);
        check_strides("v_cache", a->v_cache_stride, out, pr);
    }
    if (pr.code == R9VX_OK && a->t) {
        const uint64_t rows[2] = {a->t, st->heads}, kv[2] = {a->t, st->kv_heads}, pages[3] = {a->pages, st->page_size, st->kv_heads};
        const uint64_t nq = span(a->q_stride, rows, st->head_dim, in), ny = span(a->q_out_stride, rows, st->head_dim, out);
        const bool in_place = same_rows(a) && in == out;
        if (!in_place && overlap(a->q_out, ny, a->q, nq)) pr.add(R9VX_ERR_INVALID, "q_out must not overlap q (it may be q, with q's strides and type)");
        if (overlap(a->q_out, ny, a->positions, 4ull * a->t) || overlap(a->q_out, ny, a->freqs, 4ull * st->rot) || overlap(a->q_out, ny, a->slots, 8ull * a->t))
            pr.add(R9VX_ERR_INVALID, "q_out must not overlap positions, freqs or slots");
        if (!rows_apart(a->q_out_stride, rows, st->head_dim)) pr.add(R9VX_ERR_INVALID, "rows of q_out overlap each other");
        if (cache) {
            const uint64_t nk = span(a->k_stride, kv, st->head_dim, in), nv = span(a->v_stride, kv, st->head_dim, in);
            const uint64_t nkc = span(a->k_cache_stride, pages, st->head_dim, out), nvc = span(a->v_cache_stride, pages, st->head_dim, out);
            /* q in place may stand among k's and v's rows, as one projection leaves them, but be none of them */
            if (in_place ? !apart(a->q_out, a->q_out_stride, rows, a->k, a->k_stride, kv, st->head_dim, in) || !apart(a->q_out, a->q_out_stride, rows, a->v, a->v_stride, kv, st->head_dim, in)
                         : overlap(a->q_out, ny, a->k, nk) || overlap(a->q_out, ny, a->v, nv))
                pr.add(R9VX_ERR_INVALID, "q_out must not overlap k or v");
            if (overlap(a->k_cache, nkc, a->q, nq) || overlap(a->k_cache, nkc, a->k, nk) || overlap(a->k_cache, nkc, a->v, nv) || overlap(a->k_cache, nkc, a->q_out, ny) ||
                overlap(a->v_cache, nvc, a->q, nq) || overlap(a->v_cache, nvc, a->k, nk) || overlap(a->v_cache, nvc, a->v, nv) || overlap(a->v_cache, nvc, a->q_out, ny))
                pr.add(R9VX_ERR_INVALID, "the cache must not overlap q, k, v or q_out");
            if (overlap(a->k_cache, nkc, a->positions, 4ull * a->t) || overlap(a->k_cache, nkc, a->freqs, 4ull * st->rot) || overlap(a->k_cache, nkc, a->slots, 8ull * a->t) ||
                overlap(a->v_cache, nvc, a->positions, 4ull * a->t) || overlap(a->v_cache, nvc, a->freqs, 4ull * st->rot) || overlap(a->v_cache, nvc, a->slots, 8ull * a->t))
                pr.add(R9VX_ERR_INVALID, "the cache must not overlap positions, freqs or slots");
            /* (keys and values may take turns in one allocation) */
            if (!rows_apart(a->k_cache_stride, pages, st->head_dim) || !rows_apart(a->v_cache_stride, pages, st->head_dim) ||
                !apart(a->k_cache, a->k_cache_stride, pages, a->v_cache, a->v_cache_stride, pages, st->head_dim, out))
                pr.add(R9VX_ERR_INVALID, "rows of the cache overlap each other");
        }
    }
    const int rc = pr.finish("rope_kv");
    if (rc || a->t == 0) return rc;
    r9vx_rope_problem p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.positions = a->positions;
    p.freqs = a->freqs;
    p.q_out = a->q_out;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.slots = a->slots;
    p.status = a->status;
    memcpy(p.q_stride, a->q_stride, sizeof p.q_stride);
    memcpy(p.k_stride, a->k_stride, sizeof p.k_stride);
    memcpy(p.v_stride, a->v_stride, sizeof p.v_stride);
    memcpy(p.q_out_stride, a->q_out_stride, sizeof p.q_out_stride);
    memcpy(p.k_cache_stride, a->k_cache_stride, sizeof p.k_cache_stride);
    memcpy(p.v_cache_stride, a->v_cache_stride, sizeof p.v_cache_stride);
    p.pages = a->pages;
    p.t = a->t;
    p.heads = st->heads;
    p.kv_heads = st->kv_heads;
    p.head_dim = st->head_dim;
    p.rot = st->rot;
    p.interleaved = st->interleaved;
    p.page_shift = cache ? log2_of(st->page_size) : 0;
    p.in_dtype = st->in_dtype;
    p.out_dtype = st->out_dtype;
    p.amplitude = as_float(st->amplitude_bits);
    return hip_status("rope_kv", r9vx_launch_rope_kv(p, reinterpret_cast<hipStream_t>(stream)));
}

size_t r9vx_attn_decode_workspace_bytes(const r9vx_attn_static *st) { return attn_workspace_bytes(st, true); }
size_t r9vx_attn_prefill_workspace_bytes(const r9vx_attn_static *st) { return attn_workspace_bytes(st, false); }

int r9vx_attn_decode_launch(const r9vx_attn_static *st, const r9vx_attn_args *a, r9vx_stream_t stream) {
    return attn_launch("attn_decode", true, st, a, stream);
}
int r9vx_attn_prefill_launch(const r9vx_attn_static *st, const r9vx_attn_args *a, r9vx_stream_t stream) {
    return attn_launch("attn_prefill", false, st, a, stream);
}

}  // extern "C"
