/*
 * route_group.hip -- grouped routing on the GPU (r9vx_moe_route_group_launch).
 *
 * Per row: s = softmax(l) or sigmoid(l); c = s + bias; a group's score is its
 * largest c or the sum of its two largest; the topk_group groups of the
 * largest score stay; of their experts the K of the largest c, in that order,
 * ties to the lower index; w = s [/ their sum] * scale.
 *
 * Which experts are chosen must not depend on f32 roundings: scores and
 * comparisons are f64.  One wave per row, no workgroup talks to another.
 */
#include "r9vx_device.h"
#include "r9vx_internal.h"

namespace {

struct GroupArgs {
    const float *logits;
    const float *bias;
    uint32_t *ids;
    float *weights;
    uint32_t *status;
    uint32_t t, e, k, groups, topk_group, per; /* per: experts of a group */
    uint32_t scoring, renormalize, top2;
    double scale;
};

/* Orders doubles as unsigned integers, -0 as +0; every finite value is above 0. */
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unorder64(uint64_t k) {
    return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}
__device__ __forceinline__ uint64_t xor64(uint64_t v, int mask) {
    return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), mask, 64) << 32) | (uint32_t)__shfl_xor((int)v, mask, 64);
}
__device__ __forceinline__ double add_xor(double v) {
    for (int m = 32; m > 0; m >>= 1) v += __builtin_bit_cast(double, xor64(__builtin_bit_cast(uint64_t, v), m));
    return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, uint32_t lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), (int)lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* The larger of two, then the second largest of four: (a, b) <- the two
 * largest of (a, b) and (x, y), a >= b, x >= y. */
__device__ __forceinline__ void join2(uint64_t &a, uint64_t &b, uint64_t x, uint64_t y) {
    const uint64_t lo = a < x ? a : x;
    const uint64_t hb = b < y ? y : b;
    a = a < x ? x : a;
    b = lo < hb ? hb : lo;
}

/* The mask of the kept groups.  key[e]: order64 of c.  64 / G lanes share a
 * group (G: the groups, rounded up to a power of two). */
__device__ __forceinline__ uint64_t kept_groups(const GroupArgs &a, uint32_t lane, const uint64_t *key) {
    if (a.topk_group == a.groups) return ~0ull;
    uint32_t share = 64;
    while (share * a.groups > 64) share >>= 1;
    const uint32_t g = lane / share;
    uint64_t first = 0, second = 0; /* below every key */
    if (g < a.groups)
        for (uint32_t i = lane % share; i < a.per; i += share) join2(first, second, key[g * a.per + i], 0);
    for (uint32_t m = 1; m < share; m <<= 1) join2(first, second, xor64(first, (int)m), xor64(second, (int)m));
    const uint64_t score = a.top2 ? order64(unorder64(first) + unorder64(second)) : first;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < a.groups; ++j) {
        const uint64_t s = lane64(score, j * share);
        rank += s > score || (s == score && j < g) ? 1u : 0u;
    }
    const uint64_t in = __ballot(g < a.groups && rank < a.topk_group);
    uint64_t kept = 0; /* bit j: group j, which lane j * share speaks for */
    for (uint32_t j = 0; j < a.groups; ++j) kept |= (in >> (j * share) & 1ull) << j;
    return kept;
}

/* A row with a non-finite logit or bias, or whose selected scores sum to
 * zero: no expert (every later stage refuses the id), weight 0. */
__device__ __forceinline__ void refuse_row(const GroupArgs &a, uint32_t row, uint32_t lane, uint32_t bits) {
    if (lane < a.k) {
        a.ids[(uint64_t)row * a.k + lane] = 0xFFFFFFFFu;
        a.weights[(uint64_t)row * a.k + lane] = 0.0f;
    }
    if (lane == 0 && a.status) atomicOr(a.status, bits);
}

/* The selected experts' weights: lane j < K holds the j-th and its score. */
__device__ __forceinline__ void write_row(const GroupArgs &a, uint32_t row, uint32_t lane, uint32_t id, double s) {
    double w = s;
    if (a.renormalize) {
        const double sum = add_xor(lane < a.k ? s : 0.0);
        if (!(sum > 0.0)) {
            refuse_row(a, row, lane, R9VX_STATUS_DEGENERATE);
            return;
        }
        w = s / sum;
    }
    if (lane < a.k) {
        a.ids[(uint64_t)row * a.k + lane] = id;
        a.weights[(uint64_t)row * a.k + lane] = (float)(w * a.scale);
    }
}

/* All of a row in f64, its keys in LDS. */
__device__ void route_row64(const GroupArgs &a, uint32_t row, uint32_t lane, uint64_t *key) {
    const float *l = a.logits + (uint64_t)row * a.e;
    double top = 0.0, sum = 1.0;
    if (a.scoring == R9VX_SCORING_SOFTMAX) {
        float m = -__builtin_huge_valf();
        for (uint32_t i = lane; i < a.e; i += 64) m = fmaxf(m, l[i]);
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        top = m;
        double part = 0.0;
        for (uint32_t i = lane; i < a.e; i += 64) part += exp((double)l[i] - top);
        sum = add_xor(part);
    }
    auto score = [&](uint32_t i) {
        const double x = l[i];
        return a.scoring == R9VX_SCORING_SOFTMAX ? exp(x - top) / sum : 1.0 / (1.0 + exp(-x));
    };
    for (uint32_t i = lane; i < a.e; i += 64) key[i] = order64(score(i) + (a.bias ? (double)a.bias[i] : 0.0));
    wave_sync();
    const uint64_t kept = kept_groups(a, lane, key);
    wave_sync();
    for (uint32_t i = lane; i < a.e; i += 64)
        if (!(kept >> (a.groups > 1 ? i / a.per : 0u) & 1ull)) key[i] = 0;
    uint32_t id = 0;
    for (uint32_t j = 0; j < a.k; ++j) {
        uint64_t best = 0;
        uint32_t at = lane;
        for (uint32_t i = lane; i < a.e; i += 64)
            if (key[i] > best) best = key[i], at = i;
        for (int m = 32; m > 0; m >>= 1) {
            const uint64_t ob = xor64(best, m);
            const uint32_t oa = (uint32_t)__shfl_xor((int)at, m, 64);
            if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
        }
        if (lane == j) id = at;
        if (at % 64 == lane) key[at] = 0;
    }
    write_row(a, row, lane, id, score(id));
}

__global__ __launch_bounds__(64) void route_group_kernel(GroupArgs a) {
    __shared__ uint64_t key[1024];
    const uint32_t lane = threadIdx.x, row = blockIdx.x;
    bool bad = false;
    for (uint32_t i = lane; i < a.e; i += 64)
        bad |= !__builtin_isfinite(a.logits[(uint64_t)row * a.e + i]) || (a.bias && !__builtin_isfinite(a.bias[i]));
    if (__ballot(bad)) {
        refuse_row(a, row, lane, R9VX_STATUS_NONFINITE);
        return;
    }
    route_row64(a, row, lane, key);
}

}  // namespace

int r9vx_launch_route_group(const r9vx_route_group_problem &p, hipStream_t stream) {
    const GroupArgs a{p.logits, p.bias,   p.ids,        p.weights, p.status,      p.t,           p.e,         p.k,
                      p.n_group, p.topk_group, p.e / p.n_group, p.scoring, p.renormalize, p.group_score, (double)p.scale};
    hipLaunchKernelGGL(route_group_kernel, dim3(p.t), dim3(64), 0, stream, a);
    return (int)hipGetLastError();
}
