/*
 * route_group.hip -- grouped routing on the GPU (r9vx_moe_route_group_launch).
 *
 * Per row: s = softmax(l) or sigmoid(l); c = s + bias; a group's score is its
 * largest c or the sum of its two largest; the topk_group groups of the
 * largest score stay; of their experts the K of the largest c, in that order,
 * ties to the lower index; w = s [/ their sum] * scale.
 *
 * Which experts are chosen must not depend on f32 roundings: the definition
 * compares in f64.  A row is routed on f32 keys, and the comparisons that
 * decide (around the last kept group, around the last chosen expert, between
 * neighbours of the order) are checked against the keys' error bounds; a row
 * with one too close to call, about one in ten thousand, goes through f64 as
 * a whole.  The K weights are computed in f64 either way.  One wave per row,
 * no workgroup talks to another.
 *
 * Bound by instruction issue: 906 vector instructions a row at 512 experts,
 * K = 10 (a third of them the K + 1 maxima in turn), 8192 rows 17 us against 4
 * of their bytes; everything in f64 took 59.  5 rows of 256 experts: 6.3 us, a
 * chain of dependent steps behind a launch.
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
    uint32_t t, e, k, groups, topk_group, per, inv; /* per: experts of a group, inv: 2^22 / per, rounded up */
    uint32_t scoring, renormalize, top2;
    double scale;
};

__device__ __forceinline__ uint64_t xor64(uint64_t v, int mask) {
    return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), mask, 64) << 32) | (uint32_t)__shfl_xor((int)v, mask, 64);
}
__device__ __forceinline__ double add_xor(double v) {
    for (int m = 32; m > 0; m >>= 1) v += __builtin_bit_cast(double, xor64(__builtin_bit_cast(uint64_t, v), m));
    return v;
}
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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

template <int CTRL>
__device__ __forceinline__ uint32_t dpp32(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t max_wave(uint32_t x) {
    x = max(x, dpp32<0xB1>(x));
    x = max(x, dpp32<0x4E>(x));
    x = max(x, dpp32<0x141>(x));
    x = max(x, dpp32<0x140>(x));
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t)r[0], (uint32_t)r[1]);
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint64_t max_wave(uint64_t x) {
    const uint32_t hi = max_wave((uint32_t)(x >> 32));
    return ((uint64_t)hi << 32) | max_wave((uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
}
/* Orders floats as unsigned integers, -0 as +0; every finite value is above 0. */
__device__ __forceinline__ uint32_t order(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ float unorder(uint32_t k) { return __builtin_bit_cast(float, k >> 31 ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint32_t read_lane(uint32_t v, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, uint32_t lane) {
    return ((uint64_t)read_lane((uint32_t)(v >> 32), lane) << 32) | read_lane((uint32_t)v, lane);
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }
/* f32: the hardware's exponential and reciprocal, which score_slack counts. */
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float over(float a, float b) { return a * __builtin_amdgcn_rcpf(b); }
__device__ __forceinline__ double over(double a, double b) { return a / b; }

/* How far f32 scores are from f64's.  The exponential of v is off by (1.5 |v|
 * + 2) 2^-24 of itself (v times log2 e, rounded, and the instruction's step).
 * sigmoid: times the slope s (1 - s) that is under 2^-24, the sum and the
 * reciprocal add 3 x 2^-24: 2^-22.  softmax, v = x - the largest, rounded: under
 * 2^-22 of the largest score `top`, and the sum's rounding, the reciprocal and
 * the product add 2^-22 of each score: 2^-21 of `top`.  Twice that. */
template <bool SIGMOID>
__device__ __forceinline__ float score_slack(float top) {
    return SIGMOID ? 0x1p-21f : top * 0x1p-20f;
}

/* Whether f32 may have two keys a >= b in another order than f64.
 * Keys with a bias are f32 sums, each off by a score's slack and 2^-24 of
 * itself.  Keys without one are the logits, whose order is the scores', unless
 * f64 rounds two different scores to one value or underflows: sigmoid's slope
 * is under 2^-24 only for logits above 16 (and two f32 logits there are 2^-20
 * apart: 2^-44 in the score, f64's step is 2^-53), exp(x) > 0 for x > -600. */
template <bool BIAS, bool SIGMOID>
__device__ __forceinline__ bool unsure(float a, float b, float top) {
    if constexpr (BIAS) return !(a - b > 2.0f * score_slack<SIGMOID>(top) + (fabsf(a) + fabsf(b)) * 0x1p-23f);
    const float low = SIGMOID ? b : b - top;
    return a != b && (!(a - b > (fabsf(a) + fabsf(b) + fabsf(top) + 1.0f) * 0x1p-40f) || low < -600.0f || (SIGMOID && a > 16.0f));
}

template <class F>
struct Ordered;
template <>
struct Ordered<float> {
    typedef uint32_t type;
};
template <>
struct Ordered<double> {
    typedef uint64_t type;
};

/* A row's experts and weights from its PER logits and biases per lane; keys:
 * LDS.  F = double is the definition.  F = float returns false, having written
 * nothing, if a comparison that decides is too close to call. */
template <int PER, bool BIAS, bool SIGMOID, class F>
__device__ __forceinline__ bool route_row(const GroupArgs &a, uint32_t row, uint32_t lane, const float (&x)[PER], const float (&b)[PER],
                                          F *keys) {
    typedef typename Ordered<F>::type U;
    constexpr bool kWide = sizeof(F) == 8, kLogits = !kWide && !BIAS; /* kLogits: a logit is its expert's key */
    const bool grouped = a.topk_group < a.groups, sums = grouped && a.top2;
    F c[PER];
    float top = 0.0f; /* softmax: the largest logit */
    F largest = 0;    /* softmax: the largest score */
    double sum = 1.0;
    if constexpr (!SIGMOID) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = max(m, lane + 64 * i < a.e ? order(x[i]) : 0u);
        top = unorder(max_wave(m));
    }
    if (!kLogits || sums || (!SIGMOID && !a.renormalize)) { /* the scores themselves are needed */
        if constexpr (SIGMOID) {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = over((F)1, (F)1 + exp_of(-(F)x[i]));
        } else {
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = lane + 64 * i < a.e ? exp_of((F)x[i] - (F)top) : (F)0;
                if (kWide || a.renormalize)
                    part += (double)c[i];
                else if (lane + 64 * i < a.e) /* a weight is a share of this sum */
                    part += exp((double)x[i] - (double)top);
            }
            sum = add_xor(part);
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = over(c[i], (F)sum);
            largest = over((F)1, (F)sum);
        }
        if constexpr (BIAS)
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = c[i] + (F)b[i];
    }
    U key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = lane + 64 * i < a.e ? order(kLogits ? (F)x[i] : c[i]) : (U)0;
    bool doubt = false;
    if (grouped) {
        /* 64 / G lanes share a group (G: the groups, rounded up to a power of two) */
        wave_sync();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 64 * i < a.e) keys[lane + 64 * i] = kLogits && !sums ? (F)x[i] : c[i];
        wave_sync();
        uint32_t share = 64;
        while (share * a.groups > 64) share >>= 1;
        const uint32_t g = lane / share;
        F first = -__builtin_huge_val(), second = first;
        if (g < a.groups)
            for (uint32_t i = lane % share; i < a.per; i += share) {
                const F v = keys[g * a.per + i];
                second = larger(second, smaller(first, v));
                first = larger(first, v);
            }
        for (uint32_t m = 1; m < share; m <<= 1) {
            const F of = __shfl_xor(first, (int)m, 64), os = __shfl_xor(second, (int)m, 64);
            second = larger(smaller(first, of), larger(second, os));
            first = larger(first, of);
        }
        const F total = a.top2 ? first + second : first;
        const U mine = g < a.groups ? order(total) : (U)0;
        uint32_t rank = 0;
        for (uint32_t j = 0; j < a.groups; ++j) {
            const U s = read_lane(mine, j * share);
            rank += s > mine || (s == mine && j < g) ? 1u : 0u;
        }
        const bool in = g < a.groups && rank < a.topk_group;
        const uint64_t stay = __ballot(in);
        if constexpr (!kWide) {
            const bool out = g < a.groups && !in;
            /* a sum of two keys is off by both their errors and its own rounding */
            const float off = sums ? 2.0f * score_slack<SIGMOID>(largest) + (fabsf(first) + fabsf(second)) * 0x1p-22f : 0.0f;
            const float least = unorder(~max_wave(in ? ~order(total - off) : 0u)), next = unorder(max_wave(out ? order(total + off) : 0u));
            doubt = sums ? !(least > next) : unsure<BIAS, SIGMOID>(least, next, BIAS ? largest : top);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t e = lane + 64 * i; /* e, per <= 1024: the product by inv is exact enough */
            if (!(stay >> ((e < a.e ? e * a.inv >> 22 : 0u) * share) & 1ull)) key[i] = 0;
        }
    }
    /* The K largest keys, and in f32 the one behind them: lane j the j-th.
     * best, after: the lane's two largest keys that are left, at and then where
     * they stand; most lanes give one or none, so a look through all PER keys
     * again is rare. */
    const uint32_t left = a.topk_group * a.per, n = !kWide && a.k < left ? a.k + 1 : a.k;
    uint32_t id = 0, at = 0, then = 0;
    U mk = 0, best = 0, after = 0;
    bool stale = false; /* `after` was taken */
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool first = key[i] > best, second = key[i] > after;
        after = first ? best : second ? key[i] : after;
        then = first ? at : second ? i : then;
        best = first ? key[i] : best;
        at = first ? i : at;
    }
    for (uint32_t j = 0; j < n; ++j) {
        const U m = max_wave(best);
        const uint64_t tied = __ballot(best == m);
        const uint32_t e = lane + 64 * at;
        uint32_t won = read_lane(e, (uint32_t)__builtin_ctzll(tied));
        if (tied & (tied - 1)) won = ~max_wave(best == m ? ~e : 0u); /* ties: the lowest index */
        if (lane == j) id = won, mk = m;
        if (PER > 1 && __ballot(stale && e == won)) {
            if (stale && e == won) { /* the largest key behind (best, at) */
                after = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if ((key[i] < best || (key[i] == best && i > (int)at)) && key[i] > after) after = key[i], then = i;
                stale = false;
            }
        }
        if (e == won) best = after, at = then, stale = true;
    }
    if constexpr (!kWide) {
        const float v = unorder(mk), vn = __shfl_down(v, 1, 64);
        /* sigmoid with a bias: only which experts; their order is taken in f64 below */
        const uint32_t from = BIAS && SIGMOID ? a.k - 1 : 0u;
        doubt |= __ballot(lane >= from && lane + 1 < n && unsure<BIAS, SIGMOID>(v, vn, BIAS ? largest : top)) != 0;
        if (doubt) return false;
    }
    double s = 0.0;
    if (lane < a.k) {
        const double xl = a.logits[(uint64_t)row * a.e + id];
        s = SIGMOID ? 1.0 / (1.0 + exp(-xl)) : exp(xl - (double)top) / sum;
    }
    if constexpr (BIAS && SIGMOID && !kWide) {
        const uint64_t ck = order(lane < a.k ? s + (double)a.bias[id] : 0.0);
        uint32_t rank = 0;
        for (uint32_t j = 0; j < a.k; ++j) {
            const uint64_t o = read_lane(ck, j);
            rank += o > ck || (o == ck && read_lane(id, j) < id) ? 1u : 0u;
        }
        /* lane j takes the selection of rank j */
        const int to = (int)(lane < a.k ? rank : lane) * 4;
        id = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)id);
        const uint64_t sb = __builtin_bit_cast(uint64_t, s);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)sb);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)(sb >> 32));
        s = __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    }
    write_row(a, row, lane, id, s);
    return true;
}

/* WAVES rows per workgroup, PER = ceil(E / 64) to a power of two. */
template <int PER, int WAVES, bool BIAS, bool SIGMOID>
__global__ __launch_bounds__(64 * WAVES) void route_group_kernel(GroupArgs a) {
    __shared__ double keys[WAVES][PER * 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x * WAVES + wave;
    if (row >= a.t) return;
    const float *l = a.logits + (uint64_t)row * a.e;
    float x[PER], b[PER];
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t e = lane + 64 * i;
        x[i] = l[e < a.e ? e : a.e - 1];
        b[i] = BIAS ? a.bias[e < a.e ? e : a.e - 1] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        big = max(big, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
        if constexpr (BIAS) big = max(big, __builtin_bit_cast(uint32_t, b[i]) & 0x7FFFFFFFu);
    }
    if (__ballot(big >= 0x7F800000u)) {
        refuse_row(a, row, lane, R9VX_STATUS_NONFINITE);
        return;
    }
    const bool huge = __ballot(big > 0x7E000000u) != 0; /* f32 sums of such biases may overflow */
    if (!huge && route_row<PER, BIAS, SIGMOID>(a, row, lane, x, b, reinterpret_cast<float *>(keys[wave]))) return;
    route_row<PER, BIAS, SIGMOID>(a, row, lane, x, b, keys[wave]);
}

template <int PER, int WAVES>
void launch_rows(const GroupArgs &a, hipStream_t stream) {
    const dim3 grid((a.t + WAVES - 1) / WAVES), block(64 * WAVES);
    const bool sigmoid = a.scoring == R9VX_SCORING_SIGMOID;
    if (a.bias && sigmoid)
        hipLaunchKernelGGL((route_group_kernel<PER, WAVES, true, true>), grid, block, 0, stream, a);
    else if (a.bias)
        hipLaunchKernelGGL((route_group_kernel<PER, WAVES, true, false>), grid, block, 0, stream, a);
    else if (sigmoid)
        hipLaunchKernelGGL((route_group_kernel<PER, WAVES, false, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((route_group_kernel<PER, WAVES, false, false>), grid, block, 0, stream, a);
}

template <int PER>
int launch_per(const GroupArgs &a, hipStream_t stream) {
    /* few rows: each on a CU of its own */
    if (a.t <= 1024)
        launch_rows<PER, 1>(a, stream);
    else
        launch_rows<PER, 4>(a, stream);
    return (int)hipGetLastError();
}

}  // namespace

int r9vx_launch_route_group(const r9vx_route_group_problem &p, hipStream_t stream) {
    const GroupArgs a{p.logits, p.bias,   p.ids,        p.weights, p.status,      p.t,           p.e,         p.k,
                      p.n_group, p.topk_group, p.e / p.n_group, ((1u << 22) + p.e / p.n_group - 1) / (p.e / p.n_group), p.scoring, p.renormalize, p.group_score, (double)p.scale};
    const uint32_t per = (p.e + 63) / 64;
    if (per <= 1) return launch_per<1>(a, stream);
    if (per <= 2) return launch_per<2>(a, stream);
    if (per <= 4) return launch_per<4>(a, stream);
    if (per <= 8) return launch_per<8>(a, stream);
    return launch_per<16>(a, stream);
}
