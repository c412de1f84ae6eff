/*
 * r9vx_attn_index.h -- where the attention kernels read and write: plain integer
 * functions that a host compiler takes too, so that their bounds are tested
 * without a GPU.
 */
#ifndef R9VX_ATTN_INDEX_H
#define R9VX_ATTN_INDEX_H

#include <stdint.h>

#ifdef __HIPCC__
#define R9VX_HD __host__ __device__ __forceinline__
#else
#define R9VX_HD inline
#endif

namespace r9vx {

constexpr uint32_t kAttnNoWindow = 1u << 30; /* no sequence is longer */

/* The keys [lo, hi) that the token at position p < 2^30 of a sequence of `length`
 * tokens sees through a window of 1 .. 2^30: 0 <= lo, 0 <= hi <= length; none where
 * lo >= hi. */
R9VX_HD void attn_seen(uint32_t window, uint32_t causal, int p, int length, int start, int prefix, int &lo, int &hi) {
    lo = start > 0 ? start : 0;
    const int w = (int)((uint32_t)p - window + 1u);
    if (p >= 0 && w > lo) lo = w;
    hi = length;
    if (causal) {
        const int last = prefix > p + 1 ? prefix : p + 1;
        if (last < hi) hi = last;
    }
    if (p < 0 || hi < 0) hi = 0; /* p < 0: more new tokens than the sequence holds */
}

/* row / group as a product: magic = ceil(2^31 / group), exact while row * group < 2^31. */
R9VX_HD uint32_t attn_group_magic(uint32_t group) { return (uint32_t)(((1ull << 31) + group - 1) / group); }
R9VX_HD int attn_token(int row, uint32_t magic) { return (int)((uint64_t)(uint32_t)row * magic >> 31); }

/* Where a key's row is: in the cache, nowhere (zeros; not in [from, to)), or in a
 * page that the cache does not have (NaN). */
enum AttnPlace { kAttnKept, kAttnNone, kAttnBad };
R9VX_HD AttnPlace attn_place(uint32_t page, uint32_t pages, int key, int from, int to) {
    if (key < from || key >= to) return kAttnNone;
    return page < pages ? kAttnKept : kAttnBad;
}

/* Part `split` of the blocks [b0, b1) (of 0 .. 2^26) of a row's keys: the blocks over
 * `parts`, in whole `unit`s, at most `most` (whole units) of them.  Enough of them
 * cover every block: ceil((b1 - b0) / most) and at least `parts`. */
R9VX_HD void attn_part(int b0, int b1, uint32_t unit, uint32_t parts, uint32_t most, uint32_t split, int &begin, int &end) {
    const uint32_t n = (uint32_t)(b1 - b0), share = parts == 1 ? n : (n + parts - 1) / parts;
    const uint32_t whole = (share + unit - 1) / unit * unit, per = whole < most ? whole : most;
    const uint64_t first = (uint64_t)split * per, last = first + per;
    begin = b0 + (int)(first < n ? first : n);
    end = b0 + (int)(last < n ? last : n);
}

/* Prefill's rows of a sequence are cut into tiles of `rows`; sequence i's tiles
 * start at floor(offset[i] * group / rows) + i, which leaves each of them enough
 * without a scan: ceil(n group / rows) <= floor((o + n) group / rows) -
 * floor(o group / rows) + 1.  Offsets outside [0, t] are taken as its ends. */
R9VX_HD int attn_offset(const int32_t *offsets, uint32_t i, uint32_t t) {
    const int x = offsets[i];
    return x < 0 ? 0 : (uint32_t)x > t ? (int)t : x;
}
R9VX_HD uint32_t attn_first_tile(const int32_t *offsets, uint32_t i, uint32_t t, uint32_t group, uint32_t rows) {
    return (uint32_t)((uint64_t)attn_offset(offsets, i, t) * group / rows) + i;
}
R9VX_HD uint32_t attn_tiles(uint64_t t, uint32_t b, uint32_t group, uint32_t rows) { return (uint32_t)(t * group / rows) + b; }

/* The sequence, its first row of q, its number of rows, and where in them (token
 * times group + head) the tile begins; false where the tile has none. */
struct AttnTile {
    uint32_t b, row;
    int offset, n;
};
R9VX_HD bool attn_tile(const int32_t *offsets, uint32_t b, uint32_t t, uint32_t group, uint32_t rows, uint32_t tile, AttnTile &at) {
    at.b = 0;
    uint32_t step = 1;
    while (step < b) step <<= 1;
    for (; step; step >>= 1)
        if (at.b + step < b && attn_first_tile(offsets, at.b + step, t, group, rows) <= tile) at.b += step;
    at.offset = attn_offset(offsets, at.b, t);
    at.n = attn_offset(offsets, at.b + 1, t) - at.offset;
    const uint32_t first = attn_first_tile(offsets, at.b, t, group, rows);
    if (at.n <= 0 || tile < first) return false;
    const uint64_t row = (uint64_t)(tile - first) * rows;
    at.row = (uint32_t)row;
    return row < (uint64_t)at.n * group;
}

}  // namespace r9vx

#endif
