// Checks the index functions of the attention kernels against their bounds and
// plain counterparts, over random and hostile inputs.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "r9vx_attn_index.h"

using namespace r9vx;

#define CHECK(x)                                               \
    do {                                                       \
        if (!(x)) {                                            \
            printf("line %d: %s\n", __LINE__, #x);             \
            exit(1);                                           \
        }                                                      \
    } while (0)

static const int kHostile[] = {INT32_MIN, INT32_MIN + 1, -(1 << 30), -77, -1, 0, 1, 2, 31, 32, 33, 100, 1 << 20, 1 << 30, INT32_MAX - 8, INT32_MAX};

int main() {
    std::mt19937 rng(1);
    auto any = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };

    // seen: against the definition, and inside [0, length) whatever the data
    for (int i = 0; i < 400000; ++i) {
        const int length = any(0, 40), p = any(-3, 45), start = any(-5, 50), prefix = any(-5, 50), window = any(0, 1) ? any(1, 45) : (int)kAttnNoWindow, causal = any(0, 1);
        int lo, hi;
        attn_seen(window, causal, p, length, start, prefix, lo, hi);
        for (int j = -2; j < 60; ++j) {
            const bool want = p >= 0 && j >= 0 && j < length && j >= start && j > p - window && (!causal || j <= p || j < prefix);
            CHECK((j >= lo && j < hi) == want);
        }
    }
    for (int start : kHostile)
        for (int prefix : kHostile)
            for (uint32_t window : {1u, 100u, 1u << 29, (1u << 30) - 1, kAttnNoWindow})
                for (int length : {0, 1, 1 << 20, 1 << 30})
                    for (int back : {1, 2, 7, 1 << 24})
                        for (uint32_t causal : {0u, 1u}) {
                            int lo, hi;
                            attn_seen(window, causal, length - back, length, start, prefix, lo, hi);
                            CHECK(lo >= 0 && hi >= 0 && hi <= length);
                        }

    // tokens of decode's rows: 8 tokens of up to 1024 heads
    for (int group = 1; group <= 1024; ++group)
        for (int row = 0; row < 8 * group + 32; ++row) CHECK(attn_token(row, attn_group_magic(group)) == row / group);

    // places: a key outside [from, to) or a page outside the cache is never kept
    for (uint32_t page : {0u, 1u, 9u, 10u, 0x7FFFFFFFu, 0x80000000u, 0xFFFFFFFFu})
        for (int key : kHostile)
            for (int from : {0, 5, 32})
                for (int to : {0, 5, 33}) {
                    const AttnPlace x = attn_place(page, 10, key, from, to);
                    CHECK((x == kAttnNone) == (key < from || key >= to));
                    CHECK(x != kAttnKept || page < 10);
                }

    // parts: every block once, in order, whole units, none over the most
    for (int i = 0; i < 200000; ++i) {
        const int b0 = any(0, 1 << 25), b1 = b0 + (any(0, 3) ? any(0, 300) : any(0, 1 << 25)), unit = any(0, 1) ? 1 : 4;
        const int parts = any(0, 2) ? any(1, 8) : any(1, 256), n = b1 - b0;
        int most = unit * any(1, 64);
        if ((n + most - 1) / most > 1000) most = (n / 900 + 1) * unit;
        const int splits = std::max(parts, (n + most - 1) / most);
        int at = b0;
        for (int s = 0; s < splits; ++s) {
            int begin, end;
            attn_part(b0, b1, unit, parts, most, s, begin, end);
            CHECK(begin <= end && begin >= b0 && end <= b1 && begin == at && end - begin <= most);
            CHECK((begin - b0) % unit == 0 || begin == b1);
            at = end;
        }
        CHECK(at == b1);
    }

    // tiles of packed sequences: every row of each of them once
    for (int i = 0; i < 4000; ++i) {
        const uint32_t group = any(1, 40), rows = 128, b = any(1, 12);
        std::vector<int32_t> off(b + 1);
        off[0] = any(0, 3) ? 0 : any(0, 50);
        for (uint32_t s = 0; s < b; ++s) off[s + 1] = off[s] + (any(0, 2) ? any(0, 90) : 0);
        const uint32_t t = off[b] + (any(0, 1) ? any(0, 60) : 0);
        std::vector<std::vector<int>> hit(b);
        for (uint32_t s = 0; s < b; ++s) hit[s].assign((off[s + 1] - off[s]) * group, 0);
        for (uint32_t tile = 0; tile < attn_tiles(t, b, group, rows); ++tile) {
            AttnTile x;
            if (!attn_tile(off.data(), b, t, group, rows, tile, x)) continue;
            CHECK(x.b < b && x.offset == off[x.b] && x.n == off[x.b + 1] - off[x.b]);
            for (uint32_t r = x.row; r < x.row + rows && r < (uint32_t)x.n * group; ++r) hit[x.b][r]++;
        }
        for (auto &h : hit)
            for (int n : h) CHECK(n == 1);
    }
    // offsets that are none: rows stay inside q
    for (int i = 0; i < 100000; ++i) {
        const uint32_t group = any(0, 1) ? any(1, 1024) : 1, b = any(1, 9), t = any(0, 3) ? any(0, 300) : any(0, 1 << 20);
        std::vector<int32_t> off(b + 1);
        for (auto &x : off) x = any(0, 2) ? any(0, (int)t) : kHostile[any(0, 15)];
        const uint32_t tiles = attn_tiles(t, b, group, 128);
        for (int k = 0; k < 20; ++k) {
            const uint32_t tile = any(0, (int)tiles - 1);
            AttnTile x;
            if (!attn_tile(off.data(), b, t, group, 128, tile, x)) continue;
            CHECK(x.b < b && x.offset >= 0 && x.n > 0 && (int64_t)x.offset + x.n <= (int64_t)t && x.row < (uint64_t)x.n * group);
        }
    }
    printf("ok\n");
    return 0;
}
