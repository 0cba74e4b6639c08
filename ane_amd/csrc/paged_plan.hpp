// paged_plan.hpp -- the host's side of paged attention: which kernel a call takes,
// over how many workgroups, its keys in how many parts; and the divisions whose
// constants the host works out.
#pragma once

#include <algorithm>

#include "paged.hpp"

namespace ane {

// x / d for x < 2^30 and d <= 2^16 as (x * magic) >> shift: with shift = 30 +
// ceil(log2 d) and magic = ceil(2^shift / d), at most 2^31, the excess magic * d -
// 2^shift is below d <= 2^(shift - 30), so x * excess < 2^shift and the floor is
// exact.  (A division the compiler spells out is some 40 instructions before a
// workgroup's first load.)
struct Div {
    uint32_t magic, shift;
    __host__ __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)((uint64_t)x * magic >> shift); }
};
inline Div div_by(uint32_t d) {
    uint32_t lg = 0;
    while ((1u << lg) < d) lg++;
    return Div{(uint32_t)(((1ull << (30 + lg)) + d - 1) / d), 30 + lg};
}

// One launch: which kernel, over how many row tiles, its keys in how many parts.
struct Launch {
    bool few, each;  // each: single tokens under a rule, a wave a (token, kv head)
    uint64_t slots;
    uint32_t chunk, parts;
};

// units: sequences (groups) of the launch; tokens: theirs in all; single: one
// token each; beside: shares its launch with the batch's own keys; bent: under a
// rule, its rows seeing many keys; windowed: its window leaves fewer keys than there are,
// max_len then a bound on those that a workgroup's rows see.
//
// 32 rows a workgroup as long as its workgroups have a place each (512 of them, two
// a CU; 64-wide four a CU, three in fp32), half again as many for one sequence,
// where 128 rows a workgroup would leave most CUs idle: 512 tokens x 32 heads fp32
// 22 us, 31 with 128 rows; 768 tokens 33, 39; 8 chunks of 64 tokens after 1000
// positions 36, 50.  Under a rule scores cost the vector unit more, which one workgroup
// of 128 rows a CU leaves idle between its waves' products: half again as many places (2
// x 300 tokens after 3000, capped, fp32 151 -> 108; 64-wide, 3 x 900 after 2000, fp32
// 135 -> 107, fp16 84 -> 75, behind a window of 1024 59 -> 53 and 38 -> 37; 3 x 500 31 ->
// 28; 1.7 times the places 6 x 777 38, 39), but not where there are few keys to share
// among the waves (2 x 1488 behind a window of 256 20, 24, behind 512 23, 25; 14 x 35
// tokens over as many keys 14, 20).
// Beyond that 128 rows, since the four waves of the other kernel read every K and
// V tile for themselves: 2 x 400 tokens 27 us, 30 with 32 rows; 16 x 256 tokens
// 49, 81.  Sequences of 64 rows and less would leave half of such a tile empty:
// single tokens, and 64 chunks of 16 tokens after 1000 positions (79 us, with 128
// rows 93).  Few rows and many keys: the keys in parts, as many as fill the
// places at once but not more: a second, part-filled round costs more than the
// longer parts (200 tokens after 4000 positions 51 us, in 1.5 times the parts 63).
// A prefix beside its batch's own keys takes half the places (three or four
// 64-wide workgroups fit a CU): 8 groups of 8 sequences 48 -> 42 us.  128-row
// workgroups are more than the CUs as it is, and their keys stay whole.  Behind a window
// rows have equally many keys, so two parts spread nothing more evenly than one: single
// tokens, which memory bounds, and short windows save the join (32 tokens behind 1024
// 31.4 -> 29.7 us, behind 4096 98.7 -> 94.7; 2 x 96 tokens behind 1024 26.2 -> 23.8, but
// 3 x 64 behind 4096 55 -> 62).
inline Launch plan(const ane_paged_cache* c, uint32_t units, uint64_t tokens, bool single, uint64_t max_len, bool beside = false,
                   bool bent = false, bool windowed = false) {
    Launch l = {};
    const uint64_t G = c->n_heads / c->n_kv_heads, rows = tokens * G;
    // of equally long sequences
    auto wgs = [&](uint64_t bm) { return (rows + units * bm - 1) / (units * bm) * units * c->n_kv_heads; };
    const uint64_t room = 512 * 128 / c->head_dim;
    l.few = single || wgs(32) <= (units == 1 || bent ? room + room / 2 : room) || wgs(32) < 3 * wgs(128);
    const uint64_t bm = l.few ? 32 : 128;
    l.slots = single ? units * ((G + bm - 1) / bm) : rows / bm + units;
    const uint64_t places = beside && c->head_dim == 128 ? 256 : 512;
    uint64_t n = std::max<uint64_t>(1, l.few ? std::min(places / wgs(32), (max_len + 255) / 256) : 1);
    if (windowed && n == 2 && (single || max_len <= 2048)) n = 1;
    l.chunk = (uint32_t)(((max_len + n - 1) / n + 127) / 128 * 128);
    l.parts = (uint32_t)((max_len + l.chunk - 1) / l.chunk);
    return l;
}

inline uint64_t bound_len(const ane_paged_cache* c, uint32_t max_len) {
    return max_len == 0 || max_len > page_cap(c) ? page_cap(c) : max_len;
}

// A batch of single tokens.  each: a wave a (token, kv head), without a merge,
// where there are 1024 of them and more and few keys each: 512 tokens over 30-100
// positions 64 -> 37 us, 256 over 300 51 -> 44; over 1000 121 -> 126.  Behind a prefix
// the bounds say how few keys a row may have of its own, not how many: one in no group
// has all of max_len, one wave after the other 32 of them.  So also max_len is at most
// 1536, where that costs as much as it saves (256 sequences with 100 own positions
// behind 1024 56 -> 40 us; 120 such and 8 alone with 1024 44 -> 57, behind 2048 54 ->
// 96, behind 8192 128 -> 328).
inline bool each_pays(const ane_paged_cache* c, const Launch& l, uint64_t len) {
    return l.parts == 1 && l.slots * c->n_kv_heads >= 1024 && len <= 512;
}
struct SharedPlan {
    Launch prefix, own;
    uint32_t parts;
    bool each;
};
inline SharedPlan shared_plan(const ane_paged_cache* c, uint32_t n, uint32_t n_groups, uint32_t max_prefix, uint32_t max_len) {
    SharedPlan p = {};
    const uint64_t len = bound_len(c, max_len), prefix = n_groups ? std::min(len, bound_len(c, max_prefix)) : 0;
    p.own = plan(c, n, n, true, len);
    if (n_groups) p.prefix = plan(c, n_groups, n, false, bound_len(c, max_prefix), true);
    p.parts = p.prefix.parts + p.own.parts;
    p.each = each_pays(c, p.own, len - prefix) && len <= 1536;
    return p;
}

}  // namespace ane
