// paged_attention.hip -- attention over the paged K/V cache: causal prompts of
// packed sequences, and batches of single tokens that may share a prefix.
//
// One pass over the keys with the running maximum and sum of the softmax.  The
// query heads of a kv head's group and the tokens of a sequence form the rows of
// one matrix (row = token * G + head), so every K and V row is read once for
// all of them.  With 32 rows a wave and 32-key blocks, the products are
//   S^T = K . Q^T      v_mfma_f32_32x32x16_f16, A = K rows, B = Q rows
//   O^T += V^T . P^T   A = V^T, B = P^T
// transposed so that a query row is a column of every accumulator: lane r and
// lane r + 32 hold row r, its maximum and sum need one exchange between the two,
// its rescaling is one factor a lane, and the lane's 8 weights of a 16-key step
// are exactly the B operand of the second product when that step's keys are
// numbered k(half, j) = 8 (j / 4) + 4 half + j % 4.  V^T comes out of row-major V
// in LDS through the transposing read ds_read_b64_tr_b16: four keys of one
// dimension a lane, two reads a step in the same numbering.
//
// fp32 activations: q and the weights enter as two fp16 parts each (hi + lo, 22
// bits), twice the matrix instructions.  A q row is scaled by a power of two to a
// maximum in [2^13, 2^14) first, so any fp32 range fits fp16 (K is fp16 already,
// products and sums are fp32).
#include <math.h>

#include <algorithm>

#include "paged_plan.hpp"

namespace ane {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __fp16 hh2 __attribute__((ext_vector_type(2)));  // (what the dot product's builtin takes)
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s4* lds_s4;

enum Mode { kPrompt, kPrefix, kOwn };

struct AttnArgs {
    const void* q;
    void* out;
    float *po, *pml;          // partials: [part][row][hd] and [part][row](max, sum); row = token * n_heads + head
    const uint16_t *kp, *vp;  // this layer's pages
    const uint32_t *table, *kv_len, *seqs, *q_start, *group_start, *prefix;
    uint64_t q_stride, out_stride;
    uint32_t n, n_tokens, n_groups, n_heads, n_kv, G, ps, n_pages, max_pages, n_seqs;
    Div by_page, by_G, by_kv;      // 16-position group -> page, row -> token, workgroup -> row tile
    struct Parts {
        uint32_t chunk, n, first;  // keys a part, parts, number of the first
    } own, pre;                    // of a row's own keys (all of a prompt's), of the shared prefix
    uint32_t parts_total;
    float scale_log2e;
    // A rule (ane_decode.h), in kernels with RULE: cap and 1 / cap in log2 units
    // (0: none), slopes by head, window (0: none), the first position each token
    // sees, the prefix each batch row sees whole (null: none).
    float cap, inv_cap;
    float bend[3];  // fp16: Tanh's coefficients for scores as the products give them, or zeros
    uint32_t window;
    const float* slopes;
    const uint32_t *first, *seen;

    template <int MODE>
    __device__ __forceinline__ const Parts& parts() const { return MODE == kPrefix ? pre : own; }
};

// No branches: a load in flight next to the others costs less than its test.
__device__ __forceinline__ uint32_t seq_id(const AttnArgs& a, uint32_t s) { return a.seqs ? a.seqs[s] : s; }
__device__ __forceinline__ uint32_t raw_len(const AttnArgs& a, uint32_t id) { return a.kv_len[min(id, a.n_seqs - 1)]; }
__device__ __forceinline__ uint32_t seq_len(const AttnArgs& a, uint32_t id, uint32_t raw) {
    return id < a.n_seqs ? (uint32_t)min((uint64_t)raw, (uint64_t)a.max_pages * a.ps) : 0;
}
__device__ __forceinline__ uint32_t seq_len(const AttnArgs& a, uint32_t id) { return seq_len(a, id, raw_len(a, id)); }
__device__ __forceinline__ uint32_t lane_of(uint32_t x, uint32_t lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ uint32_t last_lane(bool yes) {  // the last lane that says yes, 0 if none
    const uint64_t m = __ballot(yes);
    return m ? 63 - (uint32_t)__builtin_clzll(m) : 0;
}

// What a workgroup computes: BM rows of one kv head of one batch row (of one
// group in kPrefix), keys [kbeg, kend) from the pages of sequence id.  All of it
// is wave-uniform and goes through v_readfirstlane: the compiler has to be told,
// or each copy to LDS loops over its lanes' (equal) descriptors.
struct Work {
    uint32_t s, id, tok0, toks, row0, rows;  // batch row or group, sequence, first token, tokens, first row, rows in all
    int32_t kbeg, kend, lo, len;             // lo: keys before it are masked (kbeg rounds it down to 16)
    bool alone;                              // kOwn: no group has the row
    uint32_t raw, prefix;                    // as loaded: the sequence's length, the group's prefix
};

__device__ __forceinline__ void uniform(uint32_t& x) { x = __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ void uniform(int32_t& x) { x = __builtin_amdgcn_readfirstlane(x); }

// The rows of slot `slot`.  Row tiles of batch row s are slots start[s] * G / BM
// + s onwards (floor), which never overlap; what is left between is empty.
template <int MODE, int BM>
__device__ __forceinline__ bool find_rows(const AttnArgs& a, uint32_t slot, Work& w) {
    const uint32_t* start = MODE == kPrefix ? a.group_start : MODE == kPrompt ? a.q_start : nullptr;
    const uint32_t n = MODE == kPrefix ? a.n_groups : a.n, lane = threadIdx.x & 63;
    uint32_t tile, first, end;
    if (start) {
        auto key = [&](uint32_t from, uint32_t i) { return (uint64_t)from * a.G / BM + i; };
        uint32_t base = 0;  // the 64 entries from `base` hold the row
        if (n > 63) {
            base = wave_search(n, slot, [&](uint32_t i) { return key(start[i], i); });
            base = base > 31 ? base - 31 : 0;
        }
        const uint32_t v = start[min(base + lane, n)];
        const uint32_t l = last_lane(base + lane < n && key(v, base + lane) <= slot);
        w.s = base + l, first = lane_of(v, l), end = min(lane_of(v, l + 1), a.n_tokens);
        const uint64_t k = key(first, w.s);
        if (k > slot) return false;
        tile = slot - (uint32_t)k;
    } else {
        const uint32_t tiles = (a.G + BM - 1) / BM;
        w.s = slot / tiles, tile = slot % tiles;
        if (w.s >= n) return false;
        first = w.s, end = w.s + 1;
    }
    w.tok0 = first, w.toks = end > first ? end - first : 0;
    w.rows = w.toks * a.G;  // below 2^30
    w.row0 = tile * BM;
    if (tile >= (1u << 24) || w.row0 >= w.rows) return false;
    w.id = seq_id(a, MODE == kPrefix ? w.tok0 : w.s);
    w.raw = raw_len(a, w.id);
    if (MODE == kPrefix) w.prefix = a.prefix[w.s];
    uniform(w.s), uniform(w.id), uniform(w.tok0), uniform(w.toks), uniform(w.row0), uniform(w.rows);
    return true;
}

// The positions batch row s shares with its group; alone: it is in none.
__device__ __forceinline__ uint32_t shared_len(const AttnArgs& a, uint32_t s, uint32_t len, bool& alone) {
    alone = true;
    if (a.n_groups == 0) return 0;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0;
    if (a.n_groups > 63) {
        base = wave_search(a.n_groups, s, [&](uint32_t i) { return (uint64_t)a.group_start[i]; });
        base = base > 31 ? base - 31 : 0;
    }
    const uint32_t v = a.group_start[min(base + lane, a.n_groups)], p = a.prefix[min(base + lane, a.n_groups - 1)];
    const uint32_t l = last_lane(base + lane < a.n_groups && v <= s), first = lane_of(v, l);
    if (first > s || s >= lane_of(v, l + 1)) return 0;
    alone = false;
    return min(min(lane_of(p, l), len), seq_len(a, seq_id(a, first)));
}

// The first position token t of the work's sees under a rule.
__device__ __forceinline__ int32_t rule_first(const AttnArgs& a, const Work& w, uint32_t t) {
    const int32_t pos = w.len - (int32_t)w.toks + (int32_t)t;
    int32_t lo = a.window ? max(pos + 1 - (int32_t)a.window, 0) : 0;
    if (a.first) lo = max(lo, (int32_t)min(a.first[w.tok0 + t], 0x7fffffffu));
    return lo;
}
// The end of what they see, whatever the token (none below 1, a negative entry among them).
__device__ __forceinline__ int32_t rule_seen(const AttnArgs& a, const Work& w) {
    return a.seen ? min((int32_t)a.seen[w.s], w.len) : 0;
}

// The keys of part `part`.
template <int MODE, bool RULE = false>
__device__ __forceinline__ void find_keys(const AttnArgs& a, uint32_t bm, uint32_t part, Work& w) {
    w.len = (int32_t)seq_len(a, w.id, w.raw);
    w.kbeg = w.lo = 0;
    w.kend = w.len;
    w.alone = true;
    if (MODE == kPrompt) {
        const int32_t last = (int32_t)a.by_G(min(w.row0 + bm, w.rows) - 1);
        w.kend = min(w.len, w.len - (int32_t)w.toks + last + 1);
        if constexpr (RULE) {
            const int32_t tok = (int32_t)a.by_G(w.row0);
            if (w.kend > 0) w.kend = max(w.kend, rule_seen(a, w));
            int32_t lo = a.window ? max(w.len - (int32_t)w.toks + tok + 1 - (int32_t)a.window, 0) : 0;
            if (a.first) {  // the least of the tile's tokens (at most 128): what none of them sees is not read
                uint32_t f = 0xffffffffu;
                for (int32_t t = tok + (int32_t)(threadIdx.x & 63); t <= last; t += 64) f = min(f, a.first[w.tok0 + t]);
#pragma unroll
                for (int x = 32; x >= 1; x >>= 1) f = min(f, (uint32_t)__shfl_xor((int)f, x, 64));
                lo = max(lo, (int32_t)min(f, 0x7fffffffu));
            }
            w.kbeg = min(lo, max(w.kend, 0)) & ~15;
        }
    } else if (MODE == kPrefix) {
        w.kend = (int32_t)min(w.prefix, (uint32_t)w.len);
    } else {
        w.lo = (int32_t)shared_len(a, w.s, (uint32_t)w.len, w.alone);
        w.kbeg = w.lo & ~15;
        if (w.lo >= w.kend) w.kend = w.kbeg;
    }
    const int64_t b = w.kbeg + (int64_t)part * a.parts<MODE>().chunk;
    if (part + 1 < a.parts<MODE>().n) w.kend = (int32_t)min((int64_t)w.kend, b + a.parts<MODE>().chunk);
    w.kbeg = (int32_t)min(b, (int64_t)max(w.kend, 0));
    uniform(w.kbeg), uniform(w.kend), uniform(w.lo), uniform(w.len);
}
// Whether the first key's position is known before any length is.
template <int MODE, bool RULE = false>
__device__ __forceinline__ bool early_keys(const AttnArgs& a) { return !RULE && (MODE != kOwn || a.n_groups == 0); }

// Keys of the work a row (token t of the work's) sees: those below.
template <int MODE, bool RULE = false>
__device__ __forceinline__ int32_t row_limit(const AttnArgs& a, const Work& w, uint32_t t) {
    int32_t l = w.len;
    if (MODE == kPrompt) l += (int32_t)t + 1 - (int32_t)w.toks;
    if (RULE && l > 0) l = max(l, rule_seen(a, w));
    if (MODE == kPrefix) l = (int32_t)seq_len(a, seq_id(a, w.tok0 + t));
    return min(l, w.kend);
}

// LDS tiles: rows of HD fp16, 16-byte chunk c of row r in slot c ^ swz(r).  A K
// fragment reads one chunk of 16 consecutive rows at a time, a V fragment four
// chunks of four consecutive rows: both then touch every bank once.
template <int HD>
__device__ __forceinline__ uint32_t swz(uint32_t r) {
    return HD == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Copies of 16-position groups of K and V to LDS.  Page numbers are looked up 64
// groups at a time, one a lane, and handed out with v_readlane: a group is
// whole within its page, so the copy's base and extent are scalars.  Rows from
// kend on, and whole groups on a broken page number, land as zeros.
template <int HD>
struct Loader {
    static constexpr uint32_t RB = HD * 2, kRows = 1024 / RB, kCopies = 16 / kRows;
    uint32_t off[kCopies];
    uint32_t ids;

    __device__ __forceinline__ void init() {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (uint32_t i = 0; i < kCopies; i++) {
            const uint32_t r = i * kRows + lane / (RB / 16);
            off[i] = r * RB + (((lane % (RB / 16)) ^ swz<HD>(r)) << 4);
        }
    }
    __device__ __forceinline__ uint32_t page(const AttnArgs& a, uint32_t u) const {
        return a.by_page(u);
    }
    // u: this lane's 16-position group
    __device__ __forceinline__ void lookup(const AttnArgs& a, uint32_t id, uint32_t u) {
        const uint32_t p = min(page(a, min(u, (1u << 27) - 1)), a.max_pages - 1);
        ids = a.table[(uint64_t)min(id, a.n_seqs - 1) * a.max_pages + p];
    }
    // the wait for the numbers here, not before each copy that follows
    __device__ __forceinline__ void settle() { asm volatile("" : "+v"(ids)); }
    // 16 rows of x from group u (wave-uniform) on, whose page number is in lane `from`, of kv head g
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t group(const AttnArgs& a, const uint16_t* x, const Work& w, uint32_t g,
                                                            uint32_t u, uint32_t from) const {
        const uint32_t id = __builtin_amdgcn_readlane(ids, from);
        const uint32_t row = u * 16 - page(a, u) * a.ps;
        const int32_t left = w.kend - (int32_t)(u * 16);
        // (a clamp goes through the vector ALU: back to a scalar, as above)
        const uint32_t bytes = __builtin_amdgcn_readfirstlane(id < a.n_pages ? (uint32_t)min(max(left, 0), 16) * RB : 0);
        const uint64_t at = (((uint64_t)(id < a.n_pages ? id : 0) * a.n_kv + g) * a.ps + row) * HD;
        return make_rsrc(x + at, bytes);
    }
    // 1 KB of such a group (nt: of keys no other workgroup reads)
    template <bool NT = false>
    __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, uint32_t i, uint8_t* dst) const {
        if constexpr (NT) copy16_to_lds_nt(r, dst + i * 1024, off[i]);
        else copy16_to_lds(r, dst + i * 1024, off[i]);
    }
    template <bool NT = false>
    __device__ __forceinline__ void copy(const AttnArgs& a, const uint16_t* x, const Work& w, uint32_t g, uint32_t u,
                                         uint32_t from, uint8_t* dst) const {
        const __amdgpu_buffer_rsrc_t r = group(a, x, w, g, u, from);
#pragma unroll
        for (uint32_t i = 0; i < kCopies; i++) copy<NT>(r, i, dst);
    }
};

__device__ __forceinline__ float other_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ h8 as_h8(v4i x) {
    h8 r;
    __builtin_memcpy(&r, &x, 16);
    return r;
}

// The transposing read.  Its pointer is restrict for the alias information that
// leaves on the read once inlined: without any, the compiler waits for every
// copy to LDS in flight first.
__device__ __forceinline__ s4 read_tr(const uint8_t* __restrict__ p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
}

// x as two fp16 parts, 22 bits in all; rest: x - hi.
__device__ __forceinline__ void split(f2 x, h2& hi, h2& lw, f2& rest) {
    hi = __builtin_convertvector(x, h2);
    // with hi read as fp16: one instruction a value
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest.x) : "v"(hi), "v"(x.x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rest.y) : "v"(hi), "v"(x.y));
    lw = __builtin_convertvector(rest, h2);
}
__device__ __forceinline__ void split(f2 x, h2& hi, h2& lw) {
    f2 rest;
    split(x, hi, lw, rest);
}

// Weights are e^s 2^kLift relative to a reference m, a maximum that may lag by
// kLag (in log2) before O and l are rescaled: at most 2^(kLag + kLift) = 2^14 in
// fp16 mode, 2^15 in fp32 mode.
//
// fp16 mode: a weight is rounded to fp16 once, with full precision down to 2^-20 of
// the largest and as a multiple of 2^-30 of it below.
//
// fp32 mode: two parts hold 22 bits of a weight of 2^-3 and more, below that a
// multiple of 2^-24, which is enough for fp32 accuracy as long as larger weights
// carry the row.  They need not: a key far above the others may hold a value of
// zeros.  So
// - the reference also goes down, to the maximum of a tile kDrop below it, but not
//   more than kDeep below the largest seen (O grows by as much);
// - a tile with weights below 2^kThin is looked at again: where 2^-25 a key and its
//   largest value are not below 2^-19 of what the row has summed up, what the two
//   parts left of the weights goes through the matrix cores too, 2^kAgain larger.
// Weights that matter so keep 18 bits down to 2^-56 of the row's largest, and are
// multiples of 2^-73 of it below.  O stays below 2^(15 + kDeep + kAgain) 2^16 a key:
// 2^30 keys fit fp32.
// The price (prompts of 250-1023 tokens x 32 heads, in a graph): 128 -> 133 us with
// scores of deviation 1.5, 122 -> 137 with a key 14 above the others, and with scores
// of deviation 3, where most tiles have such weights, 128 -> 163; with all of those
// through the matrix cores 192.  A lag of 3 instead of 4 rescales O so often that
// the first takes 137.
constexpr float kDrop = 8.0f, kDeep = 24.0f, kThin = -7.0f, kAgain = 38.0f;

// tanh(y) = y + y z P(z), z = y^2, up to |y| = kSmall (P fitted here for the least
// relative error: 2^-23.8 with five coefficients to 0.6, in fp32 arithmetic; 2^-20.5
// with three to 0.5, below what fp16 weights are rounded by), beyond that as 1 - 2 /
// (1 + e^2y), there exact to 2^-22.  A cap is chosen well above most scores, so most
// tiles are all small, and P costs half of what exponential and reciprocal do.  fp16
// rows share their factor, so P takes the scores as they are (8192 tokens x 32 heads
// behind a window of 1024 207 -> 197 us, without a window 720 -> 674; uncapped 171, 570).
template <bool F32>
struct Tanh {
    static constexpr float kSmall = F32 ? 0.6f : 0.5f;
    static constexpr float kHalf[3] = {-0.33328157663f, 0.13205355406f, -0.04475053400f};
    // tanh(y) / y - 1
    static __device__ __forceinline__ float small(float y) {
        const float z = y * y;
        float p;
        if constexpr (F32) {
            p = -0.0058951363f;
            p = __builtin_fmaf(p, z, 0.02079595252f);
            p = __builtin_fmaf(p, z, -0.0537838228f);
            p = __builtin_fmaf(p, z, 0.13331924378f);
            p = __builtin_fmaf(p, z, -0.3333329856f);
        } else {
            p = __builtin_fmaf(kHalf[2], z, kHalf[1]);
            p = __builtin_fmaf(p, z, kHalf[0]);
        }
        return p * z;
    }
    static __device__ __forceinline__ float large(float y) {
        const float e = __builtin_amdgcn_exp2f(y * 2.88539008177792681f);
        return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
    }
};

// 32 rows of a wave: lane & 31 is the row, lane >> 5 the half of its keys (of its
// dimensions in q and O).  RULE: scores capped, lowered with the distance, keys before
// a row's own first one masked (ane_decode.h).
template <int HD, bool F32, bool RULE = false>
struct Rows {
    static constexpr int NS = HD / 16, ND = HD / 32;
    static constexpr uint32_t RB = HD * 2;
    h8 qh[NS], ql[F32 ? NS : 1];  // q, its low part
    static constexpr float kLag = F32 ? 4.0f : 8.0f, kLift = F32 ? 11.0f : 6.0f;
    f16v o[ND];
    float m, l, c;  // reference (log2), this half's sum, score factor
    float peak, bottom;  // fp32: the largest reference so far; a tile's maximum below it takes the reference down
    float lost;          // fp32: largest value times keys, of the small weights left in two parts
    int32_t lim;    // keys below it are seen
    int32_t wmin, wmax;
    uint32_t half, ka, va[2 * ND];
    // RULE: keys before `begin` are masked (least and largest of the rows below), the
    // row's position and slope (log2 units), the score factor: c is 1 where there are
    // slopes, scores then are in log2 units already.
    int32_t begin, fmin, fmax, pos;
    float slope, factor;

    __device__ __forceinline__ void init_rule(const AttnArgs& a, const Work& w, uint32_t t, uint32_t head, bool live) {
        pos = w.len - (int32_t)w.toks + (int32_t)t;
        begin = rule_first(a, w, t);
        fmin = live ? begin : 0x7fffffff, fmax = live ? begin : 0;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            fmin = min(fmin, __shfl_xor(fmin, x, 64));
            fmax = max(fmax, __shfl_xor(fmax, x, 64));
        }
        fmin = __builtin_amdgcn_readfirstlane(fmin);
        fmax = __builtin_amdgcn_readfirstlane(fmax);
        slope = a.slopes ? a.slopes[head] * 1.44269504088896341f : 0.0f;
    }
    // after take_q
    __device__ __forceinline__ void init_factor(const AttnArgs& a) {
        // (in reach of 1 / cap: scores of a factor above 2^100 caps are zero or at the cap)
        if (a.cap != 0.0f) c = fminf(c, a.cap * 0x1p100f);
        factor = c;
        if (a.slopes) c = 1.0f;
    }
    // Scores as the products give them, capped: s tanh(y) / y with y = s factor / cap, in
    // the same units; then lowered with the distance, in log2 units.
    template <int KT>
    __device__ __forceinline__ void bend(const AttnArgs& a, f16v (&s)[KT], int32_t t0) const {
        if (a.cap != 0.0f) {  // uniform, as the next ones
            const float down = fmaxf(factor * a.inv_cap, 0x1p-126f);  // (as c in take_q: never 0)
            float top = 0.0f;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(top, fabsf(s[t][r])), fabsf(s[t][r + 1]));
            auto by_y = [&](float x) { return __builtin_fmaf(Tanh<F32>::small(x * down), x, x); };
            auto as_is = [&](float x) {  // fp16: the factor is one for all rows
                const float z = x * x;
                const float p = __builtin_fmaf(__builtin_fmaf(a.bend[2], z, a.bend[1]), z, a.bend[0]);
                return x * __builtin_fmaf(p, z, 1.0f);
            };
            auto all = [&](auto small) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[t][r] = small(s[t][r]);
            };
            // small scores as in a tile that has no others: which one it is hangs on keys
            // that a row does not see, and must not change what the row gets
            auto mixed = [&](auto small) {
                const float up = __builtin_amdgcn_rcpf(down);
                all([&](float x) {
                    const float l = Tanh<F32>::large(x * down) * up;
                    return fabsf(x * down) > Tanh<F32>::kSmall ? l : small(x);
                });
            };
            const bool some = __any(top * down > Tanh<F32>::kSmall);
            if constexpr (F32) {
                some ? mixed(by_y) : all(by_y);
            } else if (a.bend[0] == 0.0f) {
                mixed(by_y);
            } else {
                some ? mixed(as_is) : all(as_is);
            }
        }
        if (!a.slopes) return;
        if (a.seen) {  // keys on both sides of a row
            const float at = (float)(pos - t0 - 4 * (int32_t)half);
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    s[t][r] = __builtin_fmaf(-slope, fabsf(at - (float)(t * 32 + 8 * (r >> 2) + (r & 3))), s[t][r] * factor);
        } else {
            const float at = slope * (float)(t0 + 4 * (int32_t)half - pos);
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    s[t][r] = __builtin_fmaf(s[t][r], factor, __builtin_fmaf(slope, (float)(t * 32 + 8 * (r >> 2) + (r & 3)), at));
        }
    }

    __device__ __forceinline__ void init(float scale_log2e, int32_t limit, bool live) {
        const uint32_t lane = threadIdx.x & 63, i = lane & 15, grp = lane >> 4;
        half = lane >> 5;
        ka = lane & 31;
        const uint32_t low = (grp & 1) * 2 + ((i & 3) >> 1);
#pragma unroll
        for (uint32_t j = 0; j < 2; j++)
#pragma unroll
            for (uint32_t d = 0; d < ND; d++) {
                const uint32_t hi = HD == 128 ? d ^ (i >> 2) : d ^ (i >> 3);
                va[j * ND + d] = (4 * half + 8 * j + (i >> 2)) * RB + (((hi << 2) | (low ^ (half + 2 * j))) << 4) + (i & 1) * 8;
            }
        m = peak = bottom = -INFINITY, lost = 0.0f, l = 0.0f, c = scale_log2e;
        lim = live ? limit : 0;
        wmin = live ? limit : 0x7fffffff, wmax = lim;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            wmin = min(wmin, __shfl_xor(wmin, x, 64));
            wmax = max(wmax, __shfl_xor(wmax, x, 64));
        }
        wmin = __builtin_amdgcn_readfirstlane(wmin);
        wmax = __builtin_amdgcn_readfirstlane(wmax);
    }
    struct Raw {  // a row of q on its way
        v4i x[NS * (F32 ? 2 : 1)];
    };
    __device__ __forceinline__ void fetch_q(const void* q, uint64_t at, bool live, Raw& w) const {
        const uint32_t h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 2; e++)
                    w.x[2 * s + e] = *reinterpret_cast<const v4i*>(static_cast<const float*>(q) + at + 16 * s + 8 * h + 4 * e);
            } else {
                w.x[s] = *reinterpret_cast<const v4i*>(static_cast<const _Float16*>(q) + at + 16 * s + 8 * h);
            }
        }
        if (!live)
#pragma unroll
            for (auto& x : w.x) x = v4i{0, 0, 0, 0};
    }
    // The same by whole rows: the loads above touch 64 cache lines each, with 16 bytes
    // of every one, and all four waves of 32-row workgroups make them (a prompt of 128
    // tokens 13.6 -> 12.9 us in a graph; the few rows of single tokens share their
    // lines, and beside a busy second workgroup 128 rows take as long either way).
    // Load i takes RB bytes of kRows rows, for each of the P parts of a row; at: the
    // byte offset of lane & 31's row.
    static constexpr uint32_t kRows = 1024 / RB, kLoads = 32 / kRows, P = F32 ? 2 : 1;
    __device__ __forceinline__ void fetch_rows(const void* q, uint64_t at, Raw& w) const {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; i++) {
            const uint32_t r = i * kRows + lane / (RB / 16);
            const uint64_t row = (uint64_t)__shfl((uint32_t)(at >> 32), r, 64) << 32 | __shfl((uint32_t)at, r, 64);
            const uint8_t* p = static_cast<const uint8_t*>(q) + row + lane % (RB / 16) * 16;
#pragma unroll
            for (uint32_t k = 0; k < P; k++) w.x[k * kLoads + i] = *reinterpret_cast<const v4i*>(p + k * RB);
        }
    }
    // and through a tile of LDS to the lanes they belong to
    __device__ __forceinline__ void turn_rows(uint8_t* st, bool live, Raw& w) const {
        const uint32_t lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (uint32_t k = 0; k < P; k++) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; i++) {
                const uint32_t x = i * kRows + lane / (RB / 16);
                *reinterpret_cast<v4i*>(st + x * RB + (((lane % (RB / 16)) ^ swz<HD>(x & 15)) << 4)) = w.x[k * kLoads + i];
            }
#pragma unroll
            for (uint32_t j = 0; j < kLoads; j++) {
                const uint32_t c = F32 ? 4 * (j / 2) + 2 * h + j % 2 : 2 * j + h;
                w.x[k * kLoads + j] = *reinterpret_cast<const v4i*>(st + r * RB + ((c ^ swz<HD>(r & 15)) << 4));
            }
        }
        wait_lgkmcnt0();
        if (!live)
#pragma unroll
            for (auto& x : w.x) x = v4i{0, 0, 0, 0};
    }
    __device__ __forceinline__ void take_q(const Raw& w) {
        if constexpr (!F32) {
#pragma unroll
            for (int s = 0; s < NS; s++) {
                qh[s] = as_h8(w.x[s]);
                asm volatile("" : "+v"(qh[s]));  // the wait for q here, not in the loop
            }
#pragma unroll
            for (int e = 0; e < 8; e++) ql[0][e] = (_Float16)0.0f;
        } else {
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < 2 * NS; s++)
#pragma unroll
                for (int k = 0; k < 4; k++) top = fmaxf(top, fabsf(__int_as_float(w.x[s][k])));
            top = other_max(top);
            // 2^(140 - ex) brings the largest |q| (exponent field ex) to [2^13, 2^14)
            const uint32_t ex = max(__float_as_uint(top) >> 23, 20u);
            const float up = __uint_as_float((267 - ex) << 23);
            // (never 0 nor infinite: -inf, a masked score, and 0, that of a zero, times it stay as they are)
            c = __builtin_amdgcn_fmed3f(c * __uint_as_float((ex - 13) << 23), 0x1p-126f, 0x1p127f);
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const f2 v = {__int_as_float(w.x[2 * s + k / 4][k % 4]) * up, __int_as_float(w.x[2 * s + k / 4][k % 4 + 1]) * up};
                    h2 hi, lw;
                    split(v, hi, lw);
                    qh[s][k] = hi.x, qh[s][k + 1] = hi.y;
                    ql[s][k] = lw.x, ql[s][k + 1] = lw.y;
                }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    }
    __device__ __forceinline__ v4i vfrag(const uint8_t* v, int s, int d) const {
        const s4 a = read_tr(v + va[d] + s * 16 * RB);
        const s4 b = read_tr(v + va[ND + d] + s * 16 * RB);
        v4i r;
        __builtin_memcpy(&r, &a, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &b, 8);
        return r;
    }
    // Fragments are read kAhead products before their use and the order is
    // pinned: left alone, the scheduler reads all of them first and spills.
    static constexpr int kAhead = 4;
    // A wave in its products goes before the SIMD's other one in its weights: with
    // two parts a value the matrix unit is the busier one (4096 tokens x 32 heads
    // fp32 267 -> 253 us; fp16 the same either way).
    static __device__ __forceinline__ void products(bool on) {
        if constexpr (F32) on ? __builtin_amdgcn_s_setprio(1) : __builtin_amdgcn_s_setprio(0);
    }
    template <int KT>
    struct Weights {  // of 32 KT keys: the B operands of 16-key products
        h8 h[2 * KT], l[F32 ? 2 * KT : 1];
    };
    template <int KT, class Between>
    __device__ __forceinline__ void scores(const uint8_t* k, f16v (&s)[KT], Between between) const {
        const uint32_t kx = swz<HD>(ka & 15);
        auto frag = [&](int i) {  // products in the order (chunk e, block t)
            const int e = i / KT, t = i % KT;
            return as_h8(*reinterpret_cast<const v4i*>(k + (t * 32 + ka) * RB + (((2 * e + half) ^ kx) << 4)));
        };
        products(true);
        h8 kf[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) kf[i] = frag(i);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[t][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < NS * KT; i++) {
            const int e = i / KT, t = i % KT;
            s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % kAhead], qh[e], s[t], 0, 0, 0);
            if constexpr (F32) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % kAhead], ql[e], s[t], 0, 0, 0);
            if (i + kAhead < NS * KT) kf[i % kAhead] = frag(i + kAhead);
            between(i);
            __builtin_amdgcn_sched_barrier(0);
        }
        products(false);
    }
    template <int KT>
    __device__ __forceinline__ void mask(f16v (&s)[KT], int32_t t0, int32_t lo) const {
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int32_t key = t0 + t * 32 + 8 * (r >> 2) + 4 * (int32_t)half + (r & 3);
                if (key >= lim || key < lo || (RULE && key < begin)) s[t][r] = -INFINITY;
            }
    }
    // Scores of keys from position t0 on to weights; keys before lo are masked.
    // Whether this lane has some so small that carried() has to look at them.
    template <int KT, class Between>
    __device__ __forceinline__ bool weights(const AttnArgs& a, f16v (&s)[KT], int32_t t0, int32_t lo, Weights<KT>& p, Between between) {
        if constexpr (RULE) bend<KT>(a, s, t0);
        float low = INFINITY;  // (of the masked too, which costs a second round at worst)
        auto least = [&] {
            if constexpr (F32) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++) low = fminf(low, s[t][r]);
            }
        };
        if (t0 + 32 * KT > wmin || t0 < lo || (RULE && t0 < fmax)) {  // uniform
            asm volatile("");  // a branch, not two selects a score in every tile
            least();
            mask<KT>(s, t0, lo);
        } else {
            least();
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[t][r]);
        top = other_max(top) * c;
        if (__any(top > m + kLag || (F32 && top < bottom))) {
            float mn = top > m + kLag ? top : m;
            if constexpr (F32) {
                if (top < bottom && top != -INFINITY) mn = fmaxf(top, peak - kDeep);
                peak = fmaxf(peak, mn);
                bottom = mn > peak - kDeep ? mn - kDrop : -INFINITY;
            }
            const float w = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= w;
            if constexpr (F32) lost *= w;
            scale_o(w);
        }
        const float b = kLift - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const f2 x = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], c, b)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + 1], c, b))};
                h2 hi, lw;
                if constexpr (F32) {
                    split(x, hi, lw);
                    p.l[2 * t + r / 8][r % 8] = lw.x;
                    p.l[2 * t + r / 8][r % 8 + 1] = lw.y;
                    l += x.x + x.y;
                } else {  // the sum of the weights as they enter the product
                    hi = __builtin_convertvector(x, h2);
                    l = __builtin_amdgcn_fdot2(__builtin_bit_cast(hh2, hi), hh2{(__fp16)1.0f, (__fp16)1.0f}, l, false);
                }
                asm volatile("" : "+v"(l));  // here: put off, the sums would keep all weights alive
                p.h[2 * t + r / 8][r % 8] = hi.x;
                p.h[2 * t + r / 8][r % 8 + 1] = hi.y;
                between(t * 8 + r / 2);
            }
        return F32 && __builtin_fmaf(low, c, b) < kThin;
    }
    // Whether the sums of each row with small weights (thin) are so large that what two
    // parts leave of those, over the 32 keys of v, is below 2^-19 of them.
    __device__ __forceinline__ bool carried(const uint8_t* v, bool thin) {
        us2 x = {0, 0};
        const v4u* p = reinterpret_cast<const v4u*>(v) + (threadIdx.x & 63);
#pragma unroll 2
        for (int i = 0; i < HD / 16; i++) {
            const v4u y = p[i * 64];
#pragma unroll
            for (int k = 0; k < 4; k++) x = __builtin_elementwise_max(x, __builtin_bit_cast(us2, y[k] & 0x7fff7fffu));
        }
        uint32_t most = max(x.x, x.y);  // (fp16 magnitudes order as integers, NaN above all)
        most = max8_u32(most);
        most = max(most, dpp_u32<kDppRowMirror>(most));
        most = max(max(lane_of(most, 0), lane_of(most, 16)), max(lane_of(most, 32), lane_of(most, 48)));
        float sum = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) sum = fmaxf(sum, fabsf(o[d][r]));
        const float more = __builtin_fmaf(half_bits_to_float(most), 32.0f, lost);
        if (__any(thin && !(other_max(sum) >= more * 0x1p-6f))) return false;
        lost = more;
        return true;
    }
    // What the two parts of weights below 2^-3 left of them (of a larger one less than
    // 2^-22), from the masked scores of 32 keys: added to O, 2^kAgain larger on the way.
    __device__ __forceinline__ void leftovers(const uint8_t* v, const f16v& s) {
        const float up = __builtin_ldexpf(1.0f, (int)kAgain);
        float b = kLift - (m == -INFINITY ? 0.0f : m);
        asm volatile("" : "+v"(b));  // not the weights kept since weights(): registers
        scale_o(up);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            h8 ph, pl;
#pragma unroll
            for (int r = 0; r < 8; r += 2) {
                const f2 x = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * e + r], c, b)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * e + r + 1], c, b))};
                h2 hi, lw;
                f2 rest;
                split(x, hi, lw, rest);
                rest.x = x.x < 0.125f ? (rest.x - (float)lw.x) * up : 0.0f;
                rest.y = x.y < 0.125f ? (rest.y - (float)lw.y) * up : 0.0f;
                split(rest, hi, lw);
                ph[r] = hi.x, ph[r + 1] = hi.y;
                pl[r] = lw.x, pl[r + 1] = lw.y;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const h8 vf = as_h8(vfrag(v, e, d));
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl, o[d], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        scale_o(1.0f / up);
    }
    __device__ __forceinline__ void scale_o(float w) {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= w;
    }
    __device__ __forceinline__ void first_values(const uint8_t* v, h8 (&vf)[kAhead]) const {
#pragma unroll
        for (int i = 0; i < kAhead; i++) vf[i] = as_h8(vfrag(v, i / ND, i % ND));
    }
    template <int KT>
    __device__ __forceinline__ void values(const uint8_t* v, h8 (&vf)[kAhead], const Weights<KT>& p) {
#pragma unroll
        for (int i = 0; i < 2 * KT * ND; i++) {
            const int e = i / ND, d = i % ND;
            if (i == 1) products(true);  // (raised before the first, which waits for LDS, it gains nothing)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % kAhead], p.h[e], o[d], 0, 0, 0);
            if constexpr (F32) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % kAhead], p.l[e], o[d], 0, 0, 0);
            if (i + kAhead < 2 * KT * ND) vf[i % kAhead] = as_h8(vfrag(v, (i + kAhead) / ND, (i + kAhead) % ND));
            __builtin_amdgcn_sched_barrier(0);
        }
        products(false);
    }
    template <int KT>
    __device__ __forceinline__ void step(const AttnArgs& a, const uint8_t* k, const uint8_t* v, int32_t t0, int32_t lo) {
        f16v s[KT];
        Weights<KT> p;
        h8 vf[kAhead];
        scores<KT>(k, s, [](int) {});
        const bool thin = weights<KT>(a, s, t0, lo, p, [](int) {});
        first_values(v, vf);
        values<KT>(v, vf, p);
        if constexpr (F32) {
            static_assert(KT == 1);
            if (__any(thin) && !carried(v, thin)) leftovers(v, s[0]);
        }
    }
    // Values that are not finite and that a row sees, added to its sums (whatever
    // their weight): keys [from, to).  tidy() took them out of the products.
    __device__ __forceinline__ void add_nonfinite(const AttnArgs& a, const Work& w, uint32_t g, int32_t from, int32_t to) {
#pragma unroll 1
        for (int32_t key = max(from, w.lo); key < min(to, w.kend); key++) {
            const uint32_t p = a.by_page((uint32_t)key / 16);
            const uint32_t id = p < a.max_pages ? a.table[(uint64_t)w.id * a.max_pages + p] : ANE_NO_PAGE;
            if (id >= a.n_pages) continue;
            const uint16_t* v = a.vp + (((uint64_t)id * a.n_kv + g) * a.ps + (uint32_t)key - p * a.ps) * HD + 4 * half;
            const bool sees = key < lim && !(RULE && key < begin);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint2 u = *reinterpret_cast<const uint2*>(v + d * 32 + 8 * e);
                    const uint32_t y[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        o[d][4 * e + i] += sees && (y[i] & 0x7c00u) == 0x7c00u ? half_bits_to_float(y[i]) : 0.0f;
                }
        }
    }
};

// A masked tile's values that are not finite are taken out of LDS (a value that a
// row does not see has weight 0 there, and 0 times an infinity or NaN would be
// NaN) and added to the rows that see them at the end.  One wave does 16 rows of
// V; true: there were some.
template <int HD>
__device__ __forceinline__ bool tidy(uint8_t* v) {
    v4i* p = reinterpret_cast<v4i*>(v) + (threadIdx.x & 63);
    uint32_t bad = 0;
#pragma unroll
    for (uint32_t i = 0; i < HD / 32; i++) {
        const v4i x = p[i * 64];
#pragma unroll
        for (int k = 0; k < 4; k++) bad |= ((uint32_t)x[k] & 0x7c007c00u) + 0x04000400u;  // bit 15 of a half: exponent all ones
    }
    if (!__any((bad & 0x80008000u) != 0)) return false;
#pragma unroll 1
    for (uint32_t i = 0; i < HD / 32; i++) {
        v4i x = p[i * 64];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t e = (((uint32_t)x[k] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
            x[k] &= ~(int)((e >> 15) * 0xffffu);
        }
        p[i * 64] = x;
    }
    return true;
}

template <bool F32>
__device__ __forceinline__ void put4(void* out, uint64_t at, float4 x) {
    if constexpr (F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = x;
    } else {
        const h2 a = __builtin_convertvector((f2){x.x, x.y}, h2), b = __builtin_convertvector((f2){x.z, x.w}, h2);
        uint2 u;
        __builtin_memcpy(&u.x, &a, 4);
        __builtin_memcpy(&u.y, &b, 4);
        *reinterpret_cast<uint2*>(static_cast<_Float16*>(out) + at) = u;
    }
}

// A row that no group has: nobody else writes its parts of the prefix launch.
__device__ __forceinline__ void no_prefix(const AttnArgs& a, const Work& w, uint32_t g, uint32_t part, uint32_t rows,
                                          uint32_t thread, uint32_t threads) {
    if (part != 0 || !w.alone) return;
    const uint64_t all = (uint64_t)a.n_tokens * a.n_heads;
    for (uint32_t i = thread; i < a.pre.n * rows; i += threads) {
        const uint32_t r = w.row0 + i % rows;
        const uint32_t t = a.by_G(r);
        const uint64_t pr = i / rows * all + (uint64_t)(w.tok0 + t) * a.n_heads + g * a.G + r - t * a.G;
        *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(-INFINITY, 0.0f);
    }
}

__device__ __forceinline__ uint32_t block_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// 128 rows a workgroup, 32 a wave, all their keys; the four waves share tiles of
// 64 keys on a 2-stage LDS ring (each wave copies one 16-key group of K and V a
// tile).  Two workgroups a CU: while one wave of a SIMD is in its weights (some 650
// vector cycles a 32-key block), the other is in its products (512 matrix cycles,
// fp32 1024).  8192 tokens x 32 heads fp16: 560-615 us, 0.89-0.98 PFLOP/s, power
// being the limit: on zeros it takes 436 us, and a library fp16 product of 8192^3
// goes from 1.07 to 1.68 PFLOP/s; fp32: 930-1040 us, 0.53-0.59, so up to 1.18 of
// matrix work.  A workgroup costs some 20000 cycles besides 5000 a tile and pair of
// workgroups (fp32), so prompts of 250-1023 tokens take 127-134 us where their
// products alone would take 80.
// Weights between the products of the other half in one wave measured slower
// (584 us, 549 so), fragments 2, 3 or 6 ahead, the copies spread over the products,
// and row tiles started in descending order of keys the same.
template <int HD, bool F32, int MODE, bool RULE = false>
__global__ void __launch_bounds__(256, 2) k_attn_block(AttnArgs a, uint32_t slots) {
    constexpr uint32_t kT = 64 * HD * 2;
    // K, V of each stage, then one word a wave: its rows' least limit, and whether
    // its group of a tile of each parity holds a value that is not finite.  One
    // array on purpose: with several, the compiler tells LDS accesses apart, and
    // then waits for all copies in flight before it reads what they may alias.
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kT + (RULE ? 64 : 48)];
    int32_t *least = reinterpret_cast<int32_t*>(smem + 4 * kT), *most = least + 12;
    int32_t *odd = least + 4, odd_from = 0x7fffffff, odd_to = 0;
    const uint32_t wave = block_wave(), lane = threadIdx.x & 63, tile = a.by_kv(blockIdx.x);
    const uint32_t g = blockIdx.x - tile * a.n_kv;
    // a causal prompt's last tiles have the most keys: they start first
    Work w;
    if (!find_rows<MODE, 128>(a, slots - 1 - tile, w)) return;
    if constexpr (RULE) uniform(w.row0), uniform(w.rows), uniform(w.tok0), uniform(w.toks);  // (again: else held as vectors)

    // page numbers, length and q are under way together; then the first copies
    Loader<HD> ld;
    if (!RULE) ld.lookup(a, w.id, wave + lane * 4);
    Rows<HD, F32, RULE> r;
    typename Rows<HD, F32, RULE>::Raw raw;
    uint32_t row = w.row0 + wave * 32 + (lane & 31), tok = a.by_G(min(row, w.rows - 1));
    uint32_t head = g * a.G + min(row, w.rows - 1) - tok * a.G;
    bool live = row < w.rows;
    r.fetch_q(a.q, (w.tok0 + tok) * a.q_stride + head * HD, live, raw);
    find_keys<MODE, RULE>(a, 128, 0, w);
    const int32_t base = RULE ? w.kbeg : 0;  // the first tile's first key
    const uint32_t u0 = (uint32_t)base / 16 + wave;
    if (RULE) ld.lookup(a, w.id, u0 + lane * 4);
    ld.settle();
    ld.init();
    const uint32_t tiles = w.kend > base ? (uint32_t)(w.kend - base + 63) / 64 : 0;
    auto issue = [&](uint32_t t) {
        if (t && (t & 63) == 0) ld.lookup(a, w.id, u0 + (t + lane) * 4), ld.settle();
        uint8_t* st = smem + (t & 1) * 2 * kT + wave * (kT / 4);
        ld.copy(a, a.kp, w, g, u0 + t * 4, t & 63, st);
        ld.copy(a, a.vp, w, g, u0 + t * 4, t & 63, st + kT);
    };
    if (tiles) issue(0);
    r.init(a.scale_log2e, row_limit<MODE, RULE>(a, w, tok), live);
    if constexpr (RULE) r.init_rule(a, w, tok, head, live);
    r.take_q(raw);
    if constexpr (RULE) r.init_factor(a);
    __builtin_amdgcn_sched_barrier(0);
    r.clear();

    if (lane == 0) least[wave] = r.wmin;
    if (RULE && lane == 0) most[wave] = r.fmax;
    wait_lgkmcnt0();
    lds_barrier();
    const int32_t wg_min = min(min(least[0], least[1]), min(least[2], least[3]));
    const int32_t wg_from = RULE ? max(max(most[0], most[1]), max(most[2], most[3])) : 0;
    for (uint32_t t = 0; t < tiles; t++) {
        const int32_t t0 = base + (int32_t)t * 64;
        uint8_t* st = smem + (t & 1) * 2 * kT;
        int32_t* flag = odd + (t & 1) * 4;
        const bool masked = t0 + 64 > wg_min || (RULE && t0 < wg_from);
        wait_vmcnt<0>();  // this wave's copies of tile t
        if (masked) {
            const bool bad = tidy<HD>(st + kT + wave * (kT / 4));
            if (lane == 0) flag[wave] = bad;
        }
        wait_lgkmcnt0();  // and its reads of tile t - 1
        lds_barrier();    // everybody's
        if (t + 1 < tiles) issue(t + 1);
        if (masked && __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]))
            odd_from = min(odd_from, t0), odd_to = t0 + 64;
        if constexpr (F32) {  // 32 keys at a time: the two parts of q and of 64 weights do not fit 256 registers
#pragma unroll 1
            for (int h = 0; h < 2; h++)
                if (t0 + 32 * h < r.wmax && !(RULE && t0 + 32 * h + 32 <= r.fmin)) r.template step<1>(a, st + h * (kT / 2), st + kT + h * (kT / 2), t0 + 32 * h, 0);
        } else {
            if (t0 < r.wmax && !(RULE && t0 + 64 <= r.fmin)) r.template step<2>(a, st, st + kT, t0, 0);
        }
    }
    if (odd_from < odd_to) r.add_nonfinite(a, w, g, odd_from, odd_to);

    if constexpr (RULE) {  // worked out again: kept through the loop, they spill
        uint32_t i = lane;
        asm volatile("" : "+v"(i));
        row = w.row0 + wave * 32 + (i & 31), tok = a.by_G(min(row, w.rows - 1));
        head = g * a.G + min(row, w.rows - 1) - tok * a.G, live = row < w.rows;
    }
    if (!live) return;
    const float l = other_sum(r.l);
    if (MODE == kPrompt) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const uint64_t at = (w.tok0 + tok) * a.out_stride + head * HD + 4 * r.half;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                put4<F32>(a.out, at + d * 32 + 8 * e, make_float4(r.o[d][4 * e] * inv, r.o[d][4 * e + 1] * inv,
                                                                 r.o[d][4 * e + 2] * inv, r.o[d][4 * e + 3] * inv));
    } else {  // part 0 of a batch
        const uint64_t pr = (uint64_t)(w.tok0 + tok) * a.n_heads + head;
        if (r.half == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(r.m, l);
        if (l == 0.0f) return;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                put4<true>(a.po, pr * HD + 4 * r.half + d * 32 + 8 * e,
                           make_float4(r.o[d][4 * e], r.o[d][4 * e + 1], r.o[d][4 * e + 2], r.o[d][4 * e + 3]));
    }
}

// Few rows: 32 a workgroup, all of them in every wave; the waves take every
// fourth block of 32 keys each, through tiles of their own (no barrier until the
// end), and are merged through LDS.  A tile has one stage, so that two workgroups
// fit a CU and one's start hides behind the other: V of a block is copied during
// its scores, K of the next during its weights.  The copies go out one at a time
// between those instructions: a CU takes 1 KB to LDS every 16 cycles, and a wave
// that issued all eight at once, among seven others, stood 600 cycles a block
// (2 chunks of 96 tokens after 8000 positions 59 -> 55 us, 64 sequences behind
// 8192 shared positions 48.5 -> 45.5 in a graph).  Single tokens are bound by
// memory: 32 over 1000-4096 positions, 366 MB in 62 us, 5.9 TB/s; the others by
// the chain of a block (copy, products, weights, products: some 2200 cycles, 3100
// beside a second workgroup) and by 15000 cycles of start and merge.
template <int HD>
constexpr uint32_t few_lds() {  // K and V of four waves (or their sums), and their maxima and sums of weights
    return 8 * 32 * HD * 2 + 1024;
}
// EACH: every wave has rows and keys of its own (slot and g differ by wave), so
// there is nothing to merge.
template <int HD, bool F32, int MODE, bool EACH = false, bool RULE = false>
__device__ __forceinline__ void attn_few(const AttnArgs& a, uint32_t slot, uint32_t part, uint32_t g, uint8_t* smem) {
    constexpr uint32_t kT = 32 * HD * 2;
    constexpr int kC = 2 * Loader<HD>::kCopies;
    float4* oo = reinterpret_cast<float4*>(smem);
    float *sm = reinterpret_cast<float*>(smem + 8 * kT), *sl = sm + 128;
    constexpr uint32_t kWaves = EACH ? 1 : 4;  // that share the keys, in turn a block of 32 each
    const uint32_t wave = block_wave(), turn = EACH ? 0 : wave, lane = threadIdx.x & 63;
    Work w;
    if (!find_rows<MODE, 32>(a, slot, w)) return;

    Loader<HD> ld;
    uint32_t u0 = part * (a.parts<MODE>().chunk / 16) + turn * 2;
    if (early_keys<MODE, RULE>(a)) ld.lookup(a, w.id, u0 + lane / 2 * (2 * kWaves) + (lane & 1));
    Rows<HD, F32, RULE> r;
    typename Rows<HD, F32, RULE>::Raw raw;
    const uint32_t row = w.row0 + (lane & 31), tok = a.by_G(min(row, w.rows - 1));
    const uint32_t head = g * a.G + min(row, w.rows - 1) - tok * a.G;
    const bool live = row < w.rows;
    const uint64_t at_q = (w.tok0 + tok) * a.q_stride + head * HD;
    if constexpr (MODE == kOwn) r.fetch_q(a.q, at_q, live, raw);
    else r.fetch_rows(a.q, at_q * (F32 ? 4 : 2), raw);
    find_keys<MODE, RULE>(a, 32, part, w);
    if (!early_keys<MODE, RULE>(a)) {
        u0 = (uint32_t)w.kbeg / 16 + turn * 2;
        ld.lookup(a, w.id, u0 + lane / 2 * (2 * kWaves) + (lane & 1));
    }
    ld.settle();
    ld.init();
    constexpr int32_t kStep = 32 * kWaves;
    const int32_t first = w.kbeg + (int32_t)turn * 32;
    const uint32_t tiles = w.kend > first ? (uint32_t)(w.kend - first + kStep - 1) / kStep : 0;
    uint8_t *kt = smem + wave * 2 * kT, *vt = kt + kT;
    struct Next {  // a block's two groups
        __amdgpu_buffer_rsrc_t g[2];
    };
    auto aim = [&](const uint16_t* x, uint32_t t) {
        const uint32_t u = u0 + t * (2 * kWaves), from = (t & 31) * 2;
        return Next{ld.group(a, x, w, g, u, from), ld.group(a, x, w, g, u + 1, from + 1)};
    };
    auto copy = [&](const Next& n, int i, uint8_t* dst) {
        ld.template copy<MODE == kOwn || EACH>(n.g[2 * i / kC], i % (kC / 2), dst + 2 * i / kC * (kT / 2));
    };
    if (tiles) {
        const Next n = aim(a.kp, 0);
#pragma unroll
        for (int i = 0; i < kC; i++) copy(n, i, kt);
    }
    r.init(a.scale_log2e, row_limit<MODE, RULE>(a, w, tok), live);
    if constexpr (RULE) r.init_rule(a, w, tok, head, live);
    if constexpr (MODE != kOwn) r.turn_rows(vt, live, raw);
    r.take_q(raw);
    if constexpr (RULE) r.init_factor(a);
    __builtin_amdgcn_sched_barrier(0);
    r.clear();

    int32_t odd_from = 0x7fffffff, odd_to = 0;
    for (uint32_t t = 0; t < tiles; t++) {
        const int32_t t0 = first + (int32_t)t * kStep;
        f16v s[1];
        h8 vf[Rows<HD, F32, RULE>::kAhead];
        typename Rows<HD, F32, RULE>::template Weights<1> p;
        wait_vmcnt<0>();  // K of this block
        const Next vn = aim(a.vp, t);
        r.template scores<1>(kt, s, [&](int i) {
            if (i < kC) copy(vn, i, vt);
        });
        wait_lgkmcnt0();
        if (t + 1 < tiles && ((t + 1) & 31) == 0) {
            ld.lookup(a, w.id, u0 + (t + 1 + lane / 2) * (2 * kWaves) + (lane & 1));
            ld.settle();
        }
        const Next kn = aim(a.kp, t + 1);  // past the last: no extent, zeros that nobody reads
        const bool thin = r.template weights<1>(a, s, t0, w.lo, p, [&](int i) {
            if (i < kC) copy(kn, i, kt);
        });
        wait_vmcnt<kC>();  // V of this block
        if (t0 + 32 > r.wmin || t0 < w.lo || (RULE && t0 < r.fmax)) {
            const bool b0 = tidy<HD>(vt), b1 = tidy<HD>(vt + kT / 2);
            if (b0 || b1) odd_from = min(odd_from, t0), odd_to = t0 + 32;
            wait_lgkmcnt0();
        }
        r.first_values(vt, vf);
        r.template values<1>(vt, vf, p);
        if constexpr (F32) {
            if (__any(thin) && !r.carried(vt, thin)) r.leftovers(vt, s[0]);
        }
        wait_lgkmcnt0();
    }
    // (this wave's keys of that range only: the other waves add their own)
    for (int32_t t0 = odd_from; t0 < odd_to; t0 += kStep) r.add_nonfinite(a, w, g, t0, t0 + 32);

    wait_vmcnt<0>();
    const bool whole = a.parts_total == 1;
    const uint64_t pr = (uint64_t)(a.parts<MODE>().first + part) * a.n_tokens * a.n_heads + (uint64_t)(w.tok0 + tok) * a.n_heads + head;
    const uint64_t at = (w.tok0 + tok) * a.out_stride + head * HD;
    const float l = other_sum(r.l);
    if constexpr (EACH) {
        no_prefix(a, w, g, part, min(w.rows - w.row0, 32u), lane, 64);
        if (!live) return;
        if (!whole && r.half == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(r.m, l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 x = make_float4(r.o[d][4 * e], r.o[d][4 * e + 1], r.o[d][4 * e + 2], r.o[d][4 * e + 3]);
                const uint32_t to = d * 32 + 8 * e + 4 * r.half;
                if (whole) put4<F32>(a.out, at + to, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
                else put4<true>(a.po, pr * HD + to, x);
            }
        return;
    }
    // Merge the four waves: each puts its sums into LDS as its lanes hold them
    // (a unit of four dimensions is 1 KB, so nothing conflicts) and takes a
    // quarter of the units of all four back.
    constexpr int kUnits = HD / 8, kMine = kUnits / 4;
    __syncthreads();
    if (r.half == 0) sm[wave * 32 + lane] = r.m, sl[wave * 32 + lane] = l;
#pragma unroll
    for (int u = 0; u < kUnits; u++)
        oo[(wave * kUnits + u) * 64 + lane] = make_float4(r.o[u / 4][u % 4 * 4], r.o[u / 4][u % 4 * 4 + 1],
                                                         r.o[u / 4][u % 4 * 4 + 2], r.o[u / 4][u % 4 * 4 + 3]);
    __syncthreads();
    if (MODE == kOwn) no_prefix(a, w, g, part, min(w.rows - w.row0, 32u), threadIdx.x, 256);
    if (!live) return;
    const uint32_t i = lane & 31;
    const float M = fmaxf(fmaxf(sm[i], sm[32 + i]), fmaxf(sm[64 + i], sm[96 + i]));
    float L = 0.0f, f[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float m = sm[k * 32 + i], l1 = sl[k * 32 + i];
        f[k] = m == -INFINITY && l1 == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - M);  // 0: no key of this row
        L = __builtin_fmaf(l1, f[k], L);
    }
    if (!whole && wave == 0 && r.half == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(M, L);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int j = 0; j < kMine; j++) {
        const uint32_t u = wave * kMine + j, d = u / 4 * 32 + u % 4 * 8 + 4 * r.half;
        float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float4 y = oo[(k * kUnits + u) * 64 + lane];
            x.x = __builtin_fmaf(y.x, f[k], x.x), x.y = __builtin_fmaf(y.y, f[k], x.y);
            x.z = __builtin_fmaf(y.z, f[k], x.z), x.w = __builtin_fmaf(y.w, f[k], x.w);
        }
        if (whole) put4<F32>(a.out, at + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        else if (L != 0.0f) put4<true>(a.po, pr * HD + d, x);
    }
}

__device__ __forceinline__ float wave_max_all(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// (one LDS array in all of them, as above; of 64-wide heads at least three workgroups a CU)
template <int HD, bool F32, int MODE, bool RULE = false>
__global__ void __launch_bounds__(256, HD == 64 ? 3 : 2) k_attn_few(AttnArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[few_lds<HD>()];
    const uint32_t slot = a.by_kv(blockIdx.x);
    attn_few<HD, F32, MODE, false, RULE>(a, slot, blockIdx.y, blockIdx.x - slot * a.n_kv, smem);
}
// Single tokens with few keys, a wave each.
template <int HD, bool F32, bool RULE = false>
__global__ void __launch_bounds__(256, HD == 64 && !(RULE && F32) ? 3 : 2) k_attn_each(AttnArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[few_lds<HD>()];
    const uint32_t job = blockIdx.x * 4 + block_wave(), slot = a.by_kv(job);
    attn_few<HD, F32, RULE ? kPrompt : kOwn, true, RULE>(a, slot, 0, job - slot * a.n_kv, smem);
}
// A batch with few rows a group: prefix and own keys in one launch, the prefix's
// workgroups, which have more keys, first (64 sequences behind 8192 shared
// positions, prefix and own one after the other 58 us with the join, 49 so).
template <int HD, bool F32, bool EACH>
__global__ void __launch_bounds__(256, HD == 64 ? 3 : 2) k_attn_shared(AttnArgs a, uint32_t prefix_slots, uint32_t prefix_blocks) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[few_lds<HD>()];
    const uint32_t b = a.by_kv(blockIdx.x), g = blockIdx.x - b * a.n_kv;
    if (b < prefix_blocks) {
        attn_few<HD, F32, kPrefix>(a, b % prefix_slots, b / prefix_slots, g, smem);
    } else if constexpr (EACH) {
        const uint32_t job = (blockIdx.x - prefix_blocks * a.n_kv) * 4 + block_wave(), slot = a.by_kv(job);
        attn_few<HD, F32, kOwn, true>(a, slot, 0, job - slot * a.n_kv, smem);
    } else {
        attn_few<HD, F32, kOwn>(a, (b - prefix_blocks) / a.own.n, (b - prefix_blocks) % a.own.n, g, smem);
    }
}

// One wave per (token, head): the parts of its keys joined, o = sum o_c 2^(m_c - M).
// Every part of every covered row has its (maximum, sum) written, (-inf, 0) where
// it has no key, so nothing is looked up here: the pairs (one a lane) and the
// first parts' sums are in flight at once.  Latency: 4-5 us, most of it the launch.
template <int HD, bool F32, uint32_t kBatch>
__global__ void __launch_bounds__(64) k_attn_join(AttnArgs a) {
    constexpr int E = HD / 64;
    typedef float fe __attribute__((ext_vector_type(E)));
    const uint32_t row = blockIdx.x, lane = threadIdx.x, parts = a.parts_total;
    const uint32_t tok = row / a.n_heads, head = row % a.n_heads;
    const uint64_t rows = (uint64_t)a.n_tokens * a.n_heads;
    const float* po = a.po + (uint64_t)row * HD + lane * E;
    auto pair = [&](uint32_t i) {
        return i < parts ? *reinterpret_cast<const float2*>(a.pml + (i * rows + row) * 2) : make_float2(-INFINITY, 0.0f);
    };
    fe v[kBatch];
    const float2 p0 = pair(lane);
#pragma unroll
    for (uint32_t k = 0; k < kBatch; k++) v[k] = *reinterpret_cast<const fe*>(po + min(k, parts - 1) * rows * HD);
    if (a.q_start && (tok < a.q_start[0] || tok >= a.q_start[a.n])) return;  // a row of no sequence
    float M = p0.x;
    for (uint32_t i = lane + 64; i < parts; i += 64) M = fmaxf(M, pair(i).x);
    M = wave_max_all(M);
    float L = 0.0f;
    fe o;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    for (uint32_t c = 0; c < parts; c += 64) {
        const float2 p = c ? pair(c + lane) : p0;
        const float w = p.x == -INFINITY && p.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p.x - M);
        L += p.y == 0.0f ? 0.0f : p.y * w;
        for (uint32_t k0 = 0; k0 < min(parts - c, 64u); k0 += kBatch) {
            if (c + k0) {
#pragma unroll
                for (uint32_t k = 0; k < kBatch; k++)
                    v[k] = *reinterpret_cast<const fe*>(po + min(c + k0 + k, parts - 1) * rows * HD);
            }
#pragma unroll
            for (uint32_t k = 0; k < kBatch; k++) {
                const float wk = __shfl(w, k0 + k, 64);
                const float lk = __shfl(p.y, k0 + k, 64);
                if (lk == 0.0f) continue;  // no key: its sums are not written
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(v[k][e], wk, o[e]);
            }
        }
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) L += __shfl_xor(L, x, 64);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint64_t to = tok * a.out_stride + head * HD + lane * E;
    if constexpr (F32) {
        *reinterpret_cast<fe*>(static_cast<float*>(a.out) + to) = o * inv;
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) static_cast<_Float16*>(a.out)[to + e] = (_Float16)(o[e] * inv);
    }
}

int attention_status(const ane_paged_cache* c, uint32_t layer, uint32_t n, uint32_t n_tokens, int type, const void* q,
                     uint64_t q_stride, float scale, const void* out, uint64_t out_stride) {
    const int st = cache_status(c);
    if (st) return st;
    const uint32_t size = type == ANE_TYPE_F32 ? 4 : 2;
    const uint64_t width = (uint64_t)c->n_heads * c->head_dim;
    if (layer >= c->n_layers || n_tokens > kMaxTokens || n > kMaxTokens ||
        (type != ANE_TYPE_F32 && type != ANE_TYPE_F16) || !(scale > 0.0f) || !(scale < 1e30f))
        return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    if (!q || !out) return ANE_ERR_BAD_POINTER;
    if ((((uintptr_t)q) | ((uintptr_t)out)) & 15 || (q_stride * size) & 15 || (out_stride * size) & 15 ||
        q_stride < width || out_stride < width)
        return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}

size_t parts_bytes(const ane_paged_cache* c, uint32_t n_tokens, uint32_t parts, size_t* ml) {
    if (parts <= 1) return 0;
    const uint64_t rows = (uint64_t)n_tokens * c->n_heads * parts;
    const size_t o = ceil_to(rows * c->head_dim * 4, 256);
    if (ml) *ml = o;
    return o + ceil_to(rows * 8, 256);
}

template <int HD, bool F32, bool RULE = false>
void launch_prompt(const AttnArgs& a, const Launch& l, hipStream_t s) {
    const dim3 grid((uint32_t)(l.slots * a.n_kv), l.parts);
    if constexpr (RULE) {
        if (l.each) {
            hipLaunchKernelGGL((k_attn_each<HD, F32, true>), dim3((grid.x + 3) / 4), dim3(256), 0, s, a);
            return;
        }
    }
    if (l.few) hipLaunchKernelGGL((k_attn_few<HD, F32, kPrompt, RULE>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attn_block<HD, F32, kPrompt, RULE>), grid, dim3(256), 0, s, a, (uint32_t)l.slots);
}
template <int HD, bool F32>
void launch_shared(const AttnArgs& a, const SharedPlan& p, hipStream_t s) {
    const Launch &pre = p.prefix, &own = p.own;
    const uint32_t pb = (uint32_t)(pre.slots * pre.parts), ob = (uint32_t)(own.slots * own.parts);
    const uint32_t own_wgs = p.each ? (uint32_t)((own.slots * a.n_kv + 3) / 4) : ob * a.n_kv;
    if (a.n_groups && pre.few) {
        auto* f = p.each ? k_attn_shared<HD, F32, true> : k_attn_shared<HD, F32, false>;
        hipLaunchKernelGGL(f, dim3(pb * a.n_kv + own_wgs), dim3(256), 0, s, a, (uint32_t)pre.slots, pb);
        return;
    }
    if (a.n_groups)
        hipLaunchKernelGGL((k_attn_block<HD, F32, kPrefix>), dim3(pb * a.n_kv), dim3(256), 0, s, a, (uint32_t)pre.slots);
    if (p.each) hipLaunchKernelGGL((k_attn_each<HD, F32>), dim3(own_wgs), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attn_few<HD, F32, kOwn>), dim3((uint32_t)(own.slots * a.n_kv), own.parts), dim3(256), 0, s, a);
}
void join_as(const AttnArgs& a, uint32_t hd, int type, hipStream_t s) {
    auto pick = [&](auto few, auto many) { return a.parts_total <= 4 ? few : many; };
    auto* f = hd == 128 ? (type == ANE_TYPE_F32 ? pick(k_attn_join<128, true, 4>, k_attn_join<128, true, 16>)
                                                : pick(k_attn_join<128, false, 4>, k_attn_join<128, false, 16>))
                        : (type == ANE_TYPE_F32 ? pick(k_attn_join<64, true, 4>, k_attn_join<64, true, 16>)
                                                : pick(k_attn_join<64, false, 4>, k_attn_join<64, false, 16>));
    hipLaunchKernelGGL(f, dim3(a.n_tokens * a.n_heads), dim3(64), 0, s, a);
}

bool plan_fits(const ane_paged_cache* c, const Launch& l, uint64_t n_tokens, uint32_t parts_total) {
    return launch_fits(l.slots * l.parts * c->n_kv_heads, 512) && l.parts <= 65535 &&
           (parts_total == 1 || launch_fits(n_tokens * c->n_heads, 64));
}

AttnArgs attn_args(const ane_paged_cache* c, uint32_t layer, const uint32_t* seqs, uint32_t n, uint32_t n_tokens,
                   const void* q, uint64_t q_stride, float scale, void* out, uint64_t out_stride) {
    AttnArgs a = {};
    const uint64_t lo = page_elems(c) * c->n_pages * layer;
    a.q = q, a.out = out, a.kp = c->k_pages + lo, a.vp = c->v_pages + lo;
    a.table = c->page_table, a.kv_len = c->kv_len, a.seqs = seqs;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.n = n, a.n_tokens = n_tokens, a.n_heads = c->n_heads, a.n_kv = c->n_kv_heads, a.G = c->n_heads / c->n_kv_heads;
    a.ps = c->page_size, a.n_pages = c->n_pages, a.max_pages = c->max_pages, a.n_seqs = c->n_seqs;
    a.by_page = div_by(a.ps / 16), a.by_G = div_by(a.G), a.by_kv = div_by(a.n_kv);
    a.scale_log2e = (float)((double)scale * 1.4426950408889634);
    return a;
}

bool bad_workspace(const void* ws, size_t bytes, size_t need) {
    return need && (!ws || (((uintptr_t)ws) & 255) || bytes < need);
}

}  // namespace
}  // namespace ane

using namespace ane;

// A bound on the keys from the first to the last that a row tile's rows see under a
// rule: with a window no more than window and tile, and what a prefix lets a token see
// past its own position, which is a new token's.
static uint64_t rule_len(const ane_paged_cache* c, const ane_attention_rule* r, uint32_t n_tokens, bool single, uint32_t max_len) {
    const uint64_t len = bound_len(c, max_len);
    if (!r || !r->window) return len;
    return std::min<uint64_t>(len, (uint64_t)r->window + 32 + 16 + (r->prefix && !single ? n_tokens : 0));
}

static Launch prompt_plan(const ane_paged_cache* c, const ane_attention_rule* r, uint32_t n, uint32_t n_tokens, bool single,
                          uint32_t max_len) {
    const uint64_t len = rule_len(c, r, n_tokens, single, max_len);
    const bool windowed = r && r->window && r->window < bound_len(c, max_len);
    Launch l = plan(c, n, n_tokens, single, len, false, r && len > (windowed ? 1024 : 256), windowed);
    l.each = r && single && each_pays(c, l, len);
    return l;
}

static size_t prompt_workspace(const ane_paged_cache* cache, const ane_attention_rule* rule, uint32_t n, uint32_t n_tokens,
                               uint32_t max_len) {
    if (cache_status(cache) || n == 0 || n_tokens == 0 || n > kMaxTokens || n_tokens > kMaxTokens) return 0;
    // the same for a batch of single tokens with and without q_start
    const Launch l = prompt_plan(cache, rule, n, n_tokens, false, max_len);
    const Launch one = prompt_plan(cache, rule, n, n_tokens, true, max_len);
    return parts_bytes(cache, n_tokens, n_tokens == n ? std::max(l.parts, one.parts) : l.parts, nullptr);
}

static int prompt(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n, const uint32_t* q_start,
                  uint32_t n_tokens, uint32_t max_len, const ane_attention_rule* rule, int type, const void* q,
                  uint64_t q_stride, float scale, void* out, uint64_t out_stride, void* workspace, size_t workspace_bytes,
                  void* stream) {
    const int st = attention_status(cache, layer, n, n_tokens, type, q, q_stride, scale, out, out_stride);
    if (st) return st;
    if (!q_start && n_tokens != n) return ANE_ERR_INVALID_ARG;
    if (rule && !(rule->softcap == 0.0f || (rule->softcap >= 0x1p-20f && rule->softcap <= 0x1p20f))) return ANE_ERR_INVALID_ARG;
    if (rule && ((((uintptr_t)rule->slopes) | ((uintptr_t)rule->first) | ((uintptr_t)rule->prefix)) & 3)) return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    const Launch l = prompt_plan(cache, rule, n, n_tokens, !q_start, max_len);
    if (!plan_fits(cache, l, n_tokens, l.parts)) return ANE_ERR_INVALID_ARG;
    size_t ml = 0;
    if (bad_workspace(workspace, workspace_bytes, parts_bytes(cache, n_tokens, l.parts, &ml))) return ANE_ERR_WORKSPACE;
    AttnArgs a = attn_args(cache, layer, seqs, n, n_tokens, q, q_stride, scale, out, out_stride);
    a.q_start = q_start;
    a.po = static_cast<float*>(workspace);
    a.pml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ml);
    a.own = {l.chunk, l.parts, 0}, a.parts_total = l.parts;
    hipStream_t s = (hipStream_t)stream;
    const bool f32 = type == ANE_TYPE_F32;
    if (rule) {
        const double cap = (double)rule->softcap * 1.4426950408889634;
        a.cap = (float)cap, a.inv_cap = cap != 0.0 ? (float)(1.0 / cap) : 0.0f;
        // (neither these nor squares of scores below kSmall of the cap leave fp32's range then)
        const double d = (double)a.scale_log2e * a.inv_cap;
        const bool in_range = d >= 0x1p-20 && d <= 0x1p20;
        for (int k = 0; k < 3; k++) a.bend[k] = in_range ? (float)(Tanh<false>::kHalf[k] * std::pow(d, 2 * k + 2)) : 0.0f;
        a.slopes = rule->slopes, a.window = std::min(rule->window, 1u << 30), a.first = rule->first, a.seen = rule->prefix;
        if (cache->head_dim == 128) f32 ? launch_prompt<128, true, true>(a, l, s) : launch_prompt<128, false, true>(a, l, s);
        else f32 ? launch_prompt<64, true, true>(a, l, s) : launch_prompt<64, false, true>(a, l, s);
    } else {
        if (cache->head_dim == 128) f32 ? launch_prompt<128, true>(a, l, s) : launch_prompt<128, false>(a, l, s);
        else f32 ? launch_prompt<64, true>(a, l, s) : launch_prompt<64, false>(a, l, s);
    }
    if (l.parts > 1) join_as(a, cache->head_dim, type, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" size_t ane_hip_attention_prompt_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                                          uint32_t max_len) {
    return prompt_workspace(cache, nullptr, n, n_tokens, max_len);
}

extern "C" int ane_hip_attention_prompt(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                        const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len, int type,
                                        const void* q, uint64_t q_stride, float scale, void* out, uint64_t out_stride,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    return prompt(cache, layer, seqs, n, q_start, n_tokens, max_len, nullptr, type, q, q_stride, scale, out, out_stride,
                  workspace, workspace_bytes, stream);
}

extern "C" size_t ane_hip_attention_rule_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                                        uint32_t max_len, const ane_attention_rule* rule) {
    return prompt_workspace(cache, rule, n, n_tokens, max_len);
}

extern "C" int ane_hip_attention_rule(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                      const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len,
                                      const ane_attention_rule* rule, int type, const void* q, uint64_t q_stride,
                                      float scale, void* out, uint64_t out_stride, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    if (!rule) return ANE_ERR_BAD_POINTER;
    return prompt(cache, layer, seqs, n, q_start, n_tokens, max_len, rule, type, q, q_stride, scale, out, out_stride,
                  workspace, workspace_bytes, stream);
}

extern "C" size_t ane_hip_attention_shared_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_groups,
                                                          uint32_t max_prefix, uint32_t max_len) {
    if (cache_status(cache) || n == 0 || n > kMaxTokens || n_groups > n) return 0;
    return parts_bytes(cache, n, shared_plan(cache, n, n_groups, max_prefix, max_len).parts, nullptr);
}

extern "C" int ane_hip_attention_shared(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                        uint32_t n_groups, const uint32_t* group_start, const uint32_t* prefix_len,
                                        uint32_t max_prefix, uint32_t max_len, int type, const void* q,
                                        uint64_t q_stride, float scale, void* out, uint64_t out_stride, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int st = attention_status(cache, layer, n, n, type, q, q_stride, scale, out, out_stride);
    if (st || n == 0) return st;
    if (n_groups > n) return ANE_ERR_INVALID_ARG;
    if (n_groups && (!group_start || !prefix_len)) return ANE_ERR_BAD_POINTER;
    const SharedPlan p = shared_plan(cache, n, n_groups, max_prefix, max_len);
    if (!plan_fits(cache, p.own, n, p.parts) || !plan_fits(cache, p.prefix, n, p.parts)) return ANE_ERR_INVALID_ARG;
    size_t ml = 0;
    if (bad_workspace(workspace, workspace_bytes, parts_bytes(cache, n, p.parts, &ml))) return ANE_ERR_WORKSPACE;
    AttnArgs a = attn_args(cache, layer, seqs, n, n, q, q_stride, scale, out, out_stride);
    a.n_groups = n_groups, a.group_start = group_start, a.prefix = prefix_len;
    a.po = static_cast<float*>(workspace);
    a.pml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ml);
    a.parts_total = p.parts;
    a.pre = {p.prefix.chunk, p.prefix.parts, 0}, a.own = {p.own.chunk, p.own.parts, p.prefix.parts};
    hipStream_t s = (hipStream_t)stream;
    if (cache->head_dim == 128)
        type == ANE_TYPE_F32 ? launch_shared<128, true>(a, p, s) : launch_shared<128, false>(a, p, s);
    else
        type == ANE_TYPE_F32 ? launch_shared<64, true>(a, p, s) : launch_shared<64, false>(a, p, s);
    if (p.parts > 1) join_as(a, cache->head_dim, type, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}
