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

#include "paged.hpp"

namespace ane {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
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
    uint32_t div_magic, div_shift;                // 16-position group -> page, see page_div
    uint32_t chunk, part0, n_parts, parts_total;  // keys a part, this launch's parts
    uint32_t chunk_prefix, n_parts_prefix;        // of the prefix launch, for the merge
    float scale_log2e;
};

// u / (ps / 16) for u < 2^27 as (u * magic) >> shift: with shift = 27 +
// ceil(log2 d), magic = ceil(2^shift / d) <= 2^28, the excess magic * d - 2^shift
// is below d <= 2^(shift - 27), so u * excess < 2^shift and the floor is exact.
void page_div(uint32_t ps, uint32_t* magic, uint32_t* shift) {
    const uint32_t d = ps / 16;
    uint32_t lg = 0;
    while ((1u << lg) < d) lg++;
    *shift = 27 + lg;
    *magic = (uint32_t)(((1ull << *shift) + d - 1) / d);
}

__device__ __forceinline__ uint32_t seq_id(const AttnArgs& a, uint32_t s) { return a.seqs ? a.seqs[s] : s; }
__device__ __forceinline__ uint32_t seq_len(const AttnArgs& a, uint32_t id) {
    return id < a.n_seqs ? (uint32_t)min((uint64_t)a.kv_len[id], (uint64_t)a.max_pages * a.ps) : 0;
}
// The positions batch row s shares with its group (0: none).
__device__ __forceinline__ uint32_t shared_len(const AttnArgs& a, uint32_t s, uint32_t len) {
    if (a.n_groups == 0) return 0;
    const uint32_t g = wave_search(a.n_groups, s, [&](uint32_t i) { return (uint64_t)a.group_start[i]; });
    const uint32_t first = a.group_start[g];
    if (first > s || s >= a.group_start[g + 1]) return 0;
    return min(min(a.prefix[g], len), seq_len(a, seq_id(a, first)));
}

// What a workgroup computes: BM rows of one kv head of one batch row (of one
// group in kPrefix), keys [kbeg, kend) from the pages of sequence id.
struct Work {
    uint32_t id, tok0, toks, row0, rows;  // first token, tokens, first row of the tile, rows in all
    int32_t kbeg, kend, lo;               // lo: keys before it are masked (kbeg rounds it down to 16)
    int32_t len;

    // Every lane holds the same values; the compiler has to be told, or each
    // copy to LDS loops over its lanes' descriptors.
    __device__ __forceinline__ void uniform() {
        for (uint32_t* x : {&id, &tok0, &toks, &row0, &rows}) *x = __builtin_amdgcn_readfirstlane(*x);
        for (int32_t* x : {&kbeg, &kend, &lo, &len}) *x = __builtin_amdgcn_readfirstlane(*x);
    }
};

template <int MODE, int BM>
__device__ __forceinline__ bool find_work(const AttnArgs& a, uint32_t slot, uint32_t part, Work& w) {
    const uint32_t* start = MODE == kPrefix ? a.group_start : MODE == kPrompt ? a.q_start : nullptr;
    const uint32_t n = MODE == kPrefix ? a.n_groups : a.n;
    uint32_t s, tile;
    if (start) {  // tiles of row s: slots start[s] * G / BM + s onwards, which never overlap
        auto key = [&](uint32_t i) { return (uint64_t)start[i] * a.G / BM + i; };
        s = wave_search(n, slot, key);
        if (key(s) > slot) return false;
        tile = slot - (uint32_t)key(s);
        w.tok0 = start[s];
        const uint32_t end = min(start[s + 1], a.n_tokens);
        w.toks = end > w.tok0 ? end - w.tok0 : 0;
    } else {
        const uint32_t tiles = (a.G + BM - 1) / BM;
        s = slot / tiles, tile = slot % tiles;
        if (s >= n) return false;
        w.tok0 = s, w.toks = 1;
    }
    w.rows = w.toks * a.G;  // below 2^30
    w.row0 = tile * BM;
    if (tile >= (1u << 24) || w.row0 >= w.rows) return false;
    w.id = seq_id(a, MODE == kPrefix ? w.tok0 : s);
    w.len = (int32_t)seq_len(a, w.id);
    w.kbeg = w.lo = 0;
    w.kend = w.len;
    if (MODE == kPrompt) {
        const int32_t last = (int32_t)((min(w.row0 + BM, w.rows) - 1) / a.G);
        w.kend = min(w.len, w.len - (int32_t)w.toks + last + 1);
    } else if (MODE == kPrefix) {
        w.kend = (int32_t)min(a.prefix[s], (uint32_t)w.len);
    } else {
        w.lo = (int32_t)shared_len(a, s, (uint32_t)w.len);
        w.kbeg = w.lo & ~15;
        if (w.lo >= w.kend) w.kend = w.kbeg;
    }
    const int64_t b = w.kbeg + (int64_t)part * a.chunk;
    if (b >= w.kend && a.parts_total > 1) return false;  // the merge does not read it
    if (part + 1 < a.n_parts) w.kend = (int32_t)min((int64_t)w.kend, b + a.chunk);
    w.kbeg = (int32_t)min(b, (int64_t)max(w.kend, 0));
    return true;
}
// Keys of the work a row (token t of the work's) sees: those below.
template <int MODE>
__device__ __forceinline__ int32_t row_limit(const AttnArgs& a, const Work& w, uint32_t t) {
    int32_t l = w.len;
    if (MODE == kPrompt) l += (int32_t)t + 1 - (int32_t)w.toks;
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
        return (uint32_t)((uint64_t)u * a.div_magic >> a.div_shift);
    }
    // u: this lane's 16-position group
    __device__ __forceinline__ void lookup(const AttnArgs& a, const Work& w, uint32_t u) {
        const uint32_t p = page(a, u);
        ids = (int32_t)u * 16 < w.kend && u < (1u << 27) && p < a.max_pages
                  ? a.table[(uint64_t)w.id * a.max_pages + p] : ANE_NO_PAGE;
        asm volatile("" : "+v"(ids));  // the wait for it here, not before each copy that follows
    }
    // group u (wave-uniform), whose page number is in lane `from`, of kv head g
    __device__ __forceinline__ void copy(const AttnArgs& a, const Work& w, uint32_t g, uint32_t u, uint32_t from,
                                         uint8_t* k, uint8_t* v) const {
        const uint32_t id = __builtin_amdgcn_readlane(ids, from);
        const uint32_t row = u * 16 - page(a, u) * a.ps;
        const int32_t left = w.kend - (int32_t)(u * 16);
        // (a clamp goes through the vector ALU: back to a scalar, as above)
        const uint32_t bytes = __builtin_amdgcn_readfirstlane(id < a.n_pages ? (uint32_t)min(max(left, 0), 16) * RB : 0);
        const uint64_t at = (((uint64_t)(id < a.n_pages ? id : 0) * a.n_kv + g) * a.ps + row) * HD;
        const __amdgpu_buffer_rsrc_t rk = make_rsrc(a.kp + at, bytes), rv = make_rsrc(a.vp + at, bytes);
#pragma unroll
        for (uint32_t i = 0; i < kCopies; i++) copy16_to_lds(rk, k + i * 1024, off[i]);
#pragma unroll
        for (uint32_t i = 0; i < kCopies; i++) copy16_to_lds(rv, v + i * 1024, off[i]);
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

// The running maximum may lag by kLag (in log2) before O and l are rescaled;
// weights are e^s 2^kLift relative to it, at most 2^(kLag + kLift) = 2^14, so that
// fp16 keeps weights 2^-20 of the largest with full precision.
constexpr float kLag = 8.0f, kLift = 6.0f;

// 32 rows of a wave: lane & 31 is the row, lane >> 5 the half of its keys (of its
// dimensions in q and O).
template <int HD, bool F32>
struct Rows {
    static constexpr int NS = HD / 16, ND = HD / 32;
    static constexpr uint32_t RB = HD * 2;
    h8 qh[NS], ql[F32 ? NS : 1];  // q, its low part
    f16v o[ND];
    float m, l, c;  // maximum (log2, lagging), this half's sum, score factor
    int32_t lim;    // keys below it are seen
    int32_t wmin, wmax;
    uint32_t half, ka, va[2 * ND];

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
        m = -INFINITY, l = 0.0f, c = scale_log2e;
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
    __device__ __forceinline__ void load_q(const void* q, uint64_t at, bool live) {
        if constexpr (!F32) {
#pragma unroll
            for (int e = 0; e < 8; e++) ql[0][e] = (_Float16)0.0f;
#pragma unroll
            for (int s = 0; s < NS; s++) {
                v4i x = {0, 0, 0, 0};
                if (live) x = *reinterpret_cast<const v4i*>(static_cast<const _Float16*>(q) + at + 16 * s + 8 * half);
                qh[s] = as_h8(x);
            }
#pragma unroll
            for (int s = 0; s < NS; s++) asm volatile("" : "+v"(qh[s]));  // the wait for q here, not in the loop
        } else {
            float4 x[NS][2];
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    x[s][e] = live ? *reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + 16 * s + 8 * half + 4 * e)
                                   : make_float4(0, 0, 0, 0);
                    top = max(max(top, abs_key(x[s][e].x)), max(abs_key(x[s][e].y), max(abs_key(x[s][e].z), abs_key(x[s][e].w))));
                }
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            // 2^(140 - ex) brings the largest |q| (exponent field ex) to [2^13, 2^14)
            const uint32_t ex = max(top >> 23, 20u);
            const float up = __uint_as_float((267 - ex) << 23);
            c *= __uint_as_float((ex - 13) << 23);
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float v[4] = {x[s][e].x * up, x[s][e].y * up, x[s][e].z * up, x[s][e].w * up};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        qh[s][4 * e + k] = (_Float16)v[k];
                        ql[s][4 * e + k] = (_Float16)(v[k] - (float)qh[s][4 * e + k]);
                    }
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
    // KT blocks of 32 keys from position t0 on; keys before lo are masked.
    template <int KT>
    __device__ __forceinline__ void step(const uint8_t* k, const uint8_t* v, int32_t t0, int32_t lo) {
        // Fragments are read kAhead products before their use and the order is
        // pinned: left alone, the scheduler reads all of them first and spills.
        constexpr int kAhead = 4;
        f16v s[KT];
        const uint32_t kx = swz<HD>(ka & 15);
        auto kfrag = [&](int i) {  // products in the order (e, t)
            const int e = i / KT, t = i % KT;
            return as_h8(*reinterpret_cast<const v4i*>(k + (t * 32 + ka) * RB + (((2 * e + half) ^ kx) << 4)));
        };
        {
            h8 kf[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) kf[i] = kfrag(i);
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[t][r] = 0.0f;
#pragma unroll
            for (int i = 0; i < NS * KT; i++) {
                const int e = i / KT, t = i % KT;
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % kAhead], qh[e], s[t], 0, 0, 0);
                if constexpr (F32) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % kAhead], ql[e], s[t], 0, 0, 0);
                if (i + kAhead < NS * KT) kf[i % kAhead] = kfrag(i + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const bool masked = t0 + 32 * KT > wmin || t0 < lo;  // uniform
        if (masked) {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int32_t key = t0 + t * 32 + 8 * (r >> 2) + 4 * (int32_t)half + (r & 3);
                    if (key >= lim || key < lo) s[t][r] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[t][r]);
        top = other_max(top) * c;
        if (__any(top > m + kLag)) {
            const float mn = top > m + kLag ? top : m;
            const float w = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] *= w;
        }
        const float b = kLift - (m == -INFINITY ? 0.0f : m);
        h8 ph[2 * KT], pl[F32 ? 2 * KT : 1];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const f2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], c, b)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + 1], c, b))};
                l += p.x + p.y;
                const h2 hi = __builtin_convertvector(p, h2);
                ph[2 * t + r / 8][r % 8] = hi.x;
                ph[2 * t + r / 8][r % 8 + 1] = hi.y;
                if constexpr (F32) {
                    const f2 rest = {__builtin_fmaf((float)hi.x, -1.0f, p.x), __builtin_fmaf((float)hi.y, -1.0f, p.y)};
                    const h2 lw = __builtin_convertvector(rest, h2);
                    pl[2 * t + r / 8][r % 8] = lw.x;
                    pl[2 * t + r / 8][r % 8 + 1] = lw.y;
                }
            }
        h8 vf[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) vf[i] = as_h8(vfrag(v, i / ND, i % ND));
#pragma unroll
        for (int i = 0; i < 2 * KT * ND; i++) {
            const int e = i / ND, d = i % ND;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % kAhead], ph[e], o[d], 0, 0, 0);
            if constexpr (F32) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % kAhead], pl[e], o[d], 0, 0, 0);
            if (i + kAhead < 2 * KT * ND) vf[i % kAhead] = as_h8(vfrag(v, (i + kAhead) / ND, (i + kAhead) % ND));
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // Values that are not finite and that a row sees, added to its sums (whatever
    // their weight): keys [from, to).  tidy() took them out of the products.
    __device__ __forceinline__ void add_nonfinite(const AttnArgs& a, const Work& w, uint32_t g, int32_t from, int32_t to) {
#pragma unroll 1
        for (int32_t key = max(from, w.lo); key < min(to, w.kend); key++) {
            const uint32_t p = (uint32_t)((uint64_t)((uint32_t)key / 16) * a.div_magic >> a.div_shift);
            const uint32_t id = p < a.max_pages ? a.table[(uint64_t)w.id * a.max_pages + p] : ANE_NO_PAGE;
            if (id >= a.n_pages) continue;
            const uint16_t* v = a.vp + (((uint64_t)id * a.n_kv + g) * a.ps + (uint32_t)key - p * a.ps) * HD + 4 * half;
            const bool sees = key < lim;
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

__device__ __forceinline__ uint32_t block_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// 128 rows a workgroup, 32 a wave; the four waves share tiles of 64 keys on a
// 2-stage LDS ring (each wave copies one 16-key group of K and V a tile).
template <int HD, bool F32, int MODE>
__global__ void __launch_bounds__(256, 2) k_attn_block(AttnArgs a, uint32_t slots) {
    constexpr uint32_t kT = 64 * HD * 2;
    // K, V of each stage, then one word a wave: its rows' least limit, and whether
    // its group of a tile of each parity holds a value that is not finite.  One
    // array on purpose: with several, the compiler tells LDS accesses apart, and
    // then waits for all copies in flight before it reads what they may alias.
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kT + 48];
    int32_t* least = reinterpret_cast<int32_t*>(smem + 4 * kT);
    int32_t *odd = least + 4, odd_from = 0x7fffffff, odd_to = 0;
    const uint32_t wave = block_wave(), lane = threadIdx.x & 63, g = blockIdx.x % a.n_kv;
    // a causal prompt's last tiles have the most keys: they start first
    const uint32_t slot = slots - 1 - blockIdx.x / a.n_kv, part = blockIdx.y;
    Work w;
    if (!find_work<MODE, 128>(a, slot, part, w)) return;
    w.uniform();

    Loader<HD> ld;
    ld.init();
    const uint32_t u0 = (uint32_t)w.kbeg / 16 + wave, tiles = (uint32_t)(w.kend - w.kbeg + 63) / 64;
    auto issue = [&](uint32_t t) {
        if ((t & 63) == 0) ld.lookup(a, w, u0 + (t + lane) * 4);
        uint8_t* st = smem + (t & 1) * 2 * kT + wave * (kT / 4);
        ld.copy(a, w, g, u0 + t * 4, t & 63, st, st + kT);
    };
    if (w.kend > w.kbeg) issue(0);

    Rows<HD, F32> r;
    const uint32_t row = w.row0 + wave * 32 + (lane & 31), tok = row / a.G, head = g * a.G + row % a.G;
    const bool live = row < w.rows;
    r.init(a.scale_log2e, live ? row_limit<MODE>(a, w, tok) : 0, live);
    r.load_q(a.q, live ? (w.tok0 + tok) * a.q_stride + head * HD : 0, live);
    __builtin_amdgcn_sched_barrier(0);
    r.clear();

    if (lane == 0) least[wave] = r.wmin;
    wait_lgkmcnt0();
    lds_barrier();
    const int32_t wg_min = min(min(least[0], least[1]), min(least[2], least[3]));
    if (w.kend > w.kbeg)
        for (uint32_t t = 0; t < tiles; t++) {
            const int32_t t0 = w.kbeg + (int32_t)t * 64;
            const uint8_t* st = smem + (t & 1) * 2 * kT;
            const bool masked = t0 + 64 > wg_min || t0 < w.lo;
            wait_vmcnt<0>();  // this wave's copies of tile t
            int32_t* flag = odd + (t & 1) * 4;
            if (masked) {
                const bool bad = tidy<HD>(smem + (t & 1) * 2 * kT + kT + wave * (kT / 4));
                if (lane == 0) flag[wave] = bad;
            }
            wait_lgkmcnt0();  // and its reads of tile t - 1
            lds_barrier();    // everybody's
            if (t + 1 < tiles) issue(t + 1);
            if (masked && __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]))
                odd_from = min(odd_from, t0), odd_to = t0 + 64;
            if constexpr (F32) {  // 32 keys at a time: the two parts of q and of 64 weights do not fit 256 registers
                if (t0 < r.wmax) r.template step<1>(st, st + kT, t0, w.lo);
                if (t0 + 32 < r.wmax) r.template step<1>(st + kT / 2, st + kT + kT / 2, t0 + 32, w.lo);
            } else {
                if (t0 < r.wmax) r.template step<2>(st, st + kT, t0, w.lo);
            }
        }
    if (odd_from < odd_to) r.add_nonfinite(a, w, g, odd_from, odd_to);

    if (!live) return;
    const float l = other_sum(r.l);
    if (a.parts_total == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const uint64_t at = (w.tok0 + tok) * a.out_stride + head * HD + 4 * r.half;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                put4<F32>(a.out, at + d * 32 + 8 * e, make_float4(r.o[d][4 * e] * inv, r.o[d][4 * e + 1] * inv,
                                                                 r.o[d][4 * e + 2] * inv, r.o[d][4 * e + 3] * inv));
    } else {
        const uint64_t pr = (uint64_t)(a.part0 + part) * a.n_tokens * a.n_heads + (uint64_t)(w.tok0 + tok) * a.n_heads + head;
        if (r.half == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(r.m, l);
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                put4<true>(a.po, pr * HD + 4 * r.half + d * 32 + 8 * e,
                           make_float4(r.o[d][4 * e], r.o[d][4 * e + 1], r.o[d][4 * e + 2], r.o[d][4 * e + 3]));
    }
}

// Few rows: 32 a workgroup, all of them in every wave; the waves take every
// fourth block of 32 keys each, on rings of their own (no barrier until the
// end), and are merged through LDS.
template <int HD, bool F32, int MODE>
__global__ void __launch_bounds__(256, 2) k_attn_few(AttnArgs a) {
    constexpr uint32_t kT = 32 * HD * 2, kPad = HD + 4;
    // per wave: K, V of two stages; one array, as above, which the merge reuses
    __shared__ __attribute__((aligned(1024))) uint8_t smem[16 * kT];
    float* oo = reinterpret_cast<float*>(smem);
    float *sm = oo + 4 * 32 * kPad, *sl = sm + 128;
    static_assert((4 * 32 * kPad + 256) * 4 <= sizeof(smem), "the merge fits the rings");
    const uint32_t wave = block_wave(), lane = threadIdx.x & 63, g = blockIdx.x % a.n_kv, part = blockIdx.y;
    Work w;
    if (!find_work<MODE, 32>(a, blockIdx.x / a.n_kv, part, w)) return;
    w.uniform();

    Loader<HD> ld;
    ld.init();
    const int32_t first = w.kbeg + (int32_t)wave * 32;
    const uint32_t u0 = (uint32_t)first / 16, tiles = w.kend > first ? (uint32_t)(w.kend - first + 127) / 128 : 0;
    uint8_t* ring = smem + wave * 4 * kT;
    int32_t odd_from = 0x7fffffff, odd_to = 0;
    auto issue = [&](uint32_t t) {
        if ((t & 31) == 0) ld.lookup(a, w, u0 + (t + lane / 2) * 8 + (lane & 1));
        uint8_t* st = ring + (t & 1) * 2 * kT;
#pragma unroll
        for (uint32_t i = 0; i < 2; i++)
            ld.copy(a, w, g, u0 + t * 8 + i, (t & 31) * 2 + i, st + i * (kT / 2), st + kT + i * (kT / 2));
    };
    if (tiles) issue(0);

    Rows<HD, F32> r;
    const uint32_t row = w.row0 + (lane & 31), tok = row / a.G, head = g * a.G + row % a.G;
    const bool live = row < w.rows;
    r.init(a.scale_log2e, live ? row_limit<MODE>(a, w, tok) : 0, live);
    r.load_q(a.q, live ? (w.tok0 + tok) * a.q_stride + head * HD : 0, live);
    __builtin_amdgcn_sched_barrier(0);
    r.clear();

    for (uint32_t t = 0; t < tiles; t++) {
        if (t + 1 < tiles) {
            wait_lgkmcnt0();  // the reads of tile t - 1, whose stage is refilled
            issue(t + 1);
            wait_vmcnt<4 * Loader<HD>::kCopies>();  // tile t has landed, tile t + 1 is on its way
        } else {
            wait_vmcnt<0>();
        }
        const int32_t t0 = first + (int32_t)t * 128;
        uint8_t* st = ring + (t & 1) * 2 * kT;
        if (t0 + 32 > r.wmin || t0 < w.lo) {
            const bool b0 = tidy<HD>(st + kT), b1 = tidy<HD>(st + kT + kT / 2);
            if (b0 || b1) odd_from = min(odd_from, t0), odd_to = t0 + 32;
        }
        if (t0 < r.wmax) r.template step<1>(st, st + kT, t0, w.lo);
    }
    // (this wave's keys of that range only: the other waves add their own)
    for (int32_t t0 = odd_from; t0 < odd_to; t0 += 128) r.add_nonfinite(a, w, g, t0, t0 + 32);

    // merge the four waves: rows of HD + 4 floats keep 16-byte stores of
    // neighbouring rows on different banks
    const float l = other_sum(r.l);
    __syncthreads();
    if (r.half == 0) sm[wave * 32 + lane] = r.m, sl[wave * 32 + lane] = l;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            *reinterpret_cast<float4*>(oo + (wave * 32 + (lane & 31)) * kPad + d * 32 + 8 * e + 4 * r.half) =
                make_float4(r.o[d][4 * e], r.o[d][4 * e + 1], r.o[d][4 * e + 2], r.o[d][4 * e + 3]);
    __syncthreads();
    const uint32_t rows = min(w.rows - w.row0, 32u);
    for (uint32_t e = threadIdx.x; e < rows * (HD / 4); e += 256) {
        const uint32_t i = e / (HD / 4), d = e % (HD / 4) * 4;
        const float M = fmaxf(fmaxf(sm[i], sm[32 + i]), fmaxf(sm[64 + i], sm[96 + i]));
        float L = 0.0f;
        float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float m = sm[k * 32 + i], l1 = sl[k * 32 + i];
            if (m == -INFINITY && l1 == 0.0f) continue;  // no key of this row
            const float f = __builtin_amdgcn_exp2f(m - M);
            const float4 y = *reinterpret_cast<const float4*>(oo + (k * 32 + i) * kPad + d);
            L = __builtin_fmaf(l1, f, L);
            x.x = __builtin_fmaf(y.x, f, x.x), x.y = __builtin_fmaf(y.y, f, x.y);
            x.z = __builtin_fmaf(y.z, f, x.z), x.w = __builtin_fmaf(y.w, f, x.w);
        }
        const uint32_t t = (w.row0 + i) / a.G, h = g * a.G + (w.row0 + i) % a.G;
        if (a.parts_total == 1) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            put4<F32>(a.out, (w.tok0 + t) * a.out_stride + h * HD + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        } else {
            const uint64_t pr = (uint64_t)(a.part0 + part) * a.n_tokens * a.n_heads + (uint64_t)(w.tok0 + t) * a.n_heads + h;
            if (d == 0) *reinterpret_cast<float2*>(a.pml + pr * 2) = make_float2(M, L);
            put4<true>(a.po, pr * HD + d, x);
        }
    }
}

__device__ __forceinline__ float wave_max_all(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// One wave per (token, head): the parts of its keys joined, o = sum o_c 2^(m_c - M).
template <int HD, bool F32, int MODE>
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a) {
    constexpr int E = HD / 64;
    const uint64_t row = blockIdx.x * 4ull + block_wave();
    const uint32_t lane = threadIdx.x & 63;
    if (row >= (uint64_t)a.n_tokens * a.n_heads) return;
    const uint32_t tok = (uint32_t)(row / a.n_heads), head = (uint32_t)(row % a.n_heads);
    uint32_t s = tok, back = 0, na = 0, nb = 0;
    if (MODE == kPrompt && a.q_start) {
        s = wave_search(a.n, tok, [&](uint32_t i) { return (uint64_t)a.q_start[i]; });
        const uint32_t end = min(a.q_start[s + 1], a.n_tokens);
        if (tok < a.q_start[s] || tok >= end) return;
        back = end - 1 - tok;
    }
    const uint32_t len = seq_len(a, seq_id(a, s));
    if (MODE == kPrompt) {
        if (len > back) nb = min(a.n_parts, (len - back + a.chunk - 1) / a.chunk);
    } else {
        const uint32_t pre = shared_len(a, s, len);
        na = min(a.n_parts_prefix, pre ? (pre + a.chunk_prefix - 1) / a.chunk_prefix : 0);
        if (len > pre) nb = min(a.n_parts, (len - (pre & ~15u) + a.chunk - 1) / a.chunk);
    }
    const uint64_t rows = (uint64_t)a.n_tokens * a.n_heads;
    auto at = [&](uint32_t i) { return (uint64_t)(i < na ? i : a.n_parts_prefix + i - na) * rows + row; };
    float M = -INFINITY;
    for (uint32_t i = lane; i < na + nb; i += 64) M = fmaxf(M, a.pml[at(i) * 2]);
    M = wave_max_all(M);
    float L = 0.0f, o[E] = {};
    for (uint32_t i = 0; i < na + nb; i++) {
        const uint64_t p = at(i);
        const float2 ml = *reinterpret_cast<const float2*>(a.pml + p * 2);
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // no key of this row
        const float f = __builtin_amdgcn_exp2f(ml.x - M);
        L = __builtin_fmaf(ml.y, f, L);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(a.po[p * HD + lane * E + e], f, o[e]);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const uint64_t to = tok * a.out_stride + head * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if constexpr (F32) static_cast<float*>(a.out)[to + e] = o[e] * inv;
        else static_cast<_Float16*>(a.out)[to + e] = (_Float16)(o[e] * inv);
    }
}

int attention_status(const ane_paged_cache* c, uint32_t layer, uint32_t n, uint32_t n_tokens, int type, const void* q,
                     uint64_t q_stride, float scale, const void* out, uint64_t out_stride) {
    const int st = cache_status(c);
    if (st) return st;
    const uint32_t size = type == ANE_TYPE_F32 ? 4 : 2;
    const uint64_t width = (uint64_t)c->n_heads * c->head_dim;
    if (layer >= c->n_layers || n_tokens > kMaxTokens || n > kMaxTokens ||
        (type != ANE_TYPE_F32 && type != ANE_TYPE_F16) || !(scale > 0.0f) || !isfinite(scale))
        return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    if (!q || !out) return ANE_ERR_BAD_POINTER;
    if ((((uintptr_t)q) | ((uintptr_t)out)) & 15 || (q_stride * size) & 15 || (out_stride * size) & 15 ||
        q_stride < width || out_stride < width)
        return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}

// One launch: which kernel, over how many row tiles, its keys in how many parts.
struct Launch {
    bool few;
    uint64_t slots;
    uint32_t chunk, parts;
};

// units: sequences (groups) of the launch, tokens: rows before the heads of a
// group are counted; single: one token each.
Launch plan(const ane_paged_cache* c, uint32_t units, uint64_t tokens, bool single, uint64_t max_len) {
    Launch l;
    const uint64_t G = c->n_heads / c->n_kv_heads;
    l.few = tokens * G <= 32ull * units;
    const uint64_t bm = l.few ? 32 : 128;
    l.slots = single ? units * ((G + bm - 1) / bm) : tokens * G / bm + units;
    const uint64_t wgs = l.slots * c->n_kv_heads, step = l.few ? 128 : 64, least = l.few ? 256 : 512;
    uint64_t parts = (512 + wgs - 1) / wgs;
    parts = std::max<uint64_t>(1, std::min(parts, (max_len + least - 1) / least));
    l.chunk = (uint32_t)(((max_len + parts - 1) / parts + step - 1) / step * step);
    l.parts = (uint32_t)((max_len + l.chunk - 1) / l.chunk);
    return l;
}

uint64_t bound_len(const ane_paged_cache* c, uint32_t max_len) {
    return max_len == 0 || max_len > page_cap(c) ? page_cap(c) : max_len;
}

size_t parts_bytes(const ane_paged_cache* c, uint32_t n_tokens, uint32_t parts, size_t* ml) {
    if (parts <= 1) return 0;
    const uint64_t rows = (uint64_t)n_tokens * c->n_heads * parts;
    const size_t o = ceil_to(rows * c->head_dim * 4, 256);
    if (ml) *ml = o;
    return o + ceil_to(rows * 8, 256);
}

template <int HD, bool F32, int MODE>
void launch(const AttnArgs& a, const Launch& l, hipStream_t s) {
    const dim3 grid((uint32_t)(l.slots * a.n_kv), l.parts);
    if (l.few) hipLaunchKernelGGL((k_attn_few<HD, F32, MODE>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attn_block<HD, F32, MODE>), grid, dim3(256), 0, s, a, (uint32_t)l.slots);
}
template <int MODE>
void launch_as(const AttnArgs& a, const Launch& l, uint32_t hd, int type, hipStream_t s) {
    if (hd == 128) type == ANE_TYPE_F32 ? launch<128, true, MODE>(a, l, s) : launch<128, false, MODE>(a, l, s);
    else type == ANE_TYPE_F32 ? launch<64, true, MODE>(a, l, s) : launch<64, false, MODE>(a, l, s);
}
template <int MODE>
void join_as(const AttnArgs& a, uint32_t hd, int type, hipStream_t s) {
    auto* f = hd == 128 ? (type == ANE_TYPE_F32 ? k_attn_join<128, true, MODE> : k_attn_join<128, false, MODE>)
                        : (type == ANE_TYPE_F32 ? k_attn_join<64, true, MODE> : k_attn_join<64, false, MODE>);
    const uint64_t rows = (uint64_t)a.n_tokens * a.n_heads;
    hipLaunchKernelGGL(f, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a);
}

bool plan_fits(const ane_paged_cache* c, const Launch& l, uint64_t n_tokens, uint32_t parts_total) {
    return launch_fits(l.slots * c->n_kv_heads, 256) && l.parts <= 65535 &&
           (parts_total == 1 || launch_fits((n_tokens * c->n_heads + 3) / 4, 256));
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
    page_div(a.ps, &a.div_magic, &a.div_shift);
    a.scale_log2e = (float)((double)scale * 1.4426950408889634);
    return a;
}

bool bad_workspace(const void* ws, size_t bytes, size_t need) {
    return need && (!ws || (((uintptr_t)ws) & 255) || bytes < need);
}

}  // namespace
}  // namespace ane

using namespace ane;

extern "C" size_t ane_hip_attention_prompt_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                                          uint32_t max_len) {
    if (cache_status(cache) || n == 0 || n_tokens == 0 || n > kMaxTokens || n_tokens > kMaxTokens) return 0;
    // the same for a batch of single tokens with and without q_start
    const Launch l = plan(cache, n, n_tokens, false, bound_len(cache, max_len));
    const Launch one = plan(cache, n, n_tokens, true, bound_len(cache, max_len));
    return parts_bytes(cache, n_tokens, n_tokens == n ? std::max(l.parts, one.parts) : l.parts, nullptr);
}

extern "C" int ane_hip_attention_prompt(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                        const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len, int type,
                                        const void* q, uint64_t q_stride, float scale, void* out, uint64_t out_stride,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    const int st = attention_status(cache, layer, n, n_tokens, type, q, q_stride, scale, out, out_stride);
    if (st) return st;
    if (!q_start && n_tokens != n) return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    const Launch l = plan(cache, n, n_tokens, !q_start, bound_len(cache, max_len));
    if (!plan_fits(cache, l, n_tokens, l.parts)) return ANE_ERR_INVALID_ARG;
    size_t ml = 0;
    if (bad_workspace(workspace, workspace_bytes, parts_bytes(cache, n_tokens, l.parts, &ml))) return ANE_ERR_WORKSPACE;
    AttnArgs a = attn_args(cache, layer, seqs, n, n_tokens, q, q_stride, scale, out, out_stride);
    a.q_start = q_start;
    a.po = static_cast<float*>(workspace);
    a.pml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ml);
    a.chunk = l.chunk, a.n_parts = a.parts_total = l.parts;
    hipStream_t s = (hipStream_t)stream;
    launch_as<kPrompt>(a, l, cache->head_dim, type, s);
    if (l.parts > 1) join_as<kPrompt>(a, cache->head_dim, type, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

namespace {
struct SharedPlan {
    Launch prefix, own;
    uint32_t parts;
};
SharedPlan shared_plan(const ane_paged_cache* c, uint32_t n, uint32_t n_groups, uint32_t max_prefix, uint32_t max_len) {
    SharedPlan p = {};
    p.own = plan(c, n, n, true, bound_len(c, max_len));
    if (n_groups) p.prefix = plan(c, n_groups, n, false, bound_len(c, max_prefix));
    p.parts = p.prefix.parts + p.own.parts;
    return p;
}
}  // namespace

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
    a.chunk_prefix = p.prefix.chunk, a.n_parts_prefix = p.prefix.parts;
    hipStream_t s = (hipStream_t)stream;
    if (n_groups) {
        a.chunk = p.prefix.chunk, a.n_parts = p.prefix.parts, a.part0 = 0;
        launch_as<kPrefix>(a, p.prefix, cache->head_dim, type, s);
    }
    a.chunk = p.own.chunk, a.n_parts = p.own.parts, a.part0 = p.prefix.parts;
    launch_as<kOwn>(a, p.own, cache->head_dim, type, s);
    if (p.parts > 1) join_as<kOwn>(a, cache->head_dim, type, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}
