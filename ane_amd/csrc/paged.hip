// paged.hip -- the paged K/V cache: RoPE and append of packed tokens, and the
// page calls (reserve, fork, free, copy, compact).
//
// The page calls keep their whole state on the device: one workgroup looks
// through the reference counts and assigns pages (the lowest free ones first,
// by prefix sums and not by atomics, so that a result never depends on
// timing), then a wide launch moves the data.
#include "paged.hpp"

namespace ane {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------ RoPE + append
struct AppendArgs {
    const void *q, *k, *v;
    void* q_out;
    const float* rope;
    uint16_t *kp, *vp;  // this layer's pages
    const uint32_t *table, *kv_len, *seqs, *q_start;
    uint64_t q_stride, kv_stride, q_out_stride;
    uint32_t n, rope_len, n_heads, n_kv, hd, ps, n_pages, max_pages, n_seqs;
};

template <class T>
__device__ __forceinline__ void load8(const void* p, uint64_t i, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const h8 a = *reinterpret_cast<const h8*>(static_cast<const _Float16*>(p) + i);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)a[e];
    }
}
template <class T>
__device__ __forceinline__ void store8(void* p, uint64_t i, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        float* o = static_cast<float*>(p) + i;
        *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(o + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        h8 a;
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] = (_Float16)x[e];
        *reinterpret_cast<h8*>(static_cast<_Float16*>(p) + i) = a;
    }
}

// One workgroup per token; a thread takes 8 values (4 pairs) of one head at a
// time: [q heads | k heads | v heads] x hd/8 units.  The values of the first
// kAhead units are loaded before the token's sequence is looked up, so that
// the chain start -> length -> page runs while they arrive.  Bound by memory: 8000
// tokens of 32 + 8 + 8 128-wide heads, fp32 in and fp16 out, 347 MB in 64 us, 5.4
// TB/s; 64 single tokens 4.6 us, the chain.
constexpr uint32_t kAhead = 3;
template <class TI, class TQ>
__global__ void __launch_bounds__(256) k_paged_append(AppendArgs a) {
    const uint32_t t = blockIdx.x, tid = threadIdx.x;
    const uint32_t per = a.hd / 8, qu = a.q ? a.n_heads * per : 0, ku = a.n_kv * per, units = qu + 2 * ku;
    auto load = [&](uint32_t u, float(&x)[8]) {
        if (u < qu) load8<TI>(a.q, t * a.q_stride + u * 8, x);
        else if (u < qu + ku) load8<TI>(a.k, t * a.kv_stride + (u - qu) * 8, x);
        else if (u < units) load8<TI>(a.v, t * a.kv_stride + (u - qu - ku) * 8, x);
    };
    float x[kAhead][8];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++) load(tid + i * 256, x[i]);

    // the token's sequence, position and page
    uint32_t s = t, first = t, last = t + 1;
    if (a.q_start) {
        s = wave_search(a.n, t, [&](uint32_t i) { return (uint64_t)a.q_start[i]; });
        first = a.q_start[s];
        last = a.q_start[s + 1];
        if (t < first || t >= last) return;  // before the first sequence or behind the last
    }
    const uint32_t id = a.seqs ? a.seqs[s] : s;
    int64_t pos = -1;
    uint32_t page = ANE_NO_PAGE, row = 0;
    if (id < a.n_seqs) {
        // (the length as attention counts it, or a row would see another token's keys)
        pos = (int64_t)min((uint64_t)a.kv_len[id], (uint64_t)a.max_pages * a.ps) - (int64_t)(last - t);
        if (pos >= 0 && (!a.rope || pos < a.rope_len)) {
            page = a.table[(uint64_t)id * a.max_pages + (uint32_t)pos / a.ps];
            row = (uint32_t)pos % a.ps;
        } else {
            pos = -1;
        }
    }
    auto put = [&](uint32_t u, float(&v)[8]) {
        if (u >= units) return;
        const bool isv = u >= qu + ku;
        const uint32_t d = u % per * 8;
        if (pos < 0) {
            if (u < qu) {
                const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                store8<TQ>(a.q_out, t * a.q_out_stride + u * 8, z);
            }
            return;
        }
        if (a.rope && !isv) {
            const float* cs = a.rope + (uint64_t)pos * a.hd + d;
            float c[8];
#pragma unroll
            for (int e = 0; e < 8; e++) c[e] = cs[e];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p = v[e], r = v[e + 1];
                v[e] = __fsub_rn(__fmul_rn(p, c[e]), __fmul_rn(r, c[e + 1]));
                v[e + 1] = __fadd_rn(__fmul_rn(p, c[e + 1]), __fmul_rn(r, c[e]));
            }
        }
        if (u < qu) {
            store8<TQ>(a.q_out, t * a.q_out_stride + u * 8, v);
        } else if (page < a.n_pages) {
            const uint32_t g = (u - qu - (isv ? ku : 0)) / per;
            store8<_Float16>(isv ? a.vp : a.kp, (((uint64_t)page * a.n_kv + g) * a.ps + row) * a.hd + d, v);
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++) put(tid + i * 256, x[i]);
    for (uint32_t u = tid + kAhead * 256; u < units; u += 256) {
        load(u, x[0]);
        put(u, x[0]);
    }
}

// -------------------------------------------------------- assigning pages
constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kLook = 1 << 16;

// Prefix sums over the workgroup's 1024 threads, this thread's value included;
// *total: the sum.  Sums stop at kMany, more than any pool's pages.  Within a
// wave by DPP shifts (a row of 16 lanes, then row 0 into 1 and 2 into 3, then the
// first half into the second): as shuffles the three of a plan took 1.5 us.
constexpr uint32_t kMany = 0x7fffffff;
__device__ __forceinline__ uint32_t add_up(uint32_t a, uint32_t b) { return min(a + b, kMany); }
template <int ctrl, int rows>
__device__ __forceinline__ uint32_t add_shifted(uint32_t v) {
    return add_up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = add_shifted<0x111, 0xf>(v);  // row_shr:1
    v = add_shifted<0x112, 0xf>(v);
    v = add_shifted<0x114, 0xf>(v);
    v = add_shifted<0x118, 0xf>(v);
    v = add_shifted<0x142, 0xa>(v);  // row_bcast:15
    return add_shifted<0x143, 0xc>(v);  // row_bcast:31
}
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* total) {
    __shared__ uint32_t sums[kPlanWaves];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t s = wave_scan(v);
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    const uint32_t t = wave_scan(lane < kPlanWaves ? sums[lane] : 0);  // the waves' sums, scanned by every wave
    const uint32_t before = wave ? __builtin_amdgcn_readlane(t, wave - 1) : 0;
    *total = __builtin_amdgcn_readlane(t, kPlanWaves - 1);
    __syncthreads();
    return add_up(before, s);
}

// The free pages as bits in LDS, 65536 pages a look: a smaller pool is looked at
// once, however many passes a call makes over it.  Short loops on purpose: one
// workgroup runs them once, and what it waits for is mostly code and the few
// loads (unrolled over registers, the plan of a compaction took 13 us, not 6).
struct Pool {
    const uint32_t* refs;
    uint32_t pages;
    uint64_t* bits;    // [kLook / 64], 1: free
    uint32_t* before;  // [kLook / 64]

    __device__ __forceinline__ void look(uint64_t base) const {
        const uint32_t lane = threadIdx.x & 63, masks = (uint32_t)min((uint64_t)kLook, pages - base + 63) / 64;
        for (uint32_t j = threadIdx.x >> 6; j < masks; j += 4 * kPlanWaves) {
            uint32_t r[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint64_t i = base + (j + k * kPlanWaves) * 64 + lane;
                r[k] = i < pages ? refs[i] : 1;
            }
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint64_t m = __ballot(r[k] == 0);
                if (lane == 0 && j + k * kPlanWaves < masks) bits[j + k * kPlanWaves] = m;
            }
        }
        __syncthreads();
    }
    // The free (or live) pages i in [from, to) in ascending order: found(rank, i)
    // for each of the first `want`; returns how many there are (counting stops
    // once `want` are found).  After a look at the pool's first pages; the whole
    // workgroup calls it.
    template <class Found>
    __device__ __forceinline__ uint32_t pick(bool free, uint32_t from, uint32_t to, uint32_t want, Found found) const {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t have = 0;
        for (uint64_t base = from / kLook * kLook; base < to && have < want; base += kLook) {
            if (pages > kLook) look(base);
            const uint32_t masks = (uint32_t)min((uint64_t)kLook, pages - base + 63) / 64;
            auto mask = [&](uint32_t j) {  // those of [from, to)
                uint64_t m = free ? bits[j] : ~bits[j];
                const uint64_t i = base + j * 64ull;
                if (i < from) m &= from - i < 64 ? ~0ull << (from - i) : 0;
                if (i + 64 > to) m &= to > i ? ~0ull >> (64 - (to - i)) : 0;
                return m;
            };
            uint32_t all;
            const uint32_t mine = threadIdx.x < masks ? __popcll(mask(threadIdx.x)) : 0;
            before[threadIdx.x] = block_scan(mine, &all) - mine;
            __syncthreads();
            for (uint32_t j = threadIdx.x >> 6; j < masks; j += kPlanWaves) {
                const uint64_t m = mask(j);
                const uint32_t rank = have + before[j] + __popcll(m & ((1ull << lane) - 1));
                if ((m >> lane & 1) && rank < want) found(rank, (uint32_t)(base + j * 64 + lane));
            }
            have += all;
            __syncthreads();
        }
        return have;
    }
};
static_assert(kLook / 64 == kPlanThreads, "a thread a mask");

struct PagesWs {
    uint32_t *list, *movers, *map;  // [n_pages] each
    uint32_t* claim;                // [n_seqs]
    uint32_t *req_len, *req_page;   // [kMaxRequests]
    uint32_t* count;                // [2]: pages to move, live pages
};

size_t pages_layout(const ane_paged_cache* c, void* base, PagesWs* w) {
    size_t off = 0;
    auto take = [&](uint64_t words) {
        const size_t o = off;
        off += ceil_to(words * 4, 256);
        return base ? reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(base) + o) : nullptr;
    };
    PagesWs p;
    p.list = take(c->n_pages);
    p.movers = take(c->n_pages);
    p.map = take(c->n_pages);
    p.claim = take(c->n_seqs);
    p.req_len = take(kMaxRequests);
    p.req_page = take(kMaxRequests);
    p.count = take(2);
    if (w) *w = p;
    return off;
}

// claim[seq] = the first valid request that names it (seq(i): ANE_NO_PAGE for one
// that is not valid).  In LDS where the cache has few sequences.
constexpr uint32_t kLdsSeqs = 4096, kLdsList = 4096;
template <class Seq>
__device__ __forceinline__ void claim_first(uint32_t n, uint32_t* claim, Seq seq) {
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const uint32_t s = seq(i);
        if (s != ANE_NO_PAGE) claim[s] = ANE_NO_PAGE;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const uint32_t s = seq(i);
        if (s != ANE_NO_PAGE) atomicMin(&claim[s], i);
    }
    __syncthreads();
}

// A request of a planning pass: its sequence (ANE_NO_PAGE: not valid), the pages
// it asks for, and what its call needs besides.  A thread keeps those of the first
// 1024 requests; the others are looked up again in each pass.
struct Request {
    uint32_t seq, need, x, y;
};

// Passes over the requests: who names a sequence first, how many pages are asked
// for, which are free, and then done(i, request, served, its pages), by every
// thread (not served from i = n on).
template <class Look, class Done>
__device__ __forceinline__ void serve(const ane_paged_cache& c, uint32_t n, PagesWs& w, Look look, Done done) {
    __shared__ uint32_t claim_lds[kLdsSeqs], list_lds[kLdsList], before_lds[kPlanThreads];
    __shared__ uint64_t bits[kPlanThreads];
    const uint32_t tid = threadIdx.x;
    const Pool pool = {c.page_refs, c.n_pages, bits, before_lds};
    // (waves without a request are at the counts meanwhile)
    const Request mine = tid < n ? look(tid) : Request{ANE_NO_PAGE, 0, 0, 0};
    pool.look(0);
    auto request = [&](uint32_t i) { return i == tid ? mine : look(i); };
    uint32_t* claim = c.n_seqs <= kLdsSeqs ? claim_lds : w.claim;
    claim_first(n, claim, [&](uint32_t i) { return request(i).seq; });
    auto valid = [&](uint32_t i, const Request& r) {
        return r.seq != ANE_NO_PAGE && __atomic_load_n(&claim[r.seq], __ATOMIC_RELAXED) == i;
    };
    uint32_t total = 0;
    for (uint32_t base = 0; base < n; base += kPlanThreads) {
        const uint32_t i = base + tid;
        uint32_t k = 0, all;
        if (i < n) {
            const Request r = request(i);
            if (valid(i, r)) k = r.need;
        }
        block_scan(k, &all);
        total = add_up(total, all);
    }
    const uint32_t want = min(total, c.n_pages);
    uint32_t* list = want <= kLdsList ? list_lds : w.list;
    const uint32_t have = pool.pick(true, 0, c.n_pages, want, [&](uint32_t rank, uint32_t i) { list[rank] = i; });
    uint32_t before = 0;
    for (uint32_t base = 0; base < n; base += kPlanThreads) {
        const uint32_t i = base + tid;
        Request r = {ANE_NO_PAGE, 0, 0, 0};
        bool ok = false;
        if (i < n) {
            r = request(i);
            ok = valid(i, r);
        }
        uint32_t all;
        const uint32_t end = add_up(before, block_scan(ok ? r.need : 0, &all));
        before = add_up(before, all);
        done(i, r, ok && end <= have && end < kMany, list + (end - (ok ? r.need : 0)));
    }
}

__global__ void __launch_bounds__(kPlanThreads)
k_pages_reserve(ane_paged_cache c, uint32_t n, const uint32_t* seqs, const uint32_t* new_len, uint32_t* served,
                PagesWs w) {
    const uint64_t cap = (uint64_t)c.max_pages * c.page_size;
    serve(c, n, w,
          [&](uint32_t i) {  // x: the new length, y: the row's first new entry
              Request r = {seqs[i], 0, new_len[i], 0};
              if (r.seq >= c.n_seqs || r.x > cap) return Request{ANE_NO_PAGE, 0, 0, 0};
              r.y = (uint32_t)((min((uint64_t)c.kv_len[r.seq], cap) + c.page_size - 1) / c.page_size);
              const uint32_t to = (uint32_t)(((uint64_t)r.x + c.page_size - 1) / c.page_size);
              r.need = to > r.y ? to - r.y : 0;
              return r;
          },
          [&](uint32_t i, const Request& r, bool yes, const uint32_t* pages) {
              auto take = [&](uint32_t seq, uint32_t at, uint32_t p) {
                  c.page_table[(uint64_t)seq * c.max_pages + at] = p;
                  c.page_refs[p] = 1;
              };
              if (served && i < n) served[i] = yes;
              // a lane takes its own request's pages, one every 0.11 us, or the wave does
              // it for a few long ones, one request after the other, 0.3 us and more each
              // (one request for 8192 pages 906 -> 20 us, 32 for 256 each 55 -> 23; 1024
              // for 8 pages 24 us, by waves 42)
              const bool lengthy = yes && r.need > 16;
              const bool wide = lengthy && r.need > 4u * (uint32_t)__popcll(__ballot(lengthy));
              if (yes && !wide)
                  for (uint32_t j = 0; j < r.need; j++) take(r.seq, r.y + j, pages[j]);
              for (uint64_t m = __ballot(wide); m; m &= m - 1) {
                  const uint32_t l = __builtin_ctzll(m), lane = threadIdx.x & 63;
                  const uint32_t seq = __shfl(r.seq, l), at = __shfl(r.y, l), need = __shfl(r.need, l);
                  const uint32_t* from = reinterpret_cast<const uint32_t*>(__shfl(reinterpret_cast<uintptr_t>(pages), l));
                  for (uint32_t j = lane; j < need; j += 256) {
                      uint32_t x[4];
#pragma unroll
                      for (uint32_t k = 0; k < 4; k++) x[k] = from[min(j + k * 64, need - 1)];
#pragma unroll
                      for (uint32_t k = 0; k < 4; k++)
                          if (j + k * 64 < need) take(seq, at + j + k * 64, x[k]);
                  }
              }
              if (yes && r.x > c.kv_len[r.seq]) c.kv_len[r.seq] = r.x;
          });
}

// Which forks are served: the length each dst takes (0: none) and its fresh page.
__global__ void __launch_bounds__(kPlanThreads)
k_pages_fork_plan(ane_paged_cache c, uint32_t n, const uint32_t* src, const uint32_t* dst, uint32_t* served, PagesWs w) {
    const uint64_t cap = (uint64_t)c.max_pages * c.page_size;
    serve(c, n, w,
          [&](uint32_t i) {  // x: the length
              const uint32_t a = src[i], b = dst[i];
              if (a >= c.n_seqs || b >= c.n_seqs || a == b) return Request{ANE_NO_PAGE, 0, 0, 0};
              const uint32_t la = c.kv_len[a], lb = c.kv_len[b];
              if (lb != 0) return Request{ANE_NO_PAGE, 0, 0, 0};
              const uint32_t len = (uint32_t)min((uint64_t)la, cap);
              return Request{b, len % c.page_size != 0, len, 0};
          },
          [&](uint32_t i, const Request& r, bool yes, const uint32_t* pages) {
              if (i >= n) return;
              if (served) served[i] = yes;
              w.req_len[i] = yes ? r.x : 0;
              w.req_page[i] = yes && r.need ? pages[0] : ANE_NO_PAGE;
          });
}

// One workgroup per fork and slice of its work: slice 0 writes the row, the
// counts and the length; the used rows of the part page are copied by all
// slices, one wave per (layer, K or V, four kv heads), eight 16-byte vectors a
// lane in flight.  src rows are never written here: a src with positions is no
// dst.  56 forks of 32 layers, 99 MB in 19 us, 5.2 TB/s.
constexpr uint32_t kHeads = 4;
__global__ void __launch_bounds__(256)
k_pages_fork(ane_paged_cache c, const uint32_t* src, const uint32_t* dst, PagesWs w) {
    constexpr uint32_t kVecs = 2;
    const uint32_t i = blockIdx.x, len = w.req_len[i], fresh = w.req_page[i], from_seq = src[i];
    if (len == 0) return;
    const uint32_t whole = len / c.page_size, part = len % c.page_size;
    const uint32_t* from = c.page_table + (uint64_t)from_seq * c.max_pages;
    if (blockIdx.y == 0) {
        const uint32_t to = dst[i];
        uint32_t* row = c.page_table + (uint64_t)to * c.max_pages;
        for (uint32_t j = threadIdx.x; j < whole + (part ? 1 : 0); j += 256) {
            const uint32_t p = j < whole ? from[j] : fresh;
            row[j] = p;
            if (p < c.n_pages) atomicAdd(&c.page_refs[p], 1u);
        }
        if (threadIdx.x == 0) c.kv_len[to] = len;
    }
    if (!part) return;
    const uint32_t old = from[whole];
    if (old >= c.n_pages || fresh >= c.n_pages) return;
    const uint32_t lane = threadIdx.x & 63, hv = c.head_dim / 8;  // 16-byte vectors a row
    const uint32_t quads = (c.n_kv_heads + kHeads - 1) / kHeads, jobs = c.n_layers * 2 * quads, run = part * hv;
    const uint64_t head = (uint64_t)c.page_size * hv, page = head * c.n_kv_heads;
    for (uint32_t j = blockIdx.y * 4 + (threadIdx.x >> 6); j < jobs; j += gridDim.y * 4) {
        const uint32_t g0 = j % quads * kHeads, kv = j / quads & 1, l = j / quads / 2;
        v4u* pool = reinterpret_cast<v4u*>(kv ? c.v_pages : c.k_pages) + (uint64_t)l * c.n_pages * page + g0 * head;
        const v4u* a = pool + old * page;
        v4u* b = pool + fresh * page;
        for (uint32_t e = lane; e < run; e += kVecs * 64) {
            // unconditional loads (a vector past the end or a head past the last
            // reads one of its own again): all in flight before the first store
            v4u t[kHeads][kVecs];
#pragma unroll
            for (uint32_t h = 0; h < kHeads; h++)
#pragma unroll
                for (uint32_t k = 0; k < kVecs; k++) t[h][k] = a[min(h, c.n_kv_heads - 1 - g0) * head + min(e + k * 64, run - 1)];
#pragma unroll
            for (uint32_t h = 0; h < kHeads; h++)
#pragma unroll
                for (uint32_t k = 0; k < kVecs; k++)
                    if (g0 + h < c.n_kv_heads && e + k * 64 < run) b[h * head + e + k * 64] = t[h][k];
        }
    }
}

// One workgroup per request; of two that name a sequence the first to take its
// length gives its pages up.
__global__ void __launch_bounds__(256) k_pages_free(ane_paged_cache c, const uint32_t* seqs) {
    __shared__ uint32_t len_sh;
    const uint32_t s = seqs[blockIdx.x];
    if (s >= c.n_seqs) return;
    if (threadIdx.x == 0) len_sh = atomicExch(&c.kv_len[s], 0u);
    __syncthreads();
    const uint64_t len = min((uint64_t)len_sh, (uint64_t)c.max_pages * c.page_size);
    const uint32_t pages = (uint32_t)((len + c.page_size - 1) / c.page_size);
    uint32_t* row = c.page_table + (uint64_t)s * c.max_pages;
    for (uint32_t j = threadIdx.x; j < pages; j += 256) {
        const uint32_t p = row[j];
        row[j] = ANE_NO_PAGE;
        if (p < c.n_pages && atomicSub(&c.page_refs[p], 1u) == 0) atomicAdd(&c.page_refs[p], 1u);  // never below 0
    }
}

// The moves of a compaction: the r-th live page at or past the live count into
// the r-th free one before it; the counts and the numbers that follow.
__global__ void __launch_bounds__(kPlanThreads)
k_pages_compact_plan(ane_paged_cache c, uint32_t* refs_out, uint32_t* n_live, PagesWs w) {
    __shared__ uint32_t list_lds[kLdsList], before_lds[kPlanThreads];
    __shared__ uint64_t bits[kPlanThreads];
    const uint32_t* refs = c.page_refs;
    const Pool pool = {refs, c.n_pages, bits, before_lds};
    pool.look(0);
    const uint32_t n = pool.pick(false, 0, c.n_pages, ~0u, [](uint32_t, uint32_t) {});
    const uint32_t holes = pool.pick(true, 0, n, ~0u, [&](uint32_t rank, uint32_t i) {
        w.list[rank] = i;
        if (rank < kLdsList) list_lds[rank] = i;
    });
    // numbers at or past the live count: a live page's new one, another's own
    for (uint64_t i = n + threadIdx.x; i < c.n_pages; i += kPlanThreads) w.map[i] = (uint32_t)i;
    if (refs_out != refs)
        for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) refs_out[i] = refs[i];
    __syncthreads();
    pool.pick(false, n, c.n_pages, ~0u, [&](uint32_t rank, uint32_t i) {
        const uint32_t to = rank < kLdsList ? list_lds[rank] : w.list[rank];
        w.movers[rank] = i;
        w.map[i] = to;
        refs_out[to] = refs[i];
    });
    for (uint64_t i = n + threadIdx.x; i < c.n_pages; i += kPlanThreads) refs_out[i] = 0;
    if (threadIdx.x == 0) {
        *w.count = holes;
        if (n_live) *n_live = n;
        w.count[1] = n;
    }
}

// Page copies, 16 KB of a page a workgroup at a time; source and destination
// pages are disjoint.  n: on the device for a compaction.  256 MB in 53 us, 4.8
// TB/s, as a large copy.
constexpr uint32_t kCopyVecs = 1024;  // 16-byte vectors a step
__device__ __forceinline__ void copy_pages(const ane_paged_cache& c, uint32_t n, const uint32_t* src, const uint32_t* dst) {
    const uint64_t vecs = (uint64_t)c.n_kv_heads * c.page_size * (c.head_dim / 8);
    const uint64_t steps = (vecs + kCopyVecs - 1) / kCopyVecs, jobs = (uint64_t)n * c.n_layers * 2 * steps;
    for (uint64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const uint64_t st = j % steps, r = j / steps;
        const uint32_t kv = r & 1, l = (uint32_t)(r / 2 % c.n_layers), i = (uint32_t)(r / 2 / c.n_layers);
        const uint32_t a = src[i], b = dst[i];
        if (a >= c.n_pages || b >= c.n_pages || a == b) continue;
        v4u* pool = reinterpret_cast<v4u*>(kv ? c.v_pages : c.k_pages) + (uint64_t)l * c.n_pages * vecs;
        const v4u* from = pool + a * vecs;
        v4u* to = pool + b * vecs;
        v4u t[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint64_t e = st * kCopyVecs + k * 256 + threadIdx.x;
            if (e < vecs) t[k] = from[e];
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint64_t e = st * kCopyVecs + k * 256 + threadIdx.x;
            if (e < vecs) to[e] = t[k];
        }
    }
}
__global__ void __launch_bounds__(256)
k_pages_copy(ane_paged_cache c, uint32_t n, const uint32_t* src, const uint32_t* dst) {
    copy_pages(c, n, src, dst);
}
__global__ void __launch_bounds__(256) k_pages_compact(ane_paged_cache c, uint32_t* table_out, PagesWs w) {
    const uint32_t live = w.count[1];
    const uint64_t entries = (uint64_t)c.n_seqs * c.max_pages;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < entries; i += gridDim.x * 256ull) {
        const uint32_t p = c.page_table[i];
        const uint32_t to = p >= live && p < c.n_pages ? w.map[p] : p;
        if (to != p || table_out != c.page_table) table_out[i] = to;
    }
    copy_pages(c, *w.count, w.movers, w.list);
}

int pages_status(const ane_paged_cache* c, uint32_t n) {
    const int st = cache_status(c);
    if (st) return st;
    if (!c->page_refs) return ANE_ERR_BAD_POINTER;
    return n > kMaxRequests ? ANE_ERR_INVALID_ARG : ANE_OK;
}
bool bad_workspace(const void* ws, size_t bytes, size_t need) {
    return need && (!ws || (((uintptr_t)ws) & 255) || bytes < need);
}
uint32_t copy_grid(uint64_t jobs) { return (uint32_t)(jobs < 4096 ? (jobs ? jobs : 1) : 4096); }

}  // namespace
}  // namespace ane

using namespace ane;

extern "C" int ane_hip_paged_rope_append(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                         const uint32_t* q_start, uint32_t n_tokens, int in_type, const void* q,
                                         uint64_t q_stride, const void* k, const void* v, uint64_t kv_stride,
                                         const float* rope_table, uint32_t rope_len, int q_out_type, void* q_out,
                                         uint64_t q_out_stride, void* stream) {
    const int st = cache_status(cache);
    if (st) return st;
    if (layer >= cache->n_layers || n_tokens > kMaxTokens || (in_type != ANE_TYPE_F32 && in_type != ANE_TYPE_F16) ||
        (q_out_type != ANE_TYPE_F32 && q_out_type != ANE_TYPE_F16) || (!q_start && n_tokens != n) ||
        (rope_table && rope_len == 0))
        return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    if (!k || !v || (!q != !q_out)) return ANE_ERR_BAD_POINTER;
    const uint32_t isz = in_type == ANE_TYPE_F32 ? 4 : 2, osz = q_out_type == ANE_TYPE_F32 ? 4 : 2;
    if ((((uintptr_t)q) | ((uintptr_t)k) | ((uintptr_t)v) | ((uintptr_t)q_out) | ((uintptr_t)rope_table)) & 15 ||
        (kv_stride * isz) & 15 || kv_stride < (uint64_t)cache->n_kv_heads * cache->head_dim ||
        (q && ((q_stride * isz) & 15 || (q_out_stride * osz) & 15 ||
               q_stride < (uint64_t)cache->n_heads * cache->head_dim ||
               q_out_stride < (uint64_t)cache->n_heads * cache->head_dim)))
        return ANE_ERR_INVALID_ARG;
    AppendArgs a;
    const uint64_t lo = page_elems(cache) * cache->n_pages * layer;
    a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.rope = rope_table;
    a.kp = cache->k_pages + lo, a.vp = cache->v_pages + lo;
    a.table = cache->page_table, a.kv_len = cache->kv_len, a.seqs = seqs, a.q_start = q_start;
    a.q_stride = q_stride, a.kv_stride = kv_stride, a.q_out_stride = q_out_stride;
    a.n = n, a.rope_len = rope_len, a.n_heads = cache->n_heads, a.n_kv = cache->n_kv_heads;
    a.hd = cache->head_dim, a.ps = cache->page_size, a.n_pages = cache->n_pages, a.max_pages = cache->max_pages;
    a.n_seqs = cache->n_seqs;
    auto* f = in_type == ANE_TYPE_F32
                  ? (q_out_type == ANE_TYPE_F32 ? k_paged_append<float, float> : k_paged_append<float, _Float16>)
                  : (q_out_type == ANE_TYPE_F32 ? k_paged_append<_Float16, float> : k_paged_append<_Float16, _Float16>);
    hipLaunchKernelGGL(f, dim3(n_tokens), dim3(256), 0, (hipStream_t)stream, a);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" size_t ane_hip_pages_workspace_size(const ane_paged_cache* cache) {
    return cache_status(cache) ? 0 : pages_layout(cache, nullptr, nullptr);
}

extern "C" int ane_hip_pages_reserve(const ane_paged_cache* cache, uint32_t n, const uint32_t* seqs,
                                     const uint32_t* new_len, uint32_t* served, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    const int st = pages_status(cache, n);
    if (st || n == 0) return st;
    if (!seqs || !new_len) return ANE_ERR_BAD_POINTER;
    if (bad_workspace(workspace, workspace_bytes, pages_layout(cache, nullptr, nullptr))) return ANE_ERR_WORKSPACE;
    PagesWs w;
    pages_layout(cache, workspace, &w);
    hipLaunchKernelGGL(k_pages_reserve, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *cache, n, seqs, new_len,
                       served, w);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" int ane_hip_pages_fork(const ane_paged_cache* cache, uint32_t n, const uint32_t* src, const uint32_t* dst,
                                  uint32_t* served, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = pages_status(cache, n);
    if (st || n == 0) return st;
    if (!src || !dst) return ANE_ERR_BAD_POINTER;
    if (bad_workspace(workspace, workspace_bytes, pages_layout(cache, nullptr, nullptr))) return ANE_ERR_WORKSPACE;
    PagesWs w;
    pages_layout(cache, workspace, &w);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(k_pages_fork_plan, dim3(1), dim3(kPlanThreads), 0, s, *cache, n, src, dst, served, w);
    // four jobs a workgroup; at most 4096 workgroups more than the forks
    const uint64_t quads = (cache->n_kv_heads + kHeads - 1) / kHeads, jobs = ((uint64_t)cache->n_layers * 2 * quads + 3) / 4;
    const uint64_t room = 4096 / n + 1;
    hipLaunchKernelGGL(k_pages_fork, dim3(n, (uint32_t)(jobs < room ? jobs : room)), dim3(256), 0, s, *cache, src, dst, w);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" int ane_hip_pages_free(const ane_paged_cache* cache, uint32_t n, const uint32_t* seqs, void* stream) {
    const int st = pages_status(cache, n);
    if (st || n == 0) return st;
    if (!seqs) return ANE_ERR_BAD_POINTER;
    hipLaunchKernelGGL(k_pages_free, dim3(n), dim3(256), 0, (hipStream_t)stream, *cache, seqs);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" int ane_hip_pages_copy(const ane_paged_cache* cache, uint32_t n, const uint32_t* src, const uint32_t* dst,
                                  void* stream) {
    const int st = pages_status(cache, n);
    if (st || n == 0) return st;
    if (!src || !dst) return ANE_ERR_BAD_POINTER;
    const uint64_t steps = (page_elems(cache) / 8 + kCopyVecs - 1) / kCopyVecs;
    hipLaunchKernelGGL(k_pages_copy, dim3(copy_grid(steps * 2 * cache->n_layers * n)), dim3(256), 0, (hipStream_t)stream,
                       *cache, n, src, dst);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" int ane_hip_pages_compact(const ane_paged_cache* cache, uint32_t* page_table_out, uint32_t* page_refs_out,
                                     uint32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = pages_status(cache, 0);
    if (st) return st;
    if (bad_workspace(workspace, workspace_bytes, pages_layout(cache, nullptr, nullptr))) return ANE_ERR_WORKSPACE;
    PagesWs w;
    pages_layout(cache, workspace, &w);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(k_pages_compact_plan, dim3(1), dim3(kPlanThreads), 0, s, *cache,
                       page_refs_out ? page_refs_out : cache->page_refs, n_live, w);
    const uint64_t steps = (page_elems(cache) / 8 + kCopyVecs - 1) / kCopyVecs;
    hipLaunchKernelGGL(k_pages_compact, dim3(copy_grid(steps * 2 * cache->n_layers * (uint64_t)cache->n_pages)), dim3(256),
                       0, s, *cache, page_table_out ? page_table_out : cache->page_table, w);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}
