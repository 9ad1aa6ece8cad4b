// kv_decode.cu — attention of a few query rows per sequence over the paged 8-bit cache
// (mrl_kv_attend, include/mrl_kv.h), one launch for every 1,024 sequences.
//
// An item is 16 query rows (tokens x the query heads of one kv head) of one sequence: their K and V pages
// are read once and serve all 16. The page is the unit of work: one warp takes a page of 64 tokens,
// S = Q K^T and O += P V by m16n8k16 products with the codes widened to f16 on the way from shared
// memory (exact: |code| <= 128), and the page's two scales applied to S and to P, which are f32 there.
// Softmax statistics are kept per warp in f32, joined over the warps of a team in shared memory, and over
// teams through global partials that the last team to arrive adds up in team order, so results do not
// depend on scheduling.
//
// The page's layout is the one the products want: a row of 64 bytes has the index that is summed over
// contiguous, each of 4 lanes takes 16 of them as four k-steps' worth, and 8 lanes cover two rows, so
// every 16-byte shared-memory load of a warp is free of conflicts and needs no transposition: K's token
// order in the score tile is chosen so that a lane's scores are 16 consecutive tokens, V's row order.
//
// Bound by HBM for long contexts (2 x 64 x head_dim bytes a page), by latency for short ones. Measured on one B200, 8 kv
// heads of 128, four query heads each: 4 sequences of 130,000 tokens 175 us (6.10 TB/s), 148 of 2,304 117 us (5.96), 48
// of 2,304 53 us (4.29), 8 of 1,000 12.4 us, one of 37 9.5 us; 64 of 2,000, 4 kv heads of 256, 82 us (3.18); 128 of 8,000
// through a window of 1,024, 8 kv heads of 64, 38 us (3.53). 15 to 18 us of the mid-sized ones are not the stream: 4 until
// the work is dealt out, 3.5 until the first page is there, the rest joining the pieces of split items and uneven ends.
#include <algorithm>

#include "kv.cuh"

namespace mrl {
namespace kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLeastScale = 1e-37f;       // V scales are taken relative to this at least
// Pieces of O are summed up before they are divided by l, which may be as large as the number of keys: they are held 2^-20
// times their size, so that sums of a million values of bf16's largest stay finite.
constexpr float kDown = 1.0f / 1048576.0f, kUp = 1048576.0f;
constexpr float kNoGrowth = 1.000001f;      // a scale times the rounded reciprocal of itself
constexpr long long kWaitClocks = 4000000000ll;  // a wait for a page gives up after about two seconds

// Warps per CTA: each holds one page's K and V block, 96 to 128 KiB in all, enough in flight per SM to cover
// the latency of HBM, and few enough that a warp's tiles stay in registers.
template <int D> constexpr int kWarps = D == 64 ? 12 : 1024 / D;
template <int D> constexpr int kWidest = D == 64 ? 4 : kWarps<D>;  // warps of the widest team
template <int D> constexpr int kAccStride = D + 8;  // f32 per row of a joined tile: rows 8 banks apart

struct SeqInfo {
    unsigned start;  // first unit (or job) of the sequence
    int len, row, m; // tokens, first row of the call, rows
};

struct Params {
    mrl_kv_cache c;
    mrl_attn a;
    float* part;         // [slots][16][D] partial outputs, then [slots][16][2] their m (base 2) and l
    unsigned* counters;  // arrivals per split item, zero between launches
    int slots;
    int row0;            // rows of earlier launches of the call (one row per sequence)
};

// Pages of a sequence that any of its rows sees: [0, head) and [lo, hi).
struct PageSpan {
    int head, lo, n;
};
__device__ __forceinline__ PageSpan page_span(int len, int m, int window, int sinks) {
    PageSpan s{0, 0, 0};
    if (len <= 0 || m <= 0) return s;
    if (window > 0) {
        const int lo = max(0, len - m - window + 1);
        s.lo = min(lo / kPage, pages_of(len));
        s.head = min(pages_of(min(sinks, lo)), s.lo);
    }
    s.n = s.head + pages_of(len) - s.lo;
    return s;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void load_block(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    long long start = 0;
    for (uint32_t i = 1;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if (i % 16 == 0) {
            if (start == 0) start = clock64();
            else if (clock64() - start > kWaitClocks) return false;
        }
    }
}
// After a wait has run out: the warp does not end while its load is in flight, or before this limit.
__device__ __noinline__ void settle(uint32_t bar, uint32_t parity) { bar_wait(bar, parity); }
// A team is `threads` threads of consecutive warps; one warp needs no barrier resource.
__device__ __forceinline__ void team_sync(int team, int threads) {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four int8 codes as f16 pairs (0, 1) and (2, 3): the byte with its sign bit flipped (code + 128) becomes
// the low bits of 1024 + code + 128, and 1152 is taken off again; all steps are exact.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 a = __hsub2(*reinterpret_cast<__half2*>(&x), off), b = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    lo = *reinterpret_cast<uint32_t*>(&a);
    hi = *reinterpret_cast<uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
    return fmaxf(x, __shfl_xor_sync(~0u, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(~0u, x, 1);
    return x + __shfl_xor_sync(~0u, x, 2);
}

// How the launch's pages are dealt out to its teams: runs of consecutive warps of a CTA.
struct Plan {
    unsigned units;  // pages of all items
    int teams;       // of the launch
    bool few;        // short launch: jobs instead of equal shares of the units
};

// A run of pages [p0, p1) of one item, by one team.
struct Segment {
    int b, head, tile;     // sequence of the call, kv head, 16-row tile
    int p0, p1;
    int parts, part, first;  // pieces the item is in, this one's number, and the first one's team (or job)
};

// WIDE: teams of kWidest warps, for few items; else every warp is a team.
template <class T, int D, bool WIDE> __global__ void __launch_bounds__(kWarps<D> * 32, 1) decode_kernel(Params pr) {
    constexpr int W = WIDE ? kWidest<D> : 1, NW = kWarps<D>, kThreads = NW * 32, kBlock = kPage * D;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* ring = smem;                                              // per warp: K block, V block
    float* acc_s = reinterpret_cast<float*>(ring + (size_t)NW * 2 * kBlock);  // per warp 16 rows of kAccStride
    float* ml_s = acc_s + NW * 16 * kAccStride<D>;                           // per warp 16 x {m, l}
    uint64_t* bars = reinterpret_cast<uint64_t*>(ml_s + NW * 32);            // per warp {K, V}
    SeqInfo* info = reinterpret_cast<SeqInfo*>(bars + NW * 2);               // [n]
    int* seq_s = reinterpret_cast<int*>(info + pr.a.n_seqs);                 // [n] table row, or -1
    __shared__ unsigned scan_s[NW];
    __shared__ unsigned arrived_s[NW];

    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const mrl_kv_cache& c = pr.c;
    const mrl_attn& a = pr.a;
    const int n = (int)a.n_seqs, group = (int)(a.q_heads / c.kv_heads);
    const int window = (int)a.window, sinks = (int)a.sinks;
    const uint32_t bar_k = smem_addr(&bars[warp * 2]), bar_v = bar_k + 8;
    if (lane == 0) {
        bar_init(bar_k);
        bar_init(bar_v);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

    // ---- the call's sequences: their items and pages, summed up
    const Rows rows{a.seqs, a.cu, n, (int)a.n_tokens};
    unsigned my_units = 0;
    bool falls = false;
    for (int b = tid; b < n; b += kThreads) {
        falls = falls || rows.falls(b);
        SeqInfo s;
        s.row = a.cu ? rows.begin(b) : pr.row0 + b;
        s.m = a.cu ? rows.end(b) - s.row : 1;
        const int seq = a.seqs[b];
        const bool known = seq >= 0 && seq < (int)c.max_seqs;
        s.len = known ? min(max(c.lens[seq], 0), (int)c.max_pages * kPage) : 0;
        seq_s[b] = known ? seq : -1;
        if (blockIdx.x == 0 && s.m > 0 && (!known || s.m > s.len)) atomicOr(c.status, MRL_KV_BAD_INDEX);
        s.start = 0;
        info[b] = s;
        if (WIDE && s.m > 0)
            my_units += (unsigned)((s.m * group + 15) / 16) * c.kv_heads * (unsigned)max(1, page_span(s.len, s.m, window, sinks).n);
    }
    Plan pl;
    pl.units = 0;
    if constexpr (WIDE) {
#pragma unroll
        for (int d = 16; d; d >>= 1) my_units += __shfl_xor_sync(~0u, my_units, d);
        if (lane == 0) scan_s[warp] = my_units;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) pl.units += scan_s[w];
    }
    pl.teams = (int)gridDim.x * (NW / W);
    // Few items with no more than a page per warp are dealt out in whole jobs, so that short ones are not split at a
    // team's border; beyond that every team takes an equal share. Measured, 8 sequences of 1,000 tokens and 8 kv heads
    // of 128: 12.0 us with jobs, 15.1 us with shares.
    pl.few = WIDE && pl.units <= (unsigned)(pl.teams * W);
    const bool none = __syncthreads_or(falls);  // and scan_s is read
    if (none && blockIdx.x == 0 && tid == 0) atomicOr(c.status, MRL_KV_BAD_INDEX);
    // An item costs its pages and a fixed part (Q, joining, writing: about 1.5 pages' time of a warp), so equal
    // shares are of pages + `fixed` per item. A share that would begin in an item's fixed part begins with the item.
    const unsigned fixed = pl.few ? 0 : (unsigned)(3 * W + 1) / 2;
    // Exclusive sums over the sequences of their items' cost, or of their jobs.
    unsigned carry = 0;
    for (int at = 0; at < n; at += kThreads) {
        const int b = at + tid;
        unsigned v = 0;
        if (b < n && info[b].m > 0 && !none) {
            const int np = max(1, page_span(info[b].len, info[b].m, window, sinks).n);
            v = (unsigned)((info[b].m * group + 15) / 16) * c.kv_heads * (pl.few ? (unsigned)((np + W - 1) / W) : np + fixed);
        }
        unsigned x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) scan_s[warp] = x;
        __syncthreads();
        unsigned before = carry;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += scan_s[w];
            carry += scan_s[w];
        }
        if (b < n) info[b].start = before + x - v;
        __syncthreads();
    }
    const unsigned total = carry;  // cost of the launch, or its jobs
    if (total == 0) return;
    if (!pl.few) pl.teams = (int)min((unsigned)pl.teams, total);  // no share is empty: an item's pieces are those of consecutive teams

    // ---- this team's share
    const int team = warp / W, w_in = warp % W;
    constexpr int threads = W * 32;
    const int t_in = w_in * 32 + lane;
    const unsigned t_all = blockIdx.x + (unsigned)team * gridDim.x;  // neighbours in work on different SMs
    // Sequence of position x: the last one that starts at or before it, which passes over those without work.
    auto seq_at = [&](unsigned x) {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (info[mid].start <= x) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    // A place in the work: page p of item `item` (heads of tiles) of sequence b, or a job. A walk goes from the
    // share's begin to its end.
    struct Place {
        int b, item, p;
    };
    auto place_at = [&](unsigned x) {
        Place q;
        if (x >= total) return Place{n, 0, 0};
        q.b = seq_at(x);
        const unsigned local = x - info[q.b].start, cost = max(1, page_span(info[q.b].len, info[q.b].m, window, sinks).n) + fixed;
        q.item = (int)(local / cost);
        const unsigned o = local % cost;
        q.p = o > fixed ? (int)(o - fixed) : 0;
        return q;
    };
    struct Walk {
        Place at;          // the next segment
        unsigned job;      // few: the next job
        int np, tiles, items;  // of the sequence at.b
    };
    // begin and end of the share, by the even and the odd lanes at once
    Place edge{0, 0, 0}, stop{n, 0, 0};
    if (!pl.few) {
        const Place q = place_at((unsigned)((unsigned long long)total * (t_all + (lane & 1)) / (unsigned)pl.teams));
        edge = Place{__shfl_sync(~0u, q.b, 0), __shfl_sync(~0u, q.item, 0), __shfl_sync(~0u, q.p, 0)};
        stop = Place{__shfl_sync(~0u, q.b, 1), __shfl_sync(~0u, q.item, 1), __shfl_sync(~0u, q.p, 1)};
    }
    auto enter = [&](Walk& w) {  // sequence w.at.b, or the next one that has work
        while (w.at.b < n && info[w.at.b].m <= 0) ++w.at.b;
        if (w.at.b >= n) return;
        const SeqInfo& q = info[w.at.b];
        w.np = max(1, page_span(q.len, q.m, window, sinks).n);
        w.tiles = (q.m * group + 15) / 16;
        w.items = w.tiles * (int)c.kv_heads;
    };
    Walk walk;
    walk.job = t_all;
    walk.at = edge;
    enter(walk);
    // The next segment of a walk; false at its end.
    auto next_segment = [&](Walk& w, Segment& s) {
        if (pl.few) {
            if (w.job >= total) return false;
            w.at.b = seq_at(w.job);
            enter(w);
            const int k = (w.np + W - 1) / W;
            const unsigned local = w.job - info[w.at.b].start;
            const int item = (int)(local / (unsigned)k), piece = (int)(local % (unsigned)k);
            s.b = w.at.b;
            s.head = item / w.tiles;
            s.tile = item % w.tiles;
            s.p0 = (int)((unsigned)(piece * w.np) / (unsigned)k);
            s.p1 = (int)((unsigned)((piece + 1) * w.np) / (unsigned)k);
            s.parts = k;
            s.part = piece;
            s.first = (int)w.job - piece;
            w.job += (unsigned)pl.teams;
            return true;
        }
        if (w.at.b >= n || (w.at.b == stop.b && w.at.item == stop.item && w.at.p >= stop.p)) return false;
        if (w.at.b > stop.b || (w.at.b == stop.b && w.at.item > stop.item)) return false;
        s.b = w.at.b;
        s.head = w.tiles == 1 ? w.at.item : w.at.item / w.tiles;
        s.tile = w.tiles == 1 ? 0 : w.at.item % w.tiles;
        s.p0 = w.at.p;
        s.p1 = w.at.b == stop.b && w.at.item == stop.item ? stop.p : w.np;
        s.parts = 1;
        s.part = 0;
        s.first = 0;
        if (s.p0 > 0 || s.p1 < w.np) {
            const unsigned long long begin = info[w.at.b].start + (unsigned long long)w.at.item * (w.np + fixed), teams = (unsigned)pl.teams;
            const unsigned t0 = (unsigned)(((begin + fixed + 1) * teams - 1) / total), t1 = (unsigned)(((begin + fixed + w.np) * teams - 1) / total);
            s.parts = (int)(t1 - t0) + 1;
            s.part = (int)(t_all - t0);
            s.first = (int)t0;
        }
        w.at.p = 0;
        if (++w.at.item == w.items) {
            w.at.item = 0;
            ++w.at.b;
            enter(w);
        }
        return true;
    };
    auto slot_of = [&](const Segment& s, int part) { return pl.few ? s.first + part : (s.first + part) * 2 + (part == 0 ? 1 : 0); };

    // ---- pages ahead of the current one: the one after it is known, its K and V loaded as their slots come free; the
    // table is read for the one after that
    Segment as{};         // segment of the page looked up
    Walk awalk = walk;
    int ai = 0;           // its number in the segment's item
    bool more = true;
    int raw_page = -1, raw_index = 0, raw_head = 0;  // looked up: entry as read, page of the sequence, kv head
    int npage = -1, nindex = 0, nhead = 0;           // known
    float nks = 0.0f, nvs = 0.0f;
    uint32_t parity = 0;
    bool fine = true;  // no wait has run out
    bool fresh = true;
    auto look_up = [&]() {
        raw_page = -1;
        if (!more) return;
        if (!fresh) ai += W;
        while (fresh || ai >= as.p1) {
            fresh = false;
            if (!next_segment(awalk, as)) {
                more = false;
                return;
            }
            ai = as.p0 + w_in;
        }
        const SeqInfo& q = info[as.b];
        const PageSpan sp = page_span(q.len, q.m, window, sinks);
        raw_index = ai < sp.head ? ai : sp.lo + ai - sp.head;
        raw_head = as.head;
        if (ai < sp.n) raw_page = __ldg(c.tables + (size_t)seq_s[as.b] * c.max_pages + raw_index);
    };
    auto advance = [&]() {
        npage = raw_page >= 0 && raw_page < (int)c.pages ? raw_page : -1;
        nindex = raw_index;
        nhead = raw_head;
        look_up();
    };
    auto fetch = [&](int which) {
        if (npage < 0 || !fine) return;
        const size_t block = block_index(c, a.layer, npage, which, nhead);
        if (which == 0) {
            nks = c.scales[block];
            nvs = c.scales[block + c.kv_heads];
        }
        if (lane == 0)
            load_block(smem_addr(ring + (size_t)(warp * 2 + which) * kBlock), c.codes + block * (size_t)kBlock, kBlock, which ? bar_v : bar_k);
    };
    look_up();
    advance();
    fetch(0);
    fetch(1);

    const int g = lane >> 2, t = lane & 3;
    const unsigned char* kb = ring + (size_t)(warp * 2) * kBlock;
    const unsigned char* vb = kb + kBlock;
    Segment s{};
    while (next_segment(walk, s)) {
        const SeqInfo q = info[s.b];
        // Rows of this lane: r, token of the sequence r / group, query head r % group.
        const int r0 = s.tile * 16 + g, r1 = r0 + 8, rows_all = q.m * group;
        const int first = q.len - q.m;
        const Span v0 = visible(first + r0 / group, q.len, 1, window, sinks), v1 = visible(first + r1 / group, q.len, 1, window, sinks);
        const int low_pos = first + s.tile * 16 / group, high_pos = first + min(rows_all - 1, s.tile * 16 + 15) / group;
        // head_dim 256 keeps Q where the joined tile goes at the end of the segment: registers hold O
        constexpr bool kQApart = D == 256;
        uint32_t qf[kQApart ? 1 : D / 16][4];
        uint4* const q_s = reinterpret_cast<uint4*>(acc_s + warp * 16 * kAccStride<D>) + lane;
        float c0 = a.scale * kLog2e, c1 = c0;
        {
            const T* base = static_cast<const T*>(a.q);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = h ? r1 : r0;
                const bool in = r < rows_all;
                const T* p = base + (int64_t)(q.row + r / group) * a.q_row + (int64_t)(s.head * group + r % group) * a.q_head + 16 * t;
                uint4 raw[D / 32];
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                    raw[i] = in ? *reinterpret_cast<const uint4*>(p + (i >> 1) * 64 + (i & 1) * 8) : make_uint4(0, 0, 0, 0);
                const T* e = reinterpret_cast<const T*>(raw);
                float down = 1.0f;
                if (sizeof(T) == 2 && !__is_same(T, __half)) {
                    // bf16 has more range than f16: the row is brought to [1, 2) by a power of two, which is put
                    // back with the softmax scale. What leaves f16's range below is 2^-24 of the row's largest.
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(to_f32<T>(e[i])));
                    top = quad_max(top);
                    const uint32_t ex = __float_as_uint(top) >> 23;  // biased exponent
                    if (ex > 0 && ex < 255) {
                        const uint32_t up = min(ex, 253u);
                        down = __uint_as_float((254u - up) << 23);
                        (h ? c1 : c0) *= __uint_as_float(up << 23);
                    }
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {  // k-step i: block i / 4, word i % 4 of the lane's 16 dims
                    const T* x = e + (i >> 2) * 16 + (i & 3) * 4;
                    const uint32_t y0 = pack_half(to_f32<T>(x[0]) * down, to_f32<T>(x[1]) * down), y1 = pack_half(to_f32<T>(x[2]) * down, to_f32<T>(x[3]) * down);
                    if (kQApart) {
                        reinterpret_cast<uint32_t*>(q_s + i * 32)[h] = y0;
                        reinterpret_cast<uint32_t*>(q_s + i * 32)[2 + h] = y1;
                    } else {
                        qf[i][h] = y0;
                        qf[i][2 + h] = y1;
                    }
                }
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        // P carries V's scale relative to the largest one of the pages that the row has seen so far, and O is in units of
        // that; its reciprocal is kept. Pages that a row sees nothing of do not count: their scale may be any number of
        // times larger, and would push the P of the others out of f16.
        float per0 = 1.0f / kLeastScale, per1 = per0;

        for (int i = s.p0 + w_in; i < s.p1; i += W) {
            const int page = npage, index = nindex;
            const float ks = nks, vs = nvs;
            advance();
            if (page < 0) {  // nothing of it was loaded
                fetch(0);
                fetch(1);
                continue;
            }
            if (fine && !bar_wait(bar_k, parity)) {
                fine = false;
                settle(bar_k, parity);
                settle(bar_v, parity);
            }
            float sc[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
            if (fine) {
#pragma unroll
                for (int db = 0; db < D / 64; ++db) {
                    uint32_t qd[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (kQApart) {
                            *reinterpret_cast<uint4*>(qd[i]) = q_s[(db * 4 + i) * 32];
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) qd[i][e] = qf[db * 4 + i][e];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint4 w = *reinterpret_cast<const uint4*>(kb + db * 4096 + (16 * (g >> 1) + 2 * j + (g & 1)) * 64 + 16 * t);
                        uint32_t b0, b1;
                        widen4(w.x, b0, b1);
                        mma16816(sc[j], qd[0], b0, b1);
                        widen4(w.y, b0, b1);
                        mma16816(sc[j], qd[1], b0, b1);
                        widen4(w.z, b0, b1);
                        mma16816(sc[j], qd[2], b0, b1);
                        widen4(w.w, b0, b1);
                        mma16816(sc[j], qd[3], b0, b1);
                    }
                }
            }
            __syncwarp();
            fetch(0);
            const float f0 = c0 * ks, f1 = c1 * ks;
            const int key0 = index * kPage;
            float n0 = -INFINITY, n1 = -INFINITY;
            // Token 16 t + 2 j + e of the page is column e of score tile j here.
            if (key0 + kPage - 1 <= low_pos && (window == 0 || key0 > high_pos - window || key0 + kPage <= sinks)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sc[j][0] *= f0;
                    sc[j][1] *= f0;
                    sc[j][2] *= f1;
                    sc[j][3] *= f1;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = key0 + 16 * t + 2 * j + e;
                        sc[j][e] = key < v0.head || (key >= v0.lo && key < v0.hi) ? sc[j][e] * f0 : -INFINITY;
                        sc[j][2 + e] = key < v1.head || (key >= v1.lo && key < v1.hi) ? sc[j][2 + e] * f1 : -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                n0 = fmaxf(n0, fmaxf(sc[j][0], sc[j][1]));
                n1 = fmaxf(n1, fmaxf(sc[j][2], sc[j][3]));
            }
            n0 = quad_max(n0);
            n1 = quad_max(n1);
            const float s0 = n0 > -INFINITY ? vs : 0.0f, s1 = n1 > -INFINITY ? vs : 0.0f;
            const bool grow0 = s0 * per0 > kNoGrowth, grow1 = s1 * per1 > kNoGrowth;
            n0 = fmaxf(n0, m0);
            n1 = fmaxf(n1, m1);
            if (__any_sync(~0u, n0 != m0 || n1 != m1 || grow0 || grow1)) {
                const float k0 = m0 == -INFINITY ? 0.0f : ex2(m0 - n0), k1 = m1 == -INFINITY ? 0.0f : ex2(m1 - n1);
                l0 *= k0;
                l1 *= k1;
                float a0 = k0, a1 = k1;
                if (grow0) {
                    const float to = __fdividef(1.0f, s0);
                    a0 *= __fdividef(to, per0);
                    per0 = to;
                }
                if (grow1) {
                    const float to = __fdividef(1.0f, s1);
                    a1 *= __fdividef(to, per1);
                    per1 = to;
                }
#pragma unroll
                for (int x = 0; x < D / 8; ++x) {
                    o[x][0] *= a0;
                    o[x][1] *= a0;
                    o[x][2] *= a1;
                    o[x][3] *= a1;
                }
                m0 = n0;
                m1 = n1;
            }
            const float z0 = m0 == -INFINITY ? 0.0f : m0, z1 = m1 == -INFINITY ? 0.0f : m1;
            const float vf0 = s0 * per0, vf1 = s1 * per1;
            uint32_t pf[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float* w = sc[2 * x + y];
                    w[0] = ex2(w[0] - z0);
                    w[1] = ex2(w[1] - z0);
                    w[2] = ex2(w[2] - z1);
                    w[3] = ex2(w[3] - z1);
                    l0 += w[0] + w[1];
                    l1 += w[2] + w[3];
                    pf[x][2 * y] = pack_half(w[0] * vf0, w[1] * vf0);
                    pf[x][2 * y + 1] = pack_half(w[2] * vf1, w[3] * vf1);
                }
            }
            if (fine && !bar_wait(bar_v, parity)) {
                fine = false;
                settle(bar_v, parity);
                if (npage >= 0) settle(bar_k, parity ^ 1);
            }
            parity ^= 1;
            if (fine) {
#pragma unroll
                for (int x = 0; x < D / 8; ++x) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vb + (8 * x + g) * 64 + 16 * t);
                    uint32_t b0, b1;
                    widen4(w.x, b0, b1);
                    mma16816(o[x], pf[0], b0, b1);
                    widen4(w.y, b0, b1);
                    mma16816(o[x], pf[1], b0, b1);
                    widen4(w.z, b0, b1);
                    mma16816(o[x], pf[2], b0, b1);
                    widen4(w.w, b0, b1);
                    mma16816(o[x], pf[3], b0, b1);
                }
            }
            __syncwarp();
            fetch(1);
        }
        l0 = quad_sum(l0);
        l1 = quad_sum(l1);

        // ---- the team's warps joined: O in one unit, then rescaled to the rows' common maximum
        const float vref0 = kDown / per0, vref1 = kDown / per1;
        float* mine = acc_s + warp * 16 * kAccStride<D>;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
            if (r0 < rows_all)
                *reinterpret_cast<float2*>(mine + g * kAccStride<D> + 8 * x + 2 * t) = make_float2(o[x][0] * vref0, o[x][1] * vref0);
            if (r1 < rows_all)
                *reinterpret_cast<float2*>(mine + (g + 8) * kAccStride<D> + 8 * x + 2 * t) = make_float2(o[x][2] * vref1, o[x][3] * vref1);
        }
        if (t == 0) {
            *reinterpret_cast<float2*>(ml_s + (warp * 16 + g) * 2) = make_float2(m0, l0);
            *reinterpret_cast<float2*>(ml_s + (warp * 16 + g + 8) * 2) = make_float2(m1, l1);
        }
        team_sync(team, threads);
        const int tile_rows = min(16, rows_all - s.tile * 16);
        const int w0 = team * W;
        auto emit = [&](int r, int d, float4 x, float m, float l) {
            const int row = s.tile * 16 + r;
            const float inv = l == 0.0f ? 0.0f : kUp / l;
            T* dst = static_cast<T*>(a.out) + (int64_t)(q.row + row / group) * a.o_row + (int64_t)(s.head * group + row % group) * a.o_head + d;
            T y[4] = {from_f32<T>(x.x * inv), from_f32<T>(x.y * inv), from_f32<T>(x.z * inv), from_f32<T>(x.w * inv)};
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
            if (a.lse && d == 0)
                a.lse[(size_t)(q.row + row / group) * a.q_heads + s.head * group + row % group] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        };
        float* const ml_g = pr.part + (size_t)pr.slots * 16 * D;
        for (int i = t_in; i < tile_rows * (D / 4); i += threads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float m = -INFINITY;
            for (int w = 0; w < W; ++w) m = fmaxf(m, ml_s[((w0 + w) * 16 + r) * 2]);
            const float z = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4 x = make_float4(0, 0, 0, 0);
            for (int w = 0; w < W; ++w) {
                const float k = ex2(ml_s[((w0 + w) * 16 + r) * 2] - z);
                const float4 y = *reinterpret_cast<const float4*>(acc_s + ((w0 + w) * 16 + r) * kAccStride<D> + d);
                l = fmaf(k, ml_s[((w0 + w) * 16 + r) * 2 + 1], l);
                x.x = fmaf(k, y.x, x.x);
                x.y = fmaf(k, y.y, x.y);
                x.z = fmaf(k, y.z, x.z);
                x.w = fmaf(k, y.w, x.w);
            }
            if (s.parts == 1) {
                emit(r, d, x, m, l);
            } else {
                const size_t slot = (size_t)slot_of(s, s.part);
                __stcg(reinterpret_cast<float4*>(pr.part + (slot * 16 + r) * D + d), x);
                if (d == 0) __stcg(reinterpret_cast<float2*>(ml_g + (slot * 16 + r) * 2), make_float2(m, l));
            }
        }
        if (s.parts > 1) {
            team_sync(team, threads);  // the team's stores come before its arrival, and the others' before the last one's reads
            if (t_in == 0) {
                __threadfence();
                const unsigned before = atomicAdd(&pr.counters[s.first], 1u);
                if (before + 1 == (unsigned)s.parts) pr.counters[s.first] = 0;
                __threadfence();
                arrived_s[warp] = before + 1;
            }
            team_sync(team, threads);
            if (arrived_s[w0] == (unsigned)s.parts) {
                for (int i = t_in; i < tile_rows * (D / 4); i += threads) {
                    const int r = i / (D / 4), d = i % (D / 4) * 4;
                    float m = -INFINITY, l = 0.0f;
                    float4 x = make_float4(0, 0, 0, 0);
                    for (int k0 = 0; k0 < s.parts; k0 += 4) {  // four pieces' loads at once
                        float2 ml[4];
                        float4 y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            ml[k] = make_float2(-INFINITY, 0.0f);
                            y[k] = make_float4(0, 0, 0, 0);
                            if (k0 + k < s.parts) {
                                const size_t slot = (size_t)slot_of(s, k0 + k);
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(ml_g + (slot * 16 + r) * 2));
                                y[k] = __ldcg(reinterpret_cast<const float4*>(pr.part + (slot * 16 + r) * D + d));
                            }
                        }
                        const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x)), z = top == -INFINITY ? 0.0f : top;
                        const float keep = ex2(m - z);
                        l *= keep;
                        x = make_float4(x.x * keep, x.y * keep, x.z * keep, x.w * keep);
                        m = top;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float e = ex2(ml[k].x - z);
                            l = fmaf(e, ml[k].y, l);
                            x.x = fmaf(e, y[k].x, x.x);
                            x.y = fmaf(e, y[k].y, x.y);
                            x.z = fmaf(e, y[k].z, x.z);
                            x.w = fmaf(e, y[k].w, x.w);
                        }
                    }
                    emit(r, d, x, m, l);
                }
            }
        }
        team_sync(team, threads);  // the joined tiles are free again
    }
    if (!fine && lane == 0) atomicOr(c.status, MRL_KV_TIMEOUT);
}

template <class T, int D> cudaError_t launch(const Params& p, int sms, cudaStream_t s) {
    constexpr int NW = kWarps<D>;
    const size_t smem = (size_t)NW * 2 * kPage * D + sizeof(float) * NW * 16 * kAccStride<D> + sizeof(float) * NW * 32 + 16 * NW +
                        (sizeof(SeqInfo) + sizeof(int)) * p.a.n_seqs;
    // Teams of a whole CTA (4 warps, head_dim 64) where there is no more than an item per SM: an item is then in few
    // pieces, joined in shared memory; single warps beyond, which need no joining. Measured us, teams / warps: 8 kv heads
    // of 128, 8 sequences of 1,000 12.0 / 19.7, one of 130,000 55 / 124, 4 of 130,000 174 / 192, 48 of 2,300 59 / 52.5, 256 of
    // 512 90 / 63; 64 of 2,000 with 4 kv heads of 256 86 / 81.
    const uint64_t group = p.a.q_heads / p.c.kv_heads;
    const uint64_t tiles = p.a.cu ? std::max<uint64_t>(p.a.n_seqs, p.a.n_tokens * group / 16) : p.a.n_seqs * ((group + 15) / 16);
    if (tiles * p.c.kv_heads <= (uint64_t)sms) {
        if (const cudaError_t e = allow_smem<decode_kernel<T, D, true>>(232448 - 2048)) return e;
        decode_kernel<T, D, true><<<sms, NW * 32, smem, s>>>(p);
    } else {
        if (const cudaError_t e = allow_smem<decode_kernel<T, D, false>>(232448 - 2048)) return e;
        decode_kernel<T, D, false><<<sms, NW * 32, smem, s>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace kv

// Pieces: one per job or two per team, jobs at most pages / width + items <= 2 warps of the launch.
static int decode_slots(uint32_t head_dim, int sms) { return 2 * sms * (int)(1024 / head_dim) + 2; }  // at most 1024 / head_dim warps an SM
size_t kv_decode_bytes(uint32_t head_dim, int sms) { return (size_t)decode_slots(head_dim, sms) * 16 * (head_dim + 2) * sizeof(float); }

int launch_kv_decode(const mrl_kv_cache& c, const mrl_attn& a, int sms, void* scratch, unsigned* counters, cudaStream_t s) {
    kv::Params p;
    p.c = c;
    p.a = a;
    p.part = static_cast<float*>(scratch);
    p.counters = counters;
    p.slots = decode_slots(c.head_dim, sms);
    p.row0 = 0;
    const bool half = a.dtype == MRL_F16;
    for (uint32_t at = 0; at < a.n_seqs; at += kKvDecodeSeqs) {
        p.a.n_seqs = a.n_seqs - at < kKvDecodeSeqs ? a.n_seqs - at : kKvDecodeSeqs;  // at most so many have their table in shared memory
        p.a.seqs = a.seqs + at;
        p.a.cu = a.cu ? a.cu + at : nullptr;
        p.row0 = (int)at;
        cudaError_t e;
        if (c.head_dim == 64) e = half ? kv::launch<__half, 64>(p, sms, s) : kv::launch<__nv_bfloat16, 64>(p, sms, s);
        else if (c.head_dim == 128) e = half ? kv::launch<__half, 128>(p, sms, s) : kv::launch<__nv_bfloat16, 128>(p, sms, s);
        else e = half ? kv::launch<__half, 256>(p, sms, s) : kv::launch<__nv_bfloat16, 256>(p, sms, s);
        if (e != cudaSuccess) return (int)e;
    }
    return 0;
}

}  // namespace mrl
