// attend_tc.cu — attention on the 5th-generation tensor cores (tcgen05, sm_100a): mrl_window_attention over
// ragged 16-bit rows, and mrl_kv_attend over the paged 8-bit cache where sequences have many query rows.
//
// A tile is 128 query rows of one sequence and kv head: 128 / group tokens x the group's query heads, so
// all query heads of a kv head share its K and V. Per 128 keys a tile does S = Q K^T (both from shared
// memory, S in tensor memory), softmax on 128 threads, one row each, that put P back into tensor memory
// over S as 16-bit pairs, and O += P V with P from there. head_dim 64 and 128 run two tiles per CTA that
// share each K and V: while one tile's S is exponentiated the tensor core works for the other. head_dim 256
// has tensor memory for one O only, and runs one tile with two S buffers instead.
//
// The running maximum a row subtracts moves only when a new one exceeds it by 2^8 (base-2 logits): O and
// the sum l are kept relative to the stale one, which cancels in o = O / l, and O is rescaled rarely. P is
// at most 2^8, over the cache, where it carries V's scale in a unit that lags by up to 2^6, at most 2^14: inside f16,
// and its rounding is relative either way.
//
// Roles: warps 0-3 and 4-7 softmax and epilogue of the tiles, warp 8 issues the products, warp 9 loads Q, K
// and V by TMA (16-bit rows), where warp 10 clears V past a sequence's end; over the cache warp 9 copies blocks of codes that
// a first launch has widened to f16 (exact) in the operand layout, once for all the tiles that read them, and
// warps 10 and 11 bring in Q as f16; the blocks' scales go to S and P, which are f32 there. Every wait is bounded; when one runs out
// the kernel records it, waits for what it has in flight and ends.
//
// Bounds: per 128 keys a tile pair needs 2 x 2 x 128 x 128 x D products (2,048 clocks at head_dim 128) and 2 x 16,384
// exponentials and as many conversions (about 2,560). What a pair takes is the chain of one tile's step, about 3,500
// clocks, the other tile in the gaps: S into registers 200, maximum 250, P 1,270, hand-over 100, P V and the next S
// 1,100, waits. Measured on one B200, full attention over 2 x 8,192 tokens of unit normal values: 16 heads of 128 in bf16 937
// us, 1,173 TFLOP/s (tensor pipe 54% active); 16 heads of 64 in f16 822 us; 8 heads of 256 in bf16 1,200 us;
// causal with a window of 1,024 and 4 sinks, 16 query heads on 4, 202 us. The rows of two tiles rather than one per CTA halve
// the traffic of K and V from L2 (64 KB per step); 128 keys a step is what tensor memory holds beside two O.
// The instructions' operands have to be in uniform registers: issued from one divergent lane, each product cost
// 75 clocks and the same kernel ran at 972 instead of 1,097 TFLOP/s.
#include <cuda.h>

#include <algorithm>

#include "kv.cuh"
#include "umma.cuh"

namespace mrl {
namespace kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr long long kWaitClocks = 4000000000ll;  // about two seconds
constexpr int kKeys = 128;        // keys per step
constexpr float kSlack = 8.0f;    // log2 by which a row's maximum may lead the one it subtracts
constexpr float kScaleSlack = 64.0f;  // the same for V's scales over the cache (a factor)
constexpr int kInfo = 8;          // steps of scales kept
constexpr uint32_t kOwnNaN = 0xffffffffu;  // two NaNs that mark a row whose scores are not finite; conversions give 0x7fff

template <int D> constexpr int kWide = kPage * D * 2;  // bytes of a page and head's K or V as f16
// What a template instance is: D, two tiles or one, stages of K and V, and its threads.
template <int D, bool PAGED> struct Shape {
    static constexpr int tiles = D == 256 ? 1 : 2;
    static constexpr int sbufs = D == 256 ? 2 : 1;
    static constexpr int stages = D == 64 ? 3 : D == 128 ? 2 : 1;
    static constexpr int q_bytes = 128 * D * 2, kv_bytes = kKeys * D * 2;
    // A stage of K or V is handed over in pieces where there is only one: K by 64 dims, V by 64 keys.
    static constexpr int k_parts = D == 256 ? 4 : 1, v_parts = D == 256 ? 2 : 1;
    static constexpr int seqs = 512;  // sequences per launch (their table is in shared memory)
    static constexpr int threads = 12 * 32;
    // Registers: launched with 168 a thread, of which the two softmax warpgroups take more and the other gives up
    // as many: 8 x 208 + 4 x 88 = 12 x 168. At 216 and 72 the warps that convert Q spill: 229 instead of 217 us for 4 x 500
    // rows on 5,000 tokens, 32 heads of 128 on 8.
    static constexpr int regs_softmax = 208, regs_other = 88;
    static constexpr int tmem_s = 0;                           // S (and P) columns of tile or buffer i at 128 i
    static constexpr int tmem_o = 256;                         // O columns of tile i at 256 + D i
    static constexpr size_t smem = 1024 + (size_t)tiles * q_bytes + 2 * stages * kv_bytes;
};

struct SeqItem {
    int len, row, m;  // tokens, first row of the call, rows
};

struct TcParams {
    mrl_kv_cache c;
    mrl_attn a;
    int heads, group, tokens;  // kv heads, query heads per kv head, tokens per tile
    int causal;
    int sectors;  // out and its strides are multiples of 32 bytes
    int inner_q, inner_k, inner_v;  // the map's second dimension is the row, not the head
    // over the cache: f16 image of the layer's pool, [pages][2][kv heads][wide], and a block of zeros. The image only
    // ever holds codes, so pages of it that a step touches but no row sees are finite.
    const unsigned char *wide, *zero;
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
    if (tc::mbar_wait(bar, parity, 16)) return true;
    const long long start = clock64();
    while (!tc::mbar_wait(bar, parity, 16)) {
        if (*failed) return false;
        if (clock64() - start > kWaitClocks) {
            *failed = 1;
            return false;
        }
    }
    return true;
}
// For a copy or product that may be in flight when its CTA has no more to do, as after a wait that ran out: the CTA does not
// end before it, or before this limit.
__device__ __noinline__ void settle(uint64_t* bar, uint32_t parity) {
    const long long start = clock64();
    while (!tc::mbar_wait(bar, parity, 16) && clock64() - start <= kWaitClocks) {}
}
// The fills of up to 8 barriers that a loading thread has issued: which, and the parity of the last one's phase.
struct Fills {
    uint32_t any = 0, parity = 0;
    __device__ __forceinline__ void note(int i, uint32_t par) {
        any |= 1u << i;
        parity = (parity & ~(1u << i)) | par << i;
    }
    // barrier i's last fill is known to have landed, and its phases go on
    __device__ __forceinline__ void drop(int i) { any &= ~(1u << i); }
    __device__ __forceinline__ void settle_all(uint64_t* bars, int n) const {
        for (int i = 0; i < n; ++i)
            if (any >> i & 1) settle(&bars[i], parity >> i & 1);
    }
};
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(tc::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(tc::smem_u32(bar))
                 : "memory");
}

// kind::f16 products, f32 accumulators; A and B of the same 16-bit type.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// M 128, N n; bf: bf16 operands, else f16; mn: B is N-major.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool bf, bool mn) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Shared-memory descriptor of a 128-byte-swizzled operand: 8 rows of 128 bytes per 1024-byte atom, atoms 1024
// bytes apart along the rows, and for a B that is N-major, 64-wide column blocks `lbo` apart. The low word
// holds the address, so stepping along an operand is an addition to it.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // atom stride, version, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | (lbo >> 4) << 16; }
__device__ __forceinline__ uint64_t desc(uint32_t low) { return (uint64_t)kDescHigh << 32 | low; }
// The first active lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

#define MRL_TC_LD32(r, taddr)                                                                                                            \
    asm volatile(                                                                                                                        \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "  \
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"                                                       \
        : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]), "=r"((r)[8]),  \
          "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]), "=r"((r)[15]), "=r"((r)[16]),         \
          "=r"((r)[17]), "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]), "=r"((r)[22]), "=r"((r)[23]), "=r"((r)[24]),        \
          "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]), "=r"((r)[29]), "=r"((r)[30]), "=r"((r)[31])                        \
        : "r"(taddr)                                                                                                                     \
        : "memory")

#define MRL_TC_ST32(taddr, r)                                                                                                            \
    asm volatile(                                                                                                                        \
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "     \
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),                                      \
        "r"((r)[0]), "r"((r)[1]), "r"((r)[2]), "r"((r)[3]), "r"((r)[4]), "r"((r)[5]), "r"((r)[6]), "r"((r)[7]), "r"((r)[8]),             \
        "r"((r)[9]), "r"((r)[10]), "r"((r)[11]), "r"((r)[12]), "r"((r)[13]), "r"((r)[14]), "r"((r)[15]), "r"((r)[16]), "r"((r)[17]),     \
        "r"((r)[18]), "r"((r)[19]), "r"((r)[20]), "r"((r)[21]), "r"((r)[22]), "r"((r)[23]), "r"((r)[24]), "r"((r)[25]), "r"((r)[26]),    \
        "r"((r)[27]), "r"((r)[28]), "r"((r)[29]), "r"((r)[30]), "r"((r)[31])                                                             \
        : "memory")
// The values of loads that a wait has covered are used after it, not before.
template <int N> __device__ __forceinline__ void pin(uint32_t (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(x[i]));
}
template <int REGS> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// Two f32 operations at once.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <bool BF> __device__ __forceinline__ uint32_t pack16(float a, float b) {
    uint32_t r;
    if (BF) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        r = *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        r = *reinterpret_cast<const uint32_t*>(&h);
    }
    return r;
}
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {  // exact, as in kv_decode.cu
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 a = __hsub2(*reinterpret_cast<__half2*>(&x), off), b = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    lo = *reinterpret_cast<uint32_t*>(&a);
    hi = *reinterpret_cast<uint32_t*>(&b);
}

// 32 bytes, as one sector where the output's rows are aligned to sectors.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8], int sectors) {
    if (sectors) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                     "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// Key steps of a tile: [0, head) and [lo, hi), of 128 keys each. Empty: hi == 0.
struct Steps {
    int head, lo, hi;
    __device__ __forceinline__ bool has(int s) const { return s < head || (s >= lo && s < hi); }
};
// Of the tokens at positions [p0, p1] of a sequence of n keys.
__device__ __forceinline__ Steps steps_of(int p0, int p1, int n, int causal, int window, int sinks) {
    const Span a = visible(p0, n, causal, window, sinks), b = visible(p1, n, causal, window, sinks);
    Steps s{0, 0, 0};
    if (imax(a.hi, b.hi) <= 0) return s;
    s.hi = (imax(a.hi, b.hi) + kKeys - 1) / kKeys;
    s.lo = imin(a.lo, s.hi * kKeys) / kKeys;
    s.head = imin((imax(a.head, b.head) + kKeys - 1) / kKeys, s.lo);
    return s;
}

// One item: `tiles` tiles of consecutive tokens of one sequence and kv head.
template <int TILES> struct Item {
    int b, head, first;  // first: token (row of the sequence) of the item
    int len, row, m;
    Steps st[TILES];
    Steps all;
    __device__ __forceinline__ int next(int s) const { return s + 1 == all.head ? (all.lo > s + 1 ? all.lo : s + 1) : s + 1; }
    __device__ __forceinline__ int begin() const { return all.head > 0 ? 0 : all.lo; }
};

// The call's items, dealt out to the CTAs; the tables are in shared memory.
template <int TILES> struct Items {
    const SeqItem* info;
    const unsigned* start;   // first item of the i-th sequence in order
    const uint16_t* order;   // that sequence
    int n, tokens;
    unsigned heads, items;
    int causal, window, sinks;

    // Item i; the tiles with the latest tokens come first, they have the most keys where the mask is causal.
    __device__ __forceinline__ Item<TILES> at(unsigned i) const {
        Item<TILES> it;
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= i) lo = mid;
            else hi = mid;
        }
        const unsigned local = i - start[lo];
        lo = order[lo];
        const SeqItem q = info[lo];
        const int count = (q.m + TILES * tokens - 1) / (TILES * tokens);
        it.b = lo;
        it.head = (int)(local % heads);
        it.first = (count - 1 - (int)(local / heads)) * TILES * tokens;
        it.len = q.len;
        it.row = q.row;
        it.m = q.m;
        it.all = Steps{0, 0, 0};
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int f = it.first + t * tokens, base = q.len - q.m;
            it.st[t] = f < q.m ? steps_of(base + f, base + imin(f + tokens, q.m) - 1, q.len, causal, window, sinks) : Steps{0, 0, 0};
            if (it.st[t].hi > 0) {
                const bool none = it.all.hi == 0;
                it.all.hi = imax(it.all.hi, it.st[t].hi);
                it.all.lo = none ? it.st[t].lo : imin(it.all.lo, it.st[t].lo);
                it.all.head = imax(it.all.head, it.st[t].head);
            }
        }
        it.all.head = imin(it.all.head, it.all.lo);
        return it;
    }
    // The CTA's item in round r: there and back over the CTAs, so that a long one is followed by a short one.
    __device__ __forceinline__ unsigned number(unsigned r) const {
        const unsigned grid = gridDim.x;
        return r & 1 ? (r + 1) * grid - 1 - blockIdx.x : r * grid + blockIdx.x;
    }
};

// The softmax warps of a CTA, without the others.
template <int TILES> __device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(128 * TILES) : "memory"); }

// E 16-bit values at p, 4 to 16 bytes aligned to themselves.
template <int E> __device__ __forceinline__ void load16(const void* p, uint32_t (&w)[E / 2]) {
    if (E == 2) w[0] = *static_cast<const uint32_t*>(p);
    else if (E == 4) *reinterpret_cast<uint2*>(w) = *static_cast<const uint2*>(p);
    else *reinterpret_cast<uint4*>(w) = *static_cast<const uint4*>(p);
}
// Of 16-bit values: bit 0, one is a NaN; bit 1, one is an Inf; bit 2, one has every bit set (kOwnNaN).
template <class T, int E> __device__ __forceinline__ int odd_values(const uint32_t (&w)[E / 2]) {
    constexpr uint32_t kExp = __is_same(T, __half) ? 0x7c00u : 0x7f80u;
    int kind = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t x = w[i / 2] >> (16 * (i & 1)) & 0xffffu, mag = x & 0x7fffu;
        kind |= mag > kExp ? 1 : mag == kExp ? 2 : 0;
        if (x == 0xffffu) kind |= 4;
    }
    return kind;
}

// The exact result of one row, from its visible keys alone. A warp, lane e holds dims e D/32 ..; four keys at a time. O is kept
// divided by l, so that it is never larger than the values: also where the products' sums are too large for f32.
template <class T, int D> __device__ __noinline__ void slow_row(const mrl_attn& a, int row0, int n, int p, int t_row, int h, int kvh, int causal) {
    constexpr int E = D / 32, kTurn = 4;
    const int lane = (int)threadIdx.x & 31;
    const Span span = visible(p, n, causal, (int)a.window, (int)a.sinks);
    float q[E], o[E];
    const T* qp = static_cast<const T*>(a.q) + (int64_t)t_row * a.q_row + (int64_t)h * a.q_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = to_f32<T>(qp[e]);
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int part = 0; part < 2; ++part) {
        const int from = part ? span.lo : 0, to = part ? span.hi : span.head;
        for (int j = from; j < to; j += kTurn) {
            uint32_t kw[kTurn][E / 2], vw[kTurn][E / 2];
            float s[kTurn];
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                const int key = imin(j + u, to - 1);
                load16<E>(static_cast<const T*>(a.k) + (int64_t)(row0 + key) * a.k_row + (int64_t)kvh * a.k_head + lane * E, kw[u]);
                load16<E>(static_cast<const T*>(a.v) + (int64_t)(row0 + key) * a.v_row + (int64_t)kvh * a.v_head + lane * E, vw[u]);
            }
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                const T* k = reinterpret_cast<const T*>(kw[u]);
                s[u] = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) s[u] = fmaf(q[e], to_f32<T>(k[e]), s[u]);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1)
#pragma unroll
                for (int u = 0; u < kTurn; ++u) s[u] += __shfl_xor_sync(~0u, s[u], d);
            float top = m;
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                s[u] *= a.scale;
                if (j + u < to) top = s[u] > top || s[u] != s[u] ? s[u] : top;  // a NaN stays
            }
            const float keep = m == -INFINITY ? 0.0f : l * expf(m - top);
            m = top;
            l = keep;
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                s[u] = j + u >= to || (s[u] == -INFINITY && top == -INFINITY) ? 0.0f : expf(s[u] - top);
                l += s[u];
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = keep == 0.0f ? 0.0f : o[e] * (keep * inv);
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                if (j + u >= to) break;
                const T* v = reinterpret_cast<const T*>(vw[u]);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(s[u] * inv, to_f32<T>(v[e]), o[e]);
            }
        }
    }
    T* op = static_cast<T*>(a.out) + (int64_t)t_row * a.o_row + (int64_t)h * a.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) op[e] = from_f32<T>(l == 0.0f ? 0.0f : o[e]);
    if (a.lse && lane == 0) a.lse[(size_t)t_row * a.q_heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

// A tile's rows whose fast result is not finite, all its softmax warps. A value of V that a row does not see (a later
// key, one before its window) reaches its products as 0 x Inf: such a row is computed again from its visible keys. Where every
// odd value of V that the tile met is seen by the row, the fast result is the right one, except that an Inf under a weight that
// rounds to 0 is a NaN there. Written by the same CTA before a barrier; rows marked kOwnNaN are right as they are.
struct OddKeys {
    int lo, hi, inf, rows;  // first and last key with an odd value of V, whether one is an Inf, whether any row is to be looked at
};
template <class T, int D, int TILES> __device__ __forceinline__ void redo_tile(const mrl_attn& a, int row0, int n, int m, int first, int tokens, int group, int kvh, Steps st, int causal, OddKeys* odd) {
    constexpr int E = D / 32, kWarps = 4 * TILES;
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const int rows = imin(tokens, m - first) * group;
    auto kind_of = [&](int r) {  // of the result in row r of the tile
        uint32_t w[E / 2];
        load16<E>(static_cast<const T*>(a.out) + (int64_t)(row0 + first + r / group) * a.o_row + (int64_t)(kvh * group + r % group) * a.o_head + lane * E, w);
        const int kind = odd_values<T, E>(w);
        return __any_sync(~0u, kind & 4) ? 0 : (__any_sync(~0u, kind & 1) ? 1 : 0) | (__any_sync(~0u, kind & 2) ? 2 : 0);
    };
    if (threadIdx.x == 0) *odd = OddKeys{0x7fffffff, -1, 0, 0};
    softmax_sync<TILES>();
    bool any = false;
    for (int r = warp; r < rows; r += kWarps) any = any || kind_of(r) != 0;
    if (any && lane == 0) odd->rows = 1;
    softmax_sync<TILES>();
    const bool look = odd->rows != 0;
    if (look) {
        for (int s = 0; s < st.hi; ++s) {
            if (!st.has(s)) continue;
            for (int j = s * kKeys + warp; j < imin((s + 1) * kKeys, n); j += kWarps) {
                uint32_t w[E / 2];
                load16<E>(static_cast<const T*>(a.v) + (int64_t)(row0 + j) * a.v_row + (int64_t)kvh * a.v_head + lane * E, w);
                const int kind = odd_values<T, E>(w);
                const bool some = __any_sync(~0u, kind & 3), inf = __any_sync(~0u, kind & 2);
                if (some && lane == 0) {
                    atomicMin(&odd->lo, j);
                    atomicMax(&odd->hi, j);
                    if (inf) odd->inf = 1;
                }
            }
        }
        softmax_sync<TILES>();
        const OddKeys o = *odd;
        for (int r = warp; r < rows; r += kWarps) {
            const int kind = kind_of(r);
            if (kind == 0) continue;
            const int f = first + r / group, p = n - m + f;
            const Span v = visible(p, n, causal, (int)a.window, (int)a.sinks);
            const bool seen = o.hi >= 0 && (o.hi < v.head || (o.hi < v.hi && (o.lo >= v.lo || v.head >= v.lo)));
            if (seen && !(o.inf && (kind & 1))) continue;
            slow_row<T, D>(a, row0, n, p, row0 + f, kvh * group + r % group, kvh, causal);
        }
    }
    softmax_sync<TILES>();  // `odd` is free again
}

template <class T, int D, int TILES> __device__ __noinline__ void redo_items(const mrl_attn& a, const Items<TILES> work, int group, OddKeys* odd) {
    for (unsigned r_no = 0; r_no * gridDim.x < work.items; ++r_no) {
        const unsigned i = work.number(r_no);
        if (i >= work.items) break;
        const Item<TILES> it = work.at(i);
#pragma unroll 1
        for (int t = 0; t < TILES; ++t) {
            const Steps st = TILES == 2 && t == 1 ? it.st[TILES - 1] : it.st[0];
            if (st.hi > 0) redo_tile<T, D, TILES>(a, it.row, it.len, it.m, it.first + t * work.tokens, work.tokens, group, it.head, st, work.causal, odd);
        }
    }
}

template <class T, int D, bool PAGED>
__global__ void __launch_bounds__(Shape<D, PAGED>::threads, 1)
    tc_kernel(const __grid_constant__ TcParams pr, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v) {
    using S = Shape<D, PAGED>;
    constexpr bool kBf = !PAGED && !__is_same(T, __half);  // operand type of the products
    constexpr int TILES = S::tiles, SB = S::sbufs, ST = S::stages;
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + (1024 - (tc::smem_u32(raw) & 1023)) % 1024;
    unsigned char* q_s = smem;                                  // per tile [D/64][128 rows][128 B], swizzled
    unsigned char* k_s = q_s + (size_t)TILES * S::q_bytes;      // per stage [D/64][128 keys][128 B]
    unsigned char* v_s = k_s + (size_t)ST * S::kv_bytes;        // per stage the same, over the cache [2 pages][D][128 B]
    __shared__ SeqItem info[S::seqs];
    __shared__ unsigned start_s[S::seqs];  // first item of the i-th sequence in order
    __shared__ uint16_t order_s[S::seqs];  // that sequence
    __shared__ int seq_s[PAGED ? S::seqs : 1];
    __shared__ unsigned scan_s[32];
    constexpr int KP = S::k_parts, VP = S::v_parts;
    __shared__ uint64_t q_full[TILES], q_empty[TILES], k_full[ST * KP], k_empty[ST * KP], v_full[ST * VP], v_empty[ST * VP], v_raw[ST * VP], s_full[2], p_full[2], o_full[TILES], o_free[TILES],
        pv_done[2], drained;
    __shared__ uint32_t tmem_s;
    __shared__ volatile int failed, redo_s;  // redo_s: some row's result is not finite
    __shared__ OddKeys odd_s;
    __shared__ float4 scales_s[kInfo];  // over the cache: K scales of a step's two pages, V scales
    __shared__ int present_s[kInfo];    // bit i: page i of the step exists
    __shared__ uint8_t q_up_s[PAGED ? 2 * TILES * 128 : 1];  // over the cache: log2 + 127 of what each row of Q was divided by, of a tile's last two items with steps

    const mrl_attn& a = pr.a;
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = (int)a.n_seqs, group = pr.group, tokens = pr.tokens;
    const int window = (int)a.window, sinks = (int)a.sinks, causal = pr.causal;

    if (tid == 0) {
        failed = 0;
        redo_s = 0;
        for (int i = 0; i < TILES; ++i) {
            tc::mbar_init(&q_full[i], PAGED ? 2 : 1);
            tc::mbar_init(&q_empty[i], 1);
            tc::mbar_init(&o_full[i], 1);
            tc::mbar_init(&o_free[i], 4);
        }
        for (int i = 0; i < ST * KP; ++i) {
            tc::mbar_init(&k_full[i], 1);
            tc::mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < ST * VP; ++i) {
            tc::mbar_init(&v_full[i], 1);
            tc::mbar_init(&v_empty[i], 1);
            tc::mbar_init(&v_raw[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&p_full[i], 4);
            tc::mbar_init(&pv_done[i], 1);
        }
        tc::mbar_init(&drained, 1);
        tc::fence_mbar_init();
    }
    if (warp == 8) {
        tc::tmem_alloc(&tmem_s, 512);
        tc::tmem_relinquish();
    }
    // ---- the call's sequences, longest first where there are few, so that the last items are short ones
    bool falls = false;
    for (int b = tid; b < n; b += S::threads) {
        const Rows r{a.seqs, a.cu, n, (int)a.n_tokens};
        falls = falls || r.falls(b);
        SeqItem q{0, r.begin(b), 0};
        q.m = r.end(b) - q.row;
        q.len = q.m;
        if (PAGED) {
            const int seq = a.seqs[b];
            const bool known = seq >= 0 && seq < (int)pr.c.max_seqs;
            seq_s[b] = known ? seq : 0;
            q.len = known ? min(max(pr.c.lens[seq], 0), (int)pr.c.max_pages * kPage) : 0;
            if (blockIdx.x == 0 && q.m > 0 && (!known || q.m > q.len)) atomicOr(pr.c.status, MRL_KV_BAD_INDEX);
        }
        info[b] = q;
    }
    const bool none = __syncthreads_or(falls);  // the items
    if (none && blockIdx.x == 0 && tid == 0 && (PAGED || a.status)) atomicOr(PAGED ? pr.c.status : a.status, MRL_KV_BAD_INDEX);
    for (int b = tid; b < n; b += S::threads) {
        int rank = b;
        if (n <= 128) {
            rank = 0;
            for (int x = 0; x < n; ++x) rank += info[x].len > info[b].len || (info[x].len == info[b].len && x < b);
        }
        order_s[rank] = (uint16_t)b;
    }
    __syncthreads();
    // ---- their items
    unsigned carry = 0;
    for (int at = 0; at < n; at += S::threads) {
        const int b = at + tid;
        unsigned v = 0;
        if (b < n) {
            const int m = info[order_s[b]].m;
            v = m > 0 && !none ? (unsigned)((m + TILES * tokens - 1) / (TILES * tokens)) * (unsigned)pr.heads : 0;
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
        for (int w = 0; w < S::threads / 32; ++w) {
            if (w < warp) before += scan_s[w];
            carry += scan_s[w];
        }
        if (b < n) start_s[b] = before + x - v;
        __syncthreads();
    }
    const unsigned items = carry;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_s;

    const Items<TILES> work{info, start_s, order_s, n, tokens, (unsigned)pr.heads, items, causal, window, sinks};
    auto item_at = [&](unsigned i) { return work.at(i); };
    const unsigned grid = gridDim.x;
    auto item_no = [&](unsigned r) { return work.number(r); };

    if (warp >= 8) fewer_registers<S::regs_other>();
    else if (warp < 4 * TILES) more_registers<S::regs_softmax>();
    if (warp < 4 * TILES) {
        // ---- softmax and epilogue of tile `tile`: thread = row
        const int tile = warp >> 2, r = tid & 127;
        const uint32_t lane_off = (uint32_t)(warp & 3) << 21;  // lane 32 (warp % 4) of tensor memory
        const int tok = pr.inner_q ? r % tokens : r / group, qh = pr.inner_q ? r / tokens : r % group;
        const bool row_used = r < tokens * group;
        uint32_t s_par = 0;  // bit i: buffer i
        uint32_t o_par = 0;  // the tile's items with steps so far, mod 2
        int step_no = 0, used = 0;
        for (unsigned r_no = 0; r_no * grid < items && !failed; ++r_no) {
            const unsigned i = item_no(r_no);
            if (i >= items) break;
            const Item<TILES> it = item_at(i);
            float cur = a.scale * kLog2e;
            const int f = it.first + tile * tokens, base = it.len - it.m;
            const Steps st = it.st[tile];
            const int p = base + f + tok;
            const Span span = f + tok < it.m ? visible(p, it.len, causal, window, sinks) : Span{0, 0, 0};
            // all of the tile's rows see keys [full_lo, full_hi) (and the sinks)
            const int p_lo = base + f, p_hi = base + imin(f + tokens, it.m) - 1;
            float m = -INFINITY, l = 0.0f, vref = 0.0f;
            bool any = false;
            for (int s = it.begin(); s < it.all.hi; s = it.next(s), ++step_no) {
                if (!st.has(s)) continue;
                const int buf = SB == 2 ? used & 1 : tile;
                if (!wait(&s_full[buf], (s_par >> buf) & 1, &failed)) break;
                s_par ^= 1u << buf;
                tc::fence_after();
                const uint32_t s_col = tmem + lane_off + S::tmem_s + buf * 128;
                const int key0 = s * kKeys;
                if (PAGED && !__is_same(T, __half) && !any) cur *= __uint_as_float((uint32_t)q_up_s[(o_par * TILES + tile) * 128 + r] << 23);
                float ka = cur, kb = cur, va = 1.0f, vb = 1.0f;
                bool full = key0 + kKeys <= it.len && (!causal || key0 + kKeys - 1 <= p_lo) &&
                            (window == 0 || key0 + kKeys <= sinks || (key0 > p_hi - window && (causal || key0 + kKeys - 1 < p_lo + window)));
                int there = 3;
                if (PAGED) {
                    const float4 x = scales_s[step_no & (kInfo - 1)];
                    there = present_s[step_no & (kInfo - 1)];
                    ka = fmaxf(ka * x.x, 1e-37f);  // of a page of zeros: a masked score stays -inf
                    kb = fmaxf(kb * x.y, 1e-37f);
                    va = x.z;
                    vb = x.w;
                    full = full && there == 3;
                }
                uint32_t x[128];
                MRL_TC_LD32(x, s_col);
                MRL_TC_LD32(x + 32, s_col + 32);
                MRL_TC_LD32(x + 64, s_col + 64);
                MRL_TC_LD32(x + 96, s_col + 96);
                tc::wait_ld();
                pin(x);
                if (!full) {
                    // visible keys of this row, relative to the step: [0, head) and [lo, hi)
                    const int head = span.head - key0, lo = span.lo - key0, hi = span.hi - key0;
                    auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; };  // bits 0 .. k - 1
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t see = below(head - 32 * w) | (below(hi - 32 * w) & ~below(lo - 32 * w));
                        if (PAGED && !(there >> (w >> 1) & 1)) see = 0;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!(see & (1u << j))) x[32 * w + j] = 0xff800000u;
                    }
                }
                float mx[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) mx[j] = __uint_as_float(x[16 * j]);
#pragma unroll
                for (int i = 1; i < 15; i += 2)
#pragma unroll
                    for (int j = 0; j < 8; ++j) mx[j] = max3(mx[j], __uint_as_float(x[16 * j + i]), __uint_as_float(x[16 * j + i + 1]));
#pragma unroll
                for (int j = 0; j < 8; ++j) mx[j] = fmaxf(mx[j], __uint_as_float(x[16 * j + 15]));
                const float top_a = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), top_b = fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]));
                const float top = fmaxf(top_a * ka, top_b * kb);
                // the maximum that is subtracted, and V's scale unit, move rarely; a page that the row sees nothing of has no
                // part in the unit, however large its scale
                float keep = 1.0f;
                if (PAGED) {
                    if (!(top_a > -INFINITY)) va = 0.0f;
                    if (!(top_b > -INFINITY)) vb = 0.0f;
                }
                const float vmax = fmaxf(va, vb);
                const bool grow = top > m + kSlack;
                if (PAGED && vmax > kScaleSlack * vref) {
                    keep = vref / vmax;
                    vref = vmax;
                }
                if (grow) {
                    const float le = m == -INFINITY ? 1.0f : ex2(m - top);  // O and l are 0 until a key was seen
                    keep *= le;
                    l *= le;
                    m = top;
                }
                if (any && __any_sync(~0u, keep != 1.0f)) {
                    if (SB == 2) {  // the product of the step before may still be adding to O
                        if (!wait(&pv_done[buf ^ 1], (uint32_t)((used - 1) >> 1) & 1, &failed)) break;
                        tc::fence_after();
                    }
                    const uint32_t o_col = tmem + lane_off + S::tmem_o + tile * D;
#pragma unroll 1
                    for (int h = 0; h < D / 16; ++h) {
                        uint32_t x[16];
                        TC_LD16(x, o_col + h * 16);
                        tc::wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * keep);
                        TC_ST16(o_col + h * 16, x);
                    }
                    tc::wait_st();
                }
                any = true;
                if (PAGED) {
                    const float per = vref > 0.0f ? __fdividef(1.0f, vref) : 0.0f;
                    va *= per;
                    vb *= per;
                }
                // P over S. A masked score is -inf. Over the cache P carries V's scale, put into the exponent and
                // taken out of the sum again; below 2^-24 of the unit it would leave f16 anyway.
                const float z = m == -INFINITY ? 0.0f : -m;
                if (PAGED) {
                    va = fmaxf(va, 5.9604645e-8f);
                    vb = fmaxf(vb, 5.9604645e-8f);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float k = h ? kb : ka, zz = PAGED ? z + __log2f(h ? vb : va) : z;
                    const uint64_t k2 = two(k, k), z2 = two(zz, zz);
                    uint64_t sum[4] = {0, 0, 0, 0};
                    uint32_t y[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        float e0, e1;
                        split(fma2(two(__uint_as_float(x[64 * h + 2 * j]), __uint_as_float(x[64 * h + 2 * j + 1])), k2, z2), e0, e1);
                        e0 = ex2(e0);
                        e1 = ex2(e1);
                        sum[j & 3] = add2(sum[j & 3], two(e0, e1));
                        y[j] = pack16<kBf>(e0, e1);
                    }
                    MRL_TC_ST32(s_col + h * 32, y);
                    float s0, s1;
                    split(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
                    l += PAGED ? __fdividef(s0 + s1, h ? vb : va) : s0 + s1;
                }
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) arrive(&p_full[buf]);
                ++used;
            }
            const bool in = row_used && f + tok < it.m;
            const int t_row = it.row + f + tok, h = it.head * group + qh;
            T* dst = static_cast<T*>(a.out) + (int64_t)t_row * a.o_row + (int64_t)h * a.o_head;
            float bad = 0.0f;
            if (any) {
                if (!wait(&o_full[tile], o_par, &failed)) break;
                o_par ^= 1;
                tc::fence_after();
                const uint32_t o_col = tmem + lane_off + S::tmem_o + tile * D;
                const float inv = l == 0.0f ? 0.0f : (PAGED ? vref : 1.0f) / l;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    uint32_t x[32];
                    MRL_TC_LD32(x, o_col + j * 32);
                    tc::wait_ld();
                    if (j == D / 32 - 1) {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) arrive(&o_free[tile]);
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float u = __uint_as_float(x[k + 2 * e]), v = __uint_as_float(x[k + 2 * e + 1]);
                            if (!PAGED) bad = fmaf(u, 0.0f, fmaf(v, 0.0f, bad));
                            w[e] = pack16<!__is_same(T, __half)>(l == 0.0f ? 0.0f : u * inv, l == 0.0f ? 0.0f : v * inv);
                        }
                        if (in) store32(dst + j * 32 + k, w, pr.sectors);
                    }
                }
            } else if (in) {
                for (int j = 0; j < D / 8; ++j) *reinterpret_cast<uint4*>(dst + j * 8) = make_uint4(0, 0, 0, 0);
            }
            if (in && a.lse) a.lse[(size_t)t_row * a.q_heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
            if (!PAGED && in && !(bad == 0.0f && l < INFINITY && m < INFINITY)) {
                // not finite: by the row's own scores, which makes it NaN throughout, or by a value of V that it sees or not
                if (!(l < INFINITY && m < INFINITY)) *reinterpret_cast<uint4*>(dst) = make_uint4(kOwnNaN, kOwnNaN, kOwnNaN, kOwnNaN);
                else redo_s = 1;
            }
        }
        if constexpr (!PAGED) {
            // Rows to be looked at again, when the CTA's pipeline has nothing to wait for any more: a row from its visible keys
            // alone takes long.
            softmax_sync<TILES>();
            if (tid == 0) redo_s = redo_s && !failed;
            softmax_sync<TILES>();
            if (redo_s) redo_items<T, D, TILES>(a, Items<TILES>{info, start_s, order_s, n, tokens, (unsigned)pr.heads, items, causal, window, sinks}, group, &odd_s);
        }
    } else if (warp == 8) {
        // ---- the products: the warp runs converged, so that what the instructions take sits in uniform registers,
        // and one elected lane issues them
        {
            constexpr uint32_t id_s = idesc_f16(kKeys, kBf, false), id_o = idesc_f16(D, kBf, !PAGED);
            const uint32_t q_low = __shfl_sync(~0u, desc_low(tc::smem_u32(q_s), 16), 0), k_low = __shfl_sync(~0u, desc_low(tc::smem_u32(k_s), 16), 0),
                           v_low = __shfl_sync(~0u, desc_low(tc::smem_u32(v_s), PAGED ? 16 : kKeys / VP * 128), 0), tm = __shfl_sync(~0u, tmem, 0);
            const bool leader = elect();
            uint32_t q_par = 0, p_par = 0, free_par = 0;
            int step_no = 0, used = 0;
            bool ok = true;
            auto commit = [&](uint64_t* bar) {
                if (leader) tc::mma_commit(bar);
                __syncwarp();
            };
            auto product_s = [&](int tile, int buf, int stage, uint32_t k_par, bool last) {
                const uint32_t q = q_low + (uint32_t)tile * (S::q_bytes >> 4), k = k_low + (uint32_t)stage * (S::kv_bytes >> 4),
                               d = tm + S::tmem_s + (uint32_t)buf * 128;
                constexpr int steps = D / 16 / KP;
#pragma unroll
                for (int part = 0; part < KP; ++part) {
                    if (KP > 1) {
                        if (!wait(&k_full[stage * KP + part], k_par, &failed)) return false;
                        tc::fence_after();
                    }
                    if (leader) {
#pragma unroll
                        for (int i = part * steps; i < (part + 1) * steps; ++i) {
                            const uint32_t off = (uint32_t)((i >> 2) * 16384 + (i & 3) * 32) >> 4;
                            mma_ss(d, desc(q + off), desc(k + off), id_s, i > 0);
                        }
                        if (KP > 1) tc::mma_commit(&k_empty[stage * KP + part]);
                        if (part == KP - 1) tc::mma_commit(&s_full[buf]);
                        if (part == KP - 1 && last) tc::mma_commit(&q_empty[tile]);
                    }
                    __syncwarp();
                }
                return true;
            };
            auto product_o = [&](int tile, int buf, int stage, uint32_t v_par, bool first) {
                const uint32_t v = v_low + (uint32_t)stage * (S::kv_bytes >> 4), d = tm + S::tmem_o + (uint32_t)tile * D, p = tm + S::tmem_s + (uint32_t)buf * 128;
                constexpr int steps = kKeys / 16 / VP;
#pragma unroll
                for (int part = 0; part < VP; ++part) {
                    if (!wait(&v_full[stage * VP + part], v_par, &failed)) return false;
                    tc::fence_after();
                    if (leader) {
#pragma unroll
                        for (int i = part * steps; i < (part + 1) * steps; ++i) {
                            const uint32_t off = (uint32_t)(PAGED ? (i >> 2) * (D * 128) + (i & 3) * 32 : part * (S::kv_bytes / VP) + (i % steps) * 2048) >> 4;
                            mma_ts(d, p + i * 8, desc(v + off), id_o, !(first && i == 0));
                        }
                        if (VP > 1) tc::mma_commit(&v_empty[stage * VP + part]);
                    }
                    __syncwarp();
                }
                return true;
            };
            for (unsigned r_no = 0; r_no * grid < items && ok && !failed; ++r_no) {
                const unsigned i = item_no(r_no);
                if (i >= items) break;
                const Item<TILES> it = item_at(i);
                bool q_here[TILES], begun[TILES];
                int pend[TILES], pend_buf[TILES];  // step whose P is to come, -1: none
#pragma unroll
                for (int t = 0; t < TILES; ++t) q_here[t] = begun[t] = false, pend[t] = -1, pend_buf[t] = t;
                // O += P V of tile t's pending step
                auto finish = [&](int t) {
                    const int no = pend[t];
                    if (!begun[t]) {  // the previous item's O has been read
                        if (!wait(&o_free[t], ((free_par >> t) & 1) ^ 1, &failed)) return false;
                        free_par ^= 1u << t;
                    }
                    if (!wait(&p_full[pend_buf[t]], (p_par >> pend_buf[t]) & 1, &failed)) return false;
                    p_par ^= 1u << pend_buf[t];
                    tc::fence_after();
                    if (!product_o(t, pend_buf[t], no % ST, (uint32_t)(no / ST) & 1, !begun[t])) return false;
                    if (SB == 2) commit(&pv_done[pend_buf[t]]);
                    begun[t] = true;
                    pend[t] = -1;
                    return true;
                };
                auto begin_q = [&](int t) {
                    if (q_here[t]) return true;
                    if (!wait(&q_full[t], (q_par >> t) & 1, &failed)) return false;
                    q_par ^= 1u << t;
                    q_here[t] = true;
                    tc::fence_after();
                    return true;
                };
                int prev = -1;  // the step before, whose V the tiles may still need
                for (int s = it.begin(); s < it.all.hi && ok; s = it.next(s), ++step_no) {
                    const int stage = step_no % ST;
                    const uint32_t k_par = (uint32_t)(step_no / ST) & 1;
                    if (KP == 1) {
                        if (!wait(&k_full[stage], k_par, &failed)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after();
                    }
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        if (!ok) continue;
                        const bool has = it.st[t].has(s), last = s == it.st[t].hi - 1;
                        if (SB == 2) {
                            // S of this step first: its buffer's last P went into O two steps ago
                            const int buf = used & 1;
                            ok = begin_q(t) && product_s(t, buf, stage, k_par, last);
                            if (ok && pend[t] >= 0) ok = finish(t);
                            pend[t] = step_no;
                            pend_buf[t] = buf;
                            ++used;
                        } else {
                            if (pend[t] >= 0) ok = finish(t);
                            if (!has || !ok) continue;
                            ok = begin_q(t) && product_s(t, t, stage, k_par, last);
                            pend[t] = step_no;
                        }
                    }
                    if (!ok) break;
                    if (KP == 1) commit(&k_empty[stage]);
                    if (VP == 1 && prev >= 0) commit(&v_empty[prev % ST]);
                    prev = step_no;
                }
                if (!ok) break;
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (pend[t] >= 0 && ok) ok = finish(t);
                    if (begun[t] && ok) commit(&o_full[t]);
                }
                if (VP == 1 && prev >= 0 && ok) commit(&v_empty[prev % ST]);
            }
            // no product, and no arrival of one on a barrier, outlasts the CTA
            commit(&drained);
            settle(&drained, 0);
        }
    } else if constexpr (!PAGED) {
        // ---- Q, K and V by TMA: boxes of 64 dims x 128 rows (Q: a tile's tokens x heads, V: a part's keys)
        if (warp == 9 && lane == 0) {
            int step_no = 0;
            uint32_t q_par = 0;
            Fills q_fills, k_fills, v_fills, raw_fills;
            uint32_t raw_par = 0;
            bool ok = true;
            for (unsigned r_no = 0; r_no * grid < items && ok && !failed; ++r_no) {
                const unsigned i = item_no(r_no);
                if (i >= items) break;
                const Item<TILES> it = item_at(i);
                for (int t = 0; t < TILES && ok; ++t) {
                    if (it.st[t].hi == 0) continue;
                    ok = wait(&q_empty[t], ((q_par >> t) & 1) ^ 1, &failed);
                    if (!ok) break;
                    q_fills.note(t, (q_par >> t) & 1);
                    q_par ^= 1u << t;
                    expect(&q_full[t], (uint32_t)(tokens * group) * D * 2);
                    const int row = it.row + it.first + t * tokens, h = it.head * group;
                    for (int d = 0; d < D / 64; ++d)
                        tma3(tc::smem_u32(q_s + (size_t)t * S::q_bytes + d * 16384), &map_q, d * 64, pr.inner_q ? row : h, pr.inner_q ? h : row, &q_full[t]);
                }
                for (int s = it.begin(); s < it.all.hi && ok; s = it.next(s), ++step_no) {
                    const int stage = step_no % ST;
                    const uint32_t par = (uint32_t)(step_no / ST) & 1;
                    const int row = it.row + s * kKeys;
                    for (int part = 0; part < KP && ok; ++part) {
                        uint64_t* bar = &k_full[stage * KP + part];
                        ok = wait(&k_empty[stage * KP + part], par ^ 1, &failed);
                        if (!ok) break;
                        expect(bar, S::kv_bytes / KP);
                        k_fills.note(stage * KP + part, par);
                        for (int d = part * (D / 64 / KP); d < (part + 1) * (D / 64 / KP); ++d)
                            tma3(tc::smem_u32(k_s + (size_t)stage * S::kv_bytes + d * 16384), &map_k, d * 64, pr.inner_k ? row : it.head,
                                 pr.inner_k ? it.head : row, bar);
                    }
                    for (int part = 0; part < VP && ok; ++part) {
                        // keys past the sequence's end: warp 10 has the stage first
                        const int x = stage * VP + part;
                        const bool cut = s * kKeys + (part + 1) * (kKeys / VP) > it.len;
                        uint64_t* bar = cut ? &v_raw[x] : &v_full[x];
                        ok = wait(&v_empty[x], par ^ 1, &failed);
                        if (!ok) break;
                        expect(bar, S::kv_bytes / VP);
                        if (cut) {
                            raw_fills.note(x, (raw_par >> x) & 1);
                            raw_par ^= 1u << x;
                            v_fills.drop(x);  // warp 10 ends that barrier's phase
                        } else {
                            v_fills.note(x, par);
                        }
                        const int v_row = row + part * (kKeys / VP);
                        for (int d = 0; d < D / 64; ++d)
                            tma3(tc::smem_u32(v_s + (size_t)stage * S::kv_bytes + part * (S::kv_bytes / VP) + d * (kKeys / VP * 128)), &map_v, d * 64,
                                 pr.inner_v ? v_row : it.head, pr.inner_v ? it.head : v_row, bar);
                    }
                }
            }
            q_fills.settle_all(q_full, TILES);
            k_fills.settle_all(k_full, ST * KP);
            v_fills.settle_all(v_full, ST * VP);
            raw_fills.settle_all(v_raw, ST * VP);
        }
        if (warp == 10) {
            // ---- V of keys past the sequence's end set to zero: rows of another sequence, or of none, may hold anything, and
            // 0 x NaN would reach every row of the item. Only an item's last step has such keys.
            int step_no = 0;
            uint32_t raw_par = 0;
            bool ok = true;
            for (unsigned r_no = 0; r_no * grid < items && ok && !failed; ++r_no) {
                const unsigned i = item_no(r_no);
                if (i >= items) break;
                const Item<TILES> it = item_at(i);
                if (it.all.hi == 0) continue;
                step_no += it.all.head + it.all.hi - it.all.lo;
                const int stage = (step_no - 1) % ST;
                for (int part = 0; part < VP && ok; ++part) {
                    constexpr int kRows = kKeys / VP;
                    const int have = it.len - (it.all.hi - 1) * kKeys - part * kRows;
                    if (have >= kRows) continue;
                    const int x = stage * VP + part;
                    ok = wait(&v_raw[x], (raw_par >> x) & 1, &failed);
                    if (!ok) break;
                    raw_par ^= 1u << x;
                    unsigned char* v = v_s + (size_t)stage * S::kv_bytes + part * (S::kv_bytes / VP);
                    const int from = imax(have, 0);
                    for (int d = 0; d < D / 64; ++d)
                        for (int y = from * 8 + lane; y < kRows * 8; y += 32) *reinterpret_cast<uint4*>(v + d * (kRows * 128) + y * 16) = make_uint4(0, 0, 0, 0);
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) arrive(&v_full[x]);
                }
            }
        }
    } else if (warp == 9) {
        // ---- K and V from the cache's f16 image, scales beside them
        if (lane == 0) {
            const mrl_kv_cache& c = pr.c;
            int step_no = 0;
            Fills k_fills, v_fills;
            bool ok = true;
            for (unsigned r_no = 0; r_no * grid < items && ok && !failed; ++r_no) {
                const unsigned i = item_no(r_no);
                if (i >= items) break;
                const Item<TILES> it = item_at(i);
                const int32_t* table = c.tables + (size_t)seq_s[it.b] * c.max_pages;
                auto page_of = [&](int index) {
                    const int page = index * kPage < it.len ? table[index] : -1;
                    return page >= 0 && page < (int)c.pages ? page : -1;
                };
                auto scale_of = [&](int page, int which) { return page >= 0 ? c.scales[block_index(c, a.layer, page, which, it.head)] : 0.0f; };
                // page numbers are looked up two steps early and scales one, so that neither is waited for
                int s = it.begin(), s1 = it.next(s);
                int p0 = -1, p1 = -1, n0 = -1, n1 = -1;
                if (s < it.all.hi) p0 = page_of(2 * s), p1 = page_of(2 * s + 1);
                if (s1 < it.all.hi) n0 = page_of(2 * s1), n1 = page_of(2 * s1 + 1);
                float4 sc = make_float4(scale_of(p0, 0), scale_of(p1, 0), scale_of(p0, 1), scale_of(p1, 1));
                for (; s < it.all.hi && ok; ++step_no) {
                    const int stage = step_no % ST;
                    const uint32_t par = (uint32_t)(step_no / ST) & 1;
                    auto image = [&](int page, int which) {
                        return page >= 0 ? pr.wide + (((size_t)page * 2 + which) * c.kv_heads + it.head) * kWide<D> : pr.zero;
                    };
                    const unsigned char *w0 = image(p0, 0), *w1 = image(p1, 0);
                    // read by the softmax of a step at most stages + 1 behind this one
                    scales_s[step_no & (kInfo - 1)] = sc;
                    present_s[step_no & (kInfo - 1)] = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
                    for (int part = 0; part < KP && ok; ++part) {
                        uint64_t* bar = &k_full[stage * KP + part];
                        ok = wait(&k_empty[stage * KP + part], par ^ 1, &failed);
                        if (!ok) break;
                        expect(bar, S::kv_bytes / KP);
                        k_fills.note(stage * KP + part, par);
                        for (int d = part * (D / 64 / KP); d < (part + 1) * (D / 64 / KP); ++d) {
                            const uint32_t to = tc::smem_u32(k_s + (size_t)stage * S::kv_bytes + d * 16384);
                            bulk(to, w0 + d * 8192, 8192, bar);
                            bulk(to + 8192, w1 + d * 8192, 8192, bar);
                        }
                    }
                    for (int part = 0; part < VP && ok; ++part) {
                        uint64_t* bar = &v_full[stage * VP + part];
                        ok = wait(&v_empty[stage * VP + part], par ^ 1, &failed);
                        if (!ok) break;
                        expect(bar, S::kv_bytes / VP);
                        v_fills.note(stage * VP + part, par);
                        const uint32_t to = tc::smem_u32(v_s + (size_t)stage * S::kv_bytes);
                        if (part == 0) bulk(to, image(p0, 1), kWide<D>, bar);
                        if (part == VP - 1) bulk(to + kWide<D>, image(p1, 1), kWide<D>, bar);
                    }
                    s = s1;
                    s1 = it.next(s);
                    p0 = n0;
                    p1 = n1;
                    sc = make_float4(scale_of(p0, 0), scale_of(p1, 0), scale_of(p0, 1), scale_of(p1, 1));
                    n0 = n1 = -1;
                    if (s1 < it.all.hi) n0 = page_of(2 * s1), n1 = page_of(2 * s1 + 1);
                }
            }
            k_fills.settle_all(k_full, ST * KP);
            v_fills.settle_all(v_full, ST * VP);
        }
    } else if (warp >= 10) {
        // ---- Q of the cache's attention, as f16
        constexpr int kConv = 64;
        const int ct = tid - 10 * 32;
        uint32_t q_par = 0;  // bit t: items with steps of tile t so far, mod 2
        bool ok = true;
        for (unsigned r_no = 0; r_no * grid < items && ok && !failed; ++r_no) {
            const unsigned i = item_no(r_no);
            if (i >= items) break;
            const Item<TILES> it = item_at(i);
            // D / 8 lanes to a row, 16 bytes each, copied to where the operand wants them, and bf16 made f16 there by
            // the thread that copied it. bf16 has more range than f16: a row is brought to [1, 2) by a power of two,
            // which goes to the softmax scale; what leaves f16's range below is 2^-24 of the row's largest.
            constexpr int kLanes = D / 8, kRows = kConv / kLanes;
            const int q_row = ct / kLanes, q_col = ct % kLanes;
            auto q_at = [&](int t, int r) { return q_s + (size_t)t * S::q_bytes + (q_col >> 3) * 16384 + r * 128 + (((q_col & 7) ^ (r & 7)) << 4); };
            auto copy_q = [&](int t) {
#pragma unroll 4
                for (int r = q_row; r < 128; r += kRows) {
                    const int f = it.first + t * tokens + r / group;
                    const bool in = r < tokens * group && f < it.m;
                    const T* from = static_cast<const T*>(a.q);
                    if (in) from += (int64_t)(it.row + f) * a.q_row + (int64_t)(it.head * group + r % group) * a.q_head + q_col * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(q_at(t, r))), "l"(from), "r"(in ? 16 : 0) : "memory");
                }
            };
            auto finish_q = [&](int t) {
                constexpr int kTurn = 4;  // rows of a thread in flight
                // Of the tile's items with steps, the one two before has used its slot up: the tile's last S of the one
                // before was issued after that one's P, and q_empty waited for it.
                uint8_t* const up_s = q_up_s + ((((q_par >> t) & 1) ^ 1) * TILES + t) * 128;
                for (int r0 = q_row; r0 < 128 && !__is_same(T, __half); r0 += kTurn * kRows) {
                    uint4 x[kTurn];
                    float top[kTurn];
#pragma unroll
                    for (int i = 0; i < kTurn; ++i) x[i] = *reinterpret_cast<const uint4*>(q_at(t, r0 + i * kRows));
#pragma unroll
                    for (int i = 0; i < kTurn; ++i) {
                        const T* e = reinterpret_cast<const T*>(&x[i]);
                        top[i] = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) top[i] = fmaxf(top[i], fabsf(to_f32<T>(e[j])));
                    }
#pragma unroll
                    for (int d = kLanes / 2; d; d >>= 1)
#pragma unroll
                        for (int i = 0; i < kTurn; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], d));
#pragma unroll
                    for (int i = 0; i < kTurn; ++i) {
                        const T* e = reinterpret_cast<const T*>(&x[i]);
                        const int r = r0 + i * kRows;
                        float down = 1.0f;
                        uint32_t up = 127;
                        const uint32_t ex = __float_as_uint(top[i]) >> 23;
                        if (ex > 0 && ex < 255) {
                            up = min(ex, 253u);
                            down = __uint_as_float((254u - up) << 23);
                        }
                        uint32_t y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = pack16<false>(to_f32<T>(e[2 * j]) * down, to_f32<T>(e[2 * j + 1]) * down);
                        *reinterpret_cast<uint4*>(q_at(t, r)) = make_uint4(y[0], y[1], y[2], y[3]);
                        if (q_col == 0) up_s[r] = (uint8_t)up;
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&q_full[t]);
            };
            for (int t = 0; t < TILES && ok; ++t) {
                if (it.st[t].hi == 0) continue;
                ok = wait(&q_empty[t], ((q_par >> t) & 1) ^ 1, &failed);
                q_par ^= 1u << t;
                if (ok) copy_q(t);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            for (int t = 0; t < TILES && ok; ++t)
                if (it.st[t].hi > 0) finish_q(t);
        }
    }
    __syncthreads();
    if (warp == 8) tc::tmem_dealloc(tmem, 512);
    uint32_t* const status = PAGED ? pr.c.status : a.status;
    if (tid == 0 && failed && status) atomicOr(status, MRL_KV_TIMEOUT);
}

// The pages that the call's sequences see, codes to f16 in the operands' layout: every 64 codes of K (a
// token's dims 64 i ..) or V (a dim's tokens) become a swizzled row of 128 bytes. A page that several
// sequences share lies at the same index of their tables after a fork: the first of them widens it.
// 1 byte read, 2 written per code; a CTA takes several blocks of a page at a time, all their loads at once, since
// the way to a page (sequence, table, refs) is a chain of dependent loads. Measured, 324 pages of 8 kv heads of
// 128 (42 MB of codes, 127 MB in all): 20.5 us, 6.2 TB/s; 31 us with 16-byte stores.
constexpr int kWidenThreads = 256, kWidenSeqs = 512;
template <int D> __global__ void __launch_bounds__(kWidenThreads) widen_kernel(mrl_kv_cache c, mrl_attn a, unsigned char* wide) {
    constexpr int kBlocks = D == 256 ? 2 : 4;                             // blocks of 64 x D codes per turn
    constexpr int kPieces = kPage * D / 16 / kWidenThreads;               // of a thread, per block
    struct Seen {
        int seq, head, lo, n;  // visible pages [0, head) and [lo, lo + n - head)
    };
    __shared__ Seen seen[kWidenSeqs];
    __shared__ unsigned start[kWidenSeqs];
    __shared__ unsigned scan_s[kWidenThreads / 32];
    __shared__ int skip_s;
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, n = (int)a.n_seqs, window = (int)a.window, sinks = (int)a.sinks;
    const Rows rows{a.seqs, a.cu, n, (int)a.n_tokens};
    unsigned carry = 0;
    for (int at = 0; at < n; at += kWidenThreads) {
        const int b = at + tid;
        Seen s{0, 0, 0, 0};
        if (b < n) {
            const int seq = a.seqs[b], m = rows.end(b) - rows.begin(b);
            if (seq >= 0 && seq < (int)c.max_seqs && m > 0) {
                const int len = min(max(c.lens[seq], 0), (int)c.max_pages * kPage);
                const Span v = visible(max(len - m, 0), len, 1, window, sinks);  // the first row sees the earliest
                s.seq = seq;
                s.lo = min(v.lo, len) / kPage;
                s.head = min(pages_of(min(sinks, v.lo)), s.lo);
                s.n = s.head + pages_of(len) - s.lo;
            }
            seen[b] = s;
        }
        unsigned x = (unsigned)s.n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) scan_s[warp] = x;
        __syncthreads();
        unsigned before = carry;
        for (int w = 0; w < kWidenThreads / 32; ++w) {
            if (w < warp) before += scan_s[w];
            carry += scan_s[w];
        }
        if (b < n) start[b] = before + x - (unsigned)s.n;
        __syncthreads();
    }
    const unsigned heads = 2 * c.kv_heads, turns = (heads + kBlocks - 1) / kBlocks, units = carry * turns;
    for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
        const unsigned p = u / turns, block0 = u % turns * kBlocks;
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= p) lo = mid;
            else hi = mid;
        }
        const Seen s = seen[lo];
        const int i = (int)(p - start[lo]), index = i < s.head ? i : s.lo + i - s.head;
        const int page = c.tables[(size_t)s.seq * c.max_pages + index];
        if (page < 0 || page >= (int)c.pages) continue;
        const uint4* src = reinterpret_cast<const uint4*>(c.codes + (block_index(c, a.layer, page, 0, 0) + block0) * (size_t)(kPage * D));
        uint4 w[kBlocks][kPieces];
#pragma unroll
        for (int k = 0; k < kBlocks; ++k)
#pragma unroll
            for (int x = 0; x < kPieces; ++x)
                if (block0 + k < heads) w[k][x] = src[k * (kPage * D / 16) + x * kWidenThreads + tid];
        if (c.refs[page] > 1) {
            __syncthreads();
            if (tid == 0) skip_s = 0;
            __syncthreads();
            for (int b = tid; b < lo; b += kWidenThreads) {
                const Seen o = seen[b];
                const bool has = index < o.head || (index >= o.lo && index < o.lo + o.n - o.head);
                if (has && c.tables[(size_t)o.seq * c.max_pages + index] == page) skip_s = 1;
            }
            __syncthreads();
            if (skip_s) continue;
        }
        unsigned char* dst = wide + ((size_t)page * heads + block0) * kWide<D>;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
#pragma unroll
            for (int x = 0; x < kPieces; ++x) {
                if (block0 + k >= heads) continue;
                const int at = x * kWidenThreads + tid, line = at >> 2, quarter = at & 3, sw = line & 7;
                uint4 e0, e1;
                widen4(w[k][x].x, e0.x, e0.y);
                widen4(w[k][x].y, e0.z, e0.w);
                widen4(w[k][x].z, e1.x, e1.y);
                widen4(w[k][x].w, e1.z, e1.w);
                // the two chunks are one 32-byte sector, written as one: halves apart would be merged in L2
                unsigned char* to = dst + k * kWide<D> + line * 128 + ((((2 * quarter) ^ sw) >> 1) << 5);
                const bool odd = sw & 1;
                const uint4 f0 = odd ? e1 : e0, f1 = odd ? e0 : e1;
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(f0.x), "r"(f0.y), "r"(f0.z), "r"(f0.w), "r"(f1.x),
                             "r"(f1.y), "r"(f1.z), "r"(f1.w)
                             : "memory");
            }
        }
    }
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
    static Encode f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess) p = nullptr;
        return reinterpret_cast<Encode>(p);
    }();
    return f;
}

// [rows][heads][D] 16-bit rows: dimensions D, then head and row in the order of their strides; boxes of 64
// dims, `box_heads` heads and `box_rows` rows.
bool make_map(CUtensorMap* map, const mrl_attn& a, const void* p, int64_t row, int64_t head, uint32_t heads, int d, int box_heads, int box_rows, int* inner) {
    if (heads == 1) head = d;
    if (a.n_tokens == 1) row = (int64_t)heads * head;
    const bool in = heads > 1 && row < head;
    const cuuint64_t dims[3] = {(cuuint64_t)d, in ? a.n_tokens : heads, in ? heads : a.n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)(in ? row : head) * 2, (cuuint64_t)(in ? head : row) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)(in ? box_rows : box_heads), (cuuint32_t)(in ? box_heads : box_rows)}, one[3] = {1, 1, 1};
    *inner = in;
    if (strides[0] >= 1ull << 40 || strides[1] >= 1ull << 40) return false;  // a map's limit
    return encoder()(map, a.dtype == MRL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box,
                  one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, bool PAGED> int launch(TcParams p, int sms, cudaStream_t s) {
    using S = Shape<D, PAGED>;
    CUtensorMap mq = {}, mk = {}, mv = {};
    if (!PAGED) {
        if (!encoder()) return kTcNoMaps;
        if (!make_map(&mq, p.a, p.a.q, p.a.q_row, p.a.q_head, p.a.q_heads, D, p.group, 128 / p.group, &p.inner_q)) return kTcBadQ;
        if (!make_map(&mk, p.a, p.a.k, p.a.k_row, p.a.k_head, p.a.kv_heads, D, 1, kKeys, &p.inner_k)) return kTcBadK;
        if (!make_map(&mv, p.a, p.a.v, p.a.v_row, p.a.v_head, p.a.kv_heads, D, 1, kKeys / S::v_parts, &p.inner_v)) return kTcBadV;
    }
    p.tokens = 128 / p.group;
    if (const cudaError_t e = allow_smem<tc_kernel<T, D, PAGED>>((int)S::smem)) return (int)e;
    const mrl_attn a = p.a;
    for (uint32_t at = 0; at < a.n_seqs; at += S::seqs) {
        p.a.n_seqs = a.n_seqs - at < (uint32_t)S::seqs ? a.n_seqs - at : (uint32_t)S::seqs;
        p.a.seqs = a.seqs ? a.seqs + at : nullptr;
        p.a.cu = a.cu + at;
        if (PAGED) {
            widen_kernel<D><<<(unsigned)sms * 8, kWidenThreads, 0, s>>>(p.c, p.a, const_cast<unsigned char*>(p.wide));
            if (const cudaError_t e = cudaGetLastError()) return (int)e;
        }
        // at most one part-filled item per sequence and head
        const uint64_t span = (uint64_t)S::tiles * p.tokens, each = (a.max_rows + span - 1) / span;
        const uint64_t most = std::min(a.n_tokens / span + p.a.n_seqs, p.a.n_seqs * each) * p.heads;
        tc_kernel<T, D, PAGED><<<(unsigned)(most < (uint64_t)sms ? most : sms), S::threads, S::smem, s>>>(p, mq, mk, mv);
        if (const cudaError_t e = cudaGetLastError()) return (int)e;
    }
    return 0;
}

template <bool PAGED> int dispatch(const TcParams& p, uint32_t d, int sms, cudaStream_t s) {
    if (p.a.dtype == MRL_F16)
        return d == 64 ? launch<__half, 64, PAGED>(p, sms, s) : d == 128 ? launch<__half, 128, PAGED>(p, sms, s) : launch<__half, 256, PAGED>(p, sms, s);
    return d == 64    ? launch<__nv_bfloat16, 64, PAGED>(p, sms, s)
           : d == 128 ? launch<__nv_bfloat16, 128, PAGED>(p, sms, s)
                      : launch<__nv_bfloat16, 256, PAGED>(p, sms, s);
}

}  // namespace
}  // namespace kv

size_t kv_wide_bytes(const mrl_kv_cache& c) { return kKvZeroBytes + (size_t)c.pages * 2 * kv::page_bytes(c); }

int launch_attend_tc(const mrl_kv_cache* c, const mrl_attn& a, int sms, void* wide, cudaStream_t s) {
    kv::TcParams p;
    p.zero = static_cast<const unsigned char*>(wide);
    p.wide = p.zero + kKvZeroBytes;
    p.c = c ? *c : mrl_kv_cache{};
    p.a = a;
    p.heads = (int)(c ? c->kv_heads : a.kv_heads);
    p.group = (int)a.q_heads / p.heads;
    p.causal = c ? 1 : (int)(a.causal != 0);
    p.sectors = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.o_row % 16 == 0 && a.o_head % 16 == 0;
    p.inner_q = p.inner_k = p.inner_v = 0;
    return c ? kv::dispatch<true>(p, c->head_dim, sms, s) : kv::dispatch<false>(p, a.head_dim, sms, s);
}

}  // namespace mrl
