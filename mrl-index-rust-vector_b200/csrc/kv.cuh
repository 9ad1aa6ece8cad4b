// kv.cuh — device helpers and launchers of the paged 8-bit cache and the attention operators
// (include/mrl_kv.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/mrl_kv.h"
#include "mrl_internal.cuh"

namespace mrl {
namespace kv {

constexpr int kPage = (int)MRL_KV_PAGE;

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }

__host__ __device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// Bytes of one page of one layer, and of one head's K (or V) block in it.
__host__ __device__ __forceinline__ size_t block_bytes(const mrl_kv_cache& c) { return (size_t)kPage * c.head_dim; }
__host__ __device__ __forceinline__ size_t page_bytes(const mrl_kv_cache& c) { return 2 * c.kv_heads * block_bytes(c); }
__device__ __forceinline__ size_t block_index(const mrl_kv_cache& c, uint32_t layer, int page, int which, int head) {
    return (((size_t)layer * c.pages + page) * 2 + which) * c.kv_heads + head;
}

// A call's rows (mrl_kv.h): sequences, their row offsets, or one row per sequence (cu null).
struct Rows {
    const int32_t* seqs;
    const int32_t* cu;
    int n, tokens;
    __device__ __forceinline__ int begin(int b) const { return cu ? min(max(cu[b], 0), tokens) : b; }
    __device__ __forceinline__ int end(int b) const { return cu ? min(max(cu[b + 1], 0), tokens) : b + 1; }
    // Offsets that decrease at b. Where none do, the sequences' rows are at most `tokens` together, and sums over them
    // stay in range; else a call does nothing.
    __device__ __forceinline__ bool falls(int b) const { return cu && cu[b + 1] < cu[b]; }
};

// Largest b in [0, n) with f(b) <= x, f not decreasing, f(0) <= x: 32 probes a step by one warp.
template <class F> __device__ __forceinline__ int warp_find(int n, long long x, F f) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + lane * step;
        const unsigned ok = __ballot_sync(~0u, at < hi && f(at) <= x);
        const int last = 31 - __clz((int)(ok | 1u));
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Units of page-wise work over a call's rows: the touched pages of sequence b are units
// base(b) .. base(b) + touched - 1 with base(b) = floor(begin(b) / 64) + 2 b, which leaves room for
// them whatever the lengths are (m rows touch at most floor((m + 62) / 64) + 1 pages, and
// base(b + 1) - base(b) >= floor(m / 64) + 2). With one row per sequence unit b is its page.
struct PageUnit {
    int seq;         // table row, -1: no such sequence, or one shorter than its rows
    int index;       // page of the sequence
    int page;        // page of the pool, -1: missing
    int row;         // first row of the call in the page (seq -1: the unit's share of the rows)
    int slot, count; // its slot in the page, and rows of the call in it (0: nothing to do)
};
__host__ __device__ __forceinline__ int page_units(int n, int tokens, bool has_cu) {
    return has_cu ? tokens / kPage + 2 * n : n;
}
// Called by a full warp; the result is warp-uniform.
__device__ __forceinline__ PageUnit find_page_unit(const mrl_kv_cache& c, const Rows& r, int unit) {
    PageUnit u{-1, 0, -1, 0, 0, 0};
    int b = unit, local = 0;
    if (r.cu) {
        b = warp_find(r.n, unit, [&](int i) { return (long long)(r.begin(i) / kPage) + 2ll * i; });
        local = unit - (r.begin(b) / kPage + 2 * b);
    }
    const int seq = r.seqs[b], lo = r.begin(b), m = r.end(b) - lo;
    if (m <= 0 || local < 0) return u;
    const int len = seq >= 0 && seq < (int)c.max_seqs ? c.lens[seq] : -1;
    const int start = len - m;
    if (len < m || (long long)len > (long long)c.max_pages * kPage) {
        u.row = lo + local * kPage;
        u.count = max(0, min(kPage, m - local * kPage));
        return u;
    }
    const int index = start / kPage + local;
    const int from = max(start, index * kPage), to = min(len, (index + 1) * kPage);
    if (from >= to) return u;
    u.seq = seq;
    u.index = index;
    const int page = c.tables[(size_t)seq * c.max_pages + index];
    u.page = page >= 0 && page < (int)c.pages ? page : -1;
    u.row = lo + from - start;
    u.slot = from - index * kPage;
    u.count = to - from;
    return u;
}

// The keys a query at position p sees among keys [0, n): [0, head) and [lo, hi).
struct Span {
    int head, lo, hi;
};
__host__ __device__ __forceinline__ int imin(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }
__host__ __device__ __forceinline__ Span visible(int p, int n, int causal, int window, int sinks) {
    const int top = imax(causal ? imin(p + 1, n) : n, 0);
    if (window <= 0) return Span{0, 0, top};
    Span s;
    s.lo = imin(imax(p - window + 1, 0), top);
    s.hi = causal || window >= n - p ? top : imax(p + window, s.lo);
    s.hi = imax(s.hi, imin(sinks, top));  // sinks past the window's end: everything up to them
    s.head = imin(sinks, s.lo);
    return s;
}

// Dynamic shared memory a kernel may be launched with, set once per kernel and device.
template <auto kernel> cudaError_t allow_smem(int bytes) {
    static bool set[64] = {};
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return e;
    if (device < 64 && set[device]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) set[device] = true;
    return e;
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace kv

// Launchers: MRL_OK or a cudaError_t (> 0).
// scratch sizes in bytes of the page operations' lists
size_t kv_list_bytes(const mrl_kv_cache& c, uint32_t n);
int launch_kv_reserve(const mrl_kv_cache& c, const int32_t* seqs, const int32_t* add, uint32_t n, void* scratch, cudaStream_t s);
int launch_kv_fork(const mrl_kv_cache& c, const int32_t* parents, const int32_t* children, uint32_t n, int sms, void* scratch,
                   cudaStream_t s);
int launch_kv_release(const mrl_kv_cache& c, const int32_t* seqs, uint32_t n, uint32_t trim, uint32_t window, uint32_t sinks,
                      cudaStream_t s);
int launch_kv_compact(const mrl_kv_cache& c, int sms, void* scratch, cudaStream_t s);
int launch_kv_copy_pages(const mrl_kv_cache& c, const int32_t* src, const int32_t* dst, uint32_t n, int sms, cudaStream_t s);
int launch_kv_append(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, const void* k, int64_t k_row, int64_t k_head,
                     const void* v, int64_t v_row, int64_t v_head, const kv::Rows& r, cudaStream_t s);
int launch_kv_read(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, void* k, void* v, const kv::Rows& r, cudaStream_t s);
// Decode: scratch for the pieces of split items, and zeroed counters; sequences of one launch
constexpr uint32_t kKvDecodeSeqs = 1024;
size_t kv_decode_bytes(uint32_t head_dim, int sms);
int launch_kv_decode(const mrl_kv_cache& c, const mrl_attn& a, int sms, void* scratch, unsigned* counters, cudaStream_t s);
// Tensor-core attention: over the cache (c; `wide` is kKvZeroBytes of zeros and room for a 16-bit image of one
// layer's pool) or over the call's own k and v. Below 0: no tensor maps in this driver, or an operand
// with strides that a map cannot describe.
enum : int { kTcNoMaps = -1, kTcBadQ = -2, kTcBadK = -3, kTcBadV = -4 };
constexpr size_t kKvZeroBytes = 64 * 256 * 2;
size_t kv_wide_bytes(const mrl_kv_cache& c);
int launch_attend_tc(const mrl_kv_cache* c, const mrl_attn& a, int sms, void* wide, cudaStream_t s);
}  // namespace mrl
