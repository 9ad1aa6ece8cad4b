// kv_pages.cu — bookkeeping of the paged cache on the device (include/mrl_kv.h): reserve, fork, release,
// trim, compact, copy. Every decision is made by one CTA over the refs and the call's list, so the
// result does not depend on scheduling: free pages are taken lowest index first. Page contents are then
// moved by a second launch over the whole device.
//
// A fork or a compact has to read and write each copied page once (2 x layers x 2 x kv_heads x 64 x
// head_dim bytes a page): bound by HBM for large ones, by the two launches for small ones. Measured, 8 kv heads of 128: 48
// forks over 8 layers 5.3 us for the plan and 11.8 us for the tails (50 MB written, their 8 sources in L2); a compact that moves
// 116 MB 5.3 and 35 us (6.6 TB/s read and written); a reserve of 24 sequences 6.5 us; a release 2.7 us.
#include "kv.cuh"

namespace mrl {
namespace kv {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kScanPages = 16;        // refs per thread and step of a scan over the pool
constexpr int kCopyThreads = 256;
constexpr int kCopyVec = 8;           // 16-byte loads in flight per thread
constexpr size_t kCopyChunk = (size_t)kCopyThreads * kCopyVec * 16;  // 32 KiB
constexpr int kMark = (int)0x80000000u;

// Lists of one page operation in the context's scratch.
struct Lists {
    int* count;  // [0]: pairs to copy, [1]: pages held (compact)
    int* off;    // [n]
    int* a;      // [pages]: free pages taken / sources
    int* b;      // [pages]: destinations
    int* map;    // [pages]: compact, new index of a moved page
};

// Exclusive prefix sum over the block; *total gets the sum. All kPlanThreads threads call it.
__device__ int block_scan(int v, int* total, int* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(~0u, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();  // sh is free
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = sh[lane], s = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(~0u, s, d);
            if (lane >= d) s += y;
        }
        sh[lane] = s - w;
        if (lane == 31) sh[32] = s;
    }
    __syncthreads();
    *total = sh[32];
    return x - v + sh[warp];
}

// Refs of pages base .. base + 15 as a bit mask of the held ones, and how many of the 16 exist.
__device__ __forceinline__ unsigned held_mask(const int32_t* refs, int pages, int base, int* have) {
    unsigned m = 0;
    *have = max(0, min(kScanPages, pages - base));
    if (*have == kScanPages && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
        const int4* p = reinterpret_cast<const int4*>(refs + base);
#pragma unroll
        for (int i = 0; i < kScanPages / 4; ++i) {
            const int4 r = p[i];
            m |= (unsigned)(r.x > 0) << (4 * i) | (unsigned)(r.y > 0) << (4 * i + 1) | (unsigned)(r.z > 0) << (4 * i + 2) |
                 (unsigned)(r.w > 0) << (4 * i + 3);
        }
    } else {
        for (int i = 0; i < *have; ++i) m |= (unsigned)(refs[base + i] > 0) << i;
    }
    return m;
}

// The `want` lowest free pages into list[0 ..]; returns how many were found (want, or all free ones).
__device__ int take_free(const mrl_kv_cache& c, int want, int* list, int* sh) {
    int found = 0;
    const int pages = (int)c.pages;
    for (int at = 0; at < pages && found < want; at += kPlanThreads * kScanPages) {
        const int base = at + (int)threadIdx.x * kScanPages;
        int have, total;
        unsigned free_bits = ~held_mask(c.refs, pages, base, &have);
        free_bits &= have >= 32 ? ~0u : (1u << have) - 1u;
        int rank = found + block_scan(__popc(free_bits), &total, sh);
        while (free_bits && rank < want) {
            list[rank++] = base + __ffs((int)free_bits) - 1;
            free_bits &= free_bits - 1;
        }
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

__device__ __forceinline__ bool in_range(int i, uint32_t n) { return i >= 0 && i < (int)n; }

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(mrl_kv_cache c, const int32_t* seqs, const int32_t* add, int n, Lists l) {
    __shared__ int sh[33];
    __shared__ unsigned bad;
    const int tid = (int)threadIdx.x;
    if (tid == 0) bad = 0;
    __syncthreads();
    // Each listed sequence's length carries a mark while its need is counted: a sequence listed twice,
    // or one whose length is not a length, shows. Entries that set no mark have offset -1.
    long long need_all = 0;
    for (int at = 0; at < n; at += kPlanThreads) {
        const int i = at + tid;
        int need = 0;
        bool marked = false;
        if (i < n) {
            const int s = seqs[i], a = add[i];
            if (!in_range(s, c.max_seqs) || a < 0) {
                atomicOr(&bad, MRL_KV_BAD_INDEX);
            } else {
                const int len = atomicOr(&c.lens[s], kMark);
                marked = len >= 0;
                if (len < 0) {
                    atomicOr(&bad, MRL_KV_BAD_INDEX);
                } else if ((long long)len + a > (long long)c.max_pages * kPage) {
                    atomicOr(&bad, MRL_KV_ROW_FULL);
                } else {
                    need = pages_of(len + a) - pages_of(len);
                }
            }
        }
        int total;
        const int x = block_scan(need, &total, sh);
        if (i < n) l.off[i] = marked ? (int)min(need_all + x, (long long)INT32_MAX) : -1;
        need_all += total;
    }
    __syncthreads();
    if (tid == 0 && !bad && need_all > (long long)c.pages) bad = MRL_KV_NO_PAGES;
    __syncthreads();
    if (!bad && need_all > 0) {
        const int found = take_free(c, (int)need_all, l.a, sh);
        if (tid == 0 && found < (int)need_all) bad = MRL_KV_NO_PAGES;
    }
    __syncthreads();
    if (bad) {
        for (int i = tid; i < n; i += kPlanThreads)
            if (l.off[i] >= 0) atomicAnd(&c.lens[seqs[i]], ~kMark);
        if (tid == 0) atomicOr(c.status, bad);
        return;
    }
    // One thread per taken page: its sequence is the last one whose offset is not above it.
    for (int r = tid; r < (int)need_all; r += kPlanThreads) {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (l.off[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int s = seqs[lo], len = c.lens[s] & ~kMark, page = l.a[r];
        c.tables[(size_t)s * c.max_pages + pages_of(len) + (r - l.off[lo])] = page;
        c.refs[page] = 1;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) c.lens[seqs[i]] = (c.lens[seqs[i]] & ~kMark) + add[i];
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(mrl_kv_cache c, const int32_t* parents, const int32_t* children, int n, Lists l) {
    __shared__ int sh[33];
    __shared__ unsigned bad;
    const int tid = (int)threadIdx.x;
    if (tid == 0) bad = 0;
    __syncthreads();
    // Children must be empty and listed once (their lengths carry a mark meanwhile), parents must not be
    // empty: so no child is a parent.
    int tails = 0;
    for (int at = 0; at < n; at += kPlanThreads) {
        const int i = at + tid;
        int need = 0;
        bool marked = false;
        if (i < n) {
            const int p = parents[i], ch = children[i];
            if (!in_range(p, c.max_seqs) || !in_range(ch, c.max_seqs)) {
                atomicOr(&bad, MRL_KV_BAD_INDEX);
            } else {
                const int len = c.lens[p], was = p == ch ? -1 : atomicOr(&c.lens[ch], kMark);
                marked = was >= 0;
                if (was != 0 || len <= 0 || len > (long long)c.max_pages * kPage) {
                    atomicOr(&bad, MRL_KV_BAD_INDEX);
                } else if (len % kPage) {
                    need = in_range(c.tables[(size_t)p * c.max_pages + len / kPage], c.pages);
                }
            }
        }
        int total;
        const int x = block_scan(need, &total, sh);
        if (i < n) l.off[i] = marked ? tails + x : -1;
        tails += total;
    }
    __syncthreads();
    if (!bad) {
        const int found = tails > (int)c.pages ? -1 : take_free(c, tails, l.b, sh);
        if (tid == 0 && found < tails) bad = MRL_KV_NO_PAGES;
    }
    __syncthreads();
    if (bad) {
        for (int i = tid; i < n; i += kPlanThreads)
            if (l.off[i] >= 0) atomicAnd(&c.lens[children[i]], ~kMark);
        if (tid == 0) {
            atomicOr(c.status, bad);
            l.count[0] = -1;
        }
        return;
    }
    for (int i = tid; i < n; i += kPlanThreads) {
        const int len = c.lens[parents[i]];
        const int next = i + 1 < n ? l.off[i + 1] : tails;
        if (next > l.off[i]) {
            l.a[l.off[i]] = c.tables[(size_t)parents[i] * c.max_pages + len / kPage];
            c.refs[l.b[l.off[i]]] = 1;
        }
        c.lens[children[i]] = len;
    }
    if (tid == 0) l.count[0] = tails;
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(mrl_kv_cache c, Lists l) {
    __shared__ int sh[33];
    const int tid = (int)threadIdx.x, pages = (int)c.pages;
    int held = 0;
    for (int at = tid * kScanPages; at < pages; at += kPlanThreads * kScanPages) {
        int have;
        held += __popc(held_mask(c.refs, pages, at, &have));
    }
    int live;
    block_scan(held, &live, sh);
    int holes = 0, highs = 0;
    for (int at = 0; at < pages; at += kPlanThreads * kScanPages) {
        const int base = at + tid * kScanPages;
        int have, total;
        const unsigned m = held_mask(c.refs, pages, base, &have);
        const unsigned exist = have >= 32 ? ~0u : (1u << have) - 1u;
        const int below = max(0, min(kScanPages, live - base));  // pages of mine under `live`
        const unsigned low = below >= 32 ? ~0u : (1u << below) - 1u;
        unsigned hole = ~m & exist & low, high = m & exist & ~low;
        int rank = holes + block_scan(__popc(hole), &total, sh);
        holes += total;
        for (; hole; hole &= hole - 1) l.b[rank++] = base + __ffs((int)hole) - 1;
        rank = highs + block_scan(__popc(high), &total, sh);
        highs += total;
        for (; high; high &= high - 1) l.a[rank++] = base + __ffs((int)high) - 1;
    }
    __syncthreads();
    for (int i = tid; i < highs; i += kPlanThreads) {  // as many holes as pages to move
        const int from = l.a[i], to = l.b[i];
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
        l.map[from] = to;
    }
    if (tid == 0) {
        l.count[0] = highs;
        l.count[1] = live;
    }
}

// One chunk of a page's codes in one layer, and with the first chunk its scales.
__device__ void copy_chunk(const mrl_kv_cache& c, uint32_t layer, int from, int to, size_t chunk) {
    const size_t bytes = page_bytes(c), at = chunk * kCopyChunk;
    const uint4* src = reinterpret_cast<const uint4*>(c.codes + block_index(c, layer, from, 0, 0) * block_bytes(c) + at);
    uint4* dst = reinterpret_cast<uint4*>(c.codes + block_index(c, layer, to, 0, 0) * block_bytes(c) + at);
    const int vecs = (int)(min(kCopyChunk, bytes - at) / 16);
    uint4 x[kCopyVec];
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i) {
        const int j = (int)threadIdx.x + i * kCopyThreads;
        if (j < vecs) x[i] = src[j];
    }
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i) {
        const int j = (int)threadIdx.x + i * kCopyThreads;
        if (j < vecs) dst[j] = x[i];
    }
    if (chunk == 0)
        for (int i = (int)threadIdx.x; i < 2 * (int)c.kv_heads; i += kCopyThreads)
            c.scales[block_index(c, layer, to, 0, 0) + i] = c.scales[block_index(c, layer, from, 0, 0) + i];
}

// Copies of `pairs` pages over all layers, the units `first`, `first + step`, ...
__device__ void copy_pairs(const mrl_kv_cache& c, const int* src, const int* dst, int pairs, long long first, long long step) {
    const long long chunks = (long long)((page_bytes(c) + kCopyChunk - 1) / kCopyChunk);
    const long long per_pair = chunks * c.layers;
    for (long long u = first; u < pairs * per_pair; u += step) {
        const int i = (int)(u / per_pair);
        const long long rest = u % per_pair;
        const int from = src[i], to = dst[i];
        if (from == to || !in_range(from, c.pages) || !in_range(to, c.pages)) continue;
        copy_chunk(c, (uint32_t)(rest / chunks), from, to, (size_t)(rest % chunks));
    }
}

// Tail pages, then the children's rows: full pages shared, the tail the child's own.
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(mrl_kv_cache c, const int32_t* parents, const int32_t* children, int n, Lists l) {
    grid_wait();
    const int tails = l.count[0];
    if (tails < 0) return;
    copy_pairs(c, l.a, l.b, tails, blockIdx.x, gridDim.x);
    for (int i = (int)(gridDim.x - 1 - blockIdx.x); i < n; i += (int)gridDim.x) {
        const int ch = children[i], len = c.lens[ch], full = len / kPage;
        const int32_t* from = c.tables + (size_t)parents[i] * c.max_pages;
        int32_t* to = c.tables + (size_t)ch * c.max_pages;
        for (int p = (int)threadIdx.x; p < full; p += kCopyThreads) {
            const int page = from[p];
            to[p] = page;
            if (in_range(page, c.pages)) atomicAdd(&c.refs[page], 1);
        }
        if (threadIdx.x == 0 && len % kPage) {
            const int next = i + 1 < n ? l.off[i + 1] : tails;
            to[full] = next > l.off[i] ? l.b[l.off[i]] : -1;
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(mrl_kv_cache c, Lists l) {
    grid_wait();
    const int moved = l.count[0], live = l.count[1];
    if (moved == 0) return;
    copy_pairs(c, l.a, l.b, moved, blockIdx.x, gridDim.x);
    for (int s = (int)(gridDim.x - 1 - blockIdx.x); s < (int)c.max_seqs; s += (int)gridDim.x) {
        int32_t* row = c.tables + (size_t)s * c.max_pages;
        const int used = min(pages_of(max(c.lens[s], 0)), (int)c.max_pages);
        for (int p = (int)threadIdx.x; p < used; p += kCopyThreads) {
            const int page = row[p];
            if (page >= live && page < (int)c.pages) row[p] = l.map[page];
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(mrl_kv_cache c, const int32_t* src, const int32_t* dst, int n) {
    if (blockIdx.x == 0)
        for (int i = (int)threadIdx.x; i < n; i += kCopyThreads)
            if (!in_range(src[i], c.pages) || !in_range(dst[i], c.pages)) atomicOr(c.status, MRL_KV_BAD_INDEX);
    copy_pairs(c, src, dst, n, blockIdx.x, gridDim.x);
}

// Release (window 0) or trim: one warp per sequence. Entries are exchanged, so a page is given back once
// even where a sequence is listed twice.
__global__ void __launch_bounds__(256) release_kernel(mrl_kv_cache c, const int32_t* seqs, int n, int window, int sinks) {
    const int i = (int)(blockIdx.x * 8 + (threadIdx.x >> 5)), lane = (int)threadIdx.x & 31;
    if (i >= n) return;
    const int s = seqs[i];
    if (!in_range(s, c.max_seqs)) {
        if (lane == 0) atomicOr(c.status, MRL_KV_BAD_INDEX);
        return;
    }
    const int len = max(c.lens[s], 0);
    int from = 0, to = min(pages_of(len), (int)c.max_pages);
    if (window > 0) {  // keys below len - window + 1 are seen by no later query, the first `sinks` excepted
        from = sinks / kPage + (sinks % kPage != 0);
        to = min(to, len - window + 1 > 0 ? (len - window + 1) / kPage : 0);
    }
    int32_t* row = c.tables + (size_t)s * c.max_pages;
    for (int p = from + lane; p < to; p += 32) {
        const int page = atomicExch(&row[p], -1);
        if (in_range(page, c.pages)) atomicSub(&c.refs[page], 1);
    }
    if (window == 0 && lane == 0) c.lens[s] = 0;
}

Lists lists_at(const mrl_kv_cache& c, void* scratch) {
    int* p = static_cast<int*>(scratch);
    Lists l;
    l.count = p;
    l.a = p + 4;
    l.b = l.a + c.pages;
    l.map = l.b + c.pages;
    l.off = l.map + c.pages;
    return l;
}

template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), int grid, int threads, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
}  // namespace kv

size_t kv_list_bytes(const mrl_kv_cache& c, uint32_t n) { return sizeof(int) * (4 + 3 * (size_t)c.pages + n); }

int launch_kv_reserve(const mrl_kv_cache& c, const int32_t* seqs, const int32_t* add, uint32_t n, void* scratch, cudaStream_t s) {
    kv::reserve_kernel<<<1, kv::kPlanThreads, 0, s>>>(c, seqs, add, (int)n, kv::lists_at(c, scratch));
    return (int)cudaGetLastError();
}

int launch_kv_fork(const mrl_kv_cache& c, const int32_t* parents, const int32_t* children, uint32_t n, int sms, void* scratch,
                   cudaStream_t s) {
    const kv::Lists l = kv::lists_at(c, scratch);
    kv::fork_plan_kernel<<<1, kv::kPlanThreads, 0, s>>>(c, parents, children, (int)n, l);
    if (const cudaError_t e = cudaGetLastError()) return (int)e;
    return (int)kv::launch_after(kv::fork_apply_kernel, sms * 4, kv::kCopyThreads, s, c, parents, children, (int)n, l);
}

int launch_kv_release(const mrl_kv_cache& c, const int32_t* seqs, uint32_t n, uint32_t trim, uint32_t window, uint32_t sinks,
                      cudaStream_t s) {
    kv::release_kernel<<<(n + 7) / 8, 256, 0, s>>>(c, seqs, (int)n, trim ? (int)window : 0, (int)sinks);
    return (int)cudaGetLastError();
}

int launch_kv_compact(const mrl_kv_cache& c, int sms, void* scratch, cudaStream_t s) {
    const kv::Lists l = kv::lists_at(c, scratch);
    kv::compact_plan_kernel<<<1, kv::kPlanThreads, 0, s>>>(c, l);
    if (const cudaError_t e = cudaGetLastError()) return (int)e;
    return (int)kv::launch_after(kv::compact_apply_kernel, sms * 4, kv::kCopyThreads, s, c, l);
}

int launch_kv_copy_pages(const mrl_kv_cache& c, const int32_t* src, const int32_t* dst, uint32_t n, int sms, cudaStream_t s) {
    kv::copy_pages_kernel<<<sms * 4, kv::kCopyThreads, 0, s>>>(c, src, dst, (int)n);
    return (int)cudaGetLastError();
}

}  // namespace mrl
