// kv_capi.cu — C ABI of the paged cache and the attention operators (include/mrl_kv.h): argument checks,
// scratch and launches. Every entry point catches its own failures, as in capi.cu.
#include <algorithm>
#include <cmath>
#include <exception>

#include "ctx.cuh"
#include "kv.cuh"

namespace {

template <class F> int guarded(mrl_ctx* ctx, F f) {
    if (!ctx) return MRL_ERR_INVALID;
    try {
        if (int rc = set_device(ctx)) return rc;
        return f();
    } catch (const std::exception&) {  // std::bad_alloc of a message
        return MRL_ERR_NOMEM;
    }
}

int bad(mrl_ctx* ctx, const char* msg) { return fail(ctx, MRL_ERR_INVALID, msg); }
int done(mrl_ctx* ctx, int cuda, const char* what) {
    return cuda == 0 ? MRL_OK : cuda_fail(ctx, (cudaError_t)cuda, what);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_cache(mrl_ctx* ctx, const mrl_kv_cache* c) {
    if (!c) return bad(ctx, "kv is NULL");
    if (!c->codes || !c->scales || !c->tables || !c->lens || !c->refs || !c->status) return bad(ctx, "kv has a NULL buffer");
    if (!aligned(c->codes)) return bad(ctx, "kv codes must be 16-byte aligned");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return bad(ctx, "head_dim must be 64, 128 or 256");
    if (c->layers < 1 || c->layers > 4096) return bad(ctx, "layers must be in [1, 4096]");
    if (c->kv_heads < 1 || c->kv_heads > 1024) return bad(ctx, "kv_heads must be in [1, 1024]");
    if (c->pages < 1 || c->pages > (1u << 24)) return bad(ctx, "pages must be in [1, 2^24]");
    if (c->max_pages < 1 || c->max_pages > (1u << 20)) return bad(ctx, "max_pages must be in [1, 2^20]");
    if (c->max_seqs < 1 || c->max_seqs > (1u << 24)) return bad(ctx, "max_seqs must be in [1, 2^24]");
    return MRL_OK;
}

constexpr uint32_t kMaxSeqs = 65535, kMaxTokens = 1u << 28;

int check_rows(mrl_ctx* ctx, const int32_t* seqs, bool need_seqs, const int32_t* cu, uint32_t n_seqs, uint32_t n_tokens) {
    if (n_seqs > kMaxSeqs) return bad(ctx, "n_seqs must be at most 65535");
    if (n_tokens > kMaxTokens) return bad(ctx, "n_tokens must be at most 2^28");
    if (n_seqs && need_seqs && !seqs) return bad(ctx, "seqs is NULL");
    if (!cu && n_tokens != n_seqs) return bad(ctx, "without cu there is one row per sequence: n_tokens must equal n_seqs");
    return MRL_OK;
}

// A [rows][heads][dims] operand of 16-bit elements: 16-byte aligned pointer and strides.
int check_rows16(mrl_ctx* ctx, const char* name, const void* p, int64_t row, int64_t head) {
    if (!p) return fail(ctx, MRL_ERR_INVALID, std::string(name) + " is NULL");
    if (!aligned(p) || row % 8 || head % 8)
        return fail(ctx, MRL_ERR_INVALID, std::string(name) + " and its row and head strides must be multiples of 16 bytes");
    if (row < 0 || head < 0) return fail(ctx, MRL_ERR_INVALID, std::string(name) + " strides must not be negative");
    return MRL_OK;
}

bool capturing(const mrl_ctx* ctx) {
    cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(ctx->stream, &s) != cudaSuccess) (void)cudaGetLastError();  // the launch will say so
    return s != cudaStreamCaptureStatusNone;
}
int no_growth(mrl_ctx* ctx) { return bad(ctx, "scratch cannot grow during a stream capture: make a call of this size on the stream before it"); }

// The scratch of the context's current stream, made by the first call on it. Past kKvStreams streams the one unused for longest
// is taken over, when the device has finished, so that streams that come and go do not add up; one that a captured graph
// may use is never handed on.
int kv_stream(mrl_ctx* ctx, mrl_kv_scratch** out) {
    mrl_kv_scratch *k = nullptr, *oldest = nullptr;
    size_t free_ones = 0;
    for (mrl_kv_scratch& x : ctx->kv) {
        if (x.stream == ctx->stream) k = &x;
        if (x.work.captured || x.image.captured) continue;
        ++free_ones;
        if (!oldest || x.last < oldest->last) oldest = &x;
    }
    if (!k) {
        if (capturing(ctx)) return no_growth(ctx);
        if (free_ones < mrl_ctx::kKvStreams) {
            ctx->kv.emplace_back();
            k = &ctx->kv.back();
        } else {
            MRL_CUDA_TRY(ctx, cudaDeviceSynchronize());
            k = oldest;
        }
        k->stream = ctx->stream;
    }
    k->last = ++ctx->kv_calls;
    *out = k;
    return MRL_OK;
}

// At least `bytes` in a block of the scratch, zero when they are made. A block whose address a captured graph may hold
// is kept beside its successor; another one is freed, which waits for the device.
int kv_grow(mrl_ctx* ctx, mrl_kv_block* b, size_t bytes) {
    const bool capture = capturing(ctx);
    if (b->bytes < bytes) {
        if (capture) return no_growth(ctx);
        if (b->captured) {
            ctx->kv_kept.push_back(b->p);
            *b = mrl_kv_block{};
        }
        if (int rc = ensure_buf(ctx, &b->p, &b->bytes, (bytes + (size_t)0xfffff) & ~(size_t)0xfffff)) return rc;
        MRL_CUDA_TRY(ctx, cudaMemsetAsync(b->p, 0, b->bytes, ctx->stream));
    }
    b->captured = b->captured || capture;
    return MRL_OK;
}

// `bytes` of working memory, and counters before it (zero; the kernels that use them leave them zero). From the first
// call there is room for every mrl_kv_attend of few rows.
constexpr size_t kCounterBytes = 65536;
int kv_scratch(mrl_ctx* ctx, size_t bytes, void** out, unsigned** counters = nullptr) {
    mrl_kv_scratch* k;
    if (int rc = kv_stream(ctx, &k)) return rc;
    for (const uint32_t d : {64u, 128u, 256u}) bytes = std::max(bytes, mrl::kv_decode_bytes(d, ctx->sms));
    if (int rc = kv_grow(ctx, &k->work, bytes + kCounterBytes)) return rc;
    *out = static_cast<char*>(k->work.p) + kCounterBytes;
    if (counters) *counters = static_cast<unsigned*>(k->work.p);
    return MRL_OK;
}

// Room for a layer's pool as f16 (launch_attend_tc).
int kv_image(mrl_ctx* ctx, size_t bytes, void** out) {
    mrl_kv_scratch* k;
    if (int rc = kv_stream(ctx, &k)) return rc;
    if (int rc = kv_grow(ctx, &k->image, bytes)) return rc;
    *out = k->image.p;
    return MRL_OK;
}

// Whether mrl_kv_attend widens the pages and runs 128-row tiles (attend_tc.cu) instead of 16-row items on the codes
// (kv_decode.cu). A sequence whose rows are one item reads its pages once either way: always the latter. Else
// the smaller estimate, in ns per 128 keys of every sequence: an item pays for each of its pages, all SMs
// together; a tile pair (a tile, head_dim 256) for each step on its SM, and widening each page once. Measured us,
// items / tiles, 8 kv heads of 128, group 4: 8 sequences of 8,000 with 64 rows 116 / 220, with 128 188 / 224, with
// 256 372 / 228, with 512 706 / 232; one of 30,000 with 512 rows 327 / 549. 64 sequences of 1,000, 8 heads of 64,
// group 2: 64 rows 71 / 135, 128 119 / 137, 256 260 / 148. 8 of 4,000, 2 heads of 256, group 4: 128 rows 88 / 138, 256
// 154 / 134.
bool tensor_cores(const mrl_ctx* ctx, const mrl_kv_cache& kv, const mrl_attn& a) {
    const uint64_t group = a.q_heads / kv.kv_heads, rows = a.n_tokens * group, heads = kv.kv_heads, sms = (uint64_t)ctx->sms;
    if (!a.cu || a.max_rows * group <= 16) return false;
    const uint64_t per_page = kv.head_dim == 64 ? 630 : kv.head_dim == 128 ? 810 : 2600;  // of one SM, for two pages
    const uint64_t per_step = kv.head_dim == 64 ? 1700 : kv.head_dim == 128 ? 2100 : 2700, widen = kv.head_dim * 118ull / 1000;
    const uint64_t items = std::max<uint64_t>(a.n_seqs, rows / 16) * heads;
    const uint64_t tiles = std::max<uint64_t>(a.n_seqs, rows / (kv.head_dim == 256 ? 128 : 256)) * heads;
    return items * per_page / sms > (tiles + sms - 1) / sms * per_step + a.n_seqs * heads * widen;
}

// Windows and sinks beyond any sequence (2^28 rows) all mean the same; cut, sums with positions stay in an int.
mrl_attn cut(const mrl_attn& a) {
    mrl_attn b = a;
    b.window = std::min(b.window, 1u << 30);
    b.sinks = std::min(b.sinks, 1u << 30);
    return b;
}

int check_attn(mrl_ctx* ctx, const mrl_attn* a, uint32_t kv_heads, uint32_t head_dim, bool paged) {
    if (a->dtype != MRL_F16 && a->dtype != MRL_BF16) return bad(ctx, "dtype must be MRL_F16 or MRL_BF16");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return bad(ctx, "head_dim must be 64, 128 or 256");
    if (kv_heads < 1 || kv_heads > 1024) return bad(ctx, "kv_heads must be in [1, 1024]");
    if (a->q_heads < kv_heads || a->q_heads % kv_heads || a->q_heads / kv_heads > 64)
        return bad(ctx, "q_heads must be kv_heads times a whole number, at most 64");
    if (!(a->scale > 0.0f) || !(a->scale < INFINITY)) return bad(ctx, "scale must be positive and finite");
    if (a->window > 0x7fffffffu || a->sinks > 0x7fffffffu) return bad(ctx, "window and sinks must be below 2^31");
    if (int rc = check_rows(ctx, a->seqs, paged, a->cu, a->n_seqs, a->n_tokens)) return rc;
    if (!paged && !a->cu) return bad(ctx, "cu is NULL");
    if (a->n_tokens == 0) return MRL_OK;
    if (a->n_seqs == 0) return bad(ctx, "there are rows but no sequences");
    if (a->max_rows == 0) return bad(ctx, "max_rows must be at least the rows of every sequence");
    if (int rc = check_rows16(ctx, "q", a->q, a->q_row, a->q_head)) return rc;
    if (int rc = check_rows16(ctx, "out", a->out, a->o_row, a->o_head)) return rc;
    if (paged) return MRL_OK;
    if (int rc = check_rows16(ctx, "k", a->k, a->k_row, a->k_head)) return rc;
    return check_rows16(ctx, "v", a->v, a->v_row, a->v_head);
}

}  // namespace

extern "C" {

int mrl_kv_reserve(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, const int32_t* d_add, uint32_t n) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (n > kMaxSeqs) return bad(ctx, "n must be at most 65535");
        if (n == 0) return MRL_OK;
        if (!d_seqs || !d_add) return bad(ctx, "seqs or add is NULL");
        void* scratch;
        if (int rc = kv_scratch(ctx, mrl::kv_list_bytes(*kv, n), &scratch)) return rc;
        return done(ctx, mrl::launch_kv_reserve(*kv, d_seqs, d_add, n, scratch, ctx->stream), "mrl_kv_reserve");
    });
}

int mrl_kv_fork(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_parents, const int32_t* d_children, uint32_t n) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (n > kMaxSeqs) return bad(ctx, "n must be at most 65535");
        if (n == 0) return MRL_OK;
        if (!d_parents || !d_children) return bad(ctx, "parents or children is NULL");
        void* scratch;
        if (int rc = kv_scratch(ctx, mrl::kv_list_bytes(*kv, n), &scratch)) return rc;
        return done(ctx, mrl::launch_kv_fork(*kv, d_parents, d_children, n, ctx->sms, scratch, ctx->stream), "mrl_kv_fork");
    });
}

int mrl_kv_release(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, uint32_t n) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (n > kMaxSeqs) return bad(ctx, "n must be at most 65535");
        if (n == 0) return MRL_OK;
        if (!d_seqs) return bad(ctx, "seqs is NULL");
        return done(ctx, mrl::launch_kv_release(*kv, d_seqs, n, 0, 0, 0, ctx->stream), "mrl_kv_release");
    });
}

int mrl_kv_trim(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, uint32_t n, uint32_t window, uint32_t sinks) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (window < 1 || window > 0x7fffffffu || sinks > 0x7fffffffu) return bad(ctx, "window must be in [1, 2^31) and sinks below 2^31");
        if (n > kMaxSeqs) return bad(ctx, "n must be at most 65535");
        if (n == 0) return MRL_OK;
        if (!d_seqs) return bad(ctx, "seqs is NULL");
        return done(ctx, mrl::launch_kv_release(*kv, d_seqs, n, 1, std::min(window, 1u << 30), std::min(sinks, 1u << 30), ctx->stream), "mrl_kv_trim");
    });
}

int mrl_kv_compact(mrl_ctx* ctx, const mrl_kv_cache* kv) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        void* scratch;
        if (int rc = kv_scratch(ctx, mrl::kv_list_bytes(*kv, 0), &scratch)) return rc;
        return done(ctx, mrl::launch_kv_compact(*kv, ctx->sms, scratch, ctx->stream), "mrl_kv_compact");
    });
}

int mrl_kv_copy_pages(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_src, const int32_t* d_dst, uint32_t n) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (n > kv->pages) return bad(ctx, "n must be at most the cache's pages");
        if (n == 0) return MRL_OK;
        if (!d_src || !d_dst) return bad(ctx, "src or dst is NULL");
        return done(ctx, mrl::launch_kv_copy_pages(*kv, d_src, d_dst, n, ctx->sms, ctx->stream), "mrl_kv_copy_pages");
    });
}

int mrl_kv_append(mrl_ctx* ctx, const mrl_kv_cache* kv, uint32_t layer, uint32_t dtype, const void* k, int64_t k_row,
                  int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int32_t* d_seqs,
                  const int32_t* d_cu, uint32_t n_seqs, uint32_t n_tokens) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (layer >= kv->layers) return bad(ctx, "layer is not one of the cache's");
        if (dtype != MRL_F16 && dtype != MRL_BF16) return bad(ctx, "dtype must be MRL_F16 or MRL_BF16");
        if (int rc = check_rows(ctx, d_seqs, true, d_cu, n_seqs, n_tokens)) return rc;
        if (n_tokens == 0) return MRL_OK;
        if (n_seqs == 0) return bad(ctx, "there are rows but no sequences");
        if (int rc = check_rows16(ctx, "k", k, k_row, k_head)) return rc;
        if (int rc = check_rows16(ctx, "v", v, v_row, v_head)) return rc;
        const mrl::kv::Rows r{d_seqs, d_cu, (int)n_seqs, (int)n_tokens};
        return done(ctx, mrl::launch_kv_append(*kv, layer, dtype, k, k_row, k_head, v, v_row, v_head, r, ctx->stream), "mrl_kv_append");
    });
}

int mrl_kv_read(mrl_ctx* ctx, const mrl_kv_cache* kv, uint32_t layer, uint32_t dtype, void* k, void* v,
                const int32_t* d_seqs, const int32_t* d_cu, uint32_t n_seqs, uint32_t n_tokens) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (layer >= kv->layers) return bad(ctx, "layer is not one of the cache's");
        if (dtype > MRL_F32) return bad(ctx, "dtype must be MRL_F16, MRL_BF16 or MRL_F32");
        if (int rc = check_rows(ctx, d_seqs, true, d_cu, n_seqs, n_tokens)) return rc;
        if (n_tokens == 0) return MRL_OK;
        if (n_seqs == 0) return bad(ctx, "there are rows but no sequences");
        if (!k || !v) return bad(ctx, "k or v is NULL");
        if (!aligned(k) || !aligned(v)) return bad(ctx, "k and v must be 16-byte aligned");
        const mrl::kv::Rows r{d_seqs, d_cu, (int)n_seqs, (int)n_tokens};
        return done(ctx, mrl::launch_kv_read(*kv, layer, dtype, k, v, r, ctx->stream), "mrl_kv_read");
    });
}

int mrl_kv_attend(mrl_ctx* ctx, const mrl_kv_cache* kv, const mrl_attn* a) {
    return guarded(ctx, [&]() -> int {
        if (int rc = check_cache(ctx, kv)) return rc;
        if (!a) return bad(ctx, "args are NULL");
        if (a->layer >= kv->layers) return bad(ctx, "layer is not one of the cache's");
        if (int rc = check_attn(ctx, a, kv->kv_heads, kv->head_dim, true)) return rc;
        if (a->n_tokens == 0) return MRL_OK;
        int no_image = MRL_OK;
        if (tensor_cores(ctx, *kv, *a)) {
            void* wide;
            no_image = kv_image(ctx, mrl::kv_wide_bytes(*kv), &wide);
            if (no_image == MRL_OK) return done(ctx, mrl::launch_attend_tc(kv, cut(*a), ctx->sms, wide, ctx->stream), "mrl_kv_attend");
            if (no_image != MRL_ERR_NOMEM) return no_image;
            // no room for it: the kernel on the codes takes any number of rows
        }
        // the cost of a launch's items (pages and a fixed part of at most 16 each) is summed in 32 bits
        const uint64_t group = a->q_heads / kv->kv_heads, per_launch = std::min(a->n_seqs, mrl::kKvDecodeSeqs);
        const uint64_t tiles = a->cu ? a->n_tokens * group / 16 + per_launch : per_launch * ((group + 15) / 16);
        if (tiles * kv->kv_heads * (kv->max_pages + 16ull) >= (1ull << 32))
            return no_image ? no_image : bad(ctx, "rows x kv_heads x max_pages is too large for one call");
        void* scratch;
        unsigned* counters;
        if (int rc = kv_scratch(ctx, mrl::kv_decode_bytes(kv->head_dim, ctx->sms), &scratch, &counters)) return rc;
        return done(ctx, mrl::launch_kv_decode(*kv, cut(*a), ctx->sms, scratch, counters, ctx->stream), "mrl_kv_attend");
    });
}

int mrl_window_attention(mrl_ctx* ctx, const mrl_attn* a) {
    return guarded(ctx, [&]() -> int {
        if (!a) return bad(ctx, "args are NULL");
        if (int rc = check_attn(ctx, a, a->kv_heads, a->head_dim, false)) return rc;
        if (a->n_tokens == 0) return MRL_OK;
        const int rc = mrl::launch_attend_tc(nullptr, cut(*a), ctx->sms, nullptr, ctx->stream);
        if (rc == mrl::kTcNoMaps) return fail(ctx, MRL_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        if (rc < 0)
            return fail(ctx, MRL_ERR_INVALID, std::string(rc == mrl::kTcBadQ ? "q" : rc == mrl::kTcBadK ? "k" : "v") + " has strides that a tensor map cannot describe");
        return done(ctx, rc, "mrl_window_attention");
    });
}

int mrl_ctx_join(mrl_ctx* ctx, void* stream, int to_ctx) {
    return guarded(ctx, [&]() -> int {
        cudaStream_t other = static_cast<cudaStream_t>(stream);
        if (other == ctx->stream) return MRL_OK;
        if (!ctx->join_event) MRL_CUDA_TRY(ctx, cudaEventCreateWithFlags(&ctx->join_event, cudaEventDisableTiming));
        MRL_CUDA_TRY(ctx, cudaEventRecord(ctx->join_event, to_ctx ? other : ctx->stream));
        MRL_CUDA_TRY(ctx, cudaStreamWaitEvent(to_ctx ? ctx->stream : other, ctx->join_event, 0));
        return MRL_OK;
    });
}

}  // extern "C"
