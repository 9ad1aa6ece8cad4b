/*
 * mrl_kv.h — C ABI of the attention operators of libmrl_b200.so: a paged key/value cache held in 8
 * bits (reserve, append, fork, release, trim, copy, compact, read), attention over it, and attention
 * with a sliding window and sink tokens over ragged 16-bit inputs. They stand for the embedder beside
 * the reference's scan (its transformer forward, prefix KV cache and ragged prefill,
 * src/gemma_embed.rs), and for a reader of the passages that the scan finds.
 *
 * Conventions of mrl_cuda.h hold: int status, never an abort or an exception across the boundary,
 * mrl_last_error for the message, every call asynchronous on the context's stream. All buffers are
 * device memory owned by the caller. Index arrays (sequences, offsets, tables) live on the device, so
 * what only their contents can show is checked there: an index out of range is never followed, and the
 * page operations set a bit of *status and change nothing.
 *
 * Scratch. A context keeps scratch for each stream that these calls were made on, until it is
 * destroyed: about 20 MiB, more for pools of millions of pages, and for mrl_kv_attend of many rows
 * twice the size of one layer's codes. It grows on demand, and a call that makes it grow allocates
 * device memory and may wait for the device; so does the first call on a stream past 32, which takes
 * over what another stream has not used for longest. The others do not synchronise. During a stream capture
 * nothing can grow: such a call is refused, so make a call of the same size on the stream before the
 * capture. A captured graph goes on using the scratch of the stream it was captured on, which stays
 * where it is whatever is called later: replay it on that stream, or where nothing else runs on that
 * stream's scratch (its calls and the other graphs captured on it) at the same time. Destroy the
 * context after the graphs, and a stream only when its work is done.
 *
 * Outputs may not overlap inputs.
 */
#ifndef MRL_KV_H
#define MRL_KV_H

#include "mrl_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MRL_KV_PAGE 64u /* tokens per page */

#define MRL_F16 0u
#define MRL_BF16 1u
#define MRL_F32 2u /* mrl_kv_read outputs only */

/* Bits of mrl_kv_cache.status, set by the device and cleared by the caller. */
#define MRL_KV_NO_PAGES 1u   /* a reserve or fork needed more free pages than there are; it did nothing */
#define MRL_KV_ROW_FULL 2u   /* a reserve needed more than max_pages pages for a sequence; it did nothing */
#define MRL_KV_BAD_INDEX 4u  /* a sequence, page or count out of range, a fork of an empty sequence, onto one that is
                                not empty or onto its own parent, or attention with row offsets that decrease; the
                                operation did nothing (attention: for the 512 or 1,024 sequences around them). Also
                                rows of an unknown sequence, or more rows than it has tokens, in an append, a
                                read or an attention over the cache, and appended rows whose page is missing: those
                                are not stored, read as 0, or see no key, and the others are as they should be */
#define MRL_KV_NONFINITE 8u  /* an append met an Inf (stored as the largest code) or a NaN (stored as 0) */
#define MRL_KV_TIMEOUT 16u   /* a kernel gave up waiting for its own loads; the call's outputs mean nothing */

/* A cache of `layers` layers over one page table. Page p of a layer holds 64 consecutive tokens of a
 * sequence for all heads; K and V of each head have one f32 scale per page: value = code * scale.
 *   codes   int8  [layers][pages][2 (K, V)][kv_heads][64 * head_dim]; within a head, K is
 *                 [head_dim / 64][64 tokens][64 dims] and V is [head_dim][64 tokens]: in each the index
 *                 that its product sums over is contiguous, in rows of 64 bytes
 *   scales  f32   [layers][pages][2][kv_heads]
 *   tables  int32 [max_seqs][max_pages]: page of tokens 64 i .. 64 i + 63, -1 where there is none
 *   lens    int32 [max_seqs]: tokens of each sequence
 *   refs    int32 [pages]: sequences that hold the page (0: free)
 *   status  uint32[1]: MRL_KV_* bits
 * head_dim is 64, 128 or 256. codes must be 16-byte aligned. A new cache has tables -1 and lens,
 * refs and status 0. Where a table entry of a visible key is not a page, the key counts as not
 * visible. */
typedef struct mrl_kv_cache {
    int8_t* codes;
    float* scales;
    int32_t* tables;
    int32_t* lens;
    int32_t* refs;
    uint32_t* status;
    uint32_t layers, pages, kv_heads, head_dim, max_seqs, max_pages;
} mrl_kv_cache;

/* ---- pages: bookkeeping on the device, deterministic ------------------------------------------ */
/* d_seqs lists `n` distinct sequences. Free pages are taken lowest index first, in the order of the
 * list and of each sequence's pages. */
/* Extend sequence d_seqs[i] by d_add[i] >= 0 tokens: lens grow at once and the pages the new tokens
 * need are taken; their contents come with the mrl_kv_append of each layer. */
int mrl_kv_reserve(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, const int32_t* d_add, uint32_t n);
/* Make the empty sequence d_children[i] a copy of d_parents[i] (parents may repeat; no child may be a
 * parent): full pages are shared (refs + 1), a partly filled last page is copied, all layers, into a
 * page of the child's own, so both can be appended to. */
int mrl_kv_fork(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_parents, const int32_t* d_children, uint32_t n);
/* Drop the sequences: refs - 1 on each of their pages, table rows -1, lens 0. */
int mrl_kv_release(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, uint32_t n);
/* Drop the pages of each sequence that no later query sees through `window` (>= 1) and `sinks`:
 * those holding neither one of the first `sinks` tokens nor a token >= len - window + 1. */
int mrl_kv_trim(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_seqs, uint32_t n, uint32_t window, uint32_t sinks);
/* Move pages so that the L held ones are pages 0 .. L-1: the i-th free page below L receives the i-th
 * held page at or above L, all layers; tables and refs follow. */
int mrl_kv_compact(mrl_ctx* ctx, const mrl_kv_cache* kv);
/* Copy the contents (all layers, codes and scales) of page d_src[i] to page d_dst[i]. The
 * destinations are distinct and none of them is a source. Tables and refs do not change. */
int mrl_kv_copy_pages(mrl_ctx* ctx, const mrl_kv_cache* kv, const int32_t* d_src, const int32_t* d_dst, uint32_t n);

/* ---- tokens ----------------------------------------------------------------------------------- */
/* Rows of a call over `n_seqs` sequences: sequence d_seqs[b] owns rows d_cu[b] .. d_cu[b+1] - 1
 * (int32 [n_seqs + 1], not decreasing, from 0 to n_tokens); d_cu NULL means one row per sequence
 * (n_tokens == n_seqs). The rows of a sequence are its last ones: row r of m is at position
 * len - m + r. Row and head strides are in elements and a head's head_dim elements are contiguous;
 * pointers and strides are multiples of 16 bytes. */
/* Quantise new K/V rows (f16 or bf16) into `layer`, after mrl_kv_reserve made room. Per page, head
 * and K or V, with a the largest finite magnitude of the page's new values: a page without older
 * tokens gets scale a * (1/127); otherwise the old scale s stays where a <= 127 s, else it becomes
 * max(a * (1/127), 2 s) and the older codes are rounded to it (it at least doubles, so all such
 * roundings of a code together stay below one step). code = clamp(rint(x / scale), -127, 127), NaN
 * and scale 0 give 0. Rows whose page or sequence is missing are not stored (MRL_KV_BAD_INDEX). */
int mrl_kv_append(mrl_ctx* ctx, const mrl_kv_cache* kv, uint32_t layer, uint32_t dtype, const void* k, int64_t k_row,
                  int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int32_t* d_seqs,
                  const int32_t* d_cu, uint32_t n_seqs, uint32_t n_tokens);
/* The values the cache holds for those rows, into contiguous [n_tokens][kv_heads][head_dim] outputs of
 * dtype MRL_F16, MRL_BF16 or MRL_F32 (code * scale in f32, rounded once). Rows whose page
 * or sequence is missing are 0; where it is the sequence, MRL_KV_BAD_INDEX is set. */
int mrl_kv_read(mrl_ctx* ctx, const mrl_kv_cache* kv, uint32_t layer, uint32_t dtype, void* k, void* v,
                const int32_t* d_seqs, const int32_t* d_cu, uint32_t n_seqs, uint32_t n_tokens);

/* ---- attention -------------------------------------------------------------------------------- */
/* Query i at position p sees key j where j <= p (unless `causal` is 0) and, with window > 0, also
 * |p - j| < window or j < sinks. s = scale * q . k, o = sum softmax(s) v, lse = ln sum exp(s). A row
 * that sees no key gives o = 0 and lse = -inf. Query head h reads kv head h / (q_heads / kv_heads). */
typedef struct mrl_attn {
    const void* q;
    const void* k; /* mrl_window_attention only */
    const void* v;
    void* out;
    float* lse; /* [n_tokens][q_heads], or NULL */
    const int32_t* seqs; /* mrl_kv_attend only */
    const int32_t* cu;
    uint32_t* status; /* mrl_window_attention: receives MRL_KV_TIMEOUT and MRL_KV_BAD_INDEX, or NULL (mrl_kv_attend
                         reports to the cache's) */
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    uint32_t n_seqs, n_tokens, max_rows; /* max_rows: at least the rows of every sequence */
    uint32_t q_heads, kv_heads, head_dim, dtype;
    uint32_t causal, window, sinks;
    float scale;
    uint32_t layer; /* mrl_kv_attend only */
} mrl_attn;
/* Attention of the last rows of sequences over the cache (always causal; k, v, kv_heads, head_dim
 * and causal of `a` are not read). Rows of an unknown sequence, and rows beyond a sequence's tokens, see no
 * key, and MRL_KV_BAD_INDEX is set. Softmax statistics and sums in f32. Any max_rows is right; it
 * helps to choose the kernel: calls of few rows read the pages as codes; calls of many widen them first, into
 * scratch of twice the size of a layer's codes, or read the codes too where the device has no room for it. Work of the former is counted in 32 bits: (n_tokens x group
 * / 16 + n_seqs) x kv_heads x (max_pages + 16), per 1024 sequences where cu is NULL, must stay below 2^32. */
int mrl_kv_attend(mrl_ctx* ctx, const mrl_kv_cache* kv, const mrl_attn* a);
/* Self-attention over ragged packed rows: sequence b's q, k and v rows are cu[b] .. cu[b+1] - 1 and
 * positions count from its first row. Rows of other sequences, and keys a query does not see, do not
 * reach its result, whatever they hold (Inf and NaN included). A row that meets an Inf or NaN among the
 * values of v of a key that it does not see is computed again from its visible keys, after all others:
 * about 2 ms for the rows that one such key in 8,192 causal ones of 16 heads of 128 reaches. */
int mrl_window_attention(mrl_ctx* ctx, const mrl_attn* a);

/* Order the context's stream after the work queued on `stream` so far (to_ctx != 0), or `stream`
 * after the context's (to_ctx == 0). Nothing to do where they are the same stream. */
int mrl_ctx_join(mrl_ctx* ctx, void* stream, int to_ctx);

#ifdef __cplusplus
}
#endif
#endif /* MRL_KV_H */
