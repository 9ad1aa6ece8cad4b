// ctx.cuh — the context behind the C ABI (include/mrl_cuda.h) and the helpers its entry points share:
// error reporting, the device guard and grow-only buffers. Host-side C++.
#pragma once

#include <cstdint>
#include <deque>
#include <string>
#include <vector>

#include "mrl_internal.cuh"

// Scratch of the paged-cache and attention entry points on one stream (include/mrl_kv.h): calls on
// different streams never share a buffer.
struct mrl_kv_block {
    void* p = nullptr;
    size_t bytes = 0;
    bool captured = false;  // a graph holds the address
};
struct mrl_kv_scratch {
    cudaStream_t stream = nullptr;
    uint64_t last = 0;   // the context's call that used it last
    mrl_kv_block work;   // counters and working memory
    mrl_kv_block image;  // 16-bit image of a layer's pool
};

struct mrl_ctx {
    int device = 0;
    int sms = 0;
    cudaStream_t own_stream = nullptr;
    cudaStream_t stream = nullptr;
    std::string err;
    // scan scratch, kScratchSets sets used by consecutive scan launches in turn: launches on the
    // stream may overlap (programmatic dependent launch), and a launch touches its set only once the
    // launch that used it before has released it. Per set: per-CTA lists, control words, per-page
    // owner (grow-only; each set owns an equal share of `owner`).
    unsigned long long* cta_keys = nullptr;  // per set 2 * sms * 32: scan keys, then their exact keys
    unsigned int* ctl = nullptr;             // per set mrl::kCtlWords
    uint8_t* owner = nullptr;
    size_t owner_bytes = 0;
    uint32_t scan_seq = 0;      // launches so far; launch s uses scratch set s % kScratchSets
    uint32_t scan_ctas = 0;     // CTAs per single-query scan launch (0: one per SM)
    unsigned int* done = nullptr;  // per set: sequence number of the last launch that released it
    uint32_t list_len_override = 0;
    // grow-only scratch for host-facing calls: inputs (queries, rows, means) and outputs
    void* tmp = nullptr;
    size_t tmp_bytes = 0;
    void* tmp_out = nullptr;
    size_t tmp_out_bytes = 0;
    // device copy of the last codec centres uploaded (64 prefix + 128 mid floats) and its host
    // twin, so repeated plan builds against one EdenFit issue no host->device copy
    float* d_means = nullptr;
    float h_means[192];
    bool means_valid = false;
    // grow-only scratch of the exact paths (scores, flag)
    void* xbuf = nullptr;
    size_t xbuf_bytes = 0;
    // two merge records (scan, ring) of mrl_engine_scan
    void* ebuf = nullptr;
    size_t ebuf_bytes = 0;
    // per-(query, CTA) top lists and tensor-core operand tiles of the batched scan
    void* bbuf = nullptr;
    size_t bbuf_bytes = 0;
    uint32_t batch_engine = MRL_BATCH_TENSOR;
    // pinned host staging of mrl_query_scan, mapped into the device's address space: the query is
    // copied to the device from here, and the scan kernel stores its results straight into it
    // (no device-to-host copies on the query path)
    void* h_io = nullptr;
    void* h_io_dev = nullptr;
    size_t h_io_bytes = 0;
    // pipelined host queries (mrl_query_submit / mrl_query_collect): MRL_MAX_INFLIGHT result slots
    // in pinned, device-mapped memory, laid out for shortlists up to slot_k; the scan stores each
    // query's top-k there and then the slot's completion word, on which the host waits
    unsigned char* h_slots = nullptr;
    unsigned char* d_slots = nullptr;
    size_t slot_stride = 0;
    uint32_t slot_k = 0;
    uint32_t slot_seq[MRL_MAX_INFLIGHT] = {};
    bool slot_busy[MRL_MAX_INFLIGHT] = {};
    // paged cache and attention (kv_capi.cu): scratch per stream, blocks that were outgrown but are held by captured
    // graphs, and the event that orders a torch stream with the context's
    static constexpr size_t kKvStreams = 32;  // that scratch is kept for beside those of captured graphs
    std::deque<mrl_kv_scratch> kv;
    uint64_t kv_calls = 0;
    std::vector<void*> kv_kept;
    cudaEvent_t join_event = nullptr;
};

inline int fail(mrl_ctx* ctx, int code, const std::string& msg) {
    if (ctx) ctx->err = msg;
    // the runtime keeps a failed call's error for the next cudaGetLastError, which a later launch would report as its own
    if (code == MRL_ERR_CUDA || code == MRL_ERR_NOMEM) (void)cudaGetLastError();
    return code;
}

inline int cuda_fail(mrl_ctx* ctx, cudaError_t e, const char* what) {
    return fail(ctx, MRL_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

#define MRL_CUDA_TRY(ctx, expr)                                   \
    do {                                                          \
        cudaError_t _e = (expr);                                  \
        if (_e != cudaSuccess) return cuda_fail((ctx), _e, #expr); \
    } while (0)

inline int set_device(mrl_ctx* ctx) {
    const cudaError_t e = cudaSetDevice(ctx->device);
    return e == cudaSuccess ? MRL_OK : cuda_fail(ctx, e, "cudaSetDevice");
}

inline int ensure_buf(mrl_ctx* ctx, void** buf, size_t* have, size_t bytes) {
    if (*have >= bytes) return MRL_OK;
    if (*buf) cudaFree(*buf);  // synchronises the device: no launch still reads the old buffer
    *buf = nullptr;
    *have = 0;
    const cudaError_t e = cudaMalloc(buf, bytes);
    if (e != cudaSuccess) return fail(ctx, MRL_ERR_NOMEM, std::string("cudaMalloc scratch: ") + cudaGetErrorString(e));
    *have = bytes;
    return MRL_OK;
}
