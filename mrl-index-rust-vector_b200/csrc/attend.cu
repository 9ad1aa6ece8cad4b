// attend.cu — attention over the paged 8-bit cache and over ragged 16-bit rows (include/mrl_kv.h).
//
// One warp per query row: the running maximum m and sum l of the softmax and the output are kept in
// registers while the visible keys pass once (o and l are scaled by exp(m_old - m) when m grows).
#include "kv.cuh"

namespace mrl {
namespace kv {
namespace {

template <class T, int D, bool PAGED> __global__ void __launch_bounds__(256) rows_kernel(mrl_kv_cache c, mrl_attn a) {
    constexpr int E = D / 32;
    const int lane = (int)threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = (int)(w / a.q_heads), h = (int)(w % a.q_heads);
    if (t >= (int)a.n_tokens) return;
    const Rows r{a.seqs, a.cu, (int)a.n_seqs, (int)a.n_tokens};
    int b = t;
    if (r.cu) b = warp_find(r.n, t, [&](int i) { return (long long)r.begin(i); });
    const int lo_row = r.begin(b), m_rows = r.end(b) - lo_row;
    const int kvh = h / (int)(a.q_heads / (PAGED ? c.kv_heads : a.kv_heads));
    int seq = 0, n = m_rows;
    if (PAGED) {
        seq = a.seqs[b];
        n = seq >= 0 && seq < (int)c.max_seqs ? min(max(c.lens[seq], 0), (int)c.max_pages * kPage) : 0;
    }
    const int p = n - m_rows + t - lo_row;
    const bool in = t >= lo_row && t - lo_row < m_rows;
    const Span span = in ? visible(p, n, PAGED ? 1 : (int)a.causal, (int)a.window, (int)a.sinks) : Span{0, 0, 0};
    float q[E], o[E];
    const T* qp = static_cast<const T*>(a.q) + (int64_t)t * a.q_row + (int64_t)h * a.q_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = to_f32<T>(qp[e]);
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    auto key = [&](int j) {
        float k[E], v[E];
        if (PAGED) {
            const int page = c.tables[(size_t)seq * c.max_pages + j / kPage], slot = j % kPage;
            if (page < 0 || page >= (int)c.pages) return;
            const size_t kb = block_index(c, a.layer, page, 0, kvh), vb = block_index(c, a.layer, page, 1, kvh);
            const int8_t *kc = c.codes + kb * (size_t)(kPage * D), *vc = c.codes + vb * (size_t)(kPage * D);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = lane * E + e;
                k[e] = (float)kc[(d / 64) * (kPage * 64) + slot * 64 + d % 64] * c.scales[kb];
                v[e] = (float)vc[d * kPage + slot] * c.scales[vb];
            }
        } else {
            const T* kp = static_cast<const T*>(a.k) + (int64_t)(lo_row + j) * a.k_row + (int64_t)kvh * a.k_head + lane * E;
            const T* vp = static_cast<const T*>(a.v) + (int64_t)(lo_row + j) * a.v_row + (int64_t)kvh * a.v_head + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                k[e] = to_f32<T>(kp[e]);
                v[e] = to_f32<T>(vp[e]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        s *= a.scale;
        const float top = fmaxf(m, s);
        const float keep = m == top ? 1.0f : expf(m - top), add = s == top ? 1.0f : expf(s - top);
        m = top;
        l = fmaf(l, keep, add);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], keep, add * v[e]);
    };
    for (int j = 0; j < span.head; ++j) key(j);
    for (int j = span.lo; j < span.hi; ++j) key(j);
    T* op = static_cast<T*>(a.out) + (int64_t)t * a.o_row + (int64_t)h * a.o_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) op[e] = from_f32<T>(l == 0.0f ? 0.0f : o[e] / l);
    if (a.lse && lane == 0) a.lse[(size_t)t * a.q_heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

template <class T, int D> void rows_launch(const mrl_kv_cache* c, const mrl_attn& a, cudaStream_t s) {
    const long long warps = (long long)a.n_tokens * a.q_heads;
    const unsigned grid = (unsigned)((warps + 7) / 8);
    if (c) rows_kernel<T, D, true><<<grid, 256, 0, s>>>(*c, a);
    else rows_kernel<T, D, false><<<grid, 256, 0, s>>>(mrl_kv_cache{}, a);
}

}  // namespace
}  // namespace kv

int launch_attend_simple(const mrl_kv_cache* c, const mrl_attn& a, cudaStream_t s) {
    const uint32_t d = c ? c->head_dim : a.head_dim;
    if (a.dtype == MRL_F16) {
        if (d == 64) kv::rows_launch<__half, 64>(c, a, s);
        else if (d == 128) kv::rows_launch<__half, 128>(c, a, s);
        else kv::rows_launch<__half, 256>(c, a, s);
    } else {
        if (d == 64) kv::rows_launch<__nv_bfloat16, 64>(c, a, s);
        else if (d == 128) kv::rows_launch<__nv_bfloat16, 128>(c, a, s);
        else kv::rows_launch<__nv_bfloat16, 256>(c, a, s);
    }
    return (int)cudaGetLastError();
}

}  // namespace mrl
