// kv_append.cu — quantised appends to the paged cache, and reading tokens back (include/mrl_kv.h).
//
// One CTA per touched page, head and K or V: the page's new values are read once into registers, their
// largest magnitude gives the scale, and the codes go out in 4-byte words (a page that already holds
// tokens and whose scale grows has those codes rounded again). K keeps a token's dims together, V a
// dim's tokens, so V turns its tile in shared memory. Bound by HBM: 2 bytes in and 1 out per value.
#include "kv.cuh"

namespace mrl {
namespace kv {
namespace {

constexpr int kThreads = 256;
constexpr float kInv127 = 1.0f / 127.0f;

__device__ __forceinline__ int8_t to_code(float x, float s) {
    // s > 0. fminf / fmaxf drop a NaN, so it is taken out first.
    const float q = rintf(__fdiv_rn(x, s));
    return q != q ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
}
__device__ __forceinline__ uint32_t to_codes4(const float* x, float s) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(uint8_t)(s > 0.0f ? to_code(x[i], s) : (int8_t)0) << (8 * i);
    return w;
}

// 8 values of 16 bits as f32.
template <class T> __device__ __forceinline__ void unpack8(uint4 v, float* x) {
    const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(p[i]);
}

// Tile of 64 tokens x D: thread t holds dims 8 (t % (D/8)) .. + 7 of tokens t / (D/8) + i * (256 / (D/8)).
template <class T, int D> __global__ void __launch_bounds__(kThreads) append_kernel(mrl_kv_cache c, uint32_t layer, const T* k, int64_t k_row, int64_t k_head, const T* v, int64_t v_row, int64_t v_head, Rows r) {
    constexpr int kCols = D / 8, kStep = kThreads / kCols, kTok = kPage / kStep;
    __shared__ PageUnit su;
    __shared__ float smax[kThreads / 32];
    __shared__ uint32_t tile[D * (kPage / 4 + 1)];  // V's codes, a dim's 64 tokens and a padding word
    const int tid = (int)threadIdx.x, head = (int)blockIdx.y, which = (int)blockIdx.z;
    if (tid < 32) {
        const PageUnit u = find_page_unit(c, r, (int)blockIdx.x);
        if (tid == 0) su = u;
    }
    __syncthreads();
    const PageUnit u = su;
    if (u.page < 0 || u.count == 0) return;
    const size_t block = block_index(c, layer, u.page, which, head);
    const float old = c.scales[block];
    const T* src = which ? v + (int64_t)head * v_head : k + (int64_t)head * k_head;
    const int64_t stride = which ? v_row : k_row;
    const int col = tid % kCols, tok0 = tid / kCols;
    uint4 raw[kTok];
    float top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
        const int t = tok0 + i * kStep - u.slot;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (t >= 0 && t < u.count) raw[i] = *reinterpret_cast<const uint4*>(src + (int64_t)(u.row + t) * stride + col * 8);
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
        float x[8];
        unpack8<T>(raw[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float m = fabsf(x[j]);
            if (m < INFINITY) top = fmaxf(top, m);
            else odd = true;
        }
    }
    if (__any_sync(~0u, odd) && (tid & 31) == 0) atomicOr(c.status, MRL_KV_NONFINITE);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if ((tid & 31) == 0) smax[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, smax[i]);
    const bool had = u.slot > 0;
    float s = __fmul_rn(top, kInv127);
    if (had) s = top <= __fmul_rn(127.0f, old) ? old : fmaxf(s, __fmul_rn(2.0f, old));
    uint32_t* out = reinterpret_cast<uint32_t*>(c.codes + block * (size_t)(kPage * D));
    if (had && s > old) {
        // every code of the page: those of slots not yet filled mean nothing
        const float ratio = __fdiv_rn(old, s);
        for (int i = tid; i < kPage * D / 4; i += kThreads) {
            const uint32_t w = out[i];
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float q = rintf(__fmul_rn((float)(int8_t)(w >> (8 * j)), ratio));
                n |= (uint32_t)(uint8_t)(int8_t)(int)q << (8 * j);
            }
            out[i] = n;
        }
        __syncthreads();
    }
    if (tid == 0 && (!had || s > old)) c.scales[block] = s;
    if (which == 0) {
        // [D/64][64 tokens][64 dims]
        uint2* dst = reinterpret_cast<uint2*>(out) + (col / 8) * (kPage * 8) + col % 8;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            const int t = tok0 + i * kStep;
            float x[8];
            unpack8<T>(raw[i], x);
            if (t >= u.slot && t < u.slot + u.count) dst[t * 8] = make_uint2(to_codes4(x, s), to_codes4(x + 4, s));
        }
        return;
    }
    uint8_t* bytes = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
        const int t = tok0 + i * kStep;
        float x[8];
        unpack8<T>(raw[i], x);
        if (t >= u.slot && t < u.slot + u.count) {
            const uint32_t a = to_codes4(x, s), b = to_codes4(x + 4, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) bytes[(col * 8 + j) * (kPage + 4) + t] = (uint8_t)((j < 4 ? a : b) >> (8 * (j & 3)));
        }
    }
    __syncthreads();
    const int lo = u.slot, hi = u.slot + u.count;
    for (int i = tid; i < D * kPage / 4; i += kThreads) {
        const int d = i / (kPage / 4), w = i % (kPage / 4);
        if (4 * w >= lo && 4 * w + 4 <= hi) {
            out[i] = tile[d * (kPage / 4 + 1) + w];
        } else {
            uint8_t* o = reinterpret_cast<uint8_t*>(out + i);
            for (int j = 0; j < 4; ++j)
                if (4 * w + j >= lo && 4 * w + j < hi) o[j] = bytes[d * (kPage + 4) + 4 * w + j];
        }
    }
}

template <class O, int D> __global__ void __launch_bounds__(kThreads) read_kernel(mrl_kv_cache c, uint32_t layer, O* k, O* v, Rows r) {
    __shared__ PageUnit su;
    __shared__ uint32_t tile[D * (kPage / 4 + 1)];
    const int tid = (int)threadIdx.x, head = (int)blockIdx.y, which = (int)blockIdx.z;
    if (tid < 32) {
        const PageUnit u = find_page_unit(c, r, (int)blockIdx.x);
        if (tid == 0) su = u;
    }
    __syncthreads();
    const PageUnit u = su;
    if (u.count == 0) return;
    O* dst = (which ? v : k) + ((size_t)u.row * c.kv_heads + head) * D;
    const size_t stride = (size_t)c.kv_heads * D;
    if (u.page < 0) {
        for (int i = tid; i < u.count * D; i += kThreads) dst[(size_t)(i / D) * stride + i % D] = from_f32<O>(0.0f);
        return;
    }
    const size_t block = block_index(c, layer, u.page, which, head);
    const float s = c.scales[block];
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(c.codes + block * (size_t)(kPage * D));
    const int8_t* from = reinterpret_cast<const int8_t*>(codes);
    if (which) {
        for (int i = tid; i < D * kPage / 4; i += kThreads) tile[(i / (kPage / 4)) * (kPage / 4 + 1) + i % (kPage / 4)] = codes[i];
        __syncthreads();
    }
    const int8_t* turned = reinterpret_cast<const int8_t*>(tile);
    for (int i = tid; i < u.count * D; i += kThreads) {
        const int t = i / D, d = i % D, slot = u.slot + t;
        const int code = which ? turned[d * (kPage + 4) + slot] : from[(d / 64) * (kPage * 64) + slot * 64 + d % 64];
        dst[(size_t)t * stride + d] = from_f32<O>(__fmul_rn((float)code, s));
    }
}

template <class T> cudaError_t append_dims(const mrl_kv_cache& c, uint32_t layer, const void* k, int64_t k_row, int64_t k_head, const void* v,
                                           int64_t v_row, int64_t v_head, const Rows& r, dim3 grid, cudaStream_t s) {
    const T *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v);
    if (c.head_dim == 64) append_kernel<T, 64><<<grid, kThreads, 0, s>>>(c, layer, kp, k_row, k_head, vp, v_row, v_head, r);
    else if (c.head_dim == 128) append_kernel<T, 128><<<grid, kThreads, 0, s>>>(c, layer, kp, k_row, k_head, vp, v_row, v_head, r);
    else append_kernel<T, 256><<<grid, kThreads, 0, s>>>(c, layer, kp, k_row, k_head, vp, v_row, v_head, r);
    return cudaGetLastError();
}

template <class O> cudaError_t read_dims(const mrl_kv_cache& c, uint32_t layer, void* k, void* v, const Rows& r, dim3 grid, cudaStream_t s) {
    O *kp = static_cast<O*>(k), *vp = static_cast<O*>(v);
    if (c.head_dim == 64) read_kernel<O, 64><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r);
    else if (c.head_dim == 128) read_kernel<O, 128><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r);
    else read_kernel<O, 256><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r);
    return cudaGetLastError();
}

}  // namespace
}  // namespace kv

int launch_kv_append(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, const void* k, int64_t k_row, int64_t k_head,
                     const void* v, int64_t v_row, int64_t v_head, const kv::Rows& r, cudaStream_t s) {
    const dim3 grid((unsigned)kv::page_units(r.n, r.tokens, r.cu != nullptr), c.kv_heads, 2);
    return (int)(dtype == MRL_F16 ? kv::append_dims<__half>(c, layer, k, k_row, k_head, v, v_row, v_head, r, grid, s)
                                  : kv::append_dims<__nv_bfloat16>(c, layer, k, k_row, k_head, v, v_row, v_head, r, grid, s));
}

int launch_kv_read(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, void* k, void* v, const kv::Rows& r, cudaStream_t s) {
    const dim3 grid((unsigned)kv::page_units(r.n, r.tokens, r.cu != nullptr), c.kv_heads, 2);
    return (int)(dtype == MRL_F16    ? kv::read_dims<__half>(c, layer, k, v, r, grid, s)
                 : dtype == MRL_BF16 ? kv::read_dims<__nv_bfloat16>(c, layer, k, v, r, grid, s)
                                     : kv::read_dims<float>(c, layer, k, v, r, grid, s));
}

}  // namespace mrl
