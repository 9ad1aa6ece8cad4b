// kv_append.cu — quantised appends to the paged cache, and reading tokens back (include/mrl_kv.h).
//
// A CTA takes one touched page and some blocks of it (a block: K or V of one head). Where the call has at
// most kFew rows in the page, as when every sequence gains one token, each warp takes a block: a lane holds
// the same few dims of every row, the largest magnitude is found by shuffles, and nothing waits for the rest
// of the CTA. Otherwise the whole CTA takes the blocks in turn: the new values are read once into registers,
// their largest magnitude gives the scale, and the codes go out in words. A page that already holds tokens
// and whose scale grows has its codes rounded again. K keeps a token's dims together, V a dim's tokens, so V
// turns its tile in shared memory. Bound by HBM for many rows (2 bytes in and 1 out per value, 1 in and 4 out
// of a read into f32), by the chain of dependent loads (offsets, sequence, length, table, scale) for few. Measured, 8 kv heads
// of 128: 9,298 rows of 9 sequences in 24.7 us (57 MB, 2.3 TB/s: 1,304 CTAs in about two waves, each behind that chain),
// read into f32 in 21.8 us (95 MB, 4.4 TB/s); 256 sequences of one row in 8.7 us, read in 7.0 us. Turning V by words of four
// tokens instead of bytes changed neither.
#include "kv.cuh"

namespace mrl {
namespace kv {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kFew = 4;  // rows of a page that warps take alone
constexpr float kInv127 = 1.0f / 127.0f;

__device__ __forceinline__ int8_t to_code(float x, float s) {
    // s > 0. fminf / fmaxf drop a NaN, so it is taken out first.
    const float q = rintf(__fdiv_rn(x, s));
    return q != q ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
}
// Adding 1.5 * 2^23 rounds to a whole number, half to even, whose two's complement is the low bits.
constexpr float kMagic = 12582912.0f;
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
// Codes of 4 values whose magnitudes are at most 127 s where they are finite; inv = 1 / s, rounded. x * inv is
// within 2.5e-5 of x / s, so it rounds to the same whole number unless it lies that close to a half: there, and
// where it is not finite, the division decides. A division for each value would bound the whole append.
__device__ __forceinline__ uint32_t to_codes4(const float* x, float s, float inv) {
    if (!(s > 0.0f)) return 0;
    float t[4];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = __fmul_rn(x[i], inv);
        t[i] = __fadd_rn(q, kMagic);
        sure = sure && fabsf(__fadd_rn(q, -__fadd_rn(t[i], -kMagic))) < 0.49995f;  // false for NaN
    }
    if (sure) return low_bytes(t[0], t[1], t[2], t[3]);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(uint8_t)to_code(x[i], s) << (8 * i);
    return w;
}
// Codes rounded again to a scale that grew by 1 / ratio.
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio) {
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = __fadd_rn(__fmul_rn((float)(int8_t)(w >> (8 * j)), ratio), kMagic);
    return low_bytes(t[0], t[1], t[2], t[3]);
}
// Largest magnitude among 16-bit values, two to a word, as their bits: Inf and NaN are the largest.
__device__ __forceinline__ uint32_t max_bits(uint32_t m, uint4 v) {
    m = __vmaxu2(__vmaxu2(m, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu));
    return __vmaxu2(m, v.w & 0x7fff7fffu);
}
template <class T> __device__ __forceinline__ float bits_f32(uint32_t m) {
    const unsigned short top = (unsigned short)max(m & 0xffffu, m >> 16);
    return to_f32<T>(*reinterpret_cast<const T*>(&top));
}
// The page's scale: `top` the largest finite new magnitude, `old` its scale where it holds older tokens.
__device__ __forceinline__ float new_scale(float top, bool had, float old) {
    const float s = __fmul_rn(top, kInv127);
    return !had ? s : top <= __fmul_rn(127.0f, old) ? old : fmaxf(s, __fmul_rn(2.0f, old));
}

// 8 values of 16 bits as f32.
template <class T> __device__ __forceinline__ void unpack8(uint4 v, float* x) {
    const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(p[i]);
}
// E values of 16 bits at p (E 2, 4 or 8, aligned to them).
template <class T, int E> __device__ __forceinline__ void load_f32(const T* p, float* x) {
    uint32_t w[E / 2];
    if (E == 2) *reinterpret_cast<uint32_t*>(w) = *reinterpret_cast<const uint32_t*>(p);
    else if (E == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = to_f32<T>(e[i]);
}

// Where K's code of (token, dim) and V's lie in a block.
__device__ __forceinline__ int k_at(int token, int dim) { return (dim / 64) * (kPage * 64) + token * 64 + dim % 64; }
__device__ __forceinline__ int v_at(int token, int dim) { return dim * kPage + token; }

template <class T> struct Source {
    const T* p;
    int64_t row, head;
};

// One warp, one block, count <= kFew rows.
template <class T, int D> __device__ void append_few(const mrl_kv_cache& c, uint32_t layer, const Source<T>& src, const PageUnit& u, int head, int which) {
    constexpr int E = D / 32;
    const int lane = (int)threadIdx.x & 31;
    const size_t block = block_index(c, layer, u.page, which, head);
    const float old = c.scales[block];
    const T* from = src.p + (int64_t)head * src.head + lane * E;
    float x[kFew][E];
    float top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < kFew; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[i][e] = 0.0f;
        if (i < u.count) load_f32<T, E>(from + (int64_t)(u.row + i) * src.row, x[i]);
    }
#pragma unroll
    for (int i = 0; i < kFew; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float m = fabsf(x[i][e]);
            if (m < INFINITY) top = fmaxf(top, m);
            else odd = true;
        }
    if (__any_sync(~0u, odd) && lane == 0) atomicOr(c.status, MRL_KV_NONFINITE);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const bool had = u.slot > 0;
    const float s = new_scale(top, had, old);
    int8_t* out = c.codes + block * (size_t)(kPage * D);
    if (had && s > old) {
        const float ratio = __fdiv_rn(old, s);
        uint4* w = reinterpret_cast<uint4*>(out) + lane;
#pragma unroll 4
        for (int i = 0; i < kPage * D / 512; ++i) {
            uint4 v = w[i * 32];
            v.x = requant4(v.x, ratio);
            v.y = requant4(v.y, ratio);
            v.z = requant4(v.z, ratio);
            v.w = requant4(v.w, ratio);
            w[i * 32] = v;
        }
        __syncwarp();
    }
    if (lane == 0 && (!had || s > old)) c.scales[block] = s;
    // few values: the division itself
#pragma unroll
    for (int i = 0; i < kFew; ++i) {
        if (i >= u.count) break;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int dim = lane * E + e;
            out[which ? v_at(u.slot + i, dim) : k_at(u.slot + i, dim)] = s > 0.0f ? to_code(x[i][e], s) : (int8_t)0;
        }
    }
}

// The whole CTA, one block. Tile of 64 tokens x D: thread t holds dims 8 (t % (D/8)) .. + 7 of tokens
// t / (D/8) + i * (256 / (D/8)), i < kTok<D>.
template <int D> constexpr int kTok = kPage * D / 8 / kThreads;
template <class T, int D> __device__ __forceinline__ void load_tile(const Source<T>& src, const PageUnit& u, int head, uint4 (&raw)[kTok<D>]) {
    constexpr int kCols = D / 8, kStep = kThreads / kCols;
    const T* from = src.p + (int64_t)head * src.head + (int)threadIdx.x % kCols * 8;
#pragma unroll
    for (int i = 0; i < kTok<D>; ++i) {
        const int t = (int)threadIdx.x / kCols + i * kStep - u.slot;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (t >= 0 && t < u.count) raw[i] = *reinterpret_cast<const uint4*>(from + (int64_t)(u.row + t) * src.row);
    }
}
template <class T, int D>
__device__ void append_block(const mrl_kv_cache& c, uint32_t layer, const uint4 (&raw)[kTok<D>], const PageUnit& u, int head, int which, float* smax,
                             uint32_t* tile) {
    constexpr int kCols = D / 8, kStep = kThreads / kCols;
    const int tid = (int)threadIdx.x;
    const size_t block = block_index(c, layer, u.page, which, head);
    const float old = c.scales[block];
    const int col = tid % kCols, tok0 = tid / kCols;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kTok<D>; ++i) bits = max_bits(bits, raw[i]);
    float top = bits_f32<T>(bits);
    const bool odd = !(top < INFINITY);
    if (odd) {  // the largest finite one
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < kTok<D>; ++i) {
            float x[8];
            unpack8<T>(raw[i], x);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (fabsf(x[j]) < INFINITY) top = fmaxf(top, fabsf(x[j]));
        }
    }
    if (__any_sync(~0u, odd) && (tid & 31) == 0) atomicOr(c.status, MRL_KV_NONFINITE);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    __syncthreads();  // smax and the tile of the block before are read
    if ((tid & 31) == 0) smax[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, smax[i]);
    const bool had = u.slot > 0;
    const float s = new_scale(top, had, old);
    const float inv = __frcp_rn(s);
    uint32_t* out = reinterpret_cast<uint32_t*>(c.codes + block * (size_t)(kPage * D));
    if (had && s > old) {
        // every code of the page: those of slots not yet filled mean nothing
        const float ratio = __fdiv_rn(old, s);
        for (int i = tid; i < kPage * D / 4; i += kThreads) out[i] = requant4(out[i], ratio);
        __syncthreads();
    }
    if (tid == 0 && (!had || s > old)) c.scales[block] = s;
    if (which == 0) {
        // [D/64][64 tokens][64 dims]
        uint2* dst = reinterpret_cast<uint2*>(out) + (col / 8) * (kPage * 8) + col % 8;
#pragma unroll
        for (int i = 0; i < kTok<D>; ++i) {
            const int t = tok0 + i * kStep;
            float x[8];
            unpack8<T>(raw[i], x);
            if (t >= u.slot && t < u.slot + u.count) dst[t * 8] = make_uint2(to_codes4(x, s, inv), to_codes4(x + 4, s, inv));
        }
        return;
    }
    uint8_t* bytes = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
    for (int i = 0; i < kTok<D>; ++i) {
        const int t = tok0 + i * kStep;
        float x[8];
        unpack8<T>(raw[i], x);
        if (t >= u.slot && t < u.slot + u.count) {
            const uint32_t a = to_codes4(x, s, inv), b = to_codes4(x + 4, s, inv);
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

// The CTA's page, found by its first warp.
__device__ __forceinline__ PageUnit cta_page(const mrl_kv_cache& c, const Rows& r, PageUnit* su) {
    if (threadIdx.x < 32) {
        const PageUnit u = find_page_unit(c, r, (int)blockIdx.x);
        if (threadIdx.x == 0) *su = u;
    }
    __syncthreads();
    return *su;
}

// FEW: 8 blocks per CTA, a warp's each where the page gains few rows; else K and V of one head, both loaded
// before either is worked on.
template <class T, int D, bool FEW> __global__ void __launch_bounds__(kThreads) append_kernel(mrl_kv_cache c, uint32_t layer, Source<T> k, Source<T> v, Rows r) {
    __shared__ PageUnit su;
    __shared__ float smax[kWarps];
    __shared__ uint32_t tile[D * (kPage / 4 + 1)];  // V's codes, a dim's 64 tokens and a padding word
    const PageUnit u = cta_page(c, r, &su);
    if (u.count == 0) return;
    if (u.page < 0) {  // these rows have nowhere to go
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(c.status, MRL_KV_BAD_INDEX);
        return;
    }
    if constexpr (FEW) {
        const int first = (int)blockIdx.y * kWarps, blocks = min(kWarps, 2 * (int)c.kv_heads - first);
        if (u.count <= kFew) {
            const int b = (int)threadIdx.x >> 5;
            if (b < blocks) append_few<T, D>(c, layer, (first + b) & 1 ? v : k, u, (first + b) >> 1, (first + b) & 1);
            return;
        }
        for (int b = 0; b < blocks; ++b) {
            uint4 raw[kTok<D>];
            load_tile<T, D>((first + b) & 1 ? v : k, u, (first + b) >> 1, raw);
            append_block<T, D>(c, layer, raw, u, (first + b) >> 1, (first + b) & 1, smax, tile);
        }
    } else {
        const int head = (int)blockIdx.y;
        uint4 raw[2][kTok<D>];
        load_tile<T, D>(k, u, head, raw[0]);
        load_tile<T, D>(v, u, head, raw[1]);
        append_block<T, D>(c, layer, raw[0], u, head, 0, smax, tile);
        append_block<T, D>(c, layer, raw[1], u, head, 1, smax, tile);
    }
}

// E values of f32 to O, as one store.
template <class O, int E> __device__ __forceinline__ void store_vec(O* p, const float* x) {
    constexpr int kWords = E * (int)sizeof(O) / 4;
    uint32_t w[kWords];
    O* y = reinterpret_cast<O*>(w);
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = from_f32<O>(x[e]);
    if (kWords == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
    else if (kWords == 2) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(w);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}

template <class O, int D> __global__ void __launch_bounds__(kThreads) read_kernel(mrl_kv_cache c, uint32_t layer, O* k, O* v, Rows r, int per) {
    __shared__ PageUnit su;
    __shared__ uint32_t tile[D * (kPage / 4 + 1)];
    const int tid = (int)threadIdx.x;
    const PageUnit u = cta_page(c, r, &su);
    if (u.count == 0) return;
    if (u.seq < 0 && tid == 0 && blockIdx.y == 0) atomicOr(c.status, MRL_KV_BAD_INDEX);
    const int first = (int)blockIdx.y * per, blocks = min(per, 2 * (int)c.kv_heads - first);
    const size_t stride = (size_t)c.kv_heads * D;
    if (u.count <= kFew) {  // a warp per block
        const int b = first + (tid >> 5), lane = tid & 31, head = b >> 1, which = b & 1;
        if (b >= first + blocks) return;
        constexpr int E = D / 32;
        const size_t block = u.page < 0 ? 0 : block_index(c, layer, u.page, which, head);
        const int8_t* codes = c.codes + block * (size_t)(kPage * D);
        const float s = u.page < 0 ? 0.0f : c.scales[block];
        for (int i = 0; i < u.count; ++i) {
            O* dst = (which ? v : k) + (size_t)(u.row + i) * stride + (size_t)head * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int dim = lane * E + e;
                dst[e] = from_f32<O>(u.page < 0 ? 0.0f : __fmul_rn((float)codes[which ? v_at(u.slot + i, dim) : k_at(u.slot + i, dim)], s));
            }
        }
        return;
    }
    for (int x = 0; x < blocks; ++x) {
        const int b = first + x, head = b >> 1, which = b & 1;
        O* dst = (which ? v : k) + (size_t)u.row * stride + (size_t)head * D;
        if (u.page < 0) {
            for (int i = tid; i < u.count * D; i += kThreads) dst[(size_t)(i / D) * stride + i % D] = from_f32<O>(0.0f);
            continue;
        }
        const size_t block = block_index(c, layer, u.page, which, head);
        const float s = c.scales[block];
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(c.codes + block * (size_t)(kPage * D));
        if (which) {
            __syncthreads();  // the tile of the block before is read
            for (int i = tid; i < D * kPage / 4; i += kThreads) tile[(i / (kPage / 4)) * (kPage / 4 + 1) + i % (kPage / 4)] = codes[i];
            __syncthreads();
        }
        const int8_t* turned = reinterpret_cast<const int8_t*>(tile);
#pragma unroll 4
        for (int i = tid; i < u.count * (D / 4); i += kThreads) {
            const int t = i / (D / 4), d = i % (D / 4) * 4, slot = u.slot + t;
            uint32_t w;
            if (which) {
                w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= (uint32_t)(uint8_t)turned[(d + j) * (kPage + 4) + slot] << (8 * j);
            } else {
                w = codes[k_at(slot, d) / 4];
            }
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __fmul_rn((float)(int8_t)(w >> (8 * j)), s);
            store_vec<O, 4>(dst + (size_t)t * stride + d, y);
        }
    }
}

// Whether the call's sequences gain few rows each. Measured, 8 kv heads of 128: 256 rows of 256 sequences 36 us
// with a CTA per block and 9 us with a warp per block.
bool few_rows(const Rows& r) { return r.tokens <= kFew * r.n; }

template <class T, int D> cudaError_t append_launch(const mrl_kv_cache& c, uint32_t layer, Source<T> k, Source<T> v, const Rows& r, cudaStream_t s) {
    const unsigned units = (unsigned)page_units(r.n, r.tokens, r.cu != nullptr);
    if (few_rows(r)) append_kernel<T, D, true><<<dim3(units, (2 * c.kv_heads + kWarps - 1) / kWarps), kThreads, 0, s>>>(c, layer, k, v, r);
    else append_kernel<T, D, false><<<dim3(units, c.kv_heads), kThreads, 0, s>>>(c, layer, k, v, r);
    return cudaGetLastError();
}
template <class T> cudaError_t append_dims(const mrl_kv_cache& c, uint32_t layer, Source<T> k, Source<T> v, const Rows& r, cudaStream_t s) {
    return c.head_dim == 64    ? append_launch<T, 64>(c, layer, k, v, r, s)
           : c.head_dim == 128 ? append_launch<T, 128>(c, layer, k, v, r, s)
                               : append_launch<T, 256>(c, layer, k, v, r, s);
}

template <class O> cudaError_t read_dims(const mrl_kv_cache& c, uint32_t layer, void* k, void* v, const Rows& r, dim3 grid, int per, cudaStream_t s) {
    O *kp = static_cast<O*>(k), *vp = static_cast<O*>(v);
    if (c.head_dim == 64) read_kernel<O, 64><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r, per);
    else if (c.head_dim == 128) read_kernel<O, 128><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r, per);
    else read_kernel<O, 256><<<grid, kThreads, 0, s>>>(c, layer, kp, vp, r, per);
    return cudaGetLastError();
}

dim3 page_grid(const mrl_kv_cache& c, const Rows& r, int per) {
    return dim3((unsigned)page_units(r.n, r.tokens, r.cu != nullptr), (2 * c.kv_heads + per - 1) / per);
}

}  // namespace
}  // namespace kv

int launch_kv_append(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, const void* k, int64_t k_row, int64_t k_head,
                     const void* v, int64_t v_row, int64_t v_head, const kv::Rows& r, cudaStream_t s) {
    if (dtype == MRL_F16)
        return (int)kv::append_dims<__half>(c, layer, {static_cast<const __half*>(k), k_row, k_head}, {static_cast<const __half*>(v), v_row, v_head}, r, s);
    return (int)kv::append_dims<__nv_bfloat16>(c, layer, {static_cast<const __nv_bfloat16*>(k), k_row, k_head},
                                               {static_cast<const __nv_bfloat16*>(v), v_row, v_head}, r, s);
}

int launch_kv_read(const mrl_kv_cache& c, uint32_t layer, uint32_t dtype, void* k, void* v, const kv::Rows& r, cudaStream_t s) {
    const int per = kv::few_rows(r) ? kv::kWarps : 1;
    const dim3 grid = kv::page_grid(c, r, per);
    return (int)(dtype == MRL_F16    ? kv::read_dims<__half>(c, layer, k, v, r, grid, per, s)
                 : dtype == MRL_BF16 ? kv::read_dims<__nv_bfloat16>(c, layer, k, v, r, grid, per, s)
                                     : kv::read_dims<float>(c, layer, k, v, r, grid, per, s));
}

}  // namespace mrl
