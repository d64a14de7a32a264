// A paged cache in 8 bits with a scale for each block of 32 tokens and head:
// the append that quantises, and the reading back (of every kind of cache).
//
// Mathematics.  A block is the 32 tokens of slot / 32 of one kv head, keys and
// values apart; a code c of it stands for c s.  With Q the largest code (127, 448),
// m the largest finite magnitude of the block's tokens x in a call and s0 its scale
// before (zero if the call writes its first token: the block begins anew),
//   s = s0 2^j, the least j >= 0 with m <= Q s; the least power of two if s0 is zero,
//   c = rne(x / s) of new tokens, rne(c 2^-j) of those it held.
// Powers of two: a block that grows shifts its codes, which e4m3 does without loss
// but in its subnormals and int8 within 1/2 + 1/4 + .. < 1 step in all; the scale of
// a block that begins with a call's own tokens does not depend on how a prompt was
// cut into calls.  (A scale of m / Q keeps up to one bit more of an int8 block
// written at once, and rounds every token again each time that m rises.)
#include "rope_rows.h"

namespace qw35 {
namespace {

using namespace rows;

struct Int8 {};

template <class C>
struct Codes;

template <>
struct Codes<Int8> {
    static constexpr uint32_t kTopExponent = 6, kTopMantissa = 0x7e0000;  // 127 = 1.984375 2^6
    static constexpr float kTop = 127.0f;
    // Four numbers, nearest integers, ties to even (a sum with 1.5 2^23 leaves them in its low bits); NaN is zero.
    static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
        auto low = [](float v) {
            v = v == v ? fminf(fmaxf(v, -kTop), kTop) : 0.0f;
            return __builtin_bit_cast(uint32_t, v + 12582912.0f) & 0xffu;
        };
        return low(a) | low(b) << 8 | low(c) << 16 | low(d) << 24;
    }
    static __device__ __forceinline__ void unpack4(uint32_t w, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> 8 * i);
    }
};

template <>
struct Codes<Fp8> {
    static constexpr uint32_t kTopExponent = 8, kTopMantissa = 0x600000;  // 448 = 1.75 2^8
    static constexpr float kTop = 448.0f;
    static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
        return pack4_e4m3(a, b, c, d);
    }
    static __device__ __forceinline__ void unpack4(uint32_t w, float (&v)[4]) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    }
};

constexpr int kLeastExponent = -60;  // of a scale: its reciprocal and log2 stay far inside fp32

// The least power of two s with m <= Q s.
template <class C>
__device__ __forceinline__ float fitting(float m) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, m);
    int e = (int)(bits >> 23) - (int)Codes<C>::kTopExponent + ((bits & 0x7fffffu) > Codes<C>::kTopMantissa ? 1 : 0);
    if (e < 127 + kLeastExponent) e = 127 + kLeastExponent;
    return m > 0.0f ? __builtin_bit_cast(float, (uint32_t)e << 23) : 0.0f;
}

struct BlockAppend {
    qw35_hip_kv_cache cache;
    HeadsView k, v;
    int n_tokens;        // of the positions
    int t0, t1;          // the tokens of this launch
    const int64_t* slots;
    int per;             // tokens whose blocks a workgroup looks for
    int heads_per;       // heads of a workgroup
    RopeArgs rope;
};

// What a workgroup shares.
template <int D>
struct BlockShared {
    int src[32];        // of the block's tokens: which of the call it is (-1: none)
    float top[2][4];    // the waves' largest magnitudes, of this head and the last
    float before[2];    // the scale before
    uint2 codes[32][D / 8 + 1];
};

// The scale of a block, and what its old codes are multiplied by (zero: they are forgotten).
struct Scale {
    float now, shrink;
    bool changed;
};

template <class C>
__device__ __forceinline__ Scale scale_of(float before, bool anew, float m) {
    // (a scale that no append has written counts as none)
    const bool has = !anew && before > 0x1p-126f && before < 0x1p126f;
    Scale s = {has ? before : fitting<C>(m), has ? 1.0f : 0.0f, false};
    for (int j = 0; has && j < 256 && m > Codes<C>::kTop * s.now; ++j) {
        s.now *= 2.0f;
        s.shrink *= 0.5f;
    }
    s.changed = anew || s.now != before;
    return s;
}

// The block's scale from every thread's largest magnitude.
template <class C, int D>
__device__ __forceinline__ Scale agree(BlockShared<D>& sh, int parity, const float* at, bool anew, float m) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) sh.top[parity][threadIdx.x >> 6] = m;
    if (threadIdx.x == 0) sh.before[parity] = anew ? 0.0f : *at;
    __syncthreads();
    m = fmaxf(fmaxf(sh.top[parity][0], sh.top[parity][1]), fmaxf(sh.top[parity][2], sh.top[parity][3]));
    return scale_of<C>(sh.before[parity], anew, m);
}

// The largest finite magnitude of eight numbers; infinities become fp32's largest number (and so the largest code).
__device__ __forceinline__ float largest(float (&x)[8], float m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = fabsf(x[j]);
        m = v < __builtin_inff() && v > m ? v : m;
        if (v == __builtin_inff()) x[j] = copysignf(0x1.fffffep127f, x[j]);
    }
    return m;
}

// Four codes at another scale.
template <class C>
__device__ __forceinline__ uint32_t again(uint32_t w, float shrink) {
    float v[4];
    Codes<C>::unpack4(w, v);
    const uint32_t r = Codes<C>::pack4(v[0] * shrink, v[1] * shrink, v[2] * shrink, v[3] * shrink);
    return shrink > 0.0f ? r : 0u;
}

template <class C>
__device__ __forceinline__ uint2 pack8(const float (&x)[8], float inv) {
    return {Codes<C>::pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
            Codes<C>::pack4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv)};
}

// 4 x 4 bytes: byte j of r[i] is byte i of w[j].
__device__ __forceinline__ void transpose4(const uint32_t (&w)[4], uint32_t (&r)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
    r[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
    r[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    r[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
    r[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}

// A workgroup writes blocks: of `per` tokens of the call those that are the
// first of theirs look through the call's slots for the block's other tokens (of two
// with the same slot the last counts), so that every block has one writer, in
// whatever order the tokens come, and results do not depend on timing.  A
// thread holds eight columns of D / 64 of the block's tokens.
template <class TI, class C, int D, bool kValues>
__device__ __forceinline__ void append_blocks(const BlockAppend& a, BlockShared<D>& sh) {
    constexpr int kLanes = D / 8, kRows = D / 64, kStep = 256 / kLanes;
    const int tid = threadIdx.x, li = tid % kLanes, row0 = tid / kLanes;
    const int heads = (int)a.cache.kv_heads, blocks = (int)a.cache.page_size / 32;
    const int64_t n_slots = (int64_t)a.cache.n_pages * a.cache.page_size;
    const int h0 = ((int)blockIdx.y >> 1) * a.heads_per, h1 = h0 + a.heads_per < heads ? h0 + a.heads_per : heads;
    const HeadsView& x_view = kValues ? a.v : a.k;
    uint8_t* const pages = static_cast<uint8_t*>(kValues ? a.cache.v : a.cache.k);
    float* const scales = const_cast<float*>(kValues ? a.cache.v_scale : a.cache.k_scale);  // (the cache's, written here)
    for (int i = 0; i < a.per; ++i) {
        const int t = a.t0 + (int)blockIdx.x * a.per + i;
        if (t >= a.t1) break;
        const int64_t slot = a.slots[t];
        if (slot < 0 || slot >= n_slots) continue;
        const int64_t block = slot / 32;
        if (t > a.t0) {
            const int64_t last = a.slots[t - 1];
            if (last >= 0 && last / 32 == block) continue;
        }
        __syncthreads();
        if (tid < 32) sh.src[tid] = -1;
        __syncthreads();
        int earlier = 0;
        for (int j = a.t0 + tid; j < a.t1; j += 256) {
            const int64_t s = a.slots[j];
            if (s < 0 || s / 32 != block) continue;
            if (j < t) earlier = 1;
            else atomicMax(&sh.src[s & 31], j);
        }
        if (__syncthreads_or(earlier)) continue;
        const uint32_t written = (uint32_t)__ballot(sh.src[tid & 31] >= 0);
        const bool anew = written & 1;
        const int64_t page = block / blocks;
        const int in_page = (int)(block - page * blocks);
        int src[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) src[r] = sh.src[row0 + r * kStep];
        Turn turn[kRows];
        if constexpr (!kValues) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                turn[r] = Turn{};
                if (a.rope.freq && src[r] >= 0 && li * 8 < a.rope.rot_dim) turn[r] = turn_of(a.rope, a.n_tokens, src[r], li * 8);
            }
        }
        for (int h = h0; h < h1; ++h) {
            const int64_t tile = (page * heads + h) * blocks + in_page;
            uint8_t* const codes = pages + tile * (32 * D);
            float x[kRows][8] = {}, m = 0.0f;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (src[r] >= 0)
                    load8<TI>(x_view.data, src[r] * x_view.token_stride + h * x_view.head_stride + li * 8, x_view.vec, x[r]);
            if constexpr (!kValues) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) norm_and_turn(a.rope, D, kLanes, li, turn[r], x[r]);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) m = largest(x[r], m);
            // (values: this thread's granules, four columns of eight tokens)
            const int quad = tid % (D / 4), octet = tid / (D / 4);
            const uint32_t mine = octet < 4 ? written >> octet * 8 & 0xff : 0xff;
            uint4_t* const granules = reinterpret_cast<uint4_t*>(codes + (octet & 3) * 8 * D + quad * 32);
            uint4_t old[2] = {};
            if (kValues && !anew && mine != 0xff) {
                old[0] = granules[0];
                old[1] = granules[1];
            }
            const Scale s = agree<C>(sh, h & 1, scales + tile, anew, m);
            const float inv = s.now > 0.0f ? 1.0f / s.now : 0.0f;
            const bool rewrite = anew || s.shrink != 1.0f;  // the tokens that the call does not write change too
            if constexpr (!kValues) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    uint2* const at = reinterpret_cast<uint2*>(codes + li * 256 + (row0 + r * kStep) * 8);
                    uint2 w = pack8<C>(x[r], inv);
                    if (src[r] < 0) {
                        if (!rewrite) continue;
                        w = {0, 0};
                        if (!anew) {
                            w = *at;
                            w = {again<C>(w.x, s.shrink), again<C>(w.y, s.shrink)};
                        }
                    }
                    *at = w;
                }
            } else {
#pragma unroll
                for (int r = 0; r < kRows; ++r) sh.codes[row0 + r * kStep][li] = pack8<C>(x[r], inv);
                __syncthreads();
                if (octet < 4 && (mine || rewrite)) {
                    uint32_t w[2][4], g[2][4];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[j / 4][j % 4] = reinterpret_cast<const uint32_t*>(sh.codes[octet * 8 + j])[quad];
                    transpose4(w[0], g[0]);
                    transpose4(w[1], g[1]);
                    uint4_t out[2] = {{g[0][0], g[1][0], g[0][1], g[1][1]}, {g[0][2], g[1][2], g[0][3], g[1][3]}};
                    if (!anew && mine != 0xff) {
                        uint32_t keep[2];  // bytes of the tokens that the call writes
#pragma unroll
                        for (int j = 0; j < 2; ++j) keep[j] = ((mine >> 4 * j & 15) * 0x00204081u & 0x01010101u) * 255u;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint32_t o = old[j / 4][j % 4];
                            if (rewrite) o = again<C>(o, s.shrink);
                            out[j / 4][j % 4] = (out[j / 4][j % 4] & keep[j & 1]) | (o & ~keep[j & 1]);
                        }
                    }
                    granules[0] = out[0];
                    granules[1] = out[1];
                }
            }
            if (tid == 0 && s.changed) scales[tile] = s.now;
        }
    }
}

// blockIdx.y: even keys, odd values of a group of heads.
template <class TI, class C, int D>
__global__ __launch_bounds__(256) void kv_append_blocks_kernel(BlockAppend a) {
    __shared__ BlockShared<D> sh;
    if (blockIdx.y & 1) append_blocks<TI, C, D, true>(a, sh);
    else append_blocks<TI, C, D, false>(a, sh);
}

template <class TI, class C, int D>
hipError_t append_dim(BlockAppend a, int n, hipStream_t stream) {
    const int heads = (int)a.cache.kv_heads;
    for (a.t0 = 0; a.t0 < n; a.t0 = a.t1) {
        const int count = n - a.t0 < kAppendSlice ? n - a.t0 : kAppendSlice;
        a.t1 = a.t0 + count;
        a.per = (int64_t)count * heads > 2048 ? 32 : 1;
        a.heads_per = 1;
        const dim3 grid((unsigned)((count + a.per - 1) / a.per), (unsigned)((heads + a.heads_per - 1) / a.heads_per * 2));
        kv_append_blocks_kernel<TI, C, D><<<grid, 256, 0, stream>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <class TI, class C>
hipError_t append_codes(const BlockAppend& a, int n, hipStream_t stream) {
    switch (a.cache.head_dim) {
        case 64: return append_dim<TI, C, 64>(a, n, stream);
        case 128: return append_dim<TI, C, 128>(a, n, stream);
        default: return append_dim<TI, C, 256>(a, n, stream);
    }
}

template <class TI>
hipError_t append_type(const BlockAppend& a, int n, hipStream_t stream) {
    return a.cache.dtype == QW35_HIP_DTYPE_I8_BLOCKS ? append_codes<TI, Int8>(a, n, stream)
                                                     : append_codes<TI, Fp8>(a, n, stream);
}

// ---- reading back --------------------------------------------------------------------------------------------------

struct CacheRead {
    qw35_hip_kv_cache cache;
    HeadsView k, v;
    int n_tokens;
    const int64_t* slots;
    int by_block;  // scales: of a block; else of a head
};

template <class C>
__device__ __forceinline__ float element(const void* cache, int64_t at) {
    if constexpr (std::is_same_v<C, Int8>) {
        return (float)static_cast<const int8_t*>(cache)[at];
    } else if constexpr (std::is_same_v<C, Fp8>) {
        float v[4];
        Codes<Fp8>::unpack4(static_cast<const uint8_t*>(cache)[at], v);
        return v[0];
    } else {
        return (float)static_cast<const C*>(cache)[at];
    }
}

// A lane has eight columns of a head of a token.
template <class C, class TO>
__global__ __launch_bounds__(256) void kv_read_kernel(CacheRead a) {
    const int heads = (int)a.cache.kv_heads, dim = (int)a.cache.head_dim, page_size = (int)a.cache.page_size;
    const int lanes = dim / 8;
    const bool values = blockIdx.y != 0;
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
    const int li = threadIdx.x % lanes;
    const int64_t t = item / heads;
    const int h = (int)(item - t * heads);
    if (t >= a.n_tokens) return;
    const int64_t slot = a.slots[t];
    float x[8] = {};
    if (slot >= 0 && slot < (int64_t)a.cache.n_pages * page_size) {
        const int64_t page = slot / page_size, tile0 = (page * heads + h) * (page_size / 32);
        const int at = (int)(slot - page * page_size);
        const float* const scales = values ? a.cache.v_scale : a.cache.k_scale;
        const float scale = !scales ? 1.0f : a.by_block ? scales[tile0 + at / 32] : scales[h];
        const int64_t base = tile0 * (32 * dim);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t e = values ? base + (int64_t)(at / 8) * 8 * dim + (li * 8 + j) * 8 + at % 8
                                     : base + (int64_t)(at / 32) * 32 * dim + li * 256 + (at % 32) * 8 + j;
            x[j] = element<C>(values ? a.cache.v : a.cache.k, e) * scale;
        }
    }
    const HeadsView& y = values ? a.v : a.k;
    store8<TO>(y.data, t * y.token_stride + h * y.head_stride + li * 8, y.vec, x);
}

template <class C, class TO>
hipError_t read_as(const CacheRead& a, hipStream_t stream) {
    const int64_t items = (int64_t)a.n_tokens * a.cache.kv_heads * (a.cache.head_dim / 8);
    kv_read_kernel<C, TO><<<dim3((unsigned)((items + 255) / 256), 2), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <class C>
hipError_t read_to(const CacheRead& a, hipStream_t stream) {
    switch (a.k.dtype) {
        case QW35_HIP_DTYPE_F32: return read_as<C, float>(a, stream);
        case QW35_HIP_DTYPE_F16: return read_as<C, _Float16>(a, stream);
        default: return read_as<C, __bf16>(a, stream);
    }
}

}  // namespace

hipError_t launch_kv_append_blocks(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                                   const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    const BlockAppend a = {cache, k, v, n_tokens, 0, 0, slots, 1, 1, rope};
    switch (k.dtype) {
        case QW35_HIP_DTYPE_F32: return append_type<float>(a, n_tokens, stream);
        case QW35_HIP_DTYPE_F16: return append_type<_Float16>(a, n_tokens, stream);
        default: return append_type<__bf16>(a, n_tokens, stream);
    }
}

hipError_t launch_kv_read(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                          const int64_t* slots, hipStream_t stream) {
    const CacheRead a = {cache, k, v, n_tokens, slots, block_scaled(cache.dtype)};
    switch (cache.dtype) {
        case QW35_HIP_DTYPE_F16: return read_to<_Float16>(a, stream);
        case QW35_HIP_DTYPE_BF16: return read_to<__bf16>(a, stream);
        case QW35_HIP_DTYPE_I8_BLOCKS: return read_to<Int8>(a, stream);
        default: return read_to<Fp8>(a, stream);
    }
}

}  // namespace qw35
