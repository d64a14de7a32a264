// Rotary positions with several axes, and the append of rotated keys and of
// values to a paged cache.
//
// Mathematics.  A head's row x (dim columns) is scaled by its RMS norm,
// n_i = x_i w_i / sqrt(mean(x^2) + eps) (left out without w), and its first
// rot_dim columns turn in pairs (i, i + rot_dim / 2) by the angle
// a_i = position[axis(i)] * base^(-2 i / rot_dim):
//   y_i = n_i cos a_i - n_(i+rot/2) sin a_i,  y_(i+rot/2) = n_(i+rot/2) cos a_i + n_i sin a_i.
// The axis of pair i follows the sections (time, height, width, extra): in a
// row, or interleaved (pairs 3 j + 1 and 3 j + 2 take height and width as far
// as those sections reach, every other pair time).
//
// An angle of a far position does not fit fp32 (200000 radians keep 2^-7), so
// the frequencies are 64-bit fixed-point turns per position, base^(..)/(2 pi)
// 2^64: the wrapping product with the position is the angle's fraction of a
// turn, exact to position * 2^-65, for one 64-bit integer multiply.
//
// What bounds it: bytes (10 flop an element), once the angles, 8 sines and
// cosines a lane, serve several heads: a lane holds eight columns of up to
// eight heads of a token, so every load and store is 16 bytes a lane, a wave
// works on several rows at once, and a pair's other half is one lane exchange
// away (rot_dim is a multiple of 16).  With fewer heads a lane where a call
// would fill the card with less than 2048 waves: there latency counts
// (32 heads x 128 bf16, one, four, eight heads a lane: 8192 tokens 54, 34, 29
// us, 4096 30, 20, 16, 1024 9.5, 7.5, 8.4; one token x 16 heads x 256 fp32:
// 4.3, 6.8, 10).
#include "rope_rows.h"

namespace qw35 {
namespace {

using namespace rows;

// Workgroups of four waves; 2^log2_lanes lanes a row.  An item is a token with up
// to H heads, which share the angles.
template <class TI, class TO, int H>
__global__ __launch_bounds__(256) void rotate_kernel(HeadsView x, HeadsView y, int n_tokens, int heads, int dim,
                                                     int log2_lanes, RopeArgs rope) {
    const int lanes = 1 << log2_lanes, li = threadIdx.x & (lanes - 1);
    const int groups = (heads + H - 1) / H;
    const int item = (int)(blockIdx.x << (8 - log2_lanes) | threadIdx.x >> log2_lanes);  // below 2^31
    const int t0 = item / groups, h0 = (item - t0 * groups) * H;
    const bool live = t0 < n_tokens && li * 8 < dim;
    const int t = live ? t0 : 0;
    float v[H][8] = {};
#pragma unroll
    for (int h = 0; h < H; ++h)
        if (live && h0 + h < heads)
            load8<TI>(x.data, t * x.token_stride + (h0 + h) * x.head_stride + li * 8, x.vec, v[h]);
    Turn turn = {};
    if (rope.freq && live && li * 8 < rope.rot_dim) turn = turn_of(rope, n_tokens, t, li * 8);
#pragma unroll
    for (int h = 0; h < H; ++h) {
        norm_and_turn(rope, dim, lanes, li, turn, v[h]);
        if (live && h0 + h < heads)
            store8<TO>(y.data, t * y.token_stride + (h0 + h) * y.head_stride + li * 8, y.vec, v[h]);
    }
}

struct Slot {
    int64_t page;
    int at;
};

__device__ __forceinline__ Slot slot_of(int64_t slot, int page_size, bool small) {
    Slot s;
    s.page = small ? (int64_t)((uint32_t)slot / (uint32_t)page_size) : slot / page_size;
    s.at = (int)(slot - s.page * page_size);
    return s;
}

// Keys.  An item is a token with up to H heads, as in rotate_kernel; the rows
// of a wave are consecutive tokens, whose 16-byte granules of a key page are
// neighbours.
template <class TI, class C, int H>
__device__ __forceinline__ void append_keys(const qw35_hip_kv_cache& cache, const HeadsView& k, int n_tokens,
                                            const int64_t* slots, int log2_lanes, const RopeArgs& rope) {
    const int lanes = 1 << log2_lanes, li = threadIdx.x & (lanes - 1);
    const int dim = (int)cache.head_dim, heads = (int)cache.kv_heads, page = (int)cache.page_size;
    const int64_t n_slots = (int64_t)cache.n_pages * page;
    const int groups = (heads + H - 1) / H;
    const int item = (int)(blockIdx.x << (8 - log2_lanes) | threadIdx.x >> log2_lanes);  // below 2^31
    const int group = item / n_tokens, t = item - group * n_tokens, h0 = group * H;
    const int64_t slot = group < groups ? slots[t] : -1;
    const bool live = slot >= 0 && slot < n_slots;
    float x[H][8] = {};
#pragma unroll
    for (int h = 0; h < H; ++h)
        if (live && h0 + h < heads)
            load8<TI>(k.data, t * k.token_stride + (h0 + h) * k.head_stride + li * 8, k.vec, x[h]);
    Turn turn = {};
    if (rope.freq && live && li * 8 < rope.rot_dim) turn = turn_of(rope, n_tokens, t, li * 8);
    const Slot s = live ? slot_of(slot, page, n_slots <= 0xffffffffll) : Slot{0, 0};
    const int64_t at = s.page * heads * ((int64_t)page * dim) + (s.at / 32) * 32 * dim + li * 256 + (s.at & 31) * 8;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        norm_and_turn(rope, dim, lanes, li, turn, x[h]);
        if (live && h0 + h < heads) {
            if constexpr (std::is_same_v<C, Fp8>) {
                const float scale = cache.k_scale ? cache.k_scale[h0 + h] : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[h][j] /= scale;
            }
            store_granule<C>(cache.k, at + (int64_t)(h0 + h) * page * dim, x[h]);
        }
    }
}

// Values.  A value page holds eight tokens of a column together, so a token's
// row by itself is dim elements at a stride of eight.  A wave takes eight
// tokens of a head, eight lanes a token; where they are the eight of a granule
// (a prompt, whose first token's slot says where granules begin), they change
// places in LDS and the wave writes 64 whole granules, 1 KB, at a time.
// Otherwise every lane writes its elements.
template <class TI, class C>
__device__ __forceinline__ void append_values(const qw35_hip_kv_cache& cache, const HeadsView& v, int n_tokens,
                                              const int64_t* slots) {
    // 8 columns x 8 tokens a lane group, 8 floats apart from the next: a wave's writes and reads meet no bank twice
    __shared__ __align__(16) float block[4][8 * 72];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane >> 3, part = lane & 7;
    const int dim = (int)cache.head_dim, heads = (int)cache.kv_heads, page = (int)cache.page_size;
    const int64_t n_slots = (int64_t)cache.n_pages * page;
    const int item = (int)blockIdx.x * 4 + wave, octet = item / heads, h = item - octet * heads;
    const int shift = (int)(slots[0] & 7);
    if (octet * 8 - shift >= n_tokens) return;
    const int t = octet * 8 - shift + j;
    const bool in = t >= 0 && t < n_tokens;
    const int64_t slot = in ? slots[t] : -1;
    const bool live = slot >= 0 && slot < n_slots;
    const int64_t first = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(slot >> 32)) << 32 |
                                    (uint32_t)__builtin_amdgcn_readfirstlane((int)slot));
    const bool whole = __all(live && slot == first + j && (first & 7) == 0);
    float scale = 1.0f;
    if constexpr (std::is_same_v<C, Fp8>) {
        if (cache.v_scale) scale = cache.v_scale[h];
    }
    const Slot s = live ? slot_of(slot, page, n_slots <= 0xffffffffll) : Slot{0, 0};
    const int64_t at = (s.page * heads + h) * ((int64_t)page * dim) + (int64_t)(s.at / 8) * 8 * dim;
    for (int c0 = 0; c0 < dim; c0 += 64) {
        const int col = c0 + part * 8;
        float x[8] = {};
        if (live) load8<TI>(v.data, t * v.token_stride + h * v.head_stride + col, v.vec, x);
        if constexpr (std::is_same_v<C, Fp8>) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] /= scale;
        }
        if (whole) {
            float* const b = block[wave];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[part * 72 + i * 8 + j] = x[i];
            __builtin_amdgcn_wave_barrier();
            const float4_t* const g = reinterpret_cast<const float4_t*>(b + lane * 8 + (lane >> 3) * 8);
            const float4_t lo = g[0], hi = g[1];
            __builtin_amdgcn_wave_barrier();
            const float w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            store_granule<C>(cache.v, at + (c0 + lane) * 8, w);
        } else if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) store_one<C>(cache.v, at + (col + i) * 8 + (s.at & 7), x[i]);
        }
    }
}

// blockIdx.y 0: keys, 1: values.
template <class TI, class C, int H>
__global__ __launch_bounds__(256) void kv_append_kernel(qw35_hip_kv_cache cache, HeadsView k, HeadsView v,
                                                        int n_tokens, const int64_t* slots, int log2_lanes, RopeArgs rope) {
    if (blockIdx.y == 0) append_keys<TI, C, H>(cache, k, n_tokens, slots, log2_lanes, rope);
    else append_values<TI, C>(cache, v, n_tokens, slots);
}

// Heads of a lane: eight if they leave 2048 waves, four if they leave 1024.
int lane_heads(int n_tokens, int heads, int log2_lanes) {
    const int64_t waves = ((int64_t)n_tokens * heads << log2_lanes) / 64;
    return heads >= 8 && waves >= 8 * 2048 ? 8 : heads >= 4 && waves >= 4 * 1024 ? 4 : 1;
}

template <class TI, class TO, int H>
hipError_t rotate_heads(const HeadsView& x, const HeadsView& y, int n_tokens, int heads, int dim, int log2_lanes,
                        const RopeArgs& rope, hipStream_t stream) {
    const int64_t items = (int64_t)n_tokens * ((heads + H - 1) / H);
    rotate_kernel<TI, TO, H>
        <<<dim3((unsigned)(((items << log2_lanes) + 255) / 256)), 256, 0, stream>>>(x, y, n_tokens, heads, dim, log2_lanes,
                                                                            rope);
    return hipGetLastError();
}

template <class TI, class TO>
hipError_t rotate_as(const HeadsView& x, const HeadsView& y, int n_tokens, int heads, int dim, const RopeArgs& rope,
                     hipStream_t stream) {
    const int lanes = row_lanes_log2(dim), h = lane_heads(n_tokens, heads, lanes);
    return h == 8   ? rotate_heads<TI, TO, 8>(x, y, n_tokens, heads, dim, lanes, rope, stream)
           : h == 4 ? rotate_heads<TI, TO, 4>(x, y, n_tokens, heads, dim, lanes, rope, stream)
                    : rotate_heads<TI, TO, 1>(x, y, n_tokens, heads, dim, lanes, rope, stream);
}

template <class TI>
hipError_t rotate_from(const HeadsView& x, const HeadsView& y, int n, int heads, int dim, const RopeArgs& rope,
                       hipStream_t stream) {
    switch (y.dtype) {
        case QW35_HIP_DTYPE_F32: return rotate_as<TI, float>(x, y, n, heads, dim, rope, stream);
        case QW35_HIP_DTYPE_F16: return rotate_as<TI, _Float16>(x, y, n, heads, dim, rope, stream);
        default: return rotate_as<TI, __bf16>(x, y, n, heads, dim, rope, stream);
    }
}

template <class TI, class C, int H>
hipError_t append_heads(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n, int log2_lanes,
                        const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    const int heads = (int)cache.kv_heads;
    const int64_t keys = (((int64_t)n * ((heads + H - 1) / H) << log2_lanes) + 255) / 256;
    const int64_t values = ((int64_t)(n + 14) / 8 * heads + 3) / 4;  // (the first octet may begin before the tokens)
    kv_append_kernel<TI, C, H><<<dim3((unsigned)(keys > values ? keys : values), 2), 256, 0, stream>>>(cache, k, v, n, slots,
                                                                                                   log2_lanes, rope);
    return hipGetLastError();
}

template <class TI, class C>
hipError_t append_as(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n,
                     const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    const int lanes = row_lanes_log2((int)cache.head_dim), h = lane_heads(n, (int)cache.kv_heads, lanes);
    return h >= 4 ? append_heads<TI, C, 4>(cache, k, v, n, lanes, slots, rope, stream)
                  : append_heads<TI, C, 1>(cache, k, v, n, lanes, slots, rope, stream);
}

template <class TI>
hipError_t append_from(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n,
                       const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    switch (cache.dtype) {
        case QW35_HIP_DTYPE_F16: return append_as<TI, _Float16>(cache, k, v, n, slots, rope, stream);
        case QW35_HIP_DTYPE_BF16: return append_as<TI, __bf16>(cache, k, v, n, slots, rope, stream);
        default: return append_as<TI, Fp8>(cache, k, v, n, slots, rope, stream);
    }
}

}  // namespace

hipError_t launch_rotate(const HeadsView& x, const HeadsView& y, int n_tokens, int heads, int dim, const RopeArgs& rope,
                         hipStream_t stream) {
    switch (x.dtype) {
        case QW35_HIP_DTYPE_F32: return rotate_from<float>(x, y, n_tokens, heads, dim, rope, stream);
        case QW35_HIP_DTYPE_F16: return rotate_from<_Float16>(x, y, n_tokens, heads, dim, rope, stream);
        default: return rotate_from<__bf16>(x, y, n_tokens, heads, dim, rope, stream);
    }
}

hipError_t launch_kv_append(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                            const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    switch (k.dtype) {
        case QW35_HIP_DTYPE_F32: return append_from<float>(cache, k, v, n_tokens, slots, rope, stream);
        case QW35_HIP_DTYPE_F16: return append_from<_Float16>(cache, k, v, n_tokens, slots, rope, stream);
        default: return append_from<__bf16>(cache, k, v, n_tokens, slots, rope, stream);
    }
}

}  // namespace qw35
