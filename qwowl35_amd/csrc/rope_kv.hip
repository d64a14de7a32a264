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
// What bounds it: bytes (10 flop an element).  A lane holds eight columns, a
// row lies in dim / 8 lanes, so a wave works on several rows at once, every
// load and store is 16 bytes a lane, and a pair's other half is one lane
// exchange away (rot_dim is a multiple of 16).
#include "attention.h"
#include "qw35_device.h"

namespace qw35 {
namespace {

struct Fp8 {};  // e4m3 in a cache page

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <class T>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool vec, float (&v)[8]) {
    const T* p = static_cast<const T*>(base) + at;
    if (vec) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            const vec_t t = reinterpret_cast<const vec_t*>(p)[i];
#pragma unroll
            for (int j = 0; j < N; ++j) v[i * N + j] = (float)t[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)p[j];
    }
}

template <class T>
__device__ __forceinline__ void store8(void* base, int64_t at, bool vec, const float (&v)[8]) {
    T* p = static_cast<T*>(base) + at;
    if (vec) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            vec_t t;
#pragma unroll
            for (int j = 0; j < N; ++j) t[j] = (T)v[i * N + j];
            reinterpret_cast<vec_t*>(p)[i] = t;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (T)v[j];
    }
}

// Nearest e4m3 value, ties to even; past the largest finite value (448) that value, NaN stays NaN.
__device__ __forceinline__ float clamp_e4m3(float v) { return v > 448.0f ? 448.0f : v < -448.0f ? -448.0f : v; }
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(a), clamp_e4m3(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(c), clamp_e4m3(d), w, true);
}

// A granule of the cache: eight elements at element index `at` (a multiple of eight).
template <class C>
__device__ __forceinline__ void store_granule(void* cache, int64_t at, const float (&v)[8]) {
    if constexpr (std::is_same_v<C, Fp8>) {
        uint2 w = {pack4_e4m3(v[0], v[1], v[2], v[3]), pack4_e4m3(v[4], v[5], v[6], v[7])};
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + at) = w;
    } else {
        store8<C>(cache, at, true, v);
    }
}

template <class C>
__device__ __forceinline__ void store_one(void* cache, int64_t at, float v) {
    if constexpr (std::is_same_v<C, Fp8>)
        static_cast<uint8_t*>(cache)[at] = (uint8_t)pack4_e4m3(v, v, v, v);
    else
        static_cast<C*>(cache)[at] = (C)v;
}

// The angles of a lane's pairs at one token.
struct Turn {
    float cos[8], sin[8];
};

__device__ __forceinline__ int axis_of(const RopeArgs& r, int pair) {
    if (r.interleaved) {
        const int a = pair % 3;
        return a == 1 ? (pair < 3 * r.sections[1] ? 1 : 0) : a == 2 ? (pair < 3 * r.sections[2] ? 2 : 0) : 0;
    }
    int end = r.sections[0];
    if (pair < end) return 0;
    end += r.sections[1];
    if (pair < end) return 1;
    return pair < end + r.sections[2] ? 2 : 3;
}

// Columns col..col+7 (col < rot_dim) of a row of token t.
__device__ __forceinline__ Turn turn_of(const RopeArgs& r, int n_tokens, int t, int col) {
    Turn out;
    const int half = r.rot_dim / 2;
    const int pair = col < half ? col : col - half;
    int pos[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) pos[a] = a < r.n_axes ? r.positions[(int64_t)a * n_tokens + t] : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int p = pos[0];
        if (r.n_axes > 1) {
            const int a = axis_of(r, pair + j);
            p = a == 0 ? pos[0] : a == 1 ? pos[1] : a == 2 ? pos[2] : pos[3];
        }
        const uint64_t turns = (uint64_t)(int64_t)p * r.freq[pair + j];
        // the top 32 bits as a signed fraction of half a turn: the fp32 rounding is 2^-25 of it
        sincospif((float)(int32_t)(turns >> 32) * 0x1p-31f, &out.sin[j], &out.cos[j]);
    }
    return out;
}

// Norm and rotation of a row of which this lane holds columns li*8..+7 in v;
// the row's `lanes` (power of two) lanes call it together, lanes past the row
// (or on no row) with v = 0.
__device__ __forceinline__ void norm_and_turn(const RopeArgs& r, int dim, int lanes, int li, const Turn& turn,
                                              float (&v)[8]) {
    if (r.norm) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
        for (int o = lanes / 2; o; o >>= 1) sum += __shfl_xor(sum, o);
        const float inv = 1.0f / sqrtf(sum / (float)dim + r.eps);
        if (li * 8 < dim) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = v[j] * inv * r.norm[li * 8 + j];
        }
    }
    if (r.freq) {
        const int step = r.rot_dim / 16;  // lanes from a column to its pair's other half
        const int lane = threadIdx.x & 63;
        const bool low = li < step, in = li < 2 * step;
        const int from = in ? (low ? lane + step : lane - step) : lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float other = __shfl(v[j], from);
            if (in) v[j] = low ? v[j] * turn.cos[j] - other * turn.sin[j] : v[j] * turn.cos[j] + other * turn.sin[j];
        }
    }
}

// Workgroups of four waves; `lanes` lanes a row.  An item is a token with
// `per_item` heads, which share the angles.
template <class TI, class TO>
__global__ __launch_bounds__(256) void rotate_kernel(HeadsView x, HeadsView y, int n_tokens, int heads, int dim,
                                                     int lanes, int per_item, RopeArgs rope) {
    const int lane = threadIdx.x & 63;
    const int li = lane & (lanes - 1);
    const int groups = (heads + per_item - 1) / per_item;
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
    const int64_t t64 = item / groups;
    const bool live = t64 < n_tokens && li * 8 < dim;
    const int t = live ? (int)t64 : 0;
    const int h0 = (int)(item - t64 * groups) * per_item;
    Turn turn = {};
    if (rope.freq && live && li * 8 < rope.rot_dim) turn = turn_of(rope, n_tokens, t, li * 8);
    for (int h = h0; h < h0 + per_item; ++h) {
        const bool on = live && h < heads;
        float v[8] = {};
        if (on) load8<TI>(x.data, t * x.token_stride + h * x.head_stride + li * 8, x.vec, v);
        norm_and_turn(rope, dim, lanes, li, turn, v);
        if (on) store8<TO>(y.data, t * y.token_stride + h * y.head_stride + li * 8, y.vec, v);
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

// blockIdx.y 0: keys, 1: values.  An item is one head's row of a token; the
// rows of a wave are consecutive tokens of a head, whose 16-byte granules of a
// key page are neighbours.
//
// A value page holds eight tokens of a column together, so a single token's
// row is dim elements at a stride of eight.  Where all eight tokens of such a
// granule are in this call, in order (a prompt), the token of the first slot
// reads the eight rows and writes whole granules, and the other seven write
// nothing; which is the case each row sees from the eight slots around its own.
template <class TI, class C>
__global__ __launch_bounds__(256) void kv_append_kernel(qw35_hip_kv_cache cache, HeadsView k, HeadsView v,
                                                        int n_tokens, const int64_t* slots, int lanes, RopeArgs rope) {
    const int lane = threadIdx.x & 63;
    const int li = lane & (lanes - 1);
    const int dim = (int)cache.head_dim, heads = (int)cache.kv_heads, page = (int)cache.page_size;
    const int64_t n_slots = (int64_t)cache.n_pages * page;
    const bool small = n_slots <= 0xffffffffll;
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
    const int64_t h64 = item / n_tokens;
    const int t = (int)(item - h64 * n_tokens);
    const int64_t slot = h64 < heads ? slots[t] : -1;
    const bool live = slot >= 0 && slot < n_slots;
    const int h = live ? (int)h64 : 0;
    const Slot s = live ? slot_of(slot, page, small) : Slot{0, 0};
    const int64_t base = (s.page * heads + h) * ((int64_t)page * dim);
    float x[8] = {};
    if (blockIdx.y == 0) {
        Turn turn = {};
        if (live) {
            load8<TI>(k.data, t * k.token_stride + h * k.head_stride + li * 8, k.vec, x);
            if (rope.freq && li * 8 < rope.rot_dim) turn = turn_of(rope, n_tokens, t, li * 8);
        }
        norm_and_turn(rope, dim, lanes, li, turn, x);
        if (!live) return;
        if constexpr (std::is_same_v<C, Fp8>) {
            const float scale = cache.k_scale ? cache.k_scale[h] : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] /= scale;
        }
        store_granule<C>(cache.k, base + (int64_t)(s.at / 32) * 32 * dim + li * 256 + (s.at & 31) * 8, x);
        return;
    }
    float scale = 1.0f;
    if constexpr (std::is_same_v<C, Fp8>) {
        if (cache.v_scale) scale = cache.v_scale[h];
    }
    // the slots of this row's granule: lane j of the row looks at its j-th token
    const int first = t - (s.at & 7);
    bool mine = false;
    if (live && li < 8) {
        const int i = first + li;
        mine = i >= 0 && i < n_tokens && slots[i] == slot - (s.at & 7) + li;
    }
    const uint64_t votes = __ballot(mine) >> (lane & ~(lanes - 1));
    if (!live) return;
    const int64_t at = base + (int64_t)(s.at / 8) * 8 * dim + li * 64;
    if ((votes & 0xff) == 0xff) {
        if (s.at & 7) return;
        float w[8][8];  // [column][token]
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            load8<TI>(v.data, (t + i) * v.token_stride + h * v.head_stride + li * 8, v.vec, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j][i] = std::is_same_v<C, Fp8> ? x[j] / scale : x[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) store_granule<C>(cache.v, at + j * 8, w[j]);
        return;
    }
    load8<TI>(v.data, t * v.token_stride + h * v.head_stride + li * 8, v.vec, x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        store_one<C>(cache.v, at + j * 8 + (s.at & 7), std::is_same_v<C, Fp8> ? x[j] / scale : x[j]);
}

// Lanes of a row: the power of two that holds dim / 8.
int row_lanes(int dim) {
    int lanes = 1;
    while (lanes * 8 < dim) lanes *= 2;
    return lanes;
}

template <class TI, class TO>
hipError_t rotate_as(const HeadsView& x, const HeadsView& y, int n_tokens, int heads, int dim, const RopeArgs& rope,
                     hipStream_t stream) {
    const int lanes = row_lanes(dim);
    const int per_item = 1;
    const int64_t items = (int64_t)n_tokens * ((heads + per_item - 1) / per_item);
    const int64_t grid = (items * lanes + 255) / 256;
    rotate_kernel<TI, TO><<<dim3((unsigned)grid), 256, 0, stream>>>(x, y, n_tokens, heads, dim, lanes, per_item, rope);
    return hipGetLastError();
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

template <class TI, class C>
hipError_t append_as(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n,
                     const int64_t* slots, const RopeArgs& rope, hipStream_t stream) {
    const int lanes = row_lanes((int)cache.head_dim);
    const int64_t grid = ((int64_t)n * cache.kv_heads * lanes + 255) / 256;
    kv_append_kernel<TI, C><<<dim3((unsigned)grid, 2), 256, 0, stream>>>(cache, k, v, n, slots, lanes, rope);
    return hipGetLastError();
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
