// Rows of heads in registers, a lane with eight columns each: loads and stores of
// any element type, RMS norm and rotation (rope_kv.hip has the mathematics).
#pragma once

#include "attention.h"
#include "qw35_device.h"

namespace qw35 {
namespace rows {

struct Fp8 {};  // e4m3 in a cache page

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

// Lanes of a row: the power of two that holds dim / 8.
inline int row_lanes_log2(int dim) {
    int n = 0;
    while (8 << n < dim) ++n;
    return n;
}

}  // namespace rows
}  // namespace qw35
