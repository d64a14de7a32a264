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
    // The same of x inv, within the codes and numbers all: one instruction each.
    static __device__ __forceinline__ uint32_t pack4_fits(const float* x, float inv) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(uint32_t, fmaf(x[i], inv, 12582912.0f));
        const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
        return lo | hi;
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
    static __device__ __forceinline__ uint32_t pack4_fits(const float* x, float inv) {
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
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

// Workgroups that a launch is not cut below by giving each more heads: a workgroup
// of several looks through the slots once for them and has the next head's rows on
// their way, and needs others beside it.  Which number is best depends on how the
// workgroups of a shape fill the compute units; 1024 is within 28% of it here.  Prompts from
// a block's beginning / from its middle, int8, us:
//   tokens x heads x columns       512           1024          2048
//   8192 x 8 x 128, bf16           26.6 / 26.9   21.2 / 28.3   26.4 / 28.1
//   8192 x 4 x 256, bf16           23.8 / 23.7   24.4 / 25.8   28.5 / 28.9
//   8192 x 4 x 256, fp32           26.8 / 25.7   29.7 / 30.3   37.0 / 33.8
//   16384 x 8 x 128, bf16          34.0 / 49.3   33.9 / 49.3   45.3 / 54.8
//   4096 x 8 x 128, bf16           16.2 / 15.5   14.5 / 14.5   17.9 / 17.9
//   5000 x 8 x 64, bf16            11.7 / 11.5   14.7 / 14.7   18.5 / 18.6
constexpr int kLeastGroups = 1024;
// Places of a call, up to 32 tokens each, whose blocks are looked for apart: a
// prompt has a block for every 32 tokens, a decode step one for each.  A prompt's
// tokens / as many scattered ones, 4 heads x 256, us:
//   places       16           32            64 (taken)    128
//   128 tokens   7.5 / 9.3    7.6 / 7.1     7.6 / 7.4     11 / 11
//   256          7.6 / 16     7.6 / 9.9     7.7 / 8.0     8.5 / 12
//   512          7.9 / 29     7.8 / 17      8.2 / 12      8.8 / 13
//   1024         8.2 / 32     8.2 / 32      8.2 / 20      9.1 / 21
//   8192         30 / 134     30 / 134      30 / 133      30 / 134
constexpr int kMostLooks = 64;

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
    int per;             // tokens whose blocks a workgroup looks for (a power of two up to 32)
    int heads_per;       // heads of a workgroup
    RopeArgs rope;
};

// What a workgroup shares.
template <int D>
struct BlockShared {
    int src[4][32];     // of the block's tokens: which of the call it is (-1: none); a list, or a list a wave
    uint32_t top[2][4];  // the waves' largest magnitudes, of this head and the last
    float before[2];    // the scale before
    uint32_t count[4][2];  // the waves' counts of the tokens of a block, or of four by halves
    union {
        uint2 codes[32][D / 8 + 1];         // of values, on their way to eight tokens of a column
        alignas(16) float angles[32][D / 2 + 2][2];  // of keys: cosine and sine of each pair (the pad: rows apart in the banks)
    };
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

// The largest of every thread's magnitudes (as fp32 bits), and thread 0's `before`.
template <int D>
__device__ __forceinline__ uint32_t agree(BlockShared<D>& sh, int parity, uint32_t m, float& before) {
    m = __builtin_bit_cast(uint32_t, wave_max_abs(__builtin_bit_cast(float, m)));
    if ((threadIdx.x & 63) == 0) sh.top[parity][threadIdx.x >> 6] = m;
    if (threadIdx.x == 0) sh.before[parity] = before;
    __syncthreads();
    before = sh.before[parity];
    const uint32_t a = dpp_max_u32(sh.top[parity][0], sh.top[parity][1]), b = dpp_max_u32(sh.top[parity][2], sh.top[parity][3]);
    return dpp_max_u32(a, b);
}

constexpr uint32_t kInfinity = 0x7f800000u;

__device__ __forceinline__ uint32_t largest(const float (&x)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = dpp_max_u32(m, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
    return m;
}

// For a block with infinities or NaN: the largest of eight numbers that are finite; infinities become fp32's
// largest number, and so the largest code (and zero under a scale of zero, which a block without a number but zeros has).
__device__ __forceinline__ uint32_t largest_finite(float (&x)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t v = __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu;
        m = v < kInfinity && v > m ? v : m;
        if (v == kInfinity) x[j] = copysignf(0x1.fffffep127f, x[j]);
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
__device__ __forceinline__ uint2 pack8(const float (&x)[8], float inv, bool fits) {
    if (fits) return {Codes<C>::pack4_fits(x, inv), Codes<C>::pack4_fits(x + 4, inv)};
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

// A block of a call: its tokens there (-1: none) in the list, and which they are as bits.
struct Found {
    const int* src;
    uint32_t written;
    int64_t block;
};

__device__ __forceinline__ int64_t of_lane(int64_t v, int l) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, l));
}

// A token of the call in a lane.
struct Near {
    int token;
    int64_t slot, block;  // -1: none
};
__device__ __forceinline__ Near near(const BlockAppend& a, int token) {
    Near x = {token, token >= a.t0 && token < a.t1 ? a.slots[token] : -1, -1};
    if (x.slot >= 0 && x.slot < (int64_t)a.cache.n_pages * a.cache.page_size) x.block = x.slot >> 5;
    return x;
}

// The lanes' tokens of a block, in a wave's list.
__device__ __forceinline__ Found found(int* src, const Near& x, int64_t block) {
    const int lane = threadIdx.x & 63;
    if (lane < 32) src[lane] = -1;
    __builtin_amdgcn_wave_barrier();
    if (x.block == block) atomicMax(&src[x.slot & 31], x.token);
    __builtin_amdgcn_wave_barrier();
    return {src, (uint32_t)__ballot(src[lane & 31] >= 0), block};
}

// How many tokens of each of some blocks (as the halves of slots) the call has: this thread's share.
template <int kBlocks>
__device__ __forceinline__ void look(const BlockAppend& a, const uint32_t (&lo)[kBlocks], const uint32_t (&hi)[kBlocks],
                                     int (&count)[kBlocks]) {
    typedef uint32_t pair_t __attribute__((ext_vector_type(4), aligned(8)));
    constexpr int kAhead = 4;  // loads on their way together
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) count[b] = 0;
    for (int j0 = a.t0 + 2 * (int)threadIdx.x; j0 < a.t1; j0 += 512 * kAhead) {
        pair_t s[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int j = j0 + 512 * i;
            s[i] = pair_t{~0u, ~0u, ~0u, ~0u};
            if (j + 1 < a.t1) s[i] = *reinterpret_cast<const pair_t*>(a.slots + j);
            else if (j < a.t1) s[i] = pair_t{(uint32_t)a.slots[j], (uint32_t)(a.slots[j] >> 32), ~0u, ~0u};
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                count[b] += ((s[i][0] ^ lo[b]) & ~31u | (s[i][1] ^ hi[b])) == 0;
                count[b] += ((s[i][2] ^ lo[b]) & ~31u | (s[i][3] ^ hi[b])) == 0;
            }
    }
}

// The blocks that a workgroup writes: those of which one of its `per` tokens is
// the call's first.  Each has one writer, in whatever order the tokens come (of two
// with the same slot the last counts), so results do not depend on timing.
//   kFew, of up to 64 tokens: every wave has them all, a lane each, and a workgroup
// one.  (In the general form, whose paths wait for what they have loaded where they
// meet, 8 tokens took 8.0 us for 6.7.)
//   Else a wave has the 64 tokens before the workgroup's and the 64 from them on, two
// a lane.  A block whose first token there is the workgroup's begins with those
// (`start`), and all slots are looked through meanwhile; if there are more of the
// block it gives way to an earlier one, or begins again with all of them.
//   Several blocks of one token, as of a batch's decode step, are looked for and
// written four at a time, a wave each (`start_one`, `write_one`): 512 sequences x 4
// heads of 256 take 12 us, and 32 one after the other by the workgroup, prompts
// 0.4 us more for it.
template <bool kFew, int D, class S, class W, class S1, class W1>
__device__ __forceinline__ void each_block(const BlockAppend& a, BlockShared<D>& sh, S start, W write, S1 start_one,
                                           W1 write_one) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* const src = sh.src[wave];
    if constexpr (kFew) {
        const Near mine = near(a, a.t0 + lane);
        const int first = (int)blockIdx.x;
        const int64_t block = of_lane(mine.block, first);
        if (block < 0 || __ballot(mine.block == block) & ((1ull << first) - 1)) return;
        const Found f = found(src, mine, block);
        start(f);
        write(f);
        return;
    }
    // (workgroups begin where a prompt's blocks do: the first may have begun before it)
    const int base = a.t0 + (int)blockIdx.x * a.per - (a.per > 1 ? (int)(a.slots[a.t0] & (a.per - 1)) : 0);
    const Near below = near(a, base - 64 + lane), here = near(a, base + lane);
    const int64_t last = (int64_t)((uint64_t)(uint32_t)__shfl_up((int)(here.block >> 32), 1) << 32 | (uint32_t)__shfl_up((int)here.block, 1));
    uint32_t runs = (uint32_t)__ballot(lane < a.per && here.block >= 0 && (lane == 0 || here.block != last));
    uint32_t ones = 0;
    if (runs & (runs - 1))
        for (uint32_t left = runs; left; left &= left - 1) {
            const int l = __builtin_ctz(left);
            const int64_t block = of_lane(here.block, l);
            if (!__ballot(below.block == block) && __ballot(here.block == block) == 1ull << l) ones |= 1u << l;
        }
    if (ones & (ones - 1)) {
        runs &= ~ones;
        while (ones) {
            const int w = __builtin_amdgcn_readfirstlane(wave);
            int at[4], n[4], mine = -1;
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                at[i] = ones ? __builtin_ctz(ones) : -1;
                ones &= ones - 1;
                const int64_t block = at[i] >= 0 ? of_lane(here.block, at[i]) : -1;
                lo[i] = (uint32_t)block << 5;
                hi[i] = (uint32_t)(block >> 27);
                if (i == w) mine = at[i];
            }
            const int64_t slot = mine >= 0 ? of_lane(here.slot, mine) : -1;
            if (mine >= 0) start_one(base + mine, slot);
            look<4>(a, lo, hi, n);
            static_assert(kAppendSlice + 2048 < 1 << 16, "a count, and of no block negative slots and those past the end");
            uint32_t halves[2] = {(uint32_t)(n[0] | n[1] << 16), (uint32_t)(n[2] | n[3] << 16)};
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                halves[0] += __shfl_xor(halves[0], o);
                halves[1] += __shfl_xor(halves[1], o);
            }
            if (lane < 2) sh.count[wave][lane] = halves[lane];
            __syncthreads();
            uint32_t all[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all[0] += sh.count[i][0];
                all[1] += sh.count[i][1];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool one = (all[i / 2] >> i % 2 * 16 & 0xffff) == 1;
                if (at[i] >= 0 && !one) runs |= 1u << at[i];  // others lie elsewhere in the call
                if (i == w && one && mine >= 0) write_one(base + mine, slot);
            }
            __syncthreads();  // (the counts are read, and what the waves shared)
        }
    }
    while (runs) {
        const int l = __builtin_ctz(runs);
        runs &= runs - 1;
        const int64_t block = of_lane(here.block, l);
        const uint64_t before = __ballot(below.block == block), from = __ballot(here.block == block);
        if (before || from & ((1ull << l) - 1)) continue;
        Found f = found(src, here, block);
        start(f);
        // how many tokens of the block the call has
        int counts[1];
        look<1>(a, {(uint32_t)block << 5}, {(uint32_t)(block >> 27)}, counts);
        int count = counts[0];
#pragma unroll
        for (int o = 1; o < 64; o *= 2) count += __shfl_xor(count, o);
        if (lane == 0) sh.count[wave][0] = (uint32_t)count;
        __syncthreads();
        count = (int)(sh.count[0][0] + sh.count[1][0] + sh.count[2][0] + sh.count[3][0]);
        if (count != __popcll(from)) {  // some lie elsewhere in the call
            int* const all = sh.src[0];
            if (tid < 32) all[tid] = -1;
            __syncthreads();
            int earlier = 0;
            for (int j = a.t0 + tid; j < a.t1; j += 256) {
                const int64_t s = a.slots[j];
                if (s >> 5 != block) continue;
                if (j < base) earlier = 1;
                else atomicMax(&all[s & 31], j);
            }
            if (__syncthreads_or(earlier)) continue;
            f = Found{all, (uint32_t)__ballot(all[lane & 31] >= 0), block};
            start(f);
        }
        write(f);
        __syncthreads();  // (the lists are read)
    }
}

__device__ __forceinline__ void positions_of(const RopeArgs& r, int n_tokens, int t, int (&pos)[4]) {
#pragma unroll
    for (int a = 0; a < 4; ++a) pos[a] = a < r.n_axes ? r.positions[(int64_t)a * n_tokens + t] : 0;
}

// What turn_of and norm_and_turn (rope_rows.h) compute, of a pair, and of rows with
// the norm's weights and the angles at hand.  An angle's bits past fp32's are added to
// first order, since every error of a key is a chance of the code beside the right one.
__device__ __forceinline__ void turn_pair(const RopeArgs& r, const int (&pos)[4], int pair, uint64_t freq, float (&to)[2]) {
    int p = pos[0];
    if (r.n_axes > 1) {
        const int a = axis_of(r, pair);
        p = a == 0 ? pos[0] : a == 1 ? pos[1] : a == 2 ? pos[2] : pos[3];
    }
    const uint64_t turns = (uint64_t)(int64_t)p * freq;
    float sin, cos;
    sincospif((float)((int32_t)(turns >> 32) & ~0x7f) * 0x1p-31f, &sin, &cos);  // (24 bits and a sign: exact)
    const float rest = (float)(uint32_t)(turns >> 7) * (3.14159265f * 0x1p-56f);
    to[0] = fmaf(-rest, sin, cos);
    to[1] = fmaf(rest, cos, sin);
}

template <int D, int kRows>
__device__ __forceinline__ void norm_and_turn_rows(const RopeArgs& r, int li, int row0, const float (&weight)[8],
                                                   const BlockShared<D>& sh, float (&v)[kRows][8]) {
    constexpr int kLanes = D / 8, kStep = 256 / kLanes;
    if (r.norm) {
        float sum[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[i] = fmaf(v[i][j], v[i][j], sum[i]);
        }
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < kRows; ++i) sum[i] += __shfl_xor(sum[i], o);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float inv = 1.0f / sqrtf(sum[i] / (float)(8 * kLanes) + r.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * weight[j];
        }
    }
    if (r.freq) {
        const int step = r.rot_dim / 16;  // lanes from a column to its pair's other half
        const int lane = threadIdx.x & 63;
        const bool low = li < step, in = li < 2 * step;
        const int from = in ? (low ? lane + step : lane - step) : lane, pair = low ? li * 8 : (li - step) * 8;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float4_t* const angles = reinterpret_cast<const float4_t*>(sh.angles[row0 + i * kStep][in ? pair : 0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4_t two = angles[k];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mine = v[i][2 * k + e], other = __shfl(mine, from);
                    const float cos = two[2 * e], sin = low ? -two[2 * e + 1] : two[2 * e + 1];
                    if (in) v[i][2 * k + e] = mine * cos + other * sin;
                }
            }
            asm volatile("" ::: "memory");  // (a row's angles at a time)
        }
    }
}

// A thread holds eight columns of D / 64 of the block's tokens; the next head's
// are on their way while one is written.
template <class TI, class C, int D, bool kFew, bool kValues>
__device__ __forceinline__ void append_blocks(const BlockAppend& a, BlockShared<D>& sh) {
    constexpr int kLanes = D / 8, kRows = D / 64, kStep = 256 / kLanes;
    const int tid = threadIdx.x, li = tid % kLanes, row0 = tid / kLanes;
    const int heads = (int)a.cache.kv_heads, blocks = (int)a.cache.page_size / 32;
    const int h0 = ((int)blockIdx.y >> 1) * a.heads_per, h1 = h0 + a.heads_per < heads ? h0 + a.heads_per : heads;
    const HeadsView& x_view = kValues ? a.v : a.k;
    uint8_t* const pages = static_cast<uint8_t*>(kValues ? a.cache.v : a.cache.k);
    float* const scales = const_cast<float*>(kValues ? a.cache.v_scale : a.cache.k_scale);  // (the cache's, written here)
    // values: this thread's granules are four columns of eight tokens
    const int quad = tid % (D / 4), octet = tid / (D / 4);
    // of the block that is written, and of its next head
    bool anew = false, merge = false;  // merge: with granules that hold other tokens
    int64_t tile0 = 0;
    uint32_t mine = 0;
    int src[kRows];
    float next[kRows][8], before_next = 0.0f;
    uint4_t old_next[2] = {};
    auto load = [&](int h) {
        const int64_t tile = tile0 + (int64_t)h * blocks;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
            for (int j = 0; j < 8; ++j) next[r][j] = 0.0f;
            if (src[r] >= 0)
                load8<TI>(x_view.data, src[r] * x_view.token_stride + h * x_view.head_stride + li * 8, x_view.vec, next[r]);
        }
        before_next = tid == 0 && !anew ? scales[tile] : 0.0f;
        if (merge) {
            const uint4_t* const from = reinterpret_cast<const uint4_t*>(pages + tile * (32 * D) + octet * 8 * D + quad * 32);
            old_next[0] = from[0];
            old_next[1] = from[1];
        }
    };
    float weight[8] = {};
    if (!kValues && a.rope.norm) {
#pragma unroll
        for (int j = 0; j < 8; ++j) weight[j] = a.rope.norm[li * 8 + j];
    }
    auto start = [&](const Found& f) {
        anew = f.written & 1;
        const int64_t page = f.block / blocks;
        tile0 = page * heads * blocks + (f.block - page * blocks);
        mine = octet < 4 ? f.written >> octet * 8 & 0xff : 0xff;
        merge = kValues && !anew && mine != 0xff;
#pragma unroll
        for (int r = 0; r < kRows; ++r) src[r] = f.src[row0 + r * kStep];
        load(h0);
    };
    // The token of a block that the call has no other of, by a wave: as many heads at a time as its lanes have room for,
    // eight columns a lane.
    constexpr int kHeads = 64 / kLanes;
    const int lane = tid & 63, wave = tid >> 6, group = lane / kLanes;
    int64_t one_tile = 0;
    float one[8], one_before = 0.0f;
    auto load_one = [&](int token, int h) {
        const bool in = h < h1;
#pragma unroll
        for (int j = 0; j < 8; ++j) one[j] = 0.0f;
        if (in) load8<TI>(x_view.data, token * x_view.token_stride + h * x_view.head_stride + li * 8, x_view.vec, one);
        one_before = in ? scales[one_tile + (int64_t)h * blocks] : 0.0f;
    };
    auto start_one = [&](int token, int64_t slot) {
        const int64_t block = slot >> 5, page = block / blocks;
        one_tile = page * heads * blocks + (block - page * blocks);
        load_one(token, h0 + group);
    };
    auto write_one = [&](int token, int64_t slot) {
        if (!kValues && a.rope.freq) {
            int pos[4];
            positions_of(a.rope, a.n_tokens, token, pos);
            for (int p = lane; p < a.rope.rot_dim / 2; p += 64) turn_pair(a.rope, pos, p, a.rope.freq[p], sh.angles[wave][p]);
            __builtin_amdgcn_wave_barrier();
        }
        const int row = (int)slot & 31;
        for (int hb = h0; hb < h1; hb += kHeads) {
            const int h = hb + group;
            if (hb != h0) load_one(token, h);
            float x[1][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[0][j] = one[j];
            if constexpr (!kValues) norm_and_turn_rows<D>(a.rope, li, wave, weight, sh, x);
            uint32_t m = largest(x[0], 0);
            for (int o = kLanes / 2; o; o >>= 1) m = dpp_max_u32(m, (uint32_t)__shfl_xor((int)m, o));
            const bool finite = m < kInfinity;
            if (__any(!finite)) {
                uint32_t f = finite ? m : largest_finite(x[0], 0);
                for (int o = kLanes / 2; o; o >>= 1) f = dpp_max_u32(f, (uint32_t)__shfl_xor((int)f, o));
                m = f;
            }
            if (h >= h1) continue;
            const int64_t tile = one_tile + (int64_t)h * blocks;
            uint8_t* const codes = pages + tile * (32 * D);
            const bool first = row == 0;
            const Scale s = scale_of<C>(first ? 0.0f : one_before, first, __builtin_bit_cast(float, m));
            const float inv = s.now > 0.0f ? 1.0f / s.now : 0.0f;
            const bool rewrite = first || s.shrink != 1.0f;
            const uint2 w = pack8<C>(x[0], inv, finite);
            // the lane's columns of the block: of keys a granule a token, of values a granule a column and eight tokens
            if (rewrite) {
                uint4_t* const at = reinterpret_cast<uint4_t*>(codes + li * (kValues ? 64 : 256));
                constexpr int kStep = kValues ? D / 2 : 4;  // (of values from one octet to the next, in four)
                for (int i = 0; i < 4; ++i) {
                    uint4_t* const to = at + i * (kValues ? kStep : 4);
                    uint4_t old[4] = {};
                    if (s.shrink > 0.0f) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) old[e] = to[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) old[e][c] = again<C>(old[e][c], s.shrink);
                        to[e] = old[e];
                    }
                }
            }
            if constexpr (!kValues) {
                *reinterpret_cast<uint2*>(codes + li * 256 + row * 8) = w;
            } else {
                uint8_t* const to = codes + row / 8 * (8 * D) + li * 64 + row % 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j * 8] = (uint8_t)((j < 4 ? w.x : w.y) >> j % 4 * 8);
            }
            if (li == 0 && s.changed) scales[tile] = s.now;
        }
    };
    each_block<kFew, D>(a, sh, start, [&](const Found& f) {
        if constexpr (!kValues) {
            // the block's angles, by eight threads a token, four of each on their way together (by the lanes that take
            // them they are 12 us of a chunk of 249 tokens x 256 columns, of which 64 turn)
            const int half = a.rope.rot_dim / 2, token = f.src[tid >> 3];
            if (a.rope.freq && token >= 0) {
                int pos[4];
                positions_of(a.rope, a.n_tokens, token, pos);
                for (int p = tid & 7; p < half; p += 32) {
                    uint64_t freq[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) freq[i] = a.rope.freq[p + 8 * i < half ? p + 8 * i : p];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (p + 8 * i < half) turn_pair(a.rope, pos, p + 8 * i, freq[i], sh.angles[tid >> 3][p + 8 * i]);
                }
            }
            __syncthreads();
        }
        for (int h = h0; h < h1; ++h) {
            const int64_t tile = tile0 + (int64_t)h * blocks;
            uint8_t* const codes = pages + tile * (32 * D);
            float x[kRows][8];
            uint32_t m = 0;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[r][j] = next[r][j];
            float before = before_next;
            const uint4_t old[2] = {old_next[0], old_next[1]};
            if (h + 1 < h1) load(h + 1);
            if constexpr (!kValues) norm_and_turn_rows<D>(a.rope, li, row0, weight, sh, x);
#pragma unroll
            for (int r = 0; r < kRows; ++r) m = src[r] >= 0 ? largest(x[r], m) : m;
            m = agree<D>(sh, h & 1, m, before);
            const bool finite = m < kInfinity;
            if (!finite) {
                m = 0;
#pragma unroll
                for (int r = 0; r < kRows; ++r) m = src[r] >= 0 ? largest_finite(x[r], m) : m;
                __syncthreads();
                m = agree<D>(sh, h & 1, m, before);
            }
            const Scale s = scale_of<C>(before, anew, __builtin_bit_cast(float, m));
            const float inv = s.now > 0.0f ? 1.0f / s.now : 0.0f;
            const bool rewrite = anew || s.shrink != 1.0f;  // the tokens that the call does not write change too
            if constexpr (!kValues) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    uint2* const at = reinterpret_cast<uint2*>(codes + li * 256 + (row0 + r * kStep) * 8);
                    uint2 w = pack8<C>(x[r], inv, finite);
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
                for (int r = 0; r < kRows; ++r) sh.codes[row0 + r * kStep][li] = pack8<C>(x[r], inv, finite);
                __syncthreads();
                if (octet < 4 && (mine || rewrite)) {
                    uint32_t w[2][4], g[2][4];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[j / 4][j % 4] = reinterpret_cast<const uint32_t*>(sh.codes[octet * 8 + j])[quad];
                    transpose4(w[0], g[0]);
                    transpose4(w[1], g[1]);
                    uint4_t out[2] = {{g[0][0], g[1][0], g[0][1], g[1][1]}, {g[0][2], g[1][2], g[0][3], g[1][3]}};
                    if (merge) {
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
                    uint4_t* const to = reinterpret_cast<uint4_t*>(codes + octet * 8 * D + quad * 32);
                    to[0] = out[0];
                    to[1] = out[1];
                }
            }
            if (tid == 0 && s.changed) scales[tile] = s.now;
        }
    }, start_one, write_one);
}

// blockIdx.y: even keys, odd values of a group of heads.
//   Bytes are the least of it: a call of few tokens is one chain of slots, rows, angles,
// the largest, codes (8 tokens x 4 heads of 256, int8: 6.8 us, of 249: 9.6), and one of
// many the chain of a head after the other (8192 x 8 heads of 128, bf16: 22.7 us, 50 MB
// at 2.2 TB/s).  So a workgroup is a block, whose 32 rows of a head are all in
// registers between the reading, the largest and the codes, each read and written
// once; registers allow four of them a compute unit (three of 256 columns, without
// spills).
template <class TI, class C, int D, bool kFew>
__global__ __launch_bounds__(256, D == 256 ? 3 : 4) void kv_append_blocks_kernel(BlockAppend a) {
    __shared__ BlockShared<D> sh;
    if (blockIdx.y & 1) append_blocks<TI, C, D, kFew, true>(a, sh);
    else append_blocks<TI, C, D, kFew, false>(a, sh);
}

template <class TI, class C, int D>
hipError_t append_dim(BlockAppend a, int n, hipStream_t stream) {
    const int heads = (int)a.cache.kv_heads;
    for (a.t0 = 0; a.t0 < n; a.t0 = a.t1) {
        const int count = n - a.t0 < kAppendSlice ? n - a.t0 : kAppendSlice;
        a.t1 = a.t0 + count;
        // A prompt has a block for every 32 tokens, a decode step one for each: workgroups for up to kMostLooks places
        // keep both apart enough.
        a.per = 1;
        while (a.per < 32 && count > kMostLooks * a.per) a.per *= 2;
        const int chunks = (count + 2 * (a.per - 1)) / a.per;  // (the first may begin before the tokens)
        // (every workgroup of several heads saves one a look through the slots)
        a.heads_per = 1;
        while (count > 64 && a.heads_per < heads && (int64_t)chunks * 2 * ((heads + 2 * a.heads_per - 1) / (2 * a.heads_per)) >= kLeastGroups)
            a.heads_per *= 2;
        const dim3 grid((unsigned)chunks, (unsigned)((heads + a.heads_per - 1) / a.heads_per * 2));
        if (count <= 64) kv_append_blocks_kernel<TI, C, D, true><<<grid, 256, 0, stream>>>(a);
        else kv_append_blocks_kernel<TI, C, D, false><<<grid, 256, 0, stream>>>(a);
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

// Four consecutive elements of a cache, from where they are or out of a word of 8-bit ones.
template <class C>
struct Four {
    typedef C raw __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ void unpack(raw w, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)w[i];
    }
    static __device__ __forceinline__ float one(const void* cache, int64_t at) { return (float)static_cast<const C*>(cache)[at]; }
};
template <class C>
struct Four8 {
    typedef uint32_t raw;
    static __device__ __forceinline__ void unpack(raw w, float (&v)[4]) { Codes<C>::unpack4(w, v); }
    static __device__ __forceinline__ float one(const void* cache, int64_t at) {
        float v[4];
        unpack(static_cast<const uint8_t*>(cache)[at], v);
        return v[0];
    }
};
template <>
struct Four<Int8> : Four8<Int8> {};
template <>
struct Four<Fp8> : Four8<Fp8> {};

template <class T>
__device__ __forceinline__ void store4(void* base, int64_t at, bool vec, const float (&v)[4]) {
    T* const p = static_cast<T*>(base) + at;
    typedef T vec_t __attribute__((ext_vector_type(4)));
    if (vec) {
        *reinterpret_cast<vec_t*>(p) = vec_t{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = (T)v[i];
    }
}

// Bound by bytes (20011 tokens x 8 heads of 128, e4m3 to bf16: 23.1 us, 123 MB at
// 5.3 TB/s, where a copy of 1 GiB has 5.1; a byte a load took 91).  Of keys a thread has eight columns (a granule of the cache) of
// D / 64 tokens, a workgroup 32 tokens of a head, so that it uses whole lines of
// the granules, which lie token by token.  Of values a thread has four columns of
// eight tokens: where those are the eight of a granule it reads 32 bytes (64 of a
// 16-bit cache) and writes four elements of each token, a row at a time by its lanes.
// The eights are counted from the first token's place in its granule: the values of
// another sequence of the call that does not lie so (seven of eight) are read a byte a
// load (20 sequences of 1000 tokens x 4 heads of 256, int8: 20 us if all lie alike, 53).
template <class C, class TO, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(CacheRead a) {
    const int tid = threadIdx.x, h = (int)blockIdx.y >> 1, heads = (int)a.cache.kv_heads;
    const int64_t n_slots = (int64_t)a.cache.n_pages * a.cache.page_size;
    const bool small = n_slots <= 0xffffffffll;
    const float* const scales = blockIdx.y & 1 ? a.cache.v_scale : a.cache.k_scale;
    struct Place {
        int64_t tile;  // 32 tokens of the head
        float scale;
        int at;        // token of the tile
        bool live;
    };
    auto find = [&](int64_t slot) {
        Place p = {0, 1.0f, (int)(slot & 31), slot >= 0 && slot < n_slots};
        const int blocks = (int)a.cache.page_size / 32;
        const int64_t block = p.live ? slot >> 5 : 0;
        const int64_t page = small ? (int64_t)((uint32_t)block / (uint32_t)blocks) : block / blocks;
        p.tile = (page * heads + h) * blocks + (block - page * blocks);
        if (scales) p.scale = a.by_block ? scales[p.tile] : scales[h];
        return p;
    };
    typedef typename Four<C>::raw raw;
    if ((blockIdx.y & 1) == 0) {
        constexpr int kLanes = D / 8, kRows = D / 64, kStep = 256 / kLanes;
        const int li = tid % kLanes, t0 = (int)blockIdx.x * 32 + tid / kLanes;
        int64_t slot[kRows];
        Place p[kRows];
        raw w[kRows][2];
#pragma unroll
        for (int r = 0; r < kRows; ++r) slot[r] = t0 + r * kStep < a.n_tokens ? a.slots[t0 + r * kStep] : -1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            p[r] = find(slot[r]);
            const raw* const from = static_cast<const raw*>(a.cache.k) + (p[r].tile * (32 * D) + li * 256 + p[r].at * 8) / 4;
            w[r][0] = w[r][1] = raw{};
            if (p[r].live) {
                w[r][0] = from[0];
                w[r][1] = from[1];
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int t = t0 + r * kStep;
            if (t >= a.n_tokens) continue;
            float lo[4], hi[4], x[8];
            Four<C>::unpack(w[r][0], lo);
            Four<C>::unpack(w[r][1], hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = p[r].live ? (j < 4 ? lo[j & 3] : hi[j & 3]) * p[r].scale : 0.0f;
            store8<TO>(a.k.data, t * a.k.token_stride + h * a.k.head_stride + li * 8, a.k.vec, x);
        }
    } else {
        constexpr int kQuads = D / 4, kOctets = 256 / kQuads;
        const int shift = (int)(a.slots[0] & 7);  // where the first token lies in its granule
        const int quad = tid % kQuads, t0 = ((int)blockIdx.x * kOctets + tid / kQuads) * 8 - shift;
        if (t0 >= a.n_tokens) return;
        int64_t slot[8];
        bool whole = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) slot[j] = t0 + j >= 0 && t0 + j < a.n_tokens ? a.slots[t0 + j] : -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) whole &= slot[j] >= 0 && slot[j] < n_slots && slot[j] == slot[0] + j;
        float x[8][4];
        if (whole && (slot[0] & 7) == 0) {
            const Place p = find(slot[0]);
            const raw* const from = static_cast<const raw*>(a.cache.v) + (p.tile * (32 * D) + p.at * D + quad * 32) / 4;
            raw w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = from[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v[4];
                Four<C>::unpack(w[i], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i % 2 * 4 + j][i / 2] = v[j] * p.scale;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Place p = find(slot[j]);
                const int64_t at = p.tile * (32 * D) + p.at / 8 * (8 * D) + quad * 32 + p.at % 8;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = p.live ? Four<C>::one(a.cache.v, at + i * 8) * p.scale : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (t0 + j >= 0 && t0 + j < a.n_tokens)
                store4<TO>(a.v.data, (t0 + j) * a.v.token_stride + h * a.v.head_stride + quad * 4, a.v.vec, x[j]);
    }
}

template <class C, class TO, int D>
hipError_t read_dim(const CacheRead& a, hipStream_t stream) {
    constexpr int kTokens = 8192 / D;  // of values in a workgroup; the first octet may begin before the tokens
    const int keys = (a.n_tokens + 31) / 32, values = (a.n_tokens + 7 + kTokens - 1) / kTokens;
    const dim3 grid((unsigned)(keys > values ? keys : values), a.cache.kv_heads * 2);
    kv_read_kernel<C, TO, D><<<grid, 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <class C, class TO>
hipError_t read_as(const CacheRead& a, hipStream_t stream) {
    switch (a.cache.head_dim) {
        case 64: return read_dim<C, TO, 64>(a, stream);
        case 128: return read_dim<C, TO, 128>(a, stream);
        default: return read_dim<C, TO, 256>(a, stream);
    }
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
