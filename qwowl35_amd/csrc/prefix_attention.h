// Attention of a ragged batch over a paged cache whose sequences share a
// prefix: the kernel template (one translation unit per head dimension).
//
// Mathematics.  For a row (new token t of sequence s, query head of group h):
//   out = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q.k_i - m)
// over the tokens i the row sees, in one pass: tiles of 32 tokens keep the
// running maximum m, the sum of p and the sum of p v (fp32), rescaled when m
// rises.  Parts of a row's tokens (the shared prefix, the sequence's own
// pages, pieces of either) give (m, sum p, sum p v) each, joined at the end by
// exp(m_part - m).
//
// Units.  The rows of all sequences read the same prefix, so a prefix unit is
// a kv head and a tile of rows out of the whole batch: the prefix is read once
// for all of them.  An own unit is a kv head, a sequence and a tile of its
// rows.  Every unit's steps of 32-token tiles lie behind each other on one
// line, of which each workgroup takes an equal piece (weighted by what a
// step costs), crossing units where it has to: lengths live on the device, and
// whatever they are the load is even and the grid constant.  A workgroup's
// piece of a unit goes to the partial slot (workgroup + unit), which no other
// piece has; the combine kernel finds a row's slots by the same arithmetic.
//
// Operands.  A tile's scores are S^T = K Q^T and the output O^T = V^T P^T, on
// v_mfma_f32_32x32x16: lane l holds query row l % 32 in S, P and O alike, so
// maximum, sum and rescaling stay in a lane (and its other one of the same
// row).  The cache's granules are the A operands: eight columns of a key, or
// eight tokens of a value column.  Row i of a tile's scores is the token whose
// number is i with bits 2 and 3 exchanged, which leaves the scores a lane holds
// as the tokens of its two value granules: P needs no exchange between lanes.
//
// Data.  Tiles go from HBM to LDS by copies that take no registers, as far
// ahead as the ring has room (128 KB for 256 columns), and from there to the
// matrix instructions: 16 bytes a lane, a wave's reads consecutive.  With up to
// 64 rows in a unit each wave (or pair) has its own tiles, since then a compute
// unit only waits for HBM; more rows share a tile among the four waves, which
// reads it once for 128 or 256 rows.
//
// Rounding.  Scores, maxima, sums and O are fp32.  P is rounded once to the
// cache's 16-bit type for the second product (relative 2^-12 fp16, 2^-9 bf16
// each, signs mixed); e4m3 is exact in either 16-bit type.
#pragma once

#include "attention.h"
#include "qw35_device.h"

namespace qw35 {
namespace attn {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kSeqs = 256;  // sequences kept in LDS
constexpr uint32_t kNoBlock = 0xffffffffu;

typedef float acc_t __attribute__((ext_vector_type(16)));

// Element type of queries and 16-bit caches, and its matrix instruction.
struct Half {
    typedef _Float16 elem;
    typedef half8_t vec8;
    static __device__ __forceinline__ acc_t mfma(vec8 a, vec8 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static constexpr short kInf = 0x7c00;  // bits of +inf
    static __device__ __forceinline__ vec8 from_e4m3(uint2 w) {
        uint4_t r;
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.0f, true));
        return __builtin_bit_cast(vec8, r);
    }
};

struct Bf16 {
    typedef __bf16 elem;
    typedef bf16x8_t vec8;
    static __device__ __forceinline__ acc_t mfma(vec8 a, vec8 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static constexpr short kInf = 0x7f80, kUp = 0x3f80, kDown = 0x4280, kBoth = 0x4282;
    static __device__ __forceinline__ vec8 from_e4m3(uint2 w) {
        uint4_t r;
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, true));
        return __builtin_bit_cast(vec8, r);
    }
};

// What the combine kernel needs of a launch, at the start of the meta block:
// this, then first[n_seqs] (a sequence's first entry), then cost[entries + 1].
struct MetaHead {
    uint64_t head_cost;  // cost of one kv head's entries
    uint64_t per;        // cost of a workgroup's piece
    int entries;
    int pad;
};

__host__ __device__ inline size_t meta_first_at() { return sizeof(MetaHead); }
__host__ __device__ inline size_t meta_cost_at(int n_seqs) {
    return (sizeof(MetaHead) + 4 * (size_t)n_seqs + 7) / 8 * 8;
}

// Floats of a partial slot: rows x dim sums, then rows maxima, then rows sums.
__host__ __device__ inline uint64_t slot_floats(int rows, int dim) { return (uint64_t)rows * (dim + 2); }

// ---- who a row is and what it sees ---------------------------------------------------------------------------------

struct Seq {
    int q0, n;   // its new tokens
    int length;  // its own tokens in the cache
};

// A value that all lanes hold alike, as one the compiler knows to be.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform((int64_t)v); }

// x / d of whole numbers below 2^52.
__device__ __forceinline__ uint64_t quotient(uint64_t x, uint64_t d) {
    uint64_t q = (uint64_t)((double)x / (double)d);
    if (q * d > x) --q;
    return q;
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

__device__ __forceinline__ Seq seq_at(const AttnArgs& a, int s) {
    Seq q;
    q.q0 = a.starts ? clampi(a.starts[s], 0, a.n_tokens) : s;
    const int end = a.starts ? clampi(a.starts[s + 1], q.q0, a.n_tokens) : s + 1;
    q.n = end - q.q0;
    q.length = clampi(a.lengths[s], 0, (int)(a.pages_per_seq * a.page_blocks * 32));
    return q;
}

// The last of n ascending numbers that is at most t (-1: none).
__device__ __forceinline__ int last_at(const int* starts, int n, int t) {
    int lo = 0, hi = n;  // starts[0..lo) <= t < starts[hi..)
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo - 1;
}

// The sequence of new token t: the last whose start is at or before it (-1: none).
__device__ __forceinline__ int seq_of(const AttnArgs& a, int t) {
    return a.starts ? last_at(a.starts, a.n_seqs, t) : t;
}

// The same of a token that the wave's lanes have alike: 64 starts a load.
__device__ __forceinline__ int seq_of_wave(const AttnArgs& a, int t, int lane) {
    if (!a.starts) return t;
    int s = -1;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        const bool at = s0 + lane < a.n_seqs && a.starts[s0 + lane] <= t;
        const uint64_t votes = __ballot(at);
        if (votes) s = s0 + 63 - __builtin_clzll(votes);
        if (votes != ~0ull) break;
    }
    return s;
}

// Tokens [lo, hi) and [0, sink) of a unit's n are seen.
struct Limits {
    int lo, hi, sink;
};

// Of a unit whose first token stands at position `base`, by a token at `pos`.
__device__ __forceinline__ Limits limits_of(const AttnArgs& a, int64_t pos, int base, int n) {
    Limits l;
    const int64_t hi = pos + 1 - base;
    l.hi = hi < 0 ? 0 : hi > n ? n : (int)hi;
    l.lo = 0;
    l.sink = 0;
    if (a.window) {
        const int64_t lo = hi - a.window;
        l.lo = lo < 0 ? 0 : lo > n ? n : (int)lo;
        l.sink = clampi(a.sink - base, 0, l.hi);
    }
    return l;
}

// The 32-token tiles a unit goes through: `sink` ones from 0, then lo..hi-1.
struct Tiles {
    int sink, lo, hi;
    __device__ __forceinline__ int count() const { return sink + hi - lo; }
    __device__ __forceinline__ int at(int v) const { return v < sink ? v : v - sink + lo; }
};

__device__ __forceinline__ Tiles tiles_of(Limits l) {
    Tiles t;
    t.hi = (l.hi + 31) / 32;
    t.lo = l.lo / 32 < t.hi ? l.lo / 32 : t.hi;
    t.sink = (l.sink + 31) / 32 < t.lo ? (l.sink + 31) / 32 : t.lo;
    return t;
}

// Tiles that any row of an own entry sees: up to the last row's position, from the first one's window.
__device__ __forceinline__ Tiles own_tiles(const AttnArgs& a, const Seq& q, int tile) {
    const int rows = q.n * a.group, r0 = tile * a.plan.own.rows;
    const int last = (r0 + a.plan.own.rows < rows ? r0 + a.plan.own.rows : rows) - 1;
    const int64_t pos0 = (int64_t)a.prefix_len + q.length - q.n;
    Limits l = limits_of(a, pos0 + last / a.group, a.prefix_len, q.length);
    const Limits first = limits_of(a, pos0 + r0 / a.group, a.prefix_len, q.length);
    l.lo = first.lo;
    return tiles_of(l);
}

// Tiles of the prefix: from the window of the batch's first position.
__device__ __forceinline__ Tiles prefix_tiles(const AttnArgs& a, int64_t min_pos) {
    Limits l = limits_of(a, min_pos, 0, a.prefix_len);
    l.hi = a.prefix_len;
    l.sink = a.window ? clampi(a.sink, 0, l.hi) : 0;
    return tiles_of(l);
}

// ---- entries and the line they form --------------------------------------------------------------------------------

template <class T>
__device__ __forceinline__ T wave_scan(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const T up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// Inclusive sum over the workgroup's threads; `total` of all.
template <class T>
__device__ __forceinline__ T block_scan(T v, T* shared, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) shared[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += shared[w];
        all += shared[w];
    }
    total = all;
    return v + before;
}

struct Line {
    int entries;         // prefix row tiles, then every sequence's
    uint64_t head_cost;
    uint64_t per;
    int64_t min_pos;     // of the batch (with a window and a prefix)
};

// Fills cost[0..entries] (cost before an entry) and info[entry] (sequence << 16
// | row tile) in LDS; the first workgroup also leaves them for the combine kernel.
template <class S>
__device__ __forceinline__ Line build_line(const AttnArgs& a, uint64_t* cost, uint32_t* info, S& sh) {
    uint64_t* const scratch = sh.scratch;
    const int tid = threadIdx.x;
    const AttnPlan& p = a.plan;
    int* const meta_first = reinterpret_cast<int*>(a.meta + meta_first_at());
    uint64_t* const meta_cost = reinterpret_cast<uint64_t*>(a.meta + meta_cost_at(a.n_seqs));
    Line line;
    line.min_pos = 0;
    int base = p.prefix_entries;
    uint32_t back = 0;  // new tokens that reach furthest before their sequence's end
    for (int s0 = 0; s0 < a.n_seqs; s0 += kThreads) {
        const int s = s0 + tid;
        uint32_t n = 0;
        if (s < a.n_seqs) {
            const Seq q = seq_at(a, s);
            n = (uint32_t)((q.n * a.group + p.own.rows - 1) / p.own.rows);
            const int before = q.n - q.length;  // (> -2^31: the earliest position is prefix_len - this)
            const uint32_t b = (uint32_t)(before + 0x40000000);
            if (q.n && b > back) back = b;
            if (s < kSeqs) {
                sh.start[s] = a.starts ? a.starts[s] : s;
                sh.end[s] = q.q0 + q.n;
                sh.ahead[s] = q.length - q.n - q.q0;
            }
        }
        uint32_t total;
        const uint32_t at = base + block_scan<uint32_t>(n, reinterpret_cast<uint32_t*>(scratch), total) - n;
        for (uint32_t r = 0; r < n && at + r < (uint32_t)p.max_entries; ++r) info[at + r] = (uint32_t)s << 16 | r;
        if (blockIdx.x == 0 && s < a.n_seqs) meta_first[s] = (int)at;
        base += (int)total;
    }
    line.entries = base < p.max_entries ? base : p.max_entries;
    if (a.window && p.prefix_entries) {
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t other = (uint32_t)__shfl_xor((int)back, o);
            back = other > back ? other : back;
        }
        uint32_t* const top = reinterpret_cast<uint32_t*>(scratch);
        __syncthreads();
        if ((tid & 63) == 0) top[tid >> 6] = back;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) back = top[w] > back ? top[w] : back;
        line.min_pos = back ? (int64_t)a.prefix_len - ((int64_t)back - 0x40000000) : a.prefix_len;
    }
    __syncthreads();
    uint64_t sum = 0;
    for (int e0 = 0; e0 < line.entries; e0 += kThreads) {
        const int e = e0 + tid;
        uint64_t c = 0;
        if (e < p.prefix_entries) {
            const int step = p.prefix.step();
            c = (uint64_t)((prefix_tiles(a, line.min_pos).count() + step - 1) / step) * p.prefix.cost;
        } else if (e < line.entries) {
            const int step = p.own.step();
            const Seq q = seq_at(a, (int)(info[e] >> 16));
            c = (uint64_t)((own_tiles(a, q, (int)(info[e] & 0xffff)).count() + step - 1) / step) * p.own.cost;
        }
        uint64_t total;
        const uint64_t at = sum + block_scan<uint64_t>(c, scratch, total) - c;
        if (e < line.entries) {
            cost[e] = at;
            if (blockIdx.x == 0) meta_cost[e] = at;
        }
        sum += total;
    }
    if (tid == 0) cost[line.entries] = sum;
    line.head_cost = sum;
    const uint64_t all = sum * (uint64_t)a.kv_heads;
    uint64_t per = quotient(all + p.workgroups - 1, p.workgroups);
    const uint64_t least = p.prefix.cost > p.own.cost ? p.prefix.cost : p.own.cost;  // a piece has a step of any unit
    line.per = per < least ? least : per;
    if (blockIdx.x == 0 && tid == 0) {
        meta_cost[line.entries] = sum;
        MetaHead* m = reinterpret_cast<MetaHead*>(a.meta);
        m->head_cost = sum;
        m->per = line.per;
        m->entries = line.entries;
    }
    __syncthreads();
    line.head_cost = uniform(line.head_cost);
    line.per = uniform(line.per);
    line.min_pos = uniform(line.min_pos);
    line.entries = uniform(line.entries);
    return line;
}

// ---- a row's result ------------------------------------------------------------------------------------------------

__device__ __forceinline__ float load1(const HeadsView& v, int64_t at) {
    if (v.dtype == QW35_HIP_DTYPE_F32) return static_cast<const float*>(v.data)[at];
    if (v.dtype == QW35_HIP_DTYPE_F16) return (float)static_cast<const _Float16*>(v.data)[at];
    return (float)static_cast<const __bf16*>(v.data)[at];
}

// N (4, 2 or 1) consecutive columns from `col`, gated, in the output's type.
template <int N>
__device__ __forceinline__ void finish(const AttnArgs& a, int t, int head, int col, float (&v)[N]) {
    if (a.gate.data) {
        const int64_t at = t * a.gate.token_stride + head * a.gate.head_stride + col;
        float g[N];
        bool done = false;
        if constexpr (N > 1) {
            if (a.gate.vec && a.gate.dtype == QW35_HIP_DTYPE_F32) {
                typedef float vec_t __attribute__((ext_vector_type(N)));
                const vec_t w = *reinterpret_cast<const vec_t*>(static_cast<const float*>(a.gate.data) + at);
#pragma unroll
                for (int j = 0; j < N; ++j) g[j] = w[j];
                done = true;
            }
        }
        if (!done) {
#pragma unroll
            for (int j = 0; j < N; ++j) g[j] = load1(a.gate, at + j);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] /= 1.0f + __expf(-g[j]);
    }
    const int64_t at = t * a.out.token_stride + head * a.out.head_stride + col;
    auto put = [&](auto zero) {
        typedef decltype(zero) T;
        T* p = static_cast<T*>(a.out.data) + at;
        if (a.out.vec && N > 1) {
            typedef T vec_t __attribute__((ext_vector_type(N > 1 ? N : 2)));
            vec_t w;
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = (T)v[j];
            *reinterpret_cast<vec_t*>(p) = w;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = (T)v[j];
        }
    };
    if (a.out.dtype == QW35_HIP_DTYPE_F32) put(0.0f);
    else if (a.out.dtype == QW35_HIP_DTYPE_F16) put((_Float16)0.0f);
    else put((__bf16)0.0f);
}

// ---- the kernel ----------------------------------------------------------------------------------------------------

// Lanes l and l ^ 32: both values, in either.  (Elements of the builtin's
// result are copied before their bits are read as a float: a
// __builtin_bit_cast of an element itself reads element 0.)
struct Pair {
    float a, b;
};
__device__ __forceinline__ Pair pair_xor32(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = p[0], b = p[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
// Over the two lanes of a row.
__device__ __forceinline__ float row_max(float v) {
    const Pair p = pair_xor32(v);
    return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float row_sum(float v) {
    const Pair p = pair_xor32(v);
    return p.a + p.b;
}

// v *= f in v's own registers (the compiler's products would go to others,
// with a copy of every accumulator where the paths meet).
__device__ __forceinline__ void scale_in_place(acc_t& v, float f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x = v[i];
        asm("v_mul_f32 %0, %1, %0" : "+v"(x) : "v"(f));
        v[i] = x;
    }
}

// A part of a row whose exponents count from m, seen from the largest `top` of several: exp2(m - top), 0 for a part
// with nothing.
__device__ __forceinline__ float part_weight(float m, float top) {
    return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// Waits until at most n of this wave's vector memory operations are in flight.
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
    asm volatile("" ::: "memory");
}
// Waits until this wave's LDS reads have returned.
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (0x7 << 4));
}

// Copies kCount KB from global memory to LDS without registers: each
// instruction moves 1 KB, lane i's 16 bytes to base + 16 i.
template <int kCount>
__device__ __forceinline__ void copy_kb(const uint8_t* from, uint8_t* to, int lane) {
    typedef const __attribute__((address_space(1))) void global_t;
    typedef __attribute__((address_space(3))) void lds_t;
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
        const uint8_t* const g = from + i * 1024 + lane * 16;
        uint8_t* const l = to + i * 1024;
        __builtin_amdgcn_global_load_lds((global_t*)g, (lds_t*)l, 16, 0, 0);
        if (i + 1 < kCount) __builtin_amdgcn_global_load_lds((global_t*)g, (lds_t*)l, 16, 1024, 0);
        if (i + 2 < kCount) __builtin_amdgcn_global_load_lds((global_t*)g, (lds_t*)l, 16, 2048, 0);
        if (i + 3 < kCount) __builtin_amdgcn_global_load_lds((global_t*)g, (lds_t*)l, 16, 3072, 0);
    }
}

template <int D>
struct Shared {
    static constexpr int kRing = D == 256 ? 128 * 1024 : 64 * 1024;
    uint8_t ring[kRing];  // tiles on their way; at a unit's end the waves' sums
    float m[kWaves][32];
    float l[kWaves][32];
    Limits all[kWaves];
    // of the first sequences, for the rows of the prefix: starts[s], the end of its new tokens, and a new token's
    // position less its index and prefix_len
    int start[kSeqs], end[kSeqs], ahead[kSeqs];
    uint32_t marks[kWaves][32 * D / 16];
    uint64_t scratch[kWaves];
};

// Raw granules of a tile: 16 bytes of a 16-bit cache, 8 of an e4m3 one.
template <bool F8>
using raw8 = std::conditional_t<F8, uint2, uint4_t>;

template <class E, bool F8>
__device__ __forceinline__ typename E::vec8 operand(raw8<F8> w) {
    if constexpr (F8) return E::from_e4m3(w);
    else return __builtin_bit_cast(typename E::vec8, w);
}

template <int D, class E, bool F8>
struct Unit {
    typedef typename E::vec8 vec8;
    typedef raw8<F8> raw;
    static constexpr int kM = D / 16;  // contraction steps of a score
    static constexpr int kT = D / 32;  // 32-column tiles of the output
    static constexpr int kElem = F8 ? 1 : 2;
    static constexpr int kTile = 32 * D * kElem;  // bytes of a tile's keys, and of its values
    static constexpr int kKb = kTile / 1024;
    static constexpr int kRing = Shared<D>::kRing;
    // The exponents' reference follows the maximum only when that has risen by
    // 2^8: sums then hold up to 2^8 times a row's largest term, which costs
    // neither type precision, and most tiles rescale nothing.
    static constexpr float kRise = 8.0f;

    const AttnArgs& a;
    Shared<D>& sh;
    const int lane, wave, n, g;  // this lane's row of a 32-row tile, and its half

    __device__ Unit(const AttnArgs& a_, Shared<D>& sh_)
        : a(a_), sh(sh_), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          n(threadIdx.x & 31), g((threadIdx.x & 63) >> 5) {}

    // What a wave carries through its tiles.
    template <int R>
    struct Rows {
        vec8 q[R][kM];
        acc_t o[R][kT];
        float mx[R], l[R];
        Limits lim[R];
        int all_lo, all_hi, all_sink;  // what every row of the wave sees
        float scale;
        bool marked;  // infinities to add at the end
    };

    // The granule of step m / of column tile t and token step kk.
    __device__ __forceinline__ vec8 key(const uint8_t* tile, int m) const {
        // row i of the product is token i with bits 2 and 3 exchanged
        const int tok = (n & 19) | (n & 4) << 1 | (n & 8) >> 1;
        return operand<E, F8>(*reinterpret_cast<const raw*>(tile + ((2 * m + g) * 32 + tok) * 8 * kElem));
    }
    __device__ __forceinline__ vec8 value(const uint8_t* tile, int t, int kk) const {
        return operand<E, F8>(*reinterpret_cast<const raw*>(tile + ((2 * kk + g) * D + t * 32 + n) * 8 * kElem));
    }

    template <int R>
    __device__ __forceinline__ void scores(const uint8_t* keys, const Rows<R>& w, acc_t (&s)[R]) const {
        constexpr int kAhead = kM < 4 ? kM : 4;
        vec8 k[kAhead];
#pragma unroll
        for (int m = 0; m < kAhead; ++m) k[m] = key(keys, m);
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = acc_t{};
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            const vec8 kk = k[m % kAhead];
            if (m + kAhead < kM) k[m % kAhead] = key(keys, m + kAhead);
#pragma unroll
            for (int r = 0; r < R; ++r) s[r] = E::mfma(kk, w.q[r][m], s[r]);
        }
        interleave<kM, R, kAhead>();
    }

    // LDS reads kAhead ahead of the matrix instructions that take them.
    template <int kSteps, int R, int kAhead>
    static __device__ __forceinline__ void interleave() {
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
            if (F8) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, R, 0);
            if (m + kAhead < kSteps) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    }

    // Softmax of a tile's scores: its terms to p, the running reference, sum and output kept.
    template <int R>
    __device__ __forceinline__ void softmax(Rows<R>& w, acc_t (&s)[R], int t0, bool masked, bool there,
                                            vec8 (&p)[R][2]) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (masked) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    s[r][j] = sees(w.lim[r], t0 + token(j), there) ? s[r][j] : -__builtin_inff();
            }
            float top = s[r][0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, s[r][j]);
            top = row_max(top) * w.scale;
            if (__builtin_expect(__any(top > w.mx[r] + kRise), 0)) {
                const float m_new = fmaxf(w.mx[r], top);
                const float shrink = m_new == w.mx[r] ? 1.0f : __builtin_amdgcn_exp2f(w.mx[r] - m_new);
                w.l[r] *= shrink;
#pragma unroll
                for (int t = 0; t < kT; ++t) scale_in_place(w.o[r][t], shrink);
                w.mx[r] = m_new;
            }
            const float ref = w.mx[r] == -__builtin_inff() ? 0.0f : w.mx[r];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[r][j], w.scale, -ref));
                w.l[r] += e;
                p[r][j / 8][j % 8] = (typename E::elem)e;
            }
        }
    }

    template <int R>
    __device__ __forceinline__ void add_values(const uint8_t* values, Rows<R>& w, const vec8 (&p)[R][2]) const {
        constexpr int kSteps = 2 * kT, kAhead = kSteps < 4 ? kSteps : 4;
        vec8 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i] = value(values, i / 2, i % 2);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const vec8 vv = v[i % kAhead];
            if (i + kAhead < kSteps) v[i % kAhead] = value(values, (i + kAhead) / 2, i % 2);
#pragma unroll
            for (int r = 0; r < R; ++r) w.o[r][i / 2] = E::mfma(vv, p[r][i % 2], w.o[r][i / 2]);
        }
        interleave<kSteps, R, kAhead>();
    }

    // Keeps infinities and NaN of a tile's values, of which some rows see only
    // a part, from the product (all waves of a shared tile come here together).
    template <int R, bool kShared>
    __device__ __forceinline__ void split_off_infinities(uint8_t* tile, Rows<R>& w, int t0, bool there,
                                                         uint32_t* marks) const {
        if (__builtin_expect(!__any(not_finite(tile)), 1)) return;
        mark_infinities<R>(tile, w, t0, there, marks);
        if (kShared) __syncthreads();
        make_finite(tile, kShared ? wave : 0, kShared ? kWaves : 1);
        if (kShared) __syncthreads();
    }

    // Every step-th granule from `first` on, without its infinities and NaN.
    __device__ __forceinline__ void make_finite(uint8_t* tile, int first, int step) const {
#pragma unroll 1
        for (int i = first; i < 2 * kT; i += step) {
            uint8_t* const at = tile + ((2 * (i & 1) + g) * D + (i >> 1) * 32 + n) * 8 * kElem;
            typedef std::conditional_t<F8, uint8_t, short> part_t;
            typedef part_t bits_t __attribute__((ext_vector_type(8)));
            bits_t v = *reinterpret_cast<const bits_t*>(at);
            constexpr part_t kSize = F8 ? 0x7f : 0x7fff, kFirst = F8 ? 0x7f : E::kInf;  // (e4m3 has a NaN, no infinities)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (v[j] & kSize) >= kFirst ? part_t(0) : v[j];
            *reinterpret_cast<bits_t*>(at) = v;
        }
        wait_lds();
    }

    // Token of a lane's score j.
    __device__ __forceinline__ int token(int j) const { return (j & 8) * 2 + g * 8 + (j & 7); }

    template <int R>
    __device__ __forceinline__ bool partly(const Rows<R>& w, int t0, bool there) const {
        return !there || !((t0 >= w.all_lo && t0 + 32 <= w.all_hi) || t0 + 32 <= w.all_sink);
    }

    // Where a unit's tiles lie: 64 of them are looked up at a time, one a lane.
    struct Pages {
        const int* table;
        Tiles tiles;
        int first, step, count;  // this wave's tiles: first, first + step, ...
        int h;
        uint32_t blocks;  // lane i: the cache block of tile 64 j + i
    };

    __device__ __forceinline__ uint32_t block_of(Pages& p, int i) const {
        if ((i & 63) == 0) {
            const int mine = i + lane < p.count ? i + lane : p.count - 1;
            const uint32_t b = (uint32_t)p.tiles.at(p.first + mine * p.step);
            const uint32_t pi = b / a.page_blocks;
            const int id = p.table[pi];
            // a page outside the cache holds nothing that a row sees
            uint32_t block = ((uint32_t)id * (uint32_t)a.kv_heads + p.h) * a.page_blocks + (b - pi * a.page_blocks);
            asm("" : "+v"(block));  // (a choice of two values, not of two paths)
            p.blocks = (uint32_t)id < a.n_pages ? block : kNoBlock;
        }
        return (uint32_t)__builtin_amdgcn_readlane((int)p.blocks, i & 63);
    }
    static __device__ __forceinline__ int64_t bytes_at(uint32_t block) {
        return (int64_t)(block == kNoBlock ? 0u : block) * kTile;
    }

    // Steps [s0, s1) of an entry for kv head h; the result to `slot`, or where
    // this is all there is of the rows (slot < 0) to the output.  R: 32-row
    // tiles of a wave; kShared: the waves share their tiles.
    template <int R, bool kShared>
    __device__ __forceinline__ void run(int h, bool prefix, int seq, int tile, Tiles tiles, int s0, int s1, int64_t slot) {
        const RowSplit& split = prefix ? a.plan.prefix : a.plan.own;
        const int rg = kShared ? wave : wave & ((1 << split.log2_rg) - 1), tg = kShared ? 0 : wave >> split.log2_rg;
        const int step = kShared ? 1 : kWaves >> split.log2_rg;
        Seq sq = {0, a.n_tokens, a.prefix_len};
        if (!prefix) {
            sq = seq_at(a, seq);
            sq = {uniform(sq.q0), uniform(sq.n), uniform(sq.length)};
        }
        const int base = prefix ? 0 : a.prefix_len;
        const int row_end = sq.n * a.group;
        const int row0 = tile * split.rows + rg * 32 * R;  // this wave's first row

        // this wave's tiles: step * s0 + tg, and every step-th after it
        Pages pages;
        pages.table = prefix ? a.prefix_pages : a.pages + (int64_t)seq * a.pages_per_seq;
        pages.tiles = tiles;
        pages.first = s0 * step + tg;
        pages.step = step;
        pages.h = h;
        const int end = s1 * step < tiles.count() ? s1 * step : tiles.count();
        pages.count = (kShared || row0 < row_end) && pages.first < end ? (end - pages.first + step - 1) / step : 0;
        const uint8_t* const kbase = static_cast<const uint8_t*>(a.ck);
        const uint8_t* const vbase = static_cast<const uint8_t*>(a.cv);

        __syncthreads();  // the ring is free
        constexpr int kFit = kShared ? kRing / (2 * kTile) : kRing / kWaves / (2 * kTile);
        constexpr int kMarks = R * 32 * D / 4;  // bytes of a wave's marks; shared tiles leave room for them in the ring
        constexpr int kPairs = kFit < 4 ? kFit : 2 * kTile * 4 + kWaves * kMarks <= kRing ? 4 : 3;
        static_assert(!kShared || 2 * kTile * kPairs + kWaves * kMarks <= kRing, "tiles and marks fit the ring");
        uint32_t* const marks = kShared ? reinterpret_cast<uint32_t*>(sh.ring + 2 * kTile * kPairs + wave * kMarks)
                                        : sh.marks[wave];
        uint8_t* const ring = sh.ring + (kShared ? 0 : wave * (kRing / kWaves));
        uint32_t there_bits = 0;  // of the tiles loaded last, the newest in bit 0
        auto note = [&](uint32_t block) { there_bits = there_bits << 1 | (block != kNoBlock ? 1u : 0u); };
        // shared: this wave's quarter of a pair of tiles
        auto load_quarter = [&](int i) {
            const uint32_t block = block_of(pages, i);
            note(block);
            const int64_t at = bytes_at(block);
            uint8_t* const to = ring + (i % kPairs) * 2 * kTile;
            if constexpr (kKb >= 2) {
                const uint8_t* const from = wave < 2 ? kbase : vbase;
                const int part = (wave & 1) * (kTile / 2);
                copy_kb<kKb / 2>(from + at + part, to + (wave < 2 ? 0 : kTile) + part, lane);
            }
        };

        Rows<R> w;
        if (pages.count) block_of(pages, 0);
        load_queries<R>(w, sq, h, row0, row_end);
        int loaded = 0;
        if constexpr (kShared) {
            for (; loaded < kPairs - 1 && loaded < pages.count; ++loaded) load_quarter(loaded);
        } else {
            for (; loaded < kPairs && loaded < pages.count; ++loaded) {
                const uint32_t block = block_of(pages, loaded);
                note(block);
                uint8_t* const to = ring + loaded * 2 * kTile;
                copy_kb<kKb>(kbase + bytes_at(block), to, lane);
                copy_kb<kKb>(vbase + bytes_at(block), to + kTile, lane);
            }
        }
        start_rows<R, kShared>(w, sq, prefix, base, row0, row_end);
        use_queries<R>(w);  // (here the queries are waited for, not in the tile loop)

        if constexpr (kShared) {
            constexpr int kEach = kKb / 2;  // a wave's copies of a pair
            for (int i = 0; i < pages.count; ++i) {
                if (i + kPairs - 2 < pages.count) wait_vm<(kPairs - 2) * kEach>();
                else wait_vm<0>();
                __builtin_amdgcn_s_barrier();  // tile i is there, and tile i - 1 read by all
                asm volatile("" ::: "memory");
                if (loaded < pages.count) load_quarter(loaded++);
                uint8_t* const at = ring + (i % kPairs) * 2 * kTile;
                const bool there = there_bits >> (loaded - 1 - i) & 1;
                const int t0 = tiles.at(pages.first + i) * 32;
                const bool masked = partly<R>(w, t0, there);
                if (masked) split_off_infinities<R, true>(at + kTile, w, t0, there, marks);
                acc_t s[R];
                vec8 p[R][2];
                scores<R>(at, w, s);
                softmax<R>(w, s, t0, masked, there, p);
                add_values<R>(at + kTile, w, p);
                wait_lds();
            }
        } else {
            constexpr int kLater = (2 * kPairs - 1) * kKb;  // copies issued after the keys of a tile, or after its values
            for (int i = 0; i < pages.count; ++i) {
                uint8_t* const at = ring + (i % kPairs) * 2 * kTile;
                const bool there = there_bits >> (loaded - 1 - i) & 1;
                const bool more = loaded < pages.count;
                const int t0 = tiles.at(pages.first + i * step) * 32;
                const bool masked = partly<R>(w, t0, there);
                acc_t s[R];
                vec8 p[R][2];
                if (more) wait_vm<kLater>();
                else wait_vm<0>();
                scores<R>(at, w, s);
                uint32_t block = 0;
                if (more) {
                    wait_lds();
                    block = block_of(pages, loaded);
                    note(block);
                    ++loaded;
                    copy_kb<kKb>(kbase + bytes_at(block), at, lane);
                }
                softmax<R>(w, s, t0, masked, there, p);
                if (more) wait_vm<kLater>();
                if (masked) split_off_infinities<R, false>(at + kTile, w, t0, there, marks);
                add_values<R>(at + kTile, w, p);
                if (more) {
                    wait_lds();
                    copy_kb<kKb>(vbase + bytes_at(block), at + kTile, lane);
                }
            }
        }
        if (__builtin_expect(w.marked, 0)) add_infinities<R>(w, marks);
#pragma unroll
        for (int r = 0; r < R; ++r) w.l[r] = row_sum(w.l[r]);

        const float v_scale = F8 && a.v_scale ? a.v_scale[h] : 1.0f;
        float* const part = a.part + (slot < 0 ? 0 : slot) * slot_floats(a.plan.slot_rows, D);
        const int part_row0 = rg * 32 * R;
        float4_t* const mine = reinterpret_cast<float4_t*>(sh.ring + wave * (kRing / kWaves)) + lane;
        static_assert(32 * D * 4 <= kRing / kWaves, "a wave's sums of 32 rows fit its part of the ring");
        auto leave = [&](int r) {  // 32 rows' sums, in lane order
#pragma unroll
            for (int t = 0; t < kT; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) mine[(t * 4 + c) * 64] = quad(w.o[r][t], c);
        };
        if constexpr (kShared) {
            if (slot >= 0) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (row0 + r * 32 + n < row_end) {
                        float* const to = part + (int64_t)(part_row0 + r * 32 + n) * D + g * 4;
#pragma unroll
                        for (int t = 0; t < kT; ++t)
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                *reinterpret_cast<float4_t*>(to + t * 32 + c * 8) = quad(w.o[r][t], c);
                        if (g == 0) put_stats(part, part_row0 + r * 32 + n, w.mx[r], w.l[r]);
                    }
                }
            } else {
                __syncthreads();  // (the tiles are read)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    leave(r);
                    const int row = row0 + r * 32 + n;
                    if (row < row_end) {
#pragma unroll 1
                        for (int i = 0; i < kT * 4; ++i)
                            put(part, slot, sq.q0, row, 0, h, (i >> 2) * 32 + (i & 3) * 8 + g * 4, mine[i * 64], w.l[r],
                                v_scale);
                    }
                    wait_lds();
                }
            }
        } else {
            // The waves of a row group join: each leaves its sums in LDS in
            // lane order, then adds up every step-th of all of theirs.
            static_assert(R == 1, "a wave of its own tiles has 32 rows");
            if (g == 0) {
                sh.m[wave][n] = w.mx[0];
                sh.l[wave][n] = w.l[0];
            }
            leave(0);
            __syncthreads();
            const int row = row0 + n;
            float top = -__builtin_inff();
            for (int v = 0; v < step; ++v) top = fmaxf(top, sh.m[rg + (v << split.log2_rg)][n]);
            float weight[kWaves], sum = 0.0f;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                weight[v] = 0.0f;
                if (v < step) {
                    weight[v] = part_weight(sh.m[rg + (v << split.log2_rg)][n], top);
                    sum += weight[v] * sh.l[rg + (v << split.log2_rg)][n];
                }
            }
            if (row < row_end) {
#pragma unroll 1
                for (int i = tg; i < kT * 4; i += step) {
                    float4_t acc = {0, 0, 0, 0};
#pragma unroll
                    for (int v = 0; v < kWaves; ++v)
                        if (v < step && weight[v] != 0.0f)
                            acc += weight[v] * reinterpret_cast<const float4_t*>(
                                                   sh.ring + (rg + (v << split.log2_rg)) * (kRing / kWaves))[i * 64 + lane];
                    put(part, slot, sq.q0, row, part_row0 + n, h, (i >> 2) * 32 + (i & 3) * 8 + g * 4, acc, sum, v_scale);
                }
                if (slot >= 0 && tg == 0 && g == 0) put_stats(part, part_row0 + n, top, sum);
            }
        }
    }

    // This lane's queries (asked for; use_queries waits).
    template <int R>
    __device__ __forceinline__ void load_queries(Rows<R>& w, const Seq& sq, int h, int row0, int row_end) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + r * 32 + n;
            const bool on = row < row_end;
            const int t = sq.q0 + (on ? row / a.group : 0), head = h * a.group + (on ? row % a.group : 0);
            const typename E::elem* p = static_cast<const typename E::elem*>(a.q.data) + t * a.q.token_stride +
                                        head * a.q.head_stride + g * 8;
#pragma unroll
            for (int m = 0; m < kM; ++m) w.q[r][m] = vec8{};
            if (on && a.q.vec) {
#pragma unroll
                for (int m = 0; m < kM; ++m) w.q[r][m] = *reinterpret_cast<const vec8*>(p + m * 16);
            } else if (on) {
#pragma unroll
                for (int m = 0; m < kM; ++m) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) w.q[r][m][j] = p[m * 16 + j];
                    asm volatile("" ::: "memory");  // (eight loads at a time)
                }
            }
        }
        w.scale = a.scale_log2 * (F8 && a.k_scale ? a.k_scale[h] : 1.0f);
    }

    template <int R>
    __device__ __forceinline__ void use_queries(Rows<R>& w) const {
        // a negative scale turns the queries' signs, so that the largest score has the largest product
        const uint32_t flip = w.scale < 0.0f ? 0x80008000u : 0u;
        w.scale = fabsf(w.scale);
        if (w.scale < 2e-38f) w.scale = 2e-38f;  // (zero: every finite score alike, and a masked one still none)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                uint4_t x = __builtin_bit_cast(uint4_t, w.q[r][m]) ^ flip;
                asm volatile("" : "+v"(x));
                w.q[r][m] = __builtin_bit_cast(vec8, x);
            }
    }

    // What this lane's rows see.
    template <int R, bool kShared>
    __device__ __forceinline__ void start_rows(Rows<R>& w, const Seq& sq, bool prefix, int base, int row0,
                                               int row_end) const {
        w.marked = false;
        w.all_lo = 0;
        w.all_hi = w.all_sink = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + r * 32 + n;
            const bool on = row < row_end;
            const int t = sq.q0 + (on ? row / a.group : 0);
            w.lim[r] = Limits{0, 0, 0};
            if (on) {
                if (!prefix) {
                    w.lim[r] = limits_of(a, (int64_t)base + sq.length - sq.n + row / a.group, base, sq.length);
                } else {
                    int s, stop = 0, ahead = 0;
                    if (a.n_seqs <= kSeqs) {
                        s = a.starts ? last_at(sh.start, a.n_seqs, t) : t;
                        if (s >= 0) {
                            stop = sh.end[s];
                            ahead = sh.ahead[s];
                        }
                    } else {
                        s = seq_of(a, t);
                        if (s >= 0) {
                            const Seq mine = seq_at(a, s);
                            stop = mine.q0 + mine.n;
                            ahead = mine.length - mine.n - mine.q0;
                        }
                    }
                    if (s >= 0 && t < stop)
                        w.lim[r] = limits_of(a, (int64_t)a.prefix_len + ahead + t, 0, a.prefix_len);
                }
                w.all_lo = w.lim[r].lo > w.all_lo ? w.lim[r].lo : w.all_lo;
                w.all_hi = w.lim[r].hi < w.all_hi ? w.lim[r].hi : w.all_hi;
                w.all_sink = w.lim[r].sink < w.all_sink ? w.lim[r].sink : w.all_sink;
            }
            w.mx[r] = -__builtin_inff();
            w.l[r] = 0.0f;
#pragma unroll
            for (int t2 = 0; t2 < kT; ++t2) w.o[r][t2] = acc_t{};
        }
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int lo = __shfl_xor(w.all_lo, o), hi = __shfl_xor(w.all_hi, o), sk = __shfl_xor(w.all_sink, o);
            w.all_lo = lo > w.all_lo ? lo : w.all_lo;
            w.all_hi = hi < w.all_hi ? hi : w.all_hi;
            w.all_sink = sk < w.all_sink ? sk : w.all_sink;
        }
        w.all_lo = uniform(w.all_lo);
        w.all_hi = uniform(w.all_hi);
        w.all_sink = uniform(w.all_sink);
        if constexpr (kShared) {
            // what every row of the workgroup sees: its waves take a tile apart together or not at all
            if (lane == 0) sh.all[wave] = Limits{w.all_lo, w.all_hi, w.all_sink};
            __syncthreads();
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const Limits l = sh.all[v];
                w.all_lo = uniform(l.lo > w.all_lo ? l.lo : w.all_lo);
                w.all_hi = uniform(l.hi < w.all_hi ? l.hi : w.all_hi);
                w.all_sink = uniform(l.sink < w.all_sink ? l.sink : w.all_sink);
            }
        }
    }

    static __device__ __forceinline__ bool sees(const Limits& l, int token, bool there) {
        return there & (token < l.hi) & ((token >= l.lo) | (token < l.sink));
    }

    static __device__ __forceinline__ float4_t quad(const acc_t& v, int c) {
        return float4_t{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
    }

    // Four columns of a row: sums into the partial slot, or the finished output.
    __device__ __forceinline__ void put(float* part, int64_t slot, int q0, int row, int part_row, int h, int col,
                                        float4_t v, float sum, float v_scale) const {
        if (slot >= 0) {
            *reinterpret_cast<float4_t*>(part + (int64_t)part_row * D + col) = v;
            return;
        }
        const float inv = sum == 0.0f ? 0.0f : v_scale / sum;
        float x[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        finish<4>(a, q0 + row / a.group, h * a.group + row % a.group, col, x);
    }

    __device__ __forceinline__ void put_stats(float* part, int part_row, float m, float l) const {
        part[(int64_t)a.plan.slot_rows * D + part_row] = m;
        part[(int64_t)a.plan.slot_rows * (D + 1) + part_row] = l;
    }

    // Whether a granule of the tile of values holds an infinity or a NaN.
    __device__ __forceinline__ bool not_finite(const uint8_t* tile) const {
        typedef short bits_t __attribute__((ext_vector_type(8)));
        bits_t top = {};
#pragma unroll 4
        for (int t = 0; t < 2 * kT; ++t)
            top = __builtin_elementwise_max(
                top, __builtin_bit_cast(bits_t, value(tile, t >> 1, t & 1)) & (short)0x7fff);
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) bad |= top[j] >= E::kInf;
        return bad;
    }

    // For a tile with infinities or NaN among its values of which some rows
    // see only a part: what a row does not see must not reach it even as
    // 0 x NaN, which the matrix instruction would add.  The product takes the
    // finite values; which infinities (a NaN is both) a row saw in which column
    // is kept, a bit each, and added when the unit's tiles are done.
    //   marks: [r][t][sign][32 rows], bits of the tile's 32 columns; lane (n, g)
    // keeps sign g of row n.  (No branch here or in the tile loop depends on the
    // lane: the paths would keep copies of the accumulators where they meet.)
    template <int R>
    __device__ __forceinline__ void mark_infinities(const uint8_t* tile, Rows<R>& w, int t0, bool there,
                                                    uint32_t* marks) const {
        if (!w.marked) {
            w.marked = true;
#pragma unroll 1
            for (int i = 0; i < R * kT; ++i) marks[i * 64 + lane] = 0;
        }
#pragma unroll 1
        for (int i = 0; i < 2 * kT; ++i) {
            typedef short bits_t __attribute__((ext_vector_type(8)));
            bits_t v = __builtin_bit_cast(bits_t, value(tile, i >> 1, i & 1));
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
                const short mine = v[0], size = mine & 0x7fff;
                v = __builtin_shufflevector(v, v, 1, 2, 3, 4, 5, 6, 7, 0);
                const uint64_t up = __ballot(size > E::kInf || mine == E::kInf);
                const uint64_t down = __ballot(size > E::kInf || (size == E::kInf && mine < 0));
                if ((up | down) == 0) continue;
                const uint64_t sign = g ? down : up;  // columns 32 (i / 2) ..: of token j, and of token 8 + j
                const int at = t0 + (i & 1) * 16 + j;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    marks[(r * kT + (i >> 1)) * 64 + lane] |=
                        (sees(w.lim[r], at, there) ? (uint32_t)sign : 0u) |
                        (sees(w.lim[r], at + 8, there) ? (uint32_t)(sign >> 32) : 0u);
            }
        }
    }

    template <int R>
    __device__ __forceinline__ void add_infinities(Rows<R>& w, const uint32_t* marks) const {
        wait_lds();
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                const uint32_t up = marks[(r * kT + t) * 64 + n], down = marks[(r * kT + t) * 64 + 32 + n];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const int col = (c >> 2) * 8 + g * 4 + (c & 3);
                    const float inf = __builtin_inff();
                    w.o[r][t][c] += (up >> col & 1 ? inf : 0.0f) - (down >> col & 1 ? inf : 0.0f);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    }
};

// kR: 32-row tiles of a wave where waves share their tiles; 0: no unit of the launch does.
template <int D, class E, bool F8, int kR>
__global__ __launch_bounds__(kThreads, D == 256 || kR == 2 ? 1 : 2) void prefix_attention_kernel(AttnArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    Shared<D>& sh = *reinterpret_cast<Shared<D>*>(lds);
    uint64_t* const cost = reinterpret_cast<uint64_t*>(lds + sizeof(Shared<D>));
    uint32_t* const info = reinterpret_cast<uint32_t*>(cost + a.plan.max_entries + 1);
    const Line line = build_line(a, cost, info, sh);
    // Pieces follow each other by XCD (workgroup b runs on XCD b % 8), so that
    // the row tiles of one kv head, which read the same keys, share an L2.
    const int grid = a.plan.workgroups;
    const int w = grid % 8 ? blockIdx.x : (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8;
    const uint64_t all = line.head_cost * (uint64_t)a.kv_heads;
    const uint64_t x0 = line.per * (uint64_t)w, x1 = x0 + line.per < all ? x0 + line.per : all;
    uint64_t x = x0;
    Unit<D, E, F8> unit(a, sh);
    while (x < x1) {
        const int h = (int)quotient(x, line.head_cost);
        const uint64_t at = x - h * line.head_cost;  // within the head
        int lo = 0, hi = line.entries;               // the entry: cost[lo] <= at < cost[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (cost[mid] <= at) lo = mid;
            else hi = mid;
        }
        const int e = uniform(lo);
        const bool prefix = e < a.plan.prefix_entries;
        const RowSplit& split = prefix ? a.plan.prefix : a.plan.own;
        const uint32_t c = (uint32_t)split.cost;
        const uint64_t e0 = uniform(cost[e]), e1 = uniform(cost[e + 1]);
        const uint64_t head0 = h * line.head_cost;
        const uint64_t stop = x1 - head0 < e1 ? x1 - head0 : e1;
        // steps whose first point lies in the piece (an entry has less than 2^32)
        const int s0 = (int)(((uint32_t)(at - e0) + c - 1) / c), s1 = (int)(((uint32_t)(stop - e0) + c - 1) / c);
        const uint32_t who = prefix ? e : uniform((int)info[e]);
        const int seq = prefix ? 0 : (int)(who >> 16), tile = prefix ? e : (int)(who & 0xffff);
        Tiles tiles;
        if (prefix) tiles = prefix_tiles(a, line.min_pos);
        else tiles = own_tiles(a, seq_at(a, seq), tile);
        tiles = {uniform(tiles.sink), uniform(tiles.lo), uniform(tiles.hi)};
        // all of the entry's steps begin in this piece
        const bool alone = !a.plan.prefix_entries && x - at + e0 >= x0 && head0 + e1 - c < x0 + line.per;
        if (s0 < s1) {
            const int64_t slot = alone ? -1 : (int64_t)w + (int64_t)h * line.entries + e;
            if (kR == 0 || !split.shared) unit.template run<1, false>(h, prefix, seq, tile, tiles, s0, s1, slot);
            else unit.template run<kR ? kR : 1, true>(h, prefix, seq, tile, tiles, s0, s1, slot);
        }
        x = head0 + stop;
    }
}

// Dynamic LDS of a launch: the tiles and the line of entries.
template <int D>
size_t lds_bytes(int max_entries) {
    return sizeof(Shared<D>) + 8 * ((size_t)max_entries + 1) + 4 * (size_t)max_entries;
}

template <int D, class E, bool F8, int kR>
hipError_t launch_as(const AttnArgs& a, hipStream_t stream) {
    prefix_attention_kernel<D, E, F8, kR><<<dim3((unsigned)a.plan.workgroups), kThreads, lds_bytes<D>(a.plan.max_entries), stream>>>(a);
    return hipGetLastError();
}

template <int D, class E, bool F8>
hipError_t launch_rows(const AttnArgs& a, hipStream_t stream) {
    if (a.plan.shared_r == 0) return launch_as<D, E, F8, 0>(a, stream);
    if constexpr (D < 256) {
        if (a.plan.shared_r == 2) return launch_as<D, E, F8, 2>(a, stream);
    }
    return launch_as<D, E, F8, 1>(a, stream);
}

template <int D>
hipError_t launch_dim(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream) {
    if (bf16) return f8 ? launch_rows<D, Bf16, true>(a, stream) : launch_rows<D, Bf16, false>(a, stream);
    return f8 ? launch_rows<D, Half, true>(a, stream) : launch_rows<D, Half, false>(a, stream);
}

}  // namespace attn
}  // namespace qw35
