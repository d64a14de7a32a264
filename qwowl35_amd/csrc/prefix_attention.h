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
// v_mfma_f32_16x16x32: lane l holds query row l % 16 in S, P and O alike, so
// maximum, sum and rescaling stay in a lane (and its three others of the same
// row).  The cache's granules are the A operands: 16 bytes are eight columns of
// a key, or eight tokens of a value column, and a wave's load is 1 KB in a
// piece, straight from HBM to registers.  Key row i of half b of a tile is
// token 8 (i / 4) + 4 b + i % 4, which leaves the four scores a lane holds of
// either half as the eight tokens 8 (l / 16) .. + 7 of its value granule: P
// needs no exchange between lanes.
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
constexpr uint32_t kNoBlock = 0xffffffffu;

// Element type of queries and 16-bit caches, and its matrix instruction.
struct Half {
    typedef _Float16 elem;
    typedef half8_t vec8;
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static constexpr uint32_t kInf2 = 0x7c007c00u;
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
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static constexpr uint32_t kInf2 = 0x7f807f80u;
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

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

__device__ __forceinline__ Seq seq_at(const AttnArgs& a, int s) {
    Seq q;
    q.q0 = a.starts ? clampi(a.starts[s], 0, a.n_tokens) : s;
    const int end = a.starts ? clampi(a.starts[s + 1], q.q0, a.n_tokens) : s + 1;
    q.n = end - q.q0;
    q.length = clampi(a.lengths[s], 0, (int)(a.pages_per_seq * a.page_blocks * 32));
    return q;
}

// The sequence of new token t: the last whose start is at or before it (-1: none).
__device__ __forceinline__ int seq_of(const AttnArgs& a, int t) {
    if (!a.starts) return t;
    int lo = 0, hi = a.n_seqs;  // starts[0..lo) <= t < starts[hi..)
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo - 1;
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
__device__ __forceinline__ Line build_line(const AttnArgs& a, uint64_t* cost, uint32_t* info, uint64_t* scratch) {
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
            const int step = kWaves >> p.prefix.log2_rg;
            c = (uint64_t)((prefix_tiles(a, line.min_pos).count() + step - 1) / step) * p.prefix.cost;
        } else if (e < line.entries) {
            const int step = kWaves >> p.own.log2_rg;
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
    uint64_t per = (all + p.workgroups - 1) / p.workgroups;
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

// Lanes l and l ^ 16, l and l ^ 32: both values, in either.  (Elements of the
// builtins' results are copied before their bits are read as a float: a
// __builtin_bit_cast of an element itself reads element 0.)
struct Pair {
    float a, b;
};
__device__ __forceinline__ Pair pair_xor16(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = p[0], b = p[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Pair pair_xor32(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = p[0], b = p[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
// Over the four lanes of a row.
__device__ __forceinline__ float row_max(float v) {
    const Pair p = pair_xor16(v);
    const Pair q = pair_xor32(fmaxf(p.a, p.b));
    return fmaxf(q.a, q.b);
}
__device__ __forceinline__ float row_sum(float v) {
    const Pair p = pair_xor16(v);
    const Pair q = pair_xor32(p.a + p.b);
    return q.a + q.b;
}

// A part of a row whose maximum is m, seen from the maximum `top` of several: exp2(m - top), 0 for a part with nothing.
__device__ __forceinline__ float part_weight(float m, float top) {
    return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

template <int D>
struct Shared {
    // Four waves' sums of 16 rows, rows padded by four floats: the 16 rows a
    // wave stores at once start in 16 different 16-byte groups.
    static constexpr int kRow = D + 4;
    float o[kWaves][16][kRow];
    float m[kWaves][16];
    float l[kWaves][16];
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

template <int D, class E, bool F8, int R>
struct Unit {
    typedef typename E::vec8 vec8;
    typedef raw8<F8> raw;
    static constexpr int kM = D / 32;  // contraction steps of a score
    static constexpr int kT = D / 16;  // 16-column tiles of the output
    static constexpr int kElem = F8 ? 1 : 2;

    const AttnArgs& a;
    Shared<D>& sh;
    const int lane, wave, n, g;  // this lane's row of a 16-row tile, and its quarter

    __device__ Unit(const AttnArgs& a_, Shared<D>& sh_)
        : a(a_), sh(sh_), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          n(threadIdx.x & 15), g((threadIdx.x & 63) >> 4) {}

    __device__ __forceinline__ void load_keys(const uint8_t* tile, raw (&k)[2][kM]) const {
        const uint8_t* p = tile + (g * 256 + (8 * (n >> 2) + (n & 3)) * 8) * kElem;
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int b = 0; b < 2; ++b)
                k[b][m] = *reinterpret_cast<const raw*>(p + (m * 1024 + b * 32) * kElem);
    }

    __device__ __forceinline__ void load_values(const uint8_t* tile, raw (&v)[kT]) const {
        const uint8_t* p = tile + (g * 8 * D + n * 8) * kElem;
#pragma unroll
        for (int t = 0; t < kT; ++t) v[t] = *reinterpret_cast<const raw*>(p + t * 128 * kElem);
    }

    // Steps [s0, s1) of an entry for kv head h; the result to `slot`, or where
    // this is all there is of the rows (slot < 0) to the output.
    __device__ __forceinline__ void run(int h, bool prefix, int seq, int tile, Tiles tiles, int s0, int s1, int64_t slot) {
        const RowSplit& split = prefix ? a.plan.prefix : a.plan.own;
        const int rg = wave & ((1 << split.log2_rg) - 1), tg = wave >> split.log2_rg;
        const int step = kWaves >> split.log2_rg;
        Seq sq = {0, a.n_tokens, a.prefix_len};
        if (!prefix) sq = seq_at(a, seq);
        const int base = prefix ? 0 : a.prefix_len;
        const int row_end = sq.n * a.group;
        const int row0 = tile * split.rows + rg * 16 * R;  // this wave's first row
        const int* const table = prefix ? a.prefix_pages : a.pages + (int64_t)seq * a.pages_per_seq;

        // this lane's rows: queries and limits
        vec8 q[R][kM];
        Limits lim[R];
        int all_lo = 0, all_hi = 0x7fffffff, all_sink = 0x7fffffff;  // what every row of the wave sees
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + r * 16 + n;
            const bool on = row < row_end;
            const int t = sq.q0 + (on ? row / a.group : 0), head = h * a.group + (on ? row % a.group : 0);
            const typename E::elem* p = static_cast<const typename E::elem*>(a.q.data) + t * a.q.token_stride +
                                        head * a.q.head_stride + g * 8;
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                vec8 w = {};
                if (on) {
                    if (a.q.vec) {
                        w = *reinterpret_cast<const vec8*>(p + m * 32);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = p[m * 32 + j];
                    }
                }
                q[r][m] = w;
            }
            lim[r] = Limits{0, 0, 0};
            if (on) {
                if (!prefix) {
                    lim[r] = limits_of(a, (int64_t)base + sq.length - sq.n + row / a.group, base, sq.length);
                } else {
                    const int s = seq_of(a, t);
                    if (s >= 0) {
                        const Seq mine = seq_at(a, s);
                        if (t < mine.q0 + mine.n)
                            lim[r] = limits_of(a, (int64_t)a.prefix_len + mine.length - mine.n + t - mine.q0, 0,
                                               a.prefix_len);
                    }
                }
                all_lo = lim[r].lo > all_lo ? lim[r].lo : all_lo;
                all_hi = lim[r].hi < all_hi ? lim[r].hi : all_hi;
                all_sink = lim[r].sink < all_sink ? lim[r].sink : all_sink;
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o *= 2) {
            const int lo = __shfl_xor(all_lo, o), hi = __shfl_xor(all_hi, o), sk = __shfl_xor(all_sink, o);
            all_lo = lo > all_lo ? lo : all_lo;
            all_hi = hi < all_hi ? hi : all_hi;
            all_sink = sk < all_sink ? sk : all_sink;
        }
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);
        all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        all_sink = __builtin_amdgcn_readfirstlane(all_sink);

        float4_t o[R][kT];
        float mx[R], l[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mx[r] = -__builtin_inff();
            l[r] = 0.0f;
#pragma unroll
            for (int t = 0; t < kT; ++t) o[r][t] = float4_t{0, 0, 0, 0};
        }
        const float scale = a.scale_log2 * (F8 && a.k_scale ? a.k_scale[h] : 1.0f);

        // this wave's tiles: step * s0 + tg, and every step-th after it
        const int first = s0 * step + tg;
        const int end = s1 * step < tiles.count() ? s1 * step : tiles.count();
        const int mine = row0 < row_end && first < end ? (end - first + step - 1) / step : 0;
        const uint8_t* const kbase = static_cast<const uint8_t*>(a.ck);
        const uint8_t* const vbase = static_cast<const uint8_t*>(a.cv);
        uint32_t blocks = kNoBlock;  // lane i: the cache block of tile 64 j + i
        auto look_up = [&](int j) {
            const int v = first + (j + lane) * step;
            blocks = kNoBlock;
            if (j + lane < mine) {
                const uint32_t b = (uint32_t)tiles.at(v);
                const uint32_t pi = b / a.page_blocks;
                const int id = table[pi];
                // a page outside the cache holds nothing that a row sees
                if ((uint32_t)id < a.n_pages)
                    blocks = ((uint32_t)id * (uint32_t)a.kv_heads + h) * a.page_blocks + (b - pi * a.page_blocks);
            }
        };
        auto block_at = [&](int j) {
            return (uint32_t)__builtin_amdgcn_readlane((int)blocks, j & 63);
        };
        auto bytes_at = [&](uint32_t block) {
            return (int64_t)(block == kNoBlock ? 0u : block) * (32 * D * kElem);
        };
        raw k[2][kM];
        uint32_t block = kNoBlock;
        if (mine) {
            look_up(0);
            block = block_at(0);
            load_keys(kbase + bytes_at(block), k);
        }
        for (int i = 0; i < mine; ++i) {
            raw v[kT];
            const uint8_t* const vtile = vbase + bytes_at(block);
            load_values(vtile, v);
            float4_t s[R][2];
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const vec8 kk = operand<E, F8>(k[b][m]);
#pragma unroll
                    for (int r = 0; r < R; ++r) s[r][b] = E::mfma(kk, q[r][m], s[r][b]);
                }
            const int t0 = tiles.at(first + i * step) * 32;
            const bool there = block != kNoBlock;
            if (i + 1 < mine) {
                if (((i + 1) & 63) == 0) look_up(i + 1);
                block = block_at(i + 1);
                load_keys(kbase + bytes_at(block), k);
            }
            const bool masked = !there || !((t0 >= all_lo && t0 + 32 <= all_hi) || t0 + 32 <= all_sink);
            vec8 p[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = s[r][j >> 2][j & 3] * scale;
                if (masked) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!sees(lim[r], t0 + g * 8 + j, there)) x[j] = -__builtin_inff();
                }
                float top = x[0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
                top = row_max(top);
                const float m_new = fmaxf(mx[r], top);
                const float ref = m_new == -__builtin_inff() ? 0.0f : m_new;
                if (__any(m_new != mx[r])) {
                    const float shrink = __builtin_amdgcn_exp2f(mx[r] - ref);
                    l[r] *= shrink;
#pragma unroll
                    for (int t = 0; t < kT; ++t) o[r][t] *= shrink;
                }
                mx[r] = m_new;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float e2 = __builtin_amdgcn_exp2f(x[j] - ref);
                    l[r] += e2;
                    p[r][j] = (typename E::elem)e2;
                }
            }
            if (masked && __any(not_finite(v))) {
                add_values_seen(vtile, lim, t0, there, p, o);
            } else {
#pragma unroll
                for (int t = 0; t < kT; ++t) {
                    const vec8 vv = operand<E, F8>(v[t]);
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r][t] = E::mfma(vv, p[r], o[r][t]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) l[r] = row_sum(l[r]);

        // the waves of a row group join, 16 rows at a time
        const float v_scale = F8 && a.v_scale ? a.v_scale[h] : 1.0f;
        float* const part = a.part + (slot < 0 ? 0 : slot) * slot_floats(a.plan.slot_rows, D);
        const int part_row0 = rg * 16 * R;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (step > 1) {
                __syncthreads();
#pragma unroll
                for (int t = 0; t < kT; ++t)
                    *reinterpret_cast<float4_t*>(&sh.o[wave][n][t * 16 + g * 4]) = o[r][t];
                if (g == 0) {
                    sh.m[wave][n] = mx[r];
                    sh.l[wave][n] = l[r];
                }
                __syncthreads();
                // 64 lanes x step waves of a group: row n of lanes' 16, columns g * 4 + 16 * ...
                float top = -__builtin_inff();
                for (int w = 0; w < step; ++w) top = fmaxf(top, sh.m[rg + (w << split.log2_rg)][n]);
                float weight[kWaves], sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    weight[w] = 0.0f;
                    if (w < step) {
                        weight[w] = part_weight(sh.m[rg + (w << split.log2_rg)][n], top);
                        sum += weight[w] * sh.l[rg + (w << split.log2_rg)][n];
                    }
                }
                const int row = row0 + r * 16 + n;
                if (row < row_end) {
                    for (int t = tg; t < kT; t += step) {
                        float4_t acc = {0, 0, 0, 0};
#pragma unroll
                        for (int w = 0; w < kWaves; ++w)
                            if (w < step && weight[w] != 0.0f)
                                acc += weight[w] *
                                       *reinterpret_cast<const float4_t*>(
                                           &sh.o[rg + (w << split.log2_rg)][n][t * 16 + g * 4]);
                        put(part, slot, sq.q0, row, part_row0 + r * 16 + n, h, t * 16 + g * 4, acc, sum, v_scale);
                    }
                    if (slot >= 0 && tg == 0 && g == 0) put_stats(part, part_row0 + r * 16 + n, top, sum);
                }
            } else {
                const int row = row0 + r * 16 + n;
                if (row < row_end) {
#pragma unroll
                    for (int t = 0; t < kT; ++t)
                        put(part, slot, sq.q0, row, part_row0 + r * 16 + n, h, t * 16 + g * 4, o[r][t], l[r], v_scale);
                    if (slot >= 0 && g == 0) put_stats(part, part_row0 + r * 16 + n, mx[r], l[r]);
                }
            }
        }
    }

    static __device__ __forceinline__ bool sees(const Limits& l, int token, bool there) {
        return there && token < l.hi && (token >= l.lo || token < l.sink);
    }

    // Four columns of a row: sums into the partial slot, or the finished output.
    __device__ __forceinline__ void put(float* part, int64_t slot, int q0, int row, int part_row, int h, int col,
                                        float4_t v, float sum, float v_scale) const {
        if (slot >= 0) {
            *reinterpret_cast<float4_t*>(part + (int64_t)part_row * D + col) = v;
            return;
        }
        const float inv = sum == 0.0f ? 0.0f : v_scale / sum;
        float w[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        finish<4>(a, q0 + row / a.group, h * a.group + row % a.group, col, w);
    }

    __device__ __forceinline__ void put_stats(float* part, int part_row, float m, float l) const {
        part[(int64_t)a.plan.slot_rows * D + part_row] = m;
        part[(int64_t)a.plan.slot_rows * (D + 1) + part_row] = l;
    }

    // Whether a granule of the tile holds an infinity or a NaN.
    static __device__ __forceinline__ bool not_finite(const raw (&v)[kT]) {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 top = {0, 0};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const uint4_t w = __builtin_bit_cast(uint4_t, operand<E, F8>(v[t]));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        }
        const u16x2 inf = __builtin_bit_cast(u16x2, E::kInf2);
        return top[0] >= inf[0] || top[1] >= inf[1];
    }

    // O += V^T P^T token by token, for a tile with infinities or NaN among its
    // values of which some rows see only a part: what a row does not see must
    // not reach it even as 0 x NaN, which the matrix instruction would add.
    __device__ __forceinline__ void add_values_seen(const uint8_t* vtile, const Limits (&lim)[R], int t0, bool there,
                                                 const vec8 (&p)[R], float4_t (&o)[R][kT]) const {
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            float w[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mine = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) mine = (i & 7) == j ? (float)p[r][j] : mine;
                w[r] = __shfl(mine, (i >> 3) * 16 + n);
            }
            const uint8_t* const at = vtile + (int64_t)((i >> 3) * 8 * D + (i & 7)) * kElem;
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                __builtin_amdgcn_sched_barrier(0);  // four loads at a time: this path keeps no registers of its own
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int col = t * 16 + g * 4 + c;
                    float x;
                    if constexpr (F8) {
                        uint2 byte = {at[col * 8], 0u};
                        x = (float)E::from_e4m3(byte)[0];
                    } else {
                        x = (float)*reinterpret_cast<const typename E::elem*>(at + col * 8 * kElem);
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (sees(lim[r], t0 + i, there)) o[r][t][c] = fmaf(w[r], x, o[r][t][c]);
                }
            }
        }
    }
};

template <int D, class E, bool F8, int R>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void prefix_attention_kernel(AttnArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    Shared<D>& sh = *reinterpret_cast<Shared<D>*>(lds);
    uint64_t* const cost = reinterpret_cast<uint64_t*>(lds + sizeof(Shared<D>));
    uint32_t* const info = reinterpret_cast<uint32_t*>(cost + a.plan.max_entries + 1);
    const Line line = build_line(a, cost, info, sh.scratch);
    // Pieces follow each other by XCD (workgroup b runs on XCD b % 8), so that
    // the row tiles of one kv head, which read the same keys, share an L2.
    const int grid = a.plan.workgroups;
    const int w = grid % 8 ? blockIdx.x : (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8;
    const uint64_t all = line.head_cost * (uint64_t)a.kv_heads;
    uint64_t x = line.per * (uint64_t)w;
    const uint64_t x1 = x + line.per < all ? x + line.per : all;
    Unit<D, E, F8, R> unit(a, sh);
    while (x < x1) {
        const int h = (int)(x / line.head_cost);
        const uint64_t at = x - h * line.head_cost;  // within the head
        int lo = 0, hi = line.entries;               // the entry: cost[lo] <= at < cost[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (cost[mid] <= at) lo = mid;
            else hi = mid;
        }
        const int e = lo;
        const bool prefix = e < a.plan.prefix_entries;
        const uint32_t c = (uint32_t)(prefix ? a.plan.prefix.cost : a.plan.own.cost);
        const uint64_t e0 = cost[e], e1 = cost[e + 1];
        const uint64_t stop = x1 - h * line.head_cost < e1 ? x1 - h * line.head_cost : e1;
        // steps whose first point lies in the piece
        const int s0 = (int)((at - e0 + c - 1) / c), s1 = (int)((stop - e0 + c - 1) / c);
        const int seq = prefix ? 0 : (int)(info[e] >> 16), tile = prefix ? e : (int)(info[e] & 0xffff);
        Tiles tiles;
        if (prefix) tiles = prefix_tiles(a, line.min_pos);
        else tiles = own_tiles(a, seq_at(a, seq), tile);
        const uint64_t head0 = h * line.head_cost;
        const bool alone = !a.plan.prefix_entries && (head0 + e0) / line.per == (head0 + e1 - c) / line.per;
        if (s0 < s1)
            unit.run(h, prefix, seq, tile, tiles, s0, s1,
                     alone ? -1 : (int64_t)w + (int64_t)h * line.entries + e);
        x = head0 + stop;
    }
}

template <int D, class E, bool F8, int R>
hipError_t launch_as(const AttnArgs& a, hipStream_t stream) {
    const size_t lds = sizeof(Shared<D>) + 8 * ((size_t)a.plan.max_entries + 1) + 4 * (size_t)a.plan.max_entries;
    prefix_attention_kernel<D, E, F8, R><<<dim3((unsigned)a.plan.workgroups), kThreads, lds, stream>>>(a);
    return hipGetLastError();
}

template <int D, class E, bool F8>
hipError_t launch_rows(const AttnArgs& a, hipStream_t stream) {
    return a.plan.r == 1 ? launch_as<D, E, F8, 1>(a, stream) : launch_as<D, E, F8, 2>(a, stream);
}

template <int D>
hipError_t launch_dim(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream) {
    if (bf16) return f8 ? launch_rows<D, Bf16, true>(a, stream) : launch_rows<D, Bf16, false>(a, stream);
    return f8 ? launch_rows<D, Half, true>(a, stream) : launch_rows<D, Half, false>(a, stream);
}

}  // namespace attn
}  // namespace qw35
