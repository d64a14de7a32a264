// Attention of a ragged batch over a paged cache whose sequences share a
// prefix: the kernel template (one translation unit per head dimension).
//
// Mathematics.  For a row (new token t of sequence s, query head of group h):
//   out = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q.k_i - m)
// over the tokens i the row sees, in one pass: tiles of 32 tokens keep a
// reference m close to the running maximum, the sum of p and the sum of p v
// (fp32), rescaled when m rises.  Parts of a row's tokens (the shared prefix,
// the sequence's own pages, pieces of either) give (m, sum p, sum p v) each,
// joined at the end by exp(m_part - m).
//
// Units.  The rows of all sequences read the same prefix, so a prefix unit is
// a kv head and a tile of rows out of the whole batch: the prefix is read once
// for all of them.  An own unit is a kv head, a sequence and a tile of its
// rows.  The steps of all prefix units lie behind each other on one line, those
// of all own units on another.  The workgroups are divided between the two by
// cost, and each (on the own line each wave, unless its units share their
// tiles) takes an equal piece, crossing units where it has to: lengths live on
// the device, and whatever they are the load is even and the grid constant.
// Row tiles of a prefix head stand abreast, on the same steps at a time, so
// that all but one read them from the L2.  A piece's part of a unit goes to the
// partial slot (place of the piece + unit), which no other has; one workgroup
// lists every unit's slots for the join.
//
// A call is often a few microseconds long, of which a wave alone on its SIMD
// takes one for every 500 or so instructions that are not a tile's.  So up to
// 64 sequences of one row tile each, the own line is kept a sequence a lane, in
// 32 bits and without a barrier.
//
// Operands.  A tile's scores are S^T = K Q^T and the output O^T = V^T P^T, on
// v_mfma_f32_32x32x16 (units of more than 16 rows) or 16x16x32: a lane holds one
// query row in S, P and O alike, so maximum, sum and rescaling stay in a lane
// and the one or three others of the same row.  The cache's granules are the A
// operands: eight columns of a key, or eight tokens of a value column.  Which
// token is which row of the scores is chosen so that a lane's scores are the
// tokens of its own value granules: P needs no exchange between lanes.
//
// Data.  Tiles go from HBM to LDS by copies that take no registers, as far
// ahead as the ring has room (128 KB for 256 columns), and from there to the
// matrix instructions: 16 bytes a lane, a wave's reads consecutive.  With up to
// 64 rows in a prefix unit each wave (or pair) has its own tiles, since then a
// compute unit only waits for HBM; more rows share a tile among the four waves,
// which read it once for 128 rows.
//
// What bounds it.  Up to 64 rows HBM, where the context is long (five sequences
// of 16 heads over 100003 tokens, 256 columns e4m3: 4.7 TB/s in the tile loop,
// where a copy reaches 4.9; 58 us), else latency (one sequence of 517 tokens: 11
// us and 5 of the join).  Over that no unit by itself but the chain within a wave
// (256 columns, one wave a SIMD, 1024 rows over 32768 tokens: the matrix unit is
// busy 39% of the time, the vector unit 28%, LDS reads 20%, and the wave waits for
// a third; 690 TFLOP/s, a large product reaches 1100.  128 columns, two waves a
// SIMD, 256 rows over 98304 tokens: matrix unit 48%, 700).
//
// Rounding.  Scores, maxima, sums and O are fp32.  P is rounded once to the
// queries' 16-bit type for the second product, whatever the output's type (the
// matrix unit takes both operands of a kind: relative 2^-11 fp16, 2^-8 bf16 at
// most, signs mixed); e4m3 is exact in either 16-bit type.  The sum of P takes it
// before the rounding: a result is then off by at most that of its weights, by
// the rounded ones' sum at most twice that.
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

// Element type of queries and 16-bit caches, and its matrix instructions.
struct Half {
    typedef _Float16 elem;
    typedef half8_t vec8;
    static __device__ __forceinline__ acc_t mfma(vec8 a, vec8 b, acc_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static constexpr short kInf = 0x7f80;  // bits of +inf
    static __device__ __forceinline__ vec8 from_e4m3(uint2 w) {
        uint4_t r;
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, true));
        return __builtin_bit_cast(vec8, r);
    }
};

// What the join needs of a launch, at the start of the workspace: this, then
// first[n_seqs] (a sequence's first own entry), then [kv_heads][prefix and own
// entries] Pieces.
struct MetaHead {
    int own_entries;
    int lanes;          // first[s] is s
    int prefix_stride;  // from a prefix entry's slot to its next
    int pad;
};
struct Pieces {
    uint32_t slot0;  // the first partial slot of an entry, and how many (an own entry's follow each other)
    uint32_t n;
};

__host__ __device__ inline size_t meta_first_at() { return sizeof(MetaHead); }
__host__ __device__ inline size_t meta_pieces_at(int n_seqs) {
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

// x / d of numbers below 2^31, the quotient below 2^15.
__device__ __forceinline__ uint32_t quotient(uint32_t x, uint32_t d) {
    uint32_t q = (uint32_t)((float)x * __builtin_amdgcn_rcpf((float)d));
    if ((int32_t)(x - q * d) < 0) --q;
    if (x - q * d >= d) ++q;
    return q;
}

// Over a wave's 64 lanes, by lane exchanges inside the vector unit.
template <class Op>
__device__ __forceinline__ int lane_scan(int v, int none, Op op) {
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));  // from 1, 2, 4, 8 lanes below in 16
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));  // lane 15 to the next 16
    v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));  // lane 31 to the upper half
    return v;
}
__device__ __forceinline__ int lane_max(int v, int none) {
    return __builtin_amdgcn_readlane(lane_scan(v, none, [](int x, int y) { return x > y ? x : y; }), 63);
}
__device__ __forceinline__ int lane_min(int v, int none) {
    return __builtin_amdgcn_readlane(lane_scan(v, none, [](int x, int y) { return x < y ? x : y; }), 63);
}

// row / group (a row stays below 2^24).
__device__ __forceinline__ int token_of(const AttnArgs& a, int row) {
    return a.plan.group_magic ? (int)__umulhi((uint32_t)row, a.plan.group_magic) : row;
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

// The same of a token that the wave's lanes have alike, with the new tokens of
// that sequence (none of a token in no sequence): 64 starts a load.
struct Place {
    int s, q0, q1;
};
__device__ __forceinline__ Place place_of(const AttnArgs& a, int t, int lane) {
    if (!a.starts) return {t, t, t + 1};
    Place p = {-1, 0, 0};
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        const int at = s0 + lane < a.n_seqs ? s0 + lane : a.n_seqs - 1;
        const int start = a.starts[at], end = a.starts[at + 1];
        const uint64_t votes = __ballot(s0 + lane < a.n_seqs && start <= t);
        if (votes) {
            const int l = 63 - __builtin_clzll(votes);
            p.s = s0 + l;
            p.q0 = clampi(__builtin_amdgcn_readlane(start, l), 0, a.n_tokens);
            p.q1 = clampi(__builtin_amdgcn_readlane(end, l), p.q0, a.n_tokens);
        }
        if (votes != ~0ull) break;
    }
    if (t < p.q0 || t >= p.q1) p.s = -1;
    return p;
}

// Tokens [lo, hi) and [0, sink) of a unit's n are seen.
struct Limits {
    int lo, hi, sink;
};

// Of a unit of n tokens, from unclamped ends.
__device__ __forceinline__ Limits limits_of(const AttnArgs& a, int hi, int lo, int sink, int n) {
    Limits l = {0, clampi(hi, 0, n), 0};
    if (a.window) {
        l.lo = clampi(lo, 0, n);
        l.sink = clampi(sink, 0, l.hi);
    }
    return l;
}

// What a new token sees of its own sequence's tokens and of the prefix, `upto`
// of its own ones lying at or before it (up to 2^30, and 2^22 below zero, as
// prefix_len and window: nothing here passes 32 bits).
__device__ __forceinline__ int upto_of(const Seq& q, int tok) { return q.length - q.n + tok + 1; }
__device__ __forceinline__ Limits own_limits(const AttnArgs& a, const Seq& q, int upto) {
    return limits_of(a, upto, upto - a.window, a.sink - a.prefix_len, q.length);
}
__device__ __forceinline__ Limits prefix_limits(const AttnArgs& a, int upto) {
    return limits_of(a, upto < 0 ? a.prefix_len + upto : a.prefix_len, a.prefix_len - a.window + upto, a.sink,
                     a.prefix_len);
}

// The 32-token tiles a unit goes through: `sink` ones from 0, then lo..hi-1.
struct Tiles {
    int sink, lo, hi;
    __device__ __forceinline__ int steps(const RowSplit& s) const { return (count() + s.step() - 1) >> s.log2_tiles; }
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
    const int rows = q.n * a.group, r0 = tile << a.plan.own.log2_rows, r1 = r0 + (1 << a.plan.own.log2_rows);
    const int last = (r1 < rows ? r1 : rows) - 1;
    Limits l = own_limits(a, q, upto_of(q, token_of(a, last)));
    if (a.window) l.lo = own_limits(a, q, upto_of(q, token_of(a, r0))).lo;
    return tiles_of(l);
}

// Tiles of the prefix: from the window of the batch's first position.
__device__ __forceinline__ Tiles prefix_tiles(const AttnArgs& a, int least_upto) {
    Limits l = prefix_limits(a, least_upto);
    l.hi = a.prefix_len;
    if (a.window) l.sink = clampi(a.sink, 0, l.hi);
    return tiles_of(l);
}

__device__ __forceinline__ bool sees(const Limits& l, int token, bool there) {
    return there & (token < l.hi) & ((token >= l.lo) | (token < l.sink));
}

// An infinity of an fp16 cache whose weight is rounded to zero gives NaN in the
// product, where the formula has an infinity.  (Tiles that a row sees a part of
// keep infinities apart anyway; bf16 weights get to zero only 2^-126 below.)  For
// rows whose result is NaN though its sum of weights is not, the values that the
// row sees are looked through: bit k of `up` is set by a +inf in column(k),
// k < K, of `down` by a -inf, of both by a NaN.
struct Infinities {
    uint32_t up, down;
    __device__ __forceinline__ float of(int k, float otherwise) const {
        const bool u = up >> k & 1, d = down >> k & 1;
        return u == d ? otherwise : u ? __builtin_inff() : -__builtin_inff();
    }
};
// The kernel's arguments (its first parameter) for such a path: read where it is
// taken, not kept for it (kept, they cost 0.7 us of each call).
__device__ __forceinline__ const AttnArgs& args_again() {
    const AttnArgs* p = (const AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}
template <int D, int K, class Column>
__device__ __forceinline__ void find_infinities(const AttnArgs& a, const int32_t* table, int h, const Limits& l,
                                                Column column, Infinities& found) {
    typedef short bits_t __attribute__((ext_vector_type(8)));
    constexpr uint32_t kAll = K == 32 ? ~0u : (1u << K) - 1;
#pragma unroll 1
    for (int t0 = 0; t0 < l.hi && (found.up & found.down) != kAll; t0 += 8) {  // eight tokens of a column lie together
        if (t0 >= l.sink && t0 + 8 <= l.lo) t0 = l.lo / 8 * 8;
        if (t0 >= l.hi) break;
        const uint32_t block = (uint32_t)t0 / 32, page = block / a.page_blocks;
        const uint32_t id = (uint32_t)table[page];
        if (id >= a.n_pages) continue;
        const int64_t at = ((int64_t)id * a.kv_heads + h) * a.page_blocks + (block - page * a.page_blocks);
        const short* const from = static_cast<const short*>(a.cv) + (at * 4 + (t0 % 32) / 8) * (8 * D);
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
            const bits_t v = *reinterpret_cast<const bits_t*>(from + column(k) * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int size = v[j] & 0x7fff;
                if (size < 0x7c00 || !sees(l, t0 + j, true)) continue;
                if (size > 0x7c00 || v[j] > 0) found.up |= 1u << k;
                if (size > 0x7c00 || v[j] < 0) found.down |= 1u << k;
            }
        }
    }
}

// A value of a row that the main kernel finishes, if it is NaN.  (Inlined, it cost
// 64 sequences of 30 tokens x 8 kv heads 0.6 of 11.1 us.)
template <int D>
__attribute__((noinline)) __device__ float lost_value(const AttnArgs& a, int seq, int h, int lo, int hi, int sink, int col,
                                                      float x) {
    if (x == x) return x;
    Infinities found = {0, 0};
    find_infinities<D, 1>(a, a.pages + (int64_t)seq * a.pages_per_seq, h, Limits{lo, hi, sink}, [&](int) { return col; }, found);
    return found.of(0, x);
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

// Cost of an entry: its own, and its steps'.
__device__ __forceinline__ uint32_t entry_cost(const RowSplit& s, int steps) {
    return steps ? s.lead + ((uint32_t)steps << s.log2_cost) : 0u;
}

// A unit's part in a piece of a line.
struct Job {
    int h, seq, tile;
    Seq sq;
    Tiles tiles;
    int s0, s1;   // its steps
    float* part;  // where its sums go; null: these are all of the rows', they go to the output
};

// What is left to a workgroup (or wave) of its piece: [x, x1), which began at x0.
struct Piece {
    uint64_t per, x0, x, x1;
    int place;
};

struct Line {
    Piece prefix, own;
    int prefix_tile;       // of this workgroup, where row tiles go abreast; else -1
    uint64_t head_cost;    // of a kv head's own entries
    int own_entries;       // of a kv head
    uint32_t prefix_cost;  // of an entry of the prefix
    Tiles prefix_tiles;
    bool lanes;            // the own line is a sequence a lane
    bool plain;            // every new token sees the whole prefix
};

__device__ __forceinline__ uint64_t line_quotient(const Line& l, uint64_t x, uint64_t d) {
    return l.lanes ? quotient((uint32_t)x, (uint32_t)d) : quotient(x, d);
}

// The piece of a line of `all` at a place of several (past them: none).
__device__ __forceinline__ Piece piece_of(const Line& l, uint64_t all, int places, int place, const RowSplit& s) {
    Piece p = {1, 0, 0, 0, place};
    if (!places) return p;
    // (with 32-bit costs a little more than the quotient will do: every place has the same)
    if (l.lanes) p.per = (uint32_t)((float)(uint32_t)all * __builtin_amdgcn_rcpf((float)places) * (1.0f + 0x1p-20f)) + 1;
    else p.per = quotient(all + (uint64_t)(places - 1), (uint64_t)places);
    if (p.per < 1u << s.log2_cost) p.per = 1u << s.log2_cost;  // a step
    p.x = p.x0 = p.per * (uint64_t)place;
    p.x1 = (uint32_t)place >= (uint32_t)places ? 0 : p.x0 + p.per < all ? p.x0 + p.per : all;
    return p;
}

// The slots of an entry whose cost begins at x.
__device__ __forceinline__ Pieces pieces_of(const Line& l, uint64_t per, const RowSplit& s, uint64_t x, uint32_t cost,
                                            int unit) {
    if (!cost) return {0, 0};
    const uint32_t w0 = (uint32_t)line_quotient(l, x + s.lead, per);
    const uint32_t w1 = (uint32_t)line_quotient(l, x + cost - (1u << s.log2_cost), per);
    return {w0 + (uint32_t)unit, w1 - w0 + 1};
}

// Steps of an entry at x, cost c, whose first point, of x + lead + (step << log2_cost), lies in what is left of the
// piece; moves on behind them.  True: all of the entry's steps begin in the piece.
__device__ __forceinline__ bool take_steps(Piece& p, const RowSplit& s, uint64_t x, uint32_t c, Job& job) {
    const uint32_t up = (1u << s.log2_cost) - 1;
    const uint64_t stop = p.x1 < x + c ? p.x1 : x + c;
    const uint32_t from = (uint32_t)(p.x - x), to = (uint32_t)(stop - x);
    job.s0 = (int)((from > (uint32_t)s.lead ? from - s.lead + up : 0u) >> s.log2_cost);
    job.s1 = (int)((to > (uint32_t)s.lead ? to - s.lead + up : 0u) >> s.log2_cost);
    p.x = stop;
    return x + s.lead >= p.x0 && x + c - (up + 1) < p.x0 + p.per;
}

template <class S>
__device__ __forceinline__ void keep_seq(const AttnArgs& a, S& sh, int s, const Seq& q) {
    if (s < kSeqs) {
        sh.start[s] = a.starts ? a.starts[s] : s;
        sh.end[s] = q.q0 + q.n;
        sh.upto[s] = upto_of(q, -q.q0);
    }
}

// (of a sequence without new tokens: more than any)
__device__ __forceinline__ int least_upto_of(const Seq& q) { return q.n ? upto_of(q, 0) : 1 << 30; }

__device__ __forceinline__ void set_prefix(const AttnArgs& a, Line& line, int least_upto) {
    if (!a.plan.prefix_entries) return;
    line.prefix_tiles = prefix_tiles(a, least_upto);
    line.prefix_cost = entry_cost(a.plan.prefix, line.prefix_tiles.steps(a.plan.prefix));
}

// The own line of up to 64 sequences with a row tile each: sequence s in lane
// s, kept in LDS, where all waves write the same.  False: one has more rows.
template <class S>
__device__ __forceinline__ bool line_in_lanes(const AttnArgs& a, S& sh, Line& line) {
    const int lane = threadIdx.x & 63;
    const AttnPlan& p = a.plan;
    const bool on = lane < a.n_seqs;
    Seq q = {0, 0, 0};
    if (on) q = seq_at(a, lane);
    if (__any(q.n * a.group > 1 << p.own.log2_rows)) return false;
    line.plain = !a.window && !__any(q.length < q.n);
    int least = 1 << 30;
    if (p.prefix_entries && !line.plain) {
        if (a.window) least = lane_min(least_upto_of(q), 1 << 30);
        if (on) keep_seq(a, sh, lane, q);
        __syncthreads();
    }
    set_prefix(a, line, least);
    const uint32_t mine = q.n ? entry_cost(p.own, own_tiles(a, q, 0).steps(p.own)) : 0u;
    const uint32_t upto = (uint32_t)lane_scan((int)mine, 0, [](int x, int y) { return x + y; });
    sh.lane_line[0][lane] = on ? upto - mine : 0x7fffffffu;
    sh.lane_line[1][lane] = mine;
    sh.lane_line[2][lane] = q.q0;
    sh.lane_line[3][lane] = q.n;
    sh.lane_line[4][lane] = q.length;
    line.head_cost = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    line.own_entries = a.n_seqs;
    return true;
}

// The own line of any batch: cost[0..entries] (cost before an entry) and
// info[entry] (sequence << 16 | row tile) in LDS.
template <class S>
__device__ __forceinline__ void line_in_lds(const AttnArgs& a, uint64_t* cost, uint32_t* info, S& sh, Line& line,
                                            bool writes) {
    uint64_t* const scratch = sh.scratch;
    const int tid = threadIdx.x;
    const AttnPlan& p = a.plan;
    int* const meta_first = reinterpret_cast<int*>(a.meta + meta_first_at());
    int base = 0, least = 1 << 30;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kThreads) {
        const int s = s0 + tid;
        uint32_t n = 0;
        if (s < a.n_seqs) {
            const Seq q = seq_at(a, s);
            n = (uint32_t)((q.n * a.group + (1 << p.own.log2_rows) - 1) >> p.own.log2_rows);
            least = least_upto_of(q) < least ? least_upto_of(q) : least;
            keep_seq(a, sh, s, q);
        }
        uint32_t total;
        const uint32_t at = base + block_scan<uint32_t>(n, reinterpret_cast<uint32_t*>(scratch), total) - n;
        for (uint32_t r = 0; r < n && at + r < (uint32_t)p.own_entries; ++r) info[at + r] = (uint32_t)s << 16 | r;
        if (writes && s < a.n_seqs) meta_first[s] = (int)at;
        base += (int)total;
    }
    const int entries = base < p.own_entries ? base : p.own_entries;
    line.plain = false;
    if (p.prefix_entries && a.window) {
        least = lane_min(least, 1 << 30);
        int* const top = reinterpret_cast<int*>(scratch);
        __syncthreads();
        if ((tid & 63) == 0) top[tid >> 6] = least;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) least = top[w] < least ? top[w] : least;
    }
    least = uniform(least);
    set_prefix(a, line, least);
    __syncthreads();
    uint64_t sum = 0;
    for (int e0 = 0; e0 < entries; e0 += kThreads) {
        const int e = e0 + tid;
        uint64_t c = 0;
        if (e < entries)
            c = entry_cost(p.own, own_tiles(a, seq_at(a, (int)(info[e] >> 16)), (int)(info[e] & 0xffff)).steps(p.own));
        uint64_t total;
        const uint64_t at = sum + block_scan<uint64_t>(c, scratch, total) - c;
        if (e < entries) cost[e] = at;
        sum += total;
    }
    if (tid == 0) cost[entries] = sum;
    line.head_cost = uniform(sum);
    line.own_entries = uniform(entries);
    __syncthreads();
}

template <class S>
__device__ __forceinline__ Line build_line(const AttnArgs& a, uint64_t* cost, uint32_t* info, S& sh) {
    const AttnPlan& p = a.plan;
    const int grid = 1 << p.log2_workgroups;
    const bool writes = (int)blockIdx.x == grid - 1;
    Line line;
    line.prefix_cost = 0;
    line.prefix_tiles = {0, 0, 0};
    line.lanes = p.lanes && line_in_lanes(a, sh, line);
    if (!line.lanes) line_in_lds(a, cost, info, sh, line, writes);
    // The workgroups are divided between the lines by what they cost (a launch
    // of both phases in every workgroup pays for beginning and ending twice).
    // Those of an XCD (workgroup b runs on XCD b % 8) have pieces that follow
    // each other, so that the row tiles of a kv head, which read the same keys,
    // share an L2, and every XCD has its part of either line.
    const uint64_t prefix = (uint64_t)line.prefix_cost * (uint64_t)(p.prefix_entries * a.kv_heads);
    const uint64_t own = line.head_cost * (uint64_t)a.kv_heads;
    const uint64_t own_by_group = p.own.shared ? own : own >> 2;
    int eighth = grid / 8;  // workgroups of an XCD for the prefix
    if (!prefix) eighth = 0;
    else if (own)
        eighth = clampi((int)((float)prefix * __builtin_amdgcn_rcpf((float)(prefix + own_by_group)) * (float)eighth), 1,
                        eighth - 1);
    const int xcd = (int)(blockIdx.x & 7), at = (int)(blockIdx.x >> 3), rest = grid / 8 - eighth;
    // Several row tiles go abreast, each with its own workgroup, over the same
    // steps of a head's prefix, which they then read from the L2 (behind each
    // other 256 rows took 175 us for 98304 tokens, 150 abreast), while there
    // are at least eight workgroups for each.
    const int tiles = p.prefix_entries, abreast = tiles > 1 && tiles <= eighth ? tiles : 1;
    const int place = xcd * eighth + at, group_of = place / abreast;
    line.prefix_tile = abreast > 1 ? place - group_of * abreast : -1;
    line.prefix = piece_of(line, abreast > 1 ? (uint64_t)line.prefix_cost * (uint64_t)a.kv_heads : prefix, eighth * 8 / abreast,
                           at < eighth ? group_of : -1, p.prefix);
    const int group = at < eighth ? -1 : xcd * rest + at - eighth;
    if (p.own.shared) line.own = piece_of(line, own, rest * 8, group, p.own);
    else line.own = piece_of(line, own, rest * 8 * kWaves, group < 0 ? -1 : group * kWaves + uniform((int)(threadIdx.x >> 6)), p.own);
    if (writes) {  // for the join
        Pieces* const pieces = reinterpret_cast<Pieces*>(a.meta + meta_pieces_at(a.n_seqs));
        if (threadIdx.x == 0) *reinterpret_cast<MetaHead*>(a.meta) = MetaHead{line.own_entries, line.lanes, abreast, 0};
        const int entries = p.prefix_entries + line.own_entries;
        for (int h = threadIdx.x >> 6; h < a.kv_heads; h += kWaves)
            for (int i = threadIdx.x & 63; i < entries; i += 64) {
                Pieces c;
                if (i < p.prefix_entries) {
                    const int unit = abreast > 1 ? h : h * p.prefix_entries + i;
                    c = pieces_of(line, line.prefix.per, p.prefix, unit * (uint64_t)line.prefix_cost, line.prefix_cost,
                                  unit);
                    if (abreast > 1) c.slot0 = c.slot0 * (uint32_t)abreast + (uint32_t)i;
                } else {
                    const int e = i - p.prefix_entries;
                    const uint64_t e0 = line.lanes ? (uint64_t)(uint32_t)sh.lane_line[0][e & 63] : cost[e];
                    const uint32_t c0 = line.lanes ? (uint32_t)sh.lane_line[1][e & 63] : (uint32_t)(cost[e + 1] - e0);
                    c = pieces_of(line, line.own.per, p.own, h * line.head_cost + e0, c0, h * line.own_entries + e);
                }
                pieces[h * entries + i] = c;
            }
    }
    return line;
}

// The next unit of the piece of the prefix; false when there is none.
__device__ __forceinline__ bool next_prefix(const AttnArgs& a, Line& line, Job& job, int dim) {
    Piece& p = line.prefix;
    if (p.x >= p.x1) return false;
    const int unit = (int)line_quotient(line, p.x, line.prefix_cost), n = a.plan.prefix_entries;
    uint32_t slot = (uint32_t)(p.place + unit);
    if (line.prefix_tile >= 0) {
        job.h = unit;
        job.tile = line.prefix_tile;
        slot = slot * (uint32_t)n + (uint32_t)job.tile;
    } else {
        job.h = n > 1 ? (int)quotient((uint32_t)unit, (uint32_t)n) : unit;
        job.tile = unit - job.h * n;
    }
    job.seq = 0;
    job.sq = {0, a.n_tokens, a.prefix_len};
    job.tiles = line.prefix_tiles;
    take_steps(p, a.plan.prefix, unit * (uint64_t)line.prefix_cost, line.prefix_cost, job);
    job.part = a.part + (uint64_t)slot * slot_floats(1 << a.plan.prefix.log2_rows, dim);
    return true;
}

// The next unit of the piece of the sequences' own tokens; false when there is none.
template <class S>
__device__ __forceinline__ bool next_own(const AttnArgs& a, Line& line, const uint64_t* cost, const uint32_t* info,
                                         const S& sh, Job& job, int dim) {
    Piece& p = line.own;
    if (p.x >= p.x1) return false;
    uint64_t x;  // where the entry begins
    uint32_t c;
    int e;
    job.h = (int)line_quotient(line, p.x, line.head_cost);
    const uint64_t head0 = job.h * line.head_cost, at = p.x - head0;
    if (line.lanes) {
        const int lane = threadIdx.x & 63;
        const int first = sh.lane_line[0][lane], mine = sh.lane_line[1][lane];
        const int q0 = sh.lane_line[2][lane], n = sh.lane_line[3][lane], length = sh.lane_line[4][lane];
        e = 63 - __builtin_clzll(__ballot(first <= (int)at));
        x = head0 + (uint32_t)__builtin_amdgcn_readlane(first, e);
        c = (uint32_t)__builtin_amdgcn_readlane(mine, e);
        job.sq = {__builtin_amdgcn_readlane(q0, e), __builtin_amdgcn_readlane(n, e),
                  __builtin_amdgcn_readlane(length, e)};
        job.seq = e;
        job.tile = 0;
    } else {
        int lo = 0, hi = line.own_entries;  // the entry: cost[lo] <= at < cost[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (cost[mid] <= at) lo = mid;
            else hi = mid;
        }
        e = uniform(lo);
        x = uniform(cost[e]);
        c = (uint32_t)uniform((int)(cost[e + 1] - x));
        x += head0;
        const uint32_t who = (uint32_t)uniform((int)info[e]);
        job.seq = (int)(who >> 16);
        job.tile = (int)(who & 0xffff);
        const Seq q = seq_at(a, job.seq);
        job.sq = {uniform(q.q0), uniform(q.n), uniform(q.length)};
    }
    job.tiles = own_tiles(a, job.sq, job.tile);
    const bool alone = take_steps(p, a.plan.own, x, c, job) && !a.plan.prefix_entries;
    job.part = alone ? nullptr
                     : a.own_part + (uint64_t)(p.place + job.h * line.own_entries + e) *
                                        slot_floats(1 << a.plan.own.log2_rows, dim);
    return true;
}

// ---- a row's result ------------------------------------------------------------------------------------------------

// K groups of N (4, 2 or 1) consecutive columns, from `col` on and `stride`
// apart: the gates of a row, and the row gated, in the output's type.
template <int K, int N>
__device__ __forceinline__ void load_gates(const AttnArgs& a, int t, int head, int col, int stride, float (&g)[K][N]) {
    if (!a.gate.data) return;
    const int64_t at = t * a.gate.token_stride + head * a.gate.head_stride + col;
    auto get = [&](auto zero) {
        typedef decltype(zero) T;
        typedef T vec_t __attribute__((ext_vector_type(N > 1 ? N : 2)));
        const T* const from = static_cast<const T*>(a.gate.data) + at;
        if (N > 1 && a.gate.vec) {
            vec_t w[K];
#pragma unroll
            for (int k = 0; k < K; ++k) w[k] = *reinterpret_cast<const vec_t*>(from + k * stride);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) g[k][j] = (float)w[k][j];
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) g[k][j] = (float)from[k * stride + j];
        }
    };
    if (a.gate.dtype == QW35_HIP_DTYPE_F32) get(0.0f);
    else if (a.gate.dtype == QW35_HIP_DTYPE_F16) get((_Float16)0.0f);
    else get((__bf16)0.0f);
}

template <int K, int N>
__device__ __forceinline__ void finish(const AttnArgs& a, int t, int head, int col, int stride, const float (&g)[K][N],
                                       float (&v)[K][N]) {
    if (a.gate.data) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) v[k][j] /= 1.0f + __expf(-g[k][j]);
    }
    const int64_t at = t * a.out.token_stride + head * a.out.head_stride + col;
    auto put = [&](auto zero) {
        typedef decltype(zero) T;
        typedef T vec_t __attribute__((ext_vector_type(N > 1 ? N : 2)));
        T* const to = static_cast<T*>(a.out.data) + at;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (N > 1 && a.out.vec) {
                vec_t w;
#pragma unroll
                for (int j = 0; j < N; ++j) w[j] = (T)v[k][j];
                *reinterpret_cast<vec_t*>(to + k * stride) = w;
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) to[k * stride + j] = (T)v[k][j];
            }
        }
    };
    if (a.out.dtype == QW35_HIP_DTYPE_F32) put(0.0f);
    else if (a.out.dtype == QW35_HIP_DTYPE_F16) put((_Float16)0.0f);
    else put((__bf16)0.0f);
}

// ---- the kernel ----------------------------------------------------------------------------------------------------

// Lanes l and l ^ 32 (l ^ 16): both values, in either.  (Elements of the builtin's
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
__device__ __forceinline__ Pair pair_xor16(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = p[0], b = p[1];
    return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
// Over the lanes of a row: l, l ^ 32 and, of 16 rows, l ^ 16.
template <int kRows>
__device__ __forceinline__ float row_max(float v) {
    if constexpr (kRows == 16) {
        const Pair q = pair_xor16(v);
        v = fmaxf(q.a, q.b);
    }
    const Pair p = pair_xor32(v);
    return fmaxf(p.a, p.b);
}
template <int kRows>
__device__ __forceinline__ float row_sum(float v) {
    if constexpr (kRows == 16) {
        const Pair q = pair_xor16(v);
        v = q.a + q.b;
    }
    const Pair p = pair_xor32(v);
    return p.a + p.b;
}

// v *= f in v's own registers, accumulation ones in the kernels that have them
// (the compiler's products would go to others, and the accumulators with them
// from one kind to the other in every tile).  The compiler does not count the
// wait states from the matrix instructions that wrote v to inline assembly (12
// of 32 rows, 8 of 16).  With own tiles a tile's scores lie between, with shared
// ones the choice whether to come here, a lane exchange and an exponential; the
// tests count them in the built library.  (s_nop here: 0.5 us of a call of 53.)
template <bool kAgpr, class Acc>
__device__ __forceinline__ void scale_in_place(Acc& v, float f) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Acc) / 4); ++i) {
        float x = v[i];
        if constexpr (kAgpr) {
            float y;
            asm("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %2, %1\n\tv_accvgpr_write_b32 %0, %1" : "+a"(x), "=&v"(y) : "v"(f));
        } else {
            asm("v_mul_f32 %0, %1, %0" : "+v"(x) : "v"(f));
        }
        v[i] = x;
    }
}

// A part of a row whose exponents count from m, seen from the largest `top` of several: exp2(m - top), 0 for a part
// with nothing.
__device__ __forceinline__ float part_weight(float m, float top) {
    // (never zero otherwise: an infinity in a part that hardly counts stays one)
    return m == -__builtin_inff() ? 0.0f : fmaxf(__builtin_amdgcn_exp2f(m - top), 1e-37f);
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

// KB i of such a copy.
__device__ __forceinline__ void copy_1kb(const uint8_t* from, uint8_t* to, int i, int lane) {
    copy_kb<1>(from + i * 1024, to + i * 1024, lane);
}

template <int D>
struct Shared {
    static constexpr int kRing = D == 256 ? 128 * 1024 : 64 * 1024;
    uint8_t ring[kRing];  // tiles on their way; at a unit's end the waves' sums
    float m[kWaves][32];
    float l[kWaves][32];
    Limits all[kWaves];
    // of the first sequences, for the rows of the prefix: starts[s], the end of its new tokens, and how many own
    // tokens a new one sees, less its index
    int start[kSeqs], end[kSeqs], upto[kSeqs];
    uint32_t marks[kWaves][32 * D / 16];
    uint64_t scratch[kWaves];
    int lane_line[5][64];  // of a line in lanes: cost before, cost, and q0, n, length
};

// Raw granules of a tile: 16 bytes of a 16-bit cache, 8 of an e4m3 one.
template <bool F8>
using raw8 = std::conditional_t<F8, uint2, uint4_t>;

template <class E, bool F8>
__device__ __forceinline__ typename E::vec8 operand(raw8<F8> w) {
    if constexpr (F8) return E::from_e4m3(w);
    else return __builtin_bit_cast(typename E::vec8, w);
}

// kRows: rows of a wave's tile, 16 or 32.
template <int D, class E, bool F8, int kRows>
struct Unit {
    typedef typename E::vec8 vec8;
    typedef raw8<F8> raw;
    typedef std::conditional_t<kRows == 32, acc_t, float4_t> acc;  // of a matrix instruction
    static constexpr int kAcc = sizeof(acc) / 4;
    static constexpr int kGroups = 64 / kRows;      // lanes of a row
    static constexpr int kM = D / (8 * kGroups);    // contraction steps of a score
    static constexpr int kB = 32 / kRows;           // matrix tiles of the scores
    static constexpr int kT = D / kRows;            // column tiles of the output
    static constexpr int kK = 4 / kGroups;          // token steps of the output
    static constexpr int kScores = kB * kAcc;       // of a lane
    static constexpr int kQuads = kT * kAcc / 4;    // 4-column groups of the output in a lane: group i holds columns
    static constexpr int kQuadCols = 4 * kGroups;   // kQuadCols i + 4 g ..
    static constexpr int kElem = F8 ? 1 : 2;
    static constexpr int kTile = 32 * D * kElem;  // bytes of a tile's keys, and of its values
    static constexpr int kKb = kTile / 1024;
    static constexpr int kRing = Shared<D>::kRing;
    // The exponents' reference follows the maximum only when that has risen by
    // 2^8: sums then hold up to 2^8 times a row's largest term, which costs
    // neither type precision, and most tiles rescale nothing.  It follows to 2^7
    // below the maximum of fp16: terms of up to 2^15 fit, and one is lost below
    // 2^-32 of a row's largest instead of 2^-25 (31 terms of 2^-27 beside one
    // whose value is zero were).
    static constexpr float kLift = std::is_same_v<E, Half> ? 7.0f : 0.0f;
    static constexpr float kRise = 8.0f + kLift;
    static constexpr bool kLoses = std::is_same_v<E, Half> && !F8;  // weights of zero may meet infinities
    static constexpr bool kAgpr = D == 256;  // one wave a SIMD, accumulation registers beside the others

    const AttnArgs& a;
    Shared<D>& sh;
    const int lane, wave, n, g;  // this lane's row of a tile, and which of the row's lanes it is

    __device__ Unit(const AttnArgs& a_, Shared<D>& sh_)
        : a(a_), sh(sh_), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          n(threadIdx.x & (kRows - 1)), g((threadIdx.x & 63) / kRows) {}

    // What a wave carries through its tiles.
    struct Rows {
        vec8 q[kM];
        acc o[kT];
        float mx, l;
        Limits lim;
        int all_lo, all_hi, all_sink;  // what every row of the wave sees
        float scale;
        bool marked;  // infinities to add at the end
    };

    // The granule of step m for score tile b / of column tile t and token step kk.
    __device__ __forceinline__ vec8 key(const uint8_t* tile, int m, int b) const {
        // which token is row n of the product: token(j) of the lane that gets it
        const int tok = kRows == 32 ? (n & 19) | (n & 4) << 1 | (n & 8) >> 1 : (n >> 2) * 8 + b * 4 + (n & 3);
        return operand<E, F8>(*reinterpret_cast<const raw*>(tile + ((kGroups * m + g) * 32 + tok) * 8 * kElem));
    }
    __device__ __forceinline__ vec8 value(const uint8_t* tile, int t, int kk) const {
        return operand<E, F8>(
            *reinterpret_cast<const raw*>(tile + ((kGroups * kk + g) * D + t * kRows + n) * 8 * kElem));
    }
    // Token of a lane's score j.
    __device__ __forceinline__ int token(int j) const { return kRows == 32 ? (j & 8) * 2 + g * 8 + (j & 7) : g * 8 + j; }

    struct Nothing {
        __device__ __forceinline__ void operator()(int) const {}
    };

    // `beside`(step): other work, a part after the matrix instructions of each step.
    static constexpr int kScoreSteps = kM * kB, kValueSteps = kK * kT;
    template <class F = Nothing>
    __device__ __forceinline__ void scores(const uint8_t* keys, const Rows& w, acc (&s)[kB], F beside = {}) const {
        constexpr int kSteps = kScoreSteps, kAhead = kSteps < 4 ? kSteps : 4;
        vec8 k[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) k[i] = key(keys, i / kB, i % kB);
#pragma unroll
            for (int b = 0; b < kB; ++b) s[b] = acc{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const vec8 kk = k[i % kAhead];
            if (i + kAhead < kSteps) k[i % kAhead] = key(keys, (i + kAhead) / kB, (i + kAhead) % kB);
            s[i % kB] = E::mfma(kk, w.q[i / kB], s[i % kB]);
            beside(i);
            if (!std::is_same_v<F, Nothing>) __builtin_amdgcn_sched_barrier(0);
        }
        if (std::is_same_v<F, Nothing>) interleave<kSteps, kAhead>();
    }

    // LDS reads kAhead ahead of the matrix instructions that take them.
    template <int kSteps, int kAhead>
    static __device__ __forceinline__ void interleave() {
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
            if (F8) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (m + kAhead < kSteps) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    }

    // Scores that a row does not see leave the softmax.
    __device__ __forceinline__ void mask(const Rows& w, acc (&s)[kB], int t0, bool there) const {
#pragma unroll
            for (int j = 0; j < kScores; ++j)
                s[j / kAcc][j % kAcc] =
                    sees(w.lim, t0 + token(j), there) ? s[j / kAcc][j % kAcc] : -__builtin_inff();
    }

    // The largest of this lane's scores of row tile r.
    static __device__ __forceinline__ float largest(const acc (&s)[kB]) {
        float top = s[0][0];
#pragma unroll
        for (int j = 1; j < kScores; ++j) top = fmaxf(top, s[j / kAcc][j % kAcc]);
        return top;
    }

    // The reference follows the rows' largest scores (`largest`: of this lane's).
    __device__ __forceinline__ void follow(Rows& w, float largest) const {
        if (__builtin_expect(__any(largest * w.scale > w.mx + kRise), 0)) {
            const float m_new = fmaxf(w.mx, row_max<kRows>(largest) * w.scale - kLift);
            const float shrink = m_new == w.mx ? 1.0f : __builtin_amdgcn_exp2f(w.mx - m_new);
            w.l *= shrink;
#pragma unroll
            for (int t = 0; t < kT; ++t) scale_in_place<kAgpr>(w.o[t], shrink);
            w.mx = m_new;
        }
    }

    // The softmax' terms of a tile, and their sums: of the scores j0 .. j1 - 1 of all row tiles' together.
    __device__ __forceinline__ void terms(Rows& w, const acc (&s)[kB], vec8 (&p)[kK], int j0 = 0,
                                          int j1 = kScores) const {
#pragma unroll
        for (int i = j0; i < j1; ++i) {
            const int j = i;
            const float ref = w.mx == -__builtin_inff() ? 0.0f : w.mx;
            const float e = __builtin_amdgcn_exp2f(fmaf(s[j / kAcc][j % kAcc], w.scale, -ref));
            w.l += e;
            p[j / 8][j % 8] = (typename E::elem)e;
        }
    }

    __device__ __forceinline__ void softmax(Rows& w, acc (&s)[kB], int t0, bool masked, bool there,
                                            vec8 (&p)[kK]) const {
        if (masked) mask(w, s, t0, there);
        float top;
        top = largest(s);
        follow(w, top);
        terms(w, s, p);
    }

    template <class F = Nothing>
    __device__ __forceinline__ void add_values(const uint8_t* values, Rows& w, const vec8 (&p)[kK],
                                               F beside = {}) const {
        constexpr int kSteps = kValueSteps, kAhead = kSteps < 4 ? kSteps : 4;
        vec8 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i] = value(values, i / kK, i % kK);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const vec8 vv = v[i % kAhead];
            if (i + kAhead < kSteps) v[i % kAhead] = value(values, (i + kAhead) / kK, (i + kAhead) % kK);
            w.o[i / kK] = E::mfma(vv, p[i % kK], w.o[i / kK]);
            beside(i);
            if (!std::is_same_v<F, Nothing>) __builtin_amdgcn_sched_barrier(0);
        }
        if (std::is_same_v<F, Nothing>) interleave<kSteps, kAhead>();
    }

    // Keeps infinities and NaN of a tile's values, of which some rows see only
    // a part, from the product (all waves of a shared tile come here together).
    template <bool kShared>
    __device__ __forceinline__ void split_off_infinities(uint8_t* tile, Rows& w, int t0, bool there,
                                                         uint32_t* marks) const {
        if (__builtin_expect(!__any(not_finite(tile)), 1)) return;
        mark_infinities(tile, w, t0, there, marks);
        if (kShared) __syncthreads();
        make_finite(tile, kShared ? wave : 0, kShared ? kWaves : 1);
        if (kShared) __syncthreads();
    }

    // 1 KB (512 bytes of e4m3) i of a tile's values, this lane's granule.
    static constexpr int kParts = D / 16;
    __device__ __forceinline__ uint8_t* granule(uint8_t* tile, int i) const { return tile + (i * 64 + lane) * 8 * kElem; }

    // Whether the tile of values holds an infinity or a NaN.
    __device__ __forceinline__ bool not_finite(uint8_t* tile) const {
        typedef short bits_t __attribute__((ext_vector_type(8)));
        bits_t top = {};
#pragma unroll 4
        for (int i = 0; i < kParts; ++i)
            top = __builtin_elementwise_max(
                top, __builtin_bit_cast(bits_t, operand<E, F8>(*reinterpret_cast<const raw*>(granule(tile, i)))) &
                         (short)0x7fff);
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) bad |= top[j] >= E::kInf;
        return bad;
    }

    // Every step-th part from `first` on, without its infinities and NaN.
    __device__ __forceinline__ void make_finite(uint8_t* tile, int first, int step) const {
#pragma unroll 1
        for (int i = first; i < kParts; i += step) {
            typedef std::conditional_t<F8, uint8_t, short> part_t;
            typedef part_t bits_t __attribute__((ext_vector_type(8)));
            bits_t v = *reinterpret_cast<const bits_t*>(granule(tile, i));
            constexpr part_t kSize = F8 ? 0x7f : 0x7fff, kFirst = F8 ? 0x7f : E::kInf;  // (e4m3 has a NaN, no infinities)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (v[j] & kSize) >= kFirst ? part_t(0) : v[j];
            *reinterpret_cast<bits_t*>(granule(tile, i)) = v;
        }
        wait_lds();
    }

    // For a tile with infinities or NaN among its values of which some rows
    // see only a part: what a row does not see must not reach it even as
    // 0 x NaN, which the matrix instruction would add.  The product takes the
    // finite values; which infinities (a NaN is both) a row saw in which column
    // is kept, a bit each, and added when the unit's tiles are done.
    //   marks: [t][sign][kRows], bits of the tile's kRows columns; a lane
    // keeps sign g % 2 of row n.  (No branch here or in the tile loop depends on
    // the lane: the paths would keep copies of the accumulators where they meet.)
    __device__ __forceinline__ void mark_infinities(const uint8_t* tile, Rows& w, int t0, bool there,
                                                    uint32_t* marks) const {
        const int mine = (g & 1) * kRows + n;
        if (!w.marked) {
            w.marked = true;
#pragma unroll 1
            for (int i = 0; i < kT; ++i) marks[i * 2 * kRows + mine] = 0;
        }
#pragma unroll 1
        for (int i = 0; i < kK * kT; ++i) {
            const int t = i / kK, kk = i % kK;
            typedef short bits_t __attribute__((ext_vector_type(8)));
            bits_t v = __builtin_bit_cast(bits_t, value(tile, t, kk));
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
                const short x = v[0], size = x & 0x7fff;
                v = __builtin_shufflevector(v, v, 1, 2, 3, 4, 5, 6, 7, 0);
                const uint64_t up = __ballot(size > E::kInf || x == E::kInf);
                const uint64_t down = __ballot(size > E::kInf || (size == E::kInf && x < 0));
                if ((up | down) == 0) continue;
                uint64_t sign = g & 1 ? down : up;  // kRows columns: of token j, 8 + j ...
                const int at = t0 + kk * 16 + j;
                uint32_t see = 0;
#pragma unroll
                for (int k = 0; k < kGroups; ++k)
                    see |= sees(w.lim, at + 8 * k, there) ? (uint32_t)(sign >> kRows * k) : 0u;
                marks[t * 2 * kRows + mine] |= see;
            }
        }
    }

    __device__ __forceinline__ void add_infinities(Rows& w, const uint32_t* marks) const {
        wait_lds();
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                const uint32_t up = marks[t * 2 * kRows + n], down = marks[t * 2 * kRows + kRows + n];
#pragma unroll
                for (int c = 0; c < kAcc; ++c) {
                    const int col = (c >> 2) * 8 + g * 4 + (c & 3);
                    const float inf = __builtin_inff();
                    w.o[t][c] += (up >> col & 1 ? inf : 0.0f) - (down >> col & 1 ? inf : 0.0f);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    }

    __device__ __forceinline__ bool partly(const Rows& w, int t0, bool there) const {
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

    // Tiles i .. i + 63 (below the count).
    __device__ __forceinline__ void look_up(Pages& p, int i) const {
        const int mine = i + lane < p.count ? i + lane : p.count - 1;
        const uint32_t b = (uint32_t)p.tiles.at(p.first + mine * p.step);
        uint32_t pi = a.plan.page_magic ? __umulhi(b, a.plan.page_magic) : b;  // b / page_blocks, or one more
        if ((int32_t)(b - pi * a.page_blocks) < 0) --pi;
        const int id = p.table[pi];
        // a page outside the cache holds nothing that a row sees
        uint32_t block = ((uint32_t)id * (uint32_t)a.kv_heads + p.h) * a.page_blocks + (b - pi * a.page_blocks);
        asm("" : "+v"(block));  // (a choice of two values, not of two paths)
        p.blocks = (uint32_t)id < a.n_pages ? block : kNoBlock;
    }
    // Tile i, the last looked up or the first of the next 64.
    __device__ __forceinline__ uint32_t block_of(Pages& p, int i) const {
        if (i && (i & 63) == 0) look_up(p, i);
        return (uint32_t)__builtin_amdgcn_readlane((int)p.blocks, i & 63);
    }
    static __device__ __forceinline__ int64_t bytes_at(uint32_t block) {
        return (int64_t)(block == kNoBlock ? 0u : block) * kTile;
    }

    // A job.  kShared: the waves share their tiles; by_wave: each wave has a
    // job of its own (and meets no other in it).
    template <bool kShared>
    __device__ __forceinline__ void run(const Job& job, const RowSplit& split, bool prefix, bool by_wave, bool plain) {
        const int rg = kShared ? wave : by_wave ? 0 : wave & ((1 << split.log2_rg) - 1);
        const int tg = kShared || by_wave ? 0 : wave >> split.log2_rg;
        const int step = split.step();
        const Seq& sq = job.sq;
        const Tiles& tiles = job.tiles;
        const int h = job.h;
        const int row_end = sq.n * a.group;
        const int row0 = (job.tile << split.log2_rows) + rg * kRows;  // this wave's first row

        // this wave's tiles: step * s0 + tg, and every step-th after it
        Pages pages;
        pages.table = prefix ? a.prefix_pages : a.pages + (int64_t)job.seq * a.pages_per_seq;
        pages.tiles = tiles;
        pages.first = job.s0 * step + tg;
        pages.step = step;
        pages.h = h;
        const int end = job.s1 * step < tiles.count() ? job.s1 * step : tiles.count();
        pages.count =
            (kShared || row0 < row_end) && pages.first < end ? (end - pages.first + step - 1) >> split.log2_tiles : 0;
        const uint8_t* const kbase = static_cast<const uint8_t*>(a.ck);
        const uint8_t* const vbase = static_cast<const uint8_t*>(a.cv);

        if (!by_wave) __syncthreads();  // the ring is free
        else wait_lds();
        constexpr int kFit = kShared ? kRing / (2 * kTile) : kRing / kWaves / (2 * kTile);
        static_assert(kRows * D / 4 <= sizeof(sh.marks[0]), "room for the marks");
        constexpr int kMost = kShared ? 6 : 4;
        constexpr int kPairs = kFit < kMost ? kFit : kMost;
        uint32_t* const marks = sh.marks[wave];
        uint8_t* const ring = sh.ring + (kShared ? 0 : wave * (kRing / kWaves));
        uint32_t there_bits = 0;  // of the tiles loaded last, the newest in bit 0
        bool missing = false;     // one of them is not there
        auto note = [&](uint32_t block) {
            there_bits = there_bits << 1 | (block != kNoBlock ? 1u : 0u);
            missing |= block == kNoBlock;
        };
        // shared: this wave's quarter of a pair of tiles
        auto quarter_of = [&](int i, const uint8_t*& from, uint8_t*& to) {
            const uint32_t block = block_of(pages, i);
            note(block);
            const int part = (wave & 1) * (kTile / 2);
            from = (wave < 2 ? kbase : vbase) + bytes_at(block) + part;
            to = ring + (i % kPairs) * 2 * kTile + (wave < 2 ? 0 : kTile) + part;
        };

        Rows w;
        if (pages.count) look_up(pages, 0);
        load_queries(w, sq, h, row0, row_end);
        int loaded = 0;
        if constexpr (kShared) {
            for (; loaded < kPairs - 1 && loaded < pages.count; ++loaded) {
                const uint8_t* from;
                uint8_t* to;
                quarter_of(loaded, from, to);
                copy_kb<kKb / 2>(from, to, lane);
            }
        } else {
            for (; loaded < kPairs && loaded < pages.count; ++loaded) {
                const uint32_t block = block_of(pages, loaded);
                note(block);
                uint8_t* const to = ring + loaded * 2 * kTile;
                copy_kb<kKb>(kbase + bytes_at(block), to, lane);
                copy_kb<kKb>(vbase + bytes_at(block), to + kTile, lane);
            }
        }
        start_rows<kShared>(w, sq, prefix, plain, row0, row_end);
        use_queries(w);  // (here the queries are waited for, not in the tile loop)

        if constexpr (kShared) {
            // In one step the matrix unit makes the next tile's scores while
            // the vector unit turns this one's into the softmax' terms, then
            // the values' product while it looks for the largest of the next.
            constexpr int kEach = kKb / 2;  // a wave's copies of a pair
            acc s[kB];
            float top;
            if (kPairs - 2 < pages.count) wait_vm<(kPairs - 2) * kEach>();  // (a job has a step, and a step a tile)
            else wait_vm<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            scores(ring, w, s);
            top = largest(s);
            // steps between which every row sees all of a tile (none of the sink's)
            const int clear0 = tiles.sink + ((w.all_lo + 31) / 32 > tiles.lo ? (w.all_lo + 31) / 32 - tiles.lo : 0) - pages.first;
            const int clear1 = tiles.sink + w.all_hi / 32 - tiles.lo - pages.first;
            auto see_and_follow = [&](int i) {
                if (i < clear0 || i >= clear1 || missing) {
                    const bool there = there_bits >> (loaded - 1 - i) & 1;
                    const int t0 = tiles.at(pages.first + i) * 32;
                    split_off_infinities<true>(ring + (i % kPairs) * 2 * kTile + kTile, w, t0, there, marks);
                    mask(w, s, t0, there);
                    top = largest(s);
                }
                follow(w, top);
            };
            vec8 p[kK];
            // A tile's copies go out one by one among the matrix instructions:
            // together they would wait for each other (32 KB at 64 bytes a cycle).
            auto step = [&](int i, auto copies) {
                see_and_follow(i);
                if (copies) wait_vm<(kPairs - 3) * kEach>();
                else wait_vm<0>();
                __builtin_amdgcn_s_barrier();  // tile i + 1 is there, and tile i - 1 read by all
                asm volatile("" ::: "memory");
                const uint8_t* from = nullptr;
                uint8_t* to = nullptr;
                if (copies) quarter_of(loaded++, from, to);
                __builtin_amdgcn_sched_barrier(0);
                acc next[kB];
                static_assert(kEach <= kScoreSteps, "a copy a step");
                scores(ring + ((i + 1) % kPairs) * 2 * kTile, w, next, [&](int m) {
                    if (copies && m < kEach) copy_1kb(from, to, m, lane);
                    terms(w, s, p, kScores * m / kScoreSteps, kScores * (m + 1) / kScoreSteps);
                });
                top = -__builtin_inff();
                add_values(ring + (i % kPairs) * 2 * kTile + kTile, w, p, [&](int m) {
#pragma unroll
                    for (int j = kScores * m / kValueSteps; j < kScores * (m + 1) / kValueSteps; ++j) {
                        top = fmaxf(top, next[j / kAcc][j % kAcc]);
                        s[j / kAcc][j % kAcc] = next[j / kAcc][j % kAcc];
                    }
                });
                wait_lds();
            };
            int i = 0;
            for (; i + kPairs - 1 < pages.count; ++i) step(i, std::true_type{});
            for (; i + 1 < pages.count; ++i) step(i, std::false_type{});
            see_and_follow(i);
            terms(w, s, p);
            add_values(ring + (i % kPairs) * 2 * kTile + kTile, w, p);
            wait_lds();
        } else {
            constexpr int kLater = (2 * kPairs - 1) * kKb;  // copies issued after the keys of a tile, or after its values
            for (int i = 0; i < pages.count; ++i) {
                uint8_t* const at = ring + (i % kPairs) * 2 * kTile;
                const bool there = there_bits >> (loaded - 1 - i) & 1;
                const bool more = loaded < pages.count;
                const int t0 = tiles.at(pages.first + i * step) * 32;
                const bool masked = partly(w, t0, there);
                acc s[kB];
                vec8 p[kK];
                if (more) wait_vm<kLater>();
                else wait_vm<0>();
                scores(at, w, s);
                uint32_t block = 0;
                if (more) {
                    wait_lds();
                    block = block_of(pages, loaded);
                    note(block);
                    ++loaded;
                    copy_kb<kKb>(kbase + bytes_at(block), at, lane);
                }
                softmax(w, s, t0, masked, there, p);
                if (more) wait_vm<kLater>();
                if (masked) split_off_infinities<false>(at + kTile, w, t0, there, marks);
                add_values(at + kTile, w, p);
                if (more) {
                    wait_lds();
                    copy_kb<kKb>(vbase + bytes_at(block), at + kTile, lane);
                }
            }
        }
        if (__builtin_expect(w.marked, 0)) add_infinities(w, marks);
        w.l = row_sum<kRows>(w.l);

        const float v_scale = F8 && a.v_scale ? a.v_scale[h] : 1.0f;
        static_assert(kRows * D * 4 <= kRing / kWaves, "a wave's sums of a row tile fit its part of the ring");
        if (!kShared && !by_wave) {
            // The waves of a row group join: each leaves its sums in LDS, then
            // adds up every step-th group of all of theirs.
            if (g == 0) {
                sh.m[wave][n] = w.mx;
                sh.l[wave][n] = w.l;
            }
            leave(w);
            __syncthreads();
            if (split.log2_rg == 0) join_waves<4>(job, rg, tg, row0, row_end, v_scale);
            else join_waves<2>(job, rg, tg, row0, row_end, v_scale);
            return;
        }
        if (kShared && !job.part) __syncthreads();  // (the tiles are read)
        const int row = row0 + n, part_row = rg * kRows + n;
        if (job.part) {
            if (row < row_end) {
                float* const to = job.part + part_row * D + g * 4;
#pragma unroll
                for (int i = 0; i < kQuads; ++i)
                    *reinterpret_cast<float4_t*>(to + i * kQuadCols) = quad(w, i);
                if (g == 0) put_stats(job.part, split, part_row, w.mx, w.l);
            }
        } else {
            leave(w);
            const int tok = token_of(a, row), head = h * a.group + row - tok * a.group;
            const float inv = w.l == 0.0f ? 0.0f : v_scale / w.l;
            if (row < row_end) {
#pragma unroll 1
                for (int i = 0; i < kQuads; i += 4) {
                    float x[4][4], gates[4][4];
                    load_gates(a, sq.q0 + tok, head, i * kQuadCols + g * 4, kQuadCols, gates);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float4_t y = left(wave)[(i + c) * 64 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[c][j] = y[j] * inv;
                    }
                    if constexpr (kLoses) {
                        float all = 0.0f;
#pragma unroll
                        for (int c = 0; c < 16; ++c) all += x[c / 4][c % 4];
                        if (__builtin_expect(all != all && w.l == w.l, 0)) {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                x[c / 4][c % 4] = lost_value<D>(args_again(), job.seq, h, w.lim.lo, w.lim.hi, w.lim.sink,
                                                                (i + c / 4) * kQuadCols + g * 4 + c % 4, x[c / 4][c % 4]);
                        }
                    }
                    finish(a, sq.q0 + tok, head, i * kQuadCols + g * 4, kQuadCols, gates, x);
                }
            }
            wait_lds();
        }
    }

    // A row tile's sums in LDS, in lane order.
    __device__ __forceinline__ float4_t* left(int by) const {
        return reinterpret_cast<float4_t*>(sh.ring + by * (kRing / kWaves));
    }
    __device__ __forceinline__ void leave(const Rows& w) const {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) left(wave)[i * 64 + lane] = quad(w, i);
    }
    static __device__ __forceinline__ float4_t quad(const Rows& w, int i) {
        const acc& v = w.o[i * 4 / kAcc];
        const int c = i * 4 % kAcc;
        return float4_t{v[c], v[c + 1], v[c + 2], v[c + 3]};
    }

    template <int kStep>
    __device__ __forceinline__ void join_waves(const Job& job, int rg, int tg, int row0, int row_end,
                                               float v_scale) const {
        constexpr int kRg = kWaves / kStep, K = kQuads / kStep;
        float weight[kStep], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kStep; ++v) {
            weight[v] = sh.m[rg + v * kRg][n];
            top = fmaxf(top, weight[v]);
        }
#pragma unroll
        for (int v = 0; v < kStep; ++v) {
            weight[v] = part_weight(weight[v], top);
            sum += weight[v] * sh.l[rg + v * kRg][n];
        }
        const int row = row0 + n;
        if (row >= row_end) return;
        float x[K][4];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float4_t acc4 = {0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < kStep; ++v) acc4 += weight[v] * left(rg + v * kRg)[(tg + k * kStep) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[k][j] = acc4[j];
        }
        // (a workgroup joins its waves for the prefix only: its rows have other parts too)
        const int part_row = rg * kRows + n;
        float* const to = job.part + part_row * D + kQuadCols * tg + 4 * g;
#pragma unroll
        for (int k = 0; k < K; ++k)
            *reinterpret_cast<float4_t*>(to + k * kQuadCols * kStep) = float4_t{x[k][0], x[k][1], x[k][2], x[k][3]};
        if (tg == 0 && g == 0) put_stats(job.part, a.plan.prefix, part_row, top, sum);
    }

    // This lane's queries (asked for; use_queries waits).
    __device__ __forceinline__ void load_queries(Rows& w, const Seq& sq, int h, int row0, int row_end) const {
        const int row = row0 + n;
        const bool on = row < row_end;
        const int tok = on ? token_of(a, row) : 0;
        const int t = sq.q0 + tok, head = h * a.group + (on ? row - tok * a.group : 0);
        const typename E::elem* p = static_cast<const typename E::elem*>(a.q.data) + t * a.q.token_stride +
                                    head * a.q.head_stride + g * 8;
#pragma unroll
        for (int m = 0; m < kM; ++m) w.q[m] = vec8{};
        if (on && a.q.vec) {
#pragma unroll
            for (int m = 0; m < kM; ++m) w.q[m] = *reinterpret_cast<const vec8*>(p + m * 8 * kGroups);
        } else if (on) {
#pragma unroll
            for (int m = 0; m < kM; ++m) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w.q[m][j] = p[m * 8 * kGroups + j];
                asm volatile("" ::: "memory");  // (eight loads at a time)
            }
        }
        w.scale = a.scale_log2 * (F8 && a.k_scale ? a.k_scale[h] : 1.0f);
    }

    __device__ __forceinline__ void use_queries(Rows& w) const {
        // a negative scale turns the queries' signs, so that the largest score has the largest product
        const uint32_t flip = w.scale < 0.0f ? 0x80008000u : 0u;
        w.scale = fabsf(w.scale);
        if (w.scale < 2e-38f) w.scale = 2e-38f;  // (zero: every finite score alike, and a masked one still none)
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                uint4_t x = __builtin_bit_cast(uint4_t, w.q[m]) ^ flip;
                asm volatile("" : "+v"(x));
                w.q[m] = __builtin_bit_cast(vec8, x);
            }
    }

    // What this lane's rows see.
    template <bool kShared>
    __device__ __forceinline__ void start_rows(Rows& w, const Seq& sq, bool prefix, bool plain, int row0,
                                               int row_end) const {
        w.marked = false;
        w.all_lo = 0;
        w.all_hi = w.all_sink = 0x7fffffff;
        const int row = row0 + n;
        const bool on = row < row_end;
        const int tok = on ? token_of(a, row) : 0, t = sq.q0 + tok;
        w.lim = Limits{0, 0, 0};
        if (on) {
            if (!prefix) {
                w.lim = own_limits(a, sq, upto_of(sq, tok));
            } else if (plain) {
                w.lim.hi = a.prefix_len;
            } else {
                int s, stop = 0, upto = 0;
                if (a.n_seqs <= kSeqs) {
                    s = a.starts ? last_at(sh.start, a.n_seqs, t) : t;
                    if (s >= 0) {
                        stop = sh.end[s];
                        upto = sh.upto[s];
                    }
                } else {
                    s = seq_of(a, t);
                    if (s >= 0) {
                        const Seq mine = seq_at(a, s);
                        stop = mine.q0 + mine.n;
                        upto = upto_of(mine, -mine.q0);
                    }
                }
                if (s >= 0 && t < stop) w.lim = prefix_limits(a, upto + t);
            }
            w.all_lo = w.lim.lo > w.all_lo ? w.lim.lo : w.all_lo;
            w.all_hi = w.lim.hi < w.all_hi ? w.lim.hi : w.all_hi;
            w.all_sink = w.lim.sink < w.all_sink ? w.lim.sink : w.all_sink;
        }
        w.mx = -__builtin_inff();
        w.l = 0.0f;
#pragma unroll
        for (int t2 = 0; t2 < kT; ++t2) w.o[t2] = acc{};
        w.all_lo = lane_max(w.all_lo, 0);
        w.all_hi = lane_min(w.all_hi, 0x7fffffff);
        w.all_sink = lane_min(w.all_sink, 0x7fffffff);
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

    __device__ __forceinline__ void put_stats(float* part, const RowSplit& split, int part_row, float m, float l) const {
        part[(D << split.log2_rows) + part_row] = m;
        part[((D + 1) << split.log2_rows) + part_row] = l;
    }
};

// kWide: waves share their tiles in some unit of the launch.
template <int D, class E, bool F8, bool kWide>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void prefix_attention_kernel(AttnArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    Shared<D>& sh = *reinterpret_cast<Shared<D>*>(lds);
    uint64_t* const cost = reinterpret_cast<uint64_t*>(lds + sizeof(Shared<D>));
    uint32_t* const info = reinterpret_cast<uint32_t*>(cost + a.plan.own_entries + 1);
    Line line = build_line(a, cost, info, sh);
    const RowSplit &pre = a.plan.prefix, &own = a.plan.own;
    Job job;
    while (next_prefix(a, line, job, D)) {
        if (job.s0 >= job.s1) continue;
        if (kWide && pre.shared) Unit<D, E, F8, 32>(a, sh).template run<true>(job, pre, true, false, line.plain);
        else if (pre.narrow) Unit<D, E, F8, 16>(a, sh).template run<false>(job, pre, true, false, line.plain);
        else Unit<D, E, F8, 32>(a, sh).template run<false>(job, pre, true, false, line.plain);
    }
    while (next_own(a, line, cost, info, sh, job, D)) {
        if (job.s0 >= job.s1) continue;
        if (kWide && own.shared) Unit<D, E, F8, 32>(a, sh).template run<true>(job, own, false, false, false);
        else if (own.narrow) Unit<D, E, F8, 16>(a, sh).template run<false>(job, own, false, true, false);
        else Unit<D, E, F8, 32>(a, sh).template run<false>(job, own, false, true, false);
    }
}

// Dynamic LDS of a launch: the tiles and the line of entries.
template <int D>
constexpr size_t lds_bytes(int own_entries) {
    return sizeof(Shared<D>) + 8 * ((size_t)own_entries + 1) + 4 * (size_t)own_entries;
}

template <int D, class E, bool F8, bool kWide>
hipError_t launch_as(const AttnArgs& a, hipStream_t stream) {
    prefix_attention_kernel<D, E, F8, kWide><<<dim3(1u << a.plan.log2_workgroups), kThreads, lds_bytes<D>(a.plan.own_entries), stream>>>(a);
    return hipGetLastError();
}

template <int D, class E, bool F8>
hipError_t launch_rows(const AttnArgs& a, hipStream_t stream) {
    if (!a.plan.shared) return launch_as<D, E, F8, false>(a, stream);
    return launch_as<D, E, F8, true>(a, stream);
}

template <int D>
hipError_t launch_dim(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream) {
    if (bf16) return f8 ? launch_rows<D, Bf16, true>(a, stream) : launch_rows<D, Bf16, false>(a, stream);
    return f8 ? launch_rows<D, Half, true>(a, stream) : launch_rows<D, Half, false>(a, stream);
}

}  // namespace attn
}  // namespace qw35
