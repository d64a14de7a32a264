// Shared-prefix attention: how a launch is divided, and the joining of the
// parts (prefix_attention.h has the mathematics and the main kernel).
#include "prefix_attention.h"

namespace qw35 {

namespace {

constexpr int kBatch = 16;  // parts whose loads are in flight together

// Over a wave's 64 lanes, in each of them.
template <class Op>
__device__ __forceinline__ float over_lanes(float v, Op op) {
    auto turn = [&](auto by) {  // of 16 lanes
        const int u = __builtin_bit_cast(int, v);
        v = op(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, 0x120 + decltype(by)::value, 0xf, 0xf, false)));
    };
    turn(std::integral_constant<int, 8>{});
    turn(std::integral_constant<int, 4>{});
    turn(std::integral_constant<int, 2>{});
    turn(std::integral_constant<int, 1>{});
    const attn::Pair p = attn::pair_xor16(v);
    v = op(p.a, p.b);
    const attn::Pair q = attn::pair_xor32(v);
    return op(q.a, q.b);
}

// Leads and costs in quarters of a microsecond, measured with all compute
// units at it: a step of a wave's own tiles waits for HBM (7 us for 128 KB of a
// compute unit's waves; 2.5 where few are at it, so 4 is taken), one of shared
// tiles for the matrix unit.  (Over 16 batches, steps at half and twice these
// costs, leads of 8 and 32 for own units of 16 rows and of 64 for shared tiles
// were no faster; 16 instead of 32 for own units of 32 rows cost four windowed
// sequences 13%, 32 instead of 16 for those of 16 rows 64 short ones 11%.)
RowSplit split_prefix(int64_t rows, int dim) {
    const int wait = dim == 64 ? 3 : 4;
    if (rows <= 16) return {2, 0, 4, 1, 0, 48, wait};
    if (rows <= 32) return {2, 0, 5, 0, 0, 48, wait};
    if (rows <= 64) return {1, 1, 6, 0, 0, 48, wait};
    return {0, 2, 7, 0, 1, 32, dim == 64 ? 2 : 3};
}

}  // namespace

// Own units of 17 to 64 rows: where there are few of them, a wave alone with its
// tile waits for itself, and four waves on one tile are faster though some have
// no row.  Of 128 units and fewer that holds at every length from 20 to 12000
// tokens, alike, ragged or with one long chunk among single tokens (256 columns x 4
// kv heads, 40 rows, 3000 tokens, us by a wave each and shared: 4 units 30, 20;
// 16 30, 27; 48 63, 41; 96 106, 69; 128 97, 94; 20 rows of 20 tokens 16, 16 at 128
// units), of 192 about evenly, of 256 only over long sequences (20 tokens 16, 25;
// 64 22, 31; 12000 571, 546; 128 columns, 512 units of 20 tokens 14, 20).  With 64
// columns a tile is too little for four waves of which two have rows: 17 to 32
// rows are shared up to 16 units (20 rows, 3000 tokens: 8 units 15, 13; 16 16, 15;
// 48 20, 21; 128 27, 31; 12000 tokens: 16 21, 21; 32 27, 30; 96 57, 69).  Lost by
// this: one of four sequences under a window of 4096, 5 to 36 rows: 30.5, 32.
int few_own_units(int64_t rows, int dim) { return dim == 64 && rows <= 32 ? 16 : 128; }

namespace {

RowSplit split_own(int64_t rows, int64_t units, int dim) {
    const int wait = dim == 64 ? 3 : 4;
    if (rows <= 16) return {0, 0, 4, 1, 0, 16, wait};
    if (rows <= 64 && units > few_own_units(rows, dim)) return {0, 0, 5, 0, 0, 32, wait};
    return {0, 2, 7, 0, 1, 32, dim == 64 ? 2 : 3};
}

// One row (token, head) for each `waves` waves of a workgroup of four: with
// few rows the four waves take every fourth part of one row and join in LDS.
// Bound by latency: the row's sequence, its list of parts, their maxima and
// sums are three reads that wait for each other (the first sixteen parts come
// with the third); a lane looks up one part of 64, and a part is a load and N
// products a lane.
template <int D>
__global__ __launch_bounds__(256) void prefix_attention_join(AttnArgs a, int waves) {
    constexpr int N = D / 64;  // columns of a lane
    typedef float vec_t __attribute__((ext_vector_type(N == 1 ? 2 : N)));
    __shared__ float sh_o[4][D];
    __shared__ float sh_m[4], sh_l[4];
    const int lane = threadIdx.x & 63, wave = attn::uniform((int)(threadIdx.x >> 6));
    const int heads = a.kv_heads * a.group;
    const bool waves_join = waves > 1;
    const int item = waves == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x;  // below 2^30
    const int t = (int)((uint32_t)item / (uint32_t)heads), head = item - t * heads;
    if (t >= a.n_tokens) return;
    const int h = attn::token_of(a, head), in_group = head - h * a.group;
    const attn::MetaHead meta = *reinterpret_cast<const attn::MetaHead*>(a.meta);
    const int* const first = reinterpret_cast<const int*>(a.meta + attn::meta_first_at());
    float gates[1][N];
    if (!waves_join || wave == 0) attn::load_gates(a, t, head, lane * N, 0, gates);  // (on their way meanwhile)
    const attn::Place at = attn::place_of(a, t, lane);
    attn::Pieces own = {0, 0}, pre = {0, 0};
    int own_row = 0, pre_row = 0;
    if (at.s >= 0) {
        const attn::Pieces* const pieces =
            reinterpret_cast<const attn::Pieces*>(a.meta + attn::meta_pieces_at(a.n_seqs)) +
            (int64_t)h * (a.plan.prefix_entries + meta.own_entries);
        own_row = (t - at.q0) * a.group + in_group;
        const int e = (meta.lanes ? at.s : first[at.s]) + (own_row >> a.plan.own.log2_rows);
        own_row &= (1 << a.plan.own.log2_rows) - 1;
        if (e < meta.own_entries) own = pieces[a.plan.prefix_entries + e];
        if (a.plan.prefix_entries) {
            pre_row = t * a.group + in_group;
            pre = pieces[pre_row >> a.plan.prefix.log2_rows];
            pre_row &= (1 << a.plan.prefix.log2_rows) - 1;
        }
    }
    if (!a.plan.prefix_entries && own.n == 1) return;  // the main kernel finished this row (all waves of it return)
    const int n = attn::uniform((int)(own.n + pre.n)), own_n = (int)own.n;
    const int k0 = waves == 1 ? 0 : wave;
    float top = -__builtin_inff(), sum = 0.0f;
    float acc[N] = {};
    // 64 parts at a time: lane i reads the maximum and sum of part i, then every lane its columns of all of them
    for (int k = k0; k < n; k += 64 * waves) {
        const int mine = k + lane * waves;
        const float* row_at = a.part;
        float pm = -__builtin_inff(), pl = 0.0f;
        if (mine < n) {
            const bool is_own = mine < own_n;
            const int log2_rows = is_own ? a.plan.own.log2_rows : a.plan.prefix.log2_rows;
            const int row = is_own ? own_row : pre_row;
            const uint64_t slot = is_own ? own.slot0 + mine : pre.slot0 + (mine - own_n) * meta.prefix_stride;
            const float* const p = (is_own ? a.own_part : a.part) + slot * attn::slot_floats(1 << log2_rows, D);
            row_at = p + row * D;
            pm = p[(D << log2_rows) + row];
            pl = p[((D + 1) << log2_rows) + row];
        }
        const int rest = (n - k + waves - 1) / waves, count = rest < 64 ? rest : 64;
        const int64_t addr = reinterpret_cast<int64_t>(row_at);
        // (a part past the last: the last once more, of weight zero)
        auto load = [&](int i, vec_t (&v)[kBatch]) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int part = i + j < count ? i + j : count - 1;
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)addr, part);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(addr >> 32), part);
                const float* const from = reinterpret_cast<const float*>((uint64_t)hi << 32 | lo) + lane * N;
                if constexpr (N == 1) v[j][0] = *from;
                else v[j] = *reinterpret_cast<const vec_t*>(from);
            }
        };
        vec_t v[kBatch];
        load(0, v);  // (on their way while the weights are made)
        const float now = fmaxf(top, over_lanes(pm, [](float x, float y) { return fmaxf(x, y); }));
        const float shrink = attn::part_weight(top, now);
        top = now;
        sum *= shrink;
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= shrink;
        const float weight = attn::part_weight(pm, now);
        sum += weight * pl;
        for (int i = 0; i < count; i += kBatch) {
            if (i) load(i, v);
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), i + j));
#pragma unroll
                for (int c = 0; c < N; ++c) acc[c] += w == 0.0f ? 0.0f : w * v[j][c];
            }
        }
    }
    // each lane holds its parts' share, rescaled alike
    sum = over_lanes(sum, [](float x, float y) { return x + y; });
    if (waves_join) {
#pragma unroll
        for (int c = 0; c < N; ++c) sh_o[wave][lane * N + c] = acc[c];
        if (lane == 0) {
            sh_m[wave] = top;
            sh_l[wave] = sum;
        }
        __syncthreads();
        if (wave) return;
        const float all = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
        sum = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) acc[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float weight = attn::part_weight(sh_m[w], all);
            sum += weight * sh_l[w];
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c] += weight * sh_o[w][lane * N + c];
        }
    }
    const float inv = sum == 0.0f ? 0.0f : (a.v_scale ? a.v_scale[h] : 1.0f) / sum;
    float out[1][N];
#pragma unroll
    for (int c = 0; c < N; ++c) out[0][c] = acc[c] * inv;
    bool lost = false;
#pragma unroll
    for (int c = 0; c < N; ++c) lost |= out[0][c] != out[0][c];
    if (__builtin_expect(lost && sum == sum, 0)) {
        const AttnArgs& b = attn::args_again();
        if (b.half_values) {
            const attn::Seq q = attn::seq_at(b, at.s);
            const int upto = attn::upto_of(q, t - q.q0);
            attn::Infinities found = {0, 0};
            const auto column = [&](int k) { return lane * N + k; };
            if (b.plan.prefix_entries)
                attn::find_infinities<D, N>(b, b.prefix_pages, h, attn::prefix_limits(b, upto), column, found);
            attn::find_infinities<D, N>(b, b.pages + (int64_t)at.s * b.pages_per_seq, h, attn::own_limits(b, q, upto),
                                        column, found);
#pragma unroll
            for (int c = 0; c < N; ++c)
                if (out[0][c] != out[0][c]) out[0][c] = found.of(c, out[0][c]);
        }
    }
    attn::finish(a, t, head, lane * N, 0, gates, out);
}

template <int D>
hipError_t launch_join(const AttnArgs& a, hipStream_t stream) {
    const int64_t rows = (int64_t)a.n_tokens * a.kv_heads * a.group;
    const int waves = rows <= 1024 ? 4 : 1;
    const int64_t grid = waves == 4 ? rows : (rows + 3) / 4;
    prefix_attention_join<D><<<dim3((unsigned)grid), 256, 0, stream>>>(a, waves);
    return hipGetLastError();
}

}  // namespace

int most_own_entries(int dim) {
    constexpr size_t kLds = 160 * 1024, kEntry = 12;
    static_assert(attn::lds_bytes<64>(1) - attn::lds_bytes<64>(0) == kEntry);
    const size_t rest = kLds - (dim == 64    ? attn::lds_bytes<64>(0)
                                : dim == 128 ? attn::lds_bytes<128>(0)
                                             : attn::lds_bytes<256>(0));
    return (int)(rest / kEntry);
}

AttnPlan plan_attention(const AttnShape& s) {
    AttnPlan p = {};
    const int64_t rows_prefix = s.prefix_len ? (int64_t)s.n_tokens * s.group : 0, rows_own = (int64_t)s.max_new * s.group;
    p.prefix = split_prefix(rows_prefix, s.dim);
    p.own = split_own(rows_own, (int64_t)s.n_seqs * s.kv_heads, s.dim);
    p.shared = p.prefix.shared || p.own.shared;
    p.log2_workgroups = s.dim == 256 ? 8 : 9;
    p.group_magic = s.group > 1 ? (uint32_t)((1ull << 32) / s.group + 1) : 0;
    p.page_magic = s.page_blocks > 1 ? (uint32_t)((1ull << 32) / s.page_blocks + 1) : 0;
    p.prefix_entries = (int)((rows_prefix + (1 << p.prefix.log2_rows) - 1) >> p.prefix.log2_rows);
    if (s.single) p.own_entries = s.n_seqs * ((s.group + (1 << p.own.log2_rows) - 1) >> p.own.log2_rows);
    // every sequence's last row tile may be a part of one
    else p.own_entries = s.n_seqs + (int)((int64_t)s.n_tokens * s.group >> p.own.log2_rows);
    if (p.own_entries > s.most_entries) p.own_entries = s.most_entries;
    auto cost = [](const RowSplit& r, int64_t tokens) {
        return r.lead + (((tokens + 31) / 32 + r.step()) / r.step() << r.log2_cost);
    };
    p.lanes = s.n_seqs <= 64 && s.kv_heads * p.prefix_entries * cost(p.prefix, s.prefix_len) < 1 << 30 &&
              s.kv_heads * s.n_seqs * cost(p.own, s.own_tokens) < 1 << 30;
    const uint64_t prefix_slots = p.prefix_entries ? (1ull << p.log2_workgroups) + (uint64_t)s.kv_heads * p.prefix_entries : 0;
    const uint64_t own_slots = (p.own.shared ? 1ull : 4ull) << p.log2_workgroups;
    p.own_part = prefix_slots * attn::slot_floats(1 << p.prefix.log2_rows, s.dim);
    p.meta_bytes = (attn::meta_pieces_at(s.n_seqs) + 8 * (uint64_t)s.kv_heads * (p.prefix_entries + p.own_entries) + 255) /
                   256 * 256;
    p.workspace_bytes = p.meta_bytes + 4 * (p.own_part + (own_slots + (uint64_t)s.kv_heads * p.own_entries) *
                                                             attn::slot_floats(1 << p.own.log2_rows, s.dim));
    return p;
}

hipError_t launch_prefix_attention(const AttnArgs& a, int dim, uint32_t q_dtype, uint32_t cache_dtype,
                                   hipStream_t stream) {
    const bool bf16 = q_dtype == QW35_HIP_DTYPE_BF16, f8 = cache_dtype == QW35_HIP_DTYPE_E4M3;
    hipError_t e = dim == 64    ? launch_attn_d64(a, bf16, f8, stream)
                   : dim == 128 ? launch_attn_d128(a, bf16, f8, stream)
                                : launch_attn_d256(a, bf16, f8, stream);
    if (e != hipSuccess) return e;
    return dim == 64    ? launch_join<64>(a, stream)
           : dim == 128 ? launch_join<128>(a, stream)
                        : launch_join<256>(a, stream);
}

}  // namespace qw35
