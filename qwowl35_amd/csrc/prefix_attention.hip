// Shared-prefix attention: how a launch is divided, and the joining of the
// parts (prefix_attention.h has the mathematics and the main kernel).
#include "prefix_attention.h"

namespace qw35 {

using attn::MetaHead;

namespace {

RowSplit split_rows(int64_t rows, int shared_r) {
    if (rows <= 32) return {0, 32, 3, 0};
    if (rows <= 64) return {1, 64, 2, 0};
    return {2, 128 * shared_r, shared_r, 1};
}

// A unit's pieces: workgroups w0.., slots slot0...
struct Pieces {
    int64_t slot0;
    int n;
    int row;  // row of the slots
};

__device__ __forceinline__ Pieces pieces_of(const MetaHead& m, const uint64_t* cost, int h, int e, int row,
                                            const RowSplit& split) {
    Pieces p = {0, 0, row % split.rows};
    if (e >= m.entries) return p;
    const uint64_t e0 = cost[e], e1 = cost[e + 1];
    if (e0 == e1) return p;
    const uint64_t head0 = h * m.head_cost;
    const uint64_t w0 = (head0 + e0) / m.per, w1 = (head0 + e1 - split.cost) / m.per;
    p.slot0 = (int64_t)(w0 + (uint64_t)h * m.entries + e);
    p.n = (int)(w1 - w0) + 1;
    return p;
}

// One row (token, head) for each `waves` waves of a workgroup of four: with
// few rows the four waves take every fourth part of one row and join in LDS.
// Bound by latency there (two dependent reads and the parts), by the parts'
// bytes otherwise.
template <int D>
__global__ __launch_bounds__(256) void prefix_attention_join(AttnArgs a, int waves) {
    constexpr int N = D / 64;  // columns of a lane
    typedef float vec_t __attribute__((ext_vector_type(N == 1 ? 2 : N)));
    __shared__ float sh_o[4][D];
    __shared__ float sh_m[4], sh_l[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int heads = a.kv_heads * a.group;
    const int64_t item = waves == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (waves == 1 && item >= (int64_t)a.n_tokens * heads) return;
    const int t = (int)(item / heads), head = (int)(item % heads);
    const int h = head / a.group;
    const MetaHead m = *reinterpret_cast<const MetaHead*>(a.meta);
    const int* const first = reinterpret_cast<const int*>(a.meta + attn::meta_first_at());
    const uint64_t* const cost = reinterpret_cast<const uint64_t*>(a.meta + attn::meta_cost_at(a.n_seqs));
    const int s = attn::seq_of_wave(a, t, lane);
    Pieces own = {0, 0, 0}, pre = {0, 0, 0};
    bool on = false;
    if (s >= 0) {
        const attn::Seq q = attn::seq_at(a, s);
        on = t >= q.q0 && t < q.q0 + q.n;
        if (on) {
            const int row = (t - q.q0) * a.group + head % a.group;
            own = pieces_of(m, cost, h, first[s] + row / a.plan.own.rows, row, a.plan.own);
        }
    }
    if (a.plan.prefix_entries) {
        const int row = t * a.group + head % a.group;
        if (on) pre = pieces_of(m, cost, h, row / a.plan.prefix.rows, row, a.plan.prefix);
    } else if (own.n == 1) {
        return;  // the main kernel finished this row (all waves of it return)
    }
    const uint64_t slot_floats = attn::slot_floats(a.plan.slot_rows, D);
    const int n = own.n + pre.n;
    const int k0 = waves == 1 ? 0 : wave;
    const float* const part = a.part;
    auto slot_of = [&](int k) {
        return part + (uint64_t)(k < own.n ? own.slot0 + k : pre.slot0 + (k - own.n)) * slot_floats;
    };
    float top = -__builtin_inff(), sum = 0.0f;
    float acc[N] = {};
    // 64 parts at a time: lane i reads the maximum and sum of part i, then every lane its columns of all of them
    for (int k = k0; k < n; k += 64 * waves) {
        const int mine = k + lane * waves;
        float pm = -__builtin_inff(), pl = 0.0f;
        if (mine < n) {
            const float* const p = slot_of(mine);
            const int row = mine < own.n ? own.row : pre.row;
            pm = p[(int64_t)a.plan.slot_rows * D + row];
            pl = p[(int64_t)a.plan.slot_rows * (D + 1) + row];
        }
        float chunk = pm;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) chunk = fmaxf(chunk, __shfl_xor(chunk, o));
        const float now = fmaxf(top, chunk);
        const float shrink = attn::part_weight(top, now);
        top = now;
        sum *= shrink;
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= shrink;
        const float weight = attn::part_weight(pm, now);
        sum += weight * pl;
        const int count = (n - k + waves - 1) / waves < 64 ? (n - k + waves - 1) / waves : 64;
#pragma unroll 8
        for (int i = 0; i < count; ++i) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), i));
            const int j = k + i * waves;
            const float* const p = slot_of(j) + (int64_t)(j < own.n ? own.row : pre.row) * D + lane * N;
            if constexpr (N == 1) {
                acc[0] += w == 0.0f ? 0.0f : w * p[0];
            } else {
                const vec_t v = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
                for (int c = 0; c < N; ++c) acc[c] += w == 0.0f ? 0.0f : w * v[c];
            }
        }
    }
    // sum: each lane holds its parts' share, rescaled alike
#pragma unroll
    for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
    if (waves > 1) {
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
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] *= inv;
    attn::finish<N>(a, t, head, lane * N, acc);
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

AttnPlan plan_attention(int dim, int kv_heads, int group, int n_seqs, int n_tokens, int max_new, bool prefix) {
    AttnPlan p = {};
    const int64_t rows_prefix = prefix ? (int64_t)n_tokens * group : 0, rows_own = (int64_t)max_new * group;
    const int64_t most = rows_prefix > rows_own ? rows_prefix : rows_own;
    p.shared_r = most <= 64 ? 0 : most <= 128 || dim == 256 ? 1 : 2;
    p.prefix = split_rows(rows_prefix, p.shared_r);
    p.own = split_rows(rows_own, p.shared_r);
    p.workgroups = dim == 256 || p.shared_r == 2 ? 256 : 512;
    p.prefix_entries = (int)((rows_prefix + p.prefix.rows - 1) / p.prefix.rows);
    // every sequence's last row tile may be a part of one
    p.max_entries = p.prefix_entries + n_seqs + (int)((int64_t)n_tokens * group / p.own.rows);
    p.slot_rows = p.prefix.rows > p.own.rows && prefix ? p.prefix.rows : p.own.rows;
    p.slots = (uint64_t)p.workgroups + (uint64_t)kv_heads * p.max_entries;
    p.meta_bytes = (attn::meta_cost_at(n_seqs) + 8 * ((uint64_t)p.max_entries + 1) + 255) / 256 * 256;
    p.lds_bytes = dim == 64    ? attn::lds_bytes<64>(p.max_entries)
                  : dim == 128 ? attn::lds_bytes<128>(p.max_entries)
                               : attn::lds_bytes<256>(p.max_entries);
    p.workspace_bytes = p.meta_bytes + 4 * p.slots * attn::slot_floats(p.slot_rows, dim);
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
