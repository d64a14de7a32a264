// Host-side launch interface of the attention operators (rope_kv.hip,
// block_cache.hip, prefix_attention.hip): internal to the library, the public C ABI is
// include/qw35_hip.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/qw35_hip.h"

namespace qw35 {

// [n_tokens][heads][dim] with unit column stride; strides in elements.
struct HeadsView {
    void* data;
    int64_t token_stride;
    int64_t head_stride;
    uint32_t dtype;  // QW35_HIP_DTYPE_*
    int vec;         // rows start 16-byte aligned: vector loads and stores
};

struct RopeArgs {
    const uint64_t* freq;      // nullptr: no rotation
    const int32_t* positions;  // [n_axes][n_tokens]
    const float* norm;         // [dim] or nullptr: no RMS norm
    float eps;
    int rot_dim;
    int n_axes;
    int interleaved;
    int sections[4];
};

hipError_t launch_rotate(const HeadsView& x, const HeadsView& y, int n_tokens, int heads, int dim, const RopeArgs& rope,
                         hipStream_t stream);
hipError_t launch_kv_append(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                            const int64_t* slots, const RopeArgs& rope, hipStream_t stream);

// Caches with a scale for each block of 32 tokens and head.
inline bool block_scaled(uint32_t dtype) { return dtype == QW35_HIP_DTYPE_E4M3_BLOCKS || dtype == QW35_HIP_DTYPE_I8_BLOCKS; }
// Tokens of a launch of their append: a block's first token looks through all of them.
constexpr int kAppendSlice = 16384;
hipError_t launch_kv_append_blocks(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                                   const int64_t* slots, const RopeArgs& rope, hipStream_t stream);
hipError_t launch_kv_read(const qw35_hip_kv_cache& cache, const HeadsView& k, const HeadsView& v, int n_tokens,
                          const int64_t* slots, hipStream_t stream);

// How a launch divides the rows (new token x head of a group) of a kind of unit.
//   Own units of up to 16 rows, and of up to 64 where there are more than
// few_own_units: a wave has 16 or 32 rows and goes through the tokens by itself.
//   Prefix units of up to 64 rows: a workgroup, 16 or 32 rows a wave, the waves
// of a row group on different 32-token tiles (a step is 4 or 2 tiles).
//   All others: a workgroup, 32 rows a wave, all four on the same tile.
int few_own_units(int64_t rows, int dim);  // sequences x kv heads

struct RowSplit {
    int log2_tiles;  // tiles of a step
    int log2_rg;     // row groups of the workgroup's waves
    int log2_rows;   // rows of a unit
    int narrow;      // 16 rows a wave
    int shared;      // the waves share their tiles
    int lead;        // cost of a unit beside its steps
    int log2_cost;   // cost of a step
    __host__ __device__ int step() const { return 1 << log2_tiles; }
};

struct AttnPlan {
    RowSplit prefix, own;
    int shared;  // of either
    int log2_workgroups;
    int lanes;           // up to 64 sequences whose costs fit 32 bits
    uint32_t group_magic, page_magic;  // 2^32 / group and page_blocks, rounded up (0: they are 1)
    int prefix_entries;  // row tiles of the prefix, of every kv head
    int own_entries;     // bound of the sequences' row tiles together
    uint64_t own_part;   // floats of the prefix' partial slots
    uint64_t meta_bytes;
    uint64_t workspace_bytes;
};

struct AttnArgs {
    HeadsView q, out, gate;
    const void* ck;
    const void* cv;
    const float* k_scale;
    const float* v_scale;
    int half_values;  // the cache is fp16
    uint32_t n_pages;
    uint32_t page_blocks;  // 32-token blocks of a page
    int kv_heads;
    int group;
    int n_tokens;
    int n_seqs;
    const int32_t* starts;
    const int32_t* lengths;
    const int32_t* pages;
    uint32_t pages_per_seq;
    const int32_t* prefix_pages;
    int prefix_len;
    float scale_log2;  // softmax scale times log2(e)
    int window;
    int sink;
    uint8_t* meta;
    float* part;      // partial slots: of the prefix
    float* own_part;  // and of own units
    AttnPlan plan;
    const float* k_blocks;  // scales of a block-scaled cache, [page][kv head][block]
    const float* v_blocks;
};

// A batch as the plan sees it; `own_tokens`: the most own tokens that a
// sequence's page table holds; `single`: every sequence has one new token.
struct AttnShape {
    int dim, kv_heads, group, n_seqs, n_tokens, max_new, page_blocks, prefix_len;
    int64_t own_tokens;
    bool single;
    int most_entries;  // the plan counts no more own entries than these
};
int most_own_entries(int dim, uint32_t cache_dtype);  // that a compute unit's LDS lists
AttnPlan plan_attention(const AttnShape& s);
hipError_t launch_prefix_attention(const AttnArgs& a, int dim, uint32_t q_dtype, uint32_t cache_dtype,
                                   hipStream_t stream);

// One translation unit per head dimension (attn_d<dim>.hip).
hipError_t launch_attn_d64(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream);
hipError_t launch_attn_d128(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream);
hipError_t launch_attn_d256(const AttnArgs& a, bool bf16, bool f8, hipStream_t stream);
// And of block-scaled caches (attn_blocks_d<dim>.hip).
hipError_t launch_attn_blocks_d64(const AttnArgs& a, bool bf16, bool i8, hipStream_t stream);
hipError_t launch_attn_blocks_d128(const AttnArgs& a, bool bf16, bool i8, hipStream_t stream);
hipError_t launch_attn_blocks_d256(const AttnArgs& a, bool bf16, bool i8, hipStream_t stream);

}  // namespace qw35
