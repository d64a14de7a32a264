// extern "C" entry points of the attention operators: argument checks and launch.
#include <limits.h>
#include <math.h>

#include "abi_error.h"
#include "attention.h"
#include "qw35_kernels.h"

namespace {

using qw35::check_hip;
using qw35::HeadsView;
using qw35::RopeArgs;
using qw35::set_err;

constexpr uint32_t kMaxTokens = 1u << 22;   // rows of a call and their heads stay within 32 bits
constexpr uint32_t kMaxHeads = 256;
constexpr uint64_t kMaxLength = 1u << 30;   // positions

size_t dtype_size(uint32_t t) { return t == QW35_HIP_DTYPE_F32 ? 4 : t == QW35_HIP_DTYPE_E4M3 ? 1 : 2; }

bool check_heads(const qw35_hip_heads* v, const char* what, const char* name, HeadsView* out, char* err,
                 uintptr_t err_len) {
    if (!v || !v->data) {
        set_err(err, err_len, "%s: null %s", what, name);
        return false;
    }
    if (v->dtype != QW35_HIP_DTYPE_F32 && v->dtype != QW35_HIP_DTYPE_BF16 && v->dtype != QW35_HIP_DTYPE_F16) {
        set_err(err, err_len, "%s: %s must be f32, bf16 or f16, got dtype %u", what, name, v->dtype);
        return false;
    }
    const uint64_t size = dtype_size(v->dtype);
    if ((uintptr_t)v->data % size) {
        set_err(err, err_len, "%s: %s must be aligned to its elements", what, name);
        return false;
    }
    *out = HeadsView{v->data, v->token_stride, v->head_stride, v->dtype, 0};
    // strides as unsigned: the alignment of a negative one is the same
    out->vec = (((uintptr_t)v->data | (uint64_t)v->token_stride * size | (uint64_t)v->head_stride * size) & 15u) == 0;
    return true;
}

// The axes whose sections matter: up to the last that is not zero.
uint32_t section_axes(const qw35_hip_rope& r) {
    uint32_t n = 0;
    for (uint32_t a = 0; a < 4; ++a)
        if (r.sections[a]) n = a + 1;
    return n ? n : 1;
}

bool check_rope(const qw35_hip_rope* r, const int32_t* positions, uint32_t n_axes, const float* norm, float eps,
                uint32_t dim, const char* what, RopeArgs* out, char* err, uintptr_t err_len) {
    *out = RopeArgs{};
    if (((uintptr_t)norm & 3u) != 0) {
        set_err(err, err_len, "%s: norm must be 4-byte aligned", what);
        return false;
    }
    if (norm && !(eps >= 0.0f && eps < INFINITY)) {
        set_err(err, err_len, "%s: eps must be a finite number >= 0", what);
        return false;
    }
    out->norm = norm;
    out->eps = eps;
    if (!r) return true;
    if (!r->freq || ((uintptr_t)r->freq & 7u)) {
        set_err(err, err_len, "%s: rope frequencies must be an 8-byte aligned device array", what);
        return false;
    }
    if (r->rot_dim == 0 || r->rot_dim % 16 || r->rot_dim > dim) {
        set_err(err, err_len, "%s: rot_dim=%u must be a multiple of 16 up to dim=%u", what, r->rot_dim, dim);
        return false;
    }
    uint64_t sum = 0;
    for (uint32_t s : r->sections) sum += s;
    if (sum && sum != r->rot_dim / 2) {
        set_err(err, err_len, "%s: sections must be all zero or add up to rot_dim / 2 = %u", what, r->rot_dim / 2);
        return false;
    }
    if (r->interleaved && sum) {
        const uint32_t half = r->rot_dim / 2;
        for (uint32_t a = 1; a < 3; ++a)
            if (r->sections[a] && 3 * (r->sections[a] - 1) + a >= half) {
                set_err(err, err_len, "%s: section %u of %u pairs does not fit %u interleaved pairs", what, a,
                        r->sections[a], half);
                return false;
            }
        if (r->sections[3]) {
            set_err(err, err_len, "%s: interleaved sections have three axes", what);
            return false;
        }
    }
    if (n_axes != 1 && n_axes != section_axes(*r)) {
        set_err(err, err_len, "%s: positions have %u axes, the sections 1 or %u", what, n_axes, section_axes(*r));
        return false;
    }
    if (!positions || ((uintptr_t)positions & 3u)) {
        set_err(err, err_len, "%s: positions must be a 4-byte aligned device array", what);
        return false;
    }
    out->freq = r->freq;
    out->positions = positions;
    out->rot_dim = (int)r->rot_dim;
    out->n_axes = (int)n_axes;
    out->interleaved = r->interleaved != 0;
    for (int a = 0; a < 4; ++a) out->sections[a] = (int)r->sections[a];
    return true;
}

bool check_cache(const qw35_hip_kv_cache* c, const char* what, char* err, uintptr_t err_len) {
    if (!c || !c->k || !c->v) {
        set_err(err, err_len, "%s: null cache", what);
        return false;
    }
    if (((uintptr_t)c->k & 15u) || ((uintptr_t)c->v & 15u) || ((uintptr_t)c->k_scale & 3u) ||
        ((uintptr_t)c->v_scale & 3u)) {
        set_err(err, err_len, "%s: cache pages must be 16-byte aligned, their scales 4-byte", what);
        return false;
    }
    if (c->dtype != QW35_HIP_DTYPE_F16 && c->dtype != QW35_HIP_DTYPE_BF16 && c->dtype != QW35_HIP_DTYPE_E4M3) {
        set_err(err, err_len, "%s: a cache is f16, bf16 or e4m3, got dtype %u", what, c->dtype);
        return false;
    }
    if (c->dtype != QW35_HIP_DTYPE_E4M3 && (c->k_scale || c->v_scale)) {
        set_err(err, err_len, "%s: only an e4m3 cache has scales", what);
        return false;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_err(err, err_len, "%s: head_dim=%u must be 64, 128 or 256", what, c->head_dim);
        return false;
    }
    if (c->page_size == 0 || c->page_size % 32 || c->page_size > (1u << 20)) {
        set_err(err, err_len, "%s: page_size=%u must be a positive multiple of 32 up to 2^20", what, c->page_size);
        return false;
    }
    if (c->kv_heads == 0 || c->kv_heads > kMaxHeads || c->n_pages == 0 || c->n_pages > 0x7fffffffu) {
        set_err(err, err_len, "%s: kv_heads=%u must be 1..%u, n_pages=%u positive", what, c->kv_heads, kMaxHeads,
                c->n_pages);
        return false;
    }
    // (a tile of 32 tokens of a head is addressed by one 32-bit number)
    if ((uint64_t)c->n_pages * c->kv_heads * (c->page_size / 32) >= 0xffffffffull) {
        set_err(err, err_len, "%s: the cache has over 2^32 - 2 blocks of 32 tokens", what);
        return false;
    }
    return true;
}

}  // namespace

extern "C" {

int qw35_hip_rope_freq(uint32_t rot_dim, double base, uint64_t* freq, char* err, uintptr_t err_len) {
    if (!freq || rot_dim == 0 || rot_dim % 16 || rot_dim > 512) {
        set_err(err, err_len, "rope_freq: rot_dim=%u must be a multiple of 16 up to 512, with an array for it",
                rot_dim);
        return 0;
    }
    if (!(base > 1.0) || !(base < INFINITY)) {
        set_err(err, err_len, "rope_freq: base must be a finite number > 1");
        return 0;
    }
    // turns per position, below 1 / (2 pi): the long double product has 64 bits of it
    const long double turn = 6.283185307179586476925286766559L;
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        const long double f = powl((long double)base, -2.0L * i / rot_dim) / turn;
        freq[i] = (uint64_t)ldexpl(f, 64);
    }
    return 1;
}

int qw35_hip_rotate(const qw35_hip_heads* x, const qw35_hip_heads* y, uint32_t n_tokens, uint32_t heads, uint32_t dim,
                    const qw35_hip_rope* rope, const int32_t* positions, uint32_t n_axes, const float* norm, float eps,
                    void* stream, char* err, uintptr_t err_len) {
    if (dim == 0 || dim % 8 || dim > 512) {
        set_err(err, err_len, "rotate: dim=%u must be a multiple of 8 up to 512", dim);
        return 0;
    }
    if (heads == 0 || heads > kMaxHeads || n_tokens > kMaxTokens) {
        set_err(err, err_len, "rotate: heads=%u must be 1..%u, n_tokens=%u at most %u", heads, kMaxHeads, n_tokens,
                kMaxTokens);
        return 0;
    }
    HeadsView vx, vy;
    RopeArgs r;
    if (n_tokens == 0) return 1;
    if (!check_heads(x, "rotate", "x", &vx, err, err_len) || !check_heads(y, "rotate", "y", &vy, err, err_len) ||
        !check_rope(rope, positions, n_axes, norm, eps, dim, "rotate", &r, err, err_len))
        return 0;
    return check_hip(qw35::launch_rotate(vx, vy, (int)n_tokens, (int)heads, (int)dim, r,
                                         static_cast<hipStream_t>(stream)),
                     "rotate", err, err_len);
}

int qw35_hip_kv_append(const qw35_hip_kv_cache* cache, const qw35_hip_heads* k, const qw35_hip_heads* v,
                       uint32_t n_tokens, const int64_t* slots, const qw35_hip_rope* rope, const int32_t* positions,
                       uint32_t n_axes, const float* norm, float eps, void* stream, char* err, uintptr_t err_len) {
    HeadsView vk, vv;
    RopeArgs r;
    if (!check_cache(cache, "kv_append", err, err_len)) return 0;
    if (n_tokens > kMaxTokens) {
        set_err(err, err_len, "kv_append: n_tokens=%u is over %u", n_tokens, kMaxTokens);
        return 0;
    }
    if (n_tokens == 0) return 1;
    if (!check_heads(k, "kv_append", "k", &vk, err, err_len) || !check_heads(v, "kv_append", "v", &vv, err, err_len) ||
        !check_rope(rope, positions, n_axes, norm, eps, cache->head_dim, "kv_append", &r, err, err_len))
        return 0;
    if (vk.dtype != vv.dtype) {
        set_err(err, err_len, "kv_append: k and v must have one type, got dtypes %u and %u", vk.dtype, vv.dtype);
        return 0;
    }
    if (!slots || ((uintptr_t)slots & 7u)) {
        set_err(err, err_len, "kv_append: slots must be an 8-byte aligned device array");
        return 0;
    }
    return check_hip(qw35::launch_kv_append(*cache, vk, vv, (int)n_tokens, slots, r,
                                            static_cast<hipStream_t>(stream)),
                     "kv_append", err, err_len);
}

static bool check_batch(const qw35_hip_kv_cache* cache, uint32_t n_heads, uint32_t n_seqs, uint32_t n_tokens,
                        char* err, uintptr_t err_len) {
    if (!check_cache(cache, "prefix_attention", err, err_len)) return false;
    if (n_heads == 0 || n_heads > kMaxHeads || n_heads % cache->kv_heads) {
        set_err(err, err_len, "prefix_attention: n_heads=%u must be a multiple of kv_heads=%u up to %u", n_heads,
                cache->kv_heads, kMaxHeads);
        return false;
    }
    if (n_tokens > kMaxTokens || n_seqs > 0xffffu) {
        set_err(err, err_len, "prefix_attention: n_tokens=%u is over %u or n_seqs=%u over 65535", n_tokens, kMaxTokens,
                n_seqs);
        return false;
    }
    return true;
}

static qw35::AttnPlan plan_of(const qw35_hip_kv_cache* c, uint32_t n_heads, uint32_t n_seqs, uint32_t n_tokens,
                              uint32_t max_new, uint32_t prefix_len, uint32_t pages_per_seq, bool single,
                              int most_entries) {
    return qw35::plan_attention({(int)c->head_dim, (int)c->kv_heads, (int)(n_heads / c->kv_heads), (int)n_seqs,
                                 (int)n_tokens, (int)max_new, (int)(c->page_size / 32), (int)prefix_len,
                                 (int64_t)pages_per_seq * c->page_size, single, most_entries});
}

static uint32_t few_own_seqs(const qw35_hip_kv_cache* c, uint64_t rows) {
    return (uint32_t)qw35::few_own_units((int64_t)rows, (int)c->head_dim) / c->kv_heads;
}

uint64_t qw35_hip_prefix_attention_workspace_size(const qw35_hip_kv_cache* cache, uint32_t n_heads, uint32_t n_seqs,
                                                  uint32_t n_tokens) {
    if (!check_batch(cache, n_heads, n_seqs, n_tokens, nullptr, 0)) return 0;
    const uint32_t group = n_heads / cache->kv_heads;
    // every division of the rows that a call of this batch may take: the most rows of a sequence that each has
    const uint32_t most[] = {1, 16 / group, 32 / group, 64 / group, 64 / group + 1, n_tokens};
    // A division whose row tiles the list does not hold is refused for this
    // batch, but smaller ones may take it: its size then is that of a full list.
    const int room = qw35::most_own_entries((int)cache->head_dim);
    uint64_t need = 256;
    bool served = n_tokens == 0;
    if (n_seqs == n_tokens)
        served |= plan_of(cache, n_heads, n_seqs, n_tokens, 1, 0, 1u << 15, true, INT_MAX).own_entries <= room;
    for (uint32_t prefix = 0; prefix < 2; ++prefix)
        for (uint32_t max_new : most)
            // and the most sequences that are few, whose units have more rows
            for (uint32_t seqs : {n_seqs, few_own_seqs(cache, (uint64_t)max_new * group)}) {
                if (max_new == 0 || max_new > n_tokens || seqs > n_seqs) continue;
                const qw35::AttnPlan p = plan_of(cache, n_heads, seqs, n_tokens, max_new, prefix, 1u << 15, false, room);
                if (p.workspace_bytes > need) need = p.workspace_bytes;
                if (seqs == n_seqs)
                    served |= plan_of(cache, n_heads, seqs, n_tokens, max_new, prefix, 1u << 15, false, INT_MAX)
                                  .own_entries <= room;
            }
    return served ? need : 0;
}

int qw35_hip_prefix_attention(const qw35_hip_attention* op, const qw35_hip_kv_cache* cache, void* stream, char* err,
                              uintptr_t err_len) {
    const char* what = "prefix_attention";
    if (!op) {
        set_err(err, err_len, "%s: null op", what);
        return 0;
    }
    if (!check_batch(cache, op->n_heads, op->n_seqs, op->n_tokens, err, err_len)) return 0;
    if (op->n_tokens == 0) return 1;
    qw35::AttnArgs a = {};
    if (!check_heads(&op->q, what, "q", &a.q, err, err_len) || !check_heads(&op->out, what, "out", &a.out, err, err_len))
        return 0;
    if (op->gate.data && !check_heads(&op->gate, what, "gate", &a.gate, err, err_len)) return 0;
    if (a.q.dtype == QW35_HIP_DTYPE_F32 || (cache->dtype != QW35_HIP_DTYPE_E4M3 && a.q.dtype != cache->dtype)) {
        set_err(err, err_len, "%s: q must have the cache's type (f16 or bf16 for an e4m3 cache), got dtype %u", what,
                a.q.dtype);
        return 0;
    }
    if (!op->starts && op->n_seqs != op->n_tokens) {
        set_err(err, err_len, "%s: without starts n_seqs=%u must be n_tokens=%u", what, op->n_seqs, op->n_tokens);
        return 0;
    }
    if (op->n_seqs && (!op->lengths || (op->pages_per_seq && !op->pages))) {
        set_err(err, err_len, "%s: null lengths or pages", what);
        return 0;
    }
    if (((uintptr_t)op->starts | (uintptr_t)op->lengths | (uintptr_t)op->pages | (uintptr_t)op->prefix_pages) & 3u) {
        set_err(err, err_len, "%s: starts, lengths and pages must be 4-byte aligned", what);
        return 0;
    }
    if ((uint64_t)op->pages_per_seq * cache->page_size > kMaxLength || op->prefix_len > kMaxLength) {
        set_err(err, err_len, "%s: at most 2^30 positions, got %llu own and %u shared", what,
                (unsigned long long)op->pages_per_seq * cache->page_size, op->prefix_len);
        return 0;
    }
    if (op->prefix_len && (!op->prefix_pages || (uint64_t)op->n_prefix_pages * cache->page_size < op->prefix_len)) {
        set_err(err, err_len, "%s: %u shared pages of %u do not hold prefix_len=%u", what,
                op->prefix_pages ? op->n_prefix_pages : 0, cache->page_size, op->prefix_len);
        return 0;
    }
    if (!(op->scale > -INFINITY && op->scale < INFINITY)) {
        set_err(err, err_len, "%s: scale must be finite", what);
        return 0;
    }
    if (op->window > kMaxLength || op->sink > kMaxLength) {
        set_err(err, err_len, "%s: window=%u and sink=%u are at most 2^30", what, op->window, op->sink);
        return 0;
    }
    // (without starts every sequence has one new token, whatever max_new says)
    const uint32_t max_new = !op->starts                                          ? 1
                             : op->max_new == 0 || op->max_new > op->n_tokens ? op->n_tokens
                                                                              : op->max_new;
    a.plan = plan_of(cache, op->n_heads, op->n_seqs, op->n_tokens, max_new, op->prefix_len, op->pages_per_seq,
                     !op->starts, INT_MAX);
    const int room = qw35::most_own_entries((int)cache->head_dim);
    if (a.plan.own_entries > room) {
        set_err(err, err_len, "%s: %d row tiles in a call are %d over the list's room; give it fewer tokens or sequences",
                what, a.plan.own_entries, a.plan.own_entries - room);
        return 0;
    }
    if (!op->workspace || ((uintptr_t)op->workspace & 255u) || op->workspace_bytes < a.plan.workspace_bytes) {
        set_err(err, err_len, "%s: needs a 256-byte aligned workspace of %llu bytes, got %llu", what,
                (unsigned long long)a.plan.workspace_bytes,
                (unsigned long long)(op->workspace ? op->workspace_bytes : 0));
        return 0;
    }
    a.ck = cache->k;
    a.cv = cache->v;
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.half_values = cache->dtype == QW35_HIP_DTYPE_F16;
    a.n_pages = cache->n_pages;
    a.page_blocks = cache->page_size / 32;
    a.kv_heads = (int)cache->kv_heads;
    a.group = (int)(op->n_heads / cache->kv_heads);
    a.n_tokens = (int)op->n_tokens;
    a.n_seqs = (int)op->n_seqs;
    a.starts = op->starts;
    a.lengths = op->lengths;
    a.pages = op->pages;
    a.pages_per_seq = op->pages_per_seq;
    a.prefix_pages = op->prefix_pages;
    a.prefix_len = (int)op->prefix_len;
    a.scale_log2 = op->scale * 1.4426950408889634f;
    a.window = (int)op->window;
    a.sink = (int)op->sink;
    a.meta = static_cast<uint8_t*>(op->workspace);
    a.part = reinterpret_cast<float*>(a.meta + a.plan.meta_bytes);
    a.own_part = a.part + a.plan.own_part;
    return check_hip(qw35::launch_prefix_attention(a, (int)cache->head_dim, op->q.dtype, cache->dtype,
                                                   static_cast<hipStream_t>(stream)),
                     what, err, err_len);
}

}  // extern "C"
