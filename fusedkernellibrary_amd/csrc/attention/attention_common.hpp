// attention_common.hpp -- arguments and launchers of the kernels around a quantised key-value cache.
#pragma once

#include <stdint.h>

#include <fklhip.h>

namespace fkattn {

// ---- arguments (plain values; the host fills them from the C ABI's structures after its checks) ----------------------

struct Rows {
    char* data;
    int64_t token_stride, head_stride;      // bytes
};

struct Cache {
    char *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, page_log, kv_heads;
    int codes;
};

struct HeadArgs {
    Rows q, k, v, q_out, k_out;
    const void *q_weight, *k_weight;
    const float *cos, *sin;
    const int32_t *positions, *slots;
    Cache cache;
    uint32_t tokens, table_rows;
    uint32_t q_heads, kv_heads, head_dim, rot_dim;
    uint32_t q_chunks, k_chunks;            // chunks of the kernel's heads; behind them come the values
    int pairs;
    float eps;
};

// With positions of several axes, one array behind the other; two bits of of_pairs say a pair's.
struct AxesHeadArgs : HeadArgs {
    int64_t position_stride;
    uint32_t axes, of_pairs[8];
    uint32_t sweeps, chunks_each;           // of many tokens: groups of lanes to a token, and chunks of heads to each
};

struct ReadArgs {
    Cache cache;
    Rows k, v;
    const int32_t* slots;
    uint32_t tokens, head_dim, k_chunks;
};

struct AttentionArgs {
    Rows q, out;
    float* lse;
    const int32_t *page_table, *context, *q_start;
    const uint64_t* mask;
    Cache cache;
    float *partial, *partial_lse;           // [shares][2][unit_rows](head_dim): a share's parts of row blocks
    int64_t page_table_stride;
    uint32_t room;                          // tokens that a row of the page table has entries for
    uint32_t tokens, batch, max_new, max_context, mask_words;
    uint32_t q_heads, group;                // query heads per key head
    uint32_t group_magic;                   // x / group as a multiplication (see divide)
    uint32_t unit_rows, granule_log, lead, share_log, share_odd;    // how the work is dealt out (work_shares.hpp)
    int type;
    float scale;
};
// share_odd is 0 in a launch with a workgroup to each row block

// With scores of another shape, and rows that see other keys (fklhip_scores).
struct ShapedArgs : AttentionArgs {
    const float* slopes;
    const int32_t *positions, *first, *prefix;
    float cap_in, cap_out;                  // 2 / cap, and cap in units of log2; 0 without
};

// Launchers (defined next to their kernels). Grids are laid out by the callers' arguments alone.
struct Launched { const char* kernel; unsigned grid[3], block[3], lds; };
int launch_heads(const HeadArgs& a, int type, bool to_cache, void* stream, Launched& info);
int launch_heads(const AxesHeadArgs& a, int type, bool to_cache, void* stream, Launched& info);
int launch_read(const ReadArgs& a, int type, void* stream, Launched& info);
int launch_merge(const AttentionArgs& a, uint32_t head_dim, bool many_parts, void* stream);
int launch_merge(const ShapedArgs& a, uint32_t head_dim, bool many_parts, void* stream);
// How a call is run: 16-row tiles (and so rows) and waves to a workgroup; row blocks of a sequence; share_odd << share_log
// shares, or none; whether rows have so many parts that a workgroup joins one.
struct AttentionPlan {
    uint32_t tiles, waves, row_blocks, unit_rows, granule_log, lead, share_log, share_odd;
    bool many_parts;
    uint32_t shares() const { return share_odd << share_log; }
};
// Whether attention's products are taken on a cache's codes as they are (kCodeProducts in tree_attention.hpp), or on keys as halves.
constexpr bool code_products(int head_dim, int codes) { return codes == FKLHIP_CODES_INT8 && head_dim % 64 == 0; }
// Whether a compute unit has room for three workgroups of two tiles with shaped scores: where keys are converted or heads have 64 elements, as
// 168 registers do then.
constexpr bool three_of_two_tiles(int head_dim, bool converted) { return head_dim <= 96 || (head_dim == 128 && converted); }
// Of scores of another shape: a sequence's query rows to a key head in the mean (0: scores are as they are), and whether rows see nothing of
// what is in front, and three_of_two_tiles.
struct ScoreShape { uint32_t mean_rows; bool fronts, three; };
AttentionPlan plan_attention(uint32_t batch, uint32_t kv_heads, uint32_t rows, uint32_t keys, uint32_t head_dim, ScoreShape shape);
template <int D> int launch_attention(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info);
template <int D> int launch_attention(const ShapedArgs& a, const AttentionPlan& plan, void* stream, Launched& info);

} // namespace fkattn
