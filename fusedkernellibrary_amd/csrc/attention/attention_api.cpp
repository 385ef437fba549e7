// attention_api.cpp -- the C ABI of the operators around a quantised key-value cache (include/fklhip.h): checks of what the
// host can see, then one or two launches. Nothing here allocates, synchronises or keeps anything of a call but the text
// of its refusal.
#include "attention_checks.hpp"

#include <algorithm>
#include <cstring>

using namespace fkattn;

namespace {
thread_local const char* g_argument_error = "";
}
namespace fkattn {
int refuse(const char* what) {
    g_argument_error = what;
    return FKLHIP_EINVAL;
}
}

namespace {

int run_heads(const fklhip_heads* h, const fklhip_axes* axes, const fklhip_kv_cache* cache, void* stream) {
    NEED(h, "no heads");
    CHECK(check_type(h->type));
    CHECK(check_count(h->tokens));
    NEED(h->head_dim >= 8 && h->head_dim <= 256 && h->head_dim % 8 == 0, "head_dim has to be a multiple of 8 up to 256");
    NEED(h->rot_dim >= 0 && h->rot_dim <= h->head_dim && h->rot_dim % 8 == 0, "rot_dim has to be a multiple of 8 up to head_dim");
    NEED(h->q_heads >= 1 && h->q_heads <= 65535 && h->kv_heads >= 1 && h->kv_heads <= 65535, "q_heads and kv_heads have to be 1 to 65535");
    NEED(h->pairs == 0 || h->pairs == 1, "pairs has to be 0 or 1");
    NEED(!h->rot_dim || !h->tokens || (h->cos && h->sin && h->positions && h->table_rows >= 1), "rot_dim without tables or positions");
    NEED(!h->rot_dim || (aligned(h->cos, 16) && aligned(h->sin, 16)), "tables have to start at multiples of 16 bytes");
    NEED(aligned(h->positions, 4) && aligned(h->slots, 4), "positions and slots have to be aligned");
    NEED(h->table_rows >= 0 && h->table_rows <= std::numeric_limits<int32_t>::max(), "a table has up to 2^31 - 1 rows");
    NEED((h->q_weight == nullptr) == (h->k_weight == nullptr), "weights for both of q and k, or for none");
    NEED(!h->q_weight || (aligned(h->q_weight, 8) && aligned(h->k_weight, 8)), "weights have to start at multiples of 8 bytes");
    NEED(!h->q_weight || h->eps >= 0.0f, "eps has to be 0 or more");
    if (axes) {
        NEED(axes->count >= 1 && axes->count <= 4, "1 to 4 axes");
        for (int32_t i = 0; i < h->rot_dim / 2; ++i) NEED(axes->of_pair[i] < axes->count, "a pair's axis is none of them");
    }
    if (cache) {
        CHECK(check_cache(cache));
        NEED(cache->kv_heads == h->kv_heads && cache->head_dim == h->head_dim, "the cache is of other heads");
    }
    if (h->tokens == 0) return FKLHIP_OK;
    CHECK(check_rows(h->q, h->tokens, h->q_heads));
    CHECK(check_rows(h->k, h->tokens, h->kv_heads));
    CHECK(check_out(h->q_out, h->tokens, h->q_heads, h->head_dim));
    if (cache) {
        CHECK(check_rows(h->v, h->tokens, h->kv_heads));
        NEED(h->slots, "no slots");
    } else {
        CHECK(check_out(h->k_out, h->tokens, h->kv_heads, h->head_dim));
    }
    AxesHeadArgs a{};
    a.q = to_rows(h->q); a.k = to_rows(h->k); a.q_out = to_rows(h->q_out);
    if (cache) { a.v = to_rows(h->v); a.cache = to_cache(*cache); }
    else a.k_out = to_rows(h->k_out);
    a.q_weight = h->q_weight; a.k_weight = h->k_weight;
    a.cos = h->cos; a.sin = h->sin; a.positions = h->positions; a.slots = h->slots;
    a.tokens = uint32_t(h->tokens); a.table_rows = uint32_t(h->table_rows);
    a.q_heads = uint32_t(h->q_heads); a.kv_heads = uint32_t(h->kv_heads);
    a.head_dim = uint32_t(h->head_dim); a.rot_dim = uint32_t(h->rot_dim);
    a.pairs = h->pairs; a.eps = h->eps;
    Launched info;
    if (!axes) return finish(launch_heads(static_cast<const HeadArgs&>(a), h->type, cache != nullptr, stream, info), info);
    a.axes = uint32_t(axes->count);
    a.position_stride = axes->stride;
    for (int32_t i = 0; i < h->rot_dim / 2; ++i) a.of_pairs[i / 16] |= uint32_t(axes->of_pair[i]) << (i % 16 * 2);
    return finish(launch_heads(a, h->type, cache != nullptr, stream, info), info);
}

int plan_call(const fklhip_attention* c, const fklhip_kv_cache* cache, bool shaped, bool fronts, AttentionPlan& plan) {
    NEED(c, "no call");
    CHECK(check_type(c->type));
    CHECK(check_cache(cache));
    CHECK(check_count(c->tokens));
    NEED(cache->head_dim == 64 || cache->head_dim == 96 || cache->head_dim == 128 || cache->head_dim == 192 || cache->head_dim == 256,
         "attention takes heads of 64, 96, 128, 192 or 256 elements");
    NEED(c->q_heads >= 1 && c->q_heads % cache->kv_heads == 0 && c->q_heads <= 65535, "q_heads has to be a multiple of kv_heads up to 65535");
    NEED(c->batch >= 0 && c->batch <= 65535, "batch has to be up to 65535");
    NEED(c->max_new >= 0 && c->max_context >= 0, "max_new and max_context have to be 0 or more");
    NEED(int64_t(c->max_context) + c->max_new <= (1 << 30), "more than 2^30 tokens to a sequence");
    const int64_t group = c->q_heads / cache->kv_heads;
    NEED(c->max_new * group * group < (int64_t(1) << 32) && c->max_new * group <= (int64_t(1) << 20), "more than 2^20 query rows to a key head");
    NEED(c->tokens * c->q_heads < (int64_t(1) << 31), "more than 2^31 - 1 query rows");
    NEED(c->page_table_stride >= 0 && c->page_table_stride <= std::numeric_limits<int32_t>::max(), "page_table_stride has to be 0 to 2^31 - 1");
    const uint32_t keys = uint32_t(std::min<int64_t>(int64_t(c->max_context) + c->max_new, c->page_table_stride * cache->page_tokens));
    plan = plan_attention(uint32_t(c->batch), uint32_t(cache->kv_heads), uint32_t(c->max_new * group), keys, uint32_t(cache->head_dim),
                          {shaped ? uint32_t(std::max<int64_t>(1, c->tokens * group / std::max(1, c->batch))) : 0u, fronts,
                           shaped && three_of_two_tiles(cache->head_dim, !code_products(cache->head_dim, cache->codes))});
    return FKLHIP_OK;
}

uint64_t workspace_of(const fklhip_kv_cache& cache, const AttentionPlan& plan) {
    return uint64_t(plan.shares()) * 2 * plan.unit_rows * (cache.head_dim + 1) * 4;
}

template <typename A> int launch_any(const A& a, uint32_t head_dim, const AttentionPlan& plan, bool parts, void* stream, Launched& info) {
    int rc;
    switch (head_dim) {
    case 64: rc = launch_attention<64>(a, plan, stream, info); break;
    case 96: rc = launch_attention<96>(a, plan, stream, info); break;
    case 128: rc = launch_attention<128>(a, plan, stream, info); break;
    case 192: rc = launch_attention<192>(a, plan, stream, info); break;
    default: rc = launch_attention<256>(a, plan, stream, info); break;
    }
    if (rc == FKLHIP_OK && parts) rc = launch_merge(a, head_dim, plan.many_parts, stream);
    return rc;
}

int run_attention(const fklhip_attention* c, const fklhip_scores* h, const fklhip_kv_cache* cache, void* stream) {
    AttentionPlan plan;
    const bool shaped = h && (h->cap != 0.0f || h->slopes || h->first || h->prefix);
    CHECK(plan_call(c, cache, shaped, shaped && h->first, plan));
    NEED(std::isfinite(c->scale), "scale has to be finite");
    if (h) {
        NEED(h->cap == 0.0f || (h->cap >= 0x1p-6f && h->cap <= 0x1p9f), "cap has to be 0, or 2^-6 to 2^9");
        NEED(!h->prefix || !c->mask, "a prefix and a mask");
        NEED(aligned(h->slopes, 4) && aligned(h->positions, 4) && aligned(h->first, 4) && aligned(h->prefix, 4), "slopes, positions, first and prefix have to be aligned");
    }
    if (c->tokens == 0 || c->batch == 0 || c->max_new == 0) return FKLHIP_OK;
    CHECK(check_rows(c->q, c->tokens, c->q_heads));
    CHECK(check_out(c->out, c->tokens, c->q_heads, cache->head_dim));
    NEED(c->context && c->q_start, "no context or no q_start");
    NEED(c->page_table || c->page_table_stride == 0, "no page_table");
    NEED(aligned(c->context, 4) && aligned(c->q_start, 4) && aligned(c->page_table, 4) && aligned(c->lse, 4) && aligned(c->mask, 8), "lengths, page_table, lse and mask have to be aligned");
    NEED(!c->mask || (c->mask_words >= 1 && int64_t(c->mask_words) * 64 >= c->max_new), "mask_words has to be max_new / 64, rounded up, or more");
    const uint64_t bytes = workspace_of(*cache, plan);
    NEED(bytes == 0 || (c->workspace && c->workspace_bytes >= bytes), "the workspace is smaller than fklhip_tree_attention_workspace says");
    NEED(bytes == 0 || aligned(c->workspace, 16), "the workspace has to start at a multiple of 16 bytes");
    ShapedArgs a{};
    a.q = to_rows(c->q); a.out = to_rows(c->out); a.lse = c->lse;
    a.page_table = c->page_table; a.context = c->context; a.q_start = c->q_start; a.mask = c->mask;
    a.cache = to_cache(*cache);
    a.page_table_stride = c->page_table_stride;
    a.tokens = uint32_t(c->tokens); a.batch = uint32_t(c->batch); a.max_new = uint32_t(c->max_new); a.max_context = uint32_t(c->max_context);
    a.mask_words = uint32_t(c->mask_words); a.q_heads = uint32_t(c->q_heads); a.group = uint32_t(c->q_heads / cache->kv_heads);
    a.group_magic = magic(a.group);
    a.room = uint32_t(std::min<int64_t>(c->page_table_stride * cache->page_tokens, int64_t(c->max_context) + c->max_new));
    // (without room nobody sees anything: all rows are written like rows of no sequence, and nothing is read for them)
    if (a.room == 0) a.max_new = 0;
    a.unit_rows = plan.unit_rows;
    a.granule_log = plan.granule_log; a.lead = plan.lead; a.share_log = plan.share_log; a.share_odd = plan.share_odd;
    a.type = c->type; a.scale = c->scale;
    if (bytes) {
        a.partial = static_cast<float*>(c->workspace);
        a.partial_lse = a.partial + uint64_t(plan.shares()) * 2 * plan.unit_rows * uint64_t(cache->head_dim);
    }
    Launched info;
    if (!shaped) return finish(launch_any(static_cast<const AttentionArgs&>(a), uint32_t(cache->head_dim), plan, bytes != 0, stream, info), info);
    a.slopes = h->slopes; a.positions = h->positions; a.first = h->first; a.prefix = h->prefix;
    if (h->cap != 0.0f) {
        a.cap_in = 2.0f / h->cap;
        a.cap_out = h->cap * 1.4426950408889634f;
    }
    return finish(launch_any(a, uint32_t(cache->head_dim), plan, bytes != 0, stream, info), info);
}

} // namespace

extern "C" {

int fklhip_argument_error(const char** text) {
    if (!text) return FKLHIP_EINVAL;
    *text = g_argument_error;
    return FKLHIP_OK;
}

int fklhip_qk_norm_rope(const fklhip_heads* heads, void* stream) { return run_heads(heads, nullptr, nullptr, stream); }

int fklhip_qk_norm_rope_axes(const fklhip_heads* heads, const fklhip_axes* axes, void* stream) {
    NEED(axes, "no axes");
    return run_heads(heads, axes, nullptr, stream);
}

int fklhip_qkv_to_cache(const fklhip_heads* heads, const fklhip_kv_cache* cache, void* stream) {
    NEED(cache, "no cache");
    return run_heads(heads, nullptr, cache, stream);
}

int fklhip_qkv_to_cache_axes(const fklhip_heads* heads, const fklhip_axes* axes, const fklhip_kv_cache* cache, void* stream) {
    NEED(axes, "no axes");
    NEED(cache, "no cache");
    return run_heads(heads, axes, cache, stream);
}

int fklhip_kv_write(const fklhip_kv_cache* cache, const fklhip_rows* k, const fklhip_rows* v, const int32_t* slots, int64_t tokens, int type, void* stream) {
    CHECK(check_cache(cache));
    CHECK(check_type(type));
    CHECK(check_count(tokens));
    if (tokens == 0) return FKLHIP_OK;
    NEED(k && v && slots, "no rows or no slots");
    NEED(aligned(slots, 4), "slots have to be aligned");
    CHECK(check_rows(*k, tokens, cache->kv_heads));
    CHECK(check_rows(*v, tokens, cache->kv_heads));
    HeadArgs a{};
    a.k = to_rows(*k); a.v = to_rows(*v); a.cache = to_cache(*cache); a.slots = slots;
    a.tokens = uint32_t(tokens); a.q_heads = 0; a.kv_heads = uint32_t(cache->kv_heads); a.head_dim = uint32_t(cache->head_dim);
    Launched info;
    return finish(launch_heads(a, type, true, stream, info), info);
}

int fklhip_kv_read(const fklhip_kv_cache* cache, const int32_t* slots, int64_t tokens, const fklhip_rows* k, const fklhip_rows* v, int type, void* stream) {
    CHECK(check_cache(cache));
    CHECK(check_type(type));
    CHECK(check_count(tokens));
    if (tokens == 0) return FKLHIP_OK;
    NEED(k && v && slots, "no rows or no slots");
    NEED(aligned(slots, 4), "slots have to be aligned");
    CHECK(check_out(*k, tokens, cache->kv_heads, cache->head_dim));
    CHECK(check_out(*v, tokens, cache->kv_heads, cache->head_dim));
    ReadArgs a{to_cache(*cache), to_rows(*k), to_rows(*v), slots, uint32_t(tokens), uint32_t(cache->head_dim), 0};
    Launched info;
    return finish(launch_read(a, type, stream, info), info);
}

int fklhip_tree_attention_workspace(const fklhip_attention* call, const fklhip_kv_cache* cache, uint64_t* bytes) {
    NEED(bytes, "no place for the answer");
    AttentionPlan plan, shaped;
    CHECK(plan_call(call, cache, false, false, plan));
    CHECK(plan_call(call, cache, true, false, shaped));        // (with fronts there are shares, the same, or none)
    *bytes = std::max(workspace_of(*cache, plan), workspace_of(*cache, shaped));
    return FKLHIP_OK;
}

int fklhip_tree_attention(const fklhip_attention* c, const fklhip_kv_cache* cache, void* stream) { return run_attention(c, nullptr, cache, stream); }

int fklhip_shaped_attention(const fklhip_attention* c, const fklhip_scores* scores, const fklhip_kv_cache* cache, void* stream) {
    NEED(scores, "no scores");
    return run_attention(c, scores, cache, stream);
}

} // extern "C"

namespace fkattn {

AttentionPlan plan_attention(uint32_t batch, uint32_t kv_heads, uint32_t rows, uint32_t keys, uint32_t head_dim, ScoreShape shape) {
    const auto log2_floor = [](uint64_t n) { uint32_t l = 0; while (n >>= 1) ++l; return l; };
    AttentionPlan p;
    p.granule_log = 7;
    const uint64_t length = (uint64_t(keys) + (1u << p.granule_log) - 1) >> p.granule_log;     // of the longest sequence there may be
    const auto blocks = [&](uint32_t tiles) { return std::max(1u, (rows + 16 * tiles - 1) / (16 * tiles)); };
    const auto units = [&](uint32_t tiles) { return uint64_t(batch) * kv_heads * blocks(tiles); };
    const uint32_t most_tiles = rows <= 16 ? 1 : rows <= 32 || head_dim > 128 ? 2 : 4;         // (each takes registers)
    const uint32_t slots = head_dim > 128 ? 256 : 512;                                       // workgroups at once on 256 compute units
    // A workgroup to each row block, if all run at once and none is long: joining shares' parts costs 6 us and more. Small blocks
    // are the faster ones then, whose keys come from the L2 cache again; one tile's has eight waves if each has a compute unit.
    // Measured, 8 key heads of 128 (4 waves, 8 waves, shares, in us): one sequence of 1000 keys 12.1, 11.7, 14.4; 2000 17.8, 16.9,
    // 16.3; 3000 23.4, 22.2, 16.2: a compute unit reads 50 GB/s of what eight waves ask for. 2 key heads of 64, 2000 keys: 14.5, 11.6, 14.5.
    // 16 tokens, 16 sequences of 1000 keys: one tile 18.7, two 18.8, four 27.2, shares of two tiles 26.8; one sequence of
    // 1000: 12.5, 16.8, 25.3 and 16.8.
    p.tiles = 1;
    while (p.tiles < most_tiles && units(p.tiles) > slots) p.tiles *= 2;
    p.waves = p.tiles == 1 && units(1) <= 256 ? 8 : 4;
    const uint64_t worth = (p.waves == 8 ? 16 : p.tiles == 4 ? 6 : 8) * 128 / head_dim;
    p.share_log = 0;
    p.share_odd = 0;
    // (sequences are taken to be half as long as the longest in the mean: shares use the compute units that ended early)
    const bool whole = units(p.tiles) <= slots ? length * (2 * slots - units(p.tiles)) <= worth * 2 * slots : length <= 8;
    if (!whole) {
        // shares: the fewer blocks the less is converted and read, unless a share has so little that beginning and ending it counts more
        // Shaped scores of trees with up to 64 rows, 40 or fewer in the mean, have two tiles: most of four would be empty. 16 of 3 to 13 tokens
        // behind windows of 4096, four query heads to a key head, two tiles and four, in us: e4m3 49.8, 53.8, int8 in half precision 53.8,
        // 60.6; 5 to 13 over 500 to 4100, int8, 36.2, 43.1; but 16 tokens each 59.8, 56.6.
        // All have two where three workgroups of two tiles fit a compute unit, e4m3, in us, two and four: 16 trees of 33 to 61 over 500 to 4100 74.1,
        // 79.9; 20 to 29 behind windows 75.6, 81.4; four prompts of 100 to 130 over 2000 to 3000 51.1, 56.0; the first of the above 47.5.
        p.tiles = shape.three || (shape.mean_rows && rows <= 64 && shape.mean_rows <= 40) ? std::min(most_tiles, 2u) : most_tiles;
        p.waves = 4;
        while (p.tiles > 1 && units(p.tiles) * length < uint64_t(p.tiles == 4 ? 8 : 4) * slots) p.tiles /= 2;
    }
    p.unit_rows = 16 * p.tiles;
    p.row_blocks = blocks(p.tiles);
    p.lead = p.tiles == 1 ? 1 : p.tiles == 2 ? 3 : 5;
    if (!whole) {
        // As many shares as workgroups run at once, or a power of two that leaves two granules to each; none where the order of launch
        // evens things out, as four times as many row blocks do, or a single sequence's that are twice as many. Measured, prompts over
        // 32 and 8 heads of 128, int8 (whole blocks, shares, in us): 2048 tokens 75.5, 99.7; behind 4000 others 241, 267; 4096 tokens
        // 228, 312; two of 2048 141, 212; three of 1500 134, 186; four of 1100 114, 171; 2048 and 300 85, 125; 1500, 200 and 700 67, 98.
        // Both bounds are high: of what stays in shares, one of 1100 takes 59.2 and would take 33.7, two 98 and 63, three 124 and 87,
        // two of 1500 137 and 92.
        const uint64_t all = units(p.tiles) * (p.lead + length);
        p.share_odd = slots == 512 && (p.tiles == 1 || (shape.three && p.tiles == 2)) ? 3 : 1;
        p.share_log = p.share_odd == 3 || slots == 256 ? 8 : 9;
        bool enough = units(p.tiles) >= uint64_t(batch == 1 ? 2 : 4) * p.shares();
        // Of shaped scores fewer do: as many if none is long; one and a half times as many of prompts, or where rows do not see what is in front; 256
        // of prompts then (a block's keys are few, and shares would end within them all the same). Measured, 32 and 8 heads of 128, e4m3, half
        // precision, four tiles, which such prompts had then (whole blocks, shares, in us): capped, one of 1100 tokens 39.2, 67.4, behind 3000 others
        // 161, 140; one of 1500 62, 91, and 191, 195; two of 1100 67, 100; three of 500 behind 1000 to 3000 112, 124; windows of 512, one of 300 behind
        // 3000 20.4, 29.4, of 700 32.1, 45.5, two of 1100 behind 1000 to 3000 62, 92; four documents, two of 700 49, 70, three of 1100 64.5, 98.4.
        // Single tokens and trees that see all have shares, as one long sequence among short ones would end alone, and the host knows the
        // longest only. Capped, bfloat16, in the forms that they have now: 64 tokens, 20 heads of 128, int8, one over 131072 and the others
        // over 1000 967, 195; evenly up to 8000 271, 263; up to 2500 93, 97; 48, 16 and 8 heads of 256, evenly up to 20000 456, 393. 48 trees of 30, 32 and 8
        // heads of 128, evenly up to 4000 152, 143, up to 2000 90, 95, one over 16000 and the others over 1000 331, 108; in windows of 512 60, 75.
        if (shape.mean_rows) enough |= (2 * units(p.tiles) >= 3 * uint64_t(p.shares()) && (rows >= 512 || shape.fronts)) || (units(p.tiles) >= p.shares() && length <= 16);
        if (shape.fronts) enough |= units(p.tiles) >= 256 && rows >= 512 && length <= 64;
        if (enough || all >= (uint64_t(1) << 30)) p.share_odd = 0;
        else if (all < uint64_t(2) * p.shares()) p.share_log = log2_floor(all / 2), p.share_odd = 1;
    }
    p.many_parts = p.shares() > 16 * units(p.tiles);
    return p;
}

} // namespace fkattn
