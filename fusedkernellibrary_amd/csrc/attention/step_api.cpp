// step_api.cpp -- the C ABI of what a server's step does around attention (include/fklhip.h): checks of what the host can see,
// then a launch or two. Nothing here allocates, synchronises or keeps anything of a call but the text of its refusal.
#include "attention_checks.hpp"
#include "step_common.hpp"

#include <algorithm>

using namespace fkattn;

namespace {

constexpr int64_t kMost = std::numeric_limits<int32_t>::max();

int check_page(int32_t page_tokens) {
    NEED(page_tokens >= 16 && page_tokens <= 256 && (page_tokens & (page_tokens - 1)) == 0, "page_tokens has to be 16, 32, 64, 128 or 256");
    return FKLHIP_OK;
}
uint32_t log_of(int32_t n) { return uint32_t(__builtin_ctz(uint32_t(n))); }
constexpr int32_t kMostDrafts = 1024, kMostCaches = 1024;

int check_drafts(const fklhip_drafts* d) {
    NEED(d, "no drafts");
    NEED(d->type == FKLHIP_BF16 || d->type == FKLHIP_F16 || d->type == FKLHIP_F32, "type has to be FKLHIP_BF16, FKLHIP_F16 or FKLHIP_F32");
    CHECK(check_count(d->tokens));
    NEED(d->batch >= 0 && d->batch <= 65535, "batch has to be up to 65535");
    NEED(d->max_new >= 0 && d->max_new <= kMostDrafts, "max_new has to be up to 1024");
    NEED(d->vocab >= 1 && d->vocab <= 1 << 24, "vocab has to be 1 to 2^24");
    return FKLHIP_OK;
}
uint64_t sums_of(const fklhip_drafts& d) { return uint64_t(d.batch) * verify_chunks(uint32_t(d.vocab)) * 8; }
uint64_t workspace_of(const fklhip_drafts& d) { return d.max_new ? sums_of(d) + uint64_t(d.batch) * (kVerifyRecord + uint64_t(d.max_new)) * 4 : 0; }

// How far apart the nearest two of several caches' arrays of a kind begin, as a part of what such an array takes: 0 where one is given
// twice, below 1 where two overlap. (Two waves would move the same rows.)
double nearest_caches(const fklhip_kv_cache* caches, int32_t layers) {
    const uint64_t rows = uint64_t(caches->pages) * uint64_t(caches->kv_heads) * uint64_t(caches->page_tokens), codes = rows * uint64_t(caches->head_dim);
    uintptr_t at[kMostCaches];
    double nearest = HUGE_VAL;
    for (int kind = 0; kind < 4; ++kind) {
        for (int32_t i = 0; i < layers; ++i) {
            const fklhip_kv_cache& c = caches[i];
            at[i] = reinterpret_cast<uintptr_t>(kind == 0 ? c.k : kind == 1 ? c.v : kind == 2 ? static_cast<void*>(c.k_scale) : static_cast<void*>(c.v_scale));
        }
        if (!std::is_sorted(at, at + layers)) std::sort(at, at + layers);
        for (int32_t i = 1; i < layers; ++i) nearest = std::min(nearest, double(at[i] - at[i - 1]) / double(kind < 2 ? codes : rows * 4));
    }
    return nearest;
}

template <typename... P> bool all_aligned(size_t n, P... p) { return (aligned(p, n) && ...); }

} // namespace

extern "C" {

int fklhip_step_tables(const fklhip_tables* t, void* stream) {
    NEED(t, "no tables");
    CHECK(check_page(t->page_tokens));
    CHECK(check_count(t->tokens));
    NEED(t->batch >= 0 && t->batch <= 65535, "batch has to be up to 65535");
    NEED(t->max_new >= 0 && int64_t(t->batch) * t->max_new <= kMost, "max_new has to be 0 or more, and batch * max_new below 2^31");
    NEED(t->page_table_stride >= 0 && t->page_table_stride <= kMost && t->page_table_stride * t->batch <= kMost, "a page table has up to 2^31 - 1 entries");
    NEED(t->page_table_stride * t->page_tokens <= int64_t(1) << 30, "more than 2^30 tokens to a sequence");
    NEED(t->free_count >= 0 && t->free_count <= kMost, "free_count has to be 0 to 2^31 - 1");
    NEED(!t->parents || (t->mask_words >= 1 && t->mask_words <= 1 << 20 && int64_t(t->mask_words) * 64 >= t->max_new), "mask_words has to be max_new / 64, rounded up, or more");
    NEED(t->q_start && t->left && t->available, "no q_start, no left or no available");
    NEED(!t->batch || (t->held && t->context && t->fresh && t->held_out), "no lengths");
    NEED(!t->batch || t->page_table || !t->page_table_stride, "no page_table");
    NEED(!t->free_count || t->free_pages, "no free_pages");
    NEED(!t->tokens || (t->slots && t->positions && (!t->parents || t->mask)), "no slots, no positions or no mask");
    NEED(all_aligned(4, t->page_table, t->held, t->context, t->fresh, t->free_pages, t->available, t->parents, t->q_start, t->slots, t->positions, t->held_out, t->left) && aligned(t->mask, 8),
         "lengths and tables have to be aligned");
    NEED((!t->batch || t->held_out != t->held) && t->left != t->available, "held_out and left have to be other arrays than held and available");
    TablesArgs a{};
    a.page_table = t->page_table; a.held = t->held; a.context = t->context; a.fresh = t->fresh; a.free_pages = t->free_pages; a.available = t->available;
    a.parents = t->parents; a.q_start = t->q_start; a.slots = t->slots; a.positions = t->positions; a.held_out = t->held_out; a.left = t->left;
    a.mask = t->mask;
    a.page_table_stride = t->page_table_stride;
    a.tokens = uint32_t(t->tokens); a.batch = uint32_t(t->batch); a.width = uint32_t(t->page_table_stride); a.page_log = log_of(t->page_tokens);
    a.max_new = uint32_t(t->max_new); a.mask_words = uint32_t(t->mask_words); a.free_count = uint32_t(t->free_count);
    Launched info;
    return finish(launch_step_tables(a, stream, info), info);
}

int fklhip_verify_drafts_workspace(const fklhip_drafts* d, uint64_t* bytes) {
    NEED(bytes, "no place for the answer");
    CHECK(check_drafts(d));
    *bytes = workspace_of(*d);
    return FKLHIP_OK;
}

int fklhip_verify_drafts(const fklhip_drafts* d, void* stream) {
    CHECK(check_drafts(d));
    if (d->batch == 0 || d->max_new == 0) return FKLHIP_OK;
    NEED(d->q_start && d->path && d->count && d->out, "no q_start, or no place for the results");
    NEED(!d->tokens || (d->target && d->ids && d->uniforms), "no target, no ids or no uniforms");
    NEED(!d->draft || !d->parents, "draft's probabilities are of chains: not with parents");
    const size_t size = d->type == FKLHIP_F32 ? 4 : 2;
    NEED(all_aligned(size, d->target, d->draft) && all_aligned(4, d->ids, d->q_start, d->parents, d->uniforms, d->path, d->count, d->out), "probabilities, ids and results have to be aligned");
    const uint64_t bytes = workspace_of(*d);
    NEED(d->workspace && d->workspace_bytes >= bytes, "the workspace is smaller than fklhip_verify_drafts_workspace says");
    NEED(aligned(d->workspace, 8), "the workspace has to start at a multiple of 8 bytes");
    VerifyArgs a{};
    a.target = static_cast<const char*>(d->target); a.draft = static_cast<const char*>(d->draft);
    a.target_stride = d->target_stride * int64_t(size); a.draft_stride = d->draft_stride * int64_t(size);
    a.ids = d->ids; a.q_start = d->q_start; a.parents = d->parents; a.uniforms = d->uniforms;
    a.path = d->path; a.count = d->count; a.out = d->out;
    a.sums = static_cast<double*>(d->workspace);
    a.record = reinterpret_cast<int32_t*>(static_cast<char*>(d->workspace) + sums_of(*d));
    a.tokens = uint32_t(d->tokens); a.batch = uint32_t(d->batch); a.max_new = uint32_t(d->max_new); a.vocab = uint32_t(d->vocab);
    a.chunks = verify_chunks(a.vocab);
    Launched info;
    return finish(launch_verify(a, d->type, stream, info), info);
}

int fklhip_kv_keep(const fklhip_kv_cache* caches, int32_t layers, const int32_t* page_table, int64_t page_table_stride, const int32_t* context, const int32_t* path, const int32_t* count,
                   int32_t batch, int32_t max_new, void* stream) {
    NEED(layers >= 0 && layers <= kMostCaches, "layers has to be 0 to 1024");
    NEED(!layers || caches, "no caches");
    NEED(batch >= 0 && batch <= 65535, "batch has to be up to 65535");
    NEED(max_new >= 0 && max_new <= 1 << 20, "max_new has to be up to 2^20");
    NEED(page_table_stride >= 0 && page_table_stride <= kMost, "page_table_stride has to be 0 to 2^31 - 1");
    for (int32_t i = 0; i < layers; ++i) {
        const fklhip_kv_cache &c = caches[i], &first = caches[0];
        CHECK(check_cache(&c));
        NEED(c.pages == first.pages && c.kv_heads == first.kv_heads && c.page_tokens == first.page_tokens && c.head_dim == first.head_dim && c.codes == first.codes, "caches of different sizes");
    }
    const double nearest = layers ? nearest_caches(caches, layers) : HUGE_VAL;
    NEED(nearest > 0.0, "the same cache twice");
    if (!layers || !batch || !max_new || !page_table_stride) return FKLHIP_OK;
    NEED(page_table && context && path && count, "no page_table, no context, no path or no count");
    NEED(all_aligned(4, page_table, context, path, count), "lengths, path and page_table have to be aligned");
    NEED(nearest >= 1.0, "caches that overlap");
    KeepArgs a{};
    const Cache c = to_cache(caches[0]);
    a.page_table = page_table; a.context = context; a.path = path; a.count = count;
    a.page_table_stride = page_table_stride;
    a.pages = c.pages; a.page_log = c.page_log; a.kv_heads = c.kv_heads; a.head_dim = uint32_t(caches[0].head_dim);
    a.batch = uint32_t(batch); a.width = uint32_t(page_table_stride); a.max_new = uint32_t(max_new);
    Launched info{};
    for (int32_t done = 0; done < layers; done += kMostLayers) {
        const int32_t n = std::min(layers - done, kMostLayers);
        for (int32_t i = 0; i < n; ++i) {
            const fklhip_kv_cache& from = caches[done + i];
            a.caches[i] = {static_cast<char*>(from.k), static_cast<char*>(from.v), from.k_scale, from.v_scale};
        }
        if (const int rc = launch_keep(a, uint32_t(n), stream, info); rc != FKLHIP_OK) return rc;
    }
    return finish(FKLHIP_OK, info);
}

} // extern "C"
