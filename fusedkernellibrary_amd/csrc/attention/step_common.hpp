// step_common.hpp -- arguments and launchers of what a server's step does around attention: its tables, the verification of its
// drafted tokens, the cache rows that it keeps.
#pragma once

#include "attention_common.hpp"

namespace fkattn {

struct TablesArgs {
    int32_t* page_table;
    const int32_t *held, *context, *fresh, *free_pages, *available, *parents;
    int32_t *q_start, *slots, *positions, *held_out, *left;
    uint64_t* mask;
    int64_t page_table_stride;
    uint32_t tokens, batch, width, page_log, max_new, mask_words, free_count;
};

constexpr uint32_t kVerifyRecord = 8;
struct VerifyArgs {
    const char *target, *draft;
    int64_t target_stride, draft_stride;    // bytes
    const int32_t *ids, *q_start, *parents;
    const float* uniforms;
    int32_t *path, *count, *out;
    double* sums;                           // [batch][chunks]
    int32_t* record;                        // [batch][kVerifyRecord + max_new]
    uint32_t tokens, batch, max_new, vocab, chunks;
};

struct KeepCache {
    char *k, *v;
    float *k_scale, *v_scale;
};
constexpr int kMostLayers = 64;             // of a launch
struct KeepArgs {
    KeepCache caches[kMostLayers];
    const int32_t *page_table, *context, *path, *count;
    int64_t page_table_stride;
    uint32_t pages, page_log, kv_heads, head_dim, batch, width, max_new;
};

int launch_step_tables(const TablesArgs& a, void* stream, Launched& info);
uint32_t verify_chunks(uint32_t vocab);
int launch_verify(const VerifyArgs& a, int type, void* stream, Launched& info);
int launch_keep(const KeepArgs& a, uint32_t layers, void* stream, Launched& info);

} // namespace fkattn
