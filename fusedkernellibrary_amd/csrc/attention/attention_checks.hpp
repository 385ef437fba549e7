// attention_checks.hpp -- what the entry points around a quantised key-value cache check their arguments with.
#pragma once

#include <fklhip.h>

#include "../registry.hpp"
#include "attention_common.hpp"

#include <cmath>
#include <cstdlib>
#include <limits>
#include <utility>

namespace fkattn {

// Keeps the text for fklhip_argument_error, and is FKLHIP_EINVAL.
int refuse(const char* what);
#define NEED(condition, what) do { if (!(condition)) return refuse(what); } while (0)

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows [count][heads][dim]: null or not, 16-byte pieces.
inline int check_rows(const fklhip_rows& r, int64_t count, int64_t heads) {
    NEED(r.data, "rows without data");
    NEED(aligned(r.data, 16), "rows have to start at a multiple of 16 bytes");
    NEED(count <= 1 || r.token_stride % 8 == 0, "a token stride has to be a multiple of 8 elements");
    NEED(heads <= 1 || r.head_stride % 8 == 0, "a head stride has to be a multiple of 8 elements");
    return FKLHIP_OK;
}
// Whether two of an output's rows share bytes: two workgroups would write there, in any order.
inline bool overlaps(const fklhip_rows& r, int64_t count, int64_t heads, int64_t dim) {
    // (a stride of a dimension of one row is not looked at)
    int64_t step[2] = {std::abs(r.head_stride), std::abs(r.token_stride)}, n[2] = {heads, count};
    if (n[0] <= 1 || (n[1] > 1 && step[1] < step[0])) std::swap(step[0], step[1]), std::swap(n[0], n[1]);
    if (n[0] <= 1) return false;
    if (step[0] < dim) return true;
    if (n[1] <= 1 || (step[1] - dim) / step[0] >= n[0] - 1) return false;
    // Rows in between others: i steps of the smaller stride against j of the larger. (Negative strides are the same places from
    // another end.)
    const __int128 small = step[0], large = step[1], end = small * (n[0] - 1) + dim;
    for (int64_t j = 1; j < n[1] && large * j < end; ++j) {
        const __int128 i = large * j / small, left = large * j - i * small;
        if ((i < n[0] && left < dim) || (i + 1 < n[0] && small - left < dim)) return true;
    }
    return false;
}
inline int check_out(const fklhip_rows& r, int64_t count, int64_t heads, int64_t dim) {
    if (const int rc = check_rows(r, count, heads); rc != FKLHIP_OK) return rc;
    NEED(!overlaps(r, count, heads, dim), "rows of an output overlap");
    return FKLHIP_OK;
}
inline Rows to_rows(const fklhip_rows& r) { return {static_cast<char*>(r.data), r.token_stride * 2, r.head_stride * 2}; }

inline int check_type(int type) {
    NEED(type == FKLHIP_BF16 || type == FKLHIP_F16, "type has to be FKLHIP_BF16 or FKLHIP_F16");
    return FKLHIP_OK;
}
inline int check_count(int64_t tokens) {
    NEED(tokens >= 0, "a negative number of tokens");
    NEED(tokens < (int64_t(1) << 30), "more than 2^30 tokens");
    return FKLHIP_OK;
}
inline int check_cache(const fklhip_kv_cache* c) {
    NEED(c, "no cache");
    NEED(c->k && c->v && c->k_scale && c->v_scale, "a cache without data");
    NEED(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->k_scale, 16) && aligned(c->v_scale, 16), "a cache's arrays have to start at multiples of 16 bytes");
    NEED(c->codes == FKLHIP_CODES_INT8 || c->codes == FKLHIP_CODES_E4M3, "codes have to be FKLHIP_CODES_INT8 or FKLHIP_CODES_E4M3");
    NEED(c->page_tokens >= 16 && c->page_tokens <= 256 && (c->page_tokens & (c->page_tokens - 1)) == 0, "page_tokens has to be 16, 32, 64, 128 or 256");
    NEED(c->pages >= 1 && c->pages <= std::numeric_limits<int32_t>::max() && c->pages * c->page_tokens <= std::numeric_limits<int32_t>::max(), "a cache has 1 to 2^31 - 1 slots");
    NEED(c->kv_heads >= 1 && c->kv_heads <= 65535, "kv_heads has to be 1 to 65535");
    NEED(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0, "head_dim has to be a multiple of 8 up to 256");
    return FKLHIP_OK;
}
inline Cache to_cache(const fklhip_kv_cache& c) {
    uint32_t log = 0;
    while ((1 << log) < c.page_tokens) ++log;
    return {static_cast<char*>(c.k), static_cast<char*>(c.v), c.k_scale, c.v_scale, uint32_t(c.pages), log, uint32_t(c.kv_heads), c.codes};
}
inline uint32_t magic(uint32_t n) { return n == 1 ? 0 : uint32_t(((uint64_t(1) << 32) + n - 1) / n); }

inline int finish(int rc, const Launched& info) {
    if (rc == FKLHIP_OK) fklhip::note_launch(info.kernel, info.grid, info.block, info.lds);
    return rc;
}

#define CHECK(call) do { const int rc_ = (call); if (rc_ != FKLHIP_OK) return rc_; } while (0)

} // namespace fkattn
