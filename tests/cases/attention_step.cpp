// attention_step.cpp -- a server's step spelled with the C++ host API (algorithms/attention/attention.h): norm, rotation and write of
// the new tokens, attention over the cache, and the new tokens' rows read back. Compiled by g++ without HIP headers.
#include <fused_kernel/algorithms/attention/attention.h>

#include <cstring>
#include <exception>
#include <memory>

namespace {
thread_local char g_error[512] = "";
template <typename F> int guarded(F body) {
    try {
        body();
        return 0;
    } catch (const std::invalid_argument& e) {
        std::strncpy(g_error, e.what(), sizeof g_error - 1);
        return 2;
    } catch (const std::exception& e) {
        std::strncpy(g_error, e.what(), sizeof g_error - 1);
        return 1;
    }
}
struct Server {
    fk::KvCache cache;
    fk::TreeAttention attend;
};
} // namespace

extern "C" {

const char* attention_step_error() { return g_error; }

int attention_step_open(int64_t pages, int32_t kv_heads, int32_t page_tokens, int32_t head_dim, int32_t codes, void** server) {
    return guarded([&] { *server = new Server{fk::KvCache(pages, kv_heads, page_tokens, head_dim, static_cast<fk::CacheCodes>(codes)), {}}; });
}
void attention_step_close(void* server) { delete static_cast<Server*>(server); }

// Rows of q, k and v heads side by side; q is changed in place, out is [tokens][q_heads][head_dim], k and v as they were stored.
int attention_step_run(void* server, void* packed, void* out, void* k_out, void* v_out, const void* q_weight, const void* k_weight, const float* cos, const float* sin, int64_t table_rows,
                       const int32_t* positions, const int32_t* slots, const int32_t* page_table, int64_t entries, const int32_t* context, const int32_t* q_start, int32_t batch, int64_t tokens,
                       int32_t q_heads, int32_t max_new, int32_t max_context, int32_t type, void* stream_) {
    return guarded([&] {
        Server& s = *static_cast<Server*>(server);
        const fklhip_kv_cache& c = s.cache;
        fk::Stream_<fk::ParArch::GPU_AMD> stream(stream_);
        const int32_t in_row = q_heads + 2 * c.kv_heads;
        fklhip_heads h{};
        h.q = h.q_out = fk::headRows(packed, in_row, c.head_dim);
        h.k = fk::headRows(packed, in_row, c.head_dim, q_heads);
        h.v = fk::headRows(packed, in_row, c.head_dim, q_heads + c.kv_heads);
        h.q_weight = q_weight; h.k_weight = k_weight; h.cos = cos; h.sin = sin; h.table_rows = table_rows; h.rot_dim = c.head_dim;
        h.positions = positions; h.slots = slots; h.tokens = tokens; h.q_heads = q_heads; h.kv_heads = c.kv_heads; h.head_dim = c.head_dim;
        h.type = type; h.eps = 1e-6f;
        fk::qkvToCache(h, c, stream);
        fklhip_attention a{};
        a.q = h.q_out;
        a.out = fk::headRows(out, q_heads, c.head_dim);
        a.page_table = page_table; a.page_table_stride = entries; a.context = context; a.q_start = q_start;
        a.tokens = tokens; a.batch = batch; a.max_new = max_new; a.max_context = max_context; a.q_heads = q_heads; a.type = type;
        a.scale = 1.0f / __builtin_sqrtf(float(c.head_dim));
        s.attend(a, c, stream);
        fk::kvRead(c, slots, tokens, fk::headRows(k_out, c.kv_heads, c.head_dim), fk::headRows(v_out, c.kv_heads, c.head_dim), static_cast<fk::RowType>(type), stream);
    });
}

} // extern "C"
