// drafts_step.cpp -- a server's step of drafted tokens spelled with the C++ host API (algorithms/attention/attention.h): tables, and in
// each layer norm, rotation and write, attention; then verification and the accepted rows. Compiled by g++ without HIP headers.
#include <fused_kernel/algorithms/attention/attention.h>

#include <cstring>
#include <exception>

namespace {
thread_local char g_error[512] = "";
int failed(const int code, const std::exception& e) {
    std::strncpy(g_error, e.what(), sizeof g_error - 1);
    return code;
}
template <typename F> int guarded(F body) {
    try {
        body();
        return 0;
    } catch (const std::invalid_argument& e) {
        return failed(2, e);
    } catch (const std::logic_error& e) {
        return failed(3, e);
    } catch (const std::exception& e) {
        return failed(1, e);
    }
}
struct Server {
    fk::TreeAttention attend;
    fk::VerifyDrafts verify;
};
} // namespace

extern "C" {

const char* drafts_step_error() { return g_error; }

void* drafts_step_open() { return new Server; }
void drafts_step_close(void* server) { delete static_cast<Server*>(server); }

int drafts_step_reserve(void* server, const fklhip_attention* call, const fklhip_drafts* drafts, const fklhip_kv_cache* cache) {
    return guarded([&] {
        static_cast<Server*>(server)->attend.reserve(*call, *cache);
        static_cast<Server*>(server)->verify.reserve(*drafts);
    });
}

// heads[i], calls[i] and caches[i] are layer i's; pair j turns by axis of_pair[j].
int drafts_step_run(void* server, const fklhip_tables* tables, const fklhip_heads* heads, const uint8_t* of_pair, int32_t pairs, int32_t axes, int64_t stride, const fklhip_attention* calls,
                    const fklhip_scores* scores, const fklhip_drafts* drafts, const fklhip_kv_cache* caches, int32_t layers, void* stream_) {
    return guarded([&] {
        Server& s = *static_cast<Server*>(server);
        fk::Stream_<fk::ParArch::GPU_AMD> stream(stream_);
        const fklhip_axes turns = fk::ropeAxes(std::vector<uint8_t>(of_pair, of_pair + pairs), axes, stride);
        fk::stepTables(*tables, stream);
        for (int32_t i = 0; i < layers; ++i) {
            fk::qkvToCache(heads[i], turns, caches[i], stream);
            s.attend(calls[i], *scores, caches[i], stream);
        }
        s.verify(*drafts, stream);
        fk::kvKeep(std::vector<fklhip_kv_cache>(caches, caches + layers), tables->page_table, tables->page_table_stride, tables->context, drafts->path, drafts->count, tables->batch, tables->max_new, stream);
    });
}

// Norm and rotation without a cache.
int drafts_step_turn(const fklhip_heads* heads, const uint8_t* of_pair, int32_t pairs, int32_t axes, int64_t stride, void* stream_) {
    return guarded([&] {
        fk::Stream_<fk::ParArch::GPU_AMD> stream(stream_);
        fk::qkNormRope(*heads, fk::ropeAxes(std::vector<uint8_t>(of_pair, of_pair + pairs), axes, stride), stream);
    });
}

} // extern "C"
