// attention_objects.cpp -- the objects of the C++ host API for attention (algorithms/attention/attention.h) behind plain functions:
// what a TreeAttention does with its workspace, and a moved cache with its pages. Compiled by g++ without HIP headers.
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
} // namespace

extern "C" {

const char* attention_objects_error() { return g_error; }

void* attend_open() { return new fk::TreeAttention; }
void attend_close(void* attend) { delete static_cast<fk::TreeAttention*>(attend); }
int attend_reserve(void* attend, const fklhip_attention* call, const fklhip_kv_cache* cache) {
    return guarded([&] { static_cast<fk::TreeAttention*>(attend)->reserve(*call, *cache); });
}
int attend_run(void* attend, const fklhip_attention* call, const fklhip_kv_cache* cache, void* stream_) {
    return guarded([&] {
        fk::Stream_<fk::ParArch::GPU_AMD> stream(stream_);
        (*static_cast<fk::TreeAttention*>(attend))(*call, *cache, stream);
    });
}

// What a cache's descriptions are after it was moved to another: made from it (moves[0] of the old, moves[1] of the new one), and
// assigned to one that had pages of its own (moves[2] of the one it came from, moves[3]); `made` is what they were of before.
int cache_moves(fklhip_kv_cache* made, fklhip_kv_cache* moves) {
    return guarded([&] {
        fk::KvCache first(2, 1, 16, 64, fk::CacheCodes::INT8);
        made[0] = first.get();
        fk::KvCache second(std::move(first));
        moves[0] = first.get();
        moves[1] = second.get();
        fk::KvCache third(3, 2, 32, 128, fk::CacheCodes::E4M3);
        made[1] = third.get();
        third = std::move(second);
        moves[2] = second.get();
        moves[3] = third.get();
    });
}

} // extern "C"
