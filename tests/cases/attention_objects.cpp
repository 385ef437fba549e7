// attention_objects.cpp -- the objects of the C++ host API for attention (algorithms/attention/attention.h) behind plain functions:
// what a TreeAttention does with its workspace. Compiled by g++ without HIP headers.
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

} // extern "C"
