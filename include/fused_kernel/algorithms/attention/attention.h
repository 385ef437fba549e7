// Attention over a quantised, paged key-value cache: the operators of include/fklhip.h with the host API's streams, memory and
// errors. Interface counterpart: FK/algorithms/attention/ (attention, split decoding, int8 and fp8 cache reads), whose kernels are
// called beside executeOperations too.
//
// A step of a server, for the new or drafted tokens of some sequences:
//   fk::KvCache cache(pages, kvHeads, pageTokens, headDim, fk::CacheCodes::INT8);
//   fk::qkvToCache(heads, cache, stream);            // norm, rotation, quantising write: one launch
//   fk::TreeAttention attend;                        // keeps its workspace
//   attend(call, cache, stream);
// and what is around it: fk::stepTables before, fk::VerifyDrafts and fk::kvKeep behind.
#ifndef FK_AMD_ATTENTION_H
#define FK_AMD_ATTENTION_H

#include <fused_kernel/core/execution_model/stream.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace fk {

enum class CacheCodes : int32_t { INT8 = FKLHIP_CODES_INT8, E4M3 = FKLHIP_CODES_E4M3 };
enum class RowType : int32_t { BF16 = FKLHIP_BF16, F16 = FKLHIP_F16 };

namespace attention_detail {

// An argument that does not fit is std::invalid_argument with what is wrong with it, everything else as everywhere (gpuErrchk).
inline void check(const int code, const char* file, const int line) {
    if (code == FKLHIP_EINVAL) {
        const char* text = "";
        fklhip_argument_error(&text);
        throw std::invalid_argument(text);
    }
    gpuAssert(code, file, line);
}
#define FK_ATTENTION_CHECK(expr) ::fk::attention_detail::check((expr), __FILE__, __LINE__)

// Device memory of 64-bit size, freed with its owner.
class DeviceMemory {
    void* m_data{nullptr};
    size_t m_bytes{0};
public:
    DeviceMemory() = default;
    explicit DeviceMemory(const size_t bytes) : m_bytes(bytes) { if (bytes) gpuErrchk(fklhip_malloc(&m_data, bytes)); }
    DeviceMemory(DeviceMemory&& other) noexcept : m_data(std::exchange(other.m_data, nullptr)), m_bytes(std::exchange(other.m_bytes, 0)) {}
    DeviceMemory& operator=(DeviceMemory&& other) noexcept {
        std::swap(m_data, other.m_data);
        std::swap(m_bytes, other.m_bytes);
        return *this;
    }
    DeviceMemory(const DeviceMemory&) = delete;
    DeviceMemory& operator=(const DeviceMemory&) = delete;
    ~DeviceMemory() { if (m_data) fklhip_free(m_data); }
    void* data() const { return m_data; }
    size_t bytes() const { return m_bytes; }
};

// A workspace that grows. Those it has grown out of live as long as it does, for graphs that name them.
class Workspace {
    std::vector<DeviceMemory> m_memory;                        // the last is the one in use
public:
    size_t bytes() const { return m_memory.empty() ? 0 : m_memory.back().bytes(); }
    void* data() const { return m_memory.empty() ? nullptr : m_memory.back().data(); }
    void reserve(const uint64_t need) {
        if (need > bytes()) m_memory.emplace_back(size_t(need));
    }
    void reserve(const uint64_t need, Stream_<ParArch::GPU_AMD>& stream, const char* of) {
        if (need <= bytes()) return;
        int capturing = 0;
        gpuErrchk(fklhip_stream_is_capturing(stream.getNativeStream(), &capturing));
        if (capturing) throw std::logic_error(std::string(of) + ": a call that is captured needs its workspace beforehand (reserve)");
        reserve(need);
    }
};

} // namespace attention_detail

// Rows [token][head][element] that lie tight, `heads` of them from `firstHead` on out of `headsInRow` (packed q, k and v rows, say).
inline fklhip_rows headRows(void* data, const int32_t headsInRow, const int32_t headDim, const int32_t firstHead = 0) {
    return {static_cast<char*>(data) + 2 * int64_t(firstHead) * headDim, int64_t(headsInRow) * headDim, headDim};
}

// A cache that owns its pages (see fklhip_kv_cache for the layout). Not copied, only moved: one that was moved from has no pages,
// and calls refuse it.
class KvCache {
    attention_detail::DeviceMemory m_k, m_v, m_kScale, m_vScale;
    fklhip_kv_cache m_cache{};
public:
    KvCache(const int64_t pages, const int32_t kvHeads, const int32_t pageTokens, const int32_t headDim, const CacheCodes codes) {
        if (pages < 1 || kvHeads < 1 || pageTokens < 1 || headDim < 1) throw std::invalid_argument("a cache has pages, heads, tokens and elements");
        const size_t tokens = size_t(pages) * size_t(kvHeads) * size_t(pageTokens);
        m_k = attention_detail::DeviceMemory(tokens * size_t(headDim));
        m_v = attention_detail::DeviceMemory(tokens * size_t(headDim));
        m_kScale = attention_detail::DeviceMemory(tokens * sizeof(float));
        m_vScale = attention_detail::DeviceMemory(tokens * sizeof(float));
        m_cache = {m_k.data(), m_v.data(), static_cast<float*>(m_kScale.data()), static_cast<float*>(m_vScale.data()), pages, kvHeads, pageTokens, headDim, static_cast<int32_t>(codes)};
    }
    KvCache(KvCache&& other) noexcept
        : m_k(std::move(other.m_k)), m_v(std::move(other.m_v)), m_kScale(std::move(other.m_kScale)), m_vScale(std::move(other.m_vScale)),
          m_cache(std::exchange(other.m_cache, {})) {}
    KvCache& operator=(KvCache&& other) noexcept {
        m_k = std::move(other.m_k);                            // (these change places, so the description does too)
        m_v = std::move(other.m_v);
        m_kScale = std::move(other.m_kScale);
        m_vScale = std::move(other.m_vScale);
        std::swap(m_cache, other.m_cache);
        return *this;
    }
    const fklhip_kv_cache& get() const { return m_cache; }
    operator const fklhip_kv_cache&() const { return m_cache; }
};

inline void qkNormRope(const fklhip_heads& heads, Stream_<ParArch::GPU_AMD>& stream) { FK_ATTENTION_CHECK(fklhip_qk_norm_rope(&heads, stream.getNativeStream())); }

inline void qkvToCache(const fklhip_heads& heads, const fklhip_kv_cache& cache, Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_qkv_to_cache(&heads, &cache, stream.getNativeStream()));
}

// The same with the positions of several axes, pair i turning by those of axis ofPair[i] (fklhip_axes).
inline fklhip_axes ropeAxes(const std::vector<uint8_t>& ofPair, const int32_t count, const int64_t stride) {
    fklhip_axes axes{stride, count, {}};
    if (ofPair.size() > sizeof axes.of_pair) throw std::invalid_argument("a head has up to 128 pairs");
    std::copy(ofPair.begin(), ofPair.end(), axes.of_pair);
    return axes;
}

inline void qkNormRope(const fklhip_heads& heads, const fklhip_axes& axes, Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_qk_norm_rope_axes(&heads, &axes, stream.getNativeStream()));
}

inline void qkvToCache(const fklhip_heads& heads, const fklhip_axes& axes, const fklhip_kv_cache& cache, Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_qkv_to_cache_axes(&heads, &axes, &cache, stream.getNativeStream()));
}

inline void kvWrite(const fklhip_kv_cache& cache, const fklhip_rows& k, const fklhip_rows& v, const int32_t* slots, const int64_t tokens, const RowType type,
                    Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_kv_write(&cache, &k, &v, slots, tokens, static_cast<int>(type), stream.getNativeStream()));
}

inline void kvRead(const fklhip_kv_cache& cache, const int32_t* slots, const int64_t tokens, const fklhip_rows& k, const fklhip_rows& v, const RowType type,
                   Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_kv_read(&cache, slots, tokens, &k, &v, static_cast<int>(type), stream.getNativeStream()));
}

// Attention with a workspace that grows to what the calls so far have needed. One object serves one stream at a time: the calls
// on a stream follow each other and may share it, calls (and replays of graphs) on two streams at once may not.
//
// Calls may be captured into a graph, which then names the workspace: the object has to live as long as its graphs. It frees
// none before its own end, so a later call that needs a larger one takes nothing from them (workspaces are of a few sizes, each
// larger than the one before). Nothing can be allocated while a graph is captured: a call that would have to is refused with
// std::logic_error, and reserve() is what comes before it.
class TreeAttention {
    attention_detail::Workspace m_workspace;

    static uint64_t needed(const fklhip_attention& call, const fklhip_kv_cache& cache) {
        uint64_t bytes = 0;
        FK_ATTENTION_CHECK(fklhip_tree_attention_workspace(&call, &cache, &bytes));
        return bytes;
    }
    void prepare(fklhip_attention& call, const fklhip_kv_cache& cache, Stream_<ParArch::GPU_AMD>& stream) {
        m_workspace.reserve(needed(call, cache), stream, "TreeAttention");
        call.workspace = m_workspace.data();
        call.workspace_bytes = m_workspace.bytes();
    }
public:
    // Makes the workspace large enough for calls of these sizes (its pointers are not looked at).
    void reserve(const fklhip_attention& call, const fklhip_kv_cache& cache) { m_workspace.reserve(needed(call, cache)); }
    void operator()(fklhip_attention call, const fklhip_kv_cache& cache, Stream_<ParArch::GPU_AMD>& stream) {
        prepare(call, cache, stream);
        FK_ATTENTION_CHECK(fklhip_tree_attention(&call, &cache, stream.getNativeStream()));
    }
    // With scores of another shape, or rows that see other keys (fklhip_scores).
    void operator()(fklhip_attention call, const fklhip_scores& scores, const fklhip_kv_cache& cache, Stream_<ParArch::GPU_AMD>& stream) {
        prepare(call, cache, stream);
        FK_ATTENTION_CHECK(fklhip_shaped_attention(&call, &scores, &cache, stream.getNativeStream()));
    }
};

// The tables of a step from its requests' lengths.
inline void stepTables(const fklhip_tables& tables, Stream_<ParArch::GPU_AMD>& stream) { FK_ATTENTION_CHECK(fklhip_step_tables(&tables, stream.getNativeStream())); }

// Drafted tokens against the target's probabilities, with a workspace for which all that TreeAttention says holds.
class VerifyDrafts {
    attention_detail::Workspace m_workspace;

    static uint64_t needed(const fklhip_drafts& drafts) {
        uint64_t bytes = 0;
        FK_ATTENTION_CHECK(fklhip_verify_drafts_workspace(&drafts, &bytes));
        return bytes;
    }
public:
    void reserve(const fklhip_drafts& drafts) { m_workspace.reserve(needed(drafts)); }
    void operator()(fklhip_drafts drafts, Stream_<ParArch::GPU_AMD>& stream) {
        m_workspace.reserve(needed(drafts), stream, "VerifyDrafts");
        drafts.workspace = m_workspace.data();
        drafts.workspace_bytes = m_workspace.bytes();
        FK_ATTENTION_CHECK(fklhip_verify_drafts(&drafts, stream.getNativeStream()));
    }
};

// The cache rows of accepted tokens, moved to where their sequences go on, in all layers' caches. pageTable is [batch][entries],
// path [batch][maxNew].
inline void kvKeep(const std::vector<fklhip_kv_cache>& caches, const int32_t* pageTable, const int64_t entries, const int32_t* context, const int32_t* path, const int32_t* count, const int32_t batch,
                   const int32_t maxNew, Stream_<ParArch::GPU_AMD>& stream) {
    FK_ATTENTION_CHECK(fklhip_kv_keep(caches.data(), static_cast<int32_t>(caches.size()), pageTable, entries, context, path, count, batch, maxNew, stream.getNativeStream()));
}

#undef FK_ATTENTION_CHECK

} // namespace fk
#endif
