// step_tables.hip -- the tables of a server's step from its requests' lengths: where each sequence's rows begin, which pages it
// takes, the slot and the position of each new token and, of drafted trees, what it sees.
//
// A wave takes a request: it adds up the rows and pages of the requests in front of it (all of a workgroup's threads together), then
// its lanes take a token each, 64 at a time. A token of a tree sees its ancestors: within 64 tokens by paths of 1, 2, 4 .. steps,
// which the lanes hand each other, and beyond them what the first ancestor in front of the 64 sees, whose row is complete by then.
// The batch's last wave takes what is behind the last request's rows. Bound by latency: a launch and three dependent trips to memory:
// 2.8 us for 16 requests of a token each, 4.1 for 200 trees of up to 61 tokens, where a launch that does nothing takes 2.3.
#include <algorithm>

#include "attention_device.hpp"
#include "step_common.hpp"

namespace fkattn {
namespace {

constexpr uint32_t kWaves = 4, kTileTokens = 1024;           // tokens of a prompt to a wave

__device__ __forceinline__ uint32_t sum_wave(uint32_t v) {
    v = reduce_lanes<32>(v, [](uint32_t a, uint32_t b) { return a + b; });
    return v + uint32_t(__shfl_xor(int(v), 32));
}

// A request held inside what the host was told: its new tokens, its pages and how many more it takes.
struct Request { uint32_t fresh, context, held, need; };
__device__ __forceinline__ Request request_at(const TablesArgs& a, uint32_t b) {
    const int32_t n = a.fresh[b], c = a.context[b], h = a.held[b];
    Request r;
    r.fresh = n < 0 ? 0u : min(uint32_t(n), a.max_new);
    r.context = c < 0 ? 0u : min(uint32_t(c), 1u << 30);
    r.held = h < 0 ? 0u : min(uint32_t(h), a.width);
    const uint32_t pages = min((r.context + r.fresh + (1u << a.page_log) - 1) >> a.page_log, a.width);
    r.need = r.fresh && pages > r.held ? pages - r.held : 0u;
    return r;
}

// What a token's place in a sequence is as a slot of the cache; `ahead`: pages that go to requests in front.
__device__ __forceinline__ int32_t slot_of(const TablesArgs& a, const Request& r, uint32_t b, uint32_t ahead, uint32_t free_now, uint32_t at) {
    const uint32_t entry = at >> a.page_log, off = at & ((1u << a.page_log) - 1u);
    int32_t page = -1;
    if (entry < r.held) {
        page = a.page_table[int64_t(b) * a.page_table_stride + entry];
    } else if (entry < r.held + r.need) {
        const uint32_t nth = ahead + entry - r.held;
        if (nth < free_now) page = a.free_pages[free_now - 1 - nth];
    }
    return page < 0 || page > int32_t(0x7fffffffu >> a.page_log) ? -1 : int32_t(uint32_t(page) << a.page_log | off);
}

template <bool TREES> __global__ __launch_bounds__(kWaves * 64) void k_step_tables(const TablesArgs a) {
    __shared__ uint32_t sums[2][kWaves];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = blockIdx.x * kWaves, b = b0 + wave;
    // rows and pages of the requests in front of the workgroup's, then of those of its waves in front
    uint32_t rows = 0, pages = 0;
    for (uint32_t i = threadIdx.x; i < b0; i += kWaves * 64) {
        const Request r = request_at(a, i);
        rows += r.fresh;
        pages += r.need;
    }
    rows = sum_wave(rows);
    pages = sum_wave(pages);
    if (lane == 0) {
        sums[0][wave] = rows;
        sums[1][wave] = pages;
    }
    __syncthreads();
    rows = pages = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        rows += sums[0][w];
        pages += sums[1][w];
    }
    for (uint32_t i = b0; i < min(b, a.batch); ++i) {
        const Request r = request_at(a, i);
        rows += r.fresh;
        pages += r.need;
    }
    if (b > a.batch) return;
    const int32_t there = a.available[0];
    const uint32_t free_now = there < 0 ? 0u : min(uint32_t(there), a.free_count), start = min(rows, a.tokens);
    if (blockIdx.y == 0 && lane == 0) a.q_start[b] = int32_t(start);
    if (b == a.batch) {
        // what is behind the last request
        if (blockIdx.y == 0 && lane == 0) a.left[0] = int32_t(free_now - pages);
        for (uint32_t row = start + blockIdx.y * 64 + lane; row < a.tokens; row += gridDim.y * 64) {
            a.slots[row] = -1;
            a.positions[row] = 0;
            if constexpr (TREES)
                for (uint32_t w = 0; w < a.mask_words; ++w) a.mask[size_t(row) * a.mask_words + w] = 0;
        }
        return;
    }
    const Request r = request_at(a, b);
    if (blockIdx.y == 0) {
        const uint32_t given = min(r.need, free_now - min(pages, free_now));
        for (uint32_t i = lane; i < given; i += 64) a.page_table[int64_t(b) * a.page_table_stride + r.held + i] = a.free_pages[free_now - 1 - (pages + i)];
        if (lane == 0) a.held_out[b] = int32_t(r.held + given);
    }
    const uint32_t count = min(r.fresh, a.tokens - start);
    if constexpr (!TREES) {
        for (uint32_t t0 = blockIdx.y * kTileTokens; t0 < count; t0 += gridDim.y * kTileTokens) {
            const uint32_t end = min(count, t0 + kTileTokens);
            for (uint32_t t = t0 + lane; t < end; t += 64) {
                a.slots[start + t] = slot_of(a, r, b, pages, free_now, r.context + t);
                a.positions[start + t] = int32_t(r.context + t);
            }
        }
    } else {
        for (uint32_t t0 = 0; t0 < count; t0 += 64) {
            const uint32_t t = t0 + lane;
            const bool live = t < count;
            const int32_t p = live ? a.parents[start + t] : -1;
            // the token's nearest ancestors within these 64, the next one behind them, and how many they are
            uint64_t seen = uint64_t(lane & 32 ? 1u << (lane & 31) : 0u) << 32 | (lane & 32 ? 0u : 1u << lane);
            int32_t next = p >= 0 && uint32_t(p) < t ? p : -1;
            uint32_t depth = next >= 0 ? 1 : 0;
#pragma unroll 1
            for (int i = 0; i < 6; ++i) {
                const bool inside = next >= int32_t(t0);
                if (!__any(inside)) break;
                const int from = inside ? next - int32_t(t0) : int(lane);
                const uint32_t lo = uint32_t(__shfl(int(uint32_t(seen)), from)), hi = uint32_t(__shfl(int(uint32_t(seen >> 32)), from)), d = uint32_t(__shfl(int(depth), from));
                const int32_t n = __shfl(next, from);
                if (inside) {
                    seen |= uint64_t(hi) << 32 | lo;
                    depth += d;
                    next = n;
                }
            }
            if (!live) continue;
            uint64_t* const words = a.mask + size_t(start + t) * a.mask_words;
            if (next >= 0) depth += uint32_t(a.positions[start + next]) - r.context;
            for (uint32_t w = 0; w < a.mask_words; ++w) {
                uint64_t bits = 0;
                if (w < t0 / 64) bits = next >= 0 ? a.mask[size_t(start + next) * a.mask_words + w] : 0;
                else if (w == t0 / 64) bits = seen;
                words[w] = bits;
            }
            a.slots[start + t] = slot_of(a, r, b, pages, free_now, r.context + t);
            a.positions[start + t] = int32_t(r.context + depth);
            __threadfence_block();                                // (the next 64 read these rows)
        }
    }
}

} // namespace

int launch_step_tables(const TablesArgs& a, void* stream, Launched& info) {
    const bool trees = a.parents != nullptr;
    const uint32_t most = std::min(std::min(a.max_new, a.tokens), 65535 * kTileTokens),
                   tiles = trees || most == 0 ? 1 : (most + kTileTokens - 1) / kTileTokens;
    const dim3 grid(a.batch / kWaves + 1, tiles, 1), block(kWaves * 64);
    info = {"step_tables", {grid.x, grid.y, 1}, {block.x, 1, 1}, 0};
    return trees ? launch(k_step_tables<true>, grid, block, stream, a) : launch(k_step_tables<false>, grid, block, stream, a);
}

} // namespace fkattn
