// keep.hip -- the cache rows of a step's accepted tokens, moved to where their sequence goes on.
//
// Accepted token i of a sequence (path[i] of its new ones, i <= path[i]) goes from place context + path[i] to context + i: codes and
// scales as they are. A wave takes a head of a sequence in a layer, kAtOnce tokens at a time in their order: it reads them all and
// then writes them, so that a row which is another's place is read before it is written over (paths ascend, so nothing
// later in the path is at a place in front). A trip to memory each for the path, the page table and the rows bounds it: 4.0 us
// for 8 sequences of a layer, 8 heads of 128 (5.0 with a wave going from token to token), 10.0 us for 48 sequences and 16 layers (12.3).
#include "attention_device.hpp"
#include "step_common.hpp"

namespace fkattn {
namespace {

constexpr uint32_t kWaves = 4, kAtOnce = 8;                   // tokens at once

struct Move { uint32_t from, to; };                           // slots; the same: nothing moves

// Slot of a place of the sequence, or -1.
__device__ __forceinline__ int64_t slot_of(const KeepArgs& a, uint32_t b, uint32_t at) {
    const uint32_t entry = at >> a.page_log;
    if (entry >= a.width) return -1;
    const int32_t page = a.page_table[int64_t(b) * a.page_table_stride + entry];
    return page < 0 || uint32_t(page) >= a.pages ? -1 : int64_t(page) << a.page_log | (at & ((1u << a.page_log) - 1u));
}

__global__ __launch_bounds__(kWaves * 64) void k_keep(const KeepArgs a) {
    const uint32_t lane = threadIdx.x & 63, head = blockIdx.x * kWaves + (threadIdx.x >> 6), b = blockIdx.y;
    if (head >= a.kv_heads) return;
    const KeepCache& c = a.caches[blockIdx.z];
    const int32_t have = a.context[b], kept = a.count[b];
    const uint32_t context = have < 0 ? 0u : min(uint32_t(have), 1u << 30), count = kept < 0 ? 0u : min(uint32_t(kept), a.max_new);
    const uint32_t dim = a.head_dim;
    for (uint32_t i0 = 1; i0 < count; i0 += kAtOnce) {
        // a lane finds a token's move
        Move m{0, 0};
        const uint32_t i = i0 + lane;
        if (lane < kAtOnce && i < count) {
            const int32_t p = a.path[size_t(b) * a.max_new + i];
            if (p > int32_t(i) && p < int32_t(a.max_new)) {
                const int64_t from = slot_of(a, b, context + uint32_t(p)), to = slot_of(a, b, context + i);
                if (from >= 0 && to >= 0) m = {uint32_t(from), uint32_t(to)};
            }
        }
        if (!__any(m.from != m.to)) continue;
        const auto row_of = [&](uint32_t slot) { return ((size_t(slot >> a.page_log) * a.kv_heads + head) << a.page_log) + (slot & ((1u << a.page_log) - 1u)); };
        // Eight lanes to a token: pieces of 8 bytes of its key, dwords of four elements of its value (a byte of each is its own), its scales.
        const uint32_t from = uint32_t(__shfl(int(m.from), int(lane / 8))), to = uint32_t(__shfl(int(m.to), int(lane / 8))), at = lane % 8;
        if (from != to) {
            const size_t source = row_of(from), place = row_of(to);
            uint2_t key[4];
            uint4_t value[8];
            float scale = 0.0f;
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n)
                if ((n * 8 + at) * 8 < dim) key[n] = *reinterpret_cast<const uint2_t*>(c.k + source * dim + (n * 8 + at) * 8);
#pragma unroll
            for (uint32_t n = 0; n < 8; ++n)
                if ((n * 8 + at) * 4 < dim) value[n] = *reinterpret_cast<const uint4_t*>(c.v + (source & ~size_t(3)) * dim + (n * 8 + at) * 16);
            if (at < 2) scale = (at ? c.v_scale : c.k_scale)[source];
            // all tokens' rows are read before one is written: the wave's accesses stay in this order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n)
                if ((n * 8 + at) * 8 < dim) *reinterpret_cast<uint2_t*>(c.k + place * dim + (n * 8 + at) * 8) = key[n];
#pragma unroll
            for (uint32_t n = 0; n < 8; ++n)
                if ((n * 8 + at) * 4 < dim) {
                    char* bytes = c.v + (place & ~size_t(3)) * dim + (n * 8 + at) * 16 + (to & 3);
#pragma unroll
                    for (int k = 0; k < 4; ++k) bytes[k * 4] = char(value[n][k] >> (8 * (from & 3)));
                }
            if (at < 2) (at ? c.v_scale : c.k_scale)[place] = scale;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

} // namespace

int launch_keep(const KeepArgs& a, uint32_t layers, void* stream, Launched& info) {
    const dim3 grid((a.kv_heads + kWaves - 1) / kWaves, a.batch, layers), block(kWaves * 64);
    info = {"kv_keep", {grid.x, grid.y, grid.z}, {block.x, 1, 1}, 0};
    return launch(k_keep, grid, block, stream, a);
}

} // namespace fkattn
