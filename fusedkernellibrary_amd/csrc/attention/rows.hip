// rows.hip -- the kernels that work on whole heads of tokens: RMS norm and rotation of queries and keys, the quantising
// write into a paged cache, and the read back.
//
// All are bound by memory (a head of 128 elements is 256 bytes in and 256 or 132 out for some 20 operations per element),
// so what counts is that every access is wide, that all of a lane's rows are requested before the first is used, and
// that one launch does everything a token needs. A copy of 1 GiB runs at 5.1 TB/s here. Norm and rotation of 4099 tokens of 28 and 4
// heads of 128 (71 MB) take 15.2 us, 4.7 TB/s; of 16384 tokens of 16 and 8 heads of 64 (105 MB) 21.4 us, 4.9 TB/s. 2048 tokens'
// keys and values of 8 heads of 128 are written in 8.3 us (12.7 MB, a start and an end more than traffic), 30011 read back in
// 30.8 us (186 MB, 6.1 TB/s). One token takes 3.2 us, which is a launch and three dependent trips to memory.
#include "heads.hpp"

namespace fkattn {
namespace {

// Reads slots back, eight elements to a lane: HEADS heads of one token's keys, or four tokens of one head's values (whose
// bytes lie side by side where the slots do).
template <int LANES, int HEADS, int TYPE, int CODES>
__global__ __launch_bounds__(256) void k_read(const ReadArgs a) {
    const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES, at = lane * 8;
    const uint32_t dim = a.head_dim, heads = a.cache.kv_heads, tile = tile_of_grid();
    const bool values = blockIdx.x >= a.k_chunks;
    if (!values) {
        const uint32_t token = tile * groups + group, head0 = blockIdx.x * HEADS;
        if (token >= a.tokens || at >= dim) return;
        uint32_t page, off;
        const bool there = locate(a.cache, a.slots[token], page, off);
        uint2_t code[HEADS];
        float scale[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            code[h] = uint2_t{0, 0};
            scale[h] = 0.0f;
            if (there && head0 + h < heads) {
                const size_t row = head_row(a.cache, page, head0 + h) + off;
                code[h] = *reinterpret_cast<const uint2_t*>(a.cache.k + row * dim + at);
                scale[h] = a.cache.k_scale[row];
            }
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            if (head0 + h >= heads) break;
            float x[8];
            decode4<CODES>(code[h].x, x);
            decode4<CODES>(code[h].y, x + 4);
            uint4_t w;
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack2<TYPE>(x[2 * k] * scale[h], x[2 * k + 1] * scale[h]);
            *reinterpret_cast<uint4_t*>(a.k.data + token * a.k.token_stride + (head0 + h) * a.k.head_stride + at * 2) = w;
        }
    } else if constexpr (HEADS == 1) {
        // few tokens: each by itself
        const uint32_t token = tile * groups + group, head = blockIdx.x - a.k_chunks;
        if (token >= a.tokens || at >= dim) return;
        uint32_t page, off;
        uint4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        float scale = 0.0f;
        if (locate(a.cache, a.slots[token], page, off)) {
            const size_t row = head_row(a.cache, page, head) + off;
            // the whole dwords are read: the other bytes are other tokens' of the same page
            const uint4_t* from = reinterpret_cast<const uint4_t*>(a.cache.v + (row - (off & 3)) * dim + size_t(at) * 4);
            lo = from[0];
            hi = from[1];
            scale = a.cache.v_scale[row];
            lo >>= 8 * (off & 3);
            hi >>= 8 * (off & 3);
        }
        uint4_t w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint4_t& from = k < 2 ? lo : hi;
            float x[4];
            decode4<CODES>((from[2 * k & 3] & 0xffu) | (from[(2 * k & 3) + 1] & 0xffu) << 8, x);
            w[k] = pack2<TYPE>(x[0] * scale, x[1] * scale);
        }
        *reinterpret_cast<uint4_t*>(a.v.data + token * a.v.token_stride + head * a.v.head_stride + at * 2) = w;
    } else {
        const uint32_t head = (blockIdx.x - a.k_chunks) * 4 + group % 4, first = tile * groups + (group / 4) * 4;
        if (head >= heads || first >= a.tokens || at >= dim) return;
        int32_t slot[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) slot[i] = first + i < a.tokens ? a.slots[first + i] : -1;
        const bool run = (slot[0] & 3) == 0 && slot[1] == slot[0] + 1 && slot[2] == slot[0] + 2 && slot[3] == slot[0] + 3;
        uint32_t page, off;
        float scale[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t code[8];                                  // of element k: the four tokens' bytes
#pragma unroll
        for (int k = 0; k < 8; ++k) code[k] = 0;
        if (run) {
            if (locate(a.cache, slot[0], page, off)) {
                const size_t row = head_row(a.cache, page, head) + off;
                const uint4_t* from = reinterpret_cast<const uint4_t*>(a.cache.v + row * dim + size_t(at) * 4);
                const uint4_t lo = from[0], hi = from[1];
                const float4_t s = *reinterpret_cast<const float4_t*>(a.cache.v_scale + row);
#pragma unroll
                for (int k = 0; k < 4; ++k) { code[k] = lo[k]; code[k + 4] = hi[k]; scale[k] = s[k]; }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!locate(a.cache, slot[i], page, off)) continue;
                const size_t row = head_row(a.cache, page, head) + off;
                scale[i] = a.cache.v_scale[row];
                // the whole dwords are read: the other bytes are other tokens' of the same page
                const uint4_t* from = reinterpret_cast<const uint4_t*>(a.cache.v + (row - (off & 3)) * dim + size_t(at) * 4);
                const uint4_t lo = from[0], hi = from[1];
#pragma unroll
                for (int k = 0; k < 8; ++k) code[k] |= (((k < 4 ? lo[k & 3] : hi[k & 3]) >> (8 * (off & 3))) & 0xffu) << (8 * i);
            }
        }
        float x[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) decode4<CODES>(code[k], x[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (first + i >= a.tokens) break;
            uint4_t w;
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack2<TYPE>(x[2 * k][i] * scale[i], x[2 * k + 1][i] * scale[i]);
            *reinterpret_cast<uint4_t*>(a.v.data + (first + i) * a.v.token_stride + head * a.v.head_stride + at * 2) = w;
        }
    }
}

template <int LANES, int HEADS, int TYPE, int CODES> int start_read(ReadArgs a, uint32_t threads, void* stream, Launched& info) {
    a.k_chunks = ceil_div(a.cache.kv_heads, HEADS);
    const uint32_t tiles = ceil_div(a.tokens, threads / LANES);
    const dim3 grid(a.k_chunks + (HEADS == 1 ? a.cache.kv_heads : ceil_div(a.cache.kv_heads, 4)), tiles < kTilesY ? tiles : kTilesY, ceil_div(tiles, kTilesY));
    info = {"kv_read", {grid.x, grid.y, grid.z}, {threads, 1, 1}, 0};
    return launch(k_read<LANES, HEADS, TYPE, CODES>, grid, dim3(threads), stream, a);
}
template <int LANES, int TYPE, int CODES> int start_read(const ReadArgs& a, void* stream, Launched& info) {
    if (uint64_t(a.tokens) * a.cache.kv_heads <= kFewRows) return start_read<LANES, 1, TYPE, CODES>(a, smallest_group(LANES), stream, info);
    return start_read<LANES, kManyRead, TYPE, CODES>(a, 256, stream, info);
}
template <int LANES, int TYPE> int start_read(const ReadArgs& a, void* stream, Launched& info) {
    if (a.cache.codes == FKLHIP_CODES_INT8) return start_read<LANES, TYPE, FKLHIP_CODES_INT8>(a, stream, info);
    return start_read<LANES, TYPE, FKLHIP_CODES_E4M3>(a, stream, info);
}

} // namespace

int launch_heads(const HeadArgs& a, int type, bool to_cache, void* stream, Launched& info) { return start_heads_of_any_size<false>(a, type, to_cache, stream, info); }

int launch_read(const ReadArgs& a, int type, void* stream, Launched& info) {
    const bool bf16 = type == FKLHIP_BF16;
    if (a.head_dim <= 64) return bf16 ? start_read<8, FKLHIP_BF16>(a, stream, info) : start_read<8, FKLHIP_F16>(a, stream, info);
    if (a.head_dim <= 128) return bf16 ? start_read<16, FKLHIP_BF16>(a, stream, info) : start_read<16, FKLHIP_F16>(a, stream, info);
    return bf16 ? start_read<32, FKLHIP_BF16>(a, stream, info) : start_read<32, FKLHIP_F16>(a, stream, info);
}

} // namespace fkattn
