// rows.hip -- the kernels that work on whole heads of tokens: RMS norm and rotation of queries and keys, the quantising
// write into a paged cache, and the read back.
//
// All are bound by memory (a head of 128 elements is 256 bytes in and 256 or 132 out for some 20 operations per element),
// so what counts is that every access is wide, that all of a lane's rows are requested before the first is used, and
// that one launch does everything a token needs. A copy of 1 GiB runs at 5.1 TB/s here. Norm and rotation of 4099 tokens of 28 and 4
// heads of 128 (71 MB) take 15.2 us, 4.7 TB/s; of 16384 tokens of 16 and 8 heads of 64 (105 MB) 21.4 us, 4.9 TB/s. 2048 tokens'
// keys and values of 8 heads of 128 are written in 8.3 us (12.7 MB, a start and an end more than traffic), 30011 read back in
// 30.8 us (186 MB, 6.1 TB/s). One token takes 3.2 us, which is a launch and three dependent trips to memory.
#include "attention_device.hpp"

namespace fkattn {
namespace {

// A group of lanes takes a head, eight elements to a lane. Rotation pairs elements half of the rotated part apart; so that
// both of a pair are in one lane, a lane holds two runs of four elements: i.. and i + rot / 2.. where pairs are halves,
// eight neighbours where pairs are neighbours or nothing is rotated.
struct LanePlace {
    uint32_t at[2];      // first elements of the lane's two runs
    uint32_t turn;       // first of its four entries in the tables
    bool live, rotated;
};
__device__ __forceinline__ LanePlace place_of(uint32_t lane, uint32_t dim, uint32_t rot, int pairs) {
    LanePlace p;
    const uint32_t i = lane * 4;                                 // of dim / 2 pairs, the lane has four
    p.live = i < dim / 2;
    p.rotated = i < rot / 2;
    p.turn = i;
    const bool halves = p.rotated && !pairs;
    p.at[0] = halves ? i : 2 * i;
    p.at[1] = halves ? i + rot / 2 : 2 * i + 4;
    return p;
}

template <int TYPE> __device__ __forceinline__ void load4(const char* row, uint32_t at, float* x) {
    const uint2_t w = *reinterpret_cast<const uint2_t*>(row + at * 2);
    unpack2<TYPE>(w.x, x[0], x[1]);
    unpack2<TYPE>(w.y, x[2], x[3]);
}
template <int TYPE> __device__ __forceinline__ void store4(char* row, uint32_t at, const float* x) {
    uint2_t w;
    w.x = pack2<TYPE>(x[0], x[1]);
    w.y = pack2<TYPE>(x[2], x[3]);
    *reinterpret_cast<uint2_t*>(row + at * 2) = w;
}

// Scale of a row from the bits of its largest magnitude: one that is infinite or NaN makes the row NaN.
template <int CODES> __device__ __forceinline__ float scale_of(uint32_t bits) {
    const float top = __builtin_bit_cast(float, bits);
    return bits >= 0x7f800000u ? __builtin_nanf("") : top / (CODES == FKLHIP_CODES_INT8 ? kTopInt8 : kTopE4M3);
}
// Eight values as codes: x / scale, an IEEE division, so that codes are what the definition says bit by bit.
template <int CODES> __device__ __forceinline__ void encode8(const float* x, float scale, uint32_t* w) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = scale > 0.0f ? x[i] / scale : 0.0f;
    w[0] = encode4<CODES>(y);
    w[1] = encode4<CODES>(y + 4);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// Where a slot is in the cache: its page and its place there; false for a slot outside.
__device__ __forceinline__ bool locate(const Cache& c, int32_t slot, uint32_t& page, uint32_t& off) {
    page = uint32_t(slot) >> c.page_log;
    off = uint32_t(slot) & ((1u << c.page_log) - 1u);
    return slot >= 0 && page < c.pages;
}
__device__ __forceinline__ size_t head_row(const Cache& c, uint32_t page, uint32_t head) {
    return (size_t(page) * c.kv_heads + head) << c.page_log;     // tokens in front of the head's part of the page
}

// Tiles of tokens go along y, and along z where there are more than a grid holds.
constexpr uint32_t kTilesY = 32768;
__device__ __forceinline__ uint32_t tile_of_grid() { return blockIdx.z * kTilesY + blockIdx.y; }

// One token's values of a head, byte by byte.
template <int LANES, int TYPE, int CODES> __device__ __forceinline__ void write_value(const HeadArgs& a, uint32_t token, uint32_t head, uint32_t lane) {
    const uint32_t at = lane * 8, dim = a.head_dim;
    uint4_t raw = {0, 0, 0, 0};
    if (at < dim) raw = *reinterpret_cast<const uint4_t*>(a.v.data + token * a.v.token_stride + head * a.v.head_stride + at * 2);
    uint32_t page, off;
    const bool stored = locate(a.cache, a.slots[token], page, off);
    float x[8];
    uint32_t top = 0, code[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack2<TYPE>(raw[k], x[2 * k], x[2 * k + 1]);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, magnitude(x[k]));
    const float scale = scale_of<CODES>(max_lanes<LANES>(top));
    encode8<CODES>(x, scale, code);
    if (!stored) return;
    const size_t row = head_row(a.cache, page, head) + off;
    if (lane == 0) a.cache.v_scale[row] = scale;
    if (at < dim) {
        char* to = a.cache.v + (row - (off & 3)) * dim + size_t(at) * 4 + (off & 3);
#pragma unroll
        for (int k = 0; k < 8; ++k) to[k * 4] = char(code[k / 4] >> (8 * (k % 4)));
    }
}

// LANES to a head of up to 8 * LANES elements, HEADS heads of one token to a group of lanes.
template <int LANES, int HEADS, int TYPE, int CODES, bool TO_CACHE>
__global__ __launch_bounds__(256) void k_heads(const HeadArgs a) {
    const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES;
    const uint32_t dim = a.head_dim, tile = tile_of_grid();
    if (TO_CACHE && blockIdx.x >= a.q_chunks + a.k_chunks) {
        if constexpr (HEADS == 1) {
            // few tokens: each by itself, as few are in neighbouring slots and four at a time take longer than one (32 of 8 heads: 4.8 us, and 3.0 so)
            const uint32_t token = tile * groups + group;
            if (token < a.tokens) write_value<LANES, TYPE, CODES>(a, token, blockIdx.x - a.q_chunks - a.k_chunks, lane);
            return;
        }
        // Values: four tokens in four neighbouring slots have their bytes side by side in the cache. A group looks after four tokens of a
        // head, and stores four at once that begin at one of them and at a slot that is a multiple of four, its own or the next group's;
        // tokens that are of no such four, byte by byte. (A chunk of a prompt begins at any slot: with own ones alone at once, 2048
        // tokens of 8 heads of 128 that began at slot 3 took 17 us, and take 8.6.)
        const uint32_t head = (blockIdx.x - a.q_chunks - a.k_chunks) * 4 + group % 4, at = lane * 8, first = tile * groups + (group / 4) * 4;
        if (head >= a.kv_heads || first >= a.tokens) return;
        const char* from = a.v.data + head * a.v.head_stride + at * 2;
        uint4_t raw[7];                                        // of tokens first ..
        int32_t slot[10];                                      // of tokens first - 3 ..; none there: -1
#pragma unroll
        for (int i = 0; i < 10; ++i) slot[i] = first + i >= 3 && first + i < a.tokens + 3 ? a.slots[first + i - 3] : -1;
        const auto load = [&](int i) {
            raw[i] = uint4_t{0, 0, 0, 0};
            if (first + i < a.tokens && at < dim) raw[i] = *reinterpret_cast<const uint4_t*>(from + (first + i) * a.v.token_stride);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) load(i);
        uint32_t page, off;
        // the four that begin at one of the group's tokens: there is one at most
        int start = -1;
        uint32_t done = 0;                                     // a bit for each of the group's tokens that is of a four
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            const int32_t s = slot[i];
            const bool four = s >= 0 && (s & 3) == 0 && slot[i + 1] == s + 1 && slot[i + 2] == s + 2 && slot[i + 3] == s + 3;
            if (four) done |= (15u << i) >> 3;
            if (four && i >= 3) start = i - 3;
        }
        float x[8], scale[4];
        uint32_t code[4][2];
        const auto encode = [&](uint4_t r, float& s, uint32_t* c) {
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) unpack2<TYPE>(r[k], x[2 * k], x[2 * k + 1]);
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, magnitude(x[k]));
            s = scale_of<CODES>(max_lanes<LANES>(top));
            encode8<CODES>(x, s, c);
        };
        if (start >= 0) {
#pragma unroll
            for (int i = 4; i < 7; ++i)
                if (i - 4 < start) load(i);
                else raw[i] = uint4_t{0, 0, 0, 0};
            int32_t slot0 = slot[3];
            uint4_t four[4] = {raw[0], raw[1], raw[2], raw[3]};
#pragma unroll
            for (int k = 1; k < 4; ++k)
                if (start == k) {
                    slot0 = slot[3 + k];
#pragma unroll
                    for (int i = 0; i < 4; ++i) four[i] = raw[k + i];
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) encode(four[i], scale[i], code[i]);
            if (locate(a.cache, slot0, page, off)) {
                const size_t row = head_row(a.cache, page, head) + off;
                if (lane == 0) *reinterpret_cast<float4_t*>(a.cache.v_scale + row) = float4_t{scale[0], scale[1], scale[2], scale[3]};
                if (at < dim) {
                    // 4 x 8 bytes turned: element by element, four tokens each
                    uint4_t out[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t lo01 = __builtin_amdgcn_perm(code[1][h], code[0][h], 0x05010400u), hi01 = __builtin_amdgcn_perm(code[1][h], code[0][h], 0x07030602u);
                        const uint32_t lo23 = __builtin_amdgcn_perm(code[3][h], code[2][h], 0x05010400u), hi23 = __builtin_amdgcn_perm(code[3][h], code[2][h], 0x07030602u);
                        out[h] = uint4_t{__builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
                                         __builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
                    }
                    uint4_t* to = reinterpret_cast<uint4_t*>(a.cache.v + row * dim + size_t(at) * 4);
                    to[0] = out[0];
                    to[1] = out[1];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (done >> i & 1 || !locate(a.cache, slot[3 + i], page, off)) continue;
            encode(raw[i], scale[0], code[0]);
            const size_t row = head_row(a.cache, page, head) + off;
            if (lane == 0) a.cache.v_scale[row] = scale[0];
            if (at < dim) {
                char* to = a.cache.v + (row - (off & 3)) * dim + size_t(at) * 4 + (off & 3);
#pragma unroll
                for (int k = 0; k < 8; ++k) to[k * 4] = char(code[0][k / 4] >> (8 * (k % 4)));
            }
        }
        return;
    }
    const bool is_q = blockIdx.x < a.q_chunks;
    const uint32_t head0 = (is_q ? blockIdx.x : blockIdx.x - a.q_chunks) * HEADS, heads = is_q ? a.q_heads : a.kv_heads;
    const Rows in = is_q ? a.q : a.k, out = is_q ? a.q_out : a.k_out;
    const char* weights = static_cast<const char*>(is_q ? a.q_weight : a.k_weight);
    const LanePlace p = place_of(lane, dim, a.rot_dim, a.pairs);
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = 1.0f;
    if (weights && p.live) { load4<TYPE>(weights, p.at[0], w); load4<TYPE>(weights, p.at[1], w + 4); }
    const uint32_t token = tile * groups + group;
    if (token >= a.tokens) return;
    float x[HEADS][8];
    const char* row = in.data + token * in.token_stride;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[h][k] = 0.0f;
        if (p.live && head0 + h < heads) {
            load4<TYPE>(row + (head0 + h) * in.head_stride, p.at[0], x[h]);
            load4<TYPE>(row + (head0 + h) * in.head_stride, p.at[1], x[h] + 4);
        }
    }
    float4_t cosine = {1.0f, 1.0f, 1.0f, 1.0f}, sine = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.rotated) {
        const uint32_t position = uint32_t(a.positions[token]);
        if (position < a.table_rows) {
            const size_t at = size_t(position) * (a.rot_dim / 2) + p.turn;
            cosine = *reinterpret_cast<const float4_t*>(a.cos + at);
            sine = *reinterpret_cast<const float4_t*>(a.sin + at);
        } else {
            cosine = sine = float4_t{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        }
    }
    uint32_t page = 0, off = 0;
    bool stored = false;
    if (TO_CACHE && !is_q) stored = locate(a.cache, a.slots[token], page, off);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (head0 + h >= heads) break;
        if (weights) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(x[h][k], x[h][k], sum);
            const float r = 1.0f / __builtin_sqrtf(sum_lanes<LANES>(sum) / float(dim) + a.eps);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[h][k] = x[h][k] * r * w[k];
        }
        if (p.rotated) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // pairs are (k, k + 4) of the lane's elements as halves, (2k, 2k + 1) as neighbours
                float& u = a.pairs ? x[h][2 * k] : x[h][k];
                float& v = a.pairs ? x[h][2 * k + 1] : x[h][k + 4];
                const float s = u, t = v;
                u = s * cosine[k] - t * sine[k];
                v = t * cosine[k] + s * sine[k];
            }
        }
        if (is_q || !TO_CACHE) {
            if (p.live) {
                char* to = out.data + token * out.token_stride + (head0 + h) * out.head_stride;
                store4<TYPE>(to, p.at[0], x[h]);
                store4<TYPE>(to, p.at[1], x[h] + 4);
            }
        } else {
            uint32_t top = 0, code[2];
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, magnitude(x[h][k]));
            const float scale = scale_of<CODES>(max_lanes<LANES>(top));
            encode8<CODES>(x[h], scale, code);
            if (stored) {
                const size_t at = head_row(a.cache, page, head0 + h) + off;
                if (lane == 0) a.cache.k_scale[at] = scale;
                if (p.live) {
                    char* to = a.cache.k + at * dim;
                    *reinterpret_cast<uint32_t*>(to + p.at[0]) = code[0];
                    *reinterpret_cast<uint32_t*>(to + p.at[1]) = code[1];
                }
            }
        }
    }
}

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

uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// Few rows of keys: one head of a token to a group of lanes, so that everything runs at once (504 tokens of 28 and 4 heads of 128
// written 5.4 us, 7.0 in the form of many; 2048 tokens of 8 heads 11.1 and 8.4). Norm and rotation alone turn at about the same
// number, whatever queries there are (few, many): 500 tokens of 28 and 4 heads 4.0 and 5.3, 1000 6.1 and 6.9, 1500 7.9 and 8.3, 760 of 64
// and 8 8.4 and 9.1, 1500 of 64 and 4 12.9 and 12.5, 6000 of 8 and 1 9.5 and 9.0. Many: a group has several heads of a token, whose
// rows it asks for together and which share its cosines, sines and slot. Values of 2 and 4 heads (16384 tokens): norm and rotation
// of 40 heads of 128 71.3 and 68.8 us (one head: 86.2), of 24 of 64 20.8 and 19.7; with the write, whose quantising takes more
// registers, of 32, 8 and 8 heads of 128 82.9 and 87.9 (one: 99.4), of 16, 8 and 8 of 64 28.1 and 33.6; reading 8 heads of
// 64 10.0 and 11.2. Workgroups as small as values allow (four heads a group each) end more evenly: 28.1 us there, 28.6 with 256
// threads; only reading, which waits for nothing but a slot, has 256 (17.8 us for 8 heads of 128, and 19.9 with 64).
constexpr uint32_t kFewRows = 6144;
constexpr int kManyHeads = 4, kManyToCache = 2, kManyRead = 2;
constexpr uint32_t smallest_group(uint32_t lanes) { return lanes * 4 < 64 ? 64 : lanes * 4; }

template <int LANES, int HEADS, int TYPE, int CODES, bool TO_CACHE>
int start_heads(HeadArgs a, uint32_t threads, void* stream, Launched& info) {
    a.q_chunks = ceil_div(a.q_heads, HEADS);
    a.k_chunks = ceil_div(a.kv_heads, HEADS);
    const uint32_t tiles = ceil_div(a.tokens, threads / LANES);
    const dim3 grid(a.q_chunks + a.k_chunks + (TO_CACHE ? (HEADS == 1 ? a.kv_heads : ceil_div(a.kv_heads, 4)) : 0), tiles < kTilesY ? tiles : kTilesY, ceil_div(tiles, kTilesY));
    info = {"heads", {grid.x, grid.y, grid.z}, {threads, 1, 1}, 0};
    return launch(k_heads<LANES, HEADS, TYPE, CODES, TO_CACHE>, grid, dim3(threads), stream, a);
}
template <int LANES, int TYPE, int CODES, bool TO_CACHE> int start_heads(const HeadArgs& a, void* stream, Launched& info) {
    constexpr int kMany = TO_CACHE ? kManyToCache : kManyHeads;
    if (uint64_t(a.tokens) * a.kv_heads <= kFewRows) return start_heads<LANES, 1, TYPE, CODES, TO_CACHE>(a, smallest_group(LANES), stream, info);
    return start_heads<LANES, kMany, TYPE, CODES, TO_CACHE>(a, smallest_group(LANES), stream, info);
}
template <int LANES, int TYPE> int start_heads(const HeadArgs& a, bool to_cache, void* stream, Launched& info) {
    if (!to_cache) return start_heads<LANES, TYPE, 0, false>(a, stream, info);
    if (a.cache.codes == FKLHIP_CODES_INT8) return start_heads<LANES, TYPE, FKLHIP_CODES_INT8, true>(a, stream, info);
    return start_heads<LANES, TYPE, FKLHIP_CODES_E4M3, true>(a, stream, info);
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

int launch_heads(const HeadArgs& a, int type, bool to_cache, void* stream, Launched& info) {
    const bool bf16 = type == FKLHIP_BF16;
    if (a.head_dim <= 64) return bf16 ? start_heads<8, FKLHIP_BF16>(a, to_cache, stream, info) : start_heads<8, FKLHIP_F16>(a, to_cache, stream, info);
    if (a.head_dim <= 128) return bf16 ? start_heads<16, FKLHIP_BF16>(a, to_cache, stream, info) : start_heads<16, FKLHIP_F16>(a, to_cache, stream, info);
    return bf16 ? start_heads<32, FKLHIP_BF16>(a, to_cache, stream, info) : start_heads<32, FKLHIP_F16>(a, to_cache, stream, info);
}

int launch_read(const ReadArgs& a, int type, void* stream, Launched& info) {
    const bool bf16 = type == FKLHIP_BF16;
    if (a.head_dim <= 64) return bf16 ? start_read<8, FKLHIP_BF16>(a, stream, info) : start_read<8, FKLHIP_F16>(a, stream, info);
    if (a.head_dim <= 128) return bf16 ? start_read<16, FKLHIP_BF16>(a, stream, info) : start_read<16, FKLHIP_F16>(a, stream, info);
    return bf16 ? start_read<32, FKLHIP_BF16>(a, stream, info) : start_read<32, FKLHIP_F16>(a, stream, info);
}

} // namespace fkattn
