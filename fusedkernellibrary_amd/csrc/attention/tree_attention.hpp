// tree_attention.hpp -- attention of a few new tokens per sequence over a quantised, paged cache.
//
// Mathematics. For the rows r of a key head (its query heads times the sequence's new tokens) and the keys j a row sees:
//   s_rj = scale * ks_j * (q_r . kc_j),   o_r = sum_j e^(s_rj - m_r) vs_j vc_j / sum_j e^(s_rj - m_r)
// with kc, vc the cache's codes and ks, vs their scales. The codes are exact in half precision (int8: 8 bits, e4m3: 4 bits of
// 11), so the products run on the codes themselves and the scales enter as one factor per key: ks on the scores, vs on the
// weights. A query row is brought to a largest magnitude in [1, 2) by a power of two, which is exact in half precision too,
// but for elements 2^24 times smaller than the row's largest. The one rounding is that of the weights to half precision.
//
// One pass over the keys, 32 at a time, everything in registers: S^T = K Q^T comes out of the matrix unit with a query row to
// a lane column (lane % 16) and four keys to each of its four quarters (lane / 16), and O^T = V^T P^T wants its weights just
// so if the contraction runs over the keys in that order; the cache keeps four tokens' bytes of a value element side by
// side for that reason. So nothing moves between lanes, and the running maximum is per lane column.
//
// The running maximum m_r and the largest value scale t are references and not the exact maxima: weights are
// w = 2^(s - m) * vs / t, and m and t move only when a score leads m by more than 2^kLead or a value scale exceeds t. Only
// then are scores compared across lanes and the sums rescaled. 2^(s - m) stays below 2^kLead and starts at 2^kStart, so a
// weight is subnormal in half precision (2^-14) only 2^-(14 + kStart) below the largest of the first keys.
#pragma once

#include "attention_device.hpp"

namespace fkattn {

constexpr int kWaves = 4;                    // of a workgroup: they share out a chunk's keys, 32 at a time
constexpr float kStart = 6.0f, kLead = 14.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNothing = -1.0e30f;         // the reference of a row that has seen no key

template <int D> struct Shape {
    static constexpr int kChunk = D % 64 == 0 ? 64 : 32;   // elements of a row that one load of a lane's quarter row covers
    static constexpr int kLoads = D / kChunk;              // of a block of 16 keys (or values)
    static constexpr int kWords = kChunk / 16;             // dwords of such a load: 4 or 2
    static constexpr int kSteps = D / 32;                  // of the matrix unit over a row
    static constexpr int kTiles = D / 16;                  // of 16 output elements
};

template <int WORDS> struct Words { uint32_t w[WORDS]; };

template <int WORDS> __device__ __forceinline__ Words<WORDS> load_words(const char* p) {
    Words<WORDS> r;
    if constexpr (WORDS == 4) {
        const uint4_t v = *reinterpret_cast<const uint4_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = v[i];
    } else {
        const uint2_t v = *reinterpret_cast<const uint2_t*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    }
    return r;
}

// Four codes of a dword as half precision, exactly.
template <int CODES> __device__ __forceinline__ void halves4(uint32_t w, half2_t& lo, half2_t& hi) {
    if constexpr (CODES == FKLHIP_CODES_INT8) {
        // 0x6400 is 1024 in half precision, with a unit of 1: the code + 128 goes into its last byte
        const uint32_t u = w ^ 0x80808080u;
        const half2_t bias = {_Float16(1152.0f), _Float16(1152.0f)};
        lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
        hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
    } else {
        lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
}
template <int CODES> __device__ __forceinline__ half8_t halves8(uint32_t a, uint32_t b) {
    half2_t x[4];
    halves4<CODES>(a, x[0], x[1]);
    halves4<CODES>(b, x[2], x[3]);
    return half8_t{x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The larger of a lane column's four quarters (lanes l, l ^ 16, l ^ 32, l ^ 48), and their sum.
__device__ __forceinline__ float max_quarters(float v) {
    v = __builtin_fmaxf(v, __shfl_xor(v, 16));
    return __builtin_fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_quarters(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The lowest n of four bits.
__device__ __forceinline__ uint32_t lowest_bits(int32_t n) { return n >= 4 ? 15u : n <= 0 ? 0u : (1u << n) - 1u; }
// Bits u .. u + 3 of a row of a mask, where those below 0 (the context's) are set and those behind the row are not.
__device__ __forceinline__ uint32_t mask_bits(const uint64_t* row, uint32_t words, int32_t u) {
    const uint32_t below = u >= 0 ? 0u : u <= -4 ? 4u : uint32_t(-u), from = u >= 0 ? uint32_t(u) : 0u;
    const uint32_t lo_at = from >> 6, hi_at = (from + 3) >> 6, shift = from & 63u;
    const uint64_t lo = lo_at < words ? row[lo_at] : 0, hi = hi_at < words && hi_at != lo_at ? row[hi_at] : 0;
    const uint32_t bits = uint32_t(lo >> shift) | (shift ? uint32_t(hi << (64u - shift)) : 0u);
    return (lowest_bits(int32_t(below)) | bits << below) & 15u;
}

// 32 keys: codes and scales of two blocks of 16 as a lane holds them.
template <int D> struct Tile {
    using S = Shape<D>;
    Words<S::kWords> k[2][S::kLoads], v[2][S::kLoads];
    float4_t ks[2], vs[2];
};

template <int D, int CODES, int R>
__global__ __launch_bounds__(kWaves * 64, R == 1 && D <= 128 ? 2 : 1) void k_tree_attention(const AttentionArgs a) {
    using S = Shape<D>;
    constexpr int kRowFloats = D + 4;                              // of a row in LDS: 16 bytes further round the banks than the last
    __shared__ __attribute__((aligned(16))) float joined[kWaves][16 * kRowFloats];
    __shared__ float joined_m[kWaves][16], joined_l[kWaves][16], row_m[16], row_l[16];

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15, quarter = lane >> 4;
    const uint32_t b = blockIdx.z;
    const uint32_t split = divide(blockIdx.x, a.heads_magic), head = blockIdx.x - split * a.cache.kv_heads;
    if (split >= a.splits) return;                                 // (the grid's x is padded)

    const int32_t start = a.q_start[b];
    uint32_t first_token = uint32_t(start < 0 ? 0 : start);
    if (first_token > a.tokens) first_token = a.tokens;
    int32_t diff = a.q_start[b + 1] - int32_t(first_token);
    uint32_t fresh = diff < 0 ? 0 : uint32_t(diff);
    fresh = min(min(fresh, a.max_new), a.tokens - first_token);
    int32_t have = a.context[b];
    uint32_t context = have < 0 ? 0 : min(uint32_t(have), a.max_context);
    const uint32_t page_mask = (1u << a.cache.page_log) - 1u;
    const uint64_t room = uint64_t(a.page_table_stride) << a.cache.page_log;
    context = room < context ? uint32_t(room) : context;
    const uint32_t total = room < uint64_t(context) + fresh ? uint32_t(room) : context + fresh;

    const uint32_t rows = fresh * a.group, row0 = blockIdx.y * (16 * R);
    if (row0 >= rows) return;
    const uint32_t last_row = min(row0 + 16 * R, rows) - 1;
    // keys that every row of the workgroup sees, and keys that any of them can see
    const bool causal = a.mask == nullptr;
    const uint32_t all_see = causal ? min(context + divide(row0, a.group_magic) + 1, total) : context;
    const uint32_t any_sees = causal ? min(context + divide(last_row, a.group_magic) + 1, total) : total;
    const uint32_t key0 = split * a.chunk, key1 = min(key0 + a.chunk, any_sees);

    // the lane's rows: their new token, and their query elements as the scores want them
    uint32_t token[R];
    half8_t q[R][S::kSteps];
    float row_scale[R];
    float4_t o[R][S::kTiles];
    float m[R], l[R];
    float t = 0.0f, inv_t = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = row0 + r * 16 + col;
        token[r] = divide(min(row, last_row), a.group_magic);
        const uint32_t g = min(row, last_row) - token[r] * a.group;
        const char* from = a.q.data + int64_t(first_token + token[r]) * a.q.token_stride + int64_t(head * a.group + g) * a.q.head_stride;
        float x[S::kSteps * 8];
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            // the elements that the quarter's codes of this step are of: kChunk / 4 neighbours of each run of kChunk
            const uint32_t at = S::kChunk == 64 ? (s / 2) * 64 + quarter * 16 + (s % 2) * 8 : s * 32 + quarter * 8;
            const uint4_t w = *reinterpret_cast<const uint4_t*>(from + at * 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (a.type == FKLHIP_BF16) unpack2<FKLHIP_BF16>(w[k], x[s * 8 + 2 * k], x[s * 8 + 2 * k + 1]);
                else unpack2<FKLHIP_F16>(w[k], x[s * 8 + 2 * k], x[s * 8 + 2 * k + 1]);
            }
        }
#pragma unroll
        for (int k = 0; k < S::kSteps * 8; ++k) top = max(top, __builtin_bit_cast(uint32_t, x[k]) & 0x7fffffffu);
        top = max(top, uint32_t(__shfl_xor(int(top), 16)));
        top = max(top, uint32_t(__shfl_xor(int(top), 32)));
        // a power of two in front of the row's largest magnitude (finite; a row of zeros is left alone)
        const int e = top == 0 || top >= 0x7f800000u ? 0 : __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, top)) - 1;
        row_scale[r] = __builtin_amdgcn_ldexpf(a.scale * kLog2e, e);
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
            for (int k = 0; k < 8; ++k) q[r][s][k] = _Float16(__builtin_amdgcn_ldexpf(x[s * 8 + k], -e));
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) o[r][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m[r] = kNothing;
        l[r] = 0.0f;
    }

    const int32_t* pages = a.page_table + int64_t(b) * a.page_table_stride;
    const uint32_t lane_k = col * D + quarter * (S::kChunk / 4), lane_v = quarter * (4 * D) + col * (S::kChunk / 4);
    const uint32_t last_entry = total ? (total - 1) >> a.cache.page_log : 0;
    // The loads of 32 keys: where they are, their codes, and their scales.
    size_t rows_at[2];
    Tile<D> tile;
    auto locate = [&](uint32_t key) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = key + h * 16;
            const uint32_t page = min(uint32_t(pages[min(at >> a.cache.page_log, last_entry)]), a.cache.pages - 1);
            rows_at[h] = ((size_t(page) * a.cache.kv_heads + head) << a.cache.page_log) + (at & page_mask);
        }
    };
    auto load_k = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) tile.k[h][i] = load_words<S::kWords>(a.cache.k + rows_at[h] * D + lane_k + i * S::kChunk);
    };
    auto load_scales_and_v = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            tile.ks[h] = *reinterpret_cast<const float4_t*>(a.cache.k_scale + rows_at[h] + quarter * 4);
            tile.vs[h] = *reinterpret_cast<const float4_t*>(a.cache.v_scale + rows_at[h] + quarter * 4);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) tile.v[h][i] = load_words<S::kWords>(a.cache.v + rows_at[h] * D + lane_v + i * S::kChunk * 4);
    };

    auto process = [&](auto masked, uint32_t key, bool more) {
        constexpr bool kMasked = decltype(masked)::value;
        float4_t s[R][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][h] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < S::kSteps; ++st) {
                const half8_t k = S::kWords == 4 ? halves8<CODES>(tile.k[h][st / 2].w[(st % 2) * 2], tile.k[h][st / 2].w[(st % 2) * 2 + 1])
                                                 : halves8<CODES>(tile.k[h][S::kWords == 4 ? 0 : st].w[0], tile.k[h][S::kWords == 4 ? 0 : st].w[1]);
#pragma unroll
                for (int r = 0; r < R; ++r) s[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[r][st], s[r][h], 0, 0, 0);
            }
        }
        if (more) load_k();                                        // (the keys' registers are free now, the values' at the end)
        __builtin_amdgcn_sched_barrier(0);
        uint32_t sees[R][2];                                        // of the quarter's four keys, a bit each
        if constexpr (kMasked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t at = key + h * 16 + quarter * 4;
                const uint32_t there = lowest_bits(int32_t(total - at));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int32_t u = int32_t(at - context);
                    const uint32_t bits = causal ? lowest_bits(int32_t(token[r]) + 1 - u) : mask_bits(a.mask + int64_t(first_token + token[r]) * a.mask_words, a.mask_words, u);
                    sees[r][h] = bits & there;
                }
                // what lies behind the last token is no token's: no code of it may reach a product, as 0 * NaN is NaN
                uint32_t keep = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    keep |= there >> i & 1 ? 0xffu << (8 * i) : 0u;
                    tile.vs[h][i] = there >> i & 1 ? tile.vs[h][i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
                    for (int k = 0; k < S::kWords; ++k) tile.v[h][i].w[k] &= keep;
            }
        }
        // scores in units of log2, masked ones -inf
        float lead = kNothing, scales = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) scales = __builtin_fmaxf(scales, tile.vs[h][i]);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[r][h][i] * tile.ks[h][i] * row_scale[r];
                    if constexpr (kMasked) x = sees[r][h] >> i & 1 ? x : -__builtin_inff();
                    s[r][h][i] = x;
                    lead = __builtin_fmaxf(lead, x - m[r]);
                }
        }
        if (__any(lead > kLead || scales > t)) {
            const float most = __builtin_fmaxf(scales, __shfl_xor(scales, 16));
            const float largest = __builtin_fmaxf(most, __shfl_xor(most, 32));
            float shrink = 1.0f;
            if (largest > t) {
                const float now = __builtin_fmaxf(largest, 1.0e-30f);
                shrink = t / now;
                t = now;
                inv_t = 1.0f / now;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float top = -__builtin_inff();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = __builtin_fmaxf(top, s[r][h][i]);
                top = max_quarters(top);
                float alpha = 1.0f;
                if (top - m[r] > kLead) {
                    const float now = top - kStart;
                    alpha = exp2_fast(m[r] - now);
                    m[r] = now;
                }
                l[r] *= alpha;
                alpha *= shrink;
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) o[r][i] *= alpha;
            }
        }
        half8_t p[R];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float scaled = tile.vs[h][i] * inv_t;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float e = exp2_fast(s[r][h][i] - m[r]);
                    l[r] += e;
                    float w = e * scaled;
                    if constexpr (kMasked) w = s[r][h][i] == -__builtin_inff() ? 0.0f : w;   // (a hidden value's scale may be NaN)
                    p[r][h * 4 + i] = _Float16(w);
                }
            }
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
            // tile i: elements (i / kWords) * kChunk + column * kWords + i % kWords
            const half8_t v = halves8<CODES>(tile.v[0][i / S::kWords].w[i % S::kWords], tile.v[1][i / S::kWords].w[i % S::kWords]);
#pragma unroll
            for (int r = 0; r < R; ++r) o[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[r], o[r][i], 0, 0, 0);
        }
    };

    uint32_t key = key0 + wave * 32;
    if (key < key1) {
        locate(key);
        load_k();
        load_scales_and_v();
    }
    while (key < key1) {
        const uint32_t after = key + kWaves * 32;
        const bool more = after < key1;
        if (more) locate(after);
        if (key + 32 <= all_see) process(std::false_type{}, key, more);
        else process(std::true_type{}, key, more);
        if (more) load_scales_and_v();
        __builtin_amdgcn_sched_barrier(0);
        key = after;
    }

    // join the waves, 16 rows at a time, and write them
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = sum_quarters(l[r]);
        if (quarter == 0) {
            joined_m[wave][col] = m[r];
            joined_l[wave][col] = l[r];
        }
        __syncthreads();
        float top = joined_m[0][col], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, joined_m[w][col]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += joined_l[w][col] * exp2_fast(joined_m[w][col] - top);
        // l may be NaN (a NaN among the scores), and then the row is
        const float factor = (sum == 0.0f ? 0.0f : exp2_fast(m[r] - top) / sum) * t;
#pragma unroll
        for (int c = 0; c < S::kLoads; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // rows quarter * 4 + i of the kWords tiles of a chunk are neighbouring elements
                float* to = &joined[wave][col * kRowFloats + c * S::kChunk + (quarter * 4 + i) * S::kWords];
#pragma unroll
                for (int k = 0; k < S::kWords; ++k) to[k] = o[r][c * S::kWords + k][i] * factor;
            }
        if (wave == 0 && quarter == 0) row_l[col] = sum, row_m[col] = top;
        __syncthreads();
        // 16 rows of D elements, four to a thread
        for (uint32_t at = threadIdx.x; at < 16 * D / 4; at += kWaves * 64) {
            const uint32_t c = at / (D / 4), d = at % (D / 4) * 4;
            const uint32_t row = row0 + r * 16 + c;
            if (row >= rows) continue;
            float4_t x = *reinterpret_cast<const float4_t*>(&joined[0][c * kRowFloats + d]);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) x += *reinterpret_cast<const float4_t*>(&joined[w][c * kRowFloats + d]);
            const uint32_t tok = divide(row, a.group_magic), qh = head * a.group + row - tok * a.group;
            const size_t place = size_t(first_token + tok) * a.q_heads + qh;
            const float lse = row_l[c] == 0.0f ? -__builtin_inff() : row_m[c] + __builtin_log2f(row_l[c]);
            if (a.splits == 1) {
                uint2_t w;
                if (a.type == FKLHIP_BF16) { w.x = pack2<FKLHIP_BF16>(x[0], x[1]); w.y = pack2<FKLHIP_BF16>(x[2], x[3]); }
                else { w.x = pack2<FKLHIP_F16>(x[0], x[1]); w.y = pack2<FKLHIP_F16>(x[2], x[3]); }
                *reinterpret_cast<uint2_t*>(a.out.data + int64_t(first_token + tok) * a.out.token_stride + int64_t(qh) * a.out.head_stride + d * 2) = w;
                if (d == 0 && a.lse) a.lse[place] = lse * kLn2;
            } else {
                *reinterpret_cast<float4_t*>(a.partial + (place * a.splits + split) * D + d) = x;
                if (d == 0) a.partial_lse[place * a.splits + split] = lse;
            }
        }
        __syncthreads();
    }
}

template <int D, int CODES, int R> int start_attention(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) {
    // workgroups of the same keys and other rows are a multiple of eight apart, which is the same XCD and its L2
    uint32_t x = a.cache.kv_heads * a.splits;
    if (plan.row_blocks > 1) x = (x + 7) / 8 * 8;
    const dim3 grid(x, plan.row_blocks, a.batch);
    info = {"tree_attention", {grid.x, grid.y, grid.z}, {kWaves * 64, 1, 1}, uint32_t((kWaves * 16 * (D + 4 + 2) + 32) * 4)};
    k_tree_attention<D, CODES, R><<<grid, dim3(kWaves * 64), 0, static_cast<hipStream_t>(stream)>>>(a);
    return int(hipGetLastError());
}

template <int D> int launch_attention(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) {
    const bool int8 = a.cache.codes == FKLHIP_CODES_INT8;
    if constexpr (D <= 128) {
        if (plan.row_tiles == 2)
            return int8 ? start_attention<D, FKLHIP_CODES_INT8, 2>(a, plan, stream, info) : start_attention<D, FKLHIP_CODES_E4M3, 2>(a, plan, stream, info);
    }
    return int8 ? start_attention<D, FKLHIP_CODES_INT8, 1>(a, plan, stream, info) : start_attention<D, FKLHIP_CODES_E4M3, 1>(a, plan, stream, info);
}

} // namespace fkattn
