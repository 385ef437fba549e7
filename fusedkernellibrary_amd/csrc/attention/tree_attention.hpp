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
// Two forms. Few rows to a key head (k_split_keys): the four waves of a workgroup take the same 16 or 32 rows and other keys,
// which each loads into its registers, and the rows' parts are joined in LDS; the bound is reading the cache. Many rows
// (k_split_rows): the waves take other rows and the same keys, which pass through LDS, copied there without registers and
// several stages ahead; the bound is the arithmetic, of which turning codes into halves is shared by a wave's row tiles.
//
// How the work is dealt out. The device alone knows the sequences' lengths, so every workgroup adds them up: the keys of all
// (sequence, key head, block of rows), one behind the other, are cut into equal shares, one to a workgroup, all of which run
// at the same time. A share may hold parts of two of them and whole ones in between; whole ones are written to the output,
// parts to the workspace, from where k_merge takes them. Without shares (short sequences, or so many that the order of
// launch evens them out) a workgroup takes one whole (sequence, key head, block of rows).
//
// The running maximum is a reference m_r and not the exact maximum: weights are w = 2^(s - m) * vs, sums those of 2^(s - m), and
// m moves only when a weight exceeds 2^kLead. Only then are scores compared across lanes and the sums rescaled. The largest
// weight starts at 2^kStart, so one is subnormal in half precision (below 2^-14) only 2^-(14 + kStart) below the largest of
// the first keys. (Value scales below kLeastScale count as that: values of 10^-22 and less lose accuracy.)
#pragma once

#include <type_traits>

#include "work_shares.hpp"

namespace fkattn {

constexpr int kWaves = 4;                    // of a workgroup: they share out a chunk's keys, 32 at a time
constexpr float kStart = 6.0f, kLead = 14.0f, kLargest = 16384.0f, kLeastScale = 0x1p-80f, kMostSum = 0x1p98f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNothing = -1.0e30f;         // the reference of a row that has seen no key

// How a key's product with the queries is taken. The matrix unit has products of 8-bit codes themselves, for runs of 64 (int8) or
// 128 (e4m3) elements: a query row is then a sum of two or three rows of such codes, and no key is converted.
//   int8: in fixed point, 256 * hi + lo (bfloat16: exact for elements from 2^-7 of the row's largest on) or with a third
//         part behind them (half precision: exact from 2^-11 on); smaller elements are off by 2^-15 (2^-22) of the largest.
//   e4m3: what four bits hold of each element, and of what is left, twice (8 bits, all that bfloat16 has) or three times;
//         elements below 2^-9 of the largest are off by 2^-17 of it.
// Heads of other sizes: keys as halves.
template <int D, int CODES> constexpr bool kCodeProducts = CODES == FKLHIP_CODES_INT8 ? D % 64 == 0 : D % 128 == 0;

using int2_t = int __attribute__((ext_vector_type(2)));
using int4_t = int __attribute__((ext_vector_type(4)));
using int8_t8 = int __attribute__((ext_vector_type(8)));

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
// Bits u .. u + 3 of a row of a mask, where those below 0 (the context's) are set and those behind the row are not; `first` is
// the row's first word.
__device__ __forceinline__ uint32_t mask_bits(const uint64_t* row, uint64_t first, uint32_t words, int32_t u) {
    const uint32_t below = u >= 0 ? 0u : u <= -4 ? 4u : uint32_t(-u), from = u >= 0 ? uint32_t(u) : 0u;
    const uint32_t shift = from & 63u;
    uint64_t lo = from < 64u ? first : 0, hi = 0;
    if (words > 1) {                                          // (the same for the whole wave)
        const uint32_t lo_at = from >> 6, hi_at = (from + 3) >> 6;
        lo = lo_at < words ? row[lo_at] : 0;
        hi = hi_at < words && hi_at != lo_at ? row[hi_at] : 0;
    }
    const uint32_t bits = uint32_t(lo >> shift) | (shift ? uint32_t(hi << (64u - shift)) : 0u);
    return (lowest_bits(int32_t(below)) | bits << below) & 15u;
}

// Keys key0 .. key1 of row block `block` and key head `head` of a sequence; where its parts go.
struct Segment {
    Sequence seq;
    uint32_t b, head, row0, rows;        // rows row0 .. row0 + rows of the sequence's
    uint32_t key0, key1, all_see;        // every row sees the keys in front of all_see
    int part;                            // -1: whole, 0 or 1: the share's part
    uint32_t behind, quarter;            // keys of the share behind the segment's, and a quarter of them all
};
__device__ __forceinline__ Segment segment_of(Args& a, const Sequence& s, uint32_t b, uint32_t head, uint32_t block, uint32_t k0, uint32_t k1, int part) {
    Segment x;
    x.seq = s; x.b = b; x.head = head; x.part = part;
    x.row0 = block * a.unit_rows;
    x.rows = min(a.unit_rows, s.rows - x.row0);
    const bool causal = a.mask == nullptr;
    const uint32_t any_sees = causal ? min(s.context + divide(x.row0 + x.rows - 1, a.group_magic) + 1, s.total) : s.total;
    x.all_see = causal ? min(s.context + divide(x.row0, a.group_magic) + 1, s.total) : s.context;
    x.key0 = k0 << a.granule_log;
    x.key1 = min(k1 << a.granule_log, any_sees);
    return x;
}

__device__ __forceinline__ uint32_t to_vector(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Calls `run` for every segment of the workgroup.
template <typename F> __device__ __forceinline__ void walk(Args& a, uint32_t lane, F run) {
    // granules at .. end of all are the share's, `in` of b's are in front of them; without shares: (sequence, head, block) of the grid
    uint32_t b = blockIdx.z, in = 0, at = 0, end = 1;
    const bool shared = a.share_odd != 0;
    if (shared) {
        const uint32_t share = own_share(a);
        const Found f = find(a, lane, [&](uint32_t all, uint32_t, uint32_t, uint32_t upto) { return upto > share_begin(a, all, share); });
        at = share_begin(a, f.all, share);
        end = share_begin(a, f.all, share + 1);
        b = f.b;
        in = at - f.before;
    }
    const uint32_t whole = end - at;
    while (at < end && b < kernel_args().batch) {
        Args& a = kernel_args();
        const Sequence s = sequence_at(a, b);
        const uint32_t n = granules_of(a, s), subs = subs_of(a, s);
        uint32_t head = blockIdx.x, block = blockIdx.y, g0 = 0, g1 = n, count = end - at;
        int part = -1;
        if (shared) {
            if (n * subs == 0 || in >= n * subs * a.cache.kv_heads) {
                ++b;
                in = 0;
                continue;
            }
            head = in / (n * subs);
            const uint32_t in_head = in - head * (n * subs), block_size = n * a.block_subs;
            block = in_head / block_size;
            const uint32_t g = in_head - block * block_size, cost = min(a.block_subs, subs - block * a.block_subs), size = n * cost;
            count = min(size - g, end - at);
            part = count == size ? -1 : g == 0 ? 1 : 0;
            g0 = (g + cost - 1) >> (cost - 1);
            g1 = (g + count + cost - 1) >> (cost - 1);
        } else if (block * a.block_subs >= subs) {
            return;
        }
        // (a segment needs all scalar registers: what the walk goes on with waits in vector registers)
        const uint32_t next_at = to_vector(at + count), next_in = to_vector(in + count), next_end = to_vector(end), next_b = to_vector(b);
        Segment x = segment_of(a, s, b, head, block, g0, g1, part);
        x.quarter = whole << a.granule_log >> 2;
        x.behind = (end - at - count) << a.granule_log;
        if (!shared) x.behind = 0, x.quarter = (x.key1 - x.key0) >> 2;
        run(x);
        at = __builtin_amdgcn_readfirstlane(next_at);
        in = __builtin_amdgcn_readfirstlane(next_in);
        end = __builtin_amdgcn_readfirstlane(next_end);
        b = __builtin_amdgcn_readfirstlane(next_b);
    }
}

// A wave's priority falls as its share gets done: left alone, the oldest of the workgroups on a compute unit runs ahead, and the
// last one ends alone, without others to fill its gaps.
__device__ __forceinline__ void set_priority(const Segment& x, uint32_t key) {
    const uint32_t left = x.behind + x.key1 - key;
    if (left > 3 * x.quarter) __builtin_amdgcn_s_setprio(3);
    else if (left > 2 * x.quarter) __builtin_amdgcn_s_setprio(2);
    else if (left > x.quarter) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

// ---- a wave's rows ---------------------------------------------------------------------------------------------------

// PARTS: rows of codes that a query row is the sum of, or 0: halves.
template <int D, int CODES, int R, int PARTS> struct WaveRows {
    using S = Shape<D>;
    static constexpr int kQueryRegs = PARTS == 0 ? S::kSteps * 4 : PARTS * S::kSteps * 2;     // dwords of a lane's quarter row
    uint32_t token[R];                   // the new token of the lane's row
    uint64_t sees_first[R];              // and the first word of its mask: fetched in good time, a word is all that trees of up to 64 have
    uint32_t q[R][kQueryRegs];           // halves, or the parts one behind the other
    float row_scale[R];
    float4_t o[R][S::kTiles];
    float m[R], l[R];
    float limit[R];                      // the largest weight that is fine as it is: kLargest, or -1 while the row has seen no key

    // Rows of the tiles `tile(r)` (16 rows each) of a segment; those behind its last are its last again.
    template <typename F> __device__ __forceinline__ void start(Args& a, const Segment& x, uint32_t col, uint32_t quarter, F tile) {
        uint4_t raw[R][S::kSteps];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t row = x.row0 + min(tile(r) * 16 + col, x.rows - 1);
            token[r] = divide(row, a.group_magic);
            sees_first[r] = a.mask ? a.mask[int64_t(x.seq.first_token + token[r]) * a.mask_words] : 0;
            const uint32_t g = row - token[r] * a.group;
            const char* from = a.q.data + int64_t(x.seq.first_token + token[r]) * a.q.token_stride + int64_t(x.head * a.group + g) * a.q.head_stride;
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s) {
                // the elements that the quarter's codes of this step are of: kChunk / 4 neighbours of each run of kChunk
                const uint32_t at = S::kChunk == 64 ? (s / 2) * 64 + quarter * 16 + (s % 2) * 8 : s * 32 + quarter * 8;
                raw[r][s] = *reinterpret_cast<const uint4_t*>(from + at * 2);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float e[S::kSteps * 8];
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (a.type == FKLHIP_BF16) unpack2<FKLHIP_BF16>(raw[r][s][k], e[s * 8 + 2 * k], e[s * 8 + 2 * k + 1]);
                    else unpack2<FKLHIP_F16>(raw[r][s][k], e[s * 8 + 2 * k], e[s * 8 + 2 * k + 1]);
                }
#pragma unroll
            for (int k = 0; k < S::kSteps * 8; ++k) top = max(top, __builtin_bit_cast(uint32_t, e[k]) & 0x7fffffffu);
            top = max(top, uint32_t(__shfl_xor(int(top), 16)));
            top = max(top, uint32_t(__shfl_xor(int(top), 32)));
            // a power of two in front of the row's largest magnitude (a row of zeros, or with an infinity, is left alone)
            const bool plain = top == 0 || top >= 0x7f800000u;
            const int p = plain ? 0 : __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, top)) - 1;
            float unit = a.scale * kLog2e;
            if constexpr (PARTS == 0) {
#pragma unroll
                for (int k = 0; k < S::kSteps * 4; ++k)
                    q[r][k] = pack2<FKLHIP_F16>(__builtin_amdgcn_ldexpf(e[2 * k], -p), __builtin_amdgcn_ldexpf(e[2 * k + 1], -p));
            } else if constexpr (CODES == FKLHIP_CODES_INT8) {
                // A power of two in front of the largest magnitude that leaves it below 127.5 * 2^8 (or 2^14); a row with an
                // infinity or a NaN has scores that are NaN.
                constexpr int kBits = PARTS == 2 ? 14 : 21;
                const int up = kBits - p - (__builtin_amdgcn_ldexpf(__builtin_bit_cast(float, top), -p) >= 1.9921875f ? 1 : 0);
                unit = top >= 0x7f800000u ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(unit, -up - p);
#pragma unroll
                for (int k = 0; k < S::kSteps * 2; ++k) {
                    uint32_t w[PARTS];
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) w[part] = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        int v = int(__builtin_rintf(__builtin_amdgcn_ldexpf(e[4 * k + i], up)));
#pragma unroll
                        for (int part = PARTS - 1; part >= 0; --part) {      // the last digit of -128 .. 127, then the rest
                            const int digit = int(uint32_t(v) << 24) >> 24;
                            w[part] |= uint32_t(digit & 0xff) << (8 * i);
                            v = (v - digit) >> 8;
                        }
                    }
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) q[r][part * S::kSteps * 2 + k] = w[part];
                }
            } else {
                unit = top >= 0x7f800000u ? __builtin_nanf("") : unit * 0x1p-7f;
#pragma unroll
                for (int k = 0; k < S::kSteps * 2; ++k) {
                    float left[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) left[i] = __builtin_amdgcn_ldexpf(e[4 * k + i], 7 - p);
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        int w = __builtin_amdgcn_cvt_pk_fp8_f32(left[0], left[1], 0, false);
                        w = __builtin_amdgcn_cvt_pk_fp8_f32(left[2], left[3], w, true);
                        q[r][part * S::kSteps * 2 + k] = uint32_t(w);
                        float taken[4];
                        decode4<FKLHIP_CODES_E4M3>(uint32_t(w), taken);
#pragma unroll
                        for (int i = 0; i < 4; ++i) left[i] -= taken[i];
                    }
                }
            }
            row_scale[r] = __builtin_amdgcn_ldexpf(unit, p);
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) o[r][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            m[r] = 0.0f;
            l[r] = 0.0f;
            limit[r] = -1.0f;
        }
    }
    // The reference at the end, for comparison with others'.
    __device__ __forceinline__ float reference(int r) const { return limit[r] < 0.0f ? kNothing : m[r]; }

    // Products of a block of 16 keys with the rows, four keys to a quarter; the codes' scales are not in them.
    template <typename K> __device__ __forceinline__ void products(K get_k, float4_t (&y)[R][2]) {
        if constexpr (PARTS == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < R; ++r) y[r][h] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Words<S::kWords> w = get_k(h, i);
#pragma unroll
                    for (int k = 0; k < S::kWords / 2; ++k) {
                        const half8_t codes = halves8<CODES>(w.w[2 * k], w.w[2 * k + 1]);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const uint32_t* from = &q[r][(i * (S::kWords / 2) + k) * 4];
                            y[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, __builtin_bit_cast(half8_t, uint4_t{from[0], from[1], from[2], from[3]}), y[r][h], 0, 0, 0);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);                  // (all codes at once as halves would take 32 registers)
            }
        } else if constexpr (CODES == FKLHIP_CODES_INT8) {
            // the first two parts as one whole number, the third by itself: with it, 32 bits would not do
            int4_t sum[PARTS - 1][R][2];
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const Words<S::kWords> w = get_k(h, i);
                        const int4_t codes = {int(w.w[0]), int(w.w[1]), int(w.w[2]), int(w.w[3])};
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const uint32_t* from = &q[r][part * S::kSteps * 2 + i * 4];
                            int4_t& to = sum[part < 2 ? 0 : 1][r][h];
                            const int4_t before = i > 0 ? to : part == 1 ? to << 8 : int4_t{0, 0, 0, 0};
                            to = __builtin_amdgcn_mfma_i32_16x16x64_i8(codes, int4_t{int(from[0]), int(from[1]), int(from[2]), int(from[3])}, before, 0, 0, 0);
                        }
                    }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[r][h][i] = float(sum[0][r][h][i]);
                        if constexpr (PARTS == 3) y[r][h][i] = __builtin_fmaf(y[r][h][i], 256.0f, float(sum[1][r][h][i]));
                    }
        } else {
#pragma unroll
            for (int i = 0; i < S::kLoads; i += 2)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Words<S::kWords> lo = get_k(h, i), hi = get_k(h, i + 1);
                    const int8_t8 codes = {int(lo.w[0]), int(lo.w[1]), int(lo.w[2]), int(lo.w[3]), int(hi.w[0]), int(hi.w[1]), int(hi.w[2]), int(hi.w[3])};
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int part = 0; part < PARTS; ++part) {
                            const uint32_t* from = &q[r][part * S::kSteps * 2 + i * 4];
                            const int8_t8 row = {int(from[0]), int(from[1]), int(from[2]), int(from[3]), int(from[4]), int(from[5]), int(from[6]), int(from[7])};
                            const float4_t before = i == 0 && part == 0 ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : y[r][h];
                            y[r][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes, row, before, 0, 0, 0, 0, 0, 0);   // (e4m3 both, no scales)
                        }
                }
        }
    }

    // 32 keys from `key` on: get_k(block, load) and get_v have their codes, get_scales(block, ks, vs) their scales;
    // after_scores runs when the keys are used up.
    template <bool MASKED, typename K, typename V, typename G, typename A>
    __device__ __forceinline__ void step(const Segment& x, uint32_t key, uint32_t quarter, K get_k, V get_v, G get_scales, A after_scores) {
        float4_t y[R][2];
        products(get_k, y);
        after_scores();
        uint32_t sees[R][2], keep[2];                               // of the quarter's four keys, a bit each; bytes that are a token's
        float4_t ks[2], vs[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            get_scales(h, ks[h], vs[h]);
            if constexpr (MASKED) {
                Args& a = kernel_args();
                const uint32_t at = key + h * 16 + quarter * 4;
                const uint32_t there = lowest_bits(int32_t(x.seq.total - at));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int32_t u = int32_t(at - x.seq.context);
                    const uint32_t bits = a.mask == nullptr ? lowest_bits(int32_t(token[r]) + 1 - u)
                                                            : mask_bits(a.mask + int64_t(x.seq.first_token + token[r]) * a.mask_words, sees_first[r], a.mask_words, u);
                    sees[r][h] = bits & there;
                }
                // what lies behind the last token is no token's: no code of it may reach a product, as 0 * NaN is NaN
                keep[h] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) keep[h] |= there >> i & 1 ? 0xffu << (8 * i) : 0u;
            }
        }
        // Weights, and a look at whether a reference has to move: where a weight is too large for half precision, or where the
        // row has seen no key yet.
        float w[R][2][4], sum[R];
        bool move = false;
        auto weigh = [&](int r, int h, int i, float score) {
            float e = exp2_fast(score);
            float weight = e * vs[h][i];
            if constexpr (MASKED) {
                e = sees[r][h] >> i & 1 ? e : 0.0f;
                weight = sees[r][h] >> i & 1 ? weight : 0.0f;       // (a hidden value's scale may be NaN)
            }
            sum[r] += e;
            return weight;
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = 0.0f;
            sum[r] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[r][h][i] *= ks[h][i];
                    w[r][h][i] = weigh(r, h, i, __builtin_fmaf(y[r][h][i], row_scale[r], -m[r]));
                    top = __builtin_fmaxf(top, w[r][h][i]);
                }
            move |= top > limit[r] || sum[r] > kMostSum;
        }
        if (__builtin_expect(__any(move), 0)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                // the largest weight there would be, in units of log2
                float top = -__builtin_inff();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = y[r][h][i] * row_scale[r] + __builtin_log2f(__builtin_fmaxf(vs[h][i], kLeastScale));
                        if constexpr (MASKED) v = sees[r][h] >> i & 1 ? v : -__builtin_inff();
                        top = __builtin_fmaxf(top, v);
                    }
                top = max_quarters(top);
                float alpha = 1.0f;
                if (limit[r] < 0.0f ? top > -__builtin_inff() : top - m[r] > kLead) {
                    alpha = limit[r] < 0.0f ? 0.0f : exp2_fast(m[r] + kStart - top);
                    m[r] = top - kStart;
                    limit[r] = kLargest;
                }
                l[r] *= alpha;
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) o[r][i] *= alpha;
                // (from the rounded scores: those of 2^100 differ from their reference by more than an exponent holds)
                sum[r] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[r][h][i] = weigh(r, h, i, y[r][h][i] * row_scale[r] - m[r]);
            }
        }
        half8_t p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += sum[r];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[r][h * 4 + i] = _Float16(w[r][h][i]);
        }
#pragma unroll
        for (int c = 0; c < S::kLoads; ++c) {
            const Words<S::kWords> v0 = get_v(0, c), v1 = get_v(1, c);
#pragma unroll
            for (int k = 0; k < S::kWords; ++k) {
                // tile c * kWords + k: elements c * kChunk + column * kWords + k
                const half8_t v = MASKED ? halves8<CODES>(v0.w[k] & keep[0], v1.w[k] & keep[1]) : halves8<CODES>(v0.w[k], v1.w[k]);
#pragma unroll
                for (int r = 0; r < R; ++r) o[r][c * S::kWords + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[r], o[r][c * S::kWords + k], 0, 0, 0);
            }
        }
    }
};

// Four or two neighbouring elements of a row of the result: to the output, or to a share's part.
template <int D, int N> __device__ __forceinline__ void put(Args& a, const Segment& x, uint32_t share, uint32_t row, uint32_t d, const float* v) {
    if (x.part < 0) {
        const uint32_t tok = divide(x.row0 + row, a.group_magic), qh = x.head * a.group + x.row0 + row - tok * a.group;
        char* to = a.out.data + int64_t(x.seq.first_token + tok) * a.out.token_stride + int64_t(qh) * a.out.head_stride + d * 2;
        uint32_t w[N / 2];
#pragma unroll
        for (int k = 0; k < N / 2; ++k) w[k] = a.type == FKLHIP_BF16 ? pack2<FKLHIP_BF16>(v[2 * k], v[2 * k + 1]) : pack2<FKLHIP_F16>(v[2 * k], v[2 * k + 1]);
        if constexpr (N == 4) *reinterpret_cast<uint2_t*>(to) = uint2_t{w[0], w[1]};
        else *reinterpret_cast<uint32_t*>(to) = w[0];
    } else {
        float* to = a.partial + ((size_t(share) * 2 + x.part) * a.unit_rows + row) * D + d;
#pragma unroll
        for (int k = 0; k < N; ++k) to[k] = v[k];
    }
}
// lse is in units of log2.
__device__ __forceinline__ void put_lse(Args& a, const Segment& x, uint32_t share, uint32_t row, float m, float l) {
    const float lse = l == 0.0f ? -__builtin_inff() : m + __builtin_log2f(l);
    if (x.part < 0) {
        if (!a.lse) return;
        const uint32_t tok = divide(x.row0 + row, a.group_magic), qh = x.head * a.group + x.row0 + row - tok * a.group;
        a.lse[size_t(x.seq.first_token + tok) * a.q_heads + qh] = lse * kLn2;
    } else {
        a.partial_lse[(size_t(share) * 2 + x.part) * a.unit_rows + row] = lse;
    }
}

// A wave's way through the page table: 64 entries at a time, one to a lane. (A scalar load for each block of keys would have
// every wave wait for it; places are asked for in ascending order.)
struct Pages {
    uint32_t first, entry;
    __device__ __forceinline__ void fetch(Args& a, const Segment& x, uint32_t page, uint32_t lane) {
        first = page;
        const int32_t* entries = a.page_table + int64_t(x.b) * a.page_table_stride;
        entry = min(uint32_t(entries[min(page + lane, (x.seq.total - 1) >> a.cache.page_log)]), a.cache.pages - 1);
    }
    // Where 16 keys of the segment are in the cache: tokens in front of them.
    __device__ __forceinline__ size_t place(Args& a, const Segment& x, uint32_t key, uint32_t lane) {
        const uint32_t page = key >> a.cache.page_log;
        if (__builtin_expect(page - first >= 64, 0)) fetch(a, x, page, lane);
        const uint32_t at = __builtin_amdgcn_readlane(entry, page - first);
        return ((size_t(at) * a.cache.kv_heads + x.head) << a.cache.page_log) + (key & ((1u << a.cache.page_log) - 1u));
    }
};

// ---- few rows: the waves split the keys -------------------------------------------------------------------------------

template <int D, int CODES, int R, int PARTS>
__global__ __launch_bounds__(kWaves * 64, D > 128 ? 1 : R == 1 ? 2 : 2) void k_split_keys(const AttentionArgs) {
    using S = Shape<D>;
    constexpr int kRowFloats = D + 4;                              // of a row in LDS: 16 bytes further round the banks than the last
    __shared__ __attribute__((aligned(16))) float joined[kWaves][16 * kRowFloats];
    __shared__ float joined_m[kWaves][16], joined_l[kWaves][16], row_m[16], row_l[16];
    walk(kernel_args(), threadIdx.x & 63, [&](const Segment& x) {
        Args& a = kernel_args();
        const uint32_t thread = thread_here(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), col = lane & 15, quarter = lane >> 4;
        const uint32_t lane_k = col * D + quarter * (S::kChunk / 4), lane_v = quarter * (4 * D) + col * (S::kChunk / 4);
        size_t at[2];
        Words<S::kWords> k[2][S::kLoads], v[2][S::kLoads];
        float4_t ks[2], vs[2];
        Pages pages{0, 0};
        auto locate = [&](uint32_t key) {
#pragma unroll
            for (int h = 0; h < 2; ++h) at[h] = pages.place(a, x, key + h * 16, lane);
        };
        auto load_k = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) k[h][i] = load_words<S::kWords>(a.cache.k + at[h] * D + lane_k + i * S::kChunk);
        };
        auto load_scales_and_v = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ks[h] = *reinterpret_cast<const float4_t*>(a.cache.k_scale + at[h] + quarter * 4);
                vs[h] = *reinterpret_cast<const float4_t*>(a.cache.v_scale + at[h] + quarter * 4);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) v[h][i] = load_words<S::kWords>(a.cache.v + at[h] * D + lane_v + i * S::kChunk * 4);
        };
        uint32_t key = x.key0 + wave * 32;
        if (key < x.key1) pages.fetch(a, x, key >> a.cache.page_log, lane);
        WaveRows<D, CODES, R, PARTS> rows;
        rows.start(kernel_args(), x, col, quarter, [](int r) { return uint32_t(r); });
        if (key < x.key1) {
            locate(key);
            load_k();
            load_scales_and_v();
        }
        auto get_k = [&](int h, int i) { return k[h][i]; };
        auto get_v = [&](int h, int i) { return v[h][i]; };
        auto get_scales = [&](int h, float4_t& s, float4_t& t) { s = ks[h]; t = vs[h]; };
        // keys that all rows see, then the others
        auto keys = [&](auto masked, uint32_t end) {
#pragma unroll 1
            while (key < end) {
                const uint32_t next = key + kWaves * 32;
                const bool more = next < x.key1;
                set_priority(x, key);
                if (more) locate(next);
                // the keys' registers are free for the next once the scores are there, the others' at the end
                rows.template step<decltype(masked)::value>(x, key, quarter, get_k, get_v, get_scales, [&] {
                    if (more) load_k();
                    __builtin_amdgcn_sched_barrier(0);
                });
                if (more) load_scales_and_v();
                __builtin_amdgcn_sched_barrier(0);
                key = next;
            }
        };
        keys(std::false_type{}, min(x.key1, x.all_see & ~31u));
        keys(std::true_type{}, x.key1);
        // join the waves, 16 rows at a time, and write them
        Args& out = kernel_args();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float l = sum_quarters(rows.l[r]), m = rows.reference(r);
            if (quarter == 0) {
                joined_m[wave][col] = m;
                joined_l[wave][col] = l;
            }
            __syncthreads();
            float top = joined_m[0][col], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, joined_m[w][col]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += joined_l[w][col] * exp2_fast(joined_m[w][col] - top);
            // (a sum that is NaN, from a NaN among the scores, makes the row NaN)
            const float factor = sum == 0.0f ? 0.0f : exp2_fast(m - top) / sum;
#pragma unroll
            for (int c = 0; c < S::kLoads; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // rows quarter * 4 + i of the kWords tiles of a chunk are neighbouring elements
                    float* to = &joined[wave][col * kRowFloats + c * S::kChunk + (quarter * 4 + i) * S::kWords];
#pragma unroll
                    for (int w = 0; w < S::kWords; ++w) to[w] = rows.o[r][c * S::kWords + w][i] * factor;
                }
            if (wave == 0 && quarter == 0) row_l[col] = sum, row_m[col] = top;
            __syncthreads();
            for (uint32_t i = thread; i < 16 * D / 4; i += kWaves * 64) {
                const uint32_t c = i / (D / 4), d = i % (D / 4) * 4, row = r * 16 + c;
                if (row >= x.rows) continue;
                float4_t e = *reinterpret_cast<const float4_t*>(&joined[0][c * kRowFloats + d]);
#pragma unroll
                for (int w = 1; w < kWaves; ++w) e += *reinterpret_cast<const float4_t*>(&joined[w][c * kRowFloats + d]);
                const float f[4] = {e[0], e[1], e[2], e[3]};
                put<D, 4>(out, x, own_share(out), row, d, f);
                if (d == 0) put_lse(out, x, own_share(out), row, row_m[c], row_l[c]);
            }
            __syncthreads();
        }
    });
}

// ---- many rows: the waves split the rows ------------------------------------------------------------------------------

// A stage of keys: per block of 16 their codes, their values' codes, and the scales of both. A wave copies a block, or, where
// a stage has two (heads of more than 128 elements), the keys' or the values' half of one. Three stages stay under 64 KB.
template <int D> struct Stage {
    static constexpr uint32_t kBlocks = D <= 128 ? 4 : 2, kKeys = 16 * kBlocks, kCodes = 16 * D, kBlockBytes = 2 * kCodes + 128, kBytes = kBlocks * kBlockBytes;
    static constexpr int kStages = 3, kRuns = (kCodes + 1023) / 1024;     // runs of 1 KB (the second of 1536 bytes is half of one)
    static constexpr int kCopies = kBlocks == 4 ? 2 * kRuns + 1 : kRuns + 1;   // memory operations of a wave
};

// Copies to LDS without registers, 16 or 4 bytes a lane at `lds` + the same times the lane's number; the count of memory
// operations in flight says when they are there.
// (the compiler is told that a value is the wave's and not the lane's)
__device__ __forceinline__ uint32_t of_wave(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const char* of_wave(const char* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const char*>(uint64_t(of_wave(uint32_t(v >> 32))) << 32 | of_wave(uint32_t(v)));
}
__device__ __forceinline__ void copy16(const char* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(of_wave(lds)), "v"(offset), "s"(of_wave(base)) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const char* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(of_wave(lds)), "v"(offset), "s"(of_wave(base)) : "memory", "m0");
}
// All but the wave's last N memory operations are done; then all waves' are, and nobody reads LDS any more.
template <int N> __device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory"); }

template <int D, int CODES, int R, int PARTS>
__global__ __launch_bounds__(kWaves * 64, D > 128 ? 1 : 2) void k_split_rows(const AttentionArgs) {
    using S = Shape<D>;
    using P = Stage<D>;
    __shared__ __attribute__((aligned(1024))) char ring[P::kStages * P::kBytes];
    // Runs of 16 bytes a lane are copied so that a lane finds its own at 16 * lane; those of 8 (heads of 96) as they lie.
    constexpr bool kOwn = S::kWords == 4;
    constexpr uint32_t kNextK = kOwn ? 1024 : 32, kNextV = kOwn ? 1024 : 128;
    walk(kernel_args(), threadIdx.x & 63, [&](const Segment& x) {
        const uint32_t thread = thread_here(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), col = lane & 15, quarter = lane >> 4;
        const uint32_t from_k = kOwn ? col * D + quarter * 16 : lane * 16, from_v = kOwn ? quarter * (4 * D) + col * 16 : lane * 16;
        const uint32_t read_k = kOwn ? lane * 16 : col * D + quarter * 8, read_v = kOwn ? lane * 16 : quarter * (4 * D) + col * 8;
        const uint32_t ring_at = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)ring)));
        const uint32_t stages = x.key1 > x.key0 ? (x.key1 - x.key0 + P::kKeys - 1) / P::kKeys : 0;
        Pages pages{0, 0};
        const uint32_t block = P::kBlocks == 4 ? wave : wave & 1;
        if (stages) pages.fetch(kernel_args(), x, (x.key0 + block * 16) >> kernel_args().cache.page_log, lane);
        auto copy = [&](uint32_t stage) {
            Args& a = kernel_args();
            const size_t at = pages.place(a, x, x.key0 + stage * P::kKeys + block * 16, lane);
            const uint32_t to = ring_at + (stage % P::kStages) * P::kBytes + block * P::kBlockBytes;
#pragma unroll
            for (int i = 0; i < P::kRuns; ++i)
                if (kOwn || i == 0 || lane < 32) {
                    if (P::kBlocks == 4 || wave < 2) copy16(a.cache.k + at * D, from_k + i * (kOwn ? 64 : 1024), to + i * 1024);
                    if (P::kBlocks == 4 || wave >= 2) copy16(a.cache.v + at * D, from_v + i * (kOwn ? 256 : 1024), to + P::kCodes + i * 1024);
                }
            // 16 scales of keys and 16 of values side by side: the lanes' offsets cover the distance of the two arrays
            if (lane < 32) {
                if (P::kBlocks == 4) {
                    const char* s = reinterpret_cast<const char*>((lane < 16 ? a.cache.k_scale : a.cache.v_scale) + at) + (lane & 15) * 4;
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(of_wave(to + 2 * P::kCodes)), "v"(s) : "memory", "m0");
                } else if (lane < 16) {
                    copy4(reinterpret_cast<const char*>((wave < 2 ? a.cache.k_scale : a.cache.v_scale) + at), lane * 4, to + 2 * P::kCodes + (wave < 2 ? 0 : 64));
                }
            }
        };
#pragma unroll
        for (uint32_t i = 0; i < P::kStages - 1; ++i)
            if (i < stages) copy(i);
        const uint32_t tiles = (x.rows + 15) / 16;
        auto loop = [&](auto count) {
            constexpr int kMine = decltype(count)::value;
            WaveRows<D, CODES, kMine == 0 ? 1 : kMine, PARTS> rows;
            if constexpr (kMine > 0) rows.start(kernel_args(), x, col, quarter, [&](int r) { return wave + kWaves * r; });
            uint32_t key = x.key0, stage = 0;
            const char* piece = ring;
            // (every stage's first step; waves without rows take part in the copies and the waiting)
            auto begin = [&](uint32_t key) {
                if ((key & (P::kKeys - 1)) == 0) {
                    set_priority(x, key);
                    if (stage + 1 < stages) arrive<P::kCopies>();
                    else arrive<0>();
                    if (stage + P::kStages - 1 < stages) copy(stage + P::kStages - 1);
                    piece = ring + (stage % P::kStages) * P::kBytes;
                    ++stage;
                } else {
                    piece += 2 * P::kBlockBytes;
                }
            };
            if constexpr (kMine > 0) {
                auto get_k = [&](int h, int i) { return load_words<S::kWords>(piece + h * P::kBlockBytes + read_k + i * kNextK); };
                auto get_v = [&](int h, int i) { return load_words<S::kWords>(piece + h * P::kBlockBytes + P::kCodes + read_v + i * kNextV); };
                auto get_scales = [&](int h, float4_t& s, float4_t& t) {
                    s = *reinterpret_cast<const float4_t*>(piece + h * P::kBlockBytes + 2 * P::kCodes + quarter * 16);
                    t = *reinterpret_cast<const float4_t*>(piece + h * P::kBlockBytes + 2 * P::kCodes + 64 + quarter * 16);
                };
                // keys that all rows see, then the others
                auto keys = [&](auto masked, uint32_t end) {
#pragma unroll 1
                    for (; key < end; key += 32) {
                        begin(key);
                        rows.template step<decltype(masked)::value>(x, key, quarter, get_k, get_v, get_scales, [] {});
                    }
                };
                keys(std::false_type{}, min(x.key1, x.all_see & ~31u));
                keys(std::true_type{}, x.key1);
            } else {
                for (; key < x.key1; key += P::kKeys) begin(key);
            }
            if constexpr (kMine > 0) {
                Args& out = kernel_args();
                const uint32_t share = own_share(out);
#pragma unroll
                for (int r = 0; r < kMine; ++r) {
                    const uint32_t row = (wave + kWaves * r) * 16 + col;
                    const float l = sum_quarters(rows.l[r]);
                    const float factor = l == 0.0f ? 0.0f : 1.0f / l;
                    if (row < x.rows) {
#pragma unroll
                        for (int c = 0; c < S::kLoads; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float v[S::kWords];
#pragma unroll
                                for (int w = 0; w < S::kWords; ++w) v[w] = rows.o[r][c * S::kWords + w][i] * factor;
                                put<D, S::kWords>(out, x, share, row, c * S::kChunk + (quarter * 4 + i) * S::kWords, v);
                            }
                        if (quarter == 0) put_lse(out, x, share, row, rows.reference(r), l);
                    }
                }
            }
        };
        if (R == 2 && tiles > wave + kWaves) loop(std::integral_constant<int, R>{});
        else if (tiles > wave) loop(std::integral_constant<int, 1>{});
        else loop(std::integral_constant<int, 0>{});
        arrive<0>();                                               // before the next segment's copies
    });
}

// ---- launches ---------------------------------------------------------------------------------------------------------

template <int D, int CODES, int PARTS> int start_attention(const AttentionArgs& a, const AttentionPlan& p, void* stream, Launched& info) {
    const dim3 grid = p.shares() == 0 ? dim3(a.cache.kv_heads, p.row_blocks, a.batch) : dim3(p.shares(), 1, 1), block(kWaves * 64);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    info = {p.split_rows ? "tree_attention_rows" : "tree_attention", {grid.x, grid.y, grid.z}, {block.x, 1, 1},
            p.split_rows ? uint32_t(Stage<D>::kStages * Stage<D>::kBytes) : uint32_t((kWaves * 16 * (D + 4 + 2) + 32) * 4)};
    if constexpr (D <= 128) {
        if (p.tiles == 2) {
            if (p.split_rows) k_split_rows<D, CODES, 2, PARTS><<<grid, block, 0, s>>>(a);
            else k_split_keys<D, CODES, 2, PARTS><<<grid, block, 0, s>>>(a);
            return int(hipGetLastError());
        }
    }
    if (p.split_rows) k_split_rows<D, CODES, 1, PARTS><<<grid, block, 0, s>>>(a);
    else k_split_keys<D, CODES, 1, PARTS><<<grid, block, 0, s>>>(a);
    return int(hipGetLastError());
}

template <int D, int CODES> int start_attention(const AttentionArgs& a, const AttentionPlan& p, void* stream, Launched& info) {
    if constexpr (kCodeProducts<D, CODES>) {
        if (a.type == FKLHIP_F16) return start_attention<D, CODES, 3>(a, p, stream, info);
        return start_attention<D, CODES, 2>(a, p, stream, info);
    } else {
        return start_attention<D, CODES, 0>(a, p, stream, info);
    }
}

template <int D> int launch_attention(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) {
    if (a.cache.codes == FKLHIP_CODES_INT8) return start_attention<D, FKLHIP_CODES_INT8>(a, plan, stream, info);
    return start_attention<D, FKLHIP_CODES_E4M3>(a, plan, stream, info);
}

} // namespace fkattn
