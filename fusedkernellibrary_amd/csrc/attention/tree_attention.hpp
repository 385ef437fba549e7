// tree_attention.hpp -- attention of a few new tokens per sequence over a quantised, paged cache.
//
// Mathematics. For the rows r of a key head (its query heads times the sequence's new tokens) and the keys j a row sees:
//   s_rj = scale * ks_j * (q_r . kc_j),   o_r = sum_j e^(s_rj - m_r) vs_j vc_j / sum_j e^(s_rj - m_r)
// with kc, vc the cache's codes and ks, vs their scales. The products run on the codes, as they are or exactly in half precision,
// and the scales enter as one factor per key: ks on the scores, vs on the weights. A query row is brought to a common size by a
// power of two, which is exact, and held as a sum of 8-bit codes (kCodeProducts) or in half precision. Weights are rounded to half precision, and
// values are exact in it (int8: 8 bits, e4m3: 4 bits of 11); all sums are in 32 bits.
//
// One pass over the keys, 32 at a time, everything in registers: S^T = K Q^T comes out of the matrix unit with a query row to
// a lane column (lane % 16) and four keys to each of its four quarters (lane / 16), and O^T = V^T P^T wants its weights just
// so if the contraction runs over the keys in that order; the cache keeps four tokens' bytes of a value element side by
// side for that reason. So nothing moves between lanes, and the running maximum is per lane column.
//
// A workgroup takes R tiles of 16 rows of a key head, and its waves other keys of the same segment, 32 in turn; the waves' sums
// are joined in LDS at the end. R is 1, 2 or 4: a key's loads and scales, and a value's conversion, serve all R. One tile's queries
// stay in registers; more are in LDS, as their sums take the registers. Four tiles of 128 elements are 128 registers of
// sums, which leaves two waves to a SIMD.
//
// What bounds it (times by kernel of a profile). One tile: reading the cache. 64 sequences with 900 to 8191 keys (8 key heads of 128,
// int8, 616 MB) take 114 us and 5.8 for joining, 5.4 TB/s; 48 with 4000 to 32700 (e4m3, 1.86 GB) 326 and 8.4 us, 5.7 TB/s; a kernel
// that only reads reaches 6.3. Four tiles: waits, with two waves to a SIMD to fill them. 16 trees of up to 61 tokens over 500 to 4100
// keys (e4m3, 25.9 Gflop) take 67 us and 9.4 for joining, where the products alone are 22 at the rate of a large matrix product:
// a wave's time is 40 % waits for memory and LDS, 21 % waits to issue, 28 % vector instructions (38 and 8 exponentials for a tile and
// 32 keys: one scaling, one fused subtraction, one exponential, one value scale, one sum and half a comparison per score, besides
// conversions); the matrix unit is busy a fifth of it. Each tile waits for what it reads from LDS: its queries, or, where the next
// tile's are read ahead, its scales behind those. 131003 keys with 56 rows (int8, 277 MB) take 68 and 6.8 us, where reading is 44, with the same shares. What was tried
// on four tiles: workgroups side by side that share a unit's keys in the L2 cache (no faster per key, and slower for trees that
// leave some of them without rows), and a touch of the lines two steps ahead (88 us for 68). Two parts of int8 queries are read from
// LDS in front of the weights of the tile before theirs (1.5 us of 64).
//
// How the work is dealt out. The device alone knows the sequences' lengths, so every workgroup adds them up: the keys of all
// (sequence, key head, block of rows), one behind the other, are cut into equal shares, one to a workgroup, all of which run
// at the same time. A share may hold parts of two of them and whole ones in between; whole ones are written to the output,
// parts to the workspace, from where the kernels of merge.hip take them. Without shares (short sequences, or so many that the
// order of launch evens them out) a workgroup takes one whole (sequence, key head, block of rows). plan_attention chooses.
//
// Shaped scores are taken from the last keys to the first: a bias by distance has them rise towards the row, and the reference
// would have to move in every step (16 trees of up to 13 behind windows of 4096, 32 and 8 heads, e4m3, four tiles: 68 us that way, 50 this;
// with two tiles 46, with three workgroups of them to a compute unit 42, and 6 for joining, where reading the 138 MB takes 22: vector instructions
// 44 % of the time, waits the rest). A cap costs five of those a score, two of them at a quarter of the rate: 64 sequences with 900 to 8191
// keys take 115 us, as without one, and a chunk of 2048 tokens in three documents 75 us a pass, vector instructions for 66 % of it (products
// alone: 19). There blocks of rows begin by how many keys they see, most first: with four tiles 77.2, and 85.7 in their order.
// A workgroup of 128 rows with keys as halves in LDS, double buffered, took 123 us for it: all blocks are resident at once, the heaviest ends alone.
//
// The running maximum is a reference m_r and not the exact maximum: weights are w = 2^(s - m) * vs, sums those of 2^(s - m), and
// m moves only when a weight exceeds 2^kLead. Only then are scores compared across lanes and the sums rescaled. The largest
// weight starts at 2^kStart, so one is subnormal in half precision (below 2^-14) only 2^-(14 + kStart) below the largest of
// the first keys. (Value scales below kLeastScale count as that: values of 10^-22 and less lose accuracy.)
#pragma once

#include "work_shares.hpp"

namespace fkattn {

constexpr float kStart = 6.0f, kLead = 14.0f, kLargest = 16384.0f, kLeastScale = 0x1p-80f, kMostSum = 0x1p98f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNothing = -1.0e30f;         // the reference of a row that has seen no key

// How a key's product with the queries is taken. int8, runs of 64 elements: the matrix unit has products of the codes themselves
// whose sums are whole numbers of 32 bits; a query row is then a sum of two or three rows of codes, and no key is converted: in
// fixed point, 256 * hi + lo (bfloat16: exact for elements from 2^-7 of the row's largest on) or with a third part behind them (half
// precision: exact from 2^-11 on); smaller elements are off by 2^-15 (2^-22) of the largest.
// Everything else: keys as halves, which hold their codes exactly, and sums in 32 bits. The matrix unit has products of e4m3 codes as
// well, at a higher rate, but what it adds up of one instruction it cuts off 2^-13 below the largest product: next to one large
// element of query and key others were lost (2^16 and 2^2 made 2^16; scores were off by up to 2^-12.5 of their largest product, and
// are by 2^-22). That form took 67 us for trees of up to 61 (70 now), 57.5 for the step of trees in half precision (56.3).
template <int D, int CODES> constexpr bool kCodeProducts = code_products(D, CODES);

using int2_t = int __attribute__((ext_vector_type(2)));
using int4_t = int __attribute__((ext_vector_type(4)));

template <int D> struct Shape {
    static constexpr int kChunk = D % 64 == 0 ? 64 : 32;   // elements of a row that one load of a lane's quarter row covers
    static constexpr int kLoads = D / kChunk;              // of a block of 16 keys (or values)
    static constexpr int kWords = kChunk / 16;             // dwords of such a load: 4 or 2
    static constexpr int kSteps = D / 32;                  // of the matrix unit over a row
    static constexpr int kTiles = D / 16;                  // of 16 output elements
};

template <int WORDS> struct Words { uint32_t w[WORDS]; };

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

// The larger of a lane column's four quarters (lanes l, l ^ 16, l ^ 32, l ^ 48), and their sum: rows of sixteen lanes, then
// halves of the wave change places.
template <typename F> __device__ __forceinline__ float join_quarters(float v, F f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, uint32_t(rows[0])), __builtin_bit_cast(float, uint32_t(rows[1]))));
    const auto halves = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return f(__builtin_bit_cast(float, uint32_t(halves[0])), __builtin_bit_cast(float, uint32_t(halves[1])));
}
__device__ __forceinline__ float max_quarters(float v) { return join_quarters(v, [](float a, float b) { return __builtin_fmaxf(a, b); }); }
__device__ __forceinline__ float sum_quarters(float v) { return join_quarters(v, [](float a, float b) { return a + b; }); }

// The lowest n of four bits.
__device__ __forceinline__ uint32_t lowest_bits(int32_t n) { return n >= 4 ? 15u : n <= 0 ? 0u : (1u << n) - 1u; }
// Bits u .. u + 3 of a row of a mask, where those below 0 (the context's) are set and those behind the row are not; `first` is
// the row's first word.
template <bool HALVES> __device__ __forceinline__ uint32_t mask_bits(const uint64_t* row, uint64_t first, uint32_t words, int32_t u) {
    const uint32_t below = u >= 0 ? 0u : u <= -4 ? 4u : uint32_t(-u), from = u >= 0 ? uint32_t(u) : 0u;
    uint64_t lo = from < 64u ? first : 0, hi = 0;
    if (words > 1) {                                          // (the same for the whole wave)
        const uint32_t lo_at = from >> 6, hi_at = (from + 3) >> 6;
        lo = lo_at < words ? row[lo_at] : 0;
        hi = hi_at < words && hi_at != lo_at ? row[hi_at] : 0;
    }
    uint32_t bits;
    if constexpr (HALVES) {
        // By halves: a vector shift of 64 bits whose amount is in the last register that a wave has (v255 of 256, v167 of 168) shifts by
        // something else now and then. (Where shifts of 64 bits are taken, the build refuses a kernel with one of that kind; by halves,
        // heads of 256 elements take more registers than there are.)
        const uint32_t at = from & 32u ? uint32_t(lo >> 32) : uint32_t(lo), next = from & 32u ? uint32_t(hi) : uint32_t(lo >> 32);
        bits = __builtin_amdgcn_alignbit(next, at, from & 31u);
    } else {
        const uint32_t shift = from & 63u;
        bits = uint32_t(lo >> shift) | (shift ? uint32_t(hi << (64u - shift)) : 0u);
    }
    return (lowest_bits(int32_t(below)) | bits << below) & 15u;
}

// The place of the first key that a token's rows see.
__device__ __forceinline__ uint32_t first_of(Args& a, const Sequence& s, uint32_t token) {
    const int32_t first = shaped(a).first[s.first_token + token];
    return max(s.front, first < 0 ? 0u : min(uint32_t(first), s.total));
}

// What up to 64 rows of a sequence see: none a key in front of `from` or behind any_sees, all those from all_from to all_see. (Shaped.)
struct Sight { uint32_t from, all_from, all_see, any_sees; };
__device__ __forceinline__ Sight sight_of(Args& a, const Sequence& s, uint32_t b, uint32_t row0, uint32_t rows) {
    Shaped& h = shaped(a);
    const bool causal = a.mask == nullptr;
    Sight x{s.front, s.front, causal ? min(s.context + divide(row0, a.group_magic) + 1, s.total) : s.context, causal ? min(s.context + divide(row0 + rows - 1, a.group_magic) + 1, s.total) : s.total};
    if (causal && h.prefix) {
        const int32_t prefix = scalar(h.prefix + b);
        const uint32_t upto = prefix < 0 ? 0u : min(uint32_t(prefix), s.total);
        x.any_sees = max(x.any_sees, upto);
        x.all_see = max(x.all_see, upto);
    }
    if (h.first) {
        // (a row to a lane)
        const uint32_t first = first_of(a, s, divide(row0 + min(thread_here() & 63, rows - 1), a.group_magic));
        const uint32_t low = reduce_lanes<32>(first, [](uint32_t a, uint32_t b) { return a < b ? a : b; }), high = max_lanes<32>(first);
        x.from = min(__builtin_amdgcn_readlane(low, 0), __builtin_amdgcn_readlane(low, 32));
        x.all_from = max(__builtin_amdgcn_readlane(high, 0), __builtin_amdgcn_readlane(high, 32));
    }
    return x;
}

// Keys key0 .. key1 of row block `block` and key head `head` of a sequence; where its parts go.
struct Segment {
    Sequence seq;
    uint32_t b, head, row0, rows;        // rows row0 .. row0 + rows of the sequence's
    uint32_t key0, key1, all_see;        // every row sees the keys in front of all_see
    int part;                            // -1: whole, 0 or 1: the share's part
    uint32_t behind, quarter;            // keys of the share behind the segment's, and a quarter of them all
    uint32_t all_from = 0;               // every row may see the keys from there on (shaped)
};
template <bool SHAPED> __device__ __forceinline__ Segment segment_of(Args& a, const Sequence& s, uint32_t b, uint32_t head, uint32_t block, uint32_t k0, uint32_t k1, int part) {
    Segment x;
    x.seq = s; x.b = b; x.head = head; x.part = part;
    x.row0 = block * a.unit_rows;
    x.rows = min(a.unit_rows, s.rows - x.row0);
    if constexpr (SHAPED) {
        const Sight sight = sight_of(a, s, b, x.row0, x.rows);
        x.all_see = sight.all_see;
        x.all_from = sight.all_from;
        x.key0 = (k0 + s.skip) << a.granule_log;
        x.key1 = min((k1 + s.skip) << a.granule_log, sight.any_sees);
        x.key0 = min(max(x.key0, sight.from & ~31u), max(x.key0, x.key1));
    } else {
        const bool causal = a.mask == nullptr;
        const uint32_t any_sees = causal ? min(s.context + divide(x.row0 + x.rows - 1, a.group_magic) + 1, s.total) : s.total;
        x.all_see = causal ? min(s.context + divide(x.row0, a.group_magic) + 1, s.total) : s.context;
        x.key0 = k0 << a.granule_log;
        x.key1 = min(k1 << a.granule_log, any_sees);
    }
    return x;
}

// Rows of the result that are of no sequence, in front of the first, above max_new or behind the last: zeros, as where a row sees
// nothing. Those behind sequence b's, which end at `end`, and in front of the first's, one key head's. (With shares the kernels of
// merge.hip, which come to every row, see to it.)
template <int D, int THREADS> __device__ __forceinline__ void clear_rows(Args& a, const Sequence& s, uint32_t b, uint32_t head, int32_t end) {
    const uint32_t front = b == 0 ? s.first_token : 0u, behind = s.first_token + s.fresh;
    const uint32_t upto = b + 1 == a.batch ? a.tokens : end < 0 ? 0u : min(uint32_t(end), a.tokens);
    if (__builtin_expect(front == 0 && upto <= behind, 1)) return;
    const auto clear = [&](uint32_t token) {
        char* to = a.out.data + int64_t(token) * a.out.token_stride + int64_t(head * a.group) * a.out.head_stride;
        for (uint32_t i = threadIdx.x; i < a.group * (D / 8); i += THREADS)
            *reinterpret_cast<uint4_t*>(to + int64_t(i / (D / 8)) * a.out.head_stride + i % (D / 8) * 16) = uint4_t{0, 0, 0, 0};
        if (a.lse)
            for (uint32_t i = threadIdx.x; i < a.group; i += THREADS) a.lse[size_t(token) * a.q_heads + head * a.group + i] = -__builtin_inff();
    };
    for (uint32_t token = 0; token < front; ++token) clear(token);
    for (uint32_t token = behind; token < upto; ++token) clear(token);
}

// The block of a sequence's rows that is nth by how many keys it sees, most first; up to 256 blocks. Windows, documents and prefixes
// have blocks of all weights in any order, and one with many keys that begins last ends alone.
__device__ __forceinline__ uint32_t nth_heaviest(Args& a, const Sequence& s, uint32_t b, uint32_t blocks, uint32_t nth, uint32_t lane) {
    Shaped& h = shaped(a);
    uint32_t prefix = 0;
    if (h.prefix && !a.mask) {
        const int32_t upto = scalar(h.prefix + b);
        prefix = upto < 0 ? 0u : min(uint32_t(upto), s.total);
    }
    uint32_t weight[4];                                        // of blocks lane, lane + 64 ..: in units of 128 keys, from 1 on
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t block = k * 64 + lane, row0 = block * a.unit_rows;
        weight[k] = 0;
        if (block < blocks) {
            const uint32_t last = divide(min(row0 + a.unit_rows, s.rows) - 1, a.group_magic);
            const uint32_t from = h.first ? first_of(a, s, divide(row0, a.group_magic)) : 0u, upto = a.mask ? s.total : max(min(s.context + last + 1, s.total), prefix);
            weight[k] = 1 + (upto > from ? (upto - from) >> 7 : 0u);
        }
    }
    // the largest weight that more than nth blocks have or exceed, and which of those that have it
    const auto having = [&](uint32_t w) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) n += __builtin_popcountll(__ballot(weight[k] >= w));
        return n;
    };
    uint32_t its = 0;
    for (uint32_t bit = 1u << (32 - __builtin_clz((s.total >> 7) + 1)); bit; bit >>= 1)
        if (having(its | bit) > nth) its |= bit;
    uint32_t left = nth - having(its + 1), found = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        uint64_t same = __ballot(weight[k] == its);
        const uint32_t n = __builtin_popcountll(same);
        if (left < n) {
            for (; left; --left) same &= same - 1;
            found = k * 64 + __builtin_ctzll(same);
            left = 0xffffffffu;
        } else if (left != 0xffffffffu) {
            left -= n;
        }
    }
    return found;
}

// Calls `run` for every segment of the workgroup. `kept` is the wave's place in LDS for what the walk goes on with: a segment
// needs all registers.
template <int D, int THREADS, bool SHAPED, typename F> __device__ __forceinline__ void walk(Args& a, uint32_t lane, uint32_t* kept, F run) {
    // granules at .. end of all are the share's, `in` of b's are in front of them; without shares: (sequence, head, block) of the grid
    uint32_t b = blockIdx.z, in = 0, at = 0, end = 1;
    const bool shared = a.share_odd != 0;
    Sequence s;
    if (shared) {
        const uint32_t share = own_share(a);
        const Found f = find<SHAPED>(a, lane, [&](uint32_t all, const Sequence&, uint32_t, uint32_t upto) { return upto > share_begin(a, all, share); });
        at = share_begin(a, f.all, share);
        end = share_begin(a, f.all, share + 1);
        b = f.b;
        in = at - f.before;
        s = f.s;
    } else {
        const int32_t rows_end = scalar(a.q_start + b + 1);
        s = sequence_of(a, scalar(a.q_start + b), rows_end, scalar(a.context + b));
        if constexpr (SHAPED)
            if (shaped(a).first && s.fresh) skip_front(a, s, scalar(shaped(a).first + s.first_token));
        if (blockIdx.y == 0) clear_rows<D, THREADS>(a, s, b, blockIdx.x, rows_end);
    }
    uint32_t whole = end - at;
    while (at < end && b < kernel_args().batch) {
        Args& a = kernel_args();
        const uint32_t n = granules_of(a, s), blocks = blocks_of(a, s);
        // (the last rows of a causal sequence see most: they begin first)
        uint32_t head = blockIdx.x, block = gridDim.y - 1 - blockIdx.y, g = 0, count = n;
        int part = -1;
        if (shared) {
            const uint32_t unit = n ? in / n : 0;
            if (unit >= blocks * a.cache.kv_heads || n == 0) {
                in = 0;
                if (++b < a.batch) s = sequence_at<SHAPED>(a, b);
                continue;
            }
            head = unit / blocks;
            block = unit - head * blocks;
            g = in - unit * n;
            count = min(n - g, end - at);
            part = g > a.lead ? 0 : g + count == n ? -1 : 1;
        } else if (block >= blocks) {
            return;
        } else if constexpr (SHAPED) {
            // (a sequence's rows may be fewer than the grid's: its own blocks are the last of the grid's rows)
            if ((shaped(a).first || shaped(a).prefix) && blocks > 1 && blocks <= 256) block = nth_heaviest(a, s, b, blocks, blocks - 1 - block, lane);
        }
        kept[0] = at + count; kept[1] = in + count; kept[2] = end; kept[3] = b; kept[4] = whole;
        Segment x = segment_of<SHAPED>(a, s, b, head, block, max(g, a.lead) - a.lead, max(g + count, a.lead) - a.lead, part);
        x.quarter = whole << a.granule_log >> 2;
        x.behind = (end - at - count) << a.granule_log;
        if (!shared) x.behind = 0, x.quarter = (SHAPED && x.key1 < x.key0 ? 0 : x.key1 - x.key0) >> 2;
        if (!shared || g + count > a.lead) run(x);            // (else there is nothing but a block's beginning)
        if (!shared) return;
        at = __builtin_amdgcn_readfirstlane(kept[0]); in = __builtin_amdgcn_readfirstlane(kept[1]); end = __builtin_amdgcn_readfirstlane(kept[2]);
        b = __builtin_amdgcn_readfirstlane(kept[3]); whole = __builtin_amdgcn_readfirstlane(kept[4]);
        s = sequence_at<SHAPED>(kernel_args(), b);
    }
}

// A wave's priority falls as its share gets done: left alone, the oldest of the workgroups on a compute unit runs ahead, and the
// last one ends alone, without others to fill its gaps.
template <bool DOWN> __device__ __forceinline__ void set_priority(const Segment& x, uint32_t key) {
    const uint32_t left = x.behind + (DOWN ? key - x.key0 : x.key1 - key);
    if (left > 3 * x.quarter) __builtin_amdgcn_s_setprio(3);
    else if (left > 2 * x.quarter) __builtin_amdgcn_s_setprio(2);
    else if (left > x.quarter) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

// ---- query rows ------------------------------------------------------------------------------------------------------

// Row `row` of a segment; those behind its last are its last again.
struct RowPlace { uint32_t token, head; };
__device__ __forceinline__ RowPlace place_of_row(Args& a, const Segment& x, uint32_t row) {
    const uint32_t at = x.row0 + min(row, x.rows - 1), token = divide(at, a.group_magic);
    return {token, x.head * a.group + at - token * a.group};
}

// A lane's quarter of a query row as the products want it (halves, or PARTS rows of codes one behind the other), and what its
// scores have to be multiplied with to be in units of log2.
template <int D, int PARTS> constexpr int kQueryRegs = PARTS == 0 ? D / 8 : PARTS * D / 16;
template <int D> __device__ __forceinline__ void load_query(Args& a, const Segment& x, uint32_t row, uint32_t quarter, uint4_t (&raw)[D / 32]) {
    const RowPlace place = place_of_row(a, x, row);
    const char* from = a.q.data + int64_t(x.seq.first_token + place.token) * a.q.token_stride + int64_t(place.head) * a.q.head_stride;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        // the elements that the quarter's codes of this step are of: kChunk / 4 neighbours of each run of kChunk
        const uint32_t at = Shape<D>::kChunk == 64 ? (s / 2) * 64 + quarter * 16 + (s % 2) * 8 : s * 32 + quarter * 8;
        raw[s] = *reinterpret_cast<const uint4_t*>(from + at * 2);
    }
}
template <int D, int PARTS> __device__ __forceinline__ float prepare_query(Args& a, const uint4_t (&raw)[D / 32], uint32_t (&q)[kQueryRegs<D, PARTS>]) {
    using S = Shape<D>;
    float e[S::kSteps * 8];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (a.type == FKLHIP_BF16) unpack2<FKLHIP_BF16>(raw[s][k], e[s * 8 + 2 * k], e[s * 8 + 2 * k + 1]);
            else unpack2<FKLHIP_F16>(raw[s][k], e[s * 8 + 2 * k], e[s * 8 + 2 * k + 1]);
        }
#pragma unroll
    for (int k = 0; k < S::kSteps * 8; ++k) top = max(top, __builtin_bit_cast(uint32_t, e[k]) & 0x7fffffffu);
    top = max(top, uint32_t(__shfl_xor(int(top), 16)));
    top = max(top, uint32_t(__shfl_xor(int(top), 32)));
    // a power of two in front of the row's largest magnitude (a row of zeros, or with an infinity, is left alone)
    const bool plain = top == 0 || top >= 0x7f800000u;
    const int p = plain ? 0 : __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, top)) - 1;
    // (a negative scale turns the queries round: scores are multiplied with what is above 0)
    float unit = __builtin_fabsf(a.scale) * kLog2e;
    if (a.scale < 0.0f)
#pragma unroll
        for (int k = 0; k < S::kSteps * 8; ++k) e[k] = -e[k];
    if constexpr (PARTS == 0) {
#pragma unroll
        for (int k = 0; k < S::kSteps * 4; ++k)
            q[k] = pack2<FKLHIP_F16>(__builtin_amdgcn_ldexpf(e[2 * k], -p), __builtin_amdgcn_ldexpf(e[2 * k + 1], -p));
        // (as with codes: an infinity makes NaN of its row's scores, not an infinity of either sign)
        unit = top >= 0x7f800000u ? __builtin_nanf("") : unit;
    } else {
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
            for (int part = 0; part < PARTS; ++part) q[part * S::kSteps * 2 + k] = w[part];
        }
    }
    unit = __builtin_amdgcn_ldexpf(unit, p);
    return unit < 1.0e-37f ? 1.0e-37f : unit;                      // (above 0, as masked scores are -inf; NaN stays)
}

// ---- 32 keys ---------------------------------------------------------------------------------------------------------

// What a wave has summed up for its rows: R tiles of 16, one to a lane column; a quarter of each sum.
template <int D, int CODES, int R, int PARTS> struct Sums {
    using S = Shape<D>;
    float4_t o[R][S::kTiles];
    float m[R], l[R];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) o[r][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            m[r] = kNothing;                                        // (which the first key that a row sees leads by more than kLead)
            l[r] = 0.0f;
        }
    }

    // Products of two blocks of 16 keys with a tile's rows, four keys of each to a quarter; the codes' scales are not in them.
    template <typename K, typename Q> __device__ __forceinline__ void products(K get_k, Q get_q, float4_t (&y)[2]) {
        if constexpr (PARTS == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) y[h] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Words<S::kWords> w = get_k(h, i);
#pragma unroll
                    for (int k = 0; k < S::kWords / 2; ++k)
                        y[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves8<CODES>(w.w[2 * k], w.w[2 * k + 1]), __builtin_bit_cast(half8_t, get_q(i * (S::kWords / 2) + k)), y[h], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);                  // (all codes at once as halves would take 32 registers)
            }
        } else {
            // the first two parts as one whole number, the third by itself: with it, 32 bits would not do
            int4_t sum[PARTS - 1][2];
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) {
                    const int4_t row = __builtin_bit_cast(int4_t, get_q(part * S::kLoads + i));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const Words<S::kWords> w = get_k(h, i);
                        int4_t& to = sum[part < 2 ? 0 : 1][h];
                        const int4_t before = i > 0 ? to : part == 1 ? to << 8 : int4_t{0, 0, 0, 0};
                        to = __builtin_amdgcn_mfma_i32_16x16x64_i8(int4_t{int(w.w[0]), int(w.w[1]), int(w.w[2]), int(w.w[3])}, row, before, 0, 0, 0);
                    }
                    if constexpr (PARTS == 3) __builtin_amdgcn_sched_barrier(0);    // (one part's registers at a time)
                }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[h][i] = float(sum[0][h][i]);
                    if constexpr (PARTS == 3) y[h][i] = __builtin_fmaf(y[h][i], 256.0f, float(sum[1][h][i]));
                }
        }
    }

    // The same of all tiles.
    template <typename K, typename Q> __device__ __forceinline__ void products_of_all(K get_k, Q get_q, float4_t (&y)[R][2]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) y[r][h] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
            for (int k = 0; k < S::kWords / 2; ++k) {
                half8_t a[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Words<S::kWords> w = get_k(h, i);
                    a[h] = halves8<CODES>(w.w[2 * k], w.w[2 * k + 1]);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const half8_t q = __builtin_bit_cast(half8_t, get_q(r, i * (S::kWords / 2) + k));
#pragma unroll
                    for (int h = 0; h < 2; ++h) y[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[h], q, y[r][h], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
    }

    // 32 keys: get_k(block, load) and get_v have their codes, get_k_scales and get_v_scales the scales of the quarter's four keys of each
    // block, get_q(tile, run) the queries, get_unit(tile) what their scores are multiplied with. after_scores runs when the
    // keys are used up. Where `masked`, sees(tile, block) has a bit for each of the quarter's four keys that the lane's row
    // sees, and hide() clears the values that are no token's. (The masked way is a branch around the scores and no second copy
    // of the loop: between two loops the sums would be held twice.)
    // shape(block, row's slope and place, scores) makes products with the queries, multiplied with their unit, what the scores are;
    // std::nullptr_t: they are. get_unit has slope and place behind the unit then.
    template <typename K, typename V, typename Q, typename U, typename G, typename W, typename T, typename M, typename H, typename A>
    __device__ __forceinline__ void step(bool masked, K get_k, V get_v, Q get_q, U get_unit, G get_k_scales, W get_v_scales, T shape, M sees, H hide, A after_scores) {
        constexpr bool kShaped = !std::is_same_v<T, std::nullptr_t>;
        half8_t p[R];
        float4_t y[2], next[2];
        // The matrix unit works on the next tile's scores while this one's weights are taken. (Four tiles of 128 elements take all registers
        // without that if queries have three parts or keys are converted: trees of up to 61 took 73 us with it, and 70 without.)
        constexpr int kRuns = kQueryRegs<D, PARTS> / 4, kProducts = 2 * PARTS * S::kLoads;
        // Shaped, keys that are converted: all tiles' products first, so that the next keys are asked for sooner (2048 tokens of a prompt 77.1 us, 77.8
        // tile by tile; 16 trees of 33 to 61 78.8, 80 to 84; as many vector instructions, and 23 registers fewer for two tiles of 128 elements).
        constexpr bool kTogether = kShaped && PARTS == 0 && R > 1;
        constexpr bool kAhead = !kTogether && !(R == 4 && (PARTS == 3 || (D == 128 && (PARTS == 0 || kShaped))));
        constexpr bool kHeld = R < 4 || kRuns <= 4;
        uint4_t q[kRuns];
        auto ask_q = [&](int r) {
#pragma unroll
            for (int run = 0; run < kRuns; ++run) q[run] = get_q(r, run);
        };
        if (kAhead) products(get_k, [&](int run) { return get_q(0, run); }, y);
        if (R == 1) after_scores();
        float4_t all[kTogether ? R : 1][2];
        if constexpr (kTogether) {
            products_of_all(get_k, get_q, all);
            after_scores();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (kTogether) {
                y[0] = all[r][0];
                y[1] = all[r][1];
            }
            if (!kAhead && !kTogether) products(get_k, [&](int run) { return get_q(r, run); }, y);
            if (!kAhead && !kTogether && r + 1 == R) after_scores();
            if (kAhead && kHeld && r + 1 < R) ask_q(r + 1);
            float unit;
            float2_t bias = {0.0f, 0.0f};
            if constexpr (kShaped) {
                const float4_t its = get_unit(r);
                unit = its[0];
                bias = float2_t{its[1], its[2]};
            } else {
                unit = get_unit(r);
            }
            float4_t ks[2], vs[2];
            get_k_scales(ks);
            if constexpr (!kShaped) get_v_scales(vs);
#pragma unroll
            for (int h = 0; h < 2; ++h) y[h] *= ks[h];
            if constexpr (kShaped) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    y[h] *= unit;
                    shape(h, bias, y[h]);
                    if constexpr (R == 4 || (R == 2 && D == 256)) __builtin_amdgcn_sched_barrier(0);    // (both blocks' at once take more registers than there are)
                }
                unit = 1.0f;
                get_v_scales(vs);
            }
            if (__builtin_expect(masked, 0)) {
                uint32_t some = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t seen = sees(r, h);
                    some |= seen;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[h][i] = seen >> i & 1 ? y[h][i] : -__builtin_inff();
                        vs[h][i] = seen >> i & 1 ? vs[h][i] : 0.0f;          // (a hidden value's scale may be NaN)
                    }
                }
                // (of a row with an infinity or a NaN the unit is NaN, and -inf times that would be no score of a hidden key)
                unit = some ? unit : 1.0f;
            }
            if (kAhead && r + 1 < R) products(get_k, [&](int run) { return kHeld ? q[run] : get_q(r + 1, run); }, next);
            // Weights, and a look at whether the reference has to move: where a weight is too large for half precision.
            float w[2][4], sum = 0.0f, top = 0.0f;
            auto weigh = [&](int h, int i, float score) {
                const float e = exp2_fast(score);
                w[h][i] = e * vs[h][i];
                sum += e;
            };
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    weigh(h, i, __builtin_fmaf(y[h][i], unit, -m[r]));
                    top = __builtin_fmaxf(top, w[h][i]);
                }
            if constexpr (kAhead && R > 1 && PARTS > 0) {
                // one product of the next tile, then a share of this one's weights, again and again
#pragma unroll
                for (int i = 0; i < kProducts; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 40 / kProducts, 0);
                }
            }
            if (kAhead && r + 2 == R) after_scores();
            if (__builtin_expect(__any(top > kLargest || sum > kMostSum), 0)) {
                // the largest weight there would be, in units of log2
                top = -__builtin_inff();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        top = __builtin_fmaxf(top, y[h][i] * unit + __builtin_amdgcn_logf(__builtin_fmaxf(vs[h][i], kLeastScale)));
                top = max_quarters(top);
                float alpha = 1.0f;
                if (top - m[r] > kLead) {
                    alpha = exp2_fast(m[r] + kStart - top);
                    m[r] = top - kStart;
                }
                l[r] *= alpha;
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) o[r][i] *= alpha;
                // (from the rounded scores: those of 2^100 differ from their reference by more than an exponent holds)
                sum = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) weigh(h, i, y[h][i] * unit - m[r]);
            }
            l[r] += sum;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i) p[r][h * 4 + i] = _Float16(w[h][i]);
                if (kAhead && r + 1 < R) y[h] = next[h];
            }
            if constexpr (R > 1) __builtin_amdgcn_sched_barrier(0);     // (more tiles' scores at once take more registers than there are)
        }
        if (__builtin_expect(masked, 0)) hide();
#pragma unroll
        for (int c = 0; c < S::kLoads; ++c) {
            const Words<S::kWords> v0 = get_v(0, c), v1 = get_v(1, c);
#pragma unroll
            for (int k = 0; k < S::kWords; ++k) {
                // tile c * kWords + k: elements c * kChunk + column * kWords + k
                const half8_t v = halves8<CODES>(v0.w[k], v1.w[k]);
#pragma unroll
                for (int r = 0; r < R; ++r) o[r][c * S::kWords + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[r], o[r][c * S::kWords + k], 0, 0, 0);
            }
            if constexpr (R > 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// Four neighbouring elements of a row of the result.
__device__ __forceinline__ void put4(Args& a, const Segment& x, uint32_t row, uint32_t d, float4_t v) {
    const uint32_t tok = divide(x.row0 + row, a.group_magic), qh = x.head * a.group + x.row0 + row - tok * a.group;
    const uint2_t w = a.type == FKLHIP_BF16 ? uint2_t{pack2<FKLHIP_BF16>(v[0], v[1]), pack2<FKLHIP_BF16>(v[2], v[3])}
                                            : uint2_t{pack2<FKLHIP_F16>(v[0], v[1]), pack2<FKLHIP_F16>(v[2], v[3])};
    *reinterpret_cast<uint2_t*>(a.out.data + int64_t(x.seq.first_token + tok) * a.out.token_stride + int64_t(qh) * a.out.head_stride + d * 2) = w;
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

// Loads from an address that is the same for the whole wave, in scalar registers, and 32 bits of the lane's.
using Global = const __attribute__((address_space(1))) char*;
__device__ __forceinline__ Global of_wave(const void* p) {
    uint64_t v = reinterpret_cast<uint64_t>(p);
    asm volatile("" : "+s"(v));
    return (Global)v;
}
template <typename T> __device__ __forceinline__ T load_at(Global base, uint32_t lane_part) { return *(const __attribute__((address_space(1))) T*)(base + size_t(lane_part)); }
template <int WORDS> __device__ __forceinline__ Words<WORDS> load_words_at(Global base, uint32_t lane_part) {
    Words<WORDS> r;
    if constexpr (WORDS == 4) {
        const uint4_t v = load_at<uint4_t>(base, lane_part);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = v[i];
    } else {
        const uint2_t v = load_at<uint2_t>(base, lane_part);
        r.w[0] = v.x; r.w[1] = v.y;
    }
    return r;
}

// A wave's way through the page table: 64 entries at a time, one to a lane. (A scalar load for each block of keys would have
// every wave wait for it; places are asked for in ascending order, or, by twos, in descending order.)
template <bool DOWN> struct Pages {
    uint32_t first, entry;
    __device__ __forceinline__ void fetch(Args& a, const Segment& x, uint32_t page, uint32_t lane) {
        if constexpr (DOWN) page = max(page, 62u) - 62u;       // (the step's second place may be on the next page)
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

// ---- the kernel -------------------------------------------------------------------------------------------------------

// Workgroups of a compute unit. Their waves share out a segment's keys, 32 at a time.
template <int D, int R, int PARTS, bool SHAPED> constexpr bool kThree = SHAPED && R == 2 && three_of_two_tiles(D, PARTS == 0);
template <int D, int R, int PARTS, int WAVES, bool SHAPED> constexpr int kResident = D > 128 || WAVES == 8 ? 1 : R == 1 || kThree<D, R, PARTS, SHAPED> ? 3 : 2;

// Joins a workgroup's waves, kAtOnce tiles at a time, and writes the rows. (Of two tiles one, where LDS is for three workgroups.)
template <int D, int R, int PARTS, bool SHAPED> constexpr int kAtOnce = R > 1 && D <= 128 && !kThree<D, R, PARTS, SHAPED> ? 2 : 1;
template <int D> constexpr int kRowFloats = D + 4;                 // of a row in LDS: 16 bytes further round the banks than the last
template <int WAVES, bool SHAPED, int D, int CODES, int R, int PARTS>
__device__ __forceinline__ void join_waves(const Segment& x, Sums<D, CODES, R, PARTS>& sums, char* space, float (&joined_m)[WAVES][R * 16], float (&joined_l)[WAVES][R * 16]) {
    using S = Shape<D>;
    Args& a = kernel_args();
    const uint32_t thread = thread_here(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), col = lane & 15, quarter = lane >> 4;
    const uint32_t share = own_share(a);
    constexpr int kTilesAtOnce = kAtOnce<D, R, PARTS, SHAPED>, kRows = kTilesAtOnce * 16;
    float(*joined)[kRows * kRowFloats<D>] = reinterpret_cast<float(*)[kRows * kRowFloats<D>]>(space);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float l = sum_quarters(sums.l[r]);
        if (quarter == 0) {
            joined_m[wave][r * 16 + col] = sums.m[r];
            joined_l[wave][r * 16 + col] = l;
        }
    }
    __syncthreads();
    // what a row's waves together lead, and sum up to
    auto row_of = [&](uint32_t row, float& top, float& sum) {
        top = joined_m[0][row];
        sum = 0.0f;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = __builtin_fmaxf(top, joined_m[w][row]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += joined_l[w][row] * exp2_fast(joined_m[w][row] - top);
    };
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += kTilesAtOnce) {
        if (r0 > 0) __syncthreads();
#pragma unroll
        for (int r = r0; r < r0 + kTilesAtOnce; ++r) {
            float top, sum;
            row_of(r * 16 + col, top, sum);
            // (a sum that is NaN, from a NaN among the scores, makes the row NaN)
            const float factor = sum == 0.0f ? 0.0f : exp2_fast(joined_m[wave][r * 16 + col] - top) / sum;
#pragma unroll
            for (int c = 0; c < S::kLoads; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // rows quarter * 4 + i of the kWords tiles of a chunk are neighbouring elements
                    float* to = &joined[wave][((r - r0) * 16 + col) * kRowFloats<D> + c * S::kChunk + (quarter * 4 + i) * S::kWords];
#pragma unroll
                    for (int w = 0; w < S::kWords; ++w) to[w] = sums.o[r][c * S::kWords + w][i] * factor;
                }
        }
        __syncthreads();
        auto sum_of = [&](uint32_t i) {
            const uint32_t at = i / (D / 4) * kRowFloats<D> + i % (D / 4) * 4;
            float4_t e = *reinterpret_cast<const float4_t*>(&joined[0][at]);
#pragma unroll
            for (int w = 1; w < WAVES; ++w) e += *reinterpret_cast<const float4_t*>(&joined[w][at]);
            return e;
        };
        const uint32_t count = min(uint32_t(kRows), x.rows - min(x.rows, uint32_t(r0 * 16))) * (D / 4);
        if (x.part < 0) {
#pragma unroll 2
            for (uint32_t i = thread; i < count; i += WAVES * 64) put4(a, x, r0 * 16 + i / (D / 4), i % (D / 4) * 4, sum_of(i));
        } else {
            float4_t* to = reinterpret_cast<float4_t*>(a.partial + ((size_t(share) * 2 + x.part) * a.unit_rows + r0 * 16) * D);
#pragma unroll 4
            for (uint32_t i = thread; i < count; i += WAVES * 64) to[i] = sum_of(i);
        }
    }
    if (thread < x.rows) {
        float top, sum;
        row_of(thread, top, sum);
        put_lse(a, x, share, thread, top, sum);
    }
    __syncthreads();
}

template <int D, int CODES, int R, int PARTS, int WAVES, bool SHAPED>
__global__ __launch_bounds__(WAVES * 64, (kResident<D, R, PARTS, WAVES, SHAPED>)) void k_tree_attention(const ArgsOf<SHAPED>) {
    using S = Shape<D>;
    constexpr int kRegs = kQueryRegs<D, PARTS>, kRuns = kRegs / 4;
    // One tile's rows: in registers. More: in LDS, whose place the joining of the waves takes afterwards.
    constexpr bool kInLds = R > 1;
    constexpr uint32_t kJoin = WAVES * kAtOnce<D, R, PARTS, SHAPED> * 16 * kRowFloats<D> * 4, kQueries = kInLds ? R * kRuns * 1024 : 0;
    __shared__ __attribute__((aligned(16))) char space[kJoin > kQueries ? kJoin : kQueries];
    __shared__ float joined_m[WAVES][R * 16], joined_l[WAVES][R * 16];
    __shared__ float units[R * 16];
    __shared__ uint64_t masks[R * 16];                             // the first word of each: all there is for trees of up to 64
    __shared__ __attribute__((aligned(16))) float scales[WAVES][64];
    // Of shaped rows: unit, slope in units of log2, and where they are, from the end of the context and, for steps with new tokens, from the
    // first one's position (floats have whole numbers up to 2^24: distances are exact up to that, places need not be); the first key they
    // see. And what keys of a step with new tokens are away from where they would be by their places.
    __shared__ float4_t shapes[SHAPED ? R * 16 : 1];
    __shared__ uint32_t firsts[SHAPED ? R * 16 : 1];
    __shared__ __attribute__((aligned(16))) float moves[SHAPED ? WAVES : 1][32];
    uint4_t* queries = reinterpret_cast<uint4_t*>(space);

    __shared__ uint32_t walks[WAVES][8];
    walk<D, WAVES * 64, SHAPED>(kernel_args(), threadIdx.x & 63, walks[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)], [&](const Segment& x) {
        Args& a = kernel_args();
        const uint32_t thread = thread_here(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), col = lane & 15, quarter = lane >> 4;
        const uint32_t lane_k = col * D + quarter * (S::kChunk / 4), lane_v = quarter * (4 * D) + col * (S::kChunk / 4);
        // The pages are asked for first, which keys and values wait for, then the queries, which are made ready while those are on their way.
        uint32_t key = x.key0 + wave * 32;
        constexpr uint32_t kStride = WAVES * 32;
        // (from the last step's keys to the first's: the loop counts up all the same, as another form of it would hold the sums twice)
        uint32_t up = key, mirror = 0;
        if constexpr (SHAPED)
            if (key < x.key1) key += (x.key1 - key - 1) / kStride * kStride, mirror = up + key;
        Pages<SHAPED> pages{0, 0};
        // (There is an entry to read: a sequence with rows has a key at least, see sequence_of. A wave without keys asks for its last
        // page's: with a branch around this, heads of 192 and 256 took 6 % longer.)
        pages.fetch(a, x, key >> a.cache.page_log, lane);
        uint4_t raw[S::kSteps];
        const uint32_t tile = kInLds ? wave : 0;
        uint64_t mask = 0;                                         // (of one tile's rows, like the queries)
        if (tile < R) {
            load_query<D>(a, x, tile * 16 + col, quarter, raw);
            if (a.mask) mask = a.mask[int64_t(x.seq.first_token + place_of_row(a, x, tile * 16 + col).token) * a.mask_words];
        }
        float slope = 0.0f, from_context = 0.0f, from_new = 0.0f;
        uint32_t own_first = 0;
        if constexpr (SHAPED) {
            if (tile < R) {
                const RowPlace place = place_of_row(a, x, tile * 16 + col);
                if (shaped(a).slopes) {
                    slope = shaped(a).slopes[place.head] * kLog2e;
                    uint32_t own = x.seq.context + place.token, first = x.seq.context;
                    if (Shaped& b = shaped(kernel_args()); b.positions) {
                        own = uint32_t(b.positions[x.seq.first_token + place.token]);
                        first = uint32_t(b.positions[x.seq.first_token]);
                    }
                    from_context = float(int32_t(own - x.seq.context));
                    from_new = float(int32_t(own - first));
                }
                if (shaped(a).first) own_first = first_of(a, x.seq, place.token);
            }
        }
        size_t at[2];
        Words<S::kWords> k[2][S::kLoads], v[2][S::kLoads];
        float4_t k_scales[2], v_scales[2];
        auto locate = [&](uint32_t key) {
#pragma unroll
            for (int h = 0; h < 2; ++h) at[h] = pages.place(a, x, key + h * 16, lane);
        };
        auto load_k = [&] {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Global from = of_wave(a.cache.k + at[h] * D);
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) k[h][i] = load_words_at<S::kWords>(from + i * S::kChunk, lane_k);
            }
        };
        // Scales of several tiles' steps are used again and again, and would take 16 registers: those go through one register of each
        // lane, asked for with the step's keys, to LDS, two of the keys' and two of the values' blocks of 16 side by side.
        float scale_ahead = 0.0f;
        auto ask_scales = [&] {
            if constexpr (kInLds) {
                Args& b = kernel_args();
                const uint32_t l = thread_here();
                const size_t first = at[0], second = at[1];
                scale_ahead = ((l & 32 ? b.cache.v_scale : b.cache.k_scale) + (l & 16 ? second : first))[l & 15];
            }
        };
        auto put_scales = [&] {
            if constexpr (kInLds) {
                // (the wave's own part of LDS, which it writes and reads in order)
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
                scales[wave][lane] = scale_ahead;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            }
        };
        auto load_scales_and_v = [&] {
            if constexpr (!kInLds) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    k_scales[h] = load_at<float4_t>(of_wave(a.cache.k_scale + at[h]), quarter * 16);
                    v_scales[h] = load_at<float4_t>(of_wave(a.cache.v_scale + at[h]), quarter * 16);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Global from = of_wave(a.cache.v + at[h] * D);
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i) v[h][i] = load_words_at<S::kWords>(from + i * S::kChunk * 4, lane_v);
            }
        };
        if (key < x.key1) {
            locate(key);
            // (in the order of the steps to come: a first step that had asked for values first would have every step wait for its values)
            __builtin_amdgcn_sched_barrier(0);
            ask_scales();
            load_k();
            __builtin_amdgcn_sched_barrier(0);
            load_scales_and_v();
            __builtin_amdgcn_sched_barrier(0);
        }
        uint32_t q[kRegs];
        float unit = 0.0f;
        if (tile < R) {
            unit = prepare_query<D, PARTS>(kernel_args(), raw, q);
            if constexpr (kInLds) {
#pragma unroll
                for (int run = 0; run < kRuns; ++run) queries[(tile * kRuns + run) * 64 + lane] = uint4_t{q[run * 4], q[run * 4 + 1], q[run * 4 + 2], q[run * 4 + 3]};
                if (quarter == 0) {
                    if constexpr (SHAPED) {
                        shapes[tile * 16 + col] = float4_t{unit, slope, from_context, from_new};
                        firsts[tile * 16 + col] = own_first;
                    } else {
                        units[tile * 16 + col] = unit;
                    }
                    masks[tile * 16 + col] = mask;
                }
            }
        }
        Sums<D, CODES, R, PARTS> sums;
        sums.clear();
        if constexpr (kInLds) __syncthreads();
        auto get_k = [&](int h, int i) { return k[h][i]; };
        auto get_v = [&](int h, int i) { return v[h][i]; };
        auto get_q = [&](int r, int run) {
            if constexpr (kInLds) return queries[(r * kRuns + run) * 64 + lane];
            else return uint4_t{q[run * 4], q[run * 4 + 1], q[run * 4 + 2], q[run * 4 + 3]};
        };
        auto get_unit = [&](int r) {
            if constexpr (SHAPED) {
                const float4_t its = kInLds ? shapes[r * 16 + col] : float4_t{unit, slope, from_context, from_new};
                return float4_t{its[0], its[1], key + 32 > x.seq.context ? its[3] : its[2], 0.0f};
            } else {
                return kInLds ? units[r * 16 + col] : unit;
            }
        };
        auto get_k_scales = [&](float4_t (&s)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = kInLds ? *reinterpret_cast<const float4_t*>(&scales[wave][h * 16 + quarter * 4]) : k_scales[h];
        };
        auto get_v_scales = [&](float4_t (&s)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = kInLds ? *reinterpret_cast<const float4_t*>(&scales[wave][32 + h * 16 + quarter * 4]) : v_scales[h];
        };
        // (from the thread's number anew, and so in the next: what both compute would be kept in registers through the loop)
        auto sees = [&](int r, int h) {
            Args& b = kernel_args();
            const uint32_t t = thread_here(), col = t & 15, quarter = t >> 4 & 3;
            const uint32_t first = key + h * 16 + quarter * 4, there = lowest_bits(int32_t(x.seq.total - first));
            const int32_t u = int32_t(first - x.seq.context);
            const uint32_t token = place_of_row(b, x, r * 16 + col).token;
            uint32_t from_first = 15u;
            if constexpr (SHAPED) {
                const uint32_t its_first = kInLds ? firsts[r * 16 + col] : own_first;
                from_first = ~lowest_bits(int32_t(its_first - first));
                if (b.mask == nullptr) {
                    int32_t upto = int32_t(token) + 1;
                    if (shaped(b).prefix) upto = max(upto, max(0, min(scalar(shaped(b).prefix + x.b), 1 << 30)) - int32_t(x.seq.context));
                    return lowest_bits(upto - u) & there & from_first;
                }
            }
            if (b.mask == nullptr) return lowest_bits(int32_t(token) + 1 - u) & there;
            const uint64_t word = kInLds ? masks[r * 16 + col] : mask;
            return mask_bits<SHAPED && D < 256>(b.mask + int64_t(x.seq.first_token + token) * b.mask_words, word, b.mask_words, u) & there & from_first;
        };
        // what lies behind the last token, or in front of the first that anybody sees, is no token's (its page may have gone to another):
        // no code of it may reach a product, as 0 * NaN is NaN
        auto hide = [&] {
            const uint32_t quarter = thread_here() >> 4 & 3;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t there = lowest_bits(int32_t(x.seq.total - (key + h * 16 + quarter * 4)));
                if constexpr (SHAPED) there &= ~lowest_bits(int32_t(x.seq.front - (key + h * 16 + quarter * 4)));
                uint32_t keep = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) keep |= there >> i & 1 ? 0xffu << (8 * i) : 0u;
#pragma unroll
                for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
                    for (int w = 0; w < S::kWords; ++w) v[h][i].w[w] &= keep;
            }
        };
        // Scores in units of log2: the tanh, cap (1 - 2 r), r = 1 / (1 + e^(2 s / cap)). Its sum, reciprocal (to a unit in the last place) and
        // exponential leave r off by 3.5 2^-24 at most, so the result by twice that and what its own roundings add: 2^-20.5 of the cap (measured
        // 2^-22), which is 2^-11 in units of log2 at the largest, 2^9, where half precision's rounding of weights is 2^-11 as well; and the
        // distance's part.
        const auto shape = [&] {
            if constexpr (!SHAPED) {
                return nullptr;
            } else {
                return [&, cap_in = shaped(a).cap_in, cap_out = shaped(a).cap_out, biased = shaped(a).slopes != nullptr, placed = shaped(a).positions != nullptr](int h, float2_t its, float4_t& s) {
                    if (cap_in != 0.0f)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + exp2_fast(s[i] * cap_in)), -2.0f * cap_out, cap_out);
                    if (D < 256 ? biased : shaped(kernel_args()).slopes != nullptr) {      // (256: no register is left for it, nor for the next)
                        const float at = float(int32_t(key + h * 16 + (thread_here() >> 4 & 3) * 4 - x.seq.context)) - its.y;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(its.x, at + float(i), s[i]);
                        if (key + 32 > x.seq.context && (D < 256 ? placed : shaped(kernel_args()).positions != nullptr)) {
                            const float4_t more = *reinterpret_cast<const float4_t*>(&moves[wave][h * 16 + (thread_here() >> 4 & 3) * 4]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(its.x, more[i], s[i]);
                        }
                    }
                };
            }
        }();
        auto put_moves = [&] {
            if constexpr (SHAPED) {
                Shaped& b = shaped(kernel_args());
                if (b.slopes && b.positions && key + 32 > x.seq.context) {
                    const uint32_t l = thread_here() & 63, j = key + l;
                    const uint32_t ahead = uint32_t(scalar(b.positions + x.seq.first_token)) - x.seq.context;
                    uint32_t more = 0u - ahead;
                    if (l < 32 && j >= x.seq.context && j < x.seq.total) more += uint32_t(b.positions[x.seq.first_token + j - x.seq.context]) - j;
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
                    if (l < 32) moves[wave][l] = float(int32_t(more));
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
                }
            }
        };
        // One step; `more` is known where this is compiled, as the compiler would otherwise count on values that were not asked for
        // behind keys that were, and wait for both.
        auto run_step = [&](auto more) {
            const uint32_t next = SHAPED ? mirror - up - kStride : key + kStride;
            set_priority<SHAPED>(x, key);
            if constexpr (more()) locate(next);
            put_scales();
            put_moves();
            // the keys' registers are free for the next once the scores are there, the others' at the end
            sums.step(key + 32 > x.all_see || (SHAPED && key < x.all_from), get_k, get_v, get_q, get_unit, get_k_scales, get_v_scales, shape, sees, hide, [&] {
                if constexpr (more()) ask_scales();
                if constexpr (more()) load_k();
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (more()) load_scales_and_v();
            __builtin_amdgcn_sched_barrier(0);
            key = next;
            if constexpr (SHAPED) up += kStride;
        };
#pragma unroll 1
        while ((SHAPED ? up : key) + kStride < x.key1) run_step(std::true_type{});
        if ((SHAPED ? up : key) < x.key1) run_step(std::false_type{});
        join_waves<WAVES, SHAPED>(x, sums, space, joined_m, joined_l);
    });
}

// ---- launches ---------------------------------------------------------------------------------------------------------

template <int D, int CODES, int PARTS, bool SHAPED> int start_attention(const ArgsOf<SHAPED>& a, const AttentionPlan& p, void* stream, Launched& info) {
    const dim3 grid = p.shares() == 0 ? dim3(a.cache.kv_heads, p.row_blocks, a.batch) : dim3(p.shares(), 1, 1), block(p.waves * 64);
    const char* name = SHAPED ? p.tiles == 4 ? "shaped_attention_4x4" : p.tiles == 2 ? "shaped_attention_2x4" : p.waves == 8 ? "shaped_attention_1x8" : "shaped_attention_1x4"
                              : p.tiles == 4 ? "tree_attention_4x4" : p.tiles == 2 ? "tree_attention_2x4" : p.waves == 8 ? "tree_attention_1x8" : "tree_attention_1x4";
    info = {name, {grid.x, grid.y, grid.z}, {block.x, 1, 1}, 0};
    if constexpr (D <= 128)
        if (p.tiles == 4) return launch(k_tree_attention<D, CODES, 4, PARTS, 4, SHAPED>, grid, block, stream, a);
    if (p.tiles == 2) return launch(k_tree_attention<D, CODES, 2, PARTS, 4, SHAPED>, grid, block, stream, a);
    if (p.waves == 8) return launch(k_tree_attention<D, CODES, 1, PARTS, 8, SHAPED>, grid, block, stream, a);
    return launch(k_tree_attention<D, CODES, 1, PARTS, 4, SHAPED>, grid, block, stream, a);
}
template <int D, int CODES, bool SHAPED> int start_attention(const ArgsOf<SHAPED>& a, const AttentionPlan& p, void* stream, Launched& info) {
    if constexpr (kCodeProducts<D, CODES>) {
        if (a.type == FKLHIP_F16) return start_attention<D, CODES, 3, SHAPED>(a, p, stream, info);
        return start_attention<D, CODES, 2, SHAPED>(a, p, stream, info);
    } else {
        return start_attention<D, CODES, 0, SHAPED>(a, p, stream, info);
    }
}
template <int D, bool SHAPED> int start_attention(const ArgsOf<SHAPED>& a, const AttentionPlan& plan, void* stream, Launched& info) {
    if (a.cache.codes == FKLHIP_CODES_INT8) return start_attention<D, FKLHIP_CODES_INT8, SHAPED>(a, plan, stream, info);
    return start_attention<D, FKLHIP_CODES_E4M3, SHAPED>(a, plan, stream, info);
}

} // namespace fkattn
