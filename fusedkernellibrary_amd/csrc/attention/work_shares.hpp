// work_shares.hpp -- how attention's work is dealt out to workgroups: all of them count it the same way.
#pragma once

#include <type_traits>

#include "attention_device.hpp"

namespace fkattn {

// A kernel's only argument as it lies in the kernel-argument segment. Every call reads its fields anew, by scalar loads where
// they are used: held in registers from the start they are more than there are scalar registers.
using Args = const __attribute__((address_space(4))) AttentionArgs;
__device__ __forceinline__ Args& kernel_args() {
    auto p = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}
// The same of a kernel whose argument is ShapedArgs.
using Shaped = const __attribute__((address_space(4))) ShapedArgs;
__device__ __forceinline__ Shaped& shaped(Args& a) { return *(Shaped*)&a; }
template <bool SHAPED> using ArgsOf = std::conditional_t<SHAPED, ShapedArgs, AttentionArgs>;

// The thread's number, for a part of a kernel that is run again and again: what is computed from it stays in that part (the
// compiler would move it in front of the loop over segments, and keep it in registers through everything).
__device__ __forceinline__ uint32_t thread_here() {
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}
// What no kernel writes while it runs, at a place that is the same for the whole wave: a scalar load.
template <typename T> __device__ __forceinline__ T scalar(const T* p) { return *(const __attribute__((address_space(4))) T*)(uintptr_t)p; }

// A sequence as the device finds it, held inside what the host was told. One with rows has keys: where the page table has room for
// no token, max_new is 0 here.
// (`front`: no row sees a key in front of that, and `skip` granules hold no other; 0 where nothing is shaped.)
struct Sequence { uint32_t first_token, fresh, context, total, rows, front = 0, skip = 0; };
__device__ __forceinline__ Sequence sequence_of(Args& a, int32_t start, int32_t end, int32_t have) {
    Sequence s;
    s.first_token = start < 0 ? 0u : min(uint32_t(start), a.tokens);
    const int32_t diff = end - int32_t(s.first_token);
    s.fresh = diff < 0 ? 0u : min(min(uint32_t(diff), a.max_new), a.tokens - s.first_token);
    s.context = have < 0 ? 0u : min(min(uint32_t(have), a.max_context), a.room);
    s.total = min(s.context + s.fresh, a.room);
    s.rows = s.fresh * a.group;
    return s;
}
__device__ __forceinline__ uint32_t granules_of_keys(Args& a, uint32_t keys) { return (keys + (1u << a.granule_log) - 1) >> a.granule_log; }
// A sequence's front, by what its first row sees first. (One granule is left at least: what has rows has them written.)
__device__ __forceinline__ void skip_front(Args& a, Sequence& s, int32_t first) {
    s.front = first < 0 ? 0u : min(uint32_t(first), s.total);
    s.skip = s.total ? min(s.front >> a.granule_log, granules_of_keys(a, s.total) - 1) : 0u;
}
template <bool SHAPED> __device__ __forceinline__ Sequence sequence_at(Args& a, uint32_t b) {
    Sequence s = sequence_of(a, scalar(a.q_start + b), scalar(a.q_start + b + 1), scalar(a.context + b));
    if constexpr (SHAPED)
        if (shaped(a).first && s.fresh) skip_front(a, s, scalar(shaped(a).first + s.first_token));
    return s;
}
// Work is counted in granules: 2^granule_log keys of one key head and one block of its rows. In front of a block's keys stand
// `lead` granules for what it takes to begin and to end it.
__device__ __forceinline__ uint32_t granules_of(Args& a, const Sequence& s) { return s.total ? a.lead + granules_of_keys(a, s.total) - s.skip : 0u; }
__device__ __forceinline__ uint32_t blocks_of(Args& a, const Sequence& s) { return (s.rows + a.unit_rows - 1) >> __builtin_ctz(a.unit_rows); }
__device__ __forceinline__ uint32_t weight_of(Args& a, const Sequence& s) { return blocks_of(a, s) * a.cache.kv_heads * granules_of(a, s); }

// Sums of a wave's lanes up to and with each.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
    return v + uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t scan_wave(uint32_t v) {
    v = add_dpp<0x111, 0xf>(v);                               // row_shr 1, 2, 4, 8: within sixteen lanes
    v = add_dpp<0x112, 0xf>(v);
    v = add_dpp<0x114, 0xf>(v);
    v = add_dpp<0x118, 0xf>(v);
    v = add_dpp<0x142, 0xa>(v);                               // row_bcast 15: the second and fourth sixteen get the one before
    return add_dpp<0x143, 0xc>(v);                            // row_bcast 31: the upper half gets the lower
}

// (of the lane's own sequence; behind the last there are empty ones)
template <bool SHAPED> __device__ __forceinline__ Sequence sequence_of_lane(Args& a, uint32_t b) {
    if (b >= a.batch) return Sequence{0, 0, 0, 0, 0};
    Sequence s = sequence_of(a, a.q_start[b], a.q_start[b + 1], a.context[b]);
    if constexpr (SHAPED)
        if (shaped(a).first && s.fresh) skip_front(a, s, shaped(a).first[s.first_token]);
    return s;
}
template <bool SHAPED> __device__ __forceinline__ Sequence of_lane(const Sequence& s, uint32_t lane) {
    const auto get = [&](uint32_t x) { return uint32_t(__builtin_amdgcn_readlane(int(x), int(lane))); };
    Sequence its{get(s.first_token), get(s.fresh), get(s.context), get(s.total), get(s.rows)};
    if constexpr (SHAPED) its.front = get(s.front), its.skip = get(s.skip);
    return its;
}
// The granules of all sequences, and the first of a sequence: that of granule at(all), or that of a token; is_it(all, the lane's
// sequence, its first granule, the one behind its last). b is the batch's size if there is none.
struct Found { uint32_t all, b, before; Sequence s; };
template <bool SHAPED, typename F> __device__ __forceinline__ Found find(Args& a, uint32_t lane, F is_it) {
    uint32_t before = 0;
    Found f{0, a.batch, 0, {0, 0, 0, 0, 0}};
    if (a.batch <= 64) {
        const Sequence s = sequence_of_lane<SHAPED>(a, lane);
        const uint32_t own = weight_of(a, s), upto = scan_wave(own);
        f.all = __builtin_amdgcn_readlane(int(upto), 63);
        const uint64_t hits = __ballot(lane < a.batch && is_it(f.all, s, upto - own, upto));
        if (hits) {
            f.b = __builtin_ctzll(hits);
            f.before = __builtin_amdgcn_readlane(int(upto - own), int(f.b));
            f.s = of_lane<SHAPED>(s, f.b);
        }
        return f;
    }
    uint32_t sum = 0;
    for (uint32_t b = lane; b < a.batch; b += 64) sum += weight_of(a, sequence_of_lane<SHAPED>(a, b));
    f.all = __builtin_amdgcn_readlane(int(scan_wave(sum)), 63);
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const Sequence s = sequence_of_lane<SHAPED>(a, b0 + lane);
        const uint32_t own = weight_of(a, s), upto = before + scan_wave(own);
        const uint64_t hits = __ballot(b0 + lane < a.batch && is_it(f.all, s, upto - own, upto));
        if (hits) {
            const int hit = __builtin_ctzll(hits);
            f.b = b0 + hit;
            f.before = __builtin_amdgcn_readlane(int(upto - own), hit);
            f.s = of_lane<SHAPED>(s, hit);
            return f;
        }
        before = __builtin_amdgcn_readlane(int(upto), 63);
    }
    return f;
}
// There are share_odd << share_log shares, share_odd being 1 or 3; all granules times the shares fit 42 bits.
__device__ __forceinline__ uint32_t share_begin(Args& a, uint32_t all, uint32_t share) {
    const uint32_t x = uint32_t((uint64_t(share) * all) >> a.share_log);
    return a.share_odd == 3 ? x / 3 : x;
}
// The share that a granule is of: the last to begin at or in front of it.
__device__ __forceinline__ uint32_t share_of(Args& a, uint32_t all, uint32_t granule) {
    return uint32_t((((uint64_t(granule) + 1) * a.share_odd << a.share_log) + all - 1) / all) - 1;
}
// Neighbouring shares, which may be of the same keys, are on the same XCD (workgroups go round the eight).
__device__ __forceinline__ uint32_t own_share(Args& a) { return a.share_log >= 3 ? (blockIdx.x & 7u) * (a.share_odd << (a.share_log - 3)) + (blockIdx.x >> 3) : blockIdx.x; }

} // namespace fkattn
