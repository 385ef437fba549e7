// merge.hip -- joins the parts of a row's attention that several shares of the work computed (work_shares.hpp).
//
// o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max). Bound by latency: counting the work, reading the parts' weights,
// reading the parts (4 bytes an element), one after another. Few parts to a row: a group of lanes takes a row (k_merge_few).
// Many: a workgroup does, whose groups of lanes take a part each, so that many parts are read at once (k_merge_many).
#include "work_shares.hpp"

namespace fkattn {
namespace {

constexpr uint32_t kThreads = 256, kMostParts = 1025;         // (a row's parts are of neighbouring shares)
template <int D> struct Lanes { static constexpr uint32_t kRow = D <= 64 ? 16 : D <= 128 ? 32 : 64, kGroups = kThreads / kRow; };

// The sequence of a token, with the granules in front of it.
__device__ __forceinline__ Found sequence_of_token(Args& a, uint32_t token) {
    return find(a, threadIdx.x & 63, [&](uint32_t, const Sequence& s, uint32_t, uint32_t) { return token >= s.first_token && token - s.first_token < s.fresh; });
}
// A row's parts: those of shares share0 .. share0 + count. None: nobody had any of it. One: it has been written.
struct Parts {
    uint32_t share0, count, row;
    __device__ __forceinline__ size_t place(Args& a, uint32_t part) const { return (size_t(share0 + part) * 2 + (part == 0 ? 1 : 0)) * a.unit_rows + row; }
    // (a share of nothing, between others where there are more shares than granules, wrote nothing)
    __device__ __forceinline__ float lse(Args& a, uint32_t all, uint32_t part) const {
        return share_begin(a, all, share0 + part) == share_begin(a, all, share0 + part + 1) ? -__builtin_inff() : a.partial_lse[place(a, part)];
    }
};
__device__ __forceinline__ Parts parts_of(Args& a, const Found& f, uint32_t token, uint32_t head) {
    const uint32_t n = granules_of(a, f.s);
    const uint32_t kv_head = divide(head, a.group_magic), row = (token - f.s.first_token) * a.group + head - kv_head * a.group;
    const uint32_t block = row >> __builtin_ctz(a.unit_rows);
    if (n == 0) return {0, 0, 0};
    const uint32_t first = f.before + (kv_head * blocks_of(a, f.s) + block) * n;
    const uint32_t share0 = share_of(a, f.all, first + a.lead);  // (what stands in front of the keys is nobody's part)
    return {share0, share_of(a, f.all, first + n - 1) - share0 + 1, row - block * a.unit_rows};
}
// Four elements of a row, and its lse (in units of log2).
__device__ __forceinline__ void put4(Args& a, uint32_t token, uint32_t head, uint32_t d, float4_t x) {
    uint2_t w;
    if (a.type == FKLHIP_BF16) { w.x = pack2<FKLHIP_BF16>(x[0], x[1]); w.y = pack2<FKLHIP_BF16>(x[2], x[3]); }
    else { w.x = pack2<FKLHIP_F16>(x[0], x[1]); w.y = pack2<FKLHIP_F16>(x[2], x[3]); }
    *reinterpret_cast<uint2_t*>(a.out.data + int64_t(token) * a.out.token_stride + int64_t(head) * a.out.head_stride + d * 2) = w;
}
__device__ __forceinline__ void put_lse(Args& a, uint32_t token, uint32_t head, float lse) {
    if (a.lse) a.lse[size_t(token) * a.q_heads + head] = lse * 0.6931471805599453f;
}

// Four elements of a part, weighted. A part without weight may hold anything; it is read all the same, as a branch around each
// would have the parts come one after another.
__device__ __forceinline__ float4_t part4(const float* from, float w) {
    const float4_t x = *reinterpret_cast<const float4_t*>(from);
    float4_t y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = w != 0.0f ? x[i] * w : 0.0f;
    return y;
}

template <int D> __global__ __launch_bounds__(kThreads) void k_merge_few(const AttentionArgs) {
    constexpr uint32_t kLanes = Lanes<D>::kRow;
    Args& a = kernel_args();
    const uint32_t at = threadIdx.x % kLanes, head = blockIdx.x * Lanes<D>::kGroups + threadIdx.x / kLanes, d = at * 4;
    const uint32_t token = blockIdx.y + blockIdx.z * 32768u;
    if (token >= a.tokens) return;
    const Found f = sequence_of_token(a, token);
    if (head >= a.q_heads) return;
    if (f.b >= a.batch) {                                     // a row of no sequence
        if (d < D) put4(a, token, head, d, float4_t{0.0f, 0.0f, 0.0f, 0.0f});
        if (at == 0) put_lse(a, token, head, -__builtin_inff());
        return;
    }
    const Parts p = parts_of(a, f, token, head);
    if (p.count == 1) return;
    float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float top = -__builtin_inff(), sum = 0.0f;
    for (uint32_t i0 = 0; i0 < p.count; i0 += kLanes) {
        const float mine = i0 + at < p.count ? p.lse(a, f.all, i0 + at) : -__builtin_inff();
        float most = mine;
#pragma unroll
        for (uint32_t i = kLanes / 2; i; i >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, i, kLanes));
        const float now = __builtin_fmaxf(top, most), base = now == -__builtin_inff() ? 0.0f : now, alpha = __builtin_amdgcn_exp2f(top - base);
        top = now;
        o *= alpha;
        const float weight = __builtin_amdgcn_exp2f(mine - base);
        float all = weight;
#pragma unroll
        for (uint32_t i = kLanes / 2; i; i >>= 1) all += __shfl_xor(all, i, kLanes);
        sum = sum * alpha + all;                              // NaN where a part's is
        const uint32_t count = min(kLanes, p.count - i0);
#pragma unroll 4
        for (uint32_t i = 0; i < count; ++i) {
            const float w = __shfl(weight, i, kLanes);        // (of all lanes: those behind the row have weights too)
            if (d < D) o += part4(a.partial + p.place(a, i0 + i) * D + d, w);
        }
    }
    if (d < D) put4(a, token, head, d, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (at == 0) put_lse(a, token, head, top + __builtin_log2f(sum));
}

template <int D> __global__ __launch_bounds__(kThreads) void k_merge_many(const AttentionArgs) {
    constexpr uint32_t kLanes = Lanes<D>::kRow, kGroups = Lanes<D>::kGroups;
    __shared__ float weight[kMostParts], tops[4], sums[4];
    __shared__ __attribute__((aligned(16))) float joined[kGroups][D];
    Args& a = kernel_args();
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = threadIdx.x % kLanes, group = threadIdx.x / kLanes, d = at * 4;
    const uint32_t head = blockIdx.x, token = blockIdx.y + blockIdx.z * 32768u;
    if (token >= a.tokens) return;
    const Found f = sequence_of_token(a, token);
    if (f.b >= a.batch) {                                     // a row of no sequence
        if (group == 0 && d < D) put4(a, token, head, d, float4_t{0.0f, 0.0f, 0.0f, 0.0f});
        if (threadIdx.x == 0) put_lse(a, token, head, -__builtin_inff());
        return;
    }
    const Parts p = parts_of(a, f, token, head);
    if (p.count == 1) return;
    float top = -__builtin_inff();
    for (uint32_t i = threadIdx.x; i < p.count; i += kThreads) {
        const float x = p.lse(a, f.all, i);
        weight[i] = x;
        top = __builtin_fmaxf(top, x);
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, i));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < p.count; i += kThreads) {
        const float w = __builtin_amdgcn_exp2f(weight[i] - base);
        weight[i] = w;
        sum += w;
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (d < D) {
#pragma unroll 8
        for (uint32_t i = group; i < p.count; i += kGroups) x += part4(a.partial + p.place(a, i) * D + d, weight[i]);
        *reinterpret_cast<float4_t*>(&joined[group][d]) = x;
    }
    __syncthreads();
    if (group == 0 && d < D) {
#pragma unroll
        for (uint32_t i = 1; i < kGroups; ++i) x += *reinterpret_cast<const float4_t*>(&joined[i][d]);
        put4(a, token, head, d, x * (sum == 0.0f ? 0.0f : 1.0f / sum));
        if (at == 0) put_lse(a, token, head, top + __builtin_log2f(sum));
    }
}

template <int D> int start_merge(const AttentionArgs& a, bool many_parts, void* stream) {
    const uint32_t y = a.tokens < 32768u ? a.tokens : 32768u, z = (a.tokens + 32767u) / 32768u;
    if (many_parts) return launch(k_merge_many<D>, dim3(a.q_heads, y, z), dim3(kThreads), stream, a);
    return launch(k_merge_few<D>, dim3((a.q_heads + Lanes<D>::kGroups - 1) / Lanes<D>::kGroups, y, z), dim3(kThreads), stream, a);
}

} // namespace

int launch_merge(const AttentionArgs& a, uint32_t head_dim, bool many_parts, void* stream) {
    switch (head_dim) {
    case 64: return start_merge<64>(a, many_parts, stream);
    case 96: return start_merge<96>(a, many_parts, stream);
    case 128: return start_merge<128>(a, many_parts, stream);
    case 192: return start_merge<192>(a, many_parts, stream);
    default: return start_merge<256>(a, many_parts, stream);
    }
}

} // namespace fkattn
