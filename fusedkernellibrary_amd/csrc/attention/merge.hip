// merge.hip -- joins the parts of a row's attention that several shares of the work computed (work_shares.hpp).
//
// o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max). A workgroup to a row: its threads take the parts' weights first, then
// groups of lanes take a part each, so that many parts are read at once. Bound by latency: counting the work, reading a
// few weights, reading the parts (4 bytes an element), one after another.
#include "work_shares.hpp"

namespace fkattn {
namespace {

constexpr uint32_t kThreads = 256, kMostParts = 1025;         // (a row's parts are of neighbouring shares)

template <int D> __global__ __launch_bounds__(kThreads) void k_merge(const AttentionArgs) {
    Args& a = kernel_args();
    constexpr uint32_t kLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, kGroups = kThreads / kLanes;
    __shared__ float weight[kMostParts], tops[4], sums[4];
    __shared__ __attribute__((aligned(16))) float joined[kGroups][D];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t head = blockIdx.x, token = blockIdx.y + blockIdx.z * 32768u;
    if (token >= a.tokens) return;
    const Found f = find(a, lane, [&](uint32_t, uint32_t b, uint32_t, uint32_t) {
        const Sequence s = sequence_of_lane(a, b);
        return token >= s.first_token && token - s.first_token < s.fresh;
    });
    if (f.b >= a.batch) return;                               // a row of no sequence
    const Sequence s = sequence_at(a, f.b);
    const uint32_t n = granules_of(a, s), subs = subs_of(a, s);
    const uint32_t kv_head = divide(head, a.group_magic), row = (token - s.first_token) * a.group + head - kv_head * a.group;
    const uint32_t block = row / a.unit_rows, size = n * min(a.block_subs, subs - block * a.block_subs);
    const uint32_t first = f.before + kv_head * (n * subs) + block * a.block_subs * n;
    char* out = a.out.data + int64_t(token) * a.out.token_stride + int64_t(head) * a.out.head_stride;
    const uint32_t at = threadIdx.x % kLanes, group = threadIdx.x / kLanes, d = at * 4;
    if (size == 0) {                                          // no keys: nobody had it
        if (group == 0 && d < D) *reinterpret_cast<uint2_t*>(out + d * 2) = uint2_t{0, 0};
        if (threadIdx.x == 0 && a.lse) a.lse[size_t(token) * a.q_heads + head] = -__builtin_inff();
        return;
    }
    // the share of a granule g: the largest i with i * all / shares <= g
    const auto share_of = [&](uint32_t g) { return uint32_t((((uint64_t(g) + 1) << a.shares_log) + f.all - 1) / f.all) - 1; };
    const uint32_t share0 = share_of(first), share1 = share_of(first + size - 1);
    if (share0 == share1) return;                             // written by the one share that had all of it
    const uint32_t parts = share1 - share0 + 1, in_block = row - block * a.unit_rows;
    const auto place = [&](uint32_t part) { return (size_t(share0 + part) * 2 + (part == 0 ? 1 : 0)) * a.unit_rows + in_block; };
    float top = -__builtin_inff();
    for (uint32_t i = threadIdx.x; i < parts; i += kThreads) {
        const uint32_t share = share0 + i;
        const float x = share_begin(a, f.all, share) == share_begin(a, f.all, share + 1) ? -__builtin_inff() : a.partial_lse[place(i)];   // (shares of nothing)
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
    for (uint32_t i = threadIdx.x; i < parts; i += kThreads) {
        const float w = __builtin_amdgcn_exp2f(weight[i] - base);
        weight[i] = w;
        sum += w;
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];              // NaN where a part's is
    float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (d < D) {
#pragma unroll 4
        for (uint32_t i = group; i < parts; i += kGroups) {
            const float w = weight[i];
            if (w != 0.0f) x += *reinterpret_cast<const float4_t*>(a.partial + place(i) * D + d) * w;
        }
        *reinterpret_cast<float4_t*>(&joined[group][d]) = x;
    }
    __syncthreads();
    if (group == 0 && d < D) {
#pragma unroll
        for (uint32_t i = 1; i < kGroups; ++i) x += *reinterpret_cast<const float4_t*>(&joined[i][d]);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        x *= inv;
        uint2_t w;
        if (a.type == FKLHIP_BF16) { w.x = pack2<FKLHIP_BF16>(x[0], x[1]); w.y = pack2<FKLHIP_BF16>(x[2], x[3]); }
        else { w.x = pack2<FKLHIP_F16>(x[0], x[1]); w.y = pack2<FKLHIP_F16>(x[2], x[3]); }
        *reinterpret_cast<uint2_t*>(out + d * 2) = w;
        if (at == 0 && a.lse) a.lse[size_t(token) * a.q_heads + head] = (top + __builtin_log2f(sum)) * 0.6931471805599453f;
    }
}

} // namespace

int launch_merge(const AttentionArgs& a, uint32_t head_dim, void* stream) {
    const dim3 grid(a.q_heads, a.tokens < 32768u ? a.tokens : 32768u, (a.tokens + 32767u) / 32768u);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (head_dim) {
    case 64: k_merge<64><<<grid, kThreads, 0, s>>>(a); break;
    case 96: k_merge<96><<<grid, kThreads, 0, s>>>(a); break;
    case 128: k_merge<128><<<grid, kThreads, 0, s>>>(a); break;
    case 192: k_merge<192><<<grid, kThreads, 0, s>>>(a); break;
    default: k_merge<256><<<grid, kThreads, 0, s>>>(a); break;
    }
    return int(hipGetLastError());
}

} // namespace fkattn
