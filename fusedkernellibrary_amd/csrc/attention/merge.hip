// merge.hip -- joins the parts of attention whose keys were shared out to several workgroups.
//
// o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max): a wave to a row, its lanes over the parts first (their weights),
// then over the row's elements. Bound by reading the parts, 4 bytes an element each, which a workgroup of another XCD wrote.
#include "attention_device.hpp"

namespace fkattn {
namespace {

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int i = 32; i; i >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, i));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int i = 32; i; i >>= 1) v += __shfl_xor(v, i);
    return v;
}

__global__ __launch_bounds__(256) void k_merge(const AttentionArgs a, const uint32_t dim) {
    const uint32_t lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= a.tokens * a.q_heads) return;
    const float* lse = a.partial_lse + size_t(row) * a.splits;
    float top = -__builtin_inff();
    for (uint32_t s = lane; s < a.splits; s += 64) top = __builtin_fmaxf(top, lse[s]);
    top = wave_max(top);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t s = lane; s < a.splits; s += 64) sum += __builtin_amdgcn_exp2f(lse[s] - base);
    sum = wave_sum(sum);                                   // NaN where a part's is
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t d = lane * 4;
    float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (d < dim) {
        const float* from = a.partial + size_t(row) * a.splits * dim + d;
        for (uint32_t s = 0; s < a.splits; ++s) {
            const float w = __builtin_amdgcn_exp2f(lse[s] - base) * inv;
            if (w != 0.0f) x += *reinterpret_cast<const float4_t*>(from + size_t(s) * dim) * w;
        }
        uint2_t w;
        if (a.type == FKLHIP_BF16) { w.x = pack2<FKLHIP_BF16>(x[0], x[1]); w.y = pack2<FKLHIP_BF16>(x[2], x[3]); }
        else { w.x = pack2<FKLHIP_F16>(x[0], x[1]); w.y = pack2<FKLHIP_F16>(x[2], x[3]); }
        const uint32_t token = row / a.q_heads, head = row - token * a.q_heads;
        *reinterpret_cast<uint2_t*>(a.out.data + int64_t(token) * a.out.token_stride + int64_t(head) * a.out.head_stride + d * 2) = w;
    }
    if (lane == 0 && a.lse) a.lse[row] = (top + __builtin_log2f(sum)) * 0.6931471805599453f;
}

} // namespace

int launch_merge(const AttentionArgs& a, uint32_t head_dim, void* stream) {
    const uint32_t rows = a.tokens * a.q_heads;
    k_merge<<<dim3((rows + 3) / 4), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a, head_dim);
    return int(hipGetLastError());
}

} // namespace fkattn
