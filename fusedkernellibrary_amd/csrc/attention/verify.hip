// verify.hip -- drafted tokens against the target's probabilities, and the token that comes behind the accepted ones.
//
// Mathematics. From a sequence's first row on, the children of the row that the path has come to are asked in their order: child t
// with token x is accepted if p(x) > u_t q_t(x), where p is the target's row of its parent and q_t the distribution it was drafted from; or,
// without one, if p(x) > u_t (1 - what the refused children in front of it had). Behind the last accepted row a token is drawn from
// w = max(p - q_t, 0) (t refused), p without the refused children's tokens, or p (nobody was asked): the first whose running
// sum exceeds u times the whole sum. So the tokens are distributed as if drawn from the target's rows one by one.
//
// Sums are in 64 bits: a drawn token is a whole number, which a sum's rounding must not decide. (A sum of 10^5 float32 weights in
// 32 bits is off by up to 10^-3 of itself in the worst order; in 64 bits a border is met with a chance of 10^-11.)
//
// Two launches. The first cuts a row into chunks, one to a workgroup; each finds the path for itself (a wave, by a few gathers that
// the lanes make together: less than a launch of its own) and adds its chunk up. The second, a workgroup to a sequence, finds
// the chunk and then the token in it. Bound by memory where the batch is large, else by the trips to memory one behind the other:
// 4.6 + 4.8 us for one chain of 5 over 32000 tokens (float32), 5.6 + 4.7 for 24 trees over 100003 (bfloat16), 15.1 + 6.3 for 64 chains of
// up to 8 over 131072 (67 MB at the most, 4.4 TB/s with the path in front). The second's scans are in registers, by moves between lanes:
// with a wave's weights added in LDS it took 33 to 72 us. One launch, a workgroup of 1024 to a sequence, was slower but for many short
// rows: 23.0 us for one sequence over 131072 (8.7 in two launches), 11.7 over 32000 (9.1), 18.5 for 256 over 32000 (21.3).
#include <type_traits>

#include "attention_device.hpp"
#include "step_common.hpp"

namespace fkattn {
namespace {

constexpr uint32_t kThreads = 256, kPerThread = 16, kChunk = kThreads * kPerThread;

template <int TYPE> constexpr uint32_t kSize = TYPE == FKLHIP_F32 ? 4 : 2;
template <int TYPE> constexpr uint32_t kRun = 16 / kSize<TYPE>;             // elements of a load
template <int TYPE> constexpr uint32_t kRuns = kPerThread / kRun<TYPE>;

// A probability: what is no number above 0 counts as 0.
__device__ __forceinline__ float as_probability(float x) { return x > 0.0f && x < __builtin_inff() ? x : 0.0f; }
template <int TYPE> __device__ __forceinline__ float element(const char* row, uint32_t i) {
    if constexpr (TYPE == FKLHIP_F32) {
        return as_probability(*reinterpret_cast<const float*>(row + size_t(i) * 4));
    } else {
        float a, b;
        unpack2<TYPE>(*reinterpret_cast<const uint16_t*>(row + size_t(i) * 2), a, b);
        return as_probability(a);
    }
}
typedef uint4_t aligned4_t __attribute__((aligned(4)));
typedef uint4_t aligned2_t __attribute__((aligned(2)));
// A run of a row from element i on; elements behind the row are 0. (Rows begin at any element: 16 bytes at a time all the same.)
template <int TYPE> __device__ __forceinline__ void load_run(const char* row, uint32_t i, uint32_t vocab, float (&x)[kRun<TYPE>]) {
    using loose_t = std::conditional_t<TYPE == FKLHIP_F32, aligned4_t, aligned2_t>;
    if (i + kRun<TYPE> <= vocab) {
        const uint4_t w = *reinterpret_cast<const loose_t*>(row + size_t(i) * kSize<TYPE>);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (TYPE == FKLHIP_F32) x[k] = __builtin_bit_cast(float, uint32_t(w[k]));
            else unpack2<TYPE>(w[k], x[2 * k], x[2 * k + 1]);
        }
#pragma unroll
        for (uint32_t k = 0; k < kRun<TYPE>; ++k) x[k] = as_probability(x[k]);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < kRun<TYPE>; ++k) x[k] = i + k < vocab ? element<TYPE>(row, i + k) : 0.0f;
    }
}
__device__ __forceinline__ float as_uniform(float u) { return u > 0.0f ? __builtin_fminf(u, 1.0f - 0x1p-24f) : 0.0f; }

struct Place { uint32_t first, count; };
__device__ __forceinline__ Place place_of(const VerifyArgs& a, uint32_t b) {
    const int32_t lo = a.q_start[b], hi = a.q_start[b + 1];
    Place p;
    p.first = lo < 0 ? 0u : min(uint32_t(lo), a.tokens);
    const int32_t n = hi - int32_t(p.first);
    p.count = hi < 0 || n < 0 ? 0u : min(min(uint32_t(n), a.max_new), a.tokens - p.first);
    return p;
}

// What the path of a sequence leads to. `against`: the refused row whose q is taken off, or -1.
struct Outcome { int32_t here, against, refused, count; };
// What the second launch needs of it, rows counted from the first of all; the refused children's tokens stand behind.
struct Record { int32_t here, against, refused, count; float u; int32_t none[3]; };
static_assert(sizeof(Record) == kVerifyRecord * 4);

__device__ __forceinline__ double of_lane(double v, uint32_t lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(int(uint32_t(u)), int(lane)), hi = __builtin_amdgcn_readlane(int(uint32_t(u >> 32)), int(lane));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// Sums of a wave's lanes up to and with each.
template <int CTRL, int ROWS> __device__ __forceinline__ double add_moved(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CTRL, ROWS, 0xf, false)), hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CTRL, ROWS, 0xf, false));
    return v + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double scan_lanes(double v) {
    v = add_moved<0x111, 0xf>(v);                              // row_shr 1, 2, 4, 8: within sixteen lanes
    v = add_moved<0x112, 0xf>(v);
    v = add_moved<0x114, 0xf>(v);
    v = add_moved<0x118, 0xf>(v);
    v = add_moved<0x142, 0xa>(v);                              // row_bcast 15: the second and fourth sixteen get the one before
    return add_moved<0x143, 0xc>(v);                           // row_bcast 31: the upper half gets the lower
}

// A wave's walk from a sequence's first row; path and refused are in LDS.
template <int TYPE> __device__ __forceinline__ Outcome find_path(const VerifyArgs& a, const Place& p, uint32_t lane, int32_t* path, int32_t* refused) {
    Outcome o{0, -1, 0, 1};
    double rest = 1.0;
    if (lane == 0) path[0] = 0;
    for (uint32_t t0 = 0; t0 < p.count; t0 += 64) {
        const uint32_t t = t0 + lane, row = p.first + t;
        int32_t parent = -1, id = -1;
        float u = 0.0f;
        if (t > 0 && t < p.count) {
            parent = a.parents ? a.parents[row] : int32_t(t) - 1;
            id = a.ids[row];
            u = as_uniform(a.uniforms[row]);
            if (parent < 0 || uint32_t(parent) >= t) parent = -1;
        }
        float prob = 0.0f, drafted = 0.0f;
        if (parent >= 0 && uint32_t(id) < a.vocab) {
            prob = element<TYPE>(a.target + int64_t(p.first + parent) * a.target_stride, uint32_t(id));
            if (a.draft) drafted = element<TYPE>(a.draft + int64_t(row) * a.draft_stride, uint32_t(id));
        }
        // (a token that an elder child had, among the 64 in front, was refused with it)
        if (parent == o.here)
            for (int32_t i = 0; i < o.refused; ++i)
                if (refused[i] == id) prob = 0.0f;
        uint64_t asked = __ballot(parent == o.here);
        while (asked) {
            const uint32_t s = __builtin_ctzll(asked);
            const double pd = of_lane(double(prob), s), ud = of_lane(double(u), s), qd = of_lane(double(drafted), s);
            const int32_t its = __builtin_amdgcn_readlane(id, int(s));
            if (pd > ud * (a.draft ? qd : rest)) {
                o.here = int32_t(t0 + s);
                o.refused = 0;
                o.against = -1;
                rest = 1.0;
                if (lane == 0) path[o.count] = o.here;
                ++o.count;
                asked = __ballot(parent == o.here);
            } else {
                if (a.draft) o.against = int32_t(t0 + s);
                if (lane == 0) refused[o.refused] = its;
                ++o.refused;
                rest -= pd;
                if (id == its && lane > s && parent == o.here) prob = 0.0f;
                asked &= asked - 1;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
    return o;
}

// A thread's weights of a chunk: run k holds elements chunk * kChunk + (k * kThreads + thread) * kRun ..
template <int TYPE> struct Weights {
    double w[kRuns<TYPE>][kRun<TYPE>];
    static __device__ __forceinline__ uint32_t at(uint32_t chunk, uint32_t k) { return chunk * kChunk + (k * kThreads + threadIdx.x) * kRun<TYPE>; }
    __device__ __forceinline__ void load(const char* p, const char* q, uint32_t chunk, uint32_t vocab) {
        float x[kRuns<TYPE>][kRun<TYPE>], y[kRuns<TYPE>][kRun<TYPE>];
#pragma unroll
        for (uint32_t k = 0; k < kRuns<TYPE>; ++k) {
            load_run<TYPE>(p, at(chunk, k), vocab, x[k]);
            if (q) load_run<TYPE>(q, at(chunk, k), vocab, y[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < kRuns<TYPE>; ++k)
#pragma unroll
            for (uint32_t i = 0; i < kRun<TYPE>; ++i) w[k][i] = q ? __builtin_fmax(double(x[k][i]) - double(y[k][i]), 0.0) : double(x[k][i]);
    }
    __device__ __forceinline__ void clear(uint32_t chunk, uint32_t id) {
#pragma unroll
        for (uint32_t k = 0; k < kRuns<TYPE>; ++k)
#pragma unroll
            for (uint32_t i = 0; i < kRun<TYPE>; ++i)
                if (at(chunk, k) + i == id) w[k][i] = 0.0;
    }
    __device__ __forceinline__ double sum(uint32_t k) const {
        double s = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kRun<TYPE>; ++i) s += w[k][i];
        return s;
    }
};

// The sum of a workgroup's values, for every thread.
__device__ __forceinline__ double sum_of_all(double v, double* waves) {
    v = scan_lanes(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    return (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

template <int TYPE> __global__ __launch_bounds__(kThreads) void k_verify_sums(const VerifyArgs a) {
    extern __shared__ int32_t lists[];                                       // path and refused tokens, max_new each
    __shared__ Outcome shared;
    __shared__ double waves[4];
    const uint32_t chunk = blockIdx.x, b = blockIdx.y;
    const Place p = place_of(a, b);
    int32_t *path = lists, *refused = lists + a.max_new;
    if (p.count == 0) {
        if (chunk == 0) {
            for (uint32_t i = threadIdx.x; i < a.max_new; i += kThreads) a.path[size_t(b) * a.max_new + i] = a.out[size_t(b) * a.max_new + i] = -1;
            if (threadIdx.x == 0) {
                a.count[b] = 0;
                a.record[size_t(b) * (kVerifyRecord + a.max_new) + 3] = 0;
            }
        }
        return;
    }
    if (threadIdx.x < 64) {
        const Outcome o = find_path<TYPE>(a, p, threadIdx.x, path, refused);
        if (threadIdx.x == 0) shared = o;
    }
    __syncthreads();
    const Outcome o = shared;
    if (chunk == 0) {
        int32_t* record = a.record + size_t(b) * (kVerifyRecord + a.max_new);
        for (uint32_t i = threadIdx.x; i < a.max_new; i += kThreads) {
            const bool kept = int32_t(i) < o.count;
            a.path[size_t(b) * a.max_new + i] = kept ? path[i] : -1;
            a.out[size_t(b) * a.max_new + i] = int32_t(i) + 1 < o.count ? a.ids[p.first + path[i + 1]] : -1;
            if (int32_t(i) < o.refused) record[kVerifyRecord + i] = refused[i];
        }
        if (threadIdx.x == 0) {
            a.count[b] = o.count;
            const int32_t first = int32_t(p.first);
            *reinterpret_cast<Record*>(record) = {first + o.here, o.against < 0 ? -1 : first + o.against, a.draft ? 0 : o.refused, o.count, as_uniform(a.uniforms[first]), {0, 0, 0}};
        }
    }
    Weights<TYPE> w;
    w.load(a.target + int64_t(p.first + o.here) * a.target_stride, o.against >= 0 ? a.draft + int64_t(p.first + o.against) * a.draft_stride : nullptr, chunk, a.vocab);
    if (!a.draft)
        for (int32_t i = 0; i < o.refused; ++i) w.clear(chunk, uint32_t(refused[i]));
    double s = 0.0;
#pragma unroll
    for (uint32_t k = 0; k < kRuns<TYPE>; ++k) s += w.sum(k);
    s = sum_of_all(s, waves);
    if (threadIdx.x == 0) a.sums[size_t(b) * a.chunks + chunk] = s;
}

// Where a running sum exceeds `share` of them all: the chunk, the sum in front of it and the border; chunk < 0: all are 0.
struct Chunk { int32_t chunk; double front, border; };
__device__ __forceinline__ Chunk find_chunk(const double* sums, uint32_t chunks, float share, uint32_t lane) {
    // (every wave for itself: there is nothing to wait for)
    double own = lane < chunks ? sums[lane] : 0.0, upto = scan_lanes(own), all = of_lane(upto, 63);
    for (uint32_t c0 = 64; c0 < chunks; c0 += 64) all += of_lane(scan_lanes(c0 + lane < chunks ? sums[c0 + lane] : 0.0), 63);
    Chunk f{-1, 0.0, double(share) * all};
    if (!(all > 0.0)) return f;
    double before = 0.0;
    for (uint32_t c0 = 0;;) {
        const double in_front = before + (upto - own);
        const uint64_t some = __ballot(own > 0.0), over = __ballot(own > 0.0 && before + upto > f.border);
        if (over || some) {
            const uint32_t at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            f.chunk = int32_t(c0 + at);
            f.front = of_lane(in_front, at);
            if (over) return f;                                              // (else the last that has something, if none is over)
        }
        before += of_lane(upto, 63);
        c0 += 64;
        if (c0 >= chunks) return f;
        own = c0 + lane < chunks ? sums[c0 + lane] : 0.0;
        upto = scan_lanes(own);
    }
}

template <int TYPE> __global__ __launch_bounds__(kThreads) void k_verify_pick(const VerifyArgs a) {
    __shared__ double waves[4], runs[kRuns<TYPE>][4];
    __shared__ uint32_t found[8], last[8];
    const uint32_t b = blockIdx.x, thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
    const int32_t* record = a.record + size_t(b) * (kVerifyRecord + a.max_new);
    const Record o = *reinterpret_cast<const Record*>(record);
    if (o.count == 0) return;
    double* sums = a.sums + size_t(b) * a.chunks;
    const char *target = a.target + int64_t(o.here) * a.target_stride, *draft = o.against >= 0 ? a.draft + int64_t(o.against) * a.draft_stride : nullptr;
    Weights<TYPE> w;
    Chunk f = find_chunk(sums, a.chunks, o.u, lane);
    const bool whole = f.chunk < 0;
    if (whole) {
        // no weight is left: the target's row as it is
        __syncthreads();
        for (uint32_t c = 0; c < a.chunks; ++c) {
            w.load(target, nullptr, c, a.vocab);
            double s = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < kRuns<TYPE>; ++k) s += w.sum(k);
            s = sum_of_all(s, waves);
            if (thread == 0) sums[c] = s;
        }
        __syncthreads();
        f = find_chunk(sums, a.chunks, o.u, lane);
    }
    if (f.chunk < 0) {
        if (thread == 0) a.out[size_t(b) * a.max_new + o.count - 1] = -1;
        return;
    }
    const uint32_t chunk = uint32_t(f.chunk);
    w.load(target, whole ? nullptr : draft, chunk, a.vocab);
    if (!whole)
        for (int32_t i = 0; i < o.refused; ++i) w.clear(chunk, uint32_t(record[kVerifyRecord + i]));
    double front[kRuns<TYPE>];
#pragma unroll
    for (uint32_t k = 0; k < kRuns<TYPE>; ++k) {
        const double run = w.sum(k), upto = scan_lanes(run);
        if (lane == 63) runs[k][wave] = upto;
        front[k] = upto - run;
    }
    __syncthreads();
    // the first element at which the sum is over the border; the last that has something, if rounding leaves none
    uint32_t first = 0xffffffffu, some = 0;
    double before = f.front;
#pragma unroll
    for (uint32_t k = 0; k < kRuns<TYPE>; ++k) {
        double sum = before;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const double its = runs[k][i];
            if (i < wave) sum += its;
            before += its;
        }
        sum += front[k];
#pragma unroll
        for (uint32_t i = 0; i < kRun<TYPE>; ++i) {
            sum += w.w[k][i];
            const uint32_t at = w.at(chunk, k) + i;
            if (w.w[k][i] > 0.0) {
                some = at;
                if (sum > f.border) first = min(first, at);
            }
        }
    }
    first = reduce_lanes<32>(first, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
    some = max_lanes<32>(some);
    if ((lane & 31) == 0) {
        found[wave * 2 + lane / 32] = first;
        last[wave * 2 + lane / 32] = some;
    }
    __syncthreads();
    if (thread == 0) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            first = min(first, found[i]);
            some = max(some, last[i]);
        }
        a.out[size_t(b) * a.max_new + o.count - 1] = int32_t(first != 0xffffffffu ? first : some);
    }
}

template <int TYPE> int start_verify(const VerifyArgs& a, void* stream) {
    if (const int rc = launch(k_verify_sums<TYPE>, dim3(a.chunks, a.batch), dim3(kThreads), stream, a, a.max_new * 8)) return rc;
    return launch(k_verify_pick<TYPE>, dim3(a.batch), dim3(kThreads), stream, a);
}

} // namespace

uint32_t verify_chunks(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }

int launch_verify(const VerifyArgs& a, int type, void* stream, Launched& info) {
    info = {"verify_drafts", {a.chunks, a.batch, 1}, {kThreads, 1, 1}, a.max_new * 8};
    if (type == FKLHIP_F32) return start_verify<FKLHIP_F32>(a, stream);
    return type == FKLHIP_BF16 ? start_verify<FKLHIP_BF16>(a, stream) : start_verify<FKLHIP_F16>(a, stream);
}

} // namespace fkattn
