// Routing of rows to experts on the CUDA cores: scores and top-k (moe_route_kernel), their
// gradient (moe_route_backward_kernel), the stable order of rows by group (group_rows_kernel)
// and the weighted sum that brings expert rows back to their tokens, with its gradient.
//
// All of them move far more bytes than they compute; what bounds the small ones is the launch.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gemm_umma.cuh"  // detail::OutTraits

namespace ckl {

constexpr int kMaxExperts = 1024;    // 32 per lane
constexpr int kMaxTopK = 32;         // one lane per choice
constexpr int kMaxRouteGroups = 32;  // one lane per expert group
constexpr int kRouteWarps = 4;

struct RouteParams {
    const void* logits;
    const float* bias;  // per expert, or nullptr
    float* weights;
    int* experts;
    int ldl;
    int tokens, n_experts, top_k;
    int groups, top_groups;
    int group_size;         // experts per group
    float inv_group_size;
    int sigmoid, renormalise;
    float scale;
};

namespace detail {

constexpr float kNegInf = -__builtin_huge_valf();

// Order-preserving map of a finite key to unsigned integers; 0 stands for "never chosen".
// -0 and +0 are equal keys, so they are made the same number first.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(double x) {
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(v >> 32));
    const uint32_t lo = __reduce_max_sync(
        0xFFFFFFFFu, static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
    return (static_cast<unsigned long long>(hi) << 32) | lo;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    }
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    }
    return v;
}
__device__ __forceinline__ float warp_maxf(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    }
    return v;
}

// A logit as the operators see it: NaN counts as -inf (never chosen, score 0) and +inf as the
// largest finite number.
__device__ __forceinline__ float clean_logit(float x) {
    return x != x ? kNegInf : fminf(x, 3.402823466e38f);
}

__device__ __forceinline__ float sigmoidf(float x) { return 1.0f / (1.0f + expf(-x)); }

// Shares p_j of the chosen scores, p_j = s_j / sum of s (lane j holds choice j; `some` is false
// on lanes without one).  softmax: the row's maximum and sum cancel, so the shares come from
// the chosen logits alone and cannot underflow together.  sigmoid: far below zero
// sigmoid(l) = e^l to more digits than FP32 holds, so there the shares are the same softmax.
__device__ __forceinline__ float chosen_share(float logit, bool some, bool sigmoid) {
    const float top = warp_maxf(some ? logit : kNegInf);
    const bool direct = sigmoid && top > -30.0f;
    const float e = some ? (direct ? sigmoidf(logit) : expf(logit - top)) : 0.0f;
    const float sum = warp_sum(e);
    return sum > 0.0f ? e / sum : 0.0f;
}

}  // namespace detail

namespace detail {

// e / group size, exact for e < 2^20.
__device__ __forceinline__ int group_of(const RouteParams& p, int e) {
    return __float2int_rz((static_cast<float>(e) + 0.5f) * p.inv_group_size);
}

// Which groups take part: bit g.  A group's score is the sum of its two best keys; `keys` is shared
// memory (index e + group of e, so that the lanes' scans start in different banks), read by a few
// neighbouring lanes per group.
__device__ __forceinline__ uint32_t choose_groups(const RouteParams& p, const double* keys, int lane) {
    const double none = -__builtin_huge_val();
    const int size = p.group_size;
    int shift = 0;  // 2^shift lanes per group
    while ((2 << shift) * p.groups <= 32) {
        ++shift;
    }
    const int per = 1 << shift;
    const int g = lane >> shift;
    double first = none, second = none;
    if (g < p.groups) {
        for (int i = lane & (per - 1); i < size; i += per) {
            const double v = keys[g * (size + 1) + i];
            second = v > first ? first : (v > second ? v : second);
            first = v > first ? v : first;
        }
    }
    for (int d = 1; d < per; d <<= 1) {
        const double f = __shfl_xor_sync(0xFFFFFFFFu, first, d);
        const double s = __shfl_xor_sync(0xFFFFFFFFu, second, d);
        const double lose = f > first ? first : f;
        const double run = f > first ? s : second;
        first = f > first ? f : first;
        second = lose > run ? lose : run;
    }
    unsigned long long mine = 0ull;
    if (g < p.groups && (lane & (per - 1)) == 0 && first != none) {
        mine = order_key(first + (second == none ? 0.0 : second));
    }
    uint32_t kept = 0;
    for (int r = 0; r < p.top_groups; ++r) {
        const unsigned long long best = warp_max(mine);
        if (best == 0ull) {
            break;
        }
        const int winner = __ffs(__ballot_sync(0xFFFFFFFFu, mine == best)) - 1;
        kept |= 1u << (winner >> shift);
        if (lane == winner) {
            mine = 0ull;
        }
    }
    return kept;
}

// Bitonic sort over the lanes of a warp, largest first, equal keys by index.
__device__ __forceinline__ void sort_lanes(unsigned long long* key, uint32_t* index, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
        for (int stride = size / 2; stride > 0; stride /= 2) {
            const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, *key, stride);
            const uint32_t i = __shfl_xor_sync(0xFFFFFFFFu, *index, stride);
            const bool mine_first = *key > k || (*key == k && *index < i);
            const bool want_first = ((lane & stride) == 0) == ((lane & size) == 0);
            if (mine_first != want_first) {
                *key = k;
                *index = i;
            }
        }
    }
}
__device__ __forceinline__ uint32_t sort_lanes(uint32_t key, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
        for (int stride = size / 2; stride > 0; stride /= 2) {
            const uint32_t k = __shfl_xor_sync(0xFFFFFFFFu, key, stride);
            const bool want_larger = ((lane & stride) == 0) == ((lane & size) == 0);
            key = want_larger ? max(key, k) : min(key, k);
        }
    }
    return key;
}

// The top_k largest keys (0: never chosen), ties to the lowest index: lane j gets choice j, or -1.
// The top_k-th largest of the lanes' best keys (their upper words) bounds the answer from below; the
// few keys that reach it are gathered, one per lane, and sorted.  `room` is shared memory for 32
// keys and indices.  More than 32 such keys (large top_k, many equal upper words): one pick after
// the other.
template <int NV>
__device__ __forceinline__ int choose_experts(const RouteParams& p, unsigned long long (&key)[NV],
                                              unsigned long long* room, int lane) {
    unsigned long long candidate;
    uint32_t index;
    int count;
    if constexpr (NV == 1) {
        candidate = key[0];
        index = static_cast<uint32_t>(lane);
        count = 32;
    } else {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            best = max(best, static_cast<uint32_t>(key[i] >> 32));
        }
        const uint32_t bound = max(1u, __shfl_sync(0xFFFFFFFFu, sort_lanes(best, lane), p.top_k - 1));
        uint32_t* room_index = reinterpret_cast<uint32_t*>(room + 32);
        count = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool reaches = static_cast<uint32_t>(key[i] >> 32) >= bound;
            const uint32_t which = __ballot_sync(0xFFFFFFFFu, reaches);
            const int at = count + __popc(which & ((1u << lane) - 1u));
            if (reaches && at < 32) {
                room[at] = key[i];
                room_index[at] = static_cast<uint32_t>(i * 32 + lane);
            }
            count += __popc(which);
        }
        __syncwarp();
        candidate = lane < count ? room[lane] : 0ull;
        index = lane < count ? room_index[lane] : 0xFFFFFFFFu;
        __syncwarp();
    }
    if (count <= 32) {
        sort_lanes(&candidate, &index, lane);
        return lane < p.top_k && candidate != 0ull ? static_cast<int>(index) : -1;
    }
    int chosen = -1;
    for (int j = 0; j < p.top_k; ++j) {
        unsigned long long best = 0ull;
        int at = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        }
        const unsigned long long all = warp_max(best);
        if (all == 0ull) {
            break;
        }
        const uint32_t e = __reduce_min_sync(
            0xFFFFFFFFu, best == all ? static_cast<uint32_t>(at * 32 + lane) : 0xFFFFFFFFu);
        if (lane == j) {
            chosen = static_cast<int>(e);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            key[i] = static_cast<int>(e) == i * 32 + lane ? 0ull : key[i];
        }
    }
    return chosen;
}

// 1 / d to 64 bits for d in [1, 1e30]: the FP32 reciprocal and two Newton steps (2^-23, 2^-46, then
// rounding).
__device__ __forceinline__ double reciprocal(double d) {
    double y = static_cast<double>(__frcp_rn(static_cast<float>(d)));
    y = fma(y, fma(-d, y, 1.0), y);
    return fma(y, fma(-d, y, 1.0), y);
}

}  // namespace detail

// One warp per token; lane l holds experts l, l + 32, ...  Which experts are chosen is a whole-number
// answer, so rounding must not decide it: without a bias and groups the logits themselves are
// compared (the scores are monotone in them); with them (kWide) score + bias and the groups' sums
// are formed in 64 bits, for every token: FP32 keys with an error bound and 64-bit ones where they
// could not decide (27 of 8192 tokens) were slower, since those few warps fetched the rarely used
// code while the launch waited for them (12 of 32 us).
template <typename T, int NV, bool kWide>
__global__ void __launch_bounds__(32 * kRouteWarps, NV <= 8 ? 10 : 4) moe_route_kernel(const RouteParams p) {
    using Traits = detail::OutTraits<T>;
    extern __shared__ __align__(16) uint8_t route_smem[];
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const int token = static_cast<int>(blockIdx.x) * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    // per warp: 64-bit keys by expert (room for 32 candidates at least), then the row
    constexpr int kKeys = NV * 32 + kMaxRouteGroups;
    double* keys = reinterpret_cast<double*>(route_smem) + warp * kKeys;
    float* row = reinterpret_cast<float*>(route_smem + kRouteWarps * kKeys * 8) + warp * (NV * 32);
    const T* src = static_cast<const T*>(p.logits) + static_cast<size_t>(token) * p.ldl;

    float logit[NV];
    float top = detail::kNegInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = i * 32 + lane;
        logit[i] = e < p.n_experts ? detail::clean_logit(Traits::load(src + e)) : detail::kNegInf;
        top = fmaxf(top, logit[i]);
        row[e] = logit[i];
    }
    float inv_sum = 0.0f;
    if (!p.sigmoid) {
        top = detail::warp_maxf(top);
        if (!kWide && !p.renormalise) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                sum += logit[i] == detail::kNegInf ? 0.0f : expf(logit[i] - top);
            }
            sum = detail::warp_sum(sum);
            inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
        }
    }
    unsigned long long key[NV];
    if constexpr (kWide) {
        const double none = -__builtin_huge_val();
        double score[NV];
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const double l = static_cast<double>(logit[i]);
            const double x = exp(p.sigmoid ? -l : l - static_cast<double>(top));
            if (p.sigmoid) {
                const double d = 1.0 + x;
                score[i] = d < 1e30 ? detail::reciprocal(d) : 1.0 / d;
            } else {
                score[i] = logit[i] == detail::kNegInf ? 0.0 : x;
                sum += score[i];
            }
        }
        if (!p.sigmoid) {
            sum = detail::warp_sum(sum);
            const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
            inv_sum = static_cast<float>(inv);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                score[i] *= inv;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 32 + lane;
            if (p.bias != nullptr && e < p.n_experts) {
                score[i] += static_cast<double>(p.bias[e]);
            }
            // (a bias of -inf or NaN takes its expert out of the choice)
            const bool may = logit[i] != detail::kNegInf && score[i] > none;
            key[i] = may ? detail::order_key(score[i]) : 0ull;
            if (p.groups > 1 && e < p.n_experts) {
                keys[e + detail::group_of(p, e)] = may ? score[i] : none;
            }
        }
        if (p.groups > 1) {
            __syncwarp();
            const uint32_t kept = detail::choose_groups(p, keys, lane);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = i * 32 + lane;
                if (e < p.n_experts && !((kept >> detail::group_of(p, e)) & 1u)) {
                    key[i] = 0ull;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            key[i] = logit[i] == detail::kNegInf
                         ? 0ull
                         : static_cast<unsigned long long>(detail::order_key(logit[i])) << 32;
        }
    }
    const int chosen =
        detail::choose_experts<NV>(p, key, reinterpret_cast<unsigned long long*>(keys), lane);  // lane j: choice j
    __syncwarp();
    const bool some = chosen >= 0;
    const float l = some ? row[chosen] : detail::kNegInf;
    float w;
    if (p.renormalise) {
        w = detail::chosen_share(l, some, p.sigmoid != 0);
    } else if (p.sigmoid) {
        w = some ? detail::sigmoidf(l) : 0.0f;
    } else {
        w = some ? expf(l - top) * inv_sum : 0.0f;
    }
    if (lane < p.top_k) {
        const size_t at = static_cast<size_t>(token) * p.top_k + lane;
        p.weights[at] = some ? w * p.scale : 0.0f;
        p.experts[at] = chosen;
    }
}

struct RouteBackwardParams {
    const void* logits;
    const int* experts;
    const float* dweights;
    void* dlogits;
    int ldl, ldd;
    int tokens, n_experts, top_k;
    int sigmoid, renormalise;
    float scale;
};

// One warp per token; lane l holds experts l, l + 32, ...  With p_j the chosen scores' shares and d_j
// the incoming gradient:
//   softmax, renormalised   dl_j = scale p_j (d_j - sum d p)                  else 0
//   sigmoid, renormalised   dl_j = scale p_j (1 - s_j) (d_j - sum d p)        else 0
//   sigmoid                 dl_j = scale s_j (1 - s_j) d_j                    else 0
//   softmax                 dl_e = s_e (scale d_e - sum_j scale d_j s_j)      for every e
// (the choice itself and the bias get no gradient).  Only the last reads the whole row.
template <typename T, int NV>
__global__ void __launch_bounds__(32 * kRouteWarps)
moe_route_backward_kernel(const RouteBackwardParams p) {
    using Traits = detail::OutTraits<T>;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const int token = static_cast<int>(blockIdx.x) * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    const T* src = static_cast<const T*>(p.logits) + static_cast<size_t>(token) * p.ldl;
    T* dst = static_cast<T*>(p.dlogits) + static_cast<size_t>(token) * p.ldd;
    const bool whole_row = !p.sigmoid && !p.renormalise;
    int chosen = -1;
    float d = 0.0f;
    if (lane < p.top_k) {
        const size_t at = static_cast<size_t>(token) * p.top_k + lane;
        chosen = p.experts[at];
        d = p.dweights[at] * p.scale;
    }
    float x[NV], grad[NV];
    float top = detail::kNegInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = i * 32 + lane;
        x[i] = whole_row && e < p.n_experts ? detail::clean_logit(Traits::load(src + e)) : detail::kNegInf;
        top = fmaxf(top, x[i]);
        grad[i] = 0.0f;
    }
    const bool named = chosen >= 0 && chosen < p.n_experts;
    const float l = named ? detail::clean_logit(Traits::load(src + chosen)) : detail::kNegInf;
    const bool some = l != detail::kNegInf;
    d = some ? d : 0.0f;
    float dot = 0.0f, value;
    if (whole_row) {
        top = detail::warp_maxf(top);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = x[i] == detail::kNegInf ? 0.0f : expf(x[i] - top);
            sum += x[i];
        }
        sum = detail::warp_sum(sum);
        const float inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] *= inv_sum;  // the scores
        }
        dot = detail::warp_sum(some ? d * expf(l - top) * inv_sum : 0.0f);
        value = d;
    } else if (p.renormalise) {
        const float share = detail::chosen_share(l, some, p.sigmoid != 0);
        dot = detail::warp_sum(d * share);
        value = share * (d - dot) * (p.sigmoid && some ? detail::sigmoidf(-l) : 1.0f);
    } else {
        value = some ? d * detail::sigmoidf(l) * detail::sigmoidf(-l) : 0.0f;
    }
    // One choice at a time, so that the result does not depend on the order of threads even
    // where a row names an expert twice.
    for (int j = 0; j < p.top_k; ++j) {
        const float v = __shfl_sync(0xFFFFFFFFu, value, j);
        const int e = __shfl_sync(0xFFFFFFFFu, some ? chosen : -1, j);
        if (e >= 0 && (e & 31) == lane) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                grad[i] += i == (e >> 5) ? v : 0.0f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = i * 32 + lane;
        if (e < p.n_experts) {
            Traits::store(dst + e, whole_row ? x[i] * (grad[i] - dot) : grad[i]);
        }
    }
}

// ---- stable order of slots by group -------------------------------------------------------

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kMaxOrderCluster = 8;
constexpr int kOrderStaged = kOrderThreads * 8;  // slots of a CTA that are sorted in shared memory
constexpr int kOrderSteps = 8;  // of 32 slots that a warp holds in registers

namespace detail {

// s / d for 0 <= s < 2^31 and 1 <= d < 2^31 by a multiplication: with r = 2^64 / d rounded up,
// s r = 2^64 s / d + s e where 0 <= e < 1, and s e < 2^64 / d, so the upper word of s r is the quotient.
// (r of d = 1 does not fit in 64 bits: 0 stands for it.)
__host__ __device__ inline unsigned long long reciprocal_of(int d) {
    return d == 1 ? 0ull : ~0ull / static_cast<unsigned long long>(d) + 1ull;
}
__host__ __device__ inline int quotient(int s, unsigned long long r) {
    if (r == 0ull) {
        return s;
    }
    // the two halves of r one after the other: s < 2^32, so neither product passes 64 bits
    const unsigned long long n = static_cast<unsigned int>(s);
    return static_cast<int>((n * (r >> 32) + ((n * (r & 0xffffffffull)) >> 32)) >> 32);
}

}  // namespace detail

struct GroupRowsParams {
    const int* ids;
    int* offsets;
    int* rows;
    int* positions;
    int slots, groups;
    unsigned long long inv_row;  // reciprocal_of(slots_per_row)
    int staged;      // a CTA's slots fit in shared memory, sorted
    int warp_slots;  // consecutive slots of one warp, a multiple of 32
};

// A counting sort that keeps the order of slots inside a group, in one launch and without a
// workspace: one cluster of 1 to 8 CTAs; every warp owns a run of consecutive slots and counts
// its groups in shared memory, the counts are summed over warps and (through distributed
// shared memory) over CTAs, and each warp then walks its run again and hands out positions in
// slot order.  No result depends on the order of atomics: they only count.
// Slots whose id names no group come last, in slot order, behind offsets[groups].
__global__ void __launch_bounds__(kOrderThreads) group_rows_kernel(const GroupRowsParams p) {
    extern __shared__ __align__(16) int order_smem[];
    const int bins = p.groups + 1;
    int* hist = order_smem;                       // [warp][bin]
    int* total = hist + kOrderWarps * bins;       // [bin] of this CTA, read by the cluster
    int* start = total + bins;                    // [bin]
    int* warp_sums = start + bins;                // [32]
    int* local = warp_sums + kOrderWarps;         // [bin] first place in `sorted`
    int2* sorted = reinterpret_cast<int2*>(local + (bins + 1) / 2 * 2);  // (position, row), p.staged
    const int tid = static_cast<int>(threadIdx.x);
    const int warp = tid >> 5, lane = tid & 31;
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));

    for (int i = tid; i < kOrderWarps * bins; i += kOrderThreads) {
        hist[i] = 0;
    }
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    __syncthreads();
    const long long first =
        (static_cast<long long>(rank) * kOrderWarps + warp) * static_cast<long long>(p.warp_slots);
    const int begin = static_cast<int>(min(first, static_cast<long long>(p.slots)));
    const int end = static_cast<int>(min(first + p.warp_slots, static_cast<long long>(p.slots)));
    int* mine = hist + warp * bins;
    // The bins of kOrderSteps x 32 slots at a time, fetched together; the first batch is kept for the
    // second walk (it is the only one up to 65536 slots).
    auto fetch = [&](int from, int (&bin)[kOrderSteps]) {
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            const int s = from + i * 32 + lane;
            bin[i] = s < end ? p.ids[s] : 0;
        }
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            const int s = from + i * 32 + lane;
            bin[i] = s >= end ? -1 : bin[i] >= 0 && bin[i] < p.groups ? bin[i] : p.groups;
        }
    };
    int kept_bin[kOrderSteps];
    fetch(begin, kept_bin);
    for (int from = begin; from < end; from += 32 * kOrderSteps) {
        int bin[kOrderSteps];
        if (from == begin) {
#pragma unroll
            for (int i = 0; i < kOrderSteps; ++i) {
                bin[i] = kept_bin[i];
            }
        } else {
            fetch(from, bin);
        }
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            if (bin[i] >= 0) {
                atomicAdd(mine + bin[i], 1);
            }
        }
    }
    __syncthreads();
    for (int b = tid; b < bins; b += kOrderThreads) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < kOrderWarps; ++w) {
            const int c = hist[w * bins + b];
            hist[w * bins + b] = run;
            run += c;
        }
        total[b] = run;
    }
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
    // groups <= 1024 = the block's threads: thread b scans bin b; the bin of dropped slots
    // (b = groups) starts at the sum of all the others.
    int before = 0, all = 0;
    if (tid < p.groups) {
        for (uint32_t q = 0; q < size; ++q) {
            int v;
            asm volatile("ld.shared::cluster.s32 %0, [%1];"
                         : "=r"(v)
                         : "r"(ptx::map_to_cta(ptx::smem_u32(total + tid), q))
                         : "memory");
            before += q < rank ? v : 0;
            all += v;
        }
    }
    int scan = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, scan, d);
        scan += lane >= d ? v : 0;
    }
    if (lane == 31) {
        warp_sums[warp] = scan;
    }
    __syncthreads();
    if (warp == 0) {
        int v = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            v += lane >= d ? u : 0;
        }
        warp_sums[lane] = v;
    }
    __syncthreads();
    const int base = scan - all + (warp > 0 ? warp_sums[warp - 1] : 0);
    const int kept = warp_sums[kOrderWarps - 1];
    if (p.staged) {
        // The same scan over this CTA's own counts: where its slots of a bin lie in `sorted`.
        __syncthreads();
        const int own = tid < p.groups ? total[tid] : 0;
        int v = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            v += lane >= d ? u : 0;
        }
        if (lane == 31) {
            warp_sums[warp] = v;
        }
        __syncthreads();
        if (warp == 0) {
            int w = warp_sums[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up_sync(0xFFFFFFFFu, w, d);
                w += lane >= d ? u : 0;
            }
            warp_sums[lane] = w;
        }
        __syncthreads();
        if (tid < p.groups) {
            local[tid] = v - own + (warp > 0 ? warp_sums[warp - 1] : 0);
        }
        if (tid == 0) {
            local[p.groups] = warp_sums[kOrderWarps - 1];
        }
    }
    if (tid < p.groups) {
        start[tid] = base + before;
        if (rank == 0) {
            p.offsets[tid] = base;
        }
    }
    if (tid == 0) {
        int dropped_before = 0;
        for (uint32_t q = 0; q < rank; ++q) {
            int v;
            asm volatile("ld.shared::cluster.s32 %0, [%1];"
                         : "=r"(v)
                         : "r"(ptx::map_to_cta(ptx::smem_u32(total + p.groups), q))
                         : "memory");
            dropped_before += v;
        }
        start[p.groups] = kept + dropped_before;
        if (rank == 0) {
            p.offsets[p.groups] = kept;
        }
    }
    // All reads of the other CTAs' totals are done once every CTA is here.
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
    for (int from = begin; from < end; from += 32 * kOrderSteps) {
        int bin[kOrderSteps];
        if (from == begin) {
#pragma unroll
            for (int i = 0; i < kOrderSteps; ++i) {
                bin[i] = kept_bin[i];
            }
        } else {
            fetch(from, bin);
        }
        // Lanes with the same bin, from one ballot per bit of the bin (__match_any_sync took 100
        // cycles a step with 32 different bins: 26 of this kernel's 35 thousand at 65536 slots).
        uint32_t same[kOrderSteps];
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            same[i] = 0xFFFFFFFFu;
        }
        for (int b = 0; (p.groups >> b) != 0; ++b) {
#pragma unroll
            for (int i = 0; i < kOrderSteps; ++i) {
                const bool bit = (bin[i] >> b) & 1;
                const uint32_t set = __ballot_sync(0xFFFFFFFFu, bit);
                same[i] &= bit ? set : ~set;
            }
        }
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            same[i] &= __ballot_sync(0xFFFFFFFFu, bin[i] >= 0);  // lanes without a slot count nowhere
        }
#pragma unroll
        for (int i = 0; i < kOrderSteps; ++i) {
            const int s = from + i * 32 + lane;
            if (bin[i] >= 0) {
                const int in_bin = mine[bin[i]] + __popc(same[i] & ((1u << lane) - 1u));
                const int pos = start[bin[i]] + in_bin;
                p.positions[s] = pos;
                const int row = detail::quotient(s, p.inv_row);
                if (p.staged) {
                    sorted[local[bin[i]] + in_bin] = make_int2(pos, row);
                } else {
                    p.rows[pos] = row;
                }
            }
            __syncwarp();
            if (bin[i] >= 0 && lane == __ffs(same[i]) - 1) {
                mine[bin[i]] += __popc(same[i]);
            }
            __syncwarp();
        }
    }
    if (p.staged) {
        // Neighbours in `sorted` are neighbours in `rows` up to the end of a bin: the stores are runs
        // instead of 32 places per instruction.
        __syncthreads();
        const long long cta_first = static_cast<long long>(rank) * kOrderWarps * p.warp_slots;
        const int count = static_cast<int>(max(0ll, min(static_cast<long long>(kOrderWarps) * p.warp_slots,
                                                        static_cast<long long>(p.slots) - cta_first)));
        for (int i = tid; i < count; i += kOrderThreads) {
            const int2 v = sorted[i];
            p.rows[v.x] = v.y;
        }
    }
}

// ---- rows back to their tokens --------------------------------------------------------------

namespace detail {

// Eight consecutive elements on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    constexpr int U = OutTraits<T>::kVec;
#pragma unroll
    for (int h = 0; h < 8 / U; ++h) {
        float u[U];
        OutTraits<T>::load_vec(p + h * U, u);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            v[h * U + i] = u[i];
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    constexpr int U = OutTraits<T>::kVec;
#pragma unroll
    for (int h = 0; h < 8 / U; ++h) {
        OutTraits<T>::store_vec(p + h * U, v + h * U);
    }
}

}  // namespace detail

constexpr int kCombineThreads = 256;

struct CombineParams {
    const void* y;
    const int* positions;
    const float* weights;
    void* out;
    int tokens, top_k, n, y_rows;
    int ldy, ldo;
    const int* kept;  // or nullptr
};

namespace detail {

// Rows of y that exist: y_rows, or fewer where the device knows better (the positions behind the last
// group hold no expert's row, and nobody wrote them).
__device__ __forceinline__ int rows_that_exist(int y_rows, const int* kept) {
    return kept != nullptr ? min(y_rows, *kept) : y_rows;
}

}  // namespace detail

// out[t] = sum_j weights[t][j] * y[positions[t][j]], summed in FP32 in the order of j.  One
// thread per 8 columns of one token (kVec) or per column; memory-bound: y is read once.
// A position that names no row adds nothing, nor does a weight of 0: it may stand for a place that
// routing could not fill, whose row of y is whatever the memory held before.
template <typename T, typename OutT, bool kVec>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const CombineParams p) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    constexpr int V = kVec ? 8 : 1;
    const int units = kVec ? p.n / 8 : p.n;
    const long long id = static_cast<long long>(blockIdx.x) * kCombineThreads + threadIdx.x;
    const long long t = id / units;
    if (t >= p.tokens) {
        return;
    }
    const int col = static_cast<int>(id - t * units) * V;
    const T* y = static_cast<const T*>(p.y) + col;
    const int* pos = p.positions + t * p.top_k;
    const float* w = p.weights + t * p.top_k;
    const int rows = detail::rows_that_exist(p.y_rows, p.kept);
    float acc[V] = {};
#pragma unroll 8
    for (int j = 0; j < p.top_k; ++j) {
        const int at = pos[j];
        const float f = w[j];
        if (at < 0 || at >= rows || f == 0.0f) {
            continue;
        }
        const T* src = y + static_cast<size_t>(at) * p.ldy;
        if constexpr (kVec) {
            float v[V];
            detail::load8(src, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[i] = fmaf(f, v[i], acc[i]);
            }
        } else {
            acc[0] = fmaf(f, detail::OutTraits<T>::load(src), acc[0]);
        }
    }
    OutT* dst = static_cast<OutT*>(p.out) + static_cast<size_t>(t) * p.ldo + col;
    if constexpr (kVec) {
        detail::store8(dst, acc);
    } else {
        detail::OutTraits<OutT>::store(dst, acc[0]);
    }
}

struct CombineBackwardParams {
    const void* y;
    const int* positions;
    const float* weights;
    const void* dout;
    void* dy;
    float* dweights;
    int tokens, top_k, n, y_rows;
    int ldy, ldo, lddy;
    const int* kept;  // or nullptr
};

// One warp per slot (t, j): dy[positions[t][j]] = weights[t][j] * dout[t] and
// dweights[t][j] = <dout[t], y[positions[t][j]]> in one pass over y.  The slots of a token sit in
// one CTA, so dout comes from L1 after the first.  No sum leaves its warp: with one CTA per
// token and the choices' sums in registers, the two block-wide steps per token left the memory
// idle (2047 x 8 rows of 2048 columns: 43 us).
template <typename T, typename OutT, bool kVec>
__global__ void __launch_bounds__(kCombineThreads)
moe_combine_backward_kernel(const CombineBackwardParams p) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    constexpr int V = kVec ? 8 : 1;
    const int lane = static_cast<int>(threadIdx.x & 31);
    const long long slot = (static_cast<long long>(blockIdx.x) * kCombineThreads + threadIdx.x) >> 5;
    const long long t = slot / p.top_k;
    if (t >= p.tokens) {
        return;
    }
    const int at = p.positions[slot];
    const float w = p.weights[slot];
    const bool exists = at >= 0 && at < detail::rows_that_exist(p.y_rows, p.kept);
    float dot = 0.0f;
    if (exists) {
        const OutT* dout = static_cast<const OutT*>(p.dout) + static_cast<size_t>(t) * p.ldo;
        const T* src = static_cast<const T*>(p.y) + static_cast<size_t>(at) * p.ldy;
        T* dst = static_cast<T*>(p.dy) + static_cast<size_t>(at) * p.lddy;
#pragma unroll 4
        for (int col = lane * V; col < p.n; col += 32 * V) {
            if constexpr (kVec) {
                float g[V], v[V];
                detail::load8(dout + col, g);
                detail::load8(src + col, v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dot = fmaf(v[i], g[i], dot);
                    g[i] *= w;
                }
                detail::store8(dst + col, g);
            } else {
                const float g = detail::OutTraits<OutT>::load(dout + col);
                dot = fmaf(detail::OutTraits<T>::load(src + col), g, dot);
                detail::OutTraits<T>::store(dst + col, w * g);
            }
        }
    }
    dot = detail::warp_sum(dot);
    if (lane == 0) {
        p.dweights[slot] = dot;
    }
}

}  // namespace ckl
