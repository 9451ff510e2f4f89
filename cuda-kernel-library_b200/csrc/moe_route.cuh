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

// One warp per token.  Lane l holds the logits of experts l, l + 32, ...; each of the top_k
// picks is one redux over the lanes' best keys and one over the tied lanes' indices, so ties
// go to the lowest index.
//
// Which experts are chosen is a whole-number answer, so the keys must not be rounded into
// false ties: without a bias and groups the logits themselves are compared (the scores are
// monotone in them); with them (kWide) score + bias is formed in 64 bits.
template <typename T, int NV, bool kWide>
__global__ void __launch_bounds__(32 * kRouteWarps) moe_route_kernel(const RouteParams p) {
    using Traits = detail::OutTraits<T>;
    using Key = typename std::conditional<kWide, unsigned long long, uint32_t>::type;
    extern __shared__ __align__(16) uint8_t route_smem[];
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const int token = static_cast<int>(blockIdx.x) * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    const int e_count = p.n_experts;
    float* row = reinterpret_cast<float*>(route_smem) + warp * (NV * 32);
    const T* src = static_cast<const T*>(p.logits) + static_cast<size_t>(token) * p.ldl;

    float logit[NV];
    float top = detail::kNegInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = i * 32 + lane;
        logit[i] = e < e_count ? detail::clean_logit(Traits::load(src + e)) : detail::kNegInf;
        top = fmaxf(top, logit[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        row[i * 32 + lane] = logit[i];
    }
    const bool need_sum = !p.sigmoid && (kWide || !p.renormalise);
    float inv_sum = 0.0f;
    if (!p.sigmoid) {
        top = detail::warp_maxf(top);
        if (!kWide && need_sum) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                sum += logit[i] == detail::kNegInf ? 0.0f : expf(logit[i] - top);
            }
            sum = detail::warp_sum(sum);
            inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
        }
    }

    Key key[NV];
    if constexpr (kWide) {
        double score[NV];
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (logit[i] == detail::kNegInf) {
                score[i] = 0.0;
            } else if (p.sigmoid) {
                score[i] = 1.0 / (1.0 + exp(-static_cast<double>(logit[i])));
            } else {
                score[i] = exp(static_cast<double>(logit[i]) - static_cast<double>(top));
            }
            sum += score[i];
        }
        if (!p.sigmoid) {
            sum = detail::warp_sum(sum);
            inv_sum = sum > 0.0 ? static_cast<float>(1.0 / sum) : 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                score[i] = sum > 0.0 ? score[i] / sum : 0.0;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 32 + lane;
            if (p.bias != nullptr && e < e_count) {
                score[i] += static_cast<double>(__ldg(p.bias + e));
            }
            // (a bias of -inf or NaN takes its expert out of the choice)
            key[i] = logit[i] == detail::kNegInf || !(score[i] > -__builtin_huge_val())
                         ? 0ull
                         : detail::order_key(score[i]);
        }
        if (p.groups > 1) {
            // A group's score is the sum of its two best keys.  The keys pass through shared
            // memory so that a few neighbouring lanes can scan one group.
            double* keys = reinterpret_cast<double*>(route_smem + kRouteWarps * NV * 32 * 4) +
                           warp * (NV * 32 + kMaxRouteGroups);
            const int size = e_count / p.groups;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = i * 32 + lane;
                if (e < e_count) {
                    keys[e + e / size] = key[i] == 0ull ? -__builtin_huge_val() : score[i];
                }
            }
            __syncwarp();
            int per = 1;  // lanes per group, a power of two
            while (per * 2 * p.groups <= 32) {
                per *= 2;
            }
            const int g = lane / per;
            double first = -__builtin_huge_val(), second = first;
            if (g < p.groups) {
                for (int i = lane % per; i < size; i += per) {
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
            if (g < p.groups && lane % per == 0 && first != -__builtin_huge_val()) {
                mine = detail::order_key(first + (second == -__builtin_huge_val() ? 0.0 : second));
            }
            uint32_t kept = 0;
            for (int r = 0; r < p.top_groups; ++r) {
                const unsigned long long best = detail::warp_max(mine);
                if (best == 0ull) {
                    break;
                }
                const int winner = __ffs(__ballot_sync(0xFFFFFFFFu, mine == best)) - 1;
                kept |= 1u << (winner / per);
                if (lane == winner) {
                    mine = 0ull;
                }
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = i * 32 + lane;
                if (e < e_count && !((kept >> (e / size)) & 1u)) {
                    key[i] = 0;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            key[i] = logit[i] == detail::kNegInf ? 0u : detail::order_key(logit[i]);
        }
    }

    int chosen = -1;  // lane j: the j-th choice
    for (int j = 0; j < p.top_k; ++j) {
        Key best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        }
        const Key all = detail::warp_max(best);
        if (all == 0) {
            break;
        }
        const uint32_t e = __reduce_min_sync(
            0xFFFFFFFFu, best == all ? static_cast<uint32_t>(at * 32 + lane) : 0xFFFFFFFFu);
        if (lane == j) {
            chosen = static_cast<int>(e);
        }
        if (static_cast<int>(e & 31u) == lane) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i == static_cast<int>(e >> 5)) {
                    key[i] = 0;
                }
            }
        }
    }
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

// One warp per token.  With p_j the chosen scores' shares and d_j the incoming gradient:
//   softmax, renormalised   dl_j = scale p_j (d_j - sum d p)                  else 0
//   sigmoid, renormalised   dl_j = scale p_j (1 - s_j) (d_j - sum d p)        else 0
//   sigmoid                 dl_j = scale s_j (1 - s_j) d_j                    else 0
//   softmax                 dl_e = s_e (scale d_e - sum_j scale d_j s_j)      for every e
// (the choice itself and the bias get no gradient).  Only the last reads the whole row.
template <typename T>
__global__ void __launch_bounds__(32 * kRouteWarps)
moe_route_backward_kernel(const RouteBackwardParams p) {
    using Traits = detail::OutTraits<T>;
    extern __shared__ __align__(16) uint8_t route_smem[];
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const int token = static_cast<int>(blockIdx.x) * kRouteWarps + warp;
    if (token >= p.tokens) {
        return;
    }
    float* grad = reinterpret_cast<float*>(route_smem) + warp * p.n_experts;
    const T* src = static_cast<const T*>(p.logits) + static_cast<size_t>(token) * p.ldl;
    T* dst = static_cast<T*>(p.dlogits) + static_cast<size_t>(token) * p.ldd;
    for (int e = lane; e < p.n_experts; e += 32) {
        grad[e] = 0.0f;
    }
    int chosen = -1;
    float d = 0.0f, l = detail::kNegInf;
    if (lane < p.top_k) {
        const size_t at = static_cast<size_t>(token) * p.top_k + lane;
        chosen = p.experts[at];
        if (chosen >= 0 && chosen < p.n_experts) {
            l = detail::clean_logit(Traits::load(src + chosen));
            d = p.dweights[at] * p.scale;
        }
    }
    const bool some = l != detail::kNegInf;
    d = some ? d : 0.0f;
    float top = 0.0f, inv_sum = 0.0f, dot = 0.0f;
    const bool whole_row = !p.sigmoid && !p.renormalise;
    float value = 0.0f;
    if (whole_row) {
        float m = detail::kNegInf;
        for (int e = lane; e < p.n_experts; e += 32) {
            m = fmaxf(m, detail::clean_logit(Traits::load(src + e)));
        }
        top = detail::warp_maxf(m);
        float sum = 0.0f;
        for (int e = lane; e < p.n_experts; e += 32) {
            const float x = detail::clean_logit(Traits::load(src + e));
            sum += x == detail::kNegInf ? 0.0f : expf(x - top);
        }
        sum = detail::warp_sum(sum);
        inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
        dot = detail::warp_sum(some ? d * expf(l - top) * inv_sum : 0.0f);
        value = d;
    } else if (p.renormalise) {
        const float share = detail::chosen_share(l, some, p.sigmoid != 0);
        dot = detail::warp_sum(d * share);
        value = share * (d - dot) * (p.sigmoid && some ? detail::sigmoidf(-l) : 1.0f);
    } else {
        value = some ? d * detail::sigmoidf(l) * detail::sigmoidf(-l) : 0.0f;
    }
    __syncwarp();
    // One choice at a time, so that the result does not depend on the order of threads even
    // where a row names an expert twice.
    for (int j = 0; j < p.top_k; ++j) {
        const float v = __shfl_sync(0xFFFFFFFFu, value, j);
        const int e = __shfl_sync(0xFFFFFFFFu, some ? chosen : -1, j);
        if (lane == 0 && e >= 0) {
            grad[e] += v;
        }
    }
    __syncwarp();
    for (int e = lane; e < p.n_experts; e += 32) {
        float g = grad[e];
        if (whole_row) {
            const float x = detail::clean_logit(Traits::load(src + e));
            g = x == detail::kNegInf ? 0.0f : expf(x - top) * inv_sum * (g - dot);
        }
        Traits::store(dst + e, g);
    }
}

// ---- stable order of slots by group -------------------------------------------------------

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kMaxOrderCluster = 8;

struct GroupRowsParams {
    const int* ids;
    int* offsets;
    int* rows;
    int* positions;
    int slots, groups, slots_per_row;
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
    const int tid = static_cast<int>(threadIdx.x);
    const int warp = tid >> 5, lane = tid & 31;
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));

    for (int i = tid; i < kOrderWarps * bins; i += kOrderThreads) {
        hist[i] = 0;
    }
    __syncthreads();
    const long long first =
        (static_cast<long long>(rank) * kOrderWarps + warp) * static_cast<long long>(p.warp_slots);
    const int begin = static_cast<int>(min(first, static_cast<long long>(p.slots)));
    const int end = static_cast<int>(min(first + p.warp_slots, static_cast<long long>(p.slots)));
    int* mine = hist + warp * bins;
    for (int s = begin + lane; s < end; s += 32) {
        const int id = p.ids[s];
        atomicAdd(mine + (id >= 0 && id < p.groups ? id : p.groups), 1);
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
    for (int s0 = begin; s0 < end; s0 += 32) {
        const int s = s0 + lane;
        int bin = -1;
        if (s < end) {
            const int id = p.ids[s];
            bin = id >= 0 && id < p.groups ? id : p.groups;
        }
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, bin);
        if (bin >= 0) {
            const int pos = start[bin] + mine[bin] + __popc(same & ((1u << lane) - 1u));
            p.positions[s] = pos;
            p.rows[pos] = s / p.slots_per_row;
        }
        __syncwarp();
        if (bin >= 0 && lane == __ffs(same) - 1) {
            mine[bin] += __popc(same);
        }
        __syncwarp();
    }
}

// ---- rows back to their tokens --------------------------------------------------------------

constexpr int kCombineThreads = 256;

struct CombineParams {
    const void* y;
    const int* positions;
    const float* weights;
    void* out;
    int tokens, top_k, n, y_rows;
    int ldy, ldo;
};

// out[t] = sum_j weights[t][j] * y[positions[t][j]], summed in FP32 in the order of j.  One
// thread per 8 columns of one token (kVec) or per column; memory-bound: y is read once.
// A position outside [0, y_rows) adds nothing.
template <typename T, typename OutT, bool kVec>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const CombineParams p) {
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
    float acc[V] = {};
#pragma unroll 8
    for (int j = 0; j < p.top_k; ++j) {
        const int at = __ldg(pos + j);
        const float f = __ldg(w + j);
        if (at < 0 || at >= p.y_rows) {
            continue;
        }
        const T* src = y + static_cast<size_t>(at) * p.ldy;
        if constexpr (kVec) {
            constexpr int U = detail::OutTraits<T>::kVec;
#pragma unroll
            for (int h = 0; h < V / U; ++h) {
                float v[U];
                detail::OutTraits<T>::load_vec(src + h * U, v);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    acc[h * U + i] = fmaf(f, v[i], acc[h * U + i]);
                }
            }
        } else {
            acc[0] = fmaf(f, detail::OutTraits<T>::load(src), acc[0]);
        }
    }
    OutT* dst = static_cast<OutT*>(p.out) + static_cast<size_t>(t) * p.ldo + col;
    if constexpr (kVec) {
        constexpr int U = detail::OutTraits<OutT>::kVec;
#pragma unroll
        for (int h = 0; h < V / U; ++h) {
            detail::OutTraits<OutT>::store_vec(dst + h * U, acc + h * U);
        }
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
};

// One CTA per token: dy[positions[t][j]] = weights[t][j] * dout[t] and
// dweights[t][j] = <dout[t], y[positions[t][j]]> in one pass over y.  Eight choices at a time
// keep their dot products in registers; more choices walk dout again (it is in L1 by then).
template <typename T, typename OutT, bool kVec>
__global__ void __launch_bounds__(kCombineThreads)
moe_combine_backward_kernel(const CombineBackwardParams p) {
    constexpr int V = kVec ? 8 : 1;
    constexpr int J = 8;
    __shared__ float part[kCombineThreads / 32][J];
    const size_t t = blockIdx.x;
    const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
    const OutT* dout = static_cast<const OutT*>(p.dout) + t * p.ldo;
    for (int j0 = 0; j0 < p.top_k; j0 += J) {
        int at[J];
        float w[J], dot[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            at[j] = -1;
            w[j] = dot[j] = 0.0f;
            if (j0 + j < p.top_k) {
                at[j] = __ldg(p.positions + t * p.top_k + j0 + j);
                w[j] = __ldg(p.weights + t * p.top_k + j0 + j);
                if (at[j] >= p.y_rows) {
                    at[j] = -1;
                }
            }
        }
        for (int col = static_cast<int>(threadIdx.x) * V; col < p.n; col += kCombineThreads * V) {
            float g[V];
            if constexpr (kVec) {
                constexpr int U = detail::OutTraits<OutT>::kVec;
#pragma unroll
                for (int h = 0; h < V / U; ++h) {
                    float v[U];
                    detail::OutTraits<OutT>::load_vec(dout + col + h * U, v);
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        g[h * U + i] = v[i];
                    }
                }
            } else {
                g[0] = detail::OutTraits<OutT>::load(dout + col);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (at[j] < 0) {
                    continue;
                }
                const T* src = static_cast<const T*>(p.y) + static_cast<size_t>(at[j]) * p.ldy + col;
                T* dst = static_cast<T*>(p.dy) + static_cast<size_t>(at[j]) * p.lddy + col;
                if constexpr (kVec) {
                    constexpr int U = detail::OutTraits<T>::kVec;
#pragma unroll
                    for (int h = 0; h < V / U; ++h) {
                        float v[U], o[U];
                        detail::OutTraits<T>::load_vec(src + h * U, v);
#pragma unroll
                        for (int i = 0; i < U; ++i) {
                            dot[j] = fmaf(v[i], g[h * U + i], dot[j]);
                            o[i] = w[j] * g[h * U + i];
                        }
                        detail::OutTraits<T>::store_vec(dst + h * U, o);
                    }
                } else {
                    dot[j] = fmaf(detail::OutTraits<T>::load(src), g[0], dot[j]);
                    detail::OutTraits<T>::store(dst, w[j] * g[0]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float s = detail::warp_sum(dot[j]);
            if (lane == 0) {
                part[warp][j] = s;
            }
        }
        __syncthreads();
        if (threadIdx.x < J && j0 + static_cast<int>(threadIdx.x) < p.top_k) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < kCombineThreads / 32; ++v) {
                s += part[v][threadIdx.x];
            }
            p.dweights[t * p.top_k + j0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
}

}  // namespace ckl
