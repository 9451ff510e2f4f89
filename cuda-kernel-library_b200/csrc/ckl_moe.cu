// C entry points of the routing operators: argument checks and launches of moe_route.cuh.

#include <algorithm>
#include <mutex>

#include "ckl_gemm.h"
#include "ckl_internal.h"
#include "moe_route.cuh"

namespace {

using namespace ckl;

#define MOE_TRY_CUDA(expr)                                                                  \
    do {                                                                                    \
        const cudaError_t err__ = (expr);                                                   \
        if (err__ != cudaSuccess) {                                                         \
            return set_error(CKL_ERR_CUDA, "%s failed: %s (%s)", #expr,                     \
                             cudaGetErrorName(err__), cudaGetErrorString(err__));           \
        }                                                                                   \
    } while (0)

bool known_dtype(int d) { return d == CKL_F32 || d == CKL_F16 || d == CKL_BF16; }
int size_of(int dtype) { return dtype == CKL_F32 ? 4 : 2; }
bool aligned16(const void* p, long long pitch, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (pitch * size_of(dtype)) % 16 == 0;
}
bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// Kernels that may need more than 48 KB of dynamic shared memory are told so once per device.
template <auto kKernel>
int allow_smem(int bytes) {
    static std::mutex mu;
    static int granted[64] = {};
    int dev = 0;
    MOE_TRY_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 0 || dev >= 64 || granted[dev] < bytes) {
        MOE_TRY_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) {
            granted[dev] = bytes;
        }
    }
    return CKL_OK;
}

template <typename T, int NV, bool kWide>
int launch_route(const RouteParams& p, cudaStream_t stream) {
    const int smem = kRouteWarps * ((NV * 32 + kMaxRouteGroups) * 8 + NV * 32 * 4);
    if (smem > 48 * 1024) {
        if (const int rc = allow_smem<moe_route_kernel<T, NV, kWide>>(smem); rc != CKL_OK) {
            return rc;
        }
    }
    const unsigned grid = static_cast<unsigned>((p.tokens + kRouteWarps - 1) / kRouteWarps);
    MOE_TRY_CUDA(launch_dependent(moe_route_kernel<T, NV, kWide>, dim3(grid), 32 * kRouteWarps,
                                  static_cast<size_t>(smem), 1, stream, p));
    return CKL_OK;
}

template <typename T, bool kWide>
int launch_route_size(const RouteParams& p, cudaStream_t stream) {
    const int nv = (p.n_experts + 31) / 32;
    if (nv <= 1) return launch_route<T, 1, kWide>(p, stream);
    if (nv <= 2) return launch_route<T, 2, kWide>(p, stream);
    if (nv <= 4) return launch_route<T, 4, kWide>(p, stream);
    if (nv <= 8) return launch_route<T, 8, kWide>(p, stream);
    if (nv <= 16) return launch_route<T, 16, kWide>(p, stream);
    return launch_route<T, 32, kWide>(p, stream);
}

template <typename T>
int launch_route_type(const RouteParams& p, cudaStream_t stream) {
    return p.bias != nullptr || p.groups > 1 ? launch_route_size<T, true>(p, stream)
                                             : launch_route_size<T, false>(p, stream);
}

template <typename T, int NV>
int launch_route_backward(const RouteBackwardParams& p, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>((p.tokens + kRouteWarps - 1) / kRouteWarps);
    MOE_TRY_CUDA(launch_dependent(moe_route_backward_kernel<T, NV>, dim3(grid), 32 * kRouteWarps, 0, 1, stream, p));
    return CKL_OK;
}

template <typename T>
int launch_route_backward_size(const RouteBackwardParams& p, cudaStream_t stream) {
    const int nv = (p.n_experts + 31) / 32;
    if (nv <= 1) return launch_route_backward<T, 1>(p, stream);
    if (nv <= 2) return launch_route_backward<T, 2>(p, stream);
    if (nv <= 4) return launch_route_backward<T, 4>(p, stream);
    if (nv <= 8) return launch_route_backward<T, 8>(p, stream);
    if (nv <= 16) return launch_route_backward<T, 16>(p, stream);
    return launch_route_backward<T, 32>(p, stream);
}

int check_route(const char* what, int dtype, const void* logits, int ldl, int tokens, int n_experts,
                int top_k, int score) {
    if (!known_dtype(dtype)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: bad dtype %d", what, dtype);
    }
    if (n_experts < 1 || top_k < 1 || top_k > n_experts) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: %d experts, top_k %d", what, n_experts, top_k);
    }
    if (n_experts > kMaxExperts || top_k > kMaxTopK || tokens > kMaxExtent) {
        return set_error(CKL_ERR_TOO_LARGE, "%s: %d experts (at most %d), top_k %d (at most %d), %d tokens", what,
                         n_experts, kMaxExperts, top_k, kMaxTopK, tokens);
    }
    if (score != CKL_SCORE_SOFTMAX && score != CKL_SCORE_SIGMOID) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: bad score %d", what, score);
    }
    if (logits == nullptr || ldl < n_experts || misaligned(logits, size_of(dtype))) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: logits %p with leading dimension %d for %d experts",
                         what, logits, ldl, n_experts);
    }
    return CKL_OK;
}

template <typename T, typename OutT>
int launch_combine(const CombineParams& p, bool vec, cudaStream_t stream) {
    const long long units = static_cast<long long>(p.tokens) * (vec ? p.n / 8 : p.n);
    const long long grid = (units + kCombineThreads - 1) / kCombineThreads;
    if (grid > 0x7fffffffll) {
        return set_error(CKL_ERR_TOO_LARGE, "moe_combine: %d tokens of %d columns", p.tokens, p.n);
    }
    MOE_TRY_CUDA(launch_dependent(vec ? moe_combine_kernel<T, OutT, true> : moe_combine_kernel<T, OutT, false>,
                                  dim3(static_cast<unsigned>(grid)), kCombineThreads, 0, 1, stream, p));
    return CKL_OK;
}

template <typename T>
int launch_combine_out(int out_dtype, const CombineParams& p, bool vec, cudaStream_t stream) {
    switch (out_dtype) {
        case CKL_F16: return launch_combine<T, __half>(p, vec, stream);
        case CKL_BF16: return launch_combine<T, __nv_bfloat16>(p, vec, stream);
        default: return launch_combine<T, float>(p, vec, stream);
    }
}

template <typename T, typename OutT>
int launch_combine_backward(const CombineBackwardParams& p, bool vec, cudaStream_t stream) {
    const long long slots = static_cast<long long>(p.tokens) * p.top_k;
    const long long grid = (slots + kCombineThreads / 32 - 1) / (kCombineThreads / 32);
    if (grid > 0x7fffffffll) {
        return set_error(CKL_ERR_TOO_LARGE, "moe_combine_backward: %d tokens, top_k %d", p.tokens, p.top_k);
    }
    MOE_TRY_CUDA(launch_dependent(
        vec ? moe_combine_backward_kernel<T, OutT, true> : moe_combine_backward_kernel<T, OutT, false>,
        dim3(static_cast<unsigned>(grid)), kCombineThreads, 0, 1, stream, p));
    return CKL_OK;
}

template <typename T>
int launch_combine_backward_out(int out_dtype, const CombineBackwardParams& p, bool vec,
                                cudaStream_t stream) {
    switch (out_dtype) {
        case CKL_F16: return launch_combine_backward<T, __half>(p, vec, stream);
        case CKL_BF16: return launch_combine_backward<T, __nv_bfloat16>(p, vec, stream);
        default: return launch_combine_backward<T, float>(p, vec, stream);
    }
}

int check_combine(const char* what, int y_dtype, const void* y, const int* positions,
                  const float* weights, int out_dtype, const void* out, int top_k, int n, int y_rows,
                  int ldy, int ldo, const int* kept) {
    if (!known_dtype(y_dtype) || !known_dtype(out_dtype)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: bad dtype %d or %d", what, y_dtype, out_dtype);
    }
    if (n > kMaxExtent) {
        return set_error(CKL_ERR_TOO_LARGE, "%s: %d columns", what, n);
    }
    if (top_k < 1 || y_rows < 0 || ldy < n || ldo < n) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: top_k %d, y_rows %d, n %d, ldy %d, ldo %d", what, top_k,
                         y_rows, n, ldy, ldo);
    }
    if ((y == nullptr && y_rows > 0) || positions == nullptr || weights == nullptr || out == nullptr) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: null pointer", what);
    }
    if (misaligned(y, size_of(y_dtype)) || misaligned(out, size_of(out_dtype)) ||
        misaligned(positions, 4) || misaligned(weights, 4) || misaligned(kept, 4)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element", what);
    }
    return CKL_OK;
}

}  // namespace

extern "C" {

int ckl_moe_route(int logit_dtype, const void* logits, int ldl, const float* bias, float* weights,
                  int* experts, int tokens, int n_experts, int top_k, int score, int groups,
                  int top_groups, int renormalise, float scale, ckl_stream_t stream) {
    if (tokens <= 0) {
        return CKL_OK;
    }
    if (const int rc = check_route("moe_route", logit_dtype, logits, ldl, tokens, n_experts, top_k, score);
        rc != CKL_OK) {
        return rc;
    }
    if (weights == nullptr || experts == nullptr || misaligned(weights, 4) || misaligned(experts, 4) ||
        misaligned(bias, 4)) {
        return set_error(CKL_ERR_INVALID_ARG, "moe_route: null or misaligned weights, experts or bias");
    }
    if (groups < 1 || n_experts % groups != 0 || top_groups < 1 || top_groups > groups) {
        return set_error(CKL_ERR_INVALID_ARG, "moe_route: %d experts in %d groups of which %d are kept",
                         n_experts, groups, top_groups);
    }
    if (groups > kMaxRouteGroups) {
        return set_error(CKL_ERR_TOO_LARGE, "moe_route: %d groups (at most %d)", groups, kMaxRouteGroups);
    }
    DeviceView view;
    if (const int rc = device_view(&view); rc != CKL_OK) {
        return rc;
    }
    RouteParams p = {};
    p.logits = logits;
    p.bias = bias;
    p.weights = weights;
    p.experts = experts;
    p.ldl = ldl;
    p.tokens = tokens;
    p.n_experts = n_experts;
    p.top_k = top_k;
    // Keeping every group is keeping none apart.
    p.groups = top_groups == groups ? 1 : groups;
    p.top_groups = top_groups == groups ? 1 : top_groups;
    p.group_size = n_experts / p.groups;
    p.inv_group_size = 1.0f / static_cast<float>(p.group_size);
    p.sigmoid = score == CKL_SCORE_SIGMOID ? 1 : 0;
    p.renormalise = renormalise != 0 ? 1 : 0;
    p.scale = scale;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (logit_dtype) {
        case CKL_F16: return launch_route_type<__half>(p, s);
        case CKL_BF16: return launch_route_type<__nv_bfloat16>(p, s);
        default: return launch_route_type<float>(p, s);
    }
}

int ckl_moe_route_backward(int logit_dtype, const void* logits, int ldl, const int* experts,
                           const float* dweights, void* dlogits, int ldd, int tokens, int n_experts,
                           int top_k, int score, int renormalise, float scale, ckl_stream_t stream) {
    if (tokens <= 0) {
        return CKL_OK;
    }
    if (const int rc =
            check_route("moe_route_backward", logit_dtype, logits, ldl, tokens, n_experts, top_k, score);
        rc != CKL_OK) {
        return rc;
    }
    if (experts == nullptr || dweights == nullptr || dlogits == nullptr || ldd < n_experts ||
        misaligned(experts, 4) || misaligned(dweights, 4) || misaligned(dlogits, size_of(logit_dtype))) {
        return set_error(CKL_ERR_INVALID_ARG,
                         "moe_route_backward: null or misaligned pointer, or ldd %d for %d experts", ldd,
                         n_experts);
    }
    DeviceView view;
    if (const int rc = device_view(&view); rc != CKL_OK) {
        return rc;
    }
    RouteBackwardParams p = {};
    p.logits = logits;
    p.experts = experts;
    p.dweights = dweights;
    p.dlogits = dlogits;
    p.ldl = ldl;
    p.ldd = ldd;
    p.tokens = tokens;
    p.n_experts = n_experts;
    p.top_k = top_k;
    p.sigmoid = score == CKL_SCORE_SIGMOID ? 1 : 0;
    p.renormalise = renormalise != 0 ? 1 : 0;
    p.scale = scale;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (logit_dtype) {
        case CKL_F16: return launch_route_backward_size<__half>(p, s);
        case CKL_BF16: return launch_route_backward_size<__nv_bfloat16>(p, s);
        default: return launch_route_backward_size<float>(p, s);
    }
}

int ckl_group_rows(const int* ids, int slots, int groups, int slots_per_row, int* offsets, int* rows,
                   int* positions, ckl_stream_t stream) {
    if (groups < 1 || slots_per_row < 1 || slots < 0) {
        return set_error(CKL_ERR_INVALID_ARG, "group_rows: %d slots, %d groups, %d slots per row", slots,
                         groups, slots_per_row);
    }
    if (groups > kMaxExperts || slots > kMaxExtent) {
        return set_error(CKL_ERR_TOO_LARGE, "group_rows: %d groups (at most %d), %d slots", groups, kMaxExperts,
                         slots);
    }
    if (offsets == nullptr || (slots > 0 && (ids == nullptr || rows == nullptr || positions == nullptr))) {
        return set_error(CKL_ERR_INVALID_ARG, "group_rows: null pointer");
    }
    if (misaligned(ids, 4) || misaligned(offsets, 4) || misaligned(rows, 4) || misaligned(positions, 4)) {
        return set_error(CKL_ERR_INVALID_ARG, "group_rows: a pointer is not aligned to its element");
    }
    DeviceView view;
    if (const int rc = device_view(&view); rc != CKL_OK) {
        return rc;
    }
    // One CTA walks 1024 slots per step of its warps; from 8192 slots on more CTAs share them.
    int cluster = 1;
    while (cluster < kMaxOrderCluster && slots > cluster * 8 * kOrderThreads) {
        cluster *= 2;
    }
    const long long warps = static_cast<long long>(cluster) * kOrderWarps;
    GroupRowsParams p = {};
    p.ids = ids;
    p.offsets = offsets;
    p.rows = rows;
    p.positions = positions;
    p.slots = slots;
    p.groups = groups;
    p.inv_row = detail::reciprocal_of(slots_per_row);
    p.warp_slots = static_cast<int>(((slots + warps - 1) / warps + 31) / 32 * 32);
    const auto smem_of = [](int bins, int staged_slots) {
        return (kOrderWarps * bins + 2 * bins + kOrderWarps + (bins + 1) / 2 * 2 + 2) * 4 + staged_slots * 8;
    };
    const int cta_slots = p.warp_slots * kOrderWarps;
    p.staged = slots > kOrderThreads && cta_slots <= kOrderStaged ? 1 : 0;
    const int smem = smem_of(groups + 1, p.staged ? cta_slots : 0);
    if (const int rc = allow_smem<group_rows_kernel>(smem_of(kMaxExperts + 1, kOrderStaged)); rc != CKL_OK) {
        return rc;
    }
    MOE_TRY_CUDA(launch_dependent(group_rows_kernel, dim3(static_cast<unsigned>(cluster)), kOrderThreads,
                                  static_cast<size_t>(smem), cluster, static_cast<cudaStream_t>(stream), p));
    return CKL_OK;
}

int ckl_moe_combine_ex(int y_dtype, const void* y, const int* positions, const float* weights, void* out,
                       int out_dtype, int tokens, int top_k, int n, int y_rows, int ldy, int ldo,
                       const int* kept, ckl_stream_t stream) {
    if (tokens <= 0 || n <= 0) {
        return CKL_OK;
    }
    if (const int rc = check_combine("moe_combine", y_dtype, y, positions, weights, out_dtype, out, top_k, n,
                                     y_rows, ldy, ldo, kept);
        rc != CKL_OK) {
        return rc;
    }
    DeviceView view;
    if (const int rc = device_view(&view); rc != CKL_OK) {
        return rc;
    }
    const CombineParams p = {y, positions, weights, out, tokens, top_k, n, y_rows, ldy, ldo, kept};
    const bool vec = n % 8 == 0 && aligned16(y, ldy, y_dtype) && aligned16(out, ldo, out_dtype);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (y_dtype) {
        case CKL_F16: return launch_combine_out<__half>(out_dtype, p, vec, s);
        case CKL_BF16: return launch_combine_out<__nv_bfloat16>(out_dtype, p, vec, s);
        default: return launch_combine_out<float>(out_dtype, p, vec, s);
    }
}

int ckl_moe_combine_backward_ex(int y_dtype, const void* y, const int* positions, const float* weights,
                                const void* dout, int dout_dtype, void* dy, float* dweights, int tokens,
                                int top_k, int n, int y_rows, int ldy, int ldo, int lddy,
                                const int* kept, ckl_stream_t stream) {
    if (tokens <= 0 || n <= 0) {
        return CKL_OK;
    }
    if (const int rc = check_combine("moe_combine_backward", y_dtype, y, positions, weights, dout_dtype, dout,
                                     top_k, n, y_rows, ldy, ldo, kept);
        rc != CKL_OK) {
        return rc;
    }
    if ((dy == nullptr && y_rows > 0) || dweights == nullptr || lddy < n ||
        misaligned(dy, size_of(y_dtype)) || misaligned(dweights, 4)) {
        return set_error(CKL_ERR_INVALID_ARG,
                         "moe_combine_backward: null or misaligned dy or dweights, or lddy %d for n %d", lddy,
                         n);
    }
    DeviceView view;
    if (const int rc = device_view(&view); rc != CKL_OK) {
        return rc;
    }
    const CombineBackwardParams p = {y, positions, weights, dout, dy, dweights, tokens, top_k, n, y_rows,
                                     ldy, ldo, lddy, kept};
    const bool vec = n % 8 == 0 && aligned16(y, ldy, y_dtype) && aligned16(dout, ldo, dout_dtype) &&
                     aligned16(dy, lddy, y_dtype);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (y_dtype) {
        case CKL_F16: return launch_combine_backward_out<__half>(dout_dtype, p, vec, s);
        case CKL_BF16: return launch_combine_backward_out<__nv_bfloat16>(dout_dtype, p, vec, s);
        default: return launch_combine_backward_out<float>(dout_dtype, p, vec, s);
    }
}

int ckl_moe_combine(int y_dtype, const void* y, const int* positions, const float* weights, void* out,
                    int out_dtype, int tokens, int top_k, int n, int y_rows, int ldy, int ldo,
                    ckl_stream_t stream) {
    return ckl_moe_combine_ex(y_dtype, y, positions, weights, out, out_dtype, tokens, top_k, n, y_rows, ldy, ldo,
                              nullptr, stream);
}

int ckl_moe_combine_backward(int y_dtype, const void* y, const int* positions, const float* weights,
                             const void* dout, int dout_dtype, void* dy, float* dweights, int tokens,
                             int top_k, int n, int y_rows, int ldy, int ldo, int lddy, ckl_stream_t stream) {
    return ckl_moe_combine_backward_ex(y_dtype, y, positions, weights, dout, dout_dtype, dy, dweights, tokens, top_k,
                                       n, y_rows, ldy, ldo, lddy, nullptr, stream);
}

}  // extern "C"
