#pragma once
// ckl:: C++ entry points of the products whose weight is chosen per row: routing to experts, the
// experts' products and their gradients, and low-rank adapters beside a shared projection.  No
// counterpart in the reference.  Inline shims over the C ABI (ckl_gemm.h states the contracts):
// packed row-major matrices, device pointers, work enqueued on `stream`; failures throw
// std::runtime_error like the rest of the library.

#include <cstddef>

#include <cuda_runtime.h>

#include "../ckl_gemm.h"
#include "gemm.hpp"

namespace ckl {

inline void group_rows(const int* ids, int slots, int groups, int slots_per_row, int* offsets, int* rows,
                       int* positions, cudaStream_t stream = nullptr) {
    detail::throw_on_error(ckl_group_rows(ids, slots, groups, slots_per_row, offsets, rows, positions, stream),
                           "group_rows");
}

struct RouteOptions {
    ckl_score score = CKL_SCORE_SOFTMAX;
    const float* bias = nullptr;
    int groups = 1, top_groups = 1;
    bool renormalise = false;
    float scale = 1.0f;
};

template <typename T>
inline void moe_route(const T* logits, float* weights, int* experts, int tokens, int n_experts, int top_k,
                      const RouteOptions& o = {}, cudaStream_t stream = nullptr) {
    detail::throw_on_error(
        ckl_moe_route(detail::dtype_of(logits), logits, n_experts, o.bias, weights, experts, tokens, n_experts,
                      top_k, o.score, o.groups, o.top_groups, o.renormalise ? 1 : 0, o.scale, stream),
        "moe_route");
}

template <typename T>
inline void moe_route_backward(const T* logits, const int* experts, const float* dweights, T* dlogits, int tokens,
                               int n_experts, int top_k, const RouteOptions& o = {},
                               cudaStream_t stream = nullptr) {
    detail::throw_on_error(
        ckl_moe_route_backward(detail::dtype_of(logits), logits, n_experts, experts, dweights, dlogits, n_experts,
                               tokens, n_experts, top_k, o.score, o.renormalise ? 1 : 0, o.scale, stream),
        "moe_route_backward");
}

// C[p] = alpha * A[a_rows[p]] * B_g + beta * C[p]; with trans_b B_g is n x k.
template <typename InT, typename OutT>
inline void gemm_grouped(const InT* a, const int* a_rows, int a_count, const InT* b, OutT* c, const int* offsets,
                         int groups, int rows, int n, int k, bool trans_b = false, float alpha = 1.0f,
                         float beta = 0.0f, cudaStream_t stream = nullptr) {
    detail::throw_on_error(
        ckl_gemm_grouped(detail::dtype_of(a), a, a_rows, a_count, b, c, detail::dtype_of(c), offsets, groups, rows,
                         n, k, k, trans_b ? k : n, static_cast<long long>(n) * k, n, trans_b ? 1 : 0, alpha, beta,
                         stream),
        "gemm_grouped");
}

// dW_g = alpha * sum over p in g of A[a_rows[p]]^T G[p] + beta * dW_g, each m x n.
template <typename InT, typename OutT>
inline void gemm_grouped_wgrad(const InT* a, const int* a_rows, int a_count, const InT* g, OutT* dw,
                               const int* offsets, int groups, int rows, int m, int n, float alpha = 1.0f,
                               float beta = 0.0f, cudaStream_t stream = nullptr) {
    detail::throw_on_error(
        ckl_gemm_grouped_wgrad(detail::dtype_of(a), a, a_rows, a_count, g, dw, detail::dtype_of(dw), offsets, groups,
                               rows, m, n, m, n, n, static_cast<long long>(m) * n, alpha, beta, stream),
        "gemm_grouped_wgrad");
}

template <typename T, typename OutT>
inline void moe_combine(const T* y, const int* positions, const float* weights, OutT* out, int tokens, int top_k,
                        int n, int y_rows, cudaStream_t stream = nullptr, const int* kept = nullptr) {
    detail::throw_on_error(ckl_moe_combine_ex(detail::dtype_of(y), y, positions, weights, out, detail::dtype_of(out),
                                              tokens, top_k, n, y_rows, n, n, kept, stream),
                           "moe_combine");
}

template <typename T, typename OutT>
inline void moe_combine_backward(const T* y, const int* positions, const float* weights, const OutT* dout, T* dy,
                                 float* dweights, int tokens, int top_k, int n, int y_rows,
                                 cudaStream_t stream = nullptr, const int* kept = nullptr) {
    detail::throw_on_error(
        ckl_moe_combine_backward_ex(detail::dtype_of(y), y, positions, weights, dout, detail::dtype_of(dout), dy,
                                    dweights, tokens, top_k, n, y_rows, n, n, n, kept, stream),
        "moe_combine_backward");
}

inline std::size_t gemm_lora_workspace_bytes(int m, int rank, bool backward = false) {
    return ckl_gemm_lora_workspace_bytes(m, rank, backward ? 1 : 0);
}

// y[i] = x[i] W + scales[g] * (x[i] A_g) B_g + beta * y[i], g the adapter of row i (or none).
template <typename InT, typename OutT>
inline void gemm_lora(const InT* x, const InT* w, const InT* lora_a, const InT* lora_b, const float* scales,
                      OutT* y, const int* offsets, const int* rows, int adapters, int m, int n, int k, int rank,
                      void* workspace, std::size_t workspace_bytes, float beta = 0.0f,
                      cudaStream_t stream = nullptr) {
    detail::throw_on_error(
        ckl_gemm_lora(detail::dtype_of(x), x, w, lora_a, lora_b, scales, y, detail::dtype_of(y), offsets, rows,
                      adapters, m, n, k, rank, k, n, rank, static_cast<long long>(k) * rank, n,
                      static_cast<long long>(rank) * n, n, beta, workspace, workspace_bytes, stream),
        "gemm_lora");
}

// dx, da, db (any may be null) of gemm_lora with a frozen W; beta applies to da and db.
template <typename InT, typename DxT, typename GradT>
inline void gemm_lora_backward(const InT* dy, const InT* x, const InT* w, const InT* lora_a, const InT* lora_b,
                               const float* scales, DxT* dx, GradT* da, GradT* db, const int* offsets,
                               const int* rows, int adapters, int m, int n, int k, int rank, void* workspace,
                               std::size_t workspace_bytes, float beta = 0.0f, cudaStream_t stream = nullptr) {
    const long long a_size = static_cast<long long>(k) * rank, b_size = static_cast<long long>(rank) * n;
    detail::throw_on_error(
        ckl_gemm_lora_backward(detail::dtype_of(dy), dy, x, w, lora_a, lora_b, scales, dx, detail::dtype_of(dx), da,
                               db, detail::dtype_of(da), offsets, rows, adapters, m, n, k, rank, n, k, n, rank,
                               a_size, n, b_size, k, rank, a_size, n, b_size, beta, workspace, workspace_bytes,
                               stream),
        "gemm_lora_backward");
}

}  // namespace ckl
