// C entry points of the products whose weight is chosen per row (gemm_grouped.cuh): experts'
// products with their gradients, and low-rank adapters beside a shared projection.

#include <algorithm>
#include <cstring>
#include <mutex>

#include "ckl_gemm.h"
#include "ckl_internal.h"
#include "gemm_grouped.cuh"
#include "gemm_grouped_pair.cuh"

namespace {

using namespace ckl;

#define GRP_TRY_CUDA(expr)                                                                  \
    do {                                                                                    \
        const cudaError_t err__ = (expr);                                                   \
        if (err__ != cudaSuccess) {                                                         \
            return set_error(CKL_ERR_CUDA, "%s failed: %s (%s)", #expr,                     \
                             cudaGetErrorName(err__), cudaGetErrorString(err__));           \
        }                                                                                   \
    } while (0)
#define GRP_TRY(expr)                                       \
    do {                                                    \
        if (const int rc__ = (expr); rc__ != CKL_OK) {      \
            return rc__;                                    \
        }                                                   \
    } while (0)

int size_of(int dtype) { return dtype == CKL_F32 ? 4 : 2; }
bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// An operand that TMA reads: base on 16 bytes, pitch and stack distance multiples of 8 elements.
int check_operand(const char* what, const char* name, const void* ptr, int pitch, int columns,
                  long long stack) {
    if (ptr == nullptr || pitch < columns || pitch < 1 || stack < 0) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: %s is %p, leading dimension %d for %d columns, stride %lld",
                         what, name, ptr, pitch, columns, stack);
    }
    if (misaligned(ptr, 16) || pitch % 8 != 0 || stack % 8 != 0) {
        return set_error(CKL_ERR_UNSUPPORTED,
                         "%s: %s must be 16-byte aligned with a leading dimension (%d) and a stride (%lld) "
                         "that are multiples of 8 elements",
                         what, name, pitch, stack);
    }
    return CKL_OK;
}

int check_types(const char* what, int ab_dtype, int c_dtype) {
    if ((ab_dtype != CKL_F16 && ab_dtype != CKL_BF16) ||
        (c_dtype != CKL_F32 && c_dtype != CKL_F16 && c_dtype != CKL_BF16)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: bad dtype %d or %d", what, ab_dtype, c_dtype);
    }
    return CKL_OK;
}

int check_groups(const char* what, const int* offsets, int groups, int rows, int cols, int depth) {
    if (groups < 1 || rows < 0 || offsets == nullptr || misaligned(offsets, 4)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: offsets %p of %d groups, %d rows", what,
                         static_cast<const void*>(offsets), groups, rows);
    }
    if (groups > kMaxGemmGroups) {
        return set_error(CKL_ERR_TOO_LARGE, "%s: %d groups (at most %d)", what, groups, kMaxGemmGroups);
    }
    if (std::max(rows, std::max(cols, depth)) > kMaxExtent) {
        return set_error(CKL_ERR_TOO_LARGE, "%s: extents %d, %d, %d (at most %d)", what, rows, cols, depth,
                         kMaxExtent);
    }
    return CKL_OK;
}

// A kernel that needs `bytes` of dynamic shared memory is told so once per device.
template <auto kKernel>
int allow_smem(int device, size_t bytes) {
    static std::mutex mu;
    static bool ready[64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (device < 0 || device >= 64 || !ready[device]) {
        GRP_TRY_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          static_cast<int>(bytes)));
        if (device >= 0 && device < 64) {
            ready[device] = true;
        }
    }
    return CKL_OK;
}

template <auto kKernel, typename Arg>
int launch_kernel(int device, int threads, size_t smem, int cluster, const Arg& arg, dim3 grid,
                  cudaStream_t stream) {
    GRP_TRY(allow_smem<kKernel>(device, smem));
    GRP_TRY_CUDA(launch_dependent(kKernel, grid, threads, smem, cluster, stream, arg));
    return CKL_OK;
}

// One product in terms of its operands.
struct Product {
    int ab_dtype, c_dtype;  // c_dtype < 0: two-part C in the operand type
    GroupedParams p;
    const void *a, *b, *t, *e;
    int lda, ldb, ldt, lde;
    int a_cols, b_cols, b_outer;  // extents of A's rows, of B's rows, and B's row count (kFormRows)
    int b_depth;
    long long b_stack, e_stack;
    int e_cols, e_outer;
    // the plan
    bool pair, whole;
    long long tiles, blocks;
};

long long row_tiles(const Product& q, int height) {
    // An upper bound: the groups' sizes are known on the device only.
    const GroupedParams& p = q.p;
    return p.form == kFormWgrad ? static_cast<long long>(p.groups) * ((p.m + height - 1) / height)
           : q.whole            ? (p.rows + height - 1) / height
                                : p.rows / height + std::min(p.groups, p.rows);
}
long long single_tiles(const Product& q, int bn) { return row_tiles(q, 128) * ((q.p.n + bn - 1) / bn); }

// Chooses the kernel and its tiles.
void plan(Product& q, const DeviceView& view) {
    GroupedParams& p = q.p;
    const bool wgrad = p.form == kFormWgrad;
    p.status = view.status;
    p.fmt = q.ab_dtype == CKL_BF16 ? 1u : 0u;
    q.whole = !wgrad && (p.offsets == nullptr || q.e != nullptr);
    // CTA pairs on 256 x 256 tiles where there are enough of them; weight gradients with a two-word operand
    // or a gathered G have only a few columns or rows of output and stay with the single-CTA kernel.
    const long long pair_tiles = row_tiles(q, 256) * ((p.n + 255) / 256);
    q.pair = q.c_dtype >= 0 && p.layered == kLayeredNone && p.b_rows == nullptr && p.n > 128 &&
             (!wgrad || p.m > 128) && pair_tiles * 2 > view.max_pairs;
    // Tile width of the single-CTA kernel: with enough tiles for every SM the wider one, which
    // reads A half as often, unless its last wave leaves more of the machine idle than the narrow
    // one's extra loads cost (a tenth).
    const auto cost_of = [&](int bn) {  // waves x columns
        return static_cast<double>((single_tiles(q, bn) + view.sm_count - 1) / view.sm_count) * bn;
    };
    p.bn = p.n > 128 && cost_of(256) <= 1.1 * cost_of(128) ? 256 : p.n > 64 ? 128 : 64;
    // Blocks of 64 reduced elements behind one tile, as far as the host can tell.
    q.blocks = wgrad ? static_cast<long long>(p.rows / p.groups + 63) / 64 * p.parts
                     : (p.k + 63) / 64;
    p.split = 1;
    q.tiles = q.pair ? pair_tiles : single_tiles(q, p.bn);
}

// Fewer tiles than half of the SMs: a cluster divides the blocks of each, at least four per CTA.
bool may_split(const Product& q, const DeviceView& view) {
    return !q.pair && single_tiles(q, std::min(q.p.bn, 128)) * 2 <= view.sm_count;
}

// Clusters of `size` CTAs that are resident at once.  A cluster lives inside one GPC, so sizes that do
// not divide a GPC's SMs well leave some unused (24 clusters of 6 ran as two waves: 17.5 us, 24 of
// 4 in one: 10.7).
int resident_clusters(int device, int size) {
    static std::mutex mu;
    static int known[64][kMaxSplit + 1] = {};
    if (device < 0 || device >= 64) {
        return 0;
    }
    std::lock_guard<std::mutex> lock(mu);
    int& count = known[device][size];
    if (count == 0) {
        using Cfg = GroupedConfig<true>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(size));
        cfg.blockDim = dim3(Cfg::kThreads);
        cfg.dynamicSmemBytes = Cfg::kSmemBytes;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned>(size);
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (allow_smem<grouped_gemm_kernel<float, true, false>>(device, Cfg::kSmemBytes) != CKL_OK ||
            cudaOccupancyMaxActiveClusters(&count, grouped_gemm_kernel<float, true, false>, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            count = 0;
        }
        count = std::max(count, 1);  // (no answer: this size is never chosen)
    }
    return count;
}
int choose_split(long long tiles, long long blocks, const DeviceView& view) {
    for (int size = static_cast<int>(std::min<long long>(kMaxSplit, blocks / 4)); size > 1; --size) {
        if (resident_clusters(view.device, size) >= tiles) {
            return size;
        }
    }
    return 1;
}

// Descriptors and remaining parameters of a planned product.
int describe(Product& q, GroupedProblem* out) {
    GroupedParams& p = q.p;
    const bool wgrad = p.form == kFormWgrad;
    if (q.tiles * std::max(p.split, 2) > 0x7fffffffll) {
        return set_error(CKL_ERR_TOO_LARGE, "%lld output tiles", q.tiles);
    }
    // Few rows to a tile: the loaders fetch those alone, where a boxed copy would fetch 128.
    const bool layers = q.ab_dtype == CKL_F16;  // the loaders read a two-word operand (BF16: columns like others)
    p.load_a = p.a_rows != nullptr || (layers && p.layered == kLayeredA) ||
               (!wgrad && !q.pair && p.k > 0 && !q.whole && p.rows <= 32ll * std::min(p.groups, p.rows));
    std::memset(out, 0, sizeof *out);
    // Gathered operands are read by the loader warps, all others through these descriptors.
    if (p.load_a == 0) {
        GRP_TRY(encode_operand(&out->a_box, q.ab_dtype, q.a, q.a_cols, p.a_count, q.lda, 0, 0, 64,
                               wgrad || q.pair ? 64 : 128));
    }
    if (!wgrad || (p.b_rows == nullptr && !(layers && p.layered == kLayeredB))) {
        GRP_TRY(encode_operand(&out->b_box, q.ab_dtype, q.b, q.b_cols, wgrad ? p.b_count : q.b_outer, q.ldb,
                               static_cast<uint64_t>(q.b_depth), static_cast<uint64_t>(q.b_stack), 64, 64));
    }
    if (p.ext_mode == kExtBlocks) {
        GRP_TRY(encode_operand(&out->e_box, q.ab_dtype, q.e, q.e_cols, q.e_outer, q.lde, p.groups,
                               static_cast<uint64_t>(q.e_stack), 64, 64));
    }
    p.a = q.a;
    p.b = q.b;
    p.t = q.t;
    p.e = q.e;
    p.lda = q.lda;
    p.ldb = q.ldb;
    p.ldt = q.ldt;
    p.lde = q.lde;
    p.e_stride = q.e_stack;
    unsigned long long limit_ns = 0;
    const int fault = take_wait_fault(&limit_ns);
    p.wait_limit_ns = limit_ns;
    p.overstate_first_stage = fault == 1 ? 1 : 0;
    if (q.c_dtype >= 0) {
        const int bytes = size_of(q.c_dtype);
        p.c_vec = !misaligned(p.c, 16) && (static_cast<long long>(p.ldc) * bytes) % 16 == 0 &&
                  (p.c_stride * bytes) % 16 == 0;
        // A TMA store writes whole 16-byte units: columns that end inside one would take what lies
        // behind them along (measured: up to 7 columns of zeros in a wider matrix).
        p.c_tma = p.c_vec && (static_cast<long long>(p.n) * bytes) % 16 == 0 && p.beta == 0.0f &&
                  p.c_rows == nullptr && p.split == 1;
        if (p.c_tma) {
            GRP_TRY(encode_operand(&out->c, q.c_dtype, p.c, p.n, wgrad ? p.m : p.rows, p.ldc, wgrad ? p.groups : 1,
                                   wgrad ? p.c_stride : static_cast<long long>(p.ldc) * p.rows,
                                   static_cast<uint32_t>(q.pair ? 32 : 64 / bytes), 32));
        }
    }
    out->p = p;
    return CKL_OK;
}

template <typename OutT, bool kAdapters>
int launch_single(const GroupedProblems& problems, int count, int tiles, const DeviceView& view,
                  cudaStream_t stream) {
    const int split = problems.at[0].p.split;
    if (split > 1) {
        return launch_kernel<grouped_gemm_kernel<OutT, true, kAdapters>>(
            view.device, GroupedConfig<true>::kThreads, GroupedConfig<true>::kSmemBytes, split, problems,
            dim3(static_cast<unsigned>(tiles * split), static_cast<unsigned>(count)), stream);
    }
    return launch_kernel<grouped_gemm_kernel<OutT, false, kAdapters>>(
        view.device, GroupedConfig<false>::kThreads, GroupedConfig<false>::kSmemBytes, 1, problems,
        dim3(static_cast<unsigned>(std::min(view.sm_count, tiles)), static_cast<unsigned>(count)), stream);
}

int launch_single(const Product& q, const GroupedProblems& problems, int count, long long tiles,
                  const DeviceView& view, cudaStream_t stream) {
    const int n = static_cast<int>(tiles);
    if (q.c_dtype < 0) {
        return q.ab_dtype == CKL_BF16 ? launch_single<TwoPart<__nv_bfloat16>, false>(problems, count, n, view, stream)
                                      : launch_single<TwoPart<__half>, false>(problems, count, n, view, stream);
    }
    if (q.e != nullptr || q.p.layered != kLayeredNone) {
        switch (q.c_dtype) {
            case CKL_F16: return launch_single<__half, true>(problems, count, n, view, stream);
            case CKL_BF16: return launch_single<__nv_bfloat16, true>(problems, count, n, view, stream);
            default: return launch_single<float, true>(problems, count, n, view, stream);
        }
    }
    switch (q.c_dtype) {
        case CKL_F16: return launch_single<__half, false>(problems, count, n, view, stream);
        case CKL_BF16: return launch_single<__nv_bfloat16, false>(problems, count, n, view, stream);
        default: return launch_single<float, false>(problems, count, n, view, stream);
    }
}

template <typename OutT>
int launch_pair(const GroupedProblem& problem, long long tiles, const DeviceView& view, cudaStream_t stream) {
    const bool ext = problem.p.ext_mode != kExtNone;
    return (ext ? launch_kernel<grouped_pair_kernel<OutT, true>, GroupedProblem>
                : launch_kernel<grouped_pair_kernel<OutT, false>, GroupedProblem>)(
        view.device, GroupedPairConfig::kThreads, GroupedPairConfig::kSmemBytes, 2, problem,
        dim3(static_cast<unsigned>(2 * std::min<long long>(view.max_pairs, tiles))), stream);
}

// Finds the adapters that are not finite, see ExtMode.
int check_adapters(const Product& q, cudaStream_t stream) {
    ExtCheckParams c = {};
    c.offsets = q.p.offsets;
    c.e = static_cast<const unsigned short*>(q.e);
    c.flags = reinterpret_cast<unsigned char*>(const_cast<uint32_t*>(q.p.ext_flags));
    c.stride = q.e_stack;
    c.adapters = q.p.groups;
    c.rows = q.e_outer;
    c.cols = q.e_cols;
    c.ld = q.lde;
    c.exponent = q.ab_dtype == CKL_BF16 ? 0x7f80u : 0x7c00u;
    GRP_TRY_CUDA(launch_dependent(ext_check_kernel, dim3(static_cast<unsigned>(c.adapters), kExtChecks),
                                  kExtCheckThreads, 0, 1, stream, c));
    return CKL_OK;
}

int run(Product& q, cudaStream_t stream) {
    DeviceView view;
    GRP_TRY(device_view(&view));
    plan(q, view);
    if (may_split(q, view)) {
        q.p.bn = std::min(q.p.bn, 128);
        q.tiles = single_tiles(q, q.p.bn);
        q.p.split = choose_split(q.tiles, q.blocks, view);
    }
    if (q.tiles == 0) {
        return CKL_OK;
    }
    if (q.e != nullptr) {
        // Adapters row by row cost about 0.6 ps per row, rank and column (500 rows, 8 adapters, rank
        // 64, n 2048: 50 us, 40 with blocks and their check); up to 5 us of that a split launch saves their blocks.
        const long long products = static_cast<long long>(q.p.rows) * q.p.ext_rank * q.p.n;
        q.p.ext_mode = q.p.split > 1 && products <= (1ll << 23) ? kExtAdd : kExtBlocks;
        if (q.p.ext_mode == kExtBlocks) {
            GRP_TRY(check_adapters(q, stream));
        }
    }
    GroupedProblems problems;
    GRP_TRY(describe(q, &problems.at[0]));
    if (!q.pair) {
        return launch_single(q, problems, 1, q.tiles, view, stream);
    }
    switch (q.c_dtype) {
        case CKL_F16: return launch_pair<__half>(problems.at[0], q.tiles, view, stream);
        case CKL_BF16: return launch_pair<__nv_bfloat16>(problems.at[0], q.tiles, view, stream);
        default: return launch_pair<float>(problems.at[0], q.tiles, view, stream);
    }
}

// Two products of the same output type that do not depend on each other: in one launch where both
// are small, which spends a launch's fixed 5 us once and fills the SMs better.
int run_two(Product& q, Product& r, cudaStream_t stream) {
    DeviceView view;
    GRP_TRY(device_view(&view));
    plan(q, view);
    plan(r, view);
    if (!may_split(q, view) || !may_split(r, view) || q.tiles == 0 || r.tiles == 0) {
        GRP_TRY(run(q, stream));
        return run(r, stream);
    }
    long long tiles = 0;
    for (Product* x : {&q, &r}) {
        x->p.bn = std::min(x->p.bn, 128);
        x->tiles = single_tiles(*x, x->p.bn);
        tiles = std::max(tiles, x->tiles);
    }
    q.p.split = r.p.split = choose_split(q.tiles + r.tiles, std::min(q.blocks, r.blocks), view);
    GroupedProblems problems;
    GRP_TRY(describe(q, &problems.at[0]));
    GRP_TRY(describe(r, &problems.at[1]));
    return launch_single(q, problems, 2, tiles, view, stream);
}

Product blank(int ab_dtype, int c_dtype, int form) {
    Product q;
    std::memset(&q, 0, sizeof q);
    q.ab_dtype = ab_dtype;
    q.c_dtype = c_dtype;
    q.p.form = form;
    q.p.alpha = 1.0f;
    q.p.parts = 1;
    return q;
}

int padded_rank(int rank) { return (rank + 15) / 16 * 16; }
// The workspace begins with the adapters' flags.
constexpr size_t kFlagBytes = static_cast<size_t>(kMaxGemmGroups) * sizeof(uint32_t);
static_assert(kExtChecks == sizeof(uint32_t), "a byte per check");
size_t two_part_bytes(int m, int rank) {
    return (static_cast<size_t>(std::max(m, 0)) * 2 * padded_rank(rank) * 2 + 255) / 256 * 256;
}

int parts_of(int ab_dtype) { return ab_dtype == CKL_BF16 ? kBf16Parts : kF16Parts; }

// T[p] = scales[g] * A[rows[p]] * op(B_g) in two words, for the positions of every adapter.
Product shrink(int ab_dtype, const void* a, int lda, int k, const void* b, int ldb, long long stack,
               bool trans, int rank, const float* scales, void* t, const int* offsets, const int* rows,
               int adapters, int m) {
    Product q = blank(ab_dtype, -1, kFormRows);
    const int rp = padded_rank(rank);
    q.p.offsets = offsets;
    q.p.a_rows = rows;
    q.p.c = t;
    q.p.scales = scales;
    q.p.groups = adapters;
    q.p.rows = q.p.a_count = q.p.c_count = m;
    q.p.n = rp;  // columns rank .. rp read weights outside their matrix, and are stored as zeros
    q.p.ext_rank = rank;
    q.p.k = k;
    q.p.ldc = 2 * rp;
    q.p.c_part_cols = rp;
    q.p.trans_b = trans ? 1 : 0;
    q.a = a;
    q.lda = lda;
    q.a_cols = k;
    q.b = b;
    q.ldb = ldb;
    q.b_cols = trans ? k : rank;
    q.b_outer = trans ? rank : k;
    q.b_depth = adapters;
    q.b_stack = stack;
    return q;
}

// The same for a few rows, where one CTA per row and 32 ranks is a wave or two.
int shrink_rows(int ab_dtype, const void* x, int ldx, int k, const void* a, int lda, long long stack, int rank,
                const float* scales, void* t, const int* offsets, const int* rows, int adapters, int m,
                cudaStream_t stream) {
    DeviceView view;
    GRP_TRY(device_view(&view));
    LoraRowsParams p = {};
    p.offsets = offsets;
    p.rows = rows;
    p.scales = scales;
    p.x = static_cast<const unsigned short*>(x);
    p.a = static_cast<const unsigned short*>(a);
    p.t = static_cast<unsigned short*>(t);
    p.a_stride = stack;
    p.adapters = adapters;
    p.m = m;
    p.k = k;
    p.rank = rank;
    p.part_cols = padded_rank(rank);
    p.ldx = ldx;
    p.lda = lda;
    const dim3 grid(static_cast<unsigned>(m), static_cast<unsigned>((rank + kLoraRanks - 1) / kLoraRanks));
    GRP_TRY_CUDA(launch_dependent(ab_dtype == CKL_BF16 ? lora_rows_kernel<__nv_bfloat16> : lora_rows_kernel<__half>,
                                  grid, kLoraRowsThreads, 0, 1, stream, p));
    return CKL_OK;
}

// C[rows[p]] = A[rows[p]] * op(B) + T[p] * op(E_g) + beta * C[rows[p]], C of n columns.
Product expand(int ab_dtype, int c_dtype, const void* a, int lda, int k, const void* b, int ldb, int n,
               bool trans, const void* flags, const void* t, int rank, const void* e, int lde, long long e_stack,
               void* c, int ldc, const int* offsets, const int* rows, int adapters, int m, float beta) {
    Product q = blank(ab_dtype, c_dtype, kFormRows);
    const int rp = padded_rank(rank);
    q.p.offsets = offsets;
    q.p.a_rows = q.p.c_rows = rows;
    q.p.c = c;
    q.p.groups = adapters;
    q.p.parts = parts_of(ab_dtype);
    q.p.ext_cols = rp;
    q.p.ext_rank = rank;
    q.p.ext_flags = static_cast<const uint32_t*>(flags);
    q.p.rows = q.p.a_count = q.p.c_count = m;
    q.p.n = n;
    q.p.k = k;
    q.p.ldc = ldc;
    q.p.beta = beta;
    q.p.trans_b = trans ? 1 : 0;
    q.a = a;
    q.lda = lda;
    q.a_cols = k;
    q.b = b;
    q.ldb = ldb;
    q.b_cols = trans ? k : n;
    q.b_outer = trans ? n : k;
    q.b_depth = 1;
    q.b_stack = static_cast<long long>(ldb) * q.b_outer;
    q.t = t;
    q.ldt = 2 * rp;
    q.e = e;
    q.lde = lde;
    q.e_stack = e_stack;
    q.e_cols = trans ? rank : n;
    q.e_outer = trans ? n : rank;
    return q;
}

int check_lora(const char* what, int ab_dtype, int out_dtype, const void* w, int ldw, const void* lora_a,
               int ldla, long long stride_a, const void* lora_b, int ldlb, long long stride_b,
               const float* scales, const int* offsets, const int* rows, int adapters, int m, int n,
               int k, int rank, const void* workspace, size_t have, size_t need) {
    GRP_TRY(check_types(what, ab_dtype, out_dtype));
    GRP_TRY(check_groups(what, offsets, adapters, m, n, k));
    if (rank < 1 || rank > kMaxLoraRank) {
        return set_error(rank < 1 ? CKL_ERR_INVALID_ARG : CKL_ERR_TOO_LARGE, "%s: rank %d (1 to %d)", what,
                         rank, kMaxLoraRank);
    }
    if (k < 1) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: k = %d", what, k);
    }
    GRP_TRY(check_operand(what, "w", w, ldw, n, 0));
    GRP_TRY(check_operand(what, "lora_a", lora_a, ldla, rank, stride_a));
    GRP_TRY(check_operand(what, "lora_b", lora_b, ldlb, n, stride_b));
    if (misaligned(scales, 4) || misaligned(rows, 4)) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: misaligned scales or rows", what);
    }
    if (need > 0 && (workspace == nullptr || misaligned(workspace, 256) || have < need)) {
        return set_error(CKL_ERR_INVALID_ARG,
                         "%s: the workspace is %p of %zu bytes, needed are %zu on a 256-byte boundary", what,
                         workspace, have, need);
    }
    return CKL_OK;
}

}  // namespace

extern "C" {

int ckl_gemm_grouped(int ab_dtype, const void* a, const int* a_rows, int a_count, const void* b, void* c,
                     int c_dtype, const int* offsets, int groups, int rows, int n, int k, int lda, int ldb,
                     long long stride_b, int ldc, int trans_b, float alpha, float beta,
                     ckl_stream_t stream) {
    const char* what = "gemm_grouped";
    if (rows <= 0 || n <= 0) {
        return CKL_OK;
    }
    GRP_TRY(check_types(what, ab_dtype, c_dtype));
    GRP_TRY(check_groups(what, offsets, groups, rows, n, k));
    k = std::max(k, 0);
    if (k > 0) {
        GRP_TRY(check_operand(what, "a", a, lda, k, 0));
        GRP_TRY(check_operand(what, "b", b, ldb, trans_b ? k : n, stride_b));
    }
    if (a_rows == nullptr) {
        a_count = rows;
    }
    if (a_count < 0 || misaligned(a_rows, 4) || c == nullptr || ldc < n || misaligned(c, size_of(c_dtype))) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: a_count %d, c %p, ldc %d for n %d", what, a_count, c, ldc, n);
    }
    Product q = blank(ab_dtype, c_dtype, kFormRows);
    q.p.offsets = offsets;
    q.p.a_rows = a_rows;
    q.p.c = c;
    q.p.groups = groups;
    q.p.rows = q.p.c_count = rows;
    q.p.a_count = a_count;
    q.p.n = n;
    q.p.k = k;
    q.p.ldc = ldc;
    q.p.alpha = alpha;
    q.p.beta = beta;
    q.p.trans_b = trans_b != 0 ? 1 : 0;
    q.a = a;
    q.lda = lda;
    q.a_cols = k;
    q.b = b;
    q.ldb = ldb;
    q.b_cols = trans_b ? k : n;
    q.b_outer = trans_b ? n : k;
    q.b_depth = groups;
    q.b_stack = stride_b;
    return run(q, static_cast<cudaStream_t>(stream));
}

int ckl_gemm_grouped_wgrad(int ab_dtype, const void* a, const int* a_rows, int a_count, const void* g,
                           void* dw, int dw_dtype, const int* offsets, int groups, int rows, int m, int n,
                           int lda, int ldg, int lddw, long long stride_dw, float alpha, float beta,
                           ckl_stream_t stream) {
    const char* what = "gemm_grouped_wgrad";
    if (m <= 0 || n <= 0) {
        return CKL_OK;
    }
    rows = std::max(rows, 0);
    GRP_TRY(check_types(what, ab_dtype, dw_dtype));
    GRP_TRY(check_groups(what, offsets, groups, rows, n, m));
    if (rows > 0) {
        GRP_TRY(check_operand(what, "a", a, lda, m, 0));
        GRP_TRY(check_operand(what, "g", g, ldg, n, 0));
    }
    if (a_rows == nullptr) {
        a_count = rows;
    }
    if (a_count < 0 || misaligned(a_rows, 4) || dw == nullptr || lddw < n || stride_dw < 0 ||
        misaligned(dw, size_of(dw_dtype))) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: a_count %d, dw %p, lddw %d for n %d, stride %lld", what,
                         a_count, dw, lddw, n, stride_dw);
    }
    Product q = blank(ab_dtype, dw_dtype, kFormWgrad);
    q.p.offsets = offsets;
    q.p.a_rows = a_rows;
    q.p.c = dw;
    q.p.c_stride = stride_dw;
    q.p.groups = groups;
    q.p.rows = q.p.b_count = rows;
    q.p.a_count = a_count;
    q.p.m = m;
    q.p.n = n;
    q.p.ldc = lddw;
    q.p.alpha = alpha;
    q.p.beta = beta;
    q.a = a;
    q.lda = lda;
    q.a_cols = m;
    q.b = g;
    q.ldb = ldg;
    q.b_cols = n;
    q.b_depth = 1;
    q.b_stack = static_cast<long long>(ldg) * std::max(rows, 1);
    return run(q, static_cast<cudaStream_t>(stream));
}

size_t ckl_gemm_lora_workspace_bytes(int m, int rank, int backward) {
    return m < 1 || rank < 1 || rank > kMaxLoraRank
               ? 0
               : kFlagBytes + two_part_bytes(m, rank) * (backward != 0 ? 2 : 1);
}

int ckl_gemm_lora(int ab_dtype, const void* x, const void* w, const void* lora_a, const void* lora_b,
                  const float* scales, void* y, int y_dtype, const int* offsets, const int* rows,
                  int adapters, int m, int n, int k, int rank, int ldx, int ldw, int ldla,
                  long long stride_a, int ldlb, long long stride_b, int ldy, float beta, void* workspace,
                  size_t workspace_bytes, ckl_stream_t stream) {
    const char* what = "gemm_lora";
    if (m <= 0 || n <= 0) {
        return CKL_OK;
    }
    GRP_TRY(check_lora(what, ab_dtype, y_dtype, w, ldw, lora_a, ldla, stride_a, lora_b, ldlb, stride_b, scales,
                       offsets, rows, adapters, m, n, k, rank, workspace, workspace_bytes,
                       ckl_gemm_lora_workspace_bytes(m, rank, 0)));
    GRP_TRY(check_operand(what, "x", x, ldx, k, 0));
    if (y == nullptr || ldy < n || misaligned(y, size_of(y_dtype))) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: y %p, ldy %d for n %d", what, y, ldy, n);
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* t = static_cast<unsigned char*>(workspace) + kFlagBytes;
    DeviceView view;
    GRP_TRY(device_view(&view));
    if (static_cast<long long>(m) * ((rank + kLoraRanks - 1) / kLoraRanks) <= 2ll * view.sm_count) {
        GRP_TRY(shrink_rows(ab_dtype, x, ldx, k, lora_a, ldla, stride_a, rank, scales, t, offsets, rows,
                            adapters, m, s));
    } else {
        Product p = shrink(ab_dtype, x, ldx, k, lora_a, ldla, stride_a, false, rank, scales, t, offsets, rows,
                           adapters, m);
        GRP_TRY(run(p, s));
    }
    Product q = expand(ab_dtype, y_dtype, x, ldx, k, w, ldw, n, false, workspace, t, rank, lora_b, ldlb, stride_b,
                       y, ldy, offsets, rows, adapters, m, beta);
    return run(q, s);
}

int ckl_gemm_lora_backward(int ab_dtype, const void* dy, const void* x, const void* w, const void* lora_a,
                           const void* lora_b, const float* scales, void* dx, int dx_dtype, void* da,
                           void* db, int dab_dtype, const int* offsets, const int* rows, int adapters, int m,
                           int n, int k, int rank, int lddy, int ldx, int ldw, int ldla, long long stride_a,
                           int ldlb, long long stride_b, int lddx, int ldda, long long stride_da, int lddb,
                           long long stride_db, float beta, void* workspace, size_t workspace_bytes,
                           ckl_stream_t stream) {
    const char* what = "gemm_lora_backward";
    if (n <= 0 || k <= 0) {
        return CKL_OK;
    }
    m = std::max(m, 0);
    GRP_TRY(check_types(what, ab_dtype, dab_dtype));
    GRP_TRY(check_lora(what, ab_dtype, dx_dtype, w, ldw, lora_a, ldla, stride_a, lora_b, ldlb, stride_b, scales,
                       offsets, rows, adapters, m, n, k, rank, workspace, workspace_bytes,
                       ckl_gemm_lora_workspace_bytes(m, rank, 1)));
    if (m > 0) {
        GRP_TRY(check_operand(what, "dy", dy, lddy, n, 0));
        if (da != nullptr || db != nullptr) {
            GRP_TRY(check_operand(what, "x", x, ldx, k, 0));
        }
    }
    if ((dx != nullptr && (lddx < k || misaligned(dx, size_of(dx_dtype)))) ||
        (da != nullptr && (ldda < rank || stride_da < 0 || misaligned(da, size_of(dab_dtype)))) ||
        (db != nullptr && (lddb < n || stride_db < 0 || misaligned(db, size_of(dab_dtype))))) {
        return set_error(CKL_ERR_INVALID_ARG, "%s: a gradient is misaligned or lddx %d, ldda %d, lddb %d is too small",
                         what, lddx, ldda, lddb);
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* u = static_cast<unsigned char*>(workspace) + kFlagBytes;
    void* t = static_cast<unsigned char*>(u) + two_part_bytes(m, rank);
    const int rp = padded_rank(rank);
    const bool need_u = m > 0 && (dx != nullptr || da != nullptr), need_t = m > 0 && db != nullptr;
    Product pu = shrink(ab_dtype, dy, lddy, n, lora_b, ldlb, stride_b, true, rank, scales, u, offsets, rows,
                        adapters, m);
    Product pt = shrink(ab_dtype, x, ldx, k, lora_a, ldla, stride_a, false, rank, scales, t, offsets, rows,
                        adapters, m);
    if (need_u && need_t) {
        GRP_TRY(run_two(pu, pt, s));
    } else if (need_u) {
        GRP_TRY(run(pu, s));
    } else if (need_t) {
        GRP_TRY(run(pt, s));
    }
    Product pa = blank(ab_dtype, dab_dtype, kFormWgrad);
    pa.p.offsets = offsets;
    pa.p.a_rows = rows;
    pa.p.c = da;
    pa.p.c_stride = stride_da;
    pa.p.groups = adapters;
    pa.p.rows = pa.p.a_count = pa.p.b_count = m;
    pa.p.m = k;
    pa.p.n = rank;
    pa.p.ldc = ldda;
    pa.p.beta = beta;
    pa.p.parts = parts_of(ab_dtype);
    pa.p.layered = kLayeredB;
    pa.p.part_cols = rp;
    pa.a = x;
    pa.lda = ldx;
    pa.a_cols = k;
    pa.b = u;
    pa.ldb = pa.b_cols = 2 * rp;
    pa.b_depth = 1;
    pa.b_stack = static_cast<long long>(pa.ldb) * std::max(m, 1);
    Product pb = blank(ab_dtype, dab_dtype, kFormWgrad);
    pb.p.offsets = offsets;
    pb.p.b_rows = rows;
    pb.p.c = db;
    pb.p.c_stride = stride_db;
    pb.p.groups = adapters;
    pb.p.rows = pb.p.a_count = pb.p.b_count = m;
    pb.p.m = rank;
    pb.p.n = n;
    pb.p.ldc = lddb;
    pb.p.beta = beta;
    pb.p.parts = parts_of(ab_dtype);
    pb.p.layered = kLayeredA;
    pb.p.part_cols = rp;
    pb.a = t;
    pb.lda = pb.a_cols = 2 * rp;
    pb.b = dy;
    pb.ldb = lddy;
    pb.b_cols = n;
    pb.b_depth = 1;
    pb.b_stack = static_cast<long long>(lddy) * std::max(m, 1);
    if (da != nullptr && db != nullptr) {
        GRP_TRY(run_two(pa, pb, s));
    } else if (da != nullptr) {
        GRP_TRY(run(pa, s));
    } else if (db != nullptr) {
        GRP_TRY(run(pb, s));
    }
    if (m > 0 && dx != nullptr) {
        Product q = expand(ab_dtype, dx_dtype, dy, lddy, n, w, ldw, k, true, workspace, u, rank, lora_a, ldla, stride_a, dx,
                           lddx, offsets, rows, adapters, m, 0.0f);
        GRP_TRY(run(q, s));
    }
    return CKL_OK;
}

}  // extern "C"
