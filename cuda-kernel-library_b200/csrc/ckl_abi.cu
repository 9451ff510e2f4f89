// C ABI of the library (include/ckl_gemm.h): argument checking, the planner
// that picks a kernel and a tile schedule, TMA descriptor construction, the
// per-device state (status word, stream-K workspace, host staging buffers) and
// the launches.  Only the CUDA runtime is linked; the one driver entry point
// needed (cuTensorMapEncodeTiled) is fetched through the runtime.

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ckl_gemm.h"
#include "ckl_internal.h"
#include "gemm_fp32.cuh"
#include "gemm_simt.cuh"
#include "gemm_umma.cuh"
#include "tile_sched.h"
#include "trsm.cuh"

namespace {
thread_local std::string g_last_error;
}  // namespace

namespace ckl {
int set_error(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}
}  // namespace ckl

namespace {

using namespace ckl;

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

#define CKL_TRY_CUDA(expr)                                                                  \
    do {                                                                                    \
        const cudaError_t err__ = (expr);                                                   \
        if (err__ != cudaSuccess) {                                                         \
            return fail(CKL_ERR_CUDA, "%s failed: %s (%s)", #expr, cudaGetErrorName(err__), \
                        cudaGetErrorString(err__));                                         \
        }                                                                                   \
    } while (0)

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct Staging {
    void* ptr = nullptr;
    size_t bytes = 0;
    unsigned int epoch = 0;  // stream-K workspaces: value of the "partial is ready" flags of the last launch
};

// One encoded TMA descriptor and what it was encoded from.  A descriptor is a pure function of
// these fields, so an entry stays valid for as long as a buffer with that address and shape is
// what the caller passes, whoever allocated it.
struct MapKey {
    const void* base;
    uint64_t inner, outer, pitch;
    int dtype;
    uint32_t box_inner, box_outer;
    bool operator==(const MapKey& o) const {
        return base == o.base && inner == o.inner && outer == o.outer && pitch == o.pitch &&
               dtype == o.dtype && box_inner == o.box_inner && box_outer == o.box_outer;
    }
};
struct MapEntry {
    MapKey key = {};
    CUtensorMap map = {};
    uint64_t stamp = 0;  // 0 = empty; else the clock value of the last use
};

struct DeviceCtx {
    int device = -1;
    int sm_count = 0;
    int cc_major = 0;
    int max_pairs = 0;
    EncodeTiledFn encode = nullptr;
    unsigned int* status = nullptr;            // 4 words on the device
    std::map<cudaStream_t, Staging> workspace; // stream-K partial slots, one per stream
    std::map<cudaStream_t, Staging> repack;    // aligned copies of operands TMA cannot describe
    Staging host_a, host_b, host_c;            // device staging for ckl_gemm_host
    cudaStream_t host_stream = nullptr;        // ckl_gemm_host: compute
    cudaStream_t host_in = nullptr;            // ckl_gemm_host: host -> device copies
    cudaStream_t host_out = nullptr;           // ckl_gemm_host: device -> host copies
    static constexpr int kHostPanels = 16;
    cudaEvent_t host_events[2 * kHostPanels] = {};  // per panel: uploaded, computed
    std::mutex host_mu;                        // one ckl_gemm_host call at a time per device
    bool attrs_set = false;
    // Recently used TMA descriptors (least recently used entry is replaced).  Encoding one
    // costs a driver call; a small GEMM launched in a loop would otherwise pay three per call.
    static constexpr int kMapCache = 48;
    MapEntry map_cache[kMapCache];
    uint64_t map_clock = 0;
    std::mutex mu;
};

std::atomic<unsigned long long> g_tensor_map_encodes{0};
// Armed by ckl_test_arm_wait_fault for the calling thread's next tensor-core launch.
struct WaitFault {
    int kind = 0;
    unsigned long long limit_ns = 0;
};
thread_local WaitFault g_wait_fault;
thread_local ckl_plan g_last_plan = {};

std::mutex g_ctx_mu;
std::map<int, std::unique_ptr<DeviceCtx>> g_ctx;

template <int kMode, typename OutT>
cudaError_t set_umma_attr() {
    return cudaFuncSetAttribute(umma_gemm_kernel<kMode, OutT>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(UmmaConfig<kMode>::kSmemBytes));
}

int get_ctx(DeviceCtx** out) {
    int dev = 0;
    CKL_TRY_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(g_ctx_mu);
    auto it = g_ctx.find(dev);
    if (it != g_ctx.end()) {
        *out = it->second.get();
        return CKL_OK;
    }
    auto ctx = std::make_unique<DeviceCtx>();
    ctx->device = dev;
    cudaDeviceProp prop;
    CKL_TRY_CUDA(cudaGetDeviceProperties(&prop, dev));
    ctx->sm_count = prop.multiProcessorCount;
    ctx->cc_major = prop.major;
    if (prop.major != 10) {
        return fail(CKL_ERR_UNSUPPORTED,
                    "device %d is compute capability %d.%d; this library is built for sm_100a only",
                    dev, prop.major, prop.minor);
    }
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    CKL_TRY_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
    if (fn == nullptr || qres != cudaDriverEntryPointSuccess) {
        return fail(CKL_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    }
    ctx->encode = reinterpret_cast<EncodeTiledFn>(fn);
    CKL_TRY_CUDA(cudaMalloc(&ctx->status, 4 * sizeof(unsigned int)));
    CKL_TRY_CUDA(cudaMemset(ctx->status, 0, 4 * sizeof(unsigned int)));
    CKL_TRY_CUDA((set_umma_attr<kModeSingle, float>()));
    CKL_TRY_CUDA((set_umma_attr<kModeSingle, __half>()));
    CKL_TRY_CUDA((set_umma_attr<kModeSingle, __nv_bfloat16>()));
    CKL_TRY_CUDA((set_umma_attr<kModePair, float>()));
    CKL_TRY_CUDA((set_umma_attr<kModePair, __half>()));
    CKL_TRY_CUDA((set_umma_attr<kModePair, __nv_bfloat16>()));
    CKL_TRY_CUDA((set_umma_attr<kModePairWide, float>()));
    CKL_TRY_CUDA((set_umma_attr<kModePairWide, __half>()));
    CKL_TRY_CUDA((set_umma_attr<kModePairWide, __nv_bfloat16>()));
    // How many CTA pairs can be resident at once (pairs must share a TPC/GPC).
    {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(ctx->sm_count / 2 * 2));
        cfg.blockDim = dim3(UmmaConfig<kModePairWide>::kThreads);
        cfg.dynamicSmemBytes = UmmaConfig<kModePairWide>::kSmemBytes;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        const cudaError_t e =
            cudaOccupancyMaxActiveClusters(&clusters, umma_gemm_kernel<kModePairWide, float>, &cfg);
        if (e != cudaSuccess || clusters <= 0) {
            (void)cudaGetLastError();
            clusters = ctx->sm_count / 2;
        }
        ctx->max_pairs = std::min(clusters, ctx->sm_count / 2);
    }
    *out = ctx.get();
    g_ctx[dev] = std::move(ctx);
    return CKL_OK;
}

size_t dtype_size(int dtype) { return dtype == CKL_F32 ? 4 : 2; }

constexpr int kLastAlgo = CKL_ALGO_UMMA_1CTA_N128_SK;
bool is_tensor_algo(int algo) { return algo >= CKL_ALGO_UMMA_1CTA && algo <= kLastAlgo; }
int mode_of_algo(int algo) {
    switch (algo) {
        case CKL_ALGO_UMMA_2CTA:
        case CKL_ALGO_UMMA_2CTA_SK: return kModePair;
        case CKL_ALGO_UMMA_2CTA_WIDE:
        case CKL_ALGO_UMMA_2CTA_WIDE_SK: return kModePairWide;
        default: return kModeSingle;
    }
}
bool is_sk_algo(int algo) {
    return algo == CKL_ALGO_UMMA_SK || algo == CKL_ALGO_UMMA_2CTA_SK ||
           algo == CKL_ALGO_UMMA_2CTA_WIDE_SK || algo == CKL_ALGO_UMMA_1CTA_N128_SK;
}
bool is_narrow_algo(int algo) {
    return algo == CKL_ALGO_UMMA_1CTA_N128 || algo == CKL_ALGO_UMMA_1CTA_N128_SK;
}
struct ModeDims {
    int tile_m, tile_n, tile_k;
    size_t slot_bytes;
};
ModeDims dims_of_mode(int mode) {
    switch (mode) {
        case kModePair:
            return {UmmaConfig<kModePair>::kTileM, UmmaConfig<kModePair>::kTileN,
                    UmmaConfig<kModePair>::kTileK, UmmaConfig<kModePair>::kSlotFloats * sizeof(float)};
        case kModePairWide:
            return {UmmaConfig<kModePairWide>::kTileM, UmmaConfig<kModePairWide>::kTileN,
                    UmmaConfig<kModePairWide>::kTileK,
                    UmmaConfig<kModePairWide>::kSlotFloats * sizeof(float)};
        default:
            return {UmmaConfig<kModeSingle>::kTileM, UmmaConfig<kModeSingle>::kTileN,
                    UmmaConfig<kModeSingle>::kTileK,
                    UmmaConfig<kModeSingle>::kSlotFloats * sizeof(float)};
    }
}

// ---- planner (pure host arithmetic) ------------------------------------------

struct Plan {
    int algo = CKL_ALGO_SIMT;
    int mode = kModeSingle;
    bool pair = false;
    bool repack = false;  // AUTO only: A and/or B are first copied to an aligned pitch
    int tile_m = 64, tile_n = 64, tile_k = 16;
    int grid = 0;
    Schedule sched = {};
    size_t workspace_bytes = 0;
};

// Plan -> the public struct
void export_plan(const Plan& plan, ckl_plan* out) {
    out->algo = plan.algo;
    out->tile_m = plan.tile_m;
    out->tile_n = plan.tile_n;
    out->tile_k = plan.tile_k;
    out->tiles_m = plan.sched.tiles_m;
    out->tiles_n = plan.sched.tiles_n;
    out->k_blocks = plan.sched.k_blocks;
    out->grid = plan.grid;
    out->units = plan.sched.units;
    out->group_m = plan.sched.group_m;
    out->dp_tiles = plan.sched.dp_tiles;
    out->sk_tiles = plan.sched.sk_tiles;
    out->sk_units = plan.sched.sk_tiles > 0 ? plan.sched.units : 0;
    out->sk_iters = plan.sched.sk_iters;
    out->workspace_bytes = plan.workspace_bytes;
    out->repack = plan.repack ? 1 : 0;
}

// 2^28 multiply-adds (645^3): below this the general kernel's one launch wins.
constexpr long long kRepackMinMacs = 1LL << 28;

bool tma_legal(int k, int lda, int ldb, size_t a_align, size_t b_align) {
    return k > 0 && lda % 8 == 0 && ldb % 8 == 0 && a_align % 16 == 0 && b_align % 16 == 0;
}

// want_sk: 0 = never, 1 = always when a remainder exists, 2 = heuristic.
Schedule make_schedule(int m, int n, int k, int mode, int max_units, int want_sk, bool narrow = false) {
    Schedule s = {};
    ModeDims d = dims_of_mode(mode);
    if (narrow) {
        d.tile_n = 128;  // the single-CTA kernel's 128-column form
    }
    s.tiles_m = (m + d.tile_m - 1) / d.tile_m;
    s.tiles_n = (n + d.tile_n - 1) / d.tile_n;
    s.k_blocks = (k + d.tile_k - 1) / d.tile_k;
    // Raster group height: a wave of tiles should cover a block of C that is about as tall as
    // it is wide, so that it reads the least A + B.  256x512 tiles are twice as wide as tall,
    // so their groups are twice as high when there are columns enough (measured, 8192^3:
    // 1599 vs 1592 TFLOP/s; 6144^3: 1550 vs 1538).
    s.group_m = mode == kModeSingle ? 16 : (mode == kModePairWide && s.tiles_n >= 8) ? 16 : 8;
#ifdef CKL_EXP
    if (const char* g = std::getenv("CKL_GROUP_M")) {
        s.group_m = std::max(1, std::atoi(g));
    }
#endif
    const int tiles = s.tiles_m * s.tiles_n;
    s.units = std::max(1, std::min(max_units, tiles));
    s.dp_tiles = tiles;
    s.sk_tiles = 0;
    s.sk_iters = 0;
    if (want_sk == 0 || max_units <= 0) {
        return s;
    }
    const int full_waves = tiles / max_units;
    const int rem = tiles % max_units;
    if (rem == 0) {
        return s;
    }
    int sk_tiles = rem;
    // Give every unit a run of k blocks of split work worth its parked partial tile (2048 k):
    // if the remainder alone is too thin, fold one full wave into the split region as well.
    // (2048 x 2816 x 4096: 14 tiles over 74 pairs leave each pair 6 k blocks of 128 and one
    // parked partial tile, and the split measures no faster than none: 1041 against 1077.)
    // A forced split (tests, benchmarks) keeps the lower bar of a few k blocks per unit.
    const long long thin = want_sk != 2 ? 4 : (d.tile_k >= 128 ? 16 : 32);
    if (full_waves >= 1 && static_cast<long long>(rem) * s.k_blocks < thin * max_units) {
        sk_tiles = rem + max_units;
    }
    const long long sk_iters = static_cast<long long>(sk_tiles) * s.k_blocks;
    if (want_sk == 2) {
        // Heuristic (measured).  Fewer tiles than units: the split pays for its partial-tile
        // traffic and fix-up pass when whole tiles would leave a quarter or more of the
        // machine idle and every unit still gets a long run of k blocks.  One or more full
        // waves: the split (fused, hidden behind the whole tiles) pays when the last wave
        // would be at most 60 % full (4096^3: 34 of 74; at 78 % and above it measured a loss).
        if (full_waves >= 1) {
            if (rem * 10 > max_units * 6) {
                return s;
            }
            // Folding a wave into a thin remainder must leave every unit a whole tile to hide
            // the reduction behind; with a single full wave it would split EVERY tile and end
            // in the separate fix-up pass (2048 x 2816 x 2048: 625 TFLOP/s against 864 unsplit).
            if (tiles - sk_tiles < max_units) {
                return s;
            }
            // Parking and adding a partial tile costs the same whatever k is; below k = 4096
            // it is not won back (4096 x 4096 x 2048: 1281 split against 1425 unsplit,
            // 4096 x 2816 x 1024: 809 against 1010; from k = 4096 on the split is level or ahead).
            if (static_cast<long long>(s.k_blocks) * d.tile_k < 4096) {
                return s;
            }
        } else {
            // Every tile would be cut over f units and finished by the fix-up pass, which costs
            // about as much as 40 k blocks of 64 (20 of 128) of one tile; the cut saves
            // k_blocks * (1 - 1/f) of them (1536^3, f = 2, 24 k blocks: 369 TFLOP/s split
            // against 530 unsplit; 1024 x 1024 x 8192, f = 4, 128 k blocks: 676 against 409).
            const long long f = max_units / tiles;
            const long long saved = f >= 2 ? static_cast<long long>(s.k_blocks) * (f - 1) / f : 0;
            // ... plus a tenth of that per partial tile it adds (512 x 512 x 4096 in 128x128
            // tiles, f = 9: 113 TFLOP/s cut against 133 uncut).
            const long long pass_cost = (d.tile_k >= 128 ? 20 : 40) + (d.tile_k >= 128 ? 2 : 4) * f;
            if (tiles * 4 > max_units * 3 || saved < pass_cost) {
                return s;
            }
        }
    }
    if (sk_iters < max_units) {
        return s;  // fewer k blocks than units: nothing to balance
    }
    s.units = max_units;
    if (full_waves == 0) {
        // Every tile is split: use a whole number of units per tile, so that each tile is cut
        // at the same k offsets.  Units working on tiles of one tile row (or column) then walk
        // the same k blocks at the same time and share A (or B) in L2; with `max_units` equal
        // ranges the offsets drift from tile to tile and most of that reuse is lost
        // (1024x1024x32768 FP16, 74 pairs: 927 TFLOP/s with 74 ranges, 1106 with 16 x 4).
        s.units = tiles * (max_units / tiles);
    }
    s.sk_tiles = sk_tiles;
    s.dp_tiles = tiles - sk_tiles;
    s.sk_iters = sk_iters;
    return s;
}

// c_traffic: bytes of C moved per output element by the epilogue (element size, doubled when
// C is also read), which sets how long the exposed epilogue of the 256x512 tile is.
int make_plan(int m, int n, int k, int lda, int ldb, size_t a_align, size_t b_align, int algo,
              int sm_count, int max_pairs, int c_traffic, Plan* plan) {
    bool legal = tma_legal(k, lda, ldb, a_align, b_align);
    int resolved = algo;
    plan->repack = false;
    if (algo == CKL_ALGO_AUTO && !legal && k > 0 &&
        static_cast<long long>(m) * n * static_cast<long long>(k) >= kRepackMinMacs) {
        // Operands TMA cannot describe (base not 16-byte aligned, pitch not a multiple of 8
        // elements): from this size on two copy passes to an aligned pitch and the tensor-core
        // kernel beat the CUDA-core kernel by a wide margin.  Smaller problems keep the
        // general kernel, whose single launch is cheaper than three.
        legal = true;
        plan->repack = true;
    }
    if (algo == CKL_ALGO_AUTO) {
        // Measured on B200: once there is at least one 256x256 tile per CTA pair the pair
        // kernel wins (half the B traffic per SM); below that the 128x256 single-CTA tiles
        // fill more SMs.
        const long long pair_tiles =
            static_cast<long long>((m + 255) / 256) * static_cast<long long>((n + 255) / 256);
        const long long wide_tiles =
            static_cast<long long>((m + 255) / 256) * static_cast<long long>((n + 511) / 512);
        // The wide tile saves a quarter of the L2-to-SM traffic (higher clocks under the power
        // cap) but exposes its epilogue between tiles; measured, it wins only when the
        // main loop is long (k >= 4096; 8192 when the epilogue both reads and writes an FP32
        // C: 16384x14336x4096, FP32 C, beta 0.5: 1301 vs 1368 TFLOP/s on the 256x256 tile) and no
        // tile column is mostly padding.
        auto wave_fill = [&](long long tiles) {  // share of unit-slots the last wave leaves busy
            const long long waves = (tiles + max_pairs - 1) / max_pairs;
            return static_cast<double>(tiles) / static_cast<double>(waves * max_pairs);
        };
        const int wide_min_k = c_traffic >= 8 ? 8192 : 4096;  // FP32 C read and written: longer drain
        bool use_wide = max_pairs > 0 && wide_tiles * 5 >= max_pairs * 4LL && k >= wide_min_k &&
                        (n % 512 == 0 || n % 512 > 384) &&
                        wave_fill(wide_tiles) >= wave_fill(pair_tiles) - 0.02;
        // Between k = 4096 and 8192 the exposed epilogue is 5-9 % of a tile, and the 256x256
        // tile with its split last wave has no quantisation loss at all: there the wide tile
        // keeps the job only for at most two waves or when its own last wave is nearly full
        // (5120^3, last wave 70 % full: 1171-1281 TFLOP/s wide against 1345-1385 split
        // 256x256; 2048 x 12288 x 4096: 1137-1178 against 1239-1278; 4096^3, two waves:
        // 1455-1472 against 1415-1447).
        if (use_wide && k < 8192 && wide_tiles > 2LL * max_pairs && wave_fill(wide_tiles) < 0.95) {
            use_wide = false;
        }
        // Row pitches that are not multiples of 128 bytes double the L2 requests of every TMA
        // box row; the wide tile needs a quarter fewer of them per MMA cycle and then wins from
        // shorter k already, provided its waves fill (3000^3: 986 against 844 TFLOP/s).
        const bool odd_pitch = (static_cast<long long>(lda) * 2) % 128 != 0 ||
                               (static_cast<long long>(ldb) * 2) % 128 != 0;
        if (!use_wide && odd_pitch && max_pairs > 0 && k >= 2048 && c_traffic < 8 &&
            wide_tiles * 5 >= max_pairs * 4LL && wave_fill(wide_tiles) >= 0.9) {
            use_wide = true;
        }
        // Fewer 256x256 tiles than half the pairs: split every tile over a whole number of
        // pairs, provided each still gets a long run of k blocks (128 k each); measured better
        // than 128x256 single-CTA tiles split the same way (half the B traffic per SM).
        const long long pair_split = pair_tiles > 0 ? max_pairs / pair_tiles : 0;
        const bool use_pair_split =
            max_pairs > 0 && pair_split >= 2 && ((k + 127) / 128) / pair_split >= 24;
        const bool use_pair = max_pairs > 0 && (pair_tiles >= max_pairs || use_pair_split);
        resolved = !legal      ? CKL_ALGO_SIMT
                   : use_wide ? CKL_ALGO_UMMA_2CTA_WIDE_SK
                   : use_pair ? CKL_ALGO_UMMA_2CTA_SK
                              : CKL_ALGO_UMMA_SK;
    } else if (is_tensor_algo(algo) && !legal) {
        return fail(CKL_ERR_UNSUPPORTED,
                    "tensor-core algo %s needs k > 0, A and B 16-byte aligned and lda, ldb "
                    "multiples of 8 elements (lda=%d ldb=%d k=%d)",
                    ckl_algo_name(algo), lda, ldb, k);
    } else if (algo < CKL_ALGO_AUTO || algo > kLastAlgo) {
        return fail(CKL_ERR_INVALID_ARG, "unknown algo %d", algo);
    }
    plan->algo = resolved;
    if (resolved == CKL_ALGO_SIMT) {
        plan->pair = false;
        plan->tile_m = 64;
        plan->tile_n = 64;
        plan->tile_k = 16;
        plan->sched = {};
        plan->sched.tiles_m = (m + 63) / 64;
        plan->sched.tiles_n = (n + 63) / 64;
        plan->sched.k_blocks = (k + 15) / 16;
        plan->sched.dp_tiles = plan->sched.tiles_m * plan->sched.tiles_n;
        plan->sched.units = plan->sched.dp_tiles;
        plan->grid = plan->sched.dp_tiles;
        plan->workspace_bytes = 0;
        return CKL_OK;
    }
    const int mode = mode_of_algo(resolved);
    const bool pair = mode != kModeSingle;
    int want_sk = 0;
    if (is_sk_algo(resolved)) {
        want_sk = (algo == CKL_ALGO_AUTO) ? 2 : 1;
        if (algo == CKL_ALGO_AUTO && mode == kModePairWide) {
            want_sk = 0;  // one accumulator: a split tile's reduction cannot hide behind the next tile
        }
    }
    const int max_units = pair ? max_pairs : sm_count;
    if (max_units <= 0) {
        return fail(CKL_ERR_UNSUPPORTED, "no schedulable units (sm_count=%d)", sm_count);
    }
    const ModeDims d = dims_of_mode(mode);
    bool narrow = is_narrow_algo(resolved);
    plan->mode = mode;
    plan->pair = pair;
    plan->tile_m = d.tile_m;
    plan->tile_k = d.tile_k;
    if (algo == CKL_ALGO_AUTO && mode == kModeSingle && n > 128 &&
        2LL * ((m + d.tile_m - 1) / d.tile_m) * ((n + d.tile_n - 1) / d.tile_n) <= max_units) {
        // 128x256 tiles would keep at most half of the SMs busy: 128x128 tiles give twice as
        // many, each with half the main loop and half the epilogue (1536^3: 684 against 551
        // TFLOP/s, 1024^3: 270 against 211), and where every tile is cut over several CTAs the
        // partial tiles are half as large (1024 x 1024 x 8192: 637 against 576).
        narrow = true;
    }
    plan->sched = make_schedule(m, n, k, mode, max_units, want_sk, narrow);
    plan->tile_n = narrow ? 128 : d.tile_n;
    plan->grid = plan->sched.units * (pair ? 2 : 1);
    if (plan->sched.sk_tiles > 0) {
        plan->workspace_bytes = 2ull * static_cast<size_t>(plan->sched.units) * d.slot_bytes;
    } else {
        plan->workspace_bytes = 0;
        if (algo == CKL_ALGO_AUTO) {
            plan->algo = mode == kModePairWide ? CKL_ALGO_UMMA_2CTA_WIDE
                         : mode == kModePair   ? CKL_ALGO_UMMA_2CTA
                         : narrow              ? CKL_ALGO_UMMA_1CTA_N128
                                               : CKL_ALGO_UMMA_1CTA;
        }
    }
    if (algo == CKL_ALGO_AUTO && narrow && plan->sched.sk_tiles > 0) {
        plan->algo = CKL_ALGO_UMMA_1CTA_N128_SK;
    }
    return CKL_OK;
}

// ---- TMA descriptors -----------------------------------------------------------

int encode_2d_uncached(DeviceCtx* ctx, CUtensorMap* map, int dtype, const void* base, uint64_t inner,
                       uint64_t outer, uint64_t pitch_elems, uint32_t box_inner, uint32_t box_outer);

int encode_2d(DeviceCtx* ctx, CUtensorMap* map, int dtype, const void* base, uint64_t inner,
              uint64_t outer, uint64_t pitch_elems, uint32_t box_inner, uint32_t box_outer) {
    const MapKey key = {base, inner, outer, pitch_elems, dtype, box_inner, box_outer};
    std::lock_guard<std::mutex> lock(ctx->mu);
    MapEntry* victim = &ctx->map_cache[0];
    for (MapEntry& e : ctx->map_cache) {
        if (e.stamp != 0 && e.key == key) {
            e.stamp = ++ctx->map_clock;
            *map = e.map;
            return CKL_OK;
        }
        if (e.stamp < victim->stamp) {
            victim = &e;
        }
    }
    if (const int rc = encode_2d_uncached(ctx, map, dtype, base, inner, outer, pitch_elems, box_inner,
                                          box_outer);
        rc != CKL_OK) {
        return rc;
    }
    victim->key = key;
    victim->map = *map;
    victim->stamp = ++ctx->map_clock;
    return CKL_OK;
}

int encode_2d_uncached(DeviceCtx* ctx, CUtensorMap* map, int dtype, const void* base, uint64_t inner,
                       uint64_t outer, uint64_t pitch_elems, uint32_t box_inner, uint32_t box_outer) {
    g_tensor_map_encodes.fetch_add(1, std::memory_order_relaxed);
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {pitch_elems * dtype_size(dtype)};
    const cuuint32_t box[2] = {box_inner, box_outer};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUtensorMapDataType dt = dtype == CKL_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : dtype == CKL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    const CUresult r = ctx->encode(map, dt, 2, const_cast<void*>(base), dims, strides, box,
                                   elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        return fail(CKL_ERR_CUDA,
                    "cuTensorMapEncodeTiled failed with CUresult %d (base=%p dims=%llu x %llu "
                    "pitch=%llu box=%u x %u)",
                    static_cast<int>(r), base, static_cast<unsigned long long>(inner),
                    static_cast<unsigned long long>(outer),
                    static_cast<unsigned long long>(pitch_elems), box_inner, box_outer);
    }
    return CKL_OK;
}

// Stream-K workspace of a stream: [flag words][partial-tile slots].  The flags (one word per
// slot, 32-row group and accumulator half) are zeroed when the buffer is created; every launch
// that uses them gets a fresh non-zero epoch, so they never need clearing between launches.
constexpr size_t kFlagWordsPerSlot = 16;
size_t flag_region_bytes(const DeviceCtx* ctx) {
    const size_t bytes = 2ull * static_cast<size_t>(ctx->sm_count) * kFlagWordsPerSlot * sizeof(unsigned int);
    return (bytes + 255) / 256 * 256;
}

int get_workspace(DeviceCtx* ctx, cudaStream_t stream, size_t bytes, float** slots,
                  unsigned int** flags, unsigned int* epoch) {
    std::lock_guard<std::mutex> lock(ctx->mu);
    Staging& w = ctx->workspace[stream];
    const size_t flag_bytes = flag_region_bytes(ctx);
    const size_t total = flag_bytes + bytes;
    if (w.bytes < total) {
        if (w.ptr != nullptr) {
            CKL_TRY_CUDA(cudaStreamSynchronize(stream));
            CKL_TRY_CUDA(cudaFree(w.ptr));
            w.ptr = nullptr;
            w.bytes = 0;
        }
        CKL_TRY_CUDA(cudaMalloc(&w.ptr, total));
        w.bytes = total;
        w.epoch = 0;
        CKL_TRY_CUDA(cudaMemsetAsync(w.ptr, 0, flag_bytes, stream));
    }
    if (++w.epoch == 0) {
        w.epoch = 1;  // wrapped: zero is the "never written" value (a stale equal epoch would
                      // need 2^32 launches on one stream between two uses of the same slot)
    }
    *flags = static_cast<unsigned int*>(w.ptr);
    *slots = reinterpret_cast<float*>(static_cast<unsigned char*>(w.ptr) + flag_bytes);
    *epoch = w.epoch;
    return CKL_OK;
}

}  // namespace

namespace ckl {

int device_view(DeviceView* out) {
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    out->device = ctx->device;
    out->sm_count = ctx->sm_count;
    out->max_pairs = ctx->max_pairs;
    out->status = ctx->status;
    return CKL_OK;
}

int encode_operand(CUtensorMap* map, int dtype, const void* base, uint64_t inner, uint64_t outer,
                   uint64_t pitch, uint64_t depth, uint64_t stack, uint32_t box_inner,
                   uint32_t box_outer) {
    std::memset(map, 0, sizeof *map);
    if (inner == 0 || outer == 0) {
        return CKL_OK;
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    g_tensor_map_encodes.fetch_add(1, std::memory_order_relaxed);
    const cuuint32_t rank = depth == 0 ? 2 : 3;
    const cuuint64_t dims[3] = {inner, outer, depth};
    const uint64_t bytes = dtype_size(dtype);
    const cuuint64_t strides[2] = {pitch * bytes, stack * bytes};
    const cuuint32_t box[3] = {box_inner, box_outer, 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    const CUresult r = ctx->encode(
        map,
        dtype == CKL_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
        : dtype == CKL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
        rank, const_cast<void*>(base), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
        box_inner * bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        return fail(CKL_ERR_CUDA,
                    "cuTensorMapEncodeTiled failed with CUresult %d (base=%p dims=%llu x %llu x %llu "
                    "pitch=%llu stack=%llu box=%u x %u)",
                    static_cast<int>(r), base, static_cast<unsigned long long>(inner),
                    static_cast<unsigned long long>(outer), static_cast<unsigned long long>(depth),
                    static_cast<unsigned long long>(pitch), static_cast<unsigned long long>(stack),
                    box_inner, box_outer);
    }
    return CKL_OK;
}

int take_wait_fault(unsigned long long* limit_ns) {
    const WaitFault fault = g_wait_fault;
    g_wait_fault = WaitFault{};
    *limit_ns = fault.limit_ns;
    return fault.kind;
}

}  // namespace ckl

namespace {

// ---- launches --------------------------------------------------------------------

template <int kMode, typename OutT>
int launch_umma(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                const GemmParams& p, int grid, cudaStream_t stream) {
    using Cfg = UmmaConfig<kMode>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    unsigned num_attrs = 0;
    if (Cfg::kPair) {
        attrs[num_attrs].id = cudaLaunchAttributeClusterDimension;
        attrs[num_attrs].val.clusterDim.x = 2;
        attrs[num_attrs].val.clusterDim.y = 1;
        attrs[num_attrs].val.clusterDim.z = 1;
        ++num_attrs;
    }
    cfg.attrs = attrs;
    cfg.numAttrs = num_attrs;
    if (p.sched.sk_tiles > 0 && p.sk_flags != nullptr) {
        // Fused stream-K: CTAs of this launch wait for partials of other CTAs, so the whole
        // grid must be resident at once: cooperative launch.  If the device cannot promise
        // that, fall through to the two-kernel form, where nobody waits for anybody.
        attrs[num_attrs].id = cudaLaunchAttributeCooperative;
        attrs[num_attrs].val.cooperative = 1;
        cfg.numAttrs = num_attrs + 1;
        if (cudaLaunchKernelEx(&cfg, umma_gemm_kernel<kMode, OutT>, ta, tb, tc, p) == cudaSuccess) {
            return CKL_OK;
        }
        (void)cudaGetLastError();
        cfg.numAttrs = num_attrs;
    }
    GemmParams q = p;
    q.sk_flags = nullptr;
    // Programmatic dependent launch: the prologue (barriers, tensor memory) may overlap the
    // tail of the previous kernel in the stream; the kernel waits for that kernel before it
    // touches global memory.  Ordinary stream order for anything that is not such a kernel.
    attrs[num_attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[num_attrs].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = num_attrs + 1;
    CKL_TRY_CUDA(cudaLaunchKernelEx(&cfg, umma_gemm_kernel<kMode, OutT>, ta, tb, tc, q));
    if (q.sched.sk_tiles > 0) {
        // ordinary launch: as a programmatic dependent it measured slower (1024x1024x32768)
        streamk_fixup_kernel<Cfg::kTileM, Cfg::kTileN, OutT>
            <<<dim3(static_cast<unsigned>(q.sched.sk_tiles), Cfg::kTileM / 32 * Cfg::kNHalves), 256, 0,
               stream>>>(q);
        CKL_TRY_CUDA(cudaGetLastError());
    }
    return CKL_OK;
}

template <typename OutT>
int launch_umma_out(int mode, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                    const GemmParams& p, int grid, cudaStream_t stream) {
    switch (mode) {
        case kModePair: return launch_umma<kModePair, OutT>(ta, tb, tc, p, grid, stream);
        case kModePairWide: return launch_umma<kModePairWide, OutT>(ta, tb, tc, p, grid, stream);
        default: return launch_umma<kModeSingle, OutT>(ta, tb, tc, p, grid, stream);
    }
}

template <typename InT, typename OutT>
int launch_simt(const void* a, const void* b, void* c, const float* bias, int m, int n, int k,
                int lda, int ldb, int ldc, float alpha, float beta, int epi, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>((m + 63) / 64));
    simt_gemm_kernel<InT, OutT><<<grid, 256, 0, stream>>>(
        static_cast<const InT*>(a), static_cast<const InT*>(b), static_cast<OutT*>(c), bias, m, n, k,
        lda, ldb, ldc, alpha, beta, epi);
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}

template <typename InT>
int launch_simt_in(int c_dtype, const void* a, const void* b, void* c, const float* bias, int m,
                   int n, int k, int lda, int ldb, int ldc, float alpha, float beta, int epi,
                   cudaStream_t stream) {
    switch (c_dtype) {
        case CKL_F32:
            return launch_simt<InT, float>(a, b, c, bias, m, n, k, lda, ldb, ldc, alpha, beta, epi,
                                           stream);
        case CKL_F16:
            return launch_simt<InT, __half>(a, b, c, bias, m, n, k, lda, ldb, ldc, alpha, beta, epi,
                                            stream);
        default:
            return launch_simt<InT, __nv_bfloat16>(a, b, c, bias, m, n, k, lda, ldb, ldc, alpha,
                                                   beta, epi, stream);
    }
}

template <typename OutT>
int launch_scale(void* c, const float* bias, int m, int n, int ldc, float beta, int epi,
                 cudaStream_t stream) {
    const long long total = static_cast<long long>(m) * n;
    const int blocks = static_cast<int>(std::min<long long>((total + 255) / 256, 148LL * 16));
    scale_c_kernel<OutT><<<blocks, 256, 0, stream>>>(static_cast<OutT*>(c), bias, m, n, ldc, beta,
                                                     epi);
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}

template <typename T, bool kDstAligned>
void launch_copy_rows(const DeviceCtx* ctx, void* dst, const void* src, int rows, int cols, int src_ld,
                      size_t dst_ld, cudaStream_t stream) {
    constexpr size_t kPer = 16 / sizeof(T);
    const size_t groups = (static_cast<size_t>(cols) + kPer - 1) / kPer * static_cast<size_t>(rows);
    const int blocks = static_cast<int>(
        std::max<size_t>(1, std::min<size_t>((groups + 255) / 256, static_cast<size_t>(ctx->sm_count) * 16)));
    copy_rows_kernel<T, kDstAligned><<<blocks, 256, 0, stream>>>(
        static_cast<T*>(dst), static_cast<const T*>(src), rows, cols, static_cast<size_t>(src_ld), dst_ld);
}

int gemm_impl(int ab_dtype, const void* a, const void* b, void* c, int c_dtype, const float* bias,
              int m, int n, int k, int lda, int ldb, int ldc, float alpha, float beta, int epi,
              int algo, cudaStream_t stream) {
    if (ab_dtype != CKL_F16 && ab_dtype != CKL_BF16) {
        return fail(CKL_ERR_INVALID_ARG, "A/B dtype must be CKL_F16 or CKL_BF16 (got %d)", ab_dtype);
    }
    if (c_dtype != CKL_F32 && c_dtype != CKL_F16 && c_dtype != CKL_BF16) {
        return fail(CKL_ERR_INVALID_ARG, "C dtype must be CKL_F32, CKL_F16 or CKL_BF16 (got %d)",
                    c_dtype);
    }
    if (algo < CKL_ALGO_AUTO || algo > kLastAlgo) {
        return fail(CKL_ERR_INVALID_ARG, "unknown algo %d", algo);
    }
    if (m <= 0 || n <= 0) {
        return CKL_OK;  // nothing to write (reference: wmma_gemm.cuh:145-147)
    }
    if (c == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "C is null");
    }
    if (ldc < n) {
        return fail(CKL_ERR_INVALID_ARG, "ldc=%d is smaller than n=%d", ldc, n);
    }
    if (epi == kEpiBiasRelu && bias == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "bias is null");
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    if (k <= 0) {
        switch (c_dtype) {
            case CKL_F32: return launch_scale<float>(c, bias, m, n, ldc, beta, epi, stream);
            case CKL_F16: return launch_scale<__half>(c, bias, m, n, ldc, beta, epi, stream);
            default: return launch_scale<__nv_bfloat16>(c, bias, m, n, ldc, beta, epi, stream);
        }
    }
    if (a == nullptr || b == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "A or B is null");
    }
    if (lda < k || ldb < n) {
        return fail(CKL_ERR_INVALID_ARG, "lda=%d < k=%d or ldb=%d < n=%d", lda, k, ldb, n);
    }
    Plan plan;
    const size_t a_align = reinterpret_cast<uintptr_t>(a) % 16 == 0 ? 16 : 2;
    const size_t b_align = reinterpret_cast<uintptr_t>(b) % 16 == 0 ? 16 : 2;
    const int c_traffic = static_cast<int>(dtype_size(c_dtype)) *
                          ((epi == kEpiLinear && beta != 0.0f) ? 2 : 1);
    if (const int rc = make_plan(m, n, k, lda, ldb, a_align, b_align, algo, ctx->sm_count,
                                 ctx->max_pairs, c_traffic, &plan);
        rc != CKL_OK) {
        return rc;
    }
    export_plan(plan, &g_last_plan);
    if (plan.algo == CKL_ALGO_SIMT) {
        return ab_dtype == CKL_F16
                   ? launch_simt_in<__half>(c_dtype, a, b, c, bias, m, n, k, lda, ldb, ldc, alpha,
                                            beta, epi, stream)
                   : launch_simt_in<__nv_bfloat16>(c_dtype, a, b, c, bias, m, n, k, lda, ldb, ldc,
                                                   alpha, beta, epi, stream);
    }

    // Operands TMA cannot describe travel through aligned copies in this stream's scratch
    // (grown on demand, reused by later calls on the stream: stream order keeps a later copy
    // from overwriting what an earlier GEMM still reads).  The same goes for a C whose base, pitch
    // or last column rules out 16-byte accesses on a large problem: the kernel writes an aligned copy
    // through its TMA epilogue and one pass copies it out, instead of the register-store
    // epilogue's 2-byte stores (C_in is copied in first when it is read).
    const size_t csz = dtype_size(c_dtype);
    // A TMA store writes whole 16-byte units: columns that end inside one would take up to 7 columns
    // of a wider matrix along.
    const bool whole_units = (static_cast<size_t>(n) * csz) % 16 == 0;
    const bool c_aligned = whole_units && reinterpret_cast<uintptr_t>(c) % 16 == 0 &&
                           (static_cast<size_t>(ldc) * csz) % 16 == 0;
    const bool stage_c = algo == CKL_ALGO_AUTO && !c_aligned &&
                         static_cast<long long>(m) * n * static_cast<long long>(k) >= kRepackMinMacs;
    void* c_user = c;
    const int ldc_user = ldc;
    if (stage_c) {
        g_last_plan.repack = 1;
    }
    if (plan.repack || stage_c) {
        const bool fix_a = reinterpret_cast<uintptr_t>(a) % 16 != 0 || lda % 8 != 0;
        const bool fix_b = reinterpret_cast<uintptr_t>(b) % 16 != 0 || ldb % 8 != 0;
        const size_t pitch_a = (static_cast<size_t>(k) + 63) / 64 * 64;   // 128-byte rows
        const size_t pitch_b = (static_cast<size_t>(n) + 63) / 64 * 64;
        const size_t per_line = 128 / csz;
        const size_t pitch_c = (static_cast<size_t>(n) + per_line - 1) / per_line * per_line;
        const size_t bytes_a = fix_a ? static_cast<size_t>(m) * pitch_a * 2 : 0;
        const size_t bytes_b = fix_b ? static_cast<size_t>(k) * pitch_b * 2 : 0;
        const size_t bytes_c = stage_c ? static_cast<size_t>(m) * pitch_c * csz : 0;
        unsigned char* scratch = nullptr;
        {
            std::lock_guard<std::mutex> lock(ctx->mu);
            Staging& buf = ctx->repack[stream];
            if (buf.bytes < bytes_a + bytes_b + bytes_c) {
                if (buf.ptr != nullptr) {
                    CKL_TRY_CUDA(cudaStreamSynchronize(stream));
                    CKL_TRY_CUDA(cudaFree(buf.ptr));
                    buf.ptr = nullptr;
                    buf.bytes = 0;
                }
                CKL_TRY_CUDA(cudaMalloc(&buf.ptr, bytes_a + bytes_b + bytes_c));
                buf.bytes = bytes_a + bytes_b + bytes_c;
            }
            scratch = static_cast<unsigned char*>(buf.ptr);
        }
        if (fix_a) {
            launch_copy_rows<uint16_t, true>(ctx, scratch, a, m, k, lda, pitch_a, stream);
            a = scratch;
            lda = static_cast<int>(pitch_a);
        }
        if (fix_b) {
            launch_copy_rows<uint16_t, true>(ctx, scratch + bytes_a, b, k, n, ldb, pitch_b, stream);
            b = scratch + bytes_a;
            ldb = static_cast<int>(pitch_b);
        }
        if (stage_c) {
            unsigned char* c_copy = scratch + bytes_a + bytes_b;
            if (epi == kEpiLinear && beta != 0.0f) {
                if (csz == 4) {
                    launch_copy_rows<uint32_t, true>(ctx, c_copy, c, m, n, ldc, pitch_c, stream);
                } else {
                    launch_copy_rows<uint16_t, true>(ctx, c_copy, c, m, n, ldc, pitch_c, stream);
                }
            }
            c = c_copy;
            ldc = static_cast<int>(pitch_c);
        }
        CKL_TRY_CUDA(cudaGetLastError());
    }

    CUtensorMap ta, tb;
    if (const int rc = encode_2d(ctx, &ta, ab_dtype, a, static_cast<uint64_t>(k),
                                 static_cast<uint64_t>(m), static_cast<uint64_t>(lda), 64, 128);
        rc != CKL_OK) {
        return rc;
    }
    if (const int rc = encode_2d(ctx, &tb, ab_dtype, b, static_cast<uint64_t>(n),
                                 static_cast<uint64_t>(k), static_cast<uint64_t>(ldb), 64, 64);
        rc != CKL_OK) {
        return rc;
    }
    GemmParams p = {};
    p.c = c;
    p.bias = bias;
    p.workspace = nullptr;
    p.status = ctx->status;
    p.m = m;
    p.n = n;
    p.k = k;
    p.ldc = ldc;
    p.alpha = alpha;
    p.beta = beta;
    p.c_vec = (reinterpret_cast<uintptr_t>(c) % 16 == 0 && (static_cast<size_t>(ldc) * csz) % 16 == 0)
                  ? 1
                  : 0;
    p.epi_mode = epi;
    // The coalesced epilogue moves C through TMA (32-row x 128-byte boxes); it needs the
    // same alignment as the vector path, and rows that end with a unit or in a copy, whose padding is
    // nobody's.  Otherwise the kernel stores from registers.
    CUtensorMap tc;
    std::memset(&tc, 0, sizeof tc);
    p.c_tma = p.c_vec != 0 && (whole_units || stage_c) ? 1 : 0;
    if (p.c_tma) {
        if (const int rc = encode_2d(ctx, &tc, c_dtype, c, static_cast<uint64_t>(n),
                                     static_cast<uint64_t>(m), static_cast<uint64_t>(ldc),
                                     static_cast<uint32_t>(128 / csz), 32);
            rc != CKL_OK) {
            return rc;
        }
    }
    p.tile_n = plan.tile_n == 128 ? 128 : 0;
    p.idesc = ptx::make_idesc_f16(ab_dtype == CKL_F16 ? 0u : 1u, 0u, 1u, plan.pair ? 256u : 128u,
                                  plan.tile_n == 128 ? 128u : 256u);
    p.sched = plan.sched;
    p.wait_limit_ns = kWaitLimitNs;
    const WaitFault fault = g_wait_fault;
    g_wait_fault = WaitFault{};  // one launch only
    if (fault.kind != 0) {
        p.wait_limit_ns = fault.limit_ns != 0 ? fault.limit_ns : kWaitLimitNs;
        p.overstate_first_stage = fault.kind == 1 ? 1 : 0;
        p.sk_flag_skew = fault.kind == 2 ? 1u : 0u;
    }
    if (plan.workspace_bytes > 0) {
        unsigned int* flags = nullptr;
        unsigned int epoch = 0;
        if (const int rc = get_workspace(ctx, stream, plan.workspace_bytes, &p.workspace, &flags, &epoch);
            rc != CKL_OK) {
            return rc;
        }
        // CKL_STREAMK_FIXUP=pass keeps the separate fix-up kernel (for comparisons).
        static const bool two_pass = [] {
            const char* v = std::getenv("CKL_STREAMK_FIXUP");
            return v != nullptr && std::strcmp(v, "pass") == 0;
        }();
        // Fused where every unit has whole tiles left after its stream-K range, so the
        // reduction hides behind them; a launch that is all stream-K ends with the reduction
        // either way, and there the fix-up pass, spread over the whole GPU, measured faster.
        // Not while the stream is being captured: a replayed graph would carry the same epoch
        // every time, and the flags of the previous replay would pass for this one's.
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(stream, &capture) != cudaSuccess) {
            (void)cudaGetLastError();
            capture = cudaStreamCaptureStatusActive;  // unknown: take the form that needs no epoch
        }
        if (!two_pass && plan.sched.dp_tiles >= plan.sched.units &&
            capture == cudaStreamCaptureStatusNone) {
            p.sk_flags = flags;
            p.sk_epoch = epoch;
        }
    }
    int rc = CKL_OK;
    switch (c_dtype) {
        case CKL_F32: rc = launch_umma_out<float>(plan.mode, ta, tb, tc, p, plan.grid, stream); break;
        case CKL_F16: rc = launch_umma_out<__half>(plan.mode, ta, tb, tc, p, plan.grid, stream); break;
        default: rc = launch_umma_out<__nv_bfloat16>(plan.mode, ta, tb, tc, p, plan.grid, stream); break;
    }
    if (rc == CKL_OK && stage_c) {
        // the aligned copy of C goes to the caller's matrix
        if (csz == 4) {
            launch_copy_rows<uint32_t, false>(ctx, c_user, c, m, n, ldc, static_cast<size_t>(ldc_user), stream);
        } else {
            launch_copy_rows<uint16_t, false>(ctx, c_user, c, m, n, ldc, static_cast<size_t>(ldc_user), stream);
        }
        CKL_TRY_CUDA(cudaGetLastError());
    }
    return rc;
}

int ensure_staging(Staging* s, size_t bytes) {
    if (s->bytes >= bytes) {
        return CKL_OK;
    }
    if (s->ptr != nullptr) {
        CKL_TRY_CUDA(cudaFree(s->ptr));
        s->ptr = nullptr;
        s->bytes = 0;
    }
    CKL_TRY_CUDA(cudaMalloc(&s->ptr, bytes));
    s->bytes = bytes;
    return CKL_OK;
}

}  // namespace

extern "C" {

int ckl_gemm_ex(int ab_dtype, const void* a, const void* b, void* c, int c_dtype, int m, int n,
                int k, int lda, int ldb, int ldc, float alpha, float beta, int algo,
                ckl_stream_t stream) {
    return gemm_impl(ab_dtype, a, b, c, c_dtype, nullptr, m, n, k, lda, ldb, ldc, alpha, beta,
                     kEpiLinear, algo, static_cast<cudaStream_t>(stream));
}

int ckl_gemm_f16(const void* a, const void* b, void* c, int c_dtype, int m, int n, int k, int lda,
                 int ldb, int ldc, float alpha, float beta, ckl_stream_t stream) {
    return ckl_gemm_ex(CKL_F16, a, b, c, c_dtype, m, n, k, lda, ldb, ldc, alpha, beta,
                       CKL_ALGO_AUTO, stream);
}

int ckl_gemm_bf16(const void* a, const void* b, void* c, int c_dtype, int m, int n, int k, int lda,
                  int ldb, int ldc, float alpha, float beta, ckl_stream_t stream) {
    return ckl_gemm_ex(CKL_BF16, a, b, c, c_dtype, m, n, k, lda, ldb, ldc, alpha, beta,
                       CKL_ALGO_AUTO, stream);
}

int ckl_gemm_bias_relu_ex(int ab_dtype, const void* a, const void* b, void* c, int c_dtype,
                          const float* bias, int m, int n, int k, int lda, int ldb, int ldc,
                          float alpha, int algo, ckl_stream_t stream) {
    return gemm_impl(ab_dtype, a, b, c, c_dtype, bias, m, n, k, lda, ldb, ldc, alpha, 0.0f,
                     kEpiBiasRelu, algo, static_cast<cudaStream_t>(stream));
}

int ckl_bias_relu_f32(float* c, const float* bias, int m, int n, int ldc, ckl_stream_t stream) {
    if (m <= 0 || n <= 0) {
        return CKL_OK;
    }
    if (c == nullptr || bias == nullptr || ldc < n) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_bias_relu_f32: null pointer or ldc < n");
    }
    const long long total = static_cast<long long>(m) * n;
    const bool vec = n % 4 == 0 && ldc % 4 == 0 && reinterpret_cast<uintptr_t>(c) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(bias) % 16 == 0;
    if (vec) {
        const int blocks = static_cast<int>(std::min<long long>((total / 4 + 255) / 256, 148LL * 16));
        bias_relu_vec4_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
            reinterpret_cast<float4*>(c), reinterpret_cast<const float4*>(bias), m, n / 4, ldc / 4);
    } else {
        const int blocks = static_cast<int>(std::min<long long>((total + 255) / 256, 148LL * 16));
        bias_relu_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(c, bias, m, n, ldc);
    }
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}

int ckl_sgemm(const float* a, const float* b, float* c, int m, int n, int k, int lda, int ldb,
              int ldc, float alpha, float beta, ckl_stream_t stream) {
    if (m <= 0 || n <= 0) {
        return CKL_OK;  // nothing to write
    }
    if (c == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_sgemm: C is null");
    }
    if (ldc < n) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_sgemm: ldc=%d is smaller than n=%d", ldc, n);
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (k <= 0) {
        return launch_scale<float>(c, nullptr, m, n, ldc, beta, kEpiLinear, s);  // C = beta * C
    }
    if (a == nullptr || b == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_sgemm: A or B is null");
    }
    if (lda < k || ldb < n) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_sgemm: lda=%d < k=%d or ldb=%d < n=%d", lda, k, ldb, n);
    }
    // 128 x 128 tiles unless they would leave most of the SMs idle (two CTAs fit on an SM).
    const long long large_tiles = ((static_cast<long long>(m) + 127) / 128) * ((static_cast<long long>(n) + 127) / 128);
    const int tile = large_tiles >= ctx->sm_count ? fp32::kTileLarge : fp32::kTileSmall;
    const long long tiles_m = (static_cast<long long>(m) + tile - 1) / tile;
    const long long tiles_n = (static_cast<long long>(n) + tile - 1) / tile;
    if (tiles_m > 65535) {
        return fail(CKL_ERR_TOO_LARGE, "ckl_sgemm: m=%d needs more than 65535 tile rows", m);
    }
    const dim3 grid(static_cast<unsigned>(tiles_n), static_cast<unsigned>(tiles_m));
    const bool vec = reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(b) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(c) % 16 == 0 && lda % 4 == 0 && ldb % 4 == 0 &&
                     ldc % 4 == 0;
    if (tile == fp32::kTileLarge) {
        if (vec) {
            sgemm_kernel<true, 128><<<grid, fp32::kThreads, 0, s>>>(a, b, c, m, n, k, lda, ldb, ldc, alpha, beta);
        } else {
            sgemm_kernel<false, 128><<<grid, fp32::kThreads, 0, s>>>(a, b, c, m, n, k, lda, ldb, ldc, alpha, beta);
        }
    } else {
        if (vec) {
            sgemm_kernel<true, 64><<<grid, fp32::kThreads, 0, s>>>(a, b, c, m, n, k, lda, ldb, ldc, alpha, beta);
        } else {
            sgemm_kernel<false, 64><<<grid, fp32::kThreads, 0, s>>>(a, b, c, m, n, k, lda, ldb, ldc, alpha, beta);
        }
    }
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}

int ckl_strsm_lower(const float* l, float* b, int m, int n, int lda, int ldb, float alpha,
                    ckl_stream_t stream) {
    if (m <= 0 || n <= 0) {
        return CKL_OK;  // reference: src/trsm/trsm_blocked.cu:65-67
    }
    if (l == nullptr || b == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_strsm_lower: L or B is null");
    }
    if (lda < m || ldb < n) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_strsm_lower: lda=%d < m=%d or ldb=%d < n=%d", lda, m, ldb, n);
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (alpha != 1.0f) {
        // L X = alpha B is linear in B: scale once, then solve with alpha = 1
        if (const int rc = launch_scale<float>(b, nullptr, m, n, ldb, alpha, kEpiLinear, s); rc != CKL_OK) {
            return rc;
        }
    }
    const unsigned col_blocks = static_cast<unsigned>((n + kTrsmThreads - 1) / kTrsmThreads);
    // Recursive halving, written as an explicit stack of (first row, rows, stage) so that no
    // recursion depth depends on m.  stage 0: split or solve; stage 1: the upper half is solved,
    // update the lower half with one GEMM and descend into it.
    struct Frame {
        int r0, rows, stage;
    };
    std::vector<Frame> stack;
    stack.push_back({0, m, 0});
    while (!stack.empty()) {
        const Frame f = stack.back();
        stack.pop_back();
        if (f.rows <= kTrsmBlock) {
            trsm_diag_block_kernel<<<col_blocks, kTrsmThreads, 0, s>>>(l, b, n, lda, ldb, f.r0, f.rows);
            CKL_TRY_CUDA(cudaGetLastError());
            continue;
        }
        // upper half: a multiple of the block size, so diagonal blocks stay aligned
        const int up = ((f.rows / 2 + kTrsmBlock - 1) / kTrsmBlock) * kTrsmBlock;
        if (f.stage == 0) {
            stack.push_back({f.r0, f.rows, 1});
            stack.push_back({f.r0, up, 0});
            continue;
        }
        // B[r0+up : r0+rows, :] -= L[r0+up : r0+rows, r0 : r0+up] * X[r0 : r0+up, :]
        const float* l_low = l + static_cast<size_t>(f.r0 + up) * lda + f.r0;
        const float* x_up = b + static_cast<size_t>(f.r0) * ldb;
        float* b_low = b + static_cast<size_t>(f.r0 + up) * ldb;
        if (const int rc = ckl_sgemm(l_low, x_up, b_low, f.rows - up, n, up, lda, ldb, ldb, -1.0f, 1.0f,
                                     stream);
            rc != CKL_OK) {
            return rc;
        }
        stack.push_back({f.r0 + up, f.rows - up, 0});
    }
    return CKL_OK;
}

int ckl_gemm_host(int ab_dtype, const void* a_host, const void* b_host, void* c_host, int c_dtype,
                  int m, int n, int k, float alpha, float beta) {
    if (m <= 0 || n <= 0) {
        return CKL_OK;
    }
    if (c_host == nullptr || (k > 0 && (a_host == nullptr || b_host == nullptr))) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_gemm_host: null host pointer");
    }
    if (c_dtype != CKL_F32 && c_dtype != CKL_F16 && c_dtype != CKL_BF16) {
        return fail(CKL_ERR_INVALID_ARG, "C dtype must be CKL_F32, CKL_F16 or CKL_BF16");
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    std::lock_guard<std::mutex> one_call(ctx->host_mu);  // the staging buffers are shared
    std::unique_lock<std::mutex> lock(ctx->mu);
    if (ctx->host_stream == nullptr) {
        CKL_TRY_CUDA(cudaStreamCreateWithFlags(&ctx->host_stream, cudaStreamNonBlocking));
        CKL_TRY_CUDA(cudaStreamCreateWithFlags(&ctx->host_in, cudaStreamNonBlocking));
        CKL_TRY_CUDA(cudaStreamCreateWithFlags(&ctx->host_out, cudaStreamNonBlocking));
        for (cudaEvent_t& e : ctx->host_events) {
            CKL_TRY_CUDA(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
        }
    }
    const size_t kk = static_cast<size_t>(std::max(k, 0));
    const size_t csz = dtype_size(c_dtype);
    const size_t a_bytes = static_cast<size_t>(m) * kk * 2;
    const size_t b_bytes = kk * n * 2;
    const size_t c_bytes = static_cast<size_t>(m) * n * csz;
    if (int rc = ensure_staging(&ctx->host_a, std::max<size_t>(a_bytes, 16)); rc != CKL_OK) return rc;
    if (int rc = ensure_staging(&ctx->host_b, std::max<size_t>(b_bytes, 16)); rc != CKL_OK) return rc;
    if (int rc = ensure_staging(&ctx->host_c, c_bytes); rc != CKL_OK) return rc;
    // The call is bound by the host link, which carries both directions at once: B goes up
    // first, then A and C travel in row panels, and panel i is multiplied and sent back while
    // panel i+1 is still on its way up.  Three streams (up, compute, down) chained by events.
    constexpr int kMaxPanels = DeviceCtx::kHostPanels;
    const int panels = std::max(1, std::min(kMaxPanels, m / 1024));
    const int rows_per_panel = ((m + panels - 1) / panels + 255) / 256 * 256;
    cudaStream_t s_in = ctx->host_in, s = ctx->host_stream, s_out = ctx->host_out;
    if (b_bytes > 0) {
        CKL_TRY_CUDA(cudaMemcpyAsync(ctx->host_b.ptr, b_host, b_bytes, cudaMemcpyHostToDevice, s_in));
    }
    auto* dev_a = static_cast<unsigned char*>(ctx->host_a.ptr);
    auto* dev_c = static_cast<unsigned char*>(ctx->host_c.ptr);
    const auto* src_a = static_cast<const unsigned char*>(a_host);
    auto* host_c = static_cast<unsigned char*>(c_host);
    void* dev_b = ctx->host_b.ptr;
    // gemm_impl takes ctx->mu inside get_workspace; release ours while it runs.
    lock.unlock();
    int rc = CKL_OK;
    auto cuda_ok = [&rc](cudaError_t e, const char* what) {
        if (e != cudaSuccess && rc == CKL_OK) {
            rc = fail(CKL_ERR_CUDA, "ckl_gemm_host: %s failed: %s", what, cudaGetErrorString(e));
        }
        return rc == CKL_OK;
    };
    int used = 0;
    for (int row0 = 0; row0 < m && rc == CKL_OK; row0 += rows_per_panel, ++used) {
        const int rows = std::min(rows_per_panel, m - row0);
        const size_t a_off = static_cast<size_t>(row0) * kk * 2;
        const size_t c_off = static_cast<size_t>(row0) * n * csz;
        const size_t c_panel = static_cast<size_t>(rows) * n * csz;
        cudaEvent_t up = ctx->host_events[2 * used], done = ctx->host_events[2 * used + 1];
        if (kk > 0 && !cuda_ok(cudaMemcpyAsync(dev_a + a_off, src_a + a_off, static_cast<size_t>(rows) * kk * 2,
                                               cudaMemcpyHostToDevice, s_in), "copy of A")) {
            break;
        }
        if (beta != 0.0f && !cuda_ok(cudaMemcpyAsync(dev_c + c_off, host_c + c_off, c_panel,
                                                     cudaMemcpyHostToDevice, s_in), "copy of C")) {
            break;
        }
        if (!cuda_ok(cudaEventRecord(up, s_in), "event record") ||
            !cuda_ok(cudaStreamWaitEvent(s, up, 0), "stream wait")) {
            break;
        }
        rc = gemm_impl(ab_dtype, dev_a + a_off, dev_b, dev_c + c_off, c_dtype, nullptr, rows, n, k, k, n, n,
                       alpha, beta, kEpiLinear, CKL_ALGO_AUTO, s);
        if (rc != CKL_OK) {
            break;
        }
        if (!cuda_ok(cudaEventRecord(done, s), "event record") ||
            !cuda_ok(cudaStreamWaitEvent(s_out, done, 0), "stream wait") ||
            !cuda_ok(cudaMemcpyAsync(host_c + c_off, dev_c + c_off, c_panel, cudaMemcpyDeviceToHost, s_out),
                     "copy of the result")) {
            break;
        }
    }
    // Nothing of this call may still be in flight when it returns, whatever happened above.
    const cudaError_t e_in = cudaStreamSynchronize(s_in);
    const cudaError_t e_run = cudaStreamSynchronize(s);
    const cudaError_t e_out = cudaStreamSynchronize(s_out);
    if (rc != CKL_OK) {
        return rc;
    }
    CKL_TRY_CUDA(e_in);
    CKL_TRY_CUDA(e_run);
    CKL_TRY_CUDA(e_out);
    return CKL_OK;
}

int ckl_plan_gemm_ex(int m, int n, int k, int lda, int ldb, int ldc, int a_align, int b_align,
                     int algo, int sm_count, int max_pairs, int c_dtype, int c_is_read,
                     ckl_plan* out) {
    if (out == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_plan_gemm: out is null");
    }
    std::memset(out, 0, sizeof *out);
    if (c_dtype != CKL_F32 && c_dtype != CKL_F16 && c_dtype != CKL_BF16) {
        return fail(CKL_ERR_INVALID_ARG, "C dtype must be CKL_F32, CKL_F16 or CKL_BF16 (got %d)", c_dtype);
    }
    if (m <= 0 || n <= 0 || k <= 0) {
        out->algo = CKL_ALGO_SIMT;  // degenerate: no tiles (k <= 0 runs the scale kernel)
        return CKL_OK;
    }
    if (lda < k || ldb < n || ldc < n) {
        return fail(CKL_ERR_INVALID_ARG, "leading dimension smaller than the row length");
    }
    Plan plan;
    const int c_traffic = static_cast<int>(dtype_size(c_dtype)) * (c_is_read ? 2 : 1);
    if (const int rc = make_plan(m, n, k, lda, ldb, static_cast<size_t>(a_align),
                                 static_cast<size_t>(b_align), algo, sm_count,
                                 max_pairs > 0 ? max_pairs : sm_count / 2, c_traffic, &plan);
        rc != CKL_OK) {
        return rc;
    }
    export_plan(plan, out);
    return CKL_OK;
}

int ckl_plan_gemm(int m, int n, int k, int lda, int ldb, int ldc, int a_align, int b_align,
                  int algo, int sm_count, ckl_plan* out) {
    return ckl_plan_gemm_ex(m, n, k, lda, ldb, ldc, a_align, b_align, algo, sm_count, 0, CKL_BF16, 0, out);
}

int ckl_last_plan(ckl_plan* out) {
    if (out == nullptr) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_last_plan: out is null");
    }
    *out = g_last_plan;
    return CKL_OK;
}

int ckl_test_arm_wait_fault(int kind, unsigned long long wait_limit_ns) {
    if (kind < 0 || kind > 2) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_test_arm_wait_fault: kind must be 0, 1 or 2");
    }
    g_wait_fault.kind = kind;
    g_wait_fault.limit_ns = wait_limit_ns;
    return CKL_OK;
}

unsigned long long ckl_debug_counter(const char* name) {
    if (name != nullptr && std::strcmp(name, "tensor_map_encodes") == 0) {
        return g_tensor_map_encodes.load(std::memory_order_relaxed);
    }
    return ~0ull;
}

int ckl_plan_sk_range(const ckl_plan* plan, int u, long long* begin, long long* end) {
    if (plan == nullptr || begin == nullptr || end == nullptr || plan->sk_units <= 0 || u < 0 ||
        u >= plan->sk_units) {
        return fail(CKL_ERR_INVALID_ARG, "ckl_plan_sk_range: bad plan or unit index");
    }
    Schedule s = {};
    s.units = plan->sk_units;
    s.sk_iters = plan->sk_iters;
    *begin = sk_range_begin(s, u);
    *end = sk_range_begin(s, u + 1);
    return CKL_OK;
}

namespace {
Schedule schedule_of(const ckl_plan* plan) {
    Schedule s = {};
    s.tiles_m = plan->tiles_m;
    s.tiles_n = plan->tiles_n;
    s.k_blocks = plan->k_blocks;
    s.units = plan->units;
    s.dp_tiles = plan->dp_tiles;
    s.sk_tiles = plan->sk_tiles;
    s.group_m = plan->group_m;
    s.sk_iters = plan->sk_iters;
    return s;
}
}  // namespace

int ckl_plan_unit_segments(const ckl_plan* plan, int u, int* out, int max_segments) {
    if (plan == nullptr || u < 0 || u >= plan->units || plan->group_m <= 0 ||
        (out == nullptr && max_segments > 0)) {
        fail(CKL_ERR_INVALID_ARG, "ckl_plan_unit_segments: bad plan or unit index");
        return -CKL_ERR_INVALID_ARG;
    }
    const Schedule s = schedule_of(plan);
    SegmentCursor cur = make_cursor(s, u);
    Segment seg;
    int count = 0;
    while (next_segment(s, &cur, &seg)) {
        if (count < max_segments) {
            int tm = 0, tn = 0;
            tile_coords(s, seg.tile, &tm, &tn);
            int* o = out + 6 * count;
            o[0] = seg.tile;
            o[1] = tm;
            o[2] = tn;
            o[3] = seg.kb_begin;
            o[4] = seg.kb_end;
            o[5] = seg.slot;
        }
        ++count;
    }
    return count;
}

int ckl_plan_fixup_slots(const ckl_plan* plan, int sk_tile, int* out, int max_slots) {
    if (plan == nullptr || sk_tile < 0 || sk_tile >= plan->sk_tiles ||
        (out == nullptr && max_slots > 0)) {
        fail(CKL_ERR_INVALID_ARG, "ckl_plan_fixup_slots: bad plan or tile index");
        return -CKL_ERR_INVALID_ARG;
    }
    const Schedule s = schedule_of(plan);
    int slots[kMaxFixupSlots];
    const int count = fixup_slots(s, sk_tile, slots, kMaxFixupSlots);
    for (int i = 0; i < count && i < max_slots; ++i) {
        out[i] = slots[i];
    }
    return count;
}

int ckl_assemble_column_blocks(void* dst, const void* src, int elem_size, int m, int n_shard,
                               int parts, ckl_stream_t stream) {
    if (m <= 0 || n_shard <= 0 || parts <= 0) {
        return CKL_OK;
    }
    if (dst == nullptr || src == nullptr || (elem_size != 2 && elem_size != 4)) {
        return fail(CKL_ERR_INVALID_ARG,
                    "ckl_assemble_column_blocks: null pointer or elem_size not 2 or 4");
    }
    const size_t row_bytes = static_cast<size_t>(n_shard) * static_cast<size_t>(elem_size);
    const bool vec = row_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(dst) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(src) % 16 == 0;
    const size_t unit = vec ? 16 : static_cast<size_t>(elem_size);
    const size_t per_row = row_bytes / unit;
    const size_t total = per_row * static_cast<size_t>(m) * static_cast<size_t>(parts);
    const int blocks = static_cast<int>(std::min<size_t>((total + 255) / 256, 148 * 32));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (vec) {
        assemble_column_blocks_kernel<uint4><<<blocks, 256, 0, s>>>(
            static_cast<uint4*>(dst), static_cast<const uint4*>(src), per_row, m, parts);
    } else if (elem_size == 4) {
        assemble_column_blocks_kernel<uint32_t><<<blocks, 256, 0, s>>>(
            static_cast<uint32_t*>(dst), static_cast<const uint32_t*>(src), per_row, m, parts);
    } else {
        assemble_column_blocks_kernel<uint16_t><<<blocks, 256, 0, s>>>(
            static_cast<uint16_t*>(dst), static_cast<const uint16_t*>(src), per_row, m, parts);
    }
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}

int ckl_device_status(unsigned int* info) {
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    CKL_TRY_CUDA(cudaDeviceSynchronize());
    unsigned int words[4] = {0, 0, 0, 0};
    CKL_TRY_CUDA(cudaMemcpy(words, ctx->status, sizeof words, cudaMemcpyDeviceToHost));
    if (info != nullptr) {
        std::memcpy(info, words, sizeof words);
    }
    if (words[0] != 0) {
        CKL_TRY_CUDA(cudaMemset(ctx->status, 0, sizeof words));
        return fail(CKL_ERR_DEVICE,
                    "a kernel gave up a bounded wait: code=%u block=%u role=%u detail=0x%x",
                    words[0], words[1], words[2], words[3]);
    }
    return CKL_OK;
}

int ckl_stream_copy(void* dst, const void* src, size_t bytes, ckl_stream_t stream) {
    if (bytes == 0) {
        return CKL_OK;
    }
    if (dst == nullptr || src == nullptr || bytes % 16 != 0 ||
        reinterpret_cast<uintptr_t>(dst) % 16 != 0 || reinterpret_cast<uintptr_t>(src) % 16 != 0) {
        return fail(CKL_ERR_INVALID_ARG,
                    "ckl_stream_copy needs 16-byte aligned pointers and a multiple of 16 bytes");
    }
    DeviceCtx* ctx = nullptr;
    if (const int rc = get_ctx(&ctx); rc != CKL_OK) {
        return rc;
    }
    stream_copy_kernel<<<ctx->sm_count * 2, 1024, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<uint4*>(dst), static_cast<const uint4*>(src), bytes / 16);
    CKL_TRY_CUDA(cudaGetLastError());
    return CKL_OK;
}


const char* ckl_last_error(void) { return g_last_error.c_str(); }

const char* ckl_algo_name(int algo) {
    switch (algo) {
        case CKL_ALGO_AUTO: return "auto";
        case CKL_ALGO_SIMT: return "simt";
        case CKL_ALGO_UMMA_1CTA: return "umma_1cta";
        case CKL_ALGO_UMMA_SK: return "umma_1cta_streamk";
        case CKL_ALGO_UMMA_2CTA: return "umma_2cta";
        case CKL_ALGO_UMMA_2CTA_SK: return "umma_2cta_streamk";
        case CKL_ALGO_UMMA_2CTA_WIDE: return "umma_2cta_wide";
        case CKL_ALGO_UMMA_2CTA_WIDE_SK: return "umma_2cta_wide_streamk";
        case CKL_ALGO_UMMA_1CTA_N128: return "umma_1cta_n128";
        case CKL_ALGO_UMMA_1CTA_N128_SK: return "umma_1cta_n128_streamk";
        default: return "unknown";
    }
}

void ckl_shutdown(void) {
    std::lock_guard<std::mutex> lock(g_ctx_mu);
    int prev = 0;
    const bool have_prev = cudaGetDevice(&prev) == cudaSuccess;
    for (auto& kv : g_ctx) {
        DeviceCtx* ctx = kv.second.get();
        if (cudaSetDevice(ctx->device) != cudaSuccess) {
            continue;
        }
        cudaDeviceSynchronize();
        for (auto& w : ctx->workspace) {
            cudaFree(w.second.ptr);
        }
        for (auto& w : ctx->repack) {
            cudaFree(w.second.ptr);
        }
        cudaFree(ctx->host_a.ptr);
        cudaFree(ctx->host_b.ptr);
        cudaFree(ctx->host_c.ptr);
        cudaFree(ctx->status);
        if (ctx->host_stream != nullptr) {
            cudaStreamDestroy(ctx->host_stream);
            cudaStreamDestroy(ctx->host_in);
            cudaStreamDestroy(ctx->host_out);
            for (cudaEvent_t e : ctx->host_events) {
                cudaEventDestroy(e);
            }
        }
    }
    g_ctx.clear();
    if (have_prev) {
        cudaSetDevice(prev);
    }
}

}  // extern "C"
