// Tensor-core products whose weight is chosen per row: one tcgen05 kernel over ragged groups of
// rows.  offsets[g] .. offsets[g+1] are the positions of group g; they live on the device, so
// every CTA derives the tile schedule itself and the host never waits for them.
//
//   kFormRows   C[p] = alpha * A[row(p)] * op(B_g) for the positions p of group g (op = identity
//               or transpose); tiles of 128 positions x bn columns, never across two groups.
//   kFormWgrad  W_g = alpha * sum over p in g of A[row(p)]^T G[row(p)]: the ragged dimension is
//               the one that is summed; tiles of 128 x bn of each W_g.
//
// Either form may be "extended" (kFormRows only): all positions form one group for a shared B,
// and behind the k blocks of that product a tile runs, for each adapter g whose rows it holds,
// the k blocks of T[p] * op(E_g) into the same accumulator, with the rows of other adapters
// read as zeros.  Low-rank adapters thereby cost neither a second pass over C nor tiles cut at
// the borders of requests.
//
// Ragged edges and gathers are one mechanism: rows are fetched with TMA gather4 (four row
// indices per copy, one copy per lane of the producer warp), and an index outside the tensor
// reads zeros.  Whole tiles of consecutive rows use one boxed copy instead.
//
// Operand layout in shared memory is that of the dense kernel (gemm_umma.cuh): 128-byte rows of
// 64 elements under the 128-byte swizzle.  The matrix whose reduced dimension is contiguous in
// memory is read K-major, the other one MN-major, so nothing is ever transposed in memory.
//
// Warp roles as in the dense kernel: warp 0 producer, warp 1 MMA, warps 2-5 epilogue; two
// accumulators in tensor memory; every wait bounded.
#pragma once

#include "gemm_umma.cuh"

namespace ckl {

constexpr int kMaxGemmGroups = 1024;
constexpr int kMaxLoraRank = 128;

enum GroupedForm : int { kFormRows = 0, kFormWgrad = 1 };

// Element type of C, or the two-part form: an FP32 value v stored as 16-bit hi = round(v) and
// lo = round(v - hi), lo `part` columns behind hi.  Holds 16 (BF16) or 22 (FP16) bits of v, so an
// intermediate that feeds another tensor-core product is not cut to the operand type.
template <typename T>
struct TwoPart {};

struct GroupedParams {
    const int* offsets;  // groups + 1, nullptr: one group of all rows
    const int* a_rows;   // row of A behind each position, or nullptr (identity)
    const int* b_rows;   // kFormWgrad: row of G behind each position, or nullptr
    const int* c_rows;   // kFormRows: row of C behind each position, or nullptr
    void* c;
    const float* scales;  // per group, or nullptr
    unsigned int* status;
    long long c_stride;  // kFormWgrad: elements from W_g to W_g+1
    int groups, rows;    // rows = positions in all
    int a_count, b_count, c_count;  // rows of A, G and C that exist
    int m, n, k;         // kFormWgrad: W_g is m x n; kFormRows: k columns of A, n columns of C
    int ldc;
    float alpha, beta;
    int form;
    int trans_b;         // kFormRows: B_g is stored n x k
    int bn;              // tile columns: 64, 128 or 256
    // Two-part operands: the reduction runs over the matrix once per part, `part` columns apart.
    int a_parts, a_part_cols;
    int b_parts, b_part_cols;
    int c_part_cols;     // TwoPart output: distance of lo behind hi
    // Extension (ext_groups > 0): offsets/groups describe the adapters.
    int ext_groups, ext_cols;  // adapters; columns of one part of T (a multiple of 16)
    uint32_t fmt;        // operand format for the instruction descriptor
    int c_vec;           // 16-byte accesses to C are legal
    unsigned long long wait_limit_ns;
    int overstate_first_stage;  // test hook, see GemmParams
};

struct GroupedConfig {
    static constexpr int kStages = 4;
    static constexpr uint32_t kABytes = 128 * 64 * 2;
    static constexpr uint32_t kBoxBytes = 64 * 64 * 2;
    static constexpr uint32_t kBBytes = 4 * kBoxBytes;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kThreads = 192;
    static constexpr uint32_t kStagingBytes = 4 * 4096;
    static constexpr int kNumBarriers = 2 * kStages + 5;
    static constexpr uint32_t kTableBytes = 2 * (kMaxGemmGroups + 2) * 4;
    static constexpr uint32_t kSmemBytes =
        kStages * kStageBytes + kStagingBytes + kTableBytes + kNumBarriers * 8 + 16 + 1024;
};

namespace detail {

// The schedule as every role of a CTA walks it.
struct GroupedTile {
    int group;
    int p0, valid;  // first position and number of positions (kFormRows: of the tile;
                    // kFormWgrad: of the whole group, the reduced range)
    int m0, n0;     // kFormWgrad: first row of W_g; first column
    int cols;       // columns of the tile that exist
    int k_blocks;   // 64-wide blocks of the main product
    int ext_first, ext_last;  // adapters [first, last) that may have rows in the tile
};

struct GroupedTable {
    const int* offs;   // [groups + 1], clamped to [0, rows]
    const int* tiles;  // [groups + 1] running count of 128-row tiles (kFormRows)
    int segments;      // groups that are cut into tiles
    bool whole;        // one segment of all positions (extended, or no offsets)
    int n_tiles, m_tiles;
    int total;
};

// Last index i in [0, count) with table[i] <= v (table ascending, table[0] <= v).
__device__ __forceinline__ int last_at_most(const int* table, int count, int v) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table[mid] <= v) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ __forceinline__ GroupedTile grouped_tile(const GroupedParams& p, const GroupedTable& t,
                                                    int tile) {
    GroupedTile o;
    int mt, nt;
    int m_tiles, local;
    if (p.form == kFormWgrad) {
        const int per = t.m_tiles * t.n_tiles;
        o.group = tile / per;
        local = tile - o.group * per;
        m_tiles = t.m_tiles;
    } else {
        o.group = t.segments == 1 ? 0 : last_at_most(t.tiles, t.segments, tile / t.n_tiles);
        local = tile - t.tiles[o.group] * t.n_tiles;
        m_tiles = t.tiles[o.group + 1] - t.tiles[o.group];
    }
    // Raster inside a group: bands of 16 tile rows, row index fastest, as in the dense kernel.
    constexpr int kBand = 16;
    const int band = local / (kBand * t.n_tiles);
    const int height = min(kBand, m_tiles - band * kBand);
    const int in_band = local - band * kBand * t.n_tiles;
    nt = in_band / height;
    mt = band * kBand + in_band - nt * height;
    o.n0 = nt * p.bn;
    o.cols = min(p.bn, p.n - o.n0);
    o.ext_first = o.ext_last = 0;
    if (p.form == kFormWgrad) {
        o.p0 = t.offs[o.group];
        o.valid = max(0, t.offs[o.group + 1] - o.p0);
        o.m0 = mt * 128;
        o.k_blocks = ((o.valid + 63) / 64) * p.a_parts * p.b_parts;
    } else {
        const int seg0 = t.whole ? 0 : t.offs[o.group];
        const int seg1 = t.whole ? p.rows : t.offs[o.group + 1];
        o.p0 = seg0 + mt * 128;
        o.valid = min(128, seg1 - o.p0);
        o.m0 = 0;
        o.k_blocks = ((p.k + 63) / 64) * p.a_parts;
        if (p.ext_groups > 0 && o.p0 < t.offs[p.ext_groups]) {
            // first adapter that ends behind p0, and the one after the last that starts in here
            o.ext_first = last_at_most(t.offs, p.ext_groups, o.p0);
            o.ext_last = last_at_most(t.offs, p.ext_groups, o.p0 + o.valid - 1) + 1;
        }
    }
    return o;
}

}  // namespace detail

template <typename OutT>
struct GroupedStore {
    using Elem = OutT;
    static constexpr bool kTwo = false;
};
template <typename T>
struct GroupedStore<TwoPart<T>> {
    using Elem = T;
    static constexpr bool kTwo = true;
};

template <typename OutT>
__global__ void __launch_bounds__(GroupedConfig::kThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a_box,
                    const __grid_constant__ CUtensorMap tmap_a_row,
                    const __grid_constant__ CUtensorMap tmap_b_box,
                    const __grid_constant__ CUtensorMap tmap_b_row,
                    const __grid_constant__ CUtensorMap tmap_t_row,
                    const __grid_constant__ CUtensorMap tmap_e_box, const GroupedParams p) {
    using Cfg = GroupedConfig;
    using Elem = typename GroupedStore<OutT>::Elem;
    constexpr bool kTwo = GroupedStore<OutT>::kTwo;
    constexpr int kStages = Cfg::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t ring = (raw_addr + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw_addr);
    uint8_t* staging_ptr = ring_ptr + kStages * Cfg::kStageBytes;
    uint8_t* table_ptr = staging_ptr + Cfg::kStagingBytes;
    uint8_t* bars_ptr = table_ptr + Cfg::kTableBytes;
    const uint32_t bars = ring + (kStages * Cfg::kStageBytes + Cfg::kStagingBytes + Cfg::kTableBytes);
    auto full_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(s); };
    auto empty_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(kStages + s); };
    auto acc_full_bar = [&](uint32_t a) { return bars + 8u * (2 * kStages + a); };
    auto acc_empty_bar = [&](uint32_t a) { return bars + 8u * (2 * kStages + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * kStages + 4);
    const uint32_t tmem_slot = bars + 8u * Cfg::kNumBarriers;
    volatile uint32_t* tmem_slot_ptr =
        reinterpret_cast<volatile uint32_t*>(bars_ptr + 8 * Cfg::kNumBarriers);

    detail::Control ctl;
    ctl.abort_flag = reinterpret_cast<volatile int*>(bars_ptr + 8 * Cfg::kNumBarriers + 4);
    ctl.abort_flag_smem = tmem_slot + 4u;
    ctl.status = p.status;
    ctl.pair = false;
    ctl.peer_rank = 0;
    ctl.limit_ns = p.wait_limit_ns != 0 ? p.wait_limit_ns : kWaitLimitNs;

    const int warp = static_cast<int>(threadIdx.x >> 5);
    const uint32_t lane = ptx::lane_id();

    // ---- set-up: barriers, tensor memory, the schedule's table ------------------------------
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            ptx::mbar_init(acc_full_bar(a), 1);
            ptx::mbar_init(acc_empty_bar(a), 4);
        }
        ptx::mbar_init(drain_bar, 1);
        *ctl.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    int* offs = reinterpret_cast<int*>(table_ptr);
    int* tile_count = offs + kMaxGemmGroups + 2;
    if (p.offsets != nullptr) {
        for (int g = static_cast<int>(threadIdx.x); g <= p.groups; g += Cfg::kThreads) {
            offs[g] = min(max(p.offsets[g], 0), p.rows);
        }
    } else if (threadIdx.x == 0) {
        offs[0] = 0;
        offs[1] = p.rows;
    }
    __syncthreads();
    detail::GroupedTable table;
    table.offs = offs;
    table.tiles = tile_count;
    table.whole = p.offsets == nullptr || p.ext_groups > 0;
    table.segments = table.whole ? 1 : p.groups;
    table.n_tiles = (p.n + p.bn - 1) / p.bn;
    table.m_tiles = (p.m + 127) / 128;
    if (warp == 0) {
        if (table.whole) {
            if (lane == 0) {
                tile_count[0] = 0;
                tile_count[1] = (p.rows + 127) / 128;
            }
        } else {
            int run = 0;
            for (int g0 = 0; g0 < p.groups; g0 += 32) {
                const int g = g0 + static_cast<int>(lane);
                int v = g < p.groups ? (max(0, offs[g + 1] - offs[g]) + 127) / 128 : 0;
                const int own_tiles = v;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
                    v += static_cast<int>(lane) >= d ? u : 0;
                }
                if (g < p.groups) {
                    tile_count[g] = run + v - own_tiles;
                }
                run += __shfl_sync(0xFFFFFFFFu, v, 31);
            }
            if (lane == 0) {
                tile_count[p.groups] = run;
            }
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_ptr;
    table.total = p.form == kFormWgrad ? p.groups * table.m_tiles * table.n_tiles
                                       : tile_count[table.segments] * table.n_tiles;
    const int ext_blocks_per_part = (p.ext_cols + 63) / 64;
    const int base_blocks = (p.k + 63) / 64;

    // ---- roles ------------------------------------------------------------------------------
    if (warp == 0) {
        // Producer: all 32 lanes, each issues its own copies.
        uint32_t it = 0;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        auto acquire_stage = [&]() -> bool {
            int got = 1;
            if (lane == 0) {
                got = detail::wait_barrier(empty_bar(stage), phase ^ 1u, ctl, kRoleProducer, it) ? 1 : 0;
            }
            return __shfl_sync(0xFFFFFFFFu, got, 0) != 0;
        };
        auto announce = [&](uint32_t bytes) {
            if (lane == 0) {
                const bool wrong = p.overstate_first_stage != 0 && it == 0 && blockIdx.x == 0;
                ptx::mbar_arrive_expect_tx(full_bar(stage), bytes + (wrong ? 16u : 0u));
            }
            __syncwarp();
        };
        auto advance = [&]() {
            ++it;
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        };
        for (int tile = blockIdx.x; ok && tile < table.total; tile += gridDim.x) {
            const detail::GroupedTile t = detail::grouped_tile(p, table, tile);
            const int boxes = (t.cols + 63) / 64;
            if (p.form == kFormRows) {
                // Four rows of A per lane, the same for every k block.  Rows behind the tile's
                // last one are not stored, so copies of only such rows are left out.
                const int first = static_cast<int>(lane) * 4;
                const bool gather = p.a_rows != nullptr || t.valid < 128;
                int r[4] = {p.a_count, p.a_count, p.a_count, p.a_count};
                if (gather) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (first + i < t.valid) {
                            r[i] = p.a_rows != nullptr ? __ldg(p.a_rows + t.p0 + first + i)
                                                       : t.p0 + first + i;
                        }
                    }
                }
                const uint32_t a_bytes =
                    gather ? static_cast<uint32_t>((t.valid + 3) / 4) * 512u : Cfg::kABytes;
                const int group = table.whole ? 0 : t.group;
                for (int kb = 0; kb < t.k_blocks; ++kb) {
                    if (!acquire_stage()) {
                        ok = false;
                        break;
                    }
                    announce(a_bytes + static_cast<uint32_t>(boxes) * Cfg::kBoxBytes);
                    const uint32_t a_dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                    const uint32_t b_dst = a_dst + Cfg::kABytes;
                    const int part = kb >= base_blocks ? 1 : 0;
                    const int k0 = (kb - part * base_blocks) * 64;
                    const int ax = k0 + part * p.a_part_cols;
                    if (gather) {
                        if (first < t.valid) {
                            ptx::tma_gather4(a_dst + lane * 512u, &tmap_a_row, full_bar(stage), ax,
                                             r[0], r[1], r[2], r[3]);
                        }
                    } else if (lane == 0) {
                        ptx::tma_load_2d(a_dst, &tmap_a_box, full_bar(stage), ax, t.p0);
                    }
                    if (static_cast<int>(lane) < boxes) {
                        const int col = t.n0 + static_cast<int>(lane) * 64;
                        ptx::tma_load_3d(b_dst + lane * Cfg::kBoxBytes, &tmap_b_box, full_bar(stage),
                                         p.trans_b ? k0 : col, p.trans_b ? col : k0, group);
                    }
                    advance();
                }
                for (int g = t.ext_first; ok && g < t.ext_last; ++g) {
                    const int lo = max(offs[g], t.p0), hi = min(offs[g + 1], t.p0 + t.valid);
                    if (lo >= hi) {
                        continue;
                    }
                    int q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int pos = t.p0 + first + i;
                        q[i] = pos >= lo && pos < hi ? pos : p.rows;  // outside T: zeros
                    }
                    for (int eb = 0; eb < 2 * ext_blocks_per_part; ++eb) {
                        if (!acquire_stage()) {
                            ok = false;
                            break;
                        }
                        announce(Cfg::kABytes + static_cast<uint32_t>(boxes) * Cfg::kBoxBytes);
                        const uint32_t a_dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                        const uint32_t b_dst = a_dst + Cfg::kABytes;
                        const int part = eb >= ext_blocks_per_part ? 1 : 0;
                        const int k0 = (eb - part * ext_blocks_per_part) * 64;
                        ptx::tma_gather4(a_dst + lane * 512u, &tmap_t_row, full_bar(stage),
                                         k0 + part * p.ext_cols, q[0], q[1], q[2], q[3]);
                        if (static_cast<int>(lane) < boxes) {
                            const int col = t.n0 + static_cast<int>(lane) * 64;
                            ptx::tma_load_3d(b_dst + lane * Cfg::kBoxBytes, &tmap_e_box,
                                             full_bar(stage), p.trans_b ? k0 : col,
                                             p.trans_b ? col : k0, g);
                        }
                        advance();
                    }
                }
            } else {
                // Weight gradient: 64 positions per block, both operands MN-major.
                const int row_blocks = (t.valid + 63) / 64;
                const int a_boxes = (min(128, p.m - t.m0) + 63) / 64;
                const int quad = static_cast<int>(lane & 15u);
                const int half = static_cast<int>(lane >> 4);
                for (int kb = 0; kb < t.k_blocks; ++kb) {
                    const int part = kb >= row_blocks ? 1 : 0;
                    const int i0 = (kb - part * row_blocks) * 64;
                    const int left = t.valid - i0;
                    const bool gather_a = p.a_rows != nullptr || left < 64;
                    const bool gather_b = p.b_rows != nullptr || left < 64;
                    int ra[4] = {p.a_count, p.a_count, p.a_count, p.a_count};
                    int rb[4] = {p.b_count, p.b_count, p.b_count, p.b_count};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int in = quad * 4 + i;
                        if (in < left) {
                            const int pos = t.p0 + i0 + in;
                            if (gather_a) {
                                ra[i] = p.a_rows != nullptr ? __ldg(p.a_rows + pos) : pos;
                            }
                            if (gather_b) {
                                rb[i] = p.b_rows != nullptr ? __ldg(p.b_rows + pos) : pos;
                            }
                        }
                    }
                    if (!acquire_stage()) {
                        ok = false;
                        break;
                    }
                    announce(static_cast<uint32_t>(a_boxes + boxes) * Cfg::kBoxBytes);
                    const uint32_t a_dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                    const uint32_t b_dst = a_dst + Cfg::kABytes;
                    const int ax = t.m0 + (p.a_parts > 1 ? part * p.a_part_cols : 0);
                    const int bx = t.n0 + (p.b_parts > 1 ? part * p.b_part_cols : 0);
                    if (gather_a) {
                        if (half < a_boxes) {
                            ptx::tma_gather4(a_dst + half * Cfg::kBoxBytes + quad * 512u, &tmap_a_row,
                                             full_bar(stage), ax + half * 64, ra[0], ra[1], ra[2], ra[3]);
                        }
                    } else if (static_cast<int>(lane) < a_boxes) {
                        ptx::tma_load_2d(a_dst + lane * Cfg::kBoxBytes, &tmap_a_box, full_bar(stage),
                                         ax + static_cast<int>(lane) * 64, t.p0 + i0);
                    }
                    if (gather_b) {
                        for (int b = half; b < boxes; b += 2) {
                            ptx::tma_gather4(b_dst + b * Cfg::kBoxBytes + quad * 512u, &tmap_b_row,
                                             full_bar(stage), bx + b * 64, rb[0], rb[1], rb[2], rb[3]);
                        }
                    } else if (static_cast<int>(lane) < boxes) {
                        ptx::tma_load_3d(b_dst + lane * Cfg::kBoxBytes, &tmap_b_box, full_bar(stage),
                                         bx + static_cast<int>(lane) * 64, t.p0 + i0, 0);
                    }
                    advance();
                }
            }
        }
        // Tail: no copy may be in flight and no stage may still be signalled when the CTA ends.
        if (lane == 0) {
            const uint32_t first = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u;
            for (uint32_t i = first; i < it; ++i) {
                const int s = static_cast<int>(i % kStages);
                const uint32_t use = i / kStages;
                if (ok && !detail::wait_barrier(empty_bar(s), use & 1u, ctl, kRoleDrain, i)) {
                    ok = false;
                }
                if (!ok) {
                    detail::drain_wait(full_bar(s), use & 1u);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (ptx::elect_one_sync()) {
            // MMA issuer.  Offsets per 16 reduced elements: 32 B along a K-major row, 2048 B (16
            // rows) in an MN-major box.
            const bool a_mn = p.form == kFormWgrad;
            const bool b_mn = a_mn || !p.trans_b;
            const uint32_t a_step = a_mn ? 2048u >> 4 : 32u >> 4;
            const uint32_t b_step = b_mn ? 2048u >> 4 : 32u >> 4;
            uint32_t it = 0;
            int stage = 0;
            uint32_t phase = 0;
            uint32_t count = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < table.total; tile += gridDim.x) {
                const detail::GroupedTile t = detail::grouped_tile(p, table, tile);
                const uint32_t acc = count & 1u;
                if (!detail::wait_barrier(acc_empty_bar(acc), ((count >> 1) & 1u) ^ 1u, ctl, kRoleMma,
                                          0x80000000u | count)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * 256u;
                // An MN-major B is read in whole 64-column boxes, a K-major one in 16-row steps.
                const uint32_t width = static_cast<uint32_t>(
                    b_mn ? (t.cols + 63) / 64 * 64 : (t.cols + 15) / 16 * 16);
                const uint32_t idesc =
                    ptx::make_idesc_f16(p.fmt, a_mn ? 1u : 0u, b_mn ? 1u : 0u, 128, width);
                uint32_t accumulate = 0;
                auto block = [&](int steps) -> bool {
                    if (!detail::wait_barrier(full_bar(stage), phase, ctl, kRoleMma, it)) {
                        return false;
                    }
                    const uint32_t a_src = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                    const uint32_t b_src = a_src + Cfg::kABytes;
                    const uint64_t a_desc =
                        ptx::make_smem_desc_sw128(a_src, a_mn ? Cfg::kBoxBytes : 16u, 1024);
                    const uint64_t b_desc =
                        ptx::make_smem_desc_sw128(b_src, b_mn ? Cfg::kBoxBytes : 16u, 1024);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j < steps) {
                            ptx::umma_f16(d_tmem, a_desc + static_cast<uint64_t>(j * a_step),
                                          b_desc + static_cast<uint64_t>(j * b_step), idesc, accumulate);
                            accumulate = 1;
                        }
                    }
                    ptx::umma_commit(empty_bar(stage));
                    ++it;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    return true;
                };
                for (int kb = 0; kb < t.k_blocks; ++kb) {
                    if (!block(4)) {
                        ok = false;
                        break;
                    }
                }
                for (int g = t.ext_first; ok && g < t.ext_last; ++g) {
                    if (max(offs[g], t.p0) >= min(offs[g + 1], t.p0 + t.valid)) {
                        continue;
                    }
                    for (int eb = 0; eb < 2 * ext_blocks_per_part; ++eb) {
                        const int in_part = eb >= ext_blocks_per_part ? eb - ext_blocks_per_part : eb;
                        if (!block(min(4, (p.ext_cols - in_part * 64) / 16))) {
                            ok = false;
                            break;
                        }
                    }
                }
                if (ok) {
                    if (accumulate != 0) {
                        ptx::umma_commit(acc_full_bar(acc));
                    } else {
                        ptx::mbar_arrive(acc_full_bar(acc));  // nothing to sum: the epilogue uses zeros
                    }
                    ++count;
                }
            }
            if (ok) {
                const uint32_t first = count > 2u ? count - 2u : 0u;
                for (uint32_t i = first; i < count && ok; ++i) {
                    ok = detail::wait_barrier(acc_empty_bar(i & 1u), (i >> 1) & 1u, ctl, kRoleDrain,
                                              0x80000000u | i);
                }
            } else {
                ptx::umma_commit(drain_bar);
                detail::drain_wait(drain_bar, 0);
            }
        }
        __syncwarp();
    } else {
        // Epilogue: 32 columns at a time through shared memory (FP32, 32 rows x 128 B per warp),
        // so that a warp writes whole 64- or 128-byte runs of a row wherever that row lies.
        const uint32_t quad = static_cast<uint32_t>(warp) & 3u;
        uint8_t* stg = staging_ptr + quad * 4096;
        using T = detail::OutTraits<Elem>;
        constexpr int kVec = T::kVec;            // elements per 16 bytes
        constexpr int kLanesPerRow = 32 / kVec;  // 8 for FP32, 4 for 16-bit types
        constexpr int kRowsPerPass = 32 / kLanesPerRow;
        const int sub = static_cast<int>(lane) % kLanesPerRow;
        uint32_t count = 0;
        bool alive = true;
        for (int tile = blockIdx.x; alive && tile < table.total; tile += gridDim.x) {
            const detail::GroupedTile t = detail::grouped_tile(p, table, tile);
            const uint32_t acc = count & 1u;
            const uint32_t parity = (count >> 1) & 1u;
            // Row of C that lane `lane` of this warp stands for, -1 for none.
            const int in_tile = static_cast<int>(quad) * 32 + static_cast<int>(lane);
            int my_row = -1;
            if (p.form == kFormWgrad) {
                my_row = t.m0 + in_tile < p.m ? t.m0 + in_tile : -1;
            } else if (in_tile < t.valid) {
                my_row = p.c_rows != nullptr ? __ldg(p.c_rows + t.p0 + in_tile) : t.p0 + in_tile;
                my_row = my_row >= 0 && my_row < p.c_count ? my_row : -1;
            }
            Elem* c_base = static_cast<Elem*>(p.c) +
                           (p.form == kFormWgrad ? static_cast<long long>(t.group) * p.c_stride : 0ll);
            const float factor = p.alpha * (p.scales != nullptr ? __ldg(p.scales + t.group) : 1.0f);
            int ok = 1;
            if (lane == 0) {
                ok = detail::wait_barrier(acc_full_bar(acc), parity, ctl, kRoleEpilogue, count) ? 1 : 0;
            }
            ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
            if (!ok) {
                alive = false;
                break;
            }
            for (int i = 0; i < 1024 && !ptx::mbar_try_wait(acc_full_bar(acc), parity); ++i) {
            }
            ptx::tc_fence_after_sync();
            const bool nothing = t.k_blocks == 0 && t.ext_first == t.ext_last;
            const uint32_t t_row = tmem_base + ((quad * 32u) << 16) + acc * 256u;
            for (int c0 = 0; c0 < t.cols; c0 += 32) {
                uint32_t r[32];
                if (nothing) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        r[i] = 0;
                    }
                } else {
                    ptx::tmem_ld_32x32(t_row + static_cast<uint32_t>(c0), r);
                    ptx::tmem_ld_wait();
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    *reinterpret_cast<uint4*>(stg + lane * 128u + ((u ^ (lane & 7u)) << 4)) =
                        make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]);
                }
                __syncwarp();
                const int col = t.n0 + c0 + sub * kVec;
                const int have = min(kVec, t.n0 + t.cols - col);
#pragma unroll
                for (int pass = 0; pass < 32 / kRowsPerPass; ++pass) {
                    const int row = pass * kRowsPerPass + static_cast<int>(lane) / kLanesPerRow;
                    const int c_row = __shfl_sync(0xFFFFFFFFu, my_row, row);
                    float v[kVec];
#pragma unroll
                    for (int u = 0; u < kVec / 4; ++u) {
                        const float4 x = *reinterpret_cast<const float4*>(
                            stg + row * 128 + (((sub * (kVec / 4) + u) ^ (row & 7)) << 4));
                        v[4 * u] = x.x; v[4 * u + 1] = x.y; v[4 * u + 2] = x.z; v[4 * u + 3] = x.w;
                    }
                    if (c_row < 0 || have <= 0) {
                        continue;
                    }
                    Elem* dst = c_base + static_cast<size_t>(c_row) * p.ldc + col;
                    const bool full = p.c_vec != 0 && have == kVec;
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        v[i] *= factor;
                    }
                    if constexpr (kTwo) {
                        float lo[kVec];
#pragma unroll
                        for (int i = 0; i < kVec; ++i) {
                            Elem h;
                            T::store(&h, v[i]);
                            lo[i] = v[i] - T::load(&h);
                        }
                        T::store_vec(dst, v);  // widths are multiples of 16 columns
                        T::store_vec(dst + p.c_part_cols, lo);
                    } else {
                        if (p.beta != 0.0f) {
                            float old[kVec];
                            if (full) {
                                T::load_vec(dst, old);
                            } else {
#pragma unroll
                                for (int i = 0; i < kVec; ++i) {
                                    old[i] = i < have ? T::load(dst + i) : 0.0f;
                                }
                            }
#pragma unroll
                            for (int i = 0; i < kVec; ++i) {
                                v[i] = fmaf(p.beta, old[i], v[i]);
                            }
                        }
                        if (full) {
                            T::store_vec(dst, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < kVec; ++i) {
                                if (i < have) {
                                    T::store(dst + i, v[i]);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive(acc_empty_bar(acc));
            }
            ++count;
        }
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace ckl
