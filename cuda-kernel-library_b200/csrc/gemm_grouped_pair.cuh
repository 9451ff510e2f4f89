// The CTA-pair form of the grouped products, for launches with tiles enough for every pair.
//
// A pair computes a transposed tile: the COLUMNS of C are the 256 rows of the tensor core's
// product (128 per CTA: the weights, or G of a weight gradient) and the ROWS of C (positions, or
// the rows of W_g) are its N, up to 256 in steps of 32.  So the ragged dimension is the one the
// instruction takes in fine steps: a group of 300 rows runs as two tiles of 160 and 140 (N = 160
// each), where 128-row tiles would compute 384 and 256-row ones 512; and each CTA reads half of
// the rows and its own columns only, 32 KB per 64 k for 256 x 256 outputs, where the single-CTA
// tile reads 48 KB for half as many.
//
//   columns operand (A of the instruction): W_g, MN-major (or K-major when op is the transpose);
//       G of a weight gradient, MN-major.  Always boxed TMA copies, 64 x 64 boxes.
//   rows operand (B of the instruction, half of the rows per CTA): positions of A, K-major; columns
//       of A in a weight gradient, MN-major.  Boxed, or gathered by the loader warps.
// The last block of a group's sum in a weight gradient, when it is not whole, comes through the
// loaders in both operands, which put zeros behind the group's end.
//
// Epilogue: a lane holds one column of C and 32 rows at a time, so the staging buffer is
// written row by row across the lanes; from there rows leave as in the single-CTA kernel.
#pragma once

#include <type_traits>

#include "gemm_grouped.cuh"

namespace ckl {

struct GroupedPairConfig {
    // Five stages of 32 KB: a sixth brought nothing, its room holds the staging buffers.
    static constexpr int kStages = 5;
    static constexpr uint32_t kBoxBytes = 64 * 64 * 2;
    static constexpr uint32_t kColsBytes = 2 * kBoxBytes;
    static constexpr uint32_t kRowsBytes = 2 * kBoxBytes;
    static constexpr uint32_t kStageBytes = kColsBytes + kRowsBytes;
    static constexpr int kFirstLoader = 6;
    static constexpr int kScheduler = kFirstLoader + kStages;  // one loader warp per stage
    static constexpr int kThreads = 32 * (kScheduler + 1);
    static constexpr uint32_t kBufferBytes = 4096;
    static constexpr int kBuffers = 3;  // per epilogue warp
    static constexpr uint32_t kWarpStaging = kBuffers * kBufferBytes;
    static constexpr uint32_t kStagingBytes = 4 * kWarpStaging;
    static constexpr int kNumBarriers = 4 * kStages + 5 + 8;
    static constexpr uint32_t kTableBytes = 2 * (kMaxGemmGroups + 2) * 4 + kMaxGemmGroups / 8;
    static constexpr uint32_t kQueueBytes = 4 * 64;
    static constexpr uint32_t kRowTableBytes = 4 * 256 * 4;  // rows of C, per epilogue warp
    static constexpr uint32_t kSmemBytes =
        kStages * kStageBytes + kStagingBytes + kTableBytes + kQueueBytes + kRowTableBytes +
        kNumBarriers * 8 + 16 + 1024;
};

namespace detail {

struct PairTile {
    int group;
    int p0, valid;  // kFormRows: positions of the tile; kFormWgrad: of the group (the sum)
    int r0, rows;   // first row of C and rows of the tile (kFormRows: r0 = p0, rows = valid)
    int c0;         // first column
    int half;       // rows per CTA: 16, 32, ... 128 (kFormWgrad: 64 or 128)
    int k_blocks;
    int ext_first, ext_last;  // kExtBlocks: adapters that may have rows in the tile
};

__device__ __forceinline__ PairTile pair_tile(const GroupedParams& p, const GroupedTable& t, int tile) {
    PairTile o;
    int local, row_tiles, total_rows, seg0;
    if (p.form == kFormWgrad) {
        const int per = t.m_tiles * t.n_tiles;
        o.group = tile / per;
        local = tile - o.group * per;
        row_tiles = t.m_tiles;
        total_rows = p.m;
        seg0 = 0;
    } else {
        o.group = t.segments == 1 ? 0 : last_at_most(t.tiles, t.segments, tile / t.n_tiles);
        local = tile - t.tiles[o.group] * t.n_tiles;
        row_tiles = t.tiles[o.group + 1] - t.tiles[o.group];
        seg0 = t.whole ? 0 : t.offs[o.group];
        total_rows = (t.whole ? p.rows : t.offs[o.group + 1]) - seg0;
    }
    constexpr int kBand = 8;
    const int band = local / (kBand * t.n_tiles);
    const int height = min(kBand, row_tiles - band * kBand);
    const int in_band = local - band * kBand * t.n_tiles;
    const int ct = in_band / height;
    const int rt = band * kBand + in_band - ct * height;
    o.c0 = ct * 256;
    // Tiles of one group are equally high.
    const int unit = p.form == kFormWgrad ? 128 : 32;
    const int step = ((total_rows + row_tiles - 1) / row_tiles + unit - 1) / unit * unit;
    o.r0 = seg0 + rt * step;
    o.rows = max(0, min(step, total_rows - rt * step));
    o.half = max(unit, (o.rows + unit - 1) / unit * unit) / 2;
    o.ext_first = o.ext_last = 0;
    if (p.form == kFormWgrad) {
        o.p0 = t.offs[o.group];
        o.valid = max(0, t.offs[o.group + 1] - o.p0);
        o.k_blocks = o.rows > 0 ? (o.valid + 63) / 64 : 0;
    } else {
        o.p0 = o.r0;
        o.valid = o.rows;
        o.k_blocks = o.rows > 0 ? (p.k + 63) / 64 : 0;
        if (p.ext_mode == kExtBlocks && o.rows > 0 && o.p0 < t.offs[p.groups]) {
            o.ext_first = last_at_most(t.offs, p.groups, o.p0);
            o.ext_last = last_at_most(t.offs, p.groups, o.p0 + o.valid - 1) + 1;
        }
    }
    return o;
}

// factor * a and factor * b (FP32 bits), rounded and packed with a in the low half.
template <typename Elem>
__device__ __forceinline__ uint32_t pack16(float factor, uint32_t a, uint32_t b) {
    const float x = factor * __uint_as_float(a), y = factor * __uint_as_float(b);
    uint32_t w;
    if constexpr (std::is_same<Elem, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        w = *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        w = *reinterpret_cast<const uint32_t*>(&h);
    }
    return w;
}

}  // namespace detail

// kExt: an extended product (the single-CTA kernel says why that is a kernel of its own).
template <typename OutT, bool kExt>
__global__ void __launch_bounds__(GroupedPairConfig::kThreads, 1)
grouped_pair_kernel(const __grid_constant__ GroupedProblem problem) {
    const GroupedParams& p = problem.p;
    const CUtensorMap &tmap_rows = problem.a_box, &tmap_cols = problem.b_box;
    const CUtensorMap &tmap_ext = problem.e_box, &tmap_c = problem.c;
    using Cfg = GroupedPairConfig;
    using Elem = typename GroupedStore<OutT>::Elem;
    constexpr int kStages = Cfg::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t ring = (raw_addr + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw_addr);
    uint8_t* staging_ptr = ring_ptr + kStages * Cfg::kStageBytes;
    uint8_t* table_ptr = staging_ptr + Cfg::kStagingBytes;
    uint8_t* queue_ptr = table_ptr + Cfg::kTableBytes;
    uint8_t* rows_ptr = queue_ptr + Cfg::kQueueBytes;
    uint8_t* bars_ptr = rows_ptr + Cfg::kRowTableBytes;
    const uint32_t bars =
        ring + (kStages * Cfg::kStageBytes + Cfg::kStagingBytes + Cfg::kTableBytes + Cfg::kQueueBytes +
                Cfg::kRowTableBytes);
    auto full_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(s); };
    auto empty_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(kStages + s); };
    auto loaded_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(2 * kStages + s); };
    auto acc_full_bar = [&](uint32_t a) { return bars + 8u * (3 * kStages + a); };
    auto acc_empty_bar = [&](uint32_t a) { return bars + 8u * (3 * kStages + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (3 * kStages + 4);
    // a stage that the loaders have to write has been acquired (where not every stage is one)
    auto wanted_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(3 * kStages + 13 + s); };
    using Queue = detail::TileQueue<detail::PairTile>;
    static_assert(Queue::kBytes <= Cfg::kQueueBytes && 2 * detail::kTileSlots == 8, "queue layout");
    const Queue queue = {reinterpret_cast<int4*>(queue_ptr), bars + 8u * (3 * kStages + 5)};
    const uint32_t tmem_slot = bars + 8u * Cfg::kNumBarriers;
    volatile uint32_t* tmem_slot_ptr =
        reinterpret_cast<volatile uint32_t*>(bars_ptr + 8 * Cfg::kNumBarriers);

    const int warp = static_cast<int>(threadIdx.x >> 5);
    const uint32_t lane = ptx::lane_id();
    const uint32_t rank = ptx::cluster_cta_rank();
    const bool leader = rank == 0;
    const bool wgrad = !kExt && p.form == kFormWgrad;
    const bool gather = p.load_a != 0;
    const bool loads = kExt || wgrad || gather;  // the loaders work

    detail::Control ctl;
    ctl.abort_flag = reinterpret_cast<volatile int*>(bars_ptr + 8 * Cfg::kNumBarriers + 4);
    ctl.abort_flag_smem = tmem_slot + 4u;
    ctl.status = p.status;
    ctl.pair = true;
    ctl.peer_rank = rank ^ 1u;
    ctl.limit_ns = p.wait_limit_ns != 0 ? p.wait_limit_ns : kWaitLimitNs;

    // ---- set-up -------------------------------------------------------------------------------
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 2);    // the producers of both CTAs, at the leader
            ptx::mbar_init(empty_bar(s), 1);
            ptx::mbar_init(loaded_bar(s), 2);  // the loaders of both CTAs, at the leader
            ptx::mbar_init(wanted_bar(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            ptx::mbar_init(acc_full_bar(a), 1);
            ptx::mbar_init(acc_empty_bar(a), 8);  // four warps of either CTA, at the leader
        }
        ptx::mbar_init(drain_bar, 1);
        // producer, the leader's MMA thread, four epilogue warps, loaders
        queue.init(5u + (leader ? 1u : 0u) + (loads ? kStages : 0u));
        *ctl.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (threadIdx.x == 64) {
        ptx::prefetch_tensormap(&tmap_rows);
        ptx::prefetch_tensormap(&tmap_cols);
        ptx::prefetch_tensormap(&tmap_c);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(tmem_slot, 512);
        ptx::tmem_relinquish_pair();
    }
    // Up to here only this CTA's own memory: the kernel before this one may still be running.
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    int* offs = reinterpret_cast<int*>(table_ptr);
    const detail::GroupedTable table =
        detail::make_table(p, offs, offs + kMaxGemmGroups + 2, 256, 256, warp, lane, Cfg::kThreads);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_ptr;
    const int total = detail::total_tiles(p, table);
    const int ext_blocks = (p.ext_cols + 63) / 64;
    const bool shifts = kExt && p.fmt == 0;
    const int unit = static_cast<int>(blockIdx.x >> 1);
    const int units = static_cast<int>(gridDim.x >> 1);

    // ---- roles --------------------------------------------------------------------------------
    if (warp == 0) {
        if (ptx::elect_one_sync()) {
            // TMA producer: this CTA's columns and, unless gathered, its half of the rows.  All bytes
            // of a stage are credited to the leader's barrier.
            uint32_t it = 0;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            uint32_t bar = 0;
            // Both producers arrive for every stage, also one that they copy nothing into (columns behind
            // the last, gathered rows): a stage cannot be filled again before both have seen it free,
            // so neither falls two phases behind, which a barrier does not tell from none.
            auto acquire_stage = [&](uint32_t bytes_of_both, bool wanted) -> bool {
                if (!detail::wait_barrier(empty_bar(stage), phase ^ 1u, ctl, kRoleProducer, it)) {
                    return false;
                }
                if (wanted) {
                    ptx::mbar_arrive(wanted_bar(stage));
                }
                bar = ptx::map_to_cta(full_bar(stage), 0);
                if (leader) {
                    const bool wrong = p.overstate_first_stage != 0 && it == 0 && blockIdx.x == 0;
                    ptx::mbar_arrive_expect_tx(full_bar(stage), bytes_of_both + (wrong ? 16u : 0u));
                } else {
                    ptx::mbar_arrive_cluster(bar);
                }
                return true;
            };
            auto advance = [&]() {
                ++it;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            detail::PairTile t;
            for (uint32_t i = 0; ok && queue.pop(i, &t, ctl, false, lane); ++i) {
                const int col0 = t.c0 + static_cast<int>(rank) * 128;
                // 64-column boxes that exist, of this CTA and of both
                const int boxes = min(2, max(0, (p.n - col0 + 63) / 64));
                const uint32_t cols_bytes =
                    static_cast<uint32_t>(min(4, (p.n - t.c0 + 63) / 64)) * Cfg::kBoxBytes;
                // (all box loops are unrolled: one thread issues them, and a rolled loop spends about
                // 100 cycles on each)
                auto load_cols = [&](uint32_t dst, const CUtensorMap* map, int k0, int z) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if (b < boxes) {
                            const int col = col0 + b * 64;
                            ptx::tma_load_3d_pair(dst + b * Cfg::kBoxBytes, map, bar, p.trans_b ? k0 : col,
                                                  p.trans_b ? col : k0, z);
                        }
                    }
                };
                if (!wgrad) {
                    const int group = kExt || table.whole ? 0 : t.group;
                    const int row0 = t.p0 + static_cast<int>(rank) * t.half;
                    const int row_boxes = gather ? 0 : (t.half + 63) / 64;
                    const uint32_t rows_bytes = 2u * static_cast<uint32_t>(row_boxes) * Cfg::kBoxBytes;
                    ok = detail::for_blocks<kExt>(
                        p, table, t, ext_blocks, 0, 0x7fffffff,
                        [&](int, int g, const detail::Span&, int eb, bool) -> bool {
                            if (!acquire_stage(cols_bytes, !gather)) {
                                return false;
                            }
                            load_cols(ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes, &tmap_ext, eb * 64, g);
                            advance();
                            return true;
                        },
                        [&](int kb) -> bool {
                            if (!acquire_stage(cols_bytes + rows_bytes, false)) {
                                return false;
                            }
                            const uint32_t dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                            load_cols(dst, &tmap_cols, kb * 64, group);
                            // rows behind the tile's last are another tile's, or zeros: not stored
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                if (b < row_boxes) {
                                    ptx::tma_load_2d_pair(dst + Cfg::kColsBytes + b * Cfg::kBoxBytes, &tmap_rows, bar,
                                                          kb * 64, row0 + b * 64);
                                }
                            }
                            advance();
                            return true;
                        });
                } else {
                    const int row0 = t.r0 + static_cast<int>(rank) * t.half;
                    // boxes of 64 rows of W_g (columns of A) that exist, of this CTA and of both
                    auto existing = [&](int from) { return min(t.half / 64, max(0, (p.m - from + 63) / 64)); };
                    const int row_boxes = existing(row0);
                    const uint32_t rows_bytes =
                        gather ? 0u
                               : static_cast<uint32_t>(existing(t.r0) + existing(t.r0 + t.half)) * Cfg::kBoxBytes;
                    for (int kb = 0; kb < t.k_blocks; ++kb) {
                        // a last block that is not whole comes through the loaders
                        const bool whole = t.valid - kb * 64 >= 64;
                        if (!acquire_stage(whole ? cols_bytes + rows_bytes : 0u, !gather && !whole)) {
                            ok = false;
                            break;
                        }
                        const uint32_t dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                        const int pos = t.p0 + kb * 64;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            if (whole && b < boxes) {
                                ptx::tma_load_3d_pair(dst + b * Cfg::kBoxBytes, &tmap_cols, bar, col0 + b * 64, pos,
                                                      0);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            if (whole && !gather && b < row_boxes) {
                                ptx::tma_load_2d_pair(dst + Cfg::kColsBytes + b * Cfg::kBoxBytes, &tmap_rows, bar,
                                                      row0 + b * 64, pos);
                            }
                        }
                        advance();
                    }
                }
            }
            // Tail: no copy into this CTA may be in flight and no stage may still be signalled when
            // it ends.
            const uint32_t first = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u;
            for (uint32_t i = first; i < it; ++i) {
                const int s = static_cast<int>(i % kStages);
                const uint32_t use = i / kStages;
                if (ok && !detail::wait_barrier(empty_bar(s), use & 1u, ctl, kRoleDrain, i)) {
                    ok = false;
                }
                if (!ok) {
                    if (leader) {
                        detail::drain_wait(full_bar(s), use & 1u);
                    } else {
                        __nanosleep(20000);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (leader && ptx::elect_one_sync()) {
            // MMA issuer, for both CTAs.  Offsets per 16 reduced elements: 32 B along a K-major row,
            // 2048 B (16 rows) in an MN-major box.
            const bool cols_mn = wgrad || !p.trans_b;
            const bool rows_mn = wgrad;
            const uint32_t cols_step = cols_mn ? 2048u >> 4 : 32u >> 4;
            const uint32_t rows_step = rows_mn ? 2048u >> 4 : 32u >> 4;
            uint32_t it = 0;
            int stage = 0;
            uint32_t phase = 0;
            uint32_t loaded_phase = 0;
            uint32_t count = 0;
            bool ready = false;
            bool ok = true;
            detail::PairTile t;
            for (uint32_t i = 0; ok && queue.pop(i, &t, ctl, false, lane); ++i) {
                const uint32_t acc = count & 1u;
                if (!detail::wait_barrier(acc_empty_bar(acc), ((count >> 1) & 1u) ^ 1u, ctl, kRoleMma,
                                          0x80000000u | count)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * 256u;
                const uint32_t idesc = ptx::make_idesc_f16(p.fmt, cols_mn ? 1u : 0u, rows_mn ? 1u : 0u, 256,
                                                           static_cast<uint32_t>(2 * t.half));
                uint32_t accumulate = 0;
                auto block = [&](int steps, bool loaded, bool shift) -> bool {
                    if (!ready && !detail::wait_barrier(full_bar(stage), phase, ctl, kRoleMma, it)) {
                        return false;
                    }
                    if (loaded) {
                        if (!detail::wait_barrier<true>(loaded_bar(stage), (loaded_phase >> stage) & 1u, ctl,
                                                        kRoleMma, 0x40000000u | it)) {
                            return false;
                        }
                        loaded_phase ^= 1u << stage;
                    }
                    const uint32_t cols_src = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                    const uint64_t cols_desc =
                        ptx::make_smem_desc_sw128(cols_src, cols_mn ? Cfg::kBoxBytes : 16u, 1024);
                    const uint64_t rows_desc = ptx::make_smem_desc_sw128(
                        cols_src + Cfg::kColsBytes, rows_mn ? Cfg::kBoxBytes : 16u, 1024);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j == 0 && shift && accumulate != 0) {
                            ptx::umma_f16_pair_shift<kPartShift>(d_tmem, cols_desc, rows_desc, idesc);
                        } else if (j < steps) {
                            ptx::umma_f16_pair(d_tmem, cols_desc + static_cast<uint64_t>(j * cols_step),
                                               rows_desc + static_cast<uint64_t>(j * rows_step), idesc, accumulate);
                            accumulate = 1;
                        }
                        if (j == 0) {
                            ready = ptx::mbar_try_wait(full_bar(stage + 1 == kStages ? 0 : stage + 1),
                                                       stage + 1 == kStages ? phase ^ 1u : phase);
                        }
                    }
                    ptx::umma_commit_pair_both(empty_bar(stage));
                    ++it;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    return true;
                };
                ok = detail::for_blocks<kExt>(
                    p, table, t, ext_blocks, 0, 0x7fffffff,
                    [&](int, int, const detail::Span&, int eb, bool first) {
                        return block(min(4, (p.ext_cols - eb * 64) / 16), true, shifts && first);
                    },
                    [&](int kb) { return block(4, gather || (wgrad && t.valid - kb * 64 < 64), false); });
                if (ok) {
                    if (accumulate != 0) {
                        ptx::umma_commit_pair_both(acc_full_bar(acc));
                    } else {  // nothing to sum: the epilogue uses zeros
                        ptx::mbar_arrive(acc_full_bar(acc));
                        ptx::mbar_arrive_cluster(ptx::map_to_cta(acc_full_bar(acc), 1));
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
                ptx::umma_commit_pair(drain_bar);
                detail::drain_wait(drain_bar, 0);
            }
        }
        __syncwarp();
    } else if (warp == Cfg::kScheduler) {
        if (ptx::elect_one_sync()) {
            uint32_t i = 0;
            detail::PairTile t;
            bool ok = true;
            for (int tile = unit; ok && tile < total; tile += units, ++i) {
                t = detail::pair_tile(p, table, tile);
                ok = queue.push(i, t, ctl);
            }
            t.group = -1;  // no more
            if (ok) {
                queue.push(i, t, ctl);
            }
        }
        __syncwarp();
    } else if (warp >= Cfg::kFirstLoader) {
        // Loaders, one warp per stage as in the single-CTA kernel; a stage is handed to the leader.
        const detail::Loader<8> load(ring + static_cast<uint32_t>(warp - Cfg::kFirstLoader) * Cfg::kStageBytes, lane);
        const int own = warp - Cfg::kFirstLoader;
        uint32_t it = 0;     // blocks so far, whoever owns their stage
        uint32_t phase = 0;  // of the own stage
        bool ok = true;
        auto acquire = [&]() -> bool {  // (see the single-CTA kernel)
            const bool got = detail::wait_barrier(gather ? empty_bar(own) : wanted_bar(own), gather ? phase ^ 1u : phase,
                                                  ctl, kRoleProducer, 0x20000000u | it);
            phase ^= 1u;
            return __all_sync(0xFFFFFFFFu, got) != 0;
        };
        auto hand_over = [&]() {
            load.finish();
            if (lane == 0) {
                // The stage lies in this CTA's shared memory, the thread that issues its MMAs may be the
                // other CTA's.
                ptx::mbar_arrive_cluster_publish(ptx::map_to_cta(loaded_bar(own), 0));
            }
        };
        detail::PairTile t;
        for (uint32_t i = 0; loads && ok && queue.pop(i, &t, ctl, true, lane); ++i) {
            const int first_row = static_cast<int>(rank) * t.half;  // of this CTA, in the tile
            if (!wgrad) {
                const int rows = max(0, min(t.half, t.valid - first_row));  // of this CTA that exist
                int src[4] = {-1, -1, -1, -1};  // lane l: rows l, 32 + l, 64 + l, 96 + l of A, -1: none
                if (gather) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = q * 32 + static_cast<int>(lane);
                        const int at = r >= rows             ? -1
                                       : p.a_rows != nullptr ? ptx::ld_global(p.a_rows + t.p0 + first_row + r)
                                                             : t.p0 + first_row + r;
                        src[q] = at < p.a_count ? at : -1;
                    }
                }
                ok = detail::for_blocks<kExt>(
                    p, table, t, ext_blocks, 0, 0x7fffffff,
                    [&](int part, int, const detail::Span& span, int eb, bool) -> bool {
                        if (static_cast<int>(it++ % kStages) != own) {
                            return true;
                        }
                        if (!acquire()) {
                            return false;
                        }
                        load.adapter_rows(Cfg::kColsBytes, p, t.p0 + first_row, rows, span.lo, span.hi, part, eb * 64);
                        hand_over();
                        return true;
                    },
                    [&](int kb) -> bool {
                        const bool mine = gather && static_cast<int>(it % kStages) == own;
                        ++it;
                        if (!mine) {
                            return true;
                        }
                        if (!acquire()) {
                            return false;
                        }
                        load.rows128(Cfg::kColsBytes, p.a, p.lda, src, rows, kb * 64, p.k);
                        hand_over();
                        return true;
                    });
            } else {
                const int first = (own - static_cast<int>(it % kStages) + kStages) % kStages;
                int next[2];
                auto fetch = [&](int kb) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int r = kb * 64 + q * 32 + static_cast<int>(lane);
                        const int at = r >= t.valid          ? -1
                                       : p.a_rows != nullptr ? p.a_rows[t.p0 + r]
                                                             : t.p0 + r;
                        next[q] = at < p.a_count ? at : -1;
                    }
                };
                fetch(first);
                for (int kb = first; kb < t.k_blocks; kb += kStages) {
                    const int left = t.valid - kb * 64;
                    const int rows[2] = {next[0], next[1]};
                    fetch(kb + kStages);
                    if (!gather && left >= 64) {
                        continue;
                    }
                    if (!acquire()) {
                        ok = false;
                        break;
                    }
                    load.rows64(Cfg::kColsBytes, p.a, p.lda, rows, t.half / 64, t.r0 + first_row, p.m);
                    if (left < 64) {
                        int at[2];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int r = q * 32 + static_cast<int>(lane);
                            at[q] = r < left ? t.p0 + kb * 64 + r : -1;
                        }
                        load.rows64(0, p.b, p.ldb, at, 2, t.c0 + static_cast<int>(rank) * 128, p.n);
                    }
                    hand_over();
                }
                it += static_cast<uint32_t>(t.k_blocks);
            }
        }
        ptx::cp_async_wait_all();  // no copy may be in flight when the CTA ends
    } else {
        // Epilogue warps 2-5: TMEM lane quarter = warp id mod 4 = 32 columns of C.
        using T = detail::OutTraits<Elem>;
        constexpr int kVec = T::kVec;
        constexpr int kLanesPerRow = 32 / kVec;
        constexpr int kRowsPerPass = 32 / kLanesPerRow;
        const uint32_t quad = static_cast<uint32_t>(warp) & 3u;
        uint8_t* stg = staging_ptr + quad * Cfg::kWarpStaging;
        const uint32_t stg_addr = ring + kStages * Cfg::kStageBytes + quad * Cfg::kWarpStaging;
        const int sub = static_cast<int>(lane) % kLanesPerRow;
        int* row_table = reinterpret_cast<int*>(rows_ptr) + quad * 256;
        uint32_t buffer = 0;
        uint32_t count = 0;
        bool alive = true;
        detail::PairTile t;
        for (uint32_t i = 0; alive && queue.pop(i, &t, ctl, true, lane); ++i) {
            const uint32_t acc = count & 1u;
            // Scattered rows of C are looked up before the accumulator is ready (2050 x 2048 x 2048
            // scattered, one wave of tiles: 34 us with the look-up between the stores, 28 here).
            const bool scattered = !wgrad && p.c_rows != nullptr;
            if (scattered) {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int r = q * 32 + static_cast<int>(lane);
                    const int row = r < t.rows ? ptx::ld_global(p.c_rows + t.p0 + r) : -1;
                    row_table[r] = row < p.c_count ? row : -1;
                }
                __syncwarp();
            }
            const bool got =
                detail::wait_barrier(acc_full_bar(acc), (count >> 1) & 1u, ctl, kRoleEpilogue, count);
            if (!__all_sync(0xFFFFFFFFu, got)) {
                alive = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const bool nothing = t.k_blocks == 0;
            const int col0 = t.c0 + static_cast<int>(rank) * 128 + static_cast<int>(quad) * 32;
            const uint32_t t_row = tmem_base + ((quad * 32u) << 16) + acc * 256u;
            const int rows = col0 < p.n ? t.rows : 0;  // rows this warp stores
            Elem* c_base =
                static_cast<Elem*>(p.c) + (wgrad ? static_cast<long long>(t.group) * p.c_stride : 0ll);
            const float factor = p.alpha * (p.scales != nullptr ? p.scales[t.group] : 1.0f);
            const int z = wgrad ? t.group : 0;
            auto row_of = [&](int j) -> int {  // row of C behind row j of the tile, negative: none
                return j >= rows ? -1 : scattered ? row_table[j] : t.r0 + j;
            };
            bool released = false;
            auto release = [&]() {  // once, when the last accumulator column is in registers
                if (!released) {
                    released = true;
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive_cluster(ptx::map_to_cta(acc_empty_bar(acc), 0));
                    }
                }
            };
            // Whole runs of 32 consecutive rows leave by TMA, which clips at the edge of C; in a weight
            // gradient it clips rows as well.
            const bool flagged = kExt && detail::has_flagged(table, t);
            const int by_tma = p.c_tma == 0 || flagged ? 0 : wgrad ? (rows + 31) / 32 * 32 : rows / 32 * 32;
            int j0 = 0;
            if (sizeof(Elem) == 2 && p.beta == 0.0f && p.c_vec != 0 && !flagged) {
                // 64 rows at a time: the accumulator is read as matrix fragments (16 columns of C by
                // 32 rows), whose 8 x 8 blocks are stored transposed, 16 bytes = 8 columns of a row
                // each.  (Lane = column and 2-byte stores, 32 rows at a time, took the epilogue of a
                // 256 x 256 tile to 8000 cycles, twice its 6 blocks of MMAs in a weight gradient.)
                // Rows that do not leave by TMA are read back, four lanes a row, and stored one by one.
                uint32_t f[64];
                auto fetch = [&](int j) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        if (j + (h >> 1) * 32 < rows) {
                            ptx::tmem_ld_16x256b_x4(
                                t_row + (static_cast<uint32_t>(h & 1) << 20) + static_cast<uint32_t>(j + (h >> 1) * 32),
                                *reinterpret_cast<uint32_t(*)[16]>(&f[h * 16]));
                        }
                    }
                };
                if (nothing) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        f[i] = 0;
                    }
                } else if (rows > 0) {
                    fetch(0);
                }
                for (; j0 < rows; j0 += 64) {
                    ptx::tmem_ld_wait();
                    uint32_t w[32];  // [32-row run][8-row block][16-byte unit]
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int at = ((i >> 4) * 2 + ((i >> 1) & 1)) * 16 + ((i >> 2) & 3) * 4 + (i & 1) * 2;
                        w[i] = detail::pack16<Elem>(factor, f[at], f[at + 1]);
                    }
                    if (j0 + 64 >= rows) {
                        release();
                    } else if (!nothing) {
                        fetch(j0 + 64);
                    }
                    if (lane == 0) {
                        // the stores that last used the buffer have read it
                        ptx::bulk_wait_group_read<Cfg::kBuffers - 1>();
                    }
                    __syncwarp();
                    const uint32_t buf = stg_addr + buffer * Cfg::kBufferBytes;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // 64-byte swizzle: the 16-byte unit is exchanged by row bits 1 and 2
                        const uint32_t row = static_cast<uint32_t>(i & 3) * 8u + (lane & 7u);
                        ptx::stmatrix_x4_trans(
                            buf + (i >> 2) * 2048u + row * 64u + (((lane >> 3) ^ ((row >> 1) & 3u)) << 4), w[4 * i],
                            w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    }
                    if (j0 < by_tma) {
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            ptx::tma_store_3d(&tmap_c, buf, col0, t.r0 + j0, z);
                            if (j0 + 32 < by_tma) {
                                ptx::tma_store_3d(&tmap_c, buf + 2048u, col0, t.r0 + j0 + 32, z);
                            }
                        }
                    } else {
                        __syncwarp();
                    }
                    const int col = col0 + sub * kVec;
                    const int have = min(kVec, p.n - col);
#pragma unroll
                    for (int run = 0; run < 2; ++run) {
                        if (j0 + run * 32 < by_tma) {
                            continue;
                        }
                        int c_row[4];
                        uint4 v[4];
#pragma unroll
                        for (int pass = 0; pass < 4; ++pass) {
                            const int j = pass * 8 + static_cast<int>(lane >> 2);
                            c_row[pass] = have > 0 ? row_of(j0 + run * 32 + j) : -1;
                            v[pass] = *reinterpret_cast<const uint4*>(stg + buffer * Cfg::kBufferBytes + run * 2048 +
                                                                      j * 64 + ((sub ^ ((j >> 1) & 3)) << 4));
                        }
#pragma unroll
                        for (int pass = 0; pass < 4; ++pass) {
                            Elem* dst = c_base + static_cast<size_t>(max(c_row[pass], 0)) * p.ldc + col;
                            if (c_row[pass] >= 0 && have == kVec) {
                                *reinterpret_cast<uint4*>(dst) = v[pass];
                            } else if (c_row[pass] >= 0) {
                                for (int i = 0; i < have; ++i) {
                                    const uint32_t word = i < 2   ? v[pass].x
                                                          : i < 4 ? v[pass].y
                                                          : i < 6 ? v[pass].z
                                                                  : v[pass].w;
                                    reinterpret_cast<unsigned short*>(dst)[i] =
                                        static_cast<unsigned short>((i & 1) ? word >> 16 : word);
                                }
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) {
                        ptx::bulk_commit_group();  // one group per buffer, empty or not
                    }
                    buffer = buffer + 1 == Cfg::kBuffers ? 0u : buffer + 1;
                }
                j0 = rows;
            }
            // FP32 columns, and C that is read or not on 16 bytes: one column per lane.
            for (; j0 < rows; j0 += 32) {
                uint32_t r[32];
                if (nothing) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        r[i] = 0;
                    }
                } else {
                    ptx::tmem_ld_32x32(t_row + static_cast<uint32_t>(j0), r);
                    ptx::tmem_ld_wait();
                }
                if (j0 + 32 >= rows) {
                    release();
                }
                const bool run = j0 < by_tma;
                if (lane == 0) {
                    ptx::bulk_wait_group_read<Cfg::kBuffers - 1>();
                }
                __syncwarp();
                uint8_t* buf = stg + buffer * Cfg::kBufferBytes;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    // 128-byte swizzle: the 16-byte unit is exchanged by row bits 0 to 2
                    *reinterpret_cast<float*>(buf + j * 128 + (((lane >> 2) ^ (j & 7u)) << 4) + (lane & 3u) * 4u) =
                        __uint_as_float(r[j]) * (run ? factor : 1.0f);
                }
                if (run) {
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::tma_store_3d(&tmap_c, stg_addr + buffer * Cfg::kBufferBytes, col0, t.r0 + j0, z);
                    }
                } else {
                    __syncwarp();
                    const int col = col0 + sub * kVec;
                    const int have = min(kVec, p.n - col);
#pragma unroll
                    for (int pass = 0; pass < 32 / kRowsPerPass; ++pass) {
                        const int j = pass * kRowsPerPass + static_cast<int>(lane) / kLanesPerRow;
                        const int c_row = row_of(j0 + j);
                        float v[kVec];
#pragma unroll
                        for (int u = 0; u < kVec / 4; ++u) {
                            const float4 x = *reinterpret_cast<const float4*>(
                                buf + j * 128 + (((sub * (kVec / 4) + u) ^ (j & 7)) << 4));
                            v[4 * u] = x.x;
                            v[4 * u + 1] = x.y;
                            v[4 * u + 2] = x.z;
                            v[4 * u + 3] = x.w;
                        }
                        if (c_row >= 0 && have > 0) {
                            if (flagged) {
                                detail::add_adapter<Elem, kVec>(p, table, t.p0 + j0 + j, col, have, v);
                            }
                            detail::store_unit<OutT, kVec>(p, c_base, c_row, col, have, factor, v);
                        }
                    }
                    __syncwarp();
                }
                if (lane == 0) {
                    ptx::bulk_commit_group();
                }
                buffer = buffer + 1 == Cfg::kBuffers ? 0u : buffer + 1;
            }
            release();
            ++count;
        }
        if (lane == 0) {
            ptx::bulk_wait_group_read<0>();  // no store may read shared memory when the CTA ends
        }
        __syncwarp();
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive_release();
    ptx::cluster_wait_acquire();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace ckl
