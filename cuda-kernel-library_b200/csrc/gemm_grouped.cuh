// Tensor-core products whose weight is chosen per row: one tcgen05 kernel over ragged groups of
// rows.  offsets[g] .. offsets[g+1] are the positions of group g; they live on the device, so
// every CTA derives the tile schedule itself and the host never waits for them.
//
//   kFormRows   C[p] = alpha * A[row(p)] * op(B_g) for the positions p of group g (op = identity
//               or transpose); tiles of 128 positions x bn columns, never across two groups.
//   kFormWgrad  W_g = alpha * sum over p in g of A[row(p)]^T G[row(p)]: the ragged dimension is
//               the one that is summed; tiles of 128 x bn of each W_g.
//
// kFormRows may be "extended": one B for all positions (a shared projection), and for the rows of
// adapter g (offsets are then the adapters') T[p] * op(E_g) besides.
//   kExtBlocks  besides the k blocks of the product a tile runs, for each adapter whose rows it holds,
//               those of T and E_g into the same accumulator, the rows of other adapters read as
//               zeros: no second pass over C, and no tiles cut at the borders of requests (which
//               reads the shared weights again for each: 2000 rows, 30 adapters, 4096 x 4096:
//               157 us against 47 for the product alone).  Zero times an infinity or NaN in one
//               adapter would be NaN in another's rows, so an adapter whose E_g holds any
//               (ext_flags, found by ext_check_kernel) is left out there and added row by row when
//               the tile is stored.
//   kExtAdd     all adapters are added row by row, in FP32 on the CUDA cores: a split launch of few
//               rows, where 64-wide blocks that hold a rank of 16 for one or two rows each
//               outnumbered those of the product.
//
// T is kept in two 16-bit words a value (two_words), which the tensor core takes as operand-type parts:
// passes over the same blocks into the same accumulator.  BF16: the value rounded and what that left, 16
// bits.  FP16 has 40 binary orders of magnitude in all, and a gradient early in an adapter's training
// lies below them (4e-7 under incoming gradients of 1e-4: two plain FP16 parts, which end at 2^-25,
// kept 4 bits of it).  So there are three parts in units of 1, 2^-11 and 2^-22, of which a value uses
// the first two or, below 2^-14, the last two: 21 bits from 2^-25 to 65504, and 2^-46 beneath.  The
// finest pass runs first, and the first MMA of the next one takes the accumulator times 2^-11.
// (The tensor core does not normalise subnormal FP16 operands: it aligns their products as if they were
// 2^-14 and cuts the sum's lower bits accordingly; zeros cost nothing.  Measured: adding 2^-24 x 1 to a
// sum of 2^-24 loses the bits that 2^-14 x 1 does.  That is why a value below 2^-14 leaves the first
// part empty.)  FP32 words taken apart by the loaders held more bits, but one warp a stage took too
// long over them (lora, 4100 rows: 154 -> 216 us; gradients, 2050 rows: 60 -> 325).
//
// Consecutive rows arrive by boxed TMA copies.  Gathered rows arrive by cp.async from loader warps,
// one per stage, that write the same swizzled layout: TMA's own row gather (tile::gather4) took about 100
// cycles per four rows, 3300 per 128 x 64 stage against the 512 the stage's MMAs need (4096^3:
// 355 TFLOP/s gathered, 1113 boxed).  The loaders also write the zeros that masked rows need:
// rows of other adapters, and in a weight gradient the positions behind the end of a group.
//
// Operand layout in shared memory is that of the dense kernel (gemm_umma.cuh): 128-byte rows of
// 64 elements under the 128-byte swizzle.  The matrix whose reduced dimension is contiguous in
// memory is read K-major, the other one MN-major, so nothing is ever transposed in memory.
//
// Warp roles: warp 0 TMA producer, warp 1 MMA, warps 2-5 epilogue as in the dense kernel, then a
// loader warp per stage and the scheduler; two accumulators in tensor memory; every wait bounded.
#pragma once

#include "gemm_umma.cuh"

namespace ckl {

constexpr int kMaxGemmGroups = 1024;
constexpr int kMaxLoraRank = 128;

enum GroupedForm : int { kFormRows = 0, kFormWgrad = 1 };
constexpr int kExtChecks = 4;
enum ExtMode : int { kExtNone = 0, kExtBlocks = 1, kExtAdd = 2 };

// Element type of C, or an FP32 value in two words, the second `c_part_cols` columns behind the first.
template <typename T>
struct TwoPart {};
constexpr int kBf16Parts = 2, kF16Parts = 3;
constexpr int kPartShift = 11;  // FP16: a part's unit is 2^-11 of that of the part before
// kFormWgrad: the operand that is two words a value, read by the loaders (FP16) or as columns (BF16).
enum LayeredOperand : int { kLayeredNone = 0, kLayeredA = 1, kLayeredB = 2 };

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
    const void* a;       // what the loaders read: A, kFormWgrad's G, and T of the extension
    const void* b;
    const void* t;
    int lda, ldb, ldt;
    int a_count, b_count, c_count;  // rows of A, G and C that exist
    int m, n, k;         // kFormWgrad: W_g is m x n; kFormRows: k columns of A, n columns of C
    int ldc;
    float alpha, beta;
    int form;
    int trans_b;         // kFormRows: B_g is stored n x k
    int bn;              // tile columns: 64, 128 or 256
    int parts;           // passes that a two-word operand takes, else 1
    int layered;         // kFormWgrad: LayeredOperand
    int part_cols;       // columns from its first words to its second ones
    int c_part_cols;     // the same of a TwoPart C
    // Extension: offsets/groups describe the adapters.
    int ext_mode;              // ExtMode
    int ext_cols;              // columns from T's first words to its second ones (a multiple of 16)
    const uint32_t* ext_flags; // kExtBlocks: a word of kExtChecks bytes per adapter, not 0: E_g is not finite
    const void* e;             // E, `ext_rank` x n per adapter (n x ext_rank with trans_b)
    int ext_rank, lde;         // (a TwoPart C: columns from ext_rank on are written as zeros)
    long long e_stride;
    uint32_t fmt;        // operand format for the instruction descriptor
    int split;           // CTAs per tile (a split launch)
    int load_a;          // rows of A come through the loaders (gathered, or few per tile)
    int c_vec;           // 16-byte accesses to C are legal
    int c_tma;           // tmap_c describes C and nothing of it is read: whole 32-row runs are
                         // written by TMA
    unsigned long long wait_limit_ns;
    int overstate_first_stage;  // test hook, see GemmParams
};

// One product: descriptors (operands that are boxed, C) and parameters.  A launch of the single-CTA
// kernel runs one or two that do not depend on each other (blockIdx.y), as the two intermediates and
// the two weight gradients of the adapters.
struct GroupedProblem {
    CUtensorMap a_box, b_box, e_box, c;
    GroupedParams p;
};
struct GroupedProblems {
    GroupedProblem at[2];
};

// kSplit: a cluster of CTAs shares one tile of at most 128 columns and divides its blocks; the
// FP32 partial tiles meet in distributed shared memory.  For launches with fewer tiles than SMs.
// A split launch has one tile per CTA, whose partial then takes the place of the ring: six stages of
// 32 KB instead of four beside a 64 KB buffer.
template <bool kSplit>
struct GroupedConfig {
    static constexpr int kStages = kSplit ? 6 : 4;
    static constexpr uint32_t kABytes = 128 * 64 * 2;
    static constexpr uint32_t kBoxBytes = 64 * 64 * 2;
    static constexpr uint32_t kBBytes = (kSplit ? 2 : 4) * kBoxBytes;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kThreads = 192 + 32 * kStages + 32;  // one loader warp per stage, a scheduler
    static constexpr int kBuffers = 3;  // of 2 KB (32 rows x 64 bytes) per epilogue warp
    static constexpr uint32_t kStagingBytes = kSplit ? 0 : 4 * kBuffers * 2048;
    static constexpr int kNumBarriers = 4 * kStages + 5 + 8;
    static constexpr uint32_t kTableBytes = 2 * (kMaxGemmGroups + 2) * 4 + kMaxGemmGroups / 8;
    static constexpr uint32_t kQueueBytes = 4 * 64;
    static constexpr uint32_t kSmemBytes =
        kStages * kStageBytes + kStagingBytes + kTableBytes + kQueueBytes + kNumBarriers * 8 + 16 + 1024;
};
constexpr int kMaxSplit = 8;

namespace detail {

// The schedule as every role of a CTA walks it.
struct GroupedTile {
    int group;
    int p0, valid;  // first position and number of positions (kFormRows: of the tile;
                    // kFormWgrad: of the whole group, the reduced range)
    int m0, n0;     // kFormWgrad: first row of W_g; first column
    int cols;       // columns of the tile that exist
    int k_blocks;   // 64-wide blocks of the main product
    int ext_first, ext_last;  // kExtBlocks: adapters [first, last) that may have rows in the tile
    int begin, end;  // this CTA's share of the tile's blocks, in the order of for_blocks
    int finer;       // part in whose unit the share's sum ends up (FP16 passes), 0: the result's
};

struct GroupedTable {
    const int* offs;   // [groups + 1], clamped to [0, rows]
    const uint32_t* flagged;  // kExtBlocks: bit per adapter
    const int* tiles;  // [groups + 1] running count of row tiles (kFormRows)
    int segments;      // groups that are cut into tiles
    bool whole;        // one segment of all positions (extended, or no offsets)
    int n_tiles, m_tiles;
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

// Builds the table in shared memory; all threads of the CTA, warp 0 writes the running counts,
// which are complete after the caller's next __syncthreads().
__device__ __forceinline__ GroupedTable make_table(const GroupedParams& p, int* offs, int* tiles,
                                                   int tile_rows, int tile_cols, int warp, uint32_t lane,
                                                   int threads) {
    if (p.offsets != nullptr) {
        for (int g = static_cast<int>(threadIdx.x); g <= p.groups; g += threads) {
            offs[g] = min(max(p.offsets[g], 0), p.rows);
        }
    } else if (threadIdx.x == 0) {
        offs[0] = 0;
        offs[1] = p.rows;
    }
    uint32_t* flagged = reinterpret_cast<uint32_t*>(tiles + kMaxGemmGroups + 2);
    if (p.ext_mode == kExtBlocks) {
        for (int g0 = warp * 32; g0 < p.groups; g0 += threads) {
            const int g = g0 + static_cast<int>(lane);
            const uint32_t any = g < p.groups ? p.ext_flags[g] : 0u;
            const uint32_t bits = __ballot_sync(0xFFFFFFFFu, any != 0);
            if (lane == 0) {
                flagged[g0 / 32] = bits;
            }
        }
    }
    __syncthreads();
    GroupedTable t;
    t.offs = offs;
    t.flagged = flagged;
    t.tiles = tiles;
    t.whole = p.offsets == nullptr || p.ext_mode != kExtNone;
    t.segments = t.whole ? 1 : p.groups;
    t.n_tiles = (p.n + tile_cols - 1) / tile_cols;
    t.m_tiles = (p.m + tile_rows - 1) / tile_rows;
    if (warp == 0) {
        if (t.whole) {
            if (lane == 0) {
                tiles[0] = 0;
                tiles[1] = (p.rows + tile_rows - 1) / tile_rows;
            }
        } else {
            int run = 0;
            for (int g0 = 0; g0 < t.segments; g0 += 32) {
                const int g = g0 + static_cast<int>(lane);
                const int count =
                    g < t.segments ? (max(0, offs[g + 1] - offs[g]) + tile_rows - 1) / tile_rows : 0;
                int v = count;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
                    v += static_cast<int>(lane) >= d ? u : 0;
                }
                if (g < t.segments) {
                    tiles[g] = run + v - count;
                }
                run += __shfl_sync(0xFFFFFFFFu, v, 31);
            }
            if (lane == 0) {
                tiles[t.segments] = run;
            }
        }
    }
    return t;
}

__device__ __forceinline__ int total_tiles(const GroupedParams& p, const GroupedTable& t) {
    return p.form == kFormWgrad ? p.groups * t.m_tiles * t.n_tiles : t.tiles[t.segments] * t.n_tiles;
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
        o.k_blocks = ((o.valid + 63) / 64) * p.parts;
    } else {
        const int seg0 = t.whole ? 0 : t.offs[o.group];
        const int seg1 = t.whole ? p.rows : t.offs[o.group + 1];
        o.p0 = seg0 + mt * 128;
        o.valid = min(128, seg1 - o.p0);
        o.m0 = 0;
        o.k_blocks = (p.k + 63) / 64;
        if (p.ext_mode == kExtBlocks && o.p0 < t.offs[p.groups]) {
            o.ext_first = last_at_most(t.offs, p.groups, o.p0);
            o.ext_last = last_at_most(t.offs, p.groups, o.p0 + o.valid - 1) + 1;
        }
    }
    return o;
}

// Tiles travel from a scheduler thread to the CTA's roles through a short queue in shared memory:
// working out a tile takes some 2000 cycles of dependent integer work, which the roles would each
// spend between two tiles (24576 rows, 64 groups, weight gradient 2048 x 1408: 6 blocks of MMAs a
// tile).  A slot's full barrier has one arrival, its empty barrier one per role.
constexpr int kTileSlots = 4;
template <typename Tile>
struct TileQueue {
    static constexpr int kWords = (sizeof(Tile) + 15) / 16 * 4;
    static constexpr uint32_t kBytes = kTileSlots * kWords * 4;
    int4* slots;
    uint32_t bars;  // kTileSlots full barriers, then as many empty ones

    __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * static_cast<uint32_t>(s); }
    __device__ __forceinline__ uint32_t empty(int s) const {
        return bars + 8u * static_cast<uint32_t>(kTileSlots + s);
    }
    __device__ __forceinline__ void init(uint32_t roles) const {
        for (int s = 0; s < kTileSlots; ++s) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), roles);
        }
    }
    // Scheduler thread: the i-th tile of this CTA.
    __device__ __forceinline__ bool push(uint32_t i, const Tile& t, const Control& ctl) const {
        const int s = static_cast<int>(i % kTileSlots);
        if (!wait_barrier(empty(s), ((i / kTileSlots) & 1u) ^ 1u, ctl, kRoleProducer, 0x60000000u | i)) {
            return false;
        }
        union {
            Tile tile;
            int4 words[kWords / 4];
        } u;
        u.tile = t;
#pragma unroll
        for (int w = 0; w < kWords / 4; ++w) {
            slots[s * (kWords / 4) + w] = u.words[w];
        }
        ptx::mbar_arrive(full(s));
        return true;
    }
    // A role (a thread, or all lanes of a warp with `lane` 0 arriving for it).
    __device__ __forceinline__ bool pop(uint32_t i, Tile* t, const Control& ctl, bool whole_warp,
                                        uint32_t lane) const {
        const int s = static_cast<int>(i % kTileSlots);
        const bool got = wait_barrier(full(s), (i / kTileSlots) & 1u, ctl, kRoleProducer, 0x61000000u | i);
        if (whole_warp ? !__all_sync(0xFFFFFFFFu, got) : !got) {
            return false;
        }
        union {
            Tile tile;
            int4 words[kWords / 4];
        } u;
#pragma unroll
        for (int w = 0; w < kWords / 4; ++w) {
            u.words[w] = slots[s * (kWords / 4) + w];
        }
        *t = u.tile;
        if (whole_warp) {
            __syncwarp();
        }
        if (!whole_warp || lane == 0) {
            ptx::mbar_arrive(empty(s));
        }
        return t->group >= 0;
    }
};

// Positions [lo, hi) of a tile that belong to adapter g, none for an adapter that is added row by row.
struct Span {
    int lo, hi;
};
template <typename Tile>
__device__ __forceinline__ Span adapter_span(const GroupedTable& table, const Tile& t, int g) {
    const bool runs = ((table.flagged[g >> 5] >> (g & 31)) & 1u) == 0;
    return {max(table.offs[g], t.p0), runs ? min(table.offs[g + 1], t.p0 + t.valid) : t.p0};
}
// Whether the tile holds rows of an adapter that is added row by row.
template <typename Tile>
__device__ __forceinline__ bool has_flagged(const GroupedTable& table, const Tile& t) {
    for (int g = t.ext_first; g < t.ext_last; ++g) {
        if ((table.flagged[g >> 5] >> (g & 31)) & 1u) {
            return true;
        }
    }
    return false;
}

// Fills in the share of a tile's blocks that CTA `rank` of `size` runs.
__device__ __forceinline__ void take_share(const GroupedParams& p, const GroupedTable& table, GroupedTile* t,
                                           int rank, int size) {
    int pass = 0;  // blocks of one pass over the two-word operand
    for (int g = t->ext_first; g < t->ext_last; ++g) {
        const Span s = adapter_span(table, *t, g);
        pass += s.lo < s.hi ? (p.ext_cols + 63) / 64 : 0;
    }
    const int blocks = t->k_blocks + p.parts * pass;
    t->begin = static_cast<int>(static_cast<long long>(blocks) * rank / size);
    t->end = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / size);
    t->finer = 0;
    if (p.fmt == 0 && p.parts > 1 && t->begin < t->end) {
        if (p.form == kFormWgrad) {
            pass = (t->valid + 63) / 64;
        }
        for (int part = p.parts - 1; part > 0; --part) {  // the last part whose pass has not ended
            t->finer += pass > 0 && t->end <= (p.parts - part) * pass ? 1 : 0;
        }
    }
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

namespace detail {

// An FP32 value as two words of the operand type.
//   BF16  v rounded, and what that left of v.
//   FP16  from 2^-14 on the same, what was left times 2^11; below, both words of v times 2^11, and the
//         lowest bit of the second word is set (else it is 0: the nearest number of the right kind is taken,
//         at most one of its steps away).  Differences and products by 2^11 are exact.
__device__ __forceinline__ void two_words(float v, __nv_bfloat16* first, __nv_bfloat16* second) {
    *first = __float2bfloat16_rn(v);
    const float f = __bfloat162float(*first);
    *second = __float2bfloat16_rn(isinf(f) ? 0.0f : v - f);  // out of range stays infinite, inf - inf would not
}
__device__ __forceinline__ void two_words(float v, __half* first, __half* second) {
    constexpr float kUnit = static_cast<float>(1 << kPartShift), kSmallest = 1.0f / (1 << 14);
    const bool fine = fabsf(v) < kSmallest && v != 0.0f;
    const float x = fine ? v * kUnit : v;
    *first = __float2half_rn(x);
    const float f = __half2float(*first);
    const float r = isfinite(f) ? (x - f) * kUnit : 0.0f;
    const __half h = __float2half_rn(r);
    unsigned int bits = __half_as_ushort(h);
    if ((bits & 1u) != (fine ? 1u : 0u)) {
        bits += fabsf(r) >= fabsf(__half2float(h)) ? 1u : ~0u;  // (0 goes up: its magnitude is not above r's)
    }
    *second = __ushort_as_half(static_cast<unsigned short>(bits));
}
// Part `part` of pairs of values from their words (FP16).
__device__ __forceinline__ uint32_t layer_of(uint32_t first, uint32_t second, int part) {
    const uint32_t fine = (second & 0x00010001u) * 0xffffu;  // all ones in the halves that are fine
    return part == 0 ? first & ~fine : part == 1 ? (second & ~fine) | (first & fine) : second & fine;
}
__device__ __forceinline__ uint4 layer_of(const uint4& a, const uint4& b, int part) {
    return make_uint4(layer_of(a.x, b.x, part), layer_of(a.y, b.y, part), layer_of(a.z, b.z, part),
                      layer_of(a.w, b.w, part));
}

// Walks the blocks of a kFormRows tile that fall into the share [begin, end): main(kb) for those of the
// product, ext(part, adapter, span, block, first of its pass) for those of the adapters that have rows in
// the tile, `per` blocks each, one pass per part.  Either returns false to stop.
// FP16 adapters come before the product and the finest part first, because each pass shifts what was
// summed before it.  BF16 ones come behind it: an addition loses 2^-24 or so of what has been
// summed, which at the beginning is little (4096 x 4096, rank 64: twice as many results rounded the
// other way with the adapters in front).
// (Kernels for products without adapters have kAdapters off and none of this.)
template <bool kAdapters, typename Tile, typename Ext, typename Main>
__device__ __forceinline__ bool for_blocks(const GroupedParams& p, const GroupedTable& table, const Tile& t, int per,
                                           int begin, int end, Ext&& ext, Main&& main) {
    if constexpr (!kAdapters) {
        for (int kb = begin; kb < min(end, t.k_blocks); ++kb) {
            if (!main(kb)) {
                return false;
            }
        }
        return true;
    }
    int at = 0;
    const bool ext_first = p.fmt == 0;
    for (int turn = 0; turn < 2; ++turn) {
        if ((turn == 0) != ext_first) {
            for (int kb = max(0, begin - at); kb < min(t.k_blocks, end - at); ++kb) {
                if (!main(kb)) {
                    return false;
                }
            }
            at += t.k_blocks;
        } else if (t.ext_first < t.ext_last) {
            for (int part = p.parts - 1; part >= 0; --part) {
                bool first = true;
                for (int g = t.ext_first; g < t.ext_last; ++g) {
                    const Span span = adapter_span(table, t, g);
                    if (span.lo >= span.hi) {
                        continue;
                    }
                    for (int eb = max(0, begin - at); eb < min(per, end - at); ++eb) {
                        if (!ext(part, g, span, eb, first)) {
                            return false;
                        }
                        first = false;
                    }
                    at += per;
                }
            }
        }
    }
    return true;
}

// One 16-byte unit of row c_row of C: `have` of its columns exist, v holds the raw sums.
template <typename OutT, int kVec>
__device__ __forceinline__ void store_unit(const GroupedParams& p,
                                           typename GroupedStore<OutT>::Elem* c_base, int c_row, int col,
                                           int have, float factor, float (&v)[kVec]) {
    using Elem = typename GroupedStore<OutT>::Elem;
    using T = OutTraits<Elem>;
    Elem* dst = c_base + static_cast<size_t>(c_row) * p.ldc + col;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        v[i] *= factor;
    }
    if constexpr (GroupedStore<OutT>::kTwo) {
        // Columns behind the rank only fill it up: their sums are of zeros, but infinity times zero is NaN.
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            v[i] = col + i < p.ext_rank ? v[i] : 0.0f;
        }
        union {
            Elem e[kVec];
            uint4 unit;
        } first, second;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            two_words(v[i], &first.e[i], &second.e[i]);
        }
        *reinterpret_cast<uint4*>(dst) = first.unit;  // widths are multiples of 16 columns
        *reinterpret_cast<uint4*>(dst + p.c_part_cols) = second.unit;
    } else {
        const bool full = p.c_vec != 0 && have == kVec;
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

// One part of `rows` rows (a multiple of 32) of a two-word FP16 matrix, `units` 16-byte units of 8 columns
// each, into a box of 128-byte swizzled rows; rows outside [lo, hi) are zeros.  A whole warp, two, four or
// eight lanes a row, kBatch rows a lane in flight.
template <int kBatch>
__device__ __forceinline__ void store_layer(uint32_t dst, const unsigned short* from, int ld, int second, int row0,
                                            int rows, int lo, int hi, int units, int part) {
    const int lane = static_cast<int>(threadIdx.x & 31);
    const int shift = units <= 2 ? 1 : units <= 4 ? 2 : 3;
    const int unit = lane & ((1 << shift) - 1), sub = lane >> shift, step = 32 >> shift;
    const bool exists = unit < units;
    const unsigned short* base = from + (exists ? unit * 8 : 0);
    for (int j0 = sub; j0 < rows; j0 += kBatch * step) {
        uint4 a[kBatch], b[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int row = row0 + j0 + i * step;
            a[i] = b[i] = make_uint4(0, 0, 0, 0);
            if (exists && row >= lo && row < hi) {
                const unsigned short* src = base + static_cast<size_t>(row) * ld;
                a[i] = *reinterpret_cast<const uint4*>(src);
                b[i] = *reinterpret_cast<const uint4*>(src + second);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int j = j0 + i * step;
            if (exists && j < rows) {
                ptx::st_shared_16(dst + static_cast<uint32_t>((j >> 3) * 1024 + (j & 7) * 128 + ((unit ^ (j & 7)) << 4)),
                                  layer_of(a[i], b[i], part));
            }
        }
    }
    __syncwarp();
}

// Writes one stage for a loader warp.  Eight lanes copy the 128 bytes of one row (lane & 7 picks the
// 16-byte unit), four rows per instruction; a unit's place under the 128-byte swizzle depends on
// the row modulo 8.  Shuffles and copies go in batches of eight: one after the other each pair
// would cost its full latency (110 cycles).
// kBatch: rows of a two-word matrix that a lane has in flight; 4 in the split kernel, whose warps have 128
// registers a thread.
template <int kBatch>
struct Loader {
    uint32_t stage;      // shared address
    int unit, sub;       // lane & 7, lane >> 3
    uint32_t even, odd;  // offset of rows 4 i + sub inside the 1024-byte group of 8 rows, by i & 1

    __device__ __forceinline__ Loader(uint32_t stage_addr, uint32_t lane) {
        stage = stage_addr;
        unit = static_cast<int>(lane & 7u);
        sub = static_cast<int>(lane >> 3);
        even = static_cast<uint32_t>(sub) * 128u + (static_cast<uint32_t>(unit ^ sub) << 4);
        odd = static_cast<uint32_t>(sub) * 128u + 512u + (static_cast<uint32_t>(unit ^ (sub + 4)) << 4);
    }

    // The last unit of a row may hold fewer than 8 columns that exist: those are read one by one, so
    // that nothing behind the last row is touched.
    __device__ __forceinline__ void part_of_unit(uint32_t dst, const void* row, int col, int have) const {
        uint32_t w[4] = {0, 0, 0, 0};
        for (int e = 0; e < have; ++e) {
            const uint32_t v = ptx::ld_global(static_cast<const unsigned short*>(row) + col + e);
            w[0] |= e == 0 ? v : e == 1 ? v << 16 : 0u;
            w[1] |= e == 2 ? v : e == 3 ? v << 16 : 0u;
            w[2] |= e == 4 ? v : e == 5 ? v << 16 : 0u;
            w[3] |= e == 6 ? v : 0u;
        }
        ptx::st_shared_16(dst, make_uint4(w[0], w[1], w[2], w[3]));
    }

    // Columns [k0, k0 + 64) of up to 128 rows, K-major; lane l holds the indices of rows l, 32 + l,
    // 64 + l, 96 + l (-1: zeros).  Columns behind `limit` are zeros; rows behind `rows` are skipped.
    __device__ __forceinline__ void rows128(uint32_t offset, const void* from, int ld, const int (&src)[4],
                                            int rows, int k0, int limit) const {
        const int col = k0 + unit * 8;
        const bool whole = col + 8 <= limit;
        // (a unit that is not whole reads nothing here: any address will do)
        const char* base = static_cast<const char*>(from) + (whole ? static_cast<size_t>(col) * 2 : 0);
        const size_t pitch = static_cast<size_t>(ld) * 2;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q * 32 >= rows) {
                break;
            }
            int at[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                at[i] = __shfl_sync(0xFFFFFFFFu, src[q], i * 4 + sub);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ptx::cp_async_16(stage + offset + q * 4096u + (i >> 1) * 1024u + ((i & 1) ? odd : even),
                                 base + max(at[i], 0) * pitch, at[i] >= 0 && whole);
            }
        }
        if (k0 + 64 > limit && (limit & 7) != 0) {
            ptx::cp_async_wait_all();
            for (int r = 0; r < rows; r += 4) {
                const int at = __shfl_sync(
                    0xFFFFFFFFu, r < 32 ? src[0] : r < 64 ? src[1] : r < 96 ? src[2] : src[3], (r & 31) + sub);
                if (!whole && col < limit && at >= 0) {
                    part_of_unit(stage + offset + (r >> 3) * 1024u + ((r & 4) ? odd : even),
                                 static_cast<const char*>(from) + at * pitch, col, limit - col);
                }
            }
        }
    }

    // Columns [k0, k0 + 64) of one part of T behind positions pos0 ..; positions outside [lo, hi) and
    // columns behind the part are zeros.
    __device__ __forceinline__ void adapter_rows(uint32_t offset, const GroupedParams& p, int pos0, int rows,
                                                 int lo, int hi, int part, int k0) const {
        const int col = k0 + unit * 8;
        const bool exists = col < p.ext_cols;
        if (p.fmt == 0) {
            store_layer<kBatch>(stage + offset, static_cast<const unsigned short*>(p.t) + k0, p.ldt, p.ext_cols,
                                pos0, (rows + 31) / 32 * 32, lo, hi, min(8, (p.ext_cols - k0) / 8), part);
            return;
        }
        const char* base = static_cast<const char*>(p.t) +
                           (static_cast<size_t>(part) * p.ext_cols + (exists ? col : 0)) * 2;
        const size_t pitch = static_cast<size_t>(p.ldt) * 2;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q * 32 >= rows) {
                break;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pos = pos0 + q * 32 + i * 4 + sub;
                const bool take = pos >= lo && pos < hi && exists;
                ptx::cp_async_16(stage + offset + q * 4096u + (i >> 1) * 1024u + ((i & 1) ? odd : even),
                                 base + (take ? pos : 0) * pitch, take);
            }
        }
    }

    // One part of 64 rows of a two-word FP16 matrix, of which `left` exist, MN-major: `boxes` boxes of 64
    // columns from col0 on.  Columns behind the words are not written: no result reads them.
    __device__ __forceinline__ void layered64(uint32_t offset, const void* from, int ld, int row0, int left,
                                              int boxes, int col0, int part_cols, int part) const {
        for (int box = 0; box < boxes; ++box) {
            const int col = col0 + box * 64;
            store_layer<kBatch>(stage + offset + box * 8192u, static_cast<const unsigned short*>(from) + col, ld,
                                part_cols, row0, 64, row0, row0 + left, min(8, (part_cols - col) / 8), part);
        }
    }

    // 64 rows, MN-major: `boxes` boxes of 64 columns from col0 on; lane l holds the indices of rows l
    // and 32 + l (-1: zeros).  Columns behind `limit` are zeros.
    __device__ __forceinline__ void rows64(uint32_t offset, const void* from, int ld, const int (&src)[2],
                                           int boxes, int col0, int limit) const {
        const size_t pitch = static_cast<size_t>(ld) * 2;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const char* row[8];
            uint32_t exists = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = __shfl_sync(0xFFFFFFFFu, src[q], i * 4 + sub);
                exists |= at >= 0 ? 1u << i : 0u;
                row[i] = static_cast<const char*>(from) + max(at, 0) * pitch;
            }
            for (int b = 0; b < boxes; ++b) {
                const int col = col0 + b * 64 + unit * 8;
                const bool whole = col + 8 <= limit;
                const size_t skip = whole ? static_cast<size_t>(col) * 2 : 0;
                const uint32_t at = stage + offset + b * 8192u + q * 4096u;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ptx::cp_async_16(at + (i >> 1) * 1024u + ((i & 1) ? odd : even), row[i] + skip,
                                     ((exists >> i) & 1u) != 0 && whole);
                }
                if (!whole && col < limit) {
                    ptx::cp_async_wait_all();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if ((exists >> i) & 1u) {
                            part_of_unit(at + (i >> 1) * 1024u + ((i & 1) ? odd : even), row[i], col, limit - col);
                        }
                    }
                }
            }
            __syncwarp();
        }
    }

    // The copies have landed and are ordered before the tensor core's reads; one lane may arrive.
    __device__ __forceinline__ void finish() const {
        ptx::cp_async_wait_all();
        ptx::fence_proxy_async_smem();
        __syncwarp();
    }
};

// v[i] += sum over ranks of T[pos] * E_g, columns col .. of the row behind position pos; T's two
// words are put together first.  The operands are 16-bit words: BF16 is the upper half of an FP32 word.
__device__ __forceinline__ float from16(const GroupedParams& p, uint32_t word) {
    return p.fmt != 0 ? __uint_as_float(word << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(word)));
}
__device__ __forceinline__ float from_two_halves(uint32_t first, uint32_t second) {
    constexpr float kUnit = 1.0f / (1 << kPartShift);
    const float f = __half2float(__ushort_as_half(static_cast<unsigned short>(first)));
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(second)));
    return fmaf(s, kUnit, f) * ((second & 1u) != 0 ? kUnit : 1.0f);
}
template <typename Elem, int kVec>
__device__ __forceinline__ void add_adapter(const GroupedParams& p, const GroupedTable& table, int pos, int col,
                                            int have, float (&v)[kVec]) {
    if (pos >= table.offs[p.groups] || pos < table.offs[0]) {
        return;
    }
    const int g = last_at_most(table.offs, p.groups, pos);
    if (pos >= table.offs[g + 1] ||
        (p.ext_mode == kExtBlocks && ((table.flagged[g >> 5] >> (g & 31)) & 1u) == 0)) {
        return;
    }
    const unsigned short* t = static_cast<const unsigned short*>(p.t) + static_cast<size_t>(pos) * p.ldt;
    const unsigned short* e = static_cast<const unsigned short*>(p.e) + static_cast<size_t>(g) * p.e_stride;
    // eight ranks at a time: their T is one 16-byte word per part (parts are 16 ranks wide or more)
#pragma unroll 2
    for (int r0 = 0; r0 < p.ext_rank; r0 += 8) {
        const uint4 hi = *reinterpret_cast<const uint4*>(t + r0);
        const uint4 lo = *reinterpret_cast<const uint4*>(t + p.ext_cols + r0);
        const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p.fmt != 0) {
                f[2 * i] = __uint_as_float(h[i] << 16) + __uint_as_float(l[i] << 16);
                f[2 * i + 1] = __uint_as_float(h[i] & 0xffff0000u) + __uint_as_float(l[i] & 0xffff0000u);
            } else {
                f[2 * i] = from_two_halves(h[i] & 0xffffu, l[i] & 0xffffu);
                f[2 * i + 1] = from_two_halves(h[i] >> 16, l[i] >> 16);
            }
        }
        if (p.trans_b) {
            // one column's ranks are neighbours
#pragma unroll
            for (int c = 0; c < kVec; ++c) {
                if (c < have) {
                    const unsigned short* src = e + static_cast<size_t>(col + c) * p.lde + r0;
                    if (r0 + 8 <= p.ext_rank) {
                        const uint4 w = *reinterpret_cast<const uint4*>(src);
                        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[c] = fmaf(f[2 * i], from16(p, x[i] & 0xffffu), v[c]);
                            v[c] = fmaf(f[2 * i + 1], from16(p, x[i] >> 16), v[c]);
                        }
                    } else {
                        for (int i = 0; r0 + i < p.ext_rank; ++i) {
                            const float fi = i == 0 ? f[0] : i == 1 ? f[1] : i == 2 ? f[2] : i == 3 ? f[3]
                                             : i == 4 ? f[4] : i == 5 ? f[5] : f[6];
                            v[c] = fmaf(fi, from16(p, src[i]), v[c]);
                        }
                    }
                }
            }
        } else if (r0 + 8 <= p.ext_rank && have == kVec) {
            // eight loads in flight, then their sums
            uint32_t x[8][kVec / 2];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned short* src = e + static_cast<size_t>(r0 + i) * p.lde + col;
                if constexpr (kVec == 8) {
                    const uint4 w = *reinterpret_cast<const uint4*>(src);
                    x[i][0] = w.x;
                    x[i][1] = w.y;
                    x[i][2] = w.z;
                    x[i][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(src);
                    x[i][0] = w.x;
                    x[i][1] = w.y;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int c = 0; c < kVec / 2; ++c) {
                    v[2 * c] = fmaf(f[i], from16(p, x[i][c] & 0xffffu), v[2 * c]);
                    v[2 * c + 1] = fmaf(f[i], from16(p, x[i][c] >> 16), v[2 * c + 1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (r0 + i < p.ext_rank) {
                    const unsigned short* src = e + static_cast<size_t>(r0 + i) * p.lde + col;
#pragma unroll
                    for (int c = 0; c < kVec; ++c) {
                        if (c < have) {
                            v[c] = fmaf(f[i], from16(p, src[c]), v[c]);
                        }
                    }
                }
            }
        }
    }
}

// Pulls columns [col, col + cols) of one rank of the adapter of position pos into L2.
__device__ __forceinline__ void prefetch_adapter(const GroupedParams& p, const GroupedTable& table, int pos, int r,
                                                 int col, int cols) {
    if (pos >= table.offs[p.groups] || pos < table.offs[0]) {
        return;
    }
    const int g = last_at_most(table.offs, p.groups, pos);
    if (pos < table.offs[g + 1]) {
        const unsigned short* src = static_cast<const unsigned short*>(p.e) +
                                    static_cast<size_t>(g) * p.e_stride + static_cast<size_t>(r) * p.lde + col;
        for (int c = 0; c < cols; c += 64) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(src + c));
        }
    }
}

// Row of C behind row `in_tile` of a tile, -1 for none.
__device__ __forceinline__ int row_of_c(const GroupedParams& p, const GroupedTile& t, int in_tile) {
    if (p.form == kFormWgrad) {
        return t.m0 + in_tile < p.m ? t.m0 + in_tile : -1;
    }
    if (in_tile >= t.valid) {
        return -1;
    }
    const int row = p.c_rows != nullptr ? p.c_rows[t.p0 + in_tile] : t.p0 + in_tile;
    return row >= 0 && row < p.c_count ? row : -1;
}

}  // namespace detail

// kAdapters: extended products and the adapters' weight gradients.  (One kernel for these and the plain
// products held 5 % more time for the latter.)
template <typename OutT, bool kSplit, bool kAdapters>
__global__ void __launch_bounds__(GroupedConfig<kSplit>::kThreads, 1)
grouped_gemm_kernel(const __grid_constant__ GroupedProblems problems) {
    const GroupedProblem& problem = problems.at[blockIdx.y];
    const GroupedParams& p = problem.p;
    const CUtensorMap &tmap_a_box = problem.a_box, &tmap_b_box = problem.b_box;
    const CUtensorMap &tmap_e_box = problem.e_box, &tmap_c = problem.c;
    using Cfg = GroupedConfig<kSplit>;
    using Elem = typename GroupedStore<OutT>::Elem;
    constexpr bool kTwo = GroupedStore<OutT>::kTwo;
    constexpr int kStages = Cfg::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t ring = (raw_addr + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw_addr);
    uint8_t* staging_ptr = ring_ptr + kStages * Cfg::kStageBytes;
    uint8_t* table_ptr = staging_ptr + Cfg::kStagingBytes;
    uint8_t* queue_ptr = table_ptr + Cfg::kTableBytes;
    uint8_t* bars_ptr = queue_ptr + Cfg::kQueueBytes;
    const uint32_t bars =
        ring + (kStages * Cfg::kStageBytes + Cfg::kStagingBytes + Cfg::kTableBytes + Cfg::kQueueBytes);
    auto full_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(s); };
    auto empty_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(kStages + s); };
    auto acc_full_bar = [&](uint32_t a) { return bars + 8u * (2 * kStages + a); };
    auto acc_empty_bar = [&](uint32_t a) { return bars + 8u * (2 * kStages + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * kStages + 4);
    // a stage's rows written by the loaders (stages that need none never use it)
    auto loaded_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(2 * kStages + 5 + s); };
    // a stage that the loaders have to write has been acquired (where not every stage is one)
    auto wanted_bar = [&](int s) { return bars + 8u * static_cast<uint32_t>(3 * kStages + 13 + s); };
    using Queue = detail::TileQueue<detail::GroupedTile>;
    static_assert(Queue::kBytes <= Cfg::kQueueBytes && 2 * detail::kTileSlots == 8, "queue layout");
    const Queue queue = {reinterpret_cast<int4*>(queue_ptr), bars + 8u * (3 * kStages + 5)};
    const uint32_t tmem_slot = bars + 8u * Cfg::kNumBarriers;
    volatile uint32_t* tmem_slot_ptr =
        reinterpret_cast<volatile uint32_t*>(bars_ptr + 8 * Cfg::kNumBarriers);
    // the loaders work
    const bool loads = p.form == kFormWgrad || p.load_a != 0 || (kAdapters && p.ext_mode == kExtBlocks);

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
            ptx::mbar_init(loaded_bar(s), 1);
            ptx::mbar_init(wanted_bar(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            ptx::mbar_init(acc_full_bar(a), 1);
            ptx::mbar_init(acc_empty_bar(a), 4);
        }
        ptx::mbar_init(drain_bar, 1);
        queue.init(6u + (loads ? kStages : 0u));  // producer, MMA, four epilogue warps, loaders
        *ctl.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (threadIdx.x == 64) {
        ptx::prefetch_tensormap(&tmap_a_box);
        ptx::prefetch_tensormap(&tmap_b_box);
        ptx::prefetch_tensormap(&tmap_c);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    // Up to here only this CTA's own memory: the kernel before this one may still be running.
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    int* offs = reinterpret_cast<int*>(table_ptr);
    const detail::GroupedTable table = detail::make_table(p, offs, offs + kMaxGemmGroups + 2, 128, p.bn, warp,
                                                          lane, Cfg::kThreads);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_ptr;
    const int total = detail::total_tiles(p, table);
    const int ext_blocks = (p.ext_cols + 63) / 64;  // of an adapter and a part of T (kExtBlocks)
    // A split launch has one tile per cluster.
    const int rank = kSplit ? static_cast<int>(ptx::cluster_cta_rank()) : 0;
    const int size = kSplit ? p.split : 1;
    const int first_tile = static_cast<int>(blockIdx.x) / size;
    const int tile_step = kSplit ? 0x7fffffff - first_tile : static_cast<int>(gridDim.x);

    // ---- roles ------------------------------------------------------------------------------
    const bool gather_a = p.load_a != 0;
    const bool layers_a = kAdapters && p.layered == kLayeredA && p.fmt == 0;  // (load_a is set as well)
    const bool layers_b = kAdapters && p.layered == kLayeredB && p.fmt == 0;
    const bool gather_b = p.form == kFormWgrad && (p.b_rows != nullptr || layers_b);
    // kFormWgrad: the pass over the rows that block kb belongs to
    auto pass_of = [&](int kb, int row_blocks) {
        return !kAdapters || p.parts == 1 ? 0 : (kb >= row_blocks) + (kb >= 2 * row_blocks);
    };
    const bool shifts = kAdapters && p.fmt == 0 && p.parts > 1;  // each pass after the first begins with a shift
    const bool every = gather_a || gather_b;  // the loaders write a part of every block
    if (warp == 0) {
        if (ptx::elect_one_sync()) {
            // TMA producer.
            uint32_t it = 0;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            auto acquire_stage = [&](uint32_t bytes, bool wanted) -> bool {
                if (!detail::wait_barrier(empty_bar(stage), phase ^ 1u, ctl, kRoleProducer, it)) {
                    return false;
                }
                if (wanted) {
                    ptx::mbar_arrive(wanted_bar(stage));
                }
                const bool wrong = p.overstate_first_stage != 0 && it == 0 && blockIdx.x == 0;
                ptx::mbar_arrive_expect_tx(full_bar(stage), bytes + (wrong ? 16u : 0u));
                return true;
            };
            auto advance = [&]() {
                ++it;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            detail::GroupedTile t;
            for (uint32_t i = 0; ok && queue.pop(i, &t, ctl, false, lane); ++i) {
                const int boxes = (t.cols + 63) / 64;
                const uint32_t b_bytes = static_cast<uint32_t>(boxes) * Cfg::kBoxBytes;
                // 64 k rows of matrix z of a stack, k0 on, as columns n0 .. of the tile
                // (all box loops are unrolled: one thread issues them, and a rolled loop spends about
                // 100 cycles on each)
                auto load_b = [&](uint32_t dst, const CUtensorMap* map, int k0, int z) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if (b < boxes) {
                            const int col = t.n0 + b * 64;
                            ptx::tma_load_3d(dst + b * Cfg::kBoxBytes, map, full_bar(stage),
                                             p.trans_b ? k0 : col, p.trans_b ? col : k0, z);
                        }
                    }
                };
                if (p.form == kFormRows) {
                    const int group = kAdapters || table.whole ? 0 : t.group;
                    ok = detail::for_blocks<kAdapters>(
                        p, table, t, ext_blocks, t.begin, t.end,
                        [&](int, int g, const detail::Span&, int eb, bool) -> bool {
                            if (!acquire_stage(b_bytes, !every)) {
                                return false;
                            }
                            load_b(ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes + Cfg::kABytes, &tmap_e_box,
                                   eb * 64, g);
                            advance();
                            return true;
                        },
                        [&](int kb) -> bool {
                            if (!acquire_stage(b_bytes + (gather_a ? 0u : Cfg::kABytes), false)) {
                                return false;
                            }
                            const uint32_t a_dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                            if (!gather_a) {
                                // Rows behind the tile's last one belong to the next group (or lie
                                // outside A): computed with and not stored.
                                ptx::tma_load_2d(a_dst, &tmap_a_box, full_bar(stage), kb * 64, t.p0);
                            }
                            load_b(a_dst + Cfg::kABytes, &tmap_b_box, kb * 64, group);
                            advance();
                            return true;
                        });
                } else {
                    // Weight gradient: 64 positions per block, both operands MN-major.
                    const int row_blocks = (t.valid + 63) / 64;
                    const int a_boxes = (min(128, p.m - t.m0) + 63) / 64;
                    const uint32_t bytes =
                        (gather_b ? 0u : b_bytes) +
                        (gather_a ? 0u : static_cast<uint32_t>(a_boxes) * Cfg::kBoxBytes);
                    for (int kb = t.begin; kb < t.end; ++kb) {
                        const int pass = pass_of(kb, row_blocks);
                        const int at = (kb - pass * row_blocks) * 64;
                        const int far = kAdapters ? (p.parts - 1 - pass) * p.part_cols : 0;  // (BF16: the words as columns)
                        // A last block that is not whole comes through the loaders in both operands,
                        // with zeros behind the group's end (a zero in one alone would leave 0 * NaN).
                        const bool whole = t.valid - at >= 64;
                        if (!acquire_stage(whole ? bytes : 0u, !every && !whole)) {
                            ok = false;
                            break;
                        }
                        const uint32_t a_dst = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            if (whole && !gather_a && b < a_boxes) {
                                ptx::tma_load_2d(a_dst + b * Cfg::kBoxBytes, &tmap_a_box, full_bar(stage),
                                                 t.m0 + (kAdapters && p.layered == kLayeredA ? far : 0) + b * 64, t.p0 + at);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            if (whole && !gather_b && b < boxes) {
                                ptx::tma_load_3d(a_dst + Cfg::kABytes + b * Cfg::kBoxBytes, &tmap_b_box,
                                                 full_bar(stage), t.n0 + (kAdapters && p.layered == kLayeredB ? far : 0) + b * 64,
                                                 t.p0 + at, 0);
                            }
                        }
                        advance();
                    }
                }
            }
            // Tail: no copy may be in flight and no stage may still be signalled when the CTA ends.
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
            uint32_t loaded_phase = 0;  // bit s: next phase of loaded_bar(s)
            uint32_t count = 0;
            bool ready = false;  // the next stage's copies are known to have landed
            bool ok = true;
            detail::GroupedTile t;
            for (uint32_t i = 0; ok && queue.pop(i, &t, ctl, false, lane); ++i) {
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
                // `shift`: a new pass begins, what has been summed is 2^11 times finer
                auto block = [&](int steps, bool loaded, bool shift) -> bool {
                    if (!ready && !detail::wait_barrier(full_bar(stage), phase, ctl, kRoleMma, it)) {
                        return false;
                    }
                    if (loaded) {
                        if (!detail::wait_barrier(loaded_bar(stage), (loaded_phase >> stage) & 1u, ctl,
                                                  kRoleMma, 0x40000000u | it)) {
                            return false;
                        }
                        loaded_phase ^= 1u << stage;
                    }
                    const uint32_t a_src = ring + static_cast<uint32_t>(stage) * Cfg::kStageBytes;
                    const uint32_t b_src = a_src + Cfg::kABytes;
                    const uint64_t a_desc =
                        ptx::make_smem_desc_sw128(a_src, a_mn ? Cfg::kBoxBytes : 16u, 1024);
                    const uint64_t b_desc =
                        ptx::make_smem_desc_sw128(b_src, b_mn ? Cfg::kBoxBytes : 16u, 1024);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j == 0 && shift && accumulate != 0) {
                            ptx::umma_f16_shift<kPartShift>(d_tmem, a_desc, b_desc, idesc);
                        } else if (j < steps) {
                            ptx::umma_f16(d_tmem, a_desc + static_cast<uint64_t>(j * a_step),
                                          b_desc + static_cast<uint64_t>(j * b_step), idesc, accumulate);
                            accumulate = 1;
                        }
                        if (j == 0) {
                            // probed here so that its latency hides behind the MMAs
                            ready = ptx::mbar_try_wait(full_bar(stage + 1 == kStages ? 0 : stage + 1),
                                                       stage + 1 == kStages ? phase ^ 1u : phase);
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
                const int row_blocks = a_mn ? (t.valid + 63) / 64 : 0;
                ok = detail::for_blocks<kAdapters>(
                    p, table, t, ext_blocks, t.begin, t.end,
                    [&](int, int, const detail::Span&, int eb, bool first) {
                        return block(min(4, (p.ext_cols - eb * 64) / 16), true, shifts && first);
                    },
                    [&](int kb) {
                        const int in_pass = a_mn ? kb - pass_of(kb, row_blocks) * row_blocks : 0;
                        const bool tail = a_mn && (t.valid & 63) != 0 && in_pass + 1 == row_blocks;
                        return block(4, gather_a || gather_b || tail, a_mn && shifts && in_pass == 0);
                    });
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
    } else if (warp == 6 + kStages) {
        // Scheduler.
        if (ptx::elect_one_sync()) {
            uint32_t i = 0;
            detail::GroupedTile t;
            bool ok = true;
            for (int tile = first_tile; ok && tile < total; tile += tile_step, ++i) {
                t = detail::grouped_tile(p, table, tile);
                detail::take_share(p, table, &t, rank, size);
                ok = queue.push(i, t, ctl);
            }
            t.group = -1;  // no more
            if (ok) {
                queue.push(i, t, ctl);
            }
        }
        __syncwarp();
    } else if (warp >= 6) {
        // Loaders: warp 6 + s owns stage s, so all stages are in flight at once and each is handed
        // over the moment its own copies have landed (one warp for all stages, or all warps for each
        // stage, would hand over only in order and lag behind: 700 TFLOP/s at 4096^3).  Eight lanes
        // copy the 128 bytes of one row (lane & 7 picks the 16-byte unit), four rows per instruction;
        // the unit's place under the 128-byte swizzle depends on the row modulo 8.  The copies are
        // generic-proxy writes: after they have landed a proxy fence orders them before the tensor
        // core's reads, then one lane arrives.
        const int own = warp - 6;
        const detail::Loader<kSplit ? 4 : 8> load(ring + static_cast<uint32_t>(own) * Cfg::kStageBytes, lane);
        uint32_t it = 0;     // blocks of this CTA so far, whoever owns their stage
        uint32_t phase = 0;  // of the own stage
        bool ok = true;
        // A barrier tells two adjacent phases apart, no more.  Where every block is written here none can
        // be multiplied without this warp, so it sees each phase of its stage's barrier.  Where only a
        // few are, the others pass whether it looks or not: then the producer says which.
        auto acquire = [&]() -> bool {
            const bool got = detail::wait_barrier(every ? empty_bar(own) : wanted_bar(own), every ? phase ^ 1u : phase,
                                                  ctl, kRoleProducer, 0x20000000u | it);
            phase ^= 1u;
            return __all_sync(0xFFFFFFFFu, got) != 0;
        };
        auto hand_over = [&]() {
            load.finish();
            if (lane == 0) {
                ptx::mbar_arrive(loaded_bar(own));
            }
        };
        detail::GroupedTile t;
        for (uint32_t i = 0; loads && ok && queue.pop(i, &t, ctl, true, lane); ++i) {
            if (p.form == kFormRows) {
                int src[4] = {-1, -1, -1, -1};  // lane l: rows l, 32 + l, 64 + l, 96 + l of A, -1: none
                if (gather_a) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = q * 32 + static_cast<int>(lane);
                        const int at = r >= t.valid          ? -1
                                       : p.a_rows != nullptr ? p.a_rows[t.p0 + r]
                                                             : t.p0 + r;
                        src[q] = at < p.a_count ? at : -1;
                    }
                }
                ok = detail::for_blocks<kAdapters>(
                    p, table, t, ext_blocks, t.begin, t.end,
                    [&](int part, int, const detail::Span& span, int eb, bool) -> bool {
                        if (static_cast<int>(it++ % kStages) != own) {
                            return true;
                        }
                        if (!acquire()) {
                            return false;
                        }
                        load.adapter_rows(0, p, t.p0, t.valid, span.lo, span.hi, part, eb * 64);
                        hand_over();
                        return true;
                    },
                    [&](int kb) -> bool {
                        const bool mine = gather_a && static_cast<int>(it % kStages) == own;
                        ++it;
                        if (!mine) {
                            return true;
                        }
                        if (!acquire()) {
                            return false;
                        }
                        load.rows128(0, p.a, p.lda, src, t.valid, kb * 64, p.k);
                        hand_over();
                        return true;
                    });
            } else {
                const int row_blocks = (t.valid + 63) / 64;
                const int a_boxes = (min(128, p.m - t.m0) + 63) / 64;
                const int b_boxes = (t.cols + 63) / 64;
                // Rows of A and G behind this lane's positions l and 32 + l of block kb, -1 behind the
                // end of the group.
                int next_a[2], next_b[2];
                auto fetch = [&](int kb) {
                    const int i0 = (kb - pass_of(kb, row_blocks) * row_blocks) * 64;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int r = i0 + q * 32 + static_cast<int>(lane);
                        const bool in = kb < t.end && r < t.valid;
                        const int at_a = !in ? -1 : p.a_rows != nullptr ? p.a_rows[t.p0 + r] : t.p0 + r;
                        const int at_b = !in ? -1 : p.b_rows != nullptr ? p.b_rows[t.p0 + r] : t.p0 + r;
                        next_a[q] = at_a < p.a_count ? at_a : -1;
                        next_b[q] = at_b < p.b_count ? at_b : -1;
                    }
                };
                // the first block of this tile whose stage is the own one
                const int first =
                    t.begin + (own - static_cast<int>(it % kStages) + kStages) % kStages;
                fetch(first);
                for (int kb = first; kb < t.end; kb += kStages) {
                    const int pass = pass_of(kb, row_blocks);
                    const int i0 = (kb - pass * row_blocks) * 64, left = t.valid - i0;
                    const bool tail = left < 64;
                    const int part = p.parts - 1 - pass;
                    const int far_a = kAdapters && p.layered == kLayeredA ? part * p.part_cols : 0;
                    const int far_b = kAdapters && p.layered == kLayeredB ? part * p.part_cols : 0;
                    const int ra[2] = {next_a[0], next_a[1]}, rb[2] = {next_b[0], next_b[1]};
                    fetch(kb + kStages);
                    if (!every && !tail) {
                        continue;
                    }
                    if (!acquire()) {
                        ok = false;
                        break;
                    }
                    // the copies of the one operand fly while the other's words are taken apart
                    if ((gather_a || tail) && !layers_a) {
                        load.rows64(0, p.a, p.lda, ra, a_boxes, t.m0 + far_a, p.m + far_a);
                    }
                    if ((gather_b || tail) && !layers_b) {
                        load.rows64(Cfg::kABytes, p.b, p.ldb, rb, b_boxes, t.n0 + far_b, p.n + far_b);
                    }
                    if (layers_a) {
                        load.layered64(0, p.a, p.lda, t.p0 + i0, min(64, left), a_boxes, t.m0, p.part_cols, part);
                    } else if (layers_b) {
                        load.layered64(Cfg::kABytes, p.b, p.ldb, t.p0 + i0, min(64, left), b_boxes, t.n0, p.part_cols,
                                       part);
                    }
                    hand_over();
                }
                it += static_cast<uint32_t>(t.end - t.begin);
            }
        }
        ptx::cp_async_wait_all();  // no copy may be in flight when the CTA ends
    } else {
        // Epilogue: 32 columns at a time through shared memory (FP32, 32 rows x 128 B per warp),
        // so that a warp writes whole 64- or 128-byte runs of a row wherever that row lies.
        const uint32_t quad = static_cast<uint32_t>(warp) & 3u;
        uint8_t* stg = staging_ptr + quad * (Cfg::kBuffers * 2048);
        using T = detail::OutTraits<Elem>;
        constexpr int kVec = T::kVec;            // elements per 16 bytes
        constexpr int kLanesPerRow = 32 / kVec;  // 8 for FP32, 4 for 16-bit types
        constexpr int kRowsPerPass = 32 / kLanesPerRow;
        const int sub = static_cast<int>(lane) % kLanesPerRow;
        uint32_t count = 0;
        const uint32_t stg_addr = ring + kStages * Cfg::kStageBytes + quad * (Cfg::kBuffers * 2048u);
        uint32_t buffer = 0;
        bool alive = true;
        detail::GroupedTile t;
        if constexpr (kSplit && kAdapters) {
            if (p.ext_mode == kExtAdd && p.trans_b == 0 && first_tile < total) {
                // What add_adapter will read of E_g for this CTA's rows travels to L2 meanwhile.
                t = detail::grouped_tile(p, table, first_tile);
                const int mine = (t.valid - rank + size - 1) / size * p.ext_rank;
                for (int i = static_cast<int>(threadIdx.x) - 64; i < mine; i += 128) {
                    const int row = i / p.ext_rank;
                    detail::prefetch_adapter(p, table, t.p0 + row * size + rank, i - row * p.ext_rank, t.n0, t.cols);
                }
            }
        }
        for (uint32_t i = 0; alive && queue.pop(i, &t, ctl, true, lane); ++i) {
            const uint32_t acc = count & 1u;
            const uint32_t parity = (count >> 1) & 1u;
            // Row of C that lane `lane` of this warp stands for, -1 for none.
            const int in_tile = static_cast<int>(quad) * 32 + static_cast<int>(lane);
            const int my_row = detail::row_of_c(p, t, in_tile);
            Elem* c_base = static_cast<Elem*>(p.c) +
                           (p.form == kFormWgrad ? static_cast<long long>(t.group) * p.c_stride : 0ll);
            const float factor = p.alpha * (p.scales != nullptr ? p.scales[t.group] : 1.0f);
            // All lanes wait: after a wait by one lane the warp may stay split in two, and the
            // code behind it then runs several times slower.
            const bool got = detail::wait_barrier(acc_full_bar(acc), parity, ctl, kRoleEpilogue, count);
            if (!__all_sync(0xFFFFFFFFu, got)) {
                alive = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const bool nothing = t.begin == t.end;
            const bool flagged = kAdapters && !kSplit && detail::has_flagged(table, t);
            const uint32_t t_row = tmem_base + ((quad * 32u) << 16) + acc * 256u;
            // Hands the accumulator back to the MMA warp, once, when its last column is in registers.
            bool released = false;
            auto release = [&]() {
                if (!released) {
                    released = true;
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive(acc_empty_bar(acc));
                    }
                }
            };
            if constexpr (kSplit) {
                // Park the partial tile where the ring was (every block has been multiplied): 512 bytes a
                // row, the 16-byte units exchanged by the row so that the 32 rows of a store hit all
                // banks.
                const uint32_t row_addr = ring + static_cast<uint32_t>(in_tile) * 512u;
                // A share that ends in one of the finer passes is still in that pass's unit.
                const float unit = !kAdapters || t.finer == 0 ? 1.0f
                                   : t.finer == 1             ? 1.0f / (1 << kPartShift)
                                                              : 1.0f / (1 << 2 * kPartShift);
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
                        ptx::st_shared_16(row_addr + (((c0 / 4 + u) ^ lane) << 4),
                                          make_uint4(__float_as_uint(unit * __uint_as_float(r[4 * u])),
                                                     __float_as_uint(unit * __uint_as_float(r[4 * u + 1])),
                                                     __float_as_uint(unit * __uint_as_float(r[4 * u + 2])),
                                                     __float_as_uint(unit * __uint_as_float(r[4 * u + 3]))));
                    }
                }
                release();
                ++count;
                continue;
            }
            // All 32 rows of this warp are consecutive rows of C: 32-column chunks (64 or 128 bytes
            // a row) go through a swizzled buffer and out by TMA, which clips at the edge
            // of C.  Otherwise rows are written one by one.
            const bool by_tma = !kTwo && p.c_tma != 0 && !flagged &&
                                (p.form == kFormWgrad ? t.m0 + static_cast<int>(quad) * 32 < p.m
                                                      : static_cast<int>(quad) * 32 + 32 <= t.valid);
            if (by_tma) {
                constexpr uint32_t kRowBytes = 64;
                constexpr int kCols = static_cast<int>(kRowBytes / sizeof(Elem));  // per buffer
                const int row = p.form == kFormWgrad ? t.m0 + static_cast<int>(quad) * 32
                                                     : t.p0 + static_cast<int>(quad) * 32;
                const int z = p.form == kFormWgrad ? t.group : 0;
                uint32_t r[32];
                if (nothing) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        r[i] = 0;
                    }
                } else {
                    ptx::tmem_ld_32x32(t_row, r);
                }
                for (int c0 = 0; c0 < t.cols; c0 += 32) {
                    if (!nothing) {
                        ptx::tmem_ld_wait();
                    }
                    uint4 out[32 / kVec];
#pragma unroll
                    for (int u = 0; u < 32 / kVec; ++u) {
                        float v[kVec];
#pragma unroll
                        for (int e = 0; e < kVec; ++e) {
                            v[e] = factor * __uint_as_float(r[u * kVec + e]);
                        }
                        T::store_vec(reinterpret_cast<Elem*>(&out[u]), v);
                    }
                    // the next chunk's columns travel while this one is stored
                    if (c0 + 32 < t.cols) {
                        if (!nothing) {
                            ptx::tmem_ld_32x32(t_row + static_cast<uint32_t>(c0 + 32), r);
                        }
                    } else {
                        release();
                    }
#pragma unroll
                    for (int h = 0; h < 32 / kCols; ++h) {
                        if (lane == 0) {
                            // the store that last used this buffer has read it
                            ptx::bulk_wait_group_read<Cfg::kBuffers - 1>();
                        }
                        __syncwarp();
                        uint8_t* buf = stg + buffer * 2048u + lane * kRowBytes;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            // 64-byte swizzle: the 16-byte unit is exchanged by row bits 1 and 2
                            *reinterpret_cast<uint4*>(buf + ((static_cast<uint32_t>(u) ^ ((lane >> 1) & 3u))
                                                             << 4)) = out[h * 4 + u];
                        }
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            ptx::tma_store_3d(&tmap_c, stg_addr + buffer * 2048u, t.n0 + c0 + h * kCols, row, z);
                            ptx::bulk_commit_group();
                        }
                        buffer = buffer + 1 == Cfg::kBuffers ? 0u : buffer + 1;
                    }
                }
            } else {
                if (p.c_tma != 0) {
                    // the row-by-row path uses two of the buffers as one
                    if (lane == 0) {
                        ptx::bulk_wait_group_read<0>();
                    }
                    __syncwarp();
                }
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
                        if (c_row >= 0 && have > 0) {
                            if (flagged) {
                                detail::add_adapter<Elem, kVec>(
                                    p, table, t.p0 + static_cast<int>(quad) * 32 + row, col, have, v);
                            }
                            detail::store_unit<OutT, kVec>(p, c_base, c_row, col, have, factor, v);
                        }
                    }
                    __syncwarp();
                }
            }
            release();
            ++count;
        }
        if (lane == 0) {
            ptx::bulk_wait_group_read<0>();  // no store may read shared memory when the CTA ends
        }
        __syncwarp();
    }

    if constexpr (kSplit) {
        // The parts of the tile meet: row i of the tile is summed by CTA i mod size, part 0 first.
        ptx::cluster_arrive_release();
        ptx::cluster_wait_acquire();
        if (first_tile < total) {
            constexpr int kVec = detail::OutTraits<Elem>::kVec;
            constexpr int kLanesPerRow = 128 / kVec;
            constexpr int kRowsPerWarp = 32 / kLanesPerRow;
            constexpr int kWarps = Cfg::kThreads / 32;
            const detail::GroupedTile t = detail::grouped_tile(p, table, first_tile);
            const int rows = p.form == kFormWgrad ? min(128, p.m - t.m0) : t.valid;
            const int sub = static_cast<int>(lane) % kLanesPerRow;
            const int col = t.n0 + sub * kVec;
            const int have = min(kVec, t.n0 + t.cols - col);
            const float factor = p.alpha * (p.scales != nullptr ? p.scales[t.group] : 1.0f);
            Elem* c_base = static_cast<Elem*>(p.c) +
                           (p.form == kFormWgrad ? static_cast<long long>(t.group) * p.c_stride : 0ll);
            const uint32_t parts = ring;
            const bool add = kAdapters && (p.ext_mode == kExtAdd || detail::has_flagged(table, t));
            for (int i = warp * kRowsPerWarp + static_cast<int>(lane) / kLanesPerRow; i * size + rank < rows;
                 i += kWarps * kRowsPerWarp) {
                const int row = i * size + rank;
                const int c_row = detail::row_of_c(p, t, row);
                if (c_row < 0 || have <= 0) {
                    continue;
                }
                float v[kVec] = {};
                for (int q = 0; q < size; ++q) {
                    const uint32_t from =
                        ptx::map_to_cta(parts + static_cast<uint32_t>(row) * 512u, static_cast<uint32_t>(q));
#pragma unroll
                    for (int u = 0; u < kVec / 4; ++u) {
                        const float4 x = ptx::ld_cluster_16(
                            from + (((sub * (kVec / 4) + u) ^ (row & 31)) << 4));
                        v[4 * u] += x.x;
                        v[4 * u + 1] += x.y;
                        v[4 * u + 2] += x.z;
                        v[4 * u + 3] += x.w;
                    }
                }
                if (add) {
                    detail::add_adapter<Elem, kVec>(p, table, t.p0 + row, col, have, v);
                }
                detail::store_unit<OutT, kVec>(p, c_base, c_row, col, have, factor, v);
            }
        }
        // No CTA leaves while another still reads its part.
        __syncwarp();
        ptx::cluster_arrive_release();
        ptx::cluster_wait_acquire();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

// Whether E_g holds an infinity or NaN: kExtChecks CTAs per adapter, a byte each for the answer.
// Adapters without rows are not read.
// It reads beside the kernel before it on the stream, which is one of the same call: that one writes
// none of what is read here, and lets this one start only after its own wait, when everything before
// it has completed.  The reads go to L2 for that reason, and the wait comes at the end, so that
// nobody who waits for this kernel overtakes the other.
struct ExtCheckParams {
    const int* offsets;
    const unsigned short* e;
    unsigned char* flags;
    long long stride;
    int adapters, rows, cols, ld;  // of E_g as stored
    unsigned int exponent;         // all ones: 0x7f80 (BF16) or 0x7c00 (FP16)
};
constexpr int kExtCheckThreads = 1024;

namespace detail {

// Walks the 16-byte units of a matrix, `units` a row, in steps of `step` of them without a division.
// Rows are counted without a sign: a walk may take a few steps of up to `step` rows past the last one
// before it is looked at again, which from 2^31 - 4096 rows would turn a signed count negative.
struct UnitWalk {
    unsigned int r;
    int u, units, rows_per_step, units_per_step;

    __host__ __device__ UnitWalk(int first, int step, int units_in_row)
        : r(static_cast<unsigned int>(first / units_in_row)),
          u(first % units_in_row),
          units(units_in_row),
          rows_per_step(step / units_in_row),
          units_per_step(step % units_in_row) {}
    __host__ __device__ bool inside(int rows) const { return r < static_cast<unsigned int>(rows); }
    __host__ __device__ void advance() {
        r += static_cast<unsigned int>(rows_per_step);
        u += units_per_step;
        if (u >= units) {
            u -= units;
            ++r;
        }
    }
};

}  // namespace detail

__global__ void __launch_bounds__(kExtCheckThreads) ext_check_kernel(const ExtCheckParams p) {
    ptx::launch_dependents();
    const int g = static_cast<int>(blockIdx.x);
    const unsigned short* e = p.e + static_cast<size_t>(g) * p.stride;
    bool bad = false;
    if (__ldcg(p.offsets + g) < __ldcg(p.offsets + g + 1)) {
        // 16-byte units, dealt to the threads of the adapter's CTAs.
        detail::UnitWalk at(static_cast<int>(blockIdx.y) * kExtCheckThreads + static_cast<int>(threadIdx.x),
                            kExtChecks * kExtCheckThreads, (p.cols + 7) / 8);
        const unsigned int both = p.exponent * 0x10001u;
        auto odd = [&](uint32_t w) {
            const uint32_t x = (w & both) ^ both;  // a half that is zero has its exponent all ones
            return (x & 0xffffu) == 0 || (x >> 16) == 0;
        };
        while (at.inside(p.rows)) {
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = make_uint4(0, 0, 0, 0);
                if (at.inside(p.rows)) {
                    const unsigned short* src = e + static_cast<size_t>(at.r) * p.ld + at.u * 8;
                    if (at.u * 8 + 8 <= p.cols) {
                        w[i] = __ldcg(reinterpret_cast<const uint4*>(src));
                    } else {
                        for (int k = 0; at.u * 8 + k < p.cols; ++k) {
                            bad |= (__ldcg(src + k) & p.exponent) == p.exponent;
                        }
                    }
                }
                at.advance();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bad |= odd(w[i].x) || odd(w[i].y) || odd(w[i].z) || odd(w[i].w);
            }
        }
    }
    const int any = __syncthreads_or(bad);
    ptx::grid_dependency_wait();
    if (threadIdx.x == 0) {
        p.flags[g * kExtChecks + blockIdx.y] = any != 0 ? 1 : 0;
    }
}

// T of the adapters for a few rows, on the CUDA cores: one CTA per position and 32 ranks reads its
// adapter's A_g (k x 32 of it) once, at the rate of one SM's L2 port, and no tensor-core tile is
// filled with rows that do not exist (48 rows of 24 adapters, k 4096, rank 16: 10.7 us through the
// tensor cores, whose clusters wait for 16 blocks and each other).
struct LoraRowsParams {
    const int* offsets;
    const int* rows;       // or nullptr
    const float* scales;   // or nullptr
    const unsigned short* x;
    const unsigned short* a;
    unsigned short* t;
    long long a_stride;
    int adapters, m, k, rank, part_cols, ldx, lda;
};
constexpr int kLoraRowsThreads = 1024;  // k 4096, rank 16: one batch of eight loads per thread
constexpr int kLoraRanks = 32;

namespace detail {
// Whether k, k + step, ... k + 7 step all lie below `limit`, and k + 8 step can be formed where they do.
__host__ __device__ inline bool eight_steps_inside(int k, int step, int limit) { return k < limit - 7 * step; }
}  // namespace detail

template <typename T>
__global__ void __launch_bounds__(kLoraRowsThreads) lora_rows_kernel(const LoraRowsParams p) {
    using Traits = detail::OutTraits<T>;
    __shared__ int adapter;
    __shared__ float part[kLoraRowsThreads / 32][kLoraRanks];
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    const int pos = static_cast<int>(blockIdx.x);
    const int r0 = static_cast<int>(blockIdx.y) * kLoraRanks;
    if (threadIdx.x == 0) {
        adapter = -1;
    }
    __syncthreads();
    for (int g = static_cast<int>(threadIdx.x); g < p.adapters; g += kLoraRowsThreads) {
        if (min(max(p.offsets[g], 0), p.m) <= pos && pos < min(max(p.offsets[g + 1], 0), p.m)) {
            adapter = g;
        }
    }
    __syncthreads();
    const int g = adapter;
    if (g < 0) {
        return;
    }
    const int row = p.rows != nullptr ? p.rows[pos] : pos;
    const bool exists = row >= 0 && row < p.m;
    const int ranks = min(kLoraRanks, p.rank - r0);
    // 16-byte units (8 ranks) per row of A_g: 1, 2 or 4; the other lanes take further rows.
    const int shift = ranks <= 8 ? 0 : ranks <= 16 ? 1 : 2;
    const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
    const int unit = lane & ((1 << shift) - 1);
    const int step = kLoraRowsThreads >> shift;
    const T* x = reinterpret_cast<const T*>(p.x) + static_cast<size_t>(exists ? row : 0) * p.ldx;
    const T* a = reinterpret_cast<const T*>(p.a) + static_cast<size_t>(g) * p.a_stride + r0 + unit * 8;
    const int have = min(8, ranks - unit * 8);
    float acc[8] = {};
    int k = static_cast<int>(threadIdx.x) >> shift;
    if (exists && have == 8) {
        // eight loads of either operand in flight
        for (; detail::eight_steps_inside(k, step, p.k); k += 8 * step) {
            float f[8], v[8][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = Traits::load(x + k + i * step);
                Traits::load_vec(a + static_cast<size_t>(k + i * step) * p.lda, v[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    acc[c] = fmaf(f[i], v[i][c], acc[c]);
                }
            }
        }
    }
    if (exists) {
        for (; k < p.k; k += step) {
            const float f = Traits::load(x + k);
            const T* src = a + static_cast<size_t>(k) * p.lda;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i < have) {
                    acc[i] = fmaf(f, Traits::load(src + i), acc[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        for (int d = 16; d >= (1 << shift); d >>= 1) {
            acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], d);
        }
        if (lane < (1 << shift)) {
            part[warp][unit * 8 + i] = acc[i];
        }
    }
    __syncthreads();
    const int r = static_cast<int>(threadIdx.x);
    if (r < kLoraRanks && r0 + r < p.part_cols) {
        float v = 0.0f;
        if (r < ranks) {
#pragma unroll
            for (int w = 0; w < kLoraRowsThreads / 32; ++w) {
                v += part[w][r];
            }
            v *= p.scales != nullptr ? p.scales[g] : 1.0f;
        }
        T* dst = reinterpret_cast<T*>(p.t) + static_cast<size_t>(pos) * 2 * p.part_cols + r0 + r;
        detail::two_words(v, dst, dst + p.part_cols);
    }
}

}  // namespace ckl
