// Products of rows that lie sorted by group (tokens by expert), each group with weights of its own, and their gradients.
//
//   forward    C[r] = A[r] W[e]^T              rows r of group e
//   backward   dA[r] = dC[r] W[e],  dW[e] = sum over the group's rows of dC[r]^T A[r]
//
// On CTA pairs: TMA ring, M = 256 instructions of a pair, two accumulators in tensor memory.  The side of 256 is always the side that
// is contiguous in the result: features of C, of dA or of dW's rows.  The side of N is what is ragged: a group's rows (or the
// rows of dW[e]), any multiple of 32 up to 256.  A group of one row then costs an instruction of N = 32 and loads of 16 rows, one of
// 300 two of 160, and no tile reaches into the next group's results.  In tensor memory a lane has a feature and a column a row, so
// that a warp's 32 lanes store 32 neighbours of each row, and rows that are no group's are never touched.
//
//   forward    M side: W[e], K contiguous             N side: rows of A, K contiguous
//   dA         M side: W[e]^T as it lies, M contiguous  N side: rows of dC, K contiguous
//   dW         M side: A^T as it lies, M contiguous     N side: dC^T as it lies, N contiguous; K: the group's rows
//
// dW's sums are ragged in K: the last block of 64 rows reaches into the next group.  Its loads land on a barrier of each CTA's own, a
// warp overwrites the rows behind the group with zeros -- in these layouts a row is 128 bytes of a box, whatever the swizzle -- and then
// tells the pair's barrier.
//
// Sizes of groups are known on the device alone, so every CTA makes the list of tiles for itself, before its first load: a prefix sum
// over the groups.  Tiles are dealt to the pairs in turn, so that neighbours share operands in the L2.  Where that leaves pairs idle at
// the end for longer than it costs to put sums together, the last half to one and a half rounds are cut by cost instead, also inside their
// sums, so that all pairs finish together.  A tile that several pairs have summed is finished by the one that comes last, in
// the order of K: the sums are the same in every call.
//
// Bound by tensor cores and their power where groups are long: 8 groups of 2048 rows x 8192 x 4096 bf16 690-710 us alone (1.55-1.6 PFLOPS) and
// 860 at the power limit.  By memory where they are short: 64 rows of 64 groups x 1408 x 2048 67 us, 5.5 TB/s with the launch.  Weight
// gradients of 512 rows a group have eight K blocks a tile of 256 KB: the epilogue's stores (16 groups x 4096 x 2048, both gradients, 264 us
// alone with the tensor pipe at 64 %).  The smallest call takes 5.4 us: 1 to set up, 1.3 for the list, the rest a launch, one block's way from
// memory and the result's.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <chrono>

#include "../clpk_elements.cuh"
#include "../clpk_internal.h"
#include "../clpk_pair.cuh"
#include "../clpk_ptx.cuh"

namespace clpk {

enum GroupedKind : uint32_t { kForward = 0, kRowGrad = 1, kWeightGrad = 2 };

constexpr uint32_t kGroupedMost = 1024;                         // groups
constexpr uint32_t kGroupedPairs = 74;                          // of a whole B200: the workspace's size may not depend on the card at hand
constexpr uint32_t kGroupedM = 256, kGroupedN = 256, kGroupedK = 64;
constexpr uint32_t kGroupedStages = 6, kGroupedStageBytes = 2 * kHalfTileBytes;
constexpr int kGroupedSets = 4, kGroupedEpilogueWarps = 4 * kGroupedSets;
constexpr int kGroupedZeroWarp = 2 + kGroupedEpilogueWarps;
constexpr int kGroupedThreads = 32 * (kGroupedZeroWarp + 1);
constexpr uint32_t kGroupedChunk = 32;                          // columns of an accumulator that a warp takes at a time
constexpr uint32_t kGroupedUnits = 2 * kGroupedEpilogueWarps;   // of a tile: what a warp has of it
constexpr uint32_t kGroupedCutTiles = 2 * kGroupedPairs;        // tiles that may be cut, at most
constexpr uint32_t kGroupedCutWarps = (kGroupedCutTiles + 31) / 32;
constexpr uint32_t kGroupedSlotFloats = kGroupedM * kGroupedN;
constexpr uint32_t kGroupedLeast = 6;                           // K blocks of a part; fewer stay with the pair before or behind
constexpr uint32_t kGroupedTileCost = 6;                        // what a tile takes besides its K blocks, in K blocks
// And to put one together, in its K blocks.  Cut at this estimate: one row x 4096 x 4096 16.8 us, uncut 24.4.  Uncut, and so with 16 here: 64
// groups of a row x 1408 x 2048 66.5 and 71.2 us, 8 of a row x 4096 x 4096 49.4 and 55.2, rows' gradients of 16 x 512 x 4096 x 2048 113 and
// 124.  With 24 or 32 two rows x 4096 x 4096 would gain (19.3 -> 18.3), the 16 groups lose.
constexpr uint32_t kGroupedJoinCost = 48;

constexpr uint32_t kMnLead = 64 * kRowBytesK;                   // as in clpk_linear_grad.cuh: from one box of 64 elements along M or N to the next
constexpr uint32_t kMnStep = 16 * kRowBytesK / 16;              // 16 rows of K, in the descriptor's units of 16 bytes

constexpr uint32_t kBadOffsets = 0x401u;

// Sums over rows are written group after group: `lists` of `groups` entries each, with a kind.
struct GroupedShape {
    uint32_t m, groups, lists;
    uint32_t kind[2];
    uint32_t feature_tiles[3], k_blocks[3];                     // by kind; k_blocks of dW: by group
    uint32_t dw_cols, dw_width;                                 // tiles along dW's rows, and their width
    uint32_t pairs;
};

struct GroupTiles {
    uint32_t cols, width, features, k_blocks;                   // tiles along N and their width, tiles along M
};

__host__ __device__ __forceinline__ GroupTiles group_tiles(const GroupedShape &p, uint32_t kind, uint32_t rows)
{
    if (kind == kWeightGrad)
        return {p.dw_cols, p.dw_width, p.feature_tiles[kind], rows ? (rows + kGroupedK - 1) / kGroupedK : 1};   // of none: zeros
    const uint32_t cols = (rows + kGroupedN - 1) / kGroupedN;
    return {cols, ((cols > 1 ? (rows + cols - 1) / cols : max(rows, 1u)) + 31) / 32 * 32, p.feature_tiles[kind], p.k_blocks[kind]};
}

// What a K block takes, in units of a column: loading and multiplying 256 features and `width` rows
__device__ __forceinline__ uint32_t block_cost(uint32_t width) { return 200 + width; }

// A place in the list of tiles
struct GroupedPlace {
    uint32_t tile, kb;
};

// The workspace: for each unit of a tile that may be cut, how many K blocks have been added, and by which launch; and the partial sums,
// two slots for each pair.  Whoever adds the last blocks sets the word to zero, and a word of another launch counts as zero, so that
// nothing has to be cleared in front of a launch and a captured one can be replayed.
constexpr uint64_t kGroupedPartsAt = kGroupedCutTiles * kGroupedUnits * sizeof(unsigned long long);
constexpr uint64_t kGroupedWorkspace = kGroupedPartsAt + 2ull * kGroupedPairs * kGroupedSlotFloats * 4;
constexpr uint32_t kDoneBits = 28;                              // of a word: K blocks; above them the launch
static_assert(kGroupedPartsAt % 16 == 0, "partial sums start on 16 bytes");

// ---- the products ---------------------------------------------------------------------------------------------

struct GroupedMaps {
    CUtensorMap w;                                              // forward: boxes of 128 features x 64 of K; dA: of 64 rows of K x 64 features
    CUtensorMap rows[4];                                        // of A or dC, boxes of 16, 32, 64 and 128 rows x 64 of K
    CUtensorMap a_t, dc_t;                                      // dW: boxes of 64 rows x 64 features
};

struct GroupedResult {
    void *base;
    uint64_t ld, stride;                                        // elements; `stride`: from one group's to the next (dW)
    uint32_t features;
    int type;
};

struct GroupedParams {
    GroupedShape shape;
    GroupedResult out[3];                                       // by kind
    uint32_t dw_rows;                                           // rows of dW[e]
    const int32_t *offsets;
    unsigned long long *done;
    unsigned long long launch;                                  // its number, not 0
    float *parts;
    uint32_t *status;
};

struct GroupedSmem {
    alignas(16) uint64_t full[kGroupedStages];                  // of the leader: both CTAs' loads
    uint64_t empty[kGroupedStages];
    uint64_t tail[kGroupedStages];                              // of each CTA: a last block of dW's rows
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint32_t tmem_base;
    uint32_t dealt;                                             // tiles in front of it are dealt in turn, the others cut
    GroupedPlace start[kGroupedPairs + 1];                      // of each pair among the others
    uint32_t offsets[kGroupedMost + 1];
    uint32_t first[2 * kGroupedMost + 1];                       // tile of each entry
    // while the list is made
    uint32_t warps[kGroupedThreads / 32];
    unsigned long long load[kGroupedPairs];                     // cost of what has been dealt to a pair
    unsigned long long rest[kGroupedCutTiles + 1];              // of the tiles that may be cut, one behind another
    unsigned long long begins[kGroupedPairs];
    unsigned long long warp_cost[kGroupedCutWarps], warp_most[kGroupedCutWarps];
    uint32_t warp_join[kGroupedCutWarps];
};
constexpr uint32_t kGroupedSmemBytes = kGroupedStages * kGroupedStageBytes + (uint32_t)sizeof(GroupedSmem);
static_assert(kGroupedSmemBytes <= kSmemMax, "ring, barriers and the list of groups");

// ---- the list of tiles ----------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ T warp_before(T own)                 // exclusive sum over the lanes
{
    const uint32_t lane = threadIdx.x & 31;
    T sum = own;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const T v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= (uint32_t)o)
            sum += v;
    }
    return sum - own;
}

// Sum and maximum over the lanes of numbers below 2^51, in halves of 24 and 27 bits, for the instructions that reduce a warp's
__device__ __forceinline__ unsigned long long warp_total(unsigned long long v)
{
    return ((unsigned long long)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24)) << 24) + __reduce_add_sync(0xffffffffu, (uint32_t)v & 0xFFFFFFu);
}
__device__ __forceinline__ unsigned long long warp_most(unsigned long long v)
{
    const uint32_t high = (uint32_t)(v >> 24), top = __reduce_max_sync(0xffffffffu, high);
    return ((unsigned long long)top << 24) + __reduce_max_sync(0xffffffffu, high == top ? (uint32_t)v & 0xFFFFFFu : 0);
}

__device__ __forceinline__ uint32_t entry_of(const GroupedSmem *sh, uint32_t entries, uint32_t tile)     // the last one that does not begin behind it
{
    uint32_t lo = 0, hi = entries;
#pragma unroll 1
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (sh->first[mid] <= tile)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ GroupTiles entry_tiles(const GroupedSmem *sh, const GroupedShape &p, uint32_t entry, uint32_t &kind, uint32_t &group)
{
    const uint32_t list = entry >= p.groups ? 1 : 0;
    group = entry - list * p.groups;
    kind = list ? p.kind[1] : p.kind[0];
    return group_tiles(p, kind, sh->offsets[group + 1] - sh->offsets[group]);
}

__device__ __forceinline__ unsigned long long tile_cost(const GroupTiles &g) { return (unsigned long long)(g.k_blocks + kGroupedTileCost) * block_cost(g.width); }

// All threads of a CTA; false: the offsets are none.  The code is short rather than fast: a launch meets it cold.
__device__ __forceinline__ bool list_tiles(GroupedSmem *sh, const GroupedParams &params)
{
    const GroupedShape &p = params.shape;
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5, entries = p.lists * p.groups, P = p.pairs;
    uint32_t kind, group;
    bool bad = false;
#pragma unroll 1
    for (uint32_t i = t; i <= p.groups; i += kGroupedThreads) {
        const int32_t v = params.offsets[i], before = i ? params.offsets[i - 1] : 0;
        sh->offsets[i] = (uint32_t)v;
        bad |= v < before || v < 0 || (uint32_t)v > p.m;
    }
    if (t < kGroupedPairs)
        sh->load[t] = 0;
    if (__syncthreads_or(bad)) {                                // nothing to walk
        if (t == 0)
            sh->dealt = 0;
        if (t <= P)
            sh->start[t] = {0, 0};
        __syncthreads();
        return false;
    }
    const uint32_t each = (entries + kGroupedThreads - 1) / kGroupedThreads, i0 = min(t * each, entries), i1 = min(i0 + each, entries);
    uint32_t own = 0;
#pragma unroll 1
    for (uint32_t i = i0; i < i1; i++) {
        const GroupTiles g = entry_tiles(sh, p, i, kind, group);
        sh->first[i] = g.cols * g.features;
        own += g.cols * g.features;
    }
    uint32_t at = warp_before(own);
    if (lane == 31)
        sh->warps[warp] = at + own;
    __syncthreads();
    const uint32_t told = lane < kGroupedThreads / 32 ? sh->warps[lane] : 0, n_tiles = __reduce_add_sync(0xffffffffu, told);
    at += __reduce_add_sync(0xffffffffu, lane < warp ? told : 0);
#pragma unroll 1
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t tiles = sh->first[i];
        sh->first[i] = at;
        at += tiles;
    }
    if (t == 0)
        sh->first[entries] = n_tiles;
    __syncthreads();

    // What may be cut: half a round to one and a half, a thread for each of its tiles.
    const uint32_t whole = n_tiles >= P + P / 2 ? (n_tiles - P / 2) / P * P : 0, rest = n_tiles - whole;
    unsigned long long cost = 0;
    if (warp < kGroupedCutWarps) {
        uint32_t join = 0;
        if (t < rest) {
            const GroupTiles g = entry_tiles(sh, p, entry_of(sh, entries, whole + t), kind, group);
            cost = tile_cost(g);
            join = kGroupedJoinCost * block_cost(g.width);
        }
        const unsigned long long sum = warp_total(cost), most = warp_most(cost);
        join = __reduce_max_sync(0xffffffffu, join);
        if (lane == 0) {
            sh->warp_cost[warp] = sum;
            sh->warp_most[warp] = most;
            sh->warp_join[warp] = join;
        }
    }
    __syncthreads();
    const bool told_cut = lane < kGroupedCutWarps;
    const unsigned long long told_cost = told_cut ? sh->warp_cost[lane] : 0, total = warp_total(told_cost), most = warp_most(told_cut ? sh->warp_most[lane] : 0);
    const uint32_t join = __reduce_max_sync(0xffffffffu, told_cut ? sh->warp_join[lane] : 0);
    // dealt out: as many as a pair gets of the longest; cut: an equal share and the joining
    const bool cut = (rest + P - 1) / P * P * most > total + (unsigned long long)join * P;
    if (t == 0)
        sh->dealt = cut ? whole : n_tiles;
    if (!cut) {
        if (t <= P)
            sh->start[t] = {n_tiles, 0};
        __syncthreads();
        return true;
    }
    if (warp < kGroupedCutWarps) {
        const unsigned long long from = warp_total(lane < warp ? told_cost : 0) + warp_before(cost);
        if (t <= rest)
            sh->rest[t] = from;                                 // and the total behind the last
    }
    if (whole) {                                                // what each pair has of the others
        const uint32_t c = t % 128;
        if (c < P) {
            unsigned long long sum = 0;
#pragma unroll 1
            for (uint32_t i = t / 128; i < entries && sh->first[i] < whole; i += kGroupedThreads / 128) {
                // tiles c, c + P, ... in front of the entry's end and of its begin
                const uint32_t n = (min(sh->first[i + 1], whole) + P - 1 - c) / P - (sh->first[i] + P - 1 - c) / P;
                if (n)
                    sum += n * tile_cost(entry_tiles(sh, p, i, kind, group));
            }
            if (t < kGroupedThreads / 128 * 128)
                atomicAdd(&sh->load[c], sum);
        }
    }
    __syncthreads();
    if (warp == 0) {                                            // where the pairs begin: each fills up to one level what it has
        constexpr uint32_t kPairsEach = (kGroupedPairs + 31) / 32;
        const float all_cost = (float)total;
        unsigned long long has[kPairsEach];
        float level = 3e38f;
#pragma unroll
        for (uint32_t j = 0; j < kPairsEach; j++)
            has[j] = lane * kPairsEach + j < P ? sh->load[lane * kPairsEach + j] : ~0ull;
        uint32_t count = 0;
#pragma unroll 1
        for (int round = 0; round < 8; round++) {               // mostly two: all have about as much
            float sum = 0;
            uint32_t below = 0;
#pragma unroll
            for (uint32_t j = 0; j < kPairsEach; j++)
                if (has[j] != ~0ull && (float)has[j] < level) {
                    sum += (float)has[j];
                    below++;
                }
            below = __reduce_add_sync(0xffffffffu, below);
            if (below == count)
                break;
            count = below;
#pragma unroll
            for (int o = 16; o > 0; o /= 2)
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            level = (all_cost + sum) / (float)max(count, 1u);
        }
        // in whole numbers, so that no pair begins in front of the one before it
        const unsigned long long full = (unsigned long long)level;
        unsigned long long own_room = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPairsEach; j++)
            own_room += full > has[j] ? full - has[j] : 0;
        unsigned long long before = warp_before(own_room);
        const float all = fmaxf((float)__shfl_sync(0xffffffffu, before + own_room, 31), 1.0f);
#pragma unroll
        for (uint32_t j = 0; j < kPairsEach; j++)
            if (lane * kPairsEach + j < P) {
                sh->begins[lane * kPairsEach + j] = (unsigned long long)(all_cost * ((float)before / all));
                before += full > has[j] ? full - has[j] : 0;
            }
    }
    __syncthreads();
    if (t <= P) {
        GroupedPlace to = {t == 0 ? whole : n_tiles, 0};
        if (t > 0 && t < P && sh->begins[t] < total) {
            const unsigned long long pos = sh->begins[t];
            uint32_t lo = 0, hi = rest;
#pragma unroll 1
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (sh->rest[mid] <= pos)
                    lo = mid;
                else
                    hi = mid;
            }
            const GroupTiles g = entry_tiles(sh, p, entry_of(sh, entries, whole + lo), kind, group);
            const uint32_t blocks = (uint32_t)((pos - sh->rest[lo]) / block_cost(g.width));
            // the tile's own cost lies in front of its blocks
            to.tile = whole + lo;
            to.kb = blocks <= kGroupedTileCost ? 0 : blocks - kGroupedTileCost;
            if (to.kb < kGroupedLeast)
                to.kb = 0;
            else if (to.kb + kGroupedLeast > g.k_blocks)
                to = {to.tile + 1, 0};
        }
        sh->start[t] = to;
    }
    __syncthreads();
    return true;
}

// A tile, or the part of its sum that falls to this pair
struct GroupedTile {
    uint32_t kind, group, tile;
    uint32_t feature, row, width, rows;                         // M side; N side: first row, columns, and those of them that are the group's (or dW's)
    uint32_t k_blocks, kb0, kb1;
    uint32_t k_row, k_rows;                                     // dW: the group's rows
};

// The tiles of a pair, one after another; every role walks the same list, as a whole warp.
struct GroupedWalk {
    const GroupedParams &p;
    const GroupedSmem *sh;
    uint32_t pair, i = 0, cut = 0, entry = 0;

    __device__ __forceinline__ GroupedWalk(const GroupedParams &p, const GroupedSmem *sh, uint32_t pair) : p(p), sh(sh), pair(pair) {}

    __device__ __forceinline__ bool next(GroupedTile &t)
    {
        const GroupedShape &s = p.shape;
        uint32_t tile = pair + i * s.pairs, kb0 = 0, kb1 = 0xFFFFFFFFu;
        if (tile >= sh->dealt) {
            const GroupedPlace from = sh->start[pair], to = sh->start[pair + 1];
            tile = from.tile + cut;
            kb0 = cut == 0 ? from.kb : 0;
            if (tile > to.tile || (tile == to.tile && kb0 >= to.kb))
                return false;
            if (tile == to.tile)
                kb1 = to.kb;
            cut++;
        } else {
            i++;
        }
        // the last entry that does not begin behind the tile; a round of tiles may lie many groups on (1000 groups of two rows x 256 x 256:
        // 31 us, one group after another 60)
        uint32_t behind;
        do {
            const uint32_t at = entry + 1 + (threadIdx.x & 31);
            behind = __popc(__ballot_sync(0xffffffffu, at < s.lists * s.groups && sh->first[at] <= tile));
            entry += behind;
        } while (behind == 32);
        const GroupTiles g = entry_tiles(sh, s, entry, t.kind, t.group);
        const uint32_t begin = sh->offsets[t.group], rows = sh->offsets[t.group + 1] - begin;
        t.tile = tile;
        // strips of eight tiles along N, those fastest: neighbours share what they read
        uint32_t in = tile - sh->first[entry], before = 0, wide = g.cols;
        if (g.cols > 8) {                                       // a division takes longer than a small group's tile has
            before = in / (8 * g.features) * 8;
            in -= before * g.features;
            wide = min(8u, g.cols - before);
        }
        const uint32_t feature = wide > 1 ? in / wide : in, col = before + in - feature * wide;
        t.feature = feature * kGroupedM;
        t.width = g.width;
        t.k_blocks = g.k_blocks;
        t.kb0 = kb0;
        t.kb1 = min(kb1, g.k_blocks);
        t.k_row = begin;
        t.k_rows = rows;
        const uint32_t first = col * g.width, all = t.kind == kWeightGrad ? p.dw_rows : rows;
        t.rows = all > first ? min(all - first, g.width) : 0;
        t.row = t.kind == kWeightGrad ? first : begin + first;
        return true;
    }
};

// The last block of a group's rows has others behind them.
__device__ __forceinline__ bool has_tail(const GroupedTile &t) { return t.kind == kWeightGrad && t.k_blocks * kGroupedK != t.k_rows; }

__device__ __forceinline__ void tma_load_pair_3d(void *smem_dst, const CUtensorMap *tmap, int32_t x, int32_t y, int32_t z, uint32_t leader_bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// what another pair has written in this launch
__device__ __forceinline__ float4 load_told(const float4 *p)
{
    float4 v;
    asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

// K blocks to those that this launch has added so far; whether they are all
__device__ __forceinline__ bool add_blocks(unsigned long long *done, unsigned long long launch, uint32_t blocks, uint32_t all)
{
    unsigned long long old = *reinterpret_cast<volatile unsigned long long *>(done);
    while (true) {
        const unsigned long long sum = (old >> kDoneBits == launch ? old : launch << kDoneBits) + blocks;
        const bool last = (uint32_t)sum % (1u << kDoneBits) == all;
        const unsigned long long seen = atomicCAS(done, old, last ? 0ull : sum);
        if (seen == old)
            return last;
        old = seen;
    }
}

// 32 columns of 32 lanes -> rows of the result.  In 16 bits lanes 2i and 2i + 1 exchange halves of what they have of four columns, so that
// each has two neighbours of every other row: 4-byte stores, 64 bytes of a row by a warp.
template <int TYPE, bool WHOLE>
__device__ __forceinline__ void store_rows(const float (&v)[kGroupedChunk], const GroupedResult &out, uint64_t row0, uint32_t rows, uint32_t feature, int lane)
{
    if constexpr (TYPE == CLPK_DT_F32) {
        float *to = static_cast<float *>(out.base) + row0 * out.ld + feature + lane;
        if (WHOLE || feature + lane < out.features) {
#pragma unroll
            for (uint32_t j = 0; j < kGroupedChunk; j++, to += out.ld)
                if (WHOLE || j < rows)
                    *to = v[j];
        }
    } else {
        using E = Element<TYPE>;
        const uint32_t odd = lane & 1, f = feature + (lane & ~1), give = odd ? 0x5410 : 0x7632, one = odd ? 0x3254 : 0x5410, two = odd ? 0x3276 : 0x7610;
        uint16_t *to = static_cast<uint16_t *>(out.base) + (row0 + odd) * out.ld + f;
        const uint64_t step = 2 * out.ld;
        uint32_t w[kGroupedChunk / 2];                          // all before the first store: exchanges between stores that may be left out wait one by one
#pragma unroll
        for (uint32_t j = 0; j < kGroupedChunk; j += 4) {
            const uint32_t a = E::round2(v[j], v[j + 1]), b = E::round2(v[j + 2], v[j + 3]);
            const uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(a, b, give), 1);
            w[j / 2] = __byte_perm(a, got, one);
            w[j / 2 + 1] = __byte_perm(b, got, two);
        }
        if (WHOLE || f + 1 < out.features) {
#pragma unroll
            for (uint32_t j = 0; j < kGroupedChunk / 2; j++, to += step)
                if (WHOLE || 2 * j + odd < rows)
                    *reinterpret_cast<uint32_t *>(to) = w[j];
        } else if (f < out.features) {
#pragma unroll
            for (uint32_t j = 0; j < kGroupedChunk / 2; j++, to += step)
                if (2 * j + odd < rows)
                    *to = (uint16_t)w[j];
        }
    }
}

template <int DT>
__device__ __forceinline__ void store_tile_rows(const float (&v)[kGroupedChunk], const GroupedParams &p, const GroupedTile &t, uint32_t col, uint32_t lane_feature, int lane)
{
    const GroupedResult &out = p.out[t.kind];
    if (col >= t.rows || t.feature + lane_feature >= out.features)
        return;
    const uint32_t rows = t.rows - col;
    const uint64_t row = t.row + col;
    GroupedResult to = out;
    if (t.kind == kWeightGrad)
        to.base = static_cast<uint8_t *>(out.base) + t.group * out.stride * (out.type == CLPK_DT_F32 ? 4 : 2);
    const uint32_t feature = t.feature + lane_feature;
    const bool whole = rows >= kGroupedChunk && feature + 32 <= out.features;
    if (out.type == CLPK_DT_F32)
        whole ? store_rows<CLPK_DT_F32, true>(v, to, row, rows, feature, lane) : store_rows<CLPK_DT_F32, false>(v, to, row, rows, feature, lane);
    else
        whole ? store_rows<DT, true>(v, to, row, rows, feature, lane) : store_rows<DT, false>(v, to, row, rows, feature, lane);
}

template <int DT, bool BACKWARD>
__global__ void __launch_bounds__(kGroupedThreads) grouped_kernel(const __grid_constant__ GroupedMaps maps, const __grid_constant__ GroupedParams p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw;
    if (smem_u32(smem) % 1024 != 0) {                           // the swizzle's period; it is declared so
        griddep_wait();
        if (threadIdx.x == 0)
            *p.status = 0x406u;
        return;
    }
    GroupedSmem *sh = reinterpret_cast<GroupedSmem *>(smem + kGroupedStages * kGroupedStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t r = cluster_ctarank(), pair = blockIdx.x / 2;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kGroupedStages; s++) {
            mbar_init(&sh->full[s], 2);                         // the leader's producer twice, or both CTAs' warps that write zeros
            mbar_init(&sh->empty[s], 1);
            mbar_init(&sh->tail[s], 1);
        }
        for (int acc = 0; acc < 2; acc++) {
            mbar_init(&sh->tmem_full[acc], 1);
            mbar_init(&sh->tmem_empty[acc], 2 * kGroupedEpilogueWarps);
        }
        mbar_fence_init();
    }
    if (warp == 1)
        tmem_alloc<2>(&sh->tmem_base, 512);
    if (threadIdx.x == 0)
        for (uint32_t l = 0; l < p.shape.lists; l++) {
            const bool dw = p.shape.kind[l] == kWeightGrad;
            tma_prefetch_desc(dw ? &maps.a_t : &maps.w);
            tma_prefetch_desc(dw ? &maps.dc_t : &maps.rows[3]);
        }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    griddep_wait();
    griddep_launch_dependents();
    const bool good = list_tiles(sh, p);
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *p.status = good ? 0u : kBadOffsets;
    GroupedWalk walk(p, sh, pair);
    GroupedTile t;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const uint32_t full0 = cluster_addr(&sh->full[0], 0);
        uint32_t s = 0, parity = 1, issued = 0;                 // a fresh barrier's preceding phase counts as complete
        bool ok = true;
        while (ok && walk.next(t)) {
            const bool tail = has_tail(t);
            const uint32_t half = t.width / 2, feature = t.feature + r * 128;
            for (uint32_t kb = t.kb0; kb < t.kb1; kb++) {
                if (!warp_wait(&sh->empty[s], parity)) {
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x402u);
                    ok = false;
                    break;
                }
                uint8_t *const a = smem + (size_t)s * kGroupedStageBytes, *const b = a + kHalfTileBytes;
                const bool last = tail && kb + 1 == t.k_blocks;
                const uint32_t bytes = kHalfTileBytes + half * kRowBytesK;
                if (elect_one()) {
                    if (last) {
                        mbar_expect_tx(&sh->tail[s], bytes);
                    } else if (r == 0) {
                        mbar_expect_tx(&sh->full[s], 2 * bytes);
                        mbar_arrive(&sh->full[s]);
                    }
                    const uint32_t bar = full0 + 8 * s;
                    if constexpr (!BACKWARD) {
                        tma_load_pair_3d(a, &maps.w, (int32_t)(kb * kRowBytesK), (int32_t)feature, (int32_t)t.group, bar);
                    } else if (t.kind == kRowGrad) {
#pragma unroll
                        for (uint32_t i = 0; i < 128; i += 64)
                            tma_load_pair_3d(a + i * kRowBytesK, &maps.w, (int32_t)((feature + i) * 2), (int32_t)(kb * kGroupedK), (int32_t)t.group, bar);
                    } else {
                        const int32_t row = (int32_t)(t.k_row + kb * kGroupedK), xa = (int32_t)(feature * 2), xb = (int32_t)((t.row + r * half) * 2);
                        if (!last) {
                            tma_load_pair_at(a, &maps.a_t, xa, row, bar);
                            tma_load_pair_at(a + kMnLead, &maps.a_t, xa + 128, row, bar);
                            tma_load_pair_at(b, &maps.dc_t, xb, row, bar);
                            if (half > 64)
                                tma_load_pair_at(b + kMnLead, &maps.dc_t, xb + 128, row, bar);
                        } else {
                            tma_load_own(a, &maps.a_t, xa, row, &sh->tail[s]);
                            tma_load_own(a + kMnLead, &maps.a_t, xa + 128, row, &sh->tail[s]);
                            tma_load_own(b, &maps.dc_t, xb, row, &sh->tail[s]);
                            if (half > 64)
                                tma_load_own(b + kMnLead, &maps.dc_t, xb + 128, row, &sh->tail[s]);
                        }
                    }
                    if (!BACKWARD || t.kind == kRowGrad) {
                        uint32_t at = 0;
#pragma unroll
                        for (int i = 3; i >= 0; i--)
                            if (half & (16u << i)) {
                                tma_load_pair_at(b + at * kRowBytesK, &maps.rows[i], (int32_t)(kb * kRowBytesK), (int32_t)(t.row + r * half + at), bar);
                                at += 16u << i;
                            }
                    }
                }
                __syncwarp();
                issued++;
                if (++s == kGroupedStages) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
        if (r == 0)
            ring_settled(sh->full, kGroupedStages, issued);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the pair's leader) ----------------
        if (r == 0) {
            constexpr uint32_t kFmt = DT == CLPK_DT_BF16 ? kFmtBF16 : kFmtF16;
            uint32_t s = 0, parity = 0;
            bool ok = true;
            for (uint32_t i = 0; ok && walk.next(t); i++) {
                const uint32_t acc = i & 1, use = i >> 1;
                if (use > 0 && !warp_wait(&sh->tmem_empty[acc], (use - 1) & 1)) {
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x403u);
                    break;
                }
                tc_fence_after_sync();
                const uint32_t d = tmem + acc * kGroupedN;
                const bool a_mn = BACKWARD, b_mn = BACKWARD && t.kind == kWeightGrad;
                const uint32_t idesc = make_idesc(kGroupedM, t.width, kFmt, kFmt, kAccF32) | (a_mn ? kMajorA : 0u) | (b_mn ? kMajorB : 0u);
                const uint32_t a_lbo = a_mn ? kMnLead : 16, a_step = a_mn ? kMnStep : 2, b_lbo = b_mn ? kMnLead : 16, b_step = b_mn ? kMnStep : 2;
                for (uint32_t kb = t.kb0; kb < t.kb1; kb++) {
                    if (!warp_wait(&sh->full[s], parity)) {
                        if (lane == 0)
                            atomicCAS(p.status, 0u, 0x404u);
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t base = smem_u32(smem + (size_t)s * kGroupedStageBytes), s_now = s;
                    if (++s == kGroupedStages) {
                        s = 0;
                        parity ^= 1;
                    }
                    if (elect_one()) {
                        const uint64_t ad = make_smem_desc(base, a_lbo, 1024, kSwizzle128B), bd = make_smem_desc(base + kHalfTileBytes, b_lbo, 1024, kSwizzle128B);
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; kk++)
                            mma2_f16_ss(d, ad + kk * a_step, bd + kk * b_step, idesc, (kb != t.kb0 || kk != 0) ? 1u : 0u);
                        tc_commit_pair(&sh->empty[s_now], 3);
                    }
                    __syncwarp();
                }
                if (ok && elect_one())
                    tc_commit_pair(&sh->tmem_full[acc], 3);
                __syncwarp();
            }
        }
    } else if (warp < kGroupedZeroWarp) {
        // ---------------- epilogue: the warps of a lane quarter take chunks in turn ----------------
        const uint32_t q = (uint32_t)(warp & 3), set = (uint32_t)(warp - 2) >> 2;
        const uint32_t lanes = r * 128 + q * 32;                // the warp's features in the tile
        for (uint32_t i = 0; walk.next(t); i++) {
            const uint32_t acc = i & 1, use = i >> 1;
            if (!warp_wait(&sh->tmem_full[acc], use & 1)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x405u);
                break;
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem + acc * kGroupedN + ((q * 32) << 16), chunks = t.width / kGroupedChunk;
            const bool whole = t.kb0 == 0 && t.kb1 == t.k_blocks;
            // where the warp's sums of a chunk lie in a pair's slot: of the pair's part at its begin, or that at its end
            auto slot = [&](uint32_t of, bool at_begin, uint32_t c) {
                return reinterpret_cast<float4 *>(p.parts + (uint64_t)(2 * of + (at_begin ? 0 : 1)) * kGroupedSlotFloats + ((r * 4 + q) * kGroupedN + c * kGroupedChunk) * 32) + lane;
            };
            auto release = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster_relaxed(&sh->tmem_empty[acc], 0);
            };
            if (set >= chunks) {
                release();
                continue;
            }
            if (whole) {
                for (uint32_t c = set; c < chunks; c += kGroupedSets) {
                    float v[kGroupedChunk];
                    tmem_ld_32x32b_x32(taddr + c * kGroupedChunk, reinterpret_cast<uint32_t(&)[kGroupedChunk]>(v));
                    tmem_ld_wait();
                    if (c + kGroupedSets >= chunks)
                        release();                              // the accumulator is free as soon as it has been read
                    store_tile_rows<DT>(v, p, t, c * kGroupedChunk, lanes, lane);
                }
                continue;
            }
            // Whoever brings the last blocks adds all parts, in the order of K.  A pair that finds all others there keeps its own where they
            // are; another one writes them to its slot first.
            unsigned long long *const done = p.done + (t.tile - sh->dealt) * kGroupedUnits + (r * 4 + q) * kGroupedSets + set;
            const uint32_t blocks = t.kb1 - t.kb0;
            bool last = false, kept = false;
            if (lane == 0)
                kept = *reinterpret_cast<volatile unsigned long long *>(done) == (p.launch << kDoneBits) + (t.k_blocks - blocks);
            kept = __shfl_sync(0xffffffffu, kept, 0);
            if (!kept) {
                for (uint32_t c = set; c < chunks; c += kGroupedSets) {
                    float v[kGroupedChunk];
                    tmem_ld_32x32b_x32(taddr + c * kGroupedChunk, reinterpret_cast<uint32_t(&)[kGroupedChunk]>(v));
                    tmem_ld_wait();
                    float4 *to = slot(pair, t.kb0 > 0, c);
#pragma unroll
                    for (uint32_t j = 0; j < kGroupedChunk / 4; j++)
                        to[j * 32] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
                release();
                __threadfence();
                __syncwarp();
                if (lane == 0)
                    last = add_blocks(done, p.launch, blocks, t.k_blocks);
                if (!__shfl_sync(0xffffffffu, last, 0))
                    continue;
            } else if (lane == 0) {
                *reinterpret_cast<volatile unsigned long long *>(done) = 0;
            }
            __syncwarp();                                       // what lane 0 has seen, the others read behind it
            __threadfence();
            uint32_t begin = pair;
            while (sh->start[begin].tile == t.tile && sh->start[begin].kb > 0)
                begin--;
            for (uint32_t c = set; c < chunks; c += kGroupedSets) {
                float v[kGroupedChunk] = {};
                for (uint32_t of = begin; of < p.shape.pairs && sh->start[of].tile <= t.tile; of++) {
                    const GroupedPlace from = sh->start[of], end = sh->start[of + 1];
                    if ((from.tile == end.tile && from.kb == end.kb) || end.tile < t.tile || (end.tile == t.tile && end.kb == 0))
                        continue;                               // none, or none of this tile
                    float part[kGroupedChunk];                  // all asked for before any is waited for
                    if (kept && of == pair) {
                        tmem_ld_32x32b_x32(taddr + c * kGroupedChunk, reinterpret_cast<uint32_t(&)[kGroupedChunk]>(part));
                        tmem_ld_wait();
                    } else {
                        const float4 *at = slot(of, from.tile == t.tile && from.kb > 0, c);
#pragma unroll
                        for (uint32_t j = 0; j < kGroupedChunk / 4; j++) {
                            const float4 f = load_told(at + j * 32);
                            part[4 * j] = f.x; part[4 * j + 1] = f.y; part[4 * j + 2] = f.z; part[4 * j + 3] = f.w;
                        }
                    }
#pragma unroll
                    for (uint32_t j = 0; j < kGroupedChunk; j++)
                        v[j] += part[j];
                }
                if (kept && c + kGroupedSets >= chunks)
                    release();
                store_tile_rows<DT>(v, p, t, c * kGroupedChunk, lanes, lane);
            }
        }
    } else if (BACKWARD) {
        // ---------------- zeros behind a group's last rows ----------------
        uint32_t blocks = 0, uses = 0;                          // K blocks so far; a bit for each stage: the parity of its next tail
        const uint32_t full0 = cluster_addr(&sh->full[0], 0);
        while (walk.next(t)) {
            if (has_tail(t) && t.kb1 == t.k_blocks) {
                const uint32_t s = (blocks + (t.kb1 - t.kb0) - 1) % kGroupedStages;
                if (!warp_wait(&sh->tail[s], uses >> s & 1)) {
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x407u);
                    break;
                }
                uses ^= 1u << s;
                const uint32_t rows = t.k_rows - (t.k_blocks - 1) * kGroupedK;      // of none: zeros all
                uint8_t *const st = smem + (size_t)s * kGroupedStageBytes;
                // a row is 128 bytes of a box: eight lanes, four rows at a time
                uint8_t *const from = st + (rows + (lane >> 3)) * kRowBytesK + (lane & 7) * 16;
                for (uint32_t row = rows + (lane >> 3), at = 0; row < kGroupedK; row += 4, at += 4 * kRowBytesK) {
                    *reinterpret_cast<uint4 *>(from + at) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(from + at + kMnLead) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(from + at + 2 * kMnLead) = make_uint4(0, 0, 0, 0);
                    if (t.width > 128)
                        *reinterpret_cast<uint4 *>(from + at + 3 * kMnLead) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_remote(full0 + 8 * s);
            }
            blocks += t.kb1 - t.kb0;
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    if (warp == 1)
        tmem_dealloc<2>(tmem, 512);
}

// ---- host side ------------------------------------------------------------------------------------------------

// boxes of 128 bytes of a row times box_rows rows; of three dimensions where `groups` > 0
static int make_grouped_map(CUtensorMap *map, const void *base, uint64_t rows, uint64_t row_elems, uint64_t pitch, uint32_t box_rows, uint64_t groups = 0, uint64_t stride = 0)
{
    EncodeTiledFn enc = nullptr;
    CLPK_TRY(get_encode_fn(&enc));
    const cuuint64_t dims[3] = {row_elems * 2, rows, groups}, strides[2] = {pitch * 2, stride * 2};
    const cuuint32_t box[3] = {kRowBytesK, box_rows, 1}, estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, groups ? 3 : 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled (grouped) failed with CUresult %d", (int)r);
        return CLPK_ERR_CUDA;
    }
    return CLPK_OK;
}

static uint32_t up_div(uint64_t a, uint32_t b) { return (uint32_t)((a + b - 1) / b); }

static int run_grouped(const GroupedMaps &maps, GroupedParams &p, int dtype, bool backward, const int32_t *offsets, void *workspace, cudaStream_t s)
{
    // numbers that no other launch of this process has, and hardly one of a process before it in the same memory
    static std::atomic<unsigned long long> launches((unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() << 8);
    constexpr unsigned long long kMost = (1ull << (64 - kDoneBits)) - 1;
    p.launch = launches.fetch_add(1) % kMost + 1;
    p.offsets = offsets;
    p.done = static_cast<unsigned long long *>(workspace);
    p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kGroupedPartsAt);
    p.shape.pairs = std::max(1u, std::min(kGroupedPairs, (uint32_t)num_sms() / 2));
    const uint32_t ctas = 2 * p.shape.pairs;
    if (backward)
        return dtype == CLPK_DT_F16 ? launch_clusters(grouped_kernel<CLPK_DT_F16, true>, "grouped (gradients)", ctas, kGroupedThreads, kGroupedSmemBytes, 2, s, maps, p)
                                    : launch_clusters(grouped_kernel<CLPK_DT_BF16, true>, "grouped (gradients)", ctas, kGroupedThreads, kGroupedSmemBytes, 2, s, maps, p);
    return dtype == CLPK_DT_F16 ? launch_clusters(grouped_kernel<CLPK_DT_F16, false>, "grouped", ctas, kGroupedThreads, kGroupedSmemBytes, 2, s, maps, p)
                                : launch_clusters(grouped_kernel<CLPK_DT_BF16, false>, "grouped", ctas, kGroupedThreads, kGroupedSmemBytes, 2, s, maps, p);
}

// ---- what the calls ask of their arguments --------------------------------------------------------------------

static int check_grouped(const char *what, int dtype, int out_dtype, uint32_t m, uint32_t n, uint32_t k, uint32_t groups)
{
    CLPK_REQUIRE(dtype == CLPK_DT_BF16 || dtype == CLPK_DT_F16, "%s: dtype %d is not BF16 or F16", what, dtype);
    CLPK_REQUIRE(out_dtype == dtype || out_dtype == CLPK_DT_F32, "%s: results of type %d are neither dtype nor F32", what, out_dtype);
    CLPK_REQUIRE(n > 0 && k > 0, "%s: only the number of rows may be 0 (got %u x %u)", what, n, k);
    CLPK_REQUIRE(groups > 0 && groups <= kGroupedMost, "%s: %u groups, of 1 to %u", what, groups, kGroupedMost);
    // whole tiles and K blocks have to have 32-bit coordinates, and the tiles of both gradients a 32-bit number
    const uint64_t rows = m / kGroupedN + groups, tiles = (up_div(n, kGroupedM) + (uint64_t)up_div(k, kGroupedM)) * rows + (uint64_t)groups * up_div(k, kGroupedM) * up_div(n, 128);
    CLPK_REQUIRE(m <= 0x7FFFFE00u && n <= 0x1FFFFF00u && k <= 0x1FFFFF00u && tiles <= 1u << 30, "%s: %u x %u x %u in %u groups is too large", what, m, n, k, groups);
    return CLPK_OK;
}

// the pitch of a matrix; 0 in *ld: rows one behind another
static int check_grouped_matrix(const char *what, const char *name, const void *base, uint64_t cols, uint64_t *ld, uint64_t elem)
{
    if (*ld == 0)
        *ld = cols;
    CLPK_REQUIRE(base, "%s: %s is NULL", what, name);
    CLPK_REQUIRE(*ld >= cols && *ld < 1ull << 35, "%s: the pitch of %s, %llu, is shorter than its rows of %llu, or too large", what, name, (unsigned long long)*ld,
                 (unsigned long long)cols);
    CLPK_REQUIRE(*ld * elem % 16 == 0 && (uintptr_t)base % 16 == 0, "%s: %s must start on 16 bytes and its pitch (%llu elements of %llu bytes) be a multiple of 16 bytes",
                 what, name, (unsigned long long)*ld, (unsigned long long)elem);
    return CLPK_OK;
}

// the elements from one group's matrix to the next; 0 in *stride: one behind another
static int check_grouped_stride(const char *what, const char *name, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t *stride, uint64_t elem, uint32_t groups)
{
    if (*stride == 0 || groups == 1)
        *stride = rows * ld;
    CLPK_REQUIRE(*stride >= (rows - 1) * ld + cols && *stride < 1ull << 38, "%s: %s, %llu, is shorter than %llu rows, or too large", what, name, (unsigned long long)*stride,
                 (unsigned long long)rows);
    CLPK_REQUIRE(*stride * elem % 16 == 0, "%s: %s (%llu elements of %llu bytes) must be a multiple of 16 bytes", what, name, (unsigned long long)*stride, (unsigned long long)elem);
    return CLPK_OK;
}

static int check_grouped_rest(const char *what, const int32_t *offsets, const void *workspace, size_t bytes, const uint32_t *status)
{
    CLPK_REQUIRE(offsets && (uintptr_t)offsets % 4 == 0, "%s: d_offsets must be an array of 32-bit integers", what);
    CLPK_REQUIRE(workspace && bytes >= kGroupedWorkspace && (uintptr_t)workspace % 16 == 0, "%s: needs a 16-byte aligned workspace of %llu bytes", what,
                 (unsigned long long)kGroupedWorkspace);
    CLPK_REQUIRE(status && (uintptr_t)status % 4 == 0, "%s: d_status must be a device word", what);
    return CLPK_OK;
}

} // namespace clpk

using namespace clpk;

extern "C" {

int clpk_grouped_gemm_workspace_bytes(uint32_t groups, size_t *bytes)
{
    CLPK_REQUIRE(bytes, "bytes is NULL");
    *bytes = 0;
    CLPK_REQUIRE(groups > 0 && groups <= kGroupedMost, "clpk_grouped_gemm: %u groups, of 1 to %u", groups, kGroupedMost);
    *bytes = (size_t)kGroupedWorkspace;
    return CLPK_OK;
}

int clpk_grouped_gemm(const clpk_grouped_gemm_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_grouped_gemm";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_grouped_gemm_args_t a = *args;
    CLPK_TRY(check_grouped(what, a.dtype, a.out_dtype, a.m, a.n, a.k, a.groups));
    CLPK_TRY(check_grouped_rest(what, a.d_offsets, a.d_workspace, a.workspace_bytes, a.d_status));
    cudaStream_t s = as_stream(stream);
    if (a.m == 0) {
        CLPK_CUDA(cudaMemsetAsync(a.d_status, 0, sizeof(uint32_t), s));
        return CLPK_OK;
    }
    const uint64_t out_elem = element_bytes(a.out_dtype);
    CLPK_TRY(check_grouped_matrix(what, "d_a", a.d_a, a.k, &a.lda, 2));
    CLPK_TRY(check_grouped_matrix(what, "d_w", a.d_w, a.k, &a.ldw, 2));
    CLPK_TRY(check_grouped_stride(what, "stride_w", a.n, a.k, a.ldw, &a.stride_w, 2, a.groups));
    CLPK_TRY(check_grouped_matrix(what, "d_c", a.d_c, a.n, &a.ldc, out_elem));
    GroupedMaps maps = {};
    CLPK_TRY(make_grouped_map(&maps.w, a.d_w, a.n, a.k, a.ldw, 128, a.groups, a.stride_w));
    for (uint32_t i = 0; i < 4; i++)
        CLPK_TRY(make_grouped_map(&maps.rows[i], a.d_a, a.m, a.k, a.lda, 16u << i));
    GroupedParams p = {};
    p.shape.m = a.m;
    p.shape.groups = a.groups;
    p.shape.lists = 1;
    p.shape.kind[0] = kForward;
    p.shape.feature_tiles[kForward] = up_div(a.n, kGroupedM);
    p.shape.k_blocks[kForward] = up_div(a.k, kGroupedK);
    p.out[kForward] = {a.d_c, a.ldc, 0, a.n, a.out_dtype};
    p.status = a.d_status;
    return run_grouped(maps, p, a.dtype, false, a.d_offsets, a.d_workspace, s);
}

int clpk_grouped_gemm_backward(const clpk_grouped_gemm_backward_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_grouped_gemm_backward";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_grouped_gemm_backward_args_t a = *args;
    CLPK_TRY(check_grouped(what, a.dtype, a.dw_dtype, a.m, a.n, a.k, a.groups));
    CLPK_TRY(check_grouped_rest(what, a.d_offsets, a.d_workspace, a.workspace_bytes, a.d_status));
    const uint64_t dw_elem = element_bytes(a.dw_dtype);
    if (a.d_dw) {
        CLPK_TRY(check_grouped_matrix(what, "d_dw", a.d_dw, a.k, &a.lddw, dw_elem));
        CLPK_TRY(check_grouped_stride(what, "stride_dw", a.n, a.k, a.lddw, &a.stride_dw, dw_elem, a.groups));
    }
    cudaStream_t s = as_stream(stream);
    if (a.m == 0 || (!a.d_da && !a.d_dw)) {
        CLPK_CUDA(cudaMemsetAsync(a.d_status, 0, sizeof(uint32_t), s));
        for (uint32_t e = 0; e < a.groups && a.d_dw; e++)
            CLPK_CUDA(cudaMemset2DAsync(static_cast<uint8_t *>(a.d_dw) + e * a.stride_dw * dw_elem, a.lddw * dw_elem, 0, (size_t)a.k * dw_elem, a.n, s));
        return CLPK_OK;
    }
    CLPK_TRY(check_grouped_matrix(what, "d_dc", a.d_dc, a.n, &a.lddc, 2));
    GroupedMaps maps = {};
    GroupedParams p = {};
    p.shape.m = a.m;
    p.shape.groups = a.groups;
    p.dw_rows = a.n;
    p.status = a.d_status;
    if (a.d_da) {
        CLPK_TRY(check_grouped_matrix(what, "d_da", a.d_da, a.k, &a.ldda, 2));
        CLPK_TRY(check_grouped_matrix(what, "d_w", a.d_w, a.k, &a.ldw, 2));
        CLPK_TRY(check_grouped_stride(what, "stride_w", a.n, a.k, a.ldw, &a.stride_w, 2, a.groups));
        CLPK_TRY(make_grouped_map(&maps.w, a.d_w, a.n, a.k, a.ldw, kGroupedK, a.groups, a.stride_w));
        for (uint32_t i = 0; i < 4; i++)
            CLPK_TRY(make_grouped_map(&maps.rows[i], a.d_dc, a.m, a.n, a.lddc, 16u << i));
        p.shape.kind[p.shape.lists++] = kRowGrad;
        p.shape.feature_tiles[kRowGrad] = up_div(a.k, kGroupedM);
        p.shape.k_blocks[kRowGrad] = up_div(a.n, kGroupedK);
        p.out[kRowGrad] = {a.d_da, a.ldda, 0, a.k, a.dtype};
    }
    if (a.d_dw) {
        CLPK_TRY(check_grouped_matrix(what, "d_a", a.d_a, a.k, &a.lda, 2));
        CLPK_TRY(make_grouped_map(&maps.a_t, a.d_a, a.m, a.k, a.lda, kGroupedK));
        CLPK_TRY(make_grouped_map(&maps.dc_t, a.d_dc, a.m, a.n, a.lddc, kGroupedK));
        p.shape.kind[p.shape.lists++] = kWeightGrad;
        p.shape.feature_tiles[kWeightGrad] = up_div(a.k, kGroupedM);
        p.shape.dw_width = a.n <= 128 ? 128 : 256;              // whole boxes of 64 for each CTA
        p.shape.dw_cols = up_div(a.n, p.shape.dw_width);
        p.out[kWeightGrad] = {a.d_dw, a.lddw, a.stride_dw, a.k, a.dw_dtype};
    }
    return run_grouped(maps, p, a.dtype, true, a.d_offsets, a.d_workspace, s);
}

} // extern "C"
