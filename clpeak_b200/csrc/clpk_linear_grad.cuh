// The products of a gated feed-forward layer's backward pass as one launch of linear_kernel (included by clpk_linear.cuh).
//
//   dx = dg Wg + du Wu;   dWg = dg^T x, dWu = du^T x        (dg and du: gate_gradients_kernel)
//
//  * Operands that are contiguous along M or N instead of K: dx = dg Wg takes Wg as it lies ([K][N]), dW = dg^T x takes dg and x
//    as they lie ([K][M] and [K][N]); nothing is transposed.  A stage is then boxes of 64 elements along M or N times 64 of K, in
//    the same 128-byte swizzle; the descriptors' leading offset is the distance between two boxes, their stride that of eight rows
//    of K.
//  * dx is a sum over two pairs of operands, one K range of 2 f.
//  * The tiles of dx and those of dWg and dWu are of different length.  The longer ones come first; a cluster that has one of them
//    less gets more of the others (share_a, share_b).
//  * dx of few tokens or a narrow model has few tiles and a sum over all of 2 f, dW of a small layer few tiles and a sum over all
//    tokens.  Such a sum is cut into parts that are tiles of their own; their results go to the workspace in fp32 and
//    join_parts_kernel adds them, in the order of K, and rounds.  147 x 654 x 7749: 71 us whole, 26 in 8 parts.
#pragma once

constexpr uint32_t kMnLead = 64 * kRowBytesK;               // bytes from one box of 64 elements along M or N to the next
constexpr uint32_t kMnStep = 16 * kRowBytesK / 16;          // 16 rows of K, in the descriptor's units of 16 bytes

struct GradMaps {
    CUtensorMap dg[2], dg_t[2];                             // dg and du: boxes of 128 tokens (dx), of 64 (dW)
    CUtensorMap w[2], x;
    CUtensorMap c[3];
};

// tiles of the same length: those of dx, or those of dWg and dWu
struct GradTiles {
    uint32_t tiles, tiles_m, blocks;                        // `blocks`: of K, of all parts together
    uint32_t parts;                                         // that K is cut into; `tiles` counts each
    uint32_t products;                                      // dx, or dWg and dWu
    // of the launch
    TileOrder order;
    Divider by_product, by_parts;                           // by the tiles of a product's part, by the parts
};

struct GradParams : LinearParams {
    GradTiles first, second;
    uint32_t first_each, first_more;                        // of the first ones: what each cluster has, and how many have one more
    uint32_t share_a, share_b;                              // of the second ones, for clusters below first_more, and for the others
    uint32_t segment;                                       // K blocks of dx with dg
};

// The i-th tile of a cluster: its result (dx, dWg or dWu), its place in it, K blocks [kb0, kb1), and the rows of 256 that its
// part's results lie behind in the workspace.
__device__ __forceinline__ bool grad_tile(const GradParams &p, uint32_t cluster, uint32_t clusters, uint32_t i, LinearTile &t)
{
    const uint32_t more = p.first_more, have = p.first_each + (cluster < more ? 1 : 0);
    const GradTiles &set = i < have ? p.first : p.second;
    uint32_t tile;
    if (i < have) {
        tile = cluster + i * clusters;
    } else {
        // What clusters get that have one of the first ones less comes before what all get, so that from there on all are in step
        // and ask for the same blocks of K together: the other way round the L2 had to fetch them again (3 % at 8192 x 2048 x 8192).
        const uint32_t extra = cluster >= more ? p.share_b - p.share_a : 0, j = i - have;
        if (j < extra)
            tile = j * (clusters - more) + cluster - more;
        else if (j < extra + p.share_a)
            tile = (p.share_b - p.share_a) * (clusters - more) + (j - extra) * clusters + cluster;
        else
            return false;
        if (tile >= set.tiles)
            return false;
    }
    const uint32_t each = set.tiles_m * set.order.tiles_n, unit = divide(tile, set.by_product), part = unit >> (set.products - 1);
    t.which = set.products == 1 ? 0 : 1 + unit % 2;
    t.kb0 = divide(part * set.blocks, set.by_parts);
    t.kb1 = divide((part + 1) * set.blocks, set.by_parts);
    tile_coords(set.order, tile - unit * each, t.mb, t.nb);
    t.mb_out = part * set.tiles_m + t.mb;
    return true;
}

// a K block of a tile
__device__ __forceinline__ void grad_load(const GradMaps &maps, const GradParams &p, uint32_t which, uint8_t *blk, uint32_t kb, uint32_t row_a, uint32_t row_b,
                                          uint32_t bar)
{
    const CUtensorMap *b = &maps.x;
    if (which == 0) {
        const uint32_t o = kb >= p.segment ? 1 : 0;
        kb -= o * p.segment;
        tma_load_pair_at(blk, &maps.dg[o], (int32_t)(kb * kRowBytesK), (int32_t)row_a, bar);
        b = &maps.w[o];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 128; i += 64)
            tma_load_pair_at(blk + i * kRowBytesK, &maps.dg_t[which - 1], (int32_t)((row_a + i) * 2), (int32_t)(kb * kLinearK), bar);
    }
    for (uint32_t i = 0; i < p.tn / 2; i += 64)
        tma_load_pair_at(blk + kHalfTileBytes + i * kRowBytesK, b, (int32_t)((row_b + i) * 2), (int32_t)(kb * kLinearK), bar);
}
