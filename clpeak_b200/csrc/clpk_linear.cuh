// Products of a feed-forward layer with many tokens, on CTA pairs (included by feed_forward.cu).
//
// Same pieces as gemm_tiles_kernel -- TMA ring, M = 256 instructions of a pair, two accumulators, K over the pairs of a cluster
// -- in three forms that clpk_gemm does not have:
//
//  * kScaled: sums of 8-bit integers with scales for each token and channel and a bias in the epilogue.
//  * kGated: two products that share A in one pass.  In a pair's instruction each CTA brings half of the tile's columns of B, so
//    the leader loads Wg's rows and its peer Wu's: columns [0, tn / 2) of the accumulator are g and [tn / 2, tn) are u of the same
//    features, a thread of the epilogue holds both, and h = act(g) * u leaves without g or u having been anywhere.
//  * kGradients: the products of the backward pass (clpk_linear_grad.cuh).
//
// What bounds it.  Long sums: the tensor cores and the card's power limit.  Gated bf16 4096^3 keeps the tensor pipe busy for 94.9 % of
// the SMs' active cycles, at 1.53 GHz; 8192 x 4096 x 8192 takes 784 to 820 us in a running program, by the card (1.34 to 1.40
// PFLOPS; where it took 784 to 795, the library's plain product of that size took 800 to 813), and int8 8192^3 with scales and bias 375 to
// 393 (2.8 to 2.9 POPS), clpk_gemm's with 32-bit results 400.  A K block of a 256 x 256 tile is 512 tensor cycles: 0.28 us while half of
// the SMs work, 0.39 to 0.44 when all do.  Tiles of 512 rows, which fetch a quarter less, were 5 to 11 % slower in every form:
// tensor memory then holds one accumulator, and an epilogue with activations is too long to stand exposed.
//
// Short sums: the epilogue and the results' way to memory.  16-bit results of 4096 x 14336 x 256 leave in 35 us, and a memset of them
// takes 33; gated bf16 4096 x 128 x 14336 37 to 43 us with ReLU and 53 to 55 with SiLU, of whose two special-function results an element the
// schedulers' share is 28.  Sixteen warps do it, four on each scheduler, so that one's waits -- for tensor memory, for its box, for
// shared memory -- lie under the others' work: eight, with two boxes each, issued in a third of the cycles (66 us, ReLU 50).
#pragma once

enum LinearForm { kGated = 0, kScaled = 1, kGradients = 2 };

constexpr uint32_t kLinearMaxStages = 6;                            // of the widths there are, see linear_stages
constexpr uint32_t kLinearM = 256;
constexpr uint32_t kLinearK = 64;                                   // of 16-bit elements: 128 bytes; 128 of the 8-bit ones
constexpr uint32_t kLinearChunk = 32, kLinearPart = 16;             // columns that a warp takes in turn, and at once
constexpr int kLinearSets = 4, kLinearEpilogueWarps = 4 * kLinearSets;     // a set: a warp for each lane quarter
constexpr uint32_t kLinearBoxBytes = 2048;                          // 32 rows of 64 bytes
constexpr int kLinearThreads = 64 + 32 * kLinearEpilogueWarps;

struct LinearSmem {
    alignas(16) float cols[kLinearEpilogueWarps][32];               // a warp's scales and bias
    uint64_t full[kLinearMaxStages];
    uint64_t empty[kLinearMaxStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint32_t tmem_base;
};

// a result: h, g, u or c; dx, dWg, dWu
struct LinearResult {
    void *base;
    uint64_t ld;
    uint32_t m, n;
    uint32_t whole;                                 // columns up to the last 16 bytes that a row fills
    int type;                                       // CLPK_DT_*
};

// n / d for n < 2^31 by the multiplication of Granlund and Montgomery (1994); a division takes some 25 instructions
struct Divider {
    uint32_t mul, shift;
};
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider &d) { return (__umulhi(n, d.mul) + n) >> d.shift; }
static Divider divider(uint32_t d)
{
    uint32_t shift = 0;
    while ((1ull << shift) < d)
        shift++;
    return {(uint32_t)((((1ull << shift) - d) << 32) / d + 1), shift};
}

// Tiles are walked in groups of eight columns, M fastest inside a row of a group's.
constexpr uint32_t kLinearGroup = 8;
struct TileOrder {
    uint32_t tiles_m, tiles_n;
    Divider group, last;                            // by the tiles of a group, and by the columns of the last one where they are fewer
};
static TileOrder tile_order(uint32_t tiles_m, uint32_t tiles_n)
{
    return {tiles_m, tiles_n, divider(kLinearGroup * tiles_m), divider(std::max(tiles_n % kLinearGroup, 1u))};
}
__device__ __forceinline__ void tile_coords(const TileOrder &o, uint32_t tile, uint32_t &mb, uint32_t &nb)
{
    const uint32_t g = divide(tile, o.group), within = tile - g * kLinearGroup * o.tiles_m, first_n = g * kLinearGroup, width = o.tiles_n - first_n;
    if (width >= kLinearGroup) {
        mb = within / kLinearGroup;
        nb = first_n + within % kLinearGroup;
    } else {
        mb = divide(within, o.last);
        nb = first_n + within - mb * width;
    }
}

struct LinearParams {
    TileOrder order;
    uint32_t k_blocks;                              // of 128 bytes
    uint32_t tn, splits, stages, kps, tmem_cols;    // kps: K blocks per stage
    int activation;                                 // CLPK_ACT_*
    uint32_t keep;                                  // kGated: g and u are stored too
    LinearResult c[3];
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

// bytes of one K block in a CTA: its 128 rows of A and its half of the tile's columns of B
__host__ __device__ constexpr uint32_t linear_block_bytes(uint32_t tn) { return kHalfTileBytes + tn / 2 * kRowBytesK; }

// two K blocks per stage halve the hand-overs; at tn = 192 and 256 too few stages would be left
constexpr uint32_t linear_kps(uint32_t tn) { return tn <= 128 ? 2 : 1; }

// what a CTA has besides its ring, and the stages that fit beside it
constexpr uint32_t kLinearFixedBytes = kLinearEpilogueWarps * kLinearBoxBytes + (uint32_t)sizeof(LinearSmem);
constexpr uint32_t linear_stages(uint32_t tn) { return (kSmemMax - kLinearFixedBytes) / (linear_kps(tn) * linear_block_bytes(tn)); }
static_assert(linear_stages(64) == 4 && linear_stages(128) == 4 && linear_stages(192) == kLinearMaxStages && linear_stages(256) == 6,
              "the barriers are as many as the stages of the width that has most");

__device__ __forceinline__ uint32_t pack16(float a, float b, int type)
{
    if (type == CLPK_DT_F16) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// What a warp finishes at a time: `kLinearPart` columns of 32 rows, a row in each lane.
//
// A warp's staging is a box of 32 rows of 64 bytes, in the swizzle of that width: two parts of 16-bit results or one of fp32.  (A
// second box for fp32 gained nothing: 8192 x 8192 x 512 64.0 and 64.6 us.)  TMA stores it and clips what lies beyond C -- in units of 16 bytes: where a row of C ends inside one,
// the map's rows end before it and each lane writes the rest of its row, so that what lies behind the row stays as it is.
template <int TYPE>
__device__ __forceinline__ void fill_box(const float (&v)[kLinearPart], uint8_t *box, uint32_t first, int lane)
{
    constexpr uint32_t kPieces = TYPE == CLPK_DT_F32 ? 4 : 2;
#pragma unroll
    for (uint32_t j = 0; j < kPieces; j++) {
        uint4 w;
        if constexpr (TYPE == CLPK_DT_F32) {
            const float *x = v + 4 * j;
            w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        } else {
            const float *x = v + 8 * j;
            w = make_uint4(pack16(x[0], x[1], TYPE), pack16(x[2], x[3], TYPE), pack16(x[4], x[5], TYPE), pack16(x[6], x[7], TYPE));
        }
        *reinterpret_cast<uint4 *>(box + lane * 64 + (((first + j) ^ ((lane >> 1) & 3)) << 4)) = w;
    }
}

template <int TYPE>
__device__ __forceinline__ void store_box(const LinearResult &c, const uint8_t *box, const CUtensorMap *map, uint32_t col, uint32_t row, int lane)
{
    constexpr uint32_t kElem = TYPE == CLPK_DT_F32 ? 4 : 2, kCols = 64 / kElem;
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        if (col < c.whole)
            tma_store_2d(map, box, (int32_t)col, (int32_t)row);
        bulk_commit();
    }
    if (c.n != c.whole && c.whole - col < kCols && row + lane < c.m) {
        uint4 v = *reinterpret_cast<const uint4 *>(box + lane * 64 + (((c.whole - col) * kElem / 16 ^ ((lane >> 1) & 3)) << 4));
        uint8_t *to = static_cast<uint8_t *>(c.base) + ((uint64_t)(row + lane) * c.ld + c.whole) * kElem;
        const uint32_t bytes = (c.n - c.whole) * kElem;
        if (bytes & 8) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(v.x, v.y);
            to += 8;
            v.x = v.z;
            v.y = v.w;
        }
        if (bytes & 4) {
            *reinterpret_cast<uint32_t *>(to) = v.x;
            to += 4;
            v.x = v.y;
        }
        if (bytes & 2)
            *reinterpret_cast<uint16_t *>(to) = (uint16_t)v.x;
    }
}

template <int ACT>
__device__ __forceinline__ void gate(float (&h)[kLinearPart], const float (&u)[kLinearPart])
{
#pragma unroll
    for (int i = 0; i < kLinearPart; i += 2) {
        const float2 v = mul2(activate2<ACT>(make_float2(h[i], h[i + 1])), make_float2(u[i], u[i + 1]));
        h[i] = v.x;
        h[i + 1] = v.y;
    }
}

__device__ __forceinline__ void gate_by(int act, float (&h)[kLinearPart], const float (&u)[kLinearPart])
{
    switch (act) {
    case CLPK_ACT_SILU:      gate<CLPK_ACT_SILU>(h, u); break;
    case CLPK_ACT_GELU_TANH: gate<CLPK_ACT_GELU_TANH>(h, u); break;
    case CLPK_ACT_GELU:      gate<CLPK_ACT_GELU>(h, u); break;
    case CLPK_ACT_RELU:      gate<CLPK_ACT_RELU>(h, u); break;
    default:                 gate<CLPK_ACT_SIGMOID>(h, u); break;
    }
}

// the sums of a part in fp32; those of 8-bit integers with the scale of the lane's row and those of the columns
template <int DT>
__device__ __forceinline__ void scaled(float (&v)[kLinearPart], const uint32_t (&sum)[kLinearPart], float row_scale, const float *cols)
{
#pragma unroll
    for (int i = 0; i < kLinearPart; i += 4) {
        if constexpr (DT == CLPK_DT_I8) {
            const float4 c = *reinterpret_cast<const float4 *>(cols + i);
            const float2 rows = make_float2(row_scale, row_scale);
            const float2 a = mul2(mul2(make_float2((float)(int32_t)sum[i], (float)(int32_t)sum[i + 1]), rows), make_float2(c.x, c.y));
            const float2 b = mul2(mul2(make_float2((float)(int32_t)sum[i + 2], (float)(int32_t)sum[i + 3]), rows), make_float2(c.z, c.w));
            v[i] = a.x; v[i + 1] = a.y; v[i + 2] = b.x; v[i + 3] = b.y;
        } else {
            for (int j = i; j < i + 4; j++)
                v[j] = __uint_as_float(sum[j]);
        }
    }
}

__device__ __forceinline__ uint32_t bias_bits(const void *bias, int type, uint32_t col)
{
    return type == CLPK_DT_F32 ? static_cast<const uint32_t *>(bias)[col] : static_cast<const uint16_t *>(bias)[col];
}

__device__ __forceinline__ float bias_value(uint32_t bits, int type)
{
    if (type == CLPK_DT_F32)
        return __uint_as_float(bits);
    return type == CLPK_DT_F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}

// What a chunk's 8-bit sums are finished with: the scale of the lane's row, and of each part a column's of Wg's or B's for the lower
// half of the lanes and of Wu's, or bias, for the upper.  They are asked for a chunk ahead, and go to the lanes through shared
// memory: with a shuffle for each column the pipe that shuffles was the bound (bf16 results, 4096 x 14336 x 256 with
// bias 63 us and so 53, both with eight epilogue warps; 35 to 38 with sixteen).
struct LinearScales {
    float row = 0.0f;
    uint32_t col[2] = {};

    template <int DT, LinearForm FORM>
    __device__ __forceinline__ void rows(const LinearParams &p, uint32_t row0, int lane)
    {
        if constexpr (DT == CLPK_DT_I8)
            row = row0 + lane < p.c[0].m ? p.a_scale[row0 + lane] : 0.0f;
    }
    template <int DT, LinearForm FORM>
    __device__ __forceinline__ void cols(const LinearParams &p, uint32_t first, int lane)
    {
        if constexpr (DT == CLPK_DT_I8) {
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                const uint32_t c = first + h * kLinearPart + lane % kLinearPart;
                col[h] = 0;
                if (c < p.c[0].n) {
                    if (lane < kLinearPart)
                        col[h] = __float_as_uint(p.b_scale[c]);
                    else if (FORM == kGated)
                        col[h] = __float_as_uint(p.u_scale[c]);
                    else if (p.bias)
                        col[h] = bias_bits(p.bias, p.c[0].type, c);
                }
            }
        }
    }
    template <LinearForm FORM>
    __device__ __forceinline__ float value(const LinearParams &p, uint32_t h, int lane) const
    {
        const uint32_t bits = h ? col[1] : col[0];
        return FORM == kGated || lane < kLinearPart ? __uint_as_float(bits) : bias_value(bits, p.c[0].type);
    }
};

// a row's part of an exchanged unit, four columns every 2 KiB
__device__ __forceinline__ void load_part(uint32_t (&v)[kLinearPart], const uint8_t *at)
{
#pragma unroll
    for (uint32_t g = 0; g < kLinearPart / 4; g++) {
        const uint4 e = *reinterpret_cast<const uint4 *>(at + g * 2048);
        v[4 * g] = e.x; v[4 * g + 1] = e.y; v[4 * g + 2] = e.z; v[4 * g + 3] = e.w;
    }
}

// what a warp of the epilogue works with
struct LinearWarp {
    uint8_t *box;
    float *cols;                                        // of a part: 32 scales, or scales and bias
    int lane;
};

// What becomes of a chunk of sums, or with kGated of that of g and that of u.  fetch(h, s0, s1, last): the sums of a part; `last`:
// they are not asked for again.  `which`: the result that plain sums (kGradients) belong to.
template <int DT, LinearForm FORM, int TYPE, typename Fetch>
__device__ __forceinline__ void linear_finish_as(const CUtensorMap *maps, const LinearParams &p, const LinearScales &scales, uint32_t which, uint32_t row,
                                                 uint32_t col, const LinearWarp &w, Fetch fetch)
{
    // kGated: g and u go out first where they are kept
    for (uint32_t out = FORM == kGated && DT != CLPK_DT_I8 && p.keep ? 2 : 0;; out--) {
        const uint32_t to = FORM == kGated ? out : which;
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            uint32_t s0[kLinearPart], s1[kLinearPart];
            fetch(h, s0, s1, out == 0 && h == 1);
            if constexpr (DT == CLPK_DT_I8) {
                w.cols[w.lane] = scales.value<FORM>(p, h, w.lane);       // all lanes have read the last ones: a box's turn lies between
                __syncwarp();
            }
            float v[kLinearPart];
            scaled<DT>(v, s0, scales.row, w.cols);
            if constexpr (FORM == kGated) {
                float u[kLinearPart];
                scaled<DT>(u, s1, scales.row, w.cols + kLinearPart);
                if (DT == CLPK_DT_I8 || out == 0) {
                    gate_by(p.activation, v, u);
                } else if (out == 2) {
#pragma unroll
                    for (int i = 0; i < kLinearPart; i++)
                        v[i] = u[i];
                }
            } else if constexpr (FORM == kScaled) {
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < kLinearPart; i += 4) {
                        const float4 c = *reinterpret_cast<const float4 *>(w.cols + kLinearPart + i);
                        v[i] += c.x; v[i + 1] += c.y; v[i + 2] += c.z; v[i + 3] += c.w;
                    }
                }
            }
            constexpr bool kWide = TYPE == CLPK_DT_F32;
            if ((kWide || h == 0) && w.lane == 0)
                bulk_wait_read<0>();
            __syncwarp();
            fill_box<TYPE>(v, w.box, kWide ? 0 : 2 * h, w.lane);
            if (kWide || h == 1)
                store_box<TYPE>(p.c[to], w.box, maps + to, kWide ? col + h * kLinearPart : col, row, w.lane);
        }
        if (out == 0)
            break;
    }
}

template <int DT, LinearForm FORM, typename Fetch>
__device__ __forceinline__ void linear_finish(const CUtensorMap *maps, const LinearParams &p, const LinearScales &scales, uint32_t which, uint32_t row, uint32_t col,
                                              const LinearWarp &w, Fetch fetch)
{
    const int type = p.c[which].type;
    if constexpr (DT != CLPK_DT_I8) {                   // its own type, or fp32 for a part of a gradient's sum
        if (FORM == kGradients && type == CLPK_DT_F32)
            linear_finish_as<DT, FORM, CLPK_DT_F32>(maps, p, scales, which, row, col, w, fetch);
        else
            linear_finish_as<DT, FORM, DT>(maps, p, scales, which, row, col, w, fetch);
    } else if (type == CLPK_DT_F32) {
        linear_finish_as<DT, FORM, CLPK_DT_F32>(maps, p, scales, which, row, col, w, fetch);
    } else if (type == CLPK_DT_F16) {
        linear_finish_as<DT, FORM, CLPK_DT_F16>(maps, p, scales, which, row, col, w, fetch);
    } else {
        linear_finish_as<DT, FORM, CLPK_DT_BF16>(maps, p, scales, which, row, col, w, fetch);
    }
}

// a tile: which result, where in it (rows of 256, and for the result; columns of tn), and which K blocks of it this pair adds
struct LinearTile {
    uint32_t which, mb, mb_out, nb, kb0, kb1;
};

#include "clpk_linear_grad.cuh"

struct LinearMaps {
    CUtensorMap a, b[2], c[3];
};
template <LinearForm FORM> using LinearMapsOf = std::conditional_t<FORM == kGradients, GradMaps, LinearMaps>;
template <LinearForm FORM> using LinearParamsOf = std::conditional_t<FORM == kGradients, GradParams, LinearParams>;

// the i-th tile of a cluster; false: it has no more
template <LinearForm FORM>
__device__ __forceinline__ bool linear_tile(const LinearParamsOf<FORM> &p, uint32_t cluster, uint32_t clusters, uint32_t split, uint32_t i, LinearTile &t)
{
    if constexpr (FORM == kGradients) {
        return grad_tile(p, cluster, clusters, i, t);
    } else {
        const uint32_t tile = cluster + i * clusters;
        if (tile >= p.order.tiles_m * p.order.tiles_n)
            return false;
        tile_coords(p.order, tile, t.mb, t.nb);
        t.mb_out = t.mb;
        t.which = 0;
        t.kb0 = split * p.k_blocks / p.splits;
        t.kb1 = (split + 1) * p.k_blocks / p.splits;
        return true;
    }
}

template <int DT, LinearForm FORM>
__global__ void __launch_bounds__(kLinearThreads) linear_kernel(const __grid_constant__ LinearMapsOf<FORM> maps, const __grid_constant__ LinearParamsOf<FORM> p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw;
    // The ring and the scales leave no room to move the base up to 1024 bytes, the swizzle's period; a launch whose memory does not
    // start there, as it is declared, says so instead of computing.
    if (smem_u32(smem) % 1024 != 0) {
        griddep_wait();
        if (threadIdx.x == 0)
            *p.status = 0x306u;
        return;
    }
    const uint32_t block_bytes = linear_block_bytes(p.tn), stage_bytes = p.kps * block_bytes;
    uint8_t *staging = smem + (size_t)p.stages * stage_bytes;
    LinearSmem *sh = reinterpret_cast<LinearSmem *>(staging + kLinearEpilogueWarps * kLinearBoxBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), r = rank & 1, leader = rank & ~1u, split = rank >> 1;
    const uint32_t cluster = blockIdx.x / (2 * p.splits), clusters = gridDim.x / (2 * p.splits);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (int acc = 0; acc < 2; acc++) {
            mbar_init(&sh->tmem_full[acc], 1);
            mbar_init(&sh->tmem_empty[acc], 2 * kLinearEpilogueWarps);
        }
        mbar_fence_init();
        if constexpr (FORM != kGradients) {
            tma_prefetch_desc(&maps.a);
            tma_prefetch_desc(&maps.b[FORM == kGated ? r : 0]);
            tma_prefetch_desc(&maps.c[0]);
        }
    }
    if (warp == 1)
        tmem_alloc<2>(&sh->tmem_base, p.tmem_cols);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    griddep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *p.status = 0u;
    griddep_launch_dependents();

    const uint32_t q = (uint32_t)(warp & 3), set = (uint32_t)(warp - 2) >> 2;      // epilogue warps
    const uint32_t unit_cols = FORM == kGated ? p.tn / 2 : p.tn, units = unit_cols / kLinearChunk;
    constexpr uint32_t kSubs = FORM == kGated ? 2 : 1;                             // chunks per unit, tn / 2 columns apart
    const uint32_t me = warp < 2 ? 0 : warp - 2;
    const LinearWarp w = {staging + me * kLinearBoxBytes, sh->cols[me], lane};
    LinearTile t;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const uint32_t full0 = cluster_addr(&sh->full[0], leader);
        uint32_t s = 0, parity = 1, issued = 0;                // parity of the empty barrier's previous phase
        bool ok = true;
        for (uint32_t i = 0; ok && linear_tile<FORM>(p, cluster, clusters, split, i, t); i++) {
            const uint32_t row_a = t.mb * kLinearM + r * 128;
            const uint32_t row_b = FORM == kGated ? t.nb * (p.tn / 2) : t.nb * p.tn + r * (p.tn / 2);
            const uint32_t kb0 = t.kb0, kb1 = t.kb1;
            for (uint32_t kb = kb0; kb < kb1; kb += p.kps) {
                const uint32_t nk = kb1 - kb < p.kps ? kb1 - kb : p.kps;
                if (!warp_wait(&sh->empty[s], parity)) {       // a fresh barrier's preceding phase counts as complete
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x301u);
                    ok = false;
                    break;
                }
                uint8_t *st = smem + (size_t)s * stage_bytes;
                if (elect_one()) {
                    if (r == 0)
                        mbar_expect_tx(&sh->full[s], nk * 2 * block_bytes);
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++)
                        if (h < nk) {
                            uint8_t *blk = st + h * block_bytes;
                            if constexpr (FORM == kGradients) {
                                grad_load(maps, p, t.which, blk, kb + h, row_a, row_b, full0 + 8 * s);
                            } else {
                                tma_load_pair_at(blk, &maps.a, (int32_t)((kb + h) * kRowBytesK), (int32_t)row_a, full0 + 8 * s);
                                tma_load_pair_at(blk + kHalfTileBytes, &maps.b[FORM == kGated ? r : 0], (int32_t)((kb + h) * kRowBytesK), (int32_t)row_b, full0 + 8 * s);
                            }
                        }
                }
                __syncwarp();
                issued++;
                if (++s == p.stages) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
        if (r == 0)                                            // its barriers count the loads of both; nothing else waits for this warp
            ring_settled(sh->full, p.stages, issued);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the pair's leader) ----------------
        if (r == 0) {
            constexpr uint32_t kFmt = DT == CLPK_DT_BF16 ? kFmtBF16 : DT == CLPK_DT_F16 ? kFmtF16 : kFmtS8;
            const uint16_t pair_mask = (uint16_t)(3u << leader);
            uint32_t s = 0, parity = 0;
            bool ok = true;
            for (uint32_t i = 0; ok && linear_tile<FORM>(p, cluster, clusters, split, i, t); i++) {
                const uint32_t acc = i & 1, use = i >> 1;
                const uint32_t kb0 = t.kb0, kb1 = t.kb1;
                if (use > 0 && !warp_wait(&sh->tmem_empty[acc], (use - 1) & 1)) {
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x302u);
                    break;
                }
                tc_fence_after_sync();
                const uint32_t d = tmem + acc * p.tn;
                const bool a_mn = FORM == kGradients && t.which > 0;       // A contiguous along M
                const uint32_t idesc = make_idesc(256, p.tn, kFmt, kFmt, DT == CLPK_DT_I8 ? kAccS32 : kAccF32) | (a_mn ? kMajorA : 0u) |
                                       (FORM == kGradients ? kMajorB : 0u);
                const uint32_t a_lbo = a_mn ? kMnLead : 16, a_step = a_mn ? kMnStep : 2;
                constexpr uint32_t kBLbo = FORM == kGradients ? kMnLead : 16, kBStep = FORM == kGradients ? kMnStep : 2;
                for (uint32_t kb = kb0; kb < kb1; kb += p.kps) {
                    if (!warp_wait(&sh->full[s], parity)) {
                        if (lane == 0)
                            atomicCAS(p.status, 0u, 0x303u);
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t base = smem_u32(smem + (size_t)s * stage_bytes);
                    const uint32_t nk = kb1 - kb < p.kps ? kb1 - kb : p.kps;
                    const uint32_t s_now = s;
                    if (++s == p.stages) {
                        s = 0;
                        parity ^= 1;
                    }
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t h = 0; h < 2; h++) {
                            if (h >= nk)
                                break;
                            const uint32_t blk = base + h * block_bytes;
                            const uint64_t ad = make_smem_desc(blk, a_lbo, 1024, kSwizzle128B), bd = make_smem_desc(blk + kHalfTileBytes, kBLbo, 1024, kSwizzle128B);
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; kk++) {
                                const uint32_t accumulate = (kb != kb0 || h != 0 || kk != 0) ? 1u : 0u;
                                if constexpr (DT == CLPK_DT_I8)
                                    mma2_i8_ss(d, ad + kk * a_step, bd + kk * kBStep, idesc, accumulate);
                                else
                                    mma2_f16_ss(d, ad + kk * a_step, bd + kk * kBStep, idesc, accumulate);
                            }
                        }
                        tc_commit_pair(&sh->empty[s_now], pair_mask);
                    }
                    __syncwarp();
                }
                if (ok && elect_one())
                    tc_commit_pair(&sh->tmem_full[acc], pair_mask);
                __syncwarp();
            }
        }
    } else if (p.splits == 1) {
        // ---------------- epilogue, K not split: the warps of a lane quarter take chunks in turn ----------------
        auto ask = [&](LinearScales &scales) {                 // for a tile's first chunk
            scales.template rows<DT, FORM>(p, t.mb_out * kLinearM + r * 128 + q * 32, lane);
            scales.template cols<DT, FORM>(p, t.nb * unit_cols + set * kLinearChunk, lane);
        };
        LinearScales scales;
        bool more = linear_tile<FORM>(p, cluster, clusters, split, 0, t);
        if (more)
            ask(scales);
        for (uint32_t i = 0; more; i++) {
            const uint32_t acc = i & 1, use = i >> 1, which = t.which;
            const uint32_t row = t.mb_out * kLinearM + r * 128 + q * 32, col = t.nb * unit_cols;
            if (!warp_wait(&sh->tmem_full[acc], use & 1)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x304u);
                break;
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem + acc * p.tn + ((q * 32) << 16);
            auto release = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster_relaxed(&sh->tmem_empty[acc], leader);
            };
            if (set >= units) {
                release();
                more = linear_tile<FORM>(p, cluster, clusters, split, i + 1, t);
                continue;
            }
            for (uint32_t c = set; c < units; c += kLinearSets) {
                const bool last_chunk = c + kLinearSets >= units;
                LinearScales next = scales;
                if (!last_chunk)
                    next.template cols<DT, FORM>(p, col + (c + kLinearSets) * kLinearChunk, lane);
                else if ((more = linear_tile<FORM>(p, cluster, clusters, split, i + 1, t)))
                    ask(next);
                linear_finish<DT, FORM>(maps.c, p, scales, which, row, col + c * kLinearChunk, w,
                                        [&](uint32_t h, uint32_t (&s0)[kLinearPart], uint32_t (&s1)[kLinearPart], bool last) {
                                            const uint32_t at = taddr + c * kLinearChunk + h * kLinearPart;
                                            tmem_ld_32x32b_x16(at, s0);
                                            if (FORM == kGated)
                                                tmem_ld_32x32b_x16(at + p.tn / 2, s1);
                                            tmem_ld_wait();
                                            if (last && last_chunk)
                                                release();
                                        });
                scales = next;
            }
        }
    } else if (!warp_wait(&sh->tmem_full[0], 0)) {
        if (lane == 0)
            atomicCAS(p.status, 0u, 0x305u);
    }

    if (FORM != kGradients && p.splits > 1) {
        // ---------------- K split over the cluster's pairs (one tile per cluster) ----------------
        // Every pair's instructions have retired, so the stages of the ring are free to take partial sums: slot (src, j) of CTA
        // (owner, r) holds pair src's sums of the owner's j-th unit, src counted without the owner.  They are added in the order
        // of the pairs, whoever owns the unit.
        constexpr uint32_t kUnitBytes = kSubs * kLinearChunk * 128 * 4;
        tc_fence_before_sync();
        __syncwarp();
        cluster_sync();
        tc_fence_after_sync();
        const uint32_t slots = (units + p.splits - 1) / p.splits;
        const uint32_t taddr = tmem + ((q * 32) << 16), my_row = q * 32 + lane;
        const bool epilogue = warp >= 2;
        if (epilogue) {
            for (uint32_t i = set; i < kSubs * units; i += kLinearSets) {
                const uint32_t c = i / kSubs, sub = i % kSubs, owner = c % p.splits;
                if (owner == split)
                    continue;
                uint32_t v[32];
                tmem_ld_32x32b_x32(taddr + sub * (p.tn / 2) + c * kLinearChunk, v);
                tmem_ld_wait();
                const uint32_t src = split < owner ? split : split - 1;
                const uint32_t dst = cluster_addr(smem + (size_t)(src * slots + c / p.splits) * kUnitBytes + sub * (kUnitBytes / kSubs) + my_row * 16, owner * 2 + r);
#pragma unroll
                for (uint32_t g = 0; g < 8; g++)
                    st_cluster_v4(dst + g * 2048, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        }
        __syncwarp();
        cluster_sync();
        if (epilogue && linear_tile<FORM>(p, cluster, clusters, split, 0, t)) {
            const uint32_t row = t.mb_out * kLinearM + r * 128 + q * 32;
            // the four warps of a lane quarter share the sums, each of which takes the place of the first of its terms
            constexpr uint32_t kParts = kLinearChunk / kLinearPart * kSubs;
#pragma unroll 1
            for (uint32_t i = set; split + i / kParts * p.splits < units; i += kLinearSets) {
                const uint32_t j = i / kParts, c = split + j * p.splits, sub = i % kParts / 2, h = i % 2;
                uint8_t *const slot = smem + (size_t)j * kUnitBytes + sub * (kUnitBytes / kSubs) + h * 8192 + my_row * 16;
                uint32_t own[kLinearPart], sum[kLinearPart] = {};
                tmem_ld_32x32b_x16(taddr + sub * (p.tn / 2) + c * kLinearChunk + h * kLinearPart, own);
                tmem_ld_wait();
#pragma unroll 1
                for (uint32_t src = 0; src < p.splits; src++) {
                    uint32_t theirs[kLinearPart];
                    if (src != split)
                        load_part(theirs, slot + (size_t)(src < split ? src : src - 1) * slots * kUnitBytes);
#pragma unroll
                    for (uint32_t l = 0; l < kLinearPart; l++) {
                        const uint32_t e = src == split ? own[l] : theirs[l];
                        if (src == 0)
                            sum[l] = e;
                        else if constexpr (DT == CLPK_DT_I8)
                            sum[l] += e;
                        else
                            sum[l] = __float_as_uint(__uint_as_float(sum[l]) + __uint_as_float(e));
                    }
                }
#pragma unroll
                for (uint32_t g = 0; g < kLinearPart / 4; g++)
                    *reinterpret_cast<uint4 *>(slot + g * 2048) = make_uint4(sum[4 * g], sum[4 * g + 1], sum[4 * g + 2], sum[4 * g + 3]);
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + q), "n"(32 * kLinearSets) : "memory");
            for (uint32_t j = set; split + j * p.splits < units; j += kLinearSets) {
                const uint32_t c = split + j * p.splits, col = t.nb * unit_cols + c * kLinearChunk;
                const uint8_t *const at = smem + (size_t)j * kUnitBytes + my_row * 16;
                LinearScales scales;
                scales.rows<DT, FORM>(p, row, lane);
                scales.cols<DT, FORM>(p, col, lane);
                linear_finish<DT, FORM>(maps.c, p, scales, t.which, row, col, w, [&](uint32_t h, uint32_t (&s0)[kLinearPart], uint32_t (&s1)[kLinearPart], bool) {
                    load_part(s0, at + h * 8192);
                    if (FORM == kGated)
                        load_part(s1, at + kUnitBytes / 2 + h * 8192);
                });
            }
        }
    }
    // the staging boxes must have been read before this CTA's shared memory goes away
    if (warp >= 2 && lane == 0)
        bulk_wait_read<0>();

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    if (warp == 1)
        tmem_dealloc<2>(tmem, p.tmem_cols);
}

// ---- host side -----------------------------------------------------------------------------

// a row-major matrix, in boxes of 128 bytes of a row times box_rows rows
static int make_matrix_map(CUtensorMap *map, const void *base, uint64_t rows, uint64_t row_bytes, uint64_t pitch_bytes, uint32_t box_rows)
{
    EncodeTiledFn enc = nullptr;
    const int rc = get_encode_fn(&enc);
    if (rc != CLPK_OK)
        return rc;
    const cuuint64_t dims[2] = {row_bytes, rows}, strides[1] = {pitch_bytes};
    const cuuint32_t box[2] = {kRowBytesK, box_rows}, estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return CLPK_ERR_CUDA;
    }
    return CLPK_OK;
}

// a result, in boxes of 32 rows of 64 bytes
static int make_result_map(CUtensorMap *map, const LinearResult &c)
{
    EncodeTiledFn enc = nullptr;
    const int rc = get_encode_fn(&enc);
    if (rc != CLPK_OK)
        return rc;
    const uint32_t elem = c.type == CLPK_DT_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {std::max(c.whole, 16 / elem), c.m}, strides[1] = {c.ld * elem};
    const cuuint32_t box[2] = {64 / elem, 32}, estr[2] = {1, 1};
    const CUresult r = enc(map, elem == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c.base, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled (result) failed with CUresult %d", (int)r);
        return CLPK_ERR_CUDA;
    }
    return CLPK_OK;
}
