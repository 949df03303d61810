// Products of a feed-forward layer with few tokens (included by feed_forward.cu).
//
// Every weight is read once and multiplied by a handful of tokens, so the time is that of reading the weights.  The operands
// change places: a tile's 128 rows are rows of the weight, as they lie in memory, and the tokens are its columns (16 to 128, the
// fewest that a tcgen05 instruction of 128 rows takes), so that of the shared memory that TMA fills nearly all is weight.  With
// kGated a tile is 64 rows of Wg above the same 64 of Wu.
//
// K is split over the CTAs of a cluster, as far as it takes to give every SM some: one tile per cluster, each CTA a K range.  Each token
// belongs to one of the CTAs: all send it their partial sums of that token through distributed shared memory, and after one barrier
// it adds them in the order of K and finishes them.  Sending instead of fetching, because a fetch is a round trip of a microsecond
// per CTA that is asked; and, where a CTA's share of the SM has room for it, to a place behind the owner's ring, which may still be
// at work (in the ring it takes a barrier more).  Nothing goes through global memory.  CTAs are small: several share an SM, and
// one's set-up and exchange lie under another's loads.
//
// What bounds it: the weights' way from memory, and for few of them the chain from launch to launch (2.7 us).  bf16 1 x 4096 x
// 11008: 180 MB in 31.3 us, 5.8 TB/s; int8 1 x 16384 x 4096 13.5 us against 10.3 at the copy rate, 1 x 4096 x 4096 5.2 against
// 2.6; int8 48 x 4096 x 11008 20.0 against 14.0, of which 2.3 are the finishing of 48 tokens after the last product.  With 256
// tokens' rows of A and the weights as B, as the pairs have it, the same calls take 16 to 64 us.
#pragma once

constexpr int kFewThreads = 256, kFewResident = 4;             // CTAs that an SM has registers for
constexpr int kFewMaxStages = 8;
constexpr uint32_t kFewRows = 128;

struct FewSmem {
    uint64_t full[kFewMaxStages];
    uint64_t empty[kFewMaxStages];
    uint64_t done;
    uint32_t tmem_base;
    float a_scale[128];                             // of the tokens
};

struct FewMaps {
    CUtensorMap w[2], x;
};

struct FewParams {
    uint32_t m, n;                                  // tokens, rows of a weight
    uint32_t k_blocks, splits, stages, tokens;      // tokens: m rounded up to what the instruction takes
    uint32_t sums_at;                               // where the partial sums lie: behind the ring, or 0: in it
    uint32_t smem_bytes;                            // of the ring and the sums
    uint32_t tmem_cols;
    int out, activation;
    void *c, *g, *u;                                // g, u: kept where not NULL
    uint64_t ldc;
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

__device__ __forceinline__ void ld_shared(const float *p, uint32_t (&v)[4])
{
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void ld_shared(const float *p, uint32_t (&v)[2])
{
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    v[0] = w.x; v[1] = w.y;
}

// N neighbouring results of one token
template <int N>
__device__ __forceinline__ void few_store(void *base, int type, uint64_t at, uint32_t left, const float (&v)[N])
{
    if (type == CLPK_DT_F32) {
        float *c = static_cast<float *>(base) + at;
        if (left >= N) {
            if constexpr (N == 4)
                *reinterpret_cast<float4 *>(c) = make_float4(v[0], v[1], v[2], v[3]);
            else
                *reinterpret_cast<float2 *>(c) = make_float2(v[0], v[1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < left)
                    c[i] = v[i];
        }
        return;
    }
    uint16_t *c = static_cast<uint16_t *>(base) + at;
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2)
        w[i / 2] = pack16(v[i], v[i + 1], type);
    if (left >= N) {
        if constexpr (N == 4)
            *reinterpret_cast<uint2 *>(c) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t *>(c) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left)
                c[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
}

// What a CTA finishes: its tokens' partial sums, [K range][token][128 rows], and what they are finished with.
template <uint32_t kPerLane>
struct FewFinish {
    const float *sums;
    uint32_t slots, first;                          // tokens of an owner, the first one of this
    uint32_t col, left;                             // the lane's first feature, and how many there are from it on
    const float (&b_scale)[kPerLane], (&u_scale)[kPerLane];
    const float *a_scale;                           // of all tokens
};

// A warp takes kAtOnce tokens in a step, so that one's loads and activations do not wait for another's.
template <int DT, LinearForm FORM, int ACT, uint32_t kPerLane>
__device__ __forceinline__ void few_finish(const FewParams &p, const FewFinish<kPerLane> &f, uint32_t warp, uint32_t lane)
{
    constexpr uint32_t kSubs = FORM == kGated ? 2 : 1, kAtOnce = 2, kWarps = kFewThreads / 32;
    const uint32_t here = f.first < p.m ? (p.m - f.first < f.slots ? p.m - f.first : f.slots) : 0;
    for (uint32_t k0 = warp; k0 < here; k0 += kAtOnce * kWarps) {
        uint32_t sum[kAtOnce][kSubs][kPerLane];
        for (uint32_t src = 0; src < p.splits; src++) {
            uint32_t e[kAtOnce][kSubs][kPerLane];
#pragma unroll
            for (uint32_t t = 0; t < kAtOnce; t++) {
                const uint32_t k = k0 + t * kWarps;
                if (k < here) {
                    const float *from = f.sums + (src * f.slots + k) * kFewRows + lane * kPerLane;
#pragma unroll
                    for (uint32_t o = 0; o < kSubs; o++)
                        ld_shared(from + o * 64, e[t][o]);
                }
            }
#pragma unroll
            for (uint32_t t = 0; t < kAtOnce; t++)
#pragma unroll
                for (uint32_t o = 0; o < kSubs; o++)
#pragma unroll
                    for (uint32_t i = 0; i < kPerLane; i++) {
                        uint32_t &x = sum[t][o][i];
                        if (src == 0)
                            x = e[t][o][i];
                        else if constexpr (DT == CLPK_DT_I8)
                            x += e[t][o][i];
                        else
                            x = __float_as_uint(__uint_as_float(x) + __uint_as_float(e[t][o][i]));
                    }
        }
        float v[kAtOnce][kSubs][kPerLane], h[kAtOnce][kPerLane];
#pragma unroll
        for (uint32_t t = 0; t < kAtOnce; t++) {
            const uint32_t k = k0 + t * kWarps < here ? k0 + t * kWarps : k0;
            const float a = DT == CLPK_DT_I8 ? f.a_scale[f.first + k] : 1.0f;
#pragma unroll
            for (uint32_t i = 0; i < kPerLane; i++) {
#pragma unroll
                for (uint32_t o = 0; o < kSubs; o++) {
                    if constexpr (DT == CLPK_DT_I8)
                        v[t][o][i] = (float)(int32_t)sum[t][o][i] * a * (o ? f.u_scale[i] : f.b_scale[i]);
                    else
                        v[t][o][i] = __uint_as_float(sum[t][o][i]);
                }
                if constexpr (FORM == kGated)
                    h[t][i] = activate<ACT>(v[t][0][i]) * v[t][1][i];
                else
                    h[t][i] = p.bias ? v[t][0][i] + f.u_scale[i] : v[t][0][i];
            }
        }
#pragma unroll
        for (uint32_t t = 0; t < kAtOnce; t++) {
            if (k0 + t * kWarps >= here)
                break;
            const uint64_t at = (f.first + k0 + t * kWarps) * p.ldc + f.col;
            if constexpr (FORM == kGated)
                if (p.g) {
                    few_store(p.g, p.out, at, f.left, v[t][0]);
                    few_store(p.u, p.out, at, f.left, v[t][1]);
                }
            few_store(p.c, p.out, at, f.left, h[t]);
        }
    }
}

template <int DT, LinearForm FORM>
__global__ void __launch_bounds__(kFewThreads, kFewResident) linear_few_kernel(const __grid_constant__ FewMaps maps, FewParams p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t stage_bytes = kHalfTileBytes + p.tokens * kRowBytesK;
    FewSmem *sh = reinterpret_cast<FewSmem *>(smem + p.smem_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = cluster_ctarank(), tile = blockIdx.x / p.splits;
    const uint32_t kb0 = split * p.k_blocks / p.splits, kb1 = (split + 1) * p.k_blocks / p.splits;
    constexpr uint32_t kTileCols = FORM == kGated ? 64 : 128;                       // features per tile

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        mbar_init(&sh->done, 1);
        mbar_fence_init();
        tma_prefetch_desc(&maps.w[0]);
        tma_prefetch_desc(&maps.x);
        if constexpr (FORM == kGated)
            tma_prefetch_desc(&maps.w[1]);
    }
    if (warp == 1)
        tmem_alloc<1>(&sh->tmem_base, p.tmem_cols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    if (p.splits > 1 && p.sums_at)
        cluster_arrive();                                      // this CTA runs: the others may write to its shared memory
    griddep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *p.status = 0u;
    griddep_launch_dependents();

    uint32_t issued = 0;
    if (warp == 0) {
        // ---------------- TMA producer ----------------
        uint32_t s = 0, parity = 1;
        for (uint32_t kb = kb0; kb < kb1; kb++) {
            if (!warp_wait(&sh->empty[s], parity)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x311u);
                break;
            }
            uint8_t *st = smem + (size_t)s * stage_bytes;
            const int32_t x = (int32_t)(kb * kRowBytesK), row = (int32_t)(tile * kTileCols);
            if (elect_one()) {
                mbar_expect_tx(&sh->full[s], stage_bytes);
                tma_load_own(st, &maps.w[0], x, row, &sh->full[s]);
                if constexpr (FORM == kGated)
                    tma_load_own(st + kHalfTileBytes / 2, &maps.w[1], x, row, &sh->full[s]);
                tma_load_own(st + kHalfTileBytes, &maps.x, x, 0, &sh->full[s]);
            }
            __syncwarp();
            issued++;
            if (++s == p.stages) {
                s = 0;
                parity ^= 1;
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        constexpr uint32_t kFmt = DT == CLPK_DT_BF16 ? kFmtBF16 : DT == CLPK_DT_F16 ? kFmtF16 : kFmtS8;
        const uint32_t idesc = make_idesc(128, p.tokens, kFmt, kFmt, DT == CLPK_DT_I8 ? kAccS32 : kAccF32);
        uint32_t s = 0, parity = 0;
        bool ok = true;
        for (uint32_t kb = kb0; kb < kb1; kb++) {
            if (!warp_wait(&sh->full[s], parity)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x312u);
                ok = false;
                break;
            }
            tc_fence_after_sync();
            const uint32_t base = smem_u32(smem + (size_t)s * stage_bytes);
            if (elect_one()) {
                const uint64_t wd = make_smem_desc(base, 16, 1024, kSwizzle128B), xd = make_smem_desc(base + kHalfTileBytes, 16, 1024, kSwizzle128B);
#pragma unroll
                for (uint32_t kk = 0; kk < 4; kk++) {
                    const uint32_t accumulate = (kb != kb0 || kk != 0) ? 1u : 0u;
                    if constexpr (DT == CLPK_DT_I8)
                        mma_i8_ss(tmem, wd + 2 * kk, xd + 2 * kk, idesc, accumulate);
                    else
                        mma_f16_ss(tmem, wd + 2 * kk, xd + 2 * kk, idesc, accumulate);
                }
                tc_commit(&sh->empty[s]);
            }
            __syncwarp();
            if (++s == p.stages) {
                s = 0;
                parity ^= 1;
            }
        }
        if (ok && elect_one())
            tc_commit(&sh->done);
        __syncwarp();
    }
    __syncwarp();
    // what the results are finished with is fetched while the products are on their way
    constexpr uint32_t kPerLane = kTileCols / 32;
    const uint32_t col = tile * kTileCols + lane * kPerLane, left = col < p.n ? p.n - col : 0;
    float b_scale[kPerLane] = {}, u_scale[kPerLane] = {};
    if constexpr (DT == CLPK_DT_I8) {
#pragma unroll
        for (uint32_t i = 0; i < kPerLane; i++) {
            b_scale[i] = i < left ? p.b_scale[col + i] : 0.0f;
            if constexpr (FORM == kGated)
                u_scale[i] = i < left ? p.u_scale[col + i] : 0.0f;
            else
                u_scale[i] = p.bias && i < left ? bias_value(bias_bits(p.bias, p.out, col + i), p.out) : 0.0f;
        }
        if (threadIdx.x < p.m)
            sh->a_scale[threadIdx.x] = p.a_scale[threadIdx.x];
    }
    // ---------------- partial sums -> shared memory of the token's owner, [K range][token of its][128 rows] ----------------
    // All instructions have retired, hence all loads have landed: where K is not split the ring is free.  A wait that ran out
    // leaves sums that are wrong, and a status that says so; every CTA still comes to the barriers.
    if (!warp_wait(&sh->done, 0)) {
        if (lane == 0)
            atomicCAS(p.status, 0u, 0x313u);
        if (warp == 0)
            ring_settled(sh->full, p.stages, issued);
    }
    tc_fence_after_sync();
    if (p.splits > 1) {
        if (!p.sums_at)
            cluster_arrive();                                  // ... behind its ring's last use
        cluster_wait();
    }
    const uint32_t slots = (p.m + p.splits - 1) / p.splits;    // tokens of an owner
    float *sums = reinterpret_cast<float *>(smem + p.sums_at);
    // a warp reads 32 lanes, those of its number modulo four; the two warps of a lane quarter take every other sixteen tokens
    const uint32_t row = threadIdx.x % kFewRows, lanes = tmem + ((uint32_t)(warp % 4) * 32 << 16);
    if (p.splits == 1) {
        for (uint32_t c = 16 * (warp / 4); c < p.m; c += 32) { // the room is that of whole sixteens
            uint32_t v[16];
            tmem_ld_32x32b_x16(lanes + c, v);
            tmem_ld_wait();
#pragma unroll
            for (uint32_t i = 0; i < 16; i++)
                sums[(c + i) * kFewRows + row] = __uint_as_float(v[i]);
        }
    } else {
        const float *mine = sums + split * slots * kFewRows + row;
        for (uint32_t c = 16 * (warp / 4); c < p.m; c += 32) {
            uint32_t v[16];
            tmem_ld_32x32b_x16(lanes + c, v);
            uint32_t owner = c / slots, slot = c - owner * slots, to = cluster_addr(mine + slot * kFewRows, owner);
            tmem_ld_wait();
#pragma unroll
            for (uint32_t i = 0; i < 16; i++) {
                if (c + i < p.m)
                    st_cluster(to, v[i]);
                to += kFewRows * 4;
                if (++slot == slots) {
                    slot = 0;
                    owner = owner + 1 < p.splits ? owner + 1 : 0;
                    to = cluster_addr(mine, owner);
                }
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (p.splits > 1)
        cluster_sync();
    if (warp == 1)
        tmem_dealloc<1>(tmem, p.tmem_cols);

    // ---------------- the tokens of this CTA: add, finish, store ----------------
    const FewFinish<kPerLane> f = {sums, slots, split * slots, col, left, b_scale, u_scale, sh->a_scale};
    if constexpr (FORM == kGated) {
        switch (p.activation) {
        case CLPK_ACT_SILU:      few_finish<DT, FORM, CLPK_ACT_SILU>(p, f, warp, lane); break;
        case CLPK_ACT_GELU_TANH: few_finish<DT, FORM, CLPK_ACT_GELU_TANH>(p, f, warp, lane); break;
        case CLPK_ACT_GELU:      few_finish<DT, FORM, CLPK_ACT_GELU>(p, f, warp, lane); break;
        case CLPK_ACT_RELU:      few_finish<DT, FORM, CLPK_ACT_RELU>(p, f, warp, lane); break;
        default:                 few_finish<DT, FORM, CLPK_ACT_SIGMOID>(p, f, warp, lane); break;
        }
    } else {
        few_finish<DT, FORM, 0>(p, f, warp, lane);
    }
}
