// One step of Adam with decoupled weight decay over many tensors.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: every array passes by once.  bf16 parameters with master copies and 32-bit moments move 28 bytes an element (270 million of
// them 1.10 to 1.15 ms, 6.6 to 6.9 TB/s), with 8-bit moments and no master copy 10 or 12 (fp32 gradients: 637 to 678 us, 4.8 to 5.1 TB/s;
// instructions are the bound there, 3.4 a cycle of 4).  The table of tensors travels with the launch, so that a call is one launch for up to 440
// tensors, whatever their sizes: a CTA has a chunk of 2048 elements, and finds the tensor that its chunk belongs to by halving the
// list of the tensors' first chunks.
//
// Moments in 8 bits.  A warp has a block of 256 elements, eight in each lane: the moments are computed in fp32, the largest of the block is
// found by one reduction over the lanes, and codes are rounded from registers.  The codes stand for m = s q |q| and
// sqrt(v) = s c^2: the square spreads 127 steps over a range of 2^14, and 255 over 2^16 of sqrt(v), 2^32 of v, where equal steps would
// round to zero whatever is below 2^-8 and 2^-9 of the block's largest.  A v that is not zero keeps a code that is not: an
// element with a small v beside a large one is taken for larger than it is, and its step gets shorter, never divided by eps alone.
// No multiplication and addition are fused, so that moments and codes have one value that can be told in any arithmetic; with moments in
// fp32 that holds for the parameters too.
#include "../clpk_elements.cuh"
#include "../clpk_internal.h"
#include "../clpk_ptx.cuh"

#include <cmath>

namespace clpk {

constexpr int kStepThreads = 256, kStepElems = 8;
constexpr uint32_t kStepChunk = kStepThreads * kStepElems;
static_assert(32 * kStepElems == CLPK_ADAMW_BLOCK, "a warp has one block of 8-bit moments");

struct StepTensor {
    uint64_t n;
    void *param;
    const void *grad;
    float *master;
    void *m, *v;
    float *m_scale, *v_scale;
};

// the step's numbers
struct StepRates {
    float b1, b1_rest, b2, b2_rest, eps;
    float keep, root_scale, rate;                       // 1 - lr wd, 1 / sqrt(1 - b2^t), lr / (1 - b1^t)
    float none;                                         // -0
};

struct StepCommon {
    StepRates rates;
    double lr, beta1, beta2, decay;                     // with d_lr or d_step
    uint64_t step;
    const float *d_lr;
    const uint32_t *d_step;
    const float *grad_scale;
    uint32_t count;
};

template <int CAP> struct StepTable {
    StepCommon c;
    StepTensor tensors[CAP];
    uint32_t first[CAP];                                // chunk of the launch; `aligned` in the top bit
};
constexpr uint32_t kStepAligned = 0x80000000u;
constexpr int kStepFew = 48, kStepSome = 144, kStepMany = 440;
static_assert(sizeof(StepTable<kStepMany>) <= 32764, "parameters of a kernel");

__host__ __device__ __forceinline__ void set_rates(StepRates &r, double lr, double beta1, double beta2, double decay, double step)
{
    // 1 - beta^t without the digits that a beta near 1 loses
    const double c1 = beta1 > 0 ? -expm1(step * log(beta1)) : 1.0, c2 = beta2 > 0 ? -expm1(step * log(beta2)) : 1.0;
    r.keep = (float)(1.0 - lr * decay);
    r.root_scale = (float)(1.0 / sqrt(c2));
    r.rate = (float)(lr / c1);
}

// Two numbers at a time, each operation rounded by itself.  The assembler makes a fused multiply-add of mul.rn.f32x2 and a sum that
// follows; so a product is a fused one with -0, which it does not know (`none`: StepRates::none).
__device__ __forceinline__ float2 step_mul(float2 a, float2 b, float none)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %6};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(none));
    return d;
}
__device__ __forceinline__ float2 step_add(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 step_sub(float2 a, float2 b)          // b * -1 + a
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %6};\n\tfma.rn.f32x2 a, b, c, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(-1.0f));
    return d;
}
// the largest of three, NaN where one is NaN
__device__ __forceinline__ float step_max(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 step_both(float x) { return make_float2(x, x); }

constexpr uint32_t kByteFloat = 0x4B000000u;            // 2^23: a byte in its lowest place is added to it
constexpr float kRoundCode = 12582912.0f;               // 1.5 * 2^23: the sum's last place is 1

// bytes j and j + 1 of `w` as numbers, less `bias`
__device__ __forceinline__ float2 step_bytes(uint32_t w, uint32_t j, float bias)
{
    return step_add(make_float2(__uint_as_float(__byte_perm(w, kByteFloat, 0x7540 + j)), __uint_as_float(__byte_perm(w, kByteFloat, 0x7541 + j))),
                    step_both(-8388608.0f - bias));
}

__device__ __forceinline__ float sqrt_near(float x)     // 2^-23 of the value off; 0 below 2^-126
{
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_near(float x)      // 2^-23 of the value off
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Codes of four elements, as numbers that have them in their lowest byte: rint(sqrt(size * inverse)) with the sign of m for m, whose
// size is |m|, and of 1 at least for v, whose size is sqrt(v).
//
// Roots are taken with 2^-23 of their value first.  The one or two of them and the rounding of the product leave the last one, which is 255 at
// most, less than 2^-13 off, and that tells the code unless it lies so near to the middle between two; then the roots are
// rounded.  `exact`: that they are in any case.
template <bool V>
__device__ __forceinline__ void step_codes(float2 (&t)[2], const float2 (&of)[2], float inverse, float none, bool exact)
{
    const auto root_of = [&](float x, bool near) { return near ? sqrt_near(x) : __fsqrt_rn(x); };
    const auto codes = [&](float2 x, bool near, float2 &root) {
        const float2 size = V ? make_float2(root_of(x.x, near), root_of(x.y, near)) : make_float2(fabsf(x.x), fabsf(x.y));
        const float2 y = step_mul(size, step_both(inverse), none);
        root = make_float2(root_of(y.x, near), root_of(y.y, near));
        root = V ? make_float2(fmaxf(root.x, 1.0f), fmaxf(root.y, 1.0f)) : make_float2(copysignf(root.x, x.x), copysignf(root.y, x.y));
        return step_add(root, step_both(kRoundCode));
    };
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float2 root;
        t[i] = codes(of[i], true, root);
        const float2 off = step_sub(root, step_add(t[i], step_both(-kRoundCode)));
        far = step_max(far, fabsf(off.x), fabsf(off.y));
    }
    if (far > 0.5f - 1.0f / 8192 || exact) {            // not with a NaN, of whose block the codes are 0
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float2 root;
            t[i] = codes(of[i], false, root);
        }
    }
}

// The scale of a block from its largest size, whose bits order like the values; 1 / scale, or 0 where there is none.  The quotient by a
// constant is a product with the reciprocal and one correction by its remainder, the reciprocal a near one and a correction likewise (Markstein
// 1990): rounded as a division is.  The tests compare the quotients of all numbers between two powers of two, at 1, at both ends of fp32
// and about the least scale; the reciprocals were compared with __frcp_rn's, of every number from 2^-126 to 1e36.
template <int STEPS>
__device__ __forceinline__ float step_scale(uint32_t top, float &scale)
{
    constexpr float kSquared = (float)(STEPS * STEPS), kReciprocal = (float)(1.0 / (STEPS * STEPS));
    if (top >= 0x7F800000u) {
        scale = __uint_as_float(0x7FC00000u);
        return 0.0f;
    }
    const float size = __uint_as_float(top), near = __fmul_rn(size, kReciprocal);
    scale = __fmaf_rn(__fmaf_rn(-near, kSquared, size), kReciprocal, near);
    if (scale < 1.17549435e-38f) {
        scale = 0.0f;
        return 0.0f;
    }
    const float r = rcp_near(scale);
    return __fmaf_rn(r, __fmaf_rn(-scale, r, 1.0f), r);
}

// Eight elements of a thread, in pairs.  FAST: neighbours, in whole vectors; otherwise 32 apart, one at a time, those below `left` only.
template <int DT, int GDT, int SDT, bool MASTER, bool FAST>
__device__ __forceinline__ void step_elements(const StepTensor &t, const StepRates &r, float grad_scale, uint64_t at, uint32_t left)
{
    using P = Element<DT>;
    using G = Element<GDT>;
    constexpr int N = kStepElems;
    constexpr bool kSmall = SDT == CLPK_DT_I8;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t block = at;                          // the warp's first element
    typename P::T *const param = static_cast<typename P::T *>(t.param) + block;
    const typename G::T *const grad = static_cast<const typename G::T *>(t.grad) + block;
    float *const master = MASTER ? t.master + block : nullptr;
    float p[N], g[N], m[N], v[N];
    uint32_t qm[2] = {}, qv[2] = {};                    // codes, four a word
    auto mine = [&](int j) { return lane + 32 * j; };

    if constexpr (FAST) {
        Raw<GDT, N> raw_g;
        raw_g.load(grad + lane * N);
        if constexpr (kSmall) {
            const uint2 m8 = *reinterpret_cast<const uint2 *>(static_cast<const int8_t *>(t.m) + block + lane * N);
            const uint2 v8 = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.v) + block + lane * N);
            qm[0] = m8.x; qm[1] = m8.y; qv[0] = v8.x; qv[1] = v8.y;
        } else {
            Raw<CLPK_DT_F32, N> raw_m, raw_v;
            raw_m.load(static_cast<const float *>(t.m) + block + lane * N);
            raw_v.load(static_cast<const float *>(t.v) + block + lane * N);
            raw_m.widen(m);
            raw_v.widen(v);
        }
        if constexpr (MASTER) {
            Raw<CLPK_DT_F32, N> raw;
            raw.load(master + lane * N);
            raw.widen(p);
        } else {
            Raw<DT, N> raw;
            raw.load(param + lane * N);
            raw.widen(p);
        }
        raw_g.widen(g);
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) {
            p[j] = g[j] = m[j] = v[j] = 0.0f;
            if (mine(j) < left) {
                g[j] = G::widen(grad[mine(j)]);
                p[j] = MASTER ? master[mine(j)] : P::widen(param[mine(j)]);
                if constexpr (kSmall) {
                    qm[j / 4] |= (uint32_t)static_cast<const uint8_t *>(t.m)[block + mine(j)] << (8 * (j & 3));
                    qv[j / 4] |= (uint32_t)static_cast<const uint8_t *>(t.v)[block + mine(j)] << (8 * (j & 3));
                } else {
                    m[j] = static_cast<const float *>(t.m)[block + mine(j)];
                    v[j] = static_cast<const float *>(t.v)[block + mine(j)];
                }
            }
        }
    }
    float sm = 0.0f, sv = 0.0f;
    if constexpr (kSmall) {
        sm = t.m_scale[block / CLPK_ADAMW_BLOCK];
        sv = t.v_scale[block / CLPK_ADAMW_BLOCK];
        qm[0] ^= 0x80808080u;                           // from [-128, 127] to [0, 255]
        qm[1] ^= 0x80808080u;
    }
    const auto mul = [&](float2 a, float2 b) { return step_mul(a, b, r.none); };
    // With moments in 8 bits the instructions are the bound: root and reciprocal come with 2^-23 of their value.  A near root is 0 where v is
    // below 2^-126, so eps has to hide what is lost there, 2^-63: by 2^-22.  So the quotient's lower side is 2^-22 off, its reciprocal 2^-23
    // more, and the quotient less than 2^-21 beside what its roundings are in any case.
    const bool near = kSmall && r.eps >= r.root_scale * 4.547473508864641e-13f;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        float2 m2 = make_float2(m[j], m[j + 1]), v2 = make_float2(v[j], v[j + 1]), p2 = make_float2(p[j], p[j + 1]), step;
        const float2 g2 = mul(make_float2(g[j], g[j + 1]), step_both(grad_scale));
        if constexpr (kSmall) {
            const float2 q = step_bytes(qm[j / 4], j & 3, 128.0f), c = step_bytes(qv[j / 4], j & 3, 0.0f);
            m2 = mul(mul(q, make_float2(fabsf(q.x), fabsf(q.y))), step_both(sm));       // whole numbers below 2^16: their products are exact
            const float2 old = mul(mul(c, c), step_both(sv));
            v2 = mul(old, old);
        }
        m2 = step_add(mul(m2, step_both(r.b1)), mul(g2, step_both(r.b1_rest)));
        v2 = step_add(mul(v2, step_both(r.b2)), mul(mul(g2, g2), step_both(r.b2_rest)));
        const float2 root = near ? make_float2(sqrt_near(v2.x), sqrt_near(v2.y)) : make_float2(__fsqrt_rn(v2.x), __fsqrt_rn(v2.y));
        const float2 under = step_add(mul(root, step_both(r.root_scale)), step_both(r.eps));
        step = kSmall ? mul(m2, make_float2(rcp_near(under.x), rcp_near(under.y))) : make_float2(__fdiv_rn(m2.x, under.x), __fdiv_rn(m2.y, under.y));
        p2 = step_add(mul(p2, step_both(r.keep)), mul(step, step_both(-r.rate)));
        p[j] = p2.x;
        p[j + 1] = p2.y;
        m[j] = m2.x;
        m[j + 1] = m2.y;
        v[j] = v2.x;
        v[j + 1] = v2.y;
    }

    if constexpr (FAST) {
        Raw<DT, N> out;
        out.round(p);
        out.store(param + lane * N);
        Raw<CLPK_DT_F32, N> raw;
        if constexpr (MASTER) {
            raw.round(p);
            raw.store(master + lane * N);
        }
        if constexpr (!kSmall) {
            raw.round(m);
            raw.store(static_cast<float *>(t.m) + block + lane * N);
            raw.round(v);
            raw.store(static_cast<float *>(t.v) + block + lane * N);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (mine(j) < left) {
                param[mine(j)] = P::round(p[j]);
                if constexpr (MASTER)
                    master[mine(j)] = p[j];
                if constexpr (!kSmall) {
                    static_cast<float *>(t.m)[block + mine(j)] = m[j];
                    static_cast<float *>(t.v)[block + mine(j)] = v[j];
                }
            }
    }

    if constexpr (kSmall) {
        float most_m = 0.0f, most_v = 0.0f, least_v = v[0];
#pragma unroll
        for (int j = 0; j < N; j += 2) {                // behind the last element m and v are what became of zeros: zeros, or NaN by a factor that is none
            const bool a = FAST || mine(j) < left, b = FAST || mine(j + 1) < left;
            most_m = step_max(most_m, a ? fabsf(m[j]) : 0.0f, b ? fabsf(m[j + 1]) : 0.0f);
            most_v = step_max(most_v, a ? v[j] : 0.0f, b ? v[j + 1] : 0.0f);
            least_v = fminf(least_v, fminf(v[j], v[j + 1]));
        }
        const uint32_t top_m = __reduce_max_sync(0xffffffffu, __float_as_uint(most_m)), top_v = __reduce_max_sync(0xffffffffu, __float_as_uint(most_v));
        // the largest root is that of the largest v; where that is below 2^-90, roots that are near lose what lies below 2^-126
        const bool low = top_v < 0x12800000u;
        const float im = step_scale<127>(top_m, sm), iv = step_scale<255>(__float_as_uint(__fsqrt_rn(__uint_as_float(top_v))), sv);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float2 c[2] = {};
            const auto word = [&](float inverse) {
                const uint32_t w = __byte_perm(__byte_perm(__float_as_uint(c[0].x), __float_as_uint(c[0].y), 0x0040),
                                               __byte_perm(__float_as_uint(c[1].x), __float_as_uint(c[1].y), 0x0040), 0x5410);
                return inverse > 0.0f ? w : 0u;
            };
            const float2 m4[2] = {make_float2(m[4 * h], m[4 * h + 1]), make_float2(m[4 * h + 2], m[4 * h + 3])};
            const float2 v4[2] = {make_float2(v[4 * h], v[4 * h + 1]), make_float2(v[4 * h + 2], v[4 * h + 3])};
            step_codes<false>(c, m4, im, r.none, false);
            qm[h] = word(im);
            step_codes<true>(c, v4, iv, r.none, low);
            qv[h] = word(iv);
            if (least_v == 0.0f)                        // of a v of 0 the code is 0
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (v[4 * h + j] == 0.0f)
                        qv[h] &= ~(0xFFu << (8 * j));
        }
        if (lane == 0 && (FAST || left > 0)) {
            t.m_scale[block / CLPK_ADAMW_BLOCK] = sm;
            t.v_scale[block / CLPK_ADAMW_BLOCK] = sv;
        }
        if constexpr (FAST) {
            *reinterpret_cast<uint2 *>(static_cast<int8_t *>(t.m) + block + lane * N) = make_uint2(qm[0], qm[1]);
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(t.v) + block + lane * N) = make_uint2(qv[0], qv[1]);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (mine(j) < left) {
                    static_cast<int8_t *>(t.m)[block + mine(j)] = (int8_t)(qm[j / 4] >> (8 * (j & 3)));
                    static_cast<uint8_t *>(t.v)[block + mine(j)] = (uint8_t)(qv[j / 4] >> (8 * (j & 3)));
                }
        }
    }
}

// CTAs an SM: what the registers allow.  With moments in 8 bits six, 40 registers a thread, were 683 us where four took 770 (12 bytes an element),
// although 36 to 56 bytes a thread are spilled with 40.
template <int DT, int GDT, int SDT, bool MASTER, int CAP>
__global__ void __launch_bounds__(kStepThreads, SDT == CLPK_DT_I8 ? 6 : 4) adamw_kernel(const __grid_constant__ StepTable<CAP> table)
{
    __shared__ StepRates told;
    griddep_wait();
    griddep_launch_dependents();
    // the last tensor whose first chunk is not behind this one
    uint32_t lo = 0, hi = table.c.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((table.first[mid] & ~kStepAligned) <= blockIdx.x)
            lo = mid;
        else
            hi = mid;
    }
    const StepTensor &t = table.tensors[lo];
    const uint64_t at = (uint64_t)(blockIdx.x - (table.first[lo] & ~kStepAligned)) * kStepChunk + (threadIdx.x & ~31u) * kStepElems;
    StepRates r = table.c.rates;
    if (table.c.d_lr || table.c.d_step) {
        if (threadIdx.x == 0) {
            const double lr = table.c.d_lr ? (double)*table.c.d_lr : table.c.lr;
            set_rates(told, lr, table.c.beta1, table.c.beta2, table.c.decay, table.c.d_step ? (double)max(*table.c.d_step, 1u) : (double)table.c.step);
        }
        __syncthreads();
        r.keep = told.keep;
        r.root_scale = told.root_scale;
        r.rate = told.rate;
    }
    const float grad_scale = table.c.grad_scale ? *table.c.grad_scale : 1.0f;
    if (at >= t.n)                                      // whole warps, behind the last barrier
        return;
    const uint64_t left = t.n - at;
    if ((table.first[lo] & kStepAligned) && left >= CLPK_ADAMW_BLOCK)
        step_elements<DT, GDT, SDT, MASTER, true>(t, r, grad_scale, at, CLPK_ADAMW_BLOCK);
    else
        step_elements<DT, GDT, SDT, MASTER, false>(t, r, grad_scale, at, left < CLPK_ADAMW_BLOCK ? (uint32_t)left : CLPK_ADAMW_BLOCK);
}

// ---- host side ------------------------------------------------------------------------------------------

constexpr uint64_t kStepMostChunks = 0x7FFFFFFFu;       // of a launch

template <int DT, int GDT, int SDT, bool MASTER, int CAP>
static int launch_step(StepTable<CAP> &table, const clpk_adamw_tensor_t *tensors, uint32_t count, cudaStream_t s)
{
    uint64_t chunks = 0;
    const auto flush = [&]() {
        const int rc = table.c.count ? launch_behind(adamw_kernel<DT, GDT, SDT, MASTER, CAP>, "adamw", (unsigned)chunks, kStepThreads, 0, s, table) : CLPK_OK;
        table.c.count = 0;
        chunks = 0;
        return rc;
    };
    for (uint32_t i = 0; i < count; i++) {
        const clpk_adamw_tensor_t &t = tensors[i];
        const uint64_t own = (t.n + kStepChunk - 1) / kStepChunk;
        if (own == 0)
            continue;
        if (table.c.count == CAP || chunks + own > kStepMostChunks)
            CLPK_TRY(flush());
        uintptr_t at = (uintptr_t)t.d_param | (uintptr_t)t.d_grad | (uintptr_t)t.d_master;
        if (SDT == CLPK_DT_F32)
            at |= (uintptr_t)t.d_m | (uintptr_t)t.d_v;
        const bool aligned = at % 16 == 0 && (SDT == CLPK_DT_F32 || ((uintptr_t)t.d_m | (uintptr_t)t.d_v) % 8 == 0);
        table.tensors[table.c.count] = {t.n, t.d_param, t.d_grad, t.d_master, t.d_m, t.d_v, t.d_m_scale, t.d_v_scale};
        table.first[table.c.count++] = (uint32_t)chunks | (aligned ? kStepAligned : 0);
        chunks += own;
    }
    return flush();
}

template <int DT, int GDT, int SDT, bool MASTER>
static int run_step(const StepCommon &c, const clpk_adamw_tensor_t *tensors, uint32_t count, cudaStream_t s)
{
    const auto with = [&](auto &table) {
        table.c = c;
        return launch_step<DT, GDT, SDT, MASTER>(table, tensors, count, s);
    };
    StepTable<kStepFew> few;                            // the less to send along with the launch: 64 tensors 5.7 us with room for 440
    StepTable<kStepSome> some;
    StepTable<kStepMany> many;
    return count <= kStepFew ? with(few) : count <= kStepSome ? with(some) : with(many);
}

template <int DT, int GDT>
static int run_step_by(const StepCommon &c, int state, bool master, const clpk_adamw_tensor_t *tensors, uint32_t count, cudaStream_t s)
{
    if constexpr (DT != CLPK_DT_F32)
        if (master)
            return state == CLPK_DT_I8 ? run_step<DT, GDT, CLPK_DT_I8, true>(c, tensors, count, s) : run_step<DT, GDT, CLPK_DT_F32, true>(c, tensors, count, s);
    return state == CLPK_DT_I8 ? run_step<DT, GDT, CLPK_DT_I8, false>(c, tensors, count, s) : run_step<DT, GDT, CLPK_DT_F32, false>(c, tensors, count, s);
}

static int check_part(uint32_t i, const char *name, const void *base, uint64_t elem)
{
    CLPK_REQUIRE(base && (uintptr_t)base % elem == 0, "clpk_adamw: %s of tensor %u is NULL or not aligned to its elements", name, i);
    return CLPK_OK;
}

static int check_step_tensor(const clpk_adamw_args_t &a, uint32_t i, bool master)
{
    const clpk_adamw_tensor_t &t = a.h_tensors[i];
    if (t.n == 0)
        return CLPK_OK;
    CLPK_REQUIRE(t.n <= 1ull << 40, "clpk_adamw: tensor %u has %llu elements", i, (unsigned long long)t.n);
    CLPK_TRY(check_part(i, "d_param", t.d_param, element_bytes(a.dtype)));
    CLPK_TRY(check_part(i, "d_grad", t.d_grad, element_bytes(a.grad_dtype)));
    CLPK_REQUIRE((t.d_master != nullptr) == master, "clpk_adamw: d_master: give it for every tensor, or for none (tensor %u)", i);
    if (master)
        CLPK_TRY(check_part(i, "d_master", t.d_master, 4));
    const uint64_t state = element_bytes(a.state_dtype);
    CLPK_TRY(check_part(i, "d_m", t.d_m, state));
    CLPK_TRY(check_part(i, "d_v", t.d_v, state));
    if (a.state_dtype == CLPK_DT_I8) {
        CLPK_TRY(check_part(i, "d_m_scale", t.d_m_scale, 4));
        CLPK_TRY(check_part(i, "d_v_scale", t.d_v_scale, 4));
    }
    return CLPK_OK;
}

} // namespace clpk

using namespace clpk;

extern "C" int clpk_adamw(const clpk_adamw_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_adamw";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    const clpk_adamw_args_t &a = *args;
    CLPK_REQUIRE(a.dtype == CLPK_DT_F32 || a.dtype == CLPK_DT_F16 || a.dtype == CLPK_DT_BF16, "%s: dtype %d is not F32, F16 or BF16", what, a.dtype);
    CLPK_REQUIRE(a.grad_dtype == a.dtype || a.grad_dtype == CLPK_DT_F32, "%s: grad_dtype %d is neither dtype nor F32", what, a.grad_dtype);
    CLPK_REQUIRE(a.state_dtype == CLPK_DT_F32 || a.state_dtype == CLPK_DT_I8, "%s: state_dtype %d is not F32 or I8", what, a.state_dtype);
    CLPK_REQUIRE(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0, "%s: beta1 %g, beta2 %g: both in [0, 1)", what, a.beta1, a.beta2);
    CLPK_REQUIRE(a.eps >= 1.17549435e-38 && a.eps < 1e30, "%s: eps %g is not in [2^-126, 1e30)", what, a.eps);
    CLPK_REQUIRE(std::isfinite(a.weight_decay) && a.weight_decay >= 0.0 && (a.d_lr || (std::isfinite(a.lr) && a.lr >= 0.0)), "%s: lr %g, weight_decay %g", what, a.lr, a.weight_decay);
    CLPK_REQUIRE(a.d_step || a.step > 0, "%s: steps are counted from 1", what);
    CLPK_REQUIRE((uintptr_t)a.d_lr % 4 == 0 && (uintptr_t)a.d_step % 4 == 0 && (uintptr_t)a.d_grad_scale % 4 == 0, "%s: d_lr, d_step or d_grad_scale is not aligned to its elements", what);
    CLPK_REQUIRE(a.count == 0 || a.h_tensors, "%s: h_tensors is NULL", what);
    bool master = false;
    for (uint32_t i = 0; i < a.count && !master; i++)
        master = a.h_tensors[i].n > 0 && a.h_tensors[i].d_master;
    CLPK_REQUIRE(!master || a.dtype != CLPK_DT_F32, "%s: parameters in fp32 have no master copies", what);
    for (uint32_t i = 0; i < a.count; i++)
        CLPK_TRY(check_step_tensor(a, i, master));

    StepCommon c = {};
    c.rates.b1 = (float)a.beta1;
    c.rates.b1_rest = (float)(1.0 - a.beta1);
    c.rates.b2 = (float)a.beta2;
    c.rates.b2_rest = (float)(1.0 - a.beta2);
    c.rates.eps = (float)a.eps;
    c.rates.none = -0.0f;
    if (!a.d_lr && !a.d_step)
        set_rates(c.rates, a.lr, a.beta1, a.beta2, a.weight_decay, (double)a.step);
    c.lr = a.lr;
    c.beta1 = a.beta1;
    c.beta2 = a.beta2;
    c.decay = a.weight_decay;
    c.step = a.step;
    c.d_lr = a.d_lr;
    c.d_step = a.d_step;
    c.grad_scale = a.d_grad_scale;
    cudaStream_t s = as_stream(stream);
    if (a.dtype == CLPK_DT_F32)
        return run_step_by<CLPK_DT_F32, CLPK_DT_F32>(c, a.state_dtype, master, a.h_tensors, a.count, s);
    if (a.dtype == CLPK_DT_BF16)
        return a.grad_dtype == CLPK_DT_F32 ? run_step_by<CLPK_DT_BF16, CLPK_DT_F32>(c, a.state_dtype, master, a.h_tensors, a.count, s)
                                           : run_step_by<CLPK_DT_BF16, CLPK_DT_BF16>(c, a.state_dtype, master, a.h_tensors, a.count, s);
    return a.grad_dtype == CLPK_DT_F32 ? run_step_by<CLPK_DT_F16, CLPK_DT_F32>(c, a.state_dtype, master, a.h_tensors, a.count, s)
                                       : run_step_by<CLPK_DT_F16, CLPK_DT_F16>(c, a.state_dtype, master, a.h_tensors, a.count, s);
}
