// TEST PROGRAM: how the feed-forward products of given sizes are cut on a B200, from the product's own planning code, without a GPU.
// Reads lines "<form> <tokens> <k> <n>", writes one line for each; forms: g / i gated in 16 / 8 bits, s scaled 8 bits, b backward
// (tokens, model width, hidden width).  Exit code: launches whose shared memory or tensor memory would not fit.
#include "kernels/feed_forward.cu"

#include <cstdio>

namespace clpk {
void set_error(const char *, ...) {}
int cuda_fail(cudaError_t, const char *) { return CLPK_ERR_CUDA; }
int require_sm100() { return CLPK_ERR_NO_DEVICE; }
int num_sms() { return 148; }
int tuning(int) { return -1; }
} // namespace clpk

static int g_unfit = 0;

template <LinearForm FORM> static void forward(uint32_t m, uint32_t k, uint32_t n, int dtype)
{
    const uint32_t k_blocks = linear_k_blocks(k, dtype), sms = (uint32_t)num_sms(), tiles = ceil_div(n, few_cols<FORM>);
    if (few_tokens(m, tiles, k_blocks, sms)) {
        FewParams p = {};
        p.m = m;
        p.n = n;
        p.k_blocks = k_blocks;
        plan_few(p, tiles, sms);
        const uint32_t stage = kHalfTileBytes + p.tokens * kRowBytesK, sums = p.splits * ((m + p.splits - 1) / p.splits) * kFewRows * 4;
        if (p.stages < 2 || p.splits > k_blocks || p.smem_bytes + sizeof(FewSmem) + 1024 > kSmemMax || p.stages * stage > p.smem_bytes ||
            p.sums_at + (p.splits > 1 ? sums : p.tokens * kFewRows * 4) > p.smem_bytes || (p.sums_at && p.sums_at < p.stages * stage))
            g_unfit++;
        std::printf("few ranges %u%s\n", p.splits, p.splits == 1 ? "" : p.sums_at ? " sums behind the ring" : " sums in the ring");
    } else {
        Product w = {};
        w.m = m;
        w.n = n;
        w.k = k;
        const LinearPlan plan = plan_linear(w, FORM, k_blocks);
        const uint32_t cols = FORM == kGated ? plan.tn / 2 : plan.tn, all = ceil_div(m, kLinearM) * ceil_div(n, cols);
        // the sums that a pair is sent: a chunk of 32 columns of 128 rows for each other pair and each of its own chunks
        const uint32_t units = cols / kLinearChunk, slots = (units + plan.splits - 1) / plan.splits, subs = FORM == kGated ? 2 : 1;
        if (plan.splits > k_blocks || (plan.splits - 1) * slots * subs * kLinearChunk * 128 * 4 > linear_stages(plan.tn) * linear_kps(plan.tn) * linear_block_bytes(plan.tn))
            g_unfit++;
        std::printf("pairs columns %u ranges %u%s\n", plan.tn, plan.splits, plan.splits > 1 ? "" : all > sms / 2 ? " several tiles" : " one tile");
    }
}

static void backward(uint32_t m, uint32_t d, uint32_t f)
{
    const GradPlan plan = plan_backward(m, d, f);
    const GradTiles x = x_tiles(m, d, f, plan.tn, plan.x_parts), w = w_tiles(m, d, f, plan.tn, plan.w_parts);
    const bool x_first = &longer(x, w) == &x;
    const GradTiles &first = x_first ? x : w, &second = x_first ? w : x;
    // every tile has a cluster
    const uint32_t clusters = std::min(x.tiles + w.tiles, kGradPairs), more = first.tiles % clusters;
    uint32_t a = 0, b = 0;
    share_tiles(first, second, clusters, a, b);
    if (b < a || (uint64_t)a * clusters + (uint64_t)(b - a) * (clusters - more) < second.tiles || (x.tiles + w.tiles <= kGradPairs && (more ? (a || b > 1) : b)))
        g_unfit++;
    std::printf("gradients columns %u dx %u dw %u first %s\n", plan.tn, plan.x_parts, plan.w_parts, x_first ? "dx" : "dw");
}

int main()
{
    char form;
    unsigned m, k, n;
    while (std::scanf(" %c %u %u %u", &form, &m, &k, &n) == 4) {
        switch (form) {
        case 'g': forward<kGated>(m, k, n, CLPK_DT_BF16); break;
        case 'i': forward<kGated>(m, k, n, CLPK_DT_I8); break;
        case 's': forward<kScaled>(m, k, n, CLPK_DT_I8); break;
        default:  backward(m, k, n); break;
        }
    }
    return g_unfit > 255 ? 255 : g_unfit;
}
