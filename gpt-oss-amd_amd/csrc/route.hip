// Routing by score: router logits -> the experts of every token and their weights, for rules other than "softmax over the largest
// logits" (router.hip): softmax or sigmoid scores, a bias that takes part in the choice only, groups of experts, weights
// renormalised over the chosen and scaled.
#include "common.h"
#include "kernels.h"
#include "topk.h"

namespace moe {

namespace {

// Sort key of a choice value: as rank_key, and a value that is not a number above all others.
MOE_DEVICE uint32_t choice_key(float c) { return c == c ? rank_key(c) : 0xFFFFFFFFu; }
MOE_DEVICE float choice_value(uint32_t key) { return key == 0xFFFFFFFFu ? NAN : rank_key_value(key); }

}  // namespace

// A wave per token, C values to a lane: expert 64 c + lane.
//   s = 1 / (1 + exp(-l))  or  exp(l - max) / sum, in fp64, rounded to fp32 once: scores that differ in their last place decide between
//   experts, and a rule stated on rounded scores has one answer whatever computes it
//   c = s + bias; group value = sum of the group_top largest c of its experts; the groups_per_token largest groups stay
//   K largest c of the groups that stay (equal ones: the lower index); weight = s / (sum over the chosen) * scale
template <int C>
__global__ __launch_bounds__(256) void route_kernel(const float* __restrict__ logits, float* __restrict__ topk_v, int* __restrict__ topk_i,
                                                    int T, int E, int K, RouteRule rule) {
    __shared__ float score_s[4][64 * C];
    __shared__ uint32_t key_s[4][64 * C];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * 4 + wave;
    if (t >= T) return;
    float* const score = score_s[wave];
    uint32_t* const keys = key_s[wave];
    const float* row = logits + (size_t)t * E;
    float l[C], s[C];
#pragma unroll
    for (int c = 0; c < C; ++c) l[c] = lane + 64 * c < E ? row[lane + 64 * c] : -INFINITY;
    if (rule.scoring == MOE_ROUTE_SOFTMAX) {
        uint32_t best = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) best = max(best, choice_key(l[c]));
#define MOE_STEP(CTRL, M) best = max(best, dpp_move<CTRL, M>(0u, best));
        MOE_DPP_STEPS(MOE_STEP)
#undef MOE_STEP
        const double mx = (double)choice_value(__builtin_amdgcn_readlane(best, 63));
        double e[C], sum = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            e[c] = l[c] == -INFINITY ? 0.0 : exp((double)l[c] - mx);
            sum += e[c];
        }
        sum = wave_sum(sum);
        const double inv = sum == 0.0 ? 0.0 : 1.0 / sum;  // every expert masked: scores of zero
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = (float)(e[c] * inv);
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = (float)(1.0 / (1.0 + exp(-(double)l[c])));
    }
    uint32_t key[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int e = lane + 64 * c;
        key[c] = 0u;
        if (e < E) {
            key[c] = choice_key(rule.bias ? s[c] + rule.bias[e] : s[c]);
            score[e] = s[c];
            keys[e] = key[c];
        }
    }
    lds_in_order();
    if (rule.n_groups > 1) {
        const int size = E / rule.n_groups;
        uint32_t first = 0, second = 0;
        if (lane < rule.n_groups)
            for (int i = 0; i < size; ++i) {
                const uint32_t k = keys[lane * size + i];
                second = max(second, min(first, k));
                first = max(first, k);
            }
        uint32_t value = 0;
        if (lane < rule.n_groups) {
            float v = choice_value(first);
            if (rule.group_top == 2 && size > 1) v += choice_value(second);
            value = choice_key(v);
        }
        unsigned long long kept = 0;
        for (int r = 0; r < rule.groups_per_token; ++r) {
            uint32_t best = value;
#define MOE_STEP(CTRL, M) best = max(best, dpp_move<CTRL, M>(0u, best));
            MOE_DPP_STEPS(MOE_STEP)
#undef MOE_STEP
            best = __builtin_amdgcn_readlane(best, 63);
            const int g = (int)__builtin_ctzll(__ballot(value == best));
            kept |= 1ull << g;
            if (lane == g) value = 0;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = lane + 64 * c;
            if (e < E && !((kept >> (e / size)) & 1)) key[c] = 0;
        }
    }
    int my_i = 0;
    for (int r = 0; r < K; ++r) {
        uint32_t best = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) best = max(best, key[c]);
#define MOE_STEP(CTRL, M) best = max(best, dpp_move<CTRL, M>(0u, best));
        MOE_DPP_STEPS(MOE_STEP)
#undef MOE_STEP
        best = __builtin_amdgcn_readlane(best, 63);
        int bi = 0;
#pragma unroll
        for (int c = C - 1; c >= 0; --c) {
            const unsigned long long has = __ballot(key[c] == best);
            if (has) bi = 64 * c + (int)__builtin_ctzll(has);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) key[c] = bi == lane + 64 * c ? 0u : key[c];
        if (lane == r) my_i = bi;
    }
    double w = lane < K ? (double)score[my_i] : 0.0;
    if (rule.renormalize) {
        double sum = 0.0;
        for (int r = 0; r < K; ++r) sum += (double)lane_value((float)w, r);
        w = sum == 0.0 ? 0.0 : w / sum;
    }
    if (lane < K) {
        topk_v[(size_t)t * K + lane] = (float)(w * (double)rule.scale);
        topk_i[(size_t)t * K + lane] = my_i;
    }
}

int launch_route(const float* logits, float* topk_v, int* topk_i, int T, int E, int K, const RouteRule& rule, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(T, 4));
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, logits, topk_v, topk_i, T, E, K, rule);
        return launch_status();
    };
    if (E <= 64) return launch(route_kernel<1>);
    if (E <= 128) return launch(route_kernel<2>);
    if (E <= 256) return launch(route_kernel<4>);
    if (E <= 512) return launch(route_kernel<8>);
    return launch(route_kernel<16>);
}

}  // namespace moe
