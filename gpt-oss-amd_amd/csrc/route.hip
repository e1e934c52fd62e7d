// Routing by score: router logits -> the experts of every token and their weights, for rules other than "softmax over the largest
// logits" (router.hip): softmax or sigmoid scores, a bias that takes part in the choice only, groups of experts, weights
// renormalised over the chosen and scaled.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "topk.h"

namespace moe {

namespace {

// Sort key of a choice value: as rank_key, a value that is not a number as +infinity.
MOE_DEVICE uint32_t choice_key(float c) { return rank_key(c == c ? c : INFINITY); }

struct RouteCut {
    int log_group_lanes;  // lanes of a group
    int group_size, per_lane;
    int wide;  // a lane's logits in pieces of 16 bytes
};

// ---- scores ---------------------------------------------------------------------------------------
// exp(x) for |x| <= 139, to 2^-52: 2^f from the polynomial that meets it at the twelve Chebyshev nodes of -1/2 .. 1/2 (2^-57; as many terms of the
// Taylor series give 2^-47), f = x log2(e) less the whole number next to it, log2(e) in two parts.
MOE_DEVICE double exp_series(double x) {
    const double n = __builtin_rint(x * 0x1.71547652b82fep+0);
    const double f = fma(x, 2.0355273740931033e-17, fma(x, 0x1.71547652b82fep+0, -n));
    double p = 0x1.e9ec1fcb69a7fp-32;
    p = fma(p, f, 0x1.e6228acd1c6e5p-28);
    p = fma(p, f, 0x1.b524ebd13a55fp-24);
    p = fma(p, f, 0x1.62bfc2c86d700p-20);
    p = fma(p, f, 0x1.ffcbfc6da6ed1p-17);
    p = fma(p, f, 0x1.430913112c61bp-13);
    p = fma(p, f, 0x1.5d87fe78a3f9cp-10);
    p = fma(p, f, 0x1.3b2ab6fb9f1a5p-7);
    p = fma(p, f, 0x1.c6b08d704a0c6p-5);
    p = fma(p, f, 0x1.ebfbdff82c5aep-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// 1 / d for 1 <= d < 2^250: the hardware's estimate (2^-24) and a step of third order.
MOE_DEVICE double reciprocal(double d) {
    const double r = __builtin_amdgcn_rcp(d), e = fma(-d, r, 1.0);
    return fma(r, fma(e, e, e), r);
}

// 1 / (1 + exp(-l)) to 2^-51, rounded to fp32 once.  Past 130 either way the result is 0 or 1 in fp32.
MOE_DEVICE float sigmoid_score(float l) {
    const float near = fminf(fmaxf(l, -130.f), 130.f);
    const float s = (float)reciprocal(1.0 + exp_series(-(double)near));
    return l == l ? s : l;
}

// exp(l - mx), from exp(-138) on: what is less is 0 in fp32 whatever it is divided by.  (An infinite mx leaves no number above that.)
MOE_DEVICE double softmax_term(float l, double mx) { return exp_series(fmax((double)l - mx, -138.0)); }

// A row's sum of terms in whole numbers of 2^-52 (terms are 0 .. 1), so that it does not depend on how the row lies over lanes, and a token
// gets the same bits in a batch of any size: the bits of 1 + term rise by one for each.
MOE_DEVICE uint64_t term_units(double e) { return __builtin_bit_cast(uint64_t, e + 1.0) - __builtin_bit_cast(uint64_t, 1.0); }

// What the terms of a row with largest logit mx (+infinity if it holds a NaN) are multiplied by: 0 where all logits are -infinity.
MOE_DEVICE double softmax_scale(float mx, uint64_t units) {
    if (mx == -INFINITY) return 0.0;
    return mx < INFINITY ? reciprocal((double)units * 0x1p-52) : (double)NAN;
}

// ---- values with their place ------------------------------------------------------------------------
// A choice value and its place as one double, which v_max_f64 ranks by value and then by lower place: an fp32 value leaves 29 bits of the
// double's mantissa free.  Infinities become +-2^1023, past all fp32 values; a NaN counts as +infinity.
constexpr int kPlaceBits = 10;
constexpr uint32_t kPlaceMask = (1u << kPlaceBits) - 1u;
MOE_DEVICE double make_double(uint32_t hi, uint32_t lo) { return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo); }
MOE_DEVICE uint32_t low_word(double d) { return (uint32_t)__builtin_bit_cast(uint64_t, d); }
MOE_DEVICE uint32_t high_word(double d) { return (uint32_t)(__builtin_bit_cast(uint64_t, d) >> 32); }
MOE_DEVICE double no_choice() { return make_double(0xFFEFFFFFu, 0xFFFFFFFFu); }  // below all choices

MOE_DEVICE double choice_with_place(float c, int place) {
    const double d = fmax(fmin((double)(c + 0.f), 0x1p1023), -0x1p1023);
    const uint32_t lo = low_word(d), hi = high_word(d);
    return make_double(hi, lo | (((uint32_t)place ^ ~(uint32_t)((int32_t)hi >> 31)) & kPlaceMask));
}
MOE_DEVICE int place_of(double d) { return (int)((low_word(d) ^ ~(uint32_t)((int32_t)high_word(d) >> 31)) & kPlaceMask); }

// ---- exchange between lanes ------------------------------------------------------------------------
// v of another lane of the row of 16, for controls that give every lane one.
template <int CTRL>
MOE_DEVICE double dpp_double(double v) {
    return make_double((uint32_t)__builtin_amdgcn_mov_dpp((int)high_word(v), CTRL, 0xf, 0xf, true),
                       (uint32_t)__builtin_amdgcn_mov_dpp((int)low_word(v), CTRL, 0xf, 0xf, true));
}
// The larger and the smaller of two numbers.  (fmax and fmin quiet their arguments first, an instruction each: nothing here is a NaN.)
MOE_DEVICE double larger(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
MOE_DEVICE double smaller(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// Two doubles whose larger, lane by lane, is that of a lane and of the one 16 (or 32) further on, modulo twice that.
template <int LANES>
MOE_DEVICE void swap_double(double v, double& x, double& y) {
    const uint32_t hi = high_word(v), lo = low_word(v);
    if constexpr (LANES == 16) {
        const auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false), l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
        x = make_double(h[0], l[0]), y = make_double(h[1], l[1]);
    } else {
        const auto h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false), l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
        x = make_double(h[0], l[0]), y = make_double(h[1], l[1]);
    }
}

// Every lane of the LPT (16, 32 or 64) that share a token gets op over all of them.  Rotations of the row of 16, then rows.
template <int LPT, class Op>
MOE_DEVICE double token_reduce(double v, Op op) {
    v = op(v, dpp_double<0x128>(v));
    v = op(v, dpp_double<0x124>(v));
    v = op(v, dpp_double<0x122>(v));
    v = op(v, dpp_double<0x121>(v));
    double x, y;
    if constexpr (LPT >= 32) {
        swap_double<16>(v, x, y);
        v = op(x, y);
    }
    if constexpr (LPT >= 64) {
        swap_double<32>(v, x, y);
        v = op(x, y);
    }
    return v;
}

template <int LPT>
MOE_DEVICE uint64_t token_sum(uint64_t v) {
    const double sum = token_reduce<LPT>(__builtin_bit_cast(double, v), [](double a, double b) {
        return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, a) + __builtin_bit_cast(uint64_t, b));
    });
    return __builtin_bit_cast(uint64_t, sum);
}

// (a, b) in descending order
MOE_DEVICE void descending(double& a, double& b) {
    const double hi = larger(a, b), lo = smaller(a, b);
    a = hi;
    b = lo;
}

// d[FROM .. FROM + N) in descending order, N a power of two: merges of sorted halves, the pairs of Batcher's odd-even merge, those K
// apart, K = N / 2 .. 1, one after the other.  (K is a template parameter: a loop that halves it is not unrolled, and d then indexed at run time.)
template <int FROM, int N, int K, int V>
MOE_DEVICE void merge_pairs(double (&d)[V]) {
#pragma unroll
    for (int j = K == N / 2 ? 0 : K; j + K < N; j += 2 * K)
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (j + i + K < N) descending(d[FROM + j + i], d[FROM + j + i + K]);
    if constexpr (K > 1) merge_pairs<FROM, N, K / 2>(d);
}
template <int FROM, int N, int V>
MOE_DEVICE void sort_descending(double (&d)[V]) {
    if constexpr (N > 1) {
        sort_descending<FROM, N / 2>(d);
        sort_descending<FROM + N / 2, N / 2>(d);
        merge_pairs<FROM, N, N / 2>(d);
    }
}
// A bitonic run of N in descending order.
template <int FROM, int N, int V>
MOE_DEVICE void sort_bitonic(double (&d)[V]) {
    if constexpr (N > 1) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) descending(d[FROM + i], d[FROM + i + N / 2]);
        sort_bitonic<FROM, N / 2>(d);
        sort_bitonic<FROM + N / 2, N / 2>(d);
    }
}
// The KC largest of d[FROM .. FROM + N) in descending order at d[FROM ..): of two sorted runs of KC, the larger of each and of the other
// run's opposite are a bitonic run of the KC largest.
template <int FROM, int N, int KC, int V>
MOE_DEVICE void top_descending(double (&d)[V]) {
    if constexpr (N <= KC) {
        sort_descending<FROM, N>(d);
    } else {
        top_descending<FROM, N / 2, KC>(d);
        top_descending<FROM + N / 2, N / 2, KC>(d);
#pragma unroll
        for (int i = 0; i < KC; ++i) d[FROM + i] = larger(d[FROM + i], d[FROM + N / 2 + KC - 1 - i]);
        sort_bitonic<FROM, KC>(d);
    }
}

}  // namespace

// LPT lanes to a token (64 / LPT tokens to a wave), up to V experts to a lane, a group of experts in whole lanes.
//   s = 1 / (1 + exp(-l))  or  exp(l - max) / sum, in fp64, rounded to fp32 once: scores that differ in their last place decide between
//   experts, and a rule stated on rounded scores has one answer whatever computes it to fp64's accuracy (but for one score in some 2^26 that lies that
//   near the middle of two fp32 numbers)
//   c = s + bias; group value = sum of the group_top largest c of its experts; the groups_per_token largest groups stay
//   K largest c of the groups that stay (equal ones: the lower index); weight = s / (sum over the chosen) * scale
// Bound by its instructions: some 28 in 64 bits for every score, 300 a token (of 256 experts, 8 of them chosen) for the selection.  A lane sorts its
// values once; a round of the selection is then a maximum over the first of every lane's, and the lane that had it moves up its next.
// 16384 tokens of 256 experts: a wave a token, keys searched in every round, the library's exponential 24.6 us, so 12.4 (2.4 of them are
// an empty launch's); 2.6 would be the logits at the rate of a long read.
template <int LPT, int V, int KMAX>
__global__ __launch_bounds__(256) void route_kernel(const float* __restrict__ logits, float* __restrict__ topk_v, int* __restrict__ topk_i, int T,
                                                    int E, int K, RouteRule rule, RouteCut cut) {
    constexpr int KC = V < KMAX ? V : KMAX;  // the most that a lane can win
    constexpr int kTokens = 256 / LPT;
    __shared__ __attribute__((aligned(16))) float score_s[kTokens][LPT * V];  // by place: lane of the token x V + v, the order of the experts
    __shared__ __attribute__((aligned(16))) float value_s[kTokens][64];
    const int slot = threadIdx.x / LPT, in_token = threadIdx.x & (LPT - 1);
    // the lane's experts: first .. first + n - 1
    const int group_lanes = 1 << cut.log_group_lanes;
    const int group = in_token >> cut.log_group_lanes, within = in_token & (group_lanes - 1);
    const int first = group * cut.group_size + within * cut.per_lane;
    const int n = group < rule.n_groups ? min(cut.per_lane, cut.group_size - within * cut.per_lane) : 0;
    // Loads and LDS writes go without branches: what lies past a lane's experts is another's or, past the buffer's end, 0, and no token past
    // the last is stored; they go along because tokens share their waves' exchanges.
    const __amdgpu_buffer_rsrc_t b_rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(rule.bias), 0, rule.bias ? E * 4 : 0, 0x00020000);
    const int t0 = blockIdx.x * kTokens, t = t0 + slot;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(logits) + (size_t)t0 * E, 0,
                                                                          min(kTokens, T - t0) * E * 4, 0x00020000);
    const int at = (slot * E + first) * 4;
    float s[V], bias[V];
    if (V >= 4 && cut.wide) {  // whole 16 bytes
#pragma unroll
        for (int v = 0; v + 3 < V; v += 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 4 * v, 0);
            const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, first * 4, 4 * v, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[v + i] = __uint_as_float(x[i]), bias[v + i] = __uint_as_float(y[i]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 4 * v, 0));
            bias[v] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b_rsrc, first * 4, 4 * v, 0));
        }
    }
    if (rule.scoring == MOE_ROUTE_SOFTMAX) {
        double most = -INFINITY;
        bool nan = false;  // such a row's scores are NaN, as those of a row with +infinity
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] = v < n ? s[v] : -INFINITY;
            most = fmax(most, (double)s[v]);
            nan |= s[v] != s[v];
        }
        const float mx = (float)token_reduce<LPT>(nan ? (double)INFINITY : most, larger);
        double e[V];
        uint64_t units = 0;  // places without an expert have terms that round to none
#pragma unroll
        for (int v = 0; v < V; ++v) {
            e[v] = softmax_term(s[v], (double)mx);
            units += term_units(e[v]);
        }
        const double scale = softmax_scale(mx, token_sum<LPT>(units));
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = (float)(e[v] * scale);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = sigmoid_score(s[v]);
    }
    float* const score = score_s[slot];
    if constexpr (V >= 4) {
#pragma unroll
        for (int v = 0; v + 3 < V; v += 4) *reinterpret_cast<f32x4*>(score + in_token * V + v) = f32x4{s[v], s[v + 1], s[v + 2], s[v + 3]};
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) score[in_token * V + v] = s[v];
    }
    double d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const double c = choice_with_place(s[v] + bias[v], in_token * V + v);  // without a bias 0 is added
        d[v] = v < n ? c : no_choice();
    }
    top_descending<0, V, KC>(d);
    if (rule.n_groups > 1) {
        // the two largest of the group, in all of its lanes; lanes that differ in one bit of their number at a time
        double a = d[0], b = V > 1 ? d[V > 1 ? 1 : 0] : no_choice();
        auto merge = [&](double a2, double b2) {
            b = larger(smaller(a, a2), larger(b, b2));
            a = larger(a, a2);
        };
        if (cut.log_group_lanes > 0) merge(dpp_double<0xB1>(a), dpp_double<0xB1>(b));
        if (cut.log_group_lanes > 1) merge(dpp_double<0x4E>(a), dpp_double<0x4E>(b));
        if (cut.log_group_lanes > 2) merge(dpp_double<0x141>(a), dpp_double<0x141>(b));
        if (cut.log_group_lanes > 3) merge(dpp_double<0x140>(a), dpp_double<0x140>(b));
        if (LPT > 16 && cut.log_group_lanes > 4) {
            double a1, a2, b1, b2;
            swap_double<16>(a, a1, a2);
            swap_double<16>(b, b1, b2);
            a = a1, b = b1;
            merge(a2, b2);
        }
        // as fp32 again: the index is less than half a step
        float value = (float)a;
        if (rule.group_top == 2 && cut.group_size > 1) value += (float)b;
        value = value == value ? value : INFINITY;
        if (within == 0) value_s[slot][group] = value;
        lds_in_order();
        int better = 0;
        for (int g = 0; g < rule.n_groups; g += 4) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(&value_s[slot][g]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g + i < rule.n_groups) better += o[i] > value || (o[i] == value && g + i < group) ? 1 : 0;
        }
        if (better >= rule.groups_per_token) {
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = no_choice();
        }
    }
    double won = 0.0;
#pragma unroll
    for (int r = 0; r < KMAX; ++r) {
        if (r < K) {  // uniform
            const double best = token_reduce<LPT>(d[0], larger);
            won = in_token == r ? best : won;
            const bool mine = d[0] == best;
#pragma unroll
            for (int v = 0; v < KC; ++v) {
                // values, not places of the array: a choice between places is made by an index at run time
                const double next = v + 1 < KC ? +d[v + 1 < KC ? v + 1 : 0] : no_choice(), same = d[v];
                if (v + r < KMAX - 1) d[v] = mine ? next : same;
            }
        }
    }
    const int place = in_token < K ? place_of(won) : 0;
    lds_in_order();
    double w = (double)score[place];
    if (rule.renormalize) {
        float* const chosen = value_s[slot];
        if (in_token < 8) chosen[in_token] = in_token < K ? (float)w : 0.f;
        lds_in_order();
        double sum = 0.0;
#pragma unroll
        for (int r = 0; r < KMAX; r += 4) {
            const f32x4 c = *reinterpret_cast<const f32x4*>(chosen + r);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += (double)c[i];
        }
        w = sum == 0.0 ? 0.0 : w / sum;
    }
    if (t < T && in_token < K) {
        const int l = place / V, g = l >> cut.log_group_lanes;
        topk_v[(size_t)t * K + in_token] = (float)(w * (double)rule.scale);
        topk_i[(size_t)t * K + in_token] = g * cut.group_size + (l & (group_lanes - 1)) * cut.per_lane + place % V;
    }
}

// Groups that do not fit whole lanes of route_kernel: a wave per token, C values to a lane, expert 64 c + lane; the same rule.
template <int C>
__global__ __launch_bounds__(256) void route_any_kernel(const float* __restrict__ logits, float* __restrict__ topk_v,
                                                        int* __restrict__ topk_i, int T, int E, int K, RouteRule rule) {
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
        const float mx = rank_key_value(__builtin_amdgcn_readlane(best, 63));
        double e[C];
        uint64_t units = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            e[c] = softmax_term(l[c], (double)mx);
            units += term_units(e[c]);
        }
        const double scale = softmax_scale(mx, token_sum<64>(units));
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = (float)(e[c] * scale);
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = sigmoid_score(l[c]);
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
            float v = rank_key_value(first);
            if (rule.group_top == 2 && size > 1) v += rank_key_value(second);
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

// Lanes of a group (log2), where `lpt` lanes share a token.
static int group_lanes_log(int G, int lpt) {
    int log = 0;
    while (G << (log + 1) <= lpt) ++log;
    return log;
}
bool route_fits_lanes(int E, int n_groups) { return ceil_div(E / n_groups, 1 << group_lanes_log(n_groups, 64)) <= 16; }

// Tokens T of a batch of `total`, which is what the lanes of a token go by.
static int launch_route_part(const float* logits, float* topk_v, int* topk_i, int T, int total, int E, int K, const RouteRule& rule, int n_cus,
                             hipStream_t stream) {
    const int G = rule.n_groups, size = E / G;
    // Lanes of a token: the fewer, the less a token's exchanges between lanes cost, as long as there are three waves to a compute unit.  us at 16 :
    // 32 : 64 lanes, 256 experts in 8 groups, K = 8, 1 token 5.0 : 4.3 : 4.0, 512 tokens 5.6 : 4.6 : 4.4, 2000 tokens 5.6 : 4.8 : 5.1, 4096 tokens 6.2 :
    // 6.3 : 7.3, 16384 tokens 12.1 : 13.9 : 18.7; 32 experts, 4096 tokens 3.0 : 3.1 : 3.8.  (8 lanes of 32 experts 12.7; blocks that go through
    // several batches of tokens, the next one's logits in flight, 14.5.)
    int lanes = 16;
    while (lanes < 64 && (long long)total * lanes < 192LL * n_cus) lanes *= 2;
    for (int lpt = lanes; lpt <= 64; lpt *= 2) {
        RouteCut cut;
        if (G > lpt) continue;
        cut.log_group_lanes = group_lanes_log(G, lpt);
        cut.group_size = size;
        cut.per_lane = ceil_div(size, 1 << cut.log_group_lanes);
        if (cut.per_lane > 16) continue;
        cut.wide = cut.per_lane % 4 == 0 && E % 4 == 0 && size % 4 == 0 && (((uintptr_t)logits | (uintptr_t)rule.bias) & 15u) == 0;
        auto of = [&](auto l) {
            constexpr int LPT = decltype(l)::value;
            auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(T, 256 / LPT)), dim3(256), 0, stream, logits, topk_v, topk_i, T, E, K, rule, cut);
                return launch_status();
            };
            auto of_k = [&](auto k) {
                constexpr int KMAX = decltype(k)::value;
                if (cut.per_lane <= 1) return launch(route_kernel<LPT, 1, KMAX>);
                if (cut.per_lane <= 2) return launch(route_kernel<LPT, 2, KMAX>);
                if (cut.per_lane <= 4) return launch(route_kernel<LPT, 4, KMAX>);
                if (cut.per_lane <= 8) return launch(route_kernel<LPT, 8, KMAX>);
                return launch(route_kernel<LPT, 16, KMAX>);
            };
            return K <= 4 ? of_k(std::integral_constant<int, 4>{}) : of_k(std::integral_constant<int, 8>{});
        };
        return lpt == 16 ? of(std::integral_constant<int, 16>{}) : lpt == 32 ? of(std::integral_constant<int, 32>{}) : of(std::integral_constant<int, 64>{});
    }
    // over 512 experts in groups that leave lanes idle, as 3 of 320: 16 experts a lane do not do
    hipLaunchKernelGGL(route_any_kernel<16>, dim3((unsigned)ceil_div(T, 4)), dim3(256), 0, stream, logits, topk_v, topk_i, T, E, K, rule);
    return launch_status();
}

int launch_route(const float* logits, float* topk_v, int* topk_i, int T, int E, int K, const RouteRule& rule, int n_cus,
                 hipStream_t stream) {
    constexpr long long kTokens = kMostThreads / 64;  // a multiple of four rows, which keeps the logits' alignment
    for (long long t = 0; t < T; t += kTokens) {
        const int rc = launch_route_part(logits + t * E, topk_v + t * K, topk_i + t * K, (int)std::min(T - t, kTokens), T, E, K, rule, n_cus, stream);
        if (rc) return rc;
    }
    return MOE_OK;
}

}  // namespace moe
