// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace moe {

namespace {

constexpr int kWaves = 8, kStep = 512, kAhead = 4;  // waves of a block; values of a step, eight to a lane; steps that a wave loads at once
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kFewest = 4096;  // values of a row's part, if there are more

// What a row or a part of it holds: the largest logit, how many have it, and of the others the sums of e = exp(l - most) and of e (l - most).
// Those that have it are counted by themselves: next to their 1 the others' sum would be lost where nearly all the weight is theirs.
struct Sums {
    float most, count, rest, moment;
};
MOE_DEVICE void rebase(Sums& s, float most) {
    if (s.most == most) return;
    if (s.most > -INFINITY) {  // else nothing counts so far; a NaN stays
        const float down = s.most - most, f = __builtin_amdgcn_exp2f(down * kLog2e), rest = s.count + s.rest;
        s.moment = f * (s.moment + fmaxf(down, -256.f) * rest);
        s.rest = f * rest;
    }
    s.count = 0.f;
    s.most = most;
}
MOE_DEVICE Sums joined(Sums a, Sums b) {
    const float most = fmaxf(a.most, b.most);
    rebase(a, most);
    rebase(b, most);
    return {most, a.count + b.count, a.rest + b.rest, a.moment + b.moment};
}

// The largest values, one to a lane in order, equal ones by index; lanes from `top` on hold more of them or nothing (index kNone).
constexpr int kNone = 0x7FFFFFFF;
struct Best {
    float value;
    int index;
};
// A number that is in the order of the values; a NaN above all.
MOE_DEVICE int order_of(float v) {
    if (v != v) return 0x7FFFFFFF;
    const int b = (int)__float_as_uint(v + 0.f);  // one zero
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
// All lanes have the same v and index.
MOE_DEVICE void insert(Best& b, float v, int index) {
    const int mine = b.index == kNone ? (int)0x80000000 : order_of(b.value), other = order_of(v);
    const bool before = b.index != kNone && (mine > other || (mine == other && b.index < index));
    const int at = __builtin_popcountll(__ballot(before)), lane = threadIdx.x & 63;
    const float up_v = __shfl_up(b.value, 1);
    const int up_i = __shfl_up(b.index, 1);
    if (lane == at) b = {v, index};
    else if (lane > at) b = {up_v, up_i};
}
MOE_DEVICE float lane_value(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }
MOE_DEVICE float wave_max(float v) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v = fmaxf(v, __shfl_xor(v, i));
    return v;
}

// A wave's state over the values that it has seen, in ascending order of index.
struct Wave {
    Sums s;         // most and count: of the wave; rest and moment: of the lane
    Best best;
    float enter;    // a value below it changes neither the list nor the maximum
    int top;
    bool full;

    MOE_DEVICE void start(int k) {
        s = {-INFINITY, 0.f, 0.f, 0.f};
        best = {-INFINITY, kNone};
        enter = -INFINITY;
        top = k;
        full = k == 0;
    }
    MOE_DEVICE void set_enter() {
        if (!full) full = __builtin_amdgcn_readlane(best.index, top - 1) != kNone;
        enter = !full ? -INFINITY : top ? fminf(lane_value(best.value, top - 1), s.most) : s.most;
    }
    // N values of a lane (logits), their indices by index(j); a negative one marks no value (-infinity is in its place).
    template <int N, class F>
    MOE_DEVICE void take(const float (&x)[N], F index) {
        float most = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) most = fmaxf(most, x[j]);
        if (__any(!(most < enter))) take_some(x, index, most);
        else add<false>(x, index);
    }
    template <bool EQUAL, int N, class F>
    MOE_DEVICE void add(const float (&x)[N], F index) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float d = x[j] - s.most, e = __builtin_amdgcn_exp2f(d * kLog2e);
            if constexpr (EQUAL) {
                const bool is = x[j] >= s.most;
                s.count += (float)__builtin_popcountll(__ballot(is && index(j) >= 0));
                if (is) continue;
            }
            s.rest += e;
            s.moment = fmaf(e, fmaxf(d, -256.f), s.moment);  // of -infinity nothing
        }
    }
    template <int N, class F>
    MOE_DEVICE void take_some(const float (&x)[N], F index, float most) {
        const float now = fmaxf(s.most, wave_max(most));
        if (now > s.most) {
            // what was counted by the wave goes to lane 0
            Sums mine = s;
            if (threadIdx.x & 63) mine.count = 0.f;
            rebase(mine, now);
            s = {now, 0.f, mine.rest, mine.moment};
        }
        add<true>(x, index);
        if (top) {
            if (!full) first(x, index);
            else {
#pragma unroll
                for (int j = 0; j < N; ++j) insert_where(x[j] >= enter && index(j) >= 0, x[j], index(j));
            }
        }
        set_enter();
    }
    // The first values: the top-th largest of the lanes' largest ones bounds the list from below.
    template <int N, class F>
    MOE_DEVICE void first(const float (&x)[N], F index) {
        int largest = (int)0x80000000;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (index(j) >= 0) largest = max(largest, order_of(x[j]));
        int above = 0;
        for (int i = 0; i < 64; ++i) above += __builtin_amdgcn_readlane(largest, i) > largest;
        int bound = above < top ? largest : 0x7FFFFFFF;
#pragma unroll
        for (int i = 1; i < 64; i *= 2) bound = min(bound, __shfl_xor(bound, i));
#pragma unroll
        for (int j = 0; j < N; ++j) insert_where(index(j) >= 0 && order_of(x[j]) >= bound, x[j], index(j));
    }
    MOE_DEVICE void insert_where(bool want, float x, int index) {
        uint64_t left = __ballot(want);
        while (left) {
            const int lane = __builtin_ctzll(left);
            left &= left - 1;
            insert(best, lane_value(x, lane), __builtin_amdgcn_readlane(index, lane));
        }
    }
    // The lanes' sums as the wave's, in all of them.
    MOE_DEVICE void finish() {
#pragma unroll
        for (int i = 1; i < 64; i *= 2) {
            s.rest += __shfl_xor(s.rest, i);
            s.moment += __shfl_xor(s.moment, i);
        }
    }
};

// Of a list of n: entry i in its wave's lanes.
struct Lists {
    Sums sums[kWaves];
    float value[kWaves][64];
    int index[kWaves][64];
};

MOE_DEVICE float load_logit(const float* p) { return *p; }
MOE_DEVICE float load_logit(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// A row's results.  A NaN or +infinity makes all of them NaN, nothing but -infinity too.
template <class T>
MOE_DEVICE void write_row(const LogprobArgs& a, const T* logits, int row, const Sums& s, const Best& best) {
    const int lane = threadIdx.x & 63;
    const float rest = s.count - 1.f + s.rest;  // Z = 1 + rest
    const float log_z = fabsf(s.most) < INFINITY ? log1pf(rest) : NAN;
    auto of = [&](float x) { return (float)((double)x - (double)s.most - (double)log_z); };
    if (a.logprobs && lane == 0) {
        const int token = a.tokens[row];
        a.logprobs[row] = (unsigned)token < (unsigned)a.vocab ? of(load_logit(logits + (size_t)row * a.stride + token)) : NAN;
    }
    if (a.entropy && lane == 0) a.entropy[row] = log_z - s.moment / (1.f + rest);
    if (a.top_logprobs && lane < a.top_k) {
        a.top_logprobs[(size_t)row * a.top_k + lane] = of(best.value);
        a.top_indices[(size_t)row * a.top_k + lane] = best.index;
    }
}

}  // namespace

// A block to a row or one of `parts` of it (several where there are few rows); a wave takes every kWaves-th step of 512 values.  One pass: the running
// maximum is the wave's, so that most steps change neither it nor the list of the largest values, which is what one comparison of each lane's
// largest value asks, and cost a product, an exponential and two additions a value.  Values before the first 16-byte border and behind the
// last whole step are read one by one.  Bound by HBM.
template <class T>
__global__ __launch_bounds__(64 * kWaves) void logprob_kernel(LogprobArgs a, int parts, int part_len) {
    constexpr int kVec = 16 / sizeof(T);  // values of a load
    const T* logits = static_cast<const T*>(a.logits);
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T* x = logits + (size_t)row * a.stride;
    const int begin = min(part * part_len, a.vocab), end = min(a.vocab, begin + part_len);
    const int to_border = (int)((16 - ((uintptr_t)(x + begin) & 15)) % 16 / sizeof(T));
    const int first = min(end, begin + to_border), steps = (end - first) / kStep, behind = first + steps * kStep;

    Wave w;
    w.start(a.top_k);
    auto one_by_one = [&](int from, int to) {
        for (int i = from; i < to; i += 64) {
            const int at = i + lane;
            const float v[1] = {at < to ? load_logit(x + at) : -INFINITY};
            w.take(v, [&](int) { return at < to ? at : -1; });
        }
    };
    if (wave == 0) one_by_one(begin, first);
    auto load = [&](int step, u32x4 (&v)[8 / kVec]) {
#pragma unroll
        for (int i = 0; i < 8 / kVec; ++i) v[i] = *reinterpret_cast<const u32x4*>(x + first + step * kStep + (64 * i + lane) * kVec);
    };
    auto take = [&](int step, const u32x4 (&v)[8 / kVec]) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = sizeof(T) == 4 ? __uint_as_float(v[j / kVec][j % kVec]) : bf16_bits_to_f32(v[0][j / 2] >> (j % 2 * 16) & 0xFFFFu);
        w.take(f, [&](int j) { return first + step * kStep + (64 * (j / kVec) + lane) * kVec + j % kVec; });
    };
    int step = wave;
    for (; step + (kAhead - 1) * kWaves < steps; step += kAhead * kWaves) {
        u32x4 v[kAhead][8 / kVec];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(step + i * kWaves, v[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) take(step + i * kWaves, v[i]);
    }
    for (; step < steps; step += kWaves) {
        u32x4 v[8 / kVec];
        load(step, v);
        take(step, v);
    }
    if (wave == kWaves - 1) one_by_one(behind, end);
    w.finish();

    __shared__ Lists lists;
    if (lane == 0) lists.sums[wave] = w.s;
    lists.value[wave][lane] = w.best.value;
    lists.index[wave][lane] = w.best.index;
    __syncthreads();
    if (wave) return;
    Sums s = lists.sums[0];
    for (int i = 1; i < kWaves; ++i) s = joined(s, lists.sums[i]);
    // the waves' lists into the first one's: an entry that does not get in ends its list
    if (a.top_k)
        for (int i = 1; i < kWaves; ++i)
            for (int j = 0; j < a.top_k; ++j) {
                const int index = lists.index[i][j];
                if (index == kNone) break;
                const float v = lists.value[i][j];
                const int last = __builtin_amdgcn_readlane(w.best.index, a.top_k - 1), lo = order_of(lane_value(w.best.value, a.top_k - 1)), mine = order_of(v);
                if (last != kNone && (mine < lo || (mine == lo && index > last))) break;
                insert(w.best, v, index);
            }
    if (parts == 1) {
        write_row(a, logits, row, s, w.best);
        return;
    }
    float* out = static_cast<float*>(a.workspace) + (size_t)blockIdx.x * (4 + 2 * a.top_k);
    if (lane == 0) *reinterpret_cast<f32x2*>(out) = f32x2{s.most, s.count};
    if (lane == 0) *reinterpret_cast<f32x2*>(out + 2) = f32x2{s.rest, s.moment};
    if (lane < a.top_k) *reinterpret_cast<f32x2*>(out + 4 + 2 * lane) = f32x2{w.best.value, __uint_as_float(w.best.index)};
}

// The parts of a row, joined by a wave.
template <class T>
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobArgs a, int parts) {
    const int row = blockIdx.x, lane = threadIdx.x, size = 4 + 2 * a.top_k;
    const float* in = static_cast<const float*>(a.workspace) + (size_t)row * parts * size;
    Sums s = {-INFINITY, 0.f, 0.f, 0.f};
    for (int i = lane; i < parts; i += 64) {
        const float* p = in + (size_t)i * size;
        s = joined(s, {p[0], p[1], p[2], p[3]});
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) s = joined(s, {__shfl_xor(s.most, i), __shfl_xor(s.count, i), __shfl_xor(s.rest, i), __shfl_xor(s.moment, i)});
    Wave w;
    w.start(a.top_k);
    const int n = parts * a.top_k;
    for (int i = 0; i < n; i += 64) {
        const int at = i + lane;
        float v = -INFINITY;
        int index = -1;
        if (at < n) {
            const float* p = in + (size_t)(at / a.top_k) * size + 4 + 2 * (at % a.top_k);
            v = p[0];
            index = (int)__float_as_uint(p[1]);
            if (index == kNone) index = -1;
        }
        if (!w.full) {
            const float x[1] = {v};
            w.first(x, [&](int) { return index; });
            w.full = __builtin_amdgcn_readlane(w.best.index, a.top_k - 1) != kNone;
        } else {
            const int last = order_of(lane_value(w.best.value, a.top_k - 1));
            w.insert_where(index >= 0 && order_of(v) >= last, v, index);
        }
    }
    write_row(a, static_cast<const T*>(a.logits), row, s, w.best);
}

// Parts of a row: about 2048 blocks where there are fewer rows than 1024.
static int parts_of(int n_tokens, int vocab) {
    if (n_tokens >= 1024) return 1;
    return std::min(ceil_div(2048, n_tokens), ceil_div(vocab, kFewest));
}

size_t logprob_workspace(int n_tokens, int vocab, int top_k) {
    if (vocab <= kFewest) return 0;
    // the most of any number of rows up to this: n times its parts is below 2048 + n
    const long long rows = std::min(n_tokens, 1024), parts = std::min<long long>(2048 + rows, rows * ceil_div(vocab, kFewest));
    return (size_t)parts * (4 + 2 * top_k) * 4;
}

int launch_token_logprobs(const LogprobArgs& a, bool bf16_logits, hipStream_t stream) {
    const int parts = parts_of(a.n_tokens, a.vocab), part_len = ceil_div(ceil_div(a.vocab, parts), 8) * 8;
    auto run = [&](auto kernel, auto join) {
        const int most = (int)(kMostThreads / (64 * kWaves));  // rows of a launch; more than 1024 of them are not cut
        for (int row = 0; row < a.n_tokens; row += most) {
            LogprobArgs b = a;
            b.n_tokens = std::min(a.n_tokens - row, most);
            b.logits = static_cast<const char*>(a.logits) + (size_t)row * a.stride * (bf16_logits ? 2 : 4);
            if (a.logprobs) b.tokens += row, b.logprobs += row;
            if (a.entropy) b.entropy += row;
            if (a.top_k) b.top_logprobs += (size_t)row * a.top_k, b.top_indices += (size_t)row * a.top_k;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(b.n_tokens * parts)), dim3(64 * kWaves), 0, stream, b, parts, part_len);
            const int rc = launch_status();
            if (rc) return rc;
        }
        if (parts == 1) return (int)MOE_OK;
        hipLaunchKernelGGL(join, dim3((unsigned)a.n_tokens), dim3(64), 0, stream, a, parts);
        return launch_status();
    };
    return bf16_logits ? run(logprob_kernel<uint16_t>, logprob_join_kernel<uint16_t>) : run(logprob_kernel<float>, logprob_join_kernel<float>);
}

}  // namespace moe
