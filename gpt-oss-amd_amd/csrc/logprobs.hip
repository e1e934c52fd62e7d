// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace moe {

namespace {

constexpr int kWaves = 4, kStep = 512, kAhead = 2;  // waves of a block; values of a step, eight to a lane; steps that a wave loads at once
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kFewest = 2048;  // values of a row's part, if there are more

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

// A logit and its index as one number in the order of the values (a NaN above all), equal ones by falling index; 0 stands for nothing.
typedef uint64_t Key;
MOE_DEVICE Key key_of(float v, int index) {
    const int b = (int)__float_as_uint(v + 0.f);  // one zero
    const uint32_t order = v != v ? 0xFFFFFFFFu : (uint32_t)(b ^ ((b >> 31) | (int)0x80000000));
    return (Key)order << 32 | (uint32_t)~index;
}
MOE_DEVICE float value_of(Key k) {
    const uint32_t order = (uint32_t)(k >> 32);
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
MOE_DEVICE int index_of(Key k) { return (int)~(uint32_t)k; }
// The least value above one that value_of gives; a NaN above +infinity.
MOE_DEVICE float above(float v) {
    const int b = (int)__float_as_uint(v);
    return v != v ? v : __uint_as_float((uint32_t)(b < 0 ? b - 1 : b + 1));
}
MOE_DEVICE Key lane_key(Key k, int lane) {
    return (Key)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(k >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)k, lane);
}

// v of the lane whose number differs in bit J (a power of two) alone.
template <int J>
MOE_DEVICE uint32_t other_lane(uint32_t v) {
    if constexpr (J == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
    if constexpr (J == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
    if constexpr (J == 4) {  // from four lanes up in the even fours, from four down in the odd ones
        const int up = __builtin_amdgcn_update_dpp(0, (int)v, 0x104, 0xf, 0x5, false);
        return (uint32_t)__builtin_amdgcn_update_dpp(up, (int)v, 0x114, 0xf, 0xA, false);
    }
    if constexpr (J == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);
    if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
    if constexpr (J == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
template <int J>
MOE_DEVICE void exchange(Key& k, bool larger) {
    const Key other = (Key)other_lane<J>((uint32_t)(k >> 32)) << 32 | other_lane<J>((uint32_t)k);
    k = (other > k) == larger ? other : k;
}
// Of lanes in a bitonic order, to descending order in runs of 2 J where `down`, to ascending order in the others.
template <int J>
MOE_DEVICE void merge_runs(Key& k, bool down) {
    exchange<J>(k, ((threadIdx.x & J) == 0) == down);
    if constexpr (J > 1) merge_runs<J / 2>(k, down);
}
template <int RUN>
MOE_DEVICE void sort_runs(Key& k) {  // runs of RUN: descending and ascending in turn
    if constexpr (RUN > 2) sort_runs<RUN / 2>(k);
    merge_runs<RUN / 2>(k, RUN == 64 || (threadIdx.x & RUN) == 0);
}

// Sorting a key of every lane into the list takes as many instructions as about so many keys entered one by one.
constexpr int kFew = 16;

// The largest keys, one to a lane in descending order; 64 are kept, `top` of them count.
struct List {
    Key mine, last;  // last: the top-th, 0 as long as there are fewer
    int top;

    MOE_DEVICE void start(int k) {
        mine = last = 0;
        top = k;
    }
    MOE_DEVICE void set_last() { last = lane_key(mine, top - 1); }
    // With another list in descending order, of which lane l holds entry 63 - l.
    MOE_DEVICE void merge_reversed(Key other) {
        mine = other > mine ? other : mine;
        merge_runs<32>(mine, true);
        set_last();
    }
    MOE_DEVICE void insert(uint64_t left, Key k) {  // the keys of these lanes
        while (left) {
            const Key one = lane_key(k, __builtin_ctzll(left));
            left &= left - 1;
            const int at = __builtin_popcountll(__ballot(mine > one)), lane = threadIdx.x & 63;
            const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(mine >> 32), 0x138, 0xf, 0xf, false);  // the lane below's
            const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)mine, 0x138, 0xf, 0xf, false);
            mine = lane == at ? one : lane > at ? (Key)hi << 32 | lo : mine;
        }
    }
    // N keys of a lane: the lanes' largest ones, sorted; of what is left then few are above the top-th, or the next largest ones are sorted too.
    template <int N>
    MOE_DEVICE void fill(Key (&k)[N]) {
#pragma nounroll
        for (;;) {
            Key most = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) most = k[j] > most ? k[j] : most;
            merge(most);
            uint64_t left[N];
            int many = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                left[j] = __ballot(k[j] > last && k[j] != most);
                many += __builtin_popcountll(left[j]);
            }
            if (many <= kFew) {
#pragma unroll
                for (int j = 0; j < N; ++j) insert(left[j], k[j]);
                set_last();
                return;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) k[j] = k[j] == most ? 0 : k[j];
        }
    }
    MOE_DEVICE void merge(Key sorted) {  // with a key of every lane
        sort_runs<64>(sorted);
        const int from = (63 - (int)(threadIdx.x & 63)) * 4;
        const Key other = (Key)(uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(sorted >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)sorted);
        merge_reversed(other);
    }
};
MOE_DEVICE float wave_max(float v) {
#define MOE_STEP(C, M) v = fmaxf(v, __uint_as_float(dpp_move<C, M>(__float_as_uint(v), __float_as_uint(v))));
    MOE_DPP_STEPS(MOE_STEP)
#undef MOE_STEP
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// A wave's state over the values that it has seen.
struct Wave {
    Sums s;         // most and count: of the wave; rest and moment: of the lane
    List list;
    float entry;    // a value below it does not change the list,
    float enter;    // one below this neither the list nor the maximum

    MOE_DEVICE void start(int top) {
        s = {-INFINITY, 0.f, 0.f, 0.f};
        list.start(top);
        entry = top ? -INFINITY : INFINITY;
        enter = -INFINITY;
    }
    // N values of a lane, their indices by index(j); if not ALL, a negative one marks no value (-infinity is in its place).  No later call of the wave brings
    // an index below `next`.
    template <bool ALL, int N, class F>
    MOE_DEVICE void take(const float (&x)[N], F index, int next) {
        float most = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) most = fmaxf(most, x[j]);
        if (!__any(!(most < enter))) {
            add(x);
            return;
        }
        if (__any(!(most < s.most))) {
            const float now = fmaxf(s.most, wave_max(most));
            if (now > s.most) {
                // what was counted by the wave goes to lane 0
                Sums mine = s;
                if (threadIdx.x & 63) mine.count = 0.f;
                rebase(mine, now);
                s = {now, 0.f, mine.rest, mine.moment};
            }
            float below[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bool is = x[j] >= s.most;
                s.count += (float)__builtin_popcountll(__ballot(is && (ALL || index(j) >= 0)));
                below[j] = is ? -INFINITY : x[j];
            }
            if (s.most > -INFINITY) {
                add(below);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (x[j] != x[j]) s.rest = x[j];
            }
        } else {
            add(x);
        }
        const int lanes = list.top == 0 ? 0 : list.last == 0 ? 64 : __builtin_popcountll(__ballot(most >= entry));  // that have a value for the list
        if (lanes) {
            if (lanes > kFew) {
                Key k[N];
#pragma unroll
                for (int j = 0; j < N; ++j) k[j] = !ALL && index(j) < 0 ? 0 : key_of(x[j], index(j));
                list.fill(k);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    uint64_t left = __ballot(x[j] >= entry && (ALL || index(j) >= 0));
                    if (left) list.insert(left, key_of(x[j], index(j)));
                }
                list.set_last();
            }
            // Of equal values the first are kept: one of the last's own enters only in front of it.  Without that, rows of which most are -infinity, or equal, entered
            // every value one by one: 1000 bf16 rows of 200000 with 40 finite logits each 5284 us, with it 87
            if (list.last) entry = index_of(list.last) < next ? above(value_of(list.last)) : value_of(list.last);
        }
        enter = fminf(entry, s.most);
    }
    template <int N>
    MOE_DEVICE void add(const float (&x)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float d = x[j] - s.most, e = __builtin_amdgcn_exp2f(d * kLog2e);
            s.rest += e;
            s.moment = fmaf(e, fmaxf(d, -256.f), s.moment);  // of -infinity nothing
        }
    }
};

// The lanes' sums together, in all of them.
MOE_DEVICE Sums wave_joined(Sums s) {
    const float most = wave_max(s.most);
    rebase(s, most);
    return {most, wave_sum(s.count), wave_sum(s.rest), wave_sum(s.moment)};
}

// The waves' sums and lists as the first wave's; the others' are used up.
struct Shared {
    Sums sums[kWaves];
    Key keys[kWaves][64];
};
MOE_DEVICE void join_waves(Shared& lds, Sums& s, List& list) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (lane == 0) lds.sums[wave] = s;
    if (list.top) lds.keys[wave][lane] = list.mine;
    __syncthreads();
    if (wave == 0) {
        s = wave_joined(lane < kWaves ? lds.sums[lane] : Sums{-INFINITY, 0.f, 0.f, 0.f});
    }
    if (!list.top) return;
    for (int half = kWaves / 2; half > 0; half /= 2) {
        if (wave < half) {
            list.merge_reversed(lds.keys[wave + half][63 - lane]);
            lds.keys[wave][lane] = list.mine;
        }
        __syncthreads();
    }
}

template <bool NT>
MOE_DEVICE u32x4 load_16(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load(static_cast<const u32x4*>(p));
    else return *static_cast<const u32x4*>(p);
}
MOE_DEVICE float load_logit(const float* p) { return *p; }
MOE_DEVICE float load_logit(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// The logit of a row's token, a NaN where there is no such logit.
template <class T>
MOE_DEVICE float token_logit(const LogprobArgs& a, int row) {
    if (!a.logprobs) return 0.f;
    const int token = a.tokens[row];
    return (unsigned)token < (unsigned)a.vocab ? load_logit(static_cast<const T*>(a.logits) + (size_t)row * a.stride + token) : NAN;
}

// A row's results.  A NaN or +infinity makes all of them NaN, nothing but -infinity too.
MOE_DEVICE void write_row(const LogprobArgs& a, int row, float token, const Sums& s, Key best) {
    const int lane = threadIdx.x & 63;
    const float rest = s.count - 1.f + s.rest;  // Z = 1 + rest
    const float log_z = fabsf(s.most) < INFINITY ? log1pf(rest) : NAN;
    auto of = [&](float x) { return (float)((double)x - (double)s.most - (double)log_z); };
    if (a.logprobs && lane == 0) a.logprobs[row] = of(token);
    if (a.entropy && lane == 0) a.entropy[row] = log_z - s.moment / (1.f + rest);
    if (a.top_logprobs && lane < a.top_k) {
        a.top_logprobs[(size_t)row * a.top_k + lane] = of(value_of(best));
        a.top_indices[(size_t)row * a.top_k + lane] = index_of(best);
    }
}

}  // namespace

// A block to a row or one of `parts` of it (several where there are few rows); a wave takes every kWaves-th step of 512 values.  One pass: the running
// maximum is the wave's, so that most steps change neither it nor the list of the largest values, which is what one comparison of each lane's
// largest value asks, and cost a difference, an exponential and two sums a value.  Values before the first 16-byte border and behind the
// last whole step are read one by one, by the last wave while its first steps come.  Past the last-level cache rows are read past it.
// Bound by HBM and by its arithmetic: 1000 bf16 rows of 200000 with 5 alternatives 79 to 90 us, 4.4 to 5.1 TB/s (when it took 83: without the entropy 75, without any
// sums 70); fp32 rows of 131072 with 20 87 us, 6 TB/s.  One row of 131072 with 20 alternatives 11.0 us, 6.1 and 4.9 of them the two launches.
template <class T, bool NT>
__global__ __launch_bounds__(64 * kWaves) void logprob_kernel(LogprobArgs a, int parts, int part_len) {
    constexpr int kVec = 16 / sizeof(T);  // values of a load
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.stride;
    const int begin = min(part * part_len, a.vocab), end = min(a.vocab, begin + part_len);
    const int to_border = (int)((16 - ((uintptr_t)(x + begin) & 15)) % 16 / sizeof(T));
    const int first = min(end, begin + to_border), steps = (end - first) / kStep, behind = first + steps * kStep;

    const float token = parts == 1 ? token_logit<T>(a, row) : 0.f;
    Wave w;
    w.start(a.top_k);
    auto load = [&](int step, u32x4 (&v)[8 / kVec]) {
#pragma unroll
        for (int i = 0; i < 8 / kVec; ++i) v[i] = load_16<NT>(x + first + step * kStep + (64 * i + lane) * kVec);
    };
    auto take = [&](int step, const u32x4 (&v)[8 / kVec]) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = sizeof(T) == 4 ? __uint_as_float(v[j / kVec][j % kVec]) : bf16_bits_to_f32(v[0][j / 2] >> (j % 2 * 16) & 0xFFFFu);
        w.take<true>(f, [&](int j) { return first + step * kStep + (64 * (j / kVec) + lane) * kVec + j % kVec; }, first + (step + 1) * kStep);
    };
    int step = wave;
    auto ahead = [&](u32x4 (&v)[kAhead][8 / kVec]) {  // past the last the last again
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(min(step + i * kWaves, steps - 1), v[i]);
    };
    u32x4 v[kAhead][8 / kVec];
    if (steps > 0) ahead(v);
    if (wave == kWaves - 1 && (begin < first || behind < end)) {
        auto at = [&](int j) {
            const int i = j < 8 ? behind + 64 * j + lane : begin + lane;
            return i < (j < 8 ? end : first) ? i : -1;
        };
        float f[9];
#pragma unroll
        for (int j = 0; j < 9; ++j) f[j] = at(j) < 0 ? -INFINITY : load_logit(x + at(j));
        w.take<false>(f, at, first);
    }
    while (step < steps) {
        u32x4 next[kAhead][8 / kVec];
        const int now = step;
        step += kAhead * kWaves;
        ahead(next);
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (now + i * kWaves < steps) take(now + i * kWaves, v[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int j = 0; j < 8 / kVec; ++j) v[i][j] = next[i][j];
    }
    if (lane) w.s.count = 0.f;  // it is the wave's
    w.s = wave_joined(w.s);

    __shared__ Shared lds;
    join_waves(lds, w.s, w.list);
    if (wave) return;
    if (parts == 1) {
        write_row(a, row, token, w.s, w.list.mine);
        return;
    }
    const size_t rows = gridDim.x;  // parts of all rows
    if (lane == 0) static_cast<f32x4*>(a.workspace)[blockIdx.x] = f32x4{w.s.most, w.s.count, w.s.rest, w.s.moment};
    if (lane < a.top_k) reinterpret_cast<Key*>(static_cast<f32x4*>(a.workspace) + rows)[(size_t)blockIdx.x * a.top_k + lane] = w.list.mine;
}

// The parts of a row, joined by a block.
template <class T>
__global__ __launch_bounds__(64 * kWaves) void logprob_join_kernel(LogprobArgs a, int parts) {
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const f32x4* sums = static_cast<const f32x4*>(a.workspace) + (size_t)row * parts;
    const Key* keys = reinterpret_cast<const Key*>(static_cast<const f32x4*>(a.workspace) + (size_t)a.n_tokens * parts) + (size_t)row * parts * a.top_k;
    constexpr int kKeys = 8;
    const float token = token_logit<T>(a, row);
    Sums s = {-INFINITY, 0.f, 0.f, 0.f};
    List list;
    list.start(a.top_k);
    for (int i = threadIdx.x; i < parts; i += 64 * kWaves) {
        const f32x4 p = sums[i];
        s = joined(s, {p[0], p[1], p[2], p[3]});
    }
    for (int i = threadIdx.x; i - lane < parts * a.top_k; i += 64 * kWaves * kKeys) {  // all of a wave
        Key k[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) k[j] = i + 64 * kWaves * j < parts * a.top_k ? keys[i + 64 * kWaves * j] : 0;
        list.fill(k);
    }
    __shared__ Shared lds;
    s = wave_joined(s);
    join_waves(lds, s, list);
    if (threadIdx.x < 64) write_row(a, row, token, s, list.mine);
}

// Parts of a row: about kBlocks blocks where there are fewer rows.  A wave's first list costs it as much as ten steps.  us with 512 : 1024 : 2048 blocks:
// 1000 rows of 131072 90 : 99 : 111, 100 rows 33 : 34 : 37.
constexpr int kBlocks = 512;
static int parts_of(int n_tokens, int vocab) {
    return n_tokens >= kBlocks ? 1 : std::min(ceil_div(kBlocks, n_tokens), ceil_div(vocab, kFewest));
}

size_t logprob_workspace(int n_tokens, int vocab, int top_k) {
    if (vocab <= kFewest) return 0;
    // the most of any number of rows up to this: n times its parts is below kBlocks + n
    const long long rows = std::min(n_tokens, kBlocks), parts = std::min<long long>(kBlocks + rows, rows * ceil_div(vocab, kFewest));
    return (size_t)parts * (16 + 8 * top_k);
}

int launch_token_logprobs(const LogprobArgs& a, bool bf16_logits, hipStream_t stream) {
    const int parts = parts_of(a.n_tokens, a.vocab), part_len = ceil_div(ceil_div(a.vocab, parts), kStep) * kStep;
    auto run = [&](auto kernel, auto join) {
        const long long most = kMostThreads / (64 * kWaves);  // rows of a launch; more than 1024 of them are not cut
        for (long long row = 0; row < a.n_tokens; row += most) {
            LogprobArgs b = a;
            b.n_tokens = (int)std::min(a.n_tokens - row, most);
            b.logits = static_cast<const char*>(a.logits) + row * a.stride * (bf16_logits ? 2 : 4);
            if (a.logprobs) b.tokens += row, b.logprobs += row;
            if (a.entropy) b.entropy += row;
            if (a.top_k) b.top_logprobs += row * a.top_k, b.top_indices += row * a.top_k;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(b.n_tokens * parts)), dim3(64 * kWaves), 0, stream, b, parts, part_len);
            const int rc = launch_status();
            if (rc) return rc;
        }
        if (parts == 1) return (int)MOE_OK;
        hipLaunchKernelGGL(join, dim3((unsigned)a.n_tokens), dim3(64 * kWaves), 0, stream, a, parts);
        return launch_status();
    };
    const bool past_cache = (long long)a.n_tokens * a.vocab * (bf16_logits ? 2 : 4) > (256ll << 20);
    if (bf16_logits)
        return past_cache ? run(logprob_kernel<uint16_t, true>, logprob_join_kernel<uint16_t>) : run(logprob_kernel<uint16_t, false>, logprob_join_kernel<uint16_t>);
    return past_cache ? run(logprob_kernel<float, true>, logprob_join_kernel<float>) : run(logprob_kernel<float, false>, logprob_join_kernel<float>);
}

}  // namespace moe
