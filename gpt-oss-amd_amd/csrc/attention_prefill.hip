// Causal attention over packed prompts: out = softmax(scale q K^T, sinks) V, query heads in groups that share a key/value head.
#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "kernels.h"

namespace moe {

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves, kKeys = 64;  // query rows of a block, 32 to a wave; keys that it takes at a time

// Half a row's weights of a tile, relative to the maximum that it knows, may add up to this before it looks for a new maximum: no tile but the first few
// has to look for one, and with weights up to 2^10 sums stay as far from overflow as values of 2^118 allow.
constexpr float kMostWeight = 1024.f;

// A weight is exp2 of s scale - m in one rounding, the maximum m a product that was rounded by itself: what it lost, up to 2^-24 of m, is a factor of all weights
// of the row, which their sum takes out again.  Up to this size of m it is below 2^(1/16); from 2^31 on it would be infinity or nothing.  Rows whose
// maximum was ever past it go through the careful pass with scores rounded before the maximum is taken (where all rows of a prompt do, 2.3 times as long).
constexpr float kFar = 1048576.f;

struct Span {
    int begin, rows;
};
MOE_DEVICE Span span_of(const int* starts, int s, int total) {
    const int begin = min(max(starts[s], 0), total);
    return {begin, min(max(starts[s + 1], begin), total) - begin};
}

}  // namespace

// Block: 128 rows of one head of one sequence; wave: 32 of them, against tiles of 64 keys that the block loads into LDS a tile ahead.  S^T = K Q^T puts a
// query row into two lanes (l and l + 32), so that its maximum and sum are a lane's but for one exchange, and P^T the second product's operand as
// it stands: O^T = V^T P^T, V^T read from LDS as columns.  P is rounded to bf16 for that product (half a step is up to 2^-8 of a weight, as that of the bf16
// result; a second part would cost half as many matrix instructions again); its sum is taken before that, in fp32.  Statistics are in powers of two.
// Longest blocks first.
// A prompt of 8192, 64 heads of 64: 571 to 594 us from card to card, 925 to 963 TFLOP/s; heads of 128 975 to 1013; a large library product reaches 1394.  When it took 612 us, it took 439
// without the weights' arithmetic and 505 without matrix instructions; 64 rows to a wave, half the reads of LDS, 615 : 618, two blocks to a compute unit
// in place of three 613 : 612, four 784: what bounds it is both kinds of instruction together.
template <int D>
__global__ __launch_bounds__(64 * kWaves, D == 64 ? 3 : 2) void attention_prefill_kernel(AttentionPrefillArgs a) {
    constexpr int kRow = 2 * D, kSteps = D / 16, kDims = D / 32, kChunks = D / 8, kLoads = kKeys * kChunks / (64 * kWaves);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;

    // heads of a group on one XCD (blocks go to them in turn), where its L2 holds their keys
    const int block = a.first_block + blockIdx.x;
    int head, rank;
    if (a.n_heads % 8 == 0) {
        const int each = a.n_heads / 8, at = block / 8;
        head = block % 8 * each + at % each;
        rank = at / each;
    } else {
        head = block % a.n_heads;
        rank = block / a.n_heads;
    }
    auto tiles_of = [&](int s) { return ceil_div(span_of(a.q_starts, s, a.total_q).rows, kRows); };
    int seq, tile;
    if (!find_last_item(a.n_seqs, rank, tiles_of, seq, tile)) return;
    const Span qs = span_of(a.q_starts, seq, a.total_q), ks = span_of(a.k_starts, seq, a.total_k);
    const int ahead = ks.rows - qs.rows;  // query i sees keys up to i + ahead
    const int window = a.window < ks.rows ? a.window : 0;  // one past all keys is none: a row without keys less such a window would not fit 32 bits
    const int row0 = tile * kRows, kv_head = head / (a.n_heads / a.n_kv_heads);
    const int end = min(row0 + kRows, qs.rows) + ahead;  // past the last key that the block sees
    const int begin = window ? max(0, row0 + ahead - window + 1) & ~(kKeys - 1) : 0;

    __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][kKeys * kRow];
    __shared__ int odd[2];  // the first key of the last tile in that buffer whose values were not all finite

    const int wave_row = row0 + 32 * wave, row = min(wave_row + col, qs.rows - 1);
    const int last = row + ahead, first = window ? last - window + 1 : 0;  // what this lane's row sees
    u32x4 qf[kSteps];
    {
        const uint16_t* q = a.q + (size_t)(qs.begin + row) * a.q_stride + (size_t)head * D;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = *reinterpret_cast<const u32x4*>(q + 16 * s + 8 * hi);
    }
    f32x16 acc[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float m = -INFINITY, l = 0.f, reach = 0.f;  // reach: the largest |m| so far
    const float scale = a.scale * kLog2e;
    float before = 1.f, by = scale;  // of the careful pass: what scores are multiplied by first, and next to the maximum

    // a lane's share of a tile: kLoads pieces of 1 KiB to a wave, each linear in LDS; offsets in bytes from the tile's first row, of rows past the last key
    // the last one's
    uint32_t k_off[kLoads], v_off[kLoads];
    auto offsets = [&](int rows) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (wave * kLoads + i) * (64 / kChunks) + lane / kChunks, c = lane % kChunks;
            const uint32_t from = min(r, rows - 1);
            k_off[i] = 2 * (from * (uint32_t)a.k_stride + 8 * k_chunk<D>(r, c));
            v_off[i] = 2 * (from * (uint32_t)a.v_stride + 8 * v_chunk<D>(r, c));
        }
    };
    offsets(kKeys);
    const uint8_t* k_base = reinterpret_cast<const uint8_t*>(a.k + (size_t)ks.begin * a.k_stride + (size_t)kv_head * D);
    const uint8_t* v_base = reinterpret_cast<const uint8_t*>(a.v + (size_t)ks.begin * a.v_stride + (size_t)kv_head * D);
    const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&lds[0][0][0]) + wave * kLoads * 1024;
    auto load = [&](int buffer, int key0) {
        if (key0 + kKeys > ks.rows) offsets(ks.rows - key0);  // the last tile
        const uint8_t* k = k_base + (size_t)key0 * a.k_stride * 2;
        const uint8_t* v = v_base + (size_t)key0 * a.v_stride * 2;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            tile_dma16(k, k_off[i], lds_at + buffer * 2 * kKeys * kRow + i * 1024);
            tile_dma16(v, v_off[i], lds_at + (buffer * 2 + 1) * kKeys * kRow + i * 1024);
        }
    };
    // Whether some row of the block does not see all of these keys.  Infinities and NaNs among their values, which a weight of 0 does not undo, are taken
    // out of LDS in the careful pass; the rows that do see them get them afterwards.
    auto cut = [&](int key0) { return key0 + kKeys - 1 > row0 + ahead || (window && key0 < end - window); };
    auto clean = [&](int buffer, int key0) {
        auto not_finite = [](uint32_t x) { return ((x & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((x & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u); };
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            u32x4* at = reinterpret_cast<u32x4*>(&lds[buffer][1][0]) + threadIdx.x + 64 * kWaves * i;
            u32x4 x = *at;
            uint32_t off[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) off[w] = not_finite(x[w]);
            if (off[0] | off[1] | off[2] | off[3]) {
#pragma unroll
                for (int w = 0; w < 4; ++w) x[w] &= ~off[w];
                *at = x;
                odd[buffer] = key0;
            }
        }
        __syncthreads();
    };
    auto v_column = [&](const uint8_t* v, int key, int d) {  // keys key .. key + 3 (+ 4 in the upper half), the lane's dimension of 32 d ..
        const int i = lane & 15, r = key + 4 * hi + (i >> 2), c = 4 * d + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
        return lds_column_of_4(v + r * kRow + v_chunk<D>(r, c) * 16 + (i & 1) * 8);
    };
    auto compute = [&](int buffer, int key0, auto careful) {
        const uint8_t* k = lds[buffer][0];
        const uint8_t* v = lds[buffer][1];
        f32x16 s[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = 32 * t + col;
                s[t] = mfma_32x32x16(*reinterpret_cast<const u32x4*>(k + r * kRow + k_chunk<D>(r, 2 * j + hi) * 16), qf[j], s[t]);
            }
        settle(s[0], s[1]);
        if (key0 + kKeys - 1 > wave_row + ahead || (window && key0 < wave_row + 31 + ahead - window + 1)) {
            // a bit a key that the row sees, spread over its score; comparisons would each wait for the one before it to leave the condition register
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int from = first - key0 - 32 * t, to = last - key0 - 32 * t;  // of keys 0 .. 31
                const uint32_t upto = to < 0 ? 0u : to >= 31 ? ~0u : (2u << to) - 1u, since = from <= 0 ? ~0u : from > 31 ? 0u : ~0u << from;
                const uint32_t seen = (upto & since) >> 4 * hi;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)seen, 8 * (i / 4) + i % 4, 1);
                    s[t][i] = __uint_as_float((keep & __float_as_uint(s[t][i])) | (~keep & 0xFF800000u));
                }
            }
        }
        if constexpr (decltype(careful)::value) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[0][i] *= before;
                s[1][i] *= before;
            }
        }
        const float factor = decltype(careful)::value ? by : scale;
        u32x4 p[4];
        auto weigh = [&](float base) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[t][i], factor, -base)), y = __builtin_amdgcn_exp2f(fmaf(s[t][i + 1], factor, -base));
                    sum[0] += x;
                    sum[1] += y;
                    p[2 * t + i / 8][i % 8 / 2] = pack_bf16x2(x, y);
                }
            return sum[0] + sum[1];
        };
        float sum = weigh(m);
        if (__any(!(sum < kMostWeight))) {
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, s[t][i]);
            most = max_of_halves(sum < kMostWeight ? 0.f : 1.f) > 0.f ? fmaxf(m, max_of_halves(most) * factor) : m;  // of the rows that have to
            const float down = most == m ? 1.f : __builtin_amdgcn_exp2f(m - most);
            m = most;
            if (m > -INFINITY) reach = fmaxf(reach, fabsf(m));
            l *= down;
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[d] *= down;
            sum = weigh(m == -INFINITY ? 0.f : m);
        }
        l += sum;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                const u32x2 x = v_column(v, 16 * j, d), y = v_column(v, 16 * j + 8, d);
                acc[d] = mfma_32x32x16(u32x4{x[0], x[1], y[0], y[1]}, p[j], acc[d]);
            }
        if (decltype(careful)::value && cut(key0) && odd[buffer] == key0) {  // what was left out, a key at a time, added where it is seen
#pragma unroll
            for (int d = 0; d < kDims; ++d) settle(acc[d]);
            for (int i = 0; i < kKeys && key0 + i < ks.rows; ++i) {
                const int j = i >> 4, e = ((i >> 3) & 1) * 4 + (i & 3);  // element e of the half (i >> 2) & 1
                const bool mine = ((i >> 2) & 1) == hi, seen = key0 + i <= last && key0 + i >= first;
                const u32x4 weights = j == 0 ? p[0] : j == 1 ? p[1] : j == 2 ? p[2] : p[3];
#pragma unroll
                for (int d = 0; d < kDims; ++d) {
                    const uint32_t x = reinterpret_cast<const uint16_t*>(v_base)[(size_t)(key0 + i) * a.v_stride + 32 * d + col], left = mine && (x & 0x7F80u) == 0x7F80u ? x << (e & 1) * 16 : 0u;
                    u32x4 one;
#pragma unroll
                    for (int w = 0; w < 4; ++w) one[w] = e >> 1 == w ? left : 0u;
                    f32x16 o;
#pragma unroll
                    for (int n = 0; n < 16; ++n) o[n] = 0.f;
                    o = mfma_32x32x16(one, weights, o);
                    settle(o);
#pragma unroll
                    for (int n = 0; n < 16; ++n) acc[d][n] = seen ? acc[d][n] + o[n] : acc[d][n];
                }
            }
        }
    };

    auto pass = [&](auto careful) {
        load(0, begin);
        int buffer = 0;
        for (int key0 = begin; key0 < end; key0 += kKeys) {
            wait_and_meet<0>();  // the tile is there, and all waves have left the one before it
            if (key0 + kKeys < end) load(buffer ^ 1, key0 + kKeys);
            if (decltype(careful)::value && cut(key0)) clean(buffer, key0);
            // whether any row of the wave sees any of these keys
            if (key0 <= wave_row + 31 + ahead && (!window || key0 + kKeys > wave_row + ahead - window + 1) && wave_row < qs.rows)
                compute(buffer, key0, careful);
            buffer ^= 1;
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) settle(acc[d]);
    };
    if (begin < end) {
        pass(std::false_type{});
        // A value that is not finite under a weight of 0 has made a NaN of its row's sum.  So has one that the row sees: the careful pass tells them apart.
        float sum = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum = fmaf(acc[d][i], 0.f, sum);  // 0 if all are finite
        const bool far = reach > kFar;
        if (__syncthreads_or(!(sum == 0.f) || far)) {
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
            m = -INFINITY;
            l = 0.f;
            if (far) {
                before = scale;
                by = 1.f;
            }
            if (threadIdx.x < 2) odd[threadIdx.x] = -1;
            offsets(kKeys);
            pass(std::true_type{});
            __syncthreads();  // LDS is used anew
        }
    }
    if (a.sinks) {
        const float sink = bf16_bits_to_f32(a.sinks[head]) * kLog2e, most = fmaxf(m, sink), base = most == -INFINITY ? 0.f : most;
        const float down = __builtin_amdgcn_exp2f(m - base);
        l = sum_of_halves(l) * down + __builtin_amdgcn_exp2f(sink - base);
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[d] *= down;
    } else {
        l = sum_of_halves(l);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // whole rows to memory, by way of the wave's own part of LDS: in the order of the registers every store would touch 32 rows.  16 short-window prompts of
    // up to 3000: 70 us : 65
    uint8_t* rows = &lds[0][0][0] + wave * 32 * kRow;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<u32x2*>(rows + col * kRow + k_chunk<D>(col, 4 * d + i / 4) * 16 + 8 * hi) =
                u32x2{pack_bf16x2(acc[d][i] * inv, acc[d][i + 1] * inv), pack_bf16x2(acc[d][i + 2] * inv, acc[d][i + 3] * inv)};
    lds_in_order();
#pragma unroll
    for (int i = 0; i < 32 * kChunks / 64; ++i) {
        const int r = i * (64 / kChunks) + lane / kChunks, c = lane % kChunks;
        if (wave_row + r < qs.rows)
            *reinterpret_cast<u32x4*>(a.out + (size_t)(qs.begin + wave_row + r) * a.out_stride + (size_t)head * D + 8 * c) =
                *reinterpret_cast<const u32x4*>(rows + r * kRow + k_chunk<D>(r, c) * 16);
    }
}

int launch_attention_prefill(AttentionPrefillArgs a, int head_dim, hipStream_t stream) {
    // as many as there can be; below 2^30 rows of heads it is less than 2^27
    const int blocks = (a.total_q / kRows + std::min(a.n_seqs, a.total_q)) * a.n_heads, at_once = (int)(kMostThreads / (64 * kWaves));
    for (a.first_block = 0; a.first_block < blocks; a.first_block += at_once) {
        const dim3 grid((unsigned)std::min(at_once, blocks - a.first_block));
        if (head_dim == 64) hipLaunchKernelGGL(attention_prefill_kernel<64>, grid, dim3(64 * kWaves), 0, stream, a);
        else hipLaunchKernelGGL(attention_prefill_kernel<128>, grid, dim3(64 * kWaves), 0, stream, a);
        const int rc = launch_status();
        if (rc) return rc;
    }
    return MOE_OK;
}

}  // namespace moe
