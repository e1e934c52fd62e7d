// Attention of one query row a sequence over a paged key-value cache: out = softmax(scale q K^T, sinks) V.
#include <algorithm>

#include "attention.h"
#include "kernels.h"
#include "mx8.h"

namespace moe {

namespace {

constexpr int kWaves = 4, kTile = 32;  // waves of a block; keys that a wave takes at a time

// What a sequence's query sees: keys first .. len - 1, counted from the tile that holds the first of them.
struct Seen {
    int first, len, start;
    MOE_DEVICE int keys() const { return len - start; }
};
MOE_DEVICE Seen seen_of(const AttentionDecodeArgs& a, int b) {
    const long long room = (long long)a.max_pages << a.page_shift;
    const int len = (int)min((long long)max(a.lengths[b], 0), room);
    const int first = a.window ? max(0, len - a.window) : 0;
    return {first, len, first & ~(kTile - 1)};
}

// A wave's tile in the registers, as it comes: whole rows, 16 bytes to a lane.
template <int D, bool MX>
struct TileLoads {
    static constexpr int kRowBytes = MX ? D : 2 * D, kLanes = kRowBytes / 16, kRows = 64 / kLanes, kLoads = kTile / kRows;
    u32x4 k[kLoads], v[kLoads];
    uint32_t ks[MX ? kLoads : 1], vs[MX ? kLoads : 1];
    bool valid[2];  // whether the pages of keys 0 .. 15 and 16 .. 31 exist
};

// Scale byte of 32 values: 2^(b - 127), 255 a NaN.
MOE_DEVICE float mx_scale(uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : b << 23); }

}  // namespace

// Item (sequence, piece of its keys, KV head, 16 of the query heads that share it) to a block; pieces are as long as makes about a.pieces of
// them per head over all sequences, so that the longest sequence does not hold up the others; the whole pieces come first, the shorter ones end the launch.
// A wave takes every fourth tile of 32 keys: whole rows of K and V into registers two tiles ahead, past the caches (128 sequences of 4096 keys in 8 bits
// 201 : 178 us), through its own LDS into the matrix operands: loads in the operands' order would touch a line in two or four instructions.  S^T = K Q^T puts
// a query head into a lane column, so that its running maximum and sum are a lane's and P^T is the second product's operand as it stands: O^T = V^T P^T,
// with V^T read as columns from LDS.  P goes into that product as two bf16 parts, to 2^-16 of a weight: the matrix units have time.  Statistics are
// in powers of two: s' = scale log2(e) q.k.
// Bound by HBM: 128 sequences of 4096 keys, 8 heads of 128 in 8 bits 179 us, 6.2 TB/s; one of 131072, 8 heads of 64, 45 us, 6.0 TB/s, and 4.7 for the join.
template <int D, bool MX>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_decode_kernel(AttentionDecodeArgs a) {
    constexpr int kRow = 2 * D, kSteps = D / 32, kDims = D / 16;
    using Loads = TileLoads<D, MX>;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane & 15, g = lane >> 4;
    const int G = a.n_heads / a.n_kv_heads, group_tiles = ceil_div(G, 16);
    const int block = a.first_block + blockIdx.x, h = block % a.n_kv_heads, rest = block / a.n_kv_heads, gt = rest % group_tiles, item = rest / group_tiles;

    // the piece; up to 512 sequences are looked at once, eight to a lane
    constexpr int kHeld = 8;
    const bool held = a.batch <= 64 * kHeld;
    auto keys_of = [&](int s) { return seen_of(a, s).keys(); };
    int mine[kHeld];
    double total = 0.0;  // keys of all sequences, exact
    if (held) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            mine[i] = 0;
            if (64 * i >= a.batch) continue;
            if (64 * i + lane < a.batch) mine[i] = keys_of(64 * i + lane);
            sum += (double)mine[i];
        }
        total = wave_sum(sum);
    } else {
        for (int base = 0; base < a.batch; base += 64) total += wave_sum(base + lane < a.batch ? (double)keys_of(base + lane) : 0.0);
    }
    const long long even = (long long)(total / a.pieces) + 1;
    constexpr int kStep = kWaves * kTile;
    const int piece = (int)min(max((even + kStep - 1) / kStep * kStep, (long long)a.min_piece), (1ll << 30) + kStep);
    // items: the whole pieces of all sequences, then what is left of each
    int b = 0, part, n_whole = 0, first_part = 0, all_whole = 0;
    if (held) {
        int n[kHeld], upto[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (64 * i >= a.batch) continue;
            n[i] = mine[i] / piece;
            upto[i] = all_whole + wave_prefix_sum(n[i]);
            all_whole = __builtin_amdgcn_readlane(upto[i], 63);
        }
        if (item - all_whole >= a.batch) return;
        bool found = false;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (64 * i >= a.batch || found) continue;
            const uint64_t past = item < all_whole ? __ballot(upto[i] > item) : 64 * i + 63 >= item - all_whole ? 1ull << ((item - all_whole) & 63) : 0;
            if (past) {
                const int at = __builtin_ctzll(past);
                found = true;
                b = 64 * i + at;
                n_whole = __builtin_amdgcn_readlane(n[i], at);
                first_part = __builtin_amdgcn_readlane(upto[i], at) - n_whole;
            }
        }
    } else {
        auto whole_of = [&](int s) { return keys_of(s) / piece; };
        for (int base = 0; base < a.batch; base += 64) all_whole += wave_sum(base + lane < a.batch ? whole_of(base + lane) : 0);
        if (item - all_whole >= a.batch) return;
        if (item < all_whole) {
            find_item(a.batch, item, whole_of, b, part);
            first_part = item - part;
        } else {
            b = item - all_whole;
            for (int base = 0; base < b; base += 64) first_part += wave_sum(base + lane < b ? whole_of(base + lane) : 0);
        }
        n_whole = __builtin_amdgcn_readfirstlane(whole_of(b));
    }
    part = item < all_whole ? item - first_part : n_whole;
    const Seen seen = seen_of(a, b);
    const bool left = n_whole == 0 || n_whole * piece < seen.keys();
    const int n_parts = n_whole + (left ? 1 : 0);
    const int begin = seen.start + part * piece, end = min(seen.len, begin + piece);
    if (item >= all_whole) {
        if (h == 0 && gt == 0 && threadIdx.x == 0) {
            a.plan[3 * b] = first_part;
            a.plan[3 * b + 1] = n_whole;
            a.plan[3 * b + 2] = left ? item : -1;
        }
        if (!left) return;
    }

    __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * 2 * kTile * kRow];
    uint8_t* k_lds = lds + wave * 2 * kTile * kRow;
    uint8_t* v_lds = k_lds + kTile * kRow;

    u32x4 qf[kSteps];
    {
        const int head = 16 * gt + q;
        const uint16_t* row = a.q + ((size_t)b * a.n_heads + (size_t)h * G + min(head, G - 1)) * D;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            qf[s] = *reinterpret_cast<const u32x4*>(row + 32 * s + 8 * g);
            if (head >= G) qf[s] = u32x4{0, 0, 0, 0};
        }
    }

    // page numbers, 64 at a time, a lane to each
    const int* table = a.page_table + (size_t)b * a.max_pages;
    int pages_from = -64, pages = 0;
    auto page_at = [&](int key) {
        const int at = key >> a.page_shift;
        if (at - pages_from >= 64) {
            pages_from = at;
            pages = at + lane < a.max_pages ? table[at + lane] : -1;
        }
        return __builtin_amdgcn_readlane(pages, at - pages_from);
    };
    auto load = [&](Loads& t, int key0) {
        const uint8_t* kp[2];
        const uint8_t* vp[2];
        const uint8_t* ksp[2];
        const uint8_t* vsp[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = key0 + 16 * i;
            const int page = key < end ? page_at(key) : -1;
            t.valid[i] = (unsigned)page < (unsigned)a.n_pages;
            const size_t row = ((size_t)(t.valid[i] ? page : 0) * a.n_kv_heads + h) << a.page_shift | (size_t)(key & ((1 << a.page_shift) - 1));
            kp[i] = static_cast<const uint8_t*>(a.k) + row * Loads::kRowBytes;
            vp[i] = static_cast<const uint8_t*>(a.v) + row * Loads::kRowBytes;
            if constexpr (MX) {
                ksp[i] = a.k_scales + row * (D / 32);
                vsp[i] = a.v_scales + row * (D / 32);
            }
        }
        const int r = lane / Loads::kLanes, c = lane % Loads::kLanes;
#pragma unroll
        for (int i = 0; i < Loads::kLoads; ++i) {
            const int half = i * Loads::kRows / 16, at = i * Loads::kRows % 16 + r;
            t.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp[half] + at * Loads::kRowBytes + 16 * c));
            t.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp[half] + at * Loads::kRowBytes + 16 * c));
            if constexpr (MX) {
                t.ks[i] = ksp[half][at * (D / 32) + c / 2];
                t.vs[i] = vsp[half][at * (D / 32) + c / 2];
            }
        }
    };

    f32x4 acc[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float scale = a.scale * kLog2e;

    auto compute = [&](Loads& t, int key0) {
        const bool whole = key0 >= seen.first && key0 + kTile <= end && t.valid[0] && t.valid[1];
        auto visible = [&](int key) { return key >= seen.first && key < end && t.valid[(key - key0) >> 4]; };
        const int r0 = lane / Loads::kLanes, c = lane % Loads::kLanes;
#pragma unroll
        for (int i = 0; i < Loads::kLoads; ++i) {
            const int r = i * Loads::kRows + r0;
            if (!whole && !visible(key0 + r)) t.v[i] = u32x4{0, 0, 0, 0};  // a weight of 0 does not undo a NaN
            uint8_t* kr = k_lds + r * kRow;
            uint8_t* vr = v_lds + r * kRow;
            if constexpr (MX) {
                const float k_scale = mx_scale(t.ks[i]), v_scale = !whole && !visible(key0 + r) ? 1.f : mx_scale(t.vs[i]);
                *reinterpret_cast<u32x4*>(kr + k_chunk<D>(r, 2 * c) * 16) = e4m3x8_to_bf16(t.k[i][0], t.k[i][1], k_scale);
                *reinterpret_cast<u32x4*>(kr + k_chunk<D>(r, 2 * c + 1) * 16) = e4m3x8_to_bf16(t.k[i][2], t.k[i][3], k_scale);
                *reinterpret_cast<u32x4*>(vr + v_chunk<D>(r, 2 * c) * 16) = e4m3x8_to_bf16(t.v[i][0], t.v[i][1], v_scale);
                *reinterpret_cast<u32x4*>(vr + v_chunk<D>(r, 2 * c + 1) * 16) = e4m3x8_to_bf16(t.v[i][2], t.v[i][3], v_scale);
            } else {
                *reinterpret_cast<u32x4*>(kr + k_chunk<D>(r, c) * 16) = t.k[i];
                *reinterpret_cast<u32x4*>(vr + v_chunk<D>(r, c) * 16) = t.v[i];
            }
        }
        lds_in_order();
        f32x4 s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int r = 16 * i + q;
                s[i] = mfma_16x16x32(*reinterpret_cast<const u32x4*>(k_lds + r * kRow + k_chunk<D>(r, 4 * j + g) * 16), qf[j], s[i]);
            }
        }
        settle(s[0], s[1]);
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] *= scale;
                if (!whole && !visible(key0 + 16 * i + 4 * g + j)) s[i][j] = -INFINITY;
                most = fmaxf(most, s[i][j]);
            }
        most = fmaxf(m, max_of_groups(most));
        const float base = most == -INFINITY ? 0.f : most;
        const float down = __builtin_amdgcn_exp2f(m - base);  // nothing so far: 0
        m = most;
        l *= down;
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[d] *= down;
        u32x4 p, rest;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = __builtin_amdgcn_exp2f(s[i][j] - base);
                l += s[i][j];
            }
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const uint32_t w = pack_bf16x2(s[i][j], s[i][j + 1]);
                p[2 * i + j / 2] = w;
                rest[2 * i + j / 2] = pack_bf16x2(s[i][j] - __uint_as_float(w << 16), s[i][j + 1] - __uint_as_float(w & 0xFFFF0000u));
            }
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            u32x2 col[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 16 * i + 4 * g + (q >> 2);
                col[i] = lds_column_of_4(v_lds + r * kRow + v_chunk<D>(r, 2 * d + ((q & 3) >> 1)) * 16 + (q & 1) * 8);
            }
            const u32x4 values = {col[0][0], col[0][1], col[1][0], col[1][1]};
            acc[d] = mfma_16x16x32(values, p, acc[d]);
            acc[d] = mfma_16x16x32(values, rest, acc[d]);
        }
        lds_in_order();
    };

    int key0 = begin + wave * kTile;
    if (key0 < end) {
        Loads t0, t1;
        load(t0, key0);
        if (key0 + kStep < end) load(t1, key0 + kStep);
        for (;;) {
            compute(t0, key0);
            if (key0 + 2 * kStep < end) load(t0, key0 + 2 * kStep);
            key0 += kStep;
            if (key0 >= end) break;
            compute(t1, key0);
            if (key0 + 2 * kStep < end) load(t1, key0 + 2 * kStep);
            key0 += kStep;
            if (key0 >= end) break;
        }
    }

    // the waves' parts together
#pragma unroll
    for (int d = 0; d < kDims; ++d) settle(acc[d]);
    l = sum_of_groups(l);
    __syncthreads();
    float* o_lds = reinterpret_cast<float*>(lds);  // [waves][16][D]
    __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
#pragma unroll
    for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(o_lds + (wave * 16 + q) * D + 16 * d + 4 * g) = acc[d];
    if (g == 0) {
        m_lds[wave][q] = m;
        l_lds[wave][q] = l;
    }
    __syncthreads();
#pragma unroll
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 64 * kWaves) {
        const int row = i / (D / 4), d = i % (D / 4) * 4, head = 16 * gt + row;
        if (head >= G) continue;
        const int qh = h * G + head;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, m_lds[w][row]);
        const bool alone = n_parts == 1;
        const float sink = a.sinks && alone ? bf16_bits_to_f32(a.sinks[qh]) * kLog2e : -INFINITY;
        most = fmaxf(most, sink);
        const float base = most == -INFINITY ? 0.f : most;
        float sum = a.sinks && alone ? __builtin_amdgcn_exp2f(sink - base) : 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(m_lds[w][row] - base);
            sum += f * l_lds[w][row];
            o += f * *reinterpret_cast<const f32x4*>(o_lds + (w * 16 + row) * D + d);
        }
        if (alone) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<u32x2*>(a.out + ((size_t)b * a.n_heads + qh) * D + d) = u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
        } else {
            const size_t at = (size_t)item * a.n_heads + qh;
            *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
            if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * at) = f32x2{most, sum};
        }
    }
}

// The parts of sequences that were cut, joined: a block to a sequence and some heads; a row of D floats to D / 4 lanes, which take every kAtOnce-th part with
// a maximum of their own, so that no load waits for another's value but for the plan.
template <int D>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionDecodeArgs a, int heads_per_block) {
    constexpr int kLanes = D / 4, kAtOnce = 256 / kLanes;
    const int b = blockIdx.x, first = a.plan[3 * b], n_whole = a.plan[3 * b + 1], left = a.plan[3 * b + 2], n = n_whole + (left >= 0 ? 1 : 0);
    if (n == 1) return;
    __shared__ f32x2 stats[kAtOnce];
    __shared__ __attribute__((aligned(16))) float rows[kAtOnce][D];
    const int slot = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
    for (int head = blockIdx.y * heads_per_block; head < min(a.n_heads, (int)(blockIdx.y + 1) * heads_per_block); ++head) {
        float most = -INFINITY, sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = slot; i < n; i += kAtOnce) {
            const size_t at = (size_t)(i < n_whole ? first + i : left) * a.n_heads + head;
            const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * at);
            const f32x4 row = *reinterpret_cast<const f32x4*>(a.part_o + at * D + d);
            const float now = fmaxf(most, ml[0]), base = now == -INFINITY ? 0.f : now;
            const float f = __builtin_amdgcn_exp2f(most - base), g = __builtin_amdgcn_exp2f(ml[0] - base);
            most = now;
            sum = sum * f + ml[1] * g;
            o = o * f + row * g;
        }
        const float sink = a.sinks ? bf16_bits_to_f32(a.sinks[head]) * kLog2e : -INFINITY;
        __syncthreads();  // the last head's rows have been read
        if (d == 0) stats[slot] = f32x2{most, sum};
        *reinterpret_cast<f32x4*>(&rows[slot][d]) = o;
        __syncthreads();
        if (threadIdx.x < D / 2) {
            most = sink;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) most = fmaxf(most, stats[i][0]);
            const float base = most == -INFINITY ? 0.f : most;
            float total = a.sinks ? __builtin_amdgcn_exp2f(sink - base) : 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const float f = __builtin_amdgcn_exp2f(stats[i][0] - base);
                total += f * stats[i][1];
                x += f * rows[i][2 * threadIdx.x];
                y += f * rows[i][2 * threadIdx.x + 1];
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
            reinterpret_cast<uint32_t*>(a.out + ((size_t)b * a.n_heads + head) * D)[threadIdx.x] = pack_bf16x2(x * inv, y * inv);
        }
    }
}

// Pieces per head over all sequences: with n of them per KV head and 16 query heads there are at most n + batch.
static int most_items(int batch, int n_kv_heads, int group_tiles, int* pieces) {
    *pieces = std::max(1, kDecodePieces / (n_kv_heads * group_tiles));
    return *pieces + batch;
}
static int group_tiles_of(int n_heads, int n_kv_heads) { return ceil_div(n_heads / n_kv_heads, 16); }

size_t attention_decode_workspace(int batch, int n_heads, int n_kv_heads, int head_dim, size_t* ml, size_t* o) {
    int pieces;
    const size_t items = most_items(batch, n_kv_heads, group_tiles_of(n_heads, n_kv_heads), &pieces);
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    *ml = up((size_t)batch * 12);
    *o = *ml + up(items * n_heads * 8);
    return *o + up(items * n_heads * head_dim * 4);
}

int launch_attention_decode(AttentionDecodeArgs a, int head_dim, hipStream_t stream) {
    const int group_tiles = group_tiles_of(a.n_heads, a.n_kv_heads);
    const int items = most_items(a.batch, a.n_kv_heads, group_tiles, &a.pieces);
    const int blocks = items * a.n_kv_heads * group_tiles, at_once = (int)(kMostThreads / (64 * kWaves));
    const long long room = (long long)a.max_pages << a.page_shift;
    const long long most = a.window ? std::min<long long>(room, (long long)a.window + kTile - 1) : room;
    a.min_piece = most <= 256 ? 256 : 128;  // a short window is one piece: no parts to join
    const bool join = most > a.min_piece;
    auto run = [&](auto kernel, auto joiner) {
        for (a.first_block = 0; a.first_block < blocks; a.first_block += at_once) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(at_once, blocks - a.first_block)), dim3(64 * kWaves), 0, stream, a);
            const int rc = launch_status();
            if (rc) return rc;
        }
        if (!join) return (int)MOE_OK;
        const int per_block = std::max(1, ceil_div(a.batch * std::min(a.n_heads, 256), 2048));
        hipLaunchKernelGGL(joiner, dim3((unsigned)a.batch, (unsigned)ceil_div(a.n_heads, per_block)), dim3(256), 0, stream, a, per_block);
        return launch_status();
    };
    const bool mx = a.k_scales != nullptr;
    if (head_dim == 64)
        return mx ? run(attention_decode_kernel<64, true>, attention_join_kernel<64>) : run(attention_decode_kernel<64, false>, attention_join_kernel<64>);
    return mx ? run(attention_decode_kernel<128, true>, attention_join_kernel<128>) : run(attention_decode_kernel<128, false>, attention_join_kernel<128>);
}

}  // namespace moe
