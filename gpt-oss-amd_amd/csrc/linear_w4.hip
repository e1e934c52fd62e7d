// Products of a few rows with a matrix of 4-bit weights and group scales: y[b, n] = bias[n] + sum_k x[b, k] W[n, k].
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "mx8.h"

namespace moe {

namespace {

constexpr int kUnit = 256;  // contraction elements of a wave: two chunks of 128

// Waves of a block at most: what the registers of a wave allow (16: 128, 12: 168, 8: 256).
constexpr int max_waves(int group, int nt) {
    if (nt == 1) return 16;
    return group == 32 ? 8 : group == 64 ? 12 : 16;
}

// Floats of the LDS that a wave keeps its partial tiles in, those of two steps; a chunk of 16 rows of x goes through it while it is loaded.
__host__ __device__ constexpr int part_floats(int nt, int tiles_per_step) { return 2 * tiles_per_step * nt > 4 ? 2 * tiles_per_step * nt * 256 : 1024; }

// Unit u of rows b0 .. b0 + 16 NT - 1 of x, as xr[chunk][MFMA step][token tile]: token q, 8 elements per lane, which are 32 g + 8 j .. of the chunk
// for MXFP4 weights and 32 j + 8 g .. for int4.  Loaded in whole lines, 16 bytes of consecutive lanes side by side, and brought to the
// lanes that need them through `bounce`, 4 KiB of LDS of this wave alone: loads whose lanes follow the operand layout run at a quarter of
// the rate.  Those of one row do not and go without (2880 x 2880, through LDS : without, 1 row 4.29 : 4.15 us, 4 rows 4.41 : 4.59, 16 rows 4.88 : 6.25).
// Rows past the last and elements past K are zeros (reads past a buffer's end).
enum RowForm { kRowsBf16, kRowsE4m3, kOneRowBf16 };
template <int GROUP, int NT, int FORM>
MOE_DEVICE void load_x(const LinearArgs& a, [[maybe_unused]] uint8_t* bounce, int b0, int u, u32x4 (&xr)[2][4][NT]) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // the addresses are made anew for every unit: kept over the loops they cost registers that the weights need
    const int q = lane & 15, g = lane >> 4;
    const uint32_t rows = (uint32_t)min(a.B - b0, 16 * NT), K = (uint32_t)a.K;
    constexpr uint32_t kOutside = 0x80000000u;  // rows * K * 2 < 2^31
    if constexpr (FORM == kOneRowBf16) {
        static_assert(NT == 1);
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.x), 0, (int)(K * 2), 0x00020000);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = kUnit * u + 128 * i + (GROUP ? 32 * j + 8 * g : 32 * g + 8 * j);
                xr[i][j][0] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(q == 0 ? k * 2 : kOutside), 0, 0);
            }
    } else if constexpr (FORM == kRowsBf16) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(static_cast<const uint16_t*>(a.x) + (size_t)b0 * K), 0, (int)(rows * K * 2), 0x00020000);
        // four rows of 256 bytes to an instruction
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t k = kUnit * u + 128 * i + 8 * q;
            const uint32_t at = k < K ? (g * K + k) * 2 : kOutside;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int n = 0; n < 4; ++n) xr[i][n][t] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, (int)((16 * t + 4 * n) * K * 2), 0);
        }
        // piece c (of 16) of row r at position c ^ r of the row's 256 bytes: no two lanes of a read meet in a bank
        const uint32_t put = g * 256 + ((q ^ g) << 4), get = q * 256 + ((GROUP ? g ^ q : 4 * g ^ q) << 4);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int n = 0; n < 4; ++n) *reinterpret_cast<u32x4*>(bounce + 1024 * n + (put ^ (n << 6))) = xr[i][n][t];  // row 4n + g, piece q
                lds_in_order();
#pragma unroll
                for (int j = 0; j < 4; ++j) xr[i][j][t] = *reinterpret_cast<const u32x4*>(bounce + (get ^ (GROUP ? j << 6 : j << 4)));  // 4j + g : 4g + j
                lds_in_order();
            }
    } else {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(static_cast<const uint8_t*>(a.x) + (size_t)b0 * K), 0, (int)(rows * K), 0x00020000);
        const __amdgpu_buffer_rsrc_t s_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(a.x_scales + (size_t)b0 * (K / 32)), 0, (int)(rows * (K / 32)), 0x00020000);
        // eight rows of 128 bytes to an instruction; the scale of the lane's row q and 32 elements g
        const uint32_t put = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 4)) << 4);
        const uint32_t get = GROUP ? q * 128 + (((g ^ q) >> 1) << 4) + 8 * (g & 1) : q * 128 + ((2 * g ^ q >> 1) << 4);
        u32x4 c[2][2][NT];
        uint32_t s[2][NT];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t k = kUnit * u + 128 * i + 16 * (lane & 7), ks = kUnit * u + 128 * i + 32 * g;
            const uint32_t at = k < K ? (uint32_t)(lane >> 3) * K + k : kOutside, at_s = ks < K ? q * (K / 32) + ks / 32 : kOutside;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int n = 0; n < 2; ++n) c[i][n][t] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, (int)((16 * t + 8 * n) * K), 0);
                s[i][t] = __builtin_amdgcn_raw_buffer_load_b8(s_rsrc, (int)at_s, (int)(16 * t * (K / 32)), 0);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // piece p (of 8) of row r at position p ^ (r / 2) of the row's 128 bytes
#pragma unroll
                for (int n = 0; n < 2; ++n) *reinterpret_cast<u32x4*>(bounce + 1024 * n + (put ^ (n << 6))) = c[i][n][t];  // row 8n + lane / 8
                lds_in_order();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // bytes 32 j + 8 g .. of the row's 128 : 32 g + 8 j
                    const uint2 v = *reinterpret_cast<const uint2*>(bounce + (GROUP ? get ^ (j << 5) : (get ^ (j >> 1 << 4)) + 8 * (j & 1)));
                    const uint32_t sb = GROUP ? (uint32_t)__shfl((int)s[i][t], 16 * j + q) : s[i][t];
                    xr[i][j][t] = e4m3x8_to_bf16(v.x, v.y, mxfp4_scale_to_f32(sb));
                }
                lds_in_order();
            }
    }
}

// Codes less their zero point, exact in e4m3: weights without their scale.  Four codes 0..15 in the bytes of `q`, 128 + zero point in every byte of
// `z`.  A byte u = 128 + z - q with its top bit set is -(z - q) in sign and magnitude as it stands; in the others the magnitude is 128 - u and the
// sign plus.  Magnitudes up to 15 are e4m3 codes of themselves, in steps of 2^-9.  (The bf16 numbers 16 + code are cheaper to make, with 16 + zero
// times the sum of x taken off each group's sum.  That loses what cancels between the two, and overflows where the result does not.  So : exact, us, 16
// rows of 65536 x 2880, scales per 128 24.4 : 25.8, per 64 27.0 : 27.7, per 32 41.6 : 32.1, with room for more waves now.)
MOE_DEVICE uint32_t int4_less_zero_e4m3(uint32_t q, uint32_t z) {
    const uint32_t u = z - q;  // no byte borrows from the next
    const uint32_t positive = ~u & 0x80808080u, one = positive >> 7;
    return (u ^ (positive - one)) + one;
}
// Eight codes of a dword (order of int4_repack_kernel).
MOE_DEVICE u32x4 int4_dword_to_bf16x8(uint32_t w, uint32_t z) {
    constexpr uint32_t kCodes = 0x0F0F0F0Fu;
    return e4m3x8_to_bf16(int4_less_zero_e4m3(w & kCodes, z), int4_less_zero_e4m3((w >> 4) & kCodes, z), 512.f);
}

}  // namespace

// The weights of one unit of a tile as they come from memory.
template <int GROUP>
struct UnitWeights {
    static constexpr int kGroups = GROUP ? kUnit / GROUP : 1;
    u32x4 raw[2];
    uint32_t sw;                      // MXFP4: the scale bytes of four chunks
    u32x4 sc[GROUP ? kGroups / 2 : 1];  // int4: four rows' scales of two groups, those of the lane's results
    uint32_t zp[2];                     // and a byte zero point ^ 8 for every group of the lane's row of weights

    // Unit u of a tile; nothing is read unless `in`, without a branch: the compiler would wait for every load in flight where two paths meet.
    MOE_DEVICE void load(const LinearArgs& a, int tile, int u, bool in) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const int n_chunks = ceil_div(a.K, 128), n_units = ceil_div(a.K, kUnit);
        const uint32_t tile_bytes = GROUP ? (uint32_t)n_chunks * 1024u : (uint32_t)(a.K / 32) * 256u;
        const uint32_t scale_bytes = GROUP ? (uint32_t)n_units * (kGroups * 32u) : (uint32_t)ceil_div(n_chunks, 4) * 256u;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.w) + (size_t)(uint32_t)tile * tile_bytes, 0,
                                                                              in ? (int)tile_bytes : 0, 0x00020000);
        const __amdgpu_buffer_rsrc_t s_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(a.w_scales) + (size_t)(uint32_t)tile * scale_bytes, 0, in ? (int)scale_bytes : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < 2; ++i) raw[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane * 16, (2 * u + i) * 1024, 2 /* nt */);
        if constexpr (GROUP == 0) {
            sw = __builtin_amdgcn_raw_buffer_load_b32(s_rsrc, lane * 4, (u >> 1) * 256, 0);
        } else {
#pragma unroll
            for (int i = 0; i < kGroups / 2; ++i)
                sc[i] = __builtin_amdgcn_raw_buffer_load_b128(s_rsrc, g * kGroups * 8 + i * 16, u * kGroups * 32, 0);
            const __amdgpu_buffer_rsrc_t z_rsrc =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.w_zeros) + (size_t)(uint32_t)tile * (scale_bytes / 2), 0,
                                                  in && a.w_zeros ? (int)(scale_bytes / 2) : 0, 0x00020000);
            const int at = (lane & 15) * kGroups;  // without zero points 0 is read, which stands for 8
            if constexpr (kGroups == 8) {
                const u32x2 z = __builtin_amdgcn_raw_buffer_load_b64(z_rsrc, at, u * kGroups * 16, 0);
                zp[0] = z[0], zp[1] = z[1];
            } else if constexpr (kGroups == 4) {
                zp[0] = __builtin_amdgcn_raw_buffer_load_b32(z_rsrc, at, u * kGroups * 16, 0);
            } else {
                zp[0] = __builtin_amdgcn_raw_buffer_load_b16(z_rsrc, at, u * kGroups * 16, 0);
            }
        }
    }

    // acc = the unit's products with x, from zero
    template <int NT>
    MOE_DEVICE void multiply(int u, const u32x4 (&xr)[2][4][NT], f32x4 (&acc)[NT]) const {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = zero;
        if constexpr (GROUP == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // reads past the tile give 0, and the scale bytes of blocks that do not exist are 0
                const float s = mxfp4_scale_to_f32((sw >> (16 * (u & 1) + 8 * i)) & 0xFFu);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t d[4];
                    mxfp4_dword_to_bf16x8(raw[i][j], s, d);
                    const u32x4 av = {d[0], d[1], d[2], d[3]};
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = mfma_16x16x32(av, xr[i][j][t], acc[t]);
                }
            }
        } else {
            f32x4 p[NT];
            uint32_t z = 0;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int grp = 32 * n / GROUP;
                if (32 * n % GROUP == 0) z = __builtin_amdgcn_perm(0u, zp[grp >> 2] ^ 0x88888888u, 0x01010101u * (grp & 3));
                const u32x4 av = int4_dword_to_bf16x8(raw[n >> 2][n & 3], z);
#pragma unroll
                for (int t = 0; t < NT; ++t) p[t] = mfma_16x16x32(av, xr[n >> 2][n & 3][t], 32 * n % GROUP == 0 ? zero : p[t]);
                if (32 * (n + 1) % GROUP == 0) {
                    const uint32_t s01 = sc[grp / 2][2 * (grp & 1)], s23 = sc[grp / 2][2 * (grp & 1) + 1];
                    const float s[4] = {bf16_bits_to_f32(s01 & 0xFFFFu), bf16_bits_to_f32(s01 >> 16), bf16_bits_to_f32(s23 & 0xFFFFu),
                                        bf16_bits_to_f32(s23 >> 16)};
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t][r] = fmaf(s[r], p[t][r], acc[t][r]);
                }
            }
        }
    }
};

// Weight row of row r of a tile.
template <int GROUP>
MOE_DEVICE int weight_row(int tile, int r) {
    return GROUP ? tile * 16 + r : (tile >> 2) * 64 + tile_row_in_group(tile & 3, r);
}

// Four results of token b from weight row n on.
MOE_DEVICE void store_results(const LinearArgs& a, int b, int n, const f32x4& v) {
    float* const dst = a.y + (size_t)b * a.N + n;
    if (a.wide_stores) {  // N is a multiple of four
        if (n < a.N) *reinterpret_cast<f32x4*>(dst) = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < a.N) dst[r] = v[r];
    }
}

MOE_DEVICE f32x4 load_bias(const LinearArgs& a, int n) {  // 0 without one, and past N
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.bias), 0, a.bias ? a.N * 2 : 0, 0x00020000);
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = bf16_bits_to_f32((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(rsrc, (n + r) * 2, 0, 0));
    return v;
}

// Few tiles: a block for each, its waves take the units in turn.  Such a launch is a chain of latencies (arguments, weights and rows, LDS
// and back, the waves' meeting, stores), so its code is short and nothing waits before the first loads are out: kernels of their own for each form of
// x and (ONE) for a wave to every unit, without a loop over them.  All in one : so, us: 1 row of 2880 x 2880 4.43 : 3.96, 16 rows 4.93 : 4.78, 1 row of
// 2880 x 8192 7.5 : 7.0.  In the loop nothing is loaded ahead: with the next unit's weights on their way 1 row of 4096 x 16384 took 11.7 : 12.0.
template <int GROUP, int NT, int FORM, bool ONE>
__global__ __launch_bounds__(64 * max_waves(GROUP, NT)) void linear_tile_kernel(LinearArgs a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int tile = blockIdx.z * 8 + blockIdx.x, b0 = blockIdx.y * 16 * NT;
    const int n_units = ceil_div(a.K, kUnit);
    float* const part = lds;  // [n_units][NT][256]
    uint8_t* const bounce = reinterpret_cast<uint8_t*>(lds + n_units * NT * 256) + wave * 4096;
    if (tile * 16 >= a.N) return;
    for (int u = wave; ONE || u < n_units; u += waves) {
        UnitWeights<GROUP> w;
        w.load(a, tile, u, true);
        u32x4 xr[2][4][NT];
        load_x<GROUP, NT, FORM>(a, bounce, b0, u, xr);
        f32x4 acc[NT];
        w.template multiply<NT>(u, xr, acc);
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(part + (u * NT + t) * 256 + lane * 4) = acc[t];
        if constexpr (ONE) break;
    }
    const int n = weight_row<GROUP>(tile, 4 * (lane >> 4));
    f32x4 bias = {0.f, 0.f, 0.f, 0.f};
    if (wave < NT) bias = load_bias(a, n);
    __syncthreads();
    for (int t = wave; t < NT; t += waves) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int u = 0; u < n_units; ++u) v += *reinterpret_cast<const f32x4*>(part + (u * NT + t) * 256 + lane * 4);
        const int b = b0 + t * 16 + (lane & 15);
        if (b < a.B) store_results(a, b, n, v + bias);
    }
}

// Waves of a block of linear_w4_kernel that add up what the others leave: one for each tile of 16 x 16 of a step, up to a quarter of all.
constexpr int adders(int group, int nt, int tiles_per_step) {
    const int most = max_waves(group, nt) / 4;
    return nt * tiles_per_step < most ? nt * tiles_per_step : most;
}

// How a launch is cut: a block has wk x wr waves; the contraction's units are dealt out over wk waves, in as many slabs as that takes, and its
// tiles of 16 weight rows, tiles_per_block consecutive ones, over wr.
struct LinearCut {
    int wk, log_wr, n_slabs, tiles_per_block;
    int inv_wk;  // 65536 / wk, rounded up
    int tiles_per_step;  // tile sets between two barriers that there is room for
};

// GROUP 0: MXFP4 weights in the tiled layout of mxfp4.hip; else int4 codes with a scale per GROUP values (layout of int4_repack_kernel).
// A wave holds its unit of 16 NT rows of x in registers and goes through the block's tiles, the weights of the next D in flight; every G tiles
// the waves meet, and further waves add up the partial tiles that they have left in LDS, while they go on.  A result is the sum over units in
// ascending order, whatever the cut: it does not depend on how many rows x has.
template <int GROUP, int NT, int D, int G>
__global__ __launch_bounds__(64 * max_waves(GROUP, NT)) void linear_w4_kernel(LinearArgs a, LinearCut cut) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    constexpr int kPart = NT * 256;  // values of a tile
    constexpr int kAdders = adders(GROUP, NT, G);
    // grid (8, token blocks, tile blocks / 8): token blocks of the same weights side by side on one XCD; no quotient is formed in here, each is
    // a chain of forty instructions, and a launch for one row is little more than a few chains
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n_wr = 1 << cut.log_wr, waves = cut.wk << cut.log_wr;  // and kAdders more
    const int wr = wave * cut.inv_wk >> 16, wk = wave - wr * cut.wk;
    const int q = lane & 15, g = lane >> 4;
    const int n_units = ceil_div(a.K, kUnit);
    const int n_tiles = ceil_div(a.N, 16);
    const int token_block = blockIdx.y, tile_block = blockIdx.z * 8 + blockIdx.x;
    const int tile0 = tile_block * cut.tiles_per_block, tile1 = min(tile0 + cut.tiles_per_block, n_tiles);
    if (tile0 >= n_tiles) return;
    const int n_slabs = cut.n_slabs;
    // a wave's partial tiles, G of them in either half; x goes through the first while it is loaded
    const int per_wave = part_floats(NT, cut.tiles_per_step);
    float* const part = lds;                              // [waves][2][tiles_per_step][kPart]
    float* const bias = lds + waves * per_wave;           // [tiles_per_block][16]
    float* const sums = bias + cut.tiles_per_block * 16;    // [tiles_per_block][kPart] between slabs
    const int b0 = token_block * 16 * NT;
    const int n_bias = (tile1 - tile0) * 16;
    for (int i = threadIdx.x; i < n_bias; i += 64 * (waves + kAdders)) {
        const int n = weight_row<GROUP>(tile0 + (i >> 4), i & 15);
        bias[i] = a.bias && n < a.N ? bf16_bits_to_f32(a.bias[n]) : 0.f;
    }
    // The block's sets of n_wr tiles; blocks begin at different ones of theirs: side by side they would read from the same few channels of the
    // memory (1 row of 131072 x 2880 34.4 : 33.5 us, 16 rows of 262144 x 2880 78.1 : 74.6).  Not with more rows, where blocks with the same
    // tiles run beside each other (64 rows of 131072 x 2880 62.8 : 64.2).
    const int n_sets = (tile1 - tile0 + n_wr - 1) >> cut.log_wr;
    const int first_set = NT == 1 ? (n_sets * (tile_block & 31) >> 5) & -G : 0;
    auto first_tile = [&](int j) {
        const int set = j + first_set;
        return tile0 + ((set >= n_sets ? set - n_sets : set) << cut.log_wr);
    };
    constexpr int kPass = D > G ? D : G;
    int half = 0;  // which half of `part` a step writes

    if (wave >= waves) {
        // The waves that add up.  They load nothing: a wave's loads and stores are waited for in their order, and a store in front of the next
        // weights holds up the wave, and all others at the next meeting (131072 x 2880, by the waves themselves : by these, 16 rows 39.4 : 38.4 us,
        // 64 rows 72 : 63).
        for (int slab = 0; slab < n_slabs; ++slab) {
            const int units = min(cut.wk, n_units - slab * cut.wk);
            for (int j = 0; j < (n_sets + kPass - 1) / kPass * kPass; j += G) {
                __syncthreads();
                // item (m, w, t): token tile t of the m-th tile of row wave w
                const int items = (max(0, min(G, n_sets - j)) << cut.log_wr) * NT;
                for (int item = wave - waves; item < items; item += kAdders) {
                    const int set = item / NT, t = item - set * NT;
                    const int m = set >> cut.log_wr, w = set & (n_wr - 1);
                    const int tl = first_tile(j + m) + w;  // wave-uniform
                    if (tl >= tile1) continue;
                    const float* src = part + w * cut.wk * per_wave + (half * cut.tiles_per_step + m) * kPart + t * 256 + lane * 4;
                    float* const between = sums + (tl - tile0) * kPart + t * 256 + lane * 4;
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
                    if (slab > 0) v = *reinterpret_cast<const f32x4*>(between);
#pragma unroll 4
                    for (int i = 0; i < units; ++i) v += *reinterpret_cast<const f32x4*>(src + i * per_wave);
                    if (slab + 1 < n_slabs) {
                        *reinterpret_cast<f32x4*>(between) = v;
                        continue;
                    }
                    const int b = b0 + t * 16 + q;
                    v += *reinterpret_cast<const f32x4*>(bias + (tl - tile0) * 16 + 4 * g);
                    if (b < a.B) store_results(a, b, weight_row<GROUP>(tl, 4 * g), v);
                }
                half ^= 1;
            }
            if (slab + 1 < n_slabs) __syncthreads();
        }
        return;
    }

    UnitWeights<GROUP> w[D];
    for (int slab = 0; slab < n_slabs; ++slab) {
        const int u = slab * cut.wk + wk;
        auto load_slot = [&](int d, int j) {
            const int tile = first_tile(j) + wr;
            w[d].load(a, min(tile, n_tiles - 1), u, j < n_sets && tile < tile1 && u < n_units);
        };
        load_slot(0, 0);
        u32x4 xr[2][4][NT];
        uint8_t* const bounce = reinterpret_cast<uint8_t*>(part + wave * per_wave);
        if (a.x_scales) load_x<GROUP, NT, kRowsE4m3>(a, bounce, b0, u, xr);
        else load_x<GROUP, NT, kRowsBf16>(a, bounce, b0, u, xr);
        __builtin_amdgcn_sched_barrier(0);  // the other slots' registers are free until x is where it stays
#pragma unroll
        for (int d = 1; d < D; ++d) load_slot(d, d);
        // partial tile of set j, in slot S of the ring, the m-th of its step
        auto tile_part = [&](auto slot_tag, int m, int j) {
            constexpr int S = decltype(slot_tag)::value;
            f32x4 acc[NT];
            w[S].template multiply<NT>(u, xr, acc);
            __builtin_amdgcn_sched_barrier(0);
            load_slot(S, j + D);  // the slot is free
            __builtin_amdgcn_sched_barrier(0);
            if (j >= n_sets) return;  // block-uniform
            float* const mine = part + wave * per_wave + ((half * cut.tiles_per_step) + m) * kPart;
#pragma unroll
            for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(mine + t * 256 + lane * 4) = acc[t];
        };
        // the ring's slots are constants: D or G sets, whichever is more, to a pass of the loop
        for (int j = 0; j < n_sets; j += kPass) {
            auto at = [&](auto m_tag) {
                constexpr int M = decltype(m_tag)::value;
                if constexpr (M < kPass) {
                    tile_part(std::integral_constant<int, M % D>{}, M % G, j + M);
                    if constexpr (M % G == G - 1) {
                        __syncthreads();
                        half ^= 1;
                    }
                }
            };
            at(std::integral_constant<int, 0>{});
            at(std::integral_constant<int, 1>{});
            at(std::integral_constant<int, 2>{});
            at(std::integral_constant<int, 3>{});
        }
        if (slab + 1 < n_slabs) __syncthreads();  // the next slab's x goes through `part`
    }
}

constexpr size_t kLdsMost = 160 * 1024;

// A block for each tile: n_units partial tiles and 4 KiB a wave in LDS.
static size_t linear_tile_lds(int group, int nt, int n_units) {
    return (size_t)n_units * nt * 1024 + (size_t)std::min(n_units, max_waves(group, nt)) * 4096;
}

template <int GROUP, int NT>
static int launch_linear_tile(const LinearArgs& a, int n_units, hipStream_t stream) {
    const int waves = std::min(n_units, max_waves(GROUP, NT));
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(8, ceil_div(a.B, 16 * NT), ceil_div(ceil_div(a.N, 16), 8)), dim3(64 * waves), linear_tile_lds(GROUP, NT, n_units),
                           stream, a);
        return launch_status();
    };
    auto of = [&](auto form) {
        constexpr int FORM = decltype(form)::value;
        return n_units == waves ? launch(linear_tile_kernel<GROUP, NT, FORM, true>) : launch(linear_tile_kernel<GROUP, NT, FORM, false>);
    };
    if (a.x_scales) return of(std::integral_constant<int, kRowsE4m3>{});
    if constexpr (NT == 1)
        if (a.B == 1) return of(std::integral_constant<int, kOneRowBf16>{});
    return of(std::integral_constant<int, kRowsBf16>{});
}

template <int GROUP, int NT, int D, int G>
static int launch_linear_of(const LinearArgs& a, int n_cus, hipStream_t stream) {
    const int n_tiles = ceil_div(a.N, 16), n_units = ceil_div(a.K, kUnit);
    LinearCut cut;
    constexpr int kAdders = adders(GROUP, NT, G);
    const int slabs = ceil_div(n_units, max_waves(GROUP, NT) - kAdders);
    cut.n_slabs = slabs;
    cut.wk = ceil_div(n_units, slabs);
    cut.inv_wk = ceil_div(65536, cut.wk);
    cut.log_wr = 0;
    while ((cut.wk << (cut.log_wr + 1)) + kAdders <= std::min(12, max_waves(GROUP, NT)) && n_tiles >> cut.log_wr > n_cus) ++cut.log_wr;
    const int wr = 1 << cut.log_wr, waves = cut.wk * wr, token_blocks = ceil_div(a.B, 16 * NT);
    const int at_once = n_cus * std::max(1, max_waves(GROUP, NT) / (waves + kAdders));
    const int most = (slabs > 1 ? 32 / NT : 128) / wr;  // what the LDS has room for
    cut.tiles_per_block = std::min(most, ceil_div(n_tiles * token_blocks, at_once * wr)) * wr;
    cut.tiles_per_step = std::min(G, cut.tiles_per_block / wr);
    const size_t lds = (size_t)waves * part_floats(NT, cut.tiles_per_step) * 4 + (size_t)cut.tiles_per_block * (64 + (slabs > 1 ? NT * 1024 : 0));
    const int blocks = ceil_div(n_tiles, cut.tiles_per_block);
    hipLaunchKernelGGL((linear_w4_kernel<GROUP, NT, D, G>), dim3(8, token_blocks, ceil_div(blocks, 8)), dim3(64 * (waves + kAdders)), lds,
                       stream, a, cut);
    return launch_status();
}

// Which kernel: by the matrix and the number of rows alone, and all of them add in the same order.
template <int GROUP, int NT>
static int launch_linear_rows(const LinearArgs& a, int n_cus, hipStream_t stream) {
    const int n_units = ceil_div(a.K, kUnit);
    const long long tiles = (long long)ceil_div(a.N, 16) * ceil_div(a.B, 16 * NT);
    // Blocks of a tile that are there at once, 24 waves of them to a compute unit, up to three: us, so : the first form below, 7 rows of 5760 x 2880 with int4
    // scales per 64 6.5 : 7.1, 16 rows of 8192 x 1024 4.4 : 4.9, 8 rows of 12288 x 512 int4 4.1 : 5.5.  Not with more of them than that (16 rows of 12288 x
    // 4096 12.3 : 11.5, of 8192 x 8192 16.0 : 13.4), nor with more than three, which read x that much more often (16 rows of 16384 x 1536 7.7 : 6.3), nor
    // with 32 rows (64 rows of 5760 x 2880 12.4 : 9.1).
    const int at_once = NT == 1 ? std::clamp(24 / n_units, 1, 3) : 1;
    if (tiles <= (long long)n_cus * at_once && linear_tile_lds(GROUP, NT, n_units) <= kLdsMost) return launch_linear_tile<GROUP, NT>(a, n_units, stream);
    // With up to three tiles to a block the longer ring and the wider steps of the second form cost more code than they hide: us, first : second
    // form, 16 rows of 6144 x 8192 int4 15.7 : 19.7, 1 row of 16384 x 4096 MXFP4 11.7 : 10.1, 16 rows of 131072 x 2880 42.7 : 38.6.  int4 scales per 32 need the registers of a ring of two for more waves (65536 x 2880, 16 rows, 16 waves : 12 with the ring, 32.3 : 37.4).
    if (tiles <= 3LL * n_cus || GROUP == 32) return launch_linear_of<GROUP, NT, 1, 2>(a, n_cus, stream);
    if constexpr (GROUP != 32) return launch_linear_of<GROUP, NT, 2, 4 / NT>(a, n_cus, stream);
    return MOE_ERR_LIMIT;
}

int launch_linear_w4(const LinearArgs& args, int group, int n_cus, hipStream_t stream) {
    LinearArgs a = args;
    a.wide_stores = a.N % 4 == 0 && ((uintptr_t)a.y & 15u) == 0;
    auto rows = [&](auto g) {
        constexpr int GROUP = decltype(g)::value;
        return a.B <= 16 ? launch_linear_rows<GROUP, 1>(a, n_cus, stream) : launch_linear_rows<GROUP, 2>(a, n_cus, stream);
    };
    switch (group) {
        case 0: return rows(std::integral_constant<int, 0>{});
        case 32: return rows(std::integral_constant<int, 32>{});
        case 64: return rows(std::integral_constant<int, 64>{});
        case 128: return rows(std::integral_constant<int, 128>{});
    }
    return MOE_ERR_FORMAT;
}

// ---- int4 codes ------------------------------------------------------------------------------------
// Tiles of 16 weight rows, a tile's contraction in chunks of 128 elements (the last one filled up with zeros), lane 16 g + r of a chunk's
// 1 KiB: dword j holds elements 32 j + 8 g .. + 8 of row r, the first four in the low halves of its bytes, the others in the high ones.
// Scales bf16 [tile][unit of 256][4 lane groups][groups of the unit][4 rows]: a lane reads those of the four rows it gets from the matrix instruction
// in one piece.  Zero points as the byte z ^ 8 [tile][unit][16 rows][groups of the unit]: a lane reads those of the row it unpacks.  0 past the last
// row and group.
void int4_tiled_bytes(int rows, int K, int group, size_t* codes, size_t* scales, size_t* zeros) {
    const size_t tiles = (size_t)ceil_div(rows, 16), groups = (size_t)ceil_div(K, kUnit) * (kUnit / group);
    if (codes) *codes = tiles * (size_t)ceil_div(K, 128) * 1024;
    if (scales) *scales = tiles * groups * 32;
    if (zeros) *zeros = tiles * groups * 16;
}

__global__ __launch_bounds__(256) void int4_repack_kernel(const uint32_t* __restrict__ codes, u32x4* __restrict__ out, int rows, int K,
                                                          long long n_lanes) {
    const int n_chunks = ceil_div(K, 128);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n_lanes; i += (long long)gridDim.x * 256) {
        const long long chunk = i >> 6;
        const int lane = (int)(i & 63), c = (int)(chunk % n_chunks);
        const long long row = chunk / n_chunks * 16 + (lane & 15);
        u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 128 * c + 32 * j + 8 * (lane >> 4);
            if (row < rows && k < K) {
                const uint32_t w = codes[(size_t)row * (K / 8) + k / 8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j] |= ((w >> (4 * e)) & 0xFu) << (8 * (e & 3) + 4 * (e >> 2));
            }
        }
        out[i] = v;
    }
}

__global__ __launch_bounds__(256) void int4_scales_repack_kernel(const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                                 uint16_t* __restrict__ out_scales, uint8_t* __restrict__ out_zeros, int rows,
                                                                 int K, int group, long long n) {
    const int per_unit = kUnit / group, n_units = ceil_div(K, kUnit), n_groups = ceil_div(K, group);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long unit = i / (16 * per_unit);  // over all tiles
        const int in_unit = (int)(i - unit * (16 * per_unit));
        const long long row0 = unit / n_units * 16, group0 = unit % n_units * per_unit;
        auto source = [&](int row, int grp) {  // -1: past the last row or group
            return row0 + row < rows && group0 + grp < n_groups ? (row0 + row) * n_groups + group0 + grp : -1ll;
        };
        const long long s = source(in_unit / (4 * per_unit) * 4 + (in_unit & 3), in_unit / 4 % per_unit);
        out_scales[i] = s >= 0 ? scales[s] : 0;
        if (zeros) {
            const long long z = source(in_unit / per_unit, in_unit % per_unit);
            out_zeros[i] = z >= 0 ? (uint8_t)((zeros[z] & 15) ^ 8) : 0;
        }
    }
}

int launch_int4_repack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int rows, int K, int group, uint8_t* tiled_codes,
                       uint16_t* tiled_scales, uint8_t* tiled_zeros, hipStream_t stream) {
    const long long lanes = (long long)ceil_div(rows, 16) * ceil_div(K, 128) * 64;
    const auto blocks = [](long long items) { return dim3((unsigned)std::min(ceil_div(items, 256ll), kMostThreads / 256)); };
    hipLaunchKernelGGL(int4_repack_kernel, blocks(lanes), dim3(256), 0, stream,
                       reinterpret_cast<const uint32_t*>(codes), reinterpret_cast<u32x4*>(tiled_codes), rows, K, lanes);
    const long long n = (long long)ceil_div(rows, 16) * ceil_div(K, kUnit) * (kUnit / group) * 16;
    hipLaunchKernelGGL(int4_scales_repack_kernel, blocks(n), dim3(256), 0, stream, scales, zeros, tiled_scales,
                       tiled_zeros, rows, K, group, n);
    return launch_status();
}

}  // namespace moe
