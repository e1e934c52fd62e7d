// Products of a few rows with a matrix of 4-bit weights and group scales: y[b, n] = bias[n] + sum_k x[b, k] W[n, k].
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace moe {

namespace {

constexpr int kLinearWaves = 8;

// e4m3 values times a power of two, to bf16 (exact: three mantissa bits).
MOE_DEVICE u32x4 e4m3x8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
    u32x4 v;
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return v;
}

// Eight codes 0..15 of a dword (order of int4_repack_kernel) as the bf16 numbers 16..31: the code goes to the mantissa's top four bits.
MOE_DEVICE u32x4 int4_dword_to_bf16x8(uint32_t w) {
    constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u;
    return u32x4{((w << 3) & kMask) | kSixteen, ((w >> 1) & kMask) | kSixteen, ((w >> 5) & kMask) | kSixteen, ((w >> 9) & kMask) | kSixteen};
}

}  // namespace

// GROUP 0: MXFP4 weights in the tiled layout of mxfp4.hip; else int4 codes with a scale per GROUP values (layout of int4_repack_kernel).
// A block takes a tile of 16 weight rows against 16 NT rows of x; its waves share the contraction, in chunks of 128, and meet in LDS.
template <int GROUP, int NT, bool MX8>
__global__ __launch_bounds__(64 * kLinearWaves) void linear_w4_kernel(LinearArgs a) {
    __shared__ __attribute__((aligned(16))) float part[kLinearWaves][NT * 256];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x, K = a.K;
    const int n_chunks = ceil_div(K, 128);
    const int per_wave = ceil_div(n_chunks, kLinearWaves);
    const int c0 = wave * per_wave, c1 = min(c0 + per_wave, n_chunks);
    const uint32_t tile_bytes = GROUP ? (uint32_t)n_chunks * 1024u : (uint32_t)(K / 32) * 256u;
    const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.w) + (size_t)tile * tile_bytes, 0, (int)tile_bytes, 0x00020000);
    int tok[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) tok[t] = min((int)blockIdx.y * 16 * NT + t * 16 + q, a.B - 1);
    // the 8 contraction elements of MFMA step j for this lane: their first
    auto elem = [&](int c, int j) { return 128 * c + (GROUP ? 32 * j + 8 * g : 32 * g + 8 * j); };
    auto x_frag = [&](int c, int j, int t) {
        const int k = elem(c, j);
        if (k >= K) return u32x4{0u, 0u, 0u, 0u};
        if constexpr (MX8) {
            const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.x) + (size_t)tok[t] * K + k);
            const float s = mxfp4_scale_to_f32(a.x_scales[(size_t)tok[t] * (K / 32) + k / 32]);
            return e4m3x8_to_bf16(v.x, v.y, s);
        } else {
            return *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x) + (size_t)tok[t] * K + k);
        }
    };
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = c0; c < c1; ++c) {
        const u32x4 raw = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, lane * 16, c * 1024, 2 /* nt */);
        if constexpr (GROUP == 0) {
            // reads past the tile give 0, and the scale bytes of blocks that do not exist are 0
            const uint32_t sw = *reinterpret_cast<const uint32_t*>(a.w_scales + (size_t)tile * ceil_div(n_chunks, 4) * 256 +
                                                                   (c >> 2) * 256 + lane * 4);
            const float sc = mxfp4_scale_to_f32((sw >> (8 * (c & 3))) & 0xFFu);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t d[4];
                mxfp4_dword_to_bf16x8(raw[j], sc, d);
                const u32x4 av = {d[0], d[1], d[2], d[3]};
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t] = mfma_16x16x32(av, x_frag(c, j, t), acc[t]);
            }
        } else {
            // sum x (q - z) s = s (sum x (16 + q) - (16 + z) sum x) per group: 16 + q is a bf16 number, and the sum of x comes from a
            // product with ones
            const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
            const int n_groups = ceil_div(K, GROUP);
            f32x4 part_g[NT], sum_x[NT];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool first = 32 * j % GROUP == 0, last = 32 * (j + 1) % GROUP == 0;
                const u32x4 av = int4_dword_to_bf16x8(raw[j]);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const u32x4 xv = x_frag(c, j, t);
                    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                    part_g[t] = mfma_16x16x32(av, xv, first ? zero : part_g[t]);
                    sum_x[t] = mfma_16x16x32(ones, xv, first ? zero : sum_x[t]);
                }
                const int grp = (128 * c + 32 * j) / GROUP;
                if (last && grp < n_groups) {
                    const size_t at = ((size_t)tile * n_groups + grp) * 16 + 4 * g;
                    const uint2 sb = *reinterpret_cast<const uint2*>(a.w_scales + 2 * at);
                    const uint32_t zb = a.w_zeros ? *reinterpret_cast<const uint32_t*>(a.w_zeros + at) : 0x18181818u;
                    const float s[4] = {bf16_bits_to_f32(sb.x & 0xFFFFu), bf16_bits_to_f32(sb.x >> 16), bf16_bits_to_f32(sb.y & 0xFFFFu),
                                        bf16_bits_to_f32(sb.y >> 16)};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float z = (float)((zb >> (8 * i)) & 0xFFu);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t][i] = fmaf(s[i], fmaf(-z, sum_x[t][i], part_g[t][i]), acc[t][i]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(&part[wave][t * 256 + q * 16 + 4 * g]) = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 256; i += 64 * kLinearWaves) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kLinearWaves; ++w) v += part[w][i];
        const int r = i & 15;  // row of the tile
        const int n = GROUP ? tile * 16 + r : (tile >> 2) * 64 + tile_row_in_group(tile & 3, r);
        const int b = (int)blockIdx.y * 16 * NT + (i >> 4);
        if (b < a.B && n < a.N) {
            if (a.bias) v += bf16_bits_to_f32(a.bias[n]);
            a.y[(size_t)b * a.N + n] = v;
        }
    }
}

template <int GROUP>
static int launch_linear_of(const LinearArgs& a, hipStream_t stream) {
    const unsigned tiles = (unsigned)ceil_div(a.N, 16);
    auto launch = [&](auto kernel, int nt) {
        hipLaunchKernelGGL(kernel, dim3(tiles, ceil_div(a.B, 16 * nt)), dim3(64 * kLinearWaves), 0, stream, a);
        return launch_status();
    };
    if (a.x_scales) {
        if (a.B <= 16) return launch(linear_w4_kernel<GROUP, 1, true>, 1);
        if (a.B <= 32) return launch(linear_w4_kernel<GROUP, 2, true>, 2);
        return launch(linear_w4_kernel<GROUP, 4, true>, 4);
    }
    if (a.B <= 16) return launch(linear_w4_kernel<GROUP, 1, false>, 1);
    if (a.B <= 32) return launch(linear_w4_kernel<GROUP, 2, false>, 2);
    return launch(linear_w4_kernel<GROUP, 4, false>, 4);
}

int launch_linear_w4(const LinearArgs& a, int group, hipStream_t stream) {
    switch (group) {
        case 0: return launch_linear_of<0>(a, stream);
        case 32: return launch_linear_of<32>(a, stream);
        case 64: return launch_linear_of<64>(a, stream);
        case 128: return launch_linear_of<128>(a, stream);
    }
    return MOE_ERR_FORMAT;
}

// ---- int4 codes ------------------------------------------------------------------------------------
// Tiles of 16 weight rows, a tile's contraction in chunks of 128 elements (the last one filled up with zeros), lane 16 g + r of a chunk's
// 1 KiB: dword j holds elements 32 j + 8 g .. + 8 of row r, the element pair 2p, 2p + 1 at bits 4p and 16 + 4p, so that a shift and a mask leave a
// pair at the same place of a dword's two halves.  Scales [tile][group][16] bf16, zero points [tile][group][16] as the byte 16 + z; 0 past the
// last row.
void int4_tiled_bytes(int rows, int K, int group, size_t* codes, size_t* scales, size_t* zeros) {
    const size_t tiles = (size_t)ceil_div(rows, 16), groups = (size_t)ceil_div(K, group);
    if (codes) *codes = tiles * (size_t)ceil_div(K, 128) * 1024;
    if (scales) *scales = tiles * groups * 32;
    if (zeros) *zeros = tiles * groups * 16;
}

__global__ __launch_bounds__(256) void int4_repack_kernel(const uint32_t* __restrict__ codes, u32x4* __restrict__ out, int rows, int K,
                                                          long long n_lanes) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_lanes) return;
    const int n_chunks = ceil_div(K, 128);
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
            for (int p = 0; p < 4; ++p) v[j] |= ((w >> (8 * p)) & 0xFu) << (4 * p) | ((w >> (8 * p + 4)) & 0xFu) << (16 + 4 * p);
        }
    }
    out[i] = v;
}

__global__ __launch_bounds__(256) void int4_scales_repack_kernel(const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                                 uint16_t* __restrict__ out_scales, uint8_t* __restrict__ out_zeros, int rows,
                                                                 int n_groups, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long tg = i >> 4, row = tg / n_groups * 16 + (i & 15);
    const size_t src = (size_t)row * n_groups + (size_t)(tg % n_groups);
    out_scales[i] = row < rows ? scales[src] : 0;
    if (zeros) out_zeros[i] = row < rows ? (uint8_t)(16 + (zeros[src] & 15)) : 0;
}

int launch_int4_repack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int rows, int K, int group, uint8_t* tiled_codes,
                       uint16_t* tiled_scales, uint8_t* tiled_zeros, hipStream_t stream) {
    const long long lanes = (long long)ceil_div(rows, 16) * ceil_div(K, 128) * 64;
    hipLaunchKernelGGL(int4_repack_kernel, dim3((unsigned)ceil_div(lanes, 256ll)), dim3(256), 0, stream,
                       reinterpret_cast<const uint32_t*>(codes), reinterpret_cast<u32x4*>(tiled_codes), rows, K, lanes);
    const int groups = ceil_div(K, group);
    const long long n = (long long)ceil_div(rows, 16) * groups * 16;
    hipLaunchKernelGGL(int4_scales_repack_kernel, dim3((unsigned)ceil_div(n, 256ll)), dim3(256), 0, stream, scales, zeros, tiled_scales,
                       tiled_zeros, rows, groups, n);
    return launch_status();
}

}  // namespace moe
