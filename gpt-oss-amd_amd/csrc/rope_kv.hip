// Rows of a query/key/value projection: queries and keys rotated by position, keys and values into a paged cache.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "mx8.h"

namespace moe {

// p f / (2 pi) less the nearest whole number, to 2^-53: the product (31 by 24 bits) and 1 / (2 pi) as two numbers each, and what the product of the leading two
// leaves.  One rounding of each alone is off by 2^-21 of the angle's cosine at positions next to 2^31, and by codes of the 8-bit cache from far fewer on.
MOE_DEVICE double part_of_turn(double p, double f) {
#pragma clang fp contract(off)  // a product fused with the difference would have its rest taken twice
    constexpr double c = 0x1.45f306dc9c883p-3, c_rest = -0x1.6b01ec5417056p-57;
    const double angle = p * f, angle_rest = fma(p, f, -angle), turns = angle * c;
    return (turns - rint(turns)) + (fma(angle, c, -turns) + fma(angle_rest, c, angle * c_rest));
}

// Pairs (u, v) = (x[i], x[i + rotary_dim / 2]) of a head turn by the angle p inv_freq[i]: (u cos - v sin, v cos + u sin), times a.scale; the
// rest of a head stays.  A thread takes four pairs, so that what it holds lies in two runs of four values, eight lanes to 32 values: the groups of
// the 8-bit cache.  The angle is taken in turns, of which the fraction alone goes to fp32; cosines and sines are made once a token, in LDS.  Keys for an 8-bit cache turn in fp64 and are rounded once, so that a key next to the
// middle of two codes goes where the formula puts it.  Bound by HBM: 20 KiB in and 13 out for a token of 64 + 2 * 8 heads of 64; 8192 of them with packed
// rows 51 us, 5.3 TB/s, what a copy reaches.
template <int D, bool BF16, bool MX>
__global__ __launch_bounds__(256) void rope_kv_kernel(RopeKvArgs a, int tokens_per_block) {
    using Turn = std::conditional_t<MX, double2, float2>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Turn* turn = reinterpret_cast<Turn*>(lds);  // [tokens_per_block][rotary_dim / 2]: cosine, sine
    const int R = a.rotary_dim, half = R / 2;
    const int token0 = blockIdx.x * tokens_per_block, tokens = min(tokens_per_block, a.n_tokens - token0);
    for (int i = threadIdx.x; i < tokens * half; i += 256) {
        const double turns = part_of_turn((double)a.positions[token0 + i / half], (double)a.inv_freq[i % half]);
        decltype(Turn::x) sine, cosine;
        if constexpr (MX) sincospi(2.0 * turns, &sine, &cosine);
        else sincospif(2.f * (float)turns, &sine, &cosine);
        turn[i].x = cosine * a.scale;
        turn[i].y = sine * a.scale;
    }
    __syncthreads();
    const int heads = a.n_heads + 2 * a.n_kv_heads, units = heads * (D / 8);
    for (int i = threadIdx.x; i < tokens * units; i += 256) {
        const int t = i / units, unit = i - t * units, head = unit / (D / 8), w = unit % (D / 8);
        const bool turns = w < R / 8;
        const int lo = turns ? 4 * w : R + 4 * (w - R / 8), hi = turns ? lo + half : lo + (D - R) / 2;
        const size_t at = (size_t)(token0 + t) * a.stride + (size_t)head * D;
        float x[4], y[4];
        if constexpr (BF16) {
            const uint16_t* row = static_cast<const uint16_t*>(a.rows) + at;
            const u32x2 u = *reinterpret_cast<const u32x2*>(row + lo), v = *reinterpret_cast<const u32x2*>(row + hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = bf16_bits_to_f32(u[j / 2] >> (j % 2 * 16) & 0xFFFFu);
                y[j] = bf16_bits_to_f32(v[j / 2] >> (j % 2 * 16) & 0xFFFFu);
            }
        } else {
            const float* row = static_cast<const float*>(a.rows) + at;
            const f32x4 u = *reinterpret_cast<const f32x4*>(row + lo), v = *reinterpret_cast<const f32x4*>(row + hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = u[j];
                y[j] = v[j];
            }
        }
        if (turns && head < a.n_heads + a.n_kv_heads) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Turn cs = turn[t * half + lo + j];
                if (MX && head >= a.n_heads) {
                    const double u = x[j], v = y[j];
                    x[j] = to_odd(u * cs.x - v * cs.y);
                    y[j] = to_odd(v * cs.x + u * cs.y);
                } else {
                    const float u = x[j], v = y[j], c = (float)cs.x, s = (float)cs.y;
                    x[j] = u * c - v * s;
                    y[j] = v * c + u * s;
                }
            }
        }
        const u32x2 xb = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])}, yb = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        const int token = token0 + t;
        if (head < a.n_heads) {
            if (!a.q) continue;
            uint16_t* q = a.q + ((size_t)token * a.n_heads + head) * D;
            *reinterpret_cast<u32x2*>(q + lo) = xb;
            *reinterpret_cast<u32x2*>(q + hi) = yb;
            continue;
        }
        const bool is_v = head >= a.n_heads + a.n_kv_heads;
        const int h = head - a.n_heads - (is_v ? a.n_kv_heads : 0);
        if (uint16_t* rows = is_v ? a.v : a.k) {
            uint16_t* r = rows + ((size_t)token * a.n_kv_heads + h) * D;
            *reinterpret_cast<u32x2*>(r + lo) = xb;
            *reinterpret_cast<u32x2*>(r + hi) = yb;
        }
        if (!a.cache_k) continue;
        const int slot = a.slots[token];
        if (slot < 0 || slot >= a.n_slots) continue;
        const size_t row = ((size_t)(slot >> a.page_shift) * a.n_kv_heads + h) << a.page_shift | (size_t)(slot & ((1 << a.page_shift) - 1));
        uint8_t* cache = is_v ? a.cache_v : a.cache_k;
        if constexpr (MX) {
            uint8_t* scales = (is_v ? a.v_scales : a.k_scales) + row * (D / 32);
            auto put = [&](const float (&f)[4], int d) {
                const uint32_t b = mx_scale_byte(group_max<8>(max(max(abs_bits(f[0]), abs_bits(f[1])), max(abs_bits(f[2]), abs_bits(f[3])))));
                const float s = __uint_as_float(b == 255u ? 0x7FC00000u : (254u - b) << 23);  // 2^(127 - b): the products are exact
                int codes = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * s, f[1] * s, 0, false);
                codes = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * s, f[3] * s, codes, true);
                *reinterpret_cast<int*>(cache + row * D + d) = codes;
                if ((w & 7) == 0) scales[d / 32] = (uint8_t)b;
            };
            put(x, lo);
            put(y, hi);
        } else {
            *reinterpret_cast<u32x2*>(cache + (row * D + lo) * 2) = xb;
            *reinterpret_cast<u32x2*>(cache + (row * D + hi) * 2) = yb;
        }
    }
}

int launch_rope_kv_write(const RopeKvArgs& a, bool bf16_rows, hipStream_t stream) {
    const int units = (a.n_heads + 2 * a.n_kv_heads) * (a.head_dim / 8);
    const int per_block = std::max(1, std::min(8, 512 / units));
    const size_t lds = (size_t)per_block * (a.rotary_dim / 2) * (a.k_scales ? sizeof(double2) : sizeof(float2));
    const long long at_once = kMostThreads / 256 * per_block;
    auto run = [&](auto kernel) {
        for (long long token = 0; token < a.n_tokens; token += at_once) {
            RopeKvArgs b = a;
            b.n_tokens = (int)std::min(a.n_tokens - token, at_once);
            b.rows = static_cast<const char*>(a.rows) + token * a.stride * (bf16_rows ? 2 : 4);
            if (a.positions) b.positions += token;
            if (a.slots) b.slots += token;
            if (a.q) b.q += token * a.n_heads * a.head_dim;
            if (a.k) b.k += token * a.n_kv_heads * a.head_dim;
            if (a.v) b.v += token * a.n_kv_heads * a.head_dim;
            hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(b.n_tokens, per_block)), dim3(256), lds, stream, b, per_block);
            const int rc = launch_status();
            if (rc) return rc;
        }
        return (int)MOE_OK;
    };
    auto of_cache = [&](auto plain, auto mx) { return a.k_scales ? run(mx) : run(plain); };
    if (a.head_dim == 64)
        return bf16_rows ? of_cache(rope_kv_kernel<64, true, false>, rope_kv_kernel<64, true, true>)
                         : of_cache(rope_kv_kernel<64, false, false>, rope_kv_kernel<64, false, true>);
    return bf16_rows ? of_cache(rope_kv_kernel<128, true, false>, rope_kv_kernel<128, true, true>)
                     : of_cache(rope_kv_kernel<128, false, false>, rope_kv_kernel<128, false, true>);
}

}  // namespace moe
