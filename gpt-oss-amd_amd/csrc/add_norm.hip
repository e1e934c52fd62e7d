// Residual add, RMSNorm and its result in the type the next product reads: fp32, bf16, or e4m3 with scales.
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "norm.h"

namespace moe {

namespace {

MOE_DEVICE uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Bits of the largest |value| (those of an infinity or a NaN are above all others).
MOE_DEVICE uint32_t amax_bits(const float4& y) {
    return max(max(abs_bits(y.x), abs_bits(y.y)), max(abs_bits(y.z), abs_bits(y.w)));
}

// Maximum over the 8 (group of 32 values) or 32 lanes (group of 128) that hold a group.
template <int LANES>
MOE_DEVICE uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

// Power-of-two scale of a group (e8m0): the smallest 2^(b - 127), b >= 1, that brings its largest value to 448 or below.  448 = 1.75 * 2^8, so
// the exponent field goes up by one where the mantissa is past 1.75.  255 where the group holds an infinity or a NaN.
MOE_DEVICE uint32_t mx_scale_byte(uint32_t amax) {
    if (amax >= 0x7F800000u) return 255u;
    const int b = (int)((amax + 0x1FFFFFu) >> 23) - 8;
    return (uint32_t)max(b, 1);
}

// fp32 scale of a group, and what its values are multiplied by.
MOE_DEVICE void f32_scale(uint32_t amax, float& scale, float& mult) {
    if (amax >= 0x7F800000u) {
        scale = mult = NAN;
        return;
    }
    const float a = fmaxf(__uint_as_float(amax), 0x1p-100f);  // the quotients stay normal numbers
    scale = a / 448.0f;
    mult = 448.0f / a;
}

MOE_DEVICE uint32_t to_e4m3x4(const float4& y, float mult) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y.x * mult, y.y * mult, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(y.z * mult, y.w * mult, v, true);
    return (uint32_t)v;
}

MOE_DEVICE float4 add4(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

}  // namespace

// A block of 256 threads per row; thread i holds float4 columns i, i + 256, ...: NI of them in registers, or with NI = 0 any number,
// read again from x_out.  Q: what is written of the result besides fp32 (a.o) and bf16 (a.o_bf16) rows: e4m3 with a scale per 32 values
// (e8m0) or per 128 (fp32), which lanes of one wave hold, or per row (fp32), which takes another exchange through LDS; -1 none.
template <int NI, int Q>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(AddNormArgs a) {
    __shared__ double red[4];
    __shared__ uint32_t row_amax[4];
    const int H4 = a.size >> 2;
    const size_t row = (size_t)blockIdx.x * H4;
    const float4* x = reinterpret_cast<const float4*>(a.x) + row;
    const float4* d = a.delta ? reinterpret_cast<const float4*>(a.delta) + row : nullptr;
    float4* x_out = reinterpret_cast<float4*>(a.x_out) + row;
    const int n_cols = ceil_div(H4, 256);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v[NI > 0 ? NI : 1];
    double ss = 0.0;
    auto load = [&](int c) {
        float4 r = c < H4 ? x[c] : zero;
        if (d && c < H4) r = add4(r, d[c]);
        return r;
    };
    if constexpr (NI > 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) v[i] = load(threadIdx.x + 256 * i);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = threadIdx.x + 256 * i;
            if (c < H4) x_out[c] = v[i];
            ss = sumsq(ss, v[i]);
        }
    } else {
        for (int i = 0; i < n_cols; ++i) {
            const int c = threadIdx.x + 256 * i;
            const float4 r = load(c);
            if (c < H4) x_out[c] = r;
            ss = sumsq(ss, r);
        }
    }
    const double inv = block_inv_rms(ss, red, a.size, a.eps);
    auto result = [&](int i) {
        const int c = threadIdx.x + 256 * i;
        if (c >= H4) return zero;
        if constexpr (NI > 0) return norm_scale(v[i], a.weight, c, inv);
        else return norm_scale(x_out[c], a.weight, c, inv);
    };
    float mult = 1.0f;
    if constexpr (Q == 0) {
        uint32_t m = 0;
        if constexpr (NI > 0) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                v[i] = result(i);
                m = max(m, amax_bits(v[i]));
            }
        } else {
            for (int i = 0; i < n_cols; ++i) m = max(m, amax_bits(result(i)));
        }
        m = group_max<64>(m);
        if ((threadIdx.x & 63) == 0) row_amax[threadIdx.x >> 6] = m;
        __syncthreads();
        m = max(max(row_amax[0], row_amax[1]), max(row_amax[2], row_amax[3]));
        float scale;
        f32_scale(m, scale, mult);
        if (threadIdx.x == 0) reinterpret_cast<float*>(a.q_scales)[blockIdx.x] = scale;
    }
    auto store = [&](int i, const float4& y) {
        const int c = threadIdx.x + 256 * i;
        if (a.o && c < H4) reinterpret_cast<float4*>(a.o)[row + c] = y;
        if (a.o_bf16 && c < H4) reinterpret_cast<uint2*>(a.o_bf16)[row + c] = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
        if constexpr (Q >= 0) {
            float m = mult;
            if constexpr (Q == 32) {
                const uint32_t b = mx_scale_byte(group_max<8>(amax_bits(y)));
                m = b == 255u ? NAN : __uint_as_float((254u - b) << 23);
                if (c < H4 && (c & 7) == 0) a.q_scales[(row + c) >> 3] = (uint8_t)b;
            } else if constexpr (Q == 128) {
                float scale;
                f32_scale(group_max<32>(amax_bits(y)), scale, m);
                if (c < H4 && (c & 31) == 0)
                    reinterpret_cast<float*>(a.q_scales)[(size_t)blockIdx.x * ceil_div(H4, 32) + (c >> 5)] = scale;
            }
            if (c < H4) reinterpret_cast<uint32_t*>(a.q)[row + c] = to_e4m3x4(y, m);
        }
    };
    if constexpr (NI > 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) store(i, Q == 0 ? v[i] : result(i));
    } else {
        for (int i = 0; i < n_cols; ++i) store(i, result(i));
    }
}

int launch_add_rmsnorm(const AddNormArgs& a, int batch, hipStream_t stream) {
    auto of_q = [&](auto q) {
        constexpr int Q = decltype(q)::value;
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(batch), dim3(256), 0, stream, a);
            return launch_status();
        };
        if (a.size <= 1024) return launch(add_rmsnorm_kernel<1, Q>);
        if (a.size <= 3072) return launch(add_rmsnorm_kernel<3, Q>);
        return launch(add_rmsnorm_kernel<0, Q>);
    };
    if (!a.q) return of_q(std::integral_constant<int, -1>{});
    if (a.q_group == 32) return of_q(std::integral_constant<int, 32>{});
    if (a.q_group == 128) return of_q(std::integral_constant<int, 128>{});
    return of_q(std::integral_constant<int, 0>{});
}

}  // namespace moe
