// Residual add, RMSNorm and its result in the type the next product reads: fp32, bf16, or e4m3 with scales.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "mx8.h"
#include "norm.h"

namespace moe {

// group_max of doubles that are not negative and not NaN: their bits are in their order.
template <int LANES>
MOE_DEVICE double group_max(double v) {
    const uint32_t hi = (uint32_t)(__builtin_bit_cast(uint64_t, v) >> 32), lo = (uint32_t)__builtin_bit_cast(uint64_t, v);
    const uint32_t most = group_max<LANES>(hi);
    const uint32_t rest = group_max<LANES>(hi == most ? lo : 0u);
    return __builtin_bit_cast(double, ((uint64_t)most << 32) | rest);
}

namespace {

// Bits of the largest |value| (those of an infinity or a NaN are above all others).
MOE_DEVICE uint32_t amax_bits(const float4& y) {
    return max(max(abs_bits(y.x), abs_bits(y.y)), max(abs_bits(y.z), abs_bits(y.w)));
}
// The largest |value| before the rounding to fp32; what is not finite the bits above tell.
MOE_DEVICE double amax_of(const Double4& y) { return fmax(fmax(fabs(y.x), fabs(y.y)), fmax(fabs(y.z), fabs(y.w))); }

// fp32 scale of a group of largest |value| amax (bits: in fp32), and what its values are multiplied by: 448 / amax to 2^-48.
MOE_DEVICE void f32_scale(uint32_t bits, double amax, float& scale, double& mult) {
    if (bits >= 0x7F800000u) {
        scale = NAN;
        mult = (double)NAN;
        return;
    }
    const double a = fmax(amax, 0x1p-100);  // the quotients stay normal numbers
    scale = (float)a / 448.0f;
    const double r = __builtin_amdgcn_rcp(a);
    mult = 448.0 * fma(fma(-a, r, 1.0), r, r);
}

MOE_DEVICE uint32_t to_e4m3x4(const Double4& y, double mult) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(to_odd(y.x * mult), to_odd(y.y * mult), 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(to_odd(y.z * mult), to_odd(y.w * mult), v, true);
    return (uint32_t)v;
}

MOE_DEVICE float4 add4(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

}  // namespace

// THREADS to a row, a block of 256 or more to one or four; thread i holds float4 columns i, i + THREADS, ...: NI of them, with their weights, in
// registers, or with NI = 0 any number, read again from x_out.  Up to 256 threads the squares are added up in the order of rmsnorm_kernel: 64 at a
// time, then those sums in order.  Q: what is written of the result besides fp32 (a.o) and bf16 (a.o_bf16) rows: e4m3 with a scale per 32 values
// (e8m0) or per 128 (fp32), which lanes of one wave hold, or per row (fp32), which takes another exchange through LDS; -1 none.
template <int THREADS, int NI, int Q, bool NT>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void add_rmsnorm_kernel(AddNormArgs a, int batch) {
    constexpr int kWaves = THREADS / 64;
    constexpr bool kWaveRow = kWaves == 1;  // a row is a wave's own: nothing is exchanged through LDS
    const int at_row = kWaveRow ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    const int tid = kWaveRow ? threadIdx.x & 63 : threadIdx.x;
    if (kWaveRow && at_row >= batch) return;
    __shared__ double red[kWaves], row_amax[kWaves];
    __shared__ uint32_t row_bits[kWaves];
    const int H4 = a.size >> 2;
    const size_t row = (size_t)at_row * H4;
    const float4* x = reinterpret_cast<const float4*>(a.x) + row;
    const float4* d = a.delta ? reinterpret_cast<const float4*>(a.delta) + row : nullptr;
    const uint2* weight = reinterpret_cast<const uint2*>(a.weight);
    float4* x_out = reinterpret_cast<float4*>(a.x_out) + row;
    const int n_cols = ceil_div(H4, THREADS);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v[NI > 0 ? NI : 1];
    uint2 wb[NI > 0 ? NI : 1];
    double ss = 0.0;
    if constexpr (NI > 0) {
        float4 dv[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = tid + THREADS * i;
            v[i] = c < H4 ? load_value<NT>(x + c) : zero;
        }
        if (d) {  // uniform
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = tid + THREADS * i;
                dv[i] = c < H4 ? load_value<NT>(d + c) : zero;
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = tid + THREADS * i;
            wb[i] = c < H4 ? weight[c] : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = tid + THREADS * i;
            if (d) v[i] = add4(v[i], dv[i]);
            if (c < H4) store_value<NT>(x_out + c, v[i]);
            if constexpr (kWaveRow) ss += wave_sum(sumsq(0.0, v[i]));
            else ss = sumsq(ss, v[i]);
        }
    } else {
        for (int i = 0; i < n_cols; ++i) {
            const int c = tid + THREADS * i;
            float4 r = c < H4 ? x[c] : zero;
            if (d && c < H4) r = add4(r, d[c]);
            if (c < H4) x_out[c] = r;
            ss = sumsq(ss, r);
        }
    }
    double inv;
    if constexpr (kWaveRow) inv = inv_rms(ss, a.size, a.eps);
    else inv = block_inv_rms<kWaves>(ss, red, a.size, a.eps);
    auto result = [&](int i) {
        const int c = tid + THREADS * i;
        if constexpr (NI > 0) return norm_products(v[i], wb[i], inv);
        else return c < H4 ? norm_products(x_out[c], weight[c], inv) : Double4{0.0, 0.0, 0.0, 0.0};
    };
    double mult = 1.0;
    if constexpr (Q == 0) {
        uint32_t bits = 0;
        double most = 0.0;
        auto largest = [&](int i) {
            const Double4 y = result(i);
            bits = max(bits, amax_bits(to_float4(y)));
            most = fmax(most, amax_of(y));
        };
        if constexpr (NI > 0) {
#pragma unroll
            for (int i = 0; i < NI; ++i) largest(i);
        } else {
            for (int i = 0; i < n_cols; ++i) largest(i);
        }
        bits = group_max<64>(bits);
        most = group_max<64>(most);
        if constexpr (!kWaveRow) {
            if ((threadIdx.x & 63) == 0) {
                row_bits[threadIdx.x >> 6] = bits;
                row_amax[threadIdx.x >> 6] = most;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                bits = max(bits, row_bits[w]);
                most = fmax(most, row_amax[w]);
            }
        }
        float scale;
        f32_scale(bits, most, scale, mult);
        if (tid == 0) reinterpret_cast<float*>(a.q_scales)[at_row] = scale;
    }
    auto store = [&](int i) {
        const int c = tid + THREADS * i;
        const Double4 y = result(i);
        const float4 f = to_float4(y);
        if (a.o && c < H4) reinterpret_cast<float4*>(a.o)[row + c] = f;
        if (a.o_bf16 && c < H4) reinterpret_cast<uint2*>(a.o_bf16)[row + c] = make_uint2(pack_bf16x2(f.x, f.y), pack_bf16x2(f.z, f.w));
        if constexpr (Q >= 0) {
            double m = mult;
            if constexpr (Q == 32) {
                const uint32_t b = mx_scale_byte(group_max<8>(amax_bits(f)));
                m = b == 255u ? (double)NAN : (double)__uint_as_float((254u - b) << 23);
                if (c < H4 && (c & 7) == 0) a.q_scales[(row + c) >> 3] = (uint8_t)b;
            } else if constexpr (Q == 128) {
                float scale;
                f32_scale(group_max<32>(amax_bits(f)), group_max<32>(amax_of(y)), scale, m);
                if (c < H4 && (c & 31) == 0)
                    reinterpret_cast<float*>(a.q_scales)[(size_t)at_row * ceil_div(H4, 32) + (c >> 5)] = scale;
            }
            if (c < H4) reinterpret_cast<uint32_t*>(a.q)[row + c] = to_e4m3x4(y, m);
        }
    };
    if constexpr (NI > 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) store(i);
    } else {
        for (int i = 0; i < n_cols; ++i) store(i);
    }
}

// Whether x, delta and x_out are more than the 256 MiB of the last-level cache; they are then read and written past it.  us without : with,
// rows of 2880, out of cache: 16384 of them, scales per 128 108.7 : 95.7 (6.4 TB/s), bf16 116.2 : 98.2; 8192 of 4096 79.3 : 68.9; but 4096
// (142 MB) 27.4 : 28.3 and 1000 in bf16 9.0 : 9.5.
static bool past_cache(const AddNormArgs& a, int batch) { return (long long)batch * a.size * (a.delta ? 12 : 8) > (256ll << 20); }

// The arguments for the rows from `row` on.
static AddNormArgs rows_from(AddNormArgs a, long long row) {
    const long long at = row * a.size;
    a.x_out += at;
    a.x += at;
    if (a.delta) a.delta += at;
    if (a.o) a.o += at;
    if (a.o_bf16) a.o_bf16 += at;
    if (a.q) {
        a.q += at;
        a.q_scales += row * (a.q_group == MOE_Q_GROUP_MX ? a.size / 32 : a.q_group == MOE_Q_GROUP_128 ? 4 * ((a.size - 1) / 128 + 1) : 4);
    }
    return a;
}

// Threads to a row by its length: 64 up to 1024 values (16384 rows of 64 9.3 us, with 256 18.1), 256 up to 4096, 512 up to 8192 (64 rows of 8192 5.2 us,
// with 256 and no values in registers 8.3; 5000 rows 85 : 112), 1024 past that.
int launch_add_rmsnorm(const AddNormArgs& a, int batch, hipStream_t stream) {
    auto of = [&](auto q, auto nt) {
        constexpr int Q = decltype(q)::value;
        constexpr bool NT = decltype(nt)::value;
        auto launch = [&](auto kernel, int threads) {
            const int rows = threads < 256 ? 256 / threads : 1;
            const long long most = kMostThreads / threads;
            for (long long row = 0; row < batch; row += most) {
                const int n = (int)std::min(batch - row, most);
                hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(n, rows)), dim3(threads * rows), 0, stream, rows_from(a, row), n);
                const int rc = launch_status();
                if (rc) return rc;
            }
            return (int)MOE_OK;
        };
        if (a.size <= 256) return launch(add_rmsnorm_kernel<64, 1, Q, NT>, 64);
        if (a.size <= 512) return launch(add_rmsnorm_kernel<64, 2, Q, NT>, 64);
        if (a.size <= 1024) return launch(add_rmsnorm_kernel<64, 4, Q, NT>, 64);
        if (a.size <= 2048) return launch(add_rmsnorm_kernel<256, 2, Q, NT>, 256);
        if (a.size <= 3 * 1024) return launch(add_rmsnorm_kernel<256, 3, Q, NT>, 256);
        if (a.size <= 4096) return launch(add_rmsnorm_kernel<256, 4, Q, NT>, 256);
        if (a.size <= 8192) return launch(add_rmsnorm_kernel<512, 4, Q, NT>, 512);
        if (a.size <= 16384) return launch(add_rmsnorm_kernel<1024, 4, Q, NT>, 1024);
        return launch(add_rmsnorm_kernel<1024, 0, Q, false>, 1024);
    };
    auto of_q = [&](auto q) { return past_cache(a, batch) ? of(q, std::true_type{}) : of(q, std::false_type{}); };
    if (!a.q) return of_q(std::integral_constant<int, -1>{});
    if (a.q_group == 32) return of_q(std::integral_constant<int, 32>{});
    if (a.q_group == 128) return of_q(std::integral_constant<int, 128>{});
    return of_q(std::integral_constant<int, 0>{});
}

}  // namespace moe
