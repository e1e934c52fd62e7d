// RMSNorm of src/run.cpp:306-319 with the reference CPU's mixed precision: fp32 squares summed in
// fp64, sqrtf and the reciprocal in fp32, the scaling in fp64, one rounding to fp32 at the end.
// A row is owned by one block of 256 threads; thread i holds float4 columns i, i + 256, ... and adds
// their squares in ascending order, the fp64 sum over the block is a fixed tree over each wave and then the waves in order: results
// are run-to-run identical, and identical between the plain kernel, the one fused into the combine and, for rows of up to 4096 values, the
// one with the residual add (longer rows take more threads there, so another order of the fp64 sum).
#pragma once
#include "common.h"

namespace moe {
namespace {

MOE_DEVICE double sumsq(double ss, const float4& v) {
    ss += (double)__fmul_rn(v.x, v.x);
    ss += (double)__fmul_rn(v.y, v.y);
    ss += (double)__fmul_rn(v.z, v.z);
    ss += (double)__fmul_rn(v.w, v.w);
    return ss;
}

MOE_DEVICE double inv_rms(double sum, int size, float eps) {
    double m = sum / size;
    m += (double)eps;
    return (double)(1.0f / sqrtf((float)m));
}

// WAVES waves to the block; red: a value per wave.
template <int WAVES = 4>
MOE_DEVICE double block_inv_rms(double ss, double* red, int size, float eps = 1e-5f) {
    const int wave0 = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u);
    const double sum = 4 * wave0 < size ? wave_sum(ss) : 0.0;  // short rows: waves without a value (8192 x 64 7.6 : 4.5 us)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    double total = red[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) total += red[w];
    return inv_rms(total, size, eps);
}

// Four values before their rounding to fp32; wb: their weights (bf16).
struct Double4 {
    double x, y, z, w;
};
MOE_DEVICE Double4 norm_products(const float4& v, uint2 wb, double inv) {
    return {(double)bf16_bits_to_f32(wb.x & 0xFFFFu) * (inv * (double)v.x), (double)bf16_bits_to_f32(wb.x >> 16) * (inv * (double)v.y),
            (double)bf16_bits_to_f32(wb.y & 0xFFFFu) * (inv * (double)v.z), (double)bf16_bits_to_f32(wb.y >> 16) * (inv * (double)v.w)};
}
MOE_DEVICE float4 to_float4(const Double4& d) { return make_float4((float)d.x, (float)d.y, (float)d.z, (float)d.w); }

MOE_DEVICE float4 norm_scale(const float4& v, const uint16_t* __restrict__ weight, int c, double inv) {
    return to_float4(norm_products(v, *reinterpret_cast<const uint2*>(weight + 4 * c), inv));
}

}  // namespace
}  // namespace moe
