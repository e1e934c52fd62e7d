// What the attention kernels share: matrix operands through LDS, the running softmax's exchanges, the search for a block's sequence.
#pragma once
#include "common.h"

namespace moe {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr float kLog2e = 1.44269504088896340736f;

// D(32x32) += A(32x16) * B(16x32); lane l holds A[row l%32][8*(l/32) .. +8), B[.. same k ..][col l%32],
// D[rows 8*i + 4*(l/32) .. +4][col l%32] in elements 4*i .. 4*i+3.
MOE_DEVICE f32x16 mfma_32x32x16(const u32x4& a, const u32x4& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// To stand between matrix instructions and a branch behind which their results are read.  The hardware does not wait for a matrix instruction whose
// result another one reads; the compiler's wait goes by the longest way round an `if` between the two, so that the short way reads old values.
// Twelve states: one more than an instruction of eight passes needs.
template <class T>
MOE_DEVICE void settle(T& x) {
    asm volatile("s_nop 11" : "+v"(x));
}
template <class T>
MOE_DEVICE void settle(T& x, T& y) {
    asm volatile("s_nop 11" : "+v"(x), "+v"(y));
}

// Four 16-bit values of a column: in each 16 lanes, lane i names 8 bytes of row i/4 (its columns 4*(i%4) .. +4) and gets column i of the four rows.
MOE_DEVICE u32x2 lds_column_of_4(const void* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// Where 16-byte chunk c of row r of a tile of keys or values (2 D bytes a row) lies within its row in LDS: an exclusive or that gives 8 and 16 rows which are
// read side by side, the same chunk of each, banks of their own (keys), and two or four neighbouring chunks of 4 rows (values, read by columns).
template <int D>
MOE_DEVICE int k_chunk(int r, int c) {
    return c ^ (D == 64 ? (r & 7) ^ ((r >> 3) & 1) : r & 15);
}
template <int D>
MOE_DEVICE int v_chunk(int r, int c) {
    return c ^ (D == 64 ? (r & 3) << 1 : (r & 3) << 2 | (r & 2));
}

// Maximum or sum over the lanes that differ in bits 4 and 5 only (the four groups of 16), in all of them.
MOE_DEVICE float max_of_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
MOE_DEVICE float sum_of_halves(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
MOE_DEVICE float max_of_halves(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
MOE_DEVICE float sum_of_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_of_halves(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// Inclusive prefix sum over the lanes of a wave.
MOE_DEVICE int wave_prefix_sum(int v) {
#define MOE_STEP(C, M) v += (int)dpp_move<C, M>(0u, (uint32_t)v);
    MOE_DPP_STEPS(MOE_STEP)
#undef MOE_STEP
    return v;
}

// Sequences 0 .. n-1 have count(s) items each, numbered through: item j's sequence and its number within it.  False past the last.  All of a
// wave's lanes ask for the same j; 64 sequences at a time, a lane to each.
template <class F>
MOE_DEVICE bool find_item(int n, int j, F count, int& seq, int& within) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < n; base += 64) {
        const int c = base + lane < n ? count(base + lane) : 0;
        const int upto = wave_prefix_sum(c);
        const uint64_t past = __ballot(before + upto > j);
        if (past) {
            const int at = __builtin_ctzll(past);
            seq = base + at;
            within = j - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(c, at));
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// The same from the last item backwards: item j of the reversed order.
template <class F>
MOE_DEVICE bool find_last_item(int n, int j, F count, int& seq, int& within) {
    const int lane = threadIdx.x & 63;
    if (n <= 64) {  // one look at the counts
        const int c = lane < n ? count(lane) : 0, upto = wave_prefix_sum(c), at = __builtin_amdgcn_readlane(upto, 63) - 1 - j;
        const uint64_t past = __ballot(upto > at);
        if (at < 0) return false;
        seq = __builtin_ctzll(past);
        within = at - (__builtin_amdgcn_readlane(upto, seq) - __builtin_amdgcn_readlane(c, seq));
        return true;
    }
    int all = 0;
    for (int base = 0; base < n; base += 64) all += wave_sum(base + lane < n ? count(base + lane) : 0);
    return j < all && find_item(n, all - 1 - j, count, seq, within);
}

}  // namespace moe
