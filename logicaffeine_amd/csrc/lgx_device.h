// lgx_device.h -- device code that several of the kernel files use: vector types,
// conversions, moves and reductions between lanes, direct loads into LDS.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lgx_kargs.h"

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float h2f(uint32_t h) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

__device__ __forceinline__ uint16_t f2h(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}

__device__ __forceinline__ int shfl_xor_i(int v, int m) { return __shfl_xor(v, m, 64); }
__device__ __forceinline__ float shfl_xor_f(float v, int m) { return __shfl_xor(v, m, 64); }

// DPP lane moves for the wave reductions (VALU operations, where a shuffle
// is an LDS round trip): quad_perm [1,0,3,2] (0xB1) and [2,3,0,1] (0x4E),
// row_half_mirror (0x141: lane i <- 7 - i of its 8), row_mirror (0x140:
// lane i <- 15 - i of its 16), row_shl:S (0x100 + S: lane i <- lane i + S of
// its 16-lane row).  A lane without a source keeps its own value.
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
    const int x = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false));
}
// Maximum over each aligned group of 8 lanes, in every lane of the group
// (fmaxf is order-free, so any pairing gives the same value).
__device__ __forceinline__ float max8(float m) {
    m = fmaxf(m, dpp_f<0xB1>(m));
    m = fmaxf(m, dpp_f<0x4E>(m));
    return fmaxf(m, dpp_f<0x141>(m));
}
// Maximum over the wave, in every lane.
__device__ __forceinline__ float wave_max(float m) {
    m = max8(m);
    m = fmaxf(m, dpp_f<0x140>(m));
    m = fmaxf(m, shfl_xor_f(m, 16));
    return fmaxf(m, shfl_xor_f(m, 32));
}
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v8h as_v8h(uint4 u) { return __builtin_bit_cast(v8h, u); }

typedef __attribute__((address_space(3))) void lds_void;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// Direct global->LDS loads (a wave instruction's 64 pieces of 16 or 4 bytes
// land one after the other at l, which is uniform) that the compiler does not
// count: it makes every LDS read of a loop wait for those it knows, whichever
// buffer they fill.  They write no register; publish_lds_loads waits for them.
__device__ __forceinline__ void load_lds_16(const void* g, lds_void* l) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 : : "s"((uint32_t)(uintptr_t)l), "v"(g) : "memory", "m0");
}
__device__ __forceinline__ void load_lds_4(const void* g, lds_void* l) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 : : "s"((uint32_t)(uintptr_t)l), "v"(g) : "memory", "m0");
}
// Barrier that publishes this wave's direct global->LDS loads to the
// workgroup.  The wait is written out: the compiler waits for such a load
// where its own wave reads the data, which in a loop may be only after the
// barrier, when the other waves already read.
__device__ __forceinline__ void publish_lds_loads() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Two numbers rounded to binary16 (v_cvt_pk_f16_f32).
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){lo, hi}, v2h));
}

// w minus the low or high half of a pair of binary16 numbers, exact.  (Neither
// operand may come from a matrix instruction or a v_exp: the compiler puts no wait
// states ahead of assembly.)
template <int HI>
__device__ __forceinline__ float minus_half(float w, uint32_t pair) {
    float r;
    if (HI) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pair), "v"(w));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pair), "v"(w));
    return r;
}

// tanh: below 0.35 the odd series (the term after the last is under 1.3e-8 of
// the result), else (1 - t) / (1 + t), t = exp(-2 |x|), where 1 - t > 0.5.
__device__ __forceinline__ float a8_tanh(float x) {
    const float ax = fabsf(x), t = __builtin_amdgcn_exp2f(-2.8853900817779268f * ax);
    const float big = copysignf((1.0f - t) / (1.0f + t), x);
    const float y = x * x;
    float p = fmaf(y, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(y, p, -17.0f / 315.0f);
    p = fmaf(y, p, 2.0f / 15.0f);
    p = fmaf(y, p, -1.0f / 3.0f);
    return ax < 0.35f ? fmaf(x * y, p, x) : big;
}

// Joins over the four lanes of a column: the swaps leave a row of 16 lanes beside
// its neighbour's, then half a wave beside the other.
__device__ __forceinline__ float col_join16(float v, float& other) {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    const unsigned x = __float_as_uint(v);
    const v2u r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    other = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}
__device__ __forceinline__ float col_join32(float v, float& other) {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    const unsigned x = __float_as_uint(v);
    const v2u r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    other = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}
__device__ __forceinline__ float col_max(float v) {
    float w;
    v = col_join16(v, w);
    v = fmaxf(v, w);
    v = col_join32(v, w);
    return fmaxf(v, w);
}
__device__ __forceinline__ float col_sum(float v) {
    float w;
    v = col_join16(v, w);
    v = v + w;
    v = col_join32(v, w);
    return v + w;
}

// Inclusive sums over the wave's lanes (VALU moves within rows of 16, then of row
// 0 and 2's last lane into the next row, then of the lower half's into the upper).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
