// Wave and workgroup helpers of the kernels that are compiled without packed fp32 instructions (pk_opsel_fix.py says what is wrong with
// those; newer kernels leave them out altogether).  A function without that restriction is not inlined into one that has it unless it is
// marked always_inline, which the runtime's __shfl_xor, __syncthreads and __float_as_uint are not: these take their place.
#pragma once
#include "nfe_common.h"

#if defined(__HIP_DEVICE_COMPILE__)
#define NFE_NO_PACKED_FP32_BEGIN _Pragma("clang attribute push(__attribute__((target(\"no-packed-fp32-ops\"))), apply_to = function)")
#define NFE_NO_PACKED_FP32_END _Pragma("clang attribute pop")
#else
#define NFE_NO_PACKED_FP32_BEGIN
#define NFE_NO_PACKED_FP32_END
#endif

NFE_NO_PACKED_FP32_BEGIN
namespace nfe {
__device__ __forceinline__ unsigned bits_of(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float float_of(unsigned b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ int wave_lane() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }
// the value of lane (own ^ off); every lane of the wave has to take part
__device__ __forceinline__ unsigned wave_xor(unsigned v, int off) { return (unsigned)__builtin_amdgcn_ds_bpermute((wave_lane() ^ off) << 2, (int)v); }
__device__ __forceinline__ double wave_xor(double v, int off) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = wave_xor((unsigned)b, off), hi = wave_xor((unsigned)(b >> 32), off);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
// The same without LDS: DPP inside a row of 16 lanes, lane-row swaps beyond.  Every lane gets the result.
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned row_max(unsigned v) {              // maximum over the 16 lanes of a row
    v = umax(v, dpp<DPP_XOR1>(v));
    v = umax(v, dpp<DPP_XOR2>(v));
    v = umax(v, dpp<DPP_HALF_MIRROR>(v));
    return umax(v, dpp<DPP_MIRROR>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += float_of(dpp<DPP_XOR1>(bits_of(v)));
    v += float_of(dpp<DPP_XOR2>(bits_of(v)));
    v += float_of(dpp<DPP_HALF_MIRROR>(bits_of(v)));
    v += float_of(dpp<DPP_MIRROR>(bits_of(v)));
    const auto a = __builtin_amdgcn_permlane16_swap(bits_of(v), bits_of(v), false, false);      // (rows 0 0 2 2, rows 1 1 3 3)
    v = float_of(a[0]) + float_of(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(bits_of(v), bits_of(v), false, false);      // (lower half twice, upper half twice)
    return float_of(b[0]) + float_of(b[1]);
}
// LDS accesses of one wave: those before it come first, for every lane.  An order for the compiler, no instruction.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ void block_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}
}  // namespace nfe
NFE_NO_PACKED_FP32_END
