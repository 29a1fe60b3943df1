// 8-bit dense operators (e4m3 values, one fp32 scale for every block of 128): RMS norm / quantisation of rows, packing of weights and the
// product of the two.  Part of nfe_dense.hip's code object, beside the fp32 fully-connected layers they are the 8-bit form of.
#pragma once
#include <algorithm>
#include <cstdio>

#include "nfe_dense.h"
#include "nfe_wave.h"

NFE_NO_PACKED_FP32_BEGIN
namespace nfe {
namespace fp8 {

constexpr int BLOCK = 128;
constexpr float E4M3_MAX = 448.0f;
constexpr float SMALLEST = 1e-30f;       // lower bound of a block's maximum: an all-zero block gets a finite scale and zeros

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <int TYPE> struct Elem;
template <> struct Elem<NFE_F32> { typedef float T; };
template <> struct Elem<NFE_BF16> { typedef __bf16 T; };
template <> struct Elem<NFE_F16> { typedef _Float16 T; };
// N neighbouring values at any address that T allows, in 8- and 16-byte accesses.  (A struct of N elements is loaded and stored element by
// element as soon as the compiler has taken it apart.)
template <typename T, int N> struct Vec { T e[N]; };
typedef unsigned any8 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned any16 __attribute__((ext_vector_type(4), aligned(2)));
struct Two16 { any16 v[2]; };
template <typename T, int N> __device__ __forceinline__ Vec<T, N> load_any(const T* p) {
    constexpr int BYTES = N * (int)sizeof(T);
    static_assert(BYTES == 16 || BYTES == 32, "size");
    if constexpr (BYTES == 16) return __builtin_bit_cast(Vec<T, N>, *(const any16*)p);
    else { const Two16 t = {{*(const any16*)p, *((const any16*)p + 1)}}; return __builtin_bit_cast(Vec<T, N>, t); }
}
template <typename T, int N> __device__ __forceinline__ void store_any(T* p, const Vec<T, N>& r) {
    constexpr int BYTES = N * (int)sizeof(T);
    static_assert(BYTES == 8 || BYTES == 16 || BYTES == 32, "size");
    if constexpr (BYTES == 8) *(any8*)p = __builtin_bit_cast(any8, r);
    else if constexpr (BYTES == 16) *(any16*)p = __builtin_bit_cast(any16, r);
    else { const Two16 t = __builtin_bit_cast(Two16, r); *(any16*)p = t.v[0]; *((any16*)p + 1) = t.v[1]; }
}

__device__ __forceinline__ unsigned abs_bits(float v) { return bits_of(v) & 0x7fffffffu; }     // ordered as |v|, NaN above infinity
// four values -> four e4m3 bytes, round to nearest even
__device__ __forceinline__ unsigned e4m3x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// ------------------------------------------------------------------------------------------------
// h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight  (NORM) or y = h;  then per 128 columns
//   a = max(max |y|, 1e-30),  scale = a / 448,  q = e4m3(y / scale)
// Everything between the load of x and the rounding to e4m3 (and of h to x's type) is fp32.  The maximum is taken on the bits, so a NaN or
// an infinity in a block of y makes its scale NaN or infinite and every value of the block reads as NaN.  With the norm a NaN in h is in every
// block of y, and an infinity makes 1 / sqrt(mean) zero: NaN in its own block, zeros in the others.
// One row belongs to WAVES waves; a lane holds 8 neighbouring columns of every step, so 16 lanes share a scale.  STEPS > 0: the row stays
// in registers and is read once; STEPS = 0: longer rows, read twice.
// Bound by memory where the rows fill the chip: 16384 x 4096 bf16 with a residual (472 MB) 89.6 us = 5.27 TB/s, a large copy's rate.  A few
// thousand short rows are one round of waves and cost its latency: 10001 x 1031 fp16 (31 MB) 11.5 us.  Asking for a row's weights before its
// values, or for the next row's values early, took registers and won nothing.  Without the norm 10000 x 512 fp32 (26 MB) takes 3.9 us on the GPU
// (4.4 with it), 16384 x 4096 bf16 (203 MB, in part from cache) 33 us (34); a call takes 9 us at least.
// ------------------------------------------------------------------------------------------------
struct NormArgs {
    const void* x; const void* residual; const float* weight; void* h;
    unsigned char* q; float* scale; long long q_stride, scale_row, scale_block;
    long long rows; int cols; float eps;
};

// A lane's eight neighbouring columns of a row.  16-byte accesses take any address, so rows of any length use them; what differs is how a wave's
// 512 columns meet the row's end (all of it the same for every lane of the wave):
enum Part { FULL,        // 512 columns
            SHARED,      // fewer, and the eight columns that the last lane reads stay inside the tensor: read with the next row's first, then cleared
            LAST,        // fewer, at the tensor's end: element by element
            NONE };      // no column
template <int TYPE>
__device__ __forceinline__ void load8(float (&v)[8], const void* row, int col, int cols, Part part) {
    typedef typename Elem<TYPE>::T T;
    const T* p = (const T*)row + col;
    if (part == FULL) {
        const Vec<T, 8> r = load_any<T, 8>(p);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)r.e[k];
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    if (part == NONE) return;
    if (part == SHARED) {
        if (col < cols) {
            const Vec<T, 8> r = load_any<T, 8>(p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = col + k < cols ? (float)r.e[k] : 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (col + k < cols) v[k] = (float)p[k];
    }
}
template <int TYPE>
__device__ __forceinline__ void store8(const float (&v)[8], void* row, int col, int cols) {
    typedef typename Elem<TYPE>::T T;
    T* p = (T*)row + col;
    if (col + 8 <= cols) {
        Vec<T, 8> r;
#pragma unroll
        for (int k = 0; k < 8; ++k) r.e[k] = (T)v[k];
        store_any<T, 8>(p, r);
    } else {
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (col + k < cols) p[k] = (T)v[k];
    }
}

// What every lane of a wave knows of its row
struct NormRow {
    const NormArgs& a; long long row; const void *x, *residual; void* h; unsigned char* q; float* scale; bool shared;
    __device__ __forceinline__ NormRow(const NormArgs& args, long long r, int size) : a(args), row(r) {
        const long long at = r * args.cols * size;
        x = (const char*)args.x + at; residual = (const char*)args.residual + at; h = (char*)args.h + at;
        q = args.q + r * args.q_stride; scale = args.scale + r * args.scale_row;
        shared = (args.rows - 1 - r) * args.cols >= 7;               // up to seven elements beyond the row belong to the tensor
    }
    __device__ __forceinline__ Part part(int base, bool more) const {       // of the 512 columns from `base` on
        return base + 512 <= a.cols ? FULL : base >= a.cols ? NONE : more ? SHARED : LAST;
    }
};
template <int TYPE, bool RES>
__device__ __forceinline__ void load_h(float (&v)[8], const NormRow& R, int base, int lane) {
    const Part part = R.part(base, R.shared);
    load8<TYPE>(v, R.x, base + lane * 8, R.a.cols, part);
    if (RES) {
        float r[8];
        load8<TYPE>(r, R.residual, base + lane * 8, R.a.cols, part);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += r[k];
    }
}

// every lane of the wave takes part
template <bool NORM>
__device__ __forceinline__ void quantise8(float (&v)[8], const NormRow& R, int base, int lane, float r) {
    if (base >= R.a.cols) return;
    const int col = base + lane * 8;
    if (NORM) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= r;
        if (R.a.weight) {
            float w[8];
            load8<NFE_F32>(w, R.a.weight, col, R.a.cols, R.part(base, false));
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= w[k];
        }
    }
    unsigned m = bits_of(SMALLEST);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = umax(m, abs_bits(v[k]));
    m = row_max(m);
    const float scale = float_of(m) / E4M3_MAX;
    const float inv = 1.0f / scale;
    if (col < (R.a.cols + BLOCK - 1) / BLOCK * BLOCK) {
        uint2 w;
        w.x = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        w.y = e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *(uint2*)(R.q + col) = w;
        if ((lane & 15) == 0) R.scale[(long long)(col / BLOCK) * R.a.scale_block] = scale;
    }
}

template <int TYPE, bool NORM, bool RES, int WAVES, int STEPS>
__global__ __launch_bounds__(256) void norm_fp8_kernel(NormArgs a) {
    __shared__ float part[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long long row = WAVES == 1 ? (long long)blockIdx.x * 4 + wave : (long long)blockIdx.x;
    if (row >= a.rows) return;                                        // WAVES == 1 only: no barrier below then
    const NormRow R(a, row, (int)sizeof(typename Elem<TYPE>::T));
    const int first = WAVES == 1 ? 0 : wave * 512;
    constexpr int STRIDE = WAVES * 512, KEEP = STEPS > 0 ? STEPS : 1;
    float v[KEEP][8], sum = 0.0f;
    if (STEPS > 0) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) load_h<TYPE, RES>(v[s], R, first + s * STRIDE, lane);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (RES) store8<TYPE>(v[s], R.h, first + s * STRIDE + lane * 8, a.cols);
            if (NORM)
#pragma unroll
                for (int k = 0; k < 8; ++k) sum = fmaf(v[s][k], v[s][k], sum);
        }
    } else if (NORM) {
        for (int base = first; base < a.cols; base += STRIDE) {
            load_h<TYPE, RES>(v[0], R, base, lane);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum = fmaf(v[0][k], v[0][k], sum);
        }
    }
    float r = 1.0f;
    if (NORM) {
        sum = wave_sum(sum);
        if (WAVES > 1) {
            if (lane == 0) part[wave] = sum;
            block_sync();
            sum = (part[0] + part[1]) + (part[2] + part[3]);
        }
        r = __builtin_amdgcn_rsqf(sum / (float)a.cols + a.eps);
    }
    if (STEPS > 0) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) quantise8<NORM>(v[s], R, first + s * STRIDE, lane, r);
    } else {
        for (int base = first; base < a.cols; base += STRIDE) {
            load_h<TYPE, RES>(v[0], R, base, lane);
            if (RES) store8<TYPE>(v[0], R.h, base + lane * 8, a.cols);
            quantise8<NORM>(v[0], R, base, lane, r);
        }
    }
}

template <int TYPE, bool NORM, bool RES>
static void norm_launch(const NormArgs& a, hipStream_t st) {
    const dim3 narrow((unsigned)((a.rows + 3) / 4)), wide((unsigned)a.rows), b(256);
    // a wave for a row of up to 2048 columns, four waves for a longer one
    if (a.cols <= 512) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 1, 1>), narrow, b, 0, st, a);
    else if (a.cols <= 1024) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 1, 2>), narrow, b, 0, st, a);
    else if (a.cols <= 1536) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 1, 3>), narrow, b, 0, st, a);
    else if (a.cols <= 2048) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 1, 4>), narrow, b, 0, st, a);
    else if (a.cols <= 4096) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 4, 2>), wide, b, 0, st, a);
    else if (a.cols <= 8192) hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 4, 4>), wide, b, 0, st, a);
    else hipLaunchKernelGGL((norm_fp8_kernel<TYPE, NORM, RES, 4, 0>), wide, b, 0, st, a);
}
template <int TYPE>
static void norm_dispatch(const NormArgs& a, bool norm, hipStream_t st) {
    if (!norm) norm_launch<TYPE, false, false>(a, st);
    else if (a.residual) norm_launch<TYPE, true, true>(a, st);
    else norm_launch<TYPE, true, false>(a, st);
}

// ------------------------------------------------------------------------------------------------
// Weights [n, k] -> the operand image of v_mfma_f32_16x16x128_f8f6f4: [n/16][k/128][half 2][lane 64][16 bytes], lane l of half h holds
// columns 64 h + 16 (l / 16) .. + 15 of row l % 16, so a fragment is two contiguous kilobytes.  (The instruction sums over all 128
// columns, whose order is free as long as both operands share it.)  Rows and columns beyond n and k are zero.
// Runs once for a set of weights, so it is plain: a workgroup reads its 128 x 128 block twice (the second time from cache) and stores bytes.
// 512 x 1024 fp32 25 us, 4096 x 4096 54 us, 8192 x 8192 (335 MB) 146 us.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ long long packed_at(int n, int k, int kblocks) {
    const int c = k & 127;
    return ((((long long)(n >> 4) * kblocks + (k >> 7)) * 2 + (c >> 6)) * 64 + ((c >> 4) & 3) * 16 + (n & 15)) * 16 + (c & 15);
}

// one workgroup per 128 x 128 block; w null: q holds e4m3 bytes already
template <int TYPE>
__global__ __launch_bounds__(256) void weight_fp8_kernel(const void* w, const unsigned char* __restrict__ q, int n, int k, float gain,
                                                         unsigned char* __restrict__ packed, float* __restrict__ scale) {
    typedef typename Elem<TYPE>::T T;
    __shared__ unsigned part[4];
    const int kblocks = gridDim.x, n0 = blockIdx.y * BLOCK, k0 = blockIdx.x * BLOCK;
    const int c = threadIdx.x & 127, r0 = threadIdx.x >> 7;
    const T* src = (const T*)w;
    const int rows = (n + 15) / 16 * 16;
    float inv = 1.0f;
    if (w) {
        unsigned m = bits_of(SMALLEST);
        for (int r = r0; r < BLOCK; r += 2)
            if (n0 + r < n)
                if (k0 + c < k) m = umax(m, abs_bits((float)src[(long long)(n0 + r) * k + k0 + c]));
        for (int off = 1; off < 64; off <<= 1) m = umax(m, wave_xor(m, off));
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        block_sync();
        m = umax(umax(part[0], part[1]), umax(part[2], part[3]));
        const float s = float_of(m) / E4M3_MAX;
        if (threadIdx.x == 0) scale[(long long)blockIdx.y * kblocks + blockIdx.x] = s * gain;
        inv = 1.0f / s;
    }
    for (int r = r0; r < BLOCK; r += 2) {
        if (n0 + r >= rows) break;
        unsigned byte = 0;
        if (n0 + r < n)
            if (k0 + c < k) {
                const long long at = (long long)(n0 + r) * k + k0 + c;
                byte = w ? e4m3x4((float)src[at] * inv, 0.0f, 0.0f, 0.0f) & 255u : (unsigned)q[at];
            }
        packed[packed_at(n0 + r, k0 + c, kblocks)] = (unsigned char)byte;
    }
}

// ------------------------------------------------------------------------------------------------
// out[m, n] = act( sum_kb a_scale[m, kb] w_scale[n / 128, kb] * (sum over the 128 columns of a[m, .] w[n, .]) + bias_gain bias[n] )
// A block's sum is scaled and added in fp32, and the result is rounded once, to the output's type.  The block's own sum:
//   FP8 (bf16 and fp16 outputs): one v_mfma_f32_16x16x128_f8f6f4.  The unit adds eight products at a time in fixed point, at 2^-13 of the
//     power of two of the largest (measured: next to one product of 2^16, products below 2^3 vanish if they are among its eight and count
//     to 2^-7 otherwise; truncated towards zero), so a sum is off by less than 7 2^-13 sum|products| - 1.5e-5 of its size for normally
//     distributed values, an eighth of the rounding to fp16 and a hundredth of that to bf16.  Where products cancel, that bound is far above
//     the result's own rounding: a 16-bit result of exact sums is the fp32 output and a cast;
//   WIDE (fp32 output): both operands widened to bf16, which holds every e4m3 value, and four v_mfma_f32_16x16x32_bf16: exact products,
//     fp32 sums, half the rate.
// The weights are the instruction's first operand: lane l then holds outputs 4 (l / 16) .. + 3 of row l % 16, whose scale is one number
// per lane.
// ------------------------------------------------------------------------------------------------
struct MatmulArgs {
    const unsigned char* a; const float* a_scale; const unsigned char* w; const float* w_scale; const float* bias; void* out;
    long long a_stride, scale_row, scale_block;
    int m, n, kblocks, lrelu, out_type; float bias_gain;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bf16x8 widen8(int lo, int hi) {
    union { bf16x2 p[4]; bf16x8 v; } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return u.v;
}
// A fragment: the 32 values of 128 columns that a lane holds, in the form the instruction takes
template <bool WIDE> struct Frag;
template <> struct Frag<false> {
    i32x8 v;
    __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <> struct Frag<true> {
    bf16x8 v[4];
    __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) {
        v[0] = widen8(lo[0], lo[1]); v[1] = widen8(lo[2], lo[3]); v[2] = widen8(hi[0], hi[1]); v[3] = widen8(hi[2], hi[3]);
    }
};
__device__ __forceinline__ f32x4 mfma_block(const Frag<false>& w, const Frag<false>& a) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, zero, 0, 0, 0, 0, 0, 0);      // scales 0: the unscaled instruction
}
__device__ __forceinline__ f32x4 mfma_block(const Frag<true>& w, const Frag<true>& a) {
    f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], d, 0, 0, 0);
    return d;
}

// No instruction: what follows and needs `a` comes after what made `acc`.  Without it the compiler issues a block's products first and its
// additions after them, and spills.
__device__ __forceinline__ void in_order(f32x4& acc, i32x4& a) { asm volatile("" : "+v"(acc), "+v"(a)); }
__device__ __forceinline__ void in_order(f32x4& acc, Frag<false>& a) { asm volatile("" : "+v"(acc), "+v"(a.v)); }
__device__ __forceinline__ void in_order(f32x4& acc, Frag<true>& a) { asm volatile("" : "+v"(acc), "+v"(a.v[0]), "+v"(a.v[1]), "+v"(a.v[2]), "+v"(a.v[3])); }

template <int TYPE>
__device__ __forceinline__ void store4(const float (&v)[4], void* out, long long at, int left) {
    typedef typename Elem<TYPE>::T T;
    T* p = (T*)out + at;
    Vec<T, 4> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.e[i] = (T)v[i];
    if (left >= 4) {                              // one store at any alignment: rows of any length
        store_any<T, 4>(p, r);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) p[i] = r.e[i];
    }
}
// What a lane needs to finish columns n .. n + 3 of any row
struct Finish {
    int n, left; float bias[4];
    __device__ __forceinline__ Finish(const MatmulArgs& A, int column) : n(column), left(A.n - column) {
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = 0.0f;
        if (A.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) bias[i] = A.bias[n + i < A.n ? n + i : A.n - 1] * A.bias_gain;
    }
    template <int TYPE> __device__ __forceinline__ void store(const MatmulArgs& A, const f32x4& s, int m) const {
        if (m >= A.m) return;
        if (left <= 0) return;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = s[i] + bias[i];
        if (A.lrelu)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (v[i] < 0.0f ? v[i] * 0.2f : v[i]) * 1.4142135623730951f;      // bias_act 'lrelu': alpha 0.2, gain sqrt(2)
        store4<TYPE>(v, A.out, (long long)m * A.n + n, left);
    }
};
// each(store) calls store(sums, row) for whatever it has: one copy of it for each output type
template <bool WIDE, typename F> __device__ __forceinline__ void finish(const MatmulArgs& A, const Finish& f, F each) {
    if (WIDE) each([&](const f32x4& s, int m) { f.store<NFE_F32>(A, s, m); });
    else if (A.out_type == NFE_BF16) each([&](const f32x4& s, int m) { f.store<NFE_BF16>(A, s, m); });
    else each([&](const f32x4& s, int m) { f.store<NFE_F16>(A, s, m); });
}

// Few rows, or few tiles.  A workgroup of WAVES waves owns 16 MT rows x 16 NT columns; its waves share the K blocks, read both operands straight
// into registers, one block ahead, and join their sums through LDS in the order of the waves.  Bound by reading: every weight once for each 16 MT
// rows, every row once for each 16 NT columns.  16 x 8192 x 8192 (67.5 MB, in part from cache) 12.2 us, a library product with one scale in place of
// the blocks' 20.2; 1 x 512 x 1024 2.3 us in a replayed graph (2.9 in a trace), little more than an empty launch.
template <bool WIDE, int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, MT * NT >= 8 ? 2 : MT * NT >= 4 ? 3 : 4) void matmul_rows_kernel(MatmulArgs A) {
    __shared__ f32x4 part[WAVES][MT * NT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT), last = (A.n + 15) / 16 - 1;
    const unsigned char* ap[MT]; const float* sp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + r;
        const long long row = m < A.m ? m : A.m - 1;
        ap[i] = A.a + row * A.a_stride + g * 16;
        sp[i] = A.a_scale + row * A.scale_row;
    }
    const unsigned char* wp[NT]; const float* wsp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int nt = nt0 + j < last ? nt0 + j : last;
        wp[j] = A.w + (long long)nt * A.kblocks * 2048;
        wsp[j] = A.w_scale + (long long)(nt >> 3) * A.kblocks;
    }
    struct Block { i32x4 a[MT][2], w[NT][2]; float sa[MT], sw[NT]; };
    auto fetch = [&](Block& b, int kb) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            b.w[j][0] = *(const i32x4*)(wp[j] + (long long)kb * 2048 + lane * 16);
            b.w[j][1] = *(const i32x4*)(wp[j] + (long long)kb * 2048 + 1024 + lane * 16);
            b.sw[j] = wsp[j][kb];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            b.a[i][0] = *(const i32x4*)(ap[i] + (long long)kb * 128);
            b.a[i][1] = *(const i32x4*)(ap[i] + (long long)kb * 128 + 64);
            b.sa[i] = sp[i][kb * A.scale_block];
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const Block& b) {
        Frag<WIDE> w[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j].set(b.w[j][0], b.w[j][1]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            i32x4 lo = b.a[i][0];
            if (i > 0)
#pragma unroll
                for (int j = 0; j < NT; ++j) in_order(acc[i - 1][j], lo);
            Frag<WIDE> a;
            a.set(lo, b.a[i][1]);
            f32x4 d[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) d[j] = mfma_block(w[j], a);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float s = b.sa[i] * b.sw[j];
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[i][j][k] = fmaf(d[j][k], s, acc[i][j][k]);
            }
        }
    };
    Block even, odd;
    int kb = wave;
    if (kb < A.kblocks) fetch(even, kb);
    for (; kb + WAVES < A.kblocks; kb += 2 * WAVES) {
        fetch(odd, kb + WAVES);
        multiply(even);
        if (kb + 2 * WAVES < A.kblocks) fetch(even, kb + 2 * WAVES);
        multiply(odd);
    }
    if (kb < A.kblocks) multiply(even);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    block_sync();
    for (int t = wave; t < MT * NT; t += WAVES) {
        f32x4 s = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += part[w][t][lane];
        finish<WIDE>(A, Finish(A, (nt0 + t % NT) * 16 + g * 4), [&](auto store) { store(s, m0 + 16 * (t / NT) + r); });
    }
}

// Many rows.  A workgroup of WM x WN waves owns (16 MT WM) rows x (16 NT WN) columns; per 128 columns of K
//   * the rows' values come into a ring of LDS buffers by LDS-DMA: [row][8 chunks of 16 bytes], chunk c of row r at c ^ (r & 7) - the
//     DMA's destination is linear, so the permutation is applied to its source - which makes the fragment reads free of bank conflicts;
//     their scales beside them;
//   * the weights' fragments, already in operand order, go straight from L2 to registers: through LDS they would take it beyond its bandwidth;
//   * a wave multiplies its MT x NT fragments, MT + NT reads for MT NT matrix instructions; a product is scaled into its accumulator
//     LAG instructions after it was issued, so that the vector unit works under the matrix unit.
// Block kb begins with a wait for every load issued in the block before (rows of kb + 1, weights of kb) and issues the rows of kb + 2 and, a
// quarter into it, the weights of kb + 1.  The one barrier, in the middle of the block, says that the rows of kb + 1 are there for everybody, so no wave stops
// between blocks; and as nobody is left in block kb - 2 then, buffer (kb + 2) % 4 is free when block kb begins.
// Workgroups b, b + 8, .. run on one XCD: each XCD gets a contiguous range of tiles, GROUP row tiles deep, so that its L2 serves both operands.
// 4096^3 bf16 63 us = 2190 TFLOP/s (a library product with one scale 2730), 8191 x 8190 x 8192 fp16 462 - 477 us = 2300 - 2380 (3106): a call in a
// row of calls; the medians of a kernel trace lie above, 68 and 529 us.  The matrix unit is busy 0.53
// (4096^3) and 0.62 (8192^3) of the time, a third of a wave's life is waiting, there are no LDS conflicts, and the vector unit's scaling runs under
// the products (16.4 ns for an instruction with its four additions, 15.4 without): what is left is the waits for L2 at a block's start.
// LDS-DMA: 64 lanes x 16 (4) bytes from base + offset into 1 KiB (256 bytes) at dst.  Inline assembly, because the compiler would wait for the DMA
// into the next buffer before the reads of this one; the waits are explicit (buffer_wait).
__device__ __forceinline__ void dma16(const void* base, unsigned offset, const void* dst) {
    const unsigned l = (unsigned)(unsigned long long)(__attribute__((address_space(3))) const void*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(l), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* base, unsigned offset, const void* dst) {
    const unsigned l = (unsigned)(unsigned long long)(__attribute__((address_space(3))) const void*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(l), "v"(offset), "s"(base) : "memory", "m0");
}
// the builtin, so that the compiler counts its own loads as landed too: vmcnt(0), and nothing else
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); asm volatile("" ::: "memory"); }

constexpr int GROUP = 4;
// tile of workgroup b: bijective for any number of tiles
__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& im, int& in) {
    const int total = tm * tn, q = total / 8, r = total % 8, x = b & 7, i = b >> 3;
    const int t = x * q + (x < r ? x : r) + i;
    const int per = GROUP * tn, g = t / per, rest = t - g * per;
    const int depth = tm - g * GROUP < GROUP ? tm - g * GROUP : GROUP;
    in = rest / depth;
    im = g * GROUP + rest - in * depth;
}

template <bool WIDE, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN, 2) void matmul_tile_kernel(MatmulArgs A, int tm, int tn) {
    constexpr int THREADS = 64 * WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
    constexpr int LOADS = BM * 8 / THREADS;              // DMA instructions a wave issues for a block of rows
    static_assert(BM * 8 % THREADS == 0 && BM % 64 == 0 && BM / 64 <= WM * WN && 128 % (16 * NT) == 0, "tile shape");
    __shared__ __attribute__((aligned(16))) unsigned char rows[4][BM * 128];
    __shared__ __attribute__((aligned(16))) float scales[4][BM];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
    int im, in;
    tile_of((int)blockIdx.x, tm, tn, im, in);
    const int m0 = im * BM, n0 = in * BN + wn * (16 * NT);

    const unsigned char* a_base = A.a + (long long)m0 * A.a_stride;
    unsigned a_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int c = i * THREADS + tid, row = c >> 3;
        const int inside = m0 + row < A.m ? row : A.m - 1 - m0;
        a_off[i] = (unsigned)inside * (unsigned)A.a_stride + (unsigned)(((c & 7) ^ (row & 7)) * 16);
    }
    const int srow = wave * 64 + lane;
    const float* s_base = A.a_scale + (long long)m0 * A.scale_row;
    const unsigned s_off = (unsigned)(m0 + srow < A.m ? srow : A.m - 1 - m0) * (unsigned)A.scale_row * 4u;
    const int last = (A.n + 15) / 16 - 1;
    const unsigned char* w_base[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int nt = n0 / 16 + j < last ? n0 / 16 + j : last;
        w_base[j] = A.w + (long long)nt * A.kblocks * 2048;
    }
    const int nb = n0 / BLOCK < (A.n - 1) / BLOCK ? n0 / BLOCK : (A.n - 1) / BLOCK;
    const float* w_scale = A.w_scale + (long long)nb * A.kblocks;

    struct Weights { i32x4 v[NT][2]; float scale; };
    auto fetch_rows = [&](int kb) {
        const int buf = kb & 3;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) dma16(a_base + (long long)kb * 128, a_off[i], &rows[buf][(i * THREADS + wave * 64) * 16]);
        if (wave < BM / 64) dma4(s_base + kb * A.scale_block, s_off, &scales[buf][wave * 64]);
    };
    auto fetch_weights = [&](Weights& w, int kb) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) w.v[j][h] = *(const i32x4*)(w_base[j] + (long long)kb * 2048 + h * 1024 + lane * 16);
        w.scale = w_scale[kb];
    };
    const int at = (wm * MT * 16 + r) * 128, at0 = at + ((g ^ (r & 7)) * 16), at1 = at + (((g + 4) ^ (r & 7)) * 16), st = wm * MT * 16 + r;
    struct Row { i32x4 lo, hi; float scale; };
    auto read_row = [&](Row& a, int kb, int i) {
        const int buf = kb & 3;
        a.lo = *(const i32x4*)&rows[buf][at0 + i * 2048];
        a.hi = *(const i32x4*)&rows[buf][at1 + i * 2048];
        a.scale = scales[buf][st + i * 16];
    };

    // the row of fragments at which the next weights are asked for: not in one burst with the rows (8192^3 bf16 484 -> 468 us, 2048^3 fp32 22.8 ->
    // 22.0), except where the widened fragments leave no registers to have both in flight (8192^3 fp32 921 -> 885)
    constexpr int FETCH = WIDE && NT == 4 ? 0 : MT / 4;
    constexpr int LAG = 2, SLOTS = 4;                    // SLOTS divides MT NT: products keep their slots from block to block
    static_assert(MT * NT % SLOTS == 0 && MT % 2 == 0 && NT >= LAG, "schedule");
    f32x4 acc[MT][NT], d[SLOTS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) d[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float s_now = 0.0f, s_before = 0.0f;
    Row row;
    Weights even, odd;

    auto block = [&](int kb, const Weights& raw, Weights& next) {
        wait_loads();
        if (kb + 2 < A.kblocks) fetch_rows(kb + 2);
        Frag<WIDE> w[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j].set(raw.v[j][0], raw.v[j][1]);
        const float sw = raw.scale;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (i == MT / 2) block_sync();
            if (i == FETCH) { if (kb + 1 < A.kblocks) fetch_weights(next, kb + 1); }
            Frag<WIDE> a;
            a.set(row.lo, row.hi);
            s_before = s_now;
            s_now = row.scale * sw;
            if (i + 1 < MT) read_row(row, kb, i + 1);
            else read_row(row, kb + 1, 0);               // after the last block: whatever the ring holds, unused
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int t = i * NT + j, old = (t + SLOTS - LAG) % SLOTS;
                d[t % SLOTS] = mfma_block(w[j], a);
                const int io = j >= LAG ? i : (i + MT - 1) % MT, jo = (j + NT - LAG) % NT;
                const float s = j >= LAG ? s_now : s_before;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[io][jo][e] = fmaf(d[old][e], s, acc[io][jo][e]);
                in_order(acc[io][jo], a);
            }
        }
    };
    fetch_rows(0);
    if (A.kblocks > 1) fetch_rows(1);
    fetch_weights(even, 0);
    wait_loads();
    block_sync();
    read_row(row, 0, 0);
    int kb = 0;
    for (; kb + 1 < A.kblocks; kb += 2) {                // in pairs, so that no weights are moved between registers
        block(kb, even, odd);
        block(kb + 1, odd, even);
    }
    if (kb < A.kblocks) block(kb, even, odd);
#pragma unroll
    for (int j = NT - LAG; j < NT; ++j) {
        const int t = MT * NT - NT + j;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[MT - 1][j][e] = fmaf(d[t % SLOTS][e], s_now, acc[MT - 1][j][e]);
    }
    // A wave's results go through its part of the ring, 16-byte chunk c of row r at c ^ r, and come back as whole row segments: full cache
    // lines to store, and one copy of the finishing code (straight from the accumulators it was most of the kernel's code, and a call's first
    // workgroups wait for every line of it).
    constexpr int CHUNKS = 4 * NT, TILE = MT * NT * 1024 * WM * WN, RING = 4 * BM * 128, PARTS = TILE > RING ? TILE / RING : 1, PM = MT / PARTS;
    static_assert(MT % PARTS == 0 && TILE <= RING * PARTS, "epilogue");
    unsigned char* mine = &rows[0][0] + wave * (PM * NT * 1024);
    const int c = lane & (CHUNKS - 1), first = lane / CHUNKS;
    const Finish f(A, n0 + c * 4);
    block_sync();
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (p > 0) wave_sync();                          // other lanes still read the part before
#pragma unroll
        for (int i = 0; i < PM; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) *(f32x4*)(mine + ((i * 16 + r) * CHUNKS + ((j * 4 + g) ^ (r & (CHUNKS - 1)))) * 16) = acc[p * PM + i][j];
        wave_sync();
        finish<WIDE>(A, f, [&](auto store) {
#pragma unroll 4
            for (int t = 0; t < PM * NT; ++t) {
                const int row = t * (64 / CHUNKS) + first;
                store(*(const f32x4*)(mine + (row * CHUNKS + (c ^ (row & (CHUNKS - 1)))) * 16), m0 + (wm * MT + p * PM) * 16 + row);
            }
        });
    }
}

template <bool WIDE, int WM, int WN, int MT, int NT>
static int tile_launch(const MatmulArgs& A, hipStream_t st) {
    constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN;
    const long long tm = ((long long)A.m + BM - 1) / BM, tn = ((long long)A.n + BN - 1) / BN;
    NFE_REQUIRE(tm * tn * (64 * WM * WN) <= 0xffffffffll, "nfe_fp8_matmul: m=%d n=%d are too large", A.m, A.n);      // work items of a launch
    hipLaunchKernelGGL((matmul_tile_kernel<WIDE, WM, WN, MT, NT>), dim3((unsigned)(tm * tn)), dim3(64 * WM * WN), 0, st, A, (int)tm, (int)tn);
    return NFE_OK;
}

template <bool WIDE, int MT, int NT, int WAVES>
static int rows_launch(const MatmulArgs& A, hipStream_t st) {
    const long long x = ((long long)A.n + 16 * NT - 1) / (16 * NT), y = ((long long)A.m + 16 * MT - 1) / (16 * MT);
    NFE_REQUIRE(y <= 65535, "nfe_fp8_matmul: m=%d is too large for rows %lld bytes apart", A.m, A.a_stride);
    hipLaunchKernelGGL((matmul_rows_kernel<WIDE, MT, NT, WAVES>), dim3((unsigned)x, (unsigned)y), dim3(64 * WAVES), 0, st, A);
    return NFE_OK;
}
// Which kernel.  Up to 16 rows: one tile of rows, as a second would hold none, and eight waves to share K (against 32 x 64 on four waves, fp32
// outputs: 16 x 16384 x 4096 15.9 -> 12.7 us, 16 x 20000 x 8192 32.7 -> 27.1, 1 x 65536 x 2048 22.4 -> 21.1; bf16 13.9 -> 12.6, 31.1 -> 26.8, 21.9 -> 21.1).
// More: rows kernels: the largest tile that still gives every CU a workgroup (their waves share K, so a short chain of blocks stays
// short).  Among the widest of them and the tile kernels: the least of rounds x (time of one workgroup's K block), rounds = workgroups /
// CUs rounded up, but not less than what a lone workgroup takes for a block (loads' latency).  The times are of 256 CUs and one clock; another number
// of CUs is counted, but its choice has not been measured.  us, K block = 128; "measured": a call in a row of calls on the same operands
//                       a workgroup's block, CU full   alone     measured
//   32 x 64   rows   8-bit 0.23, widened 0.28       0.29, 0.33   128 x 8192 x 8192: 26.5 (bf16), 28.6 us (fp32); 64 rows: 16.0, 19.8
//   64 x 64   tile         0.30          0.36       0.62, 0.67   512 x 4096 x 4096: 16.8, 25.0
//   128 x 128 tile         0.66          1.15       0.82, 1.20   2048^3: 12.7, 21.2
//   256 x 256 tile         2.00                     2.00         4096^3: 63
//   128 x 256 tile                       1.94             1.94   4096^3: 118
// E.g. 10000 x 512 x 1024 fp32: 64 x 64 5 rounds x 0.36, 128 x 128 2 x 1.15, 128 x 256 1 x 1.94: 17.4 - 18.5, 24.5, 21.8 us measured.
// Offsets inside a tile are 32-bit: 256 rows of up to 2^23 bytes (and scales that far apart); anything wider stays on the rows kernels.
enum Choice { ROWS_16X16, ROWS_16X32, ROWS_32X32, ROWS_32X64, TILE_64X64, TILE_128X128, TILE_LARGE };
static Choice choose(bool wide, int m, int n, long long a_stride, long long scale_row) {
    const int cus = num_cus();
    auto count = [&](int bm, int bn) { return (((long long)m + bm - 1) / bm) * (((long long)n + bn - 1) / bn); };
    const bool near = a_stride <= (1 << 23) && scale_row <= (1 << 21);
    if (m <= 16) return count(16, 32) < cus ? ROWS_16X16 : ROWS_16X32;
    if (!near) return ROWS_32X64;
    if (count(32, 64) < cus) {
        if (count(32, 32) < cus) return count(16, 32) < cus ? ROWS_16X16 : ROWS_16X32;
        return ROWS_32X32;
    }
    auto cost = [&](int bm, int bn, double full, double alone) { return std::max(alone, full * (double)((count(bm, bn) + cus - 1) / cus)); };
    const double rows = wide ? cost(32, 64, 0.28, 0.33) : cost(32, 64, 0.23, 0.29), small = wide ? cost(64, 64, 0.36, 0.67) : cost(64, 64, 0.30, 0.62),
                 middle = wide ? cost(128, 128, 1.15, 1.20) : cost(128, 128, 0.66, 0.82), large = wide ? cost(128, 256, 1.94, 1.94) : cost(256, 256, 2.0, 2.0);
    const double best = std::min(std::min(rows, small), std::min(middle, large));
    return rows == best ? ROWS_32X64 : small == best ? TILE_64X64 : middle == best ? TILE_128X128 : TILE_LARGE;
}
template <bool WIDE>
static int matmul_launch(const MatmulArgs& A, hipStream_t st) {
    switch (choose(WIDE, A.m, A.n, A.a_stride, A.scale_row)) {
        case ROWS_16X16: return rows_launch<WIDE, 1, 1, 8>(A, st);
        case ROWS_16X32: return rows_launch<WIDE, 1, 2, 8>(A, st);
        case ROWS_32X32: return rows_launch<WIDE, 2, 2, 8>(A, st);
        case ROWS_32X64: return rows_launch<WIDE, 2, 4, 4>(A, st);
        case TILE_64X64: return tile_launch<WIDE, 2, 2, 2, 2>(A, st);
        case TILE_128X128: return tile_launch<WIDE, 2, 4, 4, 2>(A, st);
        default: return WIDE ? tile_launch<true, 2, 4, 4, 4>(A, st) : tile_launch<false, 2, 4, 8, 4>(A, st);
    }
}

static int check_rows(const char* who, long long rows, int cols) {
    NFE_REQUIRE(rows > 0 && rows <= 0x7fffffffll, "%s: rows=%lld must be in [1, 2^31)", who, rows);
    NFE_REQUIRE(cols > 0 && cols <= (1 << 30), "%s: cols=%d must be in [1, 2^30]", who, cols);
    return NFE_OK;
}
static int norm_entry(const char* who, NormArgs& a, int dtype, bool norm, nfe_stream_t stream) {
    if (int rc = check_rows(who, a.rows, a.cols)) return rc;
    NFE_REQUIRE(dtype == NFE_F32 || dtype == NFE_BF16 || dtype == NFE_F16, "%s: unknown dtype %d", who, dtype);
    NFE_REQUIRE(a.x && a.q && a.scale, "%s: null pointer", who);
    NFE_REQUIRE((a.residual != nullptr) == (a.h != nullptr), "%s: residual and h come in pairs", who);
    const int width = (a.cols + BLOCK - 1) / BLOCK * BLOCK;
    NFE_REQUIRE(a.q_stride >= width && a.q_stride % 8 == 0 && (uintptr_t)a.q % 8 == 0, "%s: q rows must be 8-byte aligned and at least %d bytes apart", who, width);
    NFE_REQUIRE(!norm || a.eps >= 1.17549435e-38f, "%s: eps must be a positive normal number", who);      // v_rsq_f32 takes less for zero
    const long long rows = a.rows, most = 1 << 22;                    // 2^32 work items are a launch's limit
    for (long long at = 0; at < rows; at += most) {
        NormArgs part = a;
        const long long first = at * a.cols * (dtype == NFE_F32 ? 4 : 2);
        part.rows = rows - at < most ? rows - at : most;
        part.x = (const char*)a.x + first;
        if (a.residual) { part.residual = (const char*)a.residual + first; part.h = (char*)a.h + first; }
        part.q = a.q + at * a.q_stride;
        part.scale = a.scale + at * a.scale_row;
        if (dtype == NFE_F32) norm_dispatch<NFE_F32>(part, norm, (hipStream_t)stream);
        else if (dtype == NFE_BF16) norm_dispatch<NFE_BF16>(part, norm, (hipStream_t)stream);
        else norm_dispatch<NFE_F16>(part, norm, (hipStream_t)stream);
        NFE_CHECK_LAUNCH(who);
    }
    return NFE_OK;
}
static int check_weight(const char* who, int n, int k) {
    NFE_REQUIRE(n > 0 && k > 0 && n <= 65535 * BLOCK && k <= (1 << 30), "%s: bad sizes n=%d k=%d", who, n, k);
    return NFE_OK;
}

}  // namespace fp8
}  // namespace nfe
NFE_NO_PACKED_FP32_END

extern "C" int nfe_rms_norm_fp8(const void* x, const void* residual, const float* weight, int dtype, int64_t rows, int cols, float eps, void* h, void* q,
                                int64_t q_stride, float* scale, int64_t scale_row_stride, int64_t scale_block_stride, nfe_stream_t stream) {
    nfe::fp8::NormArgs a{x, residual, weight, h, (unsigned char*)q, scale, q_stride, scale_row_stride, scale_block_stride, rows, cols, eps};
    return nfe::fp8::norm_entry("nfe_rms_norm_fp8", a, dtype, true, stream);
}
extern "C" int nfe_quantize_fp8(const void* x, int dtype, int64_t rows, int cols, void* q, int64_t q_stride, float* scale, int64_t scale_row_stride,
                                int64_t scale_block_stride, nfe_stream_t stream) {
    nfe::fp8::NormArgs a{x, nullptr, nullptr, nullptr, (unsigned char*)q, scale, q_stride, scale_row_stride, scale_block_stride, rows, cols, 0.0f};
    return nfe::fp8::norm_entry("nfe_quantize_fp8", a, dtype, false, stream);
}
extern "C" uint64_t nfe_fp8_weight_bytes(int n, int k) {
    return n > 0 && k > 0 ? ((uint64_t)n + 15) / 16 * (((uint64_t)k + 127) / 128) * 2048 : 0;
}
extern "C" int nfe_fp8_weight_quantize(const void* w, int dtype, int n, int k, float gain, void* packed, float* scale, nfe_stream_t stream) {
    using namespace nfe::fp8;
    if (int rc = check_weight("nfe_fp8_weight_quantize", n, k)) return rc;
    NFE_REQUIRE(w && packed && scale, "nfe_fp8_weight_quantize: null pointer");
    NFE_REQUIRE(dtype == NFE_F32 || dtype == NFE_BF16 || dtype == NFE_F16, "nfe_fp8_weight_quantize: unknown dtype %d", dtype);
    const dim3 grid((unsigned)((k + BLOCK - 1) / BLOCK), (unsigned)((n + BLOCK - 1) / BLOCK));
    auto kernel = dtype == NFE_F32 ? weight_fp8_kernel<NFE_F32> : dtype == NFE_BF16 ? weight_fp8_kernel<NFE_BF16> : weight_fp8_kernel<NFE_F16>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, w, (const unsigned char*)nullptr, n, k, gain, (unsigned char*)packed, scale);
    NFE_CHECK_LAUNCH("nfe_fp8_weight_quantize");
    return NFE_OK;
}
extern "C" int nfe_fp8_weight_pack(const void* q, int n, int k, void* packed, nfe_stream_t stream) {
    using namespace nfe::fp8;
    if (int rc = check_weight("nfe_fp8_weight_pack", n, k)) return rc;
    NFE_REQUIRE(q && packed, "nfe_fp8_weight_pack: null pointer");
    const dim3 grid((unsigned)((k + BLOCK - 1) / BLOCK), (unsigned)((n + BLOCK - 1) / BLOCK));
    hipLaunchKernelGGL(weight_fp8_kernel<NFE_F32>, grid, dim3(256), 0, (hipStream_t)stream, (const void*)nullptr, (const unsigned char*)q, n, k, 1.0f,
                       (unsigned char*)packed, (float*)nullptr);
    NFE_CHECK_LAUNCH("nfe_fp8_weight_pack");
    return NFE_OK;
}
extern "C" int nfe_fp8_matmul(const nfe_fp8_matmul_args* p, nfe_stream_t stream) {
    using namespace nfe::fp8;
    NFE_REQUIRE(p, "nfe_fp8_matmul: args is null");
    NFE_REQUIRE(p->struct_size == sizeof(*p), "nfe_fp8_matmul: struct_size %u != %zu", p->struct_size, sizeof(*p));
    NFE_REQUIRE(p->q && p->scale && p->packed && p->w_scale && p->out, "nfe_fp8_matmul: null pointer");
    if (int rc = check_weight("nfe_fp8_matmul", p->n, p->k)) return rc;
    NFE_REQUIRE(p->m > 0 && p->m <= (1 << 30), "nfe_fp8_matmul: m=%d must be in [1, 2^30]", p->m);
    const int kblocks = (p->k + BLOCK - 1) / BLOCK;
    NFE_REQUIRE(p->q_stride >= (int64_t)kblocks * BLOCK && p->q_stride % 16 == 0 && (uintptr_t)p->q % 16 == 0 && (uintptr_t)p->packed % 16 == 0,
                "nfe_fp8_matmul: q rows must be 16-byte aligned and at least %d bytes apart", kblocks * BLOCK);
    NFE_REQUIRE(p->out_dtype == NFE_F32 || p->out_dtype == NFE_BF16 || p->out_dtype == NFE_F16, "nfe_fp8_matmul: unknown out_dtype %d", p->out_dtype);
    NFE_REQUIRE(p->scale_row_stride >= 0 && p->scale_block_stride >= 0, "nfe_fp8_matmul: negative scale stride");
    const int size = p->out_dtype == NFE_F32 ? 4 : 2;
    NFE_REQUIRE((uintptr_t)p->out % size == 0, "nfe_fp8_matmul: misaligned out");
    MatmulArgs A{(const unsigned char*)p->q, p->scale, (const unsigned char*)p->packed, p->w_scale, p->bias, p->out, p->q_stride, p->scale_row_stride,
                 p->scale_block_stride, p->m, p->n, kblocks, p->lrelu, p->out_dtype, p->bias_gain};
    if (int rc = p->out_dtype == NFE_F32 ? matmul_launch<true>(A, (hipStream_t)stream) : matmul_launch<false>(A, (hipStream_t)stream)) return rc;
    NFE_CHECK_LAUNCH("nfe_fp8_matmul");
    return NFE_OK;
}
extern "C" int nfe_fp8_matmul_describe(int m, int n, int64_t q_stride, int64_t scale_row_stride, int out_dtype, char* buf, int buf_len) {
    using namespace nfe::fp8;
    NFE_REQUIRE(buf && buf_len > 0, "nfe_fp8_matmul_describe: no buffer");
    NFE_REQUIRE(m > 0 && n > 0, "nfe_fp8_matmul_describe: bad sizes m=%d n=%d", m, n);
    NFE_REQUIRE(out_dtype == NFE_F32 || out_dtype == NFE_BF16 || out_dtype == NFE_F16, "nfe_fp8_matmul_describe: unknown out_dtype %d", out_dtype);
    static const char* names[] = {"rows 16x16/8w", "rows 16x32/8w", "rows 32x32/8w", "rows 32x64/4w", "tile 64x64/4w", "tile 128x128/8w"};
    const bool wide = out_dtype == NFE_F32;
    const Choice c = choose(wide, m, n, q_stride, scale_row_stride);
    snprintf(buf, (size_t)buf_len, "%s %s", c != TILE_LARGE ? names[c] : wide ? "tile 128x256/8w" : "tile 256x256/8w", wide ? "widened" : "8-bit");
    return NFE_OK;
}
