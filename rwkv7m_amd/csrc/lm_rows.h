// Shared device helpers of the language model head's kernels (lm_norm.hip,
// lm_score.hip, lm_distill.hip): rows of a strided array, sums over a
// workgroup, and the softmax statistics of a row of logits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wkv7_common.h"
#include "wkv7_launch.h"

namespace rwkv7m {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ int64_t row_offset(const LmRows& R, int64_t row) {
    if (row < R.inner) return row * R.inner_stride;  // (no division)
    return row / R.inner * R.outer_stride + row % R.inner * R.inner_stride;
}

// 16 bytes of adjacent elements, at their element's own alignment: gfx950
// takes such a load or store as one instruction at any address.
template <typename E>
struct Vec {
    static constexpr int n = 16 / int(sizeof(E));
    typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));
    raw_t raw;

    __device__ __forceinline__ void load(const E* p) {
        raw = *reinterpret_cast<const raw_t*>(p);
    }
    __device__ __forceinline__ void store(E* p) const {
        *reinterpret_cast<raw_t*>(p) = raw;
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(E) == 4) return __uint_as_float(raw[j]);
        const uint32_t u = raw[j >> 1];
        return __uint_as_float(j & 1 ? u & 0xffff0000u : u << 16);
    }
    // Element pair j, j + 1 (j even), rounded to nearest even in bf16.
    __device__ __forceinline__ void set2(int j, float a, float b) {
        if constexpr (sizeof(E) == 4) {
            raw[j] = __float_as_uint(a);
            raw[j + 1] = __float_as_uint(b);
        } else {
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            const f32x2 f = {a, b};
            raw[j >> 1] = __builtin_bit_cast(
                uint32_t, __builtin_convertvector(f, bf16x2));
        }
    }
};

// The sum over aligned groups of G lanes (16, 64), the same in each of them.
template <int G>
__device__ __forceinline__ float lanes_sum(float x) {
    x = group_sum<16>(x);
    if constexpr (G == 64) x = add_swap<32>(add_swap<16>(x));
    return x;
}

// The larger of two, a NaN if either is one (v_maximum3_f32).
__device__ __forceinline__ float larger(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
}

// f over one value of each of the workgroup's W waves' lanes, the same in
// every thread; `s` holds W values and may be used again after the call.
template <int W, typename T, typename F>
__device__ __forceinline__ T block_fold(T x, T* s, F f) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x = f(x, __shfl_xor(x, m));
    if constexpr (W == 1) return x;
    __syncthreads();
    if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = x;
    __syncthreads();
    x = s[0];
#pragma unroll
    for (int w = 1; w < W; ++w) x = f(x, s[w]);
    return x;
}

template <int W>
__device__ __forceinline__ float block_sum(float x, float* s) {
    return block_fold<W>(x, s, [](float a, float b) { return a + b; });
}

// Softmax statistics of a set of logits x at temperature T, with c = log2(e)
// / T: d = x - ref, e = 2^(d c), s0 = sum e, s1 = sum e d, where ref is the
// largest x (0 in a set without one above -inf: there e is 0).  x - ref is
// taken before the product with c: it is exact or nearly so where e counts,
// and neither a row of the type's lowest value nor one near its largest
// overflows.  d is held above -200 / c (2^-200 is 0 in fp32), so that -inf
// adds nothing rather than NaN; NaN and +inf - inf stay NaN.
struct SoftStats {
    float ref, s0, s1;
};

__device__ __forceinline__ float ref_of(float largest) {
    return largest == -__builtin_inff() ? 0.f : largest;
}

__device__ __forceinline__ float soft_d(float x, float ref, float lowest) {
    return larger(x - ref, lowest);
}

__device__ __forceinline__ void soft_add(SoftStats& a, float x, float c,
                                         float lowest) {
    const float d = soft_d(x, a.ref, lowest);
    const float e = __builtin_amdgcn_exp2f(d * c);
    a.s0 += e;
    a.s1 = __builtin_fmaf(e, d, a.s1);
}

}  // namespace rwkv7m
