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

// One workgroup a row: a grid of 2^16 columns (a grid has fewer than 2^32
// threads along an axis) and the row a workgroup of it takes, which may be
// past the last one.  A loop over rows instead would keep what does not change
// between them in registers that the row needs: workgroups that stayed, and
// loaded the next row while they finished one, took 169 us where these take 94
// ([4088, 65536] bf16 scored), having spilled a quarter of the row.
inline dim3 row_grid(int64_t rows) {
    const int64_t most = 1 << 16;
    return rows <= most ? dim3(unsigned(rows))
                        : dim3(unsigned(most),
                               unsigned((rows + most - 1) / most));
}
__device__ __forceinline__ int64_t grid_row() {
    return int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
}

// The larger of two, a NaN if either is one (v_maximum3_f32).
__device__ __forceinline__ float larger(float a, float b) {
    return __builtin_elementwise_maximum(a, b);
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

// f over aligned groups of G lanes (2, 4, 8, 16 or 64), the same in each of
// them: lane rotations and swaps in the instructions themselves, without the
// LDS traffic and the address registers of shuffles (a row of 65536 bf16 with
// 10 alternatives is scored 4 % faster).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, 0xf, 0xf,
                                                false));
}
template <int G, typename T, typename F>
__device__ __forceinline__ T lanes_fold(T x, F f) {
    static_assert(sizeof(T) == 4 && (G == 2 || G == 4 || G == 8 || G == 16 ||
                                     G == 64), "");
    const auto bits = [](T v) { return __builtin_bit_cast(uint32_t, v); };
    const auto value = [](uint32_t u) { return __builtin_bit_cast(T, u); };
    if constexpr (G <= 8) {
        if constexpr (G == 8) x = f(x, value(dpp<0x141>(bits(x))));  // 7 - lane
        if constexpr (G >= 4) x = f(x, value(dpp<0x4e>(bits(x))));  // lane ^ 2
        return f(x, value(dpp<0xb1>(bits(x))));  // lane ^ 1
    }
    // rotations of a row of 16 lanes: after each, lanes that far apart agree
    x = f(x, value(dpp<0x128>(bits(x))));
    x = f(x, value(dpp<0x124>(bits(x))));
    x = f(x, value(dpp<0x122>(bits(x))));
    x = f(x, value(dpp<0x121>(bits(x))));
    if constexpr (G == 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(bits(x), bits(x),
                                                        false, false);
        x = f(value(a[0]), value(a[1]));
        const auto b = __builtin_amdgcn_permlane32_swap(bits(x), bits(x),
                                                        false, false);
        x = f(value(b[0]), value(b[1]));
    }
    return x;
}

template <int G, typename T>
__device__ __forceinline__ T lanes_sum(T x) {
    return lanes_fold<G>(x, [](T a, T b) { return a + b; });
}

template <int G>
__device__ __forceinline__ float lanes_larger(float x) {
    return lanes_fold<G>(x, [](float a, float b) { return larger(a, b); });
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

// f over the W values (1, 4, 8 or 16) that a workgroup's waves left in `s` (after
// a barrier), the same in every lane.
template <int W, typename F>
__device__ __forceinline__ float waves_fold(const float* s, F f) {
    if constexpr (W == 1)
        return s[0];
    else
        return lanes_fold<W>(s[threadIdx.x % W], f);
}

template <int W>
__device__ __forceinline__ float waves_sum(const float* s) {
    return waves_fold<W>(s, [](float a, float b) { return a + b; });
}
template <int W>
__device__ __forceinline__ float waves_larger(const float* s) {
    return waves_fold<W>(s, [](float a, float b) { return larger(a, b); });
}

// Waves a SIMD that a kernel with a Row of NV vectors a thread leaves room for,
// of the 512 registers a lane has there: 8 of 64 (4 NV <= 32 hold the row),
// 6 of 80 for three workgroups of 512 threads a CU, 4 of 128 where the row
// takes 64.
template <int NT, int NV>
constexpr int kRowWaves = NT == 512 ? 6 : NV <= 8 ? 8 : 4;

// An offset that is the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint64_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(x)));
    const uint64_t hi = uint32_t(__builtin_amdgcn_readfirstlane(int(x >> 32)));
    return int64_t(hi << 32 | lo);
}

__device__ __forceinline__ float uniform(float x) {
    return __uint_as_float(uint32_t(
        __builtin_amdgcn_readfirstlane(int(__float_as_uint(x)))));
}

// A row of V elements cut at the addresses that are multiples of 16 bytes:
// `lead` elements, `whole` vectors, `rest` elements.  Vectors that straddle
// such addresses load at 4.7 TB/s where these reach 5.8 ([4088, 65529] bf16).
template <typename E>
struct Cut {
    static constexpr int n = Vec<E>::n;
    int lead, whole, rest;

    __device__ __forceinline__ Cut(const E* x, int V) {
        const uint32_t past = uint32_t(reinterpret_cast<uint64_t>(x)) & 15u;
        lead = int((16u - past) & 15u) / int(sizeof(E));
        if (lead > V) lead = V;
        whole = (V - lead) / n;
        rest = (V - lead) % n;
    }
};

constexpr int kLargestRow = 1024 * 16;

// A row of V logits in the registers of the NT threads of a workgroup: NV
// whole vectors each, vector i * NT + thread, with -inf in the places past
// the row's whole vectors, and the elements before and behind those one to a
// thread (-inf in the others).  What is past the first NV * NT vectors of the
// largest variant is read again from memory each time the row is walked.
template <typename E, int NT, int NV>
struct Row {
    static constexpr int n = Vec<E>::n;
    const E* x;
    int V;
    Cut<E> cut;
    Vec<E> v[NV];
    float one;

    __device__ __forceinline__ Row(const E* p, int length)
        : x(p), V(length), cut(p, length) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i + 1) * NT <= cut.whole) {  // (the same in every thread)
                v[i].load(at(i));
            } else {
                v[i].raw = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
                if (i * NT + int(threadIdx.x) < cut.whole) v[i].load(at(i));
            }
        }
        one = has_one() ? load_f(x + one_id()) : -__builtin_inff();
    }
    // vector i * NT + thread of the row (i the same in every thread)
    __device__ __forceinline__ const E* at(int i) const {
        // (a scalar base and a 32-bit offset: the empty asm keeps the two
        // from being added up in vector registers for each i)
        int64_t base = int64_t(cut.lead + i * NT * n) * int64_t(sizeof(E));
        asm volatile("" : "+s"(base));
        return reinterpret_cast<const E*>(reinterpret_cast<const char*>(x) +
                                          base + uint32_t(threadIdx.x) * 16u);
    }
    __device__ __forceinline__ bool has_one() const {
        return int(threadIdx.x) < cut.lead + cut.rest;
    }
    __device__ __forceinline__ int one_id() const {
        const int t = threadIdx.x;
        return t < cut.lead ? t : V - cut.rest - cut.lead + t;
    }
    // f(vector, its number) over the thread's vectors, the last of which may
    // be past the row's whole vectors (-inf).  The empty asm keeps the
    // compiler from carrying one walk's unpacked elements over to the next in
    // two to four times the registers.  With COPY f gets a copy, for a walk in
    // a branch beside another one: the asm's results of both would have to
    // meet in one set of registers behind it, and the row spills.
    template <bool COPY = false, typename F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (COPY) {
                if (i * NT >= cut.whole) continue;
                Vec<E> a = v[i];
                asm volatile("" : "+v"(a.raw));
                f(a, i * NT + int(threadIdx.x));
            } else {
                asm volatile("" : "+v"(v[i].raw));
                if (i * NT < cut.whole) f(v[i], i * NT + int(threadIdx.x));
            }
        }
        // (rows of the other variants end within their registers: without
        // this loop they keep within 64 of them)
        if constexpr (NT * NV == kLargestRow)
#pragma unroll 1
            for (int i = NV; i * NT < cut.whole; i += 4) {
                Vec<E> a[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    a[u].raw = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
                    if ((i + u) * NT + int(threadIdx.x) < cut.whole)
                        a[u].load(at(i + u));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    f(a[u], (i + u) * NT + int(threadIdx.x));
            }
    }
    __device__ __forceinline__ float largest() {
        float m = one;
        each([&](const Vec<E>& a, int) {
#pragma unroll
            for (int j = 0; j < n; ++j) m = larger(m, a.get(j));
        });
        return m;
    }
};

// go(KERNEL<E, NT, NV>, NT) with the smallest workgroup that holds a row of V
// logits: where `wave` a wave up to 8 vectors a thread (4096 bf16; no barriers:
// 60000 such rows are scored in 85 us, by 256 threads each in 109), 256
// threads up to 8 (16384), 1024 threads with 4 (32768), NT8 threads up to 8192
// vectors (65536), then 1024; rows past 16 vectors of 1024 threads (131072
// bf16) read their rest again each walk.
#define RWKV7M_LM_ROW_KERNEL(KERNEL, E, V, wave, NT8, go) \
    do {                                              \
        constexpr int64_t vec = Vec<E>::n;            \
        if ((wave) && (V) <= 64 * 1 * vec)            \
            go(KERNEL<E, 64, 1>, 64);                 \
        else if ((wave) && (V) <= 64 * 2 * vec)       \
            go(KERNEL<E, 64, 2>, 64);                 \
        else if ((wave) && (V) <= 64 * 4 * vec)       \
            go(KERNEL<E, 64, 4>, 64);                 \
        else if ((wave) && (V) <= 64 * 8 * vec)       \
            go(KERNEL<E, 64, 8>, 64);                 \
        else if ((V) <= 256 * 2 * vec)                \
            go(KERNEL<E, 256, 2>, 256);               \
        else if ((V) <= 256 * 4 * vec)                \
            go(KERNEL<E, 256, 4>, 256);               \
        else if ((V) <= 256 * 8 * vec)                \
            go(KERNEL<E, 256, 8>, 256);               \
        else if ((V) <= 1024 * 4 * vec)               \
            go(KERNEL<E, 1024, 4>, 1024);             \
        else if ((V) <= 1024 * 8 * vec)               \
            go(KERNEL<E, NT8, 8192 / NT8>, NT8);      \
        else                                          \
            go(KERNEL<E, 1024, 16>, 1024);            \
    } while (0)

// Softmax over a row of logits x at temperature T in base 2: e = 2^t with t =
// (x - ref) c, c = log2(e) / T and ref the row's largest.  A row with no
// element above -inf has ref 0, and every e 0.
// Up to |ref c| = 2^16, one fma an element: t = x c - refc, refc the rounded
// product, which moves every t by the same 2^-9 or less.  e is then the
// softmax up to a factor that does not depend on x, and everything is taken
// from the same t.  That factor grows with |ref c| and leaves fp32's range at
// 2^31 (logits of -1e10, a temperature of 1e-8), so rows beyond take the
// difference first: next to ref it is exact, and t is off by its own rounding
// alone at any size.  Taken so for every row, the added operation costs rows
// of 4096 to 131072 bf16 3 to 4 % of their scoring's time.
struct RowSoftmax {
    float c, ref, refc;
    bool one_fma;  // (the same in every lane)

    // (largest is the same in every lane)
    __device__ __forceinline__ RowSoftmax(float largest, float c_)
        : c(c_), ref(uniform(largest == -__builtin_inff() ? 0.f : largest)) {
        refc = uniform(ref * c);
        one_fma = fabsf(refc) <= 0x1p16f;
    }
    // (x - ref) c, whichever form the row takes
    __device__ __forceinline__ float difference(float x) const {
        return (x - ref) * c;
    }
    // (x - ref) / 2, which does not overflow where x - ref does
    __device__ __forceinline__ float half_difference(float x) const {
        return __builtin_fmaf(x, 0.5f, -0.5f * ref);
    }
    // walk(t, each): a walk over the row with its form of t.
    template <typename R, typename F>
    __device__ __forceinline__ void with_t(R& row, F walk) const {
        if (one_fma)
            walk([this](float x) { return __builtin_fmaf(x, c, -refc); },
                 [&row](auto f) { row.each(f); });
        else
            walk([this](float x) { return difference(x); },
                 [&row](auto f) { row.template each<true>(f); });
    }
    // The largest's t: what the form moves every t by.
    __device__ __forceinline__ float largest_t() const {
        return one_fma ? __builtin_fmaf(ref, c, -refc) : 0.f;
    }
    // log2 of sum 2^((x - ref) c), from s = the sum of 2^t: 0 or more, and
    // exactly 0 where none counts beside the largest.
    __device__ __forceinline__ float log2_sum(float s) const {
        const float t = largest_t();
        return s == __builtin_amdgcn_exp2f(t) ? 0.f
                                              : larger(__log2f(s) - t, 0.f);
    }
};

}  // namespace rwkv7m
