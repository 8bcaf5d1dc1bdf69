// Pieces shared by the gated delta rule's chunk kernels (gdr_prepare.hip,
// gdr_forward.hip, gdr_backward.hip, gdr_gradients.hip).
//
// A chunk is 64 tokens.  Within it, with G the running sum of the log decays
// (in base 2, float64: E is formed from differences of sums that far tokens
// make long), S0 the state before it, [Dv][Dk]:
//
//   E_ts = 2^(G_t - G_s),  A = tril(beta_t E_ts k_t.k_s, -1),  T = (I + A)^-1
//   R = beta (V - 2^G (K S0^T)),  X = T R
//   O = scale (2^G (Q S0^T) + P X),  P = tril(E_ts q_t.k_s)
//   S_L = 2^G_L S0 + (2^(G_L - G) X)^T K
//
// Operands.  All products run on v_mfma_f32_16x16x32_bf16 with fp32 sums.  A
// number of more bits is a sum of bf16 planes, and a product the sum of the
// planes' products that count: bf16 q, k, v and do are one plane (exact), fp32
// ones and all that is computed, the state among it, three (2^-27 left out,
// less than fp32 sums round off).  Two planes for what is computed from bf16
// vectors leave out 2^-18: the final state, an fp32 output, was 4.5e-6 off (its
// norm) where fp32 products and three planes are 2e-7, and bf16 results, some of
// them rounded the other way, 1.4e-4 from those of fp32 products for 3.5e-5.
// They took 92 us for 116 (1 x 1999 tokens, 32 heads of 128 x 128), 1486 for
// 1567 (8 x 4096 with gradients, 16 of 128 x 128).
//
// Register layouts (lane l, r = l % 16, q = l / 16).  An accumulator tile D(X)
// holds X[4q + e][r], e = 0..3.  An operand of 32 places along the contracted
// axis holds X[r][32 p + 8q + i] in its slots i = 0..7, 16 bytes of a row of
// memory; the same registers are X as the left operand and X^T as the right
// one.  So that two accumulator tiles are such an operand without a move, the
// tiles of a pair share its 32 places: row (or column) m of tile 2p + u is
// place 32 p + 8 (m / 4) + 4 u + m % 4 (spread()).  Taken in their natural
// order they would be read from LDS in pairs of 8 bytes, at a quarter of the
// rate (8.1 cycles of the LDS each, where 16 bytes take 4.2).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wkv7_common.h"
#include "wkv7_launch.h"

namespace rwkv7m {
namespace gdr {

constexpr int C = kGdrChunk;
constexpr double kLog2e = 1.4426950408889634;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

template <typename E>
constexpr int kIn = sizeof(E) == 2 ? 1 : 3;  // planes of an input
constexpr int kMade = 3;                      // of a computed number

template <int N>
struct Frag {
    u32x4_t p[N];
};

__device__ __forceinline__ f32x4_t zero4() { return f32x4_t{0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t f = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
}

// Two floats to N planes, a packed pair each.  (A plane that is not finite
// leaves NaN in the next: such numbers make NaN of their products.)
template <int N>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&out)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        out[n] = pack2(a, b);
        if (n + 1 < N) {
            a -= __uint_as_float(out[n] << 16);
            b -= __uint_as_float(out[n] & 0xffff0000u);
        }
    }
}

// Slots 0..3 from a, 4..7 from b.
template <int N>
__device__ __forceinline__ Frag<N> split8(const f32x4_t& a, const f32x4_t& b) {
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t u[N];
        if (i < 2)
            split2<N>(a[2 * i], a[2 * i + 1], u);
        else
            split2<N>(b[2 * i - 4], b[2 * i - 3], u);
#pragma unroll
        for (int n = 0; n < N; ++n) f.p[n][i] = u[n];
    }
    return f;
}

// acc += a b over 32 places, the small planes' products first.
template <int NA, int NB>
__device__ __forceinline__ void mul(f32x4_t& acc, const Frag<NA>& a,
                                    const Frag<NB>& b) {
    constexpr int most = NA > NB ? NA : NB;
#pragma unroll
    for (int s = most - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = s - i;
            if (j < 0 || j >= NB) continue;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, a.p[i]),
                __builtin_bit_cast(bf16x8_t, b.p[j]), acc, 0, 0, 0);
        }
}

// acc[m] += a[m] b for M independent sums in turn, so that none waits for the
// product before it.
template <int M, int NA, int NB>
__device__ __forceinline__ void mul_each(f32x4_t (&acc)[M],
                                         const Frag<NA> (&a)[M],
                                         const Frag<NB>& b) {
    constexpr int most = NA > NB ? NA : NB;
#pragma unroll
    for (int s = most - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = s - i;
            if (j < 0 || j >= NB) continue;
#pragma unroll
            for (int m = 0; m < M; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, a[m].p[i]),
                    __builtin_bit_cast(bf16x8_t, b.p[j]), acc[m], 0, 0, 0);
        }
}
// The same with the sums' operand on the right.
template <int M, int NA, int NB>
__device__ __forceinline__ void mul_each(f32x4_t (&acc)[M], const Frag<NA>& a,
                                         const Frag<NB> (&b)[M]) {
    constexpr int most = NA > NB ? NA : NB;
#pragma unroll
    for (int s = most - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = s - i;
            if (j < 0 || j >= NB) continue;
#pragma unroll
            for (int m = 0; m < M; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, a.p[i]),
                    __builtin_bit_cast(bf16x8_t, b[m].p[j]), acc[m], 0, 0, 0);
        }
}
// Nothing is moved over this place: operands are read from LDS where they are
// written to be, ahead of the products that hide their way.
__device__ __forceinline__ void hold() { __builtin_amdgcn_sched_barrier(0); }

// Between two hold(): N products, each followed by D reads of LDS and V other
// vector instructions, as far as there are any.  A wave issues in order, a
// product every 16 cycles and a read of LDS no faster: what stands behind a
// row of either waits for all of it.
template <int N, int D, int V>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (D > 0) __builtin_amdgcn_sched_group_barrier(0x100, D, 0);
        if constexpr (V > 0) __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    }
}

__device__ __forceinline__ float exp2_of(double x) {
    return __builtin_amdgcn_exp2f(float(x));
}

// --- memory -----------------------------------------------------------------

// Eight adjoining elements of a row as they are held in memory, at 16-byte
// aligned addresses.  A row's places past Dk or Dv, and rows past T, are 0:
// they are loaded from the nearest place that there is and cleared when the
// value is used (keep).  A load under a condition has its register merged with
// the zeros behind the branch, and is waited for there and then.
template <typename E>
struct Eight;
template <>
struct Eight<bf16_t> {
    u32x4_t a;
    __device__ __forceinline__ void load(const bf16_t* p) {
        a = *reinterpret_cast<const u32x4_t*>(p);
    }
    __device__ __forceinline__ void keep(bool on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = on ? a[i] : 0u;
    }
    __device__ __forceinline__ Frag<1> planes() const { return {{a}}; }
    __device__ __forceinline__ float get(int i) const {
        return __uint_as_float(i & 1 ? a[i >> 1] & 0xffff0000u : a[i >> 1] << 16);
    }
};
template <>
struct Eight<float> {
    f32x4_t a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const f32x4_t*>(p);
        b = *reinterpret_cast<const f32x4_t*>(p + 4);
    }
    __device__ __forceinline__ void keep(bool on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = on ? a[i] : 0.f;
            b[i] = on ? b[i] : 0.f;
        }
    }
    __device__ __forceinline__ Frag<3> planes() const { return split8<3>(a, b); }
    __device__ __forceinline__ float get(int i) const {
        return i < 4 ? a[i] : b[i - 4];
    }
};

// Place of row m of tile t.
__device__ __forceinline__ int spread(int t, int m) {
    return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3);
}

// R rows of 32 KT places in LDS, NP planes.  With this pitch 16 rows' 16-byte
// pieces lie on different banks.
template <int NP, int KT, int R = C>
struct Rows {
    static constexpr int pitch = 32 * KT + 8;
    bf16_t x[NP][R][pitch];

    // The operand of rows `row` (the lane's), places 32 p ...
    __device__ __forceinline__ Frag<NP> at_row(int row, int p, int q) const {
        Frag<NP> f;
#pragma unroll
        for (int n = 0; n < NP; ++n)
            f.p[n] =
                *reinterpret_cast<const u32x4_t*>(&x[n][row][32 * p + 8 * q]);
        return f;
    }
    // .. of tile tb's rows, spread or in their order
    __device__ __forceinline__ Frag<NP> rows(int tb, int p, int lane) const {
        return at_row(spread(tb, lane & 15), p, lane >> 4);
    }
    __device__ __forceinline__ Frag<NP> rows_in_order(int tb, int p,
                                                      int lane) const {
        return at_row(16 * tb + (lane & 15), p, lane >> 4);
    }
    // X[row + e][..] of the column that each lane's place in its group of 16
    // gives: the lane reads four columns from `col` of row `row` + s / 4.
    __device__ __forceinline__ uint2 turned(int n, int row, int col,
                                            int lane) const {
        const bf16_t* p = &x[n][row + ((lane & 15) >> 2)][col];
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (lds_i16x4_t*)(p)));
    }
    // The operand of columns `col`.. (as `turned`), over the 32 rows of pair p:
    // left, rows of the transpose; right, x itself.
    __device__ __forceinline__ Frag<NP> at_column(int col, int p,
                                                  int lane) const {
        const int row = 32 * p + 8 * (lane >> 4);
        Frag<NP> f;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const uint2 lo = turned(n, row, col, lane);
            const uint2 hi = turned(n, row + 4, col, lane);
            f.p[n] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
        }
        return f;
    }
    // .. of tile jb's columns, spread or in their order
    __device__ __forceinline__ Frag<NP> columns(int jb, int p, int lane) const {
        return at_column(32 * (jb >> 1) + 8 * (lane & 3) + 4 * (jb & 1), p,
                         lane);
    }
    __device__ __forceinline__ Frag<NP> columns_in_order(int jb, int p,
                                                         int lane) const {
        return at_column(16 * jb + 4 * (lane & 3), p, lane);
    }
    // X[row + e][16 jb + r] as floats (row: the lane's first of four).
    __device__ __forceinline__ f32x4_t values(int row, int jb, int lane) const {
        f32x4_t v = zero4();
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) {
            const uint2 u = turned(n, row, 16 * jb + 4 * (lane & 3), lane);
            v[0] += __uint_as_float(u.x << 16);
            v[1] += __uint_as_float(u.x & 0xffff0000u);
            v[2] += __uint_as_float(u.y << 16);
            v[3] += __uint_as_float(u.y & 0xffff0000u);
        }
        return v;
    }
};

// Four floats as planes at four adjoining places.
template <int NP, int KT, int R>
__device__ __forceinline__ void put4(Rows<NP, KT, R>& to, int row, int col,
                                     const f32x4_t& x) {
    uint32_t lo[NP], hi[NP];
    split2<NP>(x[0], x[1], lo);
    split2<NP>(x[2], x[3], hi);
#pragma unroll
    for (int n = 0; n < NP; ++n)
        *reinterpret_cast<uint2*>(&to.x[n][row][col]) =
            make_uint2(lo[n], hi[n]);
}

__device__ __forceinline__ int near(int i, int most) {
    return i < most ? i : most;
}

// The share of a chunk's rows of one of `T` threads, on its way to LDS.
template <typename E, int KT, int T>
struct Staged {
    static constexpr int per_row = 4 * KT, n = C * per_row / T;
    Eight<E> v[n];

    // Rows 0 .. valid - 1 of `base`, `dim` places each.
    __device__ __forceinline__ void load(const E* base, int64_t stride,
                                         int valid, int dim, int thread) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int u = i * T + thread;
            v[i].load(base + near(u / per_row, valid - 1) * stride +
                      near(8 * (u % per_row), dim - 8));
        }
    }
    __device__ __forceinline__ void store(Rows<kIn<E>, KT>& to, int valid,
                                          int dim, int thread) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int u = i * T + thread;
            const int row = u / per_row, col = 8 * (u % per_row);
            Eight<E> x = v[i];
            x.keep(row < valid && col < dim);
            const auto f = x.planes();
#pragma unroll
            for (int m = 0; m < kIn<E>; ++m)
                *reinterpret_cast<u32x4_t*>(&to.x[m][row][col]) = f.p[m];
        }
    }
};

// --- what gdr_prepare.hip leaves for a chunk of a head ------------------------

// A lower triangle of 64 x 64 as the six operands of 16 rows and 32 places that
// hold anything, (tb, p) = (0, 0) .. (3, 0), (2, 1), (3, 1): rows spread(tb, r),
// places 32 p + 8q .., lane by lane.  (Row by row, with a pitch that spreads the
// banks, three planes of two triangles would take half as much again and leave
// no room for a second chunk in LDS.)
struct Triangle {
    alignas(16) bf16_t x[kMade][6][64][8];

    static __device__ __forceinline__ constexpr int operand(int tb, int p) {
        return tb + 2 * p;
    }
    __device__ __forceinline__ bf16_t* at(int n, int row, int col) {
        const int tb = 2 * (row / 32) + (row >> 2 & 1);
        const int m = 4 * (row % 32 / 8) + (row & 3);
        return &x[n][operand(tb, col / 32)][16 * (col % 32 / 8) + m][col % 8];
    }
    __device__ __forceinline__ Frag<kMade> rows(int tb, int p, int lane) const {
        Frag<kMade> f;
#pragma unroll
        for (int n = 0; n < kMade; ++n)
            f.p[n] = *reinterpret_cast<const u32x4_t*>(
                &x[n][operand(tb, p)][lane][0]);
        return f;
    }
    // The operand of the transpose's rows spread(jb, r), places 32 p ..: rows
    // 8q + (r >> 2) and four further of pair p, whose tiles are 2 p and 2 p + 1,
    // four columns a lane, transposed on the way.
    __device__ __forceinline__ Frag<kMade> columns(int jb, int p,
                                                   int lane) const {
        const int slot = 16 * (lane & 3) + 4 * (lane >> 4) + (lane >> 2 & 3);
        Frag<kMade> f;
#pragma unroll
        for (int n = 0; n < kMade; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf16_t* from =
                    &x[n][operand(2 * p + u, jb >> 1)][slot][4 * (jb & 1)];
                const uint2 w = __builtin_bit_cast(
                    uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (lds_i16x4_t*)(from)));
                f.p[n][2 * u] = w.x;
                f.p[n][2 * u + 1] = w.y;
            }
        return f;
    }
};
struct Matrices {
    Triangle t, p;
};

// The matrices and the gates.
struct Prepared {
    Matrices m;
    double G[C];                          // base 2
    float first[C], last[C], beta[C];     // 2^G, 2^(G_L - G)
};

__device__ __forceinline__ f32x4_t four(const float* p) {
    return *reinterpret_cast<const f32x4_t*>(p);
}

// Sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float sum16(float x) { return group_sum<16>(x); }

// A head's workgroups on one of the 8 XCDs (consecutive workgroups go to
// different ones), so that they share its L2: workgroup `id` of head and part.
struct Place {
    uint32_t head;
    int part;
};
__device__ __forceinline__ Place place(uint32_t id, uint32_t parts) {
    const uint32_t xcd = id % 8, slot = id / 8;
    return {slot / parts * 8 + xcd, int(slot % parts)};
}
inline unsigned places(int64_t heads, int64_t parts) {
    return unsigned((heads + 7) / 8 * 8 * parts);
}

// Batch row, value head and key head of head `id` of B * Hv (fewer than 2^24:
// a 64-bit division is 130 instructions).
struct Head {
    uint32_t b, h, hk;
    __device__ __forceinline__ Head(const GdrArgs& A, uint32_t id)
        : b(id / uint32_t(A.Hv)), h(id % uint32_t(A.Hv)),
          hk(h / (uint32_t(A.Hv) / uint32_t(A.Hk))) {}
};
__device__ __forceinline__ uint32_t chunk_count(const GdrArgs& A) {
    return uint32_t((A.T + C - 1) / C);
}

template <typename E>
__device__ __forceinline__ const E* at(const GdrTensor& t, int64_t b, int64_t h,
                                       int64_t token) {
    return static_cast<const E*>(t.p) + b * t.sb + h * t.sh + token * t.st;
}

}  // namespace gdr
}  // namespace rwkv7m
