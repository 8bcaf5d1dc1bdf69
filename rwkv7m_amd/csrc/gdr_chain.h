// What the gated delta rule's two recurrences over chunks share
// (gdr_forward.hip, gdr_backward.hip).
//
// A recurrence acts on each row of the state by itself (row i uses only
// element i of v or do), so a wave owns 16 rows, all of the state's columns,
// in accumulator registers for the whole sequence, and needs nothing from
// another wave.  One, two or four such waves make a workgroup, with four more
// that bring what a chunk needs (K, Q, T, P, the gates, V or dO) from memory
// through their registers to LDS, one chunk ahead of its use and two ahead with
// their loads.  The owning waves then wait for no load at all: where they
// brought their own operands, each wait for one was also a wait for every store
// before it, and a chunk took 14 us.
#pragma once

#include <type_traits>

#include "gdr_common.h"

namespace rwkv7m {
namespace gdr {

constexpr int BRING = 256;  // threads that bring

// 64 columns of a chunk's V or dO.
template <typename E>
struct Columns;
template <>
struct Columns<bf16_t> {
    Rows<1, 2> x;
    // [spread(tb, 4q + e)][16 wave + r]
    __device__ __forceinline__ f32x4_t values(int tb, int wave,
                                              int lane) const {
        return x.values(spread(tb, 4 * (lane >> 4)), wave, lane);
    }
    __device__ __forceinline__ void put(int row, int col,
                                        const Eight<bf16_t>& v) {
        *reinterpret_cast<u32x4_t*>(&x.x[0][row][col]) = v.a;
    }
};
template <>
struct Columns<float> {
    alignas(16) float x[C][68];
    __device__ __forceinline__ f32x4_t values(int tb, int wave,
                                              int lane) const {
        const int r = lane & 15, q = lane >> 4;
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = x[spread(tb, 4 * q + e)][16 * wave + r];
        return v;
    }
    __device__ __forceinline__ void put(int row, int col,
                                        const Eight<float>& v) {
        *reinterpret_cast<f32x4_t*>(&x[row][col]) = v.a;
        *reinterpret_cast<f32x4_t*>(&x[row][col + 4]) = v.b;
    }
};

// A chunk's X or dR of the lane's column, 64 rows of `pitch` floats: uniform
// row addresses and one 32-bit lane offset.
__device__ __forceinline__ void put_column(float* to, int pitch, int q, int v,
                                           const f32x4_t (&x)[4]) {
    const uint32_t lane = uint32_t(8 * q * pitch + v);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        (to + spread(i >> 2, i & 3) * pitch)[lane] = x[i >> 2][i & 3];
}

struct NoColumns {};

// (fp32 at 128 columns leaves no room for the 64 columns in LDS)
template <typename E, int KT>
constexpr bool kColumns = sizeof(E) == 2 || KT < 4;

template <typename E, int KT>
struct ChainChunk {
    Rows<kIn<E>, KT> k, q;
    Matrices m;
    std::conditional_t<kColumns<E, KT>, Columns<E>, NoColumns> v;
    alignas(16) float first[C], last[C], beta[C];
};
static_assert(sizeof(ChainChunk<float, 4>) <= 160 * 1024, "");
// One chunk ahead in a second buffer where two fit.
template <typename E, int KT>
constexpr int kBuffers = 2 * sizeof(ChainChunk<E, KT>) <= 160 * 1024 ? 2 : 1;

// The owning lane's column of V or dO: from LDS, or brought by itself, a chunk
// ahead of its use.
template <typename E, int KT>
struct OwnColumn {
    const E* base;  // (token 0)
    int64_t stride, T;
    bool on;
    E next[16];

    __device__ __forceinline__ OwnColumn(const GdrArgs& A, const GdrTensor& x,
                                         int64_t b, int64_t h, int v)
        : base(at<E>(x, b, h, 0) + near(v, A.Dv - 1)), stride(x.st), T(A.T),
          on(v < A.Dv) {}
    static __device__ __forceinline__ int64_t token(int64_t c, int i,
                                                    int lane) {
        return c * C + spread(i >> 2, 4 * (lane >> 4) + (i & 3));
    }
    __device__ __forceinline__ void fetch(int64_t c, int lane) {
        if constexpr (!kColumns<E, KT>)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t t = token(c, i, lane);
                next[i] = base[(t < 0 ? 0 : t < T ? t : T - 1) * stride];
            }
    }
    // The chunk's values, with the loads of chunk `then`, if any, begun.
    __device__ __forceinline__ void take(const ChainChunk<E, KT>& L, int64_t c,
                                         int64_t then, int wave, int lane,
                                         f32x4_t (&x)[4]) {
        if constexpr (kColumns<E, KT>) {
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) x[tb] = L.v.values(tb, wave, lane);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x[i >> 2][i & 3] =
                    on && token(c, i, lane) < T ? load_f(&next[i]) : 0.f;
            fetch(then, lane);
        }
    }
};

// A bringing thread's share of a chunk, for OW owning waves.
template <typename E, int KT, int OW>
struct Bring {
    Staged<E, KT, BRING> k, q;
    static constexpr int pieces = sizeof(Matrices) / 16 / BRING;
    static_assert(pieces * 16 * BRING == sizeof(Matrices), "");
    u32x4_t m[pieces];
    static constexpr int per_row = 2 * OW, turns = (OW + 1) / 2;
    Eight<E> v[turns];
    float first, last, beta;

    // (v0: the workgroup's first column; x: V or dO)
    __device__ __forceinline__ void load(const GdrArgs& A, const GdrTensor& x,
                                         const Prepared& M, int64_t b,
                                         int64_t h, int64_t hk, int64_t c,
                                         int v0, int thread) {
        const int64_t t0 = c * C;
        const int valid = int(A.T - t0 < C ? A.T - t0 : C);
        k.load(at<E>(A.k, b, hk, t0), A.k.st, valid, A.Dk, thread);
        q.load(at<E>(A.q, b, hk, t0), A.q.st, valid, A.Dk, thread);
#pragma unroll
        for (int i = 0; i < pieces; ++i)
            m[i] = reinterpret_cast<const u32x4_t*>(&M.m)[i * BRING + thread];
        if constexpr (kColumns<E, KT>)
#pragma unroll
            for (int i = 0; i < turns; ++i) {
                const int u = i * BRING + thread;
                v[i].load(at<E>(x, b, h, t0 + near(u / per_row, valid - 1)) +
                          near(v0 + 8 * (u % per_row), A.Dv - 8));
            }
        first = M.first[thread & 63];
        last = M.last[thread & 63];
        beta = M.beta[thread & 63];
    }
    __device__ __forceinline__ void store(const GdrArgs& A, ChainChunk<E, KT>& L,
                                          int64_t c, int v0,
                                          int thread) const {
        const int valid = int(A.T - c * C < C ? A.T - c * C : C);
        k.store(L.k, valid, A.Dk, thread);
        q.store(L.q, valid, A.Dk, thread);
#pragma unroll
        for (int i = 0; i < pieces; ++i)
            reinterpret_cast<u32x4_t*>(&L.m)[i * BRING + thread] = m[i];
        if constexpr (kColumns<E, KT>)
#pragma unroll
            for (int i = 0; i < turns; ++i) {
                const int u = i * BRING + thread;
                const int row = u / per_row, col = 8 * (u % per_row);
                Eight<E> x = v[i];
                x.keep(row < valid && v0 + col < A.Dv);
                if (row < C) L.v.put(row, col, x);
            }
        if (thread < C) {
            L.first[thread] = first;
            L.last[thread] = last;
            L.beta[thread] = beta;
        }
    }
};

// The six operands of T or P (or of their transposes) that hold anything, in
// the order (0, 0) .. (3, 0), (2, 1), (3, 1); transposed (0, 0), (1, 0), (0, 1)
// .. (3, 1).
template <bool TRANSPOSED>
__device__ __forceinline__ void triangle(const Triangle& x, int lane,
                                         Frag<kMade> (&f)[6]) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const int tb = TRANSPOSED ? i < 2 ? i : i - 2 : i < 4 ? i : i - 2;
        const int p = TRANSPOSED ? i >= 2 : i >= 4;
        f[i] = TRANSPOSED ? x.columns(tb, p, lane) : x.rows(tb, p, lane);
    }
}
// acc[tb] += (that matrix) f, f[p] the operand of pair p.
template <bool TRANSPOSED, int NC, int NB>
__device__ __forceinline__ void mul_triangle(f32x4_t (&acc)[4],
                                             const Frag<NC> (&m)[6],
                                             const Frag<NB> (&f)[2]) {
    constexpr int most = NC > NB ? NC : NB;
#pragma unroll
    for (int s = most - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int j = s - i;
            if (j < 0 || j >= NB) continue;
#pragma unroll
            for (int n = 0; n < 6; ++n) {
                const int tb = TRANSPOSED ? n < 2 ? n : n - 2 : n < 4 ? n : n - 2;
                const int p = TRANSPOSED ? n >= 2 : n >= 4;
                acc[tb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, m[n].p[i]),
                    __builtin_bit_cast(bf16x8_t, f[p].p[j]), acc[tb], 0, 0, 0);
            }
        }
}
// acc[tb] += f (that matrix)^T, f[p] the left operand.
template <int NC, int NA>
__device__ __forceinline__ void mul_by_triangle(f32x4_t (&acc)[4],
                                                const Frag<NA> (&f)[2],
                                                const Frag<NC> (&m)[6]) {
    constexpr int most = NC > NA ? NC : NA;
#pragma unroll
    for (int s = most - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = s - i;
            if (j < 0 || j >= NC) continue;
#pragma unroll
            for (int n = 0; n < 6; ++n) {
                const int tb = n < 4 ? n : n - 2, p = n >= 4;
                acc[tb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, f[p].p[i]),
                    __builtin_bit_cast(bf16x8_t, m[n].p[j]), acc[tb], 0, 0, 0);
            }
        }
}

// The four token blocks' operands of pair p.
template <int NI, int KT>
__device__ __forceinline__ void blocks(const Rows<NI, KT>& x, int p, int lane,
                                       Frag<NI> (&f)[4]) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb) f[tb] = x.rows(tb, p, lane);
}
// The operands of four column blocks from 4 n on, of pair p of tokens.
template <int NI, int KT>
__device__ __forceinline__ void column_blocks(const Rows<NI, KT>& x, int n,
                                              int p, int lane,
                                              Frag<NI> (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = x.columns(4 * n + i, p, lane);
}

// The loop of both: chunks first, first + step, .. (n of them).  own(L, c) by
// the threads that own rows, with the chunk in L.
template <typename E, int KT, int OW, typename F>
__device__ __forceinline__ void chain(const GdrArgs& A, const GdrTensor& x,
                                      const Prepared* M, int64_t head,
                                      int v0, int64_t first, int64_t step,
                                      int64_t n, ChainChunk<E, KT>* L, F own) {
    const Head at_head(A, uint32_t(head));
    const int64_t b = at_head.b, h = at_head.h, hk = at_head.hk;
    constexpr int NB = kBuffers<E, KT>;
    if (threadIdx.x >= 64 * OW) {
        const int thread = threadIdx.x - 64 * OW;
        Bring<E, KT, OW> s;
        s.load(A, x, M[first], b, h, hk, first, v0, thread);
        s.store(A, L[0], first, v0, thread);
        const auto ahead = [&](int64_t i) {
            const int64_t c = first + step * i;
            if (i < n) s.load(A, x, M[c], b, h, hk, c, v0, thread);
        };
        ahead(1);
        __syncthreads();
        for (int64_t i = 0; i < n; ++i) {
            if constexpr (NB == 1) __syncthreads();
            if (i + 1 < n) {
                s.store(A, L[NB == 2 ? (i + 1) & 1 : 0],
                        first + step * (i + 1), v0, thread);
                ahead(i + 2);
            }
            __syncthreads();
        }
    } else {
        // (the owning waves' step is what the others wait for)
        __builtin_amdgcn_s_setprio(2);
        __syncthreads();
        for (int64_t i = 0; i < n; ++i) {
            own(L[NB == 2 ? i & 1 : 0], first + step * i);
            if constexpr (NB == 1) __syncthreads();
            __syncthreads();
        }
    }
}

// Owning waves of a workgroup: as few as leave no more workgroups than CUs,
// and four beyond, since every workgroup brings its own K, Q, T and P and a
// CU's workgroups share its LDS.  Forward, us with one, two and four (* the
// rule's), bf16:
//   1 x 1999 tokens, 32 heads of 128 x 128  103 *  101.5   105
//   8 x 512, 12 of 64 x 64                   48     28 *    29
//   2 x 1001, 24 of 96 x 128                112     62 *    69
//   8 x 4096, 16 of 128 x 128               898    578     400 *
inline int owning_waves(int64_t heads, int dvp) {
    for (int w = 1; w < 4; w *= 2)
        if (heads * ((dvp + 16 * w - 1) / (16 * w)) <= device_cus()) return w;
    return 4;
}

}  // namespace gdr
}  // namespace rwkv7m
