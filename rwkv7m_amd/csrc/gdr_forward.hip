// The gated delta rule's recurrence over chunks (gdr_common.h has the
// formulas, gdr_chain.h the division of work): outputs, and the state before
// each chunk and X where a backward follows.
//
// With few heads bound by the way through a chunk, one after the other: 32
// heads of 128 x 128 over 1999 tokens 103 us, 3.2 a chunk, of which a wave's
// 216 matrix instructions are half.  With many, where states and X are kept, by
// memory: 8 x 4096 tokens, 16 heads of 128 x 128, move 1.65 GB in 358 to 400
// us, 4.1 to 4.6 TB/s.
#include "gdr_chain.h"

namespace rwkv7m {
namespace {

using namespace gdr;

template <typename E, int KT, int OW, bool TRAIN>
__global__ void __launch_bounds__(64 * OW + BRING)
__attribute__((amdgpu_waves_per_eu(2, 2)))
gdr_forward_kernel(const GdrArgs A, int parts) {
    constexpr int NI = kIn<E>, NC = kMade, DKP = 32 * KT;
    extern __shared__ char lds_raw[];
    const Place at_ = place(blockIdx.x, parts);
    const int64_t head = at_.head;
    if (head >= A.B * A.Hv) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const Head at_head(A, at_.head);
    const int64_t b = at_head.b, h = at_head.h, chunks = chunk_count(A);
    const int DVP = (A.Dv + 31) / 32 * 32;
    const int v0 = 16 * (OW * at_.part + wave), v = v0 + r;  // the lane's row
    const bool has = v0 < DVP, on = v < A.Dv;

    f32x4_t S[2 * KT];  // D(S^T): k = spread(kb, 4q + e), v = r
#pragma unroll
    for (int kb = 0; kb < 2 * KT; ++kb) {
        const int k = spread(kb, 4 * q);
        S[kb] = zero4();
        if (A.s0 && wave < OW && on && k < A.Dk)
            S[kb] = four(A.s0 + (head * A.Dv + v) * A.Dk + k);
    }
    E* op = static_cast<E*>(A.o) + (b * A.T * A.Hv + h) * A.Dv;
    OwnColumn<E, KT> column(A, A.v, b, h, v);
    column.fetch(0, lane);

    chain<E, KT, OW>(
        A, A.v, static_cast<const Prepared*>(A.prepared) + head * chunks,
        head, 16 * OW * at_.part, 0, 1, chunks,
        reinterpret_cast<ChainChunk<E, KT>*>(lds_raw),
        [&](const ChainChunk<E, KT>& L, int64_t c) {
        if (!has) return;
        const int64_t t0 = c * C;
        const int valid = int(A.T - t0 < C ? A.T - t0 : C);
        // What follows is in the order in which it is issued: each step's
        // operands are read from LDS between the products of the step before,
        // and so is what the vector ALU has to do and they do not need.
        // (bf16: three planes of fp32 vectors leave no registers for it.)
        constexpr bool DEEP = NI == 1;
        constexpr int TWO = DEEP ? 2 : 1, HALF = KT / 2;
        Frag<NI> kf[TWO][4], qf[TWO][4];
        Frag<NC> Tf[6], Pf[6], Sf[KT], Rf[2], Xf[2];
        f32x4_t V[4], first[4], beta[4], B0[4], O[4], X[4];
        const float whole = L.first[C - 1];
        if (DEEP) blocks(L.k, 0, lane, kf[0]);
        column.take(L, c, c + 1, wave, lane, V);
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) B0[tb] = O[tb] = X[tb] = zero4();
        if constexpr (TRAIN) {
            float* to = A.states + ((head * chunks + c) * DVP + v) * DKP;
#pragma unroll
            for (int kb = 0; kb < 2 * KT; ++kb)
                *reinterpret_cast<f32x4_t*>(to + spread(kb, 4 * q)) = S[kb];
        }
        Sf[0] = split8<NC>(S[0], S[1]);
        // K S^T, t = spread(tb, 4q + e), v = r
#pragma unroll
        for (int p = 0; p < KT; ++p) {
            if (DEEP) hold();
            if (!DEEP) {
                blocks(L.k, p, lane, kf[0]);
            } else if (p + 1 < KT) {
                blocks(L.k, p + 1, lane, kf[(p + 1) % TWO]);
            } else {
                blocks(L.q, 0, lane, qf[0]);
            }
            if (p + 1 == KT)
#pragma unroll
                for (int tb = 0; tb < 4; ++tb) {
                    first[tb] = four(L.first + spread(tb, 4 * q));
                    beta[tb] = four(L.beta + spread(tb, 4 * q));
                }
            if (!DEEP) hold();
            mul_each(B0, kf[p % TWO], Sf[p]);
            if (p + 1 < KT)
                Sf[p + 1] = split8<NC>(S[2 * p + 2], S[2 * p + 3]);
            if (DEEP && p + 1 < KT) interleave<4 * NC, 1, 3>();
            if (DEEP && p + 1 == KT) interleave<4 * NC, 2, 0>();
        }
        // S Q^T, v = 4q + e, t = spread(tb, r), and meanwhile
        const auto queries = [&](int p) {
            if (DEEP) hold();
            if (!DEEP) blocks(L.q, p, lane, qf[0]);
            else if (p + 1 < KT) blocks(L.q, p + 1, lane, qf[(p + 1) % TWO]);
            else column_blocks(L.k, 0, 0, lane, kf[0]);
            if (DEEP && p + 1 == HALF) triangle<false>(L.m.t, lane, Tf);
            if (!DEEP) hold();
            mul_each(O, Sf[p], qf[p % TWO]);
        };
        // R = beta (V - 2^G (K S^T))
#pragma unroll
        for (int p = 0; p < HALF; ++p) {
            queries(p);
#pragma unroll
            for (int i = 4 * p / HALF; i < 4 * (p + 1) / HALF; ++i)
                V[i] = beta[i] * (V[i] - first[i] * B0[i]);
#pragma unroll
            for (int i = 2 * p / HALF; i < 2 * (p + 1) / HALF; ++i)
                Rf[i] = split8<NC>(V[2 * i], V[2 * i + 1]);
            if (DEEP && p + 1 < HALF) interleave<4 * NC, 1, 6>();
            if (DEEP && p + 1 == HALF) interleave<4 * NC, 2, KT == 2 ? 20 : 8>();
        }
        // X = T R
        f32x4_t last[4];
        float own_first[4];
        if (!DEEP) triangle<false>(L.m.t, lane, Tf);
        hold();
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
            last[tb] = four(L.last + spread(tb, 4 * q));
            own_first[tb] = L.first[spread(tb, r)];
        }
        mul_triangle<false>(X, Tf, Rf);
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) S[kb] *= whole;
        if (DEEP) interleave<36, 1, 2>();
#pragma unroll
        for (int p = HALF; p < KT; ++p) {
            queries(p);
#pragma unroll
            for (int i = 2 * (p - HALF) / HALF; i < 2 * (p - HALF + 1) / HALF;
                 ++i) {
                Rf[i] = split8<NC>(X[2 * i] * last[2 * i],
                                   X[2 * i + 1] * last[2 * i + 1]);
                Xf[i] = split8<NC>(X[2 * i], X[2 * i + 1]);
            }
            if (DEEP) interleave<4 * NC, 1, KT == 2 ? 16 : 7>();
        }
        if constexpr (TRAIN) {
            put_column(A.x + (head * chunks + c) * C * DVP, DVP, q, v, X);
        }
        // S^T = 2^G_L S^T + K^T (2^(G_L - G) X)
#pragma unroll
        for (int n = 0; n < KT / 2; ++n) {
            f32x4_t sum[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = S[4 * n + i];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int at = 2 * n + p;
                if (DEEP) hold();
                if (!DEEP)
                    column_blocks(L.k, n, p, lane, kf[0]);
                else if (at + 1 < KT)
                    column_blocks(L.k, (at + 1) / 2, (at + 1) & 1, lane,
                                  kf[(at + 1) % TWO]);
                else
                    triangle<false>(L.m.p, lane, Pf);
                if (!DEEP) hold();
                mul_each(sum, kf[at % TWO], Rf[p]);
                if (at == 0)
#pragma unroll
                    for (int tb = 0; tb < 4; ++tb) O[tb] *= own_first[tb];
                if (DEEP && at == 0) interleave<4 * NC, 1, 2>();
                if (DEEP && at > 0 && at + 1 < KT) interleave<4 * NC, 1, 0>();
                if (DEEP && at + 1 == KT) interleave<4 * NC, 2, 0>();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) S[4 * n + i] = sum[i];
        }
        // O^T = scale (2^G (S Q^T) + X^T P^T)
        if (!DEEP) triangle<false>(L.m.p, lane, Pf);
        hold();
        mul_by_triangle(O, Xf, Pf);
        E* to = op + t0 * A.Hv * A.Dv + int64_t(spread(0, r)) * A.Hv * A.Dv +
                v0 + 4 * q;
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
            E* at = to + int64_t(spread(tb, 0)) * A.Hv * A.Dv;
            if (spread(tb, r) < valid && v0 + 4 * q < A.Dv) {
                O[tb] *= A.scale;
                if constexpr (sizeof(E) == 4)
                    *reinterpret_cast<f32x4_t*>(at) = O[tb];
                else
                    *reinterpret_cast<uint2*>(at) =
                        make_uint2(pack2(O[tb][0], O[tb][1]),
                                   pack2(O[tb][2], O[tb][3]));
            }
        }
    });
    if (A.s_t && wave < OW && on) {
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            const int k = spread(kb, 4 * q);
            if (k < A.Dk)
                *reinterpret_cast<f32x4_t*>(
                    A.s_t + (head * A.Dv + v) * A.Dk + k) = S[kb];
        }
    }
}

template <typename E, int KT, int OW, bool TRAIN>
hipError_t launch_with(const GdrArgs& A, hipStream_t stream) {
    const auto kernel = gdr_forward_kernel<E, KT, OW, TRAIN>;
    const int lds = int(kBuffers<E, KT> * sizeof(ChainChunk<E, KT>));
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const int parts = (gdr_dvp(A.Dv) + 16 * OW - 1) / (16 * OW);
    hipLaunchKernelGGL(kernel, dim3(places(A.B * A.Hv, parts)),
                       dim3(64 * OW + BRING), lds, stream, A, parts);
    return hipGetLastError();
}

template <typename E, int KT, bool TRAIN>
hipError_t launch(const GdrArgs& A, hipStream_t stream) {
    switch (owning_waves(A.B * A.Hv, gdr_dvp(A.Dv))) {
        case 1: return launch_with<E, KT, 1, TRAIN>(A, stream);
        case 2: return launch_with<E, KT, 2, TRAIN>(A, stream);
        default: return launch_with<E, KT, 4, TRAIN>(A, stream);
    }
}

}  // namespace

hipError_t launch_gdr_forward(bool bf16, const GdrArgs& A,
                              hipStream_t stream) {
    const bool wide = gdr_dkp(A.Dk) == 128, train = A.states != nullptr;
#define RWKV7M_GDR(E)                                                   \
    return wide ? train ? launch<E, 4, true>(A, stream)                 \
                        : launch<E, 4, false>(A, stream)                \
           : train ? launch<E, 2, true>(A, stream)                      \
                   : launch<E, 2, false>(A, stream)
    if (bf16) RWKV7M_GDR(bf16_t);
    RWKV7M_GDR(float);
#undef RWKV7M_GDR
}

}  // namespace rwkv7m
