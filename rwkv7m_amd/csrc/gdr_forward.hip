// The gated delta rule's recurrence over chunks (gdr_common.h has the
// formulas, gdr_chain.h the division of work): outputs, and the state before
// each chunk and X where a backward follows.
#include "gdr_chain.h"

namespace rwkv7m {
namespace {

using namespace gdr;

template <typename E, int KT, bool TRAIN>
__global__ void __launch_bounds__(2 * BRING)
gdr_forward_kernel(const GdrArgs A, int parts) {
    constexpr int NC = kMade<E>, DKP = 32 * KT;
    extern __shared__ char lds_raw[];
    const Place at_ = place(blockIdx.x, parts);
    const int64_t head = at_.head;
    if (head >= A.B * A.Hv) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const Head at_head(A, at_.head);
    const int64_t b = at_head.b, h = at_head.h, chunks = chunk_count(A);
    const int DVP = (A.Dv + 31) / 32 * 32;
    const int v0 = 64 * at_.part + 16 * wave, v = v0 + r;  // the lane's row
    const bool has = v0 < DVP, on = v < A.Dv;

    f32x4_t S[2 * KT];  // D(S^T): k = 16 kb + 4q + e, v = r
#pragma unroll
    for (int kb = 0; kb < 2 * KT; ++kb) {
        const int k = 16 * kb + 4 * q;
        S[kb] = zero4();
        if (A.s0 && wave < 4 && on && k < A.Dk)
            S[kb] = four(A.s0 + (head * A.Dv + v) * A.Dk + k);
    }
    E* op = static_cast<E*>(A.o) + (b * A.T * A.Hv + h) * A.Dv;
    OwnColumn<E, KT> column(A, A.v, b, h, v, wave < 4);
    column.fetch(0, lane);

    chain<E, KT>(
        A, A.v, static_cast<const Prepared<NC>*>(A.prepared) + head * chunks,
        head, 64 * at_.part, 0, 1, chunks,
        reinterpret_cast<ChainChunk<E, KT>*>(lds_raw),
        [&](const ChainChunk<E, KT>& L, int64_t c) {
        if (!has) return;
        const int64_t t0 = c * C;
        const int valid = int(A.T - t0 < C ? A.T - t0 : C);
        Frag<NC> Sf[KT];
#pragma unroll
        for (int p = 0; p < KT; ++p) Sf[p] = split8<NC>(S[2 * p], S[2 * p + 1]);
        if constexpr (TRAIN) {
            float* to = A.states + ((head * chunks + c) * DVP + v) * DKP;
#pragma unroll
            for (int kb = 0; kb < 2 * KT; ++kb)
                *reinterpret_cast<f32x4_t*>(to + 16 * kb + 4 * q) = S[kb];
        }
        // R = beta (V - 2^G (K S^T)), t = 4q + e, v = r
        f32x4_t X[4];
        {
            f32x4_t R[4], V[4];
            column.take(L, c + 1, wave, lane, V);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                f32x4_t acc = zero4();
#pragma unroll
                for (int p = 0; p < KT; ++p)
                    mul(acc, L.k.rows(tb, p, lane), Sf[p]);
                R[tb] = four(L.beta + 16 * tb + 4 * q) *
                        (V[tb] - four(L.first + 16 * tb + 4 * q) * acc);
            }
            // X = T R
            Frag<NC> Rf[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) Rf[p] = split8<NC>(R[2 * p], R[2 * p + 1]);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                X[tb] = zero4();
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    if (holds(false, tb, p))
                        mul(X[tb], L.t.rows(tb, p, lane), Rf[p]);
            }
        }
        if constexpr (TRAIN) {
            float* to = A.x + (head * chunks + c) * C * DVP + v;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                to[(16 * (i >> 2) + 4 * q + (i & 3)) * DVP] = X[i >> 2][i & 3];
        }
        // O^T: v = 4q + e, t = r
        {
            Frag<NC> Xf[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) Xf[p] = split8<NC>(X[2 * p], X[2 * p + 1]);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                f32x4_t acc = zero4();
#pragma unroll
                for (int p = 0; p < KT; ++p)
                    mul(acc, Sf[p], L.q.rows(tb, p, lane));
                acc *= L.first[16 * tb + r];
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    if (holds(false, tb, p))
                        mul(acc, Xf[p], L.p.rows(tb, p, lane));
                const int t = 16 * tb + r, col = v0 + 4 * q;
                if (t < valid && col < A.Dv) {
                    E* to = op + (t0 + t) * A.Hv * A.Dv + col;
                    acc *= A.scale;
                    if constexpr (sizeof(E) == 4)
                        *reinterpret_cast<f32x4_t*>(to) = acc;
                    else
                        *reinterpret_cast<uint2*>(to) =
                            make_uint2(pack2(acc[0], acc[1]),
                                       pack2(acc[2], acc[3]));
                }
            }
        }
        // S^T = 2^G_L S^T + K^T (2^(G_L - G) X)
        const float whole = L.first[C - 1];
        Frag<NC> Xf[2];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) X[tb] *= four(L.last + 16 * tb + 4 * q);
#pragma unroll
        for (int p = 0; p < 2; ++p) Xf[p] = split8<NC>(X[2 * p], X[2 * p + 1]);
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            S[kb] *= whole;
#pragma unroll
            for (int p = 0; p < 2; ++p)
                mul(S[kb], L.k.columns(kb, p, lane), Xf[p]);
        }
    });
    if (A.s_t && wave < 4 && on) {
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            const int k = 16 * kb + 4 * q;
            if (k < A.Dk)
                *reinterpret_cast<f32x4_t*>(
                    A.s_t + (head * A.Dv + v) * A.Dk + k) = S[kb];
        }
    }
}

template <typename E, int KT, bool TRAIN>
hipError_t launch(const GdrArgs& A, hipStream_t stream) {
    const auto kernel = gdr_forward_kernel<E, KT, TRAIN>;
    const int lds = int(kBuffers<E, KT> * sizeof(ChainChunk<E, KT>));
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const int parts = (gdr_dvp(A.Dv) + 63) / 64;
    hipLaunchKernelGGL(kernel, dim3(places(A.B * A.Hv, parts)),
                       dim3(2 * BRING), lds, stream, A, parts);
    return hipGetLastError();
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
