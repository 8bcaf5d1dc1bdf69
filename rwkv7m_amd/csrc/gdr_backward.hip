// The gated delta rule's recurrence backwards over chunks (gdr_chain.h has the
// division of work): the cotangent D of the state after each chunk, and dR,
// from which gdr_gradients.hip forms the gradients, chunk by chunk.
//
//   dX = scale P^T dO + 2^(G_L - G) (K D^T),  dR = T^T dX
//   D <- 2^G_L D + scale (2^G dO)^T Q - (beta 2^G dR)^T K
#include "gdr_chain.h"

namespace rwkv7m {
namespace {

using namespace gdr;

template <typename E, int KT>
__global__ void __launch_bounds__(2 * BRING)
gdr_backward_kernel(const GdrArgs A, int parts) {
    constexpr int NI = kIn<E>, NC = kMade<E>, DKP = 32 * KT;
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

    f32x4_t D[2 * KT];  // D(D^T): k = 16 kb + 4q + e, v = r
#pragma unroll
    for (int kb = 0; kb < 2 * KT; ++kb) {
        const int k = 16 * kb + 4 * q;
        D[kb] = zero4();
        if (A.ds_t && wave < 4 && on && k < A.Dk)
            D[kb] = four(A.ds_t + (head * A.Dv + v) * A.Dk + k);
    }

    OwnColumn<E, KT> column(A, A.dout, b, h, v);
    column.fetch(chunks - 1, lane);

    chain<E, KT>(
        A, A.dout,
        static_cast<const Prepared<NC>*>(A.prepared) + head * chunks, head,
        64 * at_.part, chunks - 1, -1, chunks,
        reinterpret_cast<ChainChunk<E, KT>*>(lds_raw),
        [&](const ChainChunk<E, KT>& L, int64_t c) {
        if (!has) return;
        float* keep = A.dstates + ((head * chunks + c) * DVP + v) * DKP;
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb)
            *reinterpret_cast<f32x4_t*>(keep + 16 * kb + 4 * q) = D[kb];

        f32x4_t dO[4], dX[4], dR[4];
        column.take(L, c, c - 1, wave, lane, dO);
        // dX: t = 4q + e, v = r
        {
            Frag<NI> f[2];
#pragma unroll
            for (int p = 0; p < 2; ++p)
                f[p] = split8<NI>(dO[2 * p], dO[2 * p + 1]);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                dX[tb] = zero4();
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    if (holds(true, tb, p))
                        mul(dX[tb], L.p.columns(tb, p, lane), f[p]);
            }
        }
        {
            Frag<NC> Df[KT];
#pragma unroll
            for (int p = 0; p < KT; ++p)
                Df[p] = split8<NC>(D[2 * p], D[2 * p + 1]);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                f32x4_t acc = zero4();
#pragma unroll
                for (int p = 0; p < KT; ++p)
                    mul(acc, L.k.rows(tb, p, lane), Df[p]);
                dX[tb] = A.scale * dX[tb] +
                         four(L.last + 16 * tb + 4 * q) * acc;
            }
        }
        {
            Frag<NC> f[2];
#pragma unroll
            for (int p = 0; p < 2; ++p)
                f[p] = split8<NC>(dX[2 * p], dX[2 * p + 1]);
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                dR[tb] = zero4();
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    if (holds(true, tb, p))
                        mul(dR[tb], L.t.columns(tb, p, lane), f[p]);
            }
        }
        float* to = A.dr + (head * chunks + c) * C * DVP + v;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            to[(16 * (i >> 2) + 4 * q + (i & 3)) * DVP] = dR[i >> 2][i & 3];

        const float whole = L.first[C - 1];
        Frag<NC> of[2], rf[2];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
            const f32x4_t first = four(L.first + 16 * tb + 4 * q);
            dO[tb] *= A.scale * first;
            dR[tb] *= -(first * four(L.beta + 16 * tb + 4 * q));
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            of[p] = split8<NC>(dO[2 * p], dO[2 * p + 1]);
            rf[p] = split8<NC>(dR[2 * p], dR[2 * p + 1]);
        }
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            D[kb] *= whole;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                mul(D[kb], L.q.columns(kb, p, lane), of[p]);
                mul(D[kb], L.k.columns(kb, p, lane), rf[p]);
            }
        }
    });
    if (A.ds0 && wave < 4 && on) {
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            const int k = 16 * kb + 4 * q;
            if (k < A.Dk)
                *reinterpret_cast<f32x4_t*>(
                    A.ds0 + (head * A.Dv + v) * A.Dk + k) = D[kb];
        }
    }
}

template <typename E, int KT>
hipError_t launch(const GdrArgs& A, hipStream_t stream) {
    const auto kernel = gdr_backward_kernel<E, KT>;
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

hipError_t launch_gdr_backward(bool bf16, const GdrArgs& A,
                               hipStream_t stream) {
    const bool wide = gdr_dkp(A.Dk) == 128;
    if (bf16)
        return wide ? launch<bf16_t, 4>(A, stream)
                    : launch<bf16_t, 2>(A, stream);
    return wide ? launch<float, 4>(A, stream) : launch<float, 2>(A, stream);
}

}  // namespace rwkv7m
