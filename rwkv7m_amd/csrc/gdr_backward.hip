// The gated delta rule's recurrence backwards over chunks (gdr_chain.h has the
// division of work): the cotangent D of the state after each chunk, and dR,
// from which gdr_gradients.hip forms the gradients, chunk by chunk.
//
//   dX = scale P^T dO + 2^(G_L - G) (K D^T),  dR = T^T dX
//   D <- 2^G_L D + scale (2^G dO)^T Q - (beta 2^G dR)^T K
//
// Bound as the forward: 8 x 512 tokens, 12 heads of 64 x 64, 26.5 us, 3.3 a
// chunk; 8 x 4096, 16 heads of 128 x 128, 1.52 GB in 355 to 400 us, 3.8 to 4.3
// TB/s.
#include "gdr_chain.h"

namespace rwkv7m {
namespace {

using namespace gdr;

template <typename E, int KT, int OW>
__global__ void __launch_bounds__(64 * OW + BRING)
__attribute__((amdgpu_waves_per_eu(2, 2)))
gdr_backward_kernel(const GdrArgs A, int parts) {
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

    f32x4_t D[2 * KT];  // D(D^T): k = spread(kb, 4q + e), v = r
#pragma unroll
    for (int kb = 0; kb < 2 * KT; ++kb) {
        const int k = spread(kb, 4 * q);
        D[kb] = zero4();
        if (A.ds_t && wave < OW && on && k < A.Dk)
            D[kb] = four(A.ds_t + (head * A.Dv + v) * A.Dk + k);
    }

    OwnColumn<E, KT> column(A, A.dout, b, h, v);
    column.fetch(chunks - 1, lane);

    chain<E, KT, OW>(
        A, A.dout,
        static_cast<const Prepared*>(A.prepared) + head * chunks, head,
        16 * OW * at_.part, chunks - 1, -1, chunks,
        reinterpret_cast<ChainChunk<E, KT>*>(lds_raw),
        [&](const ChainChunk<E, KT>& L, int64_t c) {
        if (!has) return;
        float* keep = A.dstates + ((head * chunks + c) * DVP + v) * DKP;
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb)
            *reinterpret_cast<f32x4_t*>(keep + spread(kb, 4 * q)) = D[kb];

        // (the order of issue, as in the forward)
        constexpr bool DEEP = NI == 1;
        constexpr int TWO = DEEP ? 2 : 1, HALF = KT / 2;
        Frag<NI> kf[TWO][4], of[2];
        Frag<NC> Tf[6], Pf[6], Df[KT], xf[2], rf[2], sf[2];
        f32x4_t dO[4], dX[4], dR[4], KD[4], first[4], last[4], beta[4];
        const float whole = L.first[C - 1];
        column.take(L, c, c - 1, wave, lane, dO);
        if (DEEP) {
            triangle<true>(L.m.p, lane, Pf);
            blocks(L.k, 0, lane, kf[0]);
        }
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) dX[tb] = dR[tb] = KD[tb] = zero4();
#pragma unroll
        for (int p = 0; p < 2; ++p)
            of[p] = split8<NI>(dO[2 * p], dO[2 * p + 1]);
        // P^T dO and K D^T, t = spread(tb, 4q + e), v = r
        if (!DEEP) triangle<true>(L.m.p, lane, Pf);
        hold();
        mul_triangle<true>(dX, Pf, of);
        Df[0] = split8<NC>(D[0], D[1]);
        if (DEEP) interleave<4 * NC, 0, 3>();
#pragma unroll
        for (int p = 0; p < KT; ++p) {
            if (DEEP) hold();
            if (!DEEP) blocks(L.k, p, lane, kf[0]);
            else if (p + 1 < KT) blocks(L.k, p + 1, lane, kf[(p + 1) % TWO]);
            else column_blocks(L.q, 0, 0, lane, kf[(p + 1) % TWO]);
            if (p + 1 == KT)
#pragma unroll
                for (int tb = 0; tb < 4; ++tb) {
                    first[tb] = four(L.first + spread(tb, 4 * q));
                    last[tb] = four(L.last + spread(tb, 4 * q));
                }
            if (!DEEP) hold();
            mul_each(KD, kf[p % TWO], Df[p]);
            if (p + 1 < KT)
                Df[p + 1] = split8<NC>(D[2 * p + 2], D[2 * p + 3]);
            if (DEEP && p + 1 < KT) interleave<4 * NC, 1, 3>();
            if (DEEP && p + 1 == KT) interleave<4 * NC, 2, 0>();
        }
        // D <- 2^G_L D + scale (2^G dO)^T Q - (beta 2^G dR)^T K, half of the
        // first product while dX is put together, half while dR is
#pragma unroll
        for (int p = 0; p < 2; ++p)
            sf[p] = split8<NC>(A.scale * first[2 * p] * dO[2 * p],
                               A.scale * first[2 * p + 1] * dO[2 * p + 1]);
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) D[kb] *= whole;
        const auto queries = [&](int at) {
            const int n = at / 2, p = at & 1;
            if (DEEP) hold();
            if (!DEEP)
                column_blocks(L.q, n, p, lane, kf[0]);
            else if (at + 1 < KT)
                column_blocks(L.q, (at + 1) / 2, (at + 1) & 1, lane,
                              kf[(at + 1) % TWO]);
            else
                column_blocks(L.k, 0, 0, lane, kf[(at + 1) % TWO]);
            if (DEEP && at + 1 == HALF) triangle<true>(L.m.t, lane, Tf);
            if (!DEEP) hold();
            f32x4_t sum[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = D[4 * n + i];
            mul_each(sum, kf[at % TWO], sf[p]);
#pragma unroll
            for (int i = 0; i < 4; ++i) D[4 * n + i] = sum[i];
        };
#pragma unroll
        for (int at = 0; at < HALF; ++at) {
            queries(at);
#pragma unroll
            for (int i = 4 * at / HALF; i < 4 * (at + 1) / HALF; ++i)
                dX[i] = A.scale * dX[i] + last[i] * KD[i];
#pragma unroll
            for (int i = 2 * at / HALF; i < 2 * (at + 1) / HALF; ++i)
                xf[i] = split8<NC>(dX[2 * i], dX[2 * i + 1]);
            if (DEEP && at + 1 < HALF) interleave<4 * NC, 1, 8>();
            if (DEEP && at + 1 == HALF) interleave<4 * NC, 4, 8>();
        }
        if (!DEEP) triangle<true>(L.m.t, lane, Tf);
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) beta[tb] = four(L.beta + spread(tb, 4 * q));
        hold();
        mul_triangle<true>(dR, Tf, xf);
#pragma unroll
        for (int at = HALF; at < KT; ++at) {
            queries(at);
#pragma unroll
            for (int i = 2 * (at - HALF) / HALF; i < 2 * (at - HALF + 1) / HALF;
                 ++i)
                rf[i] = split8<NC>(
                    -(first[2 * i] * beta[2 * i]) * dR[2 * i],
                    -(first[2 * i + 1] * beta[2 * i + 1]) * dR[2 * i + 1]);
            if (DEEP) interleave<4 * NC, 1, 8>();
        }
        put_column(A.dr + (head * chunks + c) * C * DVP, DVP, q, v, dR);
#pragma unroll
        for (int at = 0; at < KT; ++at) {
            const int n = at / 2, p = at & 1;
            if (DEEP) hold();
            if (!DEEP)
                column_blocks(L.k, n, p, lane, kf[0]);
            else if (at + 1 < KT)
                column_blocks(L.k, (at + 1) / 2, (at + 1) & 1, lane,
                              kf[(at + 1) % TWO]);
            if (!DEEP) hold();
            f32x4_t sum[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = D[4 * n + i];
            mul_each(sum, kf[at % TWO], rf[p]);
            if (DEEP) interleave<4 * NC, 1, 0>();
#pragma unroll
            for (int i = 0; i < 4; ++i) D[4 * n + i] = sum[i];
        }
    });
    if (A.ds0 && wave < OW && on) {
#pragma unroll
        for (int kb = 0; kb < 2 * KT; ++kb) {
            const int k = spread(kb, 4 * q);
            if (k < A.Dk)
                *reinterpret_cast<f32x4_t*>(
                    A.ds0 + (head * A.Dv + v) * A.Dk + k) = D[kb];
        }
    }
}

template <typename E, int KT, int OW>
hipError_t launch_with(const GdrArgs& A, hipStream_t stream) {
    const auto kernel = gdr_backward_kernel<E, KT, OW>;
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

template <typename E, int KT>
hipError_t launch(const GdrArgs& A, hipStream_t stream) {
    switch (owning_waves(A.B * A.Hv, gdr_dvp(A.Dv))) {
        case 1: return launch_with<E, KT, 1>(A, stream);
        case 2: return launch_with<E, KT, 2>(A, stream);
        default: return launch_with<E, KT, 4>(A, stream);
    }
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
