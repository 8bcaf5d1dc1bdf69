// The gated delta rule's chunk matrices (gdr_common.h has the formulas): T =
// (I + A)^-1 and P in planes, and the gates.
//
// One workgroup a chunk and value head, all of them independent, a wave a block
// of 16 tokens.  T's diagonal blocks are substituted forward, a lane a column:
// with keys that resemble each other the powers of A in a product form of the
// inverse grow to 1e3 and cancel, which would cost fp32 three of its digits.
// The blocks below follow by fp32 matrix products, T_ij = -T_ii sum_m A_im T_mj.
//
// A chunk's way is its latency (loads, products, 16 steps of substitution on
// one wave, up to three products after each other): 8 x 512 tokens, 12 heads of
// 64 x 64, 13.5 us, 1 x 1999, 32 of 128 x 128, 19.5 us; 8 x 4096, 16 of 128 x
// 128, 585 MB in 123 to 138 us, 4.2 to 4.8 TB/s.
#include "gdr_common.h"

namespace rwkv7m {
namespace {

using namespace gdr;

constexpr int NT = 256, PITCH = C + 4;

struct Shared {
    alignas(16) float a[C][PITCH], t[C][PITCH];
    double G[4][C];  // each wave its own
};

__device__ __forceinline__ float gate(const GdrTensor& t, bool bf16, int64_t b,
                                      int64_t h, int64_t token) {
    return bf16 ? load_f(at<bf16_t>(t, b, h, token))
                : load_f(at<float>(t, b, h, token));
}

// The sum over the lanes up to and with the calling one (lane rotations and
// scalar row totals: a shuffle of a double is two round trips through LDS).
__device__ __forceinline__ double wave_scan(double x, double* all) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
#define RWKV7M_STEP(ctrl)                                                   \
    do {                                                                    \
        i32x2 u = __builtin_bit_cast(i32x2, x);                             \
        u[0] = __builtin_amdgcn_update_dpp(0, u[0], ctrl, 0xf, 0xf, true);  \
        u[1] = __builtin_amdgcn_update_dpp(0, u[1], ctrl, 0xf, 0xf, true);  \
        x += __builtin_bit_cast(double, u);                                 \
    } while (0)
    RWKV7M_STEP(0x111);  // row_shr:1
    RWKV7M_STEP(0x112);
    RWKV7M_STEP(0x114);
    RWKV7M_STEP(0x118);
#undef RWKV7M_STEP
    const auto lane = [&](int l) {
        i32x2 u = __builtin_bit_cast(i32x2, x);
        u[0] = __builtin_amdgcn_readlane(u[0], l);
        u[1] = __builtin_amdgcn_readlane(u[1], l);
        return __builtin_bit_cast(double, u);
    };
    const int row = threadIdx.x % 64 / 16;
    const double a = lane(15), b = a + lane(31), c = b + lane(47);
    *all = c + lane(63);
    return x + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}

// D(M Y) + c from D(M^T) and D(Y) in fp32.
__device__ __forceinline__ f32x4_t mm32(const f32x4_t& mt, const f32x4_t& y,
                                        f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(mt[e], y[e], c, 0, 0, 0);
    return c;
}

template <typename E, int KT>
__global__ void __launch_bounds__(NT)
gdr_prepare_kernel(const GdrArgs A) {
    constexpr int NI = kIn<E>, NC = kMade;
    __shared__ Shared S;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const uint32_t chunks = chunk_count(A), id = blockIdx.x;
    const int64_t head = id / chunks, c = id % chunks;
    const Head at_head(A, uint32_t(head));
    const int64_t b = at_head.b, h = at_head.h, hk = at_head.hk;
    const int64_t t0 = c * C;
    const int valid = int(A.T - t0 < C ? A.T - t0 : C);
    auto* out = static_cast<Prepared*>(A.prepared) + id;

    // rows of k and q: places 32 p + 8q + i of token 16 tb + r, all loads
    // before the first is waited for
    const auto rows = [&](const GdrTensor& x, int tb, Eight<E> (&f)[KT]) {
        const E* p = at<E>(x, b, hk, t0 + near(16 * tb + r, valid - 1));
#pragma unroll
        for (int i = 0; i < KT; ++i)
            f[i].load(p + near(32 * i + 8 * q, A.Dk - 8));
    };
    const auto planes = [&](Eight<E> x, int tb, int i) {
        x.keep(16 * tb + r < valid && 32 * i + 8 * q < A.Dk);
        return x.planes();
    };
    // Each wave has the gates of all tokens, lane a token.  The running sum of
    // the log decays: a decay of 0 (-inf) is held to e^-1000, 0 in any result,
    // so that later differences stay finite.
    const int token = near(lane, valid - 1);
    const float g = gate(A.g, A.g_bf16, b, h, t0 + token);
    const float beta_ = gate(A.beta, A.beta_bf16, b, h, t0 + token);
    Eight<E> qw[KT], kj[4][KT];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j <= wave) rows(A.k, j, kj[j]);
    rows(A.q, wave, qw);
    const float beta = lane < valid ? beta_ : 0.f;
    double all;
    const double G = wave_scan(
        lane < valid ? kLog2e * double(g < -1000.f ? -1000.f : g) : 0.0, &all);
    S.G[wave][lane] = G;
    if (wave == 0) {
        out->G[lane] = G;
        out->first[lane] = exp2_of(G);
        out->last[lane] = exp2_of(all - G);
        out->beta[lane] = beta;
    }
    const float beta_own = __shfl(beta, 16 * wave + r);
    Frag<NI> qf[KT], kf[KT];  // the wave's own token block
#pragma unroll
    for (int p = 0; p < KT; ++p) {
        qf[p] = planes(qw[p], wave, p);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j == wave) kf[p] = planes(kj[j][p], j, p);
    }
    const int own = 16 * wave + r;
    const double* Gs = S.G[wave];
    const double Gw = Gs[own];
    // A's and P's block (wave, j)
    const auto block = [&](int j, const Eight<E> (&kb)[KT]) {
        f32x4_t a = zero4(), pt = zero4();
#pragma unroll
        for (int p = 0; p < KT; ++p) {
            const Frag<NI> f = planes(kb[p], j, p);
            mul(a, f, kf[p]);   // D(A^T): s = 4q + e, t = r
            mul(pt, f, qf[p]);  // D(P^T)
        }
        uint32_t lo[NC], hi[NC];
        f32x4_t at_;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int s = 16 * j + 4 * q + e;
            const float E_ = s <= own ? exp2_of(Gw - Gs[s]) : 0.f;
            at_[e] = s < own ? a[e] * (beta_own * E_) : 0.f;
            pt[e] = s <= own ? pt[e] * E_ : 0.f;
        }
        *reinterpret_cast<f32x4_t*>(&S.a[own][16 * j + 4 * q]) = at_;
        split2<NC>(pt[0], pt[1], lo);
        split2<NC>(pt[2], pt[3], hi);
#pragma unroll
        for (int n = 0; n < NC; ++n)
            *reinterpret_cast<uint2*>(out->m.p.at(n, own, 16 * j + 4 * q)) =
                make_uint2(lo[n], hi[n]);
    };
    // the diagonal blocks first: the first wave, which has no other, inverts
    // them while the rest are made
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j == wave) block(j, kj[j]);
    __syncthreads();
    if (wave == 0) {
        // block q's column r of the inverse
        float x[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            float sum[4] = {t == r ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < t; s += 4) {
                const f32x4_t a = four(&S.a[16 * q + t][16 * q + s]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s + i < t) sum[i] -= a[i] * x[s + i];
            }
            x[t] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            S.t[16 * q + t][16 * q + r] = x[t];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < wave) block(j, kj[j]);
    }
    if ((wave & 1) == 0) {
        // (the block right of the diagonal that shares a pair with it)
#pragma unroll
        for (int n = 0; n < NC; ++n)
            *reinterpret_cast<uint2*>(out->m.p.at(
                n, own, 16 * (wave + 1) + 4 * q)) = make_uint2(0, 0);
        *reinterpret_cast<f32x4_t*>(&S.t[own][16 * (wave + 1) + 4 * q]) =
            zero4();
    }
    __syncthreads();
    if (wave < 3) {
        // column block `wave`, downwards
        f32x4_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[0][e] = S.t[16 * wave + 4 * q + e][16 * wave + r];
#pragma unroll
        for (int d = 1; d < 4; ++d) {
            const int i = wave + d;
            if (i > 3) break;
            f32x4_t sum = zero4();
#pragma unroll
            for (int m = 0; m < d; ++m)
                sum = mm32(four(&S.a[16 * i + r][16 * (wave + m) + 4 * q]),
                           y[m], sum);
            y[d] = mm32(four(&S.t[16 * i + r][16 * i + 4 * q]), sum, zero4());
            y[d] = -y[d];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                S.t[16 * i + 4 * q + e][16 * wave + r] = y[d][e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = i * NT + int(threadIdx.x), l = u % 64;
        if (u >= 6 * 64) break;
        const int tb = u < 256 ? u / 64 : u / 64 - 2, p = u >= 256;
        const int row = spread(tb, l % 16), col = 32 * p + 8 * (l / 16);
        const Frag<NC> f =
            split8<NC>(four(&S.t[row][col]), four(&S.t[row][col + 4]));
#pragma unroll
        for (int n = 0; n < NC; ++n)
            *reinterpret_cast<u32x4_t*>(&out->m.t.x[n][u / 64][l][0]) = f.p[n];
    }
}

}  // namespace

int gdr_dkp(int Dk) { return Dk <= 64 ? 64 : 128; }
int gdr_dvp(int Dv) { return (Dv + 31) / 32 * 32; }

int64_t gdr_prepared_bytes() { return int64_t(sizeof(Prepared)); }

hipError_t launch_gdr_prepare(bool bf16, const GdrArgs& A,
                              hipStream_t stream) {
    const dim3 grid(unsigned(A.B * A.Hv * ((A.T + C - 1) / C)));
    const bool wide = gdr_dkp(A.Dk) == 128;
#define RWKV7M_GDR(E, KT)                                                \
    hipLaunchKernelGGL((gdr_prepare_kernel<E, KT>), grid, dim3(NT), 0,   \
                       stream, A)
    if (bf16 && wide)
        RWKV7M_GDR(bf16_t, 4);
    else if (bf16)
        RWKV7M_GDR(bf16_t, 2);
    else if (wide)
        RWKV7M_GDR(float, 4);
    else
        RWKV7M_GDR(float, 2);
#undef RWKV7M_GDR
    return hipGetLastError();
}

}  // namespace rwkv7m
