// The gated delta rule's gradients, chunk by chunk, from the states before the
// chunks (S0) and X, which the forward kept, and D and dR, which
// gdr_backward.hip left:
//
//   N = tril(dR X^T, -1) E,  dP = scale tril(dO X^T) E
//   dq = scale 2^G (dO S0) + dP K
//   left = -2^G (dR S0) - N K
//   right = 2^(G_L - G) (X D) + dP^T Q - (beta N)^T K
//   dk = beta left + right,  dv = beta dR,  dbeta = k.left + dR.v
//   dG = q.dq + beta k.left - k.right, + <D, S_L> at the last token,
//   dg = the sum of dG from the token on,
//   <D, S_L> = 2^G_L <D, S0> + sum_t k_t.(2^(G_L - G) X D)_t
//
// One workgroup a chunk and value head, all of them independent; a wave owns
// 16 tokens.  S0 and D pass through LDS in blocks of 64 rows, whose columns are
// operands by transposing reads; N and dP are formed in both orientations
// (rows of the wave's tokens, and columns), so that no wave needs another's.
#include "gdr_common.h"

namespace rwkv7m {
namespace {

using namespace gdr;

template <typename E, int KT>
struct GradShared {
    Rows64<kIn<E>, KT> k, q;
    Rows64<kMade<E>, KT> s;  // 64 rows of S0, then of D
    double G[C];
    float dG[C], rv[C], sums[4];
};

// Eight places 32 p + 8q + i of a row of X or dR, in planes.
template <int NC>
__device__ __forceinline__ Frag<NC> row8(const float* p, bool on) {
    Eight<float> v;
    if (on)
        v.load(p);
    else
        v.clear();
    return split8<NC>(v.a, v.b);
}

__device__ __forceinline__ void store_gate(void* p, bool bf16, int64_t i,
                                           float x) {
    if (bf16)
        store_f(static_cast<bf16_t*>(p) + i, x);
    else
        store_f(static_cast<float*>(p) + i, x);
}

template <typename E, int KT>
__global__ void __launch_bounds__(NT)
gdr_gradients_kernel(const GdrArgs A) {
    constexpr int NI = kIn<E>, NC = kMade<E>, DKP = 32 * KT;
    extern __shared__ char lds_raw[];
    auto& L = *reinterpret_cast<GradShared<E, KT>*>(lds_raw);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int64_t chunks = (A.T + C - 1) / C;
    const int64_t id = blockIdx.x, head = id / chunks, c = id % chunks;
    const int64_t b = head / A.Hv, h = head % A.Hv, hk = h / (A.Hv / A.Hk);
    const int64_t t0 = c * C;
    const int valid = int(A.T - t0 < C ? A.T - t0 : C);
    const int DVP = (A.Dv + 31) / 32 * 32;
    const Prepared<NC>& M =
        static_cast<const Prepared<NC>*>(A.prepared)[head * chunks + c];

    Staged<E, KT> ks, qs;
    ks.load(at<E>(A.k, b, hk, t0), A.k.st, valid, A.Dk);
    qs.load(at<E>(A.q, b, hk, t0), A.q.st, valid, A.Dk);
    if (threadIdx.x < C) L.G[threadIdx.x] = M.G[threadIdx.x];
    ks.store(L.k);
    qs.store(L.q);

    f32x4_t dq[2 * KT], left[2 * KT], right[2 * KT];
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) dq[j] = left[j] = right[j] = zero4();
    // (rows: token block `wave` against block j <= wave, t = r, s = 4q + e;
    // columns: block j >= wave against `wave`, t = 4q + e, s = r)
    f32x4_t dp_row[4], n_row[4], dp_col[4], n_col[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        dp_row[j] = n_row[j] = dp_col[j] = n_col[j] = zero4();
    float rv = 0.f, ds = 0.f;  // dR.v of token 16 wave + r; <D, S0>

    const E* dop = at<E>(A.dout, b, h, t0);
    const E* vp = at<E>(A.v, b, h, t0);
    const float* x0 = A.x + (head * chunks + c) * C * DVP;
    const float* r0 = A.dr + (head * chunks + c) * C * DVP;
    const float* s0 = A.states + (head * chunks + c) * DVP * DKP;
    const float* d0 = A.dstates + (head * chunks + c) * DVP * DKP;
    const int own = 16 * wave + r;  // the lane's token
    E* dvp = static_cast<E*>(A.dv) + ((b * A.T + t0 + own) * A.Hv + h) * A.Dv;
    const float beta_own = M.beta[own];

    for (int v0 = 0; v0 < DVP; v0 += 64) {
        // the block's rows of S0 and D, 8 places a thread and turn
        constexpr int per_row = DKP / 4, turns = 64 * per_row / NT;
        f32x4_t sv[turns], dv[turns];
#pragma unroll
        for (int i = 0; i < turns; ++i) {
            const int u = i * NT + int(threadIdx.x);
            const int row = v0 + u / per_row, col = 4 * (u % per_row);
            sv[i] = dv[i] = zero4();
            if (row < DVP) {
                sv[i] = four(s0 + row * DKP + col);
                dv[i] = four(d0 + row * DKP + col);
            }
        }
#pragma unroll
        for (int i = 0; i < turns; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) ds += sv[i][e] * dv[i][e];
        const auto put = [&](const f32x4_t (&x)[turns]) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < turns; ++i) {
                const int u = i * NT + int(threadIdx.x);
                const int row = u / per_row, col = 4 * (u % per_row);
                uint32_t lo[NC], hi[NC];
                split2<NC>(x[i][0], x[i][1], lo);
                split2<NC>(x[i][2], x[i][3], hi);
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    *reinterpret_cast<uint2*>(&L.s.x[n][row][col]) =
                        make_uint2(lo[n], hi[n]);
            }
            __syncthreads();
        };
        // operands of the wave's own tokens (left or right alike)
        Frag<NI> of[2];
        Frag<NC> xf[2], rf[2];
        const auto dout = [&](int tb, int p) {
            const int t = 16 * tb + r, col = v0 + 32 * p + 8 * q;
            Eight<E> e;
            if (t < valid && col < A.Dv)
                e.load(dop + t * A.dout.st + col);
            else
                e.clear();
            return e.planes();
        };
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int col = v0 + 32 * p + 8 * q;
            of[p] = dout(wave, p);
            xf[p] = row8<NC>(x0 + own * DVP + col, col < DVP);
            // dv and dR.v
            Eight<float> dr;
            dr.clear();
            if (col < DVP) dr.load(r0 + own * DVP + col);
            rf[p] = split8<NC>(dr.a, dr.b);
            if (own < valid && col < A.Dv) {
                Eight<E> vv;
                vv.load(vp + own * A.v.st + col);
#pragma unroll
                for (int i = 0; i < 8; ++i) rv += dr.get(i) * vv.get(i);
                dr.a *= beta_own;
                dr.b *= beta_own;
                if constexpr (sizeof(E) == 4) {
                    *reinterpret_cast<f32x4_t*>(dvp + col) = dr.a;
                    *reinterpret_cast<f32x4_t*>(dvp + col + 4) = dr.b;
                } else {
                    *reinterpret_cast<uint4*>(dvp + col) =
                        make_uint4(pack2(dr.a[0], dr.a[1]),
                                   pack2(dr.a[2], dr.a[3]),
                                   pack2(dr.b[0], dr.b[1]),
                                   pack2(dr.b[2], dr.b[3]));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j <= wave) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int col = v0 + 32 * p + 8 * q;
                    const Frag<NC> xj =
                        row8<NC>(x0 + (16 * j + r) * DVP + col, col < DVP);
                    mul(dp_row[j], xj, of[p]);
                    mul(n_row[j], xj, rf[p]);
                }
            }
            if (j >= wave) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int col = v0 + 32 * p + 8 * q;
                    mul(dp_col[j], dout(j, p), xf[p]);
                    mul(n_col[j],
                        row8<NC>(r0 + (16 * j + r) * DVP + col, col < DVP),
                        xf[p]);
                }
            }
        }
        put(sv);
#pragma unroll
        for (int jb = 0; jb < 2 * KT; ++jb)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const Frag<NC> f = L.s.columns_dense(jb, p, lane);
                mul(dq[jb], of[p], f);
                mul(left[jb], rf[p], f);
            }
        put(dv);
#pragma unroll
        for (int jb = 0; jb < 2 * KT; ++jb)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                mul(right[jb], xf[p], L.s.columns_dense(jb, p, lane));
    }

    // rows' factors, t = 16 wave + 4q + e
    const int row = 16 * wave + 4 * q;
    const f32x4_t first = four(M.first + row), last = four(M.last + row),
                  beta = four(M.beta + row);
    f32x4_t klast = zero4();
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) {
        dq[j] *= first;
        left[j] *= first;
        right[j] *= last;
        klast += L.k.values(16 * wave, j, lane) * right[j];
    }
    // E and the masks
    const double Gw = L.G[own];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j <= wave) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int s = 16 * j + 4 * q + e;
                const float E_ = s <= own ? exp2_of(Gw - L.G[s]) : 0.f;
                dp_row[j][e] = s <= own ? dp_row[j][e] * (A.scale * E_) : 0.f;
                n_row[j][e] = s < own ? n_row[j][e] * E_ : 0.f;
            }
        }
        if (j >= wave) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = 16 * j + 4 * q + e;
                const float E_ = own <= t ? exp2_of(L.G[t] - Gw) : 0.f;
                dp_col[j][e] = own <= t ? dp_col[j][e] * (A.scale * E_) : 0.f;
                n_col[j][e] =
                    own < t ? n_col[j][e] * (-M.beta[t] * E_) : 0.f;
            }
        }
    }
    // dq so far is without the scale; left with the other sign
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) dq[j] *= A.scale;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        if (2 * p <= wave) {
            const Frag<NC> a = split8<NC>(dp_row[2 * p], dp_row[2 * p + 1]);
            const Frag<NC> n = split8<NC>(n_row[2 * p], n_row[2 * p + 1]);
#pragma unroll
            for (int j = 0; j < 2 * KT; ++j) {
                const Frag<NI> f = L.k.columns(j, p, lane);
                mul(dq[j], a, f);
                mul(left[j], n, f);
            }
        }
        if (2 * p + 1 >= wave) {
            const Frag<NC> a = split8<NC>(dp_col[2 * p], dp_col[2 * p + 1]);
            const Frag<NC> n = split8<NC>(n_col[2 * p], n_col[2 * p + 1]);
#pragma unroll
            for (int j = 0; j < 2 * KT; ++j) {
                mul(right[j], a, L.q.columns(j, p, lane));
                mul(right[j], n, L.k.columns(j, p, lane));
            }
        }
    }
    f32x4_t qdq = zero4(), kleft = zero4(), kright = zero4();
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) {
        const f32x4_t kv = L.k.values(16 * wave, j, lane);
        left[j] = -left[j];
        qdq += L.q.values(16 * wave, j, lane) * dq[j];
        kleft += kv * left[j];
        kright += kv * right[j];
    }
    rv += __shfl_xor(rv, 16);
    rv += __shfl_xor(rv, 32);
    if (q == 0) L.rv[own] = rv;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) ds += __shfl_xor(ds, m);
    float kl = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        qdq[e] = sum16(qdq[e]);
        kleft[e] = sum16(kleft[e]);
        kright[e] = sum16(kright[e]);
        kl += sum16(klast[e]);
    }
    kl += __shfl_xor(kl, 16);
    kl += __shfl_xor(kl, 32);
    if (lane == 0) L.sums[wave] = kl + ds * M.first[C - 1];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r == e) L.dG[row + e] = qdq[e] + beta[e] * kleft[e] - kright[e];
    __syncthreads();
    if (r < 4) {
        const int t = row + r;
        float kt = r == 0 ? kleft[0] : r == 1 ? kleft[1] : r == 2 ? kleft[2]
                                                                  : kleft[3];
        if (t < valid)
            store_gate(A.dbeta, A.beta_bf16, (b * A.T + t0 + t) * A.Hv + h,
                       kt + L.rv[t]);
    }
    if (wave == 0) {
        double x = L.dG[lane];
        if (lane == 63)
            x += double(L.sums[0]) + double(L.sums[1]) + double(L.sums[2]) +
                 double(L.sums[3]);
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double y = __shfl_down(x, m);
            if (lane + m < 64) x += y;
        }
        if (lane < valid)
            store_gate(A.dg, A.g_bf16, (b * A.T + t0 + lane) * A.Hv + h,
                       float(x));
    }
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j) {
        const int col = 16 * j + r;
        if (col >= A.Dk) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = row + e;
            if (t >= valid) continue;
            const float dk = beta[e] * left[j][e] + right[j][e];
            if (A.dq_part) {
                const int64_t i =
                    ((b * A.T + t0 + t) * A.Hv + h) * A.Dk + col;
                A.dq_part[i] = dq[j][e];
                A.dk_part[i] = dk;
            } else {
                const int64_t i =
                    ((b * A.T + t0 + t) * A.Hk + hk) * A.Dk + col;
                store_f(static_cast<E*>(A.dq) + i, dq[j][e]);
                store_f(static_cast<E*>(A.dk) + i, dk);
            }
        }
    }
}

// The shares of the value heads that read one key head, added up in their
// order: four places a thread.
template <typename E>
__global__ void __launch_bounds__(NT)
gdr_group_kernel(const GdrArgs A, int64_t n) {
    const int per = int(A.Hv / A.Hk);
    const int64_t quads = A.Dk / 4;
    for (int64_t i = int64_t(blockIdx.x) * NT + threadIdx.x; i < n;
         i += int64_t(gridDim.x) * NT) {
        const int64_t row = i / quads, col = 4 * (i % quads);
        // (row: token and key head; its value heads are adjoining)
        const float* from[2] = {A.dq_part, A.dk_part};
        void* to[2] = {A.dq, A.dk};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4_t sum = zero4();
            for (int j = 0; j < per; ++j)
                sum += four(from[m] + (row * per + j) * A.Dk + col);
            E* out = static_cast<E*>(to[m]) + row * A.Dk + col;
            if constexpr (sizeof(E) == 4)
                *reinterpret_cast<f32x4_t*>(out) = sum;
            else
                *reinterpret_cast<uint2*>(out) = make_uint2(
                    pack2(sum[0], sum[1]), pack2(sum[2], sum[3]));
        }
    }
}

template <typename E, int KT>
hipError_t launch(const GdrArgs& A, hipStream_t stream) {
    const auto kernel = gdr_gradients_kernel<E, KT>;
    const int lds = int(sizeof(GradShared<E, KT>));
    hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const int64_t grid = A.B * A.Hv * ((A.T + C - 1) / C);
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(NT), lds, stream, A);
    e = hipGetLastError();
    if (e != hipSuccess || !A.dq_part) return e;
    const int64_t n = A.B * A.T * A.Hk * (A.Dk / 4);
    int64_t blocks = (n + NT - 1) / NT;
    if (blocks > 8192) blocks = 8192;
    hipLaunchKernelGGL(gdr_group_kernel<E>, dim3(unsigned(blocks)), dim3(NT),
                       0, stream, A, n);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gdr_gradients(bool bf16, const GdrArgs& A,
                                hipStream_t stream) {
    const bool wide = gdr_dkp(A.Dk) == 128;
    if (bf16)
        return wide ? launch<bf16_t, 4>(A, stream)
                    : launch<bf16_t, 2>(A, stream);
    return wide ? launch<float, 4>(A, stream) : launch<float, 2>(A, stream);
}

}  // namespace rwkv7m
