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
// (q.dq - dv.v is dG as well, and cheaper.  But in the running sum of the form
// above the pairs of tokens on one side of its border cancel, product by
// product; of the other they do not, and dg, a small sum of large terms, is off
// by 1.6 times as much.)
//
// One workgroup a chunk and value head, all of them independent.  A wave owns
// 32 tokens and a share of the columns of dq, left and right.  S0 and D pass
// through LDS in blocks of 32 rows, whose columns are operands by transposing
// reads; each operand so read serves two blocks of tokens.  The ten lower
// blocks of N and dP are divided among the waves and meet in LDS, whose rows
// are operands for dq and left, whose columns for right.
//
// 8 x 512 tokens, 12 heads of 64 x 64: 34.5 us.  8 x 4096, 16 of 128 x 128:
// 2.55 GB in 790 to 950 us, 2.7 to 3.2 TB/s (matrix units busy 23 % of the
// time), bound by a workgroup's own steps (one lives on a CU, its sums fill the
// registers): the loads of its first block and the gates, and four blocks
// between barriers.
#include "gdr_common.h"

namespace rwkv7m {
namespace {

using namespace gdr;

// Shares of the columns a workgroup's waves are divided over (two rows of
// waves).  bf16 up to 64 columns: 2, and two workgroups a CU (8 x 512 tokens, 12
// heads of 64 x 64: 34.5 us; with 4 and one workgroup 42).  At 128 the sums of
// half the columns leave no room for a second workgroup's registers: 4, and the
// next block's loads begun ahead (8 x 4096, 16 of 128 x 128: 800 us; with 2,
// which spill, 1720).
template <typename E, int KT>
constexpr int kShares = sizeof(E) == 2 && KT == 4 ? 4 : 2;

template <typename E, int KT>
struct GradShared {
    union {
        struct {  // a block of 32 columns of v
            Rows<kMade, KT, 32> s, d;  // S0's and D's rows
            Rows<kMade, 1> x, r;          // X, dR
            Rows<kIn<E>, 1> o;            // dO
        };
        struct {  // what is made of them
            union {
                struct {
                    Rows<kIn<E>, KT> k, q;
                };
                E out[2][C][32 * KT + 8];  // dq and dk, behind them
            };
            Rows<kMade, 2> n;  // N, then -beta N
            union {
                Rows<kMade, 2> p;  // dP
                float dots[kShares<E, KT>][2][C];  // of dG, k.left, behind it
            };
        };
    };
    double G[C];
    float first[C], last[C], beta[C], rv[C];
    float sums[2 * kShares<E, KT>];
};

// Four adjoining elements of a row.
template <typename E>
struct Four;
template <>
struct Four<bf16_t> {
    uint2 a;
    __device__ __forceinline__ void load(const bf16_t* p) {
        a = *reinterpret_cast<const uint2*>(p);
    }
    __device__ __forceinline__ void keep(bool on) {
        a.x = on ? a.x : 0u;
        a.y = on ? a.y : 0u;
    }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t u = i < 2 ? a.x : a.y;
        return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
    }
    __device__ __forceinline__ void put(Rows<1, 1>& to, int row,
                                        int col) const {
        *reinterpret_cast<uint2*>(&to.x[0][row][col]) = a;
    }
};
template <>
struct Four<float> {
    f32x4_t a;
    __device__ __forceinline__ void load(const float* p) { a = four(p); }
    __device__ __forceinline__ void keep(bool on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = on ? a[i] : 0.f;
    }
    __device__ __forceinline__ float get(int i) const { return a[i]; }
    __device__ __forceinline__ void put(Rows<3, 1>& to, int row,
                                        int col) const {
        put4(to, row, col, a);
    }
};
__device__ __forceinline__ void store4(float* p, const f32x4_t& x) {
    *reinterpret_cast<f32x4_t*>(p) = x;
}
__device__ __forceinline__ void store4(bf16_t* p, const f32x4_t& x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1]),
                                              pack2(x[2], x[3]));
}

__device__ __forceinline__ void store_gate(void* p, bool bf16, int64_t i,
                                           float x) {
    if (bf16)
        store_f(static_cast<bf16_t*>(p) + i, x);
    else
        store_f(static_cast<float*>(p) + i, x);
}

template <typename E, int KT>
__global__ void __launch_bounds__((128 * kShares<E, KT>), sizeof(E) == 2 ? 2 : 1)
gdr_gradients_kernel(const GdrArgs A) {
    constexpr int NI = kIn<E>, NC = kMade, DKP = 32 * KT;
    constexpr int KQ = kShares<E, KT>, NT = 128 * KQ;
    constexpr bool AHEAD = KQ == 4;
    extern __shared__ char lds_raw[];
    auto& L = *reinterpret_cast<GradShared<E, KT>*>(lds_raw);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int th = wave / KQ, kh = wave % KQ;  // tokens 32 th .., share kh
    constexpr int KW = 2 * KT / KQ;  // the wave's tiles of 16 columns
    const uint32_t chunks = chunk_count(A), id = blockIdx.x;
    const int64_t head = id / chunks, c = id % chunks;
    const Head at_head(A, uint32_t(head));
    const int64_t b = at_head.b, h = at_head.h, hk = at_head.hk;
    const int64_t t0 = c * C;
    const int valid = int(A.T - t0 < C ? A.T - t0 : C);
    const int DVP = (A.Dv + 31) / 32 * 32;
    const Prepared& M =
        static_cast<const Prepared*>(A.prepared)[head * chunks + c];

    const E* dop = at<E>(A.dout, b, h, t0);
    const E* vp = at<E>(A.v, b, h, t0);
    const float* x0 = A.x + (head * chunks + c) * C * DVP;
    const float* r0 = A.dr + (head * chunks + c) * C * DVP;
    const float* s0 = A.states + (head * chunks + c) * DVP * DKP;
    const float* d0 = A.dstates + (head * chunks + c) * DVP * DKP;

    Staged<E, KT, NT> ks, qs;
    const auto bring = [&]() {
        ks.load(gdr::at<E>(A.k, b, hk, t0), A.k.st, valid, A.Dk, threadIdx.x);
        qs.load(gdr::at<E>(A.q, b, hk, t0), A.q.st, valid, A.Dk, threadIdx.x);
    };
    if constexpr (AHEAD) bring();
    if (threadIdx.x < C) {
        L.G[threadIdx.x] = M.G[threadIdx.x];
        L.first[threadIdx.x] = M.first[threadIdx.x];
        L.last[threadIdx.x] = M.last[threadIdx.x];
        L.beta[threadIdx.x] = M.beta[threadIdx.x];
    }

    f32x4_t dq[2][KW], left[2][KW], right[2][KW];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KW; ++j)
            dq[i][j] = left[i][j] = right[i][j] = zero4();
    // Blocks (tb, sb) of N and dP, t = 4q + e, s = r.  The last share's waves
    // have (2 + th, 0) and (2 + th, 1), the others those of the wave's own
    // tokens, (0, 0), (1, 0), (1, 1) from 2 th on: all three, or one each.
    constexpr int OWN = KQ == 2 ? 3 : 1, TILES = KQ == 2 ? 3 : 2;
    const bool last_share = kh == KQ - 1;
    f32x4_t dp[TILES], nn[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) dp[i] = nn[i] = zero4();
    float ds = 0.f;  // <D, S0>
    // Four places of X, dR, dO and v a thread and turn, of rows trow[i]; dR.v
    constexpr int rows = 8 * C / NT, step = C / rows;
    const int trow = threadIdx.x / 8, tcol = 4 * (threadIdx.x % 8);
    float rv[rows], beta_own[rows];
#pragma unroll
    for (int i = 0; i < rows; ++i) {
        rv[i] = 0.f;
        beta_own[i] = M.beta[trow + i * step];
    }
    E* dvp = static_cast<E*>(A.dv) + ((b * A.T + t0) * A.Hv + h) * A.Dv + tcol;

    // 32 columns of v on their way to LDS: rows of S0 and D, places of X, dR,
    // dO and v
    constexpr int turns = 32 * DKP / 4 / NT;
    f32x4_t sv[turns], dv[turns], xv[rows], r4[rows];
    Four<E> ov[rows], vv[rows];
    const auto fetch = [&](int v0) {
#pragma unroll
        for (int i = 0; i < turns; ++i) {
            const int u = 4 * (i * NT + int(threadIdx.x));
            sv[i] = four(s0 + v0 * DKP + u);
            dv[i] = four(d0 + v0 * DKP + u);
        }
#pragma unroll
        for (int i = 0; i < rows; ++i) {
            const int t = trow + i * step;
            xv[i] = four(x0 + t * DVP + v0 + tcol);
            r4[i] = four(r0 + t * DVP + v0 + tcol);
            const int col = near(v0 + tcol, A.Dv - 4);
            ov[i].load(dop + near(t, valid - 1) * A.dout.st + col);
            vv[i].load(vp + near(t, valid - 1) * A.v.st + col);
        }
    };
    if constexpr (AHEAD) fetch(0);
    for (int v0 = 0; v0 < DVP; v0 += 32) {
        if constexpr (!AHEAD) fetch(v0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < turns; ++i) {
            const int u = i * NT + int(threadIdx.x);
            const int row = u / (DKP / 4), col = 4 * (u % (DKP / 4));
            put4(L.s, row, col, sv[i]);
            put4(L.d, row, col, dv[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) ds += sv[i][e] * dv[i][e];
        }
#pragma unroll
        for (int i = 0; i < rows; ++i) {
            const int t = trow + i * step;
            const bool on = t < valid && v0 + tcol < A.Dv;
            ov[i].keep(on);
            vv[i].keep(on);
            put4(L.x, t, tcol, xv[i]);
            put4(L.r, t, tcol, r4[i]);
            ov[i].put(L.o, t, tcol);
#pragma unroll
            for (int e = 0; e < 4; ++e) rv[i] += r4[i][e] * vv[i].get(e);
            if (on)
                store4(dvp + t * A.Hv * A.Dv + v0, beta_own[i] * r4[i]);
        }
        __syncthreads();
        if constexpr (AHEAD)
            if (v0 + 32 < DVP) fetch(v0 + 32);
        // operands of the wave's tokens (left or right alike)
        Frag<NI> of[2];
        Frag<NC> xf[2], rf[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            of[i] = L.o.rows_in_order(2 * th + i, 0, lane);
            xf[i] = L.x.rows_in_order(2 * th + i, 0, lane);
            rf[i] = L.r.rows_in_order(2 * th + i, 0, lane);
        }
        if (!last_share) {
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int at = KQ == 2 ? i : kh;
                if (at == 0) {
                    mul(dp[i], of[0], xf[0]);
                    mul(nn[i], rf[0], xf[0]);
                } else if (at == 1) {
                    mul(dp[i], of[1], xf[0]);
                    mul(nn[i], rf[1], xf[0]);
                } else {
                    mul(dp[i], of[1], xf[1]);
                    mul(nn[i], rf[1], xf[1]);
                }
            }
        } else {
            const Frag<NI> o = L.o.rows_in_order(2 + th, 0, lane);
            const Frag<NC> g = L.r.rows_in_order(2 + th, 0, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Frag<NC> x = L.x.rows_in_order(i, 0, lane);
                mul(dp[i], o, x);
                mul(nn[i], g, x);
            }
        }
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const Frag<NC> f = L.s.columns_in_order(kh * KW + j, 0, lane);
            const Frag<NC> g = L.d.columns_in_order(kh * KW + j, 0, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mul(dq[i][j], of[i], f);
                mul(left[i][j], rf[i], f);
                mul(right[i][j], xf[i], g);
            }
        }
    }
    __syncthreads();
    if constexpr (!AHEAD) bring();
    ks.store(L.k, valid, A.Dk, threadIdx.x);
    qs.store(L.q, valid, A.Dk, threadIdx.x);
    // N and dP with their decays, to LDS
    const auto place_tiles = [&](bool again) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            if (i >= (last_share ? 2 : OWN)) break;
            const int at = KQ == 2 ? i : kh;
            const int tb = last_share ? 2 + th : 2 * th + (at > 0),
                      sb = last_share ? i : 2 * th + (at > 1);
            const int s = 16 * sb + r;
            const double Gs = L.G[s];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = 16 * tb + 4 * q + e;
                uint32_t u[NC];
                if (!again) {
                    const float E_ = s <= t ? exp2_of(L.G[t] - Gs) : 0.f;
                    nn[i][e] = s < t ? nn[i][e] * E_ : 0.f;
                    split2<NC>(nn[i][e],
                               s <= t ? dp[i][e] * (A.scale * E_) : 0.f, u);
                } else {
                    split2<NC>(-L.beta[t] * nn[i][e], 0.f, u);
                }
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    L.n.x[n][t][s] = bf16_t(u[n]);
                    if (!again) L.p.x[n][t][s] = bf16_t(u[n] >> 16);
                }
            }
        }
    };
    place_tiles(false);
    // (the blocks right of the diagonal that share a pair with it)
    if (kh == 0) {
        const int t = 32 * th + r, s = 32 * th + 16 + 4 * q;
#pragma unroll
        for (int n = 0; n < NC; ++n)
            *reinterpret_cast<uint2*>(&L.n.x[n][t][s]) =
                *reinterpret_cast<uint2*>(&L.p.x[n][t][s]) = make_uint2(0, 0);
    }
    __syncthreads();
    // the rows' factors, t = 16 (2 th + i) + 4q + e
    float kfirst = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 16 * (2 * th + i) + 4 * q;
        const f32x4_t first = four(L.first + row), last = four(L.last + row);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            dq[i][j] *= A.scale * first;
            left[i][j] *= first;
            right[i][j] *= last;
            const f32x4_t x = L.k.values(16 * (2 * th + i) + 4 * q, kh * KW + j, lane) *
                              right[i][j];
            kfirst += (x[0] + x[1]) + (x[2] + x[3]);
        }
    }
    // left, with the other sign, and dP^T Q; (beta N)^T K after them, since
    // beta belongs to the rows of N, which it contracts
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        if (p <= th) {
            Frag<NC> a[2], n[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = L.p.rows_in_order(2 * th + i, p, lane);
                n[i] = L.n.rows_in_order(2 * th + i, p, lane);
            }
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                const Frag<NI> f = L.k.columns_in_order(kh * KW + j, p, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mul(dq[i][j], a[i], f);
                    mul(left[i][j], n[i], f);
                }
            }
        }
        if (p >= th) {
            Frag<NC> a[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) a[i] = L.p.columns_in_order(2 * th + i, p, lane);
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                const Frag<NI> f = L.q.columns_in_order(kh * KW + j, p, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i) mul(right[i][j], a[i], f);
            }
        }
    }
    __syncthreads();
    place_tiles(true);
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        if (p < th) continue;
        Frag<NC> n[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) n[i] = L.n.columns_in_order(2 * th + i, p, lane);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const Frag<NI> f = L.k.columns_in_order(kh * KW + j, p, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i) mul(right[i][j], n[i], f);
        }
    }
    // the gates' gradients
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f32x4_t kleft = zero4(), dg = zero4();
        const int row = 16 * (2 * th + i);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const f32x4_t kv = L.k.values(row + 4 * q, kh * KW + j, lane);
            left[i][j] = -left[i][j];
            dg += L.q.values(row + 4 * q, kh * KW + j, lane) * dq[i][j] -
                  kv * right[i][j];
            kleft += kv * left[i][j];
        }
        dg += four(L.beta + row + 4 * q) * kleft;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = sum16(dg[e]), y = sum16(kleft[e]);
            if (r < 2) L.dots[kh][r][row + 4 * q + e] = r ? y : x;
        }
    }
#pragma unroll
    for (int i = 0; i < rows; ++i) {
        rv[i] = group_sum<8>(rv[i]);
        if (threadIdx.x % 8 == 0) L.rv[trow + i * step] = rv[i];
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        ds += __shfl_xor(ds, m);
        kfirst += __shfl_xor(kfirst, m);
    }
    if (lane == 0) L.sums[wave] = L.first[C - 1] * ds + kfirst;
    __syncthreads();
    if (wave == 0) {
        const auto dot = [&](int i) {
            float sum = L.dots[0][i][lane];
#pragma unroll
            for (int k = 1; k < KQ; ++k) sum += L.dots[k][i][lane];
            return sum;
        };
        double x = dot(0), end = 0.0;  // <D, S_L> at the chunk's last token
#pragma unroll
        for (int w = 0; w < 2 * KQ; ++w) end += L.sums[w];
        if (lane == 63) x += end;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double y = __shfl_down(x, m);
            if (lane + m < 64) x += y;
        }
        if (lane < valid) {
            const int64_t at = (b * A.T + t0 + lane) * A.Hv + h;
            store_gate(A.dg, A.g_bf16, at, float(x));
            store_gate(A.dbeta, A.beta_bf16, at, dot(1) + L.rv[lane]);
        }
    }
    if (A.dq_part) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 16 * (2 * th + i) + 4 * q;
            const f32x4_t beta = four(L.beta + row);
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                const int col = 16 * (kh * KW + j) + r;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (row + e >= valid || col >= A.Dk) continue;
                    const int64_t at =
                        ((b * A.T + t0 + row + e) * A.Hv + h) * A.Dk + col;
                    A.dq_part[at] = dq[i][j][e];
                    A.dk_part[at] = beta[e] * left[i][j][e] + right[i][j][e];
                }
            }
        }
        return;
    }
    // dq and dk through LDS to whole rows (k and q are done with: the barrier
    // above is behind their last reads)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 16 * (2 * th + i) + 4 * q;
        const f32x4_t beta = four(L.beta + row);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const int col = 16 * (kh * KW + j) + r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                store_f(&L.out[0][row + e][col], dq[i][j][e]);
                store_f(&L.out[1][row + e][col],
                        beta[e] * left[i][j][e] + right[i][j][e]);
            }
        }
    }
    __syncthreads();
    constexpr int per16 = 16 / sizeof(E), per_row = DKP / per16;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        E* to = static_cast<E*>(m ? A.dk : A.dq) +
                ((b * A.T + t0) * A.Hk + hk) * A.Dk;
#pragma unroll
        for (int i = 0; i < C * per_row / NT; ++i) {
            const int u = i * NT + int(threadIdx.x);
            const int row = u / per_row, col = per16 * (u % per_row);
            if (row < valid && col < A.Dk)
                *reinterpret_cast<u32x4_t*>(to + row * A.Hk * A.Dk + col) =
                    *reinterpret_cast<const u32x4_t*>(&L.out[m][row][col]);
        }
    }
}

// The shares of the value heads that read one key head, added up in their
// order: four places a thread.
constexpr int GROUP = 256;  // threads

template <typename E>
__global__ void __launch_bounds__(GROUP)
gdr_group_kernel(const GdrArgs A, int64_t n) {
    const int per = int(A.Hv / A.Hk);
    const int64_t quads = A.Dk / 4;
    for (int64_t i = int64_t(blockIdx.x) * GROUP + threadIdx.x; i < n;
         i += int64_t(gridDim.x) * GROUP) {
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
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)),
                       dim3(128 * kShares<E, KT>), lds, stream, A);
    e = hipGetLastError();
    if (e != hipSuccess || !A.dq_part) return e;
    const int64_t n = A.B * A.T * A.Hk * (A.Dk / 4);
    int64_t blocks = (n + GROUP - 1) / GROUP;
    if (blocks > 8192) blocks = 8192;
    hipLaunchKernelGGL(gdr_group_kernel<E>, dim3(unsigned(blocks)), dim3(GROUP),
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
