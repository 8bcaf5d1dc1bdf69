// Verification of drafted tokens (include/rwkv7m_lm_head.h has the rule): with
// p = softmax(target / T) and q = softmax(draft / T), drafts are taken while
// u q(x) < p(x), and a token is drawn behind them from max(p - q, 0), or from
// p where all were taken.
//
// Two launches.  The first reads every row once, in parts of 8192 logits, and
// leaves each part's largest logit and sum; the second decides and draws: the
// workgroups of a sequence, one a part of the vocabulary, each find the number
// taken (a few sums), add up their part of the one row that is drawn from, and
// the last of them to finish finds the token within its part.  Which one is
// last changes nothing: the parts' sums are added in their order.
//
// What is drawn lies next to a border of a sum over 65536 numbers, one sample
// in 500 within fp32's rounding of it: exponentials and sums are float64 (a
// wave takes float64 multiply-adds at fp32's rate; 11 of them an exponential).
// The rows' bytes stay what bounds the call.

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int NT = 256;
constexpr int PART = kVerifyPart;

// 2^t for t <= 0: 2^round(t) times the exponential series of the rest, |rest|
// ln 2 <= 0.347, off by 0.347^12 / 12! = 6e-15.
__device__ __forceinline__ double exp2_64(double t) {
    t = __builtin_fmax(t, -1100.0);
    const double n = __builtin_rint(t), y = (t - n) * 0.6931471805599453094;
    double s = 1.0 / 39916800.0;
    s = __builtin_fma(s, y, 1.0 / 3628800.0);
    s = __builtin_fma(s, y, 1.0 / 362880.0);
    s = __builtin_fma(s, y, 1.0 / 40320.0);
    s = __builtin_fma(s, y, 1.0 / 5040.0);
    s = __builtin_fma(s, y, 1.0 / 720.0);
    s = __builtin_fma(s, y, 1.0 / 120.0);
    s = __builtin_fma(s, y, 1.0 / 24.0);
    s = __builtin_fma(s, y, 1.0 / 6.0);
    s = __builtin_fma(s, y, 0.5);
    s = __builtin_fma(s, y, 1.0);
    s = __builtin_fma(s, y, 1.0);
    return __builtin_amdgcn_ldexp(s, int(n));
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

// Drafts of sequence b: 0 .. K.
__device__ __forceinline__ int drafted(const LmVerifyArgs& A, int64_t b) {
    if (!A.lengths) return A.K;
    const int64_t n = A.lengths[b];
    return int(n < 0 ? 0 : n > A.K ? A.K : n);
}

// A part of a row in registers: vectors i * NT + thread of 16 bytes, -inf
// behind the row's end.
template <typename E>
struct Part {
    static constexpr int n = Vec<E>::n, nv = PART / n / NT;
    Vec<E> v[nv];
    int first;

    __device__ __forceinline__ Part(const E* row, int64_t at, int64_t V)
        : first(int(at)) {
        const int count = int(V - at < PART ? V - at : PART);
        const E* x = row + at;
#pragma unroll
        for (int i = 0; i < nv; ++i) {
            const int j = (i * NT + int(threadIdx.x)) * n;
            v[i].raw = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
            if (j + n <= count) {
                v[i].load(x + j);
            } else if (j < count) {
                // (the row's last, shorter one; each place by itself)
#pragma unroll
                for (int u = 0; u < n; ++u)
                    if (j + u < count) {
                        if constexpr (sizeof(E) == 4)
                            v[i].raw[u] = __float_as_uint(load_f(x + j + u));
                        else
                            v[i].raw[u >> 1] =
                                u & 1 ? (v[i].raw[u >> 1] & 0xffffu) |
                                            uint32_t(x[j + u]) << 16
                                      : (v[i].raw[u >> 1] & 0xffff0000u) |
                                            uint32_t(x[j + u]);
                    }
            }
        }
    }
    __device__ __forceinline__ int id(int i, int u) const {
        return first + (i * NT + int(threadIdx.x)) * n + u;
    }
};

template <typename E>
__device__ __forceinline__ const E* row_of(const void* x, const LmRows& R,
                                           int64_t row) {
    return static_cast<const E*>(x) + row_offset(R, row);
}

// Each part's largest logit, the lowest id that has it, and the sum of 2^((x -
// largest) c).  Rows 0 .. n of the target, 0 .. n - 1 of the draft.
template <typename E>
__global__ void __launch_bounds__(NT)
verify_stats_kernel(const LmVerifyArgs A) {
    __shared__ float largest[NT / 64];
    __shared__ int ids[NT / 64];
    __shared__ double sums[NT / 64];
    const int rows = A.draft ? 2 * A.K + 1 : A.K + 1;
    const int64_t id = grid_row();
    if (id >= A.B * rows * A.parts) return;
    const int part = int(id % A.parts);
    const int64_t row = id / A.parts, b = row / rows;
    const int i = int(row % rows);
    if (i == 0 && part == 0 && threadIdx.x == 0) A.arrived[b] = 0;
    const int n = drafted(A, b);
    const bool target = i <= A.K;
    if (target ? i > n : i - A.K - 1 >= n) return;
    const E* x = target ? row_of<E>(A.target, A.tr, b * (A.K + 1) + i)
                        : row_of<E>(A.draft, A.dr, b * A.K + i - A.K - 1);
    const Part<E> P(x, int64_t(part) * PART, A.V);
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < P.nv; ++j)
#pragma unroll
        for (int u = 0; u < P.n; ++u) m = larger(m, P.v[j].get(u));
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    m = lanes_larger<64>(m);
    if (lane == 0) largest[wave] = m;
    __syncthreads();
    m = waves_larger<NT / 64>(largest);
    double s = 0.0;
    int best = 0x7fffffff;
    if (A.greedy) {
#pragma unroll
        for (int j = P.nv - 1; j >= 0; --j)
#pragma unroll
            for (int u = P.n - 1; u >= 0; --u)
                if (P.v[j].get(u) == m) best = P.id(j, u);
        best = lanes_fold<64>(best, [](int a, int c) { return a < c ? a : c; });
    } else if (m > -__builtin_inff() && m < __builtin_inff()) {
#pragma unroll
        for (int j = 0; j < P.nv; ++j)
#pragma unroll
            for (int u = 0; u < P.n; ++u)
                s += exp2_64((double(P.v[j].get(u)) - double(m)) * A.c);
        s = wave_sum(s);
    }
    if (lane == 0) {
        sums[wave] = s;
        ids[wave] = best;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < NT / 64; ++w) {
            s += sums[w];
            best = ids[w] < best ? ids[w] : best;
        }
        A.stats[id] = {s, m, best};
    }
}

// A row's largest logit and 1 / sum 2^((x - largest) c); largest NaN where it
// has no softmax (NaN or +inf, nothing above -inf).
struct RowSums {
    float largest;
    int id;
    double inv;
};
__device__ __forceinline__ RowSums join(const LmVerifyStats* s, int parts,
                                        double c) {
    float m = -__builtin_inff();
    int id = -1;
    for (int i = 0; i < parts; ++i) {
        const float x = s[i].largest;
        if (x > m) id = s[i].id;
        m = larger(m, x);
    }
    if (!(m > -__builtin_inff() && m < __builtin_inff()))
        return {__builtin_nanf(""), -1, __builtin_nan("")};
    double sum = 0.0;
    for (int i = 0; i < parts; ++i)
        if (s[i].largest > -__builtin_inff())
            sum += s[i].sum * exp2_64((double(s[i].largest) - double(m)) * c);
    return {m, id, 1.0 / sum};
}
__device__ __forceinline__ double prob(const RowSums& r, float x, double c) {
    return exp2_64((double(x) - double(r.largest)) * c) * r.inv;
}

struct DrawShared {
    RowSums rows[2 * kVerifyMostDrafts + 1];
    int taken, last;
    double waves[2][NT / 64];
    int found[NT / 64], positive[NT / 64];
};

template <typename E>
__global__ void __launch_bounds__(NT)
verify_draw_kernel(const LmVerifyArgs A) {
    __shared__ DrawShared S;
    const int64_t id = grid_row();
    const int parts = A.greedy ? 1 : A.parts;
    if (id >= A.B * parts) return;
    const int64_t b = id / parts;
    const int part = int(id % parts), t = threadIdx.x;
    const int lane = t % 64, wave = t / 64;
    const int n = drafted(A, b), rows = A.draft ? 2 * A.K + 1 : A.K + 1;
    const int64_t* drafts = A.tokens + b * A.K;
    const LmVerifyStats* stats = A.stats + b * rows * A.parts;
    // (rows 0 .. n of the target, then those of the draft)
    for (int i = t; i < n + 1 + (A.draft ? n : 0); i += NT) {
        const int row = i <= n ? i : A.K + 1 + i - (n + 1);
        S.rows[i] = join(stats + int64_t(row) * A.parts, A.parts, A.c);
    }
    __syncthreads();
    if (wave == 0) {
        // draft `lane` of each 64
        int taken = n;
        for (int base = 0; base < A.K; base += 64) {
            const int i = base + lane;
            bool stop = false;
            if (i < A.K) {
                double p = 0.0, q = 0.0;
                float chance = 0.f;
                if (i < n) {
                    const int64_t x = drafts[i];
                    const bool word = x >= 0 && x < A.V;
                    const RowSums &r = S.rows[i];
                    if (A.greedy) {
                        p = word && x == r.id ? 1.0 : 0.0;
                        q = 1.0;
                        stop = p == 0.0;
                    } else {
                        q = 1.0;
                        if (word) {
                            p = prob(r, load_f(row_of<E>(A.target, A.tr,
                                                         b * (A.K + 1) + i) + x),
                                     A.c);
                            if (A.draft)
                                q = prob(S.rows[n + 1 + i],
                                         load_f(row_of<E>(A.draft, A.dr,
                                                          b * A.K + i) + x),
                                         A.c);
                        }
                        stop = !(double(A.accept[b * A.K + i]) * q < p);
                    }
                    chance = p >= q ? p > 0.0 ? 1.f : 0.f : float(p / q);
                }
                if (part == 0) A.chance[b * A.K + i] = chance;
            }
            const uint64_t stops = __builtin_amdgcn_ballot_w64(stop);
            if (stops && taken == n) taken = base + __builtin_ctzll(stops);
        }
        if (lane == 0) S.taken = taken;
    }
    __syncthreads();
    const int m = S.taken;
    const RowSums P = S.rows[m];
    const bool residual = m < n;
    const bool with_q = residual && A.draft;
    const RowSums Q = with_q ? S.rows[n + 1 + m] : RowSums{0.f, 0, 0.0};
    const bool none = !(P.largest == P.largest) || !(Q.largest == Q.largest);
    int64_t* out = A.out + b * (A.K + 1);
    const auto finish = [&](int64_t token) {
        for (int i = 0; i <= A.K; ++i)
            out[i] = i < m ? drafts[i] : i == m ? token : -1;
        A.taken[b] = m;
    };
    if (A.greedy || none) {
        if (part == 0 && t == 0) finish(none ? -1 : P.id);
        return;
    }
    const int64_t without = residual && !A.draft ? drafts[m] : -1;
    const E* x = row_of<E>(A.target, A.tr, b * (A.K + 1) + m);
    const E* y = with_q ? row_of<E>(A.draft, A.dr, b * A.K + m) : x;
    const auto mass = [&](float xv, float yv, int64_t j, double& p) {
        p = prob(P, xv, A.c);
        if (with_q) return __builtin_fmax(p - prob(Q, yv, A.c), 0.0);
        return j == without ? 0.0 : p;
    };
    double sum = 0.0, whole = 0.0;
    {
        const Part<E> a(x, int64_t(part) * PART, A.V);
        const Part<E> d(y, int64_t(part) * PART, A.V);
#pragma unroll
        for (int i = 0; i < a.nv; ++i)
#pragma unroll
            for (int u = 0; u < a.n; ++u) {
                double p;
                sum += mass(a.v[i].get(u), d.v[i].get(u), a.id(i, u), p);
                whole += p;
            }
    }
    sum = wave_sum(sum);
    whole = wave_sum(whole);
    if (lane == 0) {
        S.waves[0][wave] = sum;
        S.waves[1][wave] = whole;
    }
    __syncthreads();
    double* masses = A.masses + b * 2 * A.parts;
    if (t == 0) {
        for (int w = 1; w < NT / 64; ++w) {
            sum += S.waves[0][w];
            whole += S.waves[1][w];
        }
        __hip_atomic_store(masses + part, sum, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(masses + A.parts + part, whole, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        S.last = __hip_atomic_fetch_add(A.arrived + b, 1, __ATOMIC_ACQ_REL,
                                        __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    }
    __syncthreads();
    if (!S.last) return;
    // the sequence's last workgroup: the part that the draw falls into
    const auto mass_of = [&](int which, int i) {
        return __hip_atomic_load(masses + which * A.parts + i, __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT);
    };
    double total = 0.0;
    for (int i = 0; i < parts; ++i) total += mass_of(0, i);
    // p where nothing is left of it (p = q, to rounding)
    const bool plain = !(total > 0.0);
    if (plain) {
        total = 0.0;
        for (int i = 0; i < parts; ++i) total += mass_of(1, i);
    }
    const float u_ = A.sample[b];
    const double u = total * double(u_ > 0.f ? u_ : 0.f);
    double before = 0.0;
    int at = -1;
    for (int i = 0; i < parts; ++i) {
        const double w = mass_of(plain, i);
        if (w > 0.0) at = i;  // (the last that holds anything, if none crosses)
        if (before + w > u) break;
        if (i + 1 < parts) before += w;
    }
    // its tokens in their order, PART / NT adjoining ones a thread
    constexpr int per = PART / NT;
    const int64_t j0 = int64_t(at) * PART + t * per;
    double mine = 0.0;
    const auto weight = [&](int64_t j) {
        if (j >= A.V) return 0.0;
        double p;
        const double w = mass(load_f(x + j), load_f(y + j), j, p);
        return plain ? p : w;
    };
#pragma unroll 4
    for (int i = 0; i < per; ++i) mine += weight(j0 + i);
    double upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double z = __shfl_up(upto, s);
        if (lane >= s) upto += z;
    }
    __syncthreads();
    if (lane == 63) S.waves[0][wave] = upto;
    __syncthreads();
    double ahead = 0.0;
    for (int i = 0; i < at; ++i) ahead += mass_of(plain, i);
    for (int w = 0; w < wave; ++w) ahead += S.waves[0][w];
    // the first token whose sum passes u, and the last that has any mass
    int found = 0x7fffffff, positive = -1;
    if (mine > 0.0) {
        double run = ahead + (upto - mine);
        for (int i = 0; i < per; ++i) {
            const double w = weight(j0 + i);
            run += w;
            if (w > 0.0) {
                positive = int(j0 + i);
                if (run > u && found == 0x7fffffff) found = int(j0 + i);
            }
        }
    }
    found = lanes_fold<64>(found, [](int a, int c) { return a < c ? a : c; });
    positive = lanes_fold<64>(positive, [](int a, int c) { return a > c ? a : c; });
    if (lane == 0) {
        S.found[wave] = found;
        S.positive[wave] = positive;
    }
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < NT / 64; ++w) {
            found = S.found[w] < found ? S.found[w] : found;
            positive = S.positive[w] > positive ? S.positive[w] : positive;
        }
        finish(found != 0x7fffffff ? found : positive);
    }
}

template <typename E>
hipError_t launch(const LmVerifyArgs& A, hipStream_t stream) {
    const int64_t rows = A.draft ? 2 * A.K + 1 : A.K + 1;
    hipLaunchKernelGGL(verify_stats_kernel<E>, row_grid(A.B * rows * A.parts),
                       dim3(NT), 0, stream, A);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(verify_draw_kernel<E>,
                       row_grid(A.B * (A.greedy ? 1 : A.parts)), dim3(NT), 0,
                       stream, A);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lm_verify(bool bf16, const LmVerifyArgs& A,
                            hipStream_t stream) {
    return bf16 ? launch<bf16_t>(A, stream) : launch<float>(A, stream);
}

}  // namespace rwkv7m
