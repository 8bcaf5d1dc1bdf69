// Verification of drafted tokens (include/rwkv7m_lm_head.h has the rule): with
// p = softmax(target / T) and q = softmax(draft / T), drafts are taken while
// u q(x) < p(x), and a token is drawn behind them from max(p - q, 0), or from
// p where all were taken.
//
// Two launches.  The first reads every row once, in parts of 8192 logits, and
// leaves each part's largest logit and sum; the second decides and draws: the
// workgroups of a sequence, one a part of the vocabulary, each find the number
// taken (a few sums), add up their part of the one row that is drawn from in
// segments of 64 vectors, and the last of them to finish finds the token within
// its segment.  Which one is last changes nothing: the segments' sums are added
// in their order.
//
// What is drawn lies next to a border of a sum over 65536 numbers, one sample
// in 500 within fp32's rounding of it: exponentials and sums are float64, which
// costs the first launch as much as its bytes (a wave takes float64
// multiply-adds at fp32's rate, 16 operations a logit).  An exponential off by
// 1e-12 moves one sample in ten million.
//
// 96 sequences of 0 to 5 drafts, 65536 bf16 logits a row: 36.5 + 24 us.  The
// first launch reads 75 MB, 2.1 TB/s, bound by its float64 operations: the vector
// units are active 85 % of the time that CUs are busy, which they are for 70 % of
// it.  Rows past a sequence's drafts are not read.  One sequence of 4: 4 + 12
// us, the second launch's latency (the sums of the parts, the count, the segment
// and the token within it, one after the other).  Greedy, without exponentials
// and a draw, 96 of 5: 18.5 us, 4.1 TB/s.

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int NT = 256, DRAW = 512;  // threads
constexpr int PART = kVerifyPart;

// 2^t for t <= 0: 2^round(t) times the polynomial that meets 2^x at the nine
// Chebyshev nodes of [-1/2, 1/2], off by 1.1e-12.  The rounding and the power
// are additions (1.5 2^52 leaves the whole number in the low bits; it is added
// to the exponent), since float64's rounding, conversion and scaling
// instructions run at a fraction of its additions' rate.  Below -1000 2^-1000.
__device__ __forceinline__ double exp2_64(double t) {
    t = __builtin_fmax(t, -1000.0);
    const double big = 6755399441055744.0, n = t + big, x = t - (n - big);
    double s = 1.325522488583589e-06;
    s = __builtin_fma(s, x, 1.5310079402360393e-05);
    s = __builtin_fma(s, x, 0.00015403455852412883);
    s = __builtin_fma(s, x, 0.0013333450568000116);
    s = __builtin_fma(s, x, 0.009618129159402631);
    s = __builtin_fma(s, x, 0.055504109412059334);
    s = __builtin_fma(s, x, 0.2402265069581299);
    s = __builtin_fma(s, x, 0.6931471805459335);
    s = __builtin_fma(s, x, 1.0);
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    const uint32_t k = uint32_t(__builtin_bit_cast(uint64_t, n));
    return __builtin_bit_cast(
        double, u + (uint64_t(k << 20) << 32));
}

// x of another lane by a DPP control (0 where there is none), as two words.
template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    i32x2 u = __builtin_bit_cast(i32x2, x);
    u[0] = __builtin_amdgcn_update_dpp(0, u[0], CTRL, 0xf, 0xf, true);
    u[1] = __builtin_amdgcn_update_dpp(0, u[1], CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, u);
}
__device__ __forceinline__ double lane64(double x, int lane) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    i32x2 u = __builtin_bit_cast(i32x2, x);
    u[0] = __builtin_amdgcn_readlane(u[0], lane);
    u[1] = __builtin_amdgcn_readlane(u[1], lane);
    return __builtin_bit_cast(double, u);
}
// Sums over a wave without LDS: a shuffle of a double is two round trips
// through it, and there are twelve in a sum's way (they were a third of a
// single sequence's time).
__device__ __forceinline__ double row_sum(double x) {  // rows of 16 lanes
    x += dpp64<0x128>(x);
    x += dpp64<0x124>(x);
    x += dpp64<0x122>(x);
    return x + dpp64<0x121>(x);
}
__device__ __forceinline__ double wave_sum(double x) {
    x = row_sum(x);
    return (lane64(x, 0) + lane64(x, 16)) + (lane64(x, 32) + lane64(x, 48));
}
// The sum over the lanes up to and with the calling one; `all`: over all.
__device__ __forceinline__ double wave_scan(double x, double* all) {
    x += dpp64<0x111>(x);
    x += dpp64<0x112>(x);
    x += dpp64<0x114>(x);
    x += dpp64<0x118>(x);
    const int row = threadIdx.x % 64 / 16;
    const double a = lane64(x, 15), b = lane64(x, 31), c = lane64(x, 47);
    *all = (a + b) + (c + lane64(x, 63));
    return x + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? a + b : (a + b) + c);
}

// Drafts of sequence b: 0 .. K.
__device__ __forceinline__ int drafted(const LmVerifyArgs& A, int64_t b) {
    if (!A.lengths) return A.K;
    const int64_t n = A.lengths[b];
    return int(n < 0 ? 0 : n > A.K ? A.K : n);
}

// A part of a row in registers: vectors i * NT + thread of 16 bytes, -inf
// behind the row's end.
template <typename E, int NT>
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
    // (32 bits, which hold every id: a 64-bit division is 130 instructions)
    const uint32_t row32 = uint32_t(id) / uint32_t(A.parts);
    const int part = int(uint32_t(id) % uint32_t(A.parts));
    const int64_t row = row32, b = row32 / uint32_t(rows);
    const int i = int(row32 % uint32_t(rows));
    if (i == 0 && part == 0 && threadIdx.x == 0) A.arrived[b] = 0;
    const int n = drafted(A, b);
    const bool target = i <= A.K;
    if (target ? i > n : i - A.K - 1 >= n) return;
    const E* x = target ? row_of<E>(A.target, A.tr, b * (A.K + 1) + i)
                        : row_of<E>(A.draft, A.dr, b * A.K + i - A.K - 1);
    // (the row's drafted token, for the second launch to have at hand)
    const int which = target ? i : i - A.K - 1;
    if (part == 0 && threadIdx.x == 0 && which < n) {
        const int64_t word = A.tokens[b * A.K + which];
        A.picked[row] = word >= 0 && word < A.V ? load_f(x + word)
                                                : -__builtin_inff();
    }
    const Part<E, NT> P(x, int64_t(part) * PART, A.V);
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
// By 16 lanes, the same in each.
__device__ __forceinline__ RowSums join(const LmVerifyStats* s, int parts,
                                        double c) {
    const int l = threadIdx.x % 16;
    float m = -__builtin_inff();
    int id = 0x7fffffff;
    double sum = 0.0;
    for (int i = l; i < parts; i += 16) {
        const LmVerifyStats a = s[i];
        if (a.largest > m || a.largest != a.largest) {
            // (what came before, next to the new largest)
            sum = m > -__builtin_inff()
                      ? sum * exp2_64((double(m) - double(a.largest)) * c)
                      : 0.0;
            sum += a.sum;
            m = larger(m, a.largest);
            id = a.id;
        } else if (a.largest > -__builtin_inff()) {
            sum += a.sum * exp2_64((double(a.largest) - double(m)) * c);
        }
    }
    const float own = m;
    m = lanes_larger<16>(m);
    id = lanes_fold<16>(own == m ? id : 0x7fffffff,
                        [](int a, int b) { return a < b ? a : b; });
    if (!(m > -__builtin_inff() && m < __builtin_inff()))
        return {__builtin_nanf(""), -1, __builtin_nan("")};
    sum = own > -__builtin_inff()
              ? sum * exp2_64((double(own) - double(m)) * c)
              : 0.0;
    return {m, id, 1.0 / row_sum(sum)};
}
// (0 where exp2_64 holds at 2^-1000, for a logit of -inf above all: nothing
// masked may be drawn or taken, not by a random number of 0 either)
__device__ __forceinline__ double prob(const RowSums& r, float x, double c) {
    const double t = (double(x) - double(r.largest)) * c;
    return t < -1000.0 ? 0.0 : exp2_64(t) * r.inv;
}

struct DrawShared {
    RowSums rows[2 * kVerifyMostDrafts + 1];
    float picked[2 * kVerifyMostDrafts + 1];
    int taken, last;
};

template <typename E>
__global__ void __launch_bounds__(DRAW)
verify_draw_kernel(const LmVerifyArgs A) {
    __shared__ DrawShared S;
    const int64_t id = grid_row();
    const int parts = A.greedy ? 1 : A.parts;
    if (id >= A.B * parts) return;
    const int64_t b = uint32_t(id) / uint32_t(parts);
    const int part = int(uint32_t(id) % uint32_t(parts)), t = threadIdx.x;
    const int lane = t % 64, wave = t / 64;
    const int n = drafted(A, b), rows = A.draft ? 2 * A.K + 1 : A.K + 1;
    const int64_t* drafts = A.tokens + b * A.K;
    const LmVerifyStats* stats = A.stats + b * rows * A.parts;
    // (also those past n, which hold anything and are not used: the loads do
    // not wait for n)
    for (int i = t / 16; i < (rows + 15) / 16 * 16; i += DRAW / 16) {
        const int row = i < rows ? i : rows - 1;
        const RowSums r = join(stats + int64_t(row) * A.parts, A.parts, A.c);
        if (t % 16 == 0 && i < rows) S.rows[i] = r;
    }
    static_assert(2 * kVerifyMostDrafts + 1 <= DRAW, "");
    if (t < rows) S.picked[t] = A.picked[b * rows + t];
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
                    const RowSums& r = S.rows[i];
                    if (A.greedy) {
                        p = word && x == r.id ? 1.0 : 0.0;
                        q = 1.0;
                        stop = p == 0.0;
                        if (r.largest != r.largest) p = r.inv;  // NaN
                    } else {
                        // (outside the vocabulary 0 of 1, or NaN where the
                        // rows have no distribution)
                        p = word ? prob(r, S.picked[i], A.c) : 0.0 * r.inv;
                        q = 1.0;
                        if (A.draft) {
                            const RowSums& d = S.rows[A.K + 1 + i];
                            q = word ? prob(d, S.picked[A.K + 1 + i], A.c)
                                     : 1.0 + 0.0 * d.inv;
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
    const RowSums Q = with_q ? S.rows[A.K + 1 + m] : RowSums{0.f, 0, 0.0};
    const bool none = !(P.largest == P.largest) || !(Q.largest == Q.largest);
    int64_t* out = A.out + b * (A.K + 1);
    const auto finish = [&](int64_t token) {
        if (wave == 0)
            for (int i = t; i <= A.K; i += 64)
                out[i] = i < m ? drafts[i] : i == m ? token : -1;
        if (t == 0) A.taken[b] = m;
    };
    if (A.greedy || none) {
        if (part == 0) finish(none ? -1 : P.id);
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
    // segments of the vocabulary: a wave's vectors i of its part, in their
    // order
    constexpr int nv = Part<E, DRAW>::nv, per_part = nv * (DRAW / 64),
                  width = PART / per_part, per = width / 64;
    static_assert(per_part <= kVerifySegments && per == Vec<E>::n, "");
    double* masses = A.masses + b * 2 * A.parts * kVerifySegments;
    const int64_t segments = int64_t(A.parts) * per_part;
    {
        const Part<E, DRAW> a(x, int64_t(part) * PART, A.V);
        const Part<E, DRAW> d(y, int64_t(part) * PART, A.V);
#pragma unroll
        for (int i = 0; i < nv; ++i) {
            double sum = 0.0, whole = 0.0;
#pragma unroll
            for (int u = 0; u < a.n; ++u) {
                double p;
                sum += mass(a.v[i].get(u), d.v[i].get(u), a.id(i, u), p);
                whole += p;
            }
            sum = wave_sum(sum);
            whole = wave_sum(whole);
            const int64_t at =
                int64_t(part) * per_part + i * (DRAW / 64) + wave;
            if (lane == 0) {
                __hip_atomic_store(masses + at, sum, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(masses + segments + at, whole,
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    // Each wave's sums are out before the workgroup is counted.  They are
    // written and read past the L2s (device-scope atomics), so that waiting for
    // the writes is all it takes: a device-scope release would write the whole
    // L2 back as well, a workgroup at a time (96 sequences: 73 us for 22).
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0)
        S.last = __hip_atomic_fetch_add(A.arrived + b, 1, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    __syncthreads();
    if (!S.last) return;
    // The sequence's last workgroup, one wave of it: the segment that the draw
    // falls into, four a lane and turn.
    if (wave) return;
    const auto four_masses = [&](int which, int64_t i, double (&w)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = i + k < segments
                       ? __hip_atomic_load(masses + which * segments + i + k,
                                           __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT)
                       : 0.0;
    };
    const float u_ = A.sample[b];
    double w0[2][4], total = 0.0, whole = 0.0;
    four_masses(0, 4 * lane, w0[0]);
    four_masses(1, 4 * lane, w0[1]);
    for (int64_t i = 0; i < segments; i += 256) {
        double w[2][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[0][k] = w0[0][k];
            w[1][k] = w0[1][k];
        }
        if (i) {
            four_masses(0, i + 4 * lane, w[0]);
            four_masses(1, i + 4 * lane, w[1]);
        }
        total += wave_sum((w[0][0] + w[0][1]) + (w[0][2] + w[0][3]));
        whole += wave_sum((w[1][0] + w[1][1]) + (w[1][2] + w[1][3]));
    }
    // p where nothing is left of it (p = q, to rounding)
    const bool plain = !(total > 0.0);
    const double u = (plain ? whole : total) * double(u_ > 0.f ? u_ : 0.f);
    // the first whose running sum passes u; the last that holds anything, if
    // rounding lets none pass
    double run = 0.0, before = 0.0;
    int segment = -1, last = -1;
    for (int64_t i = 0; i < segments && segment < 0; i += 256) {
        double w[4], all;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = plain ? w0[1][k] : w0[0][k];
        if (i) four_masses(plain, i + 4 * lane, w);
        const double sum = (w[0] + w[1]) + (w[2] + w[3]);
        double ahead = run + wave_scan(sum, &all) - sum;
        int mine = -1;
        double at = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (mine < 0 && w[k] > 0.0 && ahead + w[k] > u) {
                mine = int(i) + 4 * lane + k;
                at = ahead;
            }
            ahead += w[k];
            if (w[k] > 0.0) last = int(i) + 4 * lane + k;
        }
        const uint64_t passed = __builtin_amdgcn_ballot_w64(mine >= 0);
        if (passed) {
            const int l = __builtin_ctzll(passed);
            segment = __builtin_amdgcn_readlane(mine, l);
            before = lane64(at, l);
        }
        run += all;
    }
    if (segment < 0)
        segment =
            lanes_fold<64>(last, [](int a, int c) { return a > c ? a : c; });
    // its tokens in their order, adjoining ones a lane
    const int64_t j0 = int64_t(segment) * width + lane * per;
    double w[per], mine = 0.0, all;
#pragma unroll
    for (int i = 0; i < per; ++i) {
        const int64_t j = j0 + i;
        w[i] = 0.0;
        if (j < A.V) {
            double p;
            const double r = mass(load_f(x + j), load_f(y + j), j, p);
            w[i] = plain ? p : r;
        }
        mine += w[i];
    }
    before += wave_scan(mine, &all) - mine;
    int found = 0x7fffffff, positive = -1;
#pragma unroll
    for (int i = 0; i < per; ++i) {
        before += w[i];
        if (w[i] > 0.0) {
            positive = int(j0 + i);
            if (before > u && found == 0x7fffffff) found = int(j0 + i);
        }
    }
    found = lanes_fold<64>(found, [](int a, int c) { return a < c ? a : c; });
    positive = lanes_fold<64>(positive,
                              [](int a, int c) { return a > c ? a : c; });
    finish(found != 0x7fffffff ? found : positive);
}

template <typename E>
hipError_t launch(const LmVerifyArgs& A, hipStream_t stream) {
    const int64_t rows = A.draft ? 2 * A.K + 1 : A.K + 1;
    hipLaunchKernelGGL(verify_stats_kernel<E>, row_grid(A.B * rows * A.parts),
                       dim3(NT), 0, stream, A);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(verify_draw_kernel<E>,
                       row_grid(A.B * (A.greedy ? 1 : A.parts)), dim3(DRAW), 0,
                       stream, A);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lm_verify(bool bf16, const LmVerifyArgs& A,
                            hipStream_t stream) {
    return bf16 ? launch<bf16_t>(A, stream) : launch<float>(A, stream);
}

}  // namespace rwkv7m
