// Layer norm over the last axis, forward and backward
// (include/rwkv7m_lm_head.h has the formulas).
//
// Bound by memory: about 8 operations an element forward and 14 backward
// against 4 and 6 bytes.  A row is read once and held in registers, as the
// 16-byte vectors it came in, by a group of TPR threads (16 for up to 128
// bf16 elements, a wave, 4 or 16 waves), NV vectors each; the variance is the
// mean of the squared deviations, from the registers.  Rows longer than 16
// waves hold (kLongest) are walked again from the L2.  Workgroups stay for
// many rows, with the parameters, and in the backward their gradients' sums,
// in registers; each workgroup writes one partial row of those sums and a
// second kernel adds the partial rows in a fixed order.
// [32768, 2048] bf16 with fp32 parameters, medians under a profiler: forward
// 44 us (6.0 TB/s), backward 82 + 5 us (4.9 TB/s without the second kernel).
//
// A row whose length is no multiple of the vector ends in a vector moved back
// to end with it (its first `dup` elements are the vector before's): every
// access is whole, and what the two write twice is the same value.

#include "lm_rows.h"

namespace rwkv7m {
namespace {

__device__ __forceinline__ float param(const void* p, bool bf16, int64_t i,
                                       float absent) {
    if (!p) return absent;
    return bf16 ? bf16_to_f32(static_cast<const bf16_t*>(p)[i])
                : static_cast<const float*>(p)[i];
}

// N parameters from element i on, in 16-byte loads (8 for 4 bf16).
template <int N>
__device__ __forceinline__ void params(const void* p, bool bf16, int64_t i,
                                       float absent, float (&f)[N]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = absent;
    } else if (bf16) {
        typedef uint32_t half_t
            __attribute__((ext_vector_type(N / 2), aligned(2)));
        const half_t v = *reinterpret_cast<const half_t*>(
            static_cast<const bf16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < N; ++j)
            f[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xffff0000u
                                         : v[j / 2] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            Vec<float> v;
            v.load(static_cast<const float*>(p) + i + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) f[j + k] = v.get(k);
        }
    }
}

__device__ __forceinline__ void store_param(void* p, bool bf16, int64_t i,
                                            float x) {
    if (bf16)
        store_f(static_cast<bf16_t*>(p) + i, x);
    else
        store_f(static_cast<float*>(p) + i, x);
}

// Where a thread's vectors lie in a row of C elements.
template <typename E, int TPR, int NV, bool TAIL>
struct Place {
    static constexpr int n = Vec<E>::n;
    int C, lane;

    __device__ __forceinline__ bool has(int i) const {
        return (i * TPR + lane) * n < C;
    }
    __device__ __forceinline__ int at(int i) const {
        const int a = (i * TPR + lane) * n;
        return TAIL && a + n > C ? C - n : a;
    }
    __device__ __forceinline__ int dup(int i) const {
        return TAIL ? (i * TPR + lane) * n - at(i) : 0;
    }
};

template <int TPR>
constexpr int kFwdThreads = TPR > 256 ? TPR : 256;
constexpr int kBwdThreads = 1024;

// Sums over the TPR threads of a row, the same in each of them.  Where a row
// is more than a wave's the two buffers of `s` (a value a wave of the
// workgroup) take turns: one barrier a call.
template <int TPR, int K, int W>
__device__ __forceinline__ void row_sums(float (&x)[K], float (*s)[K][W],
                                         int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] = lanes_sum<TPR < 64 ? TPR : 64>(x[k]);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x / 64, first = wave / (TPR / 64) *
                                                   (TPR / 64);
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) s[turn][k][wave] = x[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            x[k] = s[turn][k][first];
#pragma unroll
            for (int w = 1; w < TPR / 64; ++w) x[k] += s[turn][k][first + w];
        }
        turn ^= 1;
    }
}

template <typename E, int TPR, int NV, bool TAIL>
__global__ __launch_bounds__(kFwdThreads<TPR>) void norm_fwd_kernel(
    LmNormArgs A) {
    constexpr int RPB = kFwdThreads<TPR> / TPR, n = Vec<E>::n;
    __shared__ float s[2][1][kFwdThreads<TPR> / 64];
    int turn = 0;
    const Place<E, TPR, NV, TAIL> at{int(A.C), int(threadIdx.x % TPR)};
    const float inv = 1.f / float(A.C);
    float w[NV][n], b[NV][n];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.has(i)) {
            params(A.weight, A.param_bf16, at.at(i), 1.f, w[i]);
            params(A.bias, A.param_bf16, at.at(i), 0.f, b[i]);
        }
    for (int64_t row = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
         row < A.rows; row += int64_t(gridDim.x) * RPB) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        E* y = static_cast<E*>(A.y) + row * A.C;
        Vec<E> v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i)) v[i].load(x + at.at(i));
        float sum[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i))
#pragma unroll
                for (int j = 0; j < n; ++j)
                    sum[0] += j < at.dup(i) ? 0.f : v[i].get(j);
        row_sums<TPR>(sum, s, turn);
        const float mean = sum[0] * inv;
        sum[0] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i))
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const float d = j < at.dup(i) ? 0.f : v[i].get(j) - mean;
                    sum[0] = __builtin_fmaf(d, d, sum[0]);
                }
        row_sums<TPR>(sum, s, turn);
        const float rstd = 1.f / sqrtf(sum[0] * inv + A.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i)) {
                Vec<E> o;
#pragma unroll
                for (int j = 0; j < n; j += 2)
                    o.set2(j,
                           __builtin_fmaf((v[i].get(j) - mean) * rstd, w[i][j],
                                          b[i][j]),
                           __builtin_fmaf((v[i].get(j + 1) - mean) * rstd,
                                          w[i][j + 1], b[i][j + 1]));
                o.store(y + at.at(i));
            }
        if (A.mean && threadIdx.x % TPR == 0) {
            A.mean[row] = mean;
            A.rstd[row] = rstd;
        }
    }
}

// One row's operands of the backward, as they came (zeros past the last row).
template <typename E, int NV>
struct BwdRow {
    Vec<E> x[NV], dy[NV];
    float mean, rstd;

    template <typename P>
    __device__ __forceinline__ void load(const LmNormArgs& A, int64_t row,
                                         const P& at) {
        mean = rstd = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i].raw = dy[i].raw = 0;
        if (row >= A.rows) return;
        const E* px = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        const E* pd = static_cast<const E*>(A.dy) + row * A.C;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i)) {
                x[i].load(px + at.at(i));
                dy[i].load(pd + at.at(i));
            }
        mean = A.mean[row];
        rstd = A.rstd[row];
    }
};

// dx, and the workgroup's partial row of the parameters' gradients:
// workspace[block][0 / 1][C] (weight, bias).  One workgroup of 16 waves a CU,
// kBwdThreads / TPR rows at a time, so that there are few partial rows
// (their 16 C bytes, written and read again, are what a workgroup adds to
// the 6 C of each of its rows in bf16).
template <typename E, int TPR, int NV, bool TAIL>
__global__ __launch_bounds__(kBwdThreads) void norm_bwd_kernel(LmNormArgs A) {
    constexpr int RPB = kBwdThreads / TPR, n = Vec<E>::n;
    constexpr int kCols = RPB > 1 ? TPR * NV * n : 1;
    // A thread with one vector a row asks for the next row's while it works
    // on this one's ([32768, 2048] bf16: 3 % less time); with two the waves
    // have enough in flight without ([16384, 4096]: 2 % more).
    constexpr bool kAhead = NV == 1;
    __shared__ float s[2][2][kBwdThreads / 64];
    __shared__ float part[RPB][2][kCols];
    int turn = 0;
    const Place<E, TPR, NV, TAIL> at{int(A.C), int(threadIdx.x % TPR)};
    const int group = threadIdx.x / TPR;
    const int64_t step = int64_t(gridDim.x) * RPB;
    const float inv = 1.f / float(A.C);
    float w[NV][n], dw[NV][n] = {}, db[NV][n] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.has(i)) params(A.weight, A.param_bf16, at.at(i), 1.f, w[i]);
    BwdRow<E, NV> v, next;
    if constexpr (kAhead) v.load(A, int64_t(blockIdx.x) * RPB + group, at);
    // (the workgroup's threads make the same number of turns)
    for (int64_t base = int64_t(blockIdx.x) * RPB; base < A.rows;
         base += step) {
        const int64_t row = base + group;
        if constexpr (kAhead)
            next.load(A, row + step, at);
        else
            v.load(A, row, at);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i))
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const float xh = (v.x[i].get(j) - v.mean) * v.rstd;
                    const float d = j < at.dup(i) ? 0.f : v.dy[i].get(j);
                    const float g = d * w[i][j];
                    sum[0] += g;
                    sum[1] = __builtin_fmaf(g, xh, sum[1]);
                    dw[i][j] = __builtin_fmaf(d, xh, dw[i][j]);
                    db[i][j] += d;
                }
        row_sums<TPR>(sum, s, turn);
        const float sg = sum[0] * inv, sgx = sum[1] * inv;
        if (A.dx && row < A.rows) {
            E* dx = static_cast<E*>(A.dx) + row * A.C;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at.has(i)) {
                    Vec<E> o;
                    float r[n];
#pragma unroll
                    for (int j = 0; j < n; ++j) {
                        const float xh = (v.x[i].get(j) - v.mean) * v.rstd;
                        r[j] = v.rstd * (__builtin_fmaf(v.dy[i].get(j),
                                                        w[i][j], -sg) -
                                         xh * sgx);
                    }
#pragma unroll
                    for (int j = 0; j < n; j += 2) o.set2(j, r[j], r[j + 1]);
                    o.store(dx + at.at(i));
                }
        }
        if constexpr (kAhead) v = next;
    }
    if (!A.workspace) return;
    float* out = A.workspace + int64_t(blockIdx.x) * 2 * A.C;
    if constexpr (RPB > 1) {
        // the row groups' sums side by side, added in the groups' order
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i))
#pragma unroll
                for (int j = 0; j < n; ++j)
                    if (j >= at.dup(i)) {
                        part[group][0][at.at(i) + j] = dw[i][j];
                        part[group][1][at.at(i) + j] = db[i][j];
                    }
        __syncthreads();
        for (int k = 0; k < 2; ++k)
            for (int c = threadIdx.x; c < A.C; c += kBwdThreads) {
                float x = part[0][k][c];
#pragma unroll
                for (int r = 1; r < RPB; ++r) x += part[r][k][c];
                out[k * A.C + c] = x;
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.has(i))
#pragma unroll
                for (int j = 0; j < n; ++j)
                    if (j >= at.dup(i)) {
                        out[at.at(i) + j] = dw[i][j];
                        out[A.C + at.at(i) + j] = db[i][j];
                    }
    }
}

// Any length, element by element: rows shorter than a vector, and those
// longer than kLongest (their second and third reads come from the L2).
constexpr int kThreads = 256, kWaves = kThreads / 64;

template <typename E>
__global__ __launch_bounds__(kThreads) void norm_fwd_any_kernel(LmNormArgs A) {
    __shared__ float s[kWaves];
    const float n = 1.f / float(A.C);
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        E* y = static_cast<E*>(A.y) + row * A.C;
        float sum = 0.f;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads)
            sum += load_f(x + i);
        const float mean = block_sum<kWaves>(sum, s) * n;
        float sq = 0.f;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads) {
            const float d = load_f(x + i) - mean;
            sq = __builtin_fmaf(d, d, sq);
        }
        const float rstd = 1.f / sqrtf(block_sum<kWaves>(sq, s) * n + A.eps);
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads)
            store_f(y + i,
                    __builtin_fmaf((load_f(x + i) - mean) * rstd,
                                   param(A.weight, A.param_bf16, i, 1.f),
                                   param(A.bias, A.param_bf16, i, 0.f)));
        if (threadIdx.x == 0 && A.mean) {
            A.mean[row] = mean;
            A.rstd[row] = rstd;
        }
    }
}

// The workgroup's partial row is kept in the workspace itself: each thread
// adds its rows to its own columns.
template <typename E>
__global__ __launch_bounds__(kThreads) void norm_bwd_any_kernel(LmNormArgs A) {
    __shared__ float s[kWaves];
    const float n = 1.f / float(A.C);
    float* part = A.workspace + int64_t(blockIdx.x) * 2 * A.C;
    bool first = true;
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        const E* dy = static_cast<const E*>(A.dy) + row * A.C;
        const float mean = A.mean[row], rstd = A.rstd[row];
        float sg = 0.f, sgx = 0.f;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads) {
            const float d = load_f(dy + i);
            const float xh = (load_f(x + i) - mean) * rstd;
            const float g = d * param(A.weight, A.param_bf16, i, 1.f);
            sg += g;
            sgx = __builtin_fmaf(g, xh, sgx);
            if (A.workspace) {
                part[i] = __builtin_fmaf(d, xh, first ? 0.f : part[i]);
                part[A.C + i] = d + (first ? 0.f : part[A.C + i]);
            }
        }
        first = false;
        if (!A.dx) continue;
        sg = block_sum<kWaves>(sg, s) * n;
        sgx = block_sum<kWaves>(sgx, s) * n;
        E* dx = static_cast<E*>(A.dx) + row * A.C;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads) {
            const float g =
                load_f(dy + i) * param(A.weight, A.param_bf16, i, 1.f);
            store_f(dx + i, rstd * (g - sg - (load_f(x + i) - mean) * rstd *
                                                 sgx));
        }
    }
}

// dweight and dbias from the partial rows [parts][2 C]: a block sums 64
// columns over 16 interleaved shares of the rows.
__global__ __launch_bounds__(1024) void norm_sum_kernel(LmNormArgs A,
                                                        int parts) {
    __shared__ float s[16][64];
    const int64_t c = int64_t(blockIdx.x) * 64 + threadIdx.x % 64;
    const int share = threadIdx.x / 64;
    float x = 0.f;
    if (c < 2 * A.C)
#pragma unroll 8
        for (int p = share; p < parts; p += 16)
            x += A.workspace[int64_t(p) * 2 * A.C + c];
    s[share][threadIdx.x % 64] = x;
    __syncthreads();
    if (share != 0 || c >= 2 * A.C) return;
    for (int k = 1; k < 16; ++k) x += s[k][threadIdx.x];
    void* out = c < A.C ? A.dweight : A.dbias;
    if (out) store_param(out, A.param_bf16, c < A.C ? c : c - A.C, x);
}

// Vectors a thread of a group below the widest holds.  The backward has four
// arrays of them in fp32 and one workgroup of 16 waves a CU: two, or too few
// waves have room ([32768, 2048] bf16 by waves of 4 vectors, in workgroups of
// 4, takes 12 % longer than by groups of 4 waves with one vector each).
constexpr int64_t kFwdVectors = 4, kBwdVectors = 2;
constexpr int64_t kFwdBlocks = 2048, kBwdBlocks = 256;

// Elements a row may have for the widest group (16 waves of 2 vectors each).
template <typename E>
constexpr int64_t kLongest = 1024 * 2 * Vec<E>::n;

// The group that holds a row of C elements: a quarter of a wave, a wave, 4
// or 16 waves; 0: none.
template <typename E>
int threads_per_row(int64_t C, bool backward) {
    const int64_t n = Vec<E>::n, nv = backward ? kBwdVectors : kFwdVectors;
    if (C < n || C > kLongest<E>) return 0;
    return C <= 16 * n ? 16 : C <= 64 * nv * n ? 64 : C <= 256 * nv * n ? 256
                                                                        : 1024;
}

// Workgroups for `rows` rows, `at_once` in each.
int64_t row_blocks(int64_t rows, int at_once, int64_t most) {
    const int64_t blocks = (rows + at_once - 1) / at_once;
    return blocks < most ? blocks : most;
}

using NormKernel = void (*)(LmNormArgs);

template <typename E, bool BWD, int TPR, int NV>
NormKernel pick_tail(int64_t C) {
    const bool tail = C % Vec<E>::n != 0;
    if constexpr (BWD)
        return tail ? norm_bwd_kernel<E, TPR, NV, true>
                    : norm_bwd_kernel<E, TPR, NV, false>;
    else
        return tail ? norm_fwd_kernel<E, TPR, NV, true>
                    : norm_fwd_kernel<E, TPR, NV, false>;
}

template <typename E, bool BWD, int TPR>
NormKernel pick_vectors(int64_t C) {
    const int64_t nv = (C + TPR * Vec<E>::n - 1) / (TPR * Vec<E>::n);
    if (nv == 1) return pick_tail<E, BWD, TPR, 1>(C);
    if (nv == 2) return pick_tail<E, BWD, TPR, 2>(C);
    if constexpr (!BWD && TPR < 1024) {
        if (nv == 3) return pick_tail<E, BWD, TPR, 3>(C);
        return pick_tail<E, BWD, TPR, 4>(C);
    }
    return nullptr;
}

template <typename E, bool BWD>
NormKernel pick(int64_t C, int tpr) {
    switch (tpr) {
    case 16: return pick_tail<E, BWD, 16, 1>(C);
    case 64: return pick_vectors<E, BWD, 64>(C);
    case 256: return pick_vectors<E, BWD, 256>(C);
    case 1024: return pick_vectors<E, BWD, 1024>(C);
    default:
        if constexpr (BWD)
            return norm_bwd_any_kernel<E>;
        else
            return norm_fwd_any_kernel<E>;
    }
}

}  // namespace

int64_t lm_norm_workspace_floats(int64_t rows, int64_t C) {
    return 2 * C * (rows < kBwdBlocks ? rows : kBwdBlocks);
}

hipError_t launch_lm_norm(bool bf16, const LmNormArgs& A, hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    const int tpr = bf16 ? threads_per_row<bf16_t>(A.C, false)
                         : threads_per_row<float>(A.C, false);
    const int threads = tpr > 256 ? tpr : 256;
    const NormKernel kern = bf16 ? pick<bf16_t, false>(A.C, tpr)
                                 : pick<float, false>(A.C, tpr);
    if (!kern) return hipErrorInvalidValue;
    const int64_t blocks =
        row_blocks(A.rows, tpr ? threads / tpr : 1, kFwdBlocks);
    hipLaunchKernelGGL(kern, dim3(unsigned(blocks)), dim3(unsigned(threads)),
                       0, stream, A);
    return hipGetLastError();
}

hipError_t launch_lm_norm_backward(bool bf16, const LmNormArgs& A,
                                   hipStream_t stream) {
    const bool params = A.dweight || A.dbias;
    const int tpr = bf16 ? threads_per_row<bf16_t>(A.C, true)
                         : threads_per_row<float>(A.C, true);
    const int threads = tpr ? kBwdThreads : kThreads;
    const int64_t blocks =
        row_blocks(A.rows, tpr ? threads / tpr : 1, kBwdBlocks);
    if (A.rows > 0 && (A.dx || params)) {
        LmNormArgs B = A;
        if (!params) B.workspace = nullptr;
        const NormKernel kern = bf16 ? pick<bf16_t, true>(A.C, tpr)
                                     : pick<float, true>(A.C, tpr);
        if (!kern) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kern, dim3(unsigned(blocks)),
                           dim3(unsigned(threads)), 0, stream, B);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !params) return e;
    hipLaunchKernelGGL(norm_sum_kernel, dim3(unsigned((2 * A.C + 63) / 64)),
                       dim3(1024), 0, stream, A, int(blocks));
    return hipGetLastError();
}

}  // namespace rwkv7m
