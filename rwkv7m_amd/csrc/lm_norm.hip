// Layer norm over the last axis, forward and backward
// (include/rwkv7m_lm_head.h has the formulas).

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

__device__ __forceinline__ float param(const void* p, bool bf16, int64_t i,
                                       float absent) {
    if (!p) return absent;
    return bf16 ? bf16_to_f32(static_cast<const bf16_t*>(p)[i])
                : static_cast<const float*>(p)[i];
}

template <typename E>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(LmNormArgs A) {
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
            sq += d * d;
        }
        const float rstd =
            1.f / sqrtf(block_sum<kWaves>(sq, s) * n + A.eps);
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads)
            store_f(y + i, (load_f(x + i) - mean) * rstd *
                                   param(A.weight, A.param_bf16, i, 1.f) +
                               param(A.bias, A.param_bf16, i, 0.f));
        if (threadIdx.x == 0 && A.mean) {
            A.mean[row] = mean;
            A.rstd[row] = rstd;
        }
    }
}

template <typename E>
__global__ __launch_bounds__(kThreads) void norm_dx_kernel(LmNormArgs A) {
    __shared__ float s[kWaves];
    const float n = 1.f / float(A.C);
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        const E* dy = static_cast<const E*>(A.dy) + row * A.C;
        E* dx = static_cast<E*>(A.dx) + row * A.C;
        const float mean = A.mean[row], rstd = A.rstd[row];
        float sg = 0.f, sgx = 0.f;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads) {
            const float g =
                load_f(dy + i) * param(A.weight, A.param_bf16, i, 1.f);
            sg += g;
            sgx += g * ((load_f(x + i) - mean) * rstd);
        }
        sg = block_sum<kWaves>(sg, s) * n;
        sgx = block_sum<kWaves>(sgx, s) * n;
        for (int64_t i = threadIdx.x; i < A.C; i += kThreads) {
            const float g =
                load_f(dy + i) * param(A.weight, A.param_bf16, i, 1.f);
            const float xh = (load_f(x + i) - mean) * rstd;
            store_f(dx + i, rstd * (g - sg - xh * sgx));
        }
    }
}

// Partial parameter gradients: block (column tile, g) sums the rows
// g, g + groups, ... into part[g][0 / 1][C] (weight, bias).
template <typename E>
__global__ __launch_bounds__(kThreads) void norm_part_kernel(LmNormArgs A,
                                                             int groups) {
    const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= A.C) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.y; row < A.rows; row += groups) {
        const float x = load_f(static_cast<const E*>(A.x) +
                               row_offset(A.xr, row) + c);
        const float dy = load_f(static_cast<const E*>(A.dy) + row * A.C + c);
        dw += dy * ((x - A.mean[row]) * A.rstd[row]);
        db += dy;
    }
    float* p = A.workspace + int64_t(blockIdx.y) * 2 * A.C;
    p[c] = dw;
    p[A.C + c] = db;
}

__global__ __launch_bounds__(kThreads) void norm_sum_kernel(LmNormArgs A,
                                                            int groups) {
    const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= A.C) return;
    float dw = 0.f, db = 0.f;
    for (int g = 0; g < groups; ++g) {
        dw += A.workspace[int64_t(g) * 2 * A.C + c];
        db += A.workspace[int64_t(g) * 2 * A.C + A.C + c];
    }
    for (int k = 0; k < 2; ++k) {
        void* out = k ? A.dbias : A.dweight;
        if (!out) continue;
        if (A.param_bf16)
            store_f(static_cast<bf16_t*>(out) + c, k ? db : dw);
        else
            store_f(static_cast<float*>(out) + c, k ? db : dw);
    }
}

int row_groups(int64_t rows) {
    return int(rows < 1 ? 0 : rows < 256 ? rows : 256);
}

unsigned row_grid(int64_t rows) {
    return unsigned(rows < (1 << 20) ? rows : 1 << 20);
}

}  // namespace

int64_t lm_norm_workspace_floats(int64_t rows, int64_t C) {
    return 2 * C * row_groups(rows);
}

hipError_t launch_lm_norm(bool bf16, const LmNormArgs& A, hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(bf16 ? norm_fwd_kernel<bf16_t> : norm_fwd_kernel<float>,
                       dim3(row_grid(A.rows)), dim3(kThreads), 0, stream, A);
    return hipGetLastError();
}

hipError_t launch_lm_norm_backward(bool bf16, const LmNormArgs& A,
                                   hipStream_t stream) {
    if (A.rows > 0 && A.dx)
        hipLaunchKernelGGL(
            bf16 ? norm_dx_kernel<bf16_t> : norm_dx_kernel<float>,
            dim3(row_grid(A.rows)), dim3(kThreads), 0, stream, A);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!A.dweight && !A.dbias)) return e;
    const int groups = row_groups(A.rows);
    const unsigned tiles = unsigned((A.C + kThreads - 1) / kThreads);
    if (groups > 0)
        hipLaunchKernelGGL(
            bf16 ? norm_part_kernel<bf16_t> : norm_part_kernel<float>,
            dim3(tiles, unsigned(groups)), dim3(kThreads), 0, stream, A,
            groups);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(norm_sum_kernel, dim3(tiles), dim3(kThreads), 0, stream,
                       A, groups);
    return hipGetLastError();
}

}  // namespace rwkv7m
