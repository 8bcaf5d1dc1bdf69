// Distillation loss from a teacher's top logits and its gradient
// (include/rwkv7m_lm_head.h has the formulas).

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxK = 256;

// One workgroup a row: the teacher's softmax, the row's statistics, the loss
// and the gradient p, then the teacher's ids' entries once more with their q
// taken off (the first of equal ids takes all their q).
template <typename E, typename TE>
__global__ __launch_bounds__(kThreads) void distill_kernel(LmDistillArgs A) {
    static_assert(kMaxK <= kThreads, "one thread an alternative");
    __shared__ float s[kWaves];
    __shared__ int ids[kMaxK];
    __shared__ float qs[kMaxK];
    const float c = A.c, lowest = -200.f / c, T = A.temperature;
    float scale = 1.f;
    if (A.scale) {
        scale = *A.scale;
        if (A.holds_unit && scale == 1.f) return;
    }
    const int K = int(A.K), k = threadIdx.x;
    const float inf = __builtin_inff();
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        E* dx = A.dlogits ? static_cast<E*>(A.dlogits) + row * A.V : nullptr;
        const float w = A.weight ? A.weight[row] : A.mean_weight;
        int64_t id = -1;
        float t = -inf;
        if (k < K && w != 0.f) {
            id = A.ids[row * K + k];
            if (id >= 0)
                t = load_f(static_cast<const TE*>(A.teacher) + row * K + k);
        }
        const float tm = block_fold<kWaves>(t, s, larger);
        const bool used = w != 0.f && tm != -inf;
        if (!used) {
            if (dx)
                for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
                    store_f(dx + i, 0.f);
            if (threadIdx.x == 0 && A.row_losses) A.row_losses[row] = 0.f;
            continue;
        }
        const float e =
            id >= 0 ? __builtin_amdgcn_exp2f((t - tm) * c) : 0.f;
        const float es = block_sum<kWaves>(e, s);
        const float q = e / es;
        if (k < K) {
            ids[k] = id >= 0 && id < A.V ? int(id) : -1;
            qs[k] = q;
        }
        float m = -inf;
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
            m = larger(m, load_f(x + i));
        m = block_fold<kWaves>(m, s, larger);
        SoftStats st{ref_of(m), 0.f, 0.f};
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
            soft_add(st, load_f(x + i), c, lowest);
        st.s0 = block_sum<kWaves>(st.s0, s);
        const float l2 = __log2f(st.s0);
        if (A.row_losses) {
            float kl = 0.f;
            if (id >= A.V) {
                kl = __builtin_nanf("");
            } else if (q != 0.f) {
                // log2 q - log2 p
                const float lq = (t - tm) * c - __log2f(es);
                const float lp =
                    m == -inf ? -inf : (load_f(x + id) - st.ref) * c - l2;
                kl = q * (lq - lp);
            }
            kl = block_sum<kWaves>(kl, s);
            if (threadIdx.x == 0) A.row_losses[row] = kl * kLn2 * T * T;
        }
        if (!dx) continue;
        const float bad =
            block_sum<kWaves>(id >= A.V ? __builtin_nanf("") : 0.f, s);
        const float wt = w * T * scale;
        const float wp = st.s0 > 0.f || st.s0 != st.s0 ? wt / st.s0 + bad : bad;
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
            store_f(dx + i,
                    wp * __builtin_amdgcn_exp2f(
                             c * soft_d(load_f(x + i), st.ref, lowest)));
        __syncthreads();
        if (k < K && ids[k] >= 0) {
            float sum = 0.f;
            bool first = true;
            for (int j = 0; j < K; ++j) {
                if (ids[j] != ids[k]) continue;
                first = first && j >= k;
                sum += qs[j];
            }
            if (first) {
                const float p = __builtin_amdgcn_exp2f(
                    c * soft_d(load_f(x + ids[k]), st.ref, lowest));
                store_f(dx + ids[k], __builtin_fmaf(p, wp, -sum * wt));
            }
        }
        __syncthreads();
    }
}

// loss = sum_r weight[r] row_losses[r], one workgroup, in float64.
__global__ __launch_bounds__(1024) void distill_sum_kernel(LmDistillArgs A) {
    __shared__ double s[16];
    double x = 0.0;
    for (int64_t r = threadIdx.x; r < A.rows; r += 1024)
        x += double(A.weight ? A.weight[r] : A.mean_weight) *
             double(A.row_losses[r]);
    x = block_fold<16>(x, s, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) *A.loss = float(x);
}

unsigned row_grid(int64_t rows) {
    return unsigned(rows < (1 << 20) ? rows : 1 << 20);
}

}  // namespace

hipError_t launch_lm_distill(bool bf16, bool teacher_bf16,
                             const LmDistillArgs& A, hipStream_t stream) {
    auto kern = bf16 ? (teacher_bf16 ? distill_kernel<bf16_t, bf16_t>
                                     : distill_kernel<bf16_t, float>)
                     : (teacher_bf16 ? distill_kernel<float, bf16_t>
                                     : distill_kernel<float, float>);
    if (A.rows > 0)
        hipLaunchKernelGGL(kern, dim3(row_grid(A.rows)), dim3(kThreads), 0,
                           stream, A);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !A.loss) return e;
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, A);
    return hipGetLastError();
}

}  // namespace rwkv7m
