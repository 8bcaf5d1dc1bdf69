// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and their backward (include/rwkv7m_lm_head.h has the formulas).

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// The order of the alternatives as an unsigned number: that of the floats,
// -0 with +0, every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup a row.  The alternatives one at a time: the largest (key,
// lowest id) below the one before.
template <typename E>
__global__ __launch_bounds__(kThreads) void score_kernel(LmScoreArgs A) {
    __shared__ float s[kWaves];
    __shared__ uint64_t su[kWaves];
    const float c = A.c, lowest = -200.f / c, inv_t = c * kLn2;
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        float m = -__builtin_inff();
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
            m = larger(m, load_f(x + i));
        m = block_fold<kWaves>(m, s, larger);
        SoftStats st{ref_of(m), 0.f, 0.f};
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads)
            soft_add(st, load_f(x + i), c, lowest);
        st.s0 = block_sum<kWaves>(st.s0, s);
        st.s1 = block_sum<kWaves>(st.s1, s);
        const float ls = kLn2 * __log2f(st.s0);
        const auto logp = [&](float v) {
            return __builtin_fmaf(v - st.ref, inv_t, -ls);
        };
        const bool empty = m == -__builtin_inff();
        if (threadIdx.x == 0) {
            const int64_t tok = A.tokens[row];
            A.logprobs[row] = tok < 0       ? 0.f
                              : tok >= A.V  ? __builtin_nanf("")
                              : empty       ? -__builtin_inff()
                                            : logp(load_f(x + tok));
            A.entropy[row] = empty ? 0.f : ls - st.s1 / st.s0 * inv_t;
            if (A.stats) {
                A.stats[2 * row] = st.ref;
                A.stats[2 * row + 1] = empty ? __builtin_inff() : ls;
            }
        }
        uint64_t last = ~uint64_t(0);
        for (int k = 0; k < A.top_k; ++k) {
            uint64_t best = 0;
            for (int64_t i = threadIdx.x; i < A.V; i += kThreads) {
                const uint64_t key =
                    uint64_t(order_key(load_f(x + i))) << 32 |
                    uint32_t(0xffffffffu - uint32_t(i));
                if (key < last && key > best) best = key;
            }
            last = block_fold<kWaves>(
                best, su,
                [](uint64_t a, uint64_t b) { return a > b ? a : b; });
            if (threadIdx.x == 0) {
                const uint32_t id = 0xffffffffu - uint32_t(last);
                A.top_ids[row * A.top_k + k] = id;
                A.top_logprobs[row * A.top_k + k] =
                    empty ? -__builtin_inff() : logp(load_f(x + id));
            }
        }
    }
}

template <typename E>
__global__ __launch_bounds__(kThreads) void score_bwd_kernel(LmScoreArgs A) {
    const float inv_t = A.c * kLn2;
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, row);
        E* dx = static_cast<E*>(A.dlogits) + row * A.V;
        const int64_t tok = A.tokens[row];
        const float dl =
            A.d_logprobs && tok >= 0 ? A.d_logprobs[row] * inv_t : 0.f;
        const float de = A.d_entropy ? A.d_entropy[row] * inv_t : 0.f;
        const float ref = A.stats[2 * row], ls = A.stats[2 * row + 1];
        const float h = A.entropy[row];
        const bool any = dl != 0.f || de != 0.f;
        const float nan = tok >= A.V && dl != 0.f ? __builtin_nanf("") : 0.f;
        for (int64_t i = threadIdx.x; i < A.V; i += kThreads) {
            float d = 0.f;
            if (any) {
                // (held above -150, whose exp is 0 in fp32: -inf gives no NaN)
                const float lp = larger(
                    __builtin_fmaf(load_f(x + i) - ref, inv_t, -ls), -150.f);
                d = nan - __builtin_amdgcn_exp2f(lp * kLog2e) *
                              (dl + de * (lp + h));
                if (i == tok) d += dl;
            }
            store_f(dx + i, d);
        }
    }
}

unsigned row_grid(int64_t rows) {
    return unsigned(rows < (1 << 20) ? rows : 1 << 20);
}

}  // namespace

hipError_t launch_lm_score(bool bf16, const LmScoreArgs& A,
                           hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(bf16 ? score_kernel<bf16_t> : score_kernel<float>,
                       dim3(row_grid(A.rows)), dim3(kThreads), 0, stream, A);
    return hipGetLastError();
}

hipError_t launch_lm_score_backward(bool bf16, const LmScoreArgs& A,
                                    hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(
        bf16 ? score_bwd_kernel<bf16_t> : score_bwd_kernel<float>,
        dim3(row_grid(A.rows)), dim3(kThreads), 0, stream, A);
    return hipGetLastError();
}

}  // namespace rwkv7m
