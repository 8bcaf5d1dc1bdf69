// Distillation loss from a teacher's top logits and its gradient
// (include/rwkv7m_lm_head.h has the formulas).
//
// Bound by memory: a row of logits is read once and its gradient written
// once, about 16 operations an element.  One workgroup holds the row in its
// registers as it came (65536 bf16 logits: 1024 threads of 32 registers, two
// to a CU) and walks them three times: for the largest, for the sum of the
// exponentials, and for the gradient weight T p, with each exponential
// computed again rather than kept (the row would take twice the registers).
// [4088, 65536] bf16 takes 209 us (5.1 TB/s) by itself; between backward
// passes, under a profiler, 210 to 228.  The teacher's alternatives are one to
// a thread of the first 4 waves and stay in LDS; after the gradient's row is
// out, each writes its entry again with its q taken off, the first of equal
// ids with all their q, summed in the order of the alternatives.

#include "lm_rows.h"

namespace rwkv7m {
namespace {

// Threads that hold an alternative: the first 4 waves, or the only one.
template <int NT>
constexpr int kTeacher = NT < 256 ? NT : 256;

template <int NT>
struct DistillShared {
    static constexpr int KT = kTeacher<NT>, KW = KT / 64;
    float largest[NT / 64], sums[NT / 64], teacher[3][KW], bad[KW];
    // each alternative's id (-1: none, -2: past the vocabulary), teacher's
    // logit, then q, and student's logit
    int ids[KT];
    float q[KT], student[KT];
};

template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, (kRowWaves<NT, NV>)) void distill_kernel(
    LmDistillArgs A) {
    constexpr int W = NT / 64, KW = kTeacher<NT> / 64, n = Vec<E>::n;
    __shared__ DistillShared<NT> S;
    const int64_t r = grid_row();
    if (r >= A.rows) return;
    float scale = 1.f;
    if (A.scale) {
        scale = *A.scale;
        if (A.holds_unit && scale == 1.f) return;
    }
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int K = int(A.K), k = threadIdx.x, V = int(A.V);
    const float inf = __builtin_inff();
    const float w = A.weight ? A.weight[r] : A.mean_weight;
    E* dx = A.dlogits ? static_cast<E*>(A.dlogits) + r * A.V : nullptr;
    const auto clear = [&] {
        if (threadIdx.x == 0 && A.row_losses) A.row_losses[r] = 0.f;
        if (!dx) return;
        Vec<E> zero;
        zero.raw = 0;
        for (int i = threadIdx.x; i < V / n; i += NT) zero.store(dx + i * n);
        if (threadIdx.x < V % n) store_f(dx + V / n * n + threadIdx.x, 0.f);
    };
    if (w == 0.f) {
        clear();
        return;
    }
    Row<E, NT, NV> row(
        static_cast<const E*>(A.x) + uniform(row_offset(A.xr, r)), V);
    if (wave < KW) {
        int id = -1;
        float t = -inf, at_id = 0.f;
        if (k < K) {
            const int64_t i = r * K + k, full = A.ids[i];
            if (full >= 0) {
                t = A.teacher_bf16
                        ? bf16_to_f32(static_cast<const bf16_t*>(A.teacher)[i])
                        : static_cast<const float*>(A.teacher)[i];
                id = full < V ? int(full) : -2;
                if (full < V) at_id = load_f(row.x + id);
            }
        }
        S.ids[k] = id;
        S.q[k] = t;
        S.student[k] = at_id;
        const float tl = lanes_larger<64>(t);
        if (lane == 0) S.teacher[0][wave] = tl;
    }
    const float wl = lanes_larger<64>(row.largest());
    if (lane == 0) S.largest[wave] = wl;
    __syncthreads();
    const float teacher_largest = waves_larger<KW>(S.teacher[0]);
    if (teacher_largest == -inf) {
        clear();
        return;
    }
    const RowSoftmax soft(waves_larger<W>(S.largest), A.c);
    const RowSoftmax teacher(teacher_largest, A.c);
    if (wave < KW) {
        const float te =
            __builtin_amdgcn_exp2f(teacher.difference(S.q[k]));
        const float es = lanes_sum<64>(S.ids[k] == -1 ? 0.f : te);
        // an id past the vocabulary: NaN for the row
        const float bad = __any(S.ids[k] == -2) ? __builtin_nanf("") : 0.f;
        if (lane == 0) {
            S.teacher[1][wave] = es;
            S.bad[wave] = bad;
        }
    }
    float s0 = 0.f;
    soft.with_t(row, [&](auto t, auto each) {
        s0 = __builtin_amdgcn_exp2f(t(row.one));
        each([&](const Vec<E>& a, int) {
#pragma unroll
            for (int j = 0; j < n; ++j)
                s0 += __builtin_amdgcn_exp2f(t(a.get(j)));
        });
    });
    s0 = lanes_sum<64>(s0);
    if (lane == 0) S.sums[wave] = s0;
    __syncthreads();
    s0 = waves_sum<W>(S.sums);
    const float bad = waves_sum<KW>(S.bad);
    if (wave < KW) {
        const float ts = waves_sum<KW>(S.teacher[1]), t = S.q[k];
        const float te = __builtin_amdgcn_exp2f(teacher.difference(t));
        const float q = S.ids[k] == -1 ? 0.f : te / ts;
        float share = 0.f;
        if (q != 0.f) {
            // half of T (log q - log p), which fits where neither log does; a
            // row of nothing but -inf has p = 0
            const float ls = s0 == 0.f ? inf : soft.log2_sum(s0);
            share = q * (teacher.half_difference(t) -
                         soft.half_difference(S.student[k]) +
                         0.5f * kLn2 * A.temperature * (ls - __log2f(ts)));
        }
        share = lanes_sum<64>(share);
        if (lane == 0) S.teacher[2][wave] = share;
        S.q[k] = q;
    }
    const float wt = w * A.temperature * scale;
    const float wp = uniform((s0 == 0.f ? 0.f : wt / s0) + bad);
    if (dx)
        soft.with_t(row, [&](auto t, auto each) {
            const auto grad = [&](float x) {
                return wp * __builtin_amdgcn_exp2f(t(x));
            };
            each([&](const Vec<E>& a, int i) {
                Vec<E> g;
#pragma unroll
                for (int j = 0; j < n; j += 2)
                    g.set2(j, grad(a.get(j)), grad(a.get(j + 1)));
                if (i < row.cut.whole) g.store(dx + row.cut.lead + i * n);
            });
            if (row.has_one()) store_f(dx + row.one_id(), grad(row.one));
        });
    __syncthreads();
    const float half = waves_sum<KW>(S.teacher[2]) + bad;
    if (threadIdx.x == 0 && A.row_losses)
        A.row_losses[r] = half * A.temperature * 2.f;
    if (!dx || k >= K || S.ids[k] < 0) return;
    float sum = 0.f;
    bool first = true;
    for (int j = 0; j < K; ++j) {
        if (S.ids[j] != S.ids[k]) continue;
        first = first && j >= k;
        sum += S.q[j];
    }
    if (!first) return;
    soft.with_t(row, [&](auto t, auto) {
        // (p by a division: 1 where it is, so that p - q is 0)
        const float e = __builtin_amdgcn_exp2f(t(S.student[k]));
        const float p = (s0 == 0.f ? 0.f : e / s0) + bad;
        store_f(dx + S.ids[k], (p - sum) * wt);
    });
}

// loss = sum_r weight[r] row_losses[r], one workgroup, in float64: a fixed
// order, and no error beside the rows' own (5 us at 4088 rows, latency).
__global__ __launch_bounds__(1024) void distill_sum_kernel(LmDistillArgs A) {
    __shared__ double s[16];
    double x = 0.0;
    for (int64_t r = threadIdx.x; r < A.rows; r += 1024)
        x += double(A.weight ? A.weight[r] : A.mean_weight) *
             double(A.row_losses[r]);
    x = block_fold<16>(x, s, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) *A.loss = float(x);
}

}  // namespace

hipError_t launch_lm_distill(bool bf16, const LmDistillArgs& A,
                             hipStream_t stream) {
    if (A.rows > 0) {
        // (by 512 threads of 16 vectors the row does not stay within the 80
        // registers three workgroups a CU leave: 259 against 209 us)
        const bool wave = A.K <= kTeacher<64>;
        const auto go = [&](auto kern, unsigned threads) {
            hipLaunchKernelGGL(kern, row_grid(A.rows), dim3(threads), 0,
                               stream, A);
        };
        if (bf16)
            RWKV7M_LM_ROW_KERNEL(distill_kernel, bf16_t, A.V, wave, 1024, go);
        else
            RWKV7M_LM_ROW_KERNEL(distill_kernel, float, A.V, wave, 1024, go);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !A.loss) return e;
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, A);
    return hipGetLastError();
}

}  // namespace rwkv7m
