// Distillation loss from a teacher's top logits and its gradient
// (include/rwkv7m_lm_head.h has the formulas).
//
// Bound by memory: a row of logits is read once and its gradient written
// once.  One workgroup holds the row in its registers as it came (65536 bf16
// logits: 1024 threads of 32 registers) and walks them three times: for the
// largest, for the sum of the exponentials, and for the gradient weight T p,
// with each exponential computed again rather than kept (the row would take
// twice the registers).  The teacher's alternatives are one to a thread of the
// first 4 waves; after the gradient's row is out, each writes its entry again
// with its q taken off, the first of equal ids with all their q, summed in
// the order of the alternatives.

#include "lm_rows.h"

namespace rwkv7m {
namespace {

constexpr int kMaxK = 256;

template <int W>
struct DistillShared {
    float largest[W], sums[W], teacher[3][4], bad[4];
    int ids[kMaxK];
    float q[kMaxK];
};

template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, kRowWaves<NV>) void distill_kernel(
    LmDistillArgs A) {
    constexpr int W = NT / 64, n = Vec<E>::n;
    static_assert(kMaxK == 256 && NT >= kMaxK, "an alternative a thread");
    __shared__ DistillShared<W> S;
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
    Row<E, NT, NV> row;
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
    row.load(static_cast<const E*>(A.x) + uniform(row_offset(A.xr, r)), V);
    int64_t id = -1;
    float t = -inf, at_id = 0.f;  // the teacher's logit, the student's
    if (k < K) {
        id = A.ids[r * K + k];
        const int64_t i = r * K + k;
        if (id >= 0)
            t = A.teacher_bf16
                    ? bf16_to_f32(static_cast<const bf16_t*>(A.teacher)[i])
                    : static_cast<const float*>(A.teacher)[i];
        if (id >= 0 && id < V) at_id = load_f(row.x + id);
    }
    const float mine = row.largest();
    const float wl = wave_larger(mine);
    if (lane == 0) S.largest[wave] = wl;
    if (wave < 4) {
        const float tl = wave_larger(t);
        if (lane == 0) S.teacher[0][wave] = tl;
    }
    __syncthreads();
    const float largest = waves_fold<W>(S.largest, larger);
    const float teacher_largest = waves_fold<4>(S.teacher[0], larger);
    if (teacher_largest == -inf) {
        clear();
        return;
    }
    const RowSoftmax soft(largest, A.c), teacher(teacher_largest, A.c);
    float s0 = 0.f;
    row.each([&](const Vec<E>& a, int, int) {
#pragma unroll
        for (int j = 0; j < n; ++j) s0 += soft.e(a.get(j));
    });
    s0 = lanes_sum<64>(s0);
    if (lane == 0) S.sums[wave] = s0;
    const float te = id >= 0 ? teacher.e(t) : 0.f;
    if (wave < 4) {
        const float es = lanes_sum<64>(te);
        // an id past the vocabulary: NaN for the row
        const float bad = __any(id >= V) ? __builtin_nanf("") : 0.f;
        if (lane == 0) {
            S.teacher[1][wave] = es;
            S.bad[wave] = bad;
        }
    }
    __syncthreads();
    s0 = waves_sum<W>(S.sums);
    const float ts = waves_sum<4>(S.teacher[1]);
    const float bad = waves_sum<4>(S.bad);
    const float q = te / ts;
    if (wave < 4) {
        float share = 0.f;
        if (q != 0.f) {
            // log2 q - log2 p
            const float lp = largest == -inf
                                 ? -inf
                                 : (at_id - soft.ref) * A.c -
                                       soft.log2_sum(s0);
            share = q * ((t - teacher.ref) * A.c - teacher.log2_sum(ts) - lp);
        }
        share = lanes_sum<64>(share);
        if (lane == 0) S.teacher[2][wave] = share;
        S.ids[k] = id >= 0 && id < V ? int(id) : -1;
        S.q[k] = q;
    }
    const float wt = w * A.temperature * scale;
    const float wp = (s0 == 0.f ? 0.f : wt / s0) + bad;
    if (dx)
        row.each([&](const Vec<E>& a, int id, int from) {
            Vec<E> g;
#pragma unroll
            for (int j = 0; j < n; j += 2)
                g.set2(j, wp * soft.e(a.get(j)), wp * soft.e(a.get(j + 1)));
            if (from == 0)
                g.store(dx + id);
            else
                for (int j = from; j < n; ++j) store_f(dx + id + j, g.get(j));
        });
    __syncthreads();
    const float kl = waves_sum<4>(S.teacher[2]) + bad;
    if (threadIdx.x == 0 && A.row_losses)
        A.row_losses[r] = kl * kLn2 * A.temperature * A.temperature;
    if (!dx || k >= K || S.ids[k] < 0) return;
    float sum = 0.f;
    bool first = true;
    for (int j = 0; j < K; ++j) {
        if (S.ids[j] != S.ids[k]) continue;
        first = first && j >= k;
        sum += S.q[j];
    }
    if (first)
        store_f(dx + S.ids[k], __builtin_fmaf(soft.e(at_id), wp, -sum * wt));
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

}  // namespace

hipError_t launch_lm_distill(bool bf16, const LmDistillArgs& A,
                             hipStream_t stream) {
    if (A.rows > 0) {
        const auto go = [&](auto kern, unsigned threads) {
            hipLaunchKernelGGL(kern, row_grid(A.rows), dim3(threads), 0,
                               stream, A);
        };
        if (bf16)
            RWKV7M_LM_ROW_KERNEL(distill_kernel, bf16_t, A.V, go);
        else
            RWKV7M_LM_ROW_KERNEL(distill_kernel, float, A.V, go);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !A.loss) return e;
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, A);
    return hipGetLastError();
}

}  // namespace rwkv7m
