// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and their backward (include/rwkv7m_lm_head.h has the formulas).
//
// Bound by memory: a row is read once, about 10 operations an element.  One
// workgroup holds a row in its registers as it came (65536 bf16 logits: 512
// threads of 64 registers), so that the largest logit, the sums and the
// alternatives are three walks over registers and not over memory.  [4088,
// 65536] bf16 is read in 90 to 93 us (5.9 TB/s), with 10 alternatives in 98
// (5.5): what those add is mostly latency, a search of the bound, two passes
// over LDS and three barriers in which the row's registers wait.  Rows of more
// than 65536 bf16 leave room for one workgroup a CU, whose loads nothing
// overlaps: 3.8 TB/s at 131072.
//
// The alternatives.  Each thread's largest logit is known from the first
// walk; the k-th largest over g = 256 groups of threads (64 threads in a wave
// of its own) is a lower bound T of the row's k-th largest logit, and for
// logits in no particular order not many more than k of them lie at or above
// it (-g log(1 - k / g) on average, as long as the bound's 16 high bits tell
// the largest apart).
// The vectors that hold one go to LDS, their elements at or above T to a list
// there, and each of those finds its rank by counting the ones before it.
// Where they are more than LDS has room for (many equal logits, large ones at
// the same few threads, a mask that leaves fewer than k groups anything, fp32
// logits whose offset is some hundred times their spread and that agree in
// their high bits), or NaN are among them, the list's bound is found exactly,
// by counting and bisection over the order of the values and then of the ids:
// 0.40 ms for [4088, 65536] of nothing but equal logits, 1.0 ms for [1022,
// 65536] fp32 around 1000 with a spread of 2 (61 us around 0).

#include "lm_rows.h"

namespace rwkv7m {
namespace {

// Room in LDS for the vectors and the elements at or above the bound.
template <int NT>
constexpr int kVectors = NT < 256 ? 128 : 256;
template <int NT>
constexpr int kList = NT < 256 ? 256 : 512;

// The order of the alternatives as an unsigned number: that of the floats,
// -0 with +0, every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffff0000u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <int NT>
struct ScoreShared {
    static constexpr int W = NT / 64;
    float largest[W], sums[2][W], at_token;
    int64_t token;
    uint32_t groups[NT > 64 ? 256 : 1], bound;
    int vectors, listed, counts[2][W];
    // vectors that hold an element at or above the bound, with the id of
    // their first, and those elements, key above the id's complement
    uint32_t raw[kVectors<NT>][4];
    int first[kVectors<NT>];
    uint64_t list[kList<NT>];
};

// The largest 32-bit number with 16 low zeros that at least k of the 64 G keys
// reach (G in each lane of the wave), or a smaller one that exactly k reach:
// at most 16 steps of a bisection with the wave's votes.
template <int G>
__device__ __forceinline__ uint32_t group_bound(const uint32_t (&key)[G],
                                                int k) {
    uint32_t bound = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | (1u << bit);
        int count = 0;
#pragma unroll
        for (int i = 0; i < G; ++i) count += __popcll(__ballot(key[i] >= t));
        if (count >= k) bound = t;
        if (count == k) break;
    }
    return bound;
}

// f(key, id) over the thread's share of the row's first `ids` elements, from
// memory.
template <int NT, typename E, typename F>
__device__ __forceinline__ void walk_memory(const E* x, int ids, F f) {
    constexpr int n = Vec<E>::n;
    const Cut<E> cut(x, ids);
#pragma unroll 2
    for (int k = threadIdx.x; k < cut.whole; k += NT) {
        Vec<E> a;
        a.load(x + cut.lead + k * n);
#pragma unroll
        for (int j = 0; j < n; ++j)
            f(order_key(a.get(j)), cut.lead + k * n + j);
    }
    const int t = threadIdx.x, id = t < cut.lead ? t : ids - cut.rest -
                                                           cut.lead + t;
    if (t < cut.lead + cut.rest) f(order_key(load_f(x + id)), id);
}

// How many of the row's first `ids` elements have yes(key), over the
// workgroup; the two buffers of `counts` take turns.
template <int NT, typename E, typename F>
__device__ __forceinline__ int count_row(const E* x, int ids,
                                         ScoreShared<NT>& S, int& turn, F yes) {
    int count = 0;
    walk_memory<NT>(x, ids, [&](uint32_t k, int) { count += yes(k); });
    count = lanes_sum<64>(count);
    if (threadIdx.x % 64 == 0) S.counts[turn][threadIdx.x / 64] = count;
    __syncthreads();
    count = 0;
    for (int w = 0; w < NT / 64; ++w) count += S.counts[turn][w];
    turn ^= 1;
    return count;
}

// Fills the list with the row's first K elements of the order.  At least K
// have keys from `bound` on; `largest` is the row's largest key.  Most often
// the elements of the bound's own value are too many (equal logits, masks of
// -inf with fewer than K others): then the first count shows it and no
// bisection is needed.
template <int NT, typename E, typename P>
__device__ void list_exactly(const E* x, int V, int K, uint32_t bound,
                             uint32_t largest, ScoreShared<NT>& S, P put) {
    // the largest key that K elements reach, from lo on
    int turn = 0;
    const auto above = [&](uint32_t key) {
        return count_row<NT>(x, V, S, turn, [&](uint32_t k) { return k > key; });
    };
    uint32_t lo = bound, hi = bound | 0xffffu;
    if (above(hi) >= K) {
        lo = hi + 1;
        hi = largest;
    } else {
        if (hi > largest) hi = largest;
        // a bf16 value's key is the only one with its 16 high bits, -inf's is
        // the lowest
        if (sizeof(E) == 2 || hi <= 0x007fffffu)
            lo = hi = hi & 0x80000000u && sizeof(E) == 2 ? hi & 0xffff0000u
                                                         : hi;
    }
    while (lo < hi) {
        const uint32_t mid = hi - (hi - lo) / 2;
        if (above(mid - 1) >= K)
            lo = mid;
        else
            hi = mid - 1;
    }
    // the lowest id bound under which the elements of that key make K with
    // those above it: doubled from 64 until it is one, then bisected
    const int more = K - above(lo);
    const auto enough = [&](int ids) {
        return count_row<NT>(x, ids, S, turn,
                             [&](uint32_t k) { return k == lo; }) >= more;
    };
    int ilo = 0, ihi = 64;
    while (ihi < V && !enough(ihi)) {
        ilo = ihi;
        ihi *= 2;
    }
    if (ihi > V) ihi = V;
    while (ihi - ilo > 1) {
        const int mid = ilo + (ihi - ilo) / 2;
        if (enough(mid))
            ihi = mid;
        else
            ilo = mid;
    }
    if (threadIdx.x == 0) S.listed = 0;
    __syncthreads();
    walk_memory<NT>(x, V, [&](uint32_t k, int id) {
        if (k > lo || (k == lo && id < ihi)) put(k, id);
    });
    __syncthreads();
}

template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, (kRowWaves<NT, NV>)) void score_kernel(
    LmScoreArgs A) {
    constexpr int W = NT / 64, n = Vec<E>::n;
    __shared__ ScoreShared<NT> S;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int K = A.top_k, V = int(A.V);
    const float inv_t = A.c * kLn2, inf = __builtin_inff();
    const int64_t r = grid_row();
    if (r >= A.rows) return;
    Row<E, NT, NV> row(
        static_cast<const E*>(A.x) + uniform(row_offset(A.xr, r)), V);
    const float mine = row.largest();
    const float wl = lanes_larger<64>(mine);
    if (lane == 0) S.largest[wave] = wl;
    if (threadIdx.x == 0) S.vectors = S.listed = 0;
    if constexpr (NT > 64) {
        if (K > 1) {
            // the largest of one of 256 groups of threads
            float g = mine;
            if constexpr (NT > 256) g = lanes_larger<NT / 256>(g);
            if (threadIdx.x % (NT / 256) == 0)
                S.groups[threadIdx.x / (NT / 256)] = order_key(g);
        }
    }
    __syncthreads();
    const float largest = waves_larger<W>(S.largest);
    if (K && wave == 0) {
        uint32_t b = order_key(largest);
        if (K > 1) {
            constexpr int G = NT > 64 ? 4 : 1;
            uint32_t key[G] = {order_key(mine)};
            if constexpr (NT > 64)
#pragma unroll
                for (int i = 0; i < G; ++i) key[i] = S.groups[64 * i + lane];
            b = group_bound(key, K);
        }
        if (lane == 0) S.bound = b;
    }
    if (threadIdx.x == NT - 1) {
        const int64_t tok = A.tokens[r];
        S.token = tok;
        if (tok >= 0 && tok < V) S.at_token = load_f(row.x + tok);
    }
    const RowSoftmax soft(largest, A.c);
    float s0 = 0.f, s1 = 0.f;
    soft.with_t(row, [&](auto exponent, auto each) {
        const auto add = [&](float x) {
            // (held above -200, where e is 0 already: -inf adds 0, not
            // 0 * -inf)
            const float t = larger(exponent(x), -200.f);
            const float e = __builtin_amdgcn_exp2f(t);
            s0 += e;
            s1 = __builtin_fmaf(e, t, s1);
        };
        each([&](const Vec<E>& a, int) {
#pragma unroll
            for (int j = 0; j < n; ++j) add(a.get(j));
        });
        add(row.one);
    });
    s0 = lanes_sum<64>(s0);
    s1 = lanes_sum<64>(s1);
    if (lane == 0) {
        S.sums[0][wave] = s0;
        S.sums[1][wave] = s1;
    }
    __syncthreads();
    s0 = uniform(waves_sum<W>(S.sums[0]));
    s1 = uniform(waves_sum<W>(S.sums[1]));
    const uint32_t bound = K ? S.bound : 0u;
    // (below the key of -inf: the groups that hold anything are fewer
    // than k)
    const float least = bound < 0x00800000u ? -inf : key_value(bound);
    const auto put = [&](uint32_t key, int id) {
        const int at = atomicAdd(&S.listed, 1);
        if (at < kList<NT>)
            S.list[at] = uint64_t(key) << 32 | (0xffffffffu - uint32_t(id));
    };
    if (K) {
        if (mine >= least)
            row.each([&](const Vec<E>& a, int k) {
                float most = a.get(0);
#pragma unroll
                for (int j = 1; j < n; ++j) most = larger(most, a.get(j));
                if (!(most >= least) || k >= row.cut.whole) return;
                const int at = atomicAdd(&S.vectors, 1);
                if (at >= kVectors<NT>) return;
                S.first[at] = row.cut.lead + k * n;
#pragma unroll
                for (int w = 0; w < 4; ++w) S.raw[at][w] = a.raw[w];
            });
        if (row.has_one() && row.one >= least)
            put(order_key(row.one), row.one_id());
        __syncthreads();
    }
    // (after the last walk: the row's registers are free for the divisions)
    const bool empty = largest == -inf;
    const float log2_s = soft.log2_sum(s0), ls = kLn2 * log2_s;
    const auto logp = [&](float x) {
        return empty ? -inf
                     : __builtin_fmaf(soft.half_difference(x), 2.f * inv_t,
                                      -ls);
    };
    // (a thread of the last wave, which seldom has alternatives to rank)
    if (threadIdx.x == NT - 64) {
        A.logprobs[r] = S.token < 0    ? 0.f
                        : S.token >= V ? __builtin_nanf("")
                                       : logp(S.at_token);
        // s1 with every t moved back by the largest's, whose own term goes
        // first: exactly 0 where no other counts
        const float t = soft.largest_t(), e = __builtin_amdgcn_exp2f(t);
        const float own = __builtin_fmaf(e, t, 0.f);
        s1 = __builtin_fmaf(-t, s0 - e, s1 - own);
        A.entropy[r] = empty ? 0.f : kLn2 * (log2_s - s1 / s0);
        if (A.stats) {
            A.stats[2 * r] = soft.ref;
            A.stats[2 * r + 1] = empty ? inf : ls;
        }
    }
    if (!K) return;
    const int vectors = S.vectors;
    for (int i = threadIdx.x; i < vectors * n && vectors <= kVectors<NT>;
         i += NT) {
        const float x = load_f(reinterpret_cast<const E*>(S.raw[i / n]) + i % n);
        if (x >= least) put(order_key(x), S.first[i / n] + i % n);
    }
    __syncthreads();
    int listed = S.listed;
    if (vectors > kVectors<NT> || listed > kList<NT> || largest != largest) {
        list_exactly<NT>(row.x, V, K, bound, order_key(largest), S, put);
        listed = K;
    }
    for (int i = threadIdx.x; i < listed; i += NT) {
        const uint64_t own = S.list[i];
        int rank = 0;
        for (int j = 0; j < listed; ++j) rank += S.list[j] > own;
        if (rank < K) {
            A.top_ids[r * K + rank] = 0xffffffffu - uint32_t(own);
            A.top_logprobs[r * K + rank] =
                logp(key_value(uint32_t(own >> 32)));
        }
    }
}

// dlogits: a workgroup a tile of kTile vectors a thread of one row (a wave's
// where a row is no longer than that); the first tile's also takes the
// elements before and behind the row's vectors.  Bound by memory: 12
// operations and 4 bytes an element in bf16, 5.2 TB/s at [4088, 65536] behind
// the forward (207 us, the shortest of 20 175).
constexpr int kTile = 4;

template <typename E, int NT>
__global__ __launch_bounds__(NT) void score_bwd_kernel(LmScoreArgs A,
                                                       int tiles) {
    constexpr int n = Vec<E>::n;
    const float inv_t = A.c * kLn2;
    for (int64_t tile = blockIdx.x; tile < A.rows * tiles; tile += gridDim.x) {
        const int64_t r = tile / tiles;
        const int part = int(tile % tiles), V = int(A.V);
        const E* x = static_cast<const E*>(A.x) + row_offset(A.xr, r);
        E* dx = static_cast<E*>(A.dlogits) + r * A.V;
        const int64_t tok = A.tokens[r];
        const float dl =
            A.d_logprobs && tok >= 0 ? A.d_logprobs[r] * inv_t : 0.f;
        const float de = A.d_entropy ? A.d_entropy[r] * inv_t : 0.f;
        const float ref = A.stats[2 * r], ls = A.stats[2 * r + 1];
        const bool any = dl != 0.f || de != 0.f;
        // -p (dl + de (lp + h)) = p (lp g1 + g0), NaN for a token past V
        const float g1 = -de;
        const float g0 = tok >= V && dl != 0.f ? __builtin_nanf("")
                                               : -dl - de * A.entropy[r];
        const auto grad = [&](float v, int id) {
            // (held above -150, whose exp is 0 in fp32: -inf gives no NaN)
            const float lp =
                larger(__builtin_fmaf(v - ref, inv_t, -ls), -150.f);
            const float d = __builtin_amdgcn_exp2f(lp * kLog2e) *
                            __builtin_fmaf(lp, g1, g0);
            return id == tok ? d + dl : d;
        };
        const Cut<E> cut(x, V);
        const int first = part * NT * kTile + int(threadIdx.x);
        Vec<E> v[kTile];
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            const int k = first + i * NT;
            v[i].raw = 0;
            if (any && k < cut.whole) v[i].load(x + cut.lead + k * n);
        }
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            const int k = first + i * NT, at = cut.lead + k * n;
            if (k >= cut.whole) break;
            if (any) {
#pragma unroll
                for (int j = 0; j < n; j += 2)
                    v[i].set2(j, grad(v[i].get(j), at + j),
                              grad(v[i].get(j + 1), at + j + 1));
            }
            v[i].store(dx + at);
        }
        if (part == 0 && int(threadIdx.x) < cut.lead + cut.rest) {
            const int t = threadIdx.x;
            const int id = t < cut.lead ? t : V - cut.rest + t - cut.lead;
            store_f(dx + id, any ? grad(load_f(x + id), id) : 0.f);
        }
    }
}

}  // namespace

hipError_t launch_lm_score(bool bf16, const LmScoreArgs& A,
                           hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    // A wave's 64 groups bound more alternatives too loosely.
    const bool wave = A.top_k <= 40;
    // 512 threads hold 65536 bf16 in 80 registers, so that a CU has three rows
    // at work (1024 threads: two) and more to do while one ranks its
    // alternatives: [4088, 65536] with 20 of them 100 against 109 us.  A
    // single row takes 10.2 us so and 8.7 by 1024 threads, but a row's results
    // would then depend on how many others there are.
    const auto go = [&](auto kern, unsigned threads) {
        hipLaunchKernelGGL(kern, row_grid(A.rows), dim3(threads), 0, stream,
                           A);
    };
    if (bf16)
        RWKV7M_LM_ROW_KERNEL(score_kernel, bf16_t, A.V, wave, 512, go);
    else
        RWKV7M_LM_ROW_KERNEL(score_kernel, float, A.V, wave, 512, go);
    return hipGetLastError();
}

hipError_t launch_lm_score_backward(bool bf16, const LmScoreArgs& A,
                                    hipStream_t stream) {
    if (A.rows == 0) return hipSuccess;
    // [60000, 1000] bf16: 100 us by 256 threads a row, 48 by 64.
    const int64_t n = bf16 ? 8 : 4, threads = A.V <= 64 * kTile * n ? 64 : 256;
    const int64_t cols = threads * kTile * n;
    const int64_t tiles = (A.V + cols - 1) / cols, all = A.rows * tiles;
    const auto kern = threads == 64 ? (bf16 ? score_bwd_kernel<bf16_t, 64>
                                            : score_bwd_kernel<float, 64>)
                                    : (bf16 ? score_bwd_kernel<bf16_t, 256>
                                            : score_bwd_kernel<float, 256>);
    hipLaunchKernelGGL(kern, dim3(unsigned(all < (1 << 20) ? all : 1 << 20)),
                       dim3(unsigned(threads)), 0, stream, A, int(tiles));
    return hipGetLastError();
}

}  // namespace rwkv7m
