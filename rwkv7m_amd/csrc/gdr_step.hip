// The gated delta rule a token at a time on a pool of states (decode; T
// tokens of a drafted block), in fp32:
//
//   u = beta (v - a S k),  S' = a S + u k^T,  o = scale S' q,  a = e^g
//
// Bound by the state's bytes: read once, written once (or not, where the block
// is only read ahead), whatever T.  Both products are taken with the old
// state, S' q = a S q + u (k.q), so that each token walks over the registers
// once and waits for one reduction.  A workgroup holds 64 rows; a row lies
// across 16 lanes, which one DPP row sums, and a group of them has four
// adjoining rows, whose v and o are one access.
//
// 192 tokens of 32 heads of 128 x 128: 805 MB of states in 154 us, 5.2 TB/s,
// above a copy's rate (4.9).  One token of 12 heads of 64 x 64: 4.4 us, a
// launch's latency.  48 blocks of 0 to 6 tokens, 32 heads of 64 x 64, read
// ahead: 14 us for 24.5 MB, a reduction's wait a token (without the next token's
// loads ahead 17).
#include "wkv7_common.h"
#include "wkv7_launch.h"

namespace rwkv7m {
namespace {

constexpr int NT = 256, ROWS = 64;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t load4(const float* p) {
    return *reinterpret_cast<const f32x4_t*>(p);
}
__device__ __forceinline__ void store4(float* p, const f32x4_t& x) {
    *reinterpret_cast<f32x4_t*>(p) = x;
}
__device__ __forceinline__ void store4(bf16_t* p, const f32x4_t& x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(
        uint32_t(f32_to_bf16(x[0])) | uint32_t(f32_to_bf16(x[1])) << 16,
        uint32_t(f32_to_bf16(x[2])) | uint32_t(f32_to_bf16(x[3])) << 16);
}

template <typename E>
__device__ __forceinline__ const E* at(const GdrTensor& t, int64_t b, int64_t h,
                                       int64_t token) {
    return static_cast<const E*>(t.p) + b * t.sb + h * t.sh + token * t.st;
}
__device__ __forceinline__ float gate(const GdrTensor& t, bool bf16, int64_t b,
                                      int64_t h, int64_t token) {
    return bf16 ? load_f(at<bf16_t>(t, b, h, token))
                : load_f(at<float>(t, b, h, token));
}
__device__ __forceinline__ float dot(const f32x4_t& a, const f32x4_t& b) {
    return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}

// Four elements as they lie in memory.
template <typename E>
struct Raw;
template <>
struct Raw<float> {
    f32x4_t x;
    __device__ __forceinline__ void load(const float* p) { x = load4(p); }
    __device__ __forceinline__ f32x4_t get() const { return x; }
};
template <>
struct Raw<bf16_t> {
    uint2 u;
    __device__ __forceinline__ void load(const bf16_t* p) {
        u = *reinterpret_cast<const uint2*>(p);
    }
    __device__ __forceinline__ f32x4_t get() const {
        return f32x4_t{__uint_as_float(u.x << 16),
                       __uint_as_float(u.x & 0xffff0000u),
                       __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u)};
    }
};

// What the lane needs of a token, loaded without conditions (its places past
// Dk, and rows past Dv, from the last ones there are).
template <typename E, int KQ>
struct Token {
    Raw<E> k[KQ], q[KQ], v;
    float g, beta;
    __device__ __forceinline__ void load(const GdrStepArgs& A, int64_t b,
                                         int64_t h, int64_t hk, int64_t t,
                                         int row, int r) {
        const E* kp = at<E>(A.k, b, hk, t);
        const E* qp = at<E>(A.q, b, hk, t);
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int col = 64 * j + 4 * r, c = col < A.Dk ? col : A.Dk - 4;
            k[j].load(kp + c);
            q[j].load(qp + c);
        }
        v.load(at<E>(A.v, b, h, t) + (row < A.Dv ? row : A.Dv - 4));
        g = gate(A.g, A.g_bf16, b, h, t);
        beta = gate(A.beta, A.beta_bf16, b, h, t);
    }
};

// KQ: 16-lane groups of 4 places a row (Dk up to 64 KQ).
template <typename E, int KQ>
__global__ void __launch_bounds__(NT)
gdr_step_kernel(const GdrStepArgs A, uint32_t parts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15;
    // (32 bits: a 64-bit division is 130 instructions)
    const uint32_t bh = blockIdx.x / parts, Hv = uint32_t(A.Hv);
    const int64_t b = bh / Hv, h = bh % Hv,
                  hk = uint32_t(h) / (Hv / uint32_t(A.Hk));
    const int row =
        int(blockIdx.x % parts) * ROWS + wave * 16 + (lane >> 4) * 4;
    const bool on = row < A.Dv;  // (Dv is a multiple of 8)

    // the first token on its way before the slot and the state are known, and
    // each next one while the one before is worked on
    Token<E, KQ> now, next;
    now.load(A, b, h, hk, 0, row, r);
    const int64_t slot = A.slots ? A.slots[b] : b;
    int64_t len = A.lengths ? A.lengths[b] : A.T;
    len = len < 0 ? 0 : len > A.T ? A.T : len;
    if (slot < 0) len = 0;
    // A slot outside the pool, or one that an earlier row updates: NaN in
    // place of the outputs, and the state is left to the other.
    bool bad = slot >= A.pool;
    const bool use = len > 0 && !bad && on;

    float* state = A.state + ((slot * A.Hv + h) * A.Dv + row) * A.Dk;
    f32x4_t S[4][KQ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int col = 64 * j + 4 * r;
            S[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (use && col < A.Dk) S[i][j] = load4(state + i * A.Dk + col);
        }
    if (A.update && A.slots && slot >= 0 && len > 0) {
        bool twice = false;
        for (int64_t j = lane; j < b; j += 64)
            twice |= A.slots[j] == slot && (!A.lengths || A.lengths[j] > 0);
        bad |= __builtin_amdgcn_ballot_w64(twice) != 0;
    }
    E* o = static_cast<E*>(A.o) + (b * A.T * A.Hv + h) * A.Dv + row;
    for (int64_t t = 0; t < len; ++t) {
        next.load(A, b, h, hk, t + 1 < len ? t + 1 : t, row, r);
        f32x4_t k[KQ], q[KQ];
        float kq = 0.f;
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const bool in = 64 * j + 4 * r < A.Dk;
            k[j] = now.k[j].get();
            q[j] = now.q[j].get();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                k[j][e] = in ? k[j][e] : 0.f;
                q[j][e] = in ? q[j][e] : 0.f;
            }
            kq += dot(k[j], q[j]);
        }
        const f32x4_t v = now.v.get();
        const float a = expf(now.g), beta = now.beta;
        kq = group_sum<16>(kq);
        f32x4_t out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float sk = 0.f, sq = 0.f;
#pragma unroll
            for (int j = 0; j < KQ; ++j) {
                sk += dot(S[i][j], k[j]);
                sq += dot(S[i][j], q[j]);
            }
            sk = group_sum<16>(sk);
            sq = group_sum<16>(sq);
            const float u = beta * (v[i] - a * sk);
#pragma unroll
            for (int j = 0; j < KQ; ++j) S[i][j] = a * S[i][j] + u * k[j];
            out[i] = A.scale * (a * sq + u * kq);
        }
        if (bad) out = f32x4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
        if (r == 0 && on) store4(o + t * A.Hv * A.Dv, out);
        now = next;
    }
    if (r == 0 && on)
        for (int64_t t = len; t < A.T; ++t)
            store4(o + t * A.Hv * A.Dv, f32x4_t{0.f, 0.f, 0.f, 0.f});
    if (!A.update || !use || bad) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int col = 64 * j + 4 * r;
            if (col < A.Dk) store4(state + i * A.Dk + col, S[i][j]);
        }
}

}  // namespace

hipError_t launch_gdr_step(bool bf16, const GdrStepArgs& A,
                           hipStream_t stream) {
    const uint32_t parts = uint32_t(A.Dv + ROWS - 1) / ROWS;
    const dim3 grid(unsigned(A.B * A.Hv * parts));
#define RWKV7M_GDR(E, KQ)                                                   \
    hipLaunchKernelGGL((gdr_step_kernel<E, KQ>), grid, dim3(NT), 0, stream, \
                       A, parts)
    if (bf16 && A.Dk <= 64)
        RWKV7M_GDR(bf16_t, 1);
    else if (bf16)
        RWKV7M_GDR(bf16_t, 2);
    else if (A.Dk <= 64)
        RWKV7M_GDR(float, 1);
    else
        RWKV7M_GDR(float, 2);
#undef RWKV7M_GDR
    return hipGetLastError();
}

}  // namespace rwkv7m
