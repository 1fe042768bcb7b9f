// fsx_logprobs.hip — the answers of a head of several classes (include/fsx_hip.h): of every
// row of logits the log probability of a given class, the entropy and the most probable
// classes, in one pass over the row.
//
//   m = max x,  S = sum e^(x-m),  T = sum (x-m) e^(x-m)
//   log p_t = (x_t - m) - log S,  H = log S - T / S
// S and T move to a larger maximum m' as S e^(m-m') and (T + (m-m') S) e^(m-m').
#include <hip/hip_runtime.h>
#include <algorithm>

#include "fsx_head.h"

namespace fsx {

constexpr float kLowest = -3.402823466e38f;   // the maximum of no values: finite, so that -inf - m is -inf
constexpr float kLog2e = 1.4426950408889634f;

// An alternative: its value as an ordered word above its class, so that the largest word is
// the most probable class and the lowest of equal ones. 0: none.
typedef unsigned long long Alt;
__device__ __forceinline__ uint32_t ord_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 and 0 are one value
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ Alt alt_of(float x, uint32_t cls) {
    return (Alt)ord_of(x) << 32 | (uint32_t)~cls;
}

struct Sums {
    float m, s, t;
    __device__ void init() { m = kLowest; s = 0.0f; t = 0.0f; }
    __device__ void raise(float m2) {   // m2 >= m
        const float d = fmaxf(m - m2, -200.0f), f = exp2f(d * kLog2e);   // e^-200 is 0 in 32 bits
        t = (t + d * s) * f;
        s *= f;
        m = m2;
    }
    __device__ void add(float x) {      // x <= m, or -inf, or NaN
        const float z = x - m, e = exp2f(z * kLog2e);
        s += e;
        t += fmaxf(z, -200.0f) * e;     // -inf: 0 * -200; NaN goes on through e
    }
    __device__ void join(float m2, float s2, float t2) {
        Sums o{m2, s2, t2};
        const float top = fmaxf(m, m2);
        raise(top);
        o.raise(top);
        s += o.s;
        t += o.t;
    }
};

// 64 alternatives in falling order, the i-th in lane i (0: an empty place).
struct TopList {
    Alt a;
    __device__ Alt at(uint32_t lane) const {
        return (Alt)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(a >> 32), lane) << 32 |
               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)a, lane);
    }
    // c (the same in every lane) goes behind the larger ones; the last place falls out
    __device__ void insert(Alt c) {
        const uint32_t lane = __lane_id();
        const uint32_t pos = __popcll(__ballot(a > c));
        const Alt up = __shfl_up(a, 1);
        a = lane < pos ? a : lane == pos ? c : up;
    }
    // the 64 largest of both lists
    __device__ void merge(Alt other) {
        const uint32_t lane = __lane_id();
        const Alt rev = __shfl(other, 63 - lane);
        a = a > rev ? a : rev;                       // a bitonic sequence with the 64 largest
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const Alt b = __shfl_xor(a, o);
            a = (lane & o) ? (a < b ? a : b) : (a > b ? a : b);
        }
    }
};

// The row's outputs, by a whole wave (all lanes hold the same sums).
template <int DT>
__device__ void finish_row(const LogprobArgs &a, uint64_t r, const Sums &q, Alt alt) {
    using T = typename Elem<DT>::T;
    const uint32_t lane = __lane_id();
    const bool bad = q.s != q.s, empty = q.s == 0.0f;
    const float ls = logf(q.s);
    if (lane == 0) {
        if (a.target) {
            const int32_t t = a.target[r];
            float lp = NAN;
            if (t == -1) lp = 0.0f;
            else if (t >= 0 && (uint32_t)t < a.v && !bad) {
                const float x = (float)static_cast<const T *>(a.x)[r * a.ld + (uint32_t)t];
                lp = empty ? -INFINITY : (x - q.m) - ls;
            }
            a.logprob[r] = lp;
        }
        if (a.entropy) {
            const float h = ls - q.t / q.s;
            a.entropy[r] = bad ? NAN : empty || h < 0.0f ? 0.0f : h;
        }
    }
    if (lane < a.top) {
        const bool none = bad || alt == 0;
        a.top_id[r * a.top + lane] = none ? -1 : (int32_t)~(uint32_t)alt;
        a.top_lp[r * a.top + lane] = bad ? NAN : none ? -INFINITY : (value_of((uint32_t)(alt >> 32)) - q.m) - ls;
    }
}

// ---------------------------------------------------------------- long rows: a block a row

constexpr int kLW = 4;    // waves a block
constexpr int kLV = 8;    // logits a lane reads at a time

// The wave's share of a row: pieces of 64 * kLV logits, `stride` pieces apart, in rising order
// of the classes: a later logit equal to the last alternative never replaces it.
template <int DT, bool TOP>
__device__ void wave_pass(const typename Elem<DT>::T *x, uint32_t v, uint32_t first, uint32_t stride, uint32_t top,
                          Sums &q, TopList &list) {
    const uint32_t lane = __lane_id();
    constexpr uint32_t kPiece = 64 * kLV;
    float tau = -INFINITY;              // the last alternative kept so far; masked logits never pass
    for (uint64_t p = (uint64_t)first * kPiece; p < v; p += (uint64_t)stride * kPiece) {
        const uint32_t c0 = (uint32_t)p + lane * kLV;
        float e[kLV];
        load_row<typename Elem<DT>::T, kLV>(x + c0, (int64_t)v - c0, -INFINITY, e);
        float top_e = e[0];
#pragma unroll
        for (int i = 1; i < kLV; ++i) top_e = fmaxf(top_e, e[i]);
        if (top_e > q.m) q.raise(top_e);
#pragma unroll
        for (int i = 0; i < kLV; ++i) q.add(e[i]);
        if (TOP && __ballot(top_e > tau)) {
#pragma unroll
            for (int i = 0; i < kLV; ++i) {
                Alt mine = e[i] > tau ? alt_of(e[i], c0 + i) : 0;
                for (;;) {
                    const uint64_t want = __ballot(mine > list.at(top - 1));
                    if (!want) break;
                    const uint32_t src = (uint32_t)__builtin_ctzll(want);
                    list.insert(TopList{mine}.at(src));
                    if (lane == src) mine = 0;
                }
            }
            const Alt last = list.at(top - 1);
            if (last) tau = value_of((uint32_t)(last >> 32));
        }
    }
    // the wave's sums, in every lane
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(q.m, o), s2 = __shfl_xor(q.s, o), t2 = __shfl_xor(q.t, o);
        q.join(m2, s2, t2);
    }
}

// The waves' results into the first wave's (the others keep theirs).
template <bool TOP>
__device__ void block_join(Sums &q, TopList &list) {
    __shared__ float s_q[kLW][3];
    __shared__ Alt s_list[kLW][64];
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) { s_q[wave][0] = q.m; s_q[wave][1] = q.s; s_q[wave][2] = q.t; }
    if (TOP) s_list[wave][lane] = list.a;
    __syncthreads();
    if (wave == 0)
        for (int w = 1; w < kLW; ++w) {
            q.join(s_q[w][0], s_q[w][1], s_q[w][2]);
            if (TOP) list.merge(s_list[w][lane]);
        }
}

template <int DT, bool TOP>
__global__ __launch_bounds__(64 * kLW) void k_logprobs(LogprobArgs a) {
    using T = typename Elem<DT>::T;
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        Sums q;
        TopList list{0};
        q.init();
        wave_pass<DT, TOP>(static_cast<const T *>(a.x) + r * a.ld, a.v, threadIdx.x >> 6, kLW, a.top, q, list);
        block_join<TOP>(q, list);
        if (threadIdx.x < 64) finish_row<DT>(a, r, q, list.a);
    }
}

template <int DT>
static void logprobs(const LogprobArgs &a, hipStream_t st) {
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(a.rows, 1u << 20);
    if (a.top) k_logprobs<DT, true><<<blocks, 64 * kLW, 0, st>>>(a);
    else k_logprobs<DT, false><<<blocks, 64 * kLW, 0, st>>>(a);
}

uint64_t logprobs_work(uint64_t rows, uint32_t v, uint32_t top) {
    (void)rows; (void)v; (void)top;
    return 0;
}

hipError_t launch_logprobs(const LogprobArgs &a, int dtype, hipStream_t st) {
    (void)hipGetLastError();
    if (a.rows == 0) return hipSuccess;
    if (dtype == FSX_DTYPE_F32) logprobs<FSX_DTYPE_F32>(a, st);
    else if (dtype == FSX_DTYPE_F16) logprobs<FSX_DTYPE_F16>(a, st);
    else logprobs<FSX_DTYPE_BF16>(a, st);
    return hipGetLastError();
}

}  // namespace fsx
