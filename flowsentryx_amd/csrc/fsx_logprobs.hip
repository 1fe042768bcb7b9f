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

// e^z, z <= 0: v_exp_f32 gives 2^y to one unit in the last place, and 0 below 2^-126.
__device__ __forceinline__ float exp_of(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

struct Sums {
    float m, s, t;
    __device__ void init() { m = kLowest; s = 0.0f; t = 0.0f; }
    __device__ void raise(float m2) {   // m2 >= m
        const float d = fmaxf(m - m2, -200.0f), f = exp_of(d);   // e^-200 is 0 in 32 bits
        t = (t + d * s) * f;
        s *= f;
        m = m2;
    }
    __device__ void add(float x) {      // x <= m, or -inf, or NaN
        const float z = x - m, e = exp_of(z);
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

// A row's log S and what it says of the row; the outputs from them.
struct RowEnd {
    float m, ls, h;
    bool bad, empty;
    __device__ explicit RowEnd(const Sums &q) {
        m = q.m;
        bad = q.s != q.s;
        empty = q.s == 0.0f;
        ls = logf(q.s);
        const float e = ls - q.t / q.s;
        h = bad ? NAN : empty || e < 0.0f ? 0.0f : e;
    }
    // log p of the class whose logit is x
    __device__ float log_p(float x) const { return bad ? NAN : empty ? -INFINITY : (x - m) - ls; }
    __device__ int32_t id(Alt a) const { return bad || a == 0 ? -1 : (int32_t)~(uint32_t)a; }
    __device__ float id_log_p(Alt a) const {
        return bad ? NAN : a == 0 ? -INFINITY : log_p(value_of((uint32_t)(a >> 32)));
    }
};

// The given class' log probability and the entropy, by one lane.
template <int DT>
__device__ __forceinline__ void put_row(const LogprobArgs &a, uint64_t r, const RowEnd &end) {
    using T = typename Elem<DT>::T;
    if (a.target) {
        const int32_t t = a.target[r];
        float lp = t == -1 ? 0.0f : NAN;
        if (t >= 0 && (uint32_t)t < a.v) lp = end.log_p((float)static_cast<const T *>(a.x)[r * a.ld + (uint32_t)t]);
        a.logprob[r] = lp;
    }
    if (a.entropy) a.entropy[r] = end.h;
}

// The row's outputs, by a whole wave (all lanes hold the same sums).
template <int DT>
__device__ void finish_row(const LogprobArgs &a, uint64_t r, const Sums &q, Alt alt) {
    const uint32_t lane = __lane_id();
    const RowEnd end(q);
    if (lane == 0) put_row<DT>(a, r, end);
    if (lane < a.top) {
        a.top_id[r * a.top + lane] = end.id(alt);
        a.top_lp[r * a.top + lane] = end.id_log_p(alt);
    }
}

// ---------------------------------------------------------------- short rows: G lanes a row

// Up to 64 N classes: a lane holds N neighbouring logits of its row, G lanes (a power of two)
// a row, so the row is read once and its maximum is known before the sums. An alternative is
// the group's largest word; its lane clears it and the next round finds the next. The lanes
// keep the results of G rounds and store them side by side.
template <int DT, int N, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_short(LogprobArgs a, uint32_t G) {
    using T = typename Elem<DT>::T;
    const uint32_t g = threadIdx.x & (G - 1), per = 256 / G, c0 = g * N;
    for (uint64_t r0 = (uint64_t)blockIdx.x * per; r0 < a.rows; r0 += (uint64_t)gridDim.x * per) {
        const uint64_t r = r0 + threadIdx.x / G;
        const bool live = r < a.rows;
        float x[N];
        load_row<T, N>(static_cast<const T *>(a.x) + (live ? r : 0) * a.ld + c0, live ? (int64_t)a.v - c0 : 0,
                       -INFINITY, x);
        Sums q;
        q.init();
#pragma unroll
        for (int i = 0; i < N; ++i) q.m = fmaxf(q.m, x[i]);
        for (uint32_t o = 1; o < G; o <<= 1) q.m = fmaxf(q.m, __shfl_xor(q.m, o));
#pragma unroll
        for (int i = 0; i < N; ++i) q.add(x[i]);
        for (uint32_t o = 1; o < G; o <<= 1) {
            q.s += __shfl_xor(q.s, o);
            q.t += __shfl_xor(q.t, o);
        }
        const RowEnd end(q);
        if (live && g == 0) put_row<DT>(a, r, end);
        if (!TOP) continue;
        uint32_t w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = x[i] > -INFINITY ? ord_of(x[i]) : 0u;
        Alt mine = 0;
        for (uint32_t k = 0; k < a.top; ++k) {
            uint32_t b = 0, at = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (w[i] > b) { b = w[i]; at = i; }
            Alt best = b ? (Alt)b << 32 | (uint32_t)~(c0 + at) : 0;
            const Alt own = best;
            for (uint32_t o = 1; o < G; o <<= 1) {
                const Alt other = __shfl_xor(best, o);
                best = other > best ? other : best;
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (own == best && at == (uint32_t)i) w[i] = 0;
            const uint32_t place = k & (G - 1);
            if (place == g) mine = best;
            if ((place == G - 1 || k == a.top - 1) && g <= place && live) {
                const uint64_t to = r * a.top + (k - place) + g;
                a.top_id[to] = end.id(mine);
                a.top_lp[to] = end.id_log_p(mine);
            }
        }
    }
}

// ---------------------------------------------------------------- long rows: a block a row

constexpr int kLW = 4;        // waves a block
constexpr int kLV = 8;        // neighbouring logits a lane reads
constexpr int kLH = 4;        // such reads in flight
constexpr uint32_t kPiece = 64 * kLV * kLH;
constexpr uint32_t kMaxParts = 64;

// The wave's share of a row: pieces of kPiece logits, `stride` pieces apart, in rising order
// of the classes: a later logit equal to the last alternative never replaces it.
template <int DT, bool TOP>
__device__ void wave_pass(const typename Elem<DT>::T *x, uint32_t v, uint32_t first, uint32_t stride, uint32_t top,
                          Sums &q, TopList &list) {
    const uint32_t lane = __lane_id();
    float tau = -INFINITY;              // the last alternative kept so far; masked logits never pass
    for (uint64_t p = (uint64_t)first * kPiece; p < v; p += (uint64_t)stride * kPiece) {
        const uint32_t c0 = (uint32_t)p + lane * kLV;
        float e[kLH][kLV];
#pragma unroll
        for (int h = 0; h < kLH; ++h) {
            const uint32_t c = c0 + h * 64 * kLV;
            load_row<typename Elem<DT>::T, kLV>(x + c, (int64_t)v - c, -INFINITY, e[h]);
        }
        float top_e = e[0][0];
#pragma unroll
        for (int h = 0; h < kLH; ++h)
#pragma unroll
            for (int i = 0; i < kLV; ++i) top_e = fmaxf(top_e, e[h][i]);
        if (top_e > q.m) q.raise(top_e);
#pragma unroll
        for (int h = 0; h < kLH; ++h)
#pragma unroll
            for (int i = 0; i < kLV; ++i) q.add(e[h][i]);
        const uint64_t better = TOP ? __ballot(top_e > tau) : 0;
        if (better) {
            // with `top` lanes better than tau, the top-th largest of the lanes' maxima is a
            // lower bound of the last alternative after this piece: its upper 16 bits, one by one
            uint32_t floor_w = 0;
            if ((uint32_t)__popcll(better) >= top) {
                const uint32_t w = top_e > tau ? ord_of(top_e) : 0;
                for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
                    if ((uint32_t)__popcll(__ballot(w >= (floor_w | bit))) >= top) floor_w |= bit;
            }
#pragma unroll
            for (int h = 0; h < kLH; ++h)
#pragma unroll
                for (int i = 0; i < kLV; ++i) {
                    Alt mine = e[h][i] > tau && ord_of(e[h][i]) >= floor_w ? alt_of(e[h][i], c0 + h * 64 * kLV + i) : 0;
                    if (!__ballot(mine != 0)) continue;
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

// A part's results in the workspace: its sums, then its alternatives.
__host__ __device__ inline uint64_t part_bytes(uint32_t top) { return 16 + 8ull * top; }
struct Part {
    float *sums;
    Alt *alts;
    __device__ Part(const LogprobArgs &a, uint64_t i) {
        char *p = static_cast<char *>(a.work) + i * part_bytes(a.top);
        sums = reinterpret_cast<float *>(p);
        alts = reinterpret_cast<Alt *>(p + 16);
    }
};

// A row is cut into `parts` (interleaved piece by piece), a block each; with one part the
// block finishes the row.
template <int DT, bool TOP>
__global__ __launch_bounds__(64 * kLW) void k_logprobs_long(LogprobArgs a, uint32_t parts) {
    using T = typename Elem<DT>::T;
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6;
    for (uint64_t i = blockIdx.x; i < a.rows * parts; i += gridDim.x) {
        const uint64_t r = i / parts;
        const uint32_t part = (uint32_t)(i - r * parts);
        Sums q;
        TopList list{0};
        q.init();
        wave_pass<DT, TOP>(static_cast<const T *>(a.x) + r * a.ld, a.v, part * kLW + wave, parts * kLW, a.top, q,
                           list);
        block_join<TOP>(q, list);
        if (wave) continue;
        if (parts == 1) {
            finish_row<DT>(a, r, q, list.a);
        } else {
            const Part to(a, i);
            if (lane == 0) { to.sums[0] = q.m; to.sums[1] = q.s; to.sums[2] = q.t; }
            if (TOP && lane < a.top) to.alts[lane] = list.a;
        }
    }
}

template <int DT, bool TOP>
__global__ __launch_bounds__(64 * kLW) void k_logprobs_join(LogprobArgs a, uint32_t parts) {
    const uint32_t lane = __lane_id(), wave = threadIdx.x >> 6;
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        Sums q;
        TopList list{0};
        q.init();
        for (uint32_t p = wave; p < parts; p += kLW) {
            const Part from(a, r * parts + p);
            q.join(from.sums[0], from.sums[1], from.sums[2]);
            if (TOP) list.merge(lane < a.top ? from.alts[lane] : 0);
        }
        block_join<TOP>(q, list);
        if (wave == 0) finish_row<DT>(a, r, q, list.a);
    }
}

// Lanes a row and logits a lane of the short form; N 0: the long form.
struct ShortPlan {
    uint32_t n, g;
};
template <int DT> static ShortPlan short_plan(uint32_t v) {
    constexpr uint32_t wide = DT == FSX_DTYPE_F32 ? 4 : 8;   // 16 bytes a lane
    ShortPlan p{v <= 64 * wide ? wide : v <= 64 * 16 ? 16u : 0u, 1};
    while (p.n && p.g * p.n < v) p.g *= 2;
    return p;
}

// Parts of a long row: enough blocks for every CU to hold four, a piece for every wave at least.
static uint32_t long_parts(uint64_t rows, uint32_t v) {
    if (v <= 64 * 16) return 1;
    const uint64_t want = (1024 + rows - 1) / rows, most = (v + kPiece * kLW - 1) / (kPiece * kLW);
    return (uint32_t)std::min<uint64_t>({want, most, kMaxParts});
}

template <int DT, bool TOP>
static void logprobs(const LogprobArgs &a, hipStream_t st) {
    const ShortPlan p = short_plan<DT>(a.v);
    if (p.n) {
        const uint64_t blocks = (a.rows + 256 / p.g - 1) / (256 / p.g);
        const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, 1u << 16);
        if (p.n == 16) k_logprobs_short<DT, 16, TOP><<<grid, 256, 0, st>>>(a, p.g);
        else k_logprobs_short<DT, DT == FSX_DTYPE_F32 ? 4 : 8, TOP><<<grid, 256, 0, st>>>(a, p.g);
        return;
    }
    const uint32_t parts = long_parts(a.rows, a.v);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(a.rows * parts, 1u << 20);
    k_logprobs_long<DT, TOP><<<grid, 64 * kLW, 0, st>>>(a, parts);
    if (parts > 1) k_logprobs_join<DT, TOP><<<(uint32_t)std::min<uint64_t>(a.rows, 1u << 16), 64 * kLW, 0, st>>>(a, parts);
}

uint64_t logprobs_work(uint64_t rows, uint32_t v, uint32_t top) {
    const uint32_t parts = long_parts(rows, v);
    return parts > 1 ? up16(rows * parts * part_bytes(top)) : 0;
}

template <int DT>
static void logprobs(const LogprobArgs &a, hipStream_t st) {
    if (a.top) logprobs<DT, true>(a, st);
    else logprobs<DT, false>(a, st);
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
