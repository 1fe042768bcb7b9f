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

struct LargerFloat { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct LesserWord { __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return min(a, b); } };
struct PlusWord { __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a + b; } };
struct Plus { __device__ float operator()(float a, float b) const { return a + b; } };

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

// The lane's number, anew: what follows from it is not kept in registers from row to row.
__device__ __forceinline__ uint32_t lane_now() {
    uint32_t l = __lane_id();
    asm volatile("" : "+v"(l));
    return l;
}

// log s, 1 <= s (or 0, or NaN): v_log_f32 gives log2 s, which two parts of log 2 take to the
// last place.
__device__ __forceinline__ float log_of(float s) {
    const float l = __builtin_amdgcn_logf(s), hi = 0.693147182464599609375f, lo = -1.904654299957767e-9f;
    const float r = l * hi;
    return r + fmaf(l, lo, fmaf(l, hi, -r));
}

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
        t = fmaf(fmaxf(z, -200.0f), e, t);   // -inf: 0 * -200; NaN goes on through e
    }
    // the sums of the G lanes of a group, in every lane of it
    template <int G> __device__ void join_group() {
        raise(group_all<G>(m, LargerFloat()));
        s = group_all<G>(s, Plus());
        t = group_all<G>(t, Plus());
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

// A row's log S and what it says of the row; the outputs from them.
struct RowEnd {
    float m, ls, h;
    bool bad, empty;
    __device__ explicit RowEnd(const Sums &q) {
        m = q.m;
        bad = q.s != q.s;
        empty = q.s == 0.0f;
        ls = log_of(q.s);
        const float e = ls - q.t * __builtin_amdgcn_rcpf(q.s);
        h = bad ? NAN : empty || e < 0.0f ? 0.0f : e;
    }
    // log p of the class whose logit is x
    __device__ float log_p(float x) const { return bad ? NAN : empty ? -INFINITY : (x - m) - ls; }
    __device__ int32_t id(Alt a) const { return bad || a == 0 ? -1 : (int32_t)~(uint32_t)a; }
    __device__ float id_log_p(Alt a) const {
        return bad ? NAN : a == 0 ? -INFINITY : log_p(value_of((uint32_t)(a >> 32)));
    }
};

// The row's outputs, by a whole wave (all lanes hold the same sums); xt: the given class' logit.
__device__ __forceinline__ void put_row(const LogprobArgs &a, uint64_t r, const RowEnd &end, int32_t target, float xt) {
    if (a.target) a.logprob[r] = target == -1 ? 0.0f : (uint32_t)target < a.v ? end.log_p(xt) : NAN;
    if (a.entropy) a.entropy[r] = end.h;
}
__device__ void finish_row(const LogprobArgs &a, uint64_t r, const Sums &q, Alt alt, int32_t target, float xt) {
    const uint32_t lane = lane_now();
    const RowEnd end(q);
    if (lane == 0) put_row(a, r, end, target, xt);
    if (lane < a.top) {
        a.top_id[r * a.top + lane] = end.id(alt);
        a.top_lp[r * a.top + lane] = end.id_log_p(alt);
    }
}

// The upper 12 bits of the n-th largest of a wave's words, from ballots: when
// they are logits of different places, no logit below it is among the n largest.
template <int WORDS> __device__ uint32_t nth_largest(const uint32_t (&w)[WORDS], uint32_t n) {
    uint32_t f = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit >= 0x100000u; bit >>= 1) {
        uint32_t count = 0;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) count += (uint32_t)__popcll(__ballot(w[i] >= (f | bit)));
        if (count >= n) f |= bit;
    }
    return f;
}

// ---------------------------------------------------------------- short rows: G lanes a row

// A wave's RW rows: up to KEEP alternatives of each in falling order, and for RANK their words.
enum { kKeep, kRank, kChoose, kBound };   // how a row's alternatives are put in order
template <int RW, int KEEP, int PITCH, int POOL> struct ShortRows {
    Alt alts[RW * KEEP];
    Alt pool[POOL ? POOL : 1];   // kBound: the rows' candidates
    uint32_t words[PITCH ? RW * PITCH : 4];
    float2 end[RW];    // m, and log S (a bad row: NaN)
    uint32_t found[RW];
};
// What the wave's lanes have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Up to G N classes: a lane holds N neighbouring logits of its row, G lanes (a power of two)
// a row, so the row is read once and its maximum is known before the sums. A wave's alternatives
// are ordered in LDS and then stored side by side, all its rows' at once. Their order: kRank counts
// for each logit the ones before it, against the row's words from LDS; kBound first leaves out what
// cannot be one, and counts among the others; kChoose takes the group's largest word as the next
// one, and the first lane that holds it clears it; kKeep does so in registers. WHOLE: the classes are a
// multiple of N, so a lane has all of its logits or none; the next rows are then under way while
// a block works on the ones before.
template <int DT, int N, int G, bool WHOLE, int ORDER>
__global__ __launch_bounds__(256) void k_logprobs_short(LogprobArgs a, uint32_t top_inv) {
    using T = typename Elem<DT>::T;
    constexpr uint32_t PER = 256 / G, RW = 64 / G, KEEP = G * N < 64 ? G * N : 64, PITCH = G * N + 4;
    __shared__ __attribute__((aligned(16))) ShortRows<RW, KEEP, (ORDER == kRank && G > 1 ? PITCH : 0),
                                                    (ORDER == kBound ? 2 * 64 : 0)> s_rows[4];
    auto &sh = s_rows[threadIdx.x >> 6];
    const uint32_t g = threadIdx.x % G, c0 = g * N;
    const uint64_t step = (uint64_t)gridDim.x * PER;
    uint64_t r = (uint64_t)blockIdx.x * PER + threadIdx.x / G;
    const bool in_row = c0 < a.v;
    // the class of the lane's first logit: the last lanes begin so early that they end with the row, and
    // what belongs to the lane before does not count (G > 1: a row has N logits at least)
    const uint32_t cb = !WHOLE && G > 1 && c0 > a.v - N ? a.v - N : c0;
    T next[N];
    int32_t next_target = -1;
    auto fetch = [&](uint64_t row) {
        const uint64_t rr = row < a.rows ? row : a.rows - 1;
        if (a.target) next_target = a.target[rr];
        const T *p = static_cast<const T *>(a.x) + rr * a.ld + (!WHOLE && G > 1 ? cb : in_row ? c0 : 0);
        if constexpr (WHOLE || G > 1) {
            __builtin_memcpy(next, p, sizeof(next));
        } else {
            // (what follows a row's end up to the last row's can be read; it does not count)
            const int64_t ok = (int64_t)a.v, there = (int64_t)((a.rows - 1 - rr) * a.ld) + ok;
            if (there >= N) __builtin_memcpy(next, p, sizeof(next));
            else
#pragma unroll
                for (int i = 0; i < N; ++i) next[i] = p[i < ok ? i : 0];
        }
    };
    fetch(r);
    // (all lanes of a block go round together: its first row decides)
    for (uint64_t b0 = (uint64_t)blockIdx.x * PER; b0 < a.rows; b0 += step, r += step) {
        const bool live = r < a.rows;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (WHOLE ? in_row : G > 1 ? cb + i >= c0 : c0 + i < a.v) ? (float)next[i] : -INFINITY;
        const int32_t target = next_target;
        fetch(r + step);
        Sums q;
        q.init();
#pragma unroll
        for (int i = 0; i < N; ++i) q.m = fmaxf(q.m, x[i]);
        q.m = group_all<G>(q.m, LargerFloat());
#pragma unroll
        for (int i = 0; i < N; ++i) q.add(x[i]);
        q.s = group_all<G>(q.s, Plus());
        q.t = group_all<G>(q.t, Plus());
        const RowEnd end(q);
        float xt = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) xt = target == (int32_t)(cb + i) ? fmaxf(xt, x[i]) : xt;
        xt = group_all<G>(xt, LargerFloat());
        if (live && g == 0) put_row(a, r, end, target, xt);
        if (a.top == 0) continue;
        uint32_t w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = x[i] > -INFINITY ? ord_of(x[i]) : 0u;
        if constexpr (ORDER == kKeep) {
            Alt mine = 0;
            uint64_t to = r * a.top + g;
            for (uint32_t k = 0;; ++k) {
                uint32_t b = w[0];
#pragma unroll
                for (int i = 1; i < N; ++i) b = max(b, w[i]);
                const uint32_t best = group_all<G>(b, LargerWord());
                uint32_t c = ~0u;   // its first place
#pragma unroll
                for (int i = N - 1; i >= 0; --i) c = w[i] == best ? cb + i : c;
                c = group_all<G>(c, LesserWord());
                const uint32_t place = k % G;
                if (place == g) mine = best ? (Alt)best << 32 | (uint32_t)~c : 0;
                const bool last = k + 1 == a.top;
                if (last || place == G - 1) {
                    if (g <= place && live) {
                        a.top_id[to] = end.id(mine);
                        a.top_lp[to] = end.id_log_p(mine);
                    }
                    if (last) break;
                    to += G;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = c - cb == (uint32_t)i ? 0 : w[i];
            }
            continue;
        }
        const uint32_t lane = lane_now(), row = lane / G;
        Alt *to = sh.alts + row * KEEP;
        if (g == 0) sh.end[row] = {end.m, end.bad ? NAN : end.empty ? 0.0f : end.ls};
        uint32_t found = 0;   // alternatives of the row
        if constexpr (ORDER == kRank) {
            uint32_t rank[N];
#pragma unroll
            for (int i = 0; i < N; ++i) rank[i] = 0;
            if constexpr (G == 1) {
#pragma unroll
                for (int j = 1; j < N; ++j)
#pragma unroll
                    for (int i = 0; i < j; ++i) {
                        const bool before = w[i] >= w[j];
                        rank[j] += before ? 1 : 0;
                        rank[i] += before ? 0 : 1;
                    }
            } else {
                uint32_t *words = sh.words + row * PITCH;   // (in the classes' order, if not at their places)
                const uint32_t end_word = (a.v + N - 1) / N * N;
#pragma unroll
                for (int i = 0; i < N; i += 4)
                    *reinterpret_cast<uint4 *>(words + c0 + i) = uint4{w[i], w[i + 1], w[i + 2], w[i + 3]};
                wave_sync();
#pragma unroll 1
                for (uint32_t j = 0; j < end_word; j += 4) {
                    const uint4 o4 = *reinterpret_cast<const uint4 *>(words + j);
                    const uint32_t o[4] = {o4.x, o4.y, o4.z, o4.w}, ties = j < c0 ? 1 : 0;   // (equal: the lower class)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < N; ++i) rank[i] += o[e] + ties > w[i] ? 1 : 0;
                }
#pragma unroll
                for (int j = 1; j < N; ++j)
#pragma unroll
                    for (int i = 0; i < j; ++i) rank[j] += w[i] == w[j] ? 1 : 0;
                wave_sync();   // (the next rows' words come to the same place)
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                found += w[i] ? 1 : 0;
                if (w[i] && rank[i] < a.top) to[rank[i]] = (Alt)w[i] << 32 | (uint32_t)~(cb + i);
            }
            found = group_all<G>(found, PlusWord());
        } else {
            const uint64_t group = G == 64 ? ~0ull : ((1ull << G % 64) - 1) << (lane & ~(uint32_t)(G - 1));
            const uint64_t before = group & ((1ull << lane) - 1);   // lanes of the group
            uint32_t most = a.top < a.v ? a.top : a.v;
            if constexpr (ORDER == kBound) {
                // what is below the top-th largest of the lanes' largest words is no alternative
                uint32_t b[1] = {w[0]};
#pragma unroll
                for (int i = 1; i < N; ++i) b[0] = max(b[0], w[i]);
                uint32_t low = 0, n = 0;
                if constexpr (G == 64) {
                    low = nth_largest(b, a.top);
                } else {
#pragma unroll 1
                    for (uint32_t bit = 0x80000000u; bit >= 0x100000u; bit >>= 1)
                        if ((uint32_t)__popcll(__ballot(b[0] >= (low | bit)) & group) >= a.top) low |= bit;
                }
                low = max(low, 1u);
                Alt *pool = sh.pool + row * (2 * G);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint64_t m = __ballot(w[i] >= low);
                    const uint32_t place = n + (uint32_t)__popcll(m & before);
                    if (w[i] >= low && place < 2 * G) pool[place] = (Alt)w[i] << 32 | (uint32_t)~(cb + i);
                    n += (uint32_t)__popcll(m & group);
                }
                wave_sync();
                if (__ballot(n > 2 * G) == 0) {   // (else one by one)
                    const Alt x0 = g < n ? pool[g] : 0, x1 = g + G < n ? pool[g + G] : 0;
                    const uint32_t longest = G == 64 ? n : group_all<64>(n, LargerWord());
                    uint32_t r0 = 0, r1 = 0;
#pragma unroll 4
                    for (uint32_t i = 0; i < longest; ++i) {
                        const Alt o = i < n ? pool[i] : 0;
                        r0 += o > x0 ? 1 : 0;
                        r1 += o > x1 ? 1 : 0;
                    }
                    if (x0 && r0 < a.top) to[r0] = x0;
                    if (x1 && r1 < a.top) to[r1] = x1;
                    found = n < a.top ? n : a.top;
                    most = 0;
                }
            }
#pragma unroll 1
            for (uint32_t k = 0; k < most; ++k) {
                uint32_t b = w[0];
#pragma unroll
                for (int i = 1; i < N; ++i) b = max(b, w[i]);
                const uint32_t best = group_all<G>(b, LargerWord());
                if (!__ballot(best != 0)) break;
                found += best ? 1 : 0;
                const uint64_t holders = __ballot(b == best);
                if (b == best && best && !(holders & before)) {
                    uint32_t c = cb;
                    bool gone = false;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const bool it = !gone && w[i] == best;
                        c = it ? cb + i : c;
                        w[i] = it ? 0 : w[i];
                        gone = gone || it;
                    }
                    to[k] = (Alt)best << 32 | (uint32_t)~c;
                }
            }
        }
        if (g == 0) sh.found[row] = found;
        wave_sync();
        const uint64_t r0 = b0 + (threadIdx.x >> 6) * RW;
        const uint32_t rows = r0 >= a.rows ? 0 : a.rows - r0 < RW ? (uint32_t)(a.rows - r0) : RW;
#pragma unroll 1
        for (uint32_t i = lane; i < rows * a.top; i += 64) {
            const uint32_t q = i * top_inv >> 18, k = i - q * a.top;   // i / top: i < 2^12
            const float2 e = sh.end[q];
            const Alt alt = k < sh.found[q] ? sh.alts[q * KEEP + k] : 0;
            const bool none = alt == 0, bad = e.y != e.y;
            a.top_id[r0 * a.top + i] = bad || none ? -1 : (int32_t)~(uint32_t)alt;
            a.top_lp[r0 * a.top + i] = bad ? NAN : none ? -INFINITY : (value_of((uint32_t)(alt >> 32)) - e.x) - e.y;
        }
        wave_sync();
    }
}

template <int DT, int N, int G> static bool logprobs_short(const LogprobArgs &a, hipStream_t st) {
    const uint64_t blocks = (a.rows + 256 / G - 1) / (256 / G);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, 256 * 8);   // (the blocks that fit at once)
    const uint32_t top_inv = a.top ? ((1u << 18) + a.top - 1) / a.top : 0;
    // A few alternatives: kept in registers and stored as they come (us of 2^22 rows of 16 f32 logits,
    // 1 / 3 / 5 alternatives: 72 / 88 / 112, by way of LDS 77 / 92 / 115; 200000 bf16 rows of 200, 1 / 3 / 4 / 8:
    // 45 / 64 / 74 / 113 and 51 / 65 / 72 / 102). Counting costs what the row is long, choosing what is asked
    // for: about v (2 N + 2) and 3 / 5 top (4 N + 3 log2 G + 14) instructions a lane (us, counted and one by one: 2^19
    // rows of 16, 8 / 12 / 16 asked for 24 / 26 / 27 and 22 / 27 / 33; 2^18 of 33, 12 / 20 / 33 63 / 65 / 69 and 47 /
    // 67 / 101; 2^18 of 64, 24 / 32 / 48 89 / 90 / 93 and 74 / 93 / 132; 2^17 of 100, 32 / 48 / 64 124 / 125 / 128 and 96 /
    // 136 / 176; of 128, always one by one, 48 / 64 150 / 151 and 131 / 170).
    constexpr uint32_t log_g = G > 32 ? 6 : G > 16 ? 5 : G > 8 ? 4 : G > 4 ? 3 : G > 2 ? 2 : G > 1 ? 1 : 0;
    const uint32_t rank_cost = G == 1 ? 2 * N * N : a.v * (2 * N + 2),
                   rounds_cost = std::min(a.top, a.v) * (4 * N + 3 * log_g + 14);
    auto go = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(a, top_inv); };
    if (a.top <= 3) {
        if (a.v % N == 0) go(k_logprobs_short<DT, N, G, true, kKeep>);
        else go(k_logprobs_short<DT, N, G, false, kKeep>);
        return true;
    }
    if constexpr (G * N <= 512) {
        if (5 * rank_cost < 3 * rounds_cost) {
            if (a.v % N == 0) go(k_logprobs_short<DT, N, G, true, kRank>);
            else go(k_logprobs_short<DT, N, G, false, kRank>);
            return true;
        }
    }
    // Bounding costs the same for any number, if there are lanes enough for a bound (us of 20000 bf16 rows of
    // 500, 4 / 12 / 40 / 56 asked for: bounded 16.5 / 18.6 / 26 / 91, chosen 17.8 / 31 / 79 / 108; of 200, half a wave a row,
    // 5 / 9 / 20 / 22: 11.6 / 12.6 / 17.1 / 22.1 and 9.9 / 12.9 / 21.1 / 22.6, with 24 of 25 lanes 28.7 and 24.0; a
    // quarter of a wave gains nothing).
    if constexpr (G >= 32) {
        if (a.top >= (G == 64 ? 4 : 9) && 8 * ((a.v + N - 1) / N) >= 9 * a.top) {
            if (a.v % N == 0) go(k_logprobs_short<DT, N, G, true, kBound>);
            else go(k_logprobs_short<DT, N, G, false, kBound>);
            return true;
        }
    }
    if (a.v % N == 0) go(k_logprobs_short<DT, N, G, true, kChoose>);
    else go(k_logprobs_short<DT, N, G, false, kChoose>);
    return true;
}
// Eight logits a lane as far as 64 lanes reach, then sixteen, unless more alternatives are asked for than
// its lanes can bound; else in blocks (20000 bf16 rows of 1004, 0 / 1 / 5 / 20 / 40 alternatives 12.3 / 17.7 / 27 / 31 / 38
// us, in blocks 20 / 40 / 44 / 49 / 62; 40 of 600, one by one: 127 and 63). 32 a lane leave too few waves (31582 rows of
// 1279, 1 / 5 / 20: 48 / 86 / 95, in blocks 63 / 70 / 79).
constexpr uint32_t kShort = 64 * 8;
constexpr uint64_t kManyRows = 1024;   // for long rows: blocks of four waves from here on
constexpr uint32_t kPool = 128;       // a wave's candidates: 64 alternatives and one of every lane
constexpr uint32_t kFewTop = 32;       // up to here a bound from 64 words does; beyond, from 256
template <int DT> static bool logprobs_short(const LogprobArgs &a, hipStream_t st) {
    if (a.v > kShort) {
        if (a.v > 1024 || (a.top > 3 && 8 * ((a.v + 15) / 16) < 9 * a.top)) return false;
        return logprobs_short<DT, 16, 64>(a, st);
    }
    // 32-bit logits four a lane where half the lanes would do nothing, or where a bound needs more of them (us,
    // four and eight a lane: 2^22 rows of 16, 1 / 3 alternatives 79 / 107 and 71 / 87; 100000 of 175, 6 / 9 / 12 / 15 / 18 /
    // 30 56 / 59 / 61 / 64 / 67 / 85 and 50 / 58 / 62 / 67 / 75 / 148, of 256, 9 / 15 / 26 / 40 60 / 66 / 76 / 96 and 59 / 66 /
    // 100 / 173; of 140 with 40, which the lanes of neither can bound, 267 and 191)
    if constexpr (DT == FSX_DTYPE_F32) {
        if (a.v <= 4) return logprobs_short<DT, 4, 1>(a, st);
        if (a.v > 128 && a.v <= 256 && a.top > 8) return logprobs_short<DT, 4, 64>(a, st);
    }
    if (a.v <= 8) return logprobs_short<DT, 8, 1>(a, st);
    if (a.v <= 16) return logprobs_short<DT, 8, 2>(a, st);
    if (a.v <= 32) return logprobs_short<DT, 8, 4>(a, st);
    if (a.v <= 64) return logprobs_short<DT, 8, 8>(a, st);
    if (a.v <= 128) return logprobs_short<DT, 8, 16>(a, st);
    if (a.v <= 256) return logprobs_short<DT, 8, 32>(a, st);
    return logprobs_short<DT, 8, 64>(a, st);
}

// ---------------------------------------------------------------- long rows: blocks of W waves

constexpr int kLV = 8;             // neighbouring logits a lane reads
constexpr uint32_t kMaxParts = 64;

// The wave's number in its block, as the scalar that it is.
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Candidates for a row's alternatives: each wave collects its own, unordered; an order comes
// from counting for each how many are larger (their words all differ), so no list is kept
// sorted and no lane waits for another.
template <int W> struct Shared {
    Alt pool[W][kPool];
    Alt all[W * kPool];
    Alt best[64];
    uint32_t word[64 * W];
    float sums[W][3];
    uint32_t total;
};
struct Pool {
    Alt *at;
    uint32_t n;   // (the same in the wave)
    __device__ void put(uint64_t m, bool want, Alt a) {   // m: the lanes that want
        if (want) at[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = a;
        n += (uint32_t)__popcll(m);
    }
    // only the `top` largest stay, in falling order; the last one's word (there are more than `top`)
    __device__ uint32_t keep_best(uint32_t top) {
        const uint32_t lane = __lane_id();
        const Alt a = lane < n ? at[lane] : 0, b = lane + 64 < n ? at[lane + 64] : 0;
        uint32_t ra = 0, rb = 0;
#pragma unroll 1
        for (uint32_t i = 0; i < n; ++i) {
            const Alt o = at[i];
            ra += o > a;
            rb += o > b;
        }
        if (a && ra < top) at[ra] = a;
        if (b && rb < top) at[rb] = b;
        n = top;
        return __builtin_amdgcn_readfirstlane((uint32_t)(at[top - 1] >> 32));
    }
};

// A lower bound of the n-th largest of what the waves' lanes put into sh.word, from 64 words
// (each the largest of a lane of all waves) or, for many alternatives, 256.
template <int W> __device__ __forceinline__ uint32_t bound(const Shared<W> &sh, uint32_t n) {
    const uint32_t lane = lane_now();
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = sh.word[64 * i + lane];
#pragma unroll
        for (int j = i + 4; j < W; j += 4) w[i] = max(w[i], sh.word[64 * j + lane]);
    }
    if (n > kFewTop) return nth_largest(w, n);
    const uint32_t one[1] = {max(max(w[0], w[1]), max(w[2], w[3]))};
    return nth_largest(one, n);
}

// The waves' sums and pools: the block's sums in every lane, its `top` largest candidates in
// falling order, the i-th in lane i of the first wave (0: none). sh.total was 0 before a barrier.
template <int W, bool TOP>
__device__ __forceinline__ Alt block_join(Shared<W> &sh, Sums &q, const Pool &pool, uint32_t top) {
    const uint32_t lane = lane_now(), wave = wave_id();
    if (lane == 0) {
        sh.sums[wave][0] = q.m;
        sh.sums[wave][1] = q.s;
        sh.sums[wave][2] = q.t;
    }
    if (TOP) {
        if (wave == 0) sh.best[lane] = 0;
        uint32_t base = 0;
        if (lane == 0 && pool.n) base = atomicAdd(&sh.total, pool.n);   // (any order: it ends in one by value)
        base = __builtin_amdgcn_readfirstlane(base);
        if (lane < pool.n) sh.all[base + lane] = pool.at[lane];
        if (lane + 64 < pool.n) sh.all[base + lane + 64] = pool.at[lane + 64];
    }
    __syncthreads();
    q.m = sh.sums[lane & (W - 1)][0];
    q.s = sh.sums[lane & (W - 1)][1];
    q.t = sh.sums[lane & (W - 1)][2];
    q.template join_group<W>();
    if (!TOP) {
        __syncthreads();
        return 0;
    }
    const uint32_t n = __builtin_amdgcn_readfirstlane(sh.total);
#pragma unroll 1
    for (uint32_t first = wave * 64; first < n; first += W * 64) {
        const Alt a = first + lane < n ? sh.all[first + lane] : 0;
        uint32_t rank = 0, i = 0;
#pragma unroll 1
        for (; i + 8 <= n; i += 8) {
            Alt o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = sh.all[i + j];
#pragma unroll
            for (int j = 0; j < 8; ++j) rank += o[j] > a;
        }
#pragma unroll 1
        for (; i < n; ++i) rank += sh.all[i] > a;
        if (a && rank < top) sh.best[rank] = a;
    }
    __syncthreads();
    return sh.best[lane];
}

// A block's share of a row: its waves' pieces of 64 kLV H logits, in rising order of the classes,
// so that a later logit equal to a wave's last alternative never replaces it. A logit is a
// candidate if its ordered word is `low` at least.
//
// The code is kept small (one copy of each part, loops that are not unrolled): the time of a
// short call is else that of fetching its instructions.
template <int DT, int W, int H, bool TOP>
__device__ __forceinline__ void block_pass(Shared<W> &sh, const typename Elem<DT>::T *x, uint32_t v, uint32_t part,
                                           uint32_t parts, uint32_t top, Sums &q, Pool &pool) {
    using T = typename Elem<DT>::T;
    constexpr uint32_t kPiece = 64 * kLV * H;
    const uint32_t lane = lane_now(), wave = wave_id();
    q.init();
    pool.at = sh.pool[wave];
    pool.n = 0;
    uint32_t low = ord_of(kLowest);   // masked logits never pass
    uint32_t round = 0, refresh = 0;
    // the lane's reads; one that would pass the row's end (v > kLV) begins before its place and
    // what belongs to others does not count
    const uint32_t end = v - kLV, step = parts * W * kPiece;
    T raw[H][kLV];
    auto read = [&](uint32_t c0) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint32_t c = c0 + h * 64 * kLV;
            __builtin_memcpy(raw[h], x + (c < end ? c : end), sizeof(raw[h]));
        }
    };
    constexpr bool AHEAD = H == 1 && W == 16;   // (else a row is one round or few, or the registers go to more waves)
    if (AHEAD) read((part * W + wave) * kPiece + lane * kLV);
#pragma unroll 1
    for (uint32_t block_at = part * W * kPiece; block_at < v; block_at += step, ++round) {   // (< 2^32)
        const uint32_t at = block_at + wave * kPiece;
        const bool some = at < v;
        const uint32_t c0 = at + lane * kLV;
        float e[H][kLV];
        float top_e = -INFINITY;
        if (some) {
            if (!AHEAD) read(c0);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < kLV; ++i) e[h][i] = (float)raw[h][i];
            if (AHEAD) read(c0 + step);   // (behind the row: its end once more, unused)
            if (at + kPiece > v) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const uint32_t c = c0 + h * 64 * kLV;
#pragma unroll
                    for (int i = 0; i < kLV; ++i) e[h][i] = c > end && end + i < c ? -INFINITY : e[h][i];
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < kLV; ++i) top_e = fmaxf(top_e, e[h][i]);
            if (top_e > q.m) q.raise(top_e);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < kLV; ++i) q.add(e[h][i]);
            asm volatile("" : "+v"(q.s), "+v"(q.t));   // (the sums are done before the candidates)
        }
        if (!TOP) continue;
        // a lower bound of the block's last alternative, from its lanes' largest logits so far, in
        // rounds 0, 1, 4, 16, 64 ..
        if (round == refresh) {
            if (round) __syncthreads();   // (the time before still reads the words)
            else if (threadIdx.x == 0) sh.total = 0;
            refresh = round ? 4 * round : 1;
            sh.word[threadIdx.x] = ord_of(q.m);
            __syncthreads();
            low = max(low, bound(sh, top));
        }
        if (!some || !__ballot(top_e >= value_of(low))) continue;
        const float lim = value_of(low);
        uint32_t done = H * kLV;   // the first logit of a lane that found no room
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float here = e[h][0];
#pragma unroll
            for (int i = 1; i < kLV; ++i) here = fmaxf(here, e[h][i]);
            if (!__ballot(here >= lim)) continue;
            const uint32_t c = c0 + h * 64 * kLV, from = c < end ? c : end;
#pragma unroll
            for (int i = 0; i < kLV; ++i) {
                const uint64_t m = __ballot(e[h][i] >= lim);
                if (!m || done < H * kLV) continue;
                if (pool.n + (uint32_t)__popcll(m) > kPool) done = h * kLV + i;
                else pool.put(m, e[h][i] >= lim, alt_of(e[h][i], from + i));
            }
        }
        if (done == H * kLV) continue;
        // no room: one logit of each lane at a time, read again, room made before it
#pragma unroll 1
        for (uint32_t i = done; i < H * kLV; ++i) {
            const uint32_t c = c0 + i / kLV * 64 * kLV, cls = (c < end ? c : end) + i % kLV;
            const float y = cls >= c ? (float)x[cls] : -INFINITY;
            if (pool.n + 64 > kPool) low = max(low, pool.keep_best(top));
            const bool want = y >= value_of(low);
            pool.put(__ballot(want), want, alt_of(y, cls));
        }
        if (pool.n > top) low = max(low, pool.keep_best(top) + 1);   // (later an equal logit comes too late)
    }
    q.template join_group<64>();
}

// The given class and its logit, by the lanes that ask for them.
template <int DT> __device__ __forceinline__ void given(const LogprobArgs &a, uint64_t r, int32_t &t, float &x) {
    t = a.target ? a.target[r] : -1;
    x = (uint32_t)t < a.v ? (float)static_cast<const typename Elem<DT>::T *>(a.x)[r * a.ld + (uint32_t)t] : 0.0f;
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

// A row is cut into `parts` (interleaved round by round), a block each; with one part the
// block finishes the row.
template <int DT, int W, int H, bool TOP>
__global__ __launch_bounds__(64 * W, 8) void k_logprobs_long(LogprobArgs a, uint32_t parts) {
    using T = typename Elem<DT>::T;
    __shared__ Shared<W> sh;
    const uint32_t part = blockIdx.x;
#pragma unroll 1
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        Sums q;
        Pool pool;
        block_pass<DT, W, H, TOP>(sh, static_cast<const T *>(a.x) + r * a.ld, a.v, part, parts, a.top, q, pool);
        const Alt alt = block_join<W, TOP>(sh, q, pool, a.top);
        if (wave_id()) continue;
        const uint32_t lane = lane_now();
        if (parts == 1) {
            int32_t t = -1;
            float xt = 0.0f;
            if (lane == 0) given<DT>(a, r, t, xt);
            finish_row(a, r, q, alt, t, xt);
        } else {
            const Part to(a, r * parts + part);
            if (lane == 0) { to.sums[0] = q.m; to.sums[1] = q.s; to.sums[2] = q.t; }
            if (TOP && lane < a.top) to.alts[lane] = alt;
        }
    }
}

// The parts of a row, a block for each: a lane of the first wave takes a part's sums; the waves take
// the parts' alternatives in turn, above a lower bound from the first few of every part.
template <int DT, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_join(LogprobArgs a, uint32_t parts) {
    constexpr int W = 4;
    __shared__ Shared<W> sh;
    const uint32_t lane = __lane_id(), wave = wave_id();
    const uint64_t r = blockIdx.x;
    Sums q;
    Pool pool{sh.pool[wave], 0};
    q.init();
    int32_t t = -1;
    float xt = 0.0f;
    if (threadIdx.x == 0) given<DT>(a, r, t, xt);
    if (TOP) {
        const uint32_t per = (a.top > kFewTop ? 256 : 64) / parts, nth = threadIdx.x / parts;
        const Alt sample = nth < a.top && nth < per ? Part(a, r * parts + threadIdx.x % parts).alts[nth] : 0;
        if (threadIdx.x == 0) sh.total = 0;
        sh.word[threadIdx.x] = (uint32_t)(sample >> 32);
    }
    if (wave == 0 && lane < parts) {
        const Part from(a, r * parts + lane);
        q.join(from.sums[0], from.sums[1], from.sums[2]);
    }
    q.template join_group<64>();
    if (TOP) {
        __syncthreads();
        const uint32_t low = bound(sh, a.top);
#pragma unroll 1
        for (uint32_t p = wave; p < parts; p += 4 * W) {
            Alt mine[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                mine[j] = p + j * W < parts && lane < a.top ? Part(a, r * parts + p + j * W).alts[lane] : 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (pool.n + 64 > kPool) pool.keep_best(a.top);
                const bool want = mine[j] != 0 && (uint32_t)(mine[j] >> 32) >= low;
                pool.put(__ballot(want), want, mine[j]);
            }
        }
    }
    const Alt alt = block_join<W, TOP>(sh, q, pool, a.top);
    if (wave == 0) finish_row(a, r, q, alt, t, xt);
}

// Many rows: a block of four waves each. Fewer: of sixteen, each with less to do, and with
// fewer rows than half the CUs a row in parts, a round for every block at least.
static constexpr int kFewW = 16, kFewH = 1;
static uint32_t long_parts(uint64_t rows, uint32_t v) {
    if (v <= kShort || rows >= kManyRows) return 1;
    const uint64_t want = (256 + rows / 2) / rows, most = (v + 64 * kLV * kFewH * kFewW - 1) / (64 * kLV * kFewH * kFewW);
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({want, most, kMaxParts}));
}

template <int DT, bool TOP>
static void logprobs(const LogprobArgs &a, hipStream_t st) {
    const uint32_t parts = long_parts(a.rows, a.v);
    const dim3 grid(parts, (uint32_t)std::min<uint64_t>(a.rows, 65535));
    // Pieces as large as all waves of a block have some (us, pieces of 512 / 1024 / 2048): 20000 rows of 2048 with
    // 1 / 20 / 64 alternatives 42 / 43 / 47, 53 / 57 / 68, 78 / 87 / 950; 31582 of 1279 with 5 70 / 77 / 90; 9183 of
    // 3199 with 20 39 / 32 / 38; 10000 of 5000 52 / 49 / 44. 700 rows of 2048: 5.5 - 8.2 us, with sixteen waves a row
    // 8.6 - 12.8.
    if (a.v <= 2048) k_logprobs_long<DT, 4, 1, TOP><<<grid, 64 * 4, 0, st>>>(a, 1);
    else if (a.rows >= kManyRows && a.v <= 4096) k_logprobs_long<DT, 4, 2, TOP><<<grid, 64 * 4, 0, st>>>(a, 1);
    else if (a.rows >= kManyRows) k_logprobs_long<DT, 4, 4, TOP><<<grid, 64 * 4, 0, st>>>(a, 1);
    else k_logprobs_long<DT, kFewW, kFewH, TOP><<<grid, 64 * kFewW, 0, st>>>(a, parts);
    if (parts > 1) k_logprobs_join<DT, TOP><<<(uint32_t)a.rows, 256, 0, st>>>(a, parts);   // (up to 170 rows)
}

uint64_t logprobs_work(uint64_t rows, uint32_t v, uint32_t top) {
    const uint32_t parts = long_parts(rows, v);
    return parts > 1 ? up16(rows * parts * part_bytes(top)) : 0;
}

template <int DT>
static void logprobs(const LogprobArgs &a, hipStream_t st) {
    if (logprobs_short<DT>(a, st)) return;
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
