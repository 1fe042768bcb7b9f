// fsx_linear.hip — int8 layers of free size: the row quantiser and the int8 matrix product
// with a scale for every row of x and every output channel (include/fsx_hip.h).
//
//   scale_r = max(fl32(max_c |x_rc| / 127), 2^-126)      q_rc = rhe(x_rc / scale_r)
//   y_rn    = act((float)(sum_k q_rk w_nk) * scale_r * t_n + b_n)
#include <hip/hip_runtime.h>
#include <algorithm>

#include "fsx_q8_rows.h"

namespace fsx {

constexpr int kSums = -1;   // results that are sums still

// ---------------------------------------------------------------- int8 product

// ---- few rows: the weights' bytes bound it
//
// A block takes 16 channels and all of k, its FW waves 128 bytes of k (whole lines) each in turn,
// straight from memory into v_mfma_i32_16x16x64_i8, the weights first: lane l gives bytes
// 16 (l / 16) .. of row l % 16 of either operand and holds channels 4 (l / 16) .. of row l % 16
// of the result. MT groups of 16 rows; the waves' sums meet in LDS. FLOATS: up to four rows of
// floats, quantised by every block into LDS while its first weights are under way (x is small
// and comes from cache): one launch instead of two.
constexpr int kFU = 8;          // loads of weights in flight a lane
constexpr uint32_t kFusedRows = 4, kFusedBytes = 32768;

template <int XT, int MT, int FW>
__global__ __launch_bounds__(64 * FW) void k_linear_few(LinearArgs a, int yt) {
    constexpr bool FLOATS = XT != FSX_DTYPE_I8;
    constexpr uint32_t THREADS = 64 * FW;
    extern __shared__ __attribute__((aligned(16))) int8_t s_x[];   // FLOATS: the rows' codes, up64(k) + 16 apart
    __shared__ __attribute__((aligned(16))) v4i s_acc[FW][MT][64];
    __shared__ uint32_t s_max[kFusedRows];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15,
                   lq = lane >> 4;
    const uint64_t n0 = (uint64_t)blockIdx.x * 16, c = n0 + lr < a.n ? n0 + lr : a.n - 1;
    const uint32_t chunks = (a.k + 63) / 64, pitch = chunks * 64 + 16;
    const int8_t *pw = a.w + c * a.ldw + 16 * lq;
    // the wave's u-th load of round t: the place in k of 64 bytes
    auto place = [&](uint32_t t, int u) { return (2 * (wave + FW * (t * (kFU / 2) + u / 2)) + u % 2) * 64; };
    auto load = [&](const int8_t *p, uint32_t k0) {
        return k0 + 64 <= a.k ? load16(p + k0, 16) : load16(p + k0, (int64_t)a.k - k0 - 16 * lq);
    };
    v4i w[kFU];
    auto weights = [&](uint32_t t) {
#pragma unroll
        for (int u = 0; u < kFU; ++u) w[u] = load(pw, place(t, u));
    };
    weights(0);
    if constexpr (FLOATS) {
        const auto *x = static_cast<const typename Elem<XT>::T *>(a.x);
        const uint32_t per = chunks * 4, all = (uint32_t)a.rows * per;   // chunks of 16, zeros behind the end
        if (threadIdx.x < kFusedRows) s_max[threadIdx.x] = 0;
        __syncthreads();
        RawChunk<XT> first;   // (kept: rows of up to 16 THREADS values are read once)
        auto each = [&](auto f) {
            for (uint32_t q0 = 0; q0 < all; q0 += THREADS) {
                const uint32_t q = q0 + threadIdx.x, r = q < all ? q / per : 0, k0 = (q - r * per) * 16;
                f(q0, q < all, r, k0, q < all && k0 < a.k);
            }
        };
        each([&](uint32_t q0, bool, uint32_t r, uint32_t k0, bool some) {
            RawChunk<XT> raw;
            uint32_t m = 0;
            if (some) {
                raw.load(x + r * a.ldx + k0, (int64_t)a.k - k0);
                m = raw.mag();
            }
            if (q0 == 0) first = raw;
            const uint32_t r0 = __builtin_amdgcn_readfirstlane(r);
            if (__ballot(some && r != r0) == 0) {
                m = group_all<64>(m, LargerWord());
                if (lane == 0) atomicMax(&s_max[r0], m);
            } else if (some) {
                atomicMax(&s_max[r], m);
            }
        });
        __syncthreads();
        each([&](uint32_t q0, bool in, uint32_t r, uint32_t k0, bool some) {
            const float s = row_scale(mag_value<XT>(s_max[r]));
            v4i codes = {0, 0, 0, 0};
            if (some && s == s) {
                RawChunk<XT> raw = first;
                if (q0) raw.load(x + r * a.ldx + k0, (int64_t)a.k - k0);
                codes = raw.codes(1.0f / s, s);
            }
            if (in) *reinterpret_cast<v4i *>(s_x + r * pitch + k0) = codes;
        });
        __syncthreads();
    }
    v4i acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = v4i{0, 0, 0, 0};
    for (uint32_t t = 0; place(t, 0) < a.k; ++t) {
        if (t) weights(t);
#pragma unroll
        for (int u = 0; u < kFU; ++u) {
            const uint32_t k0 = place(t, u);
            if (k0 >= a.k) break;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint32_t r = 16 * m + lr, rr = r < a.rows ? r : (uint32_t)a.rows - 1;
                v4i x;
                if (FLOATS) x = *reinterpret_cast<const v4i *>(s_x + rr * pitch + k0 + 16 * lq);
                else x = load(static_cast<const int8_t *>(a.x) + rr * a.ldx + 16 * lq, k0);
                acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u], x, acc[m], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) s_acc[wave][m][lane] = acc[m];
    __syncthreads();
    if (wave >= MT) return;
    v4i sum = s_acc[0][wave][lane];
#pragma unroll
    for (int i = 1; i < FW; ++i) sum += s_acc[i][wave][lane];
    const uint64_t r = 16 * wave + lr;
    if (r >= a.rows) return;
    float xs;
    if constexpr (FLOATS) xs = row_scale(mag_value<XT>(s_max[r]));
    else xs = a.x_scale[r];
    put_sums(a, yt, sum, xs, r, n0 + 4 * lq);
}

template <int XT, int MT> static void linear_few(const LinearArgs &a, uint32_t lds, int yt, hipStream_t st) {
    const uint32_t blocks = (a.n + 15) / 16;
    // us of one row, 4096 / 8192 / 16384 channels of 4096: eight waves 6.4 / 9.1 / 16.8, sixteen
    // 5.9 / 10.9 / 20.0
    if (blocks >= 512) k_linear_few<XT, MT, 8><<<blocks, 512, lds, st>>>(a, yt);
    else k_linear_few<XT, MT, 16><<<blocks, 1024, lds, st>>>(a, yt);
}
template <int XT> static void linear_few(const LinearArgs &a, int yt, hipStream_t st) {
    if constexpr (XT != FSX_DTYPE_I8)
        linear_few<XT, 1>(a, (uint32_t)a.rows * ((a.k + 63) / 64 * 64 + 16), yt, st);
    else if (a.rows <= 16) linear_few<XT, 1>(a, 0, yt, st);
    else linear_few<XT, 2>(a, 0, yt, st);
}

// The tiles of a product over the launch's blocks. Blocks go to the 8 XCDs in turn, each with
// an L2 of its own: an XCD takes a run of neighbouring tiles, and within it groups of kGroup
// tiles along the rows, so that the tiles at work on one XCD share channels and rows.
struct TileGrid {
    static constexpr uint32_t kXcds = 8, kGroup = 8;
    uint32_t tn, tm, tiles;
    TileGrid(uint64_t n_tiles, uint64_t m_tiles) : tn((uint32_t)n_tiles), tm((uint32_t)m_tiles), tiles(tn * tm) {}
    __device__ __forceinline__ void place(uint32_t block, uint32_t &bn, uint32_t &bm) const {
        const uint32_t q = tiles / kXcds, rest = tiles % kXcds, xcd = block % kXcds, in = block / kXcds;
        const uint32_t t = xcd * q + (xcd < rest ? xcd : rest) + in;
        const uint32_t group = t / (kGroup * tn), first = group * kGroup;
        const uint32_t size = tm - first < kGroup ? tm - first : kGroup, within = t - group * kGroup * tn;
        bm = first + within % size;
        bn = within / size;
    }
};

// ---- tiles of BN channels x BM rows, waves of WN x WM, BK bytes of k at a time through LDS
//
// The weights are the first operand of v_mfma_i32_32x32x32_i8 and x the second: lane l gives
// bytes 16 (l / 32) .. of row l % 32 of either, and holds channels 8 j + 4 (l / 32) .. + 3 of
// row l % 32 of the result: four neighbouring channels of one row.
//
// LDS holds a row's BK bytes as 16-byte chunks, chunk c of row r at place c ^ key(r): sixteen
// lanes read one chunk of sixteen rows at once, and those of them whose rows share banks (256
// bytes hold 256 / BK rows) then meet different ones.
template <int BK> __device__ __forceinline__ uint32_t place_key(uint32_t row) {
    return row / (256 / BK) % (BK / 16);
}

#ifdef __HIP_DEVICE_COMPILE__   // (buffer descriptors are no host type)
// A tile's rows of one operand into LDS, LOADS chunks a thread. DMA: the loads write LDS
// themselves (chunks at 16-byte addresses); else they pass through registers.
template <int ROWS, int BK, int THREADS, bool DMA> struct Stage {
    static constexpr int LOADS = ROWS * BK / 16 / THREADS, PER = BK / 16, STEP = THREADS / PER;
    static_assert(LOADS > 0 && STEP % 16 == 0, "whole rows, the same key for a thread's chunks");
    const int8_t *base;      // the tile's first row
    __amdgpu_buffer_rsrc_t buf;   // the tile's rows (DMA): bounds for the hardware
    uint32_t at, off[LOADS]; // the thread's chunk in a row, and from `base` to its chunks (ld < 2^23)
    uint64_t row[DMA ? 1 : LOADS];
    v4i reg[DMA ? 1 : LOADS];
    // chunk i of this thread: row i STEP + threadIdx / PER, place threadIdx % PER. Rows behind
    // the last: the last one, its results are not stored.
    __device__ __forceinline__ void init(const int8_t *p, uint64_t ld, uint64_t r0, uint64_t rows,
                                         uint32_t k) {
        const uint32_t tr = threadIdx.x / PER, pos = threadIdx.x % PER;
        at = 16 * (pos ^ place_key<BK>(tr));
        base = p + r0 * ld;
        const uint32_t last = (uint32_t)(rows - r0 < ROWS ? rows - r0 : ROWS) - 1;
        // raw buffer, 32-bit data; it ends with the chunk that the last row's end lies in
        if (DMA) buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(base), 0, last * (uint32_t)ld + ((k + 15) & ~15u), 0x00020000);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t r = i * STEP + tr, rr = r < last ? r : last;
            if (DMA) off[i] = rr * (uint32_t)ld + at;
            else row[i] = rr * ld;
        }
    }
    // A chunk that starts behind the row's end: the row's first (x is cleared there); an
    // aligned chunk that starts inside the row stays in its page.
    __device__ __forceinline__ void load(int8_t *lds, uint32_t wave, uint32_t k0, uint32_t k) {
        if constexpr (DMA) {
            auto go = [&](uint32_t back) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(
                        buf, (__attribute__((address_space(3))) void *)(lds + (i * THREADS + wave * 64) * 16), 16,
                        off[i] - back, k0, 0, 0);
            };
            if (k0 + BK <= k) go(0);
            else go(k0 + at < k ? 0 : k0 + at);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) reg[i] = load16(base + row[i] + k0 + at, (int64_t)k - k0 - at);
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) {
        if (!DMA)
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                *reinterpret_cast<v4i *>(lds + (i * THREADS + threadIdx.x) * 16) = reg[i];
    }
};

// MF 32: v_mfma_i32_32x32x32_i8, 16: v_mfma_i32_16x16x64_i8.
template <int MF, int WN, int WM, int BK>
struct WaveTile {
    static constexpr int TN = WN / MF, TM = WM / MF, S = BK * MF / 1024, E = MF * MF / 64;
    typedef int Acc __attribute__((ext_vector_type(E)));
    Acc acc[TN][TM];
    struct Frag { v4i w[TN], x[TM]; };
    Frag f[2];
    __device__ __forceinline__ void read(Frag &to, const int8_t *sw, const int8_t *sx, uint32_t wn, uint32_t wm, int s) {
        const uint32_t lane = __lane_id(), lr = lane % MF, at = ((64 / MF * s + lane / MF) ^ place_key<BK>(lr)) * 16;
#pragma unroll
        for (int i = 0; i < TN; ++i) to.w[i] = *reinterpret_cast<const v4i *>(sw + (wn + MF * i + lr) * BK + at);
#pragma unroll
        for (int j = 0; j < TM; ++j) to.x[j] = *reinterpret_cast<const v4i *>(sx + (wm + MF * j + lr) * BK + at);
    }
    // Step s of a tile from f[s & 1], the next step's reads under way meanwhile.
    template <typename F> __device__ __forceinline__ void step(int s, F next) {
        __builtin_amdgcn_sched_barrier(0);
        next(f[(s + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                if constexpr (MF == 32)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[s & 1].w[i], f[s & 1].x[j], acc[i][j], 0, 0, 0);
                else
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[s & 1].w[i], f[s & 1].x[j], acc[i][j], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
    }
};

// x of the last tile behind the rows' end, `left` bytes into the tile: 0 (weights there count nothing then).
template <int BM, int BK, int THREADS>
__device__ __forceinline__ void clear_tail(int8_t *sx, uint32_t left) {
    if (left >= BK) return;
#pragma unroll 1
    for (uint32_t c = threadIdx.x; c < BM * BK / 16; c += THREADS) {
        const uint32_t r = c / (BK / 16), first = 16 * (c % (BK / 16) ^ place_key<BK>(r));
        v4i v = *reinterpret_cast<v4i *>(sx + 16 * c);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int over = (int)(first + 4 * w + 4) - (int)left;   // bytes of the word behind the end
            v[w] &= over <= 0 ? -1 : over >= 4 ? 0 : (int)(~0u >> (8 * over));
        }
        *reinterpret_cast<v4i *>(sx + 16 * c) = v;
    }
    __syncthreads();
}

// What this wave has issued has arrived but for the last LATER loads, its reads too; then all
// waves are here.
template <int LATER> __device__ __forceinline__ void tile_barrier() {
    __builtin_amdgcn_s_waitcnt((LATER & 15) | (LATER >> 4) << 14 | 0x0070);   // vmcnt LATER, lgkmcnt 0
    asm volatile("" ::: "memory");        // (no fence: it would wait for the later loads too)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

#endif

// Two buffers: tile i + 1 is loaded while tile i is multiplied. More (DMA): NS - 1 tiles are
// under way, the next one is in LDS already and its first step's reads are made ahead of the
// barrier, so that the matrix instructions go on behind it.
//
// Few tiles over a long k: block (.., p) takes bytes p k_part .. of k and leaves its sums in
// `sums` [p][rows][n]; k_linear_join adds the parts.
template <int MF, int BN, int BM, int WN, int WM, int BK, int NS, bool DMA, int YT>
__global__ __launch_bounds__(BN / WN * (BM / WM) * 64) void k_linear_tile(LinearArgs a, TileGrid tg, uint32_t k_part,
                                                                          int32_t *sums) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int THREADS = BN / WN * (BM / WM) * 64;
    constexpr bool DEEP = NS > 2;
    static_assert(DMA || !DEEP, "through registers: two buffers");
    if constexpr (YT == kSums) {
        const uint32_t from = blockIdx.y * k_part;
        a.x = static_cast<const int8_t *>(a.x) + from;
        a.w += from;
        a.k = a.k - from < k_part ? a.k - from : k_part;
    }
    // (a variable for each buffer: the compiler then knows which loads a read has to wait for)
    constexpr int SIZE = (BN + BM) * BK;
    __shared__ __attribute__((aligned(16))) int8_t s_0[SIZE], s_1[SIZE], s_2[NS > 2 ? SIZE : 16],
        s_3[NS > 3 ? SIZE : 16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane % MF,
                   part = lane / MF;
    const uint32_t wn = wave % (BN / WN) * WN, wm = wave / (BN / WN) * WM;
    uint32_t bn, bm;
    tg.place(blockIdx.x, bn, bm);
    const uint64_t n0 = (uint64_t)bn * BN, m0 = (uint64_t)bm * BM;
    WaveTile<MF, WN, WM, BK> t;
    constexpr int S = t.S;
#pragma unroll
    for (int i = 0; i < t.TN; ++i)
#pragma unroll
        for (int j = 0; j < t.TM; ++j) t.acc[i][j] = {};
    Stage<BN, BK, THREADS, DMA> lw;
    Stage<BM, BK, THREADS, DMA> lx;
    lw.init(a.w, a.ldw, n0, a.n, a.k);
    lx.init(static_cast<const int8_t *>(a.x), a.ldx, m0, a.rows, a.k);
    const uint32_t tiles = (a.k + BK - 1) / BK;
    constexpr int EACH = lw.LOADS + lx.LOADS;
    auto load = [&](uint32_t i, int8_t *to) {
        if (i >= tiles) {   // (nothing more to load: no load is under way, so that the count below holds)
            if (DMA) __builtin_amdgcn_s_waitcnt(0x0F70);
            return;
        }
        lw.load(to, wave, i * BK, a.k);
        lx.load(to + BN * BK, wave, i * BK, a.k);
    };
    auto read = [&](typename WaveTile<MF, WN, WM, BK>::Frag &to, const int8_t *from, int s) {
        t.read(to, from, from + BN * BK, wn, wm, s);
    };
    auto tail = [&](uint32_t i, int8_t *of) {
        if (i + 1 == tiles) clear_tail<BM, BK, THREADS>(of + BN * BK, a.k - i * BK);
    };
    auto multiply = [&](const int8_t *from, auto last) {   // last(f): the reads beside the last step
#pragma unroll
        for (int s = 0; s < S; ++s)
            t.step(s, [&](auto &f) {
                if (s + 1 < S) read(f, from, s + 1);
                else last(f);
            });
    };
    load(0, s_0);
    if constexpr (!DEEP) {
        lw.store(s_0);
        lx.store(s_0 + BN * BK);
        auto step = [&](uint32_t i, int8_t *from, int8_t *to) {
            tile_barrier<0>();
            tail(i, from);
            read(t.f[0], from, 0);
            load(i + 1, to);
            multiply(from, [](auto &) {});
            lw.store(to);
            lx.store(to + BN * BK);
        };
        for (uint32_t i = 0;;) {
            step(i, s_0, s_1);
            if (++i == tiles) break;
            step(i, s_1, s_0);
            if (++i == tiles) break;
        }
    } else {
        static_assert(S % 2 == 0, "a tile's first step is in f[0]");
        load(1, s_1);
        if constexpr (NS > 3) load(2, s_2);
        tile_barrier<(NS - 2) * EACH>();
        tail(0, s_0);
        read(t.f[0], s_0, 0);
        // tile i from `from`; tile i + 1 has arrived in `next`, tile i + NS - 1 goes to `to`, which
        // held tile i - 1
        auto step = [&](uint32_t i, int8_t *from, int8_t *next, int8_t *to) {
            tile_barrier<(NS - 3) * EACH>();
            tail(i + 1, next);
            load(i + NS - 1, to);
            multiply(from, [&](auto &f) { read(f, next, 0); });   // (behind the last tile: unused)
        };
        for (uint32_t i = 0;;) {
            if constexpr (NS == 3) {
                step(i, s_0, s_1, s_2);
                if (++i == tiles) break;
                step(i, s_1, s_2, s_0);
                if (++i == tiles) break;
                step(i, s_2, s_0, s_1);
                if (++i == tiles) break;
            } else {
                step(i, s_0, s_1, s_3);
                if (++i == tiles) break;
                step(i, s_1, s_2, s_0);
                if (++i == tiles) break;
                step(i, s_2, s_3, s_1);
                if (++i == tiles) break;
                step(i, s_3, s_0, s_2);
                if (++i == tiles) break;
            }
        }
    }
    if constexpr (YT == kSums) {
#pragma unroll
        for (int i = 0; i < t.TN; ++i)
#pragma unroll
            for (int j = 0; j < t.TM; ++j) {
                const uint64_t r = m0 + wm + MF * j + lr, c = n0 + wn + MF * i + 4 * part;
                if (r >= a.rows) continue;
                int32_t *to = sums + (blockIdx.y * a.rows + r) * a.n;
#pragma unroll
                for (int e = 0; e < t.E; ++e)
                    if (c + 8 * (e / 4) + e % 4 < a.n) to[c + 8 * (e / 4) + e % 4] = t.acc[i][j][e];
            }
    } else {
    using T = typename Elem<YT>::T;
    // the channels' scales and biases come through LDS
    float *s_ws = reinterpret_cast<float *>(s_0), *s_b = s_ws + BN;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < BN; c += THREADS) {
        const uint64_t cc = n0 + c < a.n ? n0 + c : a.n - 1;
        s_ws[c] = a.w_scale[cc];
        s_b[c] = a.bias ? a.bias[cc] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < t.TN; ++i) {
        const uint32_t cw = wn + MF * i + 4 * part;
        const int64_t left = (int64_t)a.n - (int64_t)(n0 + cw);   // channels from this lane's first on
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < t.TM; ++j) {
            const uint64_t r = m0 + wm + MF * j + lr;
            const float xs = a.x_scale[r < a.rows ? r : a.rows - 1];
            float v[t.E / 4][4];
#pragma unroll
            for (int e = 0; e < t.E; ++e)
                v[e / 4][e % 4] = scaled(t.acc[i][j][e], xs, s_ws[cw + 8 * (e / 4) + e % 4], s_b[cw + 8 * (e / 4) + e % 4]);
#pragma unroll
            for (int g = 0; g < t.E / 4; ++g) activate(v[g], a.act);
            if (r >= a.rows) continue;
            T *y = static_cast<T *>(a.y) + r * a.ldy + n0 + cw;
#pragma unroll
            for (int g = 0; g < t.E / 4; ++g)
                if (left > 8 * g) store4(y + 8 * g, v[g], left - 8 * g);
        }
    }
    }
#endif
}

// The parts' sums, four channels of a row a thread.
__global__ __launch_bounds__(256) void k_linear_join(LinearArgs a, int yt, uint32_t parts, const int32_t *sums) {
    const uint32_t per = (a.n + 3) / 4;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < a.rows * per; i += gridDim.x * 256ull) {
        const uint64_t r = i / per;
        const uint32_t c = (uint32_t)(i - r * per) * 4;
        v4i sum = {0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t p = 0; p < parts; ++p) {
            const int32_t *from = sums + (p * a.rows + r) * a.n + c;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += from[c + e < a.n ? e : 0];
        }
        put_sums(a, yt, sum, a.x_scale[r], r, c);
    }
}

// Rows that the DMA cannot bring into rows that it can, 16 bytes a thread; 0 behind their ends.
__global__ __launch_bounds__(256) void k_pack_rows(const int8_t *p, uint64_t ld, uint64_t rows, uint32_t k, int8_t *to) {
    const uint32_t per = (k + 15) / 16;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < rows * per; i += gridDim.x * 256ull) {
        const uint64_t r = i / per;
        const uint32_t c = (uint32_t)(i - r * per) * 16;
        *reinterpret_cast<v4i *>(to + 16 * i) = load16(p + r * ld + c, (int64_t)k - c);
    }
}

template <int MF, int BN, int BM, int WN, int WM, int BK, int NS, bool DMA>
static void linear_tile(const LinearArgs &a, int yt, hipStream_t st) {
    const TileGrid tg((a.n + BN - 1) / BN, (a.rows + BM - 1) / BM);
    constexpr int threads = BN / WN * (BM / WM) * 64;
    auto go = [&](auto kernel) { kernel<<<tg.tiles, threads, 0, st>>>(a, tg, a.k, nullptr); };
    if (yt == FSX_DTYPE_F32) go(k_linear_tile<MF, BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_F32>);
    else if (yt == FSX_DTYPE_F16) go(k_linear_tile<MF, BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_F16>);
    else go(k_linear_tile<MF, BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_BF16>);
}

// Operands that the DMA can bring: chunks at 16-byte addresses, a tile's rows within 2^31 bytes.
static bool dma_can(const void *p, uint64_t ld) { return ((uintptr_t)p | ld) % 16 == 0 && ld < (1u << 23); }

// How a product goes, by its sizes, x's type and whether the DMA can bring x and the weights.
//
// kNarrow: fsx_narrow.hip. kFewFloats, kFew: k_linear_few, for codes up to 32 rows (us at 16 / 32
// rows of 4096 to 4096 channels: 6.7 / 8.7, in tiles 9.8 / 10.8; to 16384 channels 20.7 / 28, in
// tiles 14.9 / 15.5, since those fill the CUs).
// kTiles: k_linear_tile. With few tiles over a long k in parts: enough blocks for the CUs, each
// with 1024 of k at least (223 rows of 3777 to 14 channels 23.8 -> 12.4 us). With many, operands
// that the DMA cannot bring are packed first (4096 rows of 4096 to 4096 channels at odd strides:
// 155 us through registers).
enum LinearForm { kNarrow, kFewFloats, kFew, kTiles };
struct LinearPlan {
    LinearForm form;
    uint32_t parts = 1, k_part = 0;
    bool pack_x = false, pack_w = false;
    uint64_t codes = 0, x_bytes = 0, w_bytes = 0, sums = 0;   // of the workspace, in this order
    uint64_t bytes() const { return codes + x_bytes + w_bytes + sums; }

    LinearPlan(uint64_t rows, uint32_t k, uint32_t n, int x_dtype, bool x_fits, bool w_fits) {
        const bool floats = x_dtype != FSX_DTYPE_I8;
        auto tiles = [&](uint64_t size) { return (n + size - 1) / size * ((rows + size - 1) / size); };
        if (k <= 64) form = kNarrow;
        else if (floats && rows <= kFusedRows && rows * ((k + 63) / 64 * 64 + 16) <= kFusedBytes) form = kFewFloats;
        else if ((rows <= 16 && n < 16384 && (k < 16384 || n >= 2048)) || (rows <= 32 && n < 8192 && k < 8192))
            form = kFew;
        else form = kTiles;
        if (floats && (form == kFew || form == kTiles)) codes = code_space(rows, k).bytes;
        if (form != kTiles) return;
        if (tiles(64) < 128 && k >= 2048) {
            const uint32_t want = (uint32_t)std::min<uint64_t>({256 / tiles(64), k / 1024, 64});
            k_part = ((k + want - 1) / want + 255) / 256 * 256;
            parts = (k + k_part - 1) / k_part;
            if (parts > 1) sums = up16(parts * rows * n * 4);
        } else if (tiles(128) >= 256) {
            pack_x = !floats && !x_fits;
            pack_w = !w_fits;
            if (pack_x) x_bytes = rows * up16(k);
            if (pack_w) w_bytes = n * up16(k);
        }
    }
};

// Large tiles read least for each product; with fewer of them than the CUs, smaller ones. us at
// 512 / 1024 / 2048 / 4096 rows of 4096 to 4096 channels:
//                      256 x 256     54    55    57    70    (8192 cubed: 507)
//   128 x 128, two buffers           26    28    37    71-77 (572)
//   128 x 128, four buffers          23    25    55    95    (one block a CU)
//    64 x 64                         16    33    64   119    (909)
// Eight waves a block in each: four waves of twice the size were 12 - 60 % slower, since a wave
// by itself issues an instruction in 8 cycles.
static void linear_tiles(const LinearArgs &a, int yt, const LinearPlan &ks, void *sums_at, hipStream_t st) {
    if (ks.parts > 1) {
        const TileGrid tg((a.n + 63) / 64, (a.rows + 63) / 64);
        const dim3 grid(tg.tiles, ks.parts);
        int32_t *sums = static_cast<int32_t *>(sums_at);
        if (dma_can(a.x, a.ldx) && dma_can(a.w, a.ldw))
            k_linear_tile<16, 64, 64, 32, 16, 256, 2, true, kSums><<<grid, 512, 0, st>>>(a, tg, ks.k_part, sums);
        else k_linear_tile<16, 64, 64, 32, 16, 128, 2, false, kSums><<<grid, 512, 0, st>>>(a, tg, ks.k_part, sums);
        const uint64_t blocks = (a.rows * ((a.n + 3) / 4) + 255) / 256;
        k_linear_join<<<(uint32_t)std::min<uint64_t>(blocks, 4096), 256, 0, st>>>(a, yt, ks.parts, sums);
        return;
    }
    auto tiles = [&](uint64_t size) { return (a.n + size - 1) / size * ((a.rows + size - 1) / size); };
    if (dma_can(a.x, a.ldx) && dma_can(a.w, a.ldw)) {
        if (tiles(256) >= 256) linear_tile<16, 256, 256, 128, 64, 128, 2, true>(a, yt, st);
        else if (tiles(128) >= 320) linear_tile<16, 128, 128, 64, 32, 128, 2, true>(a, yt, st);
        else if (tiles(128) >= 192) linear_tile<16, 128, 128, 64, 32, 128, 4, true>(a, yt, st);
        else linear_tile<16, 64, 64, 32, 16, 256, 2, true>(a, yt, st);
    } else linear_tile<16, 64, 64, 32, 16, 128, 2, false>(a, yt, st);
}

// A grid holds fewer than 2^32 threads: a product beyond 2^20 channels, or of more results than
// 2^38, goes out in several launches.
template <typename F>
static void slabs(const LinearArgs &a, int y_dtype, uint32_t x_size, F launch) {
    const uint64_t most_n = 1ull << 20;
    for (uint64_t n0 = 0; n0 < a.n; n0 += most_n) {
        const uint64_t n = std::min<uint64_t>(a.n - n0, most_n);
        const uint64_t most_m = (1ull << 38) / std::max<uint64_t>(n, 1024);
        for (uint64_t m0 = 0; m0 < a.rows; m0 += most_m) {
            LinearArgs b = a;
            b.n = (uint32_t)n;
            b.rows = std::min<uint64_t>(a.rows - m0, most_m);
            b.x = static_cast<const char *>(a.x) + m0 * a.ldx * x_size;
            if (a.x_scale) b.x_scale = a.x_scale + m0;
            b.w = a.w + n0 * a.ldw;
            b.w_scale = a.w_scale + n0;
            if (a.bias) b.bias = a.bias + n0;
            b.y = static_cast<char *>(a.y) + (m0 * a.ldy + n0) * elem_size(y_dtype);
            launch(b);
        }
    }
}

// What a call needs; without a pointer: as if those rows were at odd strides.
uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype, const void *x, uint64_t ldx, const void *w,
                     uint64_t ldw) {
    return LinearPlan(rows, k, n, x_dtype, x && dma_can(x, ldx), w && dma_can(w, ldw)).bytes();
}

static void pack_rows(const int8_t *p, uint64_t ld, uint64_t rows, uint32_t k, int8_t *to, hipStream_t st) {
    const uint64_t blocks = (rows * ((k + 15) / 16) + 255) / 256;
    k_pack_rows<<<(uint32_t)std::min<uint64_t>(blocks, 8192), 256, 0, st>>>(p, ld, rows, k, to);
}

hipError_t launch_linear(const LinearArgs &in, int x_dtype, int y_dtype, void *work, hipStream_t st) {
    (void)hipGetLastError();
    if (in.rows == 0 || in.n == 0) return hipSuccess;
    LinearArgs a = in;
    const LinearPlan p(a.rows, a.k, a.n, x_dtype, dma_can(a.x, a.ldx), dma_can(a.w, a.ldw));
    if (x_dtype != FSX_DTYPE_I8 && (p.form == kNarrow || p.form == kFewFloats)) {
        slabs(a, y_dtype, elem_size(x_dtype), [&](const LinearArgs &b) {
            if (p.form == kNarrow) launch_linear_narrow(b, x_dtype, y_dtype, st);
            else if (x_dtype == FSX_DTYPE_F32) linear_few<FSX_DTYPE_F32>(b, y_dtype, st);
            else if (x_dtype == FSX_DTYPE_F16) linear_few<FSX_DTYPE_F16>(b, y_dtype, st);
            else linear_few<FSX_DTYPE_BF16>(b, y_dtype, st);
        });
        return hipGetLastError();
    }
    int8_t *at = static_cast<int8_t *>(work);
    if (x_dtype != FSX_DTYPE_I8) {
        const CodeSpace s = code_space(a.rows, a.k);
        float *sc = reinterpret_cast<float *>(at + s.scale_at);
        const hipError_t e = launch_quantize_rows(a.x, x_dtype, a.rows, a.k, a.ldx, at, s.ld, sc, st);
        if (e != hipSuccess) return e;
        a.x = at;
        a.x_scale = sc;
        a.ldx = s.ld;
        at += p.codes;
    }
    if (p.pack_x) {
        pack_rows(static_cast<const int8_t *>(a.x), a.ldx, a.rows, a.k, at, st);
        a.x = at;
        a.ldx = up16(a.k);
        at += p.x_bytes;
    }
    if (p.pack_w) {
        pack_rows(a.w, a.ldw, a.n, a.k, at, st);
        a.w = at;
        a.ldw = up16(a.k);
        at += p.w_bytes;
    }
    slabs(a, y_dtype, 1, [&](const LinearArgs &b) {
        if (p.form == kNarrow) launch_linear_narrow(b, FSX_DTYPE_I8, y_dtype, st);
        else if (p.form == kFew) linear_few<FSX_DTYPE_I8>(b, y_dtype, st);
        else linear_tiles(b, y_dtype, p, at, st);   // (in parts: small enough for one launch)
    });
    return hipGetLastError();
}

}  // namespace fsx
