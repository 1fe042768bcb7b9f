// fsx_linear.hip — int8 layers of free size (include/fsx_hip.h fsx_linear_q8_device): the int8
// matrix product with a scale for every row of x and every output channel,
//
//   y_rn = act((float)(sum_k q_rk w_nk) * scale_r * t_n + b_n)
//
// and which kernel takes it. Floats become codes q as fsx_quantize.hip makes them.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <type_traits>

#include "fsx_q8_rows.h"

namespace fsx {

constexpr int kSums = -1;   // results that are sums still

// ---------------------------------------------------------------- int8 product

// ---- few rows or few channels: the longer side's bytes bound it
//
// The longer side is the rows of x (TALL) or the channels; the other one has up to 32, MT groups
// of 16. A block takes 16 of the longer side for each `kw` of its FW waves, which share its k 128
// bytes (whole lines) in turn, straight from memory into v_mfma_i32_16x16x64_i8, the weights
// first: lane l gives bytes 16 (l / 16) .. of row l % 16 of either operand and holds channels
// 4 (l / 16) .. of row l % 16 of the result. The waves' sums meet in LDS. Few blocks over a long
// k: block (.., p) takes bytes p k_part .. of k, and k_linear_join adds the parts.
//
// FLOATS: a block quantises its rows of x into LDS, in one launch with the product: all rows if
// they are few (every block does, while its first weights are under way; x is small and comes
// from cache), else (TALL) its own.
constexpr uint32_t kDirectMost = 32, kFusedRows = 4, kFusedBytes = 32768, kTallBytes = 49152;

template <int XT, int MT, int FW, bool TALL, bool ODD>
__global__ __launch_bounds__(64 * FW) void k_linear_direct(LinearArgs a, int yt, uint32_t kw, uint32_t k_part,
                                                           int32_t *sums) {
    constexpr bool FLOATS = XT != FSX_DTYPE_I8;
    constexpr uint32_t THREADS = 64 * FW;
    constexpr int U = MT == 1 && !TALL ? 8 : 4;   // loads of the longer side in flight a lane
    extern __shared__ __attribute__((aligned(16))) int8_t s_x[];   // FLOATS: the rows' codes, up64(k) + 16 apart
    __shared__ __attribute__((aligned(16))) v4i s_acc[FW][MT][64];
    __shared__ uint32_t s_max[TALL ? 16 * FW : kFusedRows];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15,
                   lq = lane >> 4;
    const uint32_t groups = FW / kw, wk = wave % kw, group = wave / kw;   // (kw divides FW)
    const uint64_t longer = TALL ? a.rows : a.n, shorter = TALL ? a.n : a.rows;
    const uint64_t l0 = (uint64_t)blockIdx.x * groups * 16;   // the block's first
    const uint32_t from = blockIdx.y * k_part, end = a.k - from < k_part ? a.k : from + k_part;
    const uint32_t chunks = (a.k + 63) / 64, pitch = chunks * 64 + 16;
    const uint64_t mine = l0 + 16 * group + lr, l = mine < longer ? mine : longer - 1;
    const int8_t *xc = static_cast<const int8_t *>(a.x);   // (codes)
    const int8_t *pl = (TALL ? xc + (FLOATS ? 0 : l * a.ldx) : a.w + l * a.ldw) + 16 * lq;
    const int8_t *ps[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const uint64_t r = 16 * m + lr, rr = r < shorter ? r : shorter - 1;
        ps[m] = (TALL ? a.w + rr * a.ldw : xc + (FLOATS ? 0 : rr * a.ldx)) + 16 * lq;
    }
    // The wave's u-th block of round t, of `whole` blocks of 64 bytes and then a rest.
    const uint32_t whole = (end - from) / 64;
    auto block = [&](uint32_t t, int u) { return 2 * (wk + kw * (t * (U / 2) + u / 2)) + u % 2; };
    auto place = [&](uint32_t i) { return from + i * 64; };
    auto code = [&](uint32_t r, uint32_t k0) {   // FLOATS: of row r in LDS
        return *reinterpret_cast<const v4i *>(s_x + r * pitch + k0 + 16 * lq);
    };
    auto lds_row = [&](int m) -> uint32_t {
        const uint32_t r = 16 * m + lr;
        return TALL ? 16 * group + lr : r < a.rows ? r : (uint32_t)a.rows - 1;
    };
    constexpr bool AHEAD = !(FLOATS && TALL);   // (those come from LDS)
    v4i v[U];
    auto longs = [&](uint32_t t) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (block(t, u) < whole)
                v[u] = AHEAD ? load16_at(pl + place(block(t, u)), ODD) : code(lds_row(0), place(block(t, u)));
    };
    if (AHEAD && block(0, 0) < whole) longs(0);
    if constexpr (FLOATS) {
        const uint64_t r0 = TALL ? l0 : 0;
        const uint32_t most = TALL ? groups * 16 : (uint32_t)a.rows;
        const uint32_t rows = a.rows - r0 < most ? (uint32_t)(a.rows - r0) : most;
        const auto *x = static_cast<const typename Elem<XT>::T *>(a.x) + r0 * a.ldx;
        const uint32_t per = chunks * 4, all = rows * per;   // chunks of 16, zeros behind the end
        for (uint32_t i = threadIdx.x; i < most; i += THREADS) s_max[i] = 0;
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
            const uint32_t r1 = __builtin_amdgcn_readfirstlane(r);
            if (__ballot(some && r != r1) == 0) {
                m = group_all<64>(m, LargerWord());
                if (lane == 0) atomicMax(&s_max[r1], m);
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
    auto multiply = [&](int m, const v4i &of_long, const v4i &of_short) {
        acc[m] = TALL ? __builtin_amdgcn_mfma_i32_16x16x64_i8(of_short, of_long, acc[m], 0, 0, 0)
                      : __builtin_amdgcn_mfma_i32_16x16x64_i8(of_long, of_short, acc[m], 0, 0, 0);
    };
#pragma unroll 1
    for (uint32_t t = 0; block(t, 0) < whole; ++t) {
        if (!AHEAD) longs(t);
        v4i w[MT][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (block(t, u) >= whole) continue;
#pragma unroll
            for (int m = 0; m < MT; ++m)
                w[m][u] = FLOATS && !TALL ? code(lds_row(m), place(block(t, u)))
                                          : load16_at(ps[m] + place(block(t, u)), ODD);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (block(t, u) >= whole) continue;
#pragma unroll
            for (int m = 0; m < MT; ++m) multiply(m, v[u], w[m][u]);
        }
        if (AHEAD && block(t + 1, 0) < whole) longs(t + 1);
    }
    if (end % 64 && wk == whole / 2 % kw) {   // the rest, by the wave whose turn it is (`from` is a multiple of 64)
        const uint32_t k0 = from + whole * 64;
        const int ok = (int)(end - k0) - (int)(16 * lq);
        const v4i rest = AHEAD ? load16_end(pl + k0, ok) : code(lds_row(0), k0);
#pragma unroll
        for (int m = 0; m < MT; ++m)
            multiply(m, rest, FLOATS && !TALL ? code(lds_row(m), k0) : load16_end(ps[m] + k0, ok));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) s_acc[wave][m][lane] = acc[m];
    __syncthreads();
    for (uint32_t i = wave; i < groups * MT; i += FW) {
        const uint32_t g = i / MT, m = i % MT;
        v4i sum = s_acc[g * kw][m][lane];
        if (kw == FW) {   // (all reads at once)
#pragma unroll
            for (int q = 1; q < FW; ++q) sum += s_acc[q][m][lane];
        } else {
            for (uint32_t q = 1; q < kw; ++q) sum += s_acc[g * kw + q][m][lane];
        }
        const uint64_t r = (TALL ? l0 + 16 * g : 16 * m) + lr, c = (TALL ? 16 * m : l0 + 16 * g) + 4 * lq;
        if (r >= a.rows) continue;
        if (!FLOATS && sums) {
            int32_t *to = sums + (blockIdx.y * a.rows + r) * a.n + c;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.n) to[e] = sum[e];
            continue;
        }
        float xs;
        if constexpr (FLOATS) xs = row_scale(mag_value<XT>(s_max[TALL ? 16 * g + lr : r]));
        else xs = a.x_scale[r];
        put_sums(a, yt, sum, xs, r, c);
    }
}

// The shape of such a product's launch.
struct DirectGrid {
    bool tall;
    uint32_t waves, kw;
    uint64_t blocks;   // (of all rows; a launch has few enough for a grid)
    static uint64_t pitch(uint32_t k) { return (k + 63) / 64 * 64 + 16; }
    // (the whole product's side: a launch of a part of its rows may hold fewer of them)
    static bool tall_of(uint64_t rows, uint32_t n, bool floats) { return n <= rows && !(floats && rows <= kFusedRows); }
    DirectGrid(uint64_t rows, uint32_t k, uint32_t n, bool floats, bool tall) : tall(tall) {
        const uint64_t sixteens = ((tall ? rows : n) + 15) / 16;
        // us of one row, 4096 / 8192 / 16384 channels of 4096: eight waves 6.4 / 9.1 / 16.8, sixteen
        // 5.9 / 10.9 / 20.0
        waves = sixteens >= 512 ? 8 : 16;
        // (256 bytes of k a wave at least, if the blocks are enough without the others)
        kw = waves;
        while (kw > 1 && k < 256 * kw && sixteens * kw / waves >= 512 &&
               !(floats && tall && waves / kw * 2 * 16 * pitch(k) > kFusedBytes))
            kw /= 2;
        blocks = (sixteens * kw + waves - 1) / waves;
    }
    uint64_t codes_bytes(uint64_t rows, uint32_t k) const { return pitch(k) * (tall ? waves / kw * 16 : rows); }
};
template <int XT, int MT, bool TALL>
static void linear_direct(const LinearArgs &a, const DirectGrid &d, uint32_t lds, uint32_t parts, uint32_t k_part,
                          int32_t *sums, int yt, hipStream_t st) {
    const bool odd = (((uintptr_t)a.w | a.ldw) & 3) || (XT == FSX_DTYPE_I8 && (((uintptr_t)a.x | a.ldx) & 3));
    auto go = [&](auto kernel) {
        kernel<<<dim3((uint32_t)d.blocks, parts), 64 * d.waves, lds, st>>>(a, yt, d.kw, k_part, sums);
    };
    if (d.waves == 8) odd ? go(k_linear_direct<XT, MT, 8, TALL, true>) : go(k_linear_direct<XT, MT, 8, TALL, false>);
    else odd ? go(k_linear_direct<XT, MT, 16, TALL, true>) : go(k_linear_direct<XT, MT, 16, TALL, false>);
}
template <int XT>
static void linear_direct(const LinearArgs &a, bool tall, uint32_t parts, uint32_t k_part, int32_t *sums, int yt,
                          hipStream_t st) {
    constexpr bool FLOATS = XT != FSX_DTYPE_I8;
    const DirectGrid d(a.rows, a.k, a.n, FLOATS, tall);
    const uint32_t groups = (uint32_t)(((d.tall ? a.n : a.rows) + 15) / 16);
    const uint32_t lds = FLOATS ? (uint32_t)d.codes_bytes(a.rows, a.k) : 0;
    auto go = [&](auto mt, auto tall) {
        linear_direct<XT, mt, tall>(a, d, lds, parts, k_part, sums, yt, st);
    };
    using std::integral_constant;
    if (d.tall) {
        if (groups == 1) go(integral_constant<int, 1>(), std::true_type());
        else go(integral_constant<int, 2>(), std::true_type());
    } else if constexpr (FLOATS) {
        go(integral_constant<int, 1>(), std::false_type());
    } else {
        if (groups == 1) go(integral_constant<int, 1>(), std::false_type());
        else go(integral_constant<int, 2>(), std::false_type());
    }
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
// The weights are the first operand of v_mfma_i32_16x16x64_i8 and x the second, as above: a lane
// holds four neighbouring channels of one row.
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
    bool odd;                // strides that are no multiple of 4
    v4i reg[DMA ? 1 : LOADS];
    // chunk i of this thread: row i STEP + threadIdx / PER, place threadIdx % PER. Rows behind
    // the last: the last one, its results are not stored.
    __device__ __forceinline__ void init(const int8_t *p, uint64_t ld, uint64_t r0, uint64_t rows,
                                         uint32_t k) {
        const uint32_t tr = threadIdx.x / PER, pos = threadIdx.x % PER;
        at = 16 * (pos ^ place_key<BK>(tr));
        base = p + r0 * ld;
        odd = (((uintptr_t)p | ld) & 3) != 0;
        const uint32_t last = (uint32_t)(rows - r0 < ROWS ? rows - r0 : ROWS) - 1;
        // raw buffer, 32-bit data; it ends with the chunk that the last row's end lies in
        if (DMA)
            buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(base), 0,
                                                    last * (uint32_t)ld + ((k + 15) & ~15u), 0x00020000);
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
            for (int i = 0; i < LOADS; ++i) {
                const int8_t *p = base + row[i] + k0 + at;
                reg[i] = k0 + BK <= k ? load16_at(p, odd) : load16_end(p, (int)(k - k0) - (int)at);
            }
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) {
        if (!DMA)
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                *reinterpret_cast<v4i *>(lds + (i * THREADS + threadIdx.x) * 16) = reg[i];
    }
};

template <int WN, int WM, int BK>
struct WaveTile {
    static constexpr int TN = WN / 16, TM = WM / 16, S = BK / 64;
    v4i acc[TN][TM];
    struct Frag { v4i w[TN], x[TM]; };
    Frag f[2];
    __device__ __forceinline__ void read(Frag &to, const int8_t *sw, const int8_t *sx, uint32_t wn, uint32_t wm,
                                         int s) {
        const uint32_t lane = __lane_id(), lr = lane % 16, at = ((4 * s + lane / 16) ^ place_key<BK>(lr)) * 16;
#pragma unroll
        for (int i = 0; i < TN; ++i) to.w[i] = *reinterpret_cast<const v4i *>(sw + (wn + 16 * i + lr) * BK + at);
#pragma unroll
        for (int j = 0; j < TM; ++j) to.x[j] = *reinterpret_cast<const v4i *>(sx + (wm + 16 * j + lr) * BK + at);
    }
    // Step s of a tile from f[s & 1], the next step's reads under way meanwhile.
    template <typename F> __device__ __forceinline__ void step(int s, F next) {
        __builtin_amdgcn_sched_barrier(0);
        next(f[(s + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[s & 1].w[i], f[s & 1].x[j], acc[i][j], 0, 0, 0);
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

// Two buffers: tile i + 1 is loaded while tile i is multiplied. Four (DMA): three tiles are
// under way, the next one is in LDS already and its first step's reads are made ahead of the
// barrier, so that the matrix instructions go on behind it.
//
// Few tiles over a long k: block (.., p) takes bytes p k_part .. of k and leaves its sums in
// `sums` [p][rows][n]; k_linear_join adds the parts.
template <int BN, int BM, int WN, int WM, int BK, int NS, bool DMA, int YT>
__global__ __launch_bounds__(BN / WN * (BM / WM) * 64) void k_linear_tile(LinearArgs a, TileGrid tg, uint32_t k_part,
                                                                          int32_t *sums) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int THREADS = BN / WN * (BM / WM) * 64;
    constexpr bool DEEP = NS == 4;
    static_assert(NS == 2 || (DEEP && DMA), "two buffers, or four by DMA");
    if constexpr (YT == kSums) {
        const uint32_t from = blockIdx.y * k_part;
        a.x = static_cast<const int8_t *>(a.x) + from;
        a.w += from;
        a.k = a.k - from < k_part ? a.k - from : k_part;
    }
    // (a variable for each buffer: the compiler then knows which loads a read has to wait for)
    constexpr int SIZE = (BN + BM) * BK;
    __shared__ __attribute__((aligned(16))) int8_t s_0[SIZE], s_1[SIZE], s_2[DEEP ? SIZE : 16],
        s_3[DEEP ? SIZE : 16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane % 16,
                   part = lane / 16;
    const uint32_t wn = wave % (BN / WN) * WN, wm = wave / (BN / WN) * WM;
    uint32_t bn, bm;
    tg.place(blockIdx.x, bn, bm);
    const uint64_t n0 = (uint64_t)bn * BN, m0 = (uint64_t)bm * BM;
    WaveTile<WN, WM, BK> t;
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
    auto read = [&](typename WaveTile<WN, WM, BK>::Frag &to, const int8_t *from, int s) {
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
        load(2, s_2);
        tile_barrier<2 * EACH>();
        tail(0, s_0);
        read(t.f[0], s_0, 0);
        // tile i from `from`; tile i + 1 has arrived in `next`, tile i + 3 goes to `to`, which
        // held tile i - 1
        auto step = [&](uint32_t i, int8_t *from, int8_t *next, int8_t *to) {
            tile_barrier<EACH>();
            tail(i + 1, next);
            load(i + 3, to);
            multiply(from, [&](auto &f) { read(f, next, 0); });   // (behind the last tile: unused)
        };
        for (uint32_t i = 0;;) {
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
    if constexpr (YT == kSums) {
#pragma unroll
        for (int i = 0; i < t.TN; ++i)
#pragma unroll
            for (int j = 0; j < t.TM; ++j) {
                const uint64_t r = m0 + wm + 16 * j + lr, c = n0 + wn + 16 * i + 4 * part;
                if (r >= a.rows) continue;
                int32_t *to = sums + (blockIdx.y * a.rows + r) * a.n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.n) to[c + e] = t.acc[i][j][e];
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
            const uint32_t cw = wn + 16 * i + 4 * part;
            const int64_t left = (int64_t)a.n - (int64_t)(n0 + cw);   // channels from this lane's first on
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < t.TM; ++j) {
                const uint64_t r = m0 + wm + 16 * j + lr;
                const float xs = a.x_scale[r < a.rows ? r : a.rows - 1];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = scaled(t.acc[i][j][e], xs, s_ws[cw + e], s_b[cw + e]);
                activate(v, a.act);
                if (r < a.rows && left > 0) store4(static_cast<T *>(a.y) + r * a.ldy + n0 + cw, v, left);
            }
        }
    }
#endif
}

// The parts' sums, four channels of a row a thread.
__global__ __launch_bounds__(256) void k_linear_join(LinearArgs a, int yt, uint32_t parts, const int32_t *sums) {
    const uint32_t per = (a.n + 3) / 4;
    const uint64_t i = blockIdx.x * 256ull + threadIdx.x, r = i / per;
    if (r >= a.rows) return;
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

static void join_parts(const LinearArgs &a, int yt, uint32_t parts, const int32_t *sums, hipStream_t st) {
    const uint64_t blocks = (a.rows * ((a.n + 3) / 4) + 255) / 256;   // (products in parts: a few thousand at most)
    k_linear_join<<<(uint32_t)blocks, 256, 0, st>>>(a, yt, parts, sums);
}

// Rows that the DMA cannot bring into rows that it can, 16 bytes a thread; 0 behind their ends.
__global__ __launch_bounds__(256) void k_pack_rows(const int8_t *p, uint64_t ld, uint64_t rows, uint32_t k,
                                                   int8_t *to) {
    const uint32_t per = (k + 15) / 16;
    const bool odd = (((uintptr_t)p | ld) & 3) != 0;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < rows * per; i += gridDim.x * 256ull) {
        const uint64_t r = i / per;
        const uint32_t c = (uint32_t)(i - r * per) * 16;
        const int8_t *from = p + r * ld + c;
        *reinterpret_cast<v4i *>(to + 16 * i) = c + 16 <= k ? load16_at(from, odd) : load16_end(from, (int)(k - c));
    }
}

template <int BN, int BM, int WN, int WM, int BK, int NS, bool DMA>
static void linear_tile(const LinearArgs &a, int yt, hipStream_t st) {
    const TileGrid tg((a.n + BN - 1) / BN, (a.rows + BM - 1) / BM);
    constexpr int threads = BN / WN * (BM / WM) * 64;
    auto go = [&](auto kernel) { kernel<<<tg.tiles, threads, 0, st>>>(a, tg, a.k, nullptr); };
    if (yt == FSX_DTYPE_F32) go(k_linear_tile<BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_F32>);
    else if (yt == FSX_DTYPE_F16) go(k_linear_tile<BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_F16>);
    else go(k_linear_tile<BN, BM, WN, WM, BK, NS, DMA, FSX_DTYPE_BF16>);
}

// Operands that the DMA can bring: chunks at 16-byte addresses, a tile's rows within 2^31 bytes.
static bool dma_can(const void *p, uint64_t ld) { return ((uintptr_t)p | ld) % 16 == 0 && ld < (1u << 23); }

// How a product goes, by its sizes, x's type and whether the DMA can bring x and the weights.
//
// kNarrow: fsx_narrow.hip. kDirectFloats, kDirect: k_linear_direct, up to 32 rows or channels. It
// takes the shorter side's bytes once for every 16 of the longer one, so large weights are better
// in tiles, that fill the CUs then (us at 1 / 16 / 32 rows of 4096, direct and in tiles: 4096
// channels 6.0 / 7.2 / 9.5 and 9.5 / 9.8 / 10.8, 16384 channels 17.1 / 20.5 / 27.6 and 14.8 / 14.9 /
// 15.5; weights at odd strides, which tiles take through registers, to 16384 channels 19.5 / 29.6
// and 28.2 / 28.4). Few channels, 2^20 rows of 1024 to 16: 277, in tiles 317.
// kTiles: k_linear_tile.
//
// Few blocks over a long k are cut into parts; the join is another launch (us of codes, whole and
// in parts).
//   Tiles by DMA: 40 rows of 4096 / 8192 / 32768 to 64 channels 8.9 / 14.9 / 78 and 8.5 / 11.1 / 27, 300
//     rows of 8192 / 16384 to 1024 23 / 41 and 18 / 21, but of 2048 / 4096 6.4 / 13.0 and 13.7 / 16.9:
//     with some 80 tiles and more the rule cuts before it pays. 128 tiles and more are not cut (603 rows of
//     3984 to 1394 15.5 and 19.1).
//   Tiles through registers: 100 rows of 1024 / 2048 / 4096 to 500 8.1 / 13.2 / 23.6 and 9.4 / 10.2 /
//     11.8; up to 256 tiles from 4096 on: 107 rows of 6581 to 6892 56 and 38, 900 of 4096 / 8192 to 900
//     24.8 / 37.5 and 28.4 / 34.3.
//   Direct, by the bytes that a block takes (400000: up to 16 rows a k of 12500, up to 32 of 8334, half of
//     it at odd strides): to 1024 channels one row of 4096 / 8192 / 12544 4.8 / 7.7 / 10.5 and 8.2 / 7.5 /
//     8.4, 14 rows of 4096 / 8192 / 12544 6.0 / 9.3 / 12.8 and 7.1 / 8.3 / 9.6, 30 rows of 4096 / 8448
//     7.7 / 13.1 and 8.2 / 9.8, 14 rows at odd strides of 4096 / 6300 7.7 / 10.2 and 7.8 / 8.7; 1000 rows
//     of 8192 / 12544 to 12 9.0 / 12.5 and 8.3 / 9.7.
// Operands that the DMA cannot bring are packed for it where the work repays the copy (us, as they
// are and packed): 4096 rows of 4096 to 4096 channels at odd strides 182 and 78, 1006 rows of 8444 to
// 2643 104 and 64; odd weights and bf16 rows of 4096 to 4096, 128 / 200 / 300 / 384 / 512 / 768 rows 24.5 /
// 34.3 / 37.3 / 38.0 / 38.9 / 43.2 and 28.7 / 29.9 / 32.3 / 32.0 / 31.1 / 37.3; odd codes of 4096 rows, 128 /
// 384 / 512 / 768 channels 19.5 / 27.0 / 27.4 / 32.8 and 25.0 / 26.1 / 25.4 / 35.3. About the least work packed it
// goes by k: 700 rows of 2000 to 2000 24.0 and 22.2, 2000 of 1000 to 2000 20.8 and 21.7, 1000 of 1003 to 2500
// 17.4 and 20.8 (both odd, codes: 11.0 and 18.4).
enum LinearForm { kNarrow, kDirectFloats, kDirect, kTiles };
struct LinearPlan {
    LinearForm form;
    uint32_t parts = 1, k_part;
    bool tall = false, pack_x = false, pack_w = false;
    uint64_t codes = 0, x_bytes = 0, w_bytes = 0, sums = 0;   // of the workspace, in this order
    uint64_t bytes() const { return codes + x_bytes + w_bytes + sums; }

    LinearPlan(uint64_t rows, uint32_t k, uint32_t n, int x_dtype, bool x_fits, bool w_fits) : k_part(k) {
        const bool floats = x_dtype != FSX_DTYPE_I8;
        auto cut = [&](uint64_t blocks, uint32_t enough, uint32_t least) {
            const uint32_t want = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({enough / blocks, k / least, 64}));
            k_part = ((k + want - 1) / want + 255) / 256 * 256;
            parts = (k + k_part - 1) / k_part;
            if (parts > 1) sums = up16(parts * rows * n * 4);
            else k_part = k;
        };
        if (k <= 64) {
            form = kNarrow;
            return;
        }
        if (floats) {
            const DirectGrid d(rows, k, n, true, DirectGrid::tall_of(rows, n, true));
            const uint64_t lds = d.codes_bytes(rows, k);
            tall = d.tall;
            if (d.tall ? n <= kDirectMost && lds <= kTallBytes : rows <= kFusedRows && lds <= kFusedBytes) {
                form = kDirectFloats;
                return;
            }
            codes = code_space(rows, k).bytes;
            x_fits = true;   // (what the quantiser leaves)
        }
        const DirectGrid d(rows, k, n, false, DirectGrid::tall_of(rows, n, false));
        tall = d.tall;
        const uint64_t shorter = d.tall ? n : rows, weights = (uint64_t)n * k;
        if (shorter <= kDirectMost && (d.tall || (shorter <= 16 ? weights < 1u << 26 || !w_fits : weights < 1u << 25))) {
            form = kDirect;
            const uint64_t taken = (shorter <= 16 ? 32 : 48) * (uint64_t)k * (x_fits && w_fits ? 1 : 2);
            if (d.blocks <= 128 && taken >= 400000) cut(d.blocks, 256, 1024);
            return;
        }
        form = kTiles;
        if ((double)rows * n * k >= 2.5e9 && (w_fits || rows >= 384) && (x_fits || n >= 384)) {
            pack_x = !x_fits;
            pack_w = !w_fits;
            if (pack_x) x_bytes = rows * up16(k);
            if (pack_w) w_bytes = n * up16(k);
        }
        const uint64_t tiles = (n + 63ull) / 64 * ((rows + 63) / 64);
        const bool dma = (x_fits || pack_x) && (w_fits || pack_w);
        if (tiles < 128 ? k >= (dma ? 2048 : 1024) : !dma && tiles < 256 && k >= 4096) cut(tiles, 512, 512);
    }
};

// Large tiles read least for each product; with fewer of them than the CUs, smaller ones, of which
// several share a CU: then also some load or store while others multiply. us at 512 / 1024 / 2048 /
// 4096 rows of 4096 to 4096 channels:
//                      256 x 256     54    55    57    70    (8192 cubed: 507)
//   128 x 128, two buffers           26    28    37    71-77 (572)
//   128 x 128, four buffers          23    25    55    95    (one block a CU)
//    64 x 64                         16    33    64   119    (909)
// Between, at 640 / 768 / 896 / 1152 rows (160 / 192 / 224 / 288 tiles of 128), 128 x 128 with four buffers and
// 64 x 64: 22.6 / 22.7 / 23.2 / 43.1 and 26.3 / 26.5 / 27.5 / 38.6, over a k of 1024 9.9 / 10.3 / 10.6 / 18.8 and
// 10.4 / 10.7 / 11.7 / 15.3.
// Over a short k what a tile loads and stores first and last counts, and 256 x 256 with one block a CU
// has nothing beside it: 8192 rows of 256 / 2048 to 8192 channels 119 / 215 us, 128 x 128 81 / 200. Up
// to 64 channels larger tiles multiply zeros: 100000 rows of 256 to 64 24 us, 128 x 128 14.0, 64 x 64
// 14.2, with half the k at a time 11.4.
// Eight waves a block in each: four waves of twice the size were 12 - 60 % slower, since a wave
// by itself issues an instruction in 8 cycles.
static void linear_tiles(const LinearArgs &a, int yt, const LinearPlan &ks, void *sums_at, hipStream_t st) {
    if (ks.parts > 1) {
        const TileGrid tg((a.n + 63) / 64, (a.rows + 63) / 64);
        const dim3 grid(tg.tiles, ks.parts);
        int32_t *sums = static_cast<int32_t *>(sums_at);
        if (dma_can(a.x, a.ldx) && dma_can(a.w, a.ldw))
            k_linear_tile<64, 64, 32, 16, 256, 2, true, kSums><<<grid, 512, 0, st>>>(a, tg, ks.k_part, sums);
        else k_linear_tile<64, 64, 32, 16, 128, 2, false, kSums><<<grid, 512, 0, st>>>(a, tg, ks.k_part, sums);
        join_parts(a, yt, ks.parts, sums, st);
        return;
    }
    auto tiles = [&](uint64_t size) { return (a.n + size - 1) / size * ((a.rows + size - 1) / size); };
    if (dma_can(a.x, a.ldx) && dma_can(a.w, a.ldw)) {
        if (a.n <= 64 && tiles(64) >= 256) linear_tile<64, 64, 32, 16, 128, 2, true>(a, yt, st);
        else if (a.k > 2048 && tiles(256) >= 256) linear_tile<256, 256, 128, 64, 128, 2, true>(a, yt, st);
        else if (tiles(128) >= 320) linear_tile<128, 128, 64, 32, 128, 2, true>(a, yt, st);
        else if (tiles(128) >= 192) linear_tile<128, 128, 64, 32, 128, 4, true>(a, yt, st);
        else linear_tile<64, 64, 32, 16, 256, 2, true>(a, yt, st);
    } else {
        linear_tile<64, 64, 32, 16, 128, 2, false>(a, yt, st);
    }
}

// A grid holds fewer than 2^32 threads: a product beyond 2^20 channels, or of more results than
// 2^34, goes out in several launches.
template <typename F>
static void slabs(const LinearArgs &a, int y_dtype, uint32_t x_size, F launch) {
    const uint64_t most_n = 1ull << 20;
    for (uint64_t n0 = 0; n0 < a.n; n0 += most_n) {
        const uint64_t n = std::min<uint64_t>(a.n - n0, most_n);
        const uint64_t most_m = (1ull << 34) / std::max<uint64_t>(n, 1024);
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

// What a call needs; without a pointer: at any place of those rows (the forms differ, and none needs
// the most at all sizes).
uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype, const void *x, uint64_t ldx, const void *w,
                     uint64_t ldw) {
    uint64_t most = 0;
    for (const bool x_fits : {false, true})
        for (const bool w_fits : {false, true})
            if ((!x || x_fits == dma_can(x, ldx)) && (!w || w_fits == dma_can(w, ldw)))
                most = std::max(most, LinearPlan(rows, k, n, x_dtype, x_fits, w_fits).bytes());
    return most;
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
    if (x_dtype != FSX_DTYPE_I8 && (p.form == kNarrow || p.form == kDirectFloats)) {
        slabs(a, y_dtype, elem_size(x_dtype), [&](const LinearArgs &b) {
            if (p.form == kNarrow) launch_linear_narrow(b, x_dtype, y_dtype, st);
            else if (x_dtype == FSX_DTYPE_F32) linear_direct<FSX_DTYPE_F32>(b, p.tall, 1, b.k, nullptr, y_dtype, st);
            else if (x_dtype == FSX_DTYPE_F16) linear_direct<FSX_DTYPE_F16>(b, p.tall, 1, b.k, nullptr, y_dtype, st);
            else linear_direct<FSX_DTYPE_BF16>(b, p.tall, 1, b.k, nullptr, y_dtype, st);
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
        else if (p.form == kDirect) {
            int32_t *sums = p.parts > 1 ? reinterpret_cast<int32_t *>(at) : nullptr;
            linear_direct<FSX_DTYPE_I8>(b, p.tall, p.parts, p.k_part, sums, y_dtype, st);
            if (sums) join_parts(b, y_dtype, p.parts, sums, st);
        }
        else linear_tiles(b, y_dtype, p, at, st);   // (in parts: small enough for one launch)
    });
    return hipGetLastError();
}

}  // namespace fsx
