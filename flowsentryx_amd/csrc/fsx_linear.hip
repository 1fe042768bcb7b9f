// fsx_linear.hip — int8 layers of free size: the row quantiser and the int8 matrix product
// with a scale for every row of x and every output channel (include/fsx_hip.h).
//
//   scale_r = max(fl32(max_c |x_rc| / 127), 2^-126)      q_rc = rhe(x_rc / scale_r)
//   y_rn    = act((float)(sum_k q_rk w_nk) * scale_r * t_n + b_n)
#include <hip/hip_runtime.h>
#include <algorithm>

#include "fsx_head.h"

namespace fsx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------- row quantiser

constexpr float kMinScale = 1.17549435e-38f;   // 2^-126

// The row's scale from its largest |x| (NaN or infinite: NaN). The quotient rounds once: a
// 53-bit quotient of 24-bit numbers rounded to 24 bits is the 24-bit quotient.
__device__ __forceinline__ float row_scale(float amax) {
    if (!(amax < INFINITY)) return NAN;
    return fmaxf(amax / 127.0f, kMinScale);
}

// rhe(x / s), exactly, of x >= 0. rint(x * (1/s)) is wrong only where x / s lies within 2^-15
// of a half: x / s <= 127.5 and the product's relative error is below 2^-22. There the
// remainder x - lo s decides, lo = floor(x / s): it is exact in 32 bits (lo = 0: x itself;
// else a multiple of the last place of s, about s / 2 in size), so comparing it with s / 2
// finds the border itself.
__device__ __forceinline__ float code_mag(float x, float inv, float s) {
    const float v = x * inv;
    float r = rintf(v);
    if (fabsf(v - r) > 0.49996f) {
        const float lo = floorf(v), rem = fmaf(-lo, s, x), h = 0.5f * s;
        r = rem > h || (rem == h && ((int)lo & 1)) ? lo + 1.0f : lo;
    }
    return r;
}
__device__ __forceinline__ int code_of(float x, float inv, float s) {
    return (int)copysignf(code_mag(fabsf(x), inv, s), x);
}

// NaN if any value of the row was NaN or infinite (a NaN is lost by fmaxf: it is counted in)
__device__ __forceinline__ float amax_of(float m, float x) {
    const float a = fabsf(x);
    return a > m || a != a ? a : m;      // once NaN, `a > m` is false and m stays NaN
}

constexpr int kQV = 16;   // codes a thread makes at a time: one 16-byte store

// A group of TPR threads takes a row. The row is read twice; the second read comes from cache.
template <int DT, int TPR>
__global__ __launch_bounds__(256) void k_quantize_rows(const void *__restrict__ xp, uint64_t rows, uint32_t cols,
                                                       uint64_t ldx, int8_t *__restrict__ q, uint64_t ldq,
                                                       float *__restrict__ scale) {
    using T = typename Elem<DT>::T;
    constexpr uint32_t RPB = 256 / TPR;
    __shared__ float s_max[4];
    const uint32_t t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    for (uint64_t r0 = (uint64_t)blockIdx.x * RPB; r0 < rows; r0 += (uint64_t)gridDim.x * RPB) {
        const uint64_t r = r0 + sub;
        const bool live = r < rows;
        const T *x = static_cast<const T *>(xp) + (live ? r : 0) * ldx;
        float m = 0.0f;
        if (live)
            for (uint32_t c = t * kQV; c < cols; c += TPR * kQV) {
                float v[kQV];
                load_row<T, kQV>(x + c, (int64_t)cols - c, 0.0f, v);
#pragma unroll
                for (int i = 0; i < kQV; ++i) m = amax_of(m, v[i]);
            }
#pragma unroll
        for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) m = amax_of(m, __shfl_xor(m, o));
        if (TPR > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
            __syncthreads();
            m = 0.0f;
#pragma unroll
            for (int w = 0; w < TPR / 64; ++w) m = amax_of(m, s_max[sub * (TPR / 64) + w]);
        }
        if (!live) continue;
        const float s = row_scale(m);
        const bool ok = s == s;
        const float inv = ok ? 1.0f / s : 0.0f;
        if (t == 0) scale[r] = s;
        int8_t *qr = q + r * ldq;
        for (uint32_t c = t * kQV; c < cols; c += TPR * kQV) {
            float v[kQV];
            int8_t o[kQV];
            load_row<T, kQV>(x + c, (int64_t)cols - c, 0.0f, v);
#pragma unroll
            for (int i = 0; i < kQV; ++i) o[i] = ok ? (int8_t)code_of(v[i], inv, s) : (int8_t)0;
            if (cols - c >= kQV) __builtin_memcpy(qr + c, o, kQV);
            else
#pragma unroll
                for (int i = 0; i < kQV; ++i) if (c + i < cols) qr[c + i] = o[i];
        }
    }
}

template <int DT>
static void quantize_rows(const void *x, uint64_t rows, uint32_t cols, uint64_t ldx, int8_t *q, uint64_t ldq,
                          float *scale, hipStream_t st) {
    const uint32_t per = (cols + kQV - 1) / kQV;   // threads that have a chunk of the row
    auto go = [&](auto kernel, uint32_t tpr) {
        const uint64_t blocks = (rows + 256 / tpr - 1) / (256 / tpr);
        kernel<<<(uint32_t)std::min<uint64_t>(blocks, 1u << 16), 256, 0, st>>>(x, rows, cols, ldx, q, ldq, scale);
    };
    if (per <= 1) go(k_quantize_rows<DT, 1>, 1);
    else if (per <= 4) go(k_quantize_rows<DT, 4>, 4);
    else if (per <= 16) go(k_quantize_rows<DT, 16>, 16);
    else if (per <= 64) go(k_quantize_rows<DT, 64>, 64);
    else go(k_quantize_rows<DT, 256>, 256);
}

hipError_t launch_quantize_rows(const void *x, int dtype, uint64_t rows, uint32_t cols, uint64_t ldx, int8_t *q,
                                uint64_t ldq, float *scale, hipStream_t st) {
    (void)hipGetLastError();
    if (rows == 0) return hipSuccess;
    if (dtype == FSX_DTYPE_F32) quantize_rows<FSX_DTYPE_F32>(x, rows, cols, ldx, q, ldq, scale, st);
    else if (dtype == FSX_DTYPE_F16) quantize_rows<FSX_DTYPE_F16>(x, rows, cols, ldx, q, ldq, scale, st);
    else quantize_rows<FSX_DTYPE_BF16>(x, rows, cols, ldx, q, ldq, scale, st);
    return hipGetLastError();
}

// ---------------------------------------------------------------- int8 product

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

// 16 code bytes from p on, of which the first `ok` exist; the others are 0.
__device__ __forceinline__ v4i load16(const int8_t *p, int64_t ok) {
    v4i v = {0, 0, 0, 0};
    if (ok >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (ok > 0) {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = p[i < ok ? i : 0];   // (no conditions: all under way at once)
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < ok ? b[i] : (int8_t)0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

__device__ __forceinline__ float scaled(int acc, float xs, float ws, float b) { return (float)acc * xs * ws + b; }
__device__ __forceinline__ float relu(float y) { return y < 0.0f ? 0.0f : y; }   // NaN stays
__device__ __forceinline__ float sigmoid(float y) {
    const float e = expf(-fabsf(y));   // never above 1: no overflow far below 0
    return (y >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// Four neighbouring channels of one row, of which the first `ok` exist.
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4], int64_t ok) {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
    if (ok >= 4) __builtin_memcpy(p, t, sizeof(t));
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < ok) p[i] = t[i];
}

template <typename T>
__device__ __forceinline__ void store4(void *y, uint64_t at, const float (&v)[4], int64_t ok) {
    store4(static_cast<T *>(y) + at, v, ok);
}
__device__ __forceinline__ void store4(void *y, int yt, uint64_t at, const float (&v)[4], int64_t ok) {
    if (yt == FSX_DTYPE_F32) store4<float>(y, at, v, ok);
    else if (yt == FSX_DTYPE_F16) store4<_Float16>(y, at, v, ok);
    else store4<__bf16>(y, at, v, ok);
}

// Four neighbouring channels' scales and biases; channels behind the last: the last one's.
struct Channels {
    float ws[4], b[4];
    __device__ __forceinline__ void load(const LinearArgs &a, uint64_t c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t cc = c + e < a.n ? c + e : a.n - 1;
            ws[e] = a.w_scale[cc];
            b[e] = a.bias ? a.bias[cc] : 0.0f;
        }
    }
    __device__ __forceinline__ void finish(const LinearArgs &a, int yt, const v4i &acc, float xs, uint64_t r,
                                           uint64_t c) const {
        if (r >= a.rows || c >= a.n) return;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled(acc[e], xs, ws[e], b[e]);
        if (a.act == FSX_ACT_RELU) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = relu(v[e]);
        } else if (a.act == FSX_ACT_SIGMOID) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = sigmoid(v[e]);
        }
        store4(a.y, yt, r * a.ldy + c, v, (int64_t)a.n - (int64_t)c);
    }
};

// Codes of up to 16 values of a row.
__device__ __forceinline__ v4i pack_codes(const float (&v)[kQV], float inv, float s, bool ok) {
    v4i q;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u |= (uint32_t)(ok ? code_of(v[4 * w + i], inv, s) & 255 : 0) << (8 * i);
        q[w] = (int)u;
    }
    return q;
}

// ---- up to 64 of k: x in registers, floats quantised there
//
// v_mfma_i32_16x16x64_i8, the weights first: lane l gives bytes 16 (l / 16) .. of row l % 16 of
// either operand and holds channels 4 (l / 16) .. of row l % 16 of the result. A row of x is CH
// chunks of 16, so a wave's lanes hold 64 / CH rows, a chunk each, in 4 / CH groups of 16 rows.
// The weights' chunks are repeated for every group; a group is multiplied with the other
// groups' lanes 0. x is read and y written once (the weights stay in registers), which bounds
// it: 2^22 rows of 8 floats to 16 floats.
template <int XT, int CH, int TN>
__global__ __launch_bounds__(256) void k_linear_narrow(LinearArgs a, int yt) {
    constexpr int GROUPS = 4 / CH;
    const uint32_t lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
    const uint32_t n0 = blockIdx.y * (16 * TN);
    const uint32_t chunk = lq % CH, my_group = lq / CH;
    v4i w[TN];
    Channels ch[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const uint64_t c = n0 + 16 * i + lr;
        w[i] = load16(a.w + (c < a.n ? c : a.n - 1) * a.ldw + 16 * chunk, (int64_t)a.k - 16 * chunk);
        ch[i].load(a, n0 + 16 * i + 4 * lq);
    }
    const uint64_t step = (uint64_t)gridDim.x * 4 * 16 * GROUPS;
    for (uint64_t r0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 * GROUPS; r0 < a.rows; r0 += step) {
        const uint64_t r = r0 + 16 * my_group + lr, rr = r < a.rows ? r : a.rows - 1;
        const int64_t ok = (int64_t)a.k - 16 * chunk;
        v4i x;
        float xs;
        if constexpr (XT == FSX_DTYPE_I8) {
            x = load16(static_cast<const int8_t *>(a.x) + rr * a.ldx + 16 * chunk, ok);
            xs = a.x_scale[rr];
        } else {
            using T = typename Elem<XT>::T;
            float v[kQV];
            load_row<T, kQV>(static_cast<const T *>(a.x) + rr * a.ldx + 16 * chunk, ok, 0.0f, v);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < kQV; ++i) m = amax_of(m, v[i]);
            if (CH > 1) m = amax_of(m, __shfl_xor(m, 16));
            if (CH > 2) m = amax_of(m, __shfl_xor(m, 32));
            xs = row_scale(m);
            x = pack_codes(v, 1.0f / xs, xs, xs == xs);
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            v4i xg;
#pragma unroll
            for (int e = 0; e < 4; ++e) xg[e] = GROUPS == 1 || my_group == (uint32_t)g ? x[e] : 0;
            const float s = GROUPS == 1 ? xs : __shfl(xs, g * CH * 16 + lr);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const v4i acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], xg, v4i{0, 0, 0, 0}, 0, 0, 0);
                ch[i].finish(a, yt, acc, s, r0 + 16 * g + lr, n0 + 16 * i + 4 * lq);
            }
        }
    }
}

template <int XT, int CH> static void linear_narrow(const LinearArgs &a, int yt, hipStream_t st) {
    const uint64_t waves = (a.rows + 16 * (4 / CH) - 1) / (16 * (4 / CH));
    const uint32_t tn = a.n <= 16 ? 1 : 4, gy = (a.n + 16 * tn - 1) / (16 * tn);
    const dim3 grid((uint32_t)std::min<uint64_t>((waves + 3) / 4, std::max<uint32_t>(1, 4096 / gy)), gy);
    if (tn == 1) k_linear_narrow<XT, CH, 1><<<grid, 256, 0, st>>>(a, yt);
    else k_linear_narrow<XT, CH, 4><<<grid, 256, 0, st>>>(a, yt);
}
template <int XT> static void linear_narrow(const LinearArgs &a, int yt, hipStream_t st) {
    if (a.k <= 16) linear_narrow<XT, 1>(a, yt, st);
    else if (a.k <= 32) linear_narrow<XT, 2>(a, yt, st);
    else linear_narrow<XT, 4>(a, yt, st);
}

// ---- few rows: the weights' bytes bound it
//
// A block takes 16 channels and all of k, its eight waves 64 of k each in turn, straight from
// memory into v_mfma_i32_16x16x64_i8 (as above) with MT groups of 16 rows; the waves' sums meet
// in LDS. FLOATS: up to four rows of floats, quantised by every block into LDS while its first
// weights are under way (x is small and comes from cache): one launch instead of two.
constexpr int kFW = 8, kFU = 8;          // waves a block, loads in flight a lane
constexpr uint32_t kFusedRows = 4, kFusedBytes = 32768;

template <int XT, int MT>
__global__ __launch_bounds__(64 * kFW) void k_linear_few(LinearArgs a, int yt) {
    constexpr bool FLOATS = XT != FSX_DTYPE_I8;
    extern __shared__ __attribute__((aligned(16))) int8_t s_x[];   // FLOATS: the rows' codes, up64(k) + 16 apart
    __shared__ __attribute__((aligned(16))) v4i s_acc[kFW][MT][64];
    __shared__ uint32_t s_max[kFusedRows];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lq = lane >> 4;
    const uint64_t n0 = (uint64_t)blockIdx.x * 16, c = n0 + lr < a.n ? n0 + lr : a.n - 1;
    const uint32_t chunks = (a.k + 63) / 64, pitch = chunks * 64 + 16;
    const int8_t *pw = a.w + c * a.ldw + 16 * lq;
    auto weights = [&](uint32_t first, v4i (&w)[kFU]) {
#pragma unroll
        for (int u = 0; u < kFU; ++u) {
            const uint32_t k0 = (first + u * kFW) * 64;
            w[u] = k0 + 64 <= a.k ? load16(pw + k0, 16) : load16(pw + k0, (int64_t)a.k - k0 - 16 * lq);
        }
    };
    v4i w[kFU];
    weights(wave, w);
    if constexpr (FLOATS) {
        using T = typename Elem<XT>::T;
        const T *x = static_cast<const T *>(a.x);
        const uint32_t per = chunks * 4, all = (uint32_t)a.rows * per;   // chunks of 16, zeros behind the end
        if (threadIdx.x < kFusedRows) s_max[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t q = threadIdx.x; q < all; q += 64 * kFW) {
            const uint32_t r = q / per, k0 = (q - r * per) * 16;
            float v[kQV], m = 0.0f;
            load_row<T, kQV>(x + r * a.ldx + k0, (int64_t)a.k - k0, 0.0f, v);
#pragma unroll
            for (int i = 0; i < kQV; ++i) m = amax_of(m, v[i]);
            // |x| as words are ordered as they are as numbers, NaN above infinity
            atomicMax(&s_max[r], __float_as_uint(m) & 0x7FFFFFFFu);
        }
        __syncthreads();
        for (uint32_t q = threadIdx.x; q < all; q += 64 * kFW) {
            const uint32_t r = q / per, k0 = (q - r * per) * 16;
            float v[kQV];
            load_row<T, kQV>(x + r * a.ldx + k0, (int64_t)a.k - k0, 0.0f, v);
            const float s = row_scale(__uint_as_float(s_max[r]));
            *reinterpret_cast<v4i *>(s_x + r * pitch + k0) = pack_codes(v, 1.0f / s, s, s == s);
        }
        __syncthreads();
    }
    v4i acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = v4i{0, 0, 0, 0};
    for (uint32_t first = wave; first < chunks; first += kFW * kFU) {
        if (first != wave) weights(first, w);
#pragma unroll
        for (int u = 0; u < kFU; ++u) {
            const uint32_t k0 = (first + u * kFW) * 64;
            if (k0 >= a.k) break;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint32_t r = 16 * m + lr, rr = r < a.rows ? r : (uint32_t)a.rows - 1;
                v4i x;
                if (FLOATS) x = *reinterpret_cast<const v4i *>(s_x + rr * pitch + k0 + 16 * lq);
                else x = load16(static_cast<const int8_t *>(a.x) + rr * a.ldx + k0 + 16 * lq,
                                k0 + 64 <= a.k ? 16 : (int64_t)a.k - k0 - 16 * lq);
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
    for (int i = 1; i < kFW; ++i) sum += s_acc[i][wave][lane];
    const uint64_t r = 16 * wave + lr;
    if (r >= a.rows) return;
    Channels ch;
    ch.load(a, n0 + 4 * lq);
    ch.finish(a, yt, sum, FLOATS ? row_scale(__uint_as_float(s_max[r & (kFusedRows - 1)])) : a.x_scale[r], r,
              n0 + 4 * lq);
}

template <int XT> static void linear_few(const LinearArgs &a, int yt, hipStream_t st) {
    const uint32_t blocks = (a.n + 15) / 16;
    if constexpr (XT != FSX_DTYPE_I8) {
        const uint32_t lds = (uint32_t)a.rows * ((a.k + 63) / 64 * 64 + 16);
        k_linear_few<XT, 1><<<blocks, 64 * kFW, lds, st>>>(a, yt);
    } else if (a.rows <= 16) k_linear_few<XT, 1><<<blocks, 64 * kFW, 0, st>>>(a, yt);
    else if (a.rows <= 32) k_linear_few<XT, 2><<<blocks, 64 * kFW, 0, st>>>(a, yt);
    else k_linear_few<XT, 4><<<blocks, 64 * kFW, 0, st>>>(a, yt);
}

// ---- tiles of BN channels x BM rows, waves of WN x WM, kBK bytes of k at a time through LDS
//
// The weights are the first operand of v_mfma_i32_32x32x32_i8 and x the second: lane l gives
// bytes 16 (l / 32) .. of row l % 32 of either, and holds channels 8 j + 4 (l / 32) .. + 3 of
// row l % 32 of the result: four neighbouring channels of one row.
//
// LDS holds a row's kBK bytes as 16-byte chunks, chunk c of row r at place c ^ (r & 7): the
// eight lanes that read one chunk of eight rows then meet all banks once. Two buffers: while
// one is multiplied, the next tile's loads fly, one barrier a tile. DMA: the loads write LDS
// themselves (operands at 16-byte strides); else they pass through registers.
constexpr int kBK = 128;

template <int ROWS, int THREADS, bool DMA> struct Stage {
    static constexpr int kLoads = ROWS * kBK / 16 / THREADS;   // chunks a thread brings
    const int8_t *base;        // the tile's first row
    uint32_t at, off[kLoads];  // the thread's chunk in a row, and from `base` to its chunks (ld < 2^23)
    uint64_t row[DMA ? 1 : kLoads];
    v4i reg[DMA ? 1 : kLoads];
    // chunk i of this thread: row i * THREADS / 8 + threadIdx / 8, place threadIdx % 8. Rows
    // behind the last: the last one, its results are not stored.
    __device__ __forceinline__ void init(const int8_t *p, uint64_t ld, uint64_t r0, uint64_t rows) {
        const uint32_t tr = threadIdx.x >> 3, pos = threadIdx.x & 7;
        at = 16 * (pos ^ (tr & 7));
        base = p + r0 * ld;
        const uint32_t last = (uint32_t)(rows - r0 < ROWS ? rows - r0 : ROWS) - 1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t r = i * (THREADS / 8) + tr, rr = r < last ? r : last;
            if (DMA) off[i] = rr * (uint32_t)ld + at;
            else row[i] = rr * ld;
        }
    }
    // A chunk that starts behind the row's end: the tile's first (x is cleared there); an
    // aligned chunk that starts inside the row stays in its page.
    __device__ __forceinline__ void load(int8_t *lds, uint32_t k0, uint32_t k) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if (DMA) {
                const int8_t *src = base + k0 + (off[i] - (k0 + at >= k ? at : 0));
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void *)src,
                    (__attribute__((address_space(3))) void *)(lds + (i * THREADS + (threadIdx.x & ~63u)) * 16), 16, 0,
                    0);
            } else {
                reg[i] = load16(base + row[i] + k0 + at, (int64_t)k - k0 - at);
            }
        }
    }
    __device__ __forceinline__ void store(int8_t *lds) {
        if (!DMA)
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                *reinterpret_cast<v4i *>(lds + (i * THREADS + threadIdx.x) * 16) = reg[i];
    }
};

template <int WN, int WM>
struct WaveTile {
    static constexpr int TN = WN / 32, TM = WM / 32, S = kBK / 32;
    v16i acc[TN][TM];
    struct Frag { v4i w[TN], x[TM]; };
    __device__ __forceinline__ void read(Frag &f, const int8_t *sw, const int8_t *sx, uint32_t wn, uint32_t wm, int s) {
        const uint32_t lane = __lane_id(), lr = lane & 31, at = ((2 * s + (lane >> 5)) ^ (lr & 7)) * 16;
#pragma unroll
        for (int i = 0; i < TN; ++i) f.w[i] = *reinterpret_cast<const v4i *>(sw + (wn + 32 * i + lr) * kBK + at);
#pragma unroll
        for (int j = 0; j < TM; ++j) f.x[j] = *reinterpret_cast<const v4i *>(sx + (wm + 32 * j + lr) * kBK + at);
    }
    // One tile of k: a step's reads fly while the step before is multiplied.
    __device__ __forceinline__ void multiply(const int8_t *sw, const int8_t *sx, uint32_t wn, uint32_t wm) {
        Frag f[2];
        read(f[0], sw, sx, wn, wm, 0);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < S) read(f[(s + 1) & 1], sw, sx, wn, wm, s + 1);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[s & 1].w[i], f[s & 1].x[j], acc[i][j], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
};

// x of the last tile behind the rows' end, `left` bytes into the tile: 0 (weights there count nothing then).
template <int BM, int THREADS>
__device__ __forceinline__ void clear_tail(int8_t *sx, uint32_t left) {
    if (left >= kBK) return;
    for (uint32_t c = threadIdx.x; c < BM * 8; c += THREADS) {
        const uint32_t r = c >> 3, first = 16 * ((c & 7) ^ (r & 7));
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

// What each wave has issued has arrived, its reads too; then all waves are here.
__device__ __forceinline__ void tile_barrier() {
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt 0, lgkmcnt 0
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

template <int BN, int BM, int WN, int WM, bool DMA, int YT>
__global__ __launch_bounds__(BN / WN * (BM / WM) * 64) void k_linear_tile(LinearArgs a, TileGrid tg) {
    constexpr int THREADS = BN / WN * (BM / WM) * 64;
    using T = typename Elem<YT>::T;
    __shared__ __attribute__((aligned(16))) int8_t s_w0[BN * kBK], s_x0[BM * kBK], s_w1[BN * kBK], s_x1[BM * kBK];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 31, half = lane >> 5;
    const uint32_t wn = wave % (BN / WN) * WN, wm = wave / (BN / WN) * WM;
    uint32_t bn, bm;
    tg.place(blockIdx.x, bn, bm);
    const uint64_t n0 = (uint64_t)bn * BN, m0 = (uint64_t)bm * BM;
    WaveTile<WN, WM> t;
#pragma unroll
    for (int i = 0; i < t.TN; ++i)
#pragma unroll
        for (int j = 0; j < t.TM; ++j) t.acc[i][j] = v16i{};
    Stage<BN, THREADS, DMA> lw;
    Stage<BM, THREADS, DMA> lx;
    lw.init(a.w, a.ldw, n0, a.n);
    lx.init(static_cast<const int8_t *>(a.x), a.ldx, m0, a.rows);
    const uint32_t tiles = (a.k + kBK - 1) / kBK;
    // tile i + 1 into (sw2, sx2) while tile i in (sw, sx) is multiplied
    auto step = [&](uint32_t i, int8_t *sw, int8_t *sx, int8_t *sw2, int8_t *sx2) {
        tile_barrier();
        if (i + 1 < tiles) {
            lw.load(sw2, (i + 1) * kBK, a.k);
            lx.load(sx2, (i + 1) * kBK, a.k);
        } else {
            clear_tail<BM, THREADS>(sx, a.k - i * kBK);
        }
        t.multiply(sw, sx, wn, wm);
        lw.store(sw2);
        lx.store(sx2);
    };
    lw.load(s_w0, 0, a.k);
    lx.load(s_x0, 0, a.k);
    lw.store(s_w0);
    lx.store(s_x0);
    for (uint32_t i = 0; i < tiles; i += 2) {
        step(i, s_w0, s_x0, s_w1, s_x1);
        if (i + 1 < tiles) step(i + 1, s_w1, s_x1, s_w0, s_x0);
    }
    // the channels' scales and biases come through LDS
    float *s_ws = reinterpret_cast<float *>(s_w0), *s_b = reinterpret_cast<float *>(s_w1);
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < BN; c += THREADS) {
        const uint64_t cc = n0 + c < a.n ? n0 + c : a.n - 1;
        s_ws[c] = a.w_scale[cc];
        s_b[c] = a.bias ? a.bias[cc] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < t.TN; ++i) {
        const uint32_t cw = wn + 32 * i + 4 * half;
        const int64_t left = (int64_t)a.n - (int64_t)(n0 + cw);   // channels from this lane's first on
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < t.TM; ++j) {
            const uint64_t r = m0 + wm + 32 * j + lr;
            const float xs = a.x_scale[r < a.rows ? r : a.rows - 1];
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                v[e] = scaled(t.acc[i][j][e], xs, s_ws[cw + 8 * (e / 4) + e % 4], s_b[cw + 8 * (e / 4) + e % 4]);
            if (a.act == FSX_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = relu(v[e]);
            } else if (a.act == FSX_ACT_SIGMOID) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = sigmoid(v[e]);
            }
            if (r >= a.rows) continue;
            T *y = static_cast<T *>(a.y) + r * a.ldy + n0 + cw;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float o[4] = {v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                if (left > 8 * g) store4(y + 8 * g, o, left - 8 * g);
            }
        }
    }
}

template <int BN, int BM, int WN, int WM, bool DMA>
static void linear_tile(const LinearArgs &a, int yt, hipStream_t st) {
    const TileGrid tg((a.n + BN - 1) / BN, (a.rows + BM - 1) / BM);
    constexpr int threads = BN / WN * (BM / WM) * 64;
    if (yt == FSX_DTYPE_F32) k_linear_tile<BN, BM, WN, WM, DMA, FSX_DTYPE_F32><<<tg.tiles, threads, 0, st>>>(a, tg);
    else if (yt == FSX_DTYPE_F16) k_linear_tile<BN, BM, WN, WM, DMA, FSX_DTYPE_F16><<<tg.tiles, threads, 0, st>>>(a, tg);
    else k_linear_tile<BN, BM, WN, WM, DMA, FSX_DTYPE_BF16><<<tg.tiles, threads, 0, st>>>(a, tg);
}

// Operands that the DMA can bring: chunks at 16-byte addresses, a tile's rows within 2^31 bytes.
static bool dma_can(const void *p, uint64_t ld) { return ((uintptr_t)p | ld) % 16 == 0 && ld < (1u << 23); }

static void linear_tiles(const LinearArgs &a, int yt, hipStream_t st) {
    const bool dma = dma_can(a.x, a.ldx) && dma_can(a.w, a.ldw);
    auto tiles = [&](uint64_t bn, uint64_t bm) { return (a.n + bn - 1) / bn * ((a.rows + bm - 1) / bm); };
    if (tiles(256, 256) >= 256) {
        if (dma) linear_tile<256, 256, 128, 64, true>(a, yt, st);
        else linear_tile<256, 256, 128, 64, false>(a, yt, st);
    } else if (tiles(128, 128) >= 256) {
        if (dma) linear_tile<128, 128, 64, 64, true>(a, yt, st);
        else linear_tile<128, 128, 64, 64, false>(a, yt, st);
    } else {
        if (dma) linear_tile<64, 64, 32, 32, true>(a, yt, st);
        else linear_tile<64, 64, 32, 32, false>(a, yt, st);
    }
}

// Which form takes a product, by its sizes and x's type alone.
enum LinearForm { kNarrow, kFewFloats, kFew, kTiles };
static LinearForm form_of(uint64_t rows, uint32_t k, int x_dtype) {
    if (k <= 64) return kNarrow;
    if (x_dtype != FSX_DTYPE_I8 && rows <= kFusedRows && rows * ((k + 63) / 64 * 64 + 16) <= kFusedBytes)
        return kFewFloats;
    return rows <= 64 ? kFew : kTiles;
}

uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype) {
    (void)n;
    const LinearForm f = form_of(rows, k, x_dtype);
    return x_dtype == FSX_DTYPE_I8 || f == kNarrow || f == kFewFloats ? 0 : code_space(rows, k).bytes;
}

// A grid holds fewer than 2^32 threads: a product beyond 2^20 channels, or of more results than
// 2^38, goes out in several launches.
template <typename F>
static void slabs(const LinearArgs &a, int y_dtype, F launch, uint32_t x_size = 1) {
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

template <int XT> static void linear_floats(const LinearArgs &a, LinearForm f, int yt, hipStream_t st) {
    if (f == kNarrow) linear_narrow<XT>(a, yt, st);
    else linear_few<XT>(a, yt, st);
}

hipError_t launch_linear(const LinearArgs &in, int x_dtype, int y_dtype, void *work, hipStream_t st) {
    (void)hipGetLastError();
    if (in.rows == 0 || in.n == 0) return hipSuccess;
    const LinearForm f = form_of(in.rows, in.k, x_dtype);
    LinearArgs a = in;
    if (x_dtype != FSX_DTYPE_I8) {
        if (f == kNarrow || f == kFewFloats) {
            slabs(a, y_dtype, [&](const LinearArgs &b) {
                if (x_dtype == FSX_DTYPE_F32) linear_floats<FSX_DTYPE_F32>(b, f, y_dtype, st);
                else if (x_dtype == FSX_DTYPE_F16) linear_floats<FSX_DTYPE_F16>(b, f, y_dtype, st);
                else linear_floats<FSX_DTYPE_BF16>(b, f, y_dtype, st);
            }, elem_size(x_dtype));
            return hipGetLastError();
        }
        const CodeSpace s = code_space(a.rows, a.k);
        int8_t *q = static_cast<int8_t *>(work);
        float *sc = reinterpret_cast<float *>(q + s.scale_at);
        const hipError_t e = launch_quantize_rows(a.x, x_dtype, a.rows, a.k, a.ldx, q, s.ld, sc, st);
        if (e != hipSuccess) return e;
        a.x = q;
        a.x_scale = sc;
        a.ldx = s.ld;
    }
    slabs(a, y_dtype, [&](const LinearArgs &b) {
        if (f == kNarrow) linear_narrow<FSX_DTYPE_I8>(b, y_dtype, st);
        else if (f == kFew) linear_few<FSX_DTYPE_I8>(b, y_dtype, st);
        else linear_tiles(b, y_dtype, st);
    });
    return hipGetLastError();
}

}  // namespace fsx
