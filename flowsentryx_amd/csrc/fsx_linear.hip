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

// 16 code bytes from p on, of which the first `ok` exist; the others are 0.
__device__ __forceinline__ v4i load16(const int8_t *p, int64_t ok) {
    v4i v = {0, 0, 0, 0};
    if (ok >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (ok > 0) {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < ok ? p[i] : (int8_t)0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

__device__ __forceinline__ float finish(int acc, float xs, float ws, float b, int act) {
    float y = (float)acc * xs * ws + b;
    if (act == FSX_ACT_RELU) y = y < 0.0f ? 0.0f : y;
    else if (act == FSX_ACT_SIGMOID) {
        const float e = expf(-fabsf(y));   // never above 1: no overflow far below 0
        y = (y >= 0.0f ? 1.0f : e) / (1.0f + e);
    }
    return y;
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

// 64 channels x 64 rows a block, 64 of k at a time through LDS, 2 x 2 waves of 32 x 32. The
// weights are the first operand of v_mfma_i32_16x16x64_i8 and x the second: a lane then holds
// four neighbouring channels of one row. Lane l gives bytes 16 (l / 16) .. of row l % 16, and
// holds channels 4 (l / 16) .. of row l % 16 of the result.
constexpr int kTB = 64, kTLd = 80;   // LDS rows 80 bytes apart: 16-byte aligned, banks spread
template <int YT>
__global__ __launch_bounds__(256) void k_linear_tile(LinearArgs a, uint32_t tiles_n, uint64_t tiles) {
    using T = typename Elem<YT>::T;
    __shared__ __attribute__((aligned(16))) int8_t s_w[kTB * kTLd], s_x[kTB * kTLd];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t wn = (wave & 1) * 32, wm = (wave >> 1) * 32, lr = lane & 15, lq = lane >> 4;
    const uint32_t sr = threadIdx.x >> 2, sc = (threadIdx.x & 3) * 16;   // staging: row, byte
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const uint64_t n0 = tile % tiles_n * kTB, m0 = tile / tiles_n * kTB;
        v4i acc[2][2] = {};
        const bool ln = n0 + sr < a.n, lm = m0 + sr < a.rows;
        const int8_t *pw = a.w + (ln ? n0 + sr : 0) * a.ldw;
        const int8_t *px = static_cast<const int8_t *>(a.x) + (lm ? m0 + sr : 0) * a.ldx;
        for (uint32_t k0 = 0; k0 < a.k; k0 += kTB) {
            const int64_t ok = (int64_t)a.k - (k0 + sc);
            const v4i vw = load16(pw + k0 + sc, ln ? ok : 0), vx = load16(px + k0 + sc, lm ? ok : 0);
            __syncthreads();
            *reinterpret_cast<v4i *>(s_w + sr * kTLd + sc) = vw;
            *reinterpret_cast<v4i *>(s_x + sr * kTLd + sc) = vx;
            __syncthreads();
            v4i fw[2], fx[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fw[i] = *reinterpret_cast<const v4i *>(s_w + (wn + 16 * i + lr) * kTLd + 16 * lq);
                fx[i] = *reinterpret_cast<const v4i *>(s_x + (wm + 16 * i + lr) * kTLd + 16 * lq);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint64_t r = m0 + wm + 16 * j + lr;
            if (r >= a.rows) continue;
            const float xs = a.x_scale[r];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint64_t c = n0 + wn + 16 * i + 4 * lq;
                if (c >= a.n) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t ce = c + e < a.n ? c + e : c;
                    v[e] = finish(acc[i][j][e], xs, a.w_scale[ce], a.bias ? a.bias[ce] : 0.0f, a.act);
                }
                store4(static_cast<T *>(a.y) + r * a.ldy + c, v, (int64_t)a.n - (int64_t)c);
            }
        }
    }
}

template <int YT>
static void linear_tile(const LinearArgs &a, hipStream_t st) {
    const uint32_t tn = (a.n + kTB - 1) / kTB;
    const uint64_t tiles = tn * ((a.rows + kTB - 1) / kTB);
    k_linear_tile<YT><<<(uint32_t)std::min<uint64_t>(tiles, 1u << 20), 256, 0, st>>>(a, tn, tiles);
}

uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype) {
    (void)n;
    return x_dtype == FSX_DTYPE_I8 ? 0 : code_space(rows, k).bytes;
}

hipError_t launch_linear(const LinearArgs &in, int x_dtype, int y_dtype, void *work, hipStream_t st) {
    (void)hipGetLastError();
    if (in.rows == 0 || in.n == 0) return hipSuccess;
    LinearArgs a = in;
    if (x_dtype != FSX_DTYPE_I8) {
        const CodeSpace s = code_space(a.rows, a.k);
        int8_t *q = static_cast<int8_t *>(work);
        float *sc = reinterpret_cast<float *>(q + s.scale_at);
        const hipError_t e = launch_quantize_rows(a.x, x_dtype, a.rows, a.k, a.ldx, q, s.ld, sc, st);
        if (e != hipSuccess) return e;
        a.x = q;
        a.x_scale = sc;
        a.ldx = s.ld;
    }
    if (y_dtype == FSX_DTYPE_F32) linear_tile<FSX_DTYPE_F32>(a, st);
    else if (y_dtype == FSX_DTYPE_F16) linear_tile<FSX_DTYPE_F16>(a, st);
    else linear_tile<FSX_DTYPE_BF16>(a, st);
    return hipGetLastError();
}

}  // namespace fsx
