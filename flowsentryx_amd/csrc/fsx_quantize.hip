// fsx_quantize.hip — rows of floats to int8 codes with one scale a row (include/fsx_hip.h
// fsx_quantize_rows_device): scale_r = max(fl32(max_c |x_rc| / 127), 2^-126),
// q_rc = x_rc / scale_r to the nearest whole number, halves to even.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "fsx_q8_rows.h"

namespace fsx {

// A group of TPR threads takes a row, up to C chunks of kQV values a thread; they stay in
// registers between the maximum and the codes (C 0: longer rows are read twice, the second
// time from cache). A row's last chunk ends with the row and repeats codes of the one before, so that
// rows of kQV values and more are read and written in whole chunks.
template <int DT, int TPR, int C>
__global__ __launch_bounds__(256) void k_quantize_rows(const void *__restrict__ xp, uint64_t rows, uint32_t cols,
                                                       uint64_t ldx, int8_t *__restrict__ q, uint64_t ldq,
                                                       float *__restrict__ scale) {
    using T = typename Elem<DT>::T;
    constexpr uint32_t RPB = 256 / TPR, STEP = TPR * kQV;
    __shared__ uint32_t s_max[4];
    const uint32_t t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    for (uint64_t r0 = (uint64_t)blockIdx.x * RPB; r0 < rows; r0 += (uint64_t)gridDim.x * RPB) {
        const uint64_t r = r0 + sub;
        const bool live = r < rows;
        const T *x = static_cast<const T *>(xp) + (live ? r : 0) * ldx;
        auto at = [&](uint32_t c) { return cols >= kQV && c + kQV > cols ? cols - kQV : c; };
        uint32_t m = 0;
        RawChunk<DT> kept[C ? C : 1];
        if constexpr (C > 0) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const uint32_t c = t * kQV + i * STEP;
                if (live && c < cols) kept[i].load(x + at(c), (int64_t)cols - at(c));
            }
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (live && t * kQV + i * STEP < cols) m = max(m, kept[i].mag());
        } else if (live) {
            for (uint64_t c = t * kQV; c < cols; c += STEP) {
                kept[0].load(x + at((uint32_t)c), (int64_t)cols - at((uint32_t)c));
                m = max(m, kept[0].mag());
            }
        }
        m = group_all<TPR < 64 ? TPR : 64>(m, LargerWord());
        if constexpr (TPR > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
            __syncthreads();
            m = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
        }
        if (!live) continue;
        const float s = row_scale(mag_value<DT>(m));
        const bool ok = s == s;
        const float inv = 1.0f / s;
        if (t == 0) scale[r] = s;
        int8_t *qr = q + r * ldq;
        auto put = [&](uint32_t c, const RawChunk<DT> &k) {
            const v4i o = ok ? k.codes(inv, s) : v4i{0, 0, 0, 0};
            if (cols - c >= kQV) __builtin_memcpy(qr + c, &o, kQV);
            else
#pragma unroll
                for (int i = 0; i < kQV; ++i) if (c + i < cols) qr[c + i] = (int8_t)(o[i / 4] >> (8 * (i % 4)));
        };
        if constexpr (C > 0) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (t * kQV + i * STEP < cols) put(at(t * kQV + i * STEP), kept[i]);
        } else {
            for (uint64_t c = t * kQV; c < cols; c += STEP) {
                kept[0].load(x + at((uint32_t)c), (int64_t)cols - at((uint32_t)c));
                put(at((uint32_t)c), kept[0]);
            }
        }
    }
}

template <int DT>
static void quantize_rows(const void *x, uint64_t rows, uint32_t cols, uint64_t ldx, int8_t *q, uint64_t ldq,
                          float *scale, hipStream_t st) {
    const uint64_t per = ((uint64_t)cols + kQV - 1) / kQV;   // chunks of a row
    auto go = [&](auto kernel, uint32_t tpr) {
        const uint64_t blocks = (rows + 256 / tpr - 1) / (256 / tpr);
        kernel<<<(uint32_t)std::min<uint64_t>(blocks, 1u << 16), 256, 0, st>>>(x, rows, cols, ldx, q, ldq, scale);
    };
    // One chunk a thread where that fills a small power of two of threads; else two, which leave fewer
    // threads idle and have more under way (us, one and two: 149075 f16 rows of 317 64 and 46, 10^5 bf16 rows of 512
    // 39 and 37, 20000 of 2000 50 and 30, but 10^5 f32 rows of 256 24.8 and 28.7).
    uint64_t full = 1;
    while (full < per) full *= 2;
    const bool one = full <= 16 && 8 * per >= 7 * full;
    if (full == 1) go(k_quantize_rows<DT, 1, 1>, 1);
    else if (full == 2) go(k_quantize_rows<DT, 2, 1>, 2);
    else if (full == 4) one ? go(k_quantize_rows<DT, 4, 1>, 4) : go(k_quantize_rows<DT, 2, 2>, 2);
    else if (full == 8) one ? go(k_quantize_rows<DT, 8, 1>, 8) : go(k_quantize_rows<DT, 4, 2>, 4);
    else if (full == 16) one ? go(k_quantize_rows<DT, 16, 1>, 16) : go(k_quantize_rows<DT, 8, 2>, 8);
    else if (full == 32) go(k_quantize_rows<DT, 16, 2>, 16);
    else if (full == 64) go(k_quantize_rows<DT, 32, 2>, 32);
    else if (full == 128) go(k_quantize_rows<DT, 64, 2>, 64);
    else if (full == 256) go(k_quantize_rows<DT, 256, 1>, 256);
    else if (full == 512) go(k_quantize_rows<DT, 256, 2>, 256);
    else go(k_quantize_rows<DT, 256, 0>, 256);   // (1574 f16 rows of 11411 17 us; four chunks in registers 36)
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

}  // namespace fsx
