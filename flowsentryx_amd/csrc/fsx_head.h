// fsx_head.h — heads of free size (fsx_linear.hip, fsx_logprobs.hip): element types, the host
// rules that the *_work functions and the launches share, and the launch functions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fsx_hip.h"

namespace fsx {

constexpr uint64_t kMaxIn = 131071;              // 128 * 128 * 131071 < 2^31: the int32 sum is exact
constexpr uint64_t kMaxDim = 0x7FFFFFFFull;      // classes, channels, columns
constexpr uint64_t kMaxRows = 1ull << 40;
constexpr uint64_t kMaxBytes = 1ull << 60;       // rows * ld * element size stays far from 2^64

__host__ __device__ inline uint32_t elem_size(int dtype) {
    return dtype == FSX_DTYPE_F32 ? 4u : dtype == FSX_DTYPE_I8 ? 1u : 2u;
}
inline uint64_t up16(uint64_t v) { return (v + 15) & ~15ull; }

// Quantised rows in a workspace: codes [rows][up16(k)], then the scales.
struct CodeSpace {
    uint64_t ld, scale_at, bytes;
};
inline CodeSpace code_space(uint64_t rows, uint64_t k) {
    CodeSpace s;
    s.ld = up16(k);
    s.scale_at = rows * s.ld;
    s.bytes = s.scale_at + up16(rows * 4);
    return s;
}

struct LinearArgs {
    const void *x;              // codes
    const float *x_scale;
    uint64_t ldx;
    const int8_t *w;
    const float *w_scale, *bias;
    uint64_t ldw;
    uint64_t rows;
    uint32_t k, n;
    int act;
    void *y;
    uint64_t ldy;
};

struct LogprobArgs {
    const void *x;
    uint64_t rows, ld;
    uint32_t v, top;
    const int32_t *target;
    float *logprob, *entropy;
    int32_t *top_id;
    float *top_lp;
    void *work;
};

hipError_t launch_quantize_rows(const void *x, int dtype, uint64_t rows, uint32_t cols, uint64_t ldx, int8_t *q,
                                uint64_t ldq, float *scale, hipStream_t st);
uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype);
hipError_t launch_linear(const LinearArgs &a, int x_dtype, int y_dtype, void *work, hipStream_t st);
uint64_t logprobs_work(uint64_t rows, uint32_t v, uint32_t top);
hipError_t launch_logprobs(const LogprobArgs &a, int dtype, hipStream_t st);

#ifdef __HIPCC__
// ---- device helpers
template <int DT> struct Elem;
template <> struct Elem<FSX_DTYPE_F32> { using T = float; };
template <> struct Elem<FSX_DTYPE_F16> { using T = _Float16; };
template <> struct Elem<FSX_DTYPE_BF16> { using T = __bf16; };

// N elements of T from p on (any alignment of p that T has: global loads need no more), of
// which the first `ok` exist; the others are `fill`.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T *p, int64_t ok, float fill, float (&v)[N]) {
    T t[N];
    if (ok >= N) {
        __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    } else {
        // (loads without conditions, behind the end the first element again: all are under way at once)
        if (ok > 0)
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = p[i < ok ? i : 0];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < ok ? (float)t[i] : fill;
    }
}
#endif

}  // namespace fsx
