// fsx_head.h — heads of free size (fsx_quantize.hip, fsx_linear.hip, fsx_narrow.hip,
// fsx_logprobs.hip): element types, the host
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
void launch_linear_narrow(const LinearArgs &a, int x_dtype, int y_dtype, hipStream_t st);   // k <= 64
uint64_t linear_work(uint64_t rows, uint32_t k, uint32_t n, int x_dtype, const void *x, uint64_t ldx, const void *w,
                     uint64_t ldw);
hipError_t launch_linear(const LinearArgs &a, int x_dtype, int y_dtype, void *work, hipStream_t st);
uint64_t logprobs_work(uint64_t rows, uint32_t v, uint32_t top);
hipError_t launch_logprobs(const LogprobArgs &a, int dtype, hipStream_t st);

#ifdef __HIPCC__
// ---- device helpers
template <int DT> struct Elem;
template <> struct Elem<FSX_DTYPE_F32> { using T = float; };
template <> struct Elem<FSX_DTYPE_F16> { using T = _Float16; };
template <> struct Elem<FSX_DTYPE_BF16> { using T = __bf16; };

// The value of lane ^ O, without LDS where the hardware has a lane permutation for it.
template <int O> __device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
    static_assert(O == 1 || O == 2 || O == 4 || O == 8 || O == 16 || O == 32, "one bit");
    if constexpr (O == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);          // quad_perm 1 0 3 2
    else if constexpr (O == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);     // quad_perm 2 3 0 1
    else if constexpr (O == 4) return __builtin_amdgcn_ds_swizzle(v, 0x101F);                // xor 4
    else if constexpr (O == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);    // row_ror 8
    else if constexpr (O == 16) return __builtin_amdgcn_ds_swizzle(v, 0x401F);               // xor 16
    else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return __lane_id() < 32 ? r[1] : r[0];
    }
}
template <int O> __device__ __forceinline__ float xor_lane(float v) {
    return __uint_as_float(xor_lane<O>(__float_as_uint(v)));
}
template <int O> __device__ __forceinline__ unsigned long long xor_lane(unsigned long long v) {
    return (unsigned long long)xor_lane<O>((uint32_t)(v >> 32)) << 32 | xor_lane<O>((uint32_t)v);
}
struct LargerWord { __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); } };
// f over the G lanes (a power of two) of a group, in every lane of it
template <int G, typename T, typename F> __device__ __forceinline__ T group_all(T v, F f) {
    if constexpr (G > 1) v = f(v, xor_lane<1>(v));
    if constexpr (G > 2) v = f(v, xor_lane<2>(v));
    if constexpr (G > 4) v = f(v, xor_lane<4>(v));
    if constexpr (G > 8) v = f(v, xor_lane<8>(v));
    if constexpr (G > 16) v = f(v, xor_lane<16>(v));
    if constexpr (G > 32) v = f(v, xor_lane<32>(v));
    return v;
}
#endif

}  // namespace fsx
