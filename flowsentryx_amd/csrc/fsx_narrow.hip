// fsx_narrow.hip — int8 layers over short rows (up to 64 of k; include/fsx_hip.h
// fsx_linear_q8_device): x in registers, floats quantised there.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "fsx_q8_rows.h"

namespace fsx {

// v_mfma_i32_16x16x64_i8, the weights first: lane l gives bytes 16 (l / 16) .. of row l % 16 of
// either operand and holds channels 4 (l / 16) .. of row l % 16 of the result. A row of x is CH
// chunks of 16, so a wave's lanes hold 64 / CH rows, a chunk each, in 4 / CH groups of 16 rows.
// The weights' chunks are repeated for every group; a group is multiplied with the other
// groups' lanes 0. x is read and y written once (the weights stay in registers), which bounds
// it: 2^22 rows of 8 floats to 16 floats. PART: k is no multiple of 8 (the loads of a row's last
// values take registers from the number of waves).
template <int XT, int CH, int TN, int YT, bool PART>
__global__ __launch_bounds__(256, TN == 1 && !PART && XT != FSX_DTYPE_I8 ? 6 : 3) void k_linear_narrow(LinearArgs a) {
    using T = typename Elem<YT>::T;
    constexpr int GROUPS = 4 / CH;
    const uint32_t lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
    const uint32_t n0 = blockIdx.y * (16 * TN);
    const uint32_t chunk = lq % CH, my_group = lq / CH;
    v4i w[TN];
    Channels ch[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const uint64_t c = n0 + 16 * i + lr, cc = c < a.n ? c : a.n - 1;
        w[i] = load16_there(a.w + cc * a.ldw + 16 * chunk, (int64_t)a.k - 16 * chunk,
                            (int64_t)((a.n - 1 - cc) * a.ldw) + (int64_t)a.k - 16 * chunk);
        ch[i].load(a, n0 + 16 * i + 4 * lq);
    }
    const uint64_t step = (uint64_t)gridDim.x * 4 * 16 * GROUPS;
    uint64_t r0 = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 * GROUPS;
    const int64_t ok = (int64_t)a.k - 16 * chunk;
    // the next rows of x are under way while a wave works on the ones before
    RawChunk<XT == FSX_DTYPE_I8 ? FSX_DTYPE_F32 : XT> raw;
    v4i next_x = {0, 0, 0, 0};
    float next_scale = 0.0f;
    auto fetch = [&](uint64_t at) {
        const uint64_t r = at + 16 * my_group + lr, rr = r < a.rows ? r : a.rows - 1;
        const int64_t there = (int64_t)((a.rows - 1 - rr) * a.ldx) + ok;   // from here to the last row's end
        if constexpr (XT == FSX_DTYPE_I8) {
            next_x = load16_there(static_cast<const int8_t *>(a.x) + rr * a.ldx + 16 * chunk, ok, there);
            next_scale = a.x_scale[rr];
        } else if (ok > 0) {
            raw.template load<PART>(static_cast<const typename Elem<XT>::T *>(a.x) + rr * a.ldx + 16 * chunk, ok, there);
        }
    };
    fetch(r0);
    for (; r0 < a.rows; r0 += step) {
        v4i x = next_x;
        float xs = next_scale;
        if constexpr (XT != FSX_DTYPE_I8) {
            uint32_t m = ok > 0 ? raw.mag() : 0;
            if (CH > 1) m = max(m, xor_lane<16>(m));
            if (CH > 2) m = max(m, xor_lane<32>(m));
            xs = row_scale(mag_value<XT>(m));
            x = ok > 0 && xs == xs ? raw.codes(1.0f / xs, xs, a.k) : v4i{0, 0, 0, 0};
        }
        if (r0 + step < a.rows) fetch(r0 + step);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            v4i xg, acc[TN];
#pragma unroll
            for (int e = 0; e < 4; ++e) xg[e] = GROUPS == 1 || my_group == (uint32_t)g ? x[e] : 0;
            const float s = GROUPS == 1 ? xs : __shfl(xs, g * CH * 16 + lr);
#pragma unroll
            for (int i = 0; i < TN; ++i)
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], xg, v4i{0, 0, 0, 0}, 0, 0, 0);
            const uint64_t row = r0 + 16 * g + lr;
            if (row >= a.rows) continue;
            T *y = static_cast<T *>(a.y) + row * a.ldy;
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const uint32_t c = n0 + 16 * i + 4 * lq;
                float v[4];
                ch[i].scale(acc[i], s, v);
                activate(v, a.act);
                if (c < a.n) store4(y + c, v, (int64_t)a.n - c);
            }
        }
    }
}

template <int XT, int CH, int TN, int YT> static void linear_narrow(const LinearArgs &a, hipStream_t st) {
    // (more blocks than fit at once only while a block's start, its weights, is short: 2^20 rows of 63 to 64
    // channels 124 us with 4096 blocks, 114 with 2048; 2^22 rows of 8 to 16 118 and 121)
    constexpr uint32_t BLOCKS = TN == 1 ? 4096 : 2048;
    const uint64_t waves = (a.rows + 16 * (4 / CH) - 1) / (16 * (4 / CH));
    const uint32_t gy = (a.n + 16 * TN - 1) / (16 * TN);
    const dim3 grid((uint32_t)std::min<uint64_t>((waves + 3) / 4, std::max<uint32_t>(1, BLOCKS / gy)), gy);
    if (XT == FSX_DTYPE_I8 || a.k % 8 == 0) k_linear_narrow<XT, CH, TN, YT, false><<<grid, 256, 0, st>>>(a);
    else k_linear_narrow<XT, CH, TN, YT, XT != FSX_DTYPE_I8><<<grid, 256, 0, st>>>(a);
}
template <int XT, int CH, int TN> static void linear_narrow(const LinearArgs &a, int yt, hipStream_t st) {
    if (yt == FSX_DTYPE_F32) linear_narrow<XT, CH, TN, FSX_DTYPE_F32>(a, st);
    else if (yt == FSX_DTYPE_F16) linear_narrow<XT, CH, TN, FSX_DTYPE_F16>(a, st);
    else linear_narrow<XT, CH, TN, FSX_DTYPE_BF16>(a, st);
}
template <int XT, int CH> static void linear_narrow(const LinearArgs &a, int yt, hipStream_t st) {
    // (64 channels a wave, or 16 where that leaves SIMDs without one)
    if (a.n <= 16 || (a.rows * CH / 64 + 1) * (a.n / 64 + 1) < 2048) linear_narrow<XT, CH, 1>(a, yt, st);
    else linear_narrow<XT, CH, 4>(a, yt, st);
}
template <int XT> static void linear_narrow(const LinearArgs &a, int yt, hipStream_t st) {
    if (a.k <= 16) linear_narrow<XT, 1>(a, yt, st);
    else if (a.k <= 32) linear_narrow<XT, 2>(a, yt, st);
    else linear_narrow<XT, 4>(a, yt, st);
}

void launch_linear_narrow(const LinearArgs &a, int x_dtype, int y_dtype, hipStream_t st) {
    if (x_dtype == FSX_DTYPE_F32) linear_narrow<FSX_DTYPE_F32>(a, y_dtype, st);
    else if (x_dtype == FSX_DTYPE_F16) linear_narrow<FSX_DTYPE_F16>(a, y_dtype, st);
    else if (x_dtype == FSX_DTYPE_BF16) linear_narrow<FSX_DTYPE_BF16>(a, y_dtype, st);
    else linear_narrow<FSX_DTYPE_I8>(a, y_dtype, st);
}

}  // namespace fsx
