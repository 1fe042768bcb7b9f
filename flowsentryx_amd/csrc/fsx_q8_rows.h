// fsx_q8_rows.h — device pieces of the int8 layers (fsx_quantize.hip, fsx_linear.hip,
// fsx_narrow.hip): rows of floats to codes, and a sum of products to an output.
#pragma once
#include "fsx_head.h"

namespace fsx {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr float kMinScale = 1.17549435e-38f;   // 2^-126

// The row's scale from its largest |x| (NaN or infinite: NaN). The quotient rounds once: a
// 53-bit quotient of 24-bit numbers rounded to 24 bits is the 24-bit quotient.
__device__ __forceinline__ float row_scale(float amax) {
    return amax < INFINITY ? fmaxf(amax / 127.0f, kMinScale) : NAN;
}

// rhe(x / s), exactly, of x >= 0 with a quotient near a half (inv = 1 / s, rounded): the remainder
// x - lo s decides, lo = floor(x / s). It is exact in 32 bits (lo = 0: x itself; else a multiple
// of the last place of s, about s / 2 in size), so comparing it with s / 2 finds the border itself.
__device__ __forceinline__ float code_near_half(float x, float inv, float s) {
    const float lo = floorf(x * inv), rem = fmaf(-lo, s, x), h = 0.5f * s;
    const bool up = rem > h || (rem == h && ((int)lo & 1));
    return lo + (up ? 1.0f : 0.0f);
}

// The codes of N values (a multiple of 4), four to a word. x inv + 1.5 2^23 rounds once, to a
// whole number whose lowest byte is the code: right unless x / s lies within 2^-16 of a half,
// since |x / s| <= 127.5 and inv is off by 2^-24 of itself. The distance from that whole number
// says so, and then the few values concerned are decided exactly.
template <int N>
__device__ __forceinline__ void encode(const float *v, float inv, float s, uint32_t *q) {
    constexpr float kWhole = 12582912.0f;
    uint32_t t[N];
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float r = fmaf(v[i], inv, kWhole);
        t[i] = __float_as_uint(r);
        far = fmaxf(far, fabsf(fmaf(v[i], inv, -(r - kWhole))));
    }
    if (far > 0.49998f)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float r = fmaf(v[i], inv, kWhole);
            const int exact = (int)copysignf(code_near_half(fabsf(v[i]), inv, s), v[i]);
            t[i] = fabsf(fmaf(v[i], inv, -(r - kWhole))) > 0.49998f ? (uint32_t)exact : t[i];
        }
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        const uint32_t lo = __builtin_amdgcn_perm(t[4 * w + 1], t[4 * w], 0x0c0c0400);
        const uint32_t hi = __builtin_amdgcn_perm(t[4 * w + 3], t[4 * w + 2], 0x0c0c0400);
        q[w] = hi << 16 | lo;
    }
}

constexpr int kQV = 16;   // codes a thread makes at a time: one 16-byte store

// Magnitudes as words that are ordered as they are, NaN above infinity: |x|'s bits.
template <int DT> __device__ __forceinline__ float mag_value(uint32_t m) {
    if constexpr (DT == FSX_DTYPE_F32) return __uint_as_float(m);
    else if constexpr (DT == FSX_DTYPE_BF16) return __uint_as_float(m << 16);
    else {
        const uint16_t h = (uint16_t)m;
        _Float16 f;
        __builtin_memcpy(&f, &h, 2);
        return (float)f;
    }
}
typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
template <int DT> struct RawChunk {   // kQV values as they lie in memory
    using T = typename Elem<DT>::T;
    static constexpr int WORDS = kQV * sizeof(T) / 4;
    uint32_t w[WORDS];
    // ok > 0 values count, behind them: 0 (PART false: a whole number of eights). `there` values can be read.
    template <bool PART = true> __device__ __forceinline__ void load(const T *p, int64_t ok, int64_t there = 0) {
        if (ok >= kQV) {
            __builtin_memcpy(w, p, sizeof(w));
            return;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // eight at a time
            uint32_t *half = w + h * WORDS / 2;
            const int64_t here = ok - 8 * h;
            if (here >= 8) {
                __builtin_memcpy(half, p + 8 * h, sizeof(w) / 2);
            } else if (PART && here > 0 && there >= 8 * h + 8) {   // (the next row's; they are read in one and cleared)
                __builtin_memcpy(half, p + 8 * h, sizeof(w) / 2);
#pragma unroll
                for (int i = 0; i < WORDS / 2; ++i) {
                    const int64_t values = here - (int64_t)(i * (4 / sizeof(T)));   // of this word on
                    half[i] = values <= 0 ? 0 : values == 1 && sizeof(T) == 2 ? half[i] & 0xFFFFu : half[i];
                }
            } else if (PART && here > 0) {
                T t[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = p[8 * h + (i < here ? i : 0)];
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = i < here ? t[i] : (T)0.0f;
                __builtin_memcpy(half, t, sizeof(w) / 2);
            } else {
#pragma unroll
                for (int i = 0; i < WORDS / 2; ++i) half[i] = 0;
            }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (DT == FSX_DTYPE_F32) return __uint_as_float(w[i]);
        else if constexpr (DT == FSX_DTYPE_BF16)
            return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        else return mag_value<DT>(w[i / 2] >> (16 * (i % 2)));
    }
    __device__ __forceinline__ uint32_t mag() const {
        if constexpr (DT == FSX_DTYPE_F32) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            v2u16 m = {0, 0};
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const uint32_t u = w[i] & 0x7FFF7FFFu;
                v2u16 h;
                __builtin_memcpy(&h, &u, 4);
                m = __builtin_elementwise_max(m, h);
            }
            return max((uint32_t)m[0], (uint32_t)m[1]);
        }
    }
    // (n: the values that count, the same in the block; beyond them 0)
    __device__ __forceinline__ v4i codes(float inv, float s, uint32_t n = kQV) const {
        uint32_t q[4] = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h && n <= 8) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = value(8 * h + i);
            encode<8>(v, inv, s, q + 2 * h);
        }
        return v4i{(int)q[0], (int)q[1], (int)q[2], (int)q[3]};
    }
};

// ---- products

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

// load16 where `there` bytes can be read from p on (the next rows'): then in one load, and cleared.
__device__ __forceinline__ v4i load16_there(const int8_t *p, int64_t ok, int64_t there) {
    if (there < 16) return load16(p, ok);
    v4i v;
    __builtin_memcpy(&v, p, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = (int)ok - 4 * i;   // of this word on
        v[i] &= left >= 4 ? -1 : left <= 0 ? 0 : (int)((1u << (8 * left)) - 1);
    }
    return v;
}

// 16 bytes from p on. A load at an address that is no multiple of 4 takes several times as long
// (16 rows of 4096 to 4096 channels at odd strides 11.9 us, at strides of 4 7.0), so with `odd` (the
// same in the wave) they come from the whole words that they lie in, shifted into place.
__device__ __forceinline__ v4i load16_at(const int8_t *p, bool odd) {
    v4i v;
    if (!odd) {
        __builtin_memcpy(&v, p, 16);
        return v;
    }
    const uint32_t back = (uint32_t)(uintptr_t)p & 3;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p - back), *last = w + (back ? 4 : 3);
    __builtin_memcpy(&v, w, 16);
    const uint32_t e = *last;
    v4i o;
    o[0] = (int)__builtin_amdgcn_alignbyte((uint32_t)v[1], (uint32_t)v[0], back);
    o[1] = (int)__builtin_amdgcn_alignbyte((uint32_t)v[2], (uint32_t)v[1], back);
    o[2] = (int)__builtin_amdgcn_alignbyte((uint32_t)v[3], (uint32_t)v[2], back);
    o[3] = (int)__builtin_amdgcn_alignbyte(e, (uint32_t)v[3], back);
    return o;
}

// load16 where the row's end lies at p + ok, 16 bytes or more behind its start; ok may be
// below 0. One load and no condition: behind the end the row's last 16 bytes, moved down.
__device__ __forceinline__ v4i load16_end(const int8_t *p, int ok) {
    const int gone = ok >= 16 ? 0 : 16 - ok;   // bytes
    unsigned long long h[2];
    __builtin_memcpy(h, p - gone, 16);
    const uint32_t bits = 8 * (gone & 7);
    if (gone & 7) {
        h[0] = h[0] >> bits | h[1] << (64 - bits);
        h[1] >>= bits;
    }
    unsigned long long lo = gone >= 16 ? 0 : gone >= 8 ? h[1] : h[0], hi = gone >= 8 ? 0 : h[1];
    v4i v;
    v[0] = (int)lo;
    v[1] = (int)(lo >> 32);
    v[2] = (int)hi;
    v[3] = (int)(hi >> 32);
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

__device__ __forceinline__ void activate(float (&v)[4], int act) {
    if (act == FSX_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = relu(v[e]);
    } else if (act == FSX_ACT_SIGMOID) {
        // (a branch: the compiler would compute it for every activation and then choose, 150 instructions)
        asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = sigmoid(v[e]);
    }
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
    __device__ __forceinline__ void scale(const v4i &acc, float xs, float (&v)[4]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled(acc[e], xs, ws[e], b[e]);
    }
};

// The sums of four neighbouring channels of row r to y.
__device__ __forceinline__ void put_sums(const LinearArgs &a, int yt, const v4i &sum, float xs, uint64_t r, uint64_t c) {
    const int64_t left = (int64_t)a.n - (int64_t)c;
    if (left <= 0) return;
    Channels ch;
    ch.load(a, c);
    float v[4];
    ch.scale(sum, xs, v);
    activate(v, a.act);
    const uint64_t at = r * a.ldy + c;
    if (yt == FSX_DTYPE_F32) store4(static_cast<float *>(a.y) + at, v, left);
    else if (yt == FSX_DTYPE_F16) store4(static_cast<_Float16 *>(a.y) + at, v, left);
    else store4(static_cast<__bf16 *>(a.y) + at, v, left);
}

}  // namespace fsx
