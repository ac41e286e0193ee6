// MXFP4 (microscaled 4-bit floating point): geometry of the packed form and the element conversions.
//
// A row is cut into blocks of 32 values; a block is 32 e2m1 codes (values +-{0, 1/2, 1, 3/2, 2, 3, 4, 6}) under one
// power-of-two scale 2^(s - 127) held as the byte s. s = max(E - 2, 0), E being the biased float32 exponent of the block's
// largest magnitude (E - 2 brings it into [4, 8), values above 6 saturate); s = 255 marks a block with an infinity or a
// NaN, and the whole block then stands for NaN (e2m1 has neither).
//   codes:  [rows][16 nb] bytes, nb = ceil(cols / 32), the even column in the low half, zeros behind the last column
//   scales: [ceil(rows / 128)][ceil(nb / 4)][32][4][4] bytes, block b of row r at [r / 128][b / 4][r % 32][r % 128 / 32][b % 4]:
//           the 512 bytes of 128 rows x 4 blocks as tcgen05.cp takes them into tensor memory, in one contiguous copy
#pragma once
#include "dc_common.cuh"

namespace dc {

constexpr int kMxBlock = 32;

__host__ __device__ inline int64_t mx4_blocks(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }
__host__ __device__ inline int64_t mx4_scale_tiles(int64_t cols) { return (mx4_blocks(cols) + 3) / 4; }
// Byte offset of the scales of blocks 4 * bt .. 4 * bt + 3 of row r, tiles = mx4_scale_tiles(cols).
__device__ __forceinline__ int64_t mx4_scale_word(int64_t r, int64_t bt, int64_t tiles) {
    return ((r >> 7) * tiles + bt) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4;
}

// Scale byte of a block from the bits of its largest magnitude, and the factor 2^(127 - s) that brings values onto the e2m1
// grid (0 for a block that stands for NaN: its codes are 0 whatever it holds).
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ float mx4_factor(uint32_t s) { return __uint_as_float((254u - (s == 255u ? 0u : s)) << 23); }
__device__ __forceinline__ float mx4_scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fffffffu) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}

// Eight values (already multiplied by the factor) to eight codes, value 0 in the lowest half byte; round to nearest even,
// saturating.
__device__ __forceinline__ uint32_t mx4_encode8(const float* v) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// The value of one code: sign, two exponent bits (bias 1), one mantissa bit.
__device__ __forceinline__ float mx4_decode(uint32_t code) {
    const uint32_t e = (code >> 1) & 3u, m = code & 1u;
    const float a = e == 0u ? 0.5f * (float)m : (float)((2u + m) << (e - 1u)) * 0.5f;
    return (code & 8u) ? -a : a;
}

// Eight values of a row starting at column col (cols in all); zeros behind the end.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const T* row, int64_t col, int64_t cols) {
    if constexpr (VEC) {
        constexpr int N = 8 / VecTraits<T>::kVec;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            Pack<T, VecTraits<T>::kVec> p;
            if (col + k * VecTraits<T>::kVec < cols) p.load(row + col + k * VecTraits<T>::kVec);
            else p.zero();
#pragma unroll
            for (int i = 0; i < VecTraits<T>::kVec; ++i) v[k * VecTraits<T>::kVec + i] = p.get(i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? to_f<T>(row[col + i]) : 0.f;
    }
}

__device__ __forceinline__ uint32_t amax8_bits(const float (&v)[8]) {
    uint32_t m = 0;      // as integers: a NaN is above every number, so it is not lost
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t encode_scaled(const float (&v)[8], uint32_t s) {
    if (s == 255u) return 0u;
    const float f = mx4_factor(s);
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = v[i] * f;
    return mx4_encode8(u);
}

}  // namespace dc
