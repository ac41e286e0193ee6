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
// The values of eight codes.
__device__ __forceinline__ void mx4_decode8(uint32_t codes, float* v) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = x.x;
        v[2 * i + 1] = x.y;
    }
}

// Eight neighbouring values of a row as they are stored, zeros behind the end.
template <typename T> struct Eight {
    static constexpr int kWords = 8 * (int)sizeof(T) / 4;
    alignas(16) uint32_t w[kWords];

    // BYTES: what an access may take, 16, 4 or an element's own (rows start and end on multiples of it).
    template <int BYTES> __device__ __forceinline__ void load(const T* row, int64_t col, int64_t cols) {
        if constexpr (BYTES == 4 && sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = col + 2 * k < cols ? *reinterpret_cast<const uint32_t*>(row + col + 2 * k) : 0u;
        } else if constexpr (BYTES == 16) {
            constexpr int N = VecTraits<T>::kVec;
#pragma unroll
            for (int k = 0; k < 8 / N; ++k)
                reinterpret_cast<uint4*>(w)[k] = col + k * N < cols ? *reinterpret_cast<const uint4*>(row + col + k * N) : make_uint4(0u, 0u, 0u, 0u);
        } else {
            T v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? row[col + i] : from_f<T>(0.f);
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
                else w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&v[2 * i]) | (uint32_t)*reinterpret_cast<const uint16_t*>(&v[2 * i + 1]) << 16;
            }
        }
    }
};

// Largest magnitudes. 16-bit types: packed maxima of two values at once (a NaN stays a NaN); float32: as integers, where a NaN is
// above every number. amax_bits gives the float32 bits.
template <typename T> __device__ __forceinline__ uint32_t amax_word(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t amax_word<float>(uint32_t a, uint32_t b) { return max(a, b & 0x7fffffffu); }
template <> __device__ __forceinline__ uint32_t amax_word<__half>(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), __habs2(*reinterpret_cast<__half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t amax_word<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), __habs2(*reinterpret_cast<__nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// A word's two values (or its one) in float32.
template <typename T> __device__ __forceinline__ float2 word_values(uint32_t w);
template <> __device__ __forceinline__ float2 word_values<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 word_values<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// float32 bits of the larger of a word's two magnitudes.
template <typename T> __device__ __forceinline__ uint32_t amax_bits(uint32_t w) {
    if constexpr (sizeof(T) == 4) return w;
    else {
        const float2 v = word_values<T>(w);
        return max(__float_as_uint(v.x), __float_as_uint(v.y));
    }
}

// Products of two float32 at once.
__device__ __forceinline__ void mul2(float& a, float& b, float f, float g) {
    uint64_t x, y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(f), "f"(g));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}

// The scale byte of the block that a lane shares with its three neighbours, and the codes of its eight values.
template <typename T> __device__ __forceinline__ uint32_t mx4_encode_lane(const Eight<T>& v, uint32_t& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Eight<T>::kWords; ++i) m = amax_word<T>(m, v.w[i]);
    m = amax_word<T>(m, __shfl_xor_sync(DC_FULL, m, 1));
    m = amax_word<T>(m, __shfl_xor_sync(DC_FULL, m, 2));
    scale = mx4_scale_byte(amax_bits<T>(m));
    const float f = mx4_factor(scale);
    float u[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = __uint_as_float(v.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 x = word_values<T>(v.w[i]); u[2 * i] = x.x; u[2 * i + 1] = x.y; }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mul2(u[2 * i], u[2 * i + 1], f, f);
    const uint32_t code = mx4_encode8(u);
    return scale == 255u ? 0u : code;
}
// The scale bytes of the four blocks of sixteen lanes as one word (in every lane).
__device__ __forceinline__ uint32_t mx4_scale_quad(uint32_t scale, int lane) {
    uint32_t word = scale << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(DC_FULL, word, 4);
    return word | __shfl_xor_sync(DC_FULL, word, 8);
}

// The widest access that rows of `cols` elements at x allow.
template <typename T> inline int row_access(const void* x, int64_t cols) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(cols * (int64_t)sizeof(T));
    return (a & 15u) == 0 ? 16 : (a & 3u) == 0 ? 4 : (int)sizeof(T);
}

int mx4_quantize_two(const void* x, void* data, void* scales, void* data_t, void* scales_t, int64_t rows, const void* x2, void* data2, void* scales2,
                     void* data_t2, void* scales_t2, int64_t rows2, int64_t cols, int dtype, cudaStream_t st);

}  // namespace dc
