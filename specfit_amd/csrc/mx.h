// Microscaled values on gfx950: 8 bits (e4m3) for activations, 4 bits (e2m1)
// for weights, 32 neighbours of a row sharing a power-of-two scale.
//
// A block's scale is 2^e, e the least integer from -127 up at which no value
// rounds past the type's largest (448: up to 464 rounds to it; 6: below 7
// does), held as the byte e + 127.  Values are rounded to nearest, ties to
// even.  A block with an infinity or a NaN has the byte 255 and reads as NaN
// throughout, which the matrix instructions honour.
//
// Layouts ("tile": 128 values of a row, 4 blocks):
//   rows     codes [rows][tiles * 128], zeros behind the row's end; scales
//            [rows][quads * 16], the byte of block b of tile t at
//            t / 4 * 16 + b * 4 + t % 4 -- a lane that holds block b of four
//            tiles in turn reads its four scales as one word.
//   weights  codes [row tiles of 16][tiles][64 lanes][16 bytes], lane b * 16 +
//            r holding block b of row r: one load of a wavefront, 1 KiB in a
//            piece, is the operand of v_mfma_scale_f32_16x16x128_f8f6f4, and
//            the pieces of two row tiles are that of the 32x32x64 form.
//            Scales [row tiles][quads][64 lanes][4], the byte of tile t in
//            t % 4.  Row tiles come in pairs, rows behind the last are zeros.
// Bytes of tiles that a row does not have (the last quad's) count for nothing.
#pragma once

#include "sf_common.h"

namespace sf_mx {

constexpr int kBlock = 32;
constexpr int kTile = 128;
constexpr int kE4m3 = 0, kE2m1 = 1;
constexpr int kBf16 = 0, kFp16 = 1, kFp32 = 2, kRows = 3;  // dtype of an operand; kRows: rows in e4m3

inline __host__ __device__ int tiles(int dim) { return (dim - 1) / kTile + 1; }
inline __host__ __device__ int quads(int dim) { return (dim - 1) / (4 * kTile) + 1; }
inline __host__ __device__ int row_tiles(int rows) { return ((rows - 1) / 32 + 1) * 2; }
inline __host__ __device__ int64_t weight_code_bytes(int rows, int dim) {
  return static_cast<int64_t>(row_tiles(rows)) * tiles(dim) * 1024;
}
inline __host__ __device__ int64_t weight_scale_bytes(int rows, int dim) {
  return static_cast<int64_t>(row_tiles(rows)) * quads(dim) * 256;
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T>
__device__ __forceinline__ T ld(const void* p) {
  return *(const __attribute__((address_space(1))) T*)(p);
}

// Element of dtype DT at p as fp32 (exact).
template <int DT>
__device__ __forceinline__ float element(const void* p) {
  if (DT == kFp32) return ld<float>(p);
  const uint16_t v = ld<uint16_t>(p);
  if (DT == kFp16) return static_cast<float>(__builtin_bit_cast(_Float16, v));
  return sf_bf16_to_f32(v);
}

template <int DT>
constexpr __host__ __device__ int size_of() {
  return DT == kFp32 ? 4 : 2;
}

template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if (DT == kFp16) {
    a = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
    b = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
  } else {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  }
}

// Pieces of 16 bytes that start at any element: one load or store all the same.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef u32x2 __attribute__((aligned(2))) u32x2_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// 8 neighbours at p as fp32.
template <int DT>
__device__ __forceinline__ void load8(const char* p, float (&f)[8]) {
  if (DT == kFp32) {
    const f32x4 a = ld<f32x4_any>(p), b = ld<f32x4_any>(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  } else {
    const u32x4 v = ld<u32x4_any>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<DT>(v[i], f[2 * i], f[2 * i + 1]);
  }
}

// fp32 -> bits of dtype, rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t narrow(float f) {
  if (DT == kFp32) return __float_as_uint(f);
  if (DT == kFp16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  return sf_f32_to_bf16(f);
}

template <int DT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if (DT == kFp16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
  }
  return narrow<DT>(a) | (narrow<DT>(b) << 16);
}

// The value that dtype holds of f.
template <int DT>
__device__ __forceinline__ float held_as(float f) {
  if (DT == kFp32) return f;
  if (DT == kFp16) return static_cast<float>(static_cast<_Float16>(f));
  return sf_round_bf16(f);
}

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// Scale byte of a block whose largest magnitude has these bits.
template <int HELD>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  const uint32_t fraction = top & 0x7fffffu;
  const int e = static_cast<int>(top >> 23) +
                (HELD == kE4m3 ? -8 + (fraction > 0x680000u) : -2 + (fraction >= 0x600000u));
  return static_cast<uint32_t>(max(e, 0));
}

// 2^-e of a scale byte (not 255), the factor that takes values to codes: a
// power of two in fp32's normal range, so the product is exact but for values
// far below the block's largest, which become 0 either way.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}

// 2^e of a scale byte; NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7fc00000u)
                     : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}

__device__ __forceinline__ uint32_t e2m1x8(const float (&f)[8]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], 1.0f, 3);
}

// Largest of four neighbouring lanes' values.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0xB1, 0xf, 0xf, false)));
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x4E, 0xf, 0xf, false)));
}

// Writes chunk c (8 values) of a row in e4m3; the four lanes of a block hold
// its chunks in turn and are all active.
__device__ __forceinline__ void store_rows_chunk(const float (&f)[8], int c, uint8_t* codes,
                                                 uint8_t* scales) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(f[i]));
  const uint32_t byte = scale_byte<kE4m3>(quad_max(top));
  u32x2 w = {0u, 0u};
  if (byte != 255) {
    const float s = inverse_scale(byte);
    w = u32x2{e4m3x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s),
              e4m3x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s)};
  }
  *reinterpret_cast<u32x2*>(codes + 8 * c) = w;
  if (c % 4 == 0) {
    const int block = c / 4, tile = block / 4;
    scales[tile / 4 * 16 + block % 4 * 4 + tile % 4] = static_cast<uint8_t>(byte);
  }
}

// Rows to e4m3, chunk `at` of all rows'.  A lane takes 8 neighbours, so a block is
// four lanes of one DPP quad, and loads and stores of a wavefront lie in a piece.
template <int DT>
__device__ __forceinline__ void quantize_rows_chunk(int64_t at, const char* __restrict__ x, int64_t row_stride,
                                                    int dim, int chunks, int64_t total, uint8_t* __restrict__ codes,
                                                    uint8_t* __restrict__ scales) {
  if (at >= total) return;  // a row's chunks are a multiple of 16: quads end together
  const int64_t row = total <= 0x7fffffff
                          ? static_cast<int64_t>(static_cast<uint32_t>(at) / static_cast<uint32_t>(chunks))
                          : at / chunks;
  const int c = static_cast<int>(at - row * chunks);
  const char* p = x + (row * row_stride + 8 * c) * size_of<DT>();
  float f[8] = {};
  if (8 * c + 8 <= dim) {
    load8<DT>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * c + i < dim) f[i] = element<DT>(p + i * size_of<DT>());
  }
  store_rows_chunk(f, c, codes + row * chunks * 8,
                   scales + row * (static_cast<int64_t>((chunks + 63) / 64) * 16));
}

// A grid's work-items are counted in 32 bits.
inline bool grid_fits(int64_t groups, int threads) { return groups <= 0xffffffffll / threads; }

inline bool aligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

}  // namespace sf_mx
