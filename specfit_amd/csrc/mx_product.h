// Products of rows in microscaled 8 bits with weights in microscaled 4 bits on
// v_mfma_scale_f32_*_f8f6f4, shared by K15 and K16.  The weights are the
// instruction's first operand, so a lane ends up with four neighbouring
// outputs of one row.
#pragma once

#include "mx.h"

namespace sf_mx {

// The 8-bit operand of the 16x16x128 form: lane g * 16 + r holds, of row r,
// values g * 16 .. + 15 and 64 + g * 16 .. + 15 of the tile, and the scale of
// block g.
struct RowsOperand {
  u32x4 lo, hi;
  uint32_t scale;  // the tile's byte lowest
};

// A lane's place in rows held in e4m3.
template <int XDT>
struct RowSource {
  const uint8_t* codes;
  const uint8_t* scales;
  __device__ __forceinline__ void set(const void* base, const void* scale_base, int64_t row,
                                      int64_t /*stride*/, int dim, int g) {
    codes = static_cast<const uint8_t*>(base) + row * (static_cast<int64_t>(tiles(dim)) * kTile) + g * 16;
    scales = static_cast<const uint8_t*>(scale_base) + row * (static_cast<int64_t>(quads(dim)) * 16) + g * 4;
  }
  struct Loaded {
    u32x4 lo, hi;
    uint32_t scale;
  };
  __device__ __forceinline__ Loaded load(int t, int /*dim*/, int /*g*/) const {
    return {ld<u32x4>(codes + t * kTile), ld<u32x4>(codes + t * kTile + 64), ld<uint32_t>(scales + t / 4 * 16)};
  }
  static __device__ __forceinline__ RowsOperand operand(const Loaded& v, int t, int /*g*/) {
    return {v.lo, v.hi, v.scale >> (8 * (t % 4))};
  }
};

// A lane's place in rows of 16-bit values, rounded to e4m3 here as K13 does:
// 16 neighbours in a lane, the other half of their block in lane ^ 16.
template <int DT>
struct RawSource {
  const char* at;
  __device__ __forceinline__ void set(const void* base, const void* /*scale_base*/, int64_t row,
                                      int64_t stride, int /*dim*/, int g) {
    at = static_cast<const char*>(base) + (row * stride + g * 16) * 2;
  }
  struct Loaded {
    u32x4 v[4];
  };
  __device__ __forceinline__ Loaded load(int t, int dim, int g) const {
    Loaded l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = t * kTile + (i / 2) * 64 + (i % 2) * 8;  // of lane group 0
      l.v[i] = u32x4{0u, 0u, 0u, 0u};
      if (k + g * 16 < dim) l.v[i] = ld<u32x4>(at + static_cast<int64_t>(k) * 2);  // rows are whole eights
    }
    return l;
  }
  static __device__ __forceinline__ RowsOperand operand(const Loaded& l, int /*t*/, int g) {
    RowsOperand o;
    uint32_t byte[2];
    u32x4* half[2] = {&o.lo, &o.hi};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[16];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) unpack2<DT>(l.v[2 * h + i / 4][i % 4], f[2 * i], f[2 * i + 1]);
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, magnitude(f[i]));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      byte[h] = scale_byte<kE4m3>(top);
      u32x4 w = {0u, 0u, 0u, 0u};
      if (byte[h] != 255) {
        const float s = inverse_scale(byte[h]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = e4m3x4(f[4 * i] * s, f[4 * i + 1] * s, f[4 * i + 2] * s, f[4 * i + 3] * s);
      }
      *half[h] = w;
    }
    // Blocks 0 and 1 are the low halves of lane groups 0, 1 and 2, 3, blocks 2
    // and 3 their high halves; the scale of block g goes to group g.
    const uint32_t other = static_cast<uint32_t>(__shfl_xor(static_cast<int>(g == 1 ? byte[1] : byte[0]), 48));
    o.scale = g == 0 ? byte[0] : g == 3 ? byte[1] : other;
    return o;
  }
};
template <>
struct RowSource<kBf16> : RawSource<kBf16> {};
template <>
struct RowSource<kFp16> : RawSource<kFp16> {};

__device__ __forceinline__ f32x4 mfma16(u32x4 w, uint32_t w_scale, const RowsOperand& x, f32x4 acc) {
  const i32x8 a = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]),
                   static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 b = {static_cast<int>(x.lo[0]), static_cast<int>(x.lo[1]), static_cast<int>(x.lo[2]),
                   static_cast<int>(x.lo[3]), static_cast<int>(x.hi[0]), static_cast<int>(x.hi[1]),
                   static_cast<int>(x.hi[2]), static_cast<int>(x.hi[3])};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, 0, static_cast<int>(w_scale), 0,
                                                          static_cast<int>(x.scale));
}

// A lane's place in the row tiles of a weight.
struct WeightSource {
  const uint8_t* codes;
  const uint8_t* scales;
  __device__ __forceinline__ void set(const uint8_t* code_base, const uint8_t* scale_base, int64_t row_tile,
                                      int dim, int lane) {
    codes = code_base + row_tile * tiles(dim) * 1024 + lane * 16;
    scales = scale_base + row_tile * quads(dim) * 256 + lane * 4;
  }
};

// acc[n][m] += rows of m times weight rows of n over tiles [begin, end), by one
// wavefront straight from memory: what few rows need, where every weight byte
// is used once.  AHEAD tiles are requested together.
template <int MT, int NT, int XDT, int AHEAD>
__device__ __forceinline__ void accumulate(f32x4 (&acc)[NT][MT], const WeightSource (&w)[NT],
                                           const RowSource<XDT> (&x)[MT], int begin, int end, int dim,
                                           int g) {
  for (int t0 = begin; t0 < end; t0 += AHEAD) {
    u32x4 wc[AHEAD][NT];
    uint32_t wsc[AHEAD][NT];
    typename RowSource<XDT>::Loaded xl[AHEAD][MT];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int t = min(t0 + u, end - 1);  // a tile of the range: its loads need no branch
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        wc[u][n] = ld<u32x4>(w[n].codes + static_cast<int64_t>(t) * 1024);
        wsc[u][n] = ld<uint32_t>(w[n].scales + static_cast<int64_t>(t / 4) * 256);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) xl[u][m] = x[m].load(t, dim, g);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int t = t0 + u;
      if (t >= end) break;  // wave-uniform
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const RowsOperand o = RowSource<XDT>::operand(xl[u][m], t, g);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][m] = mfma16(wc[u][n], wsc[u][n] >> (8 * (t % 4)), o, acc[n][m]);
      }
    }
  }
}

// The tiles of part i of n.
__device__ __forceinline__ void part_of(int count, int i, int n, int& begin, int& end) {
  begin = count * i / n;
  end = count * (i + 1) / n;
}

}  // namespace sf_mx
