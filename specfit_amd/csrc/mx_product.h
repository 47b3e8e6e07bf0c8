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

// ------------------------------------------------------- tiles of many rows --
// WN x WM wavefronts, each FN x FM products of 32 weight rows by 32 rows on
// v_mfma_scale_f32_32x32x64_f8f6f4.  A stage is one tile (128 values) of the
// workgroup's rows and weight rows; two stages alternate, the next one on its
// way into LDS (loads that write it themselves) while the present one is
// multiplied.  The scales of four tiles come together, ahead of them.
//
// Where the operands of a whole tile fit beside the accumulators they are read
// first, and the stage that they leave takes the tile after the next: twice the
// time for a load, for a second meeting (us, one ahead and two: 61 x 2,048 x
// 151,936 44.8 / 41.4; experts of 1,024 tokens 112.7 / 109.7; with 4 x 2 products
// the registers do not suffice, 8,192^3 423 / 433).
//
// LDS: rows keep their 128 bytes together, piece p (16 bytes) of row r in slot
// p ^ (r / 2 & 7): the loads then take whole lines from memory, and the sixteen
// lanes that read a piece of sixteen rows together meet sixteen different
// places of the 64 banks, a pair of rows apart in each slot.  Weight pieces
// stay in the operand's order.
template <int WN_, int WM_, int FN_, int FM_>
struct Tiling {
  static constexpr int WN = WN_, WM = WM_, FN = FN_, FM = FM_;
  static constexpr int kWaves = WN * WM, kThreads = kWaves * SF_WAVE;
  static constexpr int kRows = 32 * FM * WM, kOut = 32 * FN * WN;  // of a workgroup
  static constexpr bool kTwoAhead = FN * FM <= 4;
  static constexpr int kRowLoads = kRows / 8 / kWaves, kOutLoads = kOut / 16 / kWaves;
  static_assert(kRows / 8 % kWaves == 0 && kOut / 16 % kWaves == 0, "whole loads for a wavefront");
  static constexpr int kRowScaleLoads = (kRows + 63) / 64, kOutScaleLoads = (kOut + 63) / 64;
  struct Stage {
    uint8_t rows[kRows * kTile];
    uint8_t out[kOut * kTile / 2];
  };
  struct Scales {
    uint8_t rows[kRowScaleLoads * 1024];
    uint8_t out[kOutScaleLoads * 1024];
  };
};

// Which tile a workgroup takes.  Neighbouring workgroups run on different XCDs,
// each with its own L2: an XCD gets a run of the tiles, the run goes by bands of
// kBand row groups, so that what runs together shares rows and weights there.
constexpr int kXcds = 8, kBand = 8;

__device__ __forceinline__ void tile_of(int id, int row_groups, int out_groups, int& row_group, int& out_group) {
  const int total = row_groups * out_groups, each = total / kXcds, more = total % kXcds;
  const int xcd = id % kXcds;
  const int at = xcd * each + min(xcd, more) + id / kXcds;
  const int band = at / (kBand * out_groups);
  const int first = band * kBand, rows_here = min(kBand, row_groups - first);
  const int in_band = at - band * kBand * out_groups;
  row_group = first + in_band % rows_here;
  out_group = in_band / rows_here;
}

__device__ __forceinline__ void to_lds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Operands of s_waitcnt: at most n vector memory loads under way; no LDS reads.
constexpr int loads_left(int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; }
constexpr int kLdsRead = 0xc07f;

// This wavefront's wait, then all wavefronts' meeting.  The builtins rather than
// assembly: the compiler then knows what has landed and adds no waits of its own.
template <int WAIT>
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_sched_barrier(0);  // the products before the wait, not behind it
  __builtin_amdgcn_s_waitcnt(WAIT);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ i32x8 operand4(const uint8_t* at) {
  const u32x4 v = *reinterpret_cast<const u32x4*>(at);
  return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]),
               0, 0, 0, 0};
}

__device__ __forceinline__ i32x8 operand8(const uint8_t* lo, const uint8_t* hi) {
  const u32x4 a = *reinterpret_cast<const u32x4*>(lo), b = *reinterpret_cast<const u32x4*>(hi);
  return i32x8{static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]),
               static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
}

// acc[n][m] = the workgroup's rows times its weight rows.  row_at(r) is row r's
// number (r < kRows; any valid row for those past the end), out_tile(i) the row
// tile of the weight's i-th 16 rows as an offset of tiles from w and ws.
template <class T, class RowAt, class OutTile>
__device__ __forceinline__ void multiply(f32x16 (&acc)[T::FN][T::FM], const uint8_t* x, const uint8_t* x_scales,
                                         const uint8_t* w, const uint8_t* w_scales, int dim, RowAt row_at,
                                         OutTile out_tile, typename T::Stage& stage0, typename T::Stage& stage1,
                                         typename T::Scales (&scales)[2]) {
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / SF_WAVE);
  const int wn = wave / T::WM, wm = wave % T::WM;
  const int kt = tiles(dim), kq = quads(dim);
  const int r = lane & 31, g = lane >> 5;
  // This wavefront's loads: 8 rows each, and 16 weight rows each.
  const uint8_t* row_from[T::kRowLoads];
#pragma unroll
  for (int i = 0; i < T::kRowLoads; ++i) {
    const int row = (wave * T::kRowLoads + i) * 8 + lane / 8;
    row_from[i] = x + static_cast<int64_t>(row_at(row)) * (static_cast<int64_t>(kt) * kTile) +
                  (lane % 8 ^ (row / 2 & 7)) * 16;
  }
  const uint8_t* out_from[T::kOutLoads];
#pragma unroll
  for (int i = 0; i < T::kOutLoads; ++i)
    out_from[i] = w + (static_cast<int64_t>(out_tile(wave * T::kOutLoads + i)) * kt) * 1024;

  const uint8_t* scales_from[(T::kRowScaleLoads + T::kWaves - 1) / T::kWaves];
#pragma unroll
  for (int i = 0; i < (T::kRowScaleLoads + T::kWaves - 1) / T::kWaves; ++i)  // 64 rows each
    scales_from[i] = x_scales + static_cast<int64_t>(row_at(min((wave + i * T::kWaves) * 64 + lane, T::kRows - 1))) *
                                    (static_cast<int64_t>(kq) * 16);

  const auto load_stage = [&](typename T::Stage& s, int t) {
#pragma unroll
    for (int i = 0; i < T::kRowLoads; ++i)
      to_lds(row_from[i] + static_cast<int64_t>(t) * kTile, s.rows + (wave * T::kRowLoads + i) * 1024);
#pragma unroll
    for (int i = 0; i < T::kOutLoads; ++i)
      to_lds(out_from[i] + static_cast<int64_t>(t) * 1024 + lane * 16, s.out + (wave * T::kOutLoads + i) * 1024);
  };
  const auto load_scales = [&](int q) {
    typename T::Scales& s = scales[q % 2];
#pragma unroll
    for (int i = 0; i < (T::kRowScaleLoads + T::kWaves - 1) / T::kWaves; ++i) {
      const int at = wave + i * T::kWaves;
      if (at < T::kRowScaleLoads) to_lds(scales_from[i] + q * 16, s.rows + at * 1024);
    }
#pragma unroll
    for (int i = 0; i < (T::kOutScaleLoads + T::kWaves - 1) / T::kWaves; ++i) {
      const int at = T::kWaves - 1 - wave + i * T::kWaves;  // four row tiles, 256 bytes each
      if (at < T::kOutScaleLoads)
        to_lds(w_scales + (static_cast<int64_t>(out_tile(at * 4 + lane / 16)) * kq + q) * 256 + lane % 16 * 16,
               s.out + at * 1024);
    }
  };

#pragma unroll
  for (int n = 0; n < T::FN; ++n)
#pragma unroll
    for (int m = 0; m < T::FM; ++m) acc[n][m] = f32x16{};
  // Scale words of blocks g and 2 + g (the tile's halves), the present tile's
  // byte lowest.
  uint32_t ws[T::FN][2], xs[T::FM][2];
  const auto read_scales = [&](int q) {
    const typename T::Scales& s = scales[q % 2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < T::FN; ++n)
        ws[n][h] = *reinterpret_cast<const uint32_t*>(s.out + ((wn * T::FN + n) * 2 + r / 16) * 256 +
                                                      (2 * h + g) * 64 + r % 16 * 4);
#pragma unroll
      for (int m = 0; m < T::FM; ++m)
        xs[m][h] = *reinterpret_cast<const uint32_t*>(s.rows + ((wm * T::FM + m) * 32 + r) * 16 + (2 * h + g) * 4);
    }
  };
  const auto step = [&](typename T::Stage& here, typename T::Stage& other, int t) {
    if (t % 4 == 0) read_scales(t / 4);
    const auto request = [&](typename T::Stage& s, int ahead) {
      if (t % 4 == 0 && t + 4 < kt) load_scales(t / 4 + 1);
      // No branch here, or the products would be moved behind it: past the end
      // the last tile comes once more, unread.
      load_stage(s, min(t + ahead, kt - 1));
      __builtin_amdgcn_sched_barrier(0);
    };
    i32x8 a[2][T::FN], b[2][T::FM];
    const auto read = [&](int h) {
#pragma unroll
      for (int m = 0; m < T::FM; ++m) {
        const int row = (wm * T::FM + m) * 32 + r;
        const uint8_t* at = here.rows + row * kTile;
        b[h][m] = operand8(at + ((4 * h + g) ^ (row / 2 & 7)) * 16, at + ((4 * h + 2 + g) ^ (row / 2 & 7)) * 16);
      }
#pragma unroll
      for (int n = 0; n < T::FN; ++n)
        a[h][n] = operand4(here.out + ((wn * T::FN + n) * 2 + r / 16) * 1024 + (2 * h + g) * 256 + r % 16 * 16);
    };
    if constexpr (T::kTwoAhead) {
      read(0);
      read(1);
      meet<kLdsRead>();
      request(here, 2);
    } else {
      request(other, 1);
      read(0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!T::kTwoAhead && h) read(1);
#pragma unroll
      for (int n = 0; n < T::FN; ++n)
#pragma unroll
        for (int m = 0; m < T::FM; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              a[h][n], b[h][m], acc[n][m], 4, 0, 0, static_cast<int>(ws[n][h]), 0, static_cast<int>(xs[m][h]));
    }
    if constexpr (!T::kTwoAhead) {
      // All of the first half's reads, then the second half's among the first's
      // products.
      constexpr int kReads = T::FN + 2 * T::FM, kProducts = T::FN * T::FM, kMfma = 0x8, kDsRead = 0x100;
      __builtin_amdgcn_sched_group_barrier(kDsRead, kReads, 0);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, (kReads + kProducts - 1) / kProducts, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kMfma, kProducts, 0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < T::FN; ++n) ws[n][h] >>= 8;
#pragma unroll
      for (int m = 0; m < T::FM; ++m) xs[m][h] >>= 8;
    }
    // Two ahead: the loads of this step stay under way.
    meet<T::kTwoAhead ? loads_left(T::kRowLoads + T::kOutLoads) : loads_left(0) & kLdsRead>();
  };

  load_scales(0);
  load_stage(stage0, 0);
  if constexpr (T::kTwoAhead) load_stage(stage1, min(1, kt - 1));
  meet<loads_left(0)>();
  int t = 0;
  for (; t + 2 <= kt; t += 2) {
    step(stage0, stage1, t);
    step(stage1, stage0, t + 1);
  }
  if (t < kt) step(stage0, stage1, t);
  __builtin_amdgcn_s_waitcnt(loads_left(0));  // nothing on its way into LDS that is given back
}

// The 32 x 32 form leaves a lane four neighbours in every eight columns, the other
// four in lane + 32.  Of two such pieces (in turn) lanes 0 to 31 get the first eight
// columns' whole, lanes 32 to 63 the second's.
__device__ __forceinline__ void join(uint32_t& first, uint32_t& second) {
  const u32x2 both = __builtin_amdgcn_permlane32_swap(first, second, false, false);
  first = both[0];
  second = both[1];
}

}  // namespace sf_mx
