// K13: values to microscaled 8 and 4 bits and back; K14: the residual's
// addition and RMSNorm with an output in microscaled 8 bits besides.
//
// Formats and layouts are in mx.h.  All of it is memory traffic: a block's
// scale is an integer maximum over the magnitudes' bits, a code the conversion
// instruction's result on the value times an exact power of two.  A lane holds 8
// neighbours, which is a whole 16-byte load of 16-bit values and a quarter of a
// block, whatever the row's alignment.
//
// bf16, one MI355X (a large copy moves 5.0 TB/s):
//   8,192 x 4,096 to e4m3     20.8 us   4.9 TB/s     and back   17.4 us   5.8 TB/s
//   151,936 x 2,048 to e2m1    155 us   5.1 TB/s     and back    128 us   6.1 TB/s
//       (178 us in turn with the kernel that reads them back)
//   8,192 x 4,096 residual, norm, e4m3 output   59 us   5.1 TB/s
//   1 x 2,048: 1.6 (values) to 3 us, a launch's latency
#include "mx.h"

namespace {

using namespace sf_mx;

constexpr int kThreads = 256;

// ------------------------------------------------------------------ K13 ----
// Rows to e4m3.
template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const char* __restrict__ x,
                                                                 int64_t row_stride, int dim,
                                                                 int chunks, int64_t total,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
  quantize_rows_chunk<DT>(static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, x, row_stride, dim, chunks, total,
                          codes, scales);
}

// A weight to e2m1 tiles: a wavefront takes 16 rows by 512 columns, a lane one
// block of each of four tiles -- no exchange between lanes, and codes (1 KiB)
// and scales (256 bytes) leave in a piece.
template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_weight_kernel(
    const char* __restrict__ x, int64_t row_stride, int64_t batch_stride, int rows, int dim,
    uint8_t* __restrict__ codes, int64_t codes_batch, uint8_t* __restrict__ scales,
    int64_t scales_batch) {
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int r = lane & 15, b = lane >> 4;
  const int nt = row_tiles(rows), kt = tiles(dim), kq = quads(dim);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / SF_WAVE) + threadIdx.x / SF_WAVE;
  if (unit >= static_cast<int64_t>(nt) * kq) return;
  const int tile_row = static_cast<int>(unit / kq), q = static_cast<int>(unit % kq);
  const int row = tile_row * 16 + r;
  x += (static_cast<int64_t>(blockIdx.y) * batch_stride + static_cast<int64_t>(min(row, rows - 1)) * row_stride) *
       size_of<DT>();
  codes += blockIdx.y * codes_batch + (static_cast<int64_t>(tile_row) * kt + 4 * q) * 1024 + lane * 16;
  scales += blockIdx.y * scales_batch + (static_cast<int64_t>(tile_row) * kq + q) * 256 + lane * 4;
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (4 * q + j >= kt) break;  // wave-uniform
    const int k0 = (4 * q + j) * kTile + b * kBlock;
    float f[4][8] = {};
    if (row < rows) {
      if (k0 + kBlock <= dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load8<DT>(x + static_cast<int64_t>(k0 + 8 * i) * size_of<DT>(), f[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (k0 + i < dim) f[i / 8][i % 8] = element<DT>(x + static_cast<int64_t>(k0 + i) * size_of<DT>());
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, magnitude(f[i / 8][i % 8]));
    const uint32_t byte = scale_byte<kE2m1>(top);
    u32x4 w = {0u, 0u, 0u, 0u};
    if (byte != 255) {
      const float s = inverse_scale(byte);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[i][k] *= s;
        w[i] = e2m1x8(f[i]);
      }
    }
    *reinterpret_cast<u32x4*>(codes + j * 1024) = w;
    word |= byte << (8 * j);
  }
  *reinterpret_cast<uint32_t*>(scales) = word;
}

// 8 values to out; past the row's end nothing.
template <int DT>
__device__ __forceinline__ void store8(const float (&f)[8], char* p, int left) {
  if (left >= 8) {
    if (DT == kFp32) {
      *reinterpret_cast<f32x4_any*>(p) = f32x4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f32x4_any*>(p + 16) = f32x4{f[4], f[5], f[6], f[7]};
    } else {
      *reinterpret_cast<u32x4_any*>(p) = u32x4{narrow2<DT>(f[0], f[1]), narrow2<DT>(f[2], f[3]),
                                              narrow2<DT>(f[4], f[5]), narrow2<DT>(f[6], f[7])};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= left) break;
    if (DT == kFp32)
      reinterpret_cast<float*>(p)[i] = f[i];
    else
      reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(narrow<DT>(f[i]));
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void rows_values_kernel(const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               int dim, int chunks, int64_t total,
                                                               char* __restrict__ out) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (at >= total) return;
  const int64_t row = total <= 0x7fffffff
                          ? static_cast<int64_t>(static_cast<uint32_t>(at) / static_cast<uint32_t>(chunks))
                          : at / chunks;
  const int c = static_cast<int>(at - row * chunks);
  if (8 * c >= dim) return;
  const u32x2 w = ld<u32x2>(codes + at * 8);
  const int tile = c / 16;
  const float s = scale_value(scales[row * (static_cast<int64_t>((chunks + 63) / 64) * 16) + tile / 4 * 16 +
                                     c / 4 % 4 * 4 + tile % 4]);
  float f[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
    f[4 * i] = a[0] * s, f[4 * i + 1] = a[1] * s, f[4 * i + 2] = b[0] * s, f[4 * i + 3] = b[1] * s;
  }
  store8<DT>(f, out + (row * dim + 8 * c) * size_of<DT>(), dim - 8 * c);
}

// A wavefront to 16 rows of a tile, four rows at a time: sixteen lanes write
// a row's 128 values in a piece (a lane to a block's 32 would write a quarter of
// a line at a time: 151,936 x 2,048 from 255 us to 125).
template <int DT>
__global__ __launch_bounds__(kThreads) void weight_values_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 int rows, int dim,
                                                                 char* __restrict__ out) {
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int kt = tiles(dim), kq = quads(dim);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / SF_WAVE) + threadIdx.x / SF_WAVE;
  const int64_t tile_row = unit / kt;
  const int t = static_cast<int>(unit - tile_row * kt);
  const int c = lane & 15, k = t * kTile + 8 * c;
  if (k >= dim) return;
  const uint8_t* from = codes + unit * 1024 + c / 4 * 256 + c % 4 * 4;
  const uint8_t* scale_from = scales + (tile_row * kq + t / 4) * 256 + c / 4 * 64 + t % 4;
  uint32_t w[4], byte[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * i + (lane >> 4);
    w[i] = byte[i] = 0;
    if (tile_row * 16 + r < rows) {
      w[i] = ld<uint32_t>(from + r * 16);
      byte[i] = ld<uint8_t>(scale_from + r * 4);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = tile_row * 16 + 4 * i + (lane >> 4);
    if (row >= rows) break;
    const float s = scale_value(byte[i]);
    float f[8];
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 2);
    const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 3);
    f[0] = a[0] * s, f[1] = a[1] * s, f[2] = b[0] * s, f[3] = b[1] * s;
    f[4] = d[0] * s, f[5] = d[1] * s, f[6] = e[0] * s, f[7] = e[1] * s;
    store8<DT>(f, out + (row * dim + k) * size_of<DT>(), dim - k);
  }
}

// ------------------------------------------------------------------ K14 ----
// sum = T(x + residual); y = (sum * r) * weight with r = fp32(1 / sqrt(mean of
// sum^2 + eps)); normed = T(y), and y once more in e4m3.  y is rounded once
// for each output.  The mean is kept in 64 bits: r is then the same whatever
// the order of the sum, so are the 8-bit codes, whose borders a last bit of r
// would move values across, and the 64-bit work hides under the row's traffic.
// Addition and products are single fp32 operations (no contraction).
//
// LANES (a wavefront or a workgroup of four) take a row, a lane chunks of 8
// at LANES * 8 from each other, CHUNKS of them in registers between the two
// passes (CHUNKS = 0: any number, read again).
template <int LANES>
__device__ __forceinline__ double row_sum(double v, double* part) {
#pragma unroll
  for (int d = 1; d < SF_WAVE; d *= 2) v += __shfl_xor(v, d);
  if (LANES > SF_WAVE) {
    if ((threadIdx.x & (SF_WAVE - 1)) == 0) part[threadIdx.x / SF_WAVE] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
  }
  return v;
}

template <int DT>
__device__ __forceinline__ void load_sum(const char* x, const char* res, int c, int dim, float (&f)[8]) {
  const int64_t off = static_cast<int64_t>(c) * 8 * size_of<DT>();
  if (8 * c + 8 <= dim) {
    load8<DT>(x + off, f);
    if (res) {
      float g[8];
      load8<DT>(res + off, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = held_as<DT>(f[i] + g[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = 0.f;
    if (8 * c + i < dim) {
      f[i] = element<DT>(x + off + i * size_of<DT>());
      if (res) f[i] = held_as<DT>(f[i] + element<DT>(res + off + i * size_of<DT>()));
    }
  }
}

template <int DT, int LANES, int CHUNKS>
__global__ __launch_bounds__(kThreads) void add_rms_norm_kernel(
    const char* __restrict__ x, int64_t x_stride, const char* __restrict__ residual,
    int64_t residual_stride, int rows, int dim, const char* __restrict__ weight, double eps,
    char* __restrict__ sum, char* __restrict__ normed, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales) {
  constexpr int kRowsHere = kThreads / LANES, kHeld = CHUNKS ? CHUNKS : 1;
  __shared__ double part[kThreads / SF_WAVE];
  const int lane = threadIdx.x % LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsHere + threadIdx.x / LANES;
  if (row >= rows) return;  // a wavefront of a wavefront's row, or nobody
  const int chunks = tiles(dim) * 16;
  const char* xr = x + row * x_stride * size_of<DT>();
  const char* rr = residual ? residual + row * residual_stride * size_of<DT>() : nullptr;
  char* sr = sum ? sum + row * dim * size_of<DT>() : nullptr;
  char* nr = normed ? normed + row * dim * size_of<DT>() : nullptr;
  float f[kHeld][8];
  double total = 0;
  const int steps = CHUNKS ? CHUNKS : (chunks + LANES - 1) / LANES;
  if (CHUNKS) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) load_sum<DT>(xr, rr, lane + j * LANES, dim, f[j]);
  }
#pragma unroll kHeld
  for (int j = 0; j < steps; ++j) {
    float(&v)[8] = f[CHUNKS ? j : 0];
    const int c = lane + j * LANES;
    if (!CHUNKS) load_sum<DT>(xr, rr, c, dim, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) total = __builtin_fma(static_cast<double>(v[i]), static_cast<double>(v[i]), total);
    if (sr && 8 * c < dim) store8<DT>(v, sr + static_cast<int64_t>(c) * 8 * size_of<DT>(), dim - 8 * c);
  }
  total = row_sum<LANES>(total, part);
  const float r = static_cast<float>(1.0 / sqrt(total / dim + eps));
#pragma unroll kHeld
  for (int j = 0; j < steps; ++j) {
    float(&v)[8] = f[CHUNKS ? j : 0];
    const int c = lane + j * LANES;
    if (!CHUNKS) load_sum<DT>(xr, rr, c, dim, v);
    if (c >= chunks) continue;  // whole quads
    const char* wp = weight + static_cast<int64_t>(c) * 8 * size_of<DT>();
    float w[8] = {};
    if (8 * c + 8 <= dim) {
      load8<DT>(wp, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * c + i < dim) w[i] = element<DT>(wp + i * size_of<DT>());
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = 8 * c + i < dim ? v[i] * r * w[i] : 0.f;
    if (nr && 8 * c < dim) store8<DT>(y, nr + static_cast<int64_t>(c) * 8 * size_of<DT>(), dim - 8 * c);
    if (codes)
      store_rows_chunk(y, c, codes + row * chunks * 8,
                       scales + row * (static_cast<int64_t>((chunks + 63) / 64) * 16));
  }
}

template <int DT>
int launch_norm(const char* x, int64_t xs, const char* res, int64_t rs, int rows, int dim,
                 const char* weight, double eps, char* sum, char* normed, uint8_t* codes,
                 uint8_t* scales, hipStream_t s) {
  const int chunks = tiles(dim) * 16;
  // Wavefronts for short rows; also for 513 to 1,024 columns where there are rows
  // for all of them (with residual, us, workgroups and wavefronts: 1,000 x 800
  // 4.7 / 5.5, 4,000 10.6 / 9.2, 20,000 39 / 30; 20,000 x 2,048 75 / 91).
  const bool four = chunks <= 64 || (chunks <= 128 && rows >= 2048);
  const unsigned grid = four ? (rows - 1) / 4 + 1 : rows;
  if (!grid_fits(grid, kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
#define SF_NORM(LANES, CHUNKS)                                                                   \
  add_rms_norm_kernel<DT, LANES, CHUNKS><<<dim3(grid), dim3(kThreads), 0, s>>>(             \
      x, xs, res, rs, rows, dim, weight, eps, sum, normed, codes, scales)
  if (chunks <= 64)
    SF_NORM(64, 1);
  else if (four)
    SF_NORM(64, 2);
  else if (chunks <= 256)
    SF_NORM(256, 1);
  else if (chunks <= 512)
    SF_NORM(256, 2);
  else if (chunks <= 1024)
    SF_NORM(256, 4);
  else
    SF_NORM(256, 0);
#undef SF_NORM
  SF_LAUNCH_CHECK();
  return SF_OK;
}

template <int DT>
int quantize(const char* x, int64_t row_stride, int64_t batch_stride, int rows, int dim, int batch,
             int held, uint8_t* codes, int64_t codes_batch, uint8_t* scales, int64_t scales_batch,
             hipStream_t s) {
  if (held == kE4m3) {
    const int chunks = tiles(dim) * 16;
    const int64_t total = static_cast<int64_t>(rows) * chunks, groups = (total - 1) / kThreads + 1;
    if (!grid_fits(groups, kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid(static_cast<unsigned>(groups));
    quantize_rows_kernel<DT><<<grid, dim3(kThreads), 0, s>>>(x, row_stride, dim, chunks, total, codes, scales);
  } else {
    const int64_t groups = (static_cast<int64_t>(row_tiles(rows)) * quads(dim) - 1) / (kThreads / SF_WAVE) + 1;
    if (!grid_fits(groups, kThreads) || batch > 65535) return SF_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(batch));
    quantize_weight_kernel<DT><<<grid, dim3(kThreads), 0, s>>>(x, row_stride, batch_stride, rows, dim, codes,
                                                               codes_batch, scales, scales_batch);
  }
  SF_LAUNCH_CHECK();
  return SF_OK;
}

template <int DT>
int values(int held, const uint8_t* codes, const uint8_t* scales, int rows, int dim, char* out,
           hipStream_t s) {
  if (held == kE4m3) {
    const int chunks = tiles(dim) * 16;
    const int64_t total = static_cast<int64_t>(rows) * chunks, groups = (total - 1) / kThreads + 1;
    if (!grid_fits(groups, kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
    rows_values_kernel<DT><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, s>>>(
        codes, scales, dim, chunks, total, out);
  } else {
    const int64_t units = static_cast<int64_t>((rows - 1) / 16 + 1) * tiles(dim);
    const int64_t groups = (units - 1) / (kThreads / SF_WAVE) + 1;
    if (!grid_fits(groups, kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
    weight_values_kernel<DT><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, s>>>(
        codes, scales, rows, dim, out);
  }
  SF_LAUNCH_CHECK();
  return SF_OK;
}

// Columns up to here keep 8 * chunk numbers in 32 bits.
constexpr int kMostColumns = 1 << 30;

}  // namespace

extern "C" int sf_mx_quantize(int dtype, const void* x, int64_t row_stride, int64_t batch_stride,
                              int rows, int dim, int batch, int held, void* codes,
                              int64_t codes_batch_stride, void* scales, int64_t scales_batch_stride,
                              sf_stream_t stream) {
  if (rows < 0 || dim < 1 || batch < 0 || row_stride < 0 || batch_stride < 0 || dtype < kBf16 ||
      dtype > kFp32 || (held != kE4m3 && held != kE2m1) || (held == kE4m3 && batch > 1))
    return SF_ERR_INVALID_ARGUMENT;
  if (dim > kMostColumns) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0 || batch == 0) return SF_OK;
  if (!x || !codes || !scales) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(x, dtype == kFp32 ? 4 : 2) || !aligned(codes, 16) || !aligned(scales, 4) ||
      codes_batch_stride % 16 || scales_batch_stride % 4)
    return SF_ERR_MISALIGNED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const char* xp = static_cast<const char*>(x);
  auto* cp = static_cast<uint8_t*>(codes);
  auto* sp = static_cast<uint8_t*>(scales);
  switch (dtype) {
    case kBf16:
      return quantize<kBf16>(xp, row_stride, batch_stride, rows, dim, batch, held, cp,
                             codes_batch_stride, sp, scales_batch_stride, s);
    case kFp16:
      return quantize<kFp16>(xp, row_stride, batch_stride, rows, dim, batch, held, cp,
                             codes_batch_stride, sp, scales_batch_stride, s);
    default:
      return quantize<kFp32>(xp, row_stride, batch_stride, rows, dim, batch, held, cp,
                             codes_batch_stride, sp, scales_batch_stride, s);
  }
}

extern "C" int sf_mx_values(int held, const void* codes, const void* scales, int rows, int dim,
                            int dtype, void* out, sf_stream_t stream) {
  if (rows < 0 || dim < 1 || dtype < kBf16 || dtype > kFp32 || (held != kE4m3 && held != kE2m1))
    return SF_ERR_INVALID_ARGUMENT;
  if (dim > kMostColumns) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0) return SF_OK;
  if (!codes || !scales || !out) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(codes, 16) || !aligned(out, dtype == kFp32 ? 4 : 2)) return SF_ERR_MISALIGNED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto* cp = static_cast<const uint8_t*>(codes);
  const auto* sp = static_cast<const uint8_t*>(scales);
  char* op = static_cast<char*>(out);
  if (dtype == kBf16) return values<kBf16>(held, cp, sp, rows, dim, op, s);
  if (dtype == kFp16) return values<kFp16>(held, cp, sp, rows, dim, op, s);
  return values<kFp32>(held, cp, sp, rows, dim, op, s);
}

extern "C" int sf_add_rms_norm(int dtype, const void* x, int64_t x_stride, const void* residual,
                               int64_t residual_stride, int rows, int dim, const void* weight,
                               double eps, void* sum, void* normed, void* codes, void* scales,
                               sf_stream_t stream) {
  if (rows < 0 || dim < 1 || dtype < kBf16 || dtype > kFp32 || x_stride < 0 || residual_stride < 0 ||
      !(eps >= 0.0))
    return SF_ERR_INVALID_ARGUMENT;
  if (dim > kMostColumns) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0) return SF_OK;
  if (!x || !weight || !codes != !scales || (sum && !residual) || (!sum && !normed && !codes))
    return SF_ERR_INVALID_ARGUMENT;
  const uintptr_t size = dtype == kFp32 ? 4 : 2;
  if (!aligned(x, size) || !aligned(residual, size) || !aligned(weight, size) || !aligned(sum, size) ||
      !aligned(normed, size) || !aligned(codes, 8))
    return SF_ERR_MISALIGNED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const char *xp = static_cast<const char*>(x), *rp = static_cast<const char*>(residual),
             *wp = static_cast<const char*>(weight);
  char *sp = static_cast<char*>(sum), *np = static_cast<char*>(normed);
  auto *cp = static_cast<uint8_t*>(codes), *kp = static_cast<uint8_t*>(scales);
  if (dtype == kBf16)
    return launch_norm<kBf16>(xp, x_stride, rp, residual_stride, rows, dim, wp, eps, sp, np, cp, kp, s);
  if (dtype == kFp16)
    return launch_norm<kFp16>(xp, x_stride, rp, residual_stride, rows, dim, wp, eps, sp, np, cp, kp, s);
  return launch_norm<kFp32>(xp, x_stride, rp, residual_stride, rows, dim, wp, eps, sp, np, cp, kp, s);
}
