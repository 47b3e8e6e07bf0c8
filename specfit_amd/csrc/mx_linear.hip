// K15: rows times a weight in microscaled 4 bits,
//   out[m, n] = T(sum_k x[m, k] w[n, k] + bias[n]),
// x in e4m3 (rounded here where rows come in 16 bits), w in e2m1.  Products are
// exact, the matrix unit adds a block's in its own fixed order and width and
// accumulates in fp32; the output is rounded once, to bf16 or fp16.
//
// One MI355X (a large copy moves 5.0 TB/s, an 8,192^3 library product in e4m3 runs
// at 2,650 TFLOP/s):
//   1 x 2,048 x 5,120            5.5 us   latency: eight wavefronts cut the sum
//   61 x 2,048 x 151,936        40 us   184 MB, the output among them, at 4.6 TB/s
//   4,096 x 4,096 x 9,216      127 us   2,440 TFLOP/s, near the chip's power
//   8,192^3                    415 us   2,650 TFLOP/s, the library product's rate
#include "mx_product.h"

namespace {

using namespace sf_mx;

struct Linear {
  const void* x;
  const uint8_t* x_scales;
  int64_t x_stride;
  int rows, dim, out_features;
  const uint8_t* codes;
  const uint8_t* scales;
  const void* bias;
  int out_dtype;
  char* out;
  int64_t out_stride;
};

// Four outputs from column n on, with the bias, in the output's type.
__device__ __forceinline__ u32x2 rounded4(const Linear& p, int n, f32x4 v) {
  if (p.bias) {
    for (int i = 0; i < min(4, p.out_features - n); ++i)
      v[i] += p.out_dtype == kFp16 ? element<kFp16>(static_cast<const char*>(p.bias) + 2 * (n + i))
                                   : element<kBf16>(static_cast<const char*>(p.bias) + 2 * (n + i));
  }
  return p.out_dtype == kFp16 ? u32x2{narrow2<kFp16>(v[0], v[1]), narrow2<kFp16>(v[2], v[3])}
                              : u32x2{narrow2<kBf16>(v[0], v[1]), narrow2<kBf16>(v[2], v[3])};
}

// N outputs of 16 bits, two to a word; past the last column nothing.
template <int N, class Words, class Any>
__device__ __forceinline__ void store(const Linear& p, int row, int n, Words w) {
  if (row >= p.rows || n >= p.out_features) return;
  char* o = p.out + (row * p.out_stride + n) * 2;
  if (n + N <= p.out_features) {
    *reinterpret_cast<Any*>(o) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (n + i < p.out_features) reinterpret_cast<uint16_t*>(o)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)));
}

__device__ __forceinline__ void store4(const Linear& p, int row, int n, f32x4 v) {
  store<4, u32x2, u32x2_any>(p, row, n, rounded4(p, n, v));
}

// Few rows: a wavefront takes NT row tiles of the weight and one of KS parts of
// the sum straight from memory; the parts meet in LDS.
template <int MT, int NT, int KS, int WAVES, int XDT>
__global__ __launch_bounds__(WAVES * SF_WAVE) void linear_direct_kernel(Linear p) {
  constexpr int kAhead = MT * NT <= 4 ? 4 : MT * NT <= 8 ? 2 : 1;
  __shared__ f32x4 part[KS > 1 ? WAVES * NT * MT * SF_WAVE : 1];
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4, c = lane & 15;
  const int group = blockIdx.x * (WAVES / KS) + wave / KS;  // of NT row tiles
  const int row_tile_count = row_tiles(p.out_features);
  const int row0 = blockIdx.y * (16 * MT);
  WeightSource w[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    w[n].set(p.codes, p.scales, min(group * NT + n, row_tile_count - 1), p.dim, lane);
  RowSource<XDT> x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    x[m].set(p.x, p.x_scales, min(row0 + 16 * m + c, p.rows - 1), p.x_stride, p.dim, g);
  int begin, end;
  part_of(tiles(p.dim), wave % KS, KS, begin, end);
  f32x4 acc[NT][MT] = {};
  accumulate<MT, NT, XDT, kAhead>(acc, w, x, begin, end, p.dim, g);
  if (KS == 1) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) store4(p, row0 + 16 * m + c, (group * NT + n) * 16 + 4 * g, acc[n][m]);
    return;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) part[(wave * NT * MT + n * MT + m) * SF_WAVE + lane] = acc[n][m];
  __syncthreads();
  // Each group's NT * MT results over its KS wavefronts.
#pragma unroll
  for (int i = 0; i < (NT * MT + KS - 1) / KS; ++i) {
    const int item = i * KS + wave % KS;
    if (item >= NT * MT) break;  // wave-uniform
    f32x4 v = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) v += part[((wave / KS * KS + k) * NT * MT + item) * SF_WAVE + lane];
    store4(p, row0 + item % MT * 16 + c, (group * NT + item / MT) * 16 + 4 * g, v);
  }
}

template <int MT, int NT, int KS, int WAVES, int XDT>
void launch_direct(const Linear& p, hipStream_t s) {
  const int groups = (row_tiles(p.out_features) - 1) / NT + 1, per = WAVES / KS;
  linear_direct_kernel<MT, NT, KS, WAVES, XDT><<<dim3((groups - 1) / per + 1, (p.rows - 1) / (16 * MT) + 1),
                                                 dim3(WAVES * SF_WAVE), 0, s>>>(p);
}

// Many rows: a workgroup takes kRows of them by kOut of the weight's.
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void linear_tiled_kernel(Linear p, int row_groups, int out_groups) {
  __shared__ __attribute__((aligned(16))) typename T::Stage stage0;
  __shared__ __attribute__((aligned(16))) typename T::Stage stage1;
  __shared__ __attribute__((aligned(16))) typename T::Scales scales[2];
  int row_group, out_group;
  tile_of(blockIdx.x, row_groups, out_groups, row_group, out_group);
  const int row0 = row_group * T::kRows, tile0 = out_group * (T::kOut / 16);
  const int last_tile = row_tiles(p.out_features) - 1;
  f32x16 acc[T::FN][T::FM];
  multiply<T>(acc, static_cast<const uint8_t*>(p.x), p.x_scales, p.codes, p.scales, p.dim,
              [&](int r) { return min(row0 + r, p.rows - 1); },
              [&](int i) { return min(tile0 + i, last_tile); }, stage0, stage1, scales);
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int wn = wave / T::WM, wm = wave % T::WM;
#pragma unroll
  for (int m = 0; m < T::FM; ++m) {
    const int row = row0 + (wm * T::FM + m) * 32 + (lane & 31);
#pragma unroll
    for (int n = 0; n < T::FN; ++n)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int n0 = tile0 * 16 + (wn * T::FN + n) * 32 + 8 * i, g = lane >> 5;
        const f32x16& v = acc[n][m];
        u32x2 a = rounded4(p, n0 + 4 * g, f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]});
        u32x2 b = rounded4(p, n0 + 8 + 4 * g, f32x4{v[4 * i + 4], v[4 * i + 5], v[4 * i + 6], v[4 * i + 7]});
        uint32_t w[4] = {a[0], a[1], b[0], b[1]};
        join(w[0], w[2]);
        join(w[1], w[3]);
        store<8, u32x4, u32x4_any>(p, row, n0 + 8 * g, u32x4{w[0], w[1], w[2], w[3]});
      }
  }
}

template <class T>
int launch_tiled(const Linear& p, hipStream_t s) {
  const int row_groups = (p.rows - 1) / T::kRows + 1, out_groups = (p.out_features - 1) / T::kOut + 1;
  if (!grid_fits(static_cast<int64_t>(row_groups) * out_groups, T::kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
  linear_tiled_kernel<T><<<dim3(row_groups * out_groups), dim3(T::kThreads), 0, s>>>(p, row_groups, out_groups);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

// Rows of 16-bit values are rounded by every wavefront that reads them where that
// is cheaper than a launch of its own: one tile of rows and few wavefronts.  us on
// the device, as they are and with the launch (4 more on the host):
//   1 row of 2,048 by 5,120   5.4 / 6.0   16,384   9.4 / 7.5   40,000   22 / 13.5   151,936   77 / 36
//   16 rows                   7.2 / 7.2           12.2 / 8.7            30 / 15.4            103 / 37
constexpr int64_t kMostRawWeight = 1 << 25;  // values

bool as_they_are(int rows, int dim, int out_features) {
  return rows <= SF_MX_RAW_ROWS && dim % 8 == 0 && static_cast<int64_t>(dim) * out_features <= kMostRawWeight;
}

int64_t groups(int n, int per) { return (n - 1) / per + 1; }

// Few rows, or too small a product for tiles: 16 or 32 rows by NT row tiles of
// the weight in a workgroup of KS wavefronts that cut the sum, so that some
// thousand wavefronts have loads under way.  More row tiles to a wavefront where
// rows are read for each of them again (us, rows x dim x outputs; 1, 2 and 4 row
// tiles of 16 rows, then 4 of 32):
//   1 x 2,048 x 2,048     4.2   3.6   5.3          64 x 2,048 x 2,048     5.5   4.5   6.3   6.9
//   1 x 2,048 x 20,000    6.4   6.4   8.9          64 x 2,048 x 5,120    10.3   7.9   7.3   7.1
//   16 x 2,048 x 16,384   8.8   6.4   7.5          32 x 4,096 x 9,216    17.7  13.2  11.3  11.0
template <int XDT>
int launch_few(const Linear& p, hipStream_t s) {
  const int64_t units = groups(p.rows, 16) * row_tiles(p.out_features);
  if (XDT == kRows && p.rows > 16 && units >= 2048)
    launch_direct<2, 4, 4, 4, kRows>(p, s);
  else if (XDT == kRows && p.rows > 16 && units >= 1024)
    launch_direct<1, 4, 4, 4, kRows>(p, s);
  else if (units >= 128)
    launch_direct<1, 2, 8, 8, XDT>(p, s);
  else
    launch_direct<1, 1, 8, 8, XDT>(p, s);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

// Tiles where they make work for the 256 CUs, the larger the better they fill
// them; at most 2 workgroups of the largest run on a CU together, 4 of the others.
// us; direct form, then tiles of 32 x 128, 64 x 64, 64 x 128 and 128 x 256 rows and
// outputs:
//   16 x 2,048 x 40,000    12.9  13.5  13.5  14.2         16 x 2,048 x 80,000    22.7  19.5  19.8  19.5
//   32 x 2,048 x 16,384     8.1   9.1   8.4   9.7         32 x 2,048 x 32,768    12.6  12.5  12.7  13.1
//   256 x 2,048 x 2,048     7.0   8.4   7.8   9.1         128 x 2,048 x 5,120     9.2   8.9   8.3   9.6
//   1,024 x 2,048 x 2,048         10.4   9.3  10.0        1,024 x 2,048 x 5,120         18.2  18.3  16.8  19.9
//   2,048 x 4,096 x 9,216               101.9  81.3  86.4     (576 of the largest)
//   1,536 x 4,096 x 9,216                78.2  61.4  56.1     (432)
//   8,192 x 2,048 x 2,048                48.6  40.4  35.0     (512)
int launch_rows(const Linear& p, hipStream_t s) {
  constexpr int kCus = 256;
  const int m = p.rows, n = p.out_features;
  if (m <= 32) {
    if (groups(n, 128) >= (m <= 16 ? 2 * kCus : kCus)) return launch_tiled<Tiling<2, 1, 2, 1>>(p, s);
    return launch_few<kRows>(p, s);
  }
  const int64_t large = groups(m, 128) * groups(n, 256);
  // The largest in one nearly full round, or in several.
  if (m > 64 && (large >= 4 * kCus || (large <= 2 * kCus && large * 5 >= 2 * kCus * 4)))
    return launch_tiled<Tiling<2, 2, 4, 2>>(p, s);
  if (groups(m, 64) * groups(n, 128) >= 2 * kCus) return launch_tiled<Tiling<2, 2, 2, 1>>(p, s);
  if (groups(m, 64) * groups(n, 64) >= kCus * 5 / 8) return launch_tiled<Tiling<2, 2, 1, 1>>(p, s);
  return launch_few<kRows>(p, s);
}

// 32-bit element and tile numbers within a row, and the largest tiles' grid: that
// of the smaller ones, which run where few of these would, is far within its limit.
bool supported(int rows, int dim, int out_features) {
  return dim <= 1 << 24 && out_features <= 1 << 28 && rows <= 1 << 20 &&
         grid_fits(groups(rows, 128) * groups(out_features, 256), Tiling<2, 2, 4, 2>::kThreads);
}

}  // namespace

extern "C" int64_t sf_mx_linear_workspace(int x_dtype, int rows, int dim, int out_features) {
  if (rows < 0 || dim < 1 || out_features < 1 || (x_dtype != kBf16 && x_dtype != kFp16 && x_dtype != kRows) ||
      !supported(rows, dim, out_features))
    return -1;
  if (x_dtype == kRows || as_they_are(rows, dim, out_features)) return 0;
  return rows * (static_cast<int64_t>(tiles(dim)) * kTile + static_cast<int64_t>(quads(dim)) * 16);
}

extern "C" int sf_mx_linear(int x_dtype, const void* x, const void* x_scales, int64_t x_stride, int rows,
                            int dim, const void* codes, const void* scales, int out_features,
                            const void* bias, int out_dtype, void* out, int64_t out_stride, void* workspace,
                            sf_stream_t stream) {
  if (rows < 0 || dim < 1 || out_features < 1 || x_stride < 0 || out_stride < out_features ||
      (out_dtype != kBf16 && out_dtype != kFp16) ||
      (x_dtype != kBf16 && x_dtype != kFp16 && x_dtype != kRows))
    return SF_ERR_INVALID_ARGUMENT;
  if (!supported(rows, dim, out_features)) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0) return SF_OK;
  if (!x || !codes || !scales || !out || (x_dtype == kRows && !x_scales)) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(out, 2) || !aligned(bias, 2) || !aligned(workspace, 16) ||
      !aligned(x_scales, 16))
    return SF_ERR_MISALIGNED;
  const bool fits = aligned(x, 16) && x_stride % 8 == 0;
  if (x_dtype == kRows) {
    if (!aligned(x, 16)) return SF_ERR_MISALIGNED;
  } else if (workspace && (!fits || !as_they_are(rows, dim, out_features))) {
    uint8_t* held = static_cast<uint8_t*>(workspace);
    uint8_t* held_scales = held + rows * (static_cast<int64_t>(tiles(dim)) * kTile);
    if (const int rc = sf_mx_quantize(x_dtype, x, x_stride, 0, rows, dim, 1, kE4m3, held, 0, held_scales, 0, stream))
      return rc;
    x_dtype = kRows;
    x = held;
    x_scales = held_scales;
  } else if (rows > SF_MX_RAW_ROWS) {
    return SF_ERR_UNSUPPORTED_SHAPE;
  } else if (!fits || dim % 8) {
    return SF_ERR_MISALIGNED;
  }
  const Linear p = {x, static_cast<const uint8_t*>(x_scales), x_stride, rows, dim, out_features,
                    static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), bias,
                    out_dtype, static_cast<char*>(out), out_stride};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (x_dtype == kBf16) return launch_few<kBf16>(p, s);
  if (x_dtype == kFp16) return launch_few<kFp16>(p, s);
  return launch_rows(p, s);
}
