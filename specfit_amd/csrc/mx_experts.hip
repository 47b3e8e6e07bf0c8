// K16: grouped SwiGLU experts with weights in microscaled 4 bits, over the rows
// that K2 dispatched.  For expert e's rows r (token t = perm_pos[r] / top_k):
//   g = x[t] . gate^T, u = x[t] . up^T        x in e4m3
//   a = e4m3(silu(g) u)                       blocks of 32 of the inner size
//   rows[r] = bf16((a . down^T) * route_weight)
// with fp32 sums and one rounding between them: the activation is what the
// second product reads, so it is rounded once, from fp32, to that product's
// type.  The rows are bf16 as K3's are, for K4.  A layer's experts in one call keep
// them in 16 bits of their own kind, with three bits more, and round to bf16 once,
// behind the sum over a token's routes (0.0017 to 0.0019 of the outputs' norm
// against 64 bits; 0.0024 to 0.0026 with bf16 rows); without a dispatch that sum
// is in fp32 throughout.
//
// 128 experts of 2,048 x 768, 8 to a token, one MI355X; gate and up, then down:
//   1 token (no dispatch)        7.6 + 5.6 us   latency of two dependent launches
//   61 tokens, favourites         36 + 21 us    4.2 and 3.6 TB/s of weights
//   2,048 tokens                  76 + 57 us    1.4 and 0.9 PFLOP/s, the weights' 214
//                                               and 107 MB arriving meanwhile
// and the sum over the routes 4.6 and 13.4 us (77 MB at 5.7 TB/s).
#include <cmath>

#include "dispatch.h"
#include "mx_product.h"

namespace {

using namespace sf_mx;

// The parts of an expert's record: codes of gate, up and down, then their
// scales in that order.
struct Record {
  int64_t up_codes, down_codes, gate_scales, up_scales, down_scales, bytes;
};

Record record_of(int hidden, int inner) {
  Record r;
  r.up_codes = weight_code_bytes(inner, hidden);
  r.down_codes = 2 * r.up_codes;
  r.gate_scales = r.down_codes + weight_code_bytes(hidden, inner);
  r.up_scales = r.gate_scales + weight_scale_bytes(inner, hidden);
  r.down_scales = r.up_scales + weight_scale_bytes(inner, hidden);
  r.bytes = r.down_scales + weight_scale_bytes(hidden, inner);
  return r;
}

struct Experts {
  const void* x;
  const uint8_t* x_scales;
  int64_t x_stride;
  const int32_t* perm_pos;
  const int32_t* offsets;
  const uint16_t* route_weights;
  int top_k, hidden, inner, num_experts;
  const int32_t* slot_of_expert;
  const uint8_t* slots;
  int64_t slot_stride;
  Record record;
  uint8_t* act;         // e4m3 rows [tokens * top_k, inner]
  uint8_t* act_scales;
  uint16_t* rows;       // [tokens * top_k, hidden], bf16 or held in blocks (below)
  uint8_t* row_scales;  // of rows held in blocks: [tokens * top_k, ceil(hidden / 32)]
};

// The rows of one workgroup: up to PER of one expert's.  The chunks of more than
// LIGHT rows come first, expert by expert, then the others, so that the short
// ones fill the gaps at a launch's end.  Every wavefront finds chunk `id` from the
// dispatch's offsets: a lane counts the chunks of four experts, a scan over the
// lanes places them.
struct Chunk {
  const uint8_t* weights;  // null: there is no such chunk
  int begin, end;          // its rows
};

template <int PER, int LIGHT>
__device__ __forceinline__ Chunk chunk_of(const Experts& p, int id) {
  constexpr int kEach = SF_MAX_EXPERTS / SF_WAVE;
  const int lane = threadIdx.x & (SF_WAVE - 1);
  int first[kEach + 1], slot[kEach];
#pragma unroll
  for (int i = 0; i <= kEach; ++i) first[i] = p.offsets[min(lane * kEach + i, p.num_experts)];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = min(lane * kEach + i, p.num_experts - 1);
    slot[i] = p.slot_of_expert ? p.slot_of_expert[e] : e;
  }
  const auto count = [&](int i, bool light) {
    const int rows = slot[i] >= 0 ? first[i + 1] - first[i] : 0, over = rows % PER;
    return light ? static_cast<int>(over > 0 && over <= LIGHT) : rows / PER + (over > LIGHT);
  };
  bool light = false;
#pragma unroll
  for (int pass = 0; pass < (LIGHT ? 2 : 1); ++pass) {
    light = pass;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += count(i, light);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < SF_WAVE; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const uint64_t past = __ballot(upto > id);
    if (past == 0) {
      id -= __builtin_amdgcn_readlane(upto, SF_WAVE - 1);
      continue;
    }
    const int owner = __builtin_ctzll(past);
    int own_slot = 0, begin = 0, end = 0, before = 0;
    const int at = id - (upto - mine);  // of the owner's chunks
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int here = count(i, light);
      if (at >= before && at < before + here) {
        own_slot = slot[i];
        end = first[i + 1];
        begin = light ? end - (end - first[i]) % PER : first[i] + (at - before) * PER;
      }
      before += here;
    }
    own_slot = __builtin_amdgcn_readlane(own_slot, owner);
    begin = __builtin_amdgcn_readlane(begin, owner);
    end = min(__builtin_amdgcn_readlane(end, owner), begin + PER);
    return {p.slots + own_slot * p.slot_stride, begin, end};
  }
  return {nullptr, 0, 0};
}

// At most this many chunks.
int64_t most_chunks(int64_t routes, int experts, int per) {
  return min(routes, static_cast<int64_t>(experts)) + routes / per;
}

__device__ __forceinline__ float swiglu(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }

// Where row `row` of the activations and the scale byte of its block lie.
__device__ __forceinline__ uint8_t* act_row(const Experts& p, int row) {
  return p.act + row * (static_cast<int64_t>(tiles(p.inner)) * kTile);
}
__device__ __forceinline__ uint8_t* act_scale(const Experts& p, int row, int block) {
  return p.act_scales + row * (static_cast<int64_t>(quads(p.inner)) * 16) + block / 16 * 16 + block % 4 * 4 +
         block / 4 % 4;
}

// 32 columns of gate and up for 16 rows of one expert, the hidden size cut over
// the workgroup's wavefronts, so that the 32 activations are one block of the
// next product's rows.  Lane c of sixteen: x's row x_row, to row `row` of the
// activations where `live`.
template <int WAVES, int XDT, int AHEAD>
__device__ __forceinline__ void gate_up_block(const Experts& p, const uint8_t* weights, int block, int64_t x_row,
                                              int row, bool live, f32x4* part) {
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4;
  if (block * kBlock >= p.inner) {  // behind the activations' end, within their last tile: zeros
    if (wave == 0 && live) {
      *reinterpret_cast<u32x2*>(act_row(p, row) + block * kBlock + 8 * g) = u32x2{0u, 0u};
      if (g == 0) *act_scale(p, row, block) = 0;
    }
    return;
  }
  WeightSource w[4];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    w[n].set(weights, weights + p.record.gate_scales, 2 * block + n, p.hidden, lane);
    w[2 + n].set(weights + p.record.up_codes, weights + p.record.up_scales, 2 * block + n, p.hidden, lane);
  }
  RowSource<XDT> x[1];
  x[0].set(p.x, p.x_scales, x_row, p.x_stride, p.hidden, g);
  int begin, end;
  part_of(tiles(p.hidden), wave, WAVES, begin, end);
  f32x4 acc[4][1] = {};
  accumulate<1, 4, XDT, AHEAD>(acc, w, x, begin, end, p.hidden, g);
#pragma unroll
  for (int n = 0; n < 4; ++n) part[(wave * 4 + n) * SF_WAVE + lane] = acc[n][0];
  __syncthreads();
  if (wave > 0) return;
  f32x4 v[4] = {};
#pragma unroll
  for (int k = 0; k < WAVES; ++k)
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] += part[(k * 4 + n) * SF_WAVE + lane];
  float a[8];  // of row c: columns 4 g .. + 3 and 16 + 4 g .. + 3 of the block
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = swiglu(v[i / 4][i % 4], v[2 + i / 4][i % 4]);
    top = max(top, magnitude(a[i]));
  }
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
  const uint32_t byte = scale_byte<kE4m3>(top);
  const float s = byte == 255 ? 0.f : inverse_scale(byte);
  if (live) {
    uint8_t* o = act_row(p, row) + block * kBlock + 4 * g;
    *reinterpret_cast<uint32_t*>(o) = byte == 255 ? 0u : e4m3x4(a[0] * s, a[1] * s, a[2] * s, a[3] * s);
    *reinterpret_cast<uint32_t*>(o + 16) = byte == 255 ? 0u : e4m3x4(a[4] * s, a[5] * s, a[6] * s, a[7] * s);
    if (g == 0) *act_scale(p, row, block) = static_cast<uint8_t>(byte);
  }
}

// Few rows, as they come: a workgroup takes 16 of one expert's.
template <int WAVES, int XDT>
__global__ __launch_bounds__(WAVES * SF_WAVE) void gate_up_few_kernel(Experts p, int blocks) {
  __shared__ f32x4 part[WAVES * 4 * SF_WAVE];
  const Chunk chunk = chunk_of<16, 0>(p, blockIdx.x / blocks);
  if (!chunk.weights) return;
  const int c = threadIdx.x & 15;
  const int row = min(chunk.begin + c, chunk.end - 1);
  gate_up_block<WAVES, XDT, 2>(p, chunk.weights, blockIdx.x % blocks, p.perm_pos[row] / p.top_k, row,
                               chunk.begin + c < chunk.end, part);
}

// A route's row on its way to the sum over a token's routes: bf16 for callers, and
// for this file's own sum fp16 in blocks of 32 columns with a power of two, E - 141
// its exponent: as many bytes, and three bits more.  E is the biased exponent of
// the block's largest finite value, at least 15, so that that value becomes 2^14 to
// 2^15, nothing is lost down to 2^-28 of it, and both factors are normal.
// Infinities and NaN stay what they are.  2,048 tokens: down 53 us with bf16 rows,
// 55 to 57 so (60 with E by the lanes' exchange through LDS and byte stores).
constexpr int kHeldRows = 4;

__device__ __forceinline__ uint32_t row_exponent(uint32_t top) { return max(top >> 23, 15u); }
__device__ __forceinline__ float to_row(uint32_t e) { return __uint_as_float((268u - e) << 23); }
__device__ __forceinline__ float from_row(uint32_t e) { return __uint_as_float((e - 14u) << 23); }

// The larger of this lane's and the lane's that differs in bit 4 or 5 of its number.
__device__ __forceinline__ float max16(float x) {
  const u32x2 both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float max32(float x) {
  const u32x2 both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// The largest magnitude of N values; NaN are passed over, with FINITE infinities too.
template <int N, bool FINITE, class Values>
__device__ __forceinline__ float largest(const Values& v) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    top = fmaxf(top, FINITE && magnitude(v[i]) >= 0x7f800000u ? 0.f : fabsf(v[i]));
  return top;
}

__device__ __forceinline__ uint8_t* row_scale(const Experts& p, int row, int h) {
  return p.row_scales + row * static_cast<int64_t>((p.hidden + kBlock - 1) / kBlock) + h / kBlock;
}

// The bytes of N blocks from column h on.
typedef uint32_t __attribute__((aligned(1))) u32_any;
typedef uint16_t __attribute__((aligned(1))) u16_any;

template <int N>
__device__ __forceinline__ void store_scales(const Experts& p, int row, int h, uint32_t bytes) {
  static_assert(N == 4 || N == 2, "a word or half of one");
  uint8_t* o = row_scale(p, row, h);
  if (h + 32 * (N - 1) < p.hidden) {
    if (N == 4)
      *reinterpret_cast<u32_any*>(o) = bytes;
    else
      *reinterpret_cast<u16_any*>(o) = static_cast<uint16_t>(bytes);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (h + 32 * i < p.hidden) o[i] = static_cast<uint8_t>(bytes >> (8 * i));
}

// Columns from h on, two to a word.
template <int N, class Words, class Any>
__device__ __forceinline__ void store_row(const Experts& p, int row, int h, Words w) {
  uint16_t* o = p.rows + static_cast<int64_t>(row) * p.hidden + h;
  if (h + N <= p.hidden) {
    *reinterpret_cast<Any*>(o) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (h + i < p.hidden) o[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)));
}

__device__ __forceinline__ float route_weight(const Experts& p, int row) {
  return p.route_weights ? sf_bf16_to_f32(p.route_weights[p.perm_pos[row]]) : 1.0f;
}

// A wavefront: 32 columns of down for 16 rows, over the whole inner size.
template <int WAVES, int HELD>
__global__ __launch_bounds__(WAVES * SF_WAVE) void down_few_kernel(Experts p, int blocks) {
  const Chunk chunk = chunk_of<16, 0>(p, blockIdx.x / blocks);
  if (!chunk.weights) return;
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4, c = lane & 15;
  const int pair = blockIdx.x % blocks * WAVES + wave;  // of row tiles, which come in pairs
  if (2 * pair >= row_tiles(p.hidden)) return;
  WeightSource w[2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
    w[n].set(chunk.weights + p.record.down_codes, chunk.weights + p.record.down_scales, 2 * pair + n, p.inner, lane);
  const int row = min(chunk.begin + c, chunk.end - 1);
  RowSource<kRows> x[1];
  x[0].set(p.act, p.act_scales, row, 0, p.inner, g);
  const float route = route_weight(p, row);
  f32x4 acc[2][1] = {};
  accumulate<1, 2, kRows, 3>(acc, w, x, 0, tiles(p.inner), p.inner, g);
#pragma unroll
  for (int n = 0; n < 2; ++n) acc[n][0] *= route;
  uint32_t e = 0;
  if (HELD == kHeldRows) {
    const float v[8] = {acc[0][0][0], acc[0][0][1], acc[0][0][2], acc[0][0][3],
                        acc[1][0][0], acc[1][0][1], acc[1][0][2], acc[1][0][3]};
    float top = max32(max16(largest<8, false>(v)));
    if (__any(magnitude(top) == 0x7f800000u)) top = max32(max16(largest<8, true>(v)));
    e = row_exponent(__float_as_uint(top));
  }
  if (chunk.begin + c >= chunk.end) return;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const f32x4 v = HELD == kHeldRows ? acc[n][0] * to_row(e) : acc[n][0];
    constexpr int DT = HELD == kHeldRows ? kFp16 : kBf16;
    store_row<4, u32x2, u32x2_any>(p, row, 32 * pair + 16 * n + 4 * g,
                                   u32x2{narrow2<DT>(v[0], v[1]), narrow2<DT>(v[2], v[3])});
  }
  if (HELD == kHeldRows && g == 0) *row_scale(p, row, 32 * pair) = static_cast<uint8_t>(e);
}

// Many rows by tiles.  Half of a wavefront's weight rows are gate's, the other
// half the same of up's.
template <class T>
__device__ __forceinline__ void gate_up_tile(const Experts& p, const Chunk& chunk, int col0, typename T::Stage& stage0,
                                             typename T::Stage& stage1, typename T::Scales (&scales)[2]) {
  const int up_tiles = row_tiles(p.inner);
  f32x16 acc[T::FN][T::FM];
  multiply<T>(acc, static_cast<const uint8_t*>(p.x), p.x_scales, chunk.weights,
              chunk.weights + p.record.gate_scales, p.hidden,
              [&](int r) { return p.perm_pos[min(chunk.begin + r, chunk.end - 1)] / p.top_k; },
              [&](int i) {
                const int wn = i / (2 * T::FN), j = i % (2 * T::FN);
                const int tile = min(col0 / 16 + wn * T::FN + j % T::FN, up_tiles - 1);
                return j < T::FN ? tile : up_tiles + tile;
              },
              stage0, stage1, scales);
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int wn = wave / T::WM, wm = wave % T::WM, g = lane >> 5;
#pragma unroll
  for (int m = 0; m < T::FM; ++m) {
    const int row = chunk.begin + (wm * T::FM + m) * 32 + (lane & 31);
#pragma unroll
    for (int n = 0; n < T::FN / 2; ++n) {
      const int block = col0 / kBlock + wn * (T::FN / 2) + n;
      const bool held = block * kBlock < p.inner;
      float a[16];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        a[i] = held ? swiglu(acc[n][m][i], acc[T::FN / 2 + n][m][i]) : 0.f;
        top = max(top, magnitude(a[i]));
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      const uint32_t byte = scale_byte<kE4m3>(top);
      const float s = byte == 255 ? 0.f : inverse_scale(byte);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = byte == 255 ? 0u : e4m3x4(a[4 * i] * s, a[4 * i + 1] * s, a[4 * i + 2] * s, a[4 * i + 3] * s);
      join(w[0], w[1]);
      join(w[2], w[3]);
      if (row < chunk.end && block < tiles(p.inner) * 4) {
        uint8_t* o = act_row(p, row) + block * kBlock + 8 * g;
        *reinterpret_cast<u32x2*>(o) = u32x2{w[0], w[1]};
        *reinterpret_cast<u32x2*>(o + 16) = u32x2{w[2], w[3]};
        if (g == 0) *act_scale(p, row, block) = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <int HELD, class T>
__device__ __forceinline__ void down_tile(const Experts& p, const Chunk& chunk, int tile0, typename T::Stage& stage0,
                                          typename T::Stage& stage1, typename T::Scales (&scales)[2]) {
  const int last = row_tiles(p.hidden) - 1;
  f32x16 acc[T::FN][T::FM];
  multiply<T>(acc, p.act, p.act_scales, chunk.weights + p.record.down_codes, chunk.weights + p.record.down_scales,
              p.inner, [&](int r) { return min(chunk.begin + r, chunk.end - 1); },
              [&](int i) { return min(tile0 + i, last); }, stage0, stage1, scales);
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int wn = wave / T::WM, wm = wave % T::WM;
#pragma unroll
  for (int m = 0; m < T::FM; ++m) {
    const int row = chunk.begin + (wm * T::FM + m) * 32 + (lane & 31);
    const bool live = row < chunk.end;
    const float route = live ? route_weight(p, row) : 0.f;
    const int first = tile0 * 16 + wn * T::FN * 32;
    // The weight by itself, not with the block's power of two: of a block of zeros
    // that is 2^126, and the two factors' product infinite from a weight of 4 on.
#pragma unroll
    for (int n = 0; n < T::FN; ++n) acc[n][m] *= route;
    float top[T::FN];
    uint32_t scales_word = 0;
    if (HELD == kHeldRows) {
      bool infinite = false;
#pragma unroll
      for (int n = 0; n < T::FN; ++n) {
        top[n] = max32(largest<16, false>(acc[n][m]));
        infinite |= magnitude(top[n]) == 0x7f800000u;
      }
      if (__any(infinite)) {
#pragma unroll
        for (int n = 0; n < T::FN; ++n) top[n] = max32(largest<16, true>(acc[n][m]));
      }
    }
#pragma unroll
    for (int n = 0; n < T::FN; ++n) {
      const int h0 = first + n * 32;
      f32x16 v = acc[n][m];
      if (HELD == kHeldRows) {
        const uint32_t e = row_exponent(__float_as_uint(top[n]));
        v *= to_row(e);
        scales_word |= e << (8 * n);
      }
      constexpr int DT = HELD == kHeldRows ? kFp16 : kBf16;
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t w[4] = {narrow2<DT>(v[4 * i], v[4 * i + 1]), narrow2<DT>(v[4 * i + 2], v[4 * i + 3]),
                         narrow2<DT>(v[4 * i + 4], v[4 * i + 5]), narrow2<DT>(v[4 * i + 6], v[4 * i + 7])};
        join(w[0], w[2]);
        join(w[1], w[3]);
        if (live)
          store_row<8, u32x4, u32x4_any>(p, row, h0 + 8 * i + 8 * (lane >> 5), u32x4{w[0], w[1], w[2], w[3]});
      }
    }
    if (HELD == kHeldRows && live && lane < 32) store_scales<T::FN>(p, row, first, scales_word);
  }
}

// A chunk's workgroup takes the lowest of its tilings that holds its rows: an
// expert's last chunk is rarely full.  All have the same wavefronts and weight
// rows, the tallest first.
template <class T, class...>
struct First {
  using type = T;
};

constexpr int kGateUp = -1;  // a product: gate and up, or down with rows of this type

template <int PART, class T, class... Lower>
__device__ __forceinline__ void fitting_tile(const Experts& p, const Chunk& chunk, int out0, void* stage0, void* stage1,
                                             void* scales) {
  if constexpr (sizeof...(Lower) > 0) {
    if (chunk.end - chunk.begin <= First<Lower...>::type::kRows) {
      fitting_tile<PART, Lower...>(p, chunk, out0, stage0, stage1, scales);
      return;
    }
  }
  auto& s0 = *static_cast<typename T::Stage*>(stage0);
  auto& s1 = *static_cast<typename T::Stage*>(stage1);
  auto& sc = *static_cast<typename T::Scales(*)[2]>(scales);
  if constexpr (PART == kGateUp)
    gate_up_tile<T>(p, chunk, out0, s0, s1, sc);
  else
    down_tile<PART, T>(p, chunk, out0, s0, s1, sc);
}

// What counts as a short chunk: rows that a lower tiling holds (us, chunks in turn
// and sorted: 2,048 tokens of 128 experts 165 / 153, of 64 experts 126 / 118).
template <class... Lower>
constexpr int light_rows() {
  if constexpr (sizeof...(Lower) > 0)
    return First<Lower...>::type::kRows;
  else
    return 0;
}

template <int PART, class T, class... Lower>
__global__ __launch_bounds__(T::kThreads, 2) void experts_tiled_kernel(Experts p, int blocks) {
  static_assert(((Lower::kThreads == T::kThreads && Lower::kOut == T::kOut && Lower::kRows < T::kRows) && ...), "");
  __shared__ __attribute__((aligned(16))) typename T::Stage stage0;
  __shared__ __attribute__((aligned(16))) typename T::Stage stage1;
  __shared__ __attribute__((aligned(16))) typename T::Scales scales[2];
  // Eight chunks in turn: neighbouring workgroups run on different XCDs, so a
  // chunk's stay on one and read its rows from one L2.
  const int id = blockIdx.x / kXcds;
  const Chunk chunk = chunk_of<T::kRows, light_rows<Lower...>()>(p, id / blocks * kXcds + blockIdx.x % kXcds);
  if (!chunk.weights) return;
  const int out0 = id % blocks * (PART == kGateUp ? T::kOut / 2 : T::kOut / 16);
  fitting_tile<PART, T, Lower...>(p, chunk, out0, &stage0, &stage1, &scales);
}

// ------------------------------------------------ a token's own few routes --
// Routes that hardly share experts, without a dispatch: each multiplies its
// token's row by its expert's weights, the second kernel adds a token's up.
struct Routes {
  const int64_t* index;
  const uint16_t* weights;
  uint16_t* out;  // bf16 [tokens, hidden]
};

__device__ __forceinline__ const uint8_t* weights_of(const Experts& p, int64_t e) {
  if (e < 0 || e >= p.num_experts) return nullptr;
  const int slot = p.slot_of_expert ? p.slot_of_expert[e] : static_cast<int>(e);
  return slot < 0 ? nullptr : p.slots + slot * p.slot_stride;
}

template <int WAVES, int XDT>
__global__ __launch_bounds__(WAVES * SF_WAVE) void routed_gate_up_kernel(Experts p, Routes r, int blocks) {
  __shared__ f32x4 part[WAVES * 4 * SF_WAVE];
  const int route = blockIdx.x / blocks;
  const uint8_t* weights = weights_of(p, r.index[route]);
  if (!weights) return;
  gate_up_block<WAVES, XDT, 2>(p, weights, blockIdx.x % blocks, route / p.top_k, route, (threadIdx.x & 15) == 0, part);
}

// A workgroup: 16 columns of one token's output.  Its wavefronts take the
// routes in turn, and parts of the inner size where there are fewer routes.
template <int WAVES>
__global__ __launch_bounds__(WAVES * SF_WAVE) void routed_down_kernel(Experts p, Routes r, int cuts) {
  __shared__ float part[WAVES][16];
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4;
  const int all = row_tiles(p.hidden), token = blockIdx.x / all, tile = blockIdx.x % all;
  f32x4 sum = {};
  for (int item = wave; item < p.top_k * cuts; item += WAVES) {  // wave-uniform
    const int route = token * p.top_k + item / cuts;
    const uint8_t* weights = weights_of(p, r.index[route]);
    if (!weights) continue;
    WeightSource w[1];
    w[0].set(weights + p.record.down_codes, weights + p.record.down_scales, tile, p.inner, lane);
    RowSource<kRows> x[1];
    x[0].set(p.act, p.act_scales, route, 0, p.inner, g);
    int begin, end;
    part_of(tiles(p.inner), item % cuts, cuts, begin, end);
    f32x4 acc[1][1] = {};
    accumulate<1, 1, kRows, 6>(acc, w, x, begin, end, p.inner, g);
    sum += acc[0][0] * sf_bf16_to_f32(r.weights[route]);
  }
  if ((lane & 15) == 0)
    for (int i = 0; i < 4; ++i) part[wave][4 * g + i] = sum[i];
  __syncthreads();
  if (threadIdx.x < 16) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) v += part[k][threadIdx.x];
    const int h = tile * 16 + threadIdx.x;
    if (h < p.hidden) r.out[static_cast<int64_t>(token) * p.hidden + h] = sf_f32_to_bf16(v);
  }
}

int groups(int n, int per) { return (n - 1) / per + 1; }

// What a launcher does: kCheck only asks whether its grids fit, so that an entry
// point refuses a call before the first of its launches.
enum Do { kCheck, kLaunch };

template <int WAVES, int XDT>
int gate_up_few(const Experts& p, int64_t routes, Do what, hipStream_t s) {
  const int blocks = tiles(p.inner) * 4;
  const int64_t grid = most_chunks(routes, p.num_experts, 16) * blocks;
  if (!grid_fits(grid, WAVES * SF_WAVE)) return SF_ERR_UNSUPPORTED_SHAPE;
  if (what == kCheck) return SF_OK;
  gate_up_few_kernel<WAVES, XDT><<<dim3(static_cast<unsigned>(grid)), dim3(WAVES * SF_WAVE), 0, s>>>(p, blocks);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

template <int WAVES, int HELD>
int down_few(const Experts& p, int64_t routes, Do what, hipStream_t s) {
  const int blocks = groups(row_tiles(p.hidden) / 2, WAVES);
  const int64_t grid = most_chunks(routes, p.num_experts, 16) * blocks;
  if (!grid_fits(grid, WAVES * SF_WAVE)) return SF_ERR_UNSUPPORTED_SHAPE;
  if (what == kCheck) return SF_OK;
  down_few_kernel<WAVES, HELD><<<dim3(static_cast<unsigned>(grid)), dim3(WAVES * SF_WAVE), 0, s>>>(p, blocks);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

template <int PART, class T, class... Lower>
int tiled(const Experts& p, int64_t routes, Do what, hipStream_t s) {
  const int blocks = PART == kGateUp ? groups(tiles(p.inner) * 4, T::kOut / 64) : groups(p.hidden, T::kOut);
  const int64_t chunks = (most_chunks(routes, p.num_experts, T::kRows) + kXcds - 1) / kXcds * kXcds;
  if (!grid_fits(chunks * blocks, T::kThreads)) return SF_ERR_UNSUPPORTED_SHAPE;
  if (what == kCheck) return SF_OK;
  experts_tiled_kernel<PART, T, Lower...>
      <<<dim3(static_cast<unsigned>(chunks * blocks)), dim3(T::kThreads), 0, s>>>(p, blocks);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

using Tiles32 = Tiling<4, 1, 2, 1>;
using Tiles64 = Tiling<4, 1, 2, 2>;
using Tiles128 = Tiling<2, 2, 4, 2>;

template <int WAVES, int XDT>
int routed(const Experts& p, const Routes& r, int64_t routes, Do what, hipStream_t s) {
  const int blocks = tiles(p.inner) * 4;
  const int64_t down = routes / p.top_k * row_tiles(p.hidden);
  if (!grid_fits(routes * blocks, WAVES * SF_WAVE) || !grid_fits(down, WAVES * SF_WAVE))
    return SF_ERR_UNSUPPORTED_SHAPE;
  if (what == kCheck) return SF_OK;
  routed_gate_up_kernel<WAVES, XDT>
      <<<dim3(static_cast<unsigned>(routes * blocks)), dim3(WAVES * SF_WAVE), 0, s>>>(p, r, blocks);
  SF_LAUNCH_CHECK();
  routed_down_kernel<WAVES>
      <<<dim3(static_cast<unsigned>(down)), dim3(WAVES * SF_WAVE), 0, s>>>(p, r, max(1, WAVES / p.top_k));
  SF_LAUNCH_CHECK();
  return SF_OK;
}

// Both products over dispatched rows.
template <int HELD>
int grouped(const Experts& p, bool raw, int64_t routes, Do what, hipStream_t s) {
  // By the routes to an expert on average: how many rows share its weights.  us
  // of both products; experts of 2,048 x 768, 4,096 x 1,536 and 1,000 x 424:
  //   gate and up by tiles of at most 32 and of 128 rows
  //     16 routes an expert    70.9 / 76.5    67.7 / 68.3    21.7 / 22.8
  //     32                     90.5 / 87.5    91.0 / 78.5    32.1 / 30.4
  //   down by wavefronts and by tiles of at most 128 rows
  //     4                      63.9 / 66.1    67.3 / 64.8    21.1 / 21.5
  //     8                      67.5 / 67.3    68.5 / 65.6    22.0 / 21.7
  //     16                     77.2 / 70.7    78.0 / 68.1    23.9 / 22.0
  int rc;
  if (raw)
    rc = gate_up_few<4, kBf16>(p, routes, what, s);
  else if (routes <= 16 * p.num_experts)
    rc = tiled<kGateUp, Tiles32>(p, routes, what, s);
  else
    rc = tiled<kGateUp, Tiles128, Tiles64, Tiles32>(p, routes, what, s);
  if (rc) return rc;
  if (routes <= 8 * p.num_experts) return down_few<1, HELD>(p, routes, what, s);
  return tiled<HELD, Tiles128, Tiles64, Tiles32>(p, routes, what, s);
}

constexpr int64_t kMostRoutes = 1 << 28;

// What the entry points ask of their arguments.
int check(int x_dtype, const void* x, const void* x_scales, int64_t x_stride, int tokens, int top_k, int hidden_size,
          int intermediate_size, int num_experts, const void* slots, int64_t slot_stride, const void* act,
          const void* act_scales) {
  if (tokens < 0 || top_k < 1 || num_experts < 1 || x_stride < 0 || (x_dtype != kBf16 && x_dtype != kRows))
    return SF_ERR_INVALID_ARGUMENT;
  const int64_t bytes = sf_mx_expert_bytes(hidden_size, intermediate_size);
  if (bytes < 0) return SF_ERR_INVALID_ARGUMENT;
  if (num_experts > SF_MAX_EXPERTS || top_k > SF_MAX_TOPK) return SF_ERR_TOO_MANY_EXPERTS;
  if (static_cast<int64_t>(tokens) * top_k > kMostRoutes) return SF_ERR_UNSUPPORTED_SHAPE;
  if (tokens == 0) return SF_OK;
  if (!x || (x_dtype == kRows && !x_scales) || !slots || !act || !act_scales || slot_stride < bytes)
    return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !aligned(slots, 16) || slot_stride % 16 || !aligned(act, 16) || !aligned(act_scales, 16) ||
      (x_dtype == kRows && !aligned(x_scales, 16)))
    return SF_ERR_MISALIGNED;
  if (x_dtype != kRows) {
    if (x_stride % 8 || hidden_size % 8) return SF_ERR_MISALIGNED;
    if (tokens > SF_MX_RAW_ROWS) return SF_ERR_UNSUPPORTED_SHAPE;
  }
  return SF_OK;
}

// out[t] = bf16(sum of token t's rows, in the order of its routes, in fp32).  A
// thread: eight columns of a token.
constexpr int kSumThreads = 256, kAhead = 8;

template <bool EIGHTS>  // columns come in whole eights
__global__ __launch_bounds__(kSumThreads) void sum_rows_kernel(const uint16_t* __restrict__ rows,
                                                               const uint8_t* __restrict__ scales,
                                                               const int32_t* __restrict__ inv, int top_k, int hidden,
                                                               int blocks, uint16_t* __restrict__ out) {
  const int token = blockIdx.x / blocks;
  const int h = (blockIdx.x % blocks * kSumThreads + threadIdx.x) * 8;
  if (h >= hidden) return;
  const int scale_blocks = (hidden + kBlock - 1) / kBlock;
  inv += static_cast<int64_t>(token) * top_k;
  const bool whole = EIGHTS || h + 8 <= hidden;
  float sum[8] = {};
  for (int k0 = 0; k0 < top_k; k0 += kAhead) {  // their loads together
    int row[kAhead];
    u32x4 words[kAhead];
    uint32_t e[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) row[j] = inv[min(k0 + j, top_k - 1)];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t at = max(row[j], 0);  // of an expert that is not there: any row, not added
      const uint16_t* from = rows + at * hidden + h;
      if (whole) {
        words[j] = ld<u32x4_any>(from);
      } else {
        words[j] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (h + i < hidden) words[j][i / 2] |= static_cast<uint32_t>(ld<uint16_t>(from + i)) << (16 * (i % 2));
      }
      e[j] = ld<uint8_t>(scales + at * scale_blocks + h / kBlock);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (k0 + j >= top_k || row[j] < 0) continue;  // wave-uniform
      const float s = from_row(e[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2<kFp16>(words[j][i], a, b);
        sum[2 * i] += a * s;
        sum[2 * i + 1] += b * s;
      }
    }
  }
  uint16_t* o = out + static_cast<int64_t>(token) * hidden + h;
  if (whole) {
    *reinterpret_cast<u32x4_any*>(o) = u32x4{narrow2<kBf16>(sum[0], sum[1]), narrow2<kBf16>(sum[2], sum[3]),
                                             narrow2<kBf16>(sum[4], sum[5]), narrow2<kBf16>(sum[6], sum[7])};
    return;
  }
  for (int i = 0; i < 8; ++i)
    if (h + i < hidden) o[i] = sf_f32_to_bf16(sum[i]);
}

// The dispatch and the rows' rounding need nothing of each other: the first
// workgroups sort the routes (K2), the others round rows (K13).  61 tokens: two
// launches 4.4 + 3.9 us, one 4.8; 2,048 tokens 11.4 + 5.2 and 12.6.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void prepare_kernel(const int64_t* __restrict__ index, int routes, int experts,
                                                          int span, unsigned spans, int32_t* __restrict__ counts,
                                                          int32_t* __restrict__ perm, int32_t* __restrict__ inv,
                                                          const char* __restrict__ x, int64_t x_stride, int dim,
                                                          int chunks, int64_t total, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  if (blockIdx.x < spans)
    sf_dispatch_impl::dispatch<THREADS>(blockIdx.x, index, routes, experts, span, counts, counts + experts + 1, perm,
                                        inv, nullptr);
  else
    quantize_rows_chunk<kBf16>(static_cast<int64_t>(blockIdx.x - spans) * THREADS + threadIdx.x, x, x_stride, dim,
                               chunks, total, codes, scales);
}

// Routes that read their experts for themselves save a dispatch, a sum over rows and the
// launches of both: about 10 us on the device and 10 on the host.  They read an
// expert again for each further route to it, with even routing routes - E (1 -
// (1 - 1 / E)^routes) times; 10 us are 40 MB of such reads.  us a call on the
// device, without dispatch and with it:
//   128 experts of 2048 x 768, 8 a token    1 token 12 / 21   4: 24 / 30   8: 42 / 42   12: 60 / 53
//   32 experts of 4096 x 1536, 8 a token    1 token 27 / 34   2: 40 / 45   3: 57 / 55   4: 71 / 67
//   100 experts of 1000 x 424, 2 a token    1 token 8 / 15    16: 14 / 19  32: 19 / 23
// Beyond 128 routes the products' idle rows would count.
bool without_dispatch(int64_t routes, int experts, int64_t expert_bytes) {
  if (routes > 128) return false;
  const double again = routes - experts * (1.0 - std::pow(1.0 - 1.0 / experts, static_cast<double>(routes)));
  return again * static_cast<double>(expert_bytes) <= 40e6;
}

// sf_mx_experts' workspace: what each part starts at, in bytes.
struct Workspace {
  int64_t act, act_scales, x, x_scales, meta, perm, inv, rows, row_scales, bytes;
};

Workspace workspace_of(int tokens, int top_k, int hidden, int inner, int experts, bool dispatched) {
  Workspace w = {};
  const int64_t routes = static_cast<int64_t>(tokens) * top_k;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  w.act = take(routes * tiles(inner) * kTile);
  w.act_scales = take(routes * quads(inner) * 16);
  w.x = take(static_cast<int64_t>(tokens) * tiles(hidden) * kTile);
  w.x_scales = take(static_cast<int64_t>(tokens) * quads(hidden) * 16);
  if (dispatched) {
    w.meta = take(8ll * (experts + 1));
    w.perm = take(4 * routes);
    w.inv = take(4 * routes);
    w.rows = take(2 * routes * hidden);
    w.row_scales = take(routes * ((hidden + kBlock - 1) / kBlock));
  }
  w.bytes = at;
  return w;
}

Experts experts_of(const void* x, const void* x_scales, int64_t x_stride, const void* route_weights, int top_k,
                   int hidden_size, int intermediate_size, int num_experts, const int32_t* slot_of_expert,
                   const void* slots, int64_t slot_stride, void* act, void* act_scales) {
  Experts p = {};
  p.x = x;
  p.x_scales = static_cast<const uint8_t*>(x_scales);
  p.x_stride = x_stride;
  p.route_weights = static_cast<const uint16_t*>(route_weights);
  p.top_k = top_k;
  p.hidden = hidden_size;
  p.inner = intermediate_size;
  p.num_experts = num_experts;
  p.slot_of_expert = slot_of_expert;
  p.slots = static_cast<const uint8_t*>(slots);
  p.slot_stride = slot_stride;
  p.record = record_of(hidden_size, intermediate_size);
  p.act = static_cast<uint8_t*>(act);
  p.act_scales = static_cast<uint8_t*>(act_scales);
  return p;
}

int routed(int x_dtype, const Experts& p, const Routes& r, int64_t routes, Do what, hipStream_t s) {
  return x_dtype == kBf16 ? routed<8, kBf16>(p, r, routes, what, s) : routed<8, kRows>(p, r, routes, what, s);
}

}  // namespace

extern "C" int64_t sf_mx_expert_bytes(int hidden_size, int intermediate_size) {
  if (hidden_size < 1 || intermediate_size < 1 || hidden_size > 1 << 20 || intermediate_size > 1 << 20) return -1;
  return record_of(hidden_size, intermediate_size).bytes;
}

extern "C" int sf_mx_expert_parts(int hidden_size, int intermediate_size, int64_t* offsets) {
  if (sf_mx_expert_bytes(hidden_size, intermediate_size) < 0 || !offsets) return SF_ERR_INVALID_ARGUMENT;
  const Record r = record_of(hidden_size, intermediate_size);
  const int64_t at[6] = {0, r.up_codes, r.down_codes, r.gate_scales, r.up_scales, r.down_scales};
  for (int i = 0; i < 6; ++i) offsets[i] = at[i];
  return SF_OK;
}

extern "C" int sf_mx_grouped_swiglu(int x_dtype, const void* x, const void* x_scales, int64_t x_stride,
                                    const int32_t* perm_pos, const int32_t* offsets,
                                    const void* route_weights, int tokens, int top_k, int hidden_size,
                                    int intermediate_size, int num_experts, const int32_t* slot_of_expert,
                                    const void* slots, int64_t slot_stride, void* act, void* act_scales,
                                    void* out_rows, sf_stream_t stream) {
  if (const int rc = check(x_dtype, x, x_scales, x_stride, tokens, top_k, hidden_size, intermediate_size, num_experts,
                           slots, slot_stride, act, act_scales))
    return rc;
  if (tokens == 0) return SF_OK;
  if (!perm_pos || !offsets || !out_rows) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(out_rows, 8)) return SF_ERR_MISALIGNED;
  Experts p = experts_of(x, x_scales, x_stride, route_weights, top_k, hidden_size, intermediate_size, num_experts,
                         slot_of_expert, slots, slot_stride, act, act_scales);
  p.perm_pos = perm_pos;
  p.offsets = offsets;
  p.rows = static_cast<uint16_t*>(out_rows);
  const int64_t routes = static_cast<int64_t>(tokens) * top_k;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (const int rc = grouped<kBf16>(p, x_dtype == kBf16, routes, kCheck, s)) return rc;
  return grouped<kBf16>(p, x_dtype == kBf16, routes, kLaunch, s);
}

extern "C" int sf_mx_routed_swiglu(int x_dtype, const void* x, const void* x_scales, int64_t x_stride,
                                   const int64_t* index, const void* route_weights, int tokens, int top_k,
                                   int hidden_size, int intermediate_size, int num_experts,
                                   const int32_t* slot_of_expert, const void* slots, int64_t slot_stride, void* act,
                                   void* act_scales, void* out, sf_stream_t stream) {
  if (const int rc = check(x_dtype, x, x_scales, x_stride, tokens, top_k, hidden_size, intermediate_size, num_experts,
                           slots, slot_stride, act, act_scales))
    return rc;
  if (tokens == 0) return SF_OK;
  if (!index || !route_weights || !out) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(index, 8) || !aligned(route_weights, 2) || !aligned(out, 2)) return SF_ERR_MISALIGNED;
  const Experts p = experts_of(x, x_scales, x_stride, route_weights, top_k, hidden_size, intermediate_size, num_experts,
                               slot_of_expert, slots, slot_stride, act, act_scales);
  const Routes r = {index, static_cast<const uint16_t*>(route_weights), static_cast<uint16_t*>(out)};
  return routed(x_dtype, p, r, static_cast<int64_t>(tokens) * top_k, kLaunch, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int sf_mx_experts_form(int tokens, int top_k, int hidden_size, int intermediate_size, int num_experts) {
  const int64_t bytes = sf_mx_expert_bytes(hidden_size, intermediate_size);
  if (tokens < 0 || top_k < 1 || num_experts < 1 || bytes < 0) return -1;
  return without_dispatch(static_cast<int64_t>(tokens) * top_k, num_experts, bytes);
}

extern "C" int64_t sf_mx_experts_workspace(int tokens, int top_k, int hidden_size, int intermediate_size,
                                           int num_experts) {
  const int form = sf_mx_experts_form(tokens, top_k, hidden_size, intermediate_size, num_experts);
  if (form < 0 || top_k > SF_MAX_TOPK || num_experts > SF_MAX_EXPERTS ||
      static_cast<int64_t>(tokens) * top_k > kMostRoutes)
    return -1;
  return workspace_of(tokens, top_k, hidden_size, intermediate_size, num_experts, form == 0).bytes;
}

extern "C" int sf_mx_experts(int x_dtype, const void* x, const void* x_scales, int64_t x_stride, const int64_t* index,
                             const void* route_weights, int tokens, int top_k, int hidden_size, int intermediate_size,
                             int num_experts, const void* slots, int64_t slot_stride, void* workspace, void* out,
                             sf_stream_t stream) {
  const int64_t bytes = sf_mx_experts_workspace(tokens, top_k, hidden_size, intermediate_size, num_experts);
  if (bytes < 0) return SF_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return SF_OK;
  if (!x || !index || !route_weights || !slots || !workspace || !out) return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(workspace, 16) || !aligned(out, 2) || !aligned(index, 8) || !aligned(route_weights, 2))
    return SF_ERR_MISALIGNED;
  const int64_t routes = static_cast<int64_t>(tokens) * top_k;
  const bool dispatched = !sf_mx_experts_form(tokens, top_k, hidden_size, intermediate_size, num_experts);
  const Workspace w = workspace_of(tokens, top_k, hidden_size, intermediate_size, num_experts, dispatched);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  // Few rows are rounded by the wavefronts that read them.
  const bool rounds =
      x_dtype == kBf16 && (tokens > SF_MX_RAW_ROWS || hidden_size % 8 || x_stride % 8 || !aligned(x, 16));
  const int held = rounds ? kRows : x_dtype;  // what the products read
  if (rounds && !aligned(x, 2)) return SF_ERR_MISALIGNED;
  Experts p = experts_of(rounds ? base + w.x : x, rounds ? base + w.x_scales : x_scales, x_stride, route_weights, top_k,
                         hidden_size, intermediate_size, num_experts, nullptr, slots, slot_stride, base + w.act,
                         base + w.act_scales);
  if (const int rc = check(held, p.x, p.x_scales, x_stride, tokens, top_k, hidden_size, intermediate_size, num_experts,
                           slots, slot_stride, p.act, p.act_scales))
    return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Routes r = {index, p.route_weights, static_cast<uint16_t*>(out)};
  if (!dispatched) {
    if (const int rc = routed(held, p, r, routes, kCheck, s)) return rc;
    if (rounds) {
      if (const int rc = sf_mx_quantize(kBf16, x, x_stride, 0, tokens, hidden_size, 1, kE4m3, base + w.x, 0,
                                        base + w.x_scales, 0, stream))
        return rc;
    }
    return routed(held, p, r, routes, kLaunch, s);
  }
  int32_t* counts = reinterpret_cast<int32_t*>(base + w.meta);
  int32_t* offsets = counts + num_experts + 1;
  int32_t* perm = reinterpret_cast<int32_t*>(base + w.perm);
  int32_t* inv = reinterpret_cast<int32_t*>(base + w.inv);
  p.perm_pos = perm;
  p.offsets = offsets;
  p.rows = reinterpret_cast<uint16_t*>(base + w.rows);
  p.row_scales = base + w.row_scales;
  const sf_dispatch_impl::Cut cut = sf_dispatch_impl::cut_of(static_cast<int>(routes));
  const int chunks = tiles(hidden_size) * 16;
  const int64_t total = static_cast<int64_t>(tokens) * chunks;
  const int64_t grid = cut.spans + (total - 1) / cut.threads + 1;
  const int blocks = groups(hidden_size, 8 * kSumThreads);
  if (const int rc = grouped<kHeldRows>(p, held == kBf16, routes, kCheck, s)) return rc;
  if ((rounds && !grid_fits(grid, cut.threads)) || !grid_fits(static_cast<int64_t>(tokens) * blocks, kSumThreads))
    return SF_ERR_UNSUPPORTED_SHAPE;
  if (rounds) {
    const auto prepare = cut.threads == 256 ? prepare_kernel<256> : prepare_kernel<1024>;
    prepare<<<dim3(static_cast<unsigned>(grid)), dim3(cut.threads), 0, s>>>(
        index, static_cast<int>(routes), num_experts, cut.span, cut.spans, counts, perm, inv,
        static_cast<const char*>(x), x_stride, hidden_size, chunks, total, base + w.x, base + w.x_scales);
    SF_LAUNCH_CHECK();
  } else {
    if (const int rc = sf_dispatch(index, tokens, top_k, num_experts, counts, offsets, perm, inv, nullptr, stream))
      return rc;
  }
  if (const int rc = grouped<kHeldRows>(p, held == kBf16, routes, kLaunch, s)) return rc;
  const auto sum = hidden_size % 8 ? sum_rows_kernel<false> : sum_rows_kernel<true>;
  sum<<<dim3(static_cast<unsigned>(tokens * blocks)), dim3(kSumThreads), 0, s>>>(
      p.rows, p.row_scales, inv, top_k, hidden_size, blocks, static_cast<uint16_t*>(out));
  SF_LAUNCH_CHECK();
  return SF_OK;
}
