// K9: grouped-query attention over a block cache (kv_blocks.h): complete blocks
// in 8 bits with a power-of-two scale each, the last tokens in bf16.
//
// The Q tokens x G heads of one KV head form R = Q G query rows that share its
// keys and values; keys go by in tiles of one block.  Scores are computed
// transposed, S^T = K Q^T, so that a lane holds scores of one query row and the
// softmax state is a register; O^T += V^T P^T takes the probabilities from those
// registers as they are.  Codes become bf16 without their scale (exact): the
// key scale goes into the factor of a tile's scores, and the value scale, a
// power of two, into the exponent of its probabilities,
//   w = 2^(s c_t + (log2 v_scale - M)),  l += v_scale^-1 sum w,  O += w V,
// so neither costs an instruction per value.  M, a row's maximum in log2
// units, is a reference only: every weight of a row has the same one.
//
// direct form: a wavefront owns 16 or 32 rows and takes its operands straight
// from the cache into registers, whose order is that of the matrix
// instructions (no LDS, no barrier); the four wavefronts of a workgroup take
// every fourth tile and merge their states at the end.
#include <algorithm>

#include "kv_blocks.h"

int sf_kv_check(const sf_kv_cache* c);

namespace {

typedef float sf_f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * SF_WAVE;
constexpr int kMaxSplits = 128;

struct Args {
  sf_kv_cache c;
  int kv_heads;
  const uint16_t* q;
  int64_t q_batch, q_head, q_tok;
  const uint8_t* mask;  // of the keys from mask_begin on; nullptr: causal at the end
  int64_t mask_batch, mask_q;
  int mask_begin;
  int Q, S, G;
  int rows, row_tiles;
  int splits, split_tiles;
  float scale_log2;  // |scale| log2(e)
  uint32_t flip;     // of the query's bits: the scale's sign
  uint32_t keep;     // of the query's bits: none for a scale of 0
  uint16_t* out;     // [batch, Q, q_heads, D]
  float* part_acc;   // [splits][batch kv_heads][rows][D], splits > 1 only
  float2* part_ml;   // [splits][batch kv_heads][rows]
};

// Above this |M| its rounding could leave p far from 1 at the maximum (2^28 in
// log2 units: a factor of 2^16), so the scores are scaled before M is taken off.
constexpr float kFusedMax = 268435456.f;

__device__ __forceinline__ float max_raw(float x, float y) {
  return __builtin_amdgcn_fmed3f(x, y, INFINITY);  // one instruction; a NaN gives the other
}

__device__ __forceinline__ float swap32_max(float x) {
  const int v = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}

__device__ __forceinline__ float swap16_max(float x) {
  const int v = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}

__device__ __forceinline__ float swap32_sum(float x) {
  const int v = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

__device__ __forceinline__ float swap16_sum(float x) {
  const int v = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// Whether a row admits keys key .. key + 3, a byte each.
__device__ __forceinline__ uint32_t admitted(const uint8_t* row, int key, int mask_begin, int S) {
  uint32_t w = 0;
  if (key >= mask_begin && key + 4 <= S) {
    __builtin_memcpy(&w, row + (key - mask_begin), 4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < S)
        w |= (key + i < mask_begin ? 1u : static_cast<uint32_t>(row[key + i - mask_begin]))
             << (8 * i);
  }
  return w;
}

// The shapes of the two direct forms.  Both read the same pieces: the key of a
// row of the A operand and the contraction's order of d are free, as long as
// queries, scores and values agree on them.
template <int D, int ROWS>
struct Shape;

// v_mfma_f32_32x32x16_bf16: kScores registers hold, for query row lane % 32,
// keys 8 g + 4 (lane / 32) + i of the tile in register 4 g + i.
template <int D>
struct Shape<D, 32> {
  typedef sf_f32x16 Acc;
  static constexpr int kScoreTiles = 2, kOutTiles = D / 32, kSteps = D / 16, kPSteps = 4;
  static __device__ __forceinline__ Acc mma(sf_u32x4 a, sf_u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(sf_bf16x8, a),
                                                   __builtin_bit_cast(sf_bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int lane) { return lane & 31; }
  static __device__ __forceinline__ int group(int lane) { return lane >> 5; }
  // First d of step s of the scores, and first key of word g of the scores.
  static __device__ __forceinline__ int query_d(int lane, int s) {
    return 32 * (s >> 1) + 16 * (lane >> 5) + 8 * (s & 1);
  }
  static __device__ __forceinline__ int key(int lane, int g) { return 8 * g + 4 * (lane >> 5); }
  static constexpr int kWords = 8;  // of four scores
  // 8-bit pieces (of 16 bytes): n-th of the keys, tile n / (D / 32), steps
  // 2 (n % (D / 32)) and + 1; n-th of the values, tile n / 2, steps 2 (n % 2)
  // and + 1.  bf16 pieces: one step each.
  static __device__ __forceinline__ int key_lane(int lane) { return lane; }
  static __device__ __forceinline__ int value_lane(int lane) { return lane; }
  static __device__ __forceinline__ int key_piece(int tile, int pair) {
    return (tile * (D / 32) + pair) * SF_WAVE;
  }
  static __device__ __forceinline__ int value_piece(int tile, int pair) {
    return (tile * 2 + pair) * SF_WAVE;
  }
  static __device__ __forceinline__ int key_lane16(int lane) { return lane; }
  static __device__ __forceinline__ int value_lane16(int lane) { return lane; }
  static __device__ __forceinline__ int key_piece16(int tile, int s) {
    return (tile * (D / 16) + s) * SF_WAVE;
  }
  static __device__ __forceinline__ int value_piece16(int tile, int s) {
    return (tile * 4 + s) * SF_WAVE;
  }
  static __device__ __forceinline__ float row_max(float x) { return swap32_max(x); }
  static __device__ __forceinline__ float row_sum(float x) { return swap32_sum(x); }
  // d of registers 4 j .. 4 j + 3 of output tile t.
  static __device__ __forceinline__ int out_d(int lane, int t, int j) {
    return 32 * t + 8 * j + 4 * (lane >> 5);
  }
};

// v_mfma_f32_16x16x32_bf16, quad = lane / 16: row r of score tile g is key
// 32 (r / 8) + 8 g + r % 8, so register i of tile g holds, for query row
// lane % 16, key 32 (quad / 2) + 8 g + 4 (quad % 2) + i: the sixteen keys of
// the value pieces of half quad / 2, lane half quad % 2.
template <int D>
struct Shape<D, 16> {
  typedef sf_f32x4 Acc;
  static constexpr int kScoreTiles = 4, kOutTiles = D / 16, kSteps = D / 32, kPSteps = 2;
  static __device__ __forceinline__ Acc mma(sf_u32x4 a, sf_u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sf_bf16x8, a),
                                                   __builtin_bit_cast(sf_bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int lane) { return lane & 15; }
  static __device__ __forceinline__ int group(int lane) { return lane >> 4; }
  static __device__ __forceinline__ int query_d(int lane, int s) {
    return 64 * (s >> 1) + 16 * (lane >> 4) + 8 * (s & 1);
  }
  static __device__ __forceinline__ int key(int lane, int g) {
    return 32 * (lane >> 5) + 8 * g + 4 * ((lane >> 4) & 1);
  }
  static constexpr int kWords = 4;
  static __device__ __forceinline__ int key_lane(int lane) {
    const int r = lane & 15, quad = lane >> 4;
    return ((r >> 3) * (D / 32) + (quad >> 1)) * SF_WAVE + 32 * (quad & 1) + (r & 7);
  }
  static __device__ __forceinline__ int value_lane(int lane) {
    const int quad = lane >> 4;
    return (quad >> 1) * SF_WAVE + 32 * (quad & 1) + (lane & 15);
  }
  static __device__ __forceinline__ int key_piece(int tile, int pair) {
    return 2 * pair * SF_WAVE + 8 * tile;
  }
  static __device__ __forceinline__ int value_piece(int tile, int) {
    return (tile >> 1) * 2 * SF_WAVE + 16 * (tile & 1);
  }
  static __device__ __forceinline__ int key_lane16(int lane) {
    const int r = lane & 15, quad = lane >> 4;
    return ((r >> 3) * (D / 16) + 2 * (quad >> 1)) * SF_WAVE + 32 * (quad & 1) + (r & 7);
  }
  static __device__ __forceinline__ int value_lane16(int lane) {
    const int quad = lane >> 4;
    return 2 * (quad >> 1) * SF_WAVE + 32 * (quad & 1) + (lane & 15);
  }
  static __device__ __forceinline__ int key_piece16(int tile, int s) {
    return (4 * (s >> 1) + (s & 1)) * SF_WAVE + 8 * tile;
  }
  static __device__ __forceinline__ int value_piece16(int tile, int s) {
    return ((tile >> 1) * 4 + s) * SF_WAVE + 16 * (tile & 1);
  }
  static __device__ __forceinline__ float row_max(float x) { return swap32_max(swap16_max(x)); }
  static __device__ __forceinline__ float row_sum(float x) { return swap32_sum(swap16_sum(x)); }
  static __device__ __forceinline__ int out_d(int lane, int t, int) {
    return 16 * t + 4 * (lane >> 4);
  }
};

template <typename Acc>
constexpr int acc_size() {
  return sizeof(Acc) / 4;
}

// The state of a wavefront's rows, and what it does with the scores of a tile.
template <int D, int ROWS>
struct Rows {
  using Sh = Shape<D, ROWS>;
  using Acc = typename Sh::Acc;
  static constexpr int kN = acc_size<Acc>();
  float m = -INFINITY, l = 0.f;  // maximum in log2 units; this lane's part of the sum
  Acc acc[Sh::kOutTiles];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[t][i] = 0.f;
  }

  // Scores (in s) to weights as bf16 (in w, the B operands of the values'
  // product); factor: of the scores, to log2 units.
  __device__ __forceinline__ void softmax(Acc (&s)[Sh::kScoreTiles], float factor, float v_scale,
                                          sf_u32x4 (&w)[Sh::kPSteps]) {
    float mx[2] = {s[0][0], s[1][0]};
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) mx[t & 1] = max_raw(mx[t & 1], s[t][i]);
    const float mnew = fmaxf(m, Sh::row_max(max_raw(mx[0], mx[1])) * factor);
    if (__any(mnew > m)) {
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[t][i] *= alpha;
      m = mnew;
    }
    const float shift = static_cast<float>(static_cast<int>(__float_as_uint(v_scale) >> 23) - 127);
    float base = m == -INFINITY ? 0.f : shift - m;
    float mul = factor;
    const bool large = fabsf(m) > kFusedMax && m != -INFINITY;
    if (__any(large)) {
      const float top = large ? m : 0.f;
#pragma unroll
      for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
        for (int i = 0; i < kN; ++i) s[t][i] = s[t][i] * factor - top;
      if (large) base = shift;
      mul = 1.f;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], mul, base));
        sum[i & 1] += s[t][i];
      }
    // 1 / v_scale, a power of two.
    l = __builtin_fmaf(sum[0] + sum[1],
                       __uint_as_float((254u << 23) - __float_as_uint(v_scale)), l);
#pragma unroll
    for (int k = 0; k < Sh::kPSteps; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = 8 * k + 2 * j;  // in the order of the lane's scores
        w[k][j] = sf_pack_bf16(s[n / kN][n % kN], s[n / kN][n % kN + 1]);
      }
  }
};

// Ones (bf16) where an operand's entry is +inf (kind 0), -inf (1) or NaN (2);
// with kind 3 the entries that are none of these.  CODE: an operand made of
// int8 codes, whose NaN is kNanCodeBf16.
template <bool CODE>
__device__ __forceinline__ sf_u32x4 entries(const sf_u32x4& v, int kind) {
  sf_u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t y = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = (v[j] >> (16 * h)) & 0xffffu;
      int is = 3;
      if (CODE ? x == kNanCodeBf16 : (x & 0x7f80u) == 0x7f80u)
        is = CODE || (x & 0x7fu) ? 2 : static_cast<int>(x >> 15);
      if (is == kind) y |= (kind == 3 ? x : 0x3f80u) << (16 * h);
    }
    r[j] = y;
  }
  return r;
}

// 1 where a weight is not 0.
__device__ __forceinline__ sf_u32x4 present(const sf_u32x4& w) {
  sf_u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = (w[j] & 0x7fffu ? 0x3f80u : 0u) | (w[j] & 0x7fff0000u ? 0x3f800000u : 0u);
  return r;
}

// acc += V^T P^T for a tile whose values hold infinities or NaN: they reach the
// rows that give their key a weight and no others (0 times them in the product
// would).  operand(t, k): the values' operand of output tile t, step k.  Rare,
// so it is written for few registers: one kind after the other.
template <typename Sh, bool CODE, typename Operand>
__device__ __forceinline__ void add_special(Operand operand, const sf_u32x4 (&w)[Sh::kPSteps],
                                            typename Sh::Acc (&acc)[Sh::kOutTiles]) {
  using Acc = typename Sh::Acc;
  constexpr int kN = acc_size<Acc>();
#pragma unroll 1
  for (int t = 0; t < Sh::kOutTiles; ++t) {
    Acc o;
#pragma unroll
    for (int u = 0; u < Sh::kOutTiles; ++u)
      if (u == t) o = acc[u];
#pragma unroll
    for (int k = 0; k < Sh::kPSteps; ++k) o = Sh::mma(entries<CODE>(operand(t, k), 3), w[k], o);
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {
      Acc has;
#pragma unroll
      for (int i = 0; i < kN; ++i) has[i] = 0.f;
#pragma unroll
      for (int k = 0; k < Sh::kPSteps; ++k)
        has = Sh::mma(entries<CODE>(operand(t, k), kind), present(w[k]), has);
      const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (has[i] > 0.f) o[i] += add;
    }
#pragma unroll
    for (int u = 0; u < Sh::kOutTiles; ++u)
      if (u == t) acc[u] = o;
  }
}

// Scores of int8 keys that hold a NaN code: NaN.  operand(t, p): the keys'
// operand of score tile t, step p.
template <typename Sh, typename Operand>
__device__ __forceinline__ void mark_nan_keys(Operand operand,
                                              typename Sh::Acc (&s)[Sh::kScoreTiles]) {
  using Acc = typename Sh::Acc;
  constexpr int kN = acc_size<Acc>();
  const sf_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll 1
  for (int t = 0; t < Sh::kScoreTiles; ++t) {
    Acc has;
#pragma unroll
    for (int i = 0; i < kN; ++i) has[i] = 0.f;
#pragma unroll 1
    for (int p = 0; p < Sh::kSteps; ++p) has = Sh::mma(entries<true>(operand(t, p), 2), ones, has);
#pragma unroll
    for (int u = 0; u < Sh::kScoreTiles; ++u)
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (u == t && has[i] > 0.f) s[u][i] = __builtin_nanf("");
  }
}

template <int D, int ROWS, int HELD, bool MASK>
__global__ __launch_bounds__(kThreads, ROWS == 16 ? 2 : 1) void direct_kernel(const Args a) {
  using Sh = Shape<D, ROWS>;
  using Acc = typename Sh::Acc;
  constexpr int kN = acc_size<Acc>();
  constexpr int kPieces = D / 16;  // 8-bit pieces of a lane, keys or values
  constexpr int kKeyPairs = Sh::kSteps / 2, kValuePairs = Sh::kPSteps / 2;
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / SF_WAVE);
  // Consecutive workgroups take different heads; the last row tiles, which see
  // the most keys under the causal rule, go first.
  const int head = blockIdx.x % a.c.heads;
  const int rest = blockIdx.x / a.c.heads;
  const int split = rest % a.splits;
  const int first_row = (a.row_tiles - 1 - rest / a.splits) * ROWS;
  const int b = head / a.kv_heads;
  const int h = head - b * a.kv_heads;
  const int row = min(first_row + Sh::row(lane), a.rows - 1);
  const int tok = row / a.G;
  const int q_head = h * a.G + (row - tok * a.G);

  sf_u32x4 qf[Sh::kSteps];
  {
    const uint16_t* q = a.q + b * a.q_batch + q_head * a.q_head + tok * a.q_tok;
#pragma unroll
    for (int s = 0; s < Sh::kSteps; ++s)
      qf[s] = (sf_ld16(q + Sh::query_d(lane, s)) & a.keep) ^ a.flip;
  }

  // Tiles [begin, end) of the workgroup; keys below `full` need no look at the
  // causal rule, the mask or the end.
  const int last_tok = (min(first_row + ROWS, a.rows) - 1) / a.G;
  const int diag = a.S - a.Q + 1;  // keys that token 0 sees
  const int keys_end = MASK ? a.S : min(a.S, diag + last_tok);
  const int begin = split * a.split_tiles;
  const int end = min(begin + a.split_tiles, (keys_end + kBlockTokens - 1) / kBlockTokens);
  const int full = MASK ? min(a.S, a.mask_begin) : max(0, diag + first_row / a.G);
  const int lane_end = MASK ? a.S : diag + tok;  // keys of this lane's row (no mask)
  const uint8_t* mask = MASK ? a.mask + b * a.mask_batch + tok * a.mask_q : nullptr;

  const int64_t cap = static_cast<int64_t>(head) * a.c.capacity_blocks;
  const int64_t ring = static_cast<int64_t>(head) * a.c.ring_blocks;
  const char* k8 = static_cast<const char*>(a.c.k8) + cap * (kBlockTokens * D) +
                   16 * Sh::key_lane(lane);
  const char* v8 = static_cast<const char*>(a.c.v8) + cap * (kBlockTokens * D) +
                   16 * Sh::value_lane(lane);
  const float* k_scale = a.c.k_scale + cap;
  const float* v_scale = a.c.v_scale + cap;
  const int32_t* flags8 = a.c.flags + cap;
  const char* kt = static_cast<const char*>(a.c.k_tail) + ring * (2 * kBlockTokens * D) +
                   16 * Sh::key_lane16(lane);
  const char* vt = static_cast<const char*>(a.c.v_tail) + ring * (2 * kBlockTokens * D) +
                   16 * Sh::value_lane16(lane);
  const int32_t* tail_flags = a.c.tail_flags + ring;

  Rows<D, ROWS> r;
  r.clear();

  auto restrict_scores = [&](int tile, Acc(&s)[Sh::kScoreTiles]) {
    const int key0 = tile * kBlockTokens;
    if (key0 + kBlockTokens <= full) return;
#pragma unroll
    for (int g = 0; g < Sh::kWords; ++g) {
      const int key = key0 + Sh::key(lane, g);
      const uint32_t w = MASK ? admitted(mask, key, a.mask_begin, a.S) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = MASK ? ((w >> (8 * i)) & 0xffu) != 0 : key + i < lane_end;
        if (!ok) s[4 * g / kN][4 * g % kN + i] = -INFINITY;
      }
    }
  };

  int tile = begin + wave;
  const int end8 = min(end, a.c.folded_blocks);
  // Blocks in 8 bits.  The registers of a tile's keys (values) are filled again
  // as soon as its products are done with them.
  sf_u32x4 kr[kPieces], vr[kPieces];
  auto load_keys = [&](int t) {
    const char* p = k8 + static_cast<int64_t>(t) * (kBlockTokens * D);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
      kr[n] = sf_ld16(p + 16 * Sh::key_piece(n / kKeyPairs, n % kKeyPairs));
  };
  auto load_values = [&](int t) {
    const char* p = v8 + static_cast<int64_t>(t) * (kBlockTokens * D);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
      vr[n] = sf_ld16(p + 16 * Sh::value_piece(n / kValuePairs, n % kValuePairs));
  };
  if (tile < end8) {
    load_keys(tile);
    load_values(tile);
  }
#pragma unroll 1
  for (; tile < end8; tile += kWaves) {
    const int flag = flags8[tile];
    const float factor = a.scale_log2 * k_scale[tile];
    const float scale_v = v_scale[tile];
    Acc s[Sh::kScoreTiles];
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t) {
#pragma unroll
      for (int i = 0; i < kN; ++i) s[t][i] = 0.f;
#pragma unroll
      for (int p = 0; p < kKeyPairs; ++p) {
        sf_u32x4 x, y;
        sf_codes_frags<HELD>(kr[t * kKeyPairs + p], x, y);
        s[t] = Sh::mma(x, qf[2 * p], s[t]);
        s[t] = Sh::mma(y, qf[2 * p + 1], s[t]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // keep conversions next to their products
    if (tile + kWaves < end8) load_keys(tile + kWaves);
    if (HELD == SF_KV_INT8 && (flag & kFlagKey)) {
      const char* p8 = k8 + static_cast<int64_t>(tile) * (kBlockTokens * D);
      mark_nan_keys<Sh>(
          [&](int t, int p) {
            sf_u32x4 x, y;
            sf_codes_frags<HELD>(sf_ld16(p8 + 16 * Sh::key_piece(t, p >> 1)), x, y);
            return p & 1 ? y : x;
          },
          s);
    }
    restrict_scores(tile, s);
    sf_u32x4 w[Sh::kPSteps];
    r.softmax(s, factor, scale_v, w);
    __builtin_amdgcn_sched_barrier(0);
    if (flag & kFlagValue) {
      const char* p8 = v8 + static_cast<int64_t>(tile) * (kBlockTokens * D);
      add_special<Sh, HELD == SF_KV_INT8>(
          [&](int t, int k) {
            sf_u32x4 x, y;
            sf_codes_frags<HELD>(sf_ld16(p8 + 16 * Sh::value_piece(t, k >> 1)), x, y);
            return k & 1 ? y : x;
          },
          w, r.acc);
    } else {
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
        for (int p = 0; p < kValuePairs; ++p) {
          sf_u32x4 x, y;
          sf_codes_frags<HELD>(vr[t * kValuePairs + p], x, y);
          r.acc[t] = Sh::mma(x, w[2 * p], r.acc[t]);
          r.acc[t] = Sh::mma(y, w[2 * p + 1], r.acc[t]);
        }
    }
    if (tile + kWaves < end8) load_values(tile + kWaves);
  }
  // Blocks of the ring.
#pragma unroll 1
  for (; tile < end; tile += kWaves) {
    const int slot = tile % a.c.ring_blocks;
    const char* kp = kt + static_cast<int64_t>(slot) * (2 * kBlockTokens * D);
    const char* vp = vt + static_cast<int64_t>(slot) * (2 * kBlockTokens * D);
    const int flag = tail_flags[slot];
    Acc s[Sh::kScoreTiles];
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t) {
#pragma unroll
      for (int i = 0; i < kN; ++i) s[t][i] = 0.f;
#pragma unroll
      for (int st = 0; st < Sh::kSteps; ++st)
        s[t] = Sh::mma(sf_ld16(kp + 16 * Sh::key_piece16(t, st)), qf[st], s[t]);
    }
    restrict_scores(tile, s);
    sf_u32x4 w[Sh::kPSteps];
    r.softmax(s, a.scale_log2, 1.f, w);
    if (flag) {
      add_special<Sh, false>([&](int t, int k) { return sf_ld16(vp + 16 * Sh::value_piece16(t, k)); },
                             w, r.acc);
    } else {
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
        for (int k = 0; k < Sh::kPSteps; ++k)
          r.acc[t] = Sh::mma(sf_ld16(vp + 16 * Sh::value_piece16(t, k)), w[k], r.acc[t]);
    }
  }
  r.l = Sh::row_sum(r.l);

  // Merge the wavefronts' states in their order.
  constexpr int kRow = D + 4;
  __shared__ __attribute__((aligned(16))) float acc_lds[kWaves][ROWS * kRow];
  __shared__ float2 ml_lds[kWaves][ROWS];
  if (Sh::group(lane) == 0) ml_lds[wave][Sh::row(lane)] = make_float2(r.m, r.l);
#pragma unroll
  for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
    for (int j = 0; j < kN / 4; ++j)
      *reinterpret_cast<float4*>(&acc_lds[wave][Sh::row(lane) * kRow + Sh::out_d(lane, t, j)]) =
          make_float4(r.acc[t][4 * j], r.acc[t][4 * j + 1], r.acc[t][4 * j + 2],
                      r.acc[t][4 * j + 3]);
  __syncthreads();
  for (int n = threadIdx.x; n < ROWS * D / 4; n += kThreads) {
    const int rr = n / (D / 4);
    const int d = 4 * (n % (D / 4));
    const int out_row = first_row + rr;
    if (out_row >= a.rows) continue;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml_lds[w][rr].x);
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = ml_lds[w][rr];
        if (ml.x == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(ml.x - M);
        const float4 x = *reinterpret_cast<const float4*>(&acc_lds[w][rr * kRow + d]);
        l = __builtin_fmaf(ml.y, f, l);
        o[0] = __builtin_fmaf(x.x, f, o[0]);
        o[1] = __builtin_fmaf(x.y, f, o[1]);
        o[2] = __builtin_fmaf(x.z, f, o[2]);
        o[3] = __builtin_fmaf(x.w, f, o[3]);
      }
    }
    if (a.splits > 1) {
      const int64_t at = (static_cast<int64_t>(split) * a.c.heads + head) * a.rows + out_row;
      *reinterpret_cast<float4*>(a.part_acc + at * D + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) a.part_ml[at] = make_float2(M, l);
    } else {
      const int t = out_row / a.G;
      const int64_t to = (static_cast<int64_t>(b) * a.Q + t) * (static_cast<int64_t>(a.kv_heads) * a.G) +
                         h * a.G + (out_row - t * a.G);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<uint2*>(a.out + to * D + d) =
          make_uint2(sf_pack_bf16(o[0] * inv, o[1] * inv), sf_pack_bf16(o[2] * inv, o[3] * inv));
    }
  }
}

// Merges the splits of a row in their order: eight groups of them per row,
// D / 4 lanes each.
template <int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(const Args a) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float4 acc_lds[kGroups][kLanes];
  __shared__ float2 ml_lds[kGroups];
  const int row = blockIdx.x;
  const int head = blockIdx.y;
  const int g = threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  const int64_t step = static_cast<int64_t>(a.c.heads) * a.rows;
  const int64_t at = static_cast<int64_t>(head) * a.rows + row;
  const int per = (a.splits + kGroups - 1) / kGroups;
  const int s0 = g * per, s1 = min(a.splits, s0 + per);
  float M = -INFINITY;
  for (int s = s0; s < s1; ++s) M = fmaxf(M, a.part_ml[s * step + at].x);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float2 ml, const float4 x, float top) {
    if (ml.x == -INFINITY) return;
    const float f = __builtin_amdgcn_exp2f(ml.x - top);
    l = __builtin_fmaf(ml.y, f, l);
    o.x = __builtin_fmaf(x.x, f, o.x);
    o.y = __builtin_fmaf(x.y, f, o.y);
    o.z = __builtin_fmaf(x.z, f, o.z);
    o.w = __builtin_fmaf(x.w, f, o.w);
  };
  for (int s = s0; s < s1; ++s)
    add(a.part_ml[s * step + at],
        *reinterpret_cast<const float4*>(a.part_acc + (s * step + at) * D + d), M);
  acc_lds[g][threadIdx.x % kLanes] = o;
  if (d == 0) ml_lds[g] = make_float2(M, l);
  __syncthreads();
  if (g != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) top = fmaxf(top, ml_lds[i].x);
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kGroups; ++i) add(ml_lds[i], acc_lds[i][threadIdx.x], top);
  const int b = head / a.kv_heads, h = head - b * a.kv_heads;
  const int t = row / a.G;
  const int64_t to = (static_cast<int64_t>(b) * a.Q + t) * (static_cast<int64_t>(a.kv_heads) * a.G) +
                     h * a.G + (row - t * a.G);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(a.out + to * D + d) =
      make_uint2(sf_pack_bf16(o.x * inv, o.y * inv), sf_pack_bf16(o.z * inv, o.w * inv));
}

// How a call's rows and keys are dealt out.
struct Plan {
  int rows, tile_rows, row_tiles, splits, split_tiles;
};

Plan plan_of(int heads, int group, int queries, int keys) {
  Plan p;
  p.rows = queries * group;
  p.tile_rows = p.rows <= 16 ? 16 : 32;
  p.row_tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  const int tiles = (keys + kBlockTokens - 1) / kBlockTokens;
  // Two workgroups for each of the 256 CUs, each with a tile per wavefront.
  const int64_t base = static_cast<int64_t>(heads) * p.row_tiles;
  int64_t splits = base >= 512 ? 1 : (512 + base - 1) / base;
  splits = std::min<int64_t>(splits, (tiles + kWaves - 1) / kWaves);
  splits = std::min<int64_t>(std::max<int64_t>(splits, 1), kMaxSplits);
  p.split_tiles = static_cast<int>((tiles + splits - 1) / splits);
  p.split_tiles = (p.split_tiles + kWaves - 1) / kWaves * kWaves;
  p.splits = (tiles + p.split_tiles - 1) / p.split_tiles;
  if (p.splits < 1) p.splits = 1;
  return p;
}

template <int D, int ROWS, int HELD>
void launch(const Args& a, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(a.c.heads) * a.row_tiles * a.splits);
  if (a.mask)
    direct_kernel<D, ROWS, HELD, true><<<grid, kThreads, 0, s>>>(a);
  else
    direct_kernel<D, ROWS, HELD, false><<<grid, kThreads, 0, s>>>(a);
}

template <int D>
void launch(const Args& a, int tile_rows, hipStream_t s) {
  const bool int8 = a.c.held == SF_KV_INT8;
  if (tile_rows == 16) {
    if (int8)
      launch<D, 16, SF_KV_INT8>(a, s);
    else
      launch<D, 16, SF_KV_E4M3>(a, s);
  } else {
    if (int8)
      launch<D, 32, SF_KV_INT8>(a, s);
    else
      launch<D, 32, SF_KV_E4M3>(a, s);
  }
  if (a.splits > 1) merge_kernel<D><<<dim3(a.rows, a.c.heads), kThreads, 0, s>>>(a);
}

// Keys, and rows over all heads, of a call, so that every index of tiles, rows
// and workgroups stays in 32 bits.
constexpr int64_t kMaxKeys = 1 << 30;
constexpr int64_t kMaxRows = 1 << 24;

bool fits(int64_t heads, int64_t group, int64_t queries, int64_t keys) {
  return keys <= kMaxKeys && queries <= kMaxRows / group && heads <= 65535 &&
         queries * group * heads <= kMaxRows;
}

}  // namespace

extern "C" int64_t sf_block_attention_workspace(int batch, int queries, int keys, int q_heads,
                                                int kv_heads, int head_dim) {
  if (batch < 1 || queries < 1 || keys < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const int64_t heads = static_cast<int64_t>(batch) * kv_heads;
  if (!fits(heads, q_heads / kv_heads, queries, keys)) return 0;
  const Plan p = plan_of(static_cast<int>(heads), q_heads / kv_heads, queries, keys);
  if (p.splits == 1) return 0;
  return static_cast<int64_t>(p.splits) * heads * p.rows * (head_dim + 2) * 4;
}

extern "C" int sf_block_attention(const sf_kv_cache* cache, int batch, int kv_heads, int keys,
                                  const void* q, int64_t q_stride_batch, int64_t q_stride_head,
                                  int64_t q_stride_token, int queries, int q_heads,
                                  const uint8_t* mask, int64_t mask_stride_batch,
                                  int64_t mask_stride_query, int mask_keys, float scale, void* out,
                                  void* workspace, int64_t workspace_bytes, sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (batch < 1 || kv_heads < 1 || batch > cache->heads || batch * kv_heads != cache->heads ||
      queries < 1 || keys < 1 || !q || !out)
    return SF_ERR_INVALID_ARGUMENT;
  if (q_heads < 1 || q_heads % kv_heads) return SF_ERR_UNSUPPORTED_SHAPE;
  if (mask && (mask_keys < 0 || mask_keys > keys)) return SF_ERR_INVALID_ARGUMENT;
  const int group = q_heads / kv_heads;
  if (!fits(cache->heads, group, queries, keys)) return SF_ERR_UNSUPPORTED_SHAPE;
  const int blocks = (keys + kBlockTokens - 1) / kBlockTokens;
  if (blocks > cache->capacity_blocks || blocks - cache->folded_blocks > cache->ring_blocks)
    return SF_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(q) % 16 || q_stride_batch % 8 || q_stride_head % 8 ||
      q_stride_token % 8 || reinterpret_cast<uintptr_t>(out) % 16)
    return SF_ERR_MISALIGNED;
  Plan p = plan_of(cache->heads, group, queries, keys);
  const int64_t need = sf_block_attention_workspace(batch, queries, keys, q_heads, kv_heads,
                                                    cache->head_dim);
  if (p.splits > 1 && (!workspace || workspace_bytes < need)) {
    p.splits = 1;
    p.split_tiles = blocks;
  }
  if (p.splits > 1 && reinterpret_cast<uintptr_t>(workspace) % 16) return SF_ERR_MISALIGNED;
  Args a = {};
  a.c = *cache;
  a.kv_heads = kv_heads;
  a.q = static_cast<const uint16_t*>(q);
  a.q_batch = q_stride_batch;
  a.q_head = q_stride_head;
  a.q_tok = q_stride_token;
  a.mask = mask;
  a.mask_batch = mask_stride_batch;
  a.mask_q = mask_stride_query;
  a.mask_begin = mask ? keys - mask_keys : 0;
  a.Q = queries;
  a.S = keys;
  a.G = group;
  a.rows = p.rows;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  a.split_tiles = p.split_tiles;
  a.scale_log2 = scale == 0.f ? 1.f : __builtin_fabsf(scale) * 1.4426950408889634f;
  a.flip = scale < 0.f ? 0x80008000u : 0u;
  a.keep = scale == 0.f ? 0u : 0xffffffffu;
  a.out = static_cast<uint16_t*>(out);
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(
      a.part_acc + static_cast<int64_t>(p.splits) * cache->heads * p.rows * cache->head_dim);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    launch<128>(a, p.tile_rows, s);
  else
    launch<64>(a, p.tile_rows, s);
  SF_LAUNCH_CHECK();
  return SF_OK;
}
