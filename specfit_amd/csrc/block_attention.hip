// K10: grouped-query attention over a block cache (kv_blocks.h): complete blocks
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
// so neither costs an instruction per value.  M, at or a little above a row's
// maximum in log2 units, is a reference only: every weight of a row has the same
// one.  A state whose M is -inf belongs to a row that admits none of its keys; every
// merge and the last division go by that (see Rows::settle).
//
// Two forms, and kernels that merge splits of the keys: few rows per KV head go
// straight from the cache to registers (the direct kernel), many share tiles in
// LDS (the staged one); plan_of chooses.
#include <algorithm>

#include "kv_blocks.h"

int sf_kv_check(const sf_kv_cache* c);

namespace {

typedef float sf_f32x16 __attribute__((ext_vector_type(16)));

// Where a value is made in a branch that is rarely taken: keeps the compiler
// from running the branch always and selecting.  After a computation that is
// meant to overlap with what stands beside it: keeps it from being moved down to
// its use.
template <typename T>
__device__ __forceinline__ void pin(T& x) {
  asm volatile("" : "+v"(x));
}

// Loads and stores through pointers of the argument structs, explicitly global.
template <typename T>
__device__ __forceinline__ T ld(const T* p) {
  return *(const __attribute__((address_space(1))) T*)(p);
}

constexpr int kDirectRows = 16;
constexpr int kDirectWaves = 8;
constexpr int kDirectThreads = kDirectWaves * SF_WAVE;
constexpr int kMaxSplits = 128;
constexpr int kStagedWaves = 8;
constexpr int kStagedThreads = kStagedWaves * SF_WAVE;
constexpr int kStagedRows = 32 * kStagedWaves;

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

// M is set this far above the maximum that made it move, so that it rarely has to
// move again (a move costs a product per accumulator, and with M at the maximum a
// third of the tiles of a long prompt move one of 32 rows: 128 nodes after 32777
// tokens 174 -> 170 us).  A row's weights are at most 1, the largest at least
// 2^-kHeadroom; rounded to bf16 relative to themselves, they lose nothing by it.
constexpr float kHeadroom = 8.f;

// M of a state whose admitted scores were all -inf or NaN.
constexpr float kLowest = -3.402823466e+38f;

// Above this |M| its rounding could leave p far from 1 at the maximum (2^28 in
// log2 units: a factor of 2^16), so the scores are scaled before M is taken off.
constexpr float kFusedMax = 268435456.f;

__device__ __forceinline__ float max_raw(float x, float y) {
  return __builtin_amdgcn_fmed3f(x, y, INFINITY);  // one instruction; a NaN gives the other
}

// The largest of three (fmaxf of matrix results would canonicalise each first).
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
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

// Whether a row admits keys key .. key + 3, a byte each: one load, at the
// nearest place within the mask's keys, shifted.  Keys before the mask are
// admitted, keys past the end are not.
__device__ __forceinline__ uint32_t admitted(const uint8_t* row, int key, int mask_begin, int S) {
  const int off = key - mask_begin, count = S - mask_begin;
  if (count >= 4) {  // uniform
    const int at = min(max(off, 0), count - 4);
    uint32_t w;
    __builtin_memcpy(&w, row + at, 4);
    const int past = min(off - at, 4), before = min(at - off, 4);
    if (past > 0) w = static_cast<uint32_t>(static_cast<uint64_t>(w) >> (8 * past));
    if (before > 0)
      w = static_cast<uint32_t>(static_cast<uint64_t>(w) << (8 * before)) |
          0x01010101u >> (32 - 8 * before);
    return w;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i < S)
      w |= (key + i < mask_begin ? 1u : static_cast<uint32_t>(row[key + i - mask_begin])) << (8 * i);
  return w;
}

// The shapes of the matrix instructions: 32 rows in the staged kernel, 16 in the
// direct one.  Both read the same pieces: the key of a row of the A operand and the
// contraction's order of d are free, as long as queries, scores and values agree on
// them.
template <int D, int ROWS>
struct Shape;

// v_mfma_f32_32x32x16_bf16: the 32 scores of a lane are, for query row lane % 32,
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
  float m = -INFINITY, l = 0.f;  // M, at or above the maximum, in log2 units; this lane's part of the sum
  Acc acc[Sh::kOutTiles];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[t][i] = 0.f;
  }

  // The largest of the lane's scores.
  static __device__ __forceinline__ float top(const Acc (&s)[Sh::kScoreTiles]) {
    float mx[2] = {s[0][0], s[0][1]};
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; i += 4) {
        mx[0] = max3(mx[0], s[t][i], s[t][i + 1]);
        mx[1] = max3(mx[1], s[t][i + 2], s[t][i + 3]);
      }
    return max_raw(mx[0], mx[1]);
  }

  // Brings M to or above the scores of a tile whose largest of the lane is `most`;
  // factor: of the scores, to log2 units.  mul and base: a score's weight times the
  // value scale is 2^(s mul + base).
  __device__ __forceinline__ void raise(Acc (&s)[Sh::kScoreTiles], float most, float factor,
                                        float v_scale, float& mul, float& base) {
    const float top = Sh::row_max(most) * factor;
    if (__any(top > m)) {
      const float mnew = top > m ? top + kHeadroom : m;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[t][i] *= alpha;
      m = mnew;
    }
    const float shift = static_cast<float>(static_cast<int>(__float_as_uint(v_scale) >> 23) - 127);
    base = m == -INFINITY ? 0.f : shift - m;
    mul = factor;
    const bool large = fabsf(m) > kFusedMax && m != -INFINITY;
    if (__any(large)) {
      // Only in the rows that need it: another rounding would change the others' bits.
#pragma unroll
      for (int t = 0; t < Sh::kScoreTiles; ++t) {
#pragma unroll
        for (int i = 0; i < kN; ++i) s[t][i] = large ? s[t][i] * factor - m : s[t][i];
        pin(s[t]);
      }
      if (large) {
        base = shift;
        mul = 1.f;
      }
    }
  }

  // The n-th pair of scores to weights times the value scale, as bf16 into w (the
  // B operands of the values' product, in the order of the lane's scores), and
  // added to sum; returns the weights themselves.
  static constexpr int kPairs = Sh::kScoreTiles * kN / 2;
  static __device__ __forceinline__ float2 weigh_pair(const Acc (&s)[Sh::kScoreTiles], int n,
                                                      float mul, float base, float (&sum)[2],
                                                      sf_u32x4 (&w)[Sh::kPSteps]) {
    const float p0 =
        __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * n / kN][2 * n % kN], mul, base));
    const float p1 =
        __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * n / kN][2 * n % kN + 1], mul, base));
    sum[0] += p0;
    sum[1] += p1;
    w[n / 4][n % 4] = sf_pack_bf16(p0, p1);
    return make_float2(p0, p1);
  }
  __device__ __forceinline__ void add_sum(const float (&sum)[2], float v_scale) {
    // 1 / v_scale, a power of two.
    l = __builtin_fmaf(sum[0] + sum[1],
                       __uint_as_float((254u << 23) - __float_as_uint(v_scale)), l);
  }
  __device__ __forceinline__ void weigh(const Acc (&s)[Sh::kScoreTiles], float mul, float base,
                                        float v_scale, sf_u32x4 (&w)[Sh::kPSteps]) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < kPairs; ++n) weigh_pair(s, n, mul, base, sum, w);
    add_sum(sum, v_scale);
  }

  // After the last tile: the lanes' sums together, and M of a row that admits a key
  // (`some`, of any lane).  It is still -inf where all scores were -inf or NaN, as the
  // maximum leaves a NaN out: then the lowest finite value, so that a NaN in l reaches
  // the result of any merge (its factor may be 0) and a sum of 0 divides 0.
  __device__ __forceinline__ void settle(bool some) {
    l = Sh::row_sum(l);
    const float count = Sh::row_sum(some ? 1.f : 0.f);
    if (m == -INFINITY && count > 0.f) m = kLowest;
  }

  // All of a tile's weights, in two terms: w, and what its rounding to bf16 left, also
  // as bf16 (2^-16 of a weight is lost, where w alone loses up to 2^-8).
  __device__ __forceinline__ void softmax(Acc (&s)[Sh::kScoreTiles], float factor, float v_scale,
                                          sf_u32x4 (&w)[Sh::kPSteps],
                                          sf_u32x4 (&rest)[Sh::kPSteps]) {
    float mul, base;
    raise(s, top(s), factor, v_scale, mul, base);
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < kPairs; ++n) {
      const float2 p = weigh_pair(s, n, mul, base, sum, w);
      const uint32_t pair = w[n / 4][n % 4];
      rest[n / 4][n % 4] = sf_pack_bf16(p.x - __uint_as_float(pair << 16),
                                        p.y - __uint_as_float(pair & 0xffff0000u));
    }
    add_sum(sum, v_scale);
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

// A piece of codes with zeros for those that stand for NaN.
template <int HELD>
__device__ __forceinline__ sf_u32x4 finite_codes(const sf_u32x4& v) {
  sf_u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t y = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = (v[j] >> (8 * i)) & 0xffu;
      if (HELD == SF_KV_INT8 ? x != 0x80u : (x & 0x7fu) != 0x7fu) y |= x << (8 * i);
    }
    r[j] = y;
  }
  return r;
}

// What a lane needs to restrict the scores of a tile: its mask's bytes, loaded
// with the tile's keys, or the keys that its row sees without a mask.
template <typename Sh, bool MASK>
struct Admit {
  const uint8_t* row;  // the mask of the lane's row
  int mask_begin, S, lane_end;
  int full;            // keys below it are admitted by all of the wavefront's rows
  uint32_t some;       // not 0: the row admits a key that the lane knows of
  uint32_t words[Sh::kWords];

  __device__ __forceinline__ void load(int lane, int key0) {
    if (!MASK || key0 + kBlockTokens <= full) return;
#pragma unroll
    for (int g = 0; g < Sh::kWords; ++g) {
      words[g] = admitted(row, key0 + Sh::key(lane, g), mask_begin, S);
      pin(words[g]);
      some |= words[g];
    }
  }
  // Scores of keys that the row does not admit: -inf.
  __device__ __forceinline__ void restrict_scores(typename Sh::Acc (&s)[Sh::kScoreTiles], int lane,
                                                  int key0) const {
    constexpr int kN = acc_size<typename Sh::Acc>();
    if (key0 + kBlockTokens <= full) return;
#pragma unroll
    for (int g = 0; g < Sh::kWords; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = MASK ? ((words[g] >> (8 * i)) & 0xffu) != 0
                             : key0 + Sh::key(lane, g) + i < lane_end;
        if (!ok) s[4 * g / kN][4 * g % kN + i] = -INFINITY;
      }
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t) pin(s[t]);
  }
};

// Where a call's row of the output, or of its partial results, lies.
__device__ __forceinline__ int64_t out_row_at(const Args& a, int head, int row) {
  const int b = head / a.kv_heads, h = head - b * a.kv_heads;
  const int t = row / a.G;
  return (static_cast<int64_t>(b) * a.Q + t) * (static_cast<int64_t>(a.kv_heads) * a.G) + h * a.G +
         (row - t * a.G);
}

// A tile's operands of the two products, for the rare paths.
template <int D, int ROWS, int HELD>
struct TileOperands {
  using Sh = Shape<D, ROWS>;
  const char *k, *v;  // of the lane's first piece
  bool coded;

  __device__ __forceinline__ TileOperands(const Args& a, int head, int tile, int lane) {
    coded = tile < a.c.folded_blocks;
    if (coded) {
      const int64_t at =
          (static_cast<int64_t>(head) * a.c.capacity_blocks + tile) * (kBlockTokens * D);
      k = static_cast<const char*>(a.c.k8) + at + 16 * Sh::key_lane(lane);
      v = static_cast<const char*>(a.c.v8) + at + 16 * Sh::value_lane(lane);
    } else {
      const int64_t at = (static_cast<int64_t>(head) * a.c.ring_blocks + tile % a.c.ring_blocks) *
                         (2 * kBlockTokens * D);
      k = static_cast<const char*>(a.c.k_tail) + at + 16 * Sh::key_lane16(lane);
      v = static_cast<const char*>(a.c.v_tail) + at + 16 * Sh::value_lane16(lane);
    }
  }
  static __device__ __forceinline__ sf_u32x4 code_operand(const char* p, int step) {
    sf_u32x4 x, y;
    sf_codes_frags<HELD>(sf_ld16(p), x, y);
    return step & 1 ? y : x;
  }
  __device__ __forceinline__ sf_u32x4 key(int t, int s) const {
    return coded ? code_operand(k + 16 * Sh::key_piece(t, s >> 1), s)
                 : sf_ld16(k + 16 * Sh::key_piece16(t, s));
  }
  __device__ __forceinline__ sf_u32x4 value(int t, int s) const {
    return coded ? code_operand(v + 16 * Sh::value_piece(t, s >> 1), s)
                 : sf_ld16(v + 16 * Sh::value_piece16(t, s));
  }
  // The operand's entries of a kind (see entries).
  __device__ __forceinline__ sf_u32x4 of_kind(const sf_u32x4& x, int kind) const {
    return HELD == SF_KV_INT8 && coded ? entries<true>(x, kind) : entries<false>(x, kind);
  }
};

// What the tiles' values hold that is not finite (the loops take zeros in its
// place, as 0 times it would reach the rows that do not admit its key): an
// infinity or NaN is added to its element of the rows that admit the key.  An
// int8 key with a NaN code (which the loops take for -128) makes the rows that
// admit it NaN.  After the loops, so that their registers are free for it.
template <int D, int ROWS, int HELD, bool MASK>
__device__ __forceinline__ void add_special(Rows<D, ROWS>& r, const Args& a, int head, int lane,
                                            int begin, int end, int step,
                                            Admit<Shape<D, ROWS>, MASK>& admit) {
  using Sh = Shape<D, ROWS>;
  using Acc = typename Sh::Acc;
  constexpr int kN = acc_size<Acc>();
#pragma unroll 1
  for (int tile = begin; tile < end; tile += step) {
    const TileOperands<D, ROWS, HELD> x(a, head, tile, lane);
    const int flag =
        x.coded ? a.c.flags[static_cast<int64_t>(head) * a.c.capacity_blocks + tile]
                : a.c.tail_flags[static_cast<int64_t>(head) * a.c.ring_blocks +
                                 tile % a.c.ring_blocks];
    if (!flag) continue;
    Acc s[Sh::kScoreTiles];  // 0 where the row admits the key
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) s[t][i] = 0.f;
    admit.load(lane, tile * kBlockTokens);
    admit.restrict_scores(s, lane, tile * kBlockTokens);
    if (flag & kFlagValue) {
      sf_u32x4 w[Sh::kPSteps];
#pragma unroll
      for (int k = 0; k < Sh::kPSteps; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = 8 * k + 2 * j;
          w[k][j] = (s[n / kN][n % kN] == 0.f ? 0x3f80u : 0u) |
                    (s[n / kN][n % kN + 1] == 0.f ? 0x3f800000u : 0u);
        }
#pragma unroll 1
      for (int kind = 0; kind < 3; ++kind) {
        const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
        for (int t = 0; t < Sh::kOutTiles; ++t) {
          Acc has;
#pragma unroll
          for (int i = 0; i < kN; ++i) has[i] = 0.f;
#pragma unroll
          for (int k = 0; k < Sh::kPSteps; ++k)
            has = Sh::mma(x.of_kind(x.value(t, k), kind), w[k], has);
#pragma unroll
          for (int i = 0; i < kN; ++i)
            if (has[i] > 0.f) r.acc[t][i] += add;
        }
      }
    }
    if (HELD == SF_KV_INT8 && x.coded && (flag & kFlagKey)) {
      const sf_u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
      bool bad = false;
#pragma unroll
      for (int t = 0; t < Sh::kScoreTiles; ++t) {
        Acc has;
#pragma unroll
        for (int i = 0; i < kN; ++i) has[i] = 0.f;
#pragma unroll 1
        for (int k = 0; k < Sh::kSteps; ++k) has = Sh::mma(entries<true>(x.key(t, k), 2), ones, has);
#pragma unroll
        for (int i = 0; i < kN; ++i) bad |= has[i] > 0.f && s[t][i] == 0.f;
      }
      if (bad) r.l = __builtin_nanf("");  // a part of the row's sum
    }
  }
}

// The form of many rows: 32 rows per wavefront, 256 per workgroup, which share
// each tile.  A tile is staged in LDS as bf16 in the cache's own order, codes
// converted once for the eight wavefronts, so every operand is read as 64
// consecutive 16-byte pieces.
//
// A wavefront's own matrix and vector work overlap: while the weights of tile
// i are computed, the matrix unit forms the scores of tile i + 1, and while it
// adds the values of tile i, the maximum of those scores is taken.  So in
// iteration i the keys of i + 1 and the values of i are read, and one barrier
// is enough with two buffers of keys and three of values (what a wavefront
// writes before the barrier of iteration i, others last read before that of
// i - 1).
//
// Bound by the matrix unit at the clock that its power allows: 2048 e4m3 queries
// after 16000 keys, 32 heads of 128, take 595 - 605 us, 940 TFLOP/s (a large matrix
// product of a library reaches 1150).  Without the exponentials it is 5% less,
// without the staging 14%.  Two groups of 32 rows per wavefront, for half of the
// reads of LDS, spill: 2150 us.
//
// Probabilities meet the values as bf16, so that a row's error is 0.0023 of its norm
// against 64 bits where 0.0017 are the result's own rounding (e4m3 codes of the values
// are off by up to 2^-4).  What their rounding left, as a second product (the direct
// kernel has it), costs a third more: 602 -> 833 us here, 165 -> 212 for 128 nodes after
// 32777 tokens (729 and 195 by its matrix instructions alone).
template <int D, int HELD, bool MASK>
__global__ __launch_bounds__(kStagedThreads, 1) void block_attention_staged_kernel(const Args a) {
  using Sh = Shape<D, 32>;
  using Acc = typename Sh::Acc;
  constexpr int kPieces = kBlockTokens * D / 8;             // of a tile's keys or values, bf16
  constexpr int kLoads = 2 * kPieces / kStagedThreads;      // of both per thread, bf16
  constexpr int kCodes = kPieces / 2;                       // of keys or values in 8 bits
  __shared__ __attribute__((aligned(16))) sf_u32x4 k_lds[2][kPieces];
  __shared__ __attribute__((aligned(16))) sf_u32x4 v_lds[3][kPieces];
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / SF_WAVE);
  const int head = blockIdx.x % a.c.heads;
  const int rest = blockIdx.x / a.c.heads;
  const int split = rest % a.splits;
  const int block_row = (a.row_tiles - 1 - rest / a.splits) * (kStagedRows);
  const int wave_row = block_row + 32 * wave;
  const int b = head / a.kv_heads;
  const int h = head - b * a.kv_heads;
  const int row = wave_row + Sh::row(lane);
  const int row_c = min(row, a.rows - 1);
  const int tok = row_c / a.G;
  const int q_head = h * a.G + (row_c - tok * a.G);

  const int diag = a.S - a.Q + 1;  // keys that token 0 sees
  const int last = min(block_row + kStagedRows, a.rows) - 1;
  const int keys_end = MASK ? a.S : min(a.S, diag + last / a.G);
  const int begin = split * a.split_tiles;
  const int end = min(begin + a.split_tiles, (keys_end + kBlockTokens - 1) / kBlockTokens);
  Admit<Sh, MASK> admit;
  admit.row = MASK ? a.mask + b * a.mask_batch + tok * a.mask_q : nullptr;
  admit.mask_begin = a.mask_begin;
  admit.S = a.S;
  admit.lane_end = diag + tok;
  admit.some = MASK ? a.mask_begin > 0 : diag + tok > 0;
  admit.full = MASK ? min(a.S, a.mask_begin) : max(0, diag + min(wave_row, a.rows - 1) / a.G);

  const int64_t cap = static_cast<int64_t>(head) * a.c.capacity_blocks;
  const int64_t ring = static_cast<int64_t>(head) * a.c.ring_blocks;
  const char* k8 = static_cast<const char*>(a.c.k8) + cap * (kBlockTokens * D);
  const char* v8 = static_cast<const char*>(a.c.v8) + cap * (kBlockTokens * D);
  const float* k_scale = a.c.k_scale + cap;
  const float* v_scale = a.c.v_scale + cap;
  const int32_t* flags8 = a.c.flags + cap;
  const char* kt = static_cast<const char*>(a.c.k_tail) + ring * (2 * kBlockTokens * D);
  const char* vt = static_cast<const char*>(a.c.v_tail) + ring * (2 * kBlockTokens * D);
  const int32_t* tail_flags = a.c.tail_flags + ring;

  // A tile on its way: into registers, and from there (bf16) into LDS.
  // Its pieces are dealt out keys first, then values.
  sf_u32x4 raw[kLoads];
  int special = 0;
  // First piece of the wavefront's j-th 64: of the keys, or (- count) the values.
  auto first_piece = [&](int j) { return j * kStagedThreads + wave * SF_WAVE; };
  auto load_tile = [&](int t) {
    if (t < a.c.folded_blocks) {
      const int64_t at = static_cast<int64_t>(t) * (kBlockTokens * D);
#pragma unroll
      for (int j = 0; j < kLoads / 2; ++j) {
        const int n = first_piece(j);
        raw[j] = sf_ld16((n < kCodes ? k8 + 16 * n : v8 + 16 * (n - kCodes)) + at, 16 * lane);
      }
    } else {
      const int64_t at = static_cast<int64_t>(t % a.c.ring_blocks) * (2 * kBlockTokens * D);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int n = first_piece(j);
        raw[j] = sf_ld16((n < kPieces ? kt + 16 * n : vt + 16 * (n - kPieces)) + at, 16 * lane);
      }
    }
  };
  auto stage_tile = [&](int t, sf_u32x4* kl, sf_u32x4* vl) {
    int flag;
    if (t < a.c.folded_blocks) {
      flag = ld(flags8 + t);
#pragma unroll
      for (int j = 0; j < kLoads / 2; ++j) {
        const int n = first_piece(j);
        const bool values = n >= kCodes;
        sf_u32x4 x, y;
        sf_codes_frags<HELD>(raw[j], x, y);
        if (values && (flag & kFlagValue)) {
          x = entries<HELD == SF_KV_INT8>(x, 3);
          y = entries<HELD == SF_KV_INT8>(y, 3);
          pin(x);
          pin(y);
        }
        sf_u32x4* to = (values ? vl + 2 * (n - kCodes) : kl + 2 * n) + lane;
        to[0] = x;
        to[SF_WAVE] = y;
      }
    } else {
      flag = ld(tail_flags + t % a.c.ring_blocks);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int n = first_piece(j);
        if (n >= kPieces && flag) {
          raw[j] = entries<false>(raw[j], 3);
          pin(raw[j]);
        }
        ((n < kPieces ? kl + n : vl + (n - kPieces)) + lane)[0] = raw[j];
      }
    }
    special |= flag;
  };

  using R = Rows<D, 32>;
  R r;
  r.clear();
  sf_u32x4 qf[Sh::kSteps];
  auto scores = [&](const sf_u32x4* kl, Acc(&s)[Sh::kScoreTiles]) {
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
#pragma unroll
    for (int st = 0; st < Sh::kSteps; ++st)
#pragma unroll
      for (int t = 0; t < Sh::kScoreTiles; ++t)
        s[t] = Sh::mma(kl[Sh::key_piece16(t, st) + lane], qf[st], s[t]);
  };

  float most = -INFINITY;  // of the lane's scores of the tile at hand
  Acc s0[Sh::kScoreTiles], s1[Sh::kScoreTiles];
  int v_slot = 0;          // of the tile at hand
  if (begin < end) {
    load_tile(begin);
    {
      const uint16_t* q = a.q + b * a.q_batch + q_head * a.q_head + tok * a.q_tok;
#pragma unroll
      for (int s = 0; s < Sh::kSteps; ++s)
        qf[s] = (sf_ld16(q + Sh::query_d(lane, s)) & a.keep) ^ a.flip;
    }
    admit.load(lane, begin * kBlockTokens);
    stage_tile(begin, k_lds[begin & 1], v_lds[0]);
    if (begin + 1 < end) load_tile(begin + 1);
    __syncthreads();
    scores(k_lds[begin & 1], s0);
    admit.restrict_scores(s0, lane, begin * kBlockTokens);
    most = R::top(s0);
  }

  auto add_values = [&](const sf_u32x4* vl, const sf_u32x4(&w)[Sh::kPSteps]) {
#pragma unroll
    for (int k = 0; k < Sh::kPSteps; ++k)
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
        r.acc[t] = Sh::mma(vl[Sh::value_piece16(t, k) + lane], w[k], r.acc[t]);
  };
  auto tile_scales = [&](int tile, float& factor, float& scale_v) {
    factor = a.scale_log2;
    scale_v = 1.f;
    if (tile < a.c.folded_blocks) {
      factor *= ld(k_scale + tile);
      scale_v = ld(v_scale + tile);
    }
  };
  // Tile `tile`, whose scores are in s and which is not the last; `next` takes
  // the scores of the one after.
  auto step = [&](int tile, Acc(&s)[Sh::kScoreTiles], Acc(&next)[Sh::kScoreTiles]) {
    const sf_u32x4* vl = v_lds[v_slot];
    v_slot = v_slot == 2 ? 0 : v_slot + 1;
    float factor, scale_v, mul, base;
    tile_scales(tile, factor, scale_v);
    stage_tile(tile + 1, k_lds[(tile + 1) & 1], v_lds[v_slot]);
    if (tile + 2 < end) load_tile(tile + 2);
    admit.load(lane, (tile + 1) * kBlockTokens);
    r.raise(s, most, factor, scale_v, mul, base);
    __syncthreads();  // tile + 1 is complete
    // Both blocks are written in the order in which they are to run: an operand's
    // read kAhead products ahead of its use, a product, and vector work for the
    // time it takes.
    constexpr int kAhead = 3;
    sf_u32x4 w[Sh::kPSteps];
    {
      constexpr int kProducts = 2 * Sh::kSteps;
      const sf_u32x4* kl = k_lds[(tile + 1) & 1] + lane;
      auto read = [&](int i) { return kl[Sh::key_piece16(i & 1, i >> 1)]; };
      sf_u32x4 x[kProducts];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < Sh::kScoreTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) next[t][i] = 0.f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = read(i);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        if (i + kAhead < kProducts) x[i + kAhead] = read(i + kAhead);
        next[i & 1] = Sh::mma(x[i], qf[i >> 1], next[i & 1]);
#pragma unroll
        for (int n = i * R::kPairs / kProducts; n < (i + 1) * R::kPairs / kProducts; ++n) {
          R::weigh_pair(s, n, mul, base, sum, w);
          uint32_t pair = w[n / 4][n % 4];
          pin(pair);
          w[n / 4][n % 4] = pair;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      r.add_sum(sum, scale_v);
    }
    admit.restrict_scores(next, lane, (tile + 1) * kBlockTokens);
    {
      constexpr int kProducts = Sh::kPSteps * Sh::kOutTiles;
      auto read = [&](int i) {
        return vl[Sh::value_piece16(i % Sh::kOutTiles, i / Sh::kOutTiles) + lane];
      };
      sf_u32x4 x[kProducts];
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = read(i);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        if (i + kAhead < kProducts) x[i + kAhead] = read(i + kAhead);
        Acc& o = r.acc[i % Sh::kOutTiles];
        o = Sh::mma(x[i], w[i / Sh::kOutTiles], o);
#pragma unroll
        for (int n = i * R::kPairs / kProducts; n < (i + 1) * R::kPairs / kProducts; ++n)
          mx[n & 1] = max3(mx[n & 1], next[2 * n / 16][2 * n % 16], next[2 * n / 16][2 * n % 16 + 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      most = max_raw(mx[0], mx[1]);
    }
  };
  int tile = begin;
#pragma unroll 1
  for (; tile + 2 < end; tile += 2) {
    step(tile, s0, s1);
    step(tile + 1, s1, s0);
  }
  if (tile + 1 < end) {
    step(tile, s0, s1);
    ++tile;
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t) s0[t] = s1[t];
  }
  if (tile < end) {
    float factor, scale_v, mul, base;
    sf_u32x4 w[Sh::kPSteps];
    tile_scales(tile, factor, scale_v);
    r.raise(s0, most, factor, scale_v, mul, base);
    r.weigh(s0, mul, base, scale_v, w);
    add_values(v_lds[v_slot], w);
  }
  if (special)
    add_special<D, 32, HELD, MASK>(r, a, head, lane, begin, end, 1, admit);
  r.settle(admit.some != 0);
  if (row >= a.rows) return;
  if (a.splits > 1) {
    const int64_t at = (static_cast<int64_t>(split) * a.c.heads + head) * a.rows + row;
    if (Sh::group(lane) == 0) a.part_ml[at] = make_float2(r.m, r.l);
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(a.part_acc + at * D + Sh::out_d(lane, t, j)) =
            make_float4(r.acc[t][4 * j], r.acc[t][4 * j + 1], r.acc[t][4 * j + 2],
                        r.acc[t][4 * j + 3]);
  } else {
    const float inv = r.m == -INFINITY ? 0.f : 1.f / r.l;
    uint16_t* out = a.out + out_row_at(a, head, row) * D;
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint2*>(out + Sh::out_d(lane, t, j)) =
            make_uint2(sf_pack_bf16(r.acc[t][4 * j] * inv, r.acc[t][4 * j + 1] * inv),
                       sf_pack_bf16(r.acc[t][4 * j + 2] * inv, r.acc[t][4 * j + 3] * inv));
  }
}

// The form of few rows: 16 rows per workgroup, whose eight wavefronts take every
// eighth tile and merge their states in LDS.  Until then operands go straight from
// the cache into registers, whose order is that of the matrix instructions: the
// loop over tiles needs no LDS and no barrier.  Decoding long contexts is bound by
// the cache's bytes (131072 int8 keys of 4 heads of 128: 25 us, 5.4 TB/s), short calls
// by latency (5.3 us for one tile per wavefront), trees by the conversions of codes
// and the softmax (10.2 us for 61 nodes after 1024).  The matrix unit has room for
// probabilities in two terms, so that a row's error is the rounding of the result
// (0.0016 - 0.0017 of its norm; 0.0019 - 0.0022 with one term).  Kernel times with one
// and with two: 131072 keys 26.3 and 26.6 us, the tree 8.7 and 9.5, 512 tokens of 32 / 4
// heads of 128 18.7 and 19.1, 2000 after 4000 of 16 / 4 heads of 64 80 and 94.
template <int D, int HELD, bool MASK>
__global__ __launch_bounds__(kDirectThreads, 1) void block_attention_direct_kernel(const Args a) {
  constexpr int ROWS = kDirectRows;
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

  // Tiles [begin, end) of the workgroup.
  const int last_tok = (min(first_row + ROWS, a.rows) - 1) / a.G;
  const int diag = a.S - a.Q + 1;  // keys that token 0 sees
  const int keys_end = MASK ? a.S : min(a.S, diag + last_tok);
  const int begin = split * a.split_tiles;
  const int end = min(begin + a.split_tiles, (keys_end + kBlockTokens - 1) / kBlockTokens);
  Admit<Sh, MASK> admit;
  admit.row = MASK ? a.mask + b * a.mask_batch + tok * a.mask_q : nullptr;
  admit.mask_begin = a.mask_begin;
  admit.S = a.S;
  admit.lane_end = diag + tok;
  admit.some = MASK ? a.mask_begin > 0 : diag + tok > 0;
  admit.full = MASK ? min(a.S, a.mask_begin) : max(0, diag + first_row / a.G);

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

  int tile = begin + wave, special = 0;
  const int end8 = min(end, a.c.folded_blocks);
  // Blocks in 8 bits.  A tile's keys are loaded while the one before is worked
  // on; the registers of its values are filled again as soon as the products
  // are done with them.
  sf_u32x4 kr[kPieces], kn[kPieces], vr[kPieces];
  auto load_keys = [&](int t, sf_u32x4(&to)[kPieces]) {
    const char* p = k8 + static_cast<int64_t>(t) * (kBlockTokens * D);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
      to[n] = sf_ld16(p + 16 * Sh::key_piece(n / kKeyPairs, n % kKeyPairs));
  };
  auto load_values = [&](int t) {
    const char* p = v8 + static_cast<int64_t>(t) * (kBlockTokens * D);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
      vr[n] = sf_ld16(p + 16 * Sh::value_piece(n / kValuePairs, n % kValuePairs));
  };
  if (tile < end8) {
    load_keys(tile, kn);
    load_values(tile);
  }
  sf_u32x4 qf[Sh::kSteps];
  {
    const uint16_t* q = a.q + b * a.q_batch + q_head * a.q_head + tok * a.q_tok;
#pragma unroll
    for (int s = 0; s < Sh::kSteps; ++s)
      qf[s] = (sf_ld16(q + Sh::query_d(lane, s)) & a.keep) ^ a.flip;
  }
  Rows<D, ROWS> r;
  r.clear();
#pragma unroll 1
  for (; tile < end8; tile += kDirectWaves) {
    const int flag = ld(flags8 + tile);
    const float factor = a.scale_log2 * ld(k_scale + tile);
    const float scale_v = ld(v_scale + tile);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) kr[n] = kn[n];
    if (tile + kDirectWaves < end8) load_keys(tile + kDirectWaves, kn);
    admit.load(lane, tile * kBlockTokens);
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
    admit.restrict_scores(s, lane, tile * kBlockTokens);
    sf_u32x4 w[Sh::kPSteps], rest[Sh::kPSteps];
    r.softmax(s, factor, scale_v, w, rest);
    __builtin_amdgcn_sched_barrier(0);
    if (flag & kFlagValue) {  // in place: a second copy of the products takes registers
#pragma unroll
      for (int n = 0; n < kPieces; ++n) {
        vr[n] = finite_codes<HELD>(vr[n]);
        pin(vr[n]);
      }
    }
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int p = 0; p < kValuePairs; ++p) {
        sf_u32x4 x, y;
        sf_codes_frags<HELD>(vr[t * kValuePairs + p], x, y);
        r.acc[t] = Sh::mma(x, w[2 * p], r.acc[t]);
        r.acc[t] = Sh::mma(y, w[2 * p + 1], r.acc[t]);
        r.acc[t] = Sh::mma(x, rest[2 * p], r.acc[t]);
        r.acc[t] = Sh::mma(y, rest[2 * p + 1], r.acc[t]);
      }
    special |= flag;
    if (tile + kDirectWaves < end8) load_values(tile + kDirectWaves);
  }
  // Blocks of the ring.
#pragma unroll 1
  for (; tile < end; tile += kDirectWaves) {
    const int slot = tile % a.c.ring_blocks;
    const char* kp = kt + static_cast<int64_t>(slot) * (2 * kBlockTokens * D);
    const char* vp = vt + static_cast<int64_t>(slot) * (2 * kBlockTokens * D);
    const int flag = ld(tail_flags + slot);
    admit.load(lane, tile * kBlockTokens);
    Acc s[Sh::kScoreTiles];
#pragma unroll
    for (int t = 0; t < Sh::kScoreTiles; ++t) {
#pragma unroll
      for (int i = 0; i < kN; ++i) s[t][i] = 0.f;
#pragma unroll
      for (int st = 0; st < Sh::kSteps; ++st)
        s[t] = Sh::mma(sf_ld16(kp + 16 * Sh::key_piece16(t, st)), qf[st], s[t]);
    }
    // The values too, so that both are on their way together.
    sf_u32x4 v16[Sh::kOutTiles][Sh::kPSteps];
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int k = 0; k < Sh::kPSteps; ++k) v16[t][k] = sf_ld16(vp + 16 * Sh::value_piece16(t, k));
    admit.restrict_scores(s, lane, tile * kBlockTokens);
    sf_u32x4 w[Sh::kPSteps], rest[Sh::kPSteps];
    r.softmax(s, a.scale_log2, 1.f, w, rest);
    if (flag) {
#pragma unroll
      for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
        for (int k = 0; k < Sh::kPSteps; ++k) {
          v16[t][k] = entries<false>(v16[t][k], 3);
          pin(v16[t][k]);
        }
    }
#pragma unroll
    for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
      for (int k = 0; k < Sh::kPSteps; ++k) {
        r.acc[t] = Sh::mma(v16[t][k], w[k], r.acc[t]);
        r.acc[t] = Sh::mma(v16[t][k], rest[k], r.acc[t]);
      }
    special |= flag;
  }
  if (special)
    add_special<D, ROWS, HELD, MASK>(r, a, head, lane, begin + wave, end, kDirectWaves, admit);
  r.settle(admit.some != 0);

  // Merge the wavefronts' states in their order.
  constexpr int kRow = D + 4;
  __shared__ __attribute__((aligned(16))) float acc_lds[kDirectWaves][ROWS * kRow];
  __shared__ float2 ml_lds[kDirectWaves][ROWS];
  if (Sh::group(lane) == 0) ml_lds[wave][Sh::row(lane)] = make_float2(r.m, r.l);
#pragma unroll
  for (int t = 0; t < Sh::kOutTiles; ++t)
#pragma unroll
    for (int j = 0; j < kN / 4; ++j)
      *reinterpret_cast<float4*>(&acc_lds[wave][Sh::row(lane) * kRow + Sh::out_d(lane, t, j)]) =
          make_float4(r.acc[t][4 * j], r.acc[t][4 * j + 1], r.acc[t][4 * j + 2],
                      r.acc[t][4 * j + 3]);
  __syncthreads();
  for (int n = threadIdx.x; n < ROWS * D / 4; n += kDirectThreads) {
    const int rr = n / (D / 4);
    const int d = 4 * (n % (D / 4));
    const int out_row = first_row + rr;
    if (out_row >= a.rows) continue;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDirectWaves; ++w) M = fmaxf(M, ml_lds[w][rr].x);
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kDirectWaves; ++w) {
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
      const int64_t to = out_row_at(a, head, out_row);
      const float inv = M == -INFINITY ? 0.f : 1.f / l;
      *reinterpret_cast<uint2*>(a.out + to * D + d) =
          make_uint2(sf_pack_bf16(o[0] * inv, o[1] * inv), sf_pack_bf16(o[2] * inv, o[3] * inv));
    }
  }
}

// Elements d .. d + 3 of a row with M, divided by its sum.
template <int D>
__device__ __forceinline__ void store_merged(const Args& a, int head, int row, int d, const float4& o,
                                             float M, float l) {
  const float inv = M == -INFINITY ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(a.out + out_row_at(a, head, row) * D + d) =
      make_uint2(sf_pack_bf16(o.x * inv, o.y * inv), sf_pack_bf16(o.z * inv, o.w * inv));
}

__device__ __forceinline__ void add_scaled(float4& o, const float4& x, float f) {
  o.x = __builtin_fmaf(x.x, f, o.x);
  o.y = __builtin_fmaf(x.y, f, o.y);
  o.z = __builtin_fmaf(x.z, f, o.z);
  o.w = __builtin_fmaf(x.w, f, o.w);
}

constexpr int kMergeWaves = 4;
constexpr int kMergeThreads = kMergeWaves * SF_WAVE;
constexpr int kFewSplits = 16;
constexpr int kManyRows = 512;

// Merges few splits of many rows: D / 4 lanes per row, which go over its splits in
// their order with the values of four on their way.  Bound by the partial states'
// bytes: 8192 rows of 8 splits of 128 take 8.5 us (4 TB / s), 13.2 with a workgroup
// per row; 32 rows of 8 splits take 3.4, and 2.7 with a workgroup per row.
template <int D>
__global__ __launch_bounds__(kMergeThreads) void block_attention_merge_few_kernel(const Args a) {
  constexpr int kLanes = D / 4, kRows = kMergeThreads / kLanes;
  const int row = blockIdx.x * kRows + threadIdx.x / kLanes;
  const int head = blockIdx.y;
  const int d = 4 * (threadIdx.x % kLanes);
  if (row >= a.rows) return;
  const int64_t step = static_cast<int64_t>(a.c.heads) * a.rows;
  const int64_t at = static_cast<int64_t>(head) * a.rows + row;
  float2 ml[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) ml[s] = a.part_ml[min(s, a.splits - 1) * step + at];
  float M = -INFINITY;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) M = fmaxf(M, ml[s].x);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int s0 = 0; s0 < kFewSplits; s0 += 4) {
    if (s0 >= a.splits) break;
    float4 x[4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
      x[s] = *reinterpret_cast<const float4*>(a.part_acc +
                                              (min(s0 + s, a.splits - 1) * step + at) * D + d);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s0 + s >= a.splits || ml[s0 + s].x == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(ml[s0 + s].x - M);
      l = __builtin_fmaf(ml[s0 + s].y, f, l);
      add_scaled(o, x[s], f);
    }
  }
  store_merged<D>(a, head, row, d, o, M, l);
}

// Merges the splits of a row, if they are many or the rows few.  A thread looks at
// one split's (maximum, sum); groups of D / 4 lanes then add every kGroups-th
// accumulator, with their loads issued ahead of the weights, and the groups' sums
// are added in their order.
// (One after the other, the 128 splits of 8 rows took 16.9 us.)
template <int D>
__global__ __launch_bounds__(kMergeThreads) void block_attention_merge_kernel(const Args a) {
  constexpr int kLanes = D / 4, kGroups = kMergeThreads / kLanes;
  constexpr int kLoads = kMaxSplits / kGroups;
  static_assert(kMaxSplits <= kMergeThreads, "a thread per split");
  __shared__ float4 acc_lds[kGroups][kLanes];
  __shared__ float weight[kMaxSplits];
  __shared__ float top_lds[kMergeWaves], sum_lds[kMergeWaves];
  const int row = blockIdx.x;
  const int head = blockIdx.y;
  const int g = threadIdx.x / kLanes, d = 4 * (threadIdx.x % kLanes);
  const int64_t step = static_cast<int64_t>(a.c.heads) * a.rows;
  const int64_t at = static_cast<int64_t>(head) * a.rows + row;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (threadIdx.x < a.splits) ml = a.part_ml[threadIdx.x * step + at];
  float4 x[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
    if (j * kGroups < a.splits)
      x[j] = *reinterpret_cast<const float4*>(
          a.part_acc + (min(j * kGroups + g, a.splits - 1) * step + at) * D + d);
  const float wave_top = sf_wave_max(ml.x);
  if (threadIdx.x % SF_WAVE == 0) top_lds[threadIdx.x / SF_WAVE] = wave_top;
  __syncthreads();
  float M = top_lds[0];
#pragma unroll
  for (int w = 1; w < kMergeWaves; ++w) M = fmaxf(M, top_lds[w]);
  const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
  if (threadIdx.x < kMaxSplits) weight[threadIdx.x] = f;
  const float wave_sum = sf_wave_sum(ml.y * f);
  if (threadIdx.x % SF_WAVE == 0) sum_lds[threadIdx.x / SF_WAVE] = wave_sum;
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
    if (j * kGroups < a.splits && j * kGroups + g < a.splits) add_scaled(o, x[j], weight[j * kGroups + g]);
  acc_lds[g][threadIdx.x % kLanes] = o;
  __syncthreads();
  if (g != 0) return;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kGroups; ++i) add_scaled(o, acc_lds[i][threadIdx.x], 1.f);
  float l = sum_lds[0];
#pragma unroll
  for (int w = 1; w < kMergeWaves; ++w) l += sum_lds[w];
  store_merged<D>(a, head, row, d, o, M, l);
}

// How a call's rows and keys are dealt out.
struct Plan {
  bool staged;
  int rows, row_tiles, splits, split_tiles;
};

// The form and the splits that are expected to take the shortest, in us, with a
// workgroup per CU at a time.  Fitted to kernel times on MI355X (head dim 128; 64):
//   direct  3 + rounds (2 + 0.33 tiles)      (1 + 0.125 tiles)
//   staged  rounds (8 + 2.45 tiles)          (8 + 1.6 tiles)
//   splits  the partial states (fp32) at 4.5 MB / us, written and read, and 3 for
//           the second kernel
// The direct figures are from probabilities in one term (the second adds 2 - 9%, for
// heads of 64 up to 17%).  As the kernels are, in e4m3 at 32 / 4 heads of 128, direct / staged:
// a 61-node tree after 1024 tokens 9.5 / 19 us (split), 160 nodes after 8000 70 / 48
// (split), a prompt of 512 tokens 19 / 23, 1024 45 / 43, 2048 120 / 79; of 64: a prompt of
// 1000 21 / 30, 4000 168 / 112; 2000 tokens after 4000 at 16 / 4 heads of 64 93 / 91.
// tiles: of the longest row tile where there is one round, on average where there
// are more (as under the causal rule).
Plan plan_of(int heads, int group, int queries, int keys, int head_dim) {
  const int rows = queries * group;
  const int tiles = (keys + kBlockTokens - 1) / kBlockTokens;
  const double average = std::max(1., (keys - std::min(queries, keys) / 2) / double(kBlockTokens));
  const bool wide = head_dim == 128;
  Plan best = {};
  double best_cost = 0;
  for (const bool staged : {false, true}) {
    const int tile_rows = staged ? kStagedRows : kDirectRows;
    const int row_tiles = (rows + tile_rows - 1) / tile_rows;
    const int64_t base = static_cast<int64_t>(heads) * row_tiles;
    int last = 0;
    for (const int want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128}) {
      if (want > 1 && (base * want > 256 || want > tiles)) break;
      int split_tiles = (tiles + want - 1) / want;
      // The direct form's wavefronts take a tile each at a time.
      if (want > 1 && !staged) split_tiles = (split_tiles + kDirectWaves - 1) / kDirectWaves * kDirectWaves;
      const int splits = (tiles + split_tiles - 1) / split_tiles;
      if (splits == last) continue;
      last = splits;
      const double rounds = static_cast<double>((base * splits + 255) / 256);
      const double each = rounds > 1 ? std::min<double>(average, split_tiles) : split_tiles;
      double cost = staged ? rounds * (8 + (wide ? 2.45 : 1.6) * each)
                           : 3 + rounds * (wide ? 2 + 0.33 * each : 1 + 0.125 * each);
      if (splits > 1)
        cost += 3 + 2 * 4. * (head_dim + 2) * heads * static_cast<double>(rows) * splits / 4.5e6;
      if (best.rows == 0 || cost < best_cost) {
        best = {staged, rows, row_tiles, splits, split_tiles};
        best_cost = cost;
      }
    }
  }
  return best;
}

template <int D, int HELD>
void launch_held(const Args& a, bool staged, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(a.c.heads) * a.row_tiles * a.splits);
  if (staged) {
    if (a.mask)
      block_attention_staged_kernel<D, HELD, true><<<grid, kStagedThreads, 0, s>>>(a);
    else
      block_attention_staged_kernel<D, HELD, false><<<grid, kStagedThreads, 0, s>>>(a);
  } else {
    if (a.mask)
      block_attention_direct_kernel<D, HELD, true><<<grid, kDirectThreads, 0, s>>>(a);
    else
      block_attention_direct_kernel<D, HELD, false><<<grid, kDirectThreads, 0, s>>>(a);
  }
}

template <int D>
void launch(const Args& a, bool staged, hipStream_t s) {
  if (a.c.held == SF_KV_INT8)
    launch_held<D, SF_KV_INT8>(a, staged, s);
  else
    launch_held<D, SF_KV_E4M3>(a, staged, s);
  constexpr int kRows = kMergeThreads / (D / 4);
  if (a.splits > kFewSplits || (a.splits > 1 && a.rows * int64_t{a.c.heads} < kManyRows))
    block_attention_merge_kernel<D><<<dim3(a.rows, a.c.heads), kMergeThreads, 0, s>>>(a);
  else if (a.splits > 1)
    block_attention_merge_few_kernel<D>
        <<<dim3((a.rows + kRows - 1) / kRows, a.c.heads), kMergeThreads, 0, s>>>(a);
}

// Keys, and rows over all heads, of a call, so that every index of tiles, rows
// and workgroups stays in 32 bits.
constexpr int64_t kMaxKeys = 1 << 30;
constexpr int64_t kMaxRows = 1 << 24;

bool fits(int64_t heads, int64_t group, int64_t queries, int64_t keys) {
  return keys <= kMaxKeys && queries <= kMaxRows / group && heads <= 65535 &&
         queries * group * heads <= kMaxRows;
}

// False for shapes that no call takes.
bool plan_for(int batch, int queries, int keys, int q_heads, int kv_heads, int head_dim, Plan* p) {
  if (batch < 1 || queries < 1 || keys < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads ||
      (head_dim != 64 && head_dim != 128))
    return false;
  const int64_t heads = static_cast<int64_t>(batch) * kv_heads;
  if (!fits(heads, q_heads / kv_heads, queries, keys)) return false;
  *p = plan_of(static_cast<int>(heads), q_heads / kv_heads, queries, keys, head_dim);
  return true;
}

}  // namespace

extern "C" int64_t sf_block_attention_workspace(int batch, int queries, int keys, int q_heads,
                                                int kv_heads, int head_dim) {
  Plan p;
  if (!plan_for(batch, queries, keys, q_heads, kv_heads, head_dim, &p) || p.splits == 1) return 0;
  return static_cast<int64_t>(p.splits) * batch * kv_heads * p.rows * (head_dim + 2) * 4;
}

extern "C" int sf_block_attention_rows(int batch, int queries, int keys, int q_heads, int kv_heads,
                                       int head_dim) {
  Plan p;
  if (!plan_for(batch, queries, keys, q_heads, kv_heads, head_dim, &p)) return 0;
  return p.staged ? kStagedRows : kDirectRows;
}

extern "C" int sf_block_attention(const sf_kv_cache* cache, int batch, int kv_heads, int keys,
                                  const void* q, int64_t q_stride_batch, int64_t q_stride_head,
                                  int64_t q_stride_token, int queries, int q_heads,
                                  const uint8_t* mask, int64_t mask_stride_batch,
                                  int64_t mask_stride_query, int mask_keys, float scale, void* out,
                                  void* workspace, int64_t workspace_bytes, sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (batch < 1 || kv_heads < 1 || batch > cache->heads ||
      static_cast<int64_t>(batch) * kv_heads != cache->heads ||
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
  Plan p = plan_of(cache->heads, group, queries, keys, cache->head_dim);
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
    launch<128>(a, p.staged, s);
  else
    launch<64>(a, p.staged, s);
  SF_LAUNCH_CHECK();
  return SF_OK;
}
