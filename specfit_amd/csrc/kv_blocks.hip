// K9: writing, compacting, folding and reading the block cache (its layout is
// in kv_blocks.h).  All four are copies that change the order of values; the
// workgroup of a block owns it, so nothing is shared between workgroups.
// Bound by latency for a few tokens (3.7 - 4.7 us each) and by memory for many:
// 8192 tokens of 4 heads of 128 take 7.6 us to append (34 MB, 4.4 TB/s), 7.1 to
// fold (25 MB) and 7.5 to read back (25 MB).
#include "kv_blocks.h"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ bool nonfinite(uint32_t bf16) { return (bf16 & 0x7f80u) == 0x7f80u; }

// Piece and element of value (token row of the block, d).
template <int D>
__device__ __forceinline__ int value_at(int row, int d) {
  const int lane = 32 * ((row >> 2) & 1) + (d & 31);
  const int i = 4 * ((row >> 3) & 1) + (row & 3);
  return (((d >> 5) * 4 + (row >> 4)) * SF_WAVE + lane) * 8 + i;
}

// Piece of the eight key elements 8 p .. 8 p + 7 of a token row of the block.
template <int D>
__device__ __forceinline__ int key_piece(int row, int p) {
  const int s = 2 * (p >> 2) + (p & 1);
  return ((row >> 5) * (D / 16) + s) * SF_WAVE + 32 * ((p >> 1) & 1) + (row & 31);
}

// ---------------------------------------------------------------- append --
struct Rows {
  const uint16_t *k, *v;
  int64_t k_batch, k_head, k_tok, v_batch, v_head, v_tok;
};

template <int D>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(
    const sf_kv_cache c, const Rows in, int kv_heads, int64_t start, int64_t end, int aligned) {
  const int64_t block = start / kBlockTokens + blockIdx.x;
  const int head = blockIdx.y;
  const int b = head / kv_heads;
  const int h = head - b * kv_heads;
  const int64_t first = block * kBlockTokens;
  const int r0 = static_cast<int>(max(start - first, static_cast<int64_t>(0)));
  const int r1 = static_cast<int>(min(end - first, static_cast<int64_t>(kBlockTokens)));
  const int slot = static_cast<int>(block % c.ring_blocks);
  const int64_t at = (static_cast<int64_t>(head) * c.ring_blocks + slot) * (kBlockTokens * D);
  uint16_t* kt = static_cast<uint16_t*>(c.k_tail) + at;
  uint16_t* vt = static_cast<uint16_t*>(c.v_tail) + at;
  // Row r of the block is token first + r: row first + r - start of the input.
  const uint16_t* k = in.k + b * in.k_batch + h * in.k_head + (first - start) * in.k_tok;
  const uint16_t* v = in.v + b * in.v_batch + h * in.v_head + (first - start) * in.v_tok;

  constexpr int kPieces = D / 8;
  for (int i = r0 * kPieces + threadIdx.x; i < r1 * kPieces; i += kThreads) {
    const int row = i / kPieces;
    const int p = i - row * kPieces;
    const uint16_t* src = k + row * in.k_tok + 8 * p;
    sf_u32x4 x;
    if (aligned) {
      x = sf_ld16(src);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = src[2 * j] | static_cast<uint32_t>(src[2 * j + 1]) << 16;
    }
    *reinterpret_cast<sf_u32x4*>(kt + 8 * key_piece<D>(row, p)) = x;
  }

  // Values: a piece holds eight tokens of one d.  Rows behind the new ones
  // become zeros, so that what the ring held there before meets no product.
  // All loads of a thread are issued together (rows that are not new read a
  // new one's place and drop it): one token takes 3.7 us and 61 take 4.3; with
  // a branch around each load they took 4.1 and 7.9.
  constexpr int kValuePieces = kBlockTokens * D / 8 / kThreads;
  uint16_t y[kValuePieces][8];
  sf_u32x4 old[kValuePieces];
#pragma unroll
  for (int j = 0; j < kValuePieces; ++j) {
    const int n = j * kThreads + threadIdx.x;
    const int lane = n & (SF_WAVE - 1);
    const int d = 32 * (n >> 8) + (lane & 31);
    const int row = 16 * ((n >> 6) & 3) + 4 * (lane >> 5);  // and row + 8: four rows each
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = min(max(row + 8 * (i >> 2) + (i & 3), r0), r1 - 1);
      y[j][i] = v[r * in.v_tok + d];
    }
    if (r0) old[j] = sf_ld16(vt + 8 * n);
  }
  int bad = 0;
#pragma unroll
  for (int j = 0; j < kValuePieces; ++j) {
    const int n = j * kThreads + threadIdx.x;
    const int row = 16 * ((n >> 6) & 3) + 4 * ((n & (SF_WAVE - 1)) >> 5);
    sf_u32x4 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = row + 8 * (i >> 2) + (i & 3);
      const uint32_t fresh = r < r1 ? y[j][i] : 0u;
      bad |= nonfinite(y[j][i]);
      const uint32_t kept = r0 ? (old[j][i >> 1] >> (16 * (i & 1))) & 0xffffu : 0u;
      const uint32_t z = r < r0 ? kept : fresh;
      x[i >> 1] = i & 1 ? x[i >> 1] | z << 16 : z;
    }
    *reinterpret_cast<sf_u32x4*>(vt + 8 * n) = x;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    int32_t* flag = c.tail_flags + static_cast<int64_t>(head) * c.ring_blocks + slot;
    *flag = (bad ? kFlagValue : 0) | (r0 ? *flag : 0);
  }
}

// --------------------------------------------------------------- compact --
struct Moves {
  int32_t from[SF_KV_MAX_MOVES];
};

constexpr int kMoveRows = 16;  // rows moved between two barriers

// One workgroup per head moves its rows in ascending order: a later pass reads
// from behind every row that earlier ones wrote (positions ascend strictly, so
// from[i] >= first + i), and a pass writes after it has read.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_compact_kernel(const sf_kv_cache c, int64_t base,
                                                              int first, int count,
                                                              const Moves moves) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * c.ring_blocks * (kBlockTokens * D);
  uint16_t* kt = static_cast<uint16_t*>(c.k_tail) + at;
  uint16_t* vt = static_cast<uint16_t*>(c.v_tail) + at;
  auto slot = [&](int64_t token) {
    return ((token / kBlockTokens) % c.ring_blocks) * (kBlockTokens * D);
  };
  constexpr int kPieces = D / 8;
  constexpr int kKeyLoads = kMoveRows * kPieces / kThreads > 0 ? kMoveRows * kPieces / kThreads : 1;
  constexpr int kValueLoads = kMoveRows * D / kThreads;
  for (int i0 = 0; i0 < count; i0 += kMoveRows) {
    sf_u32x4 kx[kKeyLoads];
    uint16_t vx[kValueLoads];
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const int n = j * kThreads + threadIdx.x;
      const int i = i0 + n / kPieces;
      if (n / kPieces < kMoveRows && i < count) {
        const int64_t from = base + moves.from[i];
        kx[j] = *reinterpret_cast<const sf_u32x4*>(
            kt + slot(from) + 8 * key_piece<D>(from % kBlockTokens, n % kPieces));
      }
    }
#pragma unroll
    for (int j = 0; j < kValueLoads; ++j) {
      const int n = j * kThreads + threadIdx.x;
      const int i = i0 + n / D;
      if (i < count) {
        const int64_t from = base + moves.from[i];
        vx[j] = vt[slot(from) + value_at<D>(from % kBlockTokens, n % D)];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const int n = j * kThreads + threadIdx.x;
      const int i = i0 + n / kPieces;
      if (n / kPieces < kMoveRows && i < count) {
        const int64_t to = base + first + i;
        *reinterpret_cast<sf_u32x4*>(kt + slot(to) +
                                     8 * key_piece<D>(to % kBlockTokens, n % kPieces)) = kx[j];
      }
    }
#pragma unroll
    for (int j = 0; j < kValueLoads; ++j) {
      const int n = j * kThreads + threadIdx.x;
      const int i = i0 + n / D;
      if (i < count) {
        const int64_t to = base + first + i;
        vt[slot(to) + value_at<D>(to % kBlockTokens, n % D)] = vx[j];
      }
    }
    __syncthreads();
  }
  // A block that took rows may now hold what the blocks behind it were
  // flagged for.
  if (threadIdx.x == 0) {
    int32_t* flags = c.tail_flags + static_cast<int64_t>(blockIdx.x) * c.ring_blocks;
    const int64_t b0 = (base + first) / kBlockTokens;
    const int64_t b1 = (base + moves.from[count - 1]) / kBlockTokens;
    int any = 0;
    for (int64_t b = b0; b <= b1; ++b) any |= flags[b % c.ring_blocks];
    if (any)
      for (int64_t b = b0; b <= (base + first + count - 1) / kBlockTokens; ++b)
        flags[b % c.ring_blocks] = any;
  }
}

// ------------------------------------------------------------------ fold --
// One workgroup per (block, head, K or V): both orders pair the bf16 pieces of
// an 8-bit piece in the same way.
template <int D, int HELD>
__global__ __launch_bounds__(kThreads) void kv_fold_kernel(const sf_kv_cache c) {
  const int block = c.folded_blocks + blockIdx.x;
  const int64_t head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const uint16_t* src =
      static_cast<const uint16_t*>(values ? c.v_tail : c.k_tail) +
      (head * c.ring_blocks + block % c.ring_blocks) * (kBlockTokens * D);
  const int64_t to = head * c.capacity_blocks + block;
  uint8_t* dst = static_cast<uint8_t*>(values ? c.v8 : c.k8) + to * (kBlockTokens * D);
  constexpr int kPieces = kBlockTokens * D / 16 / kThreads;  // 8-bit pieces per thread
  static_assert(kPieces >= 1, "a thread folds whole pieces");

  sf_u32x4 x[kPieces][2];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int n = j * kThreads + threadIdx.x;
    const uint16_t* p = src + 8 * (128 * (n / SF_WAVE) + n % SF_WAVE);
    x[j][0] = sf_ld16(p);
    x[j][1] = sf_ld16(p + 8 * SF_WAVE);
  }
  uint32_t top = 0;  // of the magnitudes, as bits of fp32: they order as integers
  int bad = 0;
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t w = x[j][i >> 3][(i >> 1) & 3];
      const uint32_t m = (i & 1 ? w & 0x7fff0000u : w << 16) & 0x7fff0000u;
      if (m >= 0x7f800000u)
        bad = 1;
      else
        top = max(top, m);
    }
  __shared__ int tops[kThreads / SF_WAVE];
  top = static_cast<uint32_t>(sf_wave_max_int(static_cast<int>(top)));
  if (threadIdx.x % SF_WAVE == 0) tops[threadIdx.x / SF_WAVE] = static_cast<int>(top);
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < kThreads / SF_WAVE; ++w) top = max(top, static_cast<uint32_t>(tops[w]));

  // top = m 2^x with m in [1/2, 1): the least e with m 2^x <= q 2^e, where q
  // is 127/128 2^7 or 7/8 2^9.  (A subnormal top is below every 2^e here.)
  const int exponent = static_cast<int>(top >> 23) - 126;
  const uint32_t fraction = top & 0x7fffffu;
  const int e = max(SF_KV_MIN_EXPONENT, HELD == SF_KV_INT8
                                            ? exponent - (fraction <= 0x7e0000u ? 7 : 6)
                                            : exponent - (fraction <= 0x600000u ? 9 : 8));
  const float inverse = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    sf_u32x4 y;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t codes = 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w = x[j][q >> 1][2 * (q & 1) + half];
        const uint32_t u[2] = {w << 16, w & 0xffff0000u};
        uint32_t pair = 0;
        if (HELD == SF_KV_INT8) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = __builtin_rintf(__uint_as_float(u[i]) * inverse);
            const int code = nonfinite(u[i] >> 16) ? -128 : static_cast<int>(f);
            pair |= (static_cast<uint32_t>(code) & 0xffu) << (8 * i);
          }
        } else {
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            f[i] = nonfinite(u[i] >> 16) ? 0.f : __uint_as_float(u[i]) * inverse;
          pair = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false)) &
                 0xffffu;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (nonfinite(u[i] >> 16)) pair |= 0x7fu << (8 * i);
        }
        codes |= pair << (16 * half);
      }
      y[q] = codes;
    }
    *reinterpret_cast<sf_u32x4*>(dst + 16 * (j * kThreads + threadIdx.x)) = y;
  }
  if (threadIdx.x == 0) {
    (values ? c.v_scale : c.k_scale)[to] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    // The two workgroups of a block set a bit each.
    if (bad)
      atomicOr(&c.flags[to], values ? kFlagValue : kFlagKey);
    else
      atomicAnd(&c.flags[to], ~(values ? kFlagValue : kFlagKey));
  }
}

// ------------------------------------------------------------------ read --
template <int HELD>
__device__ __forceinline__ float code_value(uint32_t code, float scale) {
  if (HELD == SF_KV_INT8) {
    const int v = static_cast<int8_t>(code);
    return v == -128 ? __builtin_nanf("") : static_cast<float>(v) * scale;
  }
  uint32_t lo, hi;
  sf_codes_bf16<SF_KV_E4M3>(code & 0xffu, lo, hi);
  return __uint_as_float(lo << 16) * scale;
}

template <int D, int HELD>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const sf_kv_cache c, int64_t start,
                                                           int64_t end, uint16_t* k_out,
                                                           uint16_t* v_out) {
  // Rows of one of the two, padded by 16 bytes.
  constexpr int kRow = D + 8;
  __shared__ __attribute__((aligned(16))) uint16_t rows[kBlockTokens * kRow];
  const int64_t block = start / kBlockTokens + blockIdx.x;
  const int64_t head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  if (block < c.folded_blocks) {
    const int64_t at = head * c.capacity_blocks + block;
    const uint8_t* src = static_cast<const uint8_t*>(values ? c.v8 : c.k8) + at * (kBlockTokens * D);
    const float scale = (values ? c.v_scale : c.k_scale)[at];
    for (int n = threadIdx.x; n < kBlockTokens * D / 16; n += kThreads) {
      const sf_u32x4 x = sf_ld16(src + 16 * n);
      const int g = n / SF_WAVE, lane = n % SF_WAVE;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint16_t y = sf_f32_to_bf16(code_value<HELD>(x[i >> 2] >> (8 * (i & 3)) & 0xffu, scale));
        if (values) {
          const int ks = 2 * (g & 1) + (i >> 3);
          const int row = 16 * ks + 8 * ((i >> 2) & 1) + 4 * (lane >> 5) + (i & 3);
          rows[row * kRow + 32 * (g >> 1) + (lane & 31)] = y;
        } else {
          const int kh = g / (D / 32), jj = g % (D / 32);
          rows[(32 * kh + (lane & 31)) * kRow + 32 * jj + 16 * (lane >> 5) + i] = y;
        }
      }
    }
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(values ? c.v_tail : c.k_tail) +
                          (head * c.ring_blocks + block % c.ring_blocks) * (kBlockTokens * D);
    for (int n = threadIdx.x; n < kBlockTokens * D / 8; n += kThreads) {
      const sf_u32x4 x = sf_ld16(src + 8 * n);
      const int g = n / SF_WAVE, lane = n % SF_WAVE;
      if (values) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 16 * (g & 3) + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
          rows[row * kRow + 32 * (g >> 2) + (lane & 31)] =
              static_cast<uint16_t>(x[i >> 1] >> (16 * (i & 1)));
        }
      } else {
        const int kh = g / (D / 16), s = g % (D / 16);
        *reinterpret_cast<sf_u32x4*>(rows + (32 * kh + (lane & 31)) * kRow + 32 * (s >> 1) +
                                     16 * (lane >> 5) + 8 * (s & 1)) = x;
      }
    }
  }
  __syncthreads();
  uint16_t* out = (values ? v_out : k_out) + head * (end - start) * D;
  constexpr int kPieces = D / 8;
  for (int n = threadIdx.x; n < kBlockTokens * kPieces; n += kThreads) {
    const int row = n / kPieces, p = n % kPieces;
    const int64_t token = block * kBlockTokens + row;
    if (token < start || token >= end) continue;
    *reinterpret_cast<sf_u32x4*>(out + (token - start) * D + 8 * p) =
        *reinterpret_cast<const sf_u32x4*>(rows + row * kRow + 8 * p);
  }
}

}  // namespace

// What every call asks of the cache's description.
int sf_kv_check(const sf_kv_cache* c) {
  if (!c || c->heads < 1 || c->capacity_blocks < 1 || c->ring_blocks < 1 || c->folded_blocks < 0 ||
      c->folded_blocks > c->capacity_blocks || (c->held != SF_KV_E4M3 && c->held != SF_KV_INT8))
    return SF_ERR_INVALID_ARGUMENT;
  if (c->head_dim != 64 && c->head_dim != 128) return SF_ERR_UNSUPPORTED_SHAPE;
  if (c->heads > 65535) return SF_ERR_UNSUPPORTED_SHAPE;
  if (!c->k8 || !c->v8 || !c->k_scale || !c->v_scale || !c->flags || !c->k_tail || !c->v_tail ||
      !c->tail_flags)
    return SF_ERR_INVALID_ARGUMENT;
  for (const void* p : {c->k8, c->v8, c->k_tail, c->v_tail})
    if (reinterpret_cast<uintptr_t>(p) % 16) return SF_ERR_MISALIGNED;
  return SF_OK;
}

namespace {

// A start or base above it is refused before it meets a sum.
int64_t token_capacity(const sf_kv_cache* c) {
  return static_cast<int64_t>(c->capacity_blocks) * kBlockTokens;
}

// Tokens [start, end) lie in the capacity, and what is not folded of the
// sequence up to `end` in the ring.
bool in_ring(const sf_kv_cache* c, int64_t start, int64_t end) {
  if (end > token_capacity(c)) return false;
  const int64_t last = (end + kBlockTokens - 1) / kBlockTokens;
  return start >= 0 && start <= end && start >= static_cast<int64_t>(c->folded_blocks) * kBlockTokens &&
         last <= c->capacity_blocks && last - c->folded_blocks <= c->ring_blocks;
}

}  // namespace

extern "C" int sf_kv_append(const sf_kv_cache* cache, int kv_heads, const void* k,
                            int64_t k_stride_batch, int64_t k_stride_head, int64_t k_stride_token,
                            const void* v, int64_t v_stride_batch, int64_t v_stride_head,
                            int64_t v_stride_token, int64_t start, int tokens,
                            sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (kv_heads < 1 || cache->heads % kv_heads || tokens < 0) return SF_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return SF_OK;
  if (!k || !v || start < 0 || start > token_capacity(cache) ||
      !in_ring(cache, start, start + tokens))
    return SF_ERR_INVALID_ARGUMENT;
  const Rows in = {static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                   k_stride_batch, k_stride_head, k_stride_token,
                   v_stride_batch, v_stride_head, v_stride_token};
  const int aligned = reinterpret_cast<uintptr_t>(k) % 16 == 0 && k_stride_batch % 8 == 0 &&
                      k_stride_head % 8 == 0 && k_stride_token % 8 == 0;
  const int64_t end = start + tokens;
  const int blocks = static_cast<int>((end + kBlockTokens - 1) / kBlockTokens - start / kBlockTokens);
  const dim3 grid(blocks, cache->heads);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    kv_append_kernel<128><<<grid, kThreads, 0, s>>>(*cache, in, kv_heads, start, end, aligned);
  else
    kv_append_kernel<64><<<grid, kThreads, 0, s>>>(*cache, in, kv_heads, start, end, aligned);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

extern "C" int sf_kv_compact(const sf_kv_cache* cache, int64_t base, int first,
                             const int32_t* positions, int count, int64_t end,
                             sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (count < 0 || count > SF_KV_MAX_MOVES || first < 0 || base < 0) return SF_ERR_INVALID_ARGUMENT;
  if (count == 0) return SF_OK;
  if (!positions || base > token_capacity(cache) || !in_ring(cache, base + first, end))
    return SF_ERR_INVALID_ARGUMENT;
  Moves moves = {};
  for (int i = 0; i < count; ++i) {
    if (positions[i] < first + i || (i && positions[i] <= positions[i - 1]) ||
        base + positions[i] >= end)
      return SF_ERR_INVALID_ARGUMENT;
    moves.from[i] = positions[i];
  }
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    kv_compact_kernel<128><<<cache->heads, kThreads, 0, s>>>(*cache, base, first, count, moves);
  else
    kv_compact_kernel<64><<<cache->heads, kThreads, 0, s>>>(*cache, base, first, count, moves);
  SF_LAUNCH_CHECK();
  return SF_OK;
}

extern "C" int sf_kv_fold(const sf_kv_cache* cache, int blocks, sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (blocks < 0) return SF_ERR_INVALID_ARGUMENT;
  if (blocks == 0) return SF_OK;
  if (blocks > cache->ring_blocks || blocks > cache->capacity_blocks - cache->folded_blocks)
    return SF_ERR_INVALID_ARGUMENT;
  const dim3 grid(blocks, cache->heads, 2);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool int8 = cache->held == SF_KV_INT8;
  if (cache->head_dim == 128) {
    if (int8)
      kv_fold_kernel<128, SF_KV_INT8><<<grid, kThreads, 0, s>>>(*cache);
    else
      kv_fold_kernel<128, SF_KV_E4M3><<<grid, kThreads, 0, s>>>(*cache);
  } else {
    if (int8)
      kv_fold_kernel<64, SF_KV_INT8><<<grid, kThreads, 0, s>>>(*cache);
    else
      kv_fold_kernel<64, SF_KV_E4M3><<<grid, kThreads, 0, s>>>(*cache);
  }
  SF_LAUNCH_CHECK();
  return SF_OK;
}

extern "C" int sf_kv_read(const sf_kv_cache* cache, int64_t start, int tokens, void* k, void* v,
                          sf_stream_t stream) {
  if (const int rc = sf_kv_check(cache)) return rc;
  if (tokens < 0 || start < 0 || start > token_capacity(cache)) return SF_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return SF_OK;
  const int64_t end = start + tokens;
  const int64_t last = (end + kBlockTokens - 1) / kBlockTokens;
  if (!k || !v || last > cache->capacity_blocks ||
      last - cache->folded_blocks > cache->ring_blocks)
    return SF_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
    return SF_ERR_MISALIGNED;
  const dim3 grid(static_cast<int>(last - start / kBlockTokens), cache->heads, 2);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint16_t* ko = static_cast<uint16_t*>(k);
  uint16_t* vo = static_cast<uint16_t*>(v);
  const bool int8 = cache->held == SF_KV_INT8;
  if (cache->head_dim == 128) {
    if (int8)
      kv_read_kernel<128, SF_KV_INT8><<<grid, kThreads, 0, s>>>(*cache, start, end, ko, vo);
    else
      kv_read_kernel<128, SF_KV_E4M3><<<grid, kThreads, 0, s>>>(*cache, start, end, ko, vo);
  } else {
    if (int8)
      kv_read_kernel<64, SF_KV_INT8><<<grid, kThreads, 0, s>>>(*cache, start, end, ko, vo);
    else
      kv_read_kernel<64, SF_KV_E4M3><<<grid, kThreads, 0, s>>>(*cache, start, end, ko, vo);
  }
  SF_LAUNCH_CHECK();
  return SF_OK;
}
