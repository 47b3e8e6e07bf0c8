// K12: repetition penalties, a bias and an allowed set on rows of logits, and
// each row's greedy token.
//
// A thread has eight vocabulary entries of a row; the tokens of the row's own path
// are found by the wavefront that holds their entries.  The greedy token is a
// maximum of (value, lowest index) over partial results of the wavefronts, so no
// order of arrival changes it.  Bound by the bytes of the logits, and with
// penalties by their vector work (a quotient costs three instructions, see
// `divided`).
#include <algorithm>

#include "sf_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / SF_WAVE;
constexpr int kPer = 8;                     // entries of a thread
constexpr int kChunk = kThreads * kPer;     // of a workgroup
constexpr int kNone = INT32_MIN;            // key of a value that is never chosen

struct RuleArgs {
  const void* logits;
  int64_t stride;
  int rows, vocab;
  const int32_t* counts;
  const int32_t* paths;
  int path_length;
  float repetition, inverse, presence, frequency;  // inverse: of the repetition, or 0
  const float* bias;
  int64_t bias_stride;
  const int32_t* allowed;
  int64_t allowed_stride;
  void* out;
  int64_t out_stride;
  int2* parts;  // [rows][chunks * kWaves] (key, index), or nullptr
  int chunks;
};

template <int DTYPE>
struct Type;
template <>
struct Type<SF_BF16> {
  typedef uint16_t Elem;
  static __device__ __forceinline__ float load(uint16_t v) { return sf_bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t store(float v) { return sf_f32_to_bf16(v); }
};
template <>
struct Type<SF_F16> {
  typedef uint16_t Elem;
  static __device__ __forceinline__ float load(uint16_t v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  static __device__ __forceinline__ uint16_t store(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  }
};
template <>
struct Type<SF_F32> {
  typedef float Elem;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
};

// Integers in the order of floats, a NaN above all; -inf is never chosen.
__device__ __forceinline__ int order_key(float y) {
  const int u = __float_as_int(y + 0.f);  // -0 as 0
  if (y != y) return INT32_MAX;
  if (y == -INFINITY) return kNone;
  return u >= 0 ? u : u ^ 0x7fffffff;
}

// x / repetition, correctly rounded.  With the correctly rounded inverse y of b,
// q = x y is within an ulp or so of x / b, its remainder r = x - q b is exact in a
// fused multiply-add, and q + r y rounds to the quotient (Markstein, 1990), as long as
// nothing overflows or loses bits below the normal range: |x| between the two
// limits, for a repetition that has an inverse here.
__device__ __forceinline__ float divided(float x, float b, float y) {
  const float q = x * y;
  return __builtin_fmaf(__builtin_fmaf(-q, b, x), y, q);
}
constexpr float kLeastPlain = 0x1p-90f, kMostPlain = 0x1p100f;

// Entry e of thread tid: VEC neighbours, then the next kThreads * VEC.
template <int VEC>
__device__ __forceinline__ int entry(int tid, int e) {
  return (e / VEC) * (kThreads * VEC) + tid * VEC + e % VEC;
}

// The kPer entries of a thread from p (entry 0 of the chunk), n of them there.
template <int VEC, typename E>
__device__ __forceinline__ void load_entries(const E* p, int n, E (&x)[kPer]) {
  struct __attribute__((aligned(VEC * sizeof(E) > 16 ? 16 : VEC * sizeof(E)))) Piece {
    E e[VEC];
  };
#pragma unroll
  for (int e = 0; e < kPer; e += VEC) {
    const int at = entry<VEC>(threadIdx.x, e);
    if (at + VEC <= n) {
      const Piece q = *reinterpret_cast<const Piece*>(p + at);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[e + j] = q.e[j];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[e + j] = at + j < n ? p[at + j] : E(0);
    }
  }
}

// A workgroup has a chunk of one row.  Two or four rows to a workgroup read the
// counts once for them, but their registers leave half of the wavefronts: 61 rows of
// 151936 bf16 logits take 9.4 us with one, 12.5 with two, 15.4 with four (5.9
// without any rule).
template <int DTYPE, int VEC, bool PENALTY, bool OUT, bool TOKENS>
__global__ __launch_bounds__(kThreads) void logit_rules_kernel(const RuleArgs a) {
  using Ty = Type<DTYPE>;
  using Elem = typename Ty::Elem;
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int wave = threadIdx.x / SF_WAVE;
  const int c0 = blockIdx.x * kChunk;
  const int n = min(kChunk, a.vocab - c0);  // entries of the chunk
  const int r = blockIdx.y;

  // Everything the row needs is on its way together.
  Elem raw[kPer];
  load_entries<VEC>(static_cast<const Elem*>(a.logits) + r * a.stride + c0, n, raw);
  int32_t count[kPer] = {};
  if (PENALTY && a.counts) load_entries<VEC>(a.counts + c0, n, count);
  const int32_t* path = a.paths + static_cast<int64_t>(r) * a.path_length;
  int own = -1;
  if (PENALTY && a.paths && lane < a.path_length) own = path[lane];
  uint32_t good = 0;  // entries that are there and allowed
#pragma unroll
  for (int e = 0; e < kPer; ++e) good |= (entry<VEC>(threadIdx.x, e) < n ? 1u : 0u) << e;
  if (a.allowed) {
    const int32_t* words = a.allowed + r * a.allowed_stride;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < kPer; e += VEC) {
      // VEC neighbours share a word: chunks and VEC divide or are multiples of 32.
      const int v = c0 + min(entry<VEC>(threadIdx.x, e), n - 1);
      bits |= ((static_cast<uint32_t>(words[v / 32]) >> (v % 32)) & ((1u << VEC) - 1u)) << e;
    }
    good &= bits;
  }

  float y[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) y[e] = Ty::load(raw[e]);
  if (PENALTY) {
    // The row's own tokens: few chunks have any.
    if (a.paths)
      for (int p0 = 0; p0 < a.path_length; p0 += SF_WAVE) {
        if (p0) own = p0 + lane < a.path_length ? path[p0 + lane] : -1;
        uint64_t here = __ballot(own >= c0 && own < c0 + n);
        while (here) {  // uniform
          const int at =
              __builtin_amdgcn_readlane(own, static_cast<int>(__builtin_ctzll(here))) - c0;
          here &= here - 1;
#pragma unroll
          for (int e = 0; e < kPer; ++e) count[e] += entry<VEC>(threadIdx.x, e) == at;
        }
      }
    float least = fabsf(y[0]), most = fabsf(y[0]);
#pragma unroll
    for (int e = 1; e < kPer; ++e) {
      least = fminf(least, fabsf(y[e]));
      most = fmaxf(most, fabsf(y[e]));
    }
    // (A NaN is in neither: its quotient is NaN both ways.)
    const bool quick = a.inverse != 0.f && !__any(!(least >= kLeastPlain && most <= kMostPlain));
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (!__any(count[e] > 0)) continue;
      float x = quick ? divided(y[e], a.repetition, a.inverse) : y[e] / a.repetition;
      if (y[e] < 0.f) x = y[e] * a.repetition;
      x -= a.frequency * static_cast<float>(count[e]) + a.presence;
      if (count[e] > 0) y[e] = x;
    }
  }
  if (a.bias) {
    float bias[kPer];
    load_entries<VEC>(a.bias + r * a.bias_stride + c0, n, bias);
#pragma unroll
    for (int e = 0; e < kPer; ++e) y[e] += bias[e];
  }
  Elem out[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const uint32_t keep = static_cast<uint32_t>(static_cast<int32_t>(good << (31 - e)) >> 31);
    y[e] = __uint_as_float((keep & __float_as_uint(y[e])) | (~keep & 0xff800000u));
    if (OUT) out[e] = Ty::store(y[e]);
  }
  if (OUT) {
    struct __attribute__((aligned(VEC * sizeof(Elem) > 16 ? 16 : VEC * sizeof(Elem)))) Piece {
      Elem e[VEC];
    };
    Elem* to = static_cast<Elem*>(a.out) + r * a.out_stride + c0;
#pragma unroll
    for (int e = 0; e < kPer; e += VEC) {
      const int at = entry<VEC>(threadIdx.x, e);
      if (at + VEC <= n) {
        Piece p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.e[j] = out[e + j];
        *reinterpret_cast<Piece*>(to + at) = p;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at + j < n) to[at + j] = out[e + j];
      }
    }
  }
  if (TOKENS) {
    float most = y[0];  // NaN where one of them is
#pragma unroll
    for (int e = 1; e < kPer; ++e) most = __builtin_elementwise_maximum(most, y[e]);
    const int key = order_key(most);
    const int top = sf_wave_max_int(key);
    // The first entry of that value (entries ascend with e).
    int index = INT32_MAX;
    if (top == INT32_MAX) {
#pragma unroll
      for (int e = kPer - 1; e >= 0; --e)
        if (y[e] != y[e]) index = entry<VEC>(threadIdx.x, e);
    } else {
#pragma unroll
      for (int e = kPer - 1; e >= 0; --e)
        if (y[e] == most) index = entry<VEC>(threadIdx.x, e);
    }
    const int low = -sf_wave_max_int(key == top ? -index : INT32_MIN + 1);
    if (lane == 0)
      a.parts[(static_cast<int64_t>(r) * a.chunks + blockIdx.x) * kWaves + wave] =
          make_int2(top, c0 + low);
  }
}

// The best of a row's partial results: the largest key, then the lowest index.
__global__ __launch_bounds__(kThreads) void logit_token_kernel(const int2* parts, int count,
                                                         int64_t* tokens) {
  __shared__ int2 found[kWaves];
  const int2* p = parts + static_cast<int64_t>(blockIdx.x) * count;
  int best = kNone, index = INT32_MAX;
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int2 x = p[i];
    if (x.x > best || (x.x == best && x.y < index)) {
      best = x.x;
      index = x.y;
    }
  }
  const int top = sf_wave_max_int(best);
  const int low = -sf_wave_max_int(best == top ? -index : INT32_MIN + 1);
  if (threadIdx.x % SF_WAVE == 0) found[threadIdx.x / SF_WAVE] = make_int2(top, low);
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < kWaves; ++w)
    if (found[w].x > found[0].x || (found[w].x == found[0].x && found[w].y < found[0].y))
      found[0] = found[w];
  tokens[blockIdx.x] = found[0].x == kNone ? -1 : found[0].y;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

template <int DTYPE, int VEC>
void launch(const RuleArgs& a, bool penalty, hipStream_t s) {
  const bool out = a.out != nullptr, tokens = a.parts != nullptr;
  const dim3 grid(a.chunks, a.rows);
#define SF_RULES(P, O, T) logit_rules_kernel<DTYPE, VEC, P, O, T><<<grid, kThreads, 0, s>>>(a)
  if (penalty) {
    if (out && tokens) SF_RULES(true, true, true);
    else if (out) SF_RULES(true, true, false);
    else SF_RULES(true, false, true);
  } else {
    if (out && tokens) SF_RULES(false, true, true);
    else if (out) SF_RULES(false, true, false);
    else SF_RULES(false, false, true);
  }
#undef SF_RULES
}

}  // namespace

extern "C" int64_t sf_logit_rules_workspace(int rows, int vocab) {
  if (rows < 1 || vocab < 1) return 0;
  return static_cast<int64_t>(rows) * chunks_of(vocab) * kWaves * sizeof(int2);
}

extern "C" int sf_logit_rules(int dtype, const void* logits, int64_t logits_stride, int rows,
                              int vocab, const int32_t* counts, const int32_t* paths,
                              int path_length, float repetition, float presence, float frequency,
                              const float* bias, int64_t bias_stride, const int32_t* allowed,
                              int64_t allowed_stride, void* out, int64_t out_stride,
                              int64_t* tokens, void* workspace, int64_t workspace_bytes,
                              sf_stream_t stream) {
  if ((dtype != SF_BF16 && dtype != SF_F16 && dtype != SF_F32) || rows < 0 || vocab < 0 ||
      path_length < 0 || !(repetition > 0.f))
    return SF_ERR_INVALID_ARGUMENT;
  if (vocab > (1 << 30) || rows > 65535) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0 || (!out && !tokens)) return SF_OK;
  if (vocab == 0 || !logits) return SF_ERR_INVALID_ARGUMENT;
  if (tokens && (!workspace || workspace_bytes < sf_logit_rules_workspace(rows, vocab)))
    return SF_ERR_INVALID_ARGUMENT;
  if (tokens && reinterpret_cast<uintptr_t>(workspace) % sizeof(int2)) return SF_ERR_MISALIGNED;
  RuleArgs a = {logits, logits_stride, rows, vocab, counts, path_length ? paths : nullptr,
                path_length, repetition,
                repetition >= 0x1p-20f && repetition <= 0x1p20f
                    ? static_cast<float>(1.0 / static_cast<double>(repetition))
                    : 0.f,
                presence, frequency, bias, bias_stride, allowed,
                allowed_stride, out, out_stride,
                tokens ? static_cast<int2*>(workspace) : nullptr, chunks_of(vocab)};
  const bool penalty = (counts || a.paths) &&
                       (repetition != 1.f || presence != 0.f || frequency != 0.f);
  const int size = dtype == SF_F32 ? 4 : 2;
  const int vec = 16 / size;
  bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (rows == 1 || logits_stride % vec == 0);
  if (out)
    wide = wide && reinterpret_cast<uintptr_t>(out) % 16 == 0 && (rows == 1 || out_stride % vec == 0);
  if (counts) wide = wide && reinterpret_cast<uintptr_t>(counts) % 16 == 0;
  if (bias)
    wide = wide && reinterpret_cast<uintptr_t>(bias) % 16 == 0 && bias_stride % 4 == 0;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SF_BF16) {
    wide ? launch<SF_BF16, 8>(a, penalty, s) : launch<SF_BF16, 1>(a, penalty, s);
  } else if (dtype == SF_F16) {
    wide ? launch<SF_F16, 8>(a, penalty, s) : launch<SF_F16, 1>(a, penalty, s);
  } else {
    wide ? launch<SF_F32, 4>(a, penalty, s) : launch<SF_F32, 1>(a, penalty, s);
  }
  SF_LAUNCH_CHECK();
  if (tokens) {
    logit_token_kernel<<<rows, kThreads, 0, s>>>(a.parts, a.chunks * kWaves, tokens);
    SF_LAUNCH_CHECK();
  }
  return SF_OK;
}
