// K11: repetition penalties, a bias and an allowed set on rows of logits, and
// each row's greedy token.
//
// A thread keeps the counts (and a shared bias) of its eight vocabulary entries
// in registers for several rows, so a row costs its logits and one word of its
// allowed set; the tokens of a row's own path are found by the wavefront that
// holds their entries.  Bound by the bytes of the logits.  The greedy token is a
// maximum of (value, lowest index) over partial results of the wavefronts, so
// no order of arrival changes it.
#include <algorithm>

#include "sf_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / SF_WAVE;
constexpr int kPer = 8;                     // entries of a thread
constexpr int kChunk = kThreads * kPer;     // of a workgroup
constexpr int kMaxRows = 8;                 // of a workgroup
constexpr int kNone = INT32_MIN;            // key of a value that is never chosen

struct RuleArgs {
  const void* logits;
  int64_t stride;
  int rows, vocab;
  const int32_t* counts;
  const int32_t* paths;
  int path_length;
  float repetition, presence, frequency;
  const float* bias;
  int64_t bias_stride;
  const int32_t* allowed;
  int64_t allowed_stride;
  void* out;
  int64_t out_stride;
  int2* parts;  // [rows][chunks * kWaves] (key, index), or nullptr
  int chunks, group;
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

template <int DTYPE, int VEC, bool PENALTY, bool OUT, bool TOKENS>
__global__ __launch_bounds__(kThreads) void rules_kernel(const RuleArgs a) {
  using Ty = Type<DTYPE>;
  using Elem = typename Ty::Elem;
  const int lane = threadIdx.x & (SF_WAVE - 1);
  const int wave = threadIdx.x / SF_WAVE;
  const int c0 = blockIdx.x * kChunk;
  const int n = min(kChunk, a.vocab - c0);  // entries of the chunk
  const int r0 = blockIdx.y * a.group;
  const int r1 = min(r0 + a.group, a.rows);

  int32_t seen[kPer] = {};
  if (PENALTY && a.counts) load_entries<VEC>(a.counts + c0, n, seen);
  float bias[kPer] = {};
  if (a.bias && a.bias_stride == 0) load_entries<VEC>(a.bias + c0, n, bias);

  for (int r = r0; r < r1; ++r) {
    Elem raw[kPer];
    load_entries<VEC>(static_cast<const Elem*>(a.logits) + r * a.stride + c0, n, raw);
    if (a.bias && a.bias_stride) load_entries<VEC>(a.bias + r * a.bias_stride + c0, n, bias);
    uint32_t ok = 0;
#pragma unroll
    for (int e = 0; e < kPer; e += VEC) {
      const int at = entry<VEC>(threadIdx.x, e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) ok |= (at + j < n ? 1u : 0u) << (e + j);
    }
    if (a.allowed) {
      const int32_t* words = a.allowed + r * a.allowed_stride;
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < kPer; e += VEC) {
        // VEC neighbours share a word: chunks and VEC divide or are multiples of 32.
        const int v = c0 + min(entry<VEC>(threadIdx.x, e), n - 1);
        bits |= ((static_cast<uint32_t>(words[v / 32]) >> (v % 32)) & ((1u << VEC) - 1u)) << e;
      }
      ok &= bits;
    }
    int32_t count[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) count[e] = seen[e];
    if (PENALTY && a.paths) {
      const int32_t* path = a.paths + static_cast<int64_t>(r) * a.path_length;
      for (int p0 = 0; p0 < a.path_length; p0 += SF_WAVE) {
        const int token = p0 + lane < a.path_length ? path[p0 + lane] : -1;
        uint64_t here = __ballot(token >= c0 && token < c0 + n);
        while (here) {  // uniform
          const int at =
              __builtin_amdgcn_readlane(token, static_cast<int>(__builtin_ctzll(here))) - c0;
          here &= here - 1;
#pragma unroll
          for (int e = 0; e < kPer; ++e) count[e] += entry<VEC>(threadIdx.x, e) == at;
        }
      }
    }
    int best = kNone, index = 0;
    Elem out[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      float y = Ty::load(raw[e]);
      if (PENALTY) {
        if (__any(count[e] > 0)) {
          const float x = y < 0.f ? y * a.repetition : y / a.repetition;
          const float less = a.frequency * static_cast<float>(count[e]);
          const float z = x - (less + a.presence);
          if (count[e] > 0) y = z;
        }
      }
      if (a.bias) y += bias[e];
      if (!((ok >> e) & 1u)) y = -INFINITY;
      if (OUT) out[e] = Ty::store(y);
      if (TOKENS) {
        const int key = order_key(y);
        if (key > best) {  // entries ascend with e
          best = key;
          index = entry<VEC>(threadIdx.x, e);
        }
      }
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
      const int top = sf_wave_max_int(best);
      const int low = -sf_wave_max_int(best == top ? -index : INT32_MIN + 1);
      if (lane == 0)
        a.parts[(static_cast<int64_t>(r) * a.chunks + blockIdx.x) * kWaves + wave] =
            make_int2(top, c0 + low);
    }
  }
}

// The best of a row's partial results: the largest key, then the lowest index.
__global__ __launch_bounds__(kThreads) void token_kernel(const int2* parts, int count,
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
void launch(const RuleArgs& a, bool penalty, dim3 grid, hipStream_t s) {
  const bool out = a.out != nullptr, tokens = a.parts != nullptr;
#define SF_RULES(P, O, T) rules_kernel<DTYPE, VEC, P, O, T><<<grid, kThreads, 0, s>>>(a)
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
  if (vocab > (1 << 30) || rows > (1 << 18)) return SF_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0 || (!out && !tokens)) return SF_OK;
  if (vocab == 0 || !logits) return SF_ERR_INVALID_ARGUMENT;
  if (tokens && (!workspace || workspace_bytes < sf_logit_rules_workspace(rows, vocab)))
    return SF_ERR_INVALID_ARGUMENT;
  if (tokens && reinterpret_cast<uintptr_t>(workspace) % sizeof(int2)) return SF_ERR_MISALIGNED;
  RuleArgs a = {logits, logits_stride, rows, vocab, counts, path_length ? paths : nullptr,
                path_length, repetition, presence, frequency, bias, bias_stride, allowed,
                allowed_stride, out, out_stride,
                tokens ? static_cast<int2*>(workspace) : nullptr, chunks_of(vocab), 1};
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
  // Rows of a workgroup: enough workgroups for the 256 CUs first.
  const int64_t work = static_cast<int64_t>(rows) * a.chunks;
  a.group = static_cast<int>(std::min<int64_t>(kMaxRows, std::max<int64_t>(1, work / 1024)));
  const dim3 grid(a.chunks, (rows + a.group - 1) / a.group);
  if (grid.y > 65535) return SF_ERR_UNSUPPORTED_SHAPE;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == SF_BF16) {
    wide ? launch<SF_BF16, 8>(a, penalty, grid, s) : launch<SF_BF16, 1>(a, penalty, grid, s);
  } else if (dtype == SF_F16) {
    wide ? launch<SF_F16, 8>(a, penalty, grid, s) : launch<SF_F16, 1>(a, penalty, grid, s);
  } else {
    wide ? launch<SF_F32, 4>(a, penalty, grid, s) : launch<SF_F32, 1>(a, penalty, grid, s);
  }
  SF_LAUNCH_CHECK();
  if (tokens) {
    token_kernel<<<rows, kThreads, 0, s>>>(a.parts, a.chunks * kWaves, tokens);
    SF_LAUNCH_CHECK();
  }
  return SF_OK;
}
