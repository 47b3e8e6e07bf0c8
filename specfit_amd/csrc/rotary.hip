// K11: rotary positions of queries and keys.
//
// For token (b, t) and pair i the angle in turns is position * turns[i], taken
// in fp64 and reduced to half a turn before it is rounded to fp32: at position
// 10^6 an fp32 product would be off by a sixteenth of a radian.  The sines are
// the same for every head, so a workgroup computes those of its tokens once
// into LDS; (a, b) -> (a cos - b sin, b cos + a sin) then runs over its heads
// in 16-byte pieces.  Bound by the bytes of q and k, in and out.
#include <algorithm>

#include "sf_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // of a workgroup

struct RotaryArgs {
  const void* x[2];  // q, k
  int64_t batch[2], tok[2], head[2];
  int heads[2];
  void* out[2];
  const int64_t* positions;
  int64_t position_stride;
  const double* turns;
  float factor;
  int B, T, D, R;
  int tokens;  // of a workgroup
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

// VEC elements per access: those of 16 bytes, or 1.
template <int DTYPE, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryArgs a) {
  using Ty = Type<DTYPE>;
  using Elem = typename Ty::Elem;
  struct __attribute__((aligned(VEC * sizeof(Elem)))) Piece {
    Elem e[VEC];
  };
  extern __shared__ float2 turn[];  // (cos, sin) times the factor, [tokens][R / 2]
  const int half = a.R / 2;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int64_t all = static_cast<int64_t>(a.B) * a.T;
  const int count = static_cast<int>(min(static_cast<int64_t>(a.tokens), all - first));
  for (int n = threadIdx.x; n < count * half; n += kThreads) {
    const int64_t token = first + n / half;
    const int64_t b = token / a.T;
    const double p = static_cast<double>(a.positions[b * a.position_stride + (token - b * a.T)]) *
                     a.turns[n % half];
    float s, c;
    sincospif(static_cast<float>(2.0 * (p - __builtin_rint(p))), &s, &c);
    turn[n] = make_float2(c * a.factor, s * a.factor);
  }
  __syncthreads();

  // A unit of work: two pieces of VEC pairs apart (half layout), one piece of
  // VEC / 2 pairs (interleaved; VEC 1: a pair), or a piece that is copied.  A
  // thread keeps its unit (and the unit's sines in registers) over the heads, and
  // has kAtOnce of them on their way: dividing out token, head and unit for each
  // piece instead, 8002 tokens of 36 fp32 heads of 128 took 84 us; they take
  // 50 (295 MB, 5.9 TB/s).
  constexpr int kStep = INTERLEAVED ? (VEC > 1 ? VEC : 2) : VEC;
  constexpr int kPieces = INTERLEAVED ? kStep / VEC : 2;  // of a unit
  constexpr int kSines = INTERLEAVED ? kStep / 2 : VEC;
  constexpr int kAtOnce = 4;
  const int turned = (INTERLEAVED ? a.R : half) / kStep;
  const int units = turned + (a.D - a.R) / VEC;
  const int width = min(units, kThreads);
  const int rows = kThreads / width;  // heads side by side
  if (static_cast<int>(threadIdx.x) >= rows * width) return;
  const int first_head = blockIdx.y * rows + threadIdx.x / width;
  const int head_step = gridDim.y * rows;
  for (int u = threadIdx.x % width; u < units; u += width) {
    const bool copied = u >= turned;
    // First element of each of the unit's pieces.
    const int d0 = copied ? a.R + (u - turned) * VEC : u * kStep;
    const int d1 = INTERLEAVED ? d0 + VEC : d0 + half;
    const int pieces = copied ? 1 : kPieces;
    for (int i = 0; i < count; ++i) {
      const int64_t token = first + i;
      const int64_t b = token / a.T, t = token - b * a.T;
      float2 f[kSines] = {};
      if (!copied) {
#pragma unroll
        for (int e = 0; e < kSines; ++e)
          f[e] = turn[i * half + (INTERLEAVED ? d0 / 2 : d0) + e];
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Elem* x = static_cast<const Elem*>(a.x[w]) + b * a.batch[w] + t * a.tok[w];
        Elem* y = static_cast<Elem*>(a.out[w]) + (b * a.heads[w] * a.T + t) * a.D;
        const int64_t out_head = static_cast<int64_t>(a.T) * a.D;
        for (int h0 = first_head; h0 < a.heads[w]; h0 += kAtOnce * head_step) {
          Piece p[kAtOnce][2];
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) {
            const int h = h0 + j * head_step;
            if (h < a.heads[w]) {
              p[j][0] = *reinterpret_cast<const Piece*>(x + h * a.head[w] + d0);
              if (pieces > 1) p[j][1] = *reinterpret_cast<const Piece*>(x + h * a.head[w] + d1);
            }
          }
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) {
            const int h = h0 + j * head_step;
            if (h >= a.heads[w]) continue;
            if (!copied) {
#pragma unroll
              for (int e = 0; e < kSines; ++e) {
                // The pair's two elements.
                Elem& u0 = INTERLEAVED && VEC > 1 ? p[j][0].e[(2 * e) % VEC] : p[j][0].e[e % VEC];
                Elem& u1 =
                    INTERLEAVED && VEC > 1 ? p[j][0].e[(2 * e + 1) % VEC] : p[j][1].e[e % VEC];
                const float v0 = Ty::load(u0), v1 = Ty::load(u1);
                u0 = Ty::store(__builtin_fmaf(v0, f[e].x, -(v1 * f[e].y)));
                u1 = Ty::store(__builtin_fmaf(v1, f[e].x, v0 * f[e].y));
              }
            }
            *reinterpret_cast<Piece*>(y + h * out_head + d0) = p[j][0];
            if (pieces > 1) *reinterpret_cast<Piece*>(y + h * out_head + d1) = p[j][1];
          }
        }
      }
    }
  }
}

template <int DTYPE, int VEC>
void launch(const RotaryArgs& a, bool interleaved, dim3 grid, hipStream_t s) {
  const size_t lds = static_cast<size_t>(a.tokens) * (a.R / 2) * sizeof(float2);
  if (interleaved)
    rotary_kernel<DTYPE, VEC, true><<<grid, kThreads, lds, s>>>(a);
  else
    rotary_kernel<DTYPE, VEC, false><<<grid, kThreads, lds, s>>>(a);
}

}  // namespace

extern "C" int sf_rotary(int dtype, const void* q, int64_t q_stride_batch, int64_t q_stride_token,
                         int64_t q_stride_head, int q_heads, const void* k, int64_t k_stride_batch,
                         int64_t k_stride_token, int64_t k_stride_head, int k_heads,
                         const int64_t* positions, int64_t position_stride, const double* turns,
                         float factor, int batch, int tokens, int head_dim, int rotary_dim,
                         int interleaved, void* q_out, void* k_out, sf_stream_t stream) {
  if ((dtype != SF_BF16 && dtype != SF_F16 && dtype != SF_F32) || batch < 0 || tokens < 0 ||
      q_heads < 0 || k_heads < 0)
    return SF_ERR_INVALID_ARGUMENT;
  if (head_dim < 2 || head_dim > 1024 || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2 ||
      q_heads > 4096 || k_heads > 4096)
    return SF_ERR_UNSUPPORTED_SHAPE;
  const int64_t all = static_cast<int64_t>(batch) * tokens;
  if (all == 0 || q_heads + k_heads == 0) return SF_OK;
  // Below 2^32 threads of a launch.
  if (all >= int64_t{kMaxTokens} << 24) return SF_ERR_UNSUPPORTED_SHAPE;
  if (!positions || !turns || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)))
    return SF_ERR_INVALID_ARGUMENT;
  RotaryArgs a = {{q, k}, {q_stride_batch, k_stride_batch}, {q_stride_token, k_stride_token},
                  {q_stride_head, k_stride_head}, {q_heads, k_heads}, {q_out, k_out},
                  positions, position_stride, turns, factor, batch, tokens, head_dim, rotary_dim, 1};
  const int size = dtype == SF_F32 ? 4 : 2;
  const int vec = 16 / size;
  // 16-byte accesses where every row, and both halves of the turned part,
  // begin on 16 bytes.
  bool wide = head_dim % vec == 0 && rotary_dim % (interleaved ? vec : 2 * vec) == 0;
  for (int w = 0; w < 2; ++w)
    if (a.heads[w])
      wide = wide && reinterpret_cast<uintptr_t>(a.x[w]) % 16 == 0 &&
             reinterpret_cast<uintptr_t>(a.out[w]) % 16 == 0 && a.batch[w] % vec == 0 &&
             a.tok[w] % vec == 0 && a.head[w] % vec == 0;
  const int step = wide ? vec : 1;
  const int units = rotary_dim / (interleaved && wide ? vec : 2 * step) +
                    (head_dim - rotary_dim) / step;
  a.tokens = static_cast<int>(std::min<int64_t>(kMaxTokens, std::max<int64_t>(1, all / 2048)));
  // A workgroup of one token takes the heads that stand side by side in it.
  const int rows = kThreads / std::min(units, kThreads);
  const int shares = a.tokens > 1 ? 1 : std::min(16, (std::max(q_heads, k_heads) + rows - 1) / rows);
  const dim3 grid(static_cast<uint32_t>((all + a.tokens - 1) / a.tokens), shares);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool il = interleaved != 0;
  if (dtype == SF_BF16) {
    wide ? launch<SF_BF16, 8>(a, il, grid, s) : launch<SF_BF16, 1>(a, il, grid, s);
  } else if (dtype == SF_F16) {
    wide ? launch<SF_F16, 8>(a, il, grid, s) : launch<SF_F16, 1>(a, il, grid, s);
  } else {
    wide ? launch<SF_F32, 4>(a, il, grid, s) : launch<SF_F32, 1>(a, il, grid, s);
  }
  SF_LAUNCH_CHECK();
  return SF_OK;
}
