// K16: grouped SwiGLU experts with weights in microscaled 4 bits, over the rows
// that K2 dispatched.  For expert e's rows r (token t = perm_pos[r] / top_k):
//   g = x[t] . gate^T, u = x[t] . up^T        x in e4m3
//   a = e4m3(silu(g) u)                       blocks of 32 of the inner size
//   rows[r] = bf16((a . down^T) * route_weight)
// with fp32 sums and one rounding between them: the activation is what the
// second product reads, so it is rounded once, from fp32, to that product's
// type.
#include "mx_product.h"

namespace {

using namespace sf_mx;

constexpr int kThreads = 256, kWaves = kThreads / SF_WAVE;

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
  int top_k, hidden, inner;
  const int32_t* slot_of_expert;
  const uint8_t* slots;
  int64_t slot_stride;
  Record record;
  uint8_t* act;         // e4m3 rows [tokens * top_k, inner]
  uint8_t* act_scales;
  uint16_t* rows;       // bf16 [tokens * top_k, hidden]
};

// The weights of the expert of this workgroup; null where it has none to do.
__device__ __forceinline__ const uint8_t* expert_of(const Experts& p, int e, int& begin, int& end) {
  begin = p.offsets[e];
  end = p.offsets[e + 1];
  const int slot = p.slot_of_expert ? p.slot_of_expert[e] : e;
  return begin < end && slot >= 0 ? p.slots + slot * p.slot_stride : nullptr;
}

// A workgroup: 32 columns of gate and up of one expert, the hidden size cut
// over its wavefronts, so that the 32 activations are one block of the next
// product's rows.
template <int MT, int XDT>
__global__ __launch_bounds__(kThreads) void gate_up_direct_kernel(Experts p) {
  constexpr int kAhead = MT == 1 ? 2 : 1;
  __shared__ f32x4 part[kWaves * 4 * MT * SF_WAVE];
  int row_begin, row_end;
  const uint8_t* weights = expert_of(p, blockIdx.y, row_begin, row_end);
  if (!weights) return;
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4, c = lane & 15;
  const int block = blockIdx.x;
  const int64_t act_width = static_cast<int64_t>(tiles(p.inner)) * kTile;
  const int64_t act_scale_width = static_cast<int64_t>(quads(p.inner)) * 16;
  const int scale_at = block / 16 * 16 + block % 4 * 4 + block / 4 % 4;
  if (block * kBlock >= p.inner) {  // behind the activations' end, within their last tile: zeros
    for (int i = threadIdx.x; i < (row_end - row_begin) * 8; i += kThreads) {
      const int64_t row = row_begin + i / 8;
      *reinterpret_cast<uint32_t*>(p.act + row * act_width + block * kBlock + i % 8 * 4) = 0;
      if (i % 8 == 0) p.act_scales[row * act_scale_width + scale_at] = 0;
    }
    return;
  }
  WeightSource w[4];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    w[n].set(weights, weights + p.record.gate_scales, 2 * block + n, p.hidden, lane);
    w[2 + n].set(weights + p.record.up_codes, weights + p.record.up_scales, 2 * block + n, p.hidden, lane);
  }
  int begin, end;
  part_of(tiles(p.hidden), wave, kWaves, begin, end);
  for (int row0 = row_begin; row0 < row_end; row0 += 16 * MT) {
    RowSource<XDT> x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int token = p.perm_pos[min(row0 + 16 * m + c, row_end - 1)] / p.top_k;
      x[m].set(p.x, p.x_scales, token, p.x_stride, p.hidden, g);
    }
    f32x4 acc[4][MT] = {};
    accumulate<MT, 4, XDT, kAhead>(acc, w, x, begin, end, p.hidden, g);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) part[((wave * MT + m) * 4 + n) * SF_WAVE + lane] = acc[n][m];
    __syncthreads();
    if (wave < MT) {  // a wavefront to 16 rows: a lane 4 + 4 of its row's 32
      const int row = row0 + 16 * wave + c;
      f32x4 v[4] = {};
#pragma unroll
      for (int k = 0; k < kWaves; ++k)
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] += part[((k * MT + wave) * 4 + n) * SF_WAVE + lane];
      float a[8];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float gate = v[i / 4][i % 4], up = v[2 + i / 4][i % 4];
        a[i] = gate / (1.0f + __expf(-gate)) * up;
        top = max(top, magnitude(a[i]));
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      const uint32_t byte = scale_byte<kE4m3>(top);
      uint32_t lo = 0, hi = 0;
      if (byte != 255) {
        const float s = inverse_scale(byte);
        lo = e4m3x4(a[0] * s, a[1] * s, a[2] * s, a[3] * s);
        hi = e4m3x4(a[4] * s, a[5] * s, a[6] * s, a[7] * s);
      }
      if (row < row_end) {
        uint8_t* o = p.act + row * act_width + block * kBlock + 4 * g;
        *reinterpret_cast<uint32_t*>(o) = lo;
        *reinterpret_cast<uint32_t*>(o + 16) = hi;
        if (g == 0) p.act_scales[row * act_scale_width + scale_at] = static_cast<uint8_t>(byte);
      }
    }
    __syncthreads();
  }
}

// A wavefront: NT row tiles of down over the whole inner size.
template <int MT, int NT>
__global__ __launch_bounds__(kThreads) void down_direct_kernel(Experts p) {
  constexpr int kAhead = MT * NT <= 2 ? 4 : 2;
  int row_begin, row_end;
  const uint8_t* weights = expert_of(p, blockIdx.y, row_begin, row_end);
  if (!weights) return;
  const int lane = threadIdx.x & (SF_WAVE - 1), wave = threadIdx.x / SF_WAVE;
  const int g = lane >> 4, c = lane & 15;
  const int group = blockIdx.x * kWaves + wave, last = row_tiles(p.hidden) - 1;
  if (group * NT > last) return;
  WeightSource w[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    w[n].set(weights + p.record.down_codes, weights + p.record.down_scales, min(group * NT + n, last), p.inner,
             lane);
  for (int row0 = row_begin; row0 < row_end; row0 += 16 * MT) {
    RowSource<kRows> x[MT];
    float route[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = min(row0 + 16 * m + c, row_end - 1);
      x[m].set(p.act, p.act_scales, row, 0, p.inner, g);
      route[m] = p.route_weights ? sf_bf16_to_f32(p.route_weights[p.perm_pos[row]]) : 1.0f;
    }
    f32x4 acc[NT][MT] = {};
    accumulate<MT, NT, kRows, kAhead>(acc, w, x, 0, tiles(p.inner), p.inner, g);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = row0 + 16 * m + c;
      if (row >= row_end) continue;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int h = (group * NT + n) * 16 + 4 * g;
        const f32x4 v = acc[n][m] * route[m];
        uint16_t* o = p.rows + static_cast<int64_t>(row) * p.hidden + h;
        if (h + 4 <= p.hidden && p.hidden % 4 == 0) {
          *reinterpret_cast<u32x2*>(o) = u32x2{narrow2<kBf16>(v[0], v[1]), narrow2<kBf16>(v[2], v[3])};
        } else {
          for (int i = 0; i < 4; ++i)
            if (h + i < p.hidden) o[i] = sf_f32_to_bf16(v[i]);
        }
      }
    }
  }
}

template <int MT, int XDT>
void launch_direct(const Experts& p, int num_experts, hipStream_t s) {
  gate_up_direct_kernel<MT, XDT><<<dim3(tiles(p.inner) * 4, num_experts), dim3(kThreads), 0, s>>>(p);
  constexpr int NT = 2;
  const int groups = (row_tiles(p.hidden) - 1) / NT + 1;
  down_direct_kernel<MT, NT><<<dim3((groups - 1) / kWaves + 1, num_experts), dim3(kThreads), 0, s>>>(p);
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
  if (tokens < 0 || top_k < 1 || num_experts < 1 || x_stride < 0 || (x_dtype != kBf16 && x_dtype != kRows))
    return SF_ERR_INVALID_ARGUMENT;
  const int64_t bytes = sf_mx_expert_bytes(hidden_size, intermediate_size);
  if (bytes < 0) return SF_ERR_INVALID_ARGUMENT;
  if (num_experts > SF_MAX_EXPERTS || top_k > SF_MAX_TOPK) return SF_ERR_TOO_MANY_EXPERTS;
  if (static_cast<int64_t>(tokens) * top_k > 1 << 28) return SF_ERR_UNSUPPORTED_SHAPE;
  if (tokens == 0) return SF_OK;
  if (!x || (x_dtype == kRows && !x_scales) || !perm_pos || !offsets || !slots || !act || !act_scales ||
      !out_rows || slot_stride < bytes)
    return SF_ERR_INVALID_ARGUMENT;
  if (!aligned(x, 16) || !aligned(slots, 16) || slot_stride % 16 || !aligned(act, 16) || !aligned(act_scales, 4) ||
      !aligned(out_rows, 8) || (x_dtype == kRows && !aligned(x_scales, 4)))
    return SF_ERR_MISALIGNED;
  if (x_dtype != kRows) {
    if (x_stride % 8 || hidden_size % 8) return SF_ERR_MISALIGNED;
    if (tokens > 16) return SF_ERR_UNSUPPORTED_SHAPE;
  }
  const Experts p = {x, static_cast<const uint8_t*>(x_scales), x_stride, perm_pos, offsets,
                     static_cast<const uint16_t*>(route_weights), top_k, hidden_size, intermediate_size,
                     slot_of_expert, static_cast<const uint8_t*>(slots), slot_stride,
                     record_of(hidden_size, intermediate_size), static_cast<uint8_t*>(act),
                     static_cast<uint8_t*>(act_scales), static_cast<uint16_t*>(out_rows)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (x_dtype == kBf16)
    launch_direct<1, kBf16>(p, num_experts, s);
  else if (static_cast<int64_t>(tokens) * top_k <= 8 * num_experts)
    launch_direct<1, kRows>(p, num_experts, s);
  else
    launch_direct<4, kRows>(p, num_experts, s);
  SF_LAUNCH_CHECK();
  return SF_OK;
}
