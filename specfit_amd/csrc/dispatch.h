// K2's sort, shared with the kernel that rounds a prompt's rows beside it (K16).
#pragma once

#include "sf_common.h"

namespace sf_dispatch_impl {

constexpr int kMaxSpans = 256;

// How `routes` are cut: workgroups of 1024 threads, or one of 256 where one chunk
// of 256 holds all; `span` routes to each.
struct Cut {
  int threads, span;
  unsigned spans;
};

inline Cut cut_of(int routes) {
  if (routes <= 256) return {256, 256, 1u};
  const long long chunks = (static_cast<long long>(routes) + 1023) / 1024;
  const long long per = (chunks + kMaxSpans - 1) / kMaxSpans;  // chunks of a span
  return {1024, static_cast<int>(per * 1024), static_cast<unsigned>((chunks + per - 1) / per)};
}

// Workgroups of kDispatchThreads (1024, or 256 when the routes fit one
// 256-wide chunk: fewer wavefronts to synchronise), `span` routes each (a
// multiple of kDispatchThreads).  The permutation is the unique stable order
// either way.
template <int kDispatchThreads>
__device__ __forceinline__ void dispatch(
    unsigned block, const int64_t* __restrict__ idx, int N, int E, int span, int32_t* __restrict__ counts,
    int32_t* __restrict__ offsets, int32_t* __restrict__ perm_pos,
    int32_t* __restrict__ inv_perm, int32_t* __restrict__ host_meta) {
  constexpr int kDispatchWaves = kDispatchThreads / SF_WAVE;
  __shared__ int s_total[SF_MAX_EXPERTS];
  __shared__ int s_offset[SF_MAX_EXPERTS + 1];
  __shared__ int s_running[SF_MAX_EXPERTS];  // routes of e before the current chunk
  __shared__ int s_wave_count[kDispatchWaves][SF_MAX_EXPERTS];
  __shared__ int s_invalid;
  const int tid = threadIdx.x;
  const int lane = tid & (SF_WAVE - 1);
  const int wave = tid / SF_WAVE;
  const int64_t begin64 = static_cast<int64_t>(block) * span;
  const int begin = static_cast<int>(begin64);  // < N by the grid's size
  const int end = static_cast<int>(begin64 + span < N ? begin64 + span : N);

  for (int e = tid; e < SF_MAX_EXPERTS; e += kDispatchThreads) {
    s_total[e] = 0;
    s_running[e] = 0;
  }
  for (int i = tid; i < kDispatchWaves * SF_MAX_EXPERTS; i += kDispatchThreads)
    (&s_wave_count[0][0])[i] = 0;
  if (tid == 0) s_invalid = 0;
  __syncthreads();

  // Pass 1: histograms (integer atomics are order independent) of the routes
  // before the span and of the others.  Each thread keeps its id of the
  // span's first chunk.
  int64_t first = -1;
#pragma unroll 8
  for (int64_t i = tid; i < N; i += kDispatchThreads) {
    const int64_t e = idx[i];
    if (i == begin64 + tid) first = e;
    if (e >= 0 && e < E)
      atomicAdd(i < begin ? &s_running[e] : &s_total[e], 1);
    else
      atomicAdd(&s_invalid, 1);
  }
  __syncthreads();
  for (int e = tid; e < E; e += kDispatchThreads) s_total[e] += s_running[e];
  __syncthreads();
  if (wave == 0) {
    // Exclusive prefix of s_total over the experts: lane l owns experts
    // 4l .. 4l+3 (SF_MAX_EXPERTS = 256 = 4 x 64), a wavefront inclusive scan
    // of the lane sums gives each lane its starting offset.
    constexpr int kPer = SF_MAX_EXPERTS / SF_WAVE;
    int own[kPer];
    int sum = 0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int e = lane * kPer + q;
      own[q] = e < E ? s_total[e] : 0;
      sum += own[q];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < SF_WAVE; d <<= 1) {
      const int up = __shfl_up(incl, d, SF_WAVE);
      if (lane >= d) incl += up;
    }
    int run = incl - sum;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int e = lane * kPer + q;
      if (e < E) s_offset[e] = run;
      run += own[q];
    }
    if (lane == SF_WAVE - 1) s_offset[E] = incl;
  }
  __syncthreads();
  if (block == 0) {
    for (int e = tid; e < E; e += kDispatchThreads) {
      counts[e] = s_total[e];
      offsets[e] = s_offset[e];
    }
    if (tid == 0) {
      counts[E] = s_invalid;
      offsets[E] = s_offset[E];
    }
  }
  if (host_meta && block == 0) {  // the same [counts; offsets] into pinned host memory
    for (int e = tid; e < E; e += kDispatchThreads) {
      host_meta[e] = s_total[e];
      host_meta[E + 1 + e] = s_offset[e];
    }
    if (tid == 0) {
      host_meta[E] = s_invalid;
      host_meta[2 * E + 1] = s_offset[E];
    }
  }

  // Pass 2: stable scatter of the span, chunk by chunk.
  const int id_bits = E > 1 ? 32 - __builtin_clz(E - 1) : 0;
  for (int base = begin; base < end; base += kDispatchThreads) {
    const int64_t i = static_cast<int64_t>(base) + tid;
    int e = -1;
    if (i < end) {
      const int64_t v = base == begin ? first : idx[i];
      e = (v >= 0 && v < E) ? static_cast<int>(v) : -1;
    }
    // Lanes with this lane's id: the valid lanes whose ballot agrees with it
    // in every id bit.
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < id_bits; ++b) {
      const bool bit = (e >> b) & 1;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const int rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(same >> 32),
                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same), 0));
    const int group = __popcll(same);
    const bool valid = e >= 0;
    if (valid && rank == 0) s_wave_count[wave][e] = group;
    __syncthreads();
    // Exclusive prefix over the wavefronts that hold routes in this chunk
    // (the others' counts are zero), per expert, continuing the running
    // count of earlier chunks.
    const int busy_waves = min(kDispatchWaves, (min(end - base, kDispatchThreads) + SF_WAVE - 1) / SF_WAVE);
    for (int ex = tid; ex < E; ex += kDispatchThreads) {
      int run = s_running[ex];
      for (int w = 0; w < busy_waves; ++w) {
        int c = s_wave_count[w][ex];
        s_wave_count[w][ex] = run;
        run += c;
      }
      s_running[ex] = run;
    }
    __syncthreads();
    if (i < end) {
      if (valid) {
        const int pos = s_offset[e] + s_wave_count[wave][e] + rank;
        perm_pos[pos] = static_cast<int32_t>(i);
        inv_perm[i] = pos;
      } else {
        inv_perm[i] = -1;
      }
    }
    if (end - base <= kDispatchThreads) break;  // last chunk: nothing to reset
    __syncthreads();
    // Reset the per-wavefront table for the next chunk.
    for (int j = tid; j < kDispatchWaves * SF_MAX_EXPERTS; j += kDispatchThreads)
      (&s_wave_count[0][0])[j] = 0;
    __syncthreads();
  }
}

}  // namespace sf_dispatch_impl
