// Layout of the block cache: complete blocks of 64 tokens in 8 bits with one
// power-of-two scale per (head, block, K or V), the tokens after them in bf16
// in a ring of blocks of the same order.
//
// Inside a block the values stand in the order in which the matrix
// instructions of the attention take them, so a wavefront's load is 64
// consecutive 16-byte pieces and nothing is transposed or staged on the way.
// With KS = D / 16 and lane = 32 h + r (h = 0, 1; r = 0..31), a 16-byte piece
// of bf16 holds i = 0..7:
//   K  piece (kh KS + s) 64 + lane:  token 32 kh + r,
//                                    d = 32 (s / 2) + 16 h + 8 (s % 2) + i
//   V  piece (4 db + ks) 64 + lane:  d = 32 db + r,
//                                    token 16 ks + 8 (i / 4) + 4 h + i % 4
// (kh = 0, 1; s < KS; db < D / 32; ks = 0..3).  The V order of tokens is the
// one in which v_mfma_f32_32x32x16 leaves the scores of a query row in a lane.
// In 8 bits the pieces 128 g + lane and 128 g + 64 + lane of bf16 share the
// piece 64 g + lane: bytes 0..7 and 8..15.
#pragma once

#include "sf_common.h"

constexpr int kBlockTokens = SF_KV_BLOCK;
// Flags of a block: what its codes or rows hold that is not finite.
constexpr int kFlagValue = 1;
constexpr int kFlagKey = 2;

typedef unsigned int sf_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 sf_bf16x2 __attribute__((ext_vector_type(2)));

// 16-byte load, explicitly from global memory (a flat load would also hold up
// the waits for shared memory).
__device__ __forceinline__ sf_u32x4 sf_ld16(const void* p) {
  return *(const __attribute__((address_space(1))) sf_u32x4*)(p);
}

// The same at a uniform address plus a lane's offset in bytes.
__device__ __forceinline__ sf_u32x4 sf_ld16(const char* p, uint32_t offset) {
  return *(const __attribute__((address_space(1))) sf_u32x4*)(p + offset);
}

__device__ __forceinline__ uint32_t sf_pack_bf16(float lo, float hi) {
  const sf_bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}

// Four 8-bit codes as two words of bf16, without their scale (exact).
template <int HELD>
__device__ __forceinline__ void sf_codes_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (HELD == SF_KV_E4M3) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
    lo = sf_pack_bf16(f[0], f[1]);
    hi = sf_pack_bf16(f[2], f[3]);
  }
}

// A 16-byte piece of codes as the two pieces of bf16 that share it.
template <int HELD>
__device__ __forceinline__ void sf_codes_frags(sf_u32x4 raw, sf_u32x4& a, sf_u32x4& b) {
  // Opaque, or the compiler takes the bytes apart where the piece was loaded
  // and keeps them, in four times the registers, until they are used.
  asm volatile("" : "+v"(raw));
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) sf_codes_bf16<HELD>(raw[i], w[2 * i], w[2 * i + 1]);
  a = sf_u32x4{w[0], w[1], w[2], w[3]};
  b = sf_u32x4{w[4], w[5], w[6], w[7]};
}

// bf16 of the int8 code -128, which stands for a value that is not finite.
constexpr uint32_t kNanCodeBf16 = 0xC300u;
