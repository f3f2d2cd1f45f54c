// Shared device code of the float32 kernels whose workgroups split a walk (attn_f32.hip says
// why): MFMA operands straight from global memory through buffer resources, and the LDS
// layout of a wave's partial results.
#pragma once

#include "attn_common.h"

namespace mi {

constexpr int kWaves = 4;

typedef __amdgpu_buffer_rsrc_t Buf;

// Rows [0, S) of one head of a [B, S, heads, D] float tensor.
struct Head {
  Buf r;
  unsigned rb;     // bytes from one row to the next
};
__device__ __forceinline__ Head head_of(const float* base, int b, int S, long long rs, int h, int D) {
  Head x;
  float* p = const_cast<float*>(base) + (long long)b * S * rs + (long long)h * D;
  x.r = __builtin_amdgcn_make_buffer_rsrc(p, 0, (int)(((long long)(S - 1) * rs + D) * 4), 0x00020000);
  x.rb = (unsigned)(rs * 4);
  return x;
}

// Row row0 + l32, chunk 8j + 4g: c[j][e] is head dim 8j + 4g + e.
template <int D>
__device__ __forceinline__ void load_rows(f32x4 (&c)[D / 8], const Head& x, int row0, int l32, int g) {
  const unsigned off = (unsigned)(row0 + l32) * x.rb + 16u * g;
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
    c[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x.r, off + 32u * j, 0, 0));
}
// Rows row0 + crow(s, g) of columns 32 dt + l32.
template <int D>
__device__ __forceinline__ void load_cols(float (&t)[16][D / 32], const Head& x, int row0, int l32, int g) {
  const unsigned off = (unsigned)(row0 + 4 * g) * x.rb + 4u * l32;
#pragma unroll
  for (int s = 0; s < 16; ++s)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
      t[s][dt] = __builtin_bit_cast(
          float, __builtin_amdgcn_raw_buffer_load_b32(x.r, off + crow_off(s) * x.rb + 128u * dt, 0, 0));
}

// acc += rows . cols over the head dims (32 x 32).
template <int D>
__device__ __forceinline__ f32x16 dot_rows(const f32x4 (&a)[D / 8], const f32x4 (&b)[D / 8], f32x16 acc) {
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = Mfma32<float>::mma(a[j][e], b[j][e], acc);
  return acc;
}

__device__ __forceinline__ float halves(float x) { return x + __shfl_xor(x, 32); }

// A wave's 32 x D partial (acc[dt] register r: column 32 dt + crow(r, g) of row
// l32) into LDS rows of D + 4 floats.
template <int D>
__device__ __forceinline__ void put_partial(float* dst, const f32x16 (&acc)[D / 32], int l32, int g) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4*>(dst + l32 * (D + 4) + dt * 32 + 8 * j + 4 * g) =
          f32x4{acc[dt][4 * j], acc[dt][4 * j + 1], acc[dt][4 * j + 2], acc[dt][4 * j + 3]};
}

}  // namespace mi
