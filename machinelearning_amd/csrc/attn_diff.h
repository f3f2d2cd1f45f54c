// Differential attention: parameters and the pieces that its kernels share.
//
// Each head's query and key rows of E dims are two halves of E / 2, two softmax
// maps over the same values (map m in {1, 2}, scale c):
//   P_m = softmax(c q_m k_m^T + mask),   out = (P_1 - lam_h P_2) v,
// with one learned weight lam_h per query head. Its gradients, for dout:
//   G = dout v^T,  delta_m = rowsum(P_m G) = dout . (P_m v),
//   dS_1 = P_1 (G - delta_1),  dS_2 = -lam P_2 (G - delta_2),
//   dq_m = c dS_m k_m,  dk_m = c dS_m^T q_m,  dv = (P_1 - lam P_2)^T dout,
//   dlam_h = -sum over h's rows of delta_2.
// G and dv need one product each for both maps; only the forward's P_m v are two,
// since neither map's sum is known before its last key.
#pragma once

#include "attn_common.h"

namespace mi {

struct DiffParams {
  int B, S, H, Hkv, group;
  int causal;
  float scale, scale_log2;
  float resc_th;          // lazy-rescale threshold in raw score units: 8 / scale_log2
  int nblk;               // row blocks per (batch, head) of the launched kernel
  long long q_rs, kv_rs;  // row strides of q / out and of k / v, in elements
  const void* lam;        // [H], of lam_dtype (an mi_dtype)
  int lam_dtype;
  void* dlam;             // [H], of lam_dtype
  FastDiv div_h, div_hkv, div_group, div_wi;
  int wi_blocks_fastest;
  // 16-bit dK/dV dealt evenly (diff16_dkdv_kernel): steps of the whole line, of one (batch,
  // kv head) and of one workgroup; 0: a workgroup per key block.
  int line_n, line_head, line_per;
};

// A plane of [B, H, S] floats: the forward's LSE of each map, the backward's row values.
__host__ __device__ inline long long diff_plane(const DiffParams& p) { return (long long)p.B * p.H * p.S; }

__device__ __forceinline__ float load_as_float(const void* p, int dtype, long long i) {
  switch (dtype) {
    case 0: return static_cast<const float*>(p)[i];
    case 1: return (float)static_cast<const _Float16*>(p)[i];
    default: return (float)static_cast<const __bf16*>(p)[i];
  }
}
__device__ __forceinline__ void store_from_float(void* p, int dtype, long long i, float x) {
  switch (dtype) {
    case 0: static_cast<float*>(p)[i] = x; break;
    case 1: static_cast<_Float16*>(p)[i] = (_Float16)x; break;
    default: static_cast<__bf16*>(p)[i] = (__bf16)x;
  }
}

// dlam_h = -sum of delta_2 over h's rows, from its sums over p.nblk row blocks of each
// (b, h): by the last workgroups of a launch of 256 threads, a head each. `lds`: four floats.
__device__ __forceinline__ void reduce_dlam(const float* __restrict__ sums, float* lds, const DiffParams& p) {
  const int tid = threadIdx.x;
  for (int h = (int)(gridDim.x - 1 - blockIdx.x); h < p.H; h += (int)gridDim.x) {
    float x = 0.f;
    for (int i = tid; i < p.B * p.nblk; i += 256) x += sums[((long long)(i / p.nblk) * p.H + h) * p.nblk + i % p.nblk];
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s);
    if ((tid & 63) == 0) lds[tid >> 6] = x;
    __syncthreads();
    if (tid == 0) store_from_float(p.dlam, p.lam_dtype, h, -((lds[0] + lds[1]) + (lds[2] + lds[3])));
    __syncthreads();
  }
}

}  // namespace mi
