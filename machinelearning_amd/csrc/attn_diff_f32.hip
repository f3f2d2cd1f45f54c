// Differential attention (attn_diff.h's formulas) in float32: forward, dQ (with the delta
// pass) and dK/dV.
//
// As attn_f32.hip's kernels: a workgroup owns 32 rows and its four waves take every fourth
// 32-row tile of the walk, operands straight from global memory (L2), partial results summed
// through LDS in wave order. A float32 MFMA moves 4 KFLOP in 64 cycles, so a wave is bound by
// its chain of them and the split keeps the chain short; a tile's chain is E / 2 MFMAs for
// the two maps' scores, E for the forward's two value products.
// B4 H4 S256 E64, causal, us, 128-row workgroups of four whole walks (tiles through LDS) ->
// these: forward 38.5 -> 12.8, delta and dQ 45.7 -> 19.2, dK/dV and dlam 60.4 -> 19.1.
#include <type_traits>

#include "attn_diff.h"
#include "attn_f32.h"

namespace mi {

namespace {

// Scores of map m (0, 1) of 32 x 32 pairs: the head dims of its half.
template <int E, int MAP>
__device__ __forceinline__ f32x16 map_scores(const f32x4 (&a)[E / 8], const f32x4 (&b)[E / 8]) {
  f32x16 acc = zero16();
#pragma unroll
  for (int j = MAP * E / 16; j < (MAP + 1) * E / 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = Mfma32<float>::mma(a[j][e], b[j][e], acc);
  return acc;
}

// Each half's share of dQ / dK: columns of the first half take s1, of the second s2. E = 32:
// both lie in the one 32-column tile, with an accumulator each (acc[map]).
template <int E>
constexpr int half_accs() { return E == 32 ? 2 : E / 32; }
template <int E>
__device__ __forceinline__ void add_halves(f32x16 (&acc)[half_accs<E>()], const float (&cols)[16][E / 32],
                                           const f32x16& s1, const f32x16& s2) {
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int x = 0; x < half_accs<E>(); ++x)
      acc[x] = Mfma32<float>::mma(cols[r][E == 32 ? 0 : x], x < half_accs<E>() / 2 ? s1[r] : s2[r], acc[x]);
}
// The E columns of the two halves, each with its factor.
template <int E>
__device__ __forceinline__ void join_halves(f32x16 (&out)[E / 32], const f32x16 (&acc)[half_accs<E>()], float f1,
                                            float f2) {
#pragma unroll
  for (int dt = 0; dt < E / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool second = E == 32 ? r >= 8 : dt >= E / 64;
      out[dt][r] = acc[E == 32 ? (int)second : dt][r] * (second ? f2 : f1);
    }
}

// One plane's values of rows q0 + crow(r, g) of a head; rows past S read as 0.
__device__ __forceinline__ void load_rowvals(f32x4 (&v)[4], const float* plane_head, int S, int q0, int g) {
  const Buf r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(plane_head), 0, S * 4, 0x00020000);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (unsigned)(q0 + 8 * j + 4 * g) * 4u, 0, 0));
}

// The workgroup's four partials of 32 rows, summed in wave order: eight threads per row.
template <int E>
__device__ __forceinline__ void store_sum(float (&part)[kWaves][32 * (E + 4)], const f32x16 (&acc)[E / 32], float* dst,
                                          long long rs, int nvalid, int wave, int l32, int g) {
  put_partial<E>(part[wave], acc, l32, g);
  __syncthreads();
  const int row = threadIdx.x >> 3;
  if (row < nvalid) {
#pragma unroll
    for (int i = 0; i < E / 32; ++i) {
      const int d = 4 * ((threadIdx.x & 7) + 8 * i);
      f32x4 a = *reinterpret_cast<const f32x4*>(&part[0][row * (E + 4) + d]);
#pragma unroll
      for (int w = 1; w < kWaves; ++w) a += *reinterpret_cast<const f32x4*>(&part[w][row * (E + 4) + d]);
      *reinterpret_cast<f32x4*>(dst + (long long)row * rs + d) = a;
    }
  }
}

}  // namespace

template <int E>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 2 : 1, 8)))
diff_f32_fwd_kernel(const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
                    float* __restrict__ O, float* __restrict__ O2, float* __restrict__ LSE, DiffParams p) {
  constexpr int DT = E / 32;
  __shared__ __attribute__((aligned(16))) float part[kWaves][32 * (E + 4)];
  __shared__ float ml[2][2][kWaves][32];           // map; m, l
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const WorkItem wi = work_item(p.nblk, p.B * p.H, p.div_wi, p.causal, p.wi_blocks_fastest);
  const int b = (int)fdiv((unsigned)wi.bh, p.div_h), h = wi.bh - b * p.H;
  const int hkv = (int)fdiv((unsigned)h, p.div_group);
  const int q0 = wi.blk * 32, qi = q0 + l32;
  const Head hK = head_of(K, b, p.S, p.kv_rs, hkv, E), hV = head_of(V, b, p.S, p.kv_rs, hkv, E);
  f32x4 qf[E / 8], kr[E / 8];
  float vc[16][DT];
  load_rows<E>(qf, head_of(Q, b, p.S, p.q_rs, h, E), q0, l32, g);
  const int t_end = ((p.causal ? min(p.S, q0 + 32) : p.S) + 31) / 32;
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1, all_hi = p.causal ? q0 : p.S - 1;

  f32x16 o[2][DT];
  float m[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = zero16();
  const float c = p.scale_log2;
  int t = wave;
  if (t < t_end) {
    load_rows<E>(kr, hK, t * 32, l32, g);
    load_cols<E>(vc, hV, t * 32, l32, g);
  }
  for (; t < t_end; t += kWaves) {
    const int k0 = t * 32;
    f32x16 s[2] = {map_scores<E, 0>(kr, qf), map_scores<E, 1>(kr, qf)};
    if (t + kWaves < t_end) load_rows<E>(kr, hK, (t + kWaves) * 32, l32, g);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (k0 + 31 > all_hi) mask_above(s[x], key_hi - (k0 + 4 * g), -INFINITY);
      float mx = s[x][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[x][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      if (wave_any(mx > m[x] + p.resc_th)) {
        const float m_new = fmaxf(m[x], mx);
        const float alpha = fast_exp2((m[x] - m_new) * c);
        l[x] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[x][dt][r] *= alpha;
        m[x] = m_new;
      }
      const float mc = m[x] * c;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[x][r] = fast_exp2(fmaf(s[x][r], c, -mc));
        l[x] += s[x][r];
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        o[0][dt] = Mfma32<float>::mma(vc[r][dt], s[0][r], o[0][dt]);
        o[1][dt] = Mfma32<float>::mma(vc[r][dt], s[1][r], o[1][dt]);
      }
    if (t + kWaves < t_end) load_cols<E>(vc, hV, (t + kWaves) * 32, l32, g);
  }

  // Merge the waves' (max, sum, O) of each map in wave order: eight threads per row.
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float lt = halves(l[x]);
    if (g == 0) {
      ml[x][0][wave][l32] = m[x];
      ml[x][1][wave][l32] = lt;
    }
  }
  const int row = tid >> 3, qr = q0 + row;
  f32x4 y[E / 32];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x) __syncthreads();                        // the first map's partials are read
    put_partial<E>(part[wave], o[x], l32, g);
    __syncthreads();
    float M = ml[x][0][0][row], L = 0.f, wt[kWaves];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, ml[x][0][w][row]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      wt[w] = fast_exp2((ml[x][0][w][row] - M) * c);
      L = fmaf(wt[w], ml[x][1][w][row], L);
    }
    const float inv = 1.f / L;
#pragma unroll
    for (int i = 0; i < E / 32; ++i) {
      const int d = 4 * ((tid & 7) + 8 * i);
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32x4 z = *reinterpret_cast<const f32x4*>(&part[w][row * (E + 4) + d]);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(wt[w], z[e], a[e]);
      }
      a *= inv;
      const long long at = ((long long)b * p.S + qr) * p.q_rs + (long long)h * E + d;
      if (x == 0) {
        y[i] = a;
      } else {
        const float lam = load_as_float(p.lam, p.lam_dtype, h);
        if (qr < p.S) {
          if (O2) *reinterpret_cast<f32x4*>(O2 + at) = a;
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = fmaf(-lam, a[e], y[i][e]);
          *reinterpret_cast<f32x4*>(O + at) = a;
        }
      }
    }
    if (LSE && qr < p.S && (tid & 7) == 0)
      LSE[x * diff_plane(p) + (long long)wi.bh * p.S + qr] = M * p.scale + logf(L);
  }
}

// dQ of 32 queries; also their delta_1 and delta_2 (planes of ws, which dK/dV reads) and the
// block's sum of delta_2.
template <int E>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 2 : 1, 8)))
diff_f32_dq_kernel(const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
                   const float* __restrict__ O, const float* __restrict__ O2, const float* __restrict__ dO,
                   const float* __restrict__ LSE, float* __restrict__ ws, float* __restrict__ dQ, DiffParams p) {
  constexpr int DT = E / 32;
  __shared__ __attribute__((aligned(16))) float part[kWaves][32 * (E + 4)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const WorkItem wi = work_item(p.nblk, p.B * p.H, p.div_wi, p.causal, p.wi_blocks_fastest);
  const int b = (int)fdiv((unsigned)wi.bh, p.div_h), h = wi.bh - b * p.H;
  const int hkv = (int)fdiv((unsigned)h, p.div_group);
  const int q0 = wi.blk * 32, qi = q0 + l32;
  const Head hK = head_of(K, b, p.S, p.kv_rs, hkv, E), hV = head_of(V, b, p.S, p.kv_rs, hkv, E);
  f32x4 qf[E / 8], dof[E / 8], kr[E / 8], vr[E / 8];
  float kc[16][DT];
  load_rows<E>(qf, head_of(Q, b, p.S, p.q_rs, h, E), q0, l32, g);
  load_rows<E>(dof, head_of(dO, b, p.S, p.q_rs, h, E), q0, l32, g);
  const int t_end = ((p.causal ? min(p.S, q0 + 32) : p.S) + 31) / 32;
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1, all_hi = p.causal ? q0 : p.S - 1;
  int t = wave;
  if (t < t_end) {
    load_rows<E>(kr, hK, t * 32, l32, g);
    load_rows<E>(vr, hV, t * 32, l32, g);
    load_cols<E>(kc, hK, t * 32, l32, g);
  }

  const float lam = load_as_float(p.lam, p.lam_dtype, h);
  const long long ridx = (long long)wi.bh * p.S + qi, plane = diff_plane(p);
  float L[2] = {INFINITY, INFINITY}, dl[2] = {0.f, 0.f};
  {
    f32x4 of[E / 8], of2[E / 8];
    load_rows<E>(of, head_of(O, b, p.S, p.q_rs, h, E), q0, l32, g);
    load_rows<E>(of2, head_of(O2, b, p.S, p.q_rs, h, E), q0, l32, g);
    float dot = 0.f, dot2 = 0.f;
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dot = fmaf(of[j][e], dof[j][e], dot);
        dot2 = fmaf(of2[j][e], dof[j][e], dot2);
      }
    dl[1] = halves(dot2);
    dl[0] = fmaf(lam, dl[1], halves(dot));
    float sum = dl[1];                             // rows past S: dO reads as 0
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
    if (tid == 0) ws[2 * plane + (long long)wi.bh * p.nblk + wi.blk] = sum;
    if (qi < p.S) {
      L[0] = LSE[ridx] * kLog2e;
      L[1] = LSE[plane + ridx] * kLog2e;
      if (wave == 0 && g == 0) {
        ws[ridx] = dl[0];
        ws[plane + ridx] = dl[1];
      }
    }
  }

  f32x16 acc[half_accs<E>()];
#pragma unroll
  for (int x = 0; x < half_accs<E>(); ++x) acc[x] = zero16();
  const float c = p.scale_log2;
  for (; t < t_end; t += kWaves) {
    const int k0 = t * 32;
    const bool more = t + kWaves < t_end;
    f32x16 s1 = map_scores<E, 0>(kr, qf), s2 = map_scores<E, 1>(kr, qf);
    if (more) load_rows<E>(kr, hK, (t + kWaves) * 32, l32, g);
    const f32x16 ga = dot_rows<E>(vr, dof, zero16());
    if (more) load_rows<E>(vr, hV, (t + kWaves) * 32, l32, g);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s1[r] = fast_exp2(fmaf(s1[r], c, -L[0])) * (ga[r] - dl[0]);
      s2[r] = fast_exp2(fmaf(s2[r], c, -L[1])) * (ga[r] - dl[1]);
    }
    if (k0 + 31 > all_hi) {
      mask_above(s1, key_hi - (k0 + 4 * g), 0.f);
      mask_above(s2, key_hi - (k0 + 4 * g), 0.f);
    }
    add_halves<E>(acc, kc, s1, s2);
    if (more) load_cols<E>(kc, hK, (t + kWaves) * 32, l32, g);
  }
  f32x16 out[DT];
  join_halves<E>(out, acc, p.scale, -p.scale * lam);
  store_sum<E>(part, out, dQ + ((long long)b * p.S + q0) * p.q_rs + (long long)h * E, p.q_rs, p.S - q0, wave, l32, g);
}

// dK / dV of 32 keys: the walk over (head of the group, query tile) is split. The last H
// workgroups (of a causal grid the lightest) also reduce dlam.
template <int E>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 2 : 1, 8)))
diff_f32_dkdv_kernel(const float* __restrict__ Q, const float* __restrict__ K, const float* __restrict__ V,
                     const float* __restrict__ dO, const float* __restrict__ LSE, const float* __restrict__ ws,
                     float* __restrict__ dK, float* __restrict__ dV, DiffParams p) {
  constexpr int DT = E / 32;
  __shared__ __attribute__((aligned(16))) float part[kWaves][32 * (E + 4)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const long long plane = diff_plane(p);
  reduce_dlam(ws + 2 * plane, part[0], p);
  const WorkItem wi = work_item(p.nblk, p.B * p.Hkv, p.div_wi, false, p.wi_blocks_fastest);
  const int b = (int)fdiv((unsigned)wi.bh, p.div_hkv), hkv = wi.bh - b * p.Hkv;
  const int k0 = wi.blk * 32, kj = k0 + l32;
  f32x4 kf[E / 8], vf[E / 8];
  load_rows<E>(kf, head_of(K, b, p.S, p.kv_rs, hkv, E), k0, l32, g);
  load_rows<E>(vf, head_of(V, b, p.S, p.kv_rs, hkv, E), k0, l32, g);
  const int tq_begin = p.causal ? wi.blk : 0, ntq = (p.S + 31) / 32 - tq_begin;
  const int niter = p.group * ntq;
  f32x16 dk[half_accs<E>()], dv[DT];
#pragma unroll
  for (int x = 0; x < half_accs<E>(); ++x) dk[x] = zero16();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dv[dt] = zero16();
  const float c = p.scale_log2;
  int gh = 0, tq = wave;
  for (int it = wave; it < niter; it += kWaves) {
    while (tq >= ntq) {
      tq -= ntq;
      ++gh;
    }
    const int h = hkv * p.group + gh, q0 = (tq_begin + tq) * 32;
    const Head hQ = head_of(Q, b, p.S, p.q_rs, h, E), hO = head_of(dO, b, p.S, p.q_rs, h, E);
    const float lam = load_as_float(p.lam, p.lam_dtype, h);
    f32x4 qr[E / 8], orr[E / 8], Lv[2][4], dl[2][4];
    float qc[16][DT], oc[16][DT];
    load_rows<E>(qr, hQ, q0, l32, g);
    load_rows<E>(orr, hO, q0, l32, g);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const long long head = x * plane + ((long long)b * p.H + h) * p.S;
      load_rowvals(Lv[x], LSE + head, p.S, q0, g);
      load_rowvals(dl[x], ws + head, p.S, q0, g);
    }
    f32x16 s1 = map_scores<E, 0>(qr, kf), s2 = map_scores<E, 1>(qr, kf);
    const f32x16 ga = dot_rows<E>(orr, vf, zero16());
    load_cols<E>(oc, hO, q0, l32, g);
    load_cols<E>(qc, hQ, q0, l32, g);
    // Rows past S: q, dO, L and delta read as 0, so their shares are 0 in every product.
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s1[r] = fast_exp2(fmaf(s1[r], c, -(Lv[0][r >> 2][r & 3] * kLog2e)));
      s2[r] = fast_exp2(fmaf(s2[r], c, -(Lv[1][r >> 2][r & 3] * kLog2e)));
    }
    if (p.causal && q0 < k0 + 31) {
      mask_below(s1, kj - (q0 + 4 * g), 0.f);
      mask_below(s2, kj - (q0 + 4 * g), 0.f);
    }
    f32x16 w;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s2[r] *= -lam;
      w[r] = s1[r] + s2[r];
      s1[r] *= ga[r] - dl[0][r >> 2][r & 3];
      s2[r] *= ga[r] - dl[1][r >> 2][r & 3];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) dv[dt] = Mfma32<float>::mma(oc[r][dt], w[r], dv[dt]);
    add_halves<E>(dk, qc, s1, s2);
    tq += kWaves;
  }
  const long long off = ((long long)b * p.S + k0) * p.kv_rs + (long long)hkv * E;
  f32x16 out[DT];
  join_halves<E>(out, dk, p.scale, p.scale);
  store_sum<E>(part, out, dK + off, p.kv_rs, p.S - k0, wave, l32, g);
  __syncthreads();
  store_sum<E>(part, dv, dV + off, p.kv_rs, p.S - k0, wave, l32, g);
}

namespace {

template <typename F>
hipError_t by_dim(int E, F f) {
  switch (E) {
    case 32: f(std::integral_constant<int, 32>{}); break;
    case 64: f(std::integral_constant<int, 64>{}); break;
    case 128: f(std::integral_constant<int, 128>{}); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

DiffParams for_heads(DiffParams p, long long heads) {
  p.nblk = (p.S + 31) / 32;
  p.wi_blocks_fastest = !p.causal;
  p.div_wi = p.wi_blocks_fastest ? work_item_div_blocks(p.nblk) : work_item_div(heads);
  return p;
}

}  // namespace

// 16-bit inputs (attn_diff16.hip).
long long diff16_workspace_floats(const DiffParams& p, int E);
hipError_t launch_diff16_fwd(int dtype, int E, const void* q, const void* k, const void* v, void* o,
                             void* o2, float* lse, const DiffParams& p, hipStream_t st);
hipError_t launch_diff16_bwd(int dtype, int E, const void* q, const void* k, const void* v,
                             const void* o, const void* o2, const void* dout, const float* lse,
                             float* ws, void* dq, void* dk, void* dv, const DiffParams& p,
                             hipStream_t st);

long long diff_workspace_floats(int dtype, int E, const DiffParams& p) {
  if (dtype != 0) return diff16_workspace_floats(p, E);
  return 2 * diff_plane(p) + (long long)p.B * p.H * ((p.S + 31) / 32);
}

hipError_t launch_diff_fwd(int dtype, int E, const void* q, const void* k, const void* v, void* o,
                           void* o2, float* lse, const DiffParams& pa, hipStream_t st) {
  if (dtype != 0) return launch_diff16_fwd(dtype, E, q, k, v, o, o2, lse, pa, st);
  const DiffParams p = for_heads(pa, (long long)pa.B * pa.H);
  return by_dim(E, [&](auto e) {
    hipLaunchKernelGGL((diff_f32_fwd_kernel<decltype(e)::value>), dim3((unsigned)((long long)p.nblk * p.B * p.H)),
                       dim3(256), 0, st, (const float*)q, (const float*)k, (const float*)v, (float*)o,
                       (float*)o2, lse, p);
  });
}

hipError_t launch_diff_bwd(int dtype, int E, const void* q, const void* k, const void* v,
                           const void* o, const void* o2, const void* dout, const float* lse,
                           float* ws, void* dq, void* dk, void* dv, const DiffParams& pa,
                           hipStream_t st) {
  if (dtype != 0) return launch_diff16_bwd(dtype, E, q, k, v, o, o2, dout, lse, ws, dq, dk, dv, pa, st);
  const DiffParams p = for_heads(pa, (long long)pa.B * pa.H), pk = for_heads(pa, (long long)pa.B * pa.Hkv);
  return by_dim(E, [&](auto e) {
    constexpr int EE = decltype(e)::value;
    hipLaunchKernelGGL((diff_f32_dq_kernel<EE>), dim3((unsigned)((long long)p.nblk * p.B * p.H)), dim3(256), 0,
                       st, (const float*)q, (const float*)k, (const float*)v, (const float*)o,
                       (const float*)o2, (const float*)dout, lse, ws, (float*)dq, p);
    hipLaunchKernelGGL((diff_f32_dkdv_kernel<EE>), dim3((unsigned)((long long)p.nblk * p.B * p.Hkv)), dim3(256),
                       0, st, (const float*)q, (const float*)k, (const float*)v, (const float*)dout, lse, ws,
                       (float*)dk, (float*)dv, pk);
  });
}

}  // namespace mi
