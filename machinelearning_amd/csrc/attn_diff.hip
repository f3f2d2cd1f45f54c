// Differential attention (attn_diff.h's formulas) in float32: forward, delta, dQ
// and dK/dV, on [B,S,H,E] / [B,S,Hkv,E] tensors with native GQA.
//
// The walk is flash attention's: a workgroup of four waves owns 128 rows, a wave 32;
// key (or query) tiles of 32 rows are staged in LDS, double-buffered through registers;
// scores are computed transposed, so a lane owns one row and the statistics of both
// maps are lane scalars. A half's products take half the head dim's k-steps. No
// atomics: every gradient is written by the workgroup that owns its rows, and the sum
// over rows behind dlam is taken in a fixed order.
#include <type_traits>

#include "attn_diff.h"

namespace mi {

namespace {

template <typename T, int E>
struct Diff {
  using M = Mfma32<T>;
  static constexpr int EPL = M::EPL, KPI = 2 * EPL;
  static constexpr int BM = 128, BN = 32;
  static constexpr int DS = E / KPI;       // k-steps over both halves
  static constexpr int DH = DS / 2;        // ... over one
  static constexpr int DT = E / 32;
  using G = TileGeom<T, BN, E>;
  static constexpr int U = G::UNITS;
  static constexpr int UPT = (2 * U + 255) / 256;
  using Rows = typename M::frag[DS];       // 32 rows as MFMA B fragments
};

// Row `row` of a head whose rows are rs elements apart; zeros at or past S.
template <typename T, int E>
__device__ __forceinline__ void load_rows(typename Diff<T, E>::Rows& f, const T* base, long long rs,
                                          int row, int S, int g) {
  using C = Diff<T, E>;
#pragma unroll
  for (int ds = 0; ds < C::DS; ++ds)
    f[ds] = row < S ? ld_frag<T>(base + (long long)row * rs + ds * C::KPI + g * C::EPL) : zero_frag<T>();
}

}  // namespace

template <typename T, int E>
__global__ void __launch_bounds__(256)
diff_fwd_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                T* __restrict__ O, T* __restrict__ O2, float* __restrict__ LSE, DiffParams p) {
  using C = Diff<T, E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  using G = typename C::G;
  constexpr int EPL = C::EPL, KPI = C::KPI, BM = C::BM, BN = C::BN, DH = C::DH, DT = C::DT;
  constexpr int BUF = G::NAT_BYTES + G::TR_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, g = lane >> 5;
  const int BH = p.B * p.H, bh = blockIdx.x % BH;
  int qb = blockIdx.x / BH;
  if (p.causal) qb = p.nblk - 1 - qb;
  const int b = bh / p.H, h = bh % p.H, hkv = h / p.group;
  const int q0 = qb * BM, qw0 = q0 + wave * 32, qi = qw0 + l32;
  const T* Kb = K + (long long)b * p.S * p.kv_rs + (long long)hkv * E;
  const T* Vb = V + (long long)b * p.S * p.kv_rs + (long long)hkv * E;

  frag qf[C::DS];
  load_rows<T, E>(qf, Q + (long long)b * p.S * p.q_rs + (long long)h * E, p.q_rs, qi, p.S, g);
  const int kend = p.causal ? min(p.S, q0 + BM) : p.S;
  const int t_end = (kend + BN - 1) / BN;

  Unit pre[C::UPT];
  auto load_tile = [&](int t) {
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u < 2 * C::U) unit_load<T, BN, E>(pre[i], u / C::U ? Vb : Kb, p.kv_rs, t * BN, p.S, u % C::U);
    }
  };
  auto store_tile = [&](int buf) {
    char* base = smem + buf * BUF;
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u >= 2 * C::U) continue;
      if (u / C::U == 0) unit_store_nat<T, BN, E>(pre[i], base, u % C::U);
      else unit_store_tr<T, BN, E>(pre[i], base + G::NAT_BYTES, u % C::U);
    }
  };

  f32x16 oacc[2][DT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[m][dt] = zero16();
  float m_run[2] = {-1e30f, -1e30f}, l_run[2] = {0.f, 0.f};
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1;
  const float c = p.scale_log2;

  load_tile(0);
  store_tile(0);
  __syncthreads();
  for (int t = 0; t < t_end; ++t) {
    if (t + 1 < t_end) load_tile(t + 1);
    const int k0 = t * BN;
    if (qw0 < p.S && (!p.causal || k0 <= qw0 + 31)) {
      const char* Ks = smem + (t & 1) * BUF;
      const char* Vt = Ks + G::NAT_BYTES;
      const bool need_mask = k0 + BN > p.S || (p.causal && k0 + BN - 1 > qw0);
      f32x16 s[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int ds = m * DH; ds < (m + 1) * DH; ++ds)
          s[m] = M::mma(ld_frag<T>(nat_ptr<T, BN, E>(Ks, l32, ds * KPI + g * EPL)), qf[ds], s[m]);
        if (need_mask) mask_above(s[m], key_hi - (k0 + 4 * g), -INFINITY);
        float mx = s[m][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[m][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (wave_any(mx > m_run[m] + p.resc_th)) {
          const float m_new = fmaxf(m_run[m], mx);
          const float alpha = fast_exp2((m_run[m] - m_new) * c);
          l_run[m] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[m][dt][r] *= alpha;
          m_run[m] = m_new;
        }
        const float mc = m_run[m] * c;
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[m][r] = fast_exp2(fmaf(s[m][r], c, -mc));
          rs += s[m][r];
        }
        l_run[m] += rs;
      }
#pragma unroll
      for (int st = 0; st < 16 / EPL; ++st) {
        const frag p1 = pack_frag<T>(s[0], st * EPL), p2 = pack_frag<T>(s[1], st * EPL);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const frag vt = ld_frag<T>(tr_ptr<T, BN, E>(Vt, dt * 32 + l32, st * KPI + g * EPL));
          oacc[0][dt] = M::mma(vt, p1, oacc[0][dt]);
          oacc[1][dt] = M::mma(vt, p2, oacc[1][dt]);
        }
      }
    }
    if (t + 1 < t_end) store_tile((t + 1) & 1);
    __syncthreads();
  }

  float l[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) l[m] = l_run[m] + __shfl_xor(l_run[m], 32);
  if (qi >= p.S) return;
  const float lam = load_as_float(p.lam, p.lam_dtype, h);
  const float i1 = 1.f / l[0], i2 = 1.f / l[1];
  const long long off = (long long)b * p.S * p.q_rs + (long long)qi * p.q_rs + (long long)h * E;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float o[4], o2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o2[e] = oacc[1][dt][4 * j + e] * i2;
        o[e] = fmaf(-lam, o2[e], oacc[0][dt][4 * j + e] * i1);
      }
      const int d = dt * 32 + 8 * j + 4 * g;
      st_quad<T>(O + off + d, o[0], o[1], o[2], o[3]);
      if (O2) st_quad<T>(O2 + off + d, o2[0], o2[1], o2[2], o2[3]);
    }
  if (LSE && g == 0) {
    const long long idx = ((long long)b * p.H + h) * p.S + qi;
    LSE[idx] = m_run[0] * p.scale + logf(l[0]);
    LSE[diff_plane(p) + idx] = m_run[1] * p.scale + logf(l[1]);
  }
}

// delta_1, delta_2 of every row and the sums of delta_2 over blocks of 128 rows of a
// (b, h): E / 8 lanes a row, 8 elements each. One pass over dout, out and o2.
template <typename T, int E>
__global__ void __launch_bounds__(256)
diff_delta_kernel(const T* __restrict__ O, const T* __restrict__ O2, const T* __restrict__ dO,
                  float* __restrict__ ws, DiffParams p) {
  constexpr int LPR = E / 8, RPI = 256 / LPR;
  __shared__ float part[256];
  const int bh = blockIdx.x / p.nblk, blk = blockIdx.x % p.nblk;
  const int b = bh / p.H, h = bh % p.H;
  const int li = threadIdx.x % LPR;
  const float lam = load_as_float(p.lam, p.lam_dtype, h);
  float sum2 = 0.f;
  for (int r = threadIdx.x / LPR; r < 128; r += RPI) {
    const int i = blk * 128 + r;
    if (i >= p.S) break;
    const long long off = ((long long)b * p.S + i) * p.q_rs + (long long)h * E + li * 8;
    float d = 0.f, d2 = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)dO[off + e];
      d = fmaf(x, (float)O[off + e], d);
      d2 = fmaf(x, (float)O2[off + e], d2);
    }
#pragma unroll
    for (int s = 1; s < LPR; s <<= 1) {
      d += __shfl_xor(d, s);
      d2 += __shfl_xor(d2, s);
    }
    if (li == 0) {
      const long long idx = (long long)bh * p.S + i;
      ws[idx] = fmaf(lam, d2, d);
      ws[diff_plane(p) + idx] = d2;
      sum2 += d2;
    }
  }
  part[threadIdx.x] = sum2;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if (threadIdx.x < s) part[threadIdx.x] += part[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) ws[2 * diff_plane(p) + (long long)bh * p.nblk + blk] = part[0];
}

// dlam_h = -sum of h's partials, one workgroup per head.
__global__ void __launch_bounds__(256)
diff_dlam_kernel(const float* __restrict__ parts, int nblk, DiffParams p) {
  __shared__ float part[256];
  const int h = blockIdx.x;
  float sum = 0.f;
  for (long long x = threadIdx.x; x < (long long)p.B * nblk; x += 256)
    sum += parts[(x / nblk * p.H + h) * nblk + x % nblk];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if (threadIdx.x < s) part[threadIdx.x] += part[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) store_from_float(p.dlam, p.lam_dtype, h, -part[0]);
}

template <typename T, int E>
__global__ void __launch_bounds__(256)
diff_dq_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
               const T* __restrict__ dO, const float* __restrict__ LSE, const float* __restrict__ ws,
               T* __restrict__ dQ, DiffParams p) {
  using C = Diff<T, E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  using G = typename C::G;
  constexpr int EPL = C::EPL, KPI = C::KPI, BM = C::BM, BN = C::BN, DS = C::DS, DH = C::DH, DT = C::DT;
  constexpr int OFF_V = G::NAT_BYTES, OFF_KT = 2 * G::NAT_BYTES;
  constexpr int BUF = 2 * G::NAT_BYTES + G::TR_BYTES;
  // Columns of dQ: the 16 of a half with E = 32 share a 32-row tile, so both halves'
  // products run over the same K^T tile there and the lanes keep their own half's.
  constexpr bool SHARED = DT == 1;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, g = lane >> 5;
  const int BH = p.B * p.H, bh = blockIdx.x % BH;
  int qb = blockIdx.x / BH;
  if (p.causal) qb = p.nblk - 1 - qb;
  const int b = bh / p.H, h = bh % p.H, hkv = h / p.group;
  const int q0 = qb * BM, qw0 = q0 + wave * 32, qi = qw0 + l32;
  const long long qoff = (long long)b * p.S * p.q_rs + (long long)h * E;
  const T* Kb = K + (long long)b * p.S * p.kv_rs + (long long)hkv * E;
  const T* Vb = V + (long long)b * p.S * p.kv_rs + (long long)hkv * E;

  frag qf[DS], dof[DS];
  load_rows<T, E>(qf, Q + qoff, p.q_rs, qi, p.S, g);
  load_rows<T, E>(dof, dO + qoff, p.q_rs, qi, p.S, g);
  float L2[2] = {INFINITY, INFINITY}, dl[2] = {0.f, 0.f};
  if (qi < p.S) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const long long idx = m * diff_plane(p) + (long long)bh * p.S + qi;
      L2[m] = LSE[idx] * kLog2e;
      dl[m] = ws[idx];
    }
  }
  const int kend = p.causal ? min(p.S, q0 + BM) : p.S;
  const int t_end = (kend + BN - 1) / BN;

  Unit pre[C::UPT];
  auto load_tile = [&](int t) {
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u < 2 * C::U) unit_load<T, BN, E>(pre[i], u / C::U ? Vb : Kb, p.kv_rs, t * BN, p.S, u % C::U);
    }
  };
  auto store_tile = [&](int buf) {
    char* base = smem + buf * BUF;
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u >= 2 * C::U) continue;
      if (u / C::U == 0) {
        unit_store_nat<T, BN, E>(pre[i], base, u % C::U);
        unit_store_tr<T, BN, E>(pre[i], base + OFF_KT, u % C::U);
      } else {
        unit_store_nat<T, BN, E>(pre[i], base + OFF_V, u % C::U);
      }
    }
  };

  constexpr int NA = SHARED ? 2 : DT;
  f32x16 acc[NA];
#pragma unroll
  for (int x = 0; x < NA; ++x) acc[x] = zero16();
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1;
  const float c = p.scale_log2;

  load_tile(0);
  store_tile(0);
  __syncthreads();
  for (int t = 0; t < t_end; ++t) {
    if (t + 1 < t_end) load_tile(t + 1);
    const int k0 = t * BN;
    if (qw0 < p.S && (!p.causal || k0 <= qw0 + 31)) {
      const char* Ks = smem + (t & 1) * BUF;
      const char* Vs = Ks + OFF_V;
      const char* Kt = Ks + OFF_KT;
      const bool need_mask = k0 + BN > p.S || (p.causal && k0 + BN - 1 > qw0);
      f32x16 gacc = zero16(), s[2];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
        gacc = M::mma(ld_frag<T>(nat_ptr<T, BN, E>(Vs, l32, ds * KPI + g * EPL)), dof[ds], gacc);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int ds = m * DH; ds < (m + 1) * DH; ++ds)
          s[m] = M::mma(ld_frag<T>(nat_ptr<T, BN, E>(Ks, l32, ds * KPI + g * EPL)), qf[ds], s[m]);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[m][r] = fast_exp2(fmaf(s[m][r], c, -L2[m])) * (gacc[r] - dl[m]);
        if (need_mask) mask_above(s[m], key_hi - (k0 + 4 * g), 0.f);
      }
#pragma unroll
      for (int st = 0; st < 16 / EPL; ++st) {
        const frag d1 = pack_frag<T>(s[0], st * EPL), d2 = pack_frag<T>(s[1], st * EPL);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const frag kt = ld_frag<T>(tr_ptr<T, BN, E>(Kt, dt * 32 + l32, st * KPI + g * EPL));
          if constexpr (SHARED) {
            acc[0] = M::mma(kt, d1, acc[0]);
            acc[1] = M::mma(kt, d2, acc[1]);
          } else {
            acc[dt] = M::mma(kt, dt < DT / 2 ? d1 : d2, acc[dt]);
          }
        }
      }
    }
    if (t + 1 < t_end) store_tile((t + 1) & 1);
    __syncthreads();
  }

  if (qi >= p.S) return;
  const float sc[2] = {p.scale, -p.scale * load_as_float(p.lam, p.lam_dtype, h)};
  T* dst = dQ + qoff + (long long)qi * p.q_rs;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = SHARED ? j / 2 : dt >= DT / 2;
      const f32x16& a = SHARED ? acc[m] : acc[dt];
      st_quad<T>(dst + dt * 32 + 8 * j + 4 * g, a[4 * j] * sc[m], a[4 * j + 1] * sc[m],
                 a[4 * j + 2] * sc[m], a[4 * j + 3] * sc[m]);
    }
}

template <typename T, int E>
__global__ void __launch_bounds__(256)
diff_dkdv_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                 const T* __restrict__ dO, const float* __restrict__ LSE, const float* __restrict__ ws,
                 T* __restrict__ dK, T* __restrict__ dV, DiffParams p) {
  using C = Diff<T, E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  using G = typename C::G;
  constexpr int EPL = C::EPL, KPI = C::KPI, BK = 128, BQ = C::BN, DS = C::DS, DH = C::DH, DT = C::DT;
  constexpr int OFF_DO = G::NAT_BYTES, OFF_QT = 2 * G::NAT_BYTES, OFF_DOT = OFF_QT + G::TR_BYTES;
  constexpr int OFF_L = OFF_DOT + G::TR_BYTES;      // LSE of both maps (log2 units), delta of both
  constexpr int BUF = OFF_L + 4 * BQ * 4;
  constexpr bool SHARED = DT == 1;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, g = lane >> 5;
  const int BHk = p.B * p.Hkv, bhk = blockIdx.x % BHk;
  const int b = bhk / p.Hkv, hkv = bhk % p.Hkv;
  const int k0 = blockIdx.x / BHk * BK, kw0 = k0 + wave * 32, kj = kw0 + l32;
  const long long koff = (long long)b * p.S * p.kv_rs + (long long)hkv * E;

  frag kf[DS], vf[DS];
  load_rows<T, E>(kf, K + koff, p.kv_rs, kj, p.S, g);
  load_rows<T, E>(vf, V + koff, p.kv_rs, kj, p.S, g);
  constexpr int NA = SHARED ? 2 : DT;
  f32x16 dk[NA], dv[DT];
#pragma unroll
  for (int x = 0; x < NA; ++x) dk[x] = zero16();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dv[dt] = zero16();

  const int tq0 = p.causal ? k0 / BQ : 0;
  const int ntq = (p.S + BQ - 1) / BQ - tq0;
  const int niter = p.group * ntq;
  const float c = p.scale_log2;

  Unit pre[C::UPT];
  float vpre = 0.f;
  auto load_iter = [&](int it) {
    const int h = hkv * p.group + it / ntq, q0 = (tq0 + it % ntq) * BQ;
    const long long qoff = (long long)b * p.S * p.q_rs + (long long)h * E;
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u < 2 * C::U)
        unit_load<T, BQ, E>(pre[i], u / C::U ? dO + qoff : Q + qoff, p.q_rs, q0, p.S, u % C::U);
    }
    if (tid < 4 * BQ) {
      const int m = (tid / BQ) & 1, qq = q0 + tid % BQ;
      const long long idx = m * diff_plane(p) + ((long long)b * p.H + h) * p.S + qq;
      if (tid < 2 * BQ) vpre = qq < p.S ? LSE[idx] * kLog2e : INFINITY;
      else vpre = qq < p.S ? ws[idx] : 0.f;
    }
  };
  auto store_iter = [&](int buf) {
    char* base = smem + buf * BUF;
#pragma unroll
    for (int i = 0; i < C::UPT; ++i) {
      const int u = tid + i * 256;
      if (u >= 2 * C::U) continue;
      unit_store_nat<T, BQ, E>(pre[i], base + (u / C::U ? OFF_DO : 0), u % C::U);
      unit_store_tr<T, BQ, E>(pre[i], base + (u / C::U ? OFF_DOT : OFF_QT), u % C::U);
    }
    if (tid < 4 * BQ) reinterpret_cast<float*>(base + OFF_L)[tid] = vpre;
  };

  load_iter(0);
  store_iter(0);
  __syncthreads();
  for (int it = 0; it < niter; ++it) {
    if (it + 1 < niter) load_iter(it + 1);
    const int q0 = (tq0 + it % ntq) * BQ;
    if (kw0 < p.S && (!p.causal || q0 + BQ - 1 >= kw0)) {
      const char* base = smem + (it & 1) * BUF;
      const float* vec = reinterpret_cast<const float*>(base + OFF_L);
      const float lam = load_as_float(p.lam, p.lam_dtype, hkv * p.group + it / ntq);
      const bool need_mask = p.causal && q0 < kw0 + 31;
      f32x16 gacc = zero16(), s[2], w;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
        gacc = M::mma(ld_frag<T>(nat_ptr<T, BQ, E>(base + OFF_DO, l32, ds * KPI + g * EPL)), vf[ds], gacc);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int ds = m * DH; ds < (m + 1) * DH; ++ds)
          s[m] = M::mma(ld_frag<T>(nat_ptr<T, BQ, E>(base, l32, ds * KPI + g * EPL)), kf[ds], s[m]);
        // Rows past S have L = inf: P = 0.
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 L4 = *reinterpret_cast<const f32x4*>(vec + m * BQ + 8 * j + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][4 * j + e] = fast_exp2(fmaf(s[m][4 * j + e], c, -L4[e]));
        }
        if (need_mask) mask_below(s[m], kj - (q0 + 4 * g), 0.f);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[1][r] *= -lam;
        w[r] = s[0][r] + s[1][r];
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(vec + (2 + m) * BQ + 8 * j + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][4 * j + e] *= gacc[4 * j + e] - d4[e];
        }
#pragma unroll
      for (int st = 0; st < 16 / EPL; ++st) {
        const frag wf = pack_frag<T>(w, st * EPL);
        const frag d1 = pack_frag<T>(s[0], st * EPL), d2 = pack_frag<T>(s[1], st * EPL);
        const int pos = st * KPI + g * EPL;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          dv[dt] = M::mma(ld_frag<T>(tr_ptr<T, BQ, E>(base + OFF_DOT, dt * 32 + l32, pos)), wf, dv[dt]);
          const frag qt = ld_frag<T>(tr_ptr<T, BQ, E>(base + OFF_QT, dt * 32 + l32, pos));
          if constexpr (SHARED) {
            dk[0] = M::mma(qt, d1, dk[0]);
            dk[1] = M::mma(qt, d2, dk[1]);
          } else {
            dk[dt] = M::mma(qt, dt < DT / 2 ? d1 : d2, dk[dt]);
          }
        }
      }
    }
    if (it + 1 < niter) store_iter((it + 1) & 1);
    __syncthreads();
  }

  if (kj >= p.S) return;
  const float sc = p.scale;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x16& a = SHARED ? dk[j / 2] : dk[dt];
      const long long off = koff + (long long)kj * p.kv_rs + dt * 32 + 8 * j + 4 * g;
      st_quad<T>(dK + off, a[4 * j] * sc, a[4 * j + 1] * sc, a[4 * j + 2] * sc, a[4 * j + 3] * sc);
      st_quad<T>(dV + off, dv[dt][4 * j], dv[dt][4 * j + 1], dv[dt][4 * j + 2], dv[dt][4 * j + 3]);
    }
}

namespace {

template <typename T, int E>
hipError_t diff_fwd_t(const void* q, const void* k, const void* v, void* o, void* o2, float* lse,
                      DiffParams p, hipStream_t st) {
  p.nblk = (p.S + 127) / 128;
  hipLaunchKernelGGL((diff_fwd_kernel<T, E>), dim3((unsigned)((long long)p.nblk * p.B * p.H)), dim3(256), 0,
                     st, (const T*)q, (const T*)k, (const T*)v, (T*)o, (T*)o2, lse, p);
  return hipGetLastError();
}

template <typename T, int E>
hipError_t diff_bwd_t(const void* q, const void* k, const void* v, const void* o, const void* o2,
                      const void* dout, const float* lse, float* ws, void* dq, void* dk, void* dv,
                      DiffParams p, hipStream_t st) {
  p.nblk = (p.S + 127) / 128;
  const dim3 rows((unsigned)((long long)p.nblk * p.B * p.H)), keys((unsigned)((long long)p.nblk * p.B * p.Hkv));
  hipLaunchKernelGGL((diff_delta_kernel<T, E>), rows, dim3(256), 0, st, (const T*)o, (const T*)o2,
                     (const T*)dout, ws, p);
  hipLaunchKernelGGL((diff_dq_kernel<T, E>), rows, dim3(256), 0, st, (const T*)q, (const T*)k, (const T*)v,
                     (const T*)dout, lse, ws, (T*)dq, p);
  hipLaunchKernelGGL((diff_dkdv_kernel<T, E>), keys, dim3(256), 0, st, (const T*)q, (const T*)k,
                     (const T*)v, (const T*)dout, lse, ws, (T*)dk, (T*)dv, p);
  launch_diff_dlam(ws + 2 * diff_plane(p), p.nblk, p, st);
  return hipGetLastError();
}

template <typename F>
hipError_t by_dim(int E, F f) {
  switch (E) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
  }
  return hipErrorInvalidValue;
}

}  // namespace

void launch_diff_dlam(const float* parts, int nblk, const DiffParams& p, hipStream_t st) {
  hipLaunchKernelGGL(diff_dlam_kernel, dim3((unsigned)p.H), dim3(256), 0, st, parts, nblk, p);
}

// 16-bit inputs (attn_diff16.hip).
long long diff16_workspace_floats(const DiffParams& p);
hipError_t launch_diff16_fwd(int dtype, int E, const void* q, const void* k, const void* v, void* o,
                             void* o2, float* lse, const DiffParams& p, hipStream_t st);
hipError_t launch_diff16_bwd(int dtype, int E, const void* q, const void* k, const void* v,
                             const void* o, const void* o2, const void* dout, const float* lse,
                             float* ws, void* dq, void* dk, void* dv, const DiffParams& p,
                             hipStream_t st);

long long diff_workspace_floats(int dtype, const DiffParams& p) {
  if (dtype != 0) return diff16_workspace_floats(p);
  return 2 * diff_plane(p) + (long long)p.B * p.H * ((p.S + 127) / 128);
}

hipError_t launch_diff_fwd(int dtype, int E, const void* q, const void* k, const void* v, void* o,
                           void* o2, float* lse, const DiffParams& p, hipStream_t st) {
  if (dtype != 0) return launch_diff16_fwd(dtype, E, q, k, v, o, o2, lse, p, st);
  return by_dim(E, [&](auto e) {
    return diff_fwd_t<float, decltype(e)::value>(q, k, v, o, o2, lse, p, st);
  });
}

hipError_t launch_diff_bwd(int dtype, int E, const void* q, const void* k, const void* v,
                           const void* o, const void* o2, const void* dout, const float* lse,
                           float* ws, void* dq, void* dk, void* dv, const DiffParams& p,
                           hipStream_t st) {
  if (dtype != 0) return launch_diff16_bwd(dtype, E, q, k, v, o, o2, dout, lse, ws, dq, dk, dv, p, st);
  return by_dim(E, [&](auto e) {
    return diff_bwd_t<float, decltype(e)::value>(q, k, v, o, o2, dout, lse, ws, dq, dk, dv, p, st);
  });
}

}  // namespace mi
