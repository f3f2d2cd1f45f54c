// Differential attention (attn_diff.h's formulas) for 16-bit inputs: forward, dQ (with the
// delta pass) and dK/dV. Tiles come by LDS-DMA into rings and are read as attn16.h says; no
// atomics, every sum in a fixed order.
//
//  * Forward: a wave owns 32 query rows and ONE map, so its registers are those of an
//    ordinary forward with half the score depth; the four waves of a workgroup are two row
//    tiles x two maps over the same K and V tiles. The maps meet in the epilogue, lane for
//    lane through LDS: out = O_1 - lam O_2.
//  * dQ: a wave owns 32 rows of both maps: G = dO V^T is one product for both, and each
//    map's dS feeds its own half of dQ.
//  * dK/dV: a wave owns 32 keys of both maps: dV takes (P_1 - lam P_2)^T dO in one product.
//
// Rounded to the inputs' type, half a step each (2^-9 of a bf16 value, 2^-12 of fp16, on
// average), because the matrix instructions take 16-bit operands: P_m in the forward, P_1 -
// lam P_2 and both dS_m in the backward, and the stored out and P_2 v that delta comes from (a
// float32 copy would be the forward's largest write). That is small beside G where a row sees
// many keys; rows whose keys are in one tile make delta from them, and dlam is corrected by what
// dS_2's float32 sum lacks (dq and dk of sequences of 2 or 3 rows 0.0041 -> 0.0025 off, dlam
// 0.013 -> 0.0018, its own rounding; 2% of a step). Scores, statistics and sums are float32.
//
// What bounds them, at B16 S1024 H12 E64 causal | B1 S8192 H16/4 E128 causal, bf16: forward 68 |
// 439 us, dQ 82 | 502, dK/dV 93 | 677 and a join of 12. E = 64: a wave issues a MFMA in 16
// cycles, an exponential in 8, any other VALU instruction in 4; that alone is 38, 38 and 46 us.
// The VALUs issue in 79, 61 and 56% of the busy cycles, the rest is waits inside the waves that
// the other two (dK/dV: one) of a SIMD do not cover, and the ends of the grid. E = 128: the MFMA
// pipe is busy 49, 41 and 40%, at 2.0 of 2.4 GHz: fewer cycles give less than their share (of
// dK/dV's, 17% fewer gave 8% of its time).
#include <type_traits>
#include <utility>

#include "attn16.h"
#include "attn_diff.h"

namespace mi {

namespace {

template <int I>
using ic = std::integral_constant<int, I>;

// f(ic<0>), ..., f(ic<N - 1>): a loop whose counter is a constant in its body.
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(ic<I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

template <int N>
__device__ __forceinline__ void wait_ring(int n) {
  if (n <= 0) wait_vm<0>();
  else if (n == 1) wait_vm<N>();
  else wait_vm<2 * N>();
}

template <int E>
struct Diff16 {
  static constexpr int BN = 64;                    // rows of a streamed tile
  static constexpr int CH = E / 8;                 // 16-byte chunks per row
  static constexpr int TILE = BN * E * 2;          // bytes of one tile
  static constexpr int LPW = CH / 4;               // DMA instructions per wave per tile
  static constexpr int DS = E / 16, DH = E / 32;   // k-steps over both halves, over one
  static constexpr int DT = E / 32;                // 32-column output tiles
  // E = 32: both halves' columns lie in the one 32-column tile, so each map has an
  // accumulator over all of it and keeps its half.
  static constexpr bool SHARED = DT == 1;
  static constexpr int NA = SHARED ? 2 : DT;       // dQ / dK accumulators
};

// Max of 32 scores (attn_fwd16's: no NaN canonicalisation, scores are finite or -inf).
__device__ __forceinline__ float max32(const f32x16& a, const f32x16& b) {
  float ma = a[0], mb = b[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) {
    ma = __builtin_elementwise_maximum(ma, a[r]);
    mb = __builtin_elementwise_maximum(mb, b[r]);
  }
  return __builtin_elementwise_maximum(ma, mb);
}

// Planes of the backward's workspace, [B, H, S] each, and after them the sums of delta_2
// over the dQ kernel's row blocks.
enum { kDelta1 = 0, kSeed1 = 1, kSeed2 = 2, kCross = 3, kPlanes = 4 };

}  // namespace

// ---------------------------------------------------------------------------
// Forward: 64 query rows of one (batch, head) per workgroup.
// ---------------------------------------------------------------------------
template <typename T, int E>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 3 : 2, 8)))
diff16_fwd_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                  T* __restrict__ O, T* __restrict__ O2, float* __restrict__ LSE, DiffParams p) {
  using C = Diff16<E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  constexpr int BM = 64, BN = C::BN, NS = 2, DH = C::DH, DT = C::DT, LPU = 2 * C::LPW;
  // Ring slot s: K tile ring[s][0], V tile ring[s][1]; unit u = {K tile u + 1, V tile u}.
  __shared__ __attribute__((aligned(1024))) char ring[NS][2][C::TILE];
  __shared__ __attribute__((aligned(1024))) char qstage[C::TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const int rw = wave & 1, mw = wave >> 1;         // row tile, map
  const WorkItem wi = work_item(p.nblk, p.B * p.H, p.div_wi, p.causal, p.wi_blocks_fastest);
  const int b = (int)fdiv((unsigned)wi.bh, p.div_h), h = wi.bh - b * p.H;
  const int hkv = (int)fdiv((unsigned)h, p.div_group);
  const int q0 = wi.blk * BM, qw0 = q0 + rw * 32, qi = qw0 + l32;

  unsigned dvoff[C::LPW];
  dma_offsets<E>(dvoff, wave, lane, p.kv_rs);
  const unsigned m0w = lds_u32(ring[0][0] + wave * 1024);
  const RowTiles tK = row_tiles(K, b, p.S, p.kv_rs, hkv, E), tV = row_tiles(V, b, p.S, p.kv_rs, hkv, E);
  auto issue_unit = [&](int slot, int u) __attribute__((always_inline)) {
    const Rsrc rk = tile_rsrc(tK, u + 1), rv = tile_rsrc(tV, max(u, 0));
#pragma unroll
    for (int j = 0; j < C::LPW; ++j) {
      dma16_buf(rk, dvoff[j], m0w + (unsigned)((2 * slot) * C::TILE + 4096 * j));
      dma16_buf(rv, dvoff[j], m0w + (unsigned)((2 * slot + 1) * C::TILE + 4096 * j));
    }
  };
  {
    unsigned qoff[C::LPW];
    dma_offsets<E>(qoff, wave, lane, p.q_rs);
    const Rsrc rq = tile_rsrc(row_tiles(Q, b, p.S, p.q_rs, h, E), wi.blk);
    const unsigned m0q = lds_u32(qstage + wave * 1024);
#pragma unroll
    for (int j = 0; j < C::LPW; ++j) dma16_buf(rq, qoff[j], m0q + (unsigned)(4096 * j));
  }

  // The workgroup's rows end in the same key tile, so that its waves walk the same tiles and
  // only the last one needs a mask.
  static_assert(BM == BN, "one diagonal tile");
  const int t_last = ((p.causal ? min(p.S, q0 + BM) : p.S) + BN - 1) / BN - 1;

  int kaddr[DH];
#pragma unroll
  for (int ds = 0; ds < DH; ++ds) kaddr[ds] = tile_off<E>(l32, 2 * (mw * DH + ds) + g);
  int vaddr[DT][2];
  tr_offsets<E>(vaddr, lane);
  frag qf[DH];
  f32x16 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oacc[dt] = zero16();
  f32x16 sS[2][2];                                 // scores of two tiles, by parity
  float m_run = -1e30f, l_run = 0.f;
  const float c = p.scale_log2;
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1;
  const int wave_key_lo = p.causal ? qw0 : p.S - 1, wave_key_hi = min(p.causal ? qw0 + 31 : p.S, p.S - 1);

  // One key tile, of which the first HALVES x 32 keys count. LAST: the masked one, which no
  // other follows.
  auto step = [&](auto slot_fill_c, auto par_c, auto last_c, auto halves_c, int t) __attribute__((always_inline)) {
    constexpr int SF = decltype(slot_fill_c)::value, SR = (SF + 1) % NS, PAR = decltype(par_c)::value;
    constexpr bool LAST = decltype(last_c)::value != 0;
    constexpr int HALVES = decltype(halves_c)::value;
    const char* sK = ring[SR][0];
    const char* sV = ring[SR][1];
    f32x16 (&s)[2] = sS[PAR];
    if constexpr (LAST) {
#pragma unroll
      for (int mt = 0; mt < HALVES; ++mt) {
        const int kb = t * BN + mt * 32;
        if (kb + 31 > wave_key_lo) mask_above(s[mt], key_hi - (kb + 4 * g), -INFINITY);
      }
    }
    const float mx = HALVES == 2 ? max32(s[0], s[1]) : max32(s[0], s[0]);
    if (t == 0) {
      m_run = fmaxf(m_run, halves_max(mx));
    } else if (wave_any(mx > m_run + p.resc_th)) {
      const float m_new = fmaxf(m_run, halves_max(mx));
      const float alpha = fast_exp2((m_run - m_new) * c);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
      m_run = m_new;
    }
    const float mc = m_run * c;
    float rs[4] = {0.f, 0.f, 0.f, 0.f};
    auto prob = [&](int idx) __attribute__((always_inline)) {
      const int mt = idx >> 4, r = idx & 15;
      s[mt][r] = fast_exp2(fmaf(s[mt][r], c, -mc));
      if (idx < 4) rs[idx] = s[mt][r];
      else rs[idx & 3] += s[mt][r];
    };
    if constexpr (LAST) {
#pragma unroll
      for (int i = 0; i < 16 * HALVES; ++i) prob(i);
    } else {
      // The next tile's score MFMAs, each followed by a slice of this tile's exps.
      constexpr int NM = 2 * DH, EPM = 32 / NM, LAK = 2;
      f32x16 (&sn)[2] = sS[PAR ^ 1];
      frag kfr[NM];
      auto kread = [&](int i) __attribute__((always_inline)) {
        return lds_frag<T>(sK + kaddr[i >> 1] + (i & 1) * 32 * E * 2);
      };
#pragma unroll
      for (int i = 0; i < LAK; ++i) kfr[i] = kread(i);
      sn[0] = zero16();
      sn[1] = zero16();
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        if (i + LAK < NM) kfr[i + LAK] = kread(i + LAK);
        sn[i & 1] = M::mma(kfr[i], qf[i >> 1], sn[i & 1]);
#pragma unroll
        for (int e = 0; e < EPM; ++e) prob(i * EPM + e);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    // O^T += V^T P^T, V^T fragments LAV MFMAs ahead.
    constexpr int NP = 2 * HALVES * DT, LAV = E >= 128 ? 2 : 1;
    auto vread = [&](int j) __attribute__((always_inline)) {
      const int mt = j / (2 * DT), ks = (j / DT) & 1, dt = j % DT;
      const int roff = (32 * mt + 16 * ks) * E * 2;
      return lds_frag_tr<T>(sV + vaddr[dt][0] + roff, sV + vaddr[dt][1] + roff);
    };
    frag vfr[NP], pb[4];
#pragma unroll
    for (int j = 0; j < LAV; ++j) vfr[j] = vread(j);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      if (j + LAV < NP) vfr[j + LAV] = vread(j + LAV);
      const int mt = j / (2 * DT), ks = (j / DT) & 1, dt = j % DT;
      if (dt == 0) pb[2 * mt + ks] = pack_frag<T>(s[mt], ks * 8);
      oacc[dt] = M::mma(vfr[j], pb[2 * mt + ks], oacc[dt]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (i - 1 <= t_last) issue_unit(i, i - 1);
  __builtin_amdgcn_s_waitcnt(kWaitVm0);
  lds_barrier();
#pragma unroll
  for (int ds = 0; ds < DH; ++ds)
    qf[ds] = lds_frag<T>(qstage + tile_off<E>(32 * rw + l32, 2 * (mw * DH + ds) + g));
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    sS[0][mt] = zero16();
#pragma unroll
    for (int ds = 0; ds < DH; ++ds)
      sS[0][mt] = M::mma(lds_frag<T>(ring[0][0] + kaddr[ds] + mt * 32 * E * 2), qf[ds], sS[0][mt]);
  }
  // (All that the ring will ever hold has been asked for: nothing to wait for behind it.)
  auto fill = [&](auto slot_c, int t) __attribute__((always_inline)) {
    wait_ring<LPU>(min(NS - 2, t_last - t));
    lds_barrier();
    if (t + NS - 1 <= t_last) issue_unit(decltype(slot_c)::value, t + NS - 1);
  };
  auto last = [&](auto par_c) __attribute__((always_inline)) {
    fill(par_c, t_last);
    if (t_last * BN + 32 > wave_key_hi) step(par_c, par_c, ic<1>{}, ic<1>{}, t_last);
    else step(par_c, par_c, ic<1>{}, ic<2>{}, t_last);
  };
  for (int t = 0; t < t_last; t += 2) {
    fill(ic<0>{}, t);
    step(ic<0>{}, ic<0>{}, ic<0>{}, ic<2>{}, t);
    if (t + 1 < t_last) {
      fill(ic<1>{}, t + 1);
      step(ic<1>{}, ic<1>{}, ic<0>{}, ic<2>{}, t + 1);
    }
  }
  if (t_last & 1) last(ic<1>{});
  else last(ic<0>{});

  // The second map's rows, normalised, to the first map's wave: quad after quad, a lane's
  // own 16 bytes each.
  const float l_tot = halves_sum(l_run), inv = qi < p.S ? 1.f / l_tot : 0.f;
  lds_barrier();                                   // every wave has left the ring
  f32x4* xch = reinterpret_cast<f32x4*>(&ring[0][0][0] + rw * (32 * E * 4)) + lane;
  if (mw == 1) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[dt][4 * j + e] *= inv;
        xch[(dt * 4 + j) * 64] = f32x4{oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2],
                                       oacc[dt][4 * j + 3]};
      }
  }
  lds_barrier();
  T* dst = O2;
  if (mw == 0) {
    dst = O;
    const float lam = load_as_float(p.lam, p.lam_dtype, h);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 o2 = xch[(dt * 4 + j) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[dt][4 * j + e] = fmaf(-lam, o2[e], oacc[dt][4 * j + e] * inv);
      }
  }
  if (dst) {
    const long long ow = ((long long)b * p.S + qw0) * p.q_rs + (long long)h * E;
    store_rows_lds<T, E>(oacc, 1.f, &ring[0][0][0] + 2 * 32 * E * 4 + wave * (32 * E * 2), dst + ow, p.q_rs,
                         p.S - qw0, lane);
  }
  if (LSE && qi < p.S && g == 0)
    LSE[mw * diff_plane(p) + (long long)wi.bh * p.S + qi] = m_run * p.scale + logf(l_tot);
}

// ---------------------------------------------------------------------------
// dQ: 128 query rows of one (batch, head) per workgroup, over key tiles. Also the delta
// pass: delta_m from dO and the stored out and o2, the planes that dK/dV reads, and the sum
// of delta_2 over the block.
// ---------------------------------------------------------------------------
template <typename T, int E>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 3 : 2, 8)))
diff16_dq_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                 const T* __restrict__ O, const T* __restrict__ O2, const T* __restrict__ dO,
                 const float* __restrict__ LSE, float* __restrict__ ws, T* __restrict__ dQ, DiffParams p) {
  using C = Diff16<E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  constexpr int BM = 128, BN = C::BN, NS = E >= 128 ? 2 : 3, DS = C::DS, DH = C::DH, DT = C::DT, LPU = 2 * C::LPW;
  __shared__ __attribute__((aligned(1024))) char ring[NS][2][C::TILE];
  __shared__ float sums[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const WorkItem wi = work_item(p.nblk, p.B * p.H, p.div_wi, p.causal, p.wi_blocks_fastest);
  const int b = (int)fdiv((unsigned)wi.bh, p.div_h), h = wi.bh - b * p.H;
  const int hkv = (int)fdiv((unsigned)h, p.div_group);
  const int q0 = wi.blk * BM, qw0 = q0 + wave * 32, qi = qw0 + l32;
  const long long head = (long long)b * p.S * p.q_rs + (long long)h * E;

  frag qf[DS], dof[DS];
  float part = 0.f, part2 = 0.f;
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) {
    const long long off = head + (long long)qi * p.q_rs + ds * 16 + g * 8;
    qf[ds] = qi < p.S ? ld_frag<T>(Q + off) : zero_frag<T>();
    dof[ds] = qi < p.S ? ld_frag<T>(dO + off) : zero_frag<T>();
    const frag of = qi < p.S ? ld_frag<T>(O + off) : zero_frag<T>();
    const frag of2 = qi < p.S ? ld_frag<T>(O2 + off) : zero_frag<T>();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part = fmaf((float)of[e], (float)dof[ds][e], part);
      part2 = fmaf((float)of2[e], (float)dof[ds][e], part2);
    }
  }
  const float lam = load_as_float(p.lam, p.lam_dtype, h);
  float d2 = halves_sum(part2), d1 = fmaf(lam, d2, halves_sum(part));
  float L1 = INFINITY, L2 = INFINITY;              // log2 units; rows past S: P = 0
  const long long ridx = (long long)wi.bh * p.S + qi, plane = diff_plane(p);
  if (qi < p.S) {
    L1 = LSE[ridx] * kLog2e;
    L2 = LSE[plane + ridx] * kLog2e;
  }

  const int t_end = ((p.causal ? min(p.S, q0 + BM) : p.S) + BN - 1) / BN;
  int tw_end = t_end;
  if (qw0 >= p.S) tw_end = 0;
  if (p.causal) tw_end = min(tw_end, (qw0 + 31) / BN + 1);

  unsigned dvoff[C::LPW];
  dma_offsets<E>(dvoff, wave, lane, p.kv_rs);
  const unsigned m0w = lds_u32(ring[0][0] + wave * 1024);
  const RowTiles tK = row_tiles(K, b, p.S, p.kv_rs, hkv, E), tV = row_tiles(V, b, p.S, p.kv_rs, hkv, E);
  auto issue = [&](int slot, int t) __attribute__((always_inline)) {
    const Rsrc rk = tile_rsrc(tK, t), rv = tile_rsrc(tV, t);
#pragma unroll
    for (int j = 0; j < C::LPW; ++j) {
      dma16_buf(rk, dvoff[j], m0w + (unsigned)((2 * slot) * C::TILE + 4096 * j));
      dma16_buf(rv, dvoff[j], m0w + (unsigned)((2 * slot + 1) * C::TILE + 4096 * j));
    }
  };
  int kaddr[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) kaddr[ds] = tile_off<E>(l32, 2 * ds + g);
  int ktoff[DT][2];
  tr_offsets<E>(ktoff, lane);
  f32x16 acc[C::NA];
#pragma unroll
  for (int x = 0; x < C::NA; ++x) acc[x] = zero16();
  const float c = p.scale_log2;
  float cross, ds2 = 0.f;                          // ds2: the lane's sum of P_2 (G - delta_2)
  const int key_hi = p.causal ? min(qi, p.S - 1) : p.S - 1;
  const int wave_key_lo_end = p.causal ? qw0 : p.S, wave_key_hi_end = p.causal ? qw0 + 31 : p.S;

  // One key tile in halves of 32 keys.
  auto compute = [&](const char* sK, const char* sV, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int kb = t * BN + mt * 32;
      if (p.causal && kb > wave_key_hi_end) continue;            // above the diagonal
      const int roff0 = mt * 32 * E * 2;
      frag kfr[DS], vfr[DS];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) kfr[ds] = lds_frag<T>(sK + kaddr[ds] + roff0);
      f32x16 s1 = zero16(), s2 = zero16();
#pragma unroll
      for (int ds = 0; ds < DH; ++ds) {
        s1 = M::mma(kfr[ds], qf[ds], s1);
        s2 = M::mma(kfr[DH + ds], qf[DH + ds], s2);
      }
      // G - delta_1 = V dO^T + (-delta_1), each MFMA under a slice of the exps.
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) vfr[ds] = lds_frag<T>(sV + kaddr[ds] + roff0);
      f32x16 ga;
#pragma unroll
      for (int r = 0; r < 16; ++r) ga[r] = -d1;
      constexpr int EPM = 16 / DS;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        ga = M::mma(vfr[ds], dof[ds], ga);
#pragma unroll
        for (int e = ds * EPM; e < (ds + 1) * EPM; ++e) {
          s1[e] = fast_exp2(fmaf(s1[e], c, -L1));
          s2[e] = fast_exp2(fmaf(s2[e], c, -L2));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kb + 32 > p.S || (p.causal && kb + 31 > wave_key_lo_end)) {
        const unsigned keep = keep_upto(key_hi - (kb + 4 * g));
        mask_keep(s1, keep, 0.f);
        mask_keep(s2, keep, 0.f);
      }
      frag f1[2], f2[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int e = ks * 8; e < ks * 8 + 8; ++e) {
          s1[e] *= ga[e];
          s2[e] *= ga[e] + cross;
          ds2 += s2[e];
        }
        f1[ks] = pack_frag<T>(s1, ks * 8);
        f2[ks] = pack_frag<T>(s2, ks * 8);
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int roff = roff0 + 16 * ks * E * 2;
          const frag kt = lds_frag_tr<T>(sK + ktoff[dt][0] + roff, sK + ktoff[dt][1] + roff);
          if constexpr (C::SHARED) {
            acc[0] = M::mma(kt, f1[ks], acc[0]);
            acc[1] = M::mma(kt, f2[ks], acc[1]);
          } else {
            acc[dt] = M::mma(kt, dt < DT / 2 ? f1[ks] : f2[ks], acc[dt]);
          }
        }
    }
  };
  auto step = [&](auto slot_c, int t) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    wait_ring<LPU>(min(NS - 2, t_end - 1 - t));
    lds_barrier();
    if (t + NS - 1 < t_end) issue((SL + NS - 1) % NS, t + NS - 1);
    if (t < tw_end) compute(ring[SL][0], ring[SL][1], t);
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < t_end) issue(i, i);
  __builtin_amdgcn_s_waitcnt(kWaitVm0);
  lds_barrier();
  // Rows of few keys: dS is a small difference of G and delta, and the stored outputs' rounding
  // would show. Their delta_m = sum_j P_m G is made from the one key tile that they see.
  if (tw_end == 1) {
    const char* sK = ring[0][0];
    const char* sV = ring[0][1];
    float e1 = 0.f, e2 = 0.f;
    for (int mt = 0; mt < 2; ++mt) {
      const int kb = mt * 32, roff = mt * 32 * E * 2;
      f32x16 s1 = zero16(), s2 = zero16(), gr = zero16();
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const frag kf = lds_frag<T>(sK + kaddr[ds] + roff), vf = lds_frag<T>(sV + kaddr[ds] + roff);
        if (ds < DH) s1 = M::mma(kf, qf[ds], s1);
        else s2 = M::mma(kf, qf[ds], s2);
        gr = M::mma(vf, dof[ds], gr);
      }
      const unsigned keep = keep_upto(key_hi - (kb + 4 * g));
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s1[e] = fast_exp2(fmaf(s1[e], c, -L1));
        s2[e] = fast_exp2(fmaf(s2[e], c, -L2));
      }
      mask_keep(s1, keep, 0.f);
      mask_keep(s2, keep, 0.f);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        e1 = fmaf(s1[e], gr[e], e1);
        e2 = fmaf(s2[e], gr[e], e2);
      }
    }
    d1 = halves_sum(e1);
    d2 = halves_sum(e2);
  }
  cross = d1 - d2;
  if (qi < p.S && g == 0) {
    ws[kDelta1 * plane + ridx] = d1;
    ws[kSeed1 * plane + ridx] = LSE[ridx] * (-1.f / p.scale);
    ws[kSeed2 * plane + ridx] = LSE[plane + ridx] * (-1.f / p.scale);
    ws[kCross * plane + ridx] = lam * (d2 - d1);
  }
  for (int t = 0; t < t_end; t += NS) {
    step(ic<0>{}, t);
    if (t + 1 < t_end) step(ic<1>{}, t + 1);
    if constexpr (NS > 2) {
      if (t + 2 < t_end) step(ic<2 % NS>{}, t + 2);
    }
  }

  {
    // The block's sum of delta_2, exact though the stored P_2 v is not: a row's sum of
    // P_2 (G - delta_2) is what delta_2 lacks, P_2's sum being 1. Rows past S add 0 (their dO
    // and P are). Lanes 32 apart hold the same row, and half of its keys each.
    float sum = d2 + halves_sum(ds2);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
    if (lane == 0) sums[wave] = sum;
  }
  lds_barrier();
  if (tid == 0) ws[kPlanes * plane + (long long)wi.bh * p.nblk + wi.blk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  // Each half's columns with their own factor, then whole rows through LDS.
  f32x16 out[DT];
  const float sc1 = p.scale, sc2 = -p.scale * lam;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool second = C::SHARED ? r >= 8 : dt >= DT / 2;
      out[dt][r] = acc[C::SHARED ? (int)second : dt][r] * (second ? sc2 : sc1);
    }
  store_rows_lds<T, E>(out, 1.f, &ring[0][0][0] + wave * (32 * E * 2), dQ + head + (long long)qw0 * p.q_rs,
                       p.q_rs, p.S - qw0, lane);
}

// ---------------------------------------------------------------------------
// dK / dV: 128 keys of one (batch, kv head) per workgroup, over (group head, query tile).
// V is negated once and the score and G accumulators are seeded out of LDS:
//   S'_m = q_m k_m^T - L_m / scale   -> p_m = exp2(c S'_m)
//   G'   = dO (-V)^T + delta_1       -> p_1 G' = -dS_1
//   lam G' + lam (delta_2 - delta_1) -> p_2 times that = dS_2
//
// LINE: where the key blocks are few, a workgroup each leaves the chip half idle (causal
// blocks differ up to S / 64-fold, and a kv head's block walks every head of its group). The
// steps (group head, query tile) of all key blocks then form one line, block after block, cut
// into equal pieces. A block that several pieces share gets float32 partials, at most two
// slots a workgroup, which diff16_join_kernel adds in order. Each block has kLineSetup empty
// steps in front: what starting one costs.
//
// The workgroups of the line's end (the lightest blocks') also reduce dlam.
// ---------------------------------------------------------------------------
constexpr int kLineSetup = 3;

// Steps of the line before key block i of its (batch, kv head), setups included.
__host__ __device__ inline int line_before(const DiffParams& p, int i) {
  const int NT = (p.S + 63) / 64;
  return i * (p.group * NT + kLineSetup) - (p.causal ? p.group * i * (i - 1) : 0);
}
// The key block that step x of a (batch, kv head) belongs to.
__device__ __forceinline__ int line_block(const DiffParams& p, int x) {
  const int NT = (p.S + 63) / 64;
  int i;
  if (p.causal) {
    const float a = (float)(p.group * NT + kLineSetup + p.group);
    i = (int)((a - sqrtf(fmaxf(a * a - 4.f * p.group * (float)x, 0.f))) / (2.f * p.group));
    i = __builtin_amdgcn_readfirstlane(max(0, min(i, p.nblk - 1)));
    while (i > 0 && line_before(p, i) > x) --i;
    while (i + 1 < p.nblk && line_before(p, i + 1) <= x) ++i;
  } else {
    i = x / (p.group * NT + kLineSetup);
  }
  return i;
}

template <typename T, int E, bool LINE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E <= 64 ? 2 : 1, 8)))
diff16_dkdv_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                   const T* __restrict__ dO, const float* __restrict__ ws, T* __restrict__ dK,
                   T* __restrict__ dV, float* __restrict__ part, DiffParams p) {
  using C = Diff16<E>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  constexpr int BK = 128, BQ = C::BN, NS = 4, DS = C::DS, DH = C::DH, DT = C::DT;
  // Filled and drained two slots at a time: a barrier for 128 query rows.
  __shared__ __attribute__((aligned(1024))) char ring[NS][2][C::TILE];   // Q, dO
  __shared__ __attribute__((aligned(16))) float vecs[NS][kPlanes][BQ];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  reduce_dlam(ws + kPlanes * diff_plane(p), vecs[0][0], p);
  int at = 0, end = 1;
  if constexpr (LINE) {
    at = (int)blockIdx.x * p.line_per;
    end = min(at + p.line_per, p.line_n);
  }
  const int begin = at;
  do {
  WorkItem wi;
  int f0 = 0, f1 = 0x7fffffff, took = 1;
  bool whole = true;
  if constexpr (LINE) {
    wi.bh = at / p.line_head;
    const int x = at - wi.bh * p.line_head;
    wi.blk = line_block(p, x);
    const int start = line_before(p, wi.blk), from = x - start;
    const int span = line_before(p, wi.blk + 1) - start, to = min(span, from + end - at);
    f0 = max(from - kLineSetup, 0);
    f1 = to - kLineSetup;
    whole = f0 == 0 && to == span;
    took = to - from;
    if (f1 <= f0) break;                           // the piece ends in a block's empty steps
  } else {
    wi = work_item(p.nblk, p.B * p.Hkv, p.div_wi, false, p.wi_blocks_fastest);
  }
  const int b = (int)fdiv((unsigned)wi.bh, p.div_hkv), hkv = wi.bh - b * p.Hkv;
  const int k0 = wi.blk * BK, kw0 = k0 + wave * 32, kj = kw0 + l32;
  const long long koff = (long long)b * p.S * p.kv_rs + (long long)hkv * E;

  frag kf[DS], vf[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) {
    const long long off = koff + (long long)kj * p.kv_rs + ds * 16 + g * 8;
    kf[ds] = kj < p.S ? ld_frag<T>(K + off) : zero_frag<T>();
    const frag vv = kj < p.S ? ld_frag<T>(V + off) : zero_frag<T>();
    u32x4 bits = __builtin_bit_cast(u32x4, vv);
    bits ^= 0x80008000u;                           // sign of every 16-bit element
    vf[ds] = __builtin_bit_cast(frag, bits);
    if constexpr (E >= 128) {
      // One wave per SIMD: 256 more registers, which MFMA reads its operands from.
      asm("" : "+a"(kf[ds]));
      asm("" : "+a"(vf[ds]));
    }
  }
  const int tq_begin = p.causal ? k0 / BQ : 0, tq_end = (p.S + BQ - 1) / BQ;
  const int ntq = tq_end - tq_begin, niter = LINE ? f1 - f0 : p.group * ntq;

  unsigned dvoff[C::LPW];
  dma_offsets<E>(dvoff, wave, lane, p.q_rs);
  const unsigned m0w = lds_u32(ring[0][0] + wave * 1024);
  const unsigned m0v = lds_u32(vecs[0][0] + wave * 16);
  const long long plane = diff_plane(p);
  // Issue position, one unit per issue; the head's descriptors follow its head.
  const int gh0 = LINE ? f0 / ntq : 0;
  int is_gh = gh0, is_tq = tq_begin + (LINE ? f0 - gh0 * ntq : 0);
  int cp_tq = is_tq, cp_h = hkv * p.group + gh0;
  RowTiles tQ = row_tiles(Q, b, p.S, p.q_rs, cp_h, E);
  RowTiles tO = row_tiles(dO, b, p.S, p.q_rs, cp_h, E);
  const float* vec = ws + ((long long)b * p.H + cp_h) * p.S;
  auto issue = [&](int slot) __attribute__((always_inline)) {
    const Rsrc rq = tile_rsrc(tQ, is_tq), ro = tile_rsrc(tO, is_tq);
#pragma unroll
    for (int j = 0; j < C::LPW; ++j) {
      dma16_buf(rq, dvoff[j], m0w + (unsigned)((2 * slot) * C::TILE + 4096 * j));
      dma16_buf(ro, dvoff[j], m0w + (unsigned)((2 * slot + 1) * C::TILE + 4096 * j));
    }
    const int row0 = is_tq * BQ;
    const unsigned vbytes = (unsigned)min(p.S - row0, BQ) * 4u;
#pragma unroll
    for (int x = 0; x < kPlanes; ++x) {
      const Rsrc rv = make_rsrc(vec + x * plane + row0, vbytes);
      if (lane < 16) dma4_buf(rv, (unsigned)(wave * 16 + lane) * 4u, m0v + (unsigned)((slot * kPlanes + x) * BQ * 4));
    }
    if (++is_tq == tq_end) {
      is_tq = tq_begin;
      if (++is_gh < p.group) {
        const int h = hkv * p.group + is_gh;
        tQ = row_tiles(Q, b, p.S, p.q_rs, h, E);
        tO = row_tiles(dO, b, p.S, p.q_rs, h, E);
        vec += p.S;
      }
    }
  };
  int qaddr[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qaddr[ds] = tile_off<E>(l32, 2 * ds + g);
  int ttoff[DT][2];
  tr_offsets<E>(ttoff, lane);
  f32x16 dk[C::NA], dv[DT];
#pragma unroll
  for (int x = 0; x < C::NA; ++x) dk[x] = zero16();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dv[dt] = zero16();
  const float c = p.scale_log2;
  const int q_lo = p.causal ? kj : 0, wave_q_lo = p.causal ? kw0 + 31 : 0;

  // The MFMAs of 32 query rows in their order: S_1 and S_2 in turn, G, then for each 16 rows
  // dV and dK. Each one's LDS operand is read LA of them ahead, over the ends of halves and
  // tiles (of a pair) too, as the accumulators' seeds are.
  constexpr int PK = C::SHARED ? 3 : 2 * DT, NM = 2 * DS + 2 * PK, LA = E >= 128 ? 4 : 2;
  int vaddr = 4 * g;                               // floats into vecs
  auto operand = [&](int u, int mt, int i) __attribute__((always_inline)) {
    const char* sQ = &ring[0][0][0] + u * 2 * C::TILE + mt * 32 * E * 2;
    const char* sO = sQ + C::TILE;
    if (i < DS) return lds_frag<T>(sQ + qaddr[(i & 1) * DH + (i >> 1)]);
    if (i < 2 * DS) return lds_frag<T>(sO + qaddr[i - DS]);
    const int ks = (i - 2 * DS) / PK, x = (i - 2 * DS) % PK, dt = C::SHARED ? 0 : x >> 1;
    const char* t = (x & 1 ? sQ : sO) + 16 * ks * E * 2;
    return lds_frag_tr<T>(t + ttoff[dt][0], t + ttoff[dt][1]);
  };
  // Elements 4j .. 4j + 3 of an accumulator's plane.
  auto quad = [&](f32x16& a, int plane, int u, int mt, int j) __attribute__((always_inline)) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(&vecs[0][0][0] + vaddr + (u * kPlanes + plane) * BQ + mt * 32 + 8 * j);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[4 * j + e] = v[e];
  };
  f32x16 s1, s2, ga;                               // seeds of the next 32 rows, and these
  frag ahead[LA];
  auto seed = [&](int u, int mt, int x) __attribute__((always_inline)) {
    if (x < 4) quad(s1, kSeed1, u, mt, x);
    else if (x < 8) quad(s2, kSeed2, u, mt, x - 4);
    else quad(ga, kDelta1, u, mt, x - 8);
  };
  auto start = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 12; ++x) seed(u, 0, x);
#pragma unroll
    for (int i = 0; i < LA; ++i) ahead[i] = operand(u, 0, i);
  };
  // Query tile tq in slot u of the pair, in halves of 32 rows; `start` has been called for it.
  auto compute = [&](auto u_c, int tq, float lam) __attribute__((always_inline)) {
    constexpr int U = decltype(u_c)::value;
    const int q0 = tq * BQ;
    const bool need_lo = p.causal && q0 < wave_q_lo, need_hi = q0 + BQ > p.S;
    each<2>([&](auto mt_c) __attribute__((always_inline)) {
      constexpr int mt = decltype(mt_c)::value;
      constexpr bool more = mt == 0 || U == 0;     // another half follows: its unit and half
      constexpr int nu = mt == 0 ? U : 1, nmt = mt ^ 1;
      frag fr[NM];
#pragma unroll
      for (int i = 0; i < LA; ++i) fr[i] = ahead[i];
      f32x16 cr, w;
      frag wf[2], f1[2], f2[2];
      auto elem = [&](int e) __attribute__((always_inline)) {
        w[e] = fmaf(-lam, s2[e], s1[e]);
        s1[e] *= ga[e];
        s2[e] *= fmaf(lam, ga[e], cr[e]);
      };
      auto pack = [&](int ks) __attribute__((always_inline)) {
        wf[ks] = pack_frag<T>(w, ks * 8);
        f1[ks] = pack_frag<T>(s1, ks * 8);
        f2[ks] = pack_frag<T>(s2, ks * 8);
      };
      each<NM>([&](auto i_c) __attribute__((always_inline)) {
        constexpr int i = decltype(i_c)::value;
        constexpr int ks = i < 2 * DS ? -1 : (i - 2 * DS) / PK, x = i < 2 * DS ? 0 : (i - 2 * DS) % PK;
        // This one's place in time: what is read for later ones.
        if constexpr (i + LA < NM) {
          constexpr bool again = C::SHARED && i + LA >= 2 * DS && (i + LA - 2 * DS) % PK == 2;
          fr[i + LA] = again ? fr[i + LA - 1] : operand(U, mt, i + LA);
        } else if constexpr (more) {
          ahead[i + LA - NM] = operand(nu, nmt, i + LA - NM);
        }
        if constexpr (i == 2 * DS - 2) {
          quad(cr, kCross, U, mt, 0);
          quad(cr, kCross, U, mt, 1);
        }
        if constexpr (i == 2 * DS) {
          quad(cr, kCross, U, mt, 2);
          quad(cr, kCross, U, mt, 3);
        }
        if constexpr (ks == 1 && more) {
#pragma unroll
          for (int y = 12 * x / PK; y < 12 * (x + 1) / PK; ++y) seed(nu, nmt, y);
        }
        if constexpr (i == 2 * DS) {
          if (need_lo || need_hi) {
            const int qb = q0 + mt * 32 + 4 * g;
            unsigned keep = need_lo ? keep_from(q_lo - qb) : ~0u;
            if (need_hi) keep &= keep_upto(p.S - 1 - qb);
            mask_keep(s1, keep, 0.f);
            mask_keep(s2, keep, 0.f);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) elem(e);
          pack(0);
        }
        if constexpr (i < DS) {
          if constexpr (i & 1) s2 = M::mma(fr[i], kf[DH + (i >> 1)], s2);
          else s1 = M::mma(fr[i], kf[i >> 1], s1);
        } else if constexpr (i < 2 * DS) {
          ga = M::mma(fr[i], vf[i - DS], ga);
          constexpr int EPM = 16 / DS;
#pragma unroll
          for (int e = (i - DS) * EPM; e < (i - DS + 1) * EPM; ++e) {
            s1[e] = fast_exp2(s1[e] * c);
            s2[e] = fast_exp2(s2[e] * c);
          }
        } else {
          constexpr int dt = C::SHARED ? 0 : x >> 1;
          if constexpr (x == 0 || (!C::SHARED && !(x & 1))) dv[dt] = M::mma(fr[i], wf[ks], dv[dt]);
          else if constexpr (C::SHARED) dk[x - 1] = M::mma(fr[i], x == 1 ? f1[ks] : f2[ks], dk[x - 1]);
          else dk[dt] = M::mma(fr[i], dt < DT / 2 ? f1[ks] : f2[ks], dk[dt]);
          // The other 16 rows' factors under this 16 rows' MFMAs.
          if constexpr (ks == 0) {
#pragma unroll
            for (int e = 8 + 8 * x / PK; e < 8 + 8 * (x + 1) / PK; ++e) elem(e);
            if constexpr (x == PK - 1) pack(1);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };

  // (To a scalar at once: a load still open would be waited for where lam is used, and every
  // DMA in flight with it.)
  auto lam_of = [&](int h) __attribute__((always_inline)) {
    const float x = load_as_float(p.lam, p.lam_dtype, h);
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
  };
  float lam = lam_of(cp_h);
  auto advance = [&](int it) __attribute__((always_inline)) {
    if (++cp_tq == tq_end && it + 1 < niter) {
      cp_tq = tq_begin;
      lam = lam_of(++cp_h);
    }
  };
  issue(0);
  if (niter > 1) issue(1);
  int turn = 1;                                    // which way the next pair of slots lies
  for (int it = 0; it < niter; it += 2) {
    wait_vm<0>();
    lds_barrier();
    if (it + 2 < niter) issue(turn > 0 ? 2 : 0);
    if (it + 3 < niter) issue(turn > 0 ? 3 : 1);
    start(0);
    compute(ic<0>{}, cp_tq, lam);
    advance(it);
    if (it + 1 < niter) {
      compute(ic<1>{}, cp_tq, lam);
      advance(it + 1);
    }
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qaddr[ds] += turn * 4 * C::TILE;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      ttoff[dt][0] += turn * 4 * C::TILE;
      ttoff[dt][1] += turn * 4 * C::TILE;
    }
    vaddr += turn * 2 * kPlanes * BQ;
    turn = -turn;
  }

  lds_barrier();
  char* stage = &ring[0][0][0] + wave * (32 * E * 2);
  const long long off = koff + (long long)kw0 * p.kv_rs;
  f32x16 out[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool second = C::SHARED ? r >= 8 : dt >= DT / 2;
      out[dt][r] = dk[C::SHARED ? (int)second : dt][r] * (second ? p.scale : -p.scale);
    }
  if (whole) {
    store_rows_lds<T, E>(out, 1.f, stage, dK + off, p.kv_rs, p.S - kw0, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    store_rows_lds<T, E>(dv, 1.f, stage, dV + off, p.kv_rs, p.S - kw0, lane);
  } else {
    // This piece's share: [128 keys][dK | dV] floats.
    float* dst = part + ((2LL * blockIdx.x + (at != begin)) * BK + wave * 32 + l32) * (2 * E);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d0 = dt * 32 + 8 * j + 4 * g;
        *reinterpret_cast<f32x4*>(dst + d0) =
            f32x4{out[dt][4 * j], out[dt][4 * j + 1], out[dt][4 * j + 2], out[dt][4 * j + 3]};
        *reinterpret_cast<f32x4*>(dst + E + d0) =
            f32x4{dv[dt][4 * j], dv[dt][4 * j + 1], dv[dt][4 * j + 2], dv[dt][4 * j + 3]};
      }
  }
  at += took;
  if constexpr (LINE) __syncthreads();             // the ring is free for the next block
  } while (LINE && at < end);
}

// The key blocks that several pieces of the line share: their partials added in the line's
// order. A thread per 8 elements of a key's dK or dV, `per_unit` workgroups a block.
template <typename T, int E>
__global__ void __launch_bounds__(256)
diff16_join_kernel(const float* __restrict__ part, T* __restrict__ dK, T* __restrict__ dV, DiffParams p) {
  constexpr int C8 = 2 * E / 8, PER_UNIT = 128 * C8 / 256;
  const int u = blockIdx.x / PER_UNIT, x = (int)(blockIdx.x % PER_UNIT) * 256 + threadIdx.x;
  const int bh = u / p.nblk, blk = u % p.nblk;
  const int start = bh * p.line_head + line_before(p, blk), stop = bh * p.line_head + line_before(p, blk + 1);
  const int g0 = (start + kLineSetup) / p.line_per, g1 = (stop - 1) / p.line_per;
  if (g0 == g1) return;                            // written by the workgroup that had it all
  const int row = x / C8, c = x % C8, kj = blk * 128 + row;
  if (kj >= p.S) return;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, d = a;
  for (int w = g0; w <= g1; ++w) {
    // The first of them may have begun with another block.
    const float* src = part + ((2LL * w + (start > w * p.line_per)) * 128 + row) * (2 * E) + c * 8;
    a += *reinterpret_cast<const f32x4*>(src);
    d += *reinterpret_cast<const f32x4*>(src + 4);
  }
  const bool is_v = c >= C8 / 2;
  const int b = bh / p.Hkv, hkv = bh % p.Hkv;
  T* dst = (is_v ? dV : dK) + ((long long)b * p.S + kj) * p.kv_rs + (long long)hkv * E + (c % (C8 / 2)) * 8;
  st_quad<T>(dst, a[0], a[1], a[2], a[3]);
  st_quad<T>(dst + 4, d[0], d[1], d[2], d[3]);
}

namespace {

template <typename T, int E>
hipError_t diff16_fwd_t(const void* q, const void* k, const void* v, void* o, void* o2, float* lse,
                        DiffParams p, hipStream_t st) {
  p.nblk = (p.S + 63) / 64;
  p.wi_blocks_fastest = !p.causal;
  p.div_wi = p.wi_blocks_fastest ? work_item_div_blocks(p.nblk) : work_item_div((long long)p.B * p.H);
  hipLaunchKernelGGL((diff16_fwd_kernel<T, E>), dim3((unsigned)((long long)p.nblk * p.B * p.H)), dim3(256), 0,
                     st, (const T*)q, (const T*)k, (const T*)v, (T*)o, (T*)o2, lse, p);
  return hipGetLastError();
}

// Whether dK/dV deals its steps evenly, and how: where the key blocks are no more than the
// workgroups that the chip holds at once. Forward + backward, the line's us for a workgroup per
// block's: 105 blocks of E = 32 (full) 80.6 for 106.5, 256 of E = 128 (causal rows of 8192) 1522
// for 1915, 512 of E = 64 290 for 295 (rows of 4096) and 140 for 136 (of 1024); but 768 of E = 64
// 230 for 211 and 149 for 137, 384 of E = 128 385 for 383, 512 of E = 128 276 for 249. Fills the
// line's fields.
int line_slots(int E) { return E <= 64 ? 512 : 256; }

void diff16_line(DiffParams& p, int E) {
  p.line_n = p.line_head = p.line_per = 0;
  const long long nblk = (p.S + 127) / 128, units = nblk * p.B * p.Hkv;
  const long long NT = (p.S + 63) / 64;
  const long long head = nblk * (p.group * NT + kLineSetup) - (p.causal ? p.group * nblk * (nblk - 1) : 0);
  if (units > line_slots(E) || head * p.B * p.Hkv >= (1LL << 30) || p.group * NT >= (1LL << 24)) return;
  p.line_head = (int)head;
  p.line_n = (int)(head * p.B * p.Hkv);
  const int per = (p.line_n + line_slots(E) - 1) / line_slots(E);
  p.line_per = per < 6 ? 6 : per;
}

// Floats of the line's partials: two slots a workgroup.
long long line_floats(const DiffParams& p, int E) {
  return p.line_per ? 2LL * ((p.line_n + p.line_per - 1) / p.line_per) * 128 * 2 * E : 0;
}
// They follow the planes and the sums, 256-byte aligned.
long long line_offset(const DiffParams& p) {
  return (kPlanes * diff_plane(p) + (long long)p.B * p.H * ((p.S + 127) / 128) + 63) / 64 * 64;
}

template <typename T, int E>
hipError_t diff16_bwd_t(const void* q, const void* k, const void* v, const void* o, const void* o2,
                        const void* dout, const float* lse, float* ws, void* dq, void* dk, void* dv,
                        DiffParams p, hipStream_t st) {
  p.nblk = (p.S + 127) / 128;
  p.wi_blocks_fastest = !p.causal;
  p.div_wi = p.wi_blocks_fastest ? work_item_div_blocks(p.nblk) : work_item_div((long long)p.B * p.H);
  hipLaunchKernelGGL((diff16_dq_kernel<T, E>), dim3((unsigned)((long long)p.nblk * p.B * p.H)), dim3(256), 0,
                     st, (const T*)q, (const T*)k, (const T*)v, (const T*)o, (const T*)o2, (const T*)dout,
                     lse, ws, (T*)dq, p);
  DiffParams pk = p;
  pk.div_wi = p.wi_blocks_fastest ? p.div_wi : work_item_div((long long)p.B * p.Hkv);
  diff16_line(pk, E);
  const unsigned units = (unsigned)((long long)p.nblk * p.B * p.Hkv);
  float* part = ws + line_offset(p);
  if (pk.line_per) {
    hipLaunchKernelGGL((diff16_dkdv_kernel<T, E, true>), dim3((pk.line_n + pk.line_per - 1) / pk.line_per),
                       dim3(256), 0, st, (const T*)q, (const T*)k, (const T*)v, (const T*)dout, ws, (T*)dk,
                       (T*)dv, part, pk);
    hipLaunchKernelGGL((diff16_join_kernel<T, E>), dim3(units * (128 * 2 * E / 8 / 256)), dim3(256), 0, st,
                       part, (T*)dk, (T*)dv, pk);
  } else {
    hipLaunchKernelGGL((diff16_dkdv_kernel<T, E, false>), dim3(units), dim3(256), 0, st, (const T*)q,
                       (const T*)k, (const T*)v, (const T*)dout, ws, (T*)dk, (T*)dv, part, pk);
  }
  return hipGetLastError();
}

template <typename F>
hipError_t by_type(int dtype, int E, F f) {
  const auto by_dim = [&](auto t) {
    switch (E) {
      case 32: return f(t, ic<32>{});
      case 64: return f(t, ic<64>{});
      case 128: return f(t, ic<128>{});
    }
    return hipErrorInvalidValue;
  };
  return dtype == 1 ? by_dim(_Float16{}) : by_dim(__bf16{});
}

}  // namespace

long long diff16_workspace_floats(const DiffParams& p, int E) {
  DiffParams l = p;
  diff16_line(l, E);
  return line_offset(p) + line_floats(l, E);
}

hipError_t launch_diff16_fwd(int dtype, int E, const void* q, const void* k, const void* v, void* o,
                             void* o2, float* lse, const DiffParams& p, hipStream_t st) {
  return by_type(dtype, E, [&](auto t, auto e) {
    return diff16_fwd_t<decltype(t), decltype(e)::value>(q, k, v, o, o2, lse, p, st);
  });
}

hipError_t launch_diff16_bwd(int dtype, int E, const void* q, const void* k, const void* v,
                             const void* o, const void* o2, const void* dout, const float* lse,
                             float* ws, void* dq, void* dk, void* dv, const DiffParams& p,
                             hipStream_t st) {
  return by_type(dtype, E, [&](auto t, auto e) {
    return diff16_bwd_t<decltype(t), decltype(e)::value>(q, k, v, o, o2, dout, lse, ws, dq, dk, dv, p, st);
  });
}

}  // namespace mi
