// The cached step of attn_step.h for float32: keys split over workgroups, one running
// softmax per query row and map, partials merged in split order (bitwise reproducible).
//
// A workgroup of four waves walks a range of key blocks of one (batch, kv head). Its
// query rows are the T queries x the GQA group (row r = t * rep + head in group), 32 to a
// wave: up to 32 rows, the waves take a key block each (NK = 4); beyond, a row tile each
// (NK = 1) over the same block.
#include <type_traits>

#include "attn_diff.h"
#include "attn_step.h"

namespace mi {

namespace {

template <typename T, int D, int MAPS, int NK>
struct Step {
  using M = Mfma32<T>;
  static constexpr int EPL = M::EPL, KPI = 2 * EPL;
  static constexpr int DS = D / KPI, DM = DS / MAPS, DT = D / 32;   // DM: k-steps per map
  using G = TileGeom<T, 32, D>;
  static constexpr int TILE = G::NAT_BYTES + G::TR_BYTES;           // K and V of a block
  static constexpr int U = G::UNITS;
  static constexpr int UPT = (2 * NK * U + 255) / 256;
};

// Partials of a row: [row][split][MAPS * D floats of unnormalised O, then (m, l) per map].
template <int D, int MAPS>
__host__ __device__ constexpr int part_floats() { return MAPS * D + 2 * MAPS; }

// Whether four dwords hold an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool non_finite(u32x4 x) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      bad |= (x[i] & 0x7f800000u) == 0x7f800000u;
    } else {
      constexpr unsigned e = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
      bad |= (x[i] & e) == e || ((x[i] >> 16) & e) == e;
    }
  }
  return bad;
}

}  // namespace

template <typename T, int D, int MAPS, int NK>
__global__ void __launch_bounds__(256)
step_kernel(const T* __restrict__ Q, const T* __restrict__ Kc, const T* __restrict__ Vc,
            const T* __restrict__ Kn, const T* __restrict__ Vn, float* __restrict__ part,
            StepParams p) {
  using C = Step<T, D, MAPS, NK>;
  using M = Mfma32<T>;
  using frag = typename M::frag;
  using G = typename C::G;
  constexpr int EPL = C::EPL, KPI = C::KPI, DS = C::DS, DM = C::DM, DT = C::DT, NR = 4 / NK;
  __shared__ __attribute__((aligned(16))) char smem[NK * C::TILE];
  __shared__ TreeLds tree;
  __shared__ int bad[NK * 32];      // keys of the staged blocks whose values are not finite

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, g = lane >> 5;
  const int ntiles = (p.R + 31) / 32, ngrp = (ntiles + NR - 1) / NR;
  const int grp = blockIdx.x % ngrp, bk = blockIdx.x / ngrp, split = blockIdx.y;
  const int b = bk / p.Hkv, kvh = bk % p.Hkv;
  const int kw = wave % NK, tile = grp * NR + wave / NK;
  const int r = tile * 32 + l32;
  const bool row = r < p.R;
  const int t = row ? r / p.rep : 0, h = kvh * p.rep + (row ? r % p.rep : 0);

  const int Lc = step_len(p, b), ncb = (Lc + 31) / 32, nb = ncb + (p.T + 31) / 32;
  const int steps = (nb + NK - 1) / NK, per = (steps + p.nsplit - 1) / p.nsplit;
  const int s0 = split * per, s1 = min(steps, s0 + per);
  const bool has_tail = s1 > s0 && s1 * NK > ncb;
  const bool trees = p.parents != nullptr;
  if (trees && has_tail) tree_build(tree, p, b);

  frag qf[DS];
  const T* qrow = Q + (((long long)b * p.T + t) * p.H + h) * D;
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qf[ds] = row ? ld_frag<T>(qrow + ds * KPI + g * EPL) : zero_frag<T>();

  const T* kc = Kc + (long long)b * p.k_sb + (long long)kvh * p.k_sh;
  const T* vc = Vc + (long long)b * p.v_sb + (long long)kvh * p.v_sh;
  const T* kn = Kn + ((long long)b * p.T * p.Hkv + kvh) * D;
  const T* vn = Vn + ((long long)b * p.T * p.Hkv + kvh) * D;
  const long long n_rs = (long long)p.Hkv * D;

  f32x16 o[MAPS][DT];
  float m[MAPS], l[MAPS];
#pragma unroll
  for (int x = 0; x < MAPS; ++x) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = zero16();
    m[x] = kStepNegInit;
    l[x] = 0.f;
  }
  // A row outside the tree sees nothing; one that sees a value that is not finite is NaN.
  const bool dead = has_tail && trees && row && tree.up[t] != -1;
  bool poisoned = false;
  const float c = p.scale_log2;

  for (int st = s0; st < s1; ++st) {
    __syncthreads();
    if (tid < NK * 32) bad[tid] = 0;
    __syncthreads();
    for (int u = tid; u < 2 * NK * C::U; u += 256) {
      const bool is_v = u >= NK * C::U;
      const int x = (u % (NK * C::U)) / C::U, unit = u % C::U, quad = unit % G::QUADS, chunk = unit / G::QUADS;
      const int blk = st * NK + x;
      Unit un;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kr = 4 * quad + i;
        un.r[i] = u32x4{0u, 0u, 0u, 0u};
        if (blk < ncb) {
          const int j = blk * 32 + kr;
          if (j < Lc)
            un.r[i] = *reinterpret_cast<const u32x4*>((is_v ? vc : kc) + (long long)j * D + chunk * (16 / (int)sizeof(T)));
        } else {
          const int j = (blk - ncb) * 32 + kr;
          if (j < p.T && !(trees && tree.up[j] != -1)) {
            un.r[i] = *reinterpret_cast<const u32x4*>((is_v ? vn : kn) + (long long)j * n_rs + chunk * (16 / (int)sizeof(T)));
            if (trees && is_v && non_finite<T>(un.r[i])) bad[x * 32 + kr] = 1;
          }
        }
      }
      char* base = smem + x * C::TILE;
      if (is_v) unit_store_tr<T, 32, D>(un, base + G::NAT_BYTES, unit);
      else unit_store_nat<T, 32, D>(un, base, unit);
    }
    __syncthreads();
    const int blk = st * NK + kw;
    if (blk >= nb) continue;          // the barriers are at the loop's head
    unsigned see, badw = 0u;
    if (blk < ncb) {
      const int n = Lc - blk * 32;
      see = n >= 32 ? ~0u : (1u << n) - 1u;
    } else {
      see = trees ? tree.line[t][blk - ncb] : chain_word(p, t, blk - ncb);
      if (trees) badw = (unsigned)__builtin_amdgcn_ballot_w64(lane < 32 && bad[kw * 32 + l32]);
    }
    if (dead) see = 0u;
    // A value that is not finite would reach every row of the product (0 * inf): its row
    // is taken out of the tile, and the rows that see it are NaN as a whole.
    char* base = smem + kw * C::TILE;
    if (badw) {
      poisoned |= (see & badw) != 0u;
      if (NK == 4 || wave == 0)
        for (int d = lane; d < D; d += 64)
          for (int kr = 0; kr < 32; ++kr)
            if ((badw >> kr) & 1u) *const_cast<T*>(tr_ptr<T, 32, D>(base + G::NAT_BYTES, d, perm_pos<EPL>(kr))) = (T)0.f;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (NK == 1) __syncthreads();      // badw is the same in every wave
    }
    const unsigned keep = see >> (4 * g);
    f32x16 s[MAPS];
#pragma unroll
    for (int x = 0; x < MAPS; ++x) {
      s[x] = zero16();
#pragma unroll
      for (int ds = x * DM; ds < (x + 1) * DM; ++ds)
        s[x] = M::mma(ld_frag<T>(nat_ptr<T, 32, D>(base, l32, ds * KPI + g * EPL)), qf[ds], s[x]);
      mask_keep(s[x], keep, -INFINITY);
      float mx = s[x][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[x][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m[x], mx);
      const float alpha = fast_exp2((m[x] - m_new) * c);
      m[x] = m_new;
      l[x] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][dt][i] *= alpha;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[x][i] = fast_exp2(fmaf(s[x][i], c, -m_new * c));
        l[x] += s[x][i];
      }
    }
#pragma unroll
    for (int ks = 0; ks < 16 / EPL; ++ks) {
      frag pf[MAPS];
#pragma unroll
      for (int x = 0; x < MAPS; ++x) pf[x] = pack_frag<T>(s[x], ks * EPL);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const frag vt = ld_frag<T>(tr_ptr<T, 32, D>(base + G::NAT_BYTES, dt * 32 + l32, ks * KPI + g * EPL));
#pragma unroll
        for (int x = 0; x < MAPS; ++x) o[x][dt] = M::mma(vt, pf[x], o[x][dt]);
      }
    }
  }

  if (!row) return;
  // l < 0 marks a row outside the tree, m = NaN a poisoned one.
  const int splits = p.nsplit * NK;
  float* dst = part + (((long long)bk * p.R + r) * splits + split * NK + kw) * part_floats<D, MAPS>();
#pragma unroll
  for (int x = 0; x < MAPS; ++x) {
    const float lt = l[x] + __shfl_xor(l[x], 32);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float* d = dst + x * D + dt * 32 + 8 * j + 4 * g;
        d[0] = o[x][dt][4 * j];
        d[1] = o[x][dt][4 * j + 1];
        d[2] = o[x][dt][4 * j + 2];
        d[3] = o[x][dt][4 * j + 3];
      }
    if (g == 0) {
      dst[MAPS * D + 2 * x] = poisoned ? NAN : m[x];
      dst[MAPS * D + 2 * x + 1] = dead ? -1.f : lt;
    }
  }
}

// Merge of a row's partials in split order, and the output: a workgroup of D threads per
// row, one per head dim.
template <typename T, int D, int MAPS>
__global__ void __launch_bounds__(D)
step_combine_kernel(const float* __restrict__ part, T* __restrict__ out, float* __restrict__ lse,
                    int splits, StepParams p) {
  const long long gr = blockIdx.x;
  const int r = (int)(gr % p.R);
  const long long bk = gr / p.R;
  const int b = (int)(bk / p.Hkv), kvh = (int)(bk % p.Hkv);
  const int t = r / p.rep, h = kvh * p.rep + r % p.rep, d = threadIdx.x;
  constexpr int F = part_floats<D, MAPS>();
  const float* src = part + gr * splits * F;
  float o[MAPS], Mx[MAPS], L[MAPS];
  bool dead = false, poisoned = false;
#pragma unroll
  for (int x = 0; x < MAPS; ++x) {
    o[x] = L[x] = 0.f;
    Mx[x] = kStepNegInit;
    for (int s = 0; s < splits; ++s) {
      const float m = src[s * F + MAPS * D + 2 * x], l = src[s * F + MAPS * D + 2 * x + 1];
      dead |= l < 0.f;
      poisoned |= m != m;
      const float mn = fmaxf(Mx[x], m);
      const float a = fast_exp2((Mx[x] - mn) * p.scale_log2), w = fast_exp2((m - mn) * p.scale_log2);
      L[x] = L[x] * a + l * w;
      o[x] = o[x] * a + src[s * F + x * D + d] * w;
      Mx[x] = mn;
    }
  }
  float y = o[0] / L[0];
  if constexpr (MAPS == 2) y -= load_as_float(p.lam, p.lam_dtype, h) * (o[1] / L[1]);
  if (p.gate) y *= 1.f / (1.f + __expf(-p.gate[((long long)b * p.T + t) * p.H + h]));
  if (poisoned) y = NAN;
  if (dead) y = 0.f;
  out[(((long long)b * p.T + t) * p.H + h) * D + d] = (T)y;
  if (lse && d == 0)
    lse[((long long)b * p.H + h) * p.T + t] = dead ? -INFINITY : Mx[0] * p.scale + logf(L[0]);
}

namespace {

// Splits: about two workgroups per compute unit, at least four steps each.
template <int NK>
int step_splits(const StepParams& p) {
  const int NR = 4 / NK;
  const long long units = (long long)p.B * p.Hkv * (((p.R + 31) / 32 + NR - 1) / NR);
  const long long steps = ((p.rows + 31) / 32 + (p.T + 31) / 32 + NK - 1) / NK;
  const long long want = (512 + units - 1) / units, cap = steps / 4;
  return (int)(want < cap ? want : cap > 1 ? cap : 1);
}

template <typename T, int D, int MAPS, int NK>
hipError_t step_t(const void* q, const void* kc, const void* vc, const void* kn, const void* vn, void* out,
                  float* lse, float* ws, StepParams p, hipStream_t st) {
  constexpr int NR = 4 / NK;
  p.nsplit = step_splits<NK>(p);
  const long long units = (long long)p.B * p.Hkv * (((p.R + 31) / 32 + NR - 1) / NR);
  hipLaunchKernelGGL((step_kernel<T, D, MAPS, NK>), dim3((unsigned)units, (unsigned)p.nsplit), dim3(256), 0,
                     st, (const T*)q, (const T*)kc, (const T*)vc, (const T*)kn, (const T*)vn, ws, p);
  hipLaunchKernelGGL((step_combine_kernel<T, D, MAPS>), dim3((unsigned)((long long)p.B * p.Hkv * p.R)),
                     dim3(D), 0, st, ws, (T*)out, lse, p.nsplit * NK, p);
  return hipGetLastError();
}

template <typename F>
hipError_t by_shape(int D, bool two_maps, F f) {
  const auto by_maps = [&](auto t, auto d) {
    return two_maps ? f(t, d, std::integral_constant<int, 2>{}) : f(t, d, std::integral_constant<int, 1>{});
  };
  const auto by_dim = [&](auto t) {
    switch (D) {
      case 32: return by_maps(t, std::integral_constant<int, 32>{});
      case 64: return by_maps(t, std::integral_constant<int, 64>{});
      case 128: return by_maps(t, std::integral_constant<int, 128>{});
    }
    return hipErrorInvalidValue;
  };
  return by_dim(float{});
}

}  // namespace

long long step16_workspace_floats(const StepParams& p, int D, bool two_maps);
hipError_t launch_step16(int dtype, int D, const void* q, const void* kc, const void* vc, const void* kn,
                         const void* vn, void* out, float* lse, float* ws, const StepParams& p,
                         hipStream_t st);

long long step_workspace_floats(int dtype, const StepParams& p, int D, bool two_maps) {
  if (dtype != 0) return step16_workspace_floats(p, D, two_maps);
  const int maps = two_maps ? 2 : 1;
  const long long splits = p.R <= 32 ? 4LL * step_splits<4>(p) : step_splits<1>(p);
  return (long long)p.B * p.Hkv * p.R * splits * (maps * D + 2 * maps);
}

hipError_t launch_step(int dtype, int D, const void* q, const void* kc, const void* vc, const void* kn,
                       const void* vn, void* out, float* lse, float* ws, const StepParams& p,
                       hipStream_t st) {
  if (dtype != 0) return launch_step16(dtype, D, q, kc, vc, kn, vn, out, lse, ws, p, st);
  return by_shape(D, p.lam != nullptr, [&](auto t, auto d, auto m) {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value, MM = decltype(m)::value;
    return p.R <= 32 ? step_t<T, DD, MM, 4>(q, kc, vc, kn, vn, out, lse, ws, p, st)
                     : step_t<T, DD, MM, 1>(q, kc, vc, kn, vn, out, lse, ws, p, st);
  });
}

}  // namespace mi
