// The cached step of attn_step.h: MFMA tiles fed by LDS-DMA, the keys of the whole batch
// dealt evenly to the workgroups.
//
//  * Work. A unit is one (sequence, kv head, group of NR row tiles of 32 query rows); its
//    key blocks, unit after unit, form one line, cut into equal pieces, one per workgroup:
//    sequences of any lengths load the chip evenly. (Cut per sequence, the longest one sets
//    the time.) Each unit has SETUP empty blocks in front: a piece that reaches into
//    another unit starts its loads anew and writes twice, so it gets fewer keys. The
//    lengths are on the GPU, so each workgroup finds its piece itself, from a prefix sum
//    over them. A piece is one or more fragments of units;
//    a unit that one fragment covers is written at once, the others' fragments go to the
//    workspace as float32 partials (at most the first and the last of a piece are partial:
//    two slots per workgroup) and step_combine_kernel merges them in order.
//    A cache of few rows takes none of this, nor do sequences of one length whose units about
//    fill the chip: a workgroup per unit (direct_steps, even_direct).
//  * Waves. NR row waves x NM map waves x NK key groups. Up to 32 rows, each of four waves
//    takes every fourth block (its own LDS ring, no barrier in the loop) and both maps;
//    with more rows, a group's waves share the blocks of its ring, a row tile and a map
//    each (two 128-wide maps' sums of 32 rows would fill half of the registers). A wave's
//    scores are transposed, S^T = K Q^T, so a lane owns a query row and P^T feeds
//    O^T += V^T P^T from registers (attn16.h's tiles).
//  * Masks only where a block needs one: a sequence's last cached block (rows past it read
//    as zeros through the buffer's bound) and the active block's, one word per block.
//  * P^T of 16-bit inputs is rounded to their type (half a step each): the matrix
//    instructions take 16-bit operands. Partials, statistics and sums are float32.
//  * What bounds it: the cache's bytes. The loop reads 10 bytes a cycle and CU, 5.8 TB/s over
//    the chip (32 query rows a token, D = 128, bf16, 8 sequences of up to 8192 rows: 45 us of
//    kernel, 34 of them the loop; finding the piece and the first loads take 6, the partials 3,
//    and their merge in a second launch 7). Merging them in the unit's last workgroup instead
//    took 1.5 to 19 us more a call: its release and acquire write back and drop a whole L2.
//    One token, 32 sequences of up to 4000 rows: 48 us and a merge of 5, 6.0 TB/s. float32 at
//    D = 128 is bound by the MFMAs of 32 rows, 8200 cycles a block and wave: 121 us for 16
//    sequences of up to 4000 rows (61 at the memory's rate).
#include <type_traits>

#include "attn16.h"
#include "attn_diff.h"
#include "attn_step.h"

namespace mi {

namespace {

template <int I>
using ic = std::integral_constant<int, I>;

// A tile: 32 rows of K or V in LDS as they lie in memory, 16-byte chunk c of row r at chunk
// c ^ swz(r), and the MFMA operands that are read from it. A chunk of a row is a lane's part
// of one product over 2 * EV head dims (K, with Q's chunk at the same place): one MFMA of 16-bit
// elements, four of float32.
template <typename T, int D>
struct Tile {
  static constexpr int EV = 16 / (int)sizeof(T), CH = D / EV, ROW = D * (int)sizeof(T), BYTES = 32 * ROW;
  static constexpr int KS = 16 / EV;             // P^T fragments of a block
  static constexpr bool F32 = std::is_same_v<T, float>;
  using frag = std::conditional_t<F32, f32x4, typename Mfma32<T>::frag>;

  static __device__ __forceinline__ int swz(int row) {
    if constexpr (F32) return row & (CH >= 16 ? 15 : 7);
    else return mi::swz<D>(row);
  }
  static __device__ __forceinline__ frag chunk(const char* p) { return *reinterpret_cast<const frag*>(p); }
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c = Mfma32<float>::mma(a[e], b[e], c);
      return c;
    } else {
      return Mfma32<T>::mma(a, b, c);
    }
  }
  // Rows [16 / KS * ks ..) of P^T: a lane's own scores.
  static __device__ __forceinline__ frag pack(const f32x16& s, int ks) {
    if constexpr (F32) return frag{s[4 * ks], s[4 * ks + 1], s[4 * ks + 2], s[4 * ks + 3]};
    else return pack_frag<T>(s, 8 * ks);
  }

  // V^T for the keys of P^T's fragment ks, head dims [32 dt, 32 dt + 32).
  int off[F32 ? 4 : 2 * (D / 32)];
  __device__ __forceinline__ explicit Tile(int lane) {
    const int l32 = lane & 31, g = lane >> 5;
    if constexpr (F32) {
      // A lane's key of MFMA e is row 8 ks + 4 g + e; its head dim is l32's.
#pragma unroll
      for (int e = 0; e < 4; ++e)
        off[e] = (4 * g + e) * ROW + 16 * ((l32 >> 2) ^ (4 * g + e)) + 4 * (l32 & 3);
    } else {
      int t[D / 32][2];
      tr_offsets<D>(t, lane);
#pragma unroll
      for (int i = 0; i < 2 * (D / 32); ++i) off[i] = t[i / 2][i % 2];
    }
  }
  __device__ __forceinline__ frag values(const char* v, int ks, int dt) const {
    if constexpr (F32) {
      const char* p = v + 8 * ks * ROW + 128 * (CH >= 16 ? dt ^ (ks & 1) : dt);
      frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = *reinterpret_cast<const float*>(p + off[e]);
      return f;
    } else {
      const char* p = v + 16 * ks * ROW;
      return lds_frag_tr<T>(p + off[2 * dt], p + off[2 * dt + 1]);
    }
  }
};

template <typename T, int D, int MAPS, int NR, int NK>
struct Step {
  static constexpr int MW = NR == 1 ? MAPS : 1;  // maps of a wave
  static constexpr int NM = MAPS / MW, NG = NR * NM;   // map waves; waves that share a ring
  static constexpr int W = NG * NK;              // waves
  static constexpr int CH = Tile<T, D>::CH;      // 16-byte chunks per row
  static constexpr int TILE = Tile<T, D>::BYTES; // K (or V) of a block
  static constexpr int LD = TILE / 1024;         // DMA instructions per tile
  static constexpr int IPW = 2 * LD >= NG ? 2 * LD / NG : 1;   // ... of K and V per wave
  // Ring stages. (A fourth instead of the third, or the next block's scores under this one's
  // softmax: within 2%, the loop runs at the memory's rate either way.)
  static constexpr int NS = NK == 4 || NK * TILE > 16384 ? 2 : 3;
  // What starting a unit costs, in blocks (4, 16, 32 of them: 59.2, 55.5, 56.0 us for 8 sequences
  // of up to 8192 rows and 32 tokens; 66.3, 64.9, 68.4 for 32 of up to 4000 and one).
  static constexpr int SETUP = 16;
  static constexpr int RING = NK * NS * 2 * TILE;
  // The waves' float32 results, merged in LDS (the ring's bytes, after the loop).
  static constexpr bool JOIN = NK * NM > 1;
  static constexpr int MERGE = JOIN ? W * 32 * MW * D * 4 : 0;
  static constexpr int LDS = RING > MERGE ? RING : MERGE;
  static constexpr int DS = CH / 2 / NM, DM = DS / MW, DT = D / 32;   // k-steps: a wave's, a map's
  // A slot: the rows' O of each map, then their (m, l).
  static constexpr int ROWS = NR * 32, SLOT = ROWS * (MAPS * D + 2 * MAPS);
};

// The line of blocks: N of them, `per` to a workgroup (N fits 31 bits: validated).
struct Line {
  int N, per;
};

// Sum over the lanes up to and including each (DPP: six VALU instructions).
__device__ __forceinline__ int wave_scan(int x) {
  auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  add(ic<0x111>{}, ic<0xF>{});    // row_shr 1, 2, 4, 8: within rows of 16 lanes
  add(ic<0x112>{}, ic<0xF>{});
  add(ic<0x114>{}, ic<0xF>{});
  add(ic<0x118>{}, ic<0xF>{});
  add(ic<0x142>{}, ic<0xA>{});    // row_bcast15: a row's last lane to the odd rows behind it
  add(ic<0x143>{}, ic<0xC>{});    // row_bcast31: lane 31 to the upper half
  return x;
}
__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// The line as a wave sees it, 64 sequences at a time; the first 64 are kept in the lanes.
struct Scan {
  int len;            // cached rows of sequence `lane`
  int own, upto;      // blocks of one of its units; of all sequences up to it
};

template <int SETUP>
__device__ __forceinline__ Scan scan64(const StepParams& p, int b0) {
  const int i = b0 + (int)(threadIdx.x & 63);
  Scan s;
  s.len = i < p.B ? step_len(p, i) : 0;
  s.own = i < p.B ? (s.len + 31) / 32 + (p.T + 31) / 32 + SETUP : 0;
  s.upto = wave_scan(s.own);
  return s;
}

template <int SETUP>
__device__ __forceinline__ Line step_line(const StepParams& p, int units_per_seq, Scan& first) {
  first = scan64<SETUP>(p, 0);
  int N = lane_value(first.upto, 63);
  for (int b0 = 64; b0 < p.B; b0 += 64) N += lane_value(scan64<SETUP>(p, b0).upto, 63);
  N *= units_per_seq;
  return {N, max((int)(((unsigned)N + p.nsplit - 1) / (unsigned)p.nsplit), p.min_blocks)};
}

// The sequence that holds block x of one unit of each sequence, and the blocks before it.
// `s` becomes the scan that holds it.
template <int SETUP>
__device__ __forceinline__ int find_seq(const StepParams& p, Scan& s, int x, int& before) {
  before = 0;
  for (int b0 = 0;; b0 += 64) {
    if (b0) s = scan64<SETUP>(p, b0);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(before + s.upto > x);
    if (past || b0 + 64 >= p.B) {
      const int l = past ? __builtin_ctzll(past) : min(63, p.B - 1 - b0);
      before += lane_value(s.upto, l) - lane_value(s.own, l);
      return b0 + l;
    }
    before += lane_value(s.upto, 63);
  }
}

// Blocks of one unit of each sequence before `b`; `s` becomes the scan that holds b.
template <int SETUP>
__device__ __forceinline__ int blocks_before(const StepParams& p, Scan& s, int b) {
  int sum = 0;
  for (int b0 = 0; b0 + 64 <= b; b0 += 64) {
    sum += lane_value(s.upto, 63);
    s = scan64<SETUP>(p, b0 + 64);
  }
  return sum + lane_value(s.upto, b & 63) - lane_value(s.own, b & 63);
}

// A tree of at most 64 nodes in a wave's registers: lane t holds node t's line of descent
// and whether it is in the tree (tree_build's doubling, without LDS or barriers).
struct WaveTree {
  unsigned lo, hi;
  int up;
};
__device__ __forceinline__ WaveTree wave_tree(const StepParams& p, int b) {
  const int t = threadIdx.x & 63;
  WaveTree w;
  w.lo = t < 32 ? 1u << t : 0u;
  w.hi = t < 32 ? 0u : 1u << (t - 32);
  w.up = -2;
  if (t < p.T) {
    const int x = p.parents[(long long)b * p.parents_sb + t];
    if (x >= -1 && x < t) w.up = x;
  }
  while (__builtin_amdgcn_ballot_w64(w.up >= 0)) {
    const int from = w.up >= 0 ? w.up : t;
    const unsigned lo = __shfl(w.lo, from), hi = __shfl(w.hi, from);
    const int up = __shfl(w.up, from);
    w.lo |= lo;
    w.hi |= hi;
    w.up = up;
  }
  return w;
}

template <typename T, int D, int MAPS>
__device__ __forceinline__ void step_emit(const StepParams& p, T* __restrict__ out, float* __restrict__ lse,
                                            int b, int kvh, int r, int d0, const f32x4 (&o)[MAPS],
                                            const float (&M)[MAPS], const float (&L)[MAPS], bool dead,
                                            bool poisoned) {
  const int t = (int)fdiv((unsigned)r, p.div_rep), h = kvh * p.rep + r - t * p.rep;
  f32x4 y = o[0] * (1.f / L[0]);
  if constexpr (MAPS == 2) y -= o[1] * (load_as_float(p.lam, p.lam_dtype, h) / L[1]);
  if (p.gate) y *= 1.f / (1.f + __expf(-p.gate[((long long)b * p.T + t) * p.H + h]));
  if (poisoned) y = f32x4{NAN, NAN, NAN, NAN};
  if (dead) y = f32x4{0.f, 0.f, 0.f, 0.f};
  st_quad<T>(out + (((long long)b * p.T + t) * p.H + h) * D + d0, y[0], y[1], y[2], y[3]);
  if (lse && d0 == 0)
    lse[((long long)b * p.H + h) * p.T + t] = dead ? -INFINITY : poisoned ? NAN : M[0] * p.scale + logf(L[0]);
}

}  // namespace

template <typename T, int D, int MAPS, int NR, int NK, bool TREE>
__global__ void __launch_bounds__((64 * Step<T, D, MAPS, NR, NK>::W))
step_kernel(const T* __restrict__ Q, const T* __restrict__ Kc, const T* __restrict__ Vc,
              const T* __restrict__ Kn, const T* __restrict__ Vn, T* __restrict__ O,
              float* __restrict__ LSE, float* __restrict__ part, StepParams p) {
  using C = Step<T, D, MAPS, NR, NK>;
  using X = Tile<T, D>;
  using frag = typename X::frag;
  constexpr int NS = C::NS, DS = C::DS, DM = C::DM, DT = C::DT, TILE = C::TILE, NT = 64 * C::W;
  constexpr int MW = C::MW, NM = C::NM, NG = C::NG;
  // (One row tile: at most 32 nodes.)
  constexpr bool BIG = NR > 1;
  static_assert(!BIG || NT >= kTreeMax, "tree_build wants a thread per node");
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  __shared__ float ml[C::JOIN ? C::W : 1][32][2 * MW];
  __shared__ TreeLds tree;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const int rw = wave % NR, mw = wave / NR % NM, kw = wave / NG;
  const int ngrp = (p.R + C::ROWS - 1) / C::ROWS, ups = p.Hkv * ngrp;   // units per sequence
  // The arguments that are needed only behind the lengths: fetched beside them.
  asm volatile("" ::"s"(Q), "s"(Vn), "s"(part), "s"(p.k_sb), "s"(p.v_sh), "s"(p.parents), "s"(p.div_ngrp.m));
  Scan scan;
  Line line = {0, 0};
  int at = 0, end = 0, b = 0, before = 0;   // this piece of the line; blocks of one unit of each earlier sequence
  if (p.direct) {
    b = (int)fdiv(blockIdx.x, p.div_ups);
    scan.len = step_len(p, b);
    scan.own = (scan.len + 31) / 32 + (p.T + 31) / 32 + C::SETUP;
    at = ((int)blockIdx.x - b * ups) * scan.own;
    end = at + scan.own;
  } else {
    line = step_line<C::SETUP>(p, ups, scan);
    // (Pieces past the line's end: none of the products passes 31 bits, nsplit and per being
    // chosen for the largest N.)
    const long long first = (long long)blockIdx.x * line.per;
    if (first >= line.N) return;
    at = (int)first;
    end = line.N - at > line.per ? at + line.per : line.N;
    b = find_seq<C::SETUP>(p, scan, (int)fdiv((unsigned)at, p.div_ups), before);
  }
  const int begin = at;

  char* ring = lds + kw * (NS * 2 * TILE);
  int kaddr[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) kaddr[ds] = l32 * X::ROW + (((2 * (mw * DS + ds) + g) ^ X::swz(l32)) << 4);
  const X tile(lane);
  const float c = p.scale_log2;
  const bool small_tree = TREE && (!BIG || p.T <= 64);

  while (true) {
    // The fragment of unit u of sequence b that begins at `at`: its blocks [blk0, blk1).
    const int Lc = lane_value(scan.len, b & 63), ncb = (Lc + 31) / 32, nb = ncb + (p.T + 31) / 32;
    const int span = nb + C::SETUP, in_seq = at - before * ups;
    const int u = in_seq / span, from = in_seq - u * span, to = min(span, from + end - at);
    const int blk0 = max(from - C::SETUP, 0), blk1 = to - C::SETUP;
    const int kvh = (int)fdiv((unsigned)u, p.div_ngrp), grp = u - kvh * ngrp;
    const bool whole = blk0 == 0 && blk1 == nb, has_tail = blk1 > ncb;
    if (blk1 > blk0) {

    const char* kc = reinterpret_cast<const char*>(Kc + (long long)b * p.k_sb + (long long)kvh * p.k_sh);
    const char* vc = reinterpret_cast<const char*>(Vc + (long long)b * p.v_sb + (long long)kvh * p.v_sh);
    const char* kn = reinterpret_cast<const char*>(Kn + ((long long)b * p.T * p.Hkv + kvh) * D);
    const char* vn = reinterpret_cast<const char*>(Vn + ((long long)b * p.T * p.Hkv + kvh) * D);

    // Block blk of this wave's ring into a stage: each of the NG waves brings its share
    // of the 1 KB pieces of K and V.
    auto issue = [&](int stage, int blk) __attribute__((always_inline)) {
      const bool tail = blk >= ncb;
      const int k0 = (tail ? blk - ncb : blk) * 32;
      const int n = min(32, (tail ? p.T : Lc) - k0);
      const int ld = tail ? p.Hkv * D : D;                  // elements between rows
      const long long off = (long long)k0 * ld * (int)sizeof(T);
      const unsigned len = (unsigned)((n - 1) * ld + D) * (unsigned)sizeof(T);
      const Rsrc rk = make_rsrc((tail ? kn : kc) + off, len), rv = make_rsrc((tail ? vn : vc) + off, len);
      const unsigned m0 = lds_u32(ring + stage * 2 * TILE);
#pragma unroll
      for (int j = 0; j < C::IPW; ++j) {
        const int i = j * NG + wave % NG;                   // piece: K's, then V's
        if (2 * C::LD < NG && i >= 2 * C::LD) break;
        const int slot = (i % C::LD) * 64 + lane, row = slot / C::CH;
        const unsigned voff = (unsigned)(row * ld) * (unsigned)sizeof(T) + (((slot % C::CH) ^ X::swz(row)) << 4);
        if (i < C::LD) dma16_buf(rk, voff, m0 + (unsigned)(1024 * i));
        else dma16_buf(rv, voff, m0 + (unsigned)(1024 * i));
      }
    };
    const int steps = (blk1 - blk0 + NK - 1) / NK;
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
      if (blk0 + s * NK + kw < blk1) issue(s, blk0 + s * NK + kw);

    // The wave's rows, in flight with the first blocks.
    const int r = (grp * NR + rw) * 32 + l32;
    const bool row = r < p.R;
    const int t = row ? (int)fdiv((unsigned)r, p.div_rep) : 0;
    frag qf[DS];
    const T* qrow = Q + (((long long)b * p.T + t) * p.H + kvh * p.rep + (row ? r - t * p.rep : 0)) * D;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
      qf[ds] = row ? *reinterpret_cast<const frag*>(qrow + (2 * (mw * DS + ds) + g) * X::EV) : frag{};
    unsigned line_lo = 0u, line_hi = 0u;   // a small tree: t's line of descent
    bool dead = false, poisoned = false;
    if (TREE && has_tail) {
      if (small_tree) {
        const WaveTree wt = wave_tree(p, b);
        line_lo = __shfl(wt.lo, t);
        line_hi = __shfl(wt.hi, t);
        dead = __shfl(wt.up, t) != -1;
      } else if constexpr (BIG) {
        tree_build(tree, p, b);
        dead = tree.up[t] != -1;
      }
    }
    auto tree_word = [&](int i) __attribute__((always_inline)) {
      if constexpr (BIG) {
        if (!small_tree) return tree.line[t][i];
      }
      const unsigned lo = line_lo, hi = line_hi;   // (values: no choice between addresses)
      return i ? hi : lo;
    };
    f32x16 o[MW][DT];
    float m[MW], l[MW];
#pragma unroll
    for (int x = 0; x < MW; ++x) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[x][dt] = zero16();
      m[x] = kStepNegInit;
      l[x] = 0.f;
    }
    // Retires the Q loads where the compiler sees it (else it drains the ring in the loop).
    __builtin_amdgcn_s_waitcnt(kWaitVm0);

    int stage = 0;
    for (int s = 0; s < steps; ++s) {
      const int blk = blk0 + s * NK + kw;
      // This stage has landed; at most NS - 2 later ones are still on their way.
      if constexpr (NS == 2) {
        wait_vm<0>();
      } else {
        if (blk + (NS - 2) * NK < blk1) wait_vm<(NS - 2) * C::IPW>();
        else wait_vm<0>();
      }
      if constexpr (NG > 1) lds_barrier();   // everybody's pieces, and the slot refilled now is read
      const int fill = stage == 0 ? NS - 1 : stage - 1;
      if (blk + (NS - 1) * NK < blk1) issue(fill, blk + (NS - 1) * NK);
      const char* sK = ring + stage * 2 * TILE;
      const char* sV = sK + TILE;
      stage = stage + 1 == NS ? 0 : stage + 1;

      const bool tail = blk >= ncb && blk < blk1;
      if (TREE && (NG > 1 ? has_tail && blk0 + s * NK + NK > ncb : tail)) {
        // A value that is not finite would reach every row of the product (0 * inf): its
        // key is taken out of the tile, and the rows that see it are NaN as a whole.
        unsigned badw = 0u;
        if (tail) {
          constexpr unsigned e = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u, e32 = 0x7f800000u;
          for (int i = lane; i < 32 * C::CH; i += 64) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(sV + 16 * i);
            bool nf = false;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (X::F32) nf |= (x[w] & e32) == e32;
              else nf |= (x[w] & e) == e || ((x[w] >> 16) & e) == e;
            }
            // Lanes of a row are neighbours: CH of them.
            const unsigned long long any = __builtin_amdgcn_ballot_w64(nf);
#pragma unroll
            for (int q = 0; q < 64 / C::CH; ++q)
              if ((any >> (q * C::CH)) & ((1ull << (C::CH - 1)) * 2ull - 1ull))
                badw |= 1u << (i / 64 * (64 / C::CH) + q);
          }
        }
        if constexpr (NG > 1) lds_barrier();   // all have looked before any of them writes
        if (badw) {
          for (int i = lane; i < 32 * C::CH; i += 64)
            if ((badw >> (i / C::CH)) & 1u)
              *reinterpret_cast<u32x4*>(const_cast<char*>(sV) + 16 * i) = u32x4{0u, 0u, 0u, 0u};
          poisoned |= !dead && (tree_word(blk - ncb) & badw) != 0u;
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
      }
      if (blk >= blk1) continue;

      f32x16 sc[MW];
#pragma unroll
      for (int x = 0; x < MW; ++x) {
        sc[x] = zero16();
#pragma unroll
        for (int ds = x * DM; ds < (x + 1) * DM; ++ds) sc[x] = X::mma(X::chunk(sK + kaddr[ds]), qf[ds], sc[x]);
      }
      if (tail || blk * 32 + 32 > Lc) {
        unsigned see;
        if (!tail) see = (1u << (Lc - blk * 32)) - 1u;      // 1 .. 31 rows
        else if (!TREE) see = chain_word(p, t, blk - ncb);
        else see = dead ? 0u : tree_word(blk - ncb);
#pragma unroll
        for (int x = 0; x < MW; ++x) mask_keep(sc[x], see >> (4 * g), -INFINITY);
      }
#pragma unroll
      for (int x = 0; x < MW; ++x) {
        float mx = sc[x][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, sc[x][i]);
        // The running max moves only when it grows by more than 8 in log2 units.
        if (wave_any(mx > m[x] + p.resc_th)) {
          const float m_new = fmaxf(m[x], halves_max(mx));
          const float alpha = fast_exp2((m[x] - m_new) * c);
          l[x] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[x][dt][i] *= alpha;
          m[x] = m_new;
        }
        const float mc = m[x] * c;
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[x][i] = fast_exp2(fmaf(sc[x][i], c, -mc));
          rs[i & 3] += sc[x][i];
        }
        l[x] += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      }
#pragma unroll
      for (int ks = 0; ks < X::KS; ++ks) {
        frag pf[MW];
#pragma unroll
        for (int x = 0; x < MW; ++x) pf[x] = X::pack(sc[x], ks);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const frag vt = tile.values(sV, ks, dt);
#pragma unroll
          for (int x = 0; x < MW; ++x) o[x][dt] = X::mma(vt, pf[x], o[x][dt]);
        }
      }
    }

    // The fragment's result. l < 0 marks a row outside the tree, m = NaN a poisoned one.
    const int slot = 2 * blockIdx.x + (at != begin);
    float* po = part + (long long)slot * C::SLOT;
    float* pml = po + C::ROWS * MAPS * D;
#pragma unroll
    for (int x = 0; x < MW; ++x) {
      l[x] = halves_sum(l[x]);
      if (dead) l[x] = -1.f;
      if (poisoned) m[x] = NAN;
    }
    if constexpr (!C::JOIN) {                // one map, one key group: from the registers
      if (row) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d0 = dt * 32 + 8 * j + 4 * g;
            const f32x4 v[1] = {
                {o[0][dt][4 * j], o[0][dt][4 * j + 1], o[0][dt][4 * j + 2], o[0][dt][4 * j + 3]}};
            if (whole) step_emit<T, D, 1>(p, O, LSE, b, kvh, r, d0, v, m, l, dead, poisoned);
            else *reinterpret_cast<f32x4*>(po + (rw * 32 + l32) * D + d0) = v[0];
          }
        if (!whole && g == 0) {
          pml[(rw * 32 + l32) * 2] = m[0];
          pml[(rw * 32 + l32) * 2 + 1] = l[0];
        }
      }
      __syncthreads();   // the ring is free for the next fragment
    } else {
      __syncthreads();   // every wave has left the ring
      // Quad q of a row at q ^ row: the rows' quads in different banks.
      float* ob = reinterpret_cast<float*>(lds);
      constexpr int NQ = D / 4;
#pragma unroll
      for (int x = 0; x < MW; ++x) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 v = {o[x][dt][4 * j], o[x][dt][4 * j + 1], o[x][dt][4 * j + 2], o[x][dt][4 * j + 3]};
            const int q = (dt * 8 + 2 * j + g) ^ (l32 & (NQ - 1));
            *reinterpret_cast<f32x4*>(ob + ((wave * 32 + l32) * MW + x) * D + 4 * q) = v;
          }
        if (g == 0) {
          ml[wave][l32][2 * x] = m[x];
          ml[wave][l32][2 * x + 1] = l[x];
        }
      }
      __syncthreads();
      const int rows = min(p.R - grp * C::ROWS, C::ROWS);
      for (int i = tid; i < rows * NQ; i += NT) {
        const int rr = i / NQ, q = i % NQ, w0 = rr >> 5, rl = rr & 31;
        f32x4 v[MAPS];
        float Mx[MAPS], L[MAPS];
        bool gone = false, nan = false;
#pragma unroll
        for (int x = 0; x < MAPS; ++x) {
          // Map x of key group k: wave w0 + x / MW * NR + k * NG.
          const int w = w0 + x / MW * NR, y = x % MW;
          Mx[x] = ml[w][rl][2 * y];
#pragma unroll
          for (int k = 1; k < NK; ++k) Mx[x] = fmaxf(Mx[x], ml[k * NG + w][rl][2 * y]);
          v[x] = f32x4{0.f, 0.f, 0.f, 0.f};
          L[x] = 0.f;
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            const float mk = ml[k * NG + w][rl][2 * y], lk = ml[k * NG + w][rl][2 * y + 1];
            gone |= lk < 0.f;
            nan |= mk != mk;
            const float a = fast_exp2((mk - Mx[x]) * c);
            L[x] += a * lk;
            v[x] += a * *reinterpret_cast<const f32x4*>(
                            ob + (((k * NG + w) * 32 + rl) * MW + y) * D + 4 * (q ^ (rl & (NQ - 1))));
          }
        }
        if (whole) {
          step_emit<T, D, MAPS>(p, O, LSE, b, kvh, grp * C::ROWS + rr, 4 * q, v, Mx, L, gone, nan);
        } else {
#pragma unroll
          for (int x = 0; x < MAPS; ++x) {
            *reinterpret_cast<f32x4*>(po + (rr * MAPS + x) * D + 4 * q) = v[x];
            if (q == 0) {
              pml[rr * 2 * MAPS + 2 * x] = nan ? NAN : Mx[x];
              pml[rr * 2 * MAPS + 2 * x + 1] = gone ? -1.f : L[x];
            }
          }
        }
      }
      __syncthreads();
    }
    }   // blk1 > blk0

    at += to - from;
    if (at >= end) break;
    if (u + 1 == ups) {                    // the sequence's last unit is done
      before += span;
      if ((++b & 63) == 0) scan = scan64<C::SETUP>(p, b);
    }
  }
}

// The units that several workgroups share, merged in order: a wave per query row.
template <typename T, int D, int MAPS, int NR, int NK>
__global__ void __launch_bounds__(256)
step_combine_kernel(const float* __restrict__ part, T* __restrict__ O, float* __restrict__ LSE,
                      StepParams p) {
  using C = Step<T, D, MAPS, NR, NK>;
  constexpr int NQ = D / 4, FG = 64 / NQ;          // lanes per row, fragments read at once
  const long long gr = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);   // (b, kvh, r)
  if (gr >= (long long)p.B * p.Hkv * p.R) return;                        // whole waves
  const int r = (int)(gr % p.R), kvh = (int)(gr / p.R % p.Hkv), b = (int)(gr / p.R / p.Hkv);
  const int lane = threadIdx.x & 63, q = lane % NQ, fg = lane / NQ;
  const int ngrp = (p.R + C::ROWS - 1) / C::ROWS, ups = p.Hkv * ngrp;
  Scan scan;
  const Line line = step_line<C::SETUP>(p, ups, scan);
  const int grp = r / C::ROWS, rr = r % C::ROWS, before = blocks_before<C::SETUP>(p, scan, b);
  const int span = lane_value(scan.own, b & 63), start = before * ups + (kvh * ngrp + grp) * span;
  const int g0 = (start + C::SETUP) / line.per, g1 = (start + span - 1) / line.per;
  if (g0 == g1) return;                            // written by the workgroup that had it all
  const float c = p.scale_log2;
  f32x4 o[MAPS];
  float M[MAPS], L[MAPS];
  bool dead = false, poisoned = false;
#pragma unroll
  for (int x = 0; x < MAPS; ++x) {
    o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    M[x] = kStepNegInit;
    L[x] = 0.f;
  }
  for (int w = g0 + fg; w <= g1; w += FG) {
    // The first of them may have begun with another unit.
    const float* po = part + (2LL * w + (start > w * line.per)) * C::SLOT;
    const float* pml = po + C::ROWS * MAPS * D + rr * 2 * MAPS;
#pragma unroll
    for (int x = 0; x < MAPS; ++x) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(po + (rr * MAPS + x) * D + 4 * q);
      const float mk = pml[2 * x], lk = pml[2 * x + 1];
      dead |= lk < 0.f;
      poisoned |= mk != mk;
      const float mn = fmaxf(M[x], mk);
      const float a = fast_exp2((M[x] - mn) * c), f = fast_exp2((mk - mn) * c);
      L[x] = L[x] * a + lk * f;
      o[x] = o[x] * a + v * f;
      M[x] = mn;
    }
  }
#pragma unroll
  for (int off = NQ; off < 64; off <<= 1) {
    dead |= __shfl_xor((int)dead, off) != 0;
    poisoned |= __shfl_xor((int)poisoned, off) != 0;
#pragma unroll
    for (int x = 0; x < MAPS; ++x) {
      const float mo = __shfl_xor(M[x], off), lo = __shfl_xor(L[x], off);
      f32x4 oo;
#pragma unroll
      for (int e = 0; e < 4; ++e) oo[e] = __shfl_xor(o[x][e], off);
      const float mn = fmaxf(M[x], mo);
      const float a = fast_exp2((M[x] - mn) * c), f = fast_exp2((mo - mn) * c);
      L[x] = L[x] * a + lo * f;
      o[x] = o[x] * a + oo * f;
      M[x] = mn;
    }
  }
  if (fg == 0) step_emit<T, D, MAPS>(p, O, LSE, b, kvh, r, 4 * q, o, M, L, dead, poisoned);
}

namespace {

// Steps (NK blocks each) up to which a workgroup takes a whole unit by itself: up to where a
// lone workgroup's steps cost what the line's partials and second launch do. Against the line,
// us a call. 16 bits, many units: 16 sequences x 12 kv heads of D = 64, two maps, one token,
// 300 / 1000 / 1500 rows (3, 9, 12 steps) 8.4 / 15.3 / 18.8 for 13.8 / 18.9 / 22.7; 32 x 8 of
// D = 128, lengths drawn from 0 to 300 / 1000: 12.5 / 23.5 for 18.1 / 26.3; but 20 x 8 of up to
// 2000 rows (16 steps) 31.0 for 28.1. Few: 24 x 2 of D = 128, up to 400 / 600 / 800 rows (4, 5,
// 7 steps) 12.6 / 14.1 / 16.8 for 14.3 / 14.6 / 15.0; 3 x 2 of D = 64, 600 / 800 / 1000 rows
// (5, 7, 8 steps) 9.2 / 10.7 / 12.2 for 10.9 / 10.5 / 11.3. float32: 70 x 2 of D = 128, 300 /
// 500 rows (6, 9 steps) 37.4 / 51.7 for 39.9 / 50.1; 3 x 2 of D = 64, 200 / 400 / 600 rows (2,
// 4, 5 steps) 11.7 / 17.0 / 19.8 for 15.1 / 15.3 / 15.5; 4 x 2 of D = 32, 500 / 800 rows (5, 7
// steps) 12.7 / 15.8 for 14.0 / 14.8.
__host__ constexpr int direct_steps(bool f32, int D, long long units) {
  if (f32) return units >= 128 ? 7 : D >= 64 ? 3 : 5;
  return units >= 128 ? 10 : D >= 128 ? 5 : 7;
}
// Sequences of one length whose units come to three quarters of the compute units up to half as
// many again: a workgroup per unit at any length. One token, us, for the line's: 192 units of
// D = 64 (two maps) 4000 rows 42.3 for 45.7, 252 of 3000 41.0 for 44.9, 384 of 2500 49.7 for
// 55.5; of D = 128 192 of 3000 60.2 for 66.0, 384 of 2000 83.7 for 83.3; 16 tokens, 192 of D = 64,
// 4000 rows 42.2 for 49.5. But 128 of D = 128 47.7 for 48.1, 516 of D = 64 65.0 for 56.7.
__host__ constexpr bool even_direct(long long units) { return units >= 192 && units <= 384; }

// Workgroups of a launch: what the chip holds at once (by LDS and registers: two per CU for
// one, 16 sequences of up to 6000 rows, D = 64, 4 / 64 query rows: 30.0 / 36.9 for 31.2 / 38.5
// us), fewer where the longest batch that the cache can hold has less than min_blocks for each
// (two steps; one, two, four of them: one sequence, two kv heads, up to 2000 rows 14.1, 14.0,
// 15.8 us, up to 6000 20.1, 16.7, 17.7).
// `even`: the sequences have one length (a workspace's size is asked for without knowing).
template <typename T, int D, int MAPS, int NR, int NK>
void step_geometry(StepParams& p, bool even) {
  using C = Step<T, D, MAPS, NR, NK>;
  constexpr int per_cu = C::LDS > 80 * 1024 || C::W == 8 ? 1 : 2;
  const int ngrp = (p.R + C::ROWS - 1) / C::ROWS;
  const long long most = (long long)p.B * p.Hkv * ngrp * ((p.rows + 31) / 32 + (p.T + 31) / 32 + C::SETUP);
  p.min_blocks = 2 * NK;
  p.div_ups = fast_div((unsigned)(p.Hkv * ngrp));
  p.div_ngrp = fast_div((unsigned)ngrp);
  const long long want = (most + p.min_blocks - 1) / p.min_blocks;
  p.nsplit = (int)(want < 256 * per_cu ? want : 256 * per_cu);
  // Short caches: a workgroup per unit, with no line to find a place in, no partials and no
  // second launch.
  const long long units = (long long)p.B * p.Hkv * ngrp;
  p.direct = ((p.rows + 31) / 32 + (p.T + 31) / 32 + NK - 1) / NK <= direct_steps(Tile<T, D>::F32, D, units) ||
             (even && even_direct(units));
  if (p.direct) p.nsplit = (int)units;
}

template <typename T, int D, int MAPS, int NR, int NK>
hipError_t step_t(const void* q, const void* kc, const void* vc, const void* kn, const void* vn, void* out,
                    float* lse, float* ws, StepParams p, hipStream_t st) {
  step_geometry<T, D, MAPS, NR, NK>(p, !p.lens);
  const auto go = [&](auto tree) {
    hipLaunchKernelGGL((step_kernel<T, D, MAPS, NR, NK, decltype(tree)::value>), dim3((unsigned)p.nsplit),
                       dim3(64 * Step<T, D, MAPS, NR, NK>::W), 0, st, (const T*)q, (const T*)kc, (const T*)vc, (const T*)kn,
                       (const T*)vn, (T*)out, lse, ws, p);
  };
  if (p.parents) go(std::true_type{});
  else go(std::false_type{});
  if (p.direct) return hipGetLastError();
  const long long rows = (long long)p.B * p.Hkv * p.R;
  hipLaunchKernelGGL((step_combine_kernel<T, D, MAPS, NR, NK>), dim3((unsigned)((rows + 3) / 4)), dim3(256),
                     0, st, ws, (T*)out, lse, p);
  return hipGetLastError();
}

// f(T, D, MAPS, NR, NK) for a step: row waves by the row tiles of a kv head, key groups by
// what the ring of two stages takes (four 128-wide float32 ones would not fit). Against the
// next larger form, us: one tile 64.9 for 67.1 (32 sequences, D = 128, one token) and 17.5 for
// 19.8 (D = 64); two 44.8 for 52.9 (8 sequences of 4096 rows, D = 128, two maps, 16 tokens);
// three or four 55.5 for 69.4 (8 sequences of up to 8192 rows, D = 128, 32 tokens).
template <typename F>
auto step_by_shape(int dtype, const StepParams& p, int D, bool two_maps, F f) {
  const auto by_rows = [&](auto t, auto d, auto maps) {
    const int tiles = (p.R + 31) / 32;
    constexpr int wide = (int)sizeof(t) * decltype(d)::value > 256 ? 2 : 4;
    if (tiles <= 1) return f(t, d, maps, ic<1>{}, ic<wide>{});
    if (tiles <= 2) return f(t, d, maps, ic<2>{}, ic<2>{});
    if constexpr (decltype(maps)::value == 1)
      return tiles <= 4 ? f(t, d, maps, ic<4>{}, ic<2>{}) : f(t, d, maps, ic<8>{}, ic<1>{});
    else
      return f(t, d, maps, ic<4>{}, ic<1>{});
  };
  const auto by_dim = [&](auto t, auto maps) {
    return D == 32 ? by_rows(t, ic<32>{}, maps) : D == 64 ? by_rows(t, ic<64>{}, maps)
                                                          : by_rows(t, ic<128>{}, maps);
  };
  const auto by_type = [&](auto t) { return two_maps ? by_dim(t, ic<2>{}) : by_dim(t, ic<1>{}); };
  return dtype == 0 ? by_type(float{}) : dtype == 1 ? by_type(_Float16{}) : by_type(__bf16{});
}

}  // namespace

long long step_workspace_floats(int dtype, const StepParams& p, int D, bool two_maps) {
  return step_by_shape(dtype, p, D, two_maps, [&](auto t, auto d, auto m, auto nr, auto nk) {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value, MM = decltype(m)::value, RR = decltype(nr)::value,
                  KK = decltype(nk)::value;
    StepParams g = p;
    step_geometry<T, DD, MM, RR, KK>(g, false);
    return g.direct ? 0LL : 2LL * g.nsplit * Step<T, DD, MM, RR, KK>::SLOT;
  });
}

hipError_t launch_step(int dtype, int D, const void* q, const void* kc, const void* vc, const void* kn,
                       const void* vn, void* out, float* lse, float* ws, const StepParams& p,
                       hipStream_t st) {
  return step_by_shape(dtype, p, D, p.lam != nullptr, [&](auto t, auto d, auto m, auto nr, auto nk) {
    return step_t<decltype(t), decltype(d)::value, decltype(m)::value, decltype(nr)::value,
                  decltype(nk)::value>(q, kc, vc, kn, vn, out, lse, ws, p, st);
  });
}

}  // namespace mi
