// Attention forward on gfx950: one softmax map with a learned relative position bias by buckets, or two maps whose difference
// is taken with a learned weight.
//   one map:   o_i = sum_j softmax_j( scale q_i.k_j + table[bucket(j - p_i), h] ) v_j            p_i = q_start + i
//   two maps:  o_i = sum_j ( softmax_j(scale q1_i.k1_j) - lambda softmax_j(scale q2_i.k2_j) ) v_j
// One pass over the keys with running maximum and sum; a score never leaves its wave.
//
// attn_fwd_kernel: 4 waves of 32 queries share 64-key tiles of K and V in LDS (double buffered, the next tile's copies in flight
//   over the present one's products).  S^T = K Q^T puts the query on the lane: row statistics are in-lane but for one lane-half
//   exchange, and the weights are the next product's operand as they stand: O^T += V^T P^T.
//   Heads of 64 (4 x 16 heads, 2048 tokens, bfloat16): 106 us = 650 TFLOP/s, bound by the vector pipe (57 % of the cycles: exponentials,
//   bias, maximum; matrix pipe 29); heads of 128 (16 heads, 8192 causal, half): 315 us = 870 with pauses between the calls (385 back to
//   back, at the power limit), matrix 40, vector 42, LDS 41 %.
//   Held in fewer bits than f32, in 16-bit calls: a weight, rounded to the element type as the product's operand (their sum is not).  An
//   output of bfloat16 is 2.1e-3 to 2.6e-3 off with it, 1.7e-3 by its own rounding alone.  The rounding's rest as a second operand took
//   two maps' forward pass from 66 to 80 us (2 x 8 heads of 64 / 128, 2048 causal), their single-token case from 21.7 to 22.9.
// attn_step_kernel: few queries (at most 32 rows of all the heads that share a key / value head): these rows are one tile, the
//   keys are split over the grid and over the 4 waves, each with a private LDS tile and no barrier in the loop; the parts are
//   joined in LDS and, where the grid splits, by attn_join_kernel.
//   16 x 1 tokens against 37 MB of ragged caches: 13 us, of which a call of one tile takes 6.4 to 7 (launch, lengths, a tile's latency,
//   the join in LDS), and 4 for the parts' join.
#include "attn_common.h"

// One wave's 32 query rows: fragments, running statistics, the accumulated O^T.
template <int TY, int MAPS, int DQ, int DV, bool BIAS> struct FwdWave {
  typedef typename El<TY>::T T;
  typedef typename El<TY>::Frag Frag;
  typedef Tile<TY, DQ> TK;
  typedef Tile<TY, DV> TV;
  Frag q[MAPS][DQ / 16];
  f32x16 o[MAPS][DV / 32];
  float m[MAPS], l[MAPS];      // running reference (log2 units) and this lane half's part of the sum
  int limit, low;              // last key this lane's query sees; the least of the wave's
  int pos, pmin, pmax;         // the lane's position; the wave's first and last
  const float* tab;            // BIAS: this lane's head's table, at rel = 0
  float far_l, far_r;          // its values left and right of ``reach``
  bool fold;                   // both may be folded into the exponent
  bool large;                  // some value of the table is BIAS_LARGE or more
  float c2;                    // scale in log2 units
  bool both;                   // DQ = 32: the second 16 of the head's elements are not all padding

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      m[p] = -INFINITY;
      l[p] = 0.0f;
#pragma unroll
      for (int d = 0; d < DV / 32; ++d) o[p][d] = zero16();
    }
  }

  __device__ __forceinline__ void load_q(const AttnArgs& a, const T* row, bool ok, int half) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p)
#pragma unroll
      for (int s = 0; s < DQ / 16; ++s) {
        const int d = 16 * s + 8 * half;
        q[p][s] = global_frag<TY>(row + (MAPS == 2 ? p * a.sq[3] : 0) + d, ok && d < a.D);
      }
  }

  // Scores of NK keys -> weights, in place; returns by how much the accumulators shrink.  cc, add: what is left to apply to them.
  template <int NS> __device__ __forceinline__ float weights(f32x16 (&s)[NS], int p, float cc, float add, bool& grown) {
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
    mx = fmaf(half_max(mx), cc, add);
    // the reference follows the maximum only where that has grown by more than 2^8: weights stay below 2^8, far inside every
    // type's range, and most tiles leave the accumulators alone
    grown = mx > m[p] + 8.0f;
    const float mn = grown ? mx : m[p];
    const float al = grown ? exp2_(m[p] - mn) : 1.0f;
    m[p] = mn;
    const float sub = add - (mn == -INFINITY ? 0.0f : mn);
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = exp2_(fmaf(s[u][r], cc, sub));
        part[r & 3] += s[u][r];
      }
    l[p] = fmaf(l[p], al, (part[0] + part[1]) + (part[2] + part[3]));
    return al;
  }

  // NK keys from j0 on, which are rows k0 ... of the LDS tiles (maps ``mapb`` bytes apart)
  template <int NK> __device__ __forceinline__ void step(const char* kt, int mapb, const char* vt, int k0, int j0, int reach, int lane) {
    constexpr int NS = NK / 32;
    const int li = lane & 31, half = lane >> 5;
    const bool masked = low < j0 + NK - 1;
    const bool left = BIAS && j0 + NK - 1 - pmin <= -reach, right = BIAS && j0 - pmax >= reach;
    // folded: the bias is one value, which goes into the exponent; plain: every query sees every key, too
    const bool folded = BIAS && fold && (left || right), plain = !masked && (!BIAS || folded);
    Frag pf[MAPS][NK / 16];
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      f32x16 s[NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        s[u] = zero16();
#pragma unroll
        for (int k = 0; k < DQ / 16; ++k)
          if (DQ > 32 || k == 0 || both) s[u] = El<TY>::mma(TK::read_rows(kt + p * mapb, k0 + 32 * u + li, k, half), q[p][k], s[u]);
      }
      float al;
      bool grown;
      const int last = masked ? limit - j0 - 4 * half : NK;
      if (plain || folded) {
        if (masked) {
          const int to = another(last);
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + 8 * (r >> 2) + (r & 3) <= to ? s[u][r] : -INFINITY;
        }
        al = weights<NS>(s, p, c2, !BIAS ? 0.0f : left ? far_l : far_r, grown);
      } else {
        const bool near = BIAS && !left && !right;
        const float* t = tab + (j0 + 4 * half - pos);
        const float far = left ? far_l : far_r, cf = !BIAS || fabsf(far) < BIAS_FOLD ? c2 : 0.0f;
        float add = 0.0f;
        if (near && large) {
          int to = another(last);
          add = -INFINITY;                             // the largest bias that this row sees in the tile
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int c = 32 * u + 8 * (r >> 2) + (r & 3);
              add = fmaxf(add, c <= to ? t[c] : -INFINITY);
            }
          add = half_max(add);
          add = fabsf(add) < BIAS_FOLD ? add : 0.0f;
          to = another(to);
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int c = 32 * u + 8 * (r >> 2) + (r & 3);
              const float x = fmaf(s[u][r], fabsf(t[c]) < BIAS_FOLD ? c2 : 0.0f, t[c] - add);
              s[u][r] = c <= to ? x : -INFINITY;
            }
        } else {
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int c = 32 * u + 8 * (r >> 2) + (r & 3);
              float x = s[u][r] * c2;
              if (BIAS) x = fmaf(s[u][r], near ? c2 : cf, near ? t[c] : far);
              s[u][r] = c <= last ? x : -INFINITY;
            }
        }
        al = weights<NS>(s, p, 1.0f, add, grown);
      }
      if (__any(grown)) {
#pragma unroll
        for (int d = 0; d < DV / 32; ++d) o[p][d] *= al;
      }
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x8 e;
#pragma unroll
          for (int r = 0; r < 8; ++r) e[r] = s[u][8 * t + r];
          pf[p][2 * u + t] = El<TY>::frag(e);
        }
    }
#pragma unroll
    for (int t = 0; t < NK / 16; ++t)
#pragma unroll
      for (int d = 0; d < DV / 32; ++d) {
        const Frag vf = TV::read_cols(vt, k0 + 16 * t, d, lane);
#pragma unroll
        for (int p = 0; p < MAPS; ++p) o[p][d] = El<TY>::mma(vf, pf[p][t], o[p][d]);
      }
  }
};

// The work-group's place: b, key / value head, query head and query block.  Heads that share K and V run on one XCD where the head
// count allows it (work-groups b and b + 8 share one).  Without a causal mask an XCD takes one head after the other; under one the
// longest rows of all heads come first (2 x 8 heads, 2048 tokens, two maps: 65 us, head by head 74; 16 heads, 8192 tokens, back to back:
// 364, 374).
struct FwdPlace { int b, h, blk; bool ok; };
__device__ __forceinline__ FwdPlace fwd_place(const AttnArgs& a, int nblk) {
  FwdPlace w;
  const int G = a.H / a.Hkv, kvh = a.B * a.Hkv, heads = a.B * a.H;
  int bh = blockIdx.x % heads, blk = blockIdx.x / heads;
  w.ok = true;
  if (a.causal) {
    blk = nblk - 1 - blk;
    if (kvh % 8 == 0) {
      const int i = bh >> 3, kv = i / G * 8 + (bh & 7);
      bh = kv * G + i % G;
    }
  } else if (kvh % 8 == 0) {
    int o, i;
    xcd_remap(blockIdx.x, nblk * G, o, i);
    bh = o * G + i % G;
    blk = i / G;
    w.ok = o < kvh;
  } else if (heads % 8 == 0) {
    xcd_remap(blockIdx.x, nblk, bh, blk);
    w.ok = bh < heads;
  }
  w.b = bh / a.H;
  w.h = bh % a.H;
  w.blk = blk;
  return w;
}

// RW: waves by rows (4, or 2 with two waves a row, see row_waves)
template <int TY, int RW> struct KeyTile { static constexpr int KT = TY == TY_F32 && RW == 4 ? 32 : 64; };   // keys staged at a time

template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW>
__global__ __launch_bounds__(256, TY == TY_F32 && MAPS * DQ + DV > 128 ? 1 : 2) void attn_fwd_kernel(AttnArgs a, int nblk) {
  typedef typename El<TY>::T T;
  constexpr int KT = KeyTile<TY, RW>::KT, NK = RW == 2 || TY == TY_F32 || (MAPS == 2 && DV > 64) ? 32 : 64;   // keys at a time
  constexpr int MB = KT * DQ * (int)sizeof(T), KB = MAPS * MB, VB = KT * DV * (int)sizeof(T);
  extern __shared__ __align__(16) char smem[];       // 2 x (K maps, V), then the bias table
  float* tab = reinterpret_cast<float*>(smem + 2 * (KB + VB));       // nothing reads it when the epilogue lies over it
  __shared__ int large[4];
  const FwdPlace w = fwd_place(a, nblk);
  if (!w.ok) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int b = w.b, h = w.h, hk = h / (a.H / a.Hkv);
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int blk0 = w.blk * 32 * RW, part = RW == 2 ? wave >> 1 : 0;          // rows; which half of each tile's keys
  if (blk0 >= nq) return;
  const int row0 = blk0 + (RW == 2 ? wave & 1 : wave) * 32, row = row0 + li;
  const int last_row = min(blk0 + 32 * RW - 1, nq - 1);
  const int seen = a.causal ? min(nk, max(st + last_row + 1, 0)) : nk;      // keys any row of this block sees
  const int nt = (seen + KT - 1) / KT;

  const T* kp = (const T*)a.k + b * a.sk[0] + hk * a.sk[2];
  const T* vp = (const T*)a.v + b * a.sv[0] + hk * a.sv[2];
  Dma<TY, DQ, KT, 256> kd;
  Dma<TY, DV, KT, 256> vd;
  kd.init(a.sk[1], a.D, tid);
  vd.init(a.sv[1], a.Dv, tid);
  auto fetch = [&](int j0, int buf) {
    char* base = smem + buf * (KB + VB);
#pragma unroll
    for (int p = 0; p < MAPS; ++p) kd.issue(kp + (MAPS == 2 ? p * a.sk[3] : 0) + j0 * a.sk[1], seen - j0, base + p * MB, wave);
    vd.issue(vp + j0 * a.sv[1], seen - j0, base + KB, wave);
  };
  if (nt > 0) fetch(0, 0);

  FwdWave<TY, MAPS, DQ, DV, BIAS> wv;
  wv.init();
  wv.load_q(a, (const T*)a.q + b * a.sq[0] + row * a.sq[1] + h * a.sq[2], row < nq, half);
  wv.pos = st + row;
  wv.pmin = st + row0;
  wv.pmax = st + row0 + 31;
  wv.limit = min(nk - 1, a.causal ? wv.pos : nk - 1);                // rows behind the last query: computed, not stored
  wv.low = min(nk - 1, a.causal ? wv.pmin : nk - 1);
  wv.c2 = a.scale * LOG2E;
  wv.both = a.D > 16;
  if constexpr (BIAS) {
    const bool l = __any(fill_bias<TY>(a, tab, h, tid, 256));
    if (lane == 0) large[wave] = l;
    wv.tab = tab + a.reach + BIAS_PAD;
    wv.far_l = bias_log2<TY>(a, -a.reach, h);
    wv.far_r = bias_log2<TY>(a, a.reach, h);
    wv.fold = fabsf(wv.far_l) < BIAS_FOLD && fabsf(wv.far_r) < BIAS_FOLD;
  }
  const int wave_last = row0 >= nq ? -1 : a.causal ? min(seen - 1, st + min(row0 + 31, nq - 1)) : seen - 1;

  dma_wait<0>();
  __syncthreads();
  if constexpr (BIAS) wv.large = large[0] | large[1] | large[2] | large[3];
  for (int t = 0; t < nt; ++t) {
    const char* kt = smem + (t & 1) * (KB + VB);
    if (t + 1 < nt) fetch((t + 1) * KT, (t & 1) ^ 1);
#pragma unroll
    for (int u = 0; u < KT / NK; ++u)
      if ((RW == 4 || u == part) && t * KT + u * NK <= wave_last) wv.template step<NK>(kt, MB, kt + KB, u * NK, t * KT + u * NK, a.reach, lane);
    dma_wait<0>();
    __syncthreads();
  }

  if constexpr (RW == 2) {
    // the second half's state, register by register, over the tiles: every wave is past its last read
    float* x = reinterpret_cast<float*>(smem) + (wave & 1) * 64 + lane;
    if (part == 1) {
#pragma unroll
      for (int p = 0; p < MAPS; ++p) {
        float* y = x + p * (DV / 2 + 2) * 128;
        y[0] = wv.m[p];
        y[128] = wv.l[p];
#pragma unroll
        for (int d = 0; d < DV / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) y[(2 + 16 * d + r) * 128] = wv.o[p][d][r];
      }
    }
    __syncthreads();
    if (part == 0)
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      const float* y = x + p * (DV / 2 + 2) * 128;
      const float m2 = y[0], mm = fmaxf(wv.m[p], m2);
      const float w1 = wv.m[p] == -INFINITY ? 0.0f : exp2_(wv.m[p] - mm), w2 = m2 == -INFINITY ? 0.0f : exp2_(m2 - mm);
      wv.m[p] = mm;
      wv.l[p] = fmaf(wv.l[p], w1, y[128] * w2);
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) wv.o[p][d][r] = fmaf(wv.o[p][d][r], w1, y[(2 + 16 * d + r) * 128] * w2);
    }
  }
  float lam = 0.0f;
  if constexpr (MAPS == 2) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  float inv[MAPS];
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    const float l = half_sum(wv.l[p]);
    inv[p] = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.stats && row < nq && half == 0 && part == 0) {
      // log2 of the sum beside its reference; a row that sees nothing gets weights of zero in the backward pass
      float* s = a.stats + 2 * ((((long)p * a.B + b) * a.H + h) * a.Lq + row);
      s[0] = l == 0.0f ? 0.0f : wv.m[p];
      s[1] = l == 0.0f ? INFINITY : log2f(l);
    }
  }
  typedef RowStore<TY, DV> Out;
  char* piece = smem + wave * Out::BYTES;
  if constexpr (RW == 2) {
    __syncthreads();                                                 // past the join's reads
    if (part == 1) return;
  }
#pragma unroll
  for (int d = 0; d < DV / 32; ++d) {
    wv.o[0][d] *= inv[0];
    if constexpr (MAPS == 2) {
      wv.o[1][d] *= inv[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) wv.o[0][d][r] = fmaf(-lam, wv.o[1][d][r], wv.o[0][d][r]);
    }
  }
  Out::store(wv.o[0], 1.0f, piece, (T*)a.out + b * a.so[0] + row0 * a.so[1] + h * a.so[2], a.so[1], nq - row0, a.Dv, lane);
  if constexpr (MAPS == 2)
    if (a.out2) Out::store(wv.o[1], 1.0f, piece, (T*)a.out2 + (((long)b * a.Lq + row0) * a.H + h) * a.Dv, (long)a.H * a.Dv, nq - row0, a.Dv, lane);
}

// ---- few queries ---------------------------------------------------------------------------------
// Rows r = i G + g of one (b, key / value head): query i, head hk G + g; R = Lq G <= 32.  ``splits`` work-groups share the
// keys; part s of them leaves per map and row {m, l, O[0..DV)} in ws[((s B + b) Hkv + hk) ...], joined by attn_join_kernel.
template <int TY, int MAPS, int DQ, int DV> struct StepTile {
  static constexpr int SZ = sizeof(typename El<TY>::T), MB = 32 * DQ * SZ, KB = MAPS * MB, VB = 32 * DV * SZ;
  static constexpr int BUFS = 8 * (KB + VB) <= 128 * 1024 ? 2 : 1;     // private tiles of a wave: the next is fetched over the present
  static constexpr int REC = DV + 4;                                   // a row's part: O, m, l (padded to 16 bytes)
  static constexpr int LDS = 4 * BUFS * (KB + VB), JOIN = 4 * 32 * REC * 4;
};

template <int TY, int MAPS, int DQ, int DV, bool BIAS>
__global__ __launch_bounds__(256) void attn_step_kernel(AttnArgs a, int splits) {
  typedef typename El<TY>::T T;
  typedef StepTile<TY, MAPS, DQ, DV> L;
  constexpr int KT = 32, REC = L::REC;
  extern __shared__ __align__(16) char smem[];         // 4 waves x BUFS x (K maps, V) | bias tables of the G heads
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int bh = blockIdx.x / splits, sp = blockIdx.x % splits, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int G = a.H / a.Hkv, R = a.Lq * G;
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int row = li, i = row / G, g = row % G, h = hk * G + (row < R ? g : 0);
  const bool ok = row < R && i < nq;
  char* mine = smem + wave * L::BUFS * (L::KB + L::VB);
  float* tabs = reinterpret_cast<float*>(smem + L::LDS);
  __shared__ int large[4];

  // each part ends where the next begins
  const int seen = a.causal ? min(nk, max(st + nq, 0)) : nk;
  const int per = ((seen + splits - 1) / splits + 127) / 128 * 128;      // keys per part: whole rounds of the 4 waves
  const int k0 = min(sp * per, seen), k1 = min(k0 + per, seen);
  const T* kp = (const T*)a.k + b * a.sk[0] + hk * a.sk[2];
  const T* vp = (const T*)a.v + b * a.sv[0] + hk * a.sv[2];
  Dma<TY, DQ, KT, 64> kd;
  Dma<TY, DV, KT, 64> vd;
  kd.init(a.sk[1], a.D, lane);
  vd.init(a.sv[1], a.Dv, lane);
  auto fetch = [&](int j0, char* base) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) kd.issue(kp + (MAPS == 2 ? p * a.sk[3] : 0) + j0 * a.sk[1], k1 - j0, base + p * L::MB, 0);
    vd.issue(vp + j0 * a.sv[1], k1 - j0, base + L::KB, 0);
  };
  constexpr int LOADS = MAPS * Dma<TY, DQ, KT, 64>::N + Dma<TY, DV, KT, 64>::N;
  int j0 = k0 + wave * KT;
  if (j0 < k1) fetch(j0, mine);

  FwdWave<TY, MAPS, DQ, DV, BIAS> wv;
  wv.init();
  wv.load_q(a, (const T*)a.q + b * a.sq[0] + (ok ? i : 0) * a.sq[1] + h * a.sq[2], ok, half);
  wv.pos = st + (ok ? i : 0);
  wv.pmin = st;
  wv.pmax = st + a.Lq - 1;
  wv.limit = min(k1 - 1, a.causal ? wv.pos : k1 - 1);
  wv.low = min(k1 - 1, a.causal ? wv.pmin : k1 - 1);
  wv.c2 = a.scale * LOG2E;
  wv.both = a.D > 16;
  if constexpr (BIAS) {
    // the tables are read by tiles within ``reach`` of the queries only (whole tiles: the last one begins at k1 - 1 at the latest and has
    // KT keys, seen or not): most parts of a long cache have none
    const int n = bias_size(a.reach);
    bool l = false;
    if (k1 - 1 + KT - 1 - wv.pmin > -a.reach && k0 - wv.pmax < a.reach)
      for (int x = 0; x < G; ++x) l |= fill_bias<TY>(a, tabs + x * n, hk * G + x, tid, 256);
    l = __any(l);
    if (lane == 0) large[wave] = l;
    wv.tab = tabs + (row < R ? g : 0) * n + a.reach + BIAS_PAD;
    wv.far_l = bias_log2<TY>(a, -a.reach, h);
    wv.far_r = bias_log2<TY>(a, a.reach, h);
    wv.fold = !__any(fabsf(wv.far_l) >= BIAS_FOLD || fabsf(wv.far_r) >= BIAS_FOLD);
    __syncthreads();
    wv.large = large[0] | large[1] | large[2] | large[3];
  }
  for (int buf = 0; j0 < k1; j0 += 4 * KT) {
    const char* now = mine + buf * (L::KB + L::VB);
    const int nx = j0 + 4 * KT;
    if (L::BUFS == 2 && nx < k1) {
      buf ^= 1;
      fetch(nx, mine + buf * (L::KB + L::VB));
      dma_wait<LOADS>();
    } else {
      dma_wait<0>();
    }
    wv.template step<KT>(now, L::MB, now + L::KB, 0, j0, a.reach, lane);
    if (L::BUFS == 1 && nx < k1) {
      __builtin_amdgcn_s_waitcnt(0xc07f);              // this wave's reads of the tile are done
      fetch(nx, mine);
    }
  }

  // join the 4 waves: their parts in LDS, over the tiles (every wave is past its last read)
  float lam = 0.0f;
  if (MAPS == 2 && splits == 1) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  __syncthreads();
  float* rec = reinterpret_cast<float*>(smem);         // [wave][32 rows][REC]
  float accs[MAPS][DV / 8];                            // thread (row, eighth of DV): columns DV / 8 * eighth + ...
  float mt[MAPS], lt[MAPS];
  const int jr = tid >> 3, je = tid & 7;
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    const float l = half_sum(wv.l[p]);
    float* d0 = rec + (wave * 32 + li) * REC;
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = wv.o[p][d][4 * q4 + r];
        *reinterpret_cast<f32x4*>(d0 + 32 * d + 8 * q4 + 4 * half) = x;
      }
    if (half == 0) {
      d0[DV] = wv.m[p];
      d0[DV + 1] = l;
    }
    __syncthreads();
    float mm = -INFINITY;
#pragma unroll
    for (int v = 0; v < 4; ++v) mm = fmaxf(mm, rec[(v * 32 + jr) * REC + DV]);
    mt[p] = mm;
    lt[p] = 0.0f;
#pragma unroll
    for (int c = 0; c < DV / 8; ++c) accs[p][c] = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float* s = rec + (v * 32 + jr) * REC;
      const float wgt = s[DV] == -INFINITY ? 0.0f : exp2_(s[DV] - mm);
      lt[p] = fmaf(wgt, s[DV + 1], lt[p]);
#pragma unroll
      for (int c = 0; c < DV / 8; ++c) accs[p][c] = fmaf(wgt, s[je * (DV / 8) + c], accs[p][c]);
    }
    __syncthreads();
  }
  if (jr >= R) return;
  const int qi = jr / G, qh = hk * G + jr % G;
  if (splits > 1) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      float* d0 = a.ws + ((((long)sp * a.B * a.Hkv + bh) * MAPS + p) * R + jr) * REC;
#pragma unroll
      for (int c = 0; c < DV / 8; c += 4) {
        f32x4 x = {accs[p][c], accs[p][c + 1], accs[p][c + 2], accs[p][c + 3]};
        *reinterpret_cast<f32x4*>(d0 + je * (DV / 8) + c) = x;
      }
      if (je == 0) {
        d0[DV] = mt[p];
        d0[DV + 1] = lt[p];
      }
    }
    return;
  }
  if (qi >= nq) return;
  float inv[MAPS];
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    inv[p] = lt[p] == 0.0f ? 0.0f : 1.0f / lt[p];
    if (a.stats && je == 0) {
      float* s = a.stats + 2 * ((((long)p * a.B + b) * a.H + qh) * a.Lq + qi);
      s[0] = lt[p] == 0.0f ? 0.0f : mt[p];
      s[1] = lt[p] == 0.0f ? INFINITY : log2f(lt[p]);
    }
  }
  T* op = (T*)a.out + b * a.so[0] + qi * a.so[1] + qh * a.so[2];
  T* o2 = (MAPS == 2 && a.out2) ? (T*)a.out2 + (((long)b * a.Lq + qi) * a.H + qh) * a.Dv : nullptr;
#pragma unroll
  for (int c = 0; c < DV / 8; c += 4) {
    const int col = je * (DV / 8) + c;
    if (col >= a.Dv) continue;
    f32x4 x, y;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = accs[0][c + r] * inv[0];
      if constexpr (MAPS == 2) {
        y[r] = accs[1][c + r] * inv[1];
        x[r] = fmaf(-lam, y[r], x[r]);
      }
    }
    El<TY>::store4(op + col, x);
    if (MAPS == 2 && o2) El<TY>::store4(o2 + col, y);
  }
}

// A wave a row: the parts' weights from their maxima (a lane a part, at most 64), then the columns, 16 bytes a lane, the lane groups
// sharing the parts.
template <int TY, int MAPS, int DV>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int splits, int rows) {
  typedef typename El<TY>::T T;
  constexpr int REC = DV + 4, C = DV / 4, S = 64 / C;  // 16-byte columns of a row; lane groups
  const int at = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (at >= rows) return;
  const int G = a.H / a.Hkv, R = a.Lq * G;
  const int bh = at / R, jr = at % R, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int qi = jr / G, qh = hk * G + jr % G;
  if (qi >= clamp_len(a.q_len, b, a.Lq)) return;
  float lam = 0.0f;
  if constexpr (MAPS == 2) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  const int col = 4 * (lane % C), grp = lane / C;
  const float* base = a.ws + ((long)bh * MAPS * R + jr) * REC;
  const long step = (long)a.B * a.Hkv * MAPS * R * REC, map = (long)R * REC;
  constexpr int AHEAD = 8;                             // parts a lane fetches before it knows their weights
  f32x4 y[MAPS], first[MAPS][AHEAD];
  float m[MAPS], l[MAPS];
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    m[p] = lane < splits ? base[p * map + lane * step + DV] : -INFINITY;
    l[p] = lane < splits ? base[p * map + lane * step + DV + 1] : 0.0f;
  }
#pragma unroll
  for (int p = 0; p < MAPS; ++p)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) first[p][i] = *reinterpret_cast<const f32x4*>(base + p * map + min(i * S + grp, splits - 1) * step + col);
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    float mm = m[p];
#pragma unroll
    for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    const float w = m[p] == -INFINITY ? 0.0f : exp2_(m[p] - mm);
    const float lt = wave_sum(w * l[p]);
    f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float ws = __shfl(w, (i * S + grp) & 63);
      if (i * S + grp < splits) t += ws * first[p][i];
    }
    for (int s0 = AHEAD * S; s0 < splits; s0 += S) {
      const float ws = __shfl(w, (s0 + grp) & 63);
      if (s0 + grp < splits) t += ws * *reinterpret_cast<const f32x4*>(base + p * map + (s0 + grp) * step + col);
    }
#pragma unroll
    for (int d = C; d < 64; d <<= 1)
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] += __shfl_xor(t[r], d);
    y[p] = t * (lt == 0.0f ? 0.0f : 1.0f / lt);
    if (a.stats && lane == 0) {
      float* s = a.stats + 2 * ((((long)p * a.B + b) * a.H + qh) * a.Lq + qi);
      s[0] = lt == 0.0f ? 0.0f : mm;
      s[1] = lt == 0.0f ? INFINITY : log2f(lt);
    }
  }
  f32x4 x = y[0];
  if constexpr (MAPS == 2) {
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = fmaf(-lam, y[1][r], x[r]);
  }
  if (grp || col >= a.Dv) return;
  El<TY>::store4((T*)a.out + b * a.so[0] + qi * a.so[1] + qh * a.so[2] + col, x);
  if (MAPS == 2 && a.out2) El<TY>::store4((T*)a.out2 + (((long)b * a.Lq + qi) * a.H + qh) * a.Dv + col, y[MAPS - 1]);
}

// ---- host ----------------------------------------------------------------------------------------
static inline int pad_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// At most 32 rows of the heads that share a key / value head, and their bias tables within LDS.
static bool is_step(const AttnArgs* a, bool bias) {
  const int G = a->H / a->Hkv;
  return (long)a->Lq * G <= 32 && (!bias || (long)G * (2 * (a->reach + BIAS_PAD) + 1) * 4 <= 16 * 1024);
}
// Parts of at least 256 keys, and no more work-groups than the chip holds at a time (``resident`` a compute unit): a second round
// would pay each work-group's start (lengths, first tile: ~4 us) again.
static int step_splits(const AttnArgs* a, int resident) {
  const long groups = (long)a->B * a->Hkv, most = (a->Lk + 255) / 256;
  long s = (256 * resident + groups - 1) / groups;
  if (s > most) s = most;
  return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}
template <typename L> static int step_lds(const AttnArgs* a, int tab) {
  const int lds = L::LDS + a->H / a->Hkv * tab;
  return lds > L::JOIN ? lds : L::JOIN;
}
template <typename L> static int step_resident(const AttnArgs* a, int tab) {
  const int n = 160 * 1024 / step_lds<L>(a, tab);
  return n < 1 ? 1 : n > 4 ? 4 : n;
}

template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW> static int launch_rows(const AttnArgs* a, int tab, hipStream_t stream) {
  constexpr int STAGE = 2 * KeyTile<TY, RW>::KT * (MAPS * DQ + DV) * (int)sizeof(typename El<TY>::T), JOIN = MAPS * (DV / 2 + 2) * 128 * 4;
  constexpr int OUT = 4 * RowStore<TY, DV>::BYTES, A = RW == 2 && JOIN > STAGE ? JOIN : STAGE;
  const int lds = (OUT > A ? OUT : A) + tab, nblk = cdiv(a->Lq, 32 * RW);
  if (int e = allow_lds<attn_fwd_kernel<TY, MAPS, DQ, DV, BIAS, RW>>(lds)) return e;
  hipLaunchKernelGGL((attn_fwd_kernel<TY, MAPS, DQ, DV, BIAS, RW>), dim3(a->B * a->H * nblk), dim3(256), lds, stream, *a, nblk);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
template <int TY, int MAPS, int DQ, int DV, bool BIAS>
static int launch_fwd(const AttnArgs* a, hipStream_t stream) {
  const int tab = BIAS ? (2 * (a->reach + BIAS_PAD) + 1) * 4 : 0;
  if (is_step(a, BIAS)) {
    typedef StepTile<TY, MAPS, DQ, DV> L;
    const int splits = step_splits(a, step_resident<L>(a, tab)), G = a->H / a->Hkv;
    const long rows = (long)a->B * a->Hkv * MAPS * a->Lq * G;
    if (splits > 1 && (!a->ws || (uintptr_t)a->ws % 16 || a->ws_floats < splits * rows * (DV + 4))) return SGTA_EBADARG;
    const int lds = step_lds<L>(a, tab);
    if (int e = allow_lds<attn_step_kernel<TY, MAPS, DQ, DV, BIAS>>(lds)) return e;
    hipLaunchKernelGGL((attn_step_kernel<TY, MAPS, DQ, DV, BIAS>), dim3(a->B * a->Hkv * splits), dim3(256), lds, stream, *a, splits);
    SGTA_LAUNCH_CHECK();
    if (splits > 1) {
      const int rows1 = a->B * a->H * a->Lq;
      hipLaunchKernelGGL((attn_join_kernel<TY, MAPS, DV>), dim3(cdiv(rows1, 4)), dim3(256), 0, stream, *a, splits, rows1);
      SGTA_LAUNCH_CHECK();
    }
    return SGTA_OK;
  }
  const long groups = (long)a->B * a->H * cdiv(a->Lq, 128);
  return row_waves(a->q_len || a->kv_len ? groups / 2 : groups) == 2 ? launch_rows<TY, MAPS, DQ, DV, BIAS, 2>(a, tab, stream)
                                                              : launch_rows<TY, MAPS, DQ, DV, BIAS, 4>(a, tab, stream);
}

// what both directions refuse
int attn_check(const AttnArgs* a, int maps) {
  if (!a || !a->q || !a->k || !a->v || !a->w || !a->out) return SGTA_EBADARG;
  if (a->dtype < 0 || a->dtype > 2 || a->B < 1 || a->Lq < 1 || a->Lk < 1 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv) return SGTA_EBADARG;
  if (a->D < 8 || a->D % 8 || a->Dv < 8 || a->Dv % 8 || !(a->scale >= 0.99e-36f) || !(a->scale <= 1.01e36f)) return SGTA_EBADARG;
  if (maps == 1 ? (a->D > 128 || a->Dv != a->D) : (a->D > 64 || a->Dv > 128)) return SGTA_EBADARG;
  if (a->Lq >= 1 << 29 || a->Lk >= 1 << 29 || (long)a->B * a->H * cdiv(a->Lq > a->Lk ? a->Lq : a->Lk, 128) >= MAX_GROUPS) return SGTA_ETOOBIG;
  if (maps == 1 && (!a->lut || a->reach < 1 || a->reach > 1024 || a->num_buckets < 1)) return SGTA_EBADARG;
  const int al = a->dtype == TY_F32 ? 4 : 8;           // strides and pointers: whole 16-byte pieces
  const long* s[] = {a->sq, a->sk, a->sv, a->so};
  const void* p[] = {a->q, a->k, a->v, a->out};
  for (int i = 0; i < 3; ++i)
    if (s[i][1] > MAX_PITCH / (a->dtype == TY_F32 ? 4 : 2) || s[i][1] < 0) return SGTA_ETOOBIG;
  if (maps == 2 && (uintptr_t)a->out2 % 16) return SGTA_EBADARG;
  for (int i = 0; i < 4; ++i) {
    if ((uintptr_t)p[i] % 16) return SGTA_EBADARG;
    for (int j = 0; j < (i < 2 && maps == 2 ? 4 : 3); ++j)
      if (s[i][j] % al) return SGTA_EBADARG;
  }
  return SGTA_OK;
}

// the variant for a call's types and sizes: launches it, or (ws) says how many floats of workspace it takes
template <int TY, int MAPS, int DQ, int DV, bool BIAS> static int variant(const AttnArgs* a, hipStream_t st, long* ws) {
  if (!ws) return launch_fwd<TY, MAPS, DQ, DV, BIAS>(a, st);
  *ws = 0;
  if (is_step(a, BIAS)) {
    const int s = step_splits(a, step_resident<StepTile<TY, MAPS, DQ, DV>>(a, BIAS ? bias_size(a->reach) * 4 : 0));
    if (s > 1) *ws = (long)s * a->B * a->H * MAPS * a->Lq * (DV + 4);
  }
  return SGTA_OK;
}
template <int TY> static int typed(const AttnArgs* a, int maps, hipStream_t st, long* ws) {
  if (maps == 2) return a->D <= 32 && a->Dv <= 64 ? variant<TY, 2, 32, 64, false>(a, st, ws) : variant<TY, 2, 64, 128, false>(a, st, ws);
  switch (pad_dim(a->D)) {
    case 32: return variant<TY, 1, 32, 32, true>(a, st, ws);
    case 64: return variant<TY, 1, 64, 64, true>(a, st, ws);
    default: return variant<TY, 1, 128, 128, true>(a, st, ws);
  }
}
static int forward(const AttnArgs* a, int maps, hipStream_t st, long* ws) {
  if (int e = attn_check(a, maps)) return e;
  return a->dtype == TY_F32 ? typed<TY_F32>(a, maps, st, ws) : a->dtype == TY_F16 ? typed<TY_F16>(a, maps, st, ws) : typed<TY_BF16>(a, maps, st, ws);
}

extern "C" long sgta_attn_fwd_ws_floats(const sgta_attn_t* a, int maps) {
  long n = 0;
  return (maps == 1 || maps == 2) && forward(a, maps, nullptr, &n) == SGTA_OK ? n : 0;
}
extern "C" int sgta_rel_attn_fwd(const sgta_attn_t* a, sgta_stream_t stream) { return forward(a, 1, (hipStream_t)stream, nullptr); }
extern "C" int sgta_diff_attn_fwd(const sgta_attn_t* a, sgta_stream_t stream) { return forward(a, 2, (hipStream_t)stream, nullptr); }
