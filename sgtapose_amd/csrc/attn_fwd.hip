// Attention forward on gfx950: one softmax map with a learned relative position bias by buckets, or two maps whose difference
// is taken with a learned weight.
//   one map:   o_i = sum_j softmax_j( scale q_i.k_j + table[bucket(j - p_i), h] ) v_j            p_i = q_start + i
//   two maps:  o_i = sum_j ( softmax_j(scale q1_i.k1_j) - lambda softmax_j(scale q2_i.k2_j) ) v_j
// One pass over the keys with running maximum and sum; a score never leaves its wave.
//
// attn_fwd_kernel: 4 waves of 32 queries share 64-key tiles of K and V in LDS (double buffered, the next tile's global loads
//   in flight over the present one's products).  S^T = K Q^T puts the query on the lane: row statistics are in-lane but for
//   one lane-half exchange, and the weights are the next product's operand as they stand: O^T += V^T P^T.
// attn_step_kernel: few queries (at most 32 rows of all the heads that share a key / value head): these rows are one tile, the
//   keys are split over the grid and over the 4 waves, each with a private LDS tile and no barrier in the loop; the parts are
//   joined in LDS and, where the grid splits, by attn_join_kernel.
#include "attn_common.h"

// One wave's 32 query rows: fragments, running statistics, the accumulated O^T.
template <int TY, int MAPS, int DQ, int DV, bool BIAS, int KT> struct FwdWave {
  typedef typename El<TY>::T T;
  typedef typename El<TY>::Frag Frag;
  static constexpr int NS = KT / 32;
  Frag q[MAPS][DQ / 16];
  f32x16 o[MAPS][DV / 32];
  float m[MAPS], l[MAPS];      // running reference (log2 units) and this lane half's part of the sum
  int limit;                   // last key this lane's query sees (-1: none)
  int pos, pmin, pmax;         // the lane's position; the wave's first and last
  const float* tab;            // BIAS: this lane's head's table, at rel = 0
  float far_l, far_r;          // its values left and right of ``reach``
  bool fold;                   // both may be folded into the exponent

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      m[p] = -INFINITY;
      l[p] = 0.0f;
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[p][d][r] = 0.0f;
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

  // keys [j0, j0 + KT) from LDS; rows of kt beyond the last key are zero
  __device__ __forceinline__ void tile(const char* kt, const char* vt, int j0, int reach, float c2, int lane) {
    typedef Tile<TY, DQ> TK;
    typedef Tile<TY, DV> TV;
    const int li = lane & 31, half = lane >> 5;
    const bool masked = __any(limit < j0 + KT - 1);
    Frag pf[MAPS][KT / 16];
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      f32x16 s[NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < DQ / 16; ++k)
          s[u] = El<TY>::mma(TK::read_rows(kt + p * KT * TK::ROWB, 32 * u + li, k, half), q[p][k], s[u]);
      }
      float cc = c2, add = 0.0f;
      if constexpr (BIAS) {
        const bool left = j0 + KT - 1 - pmin <= -reach, right = j0 - pmax >= reach;
        if (fold && (left || right)) {
          add = left ? far_l : far_r;
        } else if (left || right) {
          const float b = left ? far_l : far_r;
          cc = 1.0f;
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], c2, b);
        } else {
          const float* t = tab + (j0 + 4 * half - pos);
          cc = 1.0f;
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], c2, t[32 * u + 8 * (r >> 2) + (r & 3)]);
        }
      }
      if (masked) {
        const int last = limit - j0 - 4 * half;
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + 8 * (r >> 2) + (r & 3) <= last ? s[u][r] : -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
      mx = fmaf(half_max(mx), cc, add);
      // the reference follows the maximum only where that has grown by more than 2^8: weights stay below 2^8, far inside
      // every type's range, and most tiles leave the accumulators alone
      if (__any(mx > m[p] + 8.0f)) {
        const float mn = fmaxf(m[p], mx);
        const float al = mn == -INFINITY ? 1.0f : exp2_(m[p] - mn);
        m[p] = mn;
        l[p] *= al;
#pragma unroll
        for (int d = 0; d < DV / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[p][d][r] *= al;
      }
      const float sub = add - (m[p] == -INFINITY ? 0.0f : m[p]);
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x8 e;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            e[r] = exp2_(fmaf(s[u][8 * t + r], cc, sub));
            part[r & 3] += e[r];
          }
          pf[p][2 * u + t] = El<TY>::frag(e);
        }
      l[p] += (part[0] + part[1]) + (part[2] + part[3]);
    }
#pragma unroll
    for (int t = 0; t < KT / 16; ++t)
#pragma unroll
      for (int d = 0; d < DV / 32; ++d) {
        const Frag vf = TV::read_cols(vt, 16 * t, d, lane);
#pragma unroll
        for (int p = 0; p < MAPS; ++p) o[p][d] = El<TY>::mma(vf, pf[p][t], o[p][d]);
      }
  }
};

// The work-group's place: b, key / value head, query head and query block.  Blocks that share K and V run on one XCD where
// the head count allows it (blocks b and b + 8 share one); under a causal mask the longest rows come first.
struct FwdPlace { int b, h, blk; bool ok; };
__device__ __forceinline__ FwdPlace fwd_place(const AttnArgs& a, int nblk) {
  FwdPlace w;
  const int G = a.H / a.Hkv, kvh = a.B * a.Hkv;
  int bh, blk;
  if (kvh % 8 == 0) {
    int o, i;
    xcd_remap(blockIdx.x, nblk * G, o, i);
    bh = (o / a.Hkv) * a.H + (o % a.Hkv) * G + i % G;
    blk = i / G;
    w.ok = o < kvh;
  } else if (a.B * a.H % 8 == 0) {
    xcd_remap(blockIdx.x, nblk, bh, blk);
    w.ok = bh < a.B * a.H;
  } else {
    bh = blockIdx.x % (a.B * a.H);
    blk = blockIdx.x / (a.B * a.H);
    w.ok = true;
  }
  w.b = bh / a.H;
  w.h = bh % a.H;
  w.blk = a.causal ? nblk - 1 - blk : blk;
  return w;
}

template <int TY, int MAPS, int DQ, int DV, bool BIAS>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnArgs a, int nblk) {
  typedef typename El<TY>::T T;
  constexpr int KT = TY == TY_F32 ? 32 : 64;
  typedef Tile<TY, DQ> TK;
  typedef Tile<TY, DV> TV;
  constexpr int KB = MAPS * KT * TK::ROWB, VB = KT * TV::ROWB;
  extern __shared__ __align__(16) char smem[];       // 2 x (K maps, V), then the bias table
  float* tab = reinterpret_cast<float*>(smem + 2 * (KB + VB));
  const FwdPlace w = fwd_place(a, nblk);
  if (!w.ok) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int b = w.b, h = w.h, hk = h / (a.H / a.Hkv);
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int blk0 = w.blk * 128;
  if (blk0 >= nq) return;
  const int row0 = blk0 + wave * 32, row = row0 + li;

  FwdWave<TY, MAPS, DQ, DV, BIAS, KT> wv;
  wv.init();
  wv.load_q(a, (const T*)a.q + b * a.sq[0] + row * a.sq[1] + h * a.sq[2], row < nq, half);
  wv.pos = st + row;
  wv.pmin = st + row0;
  wv.pmax = st + row0 + 31;
  wv.limit = row < nq ? min(nk - 1, a.causal ? wv.pos : nk - 1) : -1;
  if constexpr (BIAS) {
    fill_bias<TY>(a, tab, h, tid, 256);
    wv.tab = tab + a.reach + BIAS_PAD;
    wv.far_l = bias_log2<TY>(a, -a.reach, h);
    wv.far_r = bias_log2<TY>(a, a.reach, h);
    wv.fold = fabsf(wv.far_l) < BIAS_FOLD && fabsf(wv.far_r) < BIAS_FOLD;
  }
  const float c2 = a.scale * LOG2E;
  const int last_row = min(blk0 + 127, nq - 1);
  const int seen = a.causal ? min(nk, max(st + last_row + 1, 0)) : nk;      // keys any row of this block sees
  const int nt = (seen + KT - 1) / KT;
  const int wave_last = a.causal ? min(seen - 1, st + min(row0 + 31, nq - 1)) : seen - 1;
  const bool active = row0 < nq;

  const T* kp = (const T*)a.k + b * a.sk[0] + hk * a.sk[2];
  const T* vp = (const T*)a.v + b * a.sv[0] + hk * a.sv[2];
  Stage<TY, DQ, KT, 256> ks[MAPS];
  Stage<TY, DV, KT, 256> vs;
  auto fetch = [&](int j0) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) ks[p].load(kp + (MAPS == 2 ? p * a.sk[3] : 0), a.sk[1], j0, seen, a.D, tid);
    vs.load(vp, a.sv[1], j0, seen, a.Dv, tid);
  };
  auto put = [&](int buf) {
    char* base = smem + buf * (KB + VB);
#pragma unroll
    for (int p = 0; p < MAPS; ++p) ks[p].store(base + p * KT * TK::ROWB, tid);
    vs.store(base + KB, tid);
  };
  if (nt > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int cur = t & 1;
    if (t + 1 < nt) fetch((t + 1) * KT);
    if (active && t * KT <= wave_last) wv.tile(smem + cur * (KB + VB), smem + cur * (KB + VB) + KB, t * KT, a.reach, c2, lane);
    if (t + 1 < nt) put(cur ^ 1);
    __syncthreads();
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
    if (a.stats && row < nq && half == 0) {
      // log2 of the sum beside its reference; a row that sees nothing gets weights of zero in the backward pass
      float* s = a.stats + 2 * ((((long)p * a.B + b) * a.H + h) * a.Lq + row);
      s[0] = l == 0.0f ? 0.0f : wv.m[p];
      s[1] = l == 0.0f ? INFINITY : log2f(l);
    }
  }
  if (row < nq) {
    T* op = (T*)a.out + b * a.so[0] + row * a.so[1] + h * a.so[2];
    T* o2 = (MAPS == 2 && a.out2) ? (T*)a.out2 + (((long)b * a.Lq + row) * a.H + h) * a.Dv : nullptr;
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = 32 * d + 8 * g + 4 * half;
        if (col >= a.Dv) continue;
        f32x4 x, y;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = wv.o[0][d][4 * g + r] * inv[0];
          if constexpr (MAPS == 2) {
            y[r] = wv.o[1][d][4 * g + r] * inv[1];
            x[r] = fmaf(-lam, y[r], x[r]);
          }
        }
        El<TY>::store4(op + col, x);
        if (MAPS == 2 && o2) El<TY>::store4(o2 + col, y);
      }
  }
}

// ---- few queries ---------------------------------------------------------------------------------
// Rows r = i G + g of one (b, key / value head): query i, head hk G + g; R = Lq G <= 32.  ``splits`` work-groups share the
// keys; part s of them leaves per map and row {m, l, O[0..DV)} in ws[((s B + b) Hkv + hk) ...], joined by attn_join_kernel.
template <int TY, int MAPS, int DQ, int DV, bool BIAS>
__global__ __launch_bounds__(256) void attn_step_kernel(AttnArgs a, int splits) {
  typedef typename El<TY>::T T;
  constexpr int KT = 32;
  typedef Tile<TY, DQ> TK;
  typedef Tile<TY, DV> TV;
  constexpr int KB = MAPS * KT * TK::ROWB, VB = KT * TV::ROWB;
  constexpr int REC = DV + 4;                          // a row's part: O, m, l (padded to 16 bytes)
  extern __shared__ __align__(16) char smem[];         // 4 x (K maps, V) private tiles | bias tables of the G heads
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int bh = blockIdx.x / splits, sp = blockIdx.x % splits, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int G = a.H / a.Hkv, R = a.Lq * G;
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int row = li, i = row / G, g = row % G, h = hk * G + (row < R ? g : 0);
  const bool ok = row < R && i < nq;
  char* mine = smem + wave * (KB + VB);
  float* tabs = reinterpret_cast<float*>(smem + 4 * (KB + VB));

  FwdWave<TY, MAPS, DQ, DV, BIAS, KT> wv;
  wv.init();
  wv.load_q(a, (const T*)a.q + b * a.sq[0] + (ok ? i : 0) * a.sq[1] + h * a.sq[2], ok, half);
  wv.pos = st + (ok ? i : 0);
  wv.pmin = st;
  wv.pmax = st + a.Lq - 1;
  const int seen = a.causal ? min(nk, max(st + nq, 0)) : nk;
  wv.limit = ok ? min(seen - 1, a.causal ? wv.pos : seen - 1) : -1;
  if constexpr (BIAS) {
    const int n = bias_size(a.reach);
    for (int t = tid; t < n * G; t += 256) tabs[t] = bias_log2<TY>(a, t % n - a.reach - BIAS_PAD, hk * G + t / n);
    wv.tab = tabs + (row < R ? g : 0) * n + a.reach + BIAS_PAD;
    wv.far_l = bias_log2<TY>(a, -a.reach, h);
    wv.far_r = bias_log2<TY>(a, a.reach, h);
    wv.fold = !__any(fabsf(wv.far_l) >= BIAS_FOLD || fabsf(wv.far_r) >= BIAS_FOLD);
    __syncthreads();
  }
  const float c2 = a.scale * LOG2E;
  const int per = ((seen + splits - 1) / splits + 127) / 128 * 128;      // keys per part: whole rounds of the 4 waves
  const int k0 = min(sp * per, seen), k1 = min(k0 + per, seen);

  const T* kp = (const T*)a.k + b * a.sk[0] + hk * a.sk[2];
  const T* vp = (const T*)a.v + b * a.sv[0] + hk * a.sv[2];
  Stage<TY, DQ, KT, 64> ks[MAPS];
  Stage<TY, DV, KT, 64> vs;
  auto fetch = [&](int j0) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) ks[p].load(kp + (MAPS == 2 ? p * a.sk[3] : 0), a.sk[1], j0, k1, a.D, lane);
    vs.load(vp, a.sv[1], j0, k1, a.Dv, lane);
  };
  // each part ends where the next begins: its rows' limit goes no further
  wv.limit = min(wv.limit, k1 - 1);
  int j0 = k0 + wave * KT;
  if (j0 < k1) fetch(j0);
  for (; j0 < k1; j0 += 4 * KT) {
#pragma unroll
    for (int p = 0; p < MAPS; ++p) ks[p].store(mine + p * KT * TK::ROWB, lane);
    vs.store(mine + KB, lane);
    if (j0 + 4 * KT < k1) fetch(j0 + 4 * KT);
    wv.tile(mine, mine + KB, j0, a.reach, c2, lane);
  }

  // join the 4 waves: their parts in LDS, over the tiles (every wave is past its last read)
  float lam = 0.0f;
  if constexpr (MAPS == 2) {
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

// One wave a row: the parts' weights from their maxima, then the columns.
template <int TY, int MAPS, int DV>
__global__ __launch_bounds__(64) void attn_join_kernel(AttnArgs a, int splits) {
  typedef typename El<TY>::T T;
  constexpr int REC = DV + 4;
  const int G = a.H / a.Hkv, R = a.Lq * G;
  const int bh = blockIdx.x / R, jr = blockIdx.x % R, b = bh / a.Hkv, hk = bh % a.Hkv, lane = threadIdx.x;
  const int qi = jr / G, qh = hk * G + jr % G;
  if (qi >= clamp_len(a.q_len, b, a.Lq)) return;
  constexpr int C = DV > 64 ? 2 : 1;                   // columns lane, lane + 64
  float y[MAPS][C];
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    const float* base = a.ws + (((long)bh * MAPS + p) * R + jr) * REC;
    const long step = (long)a.B * a.Hkv * MAPS * R * REC;
    float mm = -INFINITY, lt = 0.0f;
    for (int s = lane; s < splits; s += 64) mm = fmaxf(mm, base[s * step + DV]);
#pragma unroll
    for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
#pragma unroll
    for (int c = 0; c < C; ++c) y[p][c] = 0.0f;
    for (int s = 0; s < splits; ++s) {
      const float* r = base + s * step;
      const float wgt = r[DV] == -INFINITY ? 0.0f : exp2_(r[DV] - mm);
      lt = fmaf(wgt, r[DV + 1], lt);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (lane + 64 * c < DV) y[p][c] = fmaf(wgt, r[lane + 64 * c], y[p][c]);
    }
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
    for (int c = 0; c < C; ++c) y[p][c] *= inv;
    if (a.stats && lane == 0) {
      float* s = a.stats + 2 * ((((long)p * a.B + b) * a.H + qh) * a.Lq + qi);
      s[0] = lt == 0.0f ? 0.0f : mm;
      s[1] = lt == 0.0f ? INFINITY : log2f(lt);
    }
  }
  float lam = 0.0f;
  if constexpr (MAPS == 2) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  T* op = (T*)a.out + b * a.so[0] + qi * a.so[1] + qh * a.so[2];
  T* o2 = (MAPS == 2 && a.out2) ? (T*)a.out2 + (((long)b * a.Lq + qi) * a.H + qh) * a.Dv : nullptr;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = lane + 64 * c;
    if (col >= a.Dv) continue;
    El<TY>::store(op + col, MAPS == 2 ? fmaf(-lam, y[MAPS - 1][c], y[0][c]) : y[0][c]);
    if (MAPS == 2 && o2) El<TY>::store(o2 + col, y[MAPS - 1][c]);
  }
}

// ---- host ----------------------------------------------------------------------------------------
static inline int pad_dim(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// At most 32 rows of the heads that share a key / value head, and their bias tables within LDS.
static bool is_step(const AttnArgs* a, bool bias) {
  const int G = a->H / a->Hkv;
  return (long)a->Lq * G <= 32 && (!bias || (long)G * (2 * (a->reach + BIAS_PAD) + 1) * 4 <= 16 * 1024);
}
// parts of at least 256 keys, no more than fill the chip four times
static int step_splits(const AttnArgs* a) {
  const long groups = (long)a->B * a->Hkv;
  long s = (1024 + groups - 1) / groups, most = (a->Lk + 255) / 256;
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}

template <int TY, int MAPS, int DQ, int DV, bool BIAS>
static int launch_fwd(const AttnArgs* a, hipStream_t stream) {
  constexpr int SZ = sizeof(typename El<TY>::T);
  const int tab = BIAS ? (2 * (a->reach + BIAS_PAD) + 1) * 4 : 0;
  if (is_step(a, BIAS)) {
    const int splits = step_splits(a), G = a->H / a->Hkv;
    const long rows = (long)a->B * a->Hkv * MAPS * a->Lq * G;
    if (splits > 1 && (!a->ws || a->ws_floats < splits * rows * (DV + 4))) return SGTA_EBADARG;
    int lds = 4 * 32 * (MAPS * DQ + DV) * SZ + G * tab;
    const int join = 4 * 32 * (DV + 4) * 4;
    if (lds < join) lds = join;
    if (int e = allow_lds<attn_step_kernel<TY, MAPS, DQ, DV, BIAS>>(lds)) return e;
    hipLaunchKernelGGL((attn_step_kernel<TY, MAPS, DQ, DV, BIAS>), dim3(a->B * a->Hkv * splits), dim3(256), lds, stream, *a, splits);
    SGTA_LAUNCH_CHECK();
    if (splits > 1) {
      hipLaunchKernelGGL((attn_join_kernel<TY, MAPS, DV>), dim3(a->B * a->Hkv * a->Lq * G), dim3(64), 0, stream, *a, splits);
      SGTA_LAUNCH_CHECK();
    }
    return SGTA_OK;
  }
  constexpr int KT = TY == TY_F32 ? 32 : 64;
  const int lds = 2 * KT * (MAPS * DQ + DV) * SZ + tab;
  const int nblk = cdiv(a->Lq, 128);
  if (int e = allow_lds<attn_fwd_kernel<TY, MAPS, DQ, DV, BIAS>>(lds)) return e;
  hipLaunchKernelGGL((attn_fwd_kernel<TY, MAPS, DQ, DV, BIAS>), dim3(a->B * a->H * nblk), dim3(256), lds, stream, *a, nblk);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}

// what both directions refuse
int attn_check(const AttnArgs* a, int maps) {
  if (!a || !a->q || !a->k || !a->v || !a->w || !a->out) return SGTA_EBADARG;
  if (a->dtype < 0 || a->dtype > 2 || a->B < 1 || a->Lq < 1 || a->Lk < 1 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv) return SGTA_EBADARG;
  if (a->D < 8 || a->D % 8 || a->Dv < 8 || a->Dv % 8 || !(a->scale > 0.0f) || !(a->scale < INFINITY)) return SGTA_EBADARG;
  if (maps == 1 ? (a->D > 128 || a->Dv != a->D) : (a->D > 64 || a->Dv > 128)) return SGTA_EBADARG;
  if (a->Lq >= 1 << 29 || a->Lk >= 1 << 29 || (long)a->B * a->H * cdiv(a->Lq > a->Lk ? a->Lq : a->Lk, 32) >= 1L << 31) return SGTA_ETOOBIG;
  if (maps == 1 && (!a->lut || a->reach < 1 || a->reach > 1024 || a->num_buckets < 1)) return SGTA_EBADARG;
  const int al = a->dtype == TY_F32 ? 4 : 8;           // strides and pointers: whole 16-byte pieces
  const long* s[] = {a->sq, a->sk, a->sv, a->so};
  const void* p[] = {a->q, a->k, a->v, a->out};
  for (int i = 0; i < 4; ++i) {
    if ((uintptr_t)p[i] % 16) return SGTA_EBADARG;
    for (int j = 0; j < (i < 2 && maps == 2 ? 4 : 3); ++j)
      if (s[i][j] % al) return SGTA_EBADARG;
  }
  return SGTA_OK;
}

extern "C" long sgta_attn_fwd_ws_floats(const sgta_attn_t* a, int maps) {
  if ((maps != 1 && maps != 2) || attn_check(a, maps)) return 0;
  if (!is_step(a, maps == 1)) return 0;
  const int s = step_splits(a);
  const int dv = maps == 1 ? pad_dim(a->Dv) : (a->D <= 32 && a->Dv <= 64 ? 64 : 128);
  return s > 1 ? (long)s * a->B * a->H * maps * a->Lq * (dv + 4) : 0;
}

template <int TY> static int rel_fwd(const AttnArgs* a, hipStream_t st) {
  switch (pad_dim(a->D)) {
    case 32: return launch_fwd<TY, 1, 32, 32, true>(a, st);
    case 64: return launch_fwd<TY, 1, 64, 64, true>(a, st);
    default: return launch_fwd<TY, 1, 128, 128, true>(a, st);
  }
}
template <int TY> static int diff_fwd(const AttnArgs* a, hipStream_t st) {
  return a->D <= 32 && a->Dv <= 64 ? launch_fwd<TY, 2, 32, 64, false>(a, st) : launch_fwd<TY, 2, 64, 128, false>(a, st);
}

extern "C" int sgta_rel_attn_fwd(const sgta_attn_t* a, sgta_stream_t stream) {
  if (int e = attn_check(a, 1)) return e;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == TY_F32 ? rel_fwd<TY_F32>(a, st) : a->dtype == TY_F16 ? rel_fwd<TY_F16>(a, st) : rel_fwd<TY_BF16>(a, st);
}
extern "C" int sgta_diff_attn_fwd(const sgta_attn_t* a, sgta_stream_t stream) {
  if (int e = attn_check(a, 2)) return e;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == TY_F32 ? diff_fwd<TY_F32>(a, st) : a->dtype == TY_F16 ? diff_fwd<TY_F16>(a, st) : diff_fwd<TY_BF16>(a, st);
}
