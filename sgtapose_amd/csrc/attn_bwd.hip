// Gradients of the attention in attn_fwd.hip, from the saved row statistics (reference m and log2 of the sum, so that
// P = exp2((s - m) - log2 sum) needs no second softmax):
//   X = dO V^T, delta = rowsum(dO o O), dS = P o (X - delta), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO,
//   dtable[b, h] = sum of dS over the pairs in bucket b.
// Two maps share X:  dS1 = P1 o (X - d1), dS2 = -lambda P2 o (X - d2), d_p = rowsum(dO o O_p), dV = (P1 - lambda P2)^T dO,
//   dlambda = - sum of d2.
//
// Held in fewer bits than f32, in 16-bit calls: P and dS, rounded to the element type as operands of the products that give dV, dQ and dK
// (all of which sum in f32), and delta, from the rounded output (mended below).  dQ, dK and dV of bfloat16 are 2.4e-3 off, 1.7e-3 by
// their own rounding alone; a second operand for the rest would add a product to each of the three.
//
// No atomics and no Lq x Lk array: every sum has one owner and a fixed order.
//   attn_dq_kernel   a wave owns 32 queries and walks the keys: delta, dQ, the table's gradient by distance
//                    (4 x 16 heads of 64, 2048 tokens, bfloat16: 165 us, vector pipe 55 % of the cycles, matrix 30, LDS 30)
//   attn_dkv_kernel  a wave owns 32 keys and walks the queries of all heads that share them: dK, dV
//                    (the same: 187 us, matrix 35, vector 37, LDS 37; heads beyond 64: one work-group on a CU, by registers)
//   *_dw_kernel      sums the work-groups' parts of the learned weights' gradient
// The price is that scores and X are computed twice (7 products instead of 5); what it buys is that gradients are the same from
// run to run and that dQ (f32, Lq x D a head and key block) is never read back.
//
// IEEE half: dS is rounded to half as the operand of the next product.  Gradients arrive at any magnitude, so it is first scaled
// by a power of two that brings the largest |dO| of the row (dQ) or of all queries of the shared heads (dK) next to one.  Values of some
// thousand could then still take it past the half range, though every operand and result is a half: they take the scale down with them
// (attn_vmax_kernel finds the largest).
#include "attn_common.h"

#define DIAG 768               // floats of a wave's 16 x 32 tile in rows of 47, with 15 zeros in front

int attn_check(const AttnArgs* a, int maps);

__device__ __forceinline__ float pow2_to_one(float top) {          // 2^-exponent(top), 1 for zero and for what is not finite
  const int e = (__float_as_uint(top) >> 23) & 255;
  return (e == 0 || e == 255) ? 1.0f : __uint_as_float((unsigned)(min(max(254 - e, 1), 254)) << 23);
}

#define VMAX_KEYS 128          // keys of a part at least
// the workspace, in floats
struct BwdWork {
  long delta, part, top;       // [maps][B][H][Lq]; per (b, h, query block): sums by bucket, or of d2; largest |dO|, and sum of a row's
  long vmax;                   // IEEE half: largest |v| of each part of (b, key / value head)'s keys
  long total;
  int nv;                      // parts
  int rw, nblk, nsum, nrel;    // attn_dq_kernel's waves by rows and query blocks; floats of a part; distances told apart
  __host__ __device__ BwdWork(const AttnArgs& a, int maps) {
    // (float heads beyond 64: the tiles of two halves leave no room for four waves' sums by distance of a wide table)
    rw = maps == 1 && a.dtype == TY_F32 && a.D > 64 && a.reach > 256 ? 4 : row_waves((long)a.B * a.H * ((a.Lq + 127) / 128));
    nblk = (a.Lq + 32 * rw - 1) / (32 * rw);
    nrel = 2 * (a.reach + BIAS_PAD) + 1;
    nsum = maps == 1 ? a.num_buckets : 2;                            // two maps: a sum in 64 bits, as a float and what it leaves
    const long blocks = (long)a.B * a.H * nblk;
    delta = 0;
    part = (long)maps * a.B * a.H * a.Lq;
    top = part + blocks * nsum;
    vmax = top + 2 * blocks;
    nv = a.dtype == TY_F16 ? (a.Lk + VMAX_KEYS - 1) / VMAX_KEYS : 0;
    nv = nv > 64 ? 64 : nv;
    total = vmax + (long)a.B * a.Hkv * nv;
  }
};

// Parts of the keys of a (b, key / value head): their largest |v|, infinities and not-a-numbers aside.  A launch and one read of v: 4 to 7 us
// of 77 (32 x 8 heads of 16, 343 tokens, forward and backward) to 424 (4 x 16 heads of 64, 2048).  Looking for the largest dS in the
// walks, or walking again where a sum is not finite, took 17 to 20 us there, in registers stored.
__global__ __launch_bounds__(256) void attn_vmax_kernel(AttnArgs a, BwdWork wk) {
  typedef El<TY_F16>::T T;
  __shared__ float red[4];
  const int bh = blockIdx.x / wk.nv, part = blockIdx.x % wk.nv, b = bh / a.Hkv, tid = threadIdx.x, per = a.Dv / 8;
  const int nk = clamp_len(a.kv_len, b, a.Lk), keys = (nk + wk.nv - 1) / wk.nv, j0 = min(part * keys, nk), n = min(keys, nk - j0);
  const T* p = (const T*)a.v + b * a.sv[0] + (long)j0 * a.sv[1] + bh % a.Hkv * a.sv[2];
  float top = 0.0f;
#pragma unroll 8
  for (long i = tid; i < (long)n * per; i += 256) {
    const El<TY_F16>::Raw v = *reinterpret_cast<const El<TY_F16>::Raw*>(p + i / per * a.sv[1] + i % per * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = fabsf((float)v[e]);
      top = fmaxf(top, x < INFINITY ? x : 0.0f);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  if (tid == 0) a.ws[wk.vmax + blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
// X_ij - delta_i = sum_k P_ik (X_ij - X_ik), so |P_ij (X_ij - delta_i)| is at most P (1 - P) 2 max|X| <= sum|dO| max|v| / 2, with lambda for
// the second map: the power of two that keeps that, for a row's sum ``l1`` already scaled, below 60000 of a half's 65504
__device__ __forceinline__ float value_scale(const AttnArgs& a, const BwdWork& wk, int b, int hk, float lam, float l1) {
  const int lane = threadIdx.x & 63;
  float top = lane < wk.nv ? a.ws[wk.vmax + (long)(b * a.Hkv + hk) * wk.nv + lane] : 0.0f;
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float most = top * fmaxf(fabsf(lam), 1.0f) * l1 * (0.5f / 60000.0f);
  return most > 1.0f ? 0.5f * pow2_to_one(most) : 1.0f;
}
// LDS of attn_dq_kernel before the bias table: two stages of keys, or what lies over them at the end
template <int TY, int MAPS, int DQ, int DV, int RW> struct DqLds {
  static constexpr int KT = TY == TY_F32 && RW == 4 ? 32 : 64, STAGE = 2 * KT * (MAPS * DQ + DV) * (int)sizeof(typename El<TY>::T);
  static constexpr int JOIN = RW == 2 ? MAPS * (DQ / 2 + 2) * 128 * 4 : 0, OUT = 4 * RowStore<TY, DQ>::BYTES;
  static constexpr int ALL = OUT > STAGE ? OUT : STAGE;
  static_assert(JOIN <= STAGE, "the halves' sums lie over the tiles");
};
// Work-groups on a CU that the registers are held to.  float heads of 32: three, at the price of a few registers stored outside the
// loop (32 x 8 heads, 343 tokens: 52 us where two take 67); 16-bit heads up to 64: three (4 x 16 heads, 2048 tokens: 165 us, two 188).
// Two for float heads of 64 (11 registers stored where two waves share rows) and float two-map heads of 32: there 38 are, 14 of them read
// back in the loop, and 15 in the form for large grids (2 x 777 tokens, 8 heads: 68 us, most of it one wave's latency).
constexpr int dq_groups(int ty, int maps, int dq, int dv) {
  return ty == TY_F32 ? (dq * maps + dv > 128 ? 1 : maps > 1 || dq > 32 ? 2 : 3) : maps > 1 || dq > 64 ? 2 : dq > 32 ? 3 : 4;
}
template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW>
__global__ __launch_bounds__(256, dq_groups(TY, MAPS, DQ, DV)) void attn_dq_kernel(AttnArgs a) {
  typedef typename El<TY>::T T;
  typedef typename El<TY>::Frag Frag;
  constexpr int KT = DqLds<TY, MAPS, DQ, DV, RW>::KT;
  // float, two maps: lambda's gradient is a sum of both signs over all rows, which a weight's error of 3e-7 reaches.  The scores' small
  // products have an accumulator of their own, and lg holds 2^-log2 sum, a factor: in the exponent its 10 or so would cost bits (without
  // a bias no exponent of a row that sees nothing is so large that the factor of zero would meet an infinity).  2 x 777 tokens: 69 us
  // where 62 without, the sum over 12432 rows 1e-6 to 5e-6 off where 1.5e-5.
  constexpr bool EXACT = TY == TY_F32 && !BIAS;
  typedef Tile<TY, DQ> TK;
  typedef Tile<TY, DV> TV;
  constexpr int MB = KT * TK::ROWB, KB = MAPS * MB, VB = KT * TV::ROWB;
  extern __shared__ __align__(16) char smem[];       // 2 x (K maps, V) | bias table | 4 waves: sums by distance | 4 waves: DIAG
  const BwdWork wk(a, MAPS);
  float* tab = reinterpret_cast<float*>(smem + DqLds<TY, MAPS, DQ, DV, RW>::ALL);
  __shared__ float red[2][4], mend[MAPS][4][32];
  __shared__ double sums[4];
  const int nblk = wk.nblk, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int bh = blockIdx.x % (a.B * a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hkv);
  const int blk = a.causal ? nblk - 1 - blockIdx.x / (a.B * a.H) : blockIdx.x / (a.B * a.H);
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int blk0 = blk * 32 * RW, half_of = RW == 2 ? wave >> 1 : 0;         // rows; which half of each tile's keys
  float* part = a.ws + wk.part + ((long)bh * nblk + blk) * wk.nsum;
  float* topw = a.ws + wk.top + 2 * ((long)bh * nblk + blk);
  if (blk0 >= nq) {
    for (int i = tid; i < wk.nsum; i += 256) part[i] = 0.0f;
    if (tid == 0) topw[0] = topw[1] = 0.0f;
    return;
  }
  const int row0 = blk0 + (RW == 2 ? wave & 1 : wave) * 32, row = row0 + li;
  const bool ok = row < nq;
  const int last_row = min(blk0 + 32 * RW - 1, nq - 1);
  const int seen = a.causal ? min(nk, max(st + last_row + 1, 0)) : nk;
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

  float lam = 0.0f;
  if constexpr (MAPS == 2) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  // the row's operands, delta and largest |dO|
  Frag q[MAPS][DQ / 16], g[DV / 16];
  float m[MAPS], lg[MAPS], dl[MAPS], top = 0.0f, l1 = 0.0f;
  // float: every other row's X is computed with its sign turned, so that what is left of the cut-off's mean error cancels in sums over
  // rows (lambda's gradient, the table's)
  const float sx = TY == TY_F32 && (li & 1) ? -1.0f : 1.0f;
  {
    const T* qp = (const T*)a.q + b * a.sq[0] + row * a.sq[1] + h * a.sq[2];
#pragma unroll
    for (int p = 0; p < MAPS; ++p)
#pragma unroll
      for (int s = 0; s < DQ / 16; ++s) {
        const int d = 16 * s + 8 * half;
        q[p][s] = global_frag<TY>(qp + (MAPS == 2 ? p * a.sq[3] : 0) + d, ok && d < a.D);
      }
    const T* gp = (const T*)a.dout + b * a.sdo[0] + row * a.sdo[1] + h * a.sdo[2];
    const T* op = (const T*)a.out + b * a.so[0] + row * a.so[1] + h * a.so[2];
    const T* o2 = MAPS == 2 ? (const T*)a.out2 + (((long)b * a.Lq + row) * a.H + h) * a.Dv : op;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int s = 0; s < DV / 16; ++s) {
      const int d = 16 * s + 8 * half;
      const bool in = ok && d < a.Dv;
      const typename El<TY>::Raw gr = global_raw<TY>(gp + d, in), o = global_raw<TY>(op + d, in);
      if constexpr (TY == TY_F32) g[s] = El<TY>::frag_of(gr * sx);
      else g[s] = El<TY>::frag_of(gr);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s1 = fmaf((float)gr[e], (float)o[e], s1);
        top = fmaxf(top, fabsf((float)gr[e]));
        if (TY == TY_F16) l1 += fabsf((float)gr[e]);
      }
      if constexpr (MAPS == 2) {
        const typename El<TY>::Raw y = global_raw<TY>(o2 + d, in);
#pragma unroll
        for (int e = 0; e < 8; ++e) s2 = fmaf((float)gr[e], (float)y[e], s2);
      }
    }
    s1 = half_sum(s1);
    top = half_max(top);
    if (TY == TY_F16) l1 = half_sum(l1);
    if constexpr (MAPS == 2) {
      s2 = half_sum(s2);
      dl[0] = fmaf(lam, s2, s1);
      dl[1] = s2;
    } else {
      dl[0] = s1;
    }
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      const long at = (((long)p * a.B + b) * a.H + h) * a.Lq + row;
      m[p] = ok ? a.stats[2 * at] : 0.0f;
      lg[p] = ok ? a.stats[2 * at + 1] : INFINITY;
      if (EXACT) lg[p] = exp2_(-lg[p]);
    }
    if constexpr (TY == TY_F16) {
      float t = top, u = l1;
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        t = fmaxf(t, __shfl_xor(t, d));
        u = fmaxf(u, __shfl_xor(u, d));
      }
      if (lane == 0) {
        red[0][wave] = t;
        red[1][wave] = u;
      }
      __syncthreads();
      if (tid < 2) topw[tid] = fmaxf(fmaxf(red[tid][0], red[tid][1]), fmaxf(red[tid][2], red[tid][3]));
    }
  }
  float rs = 1.0f;                                    // power of two for dS
  if constexpr (TY == TY_F16) {
    rs = pow2_to_one(top);
    rs *= value_scale(a, wk, b, hk, lam, l1 * rs);
  }
  const float irs = 1.0f / rs;

  const int pos = st + row, pmin = st + row0, pmax = st + row0 + 31;
  const int limit = min(nk - 1, a.causal ? pos : nk - 1), low = min(nk - 1, a.causal ? pmin : nk - 1);
  // by row: sums of dS over all keys; of dS and P over the keys left and right of ``reach``
  float far_l = 0.0f, far_r = 0.0f, sum_l = 0.0f, sum_r = 0.0f, p_l = 0.0f, p_r = 0.0f;
  // sums of P (X - delta) by map, which are zero but for delta's error: it comes from outputs whose weights and values were rounded
  float err[MAPS] = {};
  bool fold = true;
  const float* tb = tab;
  float *hist = nullptr, *diag = nullptr;
  if constexpr (BIAS) {
    fill_bias<TY>(a, tab, h, tid, 256);
    for (int i = tid; i < 4 * (wk.nrel + DIAG); i += 256) tab[wk.nrel + i] = 0.0f;
    far_l = bias_log2<TY>(a, -a.reach, h);
    far_r = bias_log2<TY>(a, a.reach, h);
    fold = fabsf(far_l) < BIAS_FOLD && fabsf(far_r) < BIAS_FOLD;
    tb = tab + a.reach + BIAS_PAD;
    hist = tab + (1 + wave) * wk.nrel + a.reach + BIAS_PAD;         // at distance 0
    diag = tab + 5 * wk.nrel + wave * DIAG + 15;
  }
  const float c2 = a.scale * LOG2E;
  const float c2r = fabsf(m[0]) < BIAS_FOLD ? c2 : 0.0f;             // a bias beyond absorbs its row's scores
  const bool both = a.D > 16;                         // DQ = 32: the second 16 of the head's elements are not all padding
  const int wave_last = row0 >= nq ? -1 : a.causal ? min(seen - 1, st + min(row0 + 31, nq - 1)) : seen - 1;

  f32x16 dq[MAPS][DQ / 32];
#pragma unroll
  for (int p = 0; p < MAPS; ++p)
#pragma unroll
    for (int d = 0; d < DQ / 32; ++d) dq[p][d] = zero16();

  // 32 keys from j0 on, rows 32 u of the tile: what masks and distances make of them
  struct Keys { bool masked, left, right, plain; };
  auto keys_at = [&](int j0) {
    Keys w;
    w.masked = low < j0 + 31;
    w.left = BIAS && j0 + 31 - pmin <= -a.reach;
    w.right = BIAS && j0 - pmax >= a.reach;
    w.plain = !w.masked && (!BIAS || (fold && (w.left || w.right)));
    return w;
  };
  auto products = [&](const char* vt, int u) {                       // X
    Products<TY, true> xsum(zero16());
#pragma unroll
    for (int k = 0; k < DV / 16; ++k)
      if (DV > 32 || k == 0 || both) xsum.add(TV::read_rows(vt, 32 * u + li, k, half), g[k]);
    return xsum.get();
  };
  auto weights = [&](const char* kt, int u, int j0, const Keys& w, int p) {      // P
    Products<TY, EXACT> sum(zero16());
#pragma unroll
    for (int k = 0; k < DQ / 16; ++k)
      if (DQ > 32 || k == 0 || both) sum.add(TK::read_rows(kt + p * MB, 32 * u + li, k, half), q[p][k]);
    f32x16 s = sum.get();
    if (w.plain) {
      const float add = EXACT ? -m[p] : ((BIAS ? (w.left ? far_l : far_r) : 0.0f) - m[p]) - lg[p];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = EXACT ? exp2_(fmaf(s[r], c2, add)) * lg[p] : exp2_(fmaf(s[r], c2, add));
    } else {
      const int last = w.masked ? limit - j0 - 4 * half : 32;
      const bool near = BIAS && !w.left && !w.right;
      const float far = (w.left ? far_l : far_r) - m[p];
      const float* tp = tb + (j0 + 4 * half - pos);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = 8 * (r >> 2) + (r & 3);
        const float e = BIAS ? fmaf(s[r], c2r, near ? tp[c] - m[p] : far) : s[r] * c2 - m[p];
        s[r] = c > last ? 0.0f : EXACT ? exp2_(e) * lg[p] : exp2_(e - lg[p]);
      }
    }
    return s;
  };
  dma_wait<0>();
  __syncthreads();
  if (TY != TY_F32 && nt <= 2) {
    static_assert(TY == TY_F32 || KT == 64, "two tiles of 64 keys: the first still lies in its stage afterwards");
    // Rows that see few keys (the first ones under a causal mask) have large weights, by which delta's error reaches dQ and the table's
    // near buckets: they walk their keys twice, first for that error alone.  (125 causal tokens, bfloat16: dQ 2.8e-3 off without this,
    // 2.4e-3 with; a row of n equal weights carries 1 / sqrt(n) of it, so beyond 128 keys it is lost in the roundings of dS and dQ.)
    for (int t = 0; t < nt; ++t) {
      const char* kt = smem + (t & 1) * (KB + VB);
      if (t + 1 < nt) fetch((t + 1) * KT, 1);
      for (int u = 0; u < KT / 32; ++u) {
        const int j0 = t * KT + 32 * u;
        if (j0 > wave_last || (RW == 2 && u != half_of)) continue;
        const Keys w = keys_at(j0);
        const f32x16 x = products(kt + KB, u);
#pragma unroll
        for (int p = 0; p < MAPS; ++p) {
          const f32x16 s = weights(kt, u, j0, w, p);
#pragma unroll
          for (int r = 0; r < 16; ++r) err[p] = fmaf(s[r], x[r] - dl[p], err[p]);
        }
      }
      dma_wait<0>();
      __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      err[p] = half_sum(err[p]);
      if (half == 0) mend[p][wave][li] = err[p];
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < MAPS; ++p) {
      dl[p] += RW == 2 ? mend[p][wave & 1][li] + mend[p][2 + (wave & 1)][li] : err[p];
      err[p] = 0.0f;
    }
  }
  for (int t = 0; t < nt; ++t) {
    const char* kt = smem + (t & 1) * (KB + VB);
    const char* vt = kt + KB;
    if (t + 1 < nt) fetch((t + 1) * KT, (t & 1) ^ 1);
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      const int j0 = t * KT + 32 * u;
      if (j0 > wave_last || (RW == 2 && u != half_of)) continue;
      const Keys w = keys_at(j0);
      const f32x16 x = products(vt, u);
      Frag df[MAPS][2];
#pragma unroll
      for (int p = 0; p < MAPS; ++p) {
        f32x16 s = weights(kt, u, j0, w, p);
        if constexpr (BIAS) {
          if (w.left || w.right) {
            const float sum = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])) + (((s[8] + s[9]) + (s[10] + s[11])) + ((s[12] + s[13]) + (s[14] + s[15])));
            if (w.left) p_l += sum; else p_r += sum;
          }
        }
        const float sg = (MAPS == 2 && p == 1) ? -lam : 1.0f;
        float tot[2] = {0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float d = s[r] * (TY == TY_F16 ? fmaf(x[r], rs, -dl[p] * rs) : TY == TY_F32 ? fmaf(x[r], sx, -dl[p]) : x[r] - dl[p]);
          s[r] = (MAPS == 2 && p == 1) ? d * sg : d;
          tot[r & 1] += d;
        }
        const float all = (tot[0] + tot[1]) * irs;
        err[p] += all;
        if constexpr (BIAS) {
          if (w.left) sum_l += all;
          else if (w.right) sum_r += all;
          else {
            // Sums by distance, 16 keys at a time: the tile as rows of 32 with 15 zeros between them (row k at 47 k, the zeros stay),
            // where the entries of one distance, k - q, lie 48 apart; lane u < 47 adds up those of distance 15 - u.  (LDS atomics
            // into the sums take two cycles a lane: 16 of them cost 1950 cycles a tile.)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              asm volatile("" ::: "memory");           // a wave's LDS operations are done in order; the compiler keeps it
#pragma unroll
              for (int r = 0; r < 8; ++r) diag[(8 * (r >> 2) + 4 * half + (r & 3)) * 47 + li] = s[8 * hf + r] * irs;
              asm volatile("" ::: "memory");
              float v = 0.0f, w = 0.0f;
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                v += diag[48 * k + min(lane, 46) - 15];
                w += diag[48 * (k + 1) + min(lane, 46) - 15];
              }
              if (lane < 47) hist[j0 + 16 * hf - pmin + 15 - lane] += v + w;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x8 ds;
#pragma unroll
          for (int r = 0; r < 8; ++r) ds[r] = s[8 * k + r];
          df[p][k] = El<TY>::frag(ds);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int p = 0; p < MAPS; ++p)
#pragma unroll
          for (int d = 0; d < DQ / 32; ++d) dq[p][d] = El<TY>::mma(TK::read_cols(kt + p * MB, 32 * u + 16 * k, d, lane), df[p][k], dq[p][d]);
    }
    dma_wait<0>();
    __syncthreads();
  }

#pragma unroll
  for (int p = 0; p < MAPS; ++p) err[p] = half_sum(err[p]);
  if constexpr (RW == 2) {
    // the second half's sums, register by register, over the tiles: every wave is past its last read
    float* y = reinterpret_cast<float*>(smem) + (wave & 1) * 64 + lane;
    float* z = reinterpret_cast<float*>(smem) + MAPS * DQ / 2 * 128 + (wave & 1) * (MAPS * 128) + half_of * 64 + lane;
    if (half_of == 1) {
#pragma unroll
      for (int p = 0; p < MAPS; ++p)
#pragma unroll
        for (int d = 0; d < DQ / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) y[((p * (DQ / 32) + d) * 16 + r) * 128] = dq[p][d][r];
    }
#pragma unroll
    for (int p = 0; p < MAPS; ++p) z[p * 128] = err[p];
    __syncthreads();
    if (half_of == 0) {
#pragma unroll
      for (int p = 0; p < MAPS; ++p)
#pragma unroll
        for (int d = 0; d < DQ / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dq[p][d][r] += y[((p * (DQ / 32) + d) * 16 + r) * 128];
    }
#pragma unroll
    for (int p = 0; p < MAPS; ++p) err[p] += z[p * 128 + (half_of ? -64 : 64)];
  }
  typedef RowStore<TY, DQ> Out;
  if (RW == 2) __syncthreads();                                      // past the join's reads
  if (row0 < nq && half_of == 0) {
    T* o = (T*)a.dq + b * a.sdq[0] + row0 * a.sdq[1] + h * a.sdq[2];
#pragma unroll
    for (int p = 0; p < MAPS; ++p) Out::store(dq[p], a.scale * irs, smem + wave * Out::BYTES, o + (MAPS == 2 ? p * a.sdq[3] : 0), a.sdq[1], nq - row0, a.D, lane);
  }
  // The kernel of dK and dV and the gradient of lambda get delta without its error (bfloat16, 2048 tokens: dK is 2.5e-3 off with it,
  // 2.36e-3 without, of which 1.66e-3 is dK's own rounding; lambda's 4.4e-3 and 1.2e-3).
#pragma unroll
  for (int p = 0; p < MAPS; ++p) {
    dl[p] += err[p];
    if (ok && half == 0 && half_of == 0) a.ws[wk.delta + (((long)p * a.B + b) * a.H + h) * a.Lq + row] = dl[p];
  }
  if constexpr (MAPS == 2) {
    double t2 = half == 0 && half_of == 0 && ok ? (double)dl[1] : 0.0;
#pragma unroll
    for (int d = 32; d; d >>= 1) t2 += __shfl_xor(t2, d);
    if (lane == 0) sums[wave] = t2;
    __syncthreads();
    if (tid == 0) {
      t2 = (sums[0] + sums[1]) + (sums[2] + sums[3]);
      part[0] = (float)t2;
      part[1] = (float)(t2 - (double)part[0]);
    }
  }
  if constexpr (BIAS) {
    // off the far buckets, where P's sum is large, comes the error times that sum
    sum_l = wave_sum(ok ? fmaf(-err[0], p_l, sum_l) : 0.0f);
    sum_r = wave_sum(ok ? fmaf(-err[0], p_r, sum_r) : 0.0f);
    if (lane == 0) {                                  // the ends of the table stand for everything beyond
      tab[(1 + wave) * wk.nrel] += sum_l;
      tab[(2 + wave) * wk.nrel - 1] += sum_r;
    }
    __syncthreads();
    for (int i = tid; i < wk.nrel; i += 256) {
      // over the bias itself, which is no longer needed
      tab[i] = (tab[wk.nrel + i] + tab[2 * wk.nrel + i]) + (tab[3 * wk.nrel + i] + tab[4 * wk.nrel + i]);
    }
    __syncthreads();
    // by bucket: a run of distances each, first and count behind the table of buckets; the outermost reach to the table's ends
    const int* run = a.lut + 2 * a.reach + 1;
    for (int k = tid; k < a.num_buckets; k += 256) {
      int i0 = run[k], i1 = i0 + run[a.num_buckets + k];
      float v = 0.0f;
      if (i1 > i0) {
        i0 = i0 == 0 ? 0 : i0 + BIAS_PAD;
        i1 = i1 == 2 * a.reach + 1 ? wk.nrel : i1 + BIAS_PAD;
        for (int i = i0; i < i1; ++i) v += tab[i];
      }
      part[k] = v;
    }
  }
}

// All 512 registers of a SIMD where heads are large (floats from 64, 16-bit two-map ones of 64 / 128): one work-group on a compute unit.
// Float two-map heads of 64 / 128 still store 21 and read 23 back in the loop, float heads of 128 on large grids 16.
template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW>
__global__ __launch_bounds__(256, (MAPS * DQ + DV > 128 || (TY == TY_F32 && MAPS * DQ + DV > 64)) ? 1 : 2) void attn_dkv_kernel(AttnArgs a, int nblk) {
  typedef typename El<TY>::T T;
  typedef typename El<TY>::Frag Frag;
  constexpr int QT = 64;
  typedef Tile<TY, DQ> TQ;
  typedef Tile<TY, DV> TG;
  constexpr int MB = QT * TQ::ROWB, QB = MAPS * MB, GB = QT * TG::ROWB, SB = 4 * MAPS * QT * 4, ST = QB + GB + SB;
  extern __shared__ __align__(16) char smem[];       // 2 x (Q maps, dO, per map and query: start, -delta, m, lg) | bias table
  const BwdWork wk(a, MAPS);
  float* tab = reinterpret_cast<float*>(smem + 2 * ST);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int bh = blockIdx.x % (a.B * a.Hkv), b = bh / a.Hkv, hk = bh % a.Hkv, blk = blockIdx.x / (a.B * a.Hkv);
  const int G = a.H / a.Hkv;
  const int nq = clamp_len(a.q_len, b, a.Lq), nk = clamp_len(a.kv_len, b, a.Lk), st = start_of(a.q_start, b);
  const int blk0 = blk * 32 * RW, half_of = RW == 2 ? wave >> 1 : 0;         // keys; which half of each tile's queries
  if (blk0 >= nk) return;
  const int key0 = blk0 + (RW == 2 ? wave & 1 : wave) * 32, key = key0 + li;
  const bool ok = key < nk;
  const float c2 = a.scale * LOG2E, ic2 = 1.0f / c2;
  const bool both = a.D > 16;                         // DQ = 32: the second 16 of the head's elements are not all padding
  // under a causal mask the first query that sees key blk0 stands at its position
  const int q_first = a.causal ? min(max(blk0 - st, 0), nq) / QT * QT : 0;
  const int nt = nq > q_first ? (nq - q_first + QT - 1) / QT : 0;
  const int wave_first = key0 >= nk ? 0x7fffffff : a.causal ? key0 - st : -0x7fffffff;    // first query that sees any of this wave's keys

  Dma<TY, DQ, QT, 256> qd;
  Dma<TY, DV, QT, 256> gd;
  qd.init(a.sq[1], a.D, tid);
  gd.init(a.sdo[1], a.Dv, tid);
  float st_m = 0.0f, st_l = 0.0f, st_d = 0.0f;       // thread tid < MAPS QT: one query's statistics
  auto fetch = [&](int h, int r0, int buf) {
    char* base = smem + buf * ST;
    const T* qp = (const T*)a.q + b * a.sq[0] + h * a.sq[2] + r0 * a.sq[1];
#pragma unroll
    for (int p = 0; p < MAPS; ++p) qd.issue(qp + (MAPS == 2 ? p * a.sq[3] : 0), nq - r0, base + p * MB, wave);
    gd.issue((const T*)a.dout + b * a.sdo[0] + h * a.sdo[2] + r0 * a.sdo[1], nq - r0, base + QB, wave);
    if (tid < MAPS * QT) {
      const int p = tid / QT, row = r0 + tid % QT;
      const long at = (((long)p * a.B + b) * a.H + h) * a.Lq + row;
      const bool in = row < nq;                       // a query that is none: weights of exp2(-inf)
      st_m = in ? a.stats[2 * at] : 0.0f;
      st_l = in ? a.stats[2 * at + 1] : INFINITY;
      st_d = in ? a.ws[wk.delta + at] : 0.0f;
    }
  };
  auto put = [&](int buf) {
    if (tid < MAPS * QT) {
      float* d = reinterpret_cast<float*>(smem + buf * ST + QB + GB) + (tid / QT) * 4 * QT + tid % QT;
      d[0] = (-st_m - st_l) * ic2;
      d[QT] = -st_d;
      d[2 * QT] = st_m;
      d[3 * QT] = st_l;
    }
  };
  const int steps = nt * G;
  if (steps > 0) fetch(hk * G, q_first, 0);

  float lam = 0.0f;
  if constexpr (MAPS == 2) {
    float e1, e2;
    lam = diff_lambda<TY>(a, e1, e2);
  }
  Frag kf[MAPS][DQ / 16], vf[DV / 16];
  {
    const T* kp = (const T*)a.k + b * a.sk[0] + key * a.sk[1] + hk * a.sk[2];
    const T* vp = (const T*)a.v + b * a.sv[0] + key * a.sv[1] + hk * a.sv[2];
#pragma unroll
    for (int p = 0; p < MAPS; ++p)
#pragma unroll
      for (int s = 0; s < DQ / 16; ++s) {
        const int d = 16 * s + 8 * half;
        kf[p][s] = global_frag<TY>(kp + (MAPS == 2 ? p * a.sk[3] : 0) + d, ok && d < a.D);
      }
#pragma unroll
    for (int s = 0; s < DV / 16; ++s) {
      const int d = 16 * s + 8 * half;
      vf[s] = global_frag<TY>(vp + d, ok && d < a.Dv);
    }
  }
  float rs = 1.0f;
  if constexpr (TY == TY_F16) {
    float top = 0.0f, l1 = 0.0f;
    for (int i = lane; i < G * wk.nblk; i += 64) {
      const float* t = a.ws + wk.top + 2 * (((long)b * a.H + hk * G) * wk.nblk + i);
      top = fmaxf(top, t[0]);
      l1 = fmaxf(l1, t[1]);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      top = fmaxf(top, __shfl_xor(top, d));
      l1 = fmaxf(l1, __shfl_xor(l1, d));
    }
    rs = pow2_to_one(top);
    rs *= value_scale(a, wk, b, hk, lam, l1 * rs);
  }
  f32x16 dk[MAPS][DQ / 32], dv[DV / 32];
#pragma unroll
  for (int p = 0; p < MAPS; ++p)
#pragma unroll
    for (int d = 0; d < DQ / 32; ++d) dk[p][d] = zero16();
#pragma unroll
  for (int d = 0; d < DV / 32; ++d) dv[d] = zero16();

  float far_l = 0.0f, far_r = 0.0f;
  bool fold = true;                                  // both small enough to be added to a start that -m is already in
  int h = hk * G, r0 = q_first;
  if (steps > 0) put(0);
  for (int it = 0; it < steps; ++it) {
    if (BIAS && r0 == q_first) {
      // a new head: every wave is past its last read of the old one's table, by the barrier at the end of the step before
      fill_bias<TY>(a, tab, h, tid, 256);
      far_l = bias_log2<TY>(a, -a.reach, h);
      far_r = bias_log2<TY>(a, a.reach, h);
      fold = fabsf(far_l) < BIAS_LARGE && fabsf(far_r) < BIAS_LARGE;
    }
    if (it == 0) dma_wait<0>();
    if (it == 0 || (BIAS && r0 == q_first)) __syncthreads();
    const char* qt = smem + (it & 1) * ST;
    const char* gt = qt + QB;
    const float* stat = reinterpret_cast<const float*>(gt + GB);
    int hn = h, rn = r0 + QT;
    if (rn >= nq) {
      hn = h + 1;
      rn = q_first;
    }
    if (it + 1 < steps) fetch(hn, rn, (it & 1) ^ 1);
#pragma unroll 1
    for (int u = 0; u < QT / 32; ++u) {
      const int q0 = r0 + 32 * u;
      if (q0 + 31 < wave_first || q0 >= nq || (RW == 2 && u != half_of)) continue;
      const bool diag = a.causal && q0 < key0 + 31 - st;             // some pair of the tile is masked
      const bool left = BIAS && key0 + 31 - (st + q0) <= -a.reach, right = BIAS && key0 - (st + q0 + 31) >= a.reach;
      const bool plain = !diag && (!BIAS || (fold && (left || right)));
      // register row 8 c + 4 half + r, c = 0..3: its statistics in four 16-byte pieces, the same for all lanes of a half
      auto rows16 = [&](int p, int what) {
        f32x16 v;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(stat + (4 * p + what) * QT + 32 * u + 8 * c + 4 * half);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[4 * c + r] = t[r];
        }
        return v;
      };
      Products<TY> xsum(rows16(0, 1));                               // X - delta: the sum starts from -delta
#pragma unroll
      for (int k = 0; k < DV / 16; ++k)
        if (DV > 32 || k == 0 || both) xsum.add(TG::read_rows(gt, 32 * u + li, k, half), vf[k]);
      f32x16 x = xsum.get(), w0;
      Frag dsf[MAPS][2];
#pragma unroll
      for (int p = 0; p < MAPS; ++p) {
        // and the exponent from (-m - lg) / c2
        Products<TY> ssum(plain ? rows16(p, 0) : zero16());
#pragma unroll
        for (int k = 0; k < DQ / 16; ++k)
          if (DQ > 32 || k == 0 || both) ssum.add(TQ::read_rows(qt + p * MB, 32 * u + li, k, half), kf[p][k]);
        f32x16 s = ssum.get();
        if (plain) {
          const float far = !BIAS ? 0.0f : left ? far_l : far_r;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = exp2_(BIAS ? fmaf(s[r], c2, far) : s[r] * c2);
        } else {
          const int first = diag ? key - st - q0 - 4 * half : -64;   // register rows from here on see this lane's key
          const float* tp = tab + a.reach + BIAS_PAD + (key - st - q0 - 4 * half);
          const bool near = BIAS && !left && !right;
          const float far = left ? far_l : far_r;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float* sp = stat + 4 * p * QT + 32 * u + 8 * c + 4 * half;
            const f32x4 mm = *reinterpret_cast<const f32x4*>(sp + 2 * QT), ll = *reinterpret_cast<const f32x4*>(sp + 3 * QT);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // a bias beyond BIAS_FOLD absorbs its row's scores
              const float e = BIAS ? fmaf(s[4 * c + r], fabsf(mm[r]) < BIAS_FOLD ? c2 : 0.0f, (near ? tp[-(8 * c + r)] : far) - mm[r]) : s[4 * c + r] * c2 - mm[r];
              s[4 * c + r] = 8 * c + r >= first ? exp2_(e - ll[r]) : 0.0f;
            }
          }
        }
        if (MAPS == 2 && p == 1) {
          // the second map weighs -lambda, and its delta is its own
          const f32x16 d0 = rows16(0, 1), d1 = rows16(1, 1);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] *= -lam;
            w0[r] += s[r];
            x[r] += d1[r] - d0[r];
          }
        } else {
          w0 = s;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x8 t;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            t[r] = s[8 * k + r] * x[8 * k + r];
            if (TY == TY_F16) t[r] *= rs;
          }
          dsf[p][k] = El<TY>::frag(t);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x8 t;
#pragma unroll
        for (int r = 0; r < 8; ++r) t[r] = w0[8 * k + r];
        const Frag pf = El<TY>::frag(t);
#pragma unroll
        for (int d = 0; d < DV / 32; ++d) dv[d] = El<TY>::mma(TG::read_cols(gt, 32 * u + 16 * k, d, lane), pf, dv[d]);
#pragma unroll
        for (int p = 0; p < MAPS; ++p)
#pragma unroll
          for (int d = 0; d < DQ / 32; ++d) dk[p][d] = El<TY>::mma(TQ::read_cols(qt + p * MB, 32 * u + 16 * k, d, lane), dsf[p][k], dk[p][d]);
      }
    }
    h = hn;
    r0 = rn;
    if (it + 1 < steps) put((it & 1) ^ 1);
    dma_wait<0>();
    __syncthreads();
  }
  if constexpr (RW == 2) {
    // the second half's sums, register by register, over the tiles: every wave is past its last read
    float* y = reinterpret_cast<float*>(smem) + (wave & 1) * 64 + lane;
    if (half_of == 1) {
#pragma unroll
      for (int p = 0; p < MAPS; ++p)
#pragma unroll
        for (int d = 0; d < DQ / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) y[((p * (DQ / 32) + d) * 16 + r) * 128] = dk[p][d][r];
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) y[((MAPS * (DQ / 32) + d) * 16 + r) * 128] = dv[d][r];
    }
    __syncthreads();
    if (half_of == 0) {
#pragma unroll
      for (int p = 0; p < MAPS; ++p)
#pragma unroll
        for (int d = 0; d < DQ / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dk[p][d][r] += y[((p * (DQ / 32) + d) * 16 + r) * 128];
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dv[d][r] += y[((MAPS * (DQ / 32) + d) * 16 + r) * 128];
    }
    __syncthreads();                                                 // past the join's reads
    if (half_of == 1) return;
  }
  if (key0 >= nk) return;
  T* ko = (T*)a.dk + b * a.sdk[0] + key0 * a.sdk[1] + hk * a.sdk[2];
  T* vo = (T*)a.dv + b * a.sdv[0] + key0 * a.sdv[1] + hk * a.sdv[2];
  typedef RowStore<TY, DQ> OutK;
  typedef RowStore<TY, DV> OutV;
  char* piece = smem + wave * (OutK::BYTES > OutV::BYTES ? OutK::BYTES : OutV::BYTES);
#pragma unroll
  for (int p = 0; p < MAPS; ++p) OutK::store(dk[p], a.scale / rs, piece, ko + (MAPS == 2 ? p * a.sdk[3] : 0), a.sdk[1], nk - key0, a.D, lane);
  OutV::store(dv, 1.0f, piece, vo, a.sdv[1], nk - key0, a.Dv, lane);
}

// A work-group a head and bucket: sums over samples and query blocks, in a fixed order.
template <int TY>
__global__ __launch_bounds__(256) void rel_dw_kernel(AttnArgs a) {
  typedef typename El<TY>::T T;
  const BwdWork wk(a, 1);
  __shared__ float red[4];
  const int k = blockIdx.x % a.num_buckets, h = blockIdx.x / a.num_buckets, tid = threadIdx.x;
  float v = 0.0f;
  for (int i = tid; i < a.B * wk.nblk; i += 256) {
    const int b = i / wk.nblk, c = i % wk.nblk;
    v += a.ws[wk.part + ((long)(b * a.H + h) * wk.nblk + c) * wk.nsum + k];
  }
  v = wave_sum(v);
  if ((tid & 63) == 0) red[tid >> 6] = v;
  __syncthreads();
  if (tid == 0) El<TY>::store((T*)a.dw + (long)k * a.H + h, (red[0] + red[1]) + (red[2] + red[3]));
}

// dlambda over all work-groups, then the four vectors
template <int TY>
__global__ __launch_bounds__(256) void diff_dw_kernel(AttnArgs a) {
  typedef typename El<TY>::T T;
  const BwdWork wk(a, 2);
  __shared__ double red[4];
  const int tid = threadIdx.x;
  const long n = (long)a.B * a.H * wk.nblk * wk.nsum;
  double t = 0.0;
  for (long i = tid; i < n; i += 256) t += (double)a.ws[wk.part + i];
#pragma unroll
  for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
  if ((tid & 63) == 0) red[tid >> 6] = t;
  __syncthreads();
  const float v = (float)-((red[0] + red[1]) + (red[2] + red[3]));
  float e1, e2;
  diff_lambda<TY>(a, e1, e2);
  const T* w = (const T*)a.w;
  T* o = (T*)a.dw;
  for (int d = tid; d < a.D; d += 256) {
    El<TY>::store(o + d, v * e1 * El<TY>::load(w + a.D + d));
    El<TY>::store(o + a.D + d, v * e1 * El<TY>::load(w + d));
    El<TY>::store(o + 2 * a.D + d, -v * e2 * El<TY>::load(w + 3 * a.D + d));
    El<TY>::store(o + 3 * a.D + d, -v * e2 * El<TY>::load(w + 2 * a.D + d));
  }
}

static inline int at_least(int a, int b) { return a > b ? a : b; }
template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW> static int launch_dq(const AttnArgs* a, const BwdWork& wk, hipStream_t stream) {
  const int lds = DqLds<TY, MAPS, DQ, DV, RW>::ALL + (BIAS ? (5 * wk.nrel + 4 * DIAG) * 4 : 0);
  if (int e = allow_lds<attn_dq_kernel<TY, MAPS, DQ, DV, BIAS, RW>>(lds)) return e;
  hipLaunchKernelGGL((attn_dq_kernel<TY, MAPS, DQ, DV, BIAS, RW>), dim3(a->B * a->H * wk.nblk), dim3(256), lds, stream, *a);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
template <int TY, int MAPS, int DQ, int DV, bool BIAS, int RW> static int launch_dkv(const AttnArgs* a, const BwdWork& wk, hipStream_t stream) {
  constexpr int STAGE = 2 * (64 * (MAPS * DQ + DV) * (int)sizeof(typename El<TY>::T) + 4 * MAPS * 64 * 4);
  constexpr int JOIN = RW == 2 ? (MAPS * DQ + DV) / 2 * 128 * 4 : 0;
  const int nblk = cdiv(a->Lk, 32 * RW), lds = at_least(STAGE + (BIAS ? wk.nrel * 4 : 0), at_least(JOIN, 4 * at_least(RowStore<TY, DQ>::BYTES, RowStore<TY, DV>::BYTES)));
  if (int e = allow_lds<attn_dkv_kernel<TY, MAPS, DQ, DV, BIAS, RW>>(lds)) return e;
  hipLaunchKernelGGL((attn_dkv_kernel<TY, MAPS, DQ, DV, BIAS, RW>), dim3(a->B * a->Hkv * nblk), dim3(256), lds, stream, *a, nblk);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
template <int TY, int MAPS, int DQ, int DV, bool BIAS> static int launch_bwd(const AttnArgs* a, hipStream_t stream) {
  const BwdWork wk(*a, MAPS);
  if (TY == TY_F16) {
    hipLaunchKernelGGL(attn_vmax_kernel, dim3(a->B * a->Hkv * wk.nv), dim3(256), 0, stream, *a, wk);
    SGTA_LAUNCH_CHECK();
  }
  if (int e = wk.rw == 2 ? launch_dq<TY, MAPS, DQ, DV, BIAS, 2>(a, wk, stream) : launch_dq<TY, MAPS, DQ, DV, BIAS, 4>(a, wk, stream)) return e;
  const bool two = row_waves((long)a->B * a->Hkv * cdiv(a->Lk, 128)) == 2;
  if (int e = two ? launch_dkv<TY, MAPS, DQ, DV, BIAS, 2>(a, wk, stream) : launch_dkv<TY, MAPS, DQ, DV, BIAS, 4>(a, wk, stream)) return e;
  if (MAPS == 1) hipLaunchKernelGGL((rel_dw_kernel<TY>), dim3(a->H * a->num_buckets), dim3(256), 0, stream, *a);
  else hipLaunchKernelGGL((diff_dw_kernel<TY>), dim3(1), dim3(256), 0, stream, *a);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}

static int bwd_check(const AttnArgs* a, int maps) {
  if (int e = attn_check(a, maps)) return e;
  if (!a->dout || !a->dq || !a->dk || !a->dv || !a->dw || !a->stats || !a->ws || (maps == 2 && !a->out2)) return SGTA_EBADARG;
  if (maps == 1 && (long)a->H * a->num_buckets >= MAX_GROUPS) return SGTA_ETOOBIG;
  if (a->ws_floats < BwdWork(*a, maps).total || (uintptr_t)a->ws % 16) return SGTA_EBADARG;
  const int al = a->dtype == TY_F32 ? 4 : 8;
  const long* s[] = {a->sdo, a->sdq, a->sdk, a->sdv};
  const void* p[] = {a->dout, a->dq, a->dk, a->dv};
  if (a->sdo[1] < 0 || a->sdo[1] > MAX_PITCH / (a->dtype == TY_F32 ? 4 : 2)) return SGTA_ETOOBIG;
  for (int i = 0; i < 4; ++i) {
    if ((uintptr_t)p[i] % 16) return SGTA_EBADARG;
    for (int j = 0; j < ((i == 1 || i == 2) && maps == 2 ? 4 : 3); ++j)
      if (s[i][j] % al) return SGTA_EBADARG;
  }
  return SGTA_OK;
}

extern "C" long sgta_attn_bwd_ws_floats(const sgta_attn_t* a, int maps) {
  return (maps != 1 && maps != 2) || attn_check(a, maps) ? 0 : BwdWork(*a, maps).total;
}

template <int TY> static int rel_bwd(const AttnArgs* a, hipStream_t st) {
  if (a->D <= 32) return launch_bwd<TY, 1, 32, 32, true>(a, st);
  if (a->D <= 64) return launch_bwd<TY, 1, 64, 64, true>(a, st);
  return launch_bwd<TY, 1, 128, 128, true>(a, st);
}
template <int TY> static int diff_bwd(const AttnArgs* a, hipStream_t st) {
  return a->D <= 32 && a->Dv <= 64 ? launch_bwd<TY, 2, 32, 64, false>(a, st) : launch_bwd<TY, 2, 64, 128, false>(a, st);
}

extern "C" int sgta_rel_attn_bwd(const sgta_attn_t* a, sgta_stream_t stream) {
  if (int e = bwd_check(a, 1)) return e;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == TY_F32 ? rel_bwd<TY_F32>(a, st) : a->dtype == TY_F16 ? rel_bwd<TY_F16>(a, st) : rel_bwd<TY_BF16>(a, st);
}
extern "C" int sgta_diff_attn_bwd(const sgta_attn_t* a, sgta_stream_t stream) {
  if (int e = bwd_check(a, 2)) return e;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == TY_F32 ? diff_bwd<TY_F32>(a, st) : a->dtype == TY_F16 ? diff_bwd<TY_F16>(a, st) : diff_bwd<TY_BF16>(a, st);
}
