// Token products in 8-bit integers on gfx950: rows quantised with a scale of their own, products on the integer matrix pipe,
// scales, bias and activation in the epilogue.
//   xs[m] = max_k |x[m,k]| / 127,  xq[m,k] = rint(x[m,k] / xs[m])
//   out[m,n] = relu?( (sum_k xq[m,k] wq[n,k]) xs[m] ws[n] + bias[n] )
// The sum is exact (K <= 131071: below 2^31 whatever the bytes), so it depends on no tile or order.
//
// Both operands are rows of consecutive k, which is what the matrix instructions read (16 bytes of k per lane): A holds 32
// output channels, B 32 tokens, so a lane ends up with four consecutive channels of one token.
#include "attn_common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- quantisation of rows ------------------------------------------------------------------------
// A work-group a row; up to 8192 elements stay in registers between the maximum and the quotients.  The rounding is that of the
// exact quotient: q = rint(x (1 / xs)) is at most one off, and the remainder x - q xs, exact in one fma for the q next to the
// quotient, tells.  16384 x 4096 bfloat16: 201 MB in 42 us, the rate of a copy (a wave a row: 55 us).
template <int TY> __device__ __forceinline__ void load8(const typename El<TY>::T* p, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    const typename El<TY>::Raw f = *reinterpret_cast<const typename El<TY>::Raw*>(p + k);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)f[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? El<TY>::load(p + k + e) : 0.0f;
  }
}

// one quotient with every case: subnormal scales, rows of zeros, what is not finite
__device__ __forceinline__ int quant1(float x, float s, float inv) {
  float q = rintf(x * inv);                            // inv overflows only where s is subnormal
  if (!(fabsf(q) <= 128.0f)) q = rintf(x / s);
  const float r = fmaf(-q, s, x), twice = fabsf(r + r);
  if (twice > s || (twice == s && ((int)q & 1))) q += r > 0.0f ? 1.0f : -1.0f;
  if (!(s > 0.0f) || q != q) q = 0.0f;                 // a row of zeros; not-a-number
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// eight quotients as bytes
__device__ __forceinline__ unsigned long long quant8(const float (&v)[8], float s, float inv) {
  // 1.5 2^23 + x inv: the sum's rounding is rint, and its low byte is the quotient's
  constexpr float BIG = 12582912.0f;
  unsigned t[8];
  const float h = 0.5f * s;
  bool odd = !(s >= 1e-30f && s < INFINITY);           // scales whose half or inverse may not be exact
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float b = fmaf(v[e], inv, BIG), r = fmaf(-(b - BIG), s, v[e]);
    odd |= !(fabsf(r) < h);
    t[e] = __float_as_uint(b);
  }
  if (odd) {                                           // a quotient at a half or on the other side of one: rare
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (unsigned)quant1(v[e], s, inv);
  }
  const unsigned lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u) | __builtin_amdgcn_perm(t[3], t[2], 0x04000c0cu);
  const unsigned hi = __builtin_amdgcn_perm(t[5], t[4], 0x0c0c0400u) | __builtin_amdgcn_perm(t[7], t[6], 0x04000c0cu);
  return (unsigned long long)hi << 32 | lo;
}

template <int TY>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* xv, long ldx, signed char* xq, long ldq, float* xs, int K) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long m = blockIdx.x;
  const typename El<TY>::T* x = (const typename El<TY>::T*)xv + m * ldx;
  signed char* o = xq + m * ldq;
  const bool vec = (uintptr_t)x % 16 == 0, vec8 = (uintptr_t)o % 8 == 0;
  constexpr int KEEP = 4, NT = 256;
  float v[KEEP][8];
  unsigned top = 0;                                    // |x| by its bits: a not-a-number is the largest
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int k = (i * NT + tid) * 8;
    if (k < K) {
      load8<TY>(x, k, K, vec, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
  }
  for (int k = (KEEP * NT + tid) * 8; k < K; k += NT * 8) {
    float t[8];
    load8<TY>(x, k, K, vec, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  __shared__ unsigned part[4];
  if (lane == 0) part[wave] = top;
  __syncthreads();
  top = max(max(part[0], part[1]), max(part[2], part[3]));
  const float s = __uint_as_float(top) / 127.0f, inv = 1.0f / s;
  if (tid == 0) xs[m] = s;
  auto write = [&](int k, const float (&t)[8]) {
    union { signed char c[8]; unsigned long long u; } b;
    b.u = quant8(t, s, inv);
    if (vec8 && k + 8 <= K) {
      *reinterpret_cast<unsigned long long*>(o + k) = b.u;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) o[k + e] = b.c[e];
    }
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int k = (i * NT + tid) * 8;
    if (k < K) write(k, v[i]);
  }
  for (int k = (KEEP * NT + tid) * 8; k < K; k += NT * 8) {
    float t[8];
    load8<TY>(x, k, K, vec, t);
    write(k, t);
  }
}

// ---- products ------------------------------------------------------------------------------------
struct I8Args {
  const signed char *xq, *wq;
  const float *xs, *ws;
  const void* bias;
  void* out;
  long ldx, ldw, ldo;
  int M, N, K, relu, dtype;
};

// Four consecutive channels n .. n + 3 of token m.  WHOLE: all four exist (as 16 bytes of any row do) and are aligned.
template <int TY, bool WHOLE> __device__ __forceinline__ void i8_store(const I8Args& a, int m, int n, i32x4 c, float xs) {
  typedef typename El<TY>::T T;
  T* o = (T*)a.out + (long)m * a.ldo + n;
  const T* bias = (const T*)a.bias;
  f32x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int nn = WHOLE ? n + r : min(n + r, a.N - 1);
    y[r] = (float)c[r] * (xs * a.ws[nn]);
    if (bias) y[r] += El<TY>::load(bias + nn);
    if (a.relu) y[r] = y[r] < 0.0f ? 0.0f : y[r];
  }
  if (WHOLE) El<TY>::store4(o, y);
  else
    for (int r = 0; r < 4; ++r) if (n + r < a.N) El<TY>::store(o + r, y[r]);
}
// calls f<type, WHOLE> for the output at hand: one branch for all of a wave's stores
template <typename F> __device__ __forceinline__ void i8_epilogue(const I8Args& a, F f) {
  const int per = a.dtype == TY_F32 ? 4 : 8;
  const bool whole = a.N % per == 0 && a.ldo % per == 0 && (uintptr_t)a.out % 16 == 0;
  if (a.dtype == TY_F32) {
    if (whole) f.template operator()<TY_F32, true>(); else f.template operator()<TY_F32, false>();
  } else if (a.dtype == TY_F16) {
    if (whole) f.template operator()<TY_F16, true>(); else f.template operator()<TY_F16, false>();
  } else {
    if (whole) f.template operator()<TY_BF16, true>(); else f.template operator()<TY_BF16, false>();
  }
}

// 16 bytes k .. k + 15 of a row at any alignment, zero from K on
__device__ __forceinline__ i32x4 row16(const signed char* p, int k, int K) {
  i32x4 v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, p + k, 16);
  } else if (k < K) {
    union { signed char c[16]; i32x4 v; } b;
#pragma unroll
    for (int e = 0; e < 16; ++e) b.c[e] = k + e < K ? p[k + e] : (signed char)0;
    v = b.v;
  }
  return v;
}

// A wave's accumulators: tokens m .. m + 32 MT, channels n .. n + 32 NN.  WHOLE: through a piece of LDS of the wave's own, 32 tokens
// at a time, so that every store instruction writes 16-byte pieces of whole runs of a row.  (Straight from the registers a store
// writes 16 bytes to each of 32 rows: at 16384 x 4096 x 4096 that took 130 of 380 us.)
template <int MT, int NN> struct Finish {
  const I8Args& a;
  const i32x16 (&acc)[NN][MT];
  int m, n;
  char* lds;
  static constexpr int PITCH = NN * 32 * 4 + 16, BYTES = 32 * PITCH;
  template <int TY, bool WHOLE> __device__ __forceinline__ void operator()() const {
    typedef typename El<TY>::T T;
    const int lane = threadIdx.x & 63, li = lane & 31, half = lane >> 5;
    if constexpr (!WHOLE) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int mm = m + 32 * j + li;
        if (mm >= a.M) continue;
        const float xs = a.xs[mm];
#pragma unroll
        for (int i = 0; i < NN; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int nn = n + 32 * i + 8 * g + 4 * half;
            if (nn < a.N) i8_store<TY, false>(a, mm, nn, i32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]}, xs);
          }
      }
    } else {
      constexpr int SZ = sizeof(T), PER = NN * 32 * SZ / 16;       // 16-byte pieces of a row
      f32x4 ws[NN][4], bias[NN][4];
#pragma unroll
      for (int i = 0; i < NN; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int nn = min(n + 32 * i + 8 * g + 4 * half, a.N - 4);
          __builtin_memcpy(&ws[i][g], a.ws + nn, 16);
          bias[i][g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if (a.bias)
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[i][g][r] = El<TY>::load((const T*)a.bias + nn + r);
        }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const float xs = a.xs[min(m + 32 * j + li, a.M - 1)];
        asm volatile("" ::: "memory");                 // a wave's LDS operations are done in order; the compiler keeps it
#pragma unroll
        for (int i = 0; i < NN; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              y[r] = (float)acc[i][j][4 * g + r] * (xs * ws[i][g][r]) + bias[i][g][r];
              if (a.relu) y[r] = y[r] < 0.0f ? 0.0f : y[r];
            }
            El<TY>::store4((T*)(lds + li * PITCH) + 32 * i + 8 * g + 4 * half, y);
          }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int p = 0; p < 32 * PER / 64; ++p) {
          const int row = (p * 64 + lane) / PER, c = (p * 64 + lane) % PER;
          const u32x4 v = *reinterpret_cast<const u32x4*>(lds + row * PITCH + c * 16);
          const int mm = m + 32 * j + row, nn = n + c * (16 / SZ);
          if (mm < a.M && nn < a.N) *reinterpret_cast<u32x4*>((T*)a.out + (long)mm * a.ldo + nn) = v;
        }
      }
    }
  }
};

// Tiled product: WM x WN waves, each (BM / WM) tokens x (BN / WN) channels in 32 x 32 tiles; 128-byte slices of k, double
// buffered in LDS.  RAGGED false: rows of whole 16-byte pieces, copied straight into LDS (each lane's piece chosen so that the
// pieces of a row lie XOR-swizzled by the row; rows and pieces out of range read as zero).  RAGGED true: any alignment, through
// registers.
template <int BM, int BN, int WM, int WN, bool RAGGED>
__global__ __launch_bounds__(64 * WM * WN) void linear_i8_kernel(I8Args a, int tm, int tn) {
  constexpr int NT = 64 * WM * WN, MT = BM / WM / 32, NN = BN / WN / 32, STAGE = (BM + BN) * 128;
  constexpr int PX = BM * 8 / NT, PW = BN * 8 / NT;    // pieces per thread and slice
  extern __shared__ __align__(16) char smem[];
  // consecutive tiles of one XCD: 8 token tiles by all channel tiles, so that both operands' slices are shared in its L2
  const int T = tm * tn, per = (T + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= T) return;
  const int g0 = id / (8 * tn) * 8, gm = min(8, tm - g0), rest = id - g0 * tn;
  const int m0 = (g0 + rest % gm) * BM, n0 = rest / gm * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, half = lane >> 5;
  const int wm = wave % WM, wn = wave / WM;
  const int slices = (a.K + 127) / 128;
  const signed char* xp = a.xq + (long)m0 * a.ldx;
  const signed char* wp = a.wq + (long)n0 * a.ldw;
  const int xrows = min(BM, a.M - m0), wrows = min(BN, a.N - n0);

  i32x4 rx[RAGGED ? PX : 1], rw[RAGGED ? PW : 1];
#if defined(__HIP_DEVICE_COMPILE__)
  __amdgpu_buffer_rsrc_t xr, wr;
  if (!RAGGED) {
    xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char*>(xp), (short)0, (int)((xrows - 1) * a.ldx + a.K), 0x00020000);
    wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char*>(wp), (short)0, (int)((wrows - 1) * a.ldw + a.K), 0x00020000);
  }
#endif
  typedef __attribute__((address_space(3))) void* lds_ptr_t;
  auto fetch = [&](int s, int buf) {
    char* dst = smem + buf * STAGE;
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      const int p = i * NT + tid, row = p >> 3, k = s * 128 + ((p ^ row) & 7) * 16;
      if constexpr (RAGGED) {
        rx[i] = row < xrows ? row16(xp + row * a.ldx, s * 128 + (p & 7) * 16, a.K) : i32x4{0, 0, 0, 0};
      } else {
#if defined(__HIP_DEVICE_COMPILE__)
        const unsigned off = row < xrows && k < a.K ? (unsigned)(row * a.ldx + k) : 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_ptr_t)(dst + (i * NT + wave * 64) * 16), 16, off, 0, 0, 0);
#endif
      }
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int p = i * NT + tid, row = p >> 3, k = s * 128 + ((p ^ row) & 7) * 16;
      if constexpr (RAGGED) {
        rw[i] = row < wrows ? row16(wp + row * a.ldw, s * 128 + (p & 7) * 16, a.K) : i32x4{0, 0, 0, 0};
      } else {
#if defined(__HIP_DEVICE_COMPILE__)
        const unsigned off = row < wrows && k < a.K ? (unsigned)(row * a.ldw + k) : 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_ptr_t)(dst + BM * 128 + (i * NT + wave * 64) * 16), 16, off, 0, 0, 0);
#endif
      }
    }
  };
  auto put = [&](int buf) {
    if constexpr (RAGGED) {
      char* dst = smem + buf * STAGE;
#pragma unroll
      for (int i = 0; i < PX; ++i) {
        const int p = i * NT + tid, row = p >> 3;
        *reinterpret_cast<i32x4*>(dst + row * 128 + ((p ^ row) & 7) * 16) = rx[i];
      }
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        const int p = i * NT + tid, row = p >> 3;
        *reinterpret_cast<i32x4*>(dst + BM * 128 + row * 128 + ((p ^ row) & 7) * 16) = rw[i];
      }
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of the slice has landed
    }
  };

  i32x16 acc[NN][MT];
#pragma unroll
  for (int i = 0; i < NN; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  fetch(0, 0);
  put(0);
  __syncthreads();
  for (int s = 0; s < slices; ++s) {
    const char* xb = smem + (s & 1) * STAGE;
    const char* wb = xb + BM * 128;
    if (s + 1 < slices) fetch(s + 1, (s & 1) ^ 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      i32x4 wf[NN], xf[MT];
#pragma unroll
      for (int i = 0; i < NN; ++i) {
        const int row = (wn * NN + i) * 32 + li;
        wf[i] = *reinterpret_cast<const i32x4*>(wb + row * 128 + (((2 * k + half) ^ row) & 7) * 16);
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int row = (wm * MT + j) * 32 + li;
        xf[j] = *reinterpret_cast<const i32x4*>(xb + row * 128 + (((2 * k + half) ^ row) & 7) * 16);
      }
#pragma unroll
      for (int i = 0; i < NN; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
    }
    if (s + 1 < slices) put((s & 1) ^ 1);
    __syncthreads();
  }
  static_assert(WM * WN * Finish<MT, NN>::BYTES <= 2 * STAGE, "the epilogue's pieces lie over the slices");
  const Finish<MT, NN> fin{a, acc, m0 + wm * MT * 32, n0 + wn * NN * 32, smem + __builtin_amdgcn_readfirstlane(wave) * Finish<MT, NN>::BYTES};
  i8_epilogue(a, fin);
}

// Large products: 256 x 256 tiles by 4 waves of 128 x 128, one a SIMD with its 512 registers.  LDS is what such a tile runs into
// first: 4 waves read 8 fragments of 1 KB for 16 matrix instructions (256 of 512 cycles; 8 waves of 128 x 64: 384), and a quarter
// more goes to filling it.  With one wave nothing else hides a wait, so everything is fetched ahead: the next 128-byte slice of k
// (whole cache lines of every row) into the other buffer from the last of a slice's four steps on, and the next step's fragments
// into the other set of registers, also across the slices' one barrier, which comes before the last step's products.
// 16384 x 4096 x 4096: 260 us = 2110 TOPS, matrix pipe 52 % of the cycles; from registers alone random bytes reach 3400 to 3570 (the
// chip's power), so filling and reading LDS costs the rest.
__global__ __launch_bounds__(256, 1) void linear_i8_large_kernel(I8Args a, int tm, int tn) {
  constexpr int STAGE = 512 * 128;                                // 256 token rows, then 256 channel rows
  extern __shared__ __align__(16) char smem[];
  const int T = tm * tn, per = (T + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= T) return;
  const int g0 = id / (8 * tn) * 8, gm = min(8, tm - g0), rest = id - g0 * tn;
  const int m0 = (g0 + rest % gm) * 256, n0 = rest / gm * 256;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, half = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;
  const int slices = (a.K + 127) / 128;
  const int xrows = min(256, a.M - m0), wrows = min(256, a.N - n0);
  // piece 256 i + tid: row 32 i + tid / 8, 16-byte piece (tid ^ row) & 7 of the slice, stored at its place
  const int r0 = tid >> 3, ch = ((tid ^ r0) & 7) * 16;
  unsigned xoff = r0 * (int)a.ldx + ch, woff = r0 * (int)a.ldw + ch;
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) void* lds_ptr_t;
  const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)(smem + wave * 1024);
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char*>(a.xq + (long)m0 * a.ldx), (short)0, (int)((xrows - 1) * a.ldx + a.K), 0x00020000);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char*>(a.wq + (long)n0 * a.ldw), (short)0, (int)((wrows - 1) * a.ldw + a.K), 0x00020000);
#endif
  // one of a slice's sixteen loads of this wave; rows beyond the last lie beyond the resource: zeros
  auto fetch = [&](int s, int i) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int at = s * 128;
    const bool in = at + ch < a.K;                                // the last slice may be a part of one; those behind it are none
    const int step = 32 * (i & 7), ld = (int)(i < 8 ? a.ldx : a.ldw);
    dma16(i < 8 ? xr : wr, in ? (i < 8 ? xoff : woff) + (unsigned)(step * ld + at) : 0x80000000u, lds0 + (s & 1) * STAGE + i * 4096);
#endif
  };
  const char* xb = smem + (wm * 128 + li) * 128;
  const char* wb = smem + (256 + wn * 128 + li) * 128;
  auto read = [&](i32x4 (&wf)[4], i32x4 (&xf)[4], int s, int k) {
    const int at = (s & 1) * STAGE + (((2 * k + half) ^ li) & 7) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) wf[i] = *reinterpret_cast<const i32x4*>(wb + at + i * 4096);
#pragma unroll
    for (int i = 0; i < 4; ++i) xf[i] = *reinterpret_cast<const i32x4*>(xb + at + i * 4096);
  };
  i32x16 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x16{0};
  i32x4 wf[2][4], xf[2][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) fetch(0, i);
#pragma unroll
  for (int i = 0; i < 8; ++i) fetch(1, i);
  dma_wait<8>();
  __syncthreads();
  read(wf[0], xf[0], 0, 0);
  for (int s = 0; s < slices; ++s) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k == 3) {
        dma_wait<0>();                                            // the next slice has landed,
        __builtin_amdgcn_s_waitcnt(0xc07f);                       // this one is in registers,
        __builtin_amdgcn_s_barrier();                             // for every wave
      }
      // the next step's fragments first (the scheduler would put each read next to its use), this step's products under them
      if (k < 3) read(wf[(k + 1) & 1], xf[(k + 1) & 1], s, k + 1);
      else read(wf[0], xf[0], s + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[k & 1][i], xf[k & 1][j], acc[i][j], 0, 0, 0);
        if (k == 0) {
          fetch(s + 1, 8 + 2 * i);
          fetch(s + 1, 9 + 2 * i);
        }
        if (k == 3) {
          fetch(s + 2, 2 * i);
          fetch(s + 2, 2 * i + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  dma_wait<0>();
  __syncthreads();                                                // the epilogue's pieces lie over the slices
  const Finish<4, 4> fin{a, acc, m0 + wm * 128, n0 + wn * 128, smem + wave * Finish<4, 4>::BYTES};
  i8_epilogue(a, fin);
}

struct FinishOne {
  const I8Args& a;
  int m, n;
  i32x4 c;
  template <int TY, bool WHOLE> __device__ __forceinline__ void operator()() const { i8_store<TY, WHOLE>(a, m, n, c, a.xs[m]); }
};

// Few tokens: the weights are read once, straight into registers.  A work-group has 16 channels and up to 16 MT tokens
// (blockIdx.y: the next 16 MT); its 16 waves share k in pieces of 64 bytes and are summed in LDS.  4 x 4096 x 4096: 6.4 us for 17 MB,
// most of it the latency of launch, one round of loads and the sum.  (33 to 64 tokens at any alignment: 1024 threads leave 128 registers
// each, and 44 are stored in the loop.)
template <int MT, bool RAGGED>
__global__ __launch_bounds__(1024) void linear_i8_few_kernel(I8Args a) {
  __shared__ i32x4 part[16][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const signed char* wp = a.wq + (long)min(n0 + li, a.N - 1) * a.ldw;
  const signed char* xp[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xp[j] = a.xq + (long)min(m0 + 16 * j + li, a.M - 1) * a.ldx;   // rows beyond the last are not stored
  i32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = i32x4{0, 0, 0, 0};
  const int steps = (a.K + 63) / 64;
  const int run = min(4, (steps + 15) / 16);           // consecutive pieces a wave takes
  for (int s0 = wave * run; s0 < steps; s0 += 16 * run) {
    i32x4 wf[4], xf[4][MT];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = (s0 + u) * 64 + q * 16;
      wf[u] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < MT; ++j) xf[u][j] = i32x4{0, 0, 0, 0};
      if (u < run && k < a.K) {
        if constexpr (RAGGED) {
          wf[u] = row16(wp, k, a.K);
#pragma unroll
          for (int j = 0; j < MT; ++j) xf[u][j] = row16(xp[j], k, a.K);
        } else {
          wf[u] = *reinterpret_cast<const i32x4*>(wp + k);
#pragma unroll
          for (int j = 0; j < MT; ++j) xf[u][j] = *reinterpret_cast<const i32x4*>(xp[j] + k);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][j], acc[j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave >= MT) return;
  i32x4 c = part[0][wave][lane];
#pragma unroll
  for (int v = 1; v < 16; ++v) c += part[v][wave][lane];
  const int m = m0 + 16 * wave + li, n = n0 + 4 * q;
  if (m < a.M && n < a.N) i8_epilogue(a, FinishOne{a, m, n, c});
}

template <int BM, int BN, int WM, int WN, bool RAGGED> static int launch_i8(const I8Args& a, hipStream_t st) {
  const int tm = cdiv(a.M, BM), tn = cdiv(a.N, BN), lds = 2 * (BM + BN) * 128;
  if ((long)tm * tn >= MAX_GROUPS - 8) return SGTA_ETOOBIG;
  if (int e = allow_lds<linear_i8_kernel<BM, BN, WM, WN, RAGGED>>(lds)) return e;
  hipLaunchKernelGGL((linear_i8_kernel<BM, BN, WM, WN, RAGGED>), dim3((tm * tn + 7) / 8 * 8), dim3(64 * WM * WN), lds, st, a, tm, tn);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
static int launch_i8_large(const I8Args& a, hipStream_t st) {
  const int tm = cdiv(a.M, 256), tn = cdiv(a.N, 256), lds = 2 * 512 * 128;
  if ((long)tm * tn >= MAX_GROUPS - 8) return SGTA_ETOOBIG;
  if (int e = allow_lds<linear_i8_large_kernel>(lds)) return e;
  hipLaunchKernelGGL(linear_i8_large_kernel, dim3((tm * tn + 7) / 8 * 8), dim3(256), lds, st, a, tm, tn);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
template <int MT, bool RAGGED> static int launch_few(const I8Args& a, hipStream_t st) {
  if (cdiv(a.N, 16) >= MAX_GROUPS / 4) return SGTA_ETOOBIG;          // work-groups of 1024
  hipLaunchKernelGGL((linear_i8_few_kernel<MT, RAGGED>), dim3(cdiv(a.N, 16), cdiv(a.M, 16 * MT)), dim3(1024), 0, st, a);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}

extern "C" int sgta_quant_rows_i8(const void* x, long ldx, int dtype, signed char* xq, long ldq, float* xs, int M, int K, sgta_stream_t stream) {
  if (!x || !xq || !xs || M < 1 || K < 1 || ldx < K || ldq < K || dtype < 0 || dtype > 2) return SGTA_EBADARG;
  hipStream_t st = (hipStream_t)stream;
  for (long m = 0; m < M; m += MAX_GROUPS / 2) {         // a launch each 2^23 rows
    const dim3 rows(M - m < MAX_GROUPS / 2 ? M - m : MAX_GROUPS / 2);
    const char* p = (const char*)x + m * ldx * (dtype == TY_F32 ? 4 : 2);
    signed char* o = xq + m * ldq;
    if (dtype == TY_F32) hipLaunchKernelGGL(quant_rows_kernel<TY_F32>, rows, dim3(256), 0, st, p, ldx, o, ldq, xs + m, K);
    else if (dtype == TY_F16) hipLaunchKernelGGL(quant_rows_kernel<TY_F16>, rows, dim3(256), 0, st, p, ldx, o, ldq, xs + m, K);
    else hipLaunchKernelGGL(quant_rows_kernel<TY_BF16>, rows, dim3(256), 0, st, p, ldx, o, ldq, xs + m, K);
    SGTA_LAUNCH_CHECK();
  }
  return SGTA_OK;
}

extern "C" int sgta_linear_i8(const signed char* xq, long ldx, const float* xs, const signed char* wq, long ldw, const float* ws,
                              const void* bias, void* out, long ldo, int M, int N, int K, int relu, int dtype, sgta_stream_t stream) {
  if (!xq || !xs || !wq || !ws || !out || M < 1 || N < 1 || K < 1 || ldx < K || ldw < K || ldo < N || dtype < 0 || dtype > 2) return SGTA_EBADARG;
  if (K > 131071 || ldx > 1 << 22 || ldw > 1 << 22) return SGTA_ETOOBIG;   // exact sums; a tile's rows within 2^31 bytes
  if ((uintptr_t)out % (dtype == TY_F32 ? 4 : 2) || (uintptr_t)bias % (dtype == TY_F32 ? 4 : 2)) return SGTA_EBADARG;
  const I8Args a = {xq, wq, xs, ws, bias, out, ldx, ldw, ldo, M, N, K, relu, dtype};
  hipStream_t st = (hipStream_t)stream;
  const bool ragged = K % 16 || ldx % 16 || ldw % 16 || (uintptr_t)xq % 16 || (uintptr_t)wq % 16;
  if (M <= 64) {
    if (M <= 16) return ragged ? launch_few<1, true>(a, st) : launch_few<1, false>(a, st);
    if (M <= 32) return ragged ? launch_few<2, true>(a, st) : launch_few<2, false>(a, st);
    return ragged ? launch_few<4, true>(a, st) : launch_few<4, false>(a, st);
  }
  // the largest tile that still gives most of the 256 compute units one
  if (!ragged && (long)cdiv(M, 256) * cdiv(N, 256) >= 192) return launch_i8_large(a, st);
  if ((long)cdiv(M, 128) * cdiv(N, 128) >= 192) return ragged ? launch_i8<128, 128, 2, 2, true>(a, st) : launch_i8<128, 128, 2, 2, false>(a, st);
  return ragged ? launch_i8<64, 64, 2, 2, true>(a, st) : launch_i8<64, 64, 2, 2, false>(a, st);
}
