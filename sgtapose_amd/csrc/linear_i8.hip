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
// One work-group a row; up to 8192 elements stay in registers between the maximum and the quotients.  The quotient's rounding is
// that of the exact quotient: the remainder x - q xs is exact in one fma for the q next to it, and decides.
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

__device__ __forceinline__ int quant1(float x, float s, float inv) {
  float q = rintf(x * inv);                            // inv overflows only where s is subnormal
  if (!(fabsf(q) <= 128.0f)) q = rintf(x / s);
  const float r = fmaf(-q, s, x), twice = fabsf(r + r);
  if (twice > s || (twice == s && ((int)q & 1))) q += r > 0.0f ? 1.0f : -1.0f;
  if (!(s > 0.0f) || q != q) q = 0.0f;                 // a row of zeros; not-a-number
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

template <int TY>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* xv, long ldx, signed char* xq, long ldq, float* xs, int K) {
  const long m = blockIdx.x;
  const typename El<TY>::T* x = (const typename El<TY>::T*)xv + m * ldx;
  signed char* o = xq + m * ldq;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool vec = (uintptr_t)x % 16 == 0, vec8 = (uintptr_t)o % 8 == 0;
  constexpr int KEEP = 4;
  float v[KEEP][8];
  unsigned top = 0;                                    // |x| by its bits: a not-a-number is the largest
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int k = (i * 256 + tid) * 8;
    if (k < K) {
      load8<TY>(x, k, K, vec, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
  }
  for (int k = (KEEP * 256 + tid) * 8; k < K; k += 2048) {
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
#pragma unroll
    for (int e = 0; e < 8; ++e) b.c[e] = (signed char)quant1(t[e], s, inv);
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
    const int k = (i * 256 + tid) * 8;
    if (k < K) write(k, v[i]);
  }
  for (int k = (KEEP * 256 + tid) * 8; k < K; k += 2048) {
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

// four consecutive channels n .. n + 3 of token m
__device__ __forceinline__ void i8_store(const I8Args& a, int m, int n, i32x4 c, float xs) {
  f32x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int nn = min(n + r, a.N - 1);
    float v = (float)c[r] * (xs * a.ws[nn]);
    if (a.bias)
      v += a.dtype == TY_F32 ? ((const float*)a.bias)[nn] : a.dtype == TY_F16 ? (float)((const _Float16*)a.bias)[nn] : (float)((const __bf16*)a.bias)[nn];
    y[r] = a.relu ? (v < 0.0f ? 0.0f : v) : v;
  }
  const long at = (long)m * a.ldo + n;
  const bool whole = n + 4 <= a.N && a.ldo % 4 == 0 && (uintptr_t)a.out % 16 == 0;
  if (a.dtype == TY_F32) {
    float* o = (float*)a.out + at;
    if (whole) El<TY_F32>::store4(o, y);
    else
      for (int r = 0; r < 4; ++r) if (n + r < a.N) El<TY_F32>::store(o + r, y[r]);
  } else if (a.dtype == TY_F16) {
    _Float16* o = (_Float16*)a.out + at;
    if (whole) El<TY_F16>::store4(o, y);
    else
      for (int r = 0; r < 4; ++r) if (n + r < a.N) El<TY_F16>::store(o + r, y[r]);
  } else {
    __bf16* o = (__bf16*)a.out + at;
    if (whole) El<TY_BF16>::store4(o, y);
    else
      for (int r = 0; r < 4; ++r) if (n + r < a.N) El<TY_BF16>::store(o + r, y[r]);
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
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = m0 + (wm * MT + j) * 32 + li;
    if (m >= a.M) continue;
    const float xs = a.xs[m];
#pragma unroll
    for (int i = 0; i < NN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + (wn * NN + i) * 32 + 8 * g + 4 * half;
        if (n < a.N) i8_store(a, m, n, i32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]}, xs);
      }
  }
}

// Few tokens: the weights are read once, straight into registers.  A work-group has 16 channels and up to 16 MT tokens
// (blockIdx.y: the next 16 MT); its 16 waves share k in pieces of 64 bytes and are summed in LDS.
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
  if (m < a.M && n < a.N) i8_store(a, m, n, c, a.xs[m]);
}

template <int BM, int BN, int WM, int WN, bool RAGGED> static int launch_i8(const I8Args& a, hipStream_t st) {
  const int tm = cdiv(a.M, BM), tn = cdiv(a.N, BN), lds = 2 * (BM + BN) * 128;
  if ((long)tm * tn > 0x7ffffff0L) return SGTA_ETOOBIG;
  if (int e = allow_lds<linear_i8_kernel<BM, BN, WM, WN, RAGGED>>(lds)) return e;
  hipLaunchKernelGGL((linear_i8_kernel<BM, BN, WM, WN, RAGGED>), dim3((tm * tn + 7) / 8 * 8), dim3(64 * WM * WN), lds, st, a, tm, tn);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}
template <int MT, bool RAGGED> static int launch_few(const I8Args& a, hipStream_t st) {
  hipLaunchKernelGGL((linear_i8_few_kernel<MT, RAGGED>), dim3(cdiv(a.N, 16), cdiv(a.M, 16 * MT)), dim3(1024), 0, st, a);
  SGTA_LAUNCH_CHECK();
  return SGTA_OK;
}

extern "C" int sgta_quant_rows_i8(const void* x, long ldx, int dtype, signed char* xq, long ldq, float* xs, int M, int K, sgta_stream_t stream) {
  if (!x || !xq || !xs || M < 1 || K < 1 || ldx < K || ldq < K || dtype < 0 || dtype > 2) return SGTA_EBADARG;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TY_F32) hipLaunchKernelGGL(quant_rows_kernel<TY_F32>, dim3(M), dim3(256), 0, st, x, ldx, xq, ldq, xs, K);
  else if (dtype == TY_F16) hipLaunchKernelGGL(quant_rows_kernel<TY_F16>, dim3(M), dim3(256), 0, st, x, ldx, xq, ldq, xs, K);
  else hipLaunchKernelGGL(quant_rows_kernel<TY_BF16>, dim3(M), dim3(256), 0, st, x, ldx, xq, ldq, xs, K);
  SGTA_LAUNCH_CHECK();
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
  if (!ragged && (long)cdiv(M, 256) * cdiv(N, 256) >= 192) return launch_i8<256, 256, 2, 4, false>(a, st);
  if ((long)cdiv(M, 128) * cdiv(N, 128) >= 192) return ragged ? launch_i8<128, 128, 2, 2, true>(a, st) : launch_i8<128, 128, 2, 2, false>(a, st);
  return ragged ? launch_i8<64, 64, 2, 2, true>(a, st) : launch_i8<64, 64, 2, 2, false>(a, st);
}
