// What the attention kernels share (attn_fwd.hip, attn_bwd.hip): element types, LDS tiles and their fragments, staging.
//
// Every product runs on 32x32 matrix tiles, v_mfma_f32_32x32x16_{f16,bf16}, float as three bfloat16 numbers.  A lane's operand
// fragment: lane l has row l & 31 and k = 8 (l >> 5) + 0..7 of a step of 16.
// A result has its column on the lane (l & 31) and row 8 (r >> 2) + 4 (l >> 5) + (r & 3) in register r.  Eight consecutive
// result registers are therefore an operand fragment of 16 rows in the order {0-3, 8-11} / {4-7, 12-15} of the two lane
// halves; read_cols() hands out the other operand in that same order, so softmax weights go from one product into the next
// without leaving their registers.
#pragma once
#include "common.h"
#include "../../include/sgta_hip.h"

typedef sgta_attn_t AttnArgs;

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

enum { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 2 };

template <int TY> struct El;

// float on the bfloat16 pipe.  A float's 24 significant bits are three bfloat16 numbers, x = hi + mid + lo exactly (each the upper
// half of what the ones before leave); of the nine products of two such sums the six of at least 2^-16 of the whole are taken, smallest
// first, each with all its bits into the f32 accumulator.  mid is below 2^-7 of the leading power and lo below 2^-15, so what is left out,
// mid lo + lo mid + lo lo, is below 2^-21 = 8 * 2^-24 of |a||b| (2 * 2^-24 on average), of the product's sign.  Split to the nearest it
// would be below 2^-24, but a float next to the largest would become an infinity, and that a not-a-number behind a mask's weight of zero.
// Six v_mfma_f32_32x32x16_bf16 (192 cycles) in place of eight v_mfma_f32_32x32x2_f32 (512), and the splits, ~44 vector
// instructions a fragment, overlap them.  Same range as float; what is not finite gives not-a-number in hi - hi: so does x * 0.
struct Split8 {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  x8 hi, mid, lo;
};
__device__ __forceinline__ unsigned upper_halves(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
__device__ __forceinline__ Split8 split8(f32x8 v) {
  typedef unsigned u32x4_ __attribute__((ext_vector_type(4)));
  u32x4_ h, m, l;
  f32x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e] - __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = upper_halves(v[2 * e], v[2 * e + 1]);
    m[e] = upper_halves(r[2 * e], r[2 * e + 1]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u);
#pragma unroll
  for (int e = 0; e < 4; ++e) l[e] = upper_halves(r[2 * e], r[2 * e + 1]);
  Split8 s;
  s.hi = __builtin_bit_cast(Split8::x8, h);
  s.mid = __builtin_bit_cast(Split8::x8, m);
  s.lo = __builtin_bit_cast(Split8::x8, l);
  return s;
}

template <> struct El<TY_F32> {
  typedef float T;
  typedef Split8 Frag;         // an operand fragment
  typedef f32x8 Raw;           // eight elements as they lie in memory
  static __device__ __forceinline__ f32x16 mma_small(Frag a, Frag b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.lo, b.hi, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.lo, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.mid, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.hi, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.mid, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma_large(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.hi, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return mma_large(a, b, mma_small(a, b, c)); }
  static __device__ __forceinline__ Frag frag(f32x8 v) { return split8(v); }
  static __device__ __forceinline__ Frag frag_of(Raw v) { return split8(v); }
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void store4(T* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
};
template <bool F16> struct El16 {
  typedef typename H16<F16>::T T;
  typedef typename H16<F16>::x4 x4;
  typedef typename H16<F16>::x8 Frag;
  typedef Frag Raw;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return H16<F16>::mfma32(a, b, c); }
  static __device__ __forceinline__ Frag frag_of(Raw v) { return v; }
  // to the nearest, without the clamp of the 16-bit feature maps: here what exceeds the half range becomes an infinity, by which
  // a training loop sees that its loss is scaled too far
  static __device__ __forceinline__ Frag frag(f32x8 v) { return __builtin_convertvector(v, Frag); }
  static __device__ __forceinline__ float load(const T* p) { return (float)*p; }
  static __device__ __forceinline__ void store4(T* p, f32x4 v) { *reinterpret_cast<x4*>(p) = __builtin_convertvector(v, x4); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = (T)v; }
};
template <> struct El<TY_F16> : El16<true> {};
template <> struct El<TY_BF16> : El16<false> {};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// the other lane half's value beside one's own: {value of lane l & 31, value of lane 32 + (l & 31)}
__device__ __forceinline__ void both_halves(float x, float& lo, float& hi) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_sum(float x) {
  float a, b;
  both_halves(x, a, b);
  return a + b;
}
__device__ __forceinline__ float half_max(float x) {
  float a, b;
  both_halves(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// One operand tile in LDS: rows of COLS elements in 16-byte pieces, XOR-swizzled by the row so that what LDS serves at a time
// falls on different banks: one piece of 8 consecutive rows (read_rows), and two neighbouring pieces of 4 (read_cols; a swizzle
// by the row number itself puts rows r and r ^ 1 on one pair of pieces: half of these reads' cycles were conflicts).
template <int TY, int COLS> struct Tile {
  typedef typename El<TY>::T T;
  typedef typename El<TY>::Frag Frag;
  static constexpr int SZ = sizeof(T);
  static constexpr int ROWB = COLS * SZ;              // bytes per row: 64 ... 512
  static constexpr int CH = ROWB / 16;                // pieces per row
  static constexpr int EPC = 16 / SZ;                 // elements per piece
  static __device__ __forceinline__ int swz(int row) {
    return ROWB >= 128 ? ((row & 3) << 1) | ((row >> 2) & 1) : (row & 2) | ((row >> 2) & 1);
  }
  static __device__ __forceinline__ int piece(int row, int ch) { return row * ROWB + ((ch ^ swz(row)) << 4); }

  // operand fragment of row ``row``: elements 16 s + 8 half + 0..7
  static __device__ __forceinline__ Frag read_rows(const char* lds, int row, int s, int half) {
    if constexpr (TY == TY_F32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + piece(row, 4 * s + 2 * half));
      const f32x4 b = *reinterpret_cast<const f32x4*>(lds + piece(row, 4 * s + 2 * half + 1));
      return split8(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const Frag*>(lds + piece(row, 2 * s + half));
    }
  }
  // operand fragment of COLUMN 32 blk + (lane & 31): rows row0 + {0-3, 8-11} + 4 half, the order of the result registers
  static __device__ __forceinline__ Frag read_cols(const char* lds, int row0, int blk, int lane) {
    if constexpr (TY == TY_F32) {
      const int col = 32 * blk + (lane & 31), half = lane >> 5;
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = row0 + 4 * half + (e & 3) + 8 * (e >> 2);
        f[e] = *reinterpret_cast<const float*>(lds + piece(row, col >> 2) + (col & 3) * 4);
      }
      return split8(f);
    } else {
      // transposing read: each 16 lanes fetch 4 rows x 16 columns, lane i of them gets column i of the 4 rows
      const int g = lane >> 4, i = lane & 15;
      const int row = row0 + 4 * (g >> 1) + (i >> 2), col = 32 * blk + 16 * (g & 1) + 4 * (i & 3);
      typedef __attribute__((address_space(3))) s16x4* lp;
      s16x8 v;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + piece(row, col >> 3) + (col & 4) * 2));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + piece(row + 8, col >> 3) + (col & 4) * 2));
      v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(Frag, v);
    }
  }
};

// Global memory -> LDS, 16 bytes a lane, to LDS byte ``at`` + 16 lane.  In assembly although there is a builtin: of that the
// compiler assumes that any transposing LDS read may see its data, and waits for all of it (the NEXT tile) before each of them.
// It has no result register; what was loaded is read only after dma_wait and a barrier.  Between the write of M0 and a load into LDS the
// hardware asks for one wait state, which the compiler does not add inside assembly (tests/test_wait_states.py looks for it, and for the
// five between a vector instruction's write of a scalar register and the load, in the built library).  M0 stays on the clobber list,
// so that the compiler takes no value of its own for still there; its remark, that it does not save the register, is what is wanted.
#if defined(__HIP_DEVICE_COMPILE__)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned off, unsigned at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(rs) : "memory", "m0");
}
#pragma clang diagnostic pop
#endif

// Rows of a strided matrix into a Tile by NT threads, straight into LDS (no registers, no LDS store instructions): a wave writes
// 64 consecutive pieces, so each lane fetches the piece that belongs at its place of the swizzle.  Rows from ``rows`` on and
// elements from ``cols`` on are zero and never read: what lies there may be anything.  The loads are in flight until dma_wait.
template <int TY, int COLS, int ROWS, int NT> struct Dma {
  typedef Tile<TY, COLS> Tl;
  typedef typename El<TY>::T T;
  static constexpr int ALL = ROWS * Tl::CH, N = (ALL + NT - 1) / NT;
  static_assert(ALL % 64 == 0, "whole waves");
  unsigned off[N];
  int pitch, tail;                                    // bytes from row to row; bytes of a row
  __device__ __forceinline__ void init(long ld, int cols, int tid) {
    pitch = (int)ld * Tl::SZ;                         // at most MAX_PITCH: checked at the entry points
    tail = cols * Tl::SZ;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = tid + i * NT, row = p / Tl::CH, ch = (p % Tl::CH) ^ Tl::swz(row);
      off[i] = ch * 16 < tail ? (unsigned)(row * pitch + ch * 16) : 0x80000000u;
    }
  }
  // p: the tile's first row; rows: valid rows from there on; wave: this thread's wave of the NT / 64
  __device__ __forceinline__ void issue(const T* p, int rows, char* lds, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const int n = min(rows, ROWS);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), (short)0, n > 0 ? (n - 1) * pitch + tail : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL % NT == 0 || i * NT + wave * 64 < ALL) dma16(rs, off[i], (unsigned)(size_t)(lds_ptr_t)(lds + (i * NT + wave * 64) * 16));
#endif
  }
};
// The 4 waves of a work-group own 32 rows (queries; keys for dK and dV) each; or two waves share 32 rows, each walking half of the
// other side, and are joined at the end: twice as many work-groups of half the length, for grids that would leave compute units
// idle or, ragged, make the chip wait for the longest.  ``groups``: work-groups of the first kind; 416 are 1.6 a compute unit.
// Measured over 343, 1183 and 2048 tokens with and without a causal mask (time of the second kind over the first's, ranges over one and two
// maps, bfloat16 and float, heads of 32 to 128):                  128        256        384        448        512        640 groups
//   forward                                                       0.60-0.79  0.69-0.93  0.74-1.06  0.88-1.23  0.90-1.26  0.93-1.18
//   dQ                                                            0.68-0.85  0.75-1.13  0.79-1.45  0.83-1.77  0.93-1.71  1.01-1.65
//   dK dV                                                         0.66-0.83  0.73-1.08  0.84-1.20  0.98-1.37  0.99-1.36  0.96-1.26
// Lengths spread evenly down to a tenth leave half of a forward grid empty: there it crosses at twice as many (640: 0.78-1.07, 960:
// 0.81-1.16), the gradients at as many (480: 0.83-1.54).
__host__ __device__ __forceinline__ int row_waves(long groups) { return groups < 416 ? 2 : 4; }
#define MAX_PITCH (1 << 24)
#define MAX_GROUPS (1L << 24)  // work-groups of 256 in a launch: a grid's work-items are counted in 32 bits
// until at most KEEP of this wave's loads are in flight
template <int KEEP> __device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KEEP) : "memory"); }

__device__ __forceinline__ f32x16 zero16() {
  const f32x16 z = {0};
  return z;
}

// The sum of a few products from ``start`` on.  float: the matrix pipe cuts off what lies below its largest term towards minus
// infinity.  A start far larger than the products (an exponent's maximum) would cost them bits, so the vector pipe adds it at the end
// (777 tokens: dK and dV 1.3e-6 off from such a start, 6e-7 so).  APART, from zero: the products of the upper parts, which lose nothing
// to speak of, have an accumulator of their own beside the small ones; the mean error of an instruction, -3e-8, otherwise adds up over
// the thousands of pairs of a bias table's bucket (its gradient 1.8e-6 off, and 3.5e-7 so).
template <int TY, bool APART = false> struct Products {
  f32x16 sum;
  __device__ __forceinline__ Products(f32x16 start) : sum(start) {}
  __device__ __forceinline__ void add(typename El<TY>::Frag a, typename El<TY>::Frag b) { sum = El<TY>::mma(a, b, sum); }
  __device__ __forceinline__ f32x16 get() const { return sum; }
};
template <bool APART> struct Products<TY_F32, APART> {
  f32x16 rest, sum;            // rest: the start; APART: the small products
  __device__ __forceinline__ Products(f32x16 start) : rest(start), sum(zero16()) {}
  __device__ __forceinline__ void add(Split8 a, Split8 b) {
    if (APART) {
      rest = El<TY_F32>::mma_small(a, b, rest);
      sum = El<TY_F32>::mma_large(a, b, sum);
    } else {
      sum = El<TY_F32>::mma(a, b, sum);
    }
  }
  __device__ __forceinline__ f32x16 get() const { return sum + rest; }
};

// A wave's 32 x COLS result, row li on lane li, to 32 rows of a strided matrix (those below ``rows``, elements below ``cols``): through
// a piece of LDS of the wave's own, so that a store instruction writes whole runs of a row.  Straight from the registers it would
// write 16 bytes to each of 32 rows.
template <int TY, int COLS> struct RowStore {
  typedef typename El<TY>::T T;
  static constexpr int SZ = sizeof(T), PITCH = COLS * SZ + 16, BYTES = 32 * PITCH, PER = COLS * SZ / 16;
  static __device__ __forceinline__ void store(const f32x16 (&v)[COLS / 32], float f, char* lds, T* out, long ld, int rows, int cols, int lane) {
    const int li = lane & 31, half = lane >> 5;
    asm volatile("" ::: "memory");                   // a wave's LDS operations are done in order; the compiler keeps it
#pragma unroll
    for (int d = 0; d < COLS / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = {v[d][4 * g] * f, v[d][4 * g + 1] * f, v[d][4 * g + 2] * f, v[d][4 * g + 3] * f};
        El<TY>::store4((T*)(lds + li * PITCH) + 32 * d + 8 * g + 4 * half, x);
      }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < 32 * PER / 64; ++p) {
      const int row = (p * 64 + lane) / PER, c = (p * 64 + lane) % PER * (16 / SZ);
      const u32x4 x = *reinterpret_cast<const u32x4*>(lds + row * PITCH + c * SZ);
      if (row < rows && c < cols) *reinterpret_cast<u32x4*>(out + row * ld + c) = x;
    }
    asm volatile("" ::: "memory");
  }
};

// eight consecutive elements of a global row as an operand fragment (zero where ``ok`` is false)
template <int TY> __device__ __forceinline__ typename El<TY>::Raw global_raw(const typename El<TY>::T* p, bool ok) {
  typename El<TY>::Raw f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0;
  if (ok) f = *reinterpret_cast<const typename El<TY>::Raw*>(p);
  return f;
}
template <int TY> __device__ __forceinline__ typename El<TY>::Frag global_frag(const typename El<TY>::T* p, bool ok) {
  return El<TY>::frag_of(global_raw<TY>(p, ok));
}

// lambda = exp(w0 . w1) - exp(w2 . w3) + init, by one wave; e1, e2: the two exponentials
template <int TY> __device__ __forceinline__ float diff_lambda(const AttnArgs& a, float& e1, float& e2) {
  const typename El<TY>::T* w = (const typename El<TY>::T*)a.w;
  const int lane = threadIdx.x & 63;
  float s1 = 0.0f, s2 = 0.0f;
  for (int d = lane; d < a.D; d += 64) {
    s1 = fmaf(El<TY>::load(w + d), El<TY>::load(w + a.D + d), s1);
    s2 = fmaf(El<TY>::load(w + 2 * a.D + d), El<TY>::load(w + 3 * a.D + d), s2);
  }
  e1 = expf(wave_sum(s1));
  e2 = expf(wave_sum(s2));
  return e1 - e2 + a.lam_init;
}

__device__ __forceinline__ int clamp_len(const int* len, int b, int most) { return len ? min(max(len[b], 0), most) : most; }
// positions are held in 32 bits: lengths are below 2^29, and a start beyond +- 2^30 sees the same keys at the same (farthest)
// buckets as one there
__device__ __forceinline__ int start_of(const int* start, int b) { return start ? min(max(start[b], -(1 << 30)), 1 << 30) : 0; }

// The bias of head h over distances, in LDS: entry [rel + reach + BIAS_PAD] for |rel| <= reach + BIAS_PAD, in units of log2;
// from ``reach`` on the bucket stays the same.  A tile that comes within ``reach`` of its queries' positions indexes it
// without a clamp: its distances go at most BIAS_PAD further.
#define BIAS_PAD 96
__host__ __device__ __forceinline__ int bias_size(int reach) { return 2 * (reach + BIAS_PAD) + 1; }
template <int TY> __device__ __forceinline__ float bias_log2(const AttnArgs& a, int rel, int h) {
  const int at = min(max(rel, -a.reach), a.reach) + a.reach;
  const float t = El<TY>::load((const typename El<TY>::T*)a.w + (long)a.lut[at] * a.H + h);
  // a type's lowest value stays finite (a row that has nothing else keeps equal weights), an infinity stays one
  const float s = t * LOG2E;
  return (fabsf(s) == INFINITY && fabsf(t) != INFINITY) ? copysignf(3.402823466e38f, s) : s;
}
// A softmax does not see a constant, so what a large bias has in common with a row's maximum is taken off before the score is added, in
// both directions: fma(s, c2, bias - maximum).  (Added first, a value of -1e4 costs a weight 5e-4 of itself, one of -1e6 8 %, and the
// weights of the backward pass no longer sum to one.)  Two limits, in units of log2:
//   BIAS_FOLD   from here on a bias is added first and absorbs the scores: keys that only such a value is left for weigh evenly (a type's
//               lowest value).  Below it a maximum, held in f32, is off by at most 64, and the weights with it by 2^64, which f32 and
//               bfloat16 hold; IEEE half tables end at 2^17.
//   BIAS_LARGE  heads with such a value take their near tiles' largest visible bias off first in the forward pass (one more read and two
//               instructions an element); below it the sum's rounding, 2^-20 of a weight, is that of any score of the size.  So do the
//               far tiles of attn_dkv_kernel, whose scores otherwise start from -maximum and have the far value added at the end.
#define BIAS_FOLD 2147483648.0f
#define BIAS_LARGE 16.0f
// A copy that the compiler takes for another number: branches that each compare it with an unrolled tile's columns otherwise get one set
// of 16 to 32 lane masks ahead of them all, more than the scalar registers hold (5 to 9 % of the training cases).
__device__ __forceinline__ int another(int x) {
  asm("" : "+v"(x));
  return x;
}
// -> whether this thread met a finite value of BIAS_LARGE or more
template <int TY> __device__ __forceinline__ bool fill_bias(const AttnArgs& a, float* tab, int h, int tid, int nt) {
  const int n = bias_size(a.reach);
  bool large = false;
  for (int i = tid; i < n; i += nt) {
    const float t = bias_log2<TY>(a, i - a.reach - BIAS_PAD, h);
    tab[i] = t;
    large |= fabsf(t) >= BIAS_LARGE && fabsf(t) < INFINITY;
  }
  return large;
}

// lets a kernel use up to 158 KB of dynamic LDS on the current device (once a device; 2 KB of the 160 are left for static arrays),
// refuses more
template <auto KERNEL> static int allow_lds(int bytes) {
  static bool done[SGTA_MAX_DEVICES];
  if (bytes > 158 * 1024) return SGTA_EBADARG;
  const int slot = sgta_device_slot();
  if (!done[slot]) {
    const hipError_t e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, 158 * 1024);
    if (e != hipSuccess) return (int)e;
    done[slot] = true;
  }
  return SGTA_OK;
}
