// The scan of decay attention (the mathematics: trl_decay.hip): one kernel template, instantiated for one element type per
// translation unit (trl_decay_f32.hip, trl_decay_bf16.hip, trl_decay_f16.hip).
#pragma once
#include <algorithm>
#include <type_traits>

#include "trl_io.h"

namespace trl_decay {

struct Operand {
  const void *p;
  int64_t st, sn, sh;      // strides of time, env and head, in elements; the head's own dimension is dense
};

struct Scan {
  Operand a, b, c;
  void *out;               // [T, N, H, dc] dense
  const float *decay;
  const void *start;       // [T, N] or null
  const int32_t *lengths;  // [N] or null
  const float *state_in;   // [N, H, ...] or null; transposed: [.., dc, da]
  float *state_out;        // [N, H, da, dc] or null
  float *seg_state;        // [N, H, segs, .., ..] or null (one segment)
  float *seg_coef;         // [N, H, segs]
  int64_t T, N;
  int32_t H, da, dc, segs, seg_len;
  int32_t start_u8, reverse, state_t;
  float s_inter, s_intra, s_state;
};

struct Scans {
  Scan s[3];
};

// `count` scans of equal sizes in one launch; out: the outputs, else every segment's contribution to the state
void launch_f32(const Scans &all, int count, bool out, hipStream_t st);
void launch_bf16(const Scans &all, int count, bool out, hipStream_t st);
void launch_f16(const Scans &all, int count, bool out, hipStream_t st);

// up to so many segments a workgroup joins the contributions before its own by itself: 2 us at 8 of them, against 7 us and a
// launch for the join of all; beyond, what all workgroups read grows with the square of the segments.  (Training passes: 64 heads
// of 64 in bf16, 500 steps in 7 segments: 75 us, joined by the launch 81; 8 heads of 128 in f32, 1,024 steps in 16 segments: by
// the launch 101, by the workgroups 141.)
constexpr int kJoinInside = 8;

inline int tiles_of(int dim) { return (dim + 15) / 16; }

// lambda^n in double, n < 32: each power is rounded to f32 once.  Not zero unless lambda is
__device__ __forceinline__ double power(double lam, int n) {
  const bool zero = lam == 0.0;
  double p = 1.0;
#pragma unroll
  for (int b = 0; b < 5; ++b) {
    if ((n >> b) & 1) p *= lam;
    lam *= lam;
  }
  return p == 0.0 && !zero ? __DBL_MIN__ : p;
}

__device__ __forceinline__ double power_long(double lam, int64_t n) {
  const bool zero = lam == 0.0;
  double p = 1.0;
  for (; n > 0; n >>= 1) {
    if (n & 1) p *= lam;
    lam *= lam;
  }
  return p == 0.0 && !zero ? __DBL_MIN__ : p;
}

// Rounded to f32, and not to zero: what the state is multiplied with, whose infinities stay infinite for ever
__device__ __forceinline__ float not_to_zero(double p) {
  const float f = (float)p;
  return f == 0.f && p != 0.0 ? copysignf(__FLT_DENORM_MIN__, f) : f;
}

// A power of lambda in two parts, for the state (its rounding alone would repeat in the same direction every chunk).  The large
// part is rounded down and the small one above zero, if only by the smallest float: hi s + lo s of an infinite s is s then,
// where parts of different signs, or a small part of zero, would make it a NaN.
__device__ __forceinline__ void two_parts(double p, float &hi, float &lo) {
  hi = not_to_zero(p);
  if ((double)hi > p && hi > __FLT_DENORM_MIN__) hi = __int_as_float(__float_as_int(hi) - 1);
  lo = (float)(p - (double)hi);
  if (p > 0.0) lo = fmaxf(lo, __FLT_DENORM_MIN__);
}

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- operands of the products.  `In` holds four values of k of an input, `Part` those of something computed in f32.
// f32 (and f16, which f32 holds): four 16x16x4 products.
struct Math32 {
  static constexpr bool kShare = true;
  typedef f32x4 In;
  typedef f32x4 Part;      // of an operand that is computed
  static __device__ __forceinline__ f32x4 mma(const f32x4 &a, const f32x4 &b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Part split(const f32x4 &v) { return v; }
  static __device__ __forceinline__ f32x4 mma_right(const In &a, const Part &b, f32x4 c) { return mma(a, b, c); }
  static __device__ __forceinline__ f32x4 mma_left(const Part &a, const In &b, f32x4 c) { return mma(a, b, c); }
  // w c: the right operand of S + b^T (w c)
  static __device__ __forceinline__ Part weigh(const In &c, const float (&w)[4]) {
    return f32x4{c[0] * w[0], c[1] * w[1], c[2] * w[2], c[3] * w[3]};
  }
  // whether a value is not finite (0 times it is a NaN)
  static __device__ __forceinline__ bool bad(const In &u, const In &v) {
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) d = fmaf(u[e], 0.f, fmaf(v[e], 0.f, d));
    return d != 0.f;
  }
};

// bf16: one 16x16x16 product of the inputs as they are; what is computed in f32 goes in as the sum of three bf16 parts, which
// hold its 24 bits whole, so that a product of it is rounded as it is in f32.  (With two parts, 2^-17 of a value is lost: 0.24%
// of a long sequence's outputs then round to the neighbour of the right bf16 value.)  An infinite value in f32 becomes
// inf + NaN: it stays not finite, but comes out as NaN.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));

struct Math16 {
  static constexpr bool kShare = false;
  typedef s16x4 In;
  struct Part {
    s16x4 hi, mid, lo;
  };
  static __device__ __forceinline__ f32x4 mma(const In &a, const In &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ s16x4 round(const f32x4 &v) {
    return __builtin_bit_cast(s16x4, __builtin_convertvector(v, b16x4));
  }
  static __device__ __forceinline__ f32x4 wide(const s16x4 &v) {
    return __builtin_convertvector(__builtin_bit_cast(b16x4, v), f32x4);
  }
  static __device__ __forceinline__ Part split(const f32x4 &v) {
    Part p;
    p.hi = round(v);
    const f32x4 r = v - wide(p.hi);
    p.mid = round(r);
    p.lo = round(r - wide(p.mid));
    return p;
  }
  static __device__ __forceinline__ f32x4 mma_right(const In &a, const Part &b, f32x4 c) {
    return mma(a, b.hi, mma(a, b.mid, mma(a, b.lo, c)));
  }
  static __device__ __forceinline__ f32x4 mma_left(const Part &a, const In &b, f32x4 c) {
    return mma(a.hi, b, mma(a.mid, b, mma(a.lo, b, c)));
  }
  static __device__ __forceinline__ Part weigh(const In &c, const float (&w)[4]) {
    const f32x4 u = wide(c);
    return split(f32x4{u[0] * w[0], u[1] * w[1], u[2] * w[2], u[3] * w[3]});
  }
  // whether an exponent is all ones: bit 15 or 31 after the addition
  static __device__ __forceinline__ uint32_t doubt(const In &v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 u = __builtin_bit_cast(u32x2, v);
    return ((u[0] & 0x7F807F80u) + 0x00800080u) | ((u[1] & 0x7F807F80u) + 0x00800080u);
  }
  static __device__ __forceinline__ bool bad(const In &u, const In &v) { return ((doubt(u) | doubt(v)) & 0x80008000u) != 0; }
};

// ---- four consecutive elements of one step as they are loaded (`raw`: nothing touches them before their chunk's turn, so the
// loads of a chunk fly while the one before it is worked on), and as they lie in LDS: bf16 as it is, the others in f32
template <typename T>
struct Quad {
  typedef Math32 M;
  typedef f32x4 Lds;
  typedef float L;
  uint32_t w[4];
  template <bool VEC>
  __device__ __forceinline__ Lds get() const {
    if constexpr (sizeof(T) == 4) {
      return f32x4{__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3])};
    } else {
      if constexpr (VEC) return f32x4{half(w[0]), half(w[0] >> 16), half(w[1]), half(w[1] >> 16)};
      return f32x4{half(w[0]), half(w[1]), half(w[2]), half(w[3])};
    }
  }
  static __device__ __forceinline__ float half(uint32_t u) { return (float)__builtin_bit_cast(trl_f16, (uint16_t)u); }
};

template <>
struct Quad<trl_bf16> {
  typedef Math16 M;
  typedef s16x4 Lds;
  typedef short L;
  uint32_t w[4];
  template <bool VEC>
  __device__ __forceinline__ Lds get() const {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(s16x4, VEC ? u32x2{w[0], w[1]} : u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)});
  }
};

// `n`: elements of the quad that are inside the row and the chunk (0 .. 4; 0 or 4 with VEC); the others are not read, and zero
// when the quad is staged
template <typename T, bool VEC>
__device__ __forceinline__ void fetch_quad(Quad<T> &q, const T *p, int n) {
  typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type U;
  if constexpr (VEC) {
    if (n > 0) __builtin_memcpy(q.w, p, 4 * sizeof(T));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) q.w[e] = ((const U *)p)[e];
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ typename Quad<T>::Lds quad_of(const Quad<T> &q, int n) {
  typename Quad<T>::Lds v = q.template get<VEC>();
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (VEC ? n > 0 : e < n) ? v[e] : 0;
  return v;
}

constexpr int kColStride = 20;      // LDS: elements between two columns of a transposed tile (16 steps and 4 of padding)

// Where step `row` of column `col` lies in a transposed tile.  The groups of four steps are exchanged by the column's tile, so
// that the 16 quads of a row, which a wave writes at once, fall into different banks (without: 4 writes to a bank, measured
// 65% of the LDS cycles); a reader's 16 columns are of one tile and see one permutation.
__device__ __forceinline__ int col_at(int col, int row) {
  return col * kColStride + ((((row >> 2) ^ (col >> 4)) & 3) << 2) + (row & 3);
}

// LDS: two chunks -- a by rows (16 steps of da + 4), b and c by columns -- and, for the pair products, either their parts
// (kShare) or b by rows too.
// Every wave needs all pair products.  In f32 they would be a third of its matrix instructions (16 of 52 a chunk at 64
// columns), so each wave makes the part of one tile of columns and the parts are added through LDS, behind a second barrier:
// 677 -> 592 us for a training pass over 256 steps of 2,048 heads (540 with the later steps).  Closing a chunk's output behind
// the next chunk's first barrier instead, which saves the second, took 632 (the values carried over spill; 567 with registers
// for three waves a SIMD).  On the bf16 MFMA all pairs cost 4 instructions of half the length, less than the exchange takes.
template <typename T, int KT, bool OUT>
__host__ __device__ constexpr int chunk_elems(int waves) {
  return (OUT ? (Quad<T>::M::kShare ? 1 : 2) * 16 * (16 * KT + 4) : 0) + (16 * KT + 16 * waves) * kColStride;
}
template <typename T, int KT, bool OUT>
constexpr int lds_bytes(int waves) {
  return 2 * chunk_elems<T, KT, OUT>(waves) * (int)sizeof(typename Quad<T>::L) + (OUT && Quad<T>::M::kShare ? KT * 1024 : 0);
}

// Waves of a workgroup, and quads of a (and b) that each of its threads brings.  With 8 tiles of a's dimension a workgroup of 4
// waves takes 64 of c's columns (blockIdx.z), so that two of them share a CU and one works while the other starts, ends or waits.
// Training passes against one workgroup of 8 waves: 160 heads of 64 / 128 in f32, 500 steps 369 -> 276 us, of 128 / 64 345 ->
// 299; 51 heads of 128 in bf16, 301 steps 120 -> 109; 2,048 heads, 128 steps 823 -> 764, in f32 1,028 -> 1,074.
template <int KT>
__host__ __device__ constexpr int quads_of() {
  return KT == 8 ? 2 : 1;
}
template <int KT>
inline int waves_of(int dc) {
  return KT == 8 ? 4 : std::max(KT, tiles_of(dc));
}

// A workgroup carries one (env, head, segment) of one of the scans (blockIdx.y) through time, a wave 16 of c's columns (waves
// past them only help to stage).  KT: 16-column tiles of a's (b's) dimension, which its threads bring in one quad of a and of b
// each (two with 8 tiles), and one of c.  VEC: both dimensions are multiples of four.
// Registers for four waves a SIMD; with 8 tiles for two: at 128 registers S and its operands spill (128 steps of 2,048 heads of
// 128, training: f32 2,098 -> 1,072 us, bf16 1,116 -> 763).  With 6 tiles in f32 for three (heads of 96: 876 -> 815 us; bf16 loses
// there: 691 -> 702), with 5 tiles four are best (heads of 80: f32 608 us against 714 with three, bf16 540 against 628).
// At these bounds 3, 4, 5 and 6 tiles keep 28, 60, 160 and 20 B a lane in scratch in f32, 4, 5 and 6 tiles 32, 128 and 240 B in
// bf16 (VEC; f16 like f32 or less): most of it values of the prologue and the epilogue, kept over the loop.
template <typename T, int KT, bool OUT, bool VEC>
__global__ __launch_bounds__(512, KT == 8 ? 2 : KT == 6 && Quad<T>::M::kShare ? 3 : 4) void k_scan(Scans all) {
  typedef typename Quad<T>::M M;
  typedef typename Quad<T>::Lds V4;
  typedef typename Quad<T>::L L;
  constexpr int ROW = 16 * KT + 4;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  __shared__ int bad_flag[2][8];
  __shared__ uint64_t marks[2][8];
  __shared__ float pw[48], pw_hi[32], pw_lo[32];
  const Scan &s = all.s[blockIdx.y];
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  const int lane = tid & 63, x = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (N H < 2^22: 64-bit divisions are several hundred instructions at the start of every workgroup)
  const uint32_t heads32 = (uint32_t)s.N * (uint32_t)s.H, block_seg = blockIdx.x / heads32, nh32 = blockIdx.x - block_seg * heads32;
  const uint32_t n32 = nh32 / (uint32_t)s.H;
  const int64_t heads = heads32, nh = nh32, n = n32;
  const int h = (int)(nh32 - n32 * (uint32_t)s.H);
  // (the launch that makes contributions has no need of the last segment in its direction of time)
  const int seg = (int)block_seg + (!OUT && s.reverse ? 1 : 0);
  const float decay = s.decay[h];

  const int64_t length = s.lengths ? std::min<int64_t>(std::max<int64_t>(s.lengths[n], 0), s.T) : s.T;
  const int64_t t_lo = (int64_t)seg * s.seg_len;
  const int64_t t_end = std::min<int64_t>(t_lo + s.seg_len, s.T);
  const int64_t t_hi = std::min<int64_t>(t_end, length);      // steps [t_lo, t_hi) of this workgroup
  const int steps = (int)std::max<int64_t>(t_hi - t_lo, 0);
  const int64_t t_first = s.reverse ? t_hi - 1 : t_lo, dir = s.reverse ? -1 : 1;      // step i of the scan: t_first + dir i
  const int off = s.reverse ? 0 : 1;
  const int da = s.da, dc = s.dc;
  constexpr int AQ = quads_of<KT>();
  const int c0 = AQ > 1 ? 16 * waves * (int)blockIdx.z : 0;      // first column of c here

  // this thread's quads: step and column of a and b, step and column of c
  const int arow = tid / (4 * KT), acol = 4 * (tid % (4 * KT));
  const int crow = tid / (4 * waves), ccol = 4 * (tid % (4 * waves));
  const T *pa = (const T *)s.a.p + n * s.a.sn + h * s.a.sh + (t_first + dir * arow) * s.a.st + acol;
  const T *pb = (const T *)s.b.p + n * s.b.sn + h * s.b.sh + (t_first + dir * arow) * s.b.st + acol;
  const T *pc = (const T *)s.c.p + n * s.c.sn + h * s.c.sh + (t_first + dir * crow) * s.c.st + c0 + ccol;
  const int64_t sa = dir * s.a.st, sb = dir * s.b.st, sc = dir * s.c.st;

  // Every quad of a whole chunk is inside its operand: nothing to select when it is staged.  Where that is worth code of its own:
  // bf16 with the usual sizes (128 steps of 2,048 heads of 128: 777 -> 763 us; f32 loses 4% to the longer loop).
  constexpr bool kWhole = VEC && !M::kShare && (KT & (KT - 1)) == 0;
  const bool whole = kWhole && waves * AQ == KT && da == 16 * KT && dc - c0 >= 16 * waves;
  constexpr int kRows = 16 / AQ;      // steps between a thread's quads of a and b
  struct Quads {
    Quad<T> a[AQ], b[AQ], c;
  };
  auto fetch = [&](Quads &q, int at, int cap) {      // the chunk of up to `cap` steps from `at` on (none past the end)
    const int m = std::min(cap, steps - at);
#pragma unroll
    for (int i = 0; i < AQ; ++i) {
      const int na = arow + kRows * i < m ? da - acol : 0;
      if constexpr (OUT) fetch_quad<T, VEC>(q.a[i], pa + (at + kRows * i) * sa, na);
      fetch_quad<T, VEC>(q.b[i], pb + (at + kRows * i) * sb, na);
    }
    fetch_quad<T, VEC>(q.c, pc + at * sc, crow < m ? dc - c0 - ccol : 0);
  };
  // The flags of 64 steps a wave at a time, loaded that many steps ahead; as bits in `marks` once their turn has come.  (Loaded
  // with every chunk their addresses and conversions cost more than they look: 256 steps of 2,048 heads of 64, training, float32
  // flags 554 -> 536 us, uint8 flags, whose conversion waited for the chunk's loads, 600 -> 536.)
  const int marks_len = 64 * waves;
  uint32_t flag = 0;           // as it was loaded
  auto fetch_flag = [&](int at) {
    flag = 0;
    if (s.start != nullptr && at + tid < steps) {
      const int64_t i = (t_first + dir * (at + tid)) * s.N + n;
      flag = s.start_u8 ? ((const uint8_t *)s.start)[i] : ((const uint32_t *)s.start)[i];
    }
  };
  auto lds = [&](int buf) { return (L *)lds_raw + buf * chunk_elems<T, KT, OUT>(waves); };
  f32x4 *const parts = (f32x4 *)((L *)lds_raw + 2 * chunk_elems<T, KT, OUT>(waves));
  // the chunk's m steps into a buffer; whether b or c is not finite
  auto stage = [&](const Quads &q, int buf, int m) {
    L *A = lds(buf), *B = A + 16 * ROW, *BT = A + (OUT ? (M::kShare ? 1 : 2) * 16 * ROW : 0), *CC = BT + 16 * KT * kColStride;
    const bool all = kWhole && whole && m == 16;
    const V4 c = all ? q.c.template get<VEC>() : quad_of<T, VEC>(q.c, crow < m ? dc - c0 - ccol : 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) CC[col_at(ccol, crow) + e * kColStride] = c[e];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < AQ; ++i) {
      const int row = arow + kRows * i, na = row < m ? da - acol : 0;
      const V4 b = all ? q.b[i].template get<VEC>() : quad_of<T, VEC>(q.b[i], na);
      bad |= M::bad(b, c);
      if (AQ > 1 || row < 16) {
        if constexpr (OUT) *(V4 *)(A + row * ROW + acol) = all ? q.a[i].template get<VEC>() : quad_of<T, VEC>(q.a[i], na);
        if constexpr (OUT && !M::kShare) *(V4 *)(B + row * ROW + acol) = b;
#pragma unroll
        for (int e = 0; e < 4; ++e) BT[col_at(acol, row) + e * kColStride] = b[e];
      }
    }
    return bad;
  };

  Quads q = {};
  fetch(q, 0, 16);
  fetch_flag(0);

  // the powers of lambda, by one thread each and to one rounding; zero below the 0th, so that steps after a chunk's end weigh
  // nothing
  const double lam = (double)decay;
  auto powers = [&]() {
    if (tid < 32) {
      const double p = power(lam, tid);
      pw[16 + tid] = not_to_zero(p);
      two_parts(p, pw_hi[tid], pw_lo[tid]);
      if (tid < 16) pw[tid] = 0.f;
    }
  };

  const int lcol = wave * 16 + x, col = c0 + lcol;      // this lane's column of c, of S and of the output
  f32x4 S[KT];
  {
    // state entering the segment, none: zero.  Every lane loads from an address inside it and no value has a branch of its own:
    // through each of those the compiler would carry all of S, and spill
    const int64_t size = (int64_t)da * dc;
    const float *in = s.state_in ? s.state_in + nh * size : nullptr;
    int first = 0, joins = 0;      // contributions still to be joined: segments first, first + dir, ..
    if (s.seg_state != nullptr) {
      if (s.segs > kJoinInside) {
        in = s.seg_state + (nh * s.segs + seg) * size;      // (joined by the launch before)
      } else {
        first = s.reverse ? s.segs - 1 : 0;
        joins = s.reverse ? s.segs - 1 - seg : seg;
      }
    }
    const bool have = OUT && in != nullptr;
    // a state from memory, in S's layout.  Four rows of a column lie side by side when it is read transposed.
    auto load_state = [&](const float *p, f32x4 (&v)[KT]) {
      if (VEC && s.state_t) {
        p += (int64_t)std::min(col, dc - 1) * da;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) __builtin_memcpy(&v[kt], p + std::min(kt * 16 + 4 * g, da - 4), 16);
      } else {
        const int rs = s.state_t ? 1 : dc, cs = s.state_t ? da : 1;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[kt][r] = p[std::min(kt * 16 + 4 * g + r, da - 1) * rs + std::min(col, dc - 1) * cs];
          __builtin_amdgcn_sched_barrier(0);      // (the addresses of all of them do not fit beside S)
        }
      }
    };
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) S[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (OUT) {
      if (have) load_state(in, S);
      f32x4 u[KT];
      const float *p = s.seg_state + (nh * s.segs + first) * size, *pc = s.seg_coef + nh * s.segs + first;
      if (joins > 0) load_state(p, u);
      powers();                // (while those loads are on their way)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[kt][r] = ((int)have & (int)(kt * 16 + 4 * g + r < da) & (int)(col < dc)) ? S[kt][r] : 0.f;
#pragma unroll 1
      for (int i = 0; i < joins; ++i) {
        const float cf = pc[(int)dir * i];      // < 0: a start in that segment
        f32x4 next[KT];
        p += dir * size;
        if (i + 1 < joins) load_state(p, next);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = cf < 0.f ? u[kt][r] : fmaf(cf, S[kt][r], u[kt][r]);
            S[kt][r] = ((int)(kt * 16 + 4 * g + r < da) & (int)(col < dc)) ? w : 0.f;
          }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) u[kt] = next[kt];
      }
    } else {
      powers();
    }
  }

  __syncthreads();
  float w_intra[4], w_inter[4], w_state[4];      // of a whole chunk
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    w_intra[r] = pw[16 + x - 4 * g - r] * s.s_intra;
    w_inter[r] = not_to_zero((double)pw[16 + off + 4 * g + r] * s.s_inter);
    w_state[r] = pw[32 - off - 4 * g - r] * s.s_state;
  }
  const float full_hi = pw_hi[16], full_lo = pw_lo[16];

  const int64_t out_step = dir * heads * dc;
  T *po = OUT ? (T *)s.out + ((t_first + dir * 4 * g) * heads + nh) * dc + col : nullptr;      // step 4 g of the chunk
  bool cut = false;            // a start inside this segment
  int buf = 0;
  int marks_at = -marks_len, marks_buf = 0;      // first step of those in `marks`
  // cap: 16 steps a chunk, or one up to step `until`
#pragma unroll 1
  for (int begin = 0, cap = 16, until = 0; begin < steps; buf ^= 1) {
    const int chunk = std::min(cap, steps - begin);
    const bool bad = __any(stage(q, buf, chunk));
    if (lane == 0) bad_flag[buf][wave] = bad;
    if (begin == marks_at + marks_len) {
      marks_at = begin;
      marks_buf ^= 1;
      const uint64_t bits = __ballot((s.start_u8 ? flag : flag << 1) != 0);      // (-0 is 0)
      if (lane == 0) marks[marks_buf][wave] = bits;
      fetch_flag(begin + marks_len);
    }
    // the other buffers are written only after every wave has passed this barrier
    __syncthreads();
    const int bad_any = bad_flag[buf][std::min(lane, waves - 1)];
    const int mark = ((const uint16_t *)marks[marks_buf])[(begin - marks_at) >> 4];
    const int next_cap = begin + chunk < until ? 1 : 16;
    fetch(q, begin + chunk, next_cap);      // on its way while this chunk is worked on
    const L *A = lds(buf), *B = A + 16 * ROW, *BT = A + (OUT ? (M::kShare ? 1 : 2) * 16 * ROW : 0),
            *CC = BT + 16 * KT * kColStride;
    const V4 C = *(const V4 *)(CC + col_at(lcol, 4 * g));
    f32x4 P = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
    if constexpr (OUT) {
      if (M::kShare && wave < KT) {
#pragma unroll
        for (int i = 0; i < AQ; ++i) {
          const int tile = wave + KT / AQ * i;
          const V4 av = *(const V4 *)(A + x * ROW + tile * 16 + 4 * g);
          V4 bv;
#pragma unroll
          for (int e = 0; e < 4; ++e) bv[e] = BT[col_at(tile * 16 + 4 * g + e, x)];
          parts[tile * 64 + lane] = M::mma(bv, av, P);
        }
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const V4 av = *(const V4 *)(A + x * ROW + kt * 16 + 4 * g);
        if constexpr (!M::kShare) P = M::mma(*(const V4 *)(B + x * ROW + kt * 16 + 4 * g), av, P);
        o = M::mma_right(av, M::split(S[kt]), o);
      }
      if constexpr (M::kShare) {
        if (KT > 1 || waves > 1) __syncthreads();      // (written again only after the next chunk's first barrier)
        P = parts[lane];
#pragma unroll
        for (int kt = 1; kt < KT; ++kt) {
          const f32x4 part = parts[kt * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) P[r] += part[r];
        }
      }
    }
    const bool any_bad = __any(bad_any);
    if (any_bad && chunk > 1) {
      // b or c holds an infinity or a NaN, which a weight of zero would spread over the chunk: its steps one at a time
      cap = 1;
      until = begin + chunk;
      fetch(q, begin, 1);
      continue;
    }
    // bit i: step i of the chunk is a start
    const uint32_t F = ((uint32_t)__builtin_amdgcn_readfirstlane(mark) >> (begin & 15)) & ((1u << chunk) - 1);
    if (chunk == 16 && F == 0) {
      // the usual chunk, whole and of one episode: no branch in it (the loop of a few workgroups is a chain of instructions,
      // some 4,300 cycles a chunk with a branch at every place where chunks differ)
      if constexpr (OUT) {
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = 4 * g + r <= x ? P[r] * w_intra[r] : 0.f;
          o[r] *= w_inter[r];
        }
        o = M::mma_left(M::split(p), C, o);
        if (col < dc) {
#pragma unroll
          for (int r = 0; r < 4; ++r) po[r * out_step] = (T)o[r];
        }
        po += 16 * out_step;
      }
      const typename M::Part wc = M::weigh(C, w_state);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) S[kt][r] = fmaf(S[kt][r], full_hi, S[kt][r] * full_lo);
        S[kt] = M::mma_right(*(const V4 *)(BT + col_at(kt * 16 + x, 4 * g)), wc, S[kt]);
      }
    } else {
      const int m = chunk;
      cut |= F != 0;
      if constexpr (OUT) {
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 4 * g + r;
          const uint32_t le_j = (1u << (j + off)) - 1, le_x = (1u << (x + off)) - 1;
          const bool on = (j <= x) & ((F & le_x & ~le_j) == 0);
          p[r] = on ? P[r] * w_intra[r] : 0.f;
          o[r] = (F & le_j) == 0 ? o[r] * w_inter[r] : 0.f;
        }
        o = M::mma_left(M::split(p), C, o);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((4 * g + r < m) & (col < dc)) po[r * out_step] = (T)o[r];
        po += m * out_step;
      }
      // steps that a start keeps from the chunk's end weigh nothing (b and c are finite, or this is one step alone)
      float ws[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        ws[e] = (F & ~((1u << (4 * g + e + off)) - 1)) == 0 ? pw[16 + m - off - 4 * g - e] * s.s_state : 0.f;
      const float hi = pw_hi[m], lo = pw_lo[m];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[kt][r] = F == 0 ? fmaf(S[kt][r], hi, S[kt][r] * lo) : 0.f;
      // (one step alone whose own start cuts it off -- backward in time -- leaves nothing, whatever c holds)
      if (!any_bad || off == 1 || F == 0) {
        const typename M::Part wc = M::weigh(C, ws);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
          S[kt] = M::mma_right(*(const V4 *)(BT + col_at(kt * 16 + x, 4 * g)), wc, S[kt]);
      }
      if (any_bad) {           // rows past da: 0 times a value that is not finite
        int rows = da - 4 * g;
        asm volatile("" : "+v"(rows));      // (its comparisons are made here, not kept over the loop)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kt * 16 + r >= rows) S[kt][r] = 0.f;
      }
    }
    begin += chunk;
    cap = next_cap;
  }

  // the state left behind: the caller's at the end of time, or this segment's contribution
  float *left = nullptr;
  if (!OUT) {
    left = s.seg_state + (nh * s.segs + seg) * da * dc;
    if (tid == 0 && c0 == 0) s.seg_coef[nh * s.segs + seg] = cut ? -1.f : not_to_zero(power_long(lam, steps));
  } else if (s.state_out != nullptr && seg == (s.reverse ? 0 : s.segs - 1)) {
    left = s.state_out + nh * da * dc;
  }
  if (left != nullptr) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = kt * 16 + 4 * g + r;
        if ((row < da) & (col < dc)) left[row * dc + col] = S[kt][r];
      }
  }
  if (OUT) {                   // steps past the sequence's end
    for (int64_t t = std::max<int64_t>(t_lo, length) + g; t < t_end; t += 4)
      if (col < dc) ((T *)s.out)[(t * heads + nh) * dc + col] = (T)0.f;
  }
}

template <typename T, int KT, bool OUT, bool VEC>
void launch_k(const Scans &s, dim3 grid, hipStream_t st) {
  const int waves = waves_of<KT>(s.s[0].dc);
  if (KT == 8) grid.z = (tiles_of(s.s[0].dc) + waves - 1) / waves;
  const int bytes = lds_bytes<T, KT, OUT>(waves);
  if (bytes > 48 * 1024)      // (per device and cheap; a refusal shows at the launch)
    (void)hipFuncSetAttribute((const void *)k_scan<T, KT, OUT, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  k_scan<T, KT, OUT, VEC><<<grid, 64 * waves, bytes, st>>>(s);
}

template <typename T, bool OUT, bool VEC>
void launch_t(const Scans &s, dim3 grid, hipStream_t st) {
  switch (tiles_of(s.s[0].da)) {
    case 1: return launch_k<T, 1, OUT, VEC>(s, grid, st);
    case 2: return launch_k<T, 2, OUT, VEC>(s, grid, st);
    case 3: return launch_k<T, 3, OUT, VEC>(s, grid, st);
    case 4: return launch_k<T, 4, OUT, VEC>(s, grid, st);
    case 5: return launch_k<T, 5, OUT, VEC>(s, grid, st);
    case 6: return launch_k<T, 6, OUT, VEC>(s, grid, st);
    default: return launch_k<T, 8, OUT, VEC>(s, grid, st);      // (7 tiles too)
  }
}

template <typename T>
void launch(const Scans &all, int count, bool out, hipStream_t st) {
  const Scan &f = all.s[0];
  const dim3 grid((unsigned)(f.N * f.H * (out ? f.segs : f.segs - 1)), count);
  const bool vec = f.da % 4 == 0 && f.dc % 4 == 0;
  if (out && vec)
    launch_t<T, true, true>(all, grid, st);
  else if (out)
    launch_t<T, true, false>(all, grid, st);
  else if (vec)
    launch_t<T, false, true>(all, grid, st);
  else
    launch_t<T, false, false>(all, grid, st);
}

}  // namespace
}  // namespace trl_decay
