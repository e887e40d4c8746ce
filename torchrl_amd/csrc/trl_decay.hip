// Linear attention with a decay per head: the memory over time of a policy or value network on rollouts [T, N, .].  (The
// reference's networks see one observation at a time, torchrl/contrib/models.py:6-147; this is the layer that lets them
// remember.)  For every env n and head h, with lambda = decay[h] and S a [Dk, Dv] matrix:
//     S_t = (start_t ? 0 : lambda S_{t-1}) + k_t v_t^T,        o_t = scale q_t^T S_t.
//
// Chunked form.  Over a chunk of m <= 16 steps that begins with state S, step i of it gives
//     o_i = scale (lambda^{i+1} q_i^T S + sum_{j <= i} lambda^{i-j} (q_i . k_j) v_j),
//     S'  = lambda^m S + sum_j lambda^{m-1-j} k_j v_j^T
// (terms across a start drop out), four small matrix products instead of 16 dependent rank-one updates.
//
// Gradients.  With R_t = (start_{t+1} ? 0 : lambda R_{t+1}) + scale q_t do_t^T:  dq_t = scale S_t do_t, dk_t = R_t v_t,
// dv_t = R_t^T k_t.  Each is the forward's own recurrence on other operands -- dq: (do, v, k) forward in time with S^T;
// dk: (v, do, q) and dv: (k, q, do) backward in time -- so ONE kernel computes the output and the three gradients.  Its
// operands are called a (the q role), b (the k role) and c (the v role) below.
//
// One wave carries one (env, head, group of c's columns) through time with S in MFMA accumulators: 16 steps a turn, all
// products on the exact-f32 16x16x4 MFMA.  Every accumulator is used where it lies: lane (g = lane / 16, x = lane % 16) of a
// result tile holds rows 4g .. 4g + 3 of column x, which is just what the same instruction takes as an operand with k = 4g + e
// (the sum over k may run in any order as long as both operands agree).  So the pair products are made transposed
// (P^T = b a^T: the next product's left operand) and S multiplies from the right, with no exchange between lanes and no LDS.
//
// Few rows: time is cut into segments.  A first launch makes every segment's own contribution to the state, a second joins
// them in order (state entering segment s + 1 = lambda^len state entering s + contribution), a third runs the segments.
//
// Values that are not finite stay where the recurrence puts them: masks are selections, never products with zero -- except
// of b's and c's steps inside a chunk, so a chunk whose b or c holds an infinity or a NaN is taken one step at a time.
#include <algorithm>
#include <type_traits>

#include "trl_io.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kMaxDim = 128;

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

// lambda^n in double, n < 32: each power is rounded to f32 once
__device__ __forceinline__ double power(double lam, int n) {
  double p = 1.0;
#pragma unroll
  for (int b = 0; b < 5; ++b) {
    if ((n >> b) & 1) p *= lam;
    lam *= lam;
  }
  return p;
}

__device__ double power_long(double lam, int64_t n) {
  double p = 1.0;
  for (; n > 0; n >>= 1) {
    if (n & 1) p *= lam;
    lam *= lam;
  }
  return p;
}

// four consecutive elements of a row from column col on, zero past the row's end (the single-step kernel)
template <typename T>
__device__ __forceinline__ void load4(const T *row, int col, int dim, bool live, float (&f)[4]) {
  if (live && col + 4 <= dim) {
    T t[4];
    __builtin_memcpy(t, row + col, 4 * sizeof(T));
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = live && col + e < dim ? (float)row[col + e] : 0.f;
  }
}

__device__ __forceinline__ bool not_finite(float v) { return !(__builtin_fabsf(v) <= 3.402823466e38f); }

// ---- operands of the products.  `In` holds four values of k of an input, `Part` those of something computed in f32.
// f32 (and f16, which f32 holds): four 16x16x4 products.
struct Math32 {
  typedef f32x4 In;
  typedef f32x4 Part;
  static __device__ __forceinline__ f32x4 mma(const f32x4 &a, const f32x4 &b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Part split(const f32x4 &v) { return v; }
  static __device__ __forceinline__ f32x4 mma_right(const In &a, const Part &b, f32x4 c) { return mma(a, b, c); }
  static __device__ __forceinline__ f32x4 mma_left(const Part &a, const In &b, f32x4 c) { return mma(a, b, c); }
  // s + b^T (w c)
  static __device__ __forceinline__ In weigh(const In &c, const float (&w)[4]) {
    return f32x4{c[0] * w[0], c[1] * w[1], c[2] * w[2], c[3] * w[3]};
  }
  static __device__ __forceinline__ f32x4 mma_state(const In &b, const In &wc, f32x4 s) { return mma(b, wc, s); }
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ bool bad(const In &v) {
    return (int)not_finite(v[0]) | (int)not_finite(v[1]) | (int)not_finite(v[2]) | (int)not_finite(v[3]);
  }
};

// bf16: one 16x16x16 product of the inputs as they are; what is computed in f32 goes in as a sum of bf16 parts, two of them
// (relative error 2^-17, under a bf16 output's 2^-9) or three (2^-25) for the state, which is returned in f32.  (An infinite
// value in f32 becomes inf + NaN: it stays not finite, but comes out as NaN.)
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));

struct Math16 {
  typedef s16x4 In;
  struct Part {
    s16x4 hi, lo;
  };
  struct Part3 {
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
    p.lo = round(v - wide(p.hi));
    return p;
  }
  static __device__ __forceinline__ f32x4 mma_right(const In &a, const Part &b, f32x4 c) {
    return mma(a, b.hi, mma(a, b.lo, c));
  }
  static __device__ __forceinline__ f32x4 mma_left(const Part &a, const In &b, f32x4 c) {
    return mma(a.hi, b, mma(a.lo, b, c));
  }
  static __device__ __forceinline__ Part3 weigh(const In &c, const float (&w)[4]) {
    const f32x4 u = wide(c);
    const f32x4 v = {u[0] * w[0], u[1] * w[1], u[2] * w[2], u[3] * w[3]};
    Part3 p;
    p.hi = round(v);
    const f32x4 r = v - wide(p.hi);
    p.mid = round(r);
    p.lo = round(r - wide(p.mid));
    return p;
  }
  static __device__ __forceinline__ f32x4 mma_state(const In &b, const Part3 &wc, f32x4 s) {
    return mma(b, wc.hi, mma(b, wc.mid, mma(b, wc.lo, s)));
  }
  static __device__ __forceinline__ float value(short v) { return __uint_as_float((uint32_t)(uint16_t)v << 16); }
  static __device__ __forceinline__ bool bad(const In &v) {
    bool b = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) b |= (v[e] & 0x7F80) == 0x7F80;
    return b;
  }
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

struct Scans {
  Scan s[3];
};

constexpr int kColStride = 20;      // LDS: elements between two columns of a transposed tile (16 steps and 4 of padding)

// LDS elements of one chunk: a and b by rows (16 steps of da + 4), b and c by columns
template <int KT, bool OUT>
__host__ __device__ constexpr int chunk_elems(int waves) {
  return (OUT ? 2 * 16 * (16 * KT + 4) : 0) + (16 * KT + 16 * waves) * kColStride;
}

// A workgroup carries one (env, head, segment) of one of the scans (blockIdx.y) through time, a wave 16 of c's columns (waves
// past them only help to stage).  KT: 16-column tiles of a's (b's) dimension, at most the workgroup's waves: every thread brings
// one quad of a, of b and of c.  VEC: both dimensions are multiples of four.
template <typename T, int KT, bool OUT, bool VEC>
__global__ __launch_bounds__(512, 4) void k_scan(Scans all) {
  typedef typename Quad<T>::M M;
  typedef typename Quad<T>::Lds V4;
  typedef typename Quad<T>::L L;
  constexpr int ROW = 16 * KT + 4;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  __shared__ int bad_flag[2][8];
  const Scan &s = all.s[blockIdx.y];
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  const int lane = tid & 63, x = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t heads = s.N * s.H;
  const int64_t nh = blockIdx.x % heads;
  // (the launch that makes contributions has no need of the last segment in its direction of time)
  const int seg = (int)(blockIdx.x / heads) + (!OUT && s.reverse ? 1 : 0);
  const int64_t n = nh / s.H;
  const int h = (int)(nh % s.H);

  const int64_t length = s.lengths ? std::min<int64_t>(std::max<int64_t>(s.lengths[n], 0), s.T) : s.T;
  const int64_t t_lo = (int64_t)seg * s.seg_len;
  const int64_t t_end = std::min<int64_t>(t_lo + s.seg_len, s.T);
  const int64_t t_hi = std::min<int64_t>(t_end, length);      // steps [t_lo, t_hi) of this workgroup
  const int steps = (int)std::max<int64_t>(t_hi - t_lo, 0);
  const int64_t t_first = s.reverse ? t_hi - 1 : t_lo, dir = s.reverse ? -1 : 1;      // step i of the scan: t_first + dir i
  const int off = s.reverse ? 0 : 1;
  const int da = s.da, dc = s.dc;

  // this thread's quads: step and column of a and b, step and column of c
  const int arow = tid < 64 * KT ? tid / (4 * KT) : 16, acol = 4 * (tid % (4 * KT));
  const int crow = tid / (4 * waves), ccol = 4 * (tid % (4 * waves));
  const T *pa = (const T *)s.a.p + n * s.a.sn + h * s.a.sh + (t_first + dir * arow) * s.a.st + acol;
  const T *pb = (const T *)s.b.p + n * s.b.sn + h * s.b.sh + (t_first + dir * arow) * s.b.st + acol;
  const T *pc = (const T *)s.c.p + n * s.c.sn + h * s.c.sh + (t_first + dir * crow) * s.c.st + ccol;
  const int64_t sa = 16 * dir * s.a.st, sb = 16 * dir * s.b.st, sc = 16 * dir * s.c.st;

  Quad<T> qa = {}, qb = {}, qc = {};
  float flag = 0.f;
  auto fetch = [&](int done, int m) {      // the next chunk, of m steps; advances the pointers
    const int na = arow < m ? da - acol : 0, nc = crow < m ? dc - ccol : 0;
    if constexpr (OUT) fetch_quad<T, VEC>(qa, pa, na);
    fetch_quad<T, VEC>(qb, pb, na);
    fetch_quad<T, VEC>(qc, pc, nc);
    pa += sa, pb += sb, pc += sc;
    if (s.start != nullptr && x < m) {
      const int64_t at = (t_first + dir * (done + x)) * s.N + n;
      flag = s.start_u8 ? (float)((const uint8_t *)s.start)[at] : ((const float *)s.start)[at];
    }
  };
  auto lds = [&](int buf) { return (L *)lds_raw + buf * chunk_elems<KT, OUT>(waves); };
  // the chunk's m steps (one < 0), or its step `one` alone as the first of a chunk of its own
  auto stage = [&](int buf, int m, int one) {
    L *A = lds(buf), *B = A + (OUT ? 16 * ROW : 0), *BT = B + (OUT ? 16 * ROW : 0), *CT = BT + 16 * KT * kColStride;
    bool bad = false;
    if (KT >= 8 || tid < 64 * KT) {
      const int na = (one < 0 ? arow < m : arow == one) ? da - acol : 0, row = one < 0 ? arow : (arow - one) & 15;
      if constexpr (OUT) *(V4 *)(A + row * ROW + acol) = quad_of<T, VEC>(qa, na);
      const V4 v = quad_of<T, VEC>(qb, na);
      if constexpr (OUT) *(V4 *)(B + row * ROW + acol) = v;
#pragma unroll
      for (int e = 0; e < 4; ++e) BT[(acol + e) * kColStride + row] = v[e];
      bad = M::bad(v);
    }
    const int nc = (one < 0 ? crow < m : crow == one) ? dc - ccol : 0, row = one < 0 ? crow : (crow - one) & 15;
    const V4 v = quad_of<T, VEC>(qc, nc);
#pragma unroll
    for (int e = 0; e < 4; ++e) CT[(ccol + e) * kColStride + row] = v[e];
    bad = __any((int)bad | (int)M::bad(v));
    if (lane == 0) bad_flag[buf][wave] = bad;
  };

  if (steps > 0) fetch(0, std::min(16, steps));

  const int ccolx = wave * 16 + x;      // this lane's column of c, of S and of the output
  f32x4 S[KT];
  {
    // state entering the segment: the caller's, or the joined contributions of the segments before it
    const float *in = s.seg_state ? s.seg_state + (nh * s.segs + seg) * da * dc : s.state_in;
    if (s.seg_state == nullptr && in != nullptr) in += nh * da * dc;
    const int64_t rs = s.state_t ? 1 : dc, cs = s.state_t ? da : 1;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = kt * 16 + 4 * g + r;
        S[kt][r] = 0.f;
        if (OUT && in != nullptr) {
          const float v = in[std::min(row, da - 1) * rs + std::min(ccolx, dc - 1) * cs];
          S[kt][r] = ((row < da) & (ccolx < dc)) ? v : 0.f;
        }
      }
  }

  const double lam = (double)s.decay[h];
  float w_intra[4], w_inter[4], w_state[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = 4 * g + r;
    w_intra[r] = j <= x ? (float)power(lam, x - j) * s.s_intra : 0.f;
    w_inter[r] = (float)power(lam, j + off) * s.s_inter;
    w_state[r] = (float)power(lam, 16 - off - j) * s.s_state;
  }
  const double full = power(lam, 16);
  const float full_hi = (float)full, full_lo = (float)(full - (double)full_hi);

  bool cut = false;            // a start inside this segment
  int chunk = std::min(16, steps), buf = 0, one = -1;
#pragma unroll 1
  for (int begin = 0; begin < steps; buf ^= 1) {
    stage(buf, chunk, one);
    uint32_t F = 0;            // bit i: step i of the chunk is a start
    if (s.start != nullptr) F = (uint32_t)__ballot((flag != 0.f) & (lane < chunk));
    // one barrier a chunk: the other buffer is written only after every wave has passed this one
    __syncthreads();
    const bool any_bad = __any(bad_flag[buf][std::min(lane, waves - 1)]);
    if (any_bad && chunk > 1 && one < 0) {
      // b or c holds an infinity or a NaN, which a weight of zero would spread over the chunk: its steps one at a time
      one = 0;
      continue;
    }
    const int m = one < 0 ? chunk : 1, done = begin + std::max(one, 0);
    if (one >= 0) F = (F >> one) & 1;
    cut |= F != 0;
    if (one < 0 || one == chunk - 1) {
      begin += chunk;
      chunk = std::min(16, steps - begin);
      one = -1;
      if (begin < steps) fetch(begin, chunk);
    } else {
      ++one;
    }
    const L *A = lds(buf), *B = A + (OUT ? 16 * ROW : 0), *BT = B + (OUT ? 16 * ROW : 0),
            *CT = BT + 16 * KT * kColStride;
    const V4 C = *(const V4 *)(CT + ccolx * kColStride + 4 * g);
    if constexpr (OUT) {
      f32x4 P = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const V4 av = *(const V4 *)(A + x * ROW + kt * 16 + 4 * g), bv = *(const V4 *)(B + x * ROW + kt * 16 + 4 * g);
        P = M::mma(bv, av, P);
        o = M::mma_right(av, M::split(S[kt]), o);
      }
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
      T *po = (T *)s.out + ((t_first + dir * (done + 4 * g)) * heads + nh) * dc + ccolx;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if ((4 * g + r < m) & (ccolx < dc)) po[r * dir * heads * dc] = (T)o[r];
    }
    float hi = full_hi, lo = full_lo, ws[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[e] = w_state[e];
    if (m != 16) {
      const double pm = power(lam, m);
      hi = (float)pm;
      lo = (float)(pm - (double)hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) ws[e] = (float)power(lam, std::max(m - off - (4 * g + e), 0)) * s.s_state;
    }
    // steps that a start keeps from the chunk's end weigh nothing (b and c are finite, or this is one step alone)
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[e] = (F & ~((1u << (4 * g + e + off)) - 1)) == 0 ? ws[e] : 0.f;
    if (F != 0) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) S[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
    } else {
      // (lambda^m in two parts: its rounding would otherwise repeat in the same direction every chunk)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[kt][r] = fmaf(S[kt][r], hi, S[kt][r] * lo);
    }
    // (one step alone whose own start cuts it off -- backward in time -- leaves nothing, whatever c holds)
    if (!any_bad || off == 1 || F == 0) {
      const auto wc = M::weigh(C, ws);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const V4 bt = *(const V4 *)(BT + (kt * 16 + x) * kColStride + 4 * g);
        S[kt] = M::mma_state(bt, wc, S[kt]);
      }
    }
    if (any_bad) {             // rows past da: 0 times a value that is not finite
      int rows = da - 4 * g;
      asm volatile("" : "+v"(rows));      // (its comparisons are made here, not kept over the loop)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (kt * 16 + r >= rows) S[kt][r] = 0.f;
    }
  }

  // the state left behind: the caller's at the end of time, or this segment's contribution
  float *left = nullptr;
  if (!OUT) {
    left = s.seg_state + (nh * s.segs + seg) * da * dc;
    if (tid == 0) s.seg_coef[nh * s.segs + seg] = cut ? -1.f : (float)power_long(lam, steps);
  } else if (s.state_out != nullptr && seg == (s.reverse ? 0 : s.segs - 1)) {
    left = s.state_out + nh * da * dc;
  }
  if (left != nullptr) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = kt * 16 + 4 * g + r;
        if ((row < da) & (ccolx < dc)) left[(int64_t)row * dc + ccolx] = S[kt][r];
      }
  }
  if (OUT) {                   // steps past the sequence's end
    for (int64_t t = std::max<int64_t>(t_lo, length) + g; t < t_end; t += 4)
      if (ccolx < dc) ((T *)s.out)[(t * heads + nh) * dc + ccolx] = (T)0.f;
  }
}

// seg_state[s]: contribution of segment s -> state entering segment s, in the scan's direction.  coef < 0: a start in it.
__global__ __launch_bounds__(kThreads) void k_join(float *__restrict__ seg_state, const float *__restrict__ seg_coef,
                                                   const float *__restrict__ state_in, int64_t heads, int64_t size,
                                                   int segs, int reverse) {
  const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (e >= heads * size) return;
  const int64_t nh = e / size;
  float *p = seg_state + nh * segs * size + (e - nh * size);
  const float *coef = seg_coef + nh * segs;
  float cur = state_in ? state_in[e] : 0.f;
  const int first = reverse ? segs - 1 : 0, dir = reverse ? -1 : 1;
  for (int i0 = 0; i0 < segs; i0 += 8) {
    float u[8], cf[8];         // eight contributions in flight
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool on = i0 + i < segs - 1;      // (the last one moves nothing on)
      const int sg = first + dir * (i0 + i);
      u[i] = on ? p[sg * size] : 0.f;
      cf[i] = on ? coef[sg] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i < segs) p[(first + dir * (i0 + i)) * size] = cur;
      cur = cf[i] < 0.f ? u[i] : fmaf(cf[i], cur, u[i]);
    }
  }
}

// one step: a workgroup per (env, head); LC lanes hold four columns each, the others share out the rows
template <typename T, int LC>
__global__ __launch_bounds__(kThreads) void k_step(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                   const float *__restrict__ decay, const void *__restrict__ start,
                                                   int start_u8, const float *state_in, int64_t heads, int32_t H, int32_t dk,
                                                   int32_t dv, float scale, T *__restrict__ out, float *state_out) {
  constexpr int RL = kThreads / LC;
  __shared__ float part[RL][LC * 4];
  const int64_t nh = blockIdx.x;
  const int h = (int)(nh % H);
  const int64_t n = nh / H;
  const int lc = threadIdx.x % LC, rl = threadIdx.x / LC, col = lc * 4;
  bool fresh = false;
  if (start != nullptr) fresh = start_u8 ? ((const uint8_t *)start)[n] != 0 : ((const float *)start)[n] != 0.f;
  const float lam = decay[h];
  float vv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
  load4(v + nh * dv, col, dv, true, vv);
  for (int r = rl; r < dk; r += RL) {
    const float kr = (float)k[nh * dk + r], qr = (float)q[nh * dk + r];
    const int64_t at = (nh * dk + r) * dv;
    float s[4];
    load4(state_in + at, col, dv, !fresh, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = fmaf(lam, s[e], kr * vv[e]);
      acc[e] = fmaf(qr, s[e], acc[e]);
    }
    if (col + 4 <= dv)
      __builtin_memcpy(state_out + at + col, s, 16);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < dv) state_out[at + col + e] = s[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[rl][col + e] = acc[e];
  __syncthreads();
  if (threadIdx.x < dv) {
    float o = 0.f;
    for (int i = 0; i < RL; ++i) o += part[i][threadIdx.x];
    out[nh * dv + threadIdx.x] = (T)(o * scale);
  }
}

int tiles_of(int dim) { return (dim + 15) / 16; }

// time segments: enough workgroups to fill the chip, of at least 64 steps each
void segments(int64_t T, int64_t heads, int *segs, int *seg_len) {
  int64_t want = heads > 0 ? trl_cdiv(512, heads) : 1;
  want = std::max<int64_t>(1, std::min<int64_t>(want, T / 64));
  const int64_t len = std::max<int64_t>(16, trl_cdiv(trl_cdiv(T, want), 16) * 16);
  *seg_len = (int)len;
  *segs = (int)std::max<int64_t>(1, trl_cdiv(T, len));
}

template <typename T, int KT, bool OUT, bool VEC>
void scan_launch_k(const Scans &s, dim3 grid, int waves, hipStream_t st) {
  const size_t bytes = (size_t)2 * chunk_elems<KT, OUT>(waves) * sizeof(typename Quad<T>::L);
  if (bytes > 48 * 1024)      // (per device and cheap; a refusal shows at the launch)
    (void)hipFuncSetAttribute((const void *)k_scan<T, KT, OUT, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  k_scan<T, KT, OUT, VEC><<<grid, 64 * waves, bytes, st>>>(s);
}

template <typename T, bool OUT, bool VEC>
void scan_launch_t(const Scans &s, int kt, dim3 grid, int waves, hipStream_t st) {
  switch (kt) {
    case 1: return scan_launch_k<T, 1, OUT, VEC>(s, grid, waves, st);
    case 2: return scan_launch_k<T, 2, OUT, VEC>(s, grid, waves, st);
    case 3: return scan_launch_k<T, 3, OUT, VEC>(s, grid, waves, st);
    case 4: return scan_launch_k<T, 4, OUT, VEC>(s, grid, waves, st);
    case 5: return scan_launch_k<T, 5, OUT, VEC>(s, grid, waves, st);
    case 6: return scan_launch_k<T, 6, OUT, VEC>(s, grid, waves, st);
    default: return scan_launch_k<T, 8, OUT, VEC>(s, grid, waves, st);      // (7 tiles too)
  }
}

// `count` scans of equal sizes in one launch
void scan_launch(const Scans &all, int count, int32_t dtype, bool out, hipStream_t st) {
  const Scan &f = all.s[0];
  const dim3 grid((unsigned)(f.N * f.H * (out ? f.segs : f.segs - 1)), count);
  const int kt = tiles_of(f.da), waves = std::max(kt == 7 ? 8 : kt, tiles_of(f.dc));
  const bool vec = f.da % 4 == 0 && f.dc % 4 == 0;
  TRL_FOR_DTYPE(dtype, {
    if (out && vec)
      scan_launch_t<T, true, true>(all, kt, grid, waves, st);
    else if (out)
      scan_launch_t<T, true, false>(all, kt, grid, waves, st);
    else if (vec)
      scan_launch_t<T, false, true>(all, kt, grid, waves, st);
    else
      scan_launch_t<T, false, false>(all, kt, grid, waves, st);
  });
}

void join_launch(const Scan &s, hipStream_t st) {
  const int64_t heads = s.N * s.H, size = (int64_t)s.da * s.dc;
  k_join<<<(int)trl_cdiv(heads * size, kThreads), kThreads, 0, st>>>(s.seg_state, s.seg_coef, s.state_in, heads, size, s.segs,
                                                                    s.reverse);
}

int decay_check(const char *fn, int64_t T, int64_t N, int32_t H, int32_t dk, int32_t dv, int32_t dtype) {
  TRL_REQUIRE(trl_float_dtype(dtype), "%s: dtype %d is not f32, bf16 or f16", fn, (int)dtype);
  TRL_REQUIRE(T >= 0 && N >= 0 && H >= 1, "%s: bad shape T=%lld N=%lld H=%d", fn, (long long)T, (long long)N, (int)H);
  TRL_REQUIRE(dk >= 1 && dk <= kMaxDim && dv >= 1 && dv <= kMaxDim, "%s: head sizes must be in [1, %d], got %d and %d", fn,
              kMaxDim, (int)dk, (int)dv);
  TRL_REQUIRE(T < (1ll << 30) && N < (1ll << 22) / H, "%s: too many steps or heads: T=%lld N=%lld H=%d", fn, (long long)T,
              (long long)N, (int)H);
  return TRL_OK;
}

int64_t seg_floats(int64_t heads, int segs, int32_t dk, int32_t dv) {
  return segs > 1 ? heads * segs * ((int64_t)dk * dv + 1) : 0;
}

Operand operand(const void *p, const int64_t *strides) { return {p, strides[0], strides[1], strides[2]}; }

}  // namespace

extern "C" int64_t trl_decay_attention_workspace_bytes(int64_t T, int64_t N, int32_t H, int32_t dk, int32_t dv,
                                                       int32_t backward) {
  if (decay_check("trl_decay_attention_workspace_bytes", T, N, H, dk, dv, TRL_F32)) return TRL_EINVAL;
  int segs, len;
  segments(T, N * H, &segs, &len);
  return 4 * seg_floats(N * H, segs, dk, dv) * (backward ? 2 : 1);
}

extern "C" int trl_decay_attention_fwd(const void *q, const void *k, const void *v, const int64_t *strides,
                                       const float *decay, const void *start, int32_t start_dtype, const int32_t *lengths,
                                       const float *state_in, int64_t T, int64_t N, int32_t H, int32_t dk, int32_t dv,
                                       int32_t dtype, double scale, void *out, float *state_out, void *workspace,
                                       void *stream) {
  const char *fn = "trl_decay_attention_fwd";
  if (int rc = decay_check(fn, T, N, H, dk, dv, dtype)) return rc;
  TRL_REQUIRE(start == nullptr || start_dtype == TRL_F32 || start_dtype == TRL_U8, "%s: start must be f32 or u8", fn);
  if (N == 0) return TRL_OK;
  TRL_REQUIRE(decay != nullptr && strides != nullptr && state_out != nullptr, "%s: null pointer", fn);
  TRL_REQUIRE(T == 0 || (q != nullptr && k != nullptr && v != nullptr && out != nullptr), "%s: null pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  Scan s = {};
  s.a = operand(q, strides);
  s.b = operand(k, strides + 3);
  s.c = operand(v, strides + 6);
  s.out = out;
  s.decay = decay;
  s.start = start;
  s.start_u8 = start_dtype == TRL_U8;
  s.lengths = lengths;
  s.state_in = state_in;
  s.state_out = state_out;
  s.T = T;
  s.N = N;
  s.H = H;
  s.da = dk;
  s.dc = dv;
  s.s_inter = s.s_intra = (float)scale;
  s.s_state = 1.f;
  segments(T, N * H, &s.segs, &s.seg_len);
  if (s.segs > 1) {
    TRL_REQUIRE(workspace != nullptr, "%s: null workspace", fn);
    s.seg_state = (float *)workspace;
    s.seg_coef = s.seg_state + N * H * s.segs * (int64_t)dk * dv;
    scan_launch(Scans{{s}}, 1, dtype, false, st);
    TRL_CHECK_LAUNCH(fn);
    join_launch(s, st);
    TRL_CHECK_LAUNCH(fn);
  }
  scan_launch(Scans{{s}}, 1, dtype, true, st);
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}

extern "C" int trl_decay_attention_bwd(const void *gy, const float *gstate, const void *q, const void *k, const void *v,
                                       const int64_t *strides, const float *decay, const void *start, int32_t start_dtype,
                                       const int32_t *lengths, const float *state_in, int64_t T, int64_t N, int32_t H,
                                       int32_t dk, int32_t dv, int32_t dtype, double scale, void *dq, void *dk_out,
                                       void *dv_out, float *dstate, void *workspace, void *stream) {
  const char *fn = "trl_decay_attention_bwd";
  if (int rc = decay_check(fn, T, N, H, dk, dv, dtype)) return rc;
  TRL_REQUIRE(start == nullptr || start_dtype == TRL_F32 || start_dtype == TRL_U8, "%s: start must be f32 or u8", fn);
  if (N == 0) return TRL_OK;
  TRL_REQUIRE(decay != nullptr && strides != nullptr, "%s: null pointer", fn);
  TRL_REQUIRE(T == 0 || (gy != nullptr && q != nullptr && k != nullptr && v != nullptr && dq != nullptr &&
                         dk_out != nullptr && dv_out != nullptr),
              "%s: null pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t gs[3] = {N * H * (int64_t)dv, H * (int64_t)dv, dv};
  const Operand oq = operand(q, strides), ok = operand(k, strides + 3), ov = operand(v, strides + 6), og = operand(gy, gs);
  Scan s = {};
  s.decay = decay;
  s.start = start;
  s.start_u8 = start_dtype == TRL_U8;
  s.lengths = lengths;
  s.T = T;
  s.N = N;
  s.H = H;
  segments(T, N * H, &s.segs, &s.seg_len);
  float *ws_s = nullptr, *ws_r = nullptr;
  if (s.segs > 1) {
    TRL_REQUIRE(workspace != nullptr, "%s: null workspace", fn);
    ws_s = (float *)workspace;
    ws_r = ws_s + seg_floats(N * H, s.segs, dk, dv);
  }
  const int64_t coef = N * H * s.segs * (int64_t)dk * dv;

  // S: contributions of k and v forward in time; R: of q and do backward in time
  Scan f = s, r = s;
  f.b = ok;
  f.c = ov;
  f.state_in = state_in;
  f.da = dk;
  f.dc = dv;
  f.s_state = 1.f;
  r.a = ok;
  r.b = oq;
  r.c = og;
  r.state_in = gstate;
  r.da = dk;
  r.dc = dv;
  r.reverse = 1;
  r.s_inter = 1.f;
  r.s_intra = r.s_state = (float)scale;
  if (s.segs > 1) {
    f.seg_state = ws_s;
    f.seg_coef = ws_s + coef;
    r.seg_state = ws_r;
    r.seg_coef = ws_r + coef;
    scan_launch(Scans{{f, r}}, 2, dtype, false, st);
    TRL_CHECK_LAUNCH(fn);
    join_launch(f, st);
    join_launch(r, st);
    TRL_CHECK_LAUNCH(fn);
  }
  // dv: (k, q, do) backward in time; its last state is the gradient of the initial one
  r.out = dv_out;
  r.state_out = dstate;
  // dk: (v, do, q) backward in time, R transposed
  Scan t = r;
  t.a = ov;
  t.b = og;
  t.c = oq;
  t.da = dv;
  t.dc = dk;
  t.state_t = 1;
  t.out = dk_out;
  t.state_out = nullptr;
  // dq: (do, v, k) forward in time, S transposed
  f.a = og;
  f.b = ov;
  f.c = ok;
  f.da = dv;
  f.dc = dk;
  f.state_t = 1;
  f.out = dq;
  f.s_inter = f.s_intra = (float)scale;
  if (dk == dv) {
    scan_launch(Scans{{r, t, f}}, 3, dtype, true, st);
  } else {
    scan_launch(Scans{{r}}, 1, dtype, true, st);
    scan_launch(Scans{{t, f}}, 2, dtype, true, st);
  }
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}

extern "C" int trl_decay_attention_step(const void *q, const void *k, const void *v, const float *decay, const void *start,
                                        int32_t start_dtype, const float *state_in, int64_t N, int32_t H, int32_t dk,
                                        int32_t dv, int32_t dtype, double scale, void *out, float *state_out, void *stream) {
  const char *fn = "trl_decay_attention_step";
  if (int rc = decay_check(fn, 1, N, H, dk, dv, dtype)) return rc;
  TRL_REQUIRE(start == nullptr || start_dtype == TRL_F32 || start_dtype == TRL_U8, "%s: start must be f32 or u8", fn);
  if (N == 0) return TRL_OK;
  TRL_REQUIRE(q != nullptr && k != nullptr && v != nullptr && decay != nullptr && state_in != nullptr && out != nullptr &&
                  state_out != nullptr,
              "%s: null pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t heads = N * H;
  const int u8 = start_dtype == TRL_U8;
#define STEP(LC)                                                                                                         \
  k_step<T, LC><<<(int)heads, kThreads, 0, st>>>((const T *)q, (const T *)k, (const T *)v, decay, start, u8, state_in, heads, \
                                                 H, dk, dv, (float)scale, (T *)out, state_out)
  TRL_FOR_DTYPE(dtype, {
    if (dv <= 32)
      STEP(8);
    else if (dv <= 64)
      STEP(16);
    else
      STEP(32);
  });
#undef STEP
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}
