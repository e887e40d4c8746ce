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
// c's rows inside a chunk, so a chunk whose c holds an infinity or a NaN is done again one step at a time.
#include <algorithm>

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
  int32_t H, da, dc, groups, segs, seg_len;
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

// four consecutive elements of a row from column col on, zero past the row's end
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

template <typename T, int KT, int CT, bool OUT>
__global__ __launch_bounds__(kThreads) void k_scan(Scan s) {
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int64_t heads = s.N * s.H;
  // (the launch that makes contributions has no need of the last segment in its direction of time)
  const int segs = OUT ? s.segs : s.segs - 1;
  if (wave >= heads * s.groups * segs) return;
  const int group = (int)(wave % s.groups);
  wave /= s.groups;
  const int64_t nh = wave % heads;
  const int seg = (int)(wave / heads) + (!OUT && s.reverse ? 1 : 0);
  const int64_t n = nh / s.H;
  const int h = (int)(nh % s.H);

  const int64_t length = s.lengths ? std::min<int64_t>(std::max<int64_t>(s.lengths[n], 0), s.T) : s.T;
  const int64_t t_lo = (int64_t)seg * s.seg_len;
  const int64_t t_end = std::min<int64_t>(t_lo + s.seg_len, s.T);
  const int64_t t_hi = std::min<int64_t>(t_end, length);      // steps [t_lo, t_hi) of this wave

  const T *pa = (const T *)s.a.p + n * s.a.sn + h * s.a.sh;
  const T *pb = (const T *)s.b.p + n * s.b.sn + h * s.b.sh;
  const T *pc = (const T *)s.c.p + n * s.c.sn + h * s.c.sh;
  const int col0 = group * CT * 16;
  const int off = s.reverse ? 0 : 1;

  f32x4 S[KT][CT];
  {
    // state entering the segment: the caller's, or the joined contributions of the segments before it
    const float *in = s.seg_state ? s.seg_state + (nh * s.segs + seg) * s.da * s.dc : s.state_in;
    if (s.seg_state == nullptr && in != nullptr) in += nh * s.da * s.dc;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = kt * 16 + 4 * g + r, col = col0 + ct * 16 + x;
          S[kt][ct][r] = OUT && in != nullptr && row < s.da && col < s.dc
                             ? in[s.state_t ? (int64_t)col * s.da + row : (int64_t)row * s.dc + col]
                             : 0.f;
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
  int single = 0;              // steps left to do one at a time
  int64_t done = 0;
  const int64_t steps = t_hi - t_lo;
  while (done < steps) {
    const int m = single > 0 ? 1 : (int)std::min<int64_t>(16, steps - done);
    // row x of the chunk in the order of this scan, and rows 4g + e
    const bool live = x < m;
    const int64_t tx = s.reverse ? t_hi - 1 - (done + x) : t_lo + done + x;
    float A[KT][4], B[KT][4], Bt[KT][4], C[CT][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e, col = col0 + ct * 16 + x;
        const int64_t t = s.reverse ? t_hi - 1 - (done + i) : t_lo + done + i;
        C[ct][e] = i < m && col < s.dc ? (float)pc[t * s.c.st + col] : 0.f;
      }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      if (OUT) {
        load4(pa + tx * s.a.st, kt * 16 + 4 * g, s.da, live, A[kt]);
        load4(pb + tx * s.b.st, kt * 16 + 4 * g, s.da, live, B[kt]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e, col = kt * 16 + x;
        const int64_t t = s.reverse ? t_hi - 1 - (done + i) : t_lo + done + i;
        Bt[kt][e] = i < m && col < s.da ? (float)pb[t * s.b.st + col] : 0.f;
      }
    }
    uint32_t F = 0;            // bit i: step i of the chunk is a start
    if (s.start != nullptr) {
      bool f = false;
      if (live && g == 0)
        f = s.start_u8 ? ((const uint8_t *)s.start)[tx * s.N + n] != 0 : ((const float *)s.start)[tx * s.N + n] != 0.f;
      F = (uint32_t)__ballot(f);
    }
    bool bad = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= not_finite(C[ct][e]);
    const bool any_bad = __any(bad);
    if (any_bad && m > 1) {
      single = m;
      continue;
    }

    if (OUT) {
      f32x4 P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) P = __builtin_amdgcn_mfma_f32_16x16x4f32(B[kt][e], A[kt][e], P, 0, 0, 0);
      float p[4], wi[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        const uint32_t le_j = (1u << (j + off)) - 1, le_x = (1u << (x + off)) - 1;
        const bool on = (j <= x) & ((F & le_x & ~le_j) == 0);
        p[r] = on ? P[r] * w_intra[r] : 0.f;
        wi[r] = w_inter[r];
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_16x16x4f32(A[kt][e], S[kt][ct][e], o, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t le = (1u << (4 * g + r + off)) - 1;
          o[r] = (F & le) == 0 ? o[r] * wi[r] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_16x16x4f32(p[e], C[ct][e], o, 0, 0, 0);
        const int col = col0 + ct * 16 + x;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * g + r;
          const int64_t t = s.reverse ? t_hi - 1 - (done + i) : t_lo + done + i;
          if (i < m && col < s.dc) ((T *)s.out)[(t * heads + nh) * s.dc + col] = (T)o[r];
        }
      }
    }

    float hi = full_hi, lo = full_lo, ws[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[e] = w_state[e];
    if (m != 16) {
      const double pm = power(lam, m);
      hi = (float)pm;
      lo = (float)(pm - (double)hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) ws[e] = 4 * g + e < m ? (float)power(lam, m - off - (4 * g + e)) * s.s_state : 0.f;
    }
    cut |= F != 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t le = (1u << (4 * g + e + off)) - 1;
      const bool on = (F & ~le) == 0;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) Bt[kt][e] = on ? Bt[kt][e] * ws[e] : 0.f;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
        // (lambda^m in two parts: its rounding would otherwise repeat in the same direction every chunk)
        for (int r = 0; r < 4; ++r) S[kt][ct][r] = F != 0 ? 0.f : fmaf(S[kt][ct][r], hi, S[kt][ct][r] * lo);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          S[kt][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(Bt[kt][e], C[ct][e], S[kt][ct], 0, 0, 0);
        if (any_bad) {         // rows past da: 0 times a value that is not finite
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kt * 16 + 4 * g + r >= s.da) S[kt][ct][r] = 0.f;
        }
      }
    done += m;
    if (single > 0) --single;
  }

  // the state left behind: the caller's at the end of time, or this segment's contribution
  float *left = nullptr;
  if (!OUT) {
    // (entering the segment that follows in this scan's direction: the join moves it on)
    left = s.seg_state + (nh * s.segs + seg) * s.da * s.dc;
    if (group == 0 && lane == 0) s.seg_coef[nh * s.segs + seg] = cut ? -1.f : (float)power_long(lam, steps > 0 ? steps : 0);
  } else if (s.state_out != nullptr && seg == (s.reverse ? 0 : s.segs - 1)) {
    left = s.state_out + nh * s.da * s.dc;
  }
  if (left != nullptr) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = kt * 16 + 4 * g + r, col = col0 + ct * 16 + x;
          if (row < s.da && col < s.dc) left[(int64_t)row * s.dc + col] = S[kt][ct][r];
        }
  }
  if (OUT) {                   // steps past the sequence's end
    for (int64_t t = std::max<int64_t>(t_lo, length) + g; t < t_end; t += 4)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int col = col0 + ct * 16 + x;
        if (col < s.dc) ((T *)s.out)[(t * heads + nh) * s.dc + col] = (T)0.f;
      }
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
  for (int i = 0; i < segs; ++i) {
    const int sg = reverse ? segs - 1 - i : i;
    const bool last = i == segs - 1;
    const float u = last ? 0.f : p[sg * size], cf = last ? 0.f : coef[sg];
    p[sg * size] = cur;
    cur = cf < 0.f ? u : fmaf(cf, cur, u);
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

// accumulator tiles of a's dimension a kernel is built for
int kt_of(int da) {
  const int t = tiles_of(da);
  return t <= 1 ? 1 : t <= 2 ? 2 : t <= 4 ? 4 : 8;
}

// column tiles a wave carries.  More of them read a and b fewer times and make the pair products once; fewer of them make
// more waves.  8 row tiles leave registers for two.
int ct_of(int64_t heads, int da, int dc) {
  const int t = tiles_of(dc);
  if (t == 1) return 1;
  int ct = kt_of(da) == 8 ? 2 : 4;
  while (ct > 1 && (ct >= 2 * t || heads * trl_cdiv(t, ct) < 2048)) ct /= 2;
  return ct;
}

// time segments: enough of them for two waves on every SIMD, of at least 64 steps
void segments(int64_t T, int64_t heads, int dk, int dv, int *segs, int *seg_len) {
  const int64_t waves = heads * std::min(tiles_of(dk), tiles_of(dv));
  int64_t want = waves > 0 ? trl_cdiv(2048, waves) : 1;
  want = std::max<int64_t>(1, std::min<int64_t>(want, T / 64));
  const int64_t len = std::max<int64_t>(16, trl_cdiv(trl_cdiv(T, want), 16) * 16);
  *seg_len = (int)len;
  *segs = (int)std::max<int64_t>(1, trl_cdiv(T, len));
}

template <typename T, bool OUT>
void scan_launch_t(const Scan &s, int kt, int ct, int grid, hipStream_t st) {
#define SCAN(K, C) else if (kt == K && ct == C) k_scan<T, K, C, OUT><<<grid, kThreads, 0, st>>>(s)
  if (false) {
  }
  SCAN(1, 1);
  SCAN(1, 2);
  SCAN(1, 4);
  SCAN(2, 1);
  SCAN(2, 2);
  SCAN(2, 4);
  SCAN(4, 1);
  SCAN(4, 2);
  SCAN(4, 4);
  SCAN(8, 1);
  SCAN(8, 2);
#undef SCAN
}

void scan_launch(Scan s, int32_t dtype, bool out, hipStream_t st) {
  const int64_t heads = s.N * s.H;
  const int kt = kt_of(s.da), ct = ct_of(heads * s.segs, s.da, s.dc);
  s.groups = (int)trl_cdiv(tiles_of(s.dc), ct);
  const int64_t waves = heads * s.groups * (out ? s.segs : s.segs - 1);
  const int grid = (int)trl_cdiv(waves, kThreads / 64);
  TRL_FOR_DTYPE(dtype, {
    if (out)
      scan_launch_t<T, true>(s, kt, ct, grid, st);
    else
      scan_launch_t<T, false>(s, kt, ct, grid, st);
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
  segments(T, N * H, dk, dv, &segs, &len);
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
  segments(T, N * H, dk, dv, &s.segs, &s.seg_len);
  if (s.segs > 1) {
    TRL_REQUIRE(workspace != nullptr, "%s: null workspace", fn);
    s.seg_state = (float *)workspace;
    s.seg_coef = s.seg_state + N * H * s.segs * (int64_t)dk * dv;
    scan_launch(s, dtype, false, st);
    TRL_CHECK_LAUNCH(fn);
    join_launch(s, st);
    TRL_CHECK_LAUNCH(fn);
  }
  scan_launch(s, dtype, true, st);
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
  segments(T, N * H, dk, dv, &s.segs, &s.seg_len);
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
    scan_launch(f, dtype, false, st);
    scan_launch(r, dtype, false, st);
    TRL_CHECK_LAUNCH(fn);
    join_launch(f, st);
    join_launch(r, st);
    TRL_CHECK_LAUNCH(fn);
  }
  // dv: (k, q, do) backward in time; its last state is the gradient of the initial one
  r.out = dv_out;
  r.state_out = dstate;
  scan_launch(r, dtype, true, st);
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
  scan_launch(t, dtype, true, st);
  // dq: (do, v, k) forward in time, S transposed
  f.a = og;
  f.b = ov;
  f.c = ok;
  f.da = dv;
  f.dc = dk;
  f.state_t = 1;
  f.out = dq;
  f.s_inter = f.s_intra = (float)scale;
  scan_launch(f, dtype, true, st);
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
