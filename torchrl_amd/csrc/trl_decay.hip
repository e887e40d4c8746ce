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
// One workgroup carries one (env, head, time segment), each of its waves 16 of c's columns, with the wave's columns of S in MFMA
// accumulators from the first step to the last: 16 steps a turn, products on the 16x16 MFMA (f32 and f16 inputs: exact f32;
// bf16 inputs: bf16, where a computed operand goes in whole, as three bf16 parts).  Every accumulator is used where it lies:
// lane (g = lane / 16, x = lane % 16) of a result tile holds rows 4g .. 4g + 3 of column x, which is just what the same
// instruction takes as an operand with k = 4g + e (the sum over k may run in any order as long as both operands agree).  So the
// pair products are made transposed (P^T = b a^T: the next product's left operand) and S multiplies from the right, with no
// exchange between lanes.  The inputs come through LDS, staged a chunk ahead in two buffers: a by rows, b and c transposed.
//
// Few heads: time is cut into segments.  A first launch makes every segment's own contribution to the state, the last runs the
// segments; the state that enters one (state entering segment s + 1 = lambda^len state entering s + contribution, in order) is
// made by its workgroup itself, or, with many segments, by a launch between the two.
//
// Values that are not finite stay where the recurrence puts them: masks are selections, never products with zero -- except
// of b's and c's steps inside a chunk, so a chunk whose b or c holds an infinity or a NaN is taken one step at a time.
// An infinite state stays infinite, of its sign, for ever (bf16: its products come out as NaN).
#include <algorithm>
#include <cmath>

#include "trl_decay_scan.h"

using namespace trl_decay;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 128;

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

// seg_state[s]: contribution of segment s -> state entering segment s, in the scan's direction.  coef < 0: a start in it.
// blockIdx.y: one of the scans.  A thread per element of the state, a chain of dependent sums over the segments whose operands
// are loaded sixteen at a time (64 segments of 8 heads of 64 x 64: 9.6 us; with one load in flight the chain was memory latency
// alone).
__global__ __launch_bounds__(kThreads) void k_join(Scans all, int64_t heads, int64_t size) {
  const Scan &s = all.s[blockIdx.y];
  // (time is cut where there are a few hundred heads at most: 32 bits are enough for an element's number)
  const uint32_t e32 = blockIdx.x * kThreads + threadIdx.x;
  if (e32 >= (uint32_t)(heads * size)) return;
  const int64_t e = e32, nh = e32 / (uint32_t)size;
  const int segs = s.segs, reverse = s.reverse;
  float *p = s.seg_state + nh * segs * size + (e - nh * size);
  const float *coef = s.seg_coef + nh * segs;
  float cur = s.state_in ? s.state_in[e] : 0.f;
  const int first = reverse ? segs - 1 : 0, dir = reverse ? -1 : 1;
  for (int i0 = 0; i0 < segs; i0 += 16) {
    float u[16], cf[16];       // sixteen contributions in flight
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool on = i0 + i < segs - 1;      // (the last one moves nothing on)
      const int sg = first + dir * (i0 + i);
      u[i] = on ? p[sg * size] : 0.f;
      cf[i] = on ? coef[sg] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i0 + i < segs) p[(first + dir * (i0 + i)) * size] = cur;
      cur = cf[i] < 0.f ? u[i] : fmaf(cf[i], cur, u[i]);
    }
  }
}

// One step: a workgroup per (env, head); LC lanes hold four columns each (the fewest that hold a row, so that a wave's access
// is whole rows), the others share out the rows.  Heads of 64 x 64 are bound by the state's one read and one write: 4,096 envs of
// 4 of them take 105 us, 5.1 TB/s, 1,024 of 128 x 128 113 us, 4.7; one env 3.2 us.  Small heads leave threads without work, 64 of
// 256 have some at 16 x 16 and 16 at 8 x 8: 65,536 envs of 4 heads of 16 x 16 347 us, 1.7 TB/s, 262,144 of 8 x 8 1,167, 0.6.
template <typename T, int LC>
__global__ __launch_bounds__(kThreads) void k_step(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                   const float *__restrict__ decay, const void *__restrict__ start,
                                                   int start_u8, const float *state_in, int64_t heads, int32_t H, int32_t dk,
                                                   int32_t dv, float scale, T *__restrict__ out, float *state_out) {
  constexpr int RL = kThreads / LC;
  __shared__ float part[RL][LC * 4];
  const int64_t nh = blockIdx.x, n = blockIdx.x / (uint32_t)H;
  const int h = (int)(blockIdx.x % (uint32_t)H);
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

// Time segments: as many as bring the launch to 2,048 waves (two a SIMD; a workgroup has one for 16 columns of a head), each of
// at least 64 steps, no more than sqrt(T) of them, and none where that makes fewer than three.  Training passes, us:
//  * waves, not workgroups: 128 heads of 128 in bf16, 400 steps: 2,048 waves 185, 4,096 243; 128 heads of 32 in f32, 400
//    steps: 1,536 waves 57, 1,024 65, 256 82.
//  * two halves take as long as the whole, since a contribution costs most of a segment's work again: 256 heads of 64 in f32, 256
//    steps: two segments 119, one 97; 128 heads, 128 steps: 57 and 49; but 128 heads, 1,024 steps: four 210, one 252.
//  * shorter ones are mostly start and join, longer ones a longer chain: 64 heads of 64 in bf16, 500 steps: at least 64 steps 75,
//    128 steps 85, 111 heads of 48 / 80, 333 steps: 113 and 130; 128 heads of 64, 128 steps: at least 32 steps 61, 64 steps 49.
//  * the join walks the segments one after another: one head of 16 in f32, 131,072 steps: 362 segments 176, 2,048 485, 128 237;
//    32,768 steps: 181 segments 95, 512 143.
void segments(int64_t T, int64_t heads, int32_t dk, int32_t dv, int *segs, int *seg_len) {
  const int64_t waves = tiles_of(std::max(dk, dv));
  int64_t want = heads > 0 ? (2048 / waves + heads / 2) / heads : 1;
  want = std::min(want, (int64_t)std::sqrt((double)T));
  want = std::max<int64_t>(1, std::min<int64_t>(want, T / 64));
  if (want < 3) want = 1;
  const int64_t len = std::max<int64_t>(16, trl_cdiv(trl_cdiv(T, want), 16) * 16);
  *seg_len = (int)len;
  *segs = (int)std::max<int64_t>(1, trl_cdiv(T, len));
}

void scan_launch(const Scans &all, int count, int32_t dtype, bool out, hipStream_t st) {
  if (dtype == TRL_F32)
    launch_f32(all, count, out, st);
  else if (dtype == TRL_BF16)
    launch_bf16(all, count, out, st);
  else
    launch_f16(all, count, out, st);
}

// the contributions of `count` scans of equal sizes, and their join where the workgroups do not make it themselves
int contributions(const char *fn, const Scans &all, int count, int32_t dtype, hipStream_t st) {
  scan_launch(all, count, dtype, false, st);
  TRL_CHECK_LAUNCH(fn);
  const Scan &f = all.s[0];
  if (f.segs > kJoinInside) {
    const int64_t heads = f.N * f.H, size = (int64_t)f.da * f.dc;
    k_join<<<dim3((unsigned)trl_cdiv(heads * size, kThreads), count), kThreads, 0, st>>>(all, heads, size);
    TRL_CHECK_LAUNCH(fn);
  }
  return TRL_OK;
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
    if (int rc = contributions(fn, Scans{{s}}, 1, dtype, st)) return rc;
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
    if (int rc = contributions(fn, Scans{{f, r}}, 2, dtype, st)) return rc;
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
