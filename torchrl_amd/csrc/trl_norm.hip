// Layer normalisation with its gradients, and dropout whose mask is a function of a counter: the two elementwise-and-row
// layers of a regularised Linear / ReLU stack (torchrl_amd/contrib/models.py).  The reference has neither; its stacks are
// Linear + ReLU only (torchrl/contrib/models.py:6-147).
//
// Layer norm.  For a row x of D values, with m its mean, r = 1 / sqrt(mean((x - m)^2) + eps) and n = (x - m) r:
//     y = n w + b  (then max(y, 0) with act);    with g = gy (0 where act clipped) and h = g w:
//     dx = r (h - mean(h) - n mean(h n)),   dw = sum over rows of g n,   db = sum over rows of g.
// Both directions are bound by memory: a row lives in the registers of LPR lanes from its one read to its one write, the
// mean and the centred second moment are two sums over those registers (no E[x^2] - m^2 cancellation).  (The backward pass of
// 16-bit rows of 8,193 to 16,384 elements has more than the registers hold: up to 800 B a lane of it are in scratch.)
// The weight's and the bias's gradients need a sum over all rows: every lane owns fixed columns, adds them up over the rows
// its workgroup walks, the workgroup's lane groups are added in order, and a second launch adds the workgroups' partial sums
// in order: no atomics, the same bits every run.
// Measured: 1M x 64 f32 forward 96 us (5.6 TB/s), backward 160 us (5.0 TB/s) + 5 us for the join of the parts; 16k x 1024 bf16
// 13.0, 21.8 and 4.5 us (the data stay in the last-level cache); 10007 x 257 f32 8.8, 10.0 and 4.2; 16 x 64 1.6 us.  A training
// call on small data is bound by the host and the graph engine (40 us and more), not by these.
// Rows that are not whole slots cost more, since each slot carries code for single elements beside its 16 B access: a training
// pass over 256k x 257 takes 334 us in f32 (3.2 TB/s; 260 columns 296) and 310 in bf16 (1.7 TB/s; 264 columns 149).  16-bit
// rows of many slots: 4,096 x 8,192 bf16 125 us (2.2 TB/s), 4,096 x 12,000 200 (2.0).
#include <algorithm>

#include "trl_io.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxWg = 1024;        // workgroups of a backward pass = rows of its partial sums

// sum over a row's lanes: LPR lanes of a wave, or all four waves of the workgroup (LPR == 256, through `red`)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float *red) {
  if constexpr (LPR <= 64) {
    return trl_lanes_sum<LPR>(v);
  } else {
    v = trl_lanes_sum<64>(v);
    const int w = threadIdx.x >> 6;
    __syncthreads();      // the previous sum has been read
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  }
}

// 16 B of a row as loaded, zero past the row's end; nothing touches it before its row's turn
template <typename T>
struct Slot {
  T t[TrlIo<T>::V];
};

// VEC: a row is whole slots, so that one comparison a slot decides
template <bool VEC, typename T>
__device__ __forceinline__ void load_slot(Slot<T> &q, const T *row, int64_t width, int64_t c) {
  constexpr int V = TrlIo<T>::V;
  if (c + V <= width) {
    __builtin_memcpy(q.t, row + c, 16);
  } else if constexpr (VEC) {
    q = Slot<T>{};
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      q.t[i] = (T)0.f;
      if (c + i < width) q.t[i] = row[c + i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void slot_value(const Slot<T> &q, float (&f)[TrlIo<T>::V]) {
#pragma unroll
  for (int i = 0; i < TrlIo<T>::V; ++i) f[i] = (float)q.t[i];
}

template <bool VEC, typename T>
__device__ __forceinline__ void store_slot(T *row, int64_t width, int64_t c, const float (&f)[TrlIo<T>::V]) {
  constexpr int V = TrlIo<T>::V;
  if (c + V <= width)
    trl_store16(row + c, f);
  else if (!VEC && c < width)
    trl_store_part(row + c, (int)(width - c), f);
}

// V parameters (float32) of the columns from c on
template <int V, bool VEC>
__device__ __forceinline__ void load_param(const float *p, int64_t width, int64_t c, float none, float (&f)[V]) {
  if (p != nullptr && c + V <= width) {
    __builtin_memcpy(f, p + c, 4 * V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (!VEC && p != nullptr && c + i < width) ? p[c + i] : none;
  }
}

__device__ __forceinline__ float relu_keep_nan(float z) { return z < 0.f ? 0.f : z; }
__device__ __forceinline__ float clip(float z, float g) { return z <= 0.f ? 0.f : g; }

template <typename T, int LPR, int NV, bool ACT, bool VEC>
__global__ __launch_bounds__(kThreads) void k_norm_fwd(const T *__restrict__ x, const float *__restrict__ w,
                                                       const float *__restrict__ b, int64_t rows, int64_t width, float eps,
                                                       T *__restrict__ y, float *__restrict__ mean,
                                                       float *__restrict__ rstd) {
  constexpr int V = TrlIo<T>::V, RPB = kThreads / LPR;
  __shared__ float red[4];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + group;
  Slot<T> next[NV];
  if (row < rows) {
#pragma unroll
    for (int j = 0; j < NV; ++j) load_slot<VEC>(next[j], x + row * width, width, (int64_t)(j * LPR + lane) * V);
  }
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load_param<V, VEC>(w, width, (int64_t)(j * LPR + lane) * V, 1.f, wv[j]);
    load_param<V, VEC>(b, width, (int64_t)(j * LPR + lane) * V, 0.f, bv[j]);
  }
  for (; row < rows; row += step) {
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      slot_value(next[j], v[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    }
    // the next row is on its way while this one is worked on
    if (row + step < rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) load_slot<VEC>(next[j], x + (row + step) * width, width, (int64_t)(j * LPR + lane) * V);
    }
    const float m = row_sum<LPR>(s, red) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (int64_t)(j * LPR + lane) * V + (VEC ? 0 : i) < width ? v[j][i] - m : 0.f;
        v[j][i] = d;
        q = fmaf(d, d, q);
      }
    const float r = __builtin_amdgcn_rsqf(fmaf(row_sum<LPR>(q, red), inv, eps));
    if (lane == 0) {
      if (mean != nullptr) mean[row] = m;
      if (rstd != nullptr) rstd[row] = r;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = fmaf(v[j][i] * r, wv[j][i], bv[j][i]);
        v[j][i] = ACT ? relu_keep_nan(z) : z;
      }
      store_slot<VEC>(y + row * width, width, (int64_t)(j * LPR + lane) * V, v[j]);
    }
  }
}

template <typename T, int LPR, int NV, bool ACT, bool VEC>
__global__ __launch_bounds__(kThreads) void k_norm_bwd(const T *__restrict__ gy, const T *__restrict__ x,
                                                       const float *__restrict__ w, const float *__restrict__ b,
                                                       const float *__restrict__ mean, const float *__restrict__ rstd,
                                                       int64_t rows, int64_t width, T *__restrict__ dx,
                                                       float *__restrict__ part) {
  constexpr int V = TrlIo<T>::V, RPB = kThreads / LPR;
  __shared__ float red[4];
  __shared__ float fold[kThreads * V];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const float inv = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + group;
  Slot<T> next_x[NV], next_g[NV];
  float m_next = 0.f, r_next = 0.f;
  auto bring = [&](int64_t at) {
    m_next = mean[at], r_next = rstd[at];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t col = (int64_t)(j * LPR + lane) * V;
      load_slot<VEC>(next_x[j], x + at * width, width, col);
      load_slot<VEC>(next_g[j], gy + at * width, width, col);
    }
  };
  if (row < rows) bring(row);
  float wv[NV][V], bv[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load_param<V, VEC>(w, width, (int64_t)(j * LPR + lane) * V, 1.f, wv[j]);
    if (ACT) load_param<V, VEC>(b, width, (int64_t)(j * LPR + lane) * V, 0.f, bv[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  for (; row < rows; row += step) {
    const float m = m_next, r = r_next;
    float n[NV][V], g[NV][V];
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      slot_value(next_x[j], n[j]);
      slot_value(next_g[j], g[j]);
    }
    if (row + step < rows) bring(row + step);      // the next row is on its way while this one is worked on
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // past the row's end g is 0, and u too: (0 - m) r may be infinite where every element's is finite
        const float u = (int64_t)(j * LPR + lane) * V + (VEC ? 0 : i) < width ? (n[j][i] - m) * r : 0.f;
        // the forward's own expression: its y > 0 decides, to the bit
        const float t = ACT ? clip(fmaf(u, wv[j][i], bv[j][i]), g[j][i]) : g[j][i];
        const float h = t * wv[j][i];
        dw[j][i] = fmaf(t, u, dw[j][i]);
        db[j][i] += t;
        a += h;
        c = fmaf(h, u, c);
        n[j][i] = u;
        g[j][i] = h;
      }
    if (dx != nullptr) {
      const float am = row_sum<LPR>(a, red) * inv, cm = row_sum<LPR>(c, red) * inv;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[j][i] = r * (g[j][i] - fmaf(n[j][i], cm, am));
        store_slot<VEC>(dx + row * width, width, (int64_t)(j * LPR + lane) * V, g[j]);
      }
    }
  }
  if (part == nullptr) return;
  // part[workgroup][0 = dw, 1 = db][width]: the groups of this workgroup, added in order
  float *out = part + (int64_t)blockIdx.x * 2 * width;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) fold[threadIdx.x * V + i] = s == 0 ? dw[j][i] : db[j][i];
        __syncthreads();
        for (int e = threadIdx.x; e < LPR * V; e += kThreads) {
          float t = 0.f;
          for (int gr = 0; gr < RPB; ++gr) t += fold[gr * LPR * V + e];
          const int64_t col = (int64_t)j * LPR * V + e;
          if (col < width) out[s * width + col] = t;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int64_t col = (int64_t)(j * LPR + lane) * V + i;
          if (col < width) out[s * width + col] = s == 0 ? dw[j][i] : db[j][i];
        }
      }
    }
}

// Rows of more slots than shape_of has lanes for (more than 8,192 f32 or 16,384 elements of 16 bits): one workgroup a row, the
// row read once per pass (from L2 after the first).  Correct at any width; not tuned: no network here is that wide.
template <typename T, bool ACT>
__global__ __launch_bounds__(kThreads) void k_norm_fwd_wide(const T *__restrict__ x, const float *__restrict__ w,
                                                            const float *__restrict__ b, int64_t rows, int64_t width,
                                                            float eps, T *__restrict__ y, float *__restrict__ mean,
                                                            float *__restrict__ rstd) {
  __shared__ float red[4];
  const float inv = 1.0f / (float)width;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * width;
    float s = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) s += (float)xr[c];
    const float m = row_sum<256>(s, red) * inv;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      const float d = (float)xr[c] - m;
      q = fmaf(d, d, q);
    }
    const float r = __builtin_amdgcn_rsqf(fmaf(row_sum<256>(q, red), inv, eps));
    if (threadIdx.x == 0) {
      if (mean != nullptr) mean[row] = m;
      if (rstd != nullptr) rstd[row] = r;
    }
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      const float z = fmaf(((float)xr[c] - m) * r, w ? w[c] : 1.f, b ? b[c] : 0.f);
      y[row * width + c] = (T)(ACT ? relu_keep_nan(z) : z);
    }
  }
}

template <typename T, bool ACT>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_wide_dx(const T *__restrict__ gy, const T *__restrict__ x,
                                                               const float *__restrict__ w, const float *__restrict__ b,
                                                               const float *__restrict__ mean,
                                                               const float *__restrict__ rstd, int64_t rows,
                                                               int64_t width, T *__restrict__ dx) {
  __shared__ float red[4];
  const float inv = 1.0f / (float)width;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float m = mean[row], r = rstd[row];
    const T *xr = x + row * width, *gr = gy + row * width;
    float a = 0.f, c2 = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      const float u = ((float)xr[c] - m) * r, wc = w ? w[c] : 1.f;
      const float g = (float)gr[c], t = ACT ? clip(fmaf(u, wc, b ? b[c] : 0.f), g) : g;
      a += t * wc;
      c2 = fmaf(t * wc, u, c2);
    }
    const float am = row_sum<256>(a, red) * inv, cm = row_sum<256>(c2, red) * inv;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      const float u = ((float)xr[c] - m) * r, wc = w ? w[c] : 1.f;
      const float g = (float)gr[c], t = ACT ? clip(fmaf(u, wc, b ? b[c] : 0.f), g) : g;
      dx[row * width + c] = (T)(r * (t * wc - fmaf(u, cm, am)));
    }
  }
}

// one thread a column, blockIdx.y a slab of rows
template <typename T, bool ACT>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_wide_dw(const T *__restrict__ gy, const T *__restrict__ x,
                                                               const float *__restrict__ w, const float *__restrict__ b,
                                                               const float *__restrict__ mean,
                                                               const float *__restrict__ rstd, int64_t rows,
                                                               int64_t width, float *__restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= width) return;
  const float wc = w ? w[c] : 1.f, bc = b ? b[c] : 0.f;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float u = ((float)x[row * width + c] - mean[row]) * rstd[row];
    const float g = (float)gy[row * width + c], t = ACT ? clip(fmaf(u, wc, bc), g) : g;
    dw = fmaf(t, u, dw);
    db += t;
  }
  float *out = part + (int64_t)blockIdx.y * 2 * width;
  out[c] = dw;
  out[width + c] = db;
}

// dw, db = the parts added in a fixed order: 16 columns a workgroup, 64 strips of parts, eight loads of a strip in flight
__global__ __launch_bounds__(1024) void k_norm_fold(const float *__restrict__ part, int parts, int64_t width,
                                                    float *__restrict__ dw, float *__restrict__ db) {
  __shared__ float sm[64][17], top[4][16];
  const int lc = threadIdx.x & 15, strip = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + lc, total = 2 * width;
  float s = 0.f;
  if (c < total) {
    for (int p0 = strip; p0 < parts; p0 += 64 * 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p0 + 64 * i < parts ? part[(int64_t)(p0 + 64 * i) * total + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  sm[strip][lc] = s;
  __syncthreads();
  if (threadIdx.x < 256) {
    // strips 4 k .. 4 k + 3, then the 16 sums of them
    float t = (sm[4 * strip][lc] + sm[4 * strip + 1][lc]) + (sm[4 * strip + 2][lc] + sm[4 * strip + 3][lc]);
    t += __shfl_xor(t, 16, 64);
    t += __shfl_xor(t, 32, 64);
    if ((threadIdx.x & 63) < 16) top[threadIdx.x >> 6][lc] = t;
  }
  __syncthreads();
  if (threadIdx.x < 16 && c < total) {
    const float t = (top[0][lc] + top[1][lc]) + (top[2][lc] + top[3][lc]);
    if (c < width) {
      if (dw != nullptr) dw[c] = t;
    } else if (db != nullptr) {
      db[c - width] = t;
    }
  }
}

// Lanes a row and 16 B slots a lane by the number of slots of a row: the fewest lanes that hold it in few slots, so that a
// wave works on several narrow rows at once and up to 256 slots need no barrier; 0 = more slots than it has lanes for.
// Training passes against a wave for every row of at most 64 slots and a workgroup for wider ones: 1M x 32 f32 134 us against
// 384, 1M x 64 263 / 423, 256k x 128 bf16 62 / 117, 16k x 512 f32 37 / 47, 64k x 1024 bf16 139 / 233, 10007 x 257 f32 26 / 45;
// even only for 16k x 1024 f32 (66 / 64).
struct Shape {
  int lpr, nv;
};
Shape shape_of(int64_t width, int v) {
  const int64_t n = trl_cdiv(width, v);
  if (n <= 8) return {8, 1};
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return {64, 4};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  if (n <= 2048) return {256, 8};
  return {0, 0};
}

#define FOR_BOOL(value, NAME, ...)                           \
  do {                                                       \
    if (value) { constexpr bool NAME = true; __VA_ARGS__; }  \
    else { constexpr bool NAME = false; __VA_ARGS__; }       \
  } while (0)

#define NORM_SHAPES(sh, ...)                                              \
  do {                                                                    \
    if (sh.lpr == 8) { constexpr int LPR = 8, NV = 1; __VA_ARGS__; }      \
    else if (sh.lpr == 16) { constexpr int LPR = 16, NV = 1; __VA_ARGS__; } \
    else if (sh.lpr == 32) { constexpr int LPR = 32, NV = 1; __VA_ARGS__; } \
    else if (sh.lpr == 64 && sh.nv == 1) { constexpr int LPR = 64, NV = 1; __VA_ARGS__; } \
    else if (sh.lpr == 64 && sh.nv == 2) { constexpr int LPR = 64, NV = 2; __VA_ARGS__; } \
    else if (sh.lpr == 64) { constexpr int LPR = 64, NV = 4; __VA_ARGS__; } \
    else if (sh.nv == 2) { constexpr int LPR = 256, NV = 2; __VA_ARGS__; } \
    else if (sh.nv == 4) { constexpr int LPR = 256, NV = 4; __VA_ARGS__; } \
    else { constexpr int LPR = 256, NV = 8; __VA_ARGS__; }                \
  } while (0)

int elem_bytes(int32_t dtype) { return dtype == TRL_F32 ? 4 : 2; }

// workgroups of a backward pass over rows of this width
int bwd_parts(int64_t rows, int64_t width, int32_t dtype) {
  const Shape sh = shape_of(width, 16 / elem_bytes(dtype));
  const int64_t per = sh.lpr ? kThreads / sh.lpr : 32;
  return (int)std::max<int64_t>(1, std::min<int64_t>(trl_cdiv(rows, per), sh.lpr ? kMaxWg : 64));
}

int norm_check(const char *fn, int64_t rows, int64_t width, int32_t dtype, int32_t act) {
  TRL_REQUIRE(trl_float_dtype(dtype), "%s: dtype %d is not f32, bf16 or f16", fn, (int)dtype);
  TRL_REQUIRE(rows >= 0 && width >= 1 && width < (1 << 24), "%s: bad shape [%lld, %lld]", fn, (long long)rows,
              (long long)width);
  TRL_REQUIRE(rows < ((int64_t)1 << 40) / width, "%s: too many elements: [%lld, %lld]", fn, (long long)rows,
              (long long)width);
  TRL_REQUIRE(act == 0 || act == 1, "%s: act must be 0 or 1", fn);
  return TRL_OK;
}

}  // namespace

extern "C" int trl_layer_norm_fwd(const void *x, const float *weight, const float *bias, int64_t rows, int64_t width,
                                  int32_t dtype, double eps, int32_t act, void *y, float *mean, float *rstd, void *stream) {
  const char *fn = "trl_layer_norm_fwd";
  if (int rc = norm_check(fn, rows, width, dtype, act)) return rc;
  TRL_REQUIRE((float)eps >= 1.2e-38f && eps < 1e30, "%s: eps must be positive (a normal float32)", fn);
  if (rows == 0) return TRL_OK;
  TRL_REQUIRE(x != nullptr && y != nullptr, "%s: null pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  const Shape sh = shape_of(width, 16 / elem_bytes(dtype));
  TRL_FOR_DTYPE(dtype, {
    if (sh.lpr == 0) {
      const int grid = (int)std::min<int64_t>(rows, 2048);
      FOR_BOOL(act, ACT, (k_norm_fwd_wide<T, ACT><<<grid, kThreads, 0, st>>>((const T *)x, weight, bias, rows, width, (float)eps,
                                                                       (T *)y, mean, rstd)));
    } else {
      const int grid = (int)std::min<int64_t>(trl_cdiv(rows, kThreads / sh.lpr), 2048);
      const bool vec = width % TrlIo<T>::V == 0;
      NORM_SHAPES(sh, FOR_BOOL(vec, VEC, FOR_BOOL(act, ACT, (k_norm_fwd<T, LPR, NV, ACT, VEC><<<grid, kThreads, 0, st>>>(
                                                                (const T *)x, weight, bias, rows, width, (float)eps, (T *)y,
                                                                mean, rstd)))));
    }
  });
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}

extern "C" int64_t trl_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int32_t dtype) {
  if (norm_check("trl_layer_norm_bwd_workspace_bytes", rows, width, dtype, 0)) return TRL_EINVAL;
  return (int64_t)bwd_parts(rows, width, dtype) * 2 * width * 4;
}

extern "C" int trl_layer_norm_bwd(const void *gy, const void *x, const float *weight, const float *bias, const float *mean,
                                  const float *rstd, int64_t rows, int64_t width, int32_t dtype, int32_t act, void *dx,
                                  float *dweight, float *dbias, void *workspace, void *stream) {
  const char *fn = "trl_layer_norm_bwd";
  if (int rc = norm_check(fn, rows, width, dtype, act)) return rc;
  const bool params = dweight != nullptr || dbias != nullptr;
  TRL_REQUIRE(!params || workspace != nullptr, "%s: null workspace", fn);
  TRL_REQUIRE(rows == 0 || (gy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr), "%s: null pointer", fn);
  if (!params && (rows == 0 || dx == nullptr)) return TRL_OK;
  const hipStream_t st = (hipStream_t)stream;
  const Shape sh = shape_of(width, 16 / elem_bytes(dtype));
  const int parts = bwd_parts(rows, width, dtype);
  float *part = params ? (float *)workspace : nullptr;
  TRL_FOR_DTYPE(dtype, {
    if (sh.lpr == 0) {
      const int grid = (int)std::min<int64_t>(rows, 2048);
      if (dx != nullptr && rows > 0)
        FOR_BOOL(act, ACT, (k_norm_bwd_wide_dx<T, ACT><<<grid, kThreads, 0, st>>>((const T *)gy, (const T *)x, weight, bias, mean,
                                                                            rstd, rows, width, (T *)dx)));
      if (params)
        FOR_BOOL(act, ACT, (k_norm_bwd_wide_dw<T, ACT><<<dim3((int)trl_cdiv(width, kThreads), parts), kThreads, 0, st>>>(
                         (const T *)gy, (const T *)x, weight, bias, mean, rstd, rows, width, part)));
    } else {
      const bool vec = width % TrlIo<T>::V == 0;
      NORM_SHAPES(sh, FOR_BOOL(vec, VEC, FOR_BOOL(act, ACT, (k_norm_bwd<T, LPR, NV, ACT, VEC><<<parts, kThreads, 0, st>>>(
                                                                (const T *)gy, (const T *)x, weight, bias, mean, rstd, rows,
                                                                width, (T *)dx, part)))));
    }
  });
  TRL_CHECK_LAUNCH(fn);
  if (params) {
    k_norm_fold<<<(int)trl_cdiv(2 * width, 16), 1024, 0, st>>>(part, parts, width, dweight, dbias);
    TRL_CHECK_LAUNCH(fn);
  }
  return TRL_OK;
}

// ---------------------------------------------------------------------------------------------- dropout
// Element i of call c is kept when word i % 4 of Philox-4x32-10 with key = seed and counter = (c, i / 4 with its top bit set)
// is at least round(p 2^32): the mask of a call is a function of (seed, c, i) alone, so the backward pass makes it again instead of
// reading it, and a call on a part of the memory or on another grid keeps the same elements.  (The top bit keeps the
// counters apart from those of the exploration draws, csrc/trl_act.hip, under an equal seed.)
// The generator costs 18 32 x 32 -> 64 bit products a lane for four elements (two of its 20 are the same for a whole wave).  In
// float32 and with a residual that hides behind the memory (1M x 64 bf16 + residual: 84 us, 4.8 TB/s, a copy's rate); bf16 in and
// out without one is bound by them (65 us, 4.1 TB/s; a slot more in flight made it 76).
namespace {

__device__ __forceinline__ void philox4(uint64_t seed, uint64_t call, uint32_t group, uint32_t group_hi, uint32_t (&c)[4]) {
  c[0] = (uint32_t)call;
  c[1] = (uint32_t)(call >> 32);
  c[2] = group;
  c[3] = group_hi | 0x80000000u;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  // (philox_round of trl_common.h with both exclusive ors of a word in one instruction)
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c[1], k0, 0x96);
    const uint32_t n2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c[3], k1, 0x96);
    c[1] = (uint32_t)p1;
    c[3] = (uint32_t)p0;
    c[0] = n0;
    c[2] = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

template <typename T, bool RES>
__global__ __launch_bounds__(kThreads) void k_dropout(const T *__restrict__ x, const T *__restrict__ res, int64_t n,
                                                      uint32_t threshold, float scale, uint64_t seed, uint64_t call,
                                                      const int64_t *__restrict__ call_d, T *__restrict__ y) {
  constexpr int V = TrlIo<T>::V;
  if (call_d != nullptr) call = (uint64_t)call_d[0];
  const int64_t slots = (n + V - 1) / V;
  for (int64_t s0 = (int64_t)blockIdx.x * kThreads; s0 < slots; s0 += (int64_t)gridDim.x * kThreads) {
    const int64_t s = s0 + threadIdx.x;
    if (s >= slots) return;
    // a workgroup's slots begin at a multiple of 256: one high word for all of them, and two of the generator's products
    // are the same for the whole wave
    const uint32_t group_hi = (uint32_t)((uint64_t)s0 * (V / 4) >> 32);
    const int64_t i = s * V;
    const bool whole = i + V <= n;
    float v[V], e[V];
    if (whole) {
      trl_load16(x + i, v);
      if (RES) trl_load16(res + i, e);
    } else {
      trl_load_part(x + i, (int)(n - i), 0.f, v);
      if (RES) trl_load_part(res + i, (int)(n - i), 0.f, e);
    }
#pragma unroll
    for (int g = 0; g < V / 4; ++g) {
      uint32_t u[4];
      philox4(seed, call, (uint32_t)((uint64_t)s * (V / 4) + g), group_hi, u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = u[k] >= threshold ? v[4 * g + k] * scale : 0.f;      // (whatever a dropped element holds)
        v[4 * g + k] = RES ? e[4 * g + k] + d : d;
      }
    }
    if (whole)
      trl_store16(y + i, v);
    else
      trl_store_part(y + i, (int)(n - i), v);
  }
}

__global__ void k_next_call(int64_t *counter, int64_t *call) {
  call[0] = (int64_t)atomicAdd((unsigned long long *)counter, 1ull);
}

}  // namespace

extern "C" int trl_dropout(const void *x, const void *residual, int64_t n, int32_t dtype, double p, uint64_t seed,
                           uint64_t call, const int64_t *call_d, void *y, void *stream) {
  const char *fn = "trl_dropout";
  TRL_REQUIRE(trl_float_dtype(dtype), "%s: dtype %d is not f32, bf16 or f16", fn, (int)dtype);
  TRL_REQUIRE(n >= 0 && n < ((int64_t)1 << 40), "%s: bad length %lld", fn, (long long)n);
  const double t = p * 4294967296.0 + 0.5;      // (at 2^32 no word would be large enough)
  TRL_REQUIRE(p >= 0.0 && t < 4294967296.0, "%s: p must be in [0, 1 - 2^-33)", fn);
  if (n == 0) return TRL_OK;
  TRL_REQUIRE(x != nullptr && y != nullptr, "%s: null pointer", fn);
  const hipStream_t st = (hipStream_t)stream;
  const uint32_t threshold = (uint32_t)t;
  const float scale = (float)(1.0 / (1.0 - p));
  const int grid = (int)std::min<int64_t>(trl_cdiv(n, (int64_t)kThreads * (16 / elem_bytes(dtype))), 2048);
  TRL_FOR_DTYPE(dtype, {
    if (residual != nullptr)
      k_dropout<T, true><<<grid, kThreads, 0, st>>>((const T *)x, (const T *)residual, n, threshold, scale, seed, call,
                                                    call_d, (T *)y);
    else
      k_dropout<T, false><<<grid, kThreads, 0, st>>>((const T *)x, nullptr, n, threshold, scale, seed, call, call_d, (T *)y);
  });
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}

extern "C" int trl_next_call(int64_t *counter, int64_t *call, void *stream) {
  const char *fn = "trl_next_call";
  TRL_REQUIRE(counter != nullptr && call != nullptr && counter != call, "%s: null pointer or one buffer for both", fn);
  k_next_call<<<1, 1, 0, (hipStream_t)stream>>>(counter, call);
  TRL_CHECK_LAUNCH(fn);
  return TRL_OK;
}
