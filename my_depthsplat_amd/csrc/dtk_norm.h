// dtk_norm.h — layer norm (forward, backward, the weight gradient's reduction), dropout from
// a counter-based generator, and the two fused with the residual sum, for gfx950.
//
//   z = residual + keep * x / (1 - p)      (plain norm: z = x)
//   mu = mean z, r = 1 / sqrt(mean (z - mu)^2 + eps), xh = (z - mu) r, y = xh w + b
//   a = dy w;  dz = r (a - mean a - xh mean(a xh)) + ds;  dresidual = dz, dx = keep dz / (1 - p)
//   dw = sum_rows dy xh, db = sum_rows dy
//
// Bound by memory: a row is read once into registers, the two moments are taken there (the
// second around the mean, so a large mean costs no digits), and written once. The norm is of z
// as it was rounded to the rows' type, which is what the caller holds and the backward reads
// back: taken from the unrounded sum, a row whose spread is below that rounding would get the
// gradient of another row. The mask is never stored: the backward regenerates it from the
// element's number.

#pragma once
#include "dtk_common.h"

namespace dtk {

constexpr int kThreads = 256;

struct Drop {
  const int64_t* rng;  // NULL: no dropout
  uint32_t least;      // words above it are kept
  float scale;
  uint32_t call;
};
struct Weights {
  const void *w, *b;
  bool f32;  // else of the rows' type
};

// The sum over the LPR lanes (a power of two) that share a row, in every one of them: by lane exchanges
// inside the vector unit (quads, mirrored halves of 16, swapped rows of 16 and of 32); LPR = 256: the
// workgroup, through LDS.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = add_dpp<0xB1>(v);   // lane ^ 1
  v = add_dpp<0x4E>(v);   // lane ^ 2
  v = add_dpp<0x141>(v);  // the other quad of 8
  if constexpr (LPR > 8) v = add_dpp<0x140>(v);  // the other 8 of 16
  if constexpr (LPR > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LPR > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// LPR lanes share a row, each holds NI vectors of N elements (16 bytes); vector i of a lane is
// number lane + i LPR. The vectors lie on multiples of N of the whole array, not of the row: a row whose width
// N does not divide (ODD) begins and ends inside one. So every load and whole store is an
// aligned vector and every vector is made of whole groups of the generator, at any width; the elements of
// the neighbour rows are read and left out.
template <int N, bool ODD>
struct Cols {
  int c0, lo, hi;  // the vector's first column (may be negative); its elements lo .. hi - 1 are the row's
  __device__ __forceinline__ Cols(int vec, int shift, int width)
      : c0(vec * N - (ODD ? shift : 0)), lo(ODD ? max(0, -c0) : 0), hi(ODD ? min(N, width - c0) : (c0 < width ? N : 0)) {}
  __device__ __forceinline__ bool live() const { return hi > lo; }
  __device__ __forceinline__ bool mine(int e) const { return !ODD || (e >= lo && e < hi); }
};
template <int N, bool ODD>
__device__ __forceinline__ int shift_of(int64_t row, int width) {
  return ODD ? (int)((row * width) & (N - 1)) : 0;
}

// n0: the vector's first element in the array of `total`
template <typename T, int N, bool ODD>
__device__ __forceinline__ Vec<T> load_row(const T* p, int64_t n0, int64_t total) {
  if (!ODD || n0 + N <= total) return load_vec(p + n0);
  Vec<T> v = {};  // the last row's last vector
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (n0 + e < total) v.v[e] = p[n0 + e];
  return v;
}
template <typename T, int N, bool ODD>
__device__ __forceinline__ void store_row(T* p, int64_t n0, const Cols<N, ODD>& c, const float (&f)[N]) {
  Vec<T> v;
#pragma unroll
  for (int e = 0; e < N; ++e) v.v[e] = (T)f[e];
  if (!ODD || (c.lo == 0 && c.hi == N)) {
    store_vec(p + n0, v);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c.mine(e)) p[n0 + e] = v.v[e];
  }
}
template <typename T, int N, bool ODD>
__device__ __forceinline__ void load_w(const void* p, bool f32, const Cols<N, ODD>& c, float none, float (&f)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = none;
  if (!p) return;
  if (!ODD || (c.lo == 0 && c.hi == N)) {
    if (sizeof(T) == 4 || !f32) {
      const Vec<T> v = load_vec((const T*)p + c.c0);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = (float)v.v[e];
    } else {
      const Vec<float> v0 = load_vec((const float*)p + c.c0), v1 = load_vec((const float*)p + c.c0 + N / 2);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        f[e] = v0.v[e];
        f[e + N / 2] = v1.v[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c.mine(e)) f[e] = f32 ? ((const float*)p)[c.c0 + e] : (float)((const T*)p)[c.c0 + e];
  }
}

struct FwdArgs {
  int64_t rows;
  int width;
  const void *x, *residual;
  Weights wb;
  Drop drop;
  float eps;
  void *s, *y;
  float *mean, *rstd;
};

template <typename T, int NI, int LPR, bool ADD, bool ODD>
__global__ __launch_bounds__(kThreads) void k_norm_fwd(FwdArgs a) {
  constexpr int N = Vec<T>::N, RPB = kThreads / LPR;
  __shared__ float red[kThreads / 64];
  const T *x = (const T*)a.x, *residual = (const T*)a.residual;
  const int lane = threadIdx.x % LPR, width = a.width;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR, total = a.rows * width;
  if (LPR <= 64 && row >= a.rows) return;  // whole groups of lanes
  const int shift = shift_of<N, ODD>(row, width);
  const float inv = 1.f / (float)width;
  float z[NI][N];
  float sum = 0.f;
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Cols<N, ODD> c(lane + i * LPR, shift, width);
    const int64_t n0 = row * width + c.c0;
#pragma unroll
    for (int e = 0; e < N; ++e) z[i][e] = 0.f;
    if (!c.live()) continue;
    const Vec<T> v = load_row<T, N, ODD>(x, n0, total);
    if constexpr (ADD) {
      const Vec<T> r = load_row<T, N, ODD>(residual, n0, total);
      bool keep[N];
      if (a.drop.rng) keep_mask<N>(key, (uint64_t)n0, a.drop.least, keep);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float d = (float)v.v[e];
        if (a.drop.rng) d = keep[e] ? d * a.drop.scale : 0.f;
        z[i][e] = (float)(T)(d + (float)r.v[e]);
      }
      store_row<T, N, ODD>((T*)a.s, n0, c, z[i]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) z[i][e] = (float)v.v[e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      z[i][e] = c.mine(e) ? z[i][e] : 0.f;
      sum += z[i][e];
    }
  }
  const float mu = row_sum<LPR>(sum, red) * inv;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Cols<N, ODD> c(lane + i * LPR, shift, width);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      z[i][e] -= mu;
      sq += c.live() && c.mine(e) ? z[i][e] * z[i][e] : 0.f;
    }
  }
  const float r = 1.f / sqrtf(row_sum<LPR>(sq, red) * inv + a.eps);
  if (lane == 0 && a.mean) {
    a.mean[row] = mu;
    a.rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Cols<N, ODD> c(lane + i * LPR, shift, width);
    if (!c.live()) continue;
    float w[N], b[N], o[N];
    load_w<T, N, ODD>(a.wb.w, a.wb.f32, c, 1.f, w);
    load_w<T, N, ODD>(a.wb.b, a.wb.f32, c, 0.f, b);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = z[i][e] * r * w[e] + b[e];
    store_row<T, N, ODD>((T*)a.y, row * width + c.c0, c, o);
  }
}

struct BwdArgs {
  int64_t rows;
  int width;
  const void *z, *dy, *ds;
  Weights wb;
  const float *mean, *rstd;
  Drop drop;
  void *dx, *dres;
  float* part;  // [2, gridDim, width]: the workgroups' sums of dy xh and of dy
};

// Backward: a group of LPR lanes walks rows with the stride of the grid and keeps its columns' sums
// of dy xh and dy in registers; the next row is on its way while one is worked on. (ODD: the stride is a multiple
// of N rows, so the columns of a lane stay the same.) The groups of a workgroup are folded through LDS in
// turn into one row of `part`, which k_norm_fold sums in a fixed order: no atomics, the same bits every time.
template <typename T, int NI, int LPR, bool ADD, bool ODD>
__global__ __launch_bounds__(kThreads) void k_norm_bwd(BwdArgs a) {
  constexpr int N = Vec<T>::N, RPB = kThreads / LPR;
  constexpr int kFold = LPR <= 64 ? (NI * LPR + 1) * N : 1;  // columns of a row
  __shared__ float red[kThreads / 64];
  __shared__ float fold[2][kFold];
  const T *z = (const T*)a.z, *dy = (const T*)a.dy, *ds = (const T*)a.ds;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, width = a.width;
  const int64_t total = a.rows * width, step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + group;
  const int shift = shift_of<N, ODD>(row, width);
  const float inv = 1.f / (float)width;
  float dw[NI][N] = {}, db[NI][N] = {};
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
  struct Row {
    Vec<T> z[NI], dy[NI], ds[ADD ? NI : 1];
    float mu, r;
  };
  const auto fetch = [&](Row& f, int64_t row) {
    f.mu = a.mean[row];
    f.r = a.rstd[row];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Cols<N, ODD> c(lane + i * LPR, shift, width);
      const int64_t n0 = row * width + c.c0;
      f.z[i] = f.dy[i] = Vec<T>{};
      if (ADD) f.ds[i] = Vec<T>{};
      if (!c.live()) continue;
      f.z[i] = load_row<T, N, ODD>(z, n0, total);
      if (dy) f.dy[i] = load_row<T, N, ODD>(dy, n0, total);
      if (ADD && ds) f.ds[i] = load_row<T, N, ODD>(ds, n0, total);
    }
  };
  Row next;
  if (row < a.rows) fetch(next, row);
  while (row < a.rows) {
    const Row cur = next;
    const int64_t at = row;
    row += step;
    if (row < a.rows) fetch(next, row);
    float xh[NI][N], g[NI][N];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Cols<N, ODD> c(lane + i * LPR, shift, width);
      float w[N];
      if (c.live()) load_w<T, N, ODD>(a.wb.w, a.wb.f32, c, 1.f, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool on = c.live() && c.mine(e);
        xh[i][e] = on ? ((float)cur.z[i].v[e] - cur.mu) * cur.r : 0.f;
        const float d = on ? (float)cur.dy[i].v[e] : 0.f;
        dw[i][e] += d * xh[i][e];
        db[i][e] += d;
        g[i][e] = on ? d * w[e] : 0.f;
        s1 += g[i][e];
        s2 += g[i][e] * xh[i][e];
      }
    }
    s1 = row_sum<LPR>(s1, red) * inv;
    s2 = row_sum<LPR>(s2, red) * inv;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Cols<N, ODD> c(lane + i * LPR, shift, width);
      if (!c.live()) continue;
      const int64_t n0 = at * width + c.c0;
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = cur.r * (g[i][e] - s1 - xh[i][e] * s2);
      if constexpr (ADD) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] += ds ? (float)cur.ds[i].v[e] : 0.f;
        if (a.dres) store_row<T, N, ODD>((T*)a.dres, n0, c, o);
        if (a.dx && a.drop.rng) {
          bool keep[N];
          keep_mask<N>(key, (uint64_t)n0, a.drop.least, keep);
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = keep[e] ? o[e] * a.drop.scale : 0.f;
        }
      }
      if (a.dx) store_row<T, N, ODD>((T*)a.dx, n0, c, o);
    }
  }
  if (!a.part) return;
  float* pw = a.part + (int64_t)blockIdx.x * width;
  float* pb = a.part + ((int64_t)gridDim.x + blockIdx.x) * width;
  if constexpr (LPR > 64) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Cols<N, ODD> c(lane + i * LPR, shift, width);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c.live() && c.mine(e)) {
          pw[c.c0 + e] = dw[i][e];
          pb[c.c0 + e] = db[i][e];
        }
    }
  } else {
    for (int gq = 0; gq < RPB; ++gq) {
      __syncthreads();
      if (group != gq) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const Cols<N, ODD> c(lane + i * LPR, shift, width);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (c.live() && c.mine(e)) {
            fold[0][c.c0 + e] = (gq ? fold[0][c.c0 + e] : 0.f) + dw[i][e];
            fold[1][c.c0 + e] = (gq ? fold[1][c.c0 + e] : 0.f) + db[i][e];
          }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kThreads) {
      pw[c] = fold[0][c];
      pb[c] = fold[1][c];
    }
  }
}

// Rows too wide for registers: the workgroup walks the row, once per moment.
__device__ __forceinline__ bool keep_one(const Drop& d, const RngKey& key, uint64_t n) {
  uint32_t w[4];
  philox(key, n >> 2, w);
  const uint32_t s = (uint32_t)n & 3u;
  return (s == 0 ? w[0] : s == 1 ? w[1] : s == 2 ? w[2] : w[3]) > d.least;
}
template <typename T>
__device__ __forceinline__ float weight_at(const void* p, bool f32, int c, float none) {
  return !p ? none : f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
}
template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void k_norm_fwd_wide(FwdArgs a) {
  __shared__ float red[kThreads / 64];
  const int width = a.width;
  const int64_t row = blockIdx.x;
  const T *x = (const T*)a.x + row * width, *residual = (const T*)a.residual + (ADD ? row * width : 0);
  T* s = (T*)a.s + (ADD ? row * width : 0);
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
  const T* z = ADD ? s : x;  // a thread reads back the sums that it wrote itself
  const float inv = 1.f / (float)width;
  float sum = 0.f;
  for (int c = threadIdx.x; c < width; c += kThreads) {
    float v = (float)x[c];
    if constexpr (ADD) {
      if (a.drop.rng) v = keep_one(a.drop, key, (uint64_t)row * width + c) ? v * a.drop.scale : 0.f;
      v = (float)(T)(v + (float)residual[c]);
      s[c] = (T)v;
    }
    sum += v;
  }
  const float mu = row_sum<256>(sum, red) * inv;
  float sq = 0.f;
  for (int c = threadIdx.x; c < width; c += kThreads) {
    const float d = (float)z[c] - mu;
    sq += d * d;
  }
  const float r = 1.f / sqrtf(row_sum<256>(sq, red) * inv + a.eps);
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mu;
    a.rstd[row] = r;
  }
  for (int c = threadIdx.x; c < width; c += kThreads)
    ((T*)a.y)[row * width + c] = (T)(((float)z[c] - mu) * r * weight_at<T>(a.wb.w, a.wb.f32, c, 1.f) +
                                     weight_at<T>(a.wb.b, a.wb.f32, c, 0.f));
}
template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void k_norm_bwd_wide(BwdArgs a) {
  __shared__ float red[kThreads / 64];
  const int width = a.width;
  const T *z = (const T*)a.z, *dy = (const T*)a.dy, *ds = (const T*)a.ds;
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
  const float inv = 1.f / (float)width;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mu = a.mean[row], r = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    if (dy)
      for (int c = threadIdx.x; c < width; c += kThreads) {
        const float g = (float)dy[row * width + c] * weight_at<T>(a.wb.w, a.wb.f32, c, 1.f);
        s1 += g;
        s2 += g * (((float)z[row * width + c] - mu) * r);
      }
    s1 = row_sum<256>(s1, red) * inv;
    s2 = row_sum<256>(s2, red) * inv;
    const bool first = row == blockIdx.x;
    for (int c = threadIdx.x; c < width; c += kThreads) {
      const float xh = ((float)z[row * width + c] - mu) * r;
      const float d = dy ? (float)dy[row * width + c] : 0.f;
      float g = r * (d * weight_at<T>(a.wb.w, a.wb.f32, c, 1.f) - s1 - xh * s2);
      if constexpr (ADD) {
        if (ds) g += (float)ds[row * width + c];
        if (a.dres) ((T*)a.dres)[row * width + c] = (T)g;
        if (a.dx && a.drop.rng) g = keep_one(a.drop, key, (uint64_t)row * width + c) ? g * a.drop.scale : 0.f;
      }
      if (a.dx) ((T*)a.dx)[row * width + c] = (T)g;
      if (a.part) {  // each thread owns its columns of the workgroup's partial row
        float* pw = a.part + (int64_t)blockIdx.x * width + c;
        float* pb = a.part + ((int64_t)gridDim.x + blockIdx.x) * width + c;
        *pw = (first ? 0.f : *pw) + d * xh;
        *pb = (first ? 0.f : *pb) + d;
      }
    }
  }
}

// The registers' layout of a row: LPR lanes x NI vectors. Up to 32 vectors the smallest group that holds
// the row, so narrow rows share a wave; up to 256 one wave; up to 2048 the workgroup; wider rows are
// walked (lpr 0).
struct Shape {
  int lpr, ni;
  bool odd;
};
inline Shape shape_of(int width, int dtype) {
  const int n = dtype == DTK_F32 ? 4 : 8;
  const bool odd = width % n != 0;
  const int vecs = odd ? (width + 2 * n - 2) / n : width / n;  // odd: whatever the row's place in its first vector
  if (vecs <= 8) return {8, 1, odd};
  if (vecs <= 16) return {16, 1, odd};
  if (vecs <= 32) return {32, 1, odd};
  if (vecs <= 256) return {64, (vecs + 63) / 64, odd};
  if (vecs <= 1024) return {256, (vecs + 255) / 256, odd};
  return {0, 0, odd};
}
inline int rows_per_block(const Shape& s) { return s.lpr ? kThreads / s.lpr : 1; }
// Workgroups of the backward: enough to fill 256 CUs four times, few enough that their partial rows stay small; a
// multiple of 8 where that keeps a lane's columns (k_norm_bwd, ODD).
inline int bwd_grid(int64_t rows, const Shape& s) {
  const int64_t need = (rows + rows_per_block(s) - 1) / rows_per_block(s);
  return (int)(need >= 1024 ? 1024 : s.lpr && s.odd ? (need + 7) / 8 * 8 : need);
}

template <typename T, int NI, int LPR, bool ADD>
void launch_fwd(const FwdArgs& a, bool odd, hipStream_t st) {
  const unsigned grid = (unsigned)((a.rows + kThreads / LPR - 1) / (kThreads / LPR));
  if (odd) k_norm_fwd<T, NI, LPR, ADD, true><<<grid, kThreads, 0, st>>>(a);
  else k_norm_fwd<T, NI, LPR, ADD, false><<<grid, kThreads, 0, st>>>(a);
}
template <typename T, int NI, int LPR, bool ADD>
void launch_bwd(const BwdArgs& a, int grid, bool odd, hipStream_t st) {
  if (odd) k_norm_bwd<T, NI, LPR, ADD, true><<<grid, kThreads, 0, st>>>(a);
  else k_norm_bwd<T, NI, LPR, ADD, false><<<grid, kThreads, 0, st>>>(a);
}
#define DTK_BY_SHAPE(GO, WIDE)                     \
  switch (s.lpr) {                                 \
    case 8: return GO(1, 8);                       \
    case 16: return GO(1, 16);                     \
    case 32: return GO(1, 32);                     \
    case 64:                                       \
      if (s.ni == 1) return GO(1, 64);             \
      if (s.ni == 2) return GO(2, 64);             \
      if (s.ni == 3) return GO(3, 64);             \
      return GO(4, 64);                            \
    case 256:                                      \
      if (s.ni == 2) return GO(2, 256);            \
      return GO(4, 256);                           \
  }                                                \
  WIDE
template <typename T, bool ADD>
void run_fwd(const FwdArgs& a, const Shape& s, hipStream_t st) {
#define DTK_GO(NI, LPR) launch_fwd<T, NI, LPR, ADD>(a, s.odd, st)
  DTK_BY_SHAPE(DTK_GO, (k_norm_fwd_wide<T, ADD><<<(unsigned)a.rows, kThreads, 0, st>>>(a)));
#undef DTK_GO
}
template <typename T, bool ADD>
void run_bwd(const BwdArgs& a, int grid, const Shape& s, hipStream_t st) {
#define DTK_GO(NI, LPR) launch_bwd<T, NI, LPR, ADD>(a, grid, s.odd, st)
  DTK_BY_SHAPE(DTK_GO, (k_norm_bwd_wide<T, ADD><<<grid, kThreads, 0, st>>>(a)));
#undef DTK_GO
}
template <typename T>
void run_fwd(const FwdArgs& a, const Shape& s, hipStream_t st) {
  a.residual ? run_fwd<T, true>(a, s, st) : run_fwd<T, false>(a, s, st);
}
template <typename T>
void run_bwd(const BwdArgs& a, int grid, const Shape& s, bool add, hipStream_t st) {
  add ? run_bwd<T, true>(a, grid, s, st) : run_bwd<T, false>(a, grid, s, st);
}

// One translation unit per element type compiles these.
extern template void run_fwd<float>(const FwdArgs&, const Shape&, hipStream_t);
extern template void run_fwd<bf16>(const FwdArgs&, const Shape&, hipStream_t);
extern template void run_fwd<f16>(const FwdArgs&, const Shape&, hipStream_t);
extern template void run_bwd<float>(const BwdArgs&, int, const Shape&, bool, hipStream_t);
extern template void run_bwd<bf16>(const BwdArgs&, int, const Shape&, bool, hipStream_t);
extern template void run_bwd<f16>(const BwdArgs&, int, const Shape&, bool, hipStream_t);

}  // namespace dtk
