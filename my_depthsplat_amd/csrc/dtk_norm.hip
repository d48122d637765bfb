// dtk_norm.hip — layer norm (forward, backward, the weight gradient's reduction), dropout from
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

#include "dtk_common.h"

namespace {
using namespace dtk;

constexpr int NT = 256;

struct Drop {
  const int64_t* rng;  // NULL: no dropout
  uint64_t threshold;
  float scale;
  uint32_t call;
};

// LPR lanes share a row (a power of two up to 64; 256 = the workgroup), each holds NI vectors:
// vector i of a lane is number lane + i * LPR of the row. A width that no vector divides ends in
// one vector that starts at width - N: its first elements repeat the one before (they are left
// out of the sums and written twice with the same value).
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int off = (LPR < 64 ? LPR : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (LPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// The column a lane's vector i starts at, and how many of its leading elements repeat.
template <int N>
struct Place {
  int col, skip;
  bool live;
};
template <int N>
__device__ __forceinline__ Place<N> place(int vec, int width) {
  const int at = vec * N;
  const bool live = at < width;
  const int col = at + N <= width ? at : (width - N);
  return {live ? col : 0, live ? at - col : N, live};
}

// Rows narrower than one vector: one element per "vector".
template <typename T, int N>
__device__ __forceinline__ void load_f(const T* p, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = (float)p[0];
  } else {
    const Vec<T> v = load_vec(p);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (float)v.v[e];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* p, const float (&f)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)f[0];
  } else {
    Vec<T> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = (T)f[e];
    store_vec(p, v);
  }
}
template <typename WT, int N>
__device__ __forceinline__ void load_w(const WT* p, int col, float none, float (&f)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = none;
  if (p) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (float)p[col + e];
  }
}

template <int N>
__device__ __forceinline__ void keeps(const Drop& d, const RngKey& key, uint64_t n0, bool (&keep)[N]) {
  if constexpr (N == 1) {
    uint32_t w[4];
    philox(key, n0 >> 2, w);
    const uint32_t s = (uint32_t)n0 & 3u;
    keep[0] = (s == 0 ? w[0] : s == 1 ? w[1] : s == 2 ? w[2] : w[3]) >= d.threshold;
  } else {
    keep_mask<N>(key, n0, d.threshold, keep);
  }
}

template <typename T, typename WT, int N, int NI, int LPR, bool ADD>
__global__ __launch_bounds__(NT) void k_norm_fwd(int64_t rows, int width, const T* __restrict__ x,
                                                 const T* __restrict__ residual, const WT* __restrict__ weight,
                                                 const WT* __restrict__ bias, Drop drop, float eps, T* __restrict__ s,
                                                 T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[NT / 64];
  constexpr int RPB = NT / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  if (LPR <= 64 && row >= rows) return;
  const float inv = 1.f / (float)width;
  float z[NI][N];
  float sum = 0.f;
  RngKey key = {};
  if (ADD && drop.rng) key = rng_key(drop.rng, drop.call);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Place<N> at = place<N>(lane + i * LPR, width);
#pragma unroll
    for (int e = 0; e < N; ++e) z[i][e] = 0.f;
    if (at.live) {
      load_f<T, N>(x + row * width + at.col, z[i]);
      if constexpr (ADD) {
        float r[N];
        load_f<T, N>(residual + row * width + at.col, r);
        if (drop.rng) {
          bool keep[N];
          keeps<N>(drop, key, (uint64_t)row * width + at.col, keep);
#pragma unroll
          for (int e = 0; e < N; ++e) z[i][e] = keep[e] ? z[i][e] * drop.scale : 0.f;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) z[i][e] = (float)(T)(z[i][e] + r[e]);
        store_f<T, N>(s + row * width + at.col, z[i]);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sum += e >= at.skip ? z[i][e] : 0.f;
    }
  }
  const float mu = row_sum<LPR>(sum, red) * inv;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Place<N> at = place<N>(lane + i * LPR, width);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      z[i][e] -= mu;
      sq += e >= at.skip ? z[i][e] * z[i][e] : 0.f;
    }
  }
  const float r = 1.f / sqrtf(row_sum<LPR>(sq, red) * inv + eps);
  if (lane == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Place<N> at = place<N>(lane + i * LPR, width);
    if (!at.live) continue;
    float w[N], b[N], o[N];
    load_w<WT, N>(weight, at.col, 1.f, w);
    load_w<WT, N>(bias, at.col, 0.f, b);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = z[i][e] * r * w[e] + b[e];
    store_f<T, N>(y + row * width + at.col, o);
  }
}

// Backward: a group of LPR lanes walks rows with the stride of the grid and keeps its columns'
// sums of dy xh and dy in registers; the groups of a workgroup are folded through LDS into one
// row of `part` [2, gridDim, width], which k_norm_fold sums in a fixed order (no atomics: the
// same bits every time).
template <typename T, typename WT, int N, int NI, int LPR, bool ADD>
__global__ __launch_bounds__(NT) void k_norm_bwd(int64_t rows, int width, const T* __restrict__ z,
                                                 const T* __restrict__ dy, const T* __restrict__ ds,
                                                 const WT* __restrict__ weight, const float* __restrict__ mean,
                                                 const float* __restrict__ rstd, Drop drop, T* __restrict__ dx,
                                                 T* __restrict__ dres, float* __restrict__ part) {
  constexpr int RPB = NT / LPR;
  constexpr int CPI = N * LPR;  // columns of one vector slot over the row's lanes
  __shared__ float red[NT / 64];
  __shared__ float fold[LPR <= 64 ? RPB * CPI : 1];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const float inv = 1.f / (float)width;
  float dw[NI][N] = {}, db[NI][N] = {};
  RngKey key = {};
  if (ADD && drop.rng) key = rng_key(drop.rng, drop.call);
  for (int64_t row = (int64_t)blockIdx.x * RPB + group; row < rows; row += (int64_t)gridDim.x * RPB) {
    const float mu = mean[row], r = rstd[row];
    float xh[NI][N], a[NI][N];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Place<N> at = place<N>(lane + i * LPR, width);
#pragma unroll
      for (int e = 0; e < N; ++e) xh[i][e] = a[i][e] = 0.f;
      if (!at.live) continue;
      load_f<T, N>(z + row * width + at.col, xh[i]);
      if (dy) load_f<T, N>(dy + row * width + at.col, a[i]);
      float w[N];
      load_w<WT, N>(weight, at.col, 1.f, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        xh[i][e] = (xh[i][e] - mu) * r;
        const bool once = e >= at.skip;
        dw[i][e] += once ? a[i][e] * xh[i][e] : 0.f;
        db[i][e] += once ? a[i][e] : 0.f;
        a[i][e] *= w[e];
        s1 += once ? a[i][e] : 0.f;
        s2 += once ? a[i][e] * xh[i][e] : 0.f;
      }
    }
    s1 = row_sum<LPR>(s1, red) * inv;
    s2 = row_sum<LPR>(s2, red) * inv;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const Place<N> at = place<N>(lane + i * LPR, width);
      if (!at.live) continue;
      float g[N];
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = r * (a[i][e] - s1 - xh[i][e] * s2);
      if constexpr (ADD) {
        if (ds) {
          float t[N];
          load_f<T, N>(ds + row * width + at.col, t);
#pragma unroll
          for (int e = 0; e < N; ++e) g[e] += t[e];
        }
        if (dres) store_f<T, N>(dres + row * width + at.col, g);
        if (dx && drop.rng) {
          bool keep[N];
          keeps<N>(drop, key, (uint64_t)row * width + at.col, keep);
#pragma unroll
          for (int e = 0; e < N; ++e) g[e] = keep[e] ? g[e] * drop.scale : 0.f;
        }
      }
      if (dx) store_f<T, N>(dx + row * width + at.col, g);
    }
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * width;
  float* pb = part + ((int64_t)gridDim.x + blockIdx.x) * width;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const Place<N> at = place<N>(lane + i * LPR, width);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float* out = which ? pb : pw;
      if constexpr (LPR > 64) {
        if (at.live) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e >= at.skip) out[at.col + e] = which ? db[i][e] : dw[i][e];
        }
      } else {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; ++e) fold[group * CPI + e * LPR + lane] = which ? db[i][e] : dw[i][e];
        __syncthreads();
        for (int c = threadIdx.x; c < CPI; c += NT) {
          const int l = c % LPR, e = c / LPR;
          const Place<N> pl = place<N>(l + i * LPR, width);
          float t = 0.f;
          for (int gq = 0; gq < RPB; ++gq) t += fold[gq * CPI + c];
          if (pl.live && e >= pl.skip) out[pl.col + e] = t;
        }
      }
    }
  }
}

// Rows too wide for registers: the workgroup walks the row in chunks, once per moment.
template <typename T, typename WT, bool ADD>
__global__ __launch_bounds__(NT) void k_norm_fwd_wide(int64_t rows, int width, const T* __restrict__ x,
                                                      const T* __restrict__ residual, const WT* __restrict__ weight,
                                                      const WT* __restrict__ bias, Drop drop, float eps,
                                                      T* s, T* __restrict__ y, float* __restrict__ mean,
                                                      float* __restrict__ rstd) {
  __shared__ float red[NT / 64];
  const int64_t row = blockIdx.x;
  RngKey key = {};
  if (ADD && drop.rng) key = rng_key(drop.rng, drop.call);
  const T* z = ADD ? s : x;  // a thread reads back the sums that it wrote itself
  auto value = [&](int c) { return (float)z[row * width + c]; };
  const float inv = 1.f / (float)width;
  float sum = 0.f;
  for (int c = threadIdx.x; c < width; c += NT) {
    float v = (float)x[row * width + c];
    if constexpr (ADD) {
      if (drop.rng) {
        bool keep[1];
        keeps<1>(drop, key, (uint64_t)row * width + c, keep);
        v = keep[0] ? v * drop.scale : 0.f;
      }
      v = (float)(T)(v + (float)residual[row * width + c]);
      s[row * width + c] = (T)v;
    }
    sum += v;
  }
  const float mu = row_sum<256>(sum, red) * inv;
  float sq = 0.f;
  for (int c = threadIdx.x; c < width; c += NT) {
    const float d = value(c) - mu;
    sq += d * d;
  }
  const float r = 1.f / sqrtf(row_sum<256>(sq, red) * inv + eps);
  if (threadIdx.x == 0 && mean) {
    mean[row] = mu;
    rstd[row] = r;
  }
  for (int c = threadIdx.x; c < width; c += NT)
    y[row * width + c] =
        (T)((value(c) - mu) * r * (weight ? (float)weight[c] : 1.f) + (bias ? (float)bias[c] : 0.f));
}
template <typename T, typename WT, bool ADD>
__global__ __launch_bounds__(NT) void k_norm_bwd_wide(int64_t rows, int width, const T* __restrict__ z,
                                                      const T* __restrict__ dy, const T* __restrict__ ds,
                                                      const WT* __restrict__ weight, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, Drop drop, T* __restrict__ dx,
                                                      T* __restrict__ dres, float* __restrict__ part) {
  __shared__ float red[NT / 64];
  RngKey key = {};
  if (ADD && drop.rng) key = rng_key(drop.rng, drop.call);
  const float inv = 1.f / (float)width;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    if (dy)
      for (int c = threadIdx.x; c < width; c += NT) {
        const float a = (float)dy[row * width + c] * (weight ? (float)weight[c] : 1.f);
        s1 += a;
        s2 += a * (((float)z[row * width + c] - mu) * r);
      }
    s1 = row_sum<256>(s1, red) * inv;
    s2 = row_sum<256>(s2, red) * inv;
    const bool first = row == blockIdx.x;
    for (int c = threadIdx.x; c < width; c += NT) {
      const float xh = ((float)z[row * width + c] - mu) * r;
      const float d = dy ? (float)dy[row * width + c] : 0.f;
      float g = r * (d * (weight ? (float)weight[c] : 1.f) - s1 - xh * s2);
      if constexpr (ADD) {
        if (ds) g += (float)ds[row * width + c];
        if (dres) dres[row * width + c] = (T)g;
        if (dx && drop.rng) {
          bool keep[1];
          keeps<1>(drop, key, (uint64_t)row * width + c, keep);
          g = keep[0] ? g * drop.scale : 0.f;
        }
      }
      if (dx) dx[row * width + c] = (T)g;
      if (part) {  // each thread owns its columns of the workgroup's partial row
        float* pw = part + (int64_t)blockIdx.x * width + c;
        float* pb = part + ((int64_t)gridDim.x + blockIdx.x) * width + c;
        *pw = (first ? 0.f : *pw) + d * xh;
        *pb = (first ? 0.f : *pb) + d;
      }
    }
  }
}

// part [2, n, width] -> dw, db [width]: 16 columns x 16 slices of the n rows per workgroup.
template <typename WT>
__global__ __launch_bounds__(NT) void k_norm_fold(int n, int width, const float* __restrict__ part,
                                                  WT* __restrict__ dw, WT* __restrict__ db) {
  __shared__ float t[16][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, slice = threadIdx.x / 16;
  const float* p = part + (int64_t)blockIdx.y * n * width;
  float s = 0.f;
  if (c < width)
    for (int k = slice; k < n; k += 16) s += p[(int64_t)k * width + c];
  t[slice][threadIdx.x % 16] = s;
  __syncthreads();
  WT* out = blockIdx.y ? db : dw;
  if (slice == 0 && c < width && out) {
    s = 0.f;
    for (int k = 0; k < 16; ++k) s += t[k][threadIdx.x];
    out[c] = (WT)s;
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void k_dropout(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                                                Drop drop, T* __restrict__ y) {
  constexpr int N = Vec<T>::N;
  const int64_t n0 = ((int64_t)blockIdx.x * NT + threadIdx.x) * N;
  if (n0 >= n) return;
  bool keep[N];
  if (drop.rng) {
    keep_mask<N>(rng_key(drop.rng, drop.call), (uint64_t)n0, drop.threshold, keep);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) keep[e] = true;
  }
  if (n0 + N <= n) {
    float f[N];
    load_f<T, N>(x + n0, f);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = keep[e] ? f[e] * drop.scale : 0.f;
    if (residual) {
      float r[N];
      load_f<T, N>(residual + n0, r);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] += r[e];
    }
    store_f<T, N>(y + n0, f);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (n0 + e < n) y[n0 + e] = (T)((keep[e] ? (float)x[n0 + e] * drop.scale : 0.f) + (residual ? (float)residual[n0 + e] : 0.f));
  }
}

struct FwdArgs {
  int64_t rows;
  int width;
  const void *x, *residual, *weight, *bias;
  Drop drop;
  float eps;
  void *s, *y;
  float *mean, *rstd;
  hipStream_t st;
};
struct BwdArgs {
  int64_t rows;
  int width;
  const void *z, *dy, *ds, *weight;
  const float *mean, *rstd;
  Drop drop;
  void *dx, *dres;
  float* part;
  int grid;
  hipStream_t st;
};

// The registers' layout of a row: LPR lanes x NI vectors of N. Up to 64 vectors: the smallest
// group that holds the row, so narrow rows share a wave; up to 512: one wave; up to 2048: the
// workgroup; wider rows are walked.
struct Shape {
  int n, lpr, ni;  // lpr 0: walked
};
inline Shape shape_of(int width, int dtype) {
  const int n = width < 8 && dtype != DTK_F32 ? 1 : width < 4 ? 1 : dtype == DTK_F32 ? 4 : 8;
  const int vecs = (width + n - 1) / n;
  if (vecs <= 8) return {n, 8, 1};
  if (vecs <= 16) return {n, 16, 1};
  if (vecs <= 32) return {n, 32, 1};
  if (vecs <= 256) return {n, 64, (vecs + 63) / 64};
  if (vecs <= 1024) return {n, 256, (vecs + 255) / 256};
  return {n, 0, 0};
}
inline int rows_per_block(const Shape& s) { return s.lpr ? NT / s.lpr : 1; }
// Workgroups of the backward: enough to fill 256 CUs, few enough that their partial rows stay small.
inline int bwd_grid(int64_t rows, const Shape& s) {
  const int64_t need = (rows + rows_per_block(s) - 1) / rows_per_block(s);
  return (int)(need < 1024 ? need : 1024);
}

template <typename T, typename WT, int N, int NI, int LPR, bool ADD>
void launch_fwd(const FwdArgs& a) {
  const unsigned grid = (unsigned)((a.rows + NT / LPR - 1) / (NT / LPR));
  k_norm_fwd<T, WT, N, NI, LPR, ADD><<<grid, NT, 0, a.st>>>(
      a.rows, a.width, (const T*)a.x, (const T*)a.residual, (const WT*)a.weight, (const WT*)a.bias, a.drop, a.eps,
      (T*)a.s, (T*)a.y, a.mean, a.rstd);
}
template <typename T, typename WT, int N, int NI, int LPR, bool ADD>
void launch_bwd(const BwdArgs& a) {
  k_norm_bwd<T, WT, N, NI, LPR, ADD><<<a.grid, NT, 0, a.st>>>(
      a.rows, a.width, (const T*)a.z, (const T*)a.dy, (const T*)a.ds, (const WT*)a.weight, a.mean, a.rstd, a.drop,
      (T*)a.dx, (T*)a.dres, a.part);
}
template <typename T, typename WT, bool ADD>
void run_fwd(const FwdArgs& a, const Shape& s) {
  constexpr int N = Vec<T>::N;
  if (s.n == 1) return launch_fwd<T, WT, 1, 1, 8, ADD>(a);
  switch (s.lpr) {
    case 8: return launch_fwd<T, WT, N, 1, 8, ADD>(a);
    case 16: return launch_fwd<T, WT, N, 1, 16, ADD>(a);
    case 32: return launch_fwd<T, WT, N, 1, 32, ADD>(a);
    case 64:
      switch (s.ni) {
        case 1: return launch_fwd<T, WT, N, 1, 64, ADD>(a);
        case 2: return launch_fwd<T, WT, N, 2, 64, ADD>(a);
        case 3: return launch_fwd<T, WT, N, 3, 64, ADD>(a);
        default: return launch_fwd<T, WT, N, 4, 64, ADD>(a);
      }
    case 256:
      switch (s.ni) {
        case 2: return launch_fwd<T, WT, N, 2, 256, ADD>(a);
        case 3: return launch_fwd<T, WT, N, 3, 256, ADD>(a);
        default: return launch_fwd<T, WT, N, 4, 256, ADD>(a);
      }
  }
  k_norm_fwd_wide<T, WT, ADD><<<(unsigned)a.rows, NT, 0, a.st>>>(
      a.rows, a.width, (const T*)a.x, (const T*)a.residual, (const WT*)a.weight, (const WT*)a.bias, a.drop, a.eps,
      (T*)a.s, (T*)a.y, a.mean, a.rstd);
}
template <typename T, typename WT, bool ADD>
void run_bwd(const BwdArgs& a, const Shape& s) {
  constexpr int N = Vec<T>::N;
  if (s.n == 1) return launch_bwd<T, WT, 1, 1, 8, ADD>(a);
  switch (s.lpr) {
    case 8: return launch_bwd<T, WT, N, 1, 8, ADD>(a);
    case 16: return launch_bwd<T, WT, N, 1, 16, ADD>(a);
    case 32: return launch_bwd<T, WT, N, 1, 32, ADD>(a);
    case 64:
      switch (s.ni) {
        case 1: return launch_bwd<T, WT, N, 1, 64, ADD>(a);
        case 2: return launch_bwd<T, WT, N, 2, 64, ADD>(a);
        case 3: return launch_bwd<T, WT, N, 3, 64, ADD>(a);
        default: return launch_bwd<T, WT, N, 4, 64, ADD>(a);
      }
    case 256:
      switch (s.ni) {
        case 2: return launch_bwd<T, WT, N, 2, 256, ADD>(a);
        case 3: return launch_bwd<T, WT, N, 3, 256, ADD>(a);
        default: return launch_bwd<T, WT, N, 4, 256, ADD>(a);
      }
  }
  k_norm_bwd_wide<T, WT, ADD><<<a.grid, NT, 0, a.st>>>(
      a.rows, a.width, (const T*)a.z, (const T*)a.dy, (const T*)a.ds, (const WT*)a.weight, a.mean, a.rstd, a.drop,
      (T*)a.dx, (T*)a.dres, a.part);
}

// weights are of the rows' type or f32
template <template <typename, typename> class F, typename... A>
void by_type(int dtype, int wtype, A&&... a) {
  if (dtype == DTK_F32) F<float, float>::go(a...);
  else if (dtype == DTK_BF16) wtype == DTK_F32 ? F<bf16, float>::go(a...) : F<bf16, bf16>::go(a...);
  else wtype == DTK_F32 ? F<f16, float>::go(a...) : F<f16, f16>::go(a...);
}
template <typename T, typename WT>
struct Fwd {
  static void go(const FwdArgs& a, const Shape& s) { a.residual ? run_fwd<T, WT, true>(a, s) : run_fwd<T, WT, false>(a, s); }
};
template <typename T, typename WT>
struct Bwd {
  static void go(const BwdArgs& a, const Shape& s, bool add) { add ? run_bwd<T, WT, true>(a, s) : run_bwd<T, WT, false>(a, s); }
};

}  // namespace

extern "C" {

int dtk_layer_norm_fwd(int64_t rows, int width, int dtype, int wtype, const void* x, const void* residual,
                       const void* weight, const void* bias, float eps, double p, const int64_t* rng, uint32_t call,
                       void* s, void* y, float* mean, float* rstd, void* stream) {
  DSPLAT_REQUIRE(rows >= 0 && width > 0 && rows < (1LL << 31), "dtk_layer_norm_fwd: bad sizes");
  DSPLAT_REQUIRE(type_ok(dtype) && (wtype == dtype || wtype == DTK_F32), "dtk_layer_norm_fwd: bad types");
  DSPLAT_REQUIRE(p >= 0.0 && p <= 1.0 && (p == 0.0 || (rng && residual)),
                 "dtk_layer_norm_fwd: dropout needs 0 <= p <= 1, rng and a residual");
  if (rows == 0) return 0;
  DSPLAT_REQUIRE(x && y && !mean == !rstd && !s == !residual, "dtk_layer_norm_fwd: null pointer");
  FwdArgs a = {rows, width, x, residual, weight, bias,
               {p > 0.0 ? rng : nullptr, drop_threshold(p), drop_scale(p), call}, eps, s, y, mean, rstd, (hipStream_t)stream};
  by_type<Fwd>(dtype, wtype, a, shape_of(width, dtype));
  return dsplat::check_launch("k_norm_fwd");
}

size_t dtk_layer_norm_bwd_workspace_size(int64_t rows, int width, int dtype) {
  if (rows <= 0 || width <= 0) return 0;
  return (size_t)2 * bwd_grid(rows, shape_of(width, dtype)) * width * sizeof(float);
}

int dtk_layer_norm_bwd(int64_t rows, int width, int dtype, int wtype, const void* z, const void* dy, const void* ds,
                       const void* weight, const float* mean, const float* rstd, int add, double p, const int64_t* rng,
                       uint32_t call, void* dx, void* dresidual, void* dweight, void* dbias, void* workspace,
                       void* stream) {
  DSPLAT_REQUIRE(rows >= 0 && width > 0 && rows < (1LL << 31), "dtk_layer_norm_bwd: bad sizes");
  DSPLAT_REQUIRE(type_ok(dtype) && (wtype == dtype || wtype == DTK_F32), "dtk_layer_norm_bwd: bad types");
  DSPLAT_REQUIRE(p >= 0.0 && p <= 1.0 && (p == 0.0 || (rng && add)), "dtk_layer_norm_bwd: dropout needs 0 <= p <= 1 and rng");
  DSPLAT_REQUIRE(add || (!ds && !dresidual), "dtk_layer_norm_bwd: a residual's gradient without a residual");
  const bool sums = dweight || dbias;
  DSPLAT_REQUIRE(rows == 0 || (z && mean && rstd && (!sums || workspace)), "dtk_layer_norm_bwd: null pointer");
  const Shape sh = shape_of(width, dtype);
  const int grid = rows ? bwd_grid(rows, sh) : 0;
  BwdArgs a = {rows, width, z, dy, ds, weight, mean, rstd,
               {p > 0.0 ? rng : nullptr, drop_threshold(p), drop_scale(p), call}, dx, dresidual,
               sums ? (float*)workspace : nullptr, grid, (hipStream_t)stream};
  if (rows) {
    by_type<Bwd>(dtype, wtype, a, sh, add != 0);
    if (int e = dsplat::check_launch("k_norm_bwd")) return e;
  }
  if (sums) {
    const dim3 g((width + 15) / 16, 2);
    if (wtype == DTK_F32) k_norm_fold<float><<<g, NT, 0, a.st>>>(grid, width, a.part, (float*)dweight, (float*)dbias);
    else if (wtype == DTK_BF16) k_norm_fold<bf16><<<g, NT, 0, a.st>>>(grid, width, a.part, (bf16*)dweight, (bf16*)dbias);
    else k_norm_fold<f16><<<g, NT, 0, a.st>>>(grid, width, a.part, (f16*)dweight, (f16*)dbias);
    return dsplat::check_launch("k_norm_fold");
  }
  return 0;
}

int dtk_dropout(int64_t n, int dtype, const void* x, const void* residual, double p, const int64_t* rng, uint32_t call,
                void* y, void* stream) {
  DSPLAT_REQUIRE(n >= 0 && n <= (1LL << 40), "dtk_dropout: bad sizes");
  DSPLAT_REQUIRE(type_ok(dtype), "dtk_dropout: bad type");
  DSPLAT_REQUIRE(p >= 0.0 && p <= 1.0, "dtk_dropout: p must be in [0, 1]");
  if (n == 0) return 0;
  DSPLAT_REQUIRE(x && y && (rng || p == 0.0), "dtk_dropout: null pointer");
  const Drop d = {p > 0.0 ? rng : nullptr, drop_threshold(p), drop_scale(p), call};
  const int64_t per = (int64_t)NT * (16 / (int64_t)type_size(dtype));
  const int64_t grid = (n + per - 1) / per;
  DSPLAT_REQUIRE(grid < (1LL << 31), "dtk_dropout: too large");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DTK_F32) k_dropout<float><<<grid, NT, 0, st>>>(n, (const float*)x, (const float*)residual, d, (float*)y);
  else if (dtype == DTK_BF16) k_dropout<bf16><<<grid, NT, 0, st>>>(n, (const bf16*)x, (const bf16*)residual, d, (bf16*)y);
  else k_dropout<f16><<<grid, NT, 0, st>>>(n, (const f16*)x, (const f16*)residual, d, (f16*)y);
  return dsplat::check_launch("k_dropout");
}

}  // extern "C"
