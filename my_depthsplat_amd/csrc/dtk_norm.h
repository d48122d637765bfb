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
//
// Measured (a copy of 256 MB runs at 5.4 TB/s): 42240 x 768 bf16 forward 26 us (5.0 TB/s), backward 35 us (5.6 TB/s) and
// 5.5 us for the fold of the weights' gradients; fused with dropout, 20001 x 1001 f16: forward 37.5 us (4.3 TB/s;
// without the generator 32.6), backward 56.5 us (3.5 TB/s) + 5: rows of no whole number of vectors, which take three groups
// of the generator per vector instead of two; 512 x 128 f32 forward 2.4 us, a launch.

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

// LPR lanes share a row, each holds NI vectors of N elements (16 bytes); vector i of a lane is number lane +
// i LPR of the row. How the row's width meets the vectors: kWhole: N divides it; kRagged: the last vector ends with the
// row, so its first `lo` elements are the one before's too: left out of the sums, and stored twice with the same value;
// kTiny: the row is shorter than a vector. (Vectors on multiples of N of the whole array instead, which
// read aligned and need a third less of the generator, lose more at the rows' partial stores: 1001 f16, fused forward 55
// us against 48.)
enum Fit { kWhole, kRagged, kTiny };
template <int N, Fit FIT>
struct Cols {
  int c0, lo, width;
  bool live;
  __device__ __forceinline__ Cols(int vec, int width)
      : c0(FIT == kRagged ? min(vec * N, width - N) : vec * N), lo(vec * N - c0), width(width), live(vec * N < width) {}
  __device__ __forceinline__ bool there(int e) const { return FIT != kTiny || e < width; }  // the row has this element
  __device__ __forceinline__ bool first(int e) const { return FIT == kWhole || (e >= lo && there(e)); }  // and it is this vector's
  // the sum over the elements that are this vector's
  template <typename F>
  __device__ __forceinline__ float sum(F value) const {
    float t = 0.f;
    if (FIT == kWhole || (FIT == kRagged && lo == 0)) {
#pragma unroll
      for (int e = 0; e < N; ++e) t += value(e);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) t += first(e) ? value(e) : 0.f;
    }
    return live ? t : 0.f;
  }
};
template <typename T, int N, Fit FIT>
__device__ __forceinline__ Vec<T> load_row(const T* row, const Cols<N, FIT>& c) {
  Vec<T> v = {};
  if (!c.live) return v;
  if constexpr (FIT != kTiny) return load_vec(row + c.c0);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (c.there(e)) v.v[e] = row[e];
  return v;
}
template <typename T, int N, Fit FIT>
__device__ __forceinline__ void store_row(T* row, const Cols<N, FIT>& c, const float (&f)[N]) {
  Vec<T> v;
#pragma unroll
  for (int e = 0; e < N; ++e) v.v[e] = rounded<T>(f[e]);
  if (!c.live) return;
  if constexpr (FIT != kTiny) {
    store_vec(row + c.c0, v);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c.there(e)) row[e] = v.v[e];
  }
}
template <typename T, int N, Fit FIT>
__device__ __forceinline__ void load_w(const void* p, bool f32, const Cols<N, FIT>& c, float none, float (&f)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = none;
  if (!p || !c.live) return;
  if (sizeof(T) == 4 || !f32) {
    const Vec<T> v = load_row<T, N, FIT>((const T*)p, c);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (float)v.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c.there(e)) f[e] = ((const float*)p)[c.c0 + e];
  }
}
template <int N, Fit FIT>
__device__ __forceinline__ void drop_row(const Drop& drop, const RngKey& key, uint64_t n0, float (&f)[N]) {
  if (!drop.rng) return;
  bool keep[N];
  if constexpr (FIT == kWhole) keep_mask<N>(key, n0, drop.least, keep);
  else keep_mask_anywhere<N>(key, n0, drop.least, keep);
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = keep[e] ? f[e] * drop.scale : 0.f;
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

// Waves per SIMD that the registers of NI vectors leave room for (all: the fused backward, which holds a third
// gradient and the generator's words; at 3 waves it would spill: 77 us against 55 for 20001 x 1001 f16).
constexpr int waves_of(int ni, bool all) { return ni <= 1 ? 4 : ni > 2 ? 1 : all ? 2 : 3; }

// A group of LPR lanes walks rows with the stride of the grid; the next row is on its way while one is worked on,
// the weights stay in registers.
template <typename T, int NI, int LPR, bool ADD, Fit FIT>
__global__ __launch_bounds__(kThreads, waves_of(NI, false)) void k_norm_fwd(FwdArgs a) {
  constexpr int N = Vec<T>::N, RPB = kThreads / LPR;
  using C = Cols<N, FIT>;
  __shared__ float red[kThreads / 64];
  const T *x = (const T*)a.x, *residual = (const T*)a.residual;
  const int lane = threadIdx.x % LPR, width = a.width;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const float inv = 1.f / (float)width;
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
  struct Row {
    Vec<T> x[NI], r[ADD ? NI : 1];
  };
  const auto fetch = [&](Row& f, int64_t row) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
      f.x[i] = load_row<T, N, FIT>(x + row * width, c);
      if (ADD) f.r[i] = load_row<T, N, FIT>(residual + row * width, c);
    }
  };
  Row next;
  if (row < a.rows) fetch(next, row);
  float w[NI][N], b[NI][N];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const C c(lane + i * LPR, width);
    load_w<T, N, FIT>(a.wb.w, a.wb.f32, c, 1.f, w[i]);
    load_w<T, N, FIT>(a.wb.b, a.wb.f32, c, 0.f, b[i]);
  }
  while (row < a.rows) {
    const Row cur = next;
    const int64_t at = row;
    row += step;
    if (row < a.rows) fetch(next, row);
    float z[NI][N];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
#pragma unroll
      for (int e = 0; e < N; ++e) z[i][e] = (float)cur.x[i].v[e];
      if constexpr (ADD) {
        drop_row<N, FIT>(a.drop, key, (uint64_t)(at * width + c.c0), z[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) z[i][e] = (float)rounded<T>(z[i][e] + (float)cur.r[i].v[e]);
        store_row<T, N, FIT>((T*)a.s + at * width, c, z[i]);
      }
      sum += c.sum([&](int e) { return z[i][e]; });
    }
    const float mu = row_sum<LPR>(sum, red) * inv;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
#pragma unroll
      for (int e = 0; e < N; ++e) z[i][e] -= mu;
      sq += c.sum([&](int e) { return z[i][e] * z[i][e]; });
    }
    const float r = 1.f / sqrtf(row_sum<LPR>(sq, red) * inv + a.eps);
    if (lane == 0 && a.mean) {
      a.mean[at] = mu;
      a.rstd[at] = r;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = __builtin_fmaf(z[i][e] * r, w[i][e], b[i][e]);
      store_row<T, N, FIT>((T*)a.y + at * width, C(lane + i * LPR, width), o);
    }
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

// Backward: the same walk; a lane keeps its columns' sums of dy xh and dy in registers. The groups of a workgroup are
// folded through LDS in turn into one row of `part`, which k_norm_fold sums in a fixed order: no atomics,
// the same bits every time.
template <typename T, int NI, int LPR, bool ADD, Fit FIT>
__global__ __launch_bounds__(kThreads, waves_of(NI, ADD)) void k_norm_bwd(BwdArgs a) {
  constexpr int N = Vec<T>::N, RPB = kThreads / LPR;
  using C = Cols<N, FIT>;
  __shared__ float red[kThreads / 64];
  __shared__ float fold[2][LPR <= 64 ? NI * LPR * N : 1];
  const T *z = (const T*)a.z, *dy = (const T*)a.dy, *ds = (const T*)a.ds;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, width = a.width;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + group;
  const float inv = 1.f / (float)width;
  float dw[NI][N] = {}, db[NI][N] = {};
  RngKey key = {};
  if (ADD && a.drop.rng) key = rng_key(a.drop.rng, a.drop.call);
  struct Row {
    Vec<T> z[NI], dy[NI];
    float mu, r;
  };
  const auto fetch = [&](Row& f, int64_t row) {
    f.mu = a.mean[row];
    f.r = a.rstd[row];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
      f.z[i] = load_row<T, N, FIT>(z + row * width, c);
      f.dy[i] = dy ? load_row<T, N, FIT>(dy + row * width, c) : Vec<T>{};
    }
  };
  Row next;
  if (row < a.rows) fetch(next, row);
  float w[NI][N];
#pragma unroll
  for (int i = 0; i < NI; ++i) load_w<T, N, FIT>(a.wb.w, a.wb.f32, C(lane + i * LPR, width), 1.f, w[i]);
  while (row < a.rows) {
    const Row cur = next;
    const int64_t at = row;
    row += step;
    Vec<T> add[ADD ? NI : 1];
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
        add[i] = ds ? load_row<T, N, FIT>(ds + at * width, C(lane + i * LPR, width)) : Vec<T>{};
    }
    if (row < a.rows) fetch(next, row);
    float xh[NI][N], g[NI][N];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        xh[i][e] = ((float)cur.z[i].v[e] - cur.mu) * cur.r;  // (the forward's: z r - mu r loses a large mean's digits)
        const float d = (float)cur.dy[i].v[e];
        dw[i][e] = __builtin_fmaf(d, xh[i][e], dw[i][e]);
        db[i][e] += d;
        g[i][e] = d * w[i][e];
      }
      s1 += c.sum([&](int e) { return g[i][e]; });
      s2 += c.sum([&](int e) { return g[i][e] * xh[i][e]; });
    }
    s1 = row_sum<LPR>(s1, red) * inv;
    s2 = row_sum<LPR>(s2, red) * inv;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = cur.r * __builtin_fmaf(-xh[i][e], s2, g[i][e] - s1);
      if constexpr (ADD) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] += (float)add[i].v[e];
        if (a.dres) store_row<T, N, FIT>((T*)a.dres + at * width, c, o);
        if (a.dx) drop_row<N, FIT>(a.drop, key, (uint64_t)(at * width + c.c0), o);
      }
      if (a.dx) store_row<T, N, FIT>((T*)a.dx + at * width, c, o);
    }
  }
  if (!a.part) return;
  float* pw = a.part + (int64_t)blockIdx.x * width;
  float* pb = a.part + ((int64_t)gridDim.x + blockIdx.x) * width;
  if constexpr (LPR > 64) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const C c(lane + i * LPR, width);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c.live && c.first(e)) {
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
        const C c(lane + i * LPR, width);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (c.live && c.first(e)) {
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

// Rows too wide for registers (above 4096 f32 or 8192 of 16 bits): the workgroup walks the row, once per moment, an element per
// thread, the generator's whole group for each, and the backward adds to its row of `part` in memory. 2048 x 16384 bf16:
// forward 90 us (1.5 TB/s), backward 276 + 21, with dropout 155 and 353 + 21. Left so: no layer here is that wide (a
// head's tokens have 216 channels), and vectors would need all of the above once more.
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
      v = (float)rounded<T>(v + (float)residual[c]);
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
    ((T*)a.y)[row * width + c] = rounded<T>(__builtin_fmaf(((float)z[c] - mu) * r, weight_at<T>(a.wb.w, a.wb.f32, c, 1.f),
                                                          weight_at<T>(a.wb.b, a.wb.f32, c, 0.f)));
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
        if (a.dres) ((T*)a.dres)[row * width + c] = rounded<T>(g);
        if (a.dx && a.drop.rng) g = keep_one(a.drop, key, (uint64_t)row * width + c) ? g * a.drop.scale : 0.f;
      }
      if (a.dx) ((T*)a.dx)[row * width + c] = rounded<T>(g);
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
// the row, so narrow rows share a wave; up to 128 one wave; up to 1024 the workgroup; wider rows are
// walked (lpr 0).
struct Shape {
  int lpr, ni;
  Fit fit;
};
inline Shape shape_of(int width, int dtype) {
  const int n = dtype == DTK_F32 ? 4 : 8, vecs = (width + n - 1) / n;
  const Fit fit = width < n ? kTiny : width % n ? kRagged : kWhole;
  if (vecs <= 8) return {8, 1, fit};
  if (vecs <= 16) return {16, 1, fit};
  if (vecs <= 32) return {32, 1, fit};
  if (vecs <= 128) return {64, (vecs + 63) / 64, fit};
  if (vecs <= 1024) return {256, vecs <= 256 ? 1 : vecs <= 512 ? 2 : 4, fit};
  return {0, 0, fit};
}
// Workgroups that walk the rows: no more than the chip holds at once (waves_of() per CU), and so many
// that each walks the same number of rows.
inline int walk_grid(int64_t rows, const Shape& s, bool all) {
  const int per_block = s.lpr ? kThreads / s.lpr : 1;
  const int64_t need = (rows + per_block - 1) / per_block;
  const int most = 256 * waves_of(s.ni, all);
  const int64_t turns = (need + most - 1) / most;
  return (int)((need + turns - 1) / turns);
}

template <typename T, int NI, int LPR, bool ADD>
void launch_fwd(const FwdArgs& a, Fit fit, hipStream_t st) {
  const int grid = walk_grid(a.rows, {LPR, NI, fit}, false);
  if (fit == kWhole) k_norm_fwd<T, NI, LPR, ADD, kWhole><<<grid, kThreads, 0, st>>>(a);
  else if (LPR > 8 || fit == kRagged) k_norm_fwd<T, NI, LPR, ADD, kRagged><<<grid, kThreads, 0, st>>>(a);
  else k_norm_fwd<T, 1, 8, ADD, kTiny><<<grid, kThreads, 0, st>>>(a);
}
template <typename T, int NI, int LPR, bool ADD>
void launch_bwd(const BwdArgs& a, int grid, Fit fit, hipStream_t st) {
  if (fit == kWhole) k_norm_bwd<T, NI, LPR, ADD, kWhole><<<grid, kThreads, 0, st>>>(a);
  else if (LPR > 8 || fit == kRagged) k_norm_bwd<T, NI, LPR, ADD, kRagged><<<grid, kThreads, 0, st>>>(a);
  else k_norm_bwd<T, 1, 8, ADD, kTiny><<<grid, kThreads, 0, st>>>(a);
}
#define DTK_BY_SHAPE(GO, WIDE)                     \
  switch (s.lpr) {                                 \
    case 8: return GO(1, 8);                       \
    case 16: return GO(1, 16);                     \
    case 32: return GO(1, 32);                     \
    case 64:                                       \
      if (s.ni == 1) return GO(1, 64);             \
      return GO(2, 64);                            \
    case 256:                                      \
      if (s.ni == 1) return GO(1, 256);            \
      if (s.ni == 2) return GO(2, 256);            \
      return GO(4, 256);                           \
  }                                                \
  WIDE
template <typename T, bool ADD>
void run_fwd(const FwdArgs& a, const Shape& s, hipStream_t st) {
#define DTK_GO(NI, LPR) launch_fwd<T, NI, LPR, ADD>(a, s.fit, st)
  DTK_BY_SHAPE(DTK_GO, (k_norm_fwd_wide<T, ADD><<<(unsigned)a.rows, kThreads, 0, st>>>(a)));
#undef DTK_GO
}
template <typename T, bool ADD>
void run_bwd(const BwdArgs& a, int grid, const Shape& s, hipStream_t st) {
#define DTK_GO(NI, LPR) launch_bwd<T, NI, LPR, ADD>(a, grid, s.fit, st)
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
