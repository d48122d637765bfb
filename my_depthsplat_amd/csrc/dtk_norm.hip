// dtk_norm.hip — the C ABI of layer norm and dropout (kernels of the norm: dtk_norm.h), the fold of the
// weights' gradients, and the dropout kernel.
#include "dtk_norm.h"

namespace {
using namespace dtk;

constexpr int NT = kThreads;

// part [2, n, width] -> dw, db [width]: 64 columns per workgroup, its 16 waves take every 16th of the n rows.
constexpr int kFoldThreads = 1024;
template <typename WT>
__global__ __launch_bounds__(kFoldThreads) void k_norm_fold(int n, int width, const float* __restrict__ part,
                                                            WT* __restrict__ dw, WT* __restrict__ db) {
  __shared__ float t[kFoldThreads / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const float* p = part + (int64_t)blockIdx.y * n * width;
  float s = 0.f;
  if (c < width)
#pragma unroll 8
    for (int k = wave; k < n; k += kFoldThreads / 64) s += p[(int64_t)k * width + c];
  t[wave][lane] = s;
  __syncthreads();
  WT* out = blockIdx.y ? db : dw;
  if (wave == 0 && c < width && out) {
    s = 0.f;
    for (int k = 0; k < kFoldThreads / 64; ++k) s += t[k][lane];
    out[c] = (WT)s;
  }
}

template <typename T>
__device__ __forceinline__ void drop_vec(Vec<T>& v, const Vec<T>& r, const Drop& drop, const RngKey& key, uint64_t n0, bool add) {
  constexpr int N = Vec<T>::N;
  bool keep[N];
  if (drop.rng) keep_mask<N>(key, n0, drop.least, keep);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float f = (float)v.v[e];
    if (drop.rng) f = keep[e] ? f * drop.scale : 0.f;
    v.v[e] = rounded<T>(add ? f + (float)r.v[e] : f);
  }
}
// One vector per thread. The generator takes two products a round, ten rounds per four elements: 40 per vector (f32: 20),
// which fit beside the vector's bytes (129024 x 512 bf16 with a residual: 69 us, 5.7 TB/s, with the generator and without).
// Forward with a residual and backward together 118 us, 5.6 TB/s; 2048 x 128 f32 2.6 us, a launch.
template <typename T>
__global__ __launch_bounds__(NT) void k_dropout(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                                                Drop drop, T* __restrict__ y) {
  constexpr int N = Vec<T>::N;
  const int64_t first = (int64_t)blockIdx.x * NT * N, n0 = first + (int64_t)threadIdx.x * N;
  RngKey key = {};
  if (drop.rng) key = rng_key(drop.rng, drop.call);
  if (first + NT * N <= n) {
    Vec<T> v = load_vec(x + n0), r = {};
    if (residual) r = load_vec(residual + n0);
    drop_vec(v, r, drop, key, (uint64_t)n0, residual != nullptr);
    store_vec(y + n0, v);
    return;
  }
  if (n0 >= n) return;
  Vec<T> v = {}, r = {};
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (n0 + e < n) {
      v.v[e] = x[n0 + e];
      if (residual) r.v[e] = residual[n0 + e];
    }
  drop_vec(v, r, drop, key, (uint64_t)n0, residual != nullptr);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (n0 + e < n) y[n0 + e] = v.v[e];
}

// p 2^32, rounded, is the least word that is kept; a p that rounds to 0 drops nothing.
Drop drop_of(double p, const int64_t* rng, uint32_t call) {
  const uint64_t t = (uint64_t)__builtin_llrint(p * 4294967296.0);
  return {t ? rng : nullptr, (uint32_t)(t - 1), p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f, call};
}

}  // namespace

extern "C" {

int dtk_layer_norm_fwd(int64_t rows, int width, int dtype, int wtype, const void* x, const void* residual,
                       const void* weight, const void* bias, float eps, double p, const int64_t* rng, uint32_t call,
                       void* s, void* y, float* mean, float* rstd, void* stream) {
  DSPLAT_REQUIRE(rows >= 0 && width > 0 && width <= (1 << 28) && rows < (1LL << 31), "dtk_layer_norm_fwd: bad sizes");
  DSPLAT_REQUIRE(type_ok(dtype) && (wtype == dtype || wtype == DTK_F32), "dtk_layer_norm_fwd: bad types");
  DSPLAT_REQUIRE(p >= 0.0 && p <= 1.0 && (p == 0.0 || (rng && residual)),
                 "dtk_layer_norm_fwd: dropout needs 0 <= p <= 1, rng and a residual");
  if (rows == 0) return 0;
  DSPLAT_REQUIRE(x && y && !mean == !rstd && !s == !residual, "dtk_layer_norm_fwd: null pointer");
  const FwdArgs a = {rows, width, x, residual, {weight, bias, wtype == DTK_F32}, drop_of(p, rng, call), eps, s, y, mean, rstd};
  const Shape sh = shape_of(width, dtype);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DTK_F32) run_fwd<float>(a, sh, st);
  else if (dtype == DTK_BF16) run_fwd<bf16>(a, sh, st);
  else run_fwd<f16>(a, sh, st);
  return dsplat::check_launch("k_norm_fwd");
}

size_t dtk_layer_norm_bwd_workspace_size(int64_t rows, int width, int dtype) {
  if (rows <= 0 || width <= 0) return 0;
  return (size_t)2 * walk_grid(rows, shape_of(width, dtype), false) * width * sizeof(float);
}

int dtk_layer_norm_bwd(int64_t rows, int width, int dtype, int wtype, const void* z, const void* dy, const void* ds,
                       const void* weight, const float* mean, const float* rstd, int add, double p, const int64_t* rng,
                       uint32_t call, void* dx, void* dresidual, void* dweight, void* dbias, void* workspace,
                       void* stream) {
  DSPLAT_REQUIRE(rows >= 0 && width > 0 && width <= (1 << 28) && rows < (1LL << 31), "dtk_layer_norm_bwd: bad sizes");
  DSPLAT_REQUIRE(type_ok(dtype) && (wtype == dtype || wtype == DTK_F32), "dtk_layer_norm_bwd: bad types");
  DSPLAT_REQUIRE(p >= 0.0 && p <= 1.0 && (p == 0.0 || (rng && add)), "dtk_layer_norm_bwd: dropout needs 0 <= p <= 1 and rng");
  DSPLAT_REQUIRE(add || (!ds && !dresidual), "dtk_layer_norm_bwd: a residual's gradient without a residual");
  const bool sums = dweight || dbias;
  DSPLAT_REQUIRE(rows == 0 || (z && mean && rstd && (!sums || workspace)), "dtk_layer_norm_bwd: null pointer");
  const Shape sh = shape_of(width, dtype);
  const int grid = rows ? walk_grid(rows, sh, add != 0) : 0;
  hipStream_t st = (hipStream_t)stream;
  const BwdArgs a = {rows, width, z, dy, ds, {weight, nullptr, wtype == DTK_F32}, mean, rstd, drop_of(p, rng, call), dx, dresidual,
                     sums ? (float*)workspace : nullptr};
  if (rows) {
    if (dtype == DTK_F32) run_bwd<float>(a, grid, sh, add != 0, st);
    else if (dtype == DTK_BF16) run_bwd<bf16>(a, grid, sh, add != 0, st);
    else run_bwd<f16>(a, grid, sh, add != 0, st);
    if (int e = dsplat::check_launch("k_norm_bwd")) return e;
  }
  if (sums) {
    const dim3 g((width + 63) / 64, 2);
    const float* part = (const float*)workspace;
    if (wtype == DTK_F32) k_norm_fold<float><<<g, kFoldThreads, 0, st>>>(grid, width, part, (float*)dweight, (float*)dbias);
    else if (wtype == DTK_BF16) k_norm_fold<bf16><<<g, kFoldThreads, 0, st>>>(grid, width, part, (bf16*)dweight, (bf16*)dbias);
    else k_norm_fold<f16><<<g, kFoldThreads, 0, st>>>(grid, width, part, (f16*)dweight, (f16*)dbias);
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
  const Drop d = drop_of(p, rng, call);
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
