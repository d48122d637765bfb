// dtk_attention.hip — the C ABI of attention over chosen blocks (kernels: dtk_attention.h), the join of
// split lists, and who chose which block for the backward.
#include "dtk_attention.h"

namespace {
using namespace dtk;

constexpr int NT = kThreads;

// Joins the parts of a split list: four channels of a row per thread.
template <typename T>
__global__ __launch_bounds__(NT) void k_attend_join(Args a, int64_t rows) {
  const int per = a.D / 4;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t r = id / per;
  const int d = (int)(id % per) * 4;
  if (r >= rows) return;
  float m = -INFINITY, l = 0.f, o[4] = {};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {  // eight parts' values on their way together
    float pm[8], pl[8];
    float4 po[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t at = (int64_t)min(s0 + k, a.splits - 1) * rows + r;
      pm[k] = a.part_m[at];
      pl[k] = a.part_l[at];
      po[k] = *(const float4*)(a.part + at * a.D + d);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) mn = fmaxf(mn, pm[k]);
    const float base = mn == -INFINITY ? 0.f : mn, f0 = exp2f(m - base);
    m = mn;
    l *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = s0 + k < a.splits ? exp2f(pm[k] - base) : 0.f;
      l += pl[k] * f;
      o[0] += po[k].x * f;
      o[1] += po[k].y * f;
      o[2] += po[k].z * f;
      o[3] += po[k].w * f;
    }
  }
  const int64_t i = r % a.Lq, bh = r / a.Lq, b = bh / a.Hq, h = bh % a.Hq;
  const bool valid = i < length_of(a.q_lengths, (int)b, a.Lq);
  const float inv = valid && l > 0.f ? 1.f / l : (l != l ? l : 0.f);
  store4<T>((T*)a.out + ((b * a.Lq + i) * a.Hq + h) * a.D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (d == 0 && a.lse) a.lse[r] = valid ? m + log2f(l) : -INFINITY;
}

// Which tiles chose a block: bits [B, Hkv, Tk, ceil(Tq / 32)]; and how many did (a block named twice counts
// once: whoever sets the bit counts it).
__global__ __launch_bounds__(NT) void k_attend_mark(Args a) {
  const int t = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  if ((int64_t)t * a.block >= length_of(a.q_lengths, b, a.Lq)) return;
  const int32_t* idx = a.index + (((int64_t)b * a.Hkv + hk) * a.Tq + t) * a.top;
  const int words = (a.Tq + 31) / 32;
  for (int j = threadIdx.x; j < a.top; j += NT) {
    const int v = idx[j];
    if (v < 0 || v >= a.Tk) continue;
    const int64_t item = ((int64_t)b * a.Hkv + hk) * a.Tk + v;
    const uint32_t bit = 1u << (t % 32);
    if (!(atomicOr(a.bits + item * words + t / 32, bit) & bit) && a.chosen) atomicAdd(a.chosen + item, 1u);
  }
}

// The blocks with the longest lists first: they are workgroups of dk/dv, the longest of which would
// otherwise run on alone at the end (a popular block is chosen several times as often as the mean). One
// workgroup sorts by the list's length, eight steps to a power of two; the order within a step does not matter.
constexpr int kSteps = 264, kOrderThreads = 1024;
__device__ __forceinline__ int length_step(uint32_t n) {  // 0 for the longest
  if (n < 8) return kSteps - 1 - (int)n;
  const int e = 31 - __clz(n);
  return kSteps - 1 - (8 * (e - 2) + (int)((n >> (e - 3)) & 7));
}
__global__ __launch_bounds__(kOrderThreads) void k_attend_order(Args a, int items) {
  __shared__ int at[kSteps];
  for (int i = threadIdx.x; i < kSteps; i += kOrderThreads) at[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kOrderThreads) atomicAdd(&at[length_step(a.chosen[i])], 1);
  __syncthreads();
  if (threadIdx.x < 64) {  // exclusive sums, 64 steps at a time
    int before = 0;
    for (int base = 0; base < kSteps; base += 64) {
      const int i = base + (int)threadIdx.x;
      const int n = i < kSteps ? at[i] : 0;
      const int incl = (int)dsplat::wave_incl_scan((uint32_t)n, threadIdx.x);
      if (i < kSteps) at[i] = before + incl - n;
      before += __shfl(incl, 63, 64);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kOrderThreads) a.order[atomicAdd(&at[length_step(a.chosen[i])], 1)] = i;
}

// Adds up the parts of dk and dv in order: four channels of a key per thread; 0 behind the lengths.
template <typename T>
__global__ __launch_bounds__(NT) void k_attend_dkv_join(Args a, int64_t n, int parts) {
  const int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 4;
  if (i >= n) return;
  const int64_t key = i / ((int64_t)a.Hkv * a.D), b = key / a.Lk;
  const bool valid = key - b * a.Lk < length_of(a.kv_lengths, (int)b, a.Lk);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float s[4] = {};
    if (valid)
      for (int k = 0; k < parts; ++k) {
        const float4 v = *(const float4*)(a.part + (2 * k + which) * n + i);
        s[0] += v.x;
        s[1] += v.y;
        s[2] += v.z;
        s[3] += v.w;
      }
    store4<T>((T*)(which ? a.dv : a.dk) + i, s[0], s[1], s[2], s[3]);
  }
}

template <typename F>
F* by_type(int dtype, F* f32, F* b16, F* h16) {
  return dtype == DTK_F32 ? f32 : dtype == DTK_BF16 ? b16 : h16;
}

int check(const dtk_attention* c, const char* who) {
  DSPLAT_REQUIRE(c, "%s: null pointer", who);
  DSPLAT_REQUIRE(c->B >= 0 && c->Lq >= 0 && c->Lk >= 0 && c->Hkv > 0 && c->Hq > 0 && c->Hq % c->Hkv == 0 && c->top > 0 && c->top <= 1024,
                 "%s: bad sizes", who);
  DSPLAT_REQUIRE(c->D > 0 && c->D <= 128 && c->D % 8 == 0, "%s: the head size must be a multiple of 8 up to 128", who);
  DSPLAT_REQUIRE(c->block == 32 || c->block == 64 || c->block == 128, "%s: block must be 32, 64 or 128", who);
  DSPLAT_REQUIRE(type_ok(c->dtype), "%s: bad type", who);
  DSPLAT_REQUIRE(c->Hq / c->Hkv <= 1024, "%s: more than 1024 query heads per key head", who);
  for (const int64_t* s : {c->q_strides, c->k_strides, c->v_strides})
    DSPLAT_REQUIRE(s[1] >= 0 && s[1] < (1LL << 24), "%s: a token stride must be below 2^24 elements", who);
  DSPLAT_REQUIRE(c->Lq <= (1LL << 31) - 256 && c->Lk <= (1LL << 31) - 256 && c->Hq < 65536 && c->B < 65536, "%s: too large", who);
  DSPLAT_REQUIRE(c->B == 0 || c->Lq == 0 || (c->q && c->o && c->index && (c->Lk == 0 || (c->k && c->v))), "%s: null pointer", who);
  return 0;
}
Strided strided(const void* p, const int64_t* s) { return {p, s[0], s[1], s[2]}; }
Args args_of(const dtk_attention* c) {
  Args a = {};
  a.Lq = c->Lq;
  a.Lk = c->Lk;
  a.Hq = c->Hq;
  a.Hkv = c->Hkv;
  a.G = c->Hq / c->Hkv;
  a.D = c->D;
  a.block = c->block;
  a.top = c->top;
  a.Tq = (int)((c->Lq + c->block - 1) / c->block);
  a.Tk = (int)((c->Lk + c->block - 1) / c->block);
  a.Lt = (int)(c->Lq < c->block ? (c->Lq > 0 ? c->Lq : 1) : c->block);
  a.lg = c->block == 32 ? 0 : c->block == 64 ? 1 : 2;
  a.group_magic = (uint32_t)((0x100000000ull + a.G - 1) / a.G);
  a.scale = c->scale;
  a.scale2 = fmaxf(fabsf(c->scale) * kLog2e, 1.17549435e-38f);
  a.q = strided(c->q, c->q_strides);
  a.k = strided(c->k, c->k_strides);
  a.v = strided(c->v, c->v_strides);
  a.index = c->index;
  a.q_lengths = c->q_lengths;
  a.kv_lengths = c->kv_lengths;
  a.out = c->o;
  a.lse = c->lse;
  const int per = 32 * row_waves(a);
  a.rowtiles = (a.Lt * a.G + per - 1) / per;
  a.splits = splits_of((int64_t)a.Tq * a.rowtiles * a.Hkv * c->B, a.top * (a.block / 32));
  return a;
}
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// The backward's workspace: delta, then what is cleared (the largest |do|, the lists' bits and lengths), the order.
struct BwdLayout {
  size_t gmax, bits, chosen, order, end;
  size_t part;
  int64_t items;
  bool sorted;
  int parts;
};
BwdLayout layout_of(const dtk_attention* c, const Args& a) {
  BwdLayout l;
  l.items = (int64_t)c->B * c->Hkv * a.Tk;
  l.sorted = l.items > 512;
  l.gmax = align256((size_t)c->B * c->Hq * c->Lq * 4);
  l.bits = l.gmax + 256;
  l.chosen = l.bits + (size_t)l.items * ((a.Tq + 31) / 32) * 4;
  l.order = l.chosen + (l.sorted ? (size_t)l.items * 4 : 0);
  // Parts of the lists, in f32: where the blocks are too few to fill the chip and to even out their lists, down to
  // 8 steps of the mean list each. (2 x 16384 tokens, 4 heads on one: 512 workgroups of 128 steps 390 us, four
  // parts 215 us and 27 us for their join.)
  const int64_t steps = a.Tk ? (int64_t)a.Tq * a.top * a.G * (a.block / 32) / a.Tk / (4 * 32 / a.block ? 4 * 32 / a.block : 1) : 0;
  l.parts = 1;
  while (l.items * l.parts < 2048 && l.parts * 16 <= steps) l.parts *= 2;
  l.part = align256(l.order + (l.sorted ? (size_t)l.items * 4 : 0));
  l.end = l.part + (l.parts > 1 ? (size_t)l.parts * 2 * c->B * c->Lk * c->Hkv * c->D * 4 : 0);
  return l;
}

}  // namespace

extern "C" {

size_t dtk_block_sparse_attention_fwd_workspace_size(const dtk_attention* c) {
  if (!c || c->B <= 0 || c->Lq <= 0 || c->Hq <= 0 || c->Hkv <= 0 || c->block <= 0) return 0;
  const Args a = args_of(c);
  if (a.splits == 1) return 0;
  return (size_t)a.splits * c->B * c->Hq * c->Lq * (c->D + 2) * sizeof(float);
}

int dtk_block_sparse_attention_fwd(const dtk_attention* c, void* workspace, void* stream) {
  if (int e = check(c, "dtk_block_sparse_attention_fwd")) return e;
  if (c->B == 0 || c->Lq == 0) return 0;
  Args a = args_of(c);
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = (int64_t)c->B * c->Hq * c->Lq;
  if (a.splits > 1) {
    DSPLAT_REQUIRE(workspace, "dtk_block_sparse_attention_fwd: null workspace");
    a.part = (float*)workspace;
    a.part_m = a.part + a.splits * rows * a.D;
    a.part_l = a.part_m + a.splits * rows;
  }
  const dim3 grid(a.Tq * a.rowtiles, a.Hkv, c->B * a.splits);
  if (int e = by_type(c->dtype, attend_fwd<float>, attend_fwd<bf16>, attend_fwd<f16>)(a, row_waves(a), grid, st)) return e;
  if (a.splits == 1) return 0;
  const unsigned blocks = (unsigned)((rows * (a.D / 4) + NT - 1) / NT);
  if (c->dtype == DTK_F32) k_attend_join<float><<<blocks, NT, 0, st>>>(a, rows);
  else if (c->dtype == DTK_BF16) k_attend_join<bf16><<<blocks, NT, 0, st>>>(a, rows);
  else k_attend_join<f16><<<blocks, NT, 0, st>>>(a, rows);
  return dsplat::check_launch("k_attend_join");
}

size_t dtk_block_sparse_attention_bwd_workspace_size(const dtk_attention* c) {
  if (!c || c->B <= 0 || c->Lq < 0 || c->Lk < 0 || c->Hq <= 0 || c->Hkv <= 0 || c->block <= 0) return 0;
  const Args a = args_of(c);
  return layout_of(c, a).end;
}

int dtk_block_sparse_attention_bwd(const dtk_attention* c, const void* dout, const int64_t* dout_strides, void* dq,
                                   void* dk, void* dv, void* workspace, void* stream) {
  if (int e = check(c, "dtk_block_sparse_attention_bwd")) return e;
  if (c->B == 0) return 0;
  DSPLAT_REQUIRE((c->Lq == 0 || (dout && dout_strides && dq && c->lse && workspace)) && (c->Lk == 0 || (dk && dv && workspace)),
                 "dtk_block_sparse_attention_bwd: null pointer");
  DSPLAT_REQUIRE(c->Lq == 0 || (dout_strides[1] >= 0 && dout_strides[1] < (1LL << 24)),
                 "dtk_block_sparse_attention_bwd: a token stride must be below 2^24 elements");
  Args a = args_of(c);
  a.splits = 1;
  hipStream_t st = (hipStream_t)stream;
  a.o = {c->o, c->Lq * c->Hq * c->D, (int64_t)c->Hq * c->D, c->D};
  if (c->Lq) a.g = strided(dout, dout_strides);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  char* ws = (char*)workspace;
  const BwdLayout l = layout_of(c, a);
  DSPLAT_REQUIRE(l.items < (1LL << 31), "dtk_block_sparse_attention_bwd: too large");
  a.delta = (float*)ws;
  a.gmax = (uint32_t*)(ws + l.gmax);
  a.bits = (uint32_t*)(ws + l.bits);
  if (l.sorted) {
    a.chosen = (uint32_t*)(ws + l.chosen);
    a.order = (int32_t*)(ws + l.order);
  }
  if (int e = dsplat::zero_async(a.gmax, l.order - l.gmax, st, "dtk_block_sparse_attention_bwd")) return e;
  if (c->Lq) {
    const dim3 grid(a.Tq * a.rowtiles, a.Hkv, c->B);
    if (int e = by_type(c->dtype, attend_dq<float>, attend_dq<bf16>, attend_dq<f16>)(a, row_waves(a), grid, st)) return e;
    if (a.Tk) {
      k_attend_mark<<<dim3(a.Tq, a.Hkv, c->B), NT, 0, st>>>(a);
      if (int e = dsplat::check_launch("k_attend_mark")) return e;
    }
  }
  if (!a.Tk) return 0;
  if (l.sorted) {
    k_attend_order<<<1, kOrderThreads, 0, st>>>(a, (int)l.items);
    if (int e = dsplat::check_launch("k_attend_order")) return e;
  }
  a.part = (float*)(ws + l.part);
  if (int e = by_type(c->dtype, attend_dkv<float>, attend_dkv<bf16>, attend_dkv<f16>)(a, a.block / 32, dim3((unsigned)l.items, l.parts), st)) return e;
  if (l.parts == 1) return 0;
  const int64_t n = (int64_t)c->B * c->Lk * c->Hkv * c->D;
  const unsigned blocks = (unsigned)((n / 4 + NT - 1) / NT);
  if (c->dtype == DTK_F32) k_attend_dkv_join<float><<<blocks, NT, 0, st>>>(a, n, l.parts);
  else if (c->dtype == DTK_BF16) k_attend_dkv_join<bf16><<<blocks, NT, 0, st>>>(a, n, l.parts);
  else k_attend_dkv_join<f16><<<blocks, NT, 0, st>>>(a, n, l.parts);
  return dsplat::check_launch("k_attend_dkv_join");
}

}  // extern "C"
