// dtk_attention.hip — the C ABI of attention over chosen blocks (kernels: dtk_attention.h), the joins of
// split lists, and the plan of dk/dv.
#include "dtk_attention.h"

namespace {
using namespace dtk;

constexpr int NT = kThreads;

// Joins the parts of a split list: four channels of a row per thread. (16 sequences' one token, 8 heads, 8 parts: 4 us,
// which is a launch and two dependent reads.)
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
      const bool part = s0 + k < a.splits;  // else the last part again: left out, as 0 times its infinities would be no number
      const float f = exp2f(pm[k] - base);
      l += part ? pl[k] * f : 0.f;
      o[0] += part ? po[k].x * f : 0.f;
      o[1] += part ? po[k].y * f : 0.f;
      o[2] += part ? po[k].z * f : 0.f;
      o[3] += part ? po[k].w * f : 0.f;
    }
  }
  const int64_t i = r % a.Lq, bh = r / a.Lq, b = bh / a.Hq, h = bh % a.Hq;
  const bool valid = i < length_of(a.q_lengths, (int)b, a.Lq);
  const float inv = l > 0.f ? 1.f / l : (l != l ? l : 0.f);  // (as k_attend_fwd: 0 behind the length whatever the sums are)
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = valid ? o[e] * inv : 0.f;
  const int64_t to = ((b * a.Lq + i) * a.Hq + h) * a.D + d;
  store4<T>((T*)a.out + to, o[0], o[1], o[2], o[3]);
  if (sizeof(T) == 2 && a.rest) store_rest4<T>((T*)a.rest + to, o[0], o[1], o[2], o[3]);
  if (d == 0 && a.lse) a.lse[r] = valid ? m + log2f(l) : -INFINITY;
}

// The workgroups of dk/dv: a popular block is chosen several times as often as the mean, so a list of more than `most`
// steps is cut into equal parts, and the longest parts come first (whatever starts last then ends soon). One
// workgroup sorts by the steps of a part, eight grades to a power of two; the order within a grade does not matter. (5 us for 512 blocks, 10 for 4032. In stretches
// of equal work per XCD, so that blocks of one head share an L2, it takes 7 us more and dk/dv 249 us instead of 252.)
constexpr int kGrades = 264, kPlanThreads = 1024;
__device__ __forceinline__ int grade_of(uint32_t n) {  // 0 for the longest
  if (n < 8) return kGrades - 1 - (int)n;
  const int e = 31 - __clz(n);
  return kGrades - 1 - (8 * (e - 2) + (int)((n >> (e - 3)) & 7));
}
__global__ __launch_bounds__(kPlanThreads) void k_attend_plan(Args a, int items, int most) {
  __shared__ int at[kGrades];
  __shared__ int all, slots, splits;
  for (int i = threadIdx.x; i < kGrades; i += kPlanThreads) at[i] = 0;
  if (threadIdx.x == 0) slots = splits = 0;
  const int units = a.G << a.lg, together = 128 / a.block;  // of a tile, in a step
  const auto parts_of = [&](int i, int& grade) {
    const int64_t steps = ((int64_t)a.chosen[i] * units + together - 1) / together;
    const int n = (int)max((int64_t)1, (steps + most - 1) / most);
    grade = grade_of((uint32_t)((steps + n - 1) / n));
    return n;
  };
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kPlanThreads) {
    int grade;
    const int n = parts_of(i, grade);
    atomicAdd(&at[grade], n);
  }
  __syncthreads();
  if (threadIdx.x < 64) {  // exclusive sums, 64 grades at a time
    int before = 0;
    for (int base = 0; base < kGrades; base += 64) {
      const int i = base + (int)threadIdx.x;
      const int n = i < kGrades ? at[i] : 0;
      const int incl = (int)dsplat::wave_incl_scan((uint32_t)n, threadIdx.x);
      if (i < kGrades) at[i] = before + incl - n;
      before += __shfl(incl, 63, 64);
    }
    if (threadIdx.x == 0) all = before;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += kPlanThreads) {
    int grade, slot = 0;
    const int n = parts_of(i, grade), to = atomicAdd(&at[grade], n);
    if (n > 1) {
      slot = atomicAdd(&slots, n);
      a.split[atomicAdd(&splits, 1)] = make_int4(i, slot, n, 0);
    }
    for (int k = 0; k < n; ++k) a.plan[to + k] = make_int4(i, k, n, slot);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.planned[0] = all;
    a.planned[1] = splits;
  }
}

// Adds up the parts of dk and dv in order: four channels of a key per thread; 0 behind the lengths. (9 us for the popular
// half of 512 blocks of 64 x 128.)
template <typename T>
__global__ __launch_bounds__(NT) void k_attend_dkv_join(Args a) {
  if ((int)blockIdx.x >= a.planned[1]) return;
  const int4 e = a.split[blockIdx.x];
  const int blk = e.x % a.Tk, hk = e.x / a.Tk % a.Hkv, b = e.x / a.Tk / a.Hkv;
  const int per = a.D / 4, i = blockIdx.y * NT + threadIdx.x, row = i / per, d = (i - row * per) * 4;
  const int64_t key = (int64_t)blk * a.block + row;
  if (row >= a.block || key >= a.Lk) return;
  const bool valid = key < length_of(a.kv_lengths, b, a.Lk);
  const int64_t n = (int64_t)a.block * a.D, to = ((b * a.Lk + key) * a.Hkv + hk) * a.D + d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float s[4] = {};
    if (valid)
      for (int k = 0; k < e.z; ++k) {
        const float4 v = *(const float4*)(a.part + (2 * ((int64_t)e.y + k) + which) * n + (int64_t)row * a.D + d);
        s[0] += v.x;
        s[1] += v.y;
        s[2] += v.z;
        s[3] += v.w;
      }
    store4<T>((T*)(which ? a.dv : a.dk) + to, s[0], s[1], s[2], s[3]);
  }
}

template <typename F>
F* by_type(int dtype, F* f32, F* b16, F* h16) {
  return dtype == DTK_F32 ? f32 : dtype == DTK_BF16 ? b16 : h16;
}

// What the sizes by themselves have to keep to (the workspace sizes of others are 0).
int check_sizes(const dtk_attention* c, const char* who) {
  DSPLAT_REQUIRE(c, "%s: null pointer", who);
  DSPLAT_REQUIRE(c->B >= 0 && c->Lq >= 0 && c->Lk >= 0 && c->Hkv > 0 && c->Hq > 0 && c->Hq % c->Hkv == 0 && c->top > 0 && c->top <= 1024,
                 "%s: bad sizes", who);
  DSPLAT_REQUIRE(c->D > 0 && c->D <= 128 && c->D % 8 == 0, "%s: the head size must be a multiple of 8 up to 128", who);
  DSPLAT_REQUIRE(c->block == 32 || c->block == 64 || c->block == 128, "%s: block must be 32, 64 or 128", who);
  DSPLAT_REQUIRE(type_ok(c->dtype), "%s: bad type", who);
  DSPLAT_REQUIRE(fabsf(c->scale) < INFINITY, "%s: the scale must be a finite number", who);
  DSPLAT_REQUIRE(c->Hq / c->Hkv <= 1024, "%s: more than 1024 query heads per key head", who);
  DSPLAT_REQUIRE(c->Lq <= (1LL << 31) - 256 && c->Lk <= (1LL << 31) - 256 && c->Hq < 65536 && c->B < 65536, "%s: too large", who);
  return 0;
}
int check(const dtk_attention* c, const char* who) {
  if (int e = check_sizes(c, who)) return e;
  for (const int64_t* s : {c->q_strides, c->k_strides, c->v_strides})
    DSPLAT_REQUIRE(s[1] >= 0 && s[1] < (1LL << 24), "%s: a token stride must be below 2^24 elements", who);
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
  a.rest = c->o_rest;
  const int per = 32 * row_waves(a);
  a.rowtiles = (a.Lt * a.G + per - 1) / per;
  a.splits = splits_of((int64_t)a.Tq * a.rowtiles * a.Hkv * c->B, a.top * (a.block / 32));
  return a;
}
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// The backward's workspace: delta, what is cleared (the lists' bits and lengths), the plan of dk/dv,
// the parts in f32.
struct BwdLayout {
  size_t bits, chosen, planned, plan, split, part, end;
  int64_t items, slots;  // slots: parts of split lists, at most
  int most;              // steps of a part; 0: no plan
};
BwdLayout layout_of(const dtk_attention* c, const Args& a) {
  BwdLayout l;
  const int64_t together = 128 / a.block, units = (int64_t)a.G << a.lg;
  l.items = (int64_t)c->B * c->Hkv * a.Tk;
  // Steps of all lists, at most (a list entry that stands twice counts once).
  const int64_t steps = (int64_t)c->B * c->Hkv * a.Tq * (a.top < a.Tk ? a.top : a.Tk) * units / together;
  // A part: a 1024th of all (a few per CU, whatever the lists' lengths), and 8 steps or more. 16 scenes of 2048 f32
  // tokens of 128 channels, 512 blocks: whole lists in any order 304 us, parts of 8 steps 208 us and 9 us for their join, of
  // 4 steps 230 + 16. 4 scenes of 32256 bf16 tokens, 4032 blocks: whole lists, the longest first, 293 us; 512ths 296,
  // 1024ths 264, 2048ths 265.
  const int64_t most = steps / 1024 > 8 ? steps / 1024 : 8;
  l.most = l.items > 512 || a.Tq * units > most * together ? (int)(most < (1 << 30) ? most : 1 << 30) : 0;
  l.slots = l.most ? 2 * steps / l.most + 1 : 0;  // a list of n > most steps has fewer than 2 n / most parts
  l.bits = align256((size_t)c->B * c->Hq * c->Lq * 4);
  l.chosen = l.bits + (size_t)l.items * ((a.Tq + 31) / 32) * 4;
  l.planned = align256(l.chosen + (l.most ? (size_t)l.items * 4 : 0));
  l.plan = l.planned + 256;
  l.split = l.plan + (l.most ? (size_t)(l.items + l.slots) * sizeof(int4) : 0);
  l.part = align256(l.split + (size_t)(l.slots / 2) * sizeof(int4));
  l.end = l.part + (size_t)l.slots * 2 * a.block * c->D * 4;
  return l;
}

}  // namespace

extern "C" {

size_t dtk_block_sparse_attention_fwd_workspace_size(const dtk_attention* c) {
  if (check_sizes(c, "dtk_block_sparse_attention_fwd_workspace_size") || c->B == 0 || c->Lq == 0) return 0;
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
  if (check_sizes(c, "dtk_block_sparse_attention_bwd_workspace_size") || c->B == 0) return 0;
  const Args a = args_of(c);
  return layout_of(c, a).end;
}

int dtk_block_sparse_attention_bwd(const dtk_attention* c, const void* dout, const int64_t* dout_strides, void* dq,
                                   void* dk, void* dv, void* workspace, void* stream) {
  if (int e = check(c, "dtk_block_sparse_attention_bwd")) return e;
  if (c->B == 0) return 0;
  DSPLAT_REQUIRE((c->Lq == 0 || (dout && dout_strides && dq && c->lse && workspace && (c->dtype == DTK_F32 || c->o_rest))) && !dk == !dv && (!dk || workspace),
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
  DSPLAT_REQUIRE(l.items + l.slots < (1LL << 31), "dtk_block_sparse_attention_bwd: too large");
  a.delta = (float*)ws;
  a.bits = (uint32_t*)(ws + l.bits);
  if (l.most) {
    a.chosen = (uint32_t*)(ws + l.chosen);
    a.planned = (int*)(ws + l.planned);
    a.plan = (int4*)(ws + l.plan);
    a.split = (int4*)(ws + l.split);
    a.part = (float*)(ws + l.part);
  }
  if (int e = dsplat::zero_async(a.bits, l.planned - l.bits, st, "dtk_block_sparse_attention_bwd")) return e;
  if (c->Lq) {
    const dim3 grid(a.Tq * a.rowtiles, a.Hkv, c->B);
    if (int e = by_type(c->dtype, attend_dq<float>, attend_dq<bf16>, attend_dq<f16>)(a, row_waves(a), grid, st)) return e;
  }
  if (!a.Tk || !dk) return 0;
  if (l.most) {
    k_attend_plan<<<1, kPlanThreads, 0, st>>>(a, (int)l.items, l.most);
    if (int e = dsplat::check_launch("k_attend_plan")) return e;
  }
  if (int e = by_type(c->dtype, attend_dkv<float>, attend_dkv<bf16>, attend_dkv<f16>)(a, a.block / 32, dim3((unsigned)(l.items + l.slots)), st)) return e;
  if (l.slots < 2) return 0;
  const dim3 blocks((unsigned)(l.slots / 2), (a.block * a.D / 4 + NT - 1) / NT);
  if (c->dtype == DTK_F32) k_attend_dkv_join<float><<<blocks, NT, 0, st>>>(a);
  else if (c->dtype == DTK_BF16) k_attend_dkv_join<bf16><<<blocks, NT, 0, st>>>(a);
  else k_attend_dkv_join<f16><<<blocks, NT, 0, st>>>(a);
  return dsplat::check_launch("k_attend_dkv_join");
}

}  // extern "C"
