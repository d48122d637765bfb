// dtk_select.hip — which key blocks each tile of queries attends to, for gfx950.
//
//   qm = mean of the tile's query rows over the heads that share a key head, km = mean of the
//   block's key rows (rows behind a sequence's length do not count); score = qm . km; the `top`
//   allowed blocks of the highest score, ties to the lowest block, in ascending order, -1 behind.
//
// The means, products and scores are held in 64 bits: the answer is a set of whole numbers, and
// near scores change places with the rounding of a 32-bit sum (and so with the order in which a
// kernel adds). The work is small next to reading q and k: T_q T_k D products per key head.

#include "dtk_common.h"

namespace {
using namespace dtk;

constexpr int NT = 256;

struct Rows {
  const void* p;
  int64_t b, l, h;  // strides in elements
  const int32_t* lengths;
};
__device__ __forceinline__ int64_t length_of(const int32_t* lengths, int b, int64_t L) {
  if (!lengths) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n < L ? n : L;
}

// grid (tiles, Hkv, B): out[b][hkv][tile][D] = mean over the tile's rows and the group's heads
template <typename T>
__global__ __launch_bounds__(NT) void k_pool(Rows x, int64_t L, int D, int group, int block, double* __restrict__ out) {
  __shared__ double red[NT];
  const int t = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int64_t lo = (int64_t)t * block;
  const int n = (int)max((int64_t)0, min((int64_t)block, length_of(x.lengths, b, L) - lo));
  const int lanes = min(NT, 1 << (32 - __clz(D - 1)));  // threads per row, a power of two >= D (D <= 256)
  const int c = threadIdx.x % lanes, part = threadIdx.x / lanes, parts = NT / lanes;
  double s = 0.0;
  if (c < D) {
    const T* p = (const T*)x.p + (int64_t)b * x.b + (int64_t)hk * group * x.h + c;
    for (int i = part; i < n * group; i += parts) s += (double)(float)p[(lo + i / group) * x.l + (i % group) * x.h];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (part == 0 && c < D) {
    for (int k = 1; k < parts; ++k) s += red[k * lanes + c];
    out[(((int64_t)b * gridDim.y + hk) * gridDim.x + t) * D + c] = n ? s / (double)(n * group) : 0.0;
  }
}

// grid (Tk / 64, Tq / 16, B * Hkv): 16 x 64 scores per workgroup, the pooled rows staged in LDS
constexpr int SQ = 16, SK = 64, SD = 16;
__global__ __launch_bounds__(NT) void k_scores(int Tq, int Tk, int D, const double* __restrict__ qm,
                                               const double* __restrict__ km, double* __restrict__ score) {
  __shared__ double sq[SQ][SD + 1], sk[SK][SD + 1];
  const int64_t z = blockIdx.z;
  const int q0 = blockIdx.y * SQ, k0 = blockIdx.x * SK;
  const int tk = threadIdx.x % 16, tq = threadIdx.x / 16;  // row q0 + tq, columns k0 + tk + 16 j
  double acc[4] = {};
  for (int d0 = 0; d0 < D; d0 += SD) {
    __syncthreads();
    const int d = threadIdx.x % 16, r = threadIdx.x / 16;
    sq[r][d] = q0 + r < Tq && d0 + d < D ? qm[(z * Tq + q0 + r) * D + d0 + d] : 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      sk[r + 16 * j][d] = k0 + r + 16 * j < Tk && d0 + d < D ? km[(z * Tk + k0 + r + 16 * j) * D + d0 + d] : 0.0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SD; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = __builtin_fma(sq[tq][i], sk[tk + 16 * j][i], acc[j]);
  }
  if (q0 + tq < Tq)
    for (int j = 0; j < 4; ++j)
      if (k0 + tk + 16 * j < Tk) score[(z * Tq + q0 + tq) * Tk + k0 + tk + 16 * j] = acc[j];
}

// The order of doubles as unsigned numbers; 0 is kept for blocks that may not be chosen. A score
// that is no number ranks below every number.
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return 1;
  v += 0.0;  // -0 and 0 are the same score
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// grid (Tq, B * Hkv): a radix descent over the row's keys, 8 bits at a time, finds the key of the
// last chosen place and how many equal ones are taken; a scan over the row writes the places.
__global__ __launch_bounds__(NT) void k_choose(int Tq, int Tk, int Hkv, int64_t Lq, int64_t Lk, int block, int top,
                                               const int32_t* __restrict__ q_lengths,
                                               const int32_t* __restrict__ kv_lengths,
                                               const uint8_t* __restrict__ allowed, const double* __restrict__ score,
                                               int32_t* __restrict__ index) {
  __shared__ uint32_t hist[256];
  __shared__ uint64_t s_key;
  __shared__ int s_need, s_any;
  __shared__ int wave_n[2][NT / 64];
  const int t = blockIdx.x, z = blockIdx.y, b = z / Hkv;
  const int64_t nq = length_of(q_lengths, b, Lq), nk = length_of(kv_lengths, b, Lk);
  int32_t* out = index + ((int64_t)z * Tq + t) * top;
  const int blocks = (int)((nk + block - 1) / block);  // blocks with a key
  if ((int64_t)t * block >= nq || blocks == 0) {
    for (int i = threadIdx.x; i < top; i += NT) out[i] = -1;
    return;
  }
  const double* row = score + ((int64_t)z * Tq + t) * Tk;
  const uint8_t* may = allowed ? allowed + (int64_t)t * Tk : nullptr;
  auto key_at = [&](int i) -> uint64_t { return (i < blocks && (!may || may[i])) ? order_key(row[i]) : 0ull; };
  if (threadIdx.x == 0) s_any = 0;
  __syncthreads();
  int any = 0;
  for (int i = threadIdx.x; i < blocks; i += NT) any += key_at(i) != 0;
  atomicAdd(&s_any, any);
  __syncthreads();
  const int have = s_any;
  const int want = min(top, have);
  uint64_t key = 1;   // every allowed block, if no more are allowed than wanted
  int equal = blocks;
  if (have > top) {
    uint64_t prefix = 0;
    int need = top;
    for (int shift = 56; shift >= 0; shift -= 8) {
      hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < blocks; i += NT) {
        const uint64_t k = key_at(i);
        if (k && (shift == 56 || (k >> (shift + 8)) == prefix)) atomicAdd(&hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int d = 255, n = need;
        while (d > 0 && (int)hist[d] < n) n -= hist[d--];
        s_key = (prefix << 8) | (uint64_t)d;
        s_need = n;
      }
      __syncthreads();
      prefix = s_key;
      need = s_need;
    }
    key = prefix;
    equal = need;  // of the blocks with exactly this key, the lowest `need`
  }
  // ascending places: above = key greater, tie = key equal (the first `equal` of them)
  int above0 = 0, tie0 = 0;  // before this chunk
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int base = 0; base < blocks; base += NT) {
    const uint64_t k = base + (int)threadIdx.x < blocks ? key_at(base + threadIdx.x) : 0ull;
    const bool up = have > top ? k > key : k != 0, tie = have > top && k == key;
    const uint64_t mu = __ballot(up), mt = __ballot(tie);
    if (lane == 0) {
      wave_n[0][w] = __popcll(mu);
      wave_n[1][w] = __popcll(mt);
    }
    __syncthreads();
    int u = above0 + __popcll(mu & dsplat::lanemask_lt(lane)), e = tie0 + __popcll(mt & dsplat::lanemask_lt(lane));
    for (int j = 0; j < NT / 64; ++j) {
      if (j < w) {
        u += wave_n[0][j];
        e += wave_n[1][j];
      }
      above0 += wave_n[0][j];
      tie0 += wave_n[1][j];
    }
    if (up || (tie && e < equal)) out[u + min(e, equal)] = base + threadIdx.x;
    __syncthreads();
  }
  for (int i = want + threadIdx.x; i < top; i += NT) out[i] = -1;
}

inline int64_t tiles_of(int64_t L, int block) { return (L + block - 1) / block; }

template <typename T>
void pool(const Rows& x, int64_t L, int D, int group, int block, int tiles, int Hkv, int B, double* out, hipStream_t st) {
  k_pool<T><<<dim3(tiles, Hkv, B), NT, 0, st>>>(x, L, D, group, block, out);
}

}  // namespace

extern "C" {

size_t dtk_select_blocks_workspace_size(int B, int64_t Lq, int64_t Lk, int Hkv, int D, int block) {
  if (B <= 0 || Lq <= 0 || Lk <= 0 || Hkv <= 0 || D <= 0 || block <= 0) return 0;
  const size_t tq = tiles_of(Lq, block), tk = tiles_of(Lk, block);
  return (size_t)B * Hkv * ((tq + tk) * D + tq * tk) * sizeof(double);
}

int dtk_select_blocks(int B, int64_t Lq, int64_t Lk, int Hq, int Hkv, int D, int block, int top, int dtype,
                      const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                      const int32_t* q_lengths, const int32_t* kv_lengths, const uint8_t* allowed, int32_t* index,
                      void* workspace, void* stream) {
  DSPLAT_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D > 0 && D <= 256 && top > 0,
                 "dtk_select_blocks: bad sizes");
  DSPLAT_REQUIRE(block == 32 || block == 64 || block == 128, "dtk_select_blocks: block must be 32, 64 or 128");
  DSPLAT_REQUIRE(type_ok(dtype), "dtk_select_blocks: bad type");
  DSPLAT_REQUIRE(Lq < (1LL << 31) && Lk < (1LL << 31) && (int64_t)B * Hkv < 65536 && Hq < 65536, "dtk_select_blocks: too large");
  if (B == 0 || Lq == 0) return 0;
  const int Tq = (int)tiles_of(Lq, block), Tk = (int)tiles_of(Lk, block);
  DSPLAT_REQUIRE(Tq <= 16 * 65535, "dtk_select_blocks: too large");
  DSPLAT_REQUIRE(index && (Lk == 0 || (q && k && q_strides && k_strides && workspace)), "dtk_select_blocks: null pointer");
  hipStream_t st = (hipStream_t)stream;
  double* qm = (double*)workspace;
  double* km = qm + (size_t)B * Hkv * Tq * D;
  double* score = km + (size_t)B * Hkv * Tk * D;
  if (Lk > 0) {
    const Rows rq = {q, q_strides[0], q_strides[1], q_strides[2], q_lengths};
    const Rows rk = {k, k_strides[0], k_strides[1], k_strides[2], kv_lengths};
    const int group = Hq / Hkv;
    if (dtype == DTK_F32) {
      pool<float>(rq, Lq, D, group, block, Tq, Hkv, B, qm, st);
      pool<float>(rk, Lk, D, 1, block, Tk, Hkv, B, km, st);
    } else if (dtype == DTK_BF16) {
      pool<bf16>(rq, Lq, D, group, block, Tq, Hkv, B, qm, st);
      pool<bf16>(rk, Lk, D, 1, block, Tk, Hkv, B, km, st);
    } else {
      pool<f16>(rq, Lq, D, group, block, Tq, Hkv, B, qm, st);
      pool<f16>(rk, Lk, D, 1, block, Tk, Hkv, B, km, st);
    }
    if (int e = dsplat::check_launch("k_pool")) return e;
    k_scores<<<dim3((Tk + SK - 1) / SK, (Tq + SQ - 1) / SQ, B * Hkv), NT, 0, st>>>(Tq, Tk, D, qm, km, score);
    if (int e = dsplat::check_launch("k_scores")) return e;
  }
  k_choose<<<dim3(Tq, B * Hkv), NT, 0, st>>>(Tq, Tk, Hkv, Lq, Lk, block, top, q_lengths, kv_lengths, allowed, score, index);
  return dsplat::check_launch("k_choose");
}

}  // extern "C"
