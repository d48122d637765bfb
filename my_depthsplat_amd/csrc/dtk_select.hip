// dtk_select.hip — which key blocks each tile of queries attends to, for gfx950.
//
//   qm = mean of the tile's query rows over the heads that share a key head, km = mean of the
//   block's key rows (rows behind a sequence's length do not count); score = qm . km; the `top`
//   allowed blocks of the highest score, ties to the lowest block, in ascending order, -1 behind.
//
// The means, products and scores are held in 64 bits: the answer is a set of whole numbers, and
// near scores change places with the rounding of a 32-bit sum (and so with the order in which a
// kernel adds). The work is small next to reading q and k: T_q T_k D products per key head.
//
// Measured, pooled rows / scores / choice: 4 scenes of 32256 bf16 tokens (504 x 504 blocks of 64), 2 heads of 64: 13.5 us
// (4.0 TB/s), 11.5 us, 12.5 us; 92160 tokens (1440 x 1440): 13 us, 22.5 us (24 TFLOP/s in 64 bits and 33 MB of scores), 28 us. The
// scores' and the choice's time goes into the latency of reads behind the L2 (two thirds of the choice's cycles wait).

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

// What the pooled rows of q (grid.x < Tq) and k (behind them) are made of; both in one launch.
struct PoolArgs {
  Rows x[2];
  int64_t L[2];
  int group[2];  // heads that share a pooled row
  int tiles[2];
  int D, pitch, block;
  double* out[2];  // [B, Hkv], packed (below): zeros from D on
};
inline int pitch_of(int D) { return (D + 7) & ~7; }
__host__ __device__ inline int64_t padded(int64_t tiles) { return (tiles + 15) & ~(int64_t)15; }
// Where channel d of pooled row t lies: 16 rows together, in the order in which the matrix instruction's lanes read
// them (lane group lane / 16 takes a quarter of the channels, two at a time), so that a load is 1 KB in a row. (Rows one
// after the other put the 64 lanes of a load on 64 lines: the scores of 360 x 360 and 1440 x 1440 took 28 us instead of 17 on average.)
__device__ __forceinline__ int64_t packed(int t, int d, int pitch) {
  const int per = pitch / 4, quarter = d / per, i = d % per;
  return ((int64_t)(t / 16) * (per / 2) + i / 2) * 128 + (quarter * 16 + t % 16) * 2 + i % 2;
}

// One wave per tile: a lane sums one 16-byte piece of every (64 / pieces)-th row, the lanes of a piece are folded through
// LDS in a fixed order.
template <typename T, bool VEC>
__global__ __launch_bounds__(NT) void k_pool(PoolArgs a) {
  constexpr int N = VEC ? Vec<T>::N : 1;
  __shared__ double folds[NT / 64][N * 64];
  const int lane = threadIdx.x & 63, number = blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (number >= a.tiles[0] + a.tiles[1]) return;  // (the waves share nothing)
  const int which = number >= a.tiles[0], t = number - (which ? a.tiles[0] : 0);
  const int hk = blockIdx.y, b = blockIdx.z, tiles = a.tiles[which], group = a.group[which];
  double* red = folds[threadIdx.x >> 6];
  const Rows x = a.x[which];
  const int64_t lo = (int64_t)t * a.block;
  const int n = (int)max((int64_t)0, min((int64_t)a.block, length_of(x.lengths, b, a.L[which]) - lo));
  const T* rows = (const T*)x.p + (int64_t)b * x.b + (int64_t)hk * group * x.h + lo * x.l;
  double* out = a.out[which] + ((int64_t)b * gridDim.y + hk) * padded(tiles) * a.pitch;
  // (a division: a mean by the rounded reciprocal of 75 rows may be above their common value, and equal blocks no tie)
  const double count = n ? (double)n * group : 1.0;
  for (int first = 0; first < a.pitch; first += 64 * N) {  // (once where rows are vectors: D <= 256)
    const int pieces = max(1, min(64, a.D / N - first / N)), parts = 64 / pieces;
    const int c = lane % pieces, part = lane / pieces;
    const T* p = rows + first + c * N;
    double s[N] = {};
    if (part < parts && first + c * N < a.D) {
      for (int g = 0; g < group; ++g)
#pragma unroll 8
        for (int i = part; i < n; i += parts) {
          if constexpr (VEC) {
            const Vec<T> v = load_vec(p + i * x.l + g * x.h);
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] += (double)(float)v.v[e];
          } else {
            s[0] += (double)(float)p[i * x.l + g * x.h];
          }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the sums before are read
#pragma unroll
    for (int e = 0; e < N; ++e) red[e * 64 + lane] = s[e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int end = min(a.pitch, first + 64 * N);
    for (int d = first + lane; d < end; d += 64) {
      double v = 0.0;
      if (d < a.D)
        for (int k = 0; k < parts; ++k) v += red[(d - first) % N * 64 + k * pieces + (d - first) / N];
      out[packed(t, d, a.pitch)] = v / count;
    }
  }
}

// Scores on the 64-bit matrix instruction (16 x 16 x 4): a wave takes 32 query tiles x 64 key
// blocks, the workgroup's 4 waves stand side by side over 256 blocks.
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
__global__ __launch_bounds__(NT) void k_scores(int Tq, int Tk, int pitch, const double* __restrict__ qm,
                                               const double* __restrict__ km, double* __restrict__ score) {
  const int64_t z = blockIdx.z;
  const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const int q0 = blockIdx.y * 32, k0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
  if (k0 >= Tk) return;
  const int steps = pitch / 8;
  const int qlast = (int)padded(Tq) - 16, klast = (int)padded(Tk) - 16;  // groups behind the last are read as the last
  const double *ap[2], *bp[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) ap[i] = qm + (z * padded(Tq) + min(q0 + 16 * i, qlast)) * pitch + lane * 2;
#pragma unroll
  for (int j = 0; j < 4; ++j) bp[j] = km + (z * padded(Tk) + min(k0 + 16 * j, klast)) * pitch + lane * 2;
  f64x4 acc[2][4] = {};
#pragma unroll 2
  for (int d = 0; d < steps; ++d) {
    f64x2 av[2], bv[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) av[i] = *(const f64x2*)(ap[i] + d * 128);
#pragma unroll
    for (int j = 0; j < 4; ++j) bv[j] = *(const f64x2*)(bp[j] + d * 128);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(av[i][e], bv[j][e], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int q = q0 + 16 * i + 4 * r + quarter;
      if (q >= Tq) continue;
      double* out = score + (z * Tq + q) * Tk + k0 + col;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + 16 * j + col < Tk) out[16 * j] = acc[i][j][r];
    }
}

// The order of doubles as unsigned numbers; 0 is kept for blocks that may not be chosen. A score
// that is no number ranks below every number.
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return 1;
  v += 0.0;  // -0 and 0 are the same score
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

struct ChooseArgs {
  int Tq, Tk, Hkv, block, top;
  int64_t Lq, Lk, rows;
  const int32_t *q_lengths, *kv_lengths;
  const uint8_t* allowed;
  const double *score, *qm, *km;
  int pitch;
  int32_t* index;
};

// A wave per tile, 64 NV >= Tk keys in registers (place 64 j + lane in slot j). The key of the last chosen
// place is found from its highest bit down: a bit is kept if at least `top` keys reach the number with
// it. As soon as exactly `top` do, they are the answer: for scores that differ early, as they
// do, well before the lower 32 bits are looked at. (Halving the interval of the scores instead takes
// fewer turns, but they are not what the time goes into: 27 and 13 us against 28 and 12.5 for 1440 and 360 blocks.)
// SCORE: the wave takes its tile's scores itself, a lane those of its blocks, a launch less (scored_by_choice: where that
// pays).
template <int NV, bool SCORE>
__global__ __launch_bounds__(NT) void k_choose(ChooseArgs a) {
  const int64_t row = (int64_t)blockIdx.x * (NT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 63, t = (int)(row % a.Tq), b = (int)(row / a.Tq / a.Hkv);
  const int64_t nq = length_of(a.q_lengths, b, a.Lq), nk = length_of(a.kv_lengths, b, a.Lk);
  int32_t* out = a.index + row * a.top;
  const int blocks = (int64_t)t * a.block < nq ? (int)((nk + a.block - 1) / a.block) : 0;  // blocks with a key
  const double* score = a.score + row * a.Tk;
  const uint8_t* may = a.allowed ? a.allowed + (int64_t)t * a.Tk : nullptr;
  if (blocks == 0) {  // (there may be no scores at all: nothing is read)
    for (int i = lane; i < a.top; i += 64) out[i] = -1;
    return;
  }
  uint32_t hi[NV], lo[NV];
  int have = 0;
  double v[NV];
  uint8_t ok[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {  // all on their way together
    const int i = min(64 * j + lane, a.Tk - 1);
    if (!SCORE) v[j] = score[i];
    ok[j] = may ? may[i] : 1;
  }
  if constexpr (SCORE) {
    const int64_t z = row / a.Tq;
    const double *q = a.qm + z * padded(a.Tq) * a.pitch, *k = a.km + z * padded(a.Tk) * a.pitch;
    const double* kp[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = 0.0;
      kp[j] = k + packed(min(64 * j + lane, a.Tk - 1), 0, a.pitch);
    }
    q += packed(t, 0, a.pitch);
    for (int quarter = 0; quarter < 4; ++quarter)
#pragma unroll 4
      for (int i = 0; i < a.pitch / 8; ++i) {  // two channels each
        const f64x2 qv = *(const f64x2*)(q + quarter * 32 + i * 128);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const f64x2 kv = *(const f64x2*)(kp[j] + quarter * 32 + i * 128);
          v[j] = fma(qv[0], kv[0], v[j]);
          v[j] = fma(qv[1], kv[1], v[j]);
        }
      }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint64_t k = 64 * j + lane < blocks && ok[j] ? order_key(v[j]) : 0;
    hi[j] = (uint32_t)(k >> 32);
    lo[j] = (uint32_t)k;
    have += __popcll(__ballot(k != 0));
  }
  uint32_t th = 0, tl = 1;  // every allowed block, if no more are allowed than wanted
  int reach = have;         // keys at or above (th, tl)
  if (have > a.top) {
    tl = 0;
    for (int bit = 31; bit >= 0 && reach != a.top; --bit) {
      const uint32_t c = th | (1u << bit);
      int n = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) n += __popcll(__ballot(hi[j] >= c));
      if (n >= a.top) {
        th = c;
        reach = n;
      }
    }
    if (reach != a.top) {
      int above = 0;  // keys whose upper half is larger
#pragma unroll
      for (int j = 0; j < NV; ++j) above += __popcll(__ballot(hi[j] > th));
      for (int bit = 31; bit >= 0 && reach != a.top; --bit) {
        const uint32_t c = tl | (1u << bit);
        int n = above;
#pragma unroll
        for (int j = 0; j < NV; ++j) n += __popcll(__ballot(hi[j] == th && lo[j] >= c));
        if (n >= a.top) {
          tl = c;
          reach = n;
        }
      }
    }
  }
  // equal keys beyond `top`: the lowest places of them are taken
  int ties = reach - min(reach, a.top), equal = 0;
  if (ties > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) equal += __popcll(__ballot(hi[j] == th && lo[j] == tl));
  }
  const int taken = equal - ties;
  int at = 0, tied = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const bool tie = ties > 0 && hi[j] == th && lo[j] == tl;
    const bool up = !tie && (hi[j] > th || (hi[j] == th && lo[j] >= tl));
    const uint64_t mt = __ballot(tie), mu = __ballot(up);
    const int before = tied + __popcll(mt & dsplat::lanemask_lt(lane));
    if (up || (tie && before < taken)) out[at + __popcll(mu & dsplat::lanemask_lt(lane)) + min(before, taken)] = 64 * j + lane;
    at += __popcll(mu);
    tied += __popcll(mt);
  }
  for (int i = min(have, a.top) + lane; i < a.top; i += 64) out[i] = -1;
}

// More blocks than registers hold: a workgroup per tile, a radix descent over the row's keys 8 bits at a
// time; then a scan over the row writes the places.
__global__ __launch_bounds__(NT) void k_choose_long(ChooseArgs a) {
  __shared__ int hist[256], wave_n[2][NT / 64];
  __shared__ int s_digit, s_need, s_have;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = (int)(row % a.Tq), b = (int)(row / a.Tq / a.Hkv);
  const int64_t nq = length_of(a.q_lengths, b, a.Lq), nk = length_of(a.kv_lengths, b, a.Lk);
  int32_t* out = a.index + row * a.top;
  const int blocks = (int64_t)t * a.block < nq ? (int)((nk + a.block - 1) / a.block) : 0;
  const double* score = a.score + row * a.Tk;
  const uint8_t* may = a.allowed ? a.allowed + (int64_t)t * a.Tk : nullptr;
  const auto key_at = [&](int i) -> uint64_t { return (i < blocks && (!may || may[i])) ? order_key(score[i]) : 0ull; };
  if (threadIdx.x == 0) s_have = 0;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i < blocks; i += NT) mine += key_at(i) != 0;
  atomicAdd(&s_have, mine);
  __syncthreads();
  const int have = s_have;
  uint64_t key = 0;
  int equal = 0;  // of the blocks with exactly this key, the lowest `equal` are taken
  if (have > a.top) {
    equal = a.top;
    for (int shift = 56; shift >= 0; shift -= 8) {
      hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < blocks; i += NT) {
        const uint64_t k = key_at(i);
        if (k && (shift == 56 || (k >> (shift + 8)) == key)) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      // keys in this digit or above it: the digit where that passes `equal`
      int from = hist[threadIdx.x];
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_down(from, off, 64);
        if (lane + off < 64) from += v;
      }
      if (lane == 0) wave_n[0][w] = from;
      __syncthreads();
      for (int j = w + 1; j < NT / 64; ++j) from += wave_n[0][j];
      const int over = from - hist[threadIdx.x];
      if (from >= equal && over < equal) {
        s_digit = threadIdx.x;
        s_need = equal - over;
      }
      __syncthreads();
      key = (key << 8) | (uint64_t)s_digit;
      equal = s_need;
      __syncthreads();
    }
  }
  int above0 = 0, tie0 = 0;  // before this chunk
  for (int base = 0; base < blocks; base += NT) {
    const uint64_t k = key_at(base + (int)threadIdx.x);
    const bool up = have > a.top ? k > key : k != 0, tie = have > a.top && k == key;
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
  for (int i = min(have, a.top) + threadIdx.x; i < a.top; i += NT) out[i] = -1;
}

// Every wave of the choice that takes its scores itself reads all pooled rows of its head; the matrix instructions' tiles read
// them a 32nd as often and cost a launch. 64 channels, a whole call with and without: 2 x 2048 tokens 11 and 17 us, 4 x 16000
// 23 and 27, 8 x 16000 (64 M products) 34 and 33, 16 x 16000 57 and 49; 128 channels: 4 x 16000 36 and 38, 8 x 16000 58 and
// 49; 504 blocks, eight to a lane, 53 and 24.
inline bool scored_by_choice(int64_t rows, int Tk, int pitch) { return Tk <= 64 * 4 && rows * Tk * pitch <= 1 << 26; }
inline int64_t tiles_of(int64_t L, int block) { return (L + block - 1) / block; }
inline bool block_ok(int block) { return block == 32 || block == 64 || block == 128; }

template <typename T>
void pool(const PoolArgs& a, dim3 grid, hipStream_t st) {
  if (a.D % Vec<T>::N == 0) k_pool<T, true><<<grid, NT, 0, st>>>(a);
  else k_pool<T, false><<<grid, NT, 0, st>>>(a);
}

}  // namespace

extern "C" {

size_t dtk_select_blocks_workspace_size(int B, int64_t Lq, int64_t Lk, int Hkv, int D, int block) {
  if (B <= 0 || Lq <= 0 || Lk <= 0 || Hkv <= 0 || D <= 0 || D > 256 || !block_ok(block) || Lq >= (1LL << 31) || Lk >= (1LL << 31)) return 0;
  const size_t tq = tiles_of(Lq, block), tk = tiles_of(Lk, block);
  return (size_t)B * Hkv * ((padded(tq) + padded(tk)) * pitch_of(D) + tq * tk) * sizeof(double);
}

int dtk_select_blocks(int B, int64_t Lq, int64_t Lk, int Hq, int Hkv, int D, int block, int top, int dtype,
                      const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                      const int32_t* q_lengths, const int32_t* kv_lengths, const uint8_t* allowed, int32_t* index,
                      void* workspace, void* stream) {
  DSPLAT_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D > 0 && D <= 256 && top > 0,
                 "dtk_select_blocks: bad sizes");
  DSPLAT_REQUIRE(block_ok(block), "dtk_select_blocks: block must be 32, 64 or 128");
  DSPLAT_REQUIRE(type_ok(dtype), "dtk_select_blocks: bad type");
  DSPLAT_REQUIRE(Lq < (1LL << 31) && Lk < (1LL << 31) && (int64_t)B * Hkv < 65536 && Hq < 65536, "dtk_select_blocks: too large");
  if (B == 0 || Lq == 0) return 0;
  const int Tq = (int)tiles_of(Lq, block), Tk = (int)tiles_of(Lk, block);
  DSPLAT_REQUIRE(Tq <= 32 * 65535 && Hkv < 65536 && B < 65536, "dtk_select_blocks: too large");
  DSPLAT_REQUIRE(index && (Lk == 0 || (q && k && q_strides && k_strides && workspace)), "dtk_select_blocks: null pointer");
  hipStream_t st = (hipStream_t)stream;
  const int pitch = pitch_of(D);
  const int64_t rows = (int64_t)B * Hkv * Tq;
  DSPLAT_REQUIRE(rows < (1LL << 31), "dtk_select_blocks: too large");
  const bool fused = scored_by_choice(rows, Tk, pitch);
  double* qm = (double*)workspace;
  double* km = qm + (size_t)B * Hkv * padded(Tq) * pitch;
  double* score = km + (size_t)B * Hkv * padded(Tk) * pitch;
  if (Lk > 0) {
    const PoolArgs a = {{{q, q_strides[0], q_strides[1], q_strides[2], q_lengths}, {k, k_strides[0], k_strides[1], k_strides[2], kv_lengths}},
                        {Lq, Lk}, {Hq / Hkv, 1}, {Tq, Tk}, D, pitch, block, {qm, km}};
    const dim3 grid((Tq + Tk + NT / 64 - 1) / (NT / 64), Hkv, B);
    if (dtype == DTK_F32) pool<float>(a, grid, st);
    else if (dtype == DTK_BF16) pool<bf16>(a, grid, st);
    else pool<f16>(a, grid, st);
    if (int e = dsplat::check_launch("k_pool")) return e;
    if (!fused) {
      k_scores<<<dim3((Tk + 255) / 256, (Tq + 31) / 32, B * Hkv), NT, 0, st>>>(Tq, Tk, pitch, qm, km, score);
      if (int e = dsplat::check_launch("k_scores")) return e;
    }
  }
  const ChooseArgs a = {Tq, Tk, Hkv, block, top, Lq, Lk, rows, q_lengths, kv_lengths, allowed, score, qm, km, pitch, index};
  const unsigned waves = (unsigned)((a.rows + NT / 64 - 1) / (NT / 64));
  if (fused && Tk <= 64 * 2) k_choose<2, true><<<waves, NT, 0, st>>>(a);
  else if (fused) k_choose<4, true><<<waves, NT, 0, st>>>(a);
  else if (Tk <= 64 * 8) k_choose<8, false><<<waves, NT, 0, st>>>(a);
  else if (Tk <= 64 * 16) k_choose<16, false><<<waves, NT, 0, st>>>(a);
  else if (Tk <= 64 * 24) k_choose<24, false><<<waves, NT, 0, st>>>(a);
  else if (Tk <= 64 * 32) k_choose<32, false><<<waves, NT, 0, st>>>(a);
  else k_choose_long<<<(unsigned)a.rows, NT, 0, st>>>(a);
  return dsplat::check_launch("k_choose");
}

}  // extern "C"
