// dtk_attention.h — attention of query tiles over their chosen key blocks, forward, backward
// and the form for few queries, for gfx950.
//
//   tile t = queries t block .. t block + block - 1; its keys are those of the blocks index[t]
//   x = scale q k^T, p = exp(x - lse), o = p v;  backward: dv = p^T do, dp = do v^T,
//   ds = p (dp - sum_d do o), dq = scale ds k, dk = scale ds^T q
//
// All products are 32 x 32 matrix instructions, taken transposed (keys as rows, queries as
// columns) in the forward and in dq: a lane then holds one query's scores, so the running
// maximum and sum need one exchange between the two halves of the wave, and the probabilities
// are already laid out as the second product's right operand: an instruction's k index may be
// permuted as long as both operands agree, so the accumulator's rows (8 (r / 4) + 4 half + r % 4)
// serve as they are and nothing is shuffled.
//
// Probabilities, and ds for dk, are rounded to the inputs' type for the second products (the matrix instructions' operands),
// as the inputs themselves were: a rounding of each term's own, so o, dv and dk of random rows are 0.0023 - 0.0024 of their
// norm from 64 bits in bf16, where their own rounding alone makes 0.0017. What dq is made of is taken in two pieces: ds, and
// the probabilities of a forward that trains (k_attend_dq says why); its o and dq are 0.0017 off.
// All sums, the maximum, lse and delta are held in 32 bits. f32 operands stay f32.
//
// Measured (products taken, rate; a large bf16 product reaches 1060 TFLOP/s, f32 153):
//   4 scenes of 32256 bf16 tokens (lengths from half of that on), 4 heads of 64 channels on 2, 16 blocks of 64:
//     forward 125 us 570 TFLOP/s; training forward 171 us 630 (three products), dq 218 us 660 (four), dk/dv 235 us 610
//   16 scenes of 2048 f32 tokens, one head of 128 channels, 8 blocks of 64: 89 us 93, 144 us 86, 209 us 80
//   12 views of 92160 bf16 tokens, 2 heads of 64, 16 blocks of 64, forward: 104 us 465
// What bounds them: the forward and dq at 64 channels the vector unit (some 110 of its instructions per 32 x 32 scores, half of
// its cycles, for 8 matrix instructions, a quarter of theirs; with 128 channels the forward comes to 730 TFLOP/s);
// dk/dv the rows of far tiles from behind the L2 (half of its reads miss; 4.6 TB/s) at three waves per SIMD; the
// 12 views' forward likewise (6 TB/s: one head's 64 queries share a tile); f32 the matrix instructions and the
// start of each workgroup, one or two of which fit a CU. Workgroups in stretches per XCD did not pay: the
// lists of neighbouring tiles have little in common, and ragged batches lose what even ones gain.

#pragma once
#include "dtk_common.h"

namespace dtk {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

// An operand fragment is 8 elements per lane: row (column) lane % 32, k = 8 (lane / 32) + j, or
// any other k both operands share. f32 runs as eight k = 2 instructions over the same registers.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  using Frag = bf16x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<f16> {
  using Frag = f16x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  using Frag = f32x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

struct Strided {
  const void* p;
  int64_t b, l, h;
};
struct Args {
  int64_t Lq, Lk;
  int Hq, Hkv, G, D, block, top, Tq, Tk;
  int lg;                    // block = 32 << lg
  uint32_t group_magic;      // ceil(2^32 / G)
  int Lt, rowtiles, splits;  // rows of a tile, workgroups per tile, parts of the key list
  float scale, scale2;       // scale2: |scale| log2 e, at least the smallest normal number (masked scores are
                             // -inf, and a scale of 0 must not make them no number)
  Strided q, k, v, o, g;  // g: the output's gradient
  const int32_t *index, *q_lengths, *kv_lengths;
  void *out, *dq, *dk, *dv;  // contiguous
  float *lse;                // [B, Hq, Lq], base 2; -inf for rows without a key
  void *rest;                // what the rounding of o left (kRest times it), for delta; 16-bit types that train, else NULL
  float *part, *part_m, *part_l;
  float* delta;
  uint32_t *bits, *chosen;
  int4 *plan, *split;  // NULL where every list is short and every workgroup of dk/dv fits the chip at once
  int* planned;        // how many of each
};

__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int64_t L) {  // fewer than 2^31 (the host checks)
  return lengths ? min(max(lengths[b], 0), (int)L) : (int)L;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// Row r of rows that start at p: token numbers and their strides fit 32 bits, their product is one unsigned 64-bit one.
template <typename T>
__device__ __forceinline__ const T* row_at(const T* p, int r, int64_t stride) {
  return p + (uint64_t)(uint32_t)uniform(r) * (uint32_t)uniform((int)stride);
}

// 8 channels of a row from d0 on, zeros behind D and for rows that do not count (what stands
// there may be no number).
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag row_frag(const T* row, int d0, int D, bool valid) {
  typename Mma<T>::Frag f = {};
  if (valid && d0 < D) __builtin_memcpy(&f, row + d0, sizeof(f));
  return f;
}
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag acc_frag(const f32x16& p, int s) {
  typename Mma<T>::Frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)p[8 * s + j];
  return f;
}

// What acc_frag left of it.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag rest_frag(const f32x16& p, const typename Mma<T>::Frag& of, int s) {
  typename Mma<T>::Frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)(p[8 * s + j] - (float)of[j]);
  return f;
}

// A tile of rows in LDS, R rows of DP channels. The pitch keeps both ways of reading it nearly
// free of bank conflicts: 16 rows' 16-byte pieces at one channel (the row fragments) fall on 16
// different groups of four banks, and the transposed read's 8 rows x 64 bytes on each bank three
// times at most (two is the least).
template <typename T, int DP>
struct Tile {
  static constexpr int kPitch = DP * (int)sizeof(T) + (sizeof(T) == 2 && DP == 128 ? 48 : 16);  // bytes
  static constexpr int kPieces = DP * (int)sizeof(T) / 16;                                      // per row
  static constexpr int kUnit = 32 * kPitch;                                                     // bytes of 32 rows
  using Frag = typename Mma<T>::Frag;

  // channels 16 s + 8 half .. + 7 of row lane % 32
  static __device__ __forceinline__ Frag row(const char* t, int s, int col, int half) {
    Frag f;
    __builtin_memcpy(&f, __builtin_assume_aligned(t + col * kPitch + (16 * s + 8 * half) * sizeof(T), 16), sizeof(f));
    return f;
  }
  // channel 32 d + lane % 32 of the 8 rows 16 s + {4 half .. + 3, 8 + 4 half .. + 3}: the rows an accumulator
  // holds. 16 bits: the transposing LDS read hands lane i of 16 the i-th column of the 4 rows of 16
  // that the 16 lanes' 8-byte pieces make up.
  static __device__ __forceinline__ Frag col(const char* t, int s, int d, int lane) {
    Frag f;
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds;
      const int i = lane & 15;
      const char* at = t + (16 * s + 4 * half + (i >> 2)) * kPitch + (32 * d + (lane & 16) + 4 * (i & 3)) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(at + 8 * kPitch));
      __builtin_memcpy(&f, &lo, 8);
      __builtin_memcpy((char*)&f + 8, &hi, 8);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = *(const T*)(t + (16 * s + 4 * half + (j & 3) + 8 * (j >> 2)) * kPitch + (32 * d + (lane & 31)) * 4);
    }
    return f;
  }
};

// sum += rows^T x for the 32 rows of a unit and an accumulator's 32 x 32 numbers x, which 16-bit types take in two pieces (what rounding
// the first left is the second).
template <typename T, int DP>
__device__ __forceinline__ void add_pieces(f32x16 (&sum)[DP / 32], const f32x16& x, const char* rows, int lane) {
  using Frag = typename Mma<T>::Frag;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const Frag hi = acc_frag<T>(x, s), lo = sizeof(T) == 2 ? rest_frag<T>(x, hi, s) : Frag{};
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      const Frag r = Tile<T, DP>::col(rows, s, d, lane);
      sum[d] = Mma<T>::mma(r, hi, sum[d]);
      if constexpr (sizeof(T) == 2) sum[d] = Mma<T>::mma(r, lo, sum[d]);
    }
  }
}

// The workgroup's share of U units (32 rows each) on the way from memory to LDS: loaded into
// registers while the tile before is worked on, then stored. Rows that do not count and channels
// behind D become zeros. A wave's pieces are all of one unit, so where that starts is scalar work and a
// load adds one 32-bit offset to it (31 rows' strides fit: the host checks).
template <typename T, int DP, int U>
struct Stage {
  using L = Tile<T, DP>;
  static constexpr int kPer = (U * 32 * L::kPieces + kThreads - 1) / kThreads;
  static constexpr int kWaves = 32 * L::kPieces / 64;  // waves of pieces per unit
  Vec<T> v[kPer];
  // from[j]: where the j-th unit's first row starts, n[j]: its rows that count
  __device__ __forceinline__ void load(const T* const (&from)[U], const int (&n)[U], int64_t stride, int D) {
    const int wave = uniform(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = threadIdx.x + i * kThreads, r = id / L::kPieces % 32, d = id % L::kPieces * Vec<T>::N;
      const uint32_t off = (uint32_t)r * (uint32_t)stride + (uint32_t)d;
      int have = 0;
      const T* p = nullptr;
      if constexpr (kWaves % (kThreads / 64) == 0) {
        have = n[i / (kWaves / (kThreads / 64))];
        p = from[i / (kWaves / (kThreads / 64))];
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j)
          if ((wave + i * (kThreads / 64)) / kWaves == j) {
            have = n[j];
            p = from[j];
          }
      }
      v[i] = Vec<T>{};
      if (r < have && d < D) v[i] = load_vec(p + off);
    }
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) v[i].v[e] = -v[i].v[e];
  }
  __device__ __forceinline__ void store(char* t) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = threadIdx.x + i * kThreads, r = id / L::kPieces, c = id % L::kPieces;
      if ((i + 1) * kThreads <= U * 32 * L::kPieces || r < U * 32)
        __builtin_memcpy(__builtin_assume_aligned(t + r * L::kPitch + c * 16, 16), &v[i], 16);
    }
  }
};
// Two buffers (one barrier per step) while they leave room for two workgroups per CU; f32 tiles are
// twice as large and its products eight times as long: one.
template <typename T, int DP, int U>
constexpr int kBuffers = sizeof(T) == 2 && 4 * U * Tile<T, DP>::kUnit <= 80 * 1024 ? 2 : 1;
template <typename T, int DP, int U>
constexpr int kTileBytes = 2 * kBuffers<T, DP, U> * U * Tile<T, DP>::kUnit;

__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// Units of keys that a wave of dq works off per step: where all four waves stand side by side over the rows, two, so that a
// barrier and a step's addresses serve 64 keys (4 scenes of 32256 bf16 tokens, 16 blocks of 64: 183 us with one, 166 with
// two; the forward has no registers for it at four waves per SIMD, 128 us either way).
template <typename T, int RW>
constexpr int kEach = sizeof(T) == 2 && RW == 4 ? 2 : 1;

// The tile's list without places that are no block or stand in it already, in LDS, in order. One wave, 64 places at
// a time: each is compared with those before it by broadcasts within the wave (from memory, one after the other, it took
// longer than the attention of few queries itself), and with the list so far.
// (first: this lane's place of the first 64, loaded while the lengths are on their way.)
__device__ __forceinline__ int block_list(const int32_t* idx, int first, int top, int blocks, int32_t* list, int* count) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int n = 0;
    for (int base = 0; base < top; base += 64) {
      const int v = base + lane >= top ? -1 : base == 0 ? first : idx[base + lane];
      bool ok = v >= 0 && v < blocks;
      const int here = min(64, top - base);
      for (int j = 0; j < here; ++j) ok = ok && !(j < lane && __builtin_amdgcn_readlane(v, j) == v);
      for (int j = 0; j < n; ++j) ok = ok && list[j] != v;
      const uint64_t m = __ballot(ok);
      if (ok) list[n + __popcll(m & dsplat::lanemask_lt(lane))] = v;
      n += __popcll(m);
    }
    if (lane == 0) *count = n;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*count);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  T v[4] = {(T)a, (T)b, (T)c, (T)d};
  __builtin_memcpy(p, v, sizeof(v));
}

// What the rounding of a, b, c, d left, itself rounded; f16's is taken times 2^11, out of its smallest numbers.
template <typename T>
constexpr float kRest = __is_same(T, f16) ? 2048.f : 1.f;
template <typename T>
__device__ __forceinline__ void store_rest4(T* p, float a, float b, float c, float d) {
  store4<T>(p, (a - (float)(T)a) * kRest<T>, (b - (float)(T)b) * kRest<T>, (c - (float)(T)c) * kRest<T>, (d - (float)(T)d) * kRest<T>);
}

// Where a workgroup works: tile, row group, key head, scene, part of the list.
struct Where {
  int t, rt, hk, b, split;
};
__device__ __forceinline__ Where where(const Args& a) {
  Where w;
  w.t = blockIdx.x / a.rowtiles;
  w.rt = blockIdx.x % a.rowtiles;
  w.hk = blockIdx.y;
  w.b = blockIdx.z / a.splits;
  w.split = blockIdx.z % a.splits;
  return w;
}

// A tile's units of 32 keys: unit u is part u % (block / 32) of the list's block u / (block / 32).
template <int U>
struct Span {
  int first[U];
  int n[U];  // keys that count
};
struct Keys {
  const int32_t* list;
  int lg, units, nk;
  template <int U>
  __device__ __forceinline__ Span<U> span(int u) const {
    int b[U];
    Span<U> s;
#pragma unroll
    for (int j = 0; j < U; ++j) b[j] = list[min(u + j, units - 1) >> lg];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      s.first[j] = ((uniform(b[j]) << lg) + ((u + j) & ((1 << lg) - 1))) * 32;
      s.n[j] = u + j < units ? max(0, min(32, nk - s.first[j])) : 0;
    }
    return s;
  }
};
// The unit of this wave (its number among U is uniform).
template <int U>
__device__ __forceinline__ int pick(const int (&n)[U], int w) {
  int v = n[0];
#pragma unroll
  for (int j = 1; j < U; ++j) v = w == j ? n[j] : v;
  return v;
}

// What a row's waves have in common at the end: wave kw = 0 takes in the others' sums through LDS.
template <int RW, int DP>
struct Join {
  float o[RW * 32 * (DP + 1)];
  float m[RW * 32], l[RW * 32];
};

// Forward. RW waves stand side by side over 32 rows each, 4 / RW take turns at the list's units
// of 32 keys and are joined at the end. The rows of a tile are its queries of all heads that
// share the key head (few queries: they fill the instruction's columns together). Few tiles: the list is split over
// workgroups (splits_of) and k_attend_join adds them up. PIECES: 16-bit p in two pieces, and o's rest, for a backward (an
// instance of its own: as a branch it spills at four waves per SIMD, 103 -> 182 us for the 12 views).
template <typename T, int DP, int RW, bool PIECES>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 2 ? (DP > 64 || RW == 1 ? 2 : 4) : 2)) void k_attend_fwd(Args a) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using Frag = typename M::Frag;
  constexpr int KW = 4 / RW, NS = DP / 16, ND = DP / 32, NB = kBuffers<T, DP, KW>;
  extern __shared__ __align__(16) char lds[];
  __shared__ int count;
  int32_t* list = (int32_t*)(lds + kTileBytes<T, DP, KW>);
  const Where at = where(a);
  const int32_t* idx = a.index + (((int64_t)at.b * a.Hkv + at.hk) * a.Tq + at.t) * a.top;
  const int first_places = idx[min((int)threadIdx.x & 63, a.top - 1)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int rw = uniform(wave) % RW, kw = uniform(wave) / RW;
  const int nq = length_of(a.q_lengths, at.b, a.Lq), nk = length_of(a.kv_lengths, at.b, a.Lk);
  const int row = (at.rt * RW + rw) * 32 + col;
  const int g = row / a.Lt;
  const int64_t i = (int64_t)at.t * a.block + row % a.Lt;
  const bool exists = g < a.G && i < a.Lq, valid = exists && i < nq;
  const int h = at.hk * a.G + (g < a.G ? g : 0);
  const int blocks = (nk >> (5 + a.lg)) + ((nk & (a.block - 1)) != 0);
  int n = 0;
  if (at.t * a.block < nq) n = block_list(idx, first_places, a.top, blocks, list, &count);

  const T* qp = (const T*)a.q.p + at.b * a.q.b + (valid ? i : 0) * a.q.l + h * a.q.h;
  Frag qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = row_frag<T>(qp, 16 * s + 8 * half, a.D, valid);
    if (a.scale < 0.f) qf[s] = -qf[s];
  }
  const T* kp = (const T*)a.k.p + at.b * a.k.b + at.hk * a.k.h;
  const T* vp = (const T*)a.v.p + at.b * a.v.b + at.hk * a.v.h;

  f32x16 o[ND] = {};
  // The exponents are taken relative to base2 (in powers of two), which is set to the largest score so far only when a sum of
  // 16 has passed 2^12, or at first, when it is -inf and every sum passes everything: p stays in every type's range, the
  // fast path needs no maximum, and o is rarely rescaled. (l <= 2^12 x keys, o likewise: far inside 32 bits.)
  float base2 = -INFINITY, l = 0.f;
  const int units = n << a.lg;
  const int per = (units + a.splits - 1) / a.splits;
  const int u0 = min(units, at.split * per), u1 = min(units, u0 + per);
  const Keys where_ = {list, a.lg, u1, nk};
  // A step's keys and values come together, while the step before is worked on; or, for f32 rows of more than 64
  // channels, in turn through the same registers, the values during the first product and the next keys during
  // the second (which take 4096 cycles each at 128 channels), so that two waves per SIMD fit: 16 scenes of
  // 2048 tokens of 128 channels, 8 blocks of 64 each, 91 us instead of 106. (At 64 channels three
  // waves fit as it is.)
  constexpr bool TURNS = sizeof(T) == 4 && DP > 64;
  Stage<T, DP, KW> sk, sv;
  const auto load = [&](Stage<T, DP, KW>& to, const Span<KW>& s, const T* p, int64_t stride) {
    const T* rows[KW];
#pragma unroll
    for (int j = 0; j < KW; ++j) rows[j] = row_at(p, s.first[j], stride);
    to.load(rows, s.n, stride, a.D);
  };
  Span<KW> next = {};
  const auto fetch = [&](int u) {
    next = where_.span<KW>(u);
    load(sk, next, kp, a.k.l);
    if (!TURNS) load(sv, next, vp, a.v.l);
  };
  if (u0 < u1) fetch(u0);
  for (int u = u0, step = 0; u < u1; u += KW, ++step) {
    char* tk = lds + (step % NB) * 2 * KW * L::kUnit;
    char* tv = tk + KW * L::kUnit;
    if (NB == 1 && !TURNS) __syncthreads();
    sk.store(tk);
    if (!TURNS) sv.store(tv);
    __syncthreads();
    const int left = pick(next.n, kw);
    if (TURNS) load(sk, next, vp, a.v.l);
    else if (u + KW < u1) fetch(u + KW);
    tk += kw * L::kUnit;
    if (!TURNS && left == 0) continue;
    f32x16 x = {};
    if (!TURNS || left > 0) {
#pragma unroll
      for (int s = 0; s < NS; ++s) x = M::mma(L::row(tk, s, col, half), qf[s], x);
    }
    if (TURNS) {
      sk.store(tv);  // every wave is past the products of the values before
      if (u + KW < u1) fetch(u + KW);
      __syncthreads();  // (and of these keys)
    }
    tv += kw * L::kUnit;
    if (TURNS && left == 0) continue;
    if (left < 32) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = acc_row(r, half) < left ? x[r] : -INFINITY;
    }
    f32x16 p;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.scale2, -base2));
      sum += p[r];
    }
    if (__any(!(sum <= 4096.f))) {
      float mx = x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float top = fmaxf(base2, mx * a.scale2);  // -inf as long as every score was
      const float to = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(base2 - to);
      base2 = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
      sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.scale2, -to));
        sum += p[r];
      }
    }
    l += sum;
    if constexpr (PIECES) {
      add_pieces<T, DP>(o, p, tv, lane);
    } else {
      const Frag p0 = acc_frag<T>(p, 0), p1 = acc_frag<T>(p, 1);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        o[d] = M::mma(L::col(tv, 0, d, lane), p0, o[d]);
        o[d] = M::mma(L::col(tv, 1, d, lane), p1, o[d]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if constexpr (KW > 1) {
    static_assert(sizeof(Join<RW, DP>) <= kTileBytes<T, DP, KW>, "joined in the tiles' place");
    Join<RW, DP>& join = *(Join<RW, DP>*)lds;
    float* jo = join.o + (rw * 32 + col) * (DP + 1);
    for (int k = 1; k < KW; ++k) {
      __syncthreads();
      if (kw == k) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) jo[32 * d + acc_row(r, half)] = o[d][r];
        if (half == 0) {
          join.m[rw * 32 + col] = base2;
          join.l[rw * 32 + col] = l;
        }
      }
      __syncthreads();
      if (kw == 0) {
        const float mo = join.m[rw * 32 + col], lo = join.l[rw * 32 + col];
        const float top = fmaxf(base2, mo), to = top == -INFINITY ? 0.f : top;
        const float fa = __builtin_amdgcn_exp2f(base2 - to), fb = __builtin_amdgcn_exp2f(mo - to);
        base2 = top;
        l = l * fa + lo * fb;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * fa + jo[32 * d + acc_row(r, half)] * fb;
      }
    }
  }
  if (kw != 0 || !exists) return;
  if (a.splits > 1) {
    const int64_t r = ((int64_t)at.b * a.Hq + h) * a.Lq + i, rows = (int64_t)(gridDim.z / a.splits) * a.Hq * a.Lq;
    float* po = a.part + (at.split * rows + r) * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (32 * d + 8 * c + 4 * half < a.D)
          store4<float>(po + 32 * d + 8 * c + 4 * half, o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]);
    if (half == 0) {
      a.part_m[at.split * rows + r] = base2;
      a.part_l[at.split * rows + r] = l;
    }
    return;
  }
  // a row behind the length is written as 0: its zeros beside an infinite key or value are no number
  const float inv = l > 0.f ? 1.f / l : (l != l ? l : 0.f);
  const int64_t to = (((int64_t)at.b * a.Lq + i) * a.Hq + h) * a.D;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int e = 32 * d + 8 * c + 4 * half;
      if (e >= a.D) continue;
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = valid ? o[d][4 * c + k] * inv : 0.f;
      store4<T>((T*)a.out + to + e, v[0], v[1], v[2], v[3]);
      if (PIECES) store_rest4<T>((T*)a.rest + to + e, v[0], v[1], v[2], v[3]);
    }
  if (half == 0 && a.lse) a.lse[((int64_t)at.b * a.Hq + h) * a.Lq + i] = valid ? base2 + log2f(l) : -INFINITY;
}

// ds is rounded to the inputs' type for its products. f16 has few exponents (its normal numbers end at 2^-14), so ds is taken
// there times a power of two of its own for each column, which is a query in dq and a key in dk: it starts at 2^60 and
// falls where the column's ds would pass 2^15, to put the largest at 2^12 to 2^13; what is summed so far is
// scaled with it, in 32 bits, and all is undone at the end. So a column's terms keep f16's 11 bits down to 2^-26 of its largest,
// whatever other rows, heads and scenes hold. (|ds| <= 2 D 65504^2 < 2^40: in 32 bits 2^60 times that is still a number.) p <= 1 is
// taken times 2^12 for dv, for unlikely keys: by the exponent's base, at no cost.
// 4 scenes of 32256 f16 tokens, 4 heads on 2 of 64, 16 blocks of 64: dk/dv 470 us, where one power of two of the whole call, at the
// largest |do|, took 444 and lost the digits of a scene of 2^-13 of another's gradients.
template <typename T>
constexpr bool kFewExponents = __is_same(T, f16);
constexpr int kFirstPower = 60, kLikely = 12;
// ds: 16 rows of this lane's column, the others in the lane 32 further. ldexp by 0 leaves what is no number as it is.
template <int ND>
__device__ __forceinline__ bool keep_in_range(f32x16& ds, f32x16 (&sum)[ND], int& power) {
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(ds[r]));
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
  most = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
  const bool far = most >= 32768.f && most < INFINITY;
  if (!__any(far)) return false;
  const int down = far ? 12 - ((int)(__float_as_uint(most) >> 23) - 127) : 0;
  power += down;
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_ldexpf(ds[r], down);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[d][r] = __builtin_amdgcn_ldexpf(sum[d][r], down);
  return true;
}
template <int ND>
__device__ __forceinline__ void shift(f32x16 (&sum)[ND], int power) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[d][r] = __builtin_amdgcn_ldexpf(sum[d][r], power);
}

// dq: the forward's shape; p is taken from the saved lse. delta = sum_d do o of each row on the
// way, kept for dk.
//
// A row's ds add up to 0, so what all keys have in common falls out of dq = sum ds k, and what all values have in
// common out of ds = p (dp - delta). A rounding of ds leaves a share of the keys' common part in it, one of delta
// a share of both: with 16-bit ds, and delta of an o made of 16-bit p and rounded itself, bf16 keys and values with a mean of 1 (3) times
// their spread, 1024 of them, put dq 0.037 (0.34) of its norm off. So ds is two pieces, p of the forward that trains
// likewise, and that forward keeps what the rounding of o left: 0.0017 (0.0017), which the rounding of dq alone makes. (4 scenes of
// 32256 bf16 tokens: dq 171 -> 218 us, the forward 125 -> 171. Subtracting (sum ds) times a mean of some keys at the end
// instead of the forward's second piece takes as long, and lets keys that a row does not see enter its dq.)
template <typename T, int DP, int RW>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 2 ? (DP > 64 || RW == 1 ? 2 : 3) : DP <= 64 ? 2 : 1)) void k_attend_dq(Args a) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using Frag = typename M::Frag;
  constexpr int KW = 4 / RW, NS = DP / 16, ND = DP / 32, EACH = kEach<T, RW>, U = KW * EACH, NB = kBuffers<T, DP, U>;
  extern __shared__ __align__(16) char lds[];
  __shared__ int count;
  int32_t* list = (int32_t*)(lds + kTileBytes<T, DP, U>);
  const Where at = where(a);
  const int32_t* idx = a.index + (((int64_t)at.b * a.Hkv + at.hk) * a.Tq + at.t) * a.top;
  const int first_places = idx[min((int)threadIdx.x & 63, a.top - 1)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int rw = uniform(wave) % RW, kw = uniform(wave) / RW;
  const int nq = length_of(a.q_lengths, at.b, a.Lq), nk = length_of(a.kv_lengths, at.b, a.Lk);
  const int row = (at.rt * RW + rw) * 32 + col;
  const int g = row / a.Lt;
  const int64_t i = (int64_t)at.t * a.block + row % a.Lt;
  const bool exists = g < a.G && i < a.Lq, valid = exists && i < nq;
  const int h = at.hk * a.G + (g < a.G ? g : 0);
  const int blocks = (nk >> (5 + a.lg)) + ((nk & (a.block - 1)) != 0);
  int n = 0;
  if (at.t * a.block < nq) n = block_list(idx, first_places, a.top, blocks, list, &count);
  if (at.rt == 0)  // for dk, dv: which tiles chose a block (bits [B, Hkv, Tk, ceil(Tq / 32)]), and how many did
    for (int j = threadIdx.x; j < n; j += kThreads) {
      const int64_t item = ((int64_t)at.b * a.Hkv + at.hk) * a.Tk + list[j];
      atomicOr(a.bits + item * ((a.Tq + 31) / 32) + at.t / 32, 1u << (at.t % 32));
      if (a.chosen) atomicAdd(a.chosen + item, 1u);
    }

  const int64_t ir = valid ? i : 0;
  const T* qp = (const T*)a.q.p + at.b * a.q.b + ir * a.q.l + h * a.q.h;
  const T* gp = (const T*)a.g.p + at.b * a.g.b + ir * a.g.l + h * a.g.h;
  const int64_t oat = at.b * a.o.b + ir * a.o.l + h * a.o.h;
  Frag qf[NS], gf[NS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = row_frag<T>(qp, 16 * s + 8 * half, a.D, valid);
    if (a.scale < 0.f) qf[s] = -qf[s];
    gf[s] = row_frag<T>(gp, 16 * s + 8 * half, a.D, valid);
    const Frag of = row_frag<T>((const T*)a.o.p + oat, 16 * s + 8 * half, a.D, valid);
    const Frag rest = sizeof(T) == 2 ? row_frag<T>((const T*)a.rest + oat, 16 * s + 8 * half, a.D, valid) : Frag{};
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += (float)gf[s][j] * ((float)of[j] + (float)rest[j] * (1.f / kRest<T>));
  }
  delta += __shfl_xor(delta, 32, 64);
  const int64_t stat = ((int64_t)at.b * a.Hq + h) * a.Lq + ir;
  // rows that see nothing: relative to +inf every p is 0
  const float saved = valid ? a.lse[stat] : -INFINITY, lse = saved == -INFINITY ? INFINITY : saved;
  if (kw == 0 && half == 0 && valid) a.delta[stat] = delta;
  const T* kp = (const T*)a.k.p + at.b * a.k.b + at.hk * a.k.h;
  const T* vp = (const T*)a.v.p + at.b * a.v.b + at.hk * a.v.h;

  f32x16 dq[ND] = {};
  int power = kFirstPower;  // f16: of this query's ds
  float times = __builtin_amdgcn_ldexpf(1.f, power);
  const int units = n << a.lg;
  const Keys where_ = {list, a.lg, units, nk};
  Stage<T, DP, U> sk, sv;
  Span<U> next = {};
  const auto fetch = [&](int u) {
    next = where_.span<U>(u);
    const T *pk[U], *pv[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      pk[j] = row_at(kp, next.first[j], a.k.l);
      pv[j] = row_at(vp, next.first[j], a.v.l);
    }
    sk.load(pk, next.n, a.k.l, a.D);
    sv.load(pv, next.n, a.v.l, a.D);
  };
  if (units) fetch(0);
  for (int u = 0, step = 0; u < units; u += U, ++step) {
    char* tk = lds + (step % NB) * 2 * U * L::kUnit;
    char* tv = tk + U * L::kUnit;
    if (NB == 1) __syncthreads();
    sk.store(tk);
    sv.store(tv);
    __syncthreads();
    const Span<U> now = next;
    if (u + U < units) fetch(u + U);
#pragma unroll 1
    for (int e = 0; e < EACH; ++e) {
      const char *uk = tk + (e * KW + kw) * L::kUnit, *uv = tv + (e * KW + kw) * L::kUnit;
      const int left = pick(now.n, e * KW + kw);
      if (left == 0) continue;
      f32x16 x = {}, dp = {};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        x = M::mma(L::row(uk, s, col, half), qf[s], x);
        dp = M::mma(L::row(uv, s, col, half), gf[s], dp);
      }
      if (left < 32) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = acc_row(r, half) < left ? x[r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.scale2, -lse));
        x[r] = p * (kFewExponents<T> ? (dp[r] - delta) * times : dp[r] - delta);
      }
      if constexpr (kFewExponents<T>)
        if (keep_in_range(x, dq, power)) times = __builtin_amdgcn_ldexpf(1.f, power);
      add_pieces<T, DP>(dq, x, uk, lane);
    }
  }
  if constexpr (kFewExponents<T>) shift(dq, -power);
  if constexpr (KW > 1) {
    float* jo = (float*)lds + (rw * 32 + col) * (DP + 1);
    for (int k = 1; k < KW; ++k) {
      __syncthreads();
      if (kw == k)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) jo[32 * d + acc_row(r, half)] = dq[d][r];
      __syncthreads();
      if (kw == 0)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dq[d][r] += jo[32 * d + acc_row(r, half)];
    }
  }
  if (kw != 0 || !exists) return;
  T* out = (T*)a.dq + (((int64_t)at.b * a.Lq + i) * a.Hq + h) * a.D;
  const float f = a.scale;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (32 * d + 8 * c + 4 * half < a.D) {
        if (valid)
          store4<T>(out + 32 * d + 8 * c + 4 * half, dq[d][4 * c] * f, dq[d][4 * c + 1] * f, dq[d][4 * c + 2] * f,
                    dq[d][4 * c + 3] * f);
        else
          store4<T>(out + 32 * d + 8 * c + 4 * half, 0.f, 0.f, 0.f, 0.f);
      }
}

// dk, dv of one key block: RW waves hold 32 keys each, 4 / RW take turns at the 32-query units of
// the tiles that chose the block (their bits, some at a time) and are joined at the end. Every sum
// has one order: no atomics on the gradients. A long list is worked off by several workgroups, each taking every
// parts-th step.
constexpr int kTiles = 1024;  // tiles listed at a time
// Where a key block's rows stay while its list is worked off: in LDS, from where they cost a third more of its reads and
// leave the registers to another wave per SIMD, or in registers, where that makes no room (f32: more than 64 channels'
// sums fill a SIMD with one wave; 64 channels of 32 or 128 keys fill the LDS).
template <typename T, int DP, int RW>
constexpr bool kRowsInLds = sizeof(T) == 2 || (DP == 64 && RW == 2);
template <typename T, int DP, int RW>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 2 ? (DP <= 64 ? (RW == 1 ? 2 : 3) : DP == 128 && RW == 1 ? 1 : 2) : DP <= 64 && RW > 1 || DP == 32 ? 2 : 1)) void k_attend_dkv(Args a) {
  using M = Mma<T>;
  using L = Tile<T, DP>;
  using Frag = typename M::Frag;
  constexpr int QW = 4 / RW, NS = DP / 16, ND = DP / 32, NB = 1;
  constexpr int kAhead = 1;  // steps whose rows are on their way
  constexpr bool KEEP = !kRowsInLds<T, DP, RW>;
  extern __shared__ __align__(16) char lds[];
  __shared__ int32_t tiles[kTiles];
  __shared__ int count;
  __shared__ __align__(16) float stats[NB][2][QW * 32];  // lse and delta of the staged rows
  int item = blockIdx.x, part = 0, parts = 1, slot = 0;
  if (a.plan) {
    if ((int)blockIdx.x >= a.planned[0]) return;
    const int4 e = a.plan[blockIdx.x];
    item = e.x;
    part = e.y;
    parts = e.z;
    slot = e.w;
  }
  const int blk = item % a.Tk, hk = item / a.Tk % a.Hkv, b = item / a.Tk / a.Hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int rw = uniform(wave) % RW, qw = uniform(wave) / RW;
  const int nq = length_of(a.q_lengths, b, a.Lq), nk = length_of(a.kv_lengths, b, a.Lk);
  const int64_t key = (int64_t)blk * a.block + 32 * rw + col;
  const bool exists = key < a.Lk, valid = key < nk;
  char* tkv = lds + NB * 2 * QW * L::kUnit;
  Frag kf[KEEP ? NS : 1], vf[KEEP ? NS : 1];
  if constexpr (KEEP) {
    const int64_t kr = valid ? key : 0;
    const T* kp = (const T*)a.k.p + b * a.k.b + kr * a.k.l + hk * a.k.h;
    const T* vp = (const T*)a.v.p + b * a.v.b + kr * a.v.l + hk * a.v.h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      kf[s] = row_frag<T>(kp, 16 * s + 8 * half, a.D, valid);
      if (a.scale < 0.f) kf[s] = -kf[s];
      vf[s] = row_frag<T>(vp, 16 * s + 8 * half, a.D, valid);
    }
  } else {
    Stage<T, DP, RW> sk, sv;
    const T *pk[RW], *pv[RW];
    int have[RW];
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      const int64_t k0 = (int64_t)blk * a.block + 32 * j;
      have[j] = (int)max((int64_t)0, min((int64_t)32, (int64_t)nk - k0));
      pk[j] = (const T*)a.k.p + b * a.k.b + k0 * a.k.l + hk * a.k.h;
      pv[j] = (const T*)a.v.p + b * a.v.b + k0 * a.v.l + hk * a.v.h;
    }
    sk.load(pk, have, a.k.l, a.D);
    sv.load(pv, have, a.v.l, a.D);
    if (a.scale < 0.f) sk.negate();
    sk.store(tkv);
    sv.store(tkv + RW * L::kUnit);
    tkv += rw * L::kUnit;
  }
  f32x16 dk[ND] = {}, dv[ND] = {};
  int power = kFirstPower;  // f16: of this key's ds, p's included
  float times = __builtin_amdgcn_ldexpf(1.f, power - kLikely);
  const int upt = a.G << a.lg, words = (a.Tq + 31) / 32;  // units per tile
  const uint32_t* bits = a.bits + (((int64_t)b * a.Hkv + hk) * a.Tk + blk) * words;
  const bool any = blk * a.block < nk;
  const T* qb = (const T*)a.q.p + b * a.q.b + (int64_t)hk * a.G * a.q.h;
  const T* gb = (const T*)a.g.p + b * a.g.b + (int64_t)hk * a.G * a.g.h;
  const int u0 = part * QW, stride = parts * QW;  // this part's steps
  int step = 0;
  for (int w0 = 0; any && w0 < words; w0 += kTiles / 32) {
    __syncthreads();
    if (threadIdx.x < 64) {  // the first 32 lanes hold a word each
      uint32_t m = lane < 32 && w0 + lane < words ? bits[w0 + lane] : 0u;
      const uint32_t incl = dsplat::wave_incl_scan(__popc(m), lane);
      int at = (int)incl - __popc(m);
      while (m) {
        tiles[at++] = 32 * (w0 + lane) + __ffs(m) - 1;
        m &= m - 1;
      }
      if (lane == 63) count = (int)incl;
    }
    __syncthreads();
    const int units = uniform(count) * upt;
    // Unit u: 32 rows (part u % RW; a block is RW units of keys and a tile RW units of queries) of a head of the group of a
    // listed tile. With two or four units to a tile, a step's units are of one tile and head.
    const auto listed = [&](int p) {  // p-th tile and head -> place in the list; exact: p < 2^20 and G <= 1024
      return a.G == 1 ? p : (int)__umulhi((uint32_t)p, a.group_magic);
    };
    // What is on its way: the rows of the units u .. u + QW - 1 and their statistics.
    struct Ahead {
      Stage<T, DP, QW> q, g;
      float lse, delta;
      int live;
    };
    const int64_t stats0 = ((int64_t)b * a.Hq + hk * a.G) * a.Lq;
    const auto fetch = [&](Ahead& f, int u) {
      const T *pq[QW], *pg[QW];
      int have[QW];
      f.lse = -INFINITY;
      if constexpr (RW == 1) {
        int tile[QW];
#pragma unroll
        for (int j = 0; j < QW; ++j) tile[j] = tiles[listed(min(u + j, units - 1))];
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          const int i0 = uniform(tile[j]) * 32;
          const int64_t g = u + j - listed(u + j) * a.G;
          pq[j] = row_at(qb, i0, a.q.l) + g * a.q.h;
          pg[j] = row_at(gb, i0, a.g.l) + g * a.g.h;
          have[j] = u + j < units ? max(0, min(32, nq - i0)) : 0;
        }
        const int uj = u + threadIdx.x / 32;
        if (threadIdx.x < QW * 32 && uj < units) {
          const int at = listed(uj), i = tiles[at] * 32 + threadIdx.x % 32;
          if (i < nq) {
            const int64_t stat = stats0 + (int64_t)(uj - at * a.G) * a.Lq + i;
            f.lse = a.lse[stat];
            f.delta = a.delta[stat];
          }
        }
      } else {
        const int p = (int)((uint32_t)u / RW), at = listed(p), g = p - at * a.G;
        const int i0 = (uniform(tiles[at]) * RW + (int)((uint32_t)u % RW)) * 32;
        const T *q0 = row_at(qb, i0, a.q.l) + g * a.q.h, *g0 = row_at(gb, i0, a.g.l) + g * a.g.h;
#pragma unroll
        for (int j = 0; j < QW; ++j) {
          pq[j] = q0 + j * 32 * a.q.l;
          pg[j] = g0 + j * 32 * a.g.l;
          have[j] = max(0, min(32, nq - i0 - 32 * j));
        }
        if (threadIdx.x < QW * 32 && i0 + (int)threadIdx.x < nq) {
          const int64_t stat = stats0 + (int64_t)g * a.Lq + i0;
          f.lse = (a.lse + stat)[threadIdx.x];
          f.delta = (a.delta + stat)[threadIdx.x];
        }
      }
      f.q.load(pq, have, a.q.l, a.D);
      f.g.load(pg, have, a.g.l, a.D);
      f.live = pick(have, qw);
    };
    const auto turn = [&](Ahead& f, int u) {
      char* tq = lds + (step % NB) * 2 * QW * L::kUnit;
      char* tg = tq + QW * L::kUnit;
      if (NB == 1) __syncthreads();
      f.q.store(tq);
      f.g.store(tg);
      if (threadIdx.x < QW * 32) {
        // rows that see nothing, or are none: relative to +inf every p is 0
        stats[step % NB][0][threadIdx.x] = f.lse == -INFINITY ? INFINITY : kFewExponents<T> ? f.lse - kLikely : f.lse;
        stats[step % NB][1][threadIdx.x] = f.delta;
      }
      __syncthreads();
      const int live = f.live, buffer = step++ % NB;
      if (u + kAhead * stride < units) fetch(f, u + kAhead * stride);
      if (live == 0) return;
      tq += qw * L::kUnit;
      tg += qw * L::kUnit;
      f32x16 x = {}, dp = {};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        x = M::mma(L::row(tq, s, col, half), KEEP ? kf[KEEP ? s : 0] : L::row(tkv, s, col, half), x);
        dp = M::mma(L::row(tg, s, col, half), KEEP ? vf[KEEP ? s : 0] : L::row(tkv + RW * L::kUnit, s, col, half), dp);
      }
      // (lanes whose key is none hold columns that are not written)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 lse = *(const float4*)&stats[buffer][0][qw * 32 + 8 * c + 4 * half];
        const float4 delta = *(const float4*)&stats[buffer][1][qw * 32 + 8 * c + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * c + e;
          const float ls = e == 0 ? lse.x : e == 1 ? lse.y : e == 2 ? lse.z : lse.w;
          const float de = e == 0 ? delta.x : e == 1 ? delta.y : e == 2 ? delta.z : delta.w;
          x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.scale2, -ls));
          dp[r] = x[r] * (kFewExponents<T> ? (dp[r] - de) * times : dp[r] - de);
        }
      }
      if (live < 32) {  // rows behind the length: zeros, which beside an infinite key or value are no number
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[r] = acc_row(r, half) < live ? x[r] : 0.f;
          dp[r] = acc_row(r, half) < live ? dp[r] : 0.f;
        }
      }
      if constexpr (kFewExponents<T>)
        if (keep_in_range(dp, dk, power)) times = __builtin_amdgcn_ldexpf(1.f, power - kLikely);
      const Frag p0 = acc_frag<T>(x, 0), p1 = acc_frag<T>(x, 1), s0 = acc_frag<T>(dp, 0), s1 = acc_frag<T>(dp, 1);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        dv[d] = M::mma(L::col(tg, 0, d, lane), p0, dv[d]);
        dv[d] = M::mma(L::col(tg, 1, d, lane), p1, dv[d]);
        dk[d] = M::mma(L::col(tq, 0, d, lane), s0, dk[d]);
        dk[d] = M::mma(L::col(tq, 1, d, lane), s1, dk[d]);
      }
    };
    Ahead f[kAhead] = {};
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (u0 + k * stride < units) fetch(f[k], u0 + k * stride);
    for (int u = u0; u < units; u += kAhead * stride)
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (u + k * stride < units) turn(f[k], u + k * stride);
  }
  if constexpr (kFewExponents<T>) {
    shift(dk, -power);
    shift(dv, -kLikely);
  }
  if constexpr (QW > 1) {
    float* jo = (float*)lds + (rw * 32 + col) * (DP + 1);
    for (int k = 1; k < QW; ++k)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        f32x16* acc = which ? dv : dk;
        __syncthreads();
        if (qw == k)
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) jo[32 * d + acc_row(r, half)] = acc[d][r];
        __syncthreads();
        if (qw == 0)
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] += jo[32 * d + acc_row(r, half)];
      }
  }
  if (qw != 0 || !exists) return;
  const int64_t off = (((int64_t)b * a.Lk + key) * a.Hkv + hk) * a.D;
  if (parts > 1) {  // k_attend_dkv_join adds them up
    float* pk = a.part + (((int64_t)slot + part) * 2 * a.block + 32 * rw + col) * a.D;
    float* pv = pk + (int64_t)a.block * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int e = 32 * d + 8 * c + 4 * half;
        if (e >= a.D) continue;
        store4<float>(pk + e, dk[d][4 * c] * a.scale, dk[d][4 * c + 1] * a.scale, dk[d][4 * c + 2] * a.scale,
                      dk[d][4 * c + 3] * a.scale);
        store4<float>(pv + e, dv[d][4 * c], dv[d][4 * c + 1], dv[d][4 * c + 2], dv[d][4 * c + 3]);
      }
    return;
  }
  const float f = a.scale;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int e = 32 * d + 8 * c + 4 * half;
      if (e >= a.D) continue;
      if (valid) {
        store4<T>((T*)a.dk + off + e, dk[d][4 * c] * f, dk[d][4 * c + 1] * f, dk[d][4 * c + 2] * f, dk[d][4 * c + 3] * f);
        store4<T>((T*)a.dv + off + e, dv[d][4 * c], dv[d][4 * c + 1], dv[d][4 * c + 2], dv[d][4 * c + 3]);
      } else {
        store4<T>((T*)a.dk + off + e, 0.f, 0.f, 0.f, 0.f);
        store4<T>((T*)a.dv + off + e, 0.f, 0.f, 0.f, 0.f);
      }
    }
}

template <typename K>
int launch(K kernel, const Args& a, dim3 grid, size_t lds, hipStream_t st, const char* what) {
  if (lds > 32 * 1024)
    if (int e = dsplat::ensure_dyn_lds((const void*)kernel, lds, what)) return e;
  kernel<<<grid, kThreads, lds, st>>>(a);
  return dsplat::check_launch(what);
}

// 32-row waves side by side: as many as the tile's rows fill.
inline int row_waves(const Args& a) {
  const int rows = a.Lt * a.G;
  return rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
}
// Parts of the key list: enough workgroups for the chip when there are few tiles, of 8 units or more each (one token
// of 16 sequences, 64 units: 8 parts 14.2 us and 4.0 for their join, 16 parts 13.3 and 4.8).
inline int splits_of(int64_t workgroups, int units) {
  int s = 1;
  while (workgroups * s < 512 && s * 8 < units) s *= 2;
  return s;
}

template <typename T, int DP, int RW>
struct Fwd {
  static int go(const Args& a, dim3 grid, hipStream_t st) {
    const size_t lds = kTileBytes<T, DP, 4 / RW> + a.top * sizeof(int32_t);
    if constexpr (sizeof(T) == 2)
      if (a.rest) return launch(k_attend_fwd<T, DP, RW, true>, a, grid, lds, st, "k_attend_fwd");
    return launch(k_attend_fwd<T, DP, RW, false>, a, grid, lds, st, "k_attend_fwd");
  }
};
template <typename T, int DP, int RW>
struct Dq {
  static int go(const Args& a, dim3 grid, hipStream_t st) {
    return launch(k_attend_dq<T, DP, RW>, a, grid, kTileBytes<T, DP, 4 / RW * kEach<T, RW>> + a.top * sizeof(int32_t), st, "k_attend_dq");
  }
};
template <typename T, int DP, int RW>
struct Dkv {
  static int go(const Args& a, dim3 grid, hipStream_t st) {
    return launch(k_attend_dkv<T, DP, RW>, a, grid, (2 * (4 / RW) + (kRowsInLds<T, DP, RW> ? 2 * RW : 0)) * Tile<T, DP>::kUnit, st, "k_attend_dkv");
  }
};
template <template <typename, int, int> class F, typename T, int DP>
int by_waves(int rw, const Args& a, dim3 grid, hipStream_t st) {
  return rw == 1 ? F<T, DP, 1>::go(a, grid, st) : rw == 2 ? F<T, DP, 2>::go(a, grid, st) : F<T, DP, 4>::go(a, grid, st);
}
template <template <typename, int, int> class F, typename T>
int by_width(int rw, const Args& a, dim3 grid, hipStream_t st) {
  if (a.D <= 32) return by_waves<F, T, 32>(rw, a, grid, st);
  if (a.D <= 64) return by_waves<F, T, 64>(rw, a, grid, st);
  if (a.D <= 96) return by_waves<F, T, 96>(rw, a, grid, st);
  return by_waves<F, T, 128>(rw, a, grid, st);
}

template <typename T>
int attend_fwd(const Args& a, int row_waves, dim3 grid, hipStream_t st) {
  return by_width<Fwd, T>(row_waves, a, grid, st);
}
template <typename T>
int attend_dq(const Args& a, int row_waves, dim3 grid, hipStream_t st) {
  return by_width<Dq, T>(row_waves, a, grid, st);
}
template <typename T>
int attend_dkv(const Args& a, int row_waves, dim3 grid, hipStream_t st) {
  return by_width<Dkv, T>(row_waves, a, grid, st);
}

// One translation unit per element type compiles these.
#define DTK_ATTEND(EXTERN, T)                                                \
  EXTERN template int attend_fwd<T>(const Args&, int, dim3, hipStream_t);    \
  EXTERN template int attend_dq<T>(const Args&, int, dim3, hipStream_t);     \
  EXTERN template int attend_dkv<T>(const Args&, int, dim3, hipStream_t);
DTK_ATTEND(extern, float)
DTK_ATTEND(extern, bf16)
DTK_ATTEND(extern, f16)

}  // namespace dtk
