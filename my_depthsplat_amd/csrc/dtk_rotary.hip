// dtk_rotary.hip — rotary positions of queries and keys for gfx950, forward and (the opposite
// angle) backward, both tensors in one launch.
//
//   pair i of a head turns by angle_i = position[axis(i)] freqs[i]; (a, b) -> (a c - b s, a s + b c)
//   pairs: (i, i + F) (halves) or (2i, 2i + 1) (interleaved), F = number of frequencies; the
//   channels behind 2F are copied; axis(i) = i / (F / axes).
//
// Bound by memory: each channel is read and written once. The angle is taken in 64 bits as turns
// and reduced to one turn there (a far position times a frequency needs more digits than 32
// bits hold); the sine and cosine are then of a small number in 32 bits. A thread takes the
// sines of its channels once and turns every head of its token with them.
//
// Measured: 92160 tokens, 2 + 2 heads of 64 bf16, two axes: 22 us a direction, 4.3 TB/s (a copy of 256 MB 5.4); 16 single tokens
// of 8 + 2 heads 4.0 us, a launch and the chain position, frequency, sine.

#include "dtk_common.h"

namespace {
using namespace dtk;

constexpr int NT = 256;

struct RotaryArgs {
  int64_t L, tokens;  // tokens per sequence; of all sequences
  int units;          // per token
  int Hq, Hk, D, F, per_axis, axes, groups, heads_per;
  const void *q, *k, *pos;
  int64_t qb, ql, qh, kb, kl, kh, pb, pl, pa;  // strides in elements
  const double* freqs;
  float factor;
  void *oq, *ok;  // contiguous [B, L, H, D]
};

// The sines of pairs i .. i + NP - 1 at a token. A vector's pairs have one axis where the frequencies of an axis are
// whole vectors (same).
template <typename P, int NP>
__device__ __forceinline__ void angles(const RotaryArgs& a, const P* pos, int i, bool same, bool back, float (&c)[NP], float (&s)[NP]) {
  double f[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) f[k] = a.freqs[i + k];
  const double p0 = (double)pos[(i / a.per_axis) * a.pa];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const double p = same ? p0 : (double)pos[((i + k) / a.per_axis) * a.pa];
    const double t = p * (f[k] * 0.15915494309189533577);  // turns
    float sn, cs;
    sincospif((float)(2.0 * (t - rint(t))), &sn, &cs);
    c[k] = cs * a.factor;
    s[k] = (back ? -sn : sn) * a.factor;
  }
}

template <typename T, int N>
struct Piece {
  T v[N];
  static __device__ __forceinline__ Piece load(const T* p) {
    Piece r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
  }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, this, sizeof(*this)); }
};

// N = channels of a vector (16 bytes) or 1. Units of a token: halves: the F / N vector pairs,
// then the copied vectors; interleaved: the vectors (N = 1: the pairs, then the copied channels).
template <typename T, typename P, int N, bool INTER, bool BACK>
__device__ __forceinline__ void turn_unit(const RotaryArgs& a, const P* pos, int64_t token, int64_t b, int64_t l, int g, int u) {
  constexpr bool PAIR = !INTER || N == 1;  // the unit holds both ends of its pairs as two vectors
  const int turning = PAIR ? a.F / N : 2 * a.F / N;
  const bool copy = u >= turning;
  const int c0 = copy ? (PAIR ? 2 * a.F + (u - turning) * N : u * N) : (INTER ? (N == 1 ? 2 * u : u * N) : u * N);
  const int step = INTER ? 1 : a.F;  // from a pair's first channel (vector) to its second
  constexpr int NP = PAIR ? N : N / 2;
  constexpr int K = 4;  // heads whose channels are on their way together
  const int h1 = min((g + 1) * a.heads_per, a.Hq + a.Hk);
  const auto in = [&](int h) {
    return h < a.Hq ? (const T*)a.q + b * a.qb + l * a.ql + h * a.qh : (const T*)a.k + b * a.kb + l * a.kl + (h - a.Hq) * a.kh;
  };
  const auto out = [&](int h) {
    return h < a.Hq ? (T*)a.oq + (token * a.Hq + h) * a.D : (T*)a.ok + (token * a.Hk + (h - a.Hq)) * a.D;
  };
  using V = Piece<T, N>;
  V x[K], y[K];
  const auto fetch = [&](int h) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (h + k < h1) {
        x[k] = V::load(in(h + k) + c0);
        if (PAIR && !copy) y[k] = V::load(in(h + k) + c0 + step);
      }
  };
  fetch(g * a.heads_per);
  float c[NP], s[NP];
  if (!copy) angles<P, NP>(a, pos, INTER ? c0 / 2 : c0, a.per_axis % NP == 0, BACK, c, s);
  for (int h = g * a.heads_per; h < h1; h += K) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (h + k >= h1) break;
      if (!copy) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          T& p = PAIR ? x[k].v[i] : x[k].v[2 * i % N];
          T& q = PAIR ? y[k].v[i] : x[k].v[(2 * i + 1) % N];
          const float f = (float)p, t = (float)q;
          p = (T)(f * c[i] - t * s[i]);
          q = (T)(f * s[i] + t * c[i]);
        }
        if (PAIR) y[k].store(out(h + k) + c0 + step);
      }
      x[k].store(out(h + k) + c0);
    }
    if (h + K < h1) fetch(h + K);
  }
}

template <typename T, typename P, int N, bool INTER, bool BACK>
__global__ __launch_bounds__(NT) void k_rotary(RotaryArgs a) {
  const int g = blockIdx.y;
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (token >= a.tokens) return;
  const int64_t b = (uint32_t)token / (uint32_t)a.L, l = token - b * a.L;  // fewer than 2^31 tokens (the host checks)
  const P* pos = (const P*)a.pos + b * a.pb + l * a.pl;
  for (int u = threadIdx.x; u < a.units; u += blockDim.x) turn_unit<T, P, N, INTER, BACK>(a, pos, token, b, l, g, u);
}

template <typename T, typename P, int N>
void launch(const RotaryArgs& a, bool inter, bool back, hipStream_t st) {
  const int ux = a.units < NT ? a.units : NT, ty = NT / ux;  // a token's units side by side, tokens above each other
  const dim3 block(ux, ty), grid((unsigned)((a.tokens + ty - 1) / ty), a.groups);
  if (inter)
    back ? k_rotary<T, P, N, true, true><<<grid, block, 0, st>>>(a) : k_rotary<T, P, N, true, false><<<grid, block, 0, st>>>(a);
  else
    back ? k_rotary<T, P, N, false, true><<<grid, block, 0, st>>>(a) : k_rotary<T, P, N, false, false><<<grid, block, 0, st>>>(a);
}
template <typename T>
void by_pos(const RotaryArgs& a, int ptype, bool vec, bool inter, bool back, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  if (ptype == DTK_I64) vec ? launch<T, int64_t, N>(a, inter, back, st) : launch<T, int64_t, 1>(a, inter, back, st);
  else if (ptype == DTK_I32) vec ? launch<T, int32_t, N>(a, inter, back, st) : launch<T, int32_t, 1>(a, inter, back, st);
  else vec ? launch<T, float, N>(a, inter, back, st) : launch<T, float, 1>(a, inter, back, st);
}

}  // namespace

extern "C" int dtk_rotary(int64_t B, int64_t L, int Hq, int Hk, int D, int F, int axes, int interleaved, int backward,
                          int dtype, int ptype, const void* q, const int64_t* q_strides, const void* k,
                          const int64_t* k_strides, const void* positions, const int64_t* pos_strides,
                          const double* freqs, float factor, void* q_out, void* k_out, void* stream) {
  DSPLAT_REQUIRE(B >= 0 && L >= 0 && (L == 0 || B < (1LL << 31) / L) && Hq >= 0 && Hk >= 0 && D > 0 && Hq < 65536 && Hk < 65536 && D < (1 << 20),
                 "dtk_rotary: bad sizes");
  DSPLAT_REQUIRE(F >= 0 && F <= D / 2 && axes > 0 && F % axes == 0, "dtk_rotary: bad number of frequencies");
  DSPLAT_REQUIRE(type_ok(dtype) && (ptype == DTK_I64 || ptype == DTK_I32 || ptype == DTK_F32), "dtk_rotary: bad types");
  if (B == 0 || L == 0 || Hq + Hk == 0) return 0;
  DSPLAT_REQUIRE((!Hq || (q && q_strides && q_out)) && (!Hk || (k && k_strides && k_out)) &&
                     (!F || (positions && pos_strides && freqs)),
                 "dtk_rotary: null pointer");
  RotaryArgs a = {};
  a.L = L;
  a.Hq = Hq;
  a.Hk = Hk;
  a.D = D;
  a.F = F;
  a.axes = axes;
  a.per_axis = F ? F / axes : 1;
  a.q = q;
  a.k = k;
  a.pos = positions;
  if (Hq) a.qb = q_strides[0], a.ql = q_strides[1], a.qh = q_strides[2];
  if (Hk) a.kb = k_strides[0], a.kl = k_strides[1], a.kh = k_strides[2];
  if (F) a.pb = pos_strides[0], a.pl = pos_strides[1], a.pa = pos_strides[2];
  a.freqs = freqs;
  a.factor = factor;
  a.oq = q_out;
  a.ok = k_out;
  const int n = dtype == DTK_F32 ? 4 : 8;
  const bool vec = D % n == 0 && (interleaved ? 2 * F : F) % n == 0 && (2 * F) % n == 0;
  const int m = vec ? n : 1;
  a.units = (interleaved && vec) ? D / m : F / m + (D - 2 * F) / m;
  // all heads of a token in one thread, unless that leaves the chip idle
  const int heads = Hq + Hk;
  const int64_t threads = B * L * a.units;
  int groups = 1;
  while (groups < heads && threads * groups < 256 * 1024) groups *= 2;
  a.heads_per = (heads + groups - 1) / groups;
  a.groups = (heads + a.heads_per - 1) / a.heads_per;
  a.tokens = B * L;
  DSPLAT_REQUIRE(a.tokens < (1LL << 31) && a.groups < 65536, "dtk_rotary: too large");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DTK_F32) by_pos<float>(a, ptype, vec, interleaved != 0, backward != 0, st);
  else if (dtype == DTK_BF16) by_pos<bf16>(a, ptype, vec, interleaved != 0, backward != 0, st);
  else by_pos<f16>(a, ptype, vec, interleaved != 0, backward != 0, st);
  return dsplat::check_launch("k_rotary");
}
