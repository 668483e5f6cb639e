// Per-head RMS norm and position rotation of queries and keys, alone (forward and backward) and on the way into a paged
// key / value cache.
//
//   n = x * rsqrt(mean_d x^2 + eps) * w          (skipped without weights)
//   pair i of the first `rot` values, angle t = pos * freqs[i], amplitude s:
//   y_lo = s (n_lo cos t - n_hi sin t),  y_hi = s (n_hi cos t + n_lo sin t);   y = n beyond `rot`
//   pairs: halves (i, i + rot / 2), or interleaved (2 i, 2 i + 1)
//   backward, u = R(-t) dy:   dw = sum x^ u,  dx = r (u w - x^ mean_d(u w x^)),  x^ = x r,  r = rsqrt(...)
//
// Bound by HBM: every value is read and written once (bf16, 16385 rows of 32 + 8 heads of 128: 336 MB in 73 us, 4.6 TB/s where
// a large copy reaches 4.9; forward and backward of 33920 rows of 16 + 16 heads of 64: 695 MB in 170 us; appended to a cache,
// 14590 rows of 16 + 4 + 4 heads of 64: 90 MB in 24 us).  A lane holds two 16-byte vectors of one head, chosen so that both
// members of its pairs are its own (halves: the vectors at V j and rot / 2 + V j; interleaved: neighbours), so the rotation
// needs no exchange and a load instruction still covers runs of 128 bytes at 128 values a head.  LP lanes (a power of two)
// hold a head, 64 / LP heads go through a wave at once, and a wave keeps to one row while it walks the heads: the row's
// sines and cosines are computed once and stay in registers.
// Angles are formed in 64 bits in TURNS (pos * freqs / 2 pi, the whole turns dropped): in 32 bits a position of 10^6 has
// lost a twentieth of a radian.  The sine and cosine of the remaining fraction are taken in 32 bits where the outputs have
// 16 (error 2^-22, a rounding of the output is 2^-9) and in 64 where they have 32.
#include <type_traits>

#include "common.h"

namespace {

struct HeadTensor {
  const void* x;        // (M, H, D): row and head strides in elements, unit inner stride
  long long row, head;
  const void* dy;       // backward: (M, H, D) like x, strides of its own
  long long dy_row, dy_head;
  const float* w;       // (D) or null
  void* out;            // contiguous (M, H, D)
  int H, steps;         // steps: passes of 64 / LP heads
};

struct NormRotaryParams {
  HeadTensor t[2];              // queries, keys
  const int* pos;               // (M)
  const double* freqs;          // (rot / 2) radians per position
  float amplitude, eps, inv_d;  // inv_d: 1 / D
  long long M;
  int D, rot, lp, hsplit;       // lanes per head; parts a row's steps are split into
  int rows;                     // rows a wave takes at once (MULTI; a power of two)
  float* dw_part;               // backward: (blocks, 2, D) or null
  // ---- paged cache (append)
  const int *seq, *table;       // (M); (S, width)
  long long table_ld;
  int S, width, pages, page_shift, zero_pad;
  const void* v;                // (M, Hk, D)
  long long v_row, v_head;
  void *k_pages, *v_pages;      // (pages, Hk, page size, D)
};

constexpr double INV_2PI = 0.15915494309189533577;

template <typename T>
struct V16 {
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void to_f32(u32x4 r, float* f) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = half_lo(r[e]);
        f[2 * e + 1] = half_hi(r[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(r[e]);
    }
  }
  static __device__ __forceinline__ u32x4 from_f32(const float* f) {
    if constexpr (sizeof(T) == 2)
      return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    else
      return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
  }
};

// sum over the lp (power of two) neighbouring lanes that hold a head; every one of them gets it
__device__ __forceinline__ float head_sum(float v, int lp) {
  if (lp > 1) v += dpp_move<0xB1>(v);
  if (lp > 2) v += dpp_move<0x4E>(v);
  if (lp > 4) v += dpp_move<0x141>(v);
  if (lp > 8) v += dpp_move<0x140>(v);
  if (lp > 16) v += __shfl_xor(v, 16, 64);
  return v;
}

// where this lane's two vectors lie in a head, and whether they turn
template <typename T, bool INTERLEAVED>
struct Lane {
  static constexpr int N = V16<T>::N;
  int a, b, pair0;
  bool active, turns;
  __device__ __forceinline__ Lane(int j, int D, int rot) {
    active = 2 * N * j < D;
    if (!active) j = 0;   // (its loads stay inside the head, its results are dropped)
    a = 2 * N * j;
    b = a + N;
    turns = a < rot;
    pair0 = N * j;
    if (!INTERLEAVED && turns) {
      a = N * j;
      b = rot / 2 + N * j;
    }
  }
  // members e of the pairs among the lane's 2 N values (first vector, then second)
  static __device__ __forceinline__ int lo(int e) { return INTERLEAVED ? 2 * e : e; }
  static __device__ __forceinline__ int hi(int e) { return INTERLEAVED ? 2 * e + 1 : N + e; }
};

// sine and cosine of t turns, |t| <= 1/2: the nearest quarter turn dropped, Taylor sums to x^9 / x^8 on |x| <= pi / 4 (the
// next terms are below 2^-25), the quarter put back by exchange and signs.  Half the instructions of a general routine, which
// were a third of the kernel at 16 heads of 64.
__device__ __forceinline__ void turn_sincos(float t, float& s, float& c) {
  const float k = rintf(4.f * t), x = (t - 0.25f * k) * 6.283185307179586f, y = x * x;
  const float sn = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.f);
  const float cs = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 2.4801587e-5f, -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
  const int q = (int)k;
  const bool odd = q & 1;
  s = odd ? cs : sn;
  c = odd ? sn : cs;
  if (q & 2) s = -s;
  if ((q + 1) & 2) c = -c;
}

template <typename T>
__device__ __forceinline__ void cos_sin(int pos, const double* turns_per_pos, float amplitude, float* c, float* s) {
  constexpr int N = V16<T>::N;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const double whole = rint((double)pos * turns_per_pos[e]), t = fma((double)pos, turns_per_pos[e], -whole);
    if constexpr (sizeof(T) == 2) {
      turn_sincos((float)t, s[e], c[e]);
    } else {
      double sd, cd;
      sincospi(2.0 * t, &sd, &cd);
      s[e] = (float)sd;
      c[e] = (float)cd;
    }
    c[e] *= amplitude;
    s[e] *= amplitude;
  }
}

// (products and sums are fused by hand here and below: left to hipcc, which of them it fuses differs between the kernels, and
// a key would not have the same bits in a cache as outside.  Values that do not turn are left as they are: a turn by nothing
// would multiply a neighbour by 0, and 0 * NaN is not 0.  By a choice of every result, except in the forward without a cache,
// where the lanes that do not turn skip this: 14590 rows of 16 + 4 heads of 64 in bf16 take 23 us a call into a cache, 27
// behind a branch, and 16385 of 32 + 8 of 128 without one 71 behind a branch, 73 turned by nothing.)
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void turn(float* x, const float* c, const float* s, bool turns) {
  using L = Lane<T, INTERLEAVED>;
#pragma unroll
  for (int e = 0; e < L::N; ++e) {
    const float lo = x[L::lo(e)], hi = x[L::hi(e)];
    x[L::lo(e)] = turns ? fmaf(lo, c[e], -(hi * s[e])) : lo;
    x[L::hi(e)] = turns ? fmaf(hi, c[e], lo * s[e]) : hi;
  }
}

// the transpose of `turn`, by a choice of every result: behind a branch 33920 rows of 16 + 16 heads of 64 in f32 take 124 us
// instead of 120, 16385 rows of 32 + 8 heads of 128 in bf16 100 instead of 99 (the forward is the faster behind one: 71 / 73)
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void turn_back(float* x, const float* c, const float* s, bool turns) {
  using L = Lane<T, INTERLEAVED>;
#pragma unroll
  for (int e = 0; e < L::N; ++e) {
    const float lo = x[L::lo(e)], hi = x[L::hi(e)];
    x[L::lo(e)] = turns ? fmaf(lo, c[e], hi * s[e]) : lo;
    x[L::hi(e)] = turns ? fmaf(hi, c[e], -(lo * s[e])) : hi;
  }
}

// One wave per item = (row, part of its steps), or with MULTI per `rows` rows, items strided over the grid.  PAGED: the keys go to their page, values
// are copied to theirs by further steps, and rows of negative position or sequence are padding.
template <typename T, bool INTERLEAVED, bool NORM, bool PAGED, bool MULTI>
__global__ __launch_bounds__(256) void norm_rotary_fwd_kernel(NormRotaryParams p) {
  using L = Lane<T, INTERLEAVED>;
  constexpr int N = L::N, U = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lp = p.lp, hpw = 64 / lp / (MULTI ? p.rows : 1), slot = MULTI ? lane / lp % hpw : lane / lp;
  const L at(lane % lp, p.D, p.rot);
  double freq[N];
#pragma unroll
  for (int e = 0; e < N; ++e) freq[e] = at.turns ? p.freqs[at.pair0 + e] * INV_2PI : 0.0;
  float w[2][2 * N] = {};
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        w[i][e] = p.t[i].w[at.a + e];
        w[i][N + e] = p.t[i].w[at.b + e];
      }
  }
  const int nq = p.t[0].steps, nk = p.t[1].steps, total = nq + nk + (PAGED ? nk : 0);
  const int part = (total + p.hsplit - 1) / p.hsplit;
  const long long items = MULTI ? (p.M + p.rows - 1) / p.rows : p.M * p.hsplit, stride = (long long)gridDim.x * 4;
  for (long long item = (long long)blockIdx.x * 4 + wave; item < items; item += stride) {
    long long row = MULTI ? item * p.rows + lane / lp / hpw : item;
    int s0 = 0, s1 = total;
    if constexpr (MULTI) {
      if (row >= p.M) continue;   // (all lanes of a head)
    } else if (p.hsplit > 1) {   // (few rows then: 32 bits do)
      row = (int)item / p.hsplit;
      s0 = ((int)item % p.hsplit) * part;
      s1 = min(s0 + part, total);
    }
    const int pos = p.pos[row];
    long long page_row = -1;   // PAGED: element offset of the row's slot in a page of one head (without the head's part)
    bool pad = false;
    if constexpr (PAGED) {
      const int sq = p.seq[row];
      pad = pos < 0 || sq < 0;
      const int col = pos >> p.page_shift;
      if (!pad && sq < p.S && col < p.width) {
        const int page = p.table[(long long)sq * p.table_ld + col];
        if (page >= 0 && page < p.pages)
          page_row = ((((long long)page * p.t[1].H) << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) * p.D;
      }
      if (pad && !p.zero_pad) continue;
    }
    float c[N], s[N];
    cos_sin<T>(pos, freq, p.amplitude, c, s);
    for (int st0 = s0; st0 < s1; st0 += U) {
      u32x4 ra[U], rb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {   // unconditional loads of a clamped step and head, all in flight at once
        const int st = min(st0 + u, s1 - 1);
        const T* x;
        if (!PAGED || st < nq + nk) {
          const int i = st < nq ? 0 : 1;
          const HeadTensor& t = p.t[i];
          const int h = min((st - (i ? nq : 0)) * hpw + slot, t.H - 1);
          x = (const T*)t.x + row * t.row + h * t.head;
        } else {
          const int h = min((st - nq - nk) * hpw + slot, p.t[1].H - 1);
          x = (const T*)p.v + row * p.v_row + h * p.v_head;
        }
        ra[u] = *(const u32x4*)(x + at.a);
        rb[u] = *(const u32x4*)(x + at.b);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int st = st0 + u;
        if (st >= s1) break;
        if (PAGED && st >= nq + nk) {
          const int h = (st - nq - nk) * hpw + slot;
          if (at.active && h < p.t[1].H && page_row >= 0) {
            T* o = (T*)p.v_pages + page_row + (((long long)h * p.D) << p.page_shift);
            *(u32x4*)(o + at.a) = ra[u];
            *(u32x4*)(o + at.b) = rb[u];
          }
          continue;
        }
        // (one body per tensor: a choice of weights inside one costs a select per value)
        auto head = [&](auto which, const float (&wt)[2 * N]) __attribute__((always_inline)) {
          constexpr int i = decltype(which)::value;
          const int h = (st - (i ? nq : 0)) * hpw + slot;
          float x[2 * N];
          V16<T>::to_f32(ra[u], x);
          V16<T>::to_f32(rb[u], x + N);
          if constexpr (NORM) {
            float q = 0.f;
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) q = fmaf(x[e], x[e], q);
            const float r = rsqrtf(fmaf(head_sum(at.active ? q : 0.f, lp), p.inv_d, p.eps));
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) x[e] *= r * wt[e];
          }
          if constexpr (PAGED) turn<T, INTERLEAVED>(x, c, s, at.turns);
          else if (at.turns) turn<T, INTERLEAVED>(x, c, s, true);
          if (!at.active || h >= p.t[i].H) return;
          T* o;
          if (PAGED && i == 1) {
            if (page_row < 0) return;
            o = (T*)p.k_pages + page_row + (((long long)h * p.D) << p.page_shift);
          } else {
            o = (T*)p.t[i].out + (row * p.t[i].H + h) * p.D;
          }
          const bool z = PAGED && pad;
          *(u32x4*)(o + at.a) = z ? u32x4{0u, 0u, 0u, 0u} : V16<T>::from_f32(x);
          *(u32x4*)(o + at.b) = z ? u32x4{0u, 0u, 0u, 0u} : V16<T>::from_f32(x + N);
        };
        if (st < nq) head(std::integral_constant<int, 0>(), w[0]);
        else head(std::integral_constant<int, 1>(), w[1]);
      }
    }
  }
}

// Backward: the same walk over rows and heads; the weights' gradients are summed per lane over all its rows, then over the
// workgroup in LDS in a fixed order, and written as one row of partial sums per workgroup (reduced by melgpt_reduce_rows:
// no atomics, the same bits every time).
template <typename T, bool INTERLEAVED, bool NORM, bool MULTI>
__global__ __launch_bounds__(256) void norm_rotary_bwd_kernel(NormRotaryParams p) {
  using L = Lane<T, INTERLEAVED>;
  constexpr int N = L::N, U = 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lp = p.lp, hpw = 64 / lp / (MULTI ? p.rows : 1), slot = MULTI ? lane / lp % hpw : lane / lp;
  const L at(lane % lp, p.D, p.rot);
  double freq[N];
#pragma unroll
  for (int e = 0; e < N; ++e) freq[e] = at.turns ? p.freqs[at.pair0 + e] * INV_2PI : 0.0;
  float w[2][2 * N] = {}, dw[2][2 * N] = {};
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        w[i][e] = p.t[i].w[at.a + e];
        w[i][N + e] = p.t[i].w[at.b + e];
        dw[i][e] = dw[i][N + e] = 0.f;
      }
  }
  const int nq = p.t[0].steps, total = nq + p.t[1].steps;
  const int part = (total + p.hsplit - 1) / p.hsplit;
  const long long items = MULTI ? (p.M + p.rows - 1) / p.rows : p.M * p.hsplit, stride = (long long)gridDim.x * 4;
  for (long long item = (long long)blockIdx.x * 4 + wave; item < items; item += stride) {
    long long row = MULTI ? item * p.rows + lane / lp / hpw : item;
    int s0 = 0, s1 = total;
    if constexpr (MULTI) {
      if (row >= p.M) continue;   // (all lanes of a head)
    } else if (p.hsplit > 1) {   // (few rows then: 32 bits do)
      row = (int)item / p.hsplit;
      s0 = ((int)item % p.hsplit) * part;
      s1 = min(s0 + part, total);
    }
    float c[N], s[N];
    cos_sin<T>(p.pos[row], freq, p.amplitude, c, s);
    for (int st0 = s0; st0 < s1; st0 += U) {
      u32x4 ga[U], gb[U], ra[U], rb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int st = min(st0 + u, s1 - 1), i = st < nq ? 0 : 1;
        const HeadTensor& t = p.t[i];
        const int h = min((st - (i ? nq : 0)) * hpw + slot, t.H - 1);
        const T* g = (const T*)t.dy + row * t.dy_row + h * t.dy_head;
        ga[u] = *(const u32x4*)(g + at.a);
        gb[u] = *(const u32x4*)(g + at.b);
        if constexpr (NORM) {
          const T* x = (const T*)t.x + row * t.row + h * t.head;
          ra[u] = *(const u32x4*)(x + at.a);
          rb[u] = *(const u32x4*)(x + at.b);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int st = st0 + u;
        if (st >= s1) break;
        auto head = [&](auto which, const float (&wt)[2 * N], float (&dwt)[2 * N]) __attribute__((always_inline)) {
          constexpr int i = decltype(which)::value;
          const int h = (st - (i ? nq : 0)) * hpw + slot;
          const bool mine = at.active && h < p.t[i].H;
          float g[2 * N];
          V16<T>::to_f32(ga[u], g);
          V16<T>::to_f32(gb[u], g + N);
          turn_back<T, INTERLEAVED>(g, c, s, at.turns);
          if constexpr (NORM) {
            float x[2 * N], q = 0.f;
            V16<T>::to_f32(ra[u], x);
            V16<T>::to_f32(rb[u], x + N);
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) q = fmaf(x[e], x[e], q);
            const float r = rsqrtf(fmaf(head_sum(at.active ? q : 0.f, lp), p.inv_d, p.eps));
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) {
              x[e] *= r;
              dwt[e] += mine ? g[e] * x[e] : 0.f;
              g[e] *= wt[e];
              m = fmaf(g[e], x[e], m);
            }
            m = head_sum(at.active ? m : 0.f, lp) * p.inv_d;
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) g[e] = r * fmaf(-x[e], m, g[e]);
          }
          if (!mine) return;
          T* o = (T*)p.t[i].out + (row * p.t[i].H + h) * p.D;
          *(u32x4*)(o + at.a) = V16<T>::from_f32(g);
          *(u32x4*)(o + at.b) = V16<T>::from_f32(g + N);
        };
        if (st < nq) head(std::integral_constant<int, 0>(), w[0], dw[0]);
        else head(std::integral_constant<int, 1>(), w[1], dw[1]);
      }
    }
  }
  if constexpr (NORM) {
    // 256 / lp lane groups hold partial sums of the same D values: group s writes its D values to sh[s], thread d adds them
    extern __shared__ __attribute__((aligned(16))) float sh[];
    const int groups = 256 / lp, g = threadIdx.x / lp;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i) __syncthreads();
      if (at.active) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          sh[g * p.D + at.a + e] = dw[i][e];
          sh[g * p.D + at.b + e] = dw[i][N + e];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < p.D; d += 256) {
        float a = 0.f;
        for (int k = 0; k < groups; ++k) a += sh[k * p.D + d];
        p.dw_part[((long long)blockIdx.x * 2 + i) * p.D + d] = a;
      }
    }
  }
}

int lanes_per_head(int D, int dtype) {
  const int n = 2 * (dtype == MELGPT_F32 ? 4 : 8);
  int lp = 1;
  while (lp * n < D) lp *= 2;
  return lp;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_tensor(const HeadTensor& t, int vec) {
  if (!t.x || t.H <= 0) return MELGPT_ERR_BAD_ARG;
  if (!aligned16(t.x) || t.row % vec || t.head % vec) return MELGPT_ERR_ALIGN;
  return MELGPT_OK;
}

int check_common(const NormRotaryParams& p, int dtype) {
  if (p.M < 0 || p.D <= 0 || !p.pos || p.rot < 0) return MELGPT_ERR_BAD_ARG;
  if (dtype != MELGPT_F32 && dtype != MELGPT_BF16) return MELGPT_ERR_UNSUPPORTED;
  if (p.D % 16 || p.D > 256 || p.rot % 16 || p.rot > p.D) return MELGPT_ERR_UNSUPPORTED;
  if (p.rot > 0 && !p.freqs) return MELGPT_ERR_BAD_ARG;
  if (!p.t[0].w != !p.t[1].w) return MELGPT_ERR_BAD_ARG;
  return MELGPT_OK;
}

// Where a wave has twice the room for all heads of a row or more, it takes 2, 4, .. rows at once while 2048 waves (2 a SIMD) of
// them remain: a row's sines cost its wave as much as two passes of heads.  33920 rows in bf16, one row / several: 1 + 1 heads
// of 64 40.8 / 8.9 us, of 256 43.8 / 20.5, 16 + 16 heads of 32 47 / 32; backward 69.5 / 25.1, 73.8 / 35.3, 82.7 / 56.9.
// Steps of a row are shared out over several waves only while there are too few rows to fill the card (a part computes
// the row's sines again): 2 waves for each SIMD of the 256 CUs.  Measured in bf16, 32 + 8 heads of 128, whole rows / this / 8
// waves a SIMD: 1 row 6.0 / 4.0 / 3.9 us, 256 rows 6.8 / 5.3 / 5.3, 1024 rows 8.1 / 7.5 / 10.6.
void plan(NormRotaryParams& p, int dtype, int steps_extra) {
  p.lp = lanes_per_head(p.D, dtype);
  p.inv_d = 1.f / (float)p.D;
  int hpw = 64 / p.lp;
  const int heads = p.t[0].H > p.t[1].H ? p.t[0].H : p.t[1].H;
  p.rows = 1;
  while (2 * heads <= hpw && p.M >= 4096LL * p.rows) {
    p.rows *= 2;
    hpw /= 2;
  }
  for (int i = 0; i < 2; ++i) p.t[i].steps = (p.t[i].H + hpw - 1) / hpw;
  const int total = p.t[0].steps + p.t[1].steps + (steps_extra ? p.t[1].steps : 0);
  long long want = p.M > 0 ? (2048 + p.M - 1) / p.M : 1;
  p.hsplit = (int)(want < 1 ? 1 : want > total ? total : want);   // (1 where a wave takes several rows)
}

long long blocks_for(const NormRotaryParams& p, long long most) {
  const long long b = ((p.rows > 1 ? (p.M + p.rows - 1) / p.rows : p.M * p.hsplit) + 3) / 4;
  return b < most ? b : most;
}

template <typename T, bool INTERLEAVED, bool NORM, bool PAGED>
void launch_fwd_rows(const NormRotaryParams& p, hipStream_t s) {
  const dim3 grid((unsigned)blocks_for(p, 2048)), block(256);
  if (p.rows > 1) hipLaunchKernelGGL((norm_rotary_fwd_kernel<T, INTERLEAVED, NORM, PAGED, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((norm_rotary_fwd_kernel<T, INTERLEAVED, NORM, PAGED, false>), grid, block, 0, s, p);
}

template <typename T, bool PAGED>
void launch_fwd(const NormRotaryParams& p, int interleaved, hipStream_t s) {
  const bool norm = p.t[1].w != nullptr;
  if (interleaved) {
    if (norm) launch_fwd_rows<T, true, true, PAGED>(p, s);
    else launch_fwd_rows<T, true, false, PAGED>(p, s);
  } else {
    if (norm) launch_fwd_rows<T, false, true, PAGED>(p, s);
    else launch_fwd_rows<T, false, false, PAGED>(p, s);
  }
}

template <typename T, bool INTERLEAVED, bool NORM>
void launch_bwd_rows(const NormRotaryParams& p, unsigned blocks, hipStream_t s) {
  const dim3 grid(blocks), block(256);
  const size_t lds = NORM ? (size_t)(256 / p.lp) * p.D * sizeof(float) : 0;   // <= 256 * 2 N floats: 16 KB
  if (p.rows > 1) hipLaunchKernelGGL((norm_rotary_bwd_kernel<T, INTERLEAVED, NORM, true>), grid, block, lds, s, p);
  else hipLaunchKernelGGL((norm_rotary_bwd_kernel<T, INTERLEAVED, NORM, false>), grid, block, lds, s, p);
}

template <typename T>
void launch_bwd(const NormRotaryParams& p, int interleaved, unsigned blocks, hipStream_t s) {
  const bool norm = p.t[1].w != nullptr;
  if (interleaved) {
    if (norm) launch_bwd_rows<T, true, true>(p, blocks, s);
    else launch_bwd_rows<T, true, false>(p, blocks, s);
  } else {
    if (norm) launch_bwd_rows<T, false, true>(p, blocks, s);
    else launch_bwd_rows<T, false, false>(p, blocks, s);
  }
}

}  // namespace

extern "C" int melgpt_qk_norm_rotary_fwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                         long long k_head, const int* positions, const double* freqs, int rot,
                                         int interleaved, float amplitude, const float* q_weight, const float* k_weight,
                                         float eps, void* q_out, void* k_out, long long M, int Hq, int Hk, int D, int dtype,
                                         void* stream) {
  NormRotaryParams p = {};
  p.t[0].x = q; p.t[0].row = q_row; p.t[0].head = q_head; p.t[0].w = q_weight; p.t[0].out = q_out; p.t[0].H = Hq;
  p.t[1].x = k; p.t[1].row = k_row; p.t[1].head = k_head; p.t[1].w = k_weight; p.t[1].out = k_out; p.t[1].H = Hk;
  p.pos = positions; p.freqs = freqs; p.rot = rot; p.amplitude = amplitude; p.eps = eps; p.M = M; p.D = D;
  if (M == 0) return MELGPT_OK;
  int e = check_common(p, dtype);
  if (e) return e;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  for (int i = 0; i < 2; ++i) {
    if ((e = check_tensor(p.t[i], vec))) return e;
    if (!p.t[i].out) return MELGPT_ERR_BAD_ARG;
    if (!aligned16(p.t[i].out)) return MELGPT_ERR_ALIGN;
  }
  plan(p, dtype, 0);
  if (dtype == MELGPT_F32) launch_fwd<float, false>(p, interleaved, (hipStream_t)stream);
  else launch_fwd<bf16_t, false>(p, interleaved, (hipStream_t)stream);
  return melgpt_launch_status();
}

extern "C" int melgpt_qk_norm_rotary_bwd_blocks(long long M) {
  const long long b = (M + 3) / 4;
  return (int)(b < 1 ? 1 : b < 1024 ? b : 1024);
}

extern "C" int melgpt_qk_norm_rotary_bwd(const void* dq_out, long long dq_row, long long dq_head, const void* dk_out,
                                         long long dk_row, long long dk_head, const void* q, long long q_row, long long q_head,
                                         const void* k, long long k_row, long long k_head, const int* positions,
                                         const double* freqs, int rot, int interleaved, float amplitude, const float* q_weight,
                                         const float* k_weight, float eps, void* dq, void* dk, float* dw_partials, long long M,
                                         int Hq, int Hk, int D, int dtype, void* stream) {
  NormRotaryParams p = {};
  p.t[0].dy = dq_out; p.t[0].dy_row = dq_row; p.t[0].dy_head = dq_head; p.t[0].x = q; p.t[0].row = q_row; p.t[0].head = q_head;
  p.t[0].w = q_weight; p.t[0].out = dq; p.t[0].H = Hq;
  p.t[1].dy = dk_out; p.t[1].dy_row = dk_row; p.t[1].dy_head = dk_head; p.t[1].x = k; p.t[1].row = k_row; p.t[1].head = k_head;
  p.t[1].w = k_weight; p.t[1].out = dk; p.t[1].H = Hk;
  p.pos = positions; p.freqs = freqs; p.rot = rot; p.amplitude = amplitude; p.eps = eps; p.M = M; p.D = D; p.dw_part = dw_partials;
  if (M == 0) return MELGPT_OK;
  int e = check_common(p, dtype);
  if (e) return e;
  const bool norm = q_weight != nullptr;
  if (norm && !dw_partials) return MELGPT_ERR_BAD_ARG;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  for (int i = 0; i < 2; ++i) {
    if (norm && (e = check_tensor(p.t[i], vec))) return e;
    if (!p.t[i].dy || !p.t[i].out || p.t[i].H <= 0) return MELGPT_ERR_BAD_ARG;
    if (!aligned16(p.t[i].dy) || !aligned16(p.t[i].out) || p.t[i].dy_row % vec || p.t[i].dy_head % vec) return MELGPT_ERR_ALIGN;
  }
  plan(p, dtype, 0);
  p.hsplit = 1;   // (the number of workgroups is the caller's number of partial rows)
  const unsigned blocks = (unsigned)melgpt_qk_norm_rotary_bwd_blocks(M);
  if (dtype == MELGPT_F32) launch_bwd<float>(p, interleaved, blocks, (hipStream_t)stream);
  else launch_bwd<bf16_t>(p, interleaved, blocks, (hipStream_t)stream);
  return melgpt_launch_status();
}

extern "C" int melgpt_kv_append(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                long long k_head, const void* v, long long v_row, long long v_head, const int* sequences,
                                const int* positions, const int* page_table, long long table_ld, int S, int width,
                                const double* freqs, int rot, int interleaved, float amplitude, const float* q_weight,
                                const float* k_weight, float eps, void* q_out, int zero_pad, void* k_pages, void* v_pages,
                                long long n_pages, int page_size, long long M, int Hq, int Hk, int D, int dtype, void* stream) {
  NormRotaryParams p = {};
  p.t[0].x = q; p.t[0].row = q_row; p.t[0].head = q_head; p.t[0].w = q_weight; p.t[0].out = q_out; p.t[0].H = Hq;
  p.t[1].x = k; p.t[1].row = k_row; p.t[1].head = k_head; p.t[1].w = k_weight; p.t[1].H = Hk;
  p.v = v; p.v_row = v_row; p.v_head = v_head;
  p.pos = positions; p.freqs = freqs; p.rot = rot; p.amplitude = amplitude; p.eps = eps; p.M = M; p.D = D;
  p.seq = sequences; p.table = page_table; p.table_ld = table_ld; p.S = S; p.width = width; p.zero_pad = zero_pad;
  p.k_pages = k_pages; p.v_pages = v_pages;
  if (M == 0) return MELGPT_OK;
  if (page_size <= 0 || (page_size & (page_size - 1)) || page_size > (1 << 20) || n_pages > 0x7fffffffLL) return MELGPT_ERR_UNSUPPORTED;
  if (S <= 0 || width <= 0 || n_pages <= 0 || !sequences || !page_table || !k_pages || !v_pages || !v) return MELGPT_ERR_BAD_ARG;
  p.pages = (int)n_pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  // without queries their side has no heads and no steps (its weights, when given, are the keys' norm's other half)
  if (!q) {
    p.t[0].H = 0;
    p.t[0].w = p.t[1].w;
  }
  int e = check_common(p, dtype);
  if (e) return e;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  if (q) {
    if ((e = check_tensor(p.t[0], vec))) return e;
    if (!q_out) return MELGPT_ERR_BAD_ARG;
    if (!aligned16(q_out)) return MELGPT_ERR_ALIGN;
  }
  if ((e = check_tensor(p.t[1], vec))) return e;
  if (!aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) || v_row % vec || v_head % vec) return MELGPT_ERR_ALIGN;
  plan(p, dtype, 1);
  if (dtype == MELGPT_F32) launch_fwd<float, true>(p, interleaved, (hipStream_t)stream);
  else launch_fwd<bf16_t, true>(p, interleaved, (hipStream_t)stream);
  return melgpt_launch_status();
}
