// Causal attention with grouped heads over packed sequences of different lengths, forward and backward.
//
//   sequence s: queries rows cu_q[s] .. cu_q[s+1], keys rows cu_k[s] .. cu_k[s+1] (nq, nk of them); query i sees the keys
//   j <= i + nk - nq (the last query sees every key; with nq > nk the first nq - nk queries see none: output 0, lse -inf);
//   query head h reads key head h / G.
//   forward   s_ij = scale q_i . k_j,  lse_i = log sum_j e^s_ij,  o_i = sum_j e^(s_ij - lse_i) v_j
//   backward  p_ij = e^(s_ij - lse_i),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//             dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i,h ds_ij q_i,  dv_j = sum_i,h p_ij do_i  (h over the G heads)
//
// One pass over the keys with a running maximum and sum; scores, probabilities and their gradients live in registers only.
// The backward is two kernels - queries (dq, delta), then keys (dk, dv) - that each own their rows: no atomics, the same
// bits every time, at the price of forming the scores and do . v twice (7 products instead of 5).
//
// Row tiles of a sequence: nobody knows the lengths on the host, so sequence s is allotted tiles floor(cu[s] / B) + s up to
// floor(cu[s+1] / B) + s + 1 - never fewer than it needs, one too many at most - and a workgroup finds its sequence by a
// 64-way search over the offsets.  The rows in front of the first and behind the last sequence are two sequences without keys.
#include <type_traits>

#include "mma.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct PackedParams {
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  void* o;                       // forward out / backward in
  void* low;                     // optional, 16-bit: what rounding took from o, (Mq, Hq, D) contiguous
  long long o_row, o_head;
  const void* dout;
  long long do_row, do_head;
  void *dq, *dk, *dv;
  long long dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
  float *lse, *delta;            // (Hq, Mq)
  const int *cu_q, *cu_k;        // (S + 1)
  int splits;                    // 16-bit: workgroups that share a row tile's keys (forward) or a key tile's query heads (backward)
  int usual;                     // a forward with a pool: shares of the sequences that are not long
  unsigned by_usual, by_splits;  // 2^31 over usual and splits, rounded up
  float* part;                   // splits > 1: (splits, Hq, Mq, D) sums of e^(s - m) v, then (splits, Hq, Mq, 2): m (base 2), sums;
                                 // backward: (splits, [dk, dv], Mk, Hk, D)
  int S, Hq, Hk, G, write_gaps;  // write_gaps: zero the rows no sequence owns (2: those of lse and low, not of o)
  long long Mq, Mk;
  float scale;
};

// ---------------------------------------------------------------------------------------------- which rows are mine
// Boundaries of the S + 2 row ranges over M rows: [0, cu[0]), the sequences, [cu[S], M).  Out-of-range offsets are clamped.
__device__ __forceinline__ int bound_at(const int* cu, int S, long long M, int i) {
  if (i <= 0) return 0;
  if (i > S + 1) return (int)M;
  const int b = cu[i - 1];
  return b < 0 ? 0 : b > (int)M ? (int)M : b;
}
struct Rows {
  int seq;       // -1 or S: a gap, no keys
  int lo, n;     // its first row and their number
  int tile, tiles;
  bool any;
};
// tile number t (of rows of `B`) -> its range and the tile within it; with LAST the last tile of a range comes first: the
// tiles with the most causal partners (queries: the last, keys: the first) start first
template <int B, bool LAST>
__device__ __forceinline__ Rows find_rows(const int* cu, int S, long long M, int t, int lane) {
  // the largest range i of 0 .. S + 1 with bound(i) / B + i <= t, 64 candidates at a time (the lanes of every wave)
  int lo = 0, n = S + 2;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lo + lane * step;
    const bool yes = lane * step < n && bound_at(cu, S, M, i) / B + i <= t;
    const unsigned long long m = __ballot(yes);
    const int c = m ? 63 - __builtin_clzll(m) : 0;   // (offsets that do not rise leave holes; any candidate stays in range)
    lo += c * step;
    n = min(step, n - c * step);
  }
  Rows r;
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int a = bound_at(cu, S, M, lo), b = max(bound_at(cu, S, M, lo + 1), a);
  r.seq = lo - 1;
  r.lo = a;
  r.n = b - a;
  r.tiles = (r.n + B - 1) / B;
  const int at = t - (a / B + lo);
  r.any = at >= 0 && at < r.tiles;
  r.tile = LAST ? r.tiles - 1 - at : at;
  return r;
}
// rows of the other side of sequence seq
__device__ __forceinline__ void other_rows(const int* cu, int S, long long M, int seq, int& lo, int& n) {
  if (seq < 0 || seq >= S) {
    lo = 0;
    n = 0;
    return;
  }
  lo = bound_at(cu, S, M, seq + 1);
  n = max(bound_at(cu, S, M, seq + 2) - lo, 0);
}
long long tiles_for(long long M, int S, int B) { return M / B + S + 2; }

// workgroup -> (tile, query head): consecutive workgroups go to consecutive XCDs, so with the key head fastest the
// workgroups that read one key head's rows share an XCD's L2 when the key heads are a multiple of 8
__device__ __forceinline__ void head_of(int w, const PackedParams& p, int& h) {
  const int kv = w % p.Hk, g = w / p.Hk;
  h = kv * p.G + g;
}

// ---------------------------------------------------------------------------------------------- tiles in LDS, f32 lane
// R rows of D values, 16-byte chunks xor-swizzled by the row so that neither row reads (16 rows, one chunk) nor reads along
// columns pile up on banks.
template <int D>
struct Tile {
  static constexpr int RB = 4 * D, CP = RB / 16;
  static constexpr int NKS = CP / 4;           // fragments along D
  static constexpr int DT = D / 16;            // 16-column tiles
  static __device__ __forceinline__ int off(int row, int c) { return row * RB + ((c ^ (row & 15)) << 4); }
  // fragment of 16 rows (16 tile16 + (lane & 15)), contraction along D
  static __device__ __forceinline__ u32x4 rows(const char* t, int tile16, int ks, int lane) {
    return *(const u32x4*)(t + off(16 * tile16 + (lane & 15), 4 * ks + (lane >> 4)));
  }
  // fragment of 16 columns (16 dt + (lane & 15)), contraction along rows 16 st .. + 15 (slot e: row 16 st + 4 g + e) - the
  // order in which the accumulators of the score products hold them, so those are the other operand as they stand
  static __device__ __forceinline__ u32x4 cols(const char* t, int st, int dt, int lane) {
    const int g = lane >> 4, col = 16 * dt + (lane & 15);
    u32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = *(const unsigned*)(t + off(16 * st + 4 * g + e, col >> 2) + (col & 3) * 4);
    return f;
  }
};

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
  if constexpr (Tr<T>::ES == 2) *(u32x2*)p = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  else *(f32x4*)p = v;
}
__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// ---- values that are not finite, at keys that only some queries of a workgroup see.  A masked probability is 0, but
// 0 * NaN is not: in tiles that the causal border cuts such values are stored as zeros, and what they add to the queries that
// do see them is added at the end, key by key, outside the matrix instructions.
template <typename T>
__device__ __forceinline__ bool finite_bits(unsigned v) {   // of an f32, or of both of two 16-bit values
  if constexpr (sizeof(T) == 4) return (v & 0x7f800000u) != 0x7f800000u;
#ifdef MELGPT_HALF_FP16
  else return (((v & 0x7c007c00u) + 0x04000400u) & 0x80008000u) == 0u;
#else
  else return (((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u) == 0u;
#endif
}
template <typename T>
__device__ __forceinline__ bool finite16(u32x4 v) {
  return finite_bits<T>(v[0]) && finite_bits<T>(v[1]) && finite_bits<T>(v[2]) && finite_bits<T>(v[3]);
}
// zeros in place of the values that are not finite
template <typename T>
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      if (!finite_bits<T>(v[e])) v[e] = 0u;
    } else {
      if (!finite_bits<T>(v[e] & 0xffffu)) v[e] &= 0xffff0000u;
      if (!finite_bits<T>(v[e] & 0xffff0000u)) v[e] &= 0xffffu;
    }
  }
  return v;
}
template <typename T>
__device__ __forceinline__ float value_of(const T* p) { return Elem<T>::ld(p); }
// adds the contributions of such values at keys k0 .. k1 - 1 to this lane's query (which sees keys below `sees`; running
// maximum m, base 2): get(i) / add(i, x) for the lane's n accumulators of value column col(i)
template <typename T, int D, int N, typename Col, typename Add>
__device__ __forceinline__ void add_not_finite(const T* q, const T* k, long long k_row, const T* v, long long v_row, int k0, int k1,
                                               int sees, float scale2, float m, int lane, Col col, Add add) {
  const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll 1
  for (int j = k0; j < k1; ++j) {
    bool fine = true;
    for (int d = lane; d < D; d += 64) {
      const float x = value_of(v + j * v_row + d);
      fine = fine && __builtin_isfinite(x);
    }
    if (__all(fine)) continue;
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; ++d) s = fmaf(value_of(q + d), value_of(k + j * k_row + d), s);
    const float pr = __builtin_amdgcn_exp2f(fmaf(s, scale2, -base));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = value_of(v + j * v_row + col(i));
      if (j < sees && !__builtin_isfinite(x)) add(i, pr * x);
    }
  }
}

// 32 rows of two tensors on their way into LDS: the loads of the next pair are in flight under the current pair's products.
// Rows at and beyond n are zero (their products are masked, but 0 * NaN is not 0).
template <int D>
struct Stage {
  using T = float;
  using L = Tile<D>;
  static constexpr int PER = 32 * L::CP / 256;   // chunks per thread
  u32x4 a[PER], b[PER];
  __device__ __forceinline__ void load(const T* pa, long long ra, const T* pb, long long rb, int row0, int n, int t) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = t + 256 * i, row = min(row0 + q / L::CP, n - 1), c = q % L::CP;
      a[i] = *(const u32x4*)(pa + row * ra + c * 4);
      b[i] = *(const u32x4*)(pb + row * rb + c * 4);
    }
  }
  // -> whether tensor b had values that are not finite (it has zeros there now)
  __device__ __forceinline__ bool clean_b() {
    bool fine = true;
#pragma unroll
    for (int i = 0; i < PER; ++i) fine = fine && finite16<T>(b[i]);
    if (fine) return false;
#pragma unroll
    for (int i = 0; i < PER; ++i) b[i] = finite_part<T>(b[i]);
    return true;
  }
  __device__ __forceinline__ void store(char* ta, char* tb, int row0, int n, int t) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = t + 256 * i, row = q / L::CP, c = q % L::CP;
      const bool in = row0 + row < n;
      const u32x4 z = {0u, 0u, 0u, 0u};
      *(u32x4*)(ta + L::off(row, c)) = in ? a[i] : z;
      *(u32x4*)(tb + L::off(row, c)) = in ? b[i] : z;
    }
  }
};

// a tile of B rows that no sequence owns: the forward's zeros (256 threads)
template <typename T, int D, int B>
__device__ __forceinline__ void rows_of_nobody(const PackedParams& p, const Rows& R, int h, int z, int t) {
  if (!p.write_gaps || z) return;
  constexpr int VEC = 16 / sizeof(T), C = D / VEC;                 // 16-byte pieces of a row
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const int first = B * R.tile, n = min(R.n - first, B);
  for (int i = t; i < n * C; i += 256) {
    const long long row = R.lo + first + i / C;
    const int c = i % C;
    if (p.write_gaps == 1) *(u32x4*)((T*)p.o + row * p.o_row + h * p.o_head + c * VEC) = zero;
    if (p.low) *(u32x4*)((T*)p.low + (row * p.Hq + h) * D + c * VEC) = zero;
    if (c == 0) p.lse[h * p.Mq + row] = -__builtin_inff();
  }
}

// --------------------------------------------------------------------------------------------- forward, f32 lane
// 256 threads, 64 queries of one head: a wave owns 16 queries and walks the keys 32 at a time (16 heads of 64 at length 266:
// 18 us, the time of 80 workgroups' chains of 9 steps; at 4000 rows 75 - 80 TFLOP/s, of 154 in a large product).  S^T = K Q^T puts the query
// on the lane: its maximum and sum are in registers and two exchanges away, and the probabilities are the operand of
// O^T = V^T P^T as they stand.
template <int D>
__global__ __launch_bounds__(256) void packed_fwd_f32_kernel(PackedParams p) {
  using T = float;
  using L = Tile<D>;
  __shared__ __attribute__((aligned(16))) char lds[2][2][32 * L::RB];
  __shared__ int odd;                                              // a value that is not finite in a tile the causal border cuts
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4;
  int h;
  head_of(blockIdx.x, p, h);
  const Rows R = find_rows<64, true>(p.cu_q, p.S, p.Mq, blockIdx.y, lane);
  if (!R.any) return;
  if (R.seq < 0 || R.seq >= p.S) return rows_of_nobody<T, D, 64>(p, R, h, 0, t);
  int k_lo, nk;
  other_rows(p.cu_k, p.S, p.Mk, R.seq, k_lo, nk);
  const int q_in = 64 * R.tile + 16 * wave + (lane & 15);          // this lane's query within its sequence
  const bool mine = q_in < R.n;
  const long long row = R.lo + min(q_in, R.n - 1);
  const int sees = min(max(q_in + nk - R.n + 1, 0), nk);           // keys 0 .. sees - 1
  const int last = min(64 * R.tile + 63, R.n - 1);
  const int most = min(max(last + nk - R.n + 1, 0), nk);           // of any query of the workgroup
  const T* qp = (const T*)p.q + row * p.q_row + h * p.q_head;
  u32x4 qf[L::NKS];
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) qf[ks] = *(const u32x4*)(qp + (4 * ks + g) * 4);
  const T* kp = (const T*)p.k + (long long)k_lo * p.k_row + (h / p.G) * p.k_head;
  const T* vp = (const T*)p.v + (long long)k_lo * p.v_row + (h / p.G) * p.v_head;
  const float c2 = p.scale * LOG2E;
  f32x4 o[L::DT];
#pragma unroll
  for (int d = 0; d < L::DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;
  if (most > 0) {
    Stage<D> st;
    const int full = min(max(64 * R.tile + nk - R.n + 1, 0), nk);  // keys that every query of the workgroup sees
    if (t == 0) odd = 0;
    __syncthreads();
    st.load(kp, p.k_row, vp, p.v_row, 0, nk, t);
    if (32 > full && st.clean_b()) odd = 1;
    st.store(lds[0][0], lds[0][1], 0, nk, t);
    __syncthreads();
    for (int k0 = 0, buf = 0; k0 < most; k0 += 32, buf ^= 1) {
      const bool more = k0 + 32 < most;
      if (more) st.load(kp, p.k_row, vp, p.v_row, k0 + 32, nk, t);
      const char *kt = lds[buf][0], *vt = lds[buf][1];
      f32x4 s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) mma<T>(s[i], L::rows(kt, i, ks, lane), qf[ks]);
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[i][r] = k0 + 16 * i + 4 * g + r < sees ? s[i][r] * c2 : -__builtin_inff();
          top = fmaxf(top, s[i][r]);
        }
      top = fmaxf(across_groups_max(top), m);
      const float base = top == -__builtin_inff() ? 0.f : top;     // (no key seen yet: every term stays e^-inf = 0)
      const float keep = __builtin_amdgcn_exp2f(m - base);
      m = top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - base);
          sum += s[i][r];
        }
      l = l * keep + sum;
#pragma unroll
      for (int d = 0; d < L::DT; ++d) o[d] *= keep;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < L::DT; ++d) mma<T>(o[d], L::cols(vt, e, d, lane), __builtin_bit_cast(u32x4, s[e]));
      if (more && k0 + 64 > full && st.clean_b()) odd = 1;
      if (more) st.store(lds[buf ^ 1][0], lds[buf ^ 1][1], k0 + 32, nk, t);
      __syncthreads();
    }
    l = across_groups_sum(l);
    if (odd)
      add_not_finite<T, D, 4 * L::DT>(qp, kp, p.k_row, vp, p.v_row, full & ~31, most, sees, c2, m, lane,
                                      [&](int i) { return 16 * (i >> 2) + 4 * g + (i & 3); }, [&](int i, float x) { o[i >> 2][i & 3] += x; });
  }
  if (!mine) return;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;        // (NaN stays NaN)
  T* op = (T*)p.o + row * p.o_row + h * p.o_head;
#pragma unroll
  for (int d = 0; d < L::DT; ++d) store4<T>(op + 16 * d + 4 * g, o[d] * inv);
  if (g == 0) p.lse[h * p.Mq + row] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// ------------------------------------------------------------------------------------- forward, 16-bit operands
// 256 threads, 128 queries of one head: a wave owns 32 queries (v_mfma_f32_32x32x16: twice the queries per fragment read from
// LDS, which 16-row tiles are bound by) and walks the keys 64 at a time.  bf16, 32 heads over 8 of 128: eight prompts of up to
// 4097 in 295 us (879 TFLOP/s, of 1361 in a large matrix product), 1500 queries over 16001 keys in 383 us (978 TFLOP/s).  It is
// bound by matrix and vector instructions together: a step's 32 exponentials and 100 others need nearly the time of its 16
// products, and the clock sinks under both (on zeros the same instructions run 1.4 times as fast).
template <int D>
struct Tile32 {
  static constexpr int RB = 2 * D, CP = RB / 16, NKS = D / 16, DB = D / 32;
  // keys / rows read along D, 32 rows a time
  static __device__ __forceinline__ int swz_r(int row) { return RB == 128 ? (row >> 1) & 7 : row & 15; }
  // values, read transposed: 8 rows x 64 bytes an instruction, spread over all banks
  static __device__ __forceinline__ int swz_t(int row) {
    return RB == 128 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int off_r(int row, int c) { return row * RB + ((c ^ swz_r(row)) << 4); }
  static __device__ __forceinline__ int off_t(int row, int c) { return row * RB + ((c ^ swz_t(row)) << 4); }
  static __device__ __forceinline__ u32x4 rows(const char* t, int blk, int ks, int lane) {
    return *(const u32x4*)(t + off_r(32 * blk + (lane & 31), 2 * ks + (lane >> 5)));
  }
  static __device__ __forceinline__ u32x4 rows_t(const char* t, int blk, int ks, int lane) {   // of a tile laid out for transposed reads
    return *(const u32x4*)(t + off_t(32 * blk + (lane & 31), 2 * ks + (lane >> 5)));
  }
  // 32 columns of block db, contraction over 16 rows, step st: slot j of lane half hh is row 16 st + 8 (j >> 2) + 4 hh + (j & 3),
  // the order in which accumulators 8 (st & 1) .. + 7 of a 32-row score block hold them
  static __device__ __forceinline__ u32x4 cols(const char* t, int st, int db, int lane) {
    const int hh = lane >> 5, q4 = (lane & 15) >> 2, p4 = lane & 3, g1 = (lane >> 4) & 1;
    const int row = 16 * st + 4 * hh + q4, c = 4 * db + 2 * g1 + (p4 >> 1);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, t + off_t(row, c) + 8 * (p4 & 1)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, t + off_t(row + 8, c) + 8 * (p4 & 1)));
    const s16x8 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(u32x4, f);
  }
};
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// larger of a lane's value and that of the lane 32 away (NaN wins)
__device__ __forceinline__ float halves_max(float v) {
  const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// accumulators 8 st .. 8 st + 7 of a 32-row block as the operand of a 16-row contraction.  Probabilities and score gradients are
// rounded to 16 bits here, and only here: the second products want 16-bit operands (in f32 they would run at 154 TFLOP/s, not
// 1361), and independent roundings add no more than the result's own: of its norm, in bf16, the output is 0.0020 (prompts) to
// 0.0023 (long rows) off, 0.0017 with f32 probabilities, the gradients 0.0024.  Statistics and sums are taken before it.
__device__ __forceinline__ u32x4 operand16(const f32x16& s, int st) {
  return u32x4{pack_bf16x2(s[8 * st], s[8 * st + 1]), pack_bf16x2(s[8 * st + 2], s[8 * st + 3]),
               pack_bf16x2(s[8 * st + 4], s[8 * st + 5]), pack_bf16x2(s[8 * st + 6], s[8 * st + 7])};
}

// 64 rows straight from memory into LDS (NW waves), 1 KB an instruction: LDS takes 32 bytes a cycle from registers
// (ds_write_b128: 14 ns a KB on a CU, measured) but gives 240 - a tile's stores took longer than all its reads - and the
// registers of a tile in flight are free.  An instruction's lanes fill 1 KB of LDS in order, so the swizzle is applied to
// which chunk a lane fetches.  Rows behind the last are out of the buffer's range and arrive as zeros (their scores are
// masked, but 0 * NaN is not 0).  (asm: the compiler would hold every LDS read until the builtin's data had arrived; the
// counterpart is arrive() in front of the barrier.)
typedef u32x4 buffer_t;
__device__ __forceinline__ buffer_t make_buffer(const void* base, unsigned bytes) {
  const unsigned long long a = (unsigned long long)base;
  return buffer_t{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu),
                  (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
__device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <int D, bool TR, int NW = 4>   // TR: laid out for transposed reads
struct Fetch64 {
  using L = Tile32<D>;
  static constexpr int PER = L::CP / NW, STEP = 64 / PER;   // instructions of a wave, rows between them
  static_assert(STEP % 16 == 0, "a lane's rows share their swizzle");
  unsigned from, step;                                      // bytes: this lane's first chunk, its next
  int at;                                                   // the wave's place in a tile
  __device__ __forceinline__ Fetch64(long long rs, int wave, int lane) {
    const int row = (64 / L::CP) * wave + lane / L::CP, c = (lane % L::CP) ^ (TR ? L::swz_t(row) : L::swz_r(row));
    from = 2u * ((unsigned)row * (unsigned)rs + 8u * c);
    step = 2u * STEP * (unsigned)rs;
    at = 1024 * wave;
  }
  // rows row0 .. of n (row stride rs) -> tile
  __device__ __forceinline__ void operator()(char* tile, const bf16_t* base, long long rs, int row0, int n) const {
    const int left = min(max(n - row0, 0), 64);
    (*this)(tile, make_buffer(base + row0 * rs, left > 0 ? 2u * ((unsigned)(left - 1) * (unsigned)rs + D) : 0u));
  }
  __device__ __forceinline__ void operator()(char* tile, buffer_t b) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned m0 = (unsigned)(size_t)LDS_PTR(char, tile + at + 1024 * NW * i);
      asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(m0), "v"(from + i * step), "s"(b)
                   : "memory", "m0");
    }
  }
};
// zeros in place of values that are not finite in a tile in LDS (256 threads) -> whether this thread found any
template <int D>
__device__ __forceinline__ bool clean_tile(char* tile, int t) {
  bool found = false;
#pragma unroll
  for (int i = 0; i < 64 * Tile32<D>::RB / (256 * 16); ++i) {
    u32x4* c = (u32x4*)(tile + (t + 256 * i) * 16);
    const u32x4 v = *c;
    if (!finite16<bf16_t>(v)) {
      *c = finite_part<bf16_t>(v);
      found = true;
    }
  }
  return found;
}

// Shares of a row tile's `every` key tiles: `usual` of them (which a mean length decides), but of 16 tiles at most while there
// are `splits` for that, so that one long sequence among short ones is not walked alone.
constexpr unsigned POOLED = 512;
__device__ __forceinline__ int pool_share(const PackedParams& p, int every) {
  // (quotients rounded up, exact below 2^27 for divisors up to 16: two integer divisions are a tenth of a short share's time)
  const int even = (int)__umulhi((unsigned)(every + p.usual - 1) << 1, p.by_usual);
  const int least = (int)__umulhi((unsigned)(every + p.splits - 1) << 1, p.by_splits);
  return max(max(min(even, 16), least), 1);
}
// (With 16 splits or fewer a tile that sees more keys never has fewer shares, so a sequence's last tile tells how many.)
// Those beyond the usual ones are taken by a pool of workgroups, which find them from the lengths: number e, e + POOLED, .. of
// all in order of sequence, row tile (the last first), share and query head.  128 queries over 16000 keys among 63 single ones
// over 64, 8 heads of 128: 252 us without, 94 with; 32 heads 255 / 105, 16 of 64 201 / 65.  Where there is no long one the two
// launches more cost some 6 us (100 sequences of 2 queries over 300 keys, 8 heads of 64: 21 / 28; of 1 over 1000, 16: 99 / 106).
// All lanes of a wave.
// s0, e: where the search stands (number e of those from sequence s0 on); it goes on there for the next.
__device__ __forceinline__ bool any_pooled(const PackedParams& p, int lane) {
  bool any = false;                                                // (loads side by side; the search waits for each)
#pragma unroll 4
  for (int i = lane + 1; i <= p.S; i += 64) any = any || bound_at(p.cu_k, p.S, p.Mk, i + 1) - bound_at(p.cu_k, p.S, p.Mk, i) > 1024 * p.usual;
  return __any(any);
}
__device__ __forceinline__ bool find_pooled(const PackedParams& p, int& s0, unsigned& e, int lane, Rows& r, int& h, int& z) {
  for (; s0 < p.S; s0 += 64) {
    const int i = min(s0 + lane, p.S - 1) + 1;
    const int lo = bound_at(p.cu_q, p.S, p.Mq, i), nq = max(bound_at(p.cu_q, p.S, p.Mq, i + 1) - lo, 0);
    const int every = (bound_at(p.cu_k, p.S, p.Mk, i + 1) - bound_at(p.cu_k, p.S, p.Mk, i) + 63) >> 6;
    const int some = s0 + lane < p.S && every > 0 ? (nq + 127) >> 7 : 0;
    if (!__any(some > 0 && every > 16 * p.usual)) continue;
    const int per = pool_share(p, every), more = max((every + per - 1) / per - p.usual, 0);
    const unsigned mine = (unsigned)(some * more) * p.Hq;
    unsigned upto = mine;                                          // of this and the lanes before
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const unsigned before = __shfl_up(upto, d, 64);
      if (lane >= d) upto += before;
    }
    const unsigned all = __builtin_amdgcn_readlane(upto, 63);
    if (e < all) {
      const int at = __builtin_ctzll(__ballot(upto > e));
      const unsigned k = e - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at));
      const unsigned shares = __builtin_amdgcn_readlane(more, at), j = k / (unsigned)p.Hq;
      head_of((int)(k % (unsigned)p.Hq), p, h);
      r.seq = s0 + at;
      r.lo = __builtin_amdgcn_readlane(lo, at);
      r.n = __builtin_amdgcn_readlane(nq, at);
      r.tiles = (r.n + 127) >> 7;
      r.tile = r.tiles - 1 - (int)(j / shares);
      r.any = true;
      z = p.usual + (int)(j % shares);
      return true;
    }
    e -= all;
  }
  return false;
}

// one row tile's share z of its keys
template <int D, bool POOL>
__device__ __forceinline__ void fwd32_rows(const PackedParams& p, const Rows& R, int h, int z, char (&lds)[2][2][64 * Tile32<D>::RB],
                                           int& odd) {
  using L = Tile32<D>;
  using T = bf16_t;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5;
  if (R.seq < 0 || R.seq >= p.S) return rows_of_nobody<T, D, 128>(p, R, h, z, t);
  int k_lo, nk;
  other_rows(p.cu_k, p.S, p.Mk, R.seq, k_lo, nk);
  const int w0 = 128 * R.tile + 32 * wave;                     // the wave's first query
  const int last = min(128 * R.tile + 127, R.n - 1);
  const int most = min(max(last + nk - R.n + 1, 0), nk);
  const int full = min(max(w0 + nk - R.n + 1, 0), nk);             // keys that every query of the wave sees
  const int q_in = w0 + (lane & 31);
  const int sees = min(max(q_in + nk - R.n + 1, 0), nk);           // keys 0 .. sees - 1
  const long long row = R.lo + min(q_in, R.n - 1);
  const T* qp = (const T*)p.q + row * p.q_row + h * p.q_head;
  u32x4 qf[L::NKS];
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) qf[ks] = *(const u32x4*)(qp + 16 * ks + 8 * hh);
  // the maximum is taken over the unscaled products: a negative scale goes into the queries' signs, a zero one (every key
  // alike, and no 0 * inf at the masked ones) into zero queries
  if (p.scale <= 0.f) {
    const unsigned flip = p.scale < 0.f ? 0x80008000u : 0u, keep = p.scale < 0.f ? 0xffffffffu : 0u;
#pragma unroll
    for (int ks = 0; ks < L::NKS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[ks][e] = (qf[ks][e] ^ flip) & keep;
  }
  const T* kp = (const T*)p.k + (long long)k_lo * p.k_row + (h / p.G) * p.k_head;
  const T* vp = (const T*)p.v + (long long)k_lo * p.v_row + (h / p.G) * p.v_head;
  const float c2 = p.scale == 0.f ? 1.f : fabsf(p.scale) * LOG2E;
  f32x16 o[L::DB];
#pragma unroll
  for (int d = 0; d < L::DB; ++d) o[d] = zero16();
  float m = -__builtin_inff(), l[2] = {0.f, 0.f};                  // two partial sums: independent chains
  // this workgroup's share of the key tiles
  const int every = (most + 63) >> 6, per = POOL ? pool_share(p, every) : (every + p.splits - 1) / p.splits;
  const int i0 = per * z, tiles = min(every - i0, per), k_first = 64 * i0;   // (with out_low there is one share)
  if (POOL && z > 0 && tiles <= 0) return;                         // (the join knows as much)
  if (tiles > 0) {
    const Fetch64<D, false> fetch_k(p.k_row, wave, lane);
    const Fetch64<D, true> fetch_v(p.v_row, wave, lane);
    auto scores = [&](const char* kt, int half, f32x16& s) __attribute__((always_inline)) {
      s = zero16();
#pragma unroll
      for (int ks = 0; ks < L::NKS; ++ks) s = MELGPT_MFMA_32x32x16(L::rows(kt, half, ks, lane), qf[ks], s);
    };
    auto weigh = [&](const char* vt, int half, const u32x4 (&pp)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < L::DB; ++d) o[d] = MELGPT_MFMA_32x32x16(L::cols(vt, 2 * half + e, d, lane), pp[e], o[d]);
    };
    // one step of 32 keys from k0: their scores `s` become probabilities `pn` under this step's matrix products, which are
    // the next 32 keys' scores `sn` (from kt) and the previous 32 keys' probabilities `pp` times their values (from vt) -
    // nothing here waits for anything else of the same step
    auto step = [&](int k0, f32x16& s, f32x16& sn, const char* kt, int khalf, const u32x4 (&pp)[2], u32x4 (&pn)[2], const char* vt,
                    int vhalf) __attribute__((always_inline)) {
      if (k0 + 32 > full) {
        const int lim = sees - k0 - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) < lim ? s[r] : -__builtin_inff();
      }
      scores(kt, khalf, sn);
      weigh(vt, vhalf, pp);
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = __builtin_elementwise_maximum(top, s[r]);
      top = halves_max(top) * c2;
      // the running maximum follows only when it is passed by more than 2^8: until then terms up to 2^8 are exact enough in
      // f32 sums and 16-bit operands alike, and the accumulators need no rescaling (rare after the first tiles)
      const float now = top > m + 8.f ? top : m, base = now == -__builtin_inff() ? 0.f : now;
      const bool moved = now != m;
      const float keep = moved ? __builtin_amdgcn_exp2f(m - base) : 1.f;   // (no key yet: m is -inf and the sums are 0)
      m = now;
      l[0] *= keep;
      l[1] *= keep;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -base));
        l[r & 1] += s[r];
      }
      pn[0] = operand16(s, 0);
      pn[1] = operand16(s, 1);
      // (the exponentials belong under the products above: hipcc would sink them behind the branch)
      asm volatile("" : "+v"(pn[0]), "+v"(pn[1]), "+v"(l[0]), "+v"(l[1]));
      // order: fragments ahead, then a matrix instruction, a later fragment, and its share of the softmax; hipcc alone puts
      // all of the softmax behind the products and waits for every fragment
      __builtin_amdgcn_sched_group_barrier(0x100, 5, 0);
#pragma unroll
      for (int j = 0; j < L::NKS; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
        if (j > 2) __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
      }
#pragma unroll
      for (int j = 0; j < 2 * L::DB; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
      }
      if (__any(moved)) {
#pragma unroll
        for (int d = 0; d < L::DB; ++d) o[d] *= keep;
      }
    };
    // K runs one tile ahead of V in LDS: [0] K, [1] V, two slots each, tile i in slot i & 1.  Iteration i's fetches go to
    // slots last read before its barrier and are waited for in front of the next.
    const int all = min(max(128 * R.tile + nk - R.n + 1, 0), nk);  // keys that every query of the workgroup sees
    if (t == 0) odd = 0;
    fetch_k(lds[0][0], kp, p.k_row, k_first, nk);
    fetch_k(lds[0][1], kp, p.k_row, k_first + 64, nk);
    fetch_v(lds[1][0], vp, p.v_row, k_first, nk);
#pragma unroll
    for (int i = 0; i < 64 * L::RB / (256 * 16); ++i) *(u32x4*)(lds[1][1] + (t + 256 * i) * 16) = u32x4{0u, 0u, 0u, 0u};
    arrive();
    __syncthreads();
    f32x16 s0, s1;
    u32x4 p0[2], p1[2] = {u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}};
    scores(lds[0][0], 0, s0);
    // What rounding to operands took from a sequence's first 64 probabilities, where the backward will ask (out_low): its
    // delta = do . o inherits the error of o, which against ds is as large as a rounding of ds itself for rows of few keys
    // (gradients of sequences of 4: 0.0026 of their norm, 0.0024 with this; 0.0017 is the rounding of the results) and small
    // for long ones.
    auto add_lost = [&](const f32x16& s, const u32x4 (&pn)[2], const char* vt, int half) __attribute__((always_inline)) {
      f32x16 lost;
#pragma unroll
      for (int r = 0; r < 16; ++r) lost[r] = s[r] - (r & 1 ? half_hi(pn[r >> 3][(r & 7) >> 1]) : half_lo(pn[r >> 3][(r & 7) >> 1]));
      const u32x4 pl[2] = {operand16(lost, 0), operand16(lost, 1)};
      weigh(vt, half, pl);
    };
    auto tile = [&](int i, auto par, auto first) __attribute__((always_inline)) {   // par = i & 1, known to the compiler: LDS addresses are constants
      constexpr int P = decltype(par)::value;
      constexpr bool FIRST = decltype(first)::value;
      step(k_first + 64 * i, s0, s1, lds[0][P], 1, p1, p0, lds[1][P ^ 1], 1);
      arrive();
      __syncthreads();
      fetch_k(lds[0][P], kp, p.k_row, k_first + 64 * i + 128, nk);   // (behind the last tile: zeros, never used)
      fetch_v(lds[1][P ^ 1], vp, p.v_row, k_first + 64 * i + 64, nk);
      if (k_first + 64 * i + 64 > all) {
        if (clean_tile<D>(lds[1][P], t)) odd = 1;
        __syncthreads();
      }
      if (FIRST && p.low) add_lost(s0, p0, lds[1][P], 0);
      step(k_first + 64 * i + 32, s1, s0, lds[0][P ^ 1], 0, p0, p1, lds[1][P], 0);
      if (FIRST && p.low) add_lost(s1, p1, lds[1][P], 1);
    };
    tile(0, std::integral_constant<int, 0>(), std::true_type());
    int i = 1;
    for (; i + 1 < tiles; i += 2) {
      tile(i, std::integral_constant<int, 1>(), std::false_type());
      tile(i + 1, std::integral_constant<int, 0>(), std::false_type());
    }
    if (i < tiles) tile(i, std::integral_constant<int, 1>(), std::false_type());
    weigh(lds[1][(tiles - 1) & 1], 1, p1);
    arrive();                                                      // (nothing lands in LDS that is not this workgroup's any more)
    if (odd)
      add_not_finite<T, D, 16 * L::DB>(qp, kp, p.k_row, vp, p.v_row, max(all & ~63, k_first), min(most, k_first + 64 * tiles), sees, p.scale * LOG2E, m, lane,
                                       [&](int i) { return 32 * (i >> 4) + 8 * ((i & 15) >> 2) + 4 * hh + (i & 3); },
                                       [&](int i, float x) { o[i >> 4][i & 15] += x; });
  }
  float sum = l[0] + l[1];
  sum += __shfl_xor(sum, 32, 64);
  if (q_in >= R.n) return;
  if (POOL ? per < every : p.splits > 1) {
    const long long at = ((long long)z * p.Hq + h) * p.Mq + row;
#pragma unroll
    for (int d = 0; d < L::DB; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(f32x4*)(p.part + at * D + 32 * d + 8 * j + 4 * hh) = f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
    if (hh == 0) *(f32x2*)(p.part + (long long)p.splits * p.Hq * p.Mq * D + 2 * at) = f32x2{m, sum};
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* op = (T*)p.o + row * p.o_row + h * p.o_head;
  // low: the backward's delta = do . o loses a rounding of o against ds' own size; with both halves it does not.  It is taken
  // from the bits that are stored: rounded a second time by itself, hipcc fuses the product into the conversion of the half
  // flavour (one rounding instead of two), and at a tie the two halves would not fit each other.
  auto put = [&](auto low) __attribute__((always_inline)) {
    T* lp = (T*)p.low + (row * p.Hq + h) * D;
#pragma unroll
    for (int d = 0; d < L::DB; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * d + 8 * j + 4 * hh;
        const f32x4 x = f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]} * inv;
        const u32x2 w = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
        *(u32x2*)(op + at) = w;
        if (decltype(low)::value) store4<T>(lp + at, x - f32x4{half_lo(w[0]), half_hi(w[0]), half_lo(w[1]), half_hi(w[1])});
      }
  };
  if (p.low) put(std::true_type());
  else put(std::false_type());
  if (hh == 0) p.lse[h * p.Mq + row] = sum == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * LN2;
}

template <int D, bool POOL>
__global__ __launch_bounds__(256, 2) void packed_fwd32_kernel(PackedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[2][2][64 * Tile32<D>::RB];
  __shared__ int odd;                                              // a value that is not finite in a tile the causal border cuts
  int h;
  head_of(blockIdx.x, p, h);
  const Rows R = find_rows<128, true>(p.cu_q, p.S, p.Mq, blockIdx.y, threadIdx.x & 63);
  if (R.any) fwd32_rows<D, POOL>(p, R, h, blockIdx.z, lds, odd);
}

// the pool (a launch in front: among the others it would take registers from them, and a wave of three at head size 64)
template <int D>
__global__ __launch_bounds__(256, 2) void packed_fwd32_pool_kernel(PackedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[2][2][64 * Tile32<D>::RB];
  __shared__ int odd;
  const int lane = threadIdx.x & 63;
  if (!any_pooled(p, lane)) return;
  auto at = __builtin_amdgcn_kernarg_segment_ptr();
  int s0 = 0;
  for (unsigned e = blockIdx.x;; e += POOLED) {
    asm volatile("" : "+s"(at));   // (arguments are read anew each time: kept over the loop they spill)
    PackedParams a;
    __builtin_memcpy(&a, (const void*)at, sizeof(a));
    Rows R;
    int h, z;
    if (!find_pooled(a, s0, e, lane, R, h, z)) return;
    fwd32_rows<D, true>(a, R, h, z, lds, odd);
    __syncthreads();                                               // (all waves are done with the tiles)
  }
}

// shares that the row tile of a query has behind a pool: a wave looks for its 64 / (D / 4) queries' sequences one after another
template <int D>
__device__ __forceinline__ int pooled_shares(const PackedParams& p, long long row, int lane) {
  constexpr int TPQ = D / 4;
  int shares = 0;
#pragma unroll
  for (int i = 0; i < 64 / TPQ; ++i) {
    const int r = __builtin_amdgcn_readlane((int)row, i * TPQ);
    int lo = 0, n = p.S + 2;                                       // the last range that begins at or before the row
    while (n > 1) {
      const int step = (n + 63) / 64;
      const unsigned long long m = __ballot(lane * step < n && bound_at(p.cu_q, p.S, p.Mq, lo + lane * step) <= r);
      const int c = m ? 63 - __builtin_clzll(m) : 0;
      lo += c * step;
      n = min(step, n - c * step);
    }
    const int first = bound_at(p.cu_q, p.S, p.Mq, lo), nq = bound_at(p.cu_q, p.S, p.Mq, lo + 1) - first;
    int k_lo, nk;
    other_rows(p.cu_k, p.S, p.Mk, lo - 1, k_lo, nk);
    const int last = min((r - first) | 127, nq - 1), every = (min(max(last + nk - nq + 1, 0), nk) + 63) >> 6;
    const int per = pool_share(p, every), mine = (every + per - 1) / per;
    if (lane / TPQ == i) shares = mine;
  }
  return shares;
}

// joins the splits of a query in their order: D / 4 lanes, four values each
template <int D, bool POOL>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedParams p) {
  using T = bf16_t;
  constexpr int TPQ = D / 4;
  const long long all = (long long)p.Hq * p.Mq, mine = (long long)blockIdx.x * (256 / TPQ) + threadIdx.x / TPQ, n = min(mine, all - 1);
  const int d = 4 * (threadIdx.x % TPQ), h = (int)(n / p.Mq);
  const long long row = n % p.Mq;
  const bool gap = row < bound_at(p.cu_q, p.S, p.Mq, 1) || row >= bound_at(p.cu_q, p.S, p.Mq, p.S + 1);
  const int shares = POOL ? pooled_shares<D>(p, row, threadIdx.x & 63) : p.splits;
  if (mine >= all || gap || (POOL && shares <= 1)) return;         // (written by the forward itself)
  const float* st = p.part + (long long)p.splits * all * D + 2 * n;
  float top = -__builtin_inff();
  for (int i = 0; i < shares; ++i) top = fmaxf(top, st[2 * i * all]);
  const float base = top == -__builtin_inff() ? 0.f : top;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < shares; ++i) {
    const float f = __builtin_amdgcn_exp2f(st[2 * i * all] - base);
    a += *(const f32x4*)(p.part + (i * all + n) * D + d) * f;
    sum += st[2 * i * all + 1] * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store4<T>((T*)p.o + row * p.o_row + h * p.o_head + d, a * inv);
  if (d == 0) p.lse[n] = sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// --------------------------------------------------------------------------------------------- backward, f32 lane
// dq and delta: the forward's walk with a second score product, do . v, on the same tiles
template <int D>
__global__ __launch_bounds__(256) void packed_dq_f32_kernel(PackedParams p) {
  using T = float;
  using L = Tile<D>;
  __shared__ __attribute__((aligned(16))) char lds[2][2][32 * L::RB];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4;
  int h;
  head_of(blockIdx.x, p, h);
  const Rows R = find_rows<64, true>(p.cu_q, p.S, p.Mq, blockIdx.y, lane);
  if (!R.any) return;
  int k_lo, nk;
  other_rows(p.cu_k, p.S, p.Mk, R.seq, k_lo, nk);
  if ((R.seq < 0 || R.seq >= p.S) && !p.write_gaps) return;
  const int q_in = 64 * R.tile + 16 * wave + (lane & 15);
  const bool mine = q_in < R.n;
  const long long row = R.lo + min(q_in, R.n - 1);
  const int sees = min(max(q_in + nk - R.n + 1, 0), nk);
  const int last = min(64 * R.tile + 63, R.n - 1);
  const int most = min(max(last + nk - R.n + 1, 0), nk);
  const T* qp = (const T*)p.q + row * p.q_row + h * p.q_head;
  const T* gp = (const T*)p.dout + row * p.do_row + h * p.do_head;
  const T* op = (const T*)p.o + row * p.o_row + h * p.o_head;
  u32x4 qf[L::NKS], gf[L::NKS];
  float dl = 0.f;
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) {
    qf[ks] = *(const u32x4*)(qp + (4 * ks + g) * 4);
    gf[ks] = *(const u32x4*)(gp + (4 * ks + g) * 4);
    const u32x4 of = *(const u32x4*)(op + (4 * ks + g) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) dl = fmaf(__uint_as_float(gf[ks][e]), __uint_as_float(of[e]), dl);
  }
  dl = across_groups_sum(dl);
  if (mine && g == 0) p.delta[h * p.Mq + row] = dl;
  const float lse2 = p.lse[h * p.Mq + row] * LOG2E;
  const T* kp = (const T*)p.k + (long long)k_lo * p.k_row + (h / p.G) * p.k_head;
  const T* vp = (const T*)p.v + (long long)k_lo * p.v_row + (h / p.G) * p.v_head;
  const float c2 = p.scale * LOG2E;
  f32x4 dq[L::DT];
#pragma unroll
  for (int d = 0; d < L::DT; ++d) dq[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (most > 0) {
    Stage<D> st;
    st.load(kp, p.k_row, vp, p.v_row, 0, nk, t);
    st.store(lds[0][0], lds[0][1], 0, nk, t);
    __syncthreads();
    for (int k0 = 0, buf = 0; k0 < most; k0 += 32, buf ^= 1) {
      const bool more = k0 + 32 < most;
      if (more) st.load(kp, p.k_row, vp, p.v_row, k0 + 32, nk, t);
      const char *kt = lds[buf][0], *vt = lds[buf][1];
      f32x4 s[2], dp[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = dp[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) {
          mma<T>(s[i], L::rows(kt, i, ks, lane), qf[ks]);
          mma<T>(dp[i], L::rows(vt, i, ks, lane), gf[ks]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[i][r] = k0 + 16 * i + 4 * g + r < sees ? __builtin_amdgcn_exp2f(s[i][r] * c2 - lse2) * (dp[i][r] - dl) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < L::DT; ++d) mma<T>(dq[d], L::cols(kt, e, d, lane), __builtin_bit_cast(u32x4, s[e]));
      if (more) st.store(lds[buf ^ 1][0], lds[buf ^ 1][1], k0 + 32, nk, t);
      __syncthreads();
    }
  }
  if (!mine) return;
  T* out = (T*)p.dq + row * p.dq_row + h * p.dq_head;
#pragma unroll
  for (int d = 0; d < L::DT; ++d) store4<T>(out + 16 * d + 4 * g, dq[d] * p.scale);
}

// dk and dv: 64 keys of one key head, a wave owns 16 keys (in registers) and walks the queries of its G heads that see
// them, 32 at a time.  S = Q K^T puts the key on the lane; P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS.
template <int D>
__global__ __launch_bounds__(256) void packed_dkv_f32_kernel(PackedParams p) {
  using T = float;
  using L = Tile<D>;
  __shared__ __attribute__((aligned(16))) char lds[2][2][32 * L::RB];
  __shared__ float stat[2][2][32];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4;
  const int hk = blockIdx.x;
  const Rows R = find_rows<64, false>(p.cu_k, p.S, p.Mk, blockIdx.y, lane);
  if (!R.any) return;
  int q_lo, nq;
  other_rows(p.cu_q, p.S, p.Mq, R.seq, q_lo, nq);
  if ((R.seq < 0 || R.seq >= p.S) && !p.write_gaps) return;
  const int nk = R.n;
  const int k_in = 64 * R.tile + 16 * wave + (lane & 15);
  const bool mine = k_in < nk;
  const long long row = R.lo + min(k_in, nk - 1);
  // query i sees key j <= i + nk - nq: the queries from j - (nk - nq) on
  const int from = max(k_in - (nk - nq), 0);
  const int first = max(64 * R.tile - (nk - nq), 0) & ~31;
  const T* kp = (const T*)p.k + row * p.k_row + hk * p.k_head;
  const T* vp = (const T*)p.v + row * p.v_row + hk * p.v_head;
  u32x4 kf[L::NKS], vf[L::NKS];
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) {
    kf[ks] = *(const u32x4*)(kp + (4 * ks + g) * 4);
    vf[ks] = *(const u32x4*)(vp + (4 * ks + g) * 4);
  }
  const float c2 = p.scale * LOG2E;
  f32x4 dk[L::DT], dv[L::DT];
#pragma unroll
  for (int d = 0; d < L::DT; ++d) dk[d] = dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int blocks = first < nq ? (nq - first + 31) / 32 : 0, total = blocks * p.G;
  if (total > 0) {
    Stage<D> st;
    float sv = 0.f;
    auto load = [&](int n) {
      const int h = hk * p.G + n / blocks, q0 = first + 32 * (n % blocks);
      st.load((const T*)p.q + (long long)q_lo * p.q_row + h * p.q_head, p.q_row,
              (const T*)p.dout + (long long)q_lo * p.do_row + h * p.do_head, p.do_row, q0, nq, t);
      if (t < 64) {
        const long long r = h * p.Mq + q_lo + min(q0 + (t & 31), nq - 1);
        sv = t < 32 ? p.lse[r] * LOG2E : p.delta[r];
      }
    };
    auto store = [&](int n, int buf) {
      st.store(lds[buf][0], lds[buf][1], first + 32 * (n % blocks), nq, t);
      if (t < 64) stat[buf][t >> 5][t & 31] = sv;
    };
    load(0);
    store(0, 0);
    __syncthreads();
    for (int n = 0, buf = 0; n < total; ++n, buf ^= 1) {
      if (n + 1 < total) load(n + 1);
      const int q0 = first + 32 * (n % blocks);
      const char *qt = lds[buf][0], *gt = lds[buf][1];
      f32x4 s[2], dp[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = dp[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) {
          mma<T>(s[i], L::rows(qt, i, ks, lane), kf[ks]);
          mma<T>(dp[i], L::rows(gt, i, ks, lane), vf[ks]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = 16 * i + 4 * g + r, q = q0 + at;
          const bool in = q >= from && q < nq;
          const float pr = in ? __builtin_amdgcn_exp2f(s[i][r] * c2 - stat[buf][0][at]) : 0.f;
          s[i][r] = pr;
          dp[i][r] = in ? pr * (dp[i][r] - stat[buf][1][at]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < L::DT; ++d) {
          mma<T>(dv[d], L::cols(gt, e, d, lane), __builtin_bit_cast(u32x4, s[e]));
          mma<T>(dk[d], L::cols(qt, e, d, lane), __builtin_bit_cast(u32x4, dp[e]));
        }
      if (n + 1 < total) store(n + 1, buf ^ 1);
      __syncthreads();
    }
  }
  if (!mine) return;
  T* ok = (T*)p.dk + row * p.dk_row + hk * p.dk_head;
  T* ov = (T*)p.dv + row * p.dv_row + hk * p.dv_head;
#pragma unroll
  for (int d = 0; d < L::DT; ++d) {
    store4<T>(ok + 16 * d + 4 * g, dk[d] * p.scale);
    store4<T>(ov + 16 * d + 4 * g, dv[d]);
  }
}

// ------------------------------------------------------------------------------------ backward, 16-bit operands
// dq and delta: a wave owns 32 queries, 64 keys a step; K lies in LDS in the order its transposed reads want (its row reads
// meet no bank twice in that order either).  Three products, 16 heads over 4 of 128 as below: 204 us, 770 TFLOP/s (uneven work here too:
// 67 key tiles on the longest of the 512 places, 53 evenly).
template <int D>
__global__ __launch_bounds__(256, 2) void packed_dq32_kernel(PackedParams p) {
  using L = Tile32<D>;
  using T = bf16_t;
  __shared__ __attribute__((aligned(16))) char lds[2][2][64 * L::RB];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5;
  int h;
  head_of(blockIdx.x, p, h);
  const Rows R = find_rows<128, true>(p.cu_q, p.S, p.Mq, blockIdx.y, lane);
  if (!R.any) return;
  int k_lo, nk;
  other_rows(p.cu_k, p.S, p.Mk, R.seq, k_lo, nk);
  if ((R.seq < 0 || R.seq >= p.S) && !p.write_gaps) return;
  const int w0 = 128 * R.tile + 32 * wave, q_in = w0 + (lane & 31);
  const int last = min(128 * R.tile + 127, R.n - 1);
  const int most = min(max(last + nk - R.n + 1, 0), nk);
  const int full = min(max(w0 + nk - R.n + 1, 0), nk), any = min(max(min(w0 + 31, R.n - 1) + nk - R.n + 1, 0), nk);
  const int sees = min(max(q_in + nk - R.n + 1, 0), nk);
  const long long row = R.lo + min(q_in, R.n - 1);
  const T* qp = (const T*)p.q + row * p.q_row + h * p.q_head;
  const T* gp = (const T*)p.dout + row * p.do_row + h * p.do_head;
  const T* op = (const T*)p.o + row * p.o_row + h * p.o_head;
  u32x4 qf[L::NKS], gf[L::NKS];
  float dl = 0.f;
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) {
    qf[ks] = *(const u32x4*)(qp + 16 * ks + 8 * hh);
    gf[ks] = *(const u32x4*)(gp + 16 * ks + 8 * hh);
    const u32x4 of = *(const u32x4*)(op + 16 * ks + 8 * hh);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dl = fmaf(half_lo(gf[ks][e]), half_lo(of[e]), dl);
      dl = fmaf(half_hi(gf[ks][e]), half_hi(of[e]), dl);
    }
    if (p.low) {
      const u32x4 lf = *(const u32x4*)((const T*)p.low + (row * p.Hq + h) * D + 16 * ks + 8 * hh);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dl = fmaf(half_lo(gf[ks][e]), half_lo(lf[e]), dl);
        dl = fmaf(half_hi(gf[ks][e]), half_hi(lf[e]), dl);
      }
    }
  }
  dl += __shfl_xor(dl, 32, 64);
  if (q_in < R.n && hh == 0) p.delta[h * p.Mq + row] = dl;
  const float lse2 = p.lse[h * p.Mq + row] * LOG2E, c2 = p.scale * LOG2E;
  const T* kp = (const T*)p.k + (long long)k_lo * p.k_row + (h / p.G) * p.k_head;
  const T* vp = (const T*)p.v + (long long)k_lo * p.v_row + (h / p.G) * p.v_head;
  f32x16 dq[L::DB];
#pragma unroll
  for (int d = 0; d < L::DB; ++d) dq[d] = zero16();
  if (most > 0) {
    const Fetch64<D, true> fetch_k(p.k_row, wave, lane), fetch_v(p.v_row, wave, lane);
    fetch_k(lds[0][0], kp, p.k_row, 0, nk);
    fetch_v(lds[0][1], vp, p.v_row, 0, nk);
    arrive();
    __syncthreads();
    // laid out by hand: with each matrix instruction goes the read of the fragment five later (hipcc reads it right in front
    // of the product that waits for it); the first of K^T are in flight under the probabilities
    constexpr int NP = 2 * L::NKS, NM = NP + 2 * L::DB, AHEAD = 5;
    auto half = [&](int k0, const char* kt, const char* vt, int i) __attribute__((always_inline)) {
      auto fragment = [&](int x) __attribute__((always_inline)) -> u32x4 {
        if (x < NP) return L::rows_t(x & 1 ? vt : kt, i, x >> 1, lane);
        return L::cols(kt, 2 * i + (x - NP) / L::DB, (x - NP) % L::DB, lane);
      };
      u32x4 f[NM];
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) f[x] = fragment(x);
      f32x16 s = zero16(), dp = zero16();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        if (x + AHEAD < NM) f[x + AHEAD] = fragment(x + AHEAD);
        if (x & 1) dp = MELGPT_MFMA_32x32x16(f[x], gf[x >> 1], dp);
        else s = MELGPT_MFMA_32x32x16(f[x], qf[x >> 1], s);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lse2)) * (dp[r] - dl);
      if (k0 + 32 * i + 32 > full) {
        const int lim = sees - k0 - 32 * i - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) < lim ? s[r] : 0.f;
      }
      const u32x4 sf[2] = {operand16(s, 0), operand16(s, 1)};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = NP; x < NM; ++x) {
        if (x + AHEAD < NM) f[x + AHEAD] = fragment(x + AHEAD);
        dq[(x - NP) % L::DB] = MELGPT_MFMA_32x32x16(f[x], sf[(x - NP) / L::DB], dq[(x - NP) % L::DB]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto tile = [&](int k0, auto par) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      const bool more = k0 + 64 < most;
      if (more) {
        fetch_k(lds[P ^ 1][0], kp, p.k_row, k0 + 64, nk);
        fetch_v(lds[P ^ 1][1], vp, p.v_row, k0 + 64, nk);
      }
      if (k0 < any) {
        half(k0, lds[P][0], lds[P][1], 0);
        half(k0, lds[P][0], lds[P][1], 1);
      }
      arrive();
      __syncthreads();
    };
    for (int k0 = 0; k0 < most; k0 += 128) {
      tile(k0, std::integral_constant<int, 0>());
      if (k0 + 64 < most) tile(k0 + 64, std::integral_constant<int, 1>());
    }
  }
  if (q_in >= R.n) return;
  T* out = (T*)p.dq + row * p.dq_row + h * p.dq_head;
#pragma unroll
  for (int d = 0; d < L::DB; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      store4<T>(out + 32 * d + 8 * j + 4 * hh, f32x4{dq[d][4 * j], dq[d][4 * j + 1], dq[d][4 * j + 2], dq[d][4 * j + 3]} * p.scale);
}

// dk and dv: 64 keys of one key head, 512 threads.  Pair (kb, qh) of waves owns keys 32 kb .. + 31, in registers, and of each
// 64 queries that see them, of each of the G heads, the 32 of half qh.  The two waves of a pair, on one SIMD, share a block's
// work so that each holds only one gradient (64 + 32 registers at 128 values a head instead of 128 + 64: two waves per SIMD
// fit) and one multiplies while the other computes:
//   wave A, block n:  scores of block n and dv of block n - 1, then the probabilities of block n, left in LDS for B
//   wave B, block n:  ds of block n - 1 from A's probabilities, then do . v of block n and dk of block n - 1
// one barrier a block.  Three tiles of queries and output gradients lie in LDS (the last, this one, the one being stored).
// The halves qh are added at the end, in LDS.  (One wave for both gradients, one to a SIMD, was as fast while tiles came through
// registers, but it issues every instruction of a block itself, and 400 of them take longer than its 32 products.)
// 16 heads over 4 of 128 in bf16, sequences of 4096, 265, 1999, 1, 800, 2050: 324 us for its four products (210 GFLOP), 650
// TFLOP/s; what bounds it is LDS (fragments of four tiles and the probabilities' way from A to B) beside one block in flight, and
// uneven work: a key tile has the query blocks behind it to do, one workgroup runs on a CU, and the longest of the 256 CUs'
// turns are 264 blocks there where an even share is 205.
template <int D>
__global__ __launch_bounds__(512, 2) void packed_dkv32_kernel(PackedParams p) {
  using L = Tile32<D>;
  using T = bf16_t;
  constexpr int TB = 64 * L::RB;                                   // bytes of a tile: slot i: q at 2 i TB, dout behind it
  __shared__ __attribute__((aligned(16))) char tiles_[6 * TB];
  __shared__ __attribute__((aligned(16))) float prob[3][4][4][64][4];   // [slot][pair][accumulators 4 j ..][lane]
  __shared__ __attribute__((aligned(16))) float stat[3 * 128];     // [slot][lse, delta][64]
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), hh = lane >> 5;
  const int pair = wave & 3, kb = pair & 1, qh = pair >> 1;
  const bool second = wave >= 4;                                   // wave B
  const int hk = blockIdx.x;
  const Rows R = find_rows<64, false>(p.cu_k, p.S, p.Mk, blockIdx.y, lane);
  if (!R.any) return;
  int q_lo, nq;
  other_rows(p.cu_q, p.S, p.Mq, R.seq, q_lo, nq);
  if ((R.seq < 0 || R.seq >= p.S) && !p.write_gaps) return;
  const int nk = R.n, w0 = 64 * R.tile + 32 * kb;
  const int k_in = w0 + (lane & 31);
  const long long row = R.lo + min(k_in, nk - 1);
  // query i sees key j <= i + nk - nq: the queries from j - (nk - nq) on; all of the wave's keys from `full` on
  const int from = max(k_in - (nk - nq), 0), full = max(w0 + 31 - (nk - nq), 0);
  const int first = max(64 * R.tile - (nk - nq), 0) & ~63;
  // A: keys, B: values.  Masked scores are -inf before the scale: its sign goes into the keys, a zero scale makes them zero
  // (as in the forward)
  u32x4 kv[L::NKS];
  const T* kvp = second ? (const T*)p.v + row * p.v_row + hk * p.v_head : (const T*)p.k + row * p.k_row + hk * p.k_head;
  const unsigned flip = !second && p.scale < 0.f ? 0x80008000u : 0u, keep = !second && p.scale == 0.f ? 0u : 0xffffffffu;
#pragma unroll
  for (int ks = 0; ks < L::NKS; ++ks) {
    kv[ks] = *(const u32x4*)(kvp + 16 * ks + 8 * hh);
#pragma unroll
    for (int e = 0; e < 4; ++e) kv[ks][e] = (kv[ks][e] ^ flip) & keep;
  }
  const float c2 = p.scale == 0.f ? 1.f : fabsf(p.scale) * LOG2E;
  f32x16 grad[L::DB];                                              // A: dv, B: dk
#pragma unroll
  for (int d = 0; d < L::DB; ++d) grad[d] = zero16();
  // this workgroup's share of the key head's query heads
  const int heads = (p.G + p.splits - 1) / p.splits, h0 = hk * p.G + heads * (int)blockIdx.z;
  const int blocks = first < nq ? (nq - first + 63) / 64 : 0, total = blocks * min(heads, p.G - heads * (int)blockIdx.z);
  if (total > 0) {
    // Tiles in order: head by head, the queries from the last down.  Addresses and sizes of the tile to load next are kept as
    // running scalars.  Wave parity picks the row of statistics (lse, delta) a wave fetches; waves of a parity store the same.
    const Fetch64<D, true, 8> fetch_q(p.q_row, wave, lane), fetch_g(p.do_row, wave, lane);
    const int top = first + 64 * (blocks - 1), st_row = wave & 1;
    const long long q_at = (long long)(q_lo + top) * p.q_row + (long long)h0 * p.q_head;
    const long long g_at = (long long)(q_lo + top) * p.do_row + (long long)h0 * p.do_head;
    const T *qa = (const T*)p.q + q_at, *ga = (const T*)p.dout + g_at;
    const float* sa = (st_row ? p.delta : p.lse) + (long long)h0 * p.Mq + q_lo + top;
    const long long q_down = 64 * p.q_row, g_down = 64 * p.do_row, q_next = (long long)(top - first) * p.q_row + p.q_head,
                    g_next = (long long)(top - first) * p.do_row + p.do_head, s_next = top - first + p.Mq;
    const unsigned rest = (unsigned)min(nq - top, 64);             // rows of a head's last tile
    const unsigned q_rest = 2u * ((rest - 1) * (unsigned)p.q_row + D), g_rest = 2u * ((rest - 1) * (unsigned)p.do_row + D);
    const unsigned q_full = 2u * (63u * (unsigned)p.q_row + D), g_full = 2u * (63u * (unsigned)p.do_row + D);
    const float s_mul = st_row ? 1.f : LOG2E;
    int lq = top, left = total;                                    // first query of the tile to load next, tiles left
    float sv = 0.f;
    auto load = [&](int slot) __attribute__((always_inline)) {     // (no tile left: zeros)
      const bool any = left > 0, part = lq == top;
      fetch_q(tiles_ + 2 * slot * TB, make_buffer(qa, !any ? 0u : part ? q_rest : q_full));
      fetch_g(tiles_ + (2 * slot + 1) * TB, make_buffer(ga, !any ? 0u : part ? g_rest : g_full));
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(sa, !any ? 0u : part ? 4u * rest : 256u);
      sv = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, 4u * lane, 0, 0));
      const bool wrap = lq == first;
      qa += wrap ? q_next : -q_down;
      ga += wrap ? g_next : -g_down;
      sa += wrap ? s_next : -64;
      lq = wrap ? top : lq - 64;
      --left;
    };
    auto settle = [&](int slot) __attribute__((always_inline)) {   // the tile being loaded is there
      // a query that sees no key has lse -inf; +inf makes its probabilities 0 instead of NaN
      stat[128 * slot + 64 * st_row + lane] = !st_row && sv == -__builtin_inff() ? __builtin_inff() : sv * s_mul;
      arrive();
    };
    // slot 2 stands for the block before the first: zeros (what they multiply is zero too, but 0 * NaN is not)
#pragma unroll
    for (int i = 0; i < 2 * TB / (512 * 16); ++i) *(u32x4*)(tiles_ + 4 * TB + (t + 512 * i) * 16) = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 2; ++i) *(u32x4*)((char*)&prob[2] + (t + 512 * i) * 16) = u32x4{0u, 0u, 0u, 0u};
    if (t < 128) stat[256 + t] = 0.f;
    load(0);
    settle(0);
    __syncthreads();
    int q0 = top + 32 * qh;                                        // this wave's queries of the current tile
    f32x16 acc = zero16();                                         // A: scores, B: do . v
    u32x4 w[2] = {u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}};   // A: probabilities, B: ds, as operands
    // The matrix instructions of a block, alternating: product i with the keys (or values) of tile rows, gradient i from tile
    // columns; laid out by hand, the fragment of the one four later read with each (hipcc reads it in front of its product)
    constexpr int NP = L::NKS, NM = NP + 2 * L::DB, AHEAD = 4;
    auto multiply = [&](auto slot_) __attribute__((always_inline)) {
      constexpr int SL = decltype(slot_)::value, PV = (SL + 2) % 3;
      // A: q rows of this tile, dout columns of the last; B: dout rows of this, q columns of the last
      const char* rows = tiles_ + (second ? (2 * SL + 1) * TB : 2 * SL * TB);
      const char* cols = tiles_ + (second ? 2 * PV * TB : (2 * PV + 1) * TB);
      static_assert(NP == 2 * L::DB, "one gradient instruction to a product");
      auto fragment = [&](int i) __attribute__((always_inline)) -> u32x4 {
        if (i & 1) return L::cols(cols, 2 * qh + (i >> 1) / L::DB, (i >> 1) % L::DB, lane);
        return L::rows_t(rows, qh, i >> 1, lane);
      };
      u32x4 f[NM];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) f[i] = fragment(i);
      acc = zero16();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        if (i + AHEAD < NM) f[i + AHEAD] = fragment(i + AHEAD);
        if (i & 1) grad[(i >> 1) % L::DB] = MELGPT_MFMA_32x32x16(f[i], w[(i >> 1) / L::DB], grad[(i >> 1) % L::DB]);
        else acc = MELGPT_MFMA_32x32x16(f[i], kv[i >> 1], acc);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto probabilities = [&](auto slot_) __attribute__((always_inline)) {   // of this block (A)
      constexpr int SL = decltype(slot_)::value;
      if (q0 < full || q0 + 32 > nq) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int q = q0 + 8 * (r >> 2) + 4 * hh + (r & 3);
          acc[r] = q >= from && q < nq ? acc[r] : -__builtin_inff();
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {                                // accumulators 4 j .. + 3: queries 8 j + 4 hh .. + 3
        const f32x4 ls = *(const f32x4*)&stat[128 * SL + 32 * qh + 8 * j + 4 * hh];
        f32x4 pr;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          pr[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[4 * j + r], c2, -ls[r]));
          acc[4 * j + r] = pr[r];
        }
        *(f32x4*)&prob[SL][pair][j][lane][0] = pr;
      }
      w[0] = operand16(acc, 0);
      w[1] = operand16(acc, 1);
    };
    auto score_gradients = [&](auto slot_) __attribute__((always_inline)) {   // of the block in slot_ (B)
      constexpr int SL = decltype(slot_)::value;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 de = *(const f32x4*)&stat[128 * SL + 64 + 32 * qh + 8 * j + 4 * hh];
        const f32x4 pr = *(const f32x4*)&prob[SL][pair][j][lane][0];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[4 * j + r] = pr[r] * (acc[4 * j + r] - de[r]);
      }
      w[0] = operand16(acc, 0);
      w[1] = operand16(acc, 1);
    };
    auto block = [&](auto slot_) __attribute__((always_inline)) {
      constexpr int SL = decltype(slot_)::value;
      load((SL + 1) % 3);
      if (second) score_gradients(std::integral_constant<int, (SL + 2) % 3>());
      multiply(slot_);
      if (!second) probabilities(slot_);
      settle((SL + 1) % 3);
      q0 -= 64;
      if (q0 < first) q0 = top + 32 * qh;
      __syncthreads();
    };
    auto last = [&](auto slot_) __attribute__((always_inline)) {   // what the last block still owes
      constexpr int SL = decltype(slot_)::value;
      if (second) score_gradients(slot_);
      const char* cols = tiles_ + (second ? 2 * SL * TB : (2 * SL + 1) * TB);
#pragma unroll
      for (int i = 0; i < 2 * L::DB; ++i)
        grad[i % L::DB] = MELGPT_MFMA_32x32x16(L::cols(cols, 2 * qh + i / L::DB, i % L::DB, lane), w[i / L::DB], grad[i % L::DB]);
    };
    int n = 0;
    for (; n + 3 <= total; n += 3) {
      block(std::integral_constant<int, 0>());
      block(std::integral_constant<int, 1>());
      block(std::integral_constant<int, 2>());
    }
    if (n < total) block(std::integral_constant<int, 0>());
    if (n + 1 < total) block(std::integral_constant<int, 1>());
    switch (total % 3) {
      case 1: last(std::integral_constant<int, 0>()); break;
      case 2: last(std::integral_constant<int, 1>()); break;
      default: last(std::integral_constant<int, 2>());
    }
    __syncthreads();
  }
  // the halves: waves of qh 1 hand over their 32 keys x D sums through LDS
  float* room = (float*)tiles_ + (2 * (int)second + kb) * (32 * D);
  static_assert(4 * 32 * D * 4 <= 6 * TB, "the tiles' room holds the sums");
  if (qh == 1) {
#pragma unroll
    for (int d = 0; d < L::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) room[(16 * d + r) * 64 + lane] = grad[d][r];
  }
  __syncthreads();
  if (qh == 1 || k_in >= nk) return;
  T* out = second ? (T*)p.dk + row * p.dk_row + hk * p.dk_head : (T*)p.dv + row * p.dv_row + hk * p.dv_head;
  float* part = p.splits > 1 ? p.part + ((((long long)blockIdx.z * 2 + !second) * p.Mk + row) * p.Hk + hk) * D : nullptr;
  const float f = second ? p.scale : 1.f;
#pragma unroll
  for (int d = 0; d < L::DB; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (grad[d][4 * j + r] + room[(16 * d + 4 * j + r) * 64 + lane]) * f;
      if (part) *(f32x4*)(part + 32 * d + 8 * j + 4 * hh) = x;
      else store4<T>(out + 32 * d + 8 * j + 4 * hh, x);
    }
}

// adds the shares of a key's gradients in their order: D / 4 lanes, four values each
template <int D>
__global__ __launch_bounds__(256) void packed_dkv_join_kernel(PackedParams p) {
  using T = bf16_t;
  constexpr int TPK = D / 4;
  const long long all = p.Mk * p.Hk, n = (long long)blockIdx.x * (256 / TPK) + threadIdx.x / TPK;
  if (n >= 2 * all) return;
  const bool v = n >= all;
  const long long at = v ? n - all : n, row = at / p.Hk;
  const int d = 4 * (threadIdx.x % TPK), hk = (int)(at % p.Hk);
  const bool gap = row < bound_at(p.cu_k, p.S, p.Mk, 1) || row >= bound_at(p.cu_k, p.S, p.Mk, p.S + 1);
  if (gap && !p.write_gaps) return;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < p.splits; ++i) a += *(const f32x4*)(p.part + (2 * i * all + n) * D + d);
  store4<T>((v ? (T*)p.dv + row * p.dv_row + hk * p.dv_head : (T*)p.dk + row * p.dk_row + hk * p.dk_head) + d, a);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check(const PackedParams& p, int D, int dtype) {
  if (p.S < 0 || p.Hq <= 0 || p.Hk <= 0 || p.Mq < 0 || p.Mk < 0 || !p.cu_q || !p.cu_k || !__builtin_isfinite(p.scale))
    return MELGPT_ERR_BAD_ARG;
  if (dtype != MELGPT_F32 && dtype != MELGPT_BF16) return MELGPT_ERR_UNSUPPORTED;
  if ((D != 64 && D != 128) || p.Hq % p.Hk) return MELGPT_ERR_UNSUPPORTED;
  // tile numbers and row numbers are 32-bit, a grid's second dimension ends at 65535
  if (p.Mq > (1 << 30) || p.Mk > (1 << 30) || p.S > (1 << 24)) return MELGPT_ERR_UNSUPPORTED;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  if (p.Mq > 0 && (!p.q || !p.o || !p.lse)) return MELGPT_ERR_BAD_ARG;
  if (p.Mk > 0 && (!p.k || !p.v)) return MELGPT_ERR_BAD_ARG;
  // rows do not overlap, and 64 of them lie within 4 GB of each other (the kernels' buffer loads); one row has no stride
  if (p.Mk > 1 && (p.k_row < D || p.v_row < D || p.k_row > (1 << 24) || p.v_row > (1 << 24))) return MELGPT_ERR_UNSUPPORTED;
  if (p.Mq > 1 && (p.q_row < D || p.q_row > (1 << 24))) return MELGPT_ERR_UNSUPPORTED;
  if (p.low && dtype == MELGPT_F32) return MELGPT_ERR_UNSUPPORTED;
  if (!aligned16(p.low) || !aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.o)) return MELGPT_ERR_ALIGN;
  if (p.q_row % vec || p.q_head % vec || p.k_row % vec || p.k_head % vec || p.v_row % vec || p.v_head % vec || p.o_row % vec ||
      p.o_head % vec)
    return MELGPT_ERR_ALIGN;
  return MELGPT_OK;
}

// a single row's stride is never used, but the rows behind it must lie outside its buffer
void single_rows(PackedParams& p, int D) {
  if (p.Mq <= 1) p.q_row = p.do_row = D;
  if (p.Mk <= 1) p.k_row = p.v_row = D;
}

template <typename T, int D>
int launch_fwd(const PackedParams& p, hipStream_t s) {
  const int bm = sizeof(T) == 2 ? 128 : 64;
  const long long tiles = tiles_for(p.Mq, p.S, bm);
  if (tiles > 65535) return MELGPT_ERR_UNSUPPORTED;
  if constexpr (sizeof(T) == 2) {
    const long long per = 256 / (D / 4);
    const dim3 joins((unsigned)((p.Hq * p.Mq + per - 1) / per));
    if (p.usual) {
      hipLaunchKernelGGL((packed_fwd32_pool_kernel<D>), dim3(POOLED), dim3(256), 0, s, p);
      hipLaunchKernelGGL((packed_fwd32_kernel<D, true>), dim3(p.Hq, (unsigned)tiles, p.usual), dim3(256), 0, s, p);
      hipLaunchKernelGGL((packed_join_kernel<D, true>), joins, dim3(256), 0, s, p);
    } else {
      hipLaunchKernelGGL((packed_fwd32_kernel<D, false>), dim3(p.Hq, (unsigned)tiles, (unsigned)p.splits), dim3(256), 0, s, p);
      if (p.splits > 1) hipLaunchKernelGGL((packed_join_kernel<D, false>), joins, dim3(256), 0, s, p);
    }
  } else
    hipLaunchKernelGGL((packed_fwd_f32_kernel<D>), dim3(p.Hq, (unsigned)tiles), dim3(256), 0, s, p);
  return melgpt_launch_status();
}

template <typename T, int D>
int launch_bwd(const PackedParams& p, hipStream_t s) {
  const long long tq = tiles_for(p.Mq, p.S, sizeof(T) == 2 ? 128 : 64), tk = tiles_for(p.Mk, p.S, 64);
  if (tq > 65535 || tk > 65535) return MELGPT_ERR_UNSUPPORTED;
  const dim3 gq(p.Hq, (unsigned)tq), gk(p.Hk, (unsigned)tk);
  if constexpr (sizeof(T) == 2) {
    if (p.Mq > 0) hipLaunchKernelGGL((packed_dq32_kernel<D>), gq, dim3(256), 0, s, p);
    if (p.Mk > 0) {
      hipLaunchKernelGGL((packed_dkv32_kernel<D>), dim3(p.Hk, (unsigned)tk, (unsigned)p.splits), dim3(512), 0, s, p);
      const long long per = 256 / (D / 4);
      if (p.splits > 1)
        hipLaunchKernelGGL((packed_dkv_join_kernel<D>), dim3((unsigned)((2 * p.Hk * p.Mk + per - 1) / per)), dim3(256), 0, s, p);
    }
  } else {
    if (p.Mq > 0) hipLaunchKernelGGL((packed_dq_f32_kernel<D>), gq, dim3(256), 0, s, p);
    if (p.Mk > 0) hipLaunchKernelGGL((packed_dkv_f32_kernel<D>), gk, dim3(256), 0, s, p);
  }
  return melgpt_launch_status();
}

// what the launch rules know of a forward: row tiles' workgroups, how many run at once, key tiles of a mean sequence
struct SplitModel {
  double slots, tile_us, base, keys;
  SplitModel(long long Mq, long long Mk, int S, int Hq, int D)
      : slots(D == 64 ? 768 : 512), tile_us(D == 64 ? 0.9 : 1.7), base((double)Hq * (double)((Mq + 127) / 128 + (S - 1) / 2)),
        keys((double)((Mk / S + 63) / 64)) {}
};

}  // namespace

// Workgroups that share the keys of a row tile, where the row tiles alone would not fill the card (a prompt's continuation
// over a long past), by the mean length.  By a model of the launch in microseconds: rounds of the 512 (D 128) or 768 (D 64)
// workgroups that run at once, times a workgroup's 64-key tiles (1.7 / 0.9 us each with full CUs), plus the join (4 us, and 8
// bytes a value and split at 4 TB/s).  Measured in one piece / in the n it takes, 32 heads of 128 over 16000 keys: 1500 queries
// 516 / 416 us (4), 512: 317 / 151 (4), 256: 312 / 91 (8), 128: 311 / 63 (16); 16 heads of 64, 1000 over 8000: 118 / 57 (6).
extern "C" int melgpt_packed_attn_splits(long long Mq, long long Mk, int S, int Hq, int D, int dtype) {
  if (dtype != MELGPT_BF16 || Mq <= 0 || Mk <= 0 || S <= 0 || Hq <= 0 || (D != 64 && D != 128)) return 1;
  const SplitModel m(Mq, Mk, S, Hq, D);
  if (m.base > m.slots) return 1;
  int best = 1;
  double least = 0;
  for (int n = 1; n <= 16 && n * 4 <= m.keys + 3; ++n) {
    const double rounds = (double)(long long)((m.base * n + m.slots - 1) / m.slots), each = (double)(long long)((m.keys + n - 1) / n);
    const double us = rounds * each * m.tile_us + (n > 1 ? 4 + (double)Mq * Hq * n * D * 8 / 4e6 : 0);
    if (n == 1 || us < least) {
      least = us;
      best = n;
    }
  }
  return best;
}

// The same for a batch whose longest sequence has up to `longest` keys (the rule above goes by the mean): more where that one
// would take over 100 us alone and twice the time that sequences of the mean length take together, within half a million
// partial results and for up to 512 sequences: with thousands of short ones, looking for a long one costs as much as they do.
static const int MOST_POOLED = 512;
extern "C" int melgpt_packed_attn_splits_for(long long Mq, long long Mk, int S, int Hq, int D, int dtype, long long longest) {
  const int usual = melgpt_packed_attn_splits(Mq, Mk, S, Hq, D, dtype);
  if (dtype != MELGPT_BF16 || Mq <= 0 || Mk <= 0 || S <= 1 || S > MOST_POOLED || Hq <= 0 || (D != 64 && D != 128)) return usual;
  const SplitModel m(Mq, Mk, S, Hq, D);
  const long long tiles = ((longest < Mk ? longest : Mk) + 63) / 64, room = (1 << 19) / (Hq * Mq);
  const double alone = tiles * m.tile_us / usual, even = (m.base > m.slots ? m.base / m.slots : 1.) * m.keys * m.tile_us / usual;
  long long n = (tiles + 15) / 16;
  if (n > 16) n = 16;
  if (n > room) n = room;
  return n > usual && alone > 100 && alone > 2 * even ? (int)n : usual;
}

extern "C" int melgpt_packed_attn_fwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                      long long k_head, const void* v, long long v_row, long long v_head, const int* cu_q,
                                      const int* cu_k, int S, void* out, long long o_row, long long o_head, void* out_low, float* lse,
                                      int write_gaps, int splits, float* workspace, long long Mq, long long Mk, int Hq, int Hk,
                                      int D, float scale, int dtype, void* stream) {
  PackedParams p = {};
  p.splits = splits; p.part = workspace;
  p.q = q; p.q_row = q_row; p.q_head = q_head; p.k = k; p.k_row = k_row; p.k_head = k_head;
  p.v = v; p.v_row = v_row; p.v_head = v_head; p.o = out; p.o_row = o_row; p.o_head = o_head; p.low = out_low; p.lse = lse;
  p.cu_q = cu_q; p.cu_k = cu_k; p.S = S; p.Hq = Hq; p.Hk = Hk; p.write_gaps = write_gaps; p.Mq = Mq; p.Mk = Mk; p.scale = scale;
  const int e = check(p, D, dtype);
  if (e) return e;
  if (splits < 1 || (splits > 1 && !workspace)) return MELGPT_ERR_BAD_ARG;
  if (splits > 1 && (dtype == MELGPT_F32 || out_low || splits > 1024 || Hq * Mq > (1LL << 26))) return MELGPT_ERR_UNSUPPORTED;
  if (!aligned16(workspace)) return MELGPT_ERR_ALIGN;
  if (Mq == 0) return MELGPT_OK;
  p.G = Hq / Hk;
  const int usual = melgpt_packed_attn_splits(Mq, Mk, S, Hq, D, dtype);
  // (a pool's numbers are 32-bit; 16 shares of 16 tiles or more: see find_pooled)
  if (splits > usual && splits <= 16 && S <= MOST_POOLED && Mk < (1 << 30)) {
    p.usual = usual;
    p.by_usual = ((1u << 31) + usual - 1) / usual;
    p.by_splits = ((1u << 31) + splits - 1) / splits;
  }
  single_rows(p, D);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MELGPT_F32) return D == 64 ? launch_fwd<float, 64>(p, s) : launch_fwd<float, 128>(p, s);
  return D == 64 ? launch_fwd<bf16_t, 64>(p, s) : launch_fwd<bf16_t, 128>(p, s);
}

// Workgroups that share a key tile's query heads, as many as keep a launch within 512 workgroups (two rounds of one to a CU): two
// or more while there are up to 256 key tiles.  One key head of 128 under 8, 4000 tokens, whole backward: 596 us in one piece,
// 238 in 8; two under 16: 647 / 379 in 4; four under 16, 4096 tokens: 409 / 326 in 2.  It counts tiles, not their work: from 257
// to some 400 of them two shares would still help long sequences (four heads under 16, 4700 tokens, 296 tiles: 474 / 404; 6400:
// 682 / 664; two under 14, lengths 4096 to 1: 635 / 450) but cost short ones more (17 of 265, 316 tiles: 96 / 109), and beyond
// they lose (eight under 32 heads of 64, 4000 tokens: 339 / 359).
extern "C" int melgpt_packed_attn_bwd_splits(long long Mk, int S, int Hq, int Hk, int dtype) {
  if (dtype != MELGPT_BF16 || Mk <= 0 || S <= 0 || Hk <= 0 || Hq <= Hk) return 1;
  const long long base = Hk * ((Mk + 63) / 64 + (S - 1) / 2), n = 512 / base;
  return (int)(n < 1 ? 1 : n > Hq / Hk ? Hq / Hk : n);
}

extern "C" int melgpt_packed_attn_bwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                      long long k_head, const void* v, long long v_row, long long v_head, const int* cu_q,
                                      const int* cu_k, int S, const void* out, long long o_row, long long o_head, const void* out_low,
                                      const void* dout, long long do_row, long long do_head, const float* lse, float* delta,
                                      void* dq, long long dq_row, long long dq_head, void* dk, long long dk_row,
                                      long long dk_head, void* dv, long long dv_row, long long dv_head, int write_gaps, int splits,
                                      float* workspace,
                                      long long Mq, long long Mk, int Hq, int Hk, int D, float scale, int dtype, void* stream) {
  PackedParams p = {};
  p.q = q; p.q_row = q_row; p.q_head = q_head; p.k = k; p.k_row = k_row; p.k_head = k_head;
  p.v = v; p.v_row = v_row; p.v_head = v_head; p.o = const_cast<void*>(out); p.o_row = o_row; p.o_head = o_head;
  p.low = const_cast<void*>(out_low);
  p.lse = const_cast<float*>(lse); p.delta = delta; p.dout = dout; p.do_row = do_row; p.do_head = do_head;
  p.dq = dq; p.dq_row = dq_row; p.dq_head = dq_head; p.dk = dk; p.dk_row = dk_row; p.dk_head = dk_head;
  p.dv = dv; p.dv_row = dv_row; p.dv_head = dv_head;
  p.cu_q = cu_q; p.cu_k = cu_k; p.S = S; p.Hq = Hq; p.Hk = Hk; p.write_gaps = write_gaps; p.Mq = Mq; p.Mk = Mk; p.scale = scale;
  const int e = check(p, D, dtype);
  if (e) return e;
  if (Mq > 0 && (!dout || !delta || !dq)) return MELGPT_ERR_BAD_ARG;
  if (Mk > 0 && (!dk || !dv)) return MELGPT_ERR_BAD_ARG;
  if (splits < 1 || (splits > 1 && !workspace)) return MELGPT_ERR_BAD_ARG;
  if (splits > 1 && (dtype == MELGPT_F32 || splits > 1024 || Hk * Mk > (1LL << 25))) return MELGPT_ERR_UNSUPPORTED;
  if (!aligned16(workspace)) return MELGPT_ERR_ALIGN;
  p.splits = splits; p.part = workspace;
  if (Mq > 1 && (do_row < D || do_row > (1 << 24))) return MELGPT_ERR_UNSUPPORTED;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  if (!aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || do_row % vec || do_head % vec || dq_row % vec ||
      dq_head % vec || dk_row % vec || dk_head % vec || dv_row % vec || dv_head % vec)
    return MELGPT_ERR_ALIGN;
  p.G = Hq / Hk;
  single_rows(p, D);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MELGPT_F32) return D == 64 ? launch_bwd<float, 64>(p, s) : launch_bwd<float, 128>(p, s);
  return D == 64 ? launch_bwd<bf16_t, 64>(p, s) : launch_bwd<bf16_t, 128>(p, s);
}
