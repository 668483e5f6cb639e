// Attention of one query token per sequence over a paged key / value cache (the reader of melgpt_kv_append's pages).
//
//   sequence s: keys 0 .. lengths[s] - 1, key j in page page_table[s][j / page_size], slot j % page_size;
//   query head h reads key head h / G:  o = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j e^(scale q . k_j)
//
// Bound by HBM (64 sequences of lengths up to 8192, 32 heads over 8 of 128: 1.07 GB in 211 us, 5.1 TB/s; three of 65537 to
// 131071 over 4: 4.8 TB/s): every key and value is read once, for all G query heads of its key head together - the G queries are the
// columns of a 16-wide matrix tile (one tile per 16 heads), so grouped heads cost no more reads than one.
// Keys go from memory straight into the score product's operand (S^T = K Q^T: 16 keys to a fragment, a lane holds 16 bytes
// of a key row); values take the same lanes' way through a wave's own piece of LDS, whose transposed reads are the operand
// of O^T = V^T P^T.  The waves of a workgroup share nothing until the end: each walks its own 32-key tiles with a running
// maximum and sum, one tile's loads in flight under the previous tile's softmax and second product, and the page numbers of
// the tile after that.  A sequence is split over several workgroups when there are few of them or it is long; their
// partial results are joined by a second kernel in a fixed order.
#include "mma.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct PagedParams {
  const void* q;
  long long q_row, q_head;
  const void *k_pages, *v_pages;
  const int *table, *lengths;
  long long table_ld;
  int width, pages, page_shift, S, Hq, Hk, G, splits, usual, shares, least;
  void* o;
  long long o_row, o_head;
  float* lse;     // (S, Hq)
  float* part;    // (S, Hq, splits, D) sums of e^(s - m) v, then (S, Hq, splits, 2): m (base 2), sum of e^(s - m)
  long long stats;  // offset of the second part
  float scale;
};

template <typename T, int D>
struct Geo {
  static constexpr int ES = Tr<T>::ES, RB = D * ES, CP = RB / 16, VEC = 16 / ES, NKS = CP / 4, DT = D / 16;
  static constexpr int STEPS = ES == 2 ? 1 : 2;
  static __device__ __forceinline__ int off(int row, int c) {
    if constexpr (RB == 128) return row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
    else return row * RB + ((c ^ (row & 15)) << 4);
  }
  // operand of 16 values (16 dt + (lane & 15)) contracting over 32 keys of the tile (16-bit) or 16 (f32, step st)
  static __device__ __forceinline__ u32x4 cols(const char* t, int st, int dt, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (ES == 2) {
      const int r0 = 4 * g + (i >> 2), c = 2 * dt + ((i & 3) >> 1);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, t + off(r0, c) + 8 * (i & 1)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, t + off(r0 + 16, c) + 8 * (i & 1)));
      const s16x8 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(u32x4, f);
    } else {
      const int col = 16 * dt + i;
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = *(const unsigned*)(t + off(16 * st + 4 * g + e, col >> 2) + (col & 3) * 4);
      return f;
    }
  }
};

__device__ __forceinline__ float over_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Keys of sequence s, and its 32-key tiles to a workgroup: an even share of the `usual` number of splits, but no less than
// `least` - a short sequence among long ones uses fewer of them, and the workgroups beyond end at once - and no more than 4096
// keys while there are `shares` for that (see find_pooled).  One tile to a wave where (sequence, key head) pairs are few and
// the longest way counts (one sequence of 4096 keys, 8 key heads of 128: 9.6 us, 14.2 with four to a wave), four from 256 pairs
// on, where a workgroup's start and its partial result are what more of them cost (one sequence of 65536 keys among 63 of
// 1000: 172 us, 209 with one to a wave; lengths up to 4089 in 256 sequences, 8 splits: 418 / 426).
__device__ __forceinline__ int length_of(const PagedParams& p, int s) {
  const long long cap = (long long)p.width << p.page_shift;
  return (int)min((long long)max(p.lengths[s], 0), min(cap, 0x7fffffc0LL));
}
template <bool POOL>
__device__ __forceinline__ int share_of(const PagedParams& p, int tiles) {
  const int even = max((tiles + p.usual - 1) / p.usual, p.least);
  return POOL ? max(min(even, 128), (tiles + p.shares - 1) / p.shares) : even;
}
// The shares beyond the usual ones, of sequences longer than 4096 keys a usual share, so that they do not finish alone: the
// POOLED workgroups of a launch in front take them, number e, e + POOLED, .. of all in order of sequence, share and key head.
// 8 key heads of 128, one sequence of 100000 keys among short ones of 500: 64 in all 371 us without, 160 with, 256 1403 / 207,
// 512 1445 / 291.  Where there are none but the table has room for them, the two launches more cost 2 - 9 us (256 of 500 keys:
// 105 / 110).  Among the others' workgroups the pool was no slower to help (256: 184), but its registers cost those a wave of
// four at head size 64; a grid with room for every sequence's shares cost 1 ns for each workgroup that had nothing to do.
// All lanes of a wave.
constexpr unsigned POOLED = 1024;
// s0, e: where the search stands (number e of those from sequence s0 on); it goes on there for the next.
__device__ __forceinline__ bool any_pooled(const PagedParams& p, int lane) {
  bool any = false;                                                // (loads side by side; the search waits for each)
#pragma unroll 8
  for (int i = lane; i < p.S; i += 64) any = any || p.lengths[i] > 4096LL * p.usual;
  return __any(any);
}
__device__ __forceinline__ bool find_pooled(const PagedParams& p, int& s0, unsigned& e, int lane, int& s, int& hk, int& split) {
  for (; s0 < p.S; s0 += 64) {
    const int tiles = s0 + lane < p.S ? (length_of(p, s0 + lane) + 31) >> 5 : 0;
    const int per = share_of<true>(p, tiles);
    const unsigned mine = (unsigned)max((tiles + per - 1) / per - p.usual, 0) * p.Hk;
    unsigned upto = mine;                                          // of this and the lanes before
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const unsigned before = __shfl_up(upto, d, 64);
      if (lane >= d) upto += before;
    }
    const unsigned all = __builtin_amdgcn_readlane(upto, 63);
    if (e < all) {
      const int at = __builtin_ctzll(__ballot(upto > e));
      const unsigned r = e - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at));
      s = s0 + at;
      hk = (int)(r % (unsigned)p.Hk);
      split = p.usual + (int)(r / (unsigned)p.Hk);
      return true;
    }
    e -= all;
  }
  return false;
}

// which workgroups a launch has: all (no pool), those of the usual shares, the pool
enum { ALL_SHARES, USUAL_SHARES, POOLED_SHARES };
template <typename T, int D, int WHICH>
__global__ __launch_bounds__(256) void paged_decode_kernel(PagedParams p) {
  using L = Geo<T, D>;
  __shared__ __attribute__((aligned(16))) char lds[4][32 * L::RB];
  __shared__ float stat[4][2][16];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4, i16 = lane & 15;
  const int nh = min(p.G - 16 * (int)blockIdx.z, 16);             // query heads of this workgroup
  constexpr bool POOL = WHICH == POOLED_SHARES;
  if (POOL && !any_pooled(p, lane)) return;
  int s0 = 0;
  for (unsigned e = blockIdx.x;; e += POOLED) {
    int hk = blockIdx.x % p.Hk, s = blockIdx.x / p.Hk, split = blockIdx.y;
    if (POOL && !find_pooled(p, s0, e, lane, s, hk, split)) return;
    const int h0 = hk * p.G + 16 * blockIdx.z;
    const int len = length_of(p, s), tiles = (len + 31) >> 5, per = share_of<WHICH != ALL_SHARES>(p, tiles);
    if (split > 0 && (long long)split * per >= tiles) return;        // (the join knows as much)
    const int t0 = split * per, t1 = min(t0 + per, tiles);
    const int* table = p.table + (long long)s * p.table_ld;
    const T* kb = (const T*)p.k_pages;
    const T* vb = (const T*)p.v_pages;
    const T* qp = (const T*)p.q + s * p.q_row + (h0 + min(i16, nh - 1)) * p.q_head;
    u32x4 qf[L::NKS];
#pragma unroll
    for (int ks = 0; ks < L::NKS; ++ks) qf[ks] = *(const u32x4*)(qp + (4 * ks + g) * L::VEC);
    const float c2 = p.scale * LOG2E;
    char* vt = lds[wave];
    f32x4 o[L::DT];
#pragma unroll
    for (int d = 0; d < L::DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;

    // rows i16 and 16 + i16 of a tile: page numbers, then the rows themselves
    const int mask = (1 << p.page_shift) - 1;
    int page[2];
    u32x4 kr[2][L::NKS], vr[2][L::NKS];
    unsigned ok[2];                                                  // bit j: key j of the half tile exists
    auto pages_of = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) page[i] = table[min(32 * tile + 16 * i + i16, len - 1) >> p.page_shift];
    };
    auto load = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = 32 * tile + 16 * i + i16;
        const bool in = key < len && page[i] >= 0 && page[i] < p.pages;
        ok[i] = (unsigned)__ballot(in) & 0xffffu;
        const long long at = in ? ((((long long)page[i] * p.Hk + hk) << p.page_shift) + (key & mask)) * D : 0;
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) kr[i][ks] = *(const u32x4*)(kb + at + (4 * ks + g) * L::VEC);
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) vr[i][ks] = *(const u32x4*)(vb + at + (4 * ks + g) * L::VEC);
      }
    };
    int tile = t0 + wave;
    if (tile < t1) {
      pages_of(tile);
      load(tile);
      pages_of(min(tile + 4, t1 - 1));
    }
    for (; tile < t1; tile += 4) {
      f32x4 sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks) mma<T>(sc[i], kr[i][ks], qf[ks]);
      }
      const unsigned seen[2] = {ok[0], ok[1]};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = (seen[i] >> i16) & 1;                        // (0 * NaN is not 0: rows that do not exist are zero)
#pragma unroll
        for (int ks = 0; ks < L::NKS; ++ks)
          *(u32x4*)(vt + L::off(16 * i + i16, 4 * ks + g)) = in ? vr[i][ks] : u32x4{0u, 0u, 0u, 0u};
      }
      if (tile + 4 < t1) {
        load(tile + 4);
        pages_of(min(tile + 8, t1 - 1));
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[i][r] = (seen[i] >> (4 * g + r)) & 1 ? sc[i][r] * c2 : -__builtin_inff();
          top = fmaxf(top, sc[i][r]);
        }
      top = fmaxf(over_groups_max(top), m);
      const float base = top == -__builtin_inff() ? 0.f : top;
      const float keep = __builtin_amdgcn_exp2f(m - base);
      m = top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[i][r] = __builtin_amdgcn_exp2f(sc[i][r] - base);
          sum += sc[i][r];
        }
      l = l * keep + sum;
#pragma unroll
      for (int d = 0; d < L::DT; ++d) o[d] *= keep;
#pragma unroll
      for (int e = 0; e < L::STEPS; ++e) {
        u32x4 pf;   // (16-bit lane: probabilities rounded for the second product, as in packed_attn.hip; summed in f32 above)
        if constexpr (L::ES == 2)
          pf = u32x4{pack_bf16x2(sc[0][0], sc[0][1]), pack_bf16x2(sc[0][2], sc[0][3]), pack_bf16x2(sc[1][0], sc[1][1]),
                     pack_bf16x2(sc[1][2], sc[1][3])};
        else
          pf = __builtin_bit_cast(u32x4, e ? sc[1] : sc[0]);
#pragma unroll
        for (int d = 0; d < L::DT; ++d) mma<T>(o[d], L::cols(vt, e, d, lane), pf);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
    l = over_groups_sum(l);
    // ---- the four waves' results: through LDS (each its own piece, 16 queries x D f32, once its values are read)
    static_assert(16 * D * 4 <= 32 * L::RB, "a wave's piece holds its result");
    float* mine = (float*)vt;
#pragma unroll
    for (int d = 0; d < L::DT; ++d) *(f32x4*)(mine + i16 * D + 16 * d + 4 * g) = o[d];
    if (g == 0) {
      stat[wave][0][i16] = m;
      stat[wave][1][i16] = l;
    }
    __syncthreads();
    constexpr int TPQ = D / 4;                                       // threads of one query: four values each
    for (int q = t / TPQ; q < nh; q += 256 / TPQ) {
      const int d = 4 * (t % TPQ);
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][0][q]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(stat[w][0][q] - base);
        a += *(const f32x4*)((const float*)lds[w] + q * D + d) * f;
        sum += stat[w][1][q] * f;
      }
      const long long head = (long long)s * p.Hq + h0 + q;
      if (per >= tiles) {                                            // in one piece
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* op = (T*)p.o + s * p.o_row + (h0 + q) * p.o_head + d;
        if constexpr (L::ES == 2) *(u32x2*)op = u32x2{pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv)};
        else *(f32x4*)op = a * inv;
        if (d == 0) p.lse[head] = sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * LN2;
      } else {
        *(f32x4*)(p.part + (head * p.splits + split) * D + d) = a;
        if (d == 0) {
          p.part[p.stats + 2 * (head * p.splits + split)] = top;
          p.part[p.stats + 2 * (head * p.splits + split) + 1] = sum;
        }
      }
    }
    if (!POOL) return;
    __syncthreads();                                                 // (the waves' results are read before the next share's rows)
  }
}

// joins the n splits of one (sequence, query head): 256 / (D / 4) groups of lanes, four values a lane, take every
// 256 / (D / 4)-th split each, then the groups' sums are added in order (one thread walking 86 splits took 25 us)
template <typename T, int D>
struct JoinRoom {
  static constexpr int TPQ = D / 4, NG = 256 / TPQ;
  float sh[NG][D], sums[NG];
};
template <typename T, int D>
__device__ __forceinline__ void join(const PagedParams& p, long long head, int n, JoinRoom<T, D>& room) {
  constexpr int TPQ = JoinRoom<T, D>::TPQ, NG = JoinRoom<T, D>::NG;
  const int g = threadIdx.x / TPQ, d = 4 * (threadIdx.x % TPQ), lane = threadIdx.x & 63;
  const float* st = p.part + p.stats + 2 * head * p.splits;
  const float* pp = p.part + head * p.splits * D + d;
  float top = -__builtin_inff();
  for (int i = lane; i < n; i += 64) top = fmaxf(top, st[2 * i]);
  top = wave_max(top);
  const float base = top == -__builtin_inff() ? 0.f : top;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int i = g; i < n; i += NG) {
    const float f = __builtin_amdgcn_exp2f(st[2 * i] - base);
    a += *(const f32x4*)(pp + (long long)i * D) * f;
    sum += st[2 * i + 1] * f;
  }
  *(f32x4*)&room.sh[g][d] = a;
  if (d == 0) room.sums[g] = sum;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < NG; ++i) {
    a += *(const f32x4*)&room.sh[i][d];
    sum += room.sums[i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* op = (T*)p.o + (head / p.Hq) * p.o_row + (head % p.Hq) * p.o_head + d;
  if constexpr (sizeof(T) == 2) *(u32x2*)op = u32x2{pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv)};
  else *(f32x4*)op = a * inv;
  if (d == 0) p.lse[head] = sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * LN2;
}
// without a pool a workgroup to a head; with one a few to a sequence (most have nothing to join), each some of its heads
template <typename T, int D, bool POOL>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
  __shared__ __attribute__((aligned(16))) JoinRoom<T, D> room;
  const int s = POOL ? blockIdx.x : blockIdx.x / p.Hq;
  const int tiles = (length_of(p, s) + 31) >> 5, per = share_of<POOL>(p, tiles), n = (tiles + per - 1) / per;
  if (n <= 1) return;                                              // (in one piece: there already)
  if constexpr (!POOL) {
    join<T, D>(p, blockIdx.x, n, room);
  } else {
    for (int h = blockIdx.y; h < p.Hq; h += gridDim.y) {
      join<T, D>(p, (long long)s * p.Hq + h, n, room);
      __syncthreads();
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int D, bool POOL>
int launch_as(const PagedParams& p, hipStream_t s) {
  const unsigned pairs = (unsigned)(p.S * p.Hk), z = (p.G + 15) / 16;
  if (POOL) hipLaunchKernelGGL((paged_decode_kernel<T, D, POOLED_SHARES>), dim3(POOLED, 1, z), dim3(256), 0, s, p);
  hipLaunchKernelGGL((paged_decode_kernel<T, D, POOL ? USUAL_SHARES : ALL_SHARES>), dim3(pairs, p.usual, z), dim3(256), 0, s, p);
  if (p.splits > 1) {
    const int each = p.S < 4096 ? 4096 / p.S : 1;                  // workgroups to a sequence
    const dim3 joins = POOL ? dim3((unsigned)p.S, each < p.Hq ? each : p.Hq) : dim3((unsigned)(p.S * p.Hq));
    hipLaunchKernelGGL((paged_join_kernel<T, D, POOL>), joins, dim3(256), 0, s, p);
  }
  return melgpt_launch_status();
}
template <typename T, int D>
int launch(const PagedParams& p, hipStream_t s) {
  return p.shares > p.usual ? launch_as<T, D, true>(p, s) : launch_as<T, D, false>(p, s);
}

}  // namespace

// Workgroups per (sequence, key head): 2048 in all, 128 keys (a tile to a wave) or more each; a cache of up to 512 keys is
// not split (265 keys, 16 heads of 64: 6.1 us, 7.5 in two).  Measured, heads of 128: one sequence of 4096 keys, 8 key heads
// 60 us in one piece, 9.6 in 32; three of 100000, 4 key heads 1354 / 117 in 128; 64 sequences of lengths up to 8152, 8 key
// heads 243 / 211 in 4 / 204 in 8, but all of 4096 191 / 205 in 4 / 224 in 8.
static long long usual_splits(long long base) { return (2048 + base - 1) / base; }

// Beyond these, room for a split to each 4096 keys of a sequence as long as the longest may be (find_pooled), where that is over
// four usual shares of 4096 (256 sequences of lengths up to 8192: 812 us without, 860 with a pool), within half a million
// partial results and for up to 512 sequences (thousands of short ones: looking for a long one costs as much as they do).
static const int MOST_POOLED = 512;
extern "C" int melgpt_paged_attn_splits(int S, int Hq, int Hk, long long max_length) {
  if (S <= 0 || Hk <= 0 || Hq < Hk || max_length <= 512) return 1;
  const long long base = (long long)S * Hk * ((Hq / Hk + 15) / 16), most = (max_length + 127) / 128, room = (1 << 19) / ((long long)S * Hq);
  long long n = usual_splits(base), more = (max_length + 4095) / 4096;
  if (more > room) more = room;
  if (S <= MOST_POOLED && max_length > 16384 * n && n < more) n = more;
  if (n > most) n = most;
  if (n > 128) n = 128;
  return (int)(n < 1 ? 1 : n);
}

extern "C" int melgpt_paged_attn_decode(const void* q, long long q_row, long long q_head, const void* k_pages,
                                        const void* v_pages, long long n_pages, int page_size, const int* page_table,
                                        long long table_ld, int width, const int* lengths, int S, void* out, long long o_row,
                                        long long o_head, float* lse, int splits, float* workspace, int Hq, int Hk, int D,
                                        float scale, int dtype, void* stream) {
  if (S == 0) return MELGPT_OK;
  if (S < 0 || Hq <= 0 || Hk <= 0 || width <= 0 || n_pages <= 0 || splits <= 0 || page_size <= 0 || !__builtin_isfinite(scale))
    return MELGPT_ERR_BAD_ARG;
  if (!q || !k_pages || !v_pages || !page_table || !lengths || !out || !lse || (splits > 1 && !workspace)) return MELGPT_ERR_BAD_ARG;
  if (dtype != MELGPT_F32 && dtype != MELGPT_BF16) return MELGPT_ERR_UNSUPPORTED;
  if ((D != 64 && D != 128) || Hq % Hk || (page_size & (page_size - 1)) || page_size > (1 << 20) || n_pages > 0x7fffffffLL ||
      splits > 65535 || (long long)S * Hq > 0xffffff || Hq / Hk > 1024)
    return MELGPT_ERR_UNSUPPORTED;
  const int vec = dtype == MELGPT_F32 ? 4 : 8;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) || !aligned16(workspace) || q_row % vec ||
      q_head % vec || o_row % vec || o_head % vec)
    return MELGPT_ERR_ALIGN;
  PagedParams p = {};
  p.q = q; p.q_row = q_row; p.q_head = q_head; p.k_pages = k_pages; p.v_pages = v_pages; p.table = page_table; p.lengths = lengths;
  p.table_ld = table_ld; p.width = width; p.pages = (int)n_pages; p.Hq = Hq; p.Hk = Hk; p.G = Hq / Hk; p.splits = splits;
  p.o = out; p.o_row = o_row; p.o_head = o_head; p.lse = lse; p.part = workspace; p.stats = (long long)S * Hq * splits * D;
  p.scale = scale;
  p.S = S;
  const long long pairs = (long long)S * Hk, base = pairs * ((p.G + 15) / 16), usual = usual_splits(base);
  p.least = base < 256 ? 4 : 16;
  p.shares = splits;
  p.usual = splits;
  // (the pool's numbers are 32-bit)
  if (splits > usual && S <= MOST_POOLED && pairs <= (1 << 20) && pairs * splits < (1LL << 31)) p.usual = (int)usual;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MELGPT_F32) return D == 64 ? launch<float, 64>(p, st) : launch<float, 128>(p, st);
  return D == 64 ? launch<bf16_t, 64>(p, st) : launch<bf16_t, 128>(p, st);
}
