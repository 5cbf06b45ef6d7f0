// Log probabilities of given tokens, with each row's entropy and most likely
// tokens, forward and backward (gfx950).  No counterpart in the reference.
//
// For a row x of `vocab` logits with maximum m, s = sum_j exp(x_j - m) and
// t = sum_j exp(x_j - m) (x_j - m):
//   logprob = (x_y - m) - ln s,   entropy = ln s - t / s,
//   top     = the largest x_j - m - ln s, the lowest index first among equals.
// With lp_j = x_j - m - ln s, p_j = exp(lp_j) and the gradients g, gH, gtop_i
// of the three,
//   dx_j = p_j (-(g + sum_i gtop_i) - gH (lp_j + entropy)) + g [j = y] + sum_i gtop_i [j = top_i].
//
// The forward reads a row once: a running maximum with both sums rescaled
// when it rises (per thread and batch of vectors), and per wave a list of its
// largest elements, sorted over the lanes, into which the few elements that
// beat its last entry are inserted.  Rows too few to fill the GPU are split
// over workgroups whose partial results a second kernel joins.  The backward
// reads the row again and writes its gradient once.  Sums are fp32 for every
// input type; logprob, entropy and top are fp32.
//
// Non-finite logits give what the two-pass formula gives: -inf has
// probability zero (and adds nothing to the entropy), a row with a NaN or
// +inf, or with nothing but -inf, has NaN results.

#include "common.h"

namespace scree {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpMaxTop = 64;  // a wave's list has one entry per lane
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -1e4f;  // below this exp is 0: stands for lower values where they meet that 0

typedef unsigned int u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct ElemAligned { typedef u32x4_a2 v; };
template <> struct ElemAligned<float> { typedef u32x4_a4 v; };

// 16 bytes at element alignment: rows of an odd vocabulary start anywhere.
// NT: not kept in the caches (kNtBytes).
template <bool NT, typename T> __device__ __forceinline__ uint4 ld16_elem(const T* p) {
  const auto* q = reinterpret_cast<const typename ElemAligned<T>::v*>(p);
  typename ElemAligned<T>::v v;
  if constexpr (NT) v = __builtin_nontemporal_load(q);
  else v = *q;
  return make_uint4(v.x, v.y, v.z, v.w);
}
template <typename T> __device__ __forceinline__ void st16_elem(T* p, const uint4& u) {
  typename ElemAligned<T>::v v = {u.x, u.y, u.z, u.w};
  __builtin_nontemporal_store(v, reinterpret_cast<typename ElemAligned<T>::v*>(p));
}

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.f : m; }

struct Stats {
  float m, s, t;  // maximum, sum of exp(x - m), sum of exp(x - m) (x - m)
};

// Rescale to the maximum hi >= a.m (hi finite, or the row is NaN anyway).  A
// part that saw only -inf has s = t = 0 and stays so; a NaN sum stays NaN.
__device__ __forceinline__ void rescale(Stats& a, float hi) {
  const float d = fmaxf(a.m - hi, kLowest);
  const float r = exp_of(a.m - hi);
  a.t = r * fmaf(d, a.s, a.t);
  a.s = r * a.s;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float hi = fmaxf(a.m, b.m);
  const float ref = finite_max(hi);
  rescale(a, ref);
  rescale(b, ref);
  return {hi, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ Stats wave_merge(Stats a) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)};
    a = merge(a, b);
  }
  return a;
}

// -------------------------------------------------------- a wave's top list
// Lane i holds the i-th largest (value, index) seen by the wave; unused
// entries are (-inf, INT_MAX), behind every element.  NaN is never inserted.
struct TopList {
  float v;
  int i;
  float last_v;  // entry top_k - 1, wave-uniform
  int last_i;
  __device__ __forceinline__ void init() {
    v = last_v = -__builtin_inff();
    i = last_i = 0x7fffffff;
  }
};
__device__ __forceinline__ bool ahead(float av, int ai, float bv, int bi) {
  return av > bv || (av == bv && ai < bi);
}
__device__ __forceinline__ float lane_f(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// Insert the wave-uniform (v, i): the entries behind it move down one lane
// (wave_shr:1).  The bound to beat stays while entry top_k - 1 is unused.
__device__ __forceinline__ void insert(TopList& l, float v, int i, int top_k) {
  const int lane = threadIdx.x & 63;
  const int pos = __popcll(__ballot(ahead(l.v, l.i, v, i)));
  const int lv = __builtin_bit_cast(int, l.v);
  const float pv = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(lv, lv, 0x138, 0xf, 0xf, false));
  const int pi = __builtin_amdgcn_update_dpp(l.i, l.i, 0x138, 0xf, 0xf, false);
  if (lane >= pos) {
    l.v = lane == pos ? v : pv;
    l.i = lane == pos ? i : pi;
  }
  const int last_i = __builtin_amdgcn_readlane(l.i, top_k - 1);
  if (last_i != 0x7fffffff) {
    l.last_v = lane_f(l.v, top_k - 1);
    l.last_i = last_i;
  }
}
// A first bound for an empty list: with the largest elements that N groups of
// 64 lanes hold, at least top_k elements reach the top_k-th largest of those.
// Found bit by bit in the upper half of the ordered bits, so at most 2^-7 of
// its value below; the list then takes few more than top_k elements instead of
// every new largest (16 rows x 128,000 with 20 alternatives: 54 -> 27 us, and
// 20 with the join's).
template <int N>
__device__ __forceinline__ void seed(TopList& l, const float (&mx)[N], int top_k) {
  uint32_t key[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint32_t b = __builtin_bit_cast(uint32_t, mx[n]);
    key[n] = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
  }
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = t | (1u << bit);
    int count = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) count += __popcll(__ballot(key[n] >= c));
    if (count >= top_k) t = c;
  }
  const float v = __builtin_bit_cast(float, t & 0x80000000u ? t ^ 0x80000000u : ~t);
  l.last_v = v == v ? v : -__builtin_inff();  // the bits below -inf are NaN
}
// Offer every lane's (v, i); lanes with nothing to offer pass NaN.
__device__ __forceinline__ void offer(TopList& l, float v, int i, int top_k) {
  uint64_t todo = __ballot(ahead(v, i, l.last_v, l.last_i));
  while (todo) {
    const int src = __builtin_ctzll(todo);
    insert(l, lane_f(v, src), __builtin_amdgcn_readlane(i, src), top_k);
    todo &= __ballot(ahead(v, i, l.last_v, l.last_i)) & ~(1ull << src);
  }
}

// The lanes' (v, i) for which `reach` holds, behind the `count` already there
// (those past `room` are counted only).
__device__ __forceinline__ void append(float2* found, int room, int& count, bool reach, float v, int i) {
  const uint64_t mask = __ballot(reach);
  const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
  if (reach && at < room) found[at] = make_float2(v, __builtin_bit_cast(float, i));
  count += __popcll(mask);
}
// The (v, i) of N arrays, counts[n] <= 64 each, into an empty list: each counts
// those ahead of it.  By one wave; `order` has 64 places.
template <int N>
__device__ __forceinline__ void rank_into(TopList& l, const float2 (*found)[64], const int (&counts)[N],
                                          float2* order, int top_k) {
  const int lane = threadIdx.x & 63;
  order[lane] = make_float2(-__builtin_inff(), __builtin_bit_cast(float, 0x7fffffff));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  int total = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) total += counts[n];
  for (int base = 0; base < total; base += 64) {
    int at = base + lane, from = 0;  // this lane's place, and its array
    const bool have = at < total;
    if (!have) at = 0;
#pragma unroll
    for (int n = 0; n + 1 < N; ++n)
      if (from == n && at >= counts[n]) at -= counts[n], ++from;
    const float2 mine = found[from][at];
    int rank = 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
      for (int j = 0; j < counts[n]; ++j) {
        const float2 o = found[n][j];
        rank += ahead(o.x, __builtin_bit_cast(int, o.y), mine.x, __builtin_bit_cast(int, mine.y));
      }
    if (have && rank < top_k) order[rank] = mine;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  l.v = order[lane].x;
  l.i = __builtin_bit_cast(int, order[lane].y);
  const int last_i = __builtin_amdgcn_readlane(l.i, top_k - 1);
  if (last_i != 0x7fffffff) {
    l.last_v = lane_f(l.v, top_k - 1);
    l.last_i = last_i;
  }
}

// ---------------------------------------------------------------- forward
struct LogprobOut {
  float* logprob;
  float* entropy;
  float* stats;  // (rows, 2): m, s for the backward; may be null
  float* top_logprob;
  int64_t* top_index;
};

// A row's given token and its logit: read first, so that nothing waits for
// them at the end.
struct Target {
  int64_t at;
  float logit;
};
template <typename T>
__device__ __forceinline__ Target read_target(const void* targets, int target_bytes, const T* x, int vocab,
                                              int64_t row) {
  Target t;
  t.at = target_bytes == 8 ? static_cast<const int64_t*>(targets)[row]
                           : (int64_t)static_cast<const int32_t*>(targets)[row];
  t.logit = t.at >= 0 && t.at < vocab ? to_f32(x[t.at]) : 0.f;
  return t;
}

// A row's results from its merged statistics; called by one whole wave.
__device__ __forceinline__ void finish_row(const Stats& a, const TopList& l, const Target& target,
                                           int vocab, int top_k, int64_t row, const LogprobOut& out) {
  const int lane = threadIdx.x & 63;
  const float ls = logf(a.s);
  if (lane == 0) {
    float lp = 0.f;  // a row without a target
    if (target.at >= vocab) lp = __builtin_nanf("");
    else if (target.at >= 0) lp = (target.logit - a.m) - ls;
    out.logprob[row] = lp;
    out.entropy[row] = ls - a.t / a.s;
    if (out.stats) {
      out.stats[2 * row] = a.m;
      out.stats[2 * row + 1] = a.s;
    }
  }
  if (lane < top_k) {
    out.top_logprob[row * top_k + lane] = (l.v - a.m) - ls;
    out.top_index[row * top_k + lane] = min(l.i, vocab - 1);  // fewer than top_k when NaN fill the row
  }
}

// Workspace of a split forward: per part 3 floats, then per part top_k
// (value, index) pairs.
// TOPS: how the most likely tokens are found.  A row (or part) of one trip has no
// list to keep up: what reaches the bound is collected and ranked once, by wave 0
// (with the join that ranks too, 16 rows x 128,000 with 20 alternatives: 17.6 us,
// with lists 20.2; 4,096 x 5,000 with 64: 46 against 59).  A few are in their
// lists sooner (256 x 32,000 with 5: 15.3 us against 16.4).
constexpr int kLpFewTops = 8;
enum Tops { kTopNone, kTopLists, kTopRanked };
constexpr int kLpVectors = 4;  // vectors per thread and trip, their loads issued together
template <typename T> constexpr int trip_columns() { return kLpVectors * kLpThreads * 16 / (int)sizeof(T); }
template <typename T, Tops TOPS, bool NT>
__global__ __launch_bounds__(kLpThreads) void logprob_fwd_kernel(
    const T* __restrict__ logits, int64_t stride, const void* __restrict__ targets, int target_bytes,
    int vocab, int top_k, int parts, int part_cols, float* __restrict__ part_stats,
    float2* __restrict__ part_top, LogprobOut out) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int U = kLpVectors;
  constexpr bool TOP = TOPS != kTopNone, RANKED = TOPS == kTopRanked;
  const int part = blockIdx.x % parts;
  const int64_t row = blockIdx.x / parts;
  const T* x = logits + row * stride;
  const int c0 = part * part_cols, c1 = min(vocab, c0 + part_cols);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Target target = {-1, 0.f};
  if (parts == 1 && wave == 0) target = read_target(targets, target_bytes, x, vocab, row);

  Stats a = {-__builtin_inff(), 0.f, 0.f};
  TopList l;
  if constexpr (TOP) l.init();
  const int whole = c0 + (c1 - c0) / VEC * VEC;
  __shared__ __align__(16) float lane_max[TOP ? kLpThreads : 1];
  __shared__ float2 found[RANKED ? kLpWaves : 1][64];
  __shared__ int found_n[RANKED ? kLpWaves : 1];
  int count = 0;
  // trips are uniform over a wave (its list needs every lane), the first over
  // the workgroup (its lanes' maxima bound the lists)
  int base = c0 + wave * 64 * VEC;
  do {
    uint4 v[U];
    bool have[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = base + u * kLpThreads * VEC + lane * VEC;
      have[u] = c < whole;
      if (have[u]) v[u] = ld16_elem<NT>(x + c);
    }
    float mx[U], hi = a.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mx[u] = -__builtin_inff();
      if (have[u]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) mx[u] = fmaxf(mx[u], elem<T>(v[u], e));
      }
      hi = fmaxf(hi, mx[u]);
    }
    if constexpr (TOP) {
      if (base < c0 + kLpThreads * VEC) {
        lane_max[tid] = hi;
        __syncthreads();
        float mxs[kLpWaves];
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) mxs[w] = lane_max[64 * w + lane];
        seed(l, mxs, top_k);
      }
      if constexpr (RANKED) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = base + u * kLpThreads * VEC + lane * VEC;
          if (__ballot(have[u] && mx[u] >= l.last_v)) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float f = elem<T>(v[u], e);
              append(found[wave], 64, count, have[u] && ahead(f, c + e, l.last_v, l.last_i), f, c + e);
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (RANKED && count <= 64) break;
        const int c = base + u * kLpThreads * VEC + lane * VEC;
        if (__ballot(have[u] && mx[u] >= l.last_v)) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            offer(l, have[u] ? elem<T>(v[u], e) : __builtin_nanf(""), c + e, top_k);
        }
      }
    }
    const float ref = finite_max(hi);
    rescale(a, ref);
    a.m = hi;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!have[u]) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = elem<T>(v[u], e) - ref;
        const float p = exp_of(d);
        a.s += p;
        a.t = fmaf(p, fmaxf(d, kLowest), a.t);
      }
    }
    base += U * kLpThreads * VEC;
  } while (base < whole);
  if constexpr (RANKED) {
    if (count > 64) {  // too many: the list's
      found[wave][lane] = make_float2(l.v, __builtin_bit_cast(float, l.i));
      count = min(top_k, (int)__popcll(__ballot(l.i != 0x7fffffff)));
    }
    if (lane == 0) found_n[wave] = count;
    l.init();
  }
  if (wave == 0) {  // the last columns, fewer than a vector
    const bool have = whole + lane < c1;
    const float f = have ? to_f32(x[whole + lane]) : -__builtin_inff();
    Stats b = {f, 0.f, 0.f};
    if (have) b.s = exp_of(f - finite_max(f));
    a = merge(a, b);
    if constexpr (TOP) offer(l, have ? f : __builtin_nanf(""), whole + lane, top_k);
  }

  __shared__ float red[kLpWaves][3];
  constexpr bool LISTS = TOPS == kTopLists;
  __shared__ float top_v[LISTS ? kLpWaves : 1][kLpMaxTop];
  __shared__ int top_i[LISTS ? kLpWaves : 1][kLpMaxTop];
  a = wave_merge(a);
  if (lane == 0) {
    red[wave][0] = a.m;
    red[wave][1] = a.s;
    red[wave][2] = a.t;
  }
  if constexpr (LISTS) {
    top_v[wave][lane] = l.v;
    top_i[wave][lane] = l.i;
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) a = merge(a, {red[w][0], red[w][1], red[w][2]});
  if constexpr (RANKED) {
    int counts[kLpWaves];
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) counts[w] = __builtin_amdgcn_readfirstlane(found_n[w]);
    const TopList rest = l;  // of the last columns
    l.init();
    rank_into(l, found, counts, reinterpret_cast<float2*>(lane_max), top_k);
    offer(l, lane < VEC && rest.i != 0x7fffffff ? rest.v : __builtin_nanf(""), rest.i, top_k);
  } else if constexpr (LISTS) {
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w)
      offer(l, lane < top_k ? top_v[w][lane] : __builtin_nanf(""), top_i[w][lane], top_k);
  }
  if (parts > 1) {
    if (lane == 0) {
      float* ps = part_stats + 3 * (int64_t)blockIdx.x;
      ps[0] = a.m;
      ps[1] = a.s;
      ps[2] = a.t;
    }
    if (TOP && lane < top_k)
      part_top[(int64_t)blockIdx.x * top_k + lane] = make_float2(l.v, __builtin_bit_cast(float, l.i));
    return;
  }
  finish_row(a, l, target, vocab, top_k, row, out);
}

// One wave per row joins the parts' statistics and lists.
template <typename T>
__global__ __launch_bounds__(64) void logprob_join_kernel(
    const T* __restrict__ logits, int64_t stride, const void* __restrict__ targets, int target_bytes,
    int vocab, int top_k, int parts, const float* __restrict__ part_stats,
    const float2* __restrict__ part_top, LogprobOut out) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const Target target = read_target(targets, target_bytes, logits + row * stride, vocab, row);
  Stats a = {-__builtin_inff(), 0.f, 0.f};
  for (int p = lane; p < parts; p += 64) {
    const float* ps = part_stats + 3 * (row * parts + p);
    a = merge(a, {ps[0], ps[1], ps[2]});
  }
  a = wave_merge(a);
  TopList l;
  l.init();
  if (top_k) {
    const float2* pt = part_top + row * parts * top_k;
    const int n = parts * top_k;
    constexpr int R = 12;  // a lane's candidates per turn, their loads issued together
    for (int base = 0; base < n; base += 64 * R) {
      float2 c[R];
      constexpr int G = 4;  // groups of a lane's candidates
      float mx[G] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int at = base + 64 * i + lane;
        c[i] = at < n ? pt[at] : make_float2(__builtin_nanf(""), 0.f);
        mx[i % G] = fmaxf(mx[i % G], c[i].x);
      }
      if (base == 0) {
        if (top_k > 32) {  // 64 maxima bound as many little
          seed(l, mx, top_k);
        } else {
          const float one[1] = {fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))};
          seed(l, one, top_k);
        }
      }
      if (top_k > kLpFewTops && n <= 64 * R) {
        // the few that reach the bound, side by side (one after the other into
        // the list 16 x 128,000 with 20 took 8.5 us against 6.7)
        __shared__ float2 found[G][64], order[64];
        int total = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int at = __builtin_bit_cast(int, c[i].y);
          append(found[0], 64 * G, total, ahead(c[i].x, at, l.last_v, l.last_i), c[i].x, at);
        }
        __syncthreads();
        if (total <= 64 * G) {
          int counts[G];
#pragma unroll
          for (int j = 0; j < G; ++j) counts[j] = min(max(total - 64 * j, 0), 64);
          rank_into(l, found, counts, order, top_k);
          break;
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) offer(l, c[i].x, __builtin_bit_cast(int, c[i].y), top_k);
    }
  }
  finish_row(a, l, target, vocab, top_k, row, out);
}

// --------------------------------------------------------------- backward
struct LogprobGrad {
  const float* stats;
  const float* entropy;
  const int64_t* top_index;
  const float* dlogprob;  // each gradient may be null: zero
  const float* dentropy;
  const float* dtop;
};

template <typename T, bool NT>
__global__ __launch_bounds__(kLpThreads) void logprob_bwd_kernel(
    const T* __restrict__ logits, int64_t stride, const void* __restrict__ targets, int target_bytes,
    int vocab, int top_k, int parts, int part_cols, LogprobGrad g, T* __restrict__ dlogits,
    int64_t dstride) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int U = 4;
  const int part = blockIdx.x % parts;
  const int64_t row = blockIdx.x / parts;
  const T* x = logits + row * stride;
  T* dx = dlogits + row * dstride;
  const int c0 = part * part_cols, c1 = min(vocab, c0 + part_cols);
  const int tid = threadIdx.x;

  const int64_t target = target_bytes == 8 ? static_cast<const int64_t*>(targets)[row]
                                           : (int64_t)static_cast<const int32_t*>(targets)[row];
  const float glp = g.dlogprob && target >= 0 ? g.dlogprob[row] : 0.f;
  const float gh = g.dentropy ? g.dentropy[row] : 0.f;
  float given = glp;  // the gradients that enter at single columns
  bool any = glp != 0.f || gh != 0.f;
  if (g.dtop) {
    for (int i = 0; i < top_k; ++i) {
      const float gt = g.dtop[row * top_k + i];
      given += gt;
      any = any || gt != 0.f;
    }
  }
  if (!any) {  // nothing reaches the row (a NaN is something): zeros, whatever its logits
    const int whole = c0 + (c1 - c0) / VEC * VEC;
    for (int c = c0 + tid * VEC; c < whole; c += kLpThreads * VEC) st16_elem(dx + c, make_uint4(0u, 0u, 0u, 0u));
    if (whole + tid < c1) dx[whole + tid] = from_f32<T>(0.f);
    return;
  }
  if (target >= vocab) given = __builtin_nanf("");
  const float m = g.stats[2 * row], s = g.stats[2 * row + 1];
  const float ls = logf(s), inv = 1.f / s;
  const float base_c = gh == 0.f ? -given : fmaf(-gh, g.entropy[row] - ls, -given);
  // p (-given - gh (d - ls + H)) with d = x - m
  auto grad = [&](float f) {
    const float d = f - m;
    const float p = exp_of(d) * inv;
    return p * fmaf(-gh, fmaxf(d, kLowest), base_c);
  };

  const int whole = c0 + (c1 - c0) / VEC * VEC;
  for (int base = c0 + tid * VEC; base < whole; base += U * kLpThreads * VEC) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (base + u * kLpThreads * VEC < whole) v[u] = ld16_elem<NT>(x + base + u * kLpThreads * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = base + u * kLpThreads * VEC;
      if (c >= whole) continue;
      float r[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] = grad(elem<T>(v[u], e));
      st16_elem(dx + c, pack16<T>(r));
    }
  }
  if (whole + tid < c1) dx[whole + tid] = from_f32<T>(grad(to_f32(x[whole + tid])));

  // The target's and the alternatives' columns, written again with what
  // enters at them: a thread per column (the first of equal columns), summed
  // in fp32 and rounded once.  The barrier orders the two stores.
  __syncthreads();
  const int n = 1 + (g.dtop ? top_k : 0);
  if (tid >= n) return;
  auto column = [&](int i) { return i == 0 ? target : g.top_index[row * top_k + i - 1]; };
  const int64_t col = column(tid);
  if (col < c0 || col >= c1) return;
  float sum = 0.f;
  for (int i = 0; i < n; ++i) {
    if (column(i) != col) continue;
    if (i < tid) return;
    sum += i == 0 ? glp : g.dtop[row * top_k + i - 1];
  }
  dx[col] = from_f32<T>(grad(to_f32(x[col])) + sum);
}

// ------------------------------------------------------------------- host
// Parts a row is split into: one once the rows alone make kLpFill workgroups
// (four for each CU), else enough for that, each of kLpMinCols columns or more.
constexpr int64_t kLpFill = 1024;
constexpr int64_t kLpMinCols = 4096;
constexpr int64_t kLpBwdCols = 16384;
// Logits that do not fit the 256 MB behind the L2s are gone before the
// backward reads them: streaming loads take 120 us instead of 135 at 778 MB.
// At 198 MB they would lose the backward 20 of its 62 us.
constexpr int64_t kNtBytes = 256ll << 20;

inline int fwd_parts(int64_t rows, int64_t vocab) {
  if (rows >= kLpFill) return 1;
  const int64_t want = (kLpFill + rows - 1) / rows, most = (vocab + kLpMinCols - 1) / kLpMinCols;
  return (int)(want < most ? want : most);
}
inline int part_columns(int64_t vocab, int parts) {  // whole vectors of any type
  return (int)(((vocab + parts - 1) / parts + 7) / 8 * 8);
}

int check_rows(const char* fn, int64_t rows, int64_t vocab, int64_t stride, int top_k,
               int target_bytes) {
  if (vocab < 1 || vocab > ((int64_t)1 << 24))
    return set_error(SCREE_ERR_INVALID, "%s: vocab must be in [1, 2^24], got %lld", fn, (long long)vocab);
  // a launch has one workgroup for every kLpBwdCols columns of a row
  if (rows < 0 || rows > ((int64_t)1 << 23) / ((vocab + kLpBwdCols - 1) / kLpBwdCols))
    return set_error(SCREE_ERR_INVALID, "%s: %lld rows of %lld logits out of range", fn, (long long)rows,
                     (long long)vocab);
  if (rows > 1 && stride < vocab)
    return set_error(SCREE_ERR_INVALID, "%s: row stride %lld overlaps rows", fn, (long long)stride);
  if (top_k < 0 || top_k > kLpMaxTop || top_k > vocab)
    return set_error(SCREE_ERR_INVALID, "%s: top_k must be in [0, min(%d, vocab)], got %d", fn, kLpMaxTop, top_k);
  if (target_bytes != 4 && target_bytes != 8)
    return set_error(SCREE_ERR_INVALID, "%s: targets must be of 4 or 8 bytes, got %d", fn, target_bytes);
  return SCREE_OK;
}

template <typename T>
int launch_fwd(const void* logits, int64_t stride, const void* targets, int target_bytes,
               int64_t rows, int vocab, int top_k, const LogprobOut& out, void* workspace,
               hipStream_t stream) {
  const int parts = fwd_parts(rows, vocab);
  const int cols = part_columns(vocab, parts);
  const bool nt = rows * vocab * (int64_t)sizeof(T) > kNtBytes;
  float* ps = static_cast<float*>(workspace);
  float2* pt = parts > 1 ? reinterpret_cast<float2*>(ps + (3 * rows * parts + 3) / 4 * 4) : nullptr;
  const dim3 grid((unsigned)(rows * parts));
  const T* x = static_cast<const T*>(logits);
  auto kernel = top_k == 0 ? (nt ? logprob_fwd_kernel<T, kTopNone, true> : logprob_fwd_kernel<T, kTopNone, false>)
              : top_k > kLpFewTops && cols <= trip_columns<T>()
                  ? (nt ? logprob_fwd_kernel<T, kTopRanked, true> : logprob_fwd_kernel<T, kTopRanked, false>)
                  : (nt ? logprob_fwd_kernel<T, kTopLists, true> : logprob_fwd_kernel<T, kTopLists, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(kLpThreads), 0, stream, x, stride, targets, target_bytes, vocab,
                     top_k, parts, cols, ps, pt, out);
  if (parts > 1)
    hipLaunchKernelGGL((logprob_join_kernel<T>), dim3((unsigned)rows), dim3(64), 0, stream, x, stride,
                       targets, target_bytes, vocab, top_k, parts, ps, pt, out);
  return check_launch("scree_token_logprobs");
}

template <typename T>
int launch_bwd(const void* logits, int64_t stride, const void* targets, int target_bytes,
               int64_t rows, int vocab, int top_k, const LogprobGrad& g, void* dlogits,
               int64_t dstride, hipStream_t stream) {
  const int parts = (int)((vocab + kLpBwdCols - 1) / kLpBwdCols);
  const bool nt = rows * vocab * (int64_t)sizeof(T) > kNtBytes;
  auto kernel = nt ? logprob_bwd_kernel<T, true> : logprob_bwd_kernel<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * parts)), dim3(kLpThreads), 0,
                     stream, static_cast<const T*>(logits), stride, targets, target_bytes, vocab,
                     top_k, parts, part_columns(vocab, parts), g, static_cast<T*>(dlogits), dstride);
  return check_launch("scree_token_logprobs_bwd");
}

}  // namespace
}  // namespace scree

using namespace scree;

extern "C" size_t scree_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_k) {
  if (check_rows("scree_token_logprobs_workspace_bytes", rows, vocab, vocab, top_k, 8) || rows == 0)
    return 0;
  const int64_t parts = fwd_parts(rows, vocab);
  if (parts == 1) return 0;
  return (size_t)((3 * rows * parts + 3) / 4 * 16 + rows * parts * top_k * 8);
}

extern "C" int scree_token_logprobs(const void* logits, int64_t row_stride, const void* targets,
                                    int target_bytes, int64_t rows, int64_t vocab, int top_k,
                                    float* logprob, float* entropy, float* stats,
                                    float* top_logprob, int64_t* top_index, int dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "scree_token_logprobs";
  if (int rc = check_rows(fn, rows, vocab, row_stride, top_k, target_bytes)) return rc;
  if (dtype != SCREE_DTYPE_F32 && dtype != SCREE_DTYPE_F16 && dtype != SCREE_DTYPE_BF16)
    return set_error(SCREE_ERR_UNSUPPORTED, "%s: dtype code %d unsupported (fp16, bf16, fp32)", fn, dtype);
  if (rows == 0) return SCREE_OK;
  if (!logits || !targets || !logprob || !entropy)
    return set_error(SCREE_ERR_INVALID, "%s: null pointer", fn);
  if (top_k && (!top_logprob || !top_index))
    return set_error(SCREE_ERR_INVALID, "%s: top_k without top_logprob and top_index", fn);
  const size_t need = scree_token_logprobs_workspace_bytes(rows, vocab, top_k);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(SCREE_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", fn,
                     need, workspace ? workspace_bytes : (size_t)0);
  const LogprobOut out = {logprob, entropy, stats, top_logprob, top_index};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SCREE_DTYPE_F32:
      return launch_fwd<float>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, out, workspace, s);
    case SCREE_DTYPE_F16:
      return launch_fwd<f16>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, out, workspace, s);
    default:
      return launch_fwd<bf16>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, out, workspace, s);
  }
}

extern "C" int scree_token_logprobs_bwd(const void* logits, int64_t row_stride, const void* targets,
                                        int target_bytes, int64_t rows, int64_t vocab, int top_k,
                                        const float* stats, const float* entropy,
                                        const int64_t* top_index, const float* dlogprob,
                                        const float* dentropy, const float* dtop_logprob,
                                        void* dlogits, int64_t dlogits_stride, int dtype,
                                        void* stream) {
  const char* fn = "scree_token_logprobs_bwd";
  if (int rc = check_rows(fn, rows, vocab, row_stride, top_k, target_bytes)) return rc;
  if (rows > 1 && dlogits_stride < vocab)
    return set_error(SCREE_ERR_INVALID, "%s: dlogits row stride %lld overlaps rows", fn, (long long)dlogits_stride);
  if (dtype != SCREE_DTYPE_F32 && dtype != SCREE_DTYPE_F16 && dtype != SCREE_DTYPE_BF16)
    return set_error(SCREE_ERR_UNSUPPORTED, "%s: dtype code %d unsupported (fp16, bf16, fp32)", fn, dtype);
  if (rows == 0) return SCREE_OK;
  if (!logits || !targets || !stats || !entropy || !dlogits)
    return set_error(SCREE_ERR_INVALID, "%s: null pointer", fn);
  if (dtop_logprob && (!top_index || !top_k))
    return set_error(SCREE_ERR_INVALID, "%s: dtop_logprob without top_index", fn);
  const LogprobGrad g = {stats, entropy, top_index, dlogprob, dentropy, dtop_logprob};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SCREE_DTYPE_F32:
      return launch_bwd<float>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, g, dlogits, dlogits_stride, s);
    case SCREE_DTYPE_F16:
      return launch_bwd<f16>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, g, dlogits, dlogits_stride, s);
    default:
      return launch_bwd<bf16>(logits, row_stride, targets, target_bytes, rows, (int)vocab, top_k, g, dlogits, dlogits_stride, s);
  }
}
