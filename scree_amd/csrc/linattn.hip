// Varlen linear attention with a decay per head (gfx950): chunked walks for
// packed sequences, forward and backward, and the recurrent single-token step.
// No counterpart in the reference.
//
// Per sequence and K/V head with lam = exp(log_decay):
//   S_t = lam S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,
// S_{-1} the initial state or zero; query head h reads K/V head h / group.
// With R_t = dL/dS_t = lam R_{t+1} + scale sum_group q_t do_t^T (the final
// state's gradient joins at the last token),
//   dq_t = scale S_t do_t,  dk_t = R_t v_t,  dv_t = R_t^T k_t,  dS_{-1} = lam R_0.
// All four outputs are one walk over rows i (from the sequence's end for dk, dv),
//   out_i = sum_{j <= i} lam^{i-j} (x_i . y_j) z_j + lam^{i+e} x_i A,
// with (x, y, z) = (q, k, v), (do, v, k), (v, do, q), (k, q, do) and A the
// state that came in: S, S^T, R^T, R.  e is 1 forward (the state is of the
// token before) and 0 backward (the carried state is lam R of the row after,
// or the final state's gradient itself).
//
// A workgroup walks a segment of a sequence in chunks of C rows with A in its
// accumulators (fp32): per chunk P = X Y^T weighted by lam^{i-j} below the
// diagonal, out = P Z + diag(lam^{i+e}) X A, then A = lam^n A + Y^T diag(..) Z.
// Sequences longer than a segment are first reduced to their segments' own
// states and these chained, so that segments walk side by side (a long
// sequence alone fills the GPU).

#include <type_traits>

#include "common.h"

namespace scree {
namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Frag { typedef typename VecT<T>::x8 t; };
template <> struct Frag<float> { typedef f32x8 t; };

// C(16x16, f32) += A(16x32) B(32x16): lane l holds A row l % 16 / B column
// l % 16 with k = 8 (l / 16) .. + 7; C element i of lane l is row
// 4 (l / 16) + i, column l % 16.  fp32 takes eight products of 4 k each.
__device__ __forceinline__ void mma(f32x4& c, const f16x8& a, const f16x8& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& c, const bf16x8& a, const bf16x8& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& c, const f32x8& a, const f32x8& b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
}

// A tile of D columns in LDS, row-major, rows 16 bytes apart beyond their
// length: 16 rows at one 16-byte chunk then cover the 256 bytes the LDS serves
// a pass, and every address is a lane's own base plus a constant.
//
// Operands that run along the rows (transposed ones, with k = 32 rows of the
// tile) hold in slot j of lane group g row tok(g, j), an order in which their
// reads spread over the banks as well: 16-bit reads take 4 rows x 32 bytes per
// lane group, every other row of 8 (16-byte steps would meet halfway); fp32
// reads 64 bytes of rows 4 apart.  P's columns, which meet them, follow.
template <typename T, int D>
struct Tile {
  static constexpr int PER = 16 / sizeof(T);  // elements per chunk
  static constexpr int CPR = D / PER;         // chunks per row
  static constexpr int PITCH = D + PER;       // elements from row to row
  static __device__ __forceinline__ constexpr int tok(int j) {  // without the group's part
    return sizeof(T) == 4 ? (j & 3) + 16 * (j >> 2) : j < 4 ? 2 * j : 2 * j - 7;
  }
  static constexpr int TOK_G = sizeof(T) == 4 ? 4 : 8;  // the group's part: TOK_G g

  // X is read twice: in the order in which two accumulators hold 32 rows
  // (columns 4 g .. + 3 and 16 + 4 g .. + 3 of 32) and in order.  In 16 bits it
  // lies so that the first is one read: 4 columns u = 0 .. 7 of 32 at place
  // 2 (u % 4) + u / 4.  (Two 8-byte reads in place of the one met in the banks:
  // 16 LDS cycles against 5.)
  static constexpr bool kPairs = sizeof(T) == 2;

  // This lane's place in the reads below, to which (row, col) constants add.
  static __device__ __forceinline__ const T* row8_base(const T* t, int c, int g) { return t + c * PITCH + 8 * g; }
  static __device__ __forceinline__ const T* row44_base(const T* t, int c, int g) {
    return t + c * PITCH + (kPairs ? 8 : 4) * g;
  }
  static __device__ __forceinline__ const T* x8_base(const T* t, int c, int g) {
    return kPairs ? t + c * PITCH + 16 * (g & 1) + 4 * (g >> 1) : row8_base(t, c, g);
  }
  static __device__ __forceinline__ const T* col8_base(const T* t, int c, int g) {
    if constexpr (sizeof(T) == 4) return t + TOK_G * g * PITCH + c;
    else return t + (TOK_G * g + 2 * (c >> 2)) * PITCH + 4 * (c & 3);
  }
  // columns col + 8 g .. + 7 of row + c
  static __device__ __forceinline__ typename Frag<T>::t row8(const T* base, int row, int col) {
    const T* p = base + row * PITCH + col;
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    } else {
      return __builtin_bit_cast(typename Frag<T>::t, ld16(p));
    }
  }
  // of X: columns col + 4 g .. + 3 and col + 16 + 4 g .. + 3 of row + c
  static __device__ __forceinline__ typename Frag<T>::t row44(const T* base, int row, int col) {
    if constexpr (kPairs) {
      return row8(base, row, col);
    } else {
      const T* p = base + row * PITCH + col;
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
      return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
  }
  // of X: columns col + 8 g .. + 7 of row + c
  static __device__ __forceinline__ typename Frag<T>::t x8(const T* base, int row, int col) {
    if constexpr (kPairs) {
      const T* p = base + row * PITCH + col;
      const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 8);
      return __builtin_bit_cast(typename Frag<T>::t, make_uint4(a.x, a.y, b.x, b.y));
    } else {
      return row8(base, row, col);
    }
  }
  // column col + c of rows row + TOK_G g + tok(j).  ds_read_b64_tr_b16 hands
  // lane 16 g + c, slot j, element c % 4 of the 8 bytes addressed by lane
  // 16 g + 4 j + c / 4.
  static __device__ __forceinline__ typename Frag<T>::t col8(const T* base, int row, int col) {
    const T* p = base + row * PITCH + col;
    if constexpr (sizeof(T) == 4) {
      f32x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[tok(j) * PITCH];
      return v;
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      typedef __attribute__((address_space(3))) s4* lds_s4;
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p));
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + PITCH));
      const s8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(typename Frag<T>::t, v);
    }
  }
  // P's tile (row c of a strip, columns col + 4 g .. + 3) into place
  static __device__ __forceinline__ T* score_base(T* t, int c, int g) {
    return sizeof(T) == 4 ? t + c * PITCH + 4 * g : t + c * PITCH + 8 * (g >> 1) + 2 * (g & 1);
  }
  static __device__ __forceinline__ void store_scores(T* base, int row, int col, const f32x4& p) {
    T* d = base + row * PITCH + col;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(d) = make_float4(p[0], p[1], p[2], p[3]);
    } else {
      *reinterpret_cast<uint32_t*>(d) = pack2<T>(p[0], p[2]);
      *reinterpret_cast<uint32_t*>(d + 4) = pack2<T>(p[1], p[3]);
    }
  }
  static __device__ __forceinline__ const T* scores_base(const T* t, int c, int g) {
    return row44_base(t, c, g);
  }
  static __device__ __forceinline__ typename Frag<T>::t scores(const T* base, int row, int col) {
    return row44(base, row, col);
  }
};

// A buffer descriptor over `bytes` bytes at `base`: loads past them return zeros.
[[maybe_unused]] __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
[[maybe_unused]] constexpr uint32_t kOutside = 0xfffffff0u;  // an offset past every buffer

// Rows of a tile on their way from memory to LDS, held in registers: the loads
// of the next rows are issued before the products of the present ones.
template <typename T, int D, int ROWS, int THREADS>
struct Stage {
  typedef Tile<T, D> L;
  static constexpr int N = ROWS * L::CPR / THREADS;
  static constexpr int RPT = THREADS / L::CPR;  // rows per turn of the threads
  static_assert(ROWS * L::CPR % THREADS == 0 && THREADS % L::CPR == 0, "whole chunks per thread");
  uint4 v[N];
  // Row i of the tile is the n rows' i-th from `base`, or from their end
  // (`back`); rows past n and columns past d are zeros.
  __device__ __forceinline__ void load(const T* base, int64_t row_stride, int n, int d, bool back) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t step = (uint32_t)(row_stride * sizeof(T));
    // 64 rows less than 2^24 elements apart: below 2^32 - 16 bytes
    const uint32_t bytes = n > 0 ? (uint32_t)(n - 1) * step + (uint32_t)(d * sizeof(T)) : 0u;
    const __amdgpu_buffer_rsrc_t rs = buffer_of(base, bytes);
    const int r = threadIdx.x / L::CPR, c = threadIdx.x % L::CPR;
    uint32_t at = (uint32_t)(back ? n - 1 - r : r) * step + 16u * c;
    const uint32_t turn = (back ? 0u - RPT : (uint32_t)RPT) * step;
    const int lim = c * L::PER < d ? n - r : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto u = __builtin_amdgcn_raw_buffer_load_b128(rs, i * RPT < lim ? at : kOutside, 0, 0);
      v[i] = make_uint4(u[0], u[1], u[2], u[3]);
      at += turn;
    }
#else
    (void)base, (void)row_stride, (void)n, (void)d, (void)back;
#endif
  }
  __device__ __forceinline__ void store(T* lds) const {
    T* p = lds + threadIdx.x / L::CPR * L::PITCH + threadIdx.x % L::CPR * L::PER;
#pragma unroll
    for (int i = 0; i < N; ++i) st16(p + i * RPT * L::PITCH, v[i]);
  }
  __device__ __forceinline__ void store_x(T* lds) const {
    if constexpr (L::kPairs) {
      const int c = threadIdx.x % L::CPR;  // the 4 columns 2 h and 2 h + 1 of 32, h = c % 4
      T* p = lds + threadIdx.x / L::CPR * L::PITCH + 32 * (c >> 2) + 16 * (c & 1) + 4 * ((c >> 1) & 1);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        *reinterpret_cast<uint2*>(p + i * RPT * L::PITCH) = make_uint2(v[i].x, v[i].y);
        *reinterpret_cast<uint2*>(p + i * RPT * L::PITCH + 8) = make_uint2(v[i].z, v[i].w);
      }
    } else {
      store(lds);
    }
  }
};

// Eight floats as operands of T: `rest` becomes what the operand leaves of
// them (its high bits cut off, so that the next operand takes the following).
template <typename T>
__device__ __forceinline__ typename Frag<T>::t take(float (&rest)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) {
      const uint32_t a = __builtin_bit_cast(uint32_t, rest[j]), b = __builtin_bit_cast(uint32_t, rest[j + 1]);
      w[j / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      rest[j] -= __builtin_bit_cast(float, a & 0xffff0000u);
      rest[j + 1] -= __builtin_bit_cast(float, b & 0xffff0000u);
    } else {
      const auto h = __builtin_amdgcn_cvt_pkrtz(rest[j], rest[j + 1]);
      w[j / 2] = __builtin_bit_cast(uint32_t, h);
      rest[j] = fmaf((float)h[0], -1.f, rest[j]);  // v_fma_mix_f32
      rest[j + 1] = fmaf((float)h[1], -1.f, rest[j + 1]);
    }
  }
  return __builtin_bit_cast(typename Frag<T>::t, make_uint4(w[0], w[1], w[2], w[3]));
}
// Rounded to nearest: the last operand of a sum of them, or fp32 itself.
template <typename T>
__device__ __forceinline__ typename Frag<T>::t to_frag(const float (&f)[8]) {
  if constexpr (sizeof(T) == 4)
    return f32x8{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
  else
    return __builtin_bit_cast(typename Frag<T>::t, pack16<T>(f));
}

// ------------------------------------------------------------ the work items
// Segment j of sequence b has slot cu[b] / M + b + j, M the segment length: a
// sequence of L tokens has max(1, ceil(L / M)) segments, and slots of
// different sequences never meet (floor(a) + ceil(l) <= floor(a + l) + 1), so
// a workgroup finds its segment from the offsets alone.  Slots that no
// segment has are skipped.  Offsets are clamped to [0, total].
struct Segment {
  int seq, index, count;  // the sequence, this segment's place in it, its number of segments
  int64_t row0;           // first row
  int rows;
};
__device__ __forceinline__ int64_t offset_at(const int32_t* cu, int i, int64_t total) {
  return min<int64_t>(max<int64_t>(cu[i], 0), total);
}
__device__ __forceinline__ bool find_segment(const int32_t* __restrict__ cu, int batch, int64_t total,
                                             int seg, int slot, Segment& s) {
  const uint32_t m = (uint32_t)seg;
  auto first_slot = [&](int i) { return (int)((uint32_t)offset_at(cu, i, total) / m) + i; };
  // the last sequence whose first slot is at most `slot`: halving down to a
  // wavefront of sequences, which read their offsets at once
  int lo = 0, hi = batch;  // lo's first slot is at most `slot` (or there is none), hi's is not
  while (hi - lo > 64) {
    const int mid = (lo + hi) >> 1;
    if (first_slot(mid) <= slot) lo = mid;
    else hi = mid;
  }
  const int mine = min(lo + (int)(threadIdx.x & 63), batch - 1);
  const int start = (int)offset_at(cu, mine, total), end = (int)offset_at(cu, mine + 1, total);
  const bool before = lo + (int)(threadIdx.x & 63) < hi && (int)((uint32_t)start / m) + mine <= slot;
  const int found = __popcll(__ballot(before)) - 1;
  if (found < 0) return false;  // offsets that do not begin at 0
  const int a = __builtin_amdgcn_readlane(start, found), b = max(a, __builtin_amdgcn_readlane(end, found));
  // the same in every lane: addresses built on these stay scalar
  s.seq = __builtin_amdgcn_readfirstlane(lo + found);
  s.index = __builtin_amdgcn_readfirstlane(slot - (int)((uint32_t)a / m) - s.seq);
  s.count = __builtin_amdgcn_readfirstlane(max(1, (int)(((uint32_t)(b - a) + m - 1) / m)));
  if (s.index < 0 || s.index >= s.count) return false;
  s.row0 = __builtin_amdgcn_readfirstlane(a + s.index * seg);
  s.rows = __builtin_amdgcn_readfirstlane(min(seg, b - (int)s.row0));
  return true;
}

struct Role {
  const void *x, *y, *z;  // x null: the segment's state alone
  void* out;
  int64_t x_row, x_head, y_row, y_head, z_row, z_head, o_row, o_head;
  const float* init;   // (batch, kv_heads, state): the state that comes in, may be null
  float* last;         // (batch, kv_heads, state): the state that goes out, may be null
  float* seg_state;    // (slots, kv_heads, state)
  int64_t s_x, s_z;    // the state's strides along x's and z's axes
  int x_group;         // heads of x per K/V head
  int x_loop;          // of which a workgroup takes this many, one after the other in every chunk
  int y_group;         // heads of y and z per K/V head, summed
  int dx, dz;
  int reverse;
  int zero_tail;       // rows past the last sequence become zeros (gradients)
  float in_mul, out_mul;  // the state's factors on its way in and out
};
constexpr int kMaxRoles = 3;
struct WalkArgs {
  Role role[kMaxRoles];
  const int32_t* cu;
  const float* log_decay;
  float scale;
  int64_t total;
  int batch, kv_heads, seg, slots;
  int roles, members;     // walks in this launch; workgroups of one segment and K/V head over them
  int start[kMaxRoles];   // first member of each role
  int terms;  // 16-bit operands that a weighted row of Z is split into (2 or 3)
};

template <typename T, int DX> constexpr int chunk_rows() { return sizeof(T) == 4 && DX == 256 ? 32 : 64; }

template <typename T, int DX, int NW, int NT, bool OUT>
constexpr size_t walk_lds() {
  constexpr int C = chunk_rows<T, DX>();
  return sizeof(T) * (size_t)C * ((OUT ? 2 : 1) * Tile<T, DX>::PITCH + Tile<T, 16 * NT * NW>::PITCH +
                                  (OUT ? Tile<T, C>::PITCH : 0)) +
         sizeof(float) * (OUT ? 2 : 1) * 2 * (C + 4);
}
// Waves per SIMD that the registers are held to: as many as the LDS leaves room
// for, but no more than the walk's registers allow without spills.
template <typename T, int DX, int NW, int NT, bool OUT>
constexpr int walk_waves() {
  const int w = (int)(160 * 1024 / walk_lds<T, DX, NW, NT, OUT>()) * NW / 4;
  constexpr int most = OUT ? 2 : 4;
  return w < 1 ? 1 : w > most ? most : w;
}

// NW waves; wave w owns columns [16 NT w, 16 NT (w + 1)) of z, out and the state.
// XLOOP: x's heads of a group in turn (x_loop > 1).
template <typename T, int DX, int NW, int NT, bool OUT, bool XLOOP>
__global__ __launch_bounds__(64 * NW, (walk_waves<T, DX, NW, NT, OUT>())) void lin_walk_kernel(WalkArgs a) {
  constexpr int C = chunk_rows<T, DX>();
  constexpr int CW = 16 * NT, DZ = CW * NW, THREADS = 64 * NW;
  constexpr int ST = C / 16;                   // strips of 16 rows
  constexpr int WPS = NW > ST ? NW / ST : 1;   // waves that share a strip of P
  typedef Tile<T, DX> LX;
  typedef Tile<T, DZ> LZ;
  typedef Tile<T, C> LP;
  typedef typename Frag<T>::t F;
  extern __shared__ __align__(16) char lds_raw[];
  T* ys = reinterpret_cast<T*>(lds_raw);
  T* zs = ys + C * LX::PITCH;
  T* xs = zs + C * LZ::PITCH;
  T* ps = xs + (OUT ? C * LX::PITCH : 0);
  // lam^n, -C <= n <= C, 0 for n < 0, and the same times scale
  float* pow = reinterpret_cast<float*>(ps + (OUT ? C * LP::PITCH : 0)) + C;
  float* pow_s = pow + (OUT ? 2 * (C + 4) : 0);

  // Block b runs on XCD b % 8: the walks of one segment and K/V head, which
  // read the same rows, are a group of blocks on one XCD (its L2 serves them).
  const int place = blockIdx.x >> 3;
  const int group = place / a.members * 8 + (blockIdx.x & 7);
  int member = place % a.members, role = 0;
  while (role + 1 < a.roles && member >= a.start[role + 1]) ++role;
  member -= a.start[role];
  const int kvh = group % a.kv_heads, slot = group / a.kv_heads;
  if (slot >= a.slots) return;
  const Role& r = a.role[role];
  const int slices = (r.dz + DZ - 1) / DZ;
  const int slice = member % slices, x_loop = XLOOP ? r.x_loop : 1;
  const int head = OUT ? kvh * r.x_group + member / slices * x_loop : kvh;  // the first of x's
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int z0 = slice * DZ, zcols = min(DZ, r.dz - z0);

  // Rows behind the last sequence.  The slots from that of a sequence after the
  // last one on have no segment (at least one for every seg such rows): they take
  // a share each (the last slot's alone: a backward of 8,000 tokens in 40,000 rows
  // of 16 x 64 took 161 us against 87).  Where there is none, the last slot's
  // workgroups take the rows.
  [[maybe_unused]] auto zero_tail = [&](bool shared) {
    const int64_t tail = offset_at(a.cu, a.batch, a.total);
    const int past = (int)((uint32_t)tail / (uint32_t)a.seg) + a.batch;
    if (shared ? slot < past : past < a.slots) return;
    const int64_t shares = shared ? a.slots - past : 1, share = shared ? slot - past : 0;
    const int64_t from = tail + (a.total - tail) * share / shares, to = tail + (a.total - tail) * (share + 1) / shares;
    const int per = zcols / 8;
    for (int h = 0; h < x_loop; ++h) {
      T* out = static_cast<T*>(r.out) + (head + h) * r.o_head + z0;
      for (int64_t q = threadIdx.x; q < (to - from) * per; q += THREADS) {
        T* p = out + (from + q / per) * r.o_row + (int)(q % per) * 8;
        st16(p, make_uint4(0u, 0u, 0u, 0u));
        if constexpr (sizeof(T) == 4) st16(p + 4, make_uint4(0u, 0u, 0u, 0u));
      }
    }
  };
  if constexpr (OUT)
    if (r.zero_tail && slot == a.slots - 1) zero_tail(false);
  Segment sg;
  if (!find_segment(a.cu, a.batch, a.total, a.seg, slot, sg)) {
    if constexpr (OUT)
      if (r.zero_tail) zero_tail(true);
    return;
  }
  const bool back = r.reverse;
  const int first = back ? sg.count - 1 : 0, final = sg.count - 1 - first;
  // a segment whose state nobody reads
  if (!OUT && (sg.index == final || sg.count == 1)) return;
  const int rows = sg.rows, dx = r.dx;

  const int y_group = r.y_group;
  const T* x = static_cast<const T*>(r.x) + (OUT ? sg.row0 * r.x_row + head * r.x_head : 0);
  const T* y = static_cast<const T*>(r.y) + sg.row0 * r.y_row + (int64_t)kvh * y_group * r.y_head;
  const T* z = static_cast<const T*>(r.z) + sg.row0 * r.z_row + (int64_t)kvh * y_group * r.z_head + z0;
  const int64_t x_row = r.x_row, x_head = r.x_head, y_row = r.y_row, z_row = r.z_row, y_head = r.y_head, z_head = r.z_head;
  Stage<T, DX, C, THREADS> sx, sy;
  Stage<T, DZ, C, THREADS> sz;
  // chunk ci has n rows from row `low`: the walk's order from the segment's
  // start, or from its end
  auto chunk_rows_of = [&](int ci) { return min(C, rows - ci * C); };
  auto chunk_low = [&](int ci, int n) { return (int64_t)(back ? rows - ci * C - n : ci * C); };
  // A chunk takes `turns` turns: over x's heads, which share Y and Z and the
  // state that came in, or over y's and z's, which sum into X's output.
  constexpr bool over_x = XLOOP;
  const int turns = over_x ? x_loop : y_group, chunks = (rows + C - 1) / C;
  // what chunk ci, turn `turn` brings (nothing past the last chunk: no rows)
  auto fetch = [&](int ci, int turn) {
    const int n = ci < chunks ? chunk_rows_of(ci) : 0;
    const int64_t low = chunk_low(ci, n);
    const int64_t yz = over_x ? 0 : turn;
    const int n_yz = over_x && turn ? 0 : n;
    sy.load(y + low * y_row + yz * y_head, y_row, n_yz, dx, back);
    sz.load(z + low * z_row + yz * z_head, z_row, n_yz, zcols, back);
    if constexpr (OUT)
      sx.load(x + low * x_row + (over_x ? turn : 0) * x_head, x_row, over_x || !turn ? n : 0, dx, back);
  };
  fetch(0, 0);

  const float g2 = a.log_decay[kvh] * 1.4426950408889634f;
  // lam^n; lam^0 is 1 also for a decay of -inf
  auto power = [&](int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(g2 * (float)n); };
  for (int n = (int)threadIdx.x - C; n <= C; n += THREADS) {
    const float w = n < 0 ? 0.f : power(n);
    pow[n] = w;
    if constexpr (OUT) pow_s[n] = w * a.scale;
  }
  const int e = back ? 0 : 1;

  // the state: element [m][u][i] is x-column 16 m + 4 g + i, z-column CW wave + 16 u + c
  f32x4 st[DX / 16][NT];
  const int64_t state_size = (int64_t)dx * r.dz;
  const bool whole = dx == DX && zcols == DZ;
  const float* in = nullptr;
  float in_mul = r.in_mul;  // a segment's state has it already
  if constexpr (OUT) {
    if (sg.index != first) in_mul = 1.f, in = r.seg_state + ((int64_t)slot * a.kv_heads + kvh) * state_size;
    else if (r.init) in = r.init + ((int64_t)sg.seq * a.kv_heads + kvh) * state_size;
  }
#pragma unroll
  for (int m = 0; m < DX / 16; ++m)
#pragma unroll
    for (int u = 0; u < NT; ++u) st[m][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (OUT) if (in) {
    // whole rows of the state, all loads at once, and through the LDS into the
    // accumulators' places (a lane's elements straight from memory, 4 bytes here
    // and there, took 161 us against 145 in the 12,160-token training step of 16
    // x 64, 110 against 96 in the grouped prefill)
    constexpr int RB = 64;  // rows a turn
    auto take_in = [&](auto along_z) {
      constexpr bool Z = decltype(along_z)::value;  // rows along z's columns, else along x's
      constexpr int ROWS = Z ? DX : DZ, W = Z ? DZ : DX, Q = W / 4, P = W + 4;
      constexpr int N = (ROWS * Q + THREADS - 1) / THREADS;
      static_assert((size_t)(ROWS < RB ? ROWS : RB) * P * 4 <= walk_lds<T, DX, NW, NT, OUT>() - 16 * (C + 4), "room");
      const int rows_in = Z ? dx : zcols, cols_in = Z ? zcols : dx;
      const float* src = in + (int64_t)z0 * r.s_z;
      const int64_t pitch = Z ? r.s_x : r.s_z;
      float* buf = reinterpret_cast<float*>(lds_raw);
      float4 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int q = i * THREADS + threadIdx.x, row = q / Q, col = 4 * (q % Q);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < rows_in && col < cols_in) v[i] = *reinterpret_cast<const float4*>(src + row * pitch + col);
      }
#pragma unroll
      for (int r0 = 0; r0 < ROWS; r0 += RB) {
        if (r0) __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int q = i * THREADS + threadIdx.x, row = q / Q - r0, col = 4 * (q % Q);
          if (row >= 0 && row < RB && row + r0 < ROWS) *reinterpret_cast<float4*>(buf + row * P + col) = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < DX / 16; ++m)
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            if constexpr (Z) {
              if (16 * m < r0 || 16 * m >= r0 + RB) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i) st[m][u][i] = buf[(16 * m - r0 + 4 * g + i) * P + CW * wave + 16 * u + c] * in_mul;
            } else {
              const int row = CW * wave + 16 * u - r0;
              if (row < 0 || row >= RB) continue;
              const float4 f = *reinterpret_cast<const float4*>(buf + (row + c) * P + 16 * m + 4 * g);
              st[m][u] = f32x4{f.x * in_mul, f.y * in_mul, f.z * in_mul, f.w * in_mul};
            }
          }
      }
      __syncthreads();  // before the tiles take the buffer's place
    };
    if (r.s_z == 1) take_in(std::true_type{});
    else take_in(std::false_type{});
  }

  if constexpr (OUT) {
    // the products read P in pairs of tiles: those above the diagonal stay zero
    for (int q = threadIdx.x; q < C * LP::PITCH / LP::PER; q += THREADS)
      st16(ps + q * LP::PER, make_uint4(0u, 0u, 0u, 0u));
  }
  const float keep_whole = power(C);
  const T *x8 = LX::x8_base(xs, c, g), *x44 = LX::row44_base(xs, c, g), *y8 = LX::row8_base(ys, c, g);
  const T *yt = LX::col8_base(ys, c, g), *zt = LZ::col8_base(zs, c, g) + CW * wave;
  const T* p8 = LP::scores_base(ps, c, g);
  T* pt = LP::score_base(ps, c, g);
  // weights of P's tiles d strips below the diagonal, lane (c, g) element i: row
  // t = c, column s = 4 g + i, lam^{16 d + c - 4 g - i}; of the state's share,
  // row c of strip s, lam^{16 s + c + e}
  const float *wp = pow_s + c - 4 * g, *wi = pow_s + c + e;
  const float* wz0 = pow - e - LX::TOK_G * g;
  // operands of a weighted row: an output state gets as many as fp32 has bits for
  const bool three = __is_same(T, bf16) && a.terms > 2 && (!OUT || sg.index == final);

  f32x4 o[NT][OUT ? ST : 1];
  for (int ci = 0; ci < chunks; ++ci) {
    const int n = chunk_rows_of(ci);
    for (int turn = 0; turn < turns; ++turn) {
      const bool last_turn = turn == turns - 1;
      if (!over_x || turn == 0) {
        sy.store(ys);
        sz.store(zs);
      }
      if constexpr (OUT) {
        if (over_x || turn == 0) sx.store_x(xs);
      }
      __syncthreads();
      fetch(last_turn ? ci + 1 : ci, last_turn ? 0 : turn + 1);

      if constexpr (OUT) {
        // P, a strip of 16 rows to WPS waves (every WPS-th tile each), rounded to T
#pragma unroll
        for (int s0 = 0; s0 < ST; s0 += NW) {
          const int strip = s0 + wave / WPS;
          F xf[DX / 32];
#pragma unroll
          for (int k = 0; k < DX / 32; ++k) xf[k] = LX::x8(x8, 16 * strip, 32 * k);
#pragma unroll
          for (int d = 0; d < ST; ++d) {
            if (d > strip || (WPS > 1 && d % WPS != wave % WPS)) continue;
            const int tile = strip - d;
            f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < DX / 32; ++k) mma(p, LX::row8(y8, 16 * tile, 32 * k), xf[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] *= wp[16 * d - i];
            LP::store_scores(pt, 16 * strip, 16 * tile, p);
          }
        }
        // out^T = (X A)^T lam^{i+e}: the state's accumulators are its operand as
        // they lie, in two 16-bit operands
        if (over_x || turn == 0) {
          // a state past fp16's range goes in scaled by a power of two
          float up = 1.f;
          if constexpr (__is_same(T, f16)) {
            float top = 0.f;
#pragma unroll
            for (int m = 0; m < DX / 16; ++m)
#pragma unroll
              for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(st[m][u][i]));
            if (__ballot(top > 32768.f)) {
              // the largest finite one: an infinity stays with its own column
              top = 0.f;
#pragma unroll
              for (int m = 0; m < DX / 16; ++m)
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float f = fabsf(st[m][u][i]);
                    top = fmaxf(top, f < __builtin_inff() ? f : 0.f);
                  }
#pragma unroll
              for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
              const int over = max(__builtin_amdgcn_frexp_expf(top) - 15, 0);
              up = __builtin_amdgcn_ldexpf(1.f, over);
              const float down = __builtin_amdgcn_ldexpf(1.f, -over);
#pragma unroll
              for (int m = 0; m < DX / 16; ++m)
#pragma unroll
                for (int u = 0; u < NT; ++u) st[m][u] *= down;
            }
          }
#pragma unroll
          for (int k = 0; k < DX / 32; ++k) {
            // reads hoisted over several k would not fit the registers
            __builtin_amdgcn_sched_barrier(0);
            F xf[ST];
#pragma unroll
            for (int s = 0; s < ST; ++s) xf[s] = LX::row44(x44, 16 * s, 32 * k);
#pragma unroll
            for (int u = 0; u < NT; ++u) {
              const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
              float f[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                f[i] = st[2 * k][u][i];
                f[4 + i] = st[2 * k + 1][u][i];
              }
              if constexpr (sizeof(T) == 2) {
                const F hi = take<T>(f);
#pragma unroll
                for (int s = 0; s < ST; ++s) {
                  if (k == 0) o[u][s] = zero;
                  mma(o[u][s], hi, xf[s]);
                }
              }
              const F lo = to_frag<T>(f);
#pragma unroll
              for (int s = 0; s < ST; ++s) {
                if (sizeof(T) == 4 && k == 0) o[u][s] = zero;
                mma(o[u][s], lo, xf[s]);
              }
            }
          }
#pragma unroll
          for (int s = 0; s < ST; ++s) {
            const float w = wi[16 * s] * up;
#pragma unroll
            for (int u = 0; u < NT; ++u) o[u][s] *= w;
          }
          if constexpr (__is_same(T, f16))
            if (up != 1.f)
#pragma unroll
              for (int m = 0; m < DX / 16; ++m)
#pragma unroll
                for (int u = 0; u < NT; ++u) st[m][u] *= up;
        }
        __syncthreads();
      }
      if (over_x ? last_turn : turn == 0) {
        const float w = n == C ? keep_whole : power(n);
#pragma unroll
        for (int m = 0; m < DX / 16; ++m)
#pragma unroll
          for (int u = 0; u < NT; ++u) st[m][u] *= w;
      }
      const float* wz = wz0 + n;
#pragma unroll
      for (int kk = 0; kk < C / 32; ++kk) {
        __builtin_amdgcn_sched_barrier(0);
        F zf[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) zf[u] = LZ::col8(zt, 32 * kk, 16 * u);
        if constexpr (OUT) {
#pragma unroll
          for (int s = 2 * kk; s < ST; ++s) {
            const F pf = LP::scores(p8, 16 * s, 32 * kk);
#pragma unroll
            for (int u = 0; u < NT; ++u) mma(o[u][s], zf[u], pf);
          }
        }
        if constexpr (over_x)
          if (!last_turn) continue;
        // Z weighted by lam^{n - e - i}, in two or three 16-bit operands
        float rest[NT][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = wz[-(32 * kk + LX::tok(j))];
#pragma unroll
          for (int u = 0; u < NT; ++u) rest[u][j] = (float)zf[u][j] * w;
        }
        F hi[NT], lo[NT];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int u = 0; u < NT; ++u) hi[u] = take<T>(rest[u]);
          if (three) {
#pragma unroll
            for (int m = 0; m < DX / 16; ++m) {
              const F yf = LX::col8(yt, 32 * kk, 16 * m);
#pragma unroll
              for (int u = 0; u < NT; ++u) mma(st[m][u], yf, hi[u]);
            }
#pragma unroll
            for (int u = 0; u < NT; ++u) hi[u] = take<T>(rest[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) lo[u] = to_frag<T>(rest[u]);
#pragma unroll
        for (int m = 0; m < DX / 16; ++m) {
          if (m % 4 == 0) __builtin_amdgcn_sched_barrier(0);
          const F yf = LX::col8(yt, 32 * kk, 16 * m);
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int u = 0; u < NT; ++u) mma(st[m][u], yf, hi[u]);
          }
#pragma unroll
          for (int u = 0; u < NT; ++u) mma(st[m][u], yf, lo[u]);
        }
      }
      __syncthreads();
      if constexpr (OUT) {
        if (!over_x && !last_turn) continue;
        const int64_t low = chunk_low(ci, n);
        T* out = static_cast<T*>(r.out) + (sg.row0 + low) * r.o_row + (head + (over_x ? turn : 0)) * r.o_head + z0 + CW * wave;
        // row i of the chunk lies at i, or at n - 1 - i: this lane's row of a strip,
        // and the step to the next strip's
        const int row = (NT == 1 && sizeof(T) == 2 ? 16 * (g & 1) : 0) + c;
        out += (int64_t)(back ? n - 1 - row : row) * r.o_row;
        const int64_t strip = (back ? -16 : 16) * r.o_row;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int s = 0; s < ST; ++s) {
            T* dst = out + s * strip + 4 * g;
#pragma unroll
            for (int u = 0; u < NT; ++u)
              if (16 * s + row < n && CW * wave + 16 * u + 4 * g < zcols)
                *reinterpret_cast<float4*>(dst + 16 * u) = make_float4(o[u][s][0], o[u][s][1], o[u][s][2], o[u][s][3]);
          }
        } else if constexpr (NT == 2) {
          // a lane holds 4 columns of a row in either half of 32; exchanged between
          // neighbouring groups, 8 in a row
#pragma unroll
          for (int s = 0; s < ST; ++s) {
            const auto e0 = __builtin_amdgcn_permlane16_swap(pack2<T>(o[0][s][0], o[0][s][1]),
                                                             pack2<T>(o[1][s][0], o[1][s][1]), false, false);
            const auto e1 = __builtin_amdgcn_permlane16_swap(pack2<T>(o[0][s][2], o[0][s][3]),
                                                             pack2<T>(o[1][s][2], o[1][s][3]), false, false);
            const int col = 16 * (g & 1) + 8 * (g >> 1);
            if (16 * s + row < n && CW * wave + col < zcols)
              st16(out + s * strip + col, make_uint4(e0[0], e1[0], e0[1], e1[1]));
          }
        } else {
          // a lane holds 4 columns of a row in every strip; exchanged between two
          // strips and neighbouring groups, 8 columns of a row in one of the two
#pragma unroll
          for (int s = 0; s < ST; s += 2) {
            const auto e0 = __builtin_amdgcn_permlane16_swap(pack2<T>(o[0][s][0], o[0][s][1]),
                                                             pack2<T>(o[0][s + 1][0], o[0][s + 1][1]), false, false);
            const auto e1 = __builtin_amdgcn_permlane16_swap(pack2<T>(o[0][s][2], o[0][s][3]),
                                                             pack2<T>(o[0][s + 1][2], o[0][s + 1][3]), false, false);
            const int col = 8 * (g >> 1);
            if (16 * s + row < n && CW * wave + col < zcols)
              st16(out + s * strip + col, make_uint4(e0[0], e1[0], e0[1], e1[1]));
          }
        }
      }
    }
  }

  float* to = nullptr;
  const float out_mul = OUT ? r.out_mul : 1.f;
  if constexpr (!OUT) {
    to = r.seg_state + ((int64_t)slot * a.kv_heads + kvh) * state_size;
  } else {
    if (r.last && sg.index == final && head % r.x_group == 0)
      to = r.last + ((int64_t)sg.seq * a.kv_heads + kvh) * state_size;
  }
  if (!to) return;
  // the places of the state's load, computed again: kept over the walk they
  // would take its registers
  int g_ = g, c_ = c;
  asm volatile("" : "+v"(g_), "+v"(c_));
  to += 4 * g_ * r.s_x + (z0 + CW * wave + c_) * r.s_z;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const bool col = CW * wave + 16 * u + c_ < zcols;
#pragma unroll
    for (int m = 0; m < DX / 16; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (whole || (col && 16 * m + 4 * g_ + i < dx)) to[(16 * m + i) * r.s_x + 16 * u * r.s_z] = st[m][u][i] * out_mul;
  }
}

// The segments' own states become the states that come into them: along each
// sequence, in = lam^rows in + own.  A thread per four elements.
constexpr int kChainThreads = 256;
__global__ __launch_bounds__(kChainThreads) void lin_chain_kernel(WalkArgs a) {
  const Role& r = a.role[blockIdx.y];
  const int64_t state = (int64_t)r.dx * r.dz;
  const int per = (int)((state / 4 + kChainThreads - 1) / kChainThreads);
  int item = blockIdx.x;
  const int64_t q = (int64_t)(item % per) * kChainThreads + threadIdx.x;
  item /= per;
  const int kvh = item % a.kv_heads, seq = item / a.kv_heads;
  const int64_t s0 = offset_at(a.cu, seq, a.total), s1 = max(s0, offset_at(a.cu, seq + 1, a.total));
  const int count = (int)((s1 - s0 + a.seg - 1) / a.seg);
  if (count < 2 || q * 4 >= state) return;
  const int slot0 = (int)(s0 / a.seg) + seq;
  const float g2 = a.log_decay[kvh] * 1.4426950408889634f;
  float4 cur = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r.init) {
    cur = *reinterpret_cast<const float4*>(r.init + ((int64_t)seq * a.kv_heads + kvh) * state + 4 * q);
    cur.x *= r.in_mul;
    cur.y *= r.in_mul;
    cur.z *= r.in_mul;
    cur.w *= r.in_mul;
  }
  constexpr int U = 8;
  for (int j0 = 0; j0 < count; j0 += U) {
    float4 own[U];
    float4* at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = r.reverse ? count - 1 - (j0 + u) : j0 + u;
      at[u] = reinterpret_cast<float4*>(r.seg_state + ((int64_t)(slot0 + j) * a.kv_heads + kvh) * state) + q;
      // the last segment has no state of its own
      if (j0 + u < count - 1) own[u] = *at[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + u >= count) continue;
      *at[u] = cur;
      if (j0 + u >= count - 1) continue;
      const int j = r.reverse ? count - 1 - (j0 + u) : j0 + u;
      const int rows = (int)min<int64_t>(a.seg, s1 - s0 - (int64_t)j * a.seg);
      const float w = exp2f(g2 * (float)rows);
      cur.x = fmaf(w, cur.x, own[u].x);
      cur.y = fmaf(w, cur.y, own[u].y);
      cur.z = fmaf(w, cur.z, own[u].z);
      cur.w = fmaf(w, cur.w, own[u].w);
    }
  }
}

// ------------------------------------------------------------- single tokens
// S = lam S + k v^T and o = scale S^T q for one token per row of a batch: a
// workgroup per row, K/V head and 32 columns of the state, which it reads and
// writes once (8 lanes of 4 columns by 32 rows; a thread holds its rows' 4
// columns while the group's query heads read them).
constexpr int kStepThreads = 256;
struct StepArgs {
  const void *q, *k, *v;
  void* out;
  const float* log_decay;
  const float* state;
  float* state_out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, s_row, so_row;
  int kv_heads, group, dk, dv;
  float scale;
};
// NT: the new states are stored past the caches (kStepNtBytes).
template <typename T, int ROWS, bool NT>  // ROWS * 32 >= dk
__global__ __launch_bounds__(kStepThreads) void lin_step_kernel(StepArgs a) {
  __shared__ float qs[ROWS * 32];
  __shared__ float4 part[kStepThreads / 64][8];
  const int tiles = (a.dv + 31) / 32;
  int item = blockIdx.x;
  const int tile = item % tiles;
  item /= tiles;
  const int kvh = item % a.kv_heads;
  const int64_t row = item / a.kv_heads;
  const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
  const int col = 32 * tile + 4 * cl;
  const bool live = col < a.dv;
  const float lam = expf(a.log_decay[kvh]);
  const T* k = static_cast<const T*>(a.k) + row * a.k_row + kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + row * a.v_row + kvh * a.v_head;
  const int64_t base = (int64_t)kvh * a.dk * a.dv + col;
  const float* s = a.state + row * a.s_row + base;
  float* so = a.state_out + row * a.so_row + base;
  float4 st[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = 32 * i + rl;
    st[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && d < a.dk) st[i] = *reinterpret_cast<const float4*>(s + (int64_t)d * a.dv);
  }
  float vv[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = to_f32(v[col + j]);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = 32 * i + rl;
    if (!live || d >= a.dk) continue;
    const float kd = to_f32(k[d]);
    st[i].x = fmaf(lam, st[i].x, kd * vv[0]);
    st[i].y = fmaf(lam, st[i].y, kd * vv[1]);
    st[i].z = fmaf(lam, st[i].z, kd * vv[2]);
    st[i].w = fmaf(lam, st[i].w, kd * vv[3]);
    if constexpr (NT) st16_nt(so + (int64_t)d * a.dv, __builtin_bit_cast(uint4, st[i]));
    else *reinterpret_cast<float4*>(so + (int64_t)d * a.dv) = st[i];
  }
  for (int h = 0; h < a.group; ++h) {
    const int head = kvh * a.group + h;
    const T* q = static_cast<const T*>(a.q) + row * a.q_row + head * a.q_head;
    for (int d = threadIdx.x; d < ROWS * 32; d += kStepThreads) qs[d] = d < a.dk ? to_f32(q[d]) : 0.f;
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float qd = qs[32 * i + rl];
      acc.x = fmaf(qd, st[i].x, acc.x);
      acc.y = fmaf(qd, st[i].y, acc.y);
      acc.z = fmaf(qd, st[i].z, acc.z);
      acc.w = fmaf(qd, st[i].w, acc.w);
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
      acc.x += __shfl_xor(acc.x, o);
      acc.y += __shfl_xor(acc.y, o);
      acc.z += __shfl_xor(acc.z, o);
      acc.w += __shfl_xor(acc.w, o);
    }
    if ((threadIdx.x & 63) < 8) part[threadIdx.x >> 6][cl] = acc;
    __syncthreads();
    if (threadIdx.x < 8 && live) {
      float4 t = part[0][cl];
#pragma unroll
      for (int w = 1; w < kStepThreads / 64; ++w) {
        t.x += part[w][cl].x;
        t.y += part[w][cl].y;
        t.z += part[w][cl].z;
        t.w += part[w][cl].w;
      }
      T* o = static_cast<T*>(a.out) + row * a.o_row + head * a.o_head + col;
      o[0] = from_f32<T>(t.x * a.scale);
      o[1] = from_f32<T>(t.y * a.scale);
      o[2] = from_f32<T>(t.z * a.scale);
      o[3] = from_f32<T>(t.w * a.scale);
    }
  }
}

// ------------------------------------------------------------------- host
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Tokens per segment.  The walks' workgroups, a segment and K/V head each, are
// best one round of kLinFill (two for each CU; a sequence has half a segment
// more than its tokens fill, on average): 65,536 tokens x 16 heads of 128 take
// 412 us in segments of 2,048, 463 in 1,024 and 527 in 512, and the fewer
// segments the less traffic of their states (64 KB each, read and written five
// times).  At least kLinMinSeg, at most kLinMaxSeg, so that one long sequence
// among many heads does not outlast the rest (a training step of 83,977 tokens
// of 32 x 128: 2,667 us at 4,096, 2,818 at 2,048).  A small batch of short sequences is one segment each: two
// launches less (22 us against 29 at 1,980 tokens of 16 sequences).
constexpr int64_t kLinFill = 512;
constexpr int kLinMinSeg = 128, kLinMaxSeg = 4096;
constexpr int kLinSmall = 2048, kLinSmallMean = 256;

inline int segment_tokens(int64_t total, int batch, int kv_heads) {
  if (total <= kLinSmall && total <= (int64_t)batch * kLinSmallMean && batch >= 8) return kLinSmall;
  const int64_t room = kLinFill / kv_heads - batch / 2;
  int64_t m = room < 1 ? kLinMaxSeg : ((total + room - 1) / room + 63) / 64 * 64;
  if (m < kLinMinSeg) m = kLinMinSeg;
  if (m > kLinMaxSeg) m = kLinMaxSeg;
  return (int)m;
}
inline int64_t slot_count(int64_t total, int batch, int seg) { return total / seg + batch; }

struct Shape {
  int batch, heads, kv_heads, dk, dv, dtype;
  int64_t total;
};

int check_shape(const char* fn, const Shape& s) {
  if (s.batch < 1) return set_error(SCREE_ERR_UNSUPPORTED, "%s: batch must be at least 1, got %d", fn, s.batch);
  if (s.total < 0 || s.total > ((int64_t)1 << 30))
    return set_error(SCREE_ERR_INVALID, "%s: total_tokens %lld out of range", fn, (long long)s.total);
  if (s.heads < 1 || s.heads > 4096 || s.kv_heads < 1 || s.heads % s.kv_heads)
    return set_error(SCREE_ERR_INVALID, "%s: heads %d (at most 4096) must be a multiple of kv_heads %d", fn,
                     s.heads, s.kv_heads);
  for (int d : {s.dk, s.dv})
    if (d < 8 || d > 256 || d % 8)
      return set_error(SCREE_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (multiples of 8 up to 256)", fn, d);
  if (s.dtype != SCREE_DTYPE_F16 && s.dtype != SCREE_DTYPE_BF16 && s.dtype != SCREE_DTYPE_F32)
    return set_error(SCREE_ERR_UNSUPPORTED, "%s: dtype code %d unsupported (fp16, bf16, fp32)", fn, s.dtype);
  return SCREE_OK;
}

struct Arg {
  const char* name;
  const void* p;
  const int64_t* st;
  int dim;
};
int check_args(const char* fn, const Arg* args, int n, int64_t rows) {
  for (int i = 0; i < n; ++i) {
    const Arg& t = args[i];
    if (!t.p) return set_error(SCREE_ERR_INVALID, "%s: %s is null", fn, t.name);
    if (!aligned16(t.p)) return set_error(SCREE_ERR_INVALID, "%s: %s is not 16-byte aligned", fn, t.name);
    for (int k = 0; k < 2; ++k)
      if (t.st[k] % 8 || t.st[k] < 0 || t.st[k] >= ((int64_t)1 << 24))
        return set_error(SCREE_ERR_INVALID,
                         "%s: %s strides (%lld, %lld) must be multiples of 8 elements in [0, 2^24)", fn, t.name,
                         (long long)t.st[0], (long long)t.st[1]);
    if (rows > 1 && t.st[0] < t.dim)
      return set_error(SCREE_ERR_INVALID, "%s: %s row stride %lld overlaps rows", fn, t.name, (long long)t.st[0]);
  }
  return SCREE_OK;
}
int check_states(const char* fn, const void* const* p, int n) {
  for (int i = 0; i < n; ++i)
    if (p[i] && !aligned16(p[i])) return set_error(SCREE_ERR_INVALID, "%s: a state is not 16-byte aligned", fn);
  return SCREE_OK;
}

// Bytes of one set of segment states (0: no sequence can have two segments).
size_t states_bytes(const Shape& s) {
  const int seg = segment_tokens(s.total, s.batch, s.kv_heads);
  if (s.total <= seg) return 0;
  return (size_t)slot_count(s.total, s.batch, seg) * s.kv_heads * s.dk * s.dv * sizeof(float);
}

template <typename T, int DX, int NW, int NT, bool OUT, bool XLOOP>
int launch_walk(const char* fn, WalkArgs a, int roles, hipStream_t stream) {
  a.roles = roles;
  a.members = 0;
  for (int i = 0; i < roles; ++i) {
    a.start[i] = a.members;
    a.members += (OUT ? a.role[i].x_group / a.role[i].x_loop : 1) * ((a.role[i].dz + 16 * NT * NW - 1) / (16 * NT * NW));
  }
  const int64_t items = ((int64_t)a.slots * a.kv_heads + 7) / 8 * 8 * a.members;
  if (items * 64 * NW > 0xffffffffll)
    return set_error(SCREE_ERR_INVALID, "%s: %lld workgroups are too many", fn, (long long)items);
  constexpr size_t lds = walk_lds<T, DX, NW, NT, OUT>();
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  auto kernel = lin_walk_kernel<T, DX, NW, NT, OUT, XLOOP>;
  if (lds > 64 * 1024) {
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (rc != hipSuccess) return set_error(SCREE_ERR_HIP, "%s: %s", fn, hipGetErrorString(rc));
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)items), dim3(64 * NW), lds, stream, a);
  return check_launch(fn);
}
// 32 columns to a wave instead of 16 halve the LDS reads of a walk and keep two
// waves on a SIMD instead of four.  With 16-bit states of 128 rows and enough
// walks to fill the GPU that is faster (83,977 tokens of 32 x 128 forward 719 us against 838,
// 16 x 1,000 tokens of 16 heads 118 against 131); with few walks, where each
// one's time counts, or fewer rows it is slower (1 x 500 tokens 25 us against 23,
// 16 x 1,000 tokens of 16 x 64 70 against 62).
constexpr int64_t kWideWalks = 320;
template <typename T, bool OUT, bool XLOOP, int DX>
int walk_z(const char* fn, const WalkArgs& a, int roles, hipStream_t stream) {
  const int dz = a.role[0].dz;
#define WALK(NW, NT) return launch_walk<T, DX, NW, NT, OUT, XLOOP>(fn, a, roles, stream)
  if constexpr (DX <= 64)
    if (dz <= 32) WALK(2, 1);
  if constexpr (OUT && sizeof(T) == 2 && DX == 128) {
    int64_t groups = 0;
    for (int i = 0; i < roles; ++i) groups += (int64_t)a.slots * a.kv_heads * (a.role[i].x_group / a.role[i].x_loop);
    if (dz > 64 && groups > kWideWalks) WALK(4, 2);
  }
  if constexpr (DX <= 128)
    if (DX <= 32 || dz <= 64) WALK(4, 1);
  if constexpr (DX > 32) WALK(8, 1);
#undef WALK
}
// One launch for `roles` walks of equal dims, all with x_loop > 1 or none.
template <typename T, bool OUT, bool XLOOP>
int walk(const char* fn, const WalkArgs& a, int roles, hipStream_t stream) {
  const int dx = a.role[0].dx;
  if (dx <= 32) return walk_z<T, OUT, XLOOP, 32>(fn, a, roles, stream);
  if (dx <= 64) return walk_z<T, OUT, XLOOP, 64>(fn, a, roles, stream);
  if (dx <= 128) return walk_z<T, OUT, XLOOP, 128>(fn, a, roles, stream);
  return walk_z<T, OUT, XLOOP, 256>(fn, a, roles, stream);
}
template <typename T>
int walk_out(const char* fn, const WalkArgs& a, int roles, hipStream_t stream) {
  return a.role[0].x_loop > 1 ? walk<T, true, true>(fn, a, roles, stream) : walk<T, true, false>(fn, a, roles, stream);
}
template <typename T>
int segment_states(const char* fn, const WalkArgs& a, int roles, hipStream_t stream) {
  if (int rc = walk<T, false, false>(fn, a, roles, stream)) return rc;
  const int64_t state = (int64_t)a.role[0].dx * a.role[0].dz;
  const int64_t per = (state / 4 + kChainThreads - 1) / kChainThreads;
  const int64_t items = per * a.kv_heads * a.batch;
  if (items * kChainThreads > 0xffffffffll)
    return set_error(SCREE_ERR_INVALID, "%s: %lld workgroups are too many", fn, (long long)items);
  hipLaunchKernelGGL(lin_chain_kernel, dim3((unsigned)items, roles), dim3(kChainThreads), 0, stream, a);
  return check_launch(fn);
}

WalkArgs common_args(const Shape& s, const int32_t* cu, const float* log_decay, float scale, int terms) {
  WalkArgs a = {};
  a.cu = cu;
  a.log_decay = log_decay;
  a.scale = scale;
  a.total = s.total;
  a.batch = s.batch;
  a.kv_heads = s.kv_heads;
  a.seg = segment_tokens(s.total, s.batch, s.kv_heads);
  a.slots = (int)slot_count(s.total, s.batch, a.seg);
  a.terms = terms;
  return a;
}

// Query heads that a workgroup walks together: as many of a group as leave the
// GPU kLinWalks workgroups.  They share the update of the state, its load and
// the rows of k and v.
constexpr int64_t kLinWalks = 256;
int heads_together(const WalkArgs& a, int group) {
  int n = group;
  while (n > 1 && (group % n || (int64_t)a.slots * a.kv_heads * (group / n) < kLinWalks)) --n;
  return n;
}

// 16-bit operands of a weighted row in the states' updates: 16 (bf16) or 22
// (fp16) bits where a state only feeds 16-bit outputs, fp32's 24 where it is
// an output itself.
int update_terms(int dtype, bool state_out) { return state_out && dtype == SCREE_DTYPE_BF16 ? 3 : 2; }

template <typename T>
int run_fwd(const char* fn, const Shape& s, const void* q, const void* k, const void* v, void* o,
            const float* log_decay, const int32_t* cu, const float* init, float* last,
            const int64_t* st, float scale, void* workspace, hipStream_t stream) {
  WalkArgs a = common_args(s, cu, log_decay, scale, update_terms(s.dtype, last != nullptr));
  const int group = s.heads / s.kv_heads;
  a.role[0] = {q, k, v, o, st[0], st[1], st[2], st[3], st[4], st[5], st[6], st[7],
               init, last, static_cast<float*>(workspace), s.dv, 1,
               group, heads_together(a, group), 1, s.dk, s.dv, 0, 0, 1.f, 1.f};
  if (s.total > a.seg)
    if (int rc = segment_states<T>(fn, a, 1, stream)) return rc;
  return walk_out<T>(fn, a, 1, stream);
}

// The carried state of the backward is R / scale (its operands are then the
// rows themselves): the final state's gradient comes in divided by scale, the
// initial state's goes out multiplied.
template <typename T>
int run_bwd(const char* fn, const Shape& s, const void* dout, const void* q, const void* k, const void* v,
            void* dq, void* dk, void* dv, const float* log_decay, const int32_t* cu, const float* init,
            const float* dlast, float* dinit, const float* fwd_states, const int64_t* st, float scale,
            void* workspace, hipStream_t stream) {
  WalkArgs a = common_args(s, cu, log_decay, scale, update_terms(s.dtype, dinit != nullptr));
  const int group = s.heads / s.kv_heads;
  const int64_t *sdo = st, *sq = st + 2, *sk = st + 4, *sv = st + 6, *sdq = st + 8, *sdk = st + 10, *sdv = st + 12;
  float* seg_r = static_cast<float*>(workspace);
  // only written when the forward's are not at hand
  float* seg_s = fwd_states ? const_cast<float*>(fwd_states) : seg_r + states_bytes(s) / sizeof(float);
  const float inv = 1.f / scale;
  if (s.total > a.seg) {
    // R backward from (q, dout), S forward from (k, v), both dk x dv
    a.role[0] = {nullptr, q, dout, nullptr, 0, 0, sq[0], sq[1], sdo[0], sdo[1], 0, 0,
                 dlast, nullptr, seg_r, s.dv, 1, 1, 1, group, s.dk, s.dv, 1, 0, inv, 1.f};
    a.role[1] = {nullptr, k, v, nullptr, 0, 0, sk[0], sk[1], sv[0], sv[1], 0, 0,
                 init, nullptr, seg_s, s.dv, 1, 1, 1, 1, s.dk, s.dv, 0, 0, 1.f, 1.f};
    if (int rc = segment_states<T>(fn, a, fwd_states ? 1 : 2, stream)) return rc;
  }
  const Role rdq = {dout, v, k, dq, sdo[0], sdo[1], sv[0], sv[1], sk[0], sk[1], sdq[0], sdq[1],
                    init, nullptr, seg_s, 1, s.dv, group, heads_together(a, group), 1, s.dv, s.dk, 0, 1, 1.f, 1.f};
  const Role rdk = {v, dout, q, dk, sv[0], sv[1], sdo[0], sdo[1], sq[0], sq[1], sdk[0], sdk[1],
                    dlast, nullptr, seg_r, 1, s.dv, 1, 1, group, s.dv, s.dk, 1, 1, inv, 1.f};
  const Role rdv = {k, q, dout, dv, sk[0], sk[1], sq[0], sq[1], sdo[0], sdo[1], sdv[0], sdv[1],
                    dlast, dinit, seg_r, s.dv, 1, 1, 1, group, s.dk, s.dv, 1, 1, inv, scale};
  // dk first and dv beside it: they read the same rows in the same order
  a.role[0] = rdk;
  if (s.dk == s.dv) {
    a.role[1] = rdv;
    a.role[2] = rdq;
    if (rdq.x_loop == 1) return walk_out<T>(fn, a, 3, stream);
    if (int rc = walk_out<T>(fn, a, 2, stream)) return rc;
  } else {
    if (int rc = walk_out<T>(fn, a, 1, stream)) return rc;
    a.role[0] = rdv;
    if (int rc = walk_out<T>(fn, a, 1, stream)) return rc;
  }
  a.role[0] = rdq;
  return walk_out<T>(fn, a, 1, stream);
}

// States that do not fit the 256 MB behind the L2s, old and new, are not kept
// there for the next step: 256 rows of 8 x 128 x 128 take 54 us with streaming
// stores, 61 without.
constexpr int64_t kStepNtBytes = 256ll << 20;
template <typename T>
int run_step(const char* fn, const StepArgs& a, int64_t rows, hipStream_t stream) {
  const int64_t items = rows * a.kv_heads * ((a.dv + 31) / 32);
  if (items * kStepThreads > 0xffffffffll)
    return set_error(SCREE_ERR_INVALID, "%s: %lld workgroups are too many", fn, (long long)items);
  const int64_t states = rows * a.kv_heads * a.dk * a.dv * 4;
  const bool nt = (a.state == a.state_out ? 1 : 2) * states >= kStepNtBytes;
  const int need = (a.dk + 31) / 32;
  auto kernel = need <= 1 ? (nt ? lin_step_kernel<T, 1, true> : lin_step_kernel<T, 1, false>)
              : need <= 2 ? (nt ? lin_step_kernel<T, 2, true> : lin_step_kernel<T, 2, false>)
              : need <= 4 ? (nt ? lin_step_kernel<T, 4, true> : lin_step_kernel<T, 4, false>)
                          : (nt ? lin_step_kernel<T, 8, true> : lin_step_kernel<T, 8, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)items), dim3(kStepThreads), 0, stream, a);
  return check_launch(fn);
}

}  // namespace
}  // namespace scree

using namespace scree;

extern "C" size_t scree_linear_attn_workspace_bytes(int batch, int64_t total_tokens, int heads,
                                                    int kv_heads, int k_dim, int v_dim, int backward) {
  const Shape s = {batch, heads, kv_heads, k_dim, v_dim, SCREE_DTYPE_F32, total_tokens};
  if (check_shape("scree_linear_attn_workspace_bytes", s)) return 0;
  return states_bytes(s) * (backward ? 2 : 1);
}

extern "C" int scree_linear_attn_fwd(const void* q, const void* k, const void* v, const float* log_decay,
                                     void* o, const float* initial_state, float* final_state,
                                     const int32_t* cu_seqlens, int batch, int64_t total_tokens,
                                     int heads, int kv_heads, int k_dim, int v_dim,
                                     const int64_t* strides, float scale, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* fn = "scree_linear_attn_fwd";
  const Shape s = {batch, heads, kv_heads, k_dim, v_dim, dtype, total_tokens};
  if (int rc = check_shape(fn, s)) return rc;
  if (!cu_seqlens || !log_decay || !strides)
    return set_error(SCREE_ERR_INVALID, "%s: cu_seqlens, log_decay or strides is null", fn);
  const void* states[] = {initial_state, final_state};
  if (int rc = check_states(fn, states, 2)) return rc;
  if (total_tokens) {
    const Arg args[] = {{"q", q, strides, k_dim}, {"k", k, strides + 2, k_dim},
                        {"v", v, strides + 4, v_dim}, {"o", o, strides + 6, v_dim}};
    if (int rc = check_args(fn, args, 4, total_tokens)) return rc;
  } else if (!final_state) {
    return SCREE_OK;
  }
  const size_t need = states_bytes(s);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(SCREE_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", fn, need,
                     workspace ? workspace_bytes : (size_t)0);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SCREE_DTYPE_F32:
      return run_fwd<float>(fn, s, q, k, v, o, log_decay, cu_seqlens, initial_state, final_state, strides,
                            scale, workspace, hs);
    case SCREE_DTYPE_F16:
      return run_fwd<f16>(fn, s, q, k, v, o, log_decay, cu_seqlens, initial_state, final_state, strides,
                          scale, workspace, hs);
    default:
      return run_fwd<bf16>(fn, s, q, k, v, o, log_decay, cu_seqlens, initial_state, final_state, strides,
                           scale, workspace, hs);
  }
}

extern "C" int scree_linear_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                                     const float* log_decay, void* dq, void* dk, void* dv,
                                     const float* initial_state, const float* dfinal_state,
                                     float* dinitial_state, const void* fwd_workspace,
                                     const int32_t* cu_seqlens, int batch, int64_t total_tokens,
                                     int heads, int kv_heads, int k_dim, int v_dim,
                                     const int64_t* strides, float scale, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* fn = "scree_linear_attn_bwd";
  const Shape s = {batch, heads, kv_heads, k_dim, v_dim, dtype, total_tokens};
  if (int rc = check_shape(fn, s)) return rc;
  if (!cu_seqlens || !log_decay || !strides)
    return set_error(SCREE_ERR_INVALID, "%s: cu_seqlens, log_decay or strides is null", fn);
  const void* states[] = {initial_state, dfinal_state, dinitial_state, fwd_workspace};
  if (int rc = check_states(fn, states, 4)) return rc;
  const float inv = 1.f / scale;  // run_bwd carries R / scale
  if (!(scale - scale == 0.f) || !(inv - inv == 0.f))
    return set_error(SCREE_ERR_INVALID, "%s: scale %g must be finite, and 1 / scale too", fn, (double)scale);
  if (total_tokens) {
    const Arg args[] = {{"dout", dout, strides, v_dim}, {"q", q, strides + 2, k_dim},
                        {"k", k, strides + 4, k_dim}, {"v", v, strides + 6, v_dim},
                        {"dq", dq, strides + 8, k_dim}, {"dk", dk, strides + 10, k_dim},
                        {"dv", dv, strides + 12, v_dim}};
    if (int rc = check_args(fn, args, 7, total_tokens)) return rc;
  } else if (!dinitial_state) {
    return SCREE_OK;
  }
  const size_t need = (fwd_workspace ? 1 : 2) * states_bytes(s);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(SCREE_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", fn, need,
                     workspace ? workspace_bytes : (size_t)0);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SCREE_DTYPE_F32:
      return run_bwd<float>(fn, s, dout, q, k, v, dq, dk, dv, log_decay, cu_seqlens, initial_state,
                            dfinal_state, dinitial_state, static_cast<const float*>(fwd_workspace),
                            strides, scale, workspace, hs);
    case SCREE_DTYPE_F16:
      return run_bwd<f16>(fn, s, dout, q, k, v, dq, dk, dv, log_decay, cu_seqlens, initial_state,
                          dfinal_state, dinitial_state, static_cast<const float*>(fwd_workspace), strides,
                          scale, workspace, hs);
    default:
      return run_bwd<bf16>(fn, s, dout, q, k, v, dq, dk, dv, log_decay, cu_seqlens, initial_state,
                           dfinal_state, dinitial_state, static_cast<const float*>(fwd_workspace), strides,
                           scale, workspace, hs);
  }
}

extern "C" int scree_linear_attn_step(const void* q, const void* k, const void* v, const float* log_decay,
                                      void* o, const float* state, float* state_out, int64_t rows,
                                      int heads, int kv_heads, int k_dim, int v_dim,
                                      const int64_t* strides, float scale, int dtype, void* stream) {
  const char* fn = "scree_linear_attn_step";
  const Shape s = {1, heads, kv_heads, k_dim, v_dim, dtype, rows};
  if (int rc = check_shape(fn, s)) return rc;
  if (rows == 0) return SCREE_OK;
  if (!log_decay || !strides || !state || !state_out)
    return set_error(SCREE_ERR_INVALID, "%s: log_decay, strides or a state is null", fn);
  const void* states[] = {state, state_out};
  if (int rc = check_states(fn, states, 2)) return rc;
  const Arg args[] = {{"q", q, strides, k_dim}, {"k", k, strides + 2, k_dim},
                      {"v", v, strides + 4, v_dim}, {"o", o, strides + 6, v_dim}};
  if (int rc = check_args(fn, args, 4, rows)) return rc;
  const int64_t size = (int64_t)kv_heads * k_dim * v_dim;
  for (int i = 8; i < 10; ++i)
    if (strides[i] % 4 || (rows > 1 && strides[i] < size))
      return set_error(SCREE_ERR_INVALID, "%s: state row stride %lld must be a multiple of 4 of at least %lld", fn,
                       (long long)strides[i], (long long)size);
  const StepArgs a = {q, k, v, o, log_decay, state, state_out, strides[0], strides[1], strides[2], strides[3],
                      strides[4], strides[5], strides[6], strides[7], strides[8], strides[9],
                      kv_heads, heads / kv_heads, k_dim, v_dim, scale};
  hipStream_t hs = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SCREE_DTYPE_F32: return run_step<float>(fn, a, rows, hs);
    case SCREE_DTYPE_F16: return run_step<f16>(fn, a, rows, hs);
    default: return run_step<bf16>(fn, a, rows, hs);
  }
}
