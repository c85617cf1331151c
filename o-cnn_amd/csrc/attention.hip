// Attention along the node order of an octree level: ragged sequences, a sliding window, the first `sinks`
// keys of a sequence visible to every later query, query heads that share key heads.
//
//   s_ij = scale q_i . k_j,  key j visible to the query at position p = i + keys - queries  iff
//     j <= p + right and (j >= p - left or j < sinks) and key_mask[j]
//   o_i = sum_j softmax_j(s_ij) v_j  over the visible keys; zeros where there is none
//   P = exp(s - lse), dV = P^T dO, dS = P (dO V^T - rowsum(dO o)), dQ = scale dS K, dK = scale dS^T Q
//
// Products run on the matrix cores, 32x32 tiles.  Every kernel computes the score tile TRANSPOSED to what
// its second product wants as an operand: an accumulator of v_mfma_f32_32x32 holds, in lane l, column
// l % 32 and rows 8 b + 4 (l / 32) + e, and the same lane of a B operand has to hold the same column and 8
// (bf16: rows of the contraction; fp32: 1) values of the contraction.  The order of the contraction is free
// as long as both operands agree, so the rows an accumulator lane holds are taken as they are: the
// probabilities go from the first product to the second in registers, and softmax statistics are one
// value a lane.  The other operand is read in the matching order: from LDS by ds_read_b64_tr_b16 (bf16) or
// 4 bytes a lane (fp32).
//
// Rows of a key head: the query heads that share it are packed as rows (token, head in group), so one
// pass over the keys serves the whole group, and a step of one token fills up to 32 columns.
#include "sequence.h"

#include <algorithm>
#include <cmath>

namespace ocnn {
namespace {

// Weights of the gradients -- score gradients and the probabilities of dV -- are not rounded to bf16 once but held as two bf16
// (one more product): rounded once they leave dq, dk and dv 1.42 times as far off as the rounding of these themselves does
// (16 x 1500 rows, window 512, 8 heads of 64, forward and backward: 203 us rounded once, 224 us the score gradients so, 237 all).
constexpr bool kFine = true;
// dO . o with the o that was rounded to bf16 leaves dq 2.0 times as far off as its own rounding does where a row sees 2 keys,
// 1.19 times with 9, 1.06 with 33, 1.01 with 512.  Rows that see up to kFewKeys keys -- the first of a causal sequence, those
// between masked keys -- get rowsum(P dP) from a pass of its own over the tiles of their workgroup.
constexpr int kFewKeys = 32;

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxSinks = 64;
constexpr int kFarRows = 512;   // tokens of a work item of the sinks' gradient

struct AttnArgs {
  ocnn_attention_params p;
  void* out; int64_t out_row, out_head;
  float* lse;
  const void* grad; int64_t grad_row, grad_head;              // of the output
  const void* fwd; int64_t fwd_row, fwd_head;                 // the output of the forward call
  void* dq; void* dk; void* dv;
  int64_t dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
  float* delta;
  float* part_o; float* part_ml;                              // split keys: [split][row][dim], [split][row][2]
  float* sink_part;                                           // [work item][kv head][2][sinks][dim]
  int splits, fill, group;
  int near_keys;                                              // of a workgroup of the keys' gradient: 128 or 64
  float scale2;                                               // |scale| * log2(e); a negative scale turns one operand around
};

// How an element is held: bf16; fp32 (v_mfma_f32_32x32x2_f32); Planes: fp32 in memory and three bf16 in LDS and operands,
// x = hi + mid + lo with 8 significant bits each.  A product of two is six of the nine bf16 products (mid lo, lo mid and lo lo
// stay below 2^-26 of it), 192 cycles for 16 channels instead of 512.  What is left out: below 2^-108 an element's lo (then its
// mid) is a bf16 denormal, and beyond the largest bf16 it is infinite, as the weights of a row that is taken again.
struct Planes {};
template <typename E> struct Elem { using Memory = E; using Lds = E; static constexpr int kPlanes = 1; };
template <> struct Elem<Planes> { using Memory = float; using Lds = uint16_t; static constexpr int kPlanes = 3; };
template <typename E> struct Frag { using type = bf16x8; };
template <> struct Frag<float> { using type = floatx4; };

// What a tile of rows looks like in LDS and in operands.  A 16-byte piece of an operand is kPiece elements; one step of the
// contraction over channels takes two pieces, one from each half of the wavefront.
template <typename E, int DP> struct Shape {
  using Memory = typename Elem<E>::Memory;
  using Lds = typename Elem<E>::Lds;
  static constexpr int kPiece = 16 / (int)sizeof(Lds), kMemoryPiece = 16 / (int)sizeof(Memory);
  static constexpr int kSteps = DP / (2 * kPiece);
  static constexpr int kPieces = DP / kMemoryPiece;     // of a row in memory
  static constexpr int kPitch = DP + kPiece;            // one piece of padding: rows start 4 banks apart
  static constexpr int kBlocks = DP / 32;               // 32-channel blocks of a transposed accumulator
  static constexpr int kPlanes = Elem<E>::kPlanes;
  static constexpr int kPlane = 64 * kPitch;            // (tiles in planes have 64 rows)
};
// wavefronts a SIMD that the registers leave room for
constexpr int plain_waves(int row_bytes) { return row_bytes <= 128 ? 3 : row_bytes <= 256 ? 2 : 1; }
template <typename E> constexpr int forward_waves(int dp) {
  return Elem<E>::kPlanes == 3 ? (dp <= 32 ? 2 : 1) : plain_waves(dp * (int)sizeof(E));
}
// (128 channels of bf16 spill 42 registers at two a SIMD and are faster all the same: 16 x 1500 rows, backward 435 and 451 us)
template <typename E> constexpr int grad_q_waves(int dp) {
  return Elem<E>::kPlanes == 3 ? (dp <= 32 ? 2 : 1) : dp * (int)sizeof(E) <= 64 ? 3 : dp * (int)sizeof(E) <= 256 ? 2 : 1;
}
template <typename E> constexpr int grad_kv_waves(int dp) {
  return Elem<E>::kPlanes == 3 ? (dp <= 32 ? 2 : 1) : dp * (int)sizeof(E) <= 128 ? 2 : 1;
}
// a lane's pieces of one row: a column of a B operand
template <typename E, int DP> struct Column { typename Frag<E>::type v[Shape<E, DP>::kPlanes][Shape<E, DP>::kSteps]; };

__device__ inline floatx16 mma(bf16x8 a, bf16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx16 mma(floatx4 a, floatx4 b, floatx16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

__device__ inline floatx16 zero16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

__device__ inline uint32_t pack_bf16(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
// two floats as the bf16 next to them; what that leaves stays in x, y (exact: it has fewer bits)
__device__ inline uint32_t take_bf16(float& x, float& y) {
  const uint32_t b = pack_bf16(x, y);
  x -= __uint_as_float(b << 16);
  y -= __uint_as_float(b & 0xffff0000u);
  return b;
}

// The same for weights, which are finite (a row that is not is taken again): what is left in one instruction each, x - 1 hi and
// exact too.  (-1 and 0 in either order, from registers: as constants of a packed operand they might not be what they are here.)
__device__ inline uint32_t take_weights(float& x, float& y) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const uint32_t b = pack_bf16(x, y);
  uint32_t first = 0x0000bf80u, second = 0xbf800000u;
  asm("" : "+s"(first));
  asm("" : "+s"(second));
  const bf16x2 h = __builtin_bit_cast(bf16x2, b);
  x = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), x, false);
  y = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), y, false);
  return b;
}

// The lane's pieces of a row (a column of a B operand), straight from memory; zeros where the row or the
// channels do not exist.
template <typename E, int DP>
__device__ inline void load_row(Column<E, DP>& f, const typename Elem<E>::Memory* row, bool ok, int dim, bool negate = false) {
  using S = Shape<E, DP>;
  const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    const int c = (2 * s + half) * S::kPiece;
    uintx4 v = {0, 0, 0, 0}, w = {0, 0, 0, 0};
    if (ok && c < dim) {
      v = *(const uintx4*)(row + c);
      if constexpr (S::kPlanes == 3) w = *(const uintx4*)(row + c + 4);
    }
    if (negate) {
      v ^= sizeof(typename S::Memory) == 2 ? 0x80008000u : 0x80000000u;
      if constexpr (S::kPlanes == 3) w ^= 0x80000000u;
    }
    if constexpr (S::kPlanes == 3) {
      floatx4 x = __builtin_bit_cast(floatx4, v), y = __builtin_bit_cast(floatx4, w);
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        uintx4 b;
        float t[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = take_bf16(t[2 * i], t[2 * i + 1]);
        x = floatx4{t[0], t[1], t[2], t[3]};
        y = floatx4{t[4], t[5], t[6], t[7]};
        f.v[n][s] = __builtin_bit_cast(bf16x8, b);
      }
    } else {
      f.v[0][s] = __builtin_bit_cast(typename Frag<E>::type, v);
    }
  }
}
// the row's sum of x y, a share in each half of the wavefront
template <typename T, int DP> __device__ inline float row_dot(const T* x, const T* y, bool ok, int dim) {
  using S = Shape<T, DP>;
  const int half = (threadIdx.x >> 5) & 1;
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    const int c = (2 * s + half) * S::kPiece;
    Pack<T, S::kPiece> a, b;
    a.fill(0);
    b.fill(0);
    if (ok && c < dim) {
      a.load(x + c);
      b.load(y + c);
    }
#pragma unroll
    for (int e = 0; e < S::kPiece; ++e) sum = fmaf(to_f32(a.v[e]), to_f32(b.v[e]), sum);
  }
  return sum + __shfl_xor(sum, 32, 64);
}

// Keeps the compiler from moving instructions across.  It otherwise reads each fragment right in front of the
// matrix instruction that uses it (fewer registers) and waits for LDS every time: eight times 130 cycles in
// front of 256 cycles of products.  Where the fragments of a product are 64 registers and more (rows of 256 bytes), reading
// them ahead costs spills instead, and the products are long enough: 16 x 1500 rows, window 512, 8 heads over 4 of 128, ahead
// and not: bf16 forward 117 and 93 us, backward 461 and 451; fp32 backward 2700 and 2037; 64 channels: 56 and 55, 198 and 198.
__device__ inline void in_order() { __builtin_amdgcn_sched_barrier(0); }

template <typename E, int DP> struct Ahead { static constexpr bool value = DP * (int)sizeof(typename Elem<E>::Lds) < 256; };

// The fragments of 32 rows of a tile as the left operand of tile rows . column
template <typename E, int DP> struct RowFrags {
  using S = Shape<E, DP>;
  typename Frag<E>::type v[S::kPlanes][S::kSteps];
  __device__ inline void load(const typename S::Lds* tile) {
    const int lane = threadIdx.x & 63;
    const typename S::Lds* at = tile + (lane & 31) * S::kPitch + (lane >> 5) * S::kPiece;
#pragma unroll
    for (int n = 0; n < S::kPlanes; ++n)
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) v[n][s] = *(const typename Frag<E>::type*)(at + n * S::kPlane + 2 * s * S::kPiece);
  }
};
// the planes whose products count, small ones first
constexpr int kPairs = 6, kPairA[kPairs] = {0, 1, 2, 0, 1, 0}, kPairB[kPairs] = {2, 1, 0, 1, 0, 0};
// two products whose steps alternate, so that none waits for the one before it
template <typename E, int DP>
__device__ inline void rows_times(const RowFrags<E, DP>& a, const Column<E, DP>& x, floatx16& ax, const RowFrags<E, DP>& b,
    const Column<E, DP>& y, floatx16& by) {
  constexpr int first = Elem<E>::kPlanes == 3 ? 0 : kPairs - 1;
#pragma unroll
  for (int n = first; n < kPairs; ++n)
#pragma unroll
    for (int s = 0; s < Shape<E, DP>::kSteps; ++s) {
      ax = mma(a.v[kPairA[n]][s], x.v[kPairB[n]][s], ax);
      by = mma(b.v[kPairA[n]][s], y.v[kPairB[n]][s], by);
    }
}
template <typename E, int DP>
__device__ inline void rows_times(const RowFrags<E, DP>& a, const Column<E, DP>& x, floatx16& ax) {
  constexpr int first = Elem<E>::kPlanes == 3 ? 0 : kPairs - 1;
#pragma unroll
  for (int n = first; n < kPairs; ++n)
#pragma unroll
    for (int s = 0; s < Shape<E, DP>::kSteps; ++s) ax = mma(a.v[kPairA[n]][s], x.v[kPairB[n]][s], ax);
}

__device__ inline shortx4 read_transposed(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)(p));
}

// The fragments of 32 rows of a tile, by channel, for  acc[block][channel][column] += sum over the rows of
// tile[row][channel] * w[row][column], w as an accumulator of rows_times holds it.  bf16: w is rounded to bf16 (half a
// step, 2^-9 of each weight, as the tile's own elements are); statistics and sums stay in 32 bits.  FINE: what the rounding
// left is multiplied too, rounded by itself, so that a weight is 2^-18 off at most.
template <typename E, int DP> struct ColumnFrags {            // (bf16 and planes)
  using S = Shape<E, DP>;
  bf16x8 v[S::kPlanes][2][S::kBlocks];
  __device__ inline void load(const uint16_t* tile) {
    const int lane = threadIdx.x & 63;
    // 16 lanes read 4 rows of 16 channels and get them back by channel
    const uint16_t* at = tile + ((lane >> 5) * 4 + ((lane >> 2) & 3)) * S::kPitch + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int n = 0; n < S::kPlanes; ++n)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d) {
          struct { shortx4 lo, hi; } a = {read_transposed(at + n * S::kPlane + 16 * s * S::kPitch + 32 * d),
                                          read_transposed(at + n * S::kPlane + (16 * s + 8) * S::kPitch + 32 * d)};
          v[n][s][d] = __builtin_bit_cast(bf16x8, a);
        }
  }
  template <bool FINE = false> __device__ inline void times(floatx16 (&acc)[S::kBlocks], const floatx16& w) const {
    constexpr int kParts = S::kPlanes == 3 ? 3 : FINE ? 2 : 1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 part[kParts];
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = w[8 * s + i];
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        uintx4 b;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = kParts == 2 ? take_weights(t[2 * i], t[2 * i + 1]) : take_bf16(t[2 * i], t[2 * i + 1]);
        part[n] = __builtin_bit_cast(bf16x8, b);
      }
      if constexpr (S::kPlanes == 3) {
#pragma unroll
        for (int n = 0; n < kPairs; ++n)
#pragma unroll
          for (int d = 0; d < S::kBlocks; ++d) acc[d] = mma(v[kPairA[n]][s][d], part[kPairB[n]], acc[d]);
      } else {
#pragma unroll
        for (int n = 0; n < kParts; ++n)
#pragma unroll
          for (int d = 0; d < S::kBlocks; ++d) acc[d] = mma(v[0][s][d], part[n], acc[d]);
      }
    }
  }
};
template <int DP> struct ColumnFrags<float, DP> {
  using S = Shape<float, DP>;
  float v[16][S::kBlocks];
  __device__ inline void load(const float* tile) {
    const int lane = threadIdx.x & 63;
    const float* at = tile + (lane >> 5) * 4 * S::kPitch + (lane & 31);
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d) v[r][d] = at[(8 * (r >> 2) + (r & 3)) * S::kPitch + 32 * d];
  }
  template <bool = false> __device__ inline void times(floatx16 (&acc)[S::kBlocks], const floatx16& w) const {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[r][d], w[r], acc[d], 0, 0, 0);
  }
};

// For a branch between a matrix product and the code that reads its result.  The compiler counts the wait states
// that an accumulator needs before it is read, but where a short block lies on one of two paths it counts along
// that path only, and the other path reads the last registers too early (the last key of a tile came out without
// its last channels).  So the conditions of such a branch are formed before the product (`decided`: a value
// the compiler cannot put off), and the branch that is seldom taken waits by itself.
__device__ inline bool decided(bool x) {
  int v = __builtin_amdgcn_readfirstlane(x);
  asm volatile("" : "+s"(v));
  return v != 0;
}
__device__ inline void settle() { asm volatile("s_nop 15\n\ts_nop 3"); }

// Bits 0 .. n - 1
__device__ inline uint32_t first_bits(int n) { return n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u; }
// x where the lane's bit of accumulator row r is set, `other` (as bits) elsewhere; `bits` has been moved right by 4 in the
// upper half of the wavefront.  A bit test and a select (the compiler
// makes an and, a compare and a select of it, and waits between the last two); a NaN in x does not come through.
__device__ inline float where_seen(uint32_t bits, int r, float x, uint32_t other) {
  const int n = 8 * (r >> 2) + (r & 3);
  const uint32_t keep = (uint32_t)(((int32_t)(bits << (31 - n))) >> 31);
  return __uint_as_float((__float_as_uint(x) & keep) | (other & ~keep));
}

// A tile of ROWS rows on its way from memory to LDS: the loads of the next tile are issued before the current
// one is used and wait in registers.  A thread's pieces keep their byte offsets from the tile's first row, so
// a tile costs one scalar address; a row that does not exist (or is masked) gets an offset behind the
// buffer, for which the hardware returns zeros without reading.
constexpr uint32_t kNowhere = 0xfffffff0u, kBufferBytes = 0x80000000u;

__device__ inline __amdgpu_buffer_rsrc_t buffer_at(const void* base) {
  const uint64_t u = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), (short)0, (int)kBufferBytes, 0x00020000);
}

// EVEN: rows a constant stride apart; the pieces of a thread are then too, and all but the first offset
// are scalars (where the threads of a row divide the workgroup).
template <typename E, int DP, int ROWS, int THREADS, bool EVEN> struct Staged {
  using S = Shape<E, DP>;
  using T = typename S::Memory;
  static constexpr int kEach = ROWS * S::kPieces / THREADS;
  static_assert(kEach * THREADS == ROWS * S::kPieces, "whole pieces a thread");
  static constexpr bool kScalar = EVEN && THREADS % S::kPieces == 0;
  uintx4 v[kEach];
  uint32_t at[kScalar ? 1 : kEach];
  uint32_t apart;
  __device__ static inline int row_of(int tid, int i) {
    return kScalar ? tid / S::kPieces + i * (THREADS / S::kPieces) : (tid + i * THREADS) / S::kPieces;
  }
  // offset(r): elements from the tile's first row to row r
  template <typename Offset> __device__ inline void init(int tid, int dim, Offset offset) {
#pragma unroll
    for (int i = 0; i < (kScalar ? 1 : kEach); ++i) {
      const int n = tid + i * THREADS, r = n / S::kPieces, c = (n % S::kPieces) * S::kMemoryPiece;
      at[i] = c < dim ? (uint32_t)(offset(r) + c) * (uint32_t)sizeof(T) : kNowhere;
    }
    apart = __builtin_amdgcn_readfirstlane(kScalar ? offset(THREADS / S::kPieces) * (int)sizeof(T) : 0);
  }
  __device__ inline uintx4 piece(__amdgpu_buffer_rsrc_t buf, int i, bool ok) const {
    const uint32_t o = at[kScalar ? 0 : i];
    return __builtin_amdgcn_raw_buffer_load_b128(buf, ok ? o : kNowhere, kScalar ? i * apart : 0, 0);
  }
  // the tile's first `rows` rows
  __device__ inline void load(const T* base, int tid, int rows) {
    const __amdgpu_buffer_rsrc_t buf = buffer_at(base);
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = piece(buf, i, row_of(tid, i) < rows);
  }
  __device__ inline void load_live(const T* base, int tid, uint64_t live) {
    const __amdgpu_buffer_rsrc_t buf = buffer_at(base);
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = piece(buf, i, live >> row_of(tid, i) & 1);
  }
  __device__ inline void store(typename S::Lds* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = (kScalar ? tid : tid + i * THREADS) % S::kPieces * S::kMemoryPiece;
      typename S::Lds* at = tile + row_of(tid, i) * S::kPitch + c;
      if constexpr (S::kPlanes == 3) {
        static_assert(ROWS * S::kPitch == S::kPlane, "64 rows");
        floatx4 x = __builtin_bit_cast(floatx4, v[i]);
        float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int n = 0; n < 3; ++n) {
          typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
          const uint32_t b0 = take_bf16(t[0], t[1]), b1 = take_bf16(t[2], t[3]);
          *(uintx2*)(at + n * S::kPlane) = uintx2{b0, b1};
        }
      } else {
        *(uintx4*)at = v[i];
      }
    }
  }
};

// The keys of a tile that exist and that `mask` keeps, bit i for key j0 + i: the same in every wavefront
template <int KEYS> __device__ inline uint64_t live_keys(const unsigned char* mask, int j0, int keys) {
  const int lane = threadIdx.x & 63;
  return __ballot(lane < KEYS && j0 + lane < keys && mask[j0 + lane] != 0);
}

__device__ inline float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}
__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}
__device__ inline bool finite(float x) { return fabsf(x) < __builtin_inff(); }

// orders the LDS accesses of one wavefront across its lanes
__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Work items in an order that keeps neighbours on one XCD: workgroups go round the 8 XCDs in turn, so of every 64
// items each XCD takes 8 in a row, whose windows overlap in its L2.  (Not an eighth of all items: the tiles of a
// causal sequence grow towards its end.)  Which XCD begins changes with the head, so that what the last set
// lacks is spread.  Grids are padded to whole sets of 64.
__device__ inline int near_item(int x) { return (x & ~63) + ((x + blockIdx.y) & 7) * 8 + ((x >> 3) & 7); }
inline int64_t whole_sets(int64_t n) { return n <= 64 ? n : (n + 63) & ~(int64_t)63; }
__device__ inline int item_of(int x, int n) { return n <= 64 ? x : near_item(x); }

// One sequence as the kernels see it
struct Seq {
  int q0, queries, k0, keys, room;      // room: key rows up to the next sequence
  __device__ inline int shift() const { return keys - queries; }    // position of query 0
};
__device__ inline Seq sequence(const ocnn_attention_params& p, int b) {
  Seq s;
  s.q0 = clamped(p.q_offsets, b, p.rows_q);
  s.queries = max(clamped(p.q_offsets, b + 1, p.rows_q) - s.q0, 0);
  s.k0 = clamped(p.k_offsets, b, p.rows_k);
  s.room = max(clamped(p.k_offsets, b + 1, p.rows_k) - s.k0, 0);
  s.keys = p.k_lengths ? min(max(p.k_lengths[b], 0), s.room) : s.room;
  return s;
}
// the keys a query at position pos sees through the window: [lo, hi)
__device__ inline int window_lo(const ocnn_attention_params& p, int pos) { return p.left < 0 ? 0 : max(pos - p.left, 0); }
__device__ inline int window_hi(const ocnn_attention_params& p, int pos, int keys) {
  return p.right < 0 ? keys : max(min(pos + p.right + 1, keys), 0);
}

// ---- forward -------------------------------------------------------------------------------------------
// QW = 4: a workgroup takes 128 packed rows, 32 a wavefront; tiles of 64 keys go through LDS once for all
// four.  QW = 2: 64 packed rows, and each half of a tile has a wavefront of its own for them; joined at the end.  QW = 1 (few rows a sequence): 32 packed rows, and the wavefronts take every fourth tile of 32
// keys each on their own, joined at the end.  Where rows x key heads leave compute units empty, the
// tiles are dealt out over `splits` workgroups, joined by attention_join_kernel.
// Measured: sequences of 8192 and 22184 rows, window 2047, 8 heads of 64, bf16: 168-172 us in a run of some hundred calls
// (700 TFLOP/s), 175-205 in the first ones after a pause, when the chip's clock is lower.  A 32 x 32 tile is 16 each of
// exponentials, multiply-adds and additions and 8 conversions a lane, about 420 cycles, against 256 of products: 61 % and 37 % of
// the SIMD cycles, but only 18 % both at once, so the two take turns.  One query of 262147 keys, 16 heads over 2 of 128, bf16:
// 45 us, 5.9 TB/s of keys and values, and 6 us for the join.
template <typename E, int DP, int QW> struct ForwardShape {
  static constexpr int kKeys = QW == 1 ? 32 : 64;
  static constexpr int kTile = kKeys * Shape<E, DP>::kPitch * Shape<E, DP>::kPlanes;
  static constexpr int kBuffers = QW == 1 ? 4 : 2;            // double buffer, or one a wavefront
  static constexpr size_t kJoin = (4 - QW) * (size_t)(DP / 32) * 16 * 64 * 4;
  static constexpr size_t kTiles = (size_t)kBuffers * 2 * kTile * sizeof(typename Shape<E, DP>::Lds);
  static constexpr size_t kLds = kTiles > kJoin ? kTiles : kJoin;
};

struct Softmax { float m, l; };

// One row again, visible terms only: for rows whose result is not finite.  The products above multiply the
// values of keys that a row does not see by a probability of zero, which is no zero where such a value is
// infinite or NaN.
template <typename T, int DP, int QW>
__device__ __forceinline__ void forward_row_again(const AttnArgs& a, const Seq& s, int kv, int row, int split, int tiles, int sink_tiles,
    int t0, Softmax* st, float (&o)[(DP + 63) / 64]) {
  constexpr int key_tile = QW == 1 ? 32 : 64, kWays = QW == 1 ? 4 : 1;
  const ocnn_attention_params& p = a.p;
  const int lane = threadIdx.x & 63;
  const int token = row / a.group, head = kv * a.group + row % a.group;
  const int pos = token + s.shift(), lo = window_lo(p, pos), hi = window_hi(p, pos, s.keys);
  const T* q = (const T*)p.q + (int64_t)(s.q0 + token) * p.q_row + head * p.q_head;
  float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i) o[i] = 0.0f;
  for (int n = 0;; ++n) {
    const int v = (n / kWays * a.splits + split) * kWays + n % kWays;      // the tiles of this workgroup in turn
    if (v - n % kWays >= tiles) break;
    if (v >= tiles) continue;
    const int j0 = (v < sink_tiles ? v : t0 + v - sink_tiles) * key_tile;
    const int j = j0 + lane;
    bool see = lane < key_tile && j < hi && (j >= lo || j < p.sinks);
    if (see && p.key_mask) see = p.key_mask[s.k0 + j] != 0;
    float x = -__builtin_inff();
    if (see) {
      const T* k = (const T*)p.k + (int64_t)(s.k0 + j) * p.k_row + kv * p.k_head;
      float dot = 0.0f;
      for (int c = 0; c < p.dim; ++c) dot = fmaf(to_f32(q[c]), to_f32(k[c]), dot);
      x = dot * (p.scale < 0.0f ? -a.scale2 : a.scale2);
    }
    uint64_t left = __ballot(see);
    if (!left) continue;
    // (fmax drops a NaN: it has to reach the sum)
    const float top = fmaxf(m, wave_max(x)), base = top == -__builtin_inff() ? 0.0f : top;
    const float shrink = exp2f(m - base), e = see ? exp2f(x - base) : 0.0f;
    l = l * shrink + wave_sum(e);
    m = top;
    if (l != l) {                             // a NaN stays, in every channel.  (m: the joining kernel must not weigh it by zero)
#pragma unroll
      for (int i = 0; i < (DP + 63) / 64; ++i) o[i] = l;
      st->m = __builtin_inff();
      st->l = l;
      return;
    }
#pragma unroll
    for (int i = 0; i < (DP + 63) / 64; ++i) o[i] *= shrink;
    while (left) {
      const int jj = __ffsll((unsigned long long)left) - 1;
      left &= left - 1;
      const float w = __shfl(e, jj, 64);
      const T* vr = (const T*)p.v + (int64_t)(s.k0 + j0 + jj) * p.v_row + kv * p.v_head;
#pragma unroll
      for (int i = 0; i < (DP + 63) / 64; ++i)
        if (lane + 64 * i < p.dim) o[i] = fmaf(w, to_f32(vr[lane + 64 * i]), o[i]);
    }
  }
  st->m = m;
  st->l = l;
}

template <typename E, int DP, int QW, bool SPLIT>
__global__ void __launch_bounds__(256, forward_waves<E>(DP)) attention_kernel(AttnArgs a) {
  using S = Shape<E, DP>;
  using T = typename S::Memory;
  using L = typename S::Lds;
  using F = ForwardShape<E, DP, QW>;
  constexpr int kRows = 32 * QW, kShift = Log2<kRows>::value;
  __shared__ __attribute__((aligned(16))) char lds[F::kLds];
  __shared__ Softmax stats[4][32];
  const ocnn_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  // (splits first: workgroups go round the XCDs in turn, and work items that no sequence owns must not be every second one)
  const int kv = blockIdx.y, split = SPLIT ? blockIdx.x : 0, work_id = SPLIT ? (int)blockIdx.z : item_of(blockIdx.x, gridDim.x);
  const int b = locate_packed(p.q_offsets, p.n_seq, p.rows_q, work_id, kShift, a.group);
  const int q_begin = clamped(p.q_offsets, b, p.rows_q);
  const int64_t tile = (int64_t)work_id - (((int64_t)q_begin * a.group >> kShift) + b);
  Seq s;
  if (b >= p.n_seq) {
    s.q0 = q_begin; s.queries = p.rows_q - q_begin; s.k0 = 0; s.keys = 0; s.room = 0;
  } else {
    s = sequence(p, b);
  }
  const int64_t row0 = tile * kRows;
  const int rows = s.queries * a.group;
  if (tile < 0 || row0 >= rows) return;
  const int share = wave / QW, first_row = (int)row0 + wave % QW * 32;     // of the wavefronts of the same 32 rows
  const int row = first_row + col;
  const bool have = row < rows;
  const int token = have ? row / a.group : 0, in_group = have ? row - token * a.group : 0;
  const int head = kv * a.group + in_group;
  const int64_t out_at = (int64_t)(s.q0 + token);

  if (b >= p.n_seq) {                       // rows behind the last sequence
    if (SPLIT) {
      if (have && half == 0 && share == 0) {
        float* ml = a.part_ml + (((int64_t)split * p.rows_q + out_at) * p.heads + head) * 2;
        ml[0] = -__builtin_inff();
        ml[1] = -1.0f;                      // (what the joining kernel knows them by)
      }
      return;
    }
    if (a.fill && have && share == 0) {
      T* o = (T*)a.out + out_at * a.out_row + head * a.out_head;
      for (int c = half * S::kMemoryPiece; c < p.dim; c += 2 * S::kMemoryPiece) *(uintx4*)(o + c) = uintx4{0, 0, 0, 0};
      if (a.lse && half == 0) a.lse[out_at * p.heads + head] = -__builtin_inff();
    }
    return;
  }

  // what this lane's row sees, and what the wavefront's and the workgroup's rows see
  const int pos = token + s.shift();
  const int lo = have ? window_lo(p, pos) : 0, hi = have ? window_hi(p, pos, s.keys) : 0;
  const int sinks = have ? p.sinks : 0;
  const int last_row = min(first_row + 31, rows - 1);
  int w_lo = 0, w_hi = 0, all_lo = 0, all_hi = 0;            // some row sees / every row sees
  if (first_row < rows) {
    const int pa = first_row / a.group + s.shift(), pb = last_row / a.group + s.shift();
    w_lo = window_lo(p, pa);
    w_hi = window_hi(p, pb, s.keys);
    all_lo = window_lo(p, pb);
    all_hi = first_row + 31 < rows ? window_hi(p, pa, s.keys) : 0;
  }
  const int block_last = min((int)row0 + kRows, rows) - 1;
  const int b_lo = window_lo(p, (int)row0 / a.group + s.shift());
  const int b_hi = window_hi(p, block_last / a.group + s.shift(), s.keys);
  constexpr int KT = F::kKeys;
  const int t0 = b_lo / KT, t1 = max((b_hi + KT - 1) / KT, t0);
  // tiles of the sinks in front of the window's: their keys are visible up to what causality allows
  const int sink_tiles = min((min(p.sinks, b_hi) + KT - 1) / KT, t0);
  const int tiles = sink_tiles + t1 - t0;
  auto tile_key = [&](int v) { return (v < sink_tiles ? v : t0 + v - sink_tiles) * KT; };

  Column<E, DP> q;
  load_row<E, DP>(q, (const T*)p.q + out_at * p.q_row + head * p.q_head, have, p.dim, p.scale < 0.0f);
  floatx16 o[S::kBlocks];
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d) o[d] = zero16();
  float m = -__builtin_inff(), l = 0.0f;

  const T* kbase = (const T*)p.k + (int64_t)s.k0 * p.k_row + kv * p.k_head;
  const T* vbase = (const T*)p.v + (int64_t)s.k0 * p.v_row + kv * p.v_head;
  const unsigned char* mask = p.key_mask ? p.key_mask + s.k0 : nullptr;

  // the keys j0 .. j0 + 31 that this lane's row sees, as bits for where_seen
  auto seen_bits = [&](int j0, uint32_t live) {
    return (live & first_bits(hi - j0) & (~first_bits(lo - j0) | first_bits(sinks - j0))) >> (4 * half);
  };
  auto rebase = [&](float to) {
    const float shrink = __builtin_amdgcn_exp2f(m - (to == -__builtin_inff() ? 0.0f : to));
    l *= shrink;
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= shrink;
    m = to;
  };
  // The tile's keys, from j0 on, against this wavefront's rows: scores -> probabilities -> o.  The exponentials are
  // taken against a base that follows the row's running maximum from behind: it is set by the first keys a
  // row sees, and raised after a tile whose sum has passed 2^10.  32-bit sums and bf16 weights hold larger
  // powers without loss, so most tiles need neither a maximum nor a rescaling, and the second product does
  // not wait for a vote.  Only a weight beyond 2^100 of the base is too much: the tile says so, and the
  // workgroup takes all its tiles again, with the maximum of each (careful).
  // Probabilities as operands: two bf16 for few rows, which wait for memory; one for tiles of them.  Off 64 bits, relative to
  // the result (whose own rounding is 0.0016), and us, with one and with two: one query of 262147 keys 0.0021 0.0016, 64.1 62.7;
  // 32 of 2048 keys 0.00041 0.00033, 17.1 17.7; two sequences of 8192 and 22184 rows, window 2047, 8 heads of 64: 0.0021
  // 0.0016, but 178 229.
  constexpr bool kFew = QW == 1;
  constexpr int N = QW == 4 ? 2 : 1;          // times 32 keys
  bool careful = QW == 1, over = false;       // (QW = 1 waits for memory: careful from the start)
  auto keys = [&](const L* kt, const L* vt, int j0, uint64_t live) {
    const uint64_t all = N == 2 ? ~0ull : 0xffffffffull;
    const bool masked = decided((j0 < all_lo) | (j0 + 32 * N > all_hi) | ((live & all) != all));
    const bool measure = careful || decided(__any(m == -__builtin_inff()));
    floatx16 x[N];
    if constexpr (N == 2) {
      RowFrags<E, DP> ka, kb;
      ka.load(kt);
      kb.load(kt + 32 * S::kPitch);
      if constexpr (Ahead<E, DP>::value) in_order();
      x[0] = x[1] = zero16();
      rows_times<E, DP>(ka, q, x[0], kb, q, x[1]);
    } else {
      RowFrags<E, DP> ka;
      ka.load(kt);
      if constexpr (Ahead<E, DP>::value) in_order();
      x[0] = zero16();
      rows_times<E, DP>(ka, q, x[0]);
    }
    if (masked) {
      settle();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t seen = seen_bits(j0 + 32 * i, (uint32_t)(live >> (32 * i)));
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] = where_seen(seen, r, x[i][r], 0xff800000u);
      }
    }
    if (measure) {
      settle();
      float top = x[0][0];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, x[i][r]);
      top *= a.scale2;
      rebase(fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64))));
    }
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float sums[2 * N];
    ColumnFrags<E, DP> vf[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {             // the values of one half arrive while the other half's weights are formed
      vf[i].load(vt + i * 32 * S::kPitch);
      if (i) vf[0].template times<kFew>(o, x[0]);
      sums[2 * i] = sums[2 * i + 1] = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[i][r] = __builtin_amdgcn_exp2f(fmaf(x[i][r], a.scale2, -base));
        sums[2 * i + (r & 1)] += x[i][r];
      }
    }
    vf[N - 1].template times<kFew>(o, x[N - 1]);
    float sum = sums[0] + sums[1];
    if (N == 2) sum += sums[2] + sums[3];
    l += sum;
    if (QW != 1 && __any(!(sum <= 1024.0f))) {
      settle();
      over = over || !(sum <= 1.2676506e30f);
      const float most = fmaxf(sum, __shfl_xor(sum, 32, 64));
      rebase(most > 1024.0f && most <= 1.2676506e30f ? m + rintf(__builtin_amdgcn_logf(most)) : m);
    }
  };
  auto reach = [&](int j0) { return (j0 < w_hi) & ((j0 + 32 * N > w_lo) | (j0 < p.sinks)); };
  if (!have) m = 0.0f;                        // (does not ask for a maximum)

  constexpr int kThreads = QW == 1 ? 64 : 256;
  const int mine = QW == 1 ? lane : tid;
  Staged<E, DP, KT, kThreads, true> sk, sv;
  sk.init(mine, p.dim, [&](int r) { return r * (int)p.k_row; });
  sv.init(mine, p.dim, [&](int r) { return r * (int)p.v_row; });
  uint64_t next = ~0ull;
  auto fetch = [&](int v) {
    const int j0 = tile_key(v);
    if (mask) {
      next = live_keys<KT>(mask, j0, s.keys);
      sk.load_live(kbase + (int64_t)j0 * p.k_row, mine, next);
      sv.load_live(vbase + (int64_t)j0 * p.v_row, mine, next);
    } else {
      sk.load(kbase + (int64_t)j0 * p.k_row, mine, s.keys - j0);
      sv.load(vbase + (int64_t)j0 * p.v_row, mine, s.keys - j0);
    }
  };
  if constexpr (QW != 1) {
    const int step = SPLIT ? a.splits : 1;
#pragma unroll 1
    for (;;) {
      if (split < tiles) fetch(split);
      L* kt = (L*)lds;
#pragma unroll 1
      for (int v = split; v < tiles; v += step) {
        L* vt = kt + F::kTile;
        sk.store(kt, tid);
        sv.store(vt, tid);
        const uint64_t live = next;
        __syncthreads();                      // (the other buffer's readers are done: they passed the last barrier)
        if (v + step < tiles) fetch(v + step);
        const int part = QW == 2 ? share * 32 : 0, j0 = tile_key(v) + part;
        if (reach(j0)) keys(kt + part * S::kPitch, vt + part * S::kPitch, j0, live >> part);
        kt = kt == (L*)lds ? (L*)lds + 2 * F::kTile : (L*)lds;
      }
      if (careful || !__syncthreads_or(over)) break;
      careful = true;
      m = have ? -__builtin_inff() : 0.0f;
      l = 0.0f;
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d) o[d] = zero16();
    }
  } else {
    L* kt = (L*)lds + wave * 2 * F::kTile;
    L* vt = kt + F::kTile;
    // (the splits take turns: at any time the workgroups together read one stretch of the keys, which spreads
    // over all memory channels; shares of their own, a power of two apart, met on a few of them)
    const int first = split * 4 + wave, step = 4 * (SPLIT ? a.splits : 1);
    if (first < tiles) fetch(first);
    for (int v = first; v < tiles; v += step) {
      wave_lds_fence();
      sk.store(kt, lane);
      sv.store(vt, lane);
      const uint64_t live = next;
      wave_lds_fence();
      if (v + step < tiles) fetch(v + step);
      const int j0 = tile_key(v);
      if (reach(j0)) keys(kt, vt, j0, live);
    }
  }
  if (!have) m = -__builtin_inff();
  l += __shfl_xor(l, 32, 64);

  if constexpr (QW != 4) {                    // the wavefronts' shares, joined in the first one
    constexpr int kWays = 4 / QW;
    const int w0 = wave % QW;
    if (half == 0) stats[wave][col] = Softmax{m, l};
    __syncthreads();
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWays; ++w) top = fmaxf(top, stats[w0 + QW * w][col].m);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    const float mine = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWays; ++w) sum += stats[w0 + QW * w][col].l * __builtin_amdgcn_exp2f(stats[w0 + QW * w][col].m - base);
    float* join = (float*)lds;
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[d][r] *= mine;
        if (share) join[(((wave - QW) * S::kBlocks + d) * 16 + r) * 64 + lane] = o[d][r];
      }
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int w = 0; w + 1 < kWays; ++w)
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] += join[(((w0 + QW * w) * S::kBlocks + d) * 16 + r) * 64 + lane];
    m = top;
    l = sum;
  }

  float worst = 0.0f;                         // not finite where any of them is not
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) worst += fabsf(o[d][r]);
  worst += __shfl_xor(worst, 32, 64);
  const bool good = finite(worst) && finite(l);
  const int64_t at_row = out_at * p.heads + head;
  if (have && good) {
    if (SPLIT) {
      float* po = a.part_o + ((int64_t)split * p.rows_q * p.heads + at_row) * p.dim;
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 32 * d + 8 * i + 4 * half;
          if (c < p.dim) *(floatx4*)(po + c) = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        }
      if (half == 0) {
        float* ml = a.part_ml + ((int64_t)split * p.rows_q * p.heads + at_row) * 2;
        ml[0] = m;
        ml[1] = l;
      }
    } else {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      T* po = (T*)a.out + out_at * a.out_row + head * a.out_head;
#pragma unroll
      for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 32 * d + 8 * i + 4 * half;
          Pack<T, 4> x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x.v[e] = from_f32<T>(o[d][4 * i + e] * inv);
          if (c < p.dim) x.store(po + c);
        }
      if (a.lse && half == 0) a.lse[at_row] = l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -__builtin_inff();
    }
  }
  uint32_t bad = (uint32_t)__ballot(have && !good);
  while (bad) {
    const int c = __ffs(bad) - 1;
    bad &= bad - 1;
    const int r = __shfl(row, c, 64);
    Softmax st;
    float oo[(DP + 63) / 64];
    forward_row_again<T, DP, QW>(a, s, kv, r, split, tiles, sink_tiles, t0, &st, oo);
    const int tk = r / a.group, hd = kv * a.group + r % a.group;
    const int64_t at = (int64_t)(s.q0 + tk) * p.heads + hd;
#pragma unroll
    for (int i = 0; i < (DP + 63) / 64; ++i) {
      const int ch = lane + 64 * i;
      if (ch >= p.dim) continue;
      if (SPLIT) a.part_o[((int64_t)split * p.rows_q * p.heads + at) * p.dim + ch] = oo[i];
      else ((T*)a.out)[(int64_t)(s.q0 + tk) * a.out_row + hd * a.out_head + ch] = from_f32<T>(st.l == 0.0f ? 0.0f : oo[i] / st.l);
    }
    if (lane == 0) {
      if (SPLIT) {
        float* ml = a.part_ml + ((int64_t)split * p.rows_q * p.heads + at) * 2;
        ml[0] = st.m;
        ml[1] = st.l;
      } else if (a.lse) {
        a.lse[at] = st.l == 0.0f ? -__builtin_inff() : (st.m + __builtin_amdgcn_logf(st.l)) * kLn2;
      }
    }
  }
}

// o = sum_s exp(m_s - m) o_s / sum_s exp(m_s - m) l_s.  A workgroup joins one row: its 256 threads weigh the (at
// most 256) shares, then 8 groups of 32 lanes, 4 channels each, add theirs up and are added in order.  Measured: 248 rows of 7
// shares 3.9 us, 16 rows of 128 shares of 128 channels 6.2 us: latency of two dependent reads and a launch.
constexpr int kMaxSplits = 256;
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(AttnArgs a) {
  __shared__ float weight[kMaxSplits];
  __shared__ float part[4];
  __shared__ floatx4 sums[8][32];
  const ocnn_attention_params& p = a.p;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t rows = (int64_t)p.rows_q * p.heads, row = blockIdx.x;
  const int token = (int)(row / p.heads), head = (int)(row - (int64_t)token * p.heads);
  float m = -__builtin_inff(), l = 0.0f;
  if (t < a.splits) {
    const float2 ml = *(const float2*)(a.part_ml + (t * rows + row) * 2);
    m = ml.x;
    l = ml.y;
  }
  const bool none = __syncthreads_or(l == -1.0f);       // a row of no sequence
  if (none && !a.fill) return;
  const float wm = wave_max(m);
  if (lane == 0) part[wave] = wm;
  __syncthreads();
  const float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), base = top == -__builtin_inff() ? 0.0f : top;
  // (a share without a visible key does not count, whatever its values are)
  const float w = none || l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - base);
  weight[t] = w;
  l = wave_sum(w == 0.0f ? 0.0f : w * l);
  __syncthreads();
  if (lane == 0) part[wave] = l;
  __syncthreads();
  l = part[0] + part[1] + part[2] + part[3];
  const int group = t >> 5, c = (t & 31) * 4;
  floatx4 o = {0, 0, 0, 0};
  if (c < p.dim)
#pragma unroll 8
    for (int s = group; s < a.splits; s += 8) {
      const floatx4 x = *(const floatx4*)(a.part_o + (s * rows + row) * p.dim + c);
      const float ws = weight[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = ws == 0.0f ? o[e] : fmaf(ws, x[e], o[e]);
    }
  sums[group][t & 31] = o;
  __syncthreads();
  if (group || c >= p.dim) return;
#pragma unroll
  for (int g = 1; g < 8; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += sums[g][t & 31][e];
  Pack<T, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y.v[e] = from_f32<T>(l == 0.0f ? 0.0f : o[e] / l);
  y.store((T*)a.out + (int64_t)token * a.out_row + (int64_t)head * a.out_head + c);
  if (a.lse && t == 0) a.lse[row] = l == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- gradient of the queries ---------------------------------------------------------------------------
// Rows as in the forward kernel (QW = 4); the scores are computed again from lse.  rowsum(dO o) is formed
// here, from the row's own registers, and left for the kernel of the keys.  No atomics: dQ and dK, dV each
// have a kernel that owns their rows, at the price of computing the scores twice.
// Measured: 16 x about 1500 rows, window 512, 8 heads over 4 of 64, bf16: 72 us (VALU 47 %, products 31 % of the SIMD cycles).
template <typename T, int DP>
__device__ __forceinline__ void grad_q_row_again(const AttnArgs& a, const Seq& s, int kv, int row, int t0, int t1, int sink_tiles,
    float lse2, float delta, float (&dq)[(DP + 63) / 64]) {
  const ocnn_attention_params& p = a.p;
  const int lane = threadIdx.x & 63;
  const int token = row / a.group, head = kv * a.group + row % a.group;
  const int pos = token + s.shift(), lo = window_lo(p, pos), hi = window_hi(p, pos, s.keys);
  const T* q = (const T*)p.q + (int64_t)(s.q0 + token) * p.q_row + head * p.q_head;
  const T* go = (const T*)a.grad + (int64_t)(s.q0 + token) * a.grad_row + head * a.grad_head;
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i) dq[i] = 0.0f;
  for (int v = 0; v < sink_tiles + t1 - t0; ++v) {
    const int j0 = (v < sink_tiles ? v : t0 + v - sink_tiles) * 64, j = j0 + lane;
    bool see = j < hi && (j >= lo || j < p.sinks);
    if (see && p.key_mask) see = p.key_mask[s.k0 + j] != 0;
    float ds = 0.0f;
    if (see) {
      const T* k = (const T*)p.k + (int64_t)(s.k0 + j) * p.k_row + kv * p.k_head;
      const T* vr = (const T*)p.v + (int64_t)(s.k0 + j) * p.v_row + kv * p.v_head;
      float dot = 0.0f, dp = 0.0f;
      for (int c = 0; c < p.dim; ++c) {
        dot = fmaf(to_f32(q[c]), to_f32(k[c]), dot);
        dp = fmaf(to_f32(go[c]), to_f32(vr[c]), dp);
      }
      ds = exp2f(fmaf(dot, p.scale < 0.0f ? -a.scale2 : a.scale2, -lse2)) * (dp - delta);
    }
    uint64_t left = __ballot(see);
    if (__any(ds != ds)) {                    // (stays in every channel)
#pragma unroll
      for (int i = 0; i < (DP + 63) / 64; ++i) dq[i] = __builtin_nanf("");
      return;
    }
    while (left) {
      const int jj = __ffsll((unsigned long long)left) - 1;
      left &= left - 1;
      const float w = __shfl(ds, jj, 64);
      const T* kr = (const T*)p.k + (int64_t)(s.k0 + j0 + jj) * p.k_row + kv * p.k_head;
#pragma unroll
      for (int i = 0; i < (DP + 63) / 64; ++i)
        if (lane + 64 * i < p.dim) dq[i] = fmaf(w, to_f32(kr[lane + 64 * i]), dq[i]);
    }
  }
}

template <typename E, int DP, int QW>
__global__ void __launch_bounds__(256, grad_q_waves<E>(DP)) attention_grad_q_kernel(AttnArgs a) {
  using S = Shape<E, DP>;
  using T = typename S::Memory;
  using L = typename S::Lds;
  constexpr int KT = 64, kTile = KT * S::kPitch * S::kPlanes, kRows = 32 * QW, kShift = Log2<kRows>::value;
  constexpr int N = QW == 4 ? 2 : 1;              // times 32 keys
  __shared__ __attribute__((aligned(16))) L lds[2 * 2 * kTile];
  __shared__ float sums[4][32];
  const ocnn_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int kv = blockIdx.y;
  const int work_id = item_of(blockIdx.x, gridDim.x);
  const int b = locate_packed(p.q_offsets, p.n_seq, p.rows_q, work_id, kShift, a.group);
  const int q_begin = clamped(p.q_offsets, b, p.rows_q);
  const int64_t tile = (int64_t)work_id - (((int64_t)q_begin * a.group >> kShift) + b);
  Seq s;
  if (b >= p.n_seq) {
    s.q0 = q_begin; s.queries = p.rows_q - q_begin; s.k0 = 0; s.keys = 0; s.room = 0;
  } else {
    s = sequence(p, b);
  }
  const int64_t row0 = tile * kRows;
  const int rows = s.queries * a.group;
  if (tile < 0 || row0 >= rows) return;
  const int share = wave / QW, first_row = (int)row0 + wave % QW * 32;     // of the wavefronts of the same 32 rows
  const int row = first_row + col;
  const bool have = row < rows;
  const int token = have ? row / a.group : 0, in_group = have ? row - token * a.group : 0;
  const int head = kv * a.group + in_group;
  const int64_t at = (int64_t)(s.q0 + token);
  T* dq_row = (T*)a.dq + at * a.dq_row + head * a.dq_head;
  if (b >= p.n_seq) {
    if (have && share == 0)
      for (int c = half * S::kMemoryPiece; c < p.dim; c += 2 * S::kMemoryPiece) *(uintx4*)(dq_row + c) = uintx4{0, 0, 0, 0};
    return;
  }
  const int pos = token + s.shift();
  const int lo = have ? window_lo(p, pos) : 0, hi = have ? window_hi(p, pos, s.keys) : 0, sinks = have ? p.sinks : 0;
  const int last_row = min(first_row + 31, rows - 1);
  int w_lo = 0, w_hi = 0, all_lo = 0, all_hi = 0;
  if (first_row < rows) {
    const int pa = first_row / a.group + s.shift(), pb = last_row / a.group + s.shift();
    w_lo = window_lo(p, pa);
    w_hi = window_hi(p, pb, s.keys);
    all_lo = window_lo(p, pb);
    all_hi = first_row + 31 < rows ? window_hi(p, pa, s.keys) : 0;
  }
  const int block_last = min((int)row0 + kRows, rows) - 1;
  const int b_lo = window_lo(p, (int)row0 / a.group + s.shift());
  const int b_hi = window_hi(p, block_last / a.group + s.shift(), s.keys);
  const int t0 = b_lo / KT, t1 = max((b_hi + KT - 1) / KT, t0);
  const int sink_tiles = min((min(p.sinks, b_hi) + KT - 1) / KT, t0);
  const int tiles = sink_tiles + t1 - t0;

  Column<E, DP> q, go;
  load_row<E, DP>(go, (const T*)a.grad + at * a.grad_row + head * a.grad_head, have, p.dim);
  float delta = row_dot<T, DP>((const T*)a.fwd + at * a.fwd_row + head * a.fwd_head,
      (const T*)a.grad + at * a.grad_row + head * a.grad_head, have, p.dim);
  load_row<E, DP>(q, (const T*)p.q + at * p.q_row + head * p.q_head, have, p.dim, p.scale < 0.0f);
  const int64_t at_row = at * p.heads + head;
  const float lse = have ? a.lse[at_row] : -__builtin_inff();
  const float lse2 = lse == -__builtin_inff() ? 0.0f : lse * kLog2e;

  floatx16 dq[S::kBlocks];
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d) dq[d] = zero16();
  const T* kbase = (const T*)p.k + (int64_t)s.k0 * p.k_row + kv * p.k_head;
  const T* vbase = (const T*)p.v + (int64_t)s.k0 * p.v_row + kv * p.v_head;
  const unsigned char* mask = p.key_mask ? p.key_mask + s.k0 : nullptr;

  // the keys j0 .. j0 + 31 that this lane's row sees, and as bits for where_seen
  auto visible_bits = [&](int j0, uint32_t live) { return live & first_bits(hi - j0) & (~first_bits(lo - j0) | first_bits(sinks - j0)); };
  auto seen_bits = [&](int j0, uint32_t live) { return visible_bits(j0, live) >> (4 * half); };
  auto reach = [&](int j0) { return (j0 < w_hi) & ((j0 + 32 * N > w_lo) | (j0 < p.sinks)); };
  auto keys = [&](const L* kt, const L* vt, int j0, uint64_t live) {
    const uint64_t all = N == 2 ? ~0ull : 0xffffffffull;
    const bool masked = decided((j0 < all_lo) | (j0 + 32 * N > all_hi) | ((live & all) != all));
    floatx16 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      RowFrags<E, DP> kf, vf;
      kf.load(kt + i * 32 * S::kPitch);
      vf.load(vt + i * 32 * S::kPitch);
      floatx16 dp = zero16();
      x[i] = zero16();
      rows_times<E, DP>(kf, q, x[i], vf, go, dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[i][r] = __builtin_amdgcn_exp2f(fmaf(x[i][r], a.scale2, -lse2)) * (dp[r] - delta);
    }
    ColumnFrags<E, DP> cf[N];
    cf[0].load(kt);
    if (masked) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t seen = seen_bits(j0 + 32 * i, (uint32_t)(live >> (32 * i)));
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] = where_seen(seen, r, x[i][r], 0u);
      }
    }
    if constexpr (N == 2) cf[1].load(kt + 32 * S::kPitch);
    cf[0].template times<kFine>(dq, x[0]);
    if constexpr (N == 2) cf[1].template times<kFine>(dq, x[1]);
  };
  // the share of these keys in rowsum(P dP)
  auto weigh = [&](const L* kt, const L* vt, int j0, uint64_t live) {
    float sum = 0.0f;
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      RowFrags<E, DP> kf, vf;
      kf.load(kt + i * 32 * S::kPitch);
      vf.load(vt + i * 32 * S::kPitch);
      floatx16 dp = zero16(), x = zero16();
      rows_times<E, DP>(kf, q, x, vf, go, dp);
      const uint32_t seen = seen_bits(j0 + 32 * i, (uint32_t)(live >> (32 * i)));
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += where_seen(seen, r, __builtin_amdgcn_exp2f(fmaf(x[r], a.scale2, -lse2)) * dp[r], 0u);
    }
    return sum;
  };
  auto tile_key = [&](int v) { return (v < sink_tiles ? v : t0 + v - sink_tiles) * KT; };
  Staged<E, DP, KT, 256, true> sk, sv;
  sk.init(tid, p.dim, [&](int r) { return r * (int)p.k_row; });
  sv.init(tid, p.dim, [&](int r) { return r * (int)p.v_row; });
  uint64_t next = ~0ull;
  auto fetch = [&](int v) {
    const int j0 = tile_key(v);
    if (mask) {
      next = live_keys<KT>(mask, j0, s.keys);
      sk.load_live(kbase + (int64_t)j0 * p.k_row, tid, next);
      sv.load_live(vbase + (int64_t)j0 * p.v_row, tid, next);
    } else {
      sk.load(kbase + (int64_t)j0 * p.k_row, tid, s.keys - j0);
      sv.load(vbase + (int64_t)j0 * p.v_row, tid, s.keys - j0);
    }
  };
  L* kt = lds;
  auto over = [&](auto use) {
    if (tiles > 0) fetch(0);
    for (int v = 0; v < tiles; ++v) {
      L* vt = kt + kTile;
      sk.store(kt, tid);
      sv.store(vt, tid);
      const uint64_t live = next;
      __syncthreads();
      if (v + 1 < tiles) fetch(v + 1);
      const int part = QW == 2 ? share * 32 : 0, j0 = tile_key(v) + part;
      if (reach(j0)) use(kt + part * S::kPitch, vt + part * S::kPitch, j0, live >> part);
      kt = kt == lds ? lds + 2 * kTile : lds;
    }
  };
  if constexpr (sizeof(T) == 2) {
    int sees = max(hi - lo, 0) + min(sinks, min(lo, hi));
    if (mask) {                               // (counted no further than it takes to know that there are more)
      sees = 0;
      for (int v = 0; v < tiles && __any(have && sees <= kFewKeys); ++v) {
        const int j0 = tile_key(v);
        const uint64_t live = live_keys<KT>(mask, j0, s.keys);
        sees += __popc(visible_bits(j0, (uint32_t)live)) + __popc(visible_bits(j0 + 32, (uint32_t)(live >> 32)));
      }
    }
    const bool few = have && sees <= kFewKeys;
    if (__syncthreads_or(few)) {
      float sum = 0.0f;
      over([&](const L* kt, const L* vt, int j0, uint64_t live) { sum += weigh(kt, vt, j0, live); });
      sum += __shfl_xor(sum, 32, 64);
      if constexpr (QW == 2) {
        if (half == 0) sums[wave][col] = sum;
        __syncthreads();
        sum = sums[wave % QW][col] + sums[wave % QW + QW][col];
      }
      if (few) delta = sum;
    }
  }
  if (have && half == 0 && share == 0) a.delta[at_row] = delta;
  over([&](const L* kt, const L* vt, int j0, uint64_t live) { keys(kt, vt, j0, live); });
  if constexpr (QW == 2) {                    // the second wavefront's share
    float* join = (float*)lds;
    __syncthreads();
    settle();
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (share) join[((wave % QW * S::kBlocks + d) * 16 + r) * 64 + lane] = dq[d][r];
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] += join[((wave * S::kBlocks + d) * 16 + r) * 64 + lane];
  }
  float worst = 0.0f;
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) worst += fabsf(dq[d][r]);
  worst += __shfl_xor(worst, 32, 64);
  const bool good = finite(worst);
  if (have && good)
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * d + 8 * i + 4 * half;
        Pack<T, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = from_f32<T>(dq[d][4 * i + e] * p.scale);
        if (c < p.dim) x.store(dq_row + c);
      }
  uint32_t bad = (uint32_t)__ballot(have && !good);
  while (bad) {
    const int c = __ffs(bad) - 1;
    bad &= bad - 1;
    const int r = __shfl(row, c, 64);
    float g[(DP + 63) / 64];
    grad_q_row_again<T, DP>(a, s, kv, r, t0, t1, sink_tiles, __shfl(lse2, c, 64), __shfl(delta, c, 64), g);
    const int tk = r / a.group, hd = kv * a.group + r % a.group;
#pragma unroll
    for (int i = 0; i < (DP + 63) / 64; ++i)
      if (lane + 64 * i < p.dim)
        ((T*)a.dq)[(int64_t)(s.q0 + tk) * a.dq_row + hd * a.dq_head + lane + 64 * i] = from_f32<T>(g[i] * p.scale);
  }
}

// ---- gradients of the keys and values --------------------------------------------------------------------
// A workgroup owns 128 keys of a key head, 32 a wavefront, in registers; the packed rows that see them go
// through LDS 64 at a time, so the query heads that share the key head are summed where they are
// accumulated.  Where that makes few workgroups, one owns 64 keys, and two wavefronts share the rows of 32.  The first keys (sinks) are seen by every later row: the rows beyond the window of
// their tile ("far") are dealt out in items of kFarRows tokens to workgroups of their own, in which all four
// wavefronts hold the same 32 sinks and share the rows (with a wavefront for every 32 keys, three of them had
// nothing to do).  Their sums go to memory in 32 bits and are added in order by attention_sink_kernel.
// Measured: 16 x about 1500 rows, window 512, 4 sinks, 8 heads over 4 of 64, bf16: 117 us and 5 us for the sinks (products 30 %,
// VALU 33 %: two wavefronts a SIMD, one and a half loads of the chip).
struct FarRange { int first; bool any; };        // tokens [first, queries) see the sinks only
__device__ inline FarRange far_tokens(const AttnArgs& a, const Seq& s) {
  const ocnn_attention_params& p = a.p;
  FarRange f;
  f.first = min(max(a.near_keys - 1 + p.left - s.shift() + 1, 0), s.queries);
  f.any = p.sinks > 0 && p.left >= 0 && s.keys > 0 && f.first < s.queries;
  return f;
}

template <typename T, int DP>
__device__ __forceinline__ void grad_k_row_again(const AttnArgs& a, const Seq& s, int kv, int j, int from, int to,
    float (&dk)[(DP + 63) / 64], float (&dv)[(DP + 63) / 64]) {
  const ocnn_attention_params& p = a.p;
  const int lane = threadIdx.x & 63;
  const T* k = (const T*)p.k + (int64_t)(s.k0 + j) * p.k_row + kv * p.k_head;
  const T* v = (const T*)p.v + (int64_t)(s.k0 + j) * p.v_row + kv * p.v_head;
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i) dk[i] = dv[i] = 0.0f;
  for (int r0 = from; r0 < to; r0 += 64) {
    const int r = r0 + lane;
    float w = 0.0f, ds = 0.0f;
    if (r < to) {
      const int token = r / a.group, head = kv * a.group + r % a.group;
      const int64_t at = (int64_t)(s.q0 + token);
      const T* q = (const T*)p.q + at * p.q_row + head * p.q_head;
      const T* go = (const T*)a.grad + at * a.grad_row + head * a.grad_head;
      float dot = 0.0f, dp = 0.0f;
      for (int c = 0; c < p.dim; ++c) {
        dot = fmaf(to_f32(q[c]), to_f32(k[c]), dot);
        dp = fmaf(to_f32(go[c]), to_f32(v[c]), dp);
      }
      const float lse = a.lse[at * p.heads + head];
      w = exp2f(fmaf(dot, p.scale < 0.0f ? -a.scale2 : a.scale2, lse == -__builtin_inff() ? 0.0f : -lse * kLog2e));
      ds = w * (dp - a.delta[at * p.heads + head]);
    }
    if (__any(w != w) && __any(ds != ds)) {    // (both stay in every channel)
#pragma unroll
      for (int n = 0; n < (DP + 63) / 64; ++n) dk[n] = dv[n] = __builtin_nanf("");
      return;
    }
    for (int i = 0; i < min(64, to - r0); ++i) {
      const float wi = __shfl(w, i, 64), di = __shfl(ds, i, 64);
      const int token = (r0 + i) / a.group, head = kv * a.group + (r0 + i) % a.group;
      const int64_t at = (int64_t)(s.q0 + token);
      const T* q = (const T*)p.q + at * p.q_row + head * p.q_head;
      const T* go = (const T*)a.grad + at * a.grad_row + head * a.grad_head;
#pragma unroll
      for (int n = 0; n < (DP + 63) / 64; ++n)
        if (lane + 64 * n < p.dim) {
          dk[n] = fmaf(di, to_f32(q[lane + 64 * n]), dk[n]);
          dv[n] = fmaf(wi, to_f32(go[lane + 64 * n]), dv[n]);
        }
    }
  }
}

template <typename E, int DP>
__global__ void __launch_bounds__(256, grad_kv_waves<E>(DP)) attention_grad_kv_kernel(AttnArgs a,
    int near_items) {
  using S = Shape<E, DP>;
  using T = typename S::Memory;
  using L = typename S::Lds;
  constexpr int RT = 64, kTile = RT * S::kPitch * S::kPlanes;
  constexpr bool kLate = sizeof(T) == 4;
  __shared__ __attribute__((aligned(16))) L lds[2 * 2 * kTile];
  __shared__ float row_lse[2][RT], row_delta[2][RT];
  const ocnn_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int kv = blockIdx.y;
  const bool far = (int)blockIdx.x >= near_items;
  const int sink_blocks = p.sinks > 32 ? 2 : 1;    // of 32
  // `ways` wavefronts share the rows of 32 keys; this one's share, and its 32 keys
  const int key_shift = a.near_keys == 64 ? 6 : 7, ways = far ? 4 : 128 >> key_shift;
  const int share = ways == 4 ? wave : ways == 2 ? wave >> 1 : 0, key_wave = ways == 4 ? 0 : ways == 2 ? wave & 1 : wave;
  int b, j0 = 0, far_id = 0;
  int64_t item;
  if (!far) {
    const int id = item_of(blockIdx.x, near_items);
    b = locate_packed(p.k_offsets, p.n_seq, p.rows_k, id, key_shift, 1);
    item = (int64_t)id - ((clamped(p.k_offsets, b, p.rows_k) >> key_shift) + b);
  } else {
    far_id = ((int)blockIdx.x - near_items) / sink_blocks;
    j0 = (((int)blockIdx.x - near_items) % sink_blocks) * 32;
    const int id = far_id;
    b = locate_packed(p.q_offsets, p.n_seq, p.rows_q, id, Log2<kFarRows>::value, 1);
    item = (int64_t)id - ((clamped(p.q_offsets, b, p.rows_q) >> Log2<kFarRows>::value) + b);
    if (b >= p.n_seq) return;
  }
  if (item < 0) return;
  if (b >= p.n_seq) {                              // key rows behind the last sequence
    const int k_begin = clamped(p.k_offsets, b, p.rows_k);
    const int64_t r = k_begin + item * a.near_keys + key_wave * 32 + col;
    if (r < p.rows_k && share == 0)
      for (int c = half * S::kMemoryPiece; c < p.dim; c += 2 * S::kMemoryPiece) {
        *(uintx4*)((T*)a.dk + r * a.dk_row + kv * a.dk_head + c) = uintx4{0, 0, 0, 0};
        *(uintx4*)((T*)a.dv + r * a.dv_row + kv * a.dv_head + c) = uintx4{0, 0, 0, 0};
      }
    return;
  }
  const Seq s = sequence(p, b);
  const FarRange fr = far_tokens(a, s);
  const int shift = s.shift();
  // the tokens that see the window keys [x, y]
  auto first_token = [&](int x) { return p.right < 0 ? 0 : min(max(x - p.right - shift, 0), s.queries); };
  auto end_token = [&](int y) { return p.left < 0 ? s.queries : min(max(y + p.left + 1 - shift, 0), s.queries); };
  int ta, tb;                                      // tokens of this workgroup
  if (!far) {
    if (item * a.near_keys >= s.room) return;
    j0 = (int)item * a.near_keys;
    ta = first_token(j0);
    tb = end_token(j0 + a.near_keys - 1);
  } else {
    if (!fr.any) return;
    ta = max((int)item * kFarRows, fr.first);
    tb = (int)min((item + 1) * kFarRows, (int64_t)s.queries);
    if (ta >= tb) return;
  }
  const bool sink_tile = (far || j0 == 0) && fr.any;   // its first keys' sums go to memory
  const int jw = j0 + key_wave * 32, j = jw + col;
  bool key = j < s.keys && (!far || j < p.sinks);
  if (key && p.key_mask) key = p.key_mask[s.k0 + j] != 0;
  // this key's packed rows: [lo, hi), and what some / every key of the wavefront has
  int lo = 0, hi = 0;
  if (key) {
    lo = first_token(j);
    hi = j < p.sinks ? s.queries : end_token(j);
    lo = max(lo, ta) * a.group;
    hi = min(hi, tb) * a.group;
  }
  int w_lo = 0, w_hi = 0, all_lo = 0, all_hi = 0;
  if (jw < s.keys && (!far || jw < p.sinks)) {
    const bool any_sink = jw < p.sinks;
    w_lo = max(first_token(jw), ta) * a.group;
    w_hi = min(any_sink ? s.queries : end_token(jw + 31), tb) * a.group;
    if (jw + 32 <= s.keys && !p.key_mask && (!far || jw + 32 <= p.sinks)) {
      all_lo = max(first_token(jw + 31), ta) * a.group;
      all_hi = min(end_token(jw), tb) * a.group;
    }
  }
  Column<E, DP> k, vv;
  load_row<E, DP>(k, (const T*)p.k + (int64_t)(s.k0 + j) * p.k_row + kv * p.k_head, key, p.dim, p.scale < 0.0f);
  load_row<E, DP>(vv, (const T*)p.v + (int64_t)(s.k0 + j) * p.v_row + kv * p.v_head, key, p.dim);
  floatx16 dk[S::kBlocks], dv[S::kBlocks];
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d) dk[d] = dv[d] = zero16();

  // 32 packed rows from r0 on, those before `end`
  auto subtile = [&](const L* qt, const L* gt, const float* lse2, const float* delta, int r0, int end) {
    if (r0 + 32 <= w_lo || r0 >= min(w_hi, end)) return;
    const bool masked = decided((r0 < all_lo) | (r0 + 32 > min(all_hi, end)));
    RowFrags<E, DP> qf, gf;
    qf.load(qt);
    gf.load(gt);
    // The products start from -lse and -dO . o of their rows, in the units of the scores.  fp32: the lse is taken off
    // behind, since it may be many times a score, and every step of the product would round at its size (dk and dv of
    // 700 queries: 1.1e-6 off instead of 6e-7).
    floatx16 x = zero16(), dp, ls;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const floatx4 l4 = *(const floatx4*)(lse2 + 8 * i + 4 * half), d4 = *(const floatx4*)(delta + 8 * i + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ls[4 * i + e] = l4[e];
        dp[4 * i + e] = d4[e];
      }
    }
    if constexpr (!kLate) x = ls;
    if constexpr (Ahead<E, DP>::value) in_order();
    rows_times<E, DP>(qf, k, x, gf, vv, dp);
    ColumnFrags<E, DP> gc, qc;
    gc.load(gt);
    if constexpr (Ahead<E, DP>::value) in_order();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(kLate ? fmaf(x[r], a.scale2, ls[r]) : x[r] * a.scale2);
      dp[r] *= x[r];
    }
    if (masked) {
      const uint32_t seen = (first_bits(min(hi, end) - r0) & ~first_bits(lo - r0)) >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = where_seen(seen, r, x[r], 0u);
        dp[r] = where_seen(seen, r, dp[r], 0u);
      }
    }
    qc.load(qt);
    if constexpr (Ahead<E, DP>::value) in_order();
    gc.template times<kFine>(dv, x);
    qc.template times<kFine>(dk, dp);
  };

  // a tile holds whole tokens: `step` of them, group rows each, so that a thread's rows keep their offsets
  const int step = RT / a.group, used = step * a.group;
  const int tiles = s.keys > 0 && tb > ta ? (tb - ta + step - 1) / step : 0;
  const T* qbase = (const T*)p.q + (int64_t)(s.q0 + ta) * p.q_row + (int64_t)kv * a.group * p.q_head;
  const T* gbase = (const T*)a.grad + (int64_t)(s.q0 + ta) * a.grad_row + (int64_t)kv * a.group * a.grad_head;
  Staged<E, DP, RT, 256, false> sq, sg;
  sq.init(tid, p.dim, [&](int i) { const int t = i / a.group; return t * (int)p.q_row + (i - t * a.group) * (int)p.q_head; });
  sg.init(tid, p.dim, [&](int i) { const int t = i / a.group; return t * (int)a.grad_row + (i - t * a.group) * (int)a.grad_head; });
  const int my_token = tid / a.group;
  const int64_t my_stat = (int64_t)(s.q0 + ta + my_token) * p.heads + kv * a.group + tid - my_token * a.group;
  const float lse_unit = kLate ? kLog2e : kLog2e / a.scale2;
  float one_lse = 0.0f, one_delta = 0.0f;
  auto fetch = [&](int v) {
    const int t = v * step, rows = min(tb - ta - t, step) * a.group;
    sq.load(qbase + (int64_t)t * p.q_row, tid, used < RT ? min(rows, used) : rows);
    sg.load(gbase + (int64_t)t * a.grad_row, tid, used < RT ? min(rows, used) : rows);
    if (tid < rows && tid < RT) {              // (as they are: nothing here may wait for a load)
      one_lse = a.lse[my_stat + (int64_t)t * p.heads];
      one_delta = a.delta[my_stat + (int64_t)t * p.heads];
    } else {
      one_lse = one_delta = 0.0f;
    }
  };
  auto put = [&](int buf) {
    sq.store(lds + buf * 2 * kTile, tid);
    sg.store(lds + (buf * 2 + 1) * kTile, tid);
    if (tid < RT) {
      row_lse[buf][tid] = one_lse == -__builtin_inff() ? 0.0f : -one_lse * lse_unit;
      row_delta[buf][tid] = -one_delta;
    }
  };
  auto half_tile = [&](int buf, int h, int v) {
    const int r0 = (ta + v * step) * a.group;
    if (32 * h < used)
      subtile(lds + buf * 2 * kTile + h * 32 * S::kPitch, lds + (buf * 2 + 1) * kTile + h * 32 * S::kPitch,
          row_lse[buf] + 32 * h, row_delta[buf] + 32 * h, r0 + 32 * h, r0 + used);
  };
  if (!far) {
    if (tiles > 0) fetch(0);
    for (int v = 0; v < tiles; ++v) {
      put(v & 1);
      __syncthreads();
      if (v + 1 < tiles) fetch(v + 1);
#pragma unroll 1
      for (int h = 0; h < 2; ++h)
        if (ways == 1 || h == share) half_tile(v & 1, h, v);
    }
  } else {
#pragma unroll 1
    for (int v = 0; v < tiles; v += 2) {             // two tiles, a half for each wavefront
      fetch(v);
      __syncthreads();
      put(0);
      if (v + 1 < tiles) {
        fetch(v + 1);
        put(1);
      }
      __syncthreads();
      if (v + (wave >> 1) < tiles) half_tile(wave >> 1, wave & 1, v + (wave >> 1));
    }
  }
  if (ways > 1) {
    // the shares, added in order by the wavefronts of the first
    float* join = (float*)lds;
    const int per = 4 / ways;
    auto add_up = [&](floatx16 (&x)[S::kBlocks]) {
      __syncthreads();
      if (share)
#pragma unroll
        for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) join[(((wave - per) * S::kBlocks + d) * 16 + r) * 64 + lane] = x[d][r];
      __syncthreads();
      if (!share)
        for (int w = wave; w < 4 - per; w += per)
#pragma unroll
          for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[d][r] += join[((w * S::kBlocks + d) * 16 + r) * 64 + lane];
    };
    settle();
    add_up(dk);
    add_up(dv);
    if (share) return;
  }

  float worst = 0.0f;
#pragma unroll
  for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) worst += fabsf(dk[d][r]) + fabsf(dv[d][r]);
  worst += __shfl_xor(worst, 32, 64);
  const bool good = finite(worst), mine = j < s.room;
  const bool to_memory = sink_tile && j < min(p.sinks, s.keys);
  const int64_t slot = far ? (int64_t)p.n_seq + far_id : b;
  float* part = a.sink_part + (slot * p.kv_heads + kv) * 2 * p.sinks * p.dim + (int64_t)(to_memory ? j : 0) * p.dim;
  const int64_t part_dv = (int64_t)p.sinks * p.dim;
  T* dk_row = (T*)a.dk + (int64_t)(s.k0 + j) * a.dk_row + kv * a.dk_head;
  T* dv_row = (T*)a.dv + (int64_t)(s.k0 + j) * a.dv_row + kv * a.dv_head;
  if (mine && good && (to_memory || !far))
#pragma unroll
    for (int d = 0; d < S::kBlocks; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * d + 8 * i + 4 * half;
        if (c >= p.dim) continue;
        if (to_memory) {
          *(floatx4*)(part + c) = floatx4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]};
          *(floatx4*)(part + part_dv + c) = floatx4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]};
        } else {
          Pack<T, 4> x, y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x.v[e] = from_f32<T>(dk[d][4 * i + e] * p.scale);
            y.v[e] = from_f32<T>(dv[d][4 * i + e]);
          }
          x.store(dk_row + c);
          y.store(dv_row + c);
        }
      }
  uint32_t bad = (uint32_t)__ballot(mine && !good && (to_memory || !far));
  while (bad) {
    const int c = __ffs(bad) - 1;
    bad &= bad - 1;
    const int jj = __shfl(j, c, 64);
    float gk[(DP + 63) / 64], gv[(DP + 63) / 64];
    grad_k_row_again<T, DP>(a, s, kv, jj, __shfl(lo, c, 64), __shfl(hi, c, 64), gk, gv);
    const bool mem = sink_tile && jj < min(p.sinks, s.keys);
#pragma unroll
    for (int i = 0; i < (DP + 63) / 64; ++i) {
      const int ch = lane + 64 * i;
      if (ch >= p.dim) continue;
      if (mem) {
        float* at = a.sink_part + (slot * p.kv_heads + kv) * 2 * p.sinks * p.dim + (int64_t)jj * p.dim + ch;
        at[0] = gk[i];
        at[part_dv] = gv[i];
      } else {
        ((T*)a.dk)[(int64_t)(s.k0 + jj) * a.dk_row + kv * a.dk_head + ch] = from_f32<T>(gk[i] * p.scale);
        ((T*)a.dv)[(int64_t)(s.k0 + jj) * a.dv_row + kv * a.dv_head + ch] = from_f32<T>(gv[i]);
      }
    }
  }
}

// The sinks' sums: the tile's own, then the far items in order.  Grid: (sinks, kv heads, sequences); threads:
// (dk, dv) x 128 channels x 4 shares of the items.
template <typename T>
__global__ void __launch_bounds__(1024) attention_sink_kernel(AttnArgs a) {
  __shared__ float shares[4][256];
  const ocnn_attention_params& p = a.p;
  const int j = blockIdx.x, kv = blockIdx.y, b = blockIdx.z;
  const Seq s = sequence(p, b);
  const FarRange fr = far_tokens(a, s);
  if (!fr.any || j >= s.keys) return;
  const int t = threadIdx.x & 255, share = threadIdx.x >> 8, c = t & 127, which = t >> 7;
  const int64_t one = (int64_t)p.kv_heads * 2 * p.sinks * p.dim;
  const float* base = a.sink_part + ((int64_t)kv * 2 + which) * p.sinks * p.dim + (int64_t)j * p.dim + c;
  const int i0 = fr.first / kFarRows, i1 = (s.queries - 1) / kFarRows + 1, each = (i1 - i0 + 3) / 4;
  const int64_t id0 = (int64_t)p.n_seq + (s.q0 >> Log2<kFarRows>::value) + b;
  float sum = 0.0f;
  if (c < p.dim) {
    if (share == 0) sum = base[(int64_t)b * one];
    for (int i = i0 + share * each; i < min(i0 + (share + 1) * each, i1); ++i) sum += base[(id0 + i) * one];
  }
  shares[share][t] = sum;
  __syncthreads();
  if (share || c >= p.dim) return;
  sum += shares[1][t];
  sum += shares[2][t];
  sum += shares[3][t];
  if (which) ((T*)a.dv)[(int64_t)(s.k0 + j) * a.dv_row + kv * a.dv_head + c] = from_f32<T>(sum);
  else ((T*)a.dk)[(int64_t)(s.k0 + j) * a.dk_row + kv * a.dk_head + c] = from_f32<T>(sum * p.scale);
}

// ---- host ------------------------------------------------------------------------------------------------
int check_params(const ocnn_attention_params* p) {
  OCNN_REQUIRE(p, OCNN_E_BADARG, "null pointer");
  OCNN_REQUIRE(p->dtype == OCNN_F32 || p->dtype == OCNN_BF16, OCNN_E_BADARG, "dtype %d", p->dtype);
  OCNN_REQUIRE(p->rows_q >= 0 && p->rows_k >= 0 && p->n_seq >= 1 && p->n_seq <= 65535, OCNN_E_BADARG,
      "%d queries, %d keys, %d sequences (1 .. 65535)", p->rows_q, p->rows_k, p->n_seq);
  OCNN_REQUIRE(p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->kv_heads <= 65535, OCNN_E_SHAPE,
      "%d query heads over %d key heads", p->heads, p->kv_heads);
  OCNN_REQUIRE(p->heads / p->kv_heads <= 64, OCNN_E_UNSUPPORTED, "%d query heads a key head: at most 64", p->heads / p->kv_heads);
  OCNN_REQUIRE(p->dim > 0 && p->dim <= 128 && p->dim % 8 == 0, OCNN_E_UNSUPPORTED,
      "%d channels a head: multiples of 8 up to 128", p->dim);
  OCNN_REQUIRE(p->left >= -1 && p->right >= -1, OCNN_E_BADARG, "window %d, %d: -1 for no bound", p->left, p->right);
  OCNN_REQUIRE(p->sinks >= 0 && p->sinks <= kMaxSinks, OCNN_E_UNSUPPORTED, "%d sinks: at most %d", p->sinks, kMaxSinks);
  OCNN_REQUIRE(std::isfinite(p->scale * kLog2e), OCNN_E_BADARG, "scale %g: scale x log2(e) must be finite in 32 bits", p->scale);
  // (positions and rows of a tile more, plus a bound of 2^30 in front or behind, stay below 2^31)
  OCNN_REQUIRE((int64_t)p->rows_q * p->heads <= (1ll << 30) - 1024 && p->rows_k <= (1 << 30) - 1024, OCNN_E_UNSUPPORTED,
      "%d x %d query rows, %d key rows: at most 2^30 - 1024", p->rows_q, p->heads, p->rows_k);
  OCNN_REQUIRE(p->q_offsets && p->k_offsets && (p->rows_q == 0 || p->q) && (p->rows_k == 0 || (p->k && p->v)), OCNN_E_BADARG,
      "null pointer");
  return OCNN_OK;
}

// 16-byte rows: pointers and strides of every row tensor
// and 64 rows of a group of heads lie within 2^30 elements
int check_rows(int dtype, const char* name, const void* at, int64_t row, int64_t head) {
  const int64_t piece = dtype == OCNN_F32 ? 4 : 8;
  OCNN_REQUIRE(row >= 0 && row < (1 << 22) && head >= 0 && head < (1 << 22), OCNN_E_UNSUPPORTED,
      "%s: strides %lld, %lld: below 2^22 elements", name, (long long)row, (long long)head);
  OCNN_REQUIRE((uintptr_t)at % 16 == 0 && row % piece == 0 && head % piece == 0, OCNN_E_BADARG,
      "%s: rows and heads must begin at multiples of 16 bytes", name);
  return OCNN_OK;
}

struct Plan { bool few; int splits; int64_t tiles; };
// few: 32 packed rows a workgroup, where a sequence has that many or fewer on average.  splits: the keys are
// dealt out where the row tiles leave compute units empty, as long as a workgroup keeps some tiles.
// Shares of the keys for few rows, from an estimate in us.  `blocks` workgroups a share take 128 keys at a time; such a step
// takes what its products and waits take (rows of B bytes: bf16 B / 140, fp32 B / 80; measured at 128 to 512 bytes) or what
// memory gives all workgroups that run (5 TB/s).  A load of the chip costs its steps and 2 to begin, the joining launch 3.5.  The
// shares that fill one to four loads are tried.  In us, so and with a share for every 1024 keys: 4 x 772 keys, 2 heads of 48,
// fp32 11.8 27.7; 1 x 4000 keys, 8 heads over 2 of 64, bf16 10.4 20.2, fp32 12.4 43.7; 8 x 15000 keys, 16 heads over 4 of 128,
// fp32 122 147 (32 shares: 157); 32 x 600 keys, 8 heads over 2 of 64, bf16: one share 10.8, two 12.1.
int few_splits(int64_t blocks, int64_t keys, int64_t slots, int row_bytes, bool f32) {
  const int64_t steps = std::max<int64_t>((keys + 127) / 128, 1), most = std::min<int64_t>(steps, kMaxSplits);
  const double floor_us = row_bytes / (f32 ? 80.0 : 140.0);
  auto estimate = [&](int64_t n) {
    const int64_t all = blocks * n;
    const double step = std::max(floor_us, std::min(all, slots) * 256.0 * row_bytes / 5e6);
    return (double)((all + slots - 1) / slots) * ((double)((steps + n - 1) / n) * step + 2.0) + (n > 1 ? 3.5 : 0.0);
  };
  int64_t best = 1;
  for (int64_t k = 1; k <= 4; ++k) {
    int64_t n = std::min(k * slots / std::max<int64_t>(blocks, 1), most);
    if (n <= 1) continue;
    const int64_t each = (steps + n - 1) / n;
    if (each <= 4) n = (steps + each - 1) / each;            // (no more shares than these steps need)
    if (n > 1 && estimate(n) < estimate(best)) best = n;
  }
  return (int)best;
}

Plan plan_of(const ocnn_attention_params& p) {
  Plan n;
  const int64_t group = p.heads / p.kv_heads, packed = (int64_t)p.rows_q * group;
  n.few = packed <= 32 * (int64_t)p.n_seq;
  n.tiles = (packed >> (n.few ? 5 : 7)) + p.n_seq + 1;
  int64_t keys = p.rows_k / p.n_seq;
  if (p.left >= 0 && p.right >= 0) keys = std::min<int64_t>(keys, (int64_t)p.left + p.right + p.rows_q / p.n_seq + p.sinks);
  const int64_t blocks = std::max<int64_t>((packed + (n.few ? 31 : 127)) / (n.few ? 32 : 128), n.few ? p.n_seq : 1) * p.kv_heads;
  if (n.tiles > 65535) {
    n.splits = 1;
  } else if (n.few) {
    const int row_bytes = (p.dim + 31) / 32 * 32 * (p.dtype == OCNN_F32 ? 4 : 2);
    n.splits = few_splits(blocks, keys, 256 * plain_waves(row_bytes), row_bytes, p.dtype == OCNN_F32);
  } else {
    n.splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(blocks, 1), keys / 1024, kMaxSplits}));
  }
  return n;
}
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t split_bytes(const ocnn_attention_params& p, const Plan& n) {
  if (n.splits == 1) return 0;
  const size_t rows = (size_t)n.splits * p.rows_q * p.heads;
  return round256(rows * p.dim * 4) + round256(rows * 8);
}
int64_t far_items(const ocnn_attention_params& p) { return (p.rows_q >> Log2<kFarRows>::value) + p.n_seq + 1; }
bool has_far(const ocnn_attention_params& p) { return p.sinks > 0 && p.left >= 0 && p.rows_q > 0; }
size_t sink_bytes(const ocnn_attention_params& p) {
  return has_far(p) ? (size_t)(p.n_seq + far_items(p)) * p.kv_heads * 2 * p.sinks * p.dim * 4 : 0;
}
size_t grad_bytes(const ocnn_attention_params& p) {
  return round256((size_t)p.rows_q * p.heads * 4) + round256(sink_bytes(p));
}

AttnArgs args_of(const ocnn_attention_params& p) {
  AttnArgs a = {};
  a.p = p;
  a.p.left = std::min(p.left, 1 << 30);
  a.p.right = std::min(p.right, 1 << 30);
  a.group = p.heads / p.kv_heads;
  a.scale2 = std::max(fabsf(p.scale) * kLog2e, 0x1p-100f);   // (not zero: statistics are divided by it)
  return a;
}

template <typename F> void by_dim(int dim, F f) {
  if (dim <= 32) f(std::integral_constant<int, 32>());
  else if (dim <= 64) f(std::integral_constant<int, 64>());
  else if (dim <= 96) f(std::integral_constant<int, 96>());
  else f(std::integral_constant<int, 128>());
}

// fp32 in planes, where the registers hold three of everything: 8 x 700 rows, all visible, 6 heads, in planes and not: of 32
// channels 40 and 60 us forward, 114 and 179 backward; of 64 channels 88 and 102, 255 and 369.  96 channels and more would want
// over 512 registers a lane.  (Few rows, QW = 1, wait for memory and stay in fp32.)
template <typename T, int DP> struct Held { using type = T; };
template <> struct Held<float, 32> { using type = Planes; };
template <> struct Held<float, 64> { using type = Planes; };

// 64 packed rows a workgroup instead of 128, two wavefronts on the same 32, where 128 leave a quarter of the compute units and
// more without one (us with 64 and with 128; heads of 64 channels; forward in bf16, in fp32, queries' and keys' gradient in bf16):
//   1 x 1000 rows, 4 heads over 2, window 200: 9.5 11.5, 18.0 23.8, 27.8 30.6      (about 32 workgroups of 128)
//   3 x 1800 rows, 4 heads, causal: 34.6 41.5, 111 109, 86 97                      (180)
//   9 x 800 rows, 8 heads over 4, all visible: 34.9 27.7, 137 104, 94.9 89.9       (484)
bool half_tiles(const ocnn_attention_params& p) {
  return ((int64_t)p.rows_q * (p.heads / p.kv_heads) / 128 + p.n_seq) * p.kv_heads <= 192;
}

template <typename T, int DP> void forward_launch(const AttnArgs& a, const Plan& n, hipStream_t s) {
  const dim3 grid = n.splits > 1 ? dim3(n.splits, a.p.kv_heads, (unsigned)n.tiles) : dim3((unsigned)whole_sets(n.tiles), a.p.kv_heads);
  if (n.few) {
    if (n.splits > 1) attention_kernel<T, DP, 1, true><<<grid, 256, 0, s>>>(a);
    else attention_kernel<T, DP, 1, false><<<grid, 256, 0, s>>>(a);
  } else {
    using E = typename Held<T, DP>::type;
    if (n.splits > 1) attention_kernel<E, DP, 4, true><<<grid, 256, 0, s>>>(a);
    else if (half_tiles(a.p))
      attention_kernel<E, DP, 2, false><<<dim3((unsigned)whole_sets(((int64_t)a.p.rows_q * a.group >> 6) + a.p.n_seq + 1), a.p.kv_heads), 256, 0, s>>>(a);
    else attention_kernel<E, DP, 4, false><<<grid, 256, 0, s>>>(a);
  }
  if (n.splits > 1) attention_join_kernel<T><<<(unsigned)((int64_t)a.p.rows_q * a.p.heads), 256, 0, s>>>(a);
}

template <typename T, int DP> void backward_launch(AttnArgs a, hipStream_t s) {
  const ocnn_attention_params& p = a.p;
  using E = typename Held<T, DP>::type;
  if (p.rows_q > 0) {
    const bool half = half_tiles(p);
    const dim3 grid((unsigned)whole_sets(((int64_t)p.rows_q * a.group >> (half ? 6 : 7)) + p.n_seq + 1), p.kv_heads);
    if (half) attention_grad_q_kernel<E, DP, 2><<<grid, 256, 0, s>>>(a);
    else attention_grad_q_kernel<E, DP, 4><<<grid, 256, 0, s>>>(a);
  }
  if (p.rows_k > 0) {
    // 64 keys a workgroup where 128 leave much of the chip idle: half the work each, but every row staged twice as often.
    // 1 x 1000 rows, 4 heads over 2 of 64, window 200: 99 and 73 us (fp32); 4 x 1500 rows, 8 over 4, window 512: 81 and 71 us
    // (bf16); 16 x 1500 rows (760 workgroups of 128 keys): 197 and 201 us; 2 x 20000 rows, 16 heads: 620 and 693 us.  Of 128
    // channels, one workgroup a compute unit: 64 and 53, 144 and 165, 462 and 502 us.
    const int64_t blocks = (p.rows_k / 128 + p.n_seq) * (int64_t)p.kv_heads;
    a.near_keys = blocks <= 160 * grad_kv_waves<E>(DP) ? 64 : 128;
    const int64_t near_items = whole_sets((p.rows_k / a.near_keys) + p.n_seq + 1);
    const int64_t all = near_items + (has_far(p) ? far_items(p) * (p.sinks > 32 ? 2 : 1) : 0);
    attention_grad_kv_kernel<E, DP><<<dim3((unsigned)all, p.kv_heads), 256, 0, s>>>(a, (int)near_items);
    if (has_far(p)) attention_sink_kernel<T><<<dim3(p.sinks, p.kv_heads, p.n_seq), 1024, 0, s>>>(a);
  }
}

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" {

int ocnn_attention_workspace_bytes(const ocnn_attention_params* params, size_t* workspace_bytes, size_t* grad_workspace_bytes) {
  int rc = check_params(params);
  if (rc) return rc;
  if (workspace_bytes) *workspace_bytes = split_bytes(*params, plan_of(*params));
  if (grad_workspace_bytes) *grad_workspace_bytes = grad_bytes(*params);
  return OCNN_OK;
}

int ocnn_octree_attention(void* out, int64_t out_row, int64_t out_head, float* lse, const ocnn_attention_params* params,
    int fill_rest, void* workspace_dev, size_t workspace_bytes, ocnn_stream_t stream) {
  int rc = check_params(params);
  if (rc) return rc;
  const ocnn_attention_params& p = *params;
  if (p.rows_q == 0) return OCNN_OK;
  OCNN_REQUIRE(out, OCNN_E_BADARG, "null pointer");
  if ((rc = check_rows(p.dtype, "q", p.q, p.q_row, p.q_head)) || (rc = check_rows(p.dtype, "k", p.k, p.k_row, p.k_head)) ||
      (rc = check_rows(p.dtype, "v", p.v, p.v_row, p.v_head)) || (rc = check_rows(p.dtype, "out", out, out_row, out_head)))
    return rc;
  const Plan n = plan_of(p);
  const size_t need = split_bytes(p, n);
  OCNN_REQUIRE(need == 0 || (workspace_dev && workspace_bytes >= need && (uintptr_t)workspace_dev % 16 == 0), OCNN_E_WORKSPACE,
      "octree_attention needs %zu bytes, 16-byte aligned, got %zu", need, workspace_bytes);
  AttnArgs a = args_of(p);
  a.splits = n.splits;
  a.out = out; a.out_row = out_row; a.out_head = out_head; a.lse = lse; a.fill = fill_rest != 0;
  if (n.splits > 1) {
    a.part_o = (float*)workspace_dev;
    a.part_ml = (float*)((char*)workspace_dev + round256((size_t)n.splits * p.rows_q * p.heads * p.dim * 4));
  }
  hipStream_t s = as_stream(stream);
  by_dim(p.dim, [&](auto d) {
    if (p.dtype == OCNN_F32) forward_launch<float, d.value>(a, n, s);
    else forward_launch<uint16_t, d.value>(a, n, s);
  });
  OCNN_LAUNCH_OK("octree_attention");
  return OCNN_OK;
}

int ocnn_octree_attention_grad(void* grad_q, int64_t grad_q_row, int64_t grad_q_head, void* grad_k, int64_t grad_k_row,
    int64_t grad_k_head, void* grad_v, int64_t grad_v_row, int64_t grad_v_head, const void* grad_out, int64_t grad_out_row,
    int64_t grad_out_head, const void* out, int64_t out_row, int64_t out_head, const float* lse,
    const ocnn_attention_params* params, void* workspace_dev, size_t workspace_bytes, ocnn_stream_t stream) {
  int rc = check_params(params);
  if (rc) return rc;
  const ocnn_attention_params& p = *params;
  if (p.rows_q == 0 && p.rows_k == 0) return OCNN_OK;
  OCNN_REQUIRE((p.rows_q == 0 || (grad_q && grad_out && out && lse)) && (p.rows_k == 0 || (grad_k && grad_v)), OCNN_E_BADARG,
      "null pointer");
  if ((rc = check_rows(p.dtype, "q", p.q, p.q_row, p.q_head)) || (rc = check_rows(p.dtype, "k", p.k, p.k_row, p.k_head)) ||
      (rc = check_rows(p.dtype, "v", p.v, p.v_row, p.v_head)) || (rc = check_rows(p.dtype, "out", out, out_row, out_head)) ||
      (rc = check_rows(p.dtype, "grad_out", grad_out, grad_out_row, grad_out_head)) ||
      (rc = check_rows(p.dtype, "grad_q", grad_q, grad_q_row, grad_q_head)) ||
      (rc = check_rows(p.dtype, "grad_k", grad_k, grad_k_row, grad_k_head)) ||
      (rc = check_rows(p.dtype, "grad_v", grad_v, grad_v_row, grad_v_head)))
    return rc;
  const size_t need = grad_bytes(p);
  OCNN_REQUIRE(need == 0 || (workspace_dev && workspace_bytes >= need && (uintptr_t)workspace_dev % 16 == 0), OCNN_E_WORKSPACE,
      "octree_attention_grad needs %zu bytes, 16-byte aligned, got %zu", need, workspace_bytes);
  AttnArgs a = args_of(p);
  a.dq = grad_q; a.dq_row = grad_q_row; a.dq_head = grad_q_head;
  a.dk = grad_k; a.dk_row = grad_k_row; a.dk_head = grad_k_head;
  a.dv = grad_v; a.dv_row = grad_v_row; a.dv_head = grad_v_head;
  a.grad = grad_out; a.grad_row = grad_out_row; a.grad_head = grad_out_head;
  a.fwd = out; a.fwd_row = out_row; a.fwd_head = out_head;
  a.lse = const_cast<float*>(lse);
  a.delta = (float*)workspace_dev;
  a.sink_part = (float*)((char*)workspace_dev + round256((size_t)p.rows_q * p.heads * 4));
  hipStream_t s = as_stream(stream);
  by_dim(p.dim, [&](auto d) {
    if (p.dtype == OCNN_F32) backward_launch<float, d.value>(a, s);
    else backward_launch<uint16_t, d.value>(a, s);
  });
  OCNN_LAUNCH_OK("octree_attention_grad");
  return OCNN_OK;
}

}  // extern "C"
