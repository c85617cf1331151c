// Shared by the operators along the node order of an octree level (sequence.hip, attention.hip).
#pragma once

#include "ocnn_common.h"

#include <initializer_list>
#include <type_traits>
#include <utility>

namespace ocnn {

__device__ inline float to_f32(float v) { return v; }
__device__ inline float to_f32(uint16_t v) { return bf16_to_f32(v); }
template <typename T> __device__ inline T from_f32(float v);
template <> __device__ inline float from_f32<float>(float v) { return v; }
template <> __device__ inline uint16_t from_f32<uint16_t>(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest even

// N neighbouring elements in registers; loads and stores need the alignment of one element only
template <typename T, int N> struct Pack {
  T v[N];
  __device__ inline void load(const T* p) { __builtin_memcpy(v, p, sizeof(v)); }
  __device__ inline void store(T* p) const { __builtin_memcpy(p, v, sizeof(v)); }
  // past the caches: what is written is not read again soon, and must not displace what is
  __device__ inline void store_past(T* p) const {
    if constexpr (sizeof(v) >= 8) {
      typedef uint32_t words __attribute__((ext_vector_type(sizeof(v) / 4)));
      __builtin_nontemporal_store(__builtin_bit_cast(words, v), (words*)p);
    } else {
      store(p);
    }
  }
  __device__ inline void fill(T x) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x;
  }
};

template <int N> struct Log2 { static constexpr int value = 1 + Log2<N / 2>::value; };
template <> struct Log2<1> { static constexpr int value = 0; };

// offsets[i], kept inside the rows that exist: a table the caller got wrong gives wrong results, never an
// access outside the tensors
__device__ inline int clamped(const int* offsets, int i, int rows) { return min(max(offsets[i], 0), rows); }

// Work items of 2^shift rows for sequences whose lengths only the device knows: sequence b owns the ids from
// (offsets[b] >> shift) + b on.  Two neighbours are at least ceil(length / 2^shift) apart (and 1 where the
// sequence is empty), and (rows >> shift) + n_seq ids serve all sequences, without a scan over their
// lengths.  The rows behind the last sequence count as sequence n_seq.  Returns the sequence that owns `id`.
// locate_packed: the same where every row stands for `each` items.
__device__ inline int locate_packed(const int* offsets, int n_seq, int rows, int64_t id, int shift, int each) {
  int lo = 0, hi = n_seq;                    // the largest b with start(b) <= id
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (((int64_t)clamped(offsets, mid, rows) * each >> shift) + mid <= id) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ inline int locate(const int* offsets, int n_seq, int rows, int64_t id, int shift) {
  return locate_packed(offsets, n_seq, rows, id, shift, 1);
}

}  // namespace ocnn
