// Operators along the node order of an octree level.  A level of a batched octree is one sequence
// per octree (its nodes in Morton order, octree after octree, octree/octree/merge_octrees.cpp:114-198);
// `offsets` (int32 [n_seq + 1], device) says where each begins.
//   * octree_offsets: those offsets, from the keys of the level
//   * rotary positions with several axes
//   * the gated linear recurrence and its gradient
// Tensors are row-major (a row is a node), so consecutive lanes hold consecutive channels.
#include "sequence.h"

#include <algorithm>

namespace ocnn {
namespace {

// ---- octree_offsets ---------------------------------------------------------------------------------
// The octree index is the top 16 bits of a key in both key forms, and the keys of a level are sorted by
// it: offsets[b] = the first node with index >= b.  Over the non-empty nodes it is that node's rank,
// i.e. the child entry of the first non-empty node from there on.  One wavefront per octree.
__global__ void octree_offsets_kernel(int* __restrict__ offsets, const uint64_t* __restrict__ key,
    const int* __restrict__ child, int nnum, int nnum_nempty, int batch, int nempty) {
  const int b = blockIdx.x, lane = threadIdx.x;
  int lo = 0, hi = nnum;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if ((int)(key[mid] >> 48) < b) lo = mid + 1; else hi = mid;
  }
  if (b >= batch) lo = nnum;
  int out = nempty ? nnum_nempty : lo;
  if (nempty) {
    for (int at = lo; at < nnum; at += 64) {
      const int c = at + lane < nnum ? child[at + lane] : -1;
      const uint64_t live = __ballot(c >= 0);
      if (live) { out = __shfl(c, __ffsll((unsigned long long)live) - 1, 64); break; }
    }
  }
  if (lane == 0) offsets[b] = out;
}

// ---- rotary positions -----------------------------------------------------------------------------
// Pair p of channels belongs to one axis and turns by t = position[axis] * frequency[p]:
//   (x, y) -> (x cos t - y sin t, x sin t + y cos t);  the inverse turns by -t (the gradient).
// The angle is formed in 64 bits and reduced to a fraction of a turn before it is rounded to 32: at
// position 2^20 a 32-bit product is off by 2^-5 rad, the fraction by 2^-25 of a turn.  One angle
// serves all heads of a row, so the sines (a 64-bit product, a reduction and a polynomial) are computed
// once a row into LDS and the streaming part is two fused multiply-adds per channel: bound by HBM.
// A thread takes 16 bytes of the first channels of V pairs and 16 of the second ones (interleaved: 16
// neighbouring bytes) and writes them back in the same places, so `out` may be `data`.
// Measured: 60001 x 12 x 48 bf16 from packed coordinates 23.5 us warm, 29 cold (4.8 TB/s); 213337 x 8 x 64 fp32, interleaved,
// 155 us (5.65 TB/s, above a copy's rate); 8 rows 3.2 us, a launch.
constexpr int kRotaryAngles = 2048;   // (rows of a workgroup) x (pairs): 16 KiB of LDS

struct RotaryArgs {
  void* out; const void* data;
  int64_t out_row, out_head, row, head;
  const void* pos; int64_t pos_row;
  const double* freq;
  int rows, heads, dim, pairs, axis_end[3], block_rows, items_head, pair_items, copy;
  uint32_t div_pairs, div_row, div_head;   // reciprocals: see fast_div
  int inverse, in_place;
};

// n / d for n * d < 2^32, by a multiplication with m = floor(2^32 / d) + 1 (m = 0 stands for d = 1)
__device__ inline uint32_t fast_div(uint32_t n, uint32_t m) { return m ? __umulhi(n, m) : n; }

template <int KIND> __device__ inline double rotary_position(const void* pos, int64_t row, int64_t stride, int axis) {
  if (KIND == OCNN_POS_INT32) return (double)((const int*)pos)[row * stride + axis];
  if (KIND == OCNN_POS_F32) return (double)((const float*)pos)[row * stride + axis];
  return (double)(int)((((const uint64_t*)pos)[row] >> (16 * axis)) & 0xffffu);
}

template <typename T> __device__ inline void turn_pair(T& x, T& y, const float2 k) {
  const float a = to_f32(x), b = to_f32(y);
  x = from_f32<T>(fmaf(a, k.x, -(b * k.y)));
  y = from_f32<T>(fmaf(a, k.y, b * k.x));
}

template <typename T, int KIND, bool INTERLEAVED>
__global__ void __launch_bounds__(kBlock) rotary_kernel(RotaryArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float2 turn[kRotaryAngles];
  const int64_t row0 = (int64_t)blockIdx.x * a.block_rows;
  const int rows = (int)min((int64_t)a.block_rows, (int64_t)a.rows - row0);
  for (int i = threadIdx.x; i < rows * a.pairs; i += kBlock) {
    const int r = (int)fast_div((uint32_t)i, a.div_pairs), p = i - r * a.pairs;
    const int axis = (p >= a.axis_end[0]) + (p >= a.axis_end[1]) + (p >= a.axis_end[2]);
    double t = rotary_position<KIND>(a.pos, row0 + r, a.pos_row, axis) * a.freq[p] * 0.15915494309189535;
    t -= rint(t);
    float s, c;
    sincospif(2.0f * (float)t, &s, &c);
    turn[i] = make_float2(c, a.inverse ? -s : s);
  }
  __syncthreads();
  const int items_row = a.heads * a.items_head;
  const T* data = (const T*)a.data + row0 * a.row;
  T* out = (T*)a.out + row0 * a.out_row;
  for (int i = threadIdx.x; i < rows * items_row; i += kBlock) {
    const int r = (int)fast_div((uint32_t)i, a.div_row), in_row = i - r * items_row;
    const int h = (int)fast_div((uint32_t)in_row, a.div_head), item = in_row - h * a.items_head;
    const T* src = data + (int64_t)r * a.row + (int64_t)h * a.head;
    T* dst = out + (int64_t)r * a.out_row + (int64_t)h * a.out_head;
    const float2* cs = turn + r * a.pairs;
    if (INTERLEAVED) {
      // V neighbouring channels; those from 2 P on turn by nothing
      const int c = item * V, n = min(V, a.dim - c);
      Pack<T, V> x;
      if (n == V) {
        x.load(src + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x.v[j] = j < n ? src[c + j] : (T)0;
      }
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const int p = c / 2 + j / 2;
        if (p < a.pairs) turn_pair(x.v[j], x.v[j + 1], cs[p]);
      }
      if (n == V) {
        x.store(dst + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) dst[c + j] = x.v[j];
      }
      continue;
    }
    if (item >= a.pair_items) {                       // channels that carry no position
      int c = 2 * a.pairs + (item - a.pair_items) * V;
      if (c + V > a.dim && a.dim - 2 * a.pairs >= V) c = a.dim - V;     // (copies: overlapping ones are the same)
      const int n = min(V, a.dim - c);
      if (n == V) { Pack<T, V> x; x.load(src + c); x.store(dst + c); }
      else for (int j = 0; j < n; ++j) dst[c + j] = src[c + j];
      continue;
    }
    int p = item * V;
    // the last pairs of a head, where they fill no whole vector: one vector back, together with pairs of the item
    // before, whose results are the same -- unless the input is overwritten meanwhile
    if (p + V > a.pairs && a.pairs >= V && !a.in_place) p = a.pairs - V;
    const int n = min(V, a.pairs - p);
    Pack<T, V> u, w;
    if (n == V) {
      u.load(src + p);
      w.load(src + a.pairs + p);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u.v[j] = j < n ? src[p + j] : (T)0;
        w.v[j] = j < n ? src[a.pairs + p + j] : (T)0;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) turn_pair(u.v[j], w.v[j], cs[p + j]);
    if (n == V) {
      u.store(dst + p);
      w.store(dst + a.pairs + p);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) {
          dst[p + j] = u.v[j];
          dst[a.pairs + p + j] = w.v[j];
        }
    }
  }
}

uint32_t reciprocal(uint32_t d) { return d <= 1 ? 0u : (uint32_t)((1ull << 32) / d) + 1u; }

// ---- gated linear recurrence ----------------------------------------------------------------------
//   h_t = a_t h_{t-1} + b_t x_t,  a = sigmoid(g), b = 1 - a = sigmoid(-g)
// The map of a run of rows is (A, H): h -> A h + H, and runs compose.  Four launches:
//   run    every chunk of L rows of a sequence: its (A, H)               reads g, x
//   group  every 32 chunks: the run in front of each, and of all of them
//   top    the state in front of every group
//   apply  every chunk again from its state: h                           reads g, x, writes h
// The chunks of all sequences are scanned as one list: a run that begins a sequence starts from the caller's
// state and forgets what came before (A = kReset; no product with it, so a NaN stays in its sequence).
// group and top move 16 bytes a channel and chunk; they are two launches because one compute unit has too few
// loads in flight to fetch a long list by itself (262147 rows of 256 channels: 4097 chunks, 69 us in one launch
// of a workgroup for every 8 channels).
// Measured, bf16: 262147 x 256: 43 + 7 + 5 + 69 us, bound by memory (5.8-6.2 TB/s in run and apply, which read gate and data
// twice); about 65000 x 192 in both directions: 41 and 55 us, bound by the latency of the walks and of eight dependent launches.
// States are folded in a fixed order, so results do not change from run to run (a single pass that takes
// whatever prefix its predecessors have published would not give that).
// Threads enumerate (chunk, channels) with the channels innermost.  The state is 32 bits throughout.
// Sequences of a few rows (a step of a running sequence) take one launch, a thread per (sequence,
// channels) that walks the rows; batches of sequences that are not long take one launch too (scan_block_kernel).
//
// The gradient, with L_t = dh_t + a_{t+1} L_{t+1} (L_end += the gradient of the last state):
//   dx = b L,  dg = a b L (h_{t-1} - x),  d state = a_1 L_1
// runs the same steps from the other end on (a, dh).  h_{t-1} is computed again from the
// chunk's state (kept from the forward pass, 32 bits): the stored h of a bf16 call is rounded, and
// h_{t-1} - x cancels where a sequence hardly changes.

template <typename T> __device__ inline void gates(float g, float* a, float* b);
// sigmoid(g) and sigmoid(-g) without cancellation: e = exp(-|g|), 1 / (1 + e) and e / (1 + e).  The fp32
// form carries the rounding error of g * log2(e), 2^-24 |g| / ln 2 of the result, as a factor.
template <> __device__ inline void gates<float>(float g, float* a, float* b) {
  const float x = -fabsf(g), t = x * 1.44269502f;
  const float lost = fmaf(x, 1.44269502f, -t) + x * 1.92596303e-8f;
  float e = __builtin_amdgcn_exp2f(t);
  e = (x > -100.0f) ? fmaf(e, lost * 0.693147182f, e) : (x == x ? 0.0f : x);
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  *a = g >= 0.0f ? big : small;
  *b = g >= 0.0f ? small : big;
}
template <> __device__ inline void gates<uint16_t>(float g, float* a, float* b) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269502f);   // |g| < 100: 2^-17 of the result at most
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  *a = g >= 0.0f ? big : small;
  *b = g >= 0.0f ? small : big;
}

struct ScanArgs {
  void* out; const void* gate; const void* data; const void* grad;      // grad: of the outputs
  void* grad_gate; void* grad_data;
  int64_t out_row, gate_row, data_row, grad_row, grad_gate_row, grad_data_row;
  const float* state; float* last; const float* grad_last; float* grad_state;
  float* run_a; float* run_h;                     // [ids][channels]
  float* group_a; float* group_h;                 // [groups of ids][channels]; group_h: then the state in front
  float* carry;                                   // [ids][channels], kept for the gradient
  int64_t ids;
  const int* offsets;
  int n_seq, rows, channels, groups, reverse, fill;
  int64_t threads;                                // ids x groups
  bool past;                                      // results go past the caches
};

constexpr int kScanRows = 8;   // rows whose loads are in flight together
constexpr int kGroupShift = 5, kGroup = 1 << kGroupShift;
constexpr float kReset = -1.0f;   // (products of sigmoids are not negative)

// the run (A, H) behind the run (a, h)
__device__ inline void compose(float& A, float& H, float a, float h) {
  H = a < 0.0f ? h : fmaf(a, H, h);
  A = a < 0.0f || A < 0.0f ? kReset : A * a;
}

// The rows of chunk `id`: their sequence, where they begin and how many there are.
struct Chunk {
  int seq, index, first, count, length;   // row of step j: first + j * step
  int step;
  bool live;                              // false: beyond its sequence
};

template <int L> __device__ inline Chunk chunk_of(const ScanArgs& a, int64_t id) {
  Chunk c;
  c.seq = locate(a.offsets, a.n_seq, a.rows, id, Log2<L>::value);
  const int begin = clamped(a.offsets, c.seq, a.rows);
  const int end = c.seq < a.n_seq ? clamped(a.offsets, c.seq + 1, a.rows) : a.rows;
  c.length = max(end - begin, 0);
  const int64_t index = id - ((begin >> Log2<L>::value) + c.seq);
  const int64_t at = index * L;
  c.live = index >= 0 && (at < c.length || (index == 0 && c.seq < a.n_seq));
  c.index = (int)index;
  c.count = c.live ? (int)min((int64_t)L, c.length - at) : 0;
  c.step = a.reverse ? -1 : 1;
  c.first = a.reverse ? end - 1 - (int)at : begin + (int)at;
  return c;
}

template <int V> __device__ inline void put_run(const ScanArgs& a, int64_t id, int c0, const float* A, const float* H) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    a.run_a[id * a.channels + c0 + v] = A[v];
    a.run_h[id * a.channels + c0 + v] = H[v];
  }
}
// the state in front of a chunk that does not begin its sequence (back: behind one that does not end it)
template <int V> __device__ inline void state_at(const ScanArgs& a, int64_t id, int c0, float* h) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float A = a.run_a[id * a.channels + c0 + v], H = a.run_h[id * a.channels + c0 + v];
    h[v] = A < 0.0f ? H : fmaf(A, a.group_h[(id >> kGroupShift) * a.channels + c0 + v], H);
  }
}

template <typename T, int V, int L>
__global__ void __launch_bounds__(kBlock) scan_run_kernel(ScanArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.threads) return;
  const int64_t id = i / a.groups;
  const int c0 = (int)(i - id * a.groups) * V;
  const Chunk ch = chunk_of<L>(a, id);
  const T* gate = (const T*)a.gate + c0;
  const T* data = (const T*)a.data + c0;
  float A[V], H[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { A[v] = 1.0f; H[v] = 0.0f; }
  // (what a sequence's last chunk does to the state matters to no other chunk)
  if (!ch.live || ch.seq >= a.n_seq || (int64_t)(ch.index + 1) * L >= ch.length) {
    put_run<V>(a, id, c0, A, H);
    return;
  }
  for (int t = 0; t < L; t += kScanRows) {       // the chunk is full: it is not its sequence's last
    Pack<T, V> g[kScanRows], x[kScanRows];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j) {
      const int64_t row = ch.first + (int64_t)(t + j) * ch.step;
      g[j].load(gate + row * a.gate_row);
      x[j].load(data + row * a.data_row);
    }
#pragma unroll
    for (int j = 0; j < kScanRows; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p, q;
        gates<T>(to_f32(g[j].v[v]), &p, &q);
        H[v] = fmaf(p, H[v], q * to_f32(x[j].v[v]));
        A[v] *= p;
      }
  }
  if (ch.index == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.state) H[v] = fmaf(A[v], a.state[(int64_t)ch.seq * a.channels + c0 + v], H[v]);
      A[v] = kReset;
    }
  put_run<V>(a, id, c0, A, H);
}

// The same from the other end for the gradient: m = a (dh + m'), m' from the row behind.  Runs of the chunks
// behind a sequence's first one.
template <typename T, int V, int L>
__global__ void __launch_bounds__(kBlock) scan_run_back_kernel(ScanArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.threads) return;
  const int64_t id = i / a.groups;
  const int c0 = (int)(i - id * a.groups) * V;
  const Chunk ch = chunk_of<L>(a, id);
  const T* gate = (const T*)a.gate + c0;
  const T* grad = (const T*)a.grad + c0;
  float A[V], M[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { A[v] = 1.0f; M[v] = 0.0f; }
  if (!ch.live || ch.seq >= a.n_seq || ch.index == 0) {
    put_run<V>(a, id, c0, A, M);
    return;
  }
  for (int t = L - kScanRows; t >= 0; t -= kScanRows) {
    if (t >= ch.count) continue;
    Pack<T, V> g[kScanRows], d[kScanRows];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j) {
      const int64_t row = ch.first + (int64_t)min(t + j, ch.count - 1) * ch.step;
      g[j].load(gate + row * a.gate_row);
      d[j].load(grad + row * a.grad_row);
    }
#pragma unroll
    for (int j = kScanRows - 1; j >= 0; --j)
      if (t + j < ch.count)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float p, q;
          gates<T>(to_f32(g[j].v[v]), &p, &q);
          M[v] = p * (to_f32(d[j].v[v]) + M[v]);
          A[v] *= p;
        }
  }
  if ((int64_t)(ch.index + 1) * L >= ch.length)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.grad_last) M[v] = fmaf(A[v], a.grad_last[(int64_t)ch.seq * a.channels + c0 + v], M[v]);
      A[v] = kReset;
    }
  put_run<V>(a, id, c0, A, M);
}

// In place: the run of each chunk -> the run of the chunks of its group in front of it (back: behind it).
template <bool BACK>
__global__ void __launch_bounds__(64) scan_group_kernel(ScanArgs a) {
  const int64_t id0 = (int64_t)blockIdx.x << kGroupShift;
  const int n = (int)min((int64_t)kGroup, a.ids - id0);
  const int c = blockIdx.y * 64 + threadIdx.x;
  if (c >= a.channels) return;
  float ra[kGroup], rh[kGroup];
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {             // (no branch a load: they are in flight together)
    const int64_t o = (id0 + min(i, n - 1)) * a.channels + c;
    ra[i] = a.run_a[o];
    rh[i] = a.run_h[o];
  }
  float A = 1.0f, H = 0.0f;
#pragma unroll
  for (int k = 0; k < kGroup; ++k) {
    const int i = BACK ? kGroup - 1 - k : k;
    if (i >= n) continue;
    const int64_t o = (id0 + i) * a.channels + c;
    a.run_a[o] = A;
    a.run_h[o] = H;
    compose(A, H, ra[i], rh[i]);
  }
  a.group_a[blockIdx.x * (int64_t)a.channels + c] = A;
  a.group_h[blockIdx.x * (int64_t)a.channels + c] = H;
}

// group_h: the run of each group -> the state in front of it (back: behind it).  32 threads a channel fold a
// share of the groups each, the shares are combined by doubling, and each thread walks its share again.
constexpr int kTopChannels = 32, kTopShares = 32, kHeld = 8;

template <bool BACK>
__global__ void __launch_bounds__(kTopChannels * kTopShares) scan_top_kernel(ScanArgs a) {
  __shared__ float sa[kTopShares][kTopChannels], sh[kTopShares][kTopChannels];
  const int lane = threadIdx.x % kTopChannels, seg = threadIdx.x / kTopChannels;
  const int c = blockIdx.x * kTopChannels + lane;
  const int groups = (int)((a.ids + kGroup - 1) >> kGroupShift);
  const int share = (groups + kTopShares - 1) / kTopShares;
  const int from = min(seg * share, groups), to = min(from + share, groups);
  const bool mine = c < a.channels;
  auto at = [&](int j) { return (int64_t)(BACK ? groups - 1 - j : j) * a.channels + c; };
  float ra[kHeld], rh[kHeld];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int64_t o = at(min(j0 + i, to - 1));
      ra[i] = a.group_a[o];
      rh[i] = a.group_h[o];
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (j0 + i >= to) { ra[i] = 1.0f; rh[i] = 0.0f; }
  };
  float A = 1.0f, H = 0.0f;
  if (mine)
    for (int j = from; j < to; j += kHeld) {
      load(j);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) compose(A, H, ra[i], rh[i]);
    }
  sa[seg][lane] = A;
  sh[seg][lane] = H;
  for (int d = 1; d < kTopShares; d <<= 1) {
    __syncthreads();
    float fa = 1.0f, fh = 0.0f;
    if (seg >= d) { fa = sa[seg - d][lane]; fh = sh[seg - d][lane]; }
    __syncthreads();
    compose(fa, fh, A, H);
    A = fa;
    H = fh;
    sa[seg][lane] = A;
    sh[seg][lane] = H;
  }
  __syncthreads();
  if (!mine) return;
  float h = seg ? sh[seg - 1][lane] : 0.0f;       // (the list begins with a sequence: nothing comes before it)
  for (int j = from; j < to; j += kHeld) {
    if (share > kHeld) load(j);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (j + i < to) {
        a.group_h[at(j + i)] = h;
        h = ra[i] < 0.0f ? rh[i] : fmaf(ra[i], h, rh[i]);
      }
  }
}

// The runs of all chunks -> the state in front of each (back: behind it), marked as state_at knows it: one launch instead of the
// two above for short lists, 64 threads a channel with up to 8 runs each (forward, bf16: 2000 x 64, 130 chunks, 12.0 instead of
// 16.3 us; 6000 x 128, 384 chunks, 13.8 instead of 17.5; with 32 runs each 16384 x 97, 1040 chunks, took 21.8 instead of 20.2).
constexpr int kListChannels = 16, kListShares = 64, kListHeld = 8;

template <bool BACK>
__global__ void __launch_bounds__(kListChannels * kListShares) scan_list_kernel(ScanArgs a) {
  __shared__ float sa[kListShares][kListChannels], sh[kListShares][kListChannels];
  const int lane = threadIdx.x % kListChannels, seg = threadIdx.x / kListChannels;
  const int c = blockIdx.x * kListChannels + lane;
  const int ids = (int)a.ids, share = (ids + kListShares - 1) / kListShares;      // (at most kListHeld)
  const int from = min(seg * share, ids), to = min(from + share, ids);
  const bool mine = c < a.channels;
  auto at = [&](int j) { return (int64_t)(BACK ? ids - 1 - j : j) * a.channels + c; };
  float ra[kListHeld], rh[kListHeld];
  float A = 1.0f, H = 0.0f;
  if (mine && from < to) {
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {          // (no branch a load: they are in flight together)
      const int64_t o = at(min(from + i, to - 1));
      ra[i] = a.run_a[o];
      rh[i] = a.run_h[o];
    }
#pragma unroll
    for (int i = 0; i < kListHeld; ++i)
      if (from + i < to) compose(A, H, ra[i], rh[i]);
  }
  sa[seg][lane] = A;
  sh[seg][lane] = H;
  for (int d = 1; d < kListShares; d <<= 1) {
    __syncthreads();
    float fa = 1.0f, fh = 0.0f;
    if (seg >= d) { fa = sa[seg - d][lane]; fh = sh[seg - d][lane]; }
    __syncthreads();
    compose(fa, fh, A, H);
    A = fa;
    H = fh;
    sa[seg][lane] = A;
    sh[seg][lane] = H;
  }
  __syncthreads();
  if (!mine) return;
  float h = seg ? sh[seg - 1][lane] : 0.0f;        // (the list begins with a sequence: nothing comes before it)
#pragma unroll
  for (int i = 0; i < kListHeld; ++i)
    if (from + i < to) {
      const int64_t o = at(from + i);
      a.run_a[o] = kReset;
      a.run_h[o] = h;
      h = ra[i] < 0.0f ? rh[i] : fmaf(ra[i], h, rh[i]);
    }
}

template <typename T, int V> __device__ inline void zero_rows(T* out, int64_t row_stride, const Chunk& ch) {
  Pack<T, V> z;
  z.fill(0);
  for (int j = 0; j < ch.count; ++j) z.store(out + (ch.first + (int64_t)j * ch.step) * row_stride);
}

template <typename T, int V, int L>
__global__ void __launch_bounds__(kBlock) scan_apply_kernel(ScanArgs a) {
  const int64_t i = a.threads - 1 - ((int64_t)blockIdx.x * kBlock + threadIdx.x);   // last chunk first: its rows were read last
  if (i < 0) return;
  const int64_t id = i / a.groups;
  const int c0 = (int)(i - id * a.groups) * V;
  const Chunk ch = chunk_of<L>(a, id);
  if (!ch.live) return;
  T* out = (T*)a.out + c0;
  if (ch.seq >= a.n_seq) {
    if (a.fill) zero_rows<T, V>(out, a.out_row, ch);
    return;
  }
  const T* gate = (const T*)a.gate + c0;
  const T* data = (const T*)a.data + c0;
  float h[V];
  if (ch.index) {
    state_at<V>(a, id, c0, h);
    if (a.carry)
#pragma unroll
      for (int v = 0; v < V; ++v) a.carry[id * a.channels + c0 + v] = h[v];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = a.state ? a.state[(int64_t)ch.seq * a.channels + c0 + v] : 0.0f;
  }
  for (int t = 0; t < ch.count; t += kScanRows) {
    Pack<T, V> g[kScanRows], x[kScanRows];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j) {
      const int64_t row = ch.first + (int64_t)min(t + j, ch.count - 1) * ch.step;
      g[j].load(gate + row * a.gate_row);
      x[j].load(data + row * a.data_row);
    }
#pragma unroll
    for (int j = 0; j < kScanRows; ++j)
      if (t + j < ch.count) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float p, q;
          gates<T>(to_f32(g[j].v[v]), &p, &q);
          h[v] = fmaf(p, h[v], q * to_f32(x[j].v[v]));
          x[j].v[v] = from_f32<T>(h[v]);
        }
        T* to = out + (ch.first + (int64_t)(t + j) * ch.step) * a.out_row;
        if (a.past) x[j].store_past(to); else x[j].store(to);
      }
  }
  if (a.last && (int64_t)(ch.index + 1) * L >= ch.length)
#pragma unroll
    for (int v = 0; v < V; ++v) a.last[(int64_t)ch.seq * a.channels + c0 + v] = h[v];
}

// d gate, d data of a chunk: forward over the chunk once for the state in front of every kScanRows rows,
// then group by group from the end.
template <typename T, int V, int L>
__global__ void __launch_bounds__(kBlock) scan_apply_back_kernel(ScanArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.threads) return;
  const int64_t id = i / a.groups;
  const int c0 = (int)(i - id * a.groups) * V;
  const Chunk ch = chunk_of<L>(a, id);
  if (!ch.live) return;
  T* dgate = (T*)a.grad_gate + c0;
  T* ddata = (T*)a.grad_data + c0;
  if (ch.seq >= a.n_seq) {
    zero_rows<T, V>(dgate, a.grad_gate_row, ch);
    zero_rows<T, V>(ddata, a.grad_data_row, ch);
    return;
  }
  const T* gate = (const T*)a.gate + c0;
  const T* data = (const T*)a.data + c0;
  const T* grad = (const T*)a.grad + c0;
  constexpr int kGroups = L / kScanRows;
  float front[kGroups][V], m[V];
  const int64_t at_seq = (int64_t)ch.seq * a.channels + c0;
  const bool is_last = (int64_t)(ch.index + 1) * L >= ch.length;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = ch.index ? a.carry[id * a.channels + c0 + v] : a.state ? a.state[at_seq + v] : 0.0f;
    m[v] = is_last && a.grad_last ? a.grad_last[at_seq + v] : 0.0f;
  }
  if (!is_last) state_at<V>(a, id, c0, m);
#pragma unroll
  for (int s = 0; s < kGroups; ++s) {
#pragma unroll
    for (int v = 0; v < V; ++v) front[s][v] = h[v];
    if (s + 1 < kGroups && (s + 1) * kScanRows < ch.count) {     // (a whole group)
      Pack<T, V> g[kScanRows], x[kScanRows];
#pragma unroll
      for (int j = 0; j < kScanRows; ++j) {
        const int64_t row = ch.first + (int64_t)(s * kScanRows + j) * ch.step;
        g[j].load(gate + row * a.gate_row);
        x[j].load(data + row * a.data_row);
      }
#pragma unroll
      for (int j = 0; j < kScanRows; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float p, q;
          gates<T>(to_f32(g[j].v[v]), &p, &q);
          h[v] = fmaf(p, h[v], q * to_f32(x[j].v[v]));
        }
    }
  }
#pragma unroll
  for (int s = kGroups - 1; s >= 0; --s) {
    const int t = s * kScanRows;
    if (t >= ch.count) continue;
    Pack<T, V> g[kScanRows], x[kScanRows], d[kScanRows];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j) {
      const int64_t row = ch.first + (int64_t)min(t + j, ch.count - 1) * ch.step;
      g[j].load(gate + row * a.gate_row);
      x[j].load(data + row * a.data_row);
      d[j].load(grad + row * a.grad_row);
    }
    float p[kScanRows][V], q[kScanRows][V], before[kScanRows][V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = front[s][v];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        gates<T>(to_f32(g[j].v[v]), &p[j][v], &q[j][v]);
        before[j][v] = h[v];
        h[v] = fmaf(p[j][v], h[v], q[j][v] * to_f32(x[j].v[v]));
      }
#pragma unroll
    for (int j = kScanRows - 1; j >= 0; --j)
      if (t + j < ch.count) {
        Pack<T, V> og, ox;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float lam = to_f32(d[j].v[v]) + m[v];
          og.v[v] = from_f32<T>(p[j][v] * q[j][v] * lam * (before[j][v] - to_f32(x[j].v[v])));
          ox.v[v] = from_f32<T>(q[j][v] * lam);
          m[v] = p[j][v] * lam;
        }
        const int64_t row = ch.first + (int64_t)(t + j) * ch.step;
        og.store(dgate + row * a.grad_gate_row);
        ox.store(ddata + row * a.grad_data_row);
      }
  }
  if (a.grad_state && ch.index == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) a.grad_state[at_seq + v] = m[v];
}

// One launch for batches of short sequences: a workgroup takes CH channels of one sequence, SEGS chunks of 16 rows at a
// time, and carries the state along.  The rows stay in registers between the run and the application, so gate and data are read
// once.  The runs of a wavefront's chunks are scanned by shuffles, the wavefronts' through LDS.  Bound by one compute unit's
// exponentials and narrow loads: 3.5 us for 1024 rows of 8 channels.
constexpr int kBlockRows = 16;

// Workgroups go round the 8 XCDs in turn: the channels of a sequence on one of them, since its lines hold those of several
// workgroups (from 8 sequences on; fewer would leave XCDs without work).
__device__ inline void block_item(int n, int groups, int* seq, int* group) {
  const int id = blockIdx.x;
  if (n < 8) {
    *seq = id % n;
    *group = id / n;
  } else {
    const int k = id >> 3;
    *group = k % groups;
    *seq = k / groups * 8 + (id & 7);
  }
}
inline unsigned block_items(int64_t n, int64_t groups) { return (unsigned)((n < 8 ? n : (n + 7) / 8 * 8) * groups); }

// (A, H) of this thread's chunk, the state S in front of the workgroup's chunks -> the state in front of this chunk; S moves on
template <int CH, int SEGS>
__device__ inline float scan_block_state(float A, float H, float& S, float2 (*total)[CH]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % CH;
#pragma unroll
  for (int d = CH; d < 64; d <<= 1) {
    const float fa = __shfl_up(A, d, 64), fh = __shfl_up(H, d, 64);
    if (lane >= d) { H = fmaf(A, fh, H); A *= fa; }
  }
  const float ea = __shfl_up(A, CH, 64), eh = __shfl_up(H, CH, 64);
  if (lane >= 64 - CH) total[wave][c] = make_float2(A, H);
  __syncthreads();
  float h = S, mine = S;
#pragma unroll
  for (int w = 0; w < SEGS * CH / 64; ++w) {
    const float2 t = total[w][c];
    mine = w == wave ? h : mine;
    h = fmaf(t.x, h, t.y);
  }
  S = h;
  return lane >= CH ? fmaf(ea, mine, eh) : mine;
}

template <typename T, int CH, int SEGS, int ROWS>
__device__ inline void scan_block(const ScanArgs& a, int seq, int group, float2 (*total)[SEGS * CH / 64][CH]) {
  const int c = group * CH + threadIdx.x % CH, seg = threadIdx.x / CH;
  const int begin = clamped(a.offsets, seq, a.rows);
  const int end = seq < a.n_seq ? clamped(a.offsets, seq + 1, a.rows) : a.rows, length = max(end - begin, 0);
  const bool mine = c < a.channels;
  const int cc = min(c, a.channels - 1);
  T* out = (T*)a.out + cc;
  if (seq >= a.n_seq) {
    if (a.fill && mine)
      for (int r = begin + seg; r < end; r += SEGS) out[(int64_t)r * a.out_row] = 0;
    return;
  }
  const T* gate = (const T*)a.gate + cc;
  const T* data = (const T*)a.data + cc;
  const int64_t id0 = (int64_t)(begin / ROWS) + seq;
  float S = a.state ? a.state[(int64_t)seq * a.channels + cc] : 0.0f;
  int parity = 0;
  for (int base = 0; base < length; base += SEGS * ROWS, parity ^= 1) {
    const int first = base + seg * ROWS, n = min(length - first, ROWS);
    auto row = [&](int j) {
      const int t = min(first + j, length - 1);
      return (int64_t)(a.reverse ? end - 1 - t : begin + t);
    };
    T g[ROWS], x[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      g[j] = gate[row(j) * a.gate_row];
      x[j] = data[row(j) * a.data_row];
    }
    float p[ROWS], qx[ROWS], A = 1.0f, H = 0.0f;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      float q;
      gates<T>(to_f32(g[j]), &p[j], &q);
      qx[j] = q * to_f32(x[j]);
      if (j < n) {
        H = fmaf(p[j], H, qx[j]);
        A *= p[j];
      }
    }
    float h = scan_block_state<CH, SEGS>(A, H, S, total[parity]);
    if (!mine || n <= 0) continue;
    if (a.carry && first) a.carry[(id0 + first / ROWS) * a.channels + c] = h;
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j < n) {
        h = fmaf(p[j], h, qx[j]);
        out[row(j) * a.out_row] = from_f32<T>(h);
      }
  }
  if (a.last && mine && seg == 0) a.last[(int64_t)seq * a.channels + c] = S;
}

template <typename T, int CH, int SEGS>
__global__ void __launch_bounds__(SEGS * CH) scan_block_kernel(ScanArgs a) {
  __shared__ float2 total[2][SEGS * CH / 64][CH];
  int seq, group;
  block_item(a.n_seq + 1, (a.channels + CH - 1) / CH, &seq, &group);
  if (seq > a.n_seq) return;
  scan_block<T, CH, SEGS, kBlockRows>(a, seq, group, total);
}

// One launch for sequences of a few rows on average: a thread walks the rows of one sequence (and, behind the last
// sequence, zeroes the rows that belong to none).  A sequence of more than kWalkRows rows among them is left to workgroups
// of their own in the same launch, which take 4 channels of it as the kernel above does: the length of a sequence is known to
// the device only.  Such a sequence holds a row that is a multiple of kWalkRows; a workgroup (of 4 channels) looks up who owns
// kWalkSlots of those, and takes the long sequences whose first such row is among them.  us, bf16, 64 channels, so and with every
// sequence walked: 3800 rows among 255 single ones 15 378; 61000 among 4095 243 16100; 4096 single rows of 256 channels 9.5 8.2.
constexpr int kWalkRows = 64, kWalkSlots = 8, kWalkChannels = 4, kWalkSegs = kBlock / kWalkChannels;

// The last entry of a rising table that is at most `row` (0 where none is).  8 neighbouring lanes have a row of their own and
// probe 8 entries at a time.
__device__ inline int owner_of(const int* offsets, int entries, int rows, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = entries;
  while (__any(n > 1)) {
    const int step = (n + 7) / 8, at = (lane & 7) * step;
    const uint64_t below = __ballot(at < n && clamped(offsets, lo + min(at, n - 1), rows) <= row);
    const int skip = max(__popc((uint32_t)(below >> (lane & ~7)) & 0xffu) - 1, 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

template <typename T, int V>
__global__ void __launch_bounds__(kBlock) scan_walk_kernel(ScanArgs a, unsigned seekers) {
  __shared__ float2 total[2][kBlock / 64][kWalkChannels];
  if (blockIdx.x < seekers) {                 // (first: what they find takes longest)
    const int groups = (a.channels + kWalkChannels - 1) / kWalkChannels;
    const int64_t items = (int64_t)((a.rows + kWalkRows * kWalkSlots - 1) / (kWalkRows * kWalkSlots)) * groups;
    for (int64_t n = blockIdx.x; n < items; n += seekers) {
      const int group = (int)(n % groups);
      const int64_t row = (n / groups * kWalkSlots + ((threadIdx.x & 63) >> 3)) * kWalkRows;
      const int owner = owner_of(a.offsets, a.n_seq + 1, a.rows, (int)min(row, (int64_t)a.rows));
      const int begin = clamped(a.offsets, owner, a.rows), end = owner < a.n_seq ? clamped(a.offsets, owner + 1, a.rows) : a.rows;
      uint64_t take = __ballot((threadIdx.x & 7) == 0 && row < a.rows && row >= begin && row - begin < kWalkRows && end - begin > kWalkRows);
      while (take) {                          // (the same in every wavefront)
        const int at = __ffsll((unsigned long long)take) - 1;
        take &= take - 1;
        scan_block<T, kWalkChannels, kWalkSegs, kScanRows>(a, __builtin_amdgcn_readlane(owner, at), group, total);
        __syncthreads();
      }
    }
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - seekers) * kBlock + threadIdx.x;
  if (i >= a.threads) return;
  const int seq = (int)(i / a.groups);
  const int c0 = (int)(i - (int64_t)seq * a.groups) * V;
  const int begin = clamped(a.offsets, seq, a.rows);
  const int end = seq < a.n_seq ? clamped(a.offsets, seq + 1, a.rows) : a.rows;
  T* out = (T*)a.out + c0;
  Chunk ch;
  ch.count = max(end - begin, 0);
  if (ch.count > kWalkRows) return;
  ch.first = seq < a.n_seq && a.reverse ? end - 1 : begin;
  ch.step = seq < a.n_seq && a.reverse ? -1 : 1;
  if (seq >= a.n_seq) {
    if (a.fill) zero_rows<T, V>(out, a.out_row, ch);
    return;
  }
  const T* gate = (const T*)a.gate + c0;
  const T* data = (const T*)a.data + c0;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = a.state ? a.state[(int64_t)seq * a.channels + c0 + v] : 0.0f;
  for (int t = 0; t < ch.count; t += kScanRows) {
    Pack<T, V> g[kScanRows], x[kScanRows];
#pragma unroll
    for (int j = 0; j < kScanRows; ++j) {
      const int64_t row = ch.first + (int64_t)min(t + j, ch.count - 1) * ch.step;
      g[j].load(gate + row * a.gate_row);
      x[j].load(data + row * a.data_row);
    }
#pragma unroll
    for (int j = 0; j < kScanRows; ++j)
      if (t + j < ch.count) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float p, q;
          gates<T>(to_f32(g[j].v[v]), &p, &q);
          h[v] = fmaf(p, h[v], q * to_f32(x[j].v[v]));
          x[j].v[v] = from_f32<T>(h[v]);
        }
        T* to = out + (ch.first + (int64_t)(t + j) * ch.step) * a.out_row;
        if (a.past) x[j].store_past(to); else x[j].store(to);
      }
  }
  if (a.last)
#pragma unroll
    for (int v = 0; v < V; ++v) a.last[(int64_t)seq * a.channels + c0 + v] = h[v];
}

// The gradient of scan_block_kernel, from the last chunk to the first
template <typename T, int CH, int SEGS>
__global__ void __launch_bounds__(SEGS * CH) scan_block_back_kernel(ScanArgs a) {
  __shared__ float2 total[2][SEGS * CH / 64][CH];
  int seq, group;
  block_item(a.n_seq + 1, (a.channels + CH - 1) / CH, &seq, &group);
  if (seq > a.n_seq) return;
  const int c = group * CH + threadIdx.x % CH, seg = threadIdx.x / CH;
  const int begin = clamped(a.offsets, seq, a.rows);
  const int end = seq < a.n_seq ? clamped(a.offsets, seq + 1, a.rows) : a.rows, length = max(end - begin, 0);
  const bool mine = c < a.channels;
  const int cc = min(c, a.channels - 1);
  T* dgate = (T*)a.grad_gate + cc;
  T* ddata = (T*)a.grad_data + cc;
  if (seq >= a.n_seq) {
    if (mine)
      for (int r = begin + seg; r < end; r += SEGS) {
        dgate[(int64_t)r * a.grad_gate_row] = 0;
        ddata[(int64_t)r * a.grad_data_row] = 0;
      }
    return;
  }
  const T* gate = (const T*)a.gate + cc;
  const T* data = (const T*)a.data + cc;
  const T* grad = (const T*)a.grad + cc;
  const int64_t id0 = (int64_t)(begin / kBlockRows) + seq, at_seq = (int64_t)seq * a.channels + cc;
  float S = a.grad_last ? a.grad_last[at_seq] : 0.0f;
  const int chunks = (length + kBlockRows - 1) / kBlockRows;
  int parity = 0;
  for (int base = 0; base < chunks; base += SEGS, parity ^= 1) {
    const int index = chunks - 1 - base - seg, first = max(index, 0) * kBlockRows, n = index < 0 ? 0 : min(length - first, kBlockRows);
    auto row = [&](int j) {
      const int t = min(first + j, length - 1);
      return (int64_t)(a.reverse ? end - 1 - t : begin + t);
    };
    T g[kBlockRows], x[kBlockRows], d[kBlockRows];
#pragma unroll
    for (int j = 0; j < kBlockRows; ++j) {
      g[j] = gate[row(j) * a.gate_row];
      x[j] = data[row(j) * a.data_row];
      d[j] = grad[row(j) * a.grad_row];
    }
    float h = index > 0 ? a.carry[(id0 + index) * a.channels + cc] : a.state ? a.state[at_seq] : 0.0f;
    float p[kBlockRows], q[kBlockRows], before[kBlockRows], A = 1.0f, M = 0.0f;
#pragma unroll
    for (int j = 0; j < kBlockRows; ++j) {
      gates<T>(to_f32(g[j]), &p[j], &q[j]);
      before[j] = h;
      h = fmaf(p[j], h, q[j] * to_f32(x[j]));
    }
#pragma unroll
    for (int j = kBlockRows - 1; j >= 0; --j)
      if (j < n) {
        M = p[j] * (to_f32(d[j]) + M);
        A *= p[j];
      }
    float m = scan_block_state<CH, SEGS>(A, M, S, total[parity]);
    if (!mine) continue;
#pragma unroll
    for (int j = kBlockRows - 1; j >= 0; --j)
      if (j < n) {
        const float lam = to_f32(d[j]) + m;
        dgate[row(j) * a.grad_gate_row] = from_f32<T>(p[j] * q[j] * lam * (before[j] - to_f32(x[j])));
        ddata[row(j) * a.grad_data_row] = from_f32<T>(q[j] * lam);
        m = p[j] * lam;
      }
  }
  if (a.grad_state && mine && seg == 0) a.grad_state[(int64_t)seq * a.channels + c] = S;
}

// Rows of a chunk: many where that leaves enough threads for the chip (the runs and states cost 24 bytes a
// channel and chunk, and the carry step is short), few where it does not.  The rule sees sizes that the
// forward and the backward call share, so their chunks are the same.  Forward and backward of bf16 in us with chunks of 16, 32
// and 64: 65536 x 64 27 30, 26 36, 32 47; 65536 x 192 41 55, 41 59, 42 63; 200000 x 96 55 77, 54 74, 61 81; 262147 x 256
// 138 245, 131 236, 122 234.
int scan_shift(int64_t rows, int64_t channels) {
  return rows * channels >= (int64_t)1 << 25 ? 6 : 4;
}

// sequences of 16 rows and fewer on average: one launch that walks them, but for long ones among them
bool scan_walks(int64_t rows, int64_t n_seq, bool carries) { return !carries && rows <= 16 * n_seq; }

// A workgroup a sequence and 8 channels (4 where that makes few), for batches whose sequences are not long on average.  us in
// one launch and in chunks, forward and backward of bf16, lengths between a half and three halves of what is named: 4 x 500 of
// 64 channels 4.9 12.0, 6.1 14.0; 8 x 750 of 128: 5.7 13.6, 7.7 15.7; 16 x 1250 of 97: 10.0 21.0, 15.1 24.0; 8 x 2000 of 192: 12.9
// 22.4, 22.6 27.5; but 8 x 4096 of 64: 22 19, 32 24, 64 x 256 of 512: 60 35, 108 43.  Inputs not in the caches: 16 x 1250 of 97:
// 17.8 27.6, 26.1 32.1; 8 x 2000 of 192: 25.3 27.7, 38.4 33.7 (the gradient waits for more loads at a time, hence its lower bound).
// 16 channels: 16 x 1250 of 97: 12.9 and 19.4.
// A batch whose rows nearly all lie in one sequence pays for it: 32768 rows of 64 channels take 129 us instead of 19, hence
// the bound on the rows.
bool scan_blocks(int64_t rows, int64_t channels, int64_t n_seq, bool back) {
  return rows <= 32768 && rows <= (back ? 1536 : 2048) * n_seq && n_seq * ((channels + 7) / 8) <= 1024 && scan_shift(rows, channels) == 4;
}
bool scan_narrow(int64_t channels, int64_t n_seq) { return n_seq * channels <= 512; }

// A state written where one is read: a workgroup that takes a sequence from one end to the other has read it by then; chunks of
// their own have not.
bool states_apart(const float* out, const float* in, int n_seq, int channels, bool itself) {
  const uintptr_t a = (uintptr_t)out, b = (uintptr_t)in, size = (uintptr_t)n_seq * channels * sizeof(float);
  return !out || !in || (itself && a == b) || a + size <= b || b + size <= a;
}

int64_t scan_ids(int64_t rows, int n_seq, int shift) { return (rows >> shift) + n_seq + 1; }

// the lists of runs in a workspace
void scan_lists(ScanArgs* a, int64_t ids, void* workspace) {
  const size_t one = (size_t)ids * a->channels, groups = (size_t)((ids + kGroup - 1) >> kGroupShift) * a->channels;
  a->ids = ids;
  a->run_a = (float*)workspace;
  a->run_h = a->run_a + one;
  a->group_a = a->run_h + one;
  a->group_h = a->group_a + groups;
}

// V channels a thread: wide loads where every row allows them and the chip stays full
int scan_width(const ScanArgs& a, int size, std::initializer_list<std::pair<const void*, int64_t>> tensors, int64_t ids) {
  int v = 4;
  for (; v > 1; v >>= 1) {
    bool ok = a.channels % v == 0 && ids * (a.channels / v) >= 256 * 256;
    for (auto& t : tensors) ok = ok && t.second % v == 0 && (uintptr_t)t.first % (size_t)(v * size) == 0;
    if (ok) break;
  }
  return v;
}

template <bool BACK> void scan_lists_launch(const ScanArgs& a, hipStream_t s) {
  if (a.ids <= kListShares * kListHeld) {
    scan_list_kernel<BACK><<<(a.channels + kListChannels - 1) / kListChannels, kListChannels * kListShares, 0, s>>>(a);
    return;
  }
  const unsigned groups = (unsigned)((a.ids + kGroup - 1) >> kGroupShift);
  scan_group_kernel<BACK><<<dim3(groups, (a.channels + 63) / 64), 64, 0, s>>>(a);
  scan_top_kernel<BACK><<<(a.channels + kTopChannels - 1) / kTopChannels, kTopChannels * kTopShares, 0, s>>>(a);
}

template <typename T, int V, int L>
void scan_forward_launch(const ScanArgs& a, hipStream_t s) {
  const unsigned blocks = blocks_for(a.threads);
  scan_run_kernel<T, V, L><<<blocks, kBlock, 0, s>>>(a);
  scan_lists_launch<false>(a, s);
  scan_apply_kernel<T, V, L><<<blocks, kBlock, 0, s>>>(a);
}

template <typename T, int V, int L>
void scan_backward_launch(const ScanArgs& a, hipStream_t s) {
  const unsigned blocks = blocks_for(a.threads);
  scan_run_back_kernel<T, V, L><<<blocks, kBlock, 0, s>>>(a);
  scan_lists_launch<true>(a, s);
  scan_apply_back_kernel<T, V, L><<<blocks, kBlock, 0, s>>>(a);
}

template <typename F> void by_width(int v, F f) {
  if (v == 4) f(std::integral_constant<int, 4>());
  else if (v == 2) f(std::integral_constant<int, 2>());
  else f(std::integral_constant<int, 1>());
}

template <typename F> void by_chunk(int shift, F f) {
  if (shift == 6) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 16>());
}

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" {

int ocnn_octree_offsets(int* offsets, const void* octree_dev, const void* info, int depth, int nempty,
    ocnn_stream_t stream) {
  OCNN_REQUIRE(offsets && octree_dev && info, OCNN_E_BADARG, "null pointer");
  int rc = ocnn_info_check(info);
  if (rc) return rc;
  const Info* in = as_info(info);
  OCNN_REQUIRE(depth >= 1 && depth <= in->depth, OCNN_E_BADARG, "depth %d outside 1 .. %d", depth, in->depth);
  OCNN_REQUIRE(in->has(OCNN_KEY) && in->channel(OCNN_KEY) == 1 && in->location(OCNN_KEY) == -1, OCNN_E_UNSUPPORTED,
      "the octree holds no 64-bit key per node");
  OCNN_REQUIRE(!nempty || in->has(OCNN_CHILD), OCNN_E_FORMAT, "the octree holds no children");
  const char* blob = (const char*)octree_dev;
  octree_offsets_kernel<<<in->batch_size + 1, 64, 0, as_stream(stream)>>>(offsets,
      (const uint64_t*)(blob + in->ptr_dis(OCNN_KEY, depth)),
      nempty ? (const int*)(blob + in->ptr_dis(OCNN_CHILD, depth)) : nullptr, in->nnum[depth], in->nnum_nempty[depth],
      in->batch_size, nempty != 0);
  OCNN_LAUNCH_OK("octree_offsets");
  return OCNN_OK;
}

int ocnn_octree_rotary(void* out, int64_t out_row, int64_t out_head, const void* data, int64_t row, int64_t head,
    int rows, int heads, int dim, const void* positions, int position_kind, int64_t position_row,
    const double* frequencies, const int* pairs, int axes, int interleaved, int inverse, int dtype,
    ocnn_stream_t stream) {
  OCNN_REQUIRE(rows >= 0 && heads > 0 && dim > 0, OCNN_E_BADARG, "rows %d, heads %d, dim %d", rows, heads, dim);
  OCNN_REQUIRE(dtype == OCNN_F32 || dtype == OCNN_BF16, OCNN_E_BADARG, "dtype %d", dtype);
  OCNN_REQUIRE(position_kind >= OCNN_POS_INT32 && position_kind <= OCNN_POS_XYZ, OCNN_E_BADARG, "position kind %d",
      position_kind);
  OCNN_REQUIRE(pairs && axes >= 1 && axes <= 4 && (position_kind != OCNN_POS_XYZ || axes <= 3), OCNN_E_BADARG,
      "%d axes: at most 4 (3 with packed coordinates)", axes);
  int64_t total = 0;
  int ends[4] = {0, 0, 0, 0};
  for (int i = 0; i < 4; ++i) {
    if (i < axes) {
      OCNN_REQUIRE(pairs[i] >= 0, OCNN_E_BADARG, "axis %d: %d pairs", i, pairs[i]);
      total += pairs[i];
    }
    ends[i] = i < axes ? (int)(total > 2048 ? 2048 : total) : 1 << 30;
  }
  for (int i = axes - 1; i < 4; ++i) ends[i] = 1 << 30;       // the last axis is open
  OCNN_REQUIRE(2 * total <= dim, OCNN_E_SHAPE, "%lld pairs need %lld channels, a head has %d", (long long)total,
      (long long)(2 * total), dim);
  OCNN_REQUIRE(dim <= 1024 && heads <= 1024, OCNN_E_UNSUPPORTED, "%d heads of %d channels: at most 1024 of 1024", heads, dim);
  if (rows == 0) return OCNN_OK;
  OCNN_REQUIRE(out && data && (total == 0 || (positions && frequencies)), OCNN_E_BADARG, "null pointer");
  const int size = dtype == OCNN_F32 ? 4 : 2, V = 16 / size;
  RotaryArgs a = {};
  a.out = out; a.data = data; a.out_row = out_row; a.out_head = out_head; a.row = row; a.head = head;
  a.pos = positions; a.pos_row = position_row; a.freq = frequencies;
  a.rows = rows; a.heads = heads; a.dim = dim; a.pairs = (int)total;
  for (int i = 0; i < 3; ++i) a.axis_end[i] = ends[i];
  a.in_place = out == data && out_row == row && out_head == head;
  a.pair_items = interleaved ? 0 : (a.pairs + V - 1) / V;
  if (interleaved) a.items_head = ((a.in_place ? 2 * a.pairs : dim) + V - 1) / V;
  else a.items_head = a.pair_items + (a.in_place ? 0 : (dim - 2 * a.pairs + V - 1) / V);
  if (a.items_head == 0) return OCNN_OK;
  const int items = heads * a.items_head;
  // rows of a workgroup: about 1024 items of 32 bytes (60001 rows of 12 x 48 channels bf16), fewer where that
  // would leave compute units without work
  int r = 1024 / items;
  r = r < 1 ? 1 : r > 16 ? 16 : r;
  while (r > 1 && rows / r < 2048) r >>= 1;
  if (a.pairs && r > kRotaryAngles / a.pairs) r = kRotaryAngles / a.pairs;
  a.block_rows = r;
  a.div_pairs = reciprocal(a.pairs); a.div_row = r == 1 ? 1u : reciprocal(items);   // (1: every item is of row 0)
  a.div_head = reciprocal(a.items_head);
  a.inverse = inverse != 0;
  const unsigned blocks = blocks_for(rows, r);
  hipStream_t s = as_stream(stream);
  auto launch = [&](auto type, auto kind) {
    if (interleaved) rotary_kernel<decltype(type), kind.value, true><<<blocks, kBlock, 0, s>>>(a);
    else rotary_kernel<decltype(type), kind.value, false><<<blocks, kBlock, 0, s>>>(a);
  };
  auto by_kind = [&](auto type) {
    if (position_kind == OCNN_POS_INT32) launch(type, std::integral_constant<int, OCNN_POS_INT32>());
    else if (position_kind == OCNN_POS_F32) launch(type, std::integral_constant<int, OCNN_POS_F32>());
    else launch(type, std::integral_constant<int, OCNN_POS_XYZ>());
  };
  if (dtype == OCNN_F32) by_kind(float()); else by_kind(uint16_t());
  OCNN_LAUNCH_OK("octree_rotary");
  return OCNN_OK;
}

int ocnn_recurrence_shape(int rows, int channels, int n_seq, int carries, int64_t* carry_rows, size_t* workspace_bytes,
    size_t* grad_workspace_bytes) {
  OCNN_REQUIRE(rows >= 0 && channels > 0 && n_seq >= 1 && n_seq <= 65535, OCNN_E_BADARG, "rows %d, channels %d, sequences %d",
      rows, channels, n_seq);
  const int64_t ids = scan_ids(rows, n_seq, scan_shift(rows, channels));
  const size_t lists = 2 * (size_t)(ids + ((ids + kGroup - 1) >> kGroupShift)) * channels * sizeof(float);
  OCNN_REQUIRE(ids < (1ll << 31) && (channels + 63) / 64 <= 65535, OCNN_E_UNSUPPORTED, "%d rows of %d channels", rows, channels);
  if (carry_rows) *carry_rows = ids;
  if (workspace_bytes) *workspace_bytes = scan_walks(rows, n_seq, carries) || scan_blocks(rows, channels, n_seq, false) ? 0 : lists;
  if (grad_workspace_bytes) *grad_workspace_bytes = scan_blocks(rows, channels, n_seq, true) ? 0 : lists;
  return OCNN_OK;
}

int ocnn_octree_recurrence(void* out, int64_t out_row, float* last, float* carries, const void* gate, int64_t gate_row,
    const void* data, int64_t data_row, const float* state, const int* offsets, int n_seq, int rows, int channels,
    int reverse, int fill_rest, int dtype, void* workspace_dev, size_t workspace_bytes, ocnn_stream_t stream) {
  size_t need = 0;
  int rc = ocnn_recurrence_shape(rows, channels, n_seq, carries != nullptr, nullptr, &need, nullptr);
  if (rc) return rc;
  OCNN_REQUIRE(dtype == OCNN_F32 || dtype == OCNN_BF16, OCNN_E_BADARG, "dtype %d", dtype);
  OCNN_REQUIRE(offsets && (rows == 0 || (out && gate && data)), OCNN_E_BADARG, "null pointer");
  OCNN_REQUIRE(states_apart(last, state, n_seq, channels, need == 0), OCNN_E_BADARG, "last overlaps state");
  ScanArgs a = {};
  a.out = out; a.gate = gate; a.data = data; a.out_row = out_row; a.gate_row = gate_row; a.data_row = data_row;
  a.state = state; a.last = last; a.offsets = offsets;
  a.n_seq = n_seq; a.rows = rows; a.channels = channels; a.reverse = reverse != 0; a.fill = fill_rest != 0;
  hipStream_t s = as_stream(stream);
  const int size = dtype == OCNN_F32 ? 4 : 2;
  const bool walk = scan_walks(rows, n_seq, carries != nullptr);
  const int shift = scan_shift(rows, channels);
  const int64_t ids = walk ? (int64_t)n_seq + 1 : scan_ids(rows, n_seq, shift);
  const int v = scan_width(a, size, {{out, out_row}, {gate, gate_row}, {data, data_row}}, ids);
  a.groups = (channels + v - 1) / v;
  a.threads = ids * a.groups;
  if (walk) {
    // (a grid has fewer than 2^24 workgroups; where there are more items, these take several)
    const int64_t items = rows > kWalkRows ? (int64_t)blocks_for(rows, kWalkRows * kWalkSlots) * blocks_for(channels, kWalkChannels) : 0;
    const unsigned seekers = (unsigned)std::min<int64_t>(items, 16384), blocks = seekers + blocks_for(a.threads);
    by_width(v, [&](auto w) {
      if (dtype == OCNN_F32) scan_walk_kernel<float, w.value><<<blocks, kBlock, 0, s>>>(a, seekers);
      else scan_walk_kernel<uint16_t, w.value><<<blocks, kBlock, 0, s>>>(a, seekers);
    });
    OCNN_LAUNCH_OK("octree_recurrence");
    return OCNN_OK;
  }
  a.carry = carries;
  if (scan_blocks(rows, channels, n_seq, false)) {
    auto launch = [&](auto type) {
      using T = decltype(type);
      if (scan_narrow(channels, n_seq)) scan_block_kernel<T, 4, 64><<<block_items(n_seq + 1, (channels + 3) / 4), 256, 0, s>>>(a);
      else scan_block_kernel<T, 8, 64><<<block_items(n_seq + 1, (channels + 7) / 8), 512, 0, s>>>(a);
    };
    if (dtype == OCNN_F32) launch(float()); else launch(uint16_t());
    OCNN_LAUNCH_OK("octree_recurrence");
    return OCNN_OK;
  }
  OCNN_REQUIRE(workspace_dev && workspace_bytes >= need, OCNN_E_WORKSPACE, "octree_recurrence needs %zu bytes, got %zu", need,
      workspace_bytes);
  // (bf16, 256 channels, past the caches and not: 262147 rows 123.5 / 134 us, 131072 rows 67.6 / 67.4; an operator that reads
  // the result next then loses 2 to 3 us up to 65536 rows and nothing from 200000 on)
  a.past = (int64_t)rows * channels * size >= (96ll << 20);
  scan_lists(&a, ids, workspace_dev);
  by_width(v, [&](auto w) {
    by_chunk(shift, [&](auto l) {
      if (dtype == OCNN_F32) scan_forward_launch<float, w.value, l.value>(a, s);
      else scan_forward_launch<uint16_t, w.value, l.value>(a, s);
    });
  });
  OCNN_LAUNCH_OK("octree_recurrence");
  return OCNN_OK;
}

int ocnn_octree_recurrence_grad(void* grad_gate, int64_t grad_gate_row, void* grad_data, int64_t grad_data_row,
    float* grad_state, const void* grad_out, int64_t grad_out_row, const float* grad_last, const void* gate,
    int64_t gate_row, const void* data, int64_t data_row, const float* state, const float* carries, const int* offsets,
    int n_seq, int rows, int channels, int reverse, int dtype, void* workspace_dev, size_t workspace_bytes,
    ocnn_stream_t stream) {
  size_t need = 0;
  int rc = ocnn_recurrence_shape(rows, channels, n_seq, 1, nullptr, nullptr, &need);
  if (rc) return rc;
  OCNN_REQUIRE(dtype == OCNN_F32 || dtype == OCNN_BF16, OCNN_E_BADARG, "dtype %d", dtype);
  OCNN_REQUIRE(offsets && carries && (rows == 0 || (grad_gate && grad_data && grad_out && gate && data)), OCNN_E_BADARG,
      "null pointer");
  OCNN_REQUIRE(states_apart(grad_state, grad_last, n_seq, channels, need == 0) && states_apart(grad_state, state, n_seq, channels, false),
      OCNN_E_BADARG, "grad_state overlaps a state");
  ScanArgs a = {};
  a.gate = gate; a.data = data; a.grad = grad_out; a.grad_gate = grad_gate; a.grad_data = grad_data;
  a.gate_row = gate_row; a.data_row = data_row; a.grad_row = grad_out_row; a.grad_gate_row = grad_gate_row;
  a.grad_data_row = grad_data_row;
  a.state = state; a.grad_last = grad_last; a.grad_state = grad_state; a.offsets = offsets;
  a.n_seq = n_seq; a.rows = rows; a.channels = channels; a.reverse = reverse != 0;
  a.carry = const_cast<float*>(carries);
  hipStream_t s = as_stream(stream);
  if (scan_blocks(rows, channels, n_seq, true)) {
    auto launch = [&](auto type) {
      using T = decltype(type);
      if (scan_narrow(channels, n_seq)) scan_block_back_kernel<T, 4, 64><<<block_items(n_seq + 1, (channels + 3) / 4), 256, 0, s>>>(a);
      else scan_block_back_kernel<T, 8, 64><<<block_items(n_seq + 1, (channels + 7) / 8), 512, 0, s>>>(a);
    };
    if (dtype == OCNN_F32) launch(float()); else launch(uint16_t());
    OCNN_LAUNCH_OK("octree_recurrence_grad");
    return OCNN_OK;
  }
  OCNN_REQUIRE(workspace_dev && workspace_bytes >= need, OCNN_E_WORKSPACE, "octree_recurrence_grad needs %zu bytes, got %zu",
      need, workspace_bytes);
  const int size = dtype == OCNN_F32 ? 4 : 2, shift = scan_shift(rows, channels);
  const int64_t ids = scan_ids(rows, n_seq, shift);
  int v = scan_width(a, size, {{grad_gate, grad_gate_row}, {grad_data, grad_data_row}, {grad_out, grad_out_row},
                               {gate, gate_row}, {data, data_row}}, ids);
  v = v > 2 ? 2 : v;                 // (a group of rows is held in registers: p, q, before and the three loads)
  a.groups = (channels + v - 1) / v;
  a.threads = ids * a.groups;
  scan_lists(&a, ids, workspace_dev);
  by_width(v, [&](auto w) {
    if constexpr (w.value <= 2)
      by_chunk(shift, [&](auto l) {
        if (dtype == OCNN_F32) scan_backward_launch<float, w.value, l.value>(a, s);
        else scan_backward_launch<uint16_t, w.value, l.value>(a, s);
      });
  });
  OCNN_LAUNCH_OK("octree_recurrence_grad");
  return OCNN_OK;
}

}  // extern "C"
