// Short causal convolution over the channels of a mixer's input, W = 2..4 taps:
//   y_t[d] = act(bias[d] + sum_k w[d][k] u_{t-(W-1)+k}[d])
// u being a sequence's W-1 carried rows (zero for a new one) followed by its
// tokens.  The new carried state is the last W-1 rows of u.
//
// Both forms move each element once and do 2 W + 5 operations on it, so memory
// bounds them.  A thread owns four channels (one where sizes or addresses do not
// allow 16-byte copies); its taps stay in fp32 registers and sums are fp32,
// rounded once at the end.  8192 tokens of 8192 channels: 49 us, 5.5 TB/s; of 8191, one
// channel a thread, 179 us.
#pragma once

#include "gdn_ptx.cuh"
#include "mixer_common.cuh"

namespace gdn {

constexpr int kConvThreads = 128;
constexpr int kConvVec = 4;      // channels of a thread
constexpr int kConvShort = 16;   // tokens up to which a sequence has blocks of its own

struct ConvParams {
  const void* x;               // [T, D], rows x_stride apart
  const void* weight;          // [D, W]
  const void* bias;            // [D] or nullptr
  const void* state;           // [P, W - 1, D] or nullptr (zero)
  void* new_state;             // [P, W - 1, D], may be state
  void* out;                   // [T, D], rows out_stride apart
  const void* cu;              // [N + 1]
  const void* slots;           // [N] or nullptr (slot = sequence)
  const uint8_t* has_state;    // [N] or nullptr (all)
  unsigned int* status;
  long long x_stride, out_stride, pool, tokens;
  int cu_is64, slots_is64, seqs, channels, silu;
  int tile;                    // prompts: tokens of a block
  unsigned int chan_blocks;    // blocks over the channels; the grid is those times tiles or rows
  unsigned int tile_blocks;    // prompts: blocks of tiles; those of short sequences follow
  int lookup_first;            // prompts: look for a tile's sequences before its rows are loaded
};

// The taps of V channels, two channels to a pair where V allows it.
template <typename T, int V, int W>
struct ConvTaps {
  static constexpr int kPairs = V / 2;
  uint64_t w[W][kPairs > 0 ? kPairs : 1], b[kPairs > 0 ? kPairs : 1];
  __device__ __forceinline__ void load(const ConvParams& p, int d) {
    const T* src = static_cast<const T*>(p.weight) + static_cast<long long>(d) * W;
    float f[V * W], c[V];
    // V channels' taps are V W consecutive elements
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Pack<T, V> v;
      v.load(src + i * V);
      float g[V];
      v.unpack(g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[i * V + e] = g[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = 0.0f;
    if (p.bias) {
      Pack<T, V> v;
      v.load(static_cast<const T*>(p.bias) + d);
      v.unpack(c);
    }
    // one channel: the pair's other half idles
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const int o = V > 1 ? e + 1 : e;
      b[e / 2] = pair(c[e], c[o]);
#pragma unroll
      for (int k = 0; k < W; ++k) w[k][e / 2] = pair(f[e * W + k], f[o * W + k]);
    }
  }
};

template <typename T, int V, int W>
struct ConvWindow {
  static constexpr int kPairs = V > 1 ? V / 2 : 1;
  uint64_t u[W - 1][kPairs];
  static __device__ __forceinline__ void unpack(const Pack<T, V>& v, uint64_t (&out)[kPairs]) {
    float f[V];
    v.unpack(f);
#pragma unroll
    for (int e = 0; e < V; e += 2) out[e / 2] = pair(f[e], f[V > 1 ? e + 1 : e]);
  }
  __device__ __forceinline__ void set(int k, const Pack<T, V>& v) { unpack(v, u[k]); }
  // One output row from the W - 1 rows before it and the row itself; the window
  // moves on by one.
  __device__ __forceinline__ Pack<T, V> row(const ConvTaps<T, V, W>& taps, const Pack<T, V>& in,
                                            int silu) {
    uint64_t cur[kPairs];
    unpack(in, cur);
    float y[V];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      uint64_t s = taps.b[i];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) s = fma2(taps.w[k][i], u[k][i], s);
      s = fma2(taps.w[W - 1][i], cur[i], s);
      const float2 f = unpair(silu ? silu2(s) : s);
      y[2 * i] = f.x;
      if constexpr (V > 1) y[2 * i + 1] = f.y;
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) u[k][i] = u[k + 1][i];
      u[W - 2][i] = cur[i];
    }
    Pack<T, V> out;
    out.pack(y);
    return out;
  }
};

// A whole sequence of a few tokens by each thread: old rows, tokens, new rows.
template <typename T, int V, int W>
__device__ __forceinline__ void short_sequence(const ConvParams& p, int seq, int d) {
  const long long s = index_at(p.cu, p.cu_is64, seq);
  const long long e = index_at(p.cu, p.cu_is64, seq + 1);
  if (s < 0 || e < s || e > p.tokens || e - s > kConvShort) return;   // tiles do and report those
  const long long slot = slot_of(p.slots, p.slots_is64, seq, p.pool, p.status, d == 0);
  const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[seq]);
  if (d >= p.channels) return;
  const int len = static_cast<int>(e - s);
  const T* x = static_cast<const T*>(p.x) + s * p.x_stride + d;
  T* out = static_cast<T*>(p.out) + s * p.out_stride + d;
  Pack<T, V> hist[W - 1];     // the last W - 1 rows so far
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    hist[k].zero();
    if (carried)
      hist[k].load(static_cast<const T*>(p.state) + (slot * (W - 1) + k) * p.channels + d);
  }
  Pack<T, V> next;
  if (len > 0) next.load_stream(x);
  ConvTaps<T, V, W> taps;
  taps.load(p, d);
  ConvWindow<T, V, W> win;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win.set(k, hist[k]);
  for (int t = 0; t < len; ++t) {
    const Pack<T, V> in = next;
    if (t + 1 < len) next.load_stream(x + (t + 1) * p.x_stride);
    win.row(taps, in, p.silu).store(out + t * p.out_stride);
#pragma unroll
    for (int k = 0; k + 1 < W - 1; ++k) hist[k] = hist[k + 1];
    hist[W - 2] = in;
  }
  if (slot < 0) return;
  T* ns = static_cast<T*>(p.new_state) + slot * (W - 1) * p.channels + d;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) hist[k].store(ns + static_cast<long long>(k) * p.channels);
}

// Prompts: a block takes p.tile consecutive packed tokens of kConvThreads V
// channels and walks the sequences of more than kConvShort tokens that touch them.
// The thread that holds a sequence's first token also writes its new state, after
// it has read the old one, so that the two may be the same memory.  Shorter
// sequences have blocks of their own: a tile would work through many of them one
// after the other (64 of one token, 8192 channels: 21 us).
//
// V = kConvVec: all the block's rows (and the W - 1 before them) come to shared
// memory as bulk copies that start before the sequences are looked up.  With the
// rows in registers instead, four loaded ahead, the copies in flight were too few
// (8192 tokens of 8192 channels: 63 us).  V = 1: plain loads.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_kernel(const ConvParams p) {
  extern __shared__ __align__(128) uint8_t conv_smem[];
  constexpr bool kStaged = V == kConvVec;
  constexpr int kRow = kConvThreads * V;          // elements of a staged row
  const int c0 = static_cast<int>(blockIdx.x % p.chan_blocks) * kRow;
  const int d = c0 + static_cast<int>(threadIdx.x) * V;
  if (blockIdx.x >= p.tile_blocks) {
    short_sequence<T, V, W>(p, static_cast<int>((blockIdx.x - p.tile_blocks) / p.chan_blocks), d);
    return;
  }
  // (tokens are below 2^30, so that tile ends are ints too)
  const int tokens = static_cast<int>(p.tokens);
  const int t0 = static_cast<int>(blockIdx.x / p.chan_blocks) * p.tile;
  const int t1 = min(t0 + p.tile, tokens);
  const int r0 = max(t0 - (W - 1), 0);            // rows staged: [r0, r1)
  const int r1 = min(t1 + W - 2, tokens);
  const T* rows = reinterpret_cast<const T*>(conv_smem + 128) + threadIdx.x * V;
  uint64_t* bar = reinterpret_cast<uint64_t*>(conv_smem);
  // The sequences of the tile that are done here, 32 looked at together, a lane
  // each: work(sequence, its bounds) by whole warps.
  const int lane = threadIdx.x & 31;
  int first = 0;
  auto find_first = [&] { first = max(count_below(p.cu, p.cu_is64, p.seqs, t0) - 1, 0); };
  auto for_each = [&](auto work) {
    for (int base = first; base < p.seqs; base += 32) {
      int s = 0, e = 0;
      bool past = true;
      if (base + lane < p.seqs) {
        const long long from = index_at(p.cu, p.cu_is64, base + lane);
        const long long to = index_at(p.cu, p.cu_is64, base + lane + 1);
        past = from >= t1;
        if (from >= 0 && to <= tokens && to - from > kConvShort) {
          s = static_cast<int>(from);
          e = static_cast<int>(to);
        }
      }
      unsigned int todo = __ballot_sync(0xffffffffu, !past && e > t0);
      while (todo) {
        const int k = __ffs(todo) - 1;
        todo &= todo - 1;
        work(base + k, __shfl_sync(0xffffffffu, s, k), __shfl_sync(0xffffffffu, e, k));
      }
      if (__any_sync(0xffffffffu, past)) return;
    }
  };
  if (blockIdx.x == 0 && threadIdx.x < 32) check_offsets(p.cu, p.cu_is64, p.seqs, p.tokens, p.status);
  if (p.lookup_first) {   // most sequences are short: nothing to load for many tiles
    bool any = false;
    find_first();
    for_each([&](int, int, int) { any = true; });
    if (!any) return;
  }
  if constexpr (kStaged) {
    if (threadIdx.x == 0) {
      mbar_init(bar, 1);
      fence_mbarrier_init();
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int n = r1 - r0;
      const uint32_t bytes = static_cast<uint32_t>(min(kRow, p.channels - c0) * sizeof(T));
      if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, n * bytes);
      __syncwarp();
      for (int i = threadIdx.x; i < n; i += 32)
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
            ::"r"(smem_u32(conv_smem + 128 + static_cast<size_t>(i) * kRow * sizeof(T))),
            "l"(static_cast<const T*>(p.x) + static_cast<long long>(r0 + i) * p.x_stride + c0), "r"(bytes),
            "r"(smem_u32(bar))
            : "memory");
    }
  }
  if (!p.lookup_first) find_first();   // while the rows are on their way
  const bool live = d < p.channels;
  const T* x = static_cast<const T*>(p.x) + d;
  T* out = static_cast<T*>(p.out) + d;
  ConvTaps<T, V, W> taps;
  if (live) taps.load(p, d);
  if constexpr (kStaged) {
    if (!__syncthreads_and(mbar_wait(bar, 0))) {
      if (threadIdx.x == 0) atomicOr(p.status, kStatusTmaTimeout);
      mbar_wait(bar, 0);   // no copy may outlive the block
      return;
    }
  }
  auto row_at = [&](int t) {
    Pack<T, V> v;
    if constexpr (kStaged) v.load(rows + (t - r0) * kRow);
    else v.load(x + t * p.x_stride);
    return v;
  };

  for_each([&](int i, int s, int e) {
    if (!live) return;
    // A sequence's first W - 1 tokens, which read the old state, belong to the
    // tile of its start even where they reach past it.
    const bool starts = s >= t0;
    const int a = starts ? s : max(t0, s + W - 1);   // the tokens done here: [a, z)
    const int z = starts ? min(e, max(t1, s + W - 1)) : min(e, t1);
    if (a >= z) return;

    ConvWindow<T, V, W> win;
    if (starts) {
      const long long slot = slot_of(p.slots, p.slots_is64, i, p.pool, p.status, d == 0);
      const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[i]);
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        Pack<T, V> old;
        old.zero();
        if (carried)
          old.load(static_cast<const T*>(p.state) + (slot * (W - 1) + k) * p.channels + d);
        win.set(k, old);
      }
      if (slot >= 0) {   // (longer than the window: the last rows are tokens)
        T* ns = static_cast<T*>(p.new_state) + slot * (W - 1) * p.channels + d;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
          Pack<T, V> v;
          v.load(x + static_cast<long long>(e - (W - 1) + k) * p.x_stride);
          v.store(ns + static_cast<long long>(k) * p.channels);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < W - 1; ++k) win.set(k, row_at(a - (W - 1) + k));
    }
    T* dst = out + a * p.out_stride;
#pragma unroll 8
    for (int t = a; t < z; ++t) {
      win.row(taps, row_at(t), p.silu).store(dst);
      dst += p.out_stride;
    }
  });
}

// Single tokens: one row per batch entry, its window in the pool.  64 rows of 8192
// channels take 3.0 us, of which the 8.5 MB account for 1.3.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_step_kernel(const ConvParams p) {
  const int d = static_cast<int>(blockIdx.x % p.chan_blocks * kConvThreads + threadIdx.x) * V;
  if (d >= p.channels) return;
  const long long b = blockIdx.x / p.chan_blocks;
  const long long slot = slot_of(p.slots, p.slots_is64, b, p.pool, p.status, d == 0);
  T* out = static_cast<T*>(p.out) + b * p.out_stride + d;
  if (slot < 0) {
    Pack<T, V> v;
    v.zero();
    v.store(out);
    return;
  }
  const long long at = slot * (W - 1) * p.channels + d;
  Pack<T, V> in, old[W - 1];
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
    old[k].load(static_cast<const T*>(p.state) + at + static_cast<long long>(k) * p.channels);
  in.load(static_cast<const T*>(p.x) + b * p.x_stride + d);
  ConvTaps<T, V, W> taps;
  taps.load(p, d);
  ConvWindow<T, V, W> win;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win.set(k, old[k]);
  win.row(taps, in, p.silu).store(out);
  T* ns = static_cast<T*>(p.new_state) + at;
#pragma unroll
  for (int k = 0; k + 1 < W - 1; ++k) old[k + 1].store(ns + static_cast<long long>(k) * p.channels);
  in.store(ns + static_cast<long long>(W - 2) * p.channels);
}

}  // namespace gdn
