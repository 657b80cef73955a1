// Short causal convolution over the channels of a mixer's input, W = 2..4 taps:
//   y_t[d] = act(bias[d] + sum_k w[d][k] u_{t-(W-1)+k}[d])
// u being a sequence's W-1 carried rows (zero for a new one) followed by its
// tokens.  The new carried state is the last W-1 rows of u.
//
// Both forms move each element once and do 2 W + 5 operations on it, so memory
// bounds them.  A thread owns four channels (one where sizes or addresses do not
// allow 16-byte copies); its taps stay in fp32 registers and sums are fp32,
// rounded once at the end.
#pragma once

#include "gdn_ptx.cuh"
#include "mixer_common.cuh"

namespace gdn {

constexpr int kConvThreads = 128;
constexpr int kConvVec = 4;      // channels of a thread

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

// Prompts: a block takes p.tile consecutive packed tokens of kConvThreads V
// channels and walks the sequences that touch them.  The thread that holds a
// sequence's first token also writes its new state, after it has read the old
// one, so that the two may be the same memory.
//
// V = kConvVec: all the block's rows (and the W - 1 before them) come to shared
// memory as bulk copies that start before the sequences are looked up.  With the
// rows in registers instead, four loaded ahead, the copies in flight were too few
// (8192 tokens of 8192 channels: 63 us).  V = 1: plain loads.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_kernel(const ConvParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr bool kStaged = V == kConvVec;
  constexpr int kRow = kConvThreads * V;          // elements of a staged row
  const int c0 = static_cast<int>(blockIdx.x % p.chan_blocks) * kRow;
  const int d = c0 + static_cast<int>(threadIdx.x) * V;
  const long long t0 = static_cast<long long>(blockIdx.x / p.chan_blocks) * p.tile;
  const long long t1 = min(t0 + p.tile, p.tokens);
  const bool last_tile = t1 == p.tokens;
  const long long r0 = max(t0 - (W - 1), 0LL);    // rows staged: [r0, r1)
  const long long r1 = min(t1 + W - 2, p.tokens);
  const T* rows = reinterpret_cast<const T*>(smem + 128) + threadIdx.x * V;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem);
  if constexpr (kStaged) {
    if (threadIdx.x == 0) {
      mbar_init(bar, 1);
      fence_mbarrier_init();
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int n = static_cast<int>(r1 - r0);
      const uint32_t bytes = static_cast<uint32_t>(min(kRow, p.channels - c0) * sizeof(T));
      if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, n * bytes);
      __syncwarp();
      for (int i = threadIdx.x; i < n; i += 32)
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
            ::"r"(smem_u32(smem + 128 + static_cast<size_t>(i) * kRow * sizeof(T))),
            "l"(static_cast<const T*>(p.x) + (r0 + i) * p.x_stride + c0), "r"(bytes),
            "r"(smem_u32(bar))
            : "memory");
    }
  }
  int i = count_below(p.cu, p.cu_is64, p.seqs, t0);
  if (blockIdx.x == 0 && threadIdx.x < 32) check_offsets(p.cu, p.cu_is64, p.seqs, p.tokens, p.status);
  const bool live = d < p.channels;
  const bool reporter = d == 0;
  const T* x = static_cast<const T*>(p.x) + d;
  T* out = static_cast<T*>(p.out) + d;
  ConvTaps<T, V, W> taps;
  if (live) taps.load(p, d);
  if constexpr (kStaged) {
    // (a second wait in case the first ran out: no copy may outlive the block)
    if (!mbar_wait(bar, 0)) {
      if (threadIdx.x == 0) atomicOr(p.status, kStatusTmaTimeout);
      mbar_wait(bar, 0);
      return;
    }
  }
  if (!live) return;
  auto row_at = [&](long long t) {
    Pack<T, V> v;
    if constexpr (kStaged) v.load(rows + static_cast<int>(t - r0) * kRow);
    else v.load(x + t * p.x_stride);
    return v;
  };

  // the sequence that is running at t0, then those that start in this tile
  for (i = max(i - 1, 0); i < p.seqs; ++i) {
    const long long s = index_at(p.cu, p.cu_is64, i);
    const long long e = index_at(p.cu, p.cu_is64, i + 1);
    if (s >= t1 && !(last_tile && s == p.tokens)) break;
    if (s < 0 || e < s || e > p.tokens) {
      if (reporter) atomicOr(p.status, kMixerBadSeqlens);
      continue;
    }
    // A sequence's first W - 1 tokens, which read the old state, belong to the
    // tile of its start even where they reach past it.
    const bool starts = s >= t0;
    const long long a = starts ? s : max(t0, s + W - 1);   // the tokens done here: [a, z)
    const long long z = starts ? min(e, max(t1, s + W - 1)) : min(e, t1);
    if (!starts && a >= z) continue;

    ConvWindow<T, V, W> win;
    if (starts) {
      const long long slot = slot_of(p.slots, p.slots_is64, i, p.pool, p.status, reporter);
      const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[i]);
      Pack<T, V> old[W - 1];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        old[k].zero();
        if (carried)
          old[k].load(static_cast<const T*>(p.state) + (slot * (W - 1) + k) * p.channels + d);
        win.set(k, old[k]);
      }
      if (slot >= 0) {
        const long long len = e - s;
        T* ns = static_cast<T*>(p.new_state) + slot * (W - 1) * p.channels + d;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
          const long long pos = len - (W - 1) + k;   // row k holds this position of the tokens
          T* to = ns + static_cast<long long>(k) * p.channels;
          if (pos >= 0) {
            Pack<T, V> v;
            v.load(x + (s + pos) * p.x_stride);
            v.store(to);
          }
#pragma unroll
          for (int j = k; j < W - 1; ++j)   // an old row, in a sequence shorter than the window
            if (pos + W - 1 == j) old[j].store(to);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < W - 1; ++k) win.set(k, row_at(a - (W - 1) + k));
    }
    T* dst = out + a * p.out_stride;
#pragma unroll 8
    for (long long t = a; t < z; ++t) {
      win.row(taps, row_at(t), p.silu).store(dst);
      dst += p.out_stride;
    }
  }
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
