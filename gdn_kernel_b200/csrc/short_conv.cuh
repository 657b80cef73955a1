// Short causal convolution over the channels of a mixer's input, W = 2..4 taps:
//   y_t[d] = act(bias[d] + sum_k w[d][k] u_{t-(W-1)+k}[d])
// u being a sequence's W-1 carried rows (zero for a new one) followed by its
// tokens.  The new carried state is the last W-1 rows of u.
//
// Both forms move each element once and do 2 W + 5 operations on it, so memory
// bounds them.  A thread owns one 16-byte vector of channels (one channel where
// sizes or addresses are not 16-byte multiples); its taps stay in fp32
// registers and sums are fp32, rounded once at the end.
#pragma once

#include "mixer_common.cuh"

namespace gdn {

constexpr int kConvThreads = 128;
constexpr int kConvBatch = 4;    // rows loaded while the four before them are worked on

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
  int tile;                    // tokens of a warp (prompts)
  unsigned int chan_warps;     // warps over the channels; all warps are those times tiles or rows
  unsigned int warps;
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
      const float2 f = unpair(s);
      y[2 * i] = silu ? silu_f(f.x) : f.x;
      if constexpr (V > 1) y[2 * i + 1] = silu ? silu_f(f.y) : f.y;
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) u[k][i] = u[k + 1][i];
      u[W - 2][i] = cur[i];
    }
    Pack<T, V> out;
    out.pack(y);
    return out;
  }
};

// Prompts: a warp takes p.tile consecutive packed tokens of 32 V channels and
// walks the sequences that touch them.  The thread that holds a
// sequence's first token also writes its new state, after it has read the old
// one, so that the two may be the same memory.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_kernel(const ConvParams p) {
  const unsigned int id = blockIdx.x * (kConvThreads / 32) + threadIdx.x / 32;
  if (id >= p.warps) return;
  const int d = static_cast<int>(id % p.chan_warps * 32 + threadIdx.x % 32) * V;
  const long long t0 = static_cast<long long>(id / p.chan_warps) * p.tile;
  const long long t1 = min(t0 + p.tile, p.tokens);
  const bool last_tile = t1 == p.tokens;
  int i = count_below(p.cu, p.cu_is64, p.seqs, t0);
  if (id == 0) check_offsets(p.cu, p.cu_is64, p.seqs, p.tokens, p.status);
  if (d >= p.channels) return;
  const bool reporter = d == 0;
  const T* x = static_cast<const T*>(p.x) + d;
  T* out = static_cast<T*>(p.out) + d;
  ConvTaps<T, V, W> taps;
  taps.load(p, d);

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
          Pack<T, V> v;
          v.zero();
          if (pos >= 0) v.load(x + (s + pos) * p.x_stride);
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
            if (pos < 0 && j == W - 1 + pos) v = old[j];
          v.store(ns + static_cast<long long>(k) * p.channels);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        Pack<T, V> v;
        v.load(x + (a - (W - 1) + k) * p.x_stride);
        win.set(k, v);
      }
    }

    const T* src = x + a * p.x_stride;
    T* dst = out + a * p.out_stride;
    int left = static_cast<int>(z - a);
    Pack<T, V> next[kConvBatch];
#pragma unroll
    for (int j = 0; j < kConvBatch; ++j)
      if (j < left) next[j].load_stream(src + j * p.x_stride);
    for (; left > 0; left -= kConvBatch) {
      Pack<T, V> in[kConvBatch];
      src += kConvBatch * p.x_stride;
#pragma unroll
      for (int j = 0; j < kConvBatch; ++j) {
        in[j] = next[j];
        if (j + kConvBatch < left) next[j].load_stream(src + j * p.x_stride);
      }
#pragma unroll
      for (int j = 0; j < kConvBatch; ++j)
        if (j < left) win.row(taps, in[j], p.silu).store(dst + j * p.out_stride);
      dst += kConvBatch * p.out_stride;
    }
  }
}

// Single tokens: one row per batch entry, its window in the pool.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_step_kernel(const ConvParams p) {
  const unsigned int id = blockIdx.x * (kConvThreads / 32) + threadIdx.x / 32;
  if (id >= p.warps) return;
  const int d = static_cast<int>(id % p.chan_warps * 32 + threadIdx.x % 32) * V;
  if (d >= p.channels) return;
  const long long b = id / p.chan_warps;
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
