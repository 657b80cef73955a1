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
constexpr int kConvTile = 32;    // tokens of a block
constexpr int kConvBatch = 8;    // rows whose loads are in flight together

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
  unsigned int chan_blocks;    // blocks over the channels; the grid is those times tiles or rows
};

template <typename T, int V, int W>
struct ConvTaps {
  float w[W][V], b[V];
  __device__ __forceinline__ void load(const ConvParams& p, int d) {
    const T* src = static_cast<const T*>(p.weight) + static_cast<long long>(d) * W;
    // V channels' taps are V W consecutive elements
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Pack<T, V> v;
      v.load(src + i * V);
      float f[V];
      v.unpack(f);
#pragma unroll
      for (int e = 0; e < V; ++e) w[(i * V + e) % W][(i * V + e) / W] = f[e];
    }
    if (p.bias) {
      Pack<T, V> v;
      v.load(static_cast<const T*>(p.bias) + d);
      v.unpack(b);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) b[e] = 0.0f;
    }
  }
};

// One output row from the W - 1 rows before it and the row itself; the window
// moves on by one.
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> conv_row(const ConvTaps<T, V, W>& taps,
                                               float (&win)[W - 1][V], const Pack<T, V>& in,
                                               int silu) {
  float cur[V], y[V];
  in.unpack(cur);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float s = taps.b[e];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) s = fmaf(taps.w[k][e], win[k][e], s);
    s = fmaf(taps.w[W - 1][e], cur[e], s);
    y[e] = silu ? silu_f(s) : s;
#pragma unroll
    for (int k = 0; k + 1 < W - 1; ++k) win[k][e] = win[k + 1][e];
    win[W - 2][e] = cur[e];
  }
  Pack<T, V> out;
  out.pack(y);
  return out;
}

// Prompts: a block takes kConvTile consecutive packed tokens of kConvThreads V
// channels and walks the sequences that touch them.  The thread that holds a
// sequence's first token also writes its new state, after it has read the old
// one, so that the two may be the same memory.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) gdn_short_conv_kernel(const ConvParams p) {
  const int d = static_cast<int>(blockIdx.x % p.chan_blocks * kConvThreads + threadIdx.x) * V;
  const long long t0 = static_cast<long long>(blockIdx.x / p.chan_blocks) * kConvTile;
  const long long t1 = min(t0 + kConvTile, p.tokens);
  const bool last_tile = t1 == p.tokens;
  int i = count_below(p.cu, p.cu_is64, p.seqs, t0);
  if (blockIdx.x == 0) check_offsets(p.cu, p.cu_is64, p.seqs, p.tokens, p.status);
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

    float win[W - 1][V];
    if (starts) {
      const long long slot = slot_of(p.slots, p.slots_is64, i, p.pool, p.status, reporter);
      const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[i]);
      Pack<T, V> old[W - 1];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        old[k].zero();
        if (carried)
          old[k].load(static_cast<const T*>(p.state) + (slot * (W - 1) + k) * p.channels + d);
        old[k].unpack(win[k]);
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
        v.unpack(win[k]);
      }
    }

    for (long long t = a; t < z; t += kConvBatch) {
      Pack<T, V> in[kConvBatch];
#pragma unroll
      for (int j = 0; j < kConvBatch; ++j)
        if (t + j < z) in[j].load(x + (t + j) * p.x_stride);
#pragma unroll
      for (int j = 0; j < kConvBatch; ++j)
        if (t + j < z)
          conv_row<T, V, W>(taps, win, in[j], p.silu).store(out + (t + j) * p.out_stride);
    }
  }
}

// Single tokens: one row per batch entry, its window in the pool.
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
  float win[W - 1][V];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) old[k].unpack(win[k]);
  conv_row<T, V, W>(taps, win, in, p.silu).store(out);
  T* ns = static_cast<T*>(p.new_state) + at;
#pragma unroll
  for (int k = 0; k + 1 < W - 1; ++k) old[k + 1].store(ns + static_cast<long long>(k) * p.channels);
  in.store(ns + static_cast<long long>(W - 2) * p.channels);
}

}  // namespace gdn
