// The norms around a block, each one pass over its rows.
//
// gated norm (after a mixer), by groups of a row:
//   y = rms(x) w act(g)          or          y = rms(x act(g)) w
// residual add and norm (between blocks):
//   r' = r + s u,  u = x or rms(x) w_b;      y = rms(r') (w + offset)
// with rms(v) = v / sqrt(mean(v^2) + eps) over the group.
//
// Memory bounds both (8192 rows of 32 groups of 128: 37 us, 5.5 TB/s; 8192 rows of
// 2048 with an fp32 residual and both norms: 34 us, 5.9 TB/s; a plain copy reaches
// 6.5): each element is read once, kept in registers between the
// sum of squares and the scaling, and written once.  Sums are fp32.  `kTeam`
// threads share a group (part of a warp, a warp, or with kTeam = 0 the block, as
// large as the group needs), each holding kVecs 16-byte vectors of every operand.
// Rows that no such shape fits (sizes or addresses off 16 bytes, more than 4096
// vectors) take one element per access and read their operands again, from L1 or L2,
// after the sum (gated norm of 8192 x 4095 94 us, of 1024 x 40960 131; residual add
// and norm of 8192 x 2047 52).
#pragma once

#include "mixer_common.cuh"

namespace gdn {

struct NormParams {
  const void* x;            // rows x_stride apart
  const void* gate;         // gated norm: rows gate_stride apart, or nullptr (no gate)
  const void* residual;     // add norm: rows residual_stride apart
  const void* weight;       // [group], [width] or nullptr
  const void* block_weight; // add norm: [width] or nullptr (no norm after the block)
  const float* channel_scale;   // add norm: [width] or nullptr
  void* out;
  void* new_residual;
  long long rows, x_stride, gate_stride, residual_stride, out_stride, new_residual_stride;
  int width, group, weight_shared;
  unsigned int per_row;     // groups of a row
  float inv_group, inv_width;
  int silu;                 // gate activation: silu, else sigmoid
  int norm_first;
  float eps, scale, weight_offset;
};

// Sum over the threads that share a group: kTeam of them, or the block (kTeam = 0).
template <int kTeam>
__device__ __forceinline__ float team_sum(float v, float* smem) {
  constexpr bool kBlock = kTeam == 0;
#pragma unroll
  for (int o = (kBlock ? 32 : kTeam) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (kBlock) {
    __syncthreads();   // an earlier sum's readers are done
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    // every warp adds the warps' sums, in the same order
    const int lane = threadIdx.x & 31;
    v = lane < static_cast<int>(blockDim.x >> 5) ? smem[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

__device__ __forceinline__ float gate_act(float g, int silu) { return silu ? silu_f(g) : sigmoid_f(g); }

// v[e] *= act(gate element e), two elements at a time.
template <typename T, int V>
__device__ __forceinline__ void apply_gate(float (&v)[V], const Pack<T, V>& gate, int silu) {
  float g[V];
  gate.unpack(g);
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const uint64_t gp = pair(g[e], g[e + 1]);
    const float2 y = unpair(mul2(pair(v[e], v[e + 1]), silu ? silu2(gp) : sigmoid2(gp)));
    v[e] = y.x;
    v[e + 1] = y.y;
  }
}

constexpr int kNormThreads = 128;   // of a block, where a team is a warp or less
constexpr int kNormBlock = 1024;    // largest block of one team

template <typename T, int V, int kTeam, int kVecs>
__global__ void __launch_bounds__(kTeam > 0 ? kNormThreads : kVecs == 1 ? 512 : kNormBlock)
gdn_gated_norm_kernel(const NormParams p) {
  __shared__ float smem[32];
  const int team = kTeam > 0 ? kTeam : static_cast<int>(blockDim.x);
  const int lane = kTeam > 0 ? threadIdx.x % (kTeam > 0 ? kTeam : 1) : threadIdx.x;
  // 32 bits: groups stay below 2^31, and a 64-bit division took 10 of 48 us at 8192
  // rows of 32 groups of 128
  const unsigned int id =
      kTeam > 0 ? blockIdx.x * (kNormThreads / (kTeam > 0 ? kTeam : 1)) + threadIdx.x / (kTeam > 0 ? kTeam : 1)
                : blockIdx.x;
  const bool live = id < static_cast<unsigned int>(p.rows * p.per_row);
  const unsigned int row = id / p.per_row;
  const int c0 = static_cast<int>(id - row * p.per_row) * p.group;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + c0;
  const T* gate = static_cast<const T*>(p.gate) + row * p.gate_stride + c0;
  const T* w = static_cast<const T*>(p.weight) + (p.weight_shared ? 0 : c0);
  T* out = static_cast<T*>(p.out) + row * p.out_stride + c0;

  Pack<T, V> xv[kVecs], gv[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = (lane + i * team) * V;
    xv[i].zero();
    gv[i].zero();
    if (live && c < p.group) {
      xv[i].load_stream(x + c);
      if (p.gate) gv[i].load_stream(gate + c);
    }
  }
  float xf[kVecs][V], ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    xv[i].unpack(xf[i]);
    if (p.gate && !p.norm_first) apply_gate<T, V>(xf[i], gv[i], p.silu);
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(xf[i][e], xf[i][e], ss);
  }
  const float inv = rsqrtf(team_sum<kTeam>(ss, smem) * p.inv_group + p.eps);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = (lane + i * team) * V;
    if (!live || c >= p.group) continue;
    float y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = xf[i][e] * inv;
    if (p.weight) {
      Pack<T, V> wv;
      float wf[V];
      wv.load(w + c);
      wv.unpack(wf);
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] *= wf[e];
    }
    if (p.gate && p.norm_first) apply_gate<T, V>(y, gv[i], p.silu);
    Pack<T, V> yv;
    yv.pack(y);
    yv.store(out + c);
  }
}

// Any group size and alignment: a block per group, one element per access.
template <typename T>
__global__ void __launch_bounds__(256) gdn_gated_norm_any_kernel(const NormParams p) {
  __shared__ float smem[32];
  const unsigned int per_row = p.per_row;
  const unsigned int row = blockIdx.x / per_row;
  const int c0 = static_cast<int>(blockIdx.x - row * per_row) * p.group;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + c0;
  const T* g = p.gate ? static_cast<const T*>(p.gate) + row * p.gate_stride + c0 : nullptr;
  const T* w = p.weight ? static_cast<const T*>(p.weight) + (p.weight_shared ? 0 : c0) : nullptr;
  T* out = static_cast<T*>(p.out) + row * p.out_stride + c0;
  float ss = 0.0f;
  for (int c = threadIdx.x; c < p.group; c += 256) {
    float v = to_float(x[c]);
    if (g && !p.norm_first) v *= gate_act(to_float(g[c]), p.silu);
    ss = fmaf(v, v, ss);
  }
  const float inv = rsqrtf(team_sum<0>(ss, smem) * p.inv_group + p.eps);
  for (int c = threadIdx.x; c < p.group; c += 256) {
    float v = to_float(x[c]);
    const float a = g ? gate_act(to_float(g[c]), p.silu) : 1.0f;
    v = p.norm_first ? v * inv : v * a * inv;
    if (w) v *= to_float(w[c]);
    if (p.norm_first) v *= a;
    out[c] = from_float<T>(v);
  }
}

// Residual elements R (the type of x or fp32) that go with V elements of x.
template <typename T, typename R, int V>
struct ResidualVec {
  static constexpr int kParts = static_cast<int>(sizeof(R) / sizeof(T));   // 1, or 2 for fp32 beside 16 bits
  static constexpr int kE = V / kParts == 0 ? 1 : V / kParts;
  static constexpr int kN = V == 1 ? 1 : kParts;
  Pack<R, kE> part[kN];
  __device__ __forceinline__ void load(const R* p) {
#pragma unroll
    for (int i = 0; i < kN; ++i) part[i].load_stream(p + i * kE);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kN; ++i) part[i].zero();
  }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float t[kE];
      part[i].unpack(t);
#pragma unroll
      for (int e = 0; e < kE; ++e) f[i * kE + e] = t[e];
    }
  }
  __device__ __forceinline__ void pack_store(const float (&f)[V], R* p) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float t[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) t[e] = f[i * kE + e];
      part[i].pack(t);
      part[i].store(p + i * kE);
    }
  }
};

template <typename T, typename R, int V, int kTeam, int kVecs>
__global__ void __launch_bounds__(kTeam > 0 ? kNormThreads : kVecs == 1 ? 512 : kNormBlock)
gdn_add_norm_kernel(const NormParams p) {
  __shared__ float smem[32];
  const int team = kTeam > 0 ? kTeam : static_cast<int>(blockDim.x);
  const int lane = kTeam > 0 ? threadIdx.x % (kTeam > 0 ? kTeam : 1) : threadIdx.x;
  const long long id = kTeam > 0 ? static_cast<long long>(blockIdx.x) *
                                           (kNormThreads / (kTeam > 0 ? kTeam : 1)) +
                                       threadIdx.x / (kTeam > 0 ? kTeam : 1)
                                 : blockIdx.x;
  const bool live = id < p.rows;
  const long long row = live ? id : 0;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const R* r = static_cast<const R*>(p.residual) + row * p.residual_stride;
  T* out = static_cast<T*>(p.out) + row * p.out_stride;
  R* nr = static_cast<R*>(p.new_residual) + row * p.new_residual_stride;

  Pack<T, V> xv[kVecs];
  ResidualVec<T, R, V> rv[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = (lane + i * team) * V;
    xv[i].zero();
    rv[i].zero();
    if (live && c < p.width) {
      xv[i].load_stream(x + c);
      rv[i].load(r + c);
    }
  }
  float binv = 1.0f;
  if (p.block_weight) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float f[V];
      xv[i].unpack(f);
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(f[e], f[e], ss);
    }
    binv = rsqrtf(team_sum<kTeam>(ss, smem) * p.inv_width + p.eps);
  }
  float rf[kVecs][V], ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = (lane + i * team) * V;
    float f[V];
    xv[i].unpack(f);
    rv[i].unpack(rf[i]);
    if (live && c < p.width) {
      if (p.block_weight) {
        Pack<T, V> wv;
        float wf[V];
        wv.load(static_cast<const T*>(p.block_weight) + c);
        wv.unpack(wf);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] *= binv * wf[e];
      }
      alignas(16) float s[V];
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = p.scale;
      if (p.channel_scale) {
#pragma unroll
        for (int e = 0; e < V; e += 4)
          *reinterpret_cast<float4*>(s + e) =
              *reinterpret_cast<const float4*>(p.channel_scale + c + e);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) rf[i][e] = fmaf(s[e], f[e], rf[i][e]);
      rv[i].pack_store(rf[i], nr + c);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(rf[i][e], rf[i][e], ss);
  }
  const float inv = rsqrtf(team_sum<kTeam>(ss, smem) * p.inv_width + p.eps);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = (lane + i * team) * V;
    if (!live || c >= p.width) continue;
    Pack<T, V> wv;
    float wf[V], y[V];
    wv.load(static_cast<const T*>(p.weight) + c);
    wv.unpack(wf);
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = rf[i][e] * inv * (wf[e] + p.weight_offset);
    wv.pack(y);
    wv.store(out + c);
  }
}

template <typename T, typename R>
__global__ void __launch_bounds__(256) gdn_add_norm_any_kernel(const NormParams p) {
  __shared__ float smem[32];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const R* r = static_cast<const R*>(p.residual) + row * p.residual_stride;
  const T* bw = static_cast<const T*>(p.block_weight);
  T* out = static_cast<T*>(p.out) + row * p.out_stride;
  R* nr = static_cast<R*>(p.new_residual) + row * p.new_residual_stride;
  float binv = 1.0f;
  if (bw) {
    float ss = 0.0f;
    for (int c = threadIdx.x; c < p.width; c += 256) ss = fmaf(to_float(x[c]), to_float(x[c]), ss);
    binv = rsqrtf(team_sum<0>(ss, smem) * p.inv_width + p.eps);
  }
  // r' by element, from the operands: nr may be r, so r' is formed twice before it is stored
  auto sum = [&](int c) {
    float v = to_float(x[c]);
    if (bw) v *= binv * to_float(bw[c]);
    return fmaf(p.channel_scale ? p.channel_scale[c] : p.scale, v, to_float(r[c]));
  };
  float ss = 0.0f;
  for (int c = threadIdx.x; c < p.width; c += 256) {
    const float v = sum(c);
    ss = fmaf(v, v, ss);
  }
  const float inv = rsqrtf(team_sum<0>(ss, smem) * p.inv_width + p.eps);
  for (int c = threadIdx.x; c < p.width; c += 256) {
    const float v = sum(c);
    nr[c] = from_float<R>(v);
    out[c] = from_float<T>(v * inv * (to_float(static_cast<const T*>(p.weight)[c]) + p.weight_offset));
  }
}

}  // namespace gdn
