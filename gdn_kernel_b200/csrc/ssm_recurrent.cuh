// Selective state space recurrence, token by token.  Per head, with the fp32
// state h [P, N] (N contiguous, as the GDN state is k-last):
//   step = softplus(dt + dt_bias),   h <- exp(-exp(A_log) step) h + (step x) B^T
//   y = h C + D x
// Rows p of h are independent.  Eight lanes share a row, each owning N / 8
// columns as 16-byte vectors at columns 4 lane + 32 j, so that a warp's access
// covers four rows in whole lines and a row's dot product is a three-level
// shuffle; a thread carries kRows rows, whose loads are all issued first.
//
// One token per sequence moves the state in and out once (2 P N 4 bytes of
// each head) and does 5 P N operations on it: memory bounds it.  64 sequences, 64
// heads of 64, state 128: 44 us, 6.1 TB/s, 93 % of a plain copy's rate.
#pragma once

#include "mixer_common.cuh"

namespace gdn {

constexpr int kSsmThreads = 128;
constexpr int kSsmRows = 4;                                        // rows of a thread
constexpr int kSsmBlockRows = kSsmThreads / 8 * kSsmRows;          // 64

struct SsmParams {
  const __nv_bfloat16* x;      // [T, H, P], tokens x_stride apart
  const __nv_bfloat16* dt;     // [T, H], tokens dt_stride apart
  const __nv_bfloat16* B;      // [T, G, N], tokens b_stride apart
  const __nv_bfloat16* C;      // [T, G, N], tokens c_stride apart
  const float* A_log;          // [H]
  const float* D;              // [H] or nullptr
  const float* dt_bias;        // [H] or nullptr
  const float* state;          // [pool, H, P, N] or nullptr (zero)
  float* new_state;            // [pool, H, P, N], may be state
  __nv_bfloat16* out;          // [T, H, P], contiguous
  const void* cu;              // prompts: [N + 1]
  const void* slots;           // read slots, or nullptr (slot = sequence)
  const void* write_slots;     // or nullptr (the read slots)
  const uint8_t* has_state;    // [N] or nullptr (all)
  unsigned int* status;
  long long x_stride, dt_stride, b_stride, c_stride, pool, tokens;
  int cu_is64, slots_is64, seqs, heads, groups, head_dim;
};

// softplus without overflow; large arguments are their own result.
__device__ __forceinline__ float ssm_step_size(float v) {
  return v > 20.0f ? v : log1pf(expf(v));
}

// A token's operands of one thread, as they lie in memory: eight lanes' columns
// of B and C, and the thread's rows of x.
template <int N>
struct SsmToken {
  uint2 b[N / 32], c[N / 32];
  __nv_bfloat16 x[kSsmRows], dt;
  __device__ __forceinline__ void load(const SsmParams& p, long long t, int head, int group, int l8,
                                       int row0) {
    const __nv_bfloat16* B = p.B + t * p.b_stride + group * N + 4 * l8;
    const __nv_bfloat16* C = p.C + t * p.c_stride + group * N + 4 * l8;
#pragma unroll
    for (int j = 0; j < N / 32; ++j) {
      b[j] = *reinterpret_cast<const uint2*>(B + 32 * j);
      c[j] = *reinterpret_cast<const uint2*>(C + 32 * j);
    }
    const __nv_bfloat16* src = p.x + t * p.x_stride + head * p.head_dim + row0;
#pragma unroll
    for (int i = 0; i < kSsmRows; ++i) x[i] = src[kSsmThreads / 8 * i];
    dt = p.dt[t * p.dt_stride + head];
  }
};

template <int N>
__device__ __forceinline__ void unpack_columns(const uint2 (&u)[N / 32], float (&f)[N / 8]) {
#pragma unroll
  for (int j = 0; j < N / 32; ++j) {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[j].x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[j].y));
    f[4 * j] = a.x; f[4 * j + 1] = a.y; f[4 * j + 2] = b.x; f[4 * j + 3] = b.y;
  }
}

// kPrompt: the tokens of sequence blockIdx.y in order, the next one's operands
// loaded while one is worked on; else the one token of batch entry blockIdx.y.
template <int N, bool kPrompt>
__global__ void __launch_bounds__(kSsmThreads) gdn_ssm_recurrent_kernel(const SsmParams p) {
  const int P = p.head_dim;
  const int parts = P / kSsmBlockRows;
  const int head = blockIdx.x / parts;
  const int group = head / (p.heads / p.groups);
  const int l8 = threadIdx.x & 7;
  const int row0 = (blockIdx.x % parts) * kSsmBlockRows + (threadIdx.x >> 3);   // then + 16 i
  const long long seq = blockIdx.y;
  const bool reporter = blockIdx.x == 0 && threadIdx.x == 0;
  constexpr int kStep = kSsmThreads / 8;

  long long t = seq, end = seq + 1;
  if constexpr (kPrompt) {
    t = index_at(p.cu, p.cu_is64, seq);
    end = index_at(p.cu, p.cu_is64, seq + 1);
    if (t < 0 || end < t || end > p.tokens) {
      if (reporter) atomicOr(p.status, kMixerBadSeqlens);
      return;
    }
  }
  const long long slot = slot_of(p.slots, p.slots_is64, seq, p.pool, p.status, reporter);
  const long long wslot =
      p.write_slots ? slot_of(p.write_slots, p.slots_is64, seq, p.pool, p.status, reporter) : slot;
  if (!kPrompt && slot < 0) {   // a padding entry
#pragma unroll
    for (int i = 0; i < kSsmRows; ++i)
      if (l8 == 0)
        p.out[(seq * p.heads + head) * P + row0 + kStep * i] = __float2bfloat16_rn(0.0f);
    return;
  }

  SsmToken<N> tok;
  if (t < end) tok.load(p, t, head, group, l8, row0);
  float h[kSsmRows][N / 8];
  const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[seq]);
#pragma unroll
  for (int i = 0; i < kSsmRows; ++i) {
    const float* src =
        p.state + ((slot * p.heads + head) * P + row0 + kStep * i) * static_cast<long long>(N);
#pragma unroll
    for (int j = 0; j < N / 32; ++j) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (carried) v = __ldcs(reinterpret_cast<const float4*>(src + 4 * l8 + 32 * j));
      h[i][4 * j] = v.x; h[i][4 * j + 1] = v.y; h[i][4 * j + 2] = v.z; h[i][4 * j + 3] = v.w;
    }
  }
  const float A = -expf(p.A_log[head]);
  const float bias = p.dt_bias ? p.dt_bias[head] : 0.0f;
  const float D = p.D ? p.D[head] : 0.0f;
  for (; t < end; ++t) {
    const SsmToken<N> now = tok;
    if (kPrompt && t + 1 < end) tok.load(p, t + 1, head, group, l8, row0);
    const float step = ssm_step_size(to_float(now.dt) + bias);
    const float decay = expf(A * step);
    float Bf[N / 8], Cf[N / 8];
    unpack_columns<N>(now.b, Bf);
    unpack_columns<N>(now.c, Cf);
#pragma unroll
    for (int i = 0; i < kSsmRows; ++i) {
      const float x = to_float(now.x[i]);
      const float xs = x * step;
      float y = 0.0f;
#pragma unroll
      for (int c = 0; c < N / 8; ++c) {
        h[i][c] = fmaf(decay, h[i][c], xs * Bf[c]);
        y = fmaf(h[i][c], Cf[c], y);
      }
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      y += __shfl_xor_sync(0xffffffffu, y, 4);
      if (l8 == 0)
        p.out[(t * p.heads + head) * P + row0 + kStep * i] = __float2bfloat16_rn(fmaf(D, x, y));
    }
  }
  if (wslot < 0) return;
#pragma unroll
  for (int i = 0; i < kSsmRows; ++i) {
    float* dst =
        p.new_state + ((wslot * p.heads + head) * P + row0 + kStep * i) * static_cast<long long>(N);
#pragma unroll
    for (int j = 0; j < N / 32; ++j)
      *reinterpret_cast<float4*>(dst + 4 * l8 + 32 * j) =
          make_float4(h[i][4 * j], h[i][4 * j + 1], h[i][4 * j + 2], h[i][4 * j + 3]);
  }
}

}  // namespace gdn
