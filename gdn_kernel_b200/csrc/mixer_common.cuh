// What the mixer kernels share: 16-byte vectors of the three element types, and
// the lookup of the packed sequence that a token tile belongs to.
#pragma once

#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace gdn {

// Status bits, as in the GDN kernels.
constexpr unsigned int kMixerBadSeqlens = 4u;
constexpr unsigned int kMixerBadIndex = 8u;

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }

// N consecutive elements as they lie in memory: one access of 16 or 8 bytes, or a
// single element where sizes or addresses allow no wider one.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * static_cast<int>(sizeof(T));
  using Raw = typename std::conditional<kBytes == 16, uint4,
                                        typename std::conditional<kBytes == 8, uint2, T>::type>::type;
  static_assert(kBytes == 16 || kBytes == 8 || N == 1, "a vector of 16 or 8 bytes, or one element");
  Raw raw;

  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  // Read once: no line kept in L1.
  __device__ __forceinline__ void load_stream(const T* p) {
    if constexpr (kBytes >= 8 && N > 1) raw = __ldcs(reinterpret_cast<const Raw*>(p));
    else raw = *p;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void zero() {
    if constexpr (kBytes == 16) raw = make_uint4(0u, 0u, 0u, 0u);
    else if constexpr (kBytes == 8) raw = make_uint2(0u, 0u);
    else raw = from_float<T>(0.0f);
  }
  __device__ __forceinline__ void unpack(float (&f)[N]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_float(e[i]);
  }
  __device__ __forceinline__ void pack(const float (&f)[N]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_float<T>(f[i]);
  }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair_bits(uint32_t x, uint32_t y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// sigmoid(v) = 1 / (1 + 2^(-v log2 e)) and v sigmoid(v), two at a time.  The rounded
// exponent leaves 1.5 |v| 2^-24 of the result, the rest a few units; a NaN stays one,
// and below -87 sigmoid is 0.  One reciprocal of both denominators' product is no
// faster (8192 tokens of 8192 channels: 49.1 us against 48.5 with one each; gated norm
// of 8192 x 4096: 36.5 against 36.7), and needs bounds on the exponents that lose small
// gates and NaNs, or a branch (50.4 and 39.5 us).
__device__ __forceinline__ float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fast_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint64_t sigmoid2(uint64_t v) {
  constexpr float kMinusLog2e = -1.4426950408889634f;
  const float2 t = unpair(mul2(v, pair(kMinusLog2e, kMinusLog2e)));
  const float2 f =
      unpair(add2(pair(fast_exp2(t.x), fast_exp2(t.y)), pair(1.0f, 1.0f)));
  return pair(fast_rcp(f.x), fast_rcp(f.y));
}
__device__ __forceinline__ uint64_t silu2(uint64_t v) { return mul2(v, sigmoid2(v)); }
__device__ __forceinline__ float sigmoid_f(float v) {
  return fast_rcp(1.0f + fast_exp2(-1.4426950408889634f * v));
}
__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f(v); }

// Elements of a 16-byte vector.
template <typename T> constexpr int kLanes = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i]
              : static_cast<long long>(reinterpret_cast<const int*>(p)[i]);
}

// The slot of entry i: the entry itself without indices; -1 for a padding entry
// (negative) and for one past the pool, which also raises the status bit.
__device__ __forceinline__ long long slot_of(const void* idx, int is64, long long i,
                                             long long pool, unsigned int* status, bool report) {
  if (idx == nullptr) return i;
  const long long s = index_at(idx, is64, i);
  if (s >= pool) {
    if (report) atomicOr(status, kMixerBadIndex);
    return -1;
  }
  return s < 0 ? -1 : s;
}

// One warp reports offsets that do not rise within [0, tokens].
__device__ __forceinline__ void check_offsets(const void* cu, int is64, int n, long long tokens,
                                              unsigned int* status) {
  bool bad = false;
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const long long s = index_at(cu, is64, i), e = index_at(cu, is64, i + 1);
    bad |= s < 0 || e < s || e > tokens;
  }
  if (bad) atomicOr(status, kMixerBadSeqlens);
}

// How many of the first n entries of the non-decreasing cu are below t: a
// 32-way search by one whole warp, one load of cu per lane and level.
__device__ __forceinline__ int count_below(const void* cu, int is64, int n, long long t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;   // entries before lo are below t, entries from hi on are not
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool below = at < hi && index_at(cu, is64, at) < t;
    const int k = __popc(__ballot_sync(0xffffffffu, below));   // probes below t: a prefix
    if (k == 0) return lo;
    lo = lo + (k - 1) * step + 1;
    hi = min(hi, lo - 1 + step);
  }
  return lo;
}

}  // namespace gdn
