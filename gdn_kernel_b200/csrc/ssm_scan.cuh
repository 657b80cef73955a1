// Selective state space scan over packed prompts, in chunks of Q = 128 tokens on
// the tensor cores.  With l_t = -exp(A_log) step_t and L_t the sum of l over the
// chunk's tokens up to t, a head's outputs and next state are
//   Y = M X + e^L (C h) + D X,   M_ts = (C_t . B_s) e^{L_t - L_s} step_s   (s <= t)
//   h' = e^{L_Q} h + B^T (w X),  w_s = e^{L_Q - L_s} step_s
// with h held as [N, 64], 64 of the head's P columns per CTA.
//
// A CTA carries the state of one (sequence, 64 columns of one head) from chunk
// to chunk, so x and y cross HBM once and no chunk state leaves the SM; B and C
// come from L2 for all but the first head of a group.  Four products a chunk:
//   S  = C B^T         128 x 128 x N, operands as TMA left them
//   dS = B^T [w X]     N x 192 x 128: w X is fp32, split exactly enough into
//                      three bf16 tiles side by side (24 bits), since the state
//                      is an fp32 result; summed when read back
//   Yo = C h           128 x 64 x N, h rounded to bf16
//   Yd = M X           128 x 64 x 128, M rounded to bf16 in tensor memory
// Yo and Yd stay apart because their row factors differ; the output rounds once
// more.  The roundings of h and M are 2^-9 of their terms each at most, as in
// the bf16 output itself.
//
// Decays come from sums towards the chunk's end, sfx_t = L_Q - L_t, which are
// small and hence accurate exactly where w is not; M and e^L only need the
// accuracy of bf16.  All exponents are in base 2.  M's 32 x 32 blocks below the
// diagonal ones need no exponential per element: with r the last token of the
// columns' block, L_t - L_s = (L_t - L_r) + (L_r - L_s), neither part positive,
// so e^{L_t - L_s} step_s is a row factor times a column factor.
//
// Sixteen warps with one role each, handing over through mbarriers:
//   0 TMA, two stages of {C, B, X}       1 issues the products
//   2-3 gates: sfx and log2 step         4-7 S -> M (thread = token row)
//   8-11 w X, and the state in registers (thread = token row / state row)
//   12-15 outputs (thread = token row)
// The products of a chunk are issued as dS, Yo, Yd, then S of the next chunk:
// while Yo, Yd and S run, w X of the next chunk is made from this one's end.
// Rows past a sequence's end hold other tokens: X, B and w X rows are zeroed
// there, so nothing of them (not even a NaN) enters a product's sum.
#pragma once

#include <cuda.h>

#include "gdn_ptx.cuh"
#include "ssm_recurrent.cuh"

namespace gdn {

constexpr int kScanQ = 128;
constexpr int kScanCols = 64;            // columns of P per CTA
constexpr int kScanThreads = 512;
constexpr uint32_t kScanTile = 16384;    // 128 rows x 64 bf16

// Shared memory: two stages of C (two halves of N), B (two halves) and X, the
// split w X (three tiles), h, the gates and the barriers.
constexpr uint32_t kScC = 0, kScB = 2 * kScanTile, kScX = 4 * kScanTile;
constexpr uint32_t kScStage = 5 * kScanTile;
constexpr uint32_t kScXw = 2 * kScStage;
constexpr uint32_t kScH = kScXw + 3 * kScanTile;
constexpr uint32_t kScGate = kScH + kScanTile;   // per stage: g[128], sfx[128], v[96] floats
constexpr uint32_t kScGateStage = (2 * kScanQ + 96) * 4;
constexpr uint32_t kScMisc = kScGate + 2 * kScGateStage;
constexpr uint32_t kScanSmem = kScMisc + 256;    // 227 KiB: all there is

// Tensor memory columns.
constexpr uint32_t kTmS = 0, kTmM = 128, kTmYd = 192, kTmYo = 256, kTmDs = 320;

// Registers per thread of the four warpgroups: together the 512 x 128 that the
// block is launched with.
constexpr int kScanRegs[4] = {72, 104, 208, 128};
static_assert(kScanRegs[0] + kScanRegs[1] + kScanRegs[2] + kScanRegs[3] == 4 * 128, "as launched");

template <int kRegs> __device__ __forceinline__ void scan_set_regs() {
  if constexpr (kRegs > 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  else if constexpr (kRegs < 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// 2^v; 0 for -inf (and for results below the normal range).
__device__ __forceinline__ float scan_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
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
__device__ __forceinline__ uint32_t pack_pair(uint64_t v) {
  const float2 f = unpair(v);
  return pack_bf16x2(f.x, f.y);
}
// Two packed bf16 as fp32.
__device__ __forceinline__ uint64_t unpack_pair(uint32_t u) {
  return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// The leading 8 bits of both significands as packed bf16, and what is left of
// the values: exact.  Three of these hold an fp32 value whole.
__device__ __forceinline__ uint32_t split_pair(uint64_t& v) {
  const float2 f = unpair(v);
  const uint32_t x = __float_as_uint(f.x), y = __float_as_uint(f.y);
  v = fma2(pair(__uint_as_float(x & 0xffff0000u), __uint_as_float(y & 0xffff0000u)),
           pair(-1.0f, -1.0f), v);
  return __byte_perm(x, y, 0x7632);
}

enum ScanBar {
  kBFullX = 0, kBFullBC = 2, kBEmpty = 4, kBEmptyC0 = 6, kBGateFull = 8, kBGateEmpty = 10,
  kBSFull = 12, kBMFull, kBYFull, kBYEmpty, kBXwFull, kBDsFull, kBHFull, kBHEmpty, kBDrain, kBCount
};

struct ScanParams {
  SsmParams s;
};

template <int N>
__global__ void __launch_bounds__(kScanThreads, 1)
gdn_ssm_scan_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_c, const ScanParams sp) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const SsmParams& p = sp.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, row = quad * 32 + lane;
  const int units = p.head_dim / kScanCols;
  const int head = blockIdx.x / units, col0 = blockIdx.x % units * kScanCols;
  const int group = head / (p.heads / p.groups);
  const int seq = blockIdx.y;
  const bool reporter = blockIdx.x == 0 && threadIdx.x == 0;

  const long long t_begin = index_at(p.cu, p.cu_is64, seq);
  const long long t_end = index_at(p.cu, p.cu_is64, seq + 1);
  if (t_begin < 0 || t_end < t_begin || t_end > p.tokens) {
    if (reporter) atomicOr(p.status, kMixerBadSeqlens);
    return;
  }
  const int len = static_cast<int>(t_end - t_begin);
  const int nch = (len + kScanQ - 1) / kScanQ;
  const long long slot = slot_of(p.slots, p.slots_is64, seq, p.pool, p.status, reporter);
  const bool carried = p.state && slot >= 0 && (!p.has_state || p.has_state[seq]);
  const long long sbase =
      ((slot < 0 ? 0 : slot) * p.heads + head) * static_cast<long long>(p.head_dim) * N +
      static_cast<long long>(col0) * N;
  if (nch == 0) {   // nothing but the state
    if (slot >= 0)
      for (int e = threadIdx.x; e < kScanCols * N; e += kScanThreads)
        p.new_state[sbase + e] = carried ? p.state[sbase + e] : 0.0f;
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kScMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kScMisc + 8 * kBCount);
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + kScMisc + 8 * kBCount + 4);
  float* totals = reinterpret_cast<float*>(smem + kScMisc + 8 * kBCount + 8);   // [2]
  static_assert(8 * kBCount + 16 <= 256, "barriers and flags fit");

  if (warp == 0) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kBCount; ++i) {
      int n = 1;
      if (i == kBEmpty || i == kBEmpty + 1) n = 1 + 4;   // products, output warps
      else if (i == kBGateEmpty || i == kBGateEmpty + 1) n = 12;
      else if (i == kBEmptyC0 || i == kBEmptyC0 + 1 || i == kBMFull || i == kBYEmpty ||
               i == kBXwFull || i == kBHFull)
        n = 4;
      mbar_init(bars + i, n);
    }
    fence_mbarrier_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_c);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const uint32_t tm_lane = static_cast<uint32_t>(quad * 32) << 16;

  // Waits are warp-uniform and bounded; the first to run out raises the abort
  // flag, which ends every role's loop.
  auto wait = [&](int bar, int phase, unsigned int code) {
    const int r = mbar_wait_or_abort(bars + bar, phase & 1, abort_flag);
    if (r < 0) atomicOr(p.status, code);
    return __all_sync(0xffffffffu, r == 1);
  };
  auto arrive = [&](int bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + bar);
  };
  auto chunk_len = [&](int c) { return min(kScanQ, len - c * kScanQ); };
  constexpr int kSteps = N / 16;   // k-steps over the state dimension

  if (warp < 4) {
    scan_set_regs<kScanRegs[0]>();
    if (warp == 0) {
      // ---------------------------------------------- TMA
      // C's first half is the last part of a stage to come free: the outputs
      // pass through it.
      int issued = 0;
      bool ok = true;
      for (int c = 0; c < nch; ++c) {
        const int st = c & 1;
        uint8_t* stage = smem + st * kScStage;
        const int t0 = static_cast<int>(t_begin) + c * kScanQ;
        if (c >= 2 && !(ok = wait(kBEmpty + st, (c >> 1) - 1, kStatusMmaTimeout))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bars + kBFullX + st, kScanTile);
          tma_load_3d(stage + kScX, &tm_x, bars + kBFullX + st, col0, head, t0);
          uint64_t* bar = bars + kBFullBC + st;
          mbar_arrive_expect_tx(bar, 2 * (N / 64) * kScanTile);
#pragma unroll
          for (int b = 0; b < N / 64; ++b)
            tma_load_3d(stage + kScB + b * kScanTile, &tm_b, bar, 64 * b, group, t0);
          if constexpr (N == 128) tma_load_3d(stage + kScC + kScanTile, &tm_c, bar, 64, group, t0);
        }
        __syncwarp();
        issued = c + 1;
        if (c >= 2) ok = wait(kBEmptyC0 + st, (c >> 1) - 1, kStatusMmaTimeout);
        if (elect_one()) tma_load_3d(stage + kScC, &tm_c, bars + kBFullBC + st, 0, group, t0);
        __syncwarp();
        if (!ok) break;
      }
      if (!ok)   // aborted: the copies in flight land first
        for (int c = max(issued - 2, 0); c < issued; ++c) {
          mbar_wait(bars + kBFullX + (c & 1), (c >> 1) & 1);
          mbar_wait(bars + kBFullBC + (c & 1), (c >> 1) & 1);
        }
    } else if (warp == 1) {
      // ---------------------------------------------- products
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, 0, 0);
      constexpr uint32_t idesc_y = idesc_bf16_f32(128, 64, 0, 1);
      constexpr uint32_t idesc_ds = idesc_bf16_f32(128, 192, 1, 1);
      const uint32_t base = smem_u32(smem);
      auto issue_s = [&](int c) {
        const uint32_t st = base + (c & 1) * kScStage;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const uint32_t off = (s >> 2) * kScanTile + (s & 3) * 32;
            umma_bf16(tmem + kTmS, sdesc_sw128(st + kScC + off, 16, 1024),
                      sdesc_sw128(st + kScB + off, 16, 1024), idesc_s, s > 0);
          }
          umma_commit(bars + kBSFull);
        }
        __syncwarp();
      };
      bool ok = wait(kBFullBC, 0, kStatusTmaTimeout);
      if (ok) issue_s(0);
      for (int c = 0; ok && c < nch; ++c) {
        const uint32_t st = base + (c & 1) * kScStage;
        const int ksteps = (chunk_len(c) + 15) / 16;
        if (!(ok = wait(kBXwFull, c, kStatusMmaTimeout))) break;
        tc_fence_after();
        if (elect_one()) {
          for (int s = 0; s < ksteps; ++s)
            umma_bf16(tmem + kTmDs, sdesc_sw128(st + kScB + s * 2048, kScanTile, 1024),
                      sdesc_sw128(base + kScXw + s * 2048, kScanTile, 1024), idesc_ds, s > 0);
          umma_commit(bars + kBDsFull);
        }
        __syncwarp();
        if (!(ok = wait(kBHFull, c, kStatusMmaTimeout))) break;
        if (c > 0 && !(ok = wait(kBYEmpty, c - 1, kStatusMmaTimeout))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
            umma_bf16(tmem + kTmYo,
                      sdesc_sw128(st + kScC + (s >> 2) * kScanTile + (s & 3) * 32, 16, 1024),
                      sdesc_sw128(base + kScH + s * 2048, kScanTile, 1024), idesc_y, s > 0);
          umma_commit(bars + kBHEmpty);
        }
        __syncwarp();
        if (!(ok = wait(kBMFull, c, kStatusMmaTimeout))) break;
        tc_fence_after();
        if (elect_one()) {
          for (int s = 0; s < ksteps; ++s)
            umma_bf16_ts(tmem + kTmYd, tmem + kTmM + s * 8,
                         sdesc_sw128(st + kScX + s * 2048, kScanTile, 1024), idesc_y, s > 0);
          umma_commit(bars + kBYFull);
          if (c + 2 < nch) umma_commit(bars + kBEmpty + (c & 1));
        }
        __syncwarp();
        if (c + 1 < nch) {   // M of this chunk is made, so S is read
          if (!(ok = wait(kBFullBC + ((c + 1) & 1), (c + 1) >> 1, kStatusTmaTimeout))) break;
          issue_s(c + 1);
        }
      }
      if (!ok) {   // aborted: the products in flight finish first
        if (elect_one()) umma_commit(bars + kBDrain);
        __syncwarp();
        mbar_wait(bars + kBDrain, 0);
      }
    } else {
      // ---------------------------------------------- gates
      // Two warps take turns; a chunk's dt are on their way while the chunk
      // before it (of this warp) is worked on.
      const float a2 = -expf(p.A_log[head]) * 1.4426950408889634f;
      const float bias = p.dt_bias ? p.dt_bias[head] : 0.0f;
      const __nv_bfloat16* dt = p.dt + t_begin * p.dt_stride + head;
      __nv_bfloat16 raw[4];
      auto load_dt = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = c * kScanQ + 4 * lane + i;
          raw[i] = __float2bfloat16_rn(0.0f);
          if (t < len) raw[i] = dt[t * p.dt_stride];
        }
      };
      load_dt(warp - 2);
      for (int c = warp - 2; c < nch; c += 2) {
        const int st = c & 1, n = chunk_len(c);
        float step[4], la[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          step[i] = 4 * lane + i < n ? ssm_step_size(to_float(raw[i]) + bias) : 0.0f;
          la[i] = a2 * step[i];
        }
        load_dt(c + 2);
        float sfx[4];
        sfx[3] = 0.0f;
        sfx[2] = la[3];
        sfx[1] = sfx[2] + la[2];
        sfx[0] = sfx[1] + la[1];
        float v = sfx[0] + la[0];   // sums over this lane and those after it
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float u = __shfl_down_sync(0xffffffffu, v, o);
          if (lane + o < 32) v += u;
        }
        float after = __shfl_down_sync(0xffffffffu, v, 1);
        if (lane == 31) after = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sfx[i] += after;
        // the last token of this lane's 32
        const float ref = __shfl_sync(0xffffffffu, sfx[3], lane | 7);
        if (c >= 2 && !wait(kBGateEmpty + st, (c >> 1) - 1, kStatusMmaTimeout)) break;
        float* g = reinterpret_cast<float*>(smem + kScGate + st * kScGateStage);
        reinterpret_cast<float4*>(g + kScanQ)[lane] = make_float4(sfx[0], sfx[1], sfx[2], sfx[3]);
        // log2 of a zero step is -inf: a padded token has no weight anywhere
        reinterpret_cast<float4*>(g)[lane] =
            make_float4(sfx[0] + log2f(step[0]), sfx[1] + log2f(step[1]), sfx[2] + log2f(step[2]),
                        sfx[3] + log2f(step[3]));
        if (lane < 24)
          reinterpret_cast<float4*>(g + 2 * kScanQ)[lane] =
              make_float4(step[0] * scan_exp2(sfx[0] - ref), step[1] * scan_exp2(sfx[1] - ref),
                          step[2] * scan_exp2(sfx[2] - ref), step[3] * scan_exp2(sfx[3] - ref));
        if (lane == 0) totals[st] = v;
        arrive(kBGateFull + st);
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------ S -> M
    scan_set_regs<kScanRegs[1]>();
    {   // blocks above the diagonal stay zero
      const uint32_t z[16] = {};
      for (int b = quad + 1; b < 4; ++b) tmem_st16(tmem + kTmM + 16 * b + tm_lane, z);
      tmem_wait_st();
    }
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float* g = reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage);
      const float mine = g[kScanQ + row];
      if (!wait(kBSFull, c, kStatusMmaTimeout)) break;   // also: the last M is read
      tc_fence_after();
      for (int b = 0; b < quad; ++b) {
        float s[32];
        tmem_ld32(tmem + kTmS + 32 * b + tm_lane, s);
        const float u = scan_exp2(g[kScanQ + 32 * b + 31] - mine);
        const uint64_t u2 = pair(u, u);
        const float4* v = reinterpret_cast<const float4*>(g + 2 * kScanQ + 32 * b);
        uint32_t m[16];
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 f = v[j];
          m[2 * j] = pack_pair(mul2(mul2(pair(s[4 * j], s[4 * j + 1]), u2), pair(f.x, f.y)));
          m[2 * j + 1] = pack_pair(mul2(mul2(pair(s[4 * j + 2], s[4 * j + 3]), u2), pair(f.z, f.w)));
        }
        tmem_st16(tmem + kTmM + 16 * b + tm_lane, m);
      }
      {
        float s[32];
        tmem_ld32(tmem + kTmS + 32 * quad + tm_lane, s);
        const float4* f4 = reinterpret_cast<const float4*>(g + 32 * quad);
        uint32_t m[16];
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 gv = f4[j];
          const float f[4] = {gv.x, gv.y, gv.z, gv.w};
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)   // a select: a masked S may hold anything
            v[e] = 4 * j + e <= lane ? s[4 * j + e] * scan_exp2(f[e] - mine) : 0.0f;
          m[2 * j] = pack_bf16x2(v[0], v[1]);
          m[2 * j + 1] = pack_bf16x2(v[2], v[3]);
        }
        tmem_st16(tmem + kTmM + 16 * quad + tm_lane, m);
      }
      tmem_wait_st();
      tc_fence_before();
      arrive(kBMFull);
      arrive(kBGateEmpty + st);
    }
  } else if (warp < 12) {
    // ------------------------------------------------ w X and the state
    scan_set_regs<kScanRegs[2]>();
    const bool state_row = row < N;
    uint64_t h[kScanCols / 2];
#pragma unroll
    for (int j = 0; j < kScanCols / 2; ++j) {
      const float* src = p.state + sbase + static_cast<long long>(2 * j) * N + row;
      const bool read = carried && state_row;
      h[j] = pair(read ? src[0] : 0.0f, read ? src[N] : 0.0f);
    }
    auto add_ds = [&](float decay) {
      const uint64_t d2 = pair(decay, decay);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float d[3][32];
#pragma unroll
        for (int k = 0; k < 3; ++k) tmem_ld32(tmem + kTmDs + 64 * k + 32 * b + tm_lane, d[k]);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {   // the small parts first
          const uint64_t t = add2(add2(pair(d[2][2 * j], d[2][2 * j + 1]),
                                       pair(d[1][2 * j], d[1][2 * j + 1])),
                                  pair(d[0][2 * j], d[0][2 * j + 1]));
          h[16 * b + j] = fma2(h[16 * b + j], d2, t);
        }
      }
    };
    bool ok = true;
    float decay = 1.0f;
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* stage = smem + st * kScStage;
      if (!(ok = wait(kBGateFull + st, c >> 1, kStatusMmaTimeout))) break;
      const float w = scan_exp2(reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage)[row]);
      const float next_decay = scan_exp2(totals[st]);
      arrive(kBGateEmpty + st);
      if (c > 0) {
        if (!(ok = wait(kBDsFull, c - 1, kStatusMmaTimeout))) break;
        tc_fence_after();
        add_ds(decay);
        tc_fence_before();
      }
      decay = next_decay;
      if (!(ok = wait(kBFullX + st, c >> 1, kStatusTmaTimeout))) break;
      if (n < kScanQ) {   // a last, short chunk: what lies past it must not count
        if (!(ok = wait(kBFullBC + st, c >> 1, kStatusTmaTimeout))) break;
        if (row >= n) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t off = sw128_off(row, j);
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(stage + kScX + off) = z;
#pragma unroll
            for (int b = 0; b < N / 64; ++b)
              *reinterpret_cast<uint4*>(stage + kScB + b * kScanTile + off) = z;
          }
        }
      }
      const uint64_t w2 = pair(w, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t off = sw128_off(row, j);
        const uint4 u = *reinterpret_cast<const uint4*>(stage + kScX + off);
        const uint32_t in[4] = {u.x, u.y, u.z, u.w};
        uint32_t part[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint64_t v = mul2(unpack_pair(in[i]), w2);
          part[0][i] = split_pair(v);
          part[1][i] = split_pair(v);
          part[2][i] = pack_pair(v);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<uint4*>(smem + kScXw + k * kScanTile + off) =
              make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
      }
      fence_proxy_async_smem();
      arrive(kBXwFull);
      if (c > 0 && !(ok = wait(kBHEmpty, c - 1, kStatusMmaTimeout))) break;
      if (state_row) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(smem + kScH + sw128_off(row, j)) =
              make_uint4(pack_pair(h[4 * j]), pack_pair(h[4 * j + 1]), pack_pair(h[4 * j + 2]),
                         pack_pair(h[4 * j + 3]));
      }
      fence_proxy_async_smem();
      arrive(kBHFull);
    }
    if (ok && wait(kBDsFull, nch - 1, kStatusMmaTimeout)) {
      tc_fence_after();
      add_ds(decay);
      tc_fence_before();
      if (slot >= 0 && state_row) {
#pragma unroll
        for (int j = 0; j < kScanCols / 2; ++j) {
          float* dst = p.new_state + sbase + static_cast<long long>(2 * j) * N + row;
          const float2 f = unpair(h[j]);
          dst[0] = f.x;
          dst[N] = f.y;
        }
      }
    }
  } else {
    // ------------------------------------------------ outputs
    scan_set_regs<kScanRegs[3]>();
    const float D = p.D ? p.D[head] : 0.0f;
    const uint64_t D2 = pair(D, D);
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* stage = smem + st * kScStage;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float e = scan_exp2(
          totals[st] - reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage)[kScanQ + row]);
      arrive(kBGateEmpty + st);
      if (!wait(kBFullX + st, c >> 1, kStatusTmaTimeout)) break;
      uint4 x[8];   // kept here so that the stage can be refilled early
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = *reinterpret_cast<const uint4*>(stage + kScX + sw128_off(row, j));
      arrive(kBEmpty + st);
      if (!wait(kBYFull, c, kStatusMmaTimeout)) break;
      tc_fence_after();
      // the row's results go to C's first half in shared memory (no product
      // reads it any more), from where the warp writes whole rows
      const uint64_t e2 = pair(e, e);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float yd[32], yo[32];
        tmem_ld32(tmem + kTmYd + 32 * b + tm_lane, yd);
        tmem_ld32(tmem + kTmYo + 32 * b + tm_lane, yo);
        tmem_wait_ld();
        if (b == 1) {
          tc_fence_before();
          arrive(kBYEmpty);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t in[4] = {x[4 * b + j].x, x[4 * b + j].y, x[4 * b + j].z, x[4 * b + j].w};
          uint32_t out[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = 8 * j + 2 * i;
            out[i] = pack_pair(fma2(D2, unpack_pair(in[i]),
                                    fma2(e2, pair(yo[k], yo[k + 1]), pair(yd[k], yd[k + 1]))));
          }
          *reinterpret_cast<uint4*>(stage + kScC + sw128_off(row, 4 * b + j)) =
              make_uint4(out[0], out[1], out[2], out[3]);
        }
      }
      __syncwarp();
      __nv_bfloat16* out = p.out +
          ((t_begin + static_cast<long long>(c) * kScanQ) * p.heads + head) * p.head_dim + col0;
      const long long ld = static_cast<long long>(p.heads) * p.head_dim;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = quad * 32 + 4 * i + (lane >> 3);
        const uint4 u = *reinterpret_cast<const uint4*>(stage + kScC + sw128_off(r, lane & 7));
        if (r < n) *reinterpret_cast<uint4*>(out + r * ld + 8 * (lane & 7)) = u;
      }
      fence_proxy_async_smem();   // the next copy into this half comes after these accesses
      arrive(kBEmptyC0 + st);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace gdn
