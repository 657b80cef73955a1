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
// accuracy of bf16.  All exponents are in base 2.
//
// Sixteen warps with one role each, handing over through mbarriers:
//   0 TMA, two stages of {C, B, X}       1 issues the products
//   2 gates: sfx and log2 step           4-7 S -> M (thread = token row)
//   8-11 w X, and the state in registers (thread = token row / state row)
//   12-15 outputs (thread = token row)
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
constexpr uint32_t kScGate = kScH + kScanTile;            // per stage: g[128], sfx[128]
constexpr uint32_t kScMisc = kScGate + 2 * 1024;
constexpr uint32_t kScanSmem = kScMisc + 256;

// Tensor memory columns.
constexpr uint32_t kTmS = 0, kTmM = 128, kTmYd = 192, kTmYo = 256, kTmDs = 320;

// 2^v; 0 for -inf (and for results below the normal range).
__device__ __forceinline__ float scan_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

enum ScanBar {
  kBFull = 0, kBEmpty = 2, kBGateFull = 4, kBGateEmpty = 6, kBSFull = 8, kBSEmpty, kBMFull,
  kBYFull, kBYEmpty, kBXwFull, kBDsFull, kBHFull, kBHEmpty, kBDrain, kBCount
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
      if (i == kBEmpty || i == kBEmpty + 1) n = 1 + 4;                // products, output warps
      else if (i == kBGateEmpty || i == kBGateEmpty + 1) n = 12;
      else if (i == kBSEmpty || i == kBMFull || i == kBYEmpty || i == kBXwFull || i == kBHFull) n = 4;
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

  if (warp == 0) {
    // ------------------------------------------------ TMA
    int issued = 0;
    bool ok = true;
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1;
      if (c >= 2 && !(ok = wait(kBEmpty + st, (c >> 1) - 1, kStatusMmaTimeout))) break;
      if (elect_one()) {
        uint8_t* stage = smem + st * kScStage;
        uint64_t* bar = bars + kBFull + st;
        const int t0 = static_cast<int>(t_begin) + c * kScanQ;
        mbar_arrive_expect_tx(bar, (1 + 2 * (N / 64)) * kScanTile);
#pragma unroll
        for (int b = 0; b < N / 64; ++b) {
          tma_load_3d(stage + kScC + b * kScanTile, &tm_c, bar, 64 * b, group, t0);
          tma_load_3d(stage + kScB + b * kScanTile, &tm_b, bar, 64 * b, group, t0);
        }
        tma_load_3d(stage + kScX, &tm_x, bar, col0, head, t0);
      }
      __syncwarp();
      issued = c + 1;
    }
    if (!ok)   // aborted: the copies in flight land first
      for (int c = max(issued - 2, 0); c < issued; ++c) mbar_wait(bars + kBFull + (c & 1), (c >> 1) & 1);
  } else if (warp == 1) {
    // ------------------------------------------------ products
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
    bool ok = wait(kBFull, 0, kStatusTmaTimeout);
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
      if (c + 1 < nch) {
        if (!(ok = wait(kBFull + ((c + 1) & 1), (c + 1) >> 1, kStatusTmaTimeout))) break;
        if (!(ok = wait(kBSEmpty, c, kStatusMmaTimeout))) break;
        tc_fence_after();
        issue_s(c + 1);
      }
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
    }
    if (!ok) {   // aborted: the products in flight finish first
      if (elect_one()) umma_commit(bars + kBDrain);
      __syncwarp();
      mbar_wait(bars + kBDrain, 0);
    }
  } else if (warp == 2) {
    // ------------------------------------------------ gates
    const float a2 = -expf(p.A_log[head]) * 1.4426950408889634f;
    const float bias = p.dt_bias ? p.dt_bias[head] : 0.0f;
    const __nv_bfloat16* dt = p.dt + head;
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      const long long t0 = t_begin + static_cast<long long>(c) * kScanQ;
      float step[4], la[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 4 * lane + i;
        step[i] = t < n ? ssm_step_size(to_float(dt[(t0 + t) * p.dt_stride]) + bias) : 0.0f;
        la[i] = a2 * step[i];
      }
      float s3 = 0.0f, s2 = la[3], s1 = s2 + la[2], s0 = s1 + la[1];
      const float mine = s0 + la[0];
      float v = mine;   // sums over this lane and those after it
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_down_sync(0xffffffffu, v, o);
        if (lane + o < 32) v += u;
      }
      float after = __shfl_down_sync(0xffffffffu, v, 1);
      if (lane == 31) after = 0.0f;
      if (c >= 2 && !wait(kBGateEmpty + st, (c >> 1) - 1, kStatusMmaTimeout)) break;
      float* g = reinterpret_cast<float*>(smem + kScGate + st * 1024);
      const float4 sfx = make_float4(after + s0, after + s1, after + s2, after + s3);
      reinterpret_cast<float4*>(g + kScanQ)[lane] = sfx;
      // log2 of a zero step is -inf: a padded token has no weight anywhere
      reinterpret_cast<float4*>(g)[lane] =
          make_float4(sfx.x + log2f(step[0]), sfx.y + log2f(step[1]), sfx.z + log2f(step[2]),
                      sfx.w + log2f(step[3]));
      if (lane == 0) totals[st] = v;
      arrive(kBGateFull + st);
    }
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------ S -> M
    {   // blocks above the diagonal stay zero
      const uint32_t z[16] = {};
      for (int b = quad + 1; b < 4; ++b) tmem_st16(tmem + kTmM + 16 * b + tm_lane, z);
      tmem_wait_st();
    }
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      if (!wait(kBSFull, c, kStatusMmaTimeout)) break;
      if (c > 0 && !wait(kBYFull, c - 1, kStatusMmaTimeout)) break;   // the last M is read
      tc_fence_after();
      const float* g = reinterpret_cast<const float*>(smem + kScGate + st * 1024);
      const float mine = g[kScanQ + row];
      for (int b = 0; b <= quad; ++b) {
        float s[32];
        tmem_ld32(tmem + kTmS + 32 * b + tm_lane, s);
        tmem_wait_ld();
        uint32_t m[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 gv = *reinterpret_cast<const float4*>(g + 32 * b + 4 * j);
          const float f[4] = {gv.x, gv.y, gv.z, gv.w};
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)   // a select: a masked S may hold anything
            v[e] = 32 * b + 4 * j + e <= row ? s[4 * j + e] * scan_exp2(f[e] - mine) : 0.0f;
          m[2 * j] = pack_bf16x2(v[0], v[1]);
          m[2 * j + 1] = pack_bf16x2(v[2], v[3]);
        }
        tmem_st16(tmem + kTmM + 16 * b + tm_lane, m);
      }
      tmem_wait_st();
      tc_fence_before();
      arrive(kBSEmpty);
      arrive(kBMFull);
      arrive(kBGateEmpty + st);
    }
  } else if (warp >= 8 && warp < 12) {
    // ------------------------------------------------ w X and the state
    const bool state_row = row < N;
    float h[kScanCols];
#pragma unroll
    for (int j = 0; j < kScanCols; ++j)
      h[j] = carried && state_row ? p.state[sbase + static_cast<long long>(j) * N + row] : 0.0f;
    auto add_ds = [&](float decay) {
#pragma unroll
      for (int j = 0; j < kScanCols; ++j) h[j] *= decay;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int k = 2; k >= 0; --k) {   // the small parts first
          float d[32];
          tmem_ld32(tmem + kTmDs + 64 * k + 32 * b + tm_lane, d);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) h[32 * b + j] += d[j];
        }
    };
    bool ok = true;
    float decay = 1.0f;
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* stage = smem + st * kScStage;
      if (c > 0) {
        if (!(ok = wait(kBDsFull, c - 1, kStatusMmaTimeout))) break;
        tc_fence_after();
        add_ds(decay);
        tc_fence_before();
      }
      if (!(ok = wait(kBGateFull + st, c >> 1, kStatusMmaTimeout))) break;
      if (!(ok = wait(kBFull + st, c >> 1, kStatusTmaTimeout))) break;
      const float w = scan_exp2(reinterpret_cast<const float*>(smem + kScGate + st * 1024)[row]);
      decay = scan_exp2(totals[st]);
      const bool past = row >= n;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t off = sw128_off(row, j);
        uint4 u = *reinterpret_cast<const uint4*>(stage + kScX + off);
        if (past) u = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t in[4] = {u.x, u.y, u.z, u.w};
        uint32_t part[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&in[i]));
          v.x *= past ? 0.0f : w;
          v.y *= past ? 0.0f : w;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            part[k][i] = pack_bf16x2(v.x, v.y);
            const float2 r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&part[k][i]));
            v.x -= r.x;
            v.y -= r.y;
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<uint4*>(smem + kScXw + k * kScanTile + off) =
              make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
        if (past) {
          *reinterpret_cast<uint4*>(stage + kScX + off) = u;
#pragma unroll
          for (int b = 0; b < N / 64; ++b)
            *reinterpret_cast<uint4*>(stage + kScB + b * kScanTile + off) = u;
        }
      }
      fence_proxy_async_smem();
      arrive(kBXwFull);
      arrive(kBGateEmpty + st);
      if (c > 0 && !(ok = wait(kBHEmpty, c - 1, kStatusMmaTimeout))) break;
      if (state_row) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(smem + kScH + sw128_off(row, j)) =
              make_uint4(pack_bf16x2(h[8 * j], h[8 * j + 1]), pack_bf16x2(h[8 * j + 2], h[8 * j + 3]),
                         pack_bf16x2(h[8 * j + 4], h[8 * j + 5]), pack_bf16x2(h[8 * j + 6], h[8 * j + 7]));
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
        for (int j = 0; j < kScanCols; ++j)
          p.new_state[sbase + static_cast<long long>(j) * N + row] = h[j];
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------ outputs
    const float D = p.D ? p.D[head] : 0.0f;
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* x = smem + st * kScStage + kScX;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float e = scan_exp2(totals[st] - reinterpret_cast<const float*>(smem + kScGate + st * 1024)[kScanQ + row]);
      arrive(kBGateEmpty + st);
      if (!wait(kBYFull, c, kStatusMmaTimeout)) break;
      tc_fence_after();
      // the row's results take the place of its X in shared memory (no product
      // reads it any more), and the warp writes whole rows from there
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float yd[32], yo[32];
        tmem_ld32(tmem + kTmYd + 32 * b + tm_lane, yd);
        tmem_ld32(tmem + kTmYo + 32 * b + tm_lane, yo);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t off = sw128_off(row, 4 * b + j);
          const uint4 u = *reinterpret_cast<const uint4*>(x + off);
          const uint32_t in[4] = {u.x, u.y, u.z, u.w};
          uint32_t out[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&in[i]));
            const int k = 8 * j + 2 * i;
            out[i] = pack_bf16x2(fmaf(D, v.x, fmaf(e, yo[k], yd[k])),
                                 fmaf(D, v.y, fmaf(e, yo[k + 1], yd[k + 1])));
          }
          *reinterpret_cast<uint4*>(x + off) = make_uint4(out[0], out[1], out[2], out[3]);
        }
      }
      tc_fence_before();
      arrive(kBYEmpty);
      __nv_bfloat16* out = p.out +
          ((t_begin + static_cast<long long>(c) * kScanQ) * p.heads + head) * p.head_dim + col0;
      const long long ld = static_cast<long long>(p.heads) * p.head_dim;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = quad * 32 + 4 * i + (lane >> 3);
        const uint4 u = *reinterpret_cast<const uint4*>(x + sw128_off(r, lane & 7));
        if (r < n) *reinterpret_cast<uint4*>(out + r * ld + 8 * (lane & 7)) = u;
      }
      fence_proxy_async_smem();   // the next copy into this stage comes after these accesses
      arrive(kBEmpty + st);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace gdn
