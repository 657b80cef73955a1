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
// more.  The roundings of h and M are 2^-8 of their terms each at most, as in
// the bf16 output itself.
//
// Decays come from sums over blocks of 32 tokens: after a token to its block's end,
// and of whole blocks.  w and e^L add up such sums, none of them positive, and are
// small, hence accurate, exactly where the result is not.  The only differences are
// within a block, of sums that a floor under each token's decay (kScanGone) keeps
// below 9600: off by 2^-9 at most if all 32 tokens are as steep as that, 2^-16 with
// sums of 100.  All exponents are in base 2.  M's 32 x 32 blocks below the
// diagonal ones need no exponential per element: with r the last token of the
// columns' block, L_t - L_s = (L_t - L_r) + (L_r - L_s), neither part positive,
// so e^{L_t - L_s} step_s is a row factor times a column factor.
//
// Twenty-eight warps with one role each, handing over through mbarriers:
//   0 issues the products                  3 TMA, two stages of {C, B, X}
//   1-2 gates                              4-7, 24-27 S -> M (thread = token row)
//   8-11 the state in registers (thread = state row)
//   12-15 outputs (thread = token row)     16-23 w X (thread = half a token row)
// One warp of each four works on a quarter of the rows, and M's last rows are the
// longest: the warp that issues sits with the first quarter.
// The products of a chunk are issued as dS, Yo, S of the next chunk, Yd: M is then
// made while dS and Yo run.
// Rows past a sequence's end hold other tokens: X, B and w X rows are zeroed
// there, so nothing of them (not even a NaN) enters a product's sum.
//
// Measured: 8192 tokens, 64 heads of 64, state 128, 96 us with the kernel of the
// pieces' states (20 us); 20011 ragged tokens of 32 heads of 128, state 64, 163-170.
// A chunk takes about 4000 clocks, its shared-memory traffic 3070 (384 KB: 208 of
// product operands, 80 of arriving tiles, 96 of x, w X and h), the tensor pipe is
// active for 2750; the rest is handing over.  128 tokens a chunk, because products
// of 64 rows run at half rate; 64 columns, because 128 need 320 KB of shared memory.
// The roles' loops together have to stay near 32 KB of code: at 75 KB a chunk took
// 7600 clocks, waiting for instructions.
#pragma once

#include <cuda.h>

#include "gdn_ptx.cuh"
#include "ssm_recurrent.cuh"

namespace gdn {

constexpr int kScanQ = 128;
constexpr int kScanCols = 64;            // columns of P per CTA
constexpr int kScanThreads = 896;
constexpr uint32_t kScanTile = 16384;    // 128 rows x 64 bf16

// Shared memory: two stages of C (two halves of N), B (two halves) and X, the
// split w X (three tiles), h, the gates and the barriers (with the blocks' decays).
constexpr uint32_t kScC = 0, kScB = 2 * kScanTile, kScX = 4 * kScanTile;
constexpr uint32_t kScStage = 5 * kScanTile;
constexpr uint32_t kScXw = 2 * kScStage;
constexpr uint32_t kScH = kScXw + 3 * kScanTile;
constexpr uint32_t kScGate = kScH + kScanTile;   // per stage: step[128], end[128], v[96] floats
constexpr uint32_t kScGateStage = (2 * kScanQ + 96) * 4;
constexpr uint32_t kScMisc = kScGate + 2 * kScGateStage;
constexpr uint32_t kScItem = kScMisc + 224;       // barriers and flags before it
constexpr uint32_t kScanSmem = kScMisc + 256;     // 227 KiB: all there is

// Tensor memory columns.
constexpr uint32_t kTmS = 0, kTmM = 128, kTmYd = 192, kTmYo = 256, kTmDs = 320;

// Registers per thread by role; together no more than the 896 x 72 that the block
// is launched with.
constexpr int kScanLaunchRegs = 72;
constexpr int kRegsIssue = 48, kRegsM = 72, kRegsState = 120, kRegsOut = 80, kRegsScale = 56;
static_assert(kRegsIssue + 2 * kRegsM + kRegsState + kRegsOut + 2 * kRegsScale <= 7 * kScanLaunchRegs &&
                  kScanThreads * kScanLaunchRegs <= 65536,
              "as launched");

template <int kRegs> __device__ __forceinline__ void scan_set_regs() {
  if constexpr (kRegs > kScanLaunchRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  else if constexpr (kRegs < kScanLaunchRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// 2^v; 0 for -inf (and for results below the normal range).
__device__ __forceinline__ float scan_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
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
// A value that every lane holds, so that the compiler knows it: products, copies
// and their descriptors want uniform registers, and without this each is wrapped
// in a loop over the lanes' values (50 instructions per product).
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

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
  kBFullX = 0, kBFullBC = 2, kBEmpty = 4, kBGateFull = 6, kBGateEmpty = 8, kBSFull = 10,
  kBSEmpty, kBMFull, kBYFull, kBYEmpty, kBXwFull, kBDsFull, kBDsEmpty, kBHFull, kBHEmpty,
  kBDrain, kBCount
};

// Long sequences run in pieces of seg_chunks chunks side by side: a first kernel
// makes the state that each part of a piece (`parts` of them, except in a
// sequence's last piece) adds by itself, and its decay; the scan of a piece then
// starts from the sum of those before it.
struct ScanParams {
  SsmParams s;
  int seg_chunks;      // chunks of a piece, a multiple of parts; 0: sequences are not divided
  int parts;
  int max_full;        // grid rows for whole pieces; the last piece of every sequence follows
  float* seg_state;    // [max_full (parts + 1)][H][P][N]: the parts' states, then carried states
                       // of divided sequences (read in place of a state updated in place)
  float* seg_decay;    // [max_full parts][H]: log2 of the parts' decays
};

struct ScanItem {
  int seq;             // -1: nothing to do
  int c0, chunks;      // the piece's chunks within the sequence
  int first_row;       // row of the sequence's first whole piece in seg_state
  int piece, pieces;
  int t_begin, len;    // of the sequence (tokens are below 2^31)
};

// The piece of grid row `item`.  Whole pieces come first, so that the long work
// starts first: row r is the r-th whole piece over all sequences, found by a
// running sum, 32 sequences at a time, by one warp.  A sequence of bad offsets, or
// whose pieces do not fit the grid and the workspace, is reported and skipped.
__device__ inline void scan_item(const ScanParams& sp, int item, ScanItem* out) {
  const SsmParams& p = sp.s;
  const int lane = threadIdx.x & 31;
  const int want_seq = item - sp.max_full;   // >= 0: the last piece of that sequence
  int before = 0, seq = -1, first_row = 0, begin = 0, len = -1, full = 0;
#pragma unroll 1
  for (int base = sp.seg_chunks > 0 ? 0 : want_seq; base < p.seqs; base += 32) {
    const int i = base + lane;
    begin = 0;
    len = -1;
    if (i < p.seqs) {
      const long long s = index_at(p.cu, p.cu_is64, i), e = index_at(p.cu, p.cu_is64, i + 1);
      if (s >= 0 && e >= s && e <= p.tokens) {
        begin = static_cast<int>(s);
        len = static_cast<int>(e - s);
      }
    }
    full = sp.seg_chunks > 0 && len > 0 ? (len + kScanQ - 1) / kScanQ / sp.seg_chunks : 0;
    int sum = full;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    const bool here = want_seq >= 0 ? i == want_seq
                                    : item >= before + sum - full && item < before + sum;
    const unsigned int hit = __ballot_sync(0xffffffffu, here);
    if (hit) {
      const int src = __ffs(hit) - 1;
      seq = base + src;
      first_row = before + __shfl_sync(0xffffffffu, sum - full, src);
      begin = __shfl_sync(0xffffffffu, begin, src);
      len = __shfl_sync(0xffffffffu, len, src);
      full = __shfl_sync(0xffffffffu, full, src);
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane != 0) return;
  ScanItem it;
  it.seq = seq;
  it.t_begin = begin;
  it.len = len;
  it.first_row = first_row;
  // Offsets that fall and rise again can hold more whole pieces than the tokens
  // account for, and the workspace has rows for no more than those.
  if (seq >= 0 && (len < 0 || first_row + full > sp.max_full)) {
    atomicOr(p.status, kMixerBadSeqlens);
    it.seq = -1;
  }
  const int nch = (len + kScanQ - 1) / kScanQ;
  const int rest = nch - full * sp.seg_chunks;
  it.pieces = full + (rest > 0 || nch == 0 ? 1 : 0);
  it.piece = want_seq >= 0 ? full : item - first_row;
  it.chunks = want_seq >= 0 ? rest : sp.seg_chunks;
  if (want_seq >= 0 && rest == 0 && nch > 0) it.seq = -1;
  it.c0 = it.piece * sp.seg_chunks;
  *out = it;
}

// Waits are warp-uniform and bounded: so many tries, each of which sleeps 4 us here
// (256 of them took 1.02 ms for one warp and for 28; with a hint of a microsecond the
// whole was 2-3 % slower), so 2.1 seconds, near the limit of the GDN kernels' waits.
// A system that let tries return at once would leave 10 ms, a thousand times what
// the longest wait, a few chunks' work, takes.  The first to run out raises the
// abort flag, which ends every role's loop.  (A count takes a fraction of the code of
// a clock, and the roles' loops have to fit the instruction cache together.)
constexpr int kScanWaitTries = 1 << 19;
__device__ __forceinline__ bool scan_try_wait(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(addr), "r"(parity)
      : "memory");
  return ok != 0;
}

struct ScanSync {
  uint32_t bars;              // shared-memory address
  volatile int* abort_flag;   // a status code once a wait ran out
  __device__ __forceinline__ bool wait(int bar, int phase, int code) const {
    const uint32_t addr = bars + 8 * bar;
    int left = kScanWaitTries;
    while (!__all_sync(0xffffffffu, scan_try_wait(addr, phase & 1))) {
      if (*abort_flag != 0) return false;
      if (--left == 0) *abort_flag = code;
    }
    return true;
  }
  __device__ __forceinline__ void arrive(int bar) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bars + 8 * bar) : "memory");
  }
};

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|), in a few units of 2^-24.  The
// product -|v| log2 e is carried in two parts, head and rest, with log2 e split into
// its fp32 value and the difference: e = 2^head (1 + rest ln 2), as rest is small.
// log1p(e) is the series of its hyperbolic arctangent, with z = e / (2 + e):
// 2 atanh(z) = 2 (z + z^3 / 3 + z^5 / 5 + ...), z <= 1/3, where the terms from z^15
// on are below 2^-26 of the sum.
__device__ __forceinline__ float scan_step_size(float v) {
  constexpr double kLog2e = 1.4426950408889634;
  constexpr float kHead = static_cast<float>(kLog2e);
  constexpr float kRest = static_cast<float>(kLog2e - static_cast<double>(kHead));
  const float a = fmaxf(-fabsf(v), -150.0f);   // e underflows below; and -inf is a value
  const float hi = a * kHead;
  const float lo = fmaf(a, kHead, -hi) + a * kRest;
  float e = scan_exp2(hi);
  e = fmaf(e, lo * 0.6931471805599453f, e);
  const float z = __fdividef(e, 2.0f + e);
  const float q = z * z;
  float s = fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
  s = fmaf(s, q, 1.0f / 9.0f);
  s = fmaf(s, q, 1.0f / 7.0f);
  s = fmaf(s, q, 1.0f / 5.0f);
  s = fmaf(s, q, 1.0f / 3.0f);
  s = fmaf(s * q, z, z);
  return v != v ? v : fmaxf(v, 0.0f) + (s + s);
}

// A weight below this exponent, or a decay, is zero in fp32 whatever the rest.  So no
// token's decay counts as steeper, which keeps sums of 32 of them near enough to
// zero for their differences to be accurate, and finite for an infinite step.
constexpr float kScanGone = -300.0f;

// The gates of chunks by one warp, lane owning one token of each block of 32: the
// steps, the log2 decays after a token to its block's end, and of each block.  A
// chunk's dt are loaded while the one before it (of this warp) is worked on.
struct ScanGates {
  const __nv_bfloat16* dt;    // of the piece's first token and this head
  long long stride;
  float a2, bias;             // log2 decay per step, and dt_bias
  int len;                    // tokens of the piece
  __nv_bfloat16 raw[4];
  float step[4], end[4], block[4];
  __device__ __forceinline__ void fetch(int c) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int t = c * kScanQ + 32 * b + static_cast<int>(threadIdx.x & 31);
      raw[b] = __float2bfloat16_rn(0.0f);
      if (c >= 0 && t < len) raw[b] = dt[t * stride];
    }
  }
  __device__ __forceinline__ void start(const SsmParams& p, long long t_begin, int tokens, int head,
                                        int c) {
    dt = p.dt + t_begin * p.dt_stride + head;
    stride = p.dt_stride;
    a2 = -expf(p.A_log[head]) * 1.4426950408889634f;
    bias = p.dt_bias ? p.dt_bias[head] : 0.0f;
    len = tokens;
    fetch(c);
  }
  __device__ __forceinline__ void make(int c, int next) {
    const int lane = threadIdx.x & 31;
    float v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      step[b] = scan_step_size(to_float(raw[b]) + bias);
      v[b] = a2 * step[b];
      if (v[b] < kScanGone) v[b] = kScanGone;   // (a NaN stays)
      if (c * kScanQ + 32 * b + lane >= len) step[b] = v[b] = 0.0f;
    }
    fetch(next);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)   // sums over this lane and those after it
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float u = __shfl_down_sync(0xffffffffu, v[b], o);
        if (lane + o < 32) v[b] += u;
      }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float after = __shfl_down_sync(0xffffffffu, v[b], 1);
      end[b] = lane == 31 ? 0.0f : after;
      block[b] = __shfl_sync(0xffffffffu, v[b], 0);
    }
  }
};

// kN groups of eight columns from group j0 of row `row` of w X, split exactly into
// three bf16 tiles.  (Kept small: passes of 16 columns.)
template <int kN>
__device__ __forceinline__ void scan_scale_row(uint8_t* xw, const uint8_t* x, int row, int j0,
                                               float w) {
  const uint64_t w2 = pair(w, w);
#pragma unroll 2
  for (int j = j0; j < j0 + kN; ++j) {
    const uint32_t off = sw128_off(row, j);
    const uint4 u = *reinterpret_cast<const uint4*>(x + off);
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
      *reinterpret_cast<uint4*>(xw + k * kScanTile + off) =
          make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
  }
}

// ------------------------------------------------ the states of pieces
// One CTA per part of a whole piece that is not its sequence's last, and 64
// columns of a head: the state it adds, sum over its tokens of e^{L_end - L_s} step_s B_s x_s^T,
// in one accumulator.  Chunks run from the last to the first, so that weights
// only need the decays already seen, and end where those leave nothing.
constexpr int kStateThreads = 384;
constexpr uint32_t kSsB = 0, kSsX = 2 * kScanTile, kSsStage = 3 * kScanTile;
constexpr uint32_t kSsXw = 2 * kSsStage;                       // two sets of three tiles
constexpr uint32_t kSsGate = kSsXw + 6 * kScanTile;            // per stage: weights [128]
constexpr uint32_t kSsMisc = kSsGate + 2 * kScanQ * 4;
constexpr uint32_t kSsItem = kSsMisc + 208;
constexpr uint32_t kStateSmem = kSsMisc + 256;

enum StateBar {
  kAFull = 0, kAEmpty = 2, kAGateFull = 4, kAGateEmpty = 6, kAXwFull = 8, kAXwEmpty = 10, kADone = 12,
  kACount
};

template <int N>
__global__ void __launch_bounds__(kStateThreads, 1)
gdn_ssm_piece_state_kernel(const __grid_constant__ CUtensorMap tm_x,
                           const __grid_constant__ CUtensorMap tm_b, const ScanParams sp) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const SsmParams& p = sp.s;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int quad = warp & 3, row = quad * 32 + lane;
  const int units = p.head_dim / kScanCols;
  const int head = blockIdx.x / units, col0 = blockIdx.x % units * kScanCols;
  const int group = head / (p.heads / p.groups);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSsMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSsMisc + 8 * kACount);
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + kSsMisc + 8 * kACount + 4);
  // log2 decay of the chunks done before a stage's chunk, and including it
  float* later = reinterpret_cast<float*>(smem + kSsMisc + 8 * kACount + 8);   // [2][2]
  static_assert(8 * kACount + 24 <= 208 && sizeof(ScanItem) <= 48, "they fit");
  if (warp == 0) {
    tmem_alloc(tmem_ptr, 256);
    tmem_relinquish();
  }
  if (warp == 1 && lane == 0) {
    *abort_flag = 0;
#pragma unroll 1
    for (int i = 0; i < kACount; ++i)
      mbar_init(bars + i, i == kAGateEmpty || i == kAGateEmpty + 1 ? 6   // copies, products, 4 warps
                          : i == kAXwFull || i == kAXwFull + 1     ? 4
                                                                   : 1);
    fence_mbarrier_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_b);
  }
  const int part = blockIdx.y % sp.parts;
  if (warp == 2) scan_item(sp, blockIdx.y / sp.parts, reinterpret_cast<ScanItem*>(smem + kSsItem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const ScanItem& it = *reinterpret_cast<const ScanItem*>(smem + kSsItem);
  const int nch = warp_uniform(it.seq < 0 || it.piece == it.pieces - 1 ? 0 : it.chunks / sp.parts);
  const int c0 = warp_uniform(it.c0 + part * nch);
  const long long hbase = (static_cast<long long>(head) * p.head_dim + col0) * N;
  const long long per_slot = static_cast<long long>(p.heads) * p.head_dim * N;
  const uint32_t tmem = static_cast<uint32_t>(warp_uniform(static_cast<int>(*tmem_ptr)));
  const int t_last = warp_uniform(it.t_begin + (c0 + nch - 1) * kScanQ);
  const ScanSync sync{smem_u32(bars), abort_flag};
  // Whether a chunk counts after decays of `log_decay`: not once they leave nothing of
  // it, nor after a NaN, which the state then holds already.  All roles end by this.
  auto counts = [](float log_decay) { return log_decay > kScanGone; };
  auto more = [&](int i) { return counts(later[2 * (i & 1)]); };   // chunk i, from the end

  // the scan's blocks may take the SMs that this grid leaves or has done with
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (nch == 0) {
    // no such piece, or a sequence's last
  } else if (warp == 0) {
    int issued = 0;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < nch; ++i) {
      const int st = i & 1;
      if (!(ok = sync.wait(kAGateFull + st, i >> 1, kStatusMmaTimeout))) break;
      const bool go = more(i);
      sync.arrive(kAGateEmpty + st);
      if (!go) break;
      if (i >= 2 && !(ok = sync.wait(kAEmpty + st, (i >> 1) - 1, kStatusMmaTimeout))) break;
      if (elect_one()) {
        uint8_t* stage = smem + st * kSsStage;
        uint64_t* bar = bars + kAFull + st;
        const int t0 = t_last - i * kScanQ;
        mbar_arrive_expect_tx(bar, (1 + N / 64) * kScanTile);
        tma_load_3d(stage + kSsX, &tm_x, bar, col0, head, t0);
#pragma unroll
        for (int b = 0; b < N / 64; ++b)
          tma_load_3d(stage + kSsB + b * kScanTile, &tm_b, bar, 64 * b, group, t0);
      }
      __syncwarp();
      issued = i + 1;
    }
    if (!ok)   // aborted: the copies in flight land first
      for (int i = max(issued - 2, 0); i < issued; ++i) mbar_wait(bars + kAFull + (i & 1), (i >> 1) & 1);
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_bf16_f32(128, 192, 1, 1);
    const uint32_t base = smem_u32(smem);
#pragma unroll 1
    for (int i = 0; i < nch; ++i) {
      const int st = i & 1;
      if (!sync.wait(kAGateFull + st, i >> 1, kStatusMmaTimeout)) break;
      const bool go = more(i);
      sync.arrive(kAGateEmpty + st);
      if (!go) break;
      if (!sync.wait(kAXwFull + st, i >> 1, kStatusMmaTimeout)) break;   // the copies have landed too
      tc_fence_after();
      const uint64_t b_desc = sdesc_sw128(base + st * kSsStage + kSsB, kScanTile, 1024);
      const uint64_t xw_desc = sdesc_sw128(base + kSsXw + st * 3 * kScanTile, kScanTile, 1024);
#pragma unroll
      for (int s = 0; s < kScanQ / 16; ++s)
        umma_bf16_elect(tmem, sdesc_add(b_desc, s * 2048), sdesc_add(xw_desc, s * 2048), idesc,
                        i > 0 || s > 0);
      umma_commit_elect(bars + kAEmpty + st);
      umma_commit_elect(bars + kAXwEmpty + st);
    }
    // the sum is whole, or, after an abort, nothing is in flight any more
    umma_commit_elect(bars + kADone);
    mbar_wait(bars + kADone, 0);
  } else if (warp < 4) {
    const int last = c0 + nch - 1;
    ScanGates gates;
    gates.start(p, it.t_begin, it.len, head, warp - 2 < nch ? last - (warp - 2) : -1);
#pragma unroll 1
    for (int i = warp - 2; i < nch; i += 2) {
      const int st = i & 1;
      gates.make(last - i, i + 2 < nch ? last - i - 2 : -1);
      float done = 0.0f;   // the other warp's running total
      bool ended = false;  // at the chunk before: this one only passes that on to its warpgroup
      if (i > 0) {
        if (!sync.wait(kAGateFull + (st ^ 1), (i - 1) >> 1, kStatusMmaTimeout)) break;
        done = later[2 * (st ^ 1) + 1];
        ended = !more(i - 1);
      }
      if (i >= 2 && !sync.wait(kAGateEmpty + st, (i >> 1) - 1, kStatusMmaTimeout)) break;
      float* g = reinterpret_cast<float*>(smem + kSsGate + st * kScanQ * 4);
      float total = 0.0f;
#pragma unroll
      for (int b = 3; b >= 0; --b) {
        g[32 * b + lane] = gates.step[b] * scan_exp2(done + total + gates.end[b]);
        total += gates.block[b];
      }
      if (lane == 0) {
        later[2 * st] = done;
        later[2 * st + 1] = done + total;
        if (col0 == 0 && !ended && (i == nch - 1 || !counts(done)))
          sp.seg_decay[static_cast<long long>(blockIdx.y) * p.heads + head] = done + total;
      }
      sync.arrive(kAGateFull + st);
      if (!counts(done)) break;
    }
  } else {
    // two warpgroups, one chunk each in turn
    const int wg = (warp - 4) >> 2;
#pragma unroll 1
    for (int i = wg; i < nch; i += 2) {
      const int st = i & 1;
      if (!sync.wait(kAGateFull + st, i >> 1, kStatusMmaTimeout)) break;
      const bool go = more(i);
      const float w = reinterpret_cast<const float*>(smem + kSsGate + st * kScanQ * 4)[row];
      sync.arrive(kAGateEmpty + st);
      if (!go) break;
      if (!sync.wait(kAFull + st, i >> 1, kStatusTmaTimeout)) break;
      if (i >= 2 && !sync.wait(kAXwEmpty + st, (i >> 1) - 1, kStatusMmaTimeout)) break;
      scan_scale_row<8>(smem + kSsXw + st * 3 * kScanTile, smem + st * kSsStage + kSsX, row, 0, w);
      fence_proxy_async_smem();
      sync.arrive(kAXwFull + st);
    }
    // the result, half of the columns each
    if (sync.wait(kADone, 0, kStatusMmaTimeout)) {
      tc_fence_after();
      float d[3][32];
#pragma unroll
      for (int k = 0; k < 3; ++k)
        tmem_ld32(tmem + 64 * k + 32 * wg + (static_cast<uint32_t>(quad * 32) << 16), d[k]);
      tmem_wait_ld();
      if (row < N) {
        float* dst = sp.seg_state + blockIdx.y * per_slot + hbase + 32LL * wg * N + row;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          dst[static_cast<long long>(j) * N] = (d[2][j] + d[1][j]) + d[0][j];
      }
    }
    // A state that is updated in place is kept for the first piece, which may
    // run after the last one has stored its result.
    const long long slot = slot_of(p.slots, p.slots_is64, it.seq, p.pool, p.status, false);
    if (it.piece == 0 && part == 0 && p.state == p.new_state && slot >= 0) {
      float* dst = sp.seg_state +
                   (static_cast<long long>(sp.max_full) * sp.parts + it.first_row) * per_slot + hbase;
      for (int e = threadIdx.x - 128; e < kScanCols * N; e += kStateThreads - 128)
        dst[e] = p.state[slot * per_slot + hbase + e];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, static_cast<unsigned int>(*abort_flag));
  if (warp == 0) tmem_dealloc(tmem, 256);
}

template <int N>
__global__ void __launch_bounds__(kScanThreads, 1)
gdn_ssm_scan_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_c, const ScanParams sp) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const SsmParams& p = sp.s;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int quad = warp & 3, row = quad * 32 + lane;
  const int units = p.head_dim / kScanCols;
  const int head = blockIdx.x / units, col0 = blockIdx.x % units * kScanCols;
  const int group = head / (p.heads / p.groups);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kScMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kScMisc + 8 * kBCount);
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + kScMisc + 8 * kBCount + 4);
  float4* blocks = reinterpret_cast<float4*>(smem + kScMisc + 8 * kBCount + 8);   // [2]: decays
  static_assert(8 * kBCount + 40 <= 224 && (kScMisc + 8 * kBCount + 8) % 16 == 0 &&
                    sizeof(ScanItem) <= 32,
                "they fit");

  if (warp == 0) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  if (warp == 1) {   // a barrier per lane
    const int i = lane;
    int n = 1;
    if (i == kBEmpty || i == kBEmpty + 1) n = 1 + 4;   // products, output warps
    else if (i == kBGateEmpty || i == kBGateEmpty + 1) n = 24;
    else if (i == kBXwFull || i == kBMFull || i == kBSEmpty) n = 8;
    else if (i == kBYEmpty || i == kBHFull || i == kBDsEmpty) n = 4;
    if (i < kBCount) mbar_init(bars + i, n);
    if (lane == 31) {
      *abort_flag = 0;
      prefetch_tmap(&tm_x);
      prefetch_tmap(&tm_b);
      prefetch_tmap(&tm_c);
    }
    fence_mbarrier_init();
  }
  static_assert(kBCount <= 31, "a lane each");
  if (warp == 2) scan_item(sp, blockIdx.y, reinterpret_cast<ScanItem*>(smem + kScItem));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const ScanItem& it = *reinterpret_cast<const ScanItem*>(smem + kScItem);
  const int nch = warp_uniform(it.seq < 0 ? 0 : it.chunks);
  const int t_begin = warp_uniform(it.t_begin + it.c0 * kScanQ);
  const int len = warp_uniform(min(it.len - it.c0 * kScanQ, nch * kScanQ));
  const long long hbase = (static_cast<long long>(head) * p.head_dim + col0) * N;
  const long long per_slot = static_cast<long long>(p.heads) * p.head_dim * N;
  const uint32_t tmem = static_cast<uint32_t>(warp_uniform(static_cast<int>(*tmem_ptr)));
  const uint32_t tm_lane = static_cast<uint32_t>(quad * 32) << 16;

  const ScanSync sync{smem_u32(bars), abort_flag};
  auto wait = [&](int bar, int phase, int code) { return sync.wait(bar, phase, code); };
  auto arrive = [&](int bar) { sync.arrive(bar); };
  auto chunk_len = [&](int c) { return min(kScanQ, len - c * kScanQ); };
  // The sequence's slot, and whether it starts from a carried state.
  auto find_state = [&](bool& carried) {
    const long long slot = slot_of(p.slots, p.slots_is64, it.seq, p.pool, p.status,
                                   blockIdx.x == 0 && (threadIdx.x & 31) == 0);
    carried = p.state && slot >= 0 && (!p.has_state || p.has_state[it.seq]);
    return slot;
  };
  constexpr int kSteps = N / 16;   // k-steps over the state dimension

  // The kernel before made the states of pieces.  This one may have started beside
  // it (programmatic launch); what needs them waits here, all of it, so that no
  // bounded wait below depends on how long that kernel takes.
  if (it.pieces > 1 && (it.piece > 0 || p.state == p.new_state))
    asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nch == 0) {
    if (it.seq >= 0) {   // an empty sequence: nothing but the state
      bool carried;
      const long long slot = find_state(carried);
      if (slot >= 0)
        for (int e = threadIdx.x; e < kScanCols * N; e += kScanThreads) {
          const long long at = slot * per_slot + hbase + e;
          p.new_state[at] = carried ? p.state[at] : 0.0f;
        }
    }
  } else if (warp < 4) {
    scan_set_regs<kRegsIssue>();
    if (warp == 3) {
      // ---------------------------------------------- TMA
      int issued = 0;
      bool ok = true;
#pragma unroll 1
      for (int c = 0; c < nch; ++c) {
        const int st = c & 1;
        uint8_t* stage = smem + st * kScStage;
        const int t0 = t_begin + c * kScanQ;
        if (c >= 2 && !(ok = wait(kBEmpty + st, (c >> 1) - 1, kStatusMmaTimeout))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bars + kBFullX + st, kScanTile);
          tma_load_3d(stage + kScX, &tm_x, bars + kBFullX + st, col0, head, t0);
          uint64_t* bar = bars + kBFullBC + st;
          mbar_arrive_expect_tx(bar, 2 * (N / 64) * kScanTile);
#pragma unroll
          for (int b = 0; b < N / 64; ++b) {
            tma_load_3d(stage + kScB + b * kScanTile, &tm_b, bar, 64 * b, group, t0);
            tma_load_3d(stage + kScC + b * kScanTile, &tm_c, bar, 64 * b, group, t0);
          }
        }
        __syncwarp();
        issued = c + 1;
      }
      if (!ok)   // aborted: the copies in flight land first
        for (int c = max(issued - 2, 0); c < issued; ++c) {
          mbar_wait(bars + kBFullX + (c & 1), (c >> 1) & 1);
          mbar_wait(bars + kBFullBC + (c & 1), (c >> 1) & 1);
        }
    } else if (warp == 0) {
      // ---------------------------------------------- products
      // Every lane runs the whole sequence and an elected one issues: the warp
      // never diverges, so descriptors stay in uniform registers.  (Inside a
      // branch on the elected lane each product took twice as long to issue, and
      // in a loop over k-steps four times.)
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, 0, 0);
      constexpr uint32_t idesc_y = idesc_bf16_f32(128, 64, 0, 1);
      constexpr uint32_t idesc_ds = idesc_bf16_f32(128, 192, 1, 1);
      const uint32_t base = smem_u32(smem);
      const uint64_t xw_desc = sdesc_sw128(base + kScXw, kScanTile, 1024);
      const uint64_t h_desc = sdesc_sw128(base + kScH, kScanTile, 1024);
      bool ok = true;
#pragma unroll 1
      for (int c = -1; c < nch; ++c) {
        const uint32_t st = base + (c & 1) * kScStage;
        if (c >= 0) {
          const uint64_t bt_desc = sdesc_sw128(st + kScB, kScanTile, 1024);
          const uint64_t c_desc = sdesc_sw128(st + kScC, 16, 1024);
          if (!(ok = wait(kBXwFull, c, kStatusMmaTimeout))) break;
          if (c > 0 && !(ok = wait(kBDsEmpty, c - 1, kStatusMmaTimeout))) break;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < kScanQ / 16; ++s)
            umma_bf16_elect(tmem + kTmDs, sdesc_add(bt_desc, s * 2048), sdesc_add(xw_desc, s * 2048),
                            idesc_ds, s > 0);
          umma_commit_elect(bars + kBDsFull);
          if (!(ok = wait(kBHFull, c, kStatusMmaTimeout))) break;
          if (c > 0 && !(ok = wait(kBYEmpty, c - 1, kStatusMmaTimeout))) break;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
            umma_bf16_elect(tmem + kTmYo, sdesc_add(c_desc, (s >> 2) * kScanTile + (s & 3) * 32),
                            sdesc_add(h_desc, s * 2048), idesc_y, s > 0);
          umma_commit_elect(bars + kBHEmpty);
        }
        if (c + 1 < nch) {
          const uint32_t next = base + ((c + 1) & 1) * kScStage;
          const uint64_t c_desc = sdesc_sw128(next + kScC, 16, 1024);
          const uint64_t b_desc = sdesc_sw128(next + kScB, 16, 1024);
          if (!(ok = wait(kBFullBC + ((c + 1) & 1), (c + 1) >> 1, kStatusTmaTimeout))) break;
          if (c >= 0 && !(ok = wait(kBSEmpty, c, kStatusMmaTimeout))) break;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const uint32_t off = (s >> 2) * kScanTile + (s & 3) * 32;
            umma_bf16_elect(tmem + kTmS, sdesc_add(c_desc, off), sdesc_add(b_desc, off), idesc_s, s > 0);
          }
          umma_commit_elect(bars + kBSFull);
        }
        if (c >= 0) {
          const uint64_t x_desc = sdesc_sw128(st + kScX, kScanTile, 1024);
          if (!(ok = wait(kBMFull, c, kStatusMmaTimeout))) break;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < kScanQ / 16; ++s)
            umma_bf16_ts_elect(tmem + kTmYd, tmem + kTmM + s * 8, sdesc_add(x_desc, s * 2048),
                               idesc_y, s > 0);
          umma_commit_elect(bars + kBYFull);
          if (c + 2 < nch) umma_commit_elect(bars + kBEmpty + (c & 1));
        }
      }
      if (!ok) {   // aborted: the products in flight finish first
        umma_commit_elect(bars + kBDrain);
        mbar_wait(bars + kBDrain, 0);
      }
    } else {
      // ---------------------------------------------- gates
      // Two warps take turns; a chunk's dt are on their way while the chunk
      // before it (of this warp) is worked on.
      ScanGates gates;
      gates.start(p, t_begin, len, head, warp - 1);
#pragma unroll 1
      for (int c = warp - 1; c < nch; c += 2) {
        const int st = c & 1;
        gates.make(c, c + 2);
        if (c >= 2 && !wait(kBGateEmpty + st, (c >> 1) - 1, kStatusMmaTimeout)) break;
        float* g = reinterpret_cast<float*>(smem + kScGate + st * kScGateStage) + lane;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          g[32 * b] = gates.step[b];
          g[kScanQ + 32 * b] = gates.end[b];
          if (b < 3) g[2 * kScanQ + 32 * b] = gates.step[b] * scan_exp2(gates.end[b]);
        }
        if (lane == 0)
          blocks[st] = make_float4(gates.block[0], gates.block[1], gates.block[2], gates.block[3]);
        arrive(kBGateFull + st);
      }
    }
  } else if (warp < 8 || warp >= 24) {
    // ------------------------------------------------ S -> M
    // The row quarter's 32 x 32 blocks up to the diagonal one: that one and every
    // second before it by the first warpgroup, the rest by the other.
    scan_set_regs<kRegsM>();
    const int top = warp < 8 ? quad : quad - 1;
    if (warp < 8) {   // blocks above the diagonal stay zero
      const uint32_t z[16] = {};
#pragma unroll 1
      for (int b = quad + 1; b < 4; ++b) tmem_st16(tmem + kTmM + 16 * b + tm_lane, z);
      tmem_wait_st();
    }
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float* g = reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage);
      const float* block = reinterpret_cast<const float*>(blocks + st);
      const float mine = g[kScanQ + row], since = block[quad] - mine;   // from the block's start
      if (!wait(kBSFull, c, kStatusMmaTimeout)) break;
      tc_fence_after();
      bool ok = true;
#pragma unroll 1
      for (int b = top; b >= 0 && ok; b -= 2) {
        float s[32];
        uint32_t m[16];
        tmem_ld32(tmem + kTmS + 32 * b + tm_lane, s);
        if (b == quad) {
          const float4* step4 = reinterpret_cast<const float4*>(g + 32 * b);
          const float4* end4 = reinterpret_cast<const float4*>(g + kScanQ + 32 * b);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 gv = step4[j], ev = end4[j];
            const float f[4] = {gv.x, gv.y, gv.z, gv.w}, end[4] = {ev.x, ev.y, ev.z, ev.w};
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)   // a select: a masked S may hold anything
              v[e] = 4 * j + e <= lane ? s[4 * j + e] * (f[e] * scan_exp2(end[e] - mine)) : 0.0f;
            m[2 * j] = pack_bf16x2(v[0], v[1]);
            m[2 * j + 1] = pack_bf16x2(v[2], v[3]);
          }
        } else {
          float after = since;   // and the blocks between
#pragma unroll 1
          for (int k = b + 1; k < quad; ++k) after += block[k];
          const float u = scan_exp2(after);
          const uint64_t u2 = pair(u, u);
          const float4* v = reinterpret_cast<const float4*>(g + 2 * kScanQ + 32 * b);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 f = v[j];
            m[2 * j] = pack_pair(mul2(mul2(pair(s[4 * j], s[4 * j + 1]), u2), pair(f.x, f.y)));
            m[2 * j + 1] = pack_pair(mul2(mul2(pair(s[4 * j + 2], s[4 * j + 3]), u2), pair(f.z, f.w)));
          }
        }
        if (b < 2) {   // the last of S is read
          tc_fence_before();
          arrive(kBSEmpty);
        }
        if (b == top && c > 0) ok = wait(kBYFull, c - 1, kStatusMmaTimeout);   // the last M is read
        if (ok) tmem_st16(tmem + kTmM + 16 * b + tm_lane, m);
      }
      // The warp without a block waits like the others: its arrival for this chunk must
      // not stand in for one of the last chunk's that is still to come.
      if (top < 0) {
        arrive(kBSEmpty);
        ok = c == 0 || wait(kBYFull, c - 1, kStatusMmaTimeout);
      }
      if (!ok) break;
      tmem_wait_st();
      tc_fence_before();
      arrive(kBMFull);
      arrive(kBGateEmpty + st);
    }
  } else if (warp < 12) {
    // ------------------------------------------------ the state
    scan_set_regs<kRegsState>();
    const bool state_row = row < N;
    uint64_t h[kScanCols / 2];
#pragma unroll
    for (int j = 0; j < kScanCols / 2; ++j) h[j] = 0ull;
    auto add_state = [&](const float* src, float log_decay) {
      const float f = scan_exp2(log_decay);
      const uint64_t f2 = pair(f, f);
#pragma unroll
      for (int j = 0; j < kScanCols / 2; ++j) {
        const float* s = src + 2 * j * N + row;
        h[j] = fma2(pair(__ldcg(s), __ldcg(s + N)), f2, h[j]);
      }
    };
    bool carried;
    const long long slot = find_state(carried);
    if (state_row) {   // the start: what the pieces before this one leave, and the carried state
      float log_decay = 0.0f;
      const long long row0 = static_cast<long long>(it.first_row) * sp.parts;
#pragma unroll 1
      for (int r = it.piece * sp.parts - 1; r >= (carried ? -1 : 0) && log_decay > kScanGone; --r) {
        const float* src = sp.seg_state + (row0 + r) * per_slot + hbase;
        if (r < 0)
          src = it.pieces > 1 && p.state == p.new_state
                    ? sp.seg_state +
                          (static_cast<long long>(sp.max_full) * sp.parts + it.first_row) * per_slot + hbase
                    : p.state + slot * per_slot + hbase;
        add_state(src, log_decay);
        if (r >= 0)
          log_decay += __ldcg(sp.seg_decay + (row0 + r) * p.heads + head);
      }
    }
    bool ok = true;
#pragma unroll 1
    for (int c = 0;; ++c) {
      const int st = c & 1;
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
      if (!(ok = wait(kBGateFull + st, c >> 1, kStatusMmaTimeout))) break;
      const float4 block = blocks[st];
      const float decay = scan_exp2((block.x + block.y) + (block.z + block.w));
      const uint64_t d2 = pair(decay, decay);
      arrive(kBGateEmpty + st);
      if (!(ok = wait(kBDsFull, c, kStatusMmaTimeout))) break;
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t d[3][16];
#pragma unroll
        for (int k = 0; k < 3; ++k) tmem_ld16(tmem + kTmDs + 64 * k + 16 * b + tm_lane, d[k]);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // the small parts first
          const uint64_t t = add2(add2(pair_bits(d[2][2 * j], d[2][2 * j + 1]),
                                       pair_bits(d[1][2 * j], d[1][2 * j + 1])),
                                  pair_bits(d[0][2 * j], d[0][2 * j + 1]));
          h[8 * b + j] = fma2(h[8 * b + j], d2, t);
        }
      }
      tc_fence_before();
      arrive(kBDsEmpty);
      if (c == nch - 1) break;
    }
    if (ok && slot >= 0 && it.piece == it.pieces - 1 && state_row) {
      float* dst = p.new_state + slot * per_slot + hbase + row;
#pragma unroll
      for (int j = 0; j < kScanCols / 2; ++j) {
        const float2 f = unpair(h[j]);
        dst[2 * j * N] = f.x;
        dst[(2 * j + 1) * N] = f.y;
      }
    }
  } else if (warp >= 16 && warp < 24) {
    // ------------------------------------------------ w X
    scan_set_regs<kRegsScale>();
    const int j0 = (warp - 16) >> 2 << 2;   // groups of eight columns
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* stage = smem + st * kScStage;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float* g = reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage);
      float after = g[kScanQ + row];
#pragma unroll 1
      for (int k = quad + 1; k < 4; ++k) after += reinterpret_cast<const float*>(blocks + st)[k];
      const float w = g[row] * scan_exp2(after);
      arrive(kBGateEmpty + st);
      if (!wait(kBFullX + st, c >> 1, kStatusTmaTimeout)) break;
      if (n < kScanQ) {   // a last, short chunk: what lies past it must not count
        if (!wait(kBFullBC + st, c >> 1, kStatusTmaTimeout)) break;
        if (row >= n) {
#pragma unroll 1
          for (int j = j0; j < j0 + 4; ++j) {
            const uint32_t off = sw128_off(row, j);
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(stage + kScX + off) = z;
#pragma unroll
            for (int b = 0; b < N / 64; ++b)
              *reinterpret_cast<uint4*>(stage + kScB + b * kScanTile + off) = z;
          }
        }
      }
      if (c > 0 && !wait(kBDsFull, c - 1, kStatusMmaTimeout)) break;   // the last w X is read
      scan_scale_row<4>(smem + kScXw, stage + kScX, row, j0, w);
      fence_proxy_async_smem();
      arrive(kBXwFull);
    }
  } else {
    // ------------------------------------------------ outputs
    scan_set_regs<kRegsOut>();
    const float D = p.D ? p.D[head] : 0.0f;
    const uint64_t D2 = pair(D, D);
#pragma unroll 1
    for (int c = 0; c < nch; ++c) {
      const int st = c & 1, n = chunk_len(c);
      uint8_t* stage = smem + st * kScStage;
      if (!wait(kBGateFull + st, c >> 1, kStatusMmaTimeout)) break;
      const float* block = reinterpret_cast<const float*>(blocks + st);
      float since = block[quad] -
                    reinterpret_cast<const float*>(smem + kScGate + st * kScGateStage)[kScanQ + row];
#pragma unroll 1
      for (int k = 0; k < quad; ++k) since += block[k];
      const float e = scan_exp2(since);
      arrive(kBGateEmpty + st);
      if (!wait(kBFullX + st, c >> 1, kStatusTmaTimeout)) break;
      uint4 x[8];   // kept here so that the stage can be refilled early
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = *reinterpret_cast<const uint4*>(stage + kScX + sw128_off(row, j));
      arrive(kBEmpty + st);
      if (!wait(kBYFull, c, kStatusMmaTimeout)) break;
      tc_fence_after();
      // 32 bytes of the thread's row at a time, whole sectors: no detour through
      // shared memory, which would hold up the stage
      const uint64_t e2 = pair(e, e);
      __nv_bfloat16* out = p.out +
          ((static_cast<long long>(t_begin) + c * kScanQ + row) * p.heads + head) * p.head_dim + col0;
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        uint32_t yd[16], yo[16];
        tmem_ld16(tmem + kTmYd + 16 * b + tm_lane, yd);
        tmem_ld16(tmem + kTmYo + 16 * b + tm_lane, yo);
        tmem_wait_ld();
        const uint32_t in[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = pack_pair(fma2(D2, unpack_pair(in[i]),
                                fma2(e2, pair_bits(yo[2 * i], yo[2 * i + 1]),
                                     pair_bits(yd[2 * i], yd[2 * i + 1]))));
        if (row < n)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + 16 * b),
                       "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]),
                       "r"(y[7])
                       : "memory");
#pragma unroll
        for (int j = 0; j < 6; ++j) x[j] = x[j + 2];
      }
      tc_fence_before();
      arrive(kBYEmpty);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.status, static_cast<unsigned int>(*abort_flag));
  asm volatile("griddepcontrol.wait;" ::: "memory");   // this grid ends after the one before it
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace gdn
