// C-ABI entry points of the operators around a recurrent block (declared in
// include/gdn_b200.h): short causal convolution, selective state space scan,
// gated norm, residual add and norm.  Host-side validation and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "gdn_b200.h"
#include "host_common.h"
#include "block_norm.cuh"
#include "short_conv.cuh"
#include "ssm_recurrent.cuh"
#include "ssm_scan.cuh"

namespace gdn {
namespace {

constexpr long long kMaxGrid = 0x7fffffffLL;

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }
int invalid(const char* msg) { return lib_fail(GDN_B200_ERR_INVALID_ARGUMENT, msg); }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GDN_B200_OK : lib_cuda_fail(e, what);
}

int element_size(int32_t dtype) {
  return dtype == GDN_B200_BF16 || dtype == GDN_B200_FP16 ? 2 : dtype == GDN_B200_FP32 ? 4 : 0;
}

// Rows of `stride` elements that 16-byte accesses can walk.
bool wide_rows(const void* p, long long stride, int size) {
  return aligned(p, 16) && stride * size % 16 == 0;
}

// Whether rows of `wa` bytes every `sa` bytes from a, and rows of wb every sb from b, span
// memory that they share.
bool spans_meet(const void* a, long long sa, long long wa, const void* b, long long sb,
                long long wb, long long rows) {
  const long long pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
  return rows > 0 && pb < pa + (rows - 1) * sa + wa && pa < pb + (rows - 1) * sb + wb;
}

// Whether any element of `rows` rows at a is one of those at b.  Rows of the same
// stride may lie side by side; with other strides it counts if the spans meet.
bool rows_overlap(const void* a, long long a_stride, const void* b, long long b_stride,
                  long long rows, long long width, int size) {
  const long long row = width * size, stride = a_stride * size;
  if (!spans_meet(a, stride, row, b, b_stride * size, row, rows)) return false;
  if (rows == 1 || a_stride != b_stride) return true;
  // b's row i starts `into` bytes after the start of a's row i + by
  const long long delta = reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a);
  const long long by = delta >= 0 ? delta / stride : -((stride - 1 - delta) / stride);
  const long long into = delta - by * stride;
  return (into < row && by < rows && -by < rows) ||
         (stride - into < row && by + 1 < rows && -by - 1 < rows);
}

// ------------------------------------------------------------ short convolution
template <typename T, int V, int W>
void launch_conv(const ConvParams& p, unsigned grid, bool step, cudaStream_t st) {
  const size_t smem =
      V > 1 ? 128 + static_cast<size_t>(p.tile + 2 * W - 3) * kConvThreads * V * sizeof(T) : 0;
  if (step) gdn_short_conv_step_kernel<T, V, W><<<grid, kConvThreads, 0, st>>>(p);
  else gdn_short_conv_kernel<T, V, W><<<grid, kConvThreads, smem, st>>>(p);
}

template <typename T, int V>
void launch_conv_width(const ConvParams& p, int width, unsigned grid, bool step, cudaStream_t st) {
  if (width == 2) launch_conv<T, V, 2>(p, grid, step, st);
  else if (width == 3) launch_conv<T, V, 3>(p, grid, step, st);
  else launch_conv<T, V, 4>(p, grid, step, st);
}

// Tokens of a block: long ones re-read fewer rows before their first (W - 1 each)
// and load their taps less often; short ones spread a small call over the SMs.
// 24 KiB of rows a block (8192 tokens of 8192 channels: 48 us; 51 with 16 KiB, 53
// with 32, 57 with 40).
constexpr int kConvTileBytes = 24 << 10, kConvTileShort = 16;
constexpr long long kConvFewBlocks = 148 * 6;

template <typename T>
int launch_conv_type(ConvParams& p, int width, bool step, cudaStream_t st) {
  // 16-byte copies of rows, four channels a thread, else one channel
  constexpr int size = static_cast<int>(sizeof(T));
  const bool wide = p.channels % kLanes<T> == 0 && wide_rows(p.x, p.x_stride, size) &&
                    wide_rows(p.out, p.out_stride, size) && aligned(p.weight, 16) &&
                    aligned(p.bias, 16) && aligned(p.state, 16) && aligned(p.new_state, 16);
  const int per_block = kConvThreads * (wide ? kConvVec : 1);
  p.chan_blocks = (p.channels + per_block - 1) / per_block;
  long long n = p.tokens;   // rows of a step
  if (!step) {
    p.tile = kConvTileBytes / (kConvThreads * kConvVec * size);
    if ((p.tokens / p.tile + 1) * p.chan_blocks < kConvFewBlocks) p.tile = kConvTileShort;
    n = std::max<long long>(1, (p.tokens + p.tile - 1) / p.tile);
  }
  const long long blocks = step ? n : n + p.seqs;
  if (blocks > kMaxGrid / p.chan_blocks) return invalid("tokens * channels exceeds the grid limit");
  const unsigned grid = static_cast<unsigned>(blocks * p.chan_blocks);
  p.tile_blocks = static_cast<unsigned>(n * p.chan_blocks);
  p.lookup_first = p.tokens <= 2LL * kConvShort * p.seqs;
  if (wide) launch_conv_width<T, kConvVec>(p, width, grid, step, st);
  else launch_conv_width<T, 1>(p, width, grid, step, st);
  return launched("short convolution launch");
}

int conv_call(ConvParams& p, int width, int32_t dtype, bool step, void* stream) {
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_B200_BF16) return launch_conv_type<__nv_bfloat16>(p, width, step, st);
  if (dtype == GDN_B200_FP16) return launch_conv_type<__half>(p, width, step, st);
  return launch_conv_type<float>(p, width, step, st);
}

int check_conv(int64_t rows, int64_t pool, int32_t channels, int32_t width, int32_t dtype,
               int32_t activation) {
  if (!element_size(dtype)) return invalid("dtype must be GDN_B200_BF16, _FP16 or _FP32");
  if (activation != GDN_B200_ACT_NONE && activation != GDN_B200_ACT_SILU)
    return invalid("activation must be GDN_B200_ACT_NONE or _SILU");
  if (width < 2 || width > 4) return invalid("width must be 2, 3 or 4");
  if (channels < 1 || channels > (1 << 24)) return invalid("channels must be in [1, 2^24]");
  if (rows < 0 || pool < 0) return invalid("extents must be >= 0");
  return GDN_B200_OK;
}

// ------------------------------------------------------------ norms
// Threads of a block that is one team: whole warps, as many as the vectors need.
unsigned team_threads(int nv, int vecs) { return static_cast<unsigned>((nv + 32 * vecs - 1) / (32 * vecs) * 32); }

template <typename T, int kTeam, int kVecs>
void launch_gated(const NormParams& p, long long groups, cudaStream_t st) {
  constexpr int per_block = kTeam > 0 ? kNormThreads / (kTeam > 0 ? kTeam : 1) : 1;
  gdn_gated_norm_kernel<T, kLanes<T>, kTeam, kVecs>
      <<<static_cast<unsigned>((groups + per_block - 1) / per_block),
         kTeam > 0 ? kNormThreads : team_threads(p.group / kLanes<T>, kVecs), 0, st>>>(p);
}

template <typename T>
int gated_call(const NormParams& p, cudaStream_t st) {
  const long long groups = p.rows * (p.width / p.group);
  if (groups > kMaxGrid) return invalid("rows * groups exceeds the grid limit");
  const int size = static_cast<int>(sizeof(T));
  const bool wide = p.group % kLanes<T> == 0 && wide_rows(p.x, p.x_stride, size) &&
                    (!p.gate || wide_rows(p.gate, p.gate_stride, size)) &&
                    wide_rows(p.out, p.out_stride, size) && aligned(p.weight, 16);
  // A vector of each operand per thread up to 512 threads: more per thread was
  // slower (2048 wide: 35 us with one, 40 with four, 48 with eight), as fewer warps
  // then hide the sum.
  const int nv = p.group / kLanes<T>;
  if (!wide || nv > 4096) gdn_gated_norm_any_kernel<T><<<static_cast<unsigned>(groups), 256, 0, st>>>(p);
  else if (nv <= 8) launch_gated<T, 8, 1>(p, groups, st);
  else if (nv <= 16) launch_gated<T, 16, 1>(p, groups, st);
  else if (nv <= 32) launch_gated<T, 32, 1>(p, groups, st);
  else if (nv <= 512) launch_gated<T, 0, 1>(p, groups, st);
  else if (nv <= 2048) launch_gated<T, 0, 2>(p, groups, st);
  else launch_gated<T, 0, 4>(p, groups, st);
  return launched("gated norm launch");
}

template <typename T, typename R, int kTeam, int kVecs>
void launch_add(const NormParams& p, cudaStream_t st) {
  constexpr int per_block = kTeam > 0 ? kNormThreads / (kTeam > 0 ? kTeam : 1) : 1;
  gdn_add_norm_kernel<T, R, kLanes<T>, kTeam, kVecs>
      <<<static_cast<unsigned>((p.rows + per_block - 1) / per_block),
         kTeam > 0 ? kNormThreads : team_threads(p.width / kLanes<T>, kVecs), 0, st>>>(p);
}

template <typename T, typename R>
int add_call(const NormParams& p, cudaStream_t st) {
  if (p.rows > kMaxGrid) return invalid("rows exceeds the grid limit");
  const int size = static_cast<int>(sizeof(T)), rsize = static_cast<int>(sizeof(R));
  const bool wide = p.width % kLanes<T> == 0 && wide_rows(p.x, p.x_stride, size) &&
                    wide_rows(p.out, p.out_stride, size) &&
                    wide_rows(p.residual, p.residual_stride, rsize) &&
                    wide_rows(p.new_residual, p.new_residual_stride, rsize) &&
                    aligned(p.weight, 16) && aligned(p.block_weight, 16) &&
                    aligned(p.channel_scale, 16);
  const int nv = p.width / kLanes<T>;
  if (!wide || nv > 4096) gdn_add_norm_any_kernel<T, R><<<static_cast<unsigned>(p.rows), 256, 0, st>>>(p);
  else if (nv <= 32) launch_add<T, R, 32, 1>(p, st);
  else if (nv <= 512) launch_add<T, R, 0, 1>(p, st);
  else if (nv <= 2048) launch_add<T, R, 0, 2>(p, st);
  else launch_add<T, R, 0, 4>(p, st);
  return launched("add norm launch");
}

// ------------------------------------------------------------ selective scan
int check_ssm(int64_t rows, int64_t pool, int32_t heads, int32_t groups, int32_t head_dim,
              int32_t state_dim) {
  if (head_dim != 64 && head_dim != 128) return invalid("head_dim must be 64 or 128");
  if (state_dim != 64 && state_dim != 128) return invalid("state_dim must be 64 or 128");
  if (heads < 1 || groups < 1 || heads % groups != 0)
    return invalid("num_heads must be a positive multiple of num_groups");
  if (heads > 65535) return invalid("num_heads exceeds 65535");
  if (rows < 0 || pool < 0) return invalid("extents must be >= 0");
  return GDN_B200_OK;
}

int check_ssm_rows(const SsmParams& p) {
  if (!p.x || !p.dt || !p.B || !p.C || !p.A_log || !p.out) return invalid("null pointer argument");
  if (!wide_rows(p.x, p.x_stride, 2) || !wide_rows(p.B, p.b_stride, 2) ||
      !wide_rows(p.C, p.c_stride, 2) || !aligned(p.out, 16))
    return invalid("x, B, C and output need 16-byte aligned rows");
  return GDN_B200_OK;
}

template <bool kPrompt>
int ssm_recurrent_call(const SsmParams& p, int32_t state_dim, int64_t entries, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.heads * (p.head_dim / kSsmBlockRows)),
                  static_cast<unsigned>(entries));
  if (state_dim == 64) gdn_ssm_recurrent_kernel<64, kPrompt><<<grid, kSsmThreads, 0, st>>>(p);
  else gdn_ssm_recurrent_kernel<128, kPrompt><<<grid, kSsmThreads, 0, st>>>(p);
  return launched("selective scan launch");
}

// Prompts of up to so many tokens on average (and calls without tokens) run token by
// token: a chunk costs the same however few tokens it has.  The average decides for
// the whole call, as lengths are on the device: one long prompt beside many short
// ones may run token by token too.  Sequences of equal lengths, 64 heads of 64, state
// 128, token by token / in chunks: 1 x 8 tokens 7.2 / 8.5 us, 1 x 16 11.5 / 8.4,
// 8 x 8 16 / 31, 8 x 24 38 / 31, 64 x 4 77 / 204, 64 x 16 180 / 205, 64 x 24 240 / 205.
constexpr int kScanShort = 10;

// The scan kernels' shared memory is above the default limit: raised once per
// device.
std::mutex g_scan_mu;
bool g_scan_ready[64];

int scan_setup() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return lib_cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return lib_fail(GDN_B200_ERR_CUDA, "device index out of range");
  std::lock_guard<std::mutex> lock(g_scan_mu);
  if (g_scan_ready[dev]) return GDN_B200_OK;
  for (auto fn : {gdn_ssm_scan_kernel<64>, gdn_ssm_scan_kernel<128>}) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kScanSmem));
    if (e != cudaSuccess) return lib_cuda_fail(e, "cudaFuncSetAttribute(scan smem)");
  }
  for (auto fn : {gdn_ssm_piece_state_kernel<64>, gdn_ssm_piece_state_kernel<128>}) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kStateSmem));
    if (e != cudaSuccess) return lib_cuda_fail(e, "cudaFuncSetAttribute(piece state smem)");
  }
  g_scan_ready[dev] = true;
  return GDN_B200_OK;
}

// How a call's sequences are divided.  A CTA runs 64 columns of a head, one per
// SM; its start costs about as much as two or three chunks.
//  * One sequence: as many equal pieces as fill the SMs once, of two chunks at
//    least.  8,192 tokens of 64 heads run in two pieces; five pieces, with their
//    start-ups, took longer.  1,024 tokens of 8 heads take 14 us in pieces of two
//    chunks, 18 of four, 20 of eight.
//  * Several: a piece is an SM's share of all chunks, so that a sequence that is
//    longer than that cannot hold up the rest, and most are not divided.  Where
//    whole sequences fill half of the SMs, of six chunks at least, as a piece of one
//    or two left over costs a start (4 sequences of 700 tokens: 32 heads, 21 us whole
//    and 31 divided; 8 heads, 19 whole and 16 divided).
// The states of long pieces are made in parts that fill the SMs likewise; in short
// ones a part's start and its sum cost more (32 heads, sequences of 1400, 100 and
// 50 tokens: 22 us with one part, 31 with four).
constexpr int kScanSms = 148, kScanMinPiece = 2, kScanMinPieceFilled = 6;
constexpr int kScanMaxDivided = 1024, kScanPartedPiece = 16, kScanMaxParts = 4;

struct ScanPlan {
  int seg_chunks;        // 0: not divided
  int parts;
  long long max_full;    // bound on the whole pieces
  size_t state_bytes, bytes;
};

ScanPlan scan_plan(long long seqs, long long tokens, int heads, int head_dim, int state_dim) {
  ScanPlan plan{};
  plan.parts = 1;
  const long long chunks = (tokens + kScanQ - 1) / kScanQ;
  const long long units = static_cast<long long>(heads) * (head_dim / kScanCols);
  if (seqs > kScanMaxDivided || seqs * units >= 8 * kScanSms) return plan;
  long long piece = (chunks * units + kScanSms - 1) / kScanSms;
  if (seqs == 1) {
    const long long pieces = std::max<long long>(1, kScanSms / units);
    piece = (chunks + pieces - 1) / pieces;
  }
  const bool filled = seqs > 1 && seqs * units * 2 > kScanSms;
  piece = std::max<long long>(piece, filled ? kScanMinPieceFilled : kScanMinPiece);
  if (chunks <= piece) return plan;
  const long long whole = seqs == 1 ? (chunks - 1) / piece : 1;   // pieces whose states are needed
  if (piece >= kScanPartedPiece)
    plan.parts = static_cast<int>(
        std::min<long long>(kScanMaxParts, std::max<long long>(1, kScanSms / (units * whole))));
  piece = (piece + plan.parts - 1) / plan.parts * plan.parts;
  plan.seg_chunks = static_cast<int>(piece);
  plan.max_full = (chunks + seqs) / piece;
  const size_t row = static_cast<size_t>(heads) * head_dim * state_dim * 4;
  plan.state_bytes = plan.max_full * (plan.parts + 1) * row;
  plan.bytes = plan.state_bytes + plan.max_full * plan.parts * heads * 4;
  return plan;
}

int ssm_scan_call(const SsmParams& p, int32_t state_dim, int64_t seqs, void* workspace,
                  uint64_t workspace_bytes, cudaStream_t st) {
  if (int rc = scan_setup()) return rc;
  ScanPlan plan = scan_plan(seqs, p.tokens, p.heads, p.head_dim, state_dim);
  if (!workspace || workspace_bytes < plan.bytes || plan.max_full * plan.parts + seqs > 65535)
    plan = ScanPlan{0, 1, 0, 0, 0};
  CUtensorMap tx, tb, tc;
  if (int rc = lib_token_map(&tx, p.x, p.head_dim, p.heads, p.tokens, p.x_stride, kScanQ)) return rc;
  if (int rc = lib_token_map(&tb, p.B, state_dim, p.groups, p.tokens, p.b_stride, kScanQ)) return rc;
  if (int rc = lib_token_map(&tc, p.C, state_dim, p.groups, p.tokens, p.c_stride, kScanQ)) return rc;
  ScanParams sp{};
  sp.s = p;
  sp.seg_chunks = plan.seg_chunks;
  sp.parts = plan.parts;
  sp.max_full = static_cast<int>(plan.max_full);
  sp.seg_state = static_cast<float*>(workspace);
  sp.seg_decay = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.state_bytes);
  const unsigned units = static_cast<unsigned>(p.heads * (p.head_dim / kScanCols));
  if (plan.max_full > 0) {
    const dim3 pieces(units, static_cast<unsigned>(plan.max_full * plan.parts));
    if (state_dim == 64)
      gdn_ssm_piece_state_kernel<64><<<pieces, kStateThreads, kStateSmem, st>>>(tx, tb, sp);
    else
      gdn_ssm_piece_state_kernel<128><<<pieces, kStateThreads, kStateSmem, st>>>(tx, tb, sp);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units, static_cast<unsigned>(plan.max_full + seqs));
  cfg.blockDim = dim3(kScanThreads);
  cfg.dynamicSmemBytes = kScanSmem;
  cfg.stream = st;
  cudaLaunchAttribute beside[1];
  beside[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = beside;
  cfg.numAttrs = plan.max_full > 0 ? 1 : 0;   // after the kernel of the pieces only
  const cudaError_t e =
      state_dim == 64 ? cudaLaunchKernelEx(&cfg, gdn_ssm_scan_kernel<64>, tx, tb, tc, sp)
                      : cudaLaunchKernelEx(&cfg, gdn_ssm_scan_kernel<128>, tx, tb, tc, sp);
  if (e != cudaSuccess) return lib_cuda_fail(e, "selective scan launch");
  return launched("selective scan launch");
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_b200_short_conv(const void* x, int64_t x_stride, const void* weight,
                                   const void* bias, const void* state, const void* cu_seqlens,
                                   int32_t cu_seqlens_is_int64, const void* state_indices,
                                   int32_t indices_are_int64, const uint8_t* has_state,
                                   int32_t activation, void* output, int64_t output_stride,
                                   void* new_state, int64_t num_seqs, int64_t total_tokens,
                                   int64_t pool_size, int32_t channels, int32_t width,
                                   int32_t dtype, void* stream) {
  lib_clear_error();
  if (int rc = check_conv(total_tokens, pool_size, channels, width, dtype, activation)) return rc;
  if (num_seqs < 0 || num_seqs > kMaxGrid) return invalid("num_seqs must be in [0, 2^31)");
  if (total_tokens > (1LL << 30)) return invalid("total_tokens exceeds 2^30");
  if (num_seqs == 0) return GDN_B200_OK;
  if (!weight || !cu_seqlens || !new_state || (total_tokens > 0 && (!x || !output)))
    return invalid("null pointer argument");
  if (total_tokens > 1 && (x_stride < channels || output_stride < channels))
    return invalid("rows must not overlap");
  // blocks read rows that are others' to write
  if (rows_overlap(x, x_stride, output, output_stride, total_tokens, channels, element_size(dtype)))
    return invalid("output must not overlap x");
  if (!state_indices && pool_size < num_seqs)
    return invalid("the states hold fewer rows than there are sequences");
  if (!aligned(cu_seqlens, cu_seqlens_is_int64 ? 8 : 4) ||
      !aligned(state_indices, indices_are_int64 ? 8 : 4))
    return invalid("cu_seqlens or state_indices is misaligned");
  ConvParams p{};
  int sms = 0;
  if (int rc = lib_device(&p.status, &sms)) return rc;
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.state = state;
  p.new_state = new_state;
  p.out = output;
  p.cu = cu_seqlens;
  p.slots = state_indices;
  p.has_state = has_state;
  p.x_stride = x_stride;
  p.out_stride = output_stride;
  p.pool = pool_size;
  p.tokens = total_tokens;
  p.cu_is64 = cu_seqlens_is_int64 ? 1 : 0;
  p.slots_is64 = indices_are_int64 ? 1 : 0;
  p.seqs = static_cast<int>(num_seqs);
  p.channels = channels;
  p.silu = activation == GDN_B200_ACT_SILU;
  return conv_call(p, width, dtype, false, stream);
}

extern "C" int gdn_b200_short_conv_step(const void* x, int64_t x_stride, const void* weight,
                                        const void* bias, const void* state_pool,
                                        const void* state_indices, int32_t indices_are_int64,
                                        int32_t activation, void* output, int64_t output_stride,
                                        void* new_state_pool, int64_t batch, int64_t pool_size,
                                        int32_t channels, int32_t width, int32_t dtype,
                                        void* stream) {
  lib_clear_error();
  if (int rc = check_conv(batch, pool_size, channels, width, dtype, activation)) return rc;
  if (batch == 0) return GDN_B200_OK;
  if (!x || !weight || !state_pool || !new_state_pool || !output)
    return invalid("null pointer argument");
  if (batch > 1 && (x_stride < channels || output_stride < channels))
    return invalid("rows must not overlap");
  if (!state_indices && pool_size < batch)
    return invalid("the states hold fewer rows than there are batch entries");
  if (!aligned(state_indices, indices_are_int64 ? 8 : 4))
    return invalid("state_indices is misaligned");
  ConvParams p{};
  int sms = 0;
  if (int rc = lib_device(&p.status, &sms)) return rc;
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.state = state_pool;
  p.new_state = new_state_pool;
  p.out = output;
  p.slots = state_indices;
  p.x_stride = x_stride;
  p.out_stride = output_stride;
  p.pool = pool_size;
  p.tokens = batch;
  p.slots_is64 = indices_are_int64 ? 1 : 0;
  p.channels = channels;
  p.silu = activation == GDN_B200_ACT_SILU;
  return conv_call(p, width, dtype, true, stream);
}

extern "C" uint64_t gdn_b200_ssm_prefill_workspace_size(int64_t num_seqs, int64_t total_tokens,
                                                        int32_t num_heads, int32_t head_dim,
                                                        int32_t state_dim) {
  // sizes that gdn_b200_ssm_prefill refuses need nothing (and have no plan: a head of
  // less than kScanCols columns is no unit)
  if (num_seqs <= 0 || num_seqs > 65535 || total_tokens <= 0 || total_tokens > kMaxGrid - kScanQ ||
      num_heads <= 0 || num_heads > 65535 || (head_dim != 64 && head_dim != 128) ||
      (state_dim != 64 && state_dim != 128))
    return 0;
  return scan_plan(num_seqs, total_tokens, num_heads, head_dim, state_dim).bytes;
}

extern "C" int gdn_b200_ssm_prefill(const void* x, int64_t x_stride, const void* dt,
                                    int64_t dt_stride, const float* A_log, const void* B,
                                    int64_t b_stride, const void* C, int64_t c_stride,
                                    const float* D, const float* dt_bias, const float* state,
                                    const void* cu_seqlens, int32_t cu_seqlens_is_int64,
                                    const void* state_indices, int32_t indices_are_int64,
                                    const uint8_t* has_state, void* output, float* new_state,
                                    int64_t num_seqs, int64_t total_tokens, int64_t pool_size,
                                    int32_t num_heads, int32_t num_groups, int32_t head_dim,
                                    int32_t state_dim, void* workspace, uint64_t workspace_bytes,
                                    void* stream) {
  lib_clear_error();
  if (int rc = check_ssm(total_tokens, pool_size, num_heads, num_groups, head_dim, state_dim))
    return rc;
  if (num_seqs < 0 || num_seqs > 65535) return invalid("num_seqs must be in [0, 65535]");
  if (total_tokens > kMaxGrid - kScanQ) return invalid("total_tokens exceeds the int32 range");
  if (num_seqs == 0) return GDN_B200_OK;
  if (!cu_seqlens || !new_state) return invalid("null pointer argument");
  if (!state_indices && pool_size < num_seqs)
    return invalid("the states hold fewer rows than there are sequences");
  if (!aligned(cu_seqlens, cu_seqlens_is_int64 ? 8 : 4) ||
      !aligned(state_indices, indices_are_int64 ? 8 : 4))
    return invalid("cu_seqlens or state_indices is misaligned");
  if (!aligned(workspace, 256)) return invalid("workspace needs 256-byte alignment");
  if (!aligned(state, 16) || !aligned(new_state, 16))
    return invalid("state and new_state need 16-byte alignment");
  SsmParams p{};
  int sms = 0;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.dt = static_cast<const __nv_bfloat16*>(dt);
  p.B = static_cast<const __nv_bfloat16*>(B);
  p.C = static_cast<const __nv_bfloat16*>(C);
  p.A_log = A_log;
  p.D = D;
  p.dt_bias = dt_bias;
  p.state = state;
  p.new_state = new_state;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.cu = cu_seqlens;
  p.slots = state_indices;
  p.has_state = has_state;
  p.x_stride = x_stride;
  p.dt_stride = dt_stride;
  p.b_stride = b_stride;
  p.c_stride = c_stride;
  p.pool = pool_size;
  p.tokens = total_tokens;
  p.cu_is64 = cu_seqlens_is_int64 ? 1 : 0;
  p.slots_is64 = indices_are_int64 ? 1 : 0;
  p.seqs = static_cast<int>(num_seqs);
  p.heads = num_heads;
  p.groups = num_groups;
  p.head_dim = head_dim;
  if (!A_log) return invalid("null pointer argument");
  if (total_tokens > 0) {
    if (int rc = check_ssm_rows(p)) return rc;
    if (!aligned(output, 32)) return invalid("output needs 32-byte alignment");
    // pieces of a sequence run side by side, and read tokens that others may have written
    const long long row = 2LL * num_heads * head_dim, group_row = 2LL * num_groups * state_dim;
    if (spans_meet(x, 2 * x_stride, row, output, row, row, total_tokens) ||
        spans_meet(B, 2 * b_stride, group_row, output, row, row, total_tokens) ||
        spans_meet(C, 2 * c_stride, group_row, output, row, row, total_tokens))
      return invalid("output must not overlap x, B or C");
  }
  if (int rc = lib_device(&p.status, &sms)) return rc;
  if (total_tokens <= kScanShort * num_seqs)
    return ssm_recurrent_call<true>(p, state_dim, num_seqs, static_cast<cudaStream_t>(stream));
  return ssm_scan_call(p, state_dim, num_seqs, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream));
}

extern "C" int gdn_b200_ssm_step(const void* x, int64_t x_stride, const void* dt,
                                 int64_t dt_stride, const float* A_log, const void* B,
                                 int64_t b_stride, const void* C, int64_t c_stride, const float* D,
                                 const float* dt_bias, const float* state_pool,
                                 const void* read_indices, const void* write_indices,
                                 int32_t indices_are_int64, void* output, float* new_state_pool,
                                 int64_t batch, int64_t pool_size, int32_t num_heads,
                                 int32_t num_groups, int32_t head_dim, int32_t state_dim,
                                 void* stream) {
  lib_clear_error();
  if (int rc = check_ssm(batch, pool_size, num_heads, num_groups, head_dim, state_dim)) return rc;
  if (batch > 65535) return invalid("batch exceeds 65535");
  if (batch == 0) return GDN_B200_OK;
  if (!state_pool || !new_state_pool) return invalid("null pointer argument");
  if (!read_indices && pool_size < batch)
    return invalid("the states hold fewer rows than there are batch entries");
  if (!read_indices && write_indices) return invalid("write_indices need read_indices");
  if (!aligned(read_indices, indices_are_int64 ? 8 : 4) ||
      !aligned(write_indices, indices_are_int64 ? 8 : 4))
    return invalid("state indices are misaligned");
  if (!aligned(state_pool, 16) || !aligned(new_state_pool, 16))
    return invalid("the state pools need 16-byte alignment");
  SsmParams p{};
  int sms = 0;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.dt = static_cast<const __nv_bfloat16*>(dt);
  p.B = static_cast<const __nv_bfloat16*>(B);
  p.C = static_cast<const __nv_bfloat16*>(C);
  p.A_log = A_log;
  p.D = D;
  p.dt_bias = dt_bias;
  p.state = state_pool;
  p.new_state = new_state_pool;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.slots = read_indices;
  p.write_slots = write_indices;
  p.x_stride = x_stride;
  p.dt_stride = dt_stride;
  p.b_stride = b_stride;
  p.c_stride = c_stride;
  p.pool = pool_size;
  p.tokens = batch;
  p.slots_is64 = indices_are_int64 ? 1 : 0;
  p.heads = num_heads;
  p.groups = num_groups;
  p.head_dim = head_dim;
  if (int rc = check_ssm_rows(p)) return rc;
  if (int rc = lib_device(&p.status, &sms)) return rc;
  return ssm_recurrent_call<false>(p, state_dim, batch, static_cast<cudaStream_t>(stream));
}

extern "C" int gdn_b200_gated_norm(const void* x, int64_t x_stride, const void* gate,
                                   int64_t gate_stride, const void* weight,
                                   int32_t weight_is_shared, void* output, int64_t output_stride,
                                   int64_t rows, int32_t width, int32_t group_size, double eps,
                                   int32_t activation, int32_t norm_first, int32_t dtype,
                                   void* stream) {
  lib_clear_error();
  if (!element_size(dtype)) return invalid("dtype must be GDN_B200_BF16, _FP16 or _FP32");
  if (rows < 0 || width < 1 || group_size < 1 || width % group_size != 0)
    return invalid("width must be a positive multiple of group_size");
  if (activation != GDN_B200_ACT_SILU && activation != GDN_B200_ACT_SIGMOID)
    return invalid("activation must be GDN_B200_ACT_SILU or _SIGMOID");
  if (!(eps >= 0.0)) return invalid("eps must be >= 0");
  if (rows == 0) return GDN_B200_OK;
  if (!x || !output) return invalid("null pointer argument");
  if (rows > 1 && (x_stride < width || output_stride < width || (gate && gate_stride < width)))
    return invalid("rows must not overlap");
  NormParams p{};
  p.x = x;
  p.gate = gate;
  p.weight = weight;
  p.weight_shared = weight_is_shared ? 1 : 0;
  p.out = output;
  p.rows = rows;
  p.x_stride = x_stride;
  p.gate_stride = gate_stride;
  p.out_stride = output_stride;
  p.width = width;
  p.group = group_size;
  p.per_row = static_cast<unsigned>(width / group_size);
  p.inv_group = static_cast<float>(1.0 / group_size);
  p.silu = activation == GDN_B200_ACT_SILU;
  p.norm_first = norm_first ? 1 : 0;
  p.eps = static_cast<float>(eps);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_B200_BF16) return gated_call<__nv_bfloat16>(p, st);
  if (dtype == GDN_B200_FP16) return gated_call<__half>(p, st);
  return gated_call<float>(p, st);
}

extern "C" int gdn_b200_add_norm(const void* x, int64_t x_stride, const void* residual,
                                 int64_t residual_stride, const void* weight,
                                 const void* block_weight, const float* channel_scale,
                                 double scale, void* output, int64_t output_stride,
                                 void* new_residual, int64_t new_residual_stride, int64_t rows,
                                 int32_t width, double eps, double weight_offset, int32_t dtype,
                                 int32_t residual_is_fp32, void* stream) {
  lib_clear_error();
  if (!element_size(dtype)) return invalid("dtype must be GDN_B200_BF16, _FP16 or _FP32");
  if (rows < 0 || width < 1) return invalid("rows must be >= 0 and width >= 1");
  if (!(eps >= 0.0)) return invalid("eps must be >= 0");
  if (rows == 0) return GDN_B200_OK;
  if (!x || !residual || !weight || !output || !new_residual)
    return invalid("null pointer argument");
  if (rows > 1 && (x_stride < width || residual_stride < width || output_stride < width ||
                   new_residual_stride < width))
    return invalid("rows must not overlap");
  NormParams p{};
  p.x = x;
  p.residual = residual;
  p.weight = weight;
  p.block_weight = block_weight;
  p.channel_scale = channel_scale;
  p.out = output;
  p.new_residual = new_residual;
  p.rows = rows;
  p.x_stride = x_stride;
  p.residual_stride = residual_stride;
  p.out_stride = output_stride;
  p.new_residual_stride = new_residual_stride;
  p.width = width;
  p.inv_width = static_cast<float>(1.0 / width);
  p.eps = static_cast<float>(eps);
  p.scale = static_cast<float>(scale);
  p.weight_offset = static_cast<float>(weight_offset);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == GDN_B200_FP32) return add_call<float, float>(p, st);
  if (dtype == GDN_B200_BF16)
    return residual_is_fp32 ? add_call<__nv_bfloat16, float>(p, st)
                            : add_call<__nv_bfloat16, __nv_bfloat16>(p, st);
  return residual_is_fp32 ? add_call<__half, float>(p, st) : add_call<__half, __half>(p, st);
}
