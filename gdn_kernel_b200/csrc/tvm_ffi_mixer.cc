// TVM-FFI exports of the mixer operators: what gdn_kernel_b200.mixer calls.  Each
// checks types, shapes, layouts and devices (raising ValueError), then makes one
// C call on the stream that the host framework has current.
#include "tvm_ffi_common.h"

#include <initializer_list>

namespace gdn_tvm {

using tvm::ffi::Optional;

struct DType {
  uint8_t code, bits;
};
constexpr DType kBf16{kDLBfloat, 16}, kFp32{kDLFloat, 32};

DType dtype_of(const TensorView& t) { return DType{t.dtype().code, t.dtype().bits}; }

// bfloat16, float16 or float32 as the C ABI's code.
int32_t element_code(const TensorView& t, const char* name) {
  if (is_dtype(t, kDLBfloat, 16)) return GDN_B200_BF16;
  if (is_dtype(t, kDLFloat, 16)) return GDN_B200_FP16;
  if (is_dtype(t, kDLFloat, 32)) return GDN_B200_FP32;
  TVM_FFI_THROW(ValueError) << name << ": expected bfloat16, float16 or float32";
  return 0;
}

[[noreturn]] void refuse(const char* name, const char* what) {
  TVM_FFI_THROW(ValueError) << name << ": " << what;
  std::abort();   // not reached
}

[[noreturn]] void refuse_shape(const TensorView& t, const char* name,
                               std::initializer_list<int64_t> shape) {
  std::string want, got;
  for (int64_t s : shape) want += (want.empty() ? "" : ", ") + std::to_string(s);
  for (int32_t i = 0; i < t.ndim(); ++i)
    got += (got.empty() ? "" : ", ") + std::to_string(t.size(i));
  TVM_FFI_THROW(ValueError) << name << ": expected shape (" << want << "), got (" << got << ")";
  std::abort();   // not reached
}

void check_common(const TensorView& t, const char* name, DType type,
                  std::initializer_list<int64_t> shape, const DLDevice& dev) {
  if (!is_dtype(t, type.code, type.bits)) refuse(name, "wrong dtype");
  bool same = t.ndim() == static_cast<int32_t>(shape.size());
  int32_t i = 0;
  if (same)
    for (int64_t s : shape) same &= t.size(i++) == s;
  if (!same) refuse_shape(t, name, shape);
  if (t.device().device_type != dev.device_type || t.device().device_id != dev.device_id)
    refuse(name, "must be on the same device as x");
}

// A contiguous tensor of this type and shape.
void* full(const TensorView& t, const char* name, DType type, std::initializer_list<int64_t> shape,
           const DLDevice& dev) {
  check_common(t, name, type, shape, dev);
  if (t.numel() != 0 && !t.IsContiguous()) refuse(name, "must be contiguous");
  return ptr(t);
}
void* full(const Optional<TensorView>& t, const char* name, DType type,
           std::initializer_list<int64_t> shape, const DLDevice& dev) {
  return t.has_value() ? full(t.value(), name, type, shape, dev) : nullptr;
}

// [rows, ...] whose rows are each contiguous, and the stride between rows.
struct Rows {
  void* p;
  int64_t stride;
};
Rows rows(const TensorView& t, const char* name, DType type, std::initializer_list<int64_t> shape,
          const DLDevice& dev) {
  check_common(t, name, type, shape, dev);
  int64_t want = 1;
  for (int32_t i = t.ndim() - 1; i > 0; --i) {
    if (t.size(i) != 1 && t.stride(i) != want && t.numel() != 0)
      refuse(name, "must be contiguous within a row");
    want *= t.size(i);
  }
  return Rows{ptr(t), t.size(0) > 1 ? t.stride(0) : want};
}

struct Index {
  void* p;
  int32_t is64;
};
Index index(const TensorView& t, const char* name, int64_t n, const DLDevice& dev) {
  const bool is64 = is_dtype(t, kDLInt, 64);
  if (!is64 && !is_dtype(t, kDLInt, 32)) refuse(name, "must be int32 or int64");
  return Index{full(t, name, dtype_of(t), {n}, dev), is64 ? 1 : 0};
}
Index index(const Optional<TensorView>& t, const char* name, int64_t n, const DLDevice& dev) {
  return t.has_value() ? index(t.value(), name, n, dev) : Index{nullptr, 0};
}

const uint8_t* flags(const Optional<TensorView>& t, int64_t n, const DLDevice& dev) {
  if (!t.has_value()) return nullptr;
  const TensorView& f = t.value();
  if (!is_dtype(f, kDLBool, 8) && !is_dtype(f, kDLUInt, 8))
    refuse("has_state", "must be bool or uint8");
  return static_cast<const uint8_t*>(full(f, "has_state", dtype_of(f), {n}, dev));
}

int64_t sequences(const TensorView& cu) {
  if (cu.ndim() != 1 || cu.size(0) < 1) refuse("cu_seqlens", "must be [N + 1]");
  return cu.size(0) - 1;
}

void need_slots(int64_t pool, int64_t n, const Index& slots) {
  if (slots.p == nullptr && n > 0 && pool < n)
    TVM_FFI_THROW(ValueError) << "the states hold " << pool << " rows, " << n << " are needed";
}

DLDevice cuda_device(const TensorView& x) {
  if (x.device().device_type != kDLCUDA) refuse("x", "must be a CUDA tensor");
  return x.device();
}

const float* f32(const void* p) { return static_cast<const float*>(p); }

// ------------------------------------------------------------ short convolution
void check_weight(const TensorView& x, const TensorView& weight) {
  if (x.ndim() != 2) refuse("x", "must have two dimensions");
  if (weight.ndim() != 2) refuse("weight", "must be [channels, width]");
  if (weight.size(1) < 2 || weight.size(1) > 4) refuse("weight", "width must be 2, 3 or 4");
}

void ShortConv(TensorView x, TensorView weight, Optional<TensorView> bias,
               Optional<TensorView> state, TensorView cu, TensorView output, TensorView new_state,
               Optional<TensorView> state_indices, Optional<TensorView> has_state,
               int64_t activation) {
  const int32_t code = element_code(x, "x");
  const DType type = dtype_of(x);
  const DLDevice dev = x.device();
  check_weight(x, weight);
  const int64_t T = x.size(0), D = weight.size(0), W = weight.size(1), n = sequences(cu);
  void* w = full(weight, "weight", type, {D, W}, dev);
  void* b = full(bias, "bias", type, {D}, dev);
  const Rows xr = rows(x, "x", type, {T, D}, dev);
  const Rows out = rows(output, "output", type, {T, D}, dev);
  if (new_state.ndim() != 3) refuse("new_state", "must have three dimensions");
  const int64_t pool = new_state.size(0);
  void* ns = full(new_state, "new_state", type, {pool, W - 1, D}, dev);
  void* s = full(state, "state", type, {pool, W - 1, D}, dev);
  const Index c = index(cu, "cu_seqlens", n + 1, dev);
  const Index slots = index(state_indices, "state_indices", n, dev);
  need_slots(pool, n, slots);
  const uint8_t* has = flags(has_state, n, dev);
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_short_conv(xr.p, xr.stride, w, b, s, c.p, c.is64, slots.p, slots.is64, has,
                               static_cast<int32_t>(activation), out.p, out.stride, ns, n, T, pool,
                               static_cast<int32_t>(D), static_cast<int32_t>(W), code,
                               env_stream(dev)));
}

void ShortConvStep(TensorView x, TensorView weight, Optional<TensorView> bias,
                   TensorView state_pool, Optional<TensorView> state_indices, TensorView output,
                   Optional<TensorView> new_state_pool, int64_t activation) {
  const int32_t code = element_code(x, "x");
  const DType type = dtype_of(x);
  const DLDevice dev = x.device();
  check_weight(x, weight);
  const int64_t B = x.size(0), D = weight.size(0), W = weight.size(1);
  void* w = full(weight, "weight", type, {D, W}, dev);
  void* b = full(bias, "bias", type, {D}, dev);
  const Rows xr = rows(x, "x", type, {B, D}, dev);
  const Rows out = rows(output, "output", type, {B, D}, dev);
  if (state_pool.ndim() != 3) refuse("state_pool", "must have three dimensions");
  const int64_t pool = state_pool.size(0);
  void* s = full(state_pool, "state_pool", type, {pool, W - 1, D}, dev);
  void* ns = new_state_pool.has_value()
                 ? full(new_state_pool, "new_state_pool", type, {pool, W - 1, D}, dev)
                 : s;
  const Index slots = index(state_indices, "state_indices", B, dev);
  need_slots(pool, B, slots);
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_short_conv_step(xr.p, xr.stride, w, b, s, slots.p, slots.is64,
                                    static_cast<int32_t>(activation), out.p, out.stride, ns, B,
                                    pool, static_cast<int32_t>(D), static_cast<int32_t>(W), code,
                                    env_stream(dev)));
}

// ------------------------------------------------------------ selective scan
struct ScanOperands {
  int64_t T, H, P, G, N;
  Rows x, dt, B, C;
  const float *A_log, *D, *dt_bias;
  void* out;
};

ScanOperands scan_operands(const TensorView& x, const TensorView& dt, const TensorView& A_log,
                           const TensorView& B, const TensorView& C, const Optional<TensorView>& D,
                           const Optional<TensorView>& dt_bias, const TensorView& output) {
  if (x.ndim() != 3) refuse("x", "must be [T, H, P]");
  if (B.ndim() != 3) refuse("B", "must be [T, G, N]");
  ScanOperands o;
  const DLDevice dev = x.device();
  o.T = x.size(0);
  o.H = x.size(1);
  o.P = x.size(2);
  o.G = B.size(1);
  o.N = B.size(2);
  if (o.P != 64 && o.P != 128) refuse("x", "head_dim must be 64 or 128");
  if (o.N != 64 && o.N != 128) refuse("B", "state_dim must be 64 or 128");
  if (o.H < 1 || o.G < 1 || o.H % o.G != 0)
    refuse("B", "num_heads must be a multiple of num_groups");
  o.x = rows(x, "x", kBf16, {o.T, o.H, o.P}, dev);
  o.dt = rows(dt, "dt", kBf16, {o.T, o.H}, dev);
  o.A_log = f32(full(A_log, "A_log", kFp32, {o.H}, dev));
  o.B = rows(B, "B", kBf16, {o.T, o.G, o.N}, dev);
  o.C = rows(C, "C", kBf16, {o.T, o.G, o.N}, dev);
  o.D = f32(full(D, "D", kFp32, {o.H}, dev));
  o.dt_bias = f32(full(dt_bias, "dt_bias", kFp32, {o.H}, dev));
  o.out = full(output, "output", kBf16, {o.T, o.H, o.P}, dev);
  return o;
}

int64_t SsmPrefillWorkspace(int64_t num_seqs, int64_t total_tokens, int64_t num_heads,
                            int64_t head_dim, int64_t state_dim) {
  return static_cast<int64_t>(gdn_b200_ssm_prefill_workspace_size(
      num_seqs, total_tokens, static_cast<int32_t>(num_heads), static_cast<int32_t>(head_dim),
      static_cast<int32_t>(state_dim)));
}

void SsmPrefill(TensorView x, TensorView dt, TensorView A_log, TensorView B, TensorView C,
                Optional<TensorView> D, Optional<TensorView> dt_bias, Optional<TensorView> state,
                TensorView cu, TensorView output, TensorView new_state,
                Optional<TensorView> state_indices, Optional<TensorView> has_state,
                Optional<TensorView> workspace) {
  const ScanOperands o = scan_operands(x, dt, A_log, B, C, D, dt_bias, output);
  const DLDevice dev = x.device();
  const int64_t n = sequences(cu);
  if (new_state.ndim() != 4) refuse("new_state", "must have four dimensions");
  const int64_t pool = new_state.size(0);
  void* ns = full(new_state, "new_state", kFp32, {pool, o.H, o.P, o.N}, dev);
  void* s = full(state, "state", kFp32, {pool, o.H, o.P, o.N}, dev);
  const Index c = index(cu, "cu_seqlens", n + 1, dev);
  const Index slots = index(state_indices, "state_indices", n, dev);
  need_slots(pool, n, slots);
  const uint8_t* has = flags(has_state, n, dev);
  void* ws = nullptr;
  uint64_t ws_bytes = 0;
  if (workspace.has_value()) {
    const TensorView& w = workspace.value();
    if (w.device().device_type != dev.device_type || w.device().device_id != dev.device_id)
      refuse("workspace", "must be on the same device as x");
    if (!w.IsContiguous()) refuse("workspace", "must be contiguous");
    ws = ptr(w);
    ws_bytes = static_cast<uint64_t>(w.numel()) * w.dtype().bits / 8;
    if (static_cast<int64_t>(ws_bytes) < SsmPrefillWorkspace(n, o.T, o.H, o.P, o.N))
      refuse("workspace", "is smaller than ssm_prefill_workspace_bytes()");
  }
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_ssm_prefill(
      o.x.p, o.x.stride, o.dt.p, o.dt.stride, o.A_log, o.B.p, o.B.stride, o.C.p, o.C.stride, o.D,
      o.dt_bias, f32(s), c.p, c.is64, slots.p, slots.is64, has, o.out, static_cast<float*>(ns), n,
      o.T, pool, static_cast<int32_t>(o.H), static_cast<int32_t>(o.G), static_cast<int32_t>(o.P),
      static_cast<int32_t>(o.N), ws, ws_bytes, env_stream(dev)));
}

void SsmStep(TensorView x, TensorView dt, TensorView A_log, TensorView B, TensorView C,
             Optional<TensorView> D, Optional<TensorView> dt_bias, TensorView state_pool,
             Optional<TensorView> state_indices, TensorView output,
             Optional<TensorView> new_state_pool, Optional<TensorView> output_state_indices) {
  const ScanOperands o = scan_operands(x, dt, A_log, B, C, D, dt_bias, output);
  const DLDevice dev = x.device();
  if (state_pool.ndim() != 4) refuse("state_pool", "must have four dimensions");
  const int64_t pool = state_pool.size(0);
  void* s = full(state_pool, "state_pool", kFp32, {pool, o.H, o.P, o.N}, dev);
  void* ns = new_state_pool.has_value()
                 ? full(new_state_pool, "new_state_pool", kFp32, {pool, o.H, o.P, o.N}, dev)
                 : s;
  const Index read = index(state_indices, "state_indices", o.T, dev);
  const Index write = index(output_state_indices, "output_state_indices", o.T, dev);
  if (write.p != nullptr && (read.p == nullptr || read.is64 != write.is64))
    refuse("output_state_indices", "need state_indices of the same type");
  need_slots(pool, o.T, read);
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_ssm_step(o.x.p, o.x.stride, o.dt.p, o.dt.stride, o.A_log, o.B.p, o.B.stride,
                             o.C.p, o.C.stride, o.D, o.dt_bias, f32(s), read.p, write.p, read.is64,
                             o.out, static_cast<float*>(ns), o.T, pool,
                             static_cast<int32_t>(o.H), static_cast<int32_t>(o.G),
                             static_cast<int32_t>(o.P), static_cast<int32_t>(o.N), env_stream(dev)));
}

// ------------------------------------------------------------ norms
// group_size 0: the last dimension.
void GatedNorm(TensorView x, Optional<TensorView> gate, Optional<TensorView> weight,
               TensorView output, int64_t group_size, double eps, int64_t activation,
               int64_t norm_first) {
  const int32_t code = element_code(x, "x");
  const DType type = dtype_of(x);
  const DLDevice dev = x.device();
  if (x.ndim() != 2 && x.ndim() != 3) refuse("x", "must be [T, D] or [T, H, P]");
  const int64_t T = x.size(0), last = x.size(x.ndim() - 1);
  const int64_t width = x.ndim() == 3 ? x.size(1) * last : last;
  const int64_t group = group_size == 0 ? last : group_size;
  if (group < 1 || width < 1 || width % group != 0)
    TVM_FFI_THROW(ValueError) << "group_size must divide the row's width " << width << ", got "
                              << group;
  auto view = [&](const TensorView& t, const char* name) {
    return x.ndim() == 2 ? rows(t, name, type, {T, width}, dev)
                         : rows(t, name, type, {T, x.size(1), last}, dev);
  };
  const Rows xr = view(x, "x"), out = view(output, "output");
  const Rows g = gate.has_value() ? view(gate.value(), "gate") : Rows{nullptr, 0};
  void* w = nullptr;
  int32_t shared = 0;
  if (weight.has_value()) {
    const TensorView& t = weight.value();
    if (!is_dtype(t, type.code, type.bits)) refuse("weight", "wrong dtype");
    if (t.numel() != group && t.numel() != width)
      TVM_FFI_THROW(ValueError) << "weight: expected " << group << " or " << width << " elements";
    if (!t.IsContiguous()) refuse("weight", "must be contiguous");
    if (t.device().device_type != dev.device_type || t.device().device_id != dev.device_id)
      refuse("weight", "must be on the same device as x");
    w = ptr(t);
    shared = t.numel() == group ? 1 : 0;
  }
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_gated_norm(xr.p, xr.stride, g.p, g.stride, w, shared, out.p, out.stride, T,
                               static_cast<int32_t>(width), static_cast<int32_t>(group), eps,
                               static_cast<int32_t>(activation), static_cast<int32_t>(norm_first),
                               code, env_stream(dev)));
}

void AddNorm(TensorView x, TensorView residual, TensorView weight, TensorView output,
             TensorView new_residual, Optional<TensorView> block_weight,
             Optional<TensorView> channel_scale, double scale, double eps, double weight_offset) {
  const int32_t code = element_code(x, "x");
  const DType type = dtype_of(x);
  const DLDevice dev = x.device();
  if (x.ndim() != 2) refuse("x", "must be [T, D]");
  const int64_t T = x.size(0), D = x.size(1);
  if (D < 1) refuse("x", "rows must not be empty");
  const DType rtype = dtype_of(residual);
  const bool fp32 = is_dtype(residual, kDLFloat, 32);
  if (!fp32 && !is_dtype(residual, type.code, type.bits))
    refuse("residual", "must have the type of x, or float32");
  const Rows xr = rows(x, "x", type, {T, D}, dev), out = rows(output, "output", type, {T, D}, dev);
  const Rows r = rows(residual, "residual", rtype, {T, D}, dev);
  const Rows nr = rows(new_residual, "new_residual", rtype, {T, D}, dev);
  void* w = full(weight, "weight", type, {D}, dev);
  void* bw = full(block_weight, "block_weight", type, {D}, dev);
  void* cs = full(channel_scale, "scale", kFp32, {D}, dev);
  DeviceGuard guard(cuda_device(x));
  check_rc(gdn_b200_add_norm(xr.p, xr.stride, r.p, r.stride, w, bw, f32(cs), scale, out.p,
                             out.stride, nr.p, nr.stride, T, static_cast<int32_t>(D), eps,
                             weight_offset, code, fp32 ? 1 : 0, env_stream(dev)));
}

}  // namespace gdn_tvm

TVM_FFI_DLL_EXPORT_TYPED_FUNC(short_conv, gdn_tvm::ShortConv);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(short_conv_step, gdn_tvm::ShortConvStep);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(ssm_prefill_workspace, gdn_tvm::SsmPrefillWorkspace);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(ssm_prefill, gdn_tvm::SsmPrefill);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(ssm_step, gdn_tvm::SsmStep);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(gated_norm, gdn_tvm::GatedNorm);
TVM_FFI_DLL_EXPORT_TYPED_FUNC(add_norm, gdn_tvm::AddNorm);
