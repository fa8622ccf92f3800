#include "linear.h"

#include <hip/hip_runtime.h>

#include "../common/device_guard.h"
#include "../common/span.h"

namespace hps {

#define HIP_TRY(expr)                                                                              \
  do {                                                                                             \
    hipError_t _e = (expr);                                                                        \
    if (_e != hipSuccess)                                                                          \
      return ::hps::Error(::hps::Code::kInternal, #expr, " failed: ", hipGetErrorString(_e), " (", \
                          __FILE__, ":", __LINE__, ")");                                           \
  } while (0)

namespace {

// Device memory that is freed on every way out of Create
struct DeviceBuffer {
  void* p = nullptr;
  ~DeviceBuffer() {
    if (p) (void)hipFree(p);
  }
  void* release() {
    void* q = p;
    p = nullptr;
    return q;
  }
};

}  // namespace

LinearLayers::~LinearLayers() {
  DeviceGuard guard;
  if (!w_ && !bias_) return;
  (void)guard.Enter(device_);
  if (w_) (void)hipFree(w_);
  if (bias_) (void)hipFree(bias_);
}

Status LinearLayers::Create(int device, uint32_t experts, uint32_t K, uint32_t N, ElemType type, Activation act, const void* weights,
                            ElemType from, const float* bias, bool on_device, hipStream_t stream, LinearLayers** out) {
  if (experts == 0 || experts > kMaxExperts) return Error(Code::kInvalidArg, "linear layer: 1..", kMaxExperts, " experts supported, got ", experts);
  if (K == 0 || K > kLinearMaxDim || N == 0 || N > kLinearMaxDim)
    return Error(Code::kInvalidArg, "linear layer: widths of 1..", kLinearMaxDim, " supported, got ", K, " -> ", N);
  if (type != ElemType::kF16 && type != ElemType::kBF16) return Error(Code::kInvalidArg, "linear layer: operands are fp16 or bf16, got type ", (int)type);
  if ((int)from < 0 || (int)from > 2) return Error(Code::kInvalidArg, "linear layer: unknown type of the weights ", (int)from);
  if ((int)act < 0 || (int)act > (int)Activation::kSigmoid) return Error(Code::kInvalidArg, "linear layer: unknown activation ", (int)act);
  if (!weights) return Error(Code::kInvalidArg, "linear layer: null weights");
  if (on_device && ((uintptr_t)weights % ElemBytes(from) || (uintptr_t)bias % 4))
    return Error(Code::kInvalidArg, "linear layer: weights and bias on the device are aligned to their elements");
  const uint32_t ksteps = (K + 31) / 32, npairs = (N + 31) / 32;
  const unsigned __int128 packed_bytes = (unsigned __int128)experts * npairs * ksteps * 2048, limit = (unsigned __int128)1 << 40;
  if (packed_bytes > limit) return Error(Code::kUnsupported, "linear layer: weights of more than 2^40 bytes");

  DeviceGuard guard;
  HPS_RETURN_IF_ERROR(guard.Enter(device));
  std::unique_ptr<LinearLayers> l(new LinearLayers());
  l->device_ = device;
  l->type_ = type;
  int cus = 0;
  HIP_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
  if (cus > 0) l->cu_count_ = cus;
  l->d_.K = K;
  l->d_.N = N;
  l->d_.ksteps = ksteps;
  l->d_.npairs = npairs;
  l->d_.experts = experts;
  l->d_.act = (int)act;
  DeviceBuffer staged;
  const void* src = weights;
  if (!on_device) {
    const uint64_t bytes = (uint64_t)experts * K * N * ElemBytes(from);
    HIP_TRY(hipMalloc(&staged.p, bytes));
    HIP_TRY(hipMemcpyAsync(staged.p, weights, bytes, hipMemcpyHostToDevice, stream));
    src = staged.p;
  }
  HIP_TRY(hipMalloc(&l->w_, (uint64_t)packed_bytes));
  HIP_TRY(hipMalloc(&l->bias_, (uint64_t)experts * npairs * 32 * sizeof(float)));
  HIP_TRY(LaunchLinearPack(src, from, experts, K, N, l->w_, type, stream));
  HIP_TRY(hipMemsetAsync(l->bias_, 0, (uint64_t)experts * npairs * 32 * sizeof(float), stream));
  if (bias)
    HIP_TRY(hipMemcpy2DAsync(l->bias_, (uint64_t)npairs * 32 * sizeof(float), bias, (uint64_t)N * sizeof(float), (uint64_t)N * sizeof(float),
                             experts, on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice, stream));
  HIP_TRY(hipStreamSynchronize(stream));   // the layer is ready for every stream from here on
  l->d_.w = l->w_;
  l->d_.bias = (const float*)l->bias_;
  *out = l.release();
  return Status::Ok();
}

Status LinearLayers::Forward(const LinearArgs& a, ElemType out_type, hipStream_t stream) {
  const LinearDesc& d = d_;
  if (out_type != type_ && out_type != ElemType::kF32)
    return Error(Code::kInvalidArg, "linear forward: the output has the layer's type or fp32, got type ", (int)out_type);
  if (a.rows >= (1u << 31)) return Error(Code::kUnsupported, "linear forward: more than 2^31 rows per call");
  if (a.rows == 0) return Status::Ok();
  if (!a.x || !a.out) return Error(Code::kInvalidArg, "linear forward: null device pointer");
  if (d.experts > 1 && !a.offsets) return Error(Code::kInvalidArg, "linear forward: ", d.experts, " experts need the offsets of their runs");
  if (a.x_stride < d.K || a.out_stride < d.N || (a.mul && a.mul_stride < d.N) || (a.residual && a.residual_stride < d.N))
    return Error(Code::kInvalidArg, "linear forward: rows are closer together than they are wide");
  if (a.x_rows == 0 || a.out_rows == 0) return Error(Code::kInvalidArg, "linear forward: rows without an input or an output row");
  if (!a.rows_in && a.x_rows < a.rows) return Error(Code::kInvalidArg, "linear forward: ", a.rows, " rows of an input of ", a.x_rows);
  if (!a.rows_out && a.out_rows < a.rows) return Error(Code::kInvalidArg, "linear forward: ", a.rows, " rows into an output of ", a.out_rows);
  const uint64_t in = ElemBytes(type_), ob = ElemBytes(out_type);
  if ((uintptr_t)a.x % in || (uintptr_t)a.out % ob || (uintptr_t)a.mul % in || (uintptr_t)a.residual % in || (uintptr_t)a.offsets % 4 ||
      (uintptr_t)a.rows_in % 4 || (uintptr_t)a.rows_out % 4)
    return Error(Code::kInvalidArg, "linear forward: a pointer that is not aligned to its elements");
  const Span so(a.out, a.out_rows, a.out_stride, d.N, ob), sx(a.x, a.x_rows, a.x_stride, d.K, in);
  if (so.meets(sx)) return Error(Code::kInvalidArg, "linear forward: the output overlaps the input");
  if (so.meets(Span(a.offsets, 1, 0, (uint64_t)d.experts + 1, 4)) || so.meets(Span(a.rows_in, 1, 0, a.rows, 4)) || so.meets(Span(a.rows_out, 1, 0, a.rows, 4)))
    return Error(Code::kInvalidArg, "linear forward: the output overlaps offsets or row indexes");
  // in place over mul or residual: every element is read by the thread that writes it
  auto apart = [&](const void* p, uint64_t stride) {
    const bool same = p == a.out && stride == a.out_stride && ob == in;
    return same || !so.meets(Span(p, a.out_rows, stride, d.N, in));
  };
  if ((a.mul && !apart(a.mul, a.mul_stride)) || (a.residual && !apart(a.residual, a.residual_stride)))
    return Error(Code::kInvalidArg, "linear forward: the output overlaps mul or residual without being the same rows of the same type");
  if (a.zero_rest == kZeroUnnamed && a.out_rows != a.rows)
    return Error(Code::kInvalidArg, "linear forward: rows that no position names become zeros in an output of one row per position, got ", a.out_rows, " for ", a.rows);
  DeviceGuard guard;
  HPS_RETURN_IF_ERROR(guard.Enter(device_));
  const hipError_t e = LaunchLinear(d, a, type_, out_type, cu_count_, stream);
  if (e == hipErrorInvalidConfiguration) return Error(Code::kUnsupported, "linear forward: more tiles than a launch holds; split the rows");
  if (e != hipSuccess) return Error(Code::kInternal, "linear forward launch failed: ", hipGetErrorString(e));
  return Status::Ok();
}

}  // namespace hps
