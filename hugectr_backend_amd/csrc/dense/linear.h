// Dense layers behind the interaction: y = act(x W + b) * mul + residual, one layer or one per expert over ragged runs of rows, and
// the grouping of rows by expert.  See linear_kernels.hip and group_rows.hip for the kernels, include/hps_amd.h (hps_linear_*,
// hps_group_rows_*) for the C ABI.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include <memory>

#include "../cache/qrows.h"
#include "../common/status.h"

namespace hps {

enum class Activation : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3, kSigmoid = 4 };

constexpr uint32_t kMaxExperts = 1024;
constexpr uint32_t kLinearMaxDim = 1u << 20;

// LinearArgs::zero_rest
constexpr uint16_t kZeroRest = 1;      // positions of no run write zeros (else their rows stay as they were)
constexpr uint16_t kZeroUnnamed = 2;   // and so do the rows of out that no position names (out has one row per position then)

// One call's operands, all on the device.  Strides in elements.
struct LinearArgs {
  const void* x = nullptr;            // layer type, [x_rows][x_stride]
  uint64_t x_stride = 0, x_rows = 0;
  void* out = nullptr;                // out type, [out_rows][out_stride]
  uint64_t out_stride = 0, out_rows = 0;
  const void* mul = nullptr;          // layer type, rows like out's
  uint64_t mul_stride = 0;
  const void* residual = nullptr;     // layer type, rows like out's
  uint64_t residual_stride = 0;
  const int32_t* offsets = nullptr;   // [experts + 1]; null: one run over all positions
  const int32_t* rows_in = nullptr;   // position -> row of x; null: the position itself
  const int32_t* rows_out = nullptr;  // position -> row of out, mul and residual; null: the position itself
  uint32_t rows = 0;                  // positions
  uint16_t zero_rest = 0;             // 0, kZeroRest, kZeroUnnamed
  uint16_t stream_out = 0;            // set by the launcher
};
// One kernel argument of 120 bytes or more costs the host 0.8 us a launch (2.8 -> 3.6 us, whatever its size beyond)
static_assert(sizeof(LinearArgs) <= 112, "one kernel argument");

struct LinearDesc {
  const void* w = nullptr;     // fragment order (linear_kernels.hip), [experts][npairs][ksteps][2][64][8]
  const float* bias = nullptr; // [experts][npairs * 32], zero where there is none
  uint32_t K = 0, N = 0;
  uint32_t ksteps = 0;         // ceil(K / 32)
  uint32_t npairs = 0;         // ceil(N / 32)
  uint32_t experts = 1;
  int act = 0;
};

hipError_t LaunchLinearPack(const void* d_w, ElemType from, uint32_t experts, uint32_t K, uint32_t N, void* d_packed, ElemType to,
                            hipStream_t stream);
hipError_t LaunchLinear(const LinearDesc& d, const LinearArgs& a, ElemType type, ElemType out_type, int cu_count, hipStream_t stream);

// The rows and columns a workgroup takes: which of the five kernels a call runs
struct LinearTile {
  uint32_t rows, cols;
};
LinearTile LinearTileOf(const LinearDesc& d, uint64_t rows, bool offsets, int cu_count);

uint64_t GroupRowsWorkspaceBytes(uint64_t n, uint32_t experts);
hipError_t LaunchGroupRows(const int32_t* d_ids, uint64_t n, uint32_t experts, int32_t* d_offsets, int32_t* d_order, void* d_workspace,
                           hipStream_t stream);

// Owns the packed weights on one device.  Forward keeps nothing between calls: any number of threads and streams may call it.
class LinearLayers {
 public:
  ~LinearLayers();
  // weights: [experts][K][N] row-major (the x @ W convention) of `from`; bias: [experts][N] fp32 or null; both on the host, or both on
  // the device and ready on `stream`
  static Status Create(int device, uint32_t experts, uint32_t K, uint32_t N, ElemType type, Activation act, const void* weights,
                       ElemType from, const float* bias, bool on_device, hipStream_t stream, LinearLayers** out);
  Status Forward(const LinearArgs& a, ElemType out_type, hipStream_t stream);
  LinearTile Tile(uint64_t rows, bool offsets) const { return LinearTileOf(d_, rows, offsets, cu_count_); }

 private:
  LinearLayers() = default;
  int device_ = 0;
  int cu_count_ = 256;
  ElemType type_ = ElemType::kF16;
  LinearDesc d_;
  void* w_ = nullptr;
  void* bias_ = nullptr;
};

}  // namespace hps
