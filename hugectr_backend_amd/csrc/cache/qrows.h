// Rows held in 8 or 4 bits on the device, addressed by slot: written (quantised) and read back.  See qrows_kernels.hip for the
// kernels and include/hps_amd.h (hps_qrows_*) for the C ABI.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace hps {

// types of rows, layers' operands and outputs at the C ABI (HPS_TYPE_*)
enum class ElemType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline uint32_t ElemBytes(ElemType t) { return t == ElemType::kF32 ? 4u : 2u; }

constexpr uint32_t kQRowsMaxDim = 16384;
constexpr uint32_t kQRowsListed = 65535;

struct QRowsDesc {
  uint8_t* codes = nullptr;     // [num_rows][row_bytes]
  float* scales = nullptr;      // [num_rows][groups]
  uint32_t* claim = nullptr;    // [num_rows], zero between calls
  uint32_t* stamp = nullptr;    // [num_rows]
  uint32_t* listed = nullptr;   // [1 + kQRowsListed]: how many rows, which
  uint64_t num_rows = 0;
  uint32_t dim = 0;
  uint32_t bits = 8;
  uint32_t group = 0;           // values per scale; >= dim: one scale per row
  uint32_t groups = 1;
  uint32_t row_bytes = 0;       // codes of a row, rounded up to 4 bytes
};

// 4-byte words: a lane's smallest access to codes, so that rows of any width stay aligned for it without the waste of 16
inline uint32_t QRowsRowBytes(uint32_t dim, uint32_t bits) { return ((uint32_t)(((uint64_t)dim * bits + 7) / 8) + 3) / 4 * 4; }

// what a write needs beside the store: claims, stamps and the list (zero before the first write)
inline uint64_t QRowsWorkspaceBytes(uint64_t num_rows) { return (2 * num_rows + 1 + kQRowsListed) * 4; }

hipError_t LaunchQRowsWrite(const QRowsDesc& s, const void* d_rows, ElemType type, uint64_t row_stride, const int64_t* d_slots, uint64_t n,
                            void* d_held, uint64_t held_stride, hipStream_t stream);
hipError_t LaunchQRowsRead(const QRowsDesc& s, const int64_t* d_slots, uint64_t n, float default_value, void* d_out, ElemType type,
                           uint64_t out_stride, hipStream_t stream);

}  // namespace hps
