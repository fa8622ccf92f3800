// Rows held in 8 or 4 bits, addressed by slot.
//
//   write   per group of `group` values (a whole row unless asked otherwise): a = max |x|, s = fp32(a / L) with L = 127 (8 bits) or 7
//           (4 bits), code = x / s to the nearest integer, ties to even.  a < 2^-100: s = 0 and codes 0 (below that the 32-bit quotient
//           leaves the normal numbers); a NaN or an infinity in the group: s = NaN, so that the whole group reads back as NaN.
//   read    out = code * s
//
// Both are HBM-bound byte movers.  A row belongs to a team of 2^j lanes of one wave, each lane takes V consecutive values (16 bytes
// of the wider side), so a wave reads and writes whole lines; the largest magnitude is reduced inside the team with lane exchanges.
//
// The code is exact: code = rint(x / s) of the REAL quotient.  x * (1 / s) is off by at most 127 * 2^-22 = 3.1e-5, so only a product
// within 1e-4 of a half-integer can round to the wrong side; there the sign of x - (r +- 1/2) s decides, which one fused
// multiply-add gives exactly (rounding a nonzero number never changes its sign, and 2^-100 keeps it out of the denormals).
//
// A slot that is named twice in one call keeps its LAST row, whole: a first kernel leaves the highest position in owner[slot] with
// one atomic maximum per row, the second kernel writes a row only where its own position is there and puts the zero back, so the
// array is clear again for the next call (and for a graph's next replay) without a pass over it.
#include <hip/hip_bfloat16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qrows.h"

namespace hps {

typedef float f4q __attribute__((ext_vector_type(4)));
typedef uint32_t u2q __attribute__((ext_vector_type(2)));
typedef uint32_t u4q __attribute__((ext_vector_type(4)));

constexpr int kQThreads = 256;
constexpr uint64_t kQRowsPerLaunch = 1ull << 24;   // a launch holds at most 2^32 threads; a row takes up to 64
constexpr float kQTiny = 0x1p-100f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// V values of a row: one access where the row allows it (VEC: dim, stride and base are multiples of V values), else one by one
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_values(const T* __restrict__ row, uint32_t at, uint32_t dim, float (&x)[V]) {
  if constexpr (VEC) {
    typedef T vt __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int P = 16 / sizeof(T);
    static_assert(V % P == 0, "whole 16-byte accesses");
#pragma unroll
    for (int j = 0; j < V / P; ++j) {
      const vt v = __builtin_nontemporal_load(reinterpret_cast<const vt*>(row + at) + j);
#pragma unroll
      for (int k = 0; k < P; ++k) x[j * P + k] = to_float(v[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = at + k < dim ? to_float(row[at + k]) : 0.f;
  }
}

template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_values(T* __restrict__ row, uint32_t at, uint32_t dim, const float (&x)[V]) {
  if constexpr (VEC) {
    typedef T vt __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int P = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < V / P; ++j) {
      vt v;
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = (T)x[j * P + k];
      __builtin_nontemporal_store(v, reinterpret_cast<vt*>(row + at) + j);
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (at + k < dim) row[at + k] = (T)x[k];
  }
}

// the nearest integer to x / s, ties to even (see the head of the file); inv ~ 1 / s
__device__ __forceinline__ int nearest_code(float x, float s, float inv, float levels) {
  const float q = x * inv;
  float r = rintf(q);
  if (fabsf(fabsf(q - r) - 0.5f) < 1e-4f) {
    const bool odd = ((int)r & 1) != 0;
    const float over = fmaf(-(r + 0.5f), s, x), under = fmaf(-(r - 0.5f), s, x);
    if (over > 0.f || (over == 0.f && odd)) r += 1.f;
    else if (under < 0.f || (under == 0.f && odd)) r -= 1.f;
  }
  return (int)fminf(fmaxf(r, -levels), levels);
}

__global__ __launch_bounds__(kQThreads) void hps_qrows_claim_kernel(const int64_t* __restrict__ slots, uint64_t n, uint64_t num_rows,
                                                                    uint32_t* __restrict__ owner) {
  const uint64_t i = (uint64_t)blockIdx.x * kQThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t slot = slots[i];
  if (slot >= 0 && (uint64_t)slot < num_rows) atomicMax(&owner[slot], (uint32_t)i + 1u);
}

template <typename T, int BITS>
constexpr int kQWriteV = (sizeof(T) == 2 || BITS == 4) ? 8 : 4;

// NCH chunks of V values per lane stay in registers; NCH = 0: rows wider than that are read twice
template <typename T, int BITS, bool VEC, int NCH>
__global__ __launch_bounds__(kQThreads) void hps_qrows_write_kernel(QRowsDesc s, const T* rows, uint64_t row_stride,
                                                                    const int64_t* __restrict__ slots, uint64_t first, uint64_t n, T* held,
                                                                    uint64_t held_stride, uint32_t team_log, uint32_t reduce_lanes) {
  constexpr int V = kQWriteV<T, BITS>;
  constexpr float kLevels = BITS == 8 ? 127.f : 7.f;
  constexpr int kKeep = NCH ? NCH : 1;
  const uint32_t team = 1u << team_log, lane = threadIdx.x & (team - 1);
  const uint64_t i = first + (((uint64_t)blockIdx.x * kQThreads + threadIdx.x) >> team_log);
  const bool live = i < n;                       // (a team is live or not as a whole; the wave's exchanges need every lane)
  const uint32_t dim = s.dim, chunks = (dim + V - 1) / V, rounds = (chunks + team - 1) >> team_log;
  const T* row = rows + (live ? i : 0) * row_stride;
  float x[kKeep][V];
  const int64_t slot = live ? slots[i] : -1;
  const bool inside = slot >= 0 && (uint64_t)slot < s.num_rows;
  if constexpr (NCH != 0) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const uint32_t c = lane + ((uint32_t)k << team_log);
#pragma unroll
      for (int v = 0; v < V; ++v) x[k][v] = 0.f;
      if (live && c < chunks) load_values<T, V, VEC>(row, c * V, dim, x[k]);
    }
  }
  const bool mine = inside && s.owner[slot] == (uint32_t)i + 1u;
  // magnitudes compare as integers: |NaN| > infinity > every finite value
  auto top_of = [](const float(&v)[V]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const uint32_t a = __float_as_uint(v[k]) & 0x7fffffffu;
      m = a > m ? a : m;
    }
    return m;
  };
  auto over_lanes = [](uint32_t m, uint32_t lanes) {
    for (uint32_t d = 1; d < lanes; d <<= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)m, (int)d, 64);
      m = o > m ? o : m;
    }
    return m;
  };
  const bool whole = s.groups == 1;
  uint32_t top = 0;
  if (whole) {
    if constexpr (NCH != 0) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const uint32_t t = top_of(x[k]);
        top = t > top ? t : top;
      }
    } else {
      for (uint32_t c = lane; live && c < chunks; c += team) {
        load_values<T, V, VEC>(row, c * V, dim, x[0]);
        const uint32_t t = top_of(x[0]);
        top = t > top ? t : top;
      }
    }
    top = over_lanes(top, reduce_lanes);
  }
  uint8_t* codes = s.codes + (mine ? (uint64_t)slot : 0) * s.row_bytes;
  float* scales = s.scales + (mine ? (uint64_t)slot : 0) * s.groups;
  T* out = held ? held + (live ? i : 0) * held_stride : nullptr;
  auto finish = [&](uint32_t c, float(&v)[V], uint32_t t) {   // every lane of the wave comes here (lane exchanges)
    const uint32_t m = whole ? t : over_lanes(top_of(v), reduce_lanes);
    const float a = __uint_as_float(m);
    float scale = a / kLevels;
    if (a < kQTiny) scale = 0.f;
    if (m >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
    const bool codable = scale > 0.f;
    const float inv = __builtin_amdgcn_rcpf(scale);
    if (!live || c >= chunks) return;
    int q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) q[k] = codable ? nearest_code(v[k], scale, inv, kLevels) : 0;
    if (mine) {
      const uint32_t at = c * V;
      if (whole ? c == 0 : at % s.group == 0) scales[whole ? 0 : at / s.group] = scale;
      if constexpr (BITS == 8) {
        uint32_t w[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
          w[j] = (uint32_t)(q[4 * j] & 255) | (uint32_t)(q[4 * j + 1] & 255) << 8 | (uint32_t)(q[4 * j + 2] & 255) << 16 |
                 (uint32_t)(q[4 * j + 3] & 255) << 24;
        uint32_t* dst = reinterpret_cast<uint32_t*>(codes) + c * (V / 4);
        if constexpr (V == 4) {
          *dst = w[0];
        } else if (s.row_bytes % 8 == 0) {
          *reinterpret_cast<u2q*>(dst) = u2q{w[0], w[1]};
        } else {
          dst[0] = w[0];
          if (c * 2 + 1 < s.row_bytes / 4) dst[1] = w[1];
        }
      } else {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) w |= (uint32_t)(q[k] & 15) << (4 * k);
        reinterpret_cast<uint32_t*>(codes)[c] = w;
      }
    }
    if (out) {
      float y[V];
#pragma unroll
      for (int k = 0; k < V; ++k) y[k] = (float)q[k] * scale;
      store_values<T, V, VEC>(out, c * V, dim, y);
    }
  };
  if constexpr (NCH != 0) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      if ((uint32_t)k < rounds) finish(lane + ((uint32_t)k << team_log), x[k], top);
  } else {
    for (uint32_t k = 0; k < rounds; ++k) {
      const uint32_t c = lane + (k << team_log);
#pragma unroll
      for (int v = 0; v < V; ++v) x[0][v] = 0.f;
      if (live && c < chunks) load_values<T, V, VEC>(row, c * V, dim, x[0]);
      finish(c, x[0], top);
    }
  }
  if (mine && lane == 0) s.owner[slot] = 0;
}

template <typename T, int BITS, bool VEC>
__global__ __launch_bounds__(kQThreads) void hps_qrows_read_kernel(QRowsDesc s, const int64_t* __restrict__ slots, uint64_t first, uint64_t n,
                                                                   float default_value, T* __restrict__ out, uint64_t out_stride,
                                                                   uint32_t team_log, uint32_t group_log) {
  constexpr int V = kQWriteV<T, BITS>;
  const uint32_t team = 1u << team_log, lane = threadIdx.x & (team - 1);
  const uint64_t i = first + (((uint64_t)blockIdx.x * kQThreads + threadIdx.x) >> team_log);
  if (i >= n) return;
  const int64_t slot = slots[i];
  const bool inside = slot >= 0 && (uint64_t)slot < s.num_rows;
  const uint32_t dim = s.dim, chunks = (dim + V - 1) / V, words = s.row_bytes / 4;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(s.codes + (inside ? (uint64_t)slot : 0) * s.row_bytes);
  const float* scales = s.scales + (inside ? (uint64_t)slot : 0) * s.groups;
  T* row = out + i * out_stride;
  for (uint32_t c = lane; c < chunks; c += team) {
    float y[V];
    if (inside) {
      const float scale = scales[s.groups == 1 ? 0 : (c * V) >> group_log];
      if constexpr (BITS == 8) {
        uint32_t w[V / 4];
        if constexpr (V == 4) {
          w[0] = codes[c];
        } else if (words % 2 == 0) {
          const u2q p = *reinterpret_cast<const u2q*>(codes + 2 * c);
          w[0] = p[0], w[1] = p[1];
        } else {
          w[0] = codes[2 * c];
          w[1] = 2 * c + 1 < words ? codes[2 * c + 1] : 0;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = (float)((int)(w[k / 4] << (24 - 8 * (k % 4))) >> 24) * scale;
      } else {
        const uint32_t w = codes[c];
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = (float)((int)(w << (28 - 4 * k)) >> 28) * scale;
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) y[k] = default_value;
    }
    store_values<T, V, VEC>(row, c * V, dim, y);
  }
}

namespace {

struct TeamShape {
  uint32_t team_log, rounds, reduce_lanes;
};

TeamShape TeamOf(uint32_t dim, uint32_t V, uint32_t group, uint32_t groups) {
  const uint32_t chunks = (dim + V - 1) / V;
  TeamShape t{0, 0, 0};
  while ((1u << t.team_log) < chunks && t.team_log < 6) ++t.team_log;
  t.rounds = (chunks + (1u << t.team_log) - 1) >> t.team_log;
  t.reduce_lanes = groups == 1 ? 1u << t.team_log : group / V;   // group < dim, so its lanes fit the team
  return t;
}

bool Aligned(const void* p, uint64_t stride, uint32_t dim, uint32_t V, uint32_t bytes) {
  return dim % V == 0 && (stride * bytes) % 16 == 0 && (uintptr_t)p % 16 == 0;
}

template <typename T, int BITS, bool VEC>
hipError_t WriteTyped(const QRowsDesc& s, const void* rows, uint64_t row_stride, const int64_t* slots, uint64_t n, void* held,
                      uint64_t held_stride, hipStream_t stream) {
  const TeamShape t = TeamOf(s.dim, kQWriteV<T, BITS>, s.group, s.groups);
  const uint32_t claim_blocks = (uint32_t)((n + kQThreads - 1) / kQThreads);
  hps_qrows_claim_kernel<<<claim_blocks, kQThreads, 0, stream>>>(slots, n, s.num_rows, s.owner);
#define HPS_QROWS_WRITE(NCH)                                                                                                              \
  hps_qrows_write_kernel<T, BITS, VEC, NCH><<<blocks, kQThreads, 0, stream>>>(s, (const T*)rows, row_stride, slots, first, end, (T*)held, \
                                                                              held_stride, t.team_log, t.reduce_lanes)
  for (uint64_t first = 0; first < n; first += kQRowsPerLaunch) {
    const uint64_t end = first + kQRowsPerLaunch < n ? first + kQRowsPerLaunch : n;
    const uint32_t blocks = (uint32_t)((((end - first) << t.team_log) + kQThreads - 1) / kQThreads);
    if (t.rounds == 1) HPS_QROWS_WRITE(1);
    else if (t.rounds <= 4) HPS_QROWS_WRITE(4);
    else HPS_QROWS_WRITE(0);
  }
#undef HPS_QROWS_WRITE
  return hipGetLastError();
}

template <typename T, int BITS, bool VEC>
hipError_t ReadTyped(const QRowsDesc& s, const int64_t* slots, uint64_t n, float default_value, void* out, uint64_t out_stride,
                     hipStream_t stream) {
  const TeamShape t = TeamOf(s.dim, kQWriteV<T, BITS>, s.group, s.groups);
  uint32_t group_log = 0;
  while (s.groups > 1 && (1u << group_log) < s.group) ++group_log;
  for (uint64_t first = 0; first < n; first += kQRowsPerLaunch) {
    const uint64_t end = first + kQRowsPerLaunch < n ? first + kQRowsPerLaunch : n;
    const uint32_t blocks = (uint32_t)((((end - first) << t.team_log) + kQThreads - 1) / kQThreads);
    hps_qrows_read_kernel<T, BITS, VEC><<<blocks, kQThreads, 0, stream>>>(s, slots, first, end, default_value, (T*)out, out_stride,
                                                                          t.team_log, group_log);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchQRowsWrite(const QRowsDesc& s, const void* d_rows, ElemType type, uint64_t row_stride, const int64_t* d_slots, uint64_t n,
                            void* d_held, uint64_t held_stride, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const uint32_t bytes = ElemBytes(type), V = (bytes == 2 || s.bits == 4) ? 8 : 4;
  const bool vec = Aligned(d_rows, row_stride, s.dim, V, bytes) && (!d_held || Aligned(d_held, held_stride, s.dim, V, bytes));
#define HPS_QROWS_TYPED(T, BITS)                                                                                           \
  return vec ? WriteTyped<T, BITS, true>(s, d_rows, row_stride, d_slots, n, d_held, held_stride, stream)                   \
             : WriteTyped<T, BITS, false>(s, d_rows, row_stride, d_slots, n, d_held, held_stride, stream)
  if (s.bits == 8) {
    if (type == ElemType::kF32) HPS_QROWS_TYPED(float, 8);
    if (type == ElemType::kF16) HPS_QROWS_TYPED(_Float16, 8);
    HPS_QROWS_TYPED(__bf16, 8);
  }
  if (type == ElemType::kF32) HPS_QROWS_TYPED(float, 4);
  if (type == ElemType::kF16) HPS_QROWS_TYPED(_Float16, 4);
  HPS_QROWS_TYPED(__bf16, 4);
#undef HPS_QROWS_TYPED
}

hipError_t LaunchQRowsRead(const QRowsDesc& s, const int64_t* d_slots, uint64_t n, float default_value, void* d_out, ElemType type,
                           uint64_t out_stride, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const uint32_t bytes = ElemBytes(type), V = (bytes == 2 || s.bits == 4) ? 8 : 4;
  const bool vec = Aligned(d_out, out_stride, s.dim, V, bytes);
#define HPS_QROWS_TYPED(T, BITS)                                                                              \
  return vec ? ReadTyped<T, BITS, true>(s, d_slots, n, default_value, d_out, out_stride, stream)              \
             : ReadTyped<T, BITS, false>(s, d_slots, n, default_value, d_out, out_stride, stream)
  if (s.bits == 8) {
    if (type == ElemType::kF32) HPS_QROWS_TYPED(float, 8);
    if (type == ElemType::kF16) HPS_QROWS_TYPED(_Float16, 8);
    HPS_QROWS_TYPED(__bf16, 8);
  }
  if (type == ElemType::kF32) HPS_QROWS_TYPED(float, 4);
  if (type == ElemType::kF16) HPS_QROWS_TYPED(_Float16, 4);
  HPS_QROWS_TYPED(__bf16, 4);
#undef HPS_QROWS_TYPED
}

}  // namespace hps
