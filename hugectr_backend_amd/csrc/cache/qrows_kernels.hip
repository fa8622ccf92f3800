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
// multiply-add gives exactly: rounding a nonzero number never changes its sign, and from 2^-100 on the difference is a multiple of 2^-131 at
// least or of the value's own last place, which denormals (they are on) hold.
//
// A slot that is named twice in one call keeps its LAST row, whole.  Three ways, by the number of rows:
//   few (kScan)     one launch: a block keeps its rows' slots in a table in LDS and reads the slots behind them, which leave the last
//                   position of each there
//   some (kClaim)   a first kernel leaves the highest position in claim[slot] with one atomic maximum per row; a row is written where its
//                   own position is there, and puts the zero back, so the array is clear for the next call (or a graph's next replay)
//   many (kStamp)   1.7 M atomics are 65 us, 1.7 M plain stores 23: a first kernel stores the positions into stamp[slot], any one of a
//                   slot's stays.  A row whose own is there is written; a LATER one (there are none unless a slot repeats) raises the
//                   stamp by an atomic maximum with the top bit set and goes on a list, and a last kernel writes the listed rows that
//                   still hold their slot's stamp.  Every slot's stamp is stored anew by every call: nothing has to be cleared.
#include <hip/hip_bfloat16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../common/launch.h"
#include "qrows.h"

namespace hps {

typedef uint32_t u2q __attribute__((ext_vector_type(2), aligned(4)));   // (codes are 4-byte aligned)

constexpr int kQThreads = 256;
constexpr uint64_t kQRowsPerLaunch = 1ull << 24;   // a launch holds at most 2^32 threads; a row takes up to 64
// calls of kScan against kClaim, rows of 16: 1,024 rows 5.1 us, 2,048 5.6 against 8.0, 4,096 8.7 against 8.0
constexpr uint64_t kScanRows = 2048;
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
                                                                    uint32_t* __restrict__ claim) {
  const uint64_t i = (uint64_t)blockIdx.x * kQThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t slot = slots[i];
  if (slot >= 0 && (uint64_t)slot < num_rows) atomicMax(&claim[slot], (uint32_t)i + 1u);
}

template <typename T, int BITS>
constexpr int kQWriteV = (sizeof(T) == 2 || BITS == 4) ? 8 : 4;

__global__ __launch_bounds__(kQThreads) void hps_qrows_stamp_kernel(const int64_t* __restrict__ slots, uint64_t n, uint64_t num_rows,
                                                                    uint32_t* __restrict__ stamp, uint32_t* __restrict__ listed) {
  const uint64_t i = (uint64_t)blockIdx.x * kQThreads + threadIdx.x;
  if (i == 0) listed[0] = 0;
  if (i >= n) return;
  const int64_t slot = slots[i];
  if (slot >= 0 && (uint64_t)slot < num_rows) stamp[slot] = (uint32_t)i + 1u;
}

// The last position + 1 that names `slot` (of this team's row, at position mine - 1; `insert` on the lane that enters it), for a block whose
// per_block teams hold consecutive rows.  Eight times as many places as rows: a wave searches as long as its unluckiest lane.
__device__ __forceinline__ uint32_t last_of(const int64_t* __restrict__ slots, uint64_t n, uint64_t num_rows, uint32_t per_block, int64_t slot,
                                            bool insert, uint32_t mine, uint32_t lane) {
  constexpr unsigned long long kFree = ~0ull;   // (no slot: the highest bit)
  __shared__ unsigned long long key[8 * kQThreads];
  __shared__ uint32_t last[8 * kQThreads];
  const uint32_t mask = 8 * per_block - 1;
  auto place = [&](int64_t k) { return (uint32_t)(((uint64_t)k * 0x9E3779B97F4A7C15ull) >> 40) & mask; };
  for (uint32_t i = threadIdx.x; i <= mask; i += kQThreads) {
    key[i] = kFree;
    last[i] = 0;
  }
  __syncthreads();
  uint32_t at = place(slot);
  if (insert) {
    for (;;) {
      const unsigned long long was = atomicCAS(&key[at], kFree, (unsigned long long)slot);
      if (was == kFree || was == (unsigned long long)slot) break;
      at = (at + 1) & mask;
    }
    atomicMax(&last[at], mine);
  }
  __syncthreads();
  constexpr int kEach = 4;
  for (uint64_t base = (uint64_t)(blockIdx.x + 1) * per_block; base < n; base += kQThreads * kEach) {
    int64_t k[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint64_t j = base + (uint64_t)e * kQThreads + threadIdx.x;
      k[e] = j < n ? slots[j] : -1;
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (k[e] < 0 || (uint64_t)k[e] >= num_rows) continue;
      for (uint32_t p = place(k[e]); key[p] != kFree; p = (p + 1) & mask)
        if (key[p] == (unsigned long long)k[e]) {
          atomicMax(&last[p], (uint32_t)(base + (uint64_t)e * kQThreads + threadIdx.x) + 1u);
          break;
        }
    }
  }
  __syncthreads();
  // the place belongs to the team's lane 0; the teams' lanes share a wave
  const uint32_t found = insert ? last[at] : 0u;
  return (uint32_t)__shfl((int)found, (int)((threadIdx.x & 63) - lane), 64);
}

constexpr int kScan = 0, kClaim = 1, kStamp = 2, kListed = 3;
constexpr uint32_t kRaised = 0x80000000u;

template <typename T, int BITS, bool VEC, int NCH, int U, int MODE>
__global__ __launch_bounds__(kQThreads) void hps_qrows_write_kernel(QRowsDesc s, const T* rows, uint64_t row_stride,
                                                                    const int64_t* __restrict__ slots, uint64_t first, uint64_t n, T* held,
                                                                    uint64_t held_stride, uint32_t team_log, uint32_t reduce_lanes) {
  constexpr int V = kQWriteV<T, BITS>;
  constexpr float kLevels = BITS == 8 ? 127.f : 7.f;
  constexpr int kKeep = NCH ? NCH : 1;     // chunks of V values per lane that stay in registers; NCH = 0: wider rows are read twice
  const uint32_t team = 1u << team_log, lane = threadIdx.x & (team - 1), per_block = kQThreads >> team_log;
  const uint32_t dim = s.dim, chunks = (dim + V - 1) / V, rounds = (chunks + team - 1) >> team_log;
  const bool whole = s.groups == 1;
  uint64_t at0 = first + (uint64_t)blockIdx.x * (per_block * U) + (threadIdx.x >> team_log), end = n, step = 0;
  bool by_list = false;
  if constexpr (MODE == kListed) {   // the listed rows, or, where the list was too short, all of them
    const uint32_t count = s.listed[0];
    by_list = count <= kQRowsListed;
    end = by_list ? count : n;
    at0 = (uint64_t)blockIdx.x * per_block + (threadIdx.x >> team_log);
    step = (uint64_t)gridDim.x * per_block;
  }
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
  for (;;) {
    uint64_t row[U];
    int64_t slot[U];
    bool live[U], mine[U];           // (a team is live or not as a whole; the wave's exchanges need every lane)
    float x[U][kKeep][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t at = at0 + (uint64_t)u * per_block;
      live[u] = at < end;
      row[u] = live[u] ? (by_list ? s.listed[1 + at] : at) : 0;
      slot[u] = live[u] ? slots[row[u]] : -1;
      mine[u] = slot[u] >= 0 && (uint64_t)slot[u] < s.num_rows;
    }
    if constexpr (NCH != 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          const uint32_t c = lane + ((uint32_t)k << team_log);
#pragma unroll
          for (int v = 0; v < V; ++v) x[u][k][v] = 0.f;
          if (live[u] && c < chunks) load_values<T, V, VEC>(rows + row[u] * row_stride, c * V, dim, x[u][k]);
        }
    }
    uint32_t seen[U];
    if constexpr (MODE != kScan) {
#pragma unroll
      for (int u = 0; u < U; ++u) seen[u] = mine[u] ? (MODE == kClaim ? s.claim : s.stamp)[slot[u]] : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t me = (uint32_t)row[u] + 1u;
      if constexpr (MODE == kScan) {
        const uint32_t last = last_of(slots, n, s.num_rows, per_block, slot[u], mine[u] && lane == 0, me, lane);   // (the whole block)
        mine[u] = mine[u] && last == me;
      } else if constexpr (MODE == kListed) {
        mine[u] = mine[u] && seen[u] == (kRaised | me);
      } else {
        if (MODE == kStamp && mine[u] && lane == 0 && me > (seen[u] & ~kRaised)) {
          atomicMax(&s.stamp[slot[u]], kRaised | me);
          const uint32_t k = atomicAdd(&s.listed[0], 1u);
          if (k < kQRowsListed) s.listed[1 + k] = (uint32_t)row[u];
        }
        mine[u] = mine[u] && seen[u] == me;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* from = rows + row[u] * row_stride;
      uint8_t* codes = s.codes + (mine[u] ? (uint64_t)slot[u] : 0) * s.row_bytes;
      float* scales = s.scales + (mine[u] ? (uint64_t)slot[u] : 0) * s.groups;
      T* out = held ? held + row[u] * held_stride : nullptr;
      uint32_t top = 0;
      if (whole) {
        if constexpr (NCH != 0) {
#pragma unroll
          for (int k = 0; k < NCH; ++k) {
            const uint32_t t = top_of(x[u][k]);
            top = t > top ? t : top;
          }
        } else {
          for (uint32_t c = lane; live[u] && c < chunks; c += team) {
            load_values<T, V, VEC>(from, c * V, dim, x[u][0]);
            const uint32_t t = top_of(x[u][0]);
            top = t > top ? t : top;
          }
        }
        top = over_lanes(top, reduce_lanes);
      }
      auto finish = [&](uint32_t c, float(&v)[V]) {   // every lane of the wave comes here (lane exchanges)
        const uint32_t m = whole ? top : over_lanes(top_of(v), reduce_lanes);
        const float a = __uint_as_float(m);
        float scale = a / kLevels;
        if (a < kQTiny) scale = 0.f;
        if (m >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
        const bool codable = scale > 0.f;
        const float inv = __builtin_amdgcn_rcpf(scale);
        if (!live[u] || c >= chunks) return;
        int q[V];
#pragma unroll
        for (int k = 0; k < V; ++k) q[k] = codable ? nearest_code(v[k], scale, inv, kLevels) : 0;
        if (mine[u]) {
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
              // (whole lines in no order go past the caches: 280 -> 270 us for 1.7 M rows of 128)
              if (s.row_bytes % 128 == 0) __builtin_nontemporal_store(w[0], dst);
              else *dst = w[0];
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
          if ((uint32_t)k < rounds) finish(lane + ((uint32_t)k << team_log), x[u][k]);
      } else {
        for (uint32_t k = 0; k < rounds; ++k) {
          const uint32_t c = lane + (k << team_log);
#pragma unroll
          for (int v = 0; v < V; ++v) x[u][0][v] = 0.f;
          if (live[u] && c < chunks) load_values<T, V, VEC>(from, c * V, dim, x[u][0]);
          finish(c, x[u][0]);
        }
      }
      if constexpr (MODE == kClaim) {
        if (mine[u] && lane == 0) s.claim[slot[u]] = 0;
      }
    }
    if constexpr (MODE != kListed) return;
    at0 += step;
    if (at0 - (threadIdx.x >> team_log) >= end) return;   // (the whole block at once)
  }
}

// U rows per team: their slots, then their codes, are on their way together
template <typename T, int BITS, bool VEC, int U>
__global__ __launch_bounds__(kQThreads) void hps_qrows_read_kernel(QRowsDesc s, const int64_t* __restrict__ slots, uint64_t first, uint64_t n,
                                                                   float default_value, T* __restrict__ out, uint64_t out_stride,
                                                                   uint32_t team_log, uint32_t group_log) {
  constexpr int V = kQWriteV<T, BITS>, W = BITS == 8 ? V / 4 : 1;
  const uint32_t team = 1u << team_log, lane = threadIdx.x & (team - 1), per_block = kQThreads >> team_log;
  const uint64_t i0 = first + (uint64_t)blockIdx.x * (per_block * U) + (threadIdx.x >> team_log);
  const uint32_t dim = s.dim, chunks = (dim + V - 1) / V, words = s.row_bytes / 4;
  uint64_t at[U];
  bool inside[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = i0 + (uint64_t)u * per_block;
    const int64_t slot = i < n ? slots[i] : -1;
    inside[u] = slot >= 0 && (uint64_t)slot < s.num_rows;
    at[u] = inside[u] ? (uint64_t)slot : 0;
  }
  for (uint32_t c = lane; c < chunks; c += team) {
    uint32_t w[U][W];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[u][k] = 0;
      scale[u] = 0.f;
      if (inside[u]) {
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(s.codes + at[u] * s.row_bytes) + c * W;
        scale[u] = s.scales[at[u] * s.groups + (s.groups == 1 ? 0 : (c * V) >> group_log)];
        if constexpr (W == 1) {
          w[u][0] = codes[0];
        } else if (words % 2 == 0) {
          const u2q p = *reinterpret_cast<const u2q*>(codes);
          w[u][0] = p[0], w[u][1] = p[1];
        } else {
          w[u][0] = codes[0];
          if (2 * c + 1 < words) w[u][1] = codes[1];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t i = i0 + (uint64_t)u * per_block;
      if (i >= n) continue;
      float y[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int code = BITS == 8 ? (int)(w[u][k / 4] << (24 - 8 * (k % 4))) >> 24 : (int)(w[u][0] << (28 - 4 * k)) >> 28;
        y[k] = inside[u] ? (float)code * scale[u] : default_value;
      }
      store_values<T, V, VEC>(out + i * out_stride, c * V, dim, y);
    }
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

// kStamp costs one launch more than kClaim (5 us in all) and saves 25 us a million rows
constexpr uint64_t kStampRows = 1ull << 18;
// the last pass: 1.7 M rows, 17,000 of them listed, 256 / 512 / 1,024 / 2,048 blocks 259.7 / 255.3 / 253.3 / 252.5 us, none listed 246.8 - 247.1
constexpr uint32_t kListBlocks = 1024;

template <typename T, int BITS, bool VEC, int NCH>
hipError_t WriteKept(const QRowsDesc& s, const T* rows, uint64_t row_stride, const int64_t* slots, uint64_t n, T* held, uint64_t held_stride,
                     const TeamShape& t, hipStream_t stream) {
  // rows of a team that are on their way together: 1.7 M rows of 128 fp32 in 8 bits 1 / 2 / 4: 313 / 266 / 250 us, fp16 194 / 175 / 181
  constexpr int kU = NCH != 1 ? 1 : kQWriteV<T, BITS> == 4 ? 4 : 2;
  auto blocks = [&](uint64_t rows_of, uint64_t each) {
    const uint64_t per = (uint64_t)(kQThreads >> t.team_log) * each;
    return (uint32_t)((rows_of + per - 1) / per);
  };
  auto flat = [&](uint64_t each) { return (uint32_t)((n + (uint64_t)kQThreads * each - 1) / ((uint64_t)kQThreads * each)); };
  hipError_t e;
  if (n <= kScanRows) {
    return Launch(hps_qrows_write_kernel<T, BITS, VEC, NCH, 1, kScan>, blocks(n, 1), kQThreads, stream, s, rows, row_stride, slots, 0, n, held,
                  held_stride, t.team_log, t.reduce_lanes);
  }
  // (in place, a row that the last kernel writes again would be read after it was replaced)
  if (n < kStampRows || (const void*)held == (const void*)rows) {
    e = Launch(hps_qrows_claim_kernel, flat(1), kQThreads, stream, slots, n, s.num_rows, s.claim);
    for (uint64_t first = 0; e == hipSuccess && first < n; first += kQRowsPerLaunch) {
      const uint64_t end = first + kQRowsPerLaunch < n ? first + kQRowsPerLaunch : n;
      e = Launch(hps_qrows_write_kernel<T, BITS, VEC, NCH, 1, kClaim>, blocks(end - first, 1), kQThreads, stream, s, rows, row_stride, slots, first,
                 end, held, held_stride, t.team_log, t.reduce_lanes);
    }
    return e;
  }
  e = Launch(hps_qrows_stamp_kernel, flat(1), kQThreads, stream, slots, n, s.num_rows, s.stamp, s.listed);
  for (uint64_t first = 0; e == hipSuccess && first < n; first += kQRowsPerLaunch) {
    const uint64_t end = first + kQRowsPerLaunch < n ? first + kQRowsPerLaunch : n;
    e = Launch(hps_qrows_write_kernel<T, BITS, VEC, NCH, kU, kStamp>, blocks(end - first, kU), kQThreads, stream, s, rows, row_stride, slots, first,
               end, held, held_stride, t.team_log, t.reduce_lanes);
  }
  if (e != hipSuccess) return e;
  return Launch(hps_qrows_write_kernel<T, BITS, VEC, NCH, 1, kListed>, kListBlocks, kQThreads, stream, s, rows, row_stride, slots, 0, n, (T*)nullptr,
                0, t.team_log, t.reduce_lanes);
}

template <typename T, int BITS, bool VEC>
hipError_t WriteTyped(const QRowsDesc& s, const void* rows, uint64_t row_stride, const int64_t* slots, uint64_t n, void* held,
                      uint64_t held_stride, hipStream_t stream) {
  const TeamShape t = TeamOf(s.dim, kQWriteV<T, BITS>, s.group, s.groups);
  if (t.rounds == 1) return WriteKept<T, BITS, VEC, 1>(s, (const T*)rows, row_stride, slots, n, (T*)held, held_stride, t, stream);
  if (t.rounds <= 4) return WriteKept<T, BITS, VEC, 4>(s, (const T*)rows, row_stride, slots, n, (T*)held, held_stride, t, stream);
  return WriteKept<T, BITS, VEC, 0>(s, (const T*)rows, row_stride, slots, n, (T*)held, held_stride, t, stream);
}

template <typename T, int BITS, bool VEC>
hipError_t ReadTyped(const QRowsDesc& s, const int64_t* slots, uint64_t n, float default_value, void* out, uint64_t out_stride,
                     hipStream_t stream) {
  const TeamShape t = TeamOf(s.dim, kQWriteV<T, BITS>, s.group, s.groups);
  // Four rows of a team at once: 1.7 M rows of 128 in 8 bits to fp32 311 -> 238 us.  Not where a lane writes 32 bytes (4 bits to fp32; one row /
  // four: a scale per 16 values 225 / 271 us, per 64 252 / 261, per row 318 / 293): its rows are long enough as they are.
  constexpr int kU = kQWriteV<T, BITS> * sizeof(T) <= 16 ? 4 : 1;
  uint32_t group_log = 0;
  while (s.groups > 1 && (1u << group_log) < s.group) ++group_log;
  hipError_t e = hipSuccess;
  for (uint64_t first = 0; e == hipSuccess && first < n; first += kQRowsPerLaunch) {
    const uint64_t end = first + kQRowsPerLaunch < n ? first + kQRowsPerLaunch : n;
    const uint64_t per_block = (uint64_t)(kQThreads >> t.team_log) * kU;
    const uint32_t blocks = (uint32_t)((end - first + per_block - 1) / per_block);
    e = Launch(hps_qrows_read_kernel<T, BITS, VEC, kU>, blocks, kQThreads, stream, s, slots, first, end, default_value, (T*)out, out_stride, t.team_log,
               group_log);
  }
  return e;
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
