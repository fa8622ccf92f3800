// Grouping of rows by expert: a stable counting sort of the positions 0 .. n-1 by ids[position] into E runs, plus one run behind them
// for the positions whose id is outside [0, E).
//
//   hps_group_rows_one     up to kOneBlockRows positions: one block does everything
//   hps_group_rows_count   ids per (expert, block of kGroupTile positions)
//   hps_group_rows_scan    one block per expert: where every block's ids of it start within its run
//   hps_group_rows_place   positions to their places; while the counts are few it sums them itself, one launch less
//
// Within a block a wave takes 64 consecutive positions; the lanes with the same id find each other with one ballot per bit of the id,
// so a position's place is start + lanes below it + earlier waves' counts: no atomics on the way, the order never varies.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../common/launch.h"
#include "linear.h"

namespace hps {

constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr uint32_t kGroupTile = kGroupThreads;
constexpr uint32_t kGroupBins = kMaxExperts + 1;   // the last one in use: ids of no expert
constexpr uint32_t kOneBlockRows = 4096;   // whole calls, one launch / two: 4,096 ids 7.3-10.2 us / 10.6-11.5, 8,192 12.2-18.2 / 10.5-11.6
constexpr uint32_t kFewTiles = 64;
constexpr uint32_t kFewCounts = 12288;     // summed by every block, or scanned: 8,500 counts 11.0 / 13.3 us, 12,300 13.1 / 13.2, 43,000 23.9 / 17.1

__device__ __forceinline__ uint32_t bin_of(int32_t id, uint32_t experts) { return id >= 0 && (uint32_t)id < experts ? (uint32_t)id : experts; }

// lanes of the wave that are live and hold the same bin
__device__ __forceinline__ uint64_t same_bin(uint32_t bin, bool live, uint32_t bits) {
  uint64_t m = __ballot(live);
  for (uint32_t b = 0; b < bits; ++b) {
    const bool one = (bin >> b) & 1;
    const uint64_t ones = __ballot(one);
    m &= one ? ones : ~ones;
  }
  return m;
}

// Exclusive prefix sums of value[0 .. count) for a whole block, count <= 2 * kGroupThreads; `carry` holds kGroupWaves words.
// Thread t gets the sums of elements 2 t and 2 t + 1 in `a` and `b`.
__device__ __forceinline__ void block_scan2(uint32_t va, uint32_t vb, uint32_t* carry, uint32_t& a, uint32_t& b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = va + vb;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)s, d, 64);
    if (lane >= d) s += o;
  }
  if (lane == 63) carry[wave] = s;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += carry[w];
  a = before + s - va - vb;
  b = a + va;
  __syncthreads();
}

// What the first `waves` waves of the tile hold of one bin: pairs of 16-bit counts are added as words (a tile has 1,024 ids)
__device__ __forceinline__ uint32_t count_of_waves(const uint16_t* counts, int waves) {
  const uint4 lo = *reinterpret_cast<const uint4*>(counts), hi = *reinterpret_cast<const uint4*>(counts + 8);
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += 2 * i + 1 < waves ? w[i] : 2 * i < waves ? w[i] & 0xffff : 0;
  return (sum & 0xffff) + (sum >> 16);
}

// Places of one tile: next[bin] is the first free place of every bin; with ADVANCE the call moves it behind the tile.
// in_wave[bin][wave]: the tile's ids.
template <bool ADVANCE>
__device__ __forceinline__ void place_tile(const int32_t* __restrict__ ids, uint64_t n, uint64_t base, uint32_t experts, uint32_t bits,
                                           uint32_t* next, uint16_t (*in_wave)[kGroupWaves], int32_t* __restrict__ order) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bins = experts + 1;
  const uint64_t at = base + threadIdx.x;
  const bool live = at < n;
  const uint32_t bin = live ? bin_of(ids[at], experts) : experts;
  for (uint32_t i = threadIdx.x; i < bins * kGroupWaves / 8; i += kGroupThreads) reinterpret_cast<uint4*>(in_wave)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const uint64_t same = same_bin(bin, live, bits);
  const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1));
  if (live && below == 0) in_wave[bin][wave] = (uint16_t)__popcll(same);
  __syncthreads();
  if (live) order[next[bin] + below + count_of_waves(in_wave[bin], wave)] = (int32_t)at;
  if constexpr (ADVANCE) {
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) next[b] += count_of_waves(in_wave[b], kGroupWaves);
    __syncthreads();
  }
}

__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_one(const int32_t* __restrict__ ids, uint32_t n, uint32_t experts,
                                                                    uint32_t bits, int32_t* __restrict__ offsets,
                                                                    int32_t* __restrict__ order) {
  __shared__ uint32_t next[kGroupBins + 1];
  __shared__ __attribute__((aligned(16))) uint16_t in_wave[kGroupBins][kGroupWaves];
  __shared__ uint32_t carry[kGroupWaves];
  const uint32_t bins = experts + 1;
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) next[b] = 0;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += kGroupThreads) atomicAdd(&next[bin_of(ids[i], experts)], 1u);
  __syncthreads();
  const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
  uint32_t a, b;
  block_scan2(i0 < bins ? next[i0] : 0, i1 < bins ? next[i1] : 0, carry, a, b);
  if (i0 < bins) {
    next[i0] = a;
    offsets[i0] = (int32_t)a;
  }
  if (i1 < bins) {
    next[i1] = b;
    offsets[i1] = (int32_t)b;
  }
  __syncthreads();
  for (uint32_t base = 0; base < n; base += kGroupTile) place_tile<true>(ids, n, base, experts, bits, next, in_wave, order);
}

__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_count(const int32_t* __restrict__ ids, uint64_t n, uint32_t experts,
                                                                      uint64_t of_bin, uint64_t of_tile, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kGroupBins];
  const uint32_t bins = experts + 1;
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) hist[b] = 0;
  __syncthreads();
  const uint64_t at = (uint64_t)blockIdx.x * kGroupTile + threadIdx.x;
  if (at < n) atomicAdd(&hist[bin_of(ids[at], experts)], 1u);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) counts[b * of_bin + blockIdx.x * of_tile] = hist[b];
}

// counts[bin][tile] becomes the tile's first place within the bin; total[bin] its sum.  One block per bin.
__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_scan(uint32_t tiles, uint32_t* __restrict__ counts,
                                                                     uint32_t* __restrict__ total) {
  __shared__ uint32_t carry[kGroupWaves];
  __shared__ uint32_t sum;
  uint32_t* c = counts + (uint64_t)blockIdx.x * tiles;
  uint32_t before = 0;
  for (uint32_t base = 0; base < tiles; base += 2 * kGroupThreads) {
    const uint32_t i0 = base + 2 * threadIdx.x, i1 = i0 + 1;
    const uint32_t va = i0 < tiles ? c[i0] : 0, vb = i1 < tiles ? c[i1] : 0;
    uint32_t a, b;
    block_scan2(va, vb, carry, a, b);
    if (i0 < tiles) c[i0] = before + a;
    if (i1 < tiles) c[i1] = before + b;
    if (threadIdx.x == kGroupThreads - 1) sum = b + vb;
    __syncthreads();
    before += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = before;
}

// SCANNED: counts[bin][tile] and total are the scan's; else counts[tile][bin] are plain and few
template <bool SCANNED>
__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_place(const int32_t* __restrict__ ids, uint64_t n, uint32_t experts,
                                                                      uint32_t bits, uint32_t tiles, const uint32_t* __restrict__ counts,
                                                                      const uint32_t* __restrict__ total, int32_t* __restrict__ offsets,
                                                                      int32_t* __restrict__ order) {
  __shared__ uint32_t next[kGroupBins + 1];
  __shared__ __attribute__((aligned(16))) uint16_t in_wave[kGroupBins][kGroupWaves];
  __shared__ uint32_t carry[kGroupWaves];
  __shared__ uint32_t sums[SCANNED ? 1 : kGroupBins + 1];
  const uint32_t bins = experts + 1;
  const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
  if constexpr (!SCANNED) {
    // counts[tile][bin]: as many threads per bin as there are bins to go round, each adds up its share of the tiles
    for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) sums[b] = next[b] = 0;
    __syncthreads();
    uint32_t width = 1;
    while (width < bins && width < kGroupThreads) width <<= 1;
    const uint32_t parts = kGroupThreads / width, part = threadIdx.x / width;
    for (uint32_t bin = threadIdx.x % width; bin < bins; bin += width) {
      uint32_t all = 0, before = 0;
#pragma unroll 8
      for (uint32_t t = part; t < tiles; t += parts) {
        const uint32_t c = counts[(uint64_t)t * bins + bin];
        all += c;
        before += t < blockIdx.x ? c : 0u;
      }
      if (all) atomicAdd(&sums[bin], all);
      if (before) atomicAdd(&next[bin], before);
    }
    __syncthreads();
  }
  auto total_of = [&](uint32_t i) { return i >= bins ? 0u : SCANNED ? total[i] : sums[i]; };
  auto before_of = [&](uint32_t i) { return SCANNED ? counts[(uint64_t)i * tiles + blockIdx.x] : next[i]; };
  uint32_t a, b;
  block_scan2(total_of(i0), total_of(i1), carry, a, b);
  if (i0 < bins) {
    next[i0] = a + before_of(i0);
    if (blockIdx.x == 0) offsets[i0] = (int32_t)a;
  }
  if (i1 < bins) {
    next[i1] = b + before_of(i1);
    if (blockIdx.x == 0) offsets[i1] = (int32_t)b;
  }
  __syncthreads();
  place_tile<false>(ids, n, (uint64_t)blockIdx.x * kGroupTile, experts, bits, next, in_wave, order);
}

uint64_t GroupRowsWorkspaceBytes(uint64_t n, uint32_t experts) {
  if (n <= kOneBlockRows) return 0;
  const uint64_t tiles = (n + kGroupTile - 1) / kGroupTile;
  return (uint64_t)(experts + 1) * (tiles + 1) * sizeof(uint32_t);
}

hipError_t LaunchGroupRows(const int32_t* d_ids, uint64_t n, uint32_t experts, int32_t* d_offsets, int32_t* d_order, void* d_workspace,
                           hipStream_t stream) {
  uint32_t bits = 0;
  while ((experts >> bits) != 0) ++bits;   // the bins are 0 .. experts
  if (n <= kOneBlockRows) {
    return Launch(hps_group_rows_one, 1, kGroupThreads, stream, d_ids, n, experts, bits, d_offsets, d_order);
  }
  const uint32_t tiles = (uint32_t)((n + kGroupTile - 1) / kGroupTile);
  uint32_t* counts = (uint32_t*)d_workspace;
  uint32_t* total = counts + (uint64_t)(experts + 1) * tiles;
  const uint64_t bins = experts + 1;
  const bool few = tiles <= kFewTiles && tiles * bins <= kFewCounts;
  hipError_t e = Launch(hps_group_rows_count, tiles, kGroupThreads, stream, d_ids, n, experts, few ? 1 : tiles, few ? bins : 1, counts);
  if (e != hipSuccess) return e;
  if (few) return Launch(hps_group_rows_place<false>, tiles, kGroupThreads, stream, d_ids, n, experts, bits, tiles, counts, total, d_offsets, d_order);
  e = Launch(hps_group_rows_scan, experts + 1, kGroupThreads, stream, tiles, counts, total);
  if (e != hipSuccess) return e;
  return Launch(hps_group_rows_place<true>, tiles, kGroupThreads, stream, d_ids, n, experts, bits, tiles, counts, total, d_offsets, d_order);
}

}  // namespace hps
