// Grouping of rows by expert: a stable counting sort of the positions 0 .. n-1 by ids[position] into E runs, plus one run behind them
// for the positions whose id is outside [0, E).
//
//   hps_group_rows_one     up to kOneBlockRows positions: one block does everything
//   hps_group_rows_count   ids per (expert, block of kGroupTile positions)
//   hps_group_rows_scan    one block per expert: where every block's ids of it start within its run
//   hps_group_rows_place   positions to their places; up to kFewTiles blocks it sums the counts itself (one launch less: 65,536 ids
//                          over 16 experts 14.9 -> 12.6 us with the call's own costs)
//
// Within a block a wave takes 64 consecutive positions; the lanes with the same id find each other with one ballot per bit of the id,
// so a position's place is start + lanes below it + earlier waves' counts: no atomics on the way, the order never varies.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear.h"

namespace hps {

constexpr int kGroupThreads = 1024;
constexpr int kGroupWaves = kGroupThreads / 64;
constexpr uint32_t kGroupTile = kGroupThreads;
constexpr uint32_t kGroupBins = kMaxExperts + 1;   // the last one in use: ids of no expert
constexpr uint32_t kOneBlockRows = 8192;
constexpr uint32_t kFewTiles = 64;                 // a wave's lanes hold one expert's counts

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

// Exclusive prefix sums of value[0 .. count) for a whole block, count <= 2 * kGroupThreads; `carry` holds 2 * kGroupWaves words.
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

// Places of one tile: next[bin] is the first free place of every bin and is advanced behind the tile.
__device__ __forceinline__ void place_tile(const int32_t* __restrict__ ids, uint64_t n, uint64_t base, uint32_t experts, uint32_t bits,
                                           uint32_t* next, uint16_t (*in_wave)[kGroupBins], int32_t* __restrict__ order) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bins = experts + 1;
  for (uint32_t i = threadIdx.x; i < bins * kGroupWaves; i += kGroupThreads) in_wave[i / bins][i % bins] = 0;
  __syncthreads();
  const uint64_t at = base + threadIdx.x;
  const bool live = at < n;
  const uint32_t bin = live ? bin_of(ids[at], experts) : experts;
  const uint64_t same = same_bin(bin, live, bits);
  const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1));
  if (live && below == 0) in_wave[wave][bin] = (uint16_t)__popcll(same);
  __syncthreads();
  if (live) {
    uint32_t p = next[bin] + below;
    for (int w = 0; w < wave; ++w) p += in_wave[w][bin];
    order[p] = (int32_t)at;
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) {
    uint32_t c = 0;
    for (int w = 0; w < kGroupWaves; ++w) c += in_wave[w][b];
    next[b] += c;
  }
  __syncthreads();
}

__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_one(const int32_t* __restrict__ ids, uint32_t n, uint32_t experts,
                                                                    uint32_t bits, int32_t* __restrict__ offsets,
                                                                    int32_t* __restrict__ order) {
  __shared__ uint32_t next[kGroupBins + 1];
  __shared__ uint16_t in_wave[kGroupWaves][kGroupBins];
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
  for (uint32_t base = 0; base < n; base += kGroupTile) place_tile(ids, n, base, experts, bits, next, in_wave, order);
}

__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_count(const int32_t* __restrict__ ids, uint64_t n, uint32_t experts,
                                                                      uint32_t tiles, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kGroupBins];
  const uint32_t bins = experts + 1;
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) hist[b] = 0;
  __syncthreads();
  const uint64_t at = (uint64_t)blockIdx.x * kGroupTile + threadIdx.x;
  if (at < n) atomicAdd(&hist[bin_of(ids[at], experts)], 1u);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kGroupThreads) counts[(uint64_t)b * tiles + blockIdx.x] = hist[b];
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

// SCANNED: counts and total are the scan's; else counts are plain and tiles <= kFewTiles
template <bool SCANNED>
__global__ __launch_bounds__(kGroupThreads) void hps_group_rows_place(const int32_t* __restrict__ ids, uint64_t n, uint32_t experts,
                                                                      uint32_t bits, uint32_t tiles, const uint32_t* __restrict__ counts,
                                                                      const uint32_t* __restrict__ total, int32_t* __restrict__ offsets,
                                                                      int32_t* __restrict__ order) {
  __shared__ uint32_t next[kGroupBins + 1];
  __shared__ uint16_t in_wave[kGroupWaves][kGroupBins];
  __shared__ uint32_t carry[kGroupWaves];
  __shared__ uint32_t sums[SCANNED ? 1 : kGroupBins + 1];
  const uint32_t bins = experts + 1;
  const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
  if constexpr (!SCANNED) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t bin = threadIdx.x >> 6; bin < bins; bin += kGroupWaves) {
      const uint32_t c = lane < tiles ? counts[(uint64_t)bin * tiles + lane] : 0;
      uint32_t all = c, before = lane < blockIdx.x ? c : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        all += (uint32_t)__shfl_xor((int)all, d, 64);
        before += (uint32_t)__shfl_xor((int)before, d, 64);
      }
      if (lane == 0) {
        sums[bin] = all;
        next[bin] = before;
      }
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
  place_tile(ids, n, (uint64_t)blockIdx.x * kGroupTile, experts, bits, next, in_wave, order);
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
    hps_group_rows_one<<<1, kGroupThreads, 0, stream>>>(d_ids, (uint32_t)n, experts, bits, d_offsets, d_order);
    return hipGetLastError();
  }
  const uint32_t tiles = (uint32_t)((n + kGroupTile - 1) / kGroupTile);
  uint32_t* counts = (uint32_t*)d_workspace;
  uint32_t* total = counts + (uint64_t)(experts + 1) * tiles;
  hps_group_rows_count<<<tiles, kGroupThreads, 0, stream>>>(d_ids, n, experts, tiles, counts);
  if (tiles <= kFewTiles) {
    hps_group_rows_place<false><<<tiles, kGroupThreads, 0, stream>>>(d_ids, n, experts, bits, tiles, counts, total, d_offsets, d_order);
    return hipGetLastError();
  }
  hps_group_rows_scan<<<experts + 1, kGroupThreads, 0, stream>>>(tiles, counts, total);
  hps_group_rows_place<true><<<tiles, kGroupThreads, 0, stream>>>(d_ids, n, experts, bits, tiles, counts, total, d_offsets, d_order);
  return hipGetLastError();
}

}  // namespace hps
