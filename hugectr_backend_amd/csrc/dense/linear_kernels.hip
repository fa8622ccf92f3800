// y = act(x W + b) * mul + residual on the matrix cores: operands in f16 or bf16, products exact, sums in fp32, ONE rounding at the
// end.  One layer, or one layer per expert over ragged runs of rows.
//
// Fragments (v_mfma_f32_16x16x32): the WEIGHTS are the A operand and the rows of x the B operand, so an accumulator holds the
// transposed tile: lane l has row (of x) l & 15 and the four columns 4 * (l >> 4) + reg.  The packing permutes the weights' columns
// so that a PAIR of fragments covers 32 columns and lane group g = l >> 4 has the eight CONSECUTIVE columns 8 g + 4 t + reg (t = 0, 1
// the fragment of the pair): the epilogue reads mul and residual and writes the output 16 bytes at a time straight from the
// accumulators, with no pass through LDS.
//   packed weights: [expert][pair of 32 columns][K step of 32][t][lane][8]: one fragment = one contiguous 1-KB read; columns beyond N
//   and k beyond K are zero.
#include <hip/hip_bfloat16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear.h"

namespace hps {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float acc4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4l __attribute__((ext_vector_type(4)));

template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef half8 type;
  static __device__ __forceinline__ acc4 mfma(half8 a, half8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<__bf16> {
  typedef bhalf8 type;
  static __device__ __forceinline__ acc4 mfma(bhalf8 a, bhalf8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// 16 bytes from or to an address that is only aligned to an element: rows may start anywhere (odd widths and strides)
__device__ __forceinline__ u4l load16(const void* p) {
  u4l v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void store16(void* p, u4l v) { __builtin_memcpy(p, &v, 16); }

// erf by Abramowitz and Stegun 7.1.26 (|error| <= 1.5e-7): one exponential and a polynomial of degree five
__device__ __forceinline__ float erf_as(float x) {
  const float a = fabsf(x), t = 1.f / fmaf(0.3275911f, a, 1.f);
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  return copysignf(fmaf(-p, __expf(-a * a), 1.f), x);
}

__device__ __forceinline__ float activate(float y, int act) {
  switch (act) {
    case (int)Activation::kRelu: return y > 0.f ? y : (y != y ? y : 0.f);
    case (int)Activation::kGelu: return 0.5f * y * (1.f + erf_as(y * 0.70710678f));
    case (int)Activation::kSilu: return y / (1.f + __expf(-y));
    case (int)Activation::kSigmoid: return 1.f / (1.f + __expf(-y));
    default: return y;
  }
}

// ------------------------------------------------------------------------------------------------------------
// Which rows a tile of `BM` positions covers.  Without offsets: the positions [tile * BM, ...).  With offsets every expert's run is cut
// into tiles of its own; a block finds its tile with a scan over the experts (64 a step: running maximum of the clamped offsets, so
// that offsets that descend or leave [0, rows] only make runs empty, then a prefix sum of the runs' tile counts).  Tiles behind the last
// expert's cover the positions of no run.
// ------------------------------------------------------------------------------------------------------------
struct RowTile {
  int kind;           // 0: nothing, 1: rows of `expert`, 2: positions of no run
  uint32_t expert, first, count;
};

template <int BM>
__device__ __forceinline__ RowTile find_tile(const LinearDesc& d, const LinearArgs& a, uint32_t tile, int lane) {
  const uint32_t rows = (uint32_t)a.rows;
  if (!a.offsets) {
    const uint32_t first = tile * BM;
    if (first >= rows) return {0, 0, 0, 0};
    return {1, 0, first, min((uint32_t)BM, rows - first)};
  }
  auto clamped = [&](uint32_t e) { return (uint32_t)min(max(a.offsets[e], 0), (int)rows); };
  const uint32_t head = clamped(0);
  uint32_t end = head, before = 0;
  for (uint32_t base = 0; base < d.experts; base += 64) {
    const uint32_t e = base + (uint32_t)lane;
    uint32_t v = e < d.experts ? clamped(e + 1) : 0u;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)v, s, 64);
      if (lane >= s) v = max(v, o);
    }
    v = max(v, end);
    uint32_t start = (uint32_t)__shfl_up((int)v, 1, 64);
    if (lane == 0) start = end;
    const uint32_t count = e < d.experts ? v - start : 0u, tiles = (count + BM - 1) / BM;
    uint32_t sum = tiles;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t o = (uint32_t)__shfl_up((int)sum, s, 64);
      if (lane >= s) sum += o;
    }
    const uint64_t hit = __ballot(tile >= before + sum - tiles && tile < before + sum);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      const uint32_t s0 = (uint32_t)__shfl((int)start, src, 64), c0 = (uint32_t)__shfl((int)count, src, 64);
      const uint32_t t0 = (uint32_t)__shfl((int)(before + sum - tiles), src, 64);
      const uint32_t skip = (tile - t0) * BM;
      return {1, base + (uint32_t)src, s0 + skip, min((uint32_t)BM, c0 - skip)};
    }
    before += (uint32_t)__shfl((int)sum, 63, 64);
    end = (uint32_t)__shfl((int)v, 63, 64);
  }
  if (!a.zero_rest) return {0, 0, 0, 0};
  const uint32_t t = tile - before, head_tiles = (head + BM - 1) / BM;
  if (t < head_tiles) return {2, 0, t * BM, min((uint32_t)BM, head - t * BM)};
  const uint64_t first = (uint64_t)end + (uint64_t)(t - head_tiles) * BM;
  if (first >= rows) return {0, 0, 0, 0};
  return {2, 0, (uint32_t)first, min((uint32_t)BM, rows - (uint32_t)first)};
}

// tiles of every expert's runs and of the rest, at most
static uint64_t RowTiles(const LinearDesc& d, const LinearArgs& a, uint32_t BM) {
  return a.offsets ? a.rows / BM + d.experts + 2 : (a.rows + BM - 1) / BM;
}

// Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous range of tiles, so that tiles that share rows or weights share its L2
__device__ __forceinline__ uint32_t xcd_order(uint32_t id, uint32_t total) {
  const uint32_t per = total / 8, more = total % 8, xcd = id % 8, at = id / 8;
  return xcd * per + min(xcd, more) + at;
}

// output row of a position, or -1
__device__ __forceinline__ int64_t out_row(const LinearArgs& a, uint32_t pos) {
  const int64_t r = a.rows_out ? (int64_t)a.rows_out[pos] : (int64_t)pos;
  return r >= 0 && (uint64_t)r < a.out_rows ? r : -1;
}

// row of x of a position, or null (out of range: reads as zeros)
template <typename T>
__device__ __forceinline__ const T* in_row(const LinearArgs& a, uint32_t pos) {
  const int64_t r = a.rows_in ? (int64_t)a.rows_in[pos] : (int64_t)pos;
  return r >= 0 && (uint64_t)r < a.x_rows ? reinterpret_cast<const T*>(a.x) + (uint64_t)r * a.x_stride : nullptr;
}

// eight values of a row of x from column k on, zeros beyond K and for no row
template <typename T>
__device__ __forceinline__ u4l load_x(const T* row, uint32_t k, uint32_t K) {
  u4l v = {0, 0, 0, 0};
  if (row == nullptr) return v;
  if (k + 8 <= K) return load16(row + k);
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) v[j / 2] |= (uint32_t)p[k + j] << (16 * (j % 2));
  return v;
}

// the end of eight consecutive columns [n, n + 8) of one output row: y = act(acc + bias) * mul + residual, rounded once
template <typename T, typename OutT>
__device__ __forceinline__ void finish8(const LinearDesc& d, const LinearArgs& a, int64_t row, uint32_t n, const float* __restrict__ bias,
                                        float (&y)[8]) {
  if (row < 0 || n >= d.N) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = activate(y[j] + bias[j], d.act);
  const uint32_t left = d.N - n;
  if (a.mul) {
    const T* m = reinterpret_cast<const T*>(a.mul) + (uint64_t)row * a.mul_stride + n;
    T v[8];
    const u4l r = load_x<T>(m, 0, left);
    __builtin_memcpy(v, &r, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= (float)v[j];
  }
  if (a.residual) {
    const T* m = reinterpret_cast<const T*>(a.residual) + (uint64_t)row * a.residual_stride + n;
    T v[8];
    const u4l r = load_x<T>(m, 0, left);
    __builtin_memcpy(v, &r, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] += (float)v[j];
  }
  OutT* o = reinterpret_cast<OutT*>(a.out) + (uint64_t)row * a.out_stride + n;
  if (left >= 8) {
    OutT v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (OutT)y[j];
#pragma unroll
    for (int j = 0; j < (int)sizeof(OutT) / 2; ++j) {
      u4l r;
      __builtin_memcpy(&r, reinterpret_cast<const char*>(v) + 16 * j, 16);
      store16(reinterpret_cast<char*>(o) + 16 * j, r);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((uint32_t)j < left) o[j] = (OutT)y[j];
  }
}

template <typename OutT>
__device__ __forceinline__ void zero_rows(const LinearDesc& d, const LinearArgs& a, const RowTile& t, uint32_t n0, uint32_t n1) {
  n1 = min(n1, d.N);
  for (uint32_t r = 0; r < t.count; ++r) {
    const int64_t row = out_row(a, t.first + r);
    if (row < 0) continue;
    OutT* o = reinterpret_cast<OutT*>(a.out) + (uint64_t)row * a.out_stride;
    for (uint32_t n = n0 + threadIdx.x; n < n1; n += blockDim.x) o[n] = (OutT)0.f;
  }
}

// ------------------------------------------------------------------------------------------------------------
// Tiles of BM rows x BN columns, WM x WN waves, K in steps of 64.  Both operands go through LDS, double-buffered: the step after next
// is on its way into registers while the step at hand is multiplied, the next one is written to the other buffer.  Rows of x are 128
// bytes of LDS, their 16-byte chunks swapped by chunk ^ (row & 7), so that the fragments' reads (16 rows at one chunk) are free of bank
// conflicts; weight fragments lie in LDS as in memory.
// ------------------------------------------------------------------------------------------------------------
template <typename T, typename OutT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void hps_linear_tile_kernel(LinearDesc d, LinearArgs a, uint32_t m_tiles, uint32_t n_tiles) {
  constexpr int kThreads = 64 * WM * WN;
  constexpr int FM = BM / WM / 16, FP = BN / WN / 32;     // row fragments and column pairs of a wave
  constexpr int XC = BM * 8 / kThreads, WC = BN * 8 / kThreads;   // 16-byte chunks of a step per thread
  static_assert(XC * kThreads == BM * 8 && WC * kThreads == BN * 8 && FM >= 1 && FP >= 1, "whole chunks");
  typedef typename Frag<T>::type frag;
  __shared__ __attribute__((aligned(16))) u4l lds_x[2][BM * 8];
  __shared__ __attribute__((aligned(16))) u4l lds_w[2][BN * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t id = xcd_order(blockIdx.x, m_tiles * n_tiles);
  const uint32_t nt = id % n_tiles;
  const RowTile t = find_tile<BM>(d, a, id / n_tiles, lane);
  if (t.kind == 0) return;
  if (t.kind == 2) return zero_rows<OutT>(d, a, t, nt * BN, nt * BN + BN);

  const T* xrow[XC];
#pragma unroll
  for (int i = 0; i < XC; ++i) {
    const uint32_t r = (uint32_t)(tid >> 3) + i * (kThreads / 8);
    xrow[i] = r < t.count ? in_row<T>(a, t.first + r) : nullptr;
  }
  const u4l* wbase = reinterpret_cast<const u4l*>(d.w) + (uint64_t)t.expert * d.npairs * d.ksteps * 128;
  const u4l* wsrc[WC];
#pragma unroll
  for (int i = 0; i < WC; ++i) {
    const uint32_t q = tid + i * kThreads, p = min(nt * (BN / 32) + (q >> 8), d.npairs - 1);
    wsrc[i] = wbase + (uint64_t)p * d.ksteps * 128 + (q & 255);
  }
  u4l rx[XC], rw[WC];
  const uint32_t steps = (d.ksteps + 1) / 2;
  auto fetch = [&](uint32_t s) {
#pragma unroll
    for (int i = 0; i < XC; ++i) rx[i] = load_x<T>(xrow[i], s * 64 + (tid & 7) * 8, d.K);
#pragma unroll
    for (int i = 0; i < WC; ++i) {
      const uint32_t q = tid + i * kThreads;
      rw[i] = u4l{0, 0, 0, 0};
      if (2 * s + ((q >> 7) & 1) < d.ksteps) rw[i] = wsrc[i][(uint64_t)s * 256];
    }
  };
  auto keep = [&](int b) {
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const uint32_t r = (uint32_t)(tid >> 3) + i * (kThreads / 8);
      lds_x[b][r * 8 + ((tid & 7) ^ (r & 7))] = rx[i];
    }
#pragma unroll
    for (int i = 0; i < WC; ++i) lds_w[b][tid + i * kThreads] = rw[i];
  };
  const int wm = wave / WN, wn = wave % WN;
  acc4 acc[FP][2][FM];
#pragma unroll
  for (int p = 0; p < FP; ++p)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < FM; ++m) acc[p][h][m] = acc4{0.f, 0.f, 0.f, 0.f};

  fetch(0);
  keep(0);
  if (steps > 1) fetch(1);
  __syncthreads();
  for (uint32_t s = 0; s < steps; ++s) {
    const int b = (int)(s & 1);
    if (s + 1 < steps) keep(b ^ 1);      // (the other buffer was last read before the previous barrier)
    if (s + 2 < steps) fetch(s + 2);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      frag fw[FP][2], fx[FM];
#pragma unroll
      for (int p = 0; p < FP; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          fw[p][h] = __builtin_bit_cast(frag, lds_w[b][(wn * FP + p) * 256 + ks * 128 + h * 64 + lane]);
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        const int r = (wm * FM + m) * 16 + (lane & 15);
        fx[m] = __builtin_bit_cast(frag, lds_x[b][r * 8 + ((ks * 4 + (lane >> 4)) ^ (r & 7))]);
      }
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int p = 0; p < FP; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[p][h][m] = Frag<T>::mfma(fw[p][h], fx[m], acc[p][h][m]);
    }
    __syncthreads();
  }
  const float* bias = d.bias + (uint64_t)t.expert * d.npairs * 32;
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const uint32_t r = (wm * FM + m) * 16 + (lane & 15);
    const int64_t row = r < t.count ? out_row(a, t.first + r) : -1;
#pragma unroll
    for (int p = 0; p < FP; ++p) {
      const uint32_t n = nt * BN + (wn * FP + p) * 32 + (lane >> 4) * 8;
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = acc[p][j / 4][m][j % 4];
      finish8<T, OutT>(d, a, row, n, bias + n, y);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// Few rows: bound by the weights' bytes and by latency.  A block takes one pair of 32 columns and up to 16 * MF rows; its NW waves
// split K, each reads its weight fragments and the rows' chunks straight from memory (U steps on their way at once), and the partial
// sums meet in LDS, added in the waves' order.
// ------------------------------------------------------------------------------------------------------------
template <typename T, typename OutT, int MF, int NW>
__global__ __launch_bounds__(64 * NW) void hps_linear_rows_kernel(LinearDesc d, LinearArgs a, uint32_t m_tiles) {
  constexpr int U = MF >= 4 ? 2 : 4;
  typedef typename Frag<T>::type frag;
  __shared__ __attribute__((aligned(16))) acc4 part[NW][2 * MF][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t id = xcd_order(blockIdx.x, m_tiles * d.npairs);
  const uint32_t pair = id / m_tiles;
  const RowTile t = find_tile<16 * MF>(d, a, id % m_tiles, lane);
  if (t.kind == 0) return;
  if (t.kind == 2) return zero_rows<OutT>(d, a, t, pair * 32, pair * 32 + 32);
  const T* xrow[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const uint32_t r = m * 16 + (lane & 15);
    xrow[m] = r < t.count ? in_row<T>(a, t.first + r) : nullptr;
  }
  const u4l* w = reinterpret_cast<const u4l*>(d.w) + ((uint64_t)t.expert * d.npairs + pair) * d.ksteps * 128 + lane;
  acc4 acc[2][MF];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[h][m] = acc4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = wave; s0 < d.ksteps; s0 += NW * U) {
    u4l rw[U][2], rx[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * NW;
      rw[u][0] = rw[u][1] = u4l{0, 0, 0, 0};
      if (s < d.ksteps) {
        rw[u][0] = w[(uint64_t)s * 128];
        rw[u][1] = w[(uint64_t)s * 128 + 64];
      }
#pragma unroll
      for (int m = 0; m < MF; ++m) rx[u][m] = load_x<T>(xrow[m], s * 32 + (lane >> 4) * 8, d.K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[h][m] = Frag<T>::mfma(__builtin_bit_cast(frag, rw[u][h]), __builtin_bit_cast(frag, rx[u][m]), acc[h][m]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int m = 0; m < MF; ++m) part[wave][h * MF + m][lane] = acc[h][m];
  __syncthreads();
  const float* bias = d.bias + ((uint64_t)t.expert * d.npairs + pair) * 32;
  for (int m = wave; m < MF; m += NW) {
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] += part[v][(j / 4) * MF + m][lane][j % 4];
    const uint32_t r = m * 16 + (lane & 15), n = (lane >> 4) * 8;
    const int64_t row = r < t.count ? out_row(a, t.first + r) : -1;
    finish8<T, OutT>(d, a, row, pair * 32 + n, bias + n, y);
  }
}

// ------------------------------------------------------------------------------------------------------------
// Packing, once per layer: one thread per (expert, pair, K step, fragment, lane) gathers its eight k values of one column.
// ------------------------------------------------------------------------------------------------------------
template <typename From, typename T>
__global__ __launch_bounds__(256) void hps_linear_pack_kernel(const From* __restrict__ w, uint32_t experts, uint32_t K, uint32_t N,
                                                              uint32_t ksteps, uint32_t npairs, T* __restrict__ packed) {
  const uint64_t total = (uint64_t)experts * npairs * ksteps * 128;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint32_t lane = i & 63, h = (i >> 6) & 1;
    const uint64_t b = i >> 7;
    const uint32_t ks = (uint32_t)(b % ksteps), p = (uint32_t)(b / ksteps % npairs), e = (uint32_t)(b / ksteps / npairs);
    const uint32_t c = lane & 15, n = 32 * p + 8 * (c >> 2) + 4 * h + (c & 3), k = 32 * ks + 8 * (lane >> 4);
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = n < N && k + j < K ? (T)(float)w[((uint64_t)e * K + k + j) * N + n] : (T)0.f;
    u4l r;
    __builtin_memcpy(&r, v, 16);
    reinterpret_cast<u4l*>(packed)[i] = r;
  }
}

namespace {

template <typename T, typename OutT, int BM, int BN, int WM, int WN>
hipError_t LaunchTile(const LinearDesc& d, const LinearArgs& a, hipStream_t stream) {
  const uint64_t m_tiles = RowTiles(d, a, BM), n_tiles = (d.N + BN - 1) / BN;
  if (m_tiles * n_tiles >= (1ull << 23)) return hipErrorInvalidConfiguration;   // 512 threads each: a launch holds 2^32
  hps_linear_tile_kernel<T, OutT, BM, BN, WM, WN><<<(uint32_t)(m_tiles * n_tiles), 64 * WM * WN, 0, stream>>>(d, a, (uint32_t)m_tiles,
                                                                                                             (uint32_t)n_tiles);
  return hipGetLastError();
}

template <typename T, typename OutT, int MF, int NW>
hipError_t LaunchRows(const LinearDesc& d, const LinearArgs& a, hipStream_t stream) {
  const uint64_t m_tiles = RowTiles(d, a, 16 * MF);
  if (m_tiles * d.npairs >= (1ull << 22)) return hipErrorInvalidConfiguration;
  hps_linear_rows_kernel<T, OutT, MF, NW><<<(uint32_t)(m_tiles * d.npairs), 64 * NW, 0, stream>>>(d, a, (uint32_t)m_tiles);
  return hipGetLastError();
}

template <typename T, typename OutT>
hipError_t LaunchTyped(const LinearDesc& d, const LinearArgs& a, int cu_count, hipStream_t stream) {
  const uint64_t each = a.rows / d.experts;
  if (each <= 16) return LaunchRows<T, OutT, 1, 8>(d, a, stream);
  if (each <= 64) return LaunchRows<T, OutT, 4, 8>(d, a, stream);
  const uint64_t big = (RowTiles(d, a, 256)) * ((d.N + 255) / 256);
  if (d.N > 128 && big >= (uint64_t)cu_count) return LaunchTile<T, OutT, 256, 256, 2, 4>(d, a, stream);
  return LaunchTile<T, OutT, 128, 128, 2, 2>(d, a, stream);
}

template <typename From>
hipError_t PackFrom(const void* w, uint32_t experts, uint32_t K, uint32_t N, void* packed, ElemType to, hipStream_t stream) {
  const uint32_t ksteps = (K + 31) / 32, npairs = (N + 31) / 32;
  const uint64_t total = (uint64_t)experts * npairs * ksteps * 128;
  const uint32_t blocks = (uint32_t)((total + 255) / 256 < 65536 ? (total + 255) / 256 : 65536);
  if (to == ElemType::kF16) hps_linear_pack_kernel<From, _Float16><<<blocks, 256, 0, stream>>>((const From*)w, experts, K, N, ksteps, npairs, (_Float16*)packed);
  else hps_linear_pack_kernel<From, __bf16><<<blocks, 256, 0, stream>>>((const From*)w, experts, K, N, ksteps, npairs, (__bf16*)packed);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchLinearPack(const void* d_w, ElemType from, uint32_t experts, uint32_t K, uint32_t N, void* d_packed, ElemType to,
                            hipStream_t stream) {
  if (from == ElemType::kF32) return PackFrom<float>(d_w, experts, K, N, d_packed, to, stream);
  if (from == ElemType::kF16) return PackFrom<_Float16>(d_w, experts, K, N, d_packed, to, stream);
  return PackFrom<__bf16>(d_w, experts, K, N, d_packed, to, stream);
}

hipError_t LaunchLinear(const LinearDesc& d, const LinearArgs& a, ElemType type, ElemType out_type, int cu_count, hipStream_t stream) {
  if (type == ElemType::kF16)
    return out_type == ElemType::kF32 ? LaunchTyped<_Float16, float>(d, a, cu_count, stream)
                                      : LaunchTyped<_Float16, _Float16>(d, a, cu_count, stream);
  return out_type == ElemType::kF32 ? LaunchTyped<__bf16, float>(d, a, cu_count, stream)
                                    : LaunchTyped<__bf16, __bf16>(d, a, cu_count, stream);
}

}  // namespace hps
