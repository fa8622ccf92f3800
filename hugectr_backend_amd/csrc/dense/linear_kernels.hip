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

#include "../common/launch.h"
#include "linear.h"

namespace hps {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float acc4 __attribute__((ext_vector_type(4)));
typedef float acc8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4l __attribute__((ext_vector_type(4)));
typedef uint32_t u8l __attribute__((ext_vector_type(8)));

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

// The same with accesses on 4 bytes alone: an access at an odd multiple of 2 bytes costs more than twice an aligned one (100 rows through
// 3,456 -> 3,456, rows 3,457 apart: 46.5 -> 23.8 us; 64 through 1,024 -> 1,024 5.9 -> 4.0).  The words that hold the first and the last of the
// values are the allocation's.
__device__ __forceinline__ u4l load16_odd(const void* p) {
  const uintptr_t at = (uintptr_t)p, base = at & ~(uintptr_t)3;
  const uint32_t shift = (uint32_t)(at & 2) * 8;
  typedef u4l u4l_words __attribute__((aligned(4)));
  const u4l v = *reinterpret_cast<const u4l_words*>(base);
  const uint32_t next = *reinterpret_cast<const uint32_t*>(base + 12 + 2 * (at & 2));
  return u4l{__builtin_amdgcn_alignbit(v[1], v[0], shift), __builtin_amdgcn_alignbit(v[2], v[1], shift),
             __builtin_amdgcn_alignbit(v[3], v[2], shift), __builtin_amdgcn_alignbit(next, v[3], shift)};
}

// The first `left` of eight values (all of them from 8 on), the others zero: 4 + 2 + 1 of them, nothing beyond is touched.  What is
// loaded or stored is picked by selects alone: as a chain of branches the compiler left the case of seven values unset.
__device__ __forceinline__ u4l load_halves(const void* p, uint32_t left) {
  if (left >= 8) return load16(p);
  const char* c = reinterpret_cast<const char*>(p);
  uint32_t four[2] = {0, 0}, two = 0, one = 0;
  if (left & 4) __builtin_memcpy(four, c, 8);
  if (left & 2) __builtin_memcpy(&two, c + 2 * (left & 4), 4);
  if (left & 1) {
    uint16_t h;
    __builtin_memcpy(&h, c + 2 * (left & 6), 2);
    one = h;
  }
  // word j has values 2 j and 2 j + 1
  u4l v = {four[0], four[1], 0, 0};
  v[0] |= left & 4 ? 0u : two;
  v[2] |= left & 4 ? two : 0u;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) v[j] |= (left >> 1) == j ? one : 0u;
  return v;
}

// the first `left` of eight values, of 2 or of 4 bytes
__device__ __forceinline__ void store_halves(void* p, u4l v, uint32_t left) {
  if (left >= 8) return store16(p, v);
  char* c = reinterpret_cast<char*>(p);
  uint32_t two = left & 4 ? v[2] : v[0], one = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) one |= (left >> 1) == j ? v[j] : 0u;
  const uint32_t four[2] = {v[0], v[1]};
  const uint16_t h = (uint16_t)one;
  if (left & 4) __builtin_memcpy(c, four, 8);
  if (left & 2) __builtin_memcpy(c + 2 * (left & 4), &two, 4);
  if (left & 1) __builtin_memcpy(c + 2 * (left & 6), &h, 2);
}

__device__ __forceinline__ void store_words(void* p, u8l v, uint32_t left) {
  char* c = reinterpret_cast<char*>(p);
  if (left >= 8) {
    store16(c, u4l{v[0], v[1], v[2], v[3]});
    return store16(c + 16, u4l{v[4], v[5], v[6], v[7]});
  }
  const uint32_t two[2] = {left & 4 ? v[4] : v[0], left & 4 ? v[5] : v[1]};
  uint32_t one = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) one |= (left >> 1) == j ? v[2 * j] : 0u;
  if (left & 4) store16(c, u4l{v[0], v[1], v[2], v[3]});
  if (left & 2) __builtin_memcpy(c + 4 * (left & 4), two, 8);
  if (left & 1) __builtin_memcpy(c + 4 * (left & 6), &one, 4);
}

// erfc(a / sqrt 2) / 2 for a >= 0: the Chebyshev fit of Numerical Recipes (erfcc, relative error 1.1e-7 everywhere), its argument, the exponential's
// base and the half taken into the coefficients.  Relative, because gelu's negative tail is y * erfc(-y / sqrt 2) / 2: from an error function
// that is good to 1.5e-7 of one the value at -5 was off by a quarter of itself.
__device__ __forceinline__ float normal_tail(float a) {
  const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.353553391f, 1.f));
  float p = fmaf(t, 0.246517298f, -1.18611495f);
  p = fmaf(t, p, 2.14747446f);
  p = fmaf(t, p, -1.63775315f);
  p = fmaf(t, p, 0.402321582f);
  p = fmaf(t, p, -0.26875686f);
  p = fmaf(t, p, 0.139630057f);
  p = fmaf(t, p, 0.539700616f);
  p = fmaf(t, p, 1.4427292f);
  p = fmaf(t, p, -2.82574822f);
  return t * __builtin_amdgcn_exp2f(fmaf(a * -0.72134752f, a, p));
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

// Inclusive scan over the wave's lanes by an operation whose neutral element is 0: lane exchanges within the vector units, 131072 rows over
// 16 experts 171 -> 159 us against exchanges through LDS (a scan per tile, and its latency comes before anything else)
template <typename Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op) {
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));   // row_shr:1, 2, 4, 8
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));   // row_bcast:15 to the odd rows of 16
  return op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));   // row_bcast:31 to the upper half
}

template <int BM>
__device__ __forceinline__ RowTile find_tile(const LinearDesc& d, const LinearArgs& a, uint32_t tile, int lane) {
  const uint32_t rows = a.rows;
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
    const uint32_t v = max(over_lanes(e < d.experts ? clamped(e + 1) : 0u, [](uint32_t p, uint32_t q) { return max(p, q); }), end);
    const uint32_t start = (uint32_t)__builtin_amdgcn_update_dpp((int)end, (int)v, 0x138, 0xf, 0xf, false);   // wave_shr:1
    const uint32_t count = e < d.experts ? v - start : 0u, tiles = (count + BM - 1) / BM;
    const uint32_t sum = over_lanes(tiles, [](uint32_t p, uint32_t q) { return p + q; });
    const uint64_t hit = __ballot(tile >= before + sum - tiles && tile < before + sum);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      auto of = [&](uint32_t value) { return (uint32_t)__builtin_amdgcn_readlane((int)value, src); };
      const uint32_t skip = (tile - of(before + sum - tiles)) * BM;
      RowTile t{1, base + (uint32_t)src, of(start) + skip, min((uint32_t)BM, of(count) - skip)};
      // (kept in vector registers: as scalars they led the compiler to addresses that spill the sums of a 128 x 256 tile)
      asm volatile("" : "+v"(t.expert), "+v"(t.first), "+v"(t.count));
      return t;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    end = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
  }
  if (!a.zero_rest) return {0, 0, 0, 0};
  const uint32_t t = tile - before, head_tiles = (head + BM - 1) / BM;
  if (t < head_tiles) return {2, 0, t * BM, min((uint32_t)BM, head - t * BM)};
  const uint64_t first = (uint64_t)end + (uint64_t)(t - head_tiles) * BM;
  if (first >= rows) return {0, 0, 0, 0};
  return {2, 0, (uint32_t)first, min((uint32_t)BM, rows - (uint32_t)first)};
}

// tiles of the runs that are not empty and of the rest before and behind them, at most
static uint64_t RowTiles(const LinearDesc& d, const LinearArgs& a, uint32_t BM) {
  if (!a.offsets) return (a.rows + BM - 1) / BM;
  return a.rows / BM + (d.experts < a.rows ? d.experts : a.rows) + (a.zero_rest ? 2 : 0);
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

// eight values of a row of x from column k on, zeros beyond K and for no row; ODD: rows may start on any element
template <bool ODD, typename T>
__device__ __forceinline__ u4l load_x(const T* row, uint32_t k, uint32_t K) {
  if (row == nullptr || k >= K) return u4l{0, 0, 0, 0};
  if (ODD && K - k >= 8) return load16_odd(row + k);
  return load_halves(row + k, K - k);
}

__device__ __forceinline__ acc8 activate(acc8 y, int act) {
  switch (act) {
    case (int)Activation::kRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __builtin_elementwise_maximum(y[j], 0.f);   // (a NaN stays one)
      return y;
    case (int)Activation::kGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = normal_tail(fabsf(y[j]));
        y[j] *= y[j] < 0.f ? q : 1.f - q;
      }
      return y;
    // (the hardware's reciprocal is good to one unit in the last place: 2^-23 of results that are rounded to 2^-11 or compared at 2^-20)
    case (int)Activation::kSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = y[j] * __builtin_amdgcn_rcpf(1.f + __expf(-y[j]));
      return y;
    case (int)Activation::kSigmoid:
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __builtin_amdgcn_rcpf(1.f + __expf(-y[j]));
      return y;
    default: return y;
  }
}

// What the end of eight consecutive columns [n, n + 8) of one position of a tile reads, which may pass N
struct EndsOf {
  uint64_t row;          // of the output
  bool stored, there;    // the row and the columns are the output's; the row of x is x's
  u4l mul, residual;
};

template <typename T, bool ENDS>
__device__ __forceinline__ EndsOf load_ends(const LinearDesc& d, const LinearArgs& a, const RowTile& t, uint32_t pos, uint32_t n) {
  EndsOf e = {(uint64_t)t.first + pos, pos < t.count && n < d.N, true, {0, 0, 0, 0}, {0, 0, 0, 0}};
  if (!e.stored) return e;
  if (a.rows_in) e.there = (uint64_t)(int64_t)a.rows_in[e.row] < a.x_rows;
  if (a.rows_out) {
    e.row = (uint64_t)(int64_t)a.rows_out[e.row];
    e.stored = e.row < a.out_rows;
    if (!e.stored) return e;
  }
  if (ENDS && a.mul) e.mul = load_halves(reinterpret_cast<const T*>(a.mul) + e.row * a.mul_stride + n, d.N - n);
  if (ENDS && a.residual) e.residual = load_halves(reinterpret_cast<const T*>(a.residual) + e.row * a.residual_stride + n, d.N - n);
  return e;
}

// y = act(y) * mul + residual, rounded once and stored; y has its bias, which alone is left for a row of x that is not there
template <typename T, typename OutT, bool ENDS>
__device__ __forceinline__ void finish8(const LinearDesc& d, const LinearArgs& a, const EndsOf& e, uint32_t n, acc8 bias, acc8 y) {
  typedef typename Frag<T>::type frag;
  if (!e.stored) return;
  const uint32_t left = d.N - n;
  y = activate(e.there ? y : bias, d.act);
  if (ENDS && a.mul) y *= __builtin_convertvector(__builtin_bit_cast(frag, e.mul), acc8);
  if (ENDS && a.residual) y += __builtin_convertvector(__builtin_bit_cast(frag, e.residual), acc8);
  void* o = reinterpret_cast<OutT*>(a.out) + e.row * a.out_stride + n;
  if constexpr (sizeof(OutT) == 4) store_words(o, __builtin_bit_cast(u8l, y), left);
  else store_halves(o, __builtin_bit_cast(u4l, __builtin_convertvector(y, frag)), left);
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
// Rows of out that no position names become zeros (kZeroUnnamed).  Every kernel has blocks behind its tiles for it, each with a range of
// out's rows: it reads all of rows_out, marks what it finds of its range in LDS and zeros the rest.  No tile writes these rows, so nothing is
// waited for, and the blocks run beside the last tiles.  Every row named, with these blocks / without:
// 65,536 rows over 16 experts, 1024 -> 512, 91.9 / 92.4 us, 300 over 64, 479 -> 256, 7.04 / 7.00.  A launch that leaves the positions in the
// rows they name and one that looks for them there, before the product, cost 7 us more.
// ------------------------------------------------------------------------------------------------------------
constexpr uint32_t kUnnamedRows = 1u << 17;   // a block's rows at most: one bit each

// rows per block: a sixteenth of them, 256 at least (whole waves of rows)
__host__ __device__ __forceinline__ uint32_t unnamed_range(uint32_t rows) {
  const uint32_t r = ((rows + 15) / 16 + 255) / 256 * 256;
  return r < kUnnamedRows ? r : kUnnamedRows;
}
__host__ __device__ __forceinline__ uint32_t unnamed_blocks(const LinearArgs& a) {
  return a.zero_rest == kZeroUnnamed ? (a.rows + unnamed_range(a.rows) - 1) / unnamed_range(a.rows) : 0;
}

template <typename OutT, uint32_t kThreads>
__device__ __forceinline__ void zero_unnamed(const LinearDesc& d, const LinearArgs& a, uint32_t block, uint32_t* named) {
  const uint32_t rows = a.rows, range = unnamed_range(rows), lo = block * range, count = min(range, rows - lo);
  for (uint32_t i = threadIdx.x; i < range / 32; i += kThreads) named[i] = 0;
  __syncthreads();
  auto look = [&](int32_t r) {
    const uint32_t at = (uint32_t)r - lo;
    if (at < count) atomicOr(&named[at / 32], 1u << (at & 31));
  };
  typedef u4l u4l_words __attribute__((aligned(4)));
  const uint32_t quads = rows / 4;
#pragma unroll 4
  for (uint32_t q = threadIdx.x; q < quads; q += kThreads) {
    const u4l v = reinterpret_cast<const u4l_words*>(a.rows_out)[q];
#pragma unroll
    for (int j = 0; j < 4; ++j) look((int32_t)v[j]);
  }
  if (threadIdx.x < rows % 4) look(a.rows_out[quads * 4 + threadIdx.x]);
  __syncthreads();
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t base = threadIdx.x - lane; base < count; base += kThreads) {   // a wave takes 64 rows
    const uint32_t at = base + lane;
    for (uint64_t left = __ballot(at < count && !(named[at / 32] >> (at & 31) & 1)); left; left &= left - 1) {
      OutT* o = reinterpret_cast<OutT*>(a.out) + (uint64_t)(lo + base + (uint32_t)(__ffsll((unsigned long long)left) - 1)) * a.out_stride;
      for (uint32_t n = lane; n < d.N; n += 64) o[n] = (OutT)0.f;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// Tiles of BM rows x BN columns, WM x WN waves, K in steps of 32, NB LDS buffers.  Whole steps go from memory to LDS without passing
// registers, NB - 1 of them on their way at once; one barrier a step.  The widest tile, 128 x 256 with three buffers, is made for two
// workgroups on a CU: while one waits, starts or ends its tile, the other one's products run (a single 256 x 256 workgroup: 65536 x 479
// -> 1024 101 us against 80; 65536 rows over 16 experts, 1024 -> 512, 111 against 98).
// A row of a step is 64 bytes of LDS, its 16-byte chunks swapped by chunk ^ (row / 2 % 4), so that the fragments' reads (16 rows at one
// chunk) are free of bank conflicts; weight fragments lie in LDS as in memory.  What is left of K below a step comes first, through
// registers, where what lies beyond K becomes zero: its loads' latency is the first steps' too.  Rows that do not start on 16 bytes
// (ALIGNED false) go through registers in every step.
// Rows beyond the tile's count and positions whose rows_in is outside x read some other row; the former are never stored, the sums of
// the latter are replaced in the end.
// ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void to_lds(const void* from, u4l* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// at most n memory operations of this wave left / no LDS operation left; no access moves across
template <int n>
__device__ __forceinline__ void wait_memory() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// 16 bytes of an output; a streamed output goes past the caches' usual order
typedef u4l u4l_anywhere __attribute__((aligned(2)));
__device__ __forceinline__ void put16(void* p, u4l v, bool stream) {
  if (stream) __builtin_nontemporal_store(v, reinterpret_cast<u4l_anywhere*>(p));
  else store16(p, v);
}

constexpr uint32_t kBand = 8;

// ENDS: there is mul or residual
template <typename T, typename OutT, int BM, int BN, int WM, int WN, int NB, bool ALIGNED, bool ENDS>
__global__ __launch_bounds__(64 * WM * WN, 4) void hps_linear_tile_kernel(LinearDesc d, LinearArgs a, uint32_t m_tiles, uint32_t n_tiles) {
  constexpr int kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FP = BN / WN / 32;             // row fragments and column pairs of a wave
  constexpr int XC = BM / 16 / kWaves, WC = BN / 16 / kWaves;     // 1-KB pieces (16 rows; a fragment) of a step per wave
  static_assert(XC * kWaves * 16 == BM && WC * kWaves * 16 == BN && FM >= 1 && FP >= 1 && NB >= 3, "whole pieces");
  constexpr int kStage = (BM + BN) * 4;                           // 16-byte chunks of a buffer: the rows', then the weights'
  typedef typename Frag<T>::type frag;
  __shared__ __attribute__((aligned(16))) u4l lds[NB * kStage];
  static_assert(sizeof(lds) >= kUnnamedRows / 8, "room for a block's bits");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // bands of kBand row tiles, column by column: the 64 workgroups an XCD holds at once read 8 x 8 tiles' operands, not 5 x 14
  if (blockIdx.x >= m_tiles * n_tiles) return zero_unnamed<OutT, 64 * WM * WN>(d, a, blockIdx.x - m_tiles * n_tiles, reinterpret_cast<uint32_t*>(lds));
  const uint32_t id = xcd_order(blockIdx.x, m_tiles * n_tiles), band = id / (kBand * n_tiles), in_band = id - band * kBand * n_tiles;
  const uint32_t high_of = min(kBand, m_tiles - band * kBand), nt = in_band / high_of;
  const RowTile t = find_tile<BM>(d, a, band * kBand + in_band % high_of, lane);
  if (t.kind == 0) return;
  if (t.kind == 2) return zero_rows<OutT>(d, a, t, nt * BN, nt * BN + BN);

  const uint32_t chunk = (lane & 3) ^ ((lane >> 3) & 3);          // of row lane / 4 of a piece, the one that belongs where the lane writes
  const T* xrow[XC];
#pragma unroll
  for (int i = 0; i < XC; ++i) {
    const uint32_t r = (uint32_t)(i * kWaves + wave) * 16 + (lane >> 2);
    const T* p = in_row<T>(a, t.first + min(r, t.count - 1));
    xrow[i] = (p ? p : reinterpret_cast<const T*>(a.x)) + chunk * 8;
  }
  const u4l* wsrc[WC];   // (the same for the whole wave)
#pragma unroll
  for (int i = 0; i < WC; ++i) {
    const uint32_t q = i * kWaves + wave, p = min(nt * (BN / 32) + (q >> 1), d.npairs - 1);   // fragment of the step, two per pair
    wsrc[i] = reinterpret_cast<const u4l*>(d.w) + ((uint64_t)t.expert * d.npairs + p) * d.ksteps * 128 + (q & 1) * 64;
  }
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t n0 = nt * BN + wn * FP * 32;                     // the wave's first column
  const bool idle = n0 >= d.N || (uint32_t)(wm * FM * 16) >= t.count;   // nothing of the wave's is stored: it only copies
  // the sums start from the bias (32 floats per pair of columns; pairs beyond N read the last one's and are never stored)
  acc4 acc[FP][2][FM];
  const float* const tile_bias = d.bias + (uint64_t)t.expert * d.npairs * 32;
  auto bias_of = [&](int p, int lane) {
    return *reinterpret_cast<const acc8*>(tile_bias + min(nt * (BN / 32) + wn * FP + p, d.npairs - 1) * 32 + (lane >> 4) * 8);
  };
#pragma unroll
  for (int p = 0; p < FP; ++p) {
    const acc8 b = bias_of(p, lane);
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      acc[p][0][m] = __builtin_shufflevector(b, b, 0, 1, 2, 3);
      acc[p][1][m] = __builtin_shufflevector(b, b, 4, 5, 6, 7);
    }
  }
  const uint32_t whole = d.K / 32;
  auto copy_x = [&](int i, uint32_t s, u4l* to) { to_lds(xrow[i] + s * 32, to + (i * kWaves + wave) * 64); };
  auto copy_w = [&](int i, uint32_t s, u4l* to) { to_lds(wsrc[i] + (uint64_t)s * 128 + lane, to + BM * 4 + (i * kWaves + wave) * 64); };
  u4l rx[XC];
  auto keep_x = [&](u4l* to) {
#pragma unroll
    for (int i = 0; i < XC; ++i) to[(i * kWaves + wave) * 64 + lane] = rx[i];
  };
  const int xat = wm * FM * 64 + (lane & 15) * 4 + ((lane >> 4) ^ ((lane >> 1) & 3)), wat = BM * 4 + wn * FP * 128 + lane;
  // One step from buffer b.  The copies of the step NB - 1 later (more) leave between the products, a few at a time: all at once behind the
  // barrier, every wave would wait for the others' copies to be taken before its first product.  Rows that go through registers leave one
  // step ahead (one).
  constexpr int kPieces = XC + WC, kPerRow = (kPieces + FM - 1) / FM;
  auto leave = [&](int j, uint32_t s, bool more, u4l* later, bool one) {
    if (j < XC) {
      if constexpr (ALIGNED) {
        if (more) copy_x(j, s + NB - 1, later);
      } else {
        if (one) rx[j] = load16(xrow[j] + (s + 1) * 32);
      }
    } else if (j < kPieces) {
      if (more) copy_w(j - XC, s + NB - 1, later);
    }
  };
  auto multiply = [&](const u4l* b, uint32_t s, bool more, u4l* later, bool one, u4l* next) {
    if (idle) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) leave(j, s, more, later, one);
      if constexpr (!ALIGNED) {
        if (one) keep_x(next);
      }
      return;
    }
    frag fw[FP][2], fx[FM];
#pragma unroll
    for (int p = 0; p < FP; ++p)
#pragma unroll
      for (int h = 0; h < 2; ++h) fw[p][h] = __builtin_bit_cast(frag, b[wat + p * 128 + h * 64]);
#pragma unroll
    for (int m = 0; m < FM; ++m) fx[m] = __builtin_bit_cast(frag, b[xat + m * 64]);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < FM; ++m) {
#pragma unroll
      for (int p = 0; p < FP; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[p][h][m] = Frag<T>::mfma(fw[p][h], fx[m], acc[p][h][m]);
#pragma unroll
      for (int q = 0; q < kPerRow; ++q) leave(m * kPerRow + q, s, more, later, one);
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (!ALIGNED) {
      if (one) keep_x(next);
    }
  };
  u4l tx[XC], tw[WC];
  const bool ragged = whole * 32 < d.K;
  if (ragged) {
#pragma unroll
    for (int i = 0; i < XC; ++i) tx[i] = load_x<!ALIGNED>(xrow[i] - chunk * 8, whole * 32 + chunk * 8, d.K);
#pragma unroll
    for (int i = 0; i < WC; ++i) tw[i] = wsrc[i][(uint64_t)whole * 128 + lane];
  }
  if constexpr (!ALIGNED) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < XC; ++i) rx[i] = load16(xrow[i]);
    }
  }
#pragma unroll
  for (int q = 0; q < NB - 1; ++q)
    if ((uint32_t)q < whole) {
      if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < XC; ++i) copy_x(i, q, lds + q * kStage);
      }
#pragma unroll
      for (int i = 0; i < WC; ++i) copy_w(i, q, lds + q * kStage);
    }
  if constexpr (!ALIGNED) {
    if (whole) keep_x(lds);
  }
  if (ragged) {   // in the last buffer, which the first step's copies take over behind its barrier
    u4l* b = lds + (NB - 1) * kStage;
#pragma unroll
    for (int i = 0; i < XC; ++i) b[(i * kWaves + wave) * 64 + lane] = tx[i];
#pragma unroll
    for (int i = 0; i < WC; ++i) b[BM * 4 + (i * kWaves + wave) * 64 + lane] = tw[i];
    __syncthreads();
    multiply(b, 0, false, b, false, b);
  }
  uint32_t s = 0, cur = 0;   // step and its buffer
  // (in flight behind a step's copies: those of the NB - 2 steps after it)
  constexpr int kBehind = (ALIGNED ? kPieces : WC) * (NB - 2);
#pragma unroll 1
  for (; s + NB - 1 < whole; ++s) {
    const uint32_t after = cur == NB - 1 ? 0 : cur + 1, before = cur == 0 ? NB - 1 : cur - 1;
    wait_memory<kBehind>();   // this wave's pieces of the step are in LDS,
    __syncthreads();          // everybody's are, and nobody reads the buffer before any more
    multiply(lds + cur * kStage, s, true, lds + before * kStage, true, lds + after * kStage);
    cur = after;
  }
#pragma unroll 1
  for (; s < whole; ++s) {
    const uint32_t after = cur == NB - 1 ? 0 : cur + 1;
    wait_memory<0>();
    __syncthreads();
    multiply(lds + cur * kStage, s, false, lds, s + 1 < whole, lds + after * kStage);
    cur = after;
  }
  // (what follows computes its addresses from here: kept from before the loop they would take the sums' registers)
  int lane_ = lane;
  asm volatile("" : "+v"(lane_));
  // The end of the tile.  A vector instruction costs a wave four cycles and a tile has 32,768 sums: ten of them per sum would take as long
  // as 350 of K.  none and relu over a wave's whole columns take two or three, straight from the accumulators.
  constexpr int kCols = FP * 32;
  constexpr int kRoom = NB * kStage / kWaves;   // LDS chunks of a wave, its own from here on
  u4l* const mine = lds + wave * kRoom;
  __syncthreads();                              // nobody reads the steps' buffers any more
  if (idle) return;
  if (n0 + kCols <= d.N && d.act <= (int)Activation::kRelu) {
    uint32_t at[FM];         // the position's output row, ~0: not stored
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const uint32_t r = (wm * FM + m) * 16 + (lane_ & 15);
      at[m] = r < t.count ? t.first + r : ~0u;
    }
    if (a.rows_in) {
#pragma unroll
      for (int m = 0; m < FM; ++m)
        if (at[m] != ~0u && (uint64_t)(int64_t)a.rows_in[at[m]] >= a.x_rows) {
#pragma unroll
          for (int p = 0; p < FP; ++p) {
            const acc8 b = bias_of(p, lane_);
            acc[p][0][m] = __builtin_shufflevector(b, b, 0, 1, 2, 3);
            acc[p][1][m] = __builtin_shufflevector(b, b, 4, 5, 6, 7);
          }
        }
    }
    if (a.rows_out) {
#pragma unroll
      for (int m = 0; m < FM; ++m)
        if (at[m] != ~0u) {
          const int32_t to = a.rows_out[at[m]];
          at[m] = (uint64_t)(int64_t)to < a.out_rows ? (uint32_t)to : ~0u;
        }
    }
    if (d.act == (int)Activation::kRelu) {
#pragma unroll
      for (int p = 0; p < FP; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[p][h][m][j] = __builtin_elementwise_maximum(acc[p][h][m][j], 0.f);   // (a NaN stays one)
    }
    // mul, then residual, each into the accumulators.  Rows in order: the wave's part of the tile is copied to LDS like the rows of x were,
    // all of it on its way at once and no register taken.  Rows by index, or not on 16 bytes: row by row.  A loop of two turns and one
    // fused multiply-add (sum * v + 0, then sum * 1 + v: rounded like the product and the sum they are) keep the sums in their registers.
    if constexpr (ENDS) {
      constexpr int kPart = FP * 4, kParts = FM * 16 * kPart / 64;   // 16-byte chunks of a row; pieces of 64
      static_assert(FM * 16 * kPart <= kRoom, "the wave's part of the tile fits");
#pragma unroll 1
      for (int turn = 0; turn < 2; ++turn) {
        const T* const base = reinterpret_cast<const T*>(turn ? a.residual : a.mul);
        const uint64_t stride = turn ? a.residual_stride : a.mul_stride;
        if (base == nullptr) continue;
        const bool staged = a.rows_out == nullptr && (uintptr_t)base % 16 == 0 && stride % 8 == 0;
        if (staged) {
#pragma unroll 2
          for (int i = 0; i < kParts; ++i) {
            const uint32_t q = i * 64 + lane_, r = q / kPart, c = (q % kPart) ^ (r % kPart), pos = wm * FM * 16 + r;
            to_lds(base + (uint64_t)(t.first + (pos < t.count ? pos : 0u)) * stride + n0 + c * 8, mine + i * 64);
          }
          wait_memory<0>();
        }
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
          for (int p = 0; p < FP; ++p) {
            const int r = m * 16 + (lane_ & 15), c = p * 4 + (lane_ >> 4);
            u4l v = {0, 0, 0, 0};
            if (staged) v = mine[r * kPart + (c ^ (r % kPart))];
            else if (at[m] != ~0u) v = load16(base + (uint64_t)at[m] * stride + n0 + c * 8);
            const acc8 f = __builtin_convertvector(__builtin_bit_cast(frag, v), acc8);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              acc[p][j / 4][m][j % 4] = fmaf(acc[p][j / 4][m][j % 4], turn ? 1.f : f[j], turn ? f[j] : 0.f);
          }
        wait_lds();   // the next copies come over what has been read
      }
    }
    // A lane has eight consecutive columns of a row in every pair.  Two 16-byte chunks of row r (two pairs, or a pair's halves in fp32) are
    // exchanged with the lane of row r ^ 8, so that a store writes 128 consecutive bytes of eight rows instead of 64 of sixteen.
    const bool high = (lane_ & 8) != 0, stream = a.stream_out != 0;
    auto put_two = [&](uint32_t m, u4l q0, u4l q1, uint32_t c0, uint32_t c1) {
      u4l low, up;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(high ? q0[j] : q1[j]), 0x128, 0xf, 0xf, false);   // row_ror:8
        low[j] = high ? got : q0[j];
        up[j] = high ? q1[j] : got;
      }
      const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)at[m], 0x128, 0xf, 0xf, false);
      const uint32_t rl = high ? other : at[m], ru = high ? at[m] : other, c = high ? c1 : c0;
      if (rl != ~0u) put16(reinterpret_cast<OutT*>(a.out) + (uint64_t)rl * a.out_stride + c, low, stream);
      if (ru != ~0u) put16(reinterpret_cast<OutT*>(a.out) + (uint64_t)ru * a.out_stride + c, up, stream);
    };
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const uint32_t c = n0 + (lane_ >> 4) * 8;
      if constexpr (sizeof(OutT) == 4) {
#pragma unroll
        for (int p = 0; p < FP; ++p)
          put_two(m, __builtin_bit_cast(u4l, acc[p][0][m]), __builtin_bit_cast(u4l, acc[p][1][m]), c + p * 32, c + p * 32 + 4);
      } else {
        u4l q[FP];
#pragma unroll
        for (int p = 0; p < FP; ++p)
          q[p] = __builtin_bit_cast(u4l, __builtin_convertvector(__builtin_shufflevector(acc[p][0][m], acc[p][1][m], 0, 1, 2, 3, 4, 5, 6, 7), frag));
        if constexpr (FP == 2) put_two(m, q[0], q[1], c, c + 32);
        else if (at[m] != ~0u) put16(reinterpret_cast<OutT*>(a.out) + (uint64_t)at[m] * a.out_stride + c, q[0], stream);
      }
    }
    return;
  }
  // The other activations, and columns that pass N: each wave hands its sums through LDS (its own part, kHalf row fragments at a time,
  // 16-byte chunks swapped by chunk ^ (row & 7)) and takes them back eight columns of a row per lane, so that one short loop does it.
  constexpr int kLanes = kCols / 8;                                                // lanes that share a row
  constexpr int kHalf = FM * 16 * (kCols / 4) <= kRoom ? FM : FM / 2;              // row fragments at a time
  constexpr int kIter = kHalf * 16 * kLanes / 64;
  static_assert(kHalf * 16 * (kCols / 4) <= kRoom && FM % kHalf == 0 && 64 % kLanes == 0, "a wave's sums fit its part of LDS");
  static_assert(FP <= 2, "two pairs of columns are stored together");
  const uint32_t c8 = lane_ % kLanes, n = n0 + c8 * 8;
  // (32 floats per pair of columns: eight from n < N on are there)
  const acc8 bias = *reinterpret_cast<const acc8*>(tile_bias + (n < d.N ? n : 0));
#pragma unroll 1
  for (int half = 0; half < FM / kHalf; ++half) {
#pragma unroll
    for (int m = 0; m < FM; ++m)
      if (m / kHalf == half)
#pragma unroll
        for (int p = 0; p < FP; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = (m % kHalf) * 16 + (lane_ & 15), c = p * 8 + (lane_ >> 4) * 2 + h;
            mine[r * (kCols / 4) + (c ^ (r & 7))] = __builtin_bit_cast(u4l, acc[p][h][m]);
          }
#pragma unroll 1
    for (int i = 0; i < kIter; ++i) {
      const int r = i * (64 / kLanes) + lane_ / kLanes;
      const u4l* row = mine + r * (kCols / 4);
      const acc4 v0 = __builtin_bit_cast(acc4, row[(2 * c8) ^ (r & 7)]), v1 = __builtin_bit_cast(acc4, row[(2 * c8 + 1) ^ (r & 7)]);
      finish8<T, OutT, ENDS>(d, a, load_ends<T, ENDS>(d, a, t, (wm * FM + half * kHalf) * 16 + r, n), n, bias,
                             __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// Few rows: bound by the weights' bytes and by latency.  A block takes one pair of 32 columns and up to 16 * MF rows; its NW waves
// split K, each reads its weight fragments and the rows' chunks straight from memory (U steps on their way at once), and the partial
// sums meet in LDS, added in the waves' order.
// ------------------------------------------------------------------------------------------------------------
template <typename T, typename OutT, int MF, int NW, bool ODD>
__global__ __launch_bounds__(64 * NW) void hps_linear_rows_kernel(LinearDesc d, LinearArgs a, uint32_t m_tiles) {
  constexpr int U = MF >= 4 ? 2 : 4;
  typedef typename Frag<T>::type frag;
  __shared__ __attribute__((aligned(16))) acc4 part[NW][2 * MF][64];
  static_assert(sizeof(part) >= kUnnamedRows / 8, "room for a block's bits");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x >= m_tiles * d.npairs) return zero_unnamed<OutT, 64 * NW>(d, a, blockIdx.x - m_tiles * d.npairs, reinterpret_cast<uint32_t*>(&part[0][0][0]));
  const uint32_t id = xcd_order(blockIdx.x, m_tiles * d.npairs);
  const uint32_t pair = id / m_tiles;
  const RowTile t = find_tile<16 * MF>(d, a, id % m_tiles, lane);
  if (t.kind == 0) return;
  if (t.kind == 2) return zero_rows<OutT>(d, a, t, pair * 32, pair * 32 + 32);
  // The first steps' weights leave before the rows' indexes are there, and what the end of the block reads before the products: each would
  // be one more wait for memory after the other (300 rows over 16 experts, 479 -> 256, with indexes, mul and residual 4.2 -> 3.85 us)
  const u4l* w = reinterpret_cast<const u4l*>(d.w) + ((uint64_t)t.expert * d.npairs + pair) * d.ksteps * 128 + lane;
  u4l rw[U][2];
  auto load_w = [&](uint32_t s0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * NW;
      rw[u][0] = rw[u][1] = u4l{0, 0, 0, 0};
      if (s < d.ksteps) {
        rw[u][0] = w[(uint64_t)s * 128];
        rw[u][1] = w[(uint64_t)s * 128 + 64];
      }
    }
  };
  load_w(wave);
  static_assert(MF <= NW, "a wave ends one fragment of rows at most");
  const uint32_t n = pair * 32 + (lane >> 4) * 8;
  const EndsOf ends = load_ends<T, true>(d, a, t, wave < MF ? wave * 16 + (lane & 15) : t.count, n);
  const acc8 bias = *reinterpret_cast<const acc8*>(d.bias + (uint64_t)t.expert * d.npairs * 32 + n);
  const T* xrow[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const uint32_t r = m * 16 + (lane & 15);
    xrow[m] = r < t.count ? in_row<T>(a, t.first + r) : nullptr;
  }
  acc4 acc[2][MF];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[h][m] = acc4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t s0 = wave; s0 < d.ksteps; s0 += NW * U) {
    u4l rx[U][MF];
    if (s0 != (uint32_t)wave) load_w(s0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MF; ++m) rx[u][m] = load_x<ODD>(xrow[m], (s0 + u * NW) * 32 + (lane >> 4) * 8, d.K);
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
  if (wave >= MF) return;
  acc8 y = bias;
#pragma unroll
  for (int v = 0; v < NW; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] += part[v][(j / 4) * MF + wave][lane][j % 4];
  finish8<T, OutT, true>(d, a, ends, n, bias, y);
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

// Which kernel: the one whose blocks fill the card without taking too little each.  Measured with N = 1024, K = 1024 (us): M = 128: rows
// 16 / rows 32 / 64 x 64 = 4.0 / 5.0 / 6.3; M = 512: 8.8 / 7.4 / 6.6.  A wider tile from 5/8 of the CUs on: 64 x 64 / 128 x 128 with 128 wide
// tiles 9.6 / 12.7, 160 13.4 / 13.0, 208 17.5 / 13.6 (K = 3456: 135 39.3 / 31.6, 216 50.8 / 34.4); 128 x 128 / 128 x 256 with 112 wide tiles
// (K = 3456) 34.4 / 46.9, 168 55.1 / 50.3; 160 (K = 1024) 19.3 / 19.3.  Few columns leave no room for wide tiles: M = 65536, N = 64, K = 256:
// 64 x 64 9.2, 128 x 128 11.1.  Measured with rows on 16 bytes; rows off them go by the same rule, and some would be better off in a smaller
// tile (4,096 x 1,024 -> 1,024, rows 1,025 apart: 128 x 128 23.6, 64 x 64 20.7).
// With experts the tiles are estimated as three quarters of one more per run, and one per run at least: past two blocks of the rows kernels a
// CU they wait for each other (300 rows over 64 experts, 479 -> 256: rows 16 / rows 32 / 64 x 64 = 5.8 / 4.9 / 6.1; 200 rows 4.4 / 4.8 / 6.0;
// 600 over 300, 256 -> 64: 7.4 / 7.7 / 5.5).  Runs shorter than a tile of 128 take 64 x 64: 125 rows each 10.6 us against 11.7, 250 17.5 / 15.8.
LinearTile LinearTileOf(const LinearDesc& d, uint64_t rows, bool offsets, int cu_count) {
  const uint64_t cus = (uint64_t)cu_count, runs = offsets ? (d.experts < rows ? d.experts : rows) : 0;
  auto tiles = [&](uint64_t bm, uint64_t bn) {
    const uint64_t most = (rows + bm - 1) / bm + runs * 3 / 4;
    return (most < runs ? runs : most) * ((d.N + bn - 1) / bn);
  };
  if (tiles(16, 32) <= 2 * cus) return {16, 32};
  if (tiles(32, 32) <= 2 * cus) return {32, 32};
  if (tiles(128, 128) * 8 < cus * 5 || d.N <= 64 || rows < runs * 128) return {64, 64};
  if (tiles(128, 256) * 8 < cus * 5 || d.N <= 128) return {128, 128};
  return {128, 256};
}

namespace {

template <typename T, typename OutT, int BM, int BN, int WM, int WN, int NB>
hipError_t LaunchTile(const LinearDesc& d, const LinearArgs& a, hipStream_t stream) {
  const uint64_t m_tiles = RowTiles(d, a, BM), n_tiles = (d.N + BN - 1) / BN;
  if (m_tiles * n_tiles >= (1ull << 23)) return hipErrorInvalidConfiguration;   // 512 threads each: a launch holds 2^32
  const bool aligned = (uintptr_t)a.x % 16 == 0 && a.x_stride % 8 == 0;
  auto* kernel = a.mul || a.residual ? (aligned ? hps_linear_tile_kernel<T, OutT, BM, BN, WM, WN, NB, true, true>
                                                : hps_linear_tile_kernel<T, OutT, BM, BN, WM, WN, NB, false, true>)
                                     : (aligned ? hps_linear_tile_kernel<T, OutT, BM, BN, WM, WN, NB, true, false>
                                                : hps_linear_tile_kernel<T, OutT, BM, BN, WM, WN, NB, false, false>);
  return Launch(kernel, (uint32_t)(m_tiles * n_tiles) + unnamed_blocks(a), 64 * WM * WN, stream, d, a, m_tiles, n_tiles);
}

template <typename T, typename OutT, int MF, int NW>
hipError_t LaunchRows(const LinearDesc& d, const LinearArgs& a, hipStream_t stream) {
  const uint64_t m_tiles = RowTiles(d, a, 16 * MF);
  if (m_tiles * d.npairs >= (1ull << 22)) return hipErrorInvalidConfiguration;
  const bool odd = (uintptr_t)a.x % 4 != 0 || a.x_stride % 2 != 0;
  auto* kernel = odd ? hps_linear_rows_kernel<T, OutT, MF, NW, true> : hps_linear_rows_kernel<T, OutT, MF, NW, false>;
  return Launch(kernel, (uint32_t)(m_tiles * d.npairs) + unnamed_blocks(a), 64 * NW, stream, d, a, m_tiles);
}

// An output larger than the L2s together (32 MB) leaves by streaming stores: it would push out x and the weights, which the other tiles
// still read.  65536 x 479 -> 1024 (134 MB) 103 -> 80 us, 16384 x 1024 -> 1024 (34 MB) 33 -> 32; a smaller one may stay for its reader.
constexpr uint64_t kStreamBytes = 32ull << 20;

template <typename T, typename OutT>
hipError_t LaunchTyped(const LinearDesc& d, LinearArgs a, int cu_count, hipStream_t stream) {
  const LinearTile tile = LinearTileOf(d, a.rows, a.offsets != nullptr, cu_count);
  if (a.zero_rest == kZeroUnnamed && !a.rows_out) a.zero_rest = kZeroRest;   // (every row is a position's)
  if (tile.rows == 16) return LaunchRows<T, OutT, 1, 8>(d, a, stream);
  if (tile.rows == 32) return LaunchRows<T, OutT, 2, 8>(d, a, stream);
  if (tile.rows == 64) return LaunchTile<T, OutT, 64, 64, 2, 2, 4>(d, a, stream);
  if (tile.cols == 128) return LaunchTile<T, OutT, 128, 128, 2, 4, 4>(d, a, stream);
  return LaunchTile<T, OutT, 128, 256, 2, 4, 3>(d, a, stream);
}

template <typename From>
hipError_t PackFrom(const void* w, uint32_t experts, uint32_t K, uint32_t N, void* packed, ElemType to, hipStream_t stream) {
  const uint32_t ksteps = (K + 31) / 32, npairs = (N + 31) / 32;
  const uint64_t total = (uint64_t)experts * npairs * ksteps * 128;
  const uint32_t blocks = (uint32_t)((total + 255) / 256 < 65536 ? (total + 255) / 256 : 65536);
  if (to == ElemType::kF16)
    return Launch(hps_linear_pack_kernel<From, _Float16>, blocks, 256, stream, (const From*)w, experts, K, N, ksteps, npairs, (_Float16*)packed);
  return Launch(hps_linear_pack_kernel<From, __bf16>, blocks, 256, stream, (const From*)w, experts, K, N, ksteps, npairs, (__bf16*)packed);
}

}  // namespace

hipError_t LaunchLinearPack(const void* d_w, ElemType from, uint32_t experts, uint32_t K, uint32_t N, void* d_packed, ElemType to,
                            hipStream_t stream) {
  if (from == ElemType::kF32) return PackFrom<float>(d_w, experts, K, N, d_packed, to, stream);
  if (from == ElemType::kF16) return PackFrom<_Float16>(d_w, experts, K, N, d_packed, to, stream);
  return PackFrom<__bf16>(d_w, experts, K, N, d_packed, to, stream);
}

hipError_t LaunchLinear(const LinearDesc& d, const LinearArgs& args, ElemType type, ElemType out_type, int cu_count, hipStream_t stream) {
  LinearArgs a = args;
  a.stream_out = (uint64_t)a.rows * d.N * ElemBytes(out_type) >= kStreamBytes;
  if (type == ElemType::kF16)
    return out_type == ElemType::kF32 ? LaunchTyped<_Float16, float>(d, a, cu_count, stream)
                                      : LaunchTyped<_Float16, _Float16>(d, a, cu_count, stream);
  return out_type == ElemType::kF32 ? LaunchTyped<__bf16, float>(d, a, cu_count, stream)
                                    : LaunchTyped<__bf16, __bf16>(d, a, cu_count, stream);
}

}  // namespace hps
