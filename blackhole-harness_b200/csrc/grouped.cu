// grouped.cu — products of ragged row groups with their experts' 16-bit
// matrices: y = x W[e]^T, dx = dy W[e], and the weight gradients dW[e] = dy_e^T x_e.
// Group e is rows offsets[e] .. offsets[e+1]-1.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include <atomic>
#include <mutex>

#include <cudaTypedefs.h>

#include "internal.cuh"
#include "pair.cuh"

namespace hexmoe {
namespace {

int arg_error(const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_error(HEXMOE_E_ARG, buf);
}

// The offsets of the groups, as the kernels see them: each clamped to 0..rows
// and to no less than the one before, so that whatever the array holds the
// groups are disjoint row ranges.  `bad` says that something was clamped.
struct Groups {
  const void* offsets;   // int32 or int64 [experts + 1]
  int32_t is64;
  int32_t experts;
  int64_t rows;
};

__device__ __forceinline__ int64_t raw_offset(const Groups& g, int e) {
  return g.is64 ? static_cast<const int64_t*>(g.offsets)[e] : static_cast<const int32_t*>(g.offsets)[e];
}

// A warp's walk over the groups, 32 at a time: lane l of a step holds group
// base + l.  first is carried from step to step.
struct GroupScan {
  int64_t begin, end;   // this lane's group (empty past the last expert)
  bool bad;
};
__device__ __forceinline__ GroupScan scan_groups(const Groups& g, int base, int64_t& carry) {
  const int lane = threadIdx.x % 32, e = base + lane;
  const bool in = e < g.experts;
  const int64_t raw0 = raw_offset(g, min(e, g.experts)), raw1 = raw_offset(g, min(e + 1, g.experts));
  GroupScan s;
  s.bad = in && (raw0 < 0 || raw1 < raw0 || raw1 > g.rows);
  s.begin = raw0;
  s.end = raw1;
  if (__any_sync(0xffffffffu, s.bad || raw0 < carry)) {   // something to clamp, here or in the groups before
    int64_t end = max(raw1 < 0 ? 0 : raw1 > g.rows ? g.rows : raw1, carry);
    const int64_t first = max(raw0 < 0 ? 0 : raw0 > g.rows ? g.rows : raw0, carry);
    if (lane == 0) end = max(end, first);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {   // running maximum
      const int64_t v = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end = max(end, v);
    }
    const int64_t begin = __shfl_up_sync(0xffffffffu, end, 1);
    s.begin = lane == 0 ? first : begin;
    s.end = end;
  }
  carry = __shfl_sync(0xffffffffu, s.end, 31);
  return s;
}

// The tensor core's fp32 sums cut where an fp32 addition rounds, once for every 16 products: the error grows with the
// length of a sum, always towards zero.  Results in fp32 therefore take no more than kRunLength products from one
// accumulator and add the runs in fp32.  x^T x of 500, 2000, 8000, 60000 rows, relative to its diagonal: 1e-6, 6e-6, 5e-6,
// 5e-6 (in one accumulator 1e-6, 6e-6, 2.7e-5, 3.3e-4; a plain fp32 product 3e-7, 1e-6, 1e-6, 4e-6 or, values of one
// sign, 1.3e-5).  What it costs is the additions, which L2 takes at 2.5 TB/s: f32 gradient of 8 x 8192 rows, 2048 x 2048:
// 419 us against 374, 60000 rows 393 against 339 (446 with runs of 1024); rows of 8192 to f32, 4 x 2048 x 1536: 174
// against 154.  16-bit results are rounded to 2^-9 or 2^-12 at the end and keep one accumulator: 5e-6 at 2000 products,
// 2.7e-5 at 8000.
constexpr int kRunLength = 2048;

// ---------------------------------------------------------------- plain kernel
// out(i, j) = sum_r A(i, r) B(j, r) over operands with any element strides:
// 64 x 64 tiles, mma.sync over 32-wide reduction steps staged in shared memory
// with element loads.  It takes what the TMA kernels cannot address (a base or
// row stride that is no multiple of 16 bytes); bound by those loads (weight gradient of
// 32768 rows, 96 x 1536 x 2048: 5.8 ms, where the tensor-memory kernel takes 0.2).
constexpr int kPlainTile = 64, kPlainK = 32, kPlainThreads = 128, kPlainPitch = kPlainK + 8;

struct PlainParams {
  Groups g;
  const uint16_t* a;     // ragged rows: x; weight gradient: dy
  const uint16_t* b;     // ragged rows: w; weight gradient: x
  int64_t a_i, a_r;      // element strides
  int64_t b_j, b_r, b_e;
  int32_t i_len;         // weight gradient: rows of the output
  int32_t j_len;
  int32_t r_len;         // ragged rows: reduction length
  void* out;
  int64_t out_i, out_e;
  int32_t out_f32, accumulate, bf16;
  int32_t j_tiles, i_tiles;
  int32_t* dev_err;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
  if (bf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint16_t round16(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ float widen16(uint16_t v, bool bf16) {
  return bf16 ? __bfloat162float(__ushort_as_bfloat16(v)) : __half2float(__ushort_as_half(v));
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}

// fp32 bits rounded to 16: pairs into one word each (the first half of r), or each
// into its own.  One branch on the type, none per value.
template <int N>
__device__ __forceinline__ void pack_pairs(uint32_t (&r)[N], bool bf16) {
  if (bf16) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) r[i] = pack16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), true);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) r[i] = pack16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), false);
  }
}
__device__ __forceinline__ void pack_each(uint32_t (&r)[32], bool bf16) {
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = round16(__uint_as_float(r[i]), true);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = round16(__uint_as_float(r[i]), false);
  }
}
// The first `count` (all from 8 on, none below 1) of 8 16-bit values.
__device__ __forceinline__ void store_8(uint16_t* dst, const uint4& v, int count) {
  if (count >= 8) {
    *reinterpret_cast<uint4*>(dst) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) dst[i] = static_cast<uint16_t>(w[i / 2] >> (i % 2 * 16));
}

// 64 rows x 32 reduction values into registers (16 a thread), zero outside the
// given extents; consecutive threads walk the dimension of unit stride.
__device__ __forceinline__ void plain_fetch(uint16_t (&v)[16], const uint16_t* base, int64_t s_i, int64_t s_r,
                                            int64_t rows, int64_t reds) {
#pragma unroll
  for (int t = 0; t < 16; ++t) {
    const int f = t * kPlainThreads + threadIdx.x;
    const int r = s_r == 1 ? f % kPlainK : f / kPlainTile, i = s_r == 1 ? f / kPlainK : f % kPlainTile;
    v[t] = i < rows && r < reds ? base[i * s_i + r * s_r] : 0;
  }
}
__device__ __forceinline__ void plain_stage(uint16_t (*tile)[kPlainPitch], const uint16_t (&v)[16], int64_t s_r) {
#pragma unroll
  for (int t = 0; t < 16; ++t) {
    const int f = t * kPlainThreads + threadIdx.x;
    const int r = s_r == 1 ? f % kPlainK : f / kPlainTile, i = s_r == 1 ? f / kPlainK : f % kPlainTile;
    tile[i][r] = v[t];
  }
}

template <bool WGRAD>
__global__ void __launch_bounds__(kPlainThreads) grouped_plain_kernel(const PlainParams p) {
  __shared__ __align__(16) uint16_t ta[kPlainTile][kPlainPitch], tb[kPlainTile][kPlainPitch];   // read as 32-bit words
  __shared__ int64_t s_begin, s_end;
  __shared__ int s_expert;
  __shared__ int64_t s_lo, s_hi;
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int jt = blockIdx.x % p.j_tiles;
  const int64_t it = blockIdx.x / p.j_tiles;
  const int want_e = WGRAD ? static_cast<int>(it / p.i_tiles) : -1;
  if (threadIdx.x == 0) s_expert = -1;
  __syncthreads();
  if (warp == 0) {   // the group of this tile
    int64_t carry = 0, tiles = 0;
    bool bad = false;
    for (int base = 0; base < p.g.experts; base += 32) {
      const GroupScan s = scan_groups(p.g, base, carry);
      bad |= s.bad;
      if (base == 0 && lane == 0) s_lo = s.begin;
      if constexpr (WGRAD) {
        if (base + lane == want_e) { s_begin = s.begin; s_end = s.end; s_expert = want_e; }
      } else {
        const int64_t mine = (s.end - s.begin + kPlainTile - 1) / kPlainTile;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        upto += tiles;
        if (it < upto && it >= upto - mine) {
          s_begin = s.begin + (it - (upto - mine)) * kPlainTile;
          s_end = min(s.end, s_begin + kPlainTile);
          s_expert = base + lane;
        }
        tiles = __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) s_hi = carry;
    if (bad && blockIdx.x == 0) atomicOr(p.dev_err, kDevErrOffsets);
  }
  __syncthreads();
  if constexpr (!WGRAD) {   // rows of no group
    const int64_t gap = s_lo + (p.g.rows - s_hi), total = gap * p.j_len;
    for (int64_t f = static_cast<int64_t>(blockIdx.x) * kPlainThreads + threadIdx.x; f < total;
         f += static_cast<int64_t>(gridDim.x) * kPlainThreads) {
      int64_t i = f / p.j_len;
      if (i >= s_lo) i += s_hi - s_lo;
      if (p.out_f32) static_cast<float*>(p.out)[i * p.out_i + f % p.j_len] = 0.f;
      else static_cast<uint16_t*>(p.out)[i * p.out_i + f % p.j_len] = 0;
    }
  }
  const int e = s_expert;
  if (e < 0) return;
  const int64_t begin = s_begin, end = s_end;
  const int i0 = WGRAD ? static_cast<int>(it % p.i_tiles) * kPlainTile : 0, j0 = jt * kPlainTile;
  const uint16_t* a = p.a + (WGRAD ? begin * p.a_r + i0 * p.a_i : begin * p.a_i);
  const uint16_t* b = p.b + (WGRAD ? begin * p.b_r : e * p.b_e) + j0 * p.b_j;
  const int64_t i_left = WGRAD ? p.i_len - i0 : end - begin, j_left = p.j_len - j0;
  const int64_t reds = WGRAD ? end - begin : p.r_len;
  const int wi = warp / 2 * 32, wj = warp % 2 * 32, g = lane / 4, q = lane % 4;
  float acc[2][4][4] = {}, sum[2][4][4] = {};
  auto flush = [&] {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          sum[m][n][h] += acc[m][n][h];
          acc[m][n][h] = 0.f;
        }
  };
  uint16_t va[16], vb[16];
  plain_fetch(va, a, p.a_i, p.a_r, i_left, reds);
  plain_fetch(vb, b, p.b_j, p.b_r, j_left, reds);
  for (int64_t r = 0; r < reds; r += kPlainK) {
    __syncthreads();
    plain_stage(ta, va, p.a_r);
    plain_stage(tb, vb, p.b_r);
    __syncthreads();
    if (r + kPlainK < reds) {
      plain_fetch(va, a + (r + kPlainK) * p.a_r, p.a_i, p.a_r, i_left, reds - r - kPlainK);
      plain_fetch(vb, b + (r + kPlainK) * p.b_r, p.b_j, p.b_r, j_left, reds - r - kPlainK);
    }
#pragma unroll
    for (int k = 0; k < kPlainK; k += 16) {
      uint32_t fa[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 4; ++h)
          fa[m][h] = *reinterpret_cast<const uint32_t*>(&ta[wi + m * 16 + g + (h & 1) * 8][k + q * 2 + (h >> 1) * 8]);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t b0 = *reinterpret_cast<const uint32_t*>(&tb[wj + n * 8 + g][k + q * 2]);
        const uint32_t b1 = *reinterpret_cast<const uint32_t*>(&tb[wj + n * 8 + g][k + q * 2 + 8]);
#pragma unroll
        for (int m = 0; m < 2; ++m) mma_16816(acc[m][n], fa[m], b0, b1, p.bf16);
      }
    }
    if (r / kPlainK % (kRunLength / kPlainK) == kRunLength / kPlainK - 1) flush();
  }
  flush();
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int i = wi + m * 16 + g + (h >> 1) * 8, j = wj + n * 8 + q * 2 + (h & 1);
        if (i >= i_left || j >= j_left) continue;
        const int64_t at = WGRAD ? e * p.out_e + (i0 + i) * p.out_i + j0 + j : (begin + i) * p.out_i + j0 + j;
        float v = sum[m][n][h];
        if (p.out_f32) {
          float* o = static_cast<float*>(p.out) + at;
          *o = p.accumulate ? *o + v : v;
        } else {
          uint16_t* o = static_cast<uint16_t*>(p.out) + at;
          if (p.accumulate) v += widen16(*o, p.bf16);
          *o = round16(v, p.bf16);
        }
      }
}

cudaError_t launch_plain(const PlainParams& p, bool wgrad, int64_t blocks, cudaStream_t st) {
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::max<int64_t>(blocks, 1)));
  cfg.blockDim = dim3(kPlainThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return wgrad ? cudaLaunchKernelEx(&cfg, grouped_plain_kernel<true>, p)
               : cudaLaunchKernelEx(&cfg, grouped_plain_kernel<false>, p);
}

// offsets[e] = block_m x the plan blocks whose expert is below e: a binary
// search per expert over the sorted experts of the plan's used blocks.
__global__ void group_offsets_kernel(const int32_t* expert_ids, int64_t max_blocks, const int32_t* npp, int32_t bm,
                                     int32_t experts, int32_t* offsets) {
  pdl_wait();
  const int e = blockIdx.x * blockDim.x + threadIdx.x;
  if (e > experts) return;
  int64_t lo = 0, hi = min(max_blocks, static_cast<int64_t>(npp[0]) / bm);
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (expert_ids[mid] < e) lo = mid + 1;
    else hi = mid;
  }
  offsets[e] = static_cast<int32_t>(lo * bm);
}

// ------------------------------------------------------------ tensor-memory kernel
// Persistent pairs of CTAs over tiles of one group.  Every tile is one 256-row M
// side by up to 256 N columns of fp32 accumulators in tensor memory (two such
// accumulators, so that a tile's epilogue runs under the next one's products),
// fed by a ring of 64-wide reduction steps that TMA fills, 32 KB a CTA and step.
//   rows (y = x W^T, dx = dy W)  M side: the matrix's output features, N side: the
//         group's rows.  N is a multiple of 32 chosen per tile, so a group of 341
//         rows takes two tiles of 192, not two of 256, and a group of 5 rows one
//         of 32: the weights stream once at full width whatever the group's size.
//   weight gradient              M side: n, N side: k (or the other way about, kWgradT,
//         where n would fill its 256s badly), reduction over the group's rows.  The last
//         step of a group zeroes the rows that follow it, in both operands (they are
//         another group's, and may hold anything).
// Operand majors: x and dy rows are reduction-major (K) in the row products, as
// is W for y; W for dx, and both operands of the weight gradient, are stored with
// the reduction outermost and go to the tensor core as MN-major tiles.
//
// 12 warps a CTA: 0 loads, 1 issues the products (the leader's), 2 and 3 zero tails
// (weight gradient, the leader's), 4..11 write results.  Each walks the groups' offsets by
// itself, so that no size is known on the host.
//
// Measured, bf16, 96 experts, 1536 x 2048, a call at a time and (in brackets) back to back, where the power cap
// lowers the clock at the same number of cycles: 512 rows 91..93 us (93: HBM, 6.5 TB/s); 32768 rows 174..178 us
// (206..228 at 1.12 GHz; HBM and tensor cores, each of which alone takes 145); the weight gradient of those 203..209 us
// (229..260 at 1.27 GHz; tensor cores 52 % busy, 604 MB written, which takes a plain fill 157).  A single product of
// 8192 x 8192 x 2048: 174 us (1580 TFLOP/s).
constexpr int kMaxStages = 6;
constexpr int kStepK = 64;
constexpr uint32_t kOperandBytes = 128 * kStepK * 2;   // one operand's share of a CTA and step
constexpr uint32_t kChunkBytes = kOperandBytes / 2;    // 64 rows of an MN-major operand
constexpr int kPairThreads = 384;
constexpr int kWriters = 8;
constexpr uint32_t kAccCols = 256;
constexpr uint32_t kStoreBytes = 2048;                 // a writer's staging tile: 32 lines of 64 B
constexpr uint32_t kRingBytes = 200 * 1024;            // 6 steps of A and B, 4 of A and two Bs, 5 narrow ones
constexpr uint32_t kPairSmem = 1024 + kRingBytes + kWriters * kStoreBytes + 1024;
constexpr int kBoxes = 4;                              // row boxes of 16, 32, 64, 128

enum PairMode { kRowsK = 0, kRowsMN = 1, kWgrad = 2, kWgradT = 3 };   // kWgradT: M side k, N side n

// Shapes of a tile's N side and of the ring that fits it.
//   kOne     up to 256 columns: 6 steps of 32 KB
//   kTwo     up to 512 in two accumulators: 4 steps of 48 KB
//   kNarrow  up to 64: 5 steps of 40 KB, 128 wide: with a handful of rows the matrix streams, and the ring holds
//            as much of it as it can.  Waiting for a step, issuing its products and committing them
//            takes the issuing warp some 450 cycles, more than narrow products run: twice the step
//            (one token on 96 experts, 1536 x 2048: 64 wide 14.5 us, 128 wide 13.1, 12.6 with the fifth step).
//   kMiddle  up to 128: 4 steps of 48 KB, 128 wide
enum PairShape { kOne = 0, kTwo = 1, kNarrow = 2, kMiddle = 3 };
constexpr int subs_of(int shape) { return shape >= kNarrow ? 2 : 1; }   // 64-wide blocks of a step
constexpr int span_of(int shape) {                                      // most rows of a tile
  return shape == kTwo ? 512 : shape == kNarrow ? 64 : shape == kMiddle ? 128 : 256;
}

struct PairParams {
  CUtensorMap a;             // W (3-D: reduction or features, ..., expert); weight gradient: dy, or x in kWgradT
  CUtensorMap b[kBoxes];     // the rows, by box height; weight gradient: [0] is the other of x and dy
  CUtensorMap out;           // boxes of 32 rows x 64 B; f32 of kWgradT: 16 rows x 128 B
  Groups g;
  int32_t m_len;             // M side: output features; weight gradient: n, or k in kWgradT
  int32_t n_len;             // weight gradient: k, or n in kWgradT
  int32_t red;               // row products: reduction length
  int32_t m_tiles, n_tiles, tile_n;   // n_tiles, tile_n: weight gradient
  int32_t splits;            // runs that the reduction of a tile is cut into, over several pairs
  int32_t run;               // RUNS: most steps that one accumulator sums
  void* dst;                 // splits > 1: fp32 partials, one result a run
  int64_t ld, stride_e, stride_split;
  int32_t f32, bf16, accumulate, tma_out;
  int32_t* dev_err;
};

// One tile: expert, M offset, N offset (a row offset within the group in the row
// products) and width, of `parts` accumulators side by side; row0 its first row,
// valid its real columns; steps of the reduction from `first` on, the last one of
// `tail` (0: full); split: the run of the reduction that these are.
struct Tile {
  int32_t e, m0, n0, width, parts, first, steps, tail, split;
  int64_t row0;
  int32_t valid;
  bool add;   // to what the runs before it have written
  // The columns of accumulator i: what is left of the tile, in whole 32s (341 rows: 192 and 160).
  __device__ __forceinline__ int32_t columns(int i) const { return min(width, (valid - i * width + 31) / 32 * 32); }
};

// RUNS: f32 results whose reduction may pass kRunLength.  Kernels without it are 4 % faster (16-bit gradient of 96 x
// 1536 x 2048, 341 rows: 248 us against 260 with the runs looked for).
template <int MODE, int SHAPE, bool RUNS>
struct Walker {
  int32_t base = -32;
  int64_t carry = 0, lo = 0;
  int32_t upto = 0, mine = 0, total = 0;
  int64_t begin = 0, end = 0;
  bool bad = false;
  int32_t left = 0, per = 0, end_tail = 0;   // of the tile's steps: to come, in a run, and its last one

  // The next run of a tile's reduction: all of it, or with RUNS pieces of at most p.run steps one after the other.
  __device__ __forceinline__ bool next(const PairParams& p, int32_t& unit, int32_t stride, Tile& t) {
    if (!RUNS || left == 0) {
      if (!find(p, unit, t)) return false;
      unit += stride;
      if constexpr (!RUNS) return true;
      t.add = false;
      per = left = t.steps;
      end_tail = t.tail;
      if (left > p.run) {
        const int32_t runs = (left + p.run - 1) / p.run;
        per = (left + runs - 1) / runs;
      }
    } else {
      t.first += t.steps;
      t.add = true;
    }
    t.steps = min(per, left);
    left -= t.steps;
    t.tail = left ? 0 : end_tail;
    return true;
  }

  __device__ __forceinline__ bool find(const PairParams& p, int32_t unit, Tile& t) {
    constexpr int32_t kSpan = span_of(SHAPE);
    const int32_t tile = p.splits > 1 ? unit / p.splits : unit;
    while (tile >= total) {
      if (base + 32 >= p.g.experts) return false;
      base += 32;
      const GroupScan s = scan_groups(p.g, base, carry);
      bad |= s.bad;
      begin = s.begin;
      end = s.end;
      if (base == 0) lo = __shfl_sync(0xffffffffu, begin, 0);
      const int lane = threadIdx.x % 32;
      if constexpr (MODE >= kWgrad) mine = base + lane < p.g.experts ? p.m_tiles * p.n_tiles : 0;
      else mine = static_cast<int32_t>((end - begin + kSpan - 1) / kSpan) * p.m_tiles;
      upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      upto += total;
      total = __shfl_sync(0xffffffffu, upto, 31);
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, tile < upto)) - 1;
    const int64_t b = __shfl_sync(0xffffffffu, begin, src), e = __shfl_sync(0xffffffffu, end, src);
    const int32_t local = tile - __shfl_sync(0xffffffffu, upto - mine, src);
    t.e = base + src;
    constexpr int32_t kWidth = kStepK * subs_of(SHAPE);
    if constexpr (MODE >= kWgrad) {
      t.m0 = local / p.n_tiles * 256;
      t.n0 = local % p.n_tiles * p.tile_n;
      t.width = t.valid = p.tile_n;
      t.parts = 1;
      t.row0 = b;
      t.steps = static_cast<int32_t>((e - b + kWidth - 1) / kWidth);
      t.tail = static_cast<int32_t>((e - b) % kWidth);
    } else {
      const int32_t size = static_cast<int32_t>(e - b), tiles = (size + kSpan - 1) / kSpan;
      const int32_t span = (size + tiles - 1) / tiles;
      const int32_t parts = SHAPE == kTwo && span > 256 ? 2 : 1;
      t.width = ((span + parts - 1) / parts + 31) / 32 * 32;
      t.m0 = local / tiles * 256;
      t.n0 = local % tiles * parts * t.width;
      t.row0 = b + t.n0;
      t.valid = min(parts * t.width, size - t.n0);
      t.parts = t.valid > t.width ? 2 : 1;   // the last tile of a group may end within its first accumulator
      t.steps = (p.red + kWidth - 1) / kWidth;
      t.tail = p.red % kWidth;
    }
    t.first = t.split = 0;
    if (p.splits > 1) {
      t.split = unit - tile * p.splits;
      const int32_t steps = t.steps;
      t.first = steps * t.split / p.splits;
      t.steps = steps * (t.split + 1) / p.splits - t.first;
      if (t.first + t.steps != steps) t.tail = 0;
    }
    return true;
  }
};

// Writes 32 x 32 pieces of an accumulator: one writer warp's M rows by 32 columns.
template <int MODE, bool RUNS>
struct Writer {
  const PairParams& p;
  uint8_t* stage;    // 32 lines of 64 B (their 16-byte pieces permuted as SWIZZLE_64B), or 16 plain ones of 128 B
  int lane;
  int32_t e = 0, m = 0, cols = 0;   // which result (expert, run of the reduction); first M row; columns there are
  bool add = false;                 // to what is there
  int64_t n0 = 0;                   // column 0 in the output: row products: its row; weight gradient: its column

  // An f32 result, or its addition without waiting for what is there.  Each value has one writer, whose additions
  // to an address keep their order.
  __device__ __forceinline__ void put(float* dst, float v) const {
    if (add) atomicAdd(dst, v);
    else *dst = v;
  }
  // The staging tile is free once the store before has read it.
  __device__ __forceinline__ void stage_free() const {
    if (elect_one()) bulk_wait_read();
    __syncwarp();
  }
  __device__ __forceinline__ bool f32() const { return RUNS || p.f32; }
  // Row products that leave by TMA take fragments, everything else a row of 32 columns a lane.
  __device__ __forceinline__ void load(uint32_t acc, uint32_t (&r)[32]) const {
    if (MODE != kWgrad && p.tma_out && (MODE < kWgrad || !f32())) {
      tmem_ld_fragments<0>(acc, r);
      tmem_ld_fragments<16>(acc + (16u << 16), r);
    } else {
      tmem_ld32(acc, r);
    }
  }
  __device__ __forceinline__ void write(int32_t col, uint32_t (&r)[32]) {
    if constexpr (MODE == kWgrad) write_gradient(col, r);
    else if (MODE == kWgradT && p.tma_out && f32()) write_lines(col, r);
    else if (p.tma_out) write_rows(col, r);
    else write_elements(col, r);
  }

  // Tensor memory holds a feature a lane and a row a column: 8 x 8 fragments are
  // stored transposed, into lines of 32 features of one row, and a full tile of 32
  // rows leaves by TMA (a weight gradient's always does: its matrix ends at n, not at a neighbour).
  __device__ __forceinline__ void write_rows(int32_t col, uint32_t (&r)[32]) {
    const int32_t rows = min(32, cols - col);
    pack_pairs(r, p.bf16);   // words 0..7: lanes 0..15, 8..15: lanes 16..31
    stage_free();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int line = 8 * i + lane % 8;
      stmatrix_t(smem_u32(stage) + line * 64 + ((lane / 8 ^ (line >> 1 & 3)) << 4), r[2 * i], r[2 * i + 1], r[8 + 2 * i],
                 r[8 + 2 * i + 1]);
    }
    if (MODE == kWgradT || rows == 32) {
      fence_proxy_async_smem();
      __syncwarp();
      if (elect_one()) {
        if constexpr (MODE == kWgradT) tma_store_3d(&p.out, stage, m, static_cast<int32_t>(n0) + col, e);
        else tma_store_2d(&p.out, stage, m, static_cast<int32_t>(n0) + col);
        bulk_commit();
      }
    } else {   // the group's last rows: the next ones are another group's
      __syncwarp();
      uint16_t* dst = static_cast<uint16_t*>(p.dst) + (n0 + col) * p.ld + m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int line = 8 * i + lane / 4, q = lane % 4;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + line * 64 + ((q ^ (line >> 1 & 3)) << 4));
        if (line < rows) store_8(dst + line * p.ld + q * 8, v, p.m_len - m - q * 8);
      }
      __syncwarp();
    }
  }

  // f32 of a transposed gradient, lane = k, register = n: 16 lines of 128 bytes at a time.
  __device__ __forceinline__ void write_lines(int32_t col, uint32_t (&r)[32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (16 * h >= cols - col) break;
      stage_free();
#pragma unroll
      for (int j = 0; j < 16; ++j) reinterpret_cast<uint32_t*>(stage)[32 * j + lane] = r[16 * h + j];
      fence_proxy_async_smem();
      __syncwarp();
      if (elect_one()) {
        const int32_t y = static_cast<int32_t>(n0) + col + 16 * h;
        if (add) tma_add_3d(&p.out, stage, m, y, e);
        else tma_store_3d(&p.out, stage, m, y, e);
        bulk_commit();
      }
    }
  }

  // f32 rows, and outputs that TMA cannot address: lane = feature, register = row,
  // a warp's store is 32 features of one row.
  __device__ __forceinline__ void write_elements(int32_t col, uint32_t (&r)[32]) const {
    const int32_t rows = m + lane < p.m_len ? min(32, cols - col) : 0;
    const int64_t at = e * (MODE == kWgradT ? p.stride_e : p.stride_split) + (n0 + col) * p.ld + m + lane;
    if (f32()) {
      float* dst = static_cast<float*>(p.dst) + at;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < rows) put(dst + j * p.ld, __uint_as_float(r[j]));
    } else {
      uint16_t* dst = static_cast<uint16_t*>(p.dst) + at;
      if (add) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < rows) r[j] = __float_as_uint(__uint_as_float(r[j]) + widen16(dst[j * p.ld], p.bf16));
      }
      pack_each(r, p.bf16);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < rows) dst[j * p.ld] = static_cast<uint16_t>(r[j]);
    }
    __syncwarp();
  }

  // lane = n, register = k: 64-byte lines through shared memory, stored by TMA,
  // which cuts them at the matrix's edges; by element where TMA cannot.
  __device__ __forceinline__ void write_gradient(int32_t col, uint32_t (&r)[32]) {
    if (p.tma_out) {
      if (!f32()) pack_pairs(r, p.bf16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // 16 words a line: 32 columns of 16 bits, or 16 of f32 twice
        if (h == 1 && !f32()) break;
        stage_free();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) =
              make_uint4(r[16 * h + 4 * q], r[16 * h + 4 * q + 1], r[16 * h + 4 * q + 2], r[16 * h + 4 * q + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
          const int32_t x = static_cast<int32_t>(n0) + col + 16 * h;
          if (add) tma_add_3d(&p.out, stage, x, m, e);
          else tma_store_3d(&p.out, stage, x, m, e);
          bulk_commit();
        }
      }
      return;
    }
    const int64_t at = e * p.stride_e + (m + lane) * p.ld + n0 + col;
    const int32_t count = m + lane < p.m_len ? min(32, cols - col) : 0;
    if (f32()) {
      float* dst = static_cast<float*>(p.dst) + at;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) put(dst + j, __uint_as_float(r[j]));
    } else {
      uint16_t* dst = static_cast<uint16_t*>(p.dst) + at;
      if (add) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < count) r[j] = __float_as_uint(__uint_as_float(r[j]) + widen16(dst[j], p.bf16));
      }
      pack_each(r, p.bf16);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < count) dst[j] = static_cast<uint16_t>(r[j]);
    }
    __syncwarp();
  }
};

struct PairCtrl {
  uint64_t full[kMaxStages], empty[kMaxStages], tail[kMaxStages];
  uint64_t acc_full[2], acc_empty[2], done;
  uint32_t tmem;
  int abort;
};

template <int MODE, int SHAPE, bool RUNS>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    grouped_pair_kernel(const __grid_constant__ PairParams p) {
  constexpr bool WIDE = SHAPE == kTwo;
  constexpr int kSubs = subs_of(SHAPE);
  constexpr uint32_t kStages = SHAPE == kOne ? 6 : SHAPE == kNarrow ? 5 : 4;
  constexpr uint32_t kBBytes = kOperandBytes / (SHAPE == kNarrow ? 4 : SHAPE == kMiddle ? 2 : 1);   // B of a 64-wide block
  constexpr uint32_t kStageBytes = kSubs * (kOperandBytes + (WIDE ? 2 : 1) * kBBytes);
  static_assert(kStages <= kMaxStages && kStages * kStageBytes <= kRingBytes);
  extern __shared__ uint8_t raw[];
  uint8_t* base = raw + (1024 - smem_u32(raw) % 1024) % 1024;
  uint8_t* ring = base;
  uint8_t* staging = ring + kRingBytes;
  PairCtrl* c = reinterpret_cast<PairCtrl*>(staging + kWriters * kStoreBytes);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  volatile int* abort = &c->abort;
  if (warp == 0) {   // a barrier a lane
    if (lane < kMaxStages) {
      mbar_init(&c->full[lane], 2);    // one arrival of each CTA
      mbar_init(&c->empty[lane], 1);   // the products' commit
      mbar_init(&c->tail[lane], 2);
    } else if (lane < kMaxStages + 2) {
      mbar_init(&c->acc_full[lane - kMaxStages], 1);
      mbar_init(&c->acc_empty[lane - kMaxStages], 2 * kWriters);
    } else if (lane == kMaxStages + 2) {
      mbar_init(&c->done, 1);
      c->abort = 0;
    }
    fence_mbar_init();
  } else if (warp == 1) {
    if (lane == 0) {
      prefetch_tmap(&p.a);
      prefetch_tmap(&p.b[0]);
    }
  } else if (warp == 2) pair_tmem_alloc(&c->tmem, 512);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = c->tmem;
  pdl_wait();
  pdl_launch_dependents();   // one wave: whoever waits for this grid may take its place on the SMs as they fall free

  const int32_t first = blockIdx.x / 2, stride = gridDim.x / 2;
  Walker<MODE, SHAPE, RUNS> walk;
  Tile t;
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    uint32_t it = 0, st = 0, phase = 1;
    uint32_t tails = 0, tail_odd = 0;   // a bit a stage: whether it has held a tail, whether an odd number of them
    bool ok = true;
    for (int32_t tile = first; ok && walk.next(p, tile, stride, t);) {
      const int32_t halves[2] = {t.columns(0) / 2, WIDE && t.parts > 1 ? t.columns(1) / 2 : 0};
      const int32_t m = t.m0 + static_cast<int32_t>(rank) * 128;
      const uint32_t bytes =
          kOperandBytes + (MODE >= kWgrad ? kBBytes : static_cast<uint32_t>(halves[0] + halves[1]) * kStepK * 2);
      for (int32_t s = 0; s < t.steps; ++s, ++it) {
        ok = warp_wait(&c->empty[st], phase, abort, p.dev_err);
        if (!ok) break;
        uint8_t* a = ring + st * kStageBytes;
        uint8_t* b = a + kSubs * kOperandBytes;
        // a step whose rows past the group's end are still to be zeroed lands on another barrier
        const bool last = s + 1 == t.steps;
        const bool fix = MODE >= kWgrad && last && t.tail % 16 != 0;
        const uint32_t bar = peer_addr(fix ? &c->tail[st] : &c->full[st], 0);
        if (fix) { tails |= 1u << st; tail_odd ^= 1u << st; }
        const int subs = kSubs > 1 && last && t.tail ? (t.tail + kStepK - 1) / kStepK : kSubs;
        if (elect_one()) {
          pair_arrive_expect_tx(bar, subs * bytes);
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub) {
            if (sub >= subs) break;
            const int32_t r = ((t.first + s) * kSubs + sub) * kStepK;   // where the block begins in the reduction
            if constexpr (MODE == kRowsK) {
              pair_load_3d(a, &p.a, bar, r, m, t.e);
            } else if constexpr (MODE == kRowsMN) {
              pair_load_3d(a, &p.a, bar, m, r, t.e);
              pair_load_3d(a + kChunkBytes, &p.a, bar, m + 64, r, t.e);
            } else {
              const int32_t y = static_cast<int32_t>(t.row0) + r;
              pair_load_2d(a, &p.a, bar, m, y);
              pair_load_2d(a + kChunkBytes, &p.a, bar, m + 64, y);
            }
            if constexpr (MODE >= kWgrad) {
              const int32_t y = static_cast<int32_t>(t.row0) + r, x = t.n0 + static_cast<int32_t>(rank) * halves[0];
              pair_load_2d(b, &p.b[0], bar, x, y);
              if constexpr (kBBytes > kChunkBytes) pair_load_2d(b + kChunkBytes, &p.b[0], bar, x + 64, y);
            } else {
#pragma unroll
              for (int part = 0; part < (WIDE ? 2 : 1); ++part) {
                if (part >= t.parts) break;
                const int32_t half = halves[part];
                uint8_t* to = b + part * kOperandBytes;
                int32_t y = static_cast<int32_t>(t.row0) + part * t.width + static_cast<int32_t>(rank) * half;
#pragma unroll
                for (int i = kBoxes - 1; i >= 0; --i) {   // the rows' number in boxes of 128, 64, 32, 16
                  if (half & (16 << i)) {
                    pair_load_2d(to, &p.b[i], bar, r, y);
                    to += (16 << i) * kStepK * 2;
                    y += 16 << i;
                  }
                }
              }
            }
            a += kOperandBytes;
            b += kBBytes;
          }
        }
        __syncwarp();
        if (++st == kStages) { st = 0; phase ^= 1; }
      }
    }
    if (walk.bad && blockIdx.x == 0) atomicOr(p.dev_err, kDevErrOffsets);
    if (ok && lane == 0) {   // the last steps are released to both CTAs before either leaves
      for (uint32_t back = 0; back < kStages && back < it; ++back) {
        const uint32_t j = it - 1 - back;
        mbar_wait(&c->empty[j % kStages], (j / kStages) & 1, abort, p.dev_err);
      }
    }
    if (*abort && lane == 0 && leader) {   // copies of both CTAs still in flight: wait for them, with a limit
      int ignore = 0;
      for (uint32_t back = 0; back < kStages && back < it; ++back) {
        const uint32_t j = it - 1 - back;
        mbar_wait(&c->full[j % kStages], (j / kStages) & 1, &ignore, p.dev_err);
      }
    }
    if (MODE >= kWgrad && *abort && lane == 0 && leader) {   // and for the steps that land on the tails' barriers
      int ignore = 0;
      for (uint32_t j = 0; j < kStages; ++j)
        if (tails >> j & 1) mbar_wait(&c->tail[j], ~tail_odd >> j & 1, &ignore, p.dev_err);
    }
  } else if (warp == 1 && leader) {
    // ------------------------------------------------------------- products
    uint32_t n = 0, st = 0, phase = 0;
    bool ok = true;
    for (int32_t tile = first; ok && walk.next(p, tile, stride, t);) {
      if (t.steps == 0) continue;   // an empty group's gradient: zeros, without an accumulator
      constexpr uint32_t kMajors = (MODE != kRowsK ? kIdescMajorA : 0) | (MODE >= kWgrad ? kIdescMajorB : 0);
      const uint32_t idescs[2] = {umma_idesc(p.bf16, 256, t.columns(0)) | kMajors,
                                  WIDE && t.parts > 1 ? umma_idesc(p.bf16, 256, t.columns(1)) | kMajors : 0};
      for (int32_t s = 0; ok && s < t.steps; ++s) {
        const bool last = s + 1 == t.steps;
        ok = warp_wait(&c->full[st], phase, abort, p.dev_err);
        const uint32_t a = smem_u32(ring + st * kStageBytes);
        const uint64_t da = MODE == kRowsK ? sw128_desc(a) : sw128_mn_desc(a, kChunkBytes);
        const int count = last && t.tail ? (t.tail + 15) / 16 : kSubs * kStepK / 16;   // products of 16
#pragma unroll
        for (int part = 0; part < (WIDE ? 2 : 1); ++part) {
          if (part >= t.parts) break;
          const uint32_t buf = (n + part) % 2, acc = tmem + buf * kAccCols;
          if (s == 0) ok = ok && warp_wait(&c->acc_empty[buf], ((n + part) / 2 + 1) & 1, abort, p.dev_err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b = a + kSubs * kOperandBytes + part * kOperandBytes;
          const uint64_t db = MODE >= kWgrad ? sw128_mn_desc(b, kChunkBytes) : sw128_desc(b);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kSubs * kStepK / 16; ++k)   // the next 64-wide block of an operand: its bytes / 16 on
              if (k < count)
                pair_umma_f16(acc, da + k % 4 * (MODE == kRowsK ? 2 : 128) + k / 4 * (kOperandBytes >> 4),
                              db + k % 4 * (MODE >= kWgrad ? 128 : 2) + k / 4 * (kBBytes >> 4), idescs[part], s | k);
            if (part + 1 == t.parts) pair_umma_commit(&c->empty[st]);
            if (last) pair_umma_commit(&c->acc_full[buf]);
          }
          __syncwarp();
        }
        if (++st == kStages) { st = 0; phase ^= 1; }
      }
      n += t.parts;
    }
    if (*abort && lane == 0) {   // products in flight end before their tensor memory goes
      int ignore = 0;
      pair_umma_commit(&c->done);
      mbar_wait(&c->done, 0, &ignore, p.dev_err);
    }
  } else if ((warp == 2 || warp == 3) && MODE >= kWgrad && leader) {
    // ---------------------------------------------------------------- tails
    // A warp for each CTA's shared memory, both in the leader: what they clear reaches the products by way of an
    // arrival in their own CTA.  A warp in either CTA would have to release to the other (96 x 1536 x 2048, 341 rows: 235
    // us against 214, or 219 with the wide fence in both; without clearing anything 205, mostly for want of the fence).
    const uint32_t cta = warp - 2;
    uint32_t it = 0;
    int uses = 0;   // lane s: how many tails stage s has held
    bool ok = true;
    for (int32_t tile = first; ok && walk.next(p, tile, stride, t);) {
      it += t.steps;
      if (t.tail % 16 == 0) continue;
      const uint32_t st = (it - 1) % kStages;
      ok = warp_wait(&c->tail[st], __shfl_sync(0xffffffffu, uses, st) & 1, abort, p.dev_err);
      if (lane == static_cast<int>(st)) ++uses;
      const uint32_t sub = t.tail / kStepK;
      const uint8_t* a = ring + st * kStageBytes + sub * kOperandBytes;
      const uint8_t* b = ring + st * kStageBytes + kSubs * kOperandBytes + sub * kBBytes;
      const int zeros = (16 - t.tail % 16) * 8;   // 16-byte pieces in the lines to clear, per 64-column chunk
      constexpr uint32_t kChunks = 2 + kBBytes / kChunkBytes;
#pragma unroll
      for (uint32_t chunk = 0; chunk < kChunks; ++chunk) {
        const uint32_t at =
            peer_addr(chunk < 2 ? a + chunk * kChunkBytes : b + (chunk - 2) * kChunkBytes, cta) + t.tail % kStepK * 128;
        for (int i = lane; ok && i < zeros; i += 32) pair_store_zeros(at + 16 * i);
      }
      if (cta == 0) fence_proxy_async_smem();
      else fence_proxy_async();
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&c->full[st]);
    }
  } else if (warp >= 4) {
    // -------------------------------------------------------------- results
    const int quad = warp % 4, part = (warp - 4) / 4;   // 32 of the CTA's M rows, every other 32 columns
    Writer<MODE, RUNS> out{p, staging + (warp - 4) * kStoreBytes, lane};
    uint32_t n = 0;
    bool ok = true;
    for (int32_t tile = first; ok && walk.next(p, tile, stride, t);) {
      out.e = MODE >= kWgrad ? t.split * p.g.experts + t.e : t.split;
      out.m = t.m0 + static_cast<int32_t>(rank) * 128 + quad * 32;
      out.add = p.accumulate || (RUNS && t.add);
      if (RUNS && t.add && p.tma_out) {   // the stores of the run before have arrived: additions to the same values stay in order
        if (elect_one()) bulk_wait_all();
        __syncwarp();
      }
      for (int acc_n = 0; acc_n < (WIDE ? t.parts : 1); ++acc_n) {
        const int32_t cols = MODE >= kWgrad ? min(t.width, p.n_len - t.n0) : min(t.width, t.valid - acc_n * t.width);
        const int chunks = out.m < p.m_len && cols > part * 32 ? (cols - part * 32 + 63) / 64 : 0;
        out.cols = cols;
        out.n0 = MODE >= kWgrad ? t.n0 : t.row0 + acc_n * t.width;
        uint32_t r0[32], r1[32];
        if (t.steps == 0) {   // an empty group's gradient
          if (p.accumulate) continue;
          for (int i = 0; i < chunks; ++i) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r0[j] = 0;
            out.write(part * 32 + 64 * i, r0);
          }
          continue;
        }
        const uint32_t buf = n % 2, acc = tmem + buf * kAccCols + (static_cast<uint32_t>(quad) * 32 << 16) + part * 32;
        ok = warp_wait(&c->acc_full[buf], (n / 2) & 1, abort, p.dev_err);
        if (!ok) break;
        tc_fence_after();
        ++n;
        // a chunk is written while the next one's load is under way; the accumulator is free once the last is read
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) pair_arrive(peer_addr(&c->acc_empty[buf], 0));
        };
        if (chunks == 0) release();
        else out.load(acc, r0);
        for (int i = 0; i < chunks; i += 2) {
          tmem_ld_wait_for(r0);
          if (i + 1 < chunks) out.load(acc + 64 * (i + 1), r1);
          else release();
          out.write(part * 32 + 64 * i, r0);
          if (i + 1 == chunks) break;
          tmem_ld_wait_for(r1);
          if (i + 2 < chunks) out.load(acc + 64 * (i + 2), r0);
          else release();
          out.write(part * 32 + 64 * (i + 1), r1);
        }
      }
    }
    if (p.tma_out && elect_one()) bulk_wait_all();
    if (MODE < kWgrad && ok) {   // rows of no group
      const int64_t gap = walk.lo + (p.g.rows - walk.carry);
      for (int64_t j = blockIdx.x; j < gap * p.splits; j += gridDim.x) {
        const int64_t i = j % gap, at = j / gap * p.stride_split + (i < walk.lo ? i : i - walk.lo + walk.carry) * p.ld;
        for (int32_t f = threadIdx.x - 128; f < p.m_len; f += kWriters * 32) {
          if (p.f32) static_cast<float*>(p.dst)[at + f] = 0.f;
          else static_cast<uint16_t*>(p.dst)[at + f] = 0;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 2) pair_tmem_free(tmem, 512);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &q, 12000, cudaEnableDefault, &r) == cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(q);
  });
  return fn;
}

// [outer][rows][cols] with row pitch and outer stride in bytes (dims = 2 leaves
// the outer one away).
int make_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int dims, uint64_t cols, uint64_t rows,
             uint64_t outer, uint64_t pitch, uint64_t stride, uint32_t box_cols, uint32_t box_rows,
             CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  auto fn = encode_fn();
  if (!fn) return report_error(HEXMOE_E_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t size[3] = {cols, rows, outer}, strides[2] = {pitch, stride};
  const cuuint32_t box[3] = {box_cols, box_rows, 1}, step[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(m, dt, dims, const_cast<void*>(base), size, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {   // a host thread that has launched nothing yet: runtime calls bind it, this one does not
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  }
  if (r == CUDA_SUCCESS) return HEXMOE_OK;
  char buf[96];
  snprintf(buf, sizeof(buf), "grouped product: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return report_error(HEXMOE_E_CUDA, buf);
}

// Whether TMA can address a matrix: base and strides in multiples of 16 bytes.
bool tma_rows(const void* p, int64_t ld, int64_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0 && ld * size < (1ll << 40);
}
bool tma_stack(const void* p, int64_t ld, int64_t stride, int64_t size, int32_t count) {
  return tma_rows(p, ld, size) &&
         (count == 1 || (stride * size % 16 == 0 && stride >= ld && stride * size < (1ll << 40)));
}

#define PAIR_KERNELS(MODE, SHAPE)                                             \
  reinterpret_cast<const void*>(grouped_pair_kernel<MODE, SHAPE, false>), \
      reinterpret_cast<const void*>(grouped_pair_kernel<MODE, SHAPE, true>)

int sm_count(int* sms) {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return report_cuda_error(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return report_error(HEXMOE_E_DEVICE, "device ordinal out of range");
  int v = cached[dev].load(std::memory_order_acquire);
  if (!v) {   // first call on this device: the kernels' shared memory as well
    for (const void* k : {PAIR_KERNELS(kRowsK, kOne), PAIR_KERNELS(kRowsK, kTwo), PAIR_KERNELS(kRowsK, kNarrow),
                          PAIR_KERNELS(kRowsK, kMiddle), PAIR_KERNELS(kRowsMN, kOne), PAIR_KERNELS(kRowsMN, kTwo),
                          PAIR_KERNELS(kRowsMN, kNarrow), PAIR_KERNELS(kRowsMN, kMiddle), PAIR_KERNELS(kWgrad, kOne),
                          PAIR_KERNELS(kWgrad, kMiddle), PAIR_KERNELS(kWgradT, kOne), PAIR_KERNELS(kWgradT, kMiddle)}) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
      if (e != cudaSuccess) return report_cuda_error(e, "grouped product kernel");
    }
    e = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return report_cuda_error(e, "cudaDeviceGetAttribute");
    cached[dev].store(v, std::memory_order_release);
  }
  *sms = v;
  return HEXMOE_OK;
}

template <int MODE, int SHAPE>
cudaError_t launch_pair(const PairParams& p, int64_t tiles, int sms, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(sms / 2, tiles))));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.run ? cudaLaunchKernelEx(&cfg, grouped_pair_kernel<MODE, SHAPE, true>, p)
               : cudaLaunchKernelEx(&cfg, grouped_pair_kernel<MODE, SHAPE, false>, p);
}

// ------------------------------------------------------------------- splits
// Products of few tiles leave most pairs idle while a few walk a long reduction:
// their reduction is cut into `splits` runs of steps, each with an fp32 partial
// result in the workspace, which a second kernel adds in order and rounds.
constexpr int kPairsPlanned = 74;   // pairs of a B200; what the split is planned for
constexpr int kMaxSplits = 16;

// Runs for `tiles` tiles of `steps` steps and `values` results, by what they take: step_us a step (0.28 with 256
// columns, 0.14 with up to 128, 0.15 to 0.3 for a weight gradient's, by how its rows lie in memory), value_us for
// an fp32 partial written and read (row products write theirs without TMA), some 1.2 us for the second
// kernel and 0.15 a run.  With 1, 2, 4, 8 runs: 6 rows, 776 x 1624: 9.0, 8.8, 7.8, 8.1 us; 300 rows of 4 groups, 512 x
// 4096: 13.5, 11.9, 10.7, 11.7; 500 rows, 2048 x 2048: 10.0, 14.8, 17.0, 23.1; weight gradient of 2 x 4000 rows,
// 256 x 512: 13.9, 12.1, 10.4, 12.2.
struct SplitPlan {
  int splits;
  double us;
};
SplitPlan plan_splits(int64_t tiles, int64_t steps, double step_us, int64_t values, double value_us) {
  const int64_t most = std::min<int64_t>({kPairsPlanned / std::max<int64_t>(tiles, 1), steps / 4, kMaxSplits});
  SplitPlan best = {1, step_us * static_cast<double>(steps)};
  for (int s = 2; s <= most; ++s) {
    const double us = step_us * static_cast<double>((steps + s - 1) / s) + 1.2 + 0.15 * s +
                      value_us * static_cast<double>(s * values);
    if (us < best.us) best = {s, us};
  }
  return best;
}
int64_t pitch4(int64_t n) { return (n + 3) / 4 * 4; }   // f32 rows of whole 16-byte pieces

// Most tiles that rows in groups can make with a shape.
int64_t row_tiles(int64_t rows, int32_t experts, int32_t m_len, PairShape shape) {
  return (rows / span_of(shape) + std::min<int64_t>(experts, rows)) * ((m_len + 255) / 256);
}
// The shape for groups of this mean size.  Steps 128 wide pay up to tiles of 128 columns (32 experts x 30
// rows x 512 x 2048: 11.9 us against 14.3), and narrower tiles wherever every one of them still has a pair of
// its own (1511 rows, 192 x 1472: 7.6 us narrow, 8.0 middle, 11.4 one; 3296 rows of 2 experts, 512 x 872, 106 tiles
// narrow: 9.3, 7.8, 9.6; 484 rows of 3, 3872 x 3768, 96 tiles middle: 37.0 middle, 26.9 one).  Two accumulators a
// tile where groups of 257..512 rows are the rule (the matrix is then loaded once a group, not twice: 96 x 341
// rows, 1536 x 2048: 182 us against 194) and still fill the machine; with larger groups the drain between tiles
// costs more than it saves (8192^2 x 2048: 180 us against 174).
PairShape rows_shape(int64_t rows, int32_t experts, int32_t m_len) {
  if (rows <= 64 || rows <= 32ll * experts || row_tiles(rows, experts, m_len, kNarrow) <= kPairsPlanned) return kNarrow;
  if (rows <= 128 || rows <= 96ll * experts || row_tiles(rows, experts, m_len, kMiddle) <= kPairsPlanned) return kMiddle;
  const bool fills = static_cast<int64_t>(experts) * ((m_len + 255) / 256) >= 2 * kPairsPlanned;
  return rows > 256ll * experts && rows <= 512ll * experts && fills ? kTwo : kOne;
}
int rows_splits(int64_t rows, int32_t experts, int32_t m_len, int32_t red) {
  const PairShape shape = rows_shape(rows, experts, m_len);
  return plan_splits(row_tiles(rows, experts, m_len, shape), (red + kStepK - 1) / kStepK,
                     span_of(shape) >= 256 ? 0.28 : 0.14, rows * m_len, 3.3e-6)
      .splits;
}
int64_t wgrad_tiles(int32_t experts, int32_t m_len, int32_t n_len, PairShape shape) {
  return static_cast<int64_t>(experts) * ((m_len + 255) / 256) * ((n_len + span_of(shape) - 1) / span_of(shape));
}
SplitPlan wgrad_plan(int64_t rows, int32_t experts, int32_t m_len, int32_t n_len, PairShape shape) {
  return plan_splits(wgrad_tiles(experts, m_len, n_len, shape), rows / experts / kStepK, shape == kOne ? 0.28 : 0.17,
                     static_cast<int64_t>(experts) * m_len * n_len, 1.7e-6);
}
// Tiles of 128 columns and steps of 128 rows where each tile still has a pair of its own, or where there are no more
// columns (2790 rows of 9 groups, 256 x 128: 6.2 us against 6.6; 8192 rows, 512 x 512, unsplit: 23.8 against 42.1;
// 15244 rows of 77, 120 x 112: 12.8 against 15.1).  With more tiles than pairs they lose (1125 rows of 4, 432 x 3712:
// 10.9 us against 9.4), and where twice as wide ones may share a reduction that these may not (20787 rows of 3,
// 120 x 2232 with n on the M side: 43.2 against 34.2).
PairShape wgrad_shape(int64_t rows, int32_t experts, int32_t m_len, int32_t n_len) {
  if (n_len <= span_of(kMiddle)) return kMiddle;
  if (wgrad_tiles(experts, m_len, n_len, kMiddle) > kPairsPlanned) return kOne;
  const double middle = wgrad_plan(rows, experts, m_len, n_len, kMiddle).us;
  return middle <= wgrad_plan(rows, experts, m_len, n_len, kOne).us ? kMiddle : kOne;
}
// Whether x's columns are the M side and dy's the N side (kWgradT) rather than the other way about: where that pads
// the matrix by less, and it counts because there are more tiles than pairs (2084 rows of 84 groups, 88 x 1336: 14.3
// us against 19.4; 14 rows of 90, 352 x 1464: 24.9 against 29.3) or because the runs of a split get shorter (20787
// rows of 3, 120 x 2232: 27.7 against 33.9).  Elsewhere it gains nothing (3378 rows, 352 x 2136: 16.8 against 15.8).
bool wgrad_swaps(int64_t rows, int32_t experts, int32_t n, int32_t k) {
  const auto area = [](int64_t m_len, int64_t n_len) { return (m_len + 255) / 256 * 256 * ((n_len + 63) / 64 * 64); };
  if (10 * area(k, n) >= 9 * area(n, k)) return false;
  if (wgrad_tiles(experts, n, k, kMiddle) > kPairsPlanned) return true;
  const auto us = [&](int32_t m_len, int32_t n_len) {
    return wgrad_plan(rows, experts, m_len, n_len, wgrad_shape(rows, experts, m_len, n_len)).us;
  };
  return us(k, n) < us(n, k);
}
int wgrad_splits(int64_t rows, int32_t experts, int32_t n, int32_t k) {
  const bool swap = wgrad_swaps(rows, experts, n, k);
  const int32_t m_len = swap ? k : n, n_len = swap ? n : k;
  return wgrad_plan(rows, experts, m_len, n_len, wgrad_shape(rows, experts, m_len, n_len)).splits;
}

struct JoinParams {
  const float* part;   // [splits][rows][pitch]
  int64_t rows, pitch;
  int32_t splits, cols;
  void* out;           // row r: matrix r / inner, its row r % inner
  int64_t ld, stride;
  int32_t inner, f32, bf16, accumulate, vec;
};

__global__ void __launch_bounds__(256) grouped_join_kernel(const JoinParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int32_t pieces = static_cast<int32_t>(p.pitch / 4);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.rows * pieces) return;
  const int64_t row = i / pieces;
  const int32_t col = static_cast<int32_t>(i % pieces) * 4;
  float v[4] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float4 f = *reinterpret_cast<const float4*>(p.part + (s * p.rows + row) * p.pitch + col);
    v[0] += f.x;
    v[1] += f.y;
    v[2] += f.z;
    v[3] += f.w;
  }
  const int64_t at = row / p.inner * p.stride + row % p.inner * p.ld + col;
  const int count = min(4, p.cols - col);
  if (p.f32) {
    float* o = static_cast<float*>(p.out) + at;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < count) o[j] = p.accumulate ? o[j] + v[j] : v[j];
  } else {
    uint16_t* o = static_cast<uint16_t*>(p.out) + at;
    if (p.vec && !p.accumulate && count == 4) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack16(v[0], v[1], p.bf16), pack16(v[2], v[3], p.bf16));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < count) o[j] = round16(p.accumulate ? widen16(o[j], p.bf16) + v[j] : v[j], p.bf16);
    }
  }
}

cudaError_t launch_join(const JoinParams& p, cudaStream_t st) {
  const int64_t blocks = (p.rows * (p.pitch / 4) + 255) / 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, grouped_join_kernel, p);
}

int check_groups(const char* what, int64_t rows, int32_t experts, const void* offsets, int32_t offsets_dtype) {
  if (offsets_dtype != HEXMOE_I32 && offsets_dtype != HEXMOE_I64) return report_error(HEXMOE_E_DTYPE, "offsets are I32 or I64");
  if (rows < 0 || rows >= (1ll << 31) - 512) return arg_error("%s: %lld rows", what, static_cast<long long>(rows));
  if (experts <= 0 || experts > 2048) return arg_error("%s: %d experts outside 1..2048", what, experts);
  if (!offsets || reinterpret_cast<uintptr_t>(offsets) % (offsets_dtype == HEXMOE_I64 ? 8 : 4))
    return arg_error("%s: offsets null or not aligned", what);
  return HEXMOE_OK;
}

bool is16(int32_t dt) { return dt == HEXMOE_BF16 || dt == HEXMOE_F16; }
bool off_by(const void* p, size_t z) { return reinterpret_cast<uintptr_t>(p) % z != 0; }

}  // namespace
}  // namespace hexmoe

using namespace hexmoe;

extern "C" {

int hexmoe_group_offsets(const int32_t* expert_ids, int64_t max_blocks, const int32_t* npp, int32_t block_m,
                         int32_t num_experts, int32_t* offsets, void* stream) {
  if (max_blocks < 0 || block_m <= 0 || num_experts <= 0 || num_experts > 2048 || max_blocks * block_m >= (1ll << 31))
    return arg_error("hexmoe_group_offsets: %lld blocks of %d, %d experts", static_cast<long long>(max_blocks), block_m,
                     num_experts);
  if (!npp || !offsets || (max_blocks > 0 && !expert_ids)) return arg_error("hexmoe_group_offsets: null pointer");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_experts / 256 + 1);
  cfg.blockDim = dim3(256);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, group_offsets_kernel, expert_ids, max_blocks, npp, block_m, num_experts,
                                           offsets);
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, "hexmoe_group_offsets");
}

size_t hexmoe_grouped_mm_workspace_bytes(int64_t rows, int32_t experts, int32_t n, int32_t k, int32_t transpose) {
  if (rows <= 0 || experts <= 0 || n <= 0 || k <= 0) return 0;
  const int32_t width_out = transpose ? k : n, splits = rows_splits(rows, experts, width_out, transpose ? n : k);
  return splits > 1 ? splits * rows * pitch4(width_out) * sizeof(float) : 0;
}

size_t hexmoe_grouped_wgrad_workspace_bytes(int64_t rows, int32_t experts, int32_t n, int32_t k) {
  if (rows <= 0 || experts <= 0 || n <= 0 || k <= 0) return 0;
  const int32_t splits = wgrad_splits(rows, experts, n, k);
  return splits > 1 ? splits * static_cast<size_t>(experts) * n * pitch4(k) * sizeof(float) : 0;
}

int hexmoe_grouped_mm(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int64_t stride_w, int32_t dtype,
                      int64_t rows, int32_t experts, int32_t n, int32_t k, int32_t transpose, const void* offsets,
                      int32_t offsets_dtype, void* out, int64_t ld_out, int32_t out_dtype, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* what = "hexmoe_grouped_mm";
  if (!is16(dtype)) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_mm: x and w are BF16 or F16");
  if (out_dtype != dtype && out_dtype != HEXMOE_F32) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_mm: out is of x's dtype or F32");
  if (int rc = check_groups(what, rows, experts, offsets, offsets_dtype)) return rc;
  if (n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24)) return arg_error("%s: n %d, k %d", what, n, k);
  const int32_t width_in = transpose ? n : k, width_out = transpose ? k : n;
  if (ld_x < width_in || ld_w < k || stride_w < 0 || ld_out < width_out)
    return arg_error("%s: a row stride is shorter than its row", what);
  if (rows == 0) return HEXMOE_OK;
  if (!x || !w || !out || off_by(x, 2) || off_by(w, 2) || off_by(out, out_dtype == HEXMOE_F32 ? 4 : 2))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  int32_t* dev_err = device_error_word();
  if (!dev_err) return report_error(HEXMOE_E_CUDA, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Groups groups = {offsets, offsets_dtype == HEXMOE_I64, experts, rows};
  const bool f32 = out_dtype == HEXMOE_F32, bf16 = dtype == HEXMOE_BF16;
  if (workspace && off_by(workspace, 16)) return arg_error("%s: workspace not 16-byte aligned", what);
  if (tma_rows(x, ld_x, 2) && tma_stack(w, ld_w, stride_w, 2, experts)) {
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    PairParams q{};
    q.g = groups;
    q.m_len = width_out; q.red = width_in;
    q.m_tiles = (width_out + 255) / 256;
    q.splits = rows_splits(rows, experts, width_out, width_in);
    const int64_t pitch = pitch4(width_out);
    if (workspace_bytes < q.splits * rows * pitch * sizeof(float) || !workspace) q.splits = 1;
    const bool split = q.splits > 1;
    q.dst = split ? workspace : out;
    q.ld = split ? pitch : ld_out;
    q.stride_split = rows * pitch;
    q.f32 = split || f32; q.bf16 = bf16;
    q.dev_err = dev_err;
    const PairShape shape = rows_shape(rows, experts, width_out);
    q.run = f32 && width_in > kRunLength ? kRunLength / (kStepK * subs_of(shape)) : 0;
    const int64_t tiles = row_tiles(rows, experts, width_out, shape) * q.splits;
    if (tiles >= (1ll << 30)) return arg_error("%s: too many tiles", what);
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (int rc = make_map(&q.a, w, dt, 3, k, n, experts, 2 * ld_w, experts == 1 ? 2 * ld_w : 2 * stride_w, 64,
                          transpose ? 64 : 128))
      return rc;
    // box heights up to half the widest tile that these rows can make
    const int64_t half = (std::min<int64_t>(rows, 256) + 31) / 32 * 16;
    for (int i = 0; i < kBoxes && 16 << i <= half; ++i)
      if (int rc = make_map(&q.b[i], x, dt, 2, width_in, rows, 1, 2 * ld_x, 0, 64, 16u << i)) return rc;
    // a TMA store ends at a multiple of 16 bytes: it would write over what stands behind a row that does not
    q.tma_out = !q.f32 && tma_rows(out, ld_out, 2) && width_out % 8 == 0;
    if (q.tma_out && rows >= 32)   // no full tile of 32 rows otherwise
      if (int rc = make_map(&q.out, out, dt, 2, width_out, rows, 1, 2 * ld_out, 0, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B))
        return rc;
    auto launch = [&](auto mode) {
      constexpr int MODE = decltype(mode)::value;
      return shape == kNarrow   ? launch_pair<MODE, kNarrow>(q, tiles, sms, st)
             : shape == kMiddle ? launch_pair<MODE, kMiddle>(q, tiles, sms, st)
             : shape == kTwo    ? launch_pair<MODE, kTwo>(q, tiles, sms, st)
                                : launch_pair<MODE, kOne>(q, tiles, sms, st);
    };
    cudaError_t e = transpose ? launch(std::integral_constant<int, kRowsMN>{})
                              : launch(std::integral_constant<int, kRowsK>{});
    if (e == cudaSuccess && split) {
      JoinParams j{};
      j.part = static_cast<const float*>(workspace);
      j.rows = rows; j.pitch = pitch; j.splits = q.splits; j.cols = width_out;
      j.out = out; j.ld = ld_out; j.inner = static_cast<int32_t>(rows);
      j.f32 = f32; j.bf16 = bf16; j.vec = ld_out % 4 == 0 && !off_by(out, 8);
      e = launch_join(j, st);
    }
    return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
  }
  PlainParams p{};
  p.g = groups;
  p.a = static_cast<const uint16_t*>(x); p.a_i = ld_x; p.a_r = 1;
  p.b = static_cast<const uint16_t*>(w); p.b_e = stride_w;
  p.b_j = transpose ? 1 : ld_w; p.b_r = transpose ? ld_w : 1;
  p.j_len = width_out; p.r_len = width_in;
  p.out = out; p.out_i = ld_out; p.out_f32 = f32; p.bf16 = bf16;
  p.j_tiles = (width_out + kPlainTile - 1) / kPlainTile;
  p.dev_err = dev_err;
  const int64_t plain_tiles = rows / kPlainTile + std::min<int64_t>(experts, rows);
  const cudaError_t e = launch_plain(p, false, plain_tiles * p.j_tiles, st);
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

int hexmoe_grouped_wgrad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int32_t dtype, int64_t rows,
                         int32_t experts, int32_t n, int32_t k, const void* offsets, int32_t offsets_dtype, void* out,
                         int64_t ld_out, int64_t stride_out, int32_t out_dtype, int32_t accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* what = "hexmoe_grouped_wgrad";
  if (!is16(dtype)) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_wgrad: dy and x are BF16 or F16");
  if (out_dtype != dtype && out_dtype != HEXMOE_F32) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_wgrad: out is of x's dtype or F32");
  if (int rc = check_groups(what, rows, experts, offsets, offsets_dtype)) return rc;
  if (n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24)) return arg_error("%s: n %d, k %d", what, n, k);
  if (rows >= 1ll << 28) return arg_error("%s: %lld rows", what, static_cast<long long>(rows));
  if (ld_dy < n || ld_x < k || ld_out < k || stride_out < static_cast<int64_t>(n - 1) * ld_out + k)
    return arg_error("%s: a stride is shorter than what it spans", what);
  if (!out || (rows && (!dy || !x)) || off_by(dy, 2) || off_by(x, 2) || off_by(out, out_dtype == HEXMOE_F32 ? 4 : 2))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  int32_t* dev_err = device_error_word();
  if (!dev_err) return report_error(HEXMOE_E_CUDA, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Groups groups = {offsets, offsets_dtype == HEXMOE_I64, experts, rows};
  const bool f32 = out_dtype == HEXMOE_F32, bf16 = dtype == HEXMOE_BF16;
  if (workspace && off_by(workspace, 16)) return arg_error("%s: workspace not 16-byte aligned", what);
  if (rows > 0 && tma_rows(dy, ld_dy, 2) && tma_rows(x, ld_x, 2)) {
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    PairParams q{};
    q.g = groups;
    const bool swap = wgrad_swaps(rows, experts, n, k);
    q.m_len = swap ? k : n; q.n_len = swap ? n : k;
    q.m_tiles = (q.m_len + 255) / 256;
    const PairShape shape = wgrad_shape(rows, experts, q.m_len, q.n_len);
    q.n_tiles = (q.n_len + span_of(shape) - 1) / span_of(shape);
    q.tile_n = ((q.n_len + q.n_tiles - 1) / q.n_tiles + 63) / 64 * 64;
    q.splits = wgrad_splits(rows, experts, n, k);
    const int64_t pitch = pitch4(k), lines = static_cast<int64_t>(experts) * n;
    if (workspace_bytes < q.splits * lines * pitch * sizeof(float) || !workspace) q.splits = 1;
    const bool split = q.splits > 1;
    q.dst = split ? workspace : out;
    q.ld = split ? pitch : ld_out;
    q.stride_e = split ? n * pitch : stride_out;
    q.f32 = split || f32; q.bf16 = bf16; q.accumulate = accumulate && !split;
    q.run = f32 && rows > kRunLength ? kRunLength / (kStepK * subs_of(shape)) : 0;
    q.dev_err = dev_err;
    const int64_t tiles = wgrad_tiles(experts, q.m_len, q.n_len, shape) * q.splits;
    if (tiles >= (1ll << 30)) return arg_error("%s: too many tiles", what);
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (int rc = make_map(swap ? &q.b[0] : &q.a, dy, dt, 2, n, rows, 1, 2 * ld_dy, 0, 64, 64)) return rc;
    if (int rc = make_map(swap ? &q.a : &q.b[0], x, dt, 2, k, rows, 1, 2 * ld_x, 0, 64, 64)) return rc;
    // a 16-bit sum is rounded once: that of an addition to out cannot be left to TMA, which rounds before and after
    const int64_t z = q.f32 ? 4 : 2, results = static_cast<int64_t>(experts) * q.splits;
    // (and a store ends at a multiple of 16 bytes, with zeros in what a row lacks: the partials have room for that)
    q.tma_out = tma_stack(q.dst, q.ld, q.stride_e, z, static_cast<int32_t>(results)) && (split || k * z % 16 == 0) &&
                (q.f32 || !q.accumulate);
    if (q.tma_out)
      if (int rc = make_map(&q.out, q.dst, q.f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dt, 3, k, n, results, z * q.ld,
                            results == 1 ? z * q.ld : z * q.stride_e, q.f32 && !swap ? 16 : 32, q.f32 && swap ? 16 : 32,
                            q.f32 && swap ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B))
        return rc;
    cudaError_t e = swap ? shape == kOne ? launch_pair<kWgradT, kOne>(q, tiles, sms, st)
                                         : launch_pair<kWgradT, kMiddle>(q, tiles, sms, st)
                    : shape == kOne ? launch_pair<kWgrad, kOne>(q, tiles, sms, st)
                                    : launch_pair<kWgrad, kMiddle>(q, tiles, sms, st);
    if (e == cudaSuccess && split) {
      JoinParams j{};
      j.part = static_cast<const float*>(workspace);
      j.rows = lines; j.pitch = pitch; j.splits = q.splits; j.cols = k;
      j.out = out; j.ld = ld_out; j.stride = stride_out; j.inner = n;
      j.f32 = f32; j.bf16 = bf16; j.accumulate = accumulate != 0;
      j.vec = ld_out % 4 == 0 && stride_out % 4 == 0 && !off_by(out, 8);
      e = launch_join(j, st);
    }
    return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
  }
  PlainParams p{};
  p.g = groups;
  p.a = static_cast<const uint16_t*>(dy); p.a_i = 1; p.a_r = ld_dy;
  p.b = static_cast<const uint16_t*>(x); p.b_j = 1; p.b_r = ld_x;
  p.i_len = n; p.j_len = k;
  p.out = out; p.out_i = ld_out; p.out_e = stride_out;
  p.out_f32 = f32; p.accumulate = accumulate; p.bf16 = bf16;
  p.i_tiles = (n + kPlainTile - 1) / kPlainTile;
  p.j_tiles = (k + kPlainTile - 1) / kPlainTile;
  p.dev_err = dev_err;
  const int64_t blocks = static_cast<int64_t>(experts) * p.i_tiles * p.j_tiles;
  const cudaError_t e = launch_plain(p, true, blocks, st);
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

}  // extern "C"
