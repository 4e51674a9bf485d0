// grouped.cu — products of ragged row groups with their experts' 16-bit
// matrices: y = x W[e]^T, dx = dy W[e], and the weight gradients dW[e] = dy_e^T x_e.
// Group e is rows offsets[e] .. offsets[e+1]-1.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "internal.cuh"
#include "ptx.cuh"

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
  int64_t end = max(raw1 < 0 ? 0 : raw1 > g.rows ? g.rows : raw1, carry);
  int64_t first = raw0 < 0 ? 0 : raw0 > g.rows ? g.rows : raw0;
  if (lane == 0) end = max(end, max(first, carry));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {   // running maximum
    const int64_t v = __shfl_up_sync(0xffffffffu, end, o);
    if (lane >= o) end = max(end, v);
  }
  int64_t begin = __shfl_up_sync(0xffffffffu, end, 1);
  if (lane == 0) begin = max(first, carry);
  carry = __shfl_sync(0xffffffffu, end, 31);
  s.begin = begin;
  s.end = end;
  return s;
}

// ---------------------------------------------------------------- plain kernel
// out(i, j) = sum_r A(i, r) B(j, r) over operands with any element strides:
// 64 x 64 tiles, mma.sync over 32-wide reduction steps staged in shared memory
// with element loads.  It takes what the TMA kernels cannot address (a base or
// row stride that is no multiple of 16 bytes).
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
  __shared__ uint16_t ta[kPlainTile][kPlainPitch], tb[kPlainTile][kPlainPitch];
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
  float acc[2][4][4] = {};
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
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int i = wi + m * 16 + g + (h >> 1) * 8, j = wj + n * 8 + q * 2 + (h & 1);
        if (i >= i_left || j >= j_left) continue;
        const int64_t at = WGRAD ? e * p.out_e + (i0 + i) * p.out_i + j0 + j : (begin + i) * p.out_i + j0 + j;
        float v = acc[m][n][h];
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

int hexmoe_grouped_mm(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int64_t stride_w, int32_t dtype,
                      int64_t rows, int32_t experts, int32_t n, int32_t k, int32_t transpose, const void* offsets,
                      int32_t offsets_dtype, void* out, int64_t ld_out, int32_t out_dtype, void* stream) {
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
  PlainParams p{};
  p.g = {offsets, offsets_dtype == HEXMOE_I64, experts, rows};
  p.a = static_cast<const uint16_t*>(x); p.a_i = ld_x; p.a_r = 1;
  p.b = static_cast<const uint16_t*>(w); p.b_e = stride_w;
  p.b_j = transpose ? 1 : ld_w; p.b_r = transpose ? ld_w : 1;
  p.j_len = width_out; p.r_len = width_in;
  p.out = out; p.out_i = ld_out; p.out_f32 = out_dtype == HEXMOE_F32; p.bf16 = dtype == HEXMOE_BF16;
  p.j_tiles = (width_out + kPlainTile - 1) / kPlainTile;
  p.dev_err = dev_err;
  const int64_t row_tiles = rows / kPlainTile + std::min<int64_t>(experts, rows);
  const cudaError_t e = launch_plain(p, false, row_tiles * p.j_tiles, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

int hexmoe_grouped_wgrad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int32_t dtype, int64_t rows,
                         int32_t experts, int32_t n, int32_t k, const void* offsets, int32_t offsets_dtype, void* out,
                         int64_t ld_out, int64_t stride_out, int32_t out_dtype, int32_t accumulate, void* stream) {
  const char* what = "hexmoe_grouped_wgrad";
  if (!is16(dtype)) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_wgrad: dy and x are BF16 or F16");
  if (out_dtype != dtype && out_dtype != HEXMOE_F32) return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_wgrad: out is of x's dtype or F32");
  if (int rc = check_groups(what, rows, experts, offsets, offsets_dtype)) return rc;
  if (n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24)) return arg_error("%s: n %d, k %d", what, n, k);
  if (ld_dy < n || ld_x < k || ld_out < k || stride_out < static_cast<int64_t>(n - 1) * ld_out + k)
    return arg_error("%s: a stride is shorter than what it spans", what);
  if (!out || (rows && (!dy || !x)) || off_by(dy, 2) || off_by(x, 2) || off_by(out, out_dtype == HEXMOE_F32 ? 4 : 2))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  int32_t* dev_err = device_error_word();
  if (!dev_err) return report_error(HEXMOE_E_CUDA, "device error word unavailable");
  PlainParams p{};
  p.g = {offsets, offsets_dtype == HEXMOE_I64, experts, rows};
  p.a = static_cast<const uint16_t*>(dy); p.a_i = 1; p.a_r = ld_dy;
  p.b = static_cast<const uint16_t*>(x); p.b_j = 1; p.b_r = ld_x;
  p.i_len = n; p.j_len = k;
  p.out = out; p.out_i = ld_out; p.out_e = stride_out;
  p.out_f32 = out_dtype == HEXMOE_F32; p.accumulate = accumulate; p.bf16 = dtype == HEXMOE_BF16;
  p.i_tiles = (n + kPlainTile - 1) / kPlainTile;
  p.j_tiles = (k + kPlainTile - 1) / kPlainTile;
  p.dev_err = dev_err;
  const int64_t blocks = static_cast<int64_t>(experts) * p.i_tiles * p.j_tiles;
  const cudaError_t e = launch_plain(p, true, blocks, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

}  // extern "C"
