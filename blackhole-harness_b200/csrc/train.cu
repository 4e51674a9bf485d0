// train.cu — the memory-bound operators of training a MoE layer's 16-bit
// experts: SwiGLU with the routing weight (forward and backward) and the global
// gradient norm with clipping.
#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cmath>
#include <cstdio>
#include <type_traits>
#include <vector>

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

bool known_dtype(int32_t dt) { return dt == HEXMOE_F32 || dt == HEXMOE_BF16 || dt == HEXMOE_F16; }
size_t dtype_bytes(int32_t dt) { return dt == HEXMOE_F32 ? 4 : 2; }

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// V consecutive elements as one register load or store of up to 16 bytes; their
// 32-bit words by value (an address taken would put them into local memory).
template <int BYTES>
struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

__device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
__device__ __forceinline__ uint32_t word(const uint2& r, int i) { return i == 0 ? r.x : r.y; }
__device__ __forceinline__ uint32_t word(const uint32_t& r, int) { return r; }
__device__ __forceinline__ void from_words(uint4& r, const uint32_t (&w)[4]) { r = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void from_words(uint2& r, const uint32_t (&w)[4]) { r = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void from_words(uint32_t& r, const uint32_t (&w)[4]) { r = w[0]; }

template <typename T, int V>
struct Vec {
  using Raw = typename RawOf<static_cast<int>(sizeof(T)) * V>::type;
  static __device__ __forceinline__ void unpack(Raw r, float (&x)[V]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(word(r, i));
    } else if constexpr (V == 1) {
      if constexpr (std::is_same_v<T, __half>) x[0] = __half2float(__ushort_as_half(r));
      else x[0] = __bfloat162float(__ushort_as_bfloat16(r));
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const uint32_t w = word(r, i);
        if constexpr (std::is_same_v<T, __half>) {
          x[2 * i] = __half2float(__ushort_as_half(static_cast<uint16_t>(w)));
          x[2 * i + 1] = __half2float(__ushort_as_half(static_cast<uint16_t>(w >> 16)));
        } else {
          x[2 * i] = __uint_as_float(w << 16);
          x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
        }
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&x)[V]) {
    if constexpr (V == 1 && sizeof(T) == 2) {
      if constexpr (std::is_same_v<T, __half>) return __half_as_ushort(__float2half_rn(x[0]));
      else return __bfloat16_as_ushort(__float2bfloat16_rn(x[0]));
    } else {
      uint32_t w[4] = {};
      constexpr int kWords = static_cast<int>(sizeof(Raw) / 4);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (std::is_same_v<T, float>) {
          w[i] = __float_as_uint(x[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
          w[i] = __half_as_ushort(__float2half_rn(x[2 * i])) |
                 static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i + 1]))) << 16;
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = __bfloat16_as_ushort(h.x) | static_cast<uint32_t>(__bfloat16_as_ushort(h.y)) << 16;
        }
      }
      Raw r;
      from_words(r, w);
      return r;
    }
  }
};

cudaLaunchConfig_t launch_config(dim3 grid, int threads, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// ------------------------------------------------------------------- SwiGLU
// act = w silu(g) u on rows [g | u], silu(g) = g s, s = 1 / (1 + e^-g), and with
// d = dL/dact
//   dg = w d u (s + silu(g) (1 - s)),  du = w d silu(g),  dw = sum_i d silu(g) u
// Bound by HBM: 3 values of traffic per activation forward, 5 backward.  TPR
// threads take a row (a warp for common widths, a block's 128 for wide rows or
// few of them, 4 or 8 for narrow ones), so that the sum of dw stays in one
// thread group and is added in a fixed order; each thread has kUnroll 16-byte
// loads per operand in flight.  32768 x 768 bf16 with weights: forward 23.6 us (6.4
// TB/s), backward 40.8 us (6.2 TB/s).
constexpr int kSwigluThreads = 256;
// 16-byte pieces a lane has in flight: three cover 768 16-bit values a warp.  With 1, 2, 3, 4 (bf16, forward and
// backward, us): 32768 x 768: 23.5 + 38.8, 25.5 + 41.9, 24.6 + 41.5, 26.4 + 43.0; 32768 x 96: 8.0 + 12.8, 4.9 + 7.2, 4.6
// + 6.9, 4.5 + 7.5; 8191 x 517 (by element): 11.2 + 16.8, 9.1 + 14.2, 8.8 + 12.2, 7.7 + 12.6; f32 32768 x 768: 46.8 + 77.7,
// 45.6 + 76.0, 45.6 + 75.4, 48.3 + 75.4.
constexpr int kUnroll = 3;

struct SwigluParams {
  const void* h;        // [rows, 2 * inter]
  const void* dact;     // backward: [rows, inter]
  const float* weight;  // [rows] or null
  void* out;            // forward: act [rows, inter]; backward: dh [rows, 2 * inter]
  float* dweight;       // backward: [rows] or null
  int64_t rows, ld_h, ld_dact, ld_out;
  int32_t inter;
};

// s and silu(g).  1 / (1 + e^-g) itself is zero from g = -88.7 on (from -87.3 with a fast divide), where silu is still
// a normal value down to -91.
// f32: from e = exp(-|g|), with 1 + e in 1..2, by expf and the rounded divide; below -87.3 e is no normal value and is
//   off by up to 2^-150 instead.  Against the plain formula this costs 32768 x 768 nothing and shapes that stay in L2
//   2..9 % (8192 x 768 backward: 21.3 us against 19.5); a branch for the far gates cost more (21.7).
// 16 bits: numerator and denominator scaled by 2^-32, so that the denominator is finite down to g = -110.  The exponent
//   g log2 e + 32 is rounded to 2^-20 near zero and to 2^-18 at -64, the exponential and the reciprocal err by 2^-22:
//   all of it vanishes in the result's own rounding (2^-9 or 2^-12).  No slower than the plain formula (23.7 us and
//   40.8 against 23.9 and 40.8 at 32768 x 768).
template <typename T>
__device__ __forceinline__ void sigmoid_silu(float g, float& s, float& silu) {
  if constexpr (std::is_same_v<T, float>) {
    const float e = expf(-fabsf(g)), r = 1.f / (1.f + e);
    s = g < 0.f ? e * r : r;
    silu = g * s;
  } else {
    constexpr float kScale = 0x1p-32f, kLog2E = 1.44269504f;
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -kLog2E, -32.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(kScale + e));
    s = kScale * r;
    silu = g * s;
  }
}

template <typename T, int V, int TPR, bool BWD>
__global__ void __launch_bounds__(kSwigluThreads) swiglu_kernel(const SwigluParams p) {
  using VecT = Vec<T, V>;
  using Raw = typename VecT::Raw;
  constexpr int kRows = kSwigluThreads / TPR;
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
  pdl_wait();
  const bool live = row < p.rows;
  float sum = 0.f;
  if (live) {
    const T* g_row = static_cast<const T*>(p.h) + row * p.ld_h;
    const T* u_row = g_row + p.inter;
    const T* d_row = BWD ? static_cast<const T*>(p.dact) + row * p.ld_dact : nullptr;
    T* o_row = static_cast<T*>(p.out) + row * p.ld_out;
    const float w = p.weight ? p.weight[row] : 1.f;
    const int n = p.inter / V;
    for (int c0 = lane; c0 < n; c0 += TPR * kUnroll) {
      Raw g[kUnroll], u[kUnroll], d[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int c = c0 + i * TPR;
        if (c < n) {
          g[i] = reinterpret_cast<const Raw*>(g_row)[c];
          u[i] = reinterpret_cast<const Raw*>(u_row)[c];
          if constexpr (BWD) d[i] = reinterpret_cast<const Raw*>(d_row)[c];
        }
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int c = c0 + i * TPR;
        if (c >= n) continue;
        float gf[V], uf[V], df[V], a[V], b[V];
        VecT::unpack(g[i], gf);
        VecT::unpack(u[i], uf);
        if constexpr (BWD) VecT::unpack(d[i], df);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float s, silu;
          sigmoid_silu<T>(gf[j], s, silu);
          if constexpr (BWD) {
            sum += df[j] * silu * uf[j];
            const float dw = df[j] * w;
            a[j] = dw * uf[j] * (s + silu * (1.f - s));
            b[j] = dw * silu;
          } else {
            a[j] = silu * w * uf[j];   // a weight of zero comes before the product that may overflow
          }
        }
        reinterpret_cast<Raw*>(o_row)[c] = VecT::pack(a);
        if constexpr (BWD) reinterpret_cast<Raw*>(o_row + p.inter)[c] = VecT::pack(b);
      }
    }
  }
  if constexpr (BWD) {
    if (p.dweight) {   // uniform over the grid: every thread takes part
#pragma unroll
      for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if constexpr (TPR > 32) {
        __shared__ float part[kSwigluThreads / 32];
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) sum += part[slot * (TPR / 32) + i];
      }
      if (live && lane == 0) p.dweight[row] = sum;
    }
  }
}

template <typename T, int V, int TPR, bool BWD>
cudaError_t launch_swiglu_one(const SwigluParams& p, cudaStream_t st) {
  const int64_t blocks = (p.rows + kSwigluThreads / TPR - 1) / (kSwigluThreads / TPR);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = launch_config(dim3(static_cast<unsigned>(blocks)), kSwigluThreads, st, &attr);
  return cudaLaunchKernelEx(&cfg, swiglu_kernel<T, V, TPR, BWD>, p);
}

// The threads of a row: as few as cover it with kUnroll pieces each, a block's half for wide rows unless there are
// enough rows that a warp each fills the machine.  bf16, forward and backward, us, with 4, 8, 32, 128 threads a row:
//   32768 x 64     3.2 + 5.3    3.2 + 5.8    8.2 + 16.4   17 + 54     (4 taken)
//   32768 x 96     4.6 + 6.9    5.1 + 8.0    9.3 + 17.0   18 + 56     (4)
//   65536 x 200   15.9 + 27.5  14.5 + 26.4  19.9 + 41.0   40 + 133    (32: one piece past the 24 of 8 threads)
//   512 x 768      9.7 + 12.6   5.4 + 7.0    2.2 + 2.6    1.8 + 2.2   (32)
//   512 x 4096      53 + 67      27 + 36     7.7 + 10.7   3.6 + 5.3   (128)
//   4096 x 4096     67 + 84      36 + 47    18.3 + 34.6  18.4 + 30.9  (128)
//   8192 x 4096     73 + 93      47 + 64    37.0 + 58.3  34.2 + 57.3  (32)
//   16384 x 1536    36 + 50      27 + 52    24.8 + 40.5  30.3 + 54.7  (32)
template <typename T, int V, bool BWD>
cudaError_t launch_swiglu_vec(const SwigluParams& p, cudaStream_t st) {
  const int n = p.inter / V;
  if (n <= 4 * kUnroll) return launch_swiglu_one<T, V, 4, BWD>(p, st);
  if (n <= 8 * kUnroll) return launch_swiglu_one<T, V, 8, BWD>(p, st);
  if (n <= 32 * kUnroll || p.rows >= 8192) return launch_swiglu_one<T, V, 32, BWD>(p, st);
  return launch_swiglu_one<T, V, 128, BWD>(p, st);
}

template <typename T, bool BWD>
cudaError_t launch_swiglu_type(const SwigluParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto aligned = [](const void* q, int64_t ld) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  };
  const bool vec = p.inter % V == 0 && aligned(p.h, p.ld_h) && aligned(p.out, p.ld_out) &&
                   (!BWD || aligned(p.dact, p.ld_dact));
  return vec ? launch_swiglu_vec<T, V, BWD>(p, st) : launch_swiglu_vec<T, 1, BWD>(p, st);
}

int run_swiglu(const char* what, const SwigluParams& p, int32_t dtype, bool bwd, void* stream) {
  if (!known_dtype(dtype)) return report_error(HEXMOE_E_DTYPE, "swiglu: bad dtype");
  if (p.rows < 0 || p.inter <= 0 || p.inter > (1 << 30)) return arg_error("%s: rows %lld, inter %d", what, static_cast<long long>(p.rows), p.inter);
  if (p.ld_h < 2ll * p.inter || p.ld_out < (bwd ? 2ll : 1ll) * p.inter || (bwd && p.ld_dact < p.inter))
    return arg_error("%s: a row stride is shorter than its row", what);
  if (p.rows == 0) return HEXMOE_OK;
  if (!p.h || !p.out || (bwd && !p.dact)) return arg_error("%s: null pointer", what);
  const size_t z = dtype_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(p.h) % z || reinterpret_cast<uintptr_t>(p.out) % z ||
      reinterpret_cast<uintptr_t>(p.dact) % z || reinterpret_cast<uintptr_t>(p.weight) % 4 ||
      reinterpret_cast<uintptr_t>(p.dweight) % 4)
    return arg_error("%s: a pointer is not aligned to its element", what);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    return bwd ? launch_swiglu_type<T, true>(p, st) : launch_swiglu_type<T, false>(p, st);
  };
  const cudaError_t e = dtype == HEXMOE_F32 ? go(float{}) : dtype == HEXMOE_F16 ? go(__half{}) : go(__nv_bfloat16{});
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

// ------------------------------------------- gradient norm and clipping
// norm = sqrt(sum x^2) (or max |x|) over a list of tensors, then
// out = x min(1, max_norm / (norm + 1e-6)).  Bound by HBM: a read for the norm
// and, where something is scaled or copied, a read and a write.  Two kernels:
// partial sums per block, then every block adds all partials in the same order
// (one result, whatever the order of the blocks) and scales.  The tensor list
// travels as a kernel parameter, so nothing of it is kept between calls.  All
// blocks move through the chunks side by side, the second kernel backwards: what
// the first one read last is still in L2.
constexpr int kClipThreads = 256;
// Blocks an SM, with two loads in flight a thread in the scaling and four in the norm: more requests under
// way than this mix reads and writes too finely for HBM.  604 M bf16 values copied: 566 us; with four
// loads in the scaling 578, with 3 or 5 blocks 596 and 627 (300 M f32: 560; 579, 604, 616).
constexpr int kClipPerSm = 4;
// Values of a chunk: long runs for HBM, but enough chunks for every block of a short list
// (40 tensors of 1.5 M values in all: 4096 values 8.0 us, 16384 17.7).
constexpr int kClipChunk = 16384, kClipShortChunk = 4096;
constexpr int64_t kClipShort = 16 << 20;
constexpr int kClipSmallList = 64;
constexpr int kClipList = 1000;    // 32 bytes an entry: just under the 32764 bytes of parameters

struct ClipEntry {
  const void* src;
  void* dst;
  int64_t n;
  uint32_t first;   // its first chunk
};
template <int CAP>
struct ClipTable {
  int32_t count;
  uint32_t chunks;
  int32_t chunk;   // values of one
  ClipEntry e[CAP];
};

// Sum of squares of up to 8 values, exact to f32 rounding at every magnitude:
// where the plain sum overflows or has lost small values to underflow, the
// values are scaled by a power of two first.
template <int V>
__device__ __forceinline__ double square_sum(const float (&x)[V]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) s = fmaf(x[i], x[i], s);
  if (s > 1e-25f && s < 3e38f) return static_cast<double>(s);
  const float f = s <= 1e-25f ? 0x1p100f : 0x1p-64f;
  const double back = s <= 1e-25f ? 0x1p-200 : 0x1p128;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) s = fmaf(x[i] * f, x[i] * f, s);
  return static_cast<double>(s) * back;
}

// |x| as bits: integer order is the order of magnitudes, with NaN above infinity.
template <int V>
__device__ __forceinline__ uint32_t max_bits(const float (&x)[V]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

template <bool INF>
struct ClipAcc {
  double sum = 0;
  uint32_t big = 0;
  template <int V>
  __device__ __forceinline__ void add(const float (&x)[V]) {
    if constexpr (INF) big = max(big, max_bits(x));
    else sum += square_sum(x);
  }
};

// The `count` values of a chunk into the accumulator, by one block.
template <typename T, bool INF>
__device__ __forceinline__ void clip_read(const T* src, int count, ClipAcc<INF>& acc) {
  constexpr int V = 16 / sizeof(T);
  constexpr int U = 4;
  // head: the values before the first 16-byte boundary
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  const int head = min(count, off ? V - off : 0);
  if (threadIdx.x < head) {
    const float x[1] = {to_f32(src[threadIdx.x])};
    acc.add(x);
  }
  const int n = (count - head) / V;
  using Raw = typename Vec<T, V>::Raw;
  const Raw* v = reinterpret_cast<const Raw*>(src + head);
  for (int c0 = threadIdx.x; c0 < n; c0 += kClipThreads * U) {
    Raw r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (c0 + i * kClipThreads < n) r[i] = v[c0 + i * kClipThreads];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (c0 + i * kClipThreads >= n) continue;
      float x[V];
      Vec<T, V>::unpack(r[i], x);
      acc.add(x);
    }
  }
  const int tail = head + n * V + threadIdx.x;
  if (tail < count) {
    const float x[1] = {to_f32(src[tail])};
    acc.add(x);
  }
}

// dst = src * c over the `count` values of a chunk, by one block.  Vectors where
// source and destination share their place within a vector (every in-place
// call), else one value at a time.
template <typename T, typename D>
__device__ __forceinline__ void clip_scale(const T* src, D* dst, int count, float c) {
  constexpr int V = 16 / (sizeof(T) > sizeof(D) ? sizeof(T) : sizeof(D));   // 16 bytes of the wider type
  constexpr int U = 2;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) % (V * sizeof(T)) / sizeof(T));
  if (static_cast<int>(reinterpret_cast<uintptr_t>(dst) % (V * sizeof(D)) / sizeof(D)) != off) {
    for (int i = threadIdx.x; i < count; i += kClipThreads) dst[i] = from_f32<D>(to_f32(src[i]) * c);
    return;
  }
  const int head = min(count, off ? V - off : 0);
  if (threadIdx.x < head) dst[threadIdx.x] = from_f32<D>(to_f32(src[threadIdx.x]) * c);
  const int n = (count - head) / V;
  using Raw = typename Vec<T, V>::Raw;
  using RawD = typename Vec<D, V>::Raw;
  const Raw* v = reinterpret_cast<const Raw*>(src + head);
  RawD* o = reinterpret_cast<RawD*>(dst + head);
  for (int c0 = threadIdx.x; c0 < n; c0 += kClipThreads * U) {
    Raw r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (c0 + i * kClipThreads < n) r[i] = v[c0 + i * kClipThreads];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (c0 + i * kClipThreads >= n) continue;
      float x[V];
      Vec<T, V>::unpack(r[i], x);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] *= c;
      o[c0 + i * kClipThreads] = Vec<D, V>::pack(x);
    }
  }
  const int tail = head + n * V + threadIdx.x;
  if (tail < count) dst[tail] = from_f32<D>(to_f32(src[tail]) * c);
}

// The entry that holds chunk c.
template <int CAP>
__device__ __forceinline__ int clip_entry(const ClipTable<CAP>& t, uint32_t c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.e[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T, int CAP, bool INF>
__global__ void __launch_bounds__(kClipThreads, kClipPerSm)
    clip_norm_kernel(const __grid_constant__ ClipTable<CAP> t, double* partial) {
  pdl_wait();
  pdl_launch_dependents();
  ClipAcc<INF> acc;
  if (blockIdx.x < t.chunks) {
    int i = clip_entry(t, blockIdx.x);
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
      while (i + 1 < t.count && t.e[i + 1].first <= c) ++i;
      const ClipEntry& e = t.e[i];
      const int64_t a = static_cast<int64_t>(c - e.first) * t.chunk;
      const int count = static_cast<int>(min(e.n - a, static_cast<int64_t>(t.chunk)));
      clip_read(static_cast<const T*>(e.src) + a, count, acc);
    }
  }
  __shared__ double part[kClipThreads / 32];
  if constexpr (INF) acc.sum = static_cast<double>(__uint_as_float(__reduce_max_sync(0xffffffffu, acc.big)));
  else
    for (int o = 16; o > 0; o >>= 1) acc.sum += __shfl_xor_sync(0xffffffffu, acc.sum, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = acc.sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = part[0];
    for (int i = 1; i < kClipThreads / 32; ++i) {
      if constexpr (INF) s = s != s || part[i] <= s ? s : part[i];   // a NaN stays
      else s += part[i];
    }
    partial[blockIdx.x] = s;
  }
}

template <typename T, typename D, int CAP, bool INF>
__global__ void __launch_bounds__(kClipThreads, kClipPerSm)
    clip_scale_kernel(const __grid_constant__ ClipTable<CAP> t, const double* partial, int32_t partials,
                      float max_norm, int32_t copies, float* norm_out) {
  pdl_wait();
  __shared__ double part[kClipThreads];
  double s = 0;
  for (int i = threadIdx.x; i < partials; i += kClipThreads) {
    const double v = partial[i];
    if constexpr (INF) s = s != s || v <= s ? s : v;
    else s += v;
  }
  part[threadIdx.x] = s;
  __syncthreads();
#pragma unroll
  for (int o = kClipThreads / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) {
      const double v = part[threadIdx.x + o];
      if constexpr (INF) part[threadIdx.x] = part[threadIdx.x] != part[threadIdx.x] || v <= part[threadIdx.x] ? part[threadIdx.x] : v;
      else part[threadIdx.x] += v;
    }
    __syncthreads();
  }
  const float norm = static_cast<float>(INF ? part[0] : sqrt(part[0]));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  float coef = isinf(max_norm) ? 1.f : max_norm / (norm + 1e-6f);
  if (coef > 1.f) coef = 1.f;                // a NaN stays
  if (coef == 1.f && !copies) return;        // in place and within the norm: nothing changes
  if (blockIdx.x >= t.chunks) return;
  int i = t.count - 1;
  for (int64_t c = static_cast<int64_t>(t.chunks) - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    while (t.e[i].first > c) --i;
    const ClipEntry& e = t.e[i];
    if (coef == 1.f && e.dst == e.src) continue;
    const int64_t a = static_cast<int64_t>(c - e.first) * t.chunk;
    const int count = static_cast<int>(min(e.n - a, static_cast<int64_t>(t.chunk)));
    clip_scale(static_cast<const T*>(e.src) + a, static_cast<D*>(e.dst) + a, count, coef);
  }
}

int clip_grid(uint32_t chunks, int sms) {
  return static_cast<int>(std::max<uint32_t>(1, std::min<uint32_t>(chunks, kClipPerSm * sms)));
}

// The tensors of one pair of types, and what a call passes along its launches.
struct ClipCall {
  std::vector<ClipEntry> lists[3][3];   // [source type][destination type]
  double* partial;
  int32_t partials = 0;
  int32_t chunk, copies;
  int sms;
  float max_norm;
  float* norm_out;
  cudaStream_t st;
};

template <int CAP>
int fill_table(ClipTable<CAP>& t, const std::vector<ClipEntry>& list, size_t from, const ClipCall& c) {
  const size_t to = std::min(list.size(), from + CAP);
  t.count = static_cast<int32_t>(to - from);
  t.chunks = 0;
  t.chunk = c.chunk;
  for (size_t i = from; i < to; ++i) {
    t.e[i - from] = list[i];
    t.e[i - from].first = t.chunks;
    t.chunks += static_cast<uint32_t>((list[i].n + t.chunk - 1) / t.chunk);
  }
  return clip_grid(t.chunks, c.sms);
}

// All norm kernels of the call, then all scale kernels, the lists in the reverse order.
template <typename T, typename D, int CAP, bool INF>
cudaError_t launch_clip_list(const std::vector<ClipEntry>& list, bool scale, ClipCall& c) {
  ClipTable<CAP> t;
  cudaLaunchAttribute attr;
  const size_t tables = (list.size() + CAP - 1) / CAP;
  for (size_t i = 0; i < tables; ++i) {
    const int grid = fill_table(t, list, (scale ? tables - 1 - i : i) * CAP, c);
    const cudaLaunchConfig_t cfg = launch_config(dim3(grid), kClipThreads, c.st, &attr);
    cudaError_t e;
    if (scale) {
      e = cudaLaunchKernelEx(&cfg, clip_scale_kernel<T, D, CAP, INF>, t, static_cast<const double*>(c.partial), c.partials,
                             c.max_norm, c.copies, c.norm_out);
    } else {
      e = cudaLaunchKernelEx(&cfg, clip_norm_kernel<T, CAP, INF>, t, c.partial + c.partials);
      c.partials += grid;
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int CAP, bool INF>
cudaError_t launch_clip(ClipCall& c) {
  for (int i = 0; i < 18; ++i) {
    const bool scale = i >= 9;
    const int pair = scale ? 17 - i : i, src = pair / 3, dst = pair % 3;
    const std::vector<ClipEntry>& list = c.lists[src][dst];
    auto to = [&](auto s) {
      using T = decltype(s);
      return dst == HEXMOE_F32   ? launch_clip_list<T, float, CAP, INF>(list, scale, c)
             : dst == HEXMOE_F16 ? launch_clip_list<T, __half, CAP, INF>(list, scale, c)
                                 : launch_clip_list<T, __nv_bfloat16, CAP, INF>(list, scale, c);
    };
    if (list.empty()) continue;
    const cudaError_t e = src == HEXMOE_F32 ? to(float{}) : src == HEXMOE_F16 ? to(__half{}) : to(__nv_bfloat16{});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int current_sms(int* sms) {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return report_cuda_error(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return report_error(HEXMOE_E_DEVICE, "device ordinal out of range");
  if (!cached[dev].load(std::memory_order_relaxed)) {
    int v = 0;
    e = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return report_cuda_error(e, "cudaDeviceGetAttribute");
    cached[dev].store(v, std::memory_order_relaxed);
  }
  *sms = cached[dev].load(std::memory_order_relaxed);
  return HEXMOE_OK;
}

constexpr int kClipMaxSms = 256;   // what the workspace is sized for

}  // namespace
}  // namespace hexmoe

using namespace hexmoe;

extern "C" {

int hexmoe_swiglu(const void* h, int32_t dtype, int64_t rows, int32_t inter, int64_t ld_h, const float* row_weights,
                  void* act, int64_t ld_act, void* stream) {
  SwigluParams p{};
  p.h = h; p.weight = row_weights; p.out = act;
  p.rows = rows; p.ld_h = ld_h; p.ld_out = ld_act; p.inter = inter;
  return run_swiglu("hexmoe_swiglu", p, dtype, false, stream);
}

int hexmoe_swiglu_backward(const void* dact, int64_t ld_dact, const void* h, int64_t ld_h, int32_t dtype, int64_t rows,
                           int32_t inter, const float* row_weights, void* dh, int64_t ld_dh, float* drow_weights,
                           void* stream) {
  SwigluParams p{};
  p.h = h; p.dact = dact; p.weight = row_weights; p.out = dh; p.dweight = drow_weights;
  p.rows = rows; p.ld_h = ld_h; p.ld_dact = ld_dact; p.ld_out = ld_dh; p.inter = inter;
  return run_swiglu("hexmoe_swiglu_backward", p, dtype, true, stream);
}

size_t hexmoe_clip_grad_norm_workspace_bytes(int32_t tensors) {
  if (tensors < 0) return 0;
  // launches of the norm: one for every pair of types, more for lists past a table's length
  const size_t groups = std::max(1, std::min(tensors, 9)) + static_cast<size_t>(tensors) / kClipList;
  return groups * kClipPerSm * kClipMaxSms * sizeof(double);
}

int hexmoe_clip_grad_norm(int32_t tensors, const void* const* src, const int64_t* counts, const int32_t* src_dtypes,
                          void* const* dst, const int32_t* dst_dtypes, float max_norm, int32_t inf_norm,
                          float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (tensors < 0) return arg_error("hexmoe_clip_grad_norm: %d tensors", tensors);
  if (!(max_norm >= 0.f)) return arg_error("hexmoe_clip_grad_norm: max_norm must be at least 0");
  if (!norm_out || !workspace || (tensors && (!src || !counts || !src_dtypes || (dst && !dst_dtypes))))
    return arg_error("hexmoe_clip_grad_norm: null pointer");
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm_out) % 4)
    return arg_error("hexmoe_clip_grad_norm: workspace or norm not aligned");
  const size_t need = hexmoe_clip_grad_norm_workspace_bytes(tensors);
  if (workspace_bytes < need)
    return arg_error("hexmoe_clip_grad_norm: workspace %zu bytes < %zu needed", workspace_bytes, need);
  int sms = 0;
  if (int rc = current_sms(&sms)) return rc;
  sms = std::min(sms, kClipMaxSms);
  try {
    struct Span {
      uintptr_t a, b;
      bool written;
    };
    std::vector<Span> spans;
    spans.reserve(2 * static_cast<size_t>(tensors));
    ClipCall call{};
    int64_t values = 0;
    for (int32_t i = 0; i < tensors; ++i) {
      const int32_t st = src_dtypes[i], dt = dst ? dst_dtypes[i] : st;
      if (!known_dtype(st) || !known_dtype(dt)) return report_error(HEXMOE_E_DTYPE, "hexmoe_clip_grad_norm: bad dtype");
      if (counts[i] < 0 || counts[i] > (1ll << 40)) return arg_error("hexmoe_clip_grad_norm: tensor %d has %lld values", i, static_cast<long long>(counts[i]));
      if (counts[i] == 0) continue;
      void* d = dst ? dst[i] : const_cast<void*>(src[i]);
      if (!src[i] || !d) return arg_error("hexmoe_clip_grad_norm: null pointer");
      const uintptr_t sa = reinterpret_cast<uintptr_t>(src[i]), da = reinterpret_cast<uintptr_t>(d);
      if (sa % dtype_bytes(st) || da % dtype_bytes(dt)) return arg_error("hexmoe_clip_grad_norm: tensor %d is not aligned to its element", i);
      call.lists[st][dt].push_back({src[i], d, counts[i], 0});
      values += counts[i];
      spans.push_back({da, da + counts[i] * dtype_bytes(dt), true});
      if (sa != da) spans.push_back({sa, sa + counts[i] * dtype_bytes(st), false});
      else if (st != dt) return arg_error("hexmoe_clip_grad_norm: tensor %d is written in place with another dtype", i);
      call.copies |= sa != da;
    }
    // a value that is written may be reached through one entry only: overlapping
    // entries would be scaled twice, or read after they were scaled
    std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
    uintptr_t any_end = 0, written_end = 0;
    for (const Span& s : spans) {
      if (s.a < written_end || (s.written && s.a < any_end)) return arg_error("hexmoe_clip_grad_norm: tensors overlap");
      any_end = std::max(any_end, s.b);
      if (s.written) written_end = std::max(written_end, s.b);
    }
    call.partial = static_cast<double*>(workspace);
    call.chunk = values < kClipShort ? kClipShortChunk : kClipChunk;
    call.sms = sms;
    call.max_norm = max_norm;
    call.norm_out = norm_out;
    call.st = static_cast<cudaStream_t>(stream);
    if (values == 0) {   // no values: a norm of 0
      const cudaError_t e = cudaMemsetAsync(norm_out, 0, sizeof(float), call.st);
      return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, "hexmoe_clip_grad_norm");
    }
    const bool small = tensors <= kClipSmallList;
    const cudaError_t e = inf_norm ? (small ? launch_clip<kClipSmallList, true>(call) : launch_clip<kClipList, true>(call))
                                   : (small ? launch_clip<kClipSmallList, false>(call) : launch_clip<kClipList, false>(call));
    return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, "hexmoe_clip_grad_norm");
  } catch (const std::exception&) {
    return report_error(HEXMOE_E_ARG, "hexmoe_clip_grad_norm: out of host memory");
  }
}

}  // extern "C"
