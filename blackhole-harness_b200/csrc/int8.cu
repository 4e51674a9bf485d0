// int8.cu — a MoE layer's experts in 8-bit integers: rows quantized with a scale each, the plan that puts
// routed tokens into expert order, and the layer made of them and the products in grouped.cu.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include <cooperative_groups.h>

#include "internal.cuh"
#include "ptx.cuh"

namespace hexmoe {
namespace {

namespace cg = cooperative_groups;

int arg_error(const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_error(HEXMOE_E_ARG, buf);
}

constexpr unsigned kAll = 0xffffffffu;
constexpr int64_t kMaxSum = 131071;   // products of -128 and -128 that an int32 holds

cudaLaunchConfig_t launch_config(dim3 grid, int threads, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// ------------------------------------------------------------------- rows to 8 bits
// scale = max |x| / 127, q = round(127 x / max |x|), ties to even, of every row.  The quotient is that of real numbers (x =
// max / 2, which 16-bit rows hold often, is 63.5 to the last bit): it is computed in f32, off by less than 2^-16 at 127, and
// an f32 x that close to a border n + 1/2 is decided by the sign of 254 |x| - (2 n + 1) max, which f32 products with their
// rounding errors (by FMA) give exactly; 16 bits need less (see byte()).  A row of zeros has scale 0; one that holds an
// infinity or NaN has scale NaN and zeros, so that what is made of it is NaN.
// Bound by HBM, as long as a value takes no more than some ten instructions and none of them a branch: 32768 x 2048 bf16
// 33.6 us (6.0 TB/s), 113 with borders decided in f64; 32768 x 768 f32 22.3 us (5.6 TB/s); 512 x 2048 2.4 us.  TPR threads
// take a row and keep its first kPieces 16-byte pieces each in registers; what a longer row has behind those is read again.
constexpr int kRowThreads = 256;
constexpr int kPieces = 8;

struct RowsParams {
  const void* x;
  int64_t ld_x, rows;
  int32_t cols;
  int8_t* q;              // [rows, ld_q], or with `places` [places..., ld_q]
  int64_t ld_q;
  float* scale;
  const int32_t* count;   // on the device: rows that exist, of `rows`; or null
  // The layer's tokens, each to the rows of its topk slots: slot s has row places[s] (-1: none).
  const int32_t* places;
  int32_t topk;
};

// A row's values as they lie, 16 bytes at a time, or one by one (rows that are not aligned to 16 bytes, or of odd
// lengths): the largest magnitude's bits, and the values in f32.
template <typename T, bool VEC>
struct Piece {
  static constexpr int kValues = VEC ? 16 / sizeof(T) : 1, kWords = VEC ? 4 : 1;
  uint32_t w[kWords];
  // Past L1: it is read once.
  __device__ __forceinline__ void load(const T* row, int i) {
    if constexpr (VEC) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4*>(row) + i);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = __ldcg(reinterpret_cast<const uint32_t*>(row) + i);
    } else {
      w[0] = __ldcg(reinterpret_cast<const uint16_t*>(row) + i);
    }
  }
  // The largest magnitude so far: f32 bits, or two of 16 bits.
  __device__ __forceinline__ uint32_t see(uint32_t most) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      most = sizeof(T) == 4 ? max(most, w[i] & 0x7fffffffu) : __vmaxu2(most, w[i] & 0x7fff7fffu);
    return most;
  }
  __device__ __forceinline__ float value(int j) const {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[j]);
    else if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half(static_cast<uint16_t>(w[j / 2] >> j % 2 * 16)));
    else return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
};
// The f32 bits of see()'s magnitude.
template <typename T>
__device__ __forceinline__ uint32_t f32_bits(uint32_t most) {
  if constexpr (sizeof(T) == 4) return most;
  const uint32_t v = max(most & 0xffffu, most >> 16);
  if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(v))));
  else return v << 16;
}

struct RowScale {
  float largest;   // as it is
  float fit, most, inverse;   // a power of two that keeps what follows in range, the largest times it, 127 / that
  __device__ __forceinline__ explicit RowScale(uint32_t bits) {
    largest = __uint_as_float(bits);
    fit = largest > 0x1p96f ? 0x1p-60f : largest < 0x1p-90f ? 0x1p100f : 1.f;
    most = largest * fit;
    inverse = largest == 0.f || !finite() ? 0.f : 127.f / most;
  }
  __device__ __forceinline__ bool finite() const { return __float_as_uint(largest) < 0x7f800000u; }
  __device__ __forceinline__ float scale() const { return finite() ? largest / 127.f : __uint_as_float(0x7fc00000u); }
  // 127 x / largest rounded, as the low byte of a word.
  //   16-bit x: the quotient's nearest border n + 1/2 is met exactly or missed by 2^-19 of it (254 x and (2 n + 1) largest
  //     are whole multiples of a common unit, of at most 11 + 8 bits), so rounding it to 20 bits first takes its f32 error
  //     away and leaves exact halves to the rounding to even.
  //   f32: doubt is the distance from the whole number, the largest so far; what near_border() says goes by exact_byte().
  template <typename T>
  __device__ __forceinline__ uint32_t byte(float x, float& doubt) const {
    constexpr float kWhole = 12582912.f;   // 1.5 x 2^23: f32 values here are whole numbers
    float t = __fmul_rn(__fmul_rn(x, fit), inverse);   // each rounded by itself: no FMA made of two
    if constexpr (sizeof(T) == 2) {
      const float wide = __fmul_rn(t, 17.f);
      t = __fsub_rn(wide, __fsub_rn(wide, t));
    }
    const float r = t + kWhole;
    if constexpr (sizeof(T) == 4) doubt = fmaxf(doubt, fabsf(t - (r - kWhole)));
    return __float_as_uint(r);
  }
  static __device__ __forceinline__ bool near_border(float doubt) { return doubt > 0.49998f; }
  __device__ __forceinline__ uint32_t exact_byte(float x) const {
    const float v = fabsf(x * fit), n = floorf(v * inverse + 0x1p-10f);
    if (!(fabsf(v * inverse - n - 0.5f) < 0x1p-10f)) {
      float ignore = 0.f;
      return byte<float>(x, ignore);
    }
    const float odd = 2.f * n + 1.f, p = odd * most;
    const float over = fmaf(254.f, v, -p), lost = fmaf(odd, most, -p);   // 254 v - odd most = over - lost, both exact
    const bool up = over > lost || (over == lost && (static_cast<int>(n) & 1));
    const int32_t q = static_cast<int>(n) + up;
    return static_cast<uint32_t>(x < 0.f ? -q : q);
  }
};

// A row to TPR threads.  PLACES: into the rows of its slots, which the kernel before has found.  The pieces are turned into
// bytes in registers and stored from there: what is unrolled eight times stays short, for a kernel of a few microseconds waits
// for its instructions more than for anything else.
template <typename T, bool VEC, int TPR, bool PLACES>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(const RowsParams p) {
  constexpr int kRows = kRowThreads / TPR;
  __shared__ uint32_t part[kRowThreads / 32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  const int lane = threadIdx.x % TPR;
  pdl_wait();
  pdl_launch_dependents();
  const bool live = row < p.rows && (!p.count || row < *p.count);
  using P = Piece<T, VEC>;
  constexpr int V = P::kValues, kWords = V > 4 ? V / 4 : 1;
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
  const int n = p.cols / V;
  P held[kPieces];
  uint32_t most = 0;
  if (live) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (lane + i * TPR < n) held[i].load(x, lane + i * TPR);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (lane + i * TPR < n) most = held[i].see(most);
    for (int c = lane + kPieces * TPR; c < n; c += TPR) {
      P v;
      v.load(x, c);
      most = v.see(most);
    }
  }
  uint32_t bits = f32_bits<T>(most);
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(kAll, bits, o));
  if constexpr (TPR > 32) {
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = bits;
    __syncthreads();
    const int slot = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) bits = max(bits, part[slot * (TPR / 32) + i]);
  }
  const RowScale to(bits);
  const bool finite = to.finite();
  auto bytes = [&](const P& v, uint32_t (&w)[kWords]) {
    uint32_t q[V];
    float doubt = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = to.byte<T>(v.value(j), doubt);
    if (sizeof(T) == 4 && __builtin_expect(RowScale::near_border(doubt), 0)) {
#pragma unroll
      for (int j = 0; j < V; ++j) q[j] = to.exact_byte(v.value(j));
    }
    if constexpr (V == 1) w[0] = q[0];
#pragma unroll
    for (int j = 0; j + 3 < V; j += 4) w[j / 4] = prmt(prmt(q[j], q[j + 1], 0x0040), prmt(q[j + 2], q[j + 3], 0x0040), 0x5410);
    if (!finite) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[j] = 0;
    }
  };
  auto put = [&](int64_t at, int c, const uint32_t (&w)[kWords]) {
    int8_t* dst = p.q + at * p.ld_q + static_cast<int64_t>(c) * V;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else *dst = static_cast<int8_t>(w[0]);
  };
  uint32_t w[kPieces][kWords];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    if (live && lane + i * TPR < n) bytes(held[i], w[i]);
  }
  if (!live) return;
  const int copies = PLACES ? p.topk : 1;
#pragma unroll 1
  for (int j = 0; j < copies; ++j) {
    const int64_t at = PLACES ? p.places[row * p.topk + j] : row;
    if (PLACES && at < 0) continue;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (lane + i * TPR < n) put(at, lane + i * TPR, w[i]);
    if (lane == 0) p.scale[at] = to.scale();
  }
  for (int c = lane + kPieces * TPR; c < n; c += TPR) {
    P v;
    v.load(x, c);
    bytes(v, w[0]);
#pragma unroll 1
    for (int j = 0; j < copies; ++j) {
      const int64_t at = PLACES ? p.places[row * p.topk + j] : row;
      if (!PLACES || at >= 0) put(at, c, w[0]);
    }
  }
}

// The threads of a row: as few as hold it in registers.
template <typename T, bool VEC>
cudaError_t launch_rows_vec(const RowsParams& p, cudaStream_t st) {
  const int n = p.cols / Piece<T, VEC>::kValues;
  auto go = [&](auto tpr, auto* kernel) {
    constexpr int kRows = kRowThreads / decltype(tpr)::value;
    const int64_t blocks = (p.rows + kRows - 1) / kRows;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = launch_config(dim3(static_cast<unsigned>(blocks)), kRowThreads, 0, st, &attr);
    return cudaLaunchKernelEx(&cfg, kernel, p);
  };
  auto pick = [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    return p.places ? go(tpr, quantize_rows_kernel<T, VEC, TPR, true>) : go(tpr, quantize_rows_kernel<T, VEC, TPR, false>);
  };
  if (n <= 8 * kPieces) return pick(std::integral_constant<int, 8>{});
  if (n <= 32 * kPieces) return pick(std::integral_constant<int, 32>{});
  if (n <= 64 * kPieces) return pick(std::integral_constant<int, 64>{});
  return pick(std::integral_constant<int, 256>{});
}

template <typename T>
bool rows_aligned(const RowsParams& p) {   // rows of whole pieces of 16 bytes
  constexpr int V = 16 / sizeof(T);
  return p.cols % V == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ld_x % V == 0 &&
         reinterpret_cast<uintptr_t>(p.q) % V == 0 && p.ld_q % V == 0;
}
template <typename T>
cudaError_t launch_rows_type(const RowsParams& p, cudaStream_t st) {
  return rows_aligned<T>(p) ? launch_rows_vec<T, true>(p, st) : launch_rows_vec<T, false>(p, st);
}

cudaError_t launch_rows(const RowsParams& p, int32_t dtype, cudaStream_t st) {
  if (p.rows == 0) return cudaSuccess;
  return dtype == HEXMOE_F32   ? launch_rows_type<float>(p, st)
         : dtype == HEXMOE_F16 ? launch_rows_type<__half>(p, st)
                               : launch_rows_type<__nv_bfloat16>(p, st);
}

// ------------------------------------------------------------------- plan
// The rows of routed slots in expert order: offsets[e] (exclusive counts) and every slot's row.  Within an expert the
// rows come in whatever order the counting finds: no value of the layer depends on it (a row's sums are whole
// numbers and its own).  One cluster: each CTA counts its slots in shared memory, the counts of the CTAs before it come
// over distributed shared memory, and nothing has to be cleared or handed on between kernels.
constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;
constexpr int kPlanHeld = 4;        // slots a thread keeps in registers
constexpr int kMaxExperts = 2048;

struct PlanParams {
  const void* ids;
  int32_t ids64, experts;
  int64_t slots;
  int32_t* offsets;
  int32_t* places;
  int32_t* dev_err;
};

// The experts of kPlanHeld slots, `step` apart from s on, all loads issued before the first is used; -1: of none.
__device__ __forceinline__ void plan_experts(const PlanParams& p, int64_t s, int64_t step, int64_t end, int32_t (&e)[kPlanHeld]) {
  int64_t v[kPlanHeld];
#pragma unroll
  for (int i = 0; i < kPlanHeld; ++i) {
    const int64_t at = s + i * step;
    v[i] = at < end ? (p.ids64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at]) : -1;
  }
#pragma unroll
  for (int i = 0; i < kPlanHeld; ++i) e[i] = v[i] >= 0 && v[i] < p.experts ? static_cast<int32_t>(v[i]) : -1;
}

template <int CTAS>
__global__ void __launch_bounds__(kPlanThreads, 1) plan_kernel(const PlanParams p) {
  __shared__ int32_t hist[kMaxExperts], first[kMaxExperts], sums[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = CTAS > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  auto sync = [&] {
    if constexpr (CTAS > 1) cluster.sync();
    else __syncthreads();
  };
  for (int e = threadIdx.x; e < p.experts; e += kPlanThreads) hist[e] = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  const int64_t chunk = (p.slots + CTAS - 1) / CTAS, begin = rank * chunk, end = min(begin + chunk, p.slots);
  const int64_t s0 = begin + threadIdx.x;
  int32_t held_e[kPlanHeld], held_at[kPlanHeld];   // of the first slots; those behind wait in places
  bool bad = false;
  for (int64_t s = s0; s < end; s += kPlanHeld * kPlanThreads) {
    int32_t e[kPlanHeld];
    plan_experts(p, s, kPlanThreads, end, e);
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i) {
      const int64_t at = s + i * kPlanThreads;
      const int32_t n = e[i] >= 0 ? atomicAdd(&hist[e[i]], 1) : -1;
      bad |= at < end && e[i] < 0;
      if (s == s0) {
        held_e[i] = e[i];
        held_at[i] = n;
      } else if (at < end) {
        p.places[at] = n;
      }
    }
  }
  if (bad) atomicOr(p.dev_err, kDevErrExpertId);
  sync();
  // every CTA: each expert's count over all of them, and before this one
  const int per = (p.experts + kPlanThreads - 1) / kPlanThreads;   // 1 or 2 a thread
  int32_t total[2] = {}, before[2] = {}, mine = 0;
  for (int i = 0; i < per; ++i) {
    const int e = static_cast<int>(threadIdx.x) * per + i;
    if (e >= p.experts) break;
    int32_t v[CTAS];
#pragma unroll
    for (int c = 0; c < CTAS; ++c) v[c] = CTAS > 1 ? cluster.map_shared_rank(hist, c)[e] : hist[e];
#pragma unroll
    for (int c = 0; c < CTAS; ++c) {
      total[i] += v[c];
      if (c < rank) before[i] += v[c];
    }
    mine += total[i];
  }
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(kAll, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    int32_t v = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t u = __shfl_up_sync(kAll, v, o);
      if (lane >= o) v += u;
    }
    sums[lane] = v;
  }
  __syncthreads();
  int32_t at = upto - mine + (warp ? sums[warp - 1] : 0);
  for (int i = 0; i < per; ++i) {
    const int e = static_cast<int>(threadIdx.x) * per + i;
    if (e >= p.experts) break;
    first[e] = at + before[i];
    if (rank == 0) p.offsets[e] = at;
    at += total[i];
    if (rank == 0 && e == p.experts - 1) p.offsets[p.experts] = at;
  }
  sync();   // `first` is whole, and no CTA leaves while its counts are read
#pragma unroll
  for (int i = 0; i < kPlanHeld; ++i)
    if (s0 + i * kPlanThreads < end) p.places[s0 + i * kPlanThreads] = held_e[i] < 0 ? -1 : held_at[i] + first[held_e[i]];
  for (int64_t s = s0 + kPlanHeld * kPlanThreads; s < end; s += kPlanHeld * kPlanThreads) {
    int32_t e[kPlanHeld];
    plan_experts(p, s, kPlanThreads, end, e);
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i)
      if (e[i] >= 0) p.places[s + i * kPlanThreads] += first[e[i]];
  }
}

template <int CTAS>
cudaError_t launch_plan_of(const PlanParams& p, cudaStream_t st) {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_config(dim3(CTAS), kPlanThreads, 0, st, attr);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, plan_kernel<CTAS>, p);
}
cudaError_t launch_plan(const PlanParams& p, cudaStream_t st) {
  return p.slots > 2 * kPlanThreads ? launch_plan_of<kPlanCtas>(p, st) : launch_plan_of<1>(p, st);
}

// ------------------------------------------------------------------- sum
// out[t] = sum over j of weights[t topk + j] y[places[t topk + j]], in f32 in j's order, rounded once; a slot without a row
// adds nothing.  Products are rounded by themselves (no FMA): slots that are each other's negatives leave 0.  Slots' rows are
// f32: in 16 bits, where they would be half the bytes, the layer's result was off by 0.23 % where its own rounding to bf16
// costs 0.17, fp16 rows could leave the type's range where their sum does not, and a caller with f32 rows got eight bits
// (4096 tokens, 96 experts of 2048 x 768: 287 us in a graph, 239 with 16-bit rows; 16 tokens 67 and 69).  The routing weight
// is taken here, not with the activation's scale: the product of two small ones would leave the normal numbers before the
// result does.  Bound by HBM (those 4096 tokens: 55 us, 4.9 TB/s): a thread has eight 16-byte loads in flight, of as many of
// a token's rows as there are and so many pieces of each.
constexpr int kSumThreads = 256;

struct SumParams {
  const float* y;   // [rows, hidden]
  const int32_t* places;
  const float* weights;
  void* out;
  int64_t tokens;
  int32_t topk, hidden;
};

template <typename T, int ROWS>
__global__ void __launch_bounds__(kSumThreads) sum_rows_kernel(const SumParams p) {
  constexpr int kEach = 8 / ROWS;
  const int32_t pieces = p.hidden / 4, spans = (pieces + 32 * kEach - 1) / (32 * kEach), lane = threadIdx.x % 32;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kSumThreads / 32) + threadIdx.x / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = unit / spans;
  if (t >= p.tokens) return;
  const int32_t first = static_cast<int32_t>(unit % spans) * 32 * kEach + lane;
  float4 sum[kEach] = {};
  for (int j0 = 0; j0 < p.topk; j0 += ROWS) {
    float4 v[ROWS][kEach];
    float weight[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t slot = t * p.topk + j0 + j;
      const int32_t at = j0 + j < p.topk ? p.places[slot] : -1;
      weight[j] = at >= 0 ? p.weights[slot] : 0.f;
      const float4* row = reinterpret_cast<const float4*>(p.y) + static_cast<int64_t>(at) * pieces;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        v[j][i] = at >= 0 && first + 32 * i < pieces ? row[first + 32 * i] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        sum[i].x += __fmul_rn(weight[j], v[j][i].x);
        sum[i].y += __fmul_rn(weight[j], v[j][i].y);
        sum[i].z += __fmul_rn(weight[j], v[j][i].z);
        sum[i].w += __fmul_rn(weight[j], v[j][i].w);
      }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (first + 32 * i >= pieces) continue;
    T* out = static_cast<T*>(p.out) + t * p.hidden + (first + 32 * i) * 4;
    if constexpr (std::is_same_v<T, float>) {
      *reinterpret_cast<float4*>(out) = sum[i];
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 lo = __floats2half2_rn(sum[i].x, sum[i].y), hi = __floats2half2_rn(sum[i].z, sum[i].w);
      *reinterpret_cast<uint2*>(out) = make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
    } else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(sum[i].x, sum[i].y), hi = __floats2bfloat162_rn(sum[i].z, sum[i].w);
      *reinterpret_cast<uint2*>(out) = make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
    }
  }
}

template <typename T>
cudaError_t launch_sum(const SumParams& p, cudaStream_t st) {
  auto go = [&](auto rows, auto* kernel) {
    constexpr int kEach = 8 / decltype(rows)::value;
    const int64_t spans = (p.hidden / 4 + 32 * kEach - 1) / (32 * kEach);
    const int64_t blocks = (p.tokens * spans + kSumThreads / 32 - 1) / (kSumThreads / 32);
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = launch_config(dim3(static_cast<unsigned>(blocks)), kSumThreads, 0, st, &attr);
    return cudaLaunchKernelEx(&cfg, kernel, p);
  };
  if (p.topk == 1) return go(std::integral_constant<int, 1>{}, sum_rows_kernel<T, 1>);
  if (p.topk == 2) return go(std::integral_constant<int, 2>{}, sum_rows_kernel<T, 2>);
  if (p.topk <= 4) return go(std::integral_constant<int, 4>{}, sum_rows_kernel<T, 4>);
  return go(std::integral_constant<int, 8>{}, sum_rows_kernel<T, 8>);
}

bool is16(int32_t dt) { return dt == HEXMOE_BF16 || dt == HEXMOE_F16; }
bool known_dtype(int32_t dt) { return dt == HEXMOE_F32 || is16(dt); }
bool off_by(const void* p, size_t z) { return reinterpret_cast<uintptr_t>(p) % z != 0; }
int64_t pitch16(int64_t n) { return (n + 15) / 16 * 16; }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of a workspace one after the other.
struct Carve {
  uint8_t* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += round256(count * sizeof(T));
    return p;
  }
};

struct MmScratch {
  int8_t* q;
  float* scale;
  uint8_t* partial;
  size_t partial_bytes, used;
  MmScratch(void* ws, int64_t rows, int32_t experts, int32_t n, int32_t k, bool quantizes) {
    Carve c{static_cast<uint8_t*>(ws)};
    q = c.take<int8_t>(quantizes ? rows * pitch16(k) : 0);
    scale = c.take<float>(quantizes ? rows : 0);
    partial_bytes = int8_partial_bytes(rows, experts, n, k);
    partial = c.take<uint8_t>(partial_bytes);
    used = c.used;
  }
};

struct LayerScratch {
  int32_t *offsets, *places;
  float *x_scale, *act, *act_scale, *y;
  int8_t *xq, *actq;
  uint8_t* partial;
  size_t partial_bytes, used;
  LayerScratch(void* ws, int64_t slots, int32_t experts, int32_t hidden, int32_t inter) {
    Carve c{static_cast<uint8_t*>(ws)};
    offsets = c.take<int32_t>(experts + 1);
    places = c.take<int32_t>(slots);
    x_scale = c.take<float>(slots);
    act_scale = c.take<float>(slots);
    xq = c.take<int8_t>(slots * hidden);
    act = c.take<float>(slots * inter);
    actq = c.take<int8_t>(slots * inter);
    y = c.take<float>(slots * hidden);
    partial_bytes = int8_partial_bytes(slots, experts, hidden, inter);
    partial = c.take<uint8_t>(partial_bytes);
    used = c.used;
  }
};

}  // namespace
}  // namespace hexmoe

using namespace hexmoe;

extern "C" {

int hexmoe_quantize_rows(const void* x, int32_t x_dtype, int64_t ld_x, int64_t rows, int32_t cols, int8_t* q, int64_t ld_q,
                         float* scale, void* stream) {
  const char* what = "hexmoe_quantize_rows";
  if (!known_dtype(x_dtype)) return report_error(HEXMOE_E_DTYPE, "hexmoe_quantize_rows: bad dtype");
  if (rows < 0 || cols <= 0 || cols > (1 << 30)) return arg_error("%s: rows %lld, cols %d", what, static_cast<long long>(rows), cols);
  if (ld_x < cols || ld_q < cols) return arg_error("%s: a row stride is shorter than its row", what);
  if (rows == 0) return HEXMOE_OK;
  if (!x || !q || !scale || off_by(x, x_dtype == HEXMOE_F32 ? 4 : 2) || off_by(scale, 4))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  RowsParams p{};
  p.x = x; p.ld_x = ld_x; p.rows = rows; p.cols = cols; p.q = q; p.ld_q = ld_q; p.scale = scale;
  const cudaError_t e = launch_rows(p, x_dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

size_t hexmoe_grouped_mm_int8_workspace_bytes(int64_t rows, int32_t experts, int32_t n, int32_t k, int32_t x_dtype) {
  if (rows <= 0 || experts <= 0 || n <= 0 || k <= 0) return 0;
  return MmScratch(nullptr, rows, experts, n, k, x_dtype != HEXMOE_I8).used;
}

int hexmoe_grouped_mm_int8(const void* x, int32_t x_dtype, int64_t ld_x, const float* x_scale, const int8_t* w, int64_t ld_w,
                           int64_t stride_w, const float* w_scale, int64_t rows, int32_t experts, int32_t n, int32_t k,
                           const void* offsets, int32_t offsets_dtype, void* out, int64_t ld_out, int32_t out_dtype,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "hexmoe_grouped_mm_int8";
  const bool quantizes = x_dtype != HEXMOE_I8;
  if ((quantizes && !known_dtype(x_dtype)) || !known_dtype(out_dtype))
    return report_error(HEXMOE_E_DTYPE, "hexmoe_grouped_mm_int8: x is I8, F32, BF16 or F16, out F32, BF16 or F16");
  if (offsets_dtype != HEXMOE_I32 && offsets_dtype != HEXMOE_I64) return report_error(HEXMOE_E_DTYPE, "offsets are I32 or I64");
  if (rows < 0 || rows >= (1ll << 31) - 512) return arg_error("%s: %lld rows", what, static_cast<long long>(rows));
  if (experts <= 0 || experts > kMaxExperts) return arg_error("%s: %d experts outside 1..%d", what, experts, kMaxExperts);
  if (n <= 0 || n > (1 << 24) || k <= 0 || k > kMaxSum)
    return arg_error("%s: n %d, k %d (at most %lld, or a sum may leave int32)", what, n, k, static_cast<long long>(kMaxSum));
  if (!offsets && experts != 1) return arg_error("%s: no offsets for %d experts", what, experts);
  if (off_by(offsets, offsets_dtype == HEXMOE_I64 ? 8 : 4)) return arg_error("%s: offsets not aligned", what);
  if (ld_x < k || ld_w < k || stride_w < 0 || ld_out < n) return arg_error("%s: a row stride is shorter than its row", what);
  if (rows == 0) return HEXMOE_OK;
  if (!x || !w || !w_scale || !out || (!quantizes && !x_scale) || off_by(w_scale, 4) || off_by(x_scale, 4) ||
      off_by(out, out_dtype == HEXMOE_F32 ? 4 : 2) || (quantizes && off_by(x, x_dtype == HEXMOE_F32 ? 4 : 2)))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  if (!int8_stack(w, ld_w, stride_w, experts) || (!quantizes && !int8_rows(x, ld_x)))
    return arg_error("%s: 8-bit rows must begin and repeat on multiples of 16 bytes", what);
  if (off_by(workspace, 16)) return arg_error("%s: workspace not 16-byte aligned", what);
  const MmScratch s(workspace, rows, experts, n, k, quantizes);
  if (quantizes && (!workspace || workspace_bytes < s.used))
    return arg_error("%s: a workspace of %zu bytes is needed", what, s.used);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Int8Product d{};
  d.x = static_cast<const int8_t*>(x); d.ld_x = ld_x; d.x_scale = x_scale;
  if (quantizes) {
    RowsParams p{};
    p.x = x; p.ld_x = ld_x; p.rows = rows; p.cols = k; p.q = s.q; p.ld_q = pitch16(k); p.scale = s.scale;
    const cudaError_t e = launch_rows(p, x_dtype, st);
    if (e != cudaSuccess) return report_cuda_error(e, what);
    d.x = s.q; d.ld_x = p.ld_q; d.x_scale = s.scale;
  }
  d.w = w; d.ld_w = ld_w; d.stride_w = stride_w; d.w_scale = w_scale;
  d.rows = rows; d.experts = experts; d.n = n; d.k = k;
  d.offsets = offsets; d.offsets64 = offsets_dtype == HEXMOE_I64;
  d.out = out; d.ld_out = ld_out; d.out_dtype = out_dtype;
  if (workspace && workspace_bytes >= s.used) { d.workspace = s.partial; d.workspace_bytes = s.partial_bytes; }
  return run_int8_product(what, d, st);
}

size_t hexmoe_int8_forward_workspace_bytes(int64_t tokens, int32_t topk, int32_t experts, int32_t hidden, int32_t inter) {
  if (tokens <= 0 || topk <= 0 || experts <= 0 || hidden <= 0 || inter <= 0) return 0;
  return LayerScratch(nullptr, tokens * topk, experts, hidden, inter).used;
}

int hexmoe_int8_forward(const void* x, int32_t x_dtype, int64_t ld_x, int64_t tokens, int32_t hidden, int32_t inter, int32_t topk,
                        const float* topk_weights, const void* topk_ids, int32_t ids_dtype, int32_t experts,
                        const int8_t* w13, int64_t ld_w13, int64_t stride_w13, const float* w13_scale, const int8_t* w2,
                        int64_t ld_w2, int64_t stride_w2, const float* w2_scale, void* out, int32_t out_dtype,
                        void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "hexmoe_int8_forward";
  if (!known_dtype(x_dtype) || (out_dtype != x_dtype && out_dtype != HEXMOE_F32))
    return report_error(HEXMOE_E_DTYPE, "hexmoe_int8_forward: x is F32, BF16 or F16, out the same or F32");
  if (ids_dtype != HEXMOE_I32 && ids_dtype != HEXMOE_I64) return report_error(HEXMOE_E_DTYPE, "hexmoe_int8_forward: ids are I32 or I64");
  if (tokens < 0 || topk <= 0 || topk > 1024 || tokens * topk >= (1ll << 31) - 512)
    return arg_error("%s: %lld tokens, topk %d", what, static_cast<long long>(tokens), topk);
  if (experts <= 0 || experts > kMaxExperts) return arg_error("%s: %d experts outside 1..%d", what, experts, kMaxExperts);
  if (hidden <= 0 || inter <= 0 || hidden % 16 || inter % 16 || hidden > kMaxSum || inter > kMaxSum)
    return arg_error("%s: hidden %d, inter %d (multiples of 16, at most %lld)", what, hidden, inter, static_cast<long long>(kMaxSum));
  if (ld_x < hidden || ld_w13 < hidden || ld_w2 < inter || stride_w13 < 0 || stride_w2 < 0)
    return arg_error("%s: a row stride is shorter than its row", what);
  if (tokens == 0) return HEXMOE_OK;
  if (!x || !topk_weights || !topk_ids || !w13 || !w13_scale || !w2 || !w2_scale || !out || off_by(x, x_dtype == HEXMOE_F32 ? 4 : 2) ||
      off_by(topk_weights, 4) || off_by(topk_ids, ids_dtype == HEXMOE_I64 ? 8 : 4) || off_by(w13_scale, 4) || off_by(w2_scale, 4))
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  if (off_by(out, 16)) return arg_error("%s: out not 16-byte aligned", what);
  if (!int8_stack(w13, ld_w13, stride_w13, experts) || !int8_stack(w2, ld_w2, stride_w2, experts))
    return arg_error("%s: 8-bit rows must begin and repeat on multiples of 16 bytes", what);
  const int64_t slots = tokens * topk;
  const LayerScratch s(workspace, slots, experts, hidden, inter);
  if (!workspace || off_by(workspace, 256) || workspace_bytes < s.used)
    return arg_error("%s: a workspace of %zu bytes is needed, on a multiple of 256", what, s.used);
  int32_t* dev_err = device_error_word();
  if (!dev_err) return report_error(HEXMOE_E_CUDA, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const PlanParams plan = {topk_ids, ids_dtype == HEXMOE_I64, experts, slots, s.offsets, s.places, dev_err};
  RowsParams p{};
  p.x = x; p.ld_x = ld_x; p.rows = tokens; p.cols = hidden; p.q = s.xq; p.ld_q = hidden; p.scale = s.x_scale;
  p.places = s.places; p.topk = topk;
  cudaError_t e = launch_plan(plan, st);
  if (e == cudaSuccess) e = launch_rows(p, x_dtype, st);
  if (e != cudaSuccess) return report_cuda_error(e, what);
  Int8Product d{};
  d.x = s.xq; d.ld_x = hidden; d.x_scale = s.x_scale;
  d.w = w13; d.ld_w = ld_w13; d.stride_w = stride_w13; d.w_scale = w13_scale;
  d.rows = slots; d.experts = experts; d.n = 2 * inter; d.k = hidden;
  d.offsets = s.offsets;
  d.out = s.act; d.ld_out = inter; d.out_dtype = HEXMOE_F32; d.glu = 1;
  if (int rc = run_int8_product(what, d, st)) return rc;
  p = RowsParams{};
  p.x = s.act; p.ld_x = inter; p.rows = slots; p.cols = inter; p.q = s.actq; p.ld_q = inter; p.scale = s.act_scale;
  p.count = s.offsets + experts;
  e = launch_rows(p, HEXMOE_F32, st);
  if (e != cudaSuccess) return report_cuda_error(e, what);
  d = Int8Product{};
  d.x = s.actq; d.ld_x = inter; d.x_scale = s.act_scale;
  d.w = w2; d.ld_w = ld_w2; d.stride_w = stride_w2; d.w_scale = w2_scale;
  d.rows = slots; d.experts = experts; d.n = hidden; d.k = inter;
  d.offsets = s.offsets;
  d.out = s.y; d.ld_out = hidden; d.out_dtype = HEXMOE_F32;
  d.workspace = s.partial; d.workspace_bytes = s.partial_bytes;
  if (int rc = run_int8_product(what, d, st)) return rc;
  const SumParams sum = {s.y, s.places, topk_weights, out, tokens, topk, hidden};
  e = out_dtype == HEXMOE_F32   ? launch_sum<float>(sum, st)
      : out_dtype == HEXMOE_F16 ? launch_sum<__half>(sum, st)
                                : launch_sum<__nv_bfloat16>(sum, st);
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

}  // extern "C"
