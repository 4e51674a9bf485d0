// route.cu — the router of a MoE layer: scores, choice of experts and their weights, and the gradient of the logits.
//
//   s = softmax(l) or sigmoid(l);   c = s + b with a balancing bias, else l (which has the scores' order)
//   a group's value: the sum of its 1 or 2 largest s + b; the topk_groups groups of largest value are open
//   ids: the k largest c of the open groups;   w = scale s[ids], over their sum where renormalised
//
// Ties go to the lower id.  A warp takes a token; lane l holds experts l NI .. l NI + NI - 1, so that lanes in order are
// experts in order.  Bound by latency and issue, not by bytes: a token's row is a few hundred.
//
// Order is decided as in 64 bits.  What is compared without a bias are the logits themselves, which nothing has rounded.
// Sums s + b and groups' values are computed in f32 first; where two that a decision lies between are nearer than their
// errors' bound (a token in a hundred), the warp computes them again in f64 and decides by those.
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "internal.cuh"
#include "ptx.cuh"

namespace hexmoe {
namespace {

constexpr int kRouteThreads = 256;
constexpr int kMaxTopk = 32;       // a lane a weight
constexpr int kMaxGroups = 32;     // a lane a group
constexpr int kMaxExperts = 2048;  // 64 a lane
constexpr unsigned kAll = 0xffffffffu;

int arg_error(const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_error(HEXMOE_E_ARG, buf);
}

struct RouteParams {
  const void* logits;
  const float* bias;      // [experts] or null
  float* weights;         // forward: out; backward: the gradient of the weights
  void* ids;              // int32 out; backward: int32 or int64
  void* dlogits;          // backward
  int64_t tokens, ld, ld_d;
  int32_t experts, topk, groups, topk_groups, group_top, renorm, ids64;
  float scale;
};

template <typename T>
__device__ __forceinline__ float widen(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Whole numbers in the order of the values: NaN below everything, 0 for what must not be chosen.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);   // -0 is 0
  return v != v ? 1u : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return v != v ? 1ull : b ^ (b >> 63 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return k <= 1 ? __uint_as_float(0x7fc00000u) : __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return k <= 1 ? __longlong_as_double(0x7ff8000000000000ll)
                : __longlong_as_double(static_cast<long long>(k ^ (k >> 63 ? 1ull << 63 : ~0ull)));
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// 1 / (1 + e^-l) without an overflow, and without a cancellation at either end.
template <typename F>
__device__ __forceinline__ F sigmoid(F l) {
  const F e = exp_of(l < F(0) ? l : -l), r = F(1) / (F(1) + e);
  return l < F(0) ? e * r : r;
}

// A token's logits, one warp: NI to a lane, -inf past the last expert; largest is their largest, ignoring NaN.
template <typename T, int NI>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t t, float (&l)[NI]) {
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  const int e0 = threadIdx.x % 32 * NI;
#pragma unroll
  for (int i = 0; i < NI; ++i) l[i] = e0 + i < p.experts ? widen(row[e0 + i]) : -INFINITY;
}
template <int NI>
__device__ __forceinline__ float largest_of(const float (&l)[NI]) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NI; ++i) m = fmaxf(m, l[i]);
  return warp_max(m);
}

// The scores of a row.  Masked experts (-inf) have 0, also where every one is masked.
template <typename F, int NI, bool SIGMOID>
__device__ __forceinline__ void scores_of(const float (&l)[NI], float largest, F (&s)[NI], F& sum) {
  sum = F(1);
  if constexpr (SIGMOID) {
#pragma unroll
    for (int i = 0; i < NI; ++i) s[i] = l[i] == -INFINITY ? F(0) : sigmoid(F(l[i]));
  } else {
    F part = F(0);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      s[i] = l[i] == -INFINITY ? F(0) : exp_of(F(l[i]) - F(largest));
      part += s[i];
    }
    sum = warp_sum(part);
    const F inv = sum > F(0) || sum != sum ? F(1) / sum : F(0);
#pragma unroll
    for (int i = 0; i < NI; ++i) s[i] *= inv;
  }
}

// What a selection finds: lane j holds the j-th expert and its key; next: the key behind the last one.
template <typename K>
struct Picked {
  int32_t id;
  K key, next;
};

// The k largest of a warp's keys, equal ones by lane and place.  Keys that are chosen become 0.
template <typename K, int NI>
__device__ __forceinline__ Picked<K> pick(K (&key)[NI], int k, bool want_next) {
  const int lane = threadIdx.x % 32;
  Picked<K> got{0, 0, 0};
  for (int j = 0; j < k + (want_next ? 1 : 0); ++j) {
    K best = key[0];
#pragma unroll
    for (int i = 1; i < NI; ++i) best = key[i] > best ? key[i] : best;
    const K top = warp_max_key(best);
    if (j == k) {
      got.next = top;
      break;
    }
    const int owner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    int at = 0;
#pragma unroll
    for (int i = NI - 1; i >= 0; --i) at = key[i] == top ? i : at;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i < NI; ++i) key[i] = i == at ? K(0) : key[i];
    }
    const int id = __shfl_sync(kAll, lane * NI + at, owner);
    if (lane == j) {
      got.id = id;
      got.key = top;
    }
  }
  return got;
}

// The open groups as a bit each, from the values s + b (as keys).  near: whether a decision lay between two values
// less than `tau` apart.
template <typename F, typename K, int NI>
__device__ __forceinline__ uint32_t open_groups(const RouteParams& p, const K (&key)[NI], F tau, bool& near) {
  const int lane = threadIdx.x % 32, per = p.experts / p.groups, e0 = lane * NI;
  F mine = F(0);
  for (int g = 0; g < p.groups; ++g) {
    K first = 0, second = 0;   // of this lane's experts in the group
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const K k = e0 + i >= g * per && e0 + i < (g + 1) * per ? key[i] : K(0);
      if (k > first) {
        second = first;
        first = k;
      } else if (k > second) {
        second = k;
      }
    }
    const K top = warp_max_key(first);
    F v = value_of(top);
    if (p.group_top > 1 && per > 1) {
      const int owner = __ffs(__ballot_sync(kAll, first == top)) - 1;
      v += value_of(warp_max_key(lane == owner ? second : first));
    }
    if (lane == g) mine = v;
  }
  int ahead = 0;
  const K my_key = lane < p.groups ? key_of(mine) : K(0);
  for (int g = 0; g < p.groups; ++g) {
    const K other = __shfl_sync(kAll, my_key, g);
    ahead += other > my_key || (other == my_key && g < lane);
  }
  const bool open = lane < p.groups && ahead < p.topk_groups;
  if (near) {   // asked for: the last open value and the first closed one
    const F last = value_of(__shfl_sync(kAll, my_key, __ffs(__ballot_sync(kAll, lane < p.groups && ahead == p.topk_groups - 1)) - 1));
    const F next = value_of(__shfl_sync(kAll, my_key, __ffs(__ballot_sync(kAll, lane < p.groups && ahead == p.topk_groups)) - 1));
    near = !(last - next > tau);
  }
  return __ballot_sync(kAll, open);
}

// One token's choice in type F (float, double).  near: set where f32 could not decide.
template <typename F, int NI, bool SIGMOID>
__device__ __forceinline__ int32_t choose(const RouteParams& p, const float (&l)[NI], float largest, bool& near) {
  using K = std::conditional_t<std::is_same_v<F, float>, uint32_t, uint64_t>;
  const int e0 = threadIdx.x % 32 * NI, lane = threadIdx.x % 32;
  const bool grouped = p.topk_groups < p.groups;
  K key[NI];
  F tau = F(0);
  if (p.bias || grouped) {
    F s[NI], sum;
    scores_of<F, NI, SIGMOID>(l, largest, s, sum);
    float widest = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      F c = s[i];
      if (e0 + i < p.experts) {
        if (p.bias) c = l[i] == -INFINITY ? F(-INFINITY) : c + F(p.bias[e0 + i]);
        key[i] = key_of(c);
      } else {
        key[i] = 0;
      }
      if (fabs(c) < F(INFINITY)) widest = fmaxf(widest, static_cast<float>(fabs(c)));
    }
    if constexpr (std::is_same_v<F, float>) {
      // f32 errors, in units of 2^-24: a sigmoid 8 of itself (the exponential 4, the sum, the divide); a softmax score
      // 40 (the exponent's rounding, up to 30 where the score counts, the exponential, the divide) and one for each
      // addition of its sum; the addition of the bias 1.  Two of each stand on the sides of a decision, and twice as
      // many where a group's value adds two.
      const float top = SIGMOID ? 1.f : (sum > 0.f ? 1.f / sum : 0.f);
      tau = 0x1p-23f * ((SIGMOID ? 8.f : 45.f + NI) * top + 2.f * warp_max(widest));
    }
    uint32_t open = kAll;
    if (grouped) {
      near = std::is_same_v<F, float>;
      open = open_groups<F>(p, key, F(2) * tau, near);
      if (near) return 0;
    }
    const int per = p.experts / p.groups;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (!p.bias) key[i] = e0 + i < p.experts ? K(key_of(F(l[i]))) : K(0);
      if (grouped && !(open >> ((e0 + i) / per & 31) & 1)) key[i] = 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) key[i] = e0 + i < p.experts ? K(key_of(F(l[i]))) : K(0);
  }
  const bool check = std::is_same_v<F, float> && p.bias;
  const Picked<K> got = pick(key, p.topk, check);
  near = false;
  if (check) {
    const K behind = __shfl_down_sync(kAll, got.key, 1);
    const F v = value_of(got.key), next = value_of(lane == p.topk - 1 ? got.next : behind);
    // nothing chosen lies behind the last one, or both are masked: by their ids, whatever their errors
    const bool sure = (lane == p.topk - 1 && got.next == 0) || (v == F(-INFINITY) && next == F(-INFINITY));
    near = __any_sync(kAll, lane < p.topk && !sure && !(v - next > tau));
  }
  return got.id;
}

// The share of every chosen score (lane j < k: logit l, else used = false) in their sum.
template <bool SIGMOID>
__device__ __forceinline__ float share_of(float l, float largest, bool used) {
  float x = !used || l == -INFINITY ? 0.f : SIGMOID ? sigmoid(l) : expf(l - largest);
  float sum = warp_sum(x);
  if (sum < 1e-30f) {   // scores below f32's range: there a sigmoid is e^l too
    const float top = warp_max(used ? l : -INFINITY);
    x = !used || l == -INFINITY ? 0.f : expf(l - top);
    sum = warp_sum(x);
  }
  return sum > 0.f || sum != sum ? x / sum : 0.f;
}

template <typename T, int NI, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  pdl_wait();
  if (t >= p.tokens) return;
  float l[NI];
  load_row<T>(p, t, l);
  const float largest = largest_of(l);
  bool near = false;
  int32_t id = choose<float, NI, SIGMOID>(p, l, largest, near);
  if (near) id = choose<double, NI, SIGMOID>(p, l, largest, near);
  const bool used = lane < p.topk;
  const float mine = used ? widen(static_cast<const T*>(p.logits)[t * p.ld + id]) : -INFINITY;
  float w;
  if (p.renorm) {
    w = share_of<SIGMOID>(mine, largest, used);
  } else if constexpr (SIGMOID) {
    w = mine == -INFINITY ? 0.f : sigmoid(mine);
  } else {
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) part += l[i] == -INFINITY ? 0.f : expf(l[i] - largest);
    const float sum = warp_sum(part);
    w = mine == -INFINITY && sum == sum ? 0.f : expf(mine - largest) / sum;
  }
  if (used) {
    p.weights[t * p.topk + lane] = w * p.scale;
    static_cast<int32_t*>(p.ids)[t * p.topk + lane] = id;
  }
}

// ---------------------------------------------------------------- gradient
// With d = scale dL/dw of the chosen experts j, their shares r_j = s_j / sum s and dot = sum_i r_i d_i:
//   renormalised softmax   dl_j = r_j (d_j - dot), 0 elsewhere (the softmax's own sum cancels)
//   renormalised sigmoid   dl_j = r_j (1 - s_j) (d_j - dot)
//   softmax                dl_e = s_e (d_e - sum_j s_j d_j), d_e = 0 where not chosen
//   sigmoid                dl_j = d_j s_j (1 - s_j)
// d_j - dot is summed as r_i (d_j - d_i): a share near 1 leaves no cancellation.  The row is written as what every
// expert has (0, or -s_e sum) and the chosen ones' values over it, by the same warp.  An expert that stands more than
// once among the ids has the sum of its places; ids outside 0..E-1 have no part.
template <typename T, int NI, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const RouteParams p) {
  const int lane = threadIdx.x % 32, e0 = lane * NI;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  pdl_wait();
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  T* out = static_cast<T*>(p.dlogits) + t * p.ld_d;
  int64_t id = -1 - lane;   // no two alike where there is none
  float d = 0.f;
  if (lane < p.topk) {
    const int64_t v = p.ids64 ? static_cast<const int64_t*>(p.ids)[t * p.topk + lane]
                              : static_cast<const int32_t*>(p.ids)[t * p.topk + lane];
    if (v >= 0 && v < p.experts) {
      id = v;
      d = p.weights[t * p.topk + lane] * p.scale;
    }
  }
  const bool used = id >= 0;
  const float mine = used ? widen(row[id]) : -INFINITY;
  const bool dense = !SIGMOID && !p.renorm;
  float value;
  if (dense) {
    float l[NI], s[NI], sum;
    load_row<T>(p, t, l);
    const float largest = largest_of(l);
    scores_of<float, NI, false>(l, largest, s, sum);
    const float score = mine == -INFINITY ? 0.f : expf(mine - largest) / sum;
    const float dot = warp_sum(score * d);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (e0 + i < p.experts) out[e0 + i] = narrow<T>(-s[i] * dot);
    float all = 0.f;   // of this expert's places
    for (int j = 0; j < p.topk; ++j) {
      const float dj = __shfl_sync(kAll, d, j);
      if (__shfl_sync(kAll, id, j) == id) all += dj;
    }
    value = score * (all - dot);
  } else {
    for (int e = lane; e < p.experts; e += 32) out[e] = narrow<T>(0.f);
    if (p.renorm) {
      const float r = share_of<SIGMOID>(mine, SIGMOID ? 0.f : warp_max(mine), used);
      float away = 0.f;
      for (int j = 0; j < p.topk; ++j) away += __shfl_sync(kAll, r, j) * (d - __shfl_sync(kAll, d, j));
      value = r * away;
      if constexpr (SIGMOID) value *= sigmoid(-mine);
    } else {
      value = d * sigmoid(mine) * sigmoid(-mine);
    }
    if (mine == -INFINITY) value = 0.f;
    float all = 0.f;
    for (int j = 0; j < p.topk; ++j) {
      const float vj = __shfl_sync(kAll, value, j);
      if (__shfl_sync(kAll, id, j) == id) all += vj;
    }
    value = all;
  }
  __syncwarp();   // the row's zeros (or common part) come before the chosen ones' values
  if (used) out[id] = narrow<T>(value);
}

template <typename T, int NI, bool SIGMOID>
cudaError_t launch_one(const RouteParams& p, bool backward, cudaStream_t st) {
  // a token a warp: blocks of one warp until every SM has some
  const int warps = p.tokens <= 148 * 8 ? 1 : kRouteThreads / 32;
  const int64_t blocks = (p.tokens + warps - 1) / warps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return backward ? cudaLaunchKernelEx(&cfg, route_backward_kernel<T, NI, SIGMOID>, p)
                  : cudaLaunchKernelEx(&cfg, route_kernel<T, NI, SIGMOID>, p);
}

template <typename T, bool SIGMOID>
cudaError_t launch_experts(const RouteParams& p, bool backward, cudaStream_t st) {
  const int per_lane = (p.experts + 31) / 32;
  if (per_lane <= 1) return launch_one<T, 1, SIGMOID>(p, backward, st);
  if (per_lane <= 2) return launch_one<T, 2, SIGMOID>(p, backward, st);
  if (per_lane <= 3) return launch_one<T, 3, SIGMOID>(p, backward, st);
  if (per_lane <= 4) return launch_one<T, 4, SIGMOID>(p, backward, st);
  if (per_lane <= 8) return launch_one<T, 8, SIGMOID>(p, backward, st);
  if (per_lane <= 16) return launch_one<T, 16, SIGMOID>(p, backward, st);
  return launch_one<T, 64, SIGMOID>(p, backward, st);
}

int run(const char* what, const RouteParams& p, int32_t dtype, int32_t scoring, bool backward, void* stream) {
  if (dtype != HEXMOE_F32 && dtype != HEXMOE_BF16 && dtype != HEXMOE_F16) return report_error(HEXMOE_E_DTYPE, "route: bad logits dtype");
  if (scoring != HEXMOE_SOFTMAX && scoring != HEXMOE_SIGMOID) return arg_error("%s: scoring %d", what, scoring);
  if (p.tokens < 0 || p.tokens > 0x7fffffffll || p.experts <= 0 || p.experts > kMaxExperts)
    return arg_error("%s: tokens %lld, experts %d (at most %d)", what, static_cast<long long>(p.tokens), p.experts, kMaxExperts);
  if (p.topk <= 0 || p.topk > kMaxTopk) return arg_error("%s: topk %d (1 to %d)", what, p.topk, kMaxTopk);
  if (p.ld < p.experts || (backward && p.ld_d < p.experts)) return arg_error("%s: a row stride is shorter than its row", what);
  if (p.tokens == 0) return HEXMOE_OK;
  const size_t z = dtype == HEXMOE_F32 ? 4 : 2;
  auto bad = [](const void* q, size_t size) { return !q || reinterpret_cast<uintptr_t>(q) % size; };
  if (bad(p.logits, z) || bad(p.weights, 4) || bad(p.ids, p.ids64 ? 8 : 4) || (backward && bad(p.dlogits, z)) ||
      reinterpret_cast<uintptr_t>(p.bias) % 4)
    return arg_error("%s: null pointer, or one not aligned to its element", what);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    return scoring == HEXMOE_SIGMOID ? launch_experts<T, true>(p, backward, st) : launch_experts<T, false>(p, backward, st);
  };
  const cudaError_t e = dtype == HEXMOE_F32 ? go(float{}) : dtype == HEXMOE_F16 ? go(__half{}) : go(__nv_bfloat16{});
  return e == cudaSuccess ? HEXMOE_OK : report_cuda_error(e, what);
}

}  // namespace
}  // namespace hexmoe

using namespace hexmoe;

extern "C" {

int hexmoe_route(const void* logits, int32_t logits_dtype, int64_t ld_logits, int64_t tokens, int32_t num_experts,
                 int32_t topk, int32_t scoring, const float* bias, int32_t groups, int32_t topk_groups,
                 int32_t group_top, int32_t renormalize, float scale, float* topk_weights, int32_t* topk_ids,
                 void* stream) {
  const char* what = "hexmoe_route";
  if (groups <= 0 || groups > kMaxGroups || num_experts % groups || topk_groups <= 0 || topk_groups > groups ||
      group_top < 1 || group_top > 2)
    return arg_error("%s: %d experts in %d groups (at most %d), %d of them open, %d values a group (1 or 2)", what,
                     num_experts, groups, kMaxGroups, topk_groups, group_top);
  if (num_experts > 0 && topk > num_experts / groups * topk_groups)
    return arg_error("%s: topk %d of %d experts in open groups", what, topk, num_experts / groups * topk_groups);
  RouteParams p{};
  p.logits = logits; p.bias = bias; p.weights = topk_weights; p.ids = topk_ids;
  p.tokens = tokens; p.ld = ld_logits;
  p.experts = num_experts; p.topk = topk; p.groups = groups; p.topk_groups = topk_groups; p.group_top = group_top;
  p.renorm = renormalize; p.scale = scale;
  return run(what, p, logits_dtype, scoring, false, stream);
}

int hexmoe_route_backward(const float* dweights, const void* logits, int32_t logits_dtype, int64_t ld_logits,
                          int64_t tokens, int32_t num_experts, int32_t topk, const void* topk_ids, int32_t ids_dtype,
                          int32_t scoring, int32_t renormalize, float scale, void* dlogits, int64_t ld_dlogits,
                          void* stream) {
  if (ids_dtype != HEXMOE_I32 && ids_dtype != HEXMOE_I64) return report_error(HEXMOE_E_DTYPE, "hexmoe_route_backward: ids are I32 or I64");
  RouteParams p{};
  p.logits = logits; p.weights = const_cast<float*>(dweights); p.ids = const_cast<void*>(topk_ids); p.dlogits = dlogits;
  p.tokens = tokens; p.ld = ld_logits; p.ld_d = ld_dlogits;
  p.experts = num_experts; p.topk = topk; p.groups = p.topk_groups = p.group_top = 1;
  p.renorm = renormalize; p.ids64 = ids_dtype == HEXMOE_I64; p.scale = scale;
  return run("hexmoe_route_backward", p, logits_dtype, scoring, true, stream);
}

}  // extern "C"
