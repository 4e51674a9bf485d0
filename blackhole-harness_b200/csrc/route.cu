// route.cu — the router of a MoE layer: scores, choice of experts and their weights, and the gradient of the logits.
//
//   s = softmax(l) or sigmoid(l);   c = s + b with a balancing bias, else l (which has the scores' order)
//   a group's value: the sum of its 1 or 2 largest s + b; the topk_groups groups of largest value are open
//   ids: the k largest c of the open groups;   w = scale s[ids], over their sum where renormalised
//   l = -inf masks an expert: s = 0, which is what its group is valued by; among the open groups' experts it comes last
//
// Ties go to the lower id.  A warp takes a token; lane l holds experts l NI .. l NI + NI - 1, so that lanes in order are
// experts in order.  Bound by latency and issue, not by bytes: a token's row is a few hundred.  8192 tokens of 256 experts
// in 8 groups, 4 of them open, top 8, sigmoid with a bias: 11.1 us (990 instructions a token; its 8.9 MB take HBM 1.4);
// one token 3.6 us, 4096 of 96 experts, softmax with a bias 5.2.  Above 512 experts a lane holds 64 values however few there
// are: 4096 tokens of 513 take 62 us, of 1024 37, of 2048 47 (top 8; top 32 222, 157, 201).
//
// Order is decided as in 64 bits.  What is compared without a bias are the logits themselves, which nothing has rounded.
// Sums s + b and groups' values are computed in f32 first, with fast exponentials.  Where two that a decision lies between
// are nearer than their errors' bound (a token in a thousand), the values in question alone are computed again in f64, an
// expert a lane: a warp that took its whole row through f64 would keep the kernel waiting (8192 tokens: 28 us of which 15
// were such rows').  Only where more than 32 experts are that near does the whole row go through choose_exact.
#include <algorithm>
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
constexpr size_t kRowsBytes = 40960;   // of keys, a block
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
  int32_t vec;            // rows (of logits, of their gradients, and biases) begin on 16 bytes and are whole pieces of 16 bytes
  int32_t group_lanes;    // lanes whose experts make a group, where they are whole lanes and a power of two; else 0
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
__device__ __forceinline__ uint32_t plain_key(float v) {   // of what is no NaN
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
constexpr uint32_t kMasked = 0x007fffffu;   // the key of -inf; NaN lies below
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// 1 / (1 + e^-l) without an overflow, and without a cancellation at either end.
__device__ __forceinline__ float sigmoid(float l) {
  const float e = expf(l < 0.f ? l : -l), r = 1.f / (1.f + e);
  return l < 0.f ? e * r : r;
}

// A token's values (logits, biases), NI to a lane, `none` past the last expert; in pieces of 16 bytes where p.vec says
// that rows begin on such.
template <typename T, int NI>
__device__ __forceinline__ void load_row(const RouteParams& p, const T* row, float none, float (&l)[NI]) {
  const int e0 = threadIdx.x % 32 * NI;
  if constexpr (NI * sizeof(T) % 16 == 0) {
    if (p.vec) {
      constexpr int kWords = NI * sizeof(T) / 4, kPer = 4 / sizeof(T);
      uint32_t w[kWords];
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        if (e0 + i * kPer < p.experts) {   // whole pieces: experts are a multiple of a piece
          const uint4 v = *reinterpret_cast<const uint4*>(row + e0 + i * kPer);
          w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if constexpr (sizeof(T) == 4) l[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __half>) l[i] = __half2float(__ushort_as_half(static_cast<uint16_t>(w[i / 2] >> i % 2 * 16)));
        else l[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        if (e0 + i >= p.experts) l[i] = none;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) l[i] = e0 + i < p.experts ? widen(row[e0 + i]) : none;
}
template <int NI>
__device__ __forceinline__ float largest_of(const float (&l)[NI]) {   // ignoring NaN
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NI; ++i) m = fmaxf(m, l[i]);
  return warp_max(m);
}
// Whether a row has no scores: it holds a NaN or, under a softmax, +inf (`largest`).  Its weights are all NaN, and a softmax's
// gradients: of the chosen logits alone neither would show where the NaN was not chosen.
template <int NI, bool SIGMOID>
__device__ __forceinline__ bool undefined(const float (&l)[NI], float largest) {
  bool nan = !SIGMOID && largest == INFINITY;
#pragma unroll
  for (int i = 0; i < NI; ++i) nan |= l[i] != l[i];
  return __any_sync(kAll, nan);
}
// e^x and 1 / x to 2 units in the last place, and the rounding of x log2 e (|x| 2^-24 of the result).
__device__ __forceinline__ float fast_exp(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
  return r;
}
__device__ __forceinline__ float fast_inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The scores of a row, for comparing.  Masked experts (-inf) have 0, also where every one is masked.  Returns the largest.
template <int NI, bool SIGMOID>
__device__ __forceinline__ float scores_of(const float (&l)[NI], float largest, float (&s)[NI]) {
  if constexpr (SIGMOID) {
#pragma unroll
    for (int i = 0; i < NI; ++i) s[i] = fast_inverse(1.f + fast_exp(-l[i]));
    return 1.f;
  } else {
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      s[i] = l[i] == -INFINITY ? 0.f : fast_exp(l[i] - largest);
      part += s[i];
    }
    const float sum = warp_sum(part), inv = sum == 0.f ? 0.f : fast_inverse(sum);
#pragma unroll
    for (int i = 0; i < NI; ++i) s[i] *= inv;
    return inv;
  }
}

// What is left of a row's softmax in f64: 1 for a sigmoid, the sum of e^(l - largest) otherwise.
template <typename T, bool SIGMOID>
__device__ double exact_sum(const RouteParams& p, const T* row, float largest) {
  if constexpr (SIGMOID) return 1.0;
  double part = 0.0;
#pragma unroll 1
  for (int e = threadIdx.x % 32; e < p.experts; e += 32) {
    const float l = widen(row[e]);
    if (l != -INFINITY) part += exp(static_cast<double>(l) - static_cast<double>(largest));
  }
  return warp_sum(part);
}
// s + b of one expert in f64; a masked one's s is 0.
template <typename T, bool SIGMOID>
__device__ double exact_value(const RouteParams& p, const T* row, int e, float largest, double sum) {
  const float l = widen(row[e]);
  const double d = l;
  double s = 0.0;
  if (l != -INFINITY) {
    const double x = exp(SIGMOID ? (d < 0 ? d : -d) : d - static_cast<double>(largest));
    s = SIGMOID ? (d < 0 ? x : 1.0) / (1.0 + x) : x / sum;
  }
  return p.bias ? s + static_cast<double>(p.bias[e]) : s;
}

__device__ __forceinline__ void add_top(uint32_t key, uint32_t& first, uint32_t& second) {
  const uint32_t less = min(first, key);
  first = max(first, key);
  second = max(second, less);
}

// What a selection finds.
struct Picked {
  int32_t id, count;   // lane j: the j-th expert; how many there are, 33 where they are too many for a warp
  bool near;           // two of the k first, or the last of them and what follows, lie no more than tau apart
};
__device__ __forceinline__ bool close_by(uint32_t above, uint32_t below, float tau) {
  // masked ones (-inf, NaN) are told apart by their ids, whatever their errors
  return below > kMasked && !(value_of(above) - value_of(below) > tau);
}

// The k largest of a warp's keys in order, equal ones by lane and place, one after the other; with `compare` as many
// behind them as lie no more than tau apart from one to the next.
template <int NI>
__device__ Picked pick_each(uint32_t (&key)[NI], int k, bool compare, float tau) {
  const int lane = threadIdx.x % 32;
  Picked got{0, k, false};
  uint32_t before = 0;
  for (int j = 0;; ++j) {
    if (j >= k && !compare) break;
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < NI; ++i) best = max(best, key[i]);
    const uint32_t top = __reduce_max_sync(kAll, best);
    if (compare) {
      const bool close = j > 0 && close_by(before, top, tau);
      got.near |= close;
      if (j >= k && (!close || j == 32)) {
        got.count = close ? 33 : j;
        break;
      }
      before = top;
    }
    const int owner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    int at = 0;
#pragma unroll
    for (int i = NI - 1; i >= 0; --i) at = key[i] == top ? i : at;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i < NI; ++i) key[i] = i == at ? 0u : key[i];
    }
    const int id = __shfl_sync(kAll, lane * NI + at, owner);
    if (lane == j) got.id = id;
  }
  return got;
}

// The same at a third of the instructions: the k-th largest of the lanes' largest keys bounds the k-th largest key from
// below, and few more than k keys reach it (or come within tau of it).  Those go through shared memory to a lane each, in
// the order of their ids, and are ranked by counting.  Where more than 32 do, or keys are equal too often, one by one.
struct Found {
  uint32_t key[32];
  int32_t id[32];
};
template <int NI>
__device__ __forceinline__ Picked pick(uint32_t (&key)[NI], int k, bool compare, float tau, Found& found) {
  const int lane = threadIdx.x % 32;
  uint32_t best = key[0], second = 0;
  if (k <= 8) {
#pragma unroll
    for (int i = 1; i < NI; ++i) best = max(best, key[i]);
  } else {   // more than the lanes of an open group or two may hold: two of each
#pragma unroll
    for (int i = 1; i < NI; ++i) add_top(key[i], best, second);
  }
  uint32_t bound = 0;
  for (int j = 0; j < k; ++j) {   // lanes of the same largest key leave together: the bound only falls
    bound = __reduce_max_sync(kAll, best);
    if (best == bound) {
      best = second;
      second = 0;
    }
  }
  if (compare && bound > kMasked) bound = key_of(value_of(bound) - tau);
  bound = max(bound, 1u);
  int mine = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) mine += key[i] >= bound;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kAll, upto, o);
    if (lane >= o) upto += v;
  }
  const int count = __shfl_sync(kAll, upto, 31);
  if (count > 32) {
    uint32_t copy[NI];   // what is handed on lives in memory: not the keys themselves
#pragma unroll
    for (int i = 0; i < NI; ++i) copy[i] = key[i];
    return pick_each(copy, k, compare, tau);
  }
  int at = upto - mine;
  if (mine) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (key[i] >= bound) {
        found.key[at] = key[i];
        found.id[at++] = lane * NI + i;
      }
    }
  }
  __syncwarp();
  const uint32_t my_key = lane < count ? found.key[lane] : 0u;
  const int32_t my_id = lane < count ? found.id[lane] : 0;
  int place = 0;
#pragma unroll 4
  for (int j = 0; j < count; ++j) {
    const uint32_t other = __shfl_sync(kAll, my_key, j);
    place += other > my_key || (other == my_key && j < lane);
  }
  __syncwarp();
  if (lane < count) {
    found.key[place] = my_key;
    found.id[place] = my_id;
  }
  __syncwarp();
  Picked got{0, count, false};
  if (lane < count) got.id = found.id[lane];
  if (compare) got.near = __any_sync(kAll, lane < k && lane + 1 < count && close_by(found.key[lane], found.key[lane + 1], tau));
  __syncwarp();   // the next row of this warp's may come
  return got;
}

// Where an expert's key stands in shared memory: a lane's even number of them one place on, in other banks.
template <int NI>
__device__ __forceinline__ int place_of(int e) { return NI % 2 ? e : e + e / NI; }

// The open groups as a bit each, from the values s + b (as keys); tau: what two groups' values may be off by together;
// keys: room for a row.
template <typename T, int NI, bool SIGMOID>
__device__ __forceinline__ uint32_t open_groups(const RouteParams& p, const T* row, const uint32_t (&key)[NI], float tau, float largest,
                                                uint32_t* keys) {
  const int lane = threadIdx.x % 32, per = p.experts / p.groups;
  const bool two = p.group_top > 1 && per > 1, in = lane < p.groups;
  // a lane's part of a group, or a lane's groups: lanes [g lanes, (g + 1) lanes) hold group g's two largest
  int lanes = p.group_lanes;
  uint32_t first = 0, second = 0;
  if (lanes) {   // a group is so many whole lanes, a power of two
#pragma unroll
    for (int i = 0; i < NI; ++i) add_top(key[i], first, second);
  } else {       // by way of shared memory
    lanes = 32 >> (32 - __clz(p.groups - 1));
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane * NI + i < p.experts) keys[place_of<NI>(lane * NI + i)] = key[i];
    __syncwarp();
    const int g = lane / lanes;
    if (g < p.groups)
      for (int i = lane % lanes; i < per; i += lanes) add_top(keys[place_of<NI>(g * per + i)], first, second);
    __syncwarp();
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const uint32_t f = __shfl_xor_sync(kAll, first, o), g = __shfl_xor_sync(kAll, second, o);
    add_top(f, first, second);
    second = max(second, g);
  }
  const float mine = __shfl_sync(kAll, two ? value_of(first) + value_of(second) : value_of(first), lane * lanes);
  auto rank = [&](auto k) {
    int ahead = 0;
#pragma unroll 4
    for (int g = 0; g < p.groups; ++g) {
      const auto other = __shfl_sync(kAll, k, g);
      ahead += other > k || (other == k && g < lane);
    }
    return ahead;
  };
  const uint32_t my_key = in ? key_of(mine) : 0u;
  int ahead = rank(my_key);
  // the last open group and the first closed one
  const float last = value_of(__shfl_sync(kAll, my_key, __ffs(__ballot_sync(kAll, in && ahead == p.topk_groups - 1)) - 1));
  const float next = value_of(__shfl_sync(kAll, my_key, __ffs(__ballot_sync(kAll, in && ahead == p.topk_groups)) - 1));
  if (!(last - next > tau) && !(last == -INFINITY && next == -INFINITY)) {
    // groups that near to the border: their values in f64, a warp on each
    const float away = fminf(fabsf(mine - last), fabsf(mine - next));
    const double sum = exact_sum<T, SIGMOID>(p, row, largest);
    double value = mine;
    uint32_t doubt = __ballot_sync(kAll, in && !(away > 2.f * tau));
    while (doubt) {
      const int g = __ffs(doubt) - 1;
      doubt &= doubt - 1;
      uint64_t first = 0, second = 0;
#pragma unroll 1
      for (int e = g * per + lane; e < (g + 1) * per; e += 32) {
        const uint64_t k = key_of(exact_value<T, SIGMOID>(p, row, e, largest, sum));
        second = max(second, min(first, k));
        first = max(first, k);
      }
      const uint64_t top = warp_max_key(first);
      double v = value_of(top);
      if (two) {
        const int owner = __ffs(__ballot_sync(kAll, first == top)) - 1;
        v += value_of(warp_max_key(lane == owner ? second : first));
      }
      if (lane == g) value = v;
    }
    ahead = rank(in ? key_of(value) : 0ull);
  }
  return __ballot_sync(kAll, in && ahead < p.topk_groups);
}

template <typename T, bool SIGMOID>
__device__ int32_t choose_exact(const RouteParams& p, const T* row, float largest);

// One token's experts, lane j the j-th.
template <typename T, int NI, bool SIGMOID>
__device__ __forceinline__ int32_t choose(const RouteParams& p, const T* row, const float (&l)[NI], float largest, Found& found,
                                          uint32_t* keys) {
  const int lane = threadIdx.x % 32, e0 = lane * NI;
  const bool grouped = p.topk_groups < p.groups;
  uint32_t key[NI];
  float tau = 0.f;
  if (p.bias || grouped) {
    float c[NI];
    const float top = scores_of<NI, SIGMOID>(l, largest, c);
    if (p.bias) {
      float b[NI];
      load_row(p, p.bias, 0.f, b);
#pragma unroll
      for (int i = 0; i < NI; ++i) c[i] += b[i];
    }
    // all logits and values finite, as a rule: then a key is their bits turned to their order
    const bool full = p.experts == 32 * NI;
    uint32_t most = 0, wide = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      wide = max(wide, __float_as_uint(c[i]) & 0x7fffffffu);
      most = max(most, full || e0 + i < p.experts ? __float_as_uint(l[i]) & 0x7fffffffu : 0u);
    }
    wide = __reduce_max_sync(kAll, wide);
    float widest = __uint_as_float(wide);
    const bool finite = max(wide, __reduce_max_sync(kAll, most)) < 0x7f800000u;
    if (finite) {
#pragma unroll
      for (int i = 0; i < NI; ++i) key[i] = full || e0 + i < p.experts ? plain_key(c[i]) : 0u;
    } else {
      widest = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        key[i] = e0 + i < p.experts ? key_of(c[i]) : 0u;
        const float size = fabsf(c[i]);
        widest = fmaxf(widest, size < INFINITY ? size : 0.f);
      }
      widest = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(widest)));
    }
    // Errors of the values, in units of 2^-24: a sigmoid 16 of 1 (of s (1 - s) times the exponential's 4 and its
    // argument's |l|, of s the sum's 1 and the reciprocal's 4); a softmax score, of the largest one, 48 (the exponential's
    // 4, its argument's two roundings, which count as much as |x| e^x, the reciprocal's 4, the product) and one for each
    // addition of a lane's sum and five of the warp's; the addition of the bias 1.  Two of each stand on the sides of a
    // decision, and twice as many where a group's value adds two.
    tau = 0x1p-23f * ((SIGMOID ? 16.f : 48.f + NI) * top + 2.f * widest);
    if (grouped) {
      const uint32_t open = open_groups<T, NI, SIGMOID>(p, row, key, 2.f * tau, largest, keys);
      if (!p.bias) {
#pragma unroll
        for (int i = 0; i < NI; ++i) key[i] = e0 + i < p.experts ? key_of(l[i]) : 0u;
      }
      if (p.group_lanes) {
        if (!(open >> lane / p.group_lanes & 1)) {
#pragma unroll
          for (int i = 0; i < NI; ++i) key[i] = 0;
        }
      } else {
        const int per = p.experts / p.groups;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (!(open >> ((e0 + i) / per & 31) & 1)) key[i] = 0;
      }
    }
    if (!finite) {   // what is masked, behind all others of the open groups
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (l[i] == -INFINITY && key[i] > kMasked) key[i] = kMasked;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) key[i] = e0 + i < p.experts ? key_of(l[i]) : 0u;
  }
  const Picked got = pick(key, p.topk, p.bias != nullptr, tau, found);
  if (!got.near) return got.id;
  if (got.count > 32) return choose_exact<T, SIGMOID>(p, row, largest);
  // in order of their values in f64, an expert a lane
  const double sum = exact_sum<T, SIGMOID>(p, row, largest);
  uint64_t mine = 0;
  if (lane < got.count)
    mine = key_of(widen(row[got.id]) == -INFINITY ? -INFINITY : exact_value<T, SIGMOID>(p, row, got.id, largest, sum));
  int place = 0;
#pragma unroll 1
  for (int j = 0; j < got.count; ++j) {
    const uint64_t other = __shfl_sync(kAll, mine, j);
    const int32_t id = __shfl_sync(kAll, got.id, j);
    place += other > mine || (other == mine && id < got.id);
  }
  int32_t id = 0;
#pragma unroll 1
  for (int j = 0; j < got.count; ++j) {
    const int at = __shfl_sync(kAll, place, j);
    const int32_t e = __shfl_sync(kAll, got.id, j);
    if (at == lane) id = e;
  }
  return id;
}

// The whole choice in f64, in rolled loops over local memory.
template <typename T, bool SIGMOID>
__device__ int32_t choose_exact(const RouteParams& p, const T* row, float largest) {
  const int lane = threadIdx.x % 32, held = (p.experts + 31) / 32, e0 = lane * held, per = p.experts / p.groups;
  uint64_t key[kMaxExperts / 32];
  const double sum = exact_sum<T, SIGMOID>(p, row, largest);
#pragma unroll 1
  for (int i = 0; i < held; ++i) key[i] = e0 + i < p.experts ? key_of(exact_value<T, SIGMOID>(p, row, e0 + i, largest, sum)) : 0ull;
  if (p.topk_groups < p.groups) {
    uint64_t mine = 0;
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      uint64_t first = 0, second = 0;
#pragma unroll 1
      for (int i = 0; i < held; ++i) {
        const int e = e0 + i;
        if (e < g * per || e >= (g + 1) * per) continue;
        second = max(second, min(first, key[i]));
        first = max(first, key[i]);
      }
      const uint64_t top = warp_max_key(first);
      double v = value_of(top);
      if (p.group_top > 1 && per > 1) {
        const int owner = __ffs(__ballot_sync(kAll, first == top)) - 1;
        v += value_of(warp_max_key(lane == owner ? second : first));
      }
      if (lane == g) mine = key_of(v);
    }
    int ahead = 0;
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t other = __shfl_sync(kAll, mine, g);
      ahead += other > mine || (other == mine && g < lane);
    }
    const uint32_t open = __ballot_sync(kAll, lane < p.groups && ahead < p.topk_groups);
#pragma unroll 1
    for (int i = 0; i < held; ++i)
      if (e0 + i < p.experts && !(open >> (e0 + i) / per & 1)) key[i] = 0;
  }
#pragma unroll 1
  for (int i = 0; i < held; ++i)   // what is masked, behind all others
    if (key[i] && widen(row[e0 + i]) == -INFINITY) key[i] = key_of(-static_cast<double>(INFINITY));
  int32_t id = 0;
#pragma unroll 1
  for (int j = 0; j < p.topk; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll 1
    for (int i = 0; i < held; ++i) {
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    }
    const uint64_t top = warp_max_key(best);
    const int owner = __ffs(__ballot_sync(kAll, best == top)) - 1, found = __shfl_sync(kAll, e0 + at, owner);
    if (lane == owner) key[at] = 0;
    if (lane == j) id = found;
  }
  return id;
}

// The share of every chosen score (lane j < k: logit l, else used = false) in their sum.  Where all of them are small, as a
// bias may choose, they are taken relative to their largest, or the smallest would be no normal numbers above a share of
// 2^-126; a sigmoid there is e^l but for 2^-24 of it.
template <bool SIGMOID>
__device__ __forceinline__ float share_of(float l, float largest, bool used) {
  float x = !used || l == -INFINITY ? 0.f : SIGMOID ? sigmoid(l) : expf(l - largest);
  float sum = warp_sum(x);
  if (sum < 0x1p-24f) {
    const float top = warp_max(used ? l : -INFINITY);
    x = !used || l == -INFINITY ? 0.f : expf(l - top);
    sum = warp_sum(x);
  }
  return sum > 0.f || sum != sum ? x / sum : 0.f;
}

template <typename T, int NI, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
  __shared__ Found found[kRouteThreads / 32];
  extern __shared__ __align__(16) uint8_t keys[];
  const int lane = threadIdx.x % 32;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  pdl_wait();
  if (t >= p.tokens) return;
  float l[NI];
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  load_row(p, row, -INFINITY, l);
  const float largest = SIGMOID ? 0.f : largest_of(l);
  const bool no_scores = undefined<NI, SIGMOID>(l, largest);
  const int32_t id = choose<T, NI, SIGMOID>(p, row, l, largest, found[threadIdx.x / 32],
                                            reinterpret_cast<uint32_t*>(keys) + threadIdx.x / 32 * (p.experts + 32));
  const bool used = lane < p.topk;
  const float mine = used ? widen(row[id]) : -INFINITY;
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
    p.weights[t * p.topk + lane] = no_scores ? __uint_as_float(0x7fc00000u) : w * p.scale;
    static_cast<int32_t*>(p.ids)[t * p.topk + lane] = id;
  }
}

// ---------------------------------------------------------------- gradient
// With d = scale dL/dw of the chosen experts j, their shares r_j = s_j / sum s and dot = sum_i r_i d_i:
//   renormalised softmax   dl_j = r_j (d_j - dot), 0 elsewhere (the softmax's own sum cancels)
//   renormalised sigmoid   dl_j = r_j (1 - s_j) (d_j - dot)
//   softmax                dl_e = s_e (d_e - sum_j s_j d_j), d_e = 0 where not chosen
//   sigmoid                dl_j = d_j s_j (1 - s_j)
// d_j - dot is summed as r_i (d_j - d_i), for the softmax s_i (d_j - d_i) over the chosen experts and d_j times what the
// others' scores sum to: a share or score near 1 leaves no cancellation (softmax, 4096 x 96, top 8: 3.6 us, 2.7 by the
// difference).  The row is written as what every expert has (0, or -s_e sum) and the chosen ones' values over it, by the same
// warp.  An expert that stands more than once among the ids has the sum of its places; ids outside 0..E-1 have no part.  A
// softmax's row with a NaN or +inf has a gradient of NaN, renormalised or not (which reads the row: 8191 x 256 bf16
// renormalised 5.3 us, 4.6 without); a sigmoid's chosen logits stand for themselves.
template <typename T, int NI, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const RouteParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  pdl_wait();
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  T* out = static_cast<T*>(p.dlogits) + t * p.ld_d;
  int32_t id = -1 - lane;   // no two alike where there is none
  float d = 0.f;
  if (lane < p.topk) {
    const int64_t v = p.ids64 ? static_cast<const int64_t*>(p.ids)[t * p.topk + lane]
                              : static_cast<const int32_t*>(p.ids)[t * p.topk + lane];
    if (v >= 0 && v < p.experts) {
      id = static_cast<int32_t>(v);
      d = p.weights[t * p.topk + lane] * p.scale;
    }
  }
  const bool used = id >= 0;
  const float mine = used ? widen(row[id]) : -INFINITY;
  const bool dense = !SIGMOID && !p.renorm;
  float value;
  if (dense) {
    float s[NI];   // of experts lane, lane + 32 ...: no order is asked for here
#pragma unroll
    for (int i = 0; i < NI; ++i) s[i] = lane + 32 * i < p.experts ? widen(row[lane + 32 * i]) : -INFINITY;
    const float largest = largest_of(s);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      s[i] = s[i] == -INFINITY ? 0.f : expf(s[i] - largest);
      part += s[i];
    }
    const float sum = warp_sum(part), inv = sum == 0.f ? 0.f : 1.f / sum;
    const float score = mine == -INFINITY ? 0.f : expf(mine - largest) * inv;
    const float dot = warp_sum(score * d);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane + 32 * i < p.experts) out[lane + 32 * i] = narrow<T>(-(s[i] * inv) * dot);
    float all = 0.f;   // of this expert's places
    bool again = false;   // it stands in a place before this one
    std::conditional_t<(NI > 32), uint64_t, uint32_t> chosen = 0;   // of the experts s holds
    for (int j = 0; j < p.topk; ++j) {
      const float dj = __shfl_sync(kAll, d, j);
      const int32_t other = __shfl_sync(kAll, id, j);
      all += other == id ? dj : 0.f;
      again |= other == id && j < lane;
      if (other >= 0 && (other & 31) == lane) chosen |= decltype(chosen){1} << (other >> 5);
    }
    float rest = 0.f, away = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) rest += chosen >> i & 1 ? 0.f : s[i];
    rest = warp_sum(rest) * inv;
    const float once = again ? 0.f : score;
    for (int j = 0; j < p.topk; ++j) away += __shfl_sync(kAll, once, j) * (all - __shfl_sync(kAll, all, j));
    value = score * (away + all * rest);
  } else {
    float l[NI];
    if constexpr (!SIGMOID) load_row(p, row, -INFINITY, l);   // only to see whether they are numbers
    if (p.vec) {
      for (int e = lane; e < p.experts * static_cast<int>(sizeof(T)) / 16; e += 32) reinterpret_cast<uint4*>(out)[e] = make_uint4(0, 0, 0, 0);
    } else {
      for (int e = lane; e < p.experts; e += 32) out[e] = narrow<T>(0.f);
    }
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
    if constexpr (!SIGMOID) {
      if (undefined<NI, SIGMOID>(l, largest_of(l))) {
        __syncwarp();   // over the zeros
        for (int e = lane; e < p.experts; e += 32) out[e] = narrow<T>(__uint_as_float(0x7fc00000u));
        return;
      }
    }
  }
  __syncwarp();   // the row's zeros (or common part) come before the chosen ones' values
  if (used) out[id] = narrow<T>(value);
}

template <typename T, int NI, bool SIGMOID>
cudaError_t launch_one(RouteParams p, bool backward, cudaStream_t st) {
  const int per = p.experts / p.groups, lanes = per / NI;
  p.group_lanes = per % NI == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  p.vec = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld * sizeof(T) % 16 == 0 && p.experts * sizeof(T) % 16 == 0 &&
          reinterpret_cast<uintptr_t>(p.bias) % 16 == 0 && (!p.bias || p.experts % 4 == 0) &&
          reinterpret_cast<uintptr_t>(p.dlogits) % 16 == 0 && p.ld_d * sizeof(T) % 16 == 0;
  // a token a warp: blocks of one warp until every SM has some, and no more than their rows of keys leave room for
  const size_t row = !backward && p.topk_groups < p.groups && !p.group_lanes ? sizeof(uint32_t) * (p.experts + 32) : 0;
  int warps = p.tokens <= 148 * 8 ? 1 : kRouteThreads / 32;
  if (row) warps = std::min(warps, static_cast<int>(kRowsBytes / row));
  const int64_t blocks = (p.tokens + warps - 1) / warps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = row * warps;
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
