// fgg_router.cu - the router of a mixture-of-experts layer: scores of a token's
// logits, its top-k experts and their combine weights, and the gradient of the
// logits.
//
//   s_e   = softmax(l)_e or sigmoid(l_e)
//   key_e = s_e + bias_e, or l_e without a bias (the same order)
//   ids   = the topk largest keys, largest first, ties to the lowest index
//   w_j   = scale * s_{ids_j} [ / sum_i s_{ids_i} ]
//
// An expert whose logit is -inf or NaN, or whose key is -inf or NaN, is not
// eligible; routes left over carry the id -1 (the layer's absent route) and the
// weight 0.  A row that holds a NaN (softmax: or +inf) logit has no scores: its
// weights are NaN.
//
// L lanes per token (8, 16 or 32 for up to 64, 128 or 1024 experts), each with V
// consecutive experts in registers, so that a warp works on up to four tokens and
// loads 16 bytes per lane.  Keys are compared in 32 bits; two neighbours of the
// order that lie closer than the keys' error send the tokens of the warp through
// the selection once more with 64-bit keys, computed for the few experts that can
// still be chosen, so that the order is that of the definition.  The logits are
// read once; what bounds the kernels is the chain of topk reductions for few
// tokens and their instructions for many.  Measured, one call of a replayed graph:
// 24 x 64 fp32 2.8 us; 4096 x 256 fp32 sigmoid 5.4 us, with a bias 10 us (one
// token in some hundred needs 64-bit keys, and the kernel waits for the last);
// gradient of 32768 x 64 bf16, whole softmax, top 8, 7.4 us (its 10.5 MB take 1.6 us of
// HBM), of 8 normalised weights 8.8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fgg_host.cuh"
#include "fgg_ptx.cuh"

namespace fgg {
namespace {

constexpr int kRouterMaxExperts = 1024;
constexpr int kRouterMaxTopk = 32;
constexpr int kRouterWarps = 4;
constexpr float kNegInf = -__builtin_huge_valf();

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Reductions over the L lanes of a token.
template <int L, typename V>
__device__ __forceinline__ V sub_sum(V v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float sub_max(float v) {  // NaN loses
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}

// Keys as unsigned integers of the same order; 0 = not eligible (NaN, -inf).
__device__ __forceinline__ uint32_t ordered(float f) {
  if (!(f > kNegInf)) return 0u;
  const uint32_t b = __float_as_uint(f + 0.0f);  // -0 equals +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t ordered(double f) {
  if (!(f > double(kNegInf))) return 0ull;
  const uint64_t b = uint64_t(__double_as_longlong(f + 0.0));
  return b >> 63 ? ~b : b | (1ull << 63);
}
template <int L>
__device__ __forceinline__ uint32_t sub_max_key(uint32_t k) {
  if constexpr (L == 32) return __reduce_max_sync(kFullMask, k);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(kFullMask, k, o));
  return k;
}
template <int L>
__device__ __forceinline__ uint64_t sub_max_key(uint64_t k) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(kFullMask, (unsigned long long)k, o);
    k = other > k ? other : k;
  }
  return k;
}

// The error that the order of two 32-bit keys must exceed to be trusted: scores are
// good to 1e-6, keys to that and two roundings.
__device__ __forceinline__ float key_error(float v) { return 4e-6f + 4e-7f * fabsf(v); }

// The topk largest of a token's keys, in order, into ids[0..topk) of the token (-1
// where fewer are eligible).  With `check`, one round more: false if two neighbours
// lie within their error, or one is infinite; *last: the topk-th key (or the
// smallest eligible).  The keys are used up.
template <int L, int V, bool check, class K>
__device__ __forceinline__ bool select_topk(K (&key)[V], int topk, int32_t* ids, K* last) {
  const int lane = threadIdx.x & 31, sub = lane & (L - 1);
  const unsigned group = L == 32 ? kFullMask : ((1u << L) - 1u) << (lane & ~(L - 1));
  K prev = 0;
  bool ok = true;
  const int rounds = check ? topk + 1 : topk;
  for (int j = 0; j < rounds; ++j) {
    K best = 0;
    int best_i = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] > best) {  // the lowest index among equal ones
        best = key[i];
        best_i = i;
      }
    const K top = sub_max_key<L>(best);
    if constexpr (check) {
      if (j > 0 && top != 0) {
        const float a = unordered(prev), b = unordered(top);
        ok = ok && a - b > key_error(a);  // false for infinities
      }
      if (j == topk) break;
      if (top != 0) *last = top;
      prev = top;
    }
    const unsigned same = __ballot_sync(kFullMask, best == top) & group;
    const bool win = top != 0 && lane == __ffs(same) - 1;  // the lowest lane holds the lowest index
    if (win) ids[j] = sub * V + best_i;
    if (top == 0 && sub == 0) ids[j] = -1;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (win && i == best_i) key[i] = 0;
  }
  return ok;
}

struct RouterParams {
  const void* logits;
  const float* bias;
  int32_t* ids;
  float* weights;
  const float* dweights;
  void* dlogits;
  int32_t tokens, experts, topk;
  int32_t renorm;
  int32_t vec;  // rows of logits (and dlogits) are whole, aligned 16-byte vectors
  float scale;
};

// This lane's V logits (-inf behind the last expert and for `live` false).  Whole
// 16-byte vectors where `vec` says that rows consist of them.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* row, int first, int experts, bool live,
                                            bool vec, float (&l)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) l[i] = kNegInf;
  if (!live) return;
  constexpr int N = 16 / int(sizeof(T));
  if (vec && V % N == 0) {
#pragma unroll
    for (int i = 0; i + N <= V; i += N)
      if (first + i < experts) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + first + i));
        const T* v = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int j = 0; j < N; ++j) l[i + j] = to_f32<T>(v[j]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (first + i < experts) l[i] = to_f32<T>(row[first + i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_logits(T* row, int first, int experts, bool live, bool vec,
                                             const float (&d)[V]) {
  if (!live) return;
  constexpr int N = 16 / int(sizeof(T));
  if (vec && V % N == 0) {
#pragma unroll
    for (int i = 0; i + N <= V; i += N)
      if (first + i < experts) {
        uint4 q;
        T* v = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = from_f32<T>(d[i + j]);
        *reinterpret_cast<uint4*>(row + first + i) = q;
      }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (first + i < experts) row[first + i] = from_f32<T>(d[i]);
  }
}

// Unnormalised score of a chosen expert, up to a factor that the chosen share
// (it cancels in the normalised weight): softmax exp(l - m); sigmoid divided by
// exp(min(m, 0)), so that small scores do not vanish.  m: the largest chosen logit.
template <bool kSoftmax>
__device__ __forceinline__ float chosen_score(float l, float m) {
  if (kSoftmax) return expf(l - m);
  if (l >= 0.0f) return 1.0f / (1.0f + expf(-l));
  return expf(l - fminf(m, 0.0f)) / (1.0f + expf(l));
}

template <typename T, int L, int V, bool kSoftmax>
__global__ void __launch_bounds__(32 * kRouterWarps)
    router_kernel(const __grid_constant__ RouterParams p) {
  constexpr int kTokens = kRouterWarps * 32 / L;  // of the block
  constexpr int R = (kRouterMaxTopk + L - 1) / L;  // routes of a lane: j = r L + sub
  __shared__ int32_t s_ids[kTokens][kRouterMaxTopk];
  const int lane = threadIdx.x & 31, sub = lane & (L - 1);
  const int slot = int(threadIdx.x) / L;
  const int64_t t = int64_t(blockIdx.x) * kTokens + slot;
  const bool live = t < p.tokens;
  const T* const row = static_cast<const T*>(p.logits) + (live ? t : 0) * p.experts;
  int32_t* const ids = s_ids[slot];
  float l[V];
  load_logits<T, V>(row, sub * V, p.experts, live, p.vec != 0, l);
  bool nan = false;
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    nan = nan || l[i] != l[i];
    m = fmaxf(m, l[i]);
  }
  nan = sub_max_key<L>(nan ? 1u : 0u) != 0u;
  m = sub_max<L>(m);
  if (kSoftmax && m == -kNegInf) nan = true;

  float total = 1.0f;  // softmax: sum of exp(l - m)
  if (kSoftmax && (p.bias != nullptr || !p.renorm)) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (l[i] > kNegInf) s += expf(l[i] - m);
    total = sub_sum<L>(s);
  }

  if (p.bias == nullptr) {
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = ordered(l[i]);
    select_topk<L, V, false>(key, p.topk, ids, static_cast<uint32_t*>(nullptr));
  } else {
    uint32_t key[V], used[V];
    float b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = sub * V + i;
      b[i] = e < p.experts ? __ldg(p.bias + e) : 0.0f;
      // a masked expert (-inf) stays out whatever its bias
      key[i] = 0u;
      if (l[i] > kNegInf)
        key[i] = ordered((kSoftmax ? expf(l[i] - m) / total : 1.0f / (1.0f + expf(-l[i]))) + b[i]);
      used[i] = key[i];
    }
    uint32_t last = 0;
    const bool clear = select_topk<L, V, true>(used, p.topk, ids, &last);
    if (__any_sync(kFullMask, !clear)) {
      // whoever can still be chosen has a key within both errors of the last one's
      const float v = unordered(last);
      const float least = v - 2.0f * key_error(v);
      uint64_t key64[V];
      double s64 = 1.0;
      if (kSoftmax) {
        s64 = 0.0;
#pragma unroll 1
        for (int i = 0; i < V; ++i)
          if (l[i] > kNegInf) s64 += exp(double(l[i]) - double(m));
        s64 = sub_sum<L>(s64);
      }
      uint32_t todo = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        key64[i] = 0ull;
        // (an infinite last key leaves its equals)
        if (key[i] != 0u && (key[i] >= last || unordered(key[i]) >= least)) todo |= 1u << i;
      }
      while (__any_sync(kFullMask, todo != 0u)) {
        const int at = todo != 0u ? __ffs(todo) - 1 : -1;
        todo &= todo - 1u;
        float li = 0.0f, bi = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == at) {
            li = l[i];
            bi = b[i];
          }
        const double s = kSoftmax ? exp(double(li) - double(m)) / s64 : 1.0 / (1.0 + exp(-double(li)));
        const uint64_t k = ordered(s + double(bi));
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == at) key64[i] = k;
      }
      __syncwarp();
      select_topk<L, V, false>(key64, p.topk, ids, static_cast<uint64_t*>(nullptr));
    }
  }
  __syncwarp();

  // the weights of this lane's routes
  int id[R];
  float lr[R], w[R];
  float mj = kNegInf;  // the largest chosen logit
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = r * L + sub;
    id[r] = j < p.topk ? ids[j] : -1;
    lr[r] = id[r] >= 0 && live ? to_f32<T>(row[id[r]]) : kNegInf;
    mj = fmaxf(mj, lr[r]);
  }
  mj = sub_max<L>(mj);
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    w[r] = 0.0f;
    if (id[r] >= 0) {
      if (p.renorm)
        w[r] = chosen_score<kSoftmax>(lr[r], mj);
      else
        w[r] = kSoftmax ? expf(lr[r] - m) / total : chosen_score<false>(lr[r], 0.0f);
    }
    sum += w[r];
  }
  if (p.renorm) sum = sub_sum<L>(sum);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = r * L + sub;
    if (!live || j >= p.topk) continue;
    float v = id[r] >= 0 ? w[r] * p.scale : 0.0f;
    if (p.renorm && id[r] >= 0) v = w[r] / sum * p.scale;
    if (nan) v = __int_as_float(0x7fc00000);
    p.ids[t * p.topk + j] = id[r];
    p.weights[t * p.topk + j] = v;
  }
}

// dlogits from dweights.  With c_j the share of route j,
//   softmax, normalised over the chosen   c_j = w_j sum_i w_i (dw_j - dw_i)
//   sigmoid, normalised                   c_j = w_j sum_i w_i (dw_j - dw_i) (1 - s_j)
//   sigmoid                               c_j = dw_j s_j (1 - s_j)
// (w normalised, without the scale), dl_e = sum of c_j over the routes to e.  For the
// whole softmax, with D_e the sum of dw_j over the routes to e,
//   e not chosen   dl_e = -s_e sum_f s_f D_f                          f over the chosen
//   e chosen       dl_e = s_e [ D_e (1 - sum_f s_f) + sum_f s_f (D_e - D_f) ]
// and 1 - sum_f s_f summed over the experts that are not chosen: where one expert has
// nearly all the score, s_e D_e - s_e sum_f s_f D_f would be the rounding of both.
// kDense (softmax without renormalisation): every expert's logit has a gradient.
template <typename T, int L, int V, bool kSoftmax, bool kDense>
__global__ void __launch_bounds__(32 * kRouterWarps)
    router_backward_kernel(const __grid_constant__ RouterParams p) {
  constexpr int kTokens = kRouterWarps * 32 / L;
  constexpr int R = (kRouterMaxTopk + L - 1) / L;
  __shared__ int2 s_share[kTokens][kRouterMaxTopk];  // each route's (weight, dw), (expert, share)
  static_assert(kSoftmax || !kDense, "a sigmoid's gradient is the chosen ones' own");
  // kDense: the chosen experts' gradients, each in its expert's place
  __shared__ float s_chosen[kDense ? kTokens : 1][kDense ? L * V : 1];
  const int sub = threadIdx.x & (L - 1);
  const int slot = int(threadIdx.x) / L;
  const int64_t t = int64_t(blockIdx.x) * kTokens + slot;
  const bool live = t < p.tokens;
  const T* const row = static_cast<const T*>(p.logits) + (live ? t : 0) * p.experts;
  const bool renorm = kSoftmax ? !kDense : p.renorm != 0;
  int id[R];
  float dw[R], lr[R], c[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = r * L + sub;
    id[r] = -1;
    dw[r] = 0.0f;
    if (live && j < p.topk) {
      id[r] = __ldg(p.ids + t * p.topk + j);
      dw[r] = __ldg(p.dweights + t * p.topk + j) * p.scale;
    }
    if (id[r] < 0 || id[r] >= p.experts) {  // an absent route
      id[r] = -1;
      dw[r] = 0.0f;
    }
  }
  float d[V];
  float m = 0.0f, total = 1.0f;
  if constexpr (kDense) {
    load_logits<T, V>(row, sub * V, p.experts, live, p.vec != 0, d);
    m = kNegInf;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, d[i]);
    m = sub_max<L>(m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = d[i] == kNegInf ? 0.0f : expf(d[i] - m);
      s += d[i];
    }
    total = sub_sum<L>(s);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) lr[r] = id[r] >= 0 ? to_f32<T>(row[id[r]]) : kNegInf;
  if constexpr (kDense) {
    // a masked expert has no score: its routes are absent
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r * L + sub;
      if (lr[r] == kNegInf) {
        id[r] = -1;
        dw[r] = 0.0f;
      }
      if (j < p.topk) s_share[slot][j] = make_int2(id[r], __float_as_int(dw[r]));
    }
    __syncwarp();
    uint32_t chosen = 0, twice = 0;  // of this lane's experts
    for (int i = 0; i < p.topk; ++i) {
      const unsigned at = unsigned(s_share[slot][i].x - sub * V);  // large for an absent route
      const uint32_t bit = at < unsigned(V) ? 1u << (at & 31u) : 0u;
      twice |= chosen & bit;
      chosen |= bit;
    }
    // D of this lane's routes; an expert's first route stands for it
    float all[R];
    bool first[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      all[r] = dw[r];
      first[r] = id[r] >= 0;
    }
    if (__any_sync(kFullMask, twice != 0u)) {  // a token of the warp names one twice
#pragma unroll
      for (int r = 0; r < R; ++r) all[r] = -0.0f;  // adds nothing, to -0 neither
      for (int i = 0; i < p.topk; ++i) {  // in the routes' order
        const int2 q = s_share[slot][i];
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (q.x == id[r]) {
            all[r] += __int_as_float(q.y);
            if (i < r * L + sub) first[r] = false;
          }
      }
    }
    float rest = 0.0f;  // score of the experts that are not chosen
#pragma unroll
    for (int i = 0; i < V; ++i) rest += chosen >> i & 1u ? 0.0f : d[i];
    // scores, all zero for a row that is masked whole (total 0), NaN for a NaN total
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    rest = sub_sum<L>(rest) * inv;
    float whole = 0.0f;
    __syncwarp();  // s_share is written over
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r * L + sub;
      c[r] = 0.0f;
      if (r * L < p.topk && first[r]) {
        c[r] = expf(lr[r] - m) * inv;
        whole += c[r] * all[r];
      }
      if (j < p.topk) s_share[slot][j] = make_int2(__float_as_int(c[r]), __float_as_int(all[r]));
    }
    whole = sub_sum<L>(whole);
    __syncwarp();
    float to[R];
#pragma unroll
    for (int r = 0; r < R; ++r) to[r] = rest * all[r];
    auto differences = [&](auto routes) {  // of a lane
      for (int i = 0; i < p.topk; ++i) {
        const int2 q = s_share[slot][i];
#pragma unroll
        for (int r = 0; r < decltype(routes)::value; ++r)
          to[r] = fmaf(__int_as_float(q.x), all[r] - __int_as_float(q.y), to[r]);
      }
    };
    if (p.topk <= L) differences(std::integral_constant<int, 1>());
    else differences(std::integral_constant<int, R>());
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (first[r]) s_chosen[slot][id[r]] = c[r] * to[r];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
      d[i] = chosen >> i & 1u ? s_chosen[slot][sub * V + i] : -(d[i] * inv) * whole;
  } else {
    float mj = kNegInf, sum = 0.0f;
    if (renorm) {
#pragma unroll
      for (int r = 0; r < R; ++r) mj = fmaxf(mj, lr[r]);
      mj = sub_max<L>(mj);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        c[r] = id[r] >= 0 && lr[r] != kNegInf ? chosen_score<kSoftmax>(lr[r], mj) : 0.0f;
        sum += c[r];
      }
      sum = sub_sum<L>(sum);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * L + sub;
        c[r] = sum == 0.0f ? 0.0f : c[r] / sum;
        if (j < p.topk) s_share[slot][j] = make_int2(__float_as_int(c[r]), __float_as_int(dw[r]));
      }
      __syncwarp();
      // w_j (dw_j - sum_i w_i dw_i) as w_j sum_i w_i (dw_j - dw_i): where one route has
      // nearly all the weight, the difference of the sum would be its rounding
      float to[R];
#pragma unroll
      for (int r = 0; r < R; ++r) to[r] = 0.0f;
      for (int i = 0; i < p.topk; ++i) {
        const int2 q = s_share[slot][i];
#pragma unroll
        for (int r = 0; r < R; ++r)
          to[r] = fmaf(__int_as_float(q.x), dw[r] - __int_as_float(q.y), to[r]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) c[r] *= to[r];
      __syncwarp();  // the shares are written over below
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float x = expf(-fabsf(lr[r]));
      if (renorm) {
        // 1 - sigmoid(l)
        if (!kSoftmax && id[r] >= 0) c[r] *= lr[r] >= 0.0f ? x / (1.0f + x) : 1.0f / (1.0f + x);
      } else {
        c[r] = id[r] >= 0 ? dw[r] * (x / ((1.0f + x) * (1.0f + x))) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = 0.0f;
  }
  if constexpr (!kDense) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r * L + sub;
      if (j < p.topk) s_share[slot][j] = make_int2(id[r], __float_as_int(c[r]));
    }
    __syncwarp();
    // in the routes' order, so that an expert named twice always gets the same sum
    for (int j = 0; j < p.topk; ++j) {
      const int2 q = s_share[slot][j];
      const int at = q.x - sub * V;
      if (q.x >= 0 && at >= 0 && at < V) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == at) d[i] += __int_as_float(q.y);
      }
    }
  }
  store_logits<T, V>(static_cast<T*>(p.dlogits) + (live ? t : 0) * p.experts, sub * V, p.experts,
                     live, p.vec != 0, d);
}

// Lanes per token and experts per lane by the number of experts.
template <typename T, bool kSoftmax, bool kBackward, bool kDense = false>
cudaError_t launch_router(const RouterParams& p, cudaStream_t s) {
  auto go = [&](auto lanes, auto values) {
    constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
    constexpr int kTokens = kRouterWarps * 32 / L;
    const int blocks = int((int64_t(p.tokens) + kTokens - 1) / kTokens);
    if constexpr (kBackward)
      router_backward_kernel<T, L, V, kSoftmax, kDense><<<blocks, 32 * kRouterWarps, 0, s>>>(p);
    else
      router_kernel<T, L, V, kSoftmax><<<blocks, 32 * kRouterWarps, 0, s>>>(p);
  };
  using std::integral_constant;
  if (p.experts <= 64) go(integral_constant<int, 8>(), integral_constant<int, 8>());
  else if (p.experts <= 128) go(integral_constant<int, 16>(), integral_constant<int, 8>());
  else if (p.experts <= 256) go(integral_constant<int, 32>(), integral_constant<int, 8>());
  else if (p.experts <= 512) go(integral_constant<int, 32>(), integral_constant<int, 16>());
  else go(integral_constant<int, 32>(), integral_constant<int, 32>());
  return cudaGetLastError();
}

// Rows of whole, aligned 16-byte vectors.
bool rows_of_vectors(const void* a, const void* b, int experts, int dtype) {
  return experts % (dtype == 0 ? 4 : 8) == 0 && aligned16(a) && aligned16(b);
}

template <typename T, bool kBackward>
cudaError_t launch_router(const RouterParams& p, bool softmax, cudaStream_t s) {
  if (!softmax) return launch_router<T, false, kBackward>(p, s);
  if (kBackward && !p.renorm) return launch_router<T, true, kBackward, kBackward>(p, s);
  return launch_router<T, true, kBackward>(p, s);
}
template <bool kBackward>
cudaError_t launch_router(const RouterParams& p, int dtype, bool softmax, cudaStream_t s) {
  if (dtype == 0) return launch_router<float, kBackward>(p, softmax, s);
  if (dtype == 1) return launch_router<__nv_bfloat16, kBackward>(p, softmax, s);
  return launch_router<__half, kBackward>(p, softmax, s);
}

int check_router(const void* logits, int dtype, int tokens, int experts, int topk, int score) {
  if (dtype < 0 || dtype > 2)
    return set_error(FGG_EINVAL, "dtype=%d must be 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  if (score != 0 && score != 1)
    return set_error(FGG_EINVAL, "score=%d must be 0 (softmax) or 1 (sigmoid)", score);
  if (tokens < 0) return set_error(FGG_EINVAL, "tokens=%d is negative", tokens);
  if (experts < 1 || experts > kRouterMaxExperts)
    return set_error(FGG_EBADSHAPE, "experts=%d outside [1, %d]", experts, kRouterMaxExperts);
  if (topk < 1 || topk > experts || topk > kRouterMaxTopk)
    return set_error(FGG_EBADSHAPE, "topk=%d outside [1, min(%d experts, %d)]", topk, experts,
                     kRouterMaxTopk);
  if (tokens > 0 && logits == nullptr) return set_error(FGG_EINVAL, "logits is null");
  const uintptr_t a = dtype == 0 ? 3u : 1u;
  if ((reinterpret_cast<uintptr_t>(logits) & a) != 0)
    return set_error(FGG_EALIGN, "logits is not aligned to its type");
  return FGG_OK;
}

}  // namespace
}  // namespace fgg

using namespace fgg;

extern "C" {

int fgg_moe_router(const void* logits, int32_t dtype, int32_t tokens, int32_t experts,
                   int32_t topk, int32_t score, const float* bias, int32_t renormalize,
                   float scale, int32_t* ids, float* weights, void* stream) {
  if (int rc = check_router(logits, dtype, tokens, experts, topk, score)) return rc;
  if (tokens == 0) return FGG_OK;
  if (ids == nullptr || weights == nullptr) return set_error(FGG_EINVAL, "ids / weights is null");
  if (!aligned4(bias) || !aligned4(ids) || !aligned4(weights))
    return set_error(FGG_EALIGN, "bias, ids and weights must be 4-byte aligned");
  DeviceInfo dev;
  if (int rc = current_device(&dev)) return rc;
  RouterParams p = {};
  p.logits = logits;
  p.bias = bias;
  p.ids = ids;
  p.weights = weights;
  p.tokens = tokens;
  p.experts = experts;
  p.topk = topk;
  p.renorm = renormalize != 0;
  p.vec = rows_of_vectors(logits, nullptr, experts, dtype);
  p.scale = scale;
  FGG_CUDA_CHECK(launch_router<false>(p, dtype, score == 0, reinterpret_cast<cudaStream_t>(stream)));
  return FGG_OK;
}

int fgg_moe_router_backward(const float* dweights, const void* logits, int32_t dtype,
                            const int32_t* ids, int32_t tokens, int32_t experts, int32_t topk,
                            int32_t score, int32_t renormalize, float scale, void* dlogits,
                            void* stream) {
  if (int rc = check_router(logits, dtype, tokens, experts, topk, score)) return rc;
  if (tokens == 0) return FGG_OK;
  if (dweights == nullptr || ids == nullptr || dlogits == nullptr)
    return set_error(FGG_EINVAL, "dweights / ids / dlogits is null");
  if (!aligned4(ids) || !aligned4(dweights))
    return set_error(FGG_EALIGN, "dweights and ids must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(dlogits) & (dtype == 0 ? 3u : 1u)) != 0)
    return set_error(FGG_EALIGN, "dlogits is not aligned to its type");
  DeviceInfo dev;
  if (int rc = current_device(&dev)) return rc;
  RouterParams p = {};
  p.logits = logits;
  p.ids = const_cast<int32_t*>(ids);
  p.dweights = dweights;
  p.dlogits = dlogits;
  p.tokens = tokens;
  p.experts = experts;
  p.topk = topk;
  p.renorm = renormalize != 0;
  p.vec = rows_of_vectors(logits, dlogits, experts, dtype);
  p.scale = scale;
  FGG_CUDA_CHECK(launch_router<true>(p, dtype, score == 0, reinterpret_cast<cudaStream_t>(stream)));
  return FGG_OK;
}

}  // extern "C"
