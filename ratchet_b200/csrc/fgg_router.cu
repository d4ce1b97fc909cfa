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
// One warp per token, its logits in registers (lane l holds experts 32 i + l).
// Keys are compared in 32 bits; two neighbours of the order that lie closer than
// the keys' error send the token through the same selection on 64-bit keys, so
// that the order is that of the definition.  The logits are read once; what
// bounds the kernels is that read for many tokens and one warp's chain of
// topk reductions for few.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fgg_host.cuh"
#include "fgg_ptx.cuh"

namespace fgg {
namespace {

constexpr int kRouterMaxExperts = 1024;
constexpr int kRouterMaxTopk = 32;  // a lane per route
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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {  // NaN loses
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
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
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(kFullMask, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kFullMask, uint32_t(k >> 32));
  const uint32_t lo = __reduce_max_sync(kFullMask, uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
  return uint64_t(hi) << 32 | lo;
}

// The topk largest of the warp's keys in order; lane j returns the j-th's index
// (-1 when fewer are eligible).  `runs` topk + 1 rounds are made when `gaps` is
// asked for: true unless two neighbours lie within the keys' error of each other.
template <int NV, class K>
__device__ __forceinline__ int select_topk(const K (&key)[NV], int topk, bool* clear) {
  const int lane = threadIdx.x & 31;
  uint32_t taken = 0;  // of this lane's keys
  K best = 0;
  int best_i = 0;
  auto rescan = [&]() {
    best = 0;
    best_i = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!(taken >> i & 1u) && key[i] > best) {
        best = key[i];
        best_i = i;
      }
  };
  rescan();
  int mine = -1;
  K prev = 0;
  bool ok = true;
  const int rounds = clear != nullptr ? topk + 1 : topk;
  for (int j = 0; j < rounds; ++j) {
    const K top = warp_max_key(best);
    if (top == 0) break;
    if constexpr (sizeof(K) == 4) {
      if (clear != nullptr && j > 0) {
        const float a = unordered(prev), b = unordered(top);
        // scores are good to 1e-6, keys to that and two roundings; not clear for infinities
        ok = ok && a - b > 4e-6f + 4e-7f * fabsf(a);
      }
    }
    prev = top;
    if (j == topk) break;
    // the lowest index among equal keys: lane l's are 32 i + l
    const uint32_t e = best == top ? uint32_t(32 * best_i + lane) : 0xffffffffu;
    const uint32_t win = __reduce_min_sync(kFullMask, e);
    if (lane == j) mine = int(win);
    if (e == win) {
      taken |= 1u << best_i;
      rescan();
    }
  }
  if (clear != nullptr) *clear = ok;
  return mine;
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
  float scale;
};

// This lane's logits (experts 32 i + lane; -inf behind the last).
template <typename T, int NV>
__device__ __forceinline__ void load_logits(const T* row, int experts, float (&l)[NV]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 32 * i + lane;
    l[i] = e < experts ? to_f32<T>(row[e]) : kNegInf;
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

template <typename T, int NV, bool kSoftmax>
__global__ void __launch_bounds__(32 * kRouterWarps)
    router_kernel(const __grid_constant__ RouterParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.experts;
  float l[NV];
  load_logits<T, NV>(row, p.experts, l);
  bool nan = false;
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    nan = nan || l[i] != l[i];
    m = fmaxf(m, l[i]);
  }
  nan = __any_sync(kFullMask, nan);
  m = warp_max(m);
  if (kSoftmax && m == -kNegInf) nan = true;

  float total = 1.0f;  // softmax: sum of exp(l - m)
  if (kSoftmax && (p.bias != nullptr || !p.renorm)) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (l[i] > kNegInf) s += expf(l[i] - m);
    total = warp_sum(s);
  }

  uint32_t key[NV];
  int id;
  if (p.bias == nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = ordered(l[i]);
    id = select_topk<NV, uint32_t>(key, p.topk, nullptr);
  } else {
    float b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = 32 * i + lane;
      b[i] = e < p.experts ? __ldg(p.bias + e) : 0.0f;
      // a masked expert (-inf) stays out whatever its bias
      key[i] = 0u;
      if (l[i] > kNegInf)
        key[i] = ordered((kSoftmax ? expf(l[i] - m) / total : 1.0f / (1.0f + expf(-l[i]))) + b[i]);
    }
    bool clear;
    id = select_topk<NV, uint32_t>(key, p.topk, &clear);
    if (!clear) {
      uint64_t key64[NV];
      double s64 = 0.0;
      if (kSoftmax) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (l[i] > kNegInf) s64 += exp(double(l[i]) - double(m));
        s64 = warp_sum(s64);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        key64[i] = 0ull;
        if (l[i] > kNegInf)
          key64[i] = ordered((kSoftmax ? exp(double(l[i]) - double(m)) / s64
                                       : 1.0 / (1.0 + exp(-double(l[i])))) + double(b[i]));
      }
      id = select_topk<NV, uint64_t>(key64, p.topk, nullptr);
    }
  }

  // lane j: the weight of route j
  const float lj = id >= 0 ? to_f32<T>(row[id]) : kNegInf;
  const float mj = warp_max(lj);  // the largest chosen logit
  float w = 0.0f;
  if (p.renorm) {
    const float s = id >= 0 ? chosen_score<kSoftmax>(lj, mj) : 0.0f;
    const float sum = warp_sum(s);
    w = id >= 0 ? s / sum : 0.0f;
  } else if (id >= 0) {
    w = kSoftmax ? expf(lj - m) / total : chosen_score<false>(lj, 0.0f);
  }
  w *= p.scale;
  if (nan) w = __int_as_float(0x7fc00000);
  if (lane < p.topk) {
    p.ids[t * p.topk + lane] = id;
    p.weights[t * p.topk + lane] = w;
  }
}

// dlogits from dweights.  With c_j the share of route j,
//   softmax, normalised over the chosen   c_j = w_j (dw_j - sum_i dw_i w_i)
//   softmax                               c_j = s_j dw_j
//   sigmoid, normalised                   c_j = w_j (dw_j - sum_i dw_i w_i) (1 - s_j)
//   sigmoid                               c_j = dw_j s_j (1 - s_j)
// (w normalised, without the scale), dl_e = sum of c_j over the routes to e,
// minus s_e sum_j c_j for the whole softmax.
template <typename T, int NV, bool kSoftmax>
__global__ void __launch_bounds__(32 * kRouterWarps)
    router_backward_kernel(const __grid_constant__ RouterParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.experts;
  int id = -1;
  float dw = 0.0f;
  if (lane < p.topk) {
    id = p.ids[t * p.topk + lane];
    dw = p.dweights[t * p.topk + lane] * p.scale;
  }
  if (id < 0 || id >= p.experts) {  // an absent route
    id = -1;
    dw = 0.0f;
  }
  const float lj = id >= 0 ? to_f32<T>(row[id]) : kNegInf;
  float l[NV];
  float m = 0.0f, total = 1.0f, c = 0.0f, whole = 0.0f;
  const bool dense = kSoftmax && !p.renorm;  // every expert's logit has a gradient
  if (dense) {
    load_logits<T, NV>(row, p.experts, l);
    m = kNegInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, l[i]);
    m = warp_max(m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      l[i] = l[i] == kNegInf ? 0.0f : expf(l[i] - m);
      s += l[i];
    }
    total = warp_sum(s);
#pragma unroll
    for (int i = 0; i < NV; ++i) l[i] = total > 0.0f ? l[i] / total : l[i] + (total - total);
    c = id >= 0 && lj != kNegInf ? expf(lj - m) / total * dw : 0.0f;
    whole = warp_sum(c);
  } else if (p.renorm) {
    const float mj = warp_max(lj);
    const float s = id >= 0 && lj != kNegInf ? chosen_score<kSoftmax>(lj, mj) : 0.0f;
    const float sum = warp_sum(s);
    const float w = sum == 0.0f ? 0.0f : s / sum;
    const float dot = warp_sum(w * dw);
    c = w * (dw - dot);
    if (!kSoftmax && id >= 0) c *= lj >= 0.0f ? expf(-lj) / (1.0f + expf(-lj)) : 1.0f / (1.0f + expf(lj));
  } else if (id >= 0) {
    const float x = expf(-fabsf(lj));
    c = dw * (x / ((1.0f + x) * (1.0f + x)));
  }
  T* out = static_cast<T*>(p.dlogits) + t * p.experts;
  float d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) d[i] = dense ? -l[i] * whole : 0.0f;
  for (int j = 0; j < p.topk; ++j) {
    const int ij = __shfl_sync(kFullMask, id, j);
    const float cj = __shfl_sync(kFullMask, c, j);
    if (ij >= 0 && (ij & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == ij >> 5) d[i] += cj;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 32 * i + lane;
    if (e < p.experts) out[e] = from_f32<T>(d[i]);
  }
}

// Registers for 32, 64, 128, 256, 512 or 1024 experts.
template <typename T, bool kSoftmax, bool kBackward>
cudaError_t launch_router(const RouterParams& p, cudaStream_t s) {
  const int blocks = (p.tokens + kRouterWarps - 1) / kRouterWarps;
  const int v = (p.experts + 31) / 32;
  auto go = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    if constexpr (kBackward)
      router_backward_kernel<T, NV, kSoftmax><<<blocks, 32 * kRouterWarps, 0, s>>>(p);
    else
      router_kernel<T, NV, kSoftmax><<<blocks, 32 * kRouterWarps, 0, s>>>(p);
  };
  if (v <= 1) go(std::integral_constant<int, 1>());
  else if (v <= 2) go(std::integral_constant<int, 2>());
  else if (v <= 4) go(std::integral_constant<int, 4>());
  else if (v <= 8) go(std::integral_constant<int, 8>());
  else if (v <= 16) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 32>());
  return cudaGetLastError();
}

template <bool kBackward>
cudaError_t launch_router(const RouterParams& p, int dtype, bool softmax, cudaStream_t s) {
  if (dtype == 0)
    return softmax ? launch_router<float, true, kBackward>(p, s)
                   : launch_router<float, false, kBackward>(p, s);
  if (dtype == 1)
    return softmax ? launch_router<__nv_bfloat16, true, kBackward>(p, s)
                   : launch_router<__nv_bfloat16, false, kBackward>(p, s);
  return softmax ? launch_router<__half, true, kBackward>(p, s)
                 : launch_router<__half, false, kBackward>(p, s);
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
  p.scale = scale;
  FGG_CUDA_CHECK(launch_router<true>(p, dtype, score == 0, reinterpret_cast<cudaStream_t>(stream)));
  return FGG_OK;
}

}  // extern "C"
