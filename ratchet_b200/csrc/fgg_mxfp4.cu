// fgg_mxfp4.cu - MXFP4 quantisation on the device and its inverse.
//
// The format (OCP microscaling, E2M1 elements): 32 consecutive elements share a
// power-of-two scale, stored as an UE8M0 byte.
//   e    = floor(log2(max |x|)) - 2      (2: the exponent of E2M1's largest, 6)
//   byte = max(e + 127, 0)               (0 for a block of zeros)
//   q    = e2m1_rne(x 2^-e)              ties to the even code, saturating at 6
// A block that holds a NaN or an infinity has the NaN scale 0xFF, so that it
// reads back as NaN.  e comes from the exponent bits of the maximum, and x 2^-e
// is exact in fp32 but where it vanishes, so every step is exact up to the one
// rounding to E2M1.  The exact rounding of the value's 4 bits is the hardware's
// (cuda_fp4.h's conversion).
//
// Both kernels are HBM-bound copies: one pass, 16-byte loads, four lanes per
// 32-element block.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>

#include "fgg_host.cuh"
#include "fgg_ptx.cuh"

namespace fgg {
namespace {

// Eight consecutive values as fp32, and eight fp32 as values (16-byte aligned).
template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const uint4*>(p));
    b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y);
    v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y);
    v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <>
struct Vec8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    a = __ldg(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 o;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = o;
  }
};
template <>
struct Vec8<__half> {
  uint4 a;
  __device__ __forceinline__ void load(const __half* p) {
    a = __ldg(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__half* p, const float (&v)[8]) {
    uint4 o;
    __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = o;
  }
};

// E2M1 codes of eight values, the first in the lowest four bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w |= uint32_t(__nv_cvt_float2_to_fp4x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_E2M1,
                                           cudaRoundNearest))
         << (8 * i);
  return w;
}

// Two E2M1 values of a byte, the low half first.
__device__ __forceinline__ float2 e2m1x2_values(uint32_t byte) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(__nv_fp4x2_storage_t(byte), __NV_E2M1);
  return __half22float2(__half2(h));
}

// 2^(b - 127) for a scale byte b; NaN for 255.
__device__ __forceinline__ float ue8m0_value(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255u ? 0x7fc00000u : b << 23);
}

// Four lanes per 32-element block, eight elements each; a thread takes U such
// pieces, 256 threads apart, with all its loads in flight before the first use.
// U = 4 for tensors that fill the GPU with it: 16384 x 7168 bf16 take 50 us (5.9
// TB/s; back to bf16 45 us, 6.5 TB/s) where U = 1, 16 bytes per thread in flight,
// takes 65 (59); U = 1 below, where more blocks are what shortens the call.
template <typename T, int U>
__global__ void __launch_bounds__(256)
    mxfp4_quant_kernel(const T* __restrict__ x, int64_t blocks, uint8_t* __restrict__ codes,
                       uint8_t* __restrict__ sf) {
  const int64_t h0 = int64_t(blockIdx.x) * (256 * U) + threadIdx.x;  // first piece of 8 elements
  const int64_t pieces = 4 * blocks;
  Vec8<T> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + 256 * u < pieces) in[u].load(x + (h0 + 256 * u) * 8);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t h = h0 + 256 * u;
    const bool live = h < pieces;  // the same for a block's four lanes
    float v[8];
    uint32_t top = 0;
    if (live) {
      in[u].get(v);
      // magnitudes compare as integers, NaN above infinity above every number
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(kFullMask, top, 1));
    top = max(top, __shfl_xor_sync(kFullMask, top, 2));
    if (!live) continue;
    const uint32_t eb = top >> 23;  // exponent + 127; 255: NaN or infinity
    const uint32_t byte = eb == 255u ? 255u : (eb > 2u ? eb - 2u : 0u);
    const float inv = byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = byte == 255u ? 0.0f : v[i] * inv;
    __stcs(reinterpret_cast<uint32_t*>(codes) + h, e2m1x8(v));
    if ((h & 3) == 0) sf[h >> 2] = uint8_t(byte);
  }
}

template <typename T, int U>
__global__ void __launch_bounds__(256)
    mxfp4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf,
                         int64_t blocks, T* __restrict__ x) {
  const int64_t h0 = int64_t(blockIdx.x) * (256 * U) + threadIdx.x;
  const int64_t pieces = 4 * blocks;
  uint32_t w[U], b[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + 256 * u < pieces) {
      w[u] = __ldg(reinterpret_cast<const uint32_t*>(codes) + h0 + 256 * u);
      b[u] = __ldg(sf + ((h0 + 256 * u) >> 2));
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (h0 + 256 * u >= pieces) break;
    const float s = ue8m0_value(b[u]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e2m1x2_values(w[u] >> (8 * i) & 0xffu);
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    Vec8<T>::store(x + (h0 + 256 * u) * 8, v);
  }
}

// Pieces per thread: four once the tensor gives every SM a full set of threads
// with four each.
constexpr int kPieces = 4;
inline bool many_pieces(int64_t pieces, const DeviceInfo& dev) {
  return pieces >= int64_t(dev.sm_count) * 2048 * kPieces;
}

template <typename T>
void launch_quant(const void* x, int64_t blocks, void* codes, void* sf, const DeviceInfo& dev,
                  cudaStream_t s) {
  const int64_t pieces = 4 * blocks;
  const T* in = static_cast<const T*>(x);
  auto* c = static_cast<uint8_t*>(codes);
  auto* f = static_cast<uint8_t*>(sf);
  if (many_pieces(pieces, dev))
    mxfp4_quant_kernel<T, kPieces>
        <<<int((pieces + 256 * kPieces - 1) / (256 * kPieces)), 256, 0, s>>>(in, blocks, c, f);
  else
    mxfp4_quant_kernel<T, 1><<<int((pieces + 255) / 256), 256, 0, s>>>(in, blocks, c, f);
}

template <typename T>
void launch_dequant(const void* codes, const void* sf, int64_t blocks, void* x,
                    const DeviceInfo& dev, cudaStream_t s) {
  const int64_t pieces = 4 * blocks;
  const auto* c = static_cast<const uint8_t*>(codes);
  const auto* f = static_cast<const uint8_t*>(sf);
  T* out = static_cast<T*>(x);
  if (many_pieces(pieces, dev))
    mxfp4_dequant_kernel<T, kPieces>
        <<<int((pieces + 256 * kPieces - 1) / (256 * kPieces)), 256, 0, s>>>(c, f, blocks, out);
  else
    mxfp4_dequant_kernel<T, 1><<<int((pieces + 255) / 256), 256, 0, s>>>(c, f, blocks, out);
}

int check_mx(const void* x, int dtype, int64_t count, const void* codes, const void* sf) {
  if (dtype < 0 || dtype > 2)
    return set_error(FGG_EINVAL, "dtype=%d must be 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  if (count < 0 || count % 32 != 0)
    return set_error(FGG_EBADSHAPE, "the count of elements must be a multiple of 32");
  if (count > 0 && (x == nullptr || codes == nullptr || sf == nullptr))
    return set_error(FGG_EINVAL, "null pointer");
  if (!aligned16(x)) return set_error(FGG_EALIGN, "x must be 16-byte aligned");
  if (!aligned4(codes)) return set_error(FGG_EALIGN, "codes must be 4-byte aligned");
  if (count / 8 > int64_t(INT32_MAX) * 256) return set_error(FGG_EBADSHAPE, "tensor too large");
  return FGG_OK;
}

}  // namespace
}  // namespace fgg

using namespace fgg;

extern "C" {

int fgg_mxfp4_quantize(const void* x, int32_t x_dtype, int64_t count, void* codes, void* sf,
                       void* stream) {
  if (int rc = check_mx(x, x_dtype, count, codes, sf)) return rc;
  if (count == 0) return FGG_OK;
  DeviceInfo dev;
  if (int rc = current_device(&dev)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == 0)
    launch_quant<float>(x, count / 32, codes, sf, dev, s);
  else if (x_dtype == 1)
    launch_quant<__nv_bfloat16>(x, count / 32, codes, sf, dev, s);
  else
    launch_quant<__half>(x, count / 32, codes, sf, dev, s);
  FGG_CUDA_CHECK(cudaGetLastError());
  return FGG_OK;
}

int fgg_mxfp4_dequantize(const void* codes, const void* sf, int64_t count, void* x, int32_t x_dtype,
                         void* stream) {
  if (int rc = check_mx(x, x_dtype, count, codes, sf)) return rc;
  if (count == 0) return FGG_OK;
  DeviceInfo dev;
  if (int rc = current_device(&dev)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == 0)
    launch_dequant<float>(codes, sf, count / 32, x, dev, s);
  else if (x_dtype == 1)
    launch_dequant<__nv_bfloat16>(codes, sf, count / 32, x, dev, s);
  else
    launch_dequant<__half>(codes, sf, count / 32, x, dev, s);
  FGG_CUDA_CHECK(cudaGetLastError());
  return FGG_OK;
}

}  // extern "C"
