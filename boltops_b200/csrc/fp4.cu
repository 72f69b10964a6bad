// Rows to microscaled 4-bit floats and back (fp4.cuh has the formulas).
//
// Bound by HBM: 2 (or 4) bytes a value in, 0.56 (NV) or 0.53 (MX) out.  A thread takes eight
// consecutive values, so a warp reads and writes whole lines; the two (NV) or four (MX) threads of a
// block exchange its largest magnitude.  Blocks never cross a row and all three arrays are dense,
// so the kernels see one flat array and divide by nothing.
#include "fp4.cuh"

namespace bolt {
namespace {
using namespace fp4;

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* src) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const Vec<T, 8> u = *reinterpret_cast<const Vec<T, 8>*>(src);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(u.v[i]);
  }
}

template <typename T, bool NV>
__global__ void __launch_bounds__(256) k_fp4_quant(const T* __restrict__ x, int64_t groups,
                                                   const float* __restrict__ g,
                                                   uint32_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales) {
  constexpr int kThreadsPerBlock = NV ? 2 : 4;
  const float inv_g = g != nullptr ? __frcp_rn(*g) : 1.f;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  // (whole warps run every pass: the exchange needs them)
  for (int64_t base = (int64_t)blockIdx.x * blockDim.x + (threadIdx.x & ~31); base < groups; base += stride) {
    const int64_t i = base + (threadIdx.x & 31);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i < groups) load8(v, x + 8 * i);
    if (NV && g != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv_g;
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = amax_nan(amax, v[j]);
#pragma unroll
    for (int o = 1; o < kThreadsPerBlock; o <<= 1)
      amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const uint32_t byte = scale_byte<NV>(amax);
    const uint32_t w = codes8<NV>(v, scaler_of<NV>(byte));
    if (i < groups) {
      codes[i] = w;
      if (i % kThreadsPerBlock == 0) scales[i / kThreadsPerBlock] = (uint8_t)byte;
    }
  }
}

template <typename T, bool NV>
__global__ void __launch_bounds__(256) k_fp4_dequant(const uint32_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, int64_t groups,
                                                     const float* __restrict__ g, T* __restrict__ out) {
  const float whole = g != nullptr ? *g : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < groups;
       i += (int64_t)gridDim.x * blockDim.x) {
    uint32_t h[4];
    halves8(codes[i], h);
    const float s = scale_value<NV>(scales[i / (NV ? 2 : 4)]);
    Vec<T, 8> r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      r.v[2 * j] = from_f32<T>(f.x * s * whole);       // (code * scale is exact)
      r.v[2 * j + 1] = from_f32<T>(f.y * s * whole);
    }
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out + 8 * i) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
      *reinterpret_cast<float4*>(out + 8 * i + 4) = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
    } else {
      *reinterpret_cast<uint4*>(out + 8 * i) = *reinterpret_cast<const uint4*>(&r);
    }
  }
}

int blocks_for(int64_t groups) {
  const int64_t want = (groups + 255) / 256, most = (int64_t)sm_count_of_current_device() * 16;
  return (int)(want < most ? want : most);
}

template <typename T>
int quant(const void* x, int64_t groups, bool nv, const float* g, void* codes, void* scales, cudaStream_t st) {
  const T* src = static_cast<const T*>(x);
  if (nv)
    k_fp4_quant<T, true><<<blocks_for(groups), 256, 0, st>>>(src, groups, g, static_cast<uint32_t*>(codes),
                                                             static_cast<uint8_t*>(scales));
  else
    k_fp4_quant<T, false><<<blocks_for(groups), 256, 0, st>>>(src, groups, g, static_cast<uint32_t*>(codes),
                                                              static_cast<uint8_t*>(scales));
  BOLT_LAUNCH_CHECK();
  return BOLT_OK;
}
template <typename T>
int dequant(const void* codes, const void* scales, int64_t groups, bool nv, const float* g, void* out,
            cudaStream_t st) {
  const uint32_t* c = static_cast<const uint32_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (nv) k_fp4_dequant<T, true><<<blocks_for(groups), 256, 0, st>>>(c, s, groups, g, static_cast<T*>(out));
  else k_fp4_dequant<T, false><<<blocks_for(groups), 256, 0, st>>>(c, s, groups, g, static_cast<T*>(out));
  BOLT_LAUNCH_CHECK();
  return BOLT_OK;
}

int check_sizes(const char* what, int64_t rows, int64_t cols, int format, const void* a, const void* b,
                const void* c, const void* g) {
  BOLT_REQUIRE(format == BOLT_FP4_NV || format == BOLT_FP4_MX, "%s: unknown format %d", what, format);
  const int block = format == BOLT_FP4_NV ? 16 : 32;
  BOLT_REQUIRE(rows >= 0 && cols >= 0 && cols % block == 0, "%s: %lld columns are not whole blocks of %d", what,
               (long long)cols, block);
  BOLT_REQUIRE(rows == 0 || cols == 0 || (a && b && c), "%s: null pointer", what);
  BOLT_REQUIRE(g == nullptr || format == BOLT_FP4_NV, "%s: MX has no scale of the whole tensor", what);
  return BOLT_OK;
}

}  // namespace
}  // namespace bolt

extern "C" int bolt_fp4_quant(const void* x, int dtype, int64_t rows, int64_t cols, int format,
                              const float* global_scale, void* codes, void* scales, void* stream) {
  using namespace bolt;
  const int rc = check_sizes("fp4_quant", rows, cols, format, x, codes, scales, global_scale);
  if (rc != BOLT_OK) return rc;
  if (rows * cols == 0) return BOLT_OK;
  BOLT_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0,
               "fp4_quant: operands must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t groups = rows * cols / 8;
  const bool nv = format == BOLT_FP4_NV;
  switch (dtype) {
    case BOLT_BF16: return quant<__nv_bfloat16>(x, groups, nv, global_scale, codes, scales, st);
    case BOLT_F16: return quant<__half>(x, groups, nv, global_scale, codes, scales, st);
    case BOLT_F32: return quant<float>(x, groups, nv, global_scale, codes, scales, st);
    default: set_error("fp4_quant: unsupported dtype %d", dtype); return BOLT_ERR_INVALID;
  }
}

extern "C" int bolt_fp4_dequant(const void* codes, const void* scales, int64_t rows, int64_t cols, int format,
                                const float* global_scale, void* out, int dtype, void* stream) {
  using namespace bolt;
  const int rc = check_sizes("fp4_dequant", rows, cols, format, codes, scales, out, global_scale);
  if (rc != BOLT_OK) return rc;
  if (rows * cols == 0) return BOLT_OK;
  BOLT_REQUIRE(reinterpret_cast<uintptr_t>(out) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0,
               "fp4_dequant: operands must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t groups = rows * cols / 8;
  const bool nv = format == BOLT_FP4_NV;
  switch (dtype) {
    case BOLT_BF16: return dequant<__nv_bfloat16>(codes, scales, groups, nv, global_scale, out, st);
    case BOLT_F16: return dequant<__half>(codes, scales, groups, nv, global_scale, out, st);
    case BOLT_F32: return dequant<float>(codes, scales, groups, nv, global_scale, out, st);
    default: set_error("fp4_dequant: unsupported dtype %d", dtype); return BOLT_ERR_INVALID;
  }
}
