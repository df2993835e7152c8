// Shared by the operators that work on a caller's stream (dpc_vocab.cu, dpc_norm.cu, dpc_pack.cu):
// the two tensor types, and the guard and checks of their C entries.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "dpc_internal.h"
#include "dpc_tcgen05.cuh"

namespace dpc
{
namespace ops
{
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v)
{
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v)
{
  return __float2bfloat16_rn(v);
}

// Eight values to and from bf16 in 16 bytes.
__device__ __forceinline__ uint4 pack8(const float* v)
{
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
  {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    r[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ void unpack8(const uint4& p, float* v)
{
  const uint32_t r[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
  {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  }
}

// Eight neighbours in one or two 16-byte accesses.
__device__ __forceinline__ void load8w(const float* p, float* v)
{
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8w(const __nv_bfloat16* p, float* v)
{
  unpack8(__ldg(reinterpret_cast<const uint4*>(p)), v);
}
__device__ __forceinline__ void store8w(float* p, const float* v)
{
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8w(__nv_bfloat16* p, const float* v) { *reinterpret_cast<uint4*>(p) = pack8(v); }

// Two 32-bit floats in a register pair and the instructions that work on both at once: half the issue slots of
// kernels whose arithmetic, not only their traffic, is near the limit.
typedef unsigned long long float2x;
__device__ __forceinline__ float2x pair(float a, float b)
{
  float2x r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2x pair(float a) { return pair(a, a); }
__device__ __forceinline__ float2 halves(float2x v)
{
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2x fma2(float2x a, float2x b, float2x c)
{
  float2x r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float2x mul2(float2x a, float2x b)
{
  float2x r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float2x add2(float2x a, float2x b)
{
  float2x r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float2x pair_of_bf16(uint32_t v)
{
  return pair(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint32_t bf16_of_pair(float2x v)
{
  const float2 f = halves(v);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, NULL where there is none.
inline EncodeTiledFn encode_fn()
{
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  return fn;
}

// What dpc_operators_set_wait_limit said last on this host thread.
struct Waits
{
  double milliseconds = 0.0;
  bool keep_back = false;
};
inline thread_local Waits waits;

// The limit of a call's device-side waits in cycles of the fastest clock, so that it is never shorter than asked.
inline int wait_limit_now(long long* cycles)
{
  *cycles = ptx::kWaitCyclesDefault;
  if (waits.milliseconds > 0.0)
  {
    int device = 0, khz = 0;
    DPC_CUDA(cudaGetDevice(&device));
    DPC_CUDA(cudaDeviceGetAttribute(&khz, cudaDevAttrClockRate, device));
    *cycles = (long long)(waits.milliseconds * khz) + 1;
  }
  return DPC_OK;
}

inline int launched(const char* what)
{
  const cudaError_t err = cudaPeekAtLastError();
  return err == cudaSuccess ? (int)DPC_OK : cuda_fail(cudaGetLastError(), what);
}

// No C++ exception leaves a C entry.
template <typename F>
int guarded(const char* who, F f)
{
  try
  {
    return f();
  }
  catch (const std::exception& e)
  {
    return fail(DPC_ERR_CUDA, std::string(who) + ": " + e.what());
  }
  catch (...)
  {
    return fail(DPC_ERR_CUDA, std::string(who) + ": unknown exception");
  }
}
} // namespace ops
} // namespace dpc
