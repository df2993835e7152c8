// Activations kept in 8 bits for the backward pass.
//
// A layer's gradient needs f'(x) and, for the weights of the layer after it, f(x): both come from x, so x is all
// that has to be kept.  Forward writes out = f(x) and x as whole numbers of -127..127 with one 32-bit scale
// for 128 neighbours of a row (1.03 bytes an element instead of 2 or 4); backward reads them and writes
// d_preact = d_out f'(x) and, on request, f(x) again.  |x - code * scale| <= max|x| of the block / 254.
//
// Bound by memory.  16 threads share a block, 8 elements each: 16 bytes a load of bf16, the block's maximum by four
// shuffles within the half warp, and nothing is read twice.  The code is x * (127 / max) rounded to even: one
// division a block instead of one an element, and a product whose rounding is that of 32-bit arithmetic everywhere.
// The function itself is the layers' own (dpc_math.cuh).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "dpc_internal.h"
#include "dpc_math.cuh"
#include "dpc_operators.cuh"

namespace
{
using namespace dpc::ops;

constexpr int kBlock = 128;  // elements of a row that share a scale
constexpr int kShare = 16;   // threads of a block
constexpr int kThreads = 256;

// Column of a thread's element i of the block that starts at `first`.  WIDE: 8 neighbours a thread.
template <bool WIDE>
__device__ __forceinline__ int64_t column(int64_t first, int part, int i)
{
  return WIDE ? first + part * 8 + i : first + part + kShare * i;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* row, int64_t first, int part, int64_t width, float (&v)[8])
{
  if constexpr (WIDE)
  {
    const int64_t c = column<true>(first, part, 0);
    if (c < width)
      load8w(row + c, v);
    else
    {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = 0.0f;
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
      const int64_t c = column<false>(first, part, i);
      v[i] = c < width ? to_float(row[c]) : 0.0f;
    }
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store8(T* row, int64_t first, int part, int64_t width, const float (&v)[8])
{
  if constexpr (WIDE)
  {
    const int64_t c = column<true>(first, part, 0);
    if (c < width)
      store8w(row + c, v);
  }
  else
  {
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
      const int64_t c = column<false>(first, part, i);
      if (c < width)
        row[c] = from_float<T>(v[i]);
    }
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) activate_and_pack_kernel(const T* __restrict__ x, int64_t x_ld, int64_t rows,
                                                                     int64_t width, int64_t blocks, int act,
                                                                     T* __restrict__ out, int64_t out_ld,
                                                                     int8_t* __restrict__ codes, float* __restrict__ scales)
{
  const int part = threadIdx.x & (kShare - 1);
  const int64_t total = rows * blocks, step = (int64_t)gridDim.x * (kThreads / kShare);
  // (all 32 lanes of a warp stay in the loop together: the shuffles name the whole warp)
  for (int64_t base = (int64_t)blockIdx.x * (kThreads / kShare) + (threadIdx.x / 32) * 2; base < total; base += step)
  {
    const int64_t b = base + ((threadIdx.x >> 4) & 1);
    const bool inside = b < total;
    const int64_t row = inside ? b / blocks : 0, first = inside ? (b - row * blocks) * kBlock : width;
    float v[8], f[8], d[8];
    load8<T, WIDE>(x + row * x_ld, first, part, width, v);
    // The magnitudes compare like their bit patterns, infinities and NaN above all numbers.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
      const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu;
      most = bits > most ? bits : most;
    }
#pragma unroll
    for (int o = kShare / 2; o > 0; o >>= 1)
    {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, most, o);
      most = other > most ? other : most;
    }
    if (!inside)
      continue;
    const float top = __uint_as_float(most);
    const bool finite = most < 0x7f800000u, some = finite && top >= 7.888609052210118e-31f; // 2^-100
    const float factor = some ? __fdiv_rn(127.0f, top) : 0.0f;
    int8_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = some ? (int8_t)__float2int_rn(v[i] * factor) : (int8_t)0;
    int8_t* to = codes + row * width;
    if (WIDE)
    {
      const int64_t c = column<true>(first, part, 0);
      if (c < width)
        *reinterpret_cast<uint2*>(to + c) = *reinterpret_cast<const uint2*>(q);
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 8; ++i)
      {
        const int64_t c = column<false>(first, part, i);
        if (c < width)
          to[c] = q[i];
      }
    }
    if (part == 0)
      scales[b] = !finite ? __uint_as_float(0x7fc00000u) : some ? __fdiv_rn(top, 127.0f) : 0.0f;
    if (out)
    {
      dpc::act_many<false>(act, v, f, d);
      store8<T, WIDE>(out + row * out_ld, first, part, width, f);
    }
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
    packed_backward_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows, int64_t width,
                           int64_t blocks, int act, const T* __restrict__ d_out, int64_t d_out_ld,
                           T* __restrict__ d_preact, int64_t d_preact_ld, T* __restrict__ out, int64_t out_ld)
{
  const int part = threadIdx.x & (kShare - 1);
  const int64_t total = rows * blocks, step = (int64_t)gridDim.x * (kThreads / kShare);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / kShare) + threadIdx.x / kShare; b < total; b += step)
  {
    const int64_t row = b / blocks, first = (b - row * blocks) * kBlock;
    const int8_t* from = codes + row * width;
    const float scale = __ldg(scales + b);
    float g[8], v[8], f[8], d[8];
    if (d_out)
      load8<T, WIDE>(d_out + row * d_out_ld, first, part, width, g);
    if (WIDE)
    {
      const int64_t c = column<true>(first, part, 0);
      uint2 packed = make_uint2(0, 0);
      if (c < width)
        packed = __ldg(reinterpret_cast<const uint2*>(from + c));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = scale * (float)(int8_t)((i < 4 ? packed.x : packed.y) >> (8 * (i & 3)));
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 8; ++i)
      {
        const int64_t c = column<false>(first, part, i);
        v[i] = c < width ? scale * (float)from[c] : 0.0f;
      }
    }
    dpc::act_many<true>(act, v, f, d);
    if (d_out)
    {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        g[i] *= d[i];
      // (piecewise functions have a slope even at NaN: a block that held one has a NaN here too)
      if (scale != scale)
      {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          g[i] = scale;
      }
      store8<T, WIDE>(d_preact + row * d_preact_ld, first, part, width, g);
    }
    if (out)
    {
      if (scale != scale)
      {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          f[i] = scale;
      }
      store8<T, WIDE>(out + row * out_ld, first, part, width, f);
    }
  }
}

// ------------------------------------------------------------------------------ host
int check(const std::string& who, int type, int act, int64_t rows, int64_t width)
{
  if (type != DPC_TYPE_F32 && type != DPC_TYPE_BF16)
    return dpc::fail(DPC_ERR_INVALID, who + ": type is neither DPC_TYPE_F32 nor DPC_TYPE_BF16");
  if (act < DPC_ACT_RELU || act > DPC_ACT_HARD_TANH || act % 2)
    return dpc::fail(DPC_ERR_INVALID, who + ": unknown activation");
  if (rows < 0 || width < 1)
    return dpc::fail(DPC_ERR_INVALID, who + ": rows >= 0 and width >= 1 are needed");
  if (rows > (int64_t)1 << 31 || width > (int64_t)1 << 31)
    return dpc::fail(DPC_ERR_TOO_LARGE, who + ": rows and width may be 2^31 at most");
  return DPC_OK;
}

bool stride_ok(const void* p, int64_t stride, int64_t width) { return !p || (stride >= width && stride <= (int64_t)1 << 40); }

bool wide(int type, const void* p, int64_t stride)
{
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % (type == DPC_TYPE_F32 ? 4 : 8) == 0);
}

// Blocks of the launch: 8 of 256 threads on every SM, each with a few rounds of work where there is enough.
unsigned grid_for(int64_t blocks)
{
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((blocks + 15) / 16, 148 * 8 * 4));
}

template <typename T>
void launch_pack(cudaStream_t stream, bool w, int act, int64_t rows, int64_t width, const void* x, int64_t x_ld, void* out,
                 int64_t out_ld, int8_t* codes, float* scales)
{
  const int64_t blocks = (width + kBlock - 1) / kBlock;
  const unsigned grid = grid_for(rows * blocks);
  const T* in = static_cast<const T*>(x);
  T* to = static_cast<T*>(out);
  if (w)
    activate_and_pack_kernel<T, true><<<grid, kThreads, 0, stream>>>(in, x_ld, rows, width, blocks, act, to, out_ld, codes, scales);
  else
    activate_and_pack_kernel<T, false><<<grid, kThreads, 0, stream>>>(in, x_ld, rows, width, blocks, act, to, out_ld, codes, scales);
}

template <typename T>
void launch_backward(cudaStream_t stream, bool w, int act, int64_t rows, int64_t width, const int8_t* codes,
                     const float* scales, const void* d_out, int64_t d_out_ld, void* d_preact, int64_t d_preact_ld,
                     void* out, int64_t out_ld)
{
  const int64_t blocks = (width + kBlock - 1) / kBlock;
  const unsigned grid = grid_for(rows * blocks);
  const T* g = static_cast<const T*>(d_out);
  T *dx = static_cast<T*>(d_preact), *to = static_cast<T*>(out);
  if (w)
    packed_backward_kernel<T, true><<<grid, kThreads, 0, stream>>>(codes, scales, rows, width, blocks, act, g, d_out_ld, dx, d_preact_ld, to, out_ld);
  else
    packed_backward_kernel<T, false><<<grid, kThreads, 0, stream>>>(codes, scales, rows, width, blocks, act, g, d_out_ld, dx, d_preact_ld, to, out_ld);
}
} // namespace

int dpc_activate_and_pack(void* stream, int type, int act, int64_t rows, int64_t width, const void* x, int64_t x_stride,
                          void* out, int64_t out_stride, int8_t* codes, float* scales)
{
  return guarded("dpc_activate_and_pack", [&] {
    const std::string who = "dpc_activate_and_pack";
    if (int rc = check(who, type, act, rows, width))
      return rc;
    if (rows == 0)
      return (int)DPC_OK;
    if (!x || !codes || !scales)
      return dpc::fail(DPC_ERR_INVALID, who + ": null pointer");
    if (!stride_ok(x, x_stride, width) || !stride_ok(out, out_stride, width))
      return dpc::fail(DPC_ERR_INVALID, who + ": a row stride is smaller than the width (or above 2^40)");
    const bool w = width % 8 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0 && wide(type, x, x_stride) &&
                   wide(type, out, out_stride);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == DPC_TYPE_F32)
      launch_pack<float>(st, w, act, rows, width, x, x_stride, out, out_stride, codes, scales);
    else
      launch_pack<__nv_bfloat16>(st, w, act, rows, width, x, x_stride, out, out_stride, codes, scales);
    return launched("activate_and_pack_kernel");
  });
}

int dpc_packed_activation_backward(void* stream, int type, int act, int64_t rows, int64_t width, const int8_t* codes,
                                   const float* scales, const void* d_out, int64_t d_out_stride, void* d_preact,
                                   int64_t d_preact_stride, void* out, int64_t out_stride)
{
  return guarded("dpc_packed_activation_backward", [&] {
    const std::string who = "dpc_packed_activation_backward";
    if (int rc = check(who, type, act, rows, width))
      return rc;
    if (rows == 0)
      return (int)DPC_OK;
    if (!codes || !scales || !d_out != !d_preact || (!d_out && !out))
      return dpc::fail(DPC_ERR_INVALID, who + ": null pointer");
    if (!stride_ok(d_out, d_out_stride, width) || !stride_ok(d_preact, d_preact_stride, width) ||
        !stride_ok(out, out_stride, width))
      return dpc::fail(DPC_ERR_INVALID, who + ": a row stride is smaller than the width (or above 2^40)");
    const bool w = width % 8 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0 && wide(type, d_out, d_out_stride) &&
                   wide(type, d_preact, d_preact_stride) && wide(type, out, out_stride);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == DPC_TYPE_F32)
      launch_backward<float>(st, w, act, rows, width, codes, scales, d_out, d_out_stride, d_preact, d_preact_stride, out, out_stride);
    else
      launch_backward<__nv_bfloat16>(st, w, act, rows, width, codes, scales, d_out, d_out_stride, d_preact, d_preact_stride, out, out_stride);
    return launched("packed_backward_kernel");
  });
}
