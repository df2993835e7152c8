// Activations kept in 8 bits for the backward pass.
//
// A layer's gradient needs f'(x) and, for the weights of the layer after it, f(x): both come from x, so x is all
// that has to be kept.  Forward writes out = f(x) and x as whole numbers of -127..127 with one 32-bit scale
// for 128 neighbours of a row (1.03 bytes an element instead of 2 or 4); backward reads them and writes
// d_preact = d_out f'(x) and, on request, f(x) again.  |x - code * scale| <= max|x| of the block / 254, but for blocks
// with nothing of 2^-100 or larger, which are zeros.
//
// Bound by memory.  8 threads share a block, 16 elements each, the block's maximum by three shuffles, and nothing is read
// twice; a thread reads its next part before it works on this one, in 32-byte accesses.  The code is x * (127 / max)
// rounded to even: one division a block instead of one an element, and a product whose rounding is that of 32-bit
// arithmetic everywhere.  16384 x 8192 bf16, gelu: forward 116 us (671 MB, 103 us at the rate of a copy), backward
// with f(x) 149 us (940 MB, 144), values alone 67 us (403 MB, 62).  16-byte accesses and conversions by the conversion
// unit: 187, 231 and 107.
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
constexpr int kThreads = 256;

// Threads that share a block and the elements of it that each holds: 16 neighbours where pointers, strides and the
// width allow 32-byte accesses (WIDE), else 4 that are 32 apart, so that neighbouring threads have neighbours.
template <bool WIDE>
struct Split
{
  static constexpr int kShare = WIDE ? 8 : 32, kEach = kBlock / kShare;
  static constexpr int kGroups = kThreads / kShare;
  static constexpr int kWork = WIDE ? 8 : 4; // elements at a time: registers for more would cost threads
  static __device__ __forceinline__ int64_t column(int64_t first, int part, int i)
  {
    return WIDE ? first + part * kEach + i : first + part + kShare * i;
  }
};

// 32 bytes in one access: whole sectors also where a thread's neighbours come in two halves.
__device__ __forceinline__ void load32(const void* p, uint32_t* r)
{
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* r)
{
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// A thread's part of a block as it lies in memory: read a round ahead of its use, or written when it is complete.
template <typename T, bool WIDE>
struct Cells
{
  static constexpr int kWords = WIDE ? 4 * (int)sizeof(T) : 4; // 16 elements, or 4 in 32 bits each
  uint32_t word[kWords];
  __device__ __forceinline__ void fetch(const T* row, int64_t first, int part, int64_t width)
  {
    if constexpr (WIDE)
    {
      const int64_t c = Split<WIDE>::column(first, part, 0);
      if (c < width) // (all or nothing)
      {
#pragma unroll
        for (int i = 0; i < kWords; i += 8)
          load32(reinterpret_cast<const uint32_t*>(row + c) + i, word + i);
      }
      else
      {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
          word[i] = 0;
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const int64_t c = Split<WIDE>::column(first, part, i);
        word[i] = __float_as_uint(c < width ? to_float(row[c]) : 0.0f);
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int64_t first, int part, int64_t width) const
  {
    if constexpr (WIDE)
    {
      const int64_t c = Split<WIDE>::column(first, part, 0);
      if (c < width)
      {
#pragma unroll
        for (int i = 0; i < kWords; i += 8)
          store32(reinterpret_cast<uint32_t*>(row + c) + i, word + i);
      }
    }
    else
    {
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const int64_t c = Split<WIDE>::column(first, part, i);
        if (c < width)
          row[c] = from_float<T>(__uint_as_float(word[i]));
      }
    }
  }
  // elements [8 h, 8 h + 8), or all 4
  template <int N>
  __device__ __forceinline__ void get(int h, float (&v)[N]) const
  {
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
      if constexpr (WIDE && sizeof(T) == 2)
        v[i] = __uint_as_float(i & 1 ? word[4 * h + i / 2] & 0xffff0000u : word[4 * h + i / 2] << 16);
      else
        v[i] = __uint_as_float(word[N * h + i]);
    }
  }
  template <int N>
  __device__ __forceinline__ void set(int h, const float (&v)[N])
  {
    if constexpr (WIDE && sizeof(T) == 2)
    {
#pragma unroll
      for (int i = 0; i < N; i += 2)
        word[4 * h + i / 2] = bf16_of_pair(pair(v[i], v[i + 1]));
    }
    else
    {
#pragma unroll
      for (int i = 0; i < N; ++i)
        word[N * h + i] = __float_as_uint(v[i]);
    }
  }
};

// gelu(x) = x h, h = 1 / (1 + exp(-2 u)), u = sqrt(2/pi) (x + 0.044715 x^3): the layers' 0.5 x (1 + tanh(u)) with two
// thirds of its operations, and other last bits; its slope is h + x h (1 - h) (2u)'.  Where exp overflows h is 0; x^2 stops short of
// infinity, which times that 0 would be NaN.
template <bool SLOPE, int N>
__device__ __forceinline__ void gelu_many(const float (&v)[N], float (&f)[N], float (&d)[N])
{
  constexpr float k1 = dpc::kGelu1, k2 = dpc::kGelu1 * dpc::kGelu2, log2e = 1.4426950408889634f;
#pragma unroll
  for (int i = 0; i < N; i += 2)
  {
    const float2x x = pair(v[i], v[i + 1]);
    float2x sq = mul2(x, x);
    const float2 e = halves(mul2(x, fma2(pair(-2.0f * k2 * log2e), sq, pair(-2.0f * k1 * log2e))));
    float a, b;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(e.y));
    const float2 under = halves(add2(pair(a, b), pair(1.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(under.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(under.y));
    const float2x h = pair(a, b), y = mul2(x, h);
    const float2 o = halves(y);
    f[i] = o.x, f[i + 1] = o.y;
    if (SLOPE)
    {
      const float2 s = halves(sq);
      sq = pair(fminf(s.x, 1e30f), fminf(s.y, 1e30f));
      const float2 g = halves(fma2(fma2(y, mul2(h, pair(-1.0f)), y), fma2(pair(6.0f * k2), sq, pair(2.0f * k1)), h));
      d[i] = g.x, d[i + 1] = g.y;
    }
  }
}

// tanh with an error relative to its value, since small outputs go into tensors and into the next layer's weight gradient:
// the layers' 1 - 2 / (exp(2x) + 1) cancels near 0 (0.1 % off at 1e-4, 5 % at 1e-6).  (1 - e) / (1 + e), e = exp(-2x), is
// good from a border on, below which an odd polynomial is taken; the slope is 4 e / (1 + e)^2 or 1 - tanh^2.  32-bit tensors:
// border 1/2, least squares in x^2 of (tanh(x) / x - 1) / x^2 at Chebyshev nodes (4e-10 off), 2^-20 in all.  bf16, which
// rounds by 2^-8: border 1/16 and the first two terms of the series (2 x^4 / 15 off), 2^-17 in all, since 16384 x 8192 elements in
// bf16 wait for instructions (forward 118 us with the layers' form, some 145 with the long polynomial, 133 with this one; float32 183
// with either).
template <typename T, bool SLOPE, int N>
__device__ __forceinline__ void tanh_many(const float (&v)[N], float (&f)[N], float (&d)[N])
{
  constexpr float log2e = 1.4426950408889634f, border = sizeof(T) == 4 ? 0.5f : 0.0625f;
#pragma unroll
  for (int i = 0; i < N; i += 2)
  {
    const float2x x = pair(v[i], v[i + 1]), sq = mul2(x, x);
    float2x poly = pair(-3.3333334e-1f);
    if constexpr (sizeof(T) == 4)
    {
      poly = fma2(pair(-6.6455984e-3f), sq, pair(2.1296676e-2f));
      poly = fma2(poly, sq, pair(-5.3898863e-2f));
      poly = fma2(poly, sq, pair(1.3332961e-1f));
      poly = fma2(poly, sq, pair(-3.3333325e-1f));
    }
    const float2 low = halves(fma2(mul2(x, sq), poly, x));
    // (2^125 at most, so that 1 - e is finite and 1 / (1 + e) not 0; a NaN stays one)
    const float2 at = halves(mul2(x, pair(-2.0f * log2e)));
    float a, b, ra, rb;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(at.x), "f"(125.0f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(at.y), "f"(125.0f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(a));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(b));
    const float2x e = pair(a, b);
    const float2 under = halves(add2(e, pair(1.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ra) : "f"(under.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rb) : "f"(under.y));
    const float2x r = pair(ra, rb);
    const float2 high = halves(mul2(fma2(e, pair(-1.0f), pair(1.0f)), r));
    const bool near_a = fabsf(v[i]) < border, near_b = fabsf(v[i + 1]) < border;
    f[i] = near_a ? low.x : high.x, f[i + 1] = near_b ? low.y : high.y;
    if (SLOPE)
    {
      const float2 far = halves(mul2(mul2(mul2(e, r), r), pair(4.0f)));
      d[i] = near_a ? fmaf(-low.x, low.x, 1.0f) : far.x, d[i + 1] = near_b ? fmaf(-low.y, low.y, 1.0f) : far.y;
    }
  }
}

// The layers' 1/2 + x / (2 (1 + |x|)) with h = 1 / (2 (1 + |x|)): h on the left and 1 - h on the right of 0, slope 2 h^2.  Their
// sum cancels on the left (6e-4 off at -1e4).
template <bool SLOPE, int N>
__device__ __forceinline__ void esigmoid_many(const float (&v)[N], float (&f)[N], float (&d)[N])
{
#pragma unroll
  for (int i = 0; i < N; ++i)
  {
    float h;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(1.0f + fabsf(v[i])));
    h *= 0.5f;
    f[i] = v[i] < 0.0f ? h : 1.0f - h;
    d[i] = 2.0f * h * h;
  }
}

template <typename T, bool SLOPE, int N>
__device__ __forceinline__ void activate(int act, const float (&v)[N], float (&f)[N], float (&d)[N])
{
  if (act == DPC_ACT_GELU)
    gelu_many<SLOPE>(v, f, d);
  else if (act == DPC_ACT_TANH)
    tanh_many<T, SLOPE>(v, f, d);
  else if (act == DPC_ACT_ESIGMOID)
    esigmoid_many<SLOPE>(v, f, d);
  else
    dpc::act_many<SLOPE>(act, v, f, d);
}

// Whole numbers in the low byte of a float: 1.5 * 2^23 is added, which rounds to even.  (Conversions run at an
// eighth of the rate of additions.)
constexpr float kMagic = 12582912.0f;

// Position of a group of threads among the blocks of all rows, advanced without divisions.
struct Place
{
  int64_t row, block, step_row, step_block, blocks;
  __device__ __forceinline__ Place(int64_t at, int64_t step, int64_t blocks_)
      : row(at / blocks_), block(at % blocks_), step_row(step / blocks_), step_block(step % blocks_), blocks(blocks_)
  {
  }
  __device__ __forceinline__ void next()
  {
    row += step_row, block += step_block;
    if (block >= blocks)
      block -= blocks, ++row;
  }
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3)
    activate_and_pack_kernel(const T* __restrict__ x, int64_t x_ld, int64_t rows, int64_t width, int64_t blocks, int act,
                             T* __restrict__ out, int64_t out_ld, int8_t* __restrict__ codes, float* __restrict__ scales)
{
  using S = Split<WIDE>;
  constexpr int N = S::kWork, kHalves = S::kEach / N;
  const int part = threadIdx.x & (S::kShare - 1);
  Place at((int64_t)blockIdx.x * S::kGroups + threadIdx.x / S::kShare, (int64_t)gridDim.x * S::kGroups, blocks);
  Cells<T, WIDE> next;
  auto fetch = [&] {
    const bool inside = at.row < rows;
    next.fetch(x + (inside ? at.row * x_ld : 0), at.block * kBlock, part, inside ? width : 0);
  };
  fetch();
  // (all 32 lanes of a warp stay in the loop together: the shuffles name the whole warp)
  while (__any_sync(0xffffffffu, at.row < rows))
  {
    const Cells<T, WIDE> now = next;
    const int64_t row = at.row, block = at.block, first = block * kBlock;
    at.next();
    fetch();
    // The magnitudes compare like their bit patterns, infinities and NaN above all numbers.
    uint32_t most = 0;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
    {
      float v[N];
      now.get(h, v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = S::kShare / 2; o > 0; o >>= 1)
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (row >= rows)
      continue;
    const float top = __uint_as_float(most);
    const bool finite = most < 0x7f800000u, some = finite && top >= 7.888609052210118e-31f; // 2^-100
    const float factor = __fdiv_rn(127.0f, some ? top : 1.0f);
    if (part == 0)
      scales[row * blocks + block] = !finite ? __uint_as_float(0x7fc00000u) : some ? __fdiv_rn(top, 127.0f) : 0.0f;
    uint32_t bytes[4];
    Cells<T, WIDE> result;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
    {
      float v[N];
      uint32_t q[N];
      now.get(h, v);
      // (a product rounded by itself, then to a whole number: one fused operation would round some ties otherwise,
      // and the instructions for pairs were fused)
#pragma unroll
      for (int i = 0; i < N; ++i)
        q[i] = some ? __float_as_uint(__fadd_rn(__fmul_rn(v[i], factor), kMagic)) : 0u;
      if constexpr (WIDE)
      {
#pragma unroll
        for (int i = 0; i < N; i += 4)
          bytes[(h * N + i) / 4] = __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
      }
      else
      {
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
          const int64_t c = S::column(first, part, i);
          if (c < width)
            codes[row * width + c] = (int8_t)(q[i] & 0xffu);
        }
      }
      if (out)
      {
        float f[N], d[N];
        activate<T, false>(act, v, f, d);
        result.set(h, f);
      }
    }
    if (out)
      result.store(out + row * out_ld, first, part, width);
    if constexpr (WIDE)
    {
      const int64_t c = S::column(first, part, 0);
      if (c < width)
        *reinterpret_cast<uint4*>(codes + row * width + c) = make_uint4(bytes[0], bytes[1], bytes[2], bytes[3]);
    }
  }
}

// SLOPE: d_preact (and out where it is wanted); otherwise out alone, with fewer registers and so more loads under way.
template <typename T, bool WIDE, bool SLOPE>
__global__ void __launch_bounds__(kThreads, (SLOPE ? 3 : 5) - (sizeof(T) == 4))
    packed_backward_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows, int64_t width,
                           int64_t blocks, int act, const T* __restrict__ d_out, int64_t d_out_ld,
                           T* __restrict__ d_preact, int64_t d_preact_ld, T* __restrict__ out, int64_t out_ld)
{
  using S = Split<WIDE>;
  constexpr int N = S::kWork, kHalves = S::kEach / N;
  const int part = threadIdx.x & (S::kShare - 1);
  Place at((int64_t)blockIdx.x * S::kGroups + threadIdx.x / S::kShare, (int64_t)gridDim.x * S::kGroups, blocks);
  Cells<T, WIDE> next;
  uint4 next_codes = make_uint4(0, 0, 0, 0); // 16 codes, or 4
  float next_scale = 0.0f;
  auto fetch = [&] {
    if (at.row >= rows)
      return;
    const int64_t first = at.block * kBlock;
    const int8_t* from = codes + at.row * width;
    next_scale = __ldg(scales + at.row * blocks + at.block);
    if (SLOPE)
      next.fetch(d_out + at.row * d_out_ld, first, part, width);
    if constexpr (WIDE)
    {
      const int64_t c = S::column(first, part, 0);
      if (c < width)
        next_codes = __ldg(reinterpret_cast<const uint4*>(from + c));
    }
    else
    {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
      {
        const int64_t c = S::column(first, part, i);
        r[i] = c < width ? (uint8_t)from[c] : 0u;
      }
      next_codes = make_uint4(r[0], r[1], r[2], r[3]);
    }
  };
  fetch();
  while (at.row < rows)
  {
    const Cells<T, WIDE> now = next;
    const uint32_t packed[4] = {next_codes.x, next_codes.y, next_codes.z, next_codes.w};
    const float scale = next_scale;
    const int64_t row = at.row, first = at.block * kBlock;
    at.next();
    fetch();
    // (piecewise functions have a value and a slope even at NaN: a block that held one is NaN here too)
    const bool bad = scale != scale;
    Cells<T, WIDE> slope, result;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
    {
      float v[N], f[N], d[N];
      // 2^23 + (code + 128) as the bits of a float, less 2^23 + 128
#pragma unroll
      for (int i = 0; i < N; i += 2)
      {
        const uint32_t lo = packed[WIDE ? (h * N + i) / 4 : i] ^ 0x80808080u;
        const uint32_t hi = WIDE ? lo : packed[WIDE ? 0 : i + 1] ^ 0x80808080u;
        const float2x x = pair(__uint_as_float(__byte_perm(lo, 0x4b000000u, 0x7540 | (WIDE ? i & 3 : 0))),
                               __uint_as_float(__byte_perm(hi, 0x4b000000u, 0x7540 | (WIDE ? (i + 1) & 3 : 0))));
        const float2 w = halves(mul2(add2(x, pair(-8388736.0f)), pair(scale)));
        v[i] = w.x, v[i + 1] = w.y;
      }
      if constexpr (SLOPE)
      {
        float g[N];
        now.get(h, g);
        activate<T, true>(act, v, f, d);
#pragma unroll
        for (int i = 0; i < N; i += 2)
        {
          const float2 w = halves(mul2(pair(g[i], g[i + 1]), pair(d[i], d[i + 1])));
          g[i] = bad ? scale : w.x, g[i + 1] = bad ? scale : w.y;
        }
        slope.set(h, g);
      }
      else
        activate<T, false>(act, v, f, d);
      if (out)
      {
#pragma unroll
        for (int i = 0; i < N; ++i)
          f[i] = bad ? scale : f[i];
        result.set(h, f);
      }
    }
    if (SLOPE)
      slope.store(d_preact + row * d_preact_ld, first, part, width);
    if (out)
      result.store(out + row * out_ld, first, part, width);
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
  return !p || (reinterpret_cast<uintptr_t>(p) % 32 == 0 && stride % (type == DPC_TYPE_F32 ? 8 : 16) == 0);
}

// Blocks of the launch: 32 of 256 threads for every SM at most, of which registers let 2 to 5 run at a time; each has a few rounds of
// work where there is enough.
template <bool WIDE>
unsigned grid_for(int64_t blocks)
{
  const int64_t each = Split<WIDE>::kGroups;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((blocks + each - 1) / each, 148 * 8 * 4));
}

template <typename T>
void launch_pack(cudaStream_t stream, bool w, int act, int64_t rows, int64_t width, const void* x, int64_t x_ld, void* out,
                 int64_t out_ld, int8_t* codes, float* scales)
{
  const int64_t blocks = (width + kBlock - 1) / kBlock;
  const unsigned grid = w ? grid_for<true>(rows * blocks) : grid_for<false>(rows * blocks);
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
  const unsigned grid = w ? grid_for<true>(rows * blocks) : grid_for<false>(rows * blocks);
  const T* g = static_cast<const T*>(d_out);
  T *dx = static_cast<T*>(d_preact), *to = static_cast<T*>(out);
  auto kernel = w ? (g ? packed_backward_kernel<T, true, true> : packed_backward_kernel<T, true, false>)
                  : (g ? packed_backward_kernel<T, false, true> : packed_backward_kernel<T, false, false>);
  kernel<<<grid, kThreads, 0, stream>>>(codes, scales, rows, width, blocks, act, g, d_out_ld, dx, d_preact_ld, to, out_ld);
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
    const bool w = width % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && wide(type, x, x_stride) &&
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
    const bool w = width % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && wide(type, d_out, d_out_stride) &&
                   wide(type, d_preact, d_preact_stride) && wide(type, out, out_stride);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == DPC_TYPE_F32)
      launch_backward<float>(st, w, act, rows, width, codes, scales, d_out, d_out_stride, d_preact, d_preact_stride, out, out_stride);
    else
      launch_backward<__nv_bfloat16>(st, w, act, rows, width, codes, scales, d_out, d_out_stride, d_preact, d_preact_stride, out, out_stride);
    return launched("packed_backward_kernel");
  });
}
