// The norms before and after a residual block, fused with the block's gate and residual scale, and their
// gradients.
//
//   u = norm(y) * wp + bp       r = a x + b g u       h = norm(r) * wn + bn
//
// Backward, with n = (r - mean) * rstd, m = (y - mean) * rstd, q = dh wn and <.> the mean over a row:
//   dr = dr_out + rstd (q - <q> - n <q n>)     dx = a dr       s = b dr      dg = sum s u      t = s g wp
//   dy = rstd (t - <t> - m <t m>)              dwn = sum dh n  dbn = sum dh  dwp = sum s g m   dbp = sum s g
// (an RMS norm has no <q>, <t> and no means).
//
// Bound by memory: forward reads x, y and writes r, h once; backward reads dh, dr_out, r, y and writes dx,
// dy once.  A row lives in the registers of 32 to 512 threads from its load to its last store, so the
// second norm needs no second pass; statistics are two-pass over those registers (the mean first, then the
// squares of what is left), which loses nothing where the mean is large.  Sums over rows (weights,
// biases, gates) stay in registers while a unit of threads walks its rows, are written once per unit and
// added by a second kernel in a fixed order: no atomics, the same bits every time.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "dpc_internal.h"
#include "dpc_operators.cuh"

namespace
{
using namespace dpc::ops;

constexpr int64_t kMaxWidth = 16384;

struct NormParams
{
  int64_t rows, width, rows_per_group;
  int layer, post, has_branch;
  float a, b, eps, inv_width;
  const void *x, *y, *gate, *wp, *bp, *wn, *bn;
  int64_t x_ld, y_ld, gate_ld;
  void *r, *h;
  int64_t r_ld, h_ld;
  float4* stats;
  const void *dh, *dr;
  int64_t dh_ld, dr_ld;
  void *dx, *dy, *dg;
  int64_t dx_ld, dy_ld, dg_ld;
  int64_t units, chunks, chunks_per_group, rows_per_chunk;
  float *sums, *gate_sums; // [4][units][width], [chunks][width]
};

// The elements of a row that a thread holds, VPT * 8 of them.  WIDE: vectors of 8 neighbours, 16-byte
// loads (every pointer, stride and the width allow them); otherwise neighbouring threads hold neighbouring
// elements.
template <bool WIDE, int TPR>
__device__ __forceinline__ int column(int t, int i)
{
  return WIDE ? (t + TPR * (i >> 3)) * 8 + (i & 7) : i * TPR + t;
}

template <typename T, bool WIDE, int TPR, int N>
__device__ __forceinline__ void load_row(const void* base, int64_t offset, int width, int t, float (&v)[N], float outside)
{
  const T* p = static_cast<const T*>(base) + offset;
  if (WIDE)
  {
#pragma unroll
    for (int i = 0; i < N; i += 8)
    {
      const int c = column<WIDE, TPR>(t, i);
      if (c < width)
        load8w(p + c, &v[i]);
      else
      {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          v[i + k] = outside;
      }
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
      const int c = column<WIDE, TPR>(t, i);
      v[i] = c < width ? to_float(p[c]) : outside;
    }
  }
}

template <typename T, bool WIDE, int TPR, int N>
__device__ __forceinline__ void store_row(void* base, int64_t offset, int width, int t, const float (&v)[N])
{
  T* p = static_cast<T*>(base) + offset;
  if (WIDE)
  {
#pragma unroll
    for (int i = 0; i < N; i += 8)
    {
      const int c = column<WIDE, TPR>(t, i);
      if (c < width)
        store8w(p + c, &v[i]);
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
      const int c = column<WIDE, TPR>(t, i);
      if (c < width)
        p[c] = from_float<T>(v[i]);
    }
  }
}

// Two sums over the threads of a row, to all of them.  More than a warp: through one of two buffers in turn,
// so that one barrier is enough.
template <int TPR>
struct RowSum
{
  float2 (*buffer)[TPR / 32];
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b)
  {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (TPR == 32)
      return make_float2(a, b);
    float2* now = buffer[turn & 1];
    ++turn;
    if ((threadIdx.x & 31) == 0)
      now[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w)
      s.x += now[w].x, s.y += now[w].y;
    return s;
  }
};

// mean and 1/deviation of the row in v; leaves v - mean in v (0 outside the row).
template <bool WIDE, int TPR, int N>
__device__ __forceinline__ float2 standardise(float (&v)[N], const NormParams& P, int t, RowSum<TPR>& sum)
{
  float mean = 0.0f, s = 0.0f;
  if (P.layer)
  {
#pragma unroll
    for (int i = 0; i < N; ++i)
      s += v[i];
    mean = sum(s, 0.0f).x * P.inv_width;
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = column<WIDE, TPR>(t, i) < (int)P.width ? v[i] - mean : 0.0f;
  }
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    s = fmaf(v[i], v[i], s);
  const float rstd = 1.0f / sqrtf(sum(s, 0.0f).x * P.inv_width + P.eps);
  return make_float2(mean, rstd);
}

template <typename T, bool WIDE, int TPR, int N>
__device__ __forceinline__ void affine(float (&v)[N], const void* weight, const void* bias, int width, int t)
{
  float w[N];
  if (weight)
  {
    load_row<T, WIDE, TPR>(weight, 0, width, t, w, 0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] *= w[i];
  }
  if (bias)
  {
    load_row<T, WIDE, TPR>(bias, 0, width, t, w, 0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] += w[i];
  }
}

template <int TPR>
struct Shape
{
  static constexpr int kThreads = TPR == 32 ? 128 : TPR;
  static constexpr int kUnits = kThreads / TPR; // rows that a block has under way
};

template <typename T, bool WIDE, int TPR, int VPT>
__global__ void __launch_bounds__(Shape<TPR>::kThreads) norm_forward_kernel(const NormParams P)
{
  constexpr int N = VPT * 8;
  __shared__ float2 buffer[2][TPR / 32];
  RowSum<TPR> sum{buffer};
  const int t = threadIdx.x & (TPR - 1), width = (int)P.width;
  const int64_t row = (int64_t)blockIdx.x * Shape<TPR>::kUnits + threadIdx.x / TPR;
  if (row >= P.rows)
    return; // (a whole warp, where a block has several rows)
  float v[N], x[N];
  float2 first = make_float2(0.0f, 0.0f);
  load_row<T, WIDE, TPR>(P.x, row * P.x_ld, width, t, x, 0.0f);
  if (P.has_branch)
  {
    load_row<T, WIDE, TPR>(P.y, row * P.y_ld, width, t, v, 0.0f);
    if (P.post)
    {
      first = standardise<WIDE, TPR>(v, P, t, sum);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] *= first.y;
      affine<T, WIDE, TPR>(v, P.wp, P.bp, width, t);
    }
    if (P.gate)
    {
      float g[N];
      load_row<T, WIDE, TPR>(P.gate, row / P.rows_per_group * P.gate_ld, width, t, g, 0.0f);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = fmaf(P.a, x[i], P.b * v[i]);
    store_row<T, WIDE, TPR>(P.r, row * P.r_ld, width, t, v);
  }
  else
  {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = x[i];
  }
  const float2 second = standardise<WIDE, TPR>(v, P, t, sum);
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] *= second.y;
  affine<T, WIDE, TPR>(v, P.wn, P.bn, width, t);
  store_row<T, WIDE, TPR>(P.h, row * P.h_ld, width, t, v);
  if (t == 0)
    P.stats[row] = make_float4(first.x, first.y, second.x, second.y);
}

// 0 outside the row, where v - mean would not be
template <bool WIDE, int TPR, int N>
__device__ __forceinline__ void normalise(float (&v)[N], float mean, float rstd, int width, int t)
{
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = column<WIDE, TPR>(t, i) < width ? (v[i] - mean) * rstd : 0.0f;
}

template <typename T, bool WIDE, int TPR, int VPT, bool BIAS>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, TPR <= 256 ? 512 / Shape<TPR>::kThreads : 1)
    norm_backward_kernel(const NormParams P)
{
  constexpr int N = VPT * 8;
  __shared__ float2 buffer[2][TPR / 32];
  RowSum<TPR> sum{buffer};
  const int t = threadIdx.x & (TPR - 1), width = (int)P.width;
  const int64_t unit = (int64_t)blockIdx.x * Shape<TPR>::kUnits + threadIdx.x / TPR;
  if (unit >= P.units)
    return;
  float dwn[N] = {}, dwp[N] = {}, dbn[BIAS ? N : 1] = {}, dbp[BIAS ? N : 1] = {};
  for (int64_t chunk = unit; chunk < P.chunks; chunk += P.units)
  {
    const int64_t group = chunk / P.chunks_per_group;
    const int64_t begin = group * P.rows_per_group + (chunk - group * P.chunks_per_group) * P.rows_per_chunk;
    const int64_t last = (group + 1) * P.rows_per_group;
    const int64_t end = begin + P.rows_per_chunk < last ? begin + P.rows_per_chunk : last;
    float dg[N] = {};
    for (int64_t row = begin; row < end; ++row)
    {
      const float4 st = P.stats[row];
      float n[N], q[N], w[N];
      load_row<T, WIDE, TPR>(P.r, row * P.r_ld, width, t, n, 0.0f);
      load_row<T, WIDE, TPR>(P.dh, row * P.dh_ld, width, t, q, 0.0f);
      normalise<WIDE, TPR>(n, st.z, st.w, width, t);
#pragma unroll
      for (int i = 0; i < N; ++i)
      {
        dwn[i] = fmaf(q[i], n[i], dwn[i]);
        if (BIAS)
          dbn[i] += q[i];
      }
      if (P.wn)
      {
        load_row<T, WIDE, TPR>(P.wn, 0, width, t, w, 0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i)
          q[i] *= w[i];
      }
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        s1 += q[i], s2 = fmaf(q[i], n[i], s2);
      float2 mean = sum(s1, s2);
      mean.x = P.layer ? mean.x * P.inv_width : 0.0f, mean.y *= P.inv_width;
      // (nothing outside the row: the second norm sums over q)
#pragma unroll
      for (int i = 0; i < N; ++i)
        q[i] = column<WIDE, TPR>(t, i) < width ? st.w * (q[i] - mean.x - n[i] * mean.y) : 0.0f;
      if (P.dr)
      {
        load_row<T, WIDE, TPR>(P.dr, row * P.dr_ld, width, t, w, 0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i)
          q[i] += w[i];
      }
      if (P.dx)
      {
#pragma unroll
        for (int i = 0; i < N; ++i)
          w[i] = P.a * q[i];
        store_row<T, WIDE, TPR>(P.dx, row * P.dx_ld, width, t, w);
      }
      if (!P.has_branch)
        continue;
      // q: gradient of b g u from here on.  n: the branch, standardised where it has a norm
      load_row<T, WIDE, TPR>(P.y, row * P.y_ld, width, t, n, 0.0f);
      if (P.post)
        normalise<WIDE, TPR>(n, st.x, st.y, width, t);
#pragma unroll
      for (int i = 0; i < N; ++i)
        q[i] *= P.b;
      if (P.dg)
      {
#pragma unroll
        for (int i = 0; i < N; ++i)
          w[i] = n[i];
        if (P.post)
          affine<T, WIDE, TPR>(w, P.wp, P.bp, width, t);
#pragma unroll
        for (int i = 0; i < N; ++i)
          dg[i] = fmaf(q[i], w[i], dg[i]);
      }
      if (P.gate)
      {
        load_row<T, WIDE, TPR>(P.gate, group * P.gate_ld, width, t, w, 0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i)
          q[i] *= w[i];
      }
      if (P.post)
      {
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
          dwp[i] = fmaf(q[i], n[i], dwp[i]);
          if (BIAS)
            dbp[i] += q[i];
        }
        if (P.wp)
        {
          load_row<T, WIDE, TPR>(P.wp, 0, width, t, w, 0.0f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            q[i] *= w[i];
        }
        s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
          s1 += q[i], s2 = fmaf(q[i], n[i], s2);
        mean = sum(s1, s2);
        mean.x = P.layer ? mean.x * P.inv_width : 0.0f, mean.y *= P.inv_width;
#pragma unroll
        for (int i = 0; i < N; ++i)
          q[i] = st.y * (q[i] - mean.x - n[i] * mean.y);
      }
      if (P.dy)
        store_row<T, WIDE, TPR>(P.dy, row * P.dy_ld, width, t, q);
    }
    if (P.dg)
    {
      if (P.chunks_per_group == 1)
        store_row<T, WIDE, TPR>(P.dg, group * P.dg_ld, width, t, dg);
      else
        store_row<float, WIDE, TPR>(P.gate_sums, chunk * width, width, t, dg);
    }
  }
  const int64_t plane = P.units * width, at = unit * width;
  store_row<float, WIDE, TPR>(P.sums, at, width, t, dwn);
  store_row<float, WIDE, TPR>(P.sums, at + plane, width, t, dwp);
  if (BIAS)
  {
    store_row<float, WIDE, TPR, N>(P.sums, at + 2 * plane, width, t, reinterpret_cast<const float(&)[N]>(dbn));
    store_row<float, WIDE, TPR, N>(P.sums, at + 3 * plane, width, t, reinterpret_cast<const float(&)[N]>(dbp));
  }
}

// Adds the units' sums: vector blockIdx.y of 32 columns a block; the first four are weights and biases, the
// others the gates.
struct JoinParams
{
  const float *sums, *gate_sums;
  int64_t units, width, chunks_per_group, dg_ld;
  void* out[4];
  void* dg;
};

template <typename T>
__global__ void __launch_bounds__(256) norm_join_kernel(const JoinParams P)
{
  __shared__ float parts[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + lane;
  const float* src;
  T* out;
  int64_t count;
  if (blockIdx.y < 4)
  {
    out = static_cast<T*>(P.out[blockIdx.y]);
    src = P.sums + blockIdx.y * P.units * P.width, count = P.units;
    if (!out)
      return;
  }
  else
  {
    const int64_t group = blockIdx.y - 4;
    out = static_cast<T*>(P.dg) + group * P.dg_ld;
    src = P.gate_sums + group * P.chunks_per_group * P.width, count = P.chunks_per_group;
  }
  float s = 0.0f;
  if (col < P.width)
    for (int64_t u = warp; u < count; u += 8)
      s += src[u * P.width + col];
  parts[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < P.width)
  {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w)
      s += parts[w][lane];
    out[col] = from_float<T>(s);
  }
}

// ------------------------------------------------------------------------------ host
int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// Threads of a row: two vectors of 8 a thread, four in the widest rows.
int threads_of(int64_t width) { return width <= 512 ? 32 : width <= 2048 ? 128 : width <= 4096 ? 256 : 512; }

struct Split
{
  int64_t units = 1, chunks = 1, chunks_per_group = 1, rows_per_chunk = 1;
  bool gates = false; // sums of gates go through the workspace
  size_t gate_at = 0, bytes = 0;
};

int split_rows(const dpc_residual_norm* c, Split& S)
{
  int device = 0, sms = 0;
  DPC_CUDA(cudaGetDevice(&device));
  DPC_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // Units that the GPU holds at once: 512 threads an SM, the registers of the kernel allow no more.
  const int64_t most = (int64_t)sms * (512 / threads_of(c->width));
  const int64_t groups = c->gate ? c->groups : 1, per = c->rows / groups;
  S.chunks_per_group = std::max<int64_t>(1, std::min(per, most / groups));
  S.rows_per_chunk = std::max<int64_t>(1, ceil_div(per, S.chunks_per_group));
  S.chunks_per_group = std::max<int64_t>(1, ceil_div(per, S.rows_per_chunk));
  S.chunks = S.chunks_per_group * groups;
  S.units = std::min(S.chunks, most);
  S.gates = c->gate && S.chunks_per_group > 1;
  size_t at = (size_t)S.units * c->width * 4 * sizeof(float);
  at = (at + 255) / 256 * 256;
  S.gate_at = at;
  if (S.gates)
    at += (size_t)S.chunks * c->width * sizeof(float);
  S.bytes = std::max<size_t>(at, 256);
  return DPC_OK;
}

int check(const dpc_residual_norm* c, const std::string& who)
{
  if (!c)
    return dpc::fail(DPC_ERR_INVALID, who + ": no description");
  if (c->type != DPC_TYPE_F32 && c->type != DPC_TYPE_BF16)
    return dpc::fail(DPC_ERR_INVALID, who + ": type is neither DPC_TYPE_F32 nor DPC_TYPE_BF16");
  if (c->norm != DPC_NORM_RMS && c->norm != DPC_NORM_LAYER)
    return dpc::fail(DPC_ERR_INVALID, who + ": norm is neither DPC_NORM_RMS nor DPC_NORM_LAYER");
  if (c->rows < 0 || c->width < 1)
    return dpc::fail(DPC_ERR_INVALID, who + ": rows >= 0 and width >= 1 are needed");
  if (c->width > kMaxWidth)
    return dpc::fail(DPC_ERR_TOO_LARGE, who + ": width is " + std::to_string(c->width) + ", " +
                                            std::to_string(kMaxWidth) + " at most");
  if (c->rows > (int64_t)1 << 31)
    return dpc::fail(DPC_ERR_TOO_LARGE, who + ": rows may be 2^31 at most");
  if (c->gate && (c->groups < 1 || c->rows % c->groups != 0 || c->gate_stride < c->width))
    return dpc::fail(DPC_ERR_INVALID, who + ": the gate's groups have to divide the rows, and its rows not to overlap");
  if (!c->branch && (c->gate || c->post_norm || c->post_weight || c->post_bias || c->stream_scale != 1.0f))
    return dpc::fail(DPC_ERR_INVALID, who + ": without a branch there is no gate, post norm or stream scale");
  if (!c->post_norm && (c->post_weight || c->post_bias))
    return dpc::fail(DPC_ERR_INVALID, who + ": post_weight and post_bias need post_norm");
  if (!(c->eps >= 0.0f))
    return dpc::fail(DPC_ERR_INVALID, who + ": eps is negative");
  return DPC_OK;
}

// Row strides that are used at all.
int check_strides(const dpc_residual_norm* c, const std::string& who, std::initializer_list<std::pair<const void*, int64_t>> all)
{
  for (const auto& m : all)
    if (m.first && (m.second < c->width || m.second > ((int64_t)1 << 40)))
      return dpc::fail(DPC_ERR_INVALID, who + ": a row stride is smaller than the width (or above 2^40)");
  return DPC_OK;
}

bool wide(const dpc_residual_norm* c, std::initializer_list<std::pair<const void*, int64_t>> all)
{
  const int64_t unit = c->type == DPC_TYPE_F32 ? 4 : 8;
  bool ok = c->width % 8 == 0;
  for (const auto& m : all)
    ok = ok && reinterpret_cast<uintptr_t>(m.first) % 16 == 0 && (!m.first || m.second % unit == 0);
  return ok;
}

NormParams params(const dpc_residual_norm* c)
{
  NormParams P = {};
  P.rows = c->rows, P.width = c->width;
  P.rows_per_group = std::max<int64_t>(1, c->gate ? c->rows / c->groups : c->rows);
  P.layer = c->norm == DPC_NORM_LAYER, P.post = c->post_norm != 0, P.has_branch = c->branch != nullptr;
  P.a = c->stream_scale, P.b = c->branch_scale, P.eps = c->eps, P.inv_width = 1.0f / (float)c->width;
  P.x = c->stream, P.y = c->branch, P.gate = c->gate;
  P.wp = c->post_weight, P.bp = c->post_bias, P.wn = c->pre_weight, P.bn = c->pre_bias;
  P.x_ld = c->stream_stride, P.y_ld = c->branch_stride, P.gate_ld = c->gate_stride;
  P.r = c->new_stream, P.h = c->normed;
  P.r_ld = c->new_stream_stride, P.h_ld = c->normed_stride;
  P.stats = reinterpret_cast<float4*>(c->stats);
  return P;
}

template <typename T, bool WIDE, int TPR, int VPT>
int launch_forward(cudaStream_t stream, const NormParams& P)
{
  const unsigned blocks = (unsigned)ceil_div(P.rows, Shape<TPR>::kUnits);
  norm_forward_kernel<T, WIDE, TPR, VPT><<<blocks, Shape<TPR>::kThreads, 0, stream>>>(P);
  return launched("norm_forward_kernel");
}

template <typename T, bool WIDE, int TPR, int VPT>
int launch_backward(cudaStream_t stream, const NormParams& P, bool bias)
{
  const unsigned blocks = (unsigned)ceil_div(P.units, Shape<TPR>::kUnits);
  if (bias)
    norm_backward_kernel<T, WIDE, TPR, VPT, true><<<blocks, Shape<TPR>::kThreads, 0, stream>>>(P);
  else
    norm_backward_kernel<T, WIDE, TPR, VPT, false><<<blocks, Shape<TPR>::kThreads, 0, stream>>>(P);
  return launched("norm_backward_kernel");
}

template <typename T, bool WIDE>
int dispatch(cudaStream_t stream, const NormParams& P, bool back, bool bias)
{
  switch (threads_of(P.width))
  {
  case 32:
    return back ? launch_backward<T, WIDE, 32, 2>(stream, P, bias) : launch_forward<T, WIDE, 32, 2>(stream, P);
  case 128:
    return back ? launch_backward<T, WIDE, 128, 2>(stream, P, bias) : launch_forward<T, WIDE, 128, 2>(stream, P);
  case 256:
    return back ? launch_backward<T, WIDE, 256, 2>(stream, P, bias) : launch_forward<T, WIDE, 256, 2>(stream, P);
  default:
    if (P.width <= 8192)
      return back ? launch_backward<T, WIDE, 512, 2>(stream, P, bias) : launch_forward<T, WIDE, 512, 2>(stream, P);
    return back ? launch_backward<T, WIDE, 512, 4>(stream, P, bias) : launch_forward<T, WIDE, 512, 4>(stream, P);
  }
}

int dispatch(cudaStream_t stream, int type, bool is_wide, const NormParams& P, bool back, bool bias)
{
  if (type == DPC_TYPE_F32)
    return is_wide ? dispatch<float, true>(stream, P, back, bias) : dispatch<float, false>(stream, P, back, bias);
  return is_wide ? dispatch<__nv_bfloat16, true>(stream, P, back, bias)
                 : dispatch<__nv_bfloat16, false>(stream, P, back, bias);
}

int forward(cudaStream_t stream, const dpc_residual_norm* c)
{
  const std::string who = "dpc_residual_norm_forward";
  if (int rc = check(c, who))
    return rc;
  if (c->rows == 0)
    return DPC_OK;
  if (!c->stream || !c->normed || !c->stats || (c->branch && !c->new_stream) ||
      reinterpret_cast<uintptr_t>(c->stats) % 16)
    return dpc::fail(DPC_ERR_INVALID, who + ": null pointer, or stats off a 16-byte boundary");
  const void* kept = c->branch ? c->new_stream : nullptr;
  if (int rc = check_strides(c, who, {{c->stream, c->stream_stride}, {c->branch, c->branch_stride},
                                      {kept, c->new_stream_stride}, {c->normed, c->normed_stride}}))
    return rc;
  const bool w = wide(c, {{c->stream, c->stream_stride}, {c->branch, c->branch_stride}, {c->gate, c->gate_stride},
                          {kept, c->new_stream_stride}, {c->normed, c->normed_stride}, {c->post_weight, 0},
                          {c->post_bias, 0}, {c->pre_weight, 0}, {c->pre_bias, 0}});
  return dispatch(stream, c->type, w, params(c), false, false);
}

int zero_vector(cudaStream_t stream, const dpc_residual_norm* c, void* p, int64_t rows, int64_t stride)
{
  const size_t size = c->type == DPC_TYPE_F32 ? 4 : 2;
  if (p && rows > 0)
    DPC_CUDA(cudaMemset2DAsync(p, stride * size, 0, c->width * size, rows, stream));
  return DPC_OK;
}

int backward(cudaStream_t stream, const dpc_residual_norm* c)
{
  const std::string who = "dpc_residual_norm_backward";
  if (int rc = check(c, who))
    return rc;
  if ((c->d_gate && (!c->gate || c->d_gate_stride < c->width)) || (c->d_post_weight && !c->post_norm) ||
      (c->d_post_bias && !c->post_norm) || (c->d_branch && !c->branch))
    return dpc::fail(DPC_ERR_INVALID, who + ": a gradient is asked for of what is not there");
  if (c->rows == 0)
  {
    for (void* p : {c->d_post_weight, c->d_post_bias, c->d_pre_weight, c->d_pre_bias})
      if (int rc = zero_vector(stream, c, p, 1, c->width))
        return rc;
    return zero_vector(stream, c, c->d_gate, c->groups, c->d_gate_stride);
  }
  if (!c->new_stream || !c->stats || !c->d_normed || reinterpret_cast<uintptr_t>(c->stats) % 16)
    return dpc::fail(DPC_ERR_INVALID, who + ": null pointer, or stats off a 16-byte boundary");
  if (int rc = check_strides(c, who, {{c->branch, c->branch_stride}, {c->new_stream, c->new_stream_stride},
                                      {c->d_normed, c->d_normed_stride}, {c->d_new_stream, c->d_new_stream_stride},
                                      {c->d_stream, c->d_stream_stride}, {c->d_branch, c->d_branch_stride}}))
    return rc;
  Split S;
  if (int rc = split_rows(c, S))
    return rc;
  if (!c->workspace || reinterpret_cast<uintptr_t>(c->workspace) % 256 || c->workspace_bytes < S.bytes)
    return dpc::fail(DPC_ERR_INVALID, who + ": " + std::to_string(S.bytes) +
                                          " bytes of workspace on a 256-byte boundary are needed");
  NormParams P = params(c);
  P.dh = c->d_normed, P.dr = c->d_new_stream, P.dx = c->d_stream, P.dy = c->d_branch, P.dg = c->d_gate;
  P.dh_ld = c->d_normed_stride, P.dr_ld = c->d_new_stream_stride, P.dx_ld = c->d_stream_stride;
  P.dy_ld = c->d_branch_stride, P.dg_ld = c->d_gate_stride;
  P.units = S.units, P.chunks = S.chunks, P.chunks_per_group = S.chunks_per_group, P.rows_per_chunk = S.rows_per_chunk;
  P.sums = static_cast<float*>(c->workspace);
  P.gate_sums = reinterpret_cast<float*>(static_cast<char*>(c->workspace) + S.gate_at);
  const bool w = wide(c, {{c->branch, c->branch_stride}, {c->gate, c->gate_stride},
                          {c->new_stream, c->new_stream_stride}, {c->d_normed, c->d_normed_stride},
                          {c->d_new_stream, c->d_new_stream_stride}, {c->d_stream, c->d_stream_stride},
                          {c->d_branch, c->d_branch_stride}, {c->d_gate, c->d_gate_stride}, {c->post_weight, 0},
                          {c->post_bias, 0}, {c->pre_weight, 0}});
  if (int rc = dispatch(stream, c->type, w, P, true, c->d_post_bias || c->d_pre_bias))
    return rc;
  JoinParams J = {};
  J.sums = P.sums, J.gate_sums = P.gate_sums, J.units = S.units, J.width = c->width;
  J.chunks_per_group = S.chunks_per_group, J.dg = c->d_gate, J.dg_ld = c->d_gate_stride;
  J.out[0] = c->d_pre_weight, J.out[1] = c->d_post_weight, J.out[2] = c->d_pre_bias, J.out[3] = c->d_post_bias;
  const int64_t vectors = 4 + (S.gates && c->d_gate ? c->groups : 0);
  const dim3 grid((unsigned)ceil_div(c->width, 32), (unsigned)vectors); // (groups: fewer than units there)
  if (c->type == DPC_TYPE_F32)
    norm_join_kernel<float><<<grid, 256, 0, stream>>>(J);
  else
    norm_join_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(J);
  return launched("norm_join_kernel");
}
} // namespace

int dpc_residual_norm_forward(void* stream, const dpc_residual_norm* c)
{
  return guarded("dpc_residual_norm_forward", [&] { return forward(static_cast<cudaStream_t>(stream), c); });
}

int dpc_residual_norm_workspace(const dpc_residual_norm* c, size_t* bytes)
{
  return guarded("dpc_residual_norm_workspace", [&] {
    if (!bytes)
      return dpc::fail(DPC_ERR_INVALID, "dpc_residual_norm_workspace: null pointer");
    if (int rc = check(c, "dpc_residual_norm_workspace"))
      return rc;
    Split S;
    if (int rc = split_rows(c, S))
      return rc;
    *bytes = S.bytes;
    return (int)DPC_OK;
  });
}

int dpc_residual_norm_backward(void* stream, const dpc_residual_norm* c)
{
  return guarded("dpc_residual_norm_backward", [&] { return backward(static_cast<cudaStream_t>(stream), c); });
}
