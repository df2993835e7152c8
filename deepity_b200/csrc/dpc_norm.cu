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
//
// Those sums leave registers for 512 threads an SM, too few to cover the memory's latency with loads of their
// own: backward fetches its four rows and their statistics two and more ahead into shared memory by bulk copies.
// 16384 x 4096 bf16 (805 MB, 123 us at the rate of a copy): 256 us with loads in the threads themselves, 219 with the
// copies, 160 with arithmetic on pairs and no register spilled; what is left waits for the row's two sums and for
// weights from L1.  Spills decide here: 100 bytes of them cost 50 us; a second row at once, or a warp that only
// fetches, cost more than they gave.
// Forward: 50 us at 16384 x 2048 bf16 (268 MB, 41 us); with one vector a thread 62.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "dpc_internal.h"
#include "dpc_operators.cuh"
#include "dpc_tcgen05.cuh"

namespace
{
using namespace dpc::ops;

constexpr int64_t kMaxWidth = 16384;

// (Kept at 288 bytes: 16 more took a call of few rows 0.5 us longer.)
struct NormParams
{
  int64_t rows;
  int width;
  int wait_kilocycles; // limit of a wait for a row; negative: more bytes are waited for than come, so that the waits run out
  int rows_per_group;
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
  int units, chunks, chunks_per_group, rows_per_chunk;
  float *sums, *gate_sums; // [4][units][sums_ld], [chunks][sums_ld]
  int64_t sums_ld;         // the width, up to a multiple of 8
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

// Two sums over the threads of a row (the first where `both`), to all of them.  More than a warp: through one of
// two buffers in turn, so that one barrier is enough.
template <int TPR>
struct RowSum
{
  float2 (*buffer)[TPR / 32];
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b, bool both)
  {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      b += __shfl_xor_sync(0xffffffffu, b, o);
    if (both)
    {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        a += __shfl_xor_sync(0xffffffffu, a, o);
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
    mean = sum(0.0f, s, false).y * P.inv_width;
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = column<WIDE, TPR>(t, i) < P.width ? v[i] - mean : 0.0f;
  }
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    s = fmaf(v[i], v[i], s);
  const float rstd = 1.0f / sqrtf(sum(0.0f, s, false).y * P.inv_width + P.eps);
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
  const int t = threadIdx.x & (TPR - 1), width = P.width;
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

// Backward works on pairs of neighbours (elements 2i and 2i + 1 of a thread).
template <typename T, bool WIDE, int TPR, int M>
__device__ __forceinline__ void load_pairs(const void* base, int64_t offset, int width, int t, float2x (&v)[M])
{
  const T* p = static_cast<const T*>(base) + offset;
  if constexpr (WIDE)
  {
#pragma unroll
    for (int i = 0; i < M; i += 4)
    {
      const int c = column<WIDE, TPR>(t, 2 * i);
      if constexpr (sizeof(T) == 2)
      {
        uint4 r = make_uint4(0, 0, 0, 0);
        if (c < width)
          r = *reinterpret_cast<const uint4*>(p + c);
        v[i] = pair_of_bf16(r.x), v[i + 1] = pair_of_bf16(r.y), v[i + 2] = pair_of_bf16(r.z), v[i + 3] = pair_of_bf16(r.w);
      }
      else
      {
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
        if (c < width)
          a = reinterpret_cast<const float4*>(p + c)[0], b = reinterpret_cast<const float4*>(p + c)[1];
        v[i] = pair(a.x, a.y), v[i + 1] = pair(a.z, a.w), v[i + 2] = pair(b.x, b.y), v[i + 3] = pair(b.z, b.w);
      }
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < M; ++i)
    {
      const int c = column<WIDE, TPR>(t, 2 * i), d = column<WIDE, TPR>(t, 2 * i + 1);
      v[i] = pair(c < width ? to_float(p[c]) : 0.0f, d < width ? to_float(p[d]) : 0.0f);
    }
  }
}

template <typename T, bool WIDE, int TPR, int M>
__device__ __forceinline__ void store_pairs(void* base, int64_t offset, int width, int t, const float2x (&v)[M])
{
  T* p = static_cast<T*>(base) + offset;
  if constexpr (WIDE)
  {
#pragma unroll
    for (int i = 0; i < M; i += 4)
    {
      const int c = column<WIDE, TPR>(t, 2 * i);
      if (c < width)
      {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint4*>(p + c) = make_uint4(bf16_of_pair(v[i]), bf16_of_pair(v[i + 1]), bf16_of_pair(v[i + 2]),
                                                        bf16_of_pair(v[i + 3]));
        else
        {
          const float2 a = halves(v[i]), b = halves(v[i + 1]), e = halves(v[i + 2]), f = halves(v[i + 3]);
          reinterpret_cast<float4*>(p + c)[0] = make_float4(a.x, a.y, b.x, b.y);
          reinterpret_cast<float4*>(p + c)[1] = make_float4(e.x, e.y, f.x, f.y);
        }
      }
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < M; ++i)
    {
      const int c = column<WIDE, TPR>(t, 2 * i), d = column<WIDE, TPR>(t, 2 * i + 1);
      const float2 f = halves(v[i]);
      if (c < width)
        p[c] = from_float<T>(f.x);
      if (d < width)
        p[d] = from_float<T>(f.y);
    }
  }
}

template <int M>
__device__ __forceinline__ void normalise(float2x (&v)[M], float mean, float rstd, bool layer)
{
  if (layer)
  {
#pragma unroll
    for (int i = 0; i < M; ++i)
      v[i] = add2(v[i], pair(-mean));
  }
#pragma unroll
  for (int i = 0; i < M; ++i)
    v[i] = mul2(v[i], pair(rstd));
}

// The means over the row that the gradient of a norm takes off: of q (layer norms) and of q n.
template <int TPR, int M>
__device__ __forceinline__ float2 means(const float2x (&q)[M], const float2x (&n)[M], const NormParams& P, RowSum<TPR>& sum)
{
  float2x s1 = 0, s2 = 0;
#pragma unroll
  for (int i = 0; i < M; ++i)
    s2 = fma2(q[i], n[i], s2);
  if (P.layer)
  {
#pragma unroll
    for (int i = 0; i < M; ++i)
      s1 = add2(s1, q[i]);
  }
  const float2 a = halves(s1), b = halves(s2);
  const float2 all = sum(a.x + a.y, b.x + b.y, P.layer != 0);
  return make_float2(all.x * P.inv_width, all.y * P.inv_width);
}

// q - <q> - n <q n>
template <int M>
__device__ __forceinline__ void take_off(float2x (&q)[M], const float2x (&n)[M], float2 mean, bool layer)
{
#pragma unroll
  for (int i = 0; i < M; ++i)
    q[i] = fma2(n[i], pair(-mean.y), q[i]);
  if (layer)
  {
#pragma unroll
    for (int i = 0; i < M; ++i)
      q[i] = add2(q[i], pair(-mean.x));
  }
}

// The rows of a unit in their order: chunk after chunk, `units` apart.
struct Cursor
{
  int chunk, row, end, group;
  __device__ __forceinline__ void open(const NormParams& P)
  {
    if (chunk >= P.chunks)
      return;
    group = chunk / P.chunks_per_group;
    row = group * P.rows_per_group + (chunk - group * P.chunks_per_group) * P.rows_per_chunk;
    const int last = (group + 1) * P.rows_per_group;
    end = last - row > P.rows_per_chunk ? row + P.rows_per_chunk : last;
  }
  __device__ __forceinline__ bool valid(const NormParams& P) const { return chunk < P.chunks; }
  __device__ __forceinline__ void next(const NormParams& P)
  {
    if (++row == end)
    {
      chunk = P.chunks - chunk > P.units ? chunk + P.units : P.chunks; // (nothing above their number, which may be 2^31 - 1)
      open(P);
    }
  }
};

constexpr int kFetched = 4; // new stream, d_normed, d_new_stream, branch

// STAGES > 0: rows are fetched that many ahead.  The slot of a row is filled again after the first sum over the
// next row, which every thread reaches after its last read of the slot.
template <typename T, bool WIDE, int TPR, int VPT, bool BIAS, int STAGES>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, 512 / Shape<TPR>::kThreads)
    norm_backward_kernel(const NormParams P)
{
  constexpr int M = VPT * 4, kUnits = Shape<TPR>::kUnits;
  constexpr bool kAhead = STAGES > 0;
  __shared__ float2 buffer[2][TPR / 32];
  __shared__ uint64_t filled[kUnits][kAhead ? STAGES : 1];
  __shared__ __align__(16) float4 statistics[kUnits][kAhead ? STAGES : 1];
  __shared__ __align__(16) int give_up[4];
  __shared__ Cursor ahead[kUnits]; // the next row to fetch: kept by thread 0 of a unit, out of the others' registers
  extern __shared__ __align__(128) uint8_t slots[];
  RowSum<TPR> sum{buffer};
  const int t = threadIdx.x & (TPR - 1), width = P.width, local = threadIdx.x / TPR;
  const int unit = blockIdx.x * kUnits + local;
  const uint32_t row_bytes = (uint32_t)(width * sizeof(T));
  const uint32_t slot_at = local * STAGES * kFetched * row_bytes;
  uint64_t* full = filled[local];
  if (kAhead)
  {
    if (threadIdx.x == 0)
    {
      for (int u = 0; u < kUnits; ++u)
        for (int s = 0; s < STAGES; ++s)
          dpc::ptx::mbar_init(&filled[u][s], 1);
      give_up[0] = 0;
      *reinterpret_cast<long long*>(give_up + 2) = 1000LL * abs(P.wait_kilocycles);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
  }
  if (unit >= P.units)
    return;
  auto fetch = [&](int64_t row, int s) { // by one thread of the unit
    dpc::ptx::mbar_expect_tx(&full[s], row_bytes * (2 + (P.dr != nullptr) + (P.has_branch != 0)) + (uint32_t)sizeof(float4) +
                                            (P.wait_kilocycles < 0 ? 16 : 0));
    auto bulk = [&](uint32_t to, const void* from, uint32_t bytes) {
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                   "l"(from), "r"(bytes), "r"(dpc::ptx::smem_u32(&full[s]))
                   : "memory");
    };
    auto copy = [&](int k, const void* from, int64_t ld) {
      bulk(dpc::ptx::smem_u32(slots) + slot_at + (s * kFetched + k) * row_bytes, static_cast<const T*>(from) + row * ld, row_bytes);
    };
    bulk(dpc::ptx::smem_u32(&statistics[local][s]), P.stats + row, (uint32_t)sizeof(float4));
    copy(0, P.r, P.r_ld);
    copy(1, P.dh, P.dh_ld);
    if (P.dr)
      copy(2, P.dr, P.dr_ld);
    if (P.has_branch)
      copy(3, P.y, P.y_ld);
  };
  Cursor now{unit, 0, 0, 0};
  now.open(P);
  if (kAhead && t == 0)
  {
    Cursor c = now;
    for (int s = 0; s < STAGES && c.valid(P); ++s, c.next(P))
      fetch(c.row, s);
    ahead[local] = c;
  }
  float2x dwn[M] = {}, dwp[M] = {}, dg[M] = {}, dbn[BIAS ? M : 1] = {}, dbp[BIAS ? M : 1] = {};
  const bool layer = P.layer != 0;
  bool used = false; // a row before this one has left its slot
  bool there = true; // no wait has given up: from then on all is NaN, and no slot is filled again
  for (int slot = 0, parity = 0; now.valid(P);)
  {
    const int64_t row = now.row;
    float4 st;
    if constexpr (kAhead)
    {
      there = there && dpc::ptx::mbar_wait(&full[slot], parity, give_up);
      st = statistics[local][slot];
    }
    else
      st = __ldg(P.stats + row);
    if (!there) // a copy that is never seen to arrive: NaN
      st = make_float4(NAN, NAN, NAN, NAN);
    auto get = [&](int k, const void* base, int64_t ld, float2x(&v)[M]) {
      if constexpr (kAhead)
        load_pairs<T, WIDE, TPR>(slots + slot_at + ((slot * kFetched + k) * row_bytes), 0, width, t, v);
      else
        load_pairs<T, WIDE, TPR>(base, row * ld, width, t, v);
    };
    float2x n[M], q[M], w[M];
    get(0, P.r, P.r_ld, n);
    get(1, P.dh, P.dh_ld, q);
    normalise(n, st.z, st.w, layer);
#pragma unroll
    for (int i = 0; i < M; ++i)
    {
      dwn[i] = fma2(q[i], n[i], dwn[i]);
      if (BIAS)
        dbn[i] = add2(dbn[i], there ? q[i] : pair(NAN));
    }
    if (P.wn)
    {
      load_pairs<T, WIDE, TPR>(P.wn, 0, width, t, w);
#pragma unroll
      for (int i = 0; i < M; ++i)
        q[i] = mul2(q[i], w[i]);
    }
    float2 mean = means(q, n, P, sum);
    if (kAhead && t == 0)
    {
      Cursor c = ahead[local];
      if (used && there && c.valid(P))
      {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fetch(c.row, slot == 0 ? STAGES - 1 : slot - 1);
        c.next(P);
        ahead[local] = c;
      }
      used = true;
    }
    take_off(q, n, mean, layer);
    // times 1/deviation; nothing outside the row: the second norm sums over q
    auto scale = [&](int i) {
      const float lo = column<WIDE, TPR>(t, 2 * i) < width ? st.w : 0.0f;
      return pair(lo, WIDE ? lo : column<WIDE, TPR>(t, 2 * i + 1) < width ? st.w : 0.0f);
    };
    if (P.dr)
    {
      get(2, P.dr, P.dr_ld, w);
#pragma unroll
      for (int i = 0; i < M; ++i)
        q[i] = fma2(q[i], scale(i), w[i]);
    }
    else
    {
#pragma unroll
      for (int i = 0; i < M; ++i)
        q[i] = mul2(q[i], scale(i));
    }
    if (P.dx)
    {
#pragma unroll
      for (int i = 0; i < M; ++i)
        w[i] = mul2(q[i], pair(P.a));
      store_pairs<T, WIDE, TPR>(P.dx, (int64_t)row * P.dx_ld, width, t, w);
    }
    if (P.has_branch)
    {
      // q: gradient of b g u from here on.  n: the branch, standardised where it has a norm
      get(3, P.y, P.y_ld, n);
      if (P.post)
        normalise(n, st.x, st.y, layer);
#pragma unroll
      for (int i = 0; i < M; ++i)
        q[i] = mul2(q[i], pair(P.b));
      if (P.dg)
      {
        // dg += q (n wp + bp)
        if (P.bp)
        {
          load_pairs<T, WIDE, TPR>(P.bp, 0, width, t, w);
#pragma unroll
          for (int i = 0; i < M; ++i)
            dg[i] = fma2(q[i], w[i], dg[i]);
        }
        if (P.wp)
        {
          load_pairs<T, WIDE, TPR>(P.wp, 0, width, t, w);
#pragma unroll
          for (int i = 0; i < M; ++i)
            dg[i] = fma2(q[i], mul2(w[i], n[i]), dg[i]);
        }
        else
        {
#pragma unroll
          for (int i = 0; i < M; ++i)
            dg[i] = fma2(q[i], n[i], dg[i]);
        }
      }
      if (P.gate)
      {
        load_pairs<T, WIDE, TPR>(P.gate, (int64_t)now.group * P.gate_ld, width, t, w);
#pragma unroll
        for (int i = 0; i < M; ++i)
          q[i] = mul2(q[i], w[i]);
      }
      if (P.post)
      {
#pragma unroll
        for (int i = 0; i < M; ++i)
        {
          dwp[i] = fma2(q[i], n[i], dwp[i]);
          if (BIAS)
            dbp[i] = add2(dbp[i], q[i]);
        }
        if (P.wp)
        {
          load_pairs<T, WIDE, TPR>(P.wp, 0, width, t, w);
#pragma unroll
          for (int i = 0; i < M; ++i)
            q[i] = mul2(q[i], w[i]);
        }
        mean = means(q, n, P, sum);
        take_off(q, n, mean, layer);
#pragma unroll
        for (int i = 0; i < M; ++i)
          q[i] = mul2(q[i], pair(st.y));
      }
      if (P.dy)
        store_pairs<T, WIDE, TPR>(P.dy, (int64_t)row * P.dy_ld, width, t, q);
    }
    if (++slot == STAGES || !kAhead)
      slot = 0, parity ^= 1;
    const int chunk = now.chunk, group = now.group;
    now.next(P);
    if (now.chunk != chunk && P.dg)
    {
      if (P.chunks_per_group == 1)
        store_pairs<T, WIDE, TPR>(P.dg, (int64_t)group * P.dg_ld, width, t, dg);
      else
        store_pairs<float, WIDE, TPR>(P.gate_sums, (int64_t)chunk * P.sums_ld, width, t, dg);
#pragma unroll
      for (int i = 0; i < M; ++i)
        dg[i] = 0;
    }
  }
  const int64_t plane = P.units * P.sums_ld, at = unit * P.sums_ld;
  store_pairs<float, WIDE, TPR>(P.sums, at, width, t, dwn);
  store_pairs<float, WIDE, TPR>(P.sums, at + plane, width, t, dwp);
  if constexpr (BIAS)
  {
    store_pairs<float, WIDE, TPR>(P.sums, at + 2 * plane, width, t, dbn);
    store_pairs<float, WIDE, TPR>(P.sums, at + 3 * plane, width, t, dbp);
  }
  if (kAhead && !there)
  {
    // Copies that were not seen to arrive land before the block's shared memory goes away.
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL * STAGES)
    {
    }
  }
}

// Adds the units' sums: vector blockIdx.y, 128 columns a block; the first four are weights and biases, the
// others the gates.
struct JoinParams
{
  const float *sums, *gate_sums;
  int64_t units, width, ld, chunks_per_group, dg_ld;
  void* out[4];
  void* dg;
};

constexpr int kJoinWarps = 32;

template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) norm_join_kernel(const JoinParams P)
{
  __shared__ float4 parts[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 128 + 4 * lane;
  const float* src;
  T* out;
  int64_t count;
  if (blockIdx.y < 4)
  {
    out = static_cast<T*>(P.out[blockIdx.y]);
    src = P.sums + blockIdx.y * P.units * P.ld, count = P.units;
    if (!out)
      return;
  }
  else
  {
    const int64_t group = blockIdx.y - 4;
    out = static_cast<T*>(P.dg) + group * P.dg_ld;
    src = P.gate_sums + group * P.chunks_per_group * P.ld, count = P.chunks_per_group;
  }
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (col < P.ld)
  {
#pragma unroll 8
    for (int64_t u = warp; u < count; u += kJoinWarps)
    {
      const float4 v = *reinterpret_cast<const float4*>(src + u * P.ld + col);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  parts[warp][lane] = s;
  __syncthreads();
  if (threadIdx.x < 128)
  {
    const float* all = reinterpret_cast<const float*>(parts);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w)
      total += all[w * 128 + threadIdx.x];
    const int64_t mine = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (mine < P.width)
      out[mine] = from_float<T>(total);
  }
}

// ------------------------------------------------------------------------------ host
int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// Threads of a row.  Two vectors of 8 a thread, four in the widest rows; one, as far as 512 threads go, in backward
// passes that keep sums of biases or load element by element (`lean`; two would not fit their registers) and in those of
// 32-bit rows (with two, the rows of an SM's blocks would not fit its shared memory two ahead).
int threads_of(int64_t width, bool lean)
{
  const int64_t each = lean ? 8 : 16;
  return width <= 32 * each ? 32 : width <= 128 * each ? 128 : width <= 256 * each ? 256 : 512;
}

struct Split
{
  int64_t units = 1, chunks = 1, chunks_per_group = 1, rows_per_chunk = 1;
  bool gates = false; // sums of gates go through the workspace
  size_t gate_at = 0, bytes = 0;
};

int split_rows(const dpc_residual_norm* c, bool lean, Split& S)
{
  int device = 0, sms = 0;
  DPC_CUDA(cudaGetDevice(&device));
  DPC_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // Units that the GPU holds at once: 512 threads an SM, the registers of the kernel allow no more.
  const int64_t most = (int64_t)sms * (512 / threads_of(c->width, lean));
  const int64_t groups = c->gate ? c->groups : 1, per = c->rows / groups;
  // (four rows to a unit at least: its sums are written and read again)
  S.chunks_per_group = std::max<int64_t>(1, std::min(ceil_div(per, 4), most / groups));
  S.rows_per_chunk = std::max<int64_t>(1, ceil_div(per, S.chunks_per_group));
  S.chunks_per_group = std::max<int64_t>(1, ceil_div(per, S.rows_per_chunk));
  S.chunks = S.chunks_per_group * groups;
  S.units = std::min(S.chunks, most);
  S.gates = c->gate && S.chunks_per_group > 1;
  const int64_t ld = ceil_div(c->width, 8) * 8;
  size_t at = (size_t)S.units * ld * 4 * sizeof(float);
  at = (at + 255) / 256 * 256;
  S.gate_at = at;
  if (S.gates)
    at += (size_t)S.chunks * ld * sizeof(float);
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
  if (c->rows >= (int64_t)1 << 31)
    return dpc::fail(DPC_ERR_TOO_LARGE, who + ": rows have to be below 2^31");
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
  P.rows = c->rows, P.width = (int)c->width;
  P.rows_per_group = (int)std::max<int64_t>(1, c->gate ? c->rows / c->groups : c->rows);
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

constexpr size_t kSlotBytes = 200 << 10; // shared memory of an SM for rows that are fetched ahead

template <typename T, bool WIDE, int TPR, int VPT, bool BIAS, int STAGES>
int launch_backward(cudaStream_t stream, const NormParams& P)
{
  auto kernel = norm_backward_kernel<T, WIDE, TPR, VPT, BIAS, STAGES>;
  const unsigned blocks = (unsigned)ceil_div(P.units, Shape<TPR>::kUnits);
  const size_t bytes = (size_t)Shape<TPR>::kUnits * STAGES * kFetched * P.width * sizeof(T);
  if (STAGES > 0)
  {
    // The limit belongs to the kernel, not to the launch: with the call's own size, a call on another host thread could
    // lower it between here and the launch.  The most that any width of this kernel takes is the same for all.
    constexpr size_t most = std::min(kSlotBytes, (size_t)Shape<TPR>::kThreads * VPT * 8 * STAGES * kFetched * sizeof(T));
    DPC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  }
  kernel<<<blocks, Shape<TPR>::kThreads, bytes, stream>>>(P);
  return launched("norm_backward_kernel");
}

// Three rows ahead where the blocks of an SM have the shared memory for them; of the widest rows two, or none.  (Those rows
// are longer than half of what their threads hold, so two of them take `widest` at least.)
template <typename T, bool WIDE, int TPR, int VPT, bool BIAS>
int launch_backward(cudaStream_t stream, const NormParams& P)
{
  constexpr size_t widest = (size_t)512 * VPT * 8 * kFetched * sizeof(T); // a round of 512 threads
  if constexpr (WIDE && 3 * widest <= kSlotBytes)
    return launch_backward<T, WIDE, TPR, VPT, BIAS, 3>(stream, P);
  else
  {
    if constexpr (WIDE && widest < kSlotBytes)
    {
      if ((size_t)512 / TPR * kFetched * P.width * sizeof(T) * 2 <= kSlotBytes)
        return launch_backward<T, WIDE, TPR, VPT, BIAS, 2>(stream, P);
    }
    return launch_backward<T, WIDE, TPR, VPT, BIAS, 0>(stream, P);
  }
}

template <typename T, bool WIDE>
int dispatch_forward(cudaStream_t stream, const NormParams& P)
{
  switch (threads_of(P.width, false))
  {
  case 32:
    return launch_forward<T, WIDE, 32, 2>(stream, P);
  case 128:
    return launch_forward<T, WIDE, 128, 2>(stream, P);
  case 256:
    return launch_forward<T, WIDE, 256, 2>(stream, P);
  default:
    return P.width <= 8192 ? launch_forward<T, WIDE, 512, 2>(stream, P) : launch_forward<T, WIDE, 512, 4>(stream, P);
  }
}

template <typename T, bool WIDE, bool BIAS>
int dispatch_backward(cudaStream_t stream, const NormParams& P)
{
  constexpr bool kLean = BIAS || !WIDE || sizeof(T) == 4;
  constexpr int VPT = kLean ? 1 : 2;
  switch (threads_of(P.width, kLean))
  {
  case 32:
    return launch_backward<T, WIDE, 32, VPT, BIAS>(stream, P);
  case 128:
    return launch_backward<T, WIDE, 128, VPT, BIAS>(stream, P);
  case 256:
    return launch_backward<T, WIDE, 256, VPT, BIAS>(stream, P);
  default:
    return P.width <= 512 * VPT * 8 ? launch_backward<T, WIDE, 512, VPT, BIAS>(stream, P)
           : P.width <= 8192        ? launch_backward<T, WIDE, 512, 2, BIAS>(stream, P)
                                    : launch_backward<T, WIDE, 512, 4, BIAS>(stream, P);
  }
}

template <typename T, bool WIDE>
int dispatch(cudaStream_t stream, const NormParams& P, bool back, bool bias)
{
  if (!back)
    return dispatch_forward<T, WIDE>(stream, P);
  return bias ? dispatch_backward<T, WIDE, true>(stream, P) : dispatch_backward<T, WIDE, false>(stream, P);
}

int dispatch(cudaStream_t stream, int type, bool is_wide, const NormParams& P, bool back, bool bias)
{
  if (type == DPC_TYPE_F32)
    return is_wide ? dispatch<float, true>(stream, P, back, bias) : dispatch<float, false>(stream, P, back, bias);
  return is_wide ? dispatch<__nv_bfloat16, true>(stream, P, back, bias)
                 : dispatch<__nv_bfloat16, false>(stream, P, back, bias);
}

bool wide_backward(const dpc_residual_norm* c)
{
  return wide(c, {{c->branch, c->branch_stride}, {c->gate, c->gate_stride}, {c->new_stream, c->new_stream_stride},
                  {c->d_normed, c->d_normed_stride}, {c->d_new_stream, c->d_new_stream_stride},
                  {c->d_stream, c->d_stream_stride}, {c->d_branch, c->d_branch_stride}, {c->d_gate, c->d_gate_stride},
                  {c->post_weight, 0}, {c->post_bias, 0}, {c->pre_weight, 0}});
}

bool with_bias(const dpc_residual_norm* c) { return c->d_post_bias || c->d_pre_bias; }

bool lean_backward(const dpc_residual_norm* c, bool is_wide) { return with_bias(c) || !is_wide || c->type == DPC_TYPE_F32; }

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
  const bool w = wide_backward(c);
  Split S;
  if (int rc = split_rows(c, lean_backward(c, w), S))
    return rc;
  if (!c->workspace || reinterpret_cast<uintptr_t>(c->workspace) % 256 || c->workspace_bytes < S.bytes)
    return dpc::fail(DPC_ERR_INVALID, who + ": " + std::to_string(S.bytes) +
                                          " bytes of workspace on a 256-byte boundary are needed");
  NormParams P = params(c);
  long long cycles = 0;
  if (int rc = wait_limit_now(&cycles))
    return rc;
  P.wait_kilocycles = (int)std::min<long long>(cycles / 1000 + 1, 1 << 30) * (waits.keep_back ? -1 : 1);
  P.dh = c->d_normed, P.dr = c->d_new_stream, P.dx = c->d_stream, P.dy = c->d_branch, P.dg = c->d_gate;
  P.dh_ld = c->d_normed_stride, P.dr_ld = c->d_new_stream_stride, P.dx_ld = c->d_stream_stride;
  P.dy_ld = c->d_branch_stride, P.dg_ld = c->d_gate_stride;
  P.units = (int)S.units, P.chunks = (int)S.chunks;
  P.chunks_per_group = (int)S.chunks_per_group, P.rows_per_chunk = (int)S.rows_per_chunk;
  P.sums_ld = ceil_div(c->width, 8) * 8;
  P.sums = static_cast<float*>(c->workspace);
  P.gate_sums = reinterpret_cast<float*>(static_cast<char*>(c->workspace) + S.gate_at);
  if (int rc = dispatch(stream, c->type, w, P, true, with_bias(c)))
    return rc;
  JoinParams J = {};
  J.sums = P.sums, J.gate_sums = P.gate_sums, J.units = S.units, J.width = c->width, J.ld = P.sums_ld;
  J.chunks_per_group = S.chunks_per_group, J.dg = c->d_gate, J.dg_ld = c->d_gate_stride;
  J.out[0] = c->d_pre_weight, J.out[1] = c->d_post_weight, J.out[2] = c->d_pre_bias, J.out[3] = c->d_post_bias;
  const int64_t vectors = 4 + (S.gates && c->d_gate ? c->groups : 0);
  const dim3 grid((unsigned)ceil_div(c->width, 128), (unsigned)vectors); // (groups: fewer than units there)
  if (c->type == DPC_TYPE_F32)
    norm_join_kernel<float><<<grid, 32 * kJoinWarps, 0, stream>>>(J);
  else
    norm_join_kernel<__nv_bfloat16><<<grid, 32 * kJoinWarps, 0, stream>>>(J);
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
    if (int rc = split_rows(c, lean_backward(c, wide_backward(c)), S))
      return rc;
    *bytes = S.bytes;
    return (int)DPC_OK;
  });
}

int dpc_residual_norm_backward(void* stream, const dpc_residual_norm* c)
{
  return guarded("dpc_residual_norm_backward", [&] { return backward(static_cast<cudaStream_t>(stream), c); });
}
