// Softmax cross entropy over a large vocabulary, with its gradient, in pieces of the vocabulary:
// the [rows, vocab] logits are never kept.
//
//   l[n,v] = scale * sum_k hidden[n,k] weight[v,k] + bias[v]
//   lse[n] = log sum_v exp l[n,v]          loss[n] = lse[n] - l[n, target[n]]
//   s[n,v] = g[n] / G * (exp(l[n,v] - lse[n]) - [v == target[n]])       g = dL/dloss, G = max |g|
//   d_hidden = scale G s weight      d_weight = scale G s^T hidden      d_bias = G sum_n s
//
// Forward: one product whose epilogue keeps, of every 64 columns, the maximum and the sum of the
// exponentials of a row (8 bytes instead of 64 logits), then a kernel that joins them.  Backward, for
// a piece of the vocabulary at a time: the product again with an epilogue that writes s, then
// d_hidden += s weight and d_weight = s^T hidden.  The piece bounds the memory for s (256 MB, or 2048 words where they take
// more: above 65536 rows in bf16) and the recomputed product is a quarter of the arithmetic; keeping the logits of 8192 rows x
// 128000 words in 32 bits instead would be 4.2 GB (forward's parts of them: 131 MB).
//
// One persistent kernel does all four products: 256-row tiles on CTA pairs (cta_group::2), 64-deep
// stages filled by TMA, accumulators double-buffered in tensor memory so that the epilogue warps work
// on a tile while the next one is multiplied.  A row of the vocabulary or a batch of any length is a tile
// whose outside TMA fills with zeros.
//
// bf16 tensors: tiles 256 wide.  s is rounded to bf16 (half a step, 2^-8, of each of its values): the tensor
// cores take no wider operand beside bf16 weights, and the sums over it are in 32 bits and are rounded
// to bf16 themselves.
//
// 32-bit tensors are multiplied as three bf16 planes each (24 bits: hi + mid + low, exactly) in the six products
// whose terms reach 2^-24 (what is left out is 2^-21 of a product at most, 2^-24 on average); s is held in as many planes.
// A stage holds the three planes of both operands, so that six products are made of six loads (a pass over the operands
// for each product was bound by L2: 4096 bytes a step of 256 cycles and SM).  The tensor cores truncate their 32-bit sums,
// which over the 628 additions of a contraction of 10007 left d_hidden 1.2e-5 off (2-norm; 7e-7 now); so hi x hi has an
// accumulator of its own, and a contraction is cut into runs of 8 stages (32 additions) whose sums the epilogue warps add
// up in registers, rounded to nearest.  They have registers for tiles 128 wide.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "dpc_internal.h"
#include "dpc_operators.cuh"
#include "dpc_tcgen05.cuh"

namespace
{
using namespace dpc::ptx;
using namespace dpc::ops;

constexpr int kTile = 256;       // rows of a pair's tile, and columns but for 32-bit tensors
constexpr int kRows = 128;       // rows of A that one CTA holds
constexpr int kDepth = 64;       // contraction depth of a stage: 128 bytes, one swizzle row
constexpr int kRowBytes = kDepth * 2;
constexpr int kRun = 8; // stages whose products the tensor cores add up, where the epilogue warps add the rest

enum Epilogue
{
  EPI_LSE,   // maximum and sum of exponentials of a warp's columns of a row
  EPI_SLOPE, // s of the piece, in bf16 planes
  EPI_SUM,   // 32-bit sums, added to what earlier pieces left
  EPI_OUT    // the product itself, in the type of the tensors
};

// Tiles of COLS columns: each CTA of a pair holds half of B's rows.
template <int COLS, int EPI>
struct Tile
{
  // 16 warps hide the latency of the exponentials (4096 rows x 64 against 50021 words: 124 -> 104 us, x 512: 156 -> 136); where they
  // also convert and store, or hold sums in registers, their 96 registers cost more (79 -> 89 us a piece of 25088).
  static constexpr int kEpilogueWarps = COLS == 256 && EPI == EPI_LSE ? 16 : 8;
  static constexpr int kThreads = 128 + 32 * kEpilogueWarps;

  static constexpr bool kRuns = COLS < kTile;
  static constexpr int kPlanes = kRuns ? 3 : 1; // of each operand, in a stage
  static constexpr int kABytes = kRows * kRowBytes, kBBytes = COLS / 2 * kRowBytes;
  static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
  static constexpr int kStages = kRuns ? 3 : 6;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
  static constexpr int kSets = kRuns ? 2 : 1; // accumulators of a tile: hi x hi, and the five smaller products
  static constexpr int kShare = COLS / (kEpilogueWarps / 4); // columns of an epilogue warp
};
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Bytes of slope, and of weight planes, that a piece of the vocabulary may take; but 2048 words at least, below
// which reading and writing the 32-bit sums of d_hidden again for every piece would take as long as its product.
constexpr size_t kPieceBytes = (size_t)256 << 20;
constexpr int64_t kPieceLeast = 2048;

struct GemmParams
{
  // (32 bits: divisions of 64 took longer than a tile's product where the rows are short)
  uint32_t tiles_m, tiles_n, tiles, group_m, items; // tiles = tiles_m * tiles_n, items = splits * tiles
  int splits, kblocks;
  int64_t m, n;              // rows and columns of the product
  // logits
  float factor;     // scale * log2(e)
  const void* bias; // of the piece, or NULL
  int bias_f32;
  const int64_t* targets;
  int64_t vocab, first; // first: vocabulary entry of column 0
  int64_t ignore_index;
  float2* partial; // EPI_LSE: [block of the vocabulary, a warp's columns wide][row]
  float* picked;   // EPI_LSE: logit of the target, in units of log 2
  const float* lse;
  const float* grad;
  int64_t grad_stride;
  const float* grad_top; // the largest gradient of a row's loss, which s is in units of
  float scale;
  __nv_bfloat16* slope;
  int64_t slope_ld, slope_plane;
  float* sum; // EPI_SUM
  int64_t sum_ld, sum_split;
  int add;
  void* out; // EPI_OUT
  int64_t out_ld;
  int out_f32, out_wide;
  long long wait_cycles; // limit of every wait
  int keep_back;         // the signals that a tile's sums are complete are not given: the waits for them run out
};

__device__ __forceinline__ float ex2(float x)
{
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ bool counted(int64_t target, int64_t vocab, int64_t ignore_index)
{
  return target >= 0 && target < vocab && target != ignore_index;
}

// A warp has read its accumulators: their next tile may be multiplied.  Relaxed: what was read is in registers, and
// a release would wait for the epilogue's stores as well.
__device__ __forceinline__ void accumulators_read(uint32_t bar, int lane)
{
  tc_fence_before();
  __syncwarp();
  if (lane == 0)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// 32 columns of tensor memory on their way into registers; tmem_wait ends the wait for them (the registers pass
// through it, so that nothing reads them before).
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32])
{
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
               "[%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                 "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32])
{
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// Element i of lane l becomes element l of lane i: five rounds that exchange halves of ever smaller blocks.
__device__ __forceinline__ void transpose32(float (&v)[32], int lane)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
  {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if ((i & o) == 0)
      {
        const float give = upper ? v[i] : v[i + o];
        const float got = __shfl_xor_sync(0xffffffffu, give, o);
        if (upper)
          v[i] = got;
        else
          v[i + o] = got;
      }
  }
}

// Which tile a work item is: the tiles of `group_m` row blocks go down the rows first, so that the
// CTA pairs at work share a few column blocks (weights, read once) and the rows of the group stay in L2.
__device__ __forceinline__ void locate(const GemmParams& P, uint32_t item, int& split, uint32_t& tm, uint32_t& tn)
{
  split = P.splits == 1 ? 0 : (int)(item / P.tiles);
  const uint32_t tile = item - split * P.tiles;
  const uint32_t group = P.tiles_m == P.group_m ? 0 : tile / (P.group_m * P.tiles_n);
  const uint32_t first = group * P.group_m, rest = tile - first * P.tiles_n;
  const uint32_t height = min(P.tiles_m - first, P.group_m);
  tn = rest / height;
  tm = first + rest - tn * height;
}

__device__ __forceinline__ void range_of(const GemmParams& P, int split, int& begin, int& end)
{
  begin = 0, end = P.kblocks;
  if (P.splits > 1)
    begin = (int)((int64_t)P.kblocks * split / P.splits), end = (int)((int64_t)P.kblocks * (split + 1) / P.splits);
}

// The three bf16 planes of a float (in the upper halves of words), by truncation: 8 bits each, their sum is the float
// itself, also where it is above the largest bf16, and they have its sign.  Infinities and NaN are that in every plane, and a
// plane with nothing left holds the float times 2^-32.  So every plane of a number times an infinity is an infinity of the same
// sign, and the six products add up to what the definition gives.  (Planes rounded to nearest have zeros and signs of their
// own, and inf - inf as the second plane of an infinity.  Numbers below 2^-94 have zeros here too: NaN beside an infinity.)
__device__ __forceinline__ void planes_of(float x, uint32_t (&p)[3])
{
  const uint32_t bits = __float_as_uint(x);
  const float small = x * 2.3283064365386963e-10f; // 2^-32
  p[0] = bits;
  float rest = x - __uint_as_float(bits & 0xffff0000u);
  p[1] = __float_as_uint(rest == 0.0f ? small : rest);
  rest -= __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
  p[2] = __float_as_uint(rest == 0.0f ? small : rest);
  if ((bits & 0x7f800000u) == 0x7f800000u)
    p[0] = p[1] = p[2] = bits & 0x007fffffu ? 0x7fc00000u : bits;
}

// Words of neighbours in bf16, one of each plane.
__device__ __forceinline__ void planes_of(float a, float b, uint32_t& w0, uint32_t& w1, uint32_t& w2)
{
  uint32_t p[3], q[3];
  planes_of(a, p), planes_of(b, q);
  w0 = __byte_perm(p[0], q[0], 0x7632), w1 = __byte_perm(p[1], q[1], 0x7632), w2 = __byte_perm(p[2], q[2], 0x7632);
}

// 32 logits of a row in units of log 2, -inf outside the vocabulary.
__device__ __forceinline__ void logits32(const GemmParams& P, int64_t col, float (&v)[32])
{
  if (P.bias)
  {
#pragma unroll
    for (int i = 0; i < 32; ++i)
    {
      const int64_t c = col + i < P.n ? col + i : P.n - 1;
      const float b = P.bias_f32 ? __ldg(static_cast<const float*>(P.bias) + c)
                                 : __bfloat162float(static_cast<const __nv_bfloat16*>(P.bias)[c]);
      v[i] = fmaf(v[i], P.factor, b * kLog2e);
    }
  }
  else
  {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] *= P.factor;
  }
  if (col + 32 > P.n)
  {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (col + i >= P.n)
        v[i] = -INFINITY;
  }
}

template <int EPI, bool A_MN, bool B_MN, int COLS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Tile<COLS, EPI>::kThreads, 1)
    vocab_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const GemmParams P)
{
  using C = Tile<COLS, EPI>;
  constexpr int kStages = C::kStages, kStageBytes = C::kStageBytes;
  constexpr uint32_t kTmemColumns = 2 * C::kSets * COLS;
  constexpr uint32_t kInstr = (1u << 4) | (1u << 7) | (1u << 10) | ((A_MN ? 1u : 0u) << 15) |
                              ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(COLS >> 3) << 17) |
                              ((uint32_t)(kTile >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + kStages * kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t begin = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0)
  {
    for (int s = 0; s < kStages; ++s)
    {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a)
    {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * C::kEpilogueWarps); // both CTAs' epilogue warps arrive on the leader's
    }
    *abort_flag = 0;
    *reinterpret_cast<volatile long long*>(abort_flag + 2) = P.wait_cycles;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1)
  {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync_all(); // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint32_t lead_full = mapa_u32(smem_u32(full), 0);
  const uint32_t lead_tempty = mapa_u32(smem_u32(tempty), 0);
  const uint32_t peer_empty = mapa_u32(smem_u32(empty), rank ^ 1);
  const uint32_t peer_tfull = mapa_u32(smem_u32(tfull), rank ^ 1);

  if (warp == 0)
  {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0)
    {
      int s = 0;
      uint32_t phase = 1;
      bool alive = true;
      for (uint32_t item = begin; item < P.items && alive; item += step)
      {
        int split, it, it_end;
        uint32_t tm, tn;
        locate(P, item, split, tm, tn);
        range_of(P, split, it, it_end);
        const int m0 = (int)(tm * kTile) + (int)rank * kRows, n0 = (int)(tn * COLS) + (int)rank * (COLS / 2);
        for (; it < it_end; ++it)
        {
          if (!mbar_wait_cluster(&empty[s], phase, abort_flag))
          {
            alive = false;
            break;
          }
          if (leader)
            mbar_expect_tx(&full[s], 2 * kStageBytes); // both CTAs' copies count on the leader's barrier
          const uint32_t bar = lead_full + (uint32_t)(s * 8);
          uint8_t* a = stages + s * kStageBytes;
          uint8_t* b = a + C::kPlanes * C::kABytes;
          const int k = it * kDepth;
#pragma unroll
          for (int pl = 0; pl < C::kPlanes; ++pl, a += C::kABytes, b += C::kBBytes)
          {
            if (A_MN)
            {
              tma_load_3d_pair(a, &map_a, bar, m0, k, pl);
              tma_load_3d_pair(a + 64 * kRowBytes, &map_a, bar, m0 + 64, k, pl);
            }
            else
              tma_load_3d_pair(a, &map_a, bar, k, m0, pl);
            tma_load_3d_pair(b, &map_b, bar, B_MN ? n0 : k, B_MN ? k : n0, pl);
            if (B_MN && COLS == 256)
              tma_load_3d_pair(b + 64 * kRowBytes, &map_b, bar, n0 + 64, k, pl);
          }
          if (++s == kStages)
            s = 0, phase ^= 1;
        }
      }
    }
  }
  else if (warp == 1)
  {
    // ---------------------------------------------------------------- MMA issuer (the warp together, one lane issues)
    if (leader)
    {
      // K-major: rows of 128 bytes, 8 to a swizzle atom.  MN-major: blocks of 64 columns (8 KB apart) of
      // 64 k-rows, 8 k-rows to an atom, 16 k-rows to an instruction.
      const uint64_t da0 = make_desc(smem_u32(stages), A_MN ? 64 * kRowBytes : 16, 1024, 2);
      const uint64_t db0 = make_desc(smem_u32(stages) + C::kPlanes * C::kABytes, B_MN ? 64 * kRowBytes : 16, 1024, 2);
      constexpr uint32_t adv_a = (A_MN ? 2048 : 32) >> 4, adv_b = (B_MN ? 2048 : 32) >> 4;
      int s = 0, turn = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (uint32_t item = begin; item < P.items && alive; item += step)
      {
        int it, it_end;
        range_of(P, P.splits == 1 ? 0 : (int)(item / P.tiles), it, it_end);
        while (it < it_end && alive)
        {
          const int run_end = C::kRuns && it + kRun < it_end ? it + kRun : it_end;
          const int acc = turn & 1;
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(&tempty[acc], ((turn >> 1) & 1) ^ 1, abort_flag)))
          {
            alive = false;
            break;
          }
          ++turn;
          tc_fence_after();
          const uint32_t d = tmem_base + acc * (C::kSets * COLS);
          for (uint32_t more = 0; it < run_end; ++it)
          {
            if (!__all_sync(0xffffffffu, mbar_wait_cluster(&full[s], phase, abort_flag)))
            {
              alive = false;
              break;
            }
            tc_fence_after();
            const uint64_t sa = da0 + (uint64_t)(s * (kStageBytes >> 4)), sb = db0 + (uint64_t)(s * (kStageBytes >> 4));
#pragma unroll
            for (int ks = 0; ks < kDepth / 16; ++ks)
            {
              const uint64_t a = sa + (uint64_t)(ks * adv_a), b = sb + (uint64_t)(ks * adv_b);
              if (C::kRuns)
              {
                constexpr uint64_t pa = C::kABytes >> 4, pb = C::kBBytes >> 4; // from plane to plane
                tc_mma_bf16_pair(d + COLS, a + 2 * pa, b, kInstr, more);
                tc_mma_bf16_pair(d + COLS, a, b + 2 * pb, kInstr, 1);
                tc_mma_bf16_pair(d + COLS, a + pa, b + pb, kInstr, 1);
                tc_mma_bf16_pair(d + COLS, a + pa, b, kInstr, 1);
                tc_mma_bf16_pair(d + COLS, a, b + pb, kInstr, 1);
              }
              tc_mma_bf16_pair(d, a, b, kInstr, more);
              more = 1;
            }
            tc_commit_pair(smem_u32(&empty[s])); // the stage is free in both CTAs
            tc_commit_pair(peer_empty + (uint32_t)(s * 8));
            if (++s == kStages)
              s = 0, phase ^= 1;
          }
          if (alive && !P.keep_back)
          {
            tc_commit_pair(smem_u32(&tfull[acc]));
            tc_commit_pair(peer_tfull + (uint32_t)(acc * 8));
          }
        }
      }
    }
  }
  else if (warp >= 4)
  {
    // ---------------------------------------------------------------- epilogue: a row a lane, kShare columns a warp
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    int turn = 0;
    bool alive = true; // a wait gave up: everything from then on is NaN
    for (uint32_t item = begin; item < P.items; item += step)
    {
      int split;
      uint32_t tm, tn;
      locate(P, item, split, tm, tn);
      const int64_t row = (int64_t)tm * kTile + rank * kRows + quarter * 32 + lane;
      const int64_t col0 = (int64_t)tn * COLS + part * C::kShare;
      const bool inside = row < P.m;
      int64_t target = -1; // column of the target, outside the tile: not this one
      bool count = false;
      float lse2 = 0.0f, slope_scale = 0.0f;
      if ((EPI == EPI_LSE || EPI == EPI_SLOPE) && inside)
      {
        const int64_t t = __ldg(P.targets + row);
        if (EPI == EPI_SLOPE) // (of rows that do not count as well: the loads go out together)
        {
          lse2 = __ldg(P.lse + row) * kLog2e;
          slope_scale = __fdiv_rn(__ldg(P.grad + row * P.grad_stride), __ldg(P.grad_top));
        }
        count = counted(t, P.vocab, P.ignore_index);
        if (count)
          target = t - P.first;
      }
      int it, it_end;
      range_of(P, split, it, it_end);
      float sums[C::kRuns ? C::kShare / 32 : 1][32];
      // all of the warp's rows are behind the last: nothing is read or computed (where sums take no registers: with them
      // the second way through spilled 150 bytes)
      const bool idle = !C::kRuns && row - lane >= P.m;
      const bool several = it + kRun < it_end;
      if (C::kRuns)
      {
        // the runs but the last, which the loop below adds
        for (bool first = true; alive && it + kRun < it_end; it += kRun, ++turn, first = false)
        {
          const int acc = turn & 1;
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(&tfull[acc], (turn >> 1) & 1, abort_flag)))
          {
            alive = false;
            break;
          }
          tc_fence_after();
          const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (C::kSets * COLS) + part * C::kShare;
#pragma unroll
          for (int c = 0; c < C::kShare / 32; ++c)
          {
            float v[32];
            __syncwarp();
            tc_ld32(taddr + 32 * c, v);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              sums[C::kRuns ? c : 0][i] = first ? v[i] : sums[C::kRuns ? c : 0][i] + v[i];
            tc_ld32(taddr + COLS + 32 * c, v);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              sums[C::kRuns ? c : 0][i] += v[i];
          }
          accumulators_read(lead_tempty + (uint32_t)(acc * 8), lane);
        }
      }
      const int acc = turn & 1;
      if (alive)
        alive = __all_sync(0xffffffffu, mbar_wait_cluster(&tfull[acc], (turn >> 1) & 1, abort_flag));
      ++turn;
      tc_fence_after();
      if (idle)
      {
        if (alive)
          accumulators_read(lead_tempty + (uint32_t)(acc * 8), lane);
        continue;
      }
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (C::kSets * COLS) + part * C::kShare;
      if ((EPI == EPI_LSE || EPI == EPI_SLOPE) && item + step < P.items)
      {
        // the next tile's targets come into L1 while this one is worked on
        int s;
        uint32_t m, n;
        locate(P, item + step, s, m, n);
        const int64_t next = (int64_t)m * kTile + rank * kRows + quarter * 32 + lane;
        if (next < P.m)
        {
          asm volatile("prefetch.global.L1 [%0];" ::"l"(P.targets + next));
          if (EPI == EPI_SLOPE)
          {
            asm volatile("prefetch.global.L1 [%0];" ::"l"(P.lse + next));
            asm volatile("prefetch.global.L1 [%0];" ::"l"(P.grad + next * P.grad_stride));
          }
        }
      }
      const float out_factor = EPI == EPI_OUT ? __ldg(P.grad_top) * P.scale : 1.0f;
      float top = -INFINITY, total = 0.0f;
      uint32_t raw[C::kRuns ? 1 : 2][32];
      __syncwarp();
      if (!C::kRuns)
        tmem_load(taddr, raw[0]); // (whatever is there, after a wait that gave up)
#pragma unroll
      for (int c = 0; c < C::kShare / 32; ++c)
      {
        const int64_t col = col0 + 32 * c;
        float v[32];
        __syncwarp();
        if (C::kRuns)
        {
          float w[32];
          tc_ld32(taddr + 32 * c, v);
          tc_ld32(taddr + COLS + 32 * c, w);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            v[i] += several ? sums[C::kRuns ? c : 0][i] + w[i] : w[i];
        }
        else
        {
          // the next columns come while these are worked on
          uint32_t(&now)[32] = raw[C::kRuns ? 0 : c & 1];
          tmem_wait(now);
          if (c + 1 < C::kShare / 32)
            tmem_load(taddr + 32 * (c + 1), raw[C::kRuns ? 0 : (c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            v[i] = __uint_as_float(now[i]);
        }
        if (c + 1 == C::kShare / 32 && alive) // (a warp that gave up hands nothing back: the multiplications end too)
          accumulators_read(lead_tempty + (uint32_t)(acc * 8), lane);
        if (!alive)
        {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            v[i] = NAN;
        }
        // logits are factor * v, in units of log 2
        float factor = P.factor;
        if ((EPI == EPI_LSE || EPI == EPI_SLOPE) && (P.bias || col + 32 > P.n))
        {
          logits32(P, col, v);
          factor = 1.0f;
        }
        const int hot = target >= col && target < col + 32 ? (int)(target - col) : -1;
        if (EPI == EPI_LSE)
        {
          if (hot >= 0)
          {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == hot)
                P.picked[row] = v[i] * factor;
          }
          float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int i = 4; i < 32; ++i)
            most[i & 3] = fmaxf(most[i & 3], v[i]);
          const float high = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * factor, top);
          // (nothing but -inf so far: zero in its place leaves the sum at 0, or NaN where a logit is NaN)
          const float base = high == -INFINITY ? 0.0f : high;
          float2x sum[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 32; i += 2)
          {
            const float2 e = halves(fma2(pair(v[i], v[i + 1]), pair(factor), pair(-base)));
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pair(ex2(e.x), ex2(e.y)));
          }
          const float2 all = halves(add2(sum[0], sum[1]));
          total = fmaf(total, ex2(top - base), all.x + all.y);
          top = high;
        }
        else if (EPI == EPI_SLOPE)
        {
          // (past the last column of the piece: exp(-inf) = 0 is written, and nothing reads it)
#pragma unroll
          for (int i = 0; i < 32; i += 2)
          {
            const float2 e = halves(fma2(pair(v[i], v[i + 1]), pair(factor), pair(-lse2)));
            v[i] = ex2(e.x), v[i + 1] = ex2(e.y);
          }
          if (hot >= 0)
          {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              v[i] -= i == hot ? 1.0f : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i)
            v[i] = count ? slope_scale * v[i] : 0.0f; // an ignored row is 0 whatever it holds
          if (inside)
          {
            __nv_bfloat16* dst = P.slope + row * P.slope_ld + col;
#pragma unroll
            for (int i = 0; i < 32; i += 16)
            {
              uint32_t w[C::kPlanes][8];
#pragma unroll
              for (int k = 0; k < 8; ++k)
              {
                if constexpr (C::kPlanes == 3)
                  planes_of(v[i + 2 * k], v[i + 2 * k + 1], w[0][k], w[1][k], w[2][k]);
                else
                {
                  const __nv_bfloat162 h = __floats2bfloat162_rn(v[i + 2 * k], v[i + 2 * k + 1]);
                  w[0][k] = *reinterpret_cast<const uint32_t*>(&h);
                }
              }
#pragma unroll
              for (int pl = 0; pl < C::kPlanes; ++pl)
                st8(reinterpret_cast<float*>(dst + pl * P.slope_plane + i), reinterpret_cast<const float*>(w[pl]));
            }
          }
        }
        else if (EPI == EPI_SUM)
        {
          if (inside)
          {
            float* dst = P.sum + split * P.sum_split + row * P.sum_ld + col;
            if (P.add)
            {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
              {
                float old[8];
                ld8(dst + i, old);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  v[i + k] += old[k];
              }
            }
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              st8(dst + i, v + i);
          }
        }
        else if (col < P.n)
        {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            v[i] *= out_factor;
          if (P.out_wide && col + 32 <= P.n)
          {
            if (inside && P.out_f32)
            {
              float4* dst = reinterpret_cast<float4*>(static_cast<float*>(P.out) + row * P.out_ld + col);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                dst[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
            else if (inside)
            {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(P.out) + row * P.out_ld + col);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                dst[i] = pack8(v + 8 * i);
            }
          }
          else
          {
            // neighbouring lanes write neighbours (a row a lane, element by element: 930 us instead of 89 for 100000 x
            // 1021 in bf16)
            transpose32(v, lane);
            const int64_t row0 = row - lane;
#pragma unroll
            for (int r = 0; r < 32; ++r)
              if (row0 + r < P.m && col + lane < P.n)
              {
                if (P.out_f32)
                  static_cast<float*>(P.out)[(row0 + r) * P.out_ld + col + lane] = v[r];
                else
                  static_cast<__nv_bfloat16*>(P.out)[(row0 + r) * P.out_ld + col + lane] = __float2bfloat16_rn(v[r]);
              }
          }
        }
      }
      if (EPI == EPI_LSE && inside)
        P.partial[((P.first + col0) / C::kShare) * P.m + row] = make_float2(top, total);
    }
  }

  // ------------------------------------------------------------------ teardown
  // A wait gave up: what is under way (copies into this CTA's shared memory, multiplications that read it) ends before
  // the pair leaves.  Every wait that does not come true reaches the epilogue warps of both CTAs, whichever warp gave up first, and
  // the pair leaves together: it is enough that the warps of a CTA that see its flag stay.
  if (*abort_flag)
  {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL * kStages)
    {
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all(); // neither CTA leaves while the other may still touch its memory
  if (warp == 1)
  {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns)
                 : "memory");
  }
}

// The parts of few rows without tensor cores: a tile of 256 rows would be all but empty, and the weights, read once,
// are the whole cost (65 MB for 32000 words x 1024 in bf16: 10 us at the rate of a copy).  The rows lie in shared
// memory in 32 bits; a warp multiplies them with kWords words at a time, 8 elements a lane and word, and keeps the
// maximum and the sum of exponentials of what it has seen.  ROWS: rows, rounded up.  WIDE: 16-byte loads of the weights.
// 32000 words x 1024, 1 / 2 / 4 / 8 rows: bf16 17 / 19 / 40 / 40 us where the tensor cores take 24, f32 24 / 26 / 31 / 43
// us where they take 128 (52 of them for the planes): hence up to 2 and up to 8 rows.  With widths of 256 to 4096, 4000 to 128000
// words and weights off 16 bytes (1021 columns) 3 rows on the tensor cores take 1.1 to 2.5 times as long as 2 here in bf16 (128000 x 256
// alone: 30 us against 32), 9 rows 1.6 to 3.7 times as long as 8 in f32.
template <typename T>
constexpr int kFewRows = sizeof(T) == 2 ? 2 : 8;
constexpr int kWords = 4, kFewThreads = 256;
constexpr size_t kFewBytes = 96 << 10; // shared memory for the rows: two blocks an SM

template <typename T, int ROWS, bool WIDE>
__global__ void __launch_bounds__(kFewThreads, ROWS > 4 ? 1 : 2)
    vocab_few_kernel(const T* __restrict__ hidden, int64_t hidden_ld, const T* __restrict__ weight, int64_t weight_ld,
                     int rows, int width, int64_t vocab, const T* __restrict__ bias, float factor,
                     const int64_t* __restrict__ targets, int64_t ignore_index, float2* __restrict__ partial,
                     float* __restrict__ picked)
{
  extern __shared__ __align__(16) float held[]; // [rows][chunks of 256]
  __shared__ float2 parts[kFewThreads / 32][ROWS];
  const int chunks = (width + 255) / 256, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Element k of a row: chunk k / 256; WIDE: lane (k / 8) % 32, its first four and its last four apart, so that
  // the lanes' 16-byte reads meet no bank twice; otherwise in order.
  for (int r = 0; r < ROWS; ++r)
    for (int k = threadIdx.x; k < chunks * 256; k += kFewThreads)
    {
      const int at = WIDE ? (k & ~255) + ((k >> 2) & 1) * 128 + ((k >> 3) & 31) * 4 + (k & 3) : k;
      held[r * chunks * 256 + at] = r < rows && k < width ? to_float(hidden[r * hidden_ld + k]) : 0.0f;
    }
  float top[ROWS], total[ROWS];
  int target[ROWS]; // (2^28 words at most)
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
  {
    top[r] = -INFINITY, total[r] = 0.0f, target[r] = -1;
    if (r < rows && counted(targets[r], vocab, ignore_index))
      target[r] = (int)targets[r];
  }
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * (kFewThreads / 32) * kWords;
  for (int64_t word = ((int64_t)blockIdx.x * (kFewThreads / 32) + warp) * kWords; word < vocab; word += step)
  {
    float2x sum[kWords][ROWS] = {};
#pragma unroll 2
    for (int c = 0; c < chunks; ++c)
    {
      float2x w[kWords][4];
#pragma unroll
      for (int j = 0; j < kWords; ++j)
      {
        const T* p = weight + (word + j < vocab ? word + j : vocab - 1) * weight_ld; // (a word behind the last: not used)
        float v[8];
        if constexpr (WIDE)
        {
          const int k = c * 256 + lane * 8;
          if (k < width)
            load8w(p + k, v);
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
            const int k = c * 256 + i * 32 + lane;
            v[i] = k < width ? to_float(p[k]) : 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[j][i] = pair(v[2 * i], v[2 * i + 1]);
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
      {
        const float* x = held + (r * chunks + c) * 256;
        float2x h[4];
        if constexpr (WIDE)
        {
          const float4 a = *reinterpret_cast<const float4*>(x + lane * 4), b = *reinterpret_cast<const float4*>(x + 128 + lane * 4);
          h[0] = pair(a.x, a.y), h[1] = pair(a.z, a.w), h[2] = pair(b.x, b.y), h[3] = pair(b.z, b.w);
        }
        else
        {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            h[i] = pair(x[i * 64 + lane], x[i * 64 + 32 + lane]);
        }
#pragma unroll
        for (int j = 0; j < kWords; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sum[j][r] = fma2(w[j][i], h[i], sum[j][r]);
      }
    }
#pragma unroll
    for (int j = 0; j < kWords; ++j)
    {
      if (word + j >= vocab)
        break;
      const float b = bias ? to_float(bias[word + j]) * kLog2e : 0.0f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
      {
        const float2 both = halves(sum[j][r]);
        float l = both.x + both.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          l += __shfl_xor_sync(0xffffffffu, l, o);
        l = bias ? fmaf(l, factor, b) : l * factor;
        if (word + j == target[r] && lane == 0)
          picked[r] = l;
        // (nothing but -inf so far: zero in its place leaves the sum at 0, or NaN where a logit is NaN)
        const float most = fmaxf(top[r], l), base = most == -INFINITY ? 0.0f : most;
        total[r] = fmaf(total[r], ex2(top[r] - base), ex2(l - base));
        top[r] = most;
      }
    }
  }
  if (lane == 0)
  {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      parts[warp][r] = make_float2(top[r], total[r]);
  }
  __syncthreads();
  if ((int)threadIdx.x < rows)
  {
    float most = -INFINITY, all = 0.0f;
    for (int w = 0; w < kFewThreads / 32; ++w)
      most = fmaxf(most, parts[w][threadIdx.x].x);
    const float base = most == -INFINITY ? 0.0f : most;
    for (int w = 0; w < kFewThreads / 32; ++w)
      all = fmaf(parts[w][threadIdx.x].y, ex2(parts[w][threadIdx.x].x - base), all);
    partial[(int64_t)blockIdx.x * rows + threadIdx.x] = make_float2(most, all);
  }
}

// lse and loss of every row from the parts.  A block joins `lanes` threads on each of 256 / lanes rows:
// neighbouring threads read neighbouring rows of a part, and with few rows neighbouring parts.
__global__ void __launch_bounds__(256) vocab_join_kernel(const float2* __restrict__ partial, int64_t parts, int64_t rows,
                                                         int row_shift, const float* __restrict__ picked,
                                                         const int64_t* __restrict__ targets, int64_t vocab,
                                                         int64_t ignore_index, float* __restrict__ loss, float* __restrict__ lse)
{
  __shared__ float tops[256], sums[256];
  const int per = 1 << row_shift, r = threadIdx.x & (per - 1), lanes = 256 >> row_shift;
  const int64_t row = ((int64_t)blockIdx.x << row_shift) + r;
  float top = -INFINITY, total = 0.0f;
  if (row < rows)
    for (int64_t p = threadIdx.x >> row_shift; p < parts; p += lanes)
    {
      const float2 v = partial[p * rows + row];
      const float most = fmaxf(top, v.x), base = most == -INFINITY ? 0.0f : most;
      total = total * ex2(top - base) + v.y * ex2(v.x - base);
      top = most;
    }
  tops[threadIdx.x] = top, sums[threadIdx.x] = total;
  __syncthreads();
  for (int half = lanes >> 1; half > 0; half >>= 1)
  {
    if ((int)(threadIdx.x >> row_shift) < half)
    {
      const int other = threadIdx.x + (half << row_shift);
      const float a = tops[threadIdx.x], b = tops[other], most = fmaxf(a, b), base = most == -INFINITY ? 0.0f : most;
      sums[threadIdx.x] = sums[threadIdx.x] * ex2(a - base) + sums[other] * ex2(b - base);
      tops[threadIdx.x] = most;
    }
    __syncthreads();
  }
  if ((int)threadIdx.x < per && row < rows)
  {
    const bool count = counted(targets[row], vocab, ignore_index);
    const float l = tops[r] + log2f(sums[r]), d = l - (count ? picked[row] : 0.0f);
    lse[row] = count ? l * kLn2 : 0.0f;
    loss[row] = count ? d * kLn2 : 0.0f;
  }
}

// dst[plane][row][0..ld) = src[row][0..cols) in bf16, or its three planes, zeros beyond; rows that do not count are zeros.
template <typename T>
__global__ void __launch_bounds__(256) vocab_planes_kernel(const T* __restrict__ src, int64_t src_ld, int64_t rows,
                                                           int64_t cols, __nv_bfloat16* __restrict__ dst, int64_t ld,
                                                           const int64_t* __restrict__ targets, int64_t vocab,
                                                           int64_t ignore_index)
{
  const int64_t chunks = ld / 8, total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256)
  {
    const int64_t row = i / chunks, col = (i - row * chunks) * 8;
    float v[8];
    const bool keep = !targets || counted(targets[row], vocab, ignore_index);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = keep && col + k < cols ? to_float(src[row * src_ld + col + k]) : 0.0f;
    __nv_bfloat16* to = dst + row * ld + col;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint4*>(to) = pack8(v); // (the values themselves)
    else
    {
      uint32_t w[3][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        planes_of(v[2 * k], v[2 * k + 1], w[0][k], w[1][k], w[2][k]);
#pragma unroll
      for (int pl = 0; pl < 3; ++pl)
        *reinterpret_cast<uint4*>(to + pl * rows * ld) = make_uint4(w[pl][0], w[pl][1], w[pl][2], w[pl][3]);
    }
  }
}

// The largest |g| of the rows that count: s is held in units of it, so that in a mean over the rows (all g
// alike) the -1 of a target is exactly -1 in bf16 and not a rounded 1/rows, whose error all rows would share.  1
// where it is 0 or no number.
__global__ void __launch_bounds__(1024) vocab_gradient_kernel(const float* __restrict__ grad, int64_t stride,
                                                              const int64_t* __restrict__ targets, int64_t rows,
                                                              int64_t vocab, int64_t ignore_index, float* __restrict__ top)
{
  __shared__ float tops[32];
  float most = 0.0f;
  bool bad = false;
  for (int64_t row = threadIdx.x; row < rows; row += 1024)
    if (counted(targets[row], vocab, ignore_index))
    {
      const float g = fabsf(grad[row * stride]);
      most = fmaxf(most, g), bad |= !(g < INFINITY);
    }
  if (bad)
    most = INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0)
    tops[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x < 32)
  {
    most = tops[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (threadIdx.x == 0)
      *top = most > 0.0f && most < INFINITY ? most : 1.0f;
  }
}

// out[row][col] = factor * the sum of the splits' sums, in the type of the tensors; 0 in rows that do not count, whose slope of
// 0 the tensor cores have multiplied with whatever the weights hold (0 times an infinity).
template <typename T>
__global__ void __launch_bounds__(256) vocab_sum_kernel(const float* __restrict__ sum, int64_t ld, int64_t split_stride,
                                                        int splits, int64_t rows, int64_t cols, T* __restrict__ out,
                                                        int64_t out_ld, const float* __restrict__ grad_top, float scale,
                                                        const int64_t* __restrict__ targets, int64_t vocab, int64_t ignore_index)
{
  const float factor = *grad_top * scale;
  const int64_t chunks = (cols + 3) / 4, total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256)
  {
    const int64_t row = i / chunks, col = (i - row * chunks) * 4;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < splits; ++s)
    {
      const float4 w = *reinterpret_cast<const float4*>(sum + s * split_stride + row * ld + col);
      v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    const bool keep = counted(targets[row], vocab, ignore_index);
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < cols)
        out[row * out_ld + col + k] = from_float<T>(keep ? f[k] * factor : 0.0f);
  }
}

// sums[part][col] = sum of slope over the planes and a part of the rows: 256 columns and a part a block, 8 columns a
// lane, rows in a fixed order.  (With 64 columns and all rows a block the loads under way were too few: 32 us where
// this and the kernel below take 15, for 777 rows of 10007 in three planes.)
constexpr int kColumnParts = 16;

template <int PLANES>
__global__ void __launch_bounds__(256) vocab_columns_kernel(const __nv_bfloat16* __restrict__ slope, int64_t ld,
                                                           int64_t plane, int64_t rows, float* __restrict__ sums)
{
  __shared__ float parts[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = (int64_t)blockIdx.x * 256 + 8 * lane; // (ld is a multiple of 256: always inside a row)
  const int64_t begin = rows * blockIdx.y / gridDim.y, end = rows * (blockIdx.y + 1) / gridDim.y;
  float total[8] = {};
#pragma unroll 4
  for (int64_t row = begin + warp; row < end; row += 8)
#pragma unroll
    for (int pl = PLANES - 1; pl >= 0; --pl)
    {
      float v[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(slope + pl * plane + row * ld + col)), v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        total[i] += v[i];
    }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    parts[warp][8 * lane + i] = total[i];
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w)
    s += parts[w][threadIdx.x];
  sums[blockIdx.y * ld + (int64_t)blockIdx.x * 256 + threadIdx.x] = s;
}

// out[col] = *factor * the sum of the parts
template <typename T>
__global__ void __launch_bounds__(256) vocab_columns_join_kernel(const float* __restrict__ sums, int64_t ld, int parts,
                                                                int64_t cols, const float* __restrict__ factor,
                                                                T* __restrict__ out)
{
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= cols)
    return;
  float s = 0.0f;
  for (int p = 0; p < parts; ++p)
    s += sums[p * ld + col];
  out[col] = from_float<T>(s * *factor);
}

// ------------------------------------------------------------------------------ host
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// bf16 operand [planes][rows][cols] in 128-byte swizzled boxes of 64 columns.
int operand_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t ld, int planes, int64_t plane,
                int box_rows)
{
  EncodeTiledFn fn = encode_fn();
  if (!fn)
    return dpc::fail(DPC_ERR_CUDA, "vocabulary loss: the driver has no tensor-map encoder");
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
  cuuint32_t box[3] = {kDepth, (cuuint32_t)box_rows, 1}, unit[3] = {1, 1, 1};
  if (fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, unit,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return dpc::fail(DPC_ERR_CUDA, "vocabulary loss: the driver refused a tensor map");
  return DPC_OK;
}

// One operand of a product: a matrix of bf16 planes with the contraction along its columns (K-major)
// or along its rows.
struct Operand
{
  const void* base;
  int64_t cols, rows, ld, plane;
};

template <int EPI, bool A_MN, bool B_MN, int COLS>
int product(cudaStream_t stream, int pairs, const Operand& a, const Operand& b, int planes, int64_t m, int64_t n,
            int64_t contraction, GemmParams P)
{
  using C = Tile<COLS, EPI>;
  CUtensorMap map_a, map_b;
  if (int rc = operand_map(&map_a, a.base, a.cols, a.rows, a.ld, planes, a.plane, A_MN ? kDepth : kRows))
    return rc;
  if (int rc = operand_map(&map_b, b.base, b.cols, b.rows, b.ld, planes, b.plane, B_MN ? kDepth : COLS / 2))
    return rc;
  P.m = m, P.n = n;
  P.kblocks = (int)ceil_div(contraction, kDepth);
  P.splits = std::min(P.splits, P.kblocks);
  const int64_t tiles_m = ceil_div(m, kTile), tiles_n = ceil_div(n, COLS);
  if (tiles_m * tiles_n > ((int64_t)1 << 30) / P.splits)
    return dpc::fail(DPC_ERR_TOO_LARGE, "vocabulary loss: more than 2^30 tiles of 256 rows and 128 or 256 columns");
  P.tiles_m = (uint32_t)tiles_m, P.tiles_n = (uint32_t)tiles_n, P.tiles = P.tiles_m * P.tiles_n;
  P.group_m = std::min<uint32_t>(P.tiles_m, 32);
  P.items = P.tiles * P.splits;
  auto kernel = vocab_product_kernel<EPI, A_MN, B_MN, COLS>;
  DPC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
  const int blocks = 2 * (int)std::min<int64_t>(P.items, pairs);
  kernel<<<blocks, C::kThreads, C::kSmemBytes, stream>>>(map_a, map_b, P);
  return launched("vocab_product_kernel");
}

// Tiles 128 wide, and sums in runs, for 32-bit tensors.
template <int EPI, bool A_MN, bool B_MN>
int product(cudaStream_t stream, int pairs, const Operand& a, const Operand& b, int planes, int64_t m, int64_t n,
            int64_t contraction, const GemmParams& P)
{
  return planes == 3 ? product<EPI, A_MN, B_MN, 128>(stream, pairs, a, b, planes, m, n, contraction, P)
                     : product<EPI, A_MN, B_MN, 256>(stream, pairs, a, b, planes, m, n, contraction, P);
}

struct Layout
{
  int pairs = 0, planes = 1, splits = 1;
  bool copy_hidden = false, copy_weight = false;
  int few = 0;       // blocks of the kernel for few rows
  int64_t cols = 0;  // columns of a tile
  int64_t share = 0; // columns of a partial sum of exponentials
  int64_t parts = 0; // partial sums of a row
  int64_t kp = 0;    // columns of the copies
  int64_t ks = 0;    // columns of the sums of d_hidden
  int64_t piece = 0; // vocabulary entries at a time, a multiple of the tile (or all of them)
  int column_parts = 1; // of the rows, in the sums of a bias gradient
  long long wait_cycles = 0;
  size_t grad_top = 0, columns = 0, hidden = 0, weight = 0, slope = 0, sum = 0, partial = 0, picked = 0, bytes = 0;
};

bool tma_ready(const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

int check(const dpc_vocab_ce* c, bool backward, const char* who)
{
  const std::string name = who;
  if (!c)
    return dpc::fail(DPC_ERR_INVALID, name + ": no description");
  if (c->type != DPC_TYPE_F32 && c->type != DPC_TYPE_BF16)
    return dpc::fail(DPC_ERR_INVALID, name + ": type is neither DPC_TYPE_F32 nor DPC_TYPE_BF16");
  if (c->rows < 0 || c->width < 1 || c->vocab < 1)
    return dpc::fail(DPC_ERR_INVALID, name + ": rows >= 0, width >= 1 and vocab >= 1 are needed");
  const int64_t most = (int64_t)1 << 28;
  if (c->rows > most || c->width > most || c->vocab > most)
    return dpc::fail(DPC_ERR_TOO_LARGE, name + ": rows, width and vocab may be 2^28 at most");
  if (c->hidden_stride < c->width || c->weight_stride < c->width || c->hidden_stride > most || c->weight_stride > most)
    return dpc::fail(DPC_ERR_INVALID, name + ": a row stride is smaller than the width (or above 2^28)");
  if (!(c->scale > 0.0f) || !std::isfinite(c->scale))
    return dpc::fail(DPC_ERR_INVALID, name + ": scale has to be positive and finite");
  if (backward && (c->grad_stride != 0 && c->grad_stride != 1))
    return dpc::fail(DPC_ERR_INVALID, name + ": grad_stride is 1, or 0 for one gradient for all rows");
  if (backward && (c->d_hidden_stride < c->width || c->d_weight_stride < c->width || c->d_hidden_stride > most ||
                   c->d_weight_stride > most))
    return dpc::fail(DPC_ERR_INVALID, name + ": a gradient's row stride is smaller than the width (or above 2^28)");
  return DPC_OK;
}

// Blocks of the kernel for few rows, which are its parts; 0: the tensor cores.
int few_blocks(const dpc_vocab_ce* c, int sms)
{
  if (c->rows > (c->type == DPC_TYPE_F32 ? kFewRows<float> : kFewRows<__nv_bfloat16>) || (size_t)c->rows * ceil_div(c->width, 256) * 256 * sizeof(float) > kFewBytes / 2)
    return 0;
  return (int)std::min<int64_t>((c->rows > 4 ? 1 : 2) * sms, ceil_div(c->vocab, kWords * (kFewThreads / 32)));
}

int lay_out(const dpc_vocab_ce* c, bool backward, Layout& L)
{
  int device = 0, sms = 0;
  DPC_CUDA(cudaGetDevice(&device));
  DPC_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  if (int rc = wait_limit_now(&L.wait_cycles))
    return rc;
  L.pairs = std::max(1, sms / 2);
  L.planes = c->type == DPC_TYPE_F32 ? 3 : 1;
  // (backward: the rows that do not count are zeros in the copy, so that an infinity in one of them
  // does not reach d_weight as 0 * inf)
  L.copy_hidden = backward || L.planes > 1 || !tma_ready(c->hidden, c->hidden_stride);
  L.copy_weight = L.planes > 1 || !tma_ready(c->weight, c->weight_stride);
  L.cols = L.planes == 3 ? 128 : kTile;
  L.share = L.planes == 3 ? Tile<128, EPI_LSE>::kShare : Tile<256, EPI_LSE>::kShare;
  L.kp = round_up(c->width, 8);
  L.ks = round_up(c->width, kTile);
  const int64_t all = round_up(c->vocab, kTile);
  L.piece = all;
  auto limit = [&](int64_t bytes_each) {
    L.piece = std::min(L.piece, std::max<int64_t>(kPieceLeast, (int64_t)(kPieceBytes / bytes_each) / kTile * kTile));
  };
  if (!backward)
    L.few = few_blocks(c, sms);
  if (L.few > 0)
    L.copy_hidden = L.copy_weight = false;
  if (L.copy_weight)
    limit(L.kp * 2 * L.planes);
  if (backward)
    limit(std::max<int64_t>(1, c->rows) * 2 * L.planes);
  L.piece = round_up(ceil_div(all, ceil_div(all, L.piece)), kTile); // pieces of like size
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (backward)
    L.grad_top = take(sizeof(float));
  if (L.copy_hidden)
    L.hidden = take((size_t)c->rows * L.kp * 2 * L.planes);
  if (L.copy_weight)
    L.weight = take((size_t)std::min(L.piece, c->vocab) * L.kp * 2 * L.planes);
  if (backward)
  {
    // The contraction of d_hidden, over the piece, is shared out where that fills the GPU's last round of tiles (256
    // tiles on 74 CTA pairs are 4 rounds, in halves 3.5), 4 blocks of it at least each; 3 % a share for its sums.
    const int64_t tiles = std::max<int64_t>(1, ceil_div(c->rows, kTile) * ceil_div(c->width, L.cols));
    const int64_t blocks = ceil_div(std::min(L.piece, c->vocab), kDepth);
    double best = 0.0;
    for (int64_t n = 1; n <= std::max<int64_t>(1, std::min<int64_t>(L.pairs, blocks / 4)); ++n)
    {
      const double cost = (double)ceil_div(tiles * n, L.pairs) / n * (1.0 + 0.03 * n);
      if (n == 1 || cost < best)
        best = cost, L.splits = (int)n;
    }
    L.slope = take((size_t)c->rows * L.piece * 2 * L.planes);
    L.sum = take((size_t)L.splits * c->rows * L.ks * sizeof(float));
    L.column_parts = (int)std::min<int64_t>(kColumnParts, ceil_div(c->rows, 64));
    if (c->bias)
      L.columns = take((size_t)L.column_parts * L.piece * sizeof(float));
  }
  else
  {
    L.parts = L.few > 0 ? L.few : round_up(c->vocab, L.cols) / L.share;
    L.partial = take((size_t)L.parts * c->rows * sizeof(float2));
    L.picked = take((size_t)c->rows * sizeof(float));
  }
  L.bytes = at;
  return DPC_OK;
}

int workspace_ok(const dpc_vocab_ce* c, const Layout& L, const char* who)
{
  if (!c->workspace || reinterpret_cast<uintptr_t>(c->workspace) % 256)
    return dpc::fail(DPC_ERR_INVALID, std::string(who) + ": the workspace has to be device memory on a 256-byte boundary");
  if (c->workspace_bytes < L.bytes)
    return dpc::fail(DPC_ERR_INVALID, std::string(who) + ": the workspace has " + std::to_string(c->workspace_bytes) +
                                          " bytes, " + std::to_string(L.bytes) + " are needed");
  return DPC_OK;
}

int grid_for(int64_t work)
{
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(work, 256), 148 * 16));
}

int make_planes(cudaStream_t stream, const dpc_vocab_ce* c, const void* src, int64_t src_ld, int64_t rows,
                const Layout& L, void* dst, bool mask)
{
  const int64_t* targets = mask ? c->targets : nullptr;
  __nv_bfloat16* to = static_cast<__nv_bfloat16*>(dst);
  const int blocks = grid_for(rows * (L.kp / 8));
  if (c->type == DPC_TYPE_F32)
    vocab_planes_kernel<float><<<blocks, 256, 0, stream>>>(static_cast<const float*>(src), src_ld, rows, c->width, to,
                                                           L.kp, targets, c->vocab, c->ignore_index);
  else
    vocab_planes_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(src), src_ld, rows,
                                                                   c->width, to, L.kp, targets, c->vocab, c->ignore_index);
  return launched("vocab_planes_kernel");
}

const void* at_row(const void* p, int type, int64_t elements)
{
  return static_cast<const char*>(p) + elements * (type == DPC_TYPE_F32 ? 4 : 2);
}

// Operands of a piece of the vocabulary that starts at `first`; its weights are brought into planes here.
int piece_weight(cudaStream_t stream, const dpc_vocab_ce* c, const Layout& L, int64_t first, int64_t count, char* ws,
                 Operand& weight)
{
  const void* src = at_row(c->weight, c->type, first * c->weight_stride);
  if (!L.copy_weight)
  {
    weight = {src, c->width, count, c->weight_stride, count * c->weight_stride};
    return DPC_OK;
  }
  weight = {ws + L.weight, c->width, count, L.kp, count * L.kp};
  return make_planes(stream, c, src, c->weight_stride, count, L, ws + L.weight, false);
}

int prepare_hidden(cudaStream_t stream, const dpc_vocab_ce* c, const Layout& L, bool mask, char* ws, Operand& hidden)
{
  if (!L.copy_hidden)
  {
    hidden = {c->hidden, c->width, c->rows, c->hidden_stride, c->rows * c->hidden_stride};
    return DPC_OK;
  }
  hidden = {ws + L.hidden, c->width, c->rows, L.kp, c->rows * L.kp};
  return make_planes(stream, c, c->hidden, c->hidden_stride, c->rows, L, ws + L.hidden, mask);
}

GemmParams base_params(const dpc_vocab_ce* c, const Layout& L, int64_t first, char* ws)
{
  GemmParams P = {};
  P.splits = 1;
  P.grad_top = reinterpret_cast<const float*>(ws + L.grad_top);
  P.factor = c->scale * kLog2e;
  P.scale = c->scale;
  P.bias = c->bias ? at_row(c->bias, c->type, first) : nullptr;
  P.bias_f32 = c->type == DPC_TYPE_F32;
  P.targets = c->targets;
  P.vocab = c->vocab, P.first = first, P.ignore_index = c->ignore_index;
  P.wait_cycles = L.wait_cycles, P.keep_back = waits.keep_back;
  return P;
}

template <typename T, int ROWS>
int launch_few(cudaStream_t stream, const dpc_vocab_ce* c, int blocks, float2* partial, float* picked)
{
  const size_t bytes = (size_t)ROWS * ceil_div(c->width, 256) * 256 * sizeof(float);
  const bool wide = reinterpret_cast<uintptr_t>(c->weight) % 16 == 0 && c->weight_stride % (16 / sizeof(T)) == 0 &&
                    c->width % 8 == 0;
  auto kernel = wide ? vocab_few_kernel<T, ROWS, true> : vocab_few_kernel<T, ROWS, false>;
  // (the most that a call may take: the limit belongs to the kernel, and calls on other host threads set it too)
  DPC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewBytes));
  kernel<<<blocks, kFewThreads, bytes, stream>>>(
      static_cast<const T*>(c->hidden), c->hidden_stride, static_cast<const T*>(c->weight), c->weight_stride,
      (int)c->rows, (int)c->width, c->vocab, static_cast<const T*>(c->bias), c->scale * kLog2e, c->targets,
      c->ignore_index, partial, picked);
  return launched("vocab_few_kernel");
}

template <typename T>
int launch_few(cudaStream_t stream, const dpc_vocab_ce* c, int blocks, float2* partial, float* picked)
{
  if constexpr (kFewRows<T> > 2)
  {
    if (c->rows > 2)
      return c->rows <= 4 ? launch_few<T, 4>(stream, c, blocks, partial, picked)
                          : launch_few<T, kFewRows<T>>(stream, c, blocks, partial, picked);
  }
  return c->rows == 1 ? launch_few<T, 1>(stream, c, blocks, partial, picked)
                      : launch_few<T, 2>(stream, c, blocks, partial, picked);
}

int forward(cudaStream_t stream, const dpc_vocab_ce* c)
{
  const char* who = "dpc_vocab_ce_forward";
  if (int rc = check(c, false, who))
    return rc;
  if (c->rows == 0)
    return DPC_OK;
  if (!c->hidden || !c->weight || !c->targets || !c->loss || !c->lse)
    return dpc::fail(DPC_ERR_INVALID, std::string(who) + ": null pointer");
  Layout L;
  if (int rc = lay_out(c, false, L))
    return rc;
  if (int rc = workspace_ok(c, L, who))
    return rc;
  char* ws = static_cast<char*>(c->workspace);
  float2* partial = reinterpret_cast<float2*>(ws + L.partial);
  float* picked = reinterpret_cast<float*>(ws + L.picked);
  if (L.few > 0)
  {
    if (int rc = c->type == DPC_TYPE_F32 ? launch_few<float>(stream, c, L.few, partial, picked)
                                         : launch_few<__nv_bfloat16>(stream, c, L.few, partial, picked))
      return rc;
  }
  else
  {
    Operand hidden, weight;
    if (int rc = prepare_hidden(stream, c, L, false, ws, hidden))
      return rc;
    for (int64_t first = 0; first < c->vocab; first += L.piece)
    {
      const int64_t count = std::min(L.piece, c->vocab - first);
      if (int rc = piece_weight(stream, c, L, first, count, ws, weight))
        return rc;
      GemmParams P = base_params(c, L, first, ws);
      P.partial = partial, P.picked = picked;
      if (int rc = product<EPI_LSE, false, false>(stream, L.pairs, hidden, weight, L.planes, c->rows, count, c->width, P))
        return rc;
    }
  }
  int row_shift = 0;
  while (row_shift < 3 && c->rows >> (row_shift + 1) >= 296) // (two blocks an SM before rows share one)
    ++row_shift;
  vocab_join_kernel<<<(unsigned)ceil_div(c->rows, (int64_t)1 << row_shift), 256, 0, stream>>>(
      partial, L.parts, c->rows, row_shift, picked, c->targets, c->vocab, c->ignore_index,
      c->loss, c->lse);
  return launched("vocab_join_kernel");
}

int zero_rows(cudaStream_t stream, void* p, int type, int64_t stride, int64_t width, int64_t rows)
{
  const size_t size = type == DPC_TYPE_F32 ? 4 : 2;
  DPC_CUDA(cudaMemset2DAsync(p, stride * size, 0, width * size, rows, stream));
  return DPC_OK;
}

int backward(cudaStream_t stream, const dpc_vocab_ce* c)
{
  const char* who = "dpc_vocab_ce_backward";
  if (int rc = check(c, true, who))
    return rc;
  if (!c->d_weight || (c->d_bias && !c->bias))
    return dpc::fail(DPC_ERR_INVALID, std::string(who) + ": null pointer");
  if (c->rows == 0)
  {
    if (c->d_bias)
      if (int rc = zero_rows(stream, c->d_bias, c->type, c->vocab, c->vocab, 1))
        return rc;
    return zero_rows(stream, c->d_weight, c->type, c->d_weight_stride, c->width, c->vocab);
  }
  if (!c->hidden || !c->weight || !c->targets || !c->lse || !c->grad_loss || !c->d_hidden)
    return dpc::fail(DPC_ERR_INVALID, std::string(who) + ": null pointer");
  Layout L;
  if (int rc = lay_out(c, true, L))
    return rc;
  if (int rc = workspace_ok(c, L, who))
    return rc;
  char* ws = static_cast<char*>(c->workspace);
  float* grad_top = reinterpret_cast<float*>(ws + L.grad_top);
  float* sum = reinterpret_cast<float*>(ws + L.sum);
  __nv_bfloat16* slope = reinterpret_cast<__nv_bfloat16*>(ws + L.slope);
  vocab_gradient_kernel<<<1, 1024, 0, stream>>>(c->grad_loss, c->grad_stride, c->targets, c->rows, c->vocab,
                                                c->ignore_index, grad_top);
  if (int rc = launched("vocab_gradient_kernel"))
    return rc;
  Operand hidden, weight;
  if (int rc = prepare_hidden(stream, c, L, true, ws, hidden))
    return rc;
  const int64_t plane = c->rows * L.piece;
  for (int64_t first = 0; first < c->vocab; first += L.piece)
  {
    const int64_t count = std::min(L.piece, c->vocab - first);
    if (int rc = piece_weight(stream, c, L, first, count, ws, weight))
      return rc;
    GemmParams P = base_params(c, L, first, ws);
    P.lse = c->lse, P.grad = c->grad_loss, P.grad_stride = c->grad_stride;
    P.slope = slope, P.slope_ld = L.piece, P.slope_plane = plane;
    if (int rc = product<EPI_SLOPE, false, false>(stream, L.pairs, hidden, weight, L.planes, c->rows, count, c->width, P))
      return rc;
    const Operand s = {slope, count, c->rows, L.piece, plane};
    P = base_params(c, L, first, ws);
    P.splits = L.splits;
    P.sum = sum, P.sum_ld = L.ks, P.sum_split = c->rows * L.ks, P.add = first > 0;
    if (int rc = product<EPI_SUM, false, true>(stream, L.pairs, s, weight, L.planes, c->rows, c->width, count, P))
      return rc;
    P = base_params(c, L, first, ws);
    P.out = const_cast<void*>(at_row(c->d_weight, c->type, first * c->d_weight_stride));
    P.out_ld = c->d_weight_stride, P.out_f32 = c->type == DPC_TYPE_F32;
    P.out_wide = reinterpret_cast<uintptr_t>(P.out) % 16 == 0 && c->d_weight_stride % (P.out_f32 ? 4 : 8) == 0;
    if (int rc = product<EPI_OUT, true, true>(stream, L.pairs, s, hidden, L.planes, count, c->width, c->rows, P))
      return rc;
    if (c->d_bias)
    {
      float* columns = reinterpret_cast<float*>(ws + L.columns);
      const unsigned blocks = (unsigned)ceil_div(count, 256);
      const dim3 grid(blocks, (unsigned)L.column_parts);
      if (c->type == DPC_TYPE_F32)
      {
        vocab_columns_kernel<3><<<grid, 256, 0, stream>>>(slope, L.piece, plane, c->rows, columns);
        vocab_columns_join_kernel<float><<<blocks, 256, 0, stream>>>(columns, L.piece, L.column_parts, count, grad_top,
                                                                    static_cast<float*>(c->d_bias) + first);
      }
      else
      {
        vocab_columns_kernel<1><<<grid, 256, 0, stream>>>(slope, L.piece, plane, c->rows, columns);
        vocab_columns_join_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(
            columns, L.piece, L.column_parts, count, grad_top, static_cast<__nv_bfloat16*>(c->d_bias) + first);
      }
      if (int rc = launched("vocab_columns_kernel"))
        return rc;
    }
  }
  const int blocks = grid_for(c->rows * ceil_div(c->width, 4));
  if (c->type == DPC_TYPE_F32)
    vocab_sum_kernel<float><<<blocks, 256, 0, stream>>>(sum, L.ks, c->rows * L.ks, L.splits, c->rows, c->width,
                                                        static_cast<float*>(c->d_hidden), c->d_hidden_stride, grad_top, c->scale,
                                                        c->targets, c->vocab, c->ignore_index);
  else
    vocab_sum_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(sum, L.ks, c->rows * L.ks, L.splits, c->rows, c->width,
                                                                static_cast<__nv_bfloat16*>(c->d_hidden),
                                                                c->d_hidden_stride, grad_top, c->scale, c->targets,
                                                                c->vocab, c->ignore_index);
  return launched("vocab_sum_kernel");
}
} // namespace

int dpc_operators_set_wait_limit(double milliseconds, int wait_bias)
{
  if (!(milliseconds <= 60000.0))
    return dpc::fail(DPC_ERR_INVALID, "dpc_operators_set_wait_limit: a minute at most");
  waits = {milliseconds, wait_bias != 0};
  return DPC_OK;
}

int dpc_vocab_ce_workspace(const dpc_vocab_ce* c, int backward, size_t* bytes)
{
  return guarded("dpc_vocab_ce_workspace", [&] {
    if (!bytes)
      return dpc::fail(DPC_ERR_INVALID, "dpc_vocab_ce_workspace: null pointer");
    if (int rc = check(c, backward != 0, "dpc_vocab_ce_workspace"))
      return rc;
    Layout L;
    if (int rc = lay_out(c, backward != 0, L))
      return rc;
    *bytes = L.bytes;
    return (int)DPC_OK;
  });
}

int dpc_vocab_ce_forward(void* stream, const dpc_vocab_ce* c)
{
  return guarded("dpc_vocab_ce_forward", [&] { return forward(static_cast<cudaStream_t>(stream), c); });
}

int dpc_vocab_ce_backward(void* stream, const dpc_vocab_ce* c)
{
  return guarded("dpc_vocab_ce_backward", [&] { return backward(static_cast<cudaStream_t>(stream), c); });
}
