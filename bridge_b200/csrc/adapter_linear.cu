// Low-rank adapters beside a shared projection:  y_t = W x_t + c_s B_s A_s x_t,  s the slot of row t's request.
//
//   shrink   u = c_s A_s x  (and, with B's transpose, du = c_s B_s^T dy):  a skinny product, bound by the read of x.
//   joint    y = W x + B_s u (and dx = W^T dy + A_s^T du): the projection's own GEMM whose K loop goes on over u and
//            the adapters of the slots that its tile of rows meets.  Adding the low-rank part afterwards would read
//            and write y once more; here it costs R / K of the products.
//   grads    dB_s = dy^T u and dA_s = du^T x over the rows of one slot: bound by the reads of dy and x.
//
// Rows of several requests share tiles.  Where a tile holds rows of several slots, each slot's products go into the
// same accumulator under the matrix instruction's lane mask: a row takes nothing from another request's adapter, not
// even a product with zero (which would carry that adapter's infinities over).  The gradients' sums run over rows, so
// there the blocks of rows end where a slot's rows end, and the rows behind are cleared in both operands.
//
// u and du feed matrix instructions, so they are rounded to the operands' 16 bits, and every sum is FP32.  y and dx take
// them as they are then, which costs them less than their own rounding; dA and dB, which are made of nothing else, take them in
// two parts, the rounded value and, rounded too, what it left, or their error would be 1.4 times that of their own rounding.
#include "adapter_linear.h"

#include <c10/util/Exception.h>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <vector>

#include "common.cuh"
#include "sm100_common.cuh"

namespace bb {
namespace {

constexpr int BM = 128, BK = 64;
constexpr int kThreads = 192;          // warp 0: TMA, warp 1: TMEM and MMA, warps 2-5: epilogue
constexpr int kXBytes = BM * BK * 2;   // one block of x: 128 rows x 64, 16 KB
constexpr int kPairInts = 12;

__device__ int g_error;                // first wait that gave up (per device)

__device__ __forceinline__ uint32_t pack2(float a, float b, bool half) {
  if (half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint16_t pack1(float a, bool half) {
  if (half) return __half_as_ushort(__float2half_rn(a));
  return __bfloat16_as_ushort(__float2bfloat16_rn(a));
}

// f v as 16-bit values, and what they leave of it.
__device__ __forceinline__ float unpack1(uint16_t v, bool half) {
  return half ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t rounded, bool half) {
  return pack2(a - unpack1((uint16_t)(rounded & 0xffff), half), b - unpack1((uint16_t)(rounded >> 16), half), half);
}
__device__ __forceinline__ uint4 scaled8(const float (&v)[8], float f, bool half) {
  return make_uint4(pack2(f * v[0], f * v[1], half), pack2(f * v[2], f * v[3], half), pack2(f * v[4], f * v[5], half),
                    pack2(f * v[6], f * v[7], half));
}
__device__ __forceinline__ uint4 rest8(const float (&v)[8], float f, const uint4& r, bool half) {
  return make_uint4(rest2(f * v[0], f * v[1], r.x, half), rest2(f * v[2], f * v[3], r.y, half),
                    rest2(f * v[4], f * v[5], r.z, half), rest2(f * v[6], f * v[7], r.w, half));
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Programmatic dependent launch: the next kernel of the stream may begin (its blocks find room as this grid's end); and
// the wait, until the kernel before this one is complete, of one that began so.  Every kernel here begins early, prepares
// itself and waits before it touches anything that another one makes (the plan was complete before any launch).  The
// joint products go further: behind a shrink they take x and W without a wait, and wait for u only; so a shrink lets
// them begin only when its own wait, for x and W among others, is over.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A block of rows' accumulator (TMEM, `cols` columns) into this block's shared memory, row stride cols + 4 floats
// (rows 16 bytes apart in the banks: neither these stores nor the sums' loads collide).  Warps 2-5.
__device__ __forceinline__ void spill(uint32_t tmem, float* part, int cols, bool any) {
  const int quarter = (threadIdx.x >> 5) & 3, row = quarter * 32 + (threadIdx.x & 31);
  for (int c = 0; c < cols; c += 32) {
    uint32_t r[32];
    if (any) {
      sm100::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, r);
      sm100::tmem_ld_wait();
      sm100::tmem_regs_ready(r);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      if (c + i < cols)
        *reinterpret_cast<uint4*>(part + row * (cols + 4) + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
  }
}

// The sums over the cluster's partial accumulators of eight columns, in rank order; all loads are under way together.
__device__ __forceinline__ void joined8(uint32_t part, int at, int ranks, float (&v)[8]) {
  float4 a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < ranks) {
      const uint32_t from = sm100::mapa(part + at * 4, j);
      a[j] = ld_cluster4(from);
      b[j] = ld_cluster4(from + 16);
    }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < ranks) {
      const float q[8] = {a[j].x, a[j].y, a[j].z, a[j].w, b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = j ? v[i] + q[i] : q[i];
    }
}

// ------------------------------------------------------------------------------------------------ shrink
struct ShrinkParams {
  AdapterPlan plan;
  uint16_t *u, *rest;         // rest: what u's rounding leaves, or null
  const float* scales;
  float scale;
  int T, R, cols, op_bytes, stages, nk, ranks;
  uint32_t idesc;
  bool half;
};

// A cluster of `ranks` blocks takes one slot's rows of a tile of 128, each block a stretch of K; the partial sums meet in
// shared memory.  Rows without an adapter are not written: nothing reads them.  Bound by what an SM takes in by TMA (56
// GB/s from DRAM: x and the adapter's part for every 128 rows), and by start and joining, some 8 us: 4608 rows of 2560,
// rank 16, 12 us; 8192 rows of 9728, rank 64, 45 us (3.5 TB/s of x).
template <bool OP_MN>
__global__ void __launch_bounds__(kThreads)
    adapter_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_op,
                          const ShrinkParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = kXBytes + p.op_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
  uint64_t* empty = full + p.stages;
  uint64_t* done = empty + p.stages;
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank();
  const int* unit = p.plan.units + (size_t)(blockIdx.x / p.ranks) * 8;
  const int tile = __ldg(unit), slot = __ldg(unit + 1);
  const int kb0 = (int)((long)p.nk * rank / p.ranks), kb1 = (int)((long)p.nk * (rank + 1) / p.ranks);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    sm100::mbar_init(done, 1);
    sm100::fence_mbar_init();
    sm100::prefetch_tmap(&map_x);
    sm100::prefetch_tmap(&map_op);
  }
  if (warp == 1) sm100::tmem_alloc(tmem_word, 128);
  if (warp == 0 && lane < kb1 - kb0) {     // weights into L2 while the kernel before this one ends
    if (OP_MN) sm100::tma_prefetch_3d(&map_op, 0, (kb0 + lane) * BK, slot);
    else sm100::tma_prefetch_3d(&map_op, (kb0 + lane) * BK, 0, slot);
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_word;
  wait_for_previous();
  let_next_begin();        // (not before: see there; nor before this block has its TMEM, which one that waits may take)

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&empty[stage], phase ^ 1, &g_error, 31)) break;
      unsigned char* dst = smem + stage * stage_bytes;
      sm100::mbar_expect_tx(&full[stage], stage_bytes);
      sm100::tma_load_2d(dst, &map_x, &full[stage], kb * BK, tile * BM);
      if (OP_MN) {
        for (int i = 0; i < p.cols / 64; ++i)
          sm100::tma_load_3d(dst + kXBytes + i * 8192, &map_op, &full[stage], 64 * i, kb * BK, slot);
      } else {
        sm100::tma_load_3d(dst + kXBytes, &map_op, &full[stage], kb * BK, 0, slot);
      }
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0 && kb1 > kb0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&full[stage], phase, &g_error, 32)) break;
      sm100::tc_fence_after();
      const uint32_t a = sm100::smem_addr(smem + stage * stage_bytes), b = a + kXBytes;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk)
        sm100::umma_bf16(tmem, sm100::umma_desc_sw128(a + kk * 32, 16, 1024),
                         OP_MN ? sm100::umma_desc_sw128(b + kk * 2048, 8192, 1024)
                               : sm100::umma_desc_sw128(b + kk * 32, 16, 1024),
                         p.idesc, kb > kb0 || kk > 0);
      sm100::umma_commit(&empty[stage]);
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
    sm100::umma_commit(done);
  }
  __syncwarp();
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    if (kb1 > kb0) sm100::mbar_wait(done, 0, &g_error, 33);
    __syncwarp();
    sm100::tc_fence_after();
    spill(tmem, part, p.cols, kb1 > kb0);
    sm100::tc_fence_before();
  }
  __syncthreads();
  sm100::cluster_sync();
  // this block's share of the rows: 8 columns a step, the finished values 16 bytes at a time
  const int lo = BM * rank / p.ranks, rows = BM * (rank + 1) / p.ranks - lo, groups = p.R / 8;
  const uint32_t base = sm100::smem_addr(part);
  const float f = p.scales ? p.scales[slot] : p.scale;
  for (int i = threadIdx.x; i < rows * groups; i += kThreads) {
    const int r = lo + i / groups, c = (i % groups) * 8;
    if (__ldg(unit + 4 + r / 32) >> (r % 32) & 1) continue;      // another request's row
    float v[8];
    joined8(base, r * (p.cols + 4) + c, p.ranks, v);
    const size_t at = (size_t)(tile * BM + r) * p.R + c;
    const uint4 out = scaled8(v, f, p.half);
    *reinterpret_cast<uint4*>(p.u + at) = out;
    if (p.rest) *reinterpret_cast<uint4*>(p.rest + at) = rest8(v, f, out, p.half);
  }
  sm100::cluster_sync();   // the peers' sums stay until all have read them
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 128);
  }
}

// The same for a few rows, where a cluster's start and joining would take longer than the reading: a block makes two
// columns of u for four of a slot's rows, its four warps taking 256 values of K in turn.
// Ordinary FP32 arithmetic; nothing to allocate, no barrier but one at the end.  32 rows of 16 slots, 4096 -> 2560, rank 16:
// the whole call 14.4 us, with the kernel above 17.6.
constexpr int kDotWarps = 4, kDotRows = 4;

struct DotsParams {
  AdapterPlan plan;
  const uint16_t *x, *op;
  uint16_t *u, *rest;
  const float* scales;
  float scale;
  long ldx;
  int K, R;
};

__device__ __forceinline__ float2 unpack2(uint32_t v, bool half) {
  if (half) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float s, bool half) {
  const uint32_t p[4] = {a.x, a.y, a.z, a.w}, q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(p[i], half), g = unpack2(q[i], half);
    s = fmaf(f.x, g.x, s);
    s = fmaf(f.y, g.y, s);
  }
  return s;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <bool HALF>
__global__ void __launch_bounds__(32 * kDotWarps) adapter_dots_kernel(const DotsParams p) {
  __shared__ float sums[kDotWarps][2 * kDotRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int* unit = p.plan.units + (size_t)(blockIdx.x / (p.R / 2)) * 8;
  const int tile = __ldg(unit), slot = __ldg(unit + 1), r0 = blockIdx.x % (p.R / 2) * 2;
  const uint16_t* a = p.op + ((size_t)slot * p.R + r0) * p.K;
  constexpr int kStep = 256 * kDotWarps, kUnroll = 4;
  const int k0 = warp * 256 + lane * 8;
  uint32_t mine[4];
  int skip = kDotRows * blockIdx.y;       // rows of the slot that other blocks take
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    mine[w] = ~(uint32_t)__ldg(unit + 4 + w);
    for (; skip > 0 && mine[w]; --skip) mine[w] &= mine[w] - 1;
  }
  if (!(mine[0] | mine[1] | mine[2] | mine[3])) return;
  for (int k = k0; k < p.K; k += kStep) prefetch_l2(a + k), prefetch_l2(a + p.K + k);
  wait_for_previous();
  let_next_begin();
  const float f = p.scales ? p.scales[slot] : p.scale;
  int row[kDotRows], n = 0;
#pragma unroll
  for (int j = 0; j < kDotRows; ++j) {
    row[j] = -1;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (row[j] < 0 && mine[w]) row[j] = 32 * w + __ffs(mine[w]) - 1, mine[w] &= mine[w] - 1, ++n;
  }
  const uint16_t* x[kDotRows];
  float s[2 * kDotRows];
#pragma unroll
  for (int j = 0; j < kDotRows; ++j) {
    x[j] = p.x + (size_t)(tile * BM + max(row[j], 0)) * p.ldx;
    s[2 * j] = s[2 * j + 1] = 0.f;
  }
  for (int k = k0; k < p.K; k += kUnroll * kStep) {
    uint4 q[kUnroll][2], v[kUnroll][kDotRows];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (k + i * kStep < p.K) {
        q[i][0] = *reinterpret_cast<const uint4*>(a + k + i * kStep);
        q[i][1] = *reinterpret_cast<const uint4*>(a + p.K + k + i * kStep);
#pragma unroll
        for (int j = 0; j < kDotRows; ++j)
          if (j < n) v[i][j] = *reinterpret_cast<const uint4*>(x[j] + k + i * kStep);
      }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (k + i * kStep < p.K)
#pragma unroll
        for (int j = 0; j < kDotRows; ++j)
          if (j < n) {
            s[2 * j] = dot8(q[i][0], v[i][j], s[2 * j], HALF);
            s[2 * j + 1] = dot8(q[i][1], v[i][j], s[2 * j + 1], HALF);
          }
  }
#pragma unroll
  for (int j = 0; j < 2 * kDotRows; ++j) {
    s[j] = bb::warp_sum(s[j]);
    if (lane == 0) sums[warp][j] = s[j];
  }
  __syncthreads();
  if (threadIdx.x < kDotRows) {
    const int j = threadIdx.x;
    int r = -1;
#pragma unroll
    for (int i = 0; i < kDotRows; ++i)
      if (i == j) r = row[i];
    if (r >= 0) {
      float t0 = 0.f, t1 = 0.f;
#pragma unroll
      for (int w = 0; w < kDotWarps; ++w) t0 += sums[w][2 * j], t1 += sums[w][2 * j + 1];
      const size_t at = (size_t)(tile * BM + r) * p.R + r0;
      const uint32_t out = pack2(f * t0, f * t1, HALF);
      *reinterpret_cast<uint32_t*>(p.u + at) = out;
      if (p.rest) *reinterpret_cast<uint32_t*>(p.rest + at) = rest2(f * t0, f * t1, out, HALF);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few rows
struct FewParams {
  AdapterPlan plan;
  uint16_t* y;
  int T, N, R, rows, cols, stages, nk, ranks;   // a tile: 128 rows, or T up to the next 8; columns of y
  uint32_t idesc;
  bool half;
};

// Few rows: bound by the read of W.  A cluster of `ranks` blocks takes `cols` columns of y (and 128 rows), each block a
// stretch of K and some of the slots' low-rank products; the partial sums meet in shared memory.  Only the rows that
// there are get loaded: the matrix instruction's other rows read whatever lies behind, and nobody reads what becomes of
// them.  u is waited for when W has been asked for, so that this kernel streams W while the one before it still makes
// u.  2560 -> 6144 without adapters, back to back: 1 row 9.6 us (3.3 TB/s; 5 us of it start and joining), 128 rows 14.3;
// 2560 -> 19456, 61 rows 21.5 (4.8 TB/s).
template <bool MN>
__global__ void __launch_bounds__(kThreads)
    adapter_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_low,
                       const FewParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int x_bytes = p.rows * 128, stage_bytes = x_bytes + p.cols * 128, tmem_cols = p.cols <= 128 ? 128 : 256;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
  uint64_t* empty = full + p.stages;
  uint64_t* done = empty + p.stages;
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(done + 1);
  int4* my_mask = reinterpret_cast<int4*>(full + 32);      // this block's share of the tile's units (256 bytes on)
  int* my_slot = reinterpret_cast<int*>(my_mask + BM);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / p.ranks, m_tiles = (p.T + BM - 1) / BM;    // neighbours share columns of W
  const int rank = (int)sm100::cluster_ctarank(), mt = tile % m_tiles, m0 = mt * BM, n0 = tile / m_tiles * p.cols;
  const int rows = min(BM, p.T - m0);
  const int kb0 = (int)((long)p.nk * rank / p.ranks), kb1 = (int)((long)p.nk * (rank + 1) / p.ranks);
  const int rank_blocks = (p.R + BK - 1) / BK;
  const int unit0 = __ldg(p.plan.unit_start + mt) + rank;
  const int units = max(0, (__ldg(p.plan.unit_start + mt + 1) - unit0 + p.ranks - 1) / p.ranks);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    sm100::mbar_init(done, 1);
    sm100::fence_mbar_init();
    sm100::prefetch_tmap(&map_x);
    sm100::prefetch_tmap(&map_w);
  }
  if (warp == 1) sm100::tmem_alloc(tmem_word, tmem_cols);
  if (warp >= 2 && (int)threadIdx.x - 64 < units) {        // (one at a time in the loops below, each would be a wait)
    const int4* unit = reinterpret_cast<const int4*>(p.plan.units) + 2 * (size_t)(unit0 + (threadIdx.x - 64) * p.ranks);
    my_slot[threadIdx.x - 64] = __ldg(unit).y;
    my_mask[threadIdx.x - 64] = __ldg(unit + 1);
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_word;

  if (p.plan.num_units == 0) wait_for_previous();
  let_next_begin();

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    unsigned char *x_dst = nullptr, *w_dst = nullptr;
    uint64_t* bar = nullptr;
    auto claim = [&]() {
      ok = ok && sm100::mbar_wait(&empty[stage], phase ^ 1, &g_error, 61);
      if (!ok) return false;
      bar = &full[stage];
      x_dst = smem + stage * stage_bytes, w_dst = x_dst + x_bytes;
      sm100::mbar_expect_tx(bar, stage_bytes);
      if (++stage == p.stages) stage = 0, phase ^= 1;
      return true;
    };
    for (int kb = kb0; kb < kb1 && claim(); ++kb) {
      if (MN) {
        sm100::tma_load_2d(w_dst, &map_w, bar, n0, kb * BK);
        sm100::tma_load_2d(w_dst + 8192, &map_w, bar, n0 + 64, kb * BK);
      } else {
        sm100::tma_load_2d(w_dst, &map_w, bar, kb * BK, n0);
      }
      sm100::tma_load_2d(x_dst, &map_x, bar, kb * BK, m0);
    }
    wait_for_previous();       // u, which TMA reads from here on
    asm volatile("fence.proxy.async.global;" ::: "memory");
    for (int i = 0; i < units; ++i)
      for (int rb = 0; rb < rank_blocks && claim(); ++rb) {
        if (MN) {
          sm100::tma_load_3d(w_dst, &map_low, bar, n0, rb * BK, my_slot[i]);
          sm100::tma_load_3d(w_dst + 8192, &map_low, bar, n0 + 64, rb * BK, my_slot[i]);
        } else {
          sm100::tma_load_3d(w_dst, &map_low, bar, rb * BK, n0, my_slot[i]);
        }
        sm100::tma_load_2d(x_dst, &map_u, bar, rb * BK, m0);
      }
  } else if (warp == 1 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto products = [&](int steps, bool first, const uint32_t (&off)[4]) {
      ok = ok && sm100::mbar_wait(&full[stage], phase, &g_error, 62);
      if (!ok) return;
      sm100::tc_fence_after();
      const uint32_t a = sm100::smem_addr(smem + stage * stage_bytes), b = a + x_bytes;
      for (int kk = 0; kk < steps; ++kk)
        sm100::umma_masked(tmem, sm100::umma_desc_sw128(a + kk * 32, 16, 1024),
                           MN ? sm100::umma_desc_sw128(b + kk * 2048, 8192, 1024)
                              : sm100::umma_desc_sw128(b + kk * 32, 16, 1024),
                           p.idesc, !first || kk > 0, off);
      sm100::umma_commit(&empty[stage]);
      if (++stage == p.stages) stage = 0, phase ^= 1;
    };
    const uint32_t all[4] = {0, 0, 0, 0};
    for (int kb = kb0; kb < kb1; ++kb) products(BK / 16, kb == kb0, all);
    for (int i = 0; i < units; ++i) {
      const int4 m = my_mask[i];
      const uint32_t off[4] = {(uint32_t)m.x, (uint32_t)m.y, (uint32_t)m.z, (uint32_t)m.w};
      for (int rb = 0; rb < rank_blocks; ++rb) products(min(BK / 16, (p.R - rb * BK + 15) / 16), false, off);
    }
    sm100::umma_commit(done);
  }
  __syncwarp();
  const int row_floats = p.cols + 4;     // rows 16 bytes apart in the banks
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    sm100::mbar_wait(done, 0, &g_error, 63);
    __syncwarp();
    sm100::tc_fence_after();
    if (quarter * 32 < rows)
      for (int c = 0; c < p.cols; c += 32) {
        uint32_t r[32];
        sm100::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, r);
        sm100::tmem_ld_wait();
        sm100::tmem_regs_ready(r);
        if (row < rows)
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (c + i < p.cols)
              *reinterpret_cast<uint4*>(part + row * row_floats + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        __syncwarp();        // (the next load from TMEM takes the whole warp)
      }
    sm100::tc_fence_before();
  }
  __syncthreads();
  sm100::cluster_sync();
  // this block's share of the groups of 8 columns
  const int lo = p.cols / 8 * rank / p.ranks, groups = p.cols / 8 * (rank + 1) / p.ranks - lo;
  const uint32_t base = sm100::smem_addr(part);
  for (int i = threadIdx.x; i < groups * rows; i += kThreads) {
    const int c = (lo + i % groups) * 8, t = i / groups;
    if (n0 + c >= p.N) continue;
    float v[8];
    joined8(base, t * row_floats + c, p.ranks, v);
    *reinterpret_cast<uint4*>(p.y + (size_t)(m0 + t) * p.N + n0 + c) =
        make_uint4(pack2(v[0], v[1], p.half), pack2(v[2], v[3], p.half), pack2(v[4], v[5], p.half), pack2(v[6], v[7], p.half));
  }
  sm100::cluster_sync();   // the peers' sums stay until all have read them
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------------------------------------ tokens
struct TokenParams {
  AdapterPlan plan;
  uint16_t *y, *u;
  const uint16_t* low;
  const float* scales;
  float scale;
  int T, N, R, rows, stages, nk, ranks;
  int slot_cols, columns;   // of a slot in the accumulator; of TMEM
  uint32_t idesc;
  bool half;
};

__device__ __forceinline__ float ld_cluster1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// A few rows of few slots, in one kernel: every cluster (128 columns of y, each of its blocks a stretch of K) makes
// u for itself as it goes, from the slots' rows of A beside W's: more reading from L2, but no second kernel to start, to
// end and to wait for.  The accumulator holds y's 128 columns and the products with every slot's A, of which a row takes
// its own slot's.  Where the partial sums meet, each block adds up u, rounds it as the other kernels do, and makes its
// share of the columns: a few FP32 products a value.  The first cluster keeps u if it is asked for, but only y's: du, whose
// sums here go by the columns of dx, comes from the kernels above whether dx is asked for or not, so that dA is the same
// either way.  1 row, 2560 -> 6144, rank 16: 10.7 us back to back.
template <bool MN>
__global__ void __launch_bounds__(kThreads)
    adapter_token_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                         const __grid_constant__ CUtensorMap map_op, const TokenParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int slots = p.plan.num_units, u_cols = slots * p.slot_cols;
  const int x_bytes = p.rows * 128, stage_bytes = x_bytes + kXBytes + u_cols * 128;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
  uint64_t* empty = full + p.stages;
  uint64_t* done = empty + p.stages;
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(done + 1);
  int* slot_of = reinterpret_cast<int*>(done + 2);       // of the units, at most 16
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank(), n0 = blockIdx.x / p.ranks * BM;
  const int kb0 = (int)((long)p.nk * rank / p.ranks), kb1 = (int)((long)p.nk * (rank + 1) / p.ranks);
  const int lo = BM * rank / p.ranks, cols = BM * (rank + 1) / p.ranks - lo;      // this block's columns

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    sm100::mbar_init(done, 1);
    sm100::fence_mbar_init();
    sm100::prefetch_tmap(&map_x);
    sm100::prefetch_tmap(&map_w);
    sm100::prefetch_tmap(&map_op);
  }
  if (warp == 1) sm100::tmem_alloc(tmem_word, p.columns);
  if (warp == 0 && lane < slots) slot_of[lane] = __ldg(p.plan.units + (size_t)lane * 8 + 1);
  // weights into L2 while the kernel before this one ends (whatever it still writes there, L2 has)
  if (warp == 0 && lane < kb1 - kb0) {
    if (MN) {
      sm100::tma_prefetch_2d(&map_w, n0, (kb0 + lane) * BK);
      sm100::tma_prefetch_2d(&map_w, n0 + 64, (kb0 + lane) * BK);
    } else {
      sm100::tma_prefetch_2d(&map_w, (kb0 + lane) * BK, n0);
    }
  } else if (warp >= 2) {
    const int lines = MN ? p.R * ((cols * 2 + 127) / 128) : (cols * p.R * 2 + 127) / 128;
    for (int i = threadIdx.x - 64; i < lines * slots; i += kThreads - 64) {
      const int slot = __ldg(p.plan.units + (size_t)(i / lines) * 8 + 1), l = i % lines;
      const size_t at = MN ? ((size_t)slot * p.R + l % p.R) * p.N + n0 + lo + l / p.R * 64
                           : ((size_t)slot * p.N + n0 + lo) * p.R + l * 64;
      if (n0 + lo < p.N && at < (size_t)(slot + 1) * p.N * p.R) prefetch_l2(p.low + at);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_word;
  let_next_begin();
  wait_for_previous();

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&empty[stage], phase ^ 1, &g_error, 71)) break;
      unsigned char *x_dst = smem + stage * stage_bytes, *w_dst = x_dst + x_bytes, *op_dst = w_dst + kXBytes;
      uint64_t* bar = &full[stage];
      sm100::mbar_expect_tx(bar, stage_bytes);
      if (MN) {
        sm100::tma_load_2d(w_dst, &map_w, bar, n0, kb * BK);
        sm100::tma_load_2d(w_dst + 8192, &map_w, bar, n0 + 64, kb * BK);
      } else {
        sm100::tma_load_2d(w_dst, &map_w, bar, kb * BK, n0);
      }
      sm100::tma_load_2d(x_dst, &map_x, bar, kb * BK, 0);
      for (int i = 0; i < slots; ++i) {
        const int slot = slot_of[i];
        if (MN) {
          for (int j = 0; j < p.slot_cols / 64; ++j)
            sm100::tma_load_3d(op_dst + (i * (p.slot_cols / 64) + j) * 8192, &map_op, bar, 64 * j, kb * BK, slot);
        } else {
          sm100::tma_load_3d(op_dst + i * p.slot_cols * 128, &map_op, bar, kb * BK, 0, slot);
        }
      }
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait(&full[stage], phase, &g_error, 72)) break;
      sm100::tc_fence_after();
      // the slots' rows of A lie behind W's: one instruction makes both
      const uint32_t a = sm100::smem_addr(smem + stage * stage_bytes), b = a + x_bytes;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk)
        sm100::umma_bf16(tmem, sm100::umma_desc_sw128(a + kk * 32, 16, 1024),
                         MN ? sm100::umma_desc_sw128(b + kk * 2048, 8192, 1024)
                            : sm100::umma_desc_sw128(b + kk * 32, 16, 1024), p.idesc, kb > kb0 || kk > 0);
      sm100::umma_commit(&empty[stage]);
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
    sm100::umma_commit(done);
  }
  __syncwarp();
  const int row_floats = BM + u_cols + 4;       // rows 16 bytes apart in the banks
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    sm100::mbar_wait(done, 0, &g_error, 73);
    __syncwarp();
    sm100::tc_fence_after();
    if (quarter * 32 < p.T)
      for (int c = 0; c < BM + u_cols; c += 16) {
        uint32_t r[16];
        sm100::tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c, r);
        sm100::tmem_ld_wait();
        sm100::tmem_regs_ready(r);
        if (row < p.T)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint4*>(part + row * row_floats + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        __syncwarp();        // (the next load from TMEM takes the whole warp)
      }
    sm100::tc_fence_before();
  }
  __syncthreads();
  sm100::cluster_sync();
  const uint32_t base = sm100::smem_addr(part);
  // u of every row, from its slot's columns
  uint16_t* u = reinterpret_cast<uint16_t*>(part + p.T * row_floats);
  for (int i = threadIdx.x; i < p.T * (p.R / 8); i += kThreads) {
    const int t = i / (p.R / 8), c = i % (p.R / 8) * 8, slot = __ldg(p.plan.row_slot + t);
    if (slot < 0) continue;
    int at = 0;
    while (slot_of[at] != slot) ++at;
    float v[8];
    joined8(base, t * row_floats + BM + at * p.slot_cols + c, p.ranks, v);
    const float f = p.scales ? p.scales[slot] : p.scale;
    const uint4 out = scaled8(v, f, p.half);
    *reinterpret_cast<uint4*>(u + t * p.R + c) = out;
    if (p.u && blockIdx.x == 0) {
      *reinterpret_cast<uint4*>(p.u + (size_t)t * p.R + c) = out;
      *reinterpret_cast<uint4*>(p.u + ((size_t)p.T + t) * p.R + c) = rest8(v, f, out, p.half);
    }
  }
  __syncthreads();
  // this block's columns of y
  for (int i = threadIdx.x; i < cols * p.T; i += kThreads) {
    const int c = lo + i % cols, t = i / cols, n = n0 + c;
    if (n >= p.N) continue;
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < p.ranks) q[j] = ld_cluster1(sm100::mapa(base + (t * row_floats + c) * 4, j));
    float v = q[0];
#pragma unroll
    for (int j = 1; j < 8; ++j)
      if (j < p.ranks) v += q[j];
    const int slot = __ldg(p.plan.row_slot + t);
    if (slot >= 0) {
      for (int k = 0; k < p.R; k += 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(u + t * p.R + k);
        const float2 a0 = unpack2(a.x, p.half), a1 = unpack2(a.y, p.half), a2 = unpack2(a.z, p.half), a3 = unpack2(a.w, p.half);
        if (MN) {
          const uint16_t* b = p.low + ((size_t)slot * p.R + k) * p.N + n;
          const float w[8] = {a0.x, a0.y, a1.x, a1.y, a2.x, a2.y, a3.x, a3.y};
#pragma unroll
          for (int j = 0; j < 8; ++j) v = fmaf(w[j], unpack1(b[(size_t)j * p.N], p.half), v);
        } else {
          const uint4 b = *reinterpret_cast<const uint4*>(p.low + ((size_t)slot * p.N + n) * p.R + k);
          const float2 b0 = unpack2(b.x, p.half), b1 = unpack2(b.y, p.half), b2 = unpack2(b.z, p.half), b3 = unpack2(b.w, p.half);
          v = fmaf(a0.x, b0.x, v), v = fmaf(a0.y, b0.y, v), v = fmaf(a1.x, b1.x, v), v = fmaf(a1.y, b1.y, v);
          v = fmaf(a2.x, b2.x, v), v = fmaf(a2.y, b2.y, v), v = fmaf(a3.x, b3.x, v), v = fmaf(a3.y, b3.y, v);
        }
      }
    }
    p.y[(size_t)t * p.N + n] = pack1(v, p.half);
  }
  sm100::cluster_sync();   // the peers' sums stay until all have read them
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, p.columns);
  }
}

// ------------------------------------------------------------------------------------------------ joint
// A pair of blocks (two SMs) computes tiles of 256 x 256: each holds its 128 rows of x and its half of W's 256, so that
// every block of K costs an SM 32 KB for 2 x 128 x 256 x 64 products.  Accumulators are double-buffered in TMEM: a tile's
// stores overlap the next one's products.
//
// Bound by the matrix units (85% of their cycles at 4096 x 9728 x 2560) and, when calls follow each other, by the power
// cap: 8192 rows, 2560 -> 19456, 0.53 ms alone (1.55 PFLOP/s), 0.60 sustained (1.35 at 1.34 GHz; the library's 0.61).
//
// Tiles go round the pairs; those of a last round that would leave most pairs idle are cut along K into `slices`, whose
// FP32 sums adapter_join_kernel adds up in slice order.
constexpr int kPairStages = 6;
constexpr int kPairHalf = 128 * BK * 2;
constexpr int kPairStage = 2 * kPairHalf;
constexpr int kStoreBytes = 32 * 64 * 2;       // what a warp of the epilogue stores at a time: 32 rows x 64 columns
constexpr int kPairSmem = kPairStages * kPairStage + 4 * 2 * kStoreBytes + 256 + 1024;
constexpr int kPairTile = 256 * 256;

struct JointParams {
  AdapterPlan plan;
  uint16_t* y;
  float* sums;             // [units of cut tiles][256 / 4 columns][256 rows][4]
  int T, N, R, nk;
  int group;                  // tiles of rows that go through the columns together
  int whole, slices, units;   // tiles that are not cut, cuts of each other one, pieces of work in all
  uint32_t idesc;
  bool half;
};

struct Piece {
  int mt, nt, kb0, kb1, sum;   // sum: which partial sum, or -1
  bool last;                   // takes the low-rank part
};

__device__ __forceinline__ Piece piece_at(const JointParams& p, int q) {
  const int m_tiles = (p.T + 255) / 256, n_tiles = (p.N + 255) / 256;
  Piece w;
  int tile = q;
  w.kb0 = 0, w.kb1 = p.nk, w.sum = -1, w.last = true;
  if (q >= p.whole) {
    const int j = q - p.whole, slice = j % p.slices;
    tile = p.whole + j / p.slices;
    if (p.slices > 1) {
      w.kb0 = (int)((long)p.nk * slice / p.slices), w.kb1 = (int)((long)p.nk * (slice + 1) / p.slices);
      w.sum = j, w.last = slice == p.slices - 1;
    }
  }
  // groups of tiles of rows, so that a tile of W serves all of a group from L2
  const int per_group = p.group * n_tiles, first = tile / per_group * p.group, gm = min(p.group, m_tiles - first);
  const int r = tile % per_group;
  w.mt = first + r % gm;
  w.nt = r / gm;
  return w;
}

template <bool MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    adapter_joint_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                         const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_low,
                         const __grid_constant__ CUtensorMap map_y, const __grid_constant__ JointParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* store = smem + kPairStages * kPairStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(store + 4 * 2 * kStoreBytes);
  uint64_t* empty = full + kPairStages;
  uint64_t* tfull = empty + kPairStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int rank_blocks = (p.R + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      sm100::mbar_init(&tfull[a], 1);
      sm100::mbar_init(&tempty[a], 256);
    }
    sm100::fence_mbar_init();
    sm100::prefetch_tmap(&map_x);
    sm100::prefetch_tmap(&map_w);
  }
  if (warp == 1) sm100::tmem_alloc_pair(tmem_word, 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_word;
  if (p.plan.num_units == 0) wait_for_previous();
  let_next_begin();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t bar = 0;
      unsigned char *x_dst = nullptr, *w_dst = nullptr;
      auto claim = [&]() {
        ok = ok && sm100::mbar_wait_cluster(&empty[stage], phase ^ 1, &g_error, 41);
        if (!ok) return false;
        if (rank == 0) sm100::mbar_expect_tx(&full[stage], 2 * kPairStage);
        bar = sm100::mapa(sm100::smem_addr(&full[stage]), 0);      // both blocks' loads count on the leader's barrier
        x_dst = smem + stage * kPairStage, w_dst = x_dst + kPairHalf;
        if (++stage == kPairStages) stage = 0, phase ^= 1;
        return true;
      };
      for (int q = pair; q < p.units && ok; q += pairs) {
        const Piece w = piece_at(p, q);
        const int m0 = w.mt * 256 + 128 * rank, n0 = w.nt * 256 + 128 * rank;
        const int first = __ldg(p.plan.tile_start + w.mt), end = __ldg(p.plan.tile_start + w.mt + 1);
        int next_slot = first < end ? __ldg(p.plan.pairs + (size_t)first * kPairInts) : 0;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!claim()) break;
          sm100::tma_load_2d_pair(x_dst, &map_x, bar, kb * BK, m0);
          if (MN) {
            sm100::tma_load_2d_pair(w_dst, &map_w, bar, n0, kb * BK);
            sm100::tma_load_2d_pair(w_dst + 8192, &map_w, bar, n0 + 64, kb * BK);
          } else {
            sm100::tma_load_2d_pair(w_dst, &map_w, bar, kb * BK, n0);
          }
        }
        if (q == pair) {
          wait_for_previous();       // u, which TMA reads from here on
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        if (!w.last) continue;
        for (int i = first; i < end && ok; ++i) {
          const int slot = next_slot;        // (asked for a pair ahead: the answer takes longer than the pair's products)
          if (i + 1 < end) next_slot = __ldg(p.plan.pairs + (size_t)(i + 1) * kPairInts);
          for (int rb = 0; rb < rank_blocks; ++rb) {
            if (!claim()) break;
            sm100::tma_load_2d_pair(x_dst, &map_u, bar, rb * BK, m0);
            if (MN) {
              sm100::tma_load_3d_pair(w_dst, &map_low, bar, n0, rb * BK, slot);
              sm100::tma_load_3d_pair(w_dst + 8192, &map_low, bar, n0 + 64, rb * BK, slot);
            } else {
              sm100::tma_load_3d_pair(w_dst, &map_low, bar, rb * BK, n0, slot);
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int q = pair; q < p.units && ok; q += pairs) {
        if (!sm100::mbar_wait_cluster(&tempty[acc], acc_phase ^ 1, &g_error, 42)) break;
        sm100::tc_fence_after();
        const uint32_t d = tmem + acc * 256;
        const Piece w = piece_at(p, q);
        const int4* masks = reinterpret_cast<const int4*>(p.plan.pairs);
        const int first = __ldg(p.plan.tile_start + w.mt), end = __ldg(p.plan.tile_start + w.mt + 1);
        int4 next_lo = {}, next_hi = {};
        if (first < end) next_lo = __ldg(masks + 3 * (size_t)first + 1), next_hi = __ldg(masks + 3 * (size_t)first + 2);
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          ok = sm100::mbar_wait_cluster(&full[stage], phase, &g_error, 43);
          if (!ok) break;
          sm100::tc_fence_after();
          const uint32_t a = sm100::smem_addr(smem + stage * kPairStage), b = a + kPairHalf;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            sm100::umma_bf16_pair(d, sm100::umma_desc_sw128(a + kk * 32, 16, 1024),
                                  MN ? sm100::umma_desc_sw128(b + kk * 2048, 8192, 1024)
                                     : sm100::umma_desc_sw128(b + kk * 32, 16, 1024),
                                  p.idesc, kb > w.kb0 || kk > 0);
          sm100::umma_commit_pair_mc(&empty[stage], 0x3);
          if (++stage == kPairStages) stage = 0, phase ^= 1;
        }
        if (w.last) {
          for (int i = first; i < end && ok; ++i) {
            const int4 lo = next_lo, hi = next_hi;
            if (i + 1 < end) next_lo = __ldg(masks + 3 * (size_t)i + 4), next_hi = __ldg(masks + 3 * (size_t)i + 5);
            const uint32_t off[8] = {(uint32_t)lo.x, (uint32_t)lo.y, (uint32_t)lo.z, (uint32_t)lo.w,
                                     (uint32_t)hi.x, (uint32_t)hi.y, (uint32_t)hi.z, (uint32_t)hi.w};
            for (int rb = 0; rb < rank_blocks; ++rb) {
              ok = sm100::mbar_wait_cluster(&full[stage], phase, &g_error, 45);
              if (!ok) break;
              sm100::tc_fence_after();
              const uint32_t a = sm100::smem_addr(smem + stage * kPairStage), b = a + kPairHalf;
              const int steps = min(BK / 16, (p.R - rb * BK + 15) / 16);
              for (int kk = 0; kk < steps; ++kk)
                sm100::umma_pair_masked(d, sm100::umma_desc_sw128(a + kk * 32, 16, 1024),
                                        MN ? sm100::umma_desc_sw128(b + kk * 2048, 8192, 1024)
                                           : sm100::umma_desc_sw128(b + kk * 32, 16, 1024),
                                        p.idesc, 1, off);
              sm100::umma_commit_pair_mc(&empty[stage], 0x3);
              if (++stage == kPairStages) stage = 0, phase ^= 1;
            }
          }
        }
        if (!ok) break;
        sm100::umma_commit_pair_mc(&tfull[acc], 0x3);
        if (++acc == 2) acc = 0, acc_phase ^= 1;
      }
    }
  } else {
    const int quarter = warp & 3;
    int acc = 0, turn = 0;      // turn: which of the warp's two store buffers is next, through all of its tiles
    uint32_t acc_phase = 0;
    for (int q = pair; q < p.units; q += pairs) {
      const bool got = sm100::mbar_wait_cluster(&tfull[acc], acc_phase, &g_error, 44);
      if (!__all_sync(0xffffffffu, got)) break;
      sm100::tc_fence_after();
      const Piece w = piece_at(p, q);
      const int at = 128 * rank + quarter * 32 + lane;
      const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + acc * 256;
      if (w.sum >= 0) {
#pragma unroll 1
        for (int c = 0; c < 256; c += 32) {
          uint32_t r[32];
          sm100::tmem_ld32(src + c, r);
          sm100::tmem_ld_wait();
          sm100::tmem_regs_ready(r);
          float4* dst = reinterpret_cast<float4*>(p.sums + (size_t)w.sum * kPairTile) + (size_t)(c / 4) * 256 + at;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            dst[j * 256] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                       __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
        }
      } else {
        // 32 rows x 64 columns at a time through shared memory (128-byte swizzle: 16-byte piece j of row i lies at
        // j ^ i % 8), so that y is written in whole lines; straight from the registers its sectors went out in halves.
        // The two buffers take turns from store to store, not from column to column: a tile at the right edge may have
        // an odd number of stores, and the wait below is for all but the last one.
        const int row0 = w.mt * 256 + 128 * rank + quarter * 32;
#pragma unroll 1
        for (int c = 0; c < 256; c += 64) {
          const int col = w.nt * 256 + c;
          if (row0 >= p.T || col >= p.N) break;
          uint32_t r[32], r2[32];
          sm100::tmem_ld32(src + c, r);
          sm100::tmem_ld32(src + c + 32, r2);
          sm100::tmem_ld_wait();
          sm100::tmem_regs_ready(r);
          sm100::tmem_regs_ready(r2);
          unsigned char* buf = store + (quarter * 2 + turn) * kStoreBytes;
          turn ^= 1;
          if (lane == 0) sm100::tma_store_wait_read<1>();      // the store before the last one has left this buffer
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint4 v;
            if (j < 4)
              v = make_uint4(pack2(__uint_as_float(r[8 * j]), __uint_as_float(r[8 * j + 1]), p.half),
                             pack2(__uint_as_float(r[8 * j + 2]), __uint_as_float(r[8 * j + 3]), p.half),
                             pack2(__uint_as_float(r[8 * j + 4]), __uint_as_float(r[8 * j + 5]), p.half),
                             pack2(__uint_as_float(r[8 * j + 6]), __uint_as_float(r[8 * j + 7]), p.half));
            else
              v = make_uint4(pack2(__uint_as_float(r2[8 * j - 32]), __uint_as_float(r2[8 * j - 31]), p.half),
                             pack2(__uint_as_float(r2[8 * j - 30]), __uint_as_float(r2[8 * j - 29]), p.half),
                             pack2(__uint_as_float(r2[8 * j - 28]), __uint_as_float(r2[8 * j - 27]), p.half),
                             pack2(__uint_as_float(r2[8 * j - 26]), __uint_as_float(r2[8 * j - 25]), p.half));
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((j ^ (lane & 7)) * 16)) = v;
          }
          sm100::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            sm100::tma_store_2d(&map_y, buf, col, row0);
            sm100::tma_store_commit();
          }
        }
      }
      sm100::tc_fence_before();
      sm100::mbar_arrive_cluster(sm100::mapa(sm100::smem_addr(&tempty[acc]), 0));
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
    if (lane == 0) sm100::tma_store_wait_all();
  }
  __syncwarp();
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();   // the peer's barriers and operands stay until both are done
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(tmem, 512);
  }
}

// The cut tiles: y = the sum over a tile's slices, in their order.  One block: 16 columns of the 256 rows.
__global__ void __launch_bounds__(256) adapter_join_kernel(const __grid_constant__ JointParams p) {
  const int tile = blockIdx.x / 16, c = blockIdx.x % 16 * 16;
  const Piece w = piece_at(p, p.whole + tile * p.slices);
  const int row = w.mt * 256 + threadIdx.x, col = w.nt * 256 + c;
  let_next_begin();
  wait_for_previous();
  if (row >= p.T || col >= p.N) return;
  float4 v[4] = {};
  for (int s = 0; s < p.slices; ++s) {
    const float4* src = reinterpret_cast<const float4*>(p.sums + (size_t)(tile * p.slices + s) * kPairTile) +
                        (size_t)(c / 4) * 256 + threadIdx.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 a = __ldcs(src + j * 256);
      v[j].x += a.x, v[j].y += a.y, v[j].z += a.z, v[j].w += a.w;
    }
  }
  uint16_t* dst = p.y + (size_t)row * p.N + col;
#pragma unroll
  for (int j = 0; j < 4; j += 2)
    if (col + j * 4 < p.N)
      *reinterpret_cast<uint4*>(dst + j * 4) =
          make_uint4(pack2(v[j].x, v[j].y, p.half), pack2(v[j].z, v[j].w, p.half),
                     pack2(v[j + 1].x, v[j + 1].y, p.half), pack2(v[j + 1].z, v[j + 1].w, p.half));
}

// ------------------------------------------------------------------------------------------------ grads
// Stages of 32 KB (three, so that two blocks fit an SM), or of 48 where the rank is above 64.
constexpr int grad_stages(int cols) { return cols == 64 ? 3 : 4; }

struct GradParams {
  AdapterPlan plan;
  void *da, *db;
  int K, N, S, R, cols, tiles_a, tiles_b, ranks;
  uint32_t idesc;
  bool add_a, add_b, half;
};

// What a block writes of the gradients: 128 columns of dy (rows of dB) or of x (columns of dA).
struct GradTile {
  void* out;
  int m0, limit, R;
  bool is_b, add, half;

  // four values of row m0 + r, columns c to c + 3
  __device__ __forceinline__ void put(int slot, int r, int c, float4 v) const {
    if (m0 + r >= limit) return;
    if (is_b) {
      const size_t to = ((size_t)slot * limit + m0 + r) * R + c;
      if (add) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + to);
        const float4 o = *dst;
        *dst = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + to) =
            make_uint2(pack2(v.x, v.y, half), pack2(v.z, v.w, half));
      }
    } else {
      const size_t to = ((size_t)slot * R + c) * limit + m0 + r;
      const float q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (add) static_cast<float*>(out)[to + (size_t)j * limit] += q[j];
        else static_cast<uint16_t*>(out)[to + (size_t)j * limit] = pack1(q[j], half);
      }
    }
  }
  // i-th piece of four of `rows` rows from `lo`: dB has neighbours in a row of R, dA in a column
  __device__ __forceinline__ void place(int i, int lo, int rows, int& r, int& c) const {
    r = lo + (is_b ? i / (R / 4) : i % rows);
    c = (is_b ? i % (R / 4) : i / rows) * 4;
  }
};

// A cluster takes 128 columns of dy (or x) and the rows of all slots, cut evenly over its blocks whatever the slots'
// shares: D_s [128, R] = sum over slot s's rows of dy^T u (x^T du).  A slot whose rows all fall to one block is written
// by it at once, from the accumulator, while the next slot's products go into another one; of the slots that begin or end
// in another block (at most two a block) the partial sums meet in shared memory at the end, in the blocks' order.  Bound
// like the shrink: alone and with nothing in L2, 4608 rows of 2560 and 6144 columns, rank 16, 33 us (80 MB); 8192 rows of 9728
// and 2560, rank 64, 71 us (201 MB); 3.5 and 12 us of it for the second parts of u and du.
__global__ void __launch_bounds__(kThreads)
    adapter_grads_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dy,
                         const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_du,
                         const GradParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int low_bytes = p.cols / 64 * 8192, stage_bytes = kXBytes + 2 * low_bytes, stages = grad_stages(p.cols);
  const int part_floats = BM * (p.cols + 4), tmem_cols = p.cols == 64 ? 256 : 512;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + max(stages * stage_bytes, 2 * part_floats * 4));
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;     // of the three accumulators
  uint64_t* tempty = tfull + 3;
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(tempty + 3);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank(), tile = blockIdx.x / p.ranks;
  const bool is_b = tile < p.tiles_b;
  const GradTile g{is_b ? p.db : p.da, (is_b ? tile : tile - p.tiles_b) * BM, is_b ? p.N : p.K, p.R, is_b,
                   is_b ? p.add_b : p.add_a, p.half};
  const CUtensorMap* map_wide = is_b ? &map_dy : &map_x;
  const CUtensorMap* map_thin = is_b ? &map_u : &map_du;
  const int4* blocks = reinterpret_cast<const int4*>(p.plan.blocks);
  const auto cut = [&](int r) { return (int)((long)p.plan.num_blocks * r / p.ranks); };
  const int b0 = cut(rank), b1 = cut(rank + 1);
  // the first slot's rows began in an earlier block: its sum stays in accumulator 0 to the end
  const bool began = b1 > b0 && __ldg(p.plan.block_start + __ldg(&blocks[b0]).z) < b0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 3; ++i) {
      sm100::mbar_init(&tfull[i], 1);
      sm100::mbar_init(&tempty[i], 128);
    }
    sm100::fence_mbar_init();
    sm100::prefetch_tmap(map_wide);
    sm100::prefetch_tmap(map_thin);
  }
  if (warp == 1) sm100::tmem_alloc(tmem_word, tmem_cols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_word;
  let_next_begin();
  wait_for_previous();
  float* part = reinterpret_cast<float*>(smem);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int b = b0; b < b1; ++b) {
        const int row = __ldg(&blocks[b]).x;
        if (!sm100::mbar_wait(&empty[stage], phase ^ 1, &g_error, 51)) break;
        unsigned char* dst = smem + stage * stage_bytes;
        sm100::mbar_expect_tx(&full[stage], stage_bytes);
        sm100::tma_load_2d(dst, map_wide, &full[stage], g.m0, row);
        sm100::tma_load_2d(dst + 8192, map_wide, &full[stage], g.m0 + 64, row);
        for (int i = 0; i < p.cols / 32; ++i)      // both parts of u
          sm100::tma_load_3d(dst + kXBytes + i * 8192, map_thin, &full[stage], i % (p.cols / 64) * 64, row, i / (p.cols / 64));
        if (++stage == stages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    int stage = 0, slot = -1, acc = 2;
    uint32_t phase = 0, acc_phase[3] = {0, 0, 0};
    bool ok = true;
    for (int b = b0; b < b1 && ok; ++b) {
      const int4 block = __ldg(&blocks[b]);
      const bool fresh = block.z != slot;
      if (fresh) {
        if (slot >= 0 && lane == 0) sm100::umma_commit(&tfull[acc]);
        acc = slot < 0 && began ? 0 : acc == 1 ? 2 : 1;
        slot = block.z;
        ok = sm100::mbar_wait(&tempty[acc], acc_phase[acc] ^ 1, &g_error, 54);
        acc_phase[acc] ^= 1;
      }
      ok = ok && sm100::mbar_wait(&full[stage], phase, &g_error, 52);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      unsigned char* at = smem + stage * stage_bytes;
      const int n = block.y, steps = (n + 15) / 16;
      if (n < steps * 16) {
        // rows of other requests behind the block: a row is 128 bytes of every 64 columns, in whatever order
        const int lines = (steps * 16 - n) * 8;
        for (int i = lane; i < lines * (2 + p.cols / 32); i += 32)
          *reinterpret_cast<uint4*>(at + i / lines * 8192 + n * 128 + i % lines * 16) = make_uint4(0, 0, 0, 0);
        sm100::fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) {
        sm100::tc_fence_after();
        const uint32_t a = sm100::smem_addr(at), w = a + kXBytes;
        for (int kk = 0; kk < steps; ++kk)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            sm100::umma_bf16(tmem + acc * p.cols, sm100::umma_desc_sw128(a + kk * 2048, 8192, 1024),
                             sm100::umma_desc_sw128(w + half * low_bytes + kk * 2048, 8192, 1024), p.idesc,
                             !fresh || kk > 0 || half > 0);
        sm100::umma_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == stages) stage = 0, phase ^= 1;
    }
    if (slot >= 0 && lane == 0) sm100::umma_commit(&tfull[acc]);
  } else {
    const int quarter = warp & 3;
    int acc = 2, slot = -1;
    uint32_t acc_phase[3] = {0, 0, 0};
    for (int b = b0; b < b1;) {
      acc = slot < 0 && began ? 0 : acc == 1 ? 2 : 1;
      slot = __ldg(&blocks[b]).z;
      const int end = __ldg(p.plan.block_start + slot + 1);
      const bool got = sm100::mbar_wait(&tfull[acc], acc_phase[acc], &g_error, 53);
      acc_phase[acc] ^= 1;
      if (!__all_sync(0xffffffffu, got)) break;
      sm100::tc_fence_after();
      if (!(began && acc == 0) && end <= b1) {       // all of the slot's rows were this block's
        for (int c = 0; c < p.R; c += 32) {
          uint32_t r[32];
          sm100::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + acc * p.cols + c, r);
          sm100::tmem_ld_wait();
          sm100::tmem_regs_ready(r);
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (c + j < p.R)
              g.put(slot, quarter * 32 + lane, c + j, make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]),
                                                                  __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])));
          __syncwarp();      // (rows behind the last one leave `put` early; the next load from TMEM takes the whole warp)
        }
      }
      sm100::tc_fence_before();
      if (acc) sm100::mbar_arrive(&tempty[acc]);
      b = end;
    }
    // every product is done, so the operands' memory is free: the sums that are others' too
    sm100::tc_fence_after();
    if (began) spill(tmem, part, p.cols, true);
    if (b1 > b0 && __ldg(p.plan.block_start + slot + 1) > b1 && !(began && acc == 0))
      spill(tmem + acc * p.cols, part + part_floats, p.cols, true);
    sm100::tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  sm100::cluster_sync();
  // slots that share this block's first or last rows with other blocks: each of those takes a share of the 128 rows
  const uint32_t base = sm100::smem_addr(part);
  for (int k = 0; k < 2 && b1 > b0; ++k) {
    const int slot = __ldg(&blocks[k ? b1 - 1 : b0]).z;
    const int first = __ldg(p.plan.block_start + slot), end = __ldg(p.plan.block_start + slot + 1);
    if (k ? (end <= b1 || (began && slot == __ldg(&blocks[b0]).z)) : !began) continue;
    int lo = 0, hi = p.ranks - 1;
    while (cut(lo + 1) <= first) ++lo;
    while (cut(hi) >= end) --hi;
    const int r0 = BM * (rank - lo) / (hi - lo + 1), rows = BM * (rank - lo + 1) / (hi - lo + 1) - r0;
    for (int i = threadIdx.x; i < rows * (p.R / 4); i += kThreads) {
      int r, c;
      g.place(i, r0, rows, r, c);
      // (the block where the slot begins keeps it as its last, the others as their first)
      const uint32_t at = base + (r * (p.cols + 4) + c) * 4;
      float4 v = ld_cluster4(sm100::mapa(at + part_floats * 4, lo));
      for (int j = lo + 1; j <= hi; ++j) {
        if (cut(j) == cut(j + 1)) continue;
        const float4 o = ld_cluster4(sm100::mapa(at, j));
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      g.put(slot, r, c, v);
    }
  }
  if (!g.add)        // slots without rows
    for (int s = rank; s < p.S; s += p.ranks) {
      if (s < p.plan.slots && __ldg(p.plan.block_start + s + 1) > __ldg(p.plan.block_start + s)) continue;
      for (int i = threadIdx.x; i < BM * (p.R / 4); i += kThreads) {
        int r, c;
        g.place(i, 0, BM, r, c);
        g.put(s, r, c, make_float4(0.f, 0.f, 0.f, 0.f));
      }
    }
  sm100::cluster_sync();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------------------------------------ host
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// Row-major [batch][rows, cols] of 16-bit values, boxes of 64 columns x `box` rows, 128-byte swizzle.  Reads outside
// give zeros, in each of the three dimensions: a box never reaches into the next slot.
bool encode(CUtensorMap* m, const void* base, long cols, long rows, long ld, long batch, int box, bool half) {
  const auto fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)std::max(1l, batch)};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(ld * 2 * rows)};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)box, 1}, ones[3] = {1, 1, 1};
  return fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, batch ? 3 : 2,
            const_cast<void*>(base), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The encoder works in the calling thread's context, which a thread of autograd's may not have yet.
cudaError_t have_context() {
  CUcontext cur = nullptr;
  if (cuCtxGetCurrent(&cur) == CUDA_SUCCESS && cur != nullptr) return cudaSuccess;
  return cudaFree(nullptr);
}

int sm_count() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

constexpr int kMaxSmem = 227 * 1024;

template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || ((done.load() >> (dev & 63)) & 1)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(1ull << (dev & 63));
  return e;
}

// The kernel may begin while the one before it in the stream ends (it waits by itself for what that one wrote).
// `cluster`: blocks of one, 0 where the kernel says it itself.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                   const A&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  int n = 0;
  if (cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
  }
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) launch_counter().fetch_add(1);
  return e;
}

// Blocks of a cluster: as many, at most 8, as let all clusters run at once, each with four steps of 64 of the sum; more than
// one per SM only if each has eight.  More blocks mean more loads in flight, but each costs its start and its part in
// the joining of sums.  Measured: one row through 2560 -> 6144 (48 clusters) 16.9, 11.1, 9.3, 9.6 us with 1, 2, 4 and 6
// blocks; the shrink of 71 tiles over K = 9728 68, 48, 44, 53 us with 1, 2, 4 and 6, of 30 over 2048 3 us more with 8 than
// with 4.  (Clusters lie within a GPC, so how many fit is less than blocks over SMs: 15 of 8 with a block to an SM, not 18.
// The runtime counts one block of a kernel with TMEM to an SM; there are as many as its shared memory and its `columns`
// of TMEM leave room for.)
template <typename... P>
int split(void (*kernel)(P...), int smem, int columns, int clusters, int nk) {
  struct Fit {
    const void* kernel;
    int device, smem, fits[9];
  };
  static std::mutex lock;
  static std::vector<Fit> known;
  int dev = 0;
  cudaGetDevice(&dev);
  const std::lock_guard<std::mutex> hold(lock);
  const void* key = reinterpret_cast<const void*>(kernel);
  const Fit* fit = nullptr;
  for (const Fit& f : known)
    if (f.kernel == key && f.device == dev && f.smem == smem) fit = &f;
  if (!fit) {
    Fit f{key, dev, smem, {}};
    for (int r = 2; r <= 8; ++r) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = r, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(r), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr, cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&f.fits[r], kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        f.fits[r] = 0;
      }
    }
    known.push_back(f);
    fit = &known.back();
  }
  const int sms = sm_count(), per_sm = std::max(1, std::min(kMaxSmem / (smem + 1024), 512 / columns));
  int ranks = 8;
  const auto fits = [&](int r) { return clusters <= per_sm * fit->fits[r] && nk >= (clusters * r > sms ? 8 : 4) * r; };
  while (ranks > 1 && !fits(ranks)) --ranks;
  return ranks;
}

uint16_t* rest_of(const AdapterProduct& a) {
  return a.keep_u ? static_cast<uint16_t*>(a.u) + (size_t)a.T * a.R : nullptr;
}

template <bool OP_MN>
cudaError_t run_shrink(const AdapterProduct& a, cudaStream_t stream) {
  alignas(64) CUtensorMap x, op;
  const int cols = OP_MN ? (a.R + 63) / 64 * 64 : (a.R + 15) / 16 * 16;
  if (!encode(&x, a.x, a.K, a.T, a.ldx, 0, BM, a.half)) return cudaErrorInvalidValue;
  if (!(OP_MN ? encode(&op, a.op, a.R, a.K, a.R, a.S, 64, a.half) : encode(&op, a.op, a.K, a.R, a.K, a.S, cols, a.half)))
    return cudaErrorInvalidValue;
  ShrinkParams p{};
  p.plan = a.plan;
  p.u = static_cast<uint16_t*>(a.u), p.rest = rest_of(a);
  p.scales = a.scales, p.scale = a.scale;
  p.T = a.T, p.R = a.R, p.cols = cols;
  p.op_bytes = cols * 128;
  p.nk = (a.K + BK - 1) / BK;
  p.stages = 4;
  p.idesc = sm100::umma_idesc_bf16(BM, cols, false, OP_MN) & ~(a.half ? sm100::kIdescBf16 : 0u);
  p.half = a.half;
  const int smem = std::max(p.stages * (kXBytes + p.op_bytes), BM * (cols + 4) * 4) + 256 + 1024;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(adapter_shrink_kernel<OP_MN>, kMaxSmem, done);
  if (e != cudaSuccess) return e;
  p.ranks = split(adapter_shrink_kernel<OP_MN>, smem, 128, a.plan.num_units, p.nk);
  return launch(adapter_shrink_kernel<OP_MN>, a.plan.num_units * p.ranks, kThreads, smem, p.ranks, stream, x, op, p);
}

cudaError_t run_dots(const AdapterProduct& a, cudaStream_t stream) {
  DotsParams p{};
  p.plan = a.plan;
  p.x = static_cast<const uint16_t*>(a.x), p.op = static_cast<const uint16_t*>(a.op), p.u = static_cast<uint16_t*>(a.u);
  p.rest = rest_of(a);
  p.scales = a.scales, p.scale = a.scale;
  p.ldx = a.ldx, p.K = a.K, p.R = a.R;
  const dim3 grid(a.plan.num_units * (a.R / 2), (a.T + kDotRows - 1) / kDotRows);
  return a.half ? launch(adapter_dots_kernel<true>, grid, 32 * kDotWarps, 0, 0, stream, p)
                : launch(adapter_dots_kernel<false>, grid, 32 * kDotWarps, 0, 0, stream, p);
}

// Rows and ranks up to which u is made by dot products: 2560 -> 6144, whole calls, dots and tensor cores: 8 rows of 8 slots,
// rank 16, 11.7 and 13.9 us; 64 rows of 2, rank 16, 16.7 and 17.6; 8 rows of 8 slots, rank 64, 15.2 and 14.1; 64 rows of 8
// slots, rank 32, over 9728 32 and 24.
bool few_dots(const AdapterProduct& a) { return !a.mn && a.R <= 32 && (long)a.T * a.R <= 1024; }

// Which kernel makes the joint product.  Up to 128 rows the read of W is all there is, and clusters that split K read it
// fastest; further on as long as tiles of 128 x 128 are few (to a cluster of 3 blocks or more each) and K is long:
// 4096 -> 2560, 256 rows (40 tiles): 18 us, on pairs of SMs 23; 2560 -> 6144, 256 rows (96 tiles): 22 and 18; 256 -> 512,
// 256 rows: 11 and 8.5.
bool few_rows(int T, int K, int N) {
  const long tiles = (long)((T + BM - 1) / BM) * ((N + BM - 1) / BM);
  return T <= BM || (tiles <= 48 && K >= 2048);
}

template <bool MN>
cudaError_t run_few(const AdapterProduct& a, cudaStream_t stream) {
  alignas(64) CUtensorMap x, w, u, low;
  const int rows = std::min(BM, (a.T + 7) / 8 * 8), m_tiles = (a.T + BM - 1) / BM;
  // Where tiles of 128 columns are a few more than SMs, some SMs would have two and the rest one: wider tiles, one to each.
  // 2560 -> 19456, 152 tiles of 128 and 136 of 144: 1 row 19.4 and 18.7 us, 61 rows 23.2 and 21.4, 128 rows 27.9 and 25.5;
  // 176 tiles and 141: 19.0 and 18.5; 282 tiles and 141 of 256: 31.9 and 32.5.
  constexpr int kWidest = 176;
  int cols = BM;
  if (!MN && m_tiles * ((a.N + kWidest - 1) / kWidest) <= sm_count())
    while (m_tiles * ((a.N + cols - 1) / cols) > sm_count()) cols += 16;
  bool ok = encode(&x, a.x, a.K, a.T, a.ldx, 0, rows, a.half) && encode(&u, a.u, a.R, a.T, a.R, 0, rows, a.half);
  if (MN) ok = ok && encode(&w, a.w, a.N, a.K, a.ldw, 0, 64, a.half) && encode(&low, a.low, a.N, a.R, a.N, a.S, 64, a.half);
  else ok = ok && encode(&w, a.w, a.K, a.N, a.ldw, 0, cols, a.half) && encode(&low, a.low, a.R, a.N, a.R, a.S, cols, a.half);
  if (!ok) return cudaErrorInvalidValue;
  FewParams p{};
  p.plan = a.plan;
  p.y = static_cast<uint16_t*>(a.y);
  p.T = a.T, p.N = a.N, p.R = a.R, p.rows = rows, p.cols = cols;
  p.nk = (a.K + BK - 1) / BK;
  const int tiles = m_tiles * ((a.N + cols - 1) / cols), stage = (rows + cols) * 128;
  // 69 to 128 KB; where tiles outnumber the SMs, little enough for two blocks to an SM.  (128 rows, 4 stages: 14.7 us with
  // 2 blocks a cluster and one to an SM, 18 with 3 stages and more of them; 152 tiles: 27 us with 3 stages, 42 with 4.)
  p.stages = tiles > sm_count() ? std::min(4, 110 * 1024 / stage) : 4;
  p.idesc = sm100::umma_idesc_bf16(BM, cols, false, MN) & ~(a.half ? sm100::kIdescBf16 : 0u);
  p.half = a.half;
  int smem = std::max(p.stages * stage, std::min(BM, a.T) * (cols + 4) * 4) + 256 + BM * 20 + 1024;
  if (cols > 128) smem = std::max(smem, 80 * 1024);      // (with 256 columns of TMEM: see the gradients)
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(adapter_few_kernel<MN>, kMaxSmem, done);
  if (e != cudaSuccess) return e;
  p.ranks = split(adapter_few_kernel<MN>, smem, cols <= 128 ? 128 : 256, tiles, p.nk);
  return launch(adapter_few_kernel<MN>, tiles * p.ranks, kThreads, smem, p.ranks, stream, x, w, u,
                low, p);
}

// Columns of the accumulator that a batch's slots take beside y's 128 in the one-kernel form, or 0 where it does not apply.
// Its low-rank part goes by rows x rank, its reading by the slots; what it saves is a launch (4 us of the host's 11).
// 2560 -> 6144 on the device, one kernel and two: 1 row of rank 16 10.7 and 11.1 us, 4 rows of 2 slots 11.3 and 11.1, 8 rows
// of 4 slots 12.5 and 11.4, 32 rows of 4 slots 21.5 and 13.5; calls of 1 row, host included, 9.8 and 12.5.  Larger W, where
// the host is not what counts: 1 row, 2048 -> 12352 15.2 and 13.7, 9728 -> 2560 16.0 and 14.5, 2560 -> 19456 28.3 and 20.6.
int token_columns(const AdapterProduct& a) {
  const long each = a.mn ? (a.R + 63) / 64 * 64 : (a.R + 15) / 16 * 16, all = a.plan.num_units * each;
  return (long)a.T * a.R <= 64 && all <= (a.mn ? 64 : 32) && (long)a.K * a.N <= 1 << 24 ? all : 0;
}

template <bool MN>
cudaError_t run_token(const AdapterProduct& a, int u_cols, cudaStream_t stream) {
  alignas(64) CUtensorMap x, w, op;
  const int rows = (a.T + 7) / 8 * 8, each = u_cols / a.plan.num_units;
  bool ok = encode(&x, a.x, a.K, a.T, a.ldx, 0, rows, a.half);
  if (MN) ok = ok && encode(&w, a.w, a.N, a.K, a.ldw, 0, 64, a.half) && encode(&op, a.op, a.R, a.K, a.R, a.S, 64, a.half);
  else ok = ok && encode(&w, a.w, a.K, a.N, a.ldw, 0, BM, a.half) && encode(&op, a.op, a.K, a.R, a.K, a.S, each, a.half);
  if (!ok) return cudaErrorInvalidValue;
  TokenParams p{};
  p.plan = a.plan;
  p.y = static_cast<uint16_t*>(a.y), p.u = a.keep_u && !MN ? static_cast<uint16_t*>(a.u) : nullptr;
  p.low = static_cast<const uint16_t*>(a.low);
  p.scales = a.scales, p.scale = a.scale;
  p.T = a.T, p.N = a.N, p.R = a.R, p.rows = rows, p.slot_cols = each;
  p.nk = (a.K + BK - 1) / BK;
  p.columns = 256;
  const int stage = rows * 128 + kXBytes + u_cols * 128, tiles = (a.N + BM - 1) / BM;
  p.stages = std::min(4, 220 * 1024 / stage);
  p.idesc = sm100::umma_idesc_bf16(BM, BM + u_cols, false, MN) & ~(a.half ? sm100::kIdescBf16 : 0u);
  p.half = a.half;
  int smem = std::max(p.stages * stage, a.T * (BM + u_cols + 4) * 4 + a.T * a.R * 2) + 256 + 1024;
  // (three blocks of 256 columns must not meet on an SM: see the gradients)
  smem = std::max(smem, 80 * 1024);
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(adapter_token_kernel<MN>, kMaxSmem, done);
  if (e != cudaSuccess) return e;
  p.ranks = split(adapter_token_kernel<MN>, smem, p.columns, tiles, p.nk);
  return launch(adapter_token_kernel<MN>, tiles * p.ranks, kThreads, smem, p.ranks, stream, x, w, op, p);
}

// How the tiles of 256 x 256 go to the pairs of SMs.
struct Cut {
  int pairs, whole, slices, units;
};

// A last round of `rest` tiles takes a whole tile's time of nk blocks of K; cut into slices nk / slices, the slices' sums
// (256 KB each, through L2) and another launch, together about 10 us or 28 blocks' time.
Cut cut_tiles(int T, int K, int N) {
  const int tiles = (T + 255) / 256 * ((N + 255) / 256), nk = (K + BK - 1) / BK, pairs = std::max(1, sm_count() / 2);
  Cut c{pairs, tiles, 1, tiles};
  const int rest = tiles % pairs;
  const int slices = rest ? std::min({8, pairs / rest, nk / 4}) : 1;
  if (slices >= 2 && nk - nk / slices > 28) {
    c.whole = tiles - rest;
    c.slices = slices;
    c.units = c.whole + rest * slices;
  }
  c.pairs = std::min(pairs, c.units);
  return c;
}

template <bool MN>
cudaError_t run_joint(const AdapterProduct& a, cudaStream_t stream) {
  alignas(64) CUtensorMap x, w, u, low, y;
  bool ok = encode(&x, a.x, a.K, a.T, a.ldx, 0, BM, a.half) && encode(&u, a.u, a.R, a.T, a.R, 0, BM, a.half) &&
            encode(&y, a.y, a.N, a.T, a.N, 0, 32, a.half);
  if (MN) ok = ok && encode(&w, a.w, a.N, a.K, a.ldw, 0, 64, a.half) && encode(&low, a.low, a.N, a.R, a.N, a.S, 64, a.half);
  else ok = ok && encode(&w, a.w, a.K, a.N, a.ldw, 0, BM, a.half) && encode(&low, a.low, a.R, a.N, a.R, a.S, BM, a.half);
  if (!ok) return cudaErrorInvalidValue;
  const Cut c = cut_tiles(a.T, a.K, a.N);
  JointParams p{};
  p.plan = a.plan;
  p.y = static_cast<uint16_t*>(a.y);
  p.sums = static_cast<float*>(a.workspace);
  p.T = a.T, p.N = a.N, p.R = a.R;
  p.nk = (a.K + BK - 1) / BK;
  // Wide products like larger groups (W is read once per group), tall ones smaller: 8192 rows, 2560 -> 19456, groups of 4,
  // 8, 16, 32: 643, 623, 607, 609 us under a sustained power cap; 9728 -> 2560: 316, 320, 324, 338.
  const int m_tiles = (a.T + 255) / 256, n_tiles = (a.N + 255) / 256;
  p.group = n_tiles >= 2 * m_tiles ? 16 : m_tiles >= 2 * n_tiles ? 4 : 8;
  p.whole = c.whole, p.slices = c.slices, p.units = c.units;
  p.idesc = sm100::umma_idesc_bf16(256, 256, false, MN) & ~(a.half ? sm100::kIdescBf16 : 0u);
  p.half = a.half;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(adapter_joint_kernel<MN>, kPairSmem, done);
  if (e != cudaSuccess) return e;
  e = launch(adapter_joint_kernel<MN>, 2 * c.pairs, kThreads, kPairSmem, 0, stream, x, w, u, low, y, p);
  if (e != cudaSuccess || c.units == c.whole) return e;
  return launch(adapter_join_kernel, (c.units - c.whole) / c.slices * 16, 256, 0, 0, stream, p);
}

}  // namespace

cudaError_t launch_adapter_shrink(const AdapterProduct& a, cudaStream_t stream) {
  const cudaError_t e = have_context();
  if (e != cudaSuccess || a.plan.num_units == 0) return e;
  if (few_dots(a)) return run_dots(a, stream);
  return a.mn ? run_shrink<true>(a, stream) : run_shrink<false>(a, stream);
}

AdapterNeeds adapter_product_needs(const AdapterProduct& a) {
  if (a.plan.num_units && token_columns(a)) return {a.keep_u, 0};
  if (few_rows(a.T, a.K, a.N)) return {true, 0};
  const Cut c = cut_tiles(a.T, a.K, a.N);
  return {true, (size_t)(c.units - c.whole) * kPairTile * sizeof(float)};
}

cudaError_t launch_adapter_product(const AdapterProduct& a, cudaStream_t stream) {
  cudaError_t e = have_context();
  if (e != cudaSuccess) return e;
  if (a.plan.num_units)
    if (const int columns = token_columns(a)) {
      if (a.mn && a.keep_u) e = launch_adapter_shrink(a, stream);
      if (e != cudaSuccess) return e;
      return a.mn ? run_token<true>(a, columns, stream) : run_token<false>(a, columns, stream);
    }
  e = launch_adapter_shrink(a, stream);
  if (e != cudaSuccess) return e;
  if (few_rows(a.T, a.K, a.N)) return a.mn ? run_few<true>(a, stream) : run_few<false>(a, stream);
  return a.mn ? run_joint<true>(a, stream) : run_joint<false>(a, stream);
}

cudaError_t launch_adapter_grads(const AdapterGrads& a, cudaStream_t stream) {
  cudaError_t e = have_context();
  if (e != cudaSuccess) return e;
  alignas(64) CUtensorMap x, dy, u, du;
  // (an operand that is not asked for has no pointer: any valid map stands in for its own)
  const bool ok = encode(&x, a.da ? a.x : a.dy, a.da ? a.K : a.N, a.T, a.da ? a.ldx : a.lddy, 0, 64, a.half) &&
                  encode(&dy, a.db ? a.dy : a.x, a.db ? a.N : a.K, a.T, a.db ? a.lddy : a.ldx, 0, 64, a.half) &&
                  encode(&u, a.db ? a.u : a.du, a.R, a.T, a.R, 2, 64, a.half) &&
                  encode(&du, a.da ? a.du : a.u, a.R, a.T, a.R, 2, 64, a.half);
  if (!ok) return cudaErrorInvalidValue;
  GradParams p{};
  p.plan = a.plan;
  p.da = a.da, p.db = a.db;
  p.K = a.K, p.N = a.N, p.S = a.S, p.R = a.R;
  p.cols = (a.R + 63) / 64 * 64;
  p.tiles_a = a.da ? (a.K + BM - 1) / BM : 0;
  p.tiles_b = a.db ? (a.N + BM - 1) / BM : 0;
  p.idesc = sm100::umma_idesc_bf16(BM, p.cols, true, true) & ~(a.half ? sm100::kIdescBf16 : 0u);
  p.add_a = a.add_a, p.add_b = a.add_b, p.half = a.half;
  const int smem = std::max(grad_stages(p.cols) * (kXBytes + p.cols * 256), 2 * BM * (p.cols + 4) * 4) + 256 + 1024;
  // Blocks that hold all of an SM's TMEM have the SM for themselves: of two clusters that wait for each other's, each in
  // another SM, neither would end.  (With 512 columns they take 193 KB of shared memory, with 256 97; all other blocks here
  // 69 KB or more, 80 with 256 columns: what room there is for blocks is room for their columns.)
  static std::atomic<unsigned long long> done{0};
  e = allow_smem(adapter_grads_kernel, kMaxSmem, done);
  if (e != cudaSuccess) return e;
  // (cut as for both gradients, so that one does not depend on whether the other is asked for)
  const int tiles = p.tiles_a + p.tiles_b, both = (a.K + BM - 1) / BM + (a.N + BM - 1) / BM;
  p.ranks = split(adapter_grads_kernel, smem, p.cols == 64 ? 256 : 512, both, std::max(1, a.plan.num_blocks));
  return launch(adapter_grads_kernel, tiles * p.ranks, kThreads, smem, p.ranks, stream, x, dy, u, du, p);
}

int adapter_error_code() {
  int v = -1;
  return cudaMemcpyFromSymbol(&v, g_error, sizeof v) == cudaSuccess ? v : -1;
}

}  // namespace bb
