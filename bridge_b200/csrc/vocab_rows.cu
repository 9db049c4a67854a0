// Kernels over rows of logits x [U, V]: log-probs of given tokens with entropy and the k likeliest tokens, their
// gradient, and the loss + gradient of distillation from a teacher known by its top log-probs.
//
// Everything is written in the base-2 domain of one row: c = log2(e) / T, t = x c - R for a reference R near the
// row's largest x c, e = 2^t, s = sum e.  Then p = e / s, ln p = ln 2 (t - log2 s), and the entropy is
// ln 2 (log2 s - sum e t / s), whatever R is: every thread keeps its own R, and partial (R, s, sum e t) triples are
// joined by rescaling.  Statistics are FP32; the few numbers of a row that everything else is scaled by (log s, the
// given tokens' shares) are FP64.
//
// A logit with x c <= -2^31 (-inf, the type's lowest value, any customary finite mask from -1e10 down) carries no
// probability; a row without any other has log-probs -inf, entropy 0 and gradient 0.  (In a row with others its own
// log-prob is what the fill makes it, and -inf from x c = -1e30 down.)  The bound is where FP32 ends: R is
// rounded, so t at the largest logit can be off 0 by half a unit of R's last place, 64 for |R| < 2^31 (2^64 V is still a
// number) and hundreds above, where a thread that sees nothing but a mask of -1e10 would sum to infinity.  A row with
// x c > 2^31 is NaN, as with an infinite logit.
//
// A row belongs to one cluster of 1 to 8 blocks, each with a contiguous slice; the blocks exchange partial sums
// through distributed shared memory, so no workspace and no atomics on global memory are needed and results do not
// depend on timing.
//
// What bounds them: reading the row.  8 BF16 logits cost 16 bytes, 8 exponentials (half a cycle of an SM) and about
// 40 instructions a pass, which at 6.4 TB/s is two thirds of what the SMs can issue, so the loops are kept lean (paired
// FP32 instructions, no checks inside a row) and everything that is per row overlaps other blocks' streaming.  B200,
// vocabulary 151936, BF16, device time: scoring 4096 rows with entropy 0.20 ms (6.1 TB/s at full clocks; 0.23 ms, 5.4 TB/s,
// among other calls under a sustained power cap), 1024 rows with 64 alternatives 0.076 ms; gradient of the scores 0.21 ms
// for 2048 rows (6.0 TB/s); distillation loss 0.059 ms for 1024 rows, loss and gradient 0.48 ms for 4096 (5.2 TB/s of one
// read and one write); one row with 20 alternatives 9 us, 8 rows of distillation with gradient 15 us in three launches.
#include "vocab_rows.h"

#include <c10/util/Exception.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace {

namespace cg = cooperative_groups;
using bb::DistillArgs;
using bb::kMaxTop;
using bb::RowType;
using bb::TokenArgs;

constexpr int kThreads = 512;   // at most, per block that holds its slice
constexpr int kStream = 256;    // per block that streams it
constexpr int kMaxCluster = 8;
constexpr int kCand = 2048;     // candidates of the selection kept in shared memory
constexpr float kFloor = -2147483648.f;       // -2^31, of x c: least reference of a sum
constexpr float kMasked = -1e30f;             // of x c: as good as -inf
constexpr float kOverflow = -1e29f;           // x c below this may be -inf
constexpr float kSlack = 8.f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// 2^d, log2 z and 1 / a in FP64 to about 1e-10, for the few numbers of a row that are on every block's critical path:
// short dependent chains (a Taylor series of 2^f on |f| <= 1/2, the artanh series of log2 on [sqrt 1/2, sqrt 2], one
// Newton step on an FP32 reciprocal) instead of full-precision functions.
__device__ __forceinline__ double rcp_d(double a) {      // a within FP32's normal range
  const double r = (double)(1.f / (float)a);
  return r * (2.0 - a * r);
}
__device__ __forceinline__ double exp2_d(double d) {     // 0 below 2^-1000; no branches, so calls overlap
  const double b = d < -1000.0 ? -1000.0 : (d > 1000.0 ? 1000.0 : d);
  const int n = __double2int_rn(b);
  const double f = (b - (double)n) * kLn2;
  double p = 1.0 / 40320.0;
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  p *= __hiloint2double((1023 + n) << 20, 0);
  return d < -1000.0 ? 0.0 : (d > 1000.0 ? INFINITY : p);
}
__device__ __forceinline__ double log2_d(double z) {     // -inf at 0; z >= 0, normal
  const int hi = __double2hiint(z);
  const double m1 = __hiloint2double((hi & 0xfffff) | (1023 << 20), __double2loint(z));
  const bool up = m1 > 1.4142135623730951;
  const double m = up ? 0.5 * m1 : m1;
  const int n = (hi >> 20) - 1023 + (up ? 1 : 0);
  const double s = (m - 1.0) * rcp_d(m + 1.0), q = s * s;
  double p = 1.0 / 13.0;
  p = fma(p, q, 1.0 / 11.0);
  p = fma(p, q, 1.0 / 9.0);
  p = fma(p, q, 1.0 / 7.0);
  p = fma(p, q, 1.0 / 5.0);
  p = fma(p, q, 1.0 / 3.0);
  p = fma(p, q, 1.0);
  p = fma(2.0 * kLog2e * s, p, (double)n);
  return z == 0.0 ? -INFINITY : (z < INFINITY ? p : z);      // (NaN and infinity as they are)
}

// ------------------------------------------------------------------------------------------------- rows
// 16 bytes of a row: 8 elements of 16 bits, or 4 of 32.
template <typename T>
struct Unit {
  static constexpr int kE = 16 / (int)sizeof(T);
  uint4 w;

  __device__ __forceinline__ T get(int j) const { return reinterpret_cast<const T*>(&w)[j]; }
  __device__ __forceinline__ void set(int j, T v) { reinterpret_cast<T*>(&w)[j] = v; }
  __device__ __forceinline__ void fill(T v) {
#pragma unroll
    for (int j = 0; j < kE; ++j) set(j, v);
  }
  __device__ __forceinline__ void mask(unsigned m) {      // -inf where a bit is set
#pragma unroll
    for (int j = 0; j < kE; ++j)
      if (m >> j & 1u) set(j, from_f<T>(-INFINITY));
  }
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (sizeof(T) == 4) return make_float2(get(2 * j), get(2 * j + 1));
    const uint32_t h = reinterpret_cast<const uint32_t*>(&w)[j];
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
    else
      return __half22float2(reinterpret_cast<const __half2&>(h));
  }
  __device__ __forceinline__ void set_pair(int j, float2 f) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      reinterpret_cast<__nv_bfloat162*>(&w)[j] = __floats2bfloat162_rn(f.x, f.y);
    else if constexpr (std::is_same_v<T, __half>)
      reinterpret_cast<__half2*>(&w)[j] = __floats2half2_rn(f.x, f.y);
    else
      set(2 * j, f.x), set(2 * j + 1, f.y);
  }
  __device__ __forceinline__ float max() const {          // NaN does not count
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(get(0), get(1)), fmaxf(get(2), get(3)));
    } else {
      using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      const T2* h = reinterpret_cast<const T2*>(&w);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(to_f(m.x), to_f(m.y));
    }
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// One row as units on 16-byte boundaries: unit i covers the aligned positions kE i .. kE i + kE - 1, and position a
// holds token a - shift.  Only the first and the last unit can be partly outside the row.
template <typename T>
struct Row {
  using V = std::remove_const_t<T>;
  static constexpr int kE = Unit<V>::kE;
  T* p;        // aligned base: row start - shift
  int shift;   // elements between the 16-byte boundary and the row's first element
  int end;     // V + shift
  int units;

  __device__ __forceinline__ Row(T* row, int vocab) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    p = row - shift;
    end = vocab + shift;
    units = (end + kE - 1) / kE;
  }
  __device__ __forceinline__ bool full(int i) const { return kE * i >= shift && kE * i + kE <= end; }
  __device__ __forceinline__ bool holds(int a) const { return a >= shift && a < end; }
  __device__ __forceinline__ Unit<V> load(int i) const {
    Unit<V> u;
    if (full(i)) {
      u.w = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) u.set(j, holds(kE * i + j) ? p[kE * i + j] : from_f<V>(-INFINITY));
    }
    return u;
  }
  // Stores the unit that covers the INPUT's positions kE i ..; `vec`: this row and the input's start at the same
  // offset from a 16-byte boundary.
  __device__ __forceinline__ void store(int i, const Unit<V>& u, bool vec, int in_shift) const {
    if (vec && full(i)) {
      reinterpret_cast<uint4*>(p)[i] = u.w;
    } else {
      const int a0 = kE * i - in_shift + shift;
#pragma unroll
      for (int j = 0; j < kE; ++j)
        if (holds(a0 + j)) p[a0 + j] = u.get(j);
    }
  }
};

// The block's slice of the row's units.
struct Slice {
  int lo, hi;
  __device__ __forceinline__ Slice(int units, int blocks, int rank) {
    const int per = (units + blocks - 1) >> (31 - __clz(blocks));      // (blocks is a power of two)
    lo = min(units, rank * per);
    hi = min(units, lo + per);
  }
};

// --------------------------------------------------------------------------------------------- statistics
struct Stat {
  float R, s, et;

  static __device__ __forceinline__ Stat none() { return {kFloor, 0.f, 0.f}; }
  __device__ __forceinline__ void raise(float to) {
    const float d = R - to, k = ex2(d);
    et = k * (et + d * s);
    s *= k;
    R = to;
  }
};

// The reference for a largest x c of `top`.
__device__ __forceinline__ float reference(float top) { return top > -kFloor ? NAN : fmaxf(top, kFloor); }

// A thread's running sums, two FP32 lanes to an instruction.
struct Sums {
  float R;
  float2 s, et;

  __device__ __forceinline__ Sums() : R(kFloor), s(both(0.f)), et(both(0.f)) {}
  __device__ __forceinline__ void raise(float to) {
    const float d = R - to, k = ex2(d);
    et = __fmul2_rn(both(k), __ffma2_rn(both(d), s, et));
    s = __fmul2_rn(both(k), s);
    R = to;
  }
  // kMask: some t may be -inf, whose e = 0 would make e t NaN
  template <bool kEntropy, bool kMask, typename T>
  __device__ __forceinline__ void add(const Unit<T>& u, float c) {
#pragma unroll
    for (int j = 0; j < Unit<T>::kE / 2; ++j) {
      float2 t = __ffma2_rn(u.pair(j), both(c), both(-R));
      const float2 e = make_float2(ex2(t.x), ex2(t.y));
      s = __fadd2_rn(s, e);
      if (kEntropy && kMask) t = make_float2(fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f));
      if (kEntropy) et = __ffma2_rn(e, t, et);
    }
  }
  __device__ __forceinline__ Stat get() const { return {R, s.x + s.y, et.x + et.y}; }
};

// (Volatile: it may not sink into a branch that only the lanes that use it take.)
__device__ __forceinline__ float warp_top(float v) {
  asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
  return v;
}

// Sum over the first kLanes lanes' triples (the other lanes hold none), in every one of those lanes.
template <int kLanes = 32>
__device__ __forceinline__ Stat warp_join(Stat a) {
  a.raise(warp_top(a.R));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.et += __shfl_xor_sync(0xffffffffu, a.et, o);
  }
  return a;
}

// The block's joined statistics, in every thread.  `part` holds 32 triples.
__device__ __forceinline__ Stat block_join(Stat a, Stat* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  a = warp_join(a);
  __syncthreads();
  if (lane == 0) part[warp] = a;
  __syncthreads();
  Stat b = Stat::none();
  if (lane < (int)(blockDim.x >> 5)) b = part[lane];
  return warp_join(b);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_max_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// A block's slice on its way through shared memory.  A warp takes batches of 4 x 32 consecutive units, warp w the
// batches w, w + warps, ...; every lane owns kGroups x 4 slots of 16 bytes that it alone fills (asynchronous copies)
// and reads, so a warp waits for nothing but its own copies, which run kGroups batches ahead, from before the first
// batch is needed.  With two passes the batches come once more in reverse order: the last are in their slots still, and
// what was read late is the likeliest to be in L2.  A warp barrier orders the reads of a batch's slots before the copies
// that refill them.
//
// 3 groups of 16 KB for 8 warps are 48 KB a block, 4 blocks an SM.  Distillation with gradient of 4096 x 151936 BF16, each
// step alone: 627 us with plain loads, the second pass in the order of the first; 593 us in reverse order with the stores
// and last reads marked evict-first; 533 us with the copies.
constexpr int kBatch = 4, kGroups = 3, kSpan = 32 * kBatch;
static_assert(kBatch == 4, "a batch is written out unit by unit");

__device__ __forceinline__ unsigned long long evict_first() {
  unsigned long long p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ unsigned long long evict_normal() {
  unsigned long long p;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
template <int b>
__device__ __forceinline__ void store_streaming(uint4* p, uint4 v, unsigned long long policy) {
  asm volatile("st.global.L2::cache_hint.v4.b32 [%0 + %6], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w), "l"(policy), "n"(512 * b)
               : "memory");
}

// The batches at a slice's ends, out of the way of the others.  Lane's units i, i + 32, ..: those within [lo, hi) can be
// copied; the others are read one element at a time (-inf outside the slice, which ends at `stop`).
static __device__ __noinline__ void copy_edge(uint32_t to, const uint4* from, int i, int lo, int hi) {
  for (int b = 0; b < kBatch; ++b)
    if (i + 32 * b >= lo && i + 32 * b < hi)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * b), "l"(from + 32 * b) : "memory");
}
template <typename T>
__device__ __noinline__ void read_edge(uint32_t to, const T* p, int shift, int end, int i, int lo, int hi, int stop) {
  constexpr int kE = Unit<T>::kE;
  for (int b = 0; b < kBatch; ++b, i += 32) {
    if (i >= lo && i < hi) continue;
    Unit<T> u;
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const int a = kE * i + j;
      u.set(j, i < stop && a >= shift && a < end ? p[a] : from_f<T>(-INFINITY));
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 512 * b), "r"(u.w.x), "r"(u.w.y), "r"(u.w.z),
                 "r"(u.w.w)
                 : "memory");
  }
}

// (Only two passes give L2 hints: what is read once needs none.)
template <typename T, int kPasses>
struct Feed {
  static constexpr int kGroupBytes = kSpan * 16;
  uint32_t ring;         // this lane's first slot (shared address)
  const uint4* p;        // this lane's unit of the warp's first batch
  int first, step;       // the warp's first unit (in the row), units between its batches
  int lo, hi;            // units of the row that can be copied: full ones, inside the slice
  int batches, ready;    // of this warp, and of them those to copy (none of a row that is not read)
  int inner_lo, inner_n; // batches all of whose units can be copied: the first, and how many
  uint32_t put, get;     // offsets of the slots to fill and to read

  static __host__ __device__ size_t bytes(int threads) { return (size_t)threads / 32 * kGroups * kGroupBytes; }
  // `live`: whether there is anything to read
  __device__ __forceinline__ Feed(unsigned char* smem, const Row<const T>& row, Slice sl, bool live = true) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    ring = (uint32_t)__cvta_generic_to_shared(smem) + (warp * kGroups * kGroupBytes + lane * 16);
    first = sl.lo + warp * kSpan;
    step = warps * kSpan;                       // (a power of two)
    const int shift = 31 - __clz(step);
    p = reinterpret_cast<const uint4*>(row.p) + first + lane;
    lo = max(sl.lo, row.shift ? 1 : 0);
    hi = min(sl.hi, row.end / Unit<T>::kE);
    batches = first < sl.hi ? (sl.hi - first + step - 1) >> shift : 0;
    ready = live ? batches : 0;
    inner_lo = first < lo ? 1 : 0;
    inner_n = max(0, (hi - first >= kSpan ? ((hi - first - kSpan) >> shift) + 1 : 0) - inner_lo);
    put = get = 0;
    if (!live) inner_n = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (inner(g)) issue_inner(p + g * step, evict_normal());
      else issue(g);
    }
  }
  __device__ __forceinline__ bool inner(int k) const { return (unsigned)(k - inner_lo) < (unsigned)inner_n; }
  // unit b of a lane's batch: 512 bytes on per unit, in memory and in the slots
  template <int b>
  static __device__ __forceinline__ void copy(uint32_t to, const uint4* from, unsigned long long policy) {
    if constexpr (kPasses == 2)
      asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0 + %3], [%1 + %3], 16, %2;" ::"r"(to), "l"(from),
                   "l"(policy), "n"(512 * b)
                   : "memory");
    else
      asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %2], 16;" ::"r"(to), "l"(from), "n"(512 * b) : "memory");
  }
  template <int b>
  static __device__ __forceinline__ void read(uint32_t from, uint4& v) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(from), "n"(512 * b)
                 : "memory");
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ void turn(uint32_t& at) const { at = at == (kGroups - 1) * kGroupBytes ? 0 : at + kGroupBytes; }
  // Copies of a batch whose units are all there, `from` this lane's first.
  __device__ __forceinline__ void issue_inner(const uint4* from, unsigned long long policy = 0) {
    const uint32_t to = ring + put;
    copy<0>(to, from, policy);
    copy<1>(to, from, policy);
    copy<2>(to, from, policy);
    copy<3>(to, from, policy);
    turn(put);
    commit();
  }
  // Copies of batch k: what there is of it.
  __device__ __forceinline__ void issue(int k) {
    if (k >= 0 && k < ready) {
      copy_edge(ring + put, p + k * step, first + k * step + (int)(threadIdx.x & 31), lo, hi);
      turn(put);
    }
    commit();
  }
  // The next batch, which is number k of the row, is in its slots: units that could not be copied are read here (-inf
  // outside the slice).
  __device__ __forceinline__ void wait(int k, const Row<const T>& row, Slice sl) const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
    if (!inner(k))
      read_edge<T>(ring + get, row.p, row.shift, row.end, first + k * step + (int)(threadIdx.x & 31), lo, hi, sl.hi);
  }
  // -inf at an offset of that batch from this lane's first slot
  __device__ __forceinline__ void rule_out(int offset) const {
    const uint32_t at = ring + get + offset;
    const T v = from_f<T>(-INFINITY);
    if constexpr (sizeof(T) == 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(__float_as_uint(v)) : "memory");
    else asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(reinterpret_cast<const unsigned short&>(v)) : "memory");
  }
  __device__ __forceinline__ void take(Unit<T>* u) {
    read<0>(ring + get, u[0].w);
    read<1>(ring + get, u[1].w);
    read<2>(ring + get, u[2].w);
    read<3>(ring + get, u[3].w);
    __syncwarp();      // the reads are over before a copy into these slots is issued
    turn(get);
  }
  // Second pass, from the last batch to the first: batch k's slots are those of k + kGroups, and the last batches are
  // still in theirs.  The copies that follow go where this batch was.
  __device__ __forceinline__ void take_back(int k, const Row<const T>& row, Slice sl, Unit<T>* u) {
    put = get = get == 0 ? (kGroups - 1) * kGroupBytes : get - kGroupBytes;
    const uint32_t here = get;
    wait(k, row, sl);
    take(u);
    get = here;
  }
};

// The largest (kSign = 1) or smallest (-1) element; NaN does not count.
template <int kSign, typename T, int N>
__device__ __forceinline__ float units_extreme(const Unit<T>* u) {
  const auto pick = [](auto a, auto b) {
    if constexpr (std::is_same_v<decltype(a), float>) return kSign > 0 ? fmaxf(a, b) : fminf(a, b);
    else return kSign > 0 ? __hmax2(a, b) : __hmin2(a, b);
  };
  if constexpr (sizeof(T) == 4) {
    float m = u[0].get(0);
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = pick(m, u[i / 4].get(i % 4));
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = reinterpret_cast<const T2*>(&u[0].w)[j];
#pragma unroll
      for (int n = 1; n < N; ++n) m[j] = pick(m[j], reinterpret_cast<const T2*>(&u[n].w)[j]);
    }
    m[0] = pick(pick(m[0], m[1]), pick(m[2], m[3]));
    return pick(to_f(m[0].x), to_f(m[0].y));
  }
}
template <typename T, int N>
__device__ __forceinline__ float units_max(const Unit<T>* u) {
  return units_extreme<1, T, N>(u);
}
// Whether some t of these units may be infinite.
template <typename T, int N>
__device__ __forceinline__ bool masked(const Unit<T>* u, float c) {
  return units_extreme<-1, T, N>(u) * c < kOverflow;
}
template <bool kEntropy, typename T, int N>
__device__ __forceinline__ void add_units(Sums& sums, const Unit<T>* u, float c) {
  if (kEntropy && masked<T, N>(u, c)) {
#pragma unroll
    for (int n = 0; n < N; ++n) sums.template add<kEntropy, true>(u[n], c);
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) sums.template add<kEntropy, false>(u[n], c);
  }
}

// Order-preserving map of FP32 to unsigned; -0 counts as +0 and NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  v = fmaxf(v, -INFINITY) + 0.f;
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// ---------------------------------------------------------------------------------------------- selection
// The k largest of a row, ties to the lower id.  Every thread knows the largest of its own elements.  In each of the
// cluster's C blocks the ceil(k / C)-th largest of these maxima is found by bisection; the least of the C results is
// a bound that at least k elements of the row reach, and few more do.  They are gathered in the leading block and
// ranked by counting.  Rows in which more than kCand reach the bound (many equal logits) are settled exactly by the
// leading block: the k-th largest key by bisection over the row, all above it, and the first of its equals in index
// order.
struct Select {
  unsigned long long cand[kCand];
  int count, scan[33];
};

// A value that at least k of the block's `best` reach, and not many more (0: fewer than k threads hold any).
__device__ __forceinline__ uint32_t kth_max(uint32_t best, bool any, int k) {
  constexpr int kBits = 20;      // sign, exponent and 11 bits of the significand: every FP16 and BF16 value exactly
  uint32_t bound = 0;
  if (__syncthreads_count(any) < k) return 0;
  for (int bit = 31; bit >= 32 - kBits; --bit) {
    const uint32_t trial = bound | (1u << bit);
    const int n = __syncthreads_count(any && best >= trial);
    if (n < k) continue;
    bound = trial;
    if (n <= k + (k >> 3)) break;
  }
  return bound;
}

__device__ __forceinline__ float key_value(uint32_t key) {      // the inverse of order_key
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ unsigned long long pack_key(uint32_t key, int token) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (uint32_t)token);
}

constexpr uint32_t kLowestKey = 0x007fffffu;      // of -inf

// The least value that is offered: the bound's, but -inf itself never (a row with fewer than k others is filled up).
__device__ __forceinline__ float bound_value(uint32_t bound) {
  return bound <= kLowestKey ? -3.402823466e38f : key_value(bound);
}

// Gives the elements of unit i that reach the bound to the leading block.
template <typename T>
__device__ __forceinline__ void offer(const Unit<T>& u, int i, float bound, const Row<const T>& row, Select* lead) {
  constexpr int kE = Unit<T>::kE;
  const bool full = row.full(i);
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    const float v = to_f(u.get(j));      // (NaN counts as -inf)
    if (v >= bound && (full || row.holds(kE * i + j))) {
      const int at = atomicAdd(&lead->count, 1);
      if (at < kCand) lead->cand[at] = pack_key(order_key(v), kE * i + j - row.shift);
    }
  }
}

template <typename T>
__device__ int count_ge(const Row<const T>& row, uint32_t key, int* scratch) {
  int n = 0;
  for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
    const Unit<T> u = row.load(i);
#pragma unroll
    for (int j = 0; j < Unit<T>::kE; ++j) n += row.holds(Unit<T>::kE * i + j) && order_key(to_f(u.get(j))) >= key;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = n;
  __syncthreads();
  n = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : 0;
  return __reduce_add_sync(0xffffffffu, n);
}

// The least key of the row that is at least `bound`.
template <typename T>
__device__ uint32_t least_ge(const Row<const T>& row, uint32_t bound, int* scratch) {
  uint32_t least = 0xffffffffu;
  for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
    const Unit<T> u = row.load(i);
#pragma unroll
    for (int j = 0; j < Unit<T>::kE; ++j) {
      const uint32_t key = order_key(to_f(u.get(j)));
      if (row.holds(Unit<T>::kE * i + j) && key >= bound) least = min(least, key);
    }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = (int)least;
  __syncthreads();
  least = (threadIdx.x & 31) < (blockDim.x >> 5) ? (uint32_t)scratch[threadIdx.x & 31] : 0xffffffffu;
  return __reduce_min_sync(0xffffffffu, least);
}

// One block: sel.cand[0 .. k) from the n < k candidates that are there and the first elements of key `kth`, in index
// order.
template <typename T>
__device__ void fill_equals(const Row<const T>& row, uint32_t kth, int n, int k, Select& sel) {
  constexpr int kE = Unit<T>::kE;
  for (int i0 = 0; i0 < row.units && n < k; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    uint32_t hit = 0;
    if (i < row.units) {
      const Unit<T> u = row.load(i);
#pragma unroll
      for (int j = 0; j < kE; ++j)
        if (row.holds(kE * i + j) && order_key(to_f(u.get(j))) == kth) hit |= 1u << j;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int pos = __popc(hit);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, pos, o);
      if (lane >= o) pos += v;
    }
    __syncthreads();
    if (lane == 31) sel.scan[warp] = pos;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
      if (w < warp) before += sel.scan[w];
      total += sel.scan[w];
    }
    int at = n + before + pos - __popc(hit);
    while (hit) {
      const int j = __ffs(hit) - 1;
      hit &= hit - 1;
      if (at < k) sel.cand[at] = pack_key(kth, kE * i + j - row.shift);
      ++at;
    }
    n = min(k, n + total);
  }
  __syncthreads();
}

// One block, the whole row, at least k of whose keys reach `bound`: sel.cand[0 .. k) holds the winners afterwards.
// Mostly the least of those keys is the k-th largest itself, in a crowd of equals (a row of equal logits, or one whose
// mask leaves fewer than k): two passes then; else bisection over the key's bits.
template <typename T>
__device__ void select_exactly(const Row<const T>& row, int k, uint32_t bound, Select& sel) {
  constexpr int kE = Unit<T>::kE;
  uint32_t kth = least_ge(row, bound, sel.scan);
  if (count_ge(row, kth + 1, sel.scan) >= k) {
    kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = kth | (1u << bit);
      if (count_ge(row, trial, sel.scan) >= k) kth = trial;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sel.count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
    const Unit<T> u = row.load(i);
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const uint32_t key = order_key(to_f(u.get(j)));
      if (key > kth && row.holds(kE * i + j)) sel.cand[atomicAdd(&sel.count, 1)] = pack_key(key, kE * i + j - row.shift);
    }
  }
  __syncthreads();
  fill_equals(row, kth, sel.count, k, sel);
}

// ------------------------------------------------------------------------------------- token log-probs
template <typename A>
__device__ __forceinline__ double inv_temp(const A& a, int row) {
  return a.temp ? rcp_d((double)a.temp[row]) : a.inv_temp1;
}
template <typename A>
__device__ __forceinline__ float row_c(const A& a, int row) {
  return (float)(kLog2e * inv_temp(a, row));
}

__device__ __forceinline__ float finish_logp(double x, float c, Stat st, double log2s) {
  const double xc = x * (double)c;
  if (st.s == 0.f || xc <= (double)kMasked) return st.s == st.s ? -INFINITY : st.s;
  return (float)(kLn2 * (xc - (double)st.R - log2s));
}

struct RowPart {       // what the blocks of a cluster tell one another about a row
  Stat st;
  uint32_t bound;
};

// The outputs of a row but its alternatives; by the leading block.
template <typename T, bool kEntropy>
__device__ __forceinline__ void write_row(const TokenArgs& a, int r, const T* x, float c, Stat st, double log2s) {
  for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
    const long t = a.tokens[(size_t)r * a.n + j] - a.vocab_start;
    const bool here = t >= 0 && t < a.V;
    float v = 0.f;
    if (here) v = a.open ? to_f(x[t]) * c : finish_logp(to_f(x[t]), c, st, log2s);
    a.logp[(size_t)r * a.n + j] = v;
  }
  if (threadIdx.x == 0) {
    const bool empty = st.s == 0.f;
    const double inv = rcp_d(empty ? 1.0 : (double)st.s);
    if (kEntropy) a.entropy[r] = empty ? 0.f : (float)(kLn2 * (log2s - (double)st.et * inv));
    if (!a.stats) return;
    float* o = a.stats + 3 * (size_t)r;
    o[0] = st.R;
    o[1] = a.open ? st.s : (empty ? 0.f : (float)inv);
    o[2] = a.open ? st.et : (empty ? 0.f : (float)((double)st.et * inv));
  }
}

// The alternatives from the gathered candidates; by the leading block.
template <typename T>
__device__ __forceinline__ void write_top(const TokenArgs& a, int r, const Row<const T>& row, float c, Stat st,
                                          double log2s, uint32_t bound, Select& sel) {
  int n = sel.count;
  if (n > kCand) {
    select_exactly(row, a.k, bound, sel);
    n = a.k;
  } else if (n < a.k) {      // the others of the row are -inf
    fill_equals(row, kLowestKey, n, a.k, sel);
    n = a.k;
  }
  // ranks by counting, `share` neighbouring lanes to a candidate
  int share = 1;
  while (share < 32 && 2 * share * n <= (int)blockDim.x) share *= 2;
  const int part = threadIdx.x & (share - 1), per_pass = blockDim.x / share;
  for (int i0 = 0; i0 < n; i0 += per_pass) {
    const int i = i0 + threadIdx.x / share;
    const unsigned long long own = sel.cand[min(i, n - 1)];
    int place = 0;
#pragma unroll 4
    for (int j = part; j < n; j += share) place += sel.cand[j] > own;
    for (int o = share / 2; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    if (i < n && part == 0 && place < a.k) {
      const int t = (int)(0xffffffffu - (uint32_t)own);
      const float v = key_value((uint32_t)(own >> 32));
      a.top_ids[(size_t)r * a.k + place] = t + a.vocab_start;
      a.top_logp[(size_t)r * a.k + place] = a.open ? v : finish_logp(v, c, st, log2s);
    }
  }
}

// Joins the cluster's sums and bounds; afterwards the leader's `sel` takes candidates.
__device__ __forceinline__ void join_row(RowPart& mine, Stat& st, uint32_t& bound, Select* sel,
                                         cg::cluster_group& cl) {
  const int blocks = (int)cl.num_blocks();
  if (threadIdx.x == 0) {
    mine.st = st;
    mine.bound = bound;
    if (sel) sel->count = 0;
  }
  if (blocks == 1) {
    if (sel) __syncthreads();
    return;
  }
  cl.sync();
  const int lane = threadIdx.x & 31;
  Stat other = Stat::none();
  uint32_t least = 0xffffffffu;
  if (lane < blocks) {
    const RowPart* m = cl.map_shared_rank(&mine, lane);
    other = m->st;
    least = m->bound;
  }
  st = warp_join(other);
  bound = __reduce_min_sync(0xffffffffu, least);
}

// Alternatives of short rows, and of few rows: the cluster holds the row in registers, kUnits units per thread, so the
// selection does not read it again.
template <typename T, bool kEntropy, int kUnits>
__global__ void __launch_bounds__(kThreads, kUnits == 10 ? 1 : 3) token_top_kernel(const T* __restrict__ logits, TokenArgs a) {
  __shared__ Stat part[32];
  __shared__ RowPart mine;
  extern __shared__ __align__(16) unsigned char dyn[];
  Select* sel = reinterpret_cast<Select*>(dyn);
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const Slice sl(row.units, blocks, rank);
  Unit<T> u[kUnits];
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const int i = sl.lo + threadIdx.x + n * blockDim.x;
    if (i < sl.hi) u[n] = row.load(i);
    else u[n].fill(from_f<T>(-INFINITY));
  }
  const float c = row_c(a, r);
  const float best = units_max<T, kUnits>(u);
  Sums sums;
  sums.R = reference(best * c);
  add_units<kEntropy, T, kUnits>(sums, u, c);
  Stat st = block_join(sums.get(), part);
  const bool any = sl.lo + (int)threadIdx.x < sl.hi;
  const uint32_t best_key = order_key(best);
  uint32_t bound = kth_max(best_key, any, (a.k + blocks - 1) / blocks);
  join_row(mine, st, bound, sel, cl);
  if (any && best_key >= bound) {
    Select* lead = cl.map_shared_rank(sel, 0);
    const float floor = bound_value(bound);
#pragma unroll
    for (int n = 0; n < kUnits; ++n) {
      const int i = sl.lo + threadIdx.x + n * blockDim.x;
      if (i < sl.hi && u[n].max() >= floor && *const_cast<volatile int*>(&lead->count) <= kCand)
        offer(u[n], i, floor, row, lead);
    }
  }
  if (blocks > 1) cl.sync();      // the leader has every candidate, and nobody's sums are read any more
  else __syncthreads();
  if (rank) return;
  const double log2s = log2_d((double)st.s);
  write_row<T, kEntropy>(a, r, x, c, st, log2s);
  write_top(a, r, row, c, st, log2s, bound, *sel);
}

// 16 bytes that are read once.  (Volatile: the compiler keeps the loads of a batch together, ahead of the arithmetic.)
__device__ __forceinline__ uint4 read_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Scores without alternatives: a row is read once and nothing of it is needed again, so its batches come straight into
// registers, the next while one is worked on.  Against the same pass over copies in shared memory: 203 us, not 209, for
// 4096 x 151936 BF16; 215, not 227, where the power cap holds the clock down.  (Two batches take 73-80 registers.)
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kStream, 3) token_stream_kernel(const T* __restrict__ logits, TokenArgs a) {
  __shared__ Stat part[32];
  __shared__ RowPart mine;
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank(), lane = threadIdx.x & 31;
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const Slice sl(row.units, blocks, rank);
  const int step = (int)(blockDim.x >> 5) * kSpan;
  // [lo, hi): the units that are whole and in the slice
  const int lo = max(sl.lo, row.shift ? 1 : 0), hi = min(sl.hi, row.end / Unit<T>::kE);
  const float c = row_c(a, r);
  Sums sums;
  const auto fetch = [&](int first, Unit<T>* u) {      // beyond the slice: nothing but masked logits
    if (first >= lo && first + kSpan <= hi) {
      const uint4* p = reinterpret_cast<const uint4*>(row.p) + first + lane;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) u[b].w = read_once(p + 32 * b);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = first + lane + 32 * b;
        if (i < sl.hi) u[b] = row.load(i);
        else u[b].fill(from_f<T>(-INFINITY));
      }
    }
  };
  const auto use = [&](const Unit<T>* u) {
    const float top = units_max<T, kBatch>(u) * c;
    if (top > sums.R + kSlack) sums.raise(reference(top));
    add_units<kEntropy, T, kBatch>(sums, u, c);
  };
  Unit<T> u[kBatch], v[kBatch];
  int i = sl.lo + (int)(threadIdx.x >> 5) * kSpan;
  fetch(i, u);
  for (; i < sl.hi; i += 2 * step) {
    fetch(i + step, v);
    use(u);
    fetch(i + 2 * step, u);
    use(v);
  }
  Stat st = block_join(sums.get(), part);
  uint32_t bound = 0;
  join_row(mine, st, bound, nullptr, cl);
  if (blocks > 1) cl.sync();      // nobody's sums are read any more
  if (rank) return;
  write_row<T, kEntropy>(a, r, x, c, st, log2_d((double)st.s));
}

// Alternatives of long rows, which stream through shared memory once.  A warp notes the maximum of every 32 units it
// takes; after the bound is known only those that reach it are read again.
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kStream, 4) token_top_stream_kernel(const T* __restrict__ logits, TokenArgs a) {
  __shared__ Stat part[32];
  __shared__ RowPart mine;
  __shared__ int hit_units;
  extern __shared__ __align__(16) unsigned char dyn[];
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank(), lane = threadIdx.x & 31;
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const Slice sl(row.units, blocks, rank);
  Feed<T, 1> feed(dyn, row, sl);
  // (the selection takes the ring's place once its copies are done)
  float* strips = reinterpret_cast<float*>(dyn + max(Feed<T, 1>::bytes(blockDim.x), sizeof(Select) + 4 * kCand));
  int* list = reinterpret_cast<int*>(dyn + sizeof(Select));
  if (threadIdx.x == 0) hit_units = 0;
  const float c = row_c(a, r);
  Sums sums;
  float best = -INFINITY;
  const uint4* from = feed.p + kGroups * feed.step;
  float* strip = strips + (feed.first - sl.lo) / 32 + lane;
  for (int k = 0; k < feed.batches; ++k, from += feed.step, strip += feed.step / 32) {
    feed.wait(k, row, sl);
    Unit<T> u[kBatch];
    feed.take(u);
    float m[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) m[b] = u[b].max();
    float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    best = fmaxf(best, top);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) m[b] = warp_top(m[b]);
    if (lane < kBatch) *strip = lane == 0 ? m[0] : (lane == 1 ? m[1] : (lane == 2 ? m[2] : m[3]));
    if (feed.inner(k + kGroups)) feed.issue_inner(from);
    else feed.issue(k + kGroups);
    top *= c;
    if (top > sums.R + kSlack) sums.raise(reference(top));
    add_units<kEntropy, T, kBatch>(sums, u, c);
  }
  Stat st = block_join(sums.get(), part);
  Select* sel = reinterpret_cast<Select*>(dyn);      // the ring's place: its copies are done
  const int held = sl.hi - sl.lo;
  uint32_t bound =
      kth_max(order_key(best), (int)(threadIdx.x >> 5) * kSpan + lane < held, (a.k + blocks - 1) / blocks);
  join_row(mine, st, bound, sel, cl);
  Select* lead = cl.map_shared_rank(sel, 0);
  const int count = (held + 31) / 32;
  const float floor = bound_value(bound);
  // Units that reach the bound: first found, a warp to a strip, then taken apart, a thread to a unit.  (With the
  // taking apart inside the strips' loop 32 lanes wait for one: 85 us, not 79, for 1024 x 151936 BF16 and k = 64.)
  for (int s0 = 32 * (threadIdx.x >> 5); s0 < count; s0 += blockDim.x) {
    unsigned hits = __ballot_sync(0xffffffffu, s0 + lane < count && strips[min(s0 + lane, count - 1)] >= floor);
    while (hits && *const_cast<volatile int*>(&hit_units) <= kCand) {      // (beyond, the count alone decides)
      constexpr int kAtOnce = 4;
      Unit<T> u[kAtOnce];
      int at[kAtOnce];
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        at[n] = hits ? sl.lo + 32 * (s0 + __ffs(hits) - 1) + lane : sl.hi;
        hits &= hits - 1;
        if (at[n] < sl.hi) u[n] = row.load(at[n]);
      }
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        if (at[n] >= sl.hi || !(u[n].max() >= floor)) continue;
        const int to = atomicAdd(&hit_units, 1);
        if (to < kCand) list[to] = at[n];
      }
    }
  }
  __syncthreads();
  if (hit_units > kCand) {
    if (threadIdx.x == 0) atomicAdd(&lead->count, kCand + 1);      // far too many: the exact way
  } else {
    for (int h = threadIdx.x; h < hit_units; h += blockDim.x) offer(row.load(list[h]), list[h], floor, row, lead);
  }
  if (blocks > 1) cl.sync();      // the leader has every candidate, and nobody's sums are read any more
  else __syncthreads();
  if (rank) return;
  const double log2s = log2_d((double)st.s);
  write_row<T, kEntropy>(a, r, x, c, st, log2s);
  write_top(a, r, row, c, st, log2s, bound, *sel);
}

// u = 2^t (A + B t), t = u c - R
template <bool kEntropy, bool kMask, typename T>
__device__ __forceinline__ void score_gradient(Unit<T>& u, float c, float R, float A, float B) {
#pragma unroll
  for (int j = 0; j < Unit<T>::kE / 2; ++j) {
    float2 t = __ffma2_rn(u.pair(j), both(c), both(-R));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    if (kMask) t = make_float2(fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f));
    u.set_pair(j, __fmul2_rn(e, kEntropy ? __ffma2_rn(both(B), t, both(A)) : both(A)));
  }
}

// d x_v = (e / s / T) (-G - dH ln 2 (t - E[t])) + [v = t_j] g_j / T, G = sum_j g_j
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kStream, 4)
    token_logprob_bwd_kernel(const T* __restrict__ logits, T* __restrict__ grad, TokenArgs a) {
  __shared__ float scratch[32];
  extern __shared__ __align__(16) unsigned char dyn[];
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks(), lane = threadIdx.x & 31;
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  T* g = grad + (size_t)r * a.V;
  const Row<const T> row(x, a.V);
  const Row<T> out(g, a.V);
  const Slice sl(row.units, blocks, (int)cl.block_rank());
  Feed<T, 1> feed(dyn, row, sl);
  const bool vec = row.shift == out.shift;
  const float c = row_c(a, r);
  const float it = (float)inv_temp(a, r);
  const float* st = a.stats + 3 * (size_t)r;
  const float R = st[0], inv = st[1], mean = st[2];
  float G = 0.f;      // a token outside the whole vocabulary (an ignored position) has no gradient
  for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
    const long t = a.tokens[(size_t)r * a.n + j];
    G += (t >= 0 && t < a.vocab_total) ? a.d_logp[(size_t)r * a.n + j] : 0.f;
  }
  G = bb::block_sum(G, scratch);
  const float dh = kEntropy ? a.d_entropy[r] * (float)kLn2 : 0.f;
  const float A = it * inv * (dh * mean - G), B = -it * inv * dh;
  const unsigned long long policy = evict_first();
  const uint4* from = feed.p + kGroups * feed.step;
  uint4* to = reinterpret_cast<uint4*>(out.p) + feed.first + lane;
  for (int k = 0; k < feed.batches; ++k, from += feed.step, to += feed.step) {
    feed.wait(k, row, sl);
    Unit<T> u[kBatch];
    feed.take(u);
    if (kEntropy && masked<T, kBatch>(u, c)) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) score_gradient<kEntropy, true>(u[b], c, R, A, B);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) score_gradient<kEntropy, false>(u[b], c, R, A, B);
    }
    if (feed.inner(k + kGroups)) feed.issue_inner(from);
    else feed.issue(k + kGroups);
    if (vec && feed.inner(k)) {
      store_streaming<0>(to, u[0].w, policy);
      store_streaming<1>(to, u[1].w, policy);
      store_streaming<2>(to, u[2].w, policy);
      store_streaming<3>(to, u[3].w, policy);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = feed.first + k * feed.step + lane + 32 * b;
        if (i < sl.hi) out.store(i, u[b], vec, row.shift);
      }
    }
  }
  __syncthreads();
  // the given tokens' columns, once per distinct token, by the block that wrote them
  for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
    const int64_t* tk = a.tokens + (size_t)r * a.n;
    const long t = tk[j] - a.vocab_start;
    if (t < 0 || t >= a.V) continue;
    const int unit = ((int)t + row.shift) / Unit<T>::kE;
    if (unit < sl.lo || unit >= sl.hi) continue;
    bool first = true;
    for (int i = 0; i < j; ++i) first &= tk[i] != tk[j];
    if (!first) continue;
    float add = 0.f;
    for (int i = j; i < a.n; ++i) add += tk[i] == tk[j] ? a.d_logp[(size_t)r * a.n + i] : 0.f;
    const float xt = to_f(x[t]), d = fmaf(xt, c, -R), e = ex2(d);
    const float body = e * (kEntropy ? fmaf(B, fmaxf(d, -1e4f), A) : A);
    g[t] = from_f<T>(inv == 0.f ? 0.f : fmaf(add, it, body));
  }
}

// ------------------------------------------------------------------------------------------ distillation
// Teacher side of a row, q~ = exp(log q - ref) over the entries that count, and the student's at their columns:
// e = 2^(x c - m).  A block holds the part of its slice; the parts are summed over the cluster.
struct Teacher {
  double q, qlq, qxc;   // sums of q~, q~ (log q - ref), q~ x c
  double m, z;          // max of x c, sum over distinct columns of 2^(x c - m)
};

// Everything that the gradient of a row needs.
struct Finished {
  float R, factor;      // columns outside the entries: factor 2^(x c - R)
  double per_q;         // an entry's column: per_p 2^(x c - m) - per_q q~
  double per_p, m;
  float kl;
};

__device__ __forceinline__ Teacher no_teacher() { return {0.0, 0.0, 0.0, -INFINITY, 0.0}; }

// Sum over the first kMaxCluster lanes (the others hold nothing), in those lanes.
__device__ __forceinline__ Teacher join_blocks(Teacher t) {
  double m = t.m;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
  t.z = t.z == 0.0 ? 0.0 : t.z * exp2_d(t.m - m);
  t.m = m;
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
    t.q += __shfl_xor_sync(0xffffffffu, t.q, o);
    t.qlq += __shfl_xor_sync(0xffffffffu, t.qlq, o);
    t.qxc += __shfl_xor_sync(0xffffffffu, t.qxc, o);
    t.z += __shfl_xor_sync(0xffffffffu, t.z, o);
  }
  return t;
}

// What FP32 log-probs can leave of 1 by rounding (theirs are right to 2e-6, and q to as much of itself).  Where the
// student has nothing outside the entries, as when both are under a mask that leaves fewer tokens than there are
// entries, a remainder of this size is no probability without a home: it would make the divergence infinite.
constexpr double kResidue = 3.814697265625e-6;      // 2^-18

// `some`: the row has entries that count.  `scale` includes the row's weight and 1 / T.
__device__ __forceinline__ Finished finish_row(const Teacher& t, Stat rest, bool some, bool tail, double scale) {
  // (written with selects: the long FP64 chains are independent and overlap)
  const bool out = rest.s != 0.f, in = t.z != 0.0;      // student probability outside and on the entries
  const double Rd = out ? (double)rest.R : -INFINITY, md = in ? t.m : -INFINITY;
  const double m = fmax(Rd, md);
  const bool lost = m <= (double)kFloor;                // none anywhere
  const double m0 = lost ? 0.0 : m;
  const double s = out ? (double)rest.s : 1.0;
  const double left = tail ? fmax(0.0, 1.0 - t.q) : 0.0, q_rest = out || left > kResidue ? left : 0.0, total = tail ? t.q + q_rest : 1.0;
  const double q_norm = tail ? 1.0 : t.q;
  const double log_s = log2_d(s), log_qr = log2_d(q_rest), log_norm = log2_d(q_norm);
  const double inv_s = rcp_d(s), norm = rcp_d(q_norm);
  const double share = out ? s * exp2_d(Rd - m0) : 0.0;
  const double z = lost ? 1.0 : (in ? t.z * exp2_d(md - m0) : 0.0) + share;
  const double lse = m0 + log2_d(z), inv_z = rcp_d(z), p_rest = share * inv_z;
  double kl = norm * t.qlq - kLn2 * (log_norm + norm * t.qxc - norm * t.q * lse);
  if (q_rest > 0.0) kl += out ? q_rest * kLn2 * (log_qr - (Rd + log_s - lse)) : INFINITY;
  // a teacher without probability on any entry: with a tail class all of it is there, else there is nothing to learn
  const bool nothing = !some || (!tail && t.q == 0.0);
  const bool still = nothing || lost;
  Finished f;
  f.kl = nothing ? 0.f : (lost ? INFINITY : (float)kl);
  f.R = out ? rest.R : 0.f;
  f.factor = still || !out ? 0.f : (float)(scale * (total * p_rest - q_rest) * inv_s);
  f.per_q = still ? 0.0 : scale * norm;
  f.per_p = still ? 0.0 : scale * total * inv_z;
  f.m = m0;
  return f;
}

// The teacher's entries of a row.  Those in this block's slice are chained by where they lie (a thread's units, or a
// warp's batch), so that whoever takes the logits there rules the entries' columns out.
struct Entries {
  double *xc, *q;        // of the entries in this block's slice
  Teacher* part;         // sums of 32 entries each
  float* logq;           // of every entry; -inf where dropped
  int* col;              // the shard's column if it lies in this block's slice, else -1
  int* next;             // chain, -1 at its end
  int* spot;             // where in its chain's units
  int* heads;            // chains
  unsigned char* later;  // repeats the column of an earlier entry

  static __host__ __device__ size_t bytes(int K, int chains) {
    return (K + 31) / 32 * sizeof(Teacher) + (size_t)K * 32 + (size_t)chains * 4 + K + 15;
  }
  __device__ __forceinline__ Entries(unsigned char* p, int K, int chains) {
    part = reinterpret_cast<Teacher*>(p);
    xc = reinterpret_cast<double*>(part + (K + 31) / 32);
    q = xc + K;
    logq = reinterpret_cast<float*>(q + K);
    col = reinterpret_cast<int*>(logq + K);
    next = col + K;
    spot = next + K;
    heads = spot + K;
    later = reinterpret_cast<unsigned char*>(heads + chains);
  }
};

// Reads the row's entries into `en`, chains them from en.heads[place(unit)] and sums them 32 by 32; returns whether the
// row has any that counts.  The chains are complete when it returns, the sums after the next barrier.
template <typename T, typename Place, typename Spot>
__device__ __forceinline__ bool load_entries(const Entries& en, const DistillArgs& a, int r, const T* x,
                                             const Row<const T>& row, Slice sl, float c, int chains, Place place,
                                             Spot spot) {
  const int lane = threadIdx.x & 31, padded = (a.K + 31) / 32 * 32;
  for (int i = threadIdx.x; i < chains; i += blockDim.x) en.heads[i] = -1;
  __syncthreads();
  bool some = false;
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
    const size_t at = (size_t)r * a.K + j;
    const long id = a.ids[at], t = id - a.vocab_start;
    const float lq = a.logq[at];
    const bool valid = id >= 0 && id < a.vocab_total;
    const int unit = valid && t >= 0 && t < a.V ? ((int)t + row.shift) / Unit<T>::kE : -1;
    some |= valid;
    en.logq[j] = valid ? lq : -INFINITY;
    en.col[j] = -1;
    en.later[j] = 0;
    if (unit >= sl.lo && unit < sl.hi) {
      const double xc = (double)to_f(x[t]) * (double)c;
      en.xc[j] = xc <= (double)kMasked ? -INFINITY : xc;
      en.col[j] = (int)t;
      en.spot[j] = spot(unit, ((int)t + row.shift) % Unit<T>::kE);
      en.next[j] = atomicExch(&en.heads[place(unit)], j);
    }
  }
  some = __syncthreads_or(some);
  double ref = 0.0;
  if (!a.tail) {            // relative to the largest log q: without a tail class these may be raw logits
    float top = -INFINITY;
    for (int j = lane; j < a.K; j += 32) top = fmaxf(top, en.logq[j]);
    top = warp_top(top);
    if (top > -INFINITY) ref = (double)top;
  }
  for (int j = threadIdx.x; j < padded; j += blockDim.x) {
    Teacher p = no_teacher();
    if (j < a.K && en.col[j] >= 0) {
      const double l = (double)en.logq[j] - ref, q = exp2_d(l * kLog2e), xc = en.xc[j];
      en.q[j] = q;
      p.q = q;
      p.qlq = q == 0.0 ? 0.0 : q * l;
      p.qxc = q == 0.0 ? 0.0 : q * xc;
      for (int e = en.heads[place((en.col[j] + row.shift) / Unit<T>::kE)]; e >= 0; e = en.next[e])
        if (e < j && en.col[e] == en.col[j]) en.later[j] = 1;
      if (!en.later[j] && xc > -INFINITY) {
        p.m = xc;
        p.z = 1.0;
      }
    }
    const double m = warp_max_d(p.m);
    p.z = p.z == 0.0 ? 0.0 : exp2_d(p.m - m);
    p.m = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      p.q += __shfl_xor_sync(0xffffffffu, p.q, o);
      p.qlq += __shfl_xor_sync(0xffffffffu, p.qlq, o);
      p.qxc += __shfl_xor_sync(0xffffffffu, p.qxc, o);
      p.z += __shfl_xor_sync(0xffffffffu, p.z, o);
    }
    if (lane == 0) en.part[j >> 5] = p;
  }
  return some;
}

struct Shared {
  Stat warps[32];
  struct { Stat st; Teacher teacher; } mine;
  Finished fin;
};

// Joins the block's and the cluster's sums and finishes the row: sh.fin, and the outputs that are per row.
template <typename T>
__device__ __forceinline__ void finish_block(Shared& sh, const Entries& en, Stat own, const DistillArgs& a, int r, float w, bool some,
                                             cg::cluster_group& cl) {
  const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank(), lane = threadIdx.x & 31;
  Stat st = block_join(own, sh.warps);
  Teacher t = no_teacher();
  if (threadIdx.x < 32) {
    if (lane < (a.K + 31) / 32) t = en.part[lane];
    t = join_blocks(t);
  }
  if (blocks > 1) {
    if (threadIdx.x == 0) {
      sh.mine.st = st;
      sh.mine.teacher = t;
    }
    cl.sync();
    if (threadIdx.x < 32) {
      Stat other = Stat::none();
      t = no_teacher();
      if (lane < blocks) {
        const auto* m = cl.map_shared_rank(&sh.mine, lane);
        other = m->st;
        t = m->teacher;
      }
      st = warp_join<kMaxCluster>(other);
      t = join_blocks(t);
    }
  }
  if (threadIdx.x == 0) {
    const double scale = a.num ? a.scale * ((double)a.num[0] / (double)a.den) : a.scale;
    sh.fin = finish_row(t, st, some, a.tail, (double)w * scale * inv_temp(a, r));
    if (rank == 0 && a.open) {
      a.stats[2 * (size_t)r] = st.R;
      a.stats[2 * (size_t)r + 1] = st.s;
    } else if (rank == 0 && a.rows) {
      a.rows[r] = w != 0.f ? sh.fin.kl : 0.f;
    }
  }
  __syncthreads();
  if (blocks > 1) cl.barrier_arrive();     // this block's reads of the others' sums are done
  if (a.open)
    for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
      const long t = a.ids[(size_t)r * a.K + j] - a.vocab_start;
      if (en.col[j] >= 0) a.xc[(size_t)r * a.K + j] = (float)en.xc[j];
      else if (rank == 0 && (t < 0 || t >= a.V)) a.xc[(size_t)r * a.K + j] = 0.f;
    }
}

// The entries' own columns, over what the second pass wrote there.
template <typename T, typename Place>
__device__ __forceinline__ void write_entries(const Shared& sh, const Entries& en, const DistillArgs& a, T* g,
                                              const Row<const T>& row, Place place) {
  __syncthreads();
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
    const int col = en.col[j];
    if (col < 0 || en.later[j]) continue;
    bool again = false;
    for (int e = en.heads[place((col + row.shift) / Unit<T>::kE)]; e >= 0; e = en.next[e])
      again |= e != j && en.col[e] == col;
    double q = en.q[j];
    if (again)        // in the order of the entries, whatever the chain's
      for (int i = j + 1; i < a.K; ++i)
        if (en.col[i] == col) q += en.q[i];
    const double p = sh.fin.per_p * exp2_d(en.xc[j] - sh.fin.m);
    g[col] = from_f<T>((float)(p - sh.fin.per_q * q));
  }
}

template <typename T>
__device__ __forceinline__ void gradient_unit(Unit<T>& u, float c, float R, float factor) {
#pragma unroll
  for (int j = 0; j < Unit<T>::kE / 2; ++j) {
    const float2 t = __ffma2_rn(u.pair(j), both(c), both(-R));
    u.set_pair(j, __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)), both(factor)));
  }
}

// Whether the gradient that is there needs no other factor (for every block of a launch alike).
__device__ __forceinline__ bool as_announced(const DistillArgs& a) { return a.num && a.num[0] == a.den; }

// A cluster per row, the row in registers, kUnits units per thread: the statistics of the columns outside the teacher's
// entries, the joining, the gradient.  Short rows, and few rows, where one pass's latency is what counts: of 8.8 us for 4
// FP32 rows of 24000 most goes to the launch, the entries (ids, then the logits there) and two joins, not to 0.8 MB.
template <typename T, int kUnits>
__global__ void __launch_bounds__(kThreads, 2) distill_kernel(const T* logits, T* grad, DistillArgs a) {
  if (as_announced(a)) return;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char dyn[];
  const Entries en(dyn, a.K, blockDim.x);
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks();
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const Slice sl(row.units, blocks, (int)cl.block_rank());
  const float w = a.weights ? a.weights[r] : 1.f;
  const bool live = w != 0.f;      // rows of weight 0 are not read
  Unit<T> u[kUnits];
#pragma unroll
  for (int n = 0; n < kUnits; ++n) {
    const int i = sl.lo + threadIdx.x + n * blockDim.x;
    if (live && i < sl.hi) u[n] = row.load(i);
    else u[n].fill(from_f<T>(-INFINITY));
  }
  const float c = row_c(a, r);
  const auto place = [&](int unit) { return (unit - sl.lo) % (int)blockDim.x; };
  const auto spot = [&](int unit, int j) { return (unit - sl.lo) / (int)blockDim.x * Unit<T>::kE + j; };
  const bool some = load_entries(en, a, r, x, row, sl, c, blockDim.x, place, spot);
  for (int e = en.heads[threadIdx.x]; e >= 0; e = en.next[e]) {
    const int at = en.spot[e];
#pragma unroll
    for (int n = 0; n < kUnits; ++n)
      if (at / Unit<T>::kE == n) u[n].mask(1u << at % Unit<T>::kE);
  }
  Sums sums;
  sums.R = reference(units_max<T, kUnits>(u) * c);
  add_units<false, T, kUnits>(sums, u, c);
  finish_block<T>(sh, en, sums.get(), a, r, w, some, cl);
  if (grad) {
    T* g = grad + (size_t)r * a.V;
    const Row<T> out(g, a.V);
    const bool vec = row.shift == out.shift;
    const float R = sh.fin.R, factor = live ? sh.fin.factor : 0.f;
#pragma unroll
    for (int n = 0; n < kUnits; ++n) {
      const int i = sl.lo + threadIdx.x + n * blockDim.x;
      if (i >= sl.hi) break;
      if (factor != 0.f) gradient_unit(u[n], c, R, factor);
      else u[n].fill(from_f<T>(0.f));
      out.store(i, u[n], vec, row.shift);
    }
    if (live) write_entries(sh, en, a, g, row, place);
  }
  if (blocks > 1) cl.barrier_wait();
}

// The same for many long rows: the row streams through shared memory, once for the statistics and, for the gradient,
// once more (from L2, mostly).  The copies of the first batches are on their way while the entries are prepared.
template <typename T, bool kGrad>
__global__ void __launch_bounds__(kStream, 4) distill_stream_kernel(const T* logits, T* grad, DistillArgs a) {
  if (as_announced(a)) return;
  __shared__ Shared sh;
  extern __shared__ __align__(16) unsigned char dyn[];
  cg::cluster_group cl = cg::this_cluster();
  const int blocks = (int)cl.num_blocks(), lane = threadIdx.x & 31;
  const int r = blockIdx.x / blocks;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const Slice sl(row.units, blocks, (int)cl.block_rank());
  const float w = a.weights ? a.weights[r] : 1.f;
  const bool live = w != 0.f;
  using Rows = Feed<T, kGrad ? 2 : 1>;
  Rows feed(dyn, row, sl, live);
  const int chains = (sl.hi - sl.lo + kSpan - 1) / kSpan;
  const Entries en(dyn + Rows::bytes(blockDim.x), a.K, chains);
  const float c = row_c(a, r);
  const auto place = [&](int unit) { return (unit - sl.lo) / kSpan; };
  // the lane, and the offset from its first slot of the batch
  const auto spot = [&](int unit, int j) {
    const int n = (unit - sl.lo) % kSpan;
    return n % 32 << 16 | (n / 32 * 512 + j * (int)sizeof(T));
  };
  const bool some = load_entries(en, a, r, x, row, sl, c, chains, place, spot);
  Sums sums;
  if (live) {
    const int* head = en.heads + (feed.first - sl.lo) / kSpan;
    const unsigned long long policy = evict_normal();
    const uint4* from = feed.p + kGroups * feed.step;
    for (int k = 0; k < feed.batches; ++k, from += feed.step) {
      feed.wait(k, row, sl);
      for (int e = *head; e >= 0; e = en.next[e]) {
        const int at = en.spot[e];
        if (at >> 16 == lane) feed.rule_out(at & 0xffff);
      }
      head += blockDim.x >> 5;
      Unit<T> u[kBatch];
      feed.take(u);
      const float top = units_max<T, kBatch>(u) * c;
      if (feed.inner(k + kGroups)) feed.issue_inner(from, policy);
      else feed.issue(k + kGroups);
      if (top > sums.R + kSlack) sums.raise(reference(top));
      add_units<false, T, kBatch>(sums, u, c);
    }
  }
  finish_block<T>(sh, en, sums.get(), a, r, w, some, cl);
  if constexpr (kGrad) {
    T* g = grad + (size_t)r * a.V;
    const Row<T> out(g, a.V);
    const bool vec = row.shift == out.shift;
    const float R = sh.fin.R, factor = live ? sh.fin.factor : 0.f;
    if (factor != 0.f) {
      const unsigned long long policy = evict_first();
      uint4* to = reinterpret_cast<uint4*>(out.p) + feed.first + (feed.batches - 1) * feed.step + lane;
      const uint4* from = feed.p + (feed.batches - 1 - kGroups) * feed.step;
      for (int k = feed.batches - 1; k >= 0; --k, to -= feed.step, from -= feed.step) {
        Unit<T> u[kBatch];
        feed.take_back(k, row, sl, u);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) gradient_unit(u[b], c, R, factor);
        if (feed.inner(k - kGroups)) feed.issue_inner(from, policy);
        else feed.issue(k - kGroups);
        if (vec && feed.inner(k)) {
          store_streaming<0>(to, u[0].w, policy);
          store_streaming<1>(to, u[1].w, policy);
          store_streaming<2>(to, u[2].w, policy);
          store_streaming<3>(to, u[3].w, policy);
        } else {
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int i = feed.first + k * feed.step + lane + 32 * b;
            if (i < sl.hi) out.store(i, u[b], vec, row.shift);
          }
        }
      }
    } else {      // no gradient outside the entries
      Unit<T> u;
      u.fill(from_f<T>(0.f));
      for (int i = sl.lo + threadIdx.x; i < sl.hi; i += blockDim.x) out.store(i, u, vec, row.shift);
    }
    if (live) write_entries(sh, en, a, g, row, place);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (blocks > 1) cl.barrier_wait();
}

// Vocabulary in shards: one warp per row finishes it from the joined (R, s) and x c of every entry.
__global__ void distill_finish_kernel(DistillArgs a) {
  const int r = blockIdx.x, lane = threadIdx.x;
  const int64_t* ids = a.ids + (size_t)r * a.K;
  const float *logq = a.logq + (size_t)r * a.K, *xcs = a.xc + (size_t)r * a.K;
  const auto valid = [&](int j) { return ids[j] >= 0 && ids[j] < a.vocab_total; };
  const auto entry = [&](int j) { return xcs[j] <= kMasked ? -INFINITY : (double)xcs[j]; };
  float ref = 0.f;
  bool some = false;
  if (!a.tail) {
    float top = -INFINITY;
    for (int j = lane; j < a.K; j += 32)
      if (valid(j)) top = fmaxf(top, logq[j]);
    top = warp_top(top);
    if (top > -INFINITY) ref = top;
  }
  Teacher p = no_teacher();
  for (int j = lane; j < a.K; j += 32) {
    if (!valid(j)) continue;
    some = true;
    const double q = exp2_d(((double)logq[j] - (double)ref) * kLog2e);
    p.q += q;
    if (q != 0.0) {
      p.qlq += q * ((double)logq[j] - (double)ref);
      p.qxc += q * entry(j);
    }
    p.m = fmax(p.m, entry(j));
  }
  some = __any_sync(0xffffffffu, some);
  p.q = warp_sum_d(p.q);
  p.qlq = warp_sum_d(p.qlq);
  p.qxc = warp_sum_d(p.qxc);
  p.m = warp_max_d(p.m);
  if (p.m > -INFINITY)
    for (int j = lane; j < a.K; j += 32) {
      bool first = valid(j);
      for (int i = 0; first && i < j; ++i) first = ids[i] != ids[j];
      if (first) p.z += exp2_d(entry(j) - p.m);
    }
  p.z = warp_sum_d(p.z);
  Stat st = Stat::none();
  st.R = a.stats[2 * (size_t)r];
  st.s = a.stats[2 * (size_t)r + 1];
  const float w = a.weights ? a.weights[r] : 1.f;
  const double it = inv_temp(a, r);
  const Finished f = finish_row(p, st, some, a.tail, (double)w * a.scale * it);
  if (lane == 0) {
    a.rows[r] = w == 0.f ? 0.f : f.kl;
    a.coef[2 * (size_t)r] = f.R;
    a.coef[2 * (size_t)r + 1] = w == 0.f ? 0.f : f.factor;
  }
  for (int j = lane; j < a.K; j += 32) {
    double q = 0.0;        // every entry of a repeated id carries the id's gradient
    for (int i = 0; i < a.K; ++i)
      if (valid(i) && ids[i] == ids[j]) q += exp2_d(((double)logq[i] - (double)ref) * kLog2e);
    const double s = f.per_p == 0.0 ? 0.0 : f.per_p * exp2_d(entry(j) - f.m);
    a.fix[(size_t)r * a.K + j] = w == 0.f || !valid(j) ? 0.f : (float)(s - f.per_q * q);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const T* logits, T* grad, DistillArgs a) {
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * a.stride;
  T* g = grad + (size_t)r * a.V;
  const Row<const T> row(x, a.V);
  const Row<T> out(g, a.V);
  const bool vec = row.shift == out.shift;
  const float c = row_c(a, r), R = a.coef[2 * (size_t)r], factor = a.coef[2 * (size_t)r + 1];
  for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
    Unit<T> v;
    if (factor != 0.f) v = row.load(i);
    if (factor != 0.f) gradient_unit(v, c, R, factor);
    else v.fill(from_f<T>(0.f));
    out.store(i, v, vec, row.shift);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
    const long id = a.ids[(size_t)r * a.K + j], t = id - a.vocab_start;
    if (id >= 0 && id < a.vocab_total && t >= 0 && t < a.V) g[t] = from_f<T>(a.fix[(size_t)r * a.K + j]);
  }
}

// sum_u w_u KL_u / denom in a fixed order, FP64.  A row of weight 0 counts as 0 whatever it holds.
__global__ void weighted_sum_kernel(const float* __restrict__ rows, const float* __restrict__ weights, int U,
                                    double inv_denom, float* __restrict__ out) {
  __shared__ double part[32];
  double v = 0.0;
  for (int i = threadIdx.x; i < U; i += blockDim.x) {
    const double w = weights ? (double)weights[i] : 1.0;
    if (w != 0.0) v += w * (double)rows[i];
  }
  v = warp_sum_d(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < (blockDim.x >> 5) ? part[threadIdx.x] : 0.0;
    v = warp_sum_d(v);
    if (threadIdx.x == 0) out[0] = (float)(v * inv_denom);
  }
}

// x *= num / den unless that is 1 (the factor is on the device; the usual 1 costs one read per block).  The two are
// compared and not their quotient, which is a product with a reciprocal in this build and misses 1 for many equals.
template <typename T>
__global__ void scale_unless_one_kernel(T* __restrict__ x, long n, const float* __restrict__ num, float den) {
  if (num[0] == den) return;
  const float f = __fdiv_rn(num[0], den);
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x)
    x[i] = from_f<T>(to_f(x[i]) * f);
}

// -------------------------------------------------------------------------------------------------- host
template <typename F>
cudaError_t by_type(RowType t, F&& f) {
  if (t == RowType::f32) return f((float*)nullptr);
  if (t == RowType::f16) return f((__half*)nullptr);
  return f((__nv_bfloat16*)nullptr);
}

cudaError_t launched() {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) bb::launch_counter().fetch_add(1);
  return e;
}

// How a row is spread: blocks per cluster, threads per block, units held per thread (0: streamed).
struct Shape {
  int blocks, threads, units;
};

int units_of(int V, int width) { return (V * (long)width + 30) / 16; }   // of a row at any alignment

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v;
  }();
  return n;
}

// Rows held in registers: as few blocks as hold the row with 5 units per thread, and more while every SM still gets at
// most one.  units = 0: too long.
Shape held_shape(int rows, int units) {
  int b = 1;
  while (b < kMaxCluster && b * kThreads * 5 < units) b *= 2;
  while (b < kMaxCluster && 2l * rows * b <= sm_count() && units >= 2 * b * 256) b *= 2;
  for (int n : {1, 2, 5, 10}) {
    const int t = (units + b * n - 1) / (b * n);
    if (t <= kThreads) return {b, std::max(32, (t + 31) / 32 * 32), n};
  }
  return {kMaxCluster, kThreads, 0};
}

// Rows that stream: warps for the batches of units, up to 8 and a power of two, `least` blocks per row, and more of long
// rows while they have at least `part` units and three of them are resident on every SM at once.  Up to 4/3, 2, 3, 4 for
// every SM, us, vocabulary 151936 BF16: scores of 64 rows 8.5, 7.8, 7.8, 12.2, of 74 rows 8.4, 9.5, 9.5, 12.8, of 100 rows
// 12.4, 10.7, 9.6, 9.8, of 200 rows 16.9, 16.8, 14.1, 14.1; their gradient of 100 rows 13.4, 12.0, 10.3, 10.4, of 148 rows
// 13.5, 12.4, 12.3, 15.2; distillation with gradient of 100 rows 26.1, 24.0, 20.6, 20.5, of 148 rows 26.2, 24.6, 24.7, 31.8.
// At least 512 / 1024 units, 8 rows of 50257 columns: 64 entries with gradient 10.7 / 11.8, the scores' gradient 4.3 / 5.1.
Shape stream_shape(int rows, int units, int least = 1, int part = 512) {
  int b = least;
  while (b < kMaxCluster && 2l * rows * b <= 3 * sm_count() && units >= std::max(2048, 2 * b * part)) b *= 2;
  const int batches = ((units + b - 1) / b + kSpan - 1) / kSpan;
  int warps = 1;
  while (warps < std::min(batches, kStream / 32)) warps *= 2;
  return {b, 32 * warps, 0};
}

size_t feed_bytes(int threads) { return Feed<float, 1>::bytes(threads); }

// Whether rows are held rather than streamed: short ones always (4000 rows held / streamed, us, BF16: of 12000 columns,
// 1500 units, 63 / 103 with 20 alternatives, 88 / 99 distillation; of 20000, 2500 units, 91 / 105 and 133 / 117), longer
// ones while their blocks are resident at once.
// Alternatives take little else than the row.  Vocabulary 151936 BF16, 20 of 8 rows 10.3 / 11.7, of 32 rows 13.1 / 13.8, of
// 48 rows 15.3 / 15.9.  With 10 units per thread an SM has room for one block, and clusters of 8 do not fill all SMs:
// 151936 FP32, of 8 rows 9.2 / 11.0, of 16 rows 16.1 / 12.2.
bool hold_for_top(int rows, int units, Shape s) {
  return s.units && (units <= 2560 || 4l * rows * s.blocks <= (s.units == 10 ? 2 : 11) * sm_count());
}
// Distillation has the entries to prepare as well, which a block that streams does while its copies are on their way.
// 64 entries of 16 rows with gradient, BF16: of 24000 columns 9.3 / 11.1, 50257 10.6 / 11.4, 100000 13.1 / 12.4, 151936
// 15.1 / 13.1; of 64 rows of 24000 (1500 units in each of 2 blocks) 12.6 / 11.7; 148 of 17000 (one block) 12.3 / 14.0.
bool hold_for_distill(int rows, int units, Shape s) {
  if (units <= 2048) return true;
  return 4l * rows * s.blocks <= 7 * sm_count() && (s.blocks == 1 || units <= 1024 * s.blocks);
}

template <typename K, typename... A>
cudaError_t launch_rows(K kernel, int rows, Shape s, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)s.blocks, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return e;
  return launched();
}

}  // namespace

namespace bb {

cudaError_t launch_token_logprob(RowType t, const void* logits, const TokenArgs& a, cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    using Kernel = void (*)(const T*, TokenArgs);
    const bool e = a.entropy != nullptr;
    const int units = units_of(a.V, sizeof(T));
    Shape s = held_shape(a.U, units);
    if (!a.k || !hold_for_top(a.U, units, s)) s.units = 0;
    Kernel kern;
    switch (s.units) {
      case 1: kern = e ? token_top_kernel<T, true, 1> : token_top_kernel<T, false, 1>; break;
      case 2: kern = e ? token_top_kernel<T, true, 2> : token_top_kernel<T, false, 2>; break;
      case 5: kern = e ? token_top_kernel<T, true, 5> : token_top_kernel<T, false, 5>; break;
      case 10: kern = e ? token_top_kernel<T, true, 10> : token_top_kernel<T, false, 10>; break;
      default: {
        if (!a.k) {
          // Two batches for a warp, which are on their way at once.  Blocks of at least 512 / 1024 / 2048 units, us, BF16:
          // 32 rows of 32000 columns 4.6 / 4.1 / 4.2, 8 of 100000 4.4 / 4.4 / 5.3.
          s = stream_shape(a.U, units, 1, 1024);
          kern = e ? token_stream_kernel<T, true> : token_stream_kernel<T, false>;
          return launch_rows(kern, a.U, s, 0, stream, (const T*)logits, a);
        }
        s = stream_shape(a.U, units);
        size_t smem = feed_bytes(s.threads);
        kern = e ? token_top_stream_kernel<T, true> : token_top_stream_kernel<T, false>;
        smem = std::max(smem, sizeof(Select) + 4 * kCand) + sizeof(float) * (kBatch + units / 32 / s.blocks + 2 + kStream / 32 * kBatch);
        const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
        return launch_rows(kern, a.U, s, smem, stream, (const T*)logits, a);
      }
    }
    return launch_rows(kern, a.U, s, sizeof(Select), stream, (const T*)logits, a);
  });
}

cudaError_t launch_token_logprob_bwd(RowType t, const void* logits, void* grad, const TokenArgs& a,
                                     cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto* kern = a.d_entropy ? token_logprob_bwd_kernel<T, true> : token_logprob_bwd_kernel<T, false>;
    const Shape s = stream_shape(a.U, units_of(a.V, sizeof(T)));
    const size_t smem = feed_bytes(s.threads);
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_rows(kern, a.U, s, smem, stream, (const T*)logits, (T*)grad, a);
  });
}

cudaError_t launch_distill(RowType t, const void* logits, void* grad, const DistillArgs& a, cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const int units = units_of(a.V, sizeof(T));
    Shape s = held_shape(a.U, units);
    if (!hold_for_distill(a.U, units, s)) s.units = 0;
    using Kernel = void (*)(const T*, T*, DistillArgs);
    Kernel kern;
    size_t smem = Entries::bytes(a.K, s.threads);
    switch (s.units) {
      case 1: kern = distill_kernel<T, 1>; break;
      case 2: kern = distill_kernel<T, 2>; break;
      case 5: kern = distill_kernel<T, 5>; break;
      default: {
        kern = grad ? distill_stream_kernel<T, true> : distill_stream_kernel<T, false>;
        // With a second pass the rows in work (4 blocks for every SM) should fit L2: 4096 x 151936 BF16 (180 MB with one
        // block per row) 529 us with one, 484 us with two; 1024 x 32003 FP32 (76 MB) 76 us with one, 93 us with two.
        const bool twice = grad && a.U >= 2 * sm_count() && 4l * sm_count() * units * 16 > (100l << 20);
        s = stream_shape(a.U, units, twice ? 2 : 1);
        smem = feed_bytes(s.threads) + Entries::bytes(a.K, units / s.blocks / kSpan + 2);
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
      }
    }
    return launch_rows(kern, a.U, s, smem, stream, (const T*)logits, (T*)grad, a);
  });
}

cudaError_t launch_distill_finish(const DistillArgs& a, cudaStream_t stream) {
  distill_finish_kernel<<<(unsigned)a.U, 32, 0, stream>>>(a);
  return launched();
}

cudaError_t launch_distill_grad(RowType t, const void* logits, void* grad, const DistillArgs& a, cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    distill_grad_kernel<T><<<(unsigned)a.U, kThreads, 0, stream>>>((const T*)logits, (T*)grad, a);
    return launched();
  });
}

cudaError_t launch_weighted_sum(const float* rows, const float* weights, int U, double inv_denom, float* out,
                                cudaStream_t stream) {
  weighted_sum_kernel<<<1, 1024, 0, stream>>>(rows, weights, U, inv_denom, out);
  return launched();
}

cudaError_t launch_scale_unless_one(RowType t, void* x, long n, const float* num, float den, cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const int blocks = (int)std::min<long>((n + 4095) / 4096, 4l * sm_count());
    scale_unless_one_kernel<T><<<blocks, 512, 0, stream>>>((T*)x, n, num, den);
    return launched();
  });
}

}  // namespace bb
