// Kernels over rows of logits x [U, V]: log-probs of given tokens with entropy and the k likeliest tokens, their
// gradient, and the loss + gradient of distillation from a teacher known by its top log-probs.
//
// Everything is written in the base-2 domain of one row: c = log2(e) / T, t = x c - R for a reference R near the
// row's largest x c, e = 2^t, s = sum e.  Then p = e / s, ln p = ln 2 (t - log2 s), and the entropy is
// ln 2 (log2 s - sum e t / s), whatever R is: a thread keeps its own R, raised only when a logit passes it by more
// than 8 (sums grow by 2^8 at most), and partial (R, s, sum e t) triples are joined by rescaling.  Statistics are
// FP32; the few numbers of a row that everything else is scaled by (log s, the given tokens' shares) are FP64.
//
// A logit with x c <= -1e30 (-inf, or a mask of the type's lowest value) carries no probability; a row without any
// other has log-probs -inf, entropy 0 and gradient 0.
#include "vocab_rows.h"

#include <c10/util/Exception.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace {

using bb::DistillArgs;
using bb::kMaxTop;
using bb::RowType;
using bb::TokenArgs;

constexpr int kThreads = 512;
constexpr int kCand = 2048;     // candidates of the selection kept in shared memory
constexpr float kMasked = -1e30f;
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

// One row as units of 8 elements on 16-byte boundaries: unit i covers the aligned positions 8i .. 8i + 7, and
// position a holds token a - shift.  Only the first and the last unit can be partly outside the row.
template <typename T>
struct Row {
  T* p;        // aligned base: row start - shift
  int shift;   // elements between the 16-byte boundary and the row's first element
  int end;     // V + shift
  int units;

  __device__ __forceinline__ Row(T* row, int V) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    p = row - shift;
    end = V + shift;
    units = (end + 7) >> 3;
  }
  __device__ __forceinline__ bool full(int i) const { return 8 * i >= shift && 8 * i + 8 <= end; }
  __device__ __forceinline__ void load(int i, float* f) const {
    if (full(i)) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[2 * i], b = reinterpret_cast<const float4*>(p)[2 * i + 1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
        f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
      } else {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_f(h[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int a = 8 * i + j;
        f[j] = (a >= shift && a < end) ? to_f(p[a]) : -INFINITY;
      }
    }
  }
  // `vec`: the output's rows start at the same offset from a 16-byte boundary as the input's
  __device__ __forceinline__ void store(int i, const float* f, bool vec, int in_shift) const {
    // positions are the INPUT's (in_shift); this row is the output's
    const int a0 = 8 * i - in_shift + shift;
    if (vec && full(i)) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[2 * i] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[2 * i + 1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        uint4 v;
        T* h = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = from_f<T>(f[j]);
        reinterpret_cast<uint4*>(p)[i] = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (a0 + j >= shift && a0 + j < end) p[a0 + j] = from_f<T>(f[j]);
    }
  }
};

struct Stat {
  float R, s, et;

  static __device__ __forceinline__ Stat none() { return {kMasked, 0.f, 0.f}; }
  __device__ __forceinline__ void raise(float to) {
    const float d = R - to, k = ex2(d);
    et = k * (et + d * s);
    s *= k;
    R = to;
  }
  template <bool kEntropy>
  __device__ __forceinline__ void push8(const float* f, float c) {
    float top = f[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, f[j]);
    top *= c;
    if (top > R + kSlack) raise(top);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = fmaf(f[j], c, -R), e = ex2(t);
      s += e;
      if (kEntropy) et += e * fmaxf(t, -1e4f);   // e = 0 there; -inf would make it NaN
    }
  }
  __device__ __forceinline__ void join(Stat o) {
    if (o.R > R) {
      const Stat m = *this;
      *this = o;
      o = m;
    }
    if (o.s == 0.f) return;
    o.raise(R);
    s += o.s;
    et += o.et;
  }
};

__device__ __forceinline__ Stat warp_join(Stat a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.R = __shfl_xor_sync(0xffffffffu, a.R, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.et = __shfl_xor_sync(0xffffffffu, a.et, o);
    a.join(b);
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

// Order-preserving map of FP32 to unsigned; -0 counts as +0 and NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  v = fmaxf(v, -INFINITY) + 0.f;
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// ---------------------------------------------------------------------------------------------- selection
// The k largest of a row, ties to the lower id.  `best` is the largest key that this thread saw (its stripe: units
// tid, tid + blockDim, ...).  The k-th largest of the stripes' maxima is a bound that k elements reach, so about k
// elements lie above it; they are gathered and ranked by counting.  Rows in which more than kCand reach the bound
// (many equal logits) are settled exactly: the k-th largest key by bisection over the row, all above it, and the
// first of its equals in index order.
struct Select {
  unsigned long long cand[kCand];
  int count, scan[33];
};

template <typename T>
__device__ int count_ge(const Row<T>& row, uint32_t key, int* scratch) {
  int n = 0;
  for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
    float f[8];
    row.load(i, f);
    const bool full = row.full(i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int a = 8 * i + j;
      n += (full || (a >= row.shift && a < row.end)) && order_key(f[j]) >= key;
    }
  }
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = n;
  __syncthreads();
  n = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : 0;
  return __reduce_add_sync(0xffffffffu, n);
}

__device__ __forceinline__ unsigned long long pack_key(uint32_t key, int token) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (uint32_t)token);
}

// Gathers the elements with key >= `key` into sel.cand (as many as fit) and returns their number.
template <typename T>
__device__ int gather_ge(const Row<T>& row, uint32_t key, uint32_t best, Select& sel) {
  __syncthreads();
  if (threadIdx.x == 0) sel.count = 0;
  __syncthreads();
  if (best >= key) {
    for (int i = threadIdx.x; i < row.units; i += blockDim.x) {
      float f[8];
      row.load(i, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int a = 8 * i + j;
        const uint32_t k = order_key(f[j]);
        if (k >= key && a >= row.shift && a < row.end) {
          const int at = atomicAdd(&sel.count, 1);
          if (at < kCand) sel.cand[at] = pack_key(k, a - row.shift);
        }
      }
    }
  }
  __syncthreads();
  return sel.count;
}

// After this, sel.cand[0 .. n) holds the k winners among n >= k candidates; returns n.
template <typename T>
__device__ int select_candidates(const Row<T>& row, int k, uint32_t best, bool any, Select& sel) {
  // the k-th largest of the stripes' maxima (0 when fewer than k stripes hold elements: everything)
  uint32_t bound = 0;
  if (__syncthreads_count(any) >= k) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = bound | (1u << bit);
      if (__syncthreads_count(any && best >= trial) >= k) bound = trial;
    }
  }
  int n = gather_ge(row, bound, any ? best : 0u, sel);
  if (n <= kCand) return n;
  // exact: the k-th largest key of the row
  uint32_t kth = bound;
  if (count_ge(row, bound + 1, sel.scan) >= k) {
    kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = kth | (1u << bit);
      if (count_ge(row, trial, sel.scan) >= k) kth = trial;
    }
  }
  n = gather_ge(row, kth + 1, any ? best : 0u, sel);        // fewer than k
  // its equals, in index order, until k are held
  for (int i0 = 0; i0 < row.units && n < k; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    float f[8];
    uint32_t hit = 0;
    if (i < row.units) {
      row.load(i, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int a = 8 * i + j;
        if (order_key(f[j]) == kth && a >= row.shift && a < row.end) hit |= 1u << j;
      }
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
      if (at < k) sel.cand[at] = pack_key(kth, 8 * i + j - row.shift);
      ++at;
    }
    n = min(k, n + total);
  }
  __syncthreads();
  return n;
}

// ------------------------------------------------------------------------------------- token log-probs
__device__ __forceinline__ float row_c(const float* temp, double temp1, int row) {
  return (float)(kLog2e / (temp ? (double)temp[row] : temp1));
}

__device__ __forceinline__ float finish_logp(double x, float c, Stat st, double log2s) {
  const double xc = x * (double)c;
  if (st.s == 0.f || xc <= (double)kMasked) return st.s == st.s ? -INFINITY : st.s;
  return (float)(kLn2 * (xc - (double)st.R - log2s));
}

template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads) token_logprob_kernel(const T* __restrict__ logits, TokenArgs a) {
  __shared__ Stat part[32];
  extern __shared__ __align__(16) unsigned char dyn[];
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const float c = row_c(a.temp, a.temp1, r);
  Stat st = Stat::none();
  float best = -INFINITY;
  for (int i = threadIdx.x; i < row.units; i += kThreads) {
    float f[8];
    row.load(i, f);
    st.push8<kEntropy>(f, c);
    if (kTop) {
#pragma unroll
      for (int j = 0; j < 8; ++j) best = fmaxf(best, f[j]);
    }
  }
  st = block_join(st, part);
  const double log2s = log2((double)st.s);
  for (int j = threadIdx.x; j < a.n; j += kThreads) {
    const long t = a.tokens[(size_t)r * a.n + j] - a.vocab_start;
    const bool here = t >= 0 && t < a.V;
    float v = 0.f;
    if (here) v = a.open ? to_f(x[t]) * c : finish_logp(to_f(x[t]), c, st, log2s);
    a.logp[(size_t)r * a.n + j] = v;
  }
  if (threadIdx.x == 0) {
    const bool empty = st.s == 0.f;
    if (a.entropy) a.entropy[r] = empty ? 0.f : (float)(kLn2 * (log2s - (double)st.et / (double)st.s));
    float* o = a.stats + 3 * (size_t)r;
    o[0] = st.R;
    o[1] = a.open ? st.s : (empty ? 0.f : (float)(1.0 / (double)st.s));
    o[2] = a.open ? st.et : (empty ? 0.f : (float)((double)st.et / (double)st.s));
  }
  if (kTop) {
    Select& sel = *reinterpret_cast<Select*>(dyn);
    const int n = select_candidates(row, a.k, order_key(best), (int)threadIdx.x < row.units, sel);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned long long mine = sel.cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sel.cand[j] > mine;
      if (rank < a.k) {
        const int t = (int)(0xffffffffu - (uint32_t)mine);
        a.top_ids[(size_t)r * a.k + rank] = t + a.vocab_start;
        a.top_logp[(size_t)r * a.k + rank] = a.open ? to_f(x[t]) : finish_logp(to_f(x[t]), c, st, log2s);
      }
    }
  }
}

// d x_v = (e / s / T) (-G - dH ln 2 (t - E[t])) + [v = t_j] g_j / T, G = sum_j g_j
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kThreads)
    token_logprob_bwd_kernel(const T* __restrict__ logits, T* __restrict__ grad, TokenArgs a) {
  __shared__ float scratch[32];
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * a.stride;
  T* g = grad + (size_t)r * a.V;
  const Row<const T> row(x, a.V);
  const Row<T> out(g, a.V);
  const bool vec = row.shift == out.shift;
  const float c = row_c(a.temp, a.temp1, r);
  const float it = (float)(1.0 / (a.temp ? (double)a.temp[r] : a.temp1));
  const float* st = a.stats + 3 * (size_t)r;
  const float R = st[0], inv = st[1], mean = st[2];
  float G = 0.f;      // a token outside the whole vocabulary (an ignored position) has no gradient
  for (int j = threadIdx.x; j < a.n; j += kThreads) {
    const long t = a.tokens[(size_t)r * a.n + j];
    G += (t >= 0 && t < a.vocab_total) ? a.d_logp[(size_t)r * a.n + j] : 0.f;
  }
  G = bb::block_sum(G, scratch);
  const float dh = kEntropy ? a.d_entropy[r] * (float)kLn2 : 0.f;
  const float A = it * inv * (dh * mean - G), B = -it * inv * dh;
  for (int i = threadIdx.x; i < row.units; i += kThreads) {
    float f[8];
    row.load(i, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = fmaf(f[j], c, -R), e = ex2(t);
      f[j] = e * (kEntropy ? fmaf(B, fmaxf(t, -1e4f), A) : A);
    }
    out.store(i, f, vec, row.shift);
  }
  __syncthreads();
  // the given tokens' columns, once per distinct token
  for (int j = threadIdx.x; j < a.n; j += kThreads) {
    const int64_t* tk = a.tokens + (size_t)r * a.n;
    const long t = tk[j] - a.vocab_start;
    if (t < 0 || t >= a.V) continue;
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
struct Entries {
  double xc[kMaxTop];      // x c of the entry, -inf where masked
  float logq[kMaxTop];
  float fix[kMaxTop];
  int col[kMaxTop];        // column in this shard, or -1
  unsigned char state[kMaxTop];   // 0 dropped, 1 first of its id, 2 repeats an earlier entry
  float R, factor, kl;
  int repeats;
};

// KL and gradient factors of a row from its entries and the (R, s) of everything else; warp 0, all lanes.
__device__ void finish_row(Entries& en, int K, Stat rest, bool tail, double scale, double inv_temp) {
  const int lane = threadIdx.x & 31;
  double top = -INFINITY;      // teacher: sum of q, renormalised over the entries without a tail class
  for (int j = lane; j < K; j += 32)
    if (en.state[j]) top = fmax(top, (double)en.logq[j]);
  top = warp_max_d(top);
  double shift = 0.0;
  if (!tail && top > -INFINITY) {
    double z = 0.0;
    for (int j = lane; j < K; j += 32)
      if (en.state[j]) z += exp((double)en.logq[j] - top);
    shift = top + log(warp_sum_d(z));
  }
  double q_sum = 0.0, m = rest.s == 0.f ? -INFINITY : (double)rest.R;
  for (int j = lane; j < K; j += 32) {
    if (!en.state[j]) continue;
    q_sum += exp((double)en.logq[j] - shift);
    m = fmax(m, en.xc[j]);
  }
  q_sum = warp_sum_d(q_sum);
  m = warp_max_d(m);
  const double q_rest = tail ? fmax(0.0, 1.0 - q_sum) : 0.0;
  const bool no_teacher = !tail && !(top > -INFINITY);
  bool any = false;
  for (int j = lane; j < K; j += 32) any |= en.state[j] != 0;
  any = __any_sync(0xffffffffu, any) && !no_teacher;
  if (!any || m == -INFINITY) {
    // no entry: nothing to learn.  No student probability anywhere: the divergence is infinite, without gradient
    const bool nan = rest.s != rest.s;
    for (int j = lane; j < K; j += 32) en.fix[j] = 0.f;
    if (lane == 0) {
      en.R = 0.f;
      en.factor = 0.f;
      en.kl = !any ? 0.f : (nan ? rest.s : INFINITY);
    }
    return;
  }
  const double rest_share = rest.s == 0.f ? 0.0 : (double)rest.s * exp2((double)rest.R - m);
  double z = 0.0;
  for (int j = lane; j < K; j += 32)
    if (en.state[j] == 1) z += exp2(en.xc[j] - m);
  z = warp_sum_d(z) + rest_share;
  const double log2z = log2(z), p_rest = rest_share / z, total = q_sum + q_rest;
  double kl = 0.0;
  for (int j = lane; j < K; j += 32) {
    if (!en.state[j]) {
      en.fix[j] = 0.f;
      continue;
    }
    const double lq = (double)en.logq[j] - shift, q = exp(lq);
    if (q > 0.0) kl += q * (lq - kLn2 * (en.xc[j] - m - log2z));
    else if (!(q == 0.0)) kl += q;      // NaN
    double held = q;
    if (en.repeats && en.state[j] == 1)
      for (int i = j + 1; i < K; ++i)
        if (en.state[i] == 2 && en.col[i] == en.col[j]) held += exp((double)en.logq[i] - shift);
    en.fix[j] = (float)(scale * inv_temp * (total * exp2(en.xc[j] - m) / z - held));
  }
  kl = warp_sum_d(kl);
  if (lane == 0) {
    if (q_rest > 0.0) {
      kl += q_rest * (log(q_rest) - kLn2 * ((double)rest.R - m + log2((double)rest.s) - log2z));
      if (rest.s == 0.f) kl = INFINITY;
    }
    en.kl = (float)kl;
    en.R = rest.R;
    en.factor = rest.s == 0.f ? 0.f : (float)(scale * inv_temp * (total * p_rest - q_rest) / (double)rest.s);
  }
}

// Loads the teacher's entries of row r and marks their columns in `mask` (one byte per unit).
template <typename T>
__device__ void load_entries(Entries& en, const DistillArgs& a, int r, const T* x, const Row<const T>& row, float c,
                             unsigned int* mask) {
  const int words = (row.units + 3) >> 2;
  for (int i = threadIdx.x; i < words; i += blockDim.x) mask[i] = 0u;
  if (threadIdx.x == 0) en.repeats = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
    const long id = a.ids[(size_t)r * a.K + j];
    const long t = id - a.vocab_start;
    const bool valid = id >= 0 && id < a.vocab_total, here = valid && t >= 0 && t < a.V;
    en.logq[j] = a.logq[(size_t)r * a.K + j];
    en.col[j] = here ? (int)t : -1;
    en.state[j] = valid ? 1 : 0;
    double xc = 0.0;
    if (here) {
      xc = (double)to_f(x[t]) * (double)c;
      if (xc <= (double)kMasked) xc = -INFINITY;
      const int at = (int)t + row.shift;
      if (atomicOr(&mask[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u) en.repeats = 1;
    }
    en.xc[j] = xc;
  }
  __syncthreads();
  if (en.repeats) {
    for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
      if (en.col[j] < 0) continue;
      for (int i = 0; i < j; ++i)
        if (en.col[i] == en.col[j]) en.state[j] = 2;
    }
    __syncthreads();
  }
}

// g_v = k 2^(x_v c - R); k = 0 writes zeros without reading the row.
template <typename T>
__device__ __forceinline__ void write_gradient(const Row<const T>& row, T* g, int V, float c, float R, float k) {
  const Row<T> out(g, V);
  const bool vec = row.shift == out.shift;
  for (int i = threadIdx.x; i < row.units; i += kThreads) {
    float f[8];
    if (k != 0.f) {
      row.load(i, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = k * ex2(fmaf(f[j], c, -R));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
    out.store(i, f, vec, row.shift);
  }
}

// One block per row: pass 1 takes the statistics of the columns outside the teacher's entries (their bits in `mask`
// replace a logit by -inf), warp 0 finishes the row, pass 2 reads the row again and writes its gradient.
template <typename T, bool kGrad, bool kOpen>
__global__ void __launch_bounds__(kThreads) distill_kernel(const T* logits, T* grad, DistillArgs a) {
  __shared__ Stat part[32];
  __shared__ Entries en;
  extern __shared__ __align__(16) unsigned int mask[];
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * a.stride;
  const Row<const T> row(x, a.V);
  const double inv_temp = 1.0 / (a.temp ? (double)a.temp[r] : a.temp1);
  const float c = row_c(a.temp, a.temp1, r);
  const float w = a.weights ? a.weights[r] : 1.f;
  load_entries(en, a, r, x, row, c, mask);
  Stat st = Stat::none();
  if (w != 0.f) {
    const unsigned char* bits = reinterpret_cast<const unsigned char*>(mask);
    for (int i = threadIdx.x; i < row.units; i += kThreads) {
      float f[8];
      row.load(i, f);
      const unsigned m = bits[i];
      if (m) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (m >> j & 1u) f[j] = -INFINITY;
      }
      st.push8<false>(f, c);
    }
  }
  st = block_join(st, part);
  if (kOpen) {
    for (int j = threadIdx.x; j < a.K; j += kThreads) a.xc[(size_t)r * a.K + j] = (float)en.xc[j];
    if (threadIdx.x == 0) {
      a.stats[2 * (size_t)r] = st.R;
      a.stats[2 * (size_t)r + 1] = st.s;
    }
    return;
  }
  if (threadIdx.x < 32) finish_row(en, a.K, st, a.tail, (double)w * a.scale, inv_temp);
  __syncthreads();
  if (threadIdx.x == 0) a.rows[r] = w == 0.f ? 0.f : en.kl;
  if (!kGrad) return;
  T* g = grad + (size_t)r * a.V;
  write_gradient(row, g, a.V, c, en.R, w == 0.f ? 0.f : en.factor);
  __syncthreads();
  if (w == 0.f) return;
  for (int j = threadIdx.x; j < a.K; j += kThreads)
    if (en.state[j] == 1 && en.col[j] >= 0) g[en.col[j]] = from_f<T>(en.fix[j]);
}

// Vocabulary in shards: one warp per row finishes it from the joined (R, s) and x c of every entry.
__global__ void distill_finish_kernel(DistillArgs a) {
  __shared__ Entries en;
  const int r = blockIdx.x, lane = threadIdx.x;
  const int64_t* ids = a.ids + (size_t)r * a.K;
  for (int j = lane; j < a.K; j += 32) {
    const long id = ids[j];
    en.logq[j] = a.logq[(size_t)r * a.K + j];
    en.col[j] = (int)id;
    const float xc = a.xc[(size_t)r * a.K + j];
    en.xc[j] = xc <= kMasked ? -INFINITY : (double)xc;
    bool first = true;
    for (int i = 0; i < j; ++i) first &= ids[i] != id;
    en.state[j] = id < 0 || id >= a.vocab_total ? 0 : (first ? 1 : 2);
  }
  if (lane == 0) en.repeats = 1;
  __syncwarp();
  Stat st = Stat::none();
  st.R = a.stats[2 * (size_t)r];
  st.s = a.stats[2 * (size_t)r + 1];
  const float w = a.weights ? a.weights[r] : 1.f;
  finish_row(en, a.K, st, a.tail, (double)w * a.scale, 1.0 / (a.temp ? (double)a.temp[r] : a.temp1));
  __syncwarp();
  if (lane == 0) {
    a.rows[r] = w == 0.f ? 0.f : en.kl;
    a.coef[2 * (size_t)r] = en.R;
    a.coef[2 * (size_t)r + 1] = w == 0.f ? 0.f : en.factor;
  }
  for (int j = lane; j < a.K; j += 32) {
    int first = j;      // every entry of a repeated id carries the id's gradient
    if (en.state[j] == 2)
      for (first = 0; ids[first] != ids[j];) ++first;
    a.fix[(size_t)r * a.K + j] = w == 0.f ? 0.f : en.fix[first];
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const T* logits, T* grad, DistillArgs a) {
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * a.stride;
  T* g = grad + (size_t)r * a.V;
  const Row<const T> row(x, a.V);
  const float c = row_c(a.temp, a.temp1, r);
  write_gradient(row, g, a.V, c, a.coef[2 * (size_t)r], a.coef[2 * (size_t)r + 1]);
  __syncthreads();
  for (int j = threadIdx.x; j < a.K; j += kThreads) {
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

// x *= num / den unless that is 1 (the factor is on the device; the usual 1 costs one read per block).
template <typename T>
__global__ void scale_unless_one_kernel(T* __restrict__ x, long n, const float* __restrict__ num, float den) {
  const float f = num[0] / den;
  if (f == 1.f) return;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x)
    x[i] = from_f<T>(to_f(x[i]) * f);
}

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

}  // namespace

namespace bb {

cudaError_t launch_token_logprob(RowType t, const void* logits, const TokenArgs& a, cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto* kern = a.k ? (a.entropy ? token_logprob_kernel<T, true, true> : token_logprob_kernel<T, false, true>)
                     : (a.entropy ? token_logprob_kernel<T, true, false> : token_logprob_kernel<T, false, false>);
    kern<<<(unsigned)a.U, kThreads, a.k ? sizeof(Select) : 0, stream>>>((const T*)logits, a);
    return launched();
  });
}

cudaError_t launch_token_logprob_bwd(RowType t, const void* logits, void* grad, const TokenArgs& a,
                                     cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto* kern = a.d_entropy ? token_logprob_bwd_kernel<T, true> : token_logprob_bwd_kernel<T, false>;
    kern<<<(unsigned)a.U, kThreads, 0, stream>>>((const T*)logits, (T*)grad, a);
    return launched();
  });
}

size_t distill_smem(long V) {   // one byte per unit, in words: (V + 7 + 7) / 8 units at most
  return ((size_t)(V + 14) / 8 + 3) / 4 * 4;
}

cudaError_t launch_distill(RowType t, Distill mode, const void* logits, void* grad, const DistillArgs& a,
                           cudaStream_t stream) {
  return by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto* kern = mode == Distill::open ? distill_kernel<T, false, true>
                                       : (mode == Distill::loss ? distill_kernel<T, false, false>
                                                                : distill_kernel<T, true, false>);
    const size_t smem = distill_smem(a.V);
    if (smem + sizeof(Entries) + 1024 > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return e;
    }
    kern<<<(unsigned)a.U, kThreads, smem, stream>>>((const T*)logits, (T*)grad, a);
    return launched();
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
    const int blocks = resident_grid(scale_unless_one_kernel<T>, 512, 0, (n + 4095) / 4096);
    scale_unless_one_kernel<T><<<blocks, 512, 0, stream>>>((T*)x, n, num, den);
    return launched();
  });
}

}  // namespace bb
