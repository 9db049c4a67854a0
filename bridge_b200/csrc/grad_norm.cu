// The 2-norm over many gradient tensors, of all or slot by slot, and the gradients scaled down to a bound.
//
//   sums     one block per chunk of a tensor (of one slot of it): the chunk's sum of squares, in 64 bits
//   finish   one block per slot: the sum over the slot's chunks in a fixed order, norm = sqrt(sum) / grad_scale and the
//            factor min(1, max_norm / (norm + eps)) / grad_scale
//   scale    one block per chunk: out = factor x, rounded once
//
// Lists of at most 1 MB are one launch: a cluster of eight blocks whose warps sum their chunks, meet in shared memory and
// scale them.
//
// What bounds it: reading every value once for the norm, and once more, above the L2's 126 MB, to scale it.  The second
// pass goes through the chunks backwards, so that what the first one read last is still there.  A list's pointers travel
// in the kernels' parameters: no table is uploaded, and a captured graph keeps its own.
//
// 217 M FP32 values of eight slots 0.39 ms (sums 0.137, 6.3 TB/s; scaling 0.254, 6.8 TB/s); 566 M BF16 values into FP32
// 0.69 ms (0.178 and 0.511); 16 tensors of 53 thousand values 6.6 us.
//
// Squares are FP32 in sums of eight, which are added up in 64 bits; sums outside [1e-25, 1e37] (infinite or vanishing
// squares, and zeros) are taken again value by value in 64 bits, so that no finite gradient overflows or disappears.  The
// factor is 64-bit too; where it leaves [1e-30, 1e30] the values are scaled by two factors, so that neither is a
// subnormal, which would count as 0, or infinite.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>
#include <string>
#include <vector>

#include "common.cuh"

namespace {

namespace cg = cooperative_groups;
using OptTensor = c10::optional<torch::Tensor>;
constexpr int kThreads = 256;
constexpr int kUnroll = 4;      // 16-byte loads in flight per thread

enum Kind : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct Entry {
  const void* in;
  void* out;
  long n;            // values of one slot
  int first;         // the tensor's first chunk among all of the launch
  int chunks;        // per slot
  int at;            // the tensor's first chunk among a slot's
  short kind, out_kind;
};

template <int N>
struct Table {
  Entry e[N];
  int count, slots, total, per_slot;   // total: chunks of the launch; per_slot: chunks of a slot, of all launches
  long chunk;                          // values
};

template <typename T>
struct Io;
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

template <typename T>
struct alignas(16) Vec {
  T v[16 / sizeof(T)];
};

struct Chunk {
  int entry, slot, part;   // part: the chunk among its slot's, of all tensors
  long begin, n;           // values from the tensor's base
};

template <int N>
__device__ __forceinline__ Chunk locate(const Table<N>& t, int id) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {        // the last tensor that begins at or before the chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= id) lo = mid;
    else hi = mid - 1;
  }
  const Entry& e = t.e[lo];
  const int local = id - e.first, slot = local / e.chunks, j = local - slot * e.chunks;
  const long at = (long)j * t.chunk;
  return {lo, slot, e.at + j, (long)slot * e.n + at, min(t.chunk, e.n - at)};
}

// Values before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ long lead(const T* p, long n) {
  const long k = (long)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (long)sizeof(T);
  return k < n ? k : n;
}

// A chunk's sum of squares, of thread `tid` of NT.
template <int NT, typename T>
__device__ double chunk_sum(const T* x, long n, int tid) {
  constexpr int V = 16 / sizeof(T);
  const long head = lead(x, n), vecs = (n - head) / V;
  const Vec<T>* body = reinterpret_cast<const Vec<T>*>(x + head);
  double sum = 0.0;
  const auto one = [&](float v) { sum += (double)v * (double)v; };
  const auto add = [&](const Vec<T>& a) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s = fmaf(Io<T>::get(a.v[i]), Io<T>::get(a.v[i]), s);
    if (s >= 1e-25f && s <= 1e37f) {
      sum += (double)s;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) one(Io<T>::get(a.v[i]));
    }
  };
  long i = tid;
  for (; i + (kUnroll - 1) * NT < vecs; i += kUnroll * NT) {
    Vec<T> a[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) a[k] = body[i + k * NT];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) add(a[k]);
  }
  for (; i < vecs; i += NT) add(body[i]);
  if (tid < head) one(Io<T>::get(x[tid]));
  const long tail = head + vecs * V + tid;
  if (tail < n) one(Io<T>::get(x[tail]));
  return sum;
}

__device__ __forceinline__ double block_sum_f64(double v, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += scratch[i];
  return s;
}

// A factor as two: f alone (g = 1), or f in [0.5, 1) times a power of two where one FP32 value could not hold it.
struct Factor {
  float f, g;
  __device__ __forceinline__ float operator*(float v) const { return (f * v) * g; }
};

__device__ __forceinline__ Factor split(double factor) {
  if (!(fabs(factor) > 0.0 && (fabs(factor) < 1e-30 || fabs(factor) > 1e30)) || isinf(factor)) return {(float)factor, 1.f};
  int e;
  const double m = frexp(factor, &e);
  const int at = min(max(e, -126), 127);
  return {(float)ldexp(m, e - at), (float)ldexp(1.0, at)};
}

template <int NT, typename T, typename O>
__device__ void chunk_scale(const T* x, O* y, long n, const Factor& f, int tid) {
  constexpr int V = 16 / sizeof(T);
  const long head = lead(x, n), vecs = (n - head) / V;
  const Vec<T>* body = reinterpret_cast<const Vec<T>*>(x + head);
  O* to = y + head;
  const bool wide = reinterpret_cast<uintptr_t>(to) % (V * sizeof(O)) == 0;
  const auto put = [&](const Vec<T>& a, long i) {
    alignas(32) O r[V];
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = Io<O>::put(f * Io<T>::get(a.v[k]));
    if (wide) {
      // (16-bit gradients into FP32: 32 bytes in one store, or every sector would be written in halves)
      const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
      if constexpr (V * sizeof(O) == 32)
        asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + i * V), "r"(w[0]), "r"(w[1]),
                     "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
      else
        __stcs(reinterpret_cast<uint4*>(to + i * V), *reinterpret_cast<const uint4*>(r));
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) to[i * V + k] = r[k];
    }
  };
  long i = tid;
  for (; i + (kUnroll - 1) * NT < vecs; i += kUnroll * NT) {
    Vec<T> a[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) a[k] = body[i + k * NT];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) put(a[k], i + k * NT);
  }
  for (; i < vecs; i += NT) put(body[i], i);
  if (tid < head) y[tid] = Io<O>::put(f * Io<T>::get(x[tid]));
  const long tail = head + vecs * V + tid;
  if (tail < n) y[tail] = Io<O>::put(f * Io<T>::get(x[tail]));
}

template <int NT>
__device__ double sum_of(const Entry& e, const Chunk& c, int tid) {
  if (e.kind == kF32) return chunk_sum<NT>(static_cast<const float*>(e.in) + c.begin, c.n, tid);
  if (e.kind == kBF16) return chunk_sum<NT>(static_cast<const __nv_bfloat16*>(e.in) + c.begin, c.n, tid);
  return chunk_sum<NT>(static_cast<const __half*>(e.in) + c.begin, c.n, tid);
}

template <int NT>
__device__ void scale_of(const Entry& e, const Chunk& c, const Factor& f, int tid) {
  if (f.f == 1.f && f.g == 1.f && e.in == e.out) return;
  if (e.kind == kF32) {
    chunk_scale<NT>(static_cast<const float*>(e.in) + c.begin, static_cast<float*>(e.out) + c.begin, c.n, f, tid);
  } else if (e.kind == kBF16) {
    const auto* x = static_cast<const __nv_bfloat16*>(e.in) + c.begin;
    if (e.out_kind == kF32) chunk_scale<NT>(x, static_cast<float*>(e.out) + c.begin, c.n, f, tid);
    else chunk_scale<NT>(x, static_cast<__nv_bfloat16*>(e.out) + c.begin, c.n, f, tid);
  } else {
    const auto* x = static_cast<const __half*>(e.in) + c.begin;
    if (e.out_kind == kF32) chunk_scale<NT>(x, static_cast<float*>(e.out) + c.begin, c.n, f, tid);
    else chunk_scale<NT>(x, static_cast<__half*>(e.out) + c.begin, c.n, f, tid);
  }
}

struct Bound {
  double grad_scale, max_norm;
  const float* max_norms;    // per slot, or null
  float* norm;
  bool scale;
};

__device__ __forceinline__ Factor finish(const Bound& b, int slot, double sum, bool write) {
  const double n = sqrt(sum) / b.grad_scale;
  if (write) b.norm[slot] = (float)n;
  const double most = b.max_norms ? (double)b.max_norms[slot] : b.max_norm;
  // (a NaN norm makes the factor NaN)
  return split((n + 1e-6 <= most ? 1.0 : most / (n + 1e-6)) / b.grad_scale);
}

template <int N>
__global__ void __launch_bounds__(kThreads) sums_kernel(const __grid_constant__ Table<N> t, double* parts) {
  __shared__ double scratch[kThreads / 32];
  const Chunk c = locate(t, blockIdx.x);
  const double s = block_sum_f64(sum_of<kThreads>(t.e[c.entry], c, threadIdx.x), scratch);
  if (threadIdx.x == 0) parts[(long)c.slot * t.per_slot + c.part] = s;
}

__global__ void __launch_bounds__(1024) finish_kernel(const double* parts, int per_slot, const Bound b, Factor* factor) {
  __shared__ double scratch[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < per_slot; i += 1024) s += parts[(long)blockIdx.x * per_slot + i];
  s = block_sum_f64(s, scratch);
  if (threadIdx.x) return;
  const Factor f = finish(b, blockIdx.x, s, true);
  if (b.scale) factor[blockIdx.x] = f;
}

template <int N>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table<N> t, const Factor* factor) {
  const Chunk c = locate(t, t.total - 1 - blockIdx.x);
  scale_of<kThreads>(t.e[c.entry], c, factor[c.slot], threadIdx.x);
}

// A short list: every warp of the cluster takes every 128th chunk; sums go warp by warp, in the blocks' and warps' order.
constexpr int kSmallBlocks = 8, kSmallWarps = 16, kSmallSlots = 32;

template <int N>
__global__ void __cluster_dims__(kSmallBlocks, 1, 1) __launch_bounds__(32 * kSmallWarps)
    small_kernel(const __grid_constant__ Table<N> t, const Bound b) {
  __shared__ double sums[kSmallWarps][kSmallSlots];
  __shared__ Factor factor[kSmallSlots];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * kSmallWarps + warp, step = kSmallBlocks * kSmallWarps;
  if (lane < t.slots) sums[warp][lane] = 0.0;
  __syncwarp();
  for (int id = first; id < t.total; id += step) {
    const Chunk c = locate(t, id);
    double s = sum_of<32>(t.e[c.entry], c, lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sums[warp][c.slot] += s;
  }
  cluster.sync();
  for (int slot = warp; slot < t.slots; slot += kSmallWarps) {
    double s = 0.0;       // four of the 128 warps' sums a lane
#pragma unroll
    for (int k = 0; k < kSmallBlocks * kSmallWarps / 32; ++k) {
      const int i = lane * (kSmallBlocks * kSmallWarps / 32) + k;
      s += *cluster.map_shared_rank(&sums[i % kSmallWarps][slot], i / kSmallWarps);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) factor[slot] = finish(b, slot, s, blockIdx.x == 0);
  }
  cluster.sync();         // (the peers' sums stay until all have read them)
  if (!b.scale) return;
  for (int id = first; id < t.total; id += step) {
    const Chunk c = locate(t, id);
    scale_of<32>(t.e[c.entry], c, factor[c.slot], lane);
  }
}

// ------------------------------------------------------------------------------------------------ host
short kind_of(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kHalf: return kF16;
    default: TORCH_CHECK_TYPE(false, "clip_grad_norm: gradients are float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

// A Python list or tuple of tensors, looked at where it is: hundreds of them take longer to convert than to work on.
class Tensors {
 public:
  explicit Tensors(const pybind11::object& list) : list_(list) {
    TORCH_CHECK_TYPE(PyList_Check(list.ptr()) || PyTuple_Check(list.ptr()), "clip_grad_norm: needs a list of tensors");
    n_ = (size_t)PySequence_Fast_GET_SIZE(list.ptr());
    items_ = PySequence_Fast_ITEMS(list.ptr());
    for (size_t i = 0; i < n_; ++i)
      TORCH_CHECK_TYPE(THPVariable_Check(items_[i]), "clip_grad_norm: needs a list of tensors");
  }
  size_t size() const { return n_; }
  bool empty() const { return n_ == 0; }
  const torch::Tensor& operator[](size_t i) const { return THPVariable_Unpack(items_[i]); }

 private:
  pybind11::object list_;
  PyObject** items_;
  size_t n_;
};

struct Span {
  uintptr_t lo, hi;
  bool out;
};

// Every value is scaled once, from a gradient that nothing else writes.
void check_apart(const std::vector<Entry>& e, int slots) {
  constexpr int kWidth[3] = {4, 2, 2};
  std::vector<Span> s;
  s.reserve(2 * e.size());
  bool rising = true;      // the outputs in the order of their addresses, and no other gradients: the usual list
  for (size_t i = 0; i < e.size(); ++i) {
    const auto lo = reinterpret_cast<uintptr_t>(e[i].in), to = reinterpret_cast<uintptr_t>(e[i].out);
    const size_t n = e[i].n * (size_t)slots;
    const bool same = lo == to && kWidth[e[i].kind] == kWidth[e[i].out_kind];
    if (!same || (!s.empty() && s.back().hi > to)) rising = false;
    s.push_back({to, to + n * kWidth[e[i].out_kind], true});
    if (!same) s.push_back({lo, lo + n * kWidth[e[i].kind], false});
  }
  if (rising) return;
  std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t out_end = 0, any_end = 0;     // where the outputs, and all, that began so far end
  for (const Span& v : s) {
    TORCH_CHECK_VALUE(v.lo >= (v.out ? any_end : out_end),
                      "clip_grad_norm: an output shares memory with another output or with a gradient that is not its own");
    any_end = std::max(any_end, v.hi);
    if (v.out) out_end = std::max(out_end, v.hi);
  }
}

constexpr int kFew = 48, kMany = 640;   // tensors of a launch: parameters of 2 KB, or of 30 KB

template <int N>
void fill(Table<N>& t, const std::vector<Entry>& all, size_t from, int slots, int per_slot, long chunk) {
  t.count = (int)std::min<size_t>(N, all.size() - from);
  t.slots = slots, t.per_slot = per_slot, t.chunk = chunk, t.total = 0;
  for (int i = 0; i < t.count; ++i) {
    t.e[i] = all[from + i];
    t.e[i].first = t.total;
    t.total += slots * t.e[i].chunks;
  }
}

template <int N>
void run_small(const std::vector<Entry>& all, int slots, int per_slot, long chunk, const Bound& bound, cudaStream_t stream) {
  Table<N> t;
  fill(t, all, 0, slots, per_slot, chunk);
  small_kernel<N><<<kSmallBlocks, 32 * kSmallWarps, 0, stream>>>(t, bound);
  BB_POST_LAUNCH();
}

template <int N>
void run(const std::vector<Entry>& all, int slots, int per_slot, long chunk, double* parts, const Factor* factor,
         cudaStream_t stream) {
  // (the scaling takes the lists backwards too)
  const size_t lists = (all.size() + N - 1) / N;
  for (size_t l = 0; l < lists; ++l) {
    Table<N> t;
    fill(t, all, (factor ? lists - 1 - l : l) * N, slots, per_slot, chunk);
    if (factor) scale_kernel<N><<<t.total, kThreads, 0, stream>>>(t, factor);
    else sums_kernel<N><<<t.total, kThreads, 0, stream>>>(t, parts);
    BB_POST_LAUNCH();
  }
}

}  // namespace

// Norms [slots] ([] without `per_slot`) of the gradients over `grad_scale`; with `clip`,
// out (or the gradients themselves) = gradient * min(1, max_norm / (norm + 1e-6)) / grad_scale.
torch::Tensor clip_grad_norm(const pybind11::object& grad_list, bool per_slot, double grad_scale, bool clip,
                             double max_norm, OptTensor max_norms, const pybind11::object& out_list) {
  const Tensors grads(grad_list), out(out_list);
  TORCH_CHECK_VALUE(!grads.empty(), "clip_grad_norm: no gradients");
  const auto device = grads[0].device();
  TORCH_CHECK(device.is_cuda(), "clip_grad_norm: CUDA tensors");
  const int64_t slots = per_slot ? (grads[0].dim() ? grads[0].size(0) : 0) : 1;
  TORCH_CHECK_VALUE(!per_slot || (slots >= 1 && slots < (1 << 16)), "clip_grad_norm: per_slot needs gradients stacked by slot");
  const bool in_place = out.empty();
  TORCH_CHECK_VALUE(in_place || out.size() == grads.size(), "clip_grad_norm: one output per gradient");
  const bool watched = at::GradMode::is_enabled(), inference = c10::InferenceMode::is_enabled();
  const c10::cuda::CUDAGuard guard(device);
  int64_t total = 0, bytes = 0;
  for (size_t i = 0; i < grads.size(); ++i) total += grads[i].numel(), bytes += grads[i].numel() * grads[i].element_size();
  const bool small = bytes <= (1 << 20) && slots <= kSmallSlots && grads.size() <= kMany;
  // (1 MB in 16 tensors: 10.8 us in one launch, 7.8 on the device in three, which take the host 14 us longer; twice as
  // much: 17 and 8.9)
  // chunks of 64 KB of FP32; of 8 KB where all together are too few for the SMs; of a warp's 4 KB
  const long chunk = small ? 1024 : total > (1 << 24) ? 16384 : 2048;
  std::vector<Entry> all;
  all.reserve(grads.size());
  int64_t per = 0, blocks = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    const auto& g = grads[i];
    const auto& o = in_place ? g : out[i];
    TORCH_CHECK_TYPE(g.device() == device, "clip_grad_norm: gradients are on ", device, " and ", g.device());
    TORCH_CHECK(!watched || !(g.requires_grad() || (clip && o.requires_grad())),
                "clip_grad_norm: norms and clipped gradients are not differentiable; detach the tensors");
    TORCH_CHECK(!clip || inference || !o.is_inference(),
                "clip_grad_norm: inference tensors are overwritten in inference mode only");
    Entry e{};
    e.kind = kind_of(g);
    const bool dense = per_slot ? g.is_contiguous() : (g.is_contiguous() || g.is_non_overlapping_and_dense());
    TORCH_CHECK_VALUE(dense, "clip_grad_norm: a gradient has to be dense (and contiguous where norms go by slot)");
    TORCH_CHECK_VALUE(!per_slot || (g.dim() && g.size(0) == slots), "clip_grad_norm: gradients are stacks of ",
                      std::to_string(slots), " slots, got one of ", g.dim() ? std::to_string(g.size(0)) : "none");
    if (clip && !in_place) {
      TORCH_CHECK_TYPE(o.device() == device && (o.scalar_type() == g.scalar_type() || o.scalar_type() == at::kFloat),
                       "clip_grad_norm: an output is float32 or its gradient's type, on its device");
      const bool alike = o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous());
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && alike,
                        "clip_grad_norm: an output has its gradient's sizes and strides");
    }
    if (g.numel() == 0) continue;
    e.in = g.data_ptr();
    e.out = o.data_ptr();
    e.out_kind = in_place ? e.kind : kind_of(o);
    e.n = g.numel() / slots;
    e.chunks = (int)((e.n + chunk - 1) / chunk);
    e.at = (int)per;
    per += e.chunks;
    blocks += slots * e.chunks;
    all.push_back(e);
  }
  TORCH_CHECK_VALUE(blocks < (1ll << 31), "clip_grad_norm: too many values");
  if (clip) check_apart(all, (int)slots);
  TORCH_CHECK_VALUE(!max_norms.has_value() ||
                        (max_norms->device() == device && max_norms->scalar_type() == at::kFloat &&
                         max_norms->is_contiguous() && max_norms->numel() == slots),
                    "clip_grad_norm: max_norm is a number or float32, one per slot, on the gradients' device");
  const auto f32 = at::TensorOptions().device(device).dtype(at::kFloat);
  auto norm = per_slot ? at::empty({slots}, f32) : at::empty({}, f32);
  const auto stream = at::cuda::getCurrentCUDAStream();
  const bool few = all.size() <= kFew;
  const Bound bound{grad_scale, max_norm, max_norms.has_value() ? max_norms->data_ptr<float>() : nullptr,
                    norm.data_ptr<float>(), clip};
  if (small) {
    if (few) run_small<kFew>(all, (int)slots, (int)per, chunk, bound, stream);
    else run_small<kMany>(all, (int)slots, (int)per, chunk, bound, stream);
  } else {
    auto parts = at::empty({slots * per + slots}, f32.dtype(at::kDouble));     // sums, then factors
    double* sums = parts.data_ptr<double>();
    auto* factor = reinterpret_cast<Factor*>(sums + slots * per);
    if (few) run<kFew>(all, (int)slots, (int)per, chunk, sums, nullptr, stream);
    else run<kMany>(all, (int)slots, (int)per, chunk, sums, nullptr, stream);
    finish_kernel<<<(int)slots, 1024, 0, stream>>>(sums, (int)per, bound, factor);
    BB_POST_LAUNCH();
    if (clip) {
      if (few) run<kFew>(all, (int)slots, (int)per, chunk, nullptr, factor, stream);
      else run<kMany>(all, (int)slots, (int)per, chunk, nullptr, factor, stream);
    }
  }
  const Tensors& changed = in_place ? grads : out;
  for (size_t i = 0; clip && i < changed.size(); ++i)
    if (!changed[i].is_inference()) changed[i].unsafeGetTensorImpl()->bump_version();   // (those have no version)
  return norm;
}
