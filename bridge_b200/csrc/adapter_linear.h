// Launchers of the adapter kernels (adapter_linear.cu); checked and called by adapter_ops.cpp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace bb {

constexpr int kMaxAdapterRank = 128;

// Where the rows of a batch find their adapter: device pointers into one int32 buffer that adapter_rows() lays out.
struct AdapterPlan {
  const int* row_slot;     // [T] slot, or -1
  const int* tile_start;   // [ceil(T / 256) + 1] first pair of each tile of 256 rows
  const int* pairs;        // [P][12] (slot, 0, 0, 0, 256 bits: set where a row of the tile is NOT the slot's)
  const int* unit_start;   // [2 ceil(T / 256) + 1] first unit of each tile of 128 rows
  const int* units;        // [.][8] (tile of 128 rows, slot, 0, 0, 128 bits as above): every pair by itself
  const int* block_start;  // [slots + 1] first block of each slot
  const int* blocks;       // [.][4] (first row, rows <= 64, slot, 0), slot by slot and in row order
  int num_units, num_blocks;
  int slots;               // slots the plan speaks of: the largest one + 1
};

// u[t, r] = scale_s sum_k x[t, k] op_s[r, k] for the row's slot s (rows without one are left as they are), and
// y[t, n] = sum_k x[t, k] w[n, k] + sum_r u[t, r] low_s[n, r].  With `mn` the same from transposed operands: du, dx.
struct AdapterProduct {
  const void* x;           // [T, K], row stride ldx
  const void* op;          // [S, R, K], or [S, K, R] with `mn`
  const void* w;           // [N, K], or [K, N]; row stride ldw
  const void* low;         // [S, N, R], or [S, R, N]
  void *u, *y;             // [T, R] (with keep_u [2, T, R]: and what u's rounding left, rounded too), [T, N]
  void* workspace;
  const float* scales;     // [S], or null: `scale`
  float scale;
  long ldx, ldw;
  int T, K, N, S, R;
  bool mn, half, keep_u;   // half: FP16, else BF16; keep_u: u is asked for, beside y
  AdapterPlan plan;
};

struct AdapterNeeds {
  bool u;                  // has to be there
  size_t workspace;        // bytes
};

// db[s, n, r] = sum_t dy[t, n] u[t, r],  da[s, r, k] = sum_t du[t, r] x[t, k] over the rows of slot s
struct AdapterGrads {
  const void *x, *dy;      // [T, K], [T, N]
  const void *u, *du;      // [2, T, R], as above
  void *da, *db;           // null: not asked for
  bool add_a, add_b;       // FP32, added to; else the inputs' type, written
  long ldx, lddy;
  int T, K, N, S, R;
  bool half;
  AdapterPlan plan;
};

cudaError_t launch_adapter_shrink(const AdapterProduct& a, cudaStream_t stream);      // u alone
AdapterNeeds adapter_product_needs(const AdapterProduct& a);
cudaError_t launch_adapter_product(const AdapterProduct& a, cudaStream_t stream);
cudaError_t launch_adapter_grads(const AdapterGrads& a, cudaStream_t stream);
int adapter_error_code();

}  // namespace bb
