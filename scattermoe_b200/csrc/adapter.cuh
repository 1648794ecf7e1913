// Shared by the kernels of the low-rank adapters beside a shared projection.
//
//   y_t = W x_t + b + B_a h_t,   h_t = s_a A_a x_t,   a = ids[t]      (an id outside [0, n): y_t = W x_t + b)
//
// and its gradients  g_t = s_a B_a^T dy_t;  dx_t = W^T dy_t + A_a^T g_t;  dA_a = sum g_t x_t^T;  dB_a = sum dy_t h_t^T.
// Three products cover both directions: the SHRINK into the rank (h, g), the shared product with the EXPANSION out of the rank
// added while the accumulators are at hand (y, dx), and the per-adapter sum of outer products (dA, dB).
// h and g are rows of the rank padded with zeros to a multiple of 8 (rank_pitch), in the storage type: fp32, or rounded once to the
// 16 bits that the tensor cores multiply (each rounding is at most half a step of a value that adds a correction to the product). CUDA
// cores could do without that rounding. They share the form because the products of a call choose their kernels each for itself (the
// input's width may be odd and the output's not) and backward reads the rows forward wrote; the output's error stays below 1.4 times
// that of rounding it alone.
#pragma once

#include "smoe_common.cuh"

namespace smoe {
namespace ad {

constexpr int MAX_RANK = 256;
constexpr int SM_COUNT = 148;        // of a B200. Grids, and the counts of parts that size a workspace: the size query needs no device and agrees
                                     // with the launch
constexpr int FEW_TOKENS = 128;      // up to here the product is a read of W (few_token.cu)
constexpr int SHRINK_FEW_TOKENS = 256;      // up to here a shrink with contiguous inputs takes a warp per token (adapter.cu)
constexpr int64_t rank_pitch(int r) { return (r + 7) / 8 * 8; }

struct ShrinkArgs {           // H[t, j] = s_a sum_c X[t, c] M[a][j, c]
  const void* X; int64_t T, sxm;
  const void* M; int64_t sma, smj, smc;
  const int64_t* ids;
  const float* scaling; float scale;
  void* H;
  int n, C, r, dtype;
  const int64_t* sorted_idx; const int64_t* offsets;      // the rows sorted by adapter, where the caller has them (nullable)
  cudaStream_t stream;
};

// The launch before on the stream is the shrink that writes H.
struct LinearArgs {           // Y[t, o] = sum_c X[t, c] W[c, o] + bias[o] + sum_j H[t, j] M[a][j, o]
  const void* X; int64_t T, sxm;
  const void* W; int64_t swk, swn;
  const void* bias;
  const void* H;
  const void* M; int64_t sma, smj, smo;
  const int64_t* ids;
  void* Y; int64_t sym;
  int n, C, O, r, dtype;
  int32_t* status;
  cudaStream_t stream;
};

struct GradArgs {             // D[a][j, c] = sum over rows t of adapter a of U[t, j] V[t, c]
  const void* U; int64_t T;
  const void* V; int64_t svm;
  const int64_t* sorted_idx; const int64_t* offsets;
  void* D; int64_t sda, sdj, sdc;
  int n, C, r, dtype;
  void* ws; size_t ws_bytes;
  cudaStream_t stream;
};

// Tensor-core kernels: SMOE_ERR_UNSUPPORTED (no error text) when the operands do not fit them.
int launch_linear_tc(const LinearArgs& a);
int launch_shrink_tc(const ShrinkArgs& a);
int launch_grad_tc(const GradArgs& a);
size_t grad_workspace_bytes(int64_t T, int C, int r);

int launch_shrink_simt(const ShrinkArgs& a);
int launch_linear_simt(const LinearArgs& a);
int launch_grad_simt(const GradArgs& a);

}  // namespace ad
}  // namespace smoe
