// The few-token MoE layer on CUDA cores: fp32, and 16-bit operands whose sizes, strides or alignment the streaming kernels
// (few_token.cu) cannot address. Three launches: up-projection + activation into fp32 hidden rows, down-projection into fp32 rows per
// slot, gate-weighted sum. Everything between the operands and the result stays in fp32, and every sum has a fixed order.
//
// Bound by the weights of the experts that occur, read once per job of up to 8 slots. Weights with contiguous inputs: a warp
// owns 4 weight rows and its lanes stride over K (4 x 8 partial sums per lane, one transposing reduction at the end).
// Any other strides: a lane owns a weight column, the warps of a block split K.
#include <cooperative_groups.h>

#include "act_math.cuh"
#include "few_token.cuh"

namespace smoe {
namespace ft {

constexpr int SIMT_NT = 8;
constexpr int SIMT_THREADS = 256;
constexpr int COL_CHUNK = 256;     // K elements of the inputs staged at a time by the column kernel

struct SimtParams {
  Args a;
  float* hidden;      // (R, F)
  float* per_slot;    // (R, d_out)
};

template <int ACT>
__device__ __forceinline__ float act_exact(float x) { return act_fwd<ACT, false>(x); }

// hidden value from the up-projection's one or two columns (biases added), see act_math.cuh for the layouts
__device__ __forceinline__ float hidden_value(int layout, int act, float alpha, float limit, float c0, float c1) {
  if (layout == LAYOUT_GPT_OSS) {
    const float g = min_nan(c0, limit), u = min_nan(max_nan(c1, -limit), limit);
    return (u + 1.0f) * (g * sigmoidf_<false>(alpha * g));
  }
  const float gate = layout == LAYOUT_GLU_SECOND ? c1 : c0;
  const float lin = layout == LAYOUT_PLAIN ? 1.0f : (layout == LAYOUT_GLU_SECOND ? c0 : c1);
  float r;
  SMOE_ACT_SWITCH(act, r = act_exact<ACT_>(gate);)
  return r * lin;
}

// columns of the up-projection that make hidden value p
__device__ __forceinline__ int up_column(int layout, int F, int p, int half) {
  if (layout == LAYOUT_PLAIN) return p;
  if (layout == LAYOUT_GPT_OSS) return 2 * p + half;
  return half * F + p;
}

template <bool UP, typename T>
__device__ __forceinline__ void emit(const SimtParams& q, int e, int slot, int p, float c0, float c1) {
  const Args& a = q.a;
  if (UP) {
    if (a.B1) {
      const T* b = static_cast<const T*>(a.B1) + e * a.sb1e;
      c0 += to_f32<T>(b[up_column(a.act_layout, a.F, p, 0) * a.sb1n]);
      if (a.act_layout != LAYOUT_PLAIN) c1 += to_f32<T>(b[up_column(a.act_layout, a.F, p, 1) * a.sb1n]);
    }
    q.hidden[static_cast<int64_t>(slot) * a.F + p] = hidden_value(a.act_layout, a.act, a.alpha, a.limit, c0, c1);
  } else {
    q.per_slot[static_cast<int64_t>(slot) * a.d_out + p] = c0;
  }
}

// V consecutive values as floats; V == 1 or one 16-byte load
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&out)[V]) {
  if (V == 1) {
    out[0] = to_f32<T>(__ldg(p));
  } else {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32<T>(t[i]);
  }
}
template <int V>
__device__ __forceinline__ void load_f(const float* p, float (&out)[V]) {
  if (V == 1) {
    out[0] = p[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      out[i] = f.x; out[i + 1] = f.y; out[i + 2] = f.z; out[i + 3] = f.w;
    }
  }
}

// K-contiguous weights. A warp's item is (job, 4 weight rows): 4 hidden values (plain) or 2 pairs of columns (gated), or 4
// output columns of the down-projection.
template <typename T, bool UP, int V>
__global__ void __launch_bounds__(SIMT_THREADS)
ft_rows_kernel(const SimtParams q) {
  extern __shared__ __align__(16) uint8_t scratch[];
  __shared__ Plan plan;
  const Args& a = q.a;
  make_plan(&plan, scratch, a.ids, a.sit, a.sik, a.T, a.k, a.E, SIMT_NT);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = UP ? a.d : a.F, width = UP ? a.F : a.d_out;
  const bool pairs = UP && a.act_layout != LAYOUT_PLAIN;
  const int per = pairs ? 2 : 4;
  const int blocks = (width + per - 1) / per;
  const int64_t total = static_cast<int64_t>(plan.jobs) * blocks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (SIMT_THREADS / 32);
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (SIMT_THREADS / 32) + warp; it < total; it += step) {
    const int job = static_cast<int>(it / blocks), p0 = static_cast<int>(it % blocks) * per;
    const int e = plan.job_expert[job], beg = plan.job_begin[job], n = plan.job_count[job];
    const T* w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = min(p0 + (pairs ? (i & 1) : i), width - 1);
      const int64_t col = UP ? up_column(a.act_layout, a.F, p, pairs ? i >> 1 : 0) : p;
      w[i] = (UP ? static_cast<const T*>(a.W1) + e * a.s1e + col * a.s1n : static_cast<const T*>(a.W2) + e * a.s2e + col * a.s2n);
    }
    const T* xt[SIMT_NT];
    const float* xf[SIMT_NT];
#pragma unroll
    for (int j = 0; j < SIMT_NT; ++j) {
      const int slot = plan.slots[beg + min(j, n - 1)];
      if (UP) xt[j] = static_cast<const T*>(a.X) + static_cast<int64_t>(slot / a.k) * a.sxm;
      else xf[j] = q.hidden + static_cast<int64_t>(slot) * a.F;
    }
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
    // V > 1 only when K is a multiple of V
    for (int kk = lane * V; kk < K; kk += 32 * V) {
      float wv[4][V];
#pragma unroll
      for (int i = 0; i < 4; ++i) load_v<T, V>(w[i] + kk, wv[i]);
#pragma unroll
      for (int j = 0; j < SIMT_NT; ++j) {
        if (j < n) {
          float xv[V];
          if (UP) load_v<T, V>(xt[j] + kk, xv); else load_f<V>(xf[j] + kk, xv);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < V; ++c) acc[i * 8 + j] = fmaf(wv[i][c], xv[c], acc[i * 8 + j]);
        }
      }
    }
    const float sum = transpose_reduce(acc, lane);
    const float other = __shfl_down_sync(0xffffffffu, sum, 16);      // the pair's second column (gated layouts)
    const int row = lane >> 3, j = lane & 7;
    if (j < n && (!pairs || row < 2)) {
      const int p = p0 + row;
      if (p < width) emit<UP, T>(q, e, plan.slots[beg + j], p, sum, other);
    }
  }
}

// Any strides (meant for weights with contiguous outputs). A block's item is (job, 32 hidden values or output columns); lane =
// column, the 8 warps split every staged chunk of K.
template <typename T, bool UP>
__global__ void __launch_bounds__(SIMT_THREADS)
ft_cols_kernel(const SimtParams q) {
  // the staged inputs and the reduction reuse the plan's scratch
  constexpr int XS_BYTES = SIMT_NT * COL_CHUNK * 4, RED_BYTES = 8 * 2 * SIMT_NT * 33 * 4;
  static_assert(XS_BYTES + RED_BYTES >= PLAN_WARPS * MAX_E * 2 + MAX_E * 4 + 16, "the plan's scratch does not fit");
  __shared__ __align__(16) uint8_t pool[XS_BYTES + RED_BYTES];
  __shared__ Plan plan;
  float (*xs)[COL_CHUNK] = reinterpret_cast<float (*)[COL_CHUNK]>(pool);
  float (*red)[2 * SIMT_NT][33] = reinterpret_cast<float (*)[2 * SIMT_NT][33]>(pool + XS_BYTES);
  const Args& a = q.a;
  make_plan(&plan, pool, a.ids, a.sit, a.sik, a.T, a.k, a.E, SIMT_NT);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = UP ? a.d : a.F, width = UP ? a.F : a.d_out;
  const bool pairs = UP && a.act_layout != LAYOUT_PLAIN;
  const int blocks = (width + 31) / 32;
  const int64_t total = static_cast<int64_t>(plan.jobs) * blocks;
  const int64_t swk = UP ? a.s1k : a.s2k, swn = UP ? a.s1n : a.s2n;
  for (int64_t it = blockIdx.x; it < total; it += gridDim.x) {
    const int job = static_cast<int>(it / blocks), p0 = static_cast<int>(it % blocks) * 32;
    const int e = plan.job_expert[job], beg = plan.job_begin[job], n = plan.job_count[job];
    const int p = min(p0 + lane, width - 1);
    const T* base = UP ? static_cast<const T*>(a.W1) + e * a.s1e : static_cast<const T*>(a.W2) + e * a.s2e;
    const T* w0 = base + static_cast<int64_t>(UP ? up_column(a.act_layout, a.F, p, 0) : p) * swn;
    const T* w1 = pairs ? base + static_cast<int64_t>(up_column(a.act_layout, a.F, p, 1)) * swn : w0;
    float acc0[SIMT_NT], acc1[SIMT_NT];
#pragma unroll
    for (int j = 0; j < SIMT_NT; ++j) acc0[j] = acc1[j] = 0.f;
    for (int k0 = 0; k0 < K; k0 += COL_CHUNK) {
      const int len = min(COL_CHUNK, K - k0);
      __syncthreads();
      for (int i = threadIdx.x; i < n * COL_CHUNK; i += SIMT_THREADS) {
        const int j = i / COL_CHUNK, c = i % COL_CHUNK, slot = plan.slots[beg + j];
        float v = 0.f;
        if (c < len)
          v = UP ? to_f32<T>(static_cast<const T*>(a.X)[static_cast<int64_t>(slot / a.k) * a.sxm + k0 + c])
                 : q.hidden[static_cast<int64_t>(slot) * a.F + k0 + c];
        xs[j][c] = v;
      }
      __syncthreads();
      const int c_end = min(len, (warp + 1) * (COL_CHUNK / 8));
      for (int c = warp * (COL_CHUNK / 8); c < c_end; ++c) {
        const float a0 = to_f32<T>(__ldg(w0 + (k0 + c) * swk));
        const float a1 = pairs ? to_f32<T>(__ldg(w1 + (k0 + c) * swk)) : 0.f;
#pragma unroll
        for (int j = 0; j < SIMT_NT; ++j)
          if (j < n) {
            acc0[j] = fmaf(a0, xs[j][c], acc0[j]);
            if (pairs) acc1[j] = fmaf(a1, xs[j][c], acc1[j]);
          }
      }
    }
#pragma unroll
    for (int j = 0; j < SIMT_NT; ++j) {
      red[warp][j][lane] = acc0[j];
      red[warp][SIMT_NT + j][lane] = acc1[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * 32; i += SIMT_THREADS) {
      const int j = i >> 5, c = i & 31;
      float c0 = 0.f, c1 = 0.f;
#pragma unroll
      for (int w8 = 0; w8 < 8; ++w8) {
        c0 += red[w8][j][c];
        c1 += red[w8][SIMT_NT + j][c];
      }
      if (p0 + c < width) emit<UP, T>(q, e, plan.slots[beg + j], p0 + c, c0, c1);
    }
    __syncthreads();
  }
}

// y[t, n] = sum_j gate (per_slot[t k + j, n] + b2[e, n]); slots without an expert add nothing
template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS)
ft_sum_kernel(const SimtParams q) {
  const Args& a = q.a;
  const int t = blockIdx.y, n = blockIdx.x * SIMT_THREADS + threadIdx.x;
  if (n >= a.d_out) return;
  float y = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int64_t e = a.ids[t * a.sit + j * a.sik];
    if (e < 0 || e >= a.E) continue;
    float v = q.per_slot[(static_cast<int64_t>(t) * a.k + j) * a.d_out + n];
    if (a.B2) v += to_f32<T>(static_cast<const T*>(a.B2)[e * a.sb2e + n * a.sb2n]);
    y += a.gates ? load_any(a.gates, t * a.sgt + j * a.sgk, a.gates_dtype) * v : v;
  }
  static_cast<T*>(a.Y)[t * a.sym + n] = from_f32<T>(y);
}

size_t simt_workspace_bytes(int64_t T, int k, int F, int d_out) {
  const size_t hidden = (static_cast<size_t>(T) * k * F * 4 + 255) / 256 * 256;
  return hidden + static_cast<size_t>(T) * k * d_out * 4;
}

static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, bool UP>
static int launch_linear(const SimtParams& q, int sm_count) {
  constexpr int V = 16 / sizeof(T);
  const Args& a = q.a;
  const int64_t swk = UP ? a.s1k : a.s2k, swn = UP ? a.s1n : a.s2n, swe = UP ? a.s1e : a.s2e;
  const int K = UP ? a.d : a.F;
  const void* W = UP ? a.W1 : a.W2;
  const int scratch = plan_scratch_bytes(a.E);
  const int grid = sm_count * 4;
  if (swk == 1) {
    const bool vec = K % V == 0 && swn % V == 0 && swe % V == 0 && al16(W) && (!UP || (al16(a.X) && a.sxm % V == 0));
    if (vec) ft_rows_kernel<T, UP, V><<<grid, SIMT_THREADS, scratch, a.stream>>>(q);
    else ft_rows_kernel<T, UP, 1><<<grid, SIMT_THREADS, scratch, a.stream>>>(q);
  } else {
    ft_cols_kernel<T, UP><<<grid, SIMT_THREADS, 0, a.stream>>>(q);
  }
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

template <typename T>
static int launch_typed(const SimtParams& q, int sm_count) {
  const Args& a = q.a;
  if (int rc = launch_linear<T, true>(q, sm_count)) return rc;
  if (int rc = launch_linear<T, false>(q, sm_count)) return rc;
  dim3 grid(static_cast<unsigned>(cdiv(a.d_out, SIMT_THREADS)), static_cast<unsigned>(a.T));
  ft_sum_kernel<T><<<grid, SIMT_THREADS, 0, a.stream>>>(q);
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

int launch_simt(const Args& a) {
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  SimtParams q;
  q.a = a;
  q.hidden = static_cast<float*>(a.ws);
  q.per_slot = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + (static_cast<size_t>(a.T) * a.k * a.F * 4 + 255) / 256 * 256);
  switch (a.dtype) {
    case SMOE_F32: return launch_typed<float>(q, di.sm_count);
    case SMOE_BF16: return launch_typed<__nv_bfloat16>(q, di.sm_count);
    default: return launch_typed<__half>(q, di.sm_count);
  }
}

// ---- router --------------------------------------------------------------------------------------------
// A cluster of up to 8 blocks per token: logits z_e = <x, Wr[e]> + br[e] in fp32, a warp per expert, gathered in the first block's shared
// memory, which ranks them and makes the gates. Order: larger logit first, equal logits by lower expert
// id, a NaN counts as the largest. Bound by latency: one block per token read the router's 0.5 MB (128 experts of 2048) in 25 us.
constexpr int ROUTE_THREADS = 512;
constexpr int ROUTE_CLUSTER = 8;

struct RouteParams {
  const void* X; int64_t sxm;
  const void* Wr; int64_t swm;
  const void* br; int64_t sbn;
  int64_t* ids; float* gates;
  int E, d, k, mode, renorm;
};

// whether logit v of expert i goes before logit `best` of expert bi
__device__ __forceinline__ bool beats(float v, int i, float best, int bi) {
  const bool vn = v != v, bn = best != best;
  if (vn != bn) return vn;
  if (vn || v == best) return i < bi;
  return v > best;
}

template <typename T, int V>
__global__ void __launch_bounds__(ROUTE_THREADS)
ft_route_kernel(const RouteParams p) {
  __shared__ float z[MAX_E];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the layer's kernels may take their places
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int t = blockIdx.x / parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* z0 = cluster.map_shared_rank(z, 0);
  const T* x = static_cast<const T*>(p.X) + static_cast<int64_t>(t) * p.sxm;
  cluster.sync();            // the first block runs before its memory is written
  for (int e = part * (ROUTE_THREADS / 32) + warp; e < p.E; e += parts * (ROUTE_THREADS / 32)) {
    const T* w = static_cast<const T*>(p.Wr) + static_cast<int64_t>(e) * p.swm;
    float acc = 0.f;
#pragma unroll 4
    for (int kk = lane * V; kk < p.d; kk += 32 * V) {
      float a[V], b[V];
      load_v<T, V>(x + kk, a);
      load_v<T, V>(w + kk, b);
#pragma unroll
      for (int c = 0; c < V; ++c) acc = fmaf(a[c], b[c], acc);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) z0[e] = acc + (p.br ? to_f32<T>(static_cast<const T*>(p.br)[e * p.sbn]) : 0.f);
  }
  cluster.sync();
  if (part != 0) return;
  // An expert's place is the number of experts that beat it: every thread counts for its own, all at once (k rounds of a
  // maximum over one warp took 2 us).
  __shared__ float chosen[32];
  __shared__ int chosen_id[32];
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS) {
    const float mine = z[e];
    int place = 0;
    for (int o = 0; o < p.E; ++o) place += beats(z[o], o, mine, e) && o != e;
    if (place < p.k) { chosen[place] = mine; chosen_id[place] = e; }
  }
  __syncthreads();
  if (warp != 0) return;
  const bool sel = lane < p.k;
  const float mine = sel ? chosen[lane] : 0.f, top = chosen[0];       // the largest of all logits
  const float g = sel ? expf(mine - top) : 0.f;
  float total = 0.f;
  if (p.mode == 0 && !p.renorm) {          // softmax over all experts
    for (int e = lane; e < p.E; e += 32) total += expf(z[e] - top);
  } else {
    total = g;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (sel) {
    p.ids[static_cast<int64_t>(t) * p.k + lane] = chosen_id[lane];
    p.gates[static_cast<int64_t>(t) * p.k + lane] = g / total;
  }
}

template <typename T>
static int launch_route(const RouteParams& p, int T_, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.d % V == 0 && p.sxm % V == 0 && p.swm % V == 0 && al16(p.X) && al16(p.Wr);
  int parts = 1;
  while (parts < ROUTE_CLUSTER && parts * (ROUTE_THREADS / 32) < p.E) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(T_ * parts));
  cfg.blockDim = dim3(ROUTE_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (vec) SMOE_CUDA(cudaLaunchKernelEx(&cfg, ft_route_kernel<T, V>, p));
  else SMOE_CUDA(cudaLaunchKernelEx(&cfg, ft_route_kernel<T, 1>, p));
  return SMOE_OK;
}

}  // namespace ft
}  // namespace smoe

using namespace smoe;

extern "C" int32_t smoe_few_token_max_tokens(void) { return ft::MAX_T; }

extern "C" size_t smoe_few_token_workspace_bytes(int64_t T, int32_t k, int32_t F, int32_t d_out) {
  if (T < 0 || k < 1 || F < 1 || d_out < 1) return 0;
  const size_t a = ft::simt_workspace_bytes(T, k, F, d_out), b = ft::stream_workspace_bytes(T, k, F, d_out);
  return a > b ? a : b;
}

extern "C" int smoe_few_token_route(const void* X, int64_t T, int64_t stride_xm, const void* Wr, int64_t stride_wm,
                                    const void* br, int64_t stride_bn, int32_t E, int32_t d, int32_t k, int32_t mode,
                                    int32_t renormalize, int64_t* expert_idxs, float* gates, int32_t dtype, void* stream) {
  SMOE_CHECK_ARG(dtype == SMOE_F32 || dtype == SMOE_BF16 || dtype == SMOE_F16, "few_token_route: unknown dtype %d", dtype);
  SMOE_CHECK_ARG(T >= 0 && T < (int64_t(1) << 27), "few_token_route: T=%lld out of range", (long long)T);
  SMOE_CHECK_ARG(E >= 1 && E <= ft::MAX_E && d >= 0, "few_token_route: E=%d out of range [1, %d] or d=%d negative", E, ft::MAX_E, d);
  SMOE_CHECK_ARG(k >= 1 && k <= E && k <= 32, "few_token_route: k=%d out of range [1, min(E, 32)]", k);
  SMOE_CHECK_ARG(mode == 0 || mode == 1, "few_token_route: unknown mode %d", mode);
  if (T == 0) return SMOE_OK;
  SMOE_CHECK_ARG(X && Wr && expert_idxs && gates, "few_token_route: null pointer");
  ft::RouteParams p{X, stride_xm, Wr, stride_wm, br, stride_bn, expert_idxs, gates, E, d, k, mode, renormalize ? 1 : 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SMOE_F32: return ft::launch_route<float>(p, static_cast<int>(T), st);
    case SMOE_BF16: return ft::launch_route<__nv_bfloat16>(p, static_cast<int>(T), st);
    default: return ft::launch_route<__half>(p, static_cast<int>(T), st);
  }
}

extern "C" int smoe_few_token_mlp(const void* X, int64_t T, int64_t stride_xm, const void* W1, int64_t stride_w1e,
                                  int64_t stride_w1k, int64_t stride_w1n, const void* b1, int64_t stride_b1e,
                                  int64_t stride_b1n, const void* W2, int64_t stride_w2e, int64_t stride_w2k,
                                  int64_t stride_w2n, const void* b2, int64_t stride_b2e, int64_t stride_b2n,
                                  const void* gates, int64_t stride_gt, int64_t stride_gk, int32_t gates_dtype,
                                  const int64_t* expert_idxs, int64_t stride_it, int64_t stride_ik, void* Y,
                                  int64_t stride_ym, int32_t k, int32_t d, int32_t F, int32_t d_out, int32_t E,
                                  int32_t act_layout, int32_t act, float alpha, float limit, int32_t dtype, int32_t flags,
                                  void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  SMOE_CHECK_ARG(dtype == SMOE_F32 || dtype == SMOE_BF16 || dtype == SMOE_F16, "few_token_mlp: unknown dtype %d", dtype);
  SMOE_CHECK_ARG(gates_dtype >= 0 && gates_dtype <= 2, "few_token_mlp: unknown dtype %d of the gates", gates_dtype);
  SMOE_CHECK_ARG(T >= 0 && T <= ft::MAX_T, "few_token_mlp: %lld tokens, at most %d are taken", (long long)T, ft::MAX_T);
  SMOE_CHECK_ARG(k >= 1 && T * k <= ft::MAX_R, "few_token_mlp: %lld tokens x k=%d slots, at most %d slots are taken", (long long)T,
                 k, ft::MAX_R);
  SMOE_CHECK_ARG(E >= 1 && E <= ft::MAX_E, "few_token_mlp: E=%d out of range [1, %d]", E, ft::MAX_E);
  SMOE_CHECK_ARG(d >= 1 && F >= 1 && d_out >= 1 && F < (1 << 28) && d < (1 << 28) && d_out < (1 << 28),
                 "few_token_mlp: bad sizes d=%d F=%d d_out=%d", d, F, d_out);
  SMOE_CHECK_ARG(act_layout >= 0 && act_layout <= 3 && act >= 0 && act <= 4, "few_token_mlp: layout %d / function %d", act_layout, act);
  if (T == 0) return SMOE_OK;
  SMOE_CHECK_ARG(X && W1 && W2 && expert_idxs && Y, "few_token_mlp: null pointer");
  if (workspace == nullptr || workspace_bytes < smoe_few_token_workspace_bytes(T, k, F, d_out)) {
    set_error("few_token_mlp: workspace of %zu bytes needed, %zu given", smoe_few_token_workspace_bytes(T, k, F, d_out),
              workspace_bytes);
    return SMOE_ERR_WORKSPACE;
  }
  SMOE_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "few_token_mlp: the workspace is not 16-byte aligned");
  ft::Args a{X, T == 1 ? 0 : stride_xm, W1, stride_w1e, stride_w1k, stride_w1n, b1, stride_b1e, stride_b1n,
             W2, stride_w2e, stride_w2k, stride_w2n, b2, stride_b2e, stride_b2n,
             gates, stride_gt, stride_gk, gates_dtype, expert_idxs, stride_it, stride_ik, Y, stride_ym,
             static_cast<int>(T), k, d, F, d_out, E, act_layout, act, dtype, alpha, limit,
             workspace, workspace_bytes, status, (flags & SMOE_FLAG_AFTER_ROUTER) ? 1 : 0, static_cast<cudaStream_t>(stream)};
  if (!(flags & SMOE_FLAG_FORCE_SIMT)) {
    const int rc = ft::launch_stream(a);
    if (rc != SMOE_ERR_UNSUPPORTED) {
      if (rc == SMOE_OK) set_last_path(1);
      return rc;
    }
    if (flags & SMOE_FLAG_FORCE_TC) {
      set_error("few_token_mlp: no tensor-core kernel for this dtype/alignment (dtype=%d d=%d F=%d)", dtype, d, F);
      return rc;
    }
  }
  set_last_path(0);
  return ft::launch_simt(a);
}
