// Low-rank adapters on CUDA cores (fp32, and 16-bit operands the tensor-core kernels cannot address), and the C entry points.
#include "adapter.cuh"

#include "act_math.cuh"
#include "few_token.cuh"

namespace smoe {
namespace ad {

// V consecutive values as floats: one 16-byte load, or one value
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&out)[V]) {
  if (V == 1) {
    out[0] = to_f32<T>(__ldg(p));
  } else {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32<T>(t[i]);
  }
}

// ---- shrink: a warp per (token, RW rank rows), lanes over the contracted axis, V values at a time -----------------
template <typename T, int V, int RW>
__global__ void __launch_bounds__(256)
shrink_simt_kernel(const ShrinkArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the linear may start its stream of W
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = static_cast<int>(rank_pitch(a.r) / RW);
  const int64_t total = a.T * blocks;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * 8 + warp; it < total; it += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t t = it / blocks;
    const int j0 = static_cast<int>(it % blocks) * RW;
    const int64_t id = a.ids[t];
    float acc[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) acc[i] = 0.f;
    float s = 0.f;
    if (id >= 0 && id < a.n) {
      s = a.scaling ? a.scaling[id] : a.scale;
      const T* x = static_cast<const T*>(a.X) + t * a.sxm;
      const T* m = static_cast<const T*>(a.M) + id * a.sma;
#pragma unroll (RW == 1 ? 8 : 2)
      for (int c = lane * V; c < a.C; c += 32 * V) {       // V > 1: contiguous and aligned, C a multiple of V
        float xv[V];
        load_values<T, V>(x + c, xv);
#pragma unroll
        for (int i = 0; i < RW; ++i)
          if (j0 + i < a.r) {
            float mv[V];
            load_values<T, V>(m + (j0 + i) * a.smj + c * a.smc, mv);
#pragma unroll
            for (int v = 0; v < V; ++v) acc[i] = fmaf(xv[v], mv[v], acc[i]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      // an adapter that is not there leaves a zero row, whatever the inputs hold; so does the padding
      if (lane == 0) static_cast<T*>(a.H)[t * rank_pitch(a.r) + j0 + i] = from_f32<T>((id >= 0 && id < a.n && j0 + i < a.r) ? acc[i] * s : 0.f);
    }
  }
}

// ---- shared product + expansion: 64 x 64 tiles, 4 x 4 outputs per thread ----------------------------------------
constexpr int TM = 64, TN = 64, TK = 32;      // long steps: with few tiles the kernel is bound by their number

template <typename T>
__global__ void __launch_bounds__(256)
linear_simt_kernel(const LinearArgs a) {
  __shared__ float xs[TK][TM + 4];
  __shared__ float ws[TK][TN + 4];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * TM;
  const int o0 = blockIdx.x * TN;
  const bool k_contig = a.swk == 1;
  float acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  // the next step's values are fetched while this one's are multiplied
  float xn[TM * TK / 256], wn[TN * TK / 256];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < TM * TK / 256; ++i) {
      const int idx = tid + i * 256, kk = idx % TK, m = idx / TK;
      const int64_t t = t0 + m;
      xn[i] = (t < a.T && k0 + kk < a.C) ? to_f32<T>(__ldg(static_cast<const T*>(a.X) + t * a.sxm + k0 + kk)) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < TN * TK / 256; ++i) {
      const int idx = tid + i * 256;
      const int kk = k_contig ? idx % TK : idx / TN, n = k_contig ? idx / TK : idx % TN;
      wn[i] = (o0 + n < a.O && k0 + kk < a.C)
                  ? to_f32<T>(__ldg(static_cast<const T*>(a.W) + (k0 + kk) * a.swk + (o0 + n) * a.swn)) : 0.f;
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < a.C; k0 += TK) {
#pragma unroll
    for (int i = 0; i < TM * TK / 256; ++i) xs[(tid + i * 256) % TK][(tid + i * 256) / TK] = xn[i];
#pragma unroll
    for (int i = 0; i < TN * TK / 256; ++i) {
      const int idx = tid + i * 256;
      ws[k_contig ? idx % TK : idx / TN][k_contig ? idx / TK : idx % TN] = wn[i];
    }
    __syncthreads();
    fetch(k0 + TK);
#pragma unroll
    for (int kk = 0; kk < TK; ++kk) {
      const float4 x4 = *reinterpret_cast<const float4*>(&xs[kk][ty * 4]);
      const float4 w4 = *reinterpret_cast<const float4*>(&ws[kk][tx * 4]);
      const float xv[4] = {x4.x, x4.y, x4.z, x4.w}, wv[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xv[i], wv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty * 4 + i;
    if (t >= a.T) continue;
    const int64_t id = a.ids[t];
    if (id >= 0 && id < a.n) {
      const T* m = static_cast<const T*>(a.M) + id * a.sma;
      const T* h = static_cast<const T*>(a.H) + t * rank_pitch(a.r);
      for (int jj = 0; jj < a.r; ++jj) {
        const float hv = to_f32<T>(h[jj]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int o = o0 + tx * 4 + j;
          if (o < a.O) acc[i][j] = fmaf(hv, to_f32<T>(__ldg(m + jj * a.smj + o * a.smo)), acc[i][j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = o0 + tx * 4 + j;
      if (o >= a.O) continue;
      const float b = a.bias ? to_f32<T>(static_cast<const T*>(a.bias)[o]) : 0.f;
      static_cast<T*>(a.Y)[t * a.sym + o] = from_f32<T>(acc[i][j] + b);
    }
  }
}

// ---- the same for few tokens and a weight with contiguous inputs: a warp per (4 columns, 8 tokens), lanes over the inputs ----
// A tile of 64 x 64 would leave most SMs without one (12 tokens, 3547 x 1161: 255 us in tiles).
template <typename T, int V>
__global__ void __launch_bounds__(256)
linear_rows_simt_kernel(const LinearArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int o0 = (blockIdx.x * 8 + warp) * 4;
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * 8;
  if (o0 >= a.O) return;
  const int n = static_cast<int>(min(static_cast<int64_t>(8), a.T - t0));
  const T* w[4];
  const T* x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = static_cast<const T*>(a.W) + min(o0 + i, a.O - 1) * a.swn;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = static_cast<const T*>(a.X) + (t0 + min(j, n - 1)) * a.sxm;
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
  for (int c = lane * V; c < a.C; c += 32 * V) {       // V > 1: aligned, C a multiple of V
    float wv[4][V];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_values<T, V>(w[i] + c, wv[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) {
        float xv[V];
        load_values<T, V>(x[j] + c, xv);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[i * 8 + j] = fmaf(wv[i][v], xv[v], acc[i * 8 + j]);
      }
  }
  float y = ft::transpose_reduce(acc, lane);            // lane: column lane / 8, token lane % 8
  const int o = o0 + (lane >> 3);
  const int64_t t = t0 + (lane & 7);
  if (o >= a.O || t >= a.T) return;
  const int64_t id = a.ids[t];
  if (id >= 0 && id < a.n) {
    const T* m = static_cast<const T*>(a.M) + id * a.sma + o * a.smo;
    const T* h = static_cast<const T*>(a.H) + t * rank_pitch(a.r);
    for (int j = 0; j < a.r; ++j) y = fmaf(to_f32<T>(h[j]), to_f32<T>(__ldg(m + j * a.smj)), y);
  }
  if (a.bias) y += to_f32<T>(static_cast<const T*>(a.bias)[o]);
  static_cast<T*>(a.Y)[t * a.sym + o] = from_f32<T>(y);
}

// ---- per-adapter outer products: a block per (64 columns, 16 rank rows, adapter), over the adapter's rows in order ----
constexpr int GR_SIMT_ROWS = 128;      // of a step: the kernel is bound by the latency of its steps
template <typename T>
__global__ void __launch_bounds__(256)
grad_simt_kernel(const GradArgs a) {
  __shared__ float us[GR_SIMT_ROWS][17];
  __shared__ float vs[GR_SIMT_ROWS][65];
  __shared__ int64_t rows[GR_SIMT_ROWS];
  const int tid = threadIdx.x, cx = tid & 63, jg = tid >> 6;
  const int c0 = blockIdx.x * 64, j0 = blockIdx.y * 16, e = blockIdx.z;
  const int64_t beg = e ? a.offsets[e - 1] : 0, end = a.offsets[e];
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t m0 = beg; m0 < end; m0 += GR_SIMT_ROWS) {
    const int cnt = static_cast<int>(min(static_cast<int64_t>(GR_SIMT_ROWS), end - m0));
    if (tid < GR_SIMT_ROWS) rows[tid] = tid < cnt ? a.sorted_idx[m0 + tid] : -1;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < GR_SIMT_ROWS * 16 / 256; ++q) {
      const int i = tid + q * 256;
      const int m = i >> 4, j = i & 15;
      us[m][j] = (m < cnt && j0 + j < a.r) ? to_f32<T>(static_cast<const T*>(a.U)[rows[m] * rank_pitch(a.r) + j0 + j]) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < GR_SIMT_ROWS * 64 / 256; ++q) {
      const int i = tid + q * 256;
      const int m = i >> 6, c = i & 63;
      vs[m][c] = (m < cnt && c0 + c < a.C) ? to_f32<T>(__ldg(static_cast<const T*>(a.V) + rows[m] * a.svm + c0 + c)) : 0.f;
    }
    __syncthreads();
    // a sum of its own for every step: one chain over all rows of an adapter would be off by as many roundings as there are rows
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int m = 0; m < cnt; ++m) {
      const float v = vs[m][cx];
#pragma unroll
      for (int i = 0; i < 4; ++i) part[i] = fmaf(us[m][jg * 4 + i], v, part[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += part[i];
    __syncthreads();
  }
  if (c0 + cx >= a.C) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = j0 + jg * 4 + i;
    if (j < a.r) static_cast<T*>(a.D)[e * a.sda + j * a.sdj + (c0 + cx) * a.sdc] = from_f32<T>(acc[i]);
  }
}

#define SMOE_AD_DTYPE(dtype, ...)                                      \
  switch (dtype) {                                                     \
    case SMOE_F32: { using T_ = float; __VA_ARGS__ } break;            \
    case SMOE_BF16: { using T_ = __nv_bfloat16; __VA_ARGS__ } break;   \
    default: { using T_ = __half; __VA_ARGS__ } break;                 \
  }

int launch_shrink_simt(const ShrinkArgs& a) {
  // four rank rows per warp read the token's row a quarter as often; one each where there are too few warps to fill the GPU
  const bool single = a.T * (rank_pitch(a.r) / 4) < SM_COUNT * 16;
  const int64_t warps = a.T * (rank_pitch(a.r) / (single ? 1 : 4));
  const int grid = static_cast<int>(min(cdiv64(warps, 8), static_cast<int64_t>(SM_COUNT * 32)));
  const int v = 16 / dtype_size(a.dtype);
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.smc == 1 && a.C % v == 0 && a.sxm % v == 0 && a.smj % v == 0 && a.sma % v == 0 && al16(a.X) && al16(a.M);
  if (vec && single) SMOE_AD_DTYPE(a.dtype, shrink_simt_kernel<T_, 16 / sizeof(T_), 1><<<grid, 256, 0, a.stream>>>(a);)
  else if (vec) SMOE_AD_DTYPE(a.dtype, shrink_simt_kernel<T_, 16 / sizeof(T_), 4><<<grid, 256, 0, a.stream>>>(a);)
  else SMOE_AD_DTYPE(a.dtype, shrink_simt_kernel<T_, 1, 4><<<grid, 256, 0, a.stream>>>(a);)
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

int launch_linear_simt(const LinearArgs& a) {
  if (a.T <= FEW_TOKENS && a.swk == 1) {
    const int v = 16 / dtype_size(a.dtype);
    auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = a.C % v == 0 && a.sxm % v == 0 && a.swn % v == 0 && al16(a.X) && al16(a.W);
    dim3 grid(static_cast<unsigned>(cdiv(a.O, 32)), static_cast<unsigned>(cdiv64(a.T, 8)));
    if (vec) SMOE_AD_DTYPE(a.dtype, linear_rows_simt_kernel<T_, 16 / sizeof(T_)><<<grid, 256, 0, a.stream>>>(a);)
    else SMOE_AD_DTYPE(a.dtype, linear_rows_simt_kernel<T_, 1><<<grid, 256, 0, a.stream>>>(a);)
    SMOE_LAUNCH_CHECK();
    return SMOE_OK;
  }
  // the token axis in slices of at most 65535 tiles (the grid's second axis)
  const int64_t slice = static_cast<int64_t>(65535) * TM;
  for (int64_t t0 = 0; t0 < a.T; t0 += slice) {
    LinearArgs b = a;
    const int es = dtype_size(a.dtype);
    b.X = static_cast<const uint8_t*>(a.X) + t0 * a.sxm * es;
    b.Y = static_cast<uint8_t*>(a.Y) + t0 * a.sym * es;
    b.H = static_cast<const uint8_t*>(a.H) + t0 * rank_pitch(a.r) * es;
    b.ids = a.ids + t0;
    b.T = a.T - t0 < slice ? a.T - t0 : slice;
    dim3 grid(static_cast<unsigned>(cdiv(a.O, TN)), static_cast<unsigned>(cdiv64(b.T, TM)));
    SMOE_AD_DTYPE(a.dtype, linear_simt_kernel<T_><<<grid, 256, 0, a.stream>>>(b);)
    SMOE_LAUNCH_CHECK();
  }
  return SMOE_OK;
}

int launch_grad_simt(const GradArgs& a) {
  dim3 grid(static_cast<unsigned>(cdiv(a.C, 64)), static_cast<unsigned>(cdiv(a.r, 16)), static_cast<unsigned>(a.n));
  SMOE_AD_DTYPE(a.dtype, grad_simt_kernel<T_><<<grid, 256, 0, a.stream>>>(a);)
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

// Few tokens: the product is a read of W, see few_token.cu.
static int launch_linear_few(const LinearArgs& a) {
  if (a.T > FEW_TOKENS || a.sym != a.O) return SMOE_ERR_UNSUPPORTED;
  ft::Args f = {};
  f.X = a.X; f.sxm = a.sxm;
  f.W1 = a.W; f.s1k = a.swk; f.s1n = a.swn;
  f.B1 = a.bias; f.sb1n = 1;
  f.T = static_cast<int>(a.T); f.k = 1; f.d = a.C; f.F = a.O; f.d_out = a.O; f.E = 1;
  f.act_layout = LAYOUT_PLAIN; f.act = ACT_IDENTITY; f.dtype = a.dtype;
  f.ws = a.Y;
  f.status = a.status;
  f.after_router = 0;
  f.stream = a.stream;
  const bool aligned = (reinterpret_cast<uintptr_t>(a.M) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.H) & 15) == 0;
  ft::Extension x{a.H, rank_pitch(a.r), a.M, a.sma, a.smj, a.smo, a.ids, a.n, a.r,
                  a.smj == 1 && a.smo % 8 == 0 && a.sma % 8 == 0 && a.r % 8 == 0 && aligned ? 1 : 0};
  return ft::launch_linear(f, x);
}

static int check_common(const char* who, int64_t T, int n, int in, int out, int r, int dtype) {
  SMOE_CHECK_ARG(dtype == SMOE_F32 || dtype == SMOE_BF16 || dtype == SMOE_F16, "%s: unknown dtype %d", who, dtype);
  SMOE_CHECK_ARG(T >= 0 && T < (int64_t(1) << 31) - 64, "%s: T=%lld out of range [0, 2^31 - 64)", who, (long long)T);
  SMOE_CHECK_ARG(n >= 1 && n <= 4096, "%s: %d adapters, 1 to 4096 are taken", who, n);
  SMOE_CHECK_ARG(r >= 1 && r <= MAX_RANK, "%s: rank %d, 1 to %d are taken", who, r, MAX_RANK);
  SMOE_CHECK_ARG(in >= 1 && in < (1 << 28) && out >= 1 && out < (1 << 28), "%s: bad widths in=%d out=%d", who, in, out);
  return SMOE_OK;
}

static int refuse_tc(const char* what, int dtype, int C) {
  set_error("adapter_linear: no tensor-core kernel for this dtype/alignment (%s, dtype=%d width=%d)", what, dtype, C);
  return SMOE_ERR_UNSUPPORTED;
}

static int shrink(const ShrinkArgs& a, int flags) {
  // A warp per token and 4 rank rows reads M again for every token, but spreads few tokens over the GPU: the choice for them, not a way
  // out. The whole call, 4096 x 4096, rank 16, bf16: 129 to 256 rows of one adapter 34-35 us against 44-45 on tensor cores, of 8 adapters in
  // no order 41-42 against 146; rank 64, 64 adapters 142-158 against 950 and more.
  const bool few = a.T <= SHRINK_FEW_TOKENS && a.smc == 1;
  if (!(flags & SMOE_FLAG_FORCE_SIMT) && !few) {
    const int rc = launch_shrink_tc(a);
    if (rc != SMOE_ERR_UNSUPPORTED) return rc;
    if (flags & SMOE_FLAG_FORCE_TC) return refuse_tc("shrink", a.dtype, a.C);
  }
  return launch_shrink_simt(a);
}

static int linear(const LinearArgs& a, int flags) {
  if (!(flags & SMOE_FLAG_FORCE_SIMT)) {
    int rc = launch_linear_few(a);
    if (rc == SMOE_ERR_UNSUPPORTED) rc = launch_linear_tc(a);
    if (rc != SMOE_ERR_UNSUPPORTED) {
      if (rc == SMOE_OK) set_last_path(1);
      return rc;
    }
    if (flags & SMOE_FLAG_FORCE_TC) {
      set_error("adapter_linear: no tensor-core kernel for this dtype/alignment (dtype=%d in=%d out=%d)", a.dtype, a.C, a.O);
      return rc;
    }
  }
  set_last_path(0);
  return launch_linear_simt(a);
}

static int outer(const GradArgs& a, int flags) {
  if (!(flags & SMOE_FLAG_FORCE_SIMT)) {
    const int rc = launch_grad_tc(a);
    if (rc != SMOE_ERR_UNSUPPORTED) return rc;
    if (flags & SMOE_FLAG_FORCE_TC) return refuse_tc("outer products", a.dtype, a.C);
  }
  return launch_grad_simt(a);
}

__global__ void set_rows_kernel(int64_t* rows, int64_t T) { *rows = T; }

static size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// ---- column sums (the shared bias's gradient): fp32 partial sums over slices of the rows, added up in order ----
constexpr int SUM_COLS = 256, SUM_MAX_SLICES = 64;

static int sum_slices(int64_t T, int C) {
  const int64_t by_rows = cdiv64(T, 32), by_grid = cdiv64(SM_COUNT * 8, cdiv(C, SUM_COLS));
  const int64_t s = by_rows < by_grid ? by_rows : by_grid;
  return static_cast<int>(s < 1 ? 1 : (s > SUM_MAX_SLICES ? SUM_MAX_SLICES : s));
}

template <typename T>
__global__ void __launch_bounds__(SUM_COLS)
column_partial_kernel(const T* __restrict__ V, int64_t rows, int64_t svm, int C, float* __restrict__ partial) {
  const int c = blockIdx.x * SUM_COLS + threadIdx.x;
  if (c >= C) return;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t beg = min(rows, per * blockIdx.y), end = min(rows, beg + per);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int64_t t = beg;
  for (; t + 8 <= end; t += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += to_f32<T>(__ldg(V + (t + i) * svm + c));
  }
  for (; t < end; ++t) s[0] += to_f32<T>(__ldg(V + t * svm + c));
  partial[static_cast<int64_t>(blockIdx.y) * C + c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

template <typename T>
__global__ void __launch_bounds__(SUM_COLS)
column_total_kernel(const float* __restrict__ partial, int slices, int C, T* __restrict__ out) {
  const int c = blockIdx.x * SUM_COLS + threadIdx.x;
  if (c >= C) return;
  float s = 0.f;
  for (int i = 0; i < slices; ++i) s += partial[static_cast<int64_t>(i) * C + c];
  out[c] = from_f32<T>(s);
}

static size_t column_sum_bytes(int64_t T, int C) { return static_cast<size_t>(sum_slices(T, C)) * C * 4; }

static int column_sum(const void* V, int64_t T, int64_t svm, int C, void* out, int dtype, void* ws, cudaStream_t st) {
  const int slices = sum_slices(T, C);
  float* partial = static_cast<float*>(ws);
  dim3 grid(static_cast<unsigned>(cdiv(C, SUM_COLS)), static_cast<unsigned>(slices));
  SMOE_AD_DTYPE(dtype, column_partial_kernel<T_><<<grid, SUM_COLS, 0, st>>>(static_cast<const T_*>(V), T, svm, C, partial);
                column_total_kernel<T_><<<grid.x, SUM_COLS, 0, st>>>(partial, slices, C, static_cast<T_*>(out));)
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

}  // namespace ad
}  // namespace smoe

using namespace smoe;

// forward: sorted ids and the sort's histograms; backward: g, the outer products' parts, the column sums' parts
extern "C" size_t smoe_adapter_workspace_bytes(int64_t T, int32_t n, int32_t in, int32_t out, int32_t r, int32_t dtype) {
  if (T < 0 || n < 1 || in < 1 || out < 1 || r < 1 || dtype < 0 || dtype > 2) return 0;
  const size_t forward = ad::up256(static_cast<size_t>(T) * 8) + ad::up256(smoe_sort_count_workspace_bytes(T, n));
  size_t parts = ad::grad_workspace_bytes(T, in, r);
  const size_t parts_out = ad::grad_workspace_bytes(T, out, r), sums = ad::column_sum_bytes(T, out);
  parts = parts > parts_out ? parts : parts_out;
  parts = parts > sums ? parts : sums;
  const size_t backward = ad::up256(static_cast<size_t>(T) * ad::rank_pitch(r) * dtype_size(dtype)) + ad::up256(parts);
  return (forward > backward ? forward : backward) + 256;
}

extern "C" int smoe_adapter_forward(const void* X, int64_t T, int64_t stride_xm, const void* W, int64_t stride_wo,
                                    int64_t stride_wi, const void* bias, const void* A, int64_t stride_aa, int64_t stride_aj,
                                    int64_t stride_ai, const void* B, int64_t stride_ba, int64_t stride_bo, int64_t stride_bj,
                                    const int64_t* adapter_idxs, const float* scaling, float scale, void* Y, void* H,
                                    int64_t* sorted_idx, int64_t* offsets, int32_t n, int32_t in, int32_t out, int32_t r,
                                    int32_t dtype, int32_t flags, void* workspace, size_t workspace_bytes, int32_t* status,
                                    void* stream) {
  const char* who = "adapter_forward";
  if (int rc = ad::check_common(who, T, n, in, out, r, dtype)) return rc;
  SMOE_CHECK_ARG((sorted_idx == nullptr) == (offsets == nullptr), "%s: sorted_idx and offsets go together", who);
  if (T > 0) SMOE_CHECK_ARG(X && W && A && B && adapter_idxs && Y && H, "%s: null pointer", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (offsets) {
    const size_t need = smoe_adapter_workspace_bytes(T, n, in, out, r, dtype);
    if (workspace == nullptr || workspace_bytes < need) {
      set_error("%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
      return SMOE_ERR_WORKSPACE;
    }
    int64_t* sorted_ids = static_cast<int64_t*>(workspace);
    uint8_t* rest = static_cast<uint8_t*>(workspace) + ad::up256(static_cast<size_t>(T) * 8);
    if (int rc = smoe_sort_count(adapter_idxs, T, n, sorted_ids, sorted_idx, offsets, rest, smoe_sort_count_workspace_bytes(T, n), stream))
      return rc;
  }
  if (T == 0) return SMOE_OK;
  ad::ShrinkArgs s{X, T, stride_xm, A, stride_aa, stride_aj, stride_ai, adapter_idxs, scaling, scale, H, n, in, r, dtype, sorted_idx, offsets, st};
  if (int rc = ad::shrink(s, flags)) return rc;
  ad::LinearArgs l{X, T, stride_xm, W, stride_wi, stride_wo, bias, H, B, stride_ba, stride_bj, stride_bo, adapter_idxs, Y,
                   out, n, in, out, r, dtype, status, st};
  return ad::linear(l, flags);
}

extern "C" int smoe_adapter_backward(const void* DY, int64_t T, int64_t stride_dym, const void* X, int64_t stride_xm, const void* W,
                                     int64_t stride_wo, int64_t stride_wi, const void* A, int64_t stride_aa, int64_t stride_aj,
                                     int64_t stride_ai, const void* B, int64_t stride_ba, int64_t stride_bo, int64_t stride_bj,
                                     const int64_t* adapter_idxs, const float* scaling, float scale, const void* H,
                                     const int64_t* sorted_idx, const int64_t* offsets, void* DX, void* DA, void* DB,
                                     void* DW, void* Dbias, int32_t n, int32_t in, int32_t out, int32_t r, int32_t dtype, int32_t flags,
                                     void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  const char* who = "adapter_backward";
  if (int rc = ad::check_common(who, T, n, in, out, r, dtype)) return rc;
  const size_t need = smoe_adapter_workspace_bytes(T, n, in, out, r, dtype);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
    return SMOE_ERR_WORKSPACE;
  }
  SMOE_CHECK_ARG((!DA && !DB) || (offsets && (T == 0 || sorted_idx)), "%s: the adapters' gradients need the sorted rows", who);
  if (T > 0) SMOE_CHECK_ARG(DY && X && W && A && B && adapter_idxs && H, "%s: null pointer", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* G = workspace;
  uint8_t* parts = static_cast<uint8_t*>(workspace) + ad::up256(static_cast<size_t>(T) * ad::rank_pitch(r) * dtype_size(dtype));
  const size_t parts_bytes = workspace_bytes - (parts - static_cast<uint8_t*>(workspace));
  if (T > 0 && (DX || DA)) {
    ad::ShrinkArgs s{DY, T, stride_dym, B, stride_ba, stride_bj, stride_bo, adapter_idxs, scaling, scale, G, n, out, r, dtype, sorted_idx, offsets, st};
    if (int rc = ad::shrink(s, flags)) return rc;
  }
  if (T > 0 && DX) {
    ad::LinearArgs l{DY, T, stride_dym, W, stride_wo, stride_wi, nullptr, G, A, stride_aa, stride_aj, stride_ai, adapter_idxs, DX,
                     in, n, out, in, r, dtype, status, st};
    if (int rc = ad::linear(l, flags)) return rc;
  }
  if (DA) {
    ad::GradArgs g{G, T, X, stride_xm, sorted_idx, offsets, DA, static_cast<int64_t>(r) * in, in, 1, n, in, r, dtype, parts, parts_bytes, st};
    if (int rc = ad::outer(g, flags)) return rc;
  }
  if (DB) {
    ad::GradArgs g{H, T, DY, stride_dym, sorted_idx, offsets, DB, static_cast<int64_t>(r) * out, 1, r, n, out, r, dtype, parts, parts_bytes, st};
    if (int rc = ad::outer(g, flags)) return rc;
  }
  if (DW) {      // the shared weight: one segment of the grouped weight gradient, its bias with it
    int64_t* rows = reinterpret_cast<int64_t*>(parts);
    ad::set_rows_kernel<<<1, 1, 0, st>>>(rows, T);
    SMOE_LAUNCH_CHECK();
    return smoe_group_bwd_w(DY, stride_dym, 1, X, T, stride_xm, 1, rows, nullptr, 1, DW, static_cast<int64_t>(out) * in, 1, in, Dbias,
                            out, 1, T, in, out, 1, dtype, flags & (SMOE_FLAG_FORCE_SIMT | SMOE_FLAG_FORCE_TC), status, stream);
  }
  if (Dbias) return ad::column_sum(DY, T, stride_dym, out, Dbias, dtype, parts, st);
  return SMOE_OK;
}
