// Shared by the kernels of the few-token MoE layer (decode): arguments, and the plan every block derives from the router's ids.
//
//   slot s = t*k + j with expert e = ids[t, j]:   h_s = act(x_t W1[e] + b1[e]);   y_t = sum_j g[t, j] (h_s W2[e] + b2[e])
//
// With a handful of tokens an expert has zero to a few dozen rows and the layer is bound by reading the weights of the
// experts that occur, once. The work is therefore a list of JOBS, (expert, up to NT of its slots): every weight element
// of a job's expert is read once for the job's slots together.
#pragma once

#include "smoe_common.cuh"

namespace smoe {
namespace ft {

constexpr int MAX_T = 128;      // tokens of one call
constexpr int MAX_R = 1024;     // slots of one call (T * k)
constexpr int MAX_E = 1024;
constexpr int PLAN_WARPS = 8;   // warps that sort the slots

struct Args {
  const void* X; int64_t sxm;
  const void* W1; int64_t s1e, s1k, s1n;
  const void* B1; int64_t sb1e, sb1n;
  const void* W2; int64_t s2e, s2k, s2n;
  const void* B2; int64_t sb2e, sb2n;
  const void* gates; int64_t sgt, sgk; int gates_dtype;
  const int64_t* ids; int64_t sit, sik;
  void* Y; int64_t sym;
  int T, k, d, F, d_out, E, act_layout, act, dtype;
  float alpha, limit;
  void* ws; size_t ws_bytes;
  int32_t* status;
  int after_router;     // the launch before on this stream is the router that writes ids and gates
  cudaStream_t stream;
};

// What an adapter adds to the values of a plain linear (adapter.cuh): sum over j of h[t, j] m[ids[t]][j, o]. The launch before on the
// stream writes h, and nothing else that the kernel reads.
struct Extension {
  const void* h; int64_t h_pitch;
  const void* m; int64_t sma, smj, smo;
  const int64_t* ids;      // null: nothing is added
  int n, r, m_vec;
};

inline int n_up(const Args& a) { return a.act_layout == 0 ? a.F : 2 * a.F; }

// CUDA-core kernels: fp32, and 16-bit operands the streaming kernels cannot address (any strides, any sizes).
int launch_simt(const Args& a);
size_t simt_workspace_bytes(int64_t T, int k, int F, int d_out);
// Streaming tensor-core kernels; SMOE_ERR_UNSUPPORTED (no error text) when the operands do not fit them.
int launch_stream(const Args& a);
int launch_linear(const Args& a, const Extension& ext);
size_t stream_workspace_bytes(int64_t T, int k, int F, int d_out);

// ---- plan --------------------------------------------------------------------------------------------
// Slots sorted by expert (stable, so that equal inputs give bit-equal outputs) and cut into jobs.
struct alignas(16) Plan {
  uint16_t slots[MAX_R];
  uint16_t job_expert[MAX_R];
  uint16_t job_begin[MAX_R];
  uint16_t job_count[MAX_R];
  int jobs;
};

// Bytes of scratch `make_plan` needs (dead afterwards): per-warp histograms and one packed prefix per expert.
__host__ __device__ inline int plan_scratch_bytes(int E) { return PLAN_WARPS * E * 2 + E * 4 + 16; }

// Whole-block call (at least PLAN_WARPS warps). Ids outside [0, E) belong to no job; without `ids` every slot is expert 0's. Ends with a
// barrier.
__device__ inline void make_plan(Plan* plan, uint8_t* scratch, const int64_t* ids, int64_t sit, int64_t sik, int T, int k,
                                 int E, int NT) {
  const int tid = threadIdx.x, nthreads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  uint32_t* packed = reinterpret_cast<uint32_t*>(scratch);                    // [E] count | jobs << 16, then their prefixes
  uint16_t* hist = reinterpret_cast<uint16_t*>(scratch + ((E * 4 + 15) & ~15));   // [PLAN_WARPS][E]
  const int R = T * k;
  if (R <= 32) {      // one warp sorts them in registers: position = slots of a lower expert + earlier slots of the same
    if (warp == 0) {
      int e = MAX_E + 1;
      if (lane < R) {
        const int64_t id = ids ? ids[static_cast<int64_t>(lane / k) * sit + static_cast<int64_t>(lane % k) * sik] : 0;
        if (id >= 0 && id < E) e = static_cast<int>(id);
      }
      const bool live = e < E;
      int lower = 0, same = 0, total = 0, jobs_before = 0;
      for (int o = 0; o < R; ++o) {
        const int oe = __shfl_sync(0xffffffffu, e, o);
        lower += oe < e;
        total += oe == e;
        same += oe == e && o < lane;
      }
      const bool leads = live && same == 0;
      const int my_jobs = leads ? (total + NT - 1) / NT : 0;
      int all_jobs = 0;
      for (int o = 0; o < R; ++o) {
        const int oe = __shfl_sync(0xffffffffu, e, o), oj = __shfl_sync(0xffffffffu, my_jobs, o);
        jobs_before += oe < e ? oj : 0;
        all_jobs += oj;
      }
      if (live) plan->slots[lower + same] = static_cast<uint16_t>(lane);
      if (leads)
        for (int c = 0, job = jobs_before; c < total; c += NT, ++job) {
          plan->job_expert[job] = static_cast<uint16_t>(e);
          plan->job_begin[job] = static_cast<uint16_t>(lower + c);
          plan->job_count[job] = static_cast<uint16_t>(min(NT, total - c));
        }
      if (lane == 0) plan->jobs = all_jobs;
    }
    __syncthreads();
    return;
  }
  constexpr int STEPS = MAX_R / (PLAN_WARPS * 32);
  const int steps = (R + PLAN_WARPS * 32 - 1) / (PLAN_WARPS * 32);
  for (int i = tid; i < PLAN_WARPS * E; i += nthreads) hist[i] = 0;
  __syncthreads();
  int my_e[STEPS], my_rank[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    my_e[i] = -1;
    my_rank[i] = 0;
    if (warp < PLAN_WARPS && i < steps) {
      const int s = (warp * steps + i) * 32 + lane;
      int e = -1;
      if (s < R) {
        const int64_t id = ids ? ids[static_cast<int64_t>(s / k) * sit + static_cast<int64_t>(s % k) * sik] : 0;
        e = (id >= 0 && id < E) ? static_cast<int>(id) : -1;
      }
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int before = (e >= 0) ? hist[warp * E + e] : 0;
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) hist[warp * E + e] = static_cast<uint16_t>(before + __popc(same));
      __syncwarp();
      my_e[i] = e;
      my_rank[i] = before + __popc(same & ((1u << lane) - 1u));
    }
  }
  __syncthreads();
  for (int e = tid; e < E; e += nthreads) {
    int c = 0;
    for (int w = 0; w < PLAN_WARPS; ++w) {
      const int h = hist[w * E + e];
      hist[w * E + e] = static_cast<uint16_t>(c);
      c += h;
    }
    packed[e] = static_cast<uint32_t>(c) | (static_cast<uint32_t>((c + NT - 1) / NT) << 16);
  }
  __syncthreads();
  if (warp == 0) {
    const int per = (E + 31) / 32, beg = min(lane * per, E), end = min(beg + per, E);
    uint32_t sum = 0;
    for (int e = beg; e < end; ++e) sum += packed[e];
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    uint32_t run = inc - sum;
    for (int e = beg; e < end; ++e) {
      const uint32_t mine = packed[e];
      packed[e] = run;
      const int begin = static_cast<int>(run & 0xffffu), count = static_cast<int>(mine & 0xffffu);
      int job = static_cast<int>(run >> 16);
      for (int c = 0; c < count; c += NT, ++job) {
        plan->job_expert[job] = static_cast<uint16_t>(e);
        plan->job_begin[job] = static_cast<uint16_t>(begin + c);
        plan->job_count[job] = static_cast<uint16_t>(min(NT, count - c));
      }
      run += mine;
    }
    if (lane == 31) plan->jobs = static_cast<int>(inc >> 16);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    if (my_e[i] >= 0) {
      const int at = static_cast<int>(packed[my_e[i]] & 0xffffu) + hist[warp * E + my_e[i]] + my_rank[i];
      plan->slots[at] = static_cast<uint16_t>((warp * steps + i) * 32 + lane);
    }
  __syncthreads();
}

// 32 values per lane -> lane l holds the sum over the lanes of value l.
__device__ __forceinline__ float transpose_reduce(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < o) {
        const float send = upper ? v[i] : v[i + o];
        const float keep = upper ? v[i + o] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
  }
  return v[0];
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == SMOE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SMOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

}  // namespace ft
}  // namespace smoe
