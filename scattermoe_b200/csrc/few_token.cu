// The few-token MoE layer as a stream of weights (16-bit): two launches, the up-projection with the activation and the gate, then the
// down-projection with the sum over a token's experts.
//
// Bound: the weights of the experts that occur cross HBM once; everything else is small. So the kernels are built around
// that stream. One block per SM; one thread keeps a ring of weight pieces in flight by TMA, two warps gather the token rows beside them
// (cp.async), eight warps multiply what has arrived with mma.sync: 16 weight rows x 8 slots x 16 of K per instruction. Weights are the M side, the job's slots the N side, so a
// job of 1 to 8 slots costs one instruction per 16x16 weights and the tensor pipe stays far below its limit; a
// tcgen05 tile would need 128 weight rows at a time, and with a handful of active experts the rows could not be spread evenly over
// 148 SMs. Here the split is exact: a block owns a contiguous range of hidden values (up) or of output columns (down).
//
// Weights with contiguous inputs ("K-major", nn.Linear storage): boxes of 64 of K x (16 hidden values x their 2 columns, or the block's
// output columns), starting at any row, so that a range may begin anywhere (rows that two blocks load come from L2). One bulk copy
// per weight row instead of boxes moved 1.2-3 TB/s: a block could issue one only every 40-50 ns.
// Weights with contiguous outputs ("N-major"): boxes of 32 columns x a piece of K, read
// through transposing ldmatrix; the columns of the down-projection are too few to fill the SMs, so there the list
// (column tile, job, piece of K) is cut into equal parts and partial sums are joined in a fixed order by the last block of a tile.
//
// The down-projection starts (programmatic launch) while the up-projection drains: it plans and fills its ring with weights, which do not
// depend on the hidden rows, and waits only before the first hidden row is read.
// fp32 accumulation; the hidden rows carry the gate and are rounded once, as the tensor cores need them.
#include <cuda.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "act_math.cuh"
#include "few_token.cuh"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace smoe {
namespace ft {

using namespace ptx;

constexpr int CONSUMERS = 8;                       // warps that multiply
constexpr int GATHERERS = 2;                       // warps that fetch the slots' rows
constexpr int THREADS = (CONSUMERS + 1 + GATHERERS) * 32;      // and one whose first thread loads the weights
constexpr int MAX_STAGES = 16;
constexpr int BOX = 32;                            // columns of an N-major TMA box (64 bytes)
constexpr int MAX_CTAS = 160;
constexpr int RED_PITCH = 33;

struct StreamParams {
  Args a;
  uint8_t* hidden;            // (R, F), storage type of the tokens
  float* partial;             // N-major down-projection: [block][2][T][2 * BOX]
  int* counters;              // one per column tile of it, zeroed by the up-projection
  int n_counters;
  int32_t* status;
  int NT;                     // slots of a job
  int KC, n_chunks, K;        // piece of K (a multiple of 64), pieces, K
  int box_bytes, load_bytes;  // K-major: bytes a box of 64 of K takes in the ring, and bytes it loads
  int stages, stage_bytes, x_offset, ring_bytes;
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm2(uint32_t& r0, uint32_t& r1, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// one arrival once every cp.async this thread has issued is complete
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Position in the ring: stage and the parity of its current pass.
struct RingPos {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
};

// ---- the list of runs of a block --------------------------------------------------------------------------
// A run is a stretch of K of one (weight tile, job) pair. Up-projection: the whole K of a tile of hidden values. Down-projection: the
// runs of a tile follow each other and their results add up; `last` closes the tile (for this block).
struct Run { int job, c0, c1, p0, count, tile; bool first, last; };

template <bool UP, bool KMAJOR>
struct Walker {
  int lo, hi, units, jobs, chunks, width, per_tile, r1, job;

  // up: units = hidden values (K-major) or box groups (N-major) of one job; [lo, hi) is this block's part of all jobs' units.
  // down, K-major: [lo, r1) are this block's output columns. down, N-major: [lo, hi) is its part of the flat list of pieces.
  __device__ void init(const StreamParams& p, int n_jobs) {
    jobs = n_jobs;
    chunks = p.n_chunks;
    const int64_t b = blockIdx.x, g = gridDim.x;
    const bool pairs = p.a.act_layout != LAYOUT_PLAIN, halves = pairs && p.a.act_layout != LAYOUT_GPT_OSS;
    job = 0;
    if (UP) {
      width = p.a.F;
      if (KMAJOR) {
        units = p.a.F;
        per_tile = pairs ? 16 : 32;
      } else {
        units = halves ? (p.a.F + BOX - 1) / BOX : ((pairs ? 2 * p.a.F : p.a.F) + BOX - 1) / BOX;
        per_tile = halves ? 1 : 2;
      }
      const int64_t total = static_cast<int64_t>(units) * jobs;
      lo = static_cast<int>(total * b / g);
      hi = static_cast<int>(total * (b + 1) / g);
    } else if (KMAJOR) {
      width = p.a.d_out;
      lo = static_cast<int>(static_cast<int64_t>(width) * b / g);
      r1 = static_cast<int>(static_cast<int64_t>(width) * (b + 1) / g);
    } else {
      width = p.a.d_out;
      units = jobs * chunks;      // pieces of one column tile
      const int64_t total = static_cast<int64_t>(units) * ((width + 2 * BOX - 1) / (2 * BOX));
      lo = static_cast<int>(total * b / g);
      hi = static_cast<int>(total * (b + 1) / g);
    }
  }
  __device__ bool next(Run& r) {
    if (UP) {
      if (lo >= hi) return false;
      r.job = lo / units;
      r.p0 = lo - r.job * units;
      r.count = min(min(per_tile, units - r.p0), hi - lo);
      r.c0 = 0;
      r.c1 = chunks;
      r.first = r.last = true;
      lo += r.count;
      return true;
    }
    if (KMAJOR) {
      if (lo >= r1) return false;
      r.job = job;
      r.p0 = lo;
      r.count = min(32, r1 - lo);
      r.c0 = 0;
      r.c1 = chunks;
      r.first = job == 0;
      r.last = ++job == jobs;
      if (r.last) { job = 0; lo += r.count; }
      return true;
    }
    if (lo >= hi) return false;
    r.tile = lo / units;
    const int in = lo - r.tile * units;
    r.job = in / chunks;
    r.c0 = in - r.job * chunks;
    r.c1 = min(chunks, r.c0 + (hi - lo));
    r.p0 = r.tile * 2 * BOX;
    r.count = min(2 * BOX, width - r.p0);
    r.first = job == 0 || in == 0;     // `job` only marks "not the first run of the block" here
    job = 1;
    lo += r.c1 - r.c0;
    r.last = lo >= hi || lo % units == 0;
    return true;
  }
};

// hidden value from the up-projection's one or two columns (act_math.cuh has the layouts)
__device__ __forceinline__ float hidden_fast(int layout, int act, float alpha, float limit, float c0, float c1) {
  if (layout == LAYOUT_GPT_OSS) {
    const float g = fminf(c0, limit), u = fminf(fmaxf(c1, -limit), limit);
    return (u + 1.0f) * (g * sigmoidf_<true>(alpha * g));
  }
  const float gate = layout == LAYOUT_GLU_SECOND ? c1 : c0;
  const float lin = layout == LAYOUT_PLAIN ? 1.0f : (layout == LAYOUT_GLU_SECOND ? c0 : c1);
  float r;
  SMOE_ACT_SWITCH(act, r = act_fwd<ACT_, true>(gate);)
  return r * lin;
}

template <typename T, bool UP, bool KMAJOR>
__global__ void __launch_bounds__(THREADS, 1)
ft_stream_kernel(const __grid_constant__ CUtensorMap tmap, const StreamParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);      // the ring first: 64-byte swizzle wants 512-byte alignment
  uint8_t* ring = smem;
  uint8_t* rest = ring + p.ring_bytes;
  Plan* plan = reinterpret_cast<Plan*>(rest);
  uint8_t* token = rest + sizeof(Plan);                              // token of every listed slot (T <= 128)
  uint64_t* bars = reinterpret_cast<uint64_t*>(token + MAX_R);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * MAX_STAGES);
  int* joined = reinterpret_cast<int*>(bars + 2 * MAX_STAGES) + 1;
  float* red = reinterpret_cast<float*>(bars + 2 * MAX_STAGES + 2);   // [8][NT][RED_PITCH]
  constexpr int RT = KMAJOR ? 32 : 2 * BOX;                           // weight rows (output columns) of a tile
  constexpr int OP = RT + 1;
  float* oacc = red + 8 * p.NT * RED_PITCH;                          // down: [T][OP]
  const Args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (MAX_STAGES + s); };

  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1 + GATHERERS * 32);      // the weights (expect_tx) and the gatherers' threads
      mbar_init(empty_bar(s), CONSUMERS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap);
  }
  if (UP) {
    wait_for_previous_kernel();        // ids, gates (and everything else) come from it when it is the router
    let_next_kernel_start();
    if (blockIdx.x == 0)
      for (int i = tid; i < p.n_counters; i += THREADS) p.counters[i] = 0;
  }
  // ids are older than the up-projection, so the down-projection plans before it waits
  make_plan(plan, ring, a.ids, a.sit, a.sik, a.T, a.k, a.E, p.NT);
  const int listed = plan->jobs ? plan->job_begin[plan->jobs - 1] + plan->job_count[plan->jobs - 1] : 0;
  for (int i = tid; i < listed; i += THREADS) token[i] = static_cast<uint8_t>(plan->slots[i] / a.k);
  fence_proxy_async_smem();            // the plan's scratch in the ring was written with ordinary stores
  __syncthreads();

  if (!UP && plan->jobs == 0) {        // no expert at all: rows of zeros
    wait_for_previous_kernel();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + tid; i < static_cast<int64_t>(a.T) * a.d_out;
         i += static_cast<int64_t>(gridDim.x) * THREADS)
      static_cast<T*>(a.Y)[(i / a.d_out) * a.sym + i % a.d_out] = from_f32<T>(0.f);
    return;
  }

  Walker<UP, KMAJOR> walk;
  walk.init(p, plan->jobs);
  const bool pairs = UP && a.act_layout != LAYOUT_PLAIN;
  const bool halves = pairs && a.act_layout != LAYOUT_GPT_OSS;

  if (warp == CONSUMERS) {
    // ---------------- weights: they depend on no kernel before, so nothing is waited for -----------------------------
    if (lane != 0) return;
    Run r;
    RingPos at;
    bool ok = true;
    while (walk.next(r) && ok) {
      const int e = plan->job_expert[r.job];
      for (int c = r.c0; c < r.c1; ++c, at.next(p.stages)) {
        const int s = at.stage;
        if (!mbar_wait(empty_bar(s), at.phase ^ 1, abort_flag, p.status, 21)) { ok = false; break; }
        const uint32_t dst = ring0 + s * p.stage_bytes;
        if (KMAJOR) {
          const int steps = (min(p.KC, p.K - c * p.KC) + 63) >> 6;
          mbar_arrive_expect_tx(full_bar(s), steps * p.load_bytes);
          for (int b = 0; b < steps; ++b)
            tma_load_4d(dst + b * p.box_bytes, &tmap, full_bar(s), c * p.KC + b * 64, r.p0, 0, e);
        } else {
          const int n_box = UP ? (halves ? 2 : r.count) : (r.count + BOX - 1) / BOX;
          mbar_arrive_expect_tx(full_bar(s), n_box * p.KC * BOX * 2);
          for (int b = 0; b < n_box; ++b) {
            const int col = UP ? (halves ? b * a.F + r.p0 * BOX : (r.p0 + b) * BOX) : r.p0 + b * BOX;
            tma_load_3d(dst + b * p.KC * BOX * 2, &tmap, full_bar(s), col, c * p.KC, e);
          }
        }
      }
    }
    if (!ok)      // give copies already in flight time to land before the block goes away
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    return;
  }
  if (warp > CONSUMERS) {
    // ---------------- the slots' rows: 16 bytes per thread, zeros beyond K ---------------------------------------------
    if (!UP) wait_for_previous_kernel();
    const int g = tid - (CONSUMERS + 1) * 32, chunk = g & 7, row0 = g >> 3;      // rows row0, row0 + 8, ...
    const uint32_t sw = static_cast<uint32_t>((chunk ^ row0) << 4);              // row & 7 == row0
    Run r;
    RingPos at;
    bool ok = true;
    while (walk.next(r) && ok) {
      const int n = plan->job_count[r.job], beg = plan->job_begin[r.job];
      const uint8_t* src[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = beg + min(row0 + 8 * i, n - 1);
        src[i] = UP ? static_cast<const uint8_t*>(a.X) + static_cast<int64_t>(token[j]) * a.sxm * 2
                    : p.hidden + static_cast<int64_t>(plan->slots[j]) * a.F * 2;
      }
      for (int c = r.c0; c < r.c1; ++c, at.next(p.stages)) {
        const int s = at.stage;
        if (!mbar_wait(empty_bar(s), at.phase ^ 1, abort_flag, p.status, 23)) { ok = false; break; }
        const uint32_t dst = ring0 + s * p.stage_bytes + p.x_offset + row0 * 128 + sw;
        const int k0 = c * p.KC + chunk * 8, k_end = min((c + 1) * p.KC, (p.K + 63) & ~63);
        for (int kk = k0, b = 0; kk < k_end; kk += 64, ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row0 + 8 * i < n)
              cp_async16(dst + (b * p.NT + 8 * i) * 128, src[i] + (kk < p.K ? kk * 2 : 0), kk < p.K ? 16 : 0);
        cp_async_arrive(full_bar(s));
      }
    }
    cp_async_wait<0>();
    return;
  }

  // ---------------- products -----------------------------------------------------------------------------------
  // a wait that runs out does not leave the loops: the barriers below stay matched, the results are reported as invalid
  if (!UP) wait_for_previous_kernel();
  bool ok = true;
  RingPos at;
  Run r;
  const int my_box = KMAJOR ? 0 : warp >> 2;
  // ldmatrix addresses of this lane inside a stage; the loop over K only adds multiples of a block of 64
  uint32_t a_lane[2], x_lane[2], x_lane4[2];       // K-major: the two 16-wide steps of the warp's half of a block of 64
  {
    const int row = (lane & 7) + ((lane >> 3) & 1) * 8, xrow4 = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int step = KMAJOR ? (warp & 1) * 2 + i : warp & 3;
      a_lane[i] = KMAJOR ? row * 128 + (((step * 2 + (lane >> 4)) ^ (row & 7)) << 4) : 0;
      x_lane[i] = (lane & 7) * 128 + (((step * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
      x_lane4[i] = xrow4 * 128 + (((step * 2 + ((lane >> 3) & 1)) ^ (xrow4 & 7)) << 4);
    }
    if (!KMAJOR) {
      const int krow = (warp & 3) * 16 + (lane & 7) + (lane >> 4) * 8, chunk = (lane >> 3) & 1;
#pragma unroll
      for (int i = 0; i < 2; ++i)                  // N-major: the two 16-column halves of the warp's box
        a_lane[i] = my_box * p.KC * BOX * 2 + krow * (BOX * 2) + (((chunk + 2 * i) ^ ((krow >> 1) & 3)) << 4);
    }
  }
  const int x_block = p.NT * 128;
  auto total_of = [&](int i, int row) {       // sum over the warps that share this row
    float v = 0.f;
    if (KMAJOR) {
#pragma unroll
      for (int w = 0; w < 8; ++w) v += red[(w * p.NT + i) * RED_PITCH + row];
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) v += red[(((row >> 5) * 4 + w) * p.NT + i) * RED_PITCH + (row & 31)];
    }
    return v;
  };
  while (walk.next(r)) {
    const int n = plan->job_count[r.job], beg = plan->job_begin[r.job], e = plan->job_expert[r.job];
    const int groups = (n + 7) >> 3;
    bool use0, use1;                          // the warp's two 16-row halves that hold anything
    if (KMAJOR) {
      use0 = true;
      use1 = pairs || r.count > 16;
    } else {
      const int cols = UP ? (halves ? 2 * BOX : r.count * BOX) : r.count;
      use0 = cols > my_box * BOX;
      use1 = cols > my_box * BOX + 16;
    }
    if (!UP && r.first)
      for (int i = tid; i < a.T * OP; i += CONSUMERS * 32) oacc[i] = 0.f;
    float acc[2][4][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][g][q] = 0.f;
    auto stream = [&](auto G_) {
      constexpr int G = decltype(G_)::value;           // groups of 8 slots, rounded up to 1, 2 or 4
      for (int c = r.c0; c < r.c1; ++c, at.next(p.stages)) {
        const int s = at.stage;
        if (ok) ok = mbar_wait_warp(full_bar(s), at.phase, abort_flag, p.status, 22);
        if (ok && use0) {
          const int blocks = (min(p.KC, p.K - c * p.KC) + 63) >> 6;
          const uint32_t wst = ring0 + s * p.stage_bytes, xst = wst + p.x_offset;
          auto step = [&](uint32_t w0, uint32_t w1, uint32_t x1, uint32_t x4) {
            uint32_t a0[4], a1[4] = {0, 0, 0, 0}, b[G][2];
            if (KMAJOR) {
              ldsm4(a0, w0);
              if (use1) ldsm4(a1, w1);
            } else {
              ldsm4_trans(a0, w0);
              if (use1) ldsm4_trans(a1, w1);
            }
            if (G == 1) {
              ldsm2(b[0][0], b[0][1], x1);
            } else {
#pragma unroll
              for (int g = 0; g < G; g += 2) {
                uint32_t t[4];
                ldsm4(t, x4 + g * 8 * 128);
                b[g][0] = t[0]; b[g][1] = t[1]; b[g + 1][0] = t[2]; b[g + 1][1] = t[3];
              }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              Mma<T>::run(acc[0][g], a0, b[g][0], b[g][1]);
              if (use1) Mma<T>::run(acc[1][g], a1, b[g][0], b[g][1]);
            }
          };
          if (KMAJOR) {
            for (int b = warp >> 1; b < blocks; b += 4) {
              const uint32_t w = wst + b * p.box_bytes, x = xst + b * x_block;
#pragma unroll
              for (int i = 0; i < 2; ++i) step(w + a_lane[i], w + a_lane[i] + 16 * 128, x + x_lane[i], x + x_lane4[i]);
            }
          } else {
#pragma unroll 2
            for (int b = 0; b < blocks; ++b) {
              const uint32_t w = wst + b * (64 * BOX * 2), x = xst + b * x_block;
              step(w + a_lane[0], w + a_lane[1], x + x_lane[0], x + x_lane4[0]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar(s));
      }
    };
    if (groups == 1) stream(std::integral_constant<int, 1>{});
    else if (groups == 2) stream(std::integral_constant<int, 2>{});
    else stream(std::integral_constant<int, 4>{});
    // ---- join the warps' parts of K
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if (m == 0 ? use0 : use1)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g < groups) {
            float* out = red + (warp * p.NT + g * 8 + (lane & 3) * 2) * RED_PITCH + m * 16 + (lane >> 2);
            out[0] = acc[m][g][0];
            out[RED_PITCH] = acc[m][g][1];
            out[8] = acc[m][g][2];
            out[RED_PITCH + 8] = acc[m][g][3];
          }
    consumers_sync();
    if (UP) {
      // hidden values of this tile: first value, how many, and where their columns are
      int v0, count;
      if (KMAJOR) { v0 = r.p0; count = r.count; }
      else if (halves) { v0 = r.p0 * BOX; count = min(BOX, a.F - v0); }
      else if (pairs) { v0 = r.p0 * (BOX / 2); count = min(r.count * (BOX / 2), a.F - v0); }
      else { v0 = r.p0 * BOX; count = min(r.count * BOX, a.F - v0); }
      const int second = KMAJOR ? 16 : BOX;
      for (int idx = tid; idx < n * count; idx += CONSUMERS * 32) {
        const int i = idx / count, v = idx - i * count, pv = v0 + v;
        const bool woven = !KMAJOR && pairs && !halves;       // interleaved columns stand side by side in the boxes
        float c0 = total_of(i, woven ? 2 * v : v);
        float c1 = pairs ? total_of(i, woven ? 2 * v + 1 : second + v) : 0.f;
        if (a.B1) {
          const T* bias = static_cast<const T*>(a.B1) + e * a.sb1e;
          c0 += to_f32<T>(bias[(pairs ? (halves ? pv : 2 * pv) : pv) * a.sb1n]);
          if (pairs) c1 += to_f32<T>(bias[(halves ? a.F + pv : 2 * pv + 1) * a.sb1n]);
        }
        const int slot = plan->slots[beg + i];
        float h = hidden_fast(a.act_layout, a.act, a.alpha, a.limit, c0, c1);
        if (a.gates) h *= load_any(a.gates, (slot / a.k) * a.sgt + (slot % a.k) * a.sgk, a.gates_dtype);
        reinterpret_cast<T*>(p.hidden)[static_cast<int64_t>(slot) * a.F + pv] = from_f32<T>(h);
      }
      consumers_sync();
    } else {
      // add the job's slots to their tokens; slots of one token (the same expert twice) stand together and go to one thread
      const int row = tid % RT;
      for (int i = tid / RT; i < n; i += CONSUMERS * 32 / RT) {
        const int t = token[beg + i];
        if (i > 0 && token[beg + i - 1] == t) continue;
        if (row < r.count) {
          float v = total_of(i, row);
          for (int m = i + 1; m < n && token[beg + m] == t; ++m) v += total_of(m, row);
          oacc[t * OP + row] += v;
        }
      }
      consumers_sync();
      if (r.last) {
        bool write = true;
        if (!KMAJOR) {
          // does this block hold the whole tile, or only a part of its pieces?
          const int64_t g = gridDim.x, tile_beg = static_cast<int64_t>(r.tile) * walk.units, tile_end = tile_beg + walk.units;
          const int64_t total = static_cast<int64_t>(walk.units) * ((a.d_out + 2 * BOX - 1) / (2 * BOX));
          auto begin_of = [&](int64_t b) { return total * b / g; };
          const int64_t mine0 = begin_of(blockIdx.x), mine1 = begin_of(blockIdx.x + 1);
          if (mine0 > tile_beg || mine1 < tile_end) {
            float* part = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (mine0 > tile_beg ? 0 : 1)) * a.T * RT;
            for (int i = tid; i < a.T * RT; i += CONSUMERS * 32) part[i] = oacc[(i / RT) * OP + i % RT];
            __threadfence();
            consumers_sync();
            int64_t first = tile_beg * g / total, stop = first;
            while (first > 0 && begin_of(first) > tile_beg) --first;
            while (begin_of(first + 1) <= tile_beg) ++first;
            int parts = 0;
            for (stop = first; stop < g && begin_of(stop) < tile_end; ++stop) parts += begin_of(stop + 1) > begin_of(stop);
            if (tid == 0) *joined = atomicAdd(p.counters + r.tile, 1) == parts - 1;
            consumers_sync();
            write = *joined != 0;
            if (write) {        // the last block of the tile adds the parts up, always in the same order
              __threadfence();
              for (int i = tid; i < a.T * RT; i += CONSUMERS * 32) {
                float v = 0.f;
                for (int64_t b = first; b < stop; ++b)
                  if (begin_of(b + 1) > begin_of(b))
                    v += __ldcg(p.partial + (b * 2 + (begin_of(b) > tile_beg ? 0 : 1)) * a.T * RT + i);
                oacc[(i / RT) * OP + i % RT] = v;
              }
            }
            consumers_sync();
          }
        }
        if (write)
          for (int idx = tid; idx < a.T * r.count; idx += CONSUMERS * 32) {
            const int t = idx / r.count, col = idx - t * r.count;
            float v = oacc[t * OP + col];
            if (a.B2)
              for (int j = 0; j < a.k; ++j) {
                const int64_t ex = a.ids[t * a.sit + j * a.sik];
                if (ex < 0 || ex >= a.E) continue;
                const float b = to_f32<T>(static_cast<const T*>(a.B2)[ex * a.sb2e + (r.p0 + col) * a.sb2n]);
                v += a.gates ? load_any(a.gates, t * a.sgt + j * a.sgk, a.gates_dtype) * b : b;
              }
            static_cast<T*>(a.Y)[t * a.sym + r.p0 + col] = from_f32<T>(v);
          }
        consumers_sync();
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr size_t HIDDEN_ALIGN = 256;
static size_t hidden_bytes(int64_t T, int k, int F) {
  return (static_cast<size_t>(T) * k * F * 2 + HIDDEN_ALIGN - 1) / HIDDEN_ALIGN * HIDDEN_ALIGN;
}
static int column_tiles(int d_out) { return cdiv(d_out, 2 * BOX); }
size_t stream_workspace_bytes(int64_t T, int k, int F, int d_out) {
  return hidden_bytes(T, k, F) + static_cast<size_t>(column_tiles(d_out)) * 4 + 16 +
         static_cast<size_t>(MAX_CTAS) * 2 * T * 2 * BOX * 4;
}

struct Order { bool k_major, n_major; };
static Order weight_order(const void* W, int64_t se, int64_t sk, int64_t sn, int K, int N) {
  if (!al16(W) || se % 8 || se < 0) return {false, false};
  return {sk == 1 && sn % 8 == 0 && sn >= K, sn == 1 && sk % 8 == 0 && sk >= N && N % 8 == 0};
}

// Pieces of K: multiples of 64, at most `most`, all but the last alike.
static int piece_of(int K, int most) {
  const int blocks = cdiv(K, 64), n = cdiv(blocks, most / 64);
  return cdiv(blocks, n) * 64;
}

// K-major boxes: 64 of K x `rows` x `halves` (the two columns of a hidden value; 1 without a gate) of one expert.
static bool encode_k_major(CUtensorMap* map, bool bf16, const void* W, int K, int rows_total, int64_t row_stride, int halves,
                           int64_t half_stride, int E, int64_t se, int box_rows) {
  const uint64_t dim[4] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows_total), static_cast<uint64_t>(halves),
                           static_cast<uint64_t>(E)};
  // the stride of an axis of one element is never used, but has to be valid
  const uint64_t stride[3] = {static_cast<uint64_t>(row_stride) * 2, static_cast<uint64_t>(halves > 1 ? half_stride : row_stride) * 2,
                              static_cast<uint64_t>(E > 1 ? se : row_stride) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(halves), 1};
  return encode_tensor_map(map, bf16, W, 4, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
static bool encode_n_major(CUtensorMap* map, bool bf16, const void* W, int N, int K, int64_t row_stride, int E, int64_t se, int box_k) {
  const uint64_t dim[3] = {static_cast<uint64_t>(N), static_cast<uint64_t>(K), static_cast<uint64_t>(E)};
  const uint64_t stride[2] = {static_cast<uint64_t>(row_stride) * 2, static_cast<uint64_t>(E > 1 ? se : row_stride) * 2};
  const uint32_t box[3] = {BOX, static_cast<uint32_t>(box_k), 1};
  return encode_tensor_map(map, bf16, W, 3, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

// rows of a K-major box: the hidden values of a tile, or the output columns of a block (at most 32)
static int down_rows(int d_out, int grid) { return cdiv(d_out, grid) < 32 ? cdiv(d_out, grid) : 32; }

template <typename T, bool UP, bool KMAJOR>
static int launch_one(StreamParams p, const CUtensorMap& map, const DeviceInfo& di, int grid) {
  const Args& a = p.a;
  // shared memory that is not the ring
  const int fixed = static_cast<int>(sizeof(Plan)) + MAX_R + (2 * MAX_STAGES + 2) * 8 + 8 * p.NT * RED_PITCH * 4 +
                    (UP ? 0 : a.T * ((KMAJOR ? 32 : 2 * BOX) + 1) * 4) + 1024 + 64;
  const int budget = (di.max_smem_optin < 232448 ? di.max_smem_optin : 232448) - fixed;
  if (KMAJOR) {
    const int rows = UP ? 32 : down_rows(a.d_out, grid);
    p.load_bytes = rows * 128;
    p.box_bytes = cdiv(rows, 8) * 1024;                    // boxes start on the swizzle's period
    // Stages of up to 32 KB of weights where the ring then still holds four, else 16 KB: enough of them that the stream never stops,
    // few enough that a stage is worth its waits (16 KB stages with one slot per job were bound by the warps' loop overhead).
    const int block = p.box_bytes + p.NT * 128;            // bytes of 64 of K: weights and slots
    p.KC = piece_of(p.K, 64 * (32768 / p.box_bytes));
    if ((budget - 2048) / (p.KC / 64 * block) < 4) p.KC = piece_of(p.K, 64 * (16384 / p.box_bytes));
    p.x_offset = p.KC / 64 * p.box_bytes;
  } else {
    p.load_bytes = p.box_bytes = 0;
    p.KC = piece_of(p.K, 256);                             // as the tensor map's boxes
    p.x_offset = 2 * p.KC * BOX * 2;
  }
  p.n_chunks = cdiv(p.K, p.KC);
  p.stage_bytes = p.x_offset + p.KC / 64 * p.NT * 128;
  p.stages = (budget - (KMAJOR ? 2048 : 0)) / p.stage_bytes;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  if (p.stages < 2) return SMOE_ERR_UNSUPPORTED;
  // ldmatrix reads whole 16-row blocks: up to 8 rows past a box of fewer rows (never used, but inside the ring)
  p.ring_bytes = p.stages * p.stage_bytes + (KMAJOR ? 2048 : 0);
  const int scratch = (plan_scratch_bytes(a.E) + 15) / 16 * 16;      // the plan sorts in the ring before the first copy
  if (scratch > budget) return SMOE_ERR_UNSUPPORTED;
  if (p.ring_bytes < scratch) p.ring_bytes = scratch;
  const int smem = fixed + p.ring_bytes;
  static std::mutex mu;
  static bool configured[64] = {false};
  {
    std::lock_guard<std::mutex> lock(mu);
    if (di.device < 0 || di.device >= 64 || !configured[di.device]) {
      SMOE_CUDA(cudaFuncSetAttribute(ft_stream_kernel<T, UP, KMAJOR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
      if (di.device >= 0 && di.device < 64) configured[di.device] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (!UP || a.after_router) ? 1 : 0;
  SMOE_CUDA(cudaLaunchKernelEx(&cfg, ft_stream_kernel<T, UP, KMAJOR>, map, p));
  return SMOE_OK;
}

template <typename T>
static int launch_typed(const Args& a, const DeviceInfo& di) {
  const int n_up_cols = n_up(a);
  const Order o1 = weight_order(a.W1, a.s1e, a.s1k, a.s1n, a.d, n_up_cols), o2 = weight_order(a.W2, a.s2e, a.s2k, a.s2n, a.F, a.d_out);
  if (!(o1.k_major || o1.n_major) || !(o2.k_major || o2.n_major)) return SMOE_ERR_UNSUPPORTED;
  const bool bf16 = a.dtype == SMOE_BF16;
  StreamParams p;
  p.a = a;
  p.hidden = static_cast<uint8_t*>(a.ws);
  uint8_t* after = static_cast<uint8_t*>(a.ws) + hidden_bytes(a.T, a.k, a.F);
  p.n_counters = column_tiles(a.d_out);
  p.counters = reinterpret_cast<int*>(after);
  p.partial = reinterpret_cast<float*>(after + (static_cast<size_t>(p.n_counters) * 4 + 15) / 16 * 16);
  p.status = a.status;
  p.NT = a.T <= 8 ? 8 : (a.T <= 16 ? 16 : 32);
  const int grid = di.sm_count < MAX_CTAS ? di.sm_count : MAX_CTAS;
  CUtensorMap m1, m2;
  memset(&m1, 0, sizeof(m1));
  memset(&m2, 0, sizeof(m2));
  const bool pairs = a.act_layout != LAYOUT_PLAIN, woven = a.act_layout == LAYOUT_GPT_OSS;
  const bool ok1 = o1.k_major ? encode_k_major(&m1, bf16, a.W1, a.d, a.F, woven ? 2 * a.s1n : a.s1n, pairs ? 2 : 1,
                                               woven ? a.s1n : a.s1n * a.F, a.E, a.s1e, pairs ? 16 : 32)
                              : encode_n_major(&m1, bf16, a.W1, n_up_cols, a.d, a.s1k, a.E, a.s1e, piece_of(a.d, 256));
  const bool ok2 = o2.k_major ? encode_k_major(&m2, bf16, a.W2, a.F, a.d_out, a.s2n, 1, 0, a.E, a.s2e, down_rows(a.d_out, grid))
                              : encode_n_major(&m2, bf16, a.W2, a.d_out, a.F, a.s2k, a.E, a.s2e, piece_of(a.F, 256));
  if (!ok1 || !ok2) return SMOE_ERR_UNSUPPORTED;
  p.K = a.d;
  if (int rc = o1.k_major ? launch_one<T, true, true>(p, m1, di, grid) : launch_one<T, true, false>(p, m1, di, grid)) return rc;
  p.K = a.F;
  return o2.k_major ? launch_one<T, false, true>(p, m2, di, grid) : launch_one<T, false, false>(p, m2, di, grid);
}

int launch_stream(const Args& a) {
  if (a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) return SMOE_ERR_UNSUPPORTED;
  if (a.d % 8 || a.F % 8 || a.sxm % 8 || !al16(a.X)) return SMOE_ERR_UNSUPPORTED;
  if (a.d > (1 << 20) || a.F > (1 << 20) || a.d_out > (1 << 20)) return SMOE_ERR_UNSUPPORTED;     // 32-bit unit counts
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  return a.dtype == SMOE_BF16 ? launch_typed<__nv_bfloat16>(a, di) : launch_typed<__half>(a, di);
}

}  // namespace ft
}  // namespace smoe
