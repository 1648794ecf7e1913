// The few-token MoE layer as a stream of weights (16-bit): two launches, the up-projection with the activation and the gate, then the
// down-projection with the sum over a token's experts.
//
// Bound: the weights of the experts that occur cross HBM once; everything else is small. So the kernels are built around
// that stream. One block per SM; four threads keep a ring of weight boxes in flight by TMA (4 KB each: 32 weight rows x 64 of K), two
// pairs of warps gather the slots' rows beside them, a stage each in turn (cp.async), eight warps multiply what has arrived with mma.sync:
// 16 weight rows x 8 slots x 16 of K per instruction. Weights are the M side, the job's slots the N side, so a job of 1 to 8 slots costs
// one instruction per 16x16 weights and the tensor pipe stays far below its limit up to about 16 slots. A tcgen05 tile is 64 or 128 weight
// rows at least, and 4096 output columns are 28 per SM: tiles of a handful of active experts cannot be dealt evenly over 148 SMs, and a
// stream has no use for the rate. Here the split is exact: a block owns a contiguous range of hidden values (up) or of output columns
// (down).
//
//   up    A round is up to 8 tiles of one job, a tile 32 weight rows: 16 hidden values with their two columns, or 32 without a gate. Each
//         warp owns a tile over the whole of K and makes its hidden values in registers: no exchange between warps, no barrier; the
//         slots' rows are fetched once per round. A round of few tiles gives each tile 2, 4 or 8 warps, which split the steps of K
//         and are joined through shared memory.
//   down  The block's output columns are one tile. Pairs of warps take the stages in turn, so that four jobs are under way at once, and
//         add their part of a job to token sums of their own in shared memory, joined in order once at the end. The two warps of a pair
//         hold 16 columns each, or half of K each where the tile has no more than 16.
//
// A first version gave the warps parts of K in both kernels and joined them after every tile and job: with many small jobs the
// joins cost as much as the stream (24 tokens on 128 experts of 9.4 MB: 126 + 127 us against 97 + 49 of reading).
// Issuing is what limits such a stream, not depth: one thread issues a box every 70-150 ns and spends 0.25 us more on a stage, so one
// thread moved 3.7 TB/s of 4 KB boxes (2.5 of 1.8 KB ones) with 25 to 190 KB in flight alike, two 5.4, four 5.4-5.7 (3.7-6.5), in stages of
// 32 KB; stages of 8 KB 2.2-4.2. Hence few, large stages, and as many steps of K in one as the job's slots leave room for.
// One bulk copy per weight row: 1.2-3 TB/s.
//
// Weights with contiguous inputs ("K-major", nn.Linear storage) are read through ldmatrix; weights with contiguous outputs ("N-major") through the transposing
// form, in boxes of 64 columns that two warps share (128-byte rows; with 64-byte rows the stream reached 60 %). N-major columns are too few to give every SM its own, so there the down-projection's list (column tile, job, piece of K)
// is cut into equal parts and partial sums are joined in a fixed order by the last block of a tile.
//
// The down-projection starts (programmatic launch) while the up-projection drains: it plans and fills its ring with weights, which do not
// depend on the hidden rows, and waits only before the first hidden row is read.
// fp32 accumulation; the hidden rows are rounded once, as the tensor cores need them, and carry the gate's power of two (see `carried`),
// the token sums take the rest of it.
#include <cuda.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "act_math.cuh"
#include "few_token.cuh"
#include "few_token_stages.h"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace smoe {
namespace ft {

using namespace ptx;

constexpr int CONSUMERS = 8;                       // warps that multiply
constexpr int LOADERS = 4;                         // warps whose first thread loads weights, each every fourth box of a stage
constexpr int GATHERERS = 4;                       // warps that fetch the slots' rows: two pairs that take the stages in turn
constexpr int GATHER_TURNS = 2;
constexpr int GATHER_THREADS = GATHERERS * 32 / GATHER_TURNS;
constexpr int DOWN_TURNS = 4;                      // down: pairs of multiplying warps that take the stages in turn
constexpr int THREADS = (CONSUMERS + LOADERS + GATHERERS) * 32;
// The number of stages is a multiple of the turns: every stage then always belongs to the same warps, which wait for each of its passes.
constexpr int TILE = 32;                           // weight rows (output columns) of a warp's tile
constexpr int BLOCK_K = 64;                        // K of a box: one 128-byte line of 16-bit values
constexpr int MAX_CTAS = 160;

struct StreamParams {
  Args a;
  uint8_t* hidden;            // (R, F), storage type of the tokens
  float* partial;             // N-major down-projection: [block][2][T][2 * TILE]
  int* counters;              // one per column tile of it, zeroed by the up-projection
  int n_counters;
  uint32_t part_step;         // 2^32 / blocks of the grid, rounded up
  int32_t* status;
  int NT;                     // slots of a job
  int K, blocks;              // K and its boxes
  int box_bytes, load_bytes;  // bytes a box takes in the ring, and bytes it loads
  Extension ext;              // up: added to the values before they are rounded (adapter_linear)
  Stages ring;
  int ring_bytes;
  int rows;                   // down: rows of a tile's token sums (the tile's columns)
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

// First of the units of block b when `total` units are dealt out evenly: the same for every caller, without a division.
// part_step is 2^32 / blocks, rounded up; total < 2^30.
__device__ __forceinline__ int part_begin(int total, int b, uint32_t part_step) {
  const uint64_t share = static_cast<uint64_t>(static_cast<uint32_t>(b)) * part_step;        // of 2^32
  const uint64_t at = share >= (1ull << 32) ? static_cast<uint64_t>(total) : (static_cast<uint64_t>(static_cast<uint32_t>(total)) * share) >> 32;
  return static_cast<int>(at);
}

// ---- the list of runs of a block --------------------------------------------------------------------------
// A run is a stretch of K of one job: up, a round of `tiles` tiles over the whole of K, `nb` steps of K per stage; down, (part
// of) the K of the block's tile. The runs of a tile follow each other; `last` closes the tile (for this block).
struct Run { int job, b0, b1, nb, p0, count, tiles, tile, groups, boxes, x_offset; bool first, last; };

template <bool UP, bool KMAJOR>
struct Walker {
  static constexpr int DOWN_TILE = KMAJOR ? TILE : 2 * TILE;      // output columns of a tile of the down-projection
  int lo, hi, units, jobs, blocks, width, per_tile, job, tile, step;

  // up: [lo, hi) is this block's part of all jobs' tiles.
  // down, K-major: [lo, hi) are this block's output columns; N-major: its part of the flat list of steps of K, (tile, job, step).
  __device__ void init(const StreamParams& p, int n_jobs) {
    jobs = n_jobs;
    blocks = p.blocks;
    job = -1;
    int total;
    if (UP) {
      width = p.a.F;
      per_tile = p.a.act_layout != LAYOUT_PLAIN ? TILE / 2 : TILE;
      units = (width + per_tile - 1) / per_tile;
      total = units * jobs;
    } else {
      width = p.a.d_out;
      units = jobs * blocks;      // steps of K of one column tile
      total = KMAJOR ? width : units * ((width + DOWN_TILE - 1) / DOWN_TILE);
    }
    lo = part_begin(total, blockIdx.x, p.part_step);
    hi = part_begin(total, blockIdx.x + 1, p.part_step);
  }
  __device__ bool next(Run& r) {
    if (lo >= hi) return false;
    r.b0 = 0;
    r.b1 = blocks;
    r.tiles = 1;
    if (UP) {
      r.job = lo / units;
      const int in = lo - r.job * units;
      // Whole rounds of 8 tiles and a last round of up to 3, which shares its tiles among the warps; a longer rest would leave warps
      // idle without that help, so then all rounds are made alike (12 tiles as 8 + 4: 132 us, as 6 + 6: 122 us for one token on two
      // experts of 352 MB; 33 as 4 x 8 + 1: 198 us, as 7 + 7 + 7 + 6 + 6: 203 us for 24 tokens on 128 experts of 9.4 MB).
      const int left = min(units - in, hi - lo), rounds = (left + CONSUMERS - 1) / CONSUMERS;
      r.tiles = left <= CONSUMERS ? left : ((left & (CONSUMERS - 1)) > 3 ? (left + rounds - 1) / rounds : CONSUMERS);
      lo += r.tiles;
      r.p0 = in * per_tile;
      r.count = min(r.tiles * per_tile, width - r.p0);
    } else if (KMAJOR) {
      r.first = ++job == 0;
      r.job = job;
      r.p0 = lo;
      r.count = min(TILE, hi - lo);
      r.last = job + 1 == jobs;
      if (r.last) { job = -1; lo += r.count; }
    } else {
      if (job < 0) {                       // the block's first run
        tile = lo / units;
        step = lo - tile * units;
        job = step / blocks;
        step -= job * blocks;
        r.first = true;
      } else {
        step = 0;
        if (++job == jobs) { job = 0; ++tile; }
        r.first = job == 0;
      }
      r.tile = tile;
      r.job = job;
      r.b0 = step;
      r.b1 = min(blocks, step + (hi - lo));
      r.p0 = tile * DOWN_TILE;
      r.count = min(DOWN_TILE, width - r.p0);
      lo += r.b1 - r.b0;
      r.last = lo >= hi || job + 1 == jobs;
    }
    return true;
  }
};

// Steps of K in a stage of this run, and where its slots' rows start (after the weights; `groups` x 8 rows of 128 bytes per step).
// An N-major box holds two tiles.
template <bool UP, bool KMAJOR>
__device__ __forceinline__ void shape_of(const StreamParams& p, Run& r, int n) {
  r.groups = (n + 7) >> 3;
  r.boxes = KMAJOR ? r.tiles : (r.tiles + 1) >> 1;
  r.nb = p.ring.steps_of[width_class(r.boxes)][r.groups - 1];
  r.x_offset = r.boxes * r.nb * p.box_bytes;
}

// The part of a gate that its hidden row carries: the power of two at or below it, between 1/16 and 1. Scaling by it costs no bit, and
// it leaves fp16 the headroom that a gate below 1 gives. A whole gate of 2^-18 would push fp16's rows below their normal range, where
// the step no longer shrinks (4 times the error that the rounding itself explains); no more than 1/16 keeps that at 2^-21 of a hidden
// value of 1.
__device__ __forceinline__ int carried_exponent(float gate) { return min(max(__float_as_int(gate) >> 23 & 0xff, 127 - 4), 127); }
__device__ __forceinline__ float carried(float gate) { return __int_as_float(carried_exponent(gate) << 23); }
__device__ __forceinline__ float rest_of(float gate) { return gate * __int_as_float((254 - carried_exponent(gate)) << 23); }

// hidden value from the up-projection's one or two columns (act_math.cuh has the layouts)
__device__ __forceinline__ float hidden_fast(int layout, int act, float alpha, float limit, float c0, float c1) {
  if (layout == LAYOUT_GPT_OSS) {
    const float g = min_nan(c0, limit), u = min_nan(max_nan(c1, -limit), limit);
    return (u + 1.0f) * (g * sigmoidf_<true>(alpha * g));
  }
  const float gate = layout == LAYOUT_GLU_SECOND ? c1 : c0;
  const float lin = layout == LAYOUT_PLAIN ? 1.0f : (layout == LAYOUT_GLU_SECOND ? c0 : c1);
  float r;
  SMOE_ACT_SWITCH(act, r = act_fwd<ACT_, true>(gate);)
  return r * lin;
}

// What adapter `id` adds to columns o and o + 16 of row t (second: whether the latter is wanted). h is read coherently: the kernel before
// this one writes it while this one already runs.
template <typename T>
__device__ __forceinline__ void extension_terms(const Extension& x, int t, int id, int o, bool second, float (&sum)[2]) {
  sum[0] = sum[1] = 0.f;
  if (id < 0) return;
  const T* h = static_cast<const T*>(x.h) + t * x.h_pitch;
  const T* m = static_cast<const T*>(x.m) + id * x.sma + o * x.smo;
  const int64_t next = second ? 16 * x.smo : 0;
  if (x.m_vec) {
#pragma unroll 4
    for (int j = 0; j < x.r; j += 8) {
      const uint4 hv = *reinterpret_cast<const uint4*>(h + j), m0 = __ldg(reinterpret_cast<const uint4*>(m + j)),
                  m1 = __ldg(reinterpret_cast<const uint4*>(m + next + j));
      const T *ht = reinterpret_cast<const T*>(&hv), *t0 = reinterpret_cast<const T*>(&m0), *t1 = reinterpret_cast<const T*>(&m1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[0] = fmaf(to_f32<T>(ht[i]), to_f32<T>(t0[i]), sum[0]);
        sum[1] = fmaf(to_f32<T>(ht[i]), to_f32<T>(t1[i]), sum[1]);
      }
    }
  } else {
    for (int j = 0; j < x.r; ++j) {
      sum[0] = fmaf(to_f32<T>(h[j]), to_f32<T>(__ldg(m + j * x.smj)), sum[0]);
      sum[1] = fmaf(to_f32<T>(h[j]), to_f32<T>(__ldg(m + next + j * x.smj)), sum[1]);
    }
  }
}

template <typename T, bool UP, bool KMAJOR>
__global__ void __launch_bounds__(THREADS, 1)
ft_stream_kernel(const __grid_constant__ CUtensorMap tmap, const StreamParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* ring = smem_raw + (((raw + 1023u) & ~1023u) - raw);      // the ring first: boxes start on the swizzle's period
  uint8_t* rest = ring + p.ring_bytes;
  Plan* plan = reinterpret_cast<Plan*>(rest);
  uint8_t* token = rest + sizeof(Plan);                              // token of every listed slot (T <= 128)
  uint64_t* bars = reinterpret_cast<uint64_t*>(token + MAX_R);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * MAX_STAGES);
  int* joined = reinterpret_cast<int*>(bars + 2 * MAX_STAGES) + 1;
  float* per_slot = reinterpret_cast<float*>(bars + 2 * MAX_STAGES + 2);  // the listed slots' parts of the gate (or, as integers, adapters)
  float* sums = per_slot + MAX_R;                                    // down: [warp][T][rows + 1]; up: the warps' accumulators
  const int pitch = p.rows + 1;
  const Args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (MAX_STAGES + s); };

  if (tid == 0) {
    for (int s = 0; s < p.ring.stages; ++s) {
      mbar_init(full_bar(s), LOADERS + GATHER_THREADS);      // the weights (expect_tx) and the gatherers' threads
      mbar_init(empty_bar(s), UP ? CONSUMERS : CONSUMERS / DOWN_TURNS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap);
  }
  if (UP) {
    // ids and gates come from the kernel before when it is the router; an adapter's shrink only from there on (see below)
    if (!p.ext.ids) wait_for_previous_kernel();
    let_next_kernel_start();
    if (blockIdx.x == 0)
      for (int i = tid; i < p.n_counters; i += THREADS) p.counters[i] = 0;
  }
  // ids and gates are older than the up-projection, so the down-projection plans before it waits
  make_plan(plan, ring, a.ids, a.sit, a.sik, a.T, a.k, a.E, p.NT);
  const int listed = plan->jobs ? plan->job_begin[plan->jobs - 1] + plan->job_count[plan->jobs - 1] : 0;
  for (int i = tid; i < listed; i += THREADS) {
    const int slot = plan->slots[i], t = slot / a.k;
    token[i] = static_cast<uint8_t>(t);
    if (UP && p.ext.ids) {      // the row's adapter
      const int64_t id = p.ext.ids[t];
      per_slot[i] = __int_as_float(id >= 0 && id < p.ext.n ? static_cast<int>(id) : -1);
    } else {
      const float gate = a.gates ? load_any(a.gates, t * a.sgt + (slot - t * a.k) * a.sgk, a.gates_dtype) : 1.f;
      per_slot[i] = UP ? carried(gate) : rest_of(gate);
    }
  }
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
  const bool woven = pairs && a.act_layout == LAYOUT_GPT_OSS;
  const bool halves = !KMAJOR && pairs && !woven;      // N-major: a box is 32 columns of one half and 32 of the other

  if (warp >= CONSUMERS && warp < CONSUMERS + LOADERS) {
    // ---------------- weights: they depend on no kernel before, so nothing is waited for -----------------------------
    if (lane != 0) return;
    const int mine = warp - CONSUMERS;
    Run r;
    RingPos at;
    bool ok = true;
    while (walk.next(r) && ok) {
      const int e = plan->job_expert[r.job];
      shape_of<UP, KMAJOR>(p, r, plan->job_count[r.job]);
      for (int b = r.b0; b < r.b1; b += r.nb, at.next(p.ring.stages)) {
        const int s = at.stage, steps = min(r.nb, r.b1 - b);
        if (!mbar_wait(empty_bar(s), at.phase ^ 1, abort_flag, p.status, 21)) { ok = false; break; }
        mbar_arrive_expect_tx(full_bar(s), ((UP ? r.boxes * steps : steps) - mine + LOADERS - 1) / LOADERS * p.load_bytes);
        uint32_t to = ring0 + s * p.ring.stage_bytes;
        int v = r.p0, i = mine;
        for (int t = 0; t < r.boxes; ++t, i -= steps, to += r.nb * p.box_bytes, v += UP ? (KMAJOR ? 1 : 2) * walk.per_tile : 0)
          for (; i < steps; i += LOADERS) {
            const uint32_t dst = to + i * p.box_bytes;
            const int kk = (b + i) * BLOCK_K;
            // K-major: (K, value, column of the value, expert). N-major: (column, half, K, expert).
            if (KMAJOR) tma_load_4d(dst, &tmap, full_bar(s), kk, v, 0, e);
            else tma_load_4d(dst, &tmap, full_bar(s), woven ? 2 * v : v, 0, kk, e);
            if (halves) tma_load_4d(dst + 4096, &tmap, full_bar(s), v, 1, kk, e);
          }
      }
    }
    if (!ok)      // give copies already in flight time to land before the block goes away
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    return;
  }
  if (warp >= CONSUMERS + LOADERS) {
    // ---------------- the slots' rows: 16 bytes per thread, zeros beyond K ---------------------------------------------
    if (!UP) wait_for_previous_kernel();
    const int g = tid - (CONSUMERS + LOADERS) * 32, turn = g / GATHER_THREADS;
    const int chunk = g & 7, row0 = (g % GATHER_THREADS) >> 3;                          // rows row0, row0 + 8, ...
    static_assert(GATHER_THREADS == 64, "eight rows at a time");
    const uint32_t mine = row0 * 128 + static_cast<uint32_t>((chunk ^ row0) << 4);      // row & 7 == row0
    Run r;
    RingPos at;
    bool ok = true;
    while (walk.next(r) && ok) {
      const int n = plan->job_count[r.job], beg = plan->job_begin[r.job];
      shape_of<UP, KMAJOR>(p, r, n);
      const int x_block = r.groups * 1024;
      const uint8_t* src[4];
      bool have = false;
      for (int b = r.b0; b < r.b1; b += r.nb, at.next(p.ring.stages)) {
        const int s = at.stage, steps = min(r.nb, r.b1 - b);
        if ((s & (GATHER_TURNS - 1)) != turn) continue;
        if (!have) {
          have = true;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row0 + 8 * i < n) {
              const int j = beg + row0 + 8 * i;
              src[i] = UP ? static_cast<const uint8_t*>(a.X) + static_cast<int64_t>(token[j]) * a.sxm * 2
                          : p.hidden + static_cast<int64_t>(plan->slots[j]) * a.F * 2;
            }
        }
        if (!mbar_wait(empty_bar(s), at.phase ^ 1, abort_flag, p.status, 23)) { ok = false; break; }
        const uint32_t dst = ring0 + s * p.ring.stage_bytes + r.x_offset + mine;
        const int k0 = b * BLOCK_K + chunk * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row0 + 8 * i < n) {
            uint32_t to = dst + i * 1024;
            int kk = k0;
            for (int st = 0; st < steps; ++st, kk += BLOCK_K, to += x_block)
              cp_async16(to, src[i] + (kk < p.K ? kk * 2 : 0), kk < p.K ? 16 : 0);
          }
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
  // down: the warp's half of the tile's columns, or (K-major, no more than 16 in all) its half of every box's K
  const bool by_columns = !UP && p.rows > 16;
  const int m0 = by_columns ? (warp & 1) * (KMAJOR ? 16 : 32) : 0;
  const int copies = by_columns ? CONSUMERS / 2 : CONSUMERS, copy = by_columns ? warp >> 1 : warp;
  // ldmatrix addresses of this lane inside a box and inside a step of the slots' rows; 16 of K further: see `step`
  uint32_t w_lane, w_lane1 = 0, x1_lane, x4_lane;
  {
    const int row = (lane & 7) + ((lane >> 3) & 1) * 8, xrow = (lane & 7) + (lane >> 4) * 8;
    const int krow = (lane & 7) + (lane >> 4) * 8, chunk = (lane >> 3) & 1;
    if (KMAJOR) {
      w_lane = (row + m0) * 128 + (((lane >> 4) ^ (row & 7)) << 4);
      w_lane1 = w_lane + 16 * 128;
    } else if (halves) {      // 64-byte rows, the warp's 16 columns of either half
      w_lane = krow * 64 + ((chunk ^ ((krow >> 1) & 3)) << 4);
      w_lane1 = w_lane + 4096;
    } else {                  // 128-byte rows, the warp's 32 columns
      w_lane = krow * 128 + (((chunk + (UP ? 0 : (warp & 1) * 4)) ^ (krow & 7)) << 4);
      w_lane1 = w_lane ^ 32;
    }
    x1_lane = (lane & 7) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
    x4_lane = xrow * 128 + ((((lane >> 3) & 1) ^ (xrow & 7)) << 4);
  }
  const int w_step = halves ? 1024 : 2048;
  while (walk.next(r)) {
    const int n = plan->job_count[r.job], beg = plan->job_begin[r.job], e = plan->job_expert[r.job];
    shape_of<UP, KMAJOR>(p, r, n);
    const int groups = r.groups, x_block = groups * 1024;
    // the warp's weight rows: up, a tile of the round (shared by `team` warps); down, its part of the one tile
    const int team = UP ? (r.tiles == 1 ? 8 : (r.tiles == 2 ? 4 : (r.tiles <= 4 ? 2 : 1))) : 1;
    const int tl = UP ? warp / team : 0, sub = UP ? warp - tl * team : 0;
    const int v0 = UP ? r.p0 + tl * walk.per_tile : r.p0;
    const int count = UP ? min(walk.per_tile, r.count - tl * walk.per_tile) : r.count;
    const uint32_t second_tile = UP && !KMAJOR ? (tl & 1) << (halves ? 5 : 6) : 0;       // N-major: which half of the box
    const bool use0 = count > m0, use1 = UP ? (pairs ? (woven && !KMAJOR ? count > 8 : use0) : count > 16) : count > m0 + 16;
    if (!UP && r.first && (!by_columns || !(warp & 1))) {
      for (int i = lane; i < a.T * pitch; i += 32) sums[copy * a.T * pitch + i] = 0.f;
    }
    if (!UP && r.first && by_columns) consumers_sync();        // a pair shares its sums
    constexpr int M = UP || !KMAJOR ? 2 : 1;                   // 16-row halves a warp multiplies
    float acc[M][4][4];
    bool mine = false;                                         // this warp has a part of the run
    auto stream = [&](auto G_) {
      constexpr int G = decltype(G_)::value;           // groups of 8 slots
      // independent accumulators for neighbouring steps: a chain of dependent products would leave the warp waiting
      constexpr int S = !UP && !KMAJOR ? (G == 1 ? 2 : 1) : (G == 1 ? 4 : (G == 2 ? 2 : 1));      // (registers)
      float part[S][M][G][4];
#pragma unroll
      for (int c = 0; c < S; ++c)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int q = 0; q < 4; ++q) part[c][m][g][q] = 0.f;
      for (int b = r.b0; b < r.b1; b += r.nb, at.next(p.ring.stages)) {
        const int s = at.stage;
        if (!UP && (s & (DOWN_TURNS - 1)) != (warp >> 1)) continue;
        mine = true;
        if (ok) ok = mbar_wait_warp(full_bar(s), at.phase, abort_flag, p.status, 22);
        if (ok && use0) {
          const int steps = min(r.nb, r.b1 - b);
          uint32_t w = ring0 + s * p.ring.stage_bytes + (UP ? (KMAJOR ? tl : tl >> 1) * r.nb * p.box_bytes : 0), x = ring0 + s * p.ring.stage_bytes + r.x_offset;
          auto step = [&](int i, float (&to)[M][G][4]) {       // the i-th 16 of K of a box
            uint32_t a0[4], a1[4], bx[G + 1][2];
            if (KMAJOR) {
              ldsm4(a0, w + (w_lane ^ (i << 5)));
              if (M == 2 && use1) ldsm4(a1, w + (w_lane1 ^ (i << 5)));
            } else {
              ldsm4_trans(a0, w + (w_lane ^ second_tile) + i * w_step);
              if (M == 2 && use1) ldsm4_trans(a1, w + (w_lane1 ^ second_tile) + i * w_step);
            }
            if (G == 1) {
              ldsm2(bx[0][0], bx[0][1], x + (x1_lane ^ (i << 5)));
            } else {
#pragma unroll
              for (int g = 0; g < G; g += 2) {
                uint32_t t[4];
                ldsm4(t, x + (x4_lane ^ (i << 5)) + g * 1024);
                bx[g][0] = t[0]; bx[g][1] = t[1]; bx[g + 1][0] = t[2]; bx[g + 1][1] = t[3];
              }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              Mma<T>::run(to[0][g], a0, bx[g][0], bx[g][1]);
              if (M == 2 && use1) Mma<T>::run(to[M - 1][g], a1, bx[g][0], bx[g][1]);
            }
          };
          if (UP || by_columns) {
            w += sub * p.box_bytes;
            x += sub * x_block;
            for (int i = sub; i < steps; i += team, w += team * p.box_bytes, x += team * x_block) {
#pragma unroll
              for (int q = 0; q < 4; ++q) step(q, part[q % S]);
            }
          } else {
            for (int i = 0; i < steps; i += 2) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (i + h < steps) {
                  step((warp & 1) * 2, part[(h * 2) % S]);
                  step((warp & 1) * 2 + 1, part[(h * 2 + 1) % S]);
                  w += p.box_bytes;
                  x += x_block;
                }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar(s));
      }
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v = part[0][m][g][q];
#pragma unroll
            for (int c = 1; c < S; ++c) v += part[c][m][g][q];
            acc[m][g][q] = v;
          }
    };
    if (groups == 1) stream(std::integral_constant<int, 1>{});
    else if (groups == 2) stream(std::integral_constant<int, 2>{});
    else if (groups == 3) stream(std::integral_constant<int, 3>{});
    else stream(std::integral_constant<int, 4>{});

    if (UP) {
      // The sums go through shared memory, where the warps of a tile meet (each then takes every team-th value of all) and where a
      // short loop can pick them up: unrolled over the registers the epilogue outgrew the instruction cache (10 us and more).
      float* red = sums;
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g < groups) {
#pragma unroll
            for (int q = 0; q < 4; ++q) red[(warp * 32 + (m * 4 + g) * 4 + q) * 32 + lane] = acc[m][g][q];
          }
      if (team > 1) consumers_sync(); else __syncwarp();
      if (p.ext.ids) wait_for_previous_kernel();      // the rank rows of the extension
      // accumulator q of group g: slot g*8 + 2*(lane & 3) + (q & 1), weight row (lane >> 2) + 8*(q >> 1) of each 16-row half
      if (use0) {
#pragma unroll 1
        for (int idx = sub; idx < groups * 4; idx += team) {
          const int g = idx >> 2, q = idx & 3;
          const int i = g * 8 + (lane & 3) * 2 + (q & 1), row = (lane >> 2) + (q >> 1) * 8;
          float c[2][2] = {{0.f, 0.f}, {0.f, 0.f}};       // (first, second column) of up to two values
          for (int w = 0; w < team; ++w) {
            const float* part = red + ((tl * team + w) * 32 + idx) * 32 + lane;
            c[0][0] += part[0];
            c[0][1] += part[16 * 32];
          }
          int v[2] = {row, -1};
          if (!pairs) {
            c[1][0] = c[0][1];
            v[1] = 16 + row;
          } else if (woven && !KMAJOR) {      // columns side by side: the second one sits in the neighbouring row's lane
            const float o0 = __shfl_xor_sync(0xffffffffu, c[0][0], 4), o1 = __shfl_xor_sync(0xffffffffu, c[0][1], 4);
            c[1][0] = c[0][1]; c[1][1] = o1; c[0][1] = o0;
            v[0] = (row & 1) ? -1 : row >> 1;
            v[1] = (row & 1) ? -1 : 8 + (row >> 1);
          }
          if (i >= n) continue;
          const int slot = plan->slots[beg + i];
          const float gate = p.ext.ids ? 1.f : per_slot[beg + i];
          float extra[2] = {0.f, 0.f};
          if (p.ext.ids && v[0] < count)
            extension_terms<T>(p.ext, slot, __float_as_int(per_slot[beg + i]), v0 + v[0], v[1] < count, extra);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (v[h] < 0 || v[h] >= count) continue;
            const int pv = v0 + v[h];
            float c0 = c[h][0], c1 = c[h][1];
            if (a.B1) {
              const T* bias = static_cast<const T*>(a.B1) + e * a.sb1e;
              c0 += to_f32<T>(bias[(woven ? 2 * pv : pv) * a.sb1n]);
              if (pairs) c1 += to_f32<T>(bias[(woven ? 2 * pv + 1 : a.F + pv) * a.sb1n]);
            }
            c0 += extra[h];
            reinterpret_cast<T*>(p.hidden)[static_cast<int64_t>(slot) * a.F + pv] =
                from_f32<T>(gate * hidden_fast(a.act_layout, a.act, a.alpha, a.limit, c0, c1));
          }
        }
      }
      if (team > 1) consumers_sync(); else __syncwarp();
    } else {
      // add the job's slots to this warp's token sums. Slots of one token (the same expert twice) stand together and may sit in
      // neighbouring lanes: then the lanes take turns
      if (mine && use0) {
        float* own = sums + copy * a.T * pitch + m0;       // the second 16 columns (N-major) follow 16 further
        const bool twice = __any_sync(0xffffffffu, lane > 0 && lane < n && token[beg + min(lane, n - 1)] == token[beg + min(lane, n - 1) - (lane > 0)]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (g >= groups) continue;
#pragma unroll
          for (int m = 0; m < M; ++m) {
            float* to[4];
            float gate[4];
            bool in[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int i = g * 8 + (lane & 3) * 2 + (q & 1), row = m * 16 + (lane >> 2) + (q >> 1) * 8;
              to[q] = own + token[beg + min(i, n - 1)] * pitch + row;
              gate[q] = per_slot[beg + min(i, n - 1)];
              in[q] = i < n && m0 + row < count;
            }
            if (!twice) {      // all different: read, add, write
              float v[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = in[q] ? *to[q] : 0.f;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (in[q]) *to[q] = fmaf(gate[q], acc[m][g][q], v[q]);
            } else {
              for (int turn = 0; turn < 4; ++turn) {
                if ((lane & 3) == turn) {
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    if (in[q]) *to[q] = fmaf(gate[q], acc[m][g][q], *to[q]);
                }
                __syncwarp();
              }
            }
          }
        }
        __syncwarp();
      }
      if (r.last) {
        consumers_sync();
        constexpr int DT = Walker<UP, KMAJOR>::DOWN_TILE;
        bool write = true;
        auto total_of = [&](int t, int col) {
          float v = 0.f;
          for (int w = 0; w < copies; ++w) v += sums[(w * a.T + t) * pitch + col];
          return v;
        };
        int first = 0, stop = 0, tile_beg = 0, total = 1;
        const int g = static_cast<int>(gridDim.x);
        auto begin_of = [&](int b) { return part_begin(total, b, p.part_step); };
        bool split = false;
        if (!KMAJOR) {
          // does this block hold the whole tile, or only a part of its steps?
          tile_beg = r.tile * walk.units;
          const int tile_end = tile_beg + walk.units;
          total = walk.units * ((a.d_out + DT - 1) / DT);
          const int mine0 = begin_of(blockIdx.x), mine1 = begin_of(blockIdx.x + 1);
          split = mine0 > tile_beg || mine1 < tile_end;
          if (split) {
            float* part = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (mine0 > tile_beg ? 0 : 1)) * a.T * DT;
            for (int i = tid; i < a.T * r.count; i += CONSUMERS * 32) part[(i / r.count) * DT + i % r.count] = total_of(i / r.count, i % r.count);
            __threadfence();
            consumers_sync();
            first = static_cast<int>(static_cast<int64_t>(tile_beg) * g / total);
            while (first > 0 && begin_of(first) > tile_beg) --first;
            while (begin_of(first + 1) <= tile_beg) ++first;
            int parts = 0;
            for (stop = first; stop < g && begin_of(stop) < tile_end; ++stop) parts += begin_of(stop + 1) > begin_of(stop);
            if (tid == 0) *joined = atomicAdd(p.counters + r.tile, 1) == parts - 1;
            consumers_sync();
            write = *joined != 0;      // the last block of the tile adds the parts up, always in the same order
            if (write) __threadfence();
          }
        }
        if (write)
          for (int idx = tid; idx < a.T * r.count; idx += CONSUMERS * 32) {
            const int t = idx / r.count, col = idx - t * r.count;
            float v = 0.f;
            if (split) {
              for (int b = first; b < stop; ++b)
                if (begin_of(b + 1) > begin_of(b))
                  v += __ldcg(p.partial + ((static_cast<int64_t>(b) * 2 + (begin_of(b) > tile_beg ? 0 : 1)) * a.T + t) * DT + col);
            } else {
              v = total_of(t, col);
            }
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
static int column_tiles(int d_out) { return cdiv(d_out, 2 * TILE); }
size_t stream_workspace_bytes(int64_t T, int k, int F, int d_out) {
  return hidden_bytes(T, k, F) + static_cast<size_t>(column_tiles(d_out)) * 4 + 16 + static_cast<size_t>(MAX_CTAS) * 2 * T * 2 * TILE * 4;
}

struct Order { bool k_major, n_major; };
// Experts that share one matrix (stride 0 of a broadcast view) are left to the CUDA cores: a tensor map's strides are not to be zero.
static Order weight_order(const void* W, int E, int64_t se, int64_t sk, int64_t sn, int K, int N) {
  if (!al16(W) || se % 8 || se < 0 || (se == 0 && E > 1)) return {false, false};
  return {sk == 1 && sn % 8 == 0 && sn >= K, sn == 1 && sk % 8 == 0 && sk >= N && N % 8 == 0};
}

// Boxes of one expert, 128-byte swizzle: 64 of K x `rows` x `halves` (the two columns of a hidden value; 1 without a gate).
static bool encode_k_major(CUtensorMap* map, bool bf16, const void* W, int K, int values, int64_t value_stride, int halves,
                           int64_t half_stride, int E, int64_t se, int rows) {
  const uint64_t dim[4] = {static_cast<uint64_t>(K), static_cast<uint64_t>(values), static_cast<uint64_t>(halves), static_cast<uint64_t>(E)};
  // the stride of an axis of one element is never used, but has to be valid
  const uint64_t stride[3] = {static_cast<uint64_t>(value_stride) * 2, static_cast<uint64_t>(halves > 1 ? half_stride : value_stride) * 2,
                              static_cast<uint64_t>(E > 1 ? se : value_stride) * 2};
  const uint32_t box[4] = {BLOCK_K, static_cast<uint32_t>(rows), static_cast<uint32_t>(halves), 1};
  return encode_tensor_map(map, bf16, W, 4, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Boxes of one expert: 64 columns x 64 of K, 128-byte swizzle; where the two columns of a hidden value are a half apart, 32 columns of one
// half x 64 of K, 64-byte swizzle.
static bool encode_n_major(CUtensorMap* map, bool bf16, const void* W, int N, int K, int64_t row_stride, int halves, int E, int64_t se) {
  const uint64_t dim[4] = {static_cast<uint64_t>(N / halves), static_cast<uint64_t>(halves), static_cast<uint64_t>(K), static_cast<uint64_t>(E)};
  const uint64_t stride[3] = {static_cast<uint64_t>(halves > 1 ? N / 2 : row_stride) * 2, static_cast<uint64_t>(row_stride) * 2,
                              static_cast<uint64_t>(E > 1 ? se : row_stride) * 2};
  const uint32_t box[4] = {static_cast<uint32_t>(2 * TILE / halves), 1, BLOCK_K, 1};
  // a row of a box is one 128-byte line; asking L2 for two (as the K-major boxes do, whose next step is the other one) read 25-40 % more
  // from HBM than was used
  return encode_tensor_map(map, bf16, W, 4, dim, stride, box, halves > 1 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

// rows of a K-major box of the down-projection: the output columns of a block, at most a tile
static int down_rows(int d_out, int grid) { return cdiv(d_out, grid) < TILE ? cdiv(d_out, grid) : TILE; }

template <typename T, bool UP, bool KMAJOR>
static int launch_one(StreamParams p, const CUtensorMap& map, const DeviceInfo& di, int grid) {
  const Args& a = p.a;
  p.rows = UP ? 0 : (KMAJOR ? down_rows(a.d_out, grid) : 2 * TILE);
  // shared memory that is not the ring
  const int fixed = static_cast<int>(sizeof(Plan)) + MAX_R + (2 * MAX_STAGES + 2) * 8 + MAX_R * 4 +
                    (UP ? CONSUMERS * 32 * 32 * 4 : (p.rows > 16 ? CONSUMERS / 2 : CONSUMERS) * a.T * (p.rows + 1) * 4) + 1024 + 64;
  const int budget = (di.max_smem_optin < 232448 ? di.max_smem_optin : 232448) - fixed;
  const int rows = KMAJOR ? (UP ? TILE : p.rows) : 2 * TILE;
  p.load_bytes = rows * BLOCK_K * 2;
  p.box_bytes = cdiv(rows, 8) * 1024;                      // boxes start on the swizzle's period
  p.blocks = cdiv(p.K, BLOCK_K);
  constexpr int TURNS = UP ? GATHER_TURNS : DOWN_TURNS;
  static_assert(4 % TURNS == 0, "every stage belongs to the same warps in every pass");
  if (!make_stages(&p.ring, UP, budget, p.box_bytes, p.blocks, a.T, a.k, TURNS)) return SMOE_ERR_UNSUPPORTED;
  p.ring_bytes = p.ring.stages * p.ring.stage_bytes + RING_SLACK;
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
  cfg.numAttrs = (!UP || a.after_router || p.ext.ids) ? 1 : 0;
  SMOE_CUDA(cudaLaunchKernelEx(&cfg, ft_stream_kernel<T, UP, KMAJOR>, map, p));
  return SMOE_OK;
}

template <typename T>
static int launch_typed(const Args& a, const DeviceInfo& di) {
  const int n_up_cols = n_up(a);
  const Order o1 = weight_order(a.W1, a.E, a.s1e, a.s1k, a.s1n, a.d, n_up_cols), o2 = weight_order(a.W2, a.E, a.s2e, a.s2k, a.s2n, a.F, a.d_out);
  if (!(o1.k_major || o1.n_major) || !(o2.k_major || o2.n_major)) return SMOE_ERR_UNSUPPORTED;
  const bool bf16 = a.dtype == SMOE_BF16;
  StreamParams p;
  p.a = a;
  memset(&p.ext, 0, sizeof(p.ext));
  p.hidden = static_cast<uint8_t*>(a.ws);
  uint8_t* after = static_cast<uint8_t*>(a.ws) + hidden_bytes(a.T, a.k, a.F);
  p.n_counters = column_tiles(a.d_out);
  p.counters = reinterpret_cast<int*>(after);
  p.partial = reinterpret_cast<float*>(after + (static_cast<size_t>(p.n_counters) * 4 + 15) / 16 * 16);
  p.status = a.status;
  p.NT = 32;
  const int grid = di.sm_count < MAX_CTAS ? di.sm_count : MAX_CTAS;
  p.part_step = static_cast<uint32_t>(((1ull << 32) + grid - 1) / grid);
  CUtensorMap m1, m2;
  memset(&m1, 0, sizeof(m1));
  memset(&m2, 0, sizeof(m2));
  const bool pairs = a.act_layout != LAYOUT_PLAIN, woven = a.act_layout == LAYOUT_GPT_OSS;
  const bool ok1 = o1.k_major ? encode_k_major(&m1, bf16, a.W1, a.d, a.F, woven ? 2 * a.s1n : a.s1n, pairs ? 2 : 1,
                                               woven ? a.s1n : a.s1n * a.F, a.E, a.s1e, pairs ? TILE / 2 : TILE)
                              : encode_n_major(&m1, bf16, a.W1, n_up_cols, a.d, a.s1k, pairs && !woven ? 2 : 1, a.E, a.s1e);
  const bool ok2 = o2.k_major ? encode_k_major(&m2, bf16, a.W2, a.F, a.d_out, a.s2n, 1, 0, a.E, a.s2e, down_rows(a.d_out, grid))
                              : encode_n_major(&m2, bf16, a.W2, a.d_out, a.F, a.s2k, 1, a.E, a.s2e);
  if (!ok1 || !ok2) return SMOE_ERR_UNSUPPORTED;
  p.K = a.d;
  if (int rc = o1.k_major ? launch_one<T, true, true>(p, m1, di, grid) : launch_one<T, true, false>(p, m1, di, grid)) return rc;
  p.K = a.F;
  return o2.k_major ? launch_one<T, false, true>(p, m2, di, grid) : launch_one<T, false, false>(p, m2, di, grid);
}

// The up-projection kernel as a linear of a few tokens (one expert, no activation) whose values take up an adapter's term. `ws` is the
// result (T, F), contiguous.
template <typename T>
static int launch_linear_typed(const Args& a, const Extension& ext, const DeviceInfo& di) {
  const Order o = weight_order(a.W1, 1, 0, a.s1k, a.s1n, a.d, a.F);
  if (!o.k_major && !o.n_major) return SMOE_ERR_UNSUPPORTED;
  const bool bf16 = a.dtype == SMOE_BF16;
  StreamParams p;
  p.a = a;
  p.ext = ext;
  p.hidden = static_cast<uint8_t*>(a.ws);
  p.partial = nullptr;
  p.counters = nullptr;
  p.n_counters = 0;
  p.status = a.status;
  p.NT = 32;
  const int grid = di.sm_count < MAX_CTAS ? di.sm_count : MAX_CTAS;
  p.part_step = static_cast<uint32_t>(((1ull << 32) + grid - 1) / grid);
  p.K = a.d;
  CUtensorMap map;
  const bool ok = o.k_major ? encode_k_major(&map, bf16, a.W1, a.d, a.F, a.s1n, 1, 0, 1, 0, TILE)
                            : encode_n_major(&map, bf16, a.W1, a.F, a.d, a.s1k, 1, 1, 0);
  if (!ok) return SMOE_ERR_UNSUPPORTED;
  return o.k_major ? launch_one<T, true, true>(p, map, di, grid) : launch_one<T, true, false>(p, map, di, grid);
}

int launch_linear(const Args& a, const Extension& ext) {
  if ((a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) || a.T > MAX_T) return SMOE_ERR_UNSUPPORTED;
  if (a.d % 8 || a.sxm % 8 || !al16(a.X) || static_cast<int64_t>(a.T) * cdiv(a.F, TILE) >= (int64_t(1) << 30)) return SMOE_ERR_UNSUPPORTED;
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  return a.dtype == SMOE_BF16 ? launch_linear_typed<__nv_bfloat16>(a, ext, di) : launch_linear_typed<__half>(a, ext, di);
}

int launch_stream(const Args& a) {
  if (a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) return SMOE_ERR_UNSUPPORTED;
  if (a.d % 8 || a.F % 8 || a.sxm % 8 || !al16(a.X)) return SMOE_ERR_UNSUPPORTED;
  {      // the lists of tiles and of steps of K are counted in 32 bits
    const int64_t jobs = static_cast<int64_t>(a.T) * a.k, most = int64_t(1) << 30;
    if (jobs * cdiv(a.F, TILE / 2) >= most || jobs * cdiv(a.F, BLOCK_K) * cdiv(a.d_out, TILE) >= most) return SMOE_ERR_UNSUPPORTED;
  }
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  return a.dtype == SMOE_BF16 ? launch_typed<__nv_bfloat16>(a, di) : launch_typed<__half>(a, di);
}

}  // namespace ft
}  // namespace smoe
