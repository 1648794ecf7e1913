// Shared projection with the adapters' expansion in the same accumulators (16-bit, tcgen05):
//
//   Y[t, o] = sum_c X[t, c] W[c, o] + bias[o] + sum_j H[t, j] M[a(t)][j, o]
//
// A persistent 128 x BN GEMM (TMA -> shared-memory ring -> tcgen05.mma -> tensor memory, double-buffered) whose K loop goes on after W: for
// every adapter that occurs among the tile's 128 rows, up to 64 of the rank are one more stage. Four warps build it: the rows of H
// that name the adapter, zeros for the others (so a row only meets its own adapter), and the adapter's slice
// of M, both in a swizzled layout of the ring. (Zero times infinity is not zero: infinities and NaN of M are left out of the product
// and added by the epilogue to the rows they belong to, so that one broken adapter leaves its neighbours' rows alone.) One instruction of 16 per stage at rank 16: the expansion adds 1/256 of the product at
// C = 4096 where a tile's rows share an adapter, and the output is neither read back nor rounded twice.
// Bound: the tensor cores.
#include <cuda.h>

#include <mutex>

#include "adapter.cuh"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace smoe {
namespace ad {

using namespace ptx;

constexpr int BM = 128, BK = 64, UMMA_K = 16;
constexpr int GEMM_THREADS = 320;      // warp 0 TMA, warp 1 MMA + tensor memory, warps 2-5 extension, warps 6-9 epilogue
constexpr int A_BYTES = BM * BK * 2;

template <int BN> struct GemmCfg {
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int SMEM = 1024 + STAGES * (A_BYTES + B_BYTES) + 256 + 64;
  static_assert(SMEM <= 232448, "over the shared memory a block can have");
};

struct GemmParams {
  const uint8_t* H; int64_t h_row_bytes;
  const uint8_t* M; int64_t sma, smj, smo;
  const int64_t* ids;
  const uint8_t* bias;
  uint8_t* Y; int64_t y_row_bytes;
  int64_t T;
  int n, C, O, r, is_bf16, m_pieces, wide_rows, group_m;
  uint32_t idesc, idesc_ext;
  int32_t* status;
};

// how M is read: element by element, 16-byte pieces of the rank (of a column), or 8 columns (of a rank row)
enum { PIECES_NONE = 0, PIECES_RANK = 1, PIECES_COLUMNS = 2 };

struct OutTile { int64_t t0; int rows, o0; };

// The row tiles are walked in groups of group_m, all column tiles of a group before the next group.
template <int BN>
__device__ __forceinline__ OutTile out_tile(const GemmParams& p, int t, int m_tiles, int n_tiles) {
  const int per_group = p.group_m * n_tiles;
  const int grp = t / per_group, in = t - grp * per_group;
  const int gw = min(p.group_m, m_tiles - grp * p.group_m);
  const int nt = in / gw, mt = grp * p.group_m + (in - nt * gw);
  OutTile tl;
  tl.t0 = static_cast<int64_t>(mt) * BM;
  tl.rows = static_cast<int>(min(static_cast<int64_t>(BM), p.T - tl.t0));
  tl.o0 = nt * BN;
  return tl;
}

// The adapters of a tile's rows in ascending order. Whole-warp calls; lane l holds the ids of rows 4l .. 4l+3.
struct AdapterWalk {
  uint32_t id[4];
  __device__ __forceinline__ void load(const GemmParams& p, const OutTile& tl, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = lane * 4 + i;
      const int64_t v = row < tl.rows ? p.ids[tl.t0 + row] : -1;
      id[i] = v >= 0 && v < p.n ? static_cast<uint32_t>(v) : 0xffffffffu;
    }
  }
  // smallest id >= from, 0xffffffff if none
  __device__ __forceinline__ uint32_t next(uint32_t from) const {
    uint32_t m = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (id[i] >= from) m = min(m, id[i]);
    return __reduce_min_sync(0xffffffffu, m);
  }
};

__device__ __forceinline__ uint32_t pack2(float a, float b, int is_bf16) {
  if (is_bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight 16-bit values: infinities and NaN become zeros; whether there were any.
__device__ __forceinline__ bool drop_not_finite(uint4& v, int is_bf16) {
  const uint32_t mask = is_bf16 ? 0x7f80u : 0x7c00u;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & mask) == mask) { w[i] &= 0xffff0000u; any = true; }
    if ((w[i] >> 16 & mask) == mask) { w[i] &= 0x0000ffffu; any = true; }
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
  return any;
}

__device__ __forceinline__ float to_float16bit(uint16_t raw, int is_bf16) {
  return is_bf16 ? __bfloat162float(__ushort_as_bfloat16(raw)) : __half2float(__ushort_as_half(raw));
}

// What the product left out for row t and column o: the terms of M that are not finite.
__device__ __noinline__ float not_finite_terms(const GemmParams& p, int64_t t, int64_t id, int o) {
  const uint32_t mask = p.is_bf16 ? 0x7f80u : 0x7c00u;
  float sum = 0.f;
  for (int j = 0; j < p.r; ++j) {
    const uint16_t m = __ldg(reinterpret_cast<const uint16_t*>(p.M) + id * p.sma + j * p.smj + o * p.smo);
    if ((m & mask) == mask)
      sum += to_float16bit(__ldg(reinterpret_cast<const uint16_t*>(p.H + t * p.h_row_bytes) + j), p.is_bf16) * to_float16bit(m, p.is_bf16);
  }
  return sum;
}

template <int BN, bool B_KMAJOR>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
adapter_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const GemmParams p) {
  using Cfg = GemmCfg<BN>;
  constexpr int STAGES = Cfg::STAGES, B_BYTES = Cfg::B_BYTES;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * (A_BYTES + B_BYTES));
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto build_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };       // the stage is free for the extension's builders
  auto tfull_bar = [&](int b) { return bar0 + 8u * (3 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (3 * STAGES + 2 + b); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 3 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((3 * STAGES + 4) * 8 + 8 <= 256, "the barriers do not fit");
  // entry i % 16: 1 + the block's last tile i whose extension met values of M that are not finite. The builders are at most
  // STAGES + 3 tiles ahead of the epilogue, so an entry is read before it is needed again.
  volatile int* not_finite = reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(bars) + 256);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int m_tiles = static_cast<int>((p.T + BM - 1) / BM), n_tiles = (p.O + BN - 1) / BN, total = m_tiles * n_tiles;
  const int num_kb = (p.C + BK - 1) / BK, rank_blocks = (p.r + BK - 1) / BK;
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);       // the TMA thread (expect_tx), or one builder
      mbar_init(empty_bar(s), 1);      // tcgen05.commit
      mbar_init(build_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 128);
    }
    *abort_flag = 0;
    for (int i = 0; i < 16; ++i) not_finite[i] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  struct Pos {
    int s = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next() { if (++s == STAGES) { s = 0; ph ^= 1; } }
  } at;

  if (warp == 0) {
    // ---------------- TMA -----------------------------------------------------------------------------------------
    bool ok = true;
    AdapterWalk walk;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const OutTile tl = out_tile<BN>(p, t, m_tiles, n_tiles);
      walk.load(p, tl, lane);
      for (int kb = 0; kb < num_kb; ++kb, at.next()) {
        if (!mbar_wait_warp(empty_bar(at.s), at.ph ^ 1, abort_flag, p.status, 31)) { ok = false; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(full_bar(at.s), A_BYTES + B_BYTES);
          tma_load_2d(smem_u32(sA + at.s * A_BYTES), &tmap_x, full_bar(at.s), kb * BK, static_cast<int>(tl.t0));
          const uint32_t dst = smem_u32(sB + at.s * B_BYTES);
          if (B_KMAJOR) {
            tma_load_2d(dst, &tmap_w, full_bar(at.s), kb * BK, tl.o0);
          } else {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) tma_load_2d(dst + j * (64 * BK * 2), &tmap_w, full_bar(at.s), tl.o0 + j * 64, kb * BK);
          }
        }
        __syncwarp();
      }
      for (uint32_t e = walk.next(0); ok && e != 0xffffffffu; e = walk.next(e + 1))
        for (int rb = 0; rb < rank_blocks; ++rb, at.next()) {
          if (!mbar_wait_warp(empty_bar(at.s), at.ph ^ 1, abort_flag, p.status, 32)) { ok = false; break; }
          if (lane == 0) mbar_arrive(build_bar(at.s));
          __syncwarp();
        }
    }
    if (!ok)      // give copies already in flight time to land before the block goes away
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    // ---------------- MMA issuer ---------------------------------------------------------------------------------
    bool ok = true;
    int tile_iter = 0;
    AdapterWalk walk;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++tile_iter) {
      const OutTile tl = out_tile<BN>(p, t, m_tiles, n_tiles);
      walk.load(p, tl, lane);
      const int buf = tile_iter & 1;
      if (!mbar_wait_warp(tempty_bar(buf), ((tile_iter >> 1) & 1) ^ 1, abort_flag, p.status, 33)) { ok = false; break; }
      tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + buf * BN;
      for (int kb = 0; kb < num_kb; ++kb, at.next()) {
        if (!mbar_wait_warp(full_bar(at.s), at.ph, abort_flag, p.status, 34)) { ok = false; break; }
        tc_fence_after_sync();
        if (lane == 0) {
          const uint32_t a_addr = smem_u32(sA + at.s * A_BYTES), b_addr = smem_u32(sB + at.s * B_BYTES);
#pragma unroll
          for (int j = 0; j < BK / UMMA_K; ++j) {
            const uint64_t adesc = make_smem_desc_sw128(a_addr + j * (UMMA_K * 2), 16, 1024);
            const uint64_t bdesc = B_KMAJOR ? make_smem_desc_sw128(b_addr + j * (UMMA_K * 2), 16, 1024)
                                            : make_smem_desc_sw128(b_addr + j * (UMMA_K * 128), 64 * BK * 2, 1024);
            umma_f16(d_tmem, adesc, bdesc, p.idesc, (kb | j) != 0 ? 1u : 0u);
          }
          umma_commit(empty_bar(at.s));
        }
        __syncwarp();
      }
      for (uint32_t e = walk.next(0); ok && e != 0xffffffffu; e = walk.next(e + 1))
        for (int rb = 0; rb < rank_blocks; ++rb, at.next()) {
          if (!mbar_wait_warp(full_bar(at.s), at.ph, abort_flag, p.status, 35)) { ok = false; break; }
          tc_fence_after_sync();
          if (lane == 0) {
            const uint32_t a_addr = smem_u32(sA + at.s * A_BYTES), b_addr = smem_u32(sB + at.s * B_BYTES);
            const int steps = (min(BK, p.r - rb * BK) + UMMA_K - 1) / UMMA_K;
            for (int j = 0; j < steps; ++j)
              umma_f16(d_tmem, make_smem_desc_sw128(a_addr + j * (UMMA_K * 2), 16, 1024),
                       p.m_pieces == PIECES_COLUMNS ? make_smem_desc_sw128(b_addr + j * (UMMA_K * 128), 64 * BK * 2, 1024)
                                                    : make_smem_desc_sw128(b_addr + j * (UMMA_K * 2), 16, 1024), p.idesc_ext, 1u);
            umma_commit(empty_bar(at.s));
          }
          __syncwarp();
        }
      if (ok && lane == 0) umma_commit(tfull_bar(buf));
      __syncwarp();
    }
  } else if (warp < 6) {
    // ---------------- extension: rows of H and of M into the ring ---------------------------------------------------
    const int row = tid - 64;
    // a wait that runs out does not leave the loops: the four warps' barrier stays matched
    bool ok = true;
    uint32_t passes = 0;             // bit s: parity of the next pass of build_bar(s)
    AdapterWalk walk;
    int tile_iter = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++tile_iter) {
      const OutTile tl = out_tile<BN>(p, t, m_tiles, n_tiles);
      walk.load(p, tl, lane);
      uint32_t mine = 0xffffffffu;
      if (row < tl.rows) {
        const int64_t v = p.ids[tl.t0 + row];
        if (v >= 0 && v < p.n) mine = static_cast<uint32_t>(v);
      }
      const uint4* h = reinterpret_cast<const uint4*>(p.H + (tl.t0 + row) * p.h_row_bytes);
      for (int kb = 0; kb < num_kb % STAGES; ++kb) at.next();      // the stages of W are not ours
      for (uint32_t e = walk.next(0); e != 0xffffffffu; e = walk.next(e + 1)) {
        const uint8_t* m = p.M + static_cast<int64_t>(e) * p.sma * 2;
        for (int rb = 0; rb < rank_blocks; ++rb, at.next()) {
          const int s = at.s, j0 = rb * BK, len = min(BK, p.r - j0), chunks = (len + UMMA_K - 1) / UMMA_K * 2;
          // Where M comes in 16-byte pieces everything is fetched before the wait, and at once (a piece at a time cost 3 us an
          // adapter). By rank: a thread holds two columns' rank rows, stored K-major. By column: 8 columns of one rank row, N-major.
          constexpr int PIECES = BN / 128 * 8;
          uint4 hv[8], mv[PIECES];
#pragma unroll
          for (int ch = 0; ch < 8; ++ch)            // H rows are padded to a multiple of 8 with zeros
            hv[ch] = mine == e && ch * 8 < len ? __ldg(h + j0 / 8 + ch) : make_uint4(0u, 0u, 0u, 0u);
          bool broken = false;
          if (p.m_pieces != PIECES_NONE) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              bool in;
              const uint8_t* src;
              if (p.m_pieces == PIECES_RANK) {
                const int o = (i >> 3) * 128 + row, ch = i & 7;
                in = tl.o0 + o < p.O && ch * 8 < len;
                src = m + (static_cast<int64_t>(tl.o0 + o) * p.smo + j0 + ch * 8) * 2;
              } else {
                const int idx = i * 128 + row, j = idx / (BN / 8), o = idx % (BN / 8) * 8;
                in = j < len && tl.o0 + o < p.O;
                src = m + (static_cast<int64_t>(j0 + j) * p.smj + tl.o0 + o) * 2;
              }
              mv[i] = in ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) broken |= drop_not_finite(mv[i], p.is_bf16);
          }
          if (ok) ok = mbar_wait_warp(build_bar(s), (passes >> s) & 1, abort_flag, p.status, 36);
          passes ^= 1u << s;
          if (ok) {
            uint8_t* da = sA + s * A_BYTES + row * 128;
            uint8_t* sb = sB + s * B_BYTES;
#pragma unroll
            for (int ch = 0; ch < 8; ++ch)
              if (ch < chunks) *reinterpret_cast<uint4*>(da + ((ch ^ (row & 7)) << 4)) = hv[ch];
            if (p.m_pieces == PIECES_RANK) {
#pragma unroll
              for (int i = 0; i < PIECES; ++i) {
                const int o = (i >> 3) * 128 + row, ch = i & 7;
                if (ch < chunks) *reinterpret_cast<uint4*>(sb + o * 128 + ((ch ^ (o & 7)) << 4)) = mv[i];
              }
            } else if (p.m_pieces == PIECES_COLUMNS) {
#pragma unroll
              for (int i = 0; i < PIECES; ++i) {
                const int idx = i * 128 + row, j = idx / (BN / 8), c = idx % (BN / 8);      // 64 columns x 64 rank rows of 128 bytes each
                if (j < chunks * 8) *reinterpret_cast<uint4*>(sb + (c >> 3) * (64 * BK * 2) + j * 128 + (((c & 7) ^ (j & 7)) << 4)) = mv[i];
              }
            } else {
#pragma unroll 1
              for (int half = 0; half < BN / 128; ++half) {
                const int o = half * 128 + row;
                const bool in = tl.o0 + o < p.O;
                const uint8_t* src = m + (static_cast<int64_t>(tl.o0 + o) * p.smo + j0 * p.smj) * 2;
#pragma unroll 1
                for (int ch = 0; ch < chunks; ++ch) {
                  uint32_t w[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const int j = ch * 8 + 2 * i;
                    const uint32_t lo = in && j < len ? __ldg(reinterpret_cast<const uint16_t*>(src + j * p.smj * 2)) : 0u;
                    const uint32_t hi = in && j + 1 < len ? __ldg(reinterpret_cast<const uint16_t*>(src + (j + 1) * p.smj * 2)) : 0u;
                    w[i] = lo | hi << 16;
                  }
                  uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
                  broken |= drop_not_finite(v, p.is_bf16);
                  *reinterpret_cast<uint4*>(sb + o * 128 + ((ch ^ (o & 7)) << 4)) = v;
                }
              }
            }
          }
          if (broken) not_finite[tile_iter & 15] = tile_iter + 1;
          fence_proxy_async_smem();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (ok && row == 0) mbar_arrive(full_bar(s));
        }
      }
    }
  } else {
    // ---------------- epilogue: tensor memory -> bias -> 16 bits -> rows ----------------------------------------------
    const int q = warp & 3, r = q * 32 + lane;
    int tile_iter = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++tile_iter) {
      const OutTile tl = out_tile<BN>(p, t, m_tiles, n_tiles);
      const int buf = tile_iter & 1;
      if (!mbar_wait_warp(tfull_bar(buf), (tile_iter >> 1) & 1, abort_flag, p.status, 37)) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN;
      uint8_t* yrow = p.Y + (tl.t0 + r) * p.y_row_bytes;
      int64_t broken = -1;      // the row's adapter, where the tile met values that are not finite
      if (not_finite[tile_iter & 15] == tile_iter + 1 && r < tl.rows) {
        broken = p.ids[tl.t0 + r];
        if (broken >= p.n) broken = -1;
      }
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        const int o = tl.o0 + c * 32;
        if (o >= p.O) break;
        uint32_t acc[32];
        tmem_ld_32x32b_x32(taddr + c * 32, acc);
        tmem_ld_wait();
        uint4 out[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = __uint_as_float(acc[g * 8 + i]);
            if (p.bias) {
              const uint16_t b = __ldg(reinterpret_cast<const uint16_t*>(p.bias) + min(o + g * 8 + i, p.O - 1));
              v[i] += to_float16bit(b, p.is_bf16);
            }
            if (broken >= 0 && o + g * 8 + i < p.O) v[i] += not_finite_terms(p, tl.t0 + r, broken, o + g * 8 + i);
          }
          out[g] = make_uint4(pack2(v[0], v[1], p.is_bf16), pack2(v[2], v[3], p.is_bf16), pack2(v[4], v[5], p.is_bf16), pack2(v[6], v[7], p.is_bf16));
        }
        if (r < tl.rows) {
          if (p.wide_rows) {
#pragma unroll
            for (int g = 0; g < 4; g += 2)
              if (o + g * 8 < p.O) st_global_256(yrow + static_cast<int64_t>(o + g * 8) * 2, out[g], out[g + 1]);
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if (o + g * 8 < p.O) *reinterpret_cast<uint4*>(yrow + static_cast<int64_t>(o + g * 8) * 2) = out[g];
          }
        }
      }
      tc_fence_before_sync();
      mbar_arrive(tempty_bar(buf));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * BN);
}

static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int BN, bool B_KMAJOR>
static int launch_gemm(const CUtensorMap& w, const CUtensorMap& x, const GemmParams& p, int grid, const DeviceInfo& di, cudaStream_t stream) {
  static std::mutex mu;
  static bool configured[64] = {false};
  {
    std::lock_guard<std::mutex> lock(mu);
    if (di.device < 0 || di.device >= 64 || !configured[di.device]) {
      SMOE_CUDA(cudaFuncSetAttribute(adapter_gemm_kernel<BN, B_KMAJOR>, cudaFuncAttributeMaxDynamicSharedMemorySize, GemmCfg<BN>::SMEM));
      if (di.device >= 0 && di.device < 64) configured[di.device] = true;
    }
  }
  adapter_gemm_kernel<BN, B_KMAJOR><<<grid, GEMM_THREADS, GemmCfg<BN>::SMEM, stream>>>(w, x, p);
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

int launch_linear_tc(const LinearArgs& a) {
  if (a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) return SMOE_ERR_UNSUPPORTED;
  if (a.C % 8 || a.O % 8 || a.sxm % 8 || a.sxm < a.C || a.sym % 8 || !al16(a.X) || !al16(a.W) || !al16(a.Y) || !al16(a.H)) return SMOE_ERR_UNSUPPORTED;
  const bool k_major = a.swk == 1 && a.swn % 8 == 0 && a.swn >= a.C, n_major = a.swn == 1 && a.swk % 8 == 0 && a.swk >= a.O;
  if (!k_major && !n_major) return SMOE_ERR_UNSUPPORTED;
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  const int64_t m_tiles = cdiv64(a.T, BM);
  // 256 columns per tile feed the tensor cores better; 128 where the tiles then fill the last wave so much better that it pays
  const int64_t wave256 = cdiv64(m_tiles * cdiv(a.O, 256), di.sm_count) * 256, wave128 = cdiv64(m_tiles * cdiv(a.O, 128), di.sm_count) * 128;
  const int BN = a.O > 128 && wave256 * 10 <= wave128 * 11 ? 256 : 128;
  if (m_tiles * cdiv(a.O, BN) > (int64_t(1) << 30)) return SMOE_ERR_UNSUPPORTED;
  const bool bf16 = a.dtype == SMOE_BF16;
  CUtensorMap mw, mx;
  const uint64_t xd[2] = {static_cast<uint64_t>(a.C), static_cast<uint64_t>(a.T)}, xs[1] = {static_cast<uint64_t>(a.sxm) * 2};
  const uint32_t xb[2] = {BK, BM};
  if (!encode_tensor_map(&mx, bf16, a.X, 2, xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B)) return SMOE_ERR_UNSUPPORTED;
  const uint64_t wd[2] = {static_cast<uint64_t>(k_major ? a.C : a.O), static_cast<uint64_t>(k_major ? a.O : a.C)};
  const uint64_t ws[1] = {static_cast<uint64_t>(k_major ? a.swn : a.swk) * 2};
  const uint32_t wb[2] = {64, static_cast<uint32_t>(k_major ? BN : BK)};
  if (!encode_tensor_map(&mw, bf16, a.W, 2, wd, ws, wb, CU_TENSOR_MAP_SWIZZLE_128B)) return SMOE_ERR_UNSUPPORTED;
  GemmParams p;
  p.H = static_cast<const uint8_t*>(a.H); p.h_row_bytes = rank_pitch(a.r) * 2;
  p.M = static_cast<const uint8_t*>(a.M); p.sma = a.sma; p.smj = a.smj; p.smo = a.smo;
  p.ids = a.ids;
  p.bias = static_cast<const uint8_t*>(a.bias);
  p.Y = static_cast<uint8_t*>(a.Y); p.y_row_bytes = a.sym * 2;
  p.T = a.T; p.n = a.n; p.C = a.C; p.O = a.O; p.r = a.r; p.is_bf16 = bf16 ? 1 : 0;
  p.m_pieces = PIECES_NONE;
  if (a.sma % 8 == 0 && al16(a.M)) {
    if (a.smj == 1 && a.r % 8 == 0 && a.smo % 8 == 0) p.m_pieces = PIECES_RANK;
    else if (a.smo == 1 && a.smj % 8 == 0) p.m_pieces = PIECES_COLUMNS;
  }
  p.wide_rows = a.O % 16 == 0 && a.sym % 16 == 0 && (reinterpret_cast<uintptr_t>(a.Y) & 31) == 0 ? 1 : 0;
  // while the rows of X fit L2 beside W every row tile runs beside each column tile, else groups of 16
  p.group_m = static_cast<double>(a.T) * a.C * 2.0 <= 48e6 ? (1 << 20) : 16;
  if (p.group_m > m_tiles) p.group_m = static_cast<int>(m_tiles);
  p.idesc = make_idesc_f16(bf16, false, !k_major, BM, BN);
  p.idesc_ext = make_idesc_f16(bf16, false, p.m_pieces == PIECES_COLUMNS, BM, BN);
  p.status = a.status;
  const int64_t total = m_tiles * cdiv(a.O, BN);
  const int grid = static_cast<int>(total < di.sm_count ? total : di.sm_count);
  if (BN == 256) return k_major ? launch_gemm<256, true>(mw, mx, p, grid, di, a.stream) : launch_gemm<256, false>(mw, mx, p, grid, di, a.stream);
  return k_major ? launch_gemm<128, true>(mw, mx, p, grid, di, a.stream) : launch_gemm<128, false>(mw, mx, p, grid, di, a.stream);
}

}  // namespace ad
}  // namespace smoe
