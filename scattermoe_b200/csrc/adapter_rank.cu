// The rank-sized products of the low-rank adapters on tensor cores (16-bit, mma.sync): the shrink H = s X M^T of many tokens and the
// per-adapter sums of outer products. Both are bound by reading their wide operand once (X, or x / dy): one 16-wide side keeps
// the tensor pipe far below its limit.
#include <mutex>
#include <type_traits>

#include "adapter.cuh"
#include "ptx.cuh"

namespace smoe {
namespace ad {

using namespace ptx;

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---- shrink --------------------------------------------------------------------------------------------------------
// A block owns 32 tokens: consecutive ones, or, where the caller has sorted the rows by adapter, consecutive sorted ones. Its eight warps
// take 64 of the contracted axis each, in turn, every warp with a ring of its own (cp.async, two to four stages), and are joined
// once at the end. A pass multiplies up to 64 columns: the rank rows of as many of the block's adapters as the ring holds (a
// block whose tokens share an adapter needs one pass). X comes from HBM in the first pass, from L2 in others.
constexpr int SH_MAX_SMEM = 226 * 1024;      // 1 KB less than a block can have: the static arrays
constexpr int SH_TOKENS = 32, SH_COLS = 64, SH_K = 64;
constexpr int SH_SMALL_RING = 13 * 1024;      // per warp: two blocks fit an SM

// padded against bank conflicts, but for the shortest rows: two of them then fit beside each other on an SM
__host__ __device__ inline int rank_row_bytes(int cols) { return cols <= 16 ? cols * 2 : cols * 2 + 16; }

struct ShrinkParams {
  ShrinkArgs a;
  int k_major;       // M has the contracted axis contiguous
  int m_vec;         // and 16-byte pieces of it can be copied
  int per_pass;      // adapters of a pass
  int width;         // columns an adapter takes in a pass (the rank, or a part of it, rounded up to 8)
  int ring_bytes;    // of one warp
};

template <typename T>
__global__ void __launch_bounds__(256)
shrink_tc_kernel(const ShrinkParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t chosen[8];
  const ShrinkArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * SH_TOKENS;
  __shared__ int32_t token[SH_TOKENS];
  int rows = static_cast<int>(min(static_cast<int64_t>(SH_TOKENS), a.T - t0));
  const int64_t pitch = rank_pitch(a.r);
  uint32_t id = 0xffffffffu;
  if (lane < rows) {
    const int64_t v = a.ids[t0 + lane];
    if (v >= 0 && v < a.n) id = static_cast<uint32_t>(v);
  }
  T* H = static_cast<T*>(a.H);
  const unsigned bare = __ballot_sync(0xffffffffu, lane < rows && id == 0xffffffffu);
  for (int i = tid; i < rows * static_cast<int>(pitch); i += 256) {        // rows without an adapter, and the padding
    const int t = i / static_cast<int>(pitch), j = i % static_cast<int>(pitch);
    if ((bare >> t & 1u) || j >= a.r) H[(t0 + t) * pitch + j] = from_f32<T>(0.f);
  }
  if (a.sorted_idx) {        // from here on the block's rows are sorted ones
    const int64_t live = min(a.offsets[a.n - 1], a.T);
    rows = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(SH_TOKENS), live - t0)));
    const int64_t t = lane < rows ? a.sorted_idx[t0 + lane] : 0;
    id = lane < rows ? static_cast<uint32_t>(a.ids[t]) : 0xffffffffu;
    if (warp == 0) token[lane] = static_cast<int32_t>(t);
  } else if (warp == 0) {
    token[lane] = static_cast<int32_t>(lane < rows ? t0 + lane : 0);
  }
  const uint32_t ring = smem_u32(smem) + warp * p.ring_bytes;
  uint8_t* ring_ptr = smem + warp * p.ring_bytes;
  const uint8_t* X = static_cast<const uint8_t*>(a.X);
  const uint8_t* M = static_cast<const uint8_t*>(a.M);
  uint32_t from = 0;
  for (;;) {
    // the next adapters of the block, ascending
    int adapters = 0;
    for (; adapters < p.per_pass; ++adapters) {
      const uint32_t e = __reduce_min_sync(0xffffffffu, id != 0xffffffffu && id >= from ? id : 0xffffffffu);
      if (e == 0xffffffffu) break;
      if (tid == 0) chosen[adapters] = e;
      from = e + 1;
    }
    if (adapters == 0) break;
    __syncthreads();
    for (int j0 = 0; j0 < a.r; j0 += p.width) {
      const int cols = adapters * p.width, groups = cols >> 3;
      const int m_pitch = rank_row_bytes(cols);  // M with the rank contiguous: bytes of a row in shared memory
      const int stage_bytes = SH_TOKENS * 128 + (p.k_major ? (groups + 1) / 2 * 2048 : SH_K * m_pitch);
      float acc[2][8][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int g = 0; g < 8; ++g)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[m][g][q] = 0.f;
      // what a lane copies is fixed but for the step of the contracted axis: addresses are made once
      const int chunk = lane & 7, pieces = cols >> 3;
      const uint8_t* x_row[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = (lane >> 3) + i * 4;
        x_row[i] = row < rows ? X + (static_cast<int64_t>(token[row]) * a.sxm + chunk * 8) * 2 : nullptr;
      }
      const uint8_t* m_base = M + (static_cast<int64_t>(chosen[0]) * a.sma + static_cast<int64_t>(j0) * a.smj) * 2;
      const int piece0 = lane % pieces, c_first = lane / pieces, c_step = 32 / pieces, piece_step = 32 - c_step * pieces;
      // column -> its adapter's place in `chosen` and its rank row
      auto adapter_of = [&](int col) { return adapters == 1 ? 0 : col / p.width; };
      auto load = [&](int s, int k0) {
        const uint32_t dst = ring + s * stage_bytes;
        const bool in_k = k0 + chunk * 8 < a.C;
#pragma unroll
        for (int i = 0; i < 8; ++i) {          // 32 token rows of 128 bytes
          const int row = (lane >> 3) + i * 4;
          const bool v = in_k && x_row[i] != nullptr;
          cp_async16(dst + row * 128 + ((chunk ^ (row & 7)) << 4), v ? x_row[i] + k0 * 2 : X, v ? 16 : 0);
        }
        const uint32_t dm = dst + SH_TOKENS * 128;
        uint8_t* dm_ptr = ring_ptr + s * stage_bytes + SH_TOKENS * 128;
        if (p.k_major) {                       // a row per column: 64 of the contracted axis
          for (int col = lane >> 3; col < cols; col += 4) {
            const int ad = adapter_of(col), in = col - ad * p.width;
            const bool live = j0 + in < a.r;
            const uint8_t* src = (ad == 0 ? m_base : M + (static_cast<int64_t>(chosen[ad]) * a.sma + static_cast<int64_t>(j0) * a.smj) * 2) +
                                 (in * a.smj + k0 + chunk * 8) * 2;
            const uint32_t at = col * 128 + ((chunk ^ (col & 7)) << 4);
            if (p.m_vec) {
              const bool v = in_k && live;
              cp_async16(dm + at, v ? src : M, v ? 16 : 0);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint16_t*>(dm_ptr + at)[i] =
                    live && k0 + chunk * 8 + i < a.C ? __ldg(reinterpret_cast<const uint16_t*>(src) + i) : 0;
            }
          }
        } else if (p.m_vec) {                  // a row per step of the contracted axis: the adapters' pieces of the rank
          int c = c_first, piece = piece0;
          while (c < SH_K) {
            const int col = piece * 8, ad = adapter_of(col), in = col - ad * p.width;
            const bool v = k0 + c < a.C && j0 + in < a.r;
            const uint8_t* src = ad == 0 ? m_base : M + (static_cast<int64_t>(chosen[ad]) * a.sma + j0) * 2;
            cp_async16(dm + c * m_pitch + col * 2, v ? src + (static_cast<int64_t>(k0 + c) * a.smc + in) * 2 : M, v ? 16 : 0);
            c += c_step;
            piece += piece_step;
            if (piece >= pieces) { piece -= pieces; ++c; }
          }
        } else {
          for (int i = lane; i < SH_K * cols; i += 32) {
            const int c = i / cols, col = i - c * cols, ad = adapter_of(col), j = j0 + col - ad * p.width;
            *reinterpret_cast<uint16_t*>(dm_ptr + c * m_pitch + col * 2) =
                k0 + c < a.C && j < a.r
                    ? __ldg(reinterpret_cast<const uint16_t*>(M) + static_cast<int64_t>(chosen[ad]) * a.sma +
                            static_cast<int64_t>(k0 + c) * a.smc + static_cast<int64_t>(j) * a.smj) : 0;
          }
        }
        cp_async_commit();
      };
      // One loop in which the loads run `stages - 1` turns ahead of the products: with a copy of both for every depth, and the first
      // loads unrolled, the warps waited for instructions more than for data.
      constexpr int TURN = 8 * SH_K;
      const int turns = a.C > warp * SH_K ? (a.C - warp * SH_K + TURN - 1) / TURN : 0;
      const int stages = min(4, p.ring_bytes / stage_bytes);
      int in = 0, out = 0;
#pragma unroll 1
      for (int i = 0; i < turns + stages - 1; ++i) {
        if (i < turns) {
          load(in, warp * SH_K + i * TURN);
          in = in + 1 == stages ? 0 : in + 1;
        } else {
          cp_async_commit();
        }
        if (i < stages - 1) continue;
        if (stages == 4) cp_async_wait<3>(); else if (stages == 3) cp_async_wait<2>(); else cp_async_wait<1>();
        __syncwarp();
        const uint32_t x = ring + out * stage_bytes, m = x + SH_TOKENS * 128;
        out = out + 1 == stages ? 0 : out + 1;
#pragma unroll 1
        for (int st = 0; st < SH_K / 16; ++st) {
          uint32_t af[2][4];
          const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
          const uint32_t at = x + row * 128 + (((st * 2 + (lane >> 4)) ^ (row & 7)) << 4);
          ldsm4(af[0], at);
          ldsm4(af[1], at + 16 * 128);
#pragma unroll
          for (int g = 0; g < 8; g += 2)
            if (g < groups) {
              uint32_t b[4];
              if (p.k_major) {
                const int col = (lane & 7) + (lane >> 4) * 8;
                ldsm4(b, m + (g * 8 + col) * 128 + (((st * 2 + ((lane >> 3) & 1)) ^ (col & 7)) << 4));
              } else {
                ldsm4_trans(b, m + (st * 16 + (lane & 15)) * m_pitch + (g * 8 + (lane >> 4) * 8) * 2);
              }
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) {
                mma16816<T>(acc[mt][g], af[mt], b[0], b[1]);
                if (g + 1 < groups) mma16816<T>(acc[mt][g + 1], af[mt], b[2], b[3]);
              }
            }
        }
        __syncwarp();
      }
      cp_async_wait<0>();
      __syncthreads();
      // join the warps: [warp][token][column]
      float* red = reinterpret_cast<float*>(smem);
      const int rp = cols + 1;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int g = 0; g < 8; ++g)
          if (g < groups) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              red[(warp * SH_TOKENS + mt * 16 + (lane >> 2) + (q >> 1) * 8) * rp + g * 8 + (lane & 3) * 2 + (q & 1)] = acc[mt][g][q];
          }
      __syncthreads();
      for (int i = tid; i < SH_TOKENS * cols; i += 256) {
        const int t = i / cols, col = i - t * cols, ad = col / p.width, j = j0 + col - ad * p.width;
        if (t >= rows || j >= a.r || a.ids[token[t]] != static_cast<int64_t>(chosen[ad])) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[(w * SH_TOKENS + t) * rp + col];
        H[token[t] * pitch + j] = from_f32<T>(v * (a.scaling ? a.scaling[chosen[ad]] : a.scale));
      }
      __syncthreads();
    }
  }
}

int launch_shrink_tc(const ShrinkArgs& a) {
  if (a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) return SMOE_ERR_UNSUPPORTED;
  if (a.C % 8 || a.sxm % 8 || !al16(a.X) || a.T >= (int64_t(1) << 31) - 64) return SMOE_ERR_UNSUPPORTED;
  ShrinkParams p;
  p.a = a;
  const int r8 = static_cast<int>(rank_pitch(a.r));
  p.width = r8 < SH_COLS ? r8 : SH_COLS;
  p.k_major = a.smc == 1 ? 1 : 0;
  const bool aligned = al16(a.M) && a.sma % 8 == 0;
  p.m_vec = aligned && (p.k_major ? a.smj % 8 == 0 : a.smj == 1 && a.smc % 8 == 0 && a.r % 8 == 0) ? 1 : 0;
  // Two stages of one adapter are the least. Where that is little the ring stays small enough for two blocks per SM, which is what
  // tokens in runs want; rows in no order (and not sorted) want as many adapters in a pass as fit.
  auto stage_of = [&](int cols) { return SH_TOKENS * 128 + (p.k_major ? cdiv(cols, 16) * 2048 : SH_K * rank_row_bytes(cols)); };
  const int one = 2 * stage_of(p.width);
  p.ring_bytes = one <= SH_SMALL_RING ? SH_SMALL_RING : (one > 20 * 1024 ? one : 20 * 1024);
  p.per_pass = 1;
  while (p.per_pass < 8 && (p.per_pass + 1) * p.width <= SH_COLS && 2 * stage_of((p.per_pass + 1) * p.width) <= p.ring_bytes) ++p.per_pass;
  p.ring_bytes = cdiv(p.ring_bytes, 128) * 128;
  const int cols = p.per_pass * p.width;
  const int ring = 8 * p.ring_bytes, red = 8 * SH_TOKENS * (cols + 1) * 4;
  const int smem = (ring > red ? ring : red) + 64;      // the last ldmatrix of an odd group reads 16 bytes past its row
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (smem > SH_MAX_SMEM || di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  static std::mutex mu;
  static bool configured[64] = {false};
  {
    std::lock_guard<std::mutex> lock(mu);
    if (di.device < 0 || di.device >= 64 || !configured[di.device]) {
      SMOE_CUDA(cudaFuncSetAttribute(shrink_tc_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SH_MAX_SMEM));
      SMOE_CUDA(cudaFuncSetAttribute(shrink_tc_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, SH_MAX_SMEM));
      if (di.device >= 0 && di.device < 64) configured[di.device] = true;
    }
  }
  const unsigned grid = static_cast<unsigned>(cdiv64(a.T, SH_TOKENS));
  if (a.dtype == SMOE_BF16) shrink_tc_kernel<__nv_bfloat16><<<grid, 256, smem, a.stream>>>(p);
  else shrink_tc_kernel<__half><<<grid, 256, smem, a.stream>>>(p);
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

// ---- outer products --------------------------------------------------------------------------------------------------
// D[a][j, c] = sum over the adapter's rows of U[t, j] V[t, c]. The adapter-sorted rows are cut into equal chunks; a block owns 128
// columns of V and up to 64 of the rank for one chunk and walks the adapters in it, 64 rows at a time (gathered by cp.async, four
// buffers). An adapter that lies in one chunk is written at once; one that spans chunks leaves fp32 parts (at most two per
// chunk: its first and its last adapter), which a second kernel adds up in the chunks' order. No atomics.
constexpr int GR_COLS = 128, GR_J = 64, GR_ROWS = 64, GR_STAGES = 4, GR_MAX_CHUNKS = 16;
constexpr int GR_V_PITCH = GR_COLS * 2 + 16, GR_U_PITCH = GR_J * 2 + 16;
constexpr int GR_STAGE = GR_ROWS * (GR_V_PITCH + GR_U_PITCH);
constexpr int GR_SMEM = GR_STAGES * GR_STAGE;

static int grad_chunks(int64_t T, int C, int r) {
  const int64_t by_grid = cdiv64(2 * SM_COUNT, static_cast<int64_t>(cdiv(C, GR_COLS)) * cdiv(r, GR_J)), by_rows = cdiv64(T, 256);
  const int64_t s = by_grid < by_rows ? by_grid : by_rows;
  return static_cast<int>(s < 1 ? 1 : (s > GR_MAX_CHUNKS ? GR_MAX_CHUNKS : s));
}
size_t grad_workspace_bytes(int64_t T, int C, int r) { return static_cast<size_t>(grad_chunks(T, C, r)) * 2 * r * C * 4 + 16; }

struct GradParams {
  GradArgs a;
  int chunks;
  float* parts;      // [chunk][first, last], each in the order of D: (r, C), or (C, r) where D has the rank contiguous
  int by_rank;       // the latter
};

template <typename T>
__global__ void __launch_bounds__(256)
grad_tc_kernel(const GradParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const GradArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c0 = blockIdx.x * GR_COLS, j0 = blockIdx.y * GR_J;
  const int nj = min(GR_J, static_cast<int>(rank_pitch(a.r)) - j0), groups = nj >> 3;
  const int64_t live = min(a.offsets[a.n - 1], a.T);
  const int64_t per = cdiv64(cdiv64(live, p.chunks), GR_ROWS) * GR_ROWS;
  const int64_t m0 = min(live, per * blockIdx.z), m1 = min(live, m0 + per);
  if (m0 >= m1) return;
  int e = 0;
  for (int lo = 0, hi = a.n - 1; lo < hi;) {         // first adapter whose rows end after m0
    const int mid = (lo + hi) >> 1;
    if (a.offsets[mid] > m0) hi = mid; else lo = mid + 1;
    e = lo;
  }
  const uint32_t ring = smem_u32(smem);
  const int64_t u_pitch = rank_pitch(a.r);
  const uint8_t* V = static_cast<const uint8_t*>(a.V);
  const uint8_t* U = static_cast<const uint8_t*>(a.U);
  for (int64_t beg = m0; beg < m1; ++e) {
    const int64_t all_beg = e ? a.offsets[e - 1] : 0, all_end = a.offsets[e], end = min(m1, all_end);
    if (end <= beg) continue;
    float acc[8][4];
#pragma unroll
    for (int g = 0; g < 8; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[g][q] = 0.f;
    const int tiles = static_cast<int>((end - beg + GR_ROWS - 1) / GR_ROWS);
    // the rows of the next tile to load: their numbers are fetched a tile early, or every copy would wait for them
    int32_t next_row[GR_ROWS / 16];
    auto fetch_rows = [&](int i) {
#pragma unroll
      for (int q = 0; q < GR_ROWS / 16; ++q) {
        const int64_t m = beg + static_cast<int64_t>(i) * GR_ROWS + (tid >> 4) + q * 16;
        next_row[q] = m < end ? static_cast<int32_t>(a.sorted_idx[m]) : -1;
      }
    };
    auto load = [&](int i) {
      const uint32_t dst = ring + (i % GR_STAGES) * GR_STAGE;
      const int chunk = tid & 15;
#pragma unroll
      for (int q = 0; q < GR_ROWS / 16; ++q) {
        const int row = (tid >> 4) + q * 16;
        const bool in = next_row[q] >= 0;
        const int64_t t = in ? next_row[q] : 0;
        const bool v = in && c0 + chunk * 8 < a.C;
        cp_async16(dst + row * GR_V_PITCH + chunk * 16, V + (v ? (t * a.svm + c0 + chunk * 8) * 2 : 0), v ? 16 : 0);
        if (chunk < groups)
          cp_async16(dst + GR_ROWS * GR_V_PITCH + row * GR_U_PITCH + chunk * 16, U + (in ? (t * u_pitch + j0 + chunk * 8) * 2 : 0), in ? 16 : 0);
      }
      cp_async_commit();
      fetch_rows(i + 1);
    };
    fetch_rows(0);
#pragma unroll 1
    for (int ahead = 0; ahead < tiles + GR_STAGES - 1; ++ahead) {      // the loads run GR_STAGES - 1 tiles ahead
      if (ahead >= GR_STAGES) __syncthreads();                         // everyone has read the buffer that comes next
      if (ahead < tiles) load(ahead); else cp_async_commit();
      const int i = ahead - (GR_STAGES - 1);
      if (i < 0) continue;
      cp_async_wait<GR_STAGES - 1>();
      __syncthreads();
      const uint32_t v = ring + (i % GR_STAGES) * GR_STAGE, u = v + GR_ROWS * GR_V_PITCH;
#pragma unroll 2
      for (int st = 0; st < GR_ROWS / 16; ++st) {
        uint32_t af[4];          // 16 columns of V (the M side) x 16 rows
        ldsm4_trans(af, v + (st * 16 + (lane & 7) + (lane >> 4) * 8) * GR_V_PITCH + (warp * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
        for (int g = 0; g < 8; g += 2)
          if (g < groups) {
            uint32_t b[4];
            ldsm4_trans(b, u + (st * 16 + (lane & 15)) * GR_U_PITCH + (g * 8 + (lane >> 4) * 8) * 2);
            mma16816<T>(acc[g], af, b[0], b[1]);
            if (g + 1 < groups) mma16816<T>(acc[g + 1], af, b[2], b[3]);
          }
      }
    }
    cp_async_wait<0>();
    __syncthreads();
    const bool whole = all_beg >= m0 && all_end <= m1;
    float* part = p.parts + (static_cast<int64_t>(blockIdx.z) * 2 + (all_beg < m0 ? 0 : 1)) * a.r * a.C;
#pragma unroll
    for (int g = 0; g < 8; ++g)
      if (g < groups) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = c0 + warp * 16 + (lane >> 2) + (q >> 1) * 8, j = j0 + g * 8 + (lane & 3) * 2 + (q & 1);
          if (c >= a.C || j >= a.r) continue;
          if (whole) static_cast<T*>(a.D)[e * a.sda + j * a.sdj + c * a.sdc] = from_f32<T>(acc[g][q]);
          else part[p.by_rank ? static_cast<int64_t>(c) * a.r + j : static_cast<int64_t>(j) * a.C + c] = acc[g][q];
        }
      }
    beg = end;
  }
}

// Adapters without rows get zeros, adapters that span chunks the sum of their parts.
template <typename T>
__global__ void __launch_bounds__(256)
grad_join_kernel(const GradParams p) {
  const GradArgs& a = p.a;
  const int e = blockIdx.z;
  const int64_t live = a.T ? min(a.offsets[a.n - 1], a.T) : 0;
  const int64_t beg = e ? a.offsets[e - 1] : 0, end = a.offsets[e];
  const int64_t per = cdiv64(cdiv64(live, p.chunks), GR_ROWS) * GR_ROWS;
  int z0 = 0, z1 = -1;
  if (end > beg) {
    z0 = static_cast<int>(beg / per);
    z1 = static_cast<int>((end - 1) / per);
    if (z0 == z1) return;             // written by the first kernel
  }
  const int64_t total = static_cast<int64_t>(a.r) * a.C;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    float v = 0.f;
    for (int z = z0; z <= z1; ++z) v += p.parts[(static_cast<int64_t>(z) * 2 + (beg < z * per ? 0 : 1)) * total + i];
    const int64_t inner = p.by_rank ? a.r : a.C;
    const int64_t outer_i = total < (int64_t(1) << 31) ? static_cast<uint32_t>(i) / static_cast<uint32_t>(inner) : i / inner;
    const int64_t inner_i = i - outer_i * inner, j = p.by_rank ? inner_i : outer_i, c = p.by_rank ? outer_i : inner_i;
    static_cast<T*>(a.D)[e * a.sda + j * a.sdj + c * a.sdc] = from_f32<T>(v);
  }
}

int launch_grad_tc(const GradArgs& a) {
  if (a.dtype != SMOE_BF16 && a.dtype != SMOE_F16) return SMOE_ERR_UNSUPPORTED;
  if (a.C % 8 || a.svm % 8 || !al16(a.V) || !al16(a.U) || !al16(a.ws)) return SMOE_ERR_UNSUPPORTED;
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  if (di.cc_major != 10) return SMOE_ERR_UNSUPPORTED;
  GradParams p;
  p.a = a;
  p.chunks = grad_chunks(a.T, a.C, a.r);
  p.parts = static_cast<float*>(a.ws);
  p.by_rank = a.sdj == 1 && a.sdc != 1 ? 1 : 0;
  static std::mutex mu;
  static bool configured[64] = {false};
  {
    std::lock_guard<std::mutex> lock(mu);
    if (di.device < 0 || di.device >= 64 || !configured[di.device]) {
      SMOE_CUDA(cudaFuncSetAttribute(grad_tc_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, GR_SMEM));
      SMOE_CUDA(cudaFuncSetAttribute(grad_tc_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, GR_SMEM));
      if (di.device >= 0 && di.device < 64) configured[di.device] = true;
    }
  }
  const bool bf16 = a.dtype == SMOE_BF16;
  if (a.T > 0) {
    dim3 grid(static_cast<unsigned>(cdiv(a.C, GR_COLS)), static_cast<unsigned>(cdiv(a.r, GR_J)), static_cast<unsigned>(p.chunks));
    if (bf16) grad_tc_kernel<__nv_bfloat16><<<grid, 256, GR_SMEM, a.stream>>>(p);
    else grad_tc_kernel<__half><<<grid, 256, GR_SMEM, a.stream>>>(p);
    SMOE_LAUNCH_CHECK();
  }
  const int64_t values = static_cast<int64_t>(a.r) * a.C;
  dim3 grid(static_cast<unsigned>(cdiv64(values, 256) < 256 ? cdiv64(values, 256) : 256), 1, static_cast<unsigned>(a.n));
  if (bf16) grad_join_kernel<__nv_bfloat16><<<grid, 256, 0, a.stream>>>(p);
  else grad_join_kernel<__half><<<grid, 256, 0, a.stream>>>(p);
  SMOE_LAUNCH_CHECK();
  return SMOE_OK;
}

}  // namespace ad
}  // namespace smoe
