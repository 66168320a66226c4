// y = x · w^T with fused epilogues, as persistent, warp-specialised tcgen05 kernels.
//
// Both kernels have one TMA producer warp (streams 64-wide K slices of x and w, bf16, 128-byte
// swizzle, through a shared-memory ring), one MMA warp (the whole warp walks the loop, an elected
// lane issues tcgen05.mma from shared memory into one of two 256-column fp32 accumulators in
// TMEM; tcgen05.commit releases ring slots and publishes finished accumulators) and epilogue
// warps that read their 32-lane TMEM quadrant with tcgen05.ld and apply bias / GELU /
// gate+residual in fp32.  Two accumulators let the epilogue of tile i overlap the main loop of
// tile i+1.
//
//   gemm_pair_kernel (default, 320 threads)  clusters of two CTAs share a 256x256 tile through
//               cta_group::2 MMAs; 5-stage ring of 32 KB per CTA; EIGHT epilogue warps in two
//               groups that take alternate 64-column pieces of a tile, each group with its own
//               swizzled staging tile, named barrier and TMA-store-issuing thread; up to four
//               problems per launch.  Second instantiation: the q|k|v head epilogue (QK RMS norm,
//               RoPE, head-major layout through a 5-D TMA store).
//   gemm_kernel (FLUXB_GEMM_PAIR=0, 192 threads)  one CTA per 128x256 tile, 4-stage ring of
//               48 KB, four epilogue warps, direct 16-byte stores.
//
// Tiles are handed out statically (tile = id + i * stride) in an L2-aware order (tile_coords).
// Edge tiles rely on TMA zero fill for loads and on TMA clipping / masks for stores.  Every
// barrier wait is bounded.
#include <stdio.h>
#include <stdlib.h>

#include "lora.cuh"

namespace fluxb {

namespace gemm {
constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 64;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK * 2;
constexpr int B_BYTES = BN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int THREADS = 192;
constexpr int TMEM_COLS = 512;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*alignment slack*/ + 256 /*barriers*/;

struct Params {
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  __nv_bfloat16* y2;
  const __nv_bfloat16* resid;
  const __nv_bfloat16* gate;
  int64_t ldy, ldy2, ldr, gate_stride, rows_per_batch;
  int M, N, K;
  int split, epi, epi2, round_before_act;
  int tiles_m, tiles_n, num_tiles;
  int pair_stages;  // CTA-pair kernel: ring depth in use (<= gemm2::STAGES)
  int raster_band_n, raster_group;  // tile order, see tile_coords
  DeviceStatus* status;
  // EPI_QKV_HEADS (CTA-pair kernel only): the N = 3*heads*128 columns are q | k | v of `heads`
  // heads; q and k rows are RMS-normalised per head with qk_scale[0/1] (if given) and rotated
  // with pe (if given), and everything is stored head-major through the 5-D map in tm_y.
  const float* pe;                     // [l_total, 64, 2, 2]
  const __nv_bfloat16* qk_scale[2];    // [128] each
  int row_offset, heads, l_total;      // joint position of this problem's first token
  float eps;
  // Scatter form of EPI_QKV_HEADS (scat_groups > 0): head h of q goes to
  // scat_base[h / scat_hpg] + b*scat_sb + (h % scat_hpg)*scat_sh + l*scat_sl, k and v scat_koff /
  // scat_voff elements further; the bases may be other GPUs' memory (plain 16-byte stores only).
  __nv_bfloat16* scat_base[8];
  int scat_groups, scat_hpg;
  int64_t scat_sb, scat_sh, scat_sl, scat_koff, scat_voff;
};
constexpr int EPI_QKV_HEADS = 3;  // internal epilogue code, set by fluxb_linear_qkv_grouped

// Tile order.  The tiles running at one time form a gm x gn rectangle of the output; all of
// them walk K in step, so each x row-block and w row-block is fetched from HBM once per
// rectangle and served from L2 to the others.  Across rectangles one operand is kept and the
// other swept:
//   band_n == 0: groups of `group` row-blocks of x are kept while all column-blocks are swept
//   band_n == 1: bands of `group` column-blocks (rows of w) are kept while x is swept
__device__ __forceinline__ void tile_coords(const Params& p, int tile, int tiles_m, int& m_blk, int& n_blk) {
  if (p.raster_band_n == 0) {
    const int per_group = p.raster_group * p.tiles_n;
    const int group = tile / per_group;
    const int first_m = group * p.raster_group;
    const int gsize = min(tiles_m - first_m, p.raster_group);
    const int in_group = tile - group * per_group;
    m_blk = first_m + in_group % gsize;
    n_blk = in_group / gsize;
  } else {
    const int per_band = p.raster_group * tiles_m;
    const int band = tile / per_band;
    const int first_n = band * p.raster_group;
    const int bsize = min(p.tiles_n - first_n, p.raster_group);
    const int in_band = tile - band * per_band;
    n_blk = first_n + in_band % bsize;
    m_blk = in_band / bsize;
  }
}

// Applies the epilogue to 32 consecutive columns of one output row held in registers.
// With `stage_row` == nullptr the 8-column pieces go straight to global memory with 16-byte
// stores.  Otherwise they go to this row's 128-byte line of a shared-memory staging tile in the
// 128-byte-swizzle layout (16-byte piece q of row r sits at ((q ^ (r & 7)) * 16), from where a
// TMA store writes full lines; `piece0` is the index of the first piece within the line.
__device__ __forceinline__ void epilogue_chunk(const Params& p, const uint32_t (&acc)[32], int row,
                                               int col0, bool second, uint8_t* stage_row = nullptr,
                                               int piece0 = 0, int swz = 0) {
  const int epi = second ? p.epi2 : p.epi;
  __nv_bfloat16* out = second ? p.y2 : p.y;
  const int64_t ld = second ? p.ldy2 : p.ldy;
  const int out_col0 = second ? col0 - p.split : col0;
  const bool row_ok = row < p.M;
  const int64_t b = (epi == FLUXB_EPI_GATE_RESID && row_ok) ? row / p.rows_per_batch : 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = col0 + j * 8;
    if (col >= p.N) break;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(acc[j * 8 + e]);
    if (p.bias != nullptr) {
      const uint4 bv = __ldg(reinterpret_cast<const uint4*>(p.bias + col));
      v[0] += bf16_lo(bv.x); v[1] += bf16_hi(bv.x); v[2] += bf16_lo(bv.y); v[3] += bf16_hi(bv.y);
      v[4] += bf16_lo(bv.z); v[5] += bf16_hi(bv.z); v[6] += bf16_lo(bv.w); v[7] += bf16_hi(bv.w);
    }
    if (epi == FLUXB_EPI_GELU) {
      if (p.round_before_act) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __bfloat162float(__float2bfloat16_rn(v[e]));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = gelu_tanh(v[e]);
    } else if (epi == FLUXB_EPI_GATE_RESID) {
      if (row_ok) {
        const uint4 rv = *reinterpret_cast<const uint4*>(p.resid + (int64_t)row * p.ldr + col);
        const uint4 gv = __ldg(reinterpret_cast<const uint4*>(p.gate + b * p.gate_stride + col));
        v[0] = bf16_lo(rv.x) + bf16_lo(gv.x) * v[0]; v[1] = bf16_hi(rv.x) + bf16_hi(gv.x) * v[1];
        v[2] = bf16_lo(rv.y) + bf16_lo(gv.y) * v[2]; v[3] = bf16_hi(rv.y) + bf16_hi(gv.y) * v[3];
        v[4] = bf16_lo(rv.z) + bf16_lo(gv.z) * v[4]; v[5] = bf16_hi(rv.z) + bf16_hi(gv.z) * v[5];
        v[6] = bf16_lo(rv.w) + bf16_lo(gv.w) * v[6]; v[7] = bf16_hi(rv.w) + bf16_hi(gv.w) * v[7];
      }
    }
    uint4 o;
    o.x = pack_bf16(v[0], v[1]); o.y = pack_bf16(v[2], v[3]);
    o.z = pack_bf16(v[4], v[5]); o.w = pack_bf16(v[6], v[7]);
    if (stage_row != nullptr) {
      *reinterpret_cast<uint4*>(stage_row + (((piece0 + j) ^ swz) << 4)) = o;  // rows/cols past the edge are clipped by the TMA store
    } else if (row_ok) {
      *reinterpret_cast<uint4*>(out + (int64_t)row * ld + out_col0 + j * 8) = o;
    }
  }
}

__global__ void __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
            const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_kb = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 128);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
        int m_blk, n_blk;
        tile_coords(p, tile, p.tiles_m, m_blk, n_blk);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 1)) { ok = false; break; }
          uint8_t* a_dst = smem + stage * STAGE_BYTES;
          uint8_t* b_dst = a_dst + A_BYTES;
          mbar_expect_tx(&full_bar[stage], STAGE_BYTES);
          tma_load_2d(a_dst, &tm_a, &full_bar[stage], kb * BK, m_blk * BM);
          tma_load_2d(b_dst, &tm_b, &full_bar[stage], kb * BK, n_blk * BN);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp walks the loop and an elected lane issues (warp-uniform descriptors).
    {
      constexpr uint32_t idesc = make_idesc_bf16(BM, BN, 0, 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int local = 0;
      for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x, ++local) {
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.status, 2))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 3))) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t a_addr = smem_u32(smem + stage * STAGE_BYTES);
          const uint64_t adesc = make_smem_desc(a_addr, 16, 1024);
          const uint64_t bdesc = make_smem_desc(a_addr + A_BYTES, 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              // 16 bf16 along K = 32 bytes = 2 descriptor address units
              umma_ss(d_tmem, adesc + 2 * k, bdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
            }
            umma_commit(&empty_bar[stage]);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok && elect_one()) umma_commit(&acc_full[acc]);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3;  // TMEM lane quadrant this warp may read
    int local = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x, ++local) {
      int m_blk, n_blk;
      tile_coords(p, tile, p.tiles_m, m_blk, n_blk);
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, 4)) { ok = false; break; }
      tc_fence_after_sync();
      const int row = m_blk * BM + quad * 32 + lane;
      const int n0 = n_blk * BN;
      const bool second = n0 >= p.split;
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        if (n0 + c * 32 >= p.N) break;  // uniform
        uint32_t r[32];
        tmem_ld_x32(t_addr + c * 32, r);
        tmem_wait_ld();
        epilogue_chunk(p, r, row, n0 + c * 32, second);
      }
      tc_fence_before_sync();
      mbar_arrive(&acc_empty[acc]);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace gemm

// ----------------------------------------------------------------------------------------
// CTA-pair variant: two CTAs of a cluster share one 256x256 output tile.  Each CTA loads its
// own 128 rows of x and only HALF of the w tile (128 rows); one thread of the even ("leader")
// CTA issues cta_group::2 MMAs (M=256, N=256, K=16) that run on both SMs, each tensor core
// reading the other half of w from its partner's shared memory.  Per SM this halves the
// shared-memory and L2 traffic for w, which is what bounds the single-CTA kernel.
//   - both CTAs' TMA loads count on the leader's "full" barrier (pair form of the bulk copy)
//   - slot release and accumulator-full are tcgen05.commit arrivals delivered to the barrier
//     at the same offset in BOTH CTAs, so each CTA's producer / epilogue waits locally
//   - accumulator-empty is counted on the leader (4 epilogue warps x 2 CTAs, remote arrive)
// (Relaying the slot release through the leader's producer with a remote mbarrier arrive
// instead was measured at half the throughput.)
// ----------------------------------------------------------------------------------------
namespace gemm2 {
using gemm::Params;
using gemm::epilogue_chunk;
using gemm::tile_coords;
constexpr int BM = 128;       // rows of x per CTA (256 per pair)
constexpr int BN = 256;       // output columns per tile
constexpr int BNH = 128;      // rows of w loaded by each CTA
constexpr int BK = 64;
constexpr int STAGES = 5;
constexpr int A_BYTES = BM * BK * 2;
constexpr int B_BYTES = BNH * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int OUT_CHUNK_COLS = 64;                       // output columns per staged TMA store
constexpr int OUT_BUF_BYTES = BM * OUT_CHUNK_COLS * 2;   // 128 rows x 128 bytes
constexpr int THREADS = 320;  // TMA warp, MMA warp, two groups of four epilogue warps
constexpr int TMEM_COLS = 512;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 2 * OUT_BUF_BYTES + 1024 + 256;
constexpr int MAX_PROBLEMS = 4;
constexpr int LORA_STAGES = 6;  // of kMode 3
constexpr int lora_smem(int cols) { return LORA_STAGES * (A_BYTES + cols / 2 * BK * 2) + 2 * OUT_BUF_BYTES + 1024 + 256; }

// Up to four GEMMs that differ in operands, outputs and row counts run as ONE persistent
// launch: their tiles are concatenated (problem 0's tiles first) and dealt round-robin to the
// CTA pairs.  A small problem (the 512-token text stream) would fill a third of the machine on
// its own; riding along with the image stream's GEMM it fills the tail of that launch instead.
struct Problem {
  CUtensorMap tm_a, tm_b;
  CUtensorMap tm_y, tm_y2;  // outputs (columns below / from `split`), box 64 columns x 128 rows
  Params p;
  int tile_start;  // index of this problem's first tile in the concatenated order
  int tiles_m;     // 256-row blocks
};
struct Grouped {
  Problem prob[MAX_PROBLEMS];
  int count;
  int total_tiles;
  int pair_stages;
};

static_assert(sizeof(Grouped) <= 4096, "kernel parameters are limited to 4 KB");

// One problem whose requests add low-rank adapters (kMode 3).
struct LoraGrouped {
  Problem prob[1];
  int count;
  int total_tiles;
  int pair_stages;
  CUtensorMap tm_t, tm_b;  // t [M, ld] box of one line x 128 rows, B [n, N, R] box of one group x 128 rows
  RequestAdapters req;
  LowRank low;
};

template <typename G>
__device__ __forceinline__ int find_problem(const G& g, int tile) {
  int i = 0;
#pragma unroll
  for (int k = 1; k < (int)(sizeof(g.prob) / sizeof(Problem)); ++k)
    if (k < g.count && tile >= g.prob[k].tile_start) i = k;
  return i;
}

// The adapters of a tile's W x 32 rows, as the producer warp finds them.  fetch() asks for the indices, well ahead of
// begin() and next(), so that nobody waits for them.  next() gives the adapter of the first row that is left, with the
// mask of the rows that do NOT use it (bit set: row left alone), or -1.  A tile inside one request, the ordinary case of
// long requests, is one index and an empty mask; else lane l holds rows l, 32 + l, ...
template <int W>
struct TileAdapters {
  int64_t raw[W];
  int a[W];
  int n_adapters;
  bool single;
  __device__ __forceinline__ void fetch(const RequestAdapters& req, int row0, int rows, int lane) {
    n_adapters = req.n_adapters;
    const int first = row0 / req.length;
    single = min(row0 + W * 32, rows) <= (first + 1) * (int64_t)req.length;
    if (single) {
      raw[0] = req.raw(first);
      return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int row = row0 + i * 32 + lane;
      raw[i] = row < rows ? req.raw(row / req.length) : -1;
    }
  }
  // What next() walks over, behind the K loop: the indices as 32-bit numbers, -1 for none.
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int i = 0; i < W; ++i) a[i] = raw[i] >= 0 && raw[i] < n_adapters ? (int)raw[i] : -1;
  }
  __device__ __forceinline__ int next(uint32_t (&off)[W]) {
    if (single) {
      const int cur = a[0];
      a[0] = -1;
#pragma unroll
      for (int i = 0; i < W; ++i) off[i] = 0;
      return cur;
    }
    uint32_t left = 0;
    int mine = -1;
#pragma unroll
    for (int i = W - 1; i >= 0; --i) {
      const uint32_t here = __ballot_sync(0xffffffffu, a[i] >= 0);
      if (here != 0) { left = here; mine = a[i]; }  // (the same word for all lanes)
    }
    if (left == 0) return -1;
    const int cur = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      off[i] = ~__ballot_sync(0xffffffffu, a[i] == cur);
      if (a[i] == cur) a[i] = -1;
    }
    return cur;
  }
};
// 32 accumulator columns of one row through bias and activation, packed to four 16-byte pieces.  The bias comes from
// shared memory, staged once per tile while the tile is still being multiplied: asked for eight columns at a time in the
// epilogue itself, each of those loads is waited for (8370 x 176 -> 5496, all epilogue: 75 us instead of 50).
__device__ __forceinline__ void finish32(const uint32_t (&acc)[32], const __nv_bfloat16* bias, int epi, uint4 (&out)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 b = *reinterpret_cast<const uint4*>(bias + j * 8);
    const uint32_t w[4] = {b.x, b.y, b.z, b.w};
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(acc[j * 8 + 2 * e]) + bf16_lo(w[e]);
      v[2 * e + 1] = __uint_as_float(acc[j * 8 + 2 * e + 1]) + bf16_hi(w[e]);
    }
    if (epi == FLUXB_EPI_GELU) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = gelu_tanh(v[e]);
    }
    out[j] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
}
__device__ __forceinline__ __nv_bfloat16 bias_at(const Params& p, int col) {
  return p.bias != nullptr && col < p.N ? p.bias[col] : __float2bfloat16_rn(0.f);
}
// What the producer leaves beside a ring slot for the MMA warp: of an adapter's slot the mask of the rows that it leaves
// alone, and of the last slot of a K loop and of every adapter's whether another adapter's slot follows.  The MMA warp
// reads it behind its wait for the slot (the producer's arrival there releases it) and so has nothing to find out.
struct SlotNote {
  uint32_t off[8];
  uint32_t more;
};
// A ring slot of the adapters: a line of t and a group of B; a group of 64 takes two (high parts, low parts).
__host__ __device__ __forceinline__ int lora_slots(const LowRank& low) { return low.group == 64 ? 2 * low.groups : low.groups; }

// Epilogue of one 128-row x 256-column tile (two heads of q, of k or of v) for EPI_QKV_HEADS:
// bias, rounding to bf16 (the projection's output precision in the reference), per-head RMS norm
// and rotation for q and k in fp32 with one rounding at the end, head-major 5-D TMA stores at
// (d, l, head, batch, part).  One thread of each epilogue group owns one row.  The row's sums of
// squares are taken in a first sweep over the accumulator (by both groups); in the second sweep
// a thread works 16 columns at a time for BOTH heads, because the rotation entries depend on
// the row and the pair only: each batch of eight pe entries is loaded once and used for the
// two heads.  The two groups take alternate 16-column steps; staging tile hh collects head hh
// from both groups and is stored by group hh's issuing thread.
__device__ __forceinline__ void qkv_load16(const Params& p, uint32_t taddr, int col, float (&x)[16]) {
  uint32_t r[16];
  tmem_ld_x16(taddr, r);
  tmem_wait_ld();
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(r[e]);
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 bv = __ldg(reinterpret_cast<const uint4*>(p.bias + col + j * 8));
      x[j * 8 + 0] += bf16_lo(bv.x); x[j * 8 + 1] += bf16_hi(bv.x); x[j * 8 + 2] += bf16_lo(bv.y); x[j * 8 + 3] += bf16_hi(bv.y);
      x[j * 8 + 4] += bf16_lo(bv.z); x[j * 8 + 5] += bf16_hi(bv.z); x[j * 8 + 6] += bf16_lo(bv.w); x[j * 8 + 7] += bf16_hi(bv.w);
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = __bfloat162float(__float2bfloat16_rn(x[e]));
}

template <bool kScatter>
__device__ __forceinline__ void qkv_tile_epilogue(const Params& p, const CUtensorMap* tm, uint32_t t_addr, int part,
                                                  int head0, int n0, int heads_in_tile, int b, int l0, int r_local,
                                                  bool rows_ok, uint8_t* out_stage, int eg, bool store_issuer,
                                                  int rows_left) {
  const __nv_bfloat16* w = part < 2 ? p.qk_scale[part] : nullptr;
  const bool rotate = part < 2 && p.pe != nullptr && rows_ok && (!kScatter || r_local < rows_left);
  float rstd0 = 1.f, rstd1 = 1.f;
  if (w != nullptr) {
#pragma unroll 1
    for (int hh = 0; hh < heads_in_tile; ++hh) {
      float ss = 0.f;
#pragma unroll 1
      for (int c = 0; c < 128; c += 16) {
        float x[16];
        qkv_load16(p, t_addr + hh * 128 + c, n0 + hh * 128 + c, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
      }
      const float r = rsqrtf(ss * (1.0f / 128.0f) + p.eps);
      if (hh == 0) rstd0 = r; else rstd1 = r;
    }
  }
  const float4* pr = reinterpret_cast<const float4*>(p.pe) + static_cast<int64_t>(l0 + r_local) * 64;
  // This group's four steps of 16 columns: steps eg and eg + 2 of each 64-column piece.  The pe
  // entries of the next step are requested before the current one is worked on.
  float4 f_next[8];
  if (rotate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f_next[i] = __ldg(pr + (eg * 16) / 2 + i);
  }
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int piece = it >> 1;
    const int step = eg + 2 * (it & 1);
    const int c = piece * 64 + step * 16;  // column within the head
    if ((it & 1) == 0) {
      // both staging tiles must have been read out by the stores of the piece before (each
      // issuer waits for its own), and nobody writes before both issuers are through
      if (store_issuer) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      asm volatile("bar.sync 3, 256;" ::: "memory");
    }
    float4 f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f_next[i];
    if (rotate && it < 3) {
      const int cn = ((it + 1) >> 1) * 64 + (eg + 2 * ((it + 1) & 1)) * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) f_next[i] = __ldg(pr + cn / 2 + i);
    }
#pragma unroll 1
    for (int hh = 0; hh < heads_in_tile; ++hh) {
      float x[16];
      qkv_load16(p, t_addr + hh * 128 + c, n0 + hh * 128 + c, x);
      if (w != nullptr) {
        const float r = hh == 0 ? rstd0 : rstd1;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 wv = __ldg(reinterpret_cast<const uint4*>(w + c + j * 8));
          x[j * 8 + 0] *= r * bf16_lo(wv.x); x[j * 8 + 1] *= r * bf16_hi(wv.x);
          x[j * 8 + 2] *= r * bf16_lo(wv.y); x[j * 8 + 3] *= r * bf16_hi(wv.y);
          x[j * 8 + 4] *= r * bf16_lo(wv.z); x[j * 8 + 5] *= r * bf16_hi(wv.z);
          x[j * 8 + 6] *= r * bf16_lo(wv.w); x[j * 8 + 7] *= r * bf16_hi(wv.w);
        }
      }
      if (rotate) {
        // pe[l, i] = {f00, f01, f10, f11}: out[2i] = f00 x[2i] + f01 x[2i+1], out[2i+1] = f10 x[2i] + f11 x[2i+1]
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a0 = x[2 * i], a1 = x[2 * i + 1];
          x[2 * i] = f[i].x * a0 + f[i].y * a1;
          x[2 * i + 1] = f[i].z * a0 + f[i].w * a1;
        }
      }
      uint8_t* line = out_stage + hh * OUT_BUF_BYTES + r_local * 128;
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const float* v = &x[jj * 8];
        uint4 o;
        o.x = pack_bf16(v[0], v[1]); o.y = pack_bf16(v[2], v[3]);
        o.z = pack_bf16(v[4], v[5]); o.w = pack_bf16(v[6], v[7]);
        *reinterpret_cast<uint4*>(line + (((step * 2 + jj) ^ (r_local & 7)) << 4)) = o;
      }
    }
    if ((it & 1) == 1) {
      fence_proxy_async_smem();
      asm volatile("bar.sync 3, 256;" ::: "memory");
      if (kScatter) {
        // All 256 epilogue threads copy the finished staging tiles out with plain 16-byte stores:
        // eight consecutive threads write one row's 128 bytes of one head.  The destination of a
        // head depends on its group (another GPU's arena under sequence parallelism), and rows
        // beyond the stream's end are skipped one by one, so stream lengths need not be
        // multiples of 128 here.  The barrier at the top of the next piece orders these reads
        // before the tiles are written again.
        const int tid = eg * 128 + r_local;
        const int64_t part_off = part == 0 ? 0 : (part == 1 ? p.scat_koff : p.scat_voff);
#pragma unroll 1
        for (int hh = 0; hh < heads_in_tile; ++hh) {
          const int head = head0 + hh;
          const int grp = head / p.scat_hpg;
          __nv_bfloat16* dst_head = p.scat_base[grp] + part_off + b * p.scat_sb + (head - grp * p.scat_hpg) * p.scat_sh +
                                    piece * 64;
          const uint8_t* src_tile = out_stage + hh * OUT_BUF_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int idx = tid + 256 * k;
            const int r = idx >> 3, q = idx & 7;
            if (r < rows_left) {
              const uint4 v = *reinterpret_cast<const uint4*>(src_tile + r * 128 + ((q ^ (r & 7)) << 4));
              *reinterpret_cast<uint4*>(dst_head + (int64_t)(l0 + r) * p.scat_sl + q * 8) = v;
            }
          }
        }
      } else
      // group eg's issuer stores staging tile eg = head eg of the tile
      if (store_issuer && rows_ok && eg < heads_in_tile) {
        asm volatile(
            "cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(
                reinterpret_cast<uint64_t>(tm)),
            "r"(smem_u32(out_stage + eg * OUT_BUF_BYTES)), "r"(piece * 64), "r"(l0), "r"(head0 + eg), "r"(b), "r"(part)
            : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  }
}

// kMode selects the epilogue at compile time, so that the ordinary kernel carries none of the other
// forms' code or register pressure:
//   0  ordinary (bias / GELU / gate+residual / column split)
//   1  q|k|v columns through the head epilogue, columns from `split` on ordinary
//   3  ordinary epilogue; behind the K loop of a tile the requests' adapters are added.  The low-rank
//      rows t = scale (x A^T), [M, R] in two bf16 parts (lora.cu), are K columns like any other: for
//      every adapter that the tile's rows use, the MMAs t_high B^T and t_low B^T accumulate into the
//      same TMEM tile through the same ring, with a lane mask that leaves the other requests' rows
//      alone (so a request never meets another one's adapter, not even as a product with zero).
//      Cost per adapter of a tile: one ring slot for ranks up to 32, two per 64 ranks for more, next to K / 64 of the
//      projection.
// kCols: output columns per tile.  Modes 0 to 2 have one width, 256; mode 3 takes a narrower one where that fills the
// machine better.
template <int kMode, typename G = Grouped, int kCols = BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_pair_kernel(const __grid_constant__ G g) {
  constexpr int kStages = kMode == 3 ? LORA_STAGES : STAGES;
  constexpr int kSlot = kMode == 3 ? A_BYTES + kCols / 2 * BK * 2 : STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* out_stage = smem + kStages * kSlot;  // two 16 KB output staging tiles
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(out_stage + 2 * OUT_BUF_BYTES);
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* acc_full = empty_bar + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  __shared__ SlotNote notes[kMode == 3 ? kStages : 1];  // (kMode 3 alone uses these two)
  __shared__ __align__(16) __nv_bfloat16 bias_s[2][kMode == 3 ? kCols : 8];
  static_assert(kMode == 3 ? kCols % 64 == 0 && kCols <= BN : kCols == BN, "one 64-column piece is staged at a time");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int num_tiles = g.total_tiles;
  DeviceStatus* const status = g.prob[0].p.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 16);  // one arrival per epilogue warp of both CTAs
    }
    *abort_flag = 0;
    mbar_fence_init();
    for (int i = 0; i < g.count; ++i) {
      tma_prefetch_desc(&g.prob[i].tm_a);
      tma_prefetch_desc(&g.prob[i].tm_b);
      tma_prefetch_desc(&g.prob[i].tm_y);
      tma_prefetch_desc(&g.prob[i].tm_y2);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // partner's barriers exist before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  if constexpr (kMode == 3) pdl_release();

  if (kMode == 3 && warp == 0) {
    if constexpr (kMode == 3) {
      // As below, with the whole warp walking the tiles: the adapters of a tile are found by ballots.
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const Problem& pr = g.prob[0];
      const Params& p = pr.p;
      const int num_kb = (p.K + BK - 1) / BK;
      // The next tile's coordinates and indices are taken while the current one's loads are under way: between tiles the
      // ring drains (0.6 us per tile of the joint q|k|v projection, 3 %).
      int m_blk = 0, n_blk = 0, next_m = 0, next_n = 0;
      TileAdapters<8> rows, next_rows;
      tile_coords(p, pair_id, pr.tiles_m, next_m, next_n);
      next_rows.fetch(g.req, next_m * 2 * BM, p.M, lane);
      for (int tile = pair_id; ok && tile < num_tiles; tile += num_pairs) {
        m_blk = next_m;
        n_blk = next_n;
        rows = next_rows;
        const int row0 = m_blk * 2 * BM + (int)rank * BM;
        const int col0 = n_blk * kCols + (int)rank * (kCols / 2);
        uint32_t off[8], next_off[8];
        int cur = -1;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (kb == num_kb - 1) {
            rows.begin();
            cur = rows.next(off);
          }
          ok = ok && __all_sync(0xffffffffu, mbar_wait_cluster(&empty_bar[stage], phase ^ 1, abort_flag, status, 41));
          if (ok) {
            const uint32_t full_addr = map_to_cta(smem_u32(&full_bar[stage]), 0);
            uint8_t* a_dst = smem + stage * kSlot;
            if (elect_one()) {
              if (kb == num_kb - 1) notes[stage].more = cur >= 0;
              if (leader) mbar_expect_tx(&full_bar[stage], 2 * kSlot);
              tma_load_2d_pair(a_dst, &pr.tm_a, full_addr, kb * BK, row0);
              tma_load_2d_pair(a_dst + A_BYTES, &pr.tm_b, full_addr, kb * BK, col0);
            }
            if (++stage == g.pair_stages) { stage = 0; phase ^= 1; }
          }
          if (kb == num_kb / 2 && tile + num_pairs < num_tiles) {
            tile_coords(p, tile + num_pairs, pr.tiles_m, next_m, next_n);
            next_rows.fetch(g.req, next_m * 2 * BM, p.M, lane);
          }
        }
        __syncwarp();
        if (tile == pair_id) pdl_wait();  // t is complete; every CTA passes here, with adapters or without
        const int slots = lora_slots(g.low), line = g.low.group == 16 ? 32 : 64;
        while (cur >= 0) {
          const int next = rows.next(next_off);
          for (int q = 0; ok && q < slots; ++q) {
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(&empty_bar[stage], phase ^ 1, abort_flag, status, 46));
            if (!ok) break;
            const uint32_t full_addr = map_to_cta(smem_u32(&full_bar[stage]), 0);
            uint8_t* a_dst = smem + stage * kSlot;
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < 8; ++i) notes[stage].off[i] = off[i];
              notes[stage].more = q + 1 < slots || next >= 0;
              if (leader) mbar_expect_tx(&full_bar[stage], 2 * (BM * line * 2 + kCols / 2 * g.low.group * 2));
              tma_load_2d_pair(a_dst, &g.tm_t, full_addr, q * line, row0);
              tma_load_3d_pair(a_dst + A_BYTES, &g.tm_b, full_addr, (g.low.group == 64 ? q >> 1 : q) * g.low.group, col0, cur);
            }
            if (++stage == g.pair_stages) { stage = 0; phase ^= 1; }
          }
          cur = next;
#pragma unroll
          for (int i = 0; i < 8; ++i) off[i] = next_off[i];
        }
      }
    }
    __syncwarp();
  } else if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair_id; ok && tile < num_tiles; tile += num_pairs) {
        const Problem& pr = g.prob[find_problem(g, tile)];
        const Params& p = pr.p;
        const int num_kb = (p.K + BK - 1) / BK;
        int m_blk, n_blk;
        tile_coords(p, tile - pr.tile_start, pr.tiles_m, m_blk, n_blk);
        const int row0 = m_blk * 2 * BM + (int)rank * BM;
        const int col0 = n_blk * BN + (int)rank * BNH;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_cluster(&empty_bar[stage], phase ^ 1, abort_flag, status, 41)) { ok = false; break; }
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * kSlot);
          const uint32_t full_addr = map_to_cta(smem_u32(&full_bar[stage]), 0);
          uint8_t* a_dst = smem + stage * kSlot;
          tma_load_2d_pair(a_dst, &pr.tm_a, full_addr, kb * BK, row0);
          tma_load_2d_pair(a_dst + A_BYTES, &pr.tm_b, full_addr, kb * BK, col0);
          if (++stage == g.pair_stages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp of the leader CTA walks the loop and an elected lane issues, so that
    // addresses and descriptors stay warp-uniform.
    if (leader) {
      constexpr uint32_t idesc = make_idesc_bf16(2 * BM, kCols, 0, 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int local = 0;
      for (int tile = pair_id; ok && tile < num_tiles; tile += num_pairs, ++local) {
        const int num_kb = (g.prob[find_problem(g, tile)].p.K + BK - 1) / BK;
        uint32_t more = 0;
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[acc], acc_phase ^ 1, abort_flag, status, 43))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait_cluster(&full_bar[stage], phase, abort_flag, status, 44))) { ok = false; break; }
          tc_fence_after_sync();
          if constexpr (kMode == 3) {
            if (kb == num_kb - 1) more = notes[stage].more;  // before the slot is given back
          }
          const uint32_t a_addr = smem_u32(smem + stage * kSlot);
          const uint64_t adesc = make_smem_desc(a_addr, 16, 1024);
          const uint64_t bdesc = make_smem_desc(a_addr + A_BYTES, 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_ss_pair(d_tmem, adesc + 2 * k, bdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
            umma_commit_pair_both(&empty_bar[stage]);
          }
          if (++stage == g.pair_stages) { stage = 0; phase ^= 1; }
        }
        if constexpr (kMode == 3) {
          for (int q = 0; ok && more != 0; ++q) {
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full_bar[stage], phase, abort_flag, status, 47));
            if (!ok) break;
            tc_fence_after_sync();
            const SlotNote note = notes[stage];
            more = note.more;
            const uint32_t a_addr = smem_u32(smem + stage * kSlot);
            const uint64_t adesc = g.low.desc(a_addr);
            const uint64_t bdesc = g.low.group == 64   ? make_smem_desc(a_addr + A_BYTES, 16, 1024)
                                   : g.low.group == 32 ? make_smem_desc(a_addr + A_BYTES, 16, 512, 4)
                                                       : make_smem_desc(a_addr + A_BYTES, 16, 256, 6);
            // which of the adapter's slots: of a group of 64 two, of a smaller one one
            const int first = g.low.group == 64 ? (q % (2 * g.low.groups) >> 1) * 4 : 0;
            const int n_units = min(g.low.group / 16, g.low.units - first);
            if (elect_one()) {
              for (int i = 0; i < n_units; ++i) {
                umma_ss_pair_masked(d_tmem, adesc + 2 * i, bdesc + 2 * i, idesc, note.off);
                if (g.low.group < 64) umma_ss_pair_masked(d_tmem, adesc + g.low.low(i), bdesc + 2 * i, idesc, note.off);
              }
              umma_commit_pair_both(&empty_bar[stage]);
            }
            if (++stage == g.pair_stages) { stage = 0; phase ^= 1; }
          }
        }
        if (ok && elect_one()) umma_commit_pair_both(&acc_full[acc]);
      }
    }
    __syncwarp();
  } else {
    // Two groups of four epilogue warps (warps 2-5 and 6-9; warp w reads TMEM lane quadrant w % 4).
    // A tile leaves in four 64-column pieces; group eg takes pieces eg and eg + 2 with a staging
    // tile, a named barrier and a store-issuing thread of its own.  One warp per scheduler was
    // not enough to cover the latencies inside a piece (accumulator load, bias / gate / residual
    // loads, GELU): measured per tile and CTA, 20 000 cycles for the plain epilogue, 28 000 with
    // GELU and 37 000 with gate + residual, against a main loop of 24 600 cycles at K = 3072.
    const int quad = warp & 3;
    const int eg = (warp - 2) >> 2;
    const int bar_id = 1 + eg;
    int local = 0;
    bool ok = true;
    const uint32_t acc_empty_leader0 = map_to_cta(smem_u32(&acc_empty[0]), 0);
    const bool store_issuer = warp == 2 + 4 * eg && lane == 0;
    for (int tile = pair_id; ok && tile < num_tiles; tile += num_pairs, ++local) {
      const Problem& pr = g.prob[find_problem(g, tile)];
      const Params& p = pr.p;
      int m_blk, n_blk;
      tile_coords(p, tile - pr.tile_start, pr.tiles_m, m_blk, n_blk);
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      const int row0 = m_blk * 2 * BM + (int)rank * BM;
      const int r_local = quad * 32 + lane;
      const int row = row0 + r_local;
      const int n0 = n_blk * kCols;
      const bool second = n0 >= p.split;
      if constexpr (kMode == 3) {
        // (a tile's bias is overwritten two tiles later, behind the barrier of the tile between)
        if ((int)threadIdx.x - 64 < kCols) bias_s[acc][threadIdx.x - 64] = bias_at(p, n0 + (int)threadIdx.x - 64);
        asm volatile("bar.sync 3, 256;" ::: "memory");
      }
      if (!mbar_wait_cluster(&acc_full[acc], acc_phase, abort_flag, status, 45)) { ok = false; break; }
      tc_fence_after_sync();
      const CUtensorMap* tm_out = second ? &pr.tm_y2 : &pr.tm_y;
      const int out_col0 = second ? n0 - p.split : n0;
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN;
      // The tile leaves in four 64-column pieces: registers -> swizzled staging tile in shared
      // memory -> one TMA store of full 128-byte lines.  (Storing 16 bytes per thread straight
      // to global memory, 32 different rows per warp instruction, cost 9 % of the GEMM.)
      if ((kMode == 1 || kMode == 2) && !second) {
        const int hd = p.heads * 128;
        const int part = n0 / hd;
        const int head0 = (n0 - part * hd) / 128;
        const bool rows_ok = row0 < p.M;  // M is a multiple of 128 here: a CTA's rows exist or do not
        const int b = row0 / (int)p.rows_per_batch;
        const int l0 = p.row_offset + (row0 - b * (int)p.rows_per_batch);
        const int heads_in_tile = (p.split - n0) >= BN ? BN / 128 : (p.split - n0) / 128;  // split = 3*heads*128
        qkv_tile_epilogue<kMode == 2>(p, &pr.tm_y, t_addr, part, head0, n0, heads_in_tile, b, l0, r_local, rows_ok,
                                      out_stage, eg, store_issuer, p.M - row0);
      } else {
      // ordinary columns: this group's two pieces, through its own staging tile
      uint8_t* buf = out_stage + eg * OUT_BUF_BYTES;
      uint8_t* line = buf + r_local * 128;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = eg + 2 * i;
        if (c * OUT_CHUNK_COLS < kCols && n0 + c * OUT_CHUNK_COLS < p.N) {  // uniform
          uint32_t r0[32], r1[32];
          tmem_ld_x32(t_addr + c * OUT_CHUNK_COLS, r0);
          tmem_ld_x32(t_addr + c * OUT_CHUNK_COLS + 32, r1);
          tmem_wait_ld();
          // this group's previous store must have read the staging tile out
          if (store_issuer) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");
          if constexpr (kMode == 3) {
            uint4 o0[4], o1[4];
            finish32(r0, &bias_s[acc][c * OUT_CHUNK_COLS], p.epi, o0);
            finish32(r1, &bias_s[acc][c * OUT_CHUNK_COLS + 32], p.epi, o1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              *reinterpret_cast<uint4*>(line + ((j ^ (r_local & 7)) << 4)) = o0[j];
              *reinterpret_cast<uint4*>(line + (((4 + j) ^ (r_local & 7)) << 4)) = o1[j];
            }
          } else {
            epilogue_chunk(p, r0, row, n0 + c * OUT_CHUNK_COLS, second, line, 0, r_local & 7);
            epilogue_chunk(p, r1, row, n0 + c * OUT_CHUNK_COLS + 32, second, line, 4, r_local & 7);
          }
          fence_proxy_async_smem();
          asm volatile("bar.sync %0, 128;" ::"r"(bar_id) : "memory");
          if (store_issuer) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                             reinterpret_cast<uint64_t>(tm_out)),
                         "r"(smem_u32(buf)), "r"(out_col0 + c * OUT_CHUNK_COLS), "r"(row0)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty_leader0 + acc * 8);
    }
    if (store_issuer) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // staging tiles outlive their stores
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while its partner may still touch its memory
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

}  // namespace gemm2

// ----------------------------------------------------------------------------------------
// The adapter projection for few tiles: 128 x BN tiles, one CTA each, so that a problem of a few hundred rows spreads
// over the machine instead of filling a handful of CTA pairs.  Same roles and ring as the kernels above, and a warp that
// lists the adapters of a tile's rows; the tile's low-rank rows t stay in shared memory while the adapters pass through the
// ring, up to four pieces of 64 ranks of B a slot.  With K small and many adapters it is bound by their MMAs, which read t
// from shared memory for every adapter (some 55 cycles each at 64 columns): 48 requests of 5 rows, 1024 -> 4096,
// rank 64: 14.2 us with the low-rank rows, 4.5 of them for 15 of the 16 adapters.
// ----------------------------------------------------------------------------------------
namespace gemm3 {
using gemm::BK;
using gemm::BM;
using gemm::Params;
using gemm2::TileAdapters;
using gemm2::bias_at;
using gemm2::finish32;
constexpr int THREADS = 224;  // TMA warp, MMA warp, four epilogue warps, a warp that lists the adapters
constexpr int MAX_STAGES = 16;
constexpr int MAX_SMEM = 220 * 1024;
constexpr int CHUNKS = 4;  // tiles of B per ring slot, at most

struct Tiles {
  CUtensorMap tm_a, tm_b, tm_t, tm_lb;
  Params p;
  RequestAdapters req;
  LowRank low;
  int stages;
  int subs;    // 64-wide K steps per ring slot
  int a_rows;  // rows of x per box: fewer than 128 when there are fewer; the MMAs then read what lies behind them in
               // shared memory as the other rows, whose results are never stored
};

// The adapters of a tile's rows, each with the mask of the rows that do not use it.  A warp of its own writes the list
// while the tile's K loop runs: with the search in the producer and a ring slot for each adapter, an adapter cost its warp
// and the MMA warp 850 cycles each (the search 345, waits, barrier updates and the copy's issue the rest).
struct AdapterList {
  uint4 off[BM];
  int id[BM];
  int count;
};

template <int BN>
__global__ void __launch_bounds__(THREADS, 1) lora_tile_kernel(const __grid_constant__ Tiles g) {
  constexpr int B_BYTES = BN * BK * 2;
  const int A_BYTES = g.a_rows * BK * 2, SLOT_A = g.subs * A_BYTES, STAGE_BYTES = SLOT_A + g.subs * B_BYTES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full[2], acc_empty[2], list_full[2], list_empty[2], t_full, t_empty;
  __shared__ AdapterList lists[2];
  __shared__ __align__(16) __nv_bfloat16 bias_s[2][BN];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  uint8_t* t_smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int T_BYTES = g.low.groups * g.low.tile_bytes();
  uint8_t* smem = t_smem + T_BYTES;
  volatile int* abort_flag = &abort_word;
  const Params& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (p.K + BK - 1) / BK;
  const int parts = (g.low.units + 3) / 4;  // of 64 ranks of B
  const int chunks = min(CHUNKS, STAGE_BYTES / B_BYTES);

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 128);
      mbar_init(&list_full[a], 1);
      mbar_init(&list_empty[a], 2);
    }
    mbar_init(&t_full, 1);
    mbar_init(&t_empty, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&g.tm_a);
    tma_prefetch_desc(&g.tm_b);
    tma_prefetch_desc(&g.tm_t);
    tma_prefetch_desc(&g.tm_lb);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  pdl_release();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, t_phase = 0;
    bool ok = true;
    int local = 0;
    for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x, ++local) {
      const int row0 = tile % p.tiles_m * BM, col0 = tile / p.tiles_m * BN;
      for (int kb = 0; kb < num_kb; kb += g.subs) {
        const int subs = min(g.subs, num_kb - kb);
        ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 91));
        if (!ok) break;
        uint8_t* dst = smem + stage * STAGE_BYTES;
        if (elect_one()) {
          mbar_expect_tx(&full_bar[stage], subs * (A_BYTES + B_BYTES));
          for (int i = 0; i < subs; ++i) {
            tma_load_2d(dst + i * A_BYTES, &g.tm_a, &full_bar[stage], (kb + i) * BK, row0);
            tma_load_2d(dst + SLOT_A + i * B_BYTES, &g.tm_b, &full_bar[stage], (kb + i) * BK, col0);
          }
        }
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
      }
      const int buf = local & 1;
      const AdapterList& list = lists[buf];
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&list_full[buf], (local >> 1) & 1, abort_flag, p.status, 92));
      const int total = ok ? list.count * parts : 0;
      for (int c = 0; ok && c < total; c += chunks) {
        ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 93));
        if (!ok) break;
        const int n = min(chunks, total - c);
        if (elect_one()) {
          mbar_expect_tx(&full_bar[stage], n * B_BYTES);
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            if (i >= n) break;
            const int item = parts == 1 ? c + i : (c + i) / parts;
            tma_load_3d(smem + stage * STAGE_BYTES + i * B_BYTES, &g.tm_lb, &full_bar[stage], (c + i - item * parts) * 64, col0,
                        list.id[item]);
          }
        }
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
        if (c == 0) {  // t, as soon as it is complete
          if (tile == (int)blockIdx.x) pdl_wait();
          ok = __all_sync(0xffffffffu, mbar_wait(&t_empty, t_phase ^ 1, abort_flag, p.status, 99));
          t_phase ^= 1;
          if (ok && elect_one()) {
            const int line = g.low.group == 16 ? 32 : 64;
            mbar_expect_tx(&t_full, T_BYTES);
            for (int k = 0; k < g.low.ld(); k += line) tma_load_2d(t_smem + k * BM * 2, &g.tm_t, &t_full, k, row0);
          }
        }
      }
      if (tile == (int)blockIdx.x && total == 0) pdl_wait();  // every CTA waits for the first kernel, with adapters or without
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[buf]);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_bf16(BM, BN, 0, 0);
    // of t: the first 16 ranks' high parts, how far behind a group's high parts its low parts lie, and the next group
    const uint64_t t_desc = g.low.desc(smem_u32(t_smem));
    const int to_low = g.low.low(0) - g.low.high(0), part_step = g.low.tile_bytes() >> 4;
    int stage = 0;
    uint32_t phase = 0, t_phase = 0;
    bool ok = true;
    int local = 0;
    for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x, ++local) {
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.status, 100));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int kb = 0; kb < num_kb; kb += g.subs) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 95));
        if (!ok) break;
        tc_fence_after_sync();
        const int subs = min(g.subs, num_kb - kb);
        const uint32_t a_addr = smem_u32(smem + stage * STAGE_BYTES);
        const uint64_t adesc = make_smem_desc(a_addr, 16, 1024), bdesc = make_smem_desc(a_addr + SLOT_A, 16, 1024);
        if (elect_one()) {
          for (int i = 0; i < subs; ++i) {
            const uint64_t ad = adesc + i * (A_BYTES >> 4), bd = bdesc + i * (B_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) umma_ss(d_tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | i | k) != 0 ? 1u : 0u);
          }
          umma_commit(&empty_bar[stage]);
        }
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
      }
      const int buf = local & 1;
      const AdapterList& list = lists[buf];
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&list_full[buf], (local >> 1) & 1, abort_flag, p.status, 94));
      const int total = ok ? list.count * parts : 0;
      const bool any = total > 0;
      if (any) {
        ok = __all_sync(0xffffffffu, mbar_wait(&t_full, t_phase, abort_flag, p.status, 96));
        t_phase ^= 1;
      }
      for (int c = 0; ok && c < total; c += chunks) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 97));
        if (!ok) break;
        tc_fence_after_sync();
        const int n = min(chunks, total - c);
        const uint64_t bdesc = make_smem_desc(smem_u32(smem + stage * STAGE_BYTES), 16, 1024);
        if (elect_one()) {
          // (more than 64 ranks: groups of 64, one per part; up to 64 there is one group and one part)
          int part[CHUNKS];
          uint4 o[CHUNKS];  // all asked for before the first is needed
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            if (i >= n) break;
            const int item = parts == 1 ? c + i : (c + i) / parts;
            part[i] = c + i - item * parts;
            o[i] = list.off[item];
          }
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            if (i >= n) break;
            const uint64_t ad = t_desc + part[i] * part_step, bd = bdesc + i * (B_BYTES >> 4);
            const uint32_t off[4] = {o[i].x, o[i].y, o[i].z, o[i].w};
            const int n_units = g.low.units - part[i] * 4;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (u >= n_units) break;
              umma_ss_masked(d_tmem, ad + 2 * u, bd + 2 * u, idesc, off);
              umma_ss_masked(d_tmem, ad + to_low + 2 * u, bd + 2 * u, idesc, off);
            }
          }
          umma_commit(&empty_bar[stage]);
        }
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[buf]);
      if (ok && elect_one()) {
        if (any) umma_commit(&t_empty);
        umma_commit(&acc_full[acc]);
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    int local = 0;
    for (int tile = blockIdx.x; tile < p.num_tiles; tile += gridDim.x, ++local) {
      TileAdapters<4> rows;
      rows.fetch(g.req, tile % p.tiles_m * BM, p.M, lane);
      const int buf = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&list_empty[buf], ((local >> 1) & 1) ^ 1, abort_flag, p.status, 101))) break;
      AdapterList& list = lists[buf];
      rows.begin();
      uint32_t off[4];
      int n = 0;
      for (int cur = rows.next(off); cur >= 0; cur = rows.next(off), ++n) {
        if (lane == 0) {
          list.off[n] = make_uint4(off[0], off[1], off[2], off[3]);
          list.id[n] = cur;
        }
      }
      if (lane == 0) {
        list.count = n;
        mbar_arrive(&list_full[buf]);
      }
      __syncwarp();
    }
    __syncwarp();
  } else {
    const int quad = warp & 3;
    int local = 0;
    for (int tile = blockIdx.x; tile < p.num_tiles; tile += gridDim.x, ++local) {
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      const int row0 = tile % p.tiles_m * BM, n0 = tile / p.tiles_m * BN;
      // (a tile's bias is overwritten two tiles later, behind the barrier of the tile between)
      if ((int)threadIdx.x - 64 < BN) bias_s[acc][threadIdx.x - 64] = bias_at(p, n0 + (int)threadIdx.x - 64);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, 98)) break;
      __syncwarp();
      tc_fence_after_sync();
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * BN;
      if (row0 + quad * 32 < p.M) {
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          if (n0 + c * 32 >= p.N) break;  // uniform
          uint32_t r[32];
          tmem_ld_x32(t_addr + c * 32, r);
          tmem_wait_ld();
          uint4 o[4];
          finish32(r, &bias_s[acc][c * 32], p.epi, o);
          const int row = row0 + quad * 32 + lane;
          if (row < p.M) {
            __nv_bfloat16* out = p.y + (int64_t)row * p.ldy + n0 + c * 32;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n0 + c * 32 + j * 8 < p.N) *reinterpret_cast<uint4*>(out + j * 8) = o[j];
          }
        }
      }
      tc_fence_before_sync();
      mbar_arrive(&acc_empty[acc]);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

template <int BN>
static int launch_tiles(Tiles& g, const fluxb_linear_problem& a, int64_t N, int64_t K, const void* lora_b, int64_t ldb,
                        cudaStream_t st) {
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)N}, strides[1] = {(uint64_t)a.ldw * 2};
    const uint32_t box[2] = {BK, BN};
    int rc = encode_tmap_bf16(&g.tm_b, a.w, 2, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  {
    const uint64_t dims[3] = {(uint64_t)g.low.R, (uint64_t)N, (uint64_t)g.req.n_adapters};
    const uint64_t strides[2] = {(uint64_t)ldb * 2, (uint64_t)(N * ldb) * 2};
    const uint32_t box[3] = {64, BN, 1};
    int rc = encode_tmap_bf16(&g.tm_lb, lora_b, 3, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  const int step_bytes = g.a_rows * BK * 2 + BN * BK * 2, behind = (BM - g.a_rows) * BK * 2;
  const int t_bytes = g.low.groups * g.low.group * 512, room = MAX_SMEM - 1024 - 1024 - t_bytes - behind;
  // Several K steps per slot, as long as three slots fit: a slot costs the producer and the MMA warp some 500 cycles
  // each (wait, vote, election, issue), which a step of a narrow tile does not cover (16 x 4096 -> 4096: 22.6 us with
  // one step per slot).
  g.subs = room / step_bytes >= 12 ? 4 : (room / step_bytes >= 6 ? 2 : 1);
  const int stage_bytes = g.subs * step_bytes;
  g.stages = room / stage_bytes;
  if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
  g.p.tiles_n = (int)((N + BN - 1) / BN);
  g.p.num_tiles = g.p.tiles_m * g.p.tiles_n;
  auto kern = lora_tile_kernel<BN>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: cannot set shared memory size: %s", cudaGetErrorString(e));
  const int grid = g.p.num_tiles < sm_count() ? g.p.num_tiles : sm_count();
  e = launch_after(kern, grid, THREADS, 1024 + t_bytes + g.stages * stage_bytes + behind, st, g);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

}  // namespace gemm3
}  // namespace fluxb

using namespace fluxb;

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static bool use_pair_kernel() {
  // CTA pairs (256x256 tiles) unless FLUXB_GEMM_PAIR=0 asks for the single-CTA kernel.
  static const int pair_env = [] {
    const char* s = getenv("FLUXB_GEMM_PAIR");
    return (s != nullptr && *s != 0) ? atoi(s) : 1;
  }();
  return pair_env != 0;
}

// The tile order for row blocks of `row_blk` and `concurrent` tiles at a time; p has M, N, K and tiles_n.
static void choose_raster(fluxb::gemm::Params& p, int row_blk, int concurrent) {
  // Keep the smaller operand resident in L2 when it fits, sweep the larger one.
  const int tm = (p.M + row_blk - 1) / row_blk, tn = p.tiles_n;
  const double a_bytes = 2.0 * (double)p.M * (double)p.K, w_bytes = 2.0 * (double)p.N * (double)p.K;
  const double keep_limit = 48e6;
  if (a_bytes <= w_bytes) {
    p.raster_band_n = 0;  // keep x row-blocks
    p.raster_group = a_bytes <= keep_limit ? tm : (concurrent / tn > 1 ? concurrent / tn : 1);
  } else {
    p.raster_band_n = 1;  // keep w row-blocks
    p.raster_group = w_bytes <= keep_limit ? tn : (concurrent / tm > 1 ? concurrent / tm : 1);
  }
  if (p.raster_group < 1) p.raster_group = 1;
}

// Validates one problem, encodes its tensor maps and fills its kernel parameters.
static int prepare_problem(const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, int64_t split, int epi2,
                           int round_before_act, bool use_pair, CUtensorMap* tm_a, CUtensorMap* tm_b,
                           fluxb::gemm::Params* out) {
  using namespace fluxb::gemm;
  const int64_t M = a.M;
  if (M <= 0 || N <= 0 || K <= 0) return set_error(FLUXB_ERR_BAD_ARG, "linear: bad sizes");
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear: dimension too large");
  if (!a.x || !a.w || !a.y) return set_error(FLUXB_ERR_BAD_ARG, "linear: null pointer");
  if (split < 0 || split > N) return set_error(FLUXB_ERR_BAD_ARG, "linear: split outside [0, N]");
  if (split < N) {
    if (!a.y2) return set_error(FLUXB_ERR_BAD_ARG, "linear: split < N needs a second output");
    if (split % BN) return set_error(FLUXB_ERR_BAD_ARG, "linear: split must be a multiple of %d", BN);
    if (a.ldy2 % 8 || !aligned16(a.y2)) return set_error(FLUXB_ERR_BAD_ARG, "linear: second output misaligned");
  }
  if (K % 8 || a.ldx % 8 || a.ldw % 8 || N % 8 || a.ldy % 8 || a.ldx < K || a.ldw < K)
    return set_error(FLUXB_ERR_BAD_ARG, "linear: K, N and row strides must be multiples of 8 (and strides >= K)");
  if (!aligned16(a.x) || !aligned16(a.w) || !aligned16(a.y) || !aligned16(a.bias))
    return set_error(FLUXB_ERR_BAD_ARG, "linear: pointers must be 16-byte aligned");
  const int epis[2] = {epi, split < N ? epi2 : FLUXB_EPI_NONE};
  for (int e : epis) {
    if (e != FLUXB_EPI_NONE && e != FLUXB_EPI_GELU && e != FLUXB_EPI_GATE_RESID)
      return set_error(FLUXB_ERR_UNSUPPORTED, "linear: unknown epilogue %d", e);
    if (e == FLUXB_EPI_GATE_RESID) {
      if (!a.resid || !a.gate || a.rows_per_batch <= 0 || a.ldr % 8 || a.gate_stride % 8 || !aligned16(a.resid) ||
          !aligned16(a.gate))
        return set_error(FLUXB_ERR_BAD_ARG, "linear: gate/residual epilogue needs aligned resid, gate and rows_per_batch > 0");
    }
  }
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)M};
    const uint64_t strides[1] = {(uint64_t)a.ldx * 2};
    const uint32_t box[2] = {BK, BM};
    int rc = encode_tmap_bf16(tm_a, a.x, 2, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)N};
    const uint64_t strides[1] = {(uint64_t)a.ldw * 2};
    const uint32_t box[2] = {BK, (uint32_t)(use_pair ? fluxb::gemm2::BNH : BN)};
    int rc = encode_tmap_bf16(tm_b, a.w, 2, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  Params& p = *out;
  p.bias = static_cast<const __nv_bfloat16*>(a.bias);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.y2 = static_cast<__nv_bfloat16*>(a.y2);
  p.resid = static_cast<const __nv_bfloat16*>(a.resid);
  p.gate = static_cast<const __nv_bfloat16*>(a.gate);
  p.ldy = a.ldy; p.ldy2 = a.ldy2; p.ldr = a.ldr; p.gate_stride = a.gate_stride;
  p.rows_per_batch = a.rows_per_batch > 0 ? a.rows_per_batch : 1;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.split = (int)split; p.epi = epi; p.epi2 = epi2; p.round_before_act = round_before_act;
  p.tiles_m = (int)((M + BM - 1) / BM);
  p.tiles_n = (int)((N + BN - 1) / BN);
  p.num_tiles = p.tiles_m * p.tiles_n;
  p.status = device_status_ptr();
  p.pe = nullptr; p.qk_scale[0] = p.qk_scale[1] = nullptr; p.row_offset = 0; p.heads = 0; p.l_total = 0; p.eps = 0.f;
  p.scat_groups = 0; p.scat_hpg = 1; p.scat_sb = p.scat_sh = p.scat_sl = p.scat_koff = p.scat_voff = 0;
  for (int gi = 0; gi < 8; ++gi) p.scat_base[gi] = nullptr;
  p.pair_stages = fluxb::gemm2::STAGES;
  choose_raster(p, use_pair ? 256 : 128, use_pair ? sm_count() / 2 : sm_count());
  return FLUXB_OK;
}

extern "C" int fluxb_linear_grouped(const fluxb_linear_problem* problems, int count, int64_t N, int64_t K, int epi,
                                    int64_t split, int epi2, int round_before_act, fluxb_stream_t stream) {
  using namespace fluxb::gemm;
  if (count < 0 || (count > 0 && problems == nullptr)) return set_error(FLUXB_ERR_BAD_ARG, "linear_grouped: bad problem list");
  if (count > fluxb::gemm2::MAX_PROBLEMS)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear_grouped: at most %d problems per launch", fluxb::gemm2::MAX_PROBLEMS);
  if (N < 0 || K <= 0) return set_error(FLUXB_ERR_BAD_ARG, "linear: bad sizes");
  const bool use_pair = use_pair_kernel();
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  fluxb::gemm2::Grouped g;
  g.count = 0;
  g.total_tiles = 0;
  g.pair_stages = fluxb::gemm2::STAGES;
  for (int i = 0; i < count; ++i) {
    if (problems[i].M < 0) return set_error(FLUXB_ERR_BAD_ARG, "linear: negative M");
    if (problems[i].M == 0 || N == 0) continue;  // nothing to compute for this one
    fluxb::gemm2::Problem& pr = g.prob[g.count];
    int rc = prepare_problem(problems[i], N, K, epi, split, epi2, round_before_act, use_pair, &pr.tm_a, &pr.tm_b, &pr.p);
    if (rc != FLUXB_OK) return rc;
    if (!use_pair) {  // single-CTA kernel: one launch per problem
      cudaError_t e = cudaFuncSetAttribute(gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
      if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear: cannot set shared memory size: %s", cudaGetErrorString(e));
      const int grid = pr.p.num_tiles < sm_count() ? pr.p.num_tiles : sm_count();
      gemm_kernel<<<grid, THREADS, SMEM_BYTES, st>>>(pr.tm_a, pr.tm_b, pr.p);
      continue;
    }
    {
      const fluxb_linear_problem& a = problems[i];
      const int64_t n_first = split < N ? split : N;
      const uint32_t box[2] = {fluxb::gemm2::OUT_CHUNK_COLS, fluxb::gemm2::BM};
      const uint64_t dims[2] = {(uint64_t)n_first, (uint64_t)a.M};
      const uint64_t strides[1] = {(uint64_t)a.ldy * 2};
      rc = n_first > 0 ? encode_tmap_bf16(&pr.tm_y, a.y, 2, dims, strides, box) : FLUXB_OK;
      if (rc != FLUXB_OK) return rc;
      if (split < N) {
        const uint64_t dims2[2] = {(uint64_t)(N - split), (uint64_t)a.M};
        const uint64_t strides2[1] = {(uint64_t)a.ldy2 * 2};
        rc = encode_tmap_bf16(&pr.tm_y2, a.y2, 2, dims2, strides2, box);
        if (rc != FLUXB_OK) return rc;
        if (n_first == 0) pr.tm_y = pr.tm_y2;
      } else {
        pr.tm_y2 = pr.tm_y;
      }
    }
    pr.tiles_m = (int)((problems[i].M + 255) / 256);
    pr.tile_start = g.total_tiles;
    g.total_tiles += pr.tiles_m * pr.p.tiles_n;
    ++g.count;
  }
  if (use_pair && g.count > 0) {
    auto kern = fluxb::gemm2::gemm_pair_kernel<0>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fluxb::gemm2::SMEM_BYTES);
    if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear: cannot set shared memory size: %s", cudaGetErrorString(e));
    const int pairs = g.total_tiles < sm_count() / 2 ? g.total_tiles : sm_count() / 2;
    kern<<<2 * pairs, fluxb::gemm2::THREADS, fluxb::gemm2::SMEM_BYTES, st>>>(g);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

struct QkvScatter {  // destination of the scatter form, see fluxb_linear_qkv_grouped_scatter
  void* const* bases;
  int n_groups;
  int64_t k_off, v_off, sb, sh, sl;
};

static int linear_qkv_grouped_impl(const fluxb_linear_problem* problems, const fluxb_qkv_stream* streams,
                                   int count, int64_t B, int64_t H, int64_t D, int64_t L_total, int64_t K,
                                   void* qkv_out, const QkvScatter* scat, float eps, int64_t N2, int epi2,
                                   int round_before_act, fluxb_stream_t stream) {
  using namespace fluxb::gemm;
  if (count < 1 || count > fluxb::gemm2::MAX_PROBLEMS || !problems || !streams)
    return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: 1..%d problems with their stream descriptions", fluxb::gemm2::MAX_PROBLEMS);
  if (!use_pair_kernel()) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_qkv_grouped: needs the CTA-pair kernel (FLUXB_GEMM_PAIR=0 is set)");
  if (D != 128) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_qkv_grouped: head_dim %lld (only 128)", (long long)D);
  // A 256-column tile holds two heads and is normalised as a whole with q's, k's or no scale: the
  // q|k and k|v boundaries (multiples of H*D) must therefore fall on tile boundaries.
  if ((H * D) % 256)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear_qkv_grouped: %lld heads (the head count must be even)", (long long)H);
  if (B <= 0 || H <= 0 || L_total <= 0 || K <= 0 || B > 65535 || H > 65535 || L_total > (1 << 30))
    return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: bad sizes");
  if (scat == nullptr) {
    if (!qkv_out || !aligned16(qkv_out)) return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: output null or misaligned");
  } else {
    if (scat->n_groups < 1 || scat->n_groups > 8 || !scat->bases || H % scat->n_groups)
      return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped_scatter: 1..8 head groups that divide the head count");
    for (int i = 0; i < scat->n_groups; ++i)
      if (!scat->bases[i] || !aligned16(scat->bases[i]))
        return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped_scatter: output base %d is null or misaligned", i);
    if (scat->k_off % 8 || scat->v_off % 8 || scat->sb % 8 || scat->sh % 8 || scat->sl % 8 || scat->sl < D)
      return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped_scatter: offsets and strides must be multiples of 8 elements");
  }
  if (N2 < 0 || N2 % 8) return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: N2 must be a non-negative multiple of 8");
  if (epi2 != FLUXB_EPI_NONE && epi2 != FLUXB_EPI_GELU)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear_qkv_grouped: the extra columns take no epilogue or GELU");
  const int64_t N_qkv = 3 * H * D;
  const int64_t N = N_qkv + N2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  fluxb::gemm2::Grouped g;
  g.count = 0;
  g.total_tiles = 0;
  g.pair_stages = fluxb::gemm2::STAGES;
  // one 5-D map over [3, B, H, L_total, D] for all problems
  CUtensorMap tm_out;
  if (scat == nullptr) {
    const uint64_t dims[5] = {(uint64_t)D, (uint64_t)L_total, (uint64_t)H, (uint64_t)B, 3};
    const uint64_t strides[4] = {(uint64_t)D * 2, (uint64_t)L_total * D * 2, (uint64_t)H * L_total * D * 2,
                                 (uint64_t)B * H * L_total * D * 2};
    const uint32_t box[5] = {fluxb::gemm2::OUT_CHUNK_COLS, fluxb::gemm2::BM, 1, 1, 1};
    int rc = encode_tmap_bf16(&tm_out, qkv_out, 5, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  for (int i = 0; i < count; ++i) {
    fluxb_linear_problem a = problems[i];
    const fluxb_qkv_stream& sdesc = streams[i];
    const int64_t Ls = a.rows_per_batch;
    // The head-major form leaves through 128-row TMA boxes; the scatter form masks row by row, so
    // with one batch item any stream length and offset will do.
    const int64_t align = (scat != nullptr && B == 1) ? 1 : 128;
    if (a.M <= 0 || Ls <= 0 || a.M != B * Ls || Ls % align)
      return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: each stream needs M = B * rows_per_batch with rows_per_batch a multiple of 128");
    if (sdesc.row_offset < 0 || sdesc.row_offset % align || sdesc.row_offset + Ls > L_total)
      return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: row_offset must be a multiple of 128 inside the joint sequence");
    if ((sdesc.q_scale == nullptr) != (sdesc.k_scale == nullptr) || !aligned16(sdesc.q_scale) || !aligned16(sdesc.k_scale) ||
        !aligned16(sdesc.pe))
      return set_error(FLUXB_ERR_BAD_ARG, "linear_qkv_grouped: scales go together; scales and pe must be 16-byte aligned");
    a.y = scat == nullptr ? qkv_out : scat->bases[0]; a.ldy = D;  // the q|k|v columns do not leave through y
    a.resid = nullptr; a.gate = nullptr;
    if (N2 == 0) a.y2 = nullptr;
    fluxb::gemm2::Problem& pr = g.prob[g.count];
    int rc = prepare_problem(a, N, K, FLUXB_EPI_NONE, N_qkv, epi2, round_before_act, true, &pr.tm_a, &pr.tm_b, &pr.p);
    if (rc != FLUXB_OK) return rc;
    pr.p.epi = EPI_QKV_HEADS;
    pr.p.rows_per_batch = Ls;
    pr.p.pe = sdesc.pe;
    pr.p.qk_scale[0] = static_cast<const __nv_bfloat16*>(sdesc.q_scale);
    pr.p.qk_scale[1] = static_cast<const __nv_bfloat16*>(sdesc.k_scale);
    pr.p.row_offset = (int)sdesc.row_offset;
    pr.p.heads = (int)H;
    pr.p.l_total = (int)L_total;
    pr.p.eps = eps;
    if (scat != nullptr) {
      pr.p.scat_groups = scat->n_groups;
      pr.p.scat_hpg = (int)(H / scat->n_groups);
      for (int gi = 0; gi < 8; ++gi) pr.p.scat_base[gi] = gi < scat->n_groups ? static_cast<__nv_bfloat16*>(scat->bases[gi]) : nullptr;
      pr.p.scat_sb = scat->sb; pr.p.scat_sh = scat->sh; pr.p.scat_sl = scat->sl;
      pr.p.scat_koff = scat->k_off; pr.p.scat_voff = scat->v_off;
      tm_out = pr.tm_a;  // never used for a store in this form; any valid map will do for the prefetch
    }
    pr.tm_y = tm_out;
    pr.tm_y2 = tm_out;
    if (N2 > 0) {  // extra columns [3*H*D, 3*H*D + N2): an ordinary output with epilogue epi2
      const uint32_t box[2] = {fluxb::gemm2::OUT_CHUNK_COLS, fluxb::gemm2::BM};
      const uint64_t dims2[2] = {(uint64_t)N2, (uint64_t)a.M};
      const uint64_t strides2[1] = {(uint64_t)a.ldy2 * 2};
      rc = encode_tmap_bf16(&pr.tm_y2, a.y2, 2, dims2, strides2, box);
      if (rc != FLUXB_OK) return rc;
    }
    pr.tiles_m = (int)((a.M + 255) / 256);
    pr.tile_start = g.total_tiles;
    g.total_tiles += pr.tiles_m * pr.p.tiles_n;
    ++g.count;
  }
  auto kern = scat == nullptr ? fluxb::gemm2::gemm_pair_kernel<1> : fluxb::gemm2::gemm_pair_kernel<2>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fluxb::gemm2::SMEM_BYTES);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_qkv_grouped: cannot set shared memory size: %s", cudaGetErrorString(e));
  const int pairs = g.total_tiles < sm_count() / 2 ? g.total_tiles : sm_count() / 2;
  kern<<<2 * pairs, fluxb::gemm2::THREADS, fluxb::gemm2::SMEM_BYTES, st>>>(g);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_qkv_grouped: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

extern "C" int fluxb_linear_qkv_grouped(const fluxb_linear_problem* problems, const fluxb_qkv_stream* streams,
                                        int count, int64_t B, int64_t H, int64_t D, int64_t L_total, int64_t K,
                                        void* qkv_out, float eps, int64_t N2, int epi2, int round_before_act,
                                        fluxb_stream_t stream) {
  return linear_qkv_grouped_impl(problems, streams, count, B, H, D, L_total, K, qkv_out, nullptr, eps, N2, epi2,
                                 round_before_act, stream);
}

extern "C" int fluxb_linear_qkv_grouped_scatter(const fluxb_linear_problem* problems, const fluxb_qkv_stream* streams,
                                                int count, int64_t B, int64_t H, int64_t D, int64_t L_total,
                                                int64_t K, void* const* group_bases, int n_groups, int64_t k_off,
                                                int64_t v_off, int64_t o_sb, int64_t o_sh, int64_t o_sl, float eps,
                                                int64_t N2, int epi2, int round_before_act, fluxb_stream_t stream) {
  const QkvScatter scat{group_bases, n_groups, k_off, v_off, o_sb, o_sh, o_sl};
  return linear_qkv_grouped_impl(problems, streams, count, B, H, D, L_total, K, nullptr, &scat, eps, N2, epi2,
                                 round_before_act, stream);
}

// t [M, ld] in boxes of one line x 128 rows.
static int encode_low_rank(CUtensorMap* out, const void* t_rows, int64_t M, const LowRank& low) {
  const uint64_t dims[2] = {(uint64_t)low.ld(), (uint64_t)M}, strides[1] = {(uint64_t)low.ld() * 2};
  const uint32_t box[2] = {(uint32_t)(low.group == 16 ? 32 : 64), fluxb::gemm::BM};
  return encode_tmap_bf16(out, t_rows, 2, dims, strides, box,
                          low.group == 16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

// The adapter projection on CTA pairs: tiles of 256 rows and kCols columns.
template <int kCols>
static int launch_lora_pairs(const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t_rows, const void* lora_b,
                             const LowRank& low, int64_t ldb, const RequestAdapters& req, cudaStream_t st) {
  using namespace fluxb::gemm2;
  LoraGrouped g;
  g.count = 1;
  g.pair_stages = LORA_STAGES;
  Problem& pr = g.prob[0];
  int rc = prepare_problem(a, N, K, epi, N, FLUXB_EPI_NONE, 0, true, &pr.tm_a, &pr.tm_b, &pr.p);
  if (rc != FLUXB_OK) return rc;
  {
    const uint64_t dims[2] = {(uint64_t)N, (uint64_t)a.M}, strides[1] = {(uint64_t)a.ldy * 2};
    const uint32_t box[2] = {OUT_CHUNK_COLS, BM};
    if ((rc = encode_tmap_bf16(&pr.tm_y, a.y, 2, dims, strides, box)) != FLUXB_OK) return rc;
    pr.tm_y2 = pr.tm_y;
  }
  if (kCols < BN) {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)N}, strides[1] = {(uint64_t)a.ldw * 2};
    const uint32_t box[2] = {BK, kCols / 2};
    if ((rc = encode_tmap_bf16(&pr.tm_b, a.w, 2, dims, strides, box)) != FLUXB_OK) return rc;
    pr.p.tiles_n = (int)((N + kCols - 1) / kCols);
    choose_raster(pr.p, 2 * BM, sm_count() / 2);
  }
  g.low = low;
  if ((rc = encode_low_rank(&g.tm_t, t_rows, a.M, low)) != FLUXB_OK) return rc;
  {
    const uint64_t dims[3] = {(uint64_t)low.R, (uint64_t)N, (uint64_t)req.n_adapters};
    const uint64_t strides[2] = {(uint64_t)ldb * 2, (uint64_t)(N * ldb) * 2};
    const uint32_t box[3] = {(uint32_t)low.group, kCols / 2, 1};
    const CUtensorMapSwizzle swz = low.group == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                   : low.group == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                     : CU_TENSOR_MAP_SWIZZLE_32B;
    if ((rc = encode_tmap_bf16(&g.tm_b, lora_b, 3, dims, strides, box, swz)) != FLUXB_OK) return rc;
  }
  g.req = req;
  pr.tiles_m = (int)((a.M + 255) / 256);
  pr.tile_start = 0;
  g.total_tiles = pr.tiles_m * pr.p.tiles_n;
  auto kern = gemm_pair_kernel<3, LoraGrouped, kCols>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, lora_smem(kCols));
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: cannot set shared memory size: %s", cudaGetErrorString(e));
  const int pairs = g.total_tiles < sm_count() / 2 ? g.total_tiles : sm_count() / 2;
  e = launch_after(kern, 2 * pairs, THREADS, lora_smem(kCols), st, g);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

// Which tiles, and over how many blocks the kernel of the low-rank rows splits K, by an estimate in cycles.  The tiles'
// part is fitted to the kernels over 20 problems (9 to 31131 rows, K 96 to 4696, N 72 to 5496) and within a fifth of each
// time: a tile of a CTA pair takes 400 and 75 per 64 columns for a 64-wide K step, and at least 7500 for its epilogue; a
// 128 x BN tile of one CTA takes two per operand row and step, and at least its own epilogue.  For example
// 2048 x 3072 -> 3072: pairs 256 wide 39.1 us (two rounds of 96 tiles on 74 pairs), 192 wide 36.4; 4096 x 4096 -> 4096:
// 95.4 and 105; 1024 x 2048 -> 2048: pairs 18.7, BN 128 15.5, 64 21.6, 32 34.4; 128 x 1024 -> 4096: 13.8, 10.4, 9.7, 9.2.
// The adapters that a tile's rows may use take 850 a ring slot, or, on one CTA, 80 each and 120 per sixteen ranks.
// The low-rank rows run beside the projection's first tiles, on SMs of their own: SMs whose projection blocks have a tile
// less to do than the others cost nothing as long as t is there at the end of the first K loop (4 x 512 rows, 192 wide,
// 20 spare pairs: 43.3 us with 64 blocks of low-rank rows, 37.7 with 16); others wait for some 0.6 of their time (700
// rows of three requests, K 2048, 72 tiles on 74 pairs: 20.3 us without, 25.1 with 72 blocks, 26.7 with 18).
LoraPlan fluxb::plan_lora(int64_t M, int64_t N, int64_t K, const RequestAdapters& req, const LowRank& low) {
  const int64_t L = req.length, rpad = low.units * 16;
  const int64_t shrink_rows = L < 128 ? L : 128, shrink_tiles = L <= kLoraShort ? 0 : M / L * ((L + 127) / 128);
  const int64_t kb = (K + 63) / 64, sms = sm_count();
  const int64_t a_rows = M < 128 ? (M + 7) / 8 * 8 : 128;
  LoraPlan plan{};
  int64_t best = INT64_MAX;
  for (int c : {256, 192, 128, 64, 32}) {
    const bool pair = c > 128;
    const int64_t tiles = (M + (pair ? 255 : 127)) / (pair ? 256 : 128) * ((N + c - 1) / c);
    const int64_t steps = (pair ? 400 + 75 * c / 64 : (a_rows + c) * 2 + 100) * kb, epilogue = pair ? 7500 : 1100 + 30 * c;
    const int64_t rows = pair ? 256 : 128, requests = L % rows == 0 ? 1 : (rows + L - 2) / L + 1;
    const int64_t adapters = requests < req.n_adapters ? requests : req.n_adapters;
    const int64_t each = pair ? fluxb::gemm2::lora_slots(low) * 850 : 80 + 120 * low.units;
    const int64_t tile = (steps > epilogue ? steps : epilogue) + adapters * each + (pair ? 0 : 1000);
    const int64_t units = pair ? sms / 2 : sms, rounds = (tiles + units - 1) / units;
    const int64_t spare = (rounds * units - tiles) * (pair ? 2 : 1);
    int64_t shrink = shrink_tiles > 0 ? INT64_MAX : 0;
    int ksplit = 1;
    // (clusters of eight do not all find a place at once from 16 on: 2048 rows, K 3072 alone: 16.7 us with eight, 9.9
    // with four, 12.0 with two)
    for (int ks = 1; shrink_tiles > 0 && ks <= (shrink_tiles < 12 ? 8 : 4); ks *= 2) {
      if (ks > 1 && (shrink_tiles * ks > sms || kb < ks * 4)) break;
      int64_t t = (9000 + (kb + ks - 1) / ks * ((shrink_rows + rpad) * 2 + 100)) * ((shrink_tiles * ks + sms - 1) / sms);
      t = shrink_tiles * ks <= spare ? (t > steps ? t - steps : 0) : t * 3 / 5;
      if (t < shrink) { shrink = t; ksplit = ks; }
    }
    const int64_t all = rounds * tile + (pair ? 13000 : 7000) + shrink;
    if (all < best) { best = all; plan = LoraPlan{c, ksplit}; }
  }
  return plan;
}

// The projection of fluxb_linear_lora for more rows than the row-streaming kernel takes; t as lora.cu leaves it.
int fluxb::launch_lora_gemm(const LoraPlan& plan, const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t_rows,
                            const void* lora_b, const LowRank& low, int64_t ldb, const RequestAdapters& req, cudaStream_t st) {
  if (plan.cols == 256) return launch_lora_pairs<256>(a, N, K, epi, t_rows, lora_b, low, ldb, req, st);
  if (plan.cols == 192) return launch_lora_pairs<192>(a, N, K, epi, t_rows, lora_b, low, ldb, req, st);
  fluxb::gemm3::Tiles t;
  int rc = prepare_problem(a, N, K, epi, N, FLUXB_EPI_NONE, 0, false, &t.tm_a, &t.tm_b, &t.p);
  if (rc != FLUXB_OK) return rc;
  t.req = req;
  t.low = low;
  t.a_rows = (int)(a.M < 128 ? (a.M + 7) / 8 * 8 : 128);
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)a.M}, strides[1] = {(uint64_t)a.ldx * 2};
    const uint32_t box[2] = {64, (uint32_t)t.a_rows};
    if ((rc = encode_tmap_bf16(&t.tm_a, a.x, 2, dims, strides, box)) != FLUXB_OK) return rc;
  }
  if ((rc = encode_low_rank(&t.tm_t, t_rows, a.M, low)) != FLUXB_OK) return rc;
  if (plan.cols == 128) return fluxb::gemm3::launch_tiles<128>(t, a, N, K, lora_b, ldb, st);
  if (plan.cols == 64) return fluxb::gemm3::launch_tiles<64>(t, a, N, K, lora_b, ldb, st);
  return fluxb::gemm3::launch_tiles<32>(t, a, N, K, lora_b, ldb, st);
}

extern "C" int fluxb_linear(const void* x, const void* w, const void* bias, void* y, int64_t M,
                            int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldy, int epi,
                            void* y2, int64_t ldy2, int64_t split, int epi2, const void* resid,
                            int64_t ldr, const void* gate, int64_t gate_stride,
                            int64_t rows_per_batch, int round_before_act, fluxb_stream_t stream) {
  fluxb_linear_problem a;
  a.x = x; a.w = w; a.bias = bias; a.y = y; a.M = M; a.ldx = ldx; a.ldw = ldw; a.ldy = ldy;
  a.y2 = y2; a.ldy2 = ldy2; a.resid = resid; a.ldr = ldr; a.gate = gate; a.gate_stride = gate_stride;
  a.rows_per_batch = rows_per_batch;
  if (M < 0 || N < 0 || K <= 0) return set_error(FLUXB_ERR_BAD_ARG, "linear: bad sizes");
  return fluxb_linear_grouped(&a, 1, N, K, epi, split, epi2, round_before_act, stream);
}
