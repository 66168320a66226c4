// A projection shared by all requests plus one low-rank adapter per request:
//   y[m] = act(x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T),   a = adapter[m / L]   (a < 0: no adapter)
// x holds L rows per request.  Two launches: the low-rank rows t = s_a (x A_a^T) here, then the projection with
// the adapters' second half fused in (gemm_tcgen05.cu).  t is carried as two bf16 parts, high and low
// (t = high + low to 2^-17 of |t|), so that the tensor cores take it without the rounding a single bf16 would put
// between the two products.  Both kernels may start while the one in front of them ends: the first waits for everything
// before it (in every block, before anything is read), only then does it let the second start, and that one waits for
// t alone: its x, W, bias, indices and B, which it reads without a wait of its own and partly by the read-only path, are
// complete because of that order.  So pdl_release() stays behind pdl_wait() in every kernel of this file, and a block that
// leaves early leaves behind its wait.  In a stream of such calls that took 16.4 us to 13.2 (48 x 5 rows, 1024 -> 4096, 16 adapters) and 26.0 to 24.2 (8 x 1
// row, 3072 -> 18432).  An adapter index outside [-1, n) leaves its request without an adapter and is recorded
// in the device status word (site 81).
#include "lora.cuh"
#include "vec.cuh"

namespace fluxb {

namespace shrink {
constexpr int BM = 128;
constexpr int BK = 64;
constexpr int THREADS = 192;
constexpr int MAX_STAGES = 12;
constexpr int MAX_SMEM = 200 * 1024;

struct Params {
  CUtensorMap tm_x;  // [M, K], box 64 x box_rows
  CUtensorMap tm_a;  // [n, R, K], box 64 x rpad
  RequestAdapters req;
  const float* scale;  // nullptr: ones
  __nv_bfloat16* t;    // [M, low.ld()]
  LowRank low;
  int L, tiles, tiles_per_request, box_rows;
  int num_kb, ksplit, rpad, stages, subs, tmem_cols;  // subs: 64-wide K steps per ring slot
  DeviceStatus* status;
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// One cluster of `ksplit` CTAs per 128 rows of one request (ksplit 1: clusters of two CTAs that do not meet): each CTA
// multiplies its share of K (x and A tiles by TMA, fp32 accumulator in TMEM, N = the rank in sixteens), leaves its
// partial sums in shared memory, and after a cluster barrier each takes a share of the outputs, adds the partial sums
// in a fixed order, scales, splits and stores.
__global__ void __launch_bounds__(THREADS, 1) lora_shrink_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int in_cluster = (int)cluster_ctarank(), rank = p.ksplit > 1 ? in_cluster : 0;
  const int tile = blockIdx.x / p.ksplit;
  if (tile >= p.tiles) {
    pdl_wait();  // (a block that leaves lets the projection start, too)
    return;
  }
  const int request = tile / p.tiles_per_request;
  const int l0 = (tile - request * p.tiles_per_request) * BM;
  const int row0 = request * p.L + l0;
  const int rows = min(BM, p.L - l0);
  pdl_wait();
  const int adapter = p.req.of_request(request);
  if (adapter < 0) {  // the whole cluster leaves; nobody reads these rows of t
    if (threadIdx.x == 0 && rank == 0 && l0 == 0 && p.req.raw(request) != -1) report_error(p.status, FLUXB_ERR_BAD_ARG, 81);
    return;
  }
  constexpr int x_bytes = BM * BK * 2;
  const int a_bytes = p.rpad * BK * 2, slot_x = p.subs * x_bytes, stage_bytes = slot_x + p.subs * a_bytes;
  const int kb0 = rank * p.num_kb / p.ksplit, kb1 = (rank + 1) * p.num_kb / p.ksplit;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&acc_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&p.tm_x);
    tma_prefetch_desc(&p.tm_a);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  // behind pdl_wait() above, on which the projection's own reads rely, and behind the TMEM allocation: the projection's
  // blocks take all of an SM's TMEM
  pdl_release();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t bytes = (uint32_t)(p.box_rows + p.rpad) * BK * 2;
    for (int kb = kb0; kb < kb1; kb += p.subs) {
      const int subs = min(p.subs, kb1 - kb);
      if (!__all_sync(0xffffffffu, mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 82))) break;
      uint8_t* dst = smem + stage * stage_bytes;
      if (elect_one()) {
        mbar_expect_tx(&full_bar[stage], subs * bytes);
        // rows behind the request are loaded and never stored; rows of the tile that no box covers are never read out
        for (int i = 0; i < subs; ++i) {
          tma_load_2d(dst + i * x_bytes, &p.tm_x, &full_bar[stage], (kb + i) * BK, row0);
          tma_load_3d(dst + slot_x + i * a_bytes, &p.tm_a, &full_bar[stage], (kb + i) * BK, 0, adapter);
        }
      }
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_bf16(BM, p.rpad, 0, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; kb += p.subs) {
      const int subs = min(p.subs, kb1 - kb);
      ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 83));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t a_addr = smem_u32(smem + stage * stage_bytes);
      const uint64_t adesc = make_smem_desc(a_addr, 16, 1024);
      const uint64_t bdesc = make_smem_desc(a_addr + slot_x, 16, 1024);
      if (elect_one()) {
        for (int i = 0; i < subs; ++i) {
          const uint64_t ad = adesc + i * (x_bytes >> 4), bd = bdesc + i * (a_bytes >> 4);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_ss(tmem_base, ad + 2 * k, bd + 2 * k, idesc, (kb > kb0 || i > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
      }
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (ok && elect_one()) umma_commit(&acc_full);
    __syncwarp();
  }
  // [128][rpad + 4], the ring's memory, free once the last MMA is done; the four floats behind each row spread the rows
  // over the banks
  float* part = reinterpret_cast<float*>(smem);
  const int pitch = p.rpad + 4;
  bool ok = true;
  if (warp >= 2) {
    const int quad = warp & 3;
    ok = mbar_wait(&acc_full, 0, abort_flag, p.status, 84);
    ok = __all_sync(0xffffffffu, ok);
    if (ok && quad * 32 < rows) {
      tc_fence_after_sync();
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
      for (int c = 0; c < p.rpad; c += 16) {
        uint32_t r[16];
        tmem_ld_x16(t_addr + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<uint4*>(part + (quad * 32 + lane) * pitch + c + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
  if (p.ksplit > 1) cluster_sync_all();
  const float scale = p.scale != nullptr ? p.scale[adapter] : 1.f;
  const int t_ld = p.low.ld();
  const int eights = p.rpad / 8;
  for (int i = rank * THREADS + threadIdx.x; i < eights * rows; i += p.ksplit * THREADS) {
    const int row = i / eights, c8 = (i - row * eights) * 8;
    float4 lo4[8], hi4[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (s < p.ksplit) {
        const uint32_t src = map_to_cta(smem_u32(part + row * pitch + c8), (uint32_t)(in_cluster - rank + s));
        lo4[s] = ld_cluster_f32x4(src);
        hi4[s] = ld_cluster_f32x4(src + 16);
      }
    }
    float v[8] = {};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (s < p.ksplit) {
        v[0] += lo4[s].x; v[1] += lo4[s].y; v[2] += lo4[s].z; v[3] += lo4[s].w;
        v[4] += hi4[s].x; v[5] += hi4[s].y; v[6] += hi4[s].z; v[7] += hi4[s].w;
      }
    }
    // the ranks behind R, which the projection multiplies, too: zeros would be NaN here beside an infinite x
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c8 + e < p.low.R ? v[e] : 0.f;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = v[2 * e] * scale, b = v[2 * e + 1] * scale;
      hi[e] = pack_bf16(a, b);
      // an infinite product has no low part (inf - inf would be NaN)
      const float la = a - bf16_lo(hi[e]), lb = b - bf16_hi(hi[e]);
      lo[e] = pack_bf16(isinf(bf16_lo(hi[e])) ? 0.f : la, isinf(bf16_hi(hi[e])) ? 0.f : lb);
    }
    __nv_bfloat16* dst = p.t + (int64_t)(row0 + row) * t_ld + p.low.column(c8);
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(dst + p.low.group) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  if (p.ksplit > 1) cluster_sync_all();  // no CTA leaves while another reads its partial sums
}

}  // namespace shrink

static int launch_shrink(const void* x, int64_t ldx, const void* lora_a, const float* scale, void* t, const RequestAdapters& req,
                         int64_t B, int64_t L, int64_t K, const LowRank& low, int ksplit, cudaStream_t st) {
  using namespace shrink;
  Params p;
  p.req = req;
  p.low = low;
  p.scale = scale;
  p.t = static_cast<__nv_bfloat16*>(t);
  p.L = (int)L;
  p.tiles_per_request = (int)((L + BM - 1) / BM);
  p.box_rows = (int)(L < BM ? (L + 7) / 8 * 8 : BM);
  p.rpad = low.units * 16;
  p.num_kb = (int)((K + BK - 1) / BK);
  p.status = device_status_ptr();
  const int64_t tiles = B * p.tiles_per_request;
  p.tiles = (int)tiles;
  p.ksplit = ksplit;
  const int step_bytes = BM * BK * 2 + p.rpad * BK * 2;
  // two K steps per slot where three slots fit: a slot costs its warps some 500 cycles each
  p.subs = MAX_SMEM / step_bytes >= 6 ? 2 : 1;
  const int stage_bytes = p.subs * step_bytes;
  const int steps = ((p.num_kb + p.ksplit - 1) / p.ksplit + p.subs - 1) / p.subs;
  p.stages = MAX_SMEM / stage_bytes < MAX_STAGES ? MAX_SMEM / stage_bytes : MAX_STAGES;
  if (p.stages > steps) p.stages = steps;
  int smem = p.stages * stage_bytes;
  if (smem < (p.rpad + 4) * BM * 4) smem = (p.rpad + 4) * BM * 4;
  smem += 1024;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.rpad) p.tmem_cols *= 2;
  const int64_t M = B * L;
  {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)M}, strides[1] = {(uint64_t)ldx * 2};
    const uint32_t box[2] = {BK, (uint32_t)p.box_rows};
    int rc = encode_tmap_bf16(&p.tm_x, x, 2, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  {
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)low.R, (uint64_t)req.n_adapters};
    const uint64_t strides[2] = {(uint64_t)K * 2, (uint64_t)(low.R * K) * 2};
    const uint32_t box[3] = {BK, (uint32_t)p.rpad, 1};
    int rc = encode_tmap_bf16(&p.tm_a, lora_a, 3, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  cudaError_t e = cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM + 1024);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: cannot set shared memory size: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  // Where K is not split, a cluster is two neighbouring tiles: the projection's CTA pairs start beside this kernel and
  // need both SMs of a pair free.
  const unsigned cluster = ksplit > 1 ? (unsigned)ksplit : 2;
  cfg.gridDim = dim3((unsigned)((tiles * ksplit + cluster - 1) / cluster * cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, lora_shrink_kernel, p);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

// ----------------------------------------------------------------------------------------
// Low-rank rows of short requests (up to eight rows).  The tensor-core kernel above takes 7 us for eight requests of one
// row, almost all of it set-up (tensor maps, TMEM, cluster barriers); the first kernel here 4.7.  For 48 requests of five
// rows, K 1024, rank 64, the second takes 3.4, and took 7.9 with a block per four ranks and FMAs.  They need next to no
// shared memory, so the projection can start beside them.
// ----------------------------------------------------------------------------------------
namespace shrink {
constexpr int SHORT = kLoraShort;
struct ShortParams {
  const __nv_bfloat16 *x, *a;
  const float* scale;
  __nv_bfloat16* t;
  RequestAdapters req;
  LowRank low;
  int64_t ldx;
  int K;
  DeviceStatus* status;
};

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// One value of t, scaled and split; a rank behind R (zeros, which would be NaN beside an infinite x) is zero.
__device__ __forceinline__ void store_low_rank(const ShortParams& p, int adapter, int64_t row, int j, float v) {
  v = j < p.low.R ? v * (p.scale != nullptr ? p.scale[adapter] : 1.f) : 0.f;
  const __nv_bfloat16 hi = __float2bfloat16_rn(v);
  const float h = __bfloat162float(hi);
  __nv_bfloat16* dst = p.t + row * p.low.ld() + p.low.column(j);
  dst[0] = hi;
  dst[p.low.group] = __float2bfloat16_rn(isinf(h) ? 0.f : v - h);
}

// Few requests: a block per rank, four warps sharing K, so that the reading of A is spread over the machine.
__global__ void __launch_bounds__(128) lora_shrink_one_kernel(const ShortParams p) {
  __shared__ float red[4][SHORT];
  const int ranks = p.low.units * 16;  // the ranks behind R are zeros: the tensor cores multiply them, too
  const int request = blockIdx.x / ranks, j = blockIdx.x - request * ranks;
  const int L = p.req.length, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  // behind the wait, on which the projection's own reads rely; its stream of W does not get in front: the loads here are
  // all on their way within the launch
  pdl_release();
  const int adapter = p.req.of_request(request);
  if (adapter < 0) {
    if (j == 0 && threadIdx.x == 0 && p.req.raw(request) != -1) report_error(p.status, FLUXB_ERR_BAD_ARG, 81);
    return;
  }
  const __nv_bfloat16* a = p.a + ((int64_t)adapter * p.low.R + j) * p.K;
  const __nv_bfloat16* x = p.x + (int64_t)request * L * p.ldx;
  float acc[SHORT] = {};
  constexpr int kAhead = 4;  // steps whose loads are in flight together
  for (int k0 = threadIdx.x * 8; k0 < p.K; k0 += 1024 * kAhead) {
    uint4 av[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      av[i] = k0 + i * 1024 < p.K && j < p.low.R ? ld_u4(a + k0 + i * 1024) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (k0 + i * 1024 >= p.K) break;
      const uint32_t aw[4] = {av[i].x, av[i].y, av[i].z, av[i].w};
#pragma unroll
      for (int l = 0; l < SHORT; ++l) {
        if (l < L) {
          const uint4 xv = ld_u4(x + l * p.ldx + k0 + i * 1024);
          const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[l] = fmaf(bf16_hi(aw[e]), bf16_hi(xw[e]), fmaf(bf16_lo(aw[e]), bf16_lo(xw[e]), acc[l]));
        }
      }
    }
  }
#pragma unroll
  for (int l = 0; l < SHORT; ++l) {
    if (l < L) {
      const float s = warp_sum(acc[l]);
      if (lane == 0) red[warp][l] = s;
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < L) {
    const int l = threadIdx.x;
    store_low_rank(p, adapter, request * (int64_t)L + l, j, red[0][l] + red[1][l] + red[2][l] + red[3][l]);
  }
}

// Many requests: a block per request and sixteen ranks, which reads x a sixteenth as often.  Eight warps share K; the
// products run as mma.m16n8k16 with A's rows on the M side and the rows of x on the N side, the fragments straight from
// global memory: a lane reads 16 consecutive bytes of two rows of A and one of x and uses them for two MMAs (the order of
// k does not matter as long as both sides agree).  Bound by latency.
__global__ void __launch_bounds__(256) lora_shrink_mma_kernel(const ShortParams p) {
  __shared__ float red[8][16][SHORT + 1];
  const int request = blockIdx.x / p.low.units, j0 = (blockIdx.x - request * p.low.units) * 16;
  const int L = p.req.length, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_release();  // (behind the wait, as above)
  const int adapter = p.req.of_request(request);
  if (adapter < 0) {
    if (j0 == 0 && threadIdx.x == 0 && p.req.raw(request) != -1) report_error(p.status, FLUXB_ERR_BAD_ARG, 81);
    return;
  }
  const int g = lane >> 2, t4 = lane & 3;
  const __nv_bfloat16* a = p.a + ((int64_t)adapter * p.low.R + j0 + g) * p.K;
  const __nv_bfloat16* x = p.x + ((int64_t)request * L + g) * p.ldx;
  const bool r0 = j0 + g < p.low.R, r1 = j0 + g + 8 < p.low.R, rx = g < L;
  const uint4 none = make_uint4(0, 0, 0, 0);
  float c[4] = {};
  constexpr int kAhead = 4;
  for (int k0 = warp * 32 + t4 * 8; k0 < p.K + t4 * 8; k0 += 256 * kAhead) {
    uint4 a0[kAhead], a1[kAhead], b[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k = k0 + i * 256;
      a0[i] = r0 && k < p.K ? ld_u4(a + k) : none;
      a1[i] = r1 && k < p.K ? ld_u4(a + (int64_t)8 * p.K + k) : none;
      b[i] = rx && k < p.K ? ld_u4(x + k) : none;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      mma_16x8x16(c, a0[i].x, a1[i].x, a0[i].y, a1[i].y, b[i].x, b[i].y);
      mma_16x8x16(c, a0[i].z, a1[i].z, a0[i].w, a1[i].w, b[i].z, b[i].w);
    }
  }
  red[warp][g][2 * t4] = c[0];
  red[warp][g][2 * t4 + 1] = c[1];
  red[warp][g + 8][2 * t4] = c[2];
  red[warp][g + 8][2 * t4 + 1] = c[3];
  __syncthreads();
  const int j = threadIdx.x & 15, l = threadIdx.x >> 4;
  if (l >= L) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) v += red[w][j][l];
  store_low_rank(p, adapter, request * (int64_t)L + l, j0 + j, v);
}
}  // namespace shrink

static int launch_shrink_short(const void* x, int64_t ldx, const void* lora_a, const float* scale, void* t,
                               const RequestAdapters& req, int64_t B, int64_t K, const LowRank& low, cudaStream_t st) {
  if (B * low.units * 16 > INT32_MAX) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: too many requests");
  shrink::ShortParams p{static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(lora_a), scale,
                        static_cast<__nv_bfloat16*>(t), req, low, ldx, (int)K, device_status_ptr()};
  const int64_t ranks = B * low.units * 16;
  const cudaError_t e = ranks >= 4 * sm_count() ? launch_after(shrink::lora_shrink_mma_kernel, (unsigned)(B * low.units), 256, 0, st, p)
                                                : launch_after(shrink::lora_shrink_one_kernel, (unsigned)ranks, 128, 0, st, p);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

// ----------------------------------------------------------------------------------------
// One to eight rows: the projection is a stream of W.  A block takes 16 output columns at a time; the 16 rows of W
// come through a ring in shared memory by bulk copies (a row of up to 6 KB each, 200 KB in flight per SM: the block keeps
// asking while it computes), and its eight warps share a piece's columns.  The products run as mma.m16n8k16 with W's
// rows on the M side and the rows of x on the N side; a lane reads 16 consecutive bytes of two W rows and uses them as
// its A fragments of two MMAs, with x's fragment taken from the same k positions: the order of k does not matter as
// long as both sides agree.  x's fragments stay in registers for all tiles (kPieces pieces of W; 0: read each time).
// The adapters are R more products per output, from t's two parts widened to fp32.
// Bound by HBM: 18432 x 3072, eight rows, 23.4 us with the low-rank rows (113 MB of W; 4.8 TB/s).  (With W loaded
// straight to registers, 98 KB in flight per SM: 27 us; with 2 KB copies: 25 us.)
// ----------------------------------------------------------------------------------------
namespace rows {
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32 + 32 + 128;  // and a warp that issues the copies, and four that finish the outputs
constexpr int AHEAD = 8;                  // eights of ranks that are asked for a tile ahead
constexpr int WHOLE = 3072;               // rows of up to so many columns are one piece ...
constexpr int PIECE = 1536;               // ... longer ones are cut into pieces of so many
constexpr int MAX_SLOTS = 12;
constexpr int RING_BYTES = 200 * 1024;

struct Params {
  const __nv_bfloat16 *x, *w, *bias, *t, *lora_b;
  __nv_bfloat16* y;
  RequestAdapters req;
  LowRank low;
  int64_t ldx, ldw, ldy, ldb;
  int M, N, K, epi, tiles, piece, pieces, slots;
  DeviceStatus* status;
};

__device__ __forceinline__ float dot8(const uint4& b, const float* t, float acc) {
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = fmaf(bf16_hi(w[e]), t[2 * e + 1], fmaf(bf16_lo(w[e]), t[2 * e], acc));
  return acc;
}

// kPieces: pieces per row whose fragments of x are kept (0: read each time); kSteps: most 32-column steps of a warp per piece.
template <int kPieces, int kSteps>
__global__ void __launch_bounds__(THREADS, 1) lora_rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full_bar[MAX_SLOTS], empty_bar[MAX_SLOTS], red_full[2], red_empty[2];
  __shared__ float red[2][WARPS][16][9];
  __shared__ float t_s[8][256];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // 64 bytes behind each row: eight lanes that read two rows then touch all banks once
  const int pitch = p.piece * 2 + 64, slot_bytes = 16 * pitch;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.slots; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], WARPS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&red_full[i], WARPS);
      mbar_init(&red_empty[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  pdl_release();
  int slot = 0;
  uint32_t phase = 0;
  if (warp == WARPS) {
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const int rows = min(16, p.N - tile * 16);
      for (int piece = 0; piece < p.pieces; ++piece) {
        const uint32_t bytes = min(p.piece, p.K - piece * p.piece) * 2;
        bool ok = true;
        if (lane == 0) {
          ok = mbar_wait(&empty_bar[slot], phase ^ 1, abort_flag, p.status, 85);
          if (ok) mbar_expect_tx(&full_bar[slot], rows * bytes);
        }
        if (!__shfl_sync(0xffffffffu, (int)ok, 0)) return;
        if (lane < rows) {
          const __nv_bfloat16* src = p.w + (int64_t)(tile * 16 + lane) * p.ldw + piece * p.piece;
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           smem_u32(ring + slot * slot_bytes + lane * pitch)),
                       "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(&full_bar[slot]))
                       : "memory");
        }
        if (++slot == p.slots) { slot = 0; phase ^= 1; }
      }
    }
    return;
  }
  if (warp > WARPS) {
    // One thread per output of a tile: sums the eight warps' shares and adds bias and adapter.  Warps of their own,
    // which ask for their rows of B a tile ahead, because a tile's finish is all latency: done by the streaming
    // warps it cost a third of the time (29.8 us).
    const int e = threadIdx.x - (WARPS + 1) * 32;
    const int m = e >> 4, nl = e & 15;
    const int adapter = m < p.M ? p.req.of_row(m) : -1;
    const int ahead = min(p.low.R / 8, AHEAD);
    int parity = 0;
    uint32_t red_phase = 0;
    uint4 bv[AHEAD];
    float bias = 0.f;
    auto row_of_b = [&](int n) { return p.lora_b + ((int64_t)adapter * p.N + n) * p.ldb; };
    auto ask = [&](int tile) {
      const int n = tile * 16 + nl;
      if (m >= p.M || n >= p.N) return;
      if (p.bias != nullptr) bias = __bfloat162float(p.bias[n]);
      if (adapter < 0) return;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (i < ahead) bv[i] = __ldg(reinterpret_cast<const uint4*>(row_of_b(n) + i * 8));
    };
    ask(blockIdx.x);
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const int n = tile * 16 + nl;
      const bool mine = m < p.M && n < p.N;
      if (tile == (int)blockIdx.x) {  // t of the requests that have an adapter, widened
        pdl_wait();
        for (int i = e; i < p.M * p.low.R; i += 128) {
          const int mm = i / p.low.R, j = i - mm * p.low.R;
          float w = 0.f;
          if (p.req.of_row(mm) >= 0) {
            const __nv_bfloat16* src = p.t + (int64_t)mm * p.low.ld() + p.low.column(j);
            w = __bfloat162float(src[0]) + __bfloat162float(src[p.low.group]);
          }
          t_s[mm][j] = w;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      float v = bias, s = 0.f;
      if (mine && adapter >= 0) {
        const __nv_bfloat16* b = row_of_b(n);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (i < ahead) s = dot8(bv[i], &t_s[m][i * 8], s);
        int j = ahead * 8;
#pragma unroll 4
        for (; j + 8 <= p.low.R; j += 8) s = dot8(__ldg(reinterpret_cast<const uint4*>(b + j)), &t_s[m][j], s);
        for (; j < p.low.R; ++j) s = fmaf(__bfloat162float(b[j]), t_s[m][j], s);
      }
      if (tile + (int)gridDim.x < p.tiles) ask(tile + gridDim.x);
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait(&red_full[parity], red_phase, abort_flag, p.status, 88))) return;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[parity][w][nl][m];
      __syncwarp();
      if (lane == 0) mbar_arrive(&red_empty[parity]);
      v += s;
      if (p.epi == FLUXB_EPI_GELU) v = gelu_tanh(v);
      if (mine) p.y[m * p.ldy + n] = __float2bfloat16_rn(v);
      if ((parity ^= 1) == 0) red_phase ^= 1;
    }
    return;
  }
  const int g = lane >> 2, t4 = lane & 3;
  const int steps = p.piece / (WARPS * 32);  // of 32 columns per warp and piece
  const int col = warp * (p.piece / WARPS) + t4 * 8;
  // x, like the adapters' indices, the bias and B above, is read without a wait: the low-rank kernel in front has waited for
  // everything before it in every block by the time this one starts
  const __nv_bfloat16* xr = p.x + g * p.ldx;
  auto load_x = [&](int piece, int s) {
    const int k = piece * p.piece + col + s * 32;
    return g < p.M && s < steps && k < p.K ? __ldg(reinterpret_cast<const uint4*>(xr + k)) : make_uint4(0, 0, 0, 0);
  };
  uint4 bx[kPieces > 0 ? kPieces : 1][kSteps];
  if (kPieces > 0) {
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) bx[q][s] = load_x(q, s);
  }
  int parity = 0;
  uint32_t red_phase = 0;
  for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    float c[4] = {};
    auto work = [&](int piece, const uint4 (&b)[kSteps]) -> bool {
      if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[slot], phase, abort_flag, p.status, 86))) return false;
      const uint8_t* base = ring + slot * slot_bytes + g * pitch + col * 2;
      const bool whole = (piece + 1) * p.piece <= p.K;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s < steps) {
          uint4 a0 = *reinterpret_cast<const uint4*>(base + s * 64);
          uint4 a1 = *reinterpret_cast<const uint4*>(base + 8 * pitch + s * 64);
          if (!whole && piece * p.piece + col + s * 32 >= p.K) a0 = a1 = make_uint4(0, 0, 0, 0);  // behind the copy
          shrink::mma_16x8x16(c, a0.x, a1.x, a0.y, a1.y, b[s].x, b[s].y);
          shrink::mma_16x8x16(c, a0.z, a1.z, a0.w, a1.w, b[s].z, b[s].w);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[slot]);
      if (++slot == p.slots) { slot = 0; phase ^= 1; }
      return true;
    };
    bool ok = true;
    if (kPieces > 0) {
#pragma unroll
      for (int q = 0; q < kPieces; ++q) ok = ok && work(q, bx[q]);
    } else {
      for (int q = 0; ok && q < p.pieces; ++q) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) bx[0][s] = load_x(q, s);
        ok = work(q, bx[0]);
      }
    }
    ok = ok && __all_sync(0xffffffffu, mbar_wait(&red_empty[parity], red_phase ^ 1, abort_flag, p.status, 87));
    if (!ok) return;
    red[parity][warp][g][2 * t4] = c[0];
    red[parity][warp][g][2 * t4 + 1] = c[1];
    red[parity][warp][g + 8][2 * t4] = c[2];
    red[parity][warp][g + 8][2 * t4 + 1] = c[3];
    __syncwarp();
    if (lane == 0) mbar_arrive(&red_full[parity]);
    if ((parity ^= 1) == 0) red_phase ^= 1;
  }
}

}  // namespace rows

static int launch_rows(const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t, const void* lora_b,
                       const LowRank& low, int64_t ldb, const RequestAdapters& req, cudaStream_t st) {
  using namespace rows;
  Params p;
  typedef const __nv_bfloat16* P;
  p.x = static_cast<P>(a.x); p.w = static_cast<P>(a.w); p.bias = static_cast<P>(a.bias); p.t = static_cast<P>(t);
  p.lora_b = static_cast<P>(lora_b);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.req = req;
  p.low = low;
  p.ldx = a.ldx; p.ldw = a.ldw; p.ldy = a.ldy; p.ldb = ldb;
  p.M = (int)a.M; p.N = (int)N; p.K = (int)K; p.epi = epi;
  p.tiles = (int)((N + 15) / 16);
  p.piece = K <= WHOLE ? (int)((K + 255) / 256 * 256) : PIECE;
  p.pieces = (int)((K + p.piece - 1) / p.piece);
  p.status = device_status_ptr();
  const int slot_bytes = 16 * (p.piece * 2 + 64);
  // every block the same number of tiles
  const int per = (p.tiles + sm_count() - 1) / sm_count();
  const int grid = (p.tiles + per - 1) / per;
  p.slots = RING_BYTES / slot_bytes;
  if (p.slots > MAX_SLOTS) p.slots = MAX_SLOTS;
  if (p.slots > per * p.pieces) p.slots = per * p.pieces;
  auto kern = p.pieces == 1   ? (p.piece <= 1024 ? lora_rows_kernel<1, 4> : lora_rows_kernel<1, 12>)
              : p.pieces == 3 ? lora_rows_kernel<3, 6>
                              : lora_rows_kernel<0, 6>;  // (the fragments of more pieces spill)
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: cannot set shared memory size: %s", cudaGetErrorString(e));
  e = launch_after(kern, grid, THREADS, (size_t)p.slots * slot_bytes, st, p);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

}  // namespace fluxb

using namespace fluxb;

extern "C" int64_t fluxb_linear_lora_scratch_bytes(int64_t M, int64_t N, int64_t K, int64_t R) {
  (void)N; (void)K;
  return M <= 0 || R <= 0 ? 0 : M * LowRank(R).ld() * 2;
}

extern "C" int fluxb_linear_lora(const void* x, const void* w, const void* bias, void* y, const void* lora_a,
                                 const void* lora_b, const float* lora_scale, const void* adapter, int adapter_is64,
                                 void* scratch, int64_t B, int64_t L, int64_t N, int64_t K, int64_t R, int64_t n_adapters,
                                 int64_t ldx, int64_t ldw, int64_t ldy, int64_t ldb, int epi, fluxb_stream_t stream) {
  auto off16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (epi != FLUXB_EPI_NONE && epi != FLUXB_EPI_GELU) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: epilogue %d", epi);
  if (B < 0 || L < 0 || N < 0 || K <= 0 || R <= 0 || n_adapters <= 0) return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: bad sizes");
  if (K % 8 || N % 8 || ldx % 8 || ldw % 8 || ldy % 8 || ldb % 8 || ldx < K || ldw < K || ldy < N || ldb < R)
    return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: K, N and row strides must be multiples of 8 (and strides no shorter than rows)");
  if (B == 0 || L == 0 || N == 0) return FLUXB_OK;
  if (R > 256) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: rank %lld (at most 256)", (long long)R);
  const int64_t limit = INT32_MAX / 2;
  if (B > limit || L > limit || B * L > limit || N > limit || K > limit || n_adapters > limit)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: dimension too large");
  if (!x || !w || !y || !lora_a || !lora_b || !adapter || !scratch) return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: null pointer");
  if (off16(x) || off16(w) || off16(bias) || off16(y) || off16(lora_a) || off16(lora_b) || off16(scratch))
    return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: pointers must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const RequestAdapters req{adapter, adapter_is64, (int)L, (int)n_adapters};
  const LowRank low(R);
  const bool brief = L <= kLoraShort;
  const int64_t M = B * L;
  const LoraPlan plan = M <= 8 ? LoraPlan{} : plan_lora(M, N, K, req, low);
  int rc = brief ? launch_shrink_short(x, ldx, lora_a, lora_scale, scratch, req, B, K, low, st)
                 : launch_shrink(x, ldx, lora_a, lora_scale, scratch, req, B, L, K, low, plan.ksplit, st);
  if (rc != FLUXB_OK) return rc;
  fluxb_linear_problem a = {};
  a.x = x; a.w = w; a.bias = bias; a.y = y; a.M = M; a.ldx = ldx; a.ldw = ldw; a.ldy = ldy;
  a.rows_per_batch = 1;
  rc = a.M <= 8 ? launch_rows(a, N, K, epi, scratch, lora_b, low, ldb, req, st)
                : launch_lora_gemm(plan, a, N, K, epi, scratch, lora_b, low, ldb, req, st);
  if (rc != FLUXB_OK) return rc;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}
