// A projection shared by all requests plus one low-rank adapter per request:
//   y[m] = act(x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T),   a = adapter[m / L]   (a < 0: no adapter)
// x holds L rows per request.  Two launches: the low-rank rows t = s_a (x A_a^T) here, then the projection with
// the adapters' second half fused in (gemm_tcgen05.cu).  t is carried as two bf16 parts, high and low
// (t = high + low to 2^-17 of |t|), so that the tensor cores take it without the rounding a single bf16 would put
// between the two products.  An adapter index outside [-1, n) leaves its request without an adapter and is recorded
// in the device status word (site 81).
#include "lora.cuh"

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
  __nv_bfloat16* t;    // [M, units * 32]: per 16 ranks, 16 high parts then 16 low parts
  int L, tiles_per_request, box_rows;
  int num_kb, ksplit, rpad, stages, tmem_cols;
  DeviceStatus* status;
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// One cluster of `ksplit` CTAs per 128 rows of one request: each CTA multiplies its share of K (x and A tiles by TMA,
// fp32 accumulator in TMEM, N = the rank in sixteens), leaves its partial sums in shared memory, and after a cluster
// barrier each takes a share of the outputs, adds the partial sums in a fixed order, scales, splits and stores.
__global__ void __launch_bounds__(THREADS, 1) lora_shrink_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const int tile = blockIdx.x / p.ksplit;
  const int request = tile / p.tiles_per_request;
  const int l0 = (tile - request * p.tiles_per_request) * BM;
  const int row0 = request * p.L + l0;
  const int rows = min(BM, p.L - l0);
  const int adapter = p.req.of_request(request);
  if (adapter < 0) {  // the whole cluster leaves; nobody reads these rows of t
    if (threadIdx.x == 0 && rank == 0 && l0 == 0 && p.req.raw(request) != -1) report_error(p.status, FLUXB_ERR_BAD_ARG, 81);
    return;
  }
  const int stage_bytes = BM * BK * 2 + p.rpad * BK * 2;
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

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t bytes = (uint32_t)(p.box_rows + p.rpad) * BK * 2;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 82)) break;
        uint8_t* dst = smem + stage * stage_bytes;
        mbar_expect_tx(&full_bar[stage], bytes);
        // rows behind the request are loaded and never stored; rows of the tile that no box covers are never read out
        tma_load_2d(dst, &p.tm_x, &full_bar[stage], kb * BK, row0);
        tma_load_3d(dst + BM * BK * 2, &p.tm_a, &full_bar[stage], kb * BK, 0, adapter);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_bf16(BM, p.rpad, 0, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 83));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t a_addr = smem_u32(smem + stage * stage_bytes);
      const uint64_t adesc = make_smem_desc(a_addr, 16, 1024);
      const uint64_t bdesc = make_smem_desc(a_addr + BM * BK * 2, 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          umma_ss(tmem_base, adesc + 2 * k, bdesc + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
      }
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (ok && elect_one()) umma_commit(&acc_full);
    __syncwarp();
  }
  float* part = reinterpret_cast<float*>(smem);  // [rpad][128]: the ring's memory, free once the last MMA is done
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
        for (int e = 0; e < 16; ++e) part[(c + e) * BM + quad * 32 + lane] = __uint_as_float(r[e]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
  cluster_sync_all();
  const float scale = p.scale != nullptr ? p.scale[adapter] : 1.f;
  const int t_ld = p.rpad * 2;
  for (int i = rank * THREADS + threadIdx.x; i < p.rpad / 8 * BM; i += p.ksplit * THREADS) {
    const int row = i & (BM - 1), c8 = i / BM * 8;
    if (row >= rows) continue;
    float v[8] = {};
    for (int s = 0; s < p.ksplit; ++s) {
      const uint32_t src = map_to_cta(smem_u32(part + c8 * BM + row), (uint32_t)s);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += ld_cluster_f32(src + e * BM * 4);
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = v[2 * e] * scale, b = v[2 * e + 1] * scale;
      hi[e] = pack_bf16(a, b);
      // an infinite product has no low part (inf - inf would be NaN)
      const float la = a - bf16_lo(hi[e]), lb = b - bf16_hi(hi[e]);
      lo[e] = pack_bf16(isinf(bf16_lo(hi[e])) ? 0.f : la, isinf(bf16_hi(hi[e])) ? 0.f : lb);
    }
    __nv_bfloat16* dst = p.t + (int64_t)(row0 + row) * t_ld + c8 / 16 * 32 + (c8 & 8);
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(dst + 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  cluster_sync_all();  // no CTA leaves while another reads its partial sums
}

}  // namespace shrink

static int launch_shrink(const void* x, int64_t ldx, const void* lora_a, const float* scale, void* t, const RequestAdapters& req,
                         int64_t B, int64_t L, int64_t K, int64_t R, cudaStream_t st) {
  using namespace shrink;
  Params p;
  p.req = req;
  p.scale = scale;
  p.t = static_cast<__nv_bfloat16*>(t);
  p.L = (int)L;
  p.tiles_per_request = (int)((L + BM - 1) / BM);
  p.box_rows = (int)(L < BM ? (L + 7) / 8 * 8 : BM);
  p.rpad = (int)((R + 15) / 16 * 16);
  p.num_kb = (int)((K + BK - 1) / BK);
  p.status = device_status_ptr();
  const int64_t tiles = B * p.tiles_per_request;
  // K is split until the clusters fill the machine, as long as a CTA keeps four 64-wide steps.
  p.ksplit = 1;
  while (p.ksplit < 8 && tiles * p.ksplit * 2 <= sm_count() && p.num_kb >= p.ksplit * 2 * 4) p.ksplit *= 2;
  const int steps = (p.num_kb + p.ksplit - 1) / p.ksplit;
  const int stage_bytes = BM * BK * 2 + p.rpad * BK * 2;
  p.stages = MAX_SMEM / stage_bytes < MAX_STAGES ? MAX_SMEM / stage_bytes : MAX_STAGES;
  if (p.stages > steps) p.stages = steps;
  int smem = p.stages * stage_bytes;
  if (smem < p.rpad * BM * 4) smem = p.rpad * BM * 4;
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
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)R, (uint64_t)req.n_adapters};
    const uint64_t strides[2] = {(uint64_t)K * 2, (uint64_t)R * K * 2};
    const uint32_t box[3] = {BK, (uint32_t)p.rpad, 1};
    int rc = encode_tmap_bf16(&p.tm_a, lora_a, 3, dims, strides, box);
    if (rc != FLUXB_OK) return rc;
  }
  cudaError_t e = cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM + 1024);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: cannot set shared memory size: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.ksplit));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.ksplit;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, lora_shrink_kernel, p);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}

// ----------------------------------------------------------------------------------------
// One to eight rows: the projection is a stream of W.  A block takes 16 output columns, its warps share K; a warp's
// lane loads 16 bytes of two W rows and uses them as the A fragments of mma.m16n8k16 (W's columns are the M side, the
// rows of x the N side), with x's fragment loaded from the same k positions: the order of k does not matter as long as
// both sides agree, so no shuffle or shared memory stands between the load and the product.  All 24 loads of a step
// are in flight at once, and those of the next step leave before the current one is summed over the warps.  The
// adapters are 2 R more products per output, from the high and low parts of t, in the epilogue.
// ----------------------------------------------------------------------------------------
namespace rows {
constexpr int SLICE = 384;  // k per warp and step: 12 fragments of 32
constexpr int STEPS = SLICE / 32;
constexpr int MAX_WARPS = 8;

struct Params {
  const __nv_bfloat16 *x, *w, *bias, *t, *lora_b;
  __nv_bfloat16* y;
  RequestAdapters req;
  int64_t ldx, ldw, ldy, ldb;
  int M, N, K, R, rpad, epi, tiles, slices;  // slices: steps of a warp per tile
};

__device__ __forceinline__ uint4 ld_or_zero(const __nv_bfloat16* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// sum of t[j] * b[j] over eight ranks; t as high and low parts
__device__ __forceinline__ float dot8(const uint4& b, const float* t, float acc) {
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = fmaf(bf16_hi(w[e]), t[2 * e + 1], fmaf(bf16_lo(w[e]), t[2 * e], acc));
  return acc;
}

// kOne: a warp's share of K is one step, and its fragments of x stay in registers for all tiles.
template <bool kOne>
__global__ void __launch_bounds__(MAX_WARPS * 32, 1) lora_rows_kernel(const Params p) {
  __shared__ float red[2][MAX_WARPS][16][9];
  __shared__ float t_s[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const __nv_bfloat16* xr = p.x + g * p.ldx;
  uint4 bx[STEPS], a0[STEPS], a1[STEPS];
  auto load_x = [&](int slice) {
    const int k0 = (slice * warps + warp) * SLICE + t4 * 8;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) bx[s] = ld_or_zero(xr + k0 + s * 32, g < p.M && k0 + s * 32 < p.K);
  };
  auto load_w = [&](int tile, int slice) {
    const int k0 = (slice * warps + warp) * SLICE + t4 * 8;
    const int n = tile * 16 + g;
    const __nv_bfloat16* w0 = p.w + n * p.ldw + k0;
    const __nv_bfloat16* w1 = w0 + 8 * p.ldw;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bool in = k0 + s * 32 < p.K;
      a0[s] = ld_or_zero(w0 + s * 32, in && n < p.N);
      a1[s] = ld_or_zero(w1 + s * 32, in && n + 8 < p.N);
    }
  };
  if (kOne) load_x(0);
  int tile = blockIdx.x;
  load_w(tile, 0);
  // t of the requests that have an adapter, widened
  for (int i = threadIdx.x; i < p.M * p.rpad; i += blockDim.x) {
    const int m = i / p.rpad, j = i - m * p.rpad;
    float v = 0.f;
    if (p.req.of_row(m) >= 0) {
      const __nv_bfloat16* src = p.t + (int64_t)m * p.rpad * 2 + j / 16 * 32 + j % 16;
      v = __bfloat162float(src[0]) + __bfloat162float(src[16]);
    }
    t_s[m][j] = v;
  }
  int buf = 0;
  for (; tile < p.tiles; tile += gridDim.x) {
    float c[4] = {};
    for (int slice = 0; slice < (kOne ? 1 : p.slices); ++slice) {
      if (!kOne) load_x(slice);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        mma_16x8x16(c, a0[s].x, a1[s].x, a0[s].y, a1[s].y, bx[s].x, bx[s].y);
        mma_16x8x16(c, a0[s].z, a1[s].z, a0[s].w, a1[s].w, bx[s].z, bx[s].w);
      }
      if (!kOne && slice + 1 < p.slices) load_w(tile, slice + 1);
      else if (tile + (int)gridDim.x < p.tiles) load_w(tile + gridDim.x, 0);
    }
    red[buf][warp][g][2 * t4] = c[0];
    red[buf][warp][g][2 * t4 + 1] = c[1];
    red[buf][warp][g + 8][2 * t4] = c[2];
    red[buf][warp][g + 8][2 * t4 + 1] = c[3];
    __syncthreads();  // the other buffer's readers are through before anyone gets here again
    for (int i = threadIdx.x; i < 128; i += blockDim.x) {
      const int m = i >> 4, n = tile * 16 + (i & 15);
      if (m >= p.M || n >= p.N) continue;
      float v = p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.f;
      for (int w = 0; w < warps; ++w) v += red[buf][w][i & 15][m];
      const int a = p.req.of_row(m);
      if (a >= 0) {
        const __nv_bfloat16* b = p.lora_b + ((int64_t)a * p.N + n) * p.ldb;
        float s = 0.f;
        int j = 0;
        for (; j + 8 <= p.R; j += 8) s = dot8(__ldg(reinterpret_cast<const uint4*>(b + j)), &t_s[m][j], s);
        for (; j < p.R; ++j) s = fmaf(__bfloat162float(b[j]), t_s[m][j], s);
        v += s;
      }
      if (p.epi == FLUXB_EPI_GELU) v = gelu_tanh(v);
      p.y[m * p.ldy + n] = __float2bfloat16_rn(v);
    }
    buf ^= 1;
  }
}

}  // namespace rows

static int launch_rows(const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t, const void* lora_b,
                       int64_t R, int64_t ldb, const RequestAdapters& req, cudaStream_t st) {
  rows::Params p;
  typedef const __nv_bfloat16* P;
  p.x = static_cast<P>(a.x); p.w = static_cast<P>(a.w); p.bias = static_cast<P>(a.bias); p.t = static_cast<P>(t);
  p.lora_b = static_cast<P>(lora_b);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.req = req;
  p.ldx = a.ldx; p.ldw = a.ldw; p.ldy = a.ldy; p.ldb = ldb;
  p.M = (int)a.M; p.N = (int)N; p.K = (int)K; p.R = (int)R; p.rpad = (int)((R + 15) / 16 * 16); p.epi = epi;
  p.tiles = (int)((N + 15) / 16);
  int warps = (int)((K + rows::SLICE - 1) / rows::SLICE);
  if (warps > rows::MAX_WARPS) warps = rows::MAX_WARPS;
  p.slices = (int)((K + rows::SLICE * warps - 1) / (rows::SLICE * warps));
  // every block the same number of tiles, eight warps per SM
  const int most = sm_count() * (rows::MAX_WARPS / warps);
  const int per = (p.tiles + most - 1) / most;
  const int grid = (p.tiles + per - 1) / per;
  if (p.slices == 1) rows::lora_rows_kernel<true><<<grid, warps * 32, 0, st>>>(p);
  else rows::lora_rows_kernel<false><<<grid, warps * 32, 0, st>>>(p);
  return FLUXB_OK;
}

}  // namespace fluxb

using namespace fluxb;

extern "C" int64_t fluxb_linear_lora_scratch_bytes(int64_t M, int64_t N, int64_t K, int64_t R) {
  (void)N; (void)K;
  return M <= 0 || R <= 0 ? 0 : M * ((R + 15) / 16) * 64;
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
  int rc = launch_shrink(x, ldx, lora_a, lora_scale, scratch, req, B, L, K, R, st);
  if (rc != FLUXB_OK) return rc;
  fluxb_linear_problem a = {};
  a.x = x; a.w = w; a.bias = bias; a.y = y; a.M = B * L; a.ldx = ldx; a.ldw = ldw; a.ldy = ldy;
  a.rows_per_batch = 1;
  rc = a.M <= 8 ? launch_rows(a, N, K, epi, scratch, lora_b, R, ldb, req, st)
                : launch_lora_gemm(a, N, K, epi, scratch, lora_b, R, ldb, req, st);
  if (rc != FLUXB_OK) return rc;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}
