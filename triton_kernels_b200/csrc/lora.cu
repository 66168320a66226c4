// A projection shared by all requests plus one low-rank adapter per request:
//   y[m] = act(x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T),   a = adapter[m / L]   (a < 0: no adapter)
// x holds L rows per request.  An adapter index outside [-1, n) leaves its request without an adapter and is
// recorded in the device status word (site 81).
#include "vec.cuh"

namespace fluxb {

struct LoraArgs {
  const __nv_bfloat16 *x, *w, *bias, *a, *b;
  const float* scale;  // nullptr: ones
  const void* adapter;
  __nv_bfloat16* y;
  float* t;  // [M, R]
  int64_t M, L, ldx, ldw, ldy;
  int N, K, R, n_adapters, adapter_is64, epi;
  DeviceStatus* status;
};

__device__ __forceinline__ int adapter_of(const LoraArgs& p, int64_t request) {
  const int64_t a = p.adapter_is64 ? static_cast<const int64_t*>(p.adapter)[request]
                                   : static_cast<const int32_t*>(p.adapter)[request];
  if (a < -1 || a >= p.n_adapters) {
    report_error(p.status, FLUXB_ERR_BAD_ARG, 81);
    return -1;
  }
  return static_cast<int>(a);
}

// t[m, j] = s_a sum_k x[m, k] A_a[j, k]: one warp per (row, rank).
__global__ void __launch_bounds__(256) lora_shrink_any_kernel(const LoraArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= p.M * p.R) return;
  const int64_t m = i / p.R;
  const int j = (int)(i % p.R);
  const int a = adapter_of(p, m / p.L);
  float s = 0.f;
  if (a >= 0) {
    const __nv_bfloat16* x = p.x + m * p.ldx;
    const __nv_bfloat16* w = p.a + ((int64_t)a * p.R + j) * p.K;
    for (int k = threadIdx.x & 31; k < p.K; k += 32) s = fmaf(__bfloat162float(x[k]), __bfloat162float(w[k]), s);
    s = warp_sum(s) * (p.scale != nullptr ? p.scale[a] : 1.f);
  }
  if ((threadIdx.x & 31) == 0) p.t[i] = s;
}

// 64 x 64 tiles, 4 x 4 outputs per thread, fp32 products.
__global__ void __launch_bounds__(256) lora_gemm_any_kernel(const LoraArgs p) {
  __shared__ float xs[16][65], ws[16][65];
  const int n0 = blockIdx.x * 64;
  const int64_t m0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int r = i >> 4, k = k0 + (i & 15);
      xs[i & 15][r] = m0 + r < p.M && k < p.K ? __bfloat162float(p.x[(m0 + r) * p.ldx + k]) : 0.f;
      ws[i & 15][r] = n0 + r < p.N && k < p.K ? __bfloat162float(p.w[(int64_t)(n0 + r) * p.ldw + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty + 16 * i], ws[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= p.M) continue;
    const int a = adapter_of(p, m / p.L);
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n >= p.N) continue;
      float v = acc[i][j] + (p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.f);
      if (a >= 0)
        for (int r = 0; r < p.R; ++r)
          v = fmaf(p.t[m * p.R + r], __bfloat162float(p.b[((int64_t)a * p.N + n) * p.R + r]), v);
      if (p.epi == FLUXB_EPI_GELU) v = gelu_tanh(v);
      p.y[m * p.ldy + n] = __float2bfloat16_rn(v);
    }
  }
}

}  // namespace fluxb

using namespace fluxb;

extern "C" int64_t fluxb_linear_lora_scratch_bytes(int64_t M, int64_t N, int64_t K, int64_t R) {
  (void)N; (void)K;
  return M <= 0 || R <= 0 ? 0 : M * R * 4;
}

extern "C" int fluxb_linear_lora(const void* x, const void* w, const void* bias, void* y, const void* lora_a,
                                 const void* lora_b, const float* lora_scale, const void* adapter, int adapter_is64,
                                 void* scratch, int64_t B, int64_t L, int64_t N, int64_t K, int64_t R, int64_t n_adapters,
                                 int64_t ldx, int64_t ldw, int64_t ldy, int epi, fluxb_stream_t stream) {
  auto off16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (epi != FLUXB_EPI_NONE && epi != FLUXB_EPI_GELU) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: epilogue %d", epi);
  if (B < 0 || L < 0 || N < 0 || K <= 0 || R <= 0 || n_adapters <= 0) return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: bad sizes");
  if (K % 8 || N % 8 || ldx % 8 || ldw % 8 || ldy % 8 || ldx < K || ldw < K || ldy < N)
    return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: K, N and row strides must be multiples of 8 (and strides no shorter than rows)");
  if (B == 0 || L == 0 || N == 0) return FLUXB_OK;
  const int64_t M = B * L;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > INT32_MAX / 2 || R > 1024 || n_adapters > INT32_MAX / 2)
    return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: dimension too large");
  if (!x || !w || !y || !lora_a || !lora_b || !adapter || !scratch) return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: null pointer");
  if (off16(x) || off16(w) || off16(bias) || off16(y) || off16(lora_a) || off16(lora_b) || off16(scratch))
    return set_error(FLUXB_ERR_BAD_ARG, "linear_lora: pointers must be 16-byte aligned");
  typedef const __nv_bfloat16* P;
  LoraArgs p{static_cast<P>(x), static_cast<P>(w), static_cast<P>(bias), static_cast<P>(lora_a), static_cast<P>(lora_b),
             lora_scale, adapter, static_cast<__nv_bfloat16*>(y), static_cast<float*>(scratch), M, L, ldx, ldw, ldy,
             (int)N, (int)K, (int)R, (int)n_adapters, adapter_is64, epi, device_status_ptr()};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((M + 63) / 64 > 65535 || (M * R + 7) / 8 > INT32_MAX) return set_error(FLUXB_ERR_UNSUPPORTED, "linear_lora: too many rows");
  lora_shrink_any_kernel<<<(unsigned)((M * R + 7) / 8), 256, 0, st>>>(p);
  lora_gemm_any_kernel<<<dim3((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64)), 256, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "linear_lora: launch failed: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}
