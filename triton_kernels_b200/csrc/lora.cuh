// What the low-rank adapter kernels (lora.cu) and the projection they feed (gemm_tcgen05.cu) share.
#pragma once

#include "common.cuh"

namespace fluxb {

// Which adapter a row uses: rows come in requests of `length` rows, each with an index on the device.
struct RequestAdapters {
  const void* index;  // [requests], int32 or int64
  int is64;
  int length;
  int n_adapters;
  __device__ __forceinline__ int64_t raw(int request) const {
    return is64 ? static_cast<const int64_t*>(index)[request] : static_cast<const int32_t*>(index)[request];
  }
  // -1 for none and for anything outside the adapters.
  __device__ __forceinline__ int of_request(int request) const {
    const int64_t a = raw(request);
    return a >= 0 && a < n_adapters ? static_cast<int>(a) : -1;
  }
  __device__ __forceinline__ int of_row(int row) const { return of_request(row / length); }
};

int launch_lora_gemm(const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t, const void* lora_b,
                     int64_t R, int64_t ldb, const RequestAdapters& req, cudaStream_t st);

}  // namespace fluxb
