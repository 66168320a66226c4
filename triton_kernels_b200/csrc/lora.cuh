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

// Layout of the low-rank rows t: ranks in groups of 16, 32 or 64 (the smallest that holds R, else 64), each group as
// its high parts, then its low parts: a group of 16 is a 64-byte line, of 32 a 128-byte line, of 64 two of them.  TMA
// moves a line of up to 128 bytes per request, and a ring slot costs its warps some 500 cycles whatever it holds, so
// few wide lines are asked for rather than many narrow ones; small ranks do not pay for a full group.
struct LowRank {
  int R, units, group, groups;  // units: sixteens of ranks in use
  explicit LowRank(int64_t rank = 16)
      : R((int)rank), units((int)((rank + 15) / 16)), group(rank <= 16 ? 16 : (rank <= 32 ? 32 : 64)),
        groups((int)((rank + group - 1) / group)) {}
  __host__ __device__ int ld() const { return groups * group * 2; }  // elements per row of t
  __device__ __forceinline__ int column(int rank) const { return rank / group * 2 * group + rank % group; }  // of its high part
  // Shared-memory tiles of one group, 128 rows: one tile of `group` * 4 bytes a row, or two of 128 bytes (high, low).
  __device__ __forceinline__ int tile_bytes() const { return group * 512; }
  __device__ __forceinline__ uint64_t desc(uint32_t saddr) const {
    return group == 16 ? make_smem_desc(saddr, 16, 512, 4) : make_smem_desc(saddr, 16, 1024);
  }
  // Where unit i of a group lies, in 16-byte steps: high parts and low parts
  __device__ __forceinline__ int high(int i) const { return 2 * i; }
  __device__ __forceinline__ int low(int i) const { return 2 * i + (group == 64 ? 1024 : group / 8); }
};

// How a problem of more than eight rows runs: columns per tile of the projection (256 and 192: CTA pairs, 256 rows; less:
// single CTAs, 128 rows), and the blocks among which the low-rank rows of 128 rows of a request split K.
struct LoraPlan {
  int cols, ksplit;
};
LoraPlan plan_lora(int64_t M, int64_t N, int64_t K, const RequestAdapters& req, const LowRank& low);
constexpr int kLoraShort = 8;  // requests of up to so many rows take another kernel for their low-rank rows
int launch_lora_gemm(const LoraPlan& plan, const fluxb_linear_problem& a, int64_t N, int64_t K, int epi, const void* t, const void* lora_b,
                     const LowRank& low, int64_t ldb, const RequestAdapters& req, cudaStream_t st);

}  // namespace fluxb
