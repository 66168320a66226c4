// LayerNorm with a learned scale and offset (or the adaLN modulation's): forward for any row width, and the
// backward pass of both forms with the reductions of the scale's and the offset's gradients.
//
//   forward    h = (x - mean) rstd,  y = h f + o              f = unit + factor (unit: 0 learned scale, 1 adaLN)
//   backward   g = dy f,  dx = rstd (g - mean(g) - h mean(g h)),  df = sum_rows dy h,  do = sum_rows dy
//
// A "group" is the rows that share one factor and offset vector: all rows for a learned scale, the rows of one
// batch item for the modulation.  Statistics, products and sums are fp32 whatever the storage type.  No atomics:
// column sums are partial sums per block, added in a fixed order.
#include "vec.cuh"

namespace fluxb {

template <typename T>
__device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }

// Sum over a block of 256 threads; every thread gets it.  `slot` is 8 floats of shared memory that nothing else uses.
__device__ __forceinline__ float block_sum_256(float v, float* slot) {
  v = warp_sum(v);
  __syncthreads();  // the slots' last readers are through
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += slot[i];
  return s;
}

struct LnArgs {
  const void* x;
  const void* factor;  // nullptr: ones (unit = 0)
  const void* offset;  // nullptr: zeros
  void* y;
  float* mean;  // nullptr: not wanted
  float* rstd;
  int64_t rows, rows_per_group, x_ld, y_ld, vec_stride;
  int cols;
  float unit, eps;
};

struct LnBwdArgs {
  const void* dy;
  const void* x;
  const void* factor;
  const float* mean;
  const float* rstd;
  void* dx;        // nullptr: not wanted
  float* partial;  // [groups][parts][2][cols]
  int64_t rows, rows_per_group, dy_ld, x_ld, dx_ld, vec_stride, groups;
  int cols, parts;
  float unit;
};

// ---- any width, any alignment: one block per row, elements one at a time -----------------------------------
template <typename T>
__global__ void __launch_bounds__(256) ln_fwd_any_kernel(const LnArgs a) {
  __shared__ float slot[8];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  float s = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 256) s += to_f(x[c]);
  const float mean = block_sum_256(s, slot) / a.cols;
  float q = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float d = to_f(x[c]) - mean;
    q = fmaf(d, d, q);
  }
  const float rstd = rsqrtf(block_sum_256(q, slot) / a.cols + a.eps);
  if (a.mean != nullptr && threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  const int64_t vec = row / a.rows_per_group * a.vec_stride;
  const T* f = a.factor != nullptr ? static_cast<const T*>(a.factor) + vec : nullptr;
  const T* o = a.offset != nullptr ? static_cast<const T*>(a.offset) + vec : nullptr;
  T* y = static_cast<T*>(a.y) + row * a.y_ld;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float h = __fmul_rn(to_f(x[c]) - mean, rstd);  // rounded here with and without a factor
    y[c] = static_cast<T>(fmaf(h, f != nullptr ? a.unit + to_f(f[c]) : 1.f, o != nullptr ? to_f(o[c]) : 0.f));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ln_bwd_rows_any_kernel(const LnBwdArgs a) {
  __shared__ float slot[8];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* dy = static_cast<const T*>(a.dy) + row * a.dy_ld;
  const T* f = a.factor != nullptr ? static_cast<const T*>(a.factor) + row / a.rows_per_group * a.vec_stride : nullptr;
  T* dx = static_cast<T*>(a.dx) + row * a.dx_ld;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float g = to_f(dy[c]) * (f != nullptr ? a.unit + to_f(f[c]) : 1.f);
    s1 += g;
    s2 = fmaf(g, (to_f(x[c]) - mean) * rstd, s2);
  }
  s1 = block_sum_256(s1, slot) / a.cols;
  s2 = block_sum_256(s2, slot) / a.cols;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float g = to_f(dy[c]) * (f != nullptr ? a.unit + to_f(f[c]) : 1.f);
    const float h = (to_f(x[c]) - mean) * rstd;
    dx[c] = static_cast<T>(rstd * (g - s1 - h * s2));
  }
}

// Column sums of one part of a group's rows: 32 columns per block, eight rows at a time.
template <typename T>
__global__ void __launch_bounds__(256) ln_bwd_cols_any_kernel(const LnBwdArgs a) {
  __shared__ float acc[2][8][33];
  const int col_blocks = (a.cols + 31) / 32;
  const int64_t part = blockIdx.x / col_blocks;  // group * parts + part
  const int64_t group = part / a.parts;
  const int c = (int)(blockIdx.x % col_blocks) * 32 + (threadIdx.x & 31);
  const int ty = threadIdx.x >> 5;
  float sf = 0.f, so = 0.f;
  if (c < a.cols) {
    const int64_t row0 = group * a.rows_per_group, end = row0 + a.rows_per_group;
    for (int64_t row = row0 + (part % a.parts) * 8 + ty; row < end; row += (int64_t)a.parts * 8) {
      const float d = to_f(static_cast<const T*>(a.dy)[row * a.dy_ld + c]);
      sf = fmaf(d, (to_f(static_cast<const T*>(a.x)[row * a.x_ld + c]) - a.mean[row]) * a.rstd[row], sf);
      so += d;
    }
  }
  acc[0][ty][threadIdx.x & 31] = sf;
  acc[1][ty][threadIdx.x & 31] = so;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5, cc = (int)(blockIdx.x % col_blocks) * 32 + (threadIdx.x & 31);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += acc[which][i][threadIdx.x & 31];
    if (cc < a.cols) a.partial[(part * 2 + which) * a.cols + cc] = s;
  }
}

// df, do [groups, cols] from the partial sums: a block of 32 x 8 threads per (group, which, 32 columns).
template <typename O>
__global__ void __launch_bounds__(256)
ln_bwd_reduce_kernel(const float* __restrict__ partial, O* __restrict__ df, O* __restrict__ dof, int parts, int cols) {
  __shared__ float acc[8][33];
  const int col_blocks = (cols + 31) / 32;
  const int64_t gw = blockIdx.x / col_blocks;  // group * 2 + which
  const int64_t group = gw >> 1;
  const int which = (int)(gw & 1);
  const int c = (int)(blockIdx.x % col_blocks) * 32 + (threadIdx.x & 31);
  const int ty = threadIdx.x >> 5;
  float s = 0.f;
  if (c < cols)
    for (int p = ty; p < parts; p += 8) s += partial[((group * parts + p) * 2 + which) * cols + c];
  acc[ty][threadIdx.x & 31] = s;
  __syncthreads();
  O* out = which == 0 ? df : dof;
  if (ty == 0 && c < cols && out != nullptr) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += acc[i][threadIdx.x & 31];
    out[group * cols + c] = static_cast<O>(t);
  }
}

// Blocks that share the rows of one group in the column sums: enough to fill the machine over all groups, no more
// than there are eights of rows.
static int bwd_parts(int64_t groups, int64_t rows_per_group) {
  const int64_t want = (2 * sm_count() + groups - 1) / groups;
  const int64_t most = (rows_per_group + 7) / 8;
  return (int)(want < 1 ? 1 : (want < most ? want : most));
}

}  // namespace fluxb

using namespace fluxb;

static inline bool elt_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FLUXB_BF16 ? 1u : 3u)) == 0;
}
static inline int ln_status(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return FLUXB_OK;
}
// Sizes that forward and backward share.  Sets *groups.
static int ln_check(const char* what, int64_t rows, int64_t cols, int64_t rows_per_group, int dtype, int64_t* groups) {
  if (dtype != FLUXB_F32 && dtype != FLUXB_BF16) return set_error(FLUXB_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (rows < 0 || cols <= 0 || rows_per_group < 0) return set_error(FLUXB_ERR_BAD_ARG, "%s: bad sizes", what);
  *groups = 0;
  if (rows == 0) return FLUXB_OK;
  if (rows_per_group == 0 || rows % rows_per_group)
    return set_error(FLUXB_ERR_BAD_ARG, "%s: rows must be a multiple of rows_per_group", what);
  if (rows > INT32_MAX || cols > (1 << 20)) return set_error(FLUXB_ERR_UNSUPPORTED, "%s: too many rows or columns", what);
  *groups = rows / rows_per_group;
  return FLUXB_OK;
}

extern "C" int fluxb_layer_norm(const void* x, const void* factor, const void* offset, void* y, float* mean, float* rstd,
                                int64_t rows, int64_t cols, int64_t rows_per_group, int64_t x_ld, int64_t y_ld,
                                int64_t vec_stride, float unit, float eps, int dtype, fluxb_stream_t stream) {
  int64_t groups;
  int rc = ln_check("layer_norm", rows, cols, rows_per_group, dtype, &groups);
  if (rc != FLUXB_OK || rows == 0) return rc;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr))
    return set_error(FLUXB_ERR_BAD_ARG, "layer_norm: null pointer (mean and rstd go together)");
  if (x_ld < 0 || y_ld < cols || vec_stride < 0 || !elt_aligned(x, dtype) || !elt_aligned(y, dtype) ||
      !elt_aligned(factor, dtype) || !elt_aligned(offset, dtype))
    return set_error(FLUXB_ERR_BAD_ARG, "layer_norm: bad strides or misaligned pointers");
  LnArgs a{x, factor, offset, y, mean, rstd, rows, rows_per_group, x_ld, y_ld, vec_stride, (int)cols, unit, eps};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FLUXB_BF16) ln_fwd_any_kernel<__nv_bfloat16><<<(unsigned)rows, 256, 0, st>>>(a);
  else ln_fwd_any_kernel<float><<<(unsigned)rows, 256, 0, st>>>(a);
  return ln_status("layer_norm");
}

extern "C" int64_t fluxb_layer_norm_bwd_scratch(int64_t rows, int64_t cols, int64_t rows_per_group) {
  if (rows <= 0 || cols <= 0 || rows_per_group <= 0) return 0;
  const int64_t groups = rows / rows_per_group;
  return groups * bwd_parts(groups, rows_per_group) * 2 * cols;
}

extern "C" int fluxb_layer_norm_bwd(const void* dy, const void* x, const void* factor, const float* mean, const float* rstd,
                                    void* dx, void* dfactor, void* doffset, float* scratch, int64_t rows, int64_t cols,
                                    int64_t rows_per_group, int64_t dy_ld, int64_t x_ld, int64_t dx_ld, int64_t vec_stride,
                                    float unit, int grads_f32, int dtype, fluxb_stream_t stream) {
  int64_t groups;
  int rc = ln_check("layer_norm_bwd", rows, cols, rows_per_group, dtype, &groups);
  if (rc != FLUXB_OK || rows == 0) return rc;
  const bool sums = dfactor != nullptr || doffset != nullptr;
  if (!dy || !x || !mean || !rstd || (sums && !scratch)) return set_error(FLUXB_ERR_BAD_ARG, "layer_norm_bwd: null pointer");
  if (dy_ld < 0 || x_ld < 0 || (dx != nullptr && dx_ld < cols) || vec_stride < 0 || !elt_aligned(dy, dtype) ||
      !elt_aligned(x, dtype) || !elt_aligned(factor, dtype) || !elt_aligned(dx, dtype))
    return set_error(FLUXB_ERR_BAD_ARG, "layer_norm_bwd: bad strides or misaligned pointers");
  LnBwdArgs a{dy, x, factor, mean, rstd, dx, scratch, rows, rows_per_group, dy_ld, x_ld, dx_ld, vec_stride, groups,
              (int)cols, bwd_parts(groups, rows_per_group), unit};
  const int64_t col_blocks = (cols + 31) / 32;
  if (groups * a.parts * col_blocks > INT32_MAX || groups * 2 * col_blocks > INT32_MAX)
    return set_error(FLUXB_ERR_UNSUPPORTED, "layer_norm_bwd: too many groups");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == FLUXB_BF16;
  if (dx != nullptr) {
    if (bf) ln_bwd_rows_any_kernel<__nv_bfloat16><<<(unsigned)rows, 256, 0, st>>>(a);
    else ln_bwd_rows_any_kernel<float><<<(unsigned)rows, 256, 0, st>>>(a);
  }
  if (sums) {
    const unsigned grid = (unsigned)(groups * a.parts * col_blocks), rgrid = (unsigned)(groups * 2 * col_blocks);
    if (bf) ln_bwd_cols_any_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
    else ln_bwd_cols_any_kernel<float><<<grid, 256, 0, st>>>(a);
    if (bf && !grads_f32)
      ln_bwd_reduce_kernel<__nv_bfloat16><<<rgrid, 256, 0, st>>>(scratch, static_cast<__nv_bfloat16*>(dfactor),
                                                                static_cast<__nv_bfloat16*>(doffset), a.parts, (int)cols);
    else
      ln_bwd_reduce_kernel<float><<<rgrid, 256, 0, st>>>(scratch, static_cast<float*>(dfactor), static_cast<float*>(doffset),
                                                        a.parts, (int)cols);
  }
  return ln_status("layer_norm_bwd");
}
