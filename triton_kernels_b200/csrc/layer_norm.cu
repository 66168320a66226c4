// LayerNorm with a learned scale and offset (or the adaLN modulation's): forward for any row width, and the
// backward pass of both forms with the reductions of the scale's and the offset's gradients.
//
//   forward    h = (x - mean) rstd,  y = h f + o              f = unit + factor (unit: 0 learned scale, 1 adaLN)
//   backward   g = dy f,  dx = rstd (g - mean(g) - h mean(g h)),  df = sum_rows dy h,  do = sum_rows dy
//
// A "group" is the rows that share one factor and offset vector: all rows for a learned scale, the rows of one
// batch item for the modulation.  Statistics, products and sums are fp32 whatever the storage type.  No atomics:
// column sums are partial sums per block, added in a fixed order.
#include "norm.cuh"
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
  int wpr, teams, slots;  // aligned rows: warps per row, rows at a time per block, rows on their way per team
  DeviceStatus* status;
};
constexpr int kMaxTeamSlots = 64;


// ---- any width, any alignment: one block per row, elements one at a time (more than 8192 columns, or 12288 aligned)
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

// ---- any alignment, up to 8192 columns: one block per row, kE elements per thread in registers, 512 apart (so a warp's
// loads are neighbours whatever the row starts at) -------------------------------------------------------------
constexpr int kWide = 512;  // threads

template <typename T, int kE>
__global__ void __launch_bounds__(kWide) ln_fwd_elements_kernel(const LnArgs a) {
  __shared__ float slot[2][16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  float v[kE];
#pragma unroll
  for (int i = 0; i < kE; ++i) v[i] = tid + i * kWide < a.cols ? to_f(x[tid + i * kWide]) : 0.f;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kE; ++i) s += v[i];
  s = warp_sum(s);
  if (lane == 0) slot[0][warp] = s;
  __syncthreads();
  float mean = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) mean += slot[0][w];
  mean /= a.cols;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const float d = tid + i * kWide < a.cols ? v[i] - mean : 0.f;
    q = fmaf(d, d, q);
  }
  q = warp_sum(q);
  if (lane == 0) slot[1][warp] = q;
  __syncthreads();
  q = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) q += slot[1][w];
  const float rstd = rsqrtf(q / a.cols + a.eps);
  if (a.mean != nullptr && tid == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  const int64_t vec = row / a.rows_per_group * a.vec_stride;
  const T* f = a.factor != nullptr ? static_cast<const T*>(a.factor) + vec : nullptr;
  const T* o = a.offset != nullptr ? static_cast<const T*>(a.offset) + vec : nullptr;
  T* y = static_cast<T*>(a.y) + row * a.y_ld;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int c = tid + i * kWide;
    if (c < a.cols) {
      const float h = __fmul_rn(v[i] - mean, rstd);
      y[c] = static_cast<T>(fmaf(h, f != nullptr ? a.unit + to_f(f[c]) : 1.f, o != nullptr ? to_f(o[c]) : 0.f));
    }
  }
}

// Up to 1024 columns: a warp per row, kE elements per lane.
template <typename T, int kE>
__global__ void __launch_bounds__(256) ln_fwd_narrow_kernel(const LnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  float v[kE], s = 0.f, q = 0.f;
#pragma unroll
  for (int i = 0; i < kE; ++i) v[i] = lane + i * 32 < a.cols ? to_f(x[lane + i * 32]) : 0.f;
#pragma unroll
  for (int i = 0; i < kE; ++i) s += v[i];
  const float mean = warp_sum(s) / a.cols;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const float d = lane + i * 32 < a.cols ? v[i] - mean : 0.f;
    q = fmaf(d, d, q);
  }
  const float rstd = rsqrtf(warp_sum(q) / a.cols + a.eps);
  if (a.mean != nullptr && lane == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  const int64_t vec = row / a.rows_per_group * a.vec_stride;
  const T* f = a.factor != nullptr ? static_cast<const T*>(a.factor) + vec : nullptr;
  const T* o = a.offset != nullptr ? static_cast<const T*>(a.offset) + vec : nullptr;
  T* y = static_cast<T*>(a.y) + row * a.y_ld;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int c = lane + i * 32;
    if (c < a.cols) {
      const float h = __fmul_rn(v[i] - mean, rstd);
      y[c] = static_cast<T>(fmaf(h, f != nullptr ? a.unit + to_f(f[c]) : 1.f, o != nullptr ? to_f(o[c]) : 0.f));
    }
  }
}

// One pass over x and dy: the block walks rows of its part of a group, with the next row's elements on their way.
template <typename T, int kE>
__global__ void __launch_bounds__(kWide, 1) ln_bwd_elements_kernel(const LnBwdArgs a) {
  __shared__ float2 red[2][16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t group = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int64_t base = group * a.rows_per_group;
  const T* f = a.factor != nullptr ? static_cast<const T*>(a.factor) + group * a.vec_stride : nullptr;
  float factor[kE], df[kE], dof[kE];
  T xn[kE], dn[kE];
  float mean_n = 0.f, rstd_n = 0.f;
  auto ask = [&](int64_t r) {
    if (r >= a.rows_per_group) return;
    const T* x = static_cast<const T*>(a.x) + (base + r) * a.x_ld + tid;
    const T* dy = static_cast<const T*>(a.dy) + (base + r) * a.dy_ld + tid;
    mean_n = __ldg(a.mean + base + r);
    rstd_n = __ldg(a.rstd + base + r);
#pragma unroll
    for (int i = 0; i < kE; ++i)
      if (tid + i * kWide < a.cols) {
        xn[i] = x[i * kWide];
        dn[i] = dy[i * kWide];
      }
  };
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    factor[i] = f == nullptr ? 1.f : (tid + i * kWide < a.cols ? a.unit + to_f(f[tid + i * kWide]) : 0.f);
    df[i] = dof[i] = 0.f;
    xn[i] = dn[i] = static_cast<T>(0.f);
  }
  ask(part);
  const float inv_cols = 1.f / a.cols;
  int buf = 0;
  for (int64_t r = part; r < a.rows_per_group; r += a.parts) {
    const float mean = mean_n, rstd = rstd_n;
    float g[kE], h[kE], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const bool in = tid + i * kWide < a.cols;
      const float d = in ? to_f(dn[i]) : 0.f;
      h[i] = in ? (to_f(xn[i]) - mean) * rstd : 0.f;
      g[i] = d * factor[i];
      s1 += g[i];
      s2 = fmaf(g[i], h[i], s2);
      df[i] = fmaf(d, h[i], df[i]);
      dof[i] += d;
    }
    ask(r + a.parts);
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (lane == 0) red[buf][warp] = make_float2(s1, s2);
    __syncthreads();  // (the other buffer's readers are through before anyone writes it again)
    s1 = s2 = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      s1 += red[buf][w].x;
      s2 += red[buf][w].y;
    }
    buf ^= 1;
    if (a.dx != nullptr) {
      const float k1 = -s1 * inv_cols * rstd, k2 = -s2 * inv_cols * rstd;
      T* dx = static_cast<T*>(a.dx) + (base + r) * a.dx_ld + tid;
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (tid + i * kWide < a.cols) dx[i * kWide] = static_cast<T>(fmaf(h[i], k2, fmaf(g[i], rstd, k1)));
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < kE; ++i)
    if (tid + i * kWide < a.cols) {
      out[tid + i * kWide] = df[i];
      out[a.cols + tid + i * kWide] = dof[i];
    }
}

// ---- aligned rows ------------------------------------------------------------------------------------------
// Few rows: one block per row, the row in registers (kV 16-byte pieces per thread), so that a launch is one round of
// loads and two block sums.  Bound by latency: one row of 3072 bf16 takes 2.2 us of kernel time, against 5.0 with the
// element-wise kernel above and its three passes.  (With several rows per SM the kernel that stages rows through shared
// memory takes over: it keeps more bytes in flight.)
template <typename T, int kV>
__global__ void __launch_bounds__(256) ln_fwd_block_kernel(const LnArgs a) {
  constexpr int VN = Vec<T>::N;
  __shared__ float slot[8];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const int64_t vec = row / a.rows_per_group * a.vec_stride;
  const T* fp = static_cast<const T*>(a.factor) + vec;
  const T* op = static_cast<const T*>(a.offset) + vec;
  uint4 raw[kV], fr[kV], orw[kV];
  pdl_wait();  // (the block may have started while the kernel in front was ending)
  pdl_release();
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int c = (i * 256 + threadIdx.x) * VN;
    if (c < a.cols) {
      raw[i] = ld_u4(x + c);
      fr[i] = ld_u4(fp + c);
      orw[i] = ld_u4(op + c);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    if ((i * 256 + (int)threadIdx.x) * VN < a.cols) {
      Vec<T> t;
      t.unpack(raw[i]);
#pragma unroll
      for (int j = 0; j < VN; ++j) s += t.v[j];
    }
  }
  const float mean = block_sum_256(s, slot) / a.cols;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    if ((i * 256 + (int)threadIdx.x) * VN < a.cols) {
      Vec<T> t;
      t.unpack(raw[i]);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const float d = t.v[j] - mean;
        q = fmaf(d, d, q);
      }
    }
  }
  const float rstd = rsqrtf(block_sum_256(q, slot) / a.cols + a.eps);
  if (a.mean != nullptr && threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  T* y = static_cast<T*>(a.y) + row * a.y_ld;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int c = (i * 256 + threadIdx.x) * VN;
    if (c < a.cols) {
      Vec<T> t, f, o;
      t.unpack(raw[i]);
      f.unpack(fr[i]);
      o.unpack(orw[i]);
#pragma unroll
      for (int j = 0; j < VN; ++j) t.v[j] = fmaf(__fmul_rn(t.v[j] - mean, rstd), a.unit + f.v[j], o.v[j]);
      t.store(y + c);
    }
  }
}

// Sixteen bytes as pairs of fp32: the backward kernels work on pairs (one instruction for two columns), because with
// one column at a time they were bound by the instructions that they issued (28 per element), not by memory.
template <typename T>
struct Pairs {
  static constexpr int N = 8 / sizeof(T);
  float2 v[N];
  __device__ __forceinline__ void unpack(const uint4& t) {
    if constexpr (sizeof(T) == 2) {
      v[0] = make_float2(bf16_lo(t.x), bf16_hi(t.x)); v[1] = make_float2(bf16_lo(t.y), bf16_hi(t.y));
      v[2] = make_float2(bf16_lo(t.z), bf16_hi(t.z)); v[3] = make_float2(bf16_lo(t.w), bf16_hi(t.w));
    } else {
      v[0] = make_float2(__uint_as_float(t.x), __uint_as_float(t.y));
      v[1] = make_float2(__uint_as_float(t.z), __uint_as_float(t.w));
    }
  }
  __device__ __forceinline__ uint4 pack() const {
    if constexpr (sizeof(T) == 2)
      return make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y), pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
    else
      return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The widened factor in shared memory: the first four columns of every 16-byte piece, then (bf16) the other four, so
// that neighbouring lanes read neighbouring float4s (in column order they would meet in the same banks).
template <typename T>
__device__ __forceinline__ void fill_factor(float* factor, const T* f, float unit, int cols) {
  constexpr int VN = Vec<T>::N;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const int piece = c / VN, j = c % VN;
    factor[(j / 4 * (cols / VN) + piece) * 4 + j % 4] = f != nullptr ? unit + to_f(f[c]) : 1.f;
  }
}

// What a row's piece adds: h and g for dx, the two sums of the row, the column sums.
template <typename T>
__device__ __forceinline__ void bwd_piece(const uint4& xr, const uint4& dr, const float4* factor, int piece, int pieces,
                                          float2 neg_mean, float2 rstd, Pairs<T>& g, Pairs<T>& h, float2& s1, float2& s2,
                                          Pairs<T>& df, Pairs<T>& dof) {
  Pairs<T> x, d;
  x.unpack(xr);
  d.unpack(dr);
#pragma unroll
  for (int q = 0; q < Pairs<T>::N / 2; ++q) {
    const float4 f = factor[q * pieces + piece];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * q + e;
      h.v[i] = __fmul2_rn(__fadd2_rn(x.v[i], neg_mean), rstd);
      g.v[i] = __fmul2_rn(d.v[i], e == 0 ? make_float2(f.x, f.y) : make_float2(f.z, f.w));
      s1 = __fadd2_rn(s1, g.v[i]);
      s2 = __ffma2_rn(g.v[i], h.v[i], s2);
      df.v[i] = __ffma2_rn(d.v[i], h.v[i], df.v[i]);
      dof.v[i] = __fadd2_rn(dof.v[i], d.v[i]);
    }
  }
}
// rstd (g - mean(g) - h mean(g h)) with k1 = -rstd mean(g), k2 = -rstd mean(g h)
template <typename T>
__device__ __forceinline__ uint4 bwd_dx(const Pairs<T>& g, const Pairs<T>& h, float2 rstd, float2 k1, float2 k2) {
  Pairs<T> o;
#pragma unroll
  for (int i = 0; i < Pairs<T>::N; ++i) o.v[i] = __ffma2_rn(h.v[i], k2, __ffma2_rn(g.v[i], rstd, k1));
  return o.pack();
}
// Two sums over a warp at once: lanes 0-15 get the first one's total, lanes 16-31 the second one's.
__device__ __forceinline__ float warp_sum_two(float2 s1, float2 s2, int lane) {
  const float a = s1.x + s1.y, b = s2.x + s2.y;
  const bool upper = (lane & 16) != 0;
  float keep = upper ? b : a;
  keep += __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, o);
  return keep;
}

// Backward, one pass over x and dy: a team of `wpr` warps walks whole rows and keeps the column sums of its columns in
// registers (kV 16-byte pieces per thread), so a row is read once and everything that it gives - dx, its share of df and
// do - leaves from there.  The rows come through a ring in shared memory by bulk copies, one x row and one dy row a
// slot: a row in flight costs no registers, and the ring holds about 150 KB per SM.  Two sums per row (g and g h) meet
// in the team: shuffles, then one named barrier, whose other side also frees the row's slot for the next copy.  The
// factor is kept widened in shared memory.  At the end the block's teams add up their column sums in a fixed order and
// the block writes one partial row; ln_bwd_reduce_kernel adds those.
// 3072 columns bf16: 2 x 4096 rows 34 us (151 MB read and written, 4.4 TB/s, part of it start and end of the blocks),
// 4 x 16896 rows 220 us (5.7 TB/s).
// kFull: the row is exactly kV pieces per thread.
template <typename T, int kV, bool kFull>
__global__ void __launch_bounds__(512, 1) ln_bwd_team_kernel(const LnBwdArgs a) {
  constexpr int VN = Vec<T>::N;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ uint64_t bars[kMaxTeamSlots];
  __shared__ float red[2][16][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = warp / a.wpr, team_threads = a.wpr * 32, tid = threadIdx.x - team * team_threads;
  const int group = blockIdx.x / a.parts, part = blockIdx.x - group * a.parts;
  const int pieces = a.cols / VN, rows = (int)a.rows_per_group;
  const uint32_t row_bytes = (uint32_t)a.cols * sizeof(T);
  const float4* factor = reinterpret_cast<const float4*>(dyn);  // [cols] floats, then the teams' rings
  uint8_t* ring = dyn + (a.cols * 4 + 127) / 128 * 128 + team * a.slots * 2 * row_bytes;
  uint64_t* full = bars + team * a.slots;
  if (tid == 0) {
    for (int i = 0; i < a.slots; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  const int64_t base = (int64_t)group * rows;
  const T* x = static_cast<const T*>(a.x) + base * a.x_ld;
  const T* dy = static_cast<const T*>(a.dy) + base * a.dy_ld;
  const int step = a.parts * a.teams, first = part * a.teams + team;
  auto ask = [&](int row, int slot) {
    uint8_t* dst = ring + slot * 2 * row_bytes;
    mbar_expect_tx(&full[slot], 2 * row_bytes);
    bulk_load_row(dst, x + row * a.x_ld, row_bytes, &full[slot]);
    bulk_load_row(dst + row_bytes, dy + row * a.dy_ld, row_bytes, &full[slot]);
  };
  if (tid == 0) {
    for (int i = 0; i < a.slots; ++i)
      if (first + i * step < rows) ask(first + i * step, i);
  }
  fill_factor<T>(reinterpret_cast<float*>(dyn),
                 a.factor != nullptr ? static_cast<const T*>(a.factor) + group * a.vec_stride : nullptr, a.unit, a.cols);
  __syncthreads();

  Pairs<T> df[kV], dof[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i)
#pragma unroll
    for (int j = 0; j < Pairs<T>::N; ++j) df[i].v[j] = dof[i].v[j] = both(0.f);
  const float inv_cols = 1.f / a.cols;
  int slot = 0, buf = 0;
  uint32_t phase = 0;
  const float *mean_p = a.mean + base + first, *rstd_p = a.rstd + base + first;
  float next_mean = 0.f, next_rstd = 0.f;
  if (first < rows) { next_mean = __ldg(mean_p); next_rstd = __ldg(rstd_p); }
  T* dx = static_cast<T*>(a.dx) + (base + first) * a.dx_ld + tid * VN;
  for (int r = first; r < rows; r += step) {
    const float rstd = next_rstd;
    const float2 neg_mean = both(-next_mean), rstd2 = both(rstd);
    mean_p += step;
    rstd_p += step;
    if (r + step < rows) { next_mean = __ldg(mean_p); next_rstd = __ldg(rstd_p); }
    bool ok = mbar_try_wait(&full[slot], phase);
    for (uint32_t spin = 0; spin < (1u << 24) && !ok; ++spin) ok = mbar_try_wait(&full[slot], phase);
    if (!ok) report_error(a.status, FLUXB_ERR_TIMEOUT, 72);  // carries on: the row's numbers are lost, nobody hangs
    const uint4* xs = reinterpret_cast<const uint4*>(ring + slot * 2 * row_bytes) + tid;
    const uint4* ds = xs + pieces;
    Pairs<T> g[kV], h[kV];
    float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int piece = i * team_threads + tid;
      if (kFull || piece < pieces)
        bwd_piece<T>(xs[i * team_threads], ds[i * team_threads], factor, piece, pieces, neg_mean, rstd2, g[i], h[i], s1, s2,
                     df[i], dof[i]);
    }
    const float sum = warp_sum_two(s1, s2, lane);
    if ((lane & 15) == 0) red[buf][warp][lane >> 4] = sum;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(team_threads) : "memory");
    if (tid == 0 && r + a.slots * step < rows) ask(r + a.slots * step, slot);
    float2 t = both(0.f);
    for (int w = 0; w < a.wpr; ++w) t = __fadd2_rn(t, *reinterpret_cast<const float2*>(red[buf][team * a.wpr + w]));
    if (a.dx != nullptr) {
      const float2 k1 = both(-t.x * inv_cols * rstd), k2 = both(-t.y * inv_cols * rstd);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        if (kFull || i * team_threads + tid < pieces)
          *reinterpret_cast<uint4*>(dx + i * team_threads * VN) = bwd_dx<T>(g[i], h[i], rstd2, k1, k2);
      }
      dx += step * a.dx_ld;
    }
    buf ^= 1;
    if (++slot == a.slots) { slot = 0; phase ^= 1; }
  }
  // the teams' column sums, added up by the first one; all copies have landed, the rings are free
  float2* other = reinterpret_cast<float2*>(dyn + (a.cols * 4 + 127) / 128 * 128);  // [2][cols / 2]
  for (int t = 1; t < a.teams; ++t) {
    __syncthreads();
    if (team == t) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int piece = i * team_threads + tid;
        if (kFull || piece < pieces) {
#pragma unroll
          for (int j = 0; j < Pairs<T>::N; ++j) {
            other[j * pieces + piece] = df[i].v[j];
            other[a.cols / 2 + j * pieces + piece] = dof[i].v[j];
          }
        }
      }
    }
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int piece = i * team_threads + tid;
        if (kFull || piece < pieces) {
#pragma unroll
          for (int j = 0; j < Pairs<T>::N; ++j) {
            df[i].v[j] = __fadd2_rn(df[i].v[j], other[j * pieces + piece]);
            dof[i].v[j] = __fadd2_rn(dof[i].v[j], other[a.cols / 2 + j * pieces + piece]);
          }
        }
      }
    }
  }
  if (team == 0 && a.partial != nullptr) {
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int piece = i * team_threads + tid;
      if (kFull || piece < pieces) {
#pragma unroll
        for (int j = 0; j < Pairs<T>::N; j += 2) {
          float* at = out + piece * VN + 2 * j;
          *reinterpret_cast<float4*>(at) = make_float4(df[i].v[j].x, df[i].v[j].y, df[i].v[j + 1].x, df[i].v[j + 1].y);
          *reinterpret_cast<float4*>(at + a.cols) = make_float4(dof[i].v[j].x, dof[i].v[j].y, dof[i].v[j + 1].x, dof[i].v[j + 1].y);
        }
      }
    }
  }
}

// Narrow rows: a warp per row, kV pieces per lane, the next rows (four, two or one) in registers on their way while the
// current ones are worked on.
template <typename T, int kV>
__global__ void __launch_bounds__(384, 1) ln_bwd_warp_kernel(const LnBwdArgs a) {
  constexpr int VN = Vec<T>::N;
  constexpr int kRows = kV == 1 ? 4 : (kV == 2 ? 2 : 1);
  constexpr int kWarps = 12;
  extern __shared__ __align__(128) uint8_t dyn[];
  const float4* factor = reinterpret_cast<const float4*>(dyn);                       // [cols] floats
  float2* sums = reinterpret_cast<float2*>(dyn + (size_t)(a.cols + 31) / 32 * 128);  // [kWarps][2][cols / 2]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = blockIdx.x / a.parts, part = blockIdx.x - group * a.parts;
  const int pieces = a.cols / VN, rows = (int)a.rows_per_group;
  const int64_t base = (int64_t)group * rows;
  const T* x = static_cast<const T*>(a.x) + base * a.x_ld + lane * VN;
  const T* dy = static_cast<const T*>(a.dy) + base * a.dy_ld + lane * VN;
  const int step = a.parts * kWarps * kRows;
  uint4 xn[kRows][kV], dn[kRows][kV];
  float mn[kRows], rn[kRows];
  auto ask = [&](int r0) {
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int r = r0 + q;
      if (r < rows) {
        mn[q] = __ldg(a.mean + base + r);
        rn[q] = __ldg(a.rstd + base + r);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          if (i * 32 + lane < pieces) {
            xn[q][i] = ld_nc_u4(x + r * a.x_ld + i * 32 * VN);
            dn[q][i] = ld_nc_u4(dy + r * a.dy_ld + i * 32 * VN);
          }
        }
      }
    }
  };
  int r0 = (part * kWarps + warp) * kRows;
  ask(r0);
  fill_factor<T>(reinterpret_cast<float*>(dyn),
                 a.factor != nullptr ? static_cast<const T*>(a.factor) + group * a.vec_stride : nullptr, a.unit, a.cols);
  __syncthreads();
  Pairs<T> df[kV], dof[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i)
#pragma unroll
    for (int j = 0; j < Pairs<T>::N; ++j) df[i].v[j] = dof[i].v[j] = both(0.f);
  const float inv_cols = 1.f / a.cols;
  for (; r0 < rows; r0 += step) {
    uint4 xc[kRows][kV], dc[kRows][kV];
    float mc[kRows], rc[kRows];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      mc[q] = mn[q];
      rc[q] = rn[q];
#pragma unroll
      for (int i = 0; i < kV; ++i) { xc[q][i] = xn[q][i]; dc[q][i] = dn[q][i]; }
    }
    ask(r0 + step);
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      if (r0 + q >= rows) break;
      Pairs<T> g[kV], h[kV];
      float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (i * 32 + lane < pieces)
          bwd_piece<T>(xc[q][i], dc[q][i], factor, i * 32 + lane, pieces, both(-mc[q]), both(rc[q]), g[i], h[i], s1, s2, df[i],
                       dof[i]);
      const float keep = warp_sum_two(s1, s2, lane);
      const float over = __shfl_xor_sync(0xffffffffu, keep, 16);
      if (a.dx != nullptr) {
        const float k = -inv_cols * rc[q];
        const float2 k1 = both(k * ((lane & 16) ? over : keep)), k2 = both(k * ((lane & 16) ? keep : over));
        T* dx = static_cast<T*>(a.dx) + (base + r0 + q) * a.dx_ld + lane * VN;
#pragma unroll
        for (int i = 0; i < kV; ++i)
          if (i * 32 + lane < pieces)
            *reinterpret_cast<uint4*>(dx + i * 32 * VN) = bwd_dx<T>(g[i], h[i], both(rc[q]), k1, k2);
      }
    }
  }
  if (a.partial == nullptr) return;
  float2* mine = sums + (size_t)warp * a.cols;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int piece = i * 32 + lane;
    if (piece < pieces) {
#pragma unroll
      for (int j = 0; j < Pairs<T>::N; ++j) {
        mine[piece * (VN / 2) + j] = df[i].v[j];
        mine[a.cols / 2 + piece * (VN / 2) + j] = dof[i].v[j];
      }
    }
  }
  __syncthreads();
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
  const float* all = reinterpret_cast<const float*>(sums);
  for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += all[(size_t)w * 2 * a.cols + c];
    out[c] = s;
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

// How the backward pass runs: which kernel, and how many blocks share the rows of one group (one partial row each).
struct BwdPlan {
  enum Kind { kAny, kElements, kWarp, kTeam } kind;
  int vecs;  // 16-byte pieces per thread
  int wpr, teams, slots, parts;
  size_t smem;
};
static BwdPlan bwd_plan(int64_t groups, int64_t rows_per_group, int64_t cols, int dtype, bool aligned) {
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const int64_t v = cols / vn;
  BwdPlan p{BwdPlan::kAny, 0, 0, 0, 0, 1, 0};
  int64_t blocks = 2 * sm_count(), rows_at_once = 8;  // kAny
  if (aligned && cols % vn == 0) {
    if (v <= 96) {
      p.kind = BwdPlan::kWarp;
      p.vecs = (int)((v + 31) / 32);
      blocks = sm_count();
      rows_at_once = 12;
      p.smem = ((size_t)(cols + 31) / 32 * 32 + 24 * (size_t)cols) * 4;
    } else {
      // pieces per thread: the most that registers hold (two of bf16, four of fp32; three of bf16 spill 64 to 100
      // bytes a thread and are left to rows of more than 8192), unless fewer leave fewer lanes without a column
      int64_t best = -1;
      for (int k = vn == 8 ? (v > 1024 ? 3 : 2) : 4; k >= 1; --k) {
        const int64_t w = (v + 32 * k - 1) / (32 * k);
        if (w < 2 || w > 16) continue;  // (named barriers and slots are counted for eight teams)
        const int64_t idle = (w * 32 * k - v) * 64 / v;  // in 64ths of a row
        if (best < 0 || idle < best) {
          best = idle;
          p.kind = BwdPlan::kTeam;
          p.vecs = k;
          p.wpr = (int)w;
        }
      }
      if (p.kind == BwdPlan::kTeam) {
        p.teams = 16 / p.wpr;
        const int64_t slot = 2 * cols * (vn == 8 ? 2 : 4);
        int64_t s = (152 * 1024) / (slot * p.teams);
        if (s < 3) s = 3;
        if (s > 8) s = 8;
        p.slots = (int)s;
        p.smem = (size_t)(cols * 4 + 127) / 128 * 128 + (size_t)(p.teams * s * slot);
        const size_t fold = (size_t)(cols * 4 + 127) / 128 * 128 + (size_t)cols * 8;
        if (p.teams > 1 && p.smem < fold) p.smem = fold;
        blocks = sm_count();
        rows_at_once = p.teams;
        if (p.smem > 224 * 1024) p.kind = BwdPlan::kAny;
      }
    }
  }
  if (p.kind == BwdPlan::kAny) {
    blocks = 2 * sm_count();
    rows_at_once = 8;
    if (cols <= 16 * kWide) {
      p.kind = BwdPlan::kElements;
      blocks = (cols <= 4 * kWide ? 2 : 1) * sm_count();
      rows_at_once = 1;
    }
  }
  const int64_t want = blocks / groups, most = (rows_per_group + rows_at_once - 1) / rows_at_once;
  p.parts = (int)(want < 1 ? 1 : (want < most ? want : most));
  return p;
}

}  // namespace fluxb

using namespace fluxb;

static inline bool elt_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FLUXB_BF16 ? 1u : 3u)) == 0;
}
static inline bool all16(const void* a, const void* b, const void* c, const void* d) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
           reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
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
  // row numbers and their next steps stay in 32 bits
  if (rows > (1 << 30) || cols > (1 << 20)) return set_error(FLUXB_ERR_UNSUPPORTED, "%s: too many rows or columns", what);
  *groups = rows / rows_per_group;
  return FLUXB_OK;
}

template <typename T>
static void launch_any(const LnArgs& a, cudaStream_t st) {
  const int e = (a.cols + kWide - 1) / kWide;
  const unsigned rows = (unsigned)a.rows, eights = (rows + 7) / 8;
  if (a.cols <= 128) ln_fwd_narrow_kernel<T, 4><<<eights, 256, 0, st>>>(a);
  else if (a.cols <= 512) ln_fwd_narrow_kernel<T, 16><<<eights, 256, 0, st>>>(a);
  else if (a.cols <= 1024) ln_fwd_narrow_kernel<T, 32><<<eights, 256, 0, st>>>(a);
  else if (e <= 4) ln_fwd_elements_kernel<T, 4><<<rows, kWide, 0, st>>>(a);
  else if (e <= 8) ln_fwd_elements_kernel<T, 8><<<rows, kWide, 0, st>>>(a);
  else if (e <= 16) ln_fwd_elements_kernel<T, 16><<<rows, kWide, 0, st>>>(a);
  else ln_fwd_any_kernel<T><<<rows, 256, 0, st>>>(a);
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
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const bool whole = factor != nullptr && offset != nullptr && cols % vn == 0 && x_ld % vn == 0 && y_ld % vn == 0 &&
                     vec_stride % vn == 0 && all16(x, y, factor, offset);
  if (whole && rows <= 2 * sm_count() && cols <= 1024 * vn) {
    const int v = (int)((cols / vn + 255) / 256);
#define FLUXB_LN_BLOCK(T)                                                                        \
  do {                                                                                           \
    if (v == 1) launch_after(ln_fwd_block_kernel<T, 1>, (unsigned)rows, 256, 0, st, a);          \
    else if (v == 2) launch_after(ln_fwd_block_kernel<T, 2>, (unsigned)rows, 256, 0, st, a);     \
    else launch_after(ln_fwd_block_kernel<T, 4>, (unsigned)rows, 256, 0, st, a);                 \
  } while (0)
    if (dtype == FLUXB_BF16) FLUXB_LN_BLOCK(__nv_bfloat16);
    else FLUXB_LN_BLOCK(float);
#undef FLUXB_LN_BLOCK
    return ln_status("layer_norm");
  }
  if (whole && unit == 0.f && groups == 1) {
    rc = launch_layer_norm_affine(x, factor, offset, y, mean, rstd, rows, cols, x_ld, y_ld, eps, dtype, st);
    return rc != FLUXB_OK ? rc : ln_status("layer_norm");
  }
  if (dtype == FLUXB_BF16) launch_any<__nv_bfloat16>(a, st);
  else launch_any<float>(a, st);
  return ln_status("layer_norm");
}

extern "C" int64_t fluxb_layer_norm_bwd_scratch(int64_t rows, int64_t cols, int64_t rows_per_group) {
  if (rows <= 0 || cols <= 0 || rows_per_group <= 0) return 0;
  // the most that any of the kernels asks for: two blocks per SM over all groups
  const int64_t groups = rows / rows_per_group, want = 2 * sm_count() / (groups > 0 ? groups : 1);
  const int64_t parts = want < 1 ? 1 : (want < rows_per_group ? want : rows_per_group);
  return groups * parts * 2 * cols;
}

template <typename T, bool kFull>
static auto team_kernel(int vecs) -> void (*)(LnBwdArgs) {
  if (vecs == 1) return ln_bwd_team_kernel<T, 1, kFull>;
  if (vecs == 2) return ln_bwd_team_kernel<T, 2, kFull>;
  if (vecs == 3) return ln_bwd_team_kernel<T, 3, kFull>;
  return ln_bwd_team_kernel<T, sizeof(T) == 2 ? 3 : 4, kFull>;  // (four of bf16 are never planned)
}

template <typename T>
static int launch_bwd(const LnBwdArgs& a, const BwdPlan& p, bool sums, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.groups * a.parts);
  if (p.kind == BwdPlan::kAny) {
    if (a.dx != nullptr) ln_bwd_rows_any_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a);
    if (sums) ln_bwd_cols_any_kernel<T><<<grid * (unsigned)((a.cols + 31) / 32), 256, 0, st>>>(a);
    return FLUXB_OK;
  }
  if (p.kind == BwdPlan::kElements) {
    const int e = (a.cols + kWide - 1) / kWide;
    auto kern = e <= 1   ? ln_bwd_elements_kernel<T, 1>
                : e <= 2 ? ln_bwd_elements_kernel<T, 2>
                : e <= 4 ? ln_bwd_elements_kernel<T, 4>
                : e <= 8 ? ln_bwd_elements_kernel<T, 8>
                         : ln_bwd_elements_kernel<T, 16>;
    kern<<<grid, kWide, 0, st>>>(a);
    return FLUXB_OK;
  }
  void (*kern)(LnBwdArgs) = nullptr;
  if (p.kind == BwdPlan::kWarp)
    kern = p.vecs == 1 ? ln_bwd_warp_kernel<T, 1> : (p.vecs == 2 ? ln_bwd_warp_kernel<T, 2> : ln_bwd_warp_kernel<T, 3>);
  else
    kern = a.cols * (int)sizeof(T) == p.vecs * p.wpr * 512 ? team_kernel<T, true>(p.vecs) : team_kernel<T, false>(p.vecs);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem);
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "layer_norm_bwd: cannot set shared memory size: %s", cudaGetErrorString(e));
  kern<<<grid, p.kind == BwdPlan::kWarp ? 384 : p.teams * p.wpr * 32, p.smem, st>>>(a);
  return FLUXB_OK;
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
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const bool whole = cols % vn == 0 && x_ld % vn == 0 && dy_ld % vn == 0 && (dx == nullptr || dx_ld % vn == 0) &&
                     all16(x, dy, dx, scratch);
  const BwdPlan p = bwd_plan(groups, rows_per_group, cols, dtype, whole);
  LnBwdArgs a{dy, x, factor, mean, rstd, dx, sums ? scratch : nullptr, rows, rows_per_group, dy_ld, x_ld, dx_ld, vec_stride,
              groups, (int)cols, p.parts, unit, p.wpr, p.teams, p.slots, device_status_ptr()};
  const int64_t col_blocks = (cols + 31) / 32;
  if (groups * p.parts * col_blocks > INT32_MAX || groups * 2 * col_blocks > INT32_MAX)
    return set_error(FLUXB_ERR_UNSUPPORTED, "layer_norm_bwd: too many groups");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = dtype == FLUXB_BF16 ? launch_bwd<__nv_bfloat16>(a, p, sums, st) : launch_bwd<float>(a, p, sums, st);
  if (rc != FLUXB_OK) return rc;
  if (sums) {
    const unsigned rgrid = (unsigned)(groups * 2 * col_blocks);
    if (dtype == FLUXB_BF16 && !grads_f32)
      ln_bwd_reduce_kernel<__nv_bfloat16><<<rgrid, 256, 0, st>>>(scratch, static_cast<__nv_bfloat16*>(dfactor),
                                                                static_cast<__nv_bfloat16*>(doffset), p.parts, (int)cols);
    else
      ln_bwd_reduce_kernel<float><<<rgrid, 256, 0, st>>>(scratch, static_cast<float*>(dfactor), static_cast<float*>(doffset),
                                                        p.parts, (int)cols);
  }
  return ln_status("layer_norm_bwd");
}
