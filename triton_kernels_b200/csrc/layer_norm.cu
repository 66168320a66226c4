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

// ---- aligned rows ------------------------------------------------------------------------------------------
// Few rows: one block per row, the row in registers (kV 16-byte pieces per thread), so that a launch is one round of
// loads and two block sums.  One row of 3072 bf16: 3.3 us of kernel time against 5.0 with the warp-per-row kernel that
// stages rows through shared memory (which wins from several rows per SM on).
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
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int c = (i * 256 + threadIdx.x) * VN;
    if (c < a.cols) {
      raw[i] = ld_nc_u4(x + c);
      fr[i] = ld_nc_u4(fp + c);
      orw[i] = ld_nc_u4(op + c);
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

// Backward, one pass over x and dy: a team of `wpr` warps walks whole rows and keeps the column sums of its columns in
// registers (kV 16-byte pieces per thread), so a row is read once and everything that it gives - dx, its share of df and
// do - leaves from there.  The rows come through a ring in shared memory by bulk copies, one x row and one dy row a
// slot: a row in flight costs no registers, and the ring holds about 150 KB per SM.  Two sums per row (g and g h) meet
// in the team: shuffles, then one named barrier, whose other side also frees the row's slot for the next copy.  The
// factor is kept widened in shared memory.  At the end the block's teams add up their column sums in a fixed order and
// the block writes one partial row; ln_bwd_reduce_kernel adds those.
template <typename T, int kV>
__global__ void __launch_bounds__(512, 1) ln_bwd_team_kernel(const LnBwdArgs a) {
  constexpr int VN = Vec<T>::N;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ uint64_t bars[kMaxTeamSlots];
  __shared__ float2 red[2][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = warp / a.wpr, team_threads = a.wpr * 32, tid = threadIdx.x - team * team_threads;
  const int64_t group = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const uint32_t row_bytes = (uint32_t)a.cols * sizeof(T);
  float* factor = reinterpret_cast<float*>(dyn);  // [cols], then the teams' rings
  uint8_t* ring = dyn + (size_t)(a.cols * 4 + 127) / 128 * 128 + (size_t)team * a.slots * 2 * row_bytes;
  uint64_t* full = bars + team * a.slots;
  if (tid == 0) {
    for (int i = 0; i < a.slots; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  const T* x = static_cast<const T*>(a.x) + group * a.rows_per_group * a.x_ld;
  const T* dy = static_cast<const T*>(a.dy) + group * a.rows_per_group * a.dy_ld;
  const int64_t step = (int64_t)a.parts * a.teams;
  const int64_t first = part * a.teams + team;
  auto ask = [&](int64_t row, int slot) {
    uint8_t* dst = ring + (size_t)slot * 2 * row_bytes;
    mbar_expect_tx(&full[slot], 2 * row_bytes);
    bulk_load_row(dst, x + row * a.x_ld, row_bytes, &full[slot]);
    bulk_load_row(dst + row_bytes, dy + row * a.dy_ld, row_bytes, &full[slot]);
  };
  if (tid == 0) {
    for (int i = 0; i < a.slots; ++i)
      if (first + i * step < a.rows_per_group) ask(first + i * step, i);
  }
  const T* fp = a.factor != nullptr ? static_cast<const T*>(a.factor) + group * a.vec_stride : nullptr;
  for (int c = threadIdx.x; c < a.cols; c += blockDim.x) factor[c] = fp != nullptr ? a.unit + to_f(fp[c]) : 1.f;
  __syncthreads();

  float df[kV][VN], dof[kV][VN];
#pragma unroll
  for (int i = 0; i < kV; ++i)
#pragma unroll
    for (int j = 0; j < VN; ++j) df[i][j] = dof[i][j] = 0.f;
  const float inv_cols = 1.f / a.cols;
  int slot = 0, buf = 0;
  uint32_t phase = 0;
  for (int64_t r = first; r < a.rows_per_group; r += step) {
    const int64_t row = group * a.rows_per_group + r;
    const float mean = __ldg(a.mean + row), rstd = __ldg(a.rstd + row);
    bool ok = false;
    for (uint32_t spin = 0; spin < (1u << 24) && !ok; ++spin) ok = mbar_try_wait(&full[slot], phase);
    if (!ok) report_error(a.status, FLUXB_ERR_TIMEOUT, 72);  // carries on: the row's numbers are lost, nobody hangs
    const T* xs = reinterpret_cast<const T*>(ring + (size_t)slot * 2 * row_bytes);
    const T* ds = xs + a.cols;
    float g[kV][VN], h[kV][VN];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = (i * team_threads + tid) * VN;
      if (c < a.cols) {
        Vec<T> xv, dv;
        xv.load(xs + c);
        dv.load(ds + c);
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          h[i][j] = (xv.v[j] - mean) * rstd;
          g[i][j] = dv.v[j] * factor[c + j];
          s1 += g[i][j];
          s2 = fmaf(g[i][j], h[i][j], s2);
          df[i][j] = fmaf(dv.v[j], h[i][j], df[i][j]);
          dof[i][j] += dv.v[j];
        }
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (lane == 0) red[buf][warp] = make_float2(s1, s2);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(team_threads) : "memory");
    if (tid == 0 && r + a.slots * step < a.rows_per_group) ask(r + a.slots * step, slot);
    s1 = s2 = 0.f;
    for (int w = 0; w < a.wpr; ++w) {
      const float2 v = red[buf][team * a.wpr + w];
      s1 += v.x;
      s2 += v.y;
    }
    if (a.dx != nullptr) {
      const float k1 = -s1 * inv_cols * rstd, k2 = -s2 * inv_cols * rstd;
      T* dx = static_cast<T*>(a.dx) + row * a.dx_ld;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int c = (i * team_threads + tid) * VN;
        if (c < a.cols) {
          Vec<T> o;
#pragma unroll
          for (int j = 0; j < VN; ++j) o.v[j] = fmaf(h[i][j], k2, fmaf(g[i][j], rstd, k1));
          o.store(dx + c);
        }
      }
    }
    buf ^= 1;
    if (++slot == a.slots) { slot = 0; phase ^= 1; }
  }
  // the teams' column sums, added up by the first one; all copies have landed, the rings are free
  float* other = reinterpret_cast<float*>(dyn + (size_t)(a.cols * 4 + 127) / 128 * 128);
  for (int t = 1; t < a.teams; ++t) {
    __syncthreads();
    if (team == t) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int c = (i * team_threads + tid) * VN;
        if (c < a.cols) {
#pragma unroll
          for (int j = 0; j < VN; ++j) { other[c + j] = df[i][j]; other[a.cols + c + j] = dof[i][j]; }
        }
      }
    }
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int c = (i * team_threads + tid) * VN;
        if (c < a.cols) {
#pragma unroll
          for (int j = 0; j < VN; ++j) { df[i][j] += other[c + j]; dof[i][j] += other[a.cols + c + j]; }
        }
      }
    }
  }
  if (team == 0 && a.partial != nullptr) {
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = (i * team_threads + tid) * VN;
      if (c < a.cols) {
#pragma unroll
        for (int j = 0; j < VN; j += 4) {
          *reinterpret_cast<float4*>(out + c + j) = make_float4(df[i][j], df[i][j + 1], df[i][j + 2], df[i][j + 3]);
          *reinterpret_cast<float4*>(out + a.cols + c + j) = make_float4(dof[i][j], dof[i][j + 1], dof[i][j + 2], dof[i][j + 3]);
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
  float* factor = reinterpret_cast<float*>(dyn);         // [cols]
  float* sums = factor + (a.cols + 31) / 32 * 32;        // [kWarps][2][cols]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t group = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int64_t base = group * a.rows_per_group;
  const T* x = static_cast<const T*>(a.x) + base * a.x_ld;
  const T* dy = static_cast<const T*>(a.dy) + base * a.dy_ld;
  const int64_t step = (int64_t)a.parts * kWarps * kRows;
  uint4 xn[kRows][kV], dn[kRows][kV];
  float mn[kRows], rn[kRows];
  auto ask = [&](int64_t r0) {
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int64_t r = r0 + q;
      if (r < a.rows_per_group) {
        mn[q] = __ldg(a.mean + base + r);
        rn[q] = __ldg(a.rstd + base + r);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const int c = (i * 32 + lane) * VN;
          if (c < a.cols) {
            xn[q][i] = ld_nc_u4(x + r * a.x_ld + c);
            dn[q][i] = ld_nc_u4(dy + r * a.dy_ld + c);
          }
        }
      }
    }
  };
  int64_t r0 = (part * kWarps + warp) * kRows;
  ask(r0);
  const T* fp = a.factor != nullptr ? static_cast<const T*>(a.factor) + group * a.vec_stride : nullptr;
  for (int c = threadIdx.x; c < a.cols; c += blockDim.x) factor[c] = fp != nullptr ? a.unit + to_f(fp[c]) : 1.f;
  __syncthreads();
  float df[kV][VN], dof[kV][VN];
#pragma unroll
  for (int i = 0; i < kV; ++i)
#pragma unroll
    for (int j = 0; j < VN; ++j) df[i][j] = dof[i][j] = 0.f;
  const float inv_cols = 1.f / a.cols;
  for (; r0 < a.rows_per_group; r0 += step) {
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
      if (r0 + q >= a.rows_per_group) break;
      float g[kV][VN], h[kV][VN];
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int c = (i * 32 + lane) * VN;
        if (c < a.cols) {
          Vec<T> xv, dv;
          xv.unpack(xc[q][i]);
          dv.unpack(dc[q][i]);
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            h[i][j] = (xv.v[j] - mc[q]) * rc[q];
            g[i][j] = dv.v[j] * factor[c + j];
            s1 += g[i][j];
            s2 = fmaf(g[i][j], h[i][j], s2);
            df[i][j] = fmaf(dv.v[j], h[i][j], df[i][j]);
            dof[i][j] += dv.v[j];
          }
        }
      }
      const float k1 = -warp_sum(s1) * inv_cols * rc[q], k2 = -warp_sum(s2) * inv_cols * rc[q];
      if (a.dx != nullptr) {
        T* dx = static_cast<T*>(a.dx) + (base + r0 + q) * a.dx_ld;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const int c = (i * 32 + lane) * VN;
          if (c < a.cols) {
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < VN; ++j) o.v[j] = fmaf(h[i][j], k2, fmaf(g[i][j], rc[q], k1));
            o.store(dx + c);
          }
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  float* mine = sums + (size_t)warp * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    const int c = (i * 32 + lane) * VN;
    if (c < a.cols) {
#pragma unroll
      for (int j = 0; j < VN; ++j) { mine[c + j] = df[i][j]; mine[a.cols + c + j] = dof[i][j]; }
    }
  }
  __syncthreads();
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
  for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sums[(size_t)w * 2 * a.cols + c];
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
  enum Kind { kAny, kWarp, kTeam } kind;
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
      // pieces per thread: the most that registers hold (three of bf16, four of fp32), unless fewer leave fewer
      // lanes without a column
      int64_t best = -1;
      for (int k = vn == 8 ? 3 : 4; k >= 1; --k) {
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
  if (p.kind == BwdPlan::kAny) { blocks = 2 * sm_count(); rows_at_once = 8; }
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
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const bool whole = factor != nullptr && offset != nullptr && cols % vn == 0 && x_ld % vn == 0 && y_ld % vn == 0 &&
                     vec_stride % vn == 0 && all16(x, y, factor, offset);
  if (whole && rows <= 2 * sm_count() && cols <= 1024 * vn) {
    const int v = (int)((cols / vn + 255) / 256);
#define FLUXB_LN_BLOCK(T)                                                                    \
  do {                                                                                       \
    if (v == 1) ln_fwd_block_kernel<T, 1><<<(unsigned)rows, 256, 0, st>>>(a);                \
    else if (v == 2) ln_fwd_block_kernel<T, 2><<<(unsigned)rows, 256, 0, st>>>(a);           \
    else ln_fwd_block_kernel<T, 4><<<(unsigned)rows, 256, 0, st>>>(a);                       \
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
  if (dtype == FLUXB_BF16) ln_fwd_any_kernel<__nv_bfloat16><<<(unsigned)rows, 256, 0, st>>>(a);
  else ln_fwd_any_kernel<float><<<(unsigned)rows, 256, 0, st>>>(a);
  return ln_status("layer_norm");
}

extern "C" int64_t fluxb_layer_norm_bwd_scratch(int64_t rows, int64_t cols, int64_t rows_per_group) {
  if (rows <= 0 || cols <= 0 || rows_per_group <= 0) return 0;
  // the most that any of the kernels asks for: two blocks per SM over all groups
  const int64_t groups = rows / rows_per_group, want = 2 * sm_count() / (groups > 0 ? groups : 1);
  const int64_t parts = want < 1 ? 1 : (want < rows_per_group ? want : rows_per_group);
  return groups * parts * 2 * cols;
}

template <typename T>
static int launch_bwd(const LnBwdArgs& a, const BwdPlan& p, bool sums, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.groups * a.parts);
  if (p.kind == BwdPlan::kAny) {
    if (a.dx != nullptr) ln_bwd_rows_any_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a);
    if (sums) ln_bwd_cols_any_kernel<T><<<grid * (unsigned)((a.cols + 31) / 32), 256, 0, st>>>(a);
    return FLUXB_OK;
  }
  void (*kern)(LnBwdArgs) = nullptr;
  if (p.kind == BwdPlan::kWarp)
    kern = p.vecs == 1 ? ln_bwd_warp_kernel<T, 1> : (p.vecs == 2 ? ln_bwd_warp_kernel<T, 2> : ln_bwd_warp_kernel<T, 3>);
  else
    kern = p.vecs == 1   ? ln_bwd_team_kernel<T, 1>
           : p.vecs == 2 ? ln_bwd_team_kernel<T, 2>
           : p.vecs == 3 ? ln_bwd_team_kernel<T, 3>
                         : ln_bwd_team_kernel<T, sizeof(T) == 2 ? 3 : 4>;
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
