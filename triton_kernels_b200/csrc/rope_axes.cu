// Rotary positions with several axes, from position ids: pair j of a token belongs to one axis and turns by
//   angle(l, j) = ids[b, l, axis(j)] * theta^(-2 j' / d_axis),   (a, b) -> (a cos - b sin, a sin + b cos)
// with j' the pair's index within its axis.  Every batch item has positions of its own.  The backward pass is the
// same rotation by the negative angle.
//
// Angles: the position times the pair's turns per unit position (theta^(-2j'/d) / 2 pi, from the host in fp64) is
// taken in fp64 and reduced to [-1/2, 1/2] turns there, so that positions of any size keep an angle exact to
// 2^-25 turns; sine and cosine of the reduced turn are fp32.
#include <math.h>

#include "vec.cuh"

namespace fluxb {

constexpr int kMaxPairs = 128;
constexpr int kMaxAxes = 8;

struct RopeTensor {
  const void* src;
  void* dst;
  int64_t sb, sh, sl;  // source strides in elements
  int64_t ob, oh, ol;  // destination strides
  int heads;
};

struct RopeAxesArgs {
  RopeTensor t[2];  // q, k
  const void* ids;
  int64_t id_sb, id_sl, id_sa;
  int64_t B, L;
  int groups;    // of heads, one per blockIdx.y
  int D, pairs;  // pairs <= D/2; the columns from 2*pairs on are copied
  float sign;    // +1 forward, -1 backward
  double turns[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

template <typename Id>
__device__ __forceinline__ float2 turn_of(const RopeAxesArgs& a, int64_t b, int64_t l, int j) {
  const double pos = static_cast<double>(static_cast<const Id*>(a.ids)[b * a.id_sb + l * a.id_sl + a.axis[j] * a.id_sa]);
  const double t = pos * a.turns[j];
  const float r = static_cast<float>(t - rint(t));
  float s, c;
  sincospif(2.f * r, &s, &c);
  return make_float2(c, a.sign * s);
}

// Rows of whole 16-byte pieces: a thread owns one piece of one token's rows and walks heads of q and k, so its sines and
// cosines stay in registers for all of them and no table is read or written; eight pieces are in flight per thread,
// the first eight while the angles are taken.  The heads are dealt to blockIdx.y when there are few tokens.  Bound by
// HBM: every element is read once and written once.
template <typename T, typename Id>
__global__ void __launch_bounds__(256) rope_axes_vec_kernel(const __grid_constant__ RopeAxesArgs a) {
  constexpr int VN = Vec<T>::N;
  constexpr int kAhead = 8;
  const int pieces = a.D / VN;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= (int)(a.B * a.L) * pieces) return;
  const int tok = i / pieces, piece = i - tok * pieces;
  const int b = tok / (int)a.L, l = tok - b * (int)a.L;
  const int heads = a.t[0].heads + a.t[1].heads;
  const int h0 = (int)((int64_t)blockIdx.y * heads / a.groups), h1 = (int)((int64_t)(blockIdx.y + 1) * heads / a.groups);
  const T* src[2];
  T* dst[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    src[w] = static_cast<const T*>(a.t[w].src) + b * a.t[w].sb + l * a.t[w].sl + piece * VN;
    dst[w] = static_cast<T*>(a.t[w].dst) + b * a.t[w].ob + l * a.t[w].ol + piece * VN;
  }
  const int hq = a.t[0].heads;
  uint4 raw[kAhead];
  auto ask = [&](int h) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (h + u < h1) raw[u] = ld_nc_u4(h + u < hq ? src[0] + (h + u) * a.t[0].sh : src[1] + (h + u - hq) * a.t[1].sh);
    }
  };
  ask(h0);
  const int j0 = piece * (VN / 2);
  float2 cs[VN / 2];
#pragma unroll
  for (int p = 0; p < VN / 2; ++p) cs[p] = j0 + p < a.pairs ? turn_of<Id>(a, b, l, j0 + p) : make_float2(1.f, 0.f);
  for (int h = h0; h < h1; h += kAhead) {
    if (h > h0) ask(h);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (h + u < h1) {
        T* out = h + u < hq ? dst[0] + (h + u) * a.t[0].oh : dst[1] + (h + u - hq) * a.t[1].oh;
        if (j0 >= a.pairs) {  // behind the axes: copied
          *reinterpret_cast<uint4*>(out) = raw[u];
          continue;
        }
        Vec<T> v;
        v.unpack(raw[u]);
#pragma unroll
        for (int p = 0; p < VN / 2; ++p) {
          if (j0 + p < a.pairs) {
            const float x0 = v.v[2 * p], x1 = v.v[2 * p + 1];
            v.v[2 * p] = x0 * cs[p].x - x1 * cs[p].y;
            v.v[2 * p + 1] = x0 * cs[p].y + x1 * cs[p].x;
          }
        }
        v.store(out);
      }
    }
  }
}

// Any other layout.  One thread per (token, pair or trailing element pair), over all heads of q and k.
template <typename T, typename Id>
__global__ void __launch_bounds__(256) rope_axes_any_kernel(const __grid_constant__ RopeAxesArgs a) {
  const int half = (a.D + 1) / 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.L * half) return;
  const int j = (int)(i % half);
  const int64_t tok = i / half, b = tok / a.L, l = tok % a.L;
  const bool rot = j < a.pairs;
  const float2 cs = rot ? turn_of<Id>(a, b, l, j) : make_float2(1.f, 0.f);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const RopeTensor& t = a.t[w];
    for (int h = 0; h < t.heads; ++h) {
      const T* src = static_cast<const T*>(t.src) + b * t.sb + h * t.sh + l * t.sl + 2 * j;
      T* dst = static_cast<T*>(t.dst) + b * t.ob + h * t.oh + l * t.ol + 2 * j;
      const float x0 = static_cast<float>(src[0]), x1 = 2 * j + 1 < a.D ? static_cast<float>(src[1]) : 0.f;
      if (rot) {
        dst[0] = static_cast<T>(x0 * cs.x - x1 * cs.y);
        dst[1] = static_cast<T>(x0 * cs.y + x1 * cs.x);
      } else {
        dst[0] = src[0];
        if (2 * j + 1 < a.D) dst[1] = src[1];
      }
    }
  }
}

}  // namespace fluxb

using namespace fluxb;

extern "C" int fluxb_rope_axes(const void* q, void* oq, const int64_t* q_strides, const int64_t* oq_strides, int64_t Hq,
                               const void* k, void* ok, const int64_t* k_strides, const int64_t* ok_strides, int64_t Hk,
                               const void* ids, int id_type, const int64_t* id_strides, int64_t B, int64_t L, int64_t D,
                               const int64_t* axes_dim, int n_axes, double theta, int backward, int dtype,
                               fluxb_stream_t stream) {
  if (dtype != FLUXB_F32 && dtype != FLUXB_BF16) return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: dtype %d", dtype);
  if (id_type != FLUXB_ID_F32 && id_type != FLUXB_ID_I32 && id_type != FLUXB_ID_I64)
    return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: id type %d", id_type);
  if (B < 0 || L < 0 || D <= 0 || Hq < 0 || Hk < 0) return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: bad sizes");
  if (n_axes < 1 || n_axes > kMaxAxes || !axes_dim)
    return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: 1 to %d axes, got %d", kMaxAxes, n_axes);
  if (!(theta > 0.0) || !isfinite(theta)) return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: theta must be positive");
  int64_t rot = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (axes_dim[i] <= 0 || axes_dim[i] % 2 || axes_dim[i] > D)
      return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: every axis needs an even, positive dim");
    rot += axes_dim[i];
  }
  if (rot > D) return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: the axes' dims add up to %lld, more than head_dim %lld",
                                (long long)rot, (long long)D);
  if (rot / 2 > kMaxPairs) return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: more than %d rotated pairs", kMaxPairs);
  if (B == 0 || L == 0 || Hq + Hk == 0) return FLUXB_OK;
  if (!ids || !id_strides || (Hq > 0 && (!q || !oq || !q_strides || !oq_strides)) ||
      (Hk > 0 && (!k || !ok || !k_strides || !ok_strides)))
    return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: null pointer");
  const int64_t half = (D + 1) / 2;
  if (D > (1 << 16) || Hq > (1 << 20) || Hk > (1 << 20) || B * L > INT32_MAX || (B * L * half + 255) / 256 > INT32_MAX)
    return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: too many tokens or heads");
  RopeAxesArgs a;
  const int64_t zero[3] = {0, 0, 0};
  const int64_t *qs = Hq > 0 ? q_strides : zero, *qo = Hq > 0 ? oq_strides : zero;
  const int64_t *ks = Hk > 0 ? k_strides : zero, *ko = Hk > 0 ? ok_strides : zero;
  a.t[0] = RopeTensor{q, oq, qs[0], qs[1], qs[2], qo[0], qo[1], qo[2], (int)Hq};
  a.t[1] = RopeTensor{k, ok, ks[0], ks[1], ks[2], ko[0], ko[1], ko[2], (int)Hk};
  a.ids = ids;
  a.id_sb = id_strides[0]; a.id_sl = id_strides[1]; a.id_sa = id_strides[2];
  a.B = B; a.L = L; a.D = (int)D;
  a.pairs = (int)(rot / 2);
  a.sign = backward ? -1.f : 1.f;
  const double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
  int p = 0;
  for (int i = 0; i < n_axes; ++i)
    for (int64_t j = 0; j < axes_dim[i] / 2; ++j, ++p) {
      a.turns[p] = pow(theta, -2.0 * (double)j / (double)axes_dim[i]) * kTurn;
      a.axis[p] = (uint8_t)i;
    }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const int64_t vthreads = B * L * (D / vn);
  bool whole = D % vn == 0 && vthreads <= INT32_MAX - 256;
  for (const RopeTensor& t : a.t) {
    if (t.heads == 0) continue;
    whole = whole && ((reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst)) & 15u) == 0;
    for (int64_t s : {t.sb, t.sh, t.sl, t.ob, t.oh, t.ol}) whole = whole && s % vn == 0;
  }
  if (whole) {
    // heads are split until there are about four blocks per SM, as long as a thread keeps eight
    const int64_t blocks = (vthreads + 255) / 256, heads = Hq + Hk;
    int64_t groups = 4 * sm_count() / blocks;
    if (groups > heads / 8) groups = heads / 8;
    if (groups < 1) groups = 1;
    a.groups = (int)groups;
    const dim3 vgrid((unsigned)blocks, (unsigned)groups);
#define FLUXB_ROPE_AXES(T)                                                                    \
  do {                                                                                        \
    if (id_type == FLUXB_ID_F32) rope_axes_vec_kernel<T, float><<<vgrid, 256, 0, st>>>(a);    \
    else if (id_type == FLUXB_ID_I32) rope_axes_vec_kernel<T, int><<<vgrid, 256, 0, st>>>(a); \
    else rope_axes_vec_kernel<T, long long><<<vgrid, 256, 0, st>>>(a);                        \
  } while (0)
    if (dtype == FLUXB_BF16) FLUXB_ROPE_AXES(__nv_bfloat16);
    else FLUXB_ROPE_AXES(float);
#undef FLUXB_ROPE_AXES
    cudaError_t ve = cudaGetLastError();
    if (ve != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "rope_axes: %s", cudaGetErrorString(ve));
    return FLUXB_OK;
  }
  const unsigned grid = (unsigned)((B * L * half + 255) / 256);
#define FLUXB_ROPE_AXES(T)                                                               \
  do {                                                                                   \
    if (id_type == FLUXB_ID_F32) rope_axes_any_kernel<T, float><<<grid, 256, 0, st>>>(a); \
    else if (id_type == FLUXB_ID_I32) rope_axes_any_kernel<T, int><<<grid, 256, 0, st>>>(a); \
    else rope_axes_any_kernel<T, long long><<<grid, 256, 0, st>>>(a);                    \
  } while (0)
  if (dtype == FLUXB_BF16) FLUXB_ROPE_AXES(__nv_bfloat16);
  else FLUXB_ROPE_AXES(float);
#undef FLUXB_ROPE_AXES
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FLUXB_ERR_CUDA, "rope_axes: %s", cudaGetErrorString(e));
  return FLUXB_OK;
}
