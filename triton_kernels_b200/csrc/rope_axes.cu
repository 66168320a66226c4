// Rotary positions with several axes, from position ids: pair j of a token belongs to one axis and turns by
//   angle(l, j) = ids[b, l, axis(j)] * theta^(-2 j' / d_axis),   (a, b) -> (a cos - b sin, a sin + b cos)
// with j' the pair's index within its axis.  Every batch item has positions of its own.  The backward pass is the
// same rotation by the negative angle.
//
// Angles: the position times the pair's turns per unit position (theta^(-2j'/d) / 2 pi, from the host in fp64) is
// taken exactly enough that the turn left over after whole turns is right to 2^-24 for up to 2^27 turns: in two fp32
// parts for positions below 2^24 and less than 2^22 turns (the low part's rounding 2^-26, that of adding what it gives
// 2^-26, the sum's 2^-25), in fp64 beyond (frequency and product each 2^-53 of the turns, 2^-25 at 2^27 of them, and 2^-26
// for the result in fp32; past that the error grows with the turns, and integers above 2^53 are rounded first).  (fp64
// throughout: 17.5 us instead of 15.9 for 16 heads of 8192 tokens.)  Sine and cosine of the reduced turn are fp32.
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
  int tokens, slots;  // per block (16-byte pieces)
  int D, pairs;  // pairs <= D/2; the columns from 2*pairs on are copied
  float sign;    // +1 forward, -1 backward
  double turns[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

// A frequency as two fp32 parts.
__device__ __forceinline__ float2 split(double f) {
  const float high = static_cast<float>(f);
  return make_float2(high, static_cast<float>(f - high));
}

// Cosine and signed sine of position `id` for pair j, whose frequency is `turns`.
template <typename Id>
__device__ __forceinline__ float2 turn_of(const RopeAxesArgs& a, Id id, int j, float2 turns) {
  float r;
  const float pos = static_cast<float>(id), high = pos * turns.x;
  if (id > static_cast<Id>(-(1 << 24)) && id < static_cast<Id>(1 << 24) && fabsf(high) < 4194304.f) {
    // pos is exact in fp32 and the turn count below 2^22 (a theta below one may turn faster): the product as high part
    // and error, both exact, the whole turns taken off the high part (exact, too), then what the frequency's low part
    // adds (2^-48 of the turns off)
    const float whole = (high + 12582912.f) - 12582912.f;  // 1.5 * 2^23: to the nearest integer
    r = (high - whole) + fmaf(pos, turns.y, fmaf(pos, turns.x, -high));
  } else {
    const double t = static_cast<double>(id) * a.turns[j];
    r = static_cast<float>(t - rint(t));
  }
  float s, c;
  sincospif(2.f * r, &s, &c);
  return make_float2(c, a.sign * s);
}

// Rows of whole 16-byte pieces.  A block takes a few tokens; a thread owns one piece of one token's rows, keeps its four
// pairs' sines and cosines in registers and walks every `slots`-th head of q and k.  A pair's angle is so taken once, no
// table is read or written, and the next kAhead pieces of a thread are on their way while it works on the current ones.
// Bound by HBM: every element is read once and written once; 24 + 24 heads of 4608 tokens, 128 columns bf16: 21.0 us, 5.4
// TB/s.  (With the angles taken again for every group of heads: 37 us.)  At four blocks per SM the bf16 form without
// sharing spills 28 to 44 bytes a thread.
// kShare: where several threads walk the same piece's heads (slots > 1), the block's threads first take one angle each and
// pass them on through shared memory; where a piece has one thread it takes its own.  With 512 tokens of 8 + 8 heads sharing
// takes 5.1 us and not sharing 6.2; with one thread a piece the barriers cost: 16 x 4096 tokens of 1 + 1 heads, 64 columns,
// 23.2 us sharing, 16.9 not; 16 + 4 heads of 16896 tokens fp32 31.4 and 30.4.
template <typename T, typename Id, bool kShare>
__global__ void __launch_bounds__(256, 4) rope_axes_vec_kernel(const __grid_constant__ RopeAxesArgs a) {
  constexpr int VN = Vec<T>::N;
  constexpr int kAhead = 3;
  extern __shared__ float2 table[];  // [tokens][D / 2] (kShare)
  __shared__ float2 turns[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  // (the kernel's parameters can be read at one address per warp and cycle only: with lanes that
  // each read their own pair's there, 65536 tokens with one head took 45.6 us instead of 37.7)
  if (threadIdx.x < a.pairs) {
    turns[threadIdx.x] = split(a.turns[threadIdx.x]);
    axis[threadIdx.x] = a.axis[threadIdx.x];
  }
  __syncthreads();
  pdl_wait();  // the block may have started while the kernel in front was ending
  pdl_release();
  const int pieces = a.D / VN, half = a.D / 2;
  const int tokens = (int)(a.B * a.L);
  const int piece = threadIdx.x % pieces, rest = threadIdx.x / pieces;
  const int t = rest % a.tokens, slot = rest / a.tokens;
  for (int tok0 = blockIdx.x * a.tokens; tok0 < tokens; tok0 += gridDim.x * a.tokens) {
  const int tok = tok0 + t;
  const bool active = slot < a.slots && tok < tokens;
  const int b = tok / (int)a.L, l = tok - b * (int)a.L;
  // This thread's heads are slot, slot + slots, ... of q and then of k, kAhead at a time.
  const int64_t at[4] = {b * a.t[0].sb + l * a.t[0].sl + slot * a.t[0].sh, b * a.t[1].sb + l * a.t[1].sl + slot * a.t[1].sh,
                         b * a.t[0].ob + l * a.t[0].ol + slot * a.t[0].oh, b * a.t[1].ob + l * a.t[1].ol + slot * a.t[1].oh};
  const T *sq = static_cast<const T*>(a.t[0].src) + at[0] + piece * VN, *sk = static_cast<const T*>(a.t[1].src) + at[1] + piece * VN;
  T *dq = static_cast<T*>(a.t[0].dst) + at[2] + piece * VN, *dk = static_cast<T*>(a.t[1].dst) + at[3] + piece * VN;
  const int64_t qs = a.slots * a.t[0].sh, ks = a.slots * a.t[1].sh, qo = a.slots * a.t[0].oh, ko = a.slots * a.t[1].oh;
  int nq = active && slot < a.t[0].heads ? (a.t[0].heads - slot + a.slots - 1) / a.slots : 0;
  int nk = active && slot < a.t[1].heads ? (a.t[1].heads - slot + a.slots - 1) / a.slots : 0;
  uint4 next[kAhead];
  auto load = [&](const T* p, int64_t step, int n) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u, p += step)
      if (u < n) next[u] = ld_u4(p);
  };
  if (nq > 0) load(sq, qs, nq);
  else load(sk, ks, nk);
  const int rotated = min(VN / 2, a.pairs - piece * (VN / 2));  // pairs of this piece: all, some, or none (0 or less)
  const Id* const ids = static_cast<const Id*>(a.ids);
  float2 cs[VN / 2];
  if constexpr (kShare) {
#pragma unroll 4
    for (int i = threadIdx.x; i < a.tokens * half; i += 256) {
      const int ti = i / half, j = i - ti * half;
      if (tok0 + ti < tokens && j < a.pairs) {
        const int bi = (tok0 + ti) / (int)a.L;
        const Id id = ids[bi * a.id_sb + (tok0 + ti - bi * (int)a.L) * a.id_sl + axis[j] * a.id_sa];
        table[i] = turn_of<Id>(a, id, j, turns[j]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < VN / 2; ++p)
      if (active && p < rotated) cs[p] = table[t * half + piece * (VN / 2) + p];
  } else {
    Id id[VN / 2];
#pragma unroll
    for (int p = 0; p < VN / 2; ++p)
      if (active && p < rotated) id[p] = ids[b * a.id_sb + l * a.id_sl + axis[piece * (VN / 2) + p] * a.id_sa];
#pragma unroll
    for (int p = 0; p < VN / 2; ++p)
      if (active && p < rotated) cs[p] = turn_of<Id>(a, id[p], piece * (VN / 2) + p, turns[piece * (VN / 2) + p]);
  }
  auto finish = [&](T* p, int64_t step, const uint4 (&now)[kAhead], int n) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u, p += step) {
      if (u >= n) break;
      if (rotated == VN / 2) {
        Vec<T> v;
        v.unpack(now[u]);
#pragma unroll
        for (int e = 0; e < VN / 2; ++e) {
          const float x0 = v.v[2 * e], x1 = v.v[2 * e + 1];
          v.v[2 * e] = x0 * cs[e].x - x1 * cs[e].y;
          v.v[2 * e + 1] = x0 * cs[e].y + x1 * cs[e].x;
        }
        v.store(p);
      } else if (rotated <= 0) {  // behind the axes: copied
        *reinterpret_cast<uint4*>(p) = now[u];
      } else {
        Vec<T> v;
        v.unpack(now[u]);
#pragma unroll
        for (int e = 0; e < VN / 2; ++e) {
          if (e < rotated) {
            const float x0 = v.v[2 * e], x1 = v.v[2 * e + 1];
            v.v[2 * e] = x0 * cs[e].x - x1 * cs[e].y;
            v.v[2 * e + 1] = x0 * cs[e].y + x1 * cs[e].x;
          }
        }
        v.store(p);
      }
    }
  };
  uint4 now[kAhead];
  while (nq > 0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now[u] = next[u];
    sq += kAhead * qs;
    if (nq > kAhead) load(sq, qs, nq - kAhead);
    else load(sk, ks, nk);
    finish(dq, qo, now, nq);
    dq += kAhead * qo;
    nq -= kAhead;
  }
  while (nk > 0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now[u] = next[u];
    sk += kAhead * ks;
    if (nk > kAhead) load(sk, ks, nk - kAhead);
    finish(dk, ko, now, nk);
    dk += kAhead * ko;
    nk -= kAhead;
  }
  if constexpr (kShare) __syncthreads();  // the table is free
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
  const float2 cs = rot ? turn_of<Id>(a, __ldg(static_cast<const Id*>(a.ids) + b * a.id_sb + l * a.id_sl + a.axis[j] * a.id_sa), j, split(a.turns[j])) : make_float2(1.f, 0.f);
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

extern "C" int fluxb_rope_axes(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sl, void* oq, int64_t oq_sb,
                               int64_t oq_sh, int64_t oq_sl, int64_t Hq, const void* k, int64_t k_sb, int64_t k_sh,
                               int64_t k_sl, void* ok, int64_t ok_sb, int64_t ok_sh, int64_t ok_sl, int64_t Hk,
                               const void* ids, int id_type, int64_t id_sb, int64_t id_sl, int64_t id_sa, int64_t B,
                               int64_t L, int64_t D, const int64_t* axes_dim, int n_axes, double theta, int backward,
                               int dtype, fluxb_stream_t stream) {
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
  if (!ids || (Hq > 0 && (!q || !oq)) || (Hk > 0 && (!k || !ok)))
    return set_error(FLUXB_ERR_BAD_ARG, "rope_axes: null pointer");
  const int64_t half = (D + 1) / 2;
  if (D > (1 << 16) || Hq > (1 << 20) || Hk > (1 << 20) || B > (1 << 30) || L > (1 << 30) || B * L > (1 << 30) || (B * L * half + 255) / 256 > INT32_MAX)
    return set_error(FLUXB_ERR_UNSUPPORTED, "rope_axes: too many tokens or heads");
  RopeAxesArgs a;
  a.t[0] = RopeTensor{q, oq, q_sb, q_sh, q_sl, oq_sb, oq_sh, oq_sl, (int)Hq};
  a.t[1] = RopeTensor{k, ok, k_sb, k_sh, k_sl, ok_sb, ok_sh, ok_sl, (int)Hk};
  a.ids = ids;
  a.id_sb = id_sb; a.id_sl = id_sl; a.id_sa = id_sa;
  a.B = B; a.L = L; a.D = (int)D;
  a.pairs = (int)(rot / 2);
  a.sign = backward ? -1.f : 1.f;
  // theta^(-2j/d) / 2 pi, one factor after the other in extended precision (64 bits: at most 2^-55 of the value off before
  // it is rounded to fp64).  With a pow() per pair this took the host 1.6 us of a call's 7.5; so 0.5.
  const long double kTurn = 0.15915494309189533576888L, log2_theta = log2l((long double)theta);
  int p = 0;
  for (int i = 0; i < n_axes; ++i) {
    const long double ratio = exp2l(-2.0L * log2_theta / (long double)axes_dim[i]);
    long double turn = kTurn;
    for (int64_t j = 0; j < axes_dim[i] / 2; ++j, ++p, turn *= ratio) {
      a.turns[p] = (double)turn;
      a.axis[p] = (uint8_t)i;
    }
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int vn = dtype == FLUXB_BF16 ? 8 : 4;
  const int64_t pieces = D / vn;
  bool whole = D % vn == 0 && pieces <= 256 && D <= 2048;
  for (const RopeTensor& t : a.t) {
    if (t.heads == 0) continue;
    whole = whole && ((reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst)) & 15u) == 0;
    for (int64_t s : {t.sb, t.sh, t.sl, t.ob, t.oh, t.ol}) whole = whole && s % vn == 0;
  }
  if (whole) {
    // Threads of a block: pieces x tokens x slots of heads.  A thread takes all heads (16 heads: 16.5 us with one slot,
    // 18.0 with four), unless the tokens fill too few blocks.
    int64_t slots = 1, heads = Hq + Hk;
    while (slots * 2 <= heads && pieces * slots * 2 <= 256 && B * L <= 2 * sm_count() * (256 / (pieces * slots))) slots *= 2;
    a.slots = (int)slots;
    a.tokens = (int)(256 / (pieces * slots));
    const int64_t most = 4 * sm_count(), blocks = (B * L + a.tokens - 1) / a.tokens;
    const unsigned vgrid = (unsigned)(blocks < most ? blocks : most);
    const bool share = slots > 1;
    cudaError_t ve;
    const size_t smem = share ? (size_t)a.tokens * (D / 2) * sizeof(float2) : 0;
#define FLUXB_ROPE_AXES(T, Id)                                                             \
  do {                                                                                     \
    ve = share ? launch_after(rope_axes_vec_kernel<T, Id, true>, vgrid, 256, smem, st, a)  \
               : launch_after(rope_axes_vec_kernel<T, Id, false>, vgrid, 256, 0, st, a);   \
  } while (0)
    if (dtype == FLUXB_BF16) {
      if (id_type == FLUXB_ID_F32) FLUXB_ROPE_AXES(__nv_bfloat16, float);
      else if (id_type == FLUXB_ID_I32) FLUXB_ROPE_AXES(__nv_bfloat16, int);
      else FLUXB_ROPE_AXES(__nv_bfloat16, long long);
    } else {
      if (id_type == FLUXB_ID_F32) FLUXB_ROPE_AXES(float, float);
      else if (id_type == FLUXB_ID_I32) FLUXB_ROPE_AXES(float, int);
      else FLUXB_ROPE_AXES(float, long long);
    }
#undef FLUXB_ROPE_AXES
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
