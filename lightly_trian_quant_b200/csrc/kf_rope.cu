// Rotary positions with several axes (row and column of a patch, time of a frame, ...), forward and gradient.
//
//   pair p of a head belongs to one axis; angle = pos[token][axis(p)] * freq(p)
//   (a, b) -> (a cos - b sin, b cos + a sin);  the gradient is the same turn by -angle
//   half layout: pair p = channels (p, p + P) of the first 2P, interleaved: (2p, 2p + 1); channels 2P.. pass through
//
// Bound by memory: x is read once and y written once.  An angle is worked out once per token and pair for all heads: the product in fp64
// and reduced to half turns there (a position of 10^6 times a frequency of 1 leaves fp32 with less than two digits of the angle), sine and
// cosine of the reduced angle in fp32 with its rounding put right to first order.  A thread owns one chunk of a head's channels, keeps
// its sines and cosines in registers and goes through the heads.
#include "kf_common.cuh"

namespace kf {

constexpr int ROPE_THREADS = 256, ROPE_MAX_PAIRS = 128, ROPE_TOKENS = 8;

struct RopeArgs {
  const void *x, *pos;
  void* y;
  const double* freq;                // [P] in half turns per position (freq / pi)
  const int* axis;                   // [P]
  int64_t xs_g, xs_t, xs_h, ys_g, ys_t, ys_h;   // strides in elements: outer, token, head
  int64_t ps_t, ps_a;                // strides of pos
  int G, T, H, D, P;
  int inverse;
};

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) RopeVec {
  T v[V];
};

template <typename T, typename TP, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_axes_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 turn[ROPE_TOKENS * ROPE_MAX_PAIRS];            // (cos, sin)
  pdl_wait();
  // chunks of a head: half layout: P / V pairs of chunks, then what passes through; interleaved: 2P / V chunks, then what passes through
  const int rot = INTER ? 2 * a.P / V : a.P / V, nc = rot + (a.D - 2 * a.P) / V;
  const int per = ROPE_THREADS / nc;                               // heads in flight
  const int c = threadIdx.x % nc, h0 = threadIdx.x / nc;
  for (int64_t t0 = (int64_t)blockIdx.x * ROPE_TOKENS; t0 < a.T; t0 += (int64_t)gridDim.x * ROPE_TOKENS) {
    const int nt = a.T - t0 < ROPE_TOKENS ? (int)(a.T - t0) : ROPE_TOKENS;
    for (int i = threadIdx.x; i < nt * a.P; i += ROPE_THREADS) {
      const int k = i / a.P, p = i - k * a.P;
      const double half = (double)static_cast<const TP*>(a.pos)[(t0 + k) * a.ps_t + a.axis[p] * a.ps_a] * a.freq[p];
      const double r = half - 2.0 * rint(0.5 * half);              // [-1, 1]
      const float rf = (float)r;
      const float rest = (float)(r - (double)rf) * 3.14159265358979f;
      float s, co;
      sincospif(rf, &s, &co);
      turn[k * a.P + p] = make_float2(fmaf(-s, rest, co), a.inverse ? -fmaf(co, rest, s) : fmaf(co, rest, s));
    }
    __syncthreads();
    if (h0 < per) {
      for (int k = 0; k < nt; ++k) {
        const T* xt = static_cast<const T*>(a.x) + (t0 + k) * a.xs_t;
        T* yt = static_cast<T*>(a.y) + (t0 + k) * a.ys_t;
        if (c >= rot) {
          const int e = 2 * a.P + (c - rot) * V;
          for (int g = 0; g < a.G; ++g)
            for (int h = h0; h < a.H; h += per)
              *reinterpret_cast<RopeVec<T, V>*>(yt + g * a.ys_g + h * a.ys_h + e) = *reinterpret_cast<const RopeVec<T, V>*>(xt + g * a.xs_g + h * a.xs_h + e);
        } else if constexpr (INTER) {
          float2 cs[V / 2];
#pragma unroll
          for (int j = 0; j < V / 2; ++j) cs[j] = turn[k * a.P + c * (V / 2) + j];
          for (int g = 0; g < a.G; ++g)
            for (int h = h0; h < a.H; h += per) {
              RopeVec<T, V> u = *reinterpret_cast<const RopeVec<T, V>*>(xt + g * a.xs_g + h * a.xs_h + c * V);
#pragma unroll
              for (int j = 0; j < V / 2; ++j) {
                const float p = (float)u.v[2 * j], q = (float)u.v[2 * j + 1];
                u.v[2 * j] = (T)(p * cs[j].x - q * cs[j].y);
                u.v[2 * j + 1] = (T)(q * cs[j].x + p * cs[j].y);
              }
              *reinterpret_cast<RopeVec<T, V>*>(yt + g * a.ys_g + h * a.ys_h + c * V) = u;
            }
        } else {
          float2 cs[V];
#pragma unroll
          for (int j = 0; j < V; ++j) cs[j] = turn[k * a.P + c * V + j];
          for (int g = 0; g < a.G; ++g)
            for (int h = h0; h < a.H; h += per) {
              const T* xp = xt + g * a.xs_g + h * a.xs_h + c * V;
              RopeVec<T, V> lo = *reinterpret_cast<const RopeVec<T, V>*>(xp), hi = *reinterpret_cast<const RopeVec<T, V>*>(xp + a.P);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const float p = (float)lo.v[j], q = (float)hi.v[j];
                lo.v[j] = (T)(p * cs[j].x - q * cs[j].y);
                hi.v[j] = (T)(q * cs[j].x + p * cs[j].y);
              }
              T* yp = yt + g * a.ys_g + h * a.ys_h + c * V;
              *reinterpret_cast<RopeVec<T, V>*>(yp) = lo;
              *reinterpret_cast<RopeVec<T, V>*>(yp + a.P) = hi;
            }
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace kf

using namespace kf;

template <typename T, typename TP, int V>
static int rope_launch(const RopeArgs& a, int interleaved, int grid, cudaStream_t st) {
  cudaError_t e;
  if (interleaved) {
    if constexpr (V == 1) {
      set_error("kf_rope_axes: interleaved pairs need an even alignment");
      return KF_ERR_BAD_ARGUMENT;
    } else {
      e = launch_maybe_pdl(a.T, rope_axes_kernel<T, TP, V, true>, dim3(grid), dim3(ROPE_THREADS), 0, st, a);
    }
  } else {
    e = launch_maybe_pdl(a.T, rope_axes_kernel<T, TP, V, false>, dim3(grid), dim3(ROPE_THREADS), 0, st, a);
  }
  return cuda_status(e, "kf_rope_axes launch");
}
template <typename T, typename TP>
static int rope_by_width(const RopeArgs& a, int interleaved, int V, int grid, cudaStream_t st) {
  if (V == 8) return rope_launch<T, TP, 8>(a, interleaved, grid, st);
  if (V == 4) return rope_launch<T, TP, 4>(a, interleaved, grid, st);
  if (V == 2) return rope_launch<T, TP, 2>(a, interleaved, grid, st);
  return rope_launch<T, TP, 1>(a, interleaved, grid, st);
}
template <typename T>
static int rope_by_pos(const RopeArgs& a, int pos_kind, int interleaved, int V, int grid, cudaStream_t st) {
  if (pos_kind == KF_POS_I32) return rope_by_width<T, int32_t>(a, interleaved, V, grid, st);
  if (pos_kind == KF_POS_I64) return rope_by_width<T, int64_t>(a, interleaved, V, grid, st);
  return rope_by_width<T, float>(a, interleaved, V, grid, st);
}

extern "C" int kf_rope_axes(const kf_rope_params* p, void* stream) {
  KF_REQUIRE(p, "kf_rope_axes: null parameter block");
  KF_REQUIRE(p->dtype == KF_F32 || p->dtype == KF_BF16 || p->dtype == KF_F16, "kf_rope_axes: type must be f32, bf16 or f16");
  KF_REQUIRE(p->pos_kind == KF_POS_I32 || p->pos_kind == KF_POS_I64 || p->pos_kind == KF_POS_F32, "kf_rope_axes: positions must be int32, int64 or fp32");
  KF_REQUIRE(p->G >= 0 && p->T >= 0 && p->H >= 0 && p->D > 0 && p->P >= 0 && 2 * p->P <= p->D && p->P <= ROPE_MAX_PAIRS && p->D <= 2 * ROPE_MAX_PAIRS,
             "kf_rope_axes: bad shape G=%d T=%d H=%d D=%d with %d pairs (at most %d channels)", p->G, p->T, p->H, p->D, p->P, 2 * ROPE_MAX_PAIRS);
  if (p->G == 0 || p->T == 0 || p->H == 0) return KF_OK;
  KF_REQUIRE(p->x && p->y && (p->P == 0 || (p->pos && p->freq && p->axis)), "kf_rope_axes: null pointer");
  RopeArgs a{};
  a.x = p->x; a.y = p->y; a.pos = p->pos; a.freq = p->freq; a.axis = p->axis;
  a.xs_g = p->xs_g; a.xs_t = p->xs_t; a.xs_h = p->xs_h; a.ys_g = p->ys_g; a.ys_t = p->ys_t; a.ys_h = p->ys_h; a.ps_t = p->ps_t; a.ps_a = p->ps_a;
  a.G = p->G; a.T = p->T; a.H = p->H; a.D = p->D; a.P = p->P; a.inverse = p->inverse != 0;
  // the widest access that every chunk's address is a multiple of
  const int64_t size = p->dtype == KF_F32 ? 4 : 2;
  int V = 16 / (int)size;
  const int64_t strides = p->xs_g | p->xs_t | p->xs_h | p->ys_g | p->ys_t | p->ys_h;
  const uintptr_t base = reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->y);
  auto fits = [&](int v) {
    return ((strides % v) | (p->D % v) | ((p->interleaved ? 2 * p->P : p->P) % v)) == 0 && base % (uintptr_t)(v * size) == 0 && p->D / v <= ROPE_THREADS;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  KF_REQUIRE(base % (uintptr_t)size == 0, "kf_rope_axes: misaligned tensor");
  if (p->interleaved && V == 1) {
    KF_REQUIRE(false, "kf_rope_axes: interleaved pairs need strides and addresses of whole pairs and an even number of channels");
  }
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != KF_OK) return rc;
  const int64_t blocks = ((int64_t)p->T + ROPE_TOKENS - 1) / ROPE_TOKENS;
  const int grid = (int)(blocks < 8 * sms ? blocks : 8 * sms);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == KF_F32) return rope_by_pos<float>(a, p->pos_kind, p->interleaved, V, grid, st);
  if (p->dtype == KF_BF16) return rope_by_pos<__nv_bfloat16>(a, p->pos_kind, p->interleaved, V, grid, st);
  return rope_by_pos<__half>(a, p->pos_kind, p->interleaved, V, grid, st);
}
