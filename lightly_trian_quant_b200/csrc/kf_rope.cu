// Rotary positions with several axes (row and column of a patch, time of a frame, ...), forward and gradient.
//
//   pair p of a head belongs to one axis; angle = pos[token][axis(p)] * freq(p)
//   (a, b) -> (a cos - b sin, b cos + a sin);  the gradient is the same turn by -angle
//   half layout: pair p = channels (p, p + P) of the first 2P, interleaved: (2p, 2p + 1); channels 2P.. pass through
//
// Bound by memory: x is read once and y written once.  An angle is worked out once per token and pair for all heads: the product in fp64
// and reduced to half turns there (a position of 10^6 times a frequency of 1 leaves fp32 with less than two digits of the angle), sine and
// cosine of the reduced angle in fp32 with its rounding put right to first order.  A CTA takes a few tokens; its threads ask for their
// first chunks of x, then work out the angles of the tokens while those are on their way.  51 205 x 32 x 64 bf16: 71 to 77 us (5.4 to 5.9 TB/s).
#include "kf_common.cuh"

namespace kf {

constexpr int ROPE_THREADS = 256, ROPE_MAX_PAIRS = 128, ROPE_MAX_TOKENS = 16;
// Chunks (or pairs of chunks) per thread in flight: 16 KB of loads per CTA, four CTAs per SM (with twice as many, which leave room for two CTAs, a batch of
// clips took 120 us instead of 89; with half as many interleaved ones 5003 x 9 x 80 fp32 10.6 instead of 8.2)
__host__ __device__ constexpr int rope_items(bool interleaved) { return interleaved ? 4 : 2; }

struct RopeArgs {
  const void *x, *pos;
  void* y;
  const double* freq;                // [P] in half turns per position (freq / pi)
  const int* axis;                   // [P]
  int64_t xs_g, xs_t, xs_h, ys_g, ys_t, ys_h;   // strides in elements: outer, token, head
  int64_t ps_t, ps_a;                // strides of pos
  int G, T, H, D, P;
  int inverse, tokens;               // tokens per CTA
  uint64_t by_chunks, by_heads;      // 2^32 / n rounded up: a division of less than 2^16 by a multiplication
};

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) RopeVec {
  T v[V];
};

// 16-byte accesses go through the cache as data that is used once: 51 205 x 32 x 64 bf16 91 -> 77 us.
template <typename Vec, typename T>
__device__ __forceinline__ Vec rope_load(const T* p) {
  if constexpr (sizeof(Vec) == 16) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const Vec*>(&u);
  } else {
    return *reinterpret_cast<const Vec*>(p);
  }
}
template <typename Vec, typename T>
__device__ __forceinline__ void rope_store(T* p, const Vec& v) {
  if constexpr (sizeof(Vec) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
  else *reinterpret_cast<Vec*>(p) = v;
}

template <typename T, typename TP, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS, 4) rope_axes_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int ROPE_ITEMS = rope_items(INTER);
  extern __shared__ float2 turn[];                                 // (cos, sin) [tokens][P]
  pdl_wait();
  using Vec = RopeVec<T, V>;
  // items of a head: half layout: P / V pairs of chunks, then what passes through; interleaved: 2P / V chunks, then what passes through
  const int rot = INTER ? 2 * a.P / V : a.P / V, nc = rot + (a.D - 2 * a.P) / V;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = a.T - t0 < a.tokens ? (int)(a.T - t0) : a.tokens, items = nt * a.H * nc;
  const T* const x0 = static_cast<const T*>(a.x) + blockIdx.y * a.xs_g + t0 * a.xs_t;
  T* const y0 = static_cast<T*>(a.y) + blockIdx.y * a.ys_g + t0 * a.ys_t;
  Vec lo[ROPE_ITEMS], hi[INTER ? 1 : ROPE_ITEMS];
  int at_c[ROPE_ITEMS], at_k[ROPE_ITEMS];
  int64_t to[ROPE_ITEMS];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < ROPE_ITEMS; ++u) {
      const uint32_t i = base + u * ROPE_THREADS + threadIdx.x;
      if ((int)i < items) {
        const uint32_t th = (uint32_t)(i * a.by_chunks >> 32), c = i - th * nc, k = (uint32_t)(th * a.by_heads >> 32), h = th - k * a.H;
        const int e = (int)c < rot ? c * V : 2 * a.P + ((int)c - rot) * V;
        const T* p = x0 + k * a.xs_t + h * a.xs_h + e;
        lo[u] = rope_load<Vec>(p);
        if constexpr (!INTER) {
          if ((int)c < rot) hi[u] = rope_load<Vec>(p + a.P);
        }
        at_c[u] = c;
        at_k[u] = k;
        to[u] = k * a.ys_t + h * a.ys_h + e;
      }
    }
  };
  load(0);
  for (int i = threadIdx.x; i < nt * a.P; i += ROPE_THREADS) {
    const int k = i / a.P, p = i - k * a.P;
    const double half = (double)static_cast<const TP*>(a.pos)[(t0 + k) * a.ps_t + a.axis[p] * a.ps_a] * a.freq[p];
    const double r = half - 2.0 * rint(0.5 * half);                // [-1, 1]
    const float rf = (float)r;
    const float rest = (float)(r - (double)rf) * 3.14159265358979f;
    float s, co;
    sincospif(rf, &s, &co);
    turn[i] = make_float2(fmaf(-s, rest, co), a.inverse ? -fmaf(co, rest, s) : fmaf(co, rest, s));
  }
  __syncthreads();
  for (int base = 0; base < items; base += ROPE_ITEMS * ROPE_THREADS) {
    if (base) load(base);
#pragma unroll
    for (int u = 0; u < ROPE_ITEMS; ++u) {
      if ((int)(base + u * ROPE_THREADS + threadIdx.x) >= items) break;
      T* q = y0 + to[u];
      if (at_c[u] < rot) {
        const float2* cs = turn + at_k[u] * a.P + at_c[u] * (INTER ? V / 2 : V);
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float2 t = cs[j];
            const float m = (float)lo[u].v[2 * j], n = (float)lo[u].v[2 * j + 1];
            lo[u].v[2 * j] = (T)(m * t.x - n * t.y);
            lo[u].v[2 * j + 1] = (T)(n * t.x + m * t.y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 t = cs[j];
            const float m = (float)lo[u].v[j], n = (float)hi[u].v[j];
            lo[u].v[j] = (T)(m * t.x - n * t.y);
            hi[u].v[j] = (T)(n * t.x + m * t.y);
          }
          rope_store(q + a.P, hi[u]);
        }
      }
      rope_store(q, lo[u]);
    }
  }
}

}  // namespace kf

using namespace kf;

template <typename T, typename TP, int V>
static int rope_launch(const RopeArgs& a, int interleaved, dim3 grid, cudaStream_t st) {
  // dependent launches at any number of rows (the 1): the kernel starts none early itself, so that only the gap between kernels closes (51 205 x 32 x 64 bf16 both
  // directions 147.4 -> 142.9 us)
  cudaError_t e;
  const size_t smem = (size_t)a.tokens * a.P * sizeof(float2);
  if (interleaved) {
    if constexpr (V == 1) {
      set_error("kf_rope_axes: interleaved pairs need an even alignment");
      return KF_ERR_BAD_ARGUMENT;
    } else {
      e = launch_maybe_pdl(1, rope_axes_kernel<T, TP, V, true>, grid, dim3(ROPE_THREADS), smem, st, a);
    }
  } else {
    e = launch_maybe_pdl(1, rope_axes_kernel<T, TP, V, false>, grid, dim3(ROPE_THREADS), smem, st, a);
  }
  return cuda_status(e, "kf_rope_axes launch");
}
template <typename T, typename TP>
static int rope_by_width(const RopeArgs& a, int interleaved, int V, dim3 grid, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (V == 8) return rope_launch<T, TP, 8>(a, interleaved, grid, st);
  }
  if (V == 4) return rope_launch<T, TP, 4>(a, interleaved, grid, st);
  if (V == 2) return rope_launch<T, TP, 2>(a, interleaved, grid, st);
  return rope_launch<T, TP, 1>(a, interleaved, grid, st);
}
template <typename T>
static int rope_by_pos(const RopeArgs& a, int pos_kind, int interleaved, int V, dim3 grid, cudaStream_t st) {
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
    return ((strides % v) | (p->D % v) | ((p->interleaved ? 2 * p->P : p->P) % v)) == 0 && base % (uintptr_t)(v * size) == 0;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  KF_REQUIRE(base % (uintptr_t)size == 0, "kf_rope_axes: misaligned tensor");
  if (p->interleaved && V == 1) {
    KF_REQUIRE(false, "kf_rope_axes: interleaved pairs need strides and addresses of whole pairs and an even number of channels");
  }
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != KF_OK) return rc;
  // Tokens per CTA: its threads' first items, but not so many that a short batch leaves SMs without one
  const int nc = (p->interleaved ? 2 * p->P : p->P) / V + (p->D - 2 * p->P) / V;
  KF_REQUIRE((int64_t)p->H * nc < 65536, "kf_rope_axes: %d heads of %d channels are more than a token may have", p->H, p->D);
  KF_REQUIRE(p->G < 65536, "kf_rope_axes: outer dimension of %d", p->G);
  int64_t tokens = (int64_t)rope_items(p->interleaved) * ROPE_THREADS / ((int64_t)p->H * nc);
  const int64_t spread = ((int64_t)p->T * p->G + 2 * sms - 1) / (2 * sms);
  tokens = tokens < spread ? tokens : spread;
  tokens = tokens < 1 ? 1 : tokens > ROPE_MAX_TOKENS ? ROPE_MAX_TOKENS : tokens;
  a.tokens = (int)tokens;
  a.by_chunks = ((1ull << 32) + nc - 1) / nc;
  a.by_heads = ((1ull << 32) + p->H - 1) / p->H;
  const dim3 grid((unsigned)(((int64_t)p->T + tokens - 1) / tokens), (unsigned)p->G);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == KF_F32) return rope_by_pos<float>(a, p->pos_kind, p->interleaved, V, grid, st);
  if (p->dtype == KF_BF16) return rope_by_pos<__nv_bfloat16>(a, p->pos_kind, p->interleaved, V, grid, st);
  return rope_by_pos<__half>(a, p->pos_kind, p->interleaved, V, grid, st);
}
