// LayerNorm for training: forward that keeps each row's statistics, and the gradients of rows, weight and bias.
//
//   y  = xh * w + b,  xh = (x - mean) * rstd
//   g  = dy * w;  dx = rstd * (g - mean(g) - xh * mean(g * xh)) (+ dres);  dw = sum over rows of dy * xh;  db = sum over rows of dy
//
// A row belongs to a group of W warps (1, 2, 4 or 8 of a CTA's 8), its values stay in registers between the statistics and their use: one
// pass over memory in either direction, which is what bounds both.  Rows come through shared memory by bulk copies, one row ahead of the one
// that a group works on: loads into registers left the memory idle while a warp reduced (22 470 x 1024, fp32 rows: backward 140 us).  A
// copy takes the 16-byte units that hold the row, whatever its address; they are read in chunks of 8 values where width, strides and
// addresses allow 16-byte accesses and one value per lane otherwise.  Statistics, sums and products in fp32 whatever the tensors' types.
// The weight's gradient is summed in registers over the rows of a group, over the groups of a CTA through shared memory in their order, and
// over the CTAs by a second launch: no atomics, the same bits from run to run.
// Measured, 22 470 x 1024, fp32 rows, 16-bit output: forward 26 us (5.4 TB/s), gradients with a residual's 56 us (5.7 TB/s) and 3 us for the column sums.
#include "kf_sm100.cuh"

namespace kf {

constexpr int LN_THREADS = 256, LN_WARPS = 8, LN_MAX_WIDTH = 8192;

template <typename T>
__device__ __forceinline__ float ln_to_float(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ uint32_t ln_pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 ln_unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <int CH, typename T>
__device__ __forceinline__ void ln_load(const T* p, float (&v)[CH]) {
  if constexpr (CH == 1) {
    v[0] = ln_to_float(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = ln_unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <int CH, typename T>
__device__ __forceinline__ void ln_store(T* p, const float (&v)[CH]) {
  if constexpr (CH == 1) {
    *p = static_cast<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(ln_pack2<T>(v[0], v[1]), ln_pack2<T>(v[2], v[3]), ln_pack2<T>(v[4], v[5]), ln_pack2<T>(v[6], v[7]));
  }
}

// The sum of a value over the W warps of a group; `red` has a slot per warp of the CTA.  Two calls in a row use different slots.
__device__ __forceinline__ float ln_warp_sum(float s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ float2 ln_warp_sum(float2 s) { return make_float2(ln_warp_sum(s.x), ln_warp_sum(s.y)); }
__device__ __forceinline__ void ln_add(float& s, float o) { s += o; }
__device__ __forceinline__ void ln_add(float2& s, float2 o) {
  s.x += o.x;
  s.y += o.y;
}
template <typename T>
__device__ __forceinline__ T ln_group_sum(T s, int W, int group, int warp, int lane, T* red) {
  s = ln_warp_sum(s);
  if (W > 1) {
    if (lane == 0) red[warp] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(W * 32) : "memory");
    s = red[group * W];
    for (int i = 1; i < W; ++i) ln_add(s, red[group * W + i]);
  }
  return s;
}

struct LnArgs {
  const void *x, *dy, *dres;
  const float *w, *b;
  float *mean, *rstd;
  void *y, *dx;
  float* part;                       // backward: [gridDim.x][2][d], or null: the rows' gradient alone
  int64_t ldx, lddy, ldres;
  int rows, d, W;
  int slot_x, slot_y, slot_r;        // bytes of a row's place in shared memory, per tensor (multiples of 16; 0: not there)
  float eps, inv_d;
  unsigned int* err;
};

constexpr int LN_RING = 2;

// A row's chunks of CH values among the lanes of a group: each warp takes a run of them, a lane every 32nd of the run, so that a lane's chunks lie at
// offsets that the compiler knows (with every (32 W)-th one 40 009 x 333 bf16 takes 21.4 instead of 17.6 us forward, 34.3 instead of 28.8 backward).
template <int CH>
struct LnPlace {
  int first, left;                   // column of the lane's chunk 0; chunk i is there while 32 i < left
  __device__ LnPlace(int d, int W, int warp, int lane) {
    const int chunks = (d + CH - 1) / CH, run = (chunks + W * 32 - 1) / (W * 32) * 32, at = warp * run + lane, end = (warp + 1) * run;
    first = at * CH;
    left = (end < chunks ? end : chunks) - at;
  }
  __device__ __forceinline__ bool has(int i) const { return 32 * i < left; }
};

// Row `row` of a [rows, d] tensor on its way to shared memory: the 16-byte units that hold it (they lie in the same allocation, whose
// granularity is coarser); values of the row start at byte (address & 15) of the copy.
template <typename T>
__device__ __forceinline__ uint32_t ln_row_bytes(const T* p, int d) { return (uint32_t)(((reinterpret_cast<uintptr_t>(p) & 15) + (size_t)d * sizeof(T) + 15) & ~(size_t)15); }
template <typename T>
__device__ __forceinline__ void ln_row_copy(uint8_t* dst, const T* p, int d, uint64_t* bar) {
  bulk_load_1d(dst, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15), ln_row_bytes(p, d), bar);
}
template <typename T>
__device__ __forceinline__ const T* ln_row_at(const uint8_t* slot, const T* p) { return reinterpret_cast<const T*>(slot + (reinterpret_cast<uintptr_t>(p) & 15)); }

// Behind a wait that ran out: time for the copies in flight, before the shared memory may be another CTA's.
__device__ __forceinline__ void ln_drain(bool ok) {
  if (!ok)
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
}

template <typename TI, typename TO, int CH, int NC>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_fwd_kernel(const __grid_constant__ LnArgs a) {
  extern __shared__ __align__(128) uint8_t ln_smem[];
  __shared__ float red[2][LN_WARPS];
  __shared__ uint64_t bars[LN_WARPS][LN_RING];
  __shared__ volatile uint32_t abort_flag;
  const int lane = threadIdx.x & 31, warp = warp_index();
  const int group = warp / a.W, groups = LN_WARPS / a.W, t = (warp - group * a.W) * 32 + lane;
  const LnPlace<CH> at(a.d, a.W, warp - group * a.W, lane);
  if (threadIdx.x == 0) {
    for (int i = 0; i < LN_WARPS; ++i)
      for (int k = 0; k < LN_RING; ++k) mbar_init(&bars[i][k], 1);
    abort_flag = 0u;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  const WaitCtx ctx{&abort_flag, a.err};
  uint8_t* ring = ln_smem + (size_t)group * LN_RING * a.slot_x;
  const TI* const x0 = static_cast<const TI*>(a.x);
  const int64_t first = (int64_t)blockIdx.x * groups + group, stride = (int64_t)gridDim.x * groups;
  bool ok = true;                                                // a group whose wait ran out goes on, without asking for more: its warps meet at barriers
  auto request = [&](int64_t row, int slot) {                    // one lane of the group
    if (t == 0 && row < a.rows && ok) {
      const TI* p = x0 + row * a.ldx;
      mbar_expect_tx(&bars[group][slot], ln_row_bytes(p, a.d));
      ln_row_copy(ring + slot * a.slot_x, p, a.d, &bars[group][slot]);
    }
  };
  request(first, 0);
  float w[NC][CH], b[NC][CH];                                    // read once: per row they are twice the bytes of the row
#pragma unroll
  for (int i = 0; i < NC; ++i) {
#pragma unroll
    for (int j = 0; j < CH; ++j) w[i][j] = b[i][j] = 0.f;
    if (at.has(i)) {
      ln_load<CH>(a.w + at.first + 32 * CH * i, w[i]);
      if (a.b) ln_load<CH>(a.b + at.first + 32 * CH * i, b[i]);
    }
  }
  int k = 0;
  for (int64_t row = first; row < a.rows; row += stride, ++k) {
    const int slot = k % LN_RING;
    if (a.W == 1) request(row + stride, (k + 1) % LN_RING);      // (a group of several warps asks behind the barrier of its sums)
    ok = mbar_wait_warp(&bars[group][slot], (k / LN_RING) & 1, ctx, 80) && ok;
    const TI* x = ln_row_at(ring + slot * a.slot_x, x0 + row * a.ldx) + at.first;
    float v[NC][CH];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (at.has(i)) {
        ln_load<CH>(x + 32 * CH * i, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) v[i][j] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < CH; ++j) s += v[i][j];
    const float mean = ln_group_sum(s, a.W, group, warp, lane, red[0]) * a.inv_d;
    if (a.W > 1) request(row + stride, (k + 1) % LN_RING);       // every warp is through with the row before
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (at.has(i)) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          v[i][j] -= mean;
          s = fmaf(v[i][j], v[i][j], s);
        }
      }
    }
    const float rstd = rsqrtf(ln_group_sum(s, a.W, group, warp, lane, red[1]) * a.inv_d + a.eps);
    TO* y = static_cast<TO*>(a.y) + row * a.d + at.first;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (at.has(i)) {
#pragma unroll
        for (int j = 0; j < CH; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[i][j], b[i][j]);
        ln_store<CH>(y + 32 * CH * i, v[i]);
      }
    }
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    __syncwarp();                                                // the slot's values have been read by all lanes
  }
  ln_drain(ok);
}

template <typename TI, typename TO, int CH, int NC>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_bwd_kernel(const __grid_constant__ LnArgs a) {
  extern __shared__ __align__(128) uint8_t ln_smem[];
  __shared__ float2 red[2][LN_WARPS];
  __shared__ uint64_t bars[LN_WARPS][LN_RING];
  __shared__ volatile uint32_t abort_flag;
  const int lane = threadIdx.x & 31, warp = warp_index();
  const int group = warp / a.W, groups = LN_WARPS / a.W, t = (warp - group * a.W) * 32 + lane;
  const LnPlace<CH> at(a.d, a.W, warp - group * a.W, lane);
  if (threadIdx.x == 0) {
    for (int i = 0; i < LN_WARPS; ++i)
      for (int k = 0; k < LN_RING; ++k) mbar_init(&bars[i][k], 1);
    abort_flag = 0u;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  const WaitCtx ctx{&abort_flag, a.err};
  const int slot_bytes = a.slot_x + a.slot_y + a.slot_r;
  uint8_t* ring = ln_smem + (size_t)group * LN_RING * slot_bytes;
  const TI *const x0 = static_cast<const TI*>(a.x), *const r0 = static_cast<const TI*>(a.dres);
  const TO* const y0 = static_cast<const TO*>(a.dy);
  const int64_t first = (int64_t)blockIdx.x * groups + group, stride = (int64_t)gridDim.x * groups;
  bool ok = true;                                                // a group whose wait ran out goes on, without asking for more: its warps meet at barriers
  auto request = [&](int64_t row, int slot) {                    // one lane of the group
    if (t == 0 && row < a.rows && ok) {
      const TI* p = x0 + row * a.ldx;
      const TO* q = y0 + row * a.lddy;
      uint64_t* bar = &bars[group][slot];
      uint8_t* to = ring + slot * slot_bytes;
      mbar_expect_tx(bar, ln_row_bytes(p, a.d) + ln_row_bytes(q, a.d) + (r0 ? ln_row_bytes(r0 + row * a.ldres, a.d) : 0));
      ln_row_copy(to, p, a.d, bar);
      ln_row_copy(to + a.slot_x, q, a.d, bar);
      if (r0) ln_row_copy(to + a.slot_x + a.slot_y, r0 + row * a.ldres, a.d, bar);
    }
  };
  request(first, 0);
  float w[NC][CH], aw[NC][CH], ab[NC][CH];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (at.has(i)) {
      ln_load<CH>(a.w + at.first + 32 * CH * i, w[i]);
    } else {
#pragma unroll
      for (int j = 0; j < CH; ++j) w[i][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) aw[i][j] = ab[i][j] = 0.f;
  }
  int k = 0;
  float mean = first < a.rows ? a.mean[first] : 0.f, rstd = first < a.rows ? a.rstd[first] : 0.f;
  for (int64_t row = first; row < a.rows; row += stride, ++k) {
    const int slot = k % LN_RING;
    if (a.W == 1) request(row + stride, (k + 1) % LN_RING);
    const bool more = row + stride < a.rows;
    const float next_mean = more ? a.mean[row + stride] : 0.f, next_rstd = more ? a.rstd[row + stride] : 0.f;
    ok = mbar_wait_warp(&bars[group][slot], (k / LN_RING) & 1, ctx, 81) && ok;
    const uint8_t* from = ring + slot * slot_bytes;
    const TI* x = ln_row_at(from, x0 + row * a.ldx) + at.first;
    const TO* dy = ln_row_at(from + a.slot_x, y0 + row * a.lddy) + at.first;
    float xh[NC][CH], g[NC][CH];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (at.has(i)) {
        ln_load<CH>(x + 32 * CH * i, xh[i]);
        ln_load<CH>(dy + 32 * CH * i, g[i]);
      } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          xh[i][j] = mean;
          g[i][j] = 0.f;
        }
      }
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        xh[i][j] = (xh[i][j] - mean) * rstd;
        aw[i][j] = fmaf(g[i][j], xh[i][j], aw[i][j]);
        ab[i][j] += g[i][j];
        g[i][j] *= w[i][j];
        s.x += g[i][j];
        s.y = fmaf(g[i][j], xh[i][j], s.y);
      }
    s = ln_group_sum(s, a.W, group, warp, lane, red[k & 1]);
    if (a.W > 1) request(row + stride, (k + 1) % LN_RING);       // every warp is through with the row before
    const float m1 = s.x * a.inv_d, m2 = s.y * a.inv_d;
    TI* dx = static_cast<TI*>(a.dx) + row * a.d + at.first;
    const TI* dres = r0 ? ln_row_at(from + a.slot_x + a.slot_y, r0 + row * a.ldres) + at.first : nullptr;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (at.has(i)) {
        float r[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) r[j] = 0.f;
        if (dres) ln_load<CH>(dres + 32 * CH * i, r);
#pragma unroll
        for (int j = 0; j < CH; ++j) r[j] = fmaf(rstd, g[i][j] - m1 - xh[i][j] * m2, r[j]);
        ln_store<CH>(dx + 32 * CH * i, r);
      }
    }
    mean = next_mean;
    rstd = next_rstd;
    __syncwarp();                                                // the slot's values have been read by all lanes
  }
  // the groups of this CTA, in their order, where the ring was; then the CTA's line of the partial sums
  ln_drain(ok);
  __syncthreads();
  if (abort_flag || !a.part) return;
  float* colsum = reinterpret_cast<float*>(ln_smem);             // [2][d], where a CTA has more than one group
  float* part = a.part + (size_t)blockIdx.x * 2 * a.d;
  for (int g = 0; g < groups; ++g) {
    if (group == g) {
      float* to = g == groups - 1 ? part : colsum;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = at.first + 32 * CH * i;
        if (at.has(i)) {
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            to[c + j] = g ? colsum[c + j] + aw[i][j] : aw[i][j];
            to[a.d + c + j] = g ? colsum[a.d + c + j] + ab[i][j] : ab[i][j];
          }
        }
      }
    }
    if (groups > 1) __syncthreads();
  }
}

// dw, db = the sum of `n` lines [2][d]: 32 columns per CTA, 32 threads per column
__global__ void __launch_bounds__(1024) layer_norm_cols_kernel(const float* part, int n, int d, float* dw, float* db) {
  __shared__ float sm[32][33];
  pdl_wait();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < 2 * (int64_t)d) {
#pragma unroll 8
    for (int i = ty; i < n; i += 32) s += part[(size_t)i * 2 * d + c];
  }
  sm[ty][tx] = s;
  __syncthreads();
  s = sm[tx][ty];                                                // a warp per column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t col = (int64_t)blockIdx.x * 32 + ty;
  if (tx == 0 && col < 2 * (int64_t)d) {
    if (col < d) dw[col] = s;
    else if (db) db[col - d] = s;
  }
}

// Warps per row: at most 32 values per thread; in the backward pass, which keeps four arrays of them, 16 where eight warps are enough for that
// (22 470 x 1024: one warp per row 72 us)
static int ln_warps(int d, bool bwd) {
  if (bwd) return d <= 512 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : 8;
  return d <= 1024 ? 1 : d <= 2048 ? 2 : d <= 4096 ? 4 : 8;
}

// CTAs: as many as the device holds at once with this much shared memory each, or as there are rows for
constexpr int LN_SMEM_SM = 222 * 1024, LN_MAX_PER_SM = 4;       // shared memory of an SM less what the CTAs take beside their rings; registers allow no more
static int ln_slot(int64_t d, int64_t size) { return (int)((d * size + 15 + 15) & ~15ll); }      // wherever the row starts in its first 16 bytes
static size_t ln_smem_bytes(int d, int slot_bytes, bool cols) {
  const int groups = LN_WARPS / ln_warps(d, cols);
  const size_t ring = (size_t)groups * LN_RING * slot_bytes, sums = cols && groups > 1 ? (size_t)2 * d * 4 : 0;
  return ring > sums ? ring : sums;
}
static int ln_grid(int64_t rows, int W, size_t smem, int regs, int* grid) {
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != KF_OK) return rc;
  const int groups = LN_WARPS / W;
  int per_sm = (int)(LN_SMEM_SM / (smem + 2048));
  if (regs > 0 && per_sm > 65536 / (regs * LN_THREADS)) per_sm = 65536 / (regs * LN_THREADS);
  per_sm = per_sm < 1 ? 1 : per_sm > LN_MAX_PER_SM ? LN_MAX_PER_SM : per_sm;
  const int64_t blocks = (rows + groups - 1) / groups, most = (int64_t)sms * per_sm;
  *grid = (int)(blocks < most ? blocks : most);
  return KF_OK;
}

// ws_bytes: room for the lines of the partial sums (backward; -1: none are made); *grid: the CTAs that were launched
template <void (*kern)(const LnArgs)>
static int ln_launch(const char* what, int64_t rows, size_t smem, cudaStream_t st, const LnArgs& a, int64_t ws_bytes, int* grid) {
  static PerDevice<int> kept;                                     // registers per thread of this instantiation
  int dev = 0;
  cudaGetDevice(&dev);
  int regs = kept.get(dev);
  if (!regs) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, kern);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (e != cudaSuccess) return cuda_status(e, "attributes of layer_norm");
    kept.put(dev, regs = attr.numRegs);
  }
  const int rc = ln_grid(rows, a.W, smem, regs, grid);
  if (rc != KF_OK) return rc;
  KF_REQUIRE(ws_bytes < 0 || ws_bytes >= (int64_t)*grid * 2 * a.d * 4, "kf_layer_norm_bwd: workspace of %lld bytes, needs %lld", (long long)ws_bytes, (long long)*grid * 2 * a.d * 4);
  // a dependent launch at any number of rows (the 1): it starts none early itself, so that only the gap between kernels closes (22 470 x 1024 both directions
  // 84.0 -> 79.4 us, 40 009 x 333 51.4 -> 48.1)
  return cuda_status(launch_maybe_pdl(1, kern, dim3(*grid), dim3(LN_THREADS), smem, st, a), what);
}

// f(TI, TO, CH, NC) for the types, the access width and the values per thread of a call
template <typename TI, typename TO, typename F>
static int ln_by_width(bool wide, int d, int W, F&& f) {
  const int lanes = W * 32;
  if (wide) {
    const int n = (d / 8 + lanes - 1) / lanes;
    if (n <= 1) return f(TI{}, TO{}, std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (n <= 2) return f(TI{}, TO{}, std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    if (n <= 3) return f(TI{}, TO{}, std::integral_constant<int, 8>{}, std::integral_constant<int, 3>{});
    return f(TI{}, TO{}, std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
  }
  // Steps of values per lane: every one is unrolled and its registers are there, so that with 32 behind 12 widths of 13 to 16 values took up to twice the time (26 MB of
  // bf16 rows, forward / backward: width 501 27.1 / 45.7, with a step of 16 17.1 / 28.5 us; 1001 17.2 / 43.0, now 17.2 / 24.7; 1201, with one of 24, 25.2 / 27.8, now 16.8 / 27.8)
  const int n = (d + lanes - 1) / lanes;
  if (n <= 4) return f(TI{}, TO{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  if (n <= 12) return f(TI{}, TO{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 12>{});
  if (n <= 16) return f(TI{}, TO{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  if (n <= 24) return f(TI{}, TO{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 24>{});
  return f(TI{}, TO{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
}
template <typename TI, typename F>
static int ln_by_out(int out_dtype, bool wide, int d, int W, F&& f) {
  if (out_dtype == KF_F32) return ln_by_width<TI, float>(wide, d, W, f);
  if (out_dtype == KF_BF16) return ln_by_width<TI, __nv_bfloat16>(wide, d, W, f);
  return ln_by_width<TI, __half>(wide, d, W, f);
}
template <typename F>
static int ln_by_type(int in_dtype, int out_dtype, bool wide, int d, int W, F&& f) {
  if (in_dtype == KF_F32) return ln_by_out<float>(out_dtype, wide, d, W, f);
  if (in_dtype == KF_BF16) return ln_by_out<__nv_bfloat16>(out_dtype, wide, d, W, f);
  return ln_by_out<__half>(out_dtype, wide, d, W, f);
}

static bool ln_aligned(const void* p, int64_t pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) & 15) == 0; }
static int64_t ln_size(int dtype) { return dtype == KF_F32 ? 4 : 2; }
static bool ln_float_type(int dtype) { return dtype == KF_F32 || dtype == KF_BF16 || dtype == KF_F16; }

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_layer_norm_ws_bytes(int64_t rows, int d) {
  if (rows < 0 || d <= 0 || d > LN_MAX_WIDTH) {
    set_error("kf_layer_norm_ws_bytes: bad argument rows=%lld d=%d", (long long)rows, d);
    return KF_ERR_BAD_ARGUMENT;
  }
  int grid = 0;
  const int rc = ln_grid(rows, ln_warps(d, true), 0, 0, &grid);                  // no launch makes more lines
  if (rc != KF_OK) return rc > 0 ? KF_ERR_UNSUPPORTED : rc;
  return (int64_t)grid * 2 * d * 4;
}

extern "C" int kf_layer_norm_fwd(int in_dtype, const void* x, int64_t ldx, const float* w, const float* b, float eps, int rows, int d, int out_dtype, void* y,
                                 float* mean, float* rstd, void* stream) {
  KF_REQUIRE(ln_float_type(in_dtype) && ln_float_type(out_dtype), "kf_layer_norm_fwd: types must be f32, bf16 or f16");
  KF_REQUIRE(rows >= 0 && d > 0 && d <= LN_MAX_WIDTH && ldx >= 0, "kf_layer_norm_fwd: bad shape rows=%d d=%d (at most %d wide)", rows, d, LN_MAX_WIDTH);
  if (rows == 0) return KF_OK;
  KF_REQUIRE(x && w && y && mean && rstd, "kf_layer_norm_fwd: null pointer");
  LnArgs a{};
  a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.mean = mean; a.rstd = rstd; a.y = y; a.rows = rows; a.d = d; a.W = ln_warps(d, false); a.eps = eps; a.inv_d = 1.0f / (float)d;
  a.slot_x = ln_slot(d, ln_size(in_dtype));
  a.err = dev_error_ptr();
  KF_REQUIRE(a.err != nullptr, "kf_layer_norm_fwd: device error word unavailable");
  const bool wide = d % 8 == 0 && ln_aligned(x, ldx * ln_size(in_dtype)) && ln_aligned(y, 0) && ln_aligned(w, 0) && ln_aligned(b, 0);
  const size_t smem = ln_smem_bytes(d, a.slot_x, false);
  int grid = 0;
  return ln_by_type(in_dtype, out_dtype, wide, d, a.W, [&](auto ti, auto to, auto ch, auto nc) {
    return ln_launch<layer_norm_fwd_kernel<decltype(ti), decltype(to), decltype(ch)::value, decltype(nc)::value>>("kf_layer_norm_fwd launch", rows, smem,
                     static_cast<cudaStream_t>(stream), a, -1, &grid);
  });
}

extern "C" int kf_layer_norm_bwd(int in_dtype, const void* x, int64_t ldx, int dy_dtype, const void* dy, int64_t lddy, const float* w, const float* mean,
                                 const float* rstd, const void* dres, int64_t ldres, int rows, int d, void* dx, float* dw, float* db, void* ws, int64_t ws_bytes,
                                 void* stream) {
  KF_REQUIRE(ln_float_type(in_dtype) && ln_float_type(dy_dtype), "kf_layer_norm_bwd: types must be f32, bf16 or f16");
  KF_REQUIRE(rows >= 0 && d > 0 && d <= LN_MAX_WIDTH && ldx >= 0 && lddy >= 0 && ldres >= 0, "kf_layer_norm_bwd: bad shape rows=%d d=%d (at most %d wide)", rows, d,
             LN_MAX_WIDTH);
  KF_REQUIRE(w && (dw || !db), "kf_layer_norm_bwd: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    cudaError_t e = dw ? cudaMemsetAsync(dw, 0, (size_t)d * 4, st) : cudaSuccess;
    if (e == cudaSuccess && db) e = cudaMemsetAsync(db, 0, (size_t)d * 4, st);
    return cuda_status(e, "kf_layer_norm_bwd memset");
  }
  KF_REQUIRE(x && dy && mean && rstd && dx && (ws || !dw), "kf_layer_norm_bwd: null pointer");
  LnArgs a{};
  a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.dres = dres; a.ldres = ldres; a.w = w; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.part = dw ? static_cast<float*>(ws) : nullptr; a.rows = rows; a.d = d; a.W = ln_warps(d, true); a.inv_d = 1.0f / (float)d;
  a.slot_x = ln_slot(d, ln_size(in_dtype));
  a.slot_y = ln_slot(d, ln_size(dy_dtype));
  a.slot_r = dres ? a.slot_x : 0;
  a.err = dev_error_ptr();
  KF_REQUIRE(a.err != nullptr, "kf_layer_norm_bwd: device error word unavailable");
  const size_t smem = ln_smem_bytes(d, a.slot_x + a.slot_y + a.slot_r, true);
  int grid = 0;
  const bool wide = d % 8 == 0 && ln_aligned(x, ldx * ln_size(in_dtype)) && ln_aligned(dy, lddy * ln_size(dy_dtype)) && ln_aligned(dres, ldres * ln_size(in_dtype)) &&
                    ln_aligned(dx, 0) && ln_aligned(w, 0);
  const int rc = ln_by_type(in_dtype, dy_dtype, wide, d, a.W, [&](auto ti, auto to, auto ch, auto nc) {
    return ln_launch<layer_norm_bwd_kernel<decltype(ti), decltype(to), decltype(ch)::value, decltype(nc)::value>>("kf_layer_norm_bwd launch", rows, smem, st, a, dw ? ws_bytes : -1, &grid);
  });
  if (rc != KF_OK || !dw) return rc;
  return cuda_status(launch_maybe_pdl(1, layer_norm_cols_kernel, dim3((2 * d + 31) / 32), dim3(1024), 0, st, static_cast<const float*>(ws), grid, d, dw, db),
                     "kf_layer_norm_bwd column sums launch");
}
