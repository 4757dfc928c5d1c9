// What the attention kernels share: exponentials on two pipes, packing to 16 bits, the records of a packed batch and the tensor maps
// over [token, head, 64] tensors.
#pragma once
#include "kf_sm100.cuh"

namespace kf {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^t for a pair without the special-function unit: t = n + f with n = round(t) taken from the low mantissa bits of
// t + 1.5 * 2^23 and f in [-0.5, 0.5]; 2^f by a cubic (minimax for the relative error on that interval: 7.6e-5, far
// below the rounding of the 16-bit P it feeds); n goes into the exponent field by an integer add.  t is clamped at -126
// (the result is then 2^-126 instead of 0: it vanishes in the 16-bit P and in the row sum alike) and at 127, behind which the add
// would wrap to anything, a small or a negative number too: a row with such an element has a sum that no limit lets pass.  A t that
// is no number passes the clamps and the add makes a huge element of it, with the same effect (a clamp that drops it would drop the key).  All of it runs on the
// FMA and integer pipes, as packed pairs where the operation exists.
// Clamps and no check of the largest t: that costs an instruction less, but a register through the key loop (captured, us: B 14, H 12, N 1605, MXFP8 out
// 137.5 against 135.3; B 1, H 16, N 1605 22.2 against 21.9).
__device__ __forceinline__ float clamp_ex2(float t) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;\n\tmin.NaN.f32 %0, %0, 0f42FE0000;" : "+f"(t));   // [-126, 127]
  return t;
}
__device__ __forceinline__ float2 ex2_poly2(float2 t) {
  t.x = clamp_ex2(t.x);
  t.y = clamp_ex2(t.y);
  const float2 r = add2(t, splat2(12582912.f));
  const float2 n = add2(r, splat2(-12582912.f));
  const float2 f = fma2(n, splat2(-1.f), t);
  float2 p = fma2(f, splat2(0x1.c43e56p-5f), splat2(0x1.f0df98p-3f));
  p = fma2(p, f, splat2(0x1.62f24ap-1f));
  p = fma2(p, f, splat2(0x1.fff686p-1f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int f16) {
  if (f16) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// The same with a quartic: where the sums of the exponentials are an output of their own (the log-sum-exp), one more FMA per pair.  Its constant is 1 (minimax
// for the others: 2.9e-6, 2.7e-6 with a free one) and t is clamped at -127: there f = 0, the polynomial is 1 and the add makes an exact 0 of it, so that a masked
// key, -inf, weighs nothing, not 2^-126, which a value of 10^38 would show in a bf16 output.  Between -127 and -126 the add leaves a denormal number.
__device__ __forceinline__ float2 ex2_poly2_fine(float2 t) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n\tmin.NaN.f32 %0, %0, 0f42FE0000;" : "+f"(t.x));   // [-127, 127]
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n\tmin.NaN.f32 %0, %0, 0f42FE0000;" : "+f"(t.y));
  const float2 r = add2(t, splat2(12582912.f));
  const float2 n = add2(r, splat2(-12582912.f));
  const float2 f = fma2(n, splat2(-1.f), t);
  float2 p = fma2(f, splat2(0x1.3a02b6p-7f), splat2(0x1.c9fc74p-5f));
  p = fma2(p, f, splat2(0x1.ec0378p-3f));
  p = fma2(p, f, splat2(0x1.62e12cp-1f));
  p = fma2(p, f, splat2(1.f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}

// A quartic (2.7e-6) for t that stays below 127: one clamp at -126, and the power of two goes in by a multiplication, which keeps what is no number.
__device__ __forceinline__ float2 ex2_poly2_neg(float2 t) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;\n\tmax.NaN.f32 %1, %1, 0fC2FC0000;" : "+f"(t.x), "+f"(t.y));
  const float2 r = add2(t, splat2(12582912.f));
  const float2 n = add2(r, splat2(-12582912.f));
  const float2 f = fma2(n, splat2(-1.f), t);
  float2 p = fma2(f, splat2(0x1.3997d4p-7f), splat2(0x1.ca1440p-5f));
  p = fma2(p, f, splat2(0x1.ec06dap-3f));
  p = fma2(p, f, splat2(0x1.62e0dcp-1f));
  p = fma2(p, f, splat2(0x1.ffffe8p-1f));
  return mul2(p, make_float2(__int_as_float((__float_as_int(r.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(r.y) << 23) + 0x3f800000)));
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Capped scores in units of the exponent, cap * tanh(x * scale / cap) * log2(e) of raw products x.  Anywhere: tanh(y) = 1 - 2 / (1 + e^2y), two
// operations of the special-function unit, absolute error ~1e-7 (tanh.approx would leave 2^-11, which the cap scales).  Where every score of a
// piece lies within half the cap, which is what a cap leaves alone: x times a polynomial in x^2 (minimax for the relative error of
// tanh(y) / y, |y| <= 0.5: 2.8e-8), six packed operations per pair.
struct Cap {
  float in, out;            // 2 * scale * log2(e) / cap, cap * log2(e)
  float flat;               // raw products up to here in size take the polynomial
  float inv_out;
  float c[5];               // with scale and log2(e) in them
  __host__ void set(float scale, float cap) {
    constexpr double LOG2E = 1.4426950408889634;
    const double a[5] = {0x1.0000000000000p+0, -0x1.5554a4p-2, 0x1.10e438p-3, -0x1.b20fdap-5, 0x1.18bd6ep-6}, r = (double)scale / cap;
    in = (float)(2 * r * LOG2E);
    out = (float)(cap * LOG2E);
    inv_out = 1.f / out;
    flat = (float)(0.5 / r < 1e18 ? 0.5 / r : 1e18);
    double m = scale * LOG2E;
    for (int i = 0; i < 5; ++i, m *= r * r) c[i] = (float)(a[i] * m);
    if (!(m < 1e30)) flat = -1.f;                               // a cap so small that the polynomial has no range
  }
};
__device__ __forceinline__ float2 cap_flat(const Cap& k, float2 x) {
  const float2 t = mul2(x, x);
  float2 p = fma2(t, splat2(k.c[4]), splat2(k.c[3]));
  p = fma2(p, t, splat2(k.c[2]));
  p = fma2(p, t, splat2(k.c[1]));
  p = fma2(p, t, splat2(k.c[0]));
  return mul2(x, p);
}

__device__ __forceinline__ float2 cap_any(const Cap& k, float2 x) {
  const float2 r = make_float2(rcp_approx(1.f + ex2(x.x * k.in)), rcp_approx(1.f + ex2(x.y * k.in)));
  return fma2(r, splat2(-2.f * k.out), splat2(k.out));
}
// The same with its derivative, 1 - tanh^2(y) = 4 e / (1 + e)^2 with e = e^-2|y|: formed from e it keeps its digits where tanh is 1 but for a few (1 - tanh * tanh was
// off by 1e-7, a quarter of the value at y = 8).
__device__ __forceinline__ float2 cap_any(const Cap& k, float2 x, float2& d) {
  const float2 t = mul2(x, splat2(k.in)), e = make_float2(ex2(-fabsf(t.x)), ex2(-fabsf(t.y))), u = add2(e, splat2(1.f));
  const float2 r = make_float2(rcp_approx(u.x), rcp_approx(u.y)), f = mul2(e, mul2(r, splat2(4.f)));
  const float2 s = fma2(f, splat2(-0.5f * k.out), splat2(k.out));
  d = mul2(f, r);
  return make_float2(copysignf(s.x, x.x), copysignf(s.y, x.y));
}

// ------------------------------------------------------------------------------------------------ packed batches
// One 128-row tile of queries of one sequence (a record of eight 32-bit words, built by the host; see kf_attn_pack_params).  Query r of the
// tile is at position pos + r of its keys and sees keys [0, limit(r)): all of them (prefix = k_len), or those up to itself and the prefix.
struct QTile {
  int row, rows;        // first query row of the batch, rows of the tile (1 .. 128)
  int k_row, k_len;     // the sequence's keys
  int pos, prefix;
  int slot;             // place of the tile in the order of the rows
  int pad;
  __device__ __forceinline__ int limit(int r) const {
    const int upto = pos + r + 1;
    const int l = upto > prefix ? upto : prefix;
    return l < 0 ? 0 : l < k_len ? l : k_len;
  }
};
// One 128-row tile of keys.  Key r of the tile is key first + r of its sequence and is seen by queries [lowest(r), q_len).
struct KTile {
  int row, rows;
  int q_row, q_len;     // the sequence's queries
  int first, off;       // index of the tile's first key; position of query 0
  int prefix;
  int slot0;            // slot of the sequence's first query tile
  __device__ __forceinline__ int lowest(int r) const {
    const int j = first + r, i = j - off;
    return j < prefix || i < 0 ? 0 : i;
  }
};
template <typename T>
__device__ __forceinline__ T load_tile(const int4* tiles, int index) {       // the same address in every lane
  static_assert(sizeof(T) == 32, "two 16-byte words");
  const int4 a = __ldg(tiles + 2 * (size_t)index), b = __ldg(tiles + 2 * (size_t)index + 1);
  T t;
  int* w = reinterpret_cast<int*>(&t);
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  return t;
}

// Items 0 .. n - 1, the longest first, among the CTAs of the grid: every other round in the opposite order, so that whoever got the longest of a
// round gets the shortest of the next.
__device__ __forceinline__ int items_of_cta(int n) {
  const int g = (int)gridDim.x, rounds = n / g, rest = n - rounds * g;
  const int place = rounds & 1 ? g - 1 - (int)blockIdx.x : (int)blockIdx.x;
  return rounds + (place < rest);
}
__device__ __forceinline__ int item_of_cta(int it) {
  return it * (int)gridDim.x + (it & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)), "l"(map),
               "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// Rows [from, to) of a tile of 128-byte rows become zero (whole warp): rows that a copy brought from behind the end of a sequence.  They meet
// coefficients that are zero, but 0 * NaN is NaN.  The 128-byte swizzle moves bytes inside a row only.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to, int lane) {
  for (int o = from * 128 + lane * 16; o < to * 128; o += 512) *reinterpret_cast<uint4*>(tile + o) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
}

// 3-D tensor map over [rows, heads, 64] of 16-bit elements with the given strides (elements), box (64, 1, box_rows), 128-byte swizzle; rows
// past the end read as zero.
int make_tmap_heads(CUtensorMap* map, const void* base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride, int box_rows);
int check_heads(const char* what, const kf_heads& t, int64_t rows, int heads, kf_heads* out);
int check_pack(const kf_attn_pack_params* p);

}  // namespace kf
