// Gradients of the attention over packed sequences (kf_attn_pack.cu), head dimension 64, on the sm_100a tensor cores.
//
//   P = exp(s - lse);  dV = P^T dO;  dP = dO V^T;  delta = rowsum(dO * O);  dS = P * (dP - delta) * ds/d(scale q.k);
//   dQ = scale * dS K;  dK = scale * dS^T Q        (ds/d(scale q.k) is 1, or 1 - tanh^2 with a cap)
//
// Two launches of one kernel, which share the mathematics and differ in what stays and what passes by:
//   ROWS = queries  a CTA keeps 128 queries (Q, dO) and goes through key tiles (K, V):        dQ
//   ROWS = keys     a CTA keeps 128 keys (K, V) and goes through query tiles (Q, dO) of every head that shares them:   dK, dV
// S and dP are computed in both (7 products where one pass over the pairs takes 5): each gradient is then summed in one place, in tensor
// memory, in a fixed order.  One pass would add dQ from every key tile to memory by atomics, 32 KB per pair of tiles, in an order that changes
// from run to run.
//
//   CTA      one per SM, persistent over (tile, head) items, the longest first; steps of 128 passing rows
//   roles    warps 0..7: a thread takes 64 of the 128 columns of one row: S and dP from tensor memory, P and dS in registers, as 16-bit pairs
//            back over S; warp 8: TMA (row operands in two buffers, passing operands in a ring of four); warp 9: products; warps 10, 11
//            (ROWS = queries): log-sum-exp and delta of the rows of the next item, also for the second launch
//   pipeline two S buffers, one dP buffer, the accumulators: S(G + 1) is issued before the end of step G, dP(G + 1) when dP(G) has been read,
//            the gradients' products of step G behind them
//   ROWS = keys takes the log-sum-exp and delta of its passing rows from a table with a line of 128 per query tile, +inf where there is no row:
//            P is 0 there
//   numerics P and dS are rounded to the 16-bit type of the operands (the products' A operand); everything else fp32
#include "kf_attn.cuh"

namespace kf {

constexpr int PB_T = 128, PB_D = 64;
constexpr int PB_THREADS = 384;
constexpr int PB_REGS_WORK = 208, PB_REGS_LEAN = 88;           // 256 * 208 + 128 * 88 = 384 * 168, the allocation at launch
constexpr int PB_REGS_LAUNCH = 168;
static_assert(256 * PB_REGS_WORK + 128 * PB_REGS_LEAN <= PB_THREADS * PB_REGS_LAUNCH, "register split");
constexpr int PB_RING = 4;
constexpr int PB_TILE = PB_T * PB_D * 2;                       // 16 KB
constexpr int PB_OFF_C = 4 * PB_TILE;                          // row operands: two buffers of two tiles; then the ring: two tiles per stage
constexpr int PB_OFF_STAT = PB_OFF_C + PB_RING * 2 * PB_TILE;  // per ring stage (ROWS = keys) or item buffer: lse2[128], delta[128]
constexpr int PB_OFF_BAR = PB_OFF_STAT + PB_RING * 1024;
constexpr size_t PB_SMEM = (size_t)PB_OFF_BAR + 512;
constexpr int PB_COL_S = 0, PB_COL_DP = 256, PB_COL_A1 = 384, PB_COL_A2 = 448, PB_TMEM_COLS = 512;

struct PackBwdArgs {
  const int4* tiles;
  int n_items, heads, share;     // heads of an item: query heads (ROWS = queries) or key heads
  float scale, scale_log2, cap_in, cap_out;
  const float* slopes;
  float* stats;                  // [Hq][n_q_tiles][2][128]
  int n_q_tiles;
  // ROWS = queries
  const void *O, *dO;
  int64_t o_st, o_sh, do_st, do_sh;
  const float* lse;
  int64_t lse_ld;
  // outputs: dQ, or dK and dV
  void *g1, *g2;
  int64_t g1_st, g1_sh, g2_st, g2_sh;
  unsigned int* err;
};

template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// What an item is, the same for every role.
template <bool KEYS>
struct BwdItem;
template <>
struct BwdItem<false> {
  QTile t;
  int head, n;                                                  // steps
  __device__ __forceinline__ void load(const PackBwdArgs& a, int item) {
    t = load_tile<QTile>(a.tiles, item / a.heads);
    head = item % a.heads;
    n = (t.limit(t.rows - 1) + PB_T - 1) / PB_T;
  }
  __device__ __forceinline__ int rows() const { return t.rows; }
  __device__ __forceinline__ int row0() const { return t.row; }
  __device__ __forceinline__ int slot(int) const { return t.slot; }
};
template <>
struct BwdItem<true> {
  KTile t;
  int head, n, per, first;                                      // per: query tiles per query head, from tile `first` of the sequence on
  __device__ __forceinline__ void load(const PackBwdArgs& a, int item) {
    t = load_tile<KTile>(a.tiles, item / a.heads);
    head = item % a.heads;
    first = t.lowest(0) / PB_T;
    const int tiles = (t.q_len + PB_T - 1) / PB_T;
    per = tiles > first ? tiles - first : 0;
    n = per * a.share;
  }
  __device__ __forceinline__ int rows() const { return t.rows; }
  __device__ __forceinline__ int row0() const { return t.row; }
  __device__ __forceinline__ int slot(int tile) const { return t.slot0 + tile; }
};
// Where a step's passing tile lies: first row in the batch, head, index of its first row in the sequence, rows that belong to the sequence.
struct BwdStep {
  int row, head, index, valid, tile;
};
__device__ __forceinline__ BwdStep step_of(const PackBwdArgs& a, const BwdItem<false>& i, int j) {
  return {i.t.k_row + j * PB_T, i.head / a.share, j * PB_T, i.t.k_len - j * PB_T, 0};
}
__device__ __forceinline__ BwdStep step_of(const PackBwdArgs& a, const BwdItem<true>& i, int j) {
  const int hh = j / i.per, qt = i.first + j - hh * i.per;
  return {i.t.q_row + qt * PB_T, i.head * a.share + hh, qt * PB_T, i.t.q_len - qt * PB_T, qt};
}

template <int F16, bool KEYS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(PB_THREADS, 1)
attn_pack_bwd_kernel(const __grid_constant__ CUtensorMap tmR1, const __grid_constant__ CUtensorMap tmR2, const __grid_constant__ CUtensorMap tmC1,
                     const __grid_constant__ CUtensorMap tmC2, const __grid_constant__ PackBwdArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PB_OFF_BAR);
  uint64_t *r_full = bars, *r_empty = r_full + 2, *c1_full = r_empty + 2, *c2_full = c1_full + PB_RING, *c_empty = c2_full + PB_RING, *st_full = c_empty + PB_RING,
           *st_empty = st_full + PB_RING, *s_full = st_empty + 2, *ds_full = s_full + 2, *dp_full = ds_full + 2, *dp_free = dp_full + 1, *acc_full = dp_free + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  pdl_launch_dependents();
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int n_my = (int)blockIdx.x < a.n_items ? (a.n_items - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&ds_full[i], 256);
      mbar_init(&st_empty[i], 256);
    }
    for (int i = 0; i < PB_RING; ++i) {
      mbar_init(&c1_full[i], 1);
      mbar_init(&c2_full[i], 1);
      mbar_init(&c_empty[i], 1);
      mbar_init(&st_full[i], KEYS ? 1 : 64);
    }
    mbar_init(dp_full, 1);
    mbar_init(dp_free, 256);
    mbar_init(acc_full, 1);
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_holder, PB_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = *tmem_holder;
  const WaitCtx ctx{abort_flag, a.err};
  const bool bad_align = (smem_u32(smem) & 1023u) != 0;
  if (bad_align && threadIdx.x == 0 && atomicCAS(&a.err[0], 0u, 99u) == 0u) {
    a.err[1] = 120;
    a.err[2] = blockIdx.x;
  }
  using Item = BwdItem<KEYS>;
  auto load_item = [&](Item& i, int it) { i.load(a, (int)blockIdx.x + it * (int)gridDim.x); };

  if (warp >= 8) {
  setmaxnreg_dec<PB_REGS_LEAN>();
  if (bad_align) {
    // nothing was issued; fall through to the teardown
  } else if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      prefetch_tmap(&tmR1);
      prefetch_tmap(&tmR2);
      prefetch_tmap(&tmC1);
      prefetch_tmap(&tmC2);
    }
    bool ok = !__any_sync(0xffffffffu, *static_cast<volatile unsigned int*>(a.err) != 0u);   // has an earlier launch failed?
    if (!ok) *abort_flag = 1u;
    uint32_t ri = 0, st = 0, ph = 1;
    for (int it = 0; it < n_my && ok; ++it) {
      Item I;
      load_item(I, it);
      if (I.n == 0) continue;
      const uint32_t rb = ri & 1;
      if (!mbar_wait_warp(&r_empty[rb], ((ri >> 1) & 1) ^ 1, ctx, 60)) break;
      if (elect_one()) {
        uint8_t* to = smem + rb * 2 * PB_TILE;
        mbar_expect_tx(&r_full[rb], 2 * PB_TILE);
        tma_load_3d(to, &tmR1, 0, I.head, I.row0(), &r_full[rb]);
        tma_load_3d(to + PB_TILE, &tmR2, 0, I.head, I.row0(), &r_full[rb]);
      }
      __syncwarp();
      ++ri;
      for (int j = 0; j < I.n; ++j) {
        const BwdStep s = step_of(a, I, j);
        if (!mbar_wait_warp(&c_empty[st], ph, ctx, 61)) { ok = false; break; }
        if (elect_one()) {
          uint8_t* to = smem + PB_OFF_C + st * 2 * PB_TILE;
          mbar_expect_tx(&c1_full[st], PB_TILE);
          tma_load_3d(to, &tmC1, 0, s.head, s.row, &c1_full[st]);
          if (KEYS) {
            mbar_expect_tx(&st_full[st], 1024);
            bulk_load_1d(smem + PB_OFF_STAT + st * 1024, a.stats + ((size_t)s.head * a.n_q_tiles + I.slot(s.tile)) * 256, 1024, &st_full[st]);
          }
          mbar_expect_tx(&c2_full[st], PB_TILE);
          tma_load_3d(to + PB_TILE, &tmC2, 0, s.head, s.row, &c2_full[st]);
        }
        __syncwarp();
        if (++st == PB_RING) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t fmt = F16 ? 0u : 1u;
    const uint32_t idesc_s = idesc_f16(fmt, PB_T), idesc_a = idesc_f16(fmt, PB_D) | (1u << 16);     // the passing operand of a gradient is MN-major
    const bool leader = elect_one();
    struct Cursor {
      Item i;
      int it, j;
      uint32_t ri;                                                            // items with steps so far
    };
    auto settle = [&](Cursor& c) {
      c.j = 0;
      for (; c.it < n_my; ++c.it) {
        load_item(c.i, c.it);
        if (c.i.n > 0) return;
      }
    };
    auto advance = [&](Cursor& c) {
      if (++c.j == c.i.n) {
        ++c.it;
        ++c.ri;
        settle(c);
      }
    };
    Cursor x;                                                                 // the next S and dP products
    x.it = 0;
    x.ri = 0;
    settle(x);
    uint32_t x_st = 0, x_ph = 0;                                              // their ring stage
    uint32_t G = 0;                                                           // steps whose S has been issued
    bool ok = true;
    auto product = [&](uint32_t t_d, uint32_t which) {                        // row operand `which` times the passing one, 128 x 128 x 64
      const uint64_t rdesc = smem_desc_sw128(smem_u32(smem + ((x.ri & 1) * 2 + which) * PB_TILE));
      const uint64_t cdesc = smem_desc_sw128(smem_u32(smem + PB_OFF_C + (x_st * 2 + which) * PB_TILE));
#pragma unroll
      for (int kk = 0; kk < PB_D / 16; ++kk) mma_f16(t_d, rdesc + 2 * kk, cdesc + 2 * kk, idesc_s, kk != 0);
    };
    auto issue_s = [&]() {
      ok = (x.j != 0 || mbar_wait_warp(&r_full[x.ri & 1], (x.ri >> 1) & 1, ctx, 62)) && mbar_wait_warp(&c1_full[x_st], x_ph, ctx, 63);
      if (!ok) return;
      const int valid = step_of(a, x.i, x.j).valid;
      if (valid < PB_T) zero_rows(smem + PB_OFF_C + x_st * 2 * PB_TILE, valid, PB_T, lane);
      tc_fence_after();
      if (leader) {
        product(tmem_base + PB_COL_S + (G & 1) * PB_T, 0);
        tc_commit(&s_full[G & 1]);
      }
      __syncwarp();
    };
    auto issue_dp = [&]() {                                                   // and on to the next step
      ok = mbar_wait_warp(&c2_full[x_st], x_ph, ctx, 64) && (G == 0 || mbar_wait_warp(dp_free, (G - 1) & 1, ctx, 65));
      if (!ok) return;
      const int valid = step_of(a, x.i, x.j).valid;
      if (valid < PB_T) zero_rows(smem + PB_OFF_C + (x_st * 2 + 1) * PB_TILE, valid, PB_T, lane);
      tc_fence_after();
      if (leader) {
        product(tmem_base + PB_COL_DP, 1);
        tc_commit(dp_full);
      }
      __syncwarp();
      ++G;
      if (++x_st == PB_RING) {
        x_st = 0;
        x_ph ^= 1;
      }
    };
    int a_j = 0, a_n = x.it < n_my ? x.i.n : 0;                               // the gradients' products: step and number of steps of their item
    uint32_t a_ri = 0, a_st = 0, A = 0;
    bool more = x.it < n_my;
    if (more) {
      issue_s();
      if (ok) issue_dp();
      if (ok) advance(x);
    }
    while (more && ok) {
      const bool next = x.it < n_my;
      const int n_next = x.j == 0 ? x.i.n : 0;                                // the item of step A + 1, where that is its first
      if (next) {
        issue_s();
        if (ok) issue_dp();
        if (!ok) break;
        advance(x);
      }
      if (!mbar_wait_warp(&ds_full[A & 1], (A >> 1) & 1, ctx, 66)) break;
      tc_fence_after();
      if (leader) {
        const uint32_t t_p = tmem_base + PB_COL_S + (A & 1) * PB_T;
        const uint64_t c1 = smem_desc_sw128(smem_u32(smem + PB_OFF_C + a_st * 2 * PB_TILE)), c2 = smem_desc_sw128(smem_u32(smem + PB_OFF_C + (a_st * 2 + 1) * PB_TILE));
#pragma unroll
        for (int kk = 0; kk < PB_T / 16; ++kk) {                              // 16 columns: 8 words of the half that their threads wrote
          const uint32_t p = t_p + (kk >> 2) * 64 + (kk & 3) * 8;
          if (KEYS) mma_f16_ta(tmem_base + PB_COL_A2, p, c2 + (uint64_t)(kk * (2048 >> 4)), idesc_a, (a_j | kk) != 0);
          mma_f16_ta(tmem_base + PB_COL_A1, p + 32, c1 + (uint64_t)(kk * (2048 >> 4)), idesc_a, (a_j | kk) != 0);
        }
        tc_commit(&c_empty[a_st]);
        if (a_j + 1 == a_n) {
          tc_commit(acc_full);
          tc_commit(&r_empty[a_ri & 1]);
        }
      }
      __syncwarp();
      ++A;
      if (++a_st == PB_RING) a_st = 0;
      if (++a_j == a_n) {
        a_j = 0;
        a_n = n_next;
        ++a_ri;
      }
      more = next;
    }
  } else if (!KEYS) {
    // ------------------------------------------------------------------ log-sum-exp and delta of the rows: two per thread
    bool ok = true;
    for (int it = 0; it < n_my && ok; ++it) {
      Item I;
      load_item(I, it);
      const int b = it & 1;
      ok = mbar_wait_warp(&st_empty[b], ((it >> 1) & 1) ^ 1, ctx, 67);
      if (!ok) break;
      float* sm = reinterpret_cast<float*>(smem + PB_OFF_STAT + b * 1024);
      float* gl = a.stats + ((size_t)I.head * a.n_q_tiles + I.slot(0)) * 256;
#pragma unroll 1
      for (int r = (warp - 10) * 32 + lane; r < PB_T; r += 64) {
        float lse2 = INFINITY, delta = 0.f;
        if (r < I.rows()) {
          const int64_t row = I.row0() + r;
          const float l = __ldg(a.lse + (int64_t)I.head * a.lse_ld + row);
          if (l != -INFINITY) lse2 = l * 1.4426950408889634f;
          const uint4* o = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.O) + 2 * (row * a.o_st + (int64_t)I.head * a.o_sh));
          const uint4* d = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.dO) + 2 * (row * a.do_st + (int64_t)I.head * a.do_sh));
          float2 s = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < PB_D / 8; ++i) {
            const uint4 u = __ldg(o + i), v = __ldg(d + i);
            const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) s = fma2(unpack16<F16>(uw[k]), unpack16<F16>(vw[k]), s);
          }
          delta = s.x + s.y;
        }
        sm[r] = lse2;
        sm[128 + r] = delta;
        gl[r] = lse2;
        gl[128 + r] = delta;
      }
      mbar_arrive(&st_full[b]);
    }
  }
  } else {
    setmaxnreg_inc<PB_REGS_WORK>();
    if (!bad_align) {
    // ------------------------------------------------------------------ thread = half a row
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane, c0 = wg * 64;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    bool ok = true;
    uint32_t G = 0, st = 0, st_ph = 0, acc_ph = 0;
    for (int it = 0; it < n_my && ok; ++it) {
      Item I;
      load_item(I, it);
      float lse2 = 0.f, delta = 0.f;
      if (!KEYS) {
        if (!mbar_wait_warp(&st_full[it & 1], (it >> 1) & 1, ctx, 68)) { ok = false; break; }
        const float* sm = reinterpret_cast<const float*>(smem + PB_OFF_STAT + (it & 1) * 1024);
        lse2 = sm[row];
        delta = sm[128 + row];
        mbar_arrive(&st_empty[it & 1]);
      }
      // ROWS = queries: columns below `edge` are seen; ROWS = keys: columns from `edge` on
      int edge, warp_edge;
      float at;
      if constexpr (KEYS) {
        edge = row < I.rows() ? I.t.lowest(row) : 0;
        warp_edge = I.t.lowest((warp & 3) * 32 + 31);            // the largest of the warp's
        at = (float)(I.t.first + row - I.t.off);                 // the query at whose position the key is
      } else {
        edge = row < I.rows() ? I.t.limit(row) : 0x7fffffff;
        warp_edge = I.t.limit((warp & 3) * 32);
        at = (float)(I.t.pos + row);
      }
      float slope = 0.f;
      for (int j = 0; j < I.n; ++j, ++G) {
        const BwdStep s = step_of(a, I, j);
        const uint32_t buf = G & 1, t_s = t_lane + PB_COL_S + buf * PB_T + c0;
        if (BIAS && (KEYS || j == 0)) slope = __ldg(a.slopes + (KEYS ? s.head : I.head)) * 1.4426950408889634f;
        uint32_t p[64];
        if (!mbar_wait_warp(&s_full[buf], (G >> 1) & 1, ctx, 69)) { ok = false; break; }
        tc_fence_after();
        {
          uint32_t(&p0)[32] = *reinterpret_cast<uint32_t(*)[32]>(p);
          uint32_t(&p1)[32] = *reinterpret_cast<uint32_t(*)[32]>(p + 32);
          tmem_ld32(t_s, p0);
          tmem_ld32(t_s + 32, p1);
          tmem_ld_wait();
          tmem_ld_fence(p0);
          tmem_ld_fence(p1);
        }
        const float* stat = reinterpret_cast<const float*>(smem + PB_OFF_STAT + st * 1024) + c0;
        if (KEYS && !mbar_wait_warp(&st_full[st], st_ph, ctx, 70)) { ok = false; break; }
        const float gap = at - (float)(s.index + c0);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          float2 l[2];
          if (KEYS) {
            const float4 v = *reinterpret_cast<const float4*>(stat + i);
            l[0] = make_float2(-v.x, -v.y);
            l[1] = make_float2(-v.z, -v.w);
          } else {
            l[0] = l[1] = splat2(-lse2);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int c = i + 2 * k;
            float2 x = make_float2(__uint_as_float(p[c]), __uint_as_float(p[c + 1]));
            if constexpr (CAP) {
              const float2 rc = make_float2(rcp_approx(1.f + ex2(x.x * a.cap_in)), rcp_approx(1.f + ex2(x.y * a.cap_in)));
              x = fma2(rc, splat2(-2.f * a.cap_out), splat2(a.cap_out));
            } else if constexpr (BIAS) {
              x = mul2(x, splat2(a.scale_log2));
            }
            if constexpr (BIAS) {
              l[k].x = fmaf(-slope, fabsf(gap - (float)c), l[k].x);
              l[k].y = fmaf(-slope, fabsf(gap - (float)(c + 1)), l[k].y);
            }
            x = CAP || BIAS ? add2(x, l[k]) : fma2(x, splat2(a.scale_log2), l[k]);
            p[c] = __float_as_uint(ex2(x.x));
            p[c + 1] = __float_as_uint(ex2(x.y));
          }
        }
        const bool masked = KEYS ? s.index + c0 < warp_edge : s.index + c0 + 64 > warp_edge;
        if (KEYS && masked) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (s.index + c0 + i < edge) p[i] = 0u;
        }
        if (!mbar_wait_warp(dp_full, G & 1, ctx, 71)) { ok = false; break; }
        tc_fence_after();
        uint32_t d[64];
        {
          uint32_t(&d0)[32] = *reinterpret_cast<uint32_t(*)[32]>(d);
          uint32_t(&d1)[32] = *reinterpret_cast<uint32_t(*)[32]>(d + 32);
          tmem_ld32(t_lane + PB_COL_DP + c0, d0);
          tmem_ld32(t_lane + PB_COL_DP + c0 + 32, d1);
          tmem_ld_wait();
          tmem_ld_fence(d0);
          tmem_ld_fence(d1);
        }
        tc_fence_before();
        mbar_arrive(dp_free);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          float2 m[2];
          if (KEYS) {
            const float4 v = *reinterpret_cast<const float4*>(stat + 128 + i);
            m[0] = make_float2(-v.x, -v.y);
            m[1] = make_float2(-v.z, -v.w);
          } else {
            m[0] = m[1] = splat2(-delta);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int c = i + 2 * k;
            float2 g = add2(make_float2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), m[k]);
            g = mul2(g, make_float2(__uint_as_float(p[c]), __uint_as_float(p[c + 1])));
            d[c] = __float_as_uint(g.x);
            d[c + 1] = __float_as_uint(g.y);
          }
        }
        if constexpr (CAP) {                                     // S is still in tensor memory: the factor from it again, 4 r (1 - r), r = 1 / (1 + e^2y)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t y[32];
            tmem_ld32(t_s + 32 * half, y);
            tmem_ld_wait();
            tmem_ld_fence(y);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float r = rcp_approx(1.f + ex2(__uint_as_float(y[i]) * a.cap_in));
              d[32 * half + i] = __float_as_uint(__uint_as_float(d[32 * half + i]) * (4.f * r * (1.f - r)));
            }
          }
        }
        if (masked) {                                            // 0 * something that is no number
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (KEYS ? s.index + c0 + i < edge : s.index + c0 + i >= edge) d[i] = 0u;
        }
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = pack16(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1]), F16);
        tmem_st32(t_s + 32, w);
        if (KEYS) {
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = pack16(__uint_as_float(p[2 * i]), __uint_as_float(p[2 * i + 1]), F16);
          tmem_st32(t_s, w);
          if (++st == PB_RING) {
            st = 0;
            st_ph ^= 1;
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&ds_full[buf]);
      }
      if (!ok) break;
      if (I.n > 0) {
        if (!mbar_wait_warp(acc_full, acc_ph, ctx, 72)) { ok = false; break; }
        acc_ph ^= 1;
        tc_fence_after();
      }
      // ROWS = queries: 32 columns of dQ per thread; ROWS = keys: dK by one half of the threads, dV by the other
      constexpr int COLS = KEYS ? 64 : 32;
#pragma unroll
      for (int half = 0; half < COLS / 32; ++half) {
        uint32_t r[32];
        const uint32_t col = KEYS ? (wg ? PB_COL_A2 : PB_COL_A1) + 32 * half : PB_COL_A1 + 32 * wg;
        if (I.n > 0) {
          tmem_ld32(t_lane + col, r);
          tmem_ld_wait();
          tmem_ld_fence(r);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        if (row < I.rows()) {
          const float f = KEYS && wg ? 1.f : a.scale;
          uint8_t* dst;
          if (KEYS && wg) dst = static_cast<uint8_t*>(a.g2) + 2 * ((int64_t)(I.row0() + row) * a.g2_st + (int64_t)I.head * a.g2_sh + 32 * half);
          else dst = static_cast<uint8_t*>(a.g1) + 2 * ((int64_t)(I.row0() + row) * a.g1_st + (int64_t)I.head * a.g1_sh + (KEYS ? 32 * half : 32 * wg));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack16(__uint_as_float(r[8 * i + 2 * k]) * f, __uint_as_float(r[8 * i + 2 * k + 1]) * f, F16);
            *reinterpret_cast<uint4*>(dst + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      tc_fence_before();                                         // the accumulators have been read when the next step is handed over
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && !bad_align) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, PB_TMEM_COLS);
  }
}

using BwdFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, PackBwdArgs);
template <int F16, bool KEYS>
static BwdFn bwd_kernel(bool cap, bool bias) {
  if (cap) return bias ? attn_pack_bwd_kernel<F16, KEYS, true, true> : attn_pack_bwd_kernel<F16, KEYS, true, false>;
  return bias ? attn_pack_bwd_kernel<F16, KEYS, false, true> : attn_pack_bwd_kernel<F16, KEYS, false, false>;
}

// The register split draws on what the block was launched with: a build that allocates less is refused here, it would wait forever.
static int bwd_ready(BwdFn kern, int which) {
  static PerDevice<bool> ready[16];
  int dev = 0;
  cudaGetDevice(&dev);
  if (ready[which].get(dev)) return KF_OK;
  cudaFuncAttributes attr;
  cudaError_t e = cudaFuncGetAttributes(&attr, kern);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncGetAttributes(attn_pack_bwd_kernel)");
  KF_REQUIRE(attr.numRegs >= PB_REGS_LAUNCH, "kf_attn_pack_bwd: the kernel was built with %d registers per thread, its split needs %d", attr.numRegs, PB_REGS_LAUNCH);
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PB_SMEM);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(attn_pack_bwd_kernel)");
  ready[which].put(dev, true);
  return KF_OK;
}

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_attn_pack_ws_bytes(int Hq, int n_q_tiles) {
  if (Hq <= 0 || n_q_tiles < 0) {
    set_error("kf_attn_pack_ws_bytes: bad argument Hq=%d n_q_tiles=%d", Hq, n_q_tiles);
    return KF_ERR_BAD_ARGUMENT;
  }
  return (int64_t)Hq * n_q_tiles * 256 * 4;
}

extern "C" int kf_attn_pack_bwd(const kf_attn_pack_params* p, void* stream) {
  int rc = check_pack(p);
  if (rc != KF_OK) return rc;
  if (p->n_q_tiles == 0 && p->n_k_tiles == 0) return KF_OK;
  constexpr float LOG2E = 1.4426950408889634f;
  kf_heads q{}, k{}, v{}, o{}, go{}, gq{}, gk{}, gv{};
  if (p->n_q_tiles > 0) {
    KF_REQUIRE(p->Tq > 0 && p->q_tiles && p->lse, "kf_attn_pack_bwd: null pointer");
    if ((rc = check_heads("q", p->q, p->Tq, p->Hq, &q)) != KF_OK) return rc;
    if ((rc = check_heads("o", p->o, p->Tq, p->Hq, &o)) != KF_OK) return rc;
    if ((rc = check_heads("dout", p->dout, p->Tq, p->Hq, &go)) != KF_OK) return rc;
    if ((rc = check_heads("dq", p->dq, p->Tq, p->Hq, &gq)) != KF_OK) return rc;
    KF_REQUIRE(p->ws && (reinterpret_cast<uintptr_t>(p->ws) & 15) == 0 && p->ws_bytes >= kf_attn_pack_ws_bytes(p->Hq, p->n_q_tiles),
               "kf_attn_pack_bwd: workspace of %lld bytes, needs %lld, 16-byte aligned", (long long)p->ws_bytes, (long long)kf_attn_pack_ws_bytes(p->Hq, p->n_q_tiles));
  }
  if (p->n_k_tiles > 0) {
    KF_REQUIRE(p->Tk > 0 && p->k_tiles, "kf_attn_pack_bwd: null pointer");
    if ((rc = check_heads("k", p->k, p->Tk, p->Hk, &k)) != KF_OK) return rc;
    if ((rc = check_heads("v", p->v, p->Tk, p->Hk, &v)) != KF_OK) return rc;
    if ((rc = check_heads("dk", p->dk, p->Tk, p->Hk, &gk)) != KF_OK) return rc;
    if ((rc = check_heads("dv", p->dv, p->Tk, p->Hk, &gv)) != KF_OK) return rc;
  }
  // without queries (or keys) at all the maps over them are never used: they then describe the other side
  const bool any_q = p->n_q_tiles > 0, any_k = p->n_k_tiles > 0;
  CUtensorMap tq, tgo, tk, tv;
  auto maps = [&](const kf_heads& x, const kf_heads& y, int64_t rows, int heads, CUtensorMap* mx, CUtensorMap* my) {
    const int r = make_tmap_heads(mx, x.ptr, rows, heads, x.row_stride, x.head_stride, PB_T);
    return r != KF_OK ? r : make_tmap_heads(my, y.ptr, rows, heads, y.row_stride, y.head_stride, PB_T);
  };
  if (any_q && (rc = maps(q, go, p->Tq, p->Hq, &tq, &tgo)) != KF_OK) return rc;
  if (any_k && (rc = maps(k, v, p->Tk, p->Hk, &tk, &tv)) != KF_OK) return rc;
  if (!any_q) { tq = tk; tgo = tv; }
  if (!any_k) { tk = tq; tv = tgo; }
  int sms = 0;
  if ((rc = device_sm_count(&sms)) != KF_OK) return rc;
  const bool f = p->dtype == KF_F16, c = p->cap > 0.f, b = p->slopes != nullptr;
  PackBwdArgs a{};
  a.share = p->Hq / p->Hk;
  a.scale = p->scale;
  a.scale_log2 = p->scale * LOG2E;
  if (c) {
    a.cap_in = 2.f * p->scale * LOG2E / p->cap;
    a.cap_out = p->cap * LOG2E;
  }
  a.slopes = p->slopes;
  a.stats = static_cast<float*>(p->ws);
  a.n_q_tiles = p->n_q_tiles;
  a.err = dev_error_ptr();
  KF_REQUIRE(a.err != nullptr, "kf_attn_pack_bwd: device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (any_q) {
    a.tiles = reinterpret_cast<const int4*>(p->q_tiles);
    a.heads = p->Hq;
    a.n_items = p->n_q_tiles * p->Hq;
    a.O = o.ptr; a.o_st = o.row_stride; a.o_sh = o.head_stride;
    a.dO = go.ptr; a.do_st = go.row_stride; a.do_sh = go.head_stride;
    a.lse = p->lse; a.lse_ld = p->Tq;
    a.g1 = gq.ptr; a.g1_st = gq.row_stride; a.g1_sh = gq.head_stride;
    const BwdFn kern = f ? bwd_kernel<1, false>(c, b) : bwd_kernel<0, false>(c, b);
    if ((rc = bwd_ready(kern, f * 8 + c * 2 + b)) != KF_OK) return rc;
    const cudaError_t e = launch_maybe_pdl(p->Tq, kern, dim3(a.n_items < sms ? a.n_items : sms), dim3(PB_THREADS), PB_SMEM, st, tq, tgo, tk, tv, a);
    if (e != cudaSuccess) return cuda_status(e, "kf_attn_pack_bwd launch (queries)");
  }
  if (any_k) {
    a.tiles = reinterpret_cast<const int4*>(p->k_tiles);
    a.heads = p->Hk;
    a.n_items = p->n_k_tiles * p->Hk;
    a.g1 = gk.ptr; a.g1_st = gk.row_stride; a.g1_sh = gk.head_stride;
    a.g2 = gv.ptr; a.g2_st = gv.row_stride; a.g2_sh = gv.head_stride;
    const BwdFn kern = f ? bwd_kernel<1, true>(c, b) : bwd_kernel<0, true>(c, b);
    if ((rc = bwd_ready(kern, f * 8 + 4 + c * 2 + b)) != KF_OK) return rc;
    const cudaError_t e = launch_maybe_pdl(p->Tk, kern, dim3(a.n_items < sms ? a.n_items : sms), dim3(PB_THREADS), PB_SMEM, st, tk, tv, tq, tgo, a);
    if (e != cudaSuccess) return cuda_status(e, "kf_attn_pack_bwd launch (keys)");
  }
  return KF_OK;
}
