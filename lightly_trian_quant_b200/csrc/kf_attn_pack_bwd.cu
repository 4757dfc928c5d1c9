// Gradients of the attention over packed sequences (kf_attn_pack.cu), head dimension 64, on the sm_100a tensor cores.
//
//   P = exp(s - lse);  dV = P^T dO;  dP = dO V^T;  delta = rowsum(dO * O);  dS = P * (dP - delta) * ds/d(scale q.k);
//   dQ = scale * dS K;  dK = scale * dS^T Q        (ds/d(scale q.k) is 1, or 1 - tanh^2 with a cap)
//
// Two launches of one kernel, which share the mathematics and differ in what stays and what passes by:
//   ROWS = queries  a CTA keeps 128 queries (Q, dO) and goes through key tiles (K, V):        dQ
//   ROWS = keys     a CTA keeps 128 keys (K, V) and goes through query tiles (Q, dO) of every head that shares them:   dK, dV
// S and dP are computed in both (8 products, the one for delta below among them, where one pass over the pairs takes 5): each gradient is then summed in one place, in
// tensor memory, in a fixed order.  One pass would add dQ from every key tile to memory by atomics, 32 KB per pair of tiles, in an order that changes
// from run to run.
//
//   CTA      one per SM, persistent over (tile, head) items, the longest first; steps of 96 passing rows
//   roles    two pairs of groups of four warps take the steps in turn, a thread half a row: S and dP from tensor memory, P and dS as 16-bit
//            pairs back over dP; warp 16: TMA (row operands in two buffers, passing operands in a ring); warps 17, 18, 19: the products S, dP
//            and those of the gradients
//   pipeline two S buffers, two dP buffers, the accumulators (2 x 96 + 2 x 96 + 2 x 64 columns).  The groups read their S at once, so
//            S(G + 2) is issued while it works on step G; dP(G + 2) goes behind the gradients' products of step G, which read P and dS from
//            the same buffer, and is needed when the exponentials of step G + 2 are done.  The groups of an item's last step write the
//            item's gradients, the others go on with the next item.
//   delta    dO . O takes the output as it was rounded; with ROWS = queries the sum of P (dP - delta) along a row, which should be 0, tells by how
//            much delta is off, and dQ is put right by that times the product P K (which dQ's error is), as is the delta that the second
//            launch takes.  Without it dQ and dK of a few queries with steep slopes were 1.53 times as far off as a single
//            rounding of the result, now 1.4 times; it costs one product more in the first launch
//   numerics P and dS are rounded to the 16-bit type of the operands (the products' A operand); everything else fp32.  With f16 P is 2^14 times what it is, by the
//            exponent's offset: probabilities of long rows lie below f16's normal range (at 818 401 keys dV was 2.4 % off, the same way in every row).  Delta and dP take
//            the power of two back in front of dS, by the multiplication that was an addition; dV and the product P K at the end.
//   measured 8 x 1605 tokens, 16 heads, bf16: first launch 162 us, second 177 (four products in each: 1.04 and 0.95 PFLOP/s); cold, issue slots 53 and 47 % busy,
//            tensor cores 52 and 47 %, special-function unit 50 and 53 %: warps wait for tensor memory, with ROWS = keys for shared memory too
#include "kf_attn.cuh"

namespace kf {

constexpr int PB_T = 128, PB_W = 96, PB_D = 64;                // rows of a tile that stays, rows of a passing one
constexpr int PB_THREADS = 640;
constexpr int PB_REGS_WORK = 104, PB_REGS_LEAN = 64, PB_REGS = split_regs(512, PB_REGS_WORK, 128, PB_REGS_LEAN);
static_assert(PB_THREADS * PB_REGS <= 65536, "registers of an SM");
constexpr int PB_RTILE = PB_T * PB_D * 2, PB_CTILE = PB_W * PB_D * 2;     // 16 KB, 12 KB
// Shared memory: row operands in two buffers (with ROWS = queries also O, for delta), a ring of passing ones; with ROWS = keys the log-sum-exp
// and delta of the passing rows (1 KB per stage), with ROWS = queries the row sums of dS of four items (2 KB each); barriers.
template <bool KEYS>
struct BwdMem {
  static constexpr int RING = KEYS ? 6 : 5, RTILES = KEYS ? 2 : 3;
  static constexpr int OFF_C = 2 * RTILES * PB_RTILE, OFF_STAT = OFF_C + RING * 2 * PB_CTILE, OFF_BAR = OFF_STAT + (KEYS ? RING : 8) * 1024;
  static constexpr size_t BYTES = (size_t)OFF_BAR + 512;
  static_assert(BYTES <= 227 * 1024, "shared memory");
};
constexpr int PB_COL_S = 0, PB_COL_D = 2 * PB_W, PB_COL_A1 = 4 * PB_W, PB_COL_A2 = PB_COL_A1 + PB_D, PB_TMEM_COLS = 512;
static_assert(PB_COL_A2 + PB_D <= PB_TMEM_COLS, "TMEM budget");
// Which of eight element pairs take the polynomial exponential: where instructions are shorter than the special-function unit's time.  8 x 1605 tokens:
// first launch none / one / two of eight 166.8 / 164.4 / 165.3 us, with a cap (fewer tokens) 69.1 / 72.9 / 74.8, second launch none / one / two 191 / 194 / 201
__host__ __device__ constexpr int bwd_poly(bool keys, bool cap) { return keys || cap ? 0 : 0x80; }

// P is computed 2^shift times as large
__host__ __device__ constexpr int bwd_shift(int f16) { return f16 ? 14 : 0; }
__host__ __device__ constexpr float bwd_unshift(int f16) { return f16 ? 0x1p-14f : 1.f; }

struct PackBwdArgs {
  const int4* tiles;
  int n_items, heads, share;     // heads of the items: query heads (ROWS = queries), key heads times `split`
  int split;                     // ROWS = keys: items per key head: 1, or the query heads that share it; their sums are then joined by bwd_join_kernel
  float* parts;                  // [n_items][2][128][64] of a split
  float scale, scale_log2;
  Cap cap;
  const float* slopes;
  float *lse2, *delta;           // shift - lse * log2(e) (-inf: no row, or one that sees nothing) and -delta / 2^shift: [Hq][n_q_tiles * 128], a sequence's rows from its first tile's slot on
  int64_t stat_ld;
  // ROWS = queries
  const float* lse;
  int64_t lse_ld;
  // outputs: dQ, or dK and dV
  void *g1, *g2;
  int64_t g1_st, g1_sh, g2_st, g2_sh;
  int wide;                      // rows of the outputs are 32-byte aligned
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
    n = (t.limit(t.rows - 1) + PB_W - 1) / PB_W;
  }
  __device__ __forceinline__ int rows() const { return t.rows; }
  __device__ __forceinline__ int row0() const { return t.row; }
  __device__ __forceinline__ int slot() const { return t.slot; }
};
template <>
struct BwdItem<true> {
  KTile t;
  int head, n, per, first, q_head;                              // per: passing tiles per query head, from tile `first` of the sequence on; q_head: the first one
  __device__ __forceinline__ void load(const PackBwdArgs& a, int item) {
    t = load_tile<KTile>(a.tiles, item / a.heads);
    const int h = item % a.heads, each = a.share / a.split;     // query heads of an item
    head = h / a.split;
    q_head = h * each;
    first = t.lowest(0) / PB_W;
    const int tiles = (t.q_len + PB_W - 1) / PB_W;
    per = tiles > first ? tiles - first : 0;
    n = per * each;
  }
  __device__ __forceinline__ int rows() const { return t.rows; }
  __device__ __forceinline__ int row0() const { return t.row; }
  __device__ __forceinline__ int slot() const { return t.slot0; }
};
// Where a step's passing tile lies: first row in the batch, head, index of its first row in the sequence, rows that belong to the sequence.
struct BwdStep {
  int row, head, index, valid;
};
__device__ __forceinline__ BwdStep step_of(const PackBwdArgs& a, const BwdItem<false>& i, int j) {
  return {i.t.k_row + j * PB_W, i.head / a.share, j * PB_W, i.t.k_len - j * PB_W};
}
__device__ __forceinline__ BwdStep step_of(const PackBwdArgs& a, const BwdItem<true>& i, int j) {
  const int hh = j / i.per, qt = i.first + j - hh * i.per;
  return {i.t.q_row + qt * PB_W, i.q_head + hh, qt * PB_W, i.t.q_len - qt * PB_W};
}

template <int F16, bool KEYS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(PB_THREADS, 1)
attn_pack_bwd_kernel(const __grid_constant__ CUtensorMap tmR1, const __grid_constant__ CUtensorMap tmR2, const __grid_constant__ CUtensorMap tmR3,
                     const __grid_constant__ CUtensorMap tmC1, const __grid_constant__ CUtensorMap tmC2, const __grid_constant__ PackBwdArgs a) {
  using Mem = BwdMem<KEYS>;
  constexpr float UNSHIFT = bwd_unshift(F16);
  constexpr int PB_RING = Mem::RING, RTILES = Mem::RTILES, PB_OFF_C = Mem::OFF_C, PB_OFF_STAT = Mem::OFF_STAT, PB_OFF_BAR = Mem::OFF_BAR;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PB_OFF_BAR);
  uint64_t *r_full = bars, *r_empty = r_full + 2, *c1_full = r_empty + 2, *c2_full = c1_full + PB_RING, *c_empty = c2_full + PB_RING, *st_full = c_empty + PB_RING,
           *s_full = st_full + PB_RING, *s_free = s_full + 2, *dp_full = s_free + 2, *ds_full = dp_full + 2, *d_free = ds_full + 2, *acc_full = d_free + 2,
           *acc_free = acc_full + 2, *rs_full = acc_free + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(rs_full + 4);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  pdl_launch_dependents();
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int n_my = items_of_cta(a.n_items);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], KEYS ? 2 : 2 + 16);                  // S, dP; the warps that read O and dO
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 256);
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 256);
      mbar_init(&d_free[i], 1);
      mbar_init(&acc_full[i], 1);                                // items in turn: a group may ask for its item before the other's is complete
    }
    for (int i = 0; i < PB_RING; ++i) {
      mbar_init(&c1_full[i], 1);
      mbar_init(&c2_full[i], 1);
      mbar_init(&c_empty[i], 1);
      mbar_init(&st_full[i], 1);
    }
    mbar_init(acc_free, 256);
    for (int i = 0; i < 4; ++i) mbar_init(&rs_full[i], 512);
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(tmem_holder, PB_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = (uint32_t)uniform_int((int)*tmem_holder);
  const WaitCtx ctx{abort_flag, a.err};
  const bool bad_align = (smem_u32(smem) & 1023u) != 0;
  if (bad_align && threadIdx.x == 0 && atomicCAS(&a.err[0], 0u, 99u) == 0u) {
    a.err[1] = 120;
    a.err[2] = blockIdx.x;
  }
  using Item = BwdItem<KEYS>;
  auto load_item = [&](Item& i, int it) { i.load(a, item_of_cta(it)); };

  if (warp >= 16) {
  setmaxnreg_dec<PB_REGS_LEAN>();
  if (bad_align) {
    // nothing was issued; fall through to the teardown
  } else if (warp == 16) {
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
        uint8_t* to = smem + rb * RTILES * PB_RTILE;
        mbar_expect_tx(&r_full[rb], RTILES * PB_RTILE);
        tma_load_3d(to, &tmR1, 0, I.head, I.row0(), &r_full[rb]);
        tma_load_3d(to + PB_RTILE, &tmR2, 0, I.head, I.row0(), &r_full[rb]);
        if (!KEYS) tma_load_3d(to + 2 * PB_RTILE, &tmR3, 0, I.head, I.row0(), &r_full[rb]);
      }
      __syncwarp();
      ++ri;
      for (int j = 0; j < I.n; ++j) {
        const BwdStep s = step_of(a, I, j);
        if (!mbar_wait_warp(&c_empty[st], ph, ctx, 61)) { ok = false; break; }
        if (elect_one()) {
          uint8_t* to = smem + PB_OFF_C + st * 2 * PB_CTILE;
          mbar_expect_tx(&c1_full[st], PB_CTILE + (KEYS ? 2 * PB_W * 4 : 0));
          tma_load_3d(to, &tmC1, 0, s.head, s.row, &c1_full[st]);
          if (KEYS) {                                                         // 96 values each; what is behind the sequence's end is put right by the issuer
            const int64_t at = s.head * a.stat_ld + (int64_t)I.slot() * PB_T + s.index;
            uint8_t* sm = smem + PB_OFF_STAT + st * 1024;
            bulk_load_1d(sm, a.lse2 + at, PB_W * 4, &c1_full[st]);
            bulk_load_1d(sm + 512, a.delta + at, PB_W * 4, &c1_full[st]);
          }
          mbar_expect_tx(&c2_full[st], PB_CTILE);
          tma_load_3d(to + PB_CTILE, &tmC2, 0, s.head, s.row, &c2_full[st]);
        }
        __syncwarp();
        if (++st == PB_RING) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ MMA issuers: warp 17 S, warp 18 dP, warp 19 the gradients
    // One warp for all three spent 1700 clk per step on waiting, addresses and issue, twice the time of the products.
    // Everything the products take is worked out by the whole warp, in front of the branch that one lane takes: behind it each address would
    // be one lane's, moved to a uniform register in front of every instruction.
    const bool leader = elect_one();
    int it = 0, next_n = -1, next_per = 0, next_rows = 0;                     // the item behind this one is asked for ahead
    auto fetch = [&]() {
      next_n = -1;
      if (it < n_my) {
        Item I;
        load_item(I, it++);
        next_n = I.n;
        if constexpr (KEYS) {
          next_per = I.per;
          next_rows = I.t.q_len - I.first * PB_W;
        } else {
          next_per = I.n;
          next_rows = I.t.k_len;
        }
      }
    };
    int j, n, jj, per, rows;                                                  // step of the item and their number (-1: no item left); step of the sequence, their number, its rows
    uint32_t G = 0, ri = 0, st = 0, ph = 0;                                   // steps and items before, ring stage and its parity
    auto open = [&]() {                                                       // the next item that has steps
      do {
        n = uniform_int(next_n);
        per = uniform_int(next_per);
        rows = uniform_int(next_rows);
        fetch();
      } while (n == 0);
      j = jj = 0;
    };
    auto advance = [&]() {
      ++G;
      if (++st == PB_RING) {
        st = 0;
        ph ^= 1;
      }
      if (++jj == per) jj = 0;
      if (++j == n) {
        ++ri;
        open();
      }
    };
    fetch();
    open();
    const uint32_t fmt = F16 ? 0u : 1u;
    if (warp < 19) {
      // row operand `which` times the passing one, 128 x 96 x 64, into the buffer that the step before the last has left
      const uint32_t which = warp - 17;
      const uint32_t idesc = idesc_f16(fmt, PB_W), col = which ? PB_COL_D : PB_COL_S;
      uint64_t *const c_full = which ? c2_full : c1_full, *const room = which ? d_free : s_free, *const full = which ? dp_full : s_full;
      while (n > 0) {
        const uint32_t b = G & 1, b_ph = ((G >> 1) & 1) ^ 1;
        if (j == 0 && !mbar_wait_warp(&r_full[ri & 1], (ri >> 1) & 1, ctx, 62)) break;
        if (!mbar_wait_warp3(&c_full[st], ph, &room[b], b_ph, &room[b], b_ph, ctx, 63)) break;
        uint8_t* const tile = smem + PB_OFF_C + (st * 2 + which) * PB_CTILE;
        const int valid = rows - jj * PB_W;
        if (valid < PB_W) {                                                   // what the tile holds behind the end of the sequence becomes zero
          if (KEYS && which == 0) {                                           // the rows' values there: P = 0
            float* sm = reinterpret_cast<float*>(smem + PB_OFF_STAT + st * 1024);
            for (int i = valid + lane; i < PB_W; i += 32) {
              sm[i] = -INFINITY;
              sm[128 + i] = 0.f;
            }
          }
          zero_rows(tile, valid, PB_W, lane);
        }
        if (KEYS && which == 0 && lane == 0) mbar_arrive(&st_full[st]);
        const uint32_t d = tmem_base + col + b * PB_W;
        const uint64_t r = smem_desc_sw128(smem_u32(smem + ((ri & 1) * RTILES + which) * PB_RTILE)), p = smem_desc_sw128(smem_u32(tile));
        uint64_t *const done = &full[b], *const r_done = &r_empty[ri & 1];
        const bool last = j + 1 == n;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < PB_D / 16; ++kk) mma_f16(d, r + 2 * kk, p + 2 * kk, idesc, kk != 0);
          tc_commit(done);
          if (last) tc_commit(r_done);
        }
        __syncwarp();
        advance();
      }
    } else {
      const uint32_t idesc = idesc_f16(fmt, PB_D) | (1u << 16);               // the passing operand is MN-major
      while (n > 0) {
        const uint32_t b = G & 1;
        if (!mbar_wait_warp(&ds_full[b], (G >> 1) & 1, ctx, 67)) break;
        if (j == 0 && ri > 0 && !mbar_wait_warp(acc_free, (ri - 1) & 1, ctx, 68)) break;   // the last item's gradients have been read
        tc_fence_after();
        const uint32_t t_d = tmem_base + PB_COL_D + b * PB_W;
        const uint64_t c1 = smem_desc_sw128(smem_u32(smem + PB_OFF_C + st * 2 * PB_CTILE)), c2 = c1 + (PB_CTILE >> 4);
        uint64_t *const c_done = &c_empty[st], *const d_done = &d_free[b], *const a_done = &acc_full[ri & 1];
        const bool last = j + 1 == n;
        const uint32_t more = j != 0;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < PB_W / 16; ++kk) {                            // 16 columns of dP hold 8 words of dS and 8 of P
            const uint32_t d = t_d + kk * 16;
            mma_f16_ta(tmem_base + PB_COL_A2, d + 8, (KEYS ? c2 : c1) + (uint64_t)(kk * (2048 >> 4)), idesc, kk ? 1u : more);
            mma_f16_ta(tmem_base + PB_COL_A1, d, c1 + (uint64_t)(kk * (2048 >> 4)), idesc, kk ? 1u : more);
          }
          tc_commit(d_done);
          tc_commit(c_done);
          if (last) tc_commit(a_done);
        }
        __syncwarp();
        advance();
      }
    }
  }
  } else {
    setmaxnreg_inc<PB_REGS_WORK>();
    if (!bad_align) {
    // ------------------------------------------------------------------ a thread half a row of every other step
    const uint32_t par = (warp >> 2) & 1, half = warp >> 3;
    const int row = (warp & 3) * 32 + lane;
    constexpr int COLS = PB_W / 2;
    const int c0 = (int)half * COLS;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + PB_COL_S + par * PB_W + c0, t_d = t_lane + PB_COL_D + par * PB_W + c0;     // step G uses buffers G & 1
    bool ok = true;
    uint32_t G0 = 0, ph = 0, ri = 0;                             // steps before this item; parity of the next step of this kind; items with steps
    uint32_t st = par, st_ph = 0;                                // ring stage of the next step and its parity
    for (int it = 0; it < n_my && ok; ++it) {
      Item I;
      load_item(I, it);
      const int n = I.n;
      // ROWS = queries: the row's log-sum-exp and delta (negated: they are added), also for the second launch
      float nlse2 = 0.f, ndelta = 0.f;
      if constexpr (!KEYS) {
        nlse2 = row < I.rows() ? a.lse[(int64_t)I.head * a.lse_ld + I.row0() + row] : -INFINITY;
        if (n > 0) {
          if (!mbar_wait_warp(&r_full[ri & 1], (ri >> 1) & 1, ctx, 65)) break;
          const uint8_t* d = smem + ((ri & 1) * RTILES + 1) * PB_RTILE + row * 128;
          float2 s = make_float2(0.f, 0.f);
#pragma unroll 4
          for (int c = 0; c < 8; ++c) {
            const int o = (c ^ (row & 7)) << 4;                  // the swizzle of the tile
            const uint4 u = *reinterpret_cast<const uint4*>(d + o), v = *reinterpret_cast<const uint4*>(d + PB_RTILE + o);
            s = fma2(unpack16<F16>(u.x), unpack16<F16>(v.x), s);
            s = fma2(unpack16<F16>(u.y), unpack16<F16>(v.y), s);
            s = fma2(unpack16<F16>(u.z), unpack16<F16>(v.z), s);
            s = fma2(unpack16<F16>(u.w), unpack16<F16>(v.w), s);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&r_empty[ri & 1]);
          if (row < I.rows()) ndelta = -(s.x + s.y) * UNSHIFT;
        }
        nlse2 = nlse2 == -INFINITY ? -INFINITY : fmaf(nlse2, -1.4426950408889634f, (float)bwd_shift(F16));
        if (warp < 4) {
          const int64_t o = I.head * a.stat_ld + (int64_t)I.slot() * PB_T + row;
          a.lse2[o] = nlse2;
          if (n == 0) a.delta[o] = 0.f;
        }
      }
      float2 vsum = make_float2(0.f, 0.f);                       // ROWS = queries: sum of P (dP - delta) over this thread's columns
      // ROWS = queries: the row sees columns below `edge`; ROWS = keys: from `edge` on
      int edge, warp_edge;
      int at;                                                    // ROWS = queries: position; ROWS = keys: the query that stands at the key
      if constexpr (KEYS) {
        edge = row < I.rows() ? I.t.lowest(row) : 0;
        warp_edge = I.t.lowest((warp & 3) * 32 + 31);            // the largest of the warp's
        at = I.t.first + row - I.t.off;
      } else {
        edge = row < I.rows() ? I.t.limit(row) : 0x7fffffff;
        warp_edge = I.t.limit((warp & 3) * 32);
        at = I.t.pos + row;
      }
      float slope = 0.f;
      if (BIAS && !KEYS) slope = __ldg(a.slopes + I.head) * 1.4426950408889634f;
      int index = c0, end = 0x7fffffff, head = 0, per_rows = 0;  // of this thread's first column: its place in the sequence; the sequence's end; head
      if constexpr (KEYS) {
        index += I.first * PB_W;
        end = I.t.q_len;
        head = I.q_head;
        per_rows = I.per * PB_W;
      }
      const int start = index;
      auto move = [&](int steps) {                               // from one query head to the next one that shares the keys
        index += steps * PB_W;
        if constexpr (KEYS) {
          while (index >= start + per_rows) {
            index -= per_rows;
            ++head;
          }
        }
      };
      const int j0 = (int)((G0 + par) & 1);
      if (j0 < n) move(j0);
      for (int j = j0; j < n; j += 2) {
        if (BIAS && KEYS) slope = __ldg(a.slopes + head) * 1.4426950408889634f;
        uint32_t p[3][16];
        if (!mbar_wait_warp(&s_full[par], ph, ctx, 70)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 3; ++q) tmem_ld16(t_s + 16 * q, p[q]);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 3; ++q) tmem_ld_fence(p[q]);
        if (!CAP) {
          tc_fence_before();
          mbar_arrive(&s_free[par]);
        }
        const float* stat = reinterpret_cast<const float*>(smem + PB_OFF_STAT + st * 1024) + c0;
        if (KEYS && !mbar_wait_warp(&st_full[st], st_ph, ctx, 71)) { ok = false; break; }
        const float gap = (float)(at - index);                   // (only the difference fits fp32 behind 2^24)
        bool flat = false;
        if constexpr (CAP) {
          float m4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < COLS; i += 2) m4[(i / 2) & 3] = max3(m4[(i / 2) & 3], fabsf(__uint_as_float(p[i / 16][i % 16])), fabsf(__uint_as_float(p[i / 16][i % 16 + 1])));
          flat = __all_sync(0xffffffffu, amax_nan(amax_nan(m4[0], m4[1]), amax_nan(m4[2], m4[3])) <= a.cap.flat);
        }
        auto exponentials = [&](auto small) {                    // with a cap: every score is small
#pragma unroll
          for (int i = 0; i < COLS; i += 8) {
            uint32_t f[8];                                         // with a cap: 1 - tanh^2
            float v[8];
            if (KEYS) {
              *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(stat + i);
              *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(stat + i + 4);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int c = i + 2 * k;
              float2 l = KEYS ? make_float2(v[2 * k], v[2 * k + 1]) : splat2(nlse2);
              float2 x = make_float2(__uint_as_float(p[c / 16][c % 16]), __uint_as_float(p[c / 16][c % 16 + 1]));
              if constexpr (CAP) {
                float2 d;
                if constexpr (decltype(small)::value) {            // |y| <= 1/2
                  x = cap_flat(a.cap, x);
                  const float2 y = mul2(x, splat2(a.cap.inv_out));
                  d = fma2(make_float2(-y.x, -y.y), y, splat2(1.f));
                } else {
                  x = cap_any(a.cap, x, d);
                }
                f[2 * k] = __float_as_uint(d.x);
                f[2 * k + 1] = __float_as_uint(d.y);
              } else if constexpr (BIAS) {
                x = mul2(x, splat2(a.scale_log2));
              }
              if constexpr (BIAS) {
                l.x = fmaf(-slope, fabsf(gap - (float)c), l.x);
                l.y = fmaf(-slope, fabsf(gap - (float)(c + 1)), l.y);
              }
              x = CAP || BIAS ? add2(x, l) : fma2(x, splat2(a.scale_log2), l);
              x = (bwd_poly(KEYS, CAP) >> ((i / 2 + k) % 8)) & 1 ? ex2_poly2_neg(x) : make_float2(ex2(x.x), ex2(x.y));
              p[c / 16][c % 16] = __float_as_uint(x.x);
              p[c / 16][c % 16 + 1] = __float_as_uint(x.y);
            }
            if constexpr (CAP) tmem_st8(t_s + i, f);               // over S, for the other half of the step
          }
        };
        if (CAP && flat) exponentials(std::true_type{});
        else exponentials(std::false_type{});
        if constexpr (CAP) tmem_st_wait();
        // the columns that the row sees (operands behind the end of a sequence are zero, so that P = 0 is enough)
        if (KEYS ? index < warp_edge || end - index < COLS : index + COLS > warp_edge) {
          const int lo = KEYS ? edge - index : 0, hi = KEYS ? end - index : edge - index;
#pragma unroll
          for (int i = 0; i < COLS; ++i)
            if (i < lo || i >= hi) p[i / 16][i % 16] = 0u;
        }
        if (!mbar_wait_warp(&dp_full[par], ph, ctx, 72)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 3; ++q) {                            // 16 columns: dP in, dS and P out in its place
          uint32_t d[16], f[CAP ? 16 : 1];
          tmem_ld16(t_d + 16 * q, d);
          if constexpr (CAP) tmem_ld16(t_s + 16 * q, f);
          tmem_ld_wait();
          tmem_ld_fence(d);
          if constexpr (CAP) tmem_ld_fence(f);
          uint32_t w[16];
          float u[4];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            if (KEYS && i % 4 == 0) *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(stat + 128 + 16 * q + i);
            const float2 m = KEYS ? make_float2(u[i % 4], u[i % 4 + 1]) : splat2(ndelta);
            const float2 pp = make_float2(__uint_as_float(p[q][i]), __uint_as_float(p[q][i + 1]));
            const float2 dp = make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1]));
            float2 v = mul2(F16 ? fma2(dp, splat2(UNSHIFT), m) : add2(dp, m), pp), g = pp;
            if constexpr (!KEYS) vsum = add2(vsum, v);
            if constexpr (CAP) {
              const float2 b = make_float2(__uint_as_float(f[i]), __uint_as_float(f[i + 1]));
              v = mul2(v, b);
              if constexpr (!KEYS) g = mul2(g, b);
            }
            w[i >> 1] = pack16(v.x, v.y, F16);
            w[8 + (i >> 1)] = pack16(g.x, g.y, F16);
          }
          tmem_st16(t_d + 16 * q, w);
        }
        tmem_st_wait();
        tc_fence_before();
        if (CAP) mbar_arrive(&s_free[par]);
        mbar_arrive(&ds_full[par]);
        ph ^= 1;
        if (KEYS) {
          st += 2;
          if (st >= PB_RING) {
            st -= PB_RING;
            st_ph ^= 1;
          }
        }
        move(2);
      }
      if (!ok) break;
      G0 += n;
      float* const rs = reinterpret_cast<float*>(smem + PB_OFF_STAT) + (ri & 3) * 4 * PB_T + row;      // [part][row]
      const uint32_t rs_ph = (ri >> 2) & 1;
      uint64_t* const rs_bar = &rs_full[ri & 3];
      if (n > 0) {
        if (!KEYS) {
          rs[(par * 2 + half) * PB_T] = vsum.x + vsum.y;
          mbar_arrive(rs_bar);
        }
        ++ri;
      }
      // the groups of the last step write the item's gradients, those of an item without steps (zeros) groups 0
      if (par != (n > 0 ? (G0 - 1) & 1 : 0u)) continue;
      if (n > 0) {
        if (!mbar_wait_warp(&acc_full[(ri - 1) & 1], ((ri - 1) >> 1) & 1, ctx, 73)) { ok = false; break; }
        tc_fence_after();
      }
      load_item(I, it);
      // ROWS = queries: 32 columns of dQ; ROWS = keys: 64 of dK or of dV.  All of them packed in registers, then the accumulators are the next item's.
      constexpr int PIECES = KEYS ? 2 : 1;
      uint32_t w[PIECES][16];
      const uint32_t t_a = t_lane + PB_COL_A1 + half * (32 * PIECES);
      const float scale = KEYS && half ? UNSHIFT : a.scale;
      float gap_d = 0.f;                                         // delta as it was used less what it should have been
      if (!KEYS && n > 0) {
        if (!mbar_wait_warp(rs_bar, rs_ph, ctx, 74)) { ok = false; break; }
        gap_d = -((rs[0] + rs[PB_T]) + (rs[2 * PB_T] + rs[3 * PB_T]));
        if (half == 0) a.delta[I.head * a.stat_ld + (int64_t)I.slot() * PB_T + row] = row < I.rows() ? fmaf(gap_d, UNSHIFT, ndelta) : 0.f;
        gap_d *= UNSHIFT;                                        // for the product P K
      }
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        uint32_t r[32];
        if (n > 0) {
          tmem_ld32(t_a + 32 * i, r);
          tmem_ld_wait();
          tmem_ld_fence(r);
          if (!KEYS) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t u[16];
              tmem_ld16(t_a + PB_D + 16 * q, u);
              tmem_ld_wait();
              tmem_ld_fence(u);
#pragma unroll
              for (int k = 0; k < 16; ++k) r[16 * q + k] = __float_as_uint(fmaf(gap_d, __uint_as_float(u[k]), __uint_as_float(r[16 * q + k])));
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0u;
        }
        if (KEYS && a.split > 1) {                               // the item's sums as they are
          float* to = a.parts + (((int64_t)item_of_cta(it) * 2 + half) * PB_T + row) * PB_D + 32 * i;
#pragma unroll
          for (int k = 0; k < 32; k += 8) stg8w(to + k, r + k);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) w[i][k] = pack16(__uint_as_float(r[2 * k]) * scale, __uint_as_float(r[2 * k + 1]) * scale, F16);
      }
      if (n > 0) {
        tc_fence_before();
        mbar_arrive(acc_free);
      }
      if (KEYS && a.split > 1) continue;
      if (row < I.rows()) {
        const int64_t r = I.row0() + row;
        uint8_t* dst = KEYS && half ? static_cast<uint8_t*>(a.g2) + 2 * (r * a.g2_st + (int64_t)I.head * a.g2_sh)
                                    : static_cast<uint8_t*>(a.g1) + 2 * (r * a.g1_st + (int64_t)I.head * a.g1_sh + (KEYS ? 0 : 32 * (int)half));
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          if (a.wide) {
            stg8w(dst + 64 * i, w[i]);
            stg8w(dst + 64 * i + 32, w[i] + 8);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) reinterpret_cast<uint4*>(dst + 64 * i)[k] = make_uint4(w[i][4 * k], w[i][4 * k + 1], w[i][4 * k + 2], w[i][4 * k + 3]);
          }
        }
      }
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && !bad_align) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem_base, PB_TMEM_COLS);
  }
}

// dK and dV of a key tile and head: the sums of the query heads that share it, in their order.  blockIdx.x: (tile, key head); blockIdx.y: a share of
// its chunks of 8 channels, one per thread, whose loads are in flight together (a CTA per tile and head: 11.6 us for 236 of them and 3 heads, now 7.6).
constexpr int JOIN_THREADS = 256, JOIN_CTAS = 2 * PB_T * (PB_D / 8) / JOIN_THREADS;
template <int F16>
__global__ void __launch_bounds__(JOIN_THREADS) bwd_join_kernel(const __grid_constant__ PackBwdArgs a) {
  pdl_wait();
  const int heads = a.heads / a.split, head = blockIdx.x % heads;
  const KTile t = load_tile<KTile>(a.tiles, blockIdx.x / heads);
  const int i = blockIdx.y * JOIN_THREADS + threadIdx.x, which = i / (PB_T * (PB_D / 8)), rest = i - which * PB_T * (PB_D / 8), row = rest / (PB_D / 8), c = rest % (PB_D / 8) * 8;
  if (row >= t.rows) return;
  const float4* p = reinterpret_cast<const float4*>(a.parts + (int64_t)blockIdx.x * a.split * 2 * PB_T * PB_D + (which * PB_T + row) * PB_D + c);
  constexpr int PART = 2 * PB_T * PB_D / 4, AHEAD = 4;
  float s[8] = {};
  for (int k0 = 0; k0 < a.split; k0 += AHEAD) {
    float4 u[AHEAD], v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (k0 + k < a.split) {
        u[k] = p[(int64_t)(k0 + k) * PART];
        v[k] = p[(int64_t)(k0 + k) * PART + 1];
      }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (k0 + k < a.split) {
        s[0] += u[k].x; s[1] += u[k].y; s[2] += u[k].z; s[3] += u[k].w;
        s[4] += v[k].x; s[5] += v[k].y; s[6] += v[k].z; s[7] += v[k].w;
      }
  }
  const float f = which ? bwd_unshift(F16) : a.scale;
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = pack16(s[2 * k] * f, s[2 * k + 1] * f, F16);
  const int64_t r = t.row + row;
  uint8_t* dst = which ? static_cast<uint8_t*>(a.g2) + 2 * (r * a.g2_st + (int64_t)head * a.g2_sh + c) : static_cast<uint8_t*>(a.g1) + 2 * (r * a.g1_st + (int64_t)head * a.g1_sh + c);
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Items per key head in the second launch: one, or one for every query head that shares it, whose sums go through memory in fp32 (64 KB each).  Whole items of many
// query heads are long chains, split ones fill the device evenly; which is shorter is worked out in steps (0.7 us) from the batch's lengths, the longest chain or the
// mean of an SM: an item costs 6 steps beside its own, the join 6.  Measured, both directions in us, whole / split:
//   16 heads on 1   1 x 1605 tokens 242 / 77, 8 x 1605 371 / 367, 16 x 1605 710 / 758; 20 x 130 54 / 70, 60 x 130 84 / 155, 150 x 130 215 / 352
//   12 heads on 4   1 x 1605 causal 63 / 43, 4 x 1605 causal 92 / 102, 4 x 1605 154 / 158, 60 x 130 81 / 121; ten causal clips of 1 to 2053 with a cap, f16 209 / 189
// (a choice by the number of items alone, fewer than four rounds, took up to 1.84 times the shorter time over 218 such cases, this one up to 1.15)
static int bwd_split(const kf_attn_pack_params* p, int n_k_tiles, int sms) {
  const int share = p->Hq / p->Hk;
  if (share == 1 || n_k_tiles == 0) return 1;
  if (p->k_work <= 0) return (int64_t)n_k_tiles * p->Hq <= sms ? share : 1;
  constexpr double ITEM = 6, JOIN = 6;
  const double n = n_k_tiles, longest = (p->k_longest + PB_W - 1) / PB_W, all = (double)p->k_work / PB_W + 0.5 * n, per_sm = (double)p->Hk / sms;
  const auto larger = [](double x, double y) { return x > y ? x : y; };
  const double whole = larger(longest * share + ITEM, (all * share + n * ITEM) * per_sm), split = larger(longest + ITEM, (all + n * ITEM) * share * per_sm) + JOIN;
  return split < whole ? share : 1;
}
static int64_t bwd_stat_bytes(int Hq, int n_q_tiles) { return 2 * ((int64_t)Hq * n_q_tiles + 1) * PB_T * 4; }      // the last passing tile may reach behind the last row

using BwdFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, PackBwdArgs);
template <int F16, bool KEYS>
static BwdFn bwd_kernel(bool cap, bool bias) {
  if (cap) return bias ? attn_pack_bwd_kernel<F16, KEYS, true, true> : attn_pack_bwd_kernel<F16, KEYS, true, false>;
  return bias ? attn_pack_bwd_kernel<F16, KEYS, false, true> : attn_pack_bwd_kernel<F16, KEYS, false, false>;
}

static int wide_rows(const kf_heads& t) {
  return ((reinterpret_cast<uintptr_t>(t.ptr) | (uintptr_t)(t.row_stride * 2) | (uintptr_t)(t.head_stride * 2)) & 31) == 0;
}

static int bwd_ready(BwdFn kern, int which, size_t smem) {
  static PerDevice<bool> ready[16];
  return split_ready(reinterpret_cast<const void*>(kern), ready[which], PB_REGS, smem, "kf_attn_pack_bwd");
}

static bool wants_keys(const kf_attn_pack_params* p) { return p->dk.ptr || p->dv.ptr; }      // else dq alone: the first launch

static int64_t bwd_ws_bytes(const kf_attn_pack_params* p, int n_k_tiles) {
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != KF_OK) return rc > 0 ? KF_ERR_UNSUPPORTED : rc;
  const int64_t split = bwd_split(p, n_k_tiles, sms);
  return bwd_stat_bytes(p->Hq, p->n_q_tiles) + (split > 1 ? split * n_k_tiles * p->Hk * 2 * PB_T * PB_D * 4 : 0);
}

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_attn_pack_ws_bytes(int Hq, int Hk, int n_q_tiles, int n_k_tiles) {
  if (Hq <= 0 || Hk <= 0 || Hq % Hk || n_q_tiles < 0 || n_k_tiles < 0) {
    set_error("kf_attn_pack_ws_bytes: bad argument Hq=%d Hk=%d n_q_tiles=%d n_k_tiles=%d", Hq, Hk, n_q_tiles, n_k_tiles);
    return KF_ERR_BAD_ARGUMENT;
  }
  kf_attn_pack_params p{};
  p.Hq = Hq; p.Hk = Hk; p.n_q_tiles = n_q_tiles;
  return bwd_ws_bytes(&p, n_k_tiles);
}

extern "C" int64_t kf_attn_pack_bwd_ws_bytes(const kf_attn_pack_params* p) {
  const int rc = check_pack(p);
  return rc != KF_OK ? rc : bwd_ws_bytes(p, wants_keys(p) ? p->n_k_tiles : 0);
}

extern "C" int kf_attn_pack_bwd(const kf_attn_pack_params* p, void* stream) {
  int rc = check_pack(p);
  if (rc != KF_OK) return rc;
  if (p->n_q_tiles == 0 && p->n_k_tiles == 0) return KF_OK;
  constexpr float LOG2E = 1.4426950408889634f;
  kf_heads q{}, k{}, v{}, o{}, go{}, gq{}, gk{}, gv{};
  const bool any_q = p->n_q_tiles > 0, any_k = p->n_k_tiles > 0 && wants_keys(p);
  KF_REQUIRE((!any_q || (p->Tq > 0 && p->q_tiles && p->lse)) && (!any_k || (p->Tk > 0 && p->k_tiles)), "kf_attn_pack_bwd: null pointer");
  if (p->Tq > 0) {
    if ((rc = check_heads("q", p->q, p->Tq, p->Hq, &q)) != KF_OK) return rc;
    if ((rc = check_heads("o", p->o, p->Tq, p->Hq, &o)) != KF_OK) return rc;
    if ((rc = check_heads("dout", p->dout, p->Tq, p->Hq, &go)) != KF_OK) return rc;
    if ((rc = check_heads("dq", p->dq, p->Tq, p->Hq, &gq)) != KF_OK) return rc;
  }
  if (p->Tk > 0) {
    if ((rc = check_heads("k", p->k, p->Tk, p->Hk, &k)) != KF_OK) return rc;
    if ((rc = check_heads("v", p->v, p->Tk, p->Hk, &v)) != KF_OK) return rc;
    if (any_k && (rc = check_heads("dk", p->dk, p->Tk, p->Hk, &gk)) != KF_OK) return rc;
    if (any_k && (rc = check_heads("dv", p->dv, p->Tk, p->Hk, &gv)) != KF_OK) return rc;
  }
  const int64_t need = bwd_ws_bytes(p, any_k ? p->n_k_tiles : 0);
  if (need < 0) return (int)need;
  KF_REQUIRE(p->ws && (reinterpret_cast<uintptr_t>(p->ws) & 31) == 0 && p->ws_bytes >= need, "kf_attn_pack_bwd: workspace of %lld bytes, needs %lld, 32-byte aligned",
             (long long)p->ws_bytes, (long long)need);
  CUtensorMap r1, r2, r3, c1, c2;
  // (a side stays in boxes of 128 rows in one launch and passes in boxes of 96 in the other)
  auto maps = [&](const kf_heads& x, const kf_heads& y, int64_t rows, int heads, int box, CUtensorMap* mx, CUtensorMap* my) {
    const int r = make_tmap_heads(mx, x.ptr, rows, heads, x.row_stride, x.head_stride, box);
    return r != KF_OK ? r : make_tmap_heads(my, y.ptr, rows, heads, y.row_stride, y.head_stride, box);
  };
  int sms = 0;
  if ((rc = device_sm_count(&sms)) != KF_OK) return rc;
  const bool f = p->dtype == KF_F16, c = p->cap > 0.f, b = p->slopes != nullptr;
  PackBwdArgs a{};
  a.share = p->Hq / p->Hk;
  a.split = 1;
  a.scale = p->scale;
  a.scale_log2 = p->scale * LOG2E;
  if (c) a.cap.set(p->scale, p->cap);
  a.slopes = p->slopes;
  a.stat_ld = (int64_t)p->n_q_tiles * PB_T;
  a.lse2 = static_cast<float*>(p->ws);
  a.delta = a.lse2 + a.stat_ld * p->Hq + PB_T;
  a.err = dev_error_ptr();
  KF_REQUIRE(a.err != nullptr, "kf_attn_pack_bwd: device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (any_q) {
    a.tiles = reinterpret_cast<const int4*>(p->q_tiles);
    a.heads = p->Hq;
    a.n_items = p->n_q_tiles * p->Hq;
    a.lse = p->lse; a.lse_ld = p->Tq;
    a.g1 = gq.ptr; a.g1_st = gq.row_stride; a.g1_sh = gq.head_stride;
    a.wide = wide_rows(gq);
    if ((rc = maps(q, go, p->Tq, p->Hq, PB_T, &r1, &r2)) != KF_OK) return rc;
    if ((rc = make_tmap_heads(&r3, o.ptr, p->Tq, p->Hq, o.row_stride, o.head_stride, PB_T)) != KF_OK) return rc;
    if (p->Tk > 0) {
      if ((rc = maps(k, v, p->Tk, p->Hk, PB_W, &c1, &c2)) != KF_OK) return rc;
    } else {                                                  // nothing passes: never used
      c1 = r1;
      c2 = r2;
    }
    const BwdFn kern = f ? bwd_kernel<1, false>(c, b) : bwd_kernel<0, false>(c, b);
    if ((rc = bwd_ready(kern, f * 8 + c * 2 + b, BwdMem<false>::BYTES)) != KF_OK) return rc;
    const cudaError_t e = launch_maybe_pdl(p->Tq, kern, dim3(a.n_items < sms ? a.n_items : sms), dim3(PB_THREADS), BwdMem<false>::BYTES, st, r1, r2, r3, c1, c2, a);
    if (e != cudaSuccess) return cuda_status(e, "kf_attn_pack_bwd launch (queries)");
  }
  if (any_k) {
    a.tiles = reinterpret_cast<const int4*>(p->k_tiles);
    a.split = bwd_split(p, p->n_k_tiles, sms);
    a.heads = p->Hk * a.split;
    a.n_items = p->n_k_tiles * a.heads;
    a.parts = static_cast<float*>(p->ws) + bwd_stat_bytes(p->Hq, p->n_q_tiles) / 4;
    a.g1 = gk.ptr; a.g1_st = gk.row_stride; a.g1_sh = gk.head_stride;
    a.g2 = gv.ptr; a.g2_st = gv.row_stride; a.g2_sh = gv.head_stride;
    a.wide = wide_rows(gk) && wide_rows(gv);
    if ((rc = maps(k, v, p->Tk, p->Hk, PB_T, &r1, &r2)) != KF_OK) return rc;
    if (p->Tq > 0) {
      if ((rc = maps(q, go, p->Tq, p->Hq, PB_W, &c1, &c2)) != KF_OK) return rc;
    } else {
      c1 = r1;
      c2 = r2;
    }
    const BwdFn kern = f ? bwd_kernel<1, true>(c, b) : bwd_kernel<0, true>(c, b);
    if ((rc = bwd_ready(kern, f * 8 + 4 + c * 2 + b, BwdMem<true>::BYTES)) != KF_OK) return rc;
    const cudaError_t e = launch_maybe_pdl(p->Tk, kern, dim3(a.n_items < sms ? a.n_items : sms), dim3(PB_THREADS), BwdMem<true>::BYTES, st, r1, r2, r1, c1, c2, a);
    if (e != cudaSuccess) return cuda_status(e, "kf_attn_pack_bwd launch (keys)");
    if (a.split > 1) {
      const cudaError_t j = launch_maybe_pdl(p->Tk, f ? bwd_join_kernel<1> : bwd_join_kernel<0>, dim3(p->n_k_tiles * p->Hk, JOIN_CTAS), dim3(JOIN_THREADS), 0, st, a);
      if (j != cudaSuccess) return cuda_status(j, "kf_attn_pack_bwd launch (join)");
    }
  }
  return KF_OK;
}
