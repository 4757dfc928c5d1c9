// Attention forward over packed sequences (images or clips of different lengths behind one another), head dimension 64, on the sm_100a
// tensor cores.
//
//   s = scale * q . k;  with a cap: s = cap * tanh(s / cap);  with slopes: s -= slope(head) * |position of q - index of k|
//   a query sees keys [0, limit) of its own sequence (QTile::limit: all, or up to itself and the prefix); o = softmax(s) v over them,
//   lse = log sum exp(s); a query that sees nothing has o = 0 and lse = -inf
//
// The machine is that of the forward over equal images (kf_attn.cu: roles, S buffers in tensor memory, P over the first half of its S,
// key tiles of 96, the running maximum that is only looked for where a tile's row sum came out too large).  What differs:
//   - an item is a record of the host's table and a head; items have different numbers of key tiles, the longest first, and none is
//     possible: every role steps from item to item with its own cursor
//   - a tile may reach behind the end of its sequence: the scores there are masked one by one, the rows of V are set to zero in shared
//     memory by the warp that issues the products (P is 0 there, but 0 * NaN is not)
//   - with a cap or slopes the scores are brought to the exponent's scale in registers before the maximum
//   - with slopes the key tiles start at the one where the first query stands, go up to the last and then down to the first: scores mostly
//     fall with the distance, and a maximum that rises from tile to tile sends every tile down the slow path (200 queries behind 1605
//     keys, slope 1/16: 49 us in the keys' order)
//   - the polynomial exponential is a degree finer, for the log-sum-exp, and 0 for masked keys
//   - few items over long keys (SPLIT): a cluster of up to eight CTAs takes an item, each a share of the key tiles, and joins its parts through the
//     shared memory of its CTAs: accumulators, maxima and sums in fp32, in the order of the parts
// Measured (16 heads, bf16 unless noted): 8 x 1605 tokens 124.6 us (0.68 PFLOP/s), sizes of 1 to 4101 tokens 143, a causal clip of 8197 tokens in f16 187.  No unit is full
// (8 x 1605, cold: issue slots 50 %, exponential unit 53 %, FMA pipes 39 %, tensor cores 33 %): the two softmax warps of a scheduler wait for tensor memory and for
// their own instructions, one after the other in each step
#include <cfloat>
#include <type_traits>

#include "kf_attn.cuh"
#include "kf_sm100_pair.cuh"

namespace kf {

constexpr int PK_BM = 128, PK_BN = 96, PK_D = 64;
constexpr int PK_THREADS = 256;                        // warps 0..3 softmax, 4 TMA, 5 MMA issuer, 6 and 7 idle
constexpr int PK_REGS_SOFTMAX = 208, PK_REGS_LEAN = 48, PK_REGS = split_regs(128, PK_REGS_SOFTMAX, 128, PK_REGS_LEAN);
static_assert(2 * PK_THREADS * PK_REGS <= 65536, "two CTAs per SM");
constexpr int PK_KV = 3;
constexpr int PK_QTILE = PK_BM * PK_D * 2, PK_KTILE = PK_BN * PK_D * 2;
constexpr int PK_OFF_K = 2 * PK_QTILE, PK_OFF_V = PK_OFF_K + PK_KV * PK_KTILE, PK_OFF_BAR = PK_OFF_V + PK_KV * PK_KTILE;
constexpr size_t PK_SMEM = (size_t)PK_OFF_BAR + 256;
// P is 2^shift times the weight relative to the running maximum, which stays as it is while a tile's sum keeps to the limit (and with it each P to f16's range).  In f16
// weights far below the maximum would lose their digits (one key and 400 002 others that weigh as much together: 2.2 % off), and with 2^8 rows that start with few keys, as causal
// ones do, leave the limit too often (capped f16 clips 49.4 -> 53.4 us).
__host__ __device__ constexpr float pk_shift(int f16) { return f16 ? 6.f : 0.f; }
__host__ __device__ constexpr float pk_sum_limit(int f16) { return f16 ? 65504.f : 32768.f; }
constexpr int PK_POLY_K = 3;                           // element pairs PK_POLY_K .. 3 of every four take the polynomial exponential
constexpr int PK_SBUF = 2;
constexpr int PK_TMEM_COLS = 256, PK_COL_O = PK_SBUF * PK_BN;
static_assert(PK_COL_O + PK_D <= PK_TMEM_COLS, "TMEM budget");
// A split item: the CTAs of a cluster take a share of its key tiles each, leave their accumulators, maxima and sums in shared memory (where K and V
// were) and put a share of the rows together each.
constexpr int PK_PARTS = 8, PK_LD = PK_D + 4;             // rows of 68 floats: no two of eight neighbours in the same banks
constexpr int PK_OFF_PART = PK_OFF_K, PK_OFF_ML = PK_OFF_PART + PK_BM * PK_LD * 4;
static_assert(PK_OFF_ML + PK_BM * 8 <= PK_OFF_BAR, "a part's results take the place of K and V");

struct PackFwdArgs {
  void* O;
  int64_t o_st, o_sh;       // strides of O in elements
  float* lse;               // [Hq, lse_ld]
  int64_t lse_ld;
  const int4* tiles;        // QTile records
  int n_tiles, Hq, share;   // share = query heads per key head
  float scale_log2;         // scale * log2(e)
  Cap cap;
  const float* slopes;      // [Hq]
  int wide;                 // rows of O are 32-byte aligned
  int parts;                // CTAs per item (SPLIT)
  unsigned int* err;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <int F16, bool CAP, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(PK_THREADS, 2)
attn_pack_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ PackFwdArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PK_OFF_BAR);
  uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = k_full + PK_KV, *v_full = k_empty + PK_KV, *v_empty = v_full + PK_KV,
           *s_full = v_empty + PK_KV, *p_full = s_full + PK_SBUF, *o_full = p_full + PK_SBUF;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_full + PK_SBUF);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  pdl_launch_dependents();
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int items = a.n_tiles * a.Hq;
  const int n_my = SPLIT ? 1 : items_of_cta(items);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < PK_KV; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < PK_SBUF; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
    }
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_holder, PK_TMEM_COLS);
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
    a.err[1] = 110;
    a.err[2] = blockIdx.x;
  }
  const int rank = SPLIT ? (int)cluster_ctarank() : 0;
  auto item_at = [&](int it) { return SPLIT ? (int)blockIdx.x / a.parts : item_of_cta(it); };
  auto tile_of = [&](int it) { return load_tile<QTile>(a.tiles, item_at(it) / a.Hq); };
  auto head_of = [&](int it) { return item_at(it) % a.Hq; };
  auto all_tiles = [](const QTile& t) { return (t.limit(t.rows - 1) + PK_BN - 1) / PK_BN; };
  int all = 0, first = 0, mine = 0;                        // SPLIT: the item's key tiles and this CTA's of them, in the order of tile_at
  if constexpr (SPLIT) {
    all = all_tiles(tile_of(0));
    first = all * rank / a.parts;
    mine = all * (rank + 1) / a.parts - first;
  }
  auto key_tiles = [&](const QTile& t) { return SPLIT ? mine : all_tiles(t); };
  // the order of an item's n key tiles: from tile `start` up, then from the one in front of it down
  auto start_of = [&](const QTile& t, int n) {
    if (SPLIT) n = all;
    return !BIAS || t.pos < 0 ? 0 : t.pos / PK_BN < n ? t.pos / PK_BN : n - 1;
  };
  auto tile_at = [&](int i, int start, int n) {
    if (SPLIT) {
      i += first;
      n = all;
    }
    return !BIAS ? i : start + i < n ? start + i : n - 1 - i;
  };

  // every warp: the CTA's tensor memory goes back, behind the last access to it.  A part of an item says that it is done and gives it back before it waits for the others: a CTA
  // that held it meanwhile could stand against a cluster of another stream that holds the partner's SM.
  auto release = [&]() {
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && !bad_align) {
      for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
    if constexpr (SPLIT) {
      __syncwarp();
      cluster_arrive();
    }
    if (warp == 5) {
      tc_fence_after();
      tmem_dealloc(tmem_base, PK_TMEM_COLS);
    }
  };

  if (warp >= 4) {
  setmaxnreg_dec<PK_REGS_LEAN>();
  if (bad_align) {
    // nothing was issued; fall through to the teardown
  } else if (warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    uint32_t st = 0, ph = 1;
    bool ok = !__any_sync(0xffffffffu, *static_cast<volatile unsigned int*>(a.err) != 0u);   // has an earlier launch failed?
    if (!ok) *abort_flag = 1u;
    uint32_t qi = 0;                                                              // items with keys so far
    for (int it = 0; it < n_my && ok; ++it) {
      const QTile t = tile_of(it);
      const int n_kt = key_tiles(t), h = head_of(it), hk = h / a.share, start = start_of(t, n_kt);
      if (n_kt == 0) continue;
      const uint32_t qb = qi & 1;
      if (!mbar_wait_warp(&q_empty[qb], ((qi >> 1) & 1) ^ 1, ctx, 40)) break;
      if (elect_one()) {
        mbar_expect_tx(&q_full[qb], PK_QTILE);
        tma_load_3d(smem + qb * PK_QTILE, &tmQ, 0, h, t.row, &q_full[qb]);
      }
      __syncwarp();
      ++qi;
      for (int i = 0; i < n_kt; ++i) {
        const int key = t.k_row + tile_at(i, start, n_kt) * PK_BN;
        if (!mbar_wait_warp(&k_empty[st], ph, ctx, 41)) { ok = false; break; }
        if (elect_one()) {
          mbar_expect_tx(&k_full[st], PK_KTILE);
          tma_load_3d(smem + PK_OFF_K + st * PK_KTILE, &tmK, 0, hk, key, &k_full[st]);
        }
        __syncwarp();
        if (!mbar_wait_warp(&v_empty[st], ph, ctx, 42)) { ok = false; break; }
        if (elect_one()) {
          mbar_expect_tx(&v_full[st], PK_KTILE);
          tma_load_3d(smem + PK_OFF_V + st * PK_KTILE, &tmV, 0, hk, key, &v_full[st]);
        }
        __syncwarp();
        if (++st == PK_KV) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer: S(0), S(1), then PV(G) and S(G + 2) for every step
    const uint32_t idesc_s = idesc_f16(F16 ? 0u : 1u, PK_BN);
    const uint32_t idesc_o = idesc_f16(F16 ? 0u : 1u, PK_D) | (1u << 16);     // B (= V) is MN-major
    const uint32_t t_o = tmem_base + PK_COL_O;
    const bool leader = elect_one();
    struct Cursor {                                                          // a key tile of an item; items without keys are stepped over
      int it, next_n, next_len, next_start;                                  // the item behind this one: asked for ahead
      int j, n, k_len, start;                                                // n = -1: no item left
    };
    auto fetch = [&](Cursor& c) {
      c.next_n = -1;
      if (c.it < n_my) {
        const QTile t = tile_of(c.it++);
        c.next_n = key_tiles(t);
        c.next_len = t.k_len;
        c.next_start = start_of(t, c.next_n);
      }
    };
    auto open = [&](Cursor& c) {
      do {
        c.n = uniform_int(c.next_n);
        c.k_len = uniform_int(c.next_len);
        if (BIAS) c.start = uniform_int(c.next_start);
        fetch(c);
      } while (c.n == 0);
      c.j = 0;
    };
    auto advance = [&](Cursor& c) {
      if (++c.j == c.n) open(c);
    };
    Cursor s{};                                                              // the next S product
    fetch(s);
    open(s);
    Cursor v = s;                                                            // the next PV product
    uint32_t s_qi = 0, k_st = 0, k_ph = 0;
    auto issue_s = [&](uint32_t buf) {
      const uint64_t qdesc = smem_desc_sw128(smem_u32(smem + (s_qi & 1) * PK_QTILE));
      const uint64_t kdesc = smem_desc_sw128(smem_u32(smem + PK_OFF_K + k_st * PK_KTILE));
      const uint32_t t_s = tmem_base + buf * PK_BN;
      const bool last = s.j + 1 == s.n;
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < PK_D / 16; ++kk) mma_f16(t_s, qdesc + 2 * kk, kdesc + 2 * kk, idesc_s, kk != 0);
        tc_commit(&s_full[buf]);
        tc_commit(&k_empty[k_st]);
        if (last) tc_commit(&q_empty[s_qi & 1]);
      }
      __syncwarp();
      if (last) ++s_qi;
      advance(s);
      if (++k_st == PK_KV) {
        k_st = 0;
        k_ph ^= 1;
      }
    };
    bool ok = true;
    for (uint32_t G = 0; G < PK_SBUF && s.n > 0 && ok; ++G) {
      ok = (s.j != 0 || mbar_wait_warp(&q_full[s_qi & 1], (s_qi >> 1) & 1, ctx, 43)) && mbar_wait_warp(&k_full[k_st], k_ph, ctx, 44);
      tc_fence_after();
      if (ok) issue_s(G);
    }
    uint32_t buf = 0, pph = 0, st = 0, vph = 0;
    while (v.n > 0 && ok) {
      const bool more = s.n > 0;
      if (more && s.j == 0 && !mbar_wait_warp(&q_full[s_qi & 1], (s_qi >> 1) & 1, ctx, 43)) break;
      const int valid = v.k_len - tile_at(v.j, v.start, v.n) * PK_BN;                               // rows of this V tile that belong to the sequence
      if (valid < PK_BN) {
        if (!mbar_wait_warp(&v_full[st], vph, ctx, 45)) break;
        zero_rows(smem + PK_OFF_V + st * PK_KTILE, valid, PK_BN, lane);
      }
      if (more) {
        if (!mbar_wait_warp3(&p_full[buf], pph, &v_full[st], vph, &k_full[k_st], k_ph, ctx, 46)) break;
      } else {
        if (!mbar_wait_warp3(&p_full[buf], pph, &v_full[st], vph, &v_full[st], vph, ctx, 46)) break;
      }
      tc_fence_after();
      const uint32_t t_p = tmem_base + buf * PK_BN;
      const uint64_t vdesc = smem_desc_sw128(smem_u32(smem + PK_OFF_V + st * PK_KTILE));
      const uint32_t add = v.j != 0;
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < PK_BN / 16; ++kk)
          mma_f16_ta(t_o, t_p + 8 * kk, vdesc + (uint64_t)(kk * (2048 >> 4)), idesc_o, kk ? 1u : add);
        tc_commit(&o_full[buf]);
        tc_commit(&v_empty[st]);
      }
      __syncwarp();
      if (more) issue_s(buf);
      advance(v);
      if (++buf == PK_SBUF) {
        buf = 0;
        pph ^= 1;
      }
      if (++st == PK_KV) {
        st = 0;
        vph ^= 1;
      }
    }
  }
  } else {
    setmaxnreg_inc<PK_REGS_SOFTMAX>();
    if (!bad_align) {
    // ------------------------------------------------------------------ softmax: thread = query row
    const int row = warp * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(warp * 32) << 16);
    constexpr bool RAW = !CAP && !BIAS;                          // the registers hold raw products: the scale is applied with the maximum
    const float sc = RAW ? a.scale_log2 : 1.f;
    const float2 sc2 = splat2(sc);
    constexpr float SHIFT = pk_shift(F16);
    bool ok = true;
    uint32_t buf = 0, sph = 0;
    auto exp_half = [&](const uint32_t (&r)[32], uint32_t* w, float2 mn2, float2& s0, float2& s1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = make_float2(__uint_as_float(r[8 * i + 2 * k]), __uint_as_float(r[8 * i + 2 * k + 1]));
          const float2 t = RAW ? fma2(x, sc2, mn2) : add2(x, mn2);
          p[k] = k >= PK_POLY_K ? ex2_poly2_fine(t) : make_float2(ex2(t.x), ex2(t.y));
        }
        s0 = add2(s0, add2(p[0], p[1]));
        s1 = add2(s1, add2(p[2], p[3]));
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * i + k] = pack16(p[k].x, p[k].y, F16);
      }
    };
    auto row_max = [](const uint32_t (&r)[32], float mx) {
      float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 16; ++i) m4[i & 3] = max3(m4[i & 3], __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
      return amax_nan(amax_nan(m4[0], m4[1]), amax_nan(m4[2], m4[3]));
    };
    auto store32 = [&](uint8_t* dst, const uint32_t* w) {
      if (a.wide) {
        stg8w(dst, w);
      } else {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    };
    for (int it = 0; it < n_my && ok; ++it) {
    // little of the record lives through the key loop: where the rows go is looked up again behind it
    int n_kt, lim, warp_lim;                                     // lim: keys this row sees (-1: no row); warp_lim: the fewest of the warp's rows that exist
    float slope = 0.f;
    int start, at = 0;                                           // at: the row's position
    {
      const QTile tile = tile_of(it);
      n_kt = key_tiles(tile);
      lim = row < tile.rows ? tile.limit(row) : -1;
      warp_lim = tile.limit(warp * 32);
      start = start_of(tile, n_kt);
      if constexpr (BIAS) {
        slope = __ldg(a.slopes + head_of(it)) * 1.4426950408889634f;
        at = tile.pos + row;
      }
    }
    // raw products -> logits in units of the exponent, then the keys that the row does not see
    auto logits = [&](uint32_t (&r)[32], int key0) {
      if constexpr (!RAW) {
        const float gap = (float)(at - key0);                    // behind 2^24 only the difference is a number that fp32 holds
        bool flat = false;
        if constexpr (CAP) {
          float m4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 16; ++i) m4[i & 3] = max3(m4[i & 3], fabsf(__uint_as_float(r[2 * i])), fabsf(__uint_as_float(r[2 * i + 1])));
          flat = __all_sync(0xffffffffu, amax_nan(amax_nan(m4[0], m4[1]), amax_nan(m4[2], m4[3])) <= a.cap.flat);
        }
        auto each = [&](auto kind) {                             // 0: no cap, 1: small scores, 2: any
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 x = make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            if constexpr (decltype(kind)::value == 0) x = mul2(x, splat2(a.scale_log2));
            else if constexpr (decltype(kind)::value == 1) x = cap_flat(a.cap, x);
            else x = cap_any(a.cap, x);
            if constexpr (BIAS) {
              x.x = fmaf(-slope, fabsf(gap - (float)i), x.x);
              x.y = fmaf(-slope, fabsf(gap - (float)(i + 1)), x.y);
            }
            r[i] = __float_as_uint(x.x);
            r[i + 1] = __float_as_uint(x.y);
          }
        };
        if constexpr (!CAP) each(std::integral_constant<int, 0>{});
        else if (flat) each(std::integral_constant<int, 1>{});
        else each(std::integral_constant<int, 2>{});
      }
      if (key0 + 32 > warp_lim) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (key0 + i >= lim) r[i] = 0xff800000u;
      }
    };
    float m_run = 0.f, l_run = 0.f;
    uint32_t ra[32], rb[32], rc[32];                             // the S row of this step: keys 0..31, 32..63 and 64..95 of the tile
    if (n_kt > 0) {
      ok = mbar_wait_warp(&s_full[buf], sph, ctx, 47);
      if (!ok) break;
      tc_fence_after();
      tmem_ld32(t_lane + buf * PK_BN, ra);
      tmem_ld32(t_lane + buf * PK_BN + 32, rb);
      tmem_ld32(t_lane + buf * PK_BN + 64, rc);
    }
    for (int j = 0; j < n_kt; ++j) {
      const uint32_t t_s = t_lane + buf * PK_BN, cur = buf, cph = sph;
      if (++buf == PK_SBUF) {
        buf = 0;
        sph ^= 1;
      }
      const bool prefetch = j + 1 < n_kt;
      const int kbase = tile_at(j, start, n_kt) * PK_BN;
      tmem_ld_wait();
      tmem_ld_fence(ra);
      tmem_ld_fence(rb);
      tmem_ld_fence(rc);
      logits(ra, kbase);
      logits(rb, kbase + 32);
      logits(rc, kbase + 64);
      if (j == 0) {
        m_run = row_max(rb, row_max(ra, -INFINITY));
        if (!BIAS && m_run == -INFINITY) m_run = 0.f;            // a row that sees nothing
      }
      const bool unseen = BIAS && m_run == -INFINITY;            // none of its keys so far
      const float2 mn2 = splat2(unseen ? 0.f : fmaf(-m_run, sc, SHIFT));
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
      uint32_t w[48];
      exp_half(ra, w, mn2, s0, s1);
      const bool ready = mbar_test_wait(&s_full[buf], sph);
      exp_half(rb, w + 16, mn2, s0, s1);
      if (prefetch) {
        if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp(&s_full[buf], sph, ctx, 47)) { ok = false; break; }
        tc_fence_after();
        tmem_ld32(t_lane + buf * PK_BN, ra);
        tmem_ld32(t_lane + buf * PK_BN + 32, rb);
      }
      exp_half(rc, w + 32, mn2, s0, s1);
      if (prefetch) tmem_ld32(t_lane + buf * PK_BN + 64, rc);
      float sum = (s0.x + s0.y) + (s1.x + s1.y), alpha = 1.f;
      const bool need = lim >= 0 && (!(sum <= pk_sum_limit(F16)) || (unseen && lim > 0));   // rows that are not stored go on with whatever they have
      if (__any_sync(0xffffffffu, need)) {
        uint32_t r[32];
        float mx = m_run;
#pragma unroll 1
        for (int c = 0; c < PK_BN / 32; ++c) {
          tmem_ld32(t_s + 32 * c, r);
          tmem_ld_wait();
          tmem_ld_fence(r);
          logits(r, kbase + 32 * c);
          mx = row_max(r, mx);
        }
        if (need && !(BIAS && mx == -INFINITY)) {
          alpha = ex2((m_run - mx) * sc);
          m_run = mx;
        }
        const float2 mn = splat2(BIAS && m_run == -INFINITY ? 0.f : fmaf(-m_run, sc, SHIFT));
        s0 = s1 = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < PK_BN / 32; ++c) {
          tmem_ld32(t_s + 32 * c, r);
          tmem_ld_wait();
          tmem_ld_fence(r);
          logits(r, kbase + 32 * c);
          if (c == 0) exp_half(r, w, mn, s0, s1);
          else if (c == 1) exp_half(r, w + 16, mn, s0, s1);
          else exp_half(r, w + 32, mn, s0, s1);
        }
        sum = (s0.x + s0.y) + (s1.x + s1.y);
        if (j > 0) {                                             // rescale O: PV(G - 1) must have landed first
          const uint32_t pb = cur == 0 ? PK_SBUF - 1 : cur - 1;
          if (!mbar_wait_warp(&o_full[pb], cur == 0 ? cph ^ 1 : cph, ctx, 48)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            tmem_ld32(t_lane + PK_COL_O + 32 * c, r);
            tmem_ld_wait();
            tmem_ld_fence(r);
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st32(t_lane + PK_COL_O + 32 * c, r);
          }
        }
      }
      l_run = l_run * alpha + sum;
      tmem_st32(t_s, *reinterpret_cast<const uint32_t(*)[32]>(w));
      tmem_st16(t_s + 32, w + 32);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[cur]);
    }
    // the item's last PV product
    if (ok && n_kt > 0) ok = mbar_wait_warp(&o_full[buf == 0 ? PK_SBUF - 1 : buf - 1], buf == 0 ? sph ^ 1 : sph, ctx, 49);
    if (SPLIT && ok) {
      float* part = reinterpret_cast<float*>(smem + PK_OFF_PART) + row * PK_LD;
      if (n_kt > 0) tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32];
        if (n_kt > 0) {
          tmem_ld32(t_lane + PK_COL_O + 32 * c, r);
          tmem_ld_wait();
          tmem_ld_fence(r);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(part)[8 * c + i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
      }
      // a part of which the row sees nothing has no maximum
      const bool nothing = n_kt == 0 || (BIAS ? m_run == -INFINITY : lim <= first * PK_BN);
      reinterpret_cast<float2*>(smem + PK_OFF_ML)[row] = nothing ? make_float2(-INFINITY, 0.f) : make_float2(m_run * sc, l_run);
    }
    if (!SPLIT && ok) {
      uint32_t r0[32], r1[32];
      if (n_kt > 0) {
        tc_fence_after();
        tmem_ld32(t_lane + PK_COL_O, r0);
        tmem_ld32(t_lane + PK_COL_O + 32, r1);
        tmem_ld_wait();
        tmem_ld_fence(r0);
        tmem_ld_fence(r1);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) r0[i] = r1[i] = 0u;
      }
      if (lim >= 0) {
        const QTile tile = tile_of(it);
        const int h = head_of(it);
        const bool none = lim == 0;
        const float inv = 1.0f / l_run;
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          w[i] = pack16(__uint_as_float(r0[2 * i]) * inv, __uint_as_float(r0[2 * i + 1]) * inv, F16);
          w[16 + i] = pack16(__uint_as_float(r1[2 * i]) * inv, __uint_as_float(r1[2 * i + 1]) * inv, F16);
        }
        if (none) {
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0u;
        }
        uint8_t* dst = static_cast<uint8_t*>(a.O) + 2 * ((int64_t)(tile.row + row) * a.o_st + (int64_t)h * a.o_sh);
#pragma unroll
        for (int i = 0; i < 4; ++i) store32(dst + 32 * i, w + 8 * i);
        a.lse[(int64_t)h * a.lse_ld + tile.row + row] = none ? -INFINITY : (fmaf(m_run, sc, -SHIFT) + log2f(l_run)) * 0.6931471805599453f;
      }
    }
    }   // items
    if constexpr (SPLIT) {
      __syncwarp();
      release();
      cluster_wait();                                            // every part of the item lies in its CTA's shared memory
      const QTile tile = tile_of(0);
      const int h = head_of(0), r1 = PK_BM * (rank + 1) / a.parts;
      const uint32_t part0 = smem_u32(smem + PK_OFF_PART), ml0 = smem_u32(smem + PK_OFF_ML);
      for (int r = PK_BM * rank / a.parts + (int)(threadIdx.x >> 3); r < r1 && r < tile.rows; r += 16) {      // eight threads a row, eight channels each
        const int c = threadIdx.x & 7;
        float2 ml[PK_PARTS];
        float4 x[PK_PARTS], y[PK_PARTS];
#pragma unroll
        for (int p = 0; p < PK_PARTS; ++p) {
          ml[p] = make_float2(-INFINITY, 0.f);
          if (p < a.parts) {                                     // all on their way before the first is used
            const uint32_t at = map_addr(part0 + (r * PK_LD + c * 8) * 4, p);
            ml[p] = ld_cluster2(map_addr(ml0 + r * 8, p));
            x[p] = ld_cluster4(at);
            y[p] = ld_cluster4(at + 16);
          }
        }
        float m = -INFINITY, l = 0.f, o[8] = {};
#pragma unroll
        for (int p = 0; p < PK_PARTS; ++p) m = amax_nan(m, ml[p].x);
#pragma unroll
        for (int p = 0; p < PK_PARTS; ++p) {
          if (p < a.parts) {
            const float w = ml[p].x == -INFINITY ? 0.f : ex2(ml[p].x - m);
            l = fmaf(w, ml[p].y, l);
            o[0] = fmaf(w, x[p].x, o[0]); o[1] = fmaf(w, x[p].y, o[1]); o[2] = fmaf(w, x[p].z, o[2]); o[3] = fmaf(w, x[p].w, o[3]);
            o[4] = fmaf(w, y[p].x, o[4]); o[5] = fmaf(w, y[p].y, o[5]); o[6] = fmaf(w, y[p].z, o[6]); o[7] = fmaf(w, y[p].w, o[7]);
          }
        }
        const bool none = tile.limit(r) == 0;
        const float inv = 1.0f / l;
        const uint4 w = none ? make_uint4(0u, 0u, 0u, 0u)
                             : make_uint4(pack16(o[0] * inv, o[1] * inv, F16), pack16(o[2] * inv, o[3] * inv, F16), pack16(o[4] * inv, o[5] * inv, F16), pack16(o[6] * inv, o[7] * inv, F16));
        uint8_t* dst = static_cast<uint8_t*>(a.O) + 2 * ((int64_t)(tile.row + r) * a.o_st + (int64_t)h * a.o_sh);
        reinterpret_cast<uint4*>(dst)[c] = w;
        if (c == 0) a.lse[(int64_t)h * a.lse_ld + tile.row + r] = none ? -INFINITY : (m - pk_shift(F16) + log2f(l)) * 0.6931471805599453f;
      }
    }
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    if (warp >= 4 || bad_align) {                                // the softmax warps have been there
      release();
      __syncwarp();
      cluster_wait();
    }
    cluster_sync_all();                                          // nobody reads this CTA's shared memory any more
  } else {
    release();
  }
}

// Encoding costs about a microsecond of host time: kept per thread, direct-mapped by the arguments.
int make_tmap_heads(CUtensorMap* map, const void* base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride, int box_rows) {
  struct Slot {
    const void* base;
    int64_t rows, row_stride, head_stride;
    int heads, box_rows;
    CUtensorMap map;
  };
  constexpr int SLOTS = 64;
  static thread_local Slot cache[SLOTS] = {};
  const uintptr_t k = (reinterpret_cast<uintptr_t>(base) >> 4) * 0x9E3779B97F4A7C15ull + (uintptr_t)rows * 31 + (uintptr_t)row_stride * 7 + (uintptr_t)box_rows;
  Slot& slot = cache[(k >> 32 ^ k) % SLOTS];
  if (slot.base == base && slot.rows == rows && slot.row_stride == row_stride && slot.head_stride == head_stride && slot.heads == heads && slot.box_rows == box_rows) {
    *map = slot.map;
    return KF_OK;
  }
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return KF_ERR_UNSUPPORTED;
  }
  cuuint64_t dims[3] = {64, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled (heads) failed with CUresult %d", (int)r);
    return KF_ERR_BAD_ARGUMENT;
  }
  slot = Slot{base, rows, row_stride, head_stride, heads, box_rows, *map};
  return KF_OK;
}

// A [rows, heads, 64] operand as the copies and the stores take it: 16-byte aligned, strides in whole 16-byte units; what has one row or
// head gets a stride that means nothing.
int check_heads(const char* what, const kf_heads& t, int64_t rows, int heads, kf_heads* out) {
  *out = t;
  if (heads == 1) out->head_stride = 64;
  if (rows == 1) out->row_stride = (int64_t)64 * heads;
  KF_REQUIRE(t.ptr && (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0, "kf_attn_pack: %s must be non-null and 16-byte aligned", what);
  KF_REQUIRE(out->row_stride >= 64 && out->head_stride >= 64 && out->row_stride % 8 == 0 && out->head_stride % 8 == 0 && out->row_stride < (1ll << 38) &&
                 out->head_stride < (1ll << 38),
             "kf_attn_pack: strides of %s (%lld, %lld elements) must be multiples of 8, 64 at least", what, (long long)t.row_stride, (long long)t.head_stride);
  return KF_OK;
}

int check_pack(const kf_attn_pack_params* p) {
  KF_REQUIRE(p, "kf_attn_pack: null parameter block");
  KF_REQUIRE(p->dtype == KF_BF16 || p->dtype == KF_F16, "kf_attn_pack: dtype must be bf16 or f16");
  KF_REQUIRE(p->Hq > 0 && p->Hk > 0 && p->Hq % p->Hk == 0, "kf_attn_pack: %d query heads do not share %d key heads evenly", p->Hq, p->Hk);
  KF_REQUIRE(p->Tq >= 0 && p->Tk >= 0 && p->Tq < (1ll << 31) - 256 && p->Tk < (1ll << 31) - 256, "kf_attn_pack: bad numbers of rows");
  KF_REQUIRE(p->n_q_tiles >= 0 && p->n_k_tiles >= 0 && (int64_t)p->n_q_tiles * p->Hq < (1ll << 30) && (int64_t)p->n_k_tiles * p->Hk < (1ll << 30),
             "kf_attn_pack: too many (tile, head) items");
  KF_REQUIRE(p->scale > 0.f && p->scale < 1e30f && p->cap >= 0.f && p->cap < 1e30f, "kf_attn_pack: scale must be positive and cap not negative, both finite");
  // what Cap::set makes of them: fp32 numbers with all their digits (an infinity would meet scores of 0)
  KF_REQUIRE(p->cap == 0.f || (p->cap >= FLT_MIN && 2.9 * p->scale / p->cap < FLT_MAX), "kf_attn_pack: cap %g with scale %g leaves fp32's range", p->cap, p->scale);
  return KF_OK;
}

}  // namespace kf

using namespace kf;

// CTAs per item: more than one where the items leave room for them and the longest has three tiles or more for each.  The join costs about 3 us (32 KB per
// part and item pass between SMs), a tile 0.8 us: 4 items of 128 queries on 1029 keys (11 tiles) 12.4 us unsplit, 11.9 / 10.1 / 9.2 / 9.6 / 9.3 in 2 / 3 / 4 / 5 / 6
// parts; 8 items on 517 keys (6 tiles) 8.6 unsplit, 9.8 / 8.7 in 2 / 3; 24 items on 8197 keys 74 unsplit, 23 in 8
static int fwd_parts(int64_t items, int longest, int slots) {
  const int64_t tiles = (longest + PK_BN - 1) / PK_BN, room = slots / items;
  const int64_t most = tiles < 9 ? 1 : tiles / 3 < room ? tiles / 3 : room;
  return most < 2 ? 1 : most < PK_PARTS ? (int)most : PK_PARTS;
}

extern "C" int kf_attn_pack_fwd(const kf_attn_pack_params* p, void* stream) {
  int rc = check_pack(p);
  if (rc != KF_OK) return rc;
  if (p->n_q_tiles == 0) return KF_OK;
  KF_REQUIRE(p->Tq > 0 && p->q_tiles && p->lse, "kf_attn_pack_fwd: null pointer");
  kf_heads q, k, v, o;
  if ((rc = check_heads("q", p->q, p->Tq, p->Hq, &q)) != KF_OK) return rc;
  if ((rc = check_heads("o", p->o, p->Tq, p->Hq, &o)) != KF_OK) return rc;
  k = v = q;
  int k_heads = p->Hq;
  int64_t k_rows = p->Tq;
  if (p->Tk > 0) {                                            // without keys at all the maps are never used
    if ((rc = check_heads("k", p->k, p->Tk, p->Hk, &k)) != KF_OK) return rc;
    if ((rc = check_heads("v", p->v, p->Tk, p->Hk, &v)) != KF_OK) return rc;
    k_heads = p->Hk;
    k_rows = p->Tk;
  }
  CUtensorMap tq, tk, tv;
  if ((rc = make_tmap_heads(&tq, q.ptr, p->Tq, p->Hq, q.row_stride, q.head_stride, PK_BM)) != KF_OK) return rc;
  if ((rc = make_tmap_heads(&tk, k.ptr, k_rows, k_heads, k.row_stride, k.head_stride, PK_BN)) != KF_OK) return rc;
  if ((rc = make_tmap_heads(&tv, v.ptr, k_rows, k_heads, v.row_stride, v.head_stride, PK_BN)) != KF_OK) return rc;
  using KernelFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, PackFwdArgs);
  int sms = 0;
  if ((rc = device_sm_count(&sms)) != KF_OK) return rc;
  const int64_t items = (int64_t)p->n_q_tiles * p->Hq;
  const int parts = fwd_parts(items, p->longest, 2 * sms);    // two CTAs are resident per SM
  static const KernelFn table[2][2][2][2] = {
      {{{attn_pack_fwd_kernel<0, false, false, false>, attn_pack_fwd_kernel<0, false, false, true>}, {attn_pack_fwd_kernel<0, false, true, false>, attn_pack_fwd_kernel<0, false, true, true>}},
       {{attn_pack_fwd_kernel<0, true, false, false>, attn_pack_fwd_kernel<0, true, false, true>}, {attn_pack_fwd_kernel<0, true, true, false>, attn_pack_fwd_kernel<0, true, true, true>}}},
      {{{attn_pack_fwd_kernel<1, false, false, false>, attn_pack_fwd_kernel<1, false, false, true>}, {attn_pack_fwd_kernel<1, false, true, false>, attn_pack_fwd_kernel<1, false, true, true>}},
       {{attn_pack_fwd_kernel<1, true, false, false>, attn_pack_fwd_kernel<1, true, false, true>}, {attn_pack_fwd_kernel<1, true, true, false>, attn_pack_fwd_kernel<1, true, true, true>}}}};
  const int f = p->dtype == KF_F16, c = p->cap > 0.f, b = p->slopes != nullptr, s = parts > 1;
  const KernelFn kern = table[f][c][b][s];
  static PerDevice<bool> ready[2][2][2][2];
  if ((rc = split_ready(reinterpret_cast<const void*>(kern), ready[f][c][b][s], PK_REGS, PK_SMEM, "kf_attn_pack_fwd")) != KF_OK) return rc;
  constexpr float LOG2E = 1.4426950408889634f;
  PackFwdArgs a{};
  a.O = o.ptr; a.o_st = o.row_stride; a.o_sh = o.head_stride; a.lse = p->lse; a.lse_ld = p->Tq;
  a.tiles = reinterpret_cast<const int4*>(p->q_tiles); a.n_tiles = p->n_q_tiles; a.Hq = p->Hq; a.share = p->Hq / p->Hk;
  a.scale_log2 = p->scale * LOG2E;
  if (c) a.cap.set(p->scale, p->cap);
  a.slopes = p->slopes;
  a.wide = ((reinterpret_cast<uintptr_t>(o.ptr) | (uintptr_t)(o.row_stride * 2) | (uintptr_t)(o.head_stride * 2)) & 31) == 0;
  a.err = dev_error_ptr();
  KF_REQUIRE(a.err != nullptr, "kf_attn_pack_fwd: device error word unavailable");
  a.parts = parts;
  const int grid = parts > 1 ? (int)items * parts : items < 2 * sms ? (int)items : 2 * sms;
  return cuda_status(launch_maybe_pdl_cluster(p->Tq, parts, kern, dim3(grid), dim3(PK_THREADS), PK_SMEM, static_cast<cudaStream_t>(stream), tq, tk, tv, a),
                     "kf_attn_pack_fwd launch");
}
