// Causal softmax attention forward over packed sequences with grouped heads.
//
//   o_i = sum_{j <= i} p_ij v_j,  p_i = softmax_j(scale q_i . k_j)
// within each sequence, in one pass over its keys with the running row maximum
// and sum.  lse2 = max + log2(sum) per row (log2 units) is kept for the backward.
//
// One CTA = one query tile of the plan (tt tokens x p heads, 128 rows), two
// CTAs per SM, so one CTA's MMAs run under the other's exponentials.  Warp 0
// brings in Q once and K, V through TMA rings; warp 1 issues S = Q K^T and
// O += P V with P read from TMEM; warps 2..5 run the softmax, one row per
// thread.  TMEM (256 columns): HD = 64 keeps P in columns of its own and takes
// S in two 64-key halves, so the next tile's scores are computed under this
// tile's exponentials; HD = 128 writes P over S.
//
// Rows of other sequences never reach a result: the last key tile's V rows past
// the sequence's end are cleared in shared memory (their P is zero, but zero
// times an inf or NaN is not), and so are the inf or NaN elements of V in the
// tile's masked triangle, which are added back to the rows that do see them.
#include "attn_packed.h"
#include "attn_packed.cuh"

namespace mea {

struct PackedFwdParams {
  PackedDims d;
  PackedPlan plan;
  float scale_log2;  // scale * log2(e)
  const void* v;     // the map's tensor, for the rows with inf or NaN
  long long v_tok, v_head;
  void* o;      // [total, Hq, N]
  float* lse2;  // [total, Hq]
  int* status;
};
struct PackedFwdMaps {
  CUtensorMap q, k, v;
};

template <int HD>
struct PackedFwdCfg {
  static constexpr int KS = HD <= 64 ? 2 : 1, VS = KS;  // K and V ring depth
  static constexpr uint32_t TB = 128 * HD * 2;
  static constexpr bool SEP_P = HD <= 64;
  static constexpr uint32_t S_COL = 0, P_COL = SEP_P ? 128 : 0, O_COL = SEP_P ? 192 : 128;
  static constexpr uint32_t TMEM_COLS = 256;
  static constexpr uint32_t OFF_BAR = TB * (1 + KS + VS);
  static constexpr size_t SMEM = 1024 + OFF_BAR + 256;
};

// Row maximum (NaN if any score is) of 128 raw scores in TMEM; MASK drops columns > cmax.
template <bool MASK>
__device__ __forceinline__ float packed_row_max(uint32_t sb, int cmax) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  auto chunk = [&](const uint32_t(&v)[16], int c) {
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = (MASK && 16 * c + e > cmax) ? -INFINITY : __uint_as_float(v[e]);
#pragma unroll
    for (int e = 0; e < 16; e += 8)
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = max3f_nan(m[i], x[e + 2 * i], x[e + 2 * i + 1]);
  };
  uint32_t a[16], b[16];
  tmem_ld16(sb, a);
  tmem_wait_ld_tied(a);
#pragma unroll
  for (int c = 0; c < 8; c += 2) {
    tmem_ld16(sb + 16 * (c + 1), b);
    chunk(a, c);
    tmem_wait_ld_tied(b);
    if (c + 2 < 8) tmem_ld16(sb + 16 * (c + 2), a);
    chunk(b, c + 1);
    if (c + 2 < 8) tmem_wait_ld_tied(a);
  }
  return max3f_nan(max3f_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// P = exp2(s * sl2 - m) of the 64 columns [col0, col0 + 64): packed pairs
// through out(c, pk) per 16-column chunk c; returns their sum.
template <class T, bool MASK, class Out>
__device__ __forceinline__ float packed_exp64(uint32_t sb, int col0, int cmax, float sl2, float neg_m, Out&& out) {
  float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
  const float2 scale2 = make_float2(sl2, sl2), bias2 = make_float2(neg_m, neg_m);
  auto chunk = [&](const uint32_t(&v)[16], int c) {
    uint32_t pk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 t = ffma2(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale2, bias2);
      float2 pp = exp2_pair(t, (kPolyPairsFwd >> e) & 1);
      if (MASK) {
        const int c0 = col0 + 16 * c + 2 * e;
        pp.x = c0 > cmax ? 0.f : pp.x;
        pp.y = c0 + 1 > cmax ? 0.f : pp.y;
      }
      if (e & 1)
        acc1 = fadd2(acc1, pp);
      else
        acc0 = fadd2(acc0, pp);
      pk[e] = T::pack(pp.x, pp.y);
    }
    out(c, pk);
  };
  uint32_t a[16], b[16];
  tmem_ld16(sb + col0, a);
  tmem_wait_ld_tied(a);
#pragma unroll
  for (int c = 0; c < 4; c += 2) {
    tmem_ld16(sb + col0 + 16 * (c + 1), b);
    chunk(a, c);
    tmem_wait_ld_tied(b);
    if (c + 2 < 4) tmem_ld16(sb + col0 + 16 * (c + 2), a);
    chunk(b, c + 1);
    if (c + 2 < 4) tmem_wait_ld_tied(a);
  }
  return (acc0.x + acc0.y) + (acc1.x + acc1.y);
}

// Clears the inf and NaN elements of rows [r0, r1) of a V tile (one warp); true if there were any.
template <int HD, class T>
__device__ __forceinline__ bool clear_nonfinite(uint32_t tile, int r0, int r1, int lane) {
  uint32_t acc = 0;
  const int units = r1 > r0 ? (r1 - r0) * 8 : 0;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c)
    for (int u = lane; u < units; u += 32) {
      uint32_t w[4];
      lds128(tile + c * 16384 + r0 * 128 + u * 16, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) T::probe(acc, w[i]);
    }
  const bool mine = half_nonfinite<T>(acc) || half_nonfinite<T>(acc >> 16);
  if (!__any_sync(0xffffffffu, mine)) return false;
  for (int c = 0; c < HD / 64; ++c)
    for (int u = lane; u < units; u += 32) {
      const uint32_t at = tile + c * 16384 + r0 * 128 + u * 16;
      uint32_t w[4];
      lds128(at, w);
      for (int i = 0; i < 4; ++i) {
        if (half_nonfinite<T>(w[i])) w[i] &= 0xFFFF0000u;
        if (half_nonfinite<T>(w[i] >> 16)) w[i] &= 0x0000FFFFu;
      }
      sts128(at, w[0], w[1], w[2], w[3]);
    }
  return true;
}

template <int HD, class T>
__global__ void __launch_bounds__(192, 2) packed_fwd_kernel(const __grid_constant__ PackedFwdMaps maps,
                                                            const __grid_constant__ PackedFwdParams p) {
  using Cfg = PackedFwdCfg<HD>;
  using Tile = HeadTile<HD>;
  constexpr int KS = Cfg::KS, VS = Cfg::VS;
  constexpr uint32_t TB = Cfg::TB;
  constexpr uint32_t IDESC_S = idesc_16bit(T::FMT, 128, 128, 0, 0);
  constexpr uint32_t IDESC_SH = idesc_16bit(T::FMT, 128, 64, 0, 0);  // (SEP_P) one 64-key half of S
  constexpr uint32_t IDESC_O = idesc_16bit(T::FMT, 128, HD, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sQ = smem_u32(smem);
  const uint32_t sK = sQ + TB;       // KS K tiles
  const uint32_t sV = sK + KS * TB;  // VS V tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  const uint32_t b0 = smem_u32(bars);
  const uint32_t q_full = b0;
  auto k_full = [&](int s) { return b0 + 8u * (1 + s); };
  auto k_empty = [&](int s) { return b0 + 8u * (1 + KS + s); };
  auto v_full = [&](int s) { return b0 + 8u * (1 + 2 * KS + s); };
  auto v_empty = [&](int s) { return b0 + 8u * (1 + 2 * KS + VS + s); };
  const uint32_t s_full = b0 + 8u * (1 + 2 * KS + 2 * VS);  // S_j (SEP_P: its keys [0, 64)) computed
  const uint32_t p_full = s_full + 8;                        // P_j written
  const uint32_t o_bar = s_full + 16;                        // every MMA done
  const uint32_t drain_bar = s_full + 24;
  const uint32_t s_empty = s_full + 32;    // (SEP_P) the softmax has read the half [0, 64)
  const uint32_t pv_done = s_full + 40;    // (SEP_P) PV_j done
  const uint32_t s_full_b = s_full + 48;   // (SEP_P) the half [64, 128)
  const uint32_t s_empty_b = s_full + 56;
  const uint32_t v_raw = s_full + 64;      // a V tile that warp 0 looks over before the MMA may read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 1 + 2 * KS + 2 * VS + 9);
  uint32_t* bad_slot = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 128);
    mbar_init(o_bar, 1);
    mbar_init(drain_bar, 1);
    mbar_init(s_empty, 128);
    mbar_init(pv_done, 1);
    mbar_init(s_full_b, 1);
    mbar_init(s_empty_b, 128);
    mbar_init(v_raw, 1);
    *bad_slot = 0;
    fence_mbar_init();
  }
  pdl_wait();

  const PackedHeader hd = *p.plan.head;
  zero_outside(static_cast<uint4*>(p.o), p.d.total, hd.first, hd.end, (long long)p.d.Hq * p.d.N / 8, blockIdx.x,
               gridDim.x, threadIdx.x, blockDim.x);
  if (int(blockIdx.x) / p.d.hg >= hd.n_q) return;
  const PackedTile<true> item(p.plan.q_items, blockIdx.x, p.d.hg, p.d.tt);
  const int h0 = item.head * p.d.p;  // first head
  const int kvh = h0 / (p.d.Hq / p.d.Hkv);
  const int seq0 = item.seq0, len = item.len;
  const int t0 = item.tile * p.d.tt;
  const int t1 = min(t0 + p.d.tt, len);
  const int nkv = (t1 + 127) >> 7;

  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Guard g(p.status, KID_PACKED_FWD);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    const bool lead = lane == 0;
    if (lead) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
      mbar_expect_tx(q_full, uint32_t(p.d.p * p.d.tt) * 128 * Tile::NCHUNK);
#pragma unroll
      for (int c = 0; c < Tile::NCHUNK; ++c) tma_load_3d(sQ + c * 16384, &maps.q, q_full, c * 64, h0, seq0 + t0);
    }
    int kpar[KS], vpar[VS];
    for (int s = 0; s < KS; ++s) kpar[s] = -1;
    for (int s = 0; s < VS; ++s) vpar[s] = -1;
    int raw = 0;  // uses of v_raw
    for (int j = 0; j < nkv && g.ok; ++j) {
      const int sk = j % KS, sv = j % VS;
      const uint32_t pk = (j / KS) & 1, pv = (j / VS) & 1;
      // Rows [from, to) of this V tile are masked for some rows of the query
      // tile only, rows [to, 128) for all of them.
      const int from = max(t0 + 1 - 128 * j, 0), to = min(t1 - 128 * j, 128);
      const bool look = from < 128;
      if (lead) {
        if (mbar_wait(k_empty(sk), pk ^ 1, g, 1)) {
          mbar_expect_tx(k_full(sk), TB);
#pragma unroll
          for (int c = 0; c < Tile::NCHUNK; ++c)
            tma_load_3d(sK + sk * TB + c * 16384, &maps.k, k_full(sk), c * 64, kvh, seq0 + j * 128);
          kpar[sk] = int(pk);
        }
        if (mbar_wait(v_empty(sv), pv ^ 1, g, 9)) {
          const uint32_t full = look ? v_raw : v_full(sv);
          mbar_expect_tx(full, TB);
#pragma unroll
          for (int c = 0; c < Tile::NCHUNK; ++c)
            tma_load_3d(sV + sv * TB + c * 16384, &maps.v, full, c * 64, kvh, seq0 + j * 128);
          vpar[sv] = int(pv);
        }
      }
      g.ok = __all_sync(0xffffffffu, g.ok);
      if (look && g.ok) {
        g.ok = __all_sync(0xffffffffu, mbar_wait(v_raw, raw & 1, g, 13));
        ++raw;
        if (!g.ok) break;
        zero_rows<HD>(sV + sv * TB, to, lane);
        if (clear_nonfinite<HD, T>(sV + sv * TB, from, to, lane) && lead) *bad_slot = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lead) mbar_arrive(v_full(sv));
      }
    }
    if (lead) {
      if (!g.ok) {
        mbar_drain(q_full, 0);
        for (int s = 0; s < KS; ++s)
          if (kpar[s] >= 0) mbar_drain(k_full(s), uint32_t(kpar[s]));
        for (int s = 0; s < VS; ++s)
          if (vpar[s] >= 0) mbar_drain(v_full(s), uint32_t(vpar[s]));
        mbar_drain(v_raw, uint32_t(raw & 1));
      } else {
        // The MMA warp's last releases have landed before this CTA's shared memory goes away.
        for (int s = 0; s < KS; ++s)
          if (kpar[s] >= 0) mbar_wait(k_empty(s), uint32_t(kpar[s]), g, 14);
        for (int s = 0; s < VS; ++s)
          if (vpar[s] >= 0) mbar_wait(v_empty(s), uint32_t(vpar[s]), g, 15);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      bool any = false;
      auto issue_pv = [&](int j) {
        const int sv = j % VS;
#pragma unroll
        for (int kc = 0; kc < 8; ++kc)
          mma_ts(tmem + Cfg::O_COL, tmem + Cfg::P_COL + kc * 8, Tile::mnmajor(sV + sv * TB, 128, kc), IDESC_O,
                 (j > 0 || kc > 0) ? 1u : 0u);
        mma_commit(v_empty(sv));
      };
      if constexpr (Cfg::SEP_P) {
        auto issue_half = [&](int j, int hf) {
          const int sk = j % KS;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + Cfg::S_COL + 64 * hf, Tile::kmajor(sQ, 128, kk),
                   Tile::kmajor(sK + sk * TB + hf * 64 * Tile::SWB, 128, kk), IDESC_SH, kk > 0 ? 1u : 0u);
          if (hf) mma_commit(k_empty(sk));
          mma_commit(hf ? s_full_b : s_full);
        };
        if (mbar_wait(q_full, 0, g, 5) && mbar_wait(k_full(0), 0, g, 2)) {
          tc_fence_after();
          issue_half(0, 0);
          issue_half(0, 1);
          any = true;
          for (int j = 0; j < nkv; ++j) {
            if (j + 1 < nkv) {  // each half of S_{j+1} as soon as that half of S_j has been read
              if (!mbar_wait(s_empty, j & 1, g, 10)) break;
              if (!mbar_wait(k_full((j + 1) % KS), ((j + 1) / KS) & 1, g, 2)) break;
              tc_fence_after();
              issue_half(j + 1, 0);
              if (!mbar_wait(s_empty_b, j & 1, g, 16)) break;
              tc_fence_after();
              issue_half(j + 1, 1);
            }
            if (!mbar_wait(p_full, j & 1, g, 3)) break;
            if (!mbar_wait(v_full(j % VS), (j / VS) & 1, g, 4)) break;
            tc_fence_after();
            issue_pv(j);
            mma_commit(pv_done);
          }
          if (g.ok) mma_commit(o_bar);
        }
      } else if (mbar_wait(q_full, 0, g, 5)) {
        for (int j = 0; j < nkv; ++j) {
          const int sk = j % KS;
          if (!mbar_wait(k_full(sk), (j / KS) & 1, g, 2)) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + Cfg::S_COL, Tile::kmajor(sQ, 128, kk), Tile::kmajor(sK + sk * TB, 128, kk), IDESC_S,
                   kk > 0 ? 1u : 0u);
          mma_commit(k_empty(sk));
          mma_commit(s_full);
          any = true;
          if (!mbar_wait(p_full, j & 1, g, 3)) break;
          if (!mbar_wait(v_full(j % VS), (j / VS) & 1, g, 4)) break;
          tc_fence_after();
          issue_pv(j);
        }
        if (g.ok) mma_commit(o_bar);
      }
      if (!g.ok && any) {
        mma_commit(drain_bar);
        mbar_drain(drain_bar, 0);
      }
    }
  } else {
    // ---------------- softmax + epilogue: warps 2..5 ----------------
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the query tile
    const int t = t0 + r / p.d.p;       // token within the sequence
    const bool live = r < p.d.p * p.d.tt && t < t1;
    const uint32_t lane_base = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t sb = lane_base + Cfg::S_COL;
    const float sl2 = p.scale_log2;
    float m_run = -INFINITY, l_run = 0.f;  // m_run in scaled log2 units
    bool ok = true, nan_row = false;
    // Takes S_j's row maximum mx (raw) into the running maximum.  Lazy: the
    // reference moves only when the maximum grows by more than 8 (log2 units), so
    // P stays <= 2^8; O and the sum are rescaled only then.  `o_ready` makes O stable.
    auto rescale = [&](float mx_raw, int j, auto&& o_ready) {
      const float mx = mx_raw * sl2;
      nan_row |= mx != mx;
      const bool need = mx > m_run + 8.0f || (m_run == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, need)) {
        const float m_new = need ? mx : m_run;
        const float alpha = need ? ex2(m_run - m_new) : 1.0f;  // 0 when m_run = -inf
        if (j > 0) {
          if (!o_ready()) return;
#pragma unroll
          for (int c = 0; c < HD; c += 16) {
            uint32_t ov[16];
            tmem_load16(lane_base + Cfg::O_COL + c, ov);
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st16(lane_base + Cfg::O_COL + c, ov);
          }
        }
        l_run *= alpha;
        m_run = m_new;
      }
    };
    for (int j = 0; j < nkv && ok; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(s_full, j & 1, g, 6));
      if (!ok) break;
      const bool mask = 128 * j + 127 > t0;
      const int cmax = t - 128 * j;  // last column this row sees
      if constexpr (Cfg::SEP_P) {
        ok = __all_sync(0xffffffffu, mbar_wait(s_full_b, j & 1, g, 17));
        if (!ok) break;
        tc_fence_after();
        bool pv_seen = (j == 0);  // PV_{j-1} has completed: O and the P columns are free
        auto wait_pv = [&]() -> bool {
          ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (j - 1) & 1, g, 11));
          if (ok) tc_fence_after();
          pv_seen = true;
          return ok;
        };
        rescale(mask ? packed_row_max<true>(sb, cmax) : packed_row_max<false>(sb, cmax), j, wait_pv);
        if (!ok) break;
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
        // Keys [0, 64), then [64, 128): one loop, so the exponential code exists once per mask.
#pragma unroll 1
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t pk[32];
          auto keep = [&](int c, const uint32_t(&w)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[8 * c + e] = w[e];
          };
          l_run += mask ? packed_exp64<T, true>(sb, 64 * hh, cmax, sl2, neg_m, keep)
                        : packed_exp64<T, false>(sb, 64 * hh, cmax, sl2, neg_m, keep);
          tc_fence_before();
          mbar_arrive(hh ? s_empty_b : s_empty);
          if (!pv_seen && !wait_pv()) break;
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2)
            tmem_st16(lane_base + Cfg::P_COL + 32 * hh + 16 * q2, *reinterpret_cast<const uint32_t(*)[16]>(pk + 16 * q2));
          tmem_st_wait();  // the next half rewrites the registers of pk
        }
        if (!ok) break;
      } else {
        tc_fence_after();
        // S_j was issued after PV_{j-1} on the in-order tensor pipe: O is stable.
        rescale(mask ? packed_row_max<true>(sb, cmax) : packed_row_max<false>(sb, cmax), j, [] { return true; });
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll 1
        for (int hh = 0; hh < 2; ++hh) {
          auto store = [&](int c, const uint32_t(&w)[8]) { tmem_st8(sb + 32 * hh + 8 * c, w); };
          l_run += mask ? packed_exp64<T, true>(sb, 64 * hh, cmax, sl2, neg_m, store)
                        : packed_exp64<T, false>(sb, 64 * hh, cmax, sl2, neg_m, store);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(p_full);
    }
    // ---- epilogue: O / l ----
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_bar, 0, g, 8));
    if (ok && Cfg::SEP_P) ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (nkv - 1) & 1, g, 12));
    if (ok) {
      tc_fence_after();
      const bool bad = *reinterpret_cast<volatile uint32_t*>(bad_slot) != 0;
      nan_row |= m_run == -INFINITY;  // no finite score: 0 / 0
      const float inv_l = nan_row ? __int_as_float(0x7fffffff) : 1.0f / l_run;
      const int h = h0 + r % p.d.p;
      const long long row = (long long)(seq0 + t) * p.d.Hq + h;
      uint16_t* orow = static_cast<uint16_t*>(p.o) + row * p.d.N;
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t ov[16];
        __syncwarp();
        tmem_load16(lane_base + Cfg::O_COL + c, ov);
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(ov[e]) * inv_l;
        if (bad && live) {  // the inf and NaN elements that were cleared, for the rows that see them
          for (int key = t0 + 1; key <= t; ++key) {
            const uint16_t* vr = static_cast<const uint16_t*>(p.v) + (long long)(seq0 + key) * p.v_tok + kvh * p.v_head;
            for (int e = 0; e < 16; ++e)
              if (c + e < p.d.N && half_nonfinite<T>(vr[c + e])) f[e] += T::lo(vr[c + e]);
          }
        }
        if (live) {
          if (c < p.d.N)
            st_global_v4(orow + c, T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7]));
          if (c + 8 < p.d.N)
            st_global_v4(orow + c + 8, T::pack(f[8], f[9]), T::pack(f[10], f[11]), T::pack(f[12], f[13]),
                         T::pack(f[14], f[15]));
        }
      }
      if (live) p.lse2[row] = nan_row ? __int_as_float(0x7fffffff) : m_run + __log2f(l_run);
    }
    if (!ok) g.ok = false;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

template <int HD, class T>
static int launch_packed_fwd(const PackedFwdMaps& maps, const PackedFwdParams& p, cudaStream_t st) {
  using Cfg = PackedFwdCfg<HD>;
  auto kern = packed_fwd_kernel<HD, T>;
  if (!smem_attr_set(reinterpret_cast<const void*>(kern), int(Cfg::SMEM)))
    return set_error(MEA_ERR_CUDA, "cudaFuncSetAttribute(packed_fwd) failed");
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = packed_launch(p.d.cap_q * p.d.hg, 192, Cfg::SMEM, st, &attr);
  cudaLaunchKernelEx(&cfg, kern, maps, p);
  return check_launch("packed_fwd_kernel");
}

}  // namespace mea

extern "C" int mea_packed_attention_forward(const mea_packed_dims* d, const void* q, const void* k, const void* v,
                                            const int* cu_seqlens, void* o, float* lse2, void* plan, size_t plan_bytes,
                                            int* status, void* stream) {
  using namespace mea;
  PackedDims pd;
  int rc = packed_dims(d, &pd);
  if (rc != MEA_OK) return rc;
  if (pd.total == 0) return MEA_OK;
  if ((rc = packed_check_rows("q", q, d->q_row, d->q_head, pd, pd.Hq)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("k", k, d->k_row, d->k_head, pd, pd.Hkv)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("v", v, d->v_row, d->v_head, pd, pd.Hkv)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("o", o, (long long)pd.Hq * pd.N, pd.N, pd, pd.Hq)) != MEA_OK) return rc;
  if (!cu_seqlens || !lse2 || !plan)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: cu_seqlens, lse2 and plan must be non-NULL");
  if ((reinterpret_cast<uintptr_t>(cu_seqlens) | reinterpret_cast<uintptr_t>(lse2)) & 3 ||
      reinterpret_cast<uintptr_t>(plan) & 255)
    return set_error(MEA_ERR_ALIGNMENT, "packed attention: cu_seqlens and lse2 must be 4-byte, plan 256-byte aligned");
  if (plan_bytes < packed_plan_bytes(pd))
    return set_error(MEA_ERR_WORKSPACE, "packed attention: plan has %zu bytes, needs %zu", plan_bytes, packed_plan_bytes(pd));
  PackedFwdMaps maps;
  rc = packed_map(&maps.q, pd, d->dtype, q, d->q_row, d->q_head, pd.Hq, pd.p, pd.tt);
  rc |= packed_map(&maps.k, pd, d->dtype, k, d->k_row, d->k_head, pd.Hkv, 1, 128);
  rc |= packed_map(&maps.v, pd, d->dtype, v, d->v_row, d->v_head, pd.Hkv, 1, 128);
  if (rc) return set_error(MEA_ERR_CUDA, "packed attention: tensor map encode failed (%d)", rc);
  auto st = static_cast<cudaStream_t>(stream);
  if ((rc = run_packed_plan(pd, cu_seqlens, plan, status, st)) != MEA_OK) return rc;
  PackedFwdParams p;
  p.d = pd;
  p.plan = packed_plan_view(pd, plan);
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.v = v;
  p.v_tok = d->v_row;
  p.v_head = d->v_head;
  p.o = o;
  p.lse2 = lse2;
  p.status = status;
  if (pd.cap_q == 0) {
    // n_seqs = 0: no query tile can exist, every row of o is outside.
    if (cudaMemsetAsync(o, 0, size_t(pd.total) * pd.Hq * pd.N * 2, st) != cudaSuccess)
      return set_error(MEA_ERR_CUDA, "packed attention: clearing o failed");
    return MEA_OK;
  }
  if (d->dtype == MEA_BF16)
    return pd.N <= 64 ? launch_packed_fwd<64, Bf16>(maps, p, st) : launch_packed_fwd<128, Bf16>(maps, p, st);
  return pd.N <= 64 ? launch_packed_fwd<64, Fp16>(maps, p, st) : launch_packed_fwd<128, Fp16>(maps, p, st);
}
