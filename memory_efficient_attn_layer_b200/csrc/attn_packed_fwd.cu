// Causal softmax attention forward over packed sequences with grouped heads.
//
//   o_i = sum_{j <= i} p_ij v_j,  p_i = softmax_j(scale q_i . k_j)
// within each sequence, in one pass over its keys with the running row maximum
// and sum.  lse2 = max + log2(sum) per row (log2 units) is kept for the backward.
//
// Persistent, one CTA per SM.  An item is two neighbouring query tiles (tt tokens
// x p heads each) of one sequence and head group: two streams that share every K
// and V tile, each with its own softmax warpgroup.  While one stream's
// exponentials run, the tensor core works on the other's products:
//   PV_0(j), S_0(j+1) | PV_1(j), S_1(j+1) | ...
// Warp 0 brings in Q, K and V by TMA, warp 1 issues the MMAs, warp 2 looks over V
// tiles that the mask cuts, warps 4..7 and 8..11 are the softmax of streams 0 and
// 1, one row per thread with its 128 scores in registers.  TMEM: HD = 128 writes P
// over S (S_0 S_1 O_0 O_1); HD = 64 has columns for P, so the next scores are
// computed as soon as these are in registers.
//
// What bounds it: at HD = 128 the chain of one stream's step (scores, maximum and
// exponentials about 1900 clocks, then 1024 of MMAs and their hand-overs), which
// the other stream hides in part (tensor pipe 61 to 66% busy); at HD = 64, where a
// step has half the MMA work, the exponentials (a quarter of them as a
// polynomial on the FMA pipe).  16384 tokens with 16/2 heads of 128: 865 us, 1.27
// PF/s; with 8/8 heads of 64: 385 us; 16 documents of 21267 tokens, 8/8 heads of
// 64: 81 us.  One query tile to a CTA and eight softmax warps took 1320 us and more
// for the first.
//
// Rows of other sequences never reach a result: the last key tile's V rows past
// the sequence's end are cleared in shared memory (their P is zero, but zero
// times an inf or NaN is not), and so are the inf or NaN elements of V in the
// tile's masked triangle, which are added back to the rows that do see them.
#include <type_traits>

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
  static constexpr bool SEP_P = HD <= 64;
  static constexpr int QB = HD <= 64 ? 2 : 1;  // Q buffers (of two tiles)
  static constexpr int KS = 2, VS = 2;
  static constexpr uint32_t TB = 128 * HD * 2;
  static constexpr uint32_t S_COL = 0, P_COL = SEP_P ? 256 : 0, P_STEP = SEP_P ? 64 : 128;
  static constexpr uint32_t O_COL = SEP_P ? 384 : 256;
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr uint32_t OFF_K = QB * 2 * TB, OFF_V = OFF_K + KS * TB, OFF_BAR = OFF_V + VS * TB;
  static constexpr uint32_t OFF_OUT = OFF_BAR + 768;
  static constexpr size_t SMEM = 1024 + OFF_OUT + 8 * WarpRows<(HD > 64)>::BYTES;
  // Which of eight pairs of exponentials run on the FMA pipe: a quarter, where the
  // other attention kernels' share is three eighths (16384 tokens with 8/8 heads of
  // 64: 384 us, three eighths 410, half 438, none 418; 16/2 heads of 128: 865, 881,
  // 950, 904).
  static constexpr uint32_t POLY_PAIRS = HD <= 64 ? 0x44 : 0x42;
  static constexpr int REG_SOFTMAX = 208, REG_REST = 88;  // 256 x 208 + 128 x 88 = 384 x 168
};

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

// One item: the query tiles [t0, t0 + tt) and, with two streams, [t0 + tt, t0 + 2 tt) of a sequence.
struct FwdItem {
  int seq0, t0, end, h0, kvh;
  int nkv[2];  // key tiles of each stream (0: no such tile)
  int n;       // the larger: stream 1 never has fewer, unless it is not there; -1: no item
  __device__ FwdItem() {}
  __device__ FwdItem(const PackedFwdParams& p, int idx, int n_items) {
    n = -1;
    if (idx >= n_items) return;
    const int rows = p.d.rows[LIST_FWD];
    const PackedTile<true> it(p.plan.list[LIST_FWD], idx, p.d.hg, rows);
    seq0 = it.seq0;
    t0 = it.tile * rows;
    end = min(t0 + rows, it.len);
    h0 = it.head * p.d.p;
    kvh = h0 / (p.d.Hq / p.d.Hkv);
    nkv[0] = (min(t0 + p.d.tt, end) + 127) >> 7;
    nkv[1] = end > t0 + p.d.tt ? (end + 127) >> 7 : 0;
    n = max(nkv[0], nkv[1]);
  }
  __device__ bool there() const volatile { return n > 0; }
};

// HALVES: P goes to the MMA warp in two halves of 64 keys, so that PV begins before
// the last exponentials are through.  Measured (N = 128), whole and in halves:
// 16384 tokens with 16/2 heads 917 and 867 us, eight ragged prompts with 16/4 heads
// 69.6 and 67.4; 16 x 2048 tokens with 16/16 heads, the order by sequence (K and V
// 268 MB), 355 and 366.  So it is taken where the plan goes by work.  At HD = 64 the
// next scores are computed meanwhile anyway (no change).
template <int HD, class T, bool HALVES>
__global__ void __launch_bounds__(384, 1) packed_fwd_kernel(const __grid_constant__ PackedFwdMaps maps,
                                                            const __grid_constant__ PackedFwdParams p) {
  using Cfg = PackedFwdCfg<HD>;
  using Tile = HeadTile<HD>;
  constexpr int KS = Cfg::KS, VS = Cfg::VS, QB = Cfg::QB;
  constexpr uint32_t TB = Cfg::TB;
  constexpr uint32_t IDESC_S = idesc_16bit(T::FMT, 128, 128, 0, 0);
  constexpr uint32_t IDESC_O = idesc_16bit(T::FMT, 128, HD, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  auto sQ = [&](int b, int x) { return base + (2 * b + x) * TB; };
  auto sK = [&](int s) { return base + Cfg::OFF_K + s * TB; };
  auto sV = [&](int s) { return base + Cfg::OFF_V + s * TB; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  const uint32_t b0 = smem_u32(bars);
  auto q_full = [&](int b) { return b0 + 8u * b; };
  auto q_empty = [&](int b) { return b0 + 8u * (2 + b); };
  auto k_full = [&](int s) { return b0 + 8u * (4 + s); };
  auto k_empty = [&](int s) { return b0 + 8u * (6 + s); };
  auto v_full = [&](int s) { return b0 + 8u * (8 + s); };
  auto v_empty = [&](int s) { return b0 + 8u * (10 + s); };
  auto v_raw = [&](int s) { return b0 + 8u * (12 + s); };    // landed, for warp 2 to look over
  auto s_full = [&](int x) { return b0 + 8u * (14 + x); };   // S_x(j) computed
  auto s_empty = [&](int x) { return b0 + 8u * (16 + x); };  // (SEP_P) and in registers
  auto p_full = [&](int x) { return b0 + 8u * (18 + x); };   // P_x(j) written
  auto pv_done = [&](int x) { return b0 + 8u * (20 + x); };  // (SEP_P) PV_x(j) done
  auto o_full = [&](int x) { return b0 + 8u * (22 + x); };   // an item's O_x complete
  auto o_empty = [&](int x) { return b0 + 8u * (24 + x); };  // and read out
  auto p_half = [&](int x) { return b0 + 8u * (26 + x); };   // the first 64 columns of P_x(j) written
  const uint32_t drain_bar = b0 + 8u * 28;
  const Feed<FwdItem> feed{b0 + 8u * 29, b0 + 8u * 33, reinterpret_cast<FwdItem*>(bars + 42)};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 37);
  volatile int* bad = reinterpret_cast<int*>(bars + 38);  // per item (mod 4) and stream: V held inf or NaN behind the mask

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 16; ++i) mbar_init(b0 + 8u * i, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_empty(x), 128);
      mbar_init(p_full(x), 128);
      mbar_init(p_half(x), 128);
      mbar_init(pv_done(x), 1);
      mbar_init(o_full(x), 1);
      mbar_init(o_empty(x), 128);
    }
    mbar_init(drain_bar, 1);
    static_assert(8 * 42 + Feed<FwdItem>::BYTES <= 768, "barrier space");
    for (int i = 0; i < feed.SLOTS; ++i) {
      mbar_init(feed.full + 8u * i, 1);
      mbar_init(feed.empty + 8u * i, 10);  // MMA, warp 2, eight softmax warps
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  Guard g(p.status, KID_PACKED_FWD);
  auto finish = [&]() {
    tc_fence_before();
    named_bar_sync(1, 384);
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, Cfg::TMEM_COLS);
    }
  };

  if (warp < 4) {
    reg_dealloc<Cfg::REG_REST>();
    if (warp == 0) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        const int n_items = p.plan.head->n[LIST_FWD] * p.d.hg;
        const uint32_t box = uint32_t(p.d.p * p.d.tt) * 128 * Tile::NCHUNK;
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        int qpar[2] = {-1, -1}, kpar[KS], vpar[VS];
        for (int s = 0; s < KS; ++s) kpar[s] = -1;
        for (int s = 0; s < VS; ++s) vpar[s] = -1;
        int n = 0;
        FwdItem w(p, blockIdx.x, n_items);
        feed.put(0, w, g);
        for (int item = 0; w.there() && g.ok; ++item) {
          FwdItem next;
          const int qb = item % QB;
          if (item >= QB && !mbar_wait(q_empty(qb), uint32_t((item / QB - 1) & 1), g, 1)) break;
          mbar_expect_tx(q_full(qb), w.nkv[1] ? 2 * box : box);
          for (int x = 0; x < (w.nkv[1] ? 2 : 1); ++x)
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c)
              tma_load_3d(sQ(qb, x) + c * 16384, &maps.q, q_full(qb), c * 64, w.h0, w.seq0 + w.t0 + x * p.d.tt);
          qpar[qb] = (item / QB) & 1;
          for (int j = 0; j < w.n; ++j, ++n) {
            const int sk = n % KS, sv = n % VS;
            const uint32_t pk = (n / KS) & 1, pv = (n / VS) & 1;
            if (!mbar_wait(k_empty(sk), pk ^ 1, g, 2)) break;
            mbar_expect_tx(k_full(sk), TB);
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c)
              tma_load_3d(sK(sk) + c * 16384, &maps.k, k_full(sk), c * 64, w.kvh, w.seq0 + j * 128);
            kpar[sk] = int(pk);
            if (!mbar_wait(v_empty(sv), pv ^ 1, g, 3)) break;
            mbar_expect_tx(v_raw(sv), TB);
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c)
              tma_load_3d(sV(sv) + c * 16384, &maps.v, v_raw(sv), c * 64, w.kvh, w.seq0 + j * 128);
            vpar[sv] = int(pv);
            if (j == max(w.n - 3, 0)) {
              next = FwdItem(p, int(gridDim.x) + atomicAdd(&p.plan.head->next, 1), n_items);
              feed.put(item + 1, next, g);
            }
          }
          w = next;
        }
        if (!g.ok) {
          for (int b = 0; b < QB; ++b)
            if (qpar[b] >= 0) mbar_drain(q_full(b), uint32_t(qpar[b]));
          for (int s = 0; s < KS; ++s)
            if (kpar[s] >= 0) mbar_drain(k_full(s), uint32_t(kpar[s]));
          for (int s = 0; s < VS; ++s)
            if (vpar[s] >= 0) mbar_drain(v_raw(s), uint32_t(vpar[s]));
        } else {
          // The MMA warp's last releases have landed before this CTA's shared memory goes away.
          for (int b = 0; b < QB; ++b)
            if (qpar[b] >= 0) mbar_wait(q_empty(b), uint32_t(qpar[b]), g, 4);
          for (int s = 0; s < KS; ++s)
            if (kpar[s] >= 0) mbar_wait(k_empty(s), uint32_t(kpar[s]), g, 5);
          for (int s = 0; s < VS; ++s)
            if (vpar[s] >= 0) mbar_wait(v_empty(s), uint32_t(vpar[s]), g, 6);
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      if (elect_one()) {
        bool any = false;
        int done[2] = {0, 0};  // steps of each stream so far (parities of p_full, s_empty)
        // S_x(j) of an item whose first K tile is number k0; the last stream to use the tile gives it back.
        auto issue_s = [&](const FwdItem& w, int item, int k0, int x, int j) -> bool {
          const int qb = item % QB, sk = (k0 + j) % KS;
          if (j == 0 && !mbar_wait(q_full(qb), (item / QB) & 1, g, 7)) return false;
          if (!mbar_wait(k_full(sk), ((k0 + j) / KS) & 1, g, 8)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + Cfg::S_COL + 128 * x, Tile::kmajor(sQ(qb, x), 128, kk), Tile::kmajor(sK(sk), 128, kk), IDESC_S,
                   kk > 0 ? 1u : 0u);
          mma_commit(s_full(x));
          if (x == 1 || j >= w.nkv[1]) mma_commit(k_empty(sk));
          if (j + 1 == w.n && (x == 1 || !w.nkv[1])) mma_commit(q_empty(qb));  // the item's last read of Q
          any = true;
          return true;
        };
        FwdItem w;
        int k0 = 0, outs[2] = {0, 0};  // K tile number at the item's start; items that each stream has had
        bool have = feed.get(0, w, g);
        if (have && issue_s(w, 0, 0, 0, 0) && w.nkv[1]) issue_s(w, 0, 0, 1, 0);
        for (int item = 0; have && g.ok; ++item) {
          for (int j = 0; j < w.n && g.ok; ++j) {
            const int sv = (k0 + j) % VS;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= w.nkv[x]) continue;
              const bool more = j + 1 < w.nkv[x];
              if (Cfg::SEP_P && more) {  // the next scores as soon as these are in registers
                if (!mbar_wait(s_empty(x), done[x] & 1, g, 9) || !issue_s(w, item, k0, x, j + 1)) break;
              }
              if (!mbar_wait(HALVES ? p_half(x) : p_full(x), done[x] & 1, g, 10)) break;
              if (!mbar_wait(v_full(sv), ((k0 + j) / VS) & 1, g, 11)) break;
              if (j == 0 && outs[x] > 0 && !mbar_wait(o_empty(x), (outs[x] - 1) & 1, g, 12)) break;
              tc_fence_after();
#pragma unroll
              for (int kc = 0; kc < 8; ++kc) {
                if (HALVES && kc == 4) {
                  if (!mbar_wait(p_full(x), done[x] & 1, g, 10)) break;
                  tc_fence_after();
                }
                mma_ts(tmem + Cfg::O_COL + HD * x, tmem + Cfg::P_COL + Cfg::P_STEP * x + kc * 8, Tile::mnmajor(sV(sv), 128, kc),
                       IDESC_O, (j > 0 || kc > 0) ? 1u : 0u);
              }
              if (!g.ok) break;
              if (Cfg::SEP_P) mma_commit(pv_done(x));
              if (x == 1 || j >= w.nkv[1]) mma_commit(v_empty(sv));
              if (!more) {
                mma_commit(o_full(x));
                ++outs[x];
              }
              ++done[x];
              if (!Cfg::SEP_P && more && !issue_s(w, item, k0, x, j + 1)) break;
            }
          }
          if (!g.ok) break;
          k0 += w.n;
          FwdItem nx;
          have = feed.get(item + 1, nx, g);
          if (have) {
            // SEP_P: the last scores must be in registers before the next item's are written.
            for (int x = 0; x < (nx.nkv[1] ? 2 : 1); ++x) {
              if (Cfg::SEP_P && done[x] > 0 && !mbar_wait(s_empty(x), (done[x] - 1) & 1, g, 13)) break;
              if (!issue_s(nx, item + 1, k0, x, 0)) break;
            }
            w = nx;
          }
        }
        if (!g.ok && any) {
          mma_commit(drain_bar);
          mbar_drain(drain_bar, 0);
        }
      }
    } else if (warp == 2) {
      // ---------------- V tiles: passed on, or looked over where the mask cuts them ----------------
      int n = 0;
      for (int item = 0; g.ok; ++item) {
        const volatile FwdItem& w = *feed.look(item, g);
        if (!g.ok || !w.there()) break;
        bool found = false;
        for (int j = 0; j < w.n; ++j, ++n) {
          const int sv = n % VS;
          g.ok = __all_sync(0xffffffffu, mbar_wait(v_raw(sv), (n / VS) & 1, g, 14));
          if (!g.ok) break;
          // Rows [from, to) of the tile are masked for some rows of the item only, rows [to, 128) for all of them.
          const int from = max(w.t0 + 1 - 128 * j, 0), to = min(w.end - 128 * j, 128);
          if (from < 128) {
            zero_rows<HD>(sV(sv), to, lane);
            found |= clear_nonfinite<HD, T>(sV(sv), from, to, lane);
            fence_proxy_async_smem();
          }
          if (lane == 0)  // with the stream's last V tile, which its O waits for
            for (int x = 0; x < 2; ++x)
              if (j + 1 == w.nkv[x]) bad[(item & 3) * 2 + x] = found;
          __syncwarp();
          if (lane == 0) mbar_arrive(v_full(sv));
        }
        feed.done(item, lane);
      }
    }
    finish();
    return;
  }
  reg_alloc<Cfg::REG_SOFTMAX>();
  // ---------------- softmax + epilogue: stream x, row r ----------------
  {
    const PackedHeader hd = *p.plan.head;
    zero_outside(static_cast<uint4*>(p.o), p.d.total, hd.first, hd.end, (long long)p.d.Hq * p.d.N / 8, blockIdx.x,
                 gridDim.x, threadIdx.x - 128, 256);
    const int x = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;
    const int tok = token_of(p.d, r);
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t st = lane_base + Cfg::S_COL + 128 * x, pt = lane_base + Cfg::P_COL + Cfg::P_STEP * x;
    const uint32_t ot = lane_base + Cfg::O_COL + HD * x;
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int n = 0, outs = 0;  // steps and items of this stream
    for (int item = 0; ok; ++item) {
      const volatile FwdItem& w = *feed.look(item, g);
      ok = g.ok;
      if (!ok || !w.there()) break;
      const int nkv = w.nkv[x];
      if (!nkv) {
        feed.done(item, lane);
        continue;
      }
      const int first = w.t0 + x * p.d.tt;  // the tile's first token
      const int t = first + tok;
      const bool live = tok < p.d.tt && t < w.end;
      float m_run = -INFINITY, l_run = 0.f;  // m_run in scaled log2 units
      bool nan_row = false;
#pragma unroll 1
      for (int j = 0; j < nkv; ++j, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait(s_full(x), n & 1, g, 15));
        if (!ok) break;
        tc_fence_after();
        float s[128];
        {
          uint32_t a[32], b[32], c[32], d[32];
          tmem_ld32(st, a);
          tmem_ld32(st + 32, b);
          tmem_ld32(st + 64, c);
          tmem_ld32(st + 96, d);
          tmem_wait_ld_tied2x32(a, b);
          reg_tie(c);
          reg_tie(d);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            s[e] = __uint_as_float(a[e]);
            s[32 + e] = __uint_as_float(b[e]);
            s[64 + e] = __uint_as_float(c[e]);
            s[96 + e] = __uint_as_float(d[e]);
          }
        }
        if (Cfg::SEP_P) {
          tc_fence_before();
          mbar_arrive(s_empty(x));
        }
        const bool mask = 128 * j + 127 > first;
        if (mask) {
          const int cmax = t - 128 * j;  // last column this row sees
#pragma unroll
          for (int e = 0; e < 128; ++e) s[e] = e > cmax ? -INFINITY : s[e];
        }
        float m[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int e = 4; e < 124; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) m[i] = max3f_nan(m[i], s[e + 2 * i], s[e + 2 * i + 1]);
        m[0] = max3f_nan(m[0], s[124], s[125]);
        m[1] = max3f_nan(m[1], s[126], s[127]);
        const float mx = max3f_nan(max3f_nan(m[0], m[1], m[2]), m[3], m[3]) * p.scale_log2;
        nan_row |= mx != mx;
        // PV(j - 1) is done: O is stable and the P columns are free.  (HD = 128: S(j)
        // was issued after it on the in-order tensor pipe.)
        if (Cfg::SEP_P && n > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(pv_done(x), (n - 1) & 1, g, 16));
          if (!ok) break;
          tc_fence_after();
        }
        // Lazy: the reference moves only when the maximum grows by more than 8 (log2
        // units), so P stays <= 2^8; O and the sum are rescaled only then.
        const bool need = mx > m_run + 8.0f || (m_run == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, need)) {
          const float m_new = need ? mx : m_run;
          const float alpha = need ? ex2(m_run - m_new) : 1.0f;  // 0 when m_run = -inf
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t ov[16];
              tmem_load16(ot + c, ov);
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st16(ot + c, ov);
            }
          }
          l_run *= alpha;
          m_run = m_new;
        }
        const float nm = m_run == -INFINITY ? 0.f : -m_run;
        const float2 neg_m = make_float2(nm, nm);
        float2 acc0 = make_float2(0.f, 0.f), acc1 = acc0;
        // In a masked tile every exponential runs on MUFU, which turns -inf into exactly 0.
        auto exps = [&](auto masked) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 pp = exp2_pair(ffma2(make_float2(s[16 * c + 2 * e], s[16 * c + 2 * e + 1]), sl2, neg_m),
                                          !masked() && ((Cfg::POLY_PAIRS >> e) & 1));
              if (e & 1)
                acc1 = fadd2(acc1, pp);
              else
                acc0 = fadd2(acc0, pp);
              pk[e] = T::pack(pp.x, pp.y);
            }
            tmem_st8(pt + 8 * c, pk);
            if (HALVES && c == 3) {
              tmem_st_wait();
              tc_fence_before();
              mbar_arrive(p_half(x));
            }
          }
        };
        if (mask)
          exps(std::true_type());
        else
          exps(std::false_type());
        l_run += (acc0.x + acc0.y) + (acc1.x + acc1.y);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(x));
      }
      if (!ok) break;
      // ---- epilogue: O / l ----
      ok = __all_sync(0xffffffffu, mbar_wait(o_full(x), outs & 1, g, 17));
      if (!ok) break;
      tc_fence_after();
      ++outs;
      float2 f[HD / 2];
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) tmem_load64(ot + 64 * c, *reinterpret_cast<float2(*)[32]>(f + 32 * c));
      tc_fence_before();
      mbar_arrive(o_empty(x));
      nan_row |= m_run == -INFINITY;  // no finite score: 0 / 0
      const float inv_l = nan_row ? __int_as_float(0x7fffffff) : 1.0f / l_run;
      if (bad[(item & 3) * 2 + x] && live) {  // the inf and NaN elements that were cleared, for the rows that see them
#pragma unroll 1
        for (int key = w.t0 + 1; key <= t; ++key) {
          const uint16_t* vr = static_cast<const uint16_t*>(p.v) + (long long)(w.seq0 + key) * p.v_tok + w.kvh * p.v_head;
#pragma unroll
          for (int e = 0; e < HD / 2; ++e) {
            if (2 * e < p.d.N && half_nonfinite<T>(vr[2 * e])) f[e].x += T::lo(vr[2 * e]);
            if (2 * e < p.d.N && half_nonfinite<T>(vr[2 * e + 1])) f[e].y += T::lo(vr[2 * e + 1]);
          }
        }
      }
      __syncwarp();
      WarpRows<(HD > 64)> out(base + Cfg::OFF_OUT + (warp - 4) * WarpRows<(HD > 64)>::BYTES, lane, (warp & 3) * 32);
#pragma unroll
      for (int i = 0; i < out.rows(); ++i) {
        const int row_tok = token_of(p.d, out.row(i));
        out.off[i] = (row_tok * p.d.Hq + out.row(i) - row_tok * p.d.p) * p.d.N;
        out.live[i] = row_tok < min(p.d.tt, w.end - first);
      }
      uint16_t* tile = static_cast<uint16_t*>(p.o) + ((long long)(w.seq0 + first) * p.d.Hq + w.h0) * p.d.N;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) out.template store32<T>(f + 16 * c, inv_l, tile, 32 * c, p.d.N);
      const long long row = (long long)(w.seq0 + t) * p.d.Hq + w.h0 + r - tok * p.d.p;
      if (live) p.lse2[row] = nan_row ? __int_as_float(0x7fffffff) : m_run + __log2f(l_run);
      feed.done(item, lane);
    }
    // The last pv_done has landed before this CTA's shared memory goes away.
    if (Cfg::SEP_P && ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(pv_done(x), (n - 1) & 1, g, 18));
    if (!ok) g.ok = false;
    finish();
  }
}

template <int HD, class T>
static int launch_packed_fwd(const PackedFwdMaps& maps, const PackedFwdParams& p, cudaStream_t st) {
  using Cfg = PackedFwdCfg<HD>;
  static_assert(Cfg::SMEM <= 232448, "shared memory");
  // (as the plan kernel decides from the lengths)
  const bool by_seq = packed_wide(p.d, LIST_FWD) && (long long)p.d.total / p.d.rows[LIST_FWD] * p.d.hg >= 8LL * num_sms();
  auto kern = HD <= 64 || by_seq ? packed_fwd_kernel<HD, T, false> : packed_fwd_kernel<HD, T, (HD > 64)>;
  if (!smem_attr_set(reinterpret_cast<const void*>(kern), int(Cfg::SMEM)))
    return set_error(MEA_ERR_CUDA, "cudaFuncSetAttribute(packed_fwd) failed");
  cudaLaunchAttribute attr;
  const long long items = (long long)p.d.cap[LIST_FWD] * p.d.hg;
  const cudaLaunchConfig_t cfg = packed_launch(int(items < num_sms() ? items : num_sms()), 384, Cfg::SMEM, st, &attr);
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
  if (pd.cap[LIST_FWD] == 0) {
    // n_seqs = 0: no query tile can exist, every row of o is outside.
    if (cudaMemsetAsync(o, 0, size_t(pd.total) * pd.Hq * pd.N * 2, st) != cudaSuccess)
      return set_error(MEA_ERR_CUDA, "packed attention: clearing o failed");
    return MEA_OK;
  }
  if (d->dtype == MEA_BF16)
    return pd.N <= 64 ? launch_packed_fwd<64, Bf16>(maps, p, st) : launch_packed_fwd<128, Bf16>(maps, p, st);
  return pd.N <= 64 ? launch_packed_fwd<64, Fp16>(maps, p, st) : launch_packed_fwd<128, Fp16>(maps, p, st);
}
