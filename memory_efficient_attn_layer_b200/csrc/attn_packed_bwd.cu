// Causal softmax attention backward over packed sequences with grouped heads.
//
//   delta_i = sum_d dO_id O_id           (packed_delta_kernel; the first 128 tokens'
//                                         again in fp32 by the dQ kernel)
//   P_ij = exp2(scale_log2 q_i.k_j - lse2_i),  dS_ij = P_ij (dO_i.v_j - delta_i)
//   dQ_i = scale sum_j dS_ij k_j         (packed_dq_kernel: a query tile walks its key tiles)
//   dV_j = sum_i P_ij dO_i, dK_j = scale sum_i dS_ij q_i
//                                        (packed_dkv_kernel: a key tile walks its query tiles)
//
// Every sum has one owner: dQ stays in TMEM for a query tile, dK and dV for a
// key tile, where the walk also runs over the group's query heads.  So there are
// no atomics and no fp32 buffer in global memory, and the results do not depend
// on the order in which tiles run; the price is that both kernels form S and dP
// (7 tile products where an accumulating kernel has 5).
//
// Both kernels feed the second product of each pair from TMEM.  In the dQ kernel
// rows are queries and dS is its A operand; the dK/dV kernel computes S^T = K Q^T
// and dP^T = V dO^T with keys as rows, so P^T and dS^T, written in place over
// them, are the A operands of dV and dK.  P and dS never pass through shared
// memory, whose bandwidth the S and dP products (both operands there) need.
//
// With few key tiles (few key/value heads, not many rows) a tile's walk over the
// queries is cut into parts that leave fp32 partial sums, added in their order by
// packed_dkv_sum_kernel.
//
// What bounds it: the MMAs, at 1.2 to 1.4 PF/s (60 to 72% of the tensor pipe; S and
// dP read both operands from shared memory at its full rate), and at HD = 64 the
// exponentials beside MMAs of half the work.  12289 + 4095 tokens with 16/4 heads of
// 128: dQ 874 us, dK/dV 1003 us; 16 documents of 21267 tokens with 8/8 heads of 64:
// dQ 104 us, dK/dV 128 us; delta 14 us (HBM).
//
// Warps (384 threads, persistent, one CTA per SM): 0 TMA, 1 MMA issue, 2 (dK/dV)
// lse2 and delta rows, 4..11 softmax: two warps per TMEM lane quarter, half a row
// each.
#include <type_traits>

#include "attn_packed.h"
#include "attn_packed.cuh"

namespace mea {

struct PackedBwdParams {
  PackedDims d;
  PackedPlan plan;
  float scale, scale_log2;
  const float* lse2;   // [total, Hq]
  float* delta;        // [total, Hq]
  int* next;           // next tile to be drawn from LIST_Q and LIST_K
  uint16_t* dq;        // [total, Hq, N]
  uint16_t* dk;        // [total, Hkv, N]
  uint16_t* dv;
  float* parts;        // [splits][dK, dV][total, Hkv, N] of cut walks
  int* status;
};
struct PackedBwdMaps {
  CUtensorMap q, k, v, dO;
};

// ---------------------------------------------------------------- delta
// 16 lanes per (token, head) row, 16 bytes of O and dO each, four rows in
// flight; also clears the rows of dQ, dK and dV that no sequence owns, and the
// counters that the next two kernels draw their tiles from.
constexpr int DELTA_ROWS = 64;  // rows per 256-thread block
template <class T>
__global__ void __launch_bounds__(256) packed_delta_kernel(PackedDims d, const PackedHeader* head, int* next, const uint16_t* o,
                                                           const uint16_t* dO, long long do_row, long long do_head,
                                                           float* delta, uint4* dq, uint4* dk, uint4* dv) {
  pdl_launch();
  if (blockIdx.x == 0 && threadIdx.x == 0) next[LIST_Q] = next[LIST_K] = 0;
  const long long rows = (long long)d.total * d.Hq;
  const int sub = threadIdx.x & 15;
  const long long r0 = (long long)blockIdx.x * DELTA_ROWS + (threadIdx.x >> 4);
  uint4 a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long r = r0 + 16 * i;
    a[i] = b[i] = make_uint4(0, 0, 0, 0);
    if (r < rows && sub * 8 < d.N) {
      const long long t = r / d.Hq;
      const int h = int(r - t * d.Hq);
      a[i] = __ldg(reinterpret_cast<const uint4*>(o + r * d.N) + sub);
      b[i] = __ldg(reinterpret_cast<const uint4*>(dO + t * do_row + h * do_head) + sub);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, y[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += T::lo(x[e]) * T::lo(y[e]) + T::hi(x[e]) * T::hi(y[e]);
#pragma unroll
    for (int m = 8; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (sub == 0 && r0 + 16 * i < rows) delta[r0 + 16 * i] = s;
  }
  const PackedHeader hd = *head;
  const long long wq = (long long)d.Hq * d.N / 8, wk = (long long)d.Hkv * d.N / 8;
  zero_outside(dq, d.total, hd.first, hd.end, wq, blockIdx.x, gridDim.x, threadIdx.x, blockDim.x);
  zero_outside(dk, d.total, hd.first, hd.end, wk, blockIdx.x, gridDim.x, threadIdx.x, blockDim.x);
  zero_outside(dv, d.total, hd.first, hd.end, wk, blockIdx.x, gridDim.x, threadIdx.x, blockDim.x);
}

// ---------------------------------------------------------------- common
// ---------------------------------------------------------------- dQ
template <int HD>
struct PackedDqCfg {
  static constexpr int QB = HD <= 64 ? 2 : 1;  // Q/dO buffers: the next item's load overlaps this one
  static constexpr int KS = 2, VS = 2;
  static constexpr uint32_t TB = 128 * HD * 2;
  static constexpr uint32_t S_COL = 0, DP_COL = 128, DS_COL = 256, DQ_COL = 384;  // two dS buffers
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr uint32_t OFF_K = QB * 2 * TB, OFF_V = OFF_K + KS * TB, OFF_BAR = OFF_V + VS * TB;
  static constexpr uint32_t OFF_OUT = OFF_BAR + 768, OFF_X = OFF_OUT + 8 * WarpRows<true>::BYTES;
  static constexpr size_t SMEM = 1024 + OFF_X + 1024;
};

struct DqItem {
  int seq0, len, t0, t1, h0, kvh;
  int nkv;  // key tiles; 0: no item
  __device__ DqItem() {}
  __device__ DqItem(const PackedDims& d, const PackedPlan& plan, int idx, int n_items) {
    nkv = 0;
    if (idx >= n_items) return;
    const PackedTile<true> it(plan.list[LIST_Q], idx, d.hg, d.tt);
    seq0 = it.seq0;
    len = it.len;
    t0 = it.tile * d.tt;
    t1 = min(t0 + d.tt, len);
    nkv = (t1 + 127) >> 7;
    h0 = it.head * d.p;
    kvh = h0 / (d.Hq / d.Hkv);
  }
  __device__ bool there() const volatile { return nkv > 0; }
};

template <int HD, class T>
__global__ void __launch_bounds__(384, 1) packed_dq_kernel(const __grid_constant__ PackedBwdMaps maps,
                                                           const __grid_constant__ PackedBwdParams p) {
  using Cfg = PackedDqCfg<HD>;
  using Tile = HeadTile<HD>;
  constexpr int QB = Cfg::QB, KS = Cfg::KS, VS = Cfg::VS;
  constexpr uint32_t TB = Cfg::TB;
  constexpr uint32_t IDESC_SS = idesc_16bit(T::FMT, 128, 128, 0, 0);
  constexpr uint32_t IDESC_DQ = idesc_16bit(T::FMT, 128, HD, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  auto sQ = [&](int b) { return base + 2 * TB * b; };
  auto sdO = [&](int b) { return base + 2 * TB * b + TB; };
  auto sK = [&](int s) { return base + Cfg::OFF_K + TB * s; };
  auto sV = [&](int s) { return base + Cfg::OFF_V + TB * s; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  const uint32_t b0 = smem_u32(bars);
  auto q_full = [&](int b) { return b0 + 8u * b; };
  auto q_empty = [&](int b) { return b0 + 8u * (2 + b); };
  auto k_full = [&](int s) { return b0 + 8u * (4 + s); };
  auto k_empty = [&](int s) { return b0 + 8u * (6 + s); };
  auto v_full = [&](int s) { return b0 + 8u * (8 + s); };
  auto v_empty = [&](int s) { return b0 + 8u * (10 + s); };
  const uint32_t s_full = b0 + 8u * 12, s_empty = b0 + 8u * 13;    // S computed / read by the softmax
  const uint32_t dp_full = b0 + 8u * 14, dp_empty = b0 + 8u * 15;  // dP the same
  const uint32_t ds_full = b0 + 8u * 16;                           // dS written
  auto ds_free = [&](int b) { return b0 + 8u * (17 + b); };        // read by the dQ MMAs, per buffer
  const uint32_t dq_full = b0 + 8u * 19, dq_empty = b0 + 8u * 20;  // an item's dQ complete / read out
  const uint32_t k_raw = b0 + 8u * 21, drain_bar = b0 + 8u * 22;
  const Feed<DqItem> feed{b0 + 8u * 23, b0 + 8u * 27, reinterpret_cast<DqItem*>(bars + 32)};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 12; ++i) mbar_init(b0 + 8u * i, 1);
    mbar_init(s_full, 1);
    mbar_init(s_empty, 256);
    mbar_init(dp_full, 1);
    mbar_init(dp_empty, 256);
    mbar_init(ds_full, 256);
    mbar_init(ds_free(0), 1);
    mbar_init(ds_free(1), 1);
    mbar_init(dq_full, 1);
    mbar_init(dq_empty, 256);
    mbar_init(k_raw, 1);
    mbar_init(drain_bar, 1);
    static_assert(8 * 32 + Feed<DqItem>::BYTES <= 768, "barrier space");
    for (int i = 0; i < feed.SLOTS; ++i) {
      mbar_init(feed.full + 8u * i, 1);
      mbar_init(feed.empty + 8u * i, 9);  // MMA, eight softmax warps
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
  pdl_launch();
  const int n_items = p.plan.head->n[LIST_Q] * p.d.hg;
  Guard g(p.status, KID_PACKED_DQ);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    const bool lead = lane == 0;
    int qpar[2] = {-1, -1}, kpar[KS], vpar[VS];
    for (int s = 0; s < KS; ++s) kpar[s] = -1;
    for (int s = 0; s < VS; ++s) vpar[s] = -1;
    int n = 0, item = 0, raw = 0;
    DqItem w(p.d, p.plan, blockIdx.x, n_items), next;
    if (lead) feed.put(0, w, g);
    while (w.there() && g.ok) {
      const int qb = item % QB;
      if (lead && (item < QB || mbar_wait(q_empty(qb), uint32_t((item / QB - 1) & 1), g, 1))) {
        mbar_expect_tx(q_full(qb), 2u * uint32_t(p.d.p * p.d.tt) * 128 * Tile::NCHUNK);
#pragma unroll
        for (int c = 0; c < Tile::NCHUNK; ++c) {
          tma_load_3d(sQ(qb) + c * 16384, &maps.q, q_full(qb), c * 64, w.h0, w.seq0 + w.t0);
          tma_load_3d(sdO(qb) + c * 16384, &maps.dO, q_full(qb), c * 64, w.h0, w.seq0 + w.t0);
        }
        qpar[qb] = (item / QB) & 1;
      }
      ++item;
      for (int j = 0; j < w.nkv; ++j, ++n) {
        const int sk = n % KS, sv = n % VS;
        const uint32_t pk = (n / KS) & 1, pv = (n / VS) & 1;
        // Rows of other sequences in the last key tile: dS is zero there, but the
        // dQ product would still multiply it by whatever they hold.
        const bool tail = 128 * (j + 1) > w.len;
        if (lead) {
          if (mbar_wait(k_empty(sk), pk ^ 1, g, 2)) {
            const uint32_t full = tail ? k_raw : k_full(sk);
            mbar_expect_tx(full, TB);
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c)
              tma_load_3d(sK(sk) + c * 16384, &maps.k, full, c * 64, w.kvh, w.seq0 + j * 128);
            kpar[sk] = int(pk);
          }
          if (mbar_wait(v_empty(sv), pv ^ 1, g, 3)) {
            mbar_expect_tx(v_full(sv), TB);
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c)
              tma_load_3d(sV(sv) + c * 16384, &maps.v, v_full(sv), c * 64, w.kvh, w.seq0 + j * 128);
            vpar[sv] = int(pv);
          }
        }
        if (j == max(w.nkv - 3, 0)) {
          int idx = 0;
          if (lead) idx = int(gridDim.x) + atomicAdd(p.next + LIST_Q, 1);
          next = DqItem(p.d, p.plan, __shfl_sync(0xffffffffu, idx, 0), n_items);
          if (lead) feed.put(item, next, g);  // (item counts this one already)
        }
        g.ok = __all_sync(0xffffffffu, g.ok);
        if (!g.ok) break;
        if (tail) {
          g.ok = __all_sync(0xffffffffu, mbar_wait(k_raw, raw & 1, g, 4));
          ++raw;
          if (!g.ok) break;
          zero_rows<HD>(sK(sk), w.len - 128 * j, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lead) mbar_arrive(k_full(sk));
        }
      }
      w = next;
    }
    if (lead) {
      if (!g.ok) {
        for (int b = 0; b < QB; ++b)
          if (qpar[b] >= 0) mbar_drain(q_full(b), uint32_t(qpar[b]));
        for (int s = 0; s < KS; ++s)
          if (kpar[s] >= 0) mbar_drain(k_full(s), uint32_t(kpar[s]));
        for (int s = 0; s < VS; ++s)
          if (vpar[s] >= 0) mbar_drain(v_full(s), uint32_t(vpar[s]));
        mbar_drain(k_raw, uint32_t(raw & 1));
      } else {
        // The MMA warp's last releases have landed before this CTA's shared memory goes away.
        for (int b = 0; b < QB; ++b)
          if (qpar[b] >= 0) mbar_wait(q_empty(b), uint32_t(qpar[b]), g, 5);
        for (int s = 0; s < KS; ++s)
          if (kpar[s] >= 0) mbar_wait(k_empty(s), uint32_t(kpar[s]), g, 6);
        for (int s = 0; s < VS; ++s)
          if (vpar[s] >= 0) mbar_wait(v_empty(s), uint32_t(vpar[s]), g, 7);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      bool any = false;
      // S and dP run one step ahead of dQ, across items: (n1, item1, j1) is their next step.
      int n1 = 0, item1 = 0, j1 = 0, nkv1 = 0;  // nkv1 = 0: no more items
      auto settle = [&]() {
        DqItem w;
        nkv1 = feed.get(item1, w, g) ? w.nkv : 0;
      };
      settle();
      auto issue_s = [&]() -> bool {
        const int qb = item1 % QB, sk = n1 % KS;
        if (j1 == 0 && !mbar_wait(q_full(qb), (item1 / QB) & 1, g, 8)) return false;
        if (!mbar_wait(k_full(sk), (n1 / KS) & 1, g, 9)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_ss(tmem + Cfg::S_COL, Tile::kmajor(sQ(qb), 128, kk), Tile::kmajor(sK(sk), 128, kk), IDESC_SS,
                 kk > 0 ? 1u : 0u);
        mma_commit(s_full);
        any = true;
        return true;
      };
      auto issue_dp = [&]() -> bool {
        const int qb = item1 % QB, sv = n1 % VS;
        if (!mbar_wait(v_full(sv), (n1 / VS) & 1, g, 10)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_ss(tmem + Cfg::DP_COL, Tile::kmajor(sdO(qb), 128, kk), Tile::kmajor(sV(sv), 128, kk), IDESC_SS,
                 kk > 0 ? 1u : 0u);
        mma_commit(v_empty(sv));
        if (j1 + 1 == nkv1) mma_commit(q_empty(qb));  // the item's last read of Q and dO
        mma_commit(dp_full);
        ++n1;
        if (++j1 == nkv1) {
          j1 = 0;
          ++item1;
          settle();
        }
        return true;
      };
      int n = 0, item = 0, nkv = nkv1;
      if (nkv && issue_s()) issue_dp();
      while (nkv && g.ok) {
        int nkv_next = 0;
        for (int j = 0; j < nkv; ++j, ++n) {
          const int sk = n % KS;
          const bool more = nkv1 > 0;
          if (j + 1 == nkv) nkv_next = nkv1;  // the lookahead stands at the next item by now
          // With one Q/dO buffer the next item's rows arrive late: this item's last dQ goes first.
          // (dP behind dQ: before it, 16384 tokens with 16/2 heads take 1419 us instead of 1272.)
          const bool early = more && (QB == 2 || j + 1 < nkv);
          if (early && !(mbar_wait(s_empty, n & 1, g, 11) && issue_s())) break;
          if (!mbar_wait(ds_full, n & 1, g, 13)) break;
          if (j == 0 && item > 0 && !mbar_wait(dq_empty, (item - 1) & 1, g, 14)) break;
          tc_fence_after();
#pragma unroll
          for (int kc = 0; kc < 8; ++kc)
            mma_ts(tmem + Cfg::DQ_COL, tmem + Cfg::DS_COL + 64 * (n & 1) + kc * 8, Tile::mnmajor(sK(sk), 128, kc), IDESC_DQ,
                   (j > 0 || kc > 0) ? 1u : 0u);
          mma_commit(k_empty(sk));
          mma_commit(ds_free(n & 1));
          if (j + 1 == nkv) mma_commit(dq_full);
          if (more && !early && !(mbar_wait(s_empty, n & 1, g, 11) && issue_s())) break;
          if (more && !(mbar_wait(dp_empty, n & 1, g, 12) && issue_dp())) break;
        }
        nkv = nkv_next;
        ++item;
      }
      if (!g.ok && any) {
        mma_commit(drain_bar);
        mbar_drain(drain_bar, 0);
      }
    }
  } else if (warp >= 4) {
    // ---------------- softmax warps 4..11: row r, columns [64 hh, 64 hh + 64) ----------------
    const int quarter = warp & 3, hh = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = tmem + (uint32_t(quarter * 32) << 16);
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    const int tok = token_of(p.d, r), hr = r - tok * p.d.p;
    WarpRows<true> out(base + Cfg::OFF_OUT + (warp - 4) * WarpRows<true>::BYTES, lane, quarter * 32);
    bool ok = true;
    int n = 0, item = 0;
    while (ok) {
      const volatile DqItem& w = *feed.look(item, g);
      ok = g.ok;
      if (!ok || !w.there()) break;
      const int nkv = w.nkv, t0 = w.t0;
      const int t = t0 + tok;
      const bool live = r < p.d.p * p.d.tt && t < w.t1;
      const long long row = (long long)(w.seq0 + t) * p.d.Hq + w.h0 + hr;
      const float lse = live ? __ldg(p.lse2 + row) : INFINITY;  // P = 0 in rows that are not there
      const float dl = live ? p.delta[row] : 0.f;
      const float2 neg_lse = make_float2(-lse, -lse);
      float2 dl2 = make_float2(dl, dl);
      for (int j = 0; j < nkv; ++j, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait(s_full, n & 1, g, 15));
        if (!ok) break;
        tc_fence_after();
        const bool mask = 128 * j + 127 > t0;
        const int cmax = t - 128 * j - 64 * hh;  // last of this thread's columns that the row sees
        float2 P[32];
        tmem_load64(lane_base + Cfg::S_COL + 64 * hh, P);
        tc_fence_before();
        mbar_arrive(s_empty);  // the scores are in registers
#pragma unroll
        for (int e = 0; e < 32; ++e) P[e] = exp2_pair(ffma2(P[e], sl2, neg_lse), (kPolyPairsBwd >> (e & 7)) & 1);
        ok = __all_sync(0xffffffffu, mbar_wait(dp_full, n & 1, g, 16));
        if (!ok) break;
        tc_fence_after();
        float2 dp[32];
        tmem_load64(lane_base + Cfg::DP_COL + 64 * hh, dp);
        tc_fence_before();
        mbar_arrive(dp_empty);
        if (n > 1) {
          ok = __all_sync(0xffffffffu, mbar_wait(ds_free(n & 1), ((n >> 1) - 1) & 1, g, 17));
          if (!ok) break;
          tc_fence_after();
        }
        if (nkv == 1) {
          // The first 128 tokens of a sequence have all their keys here, so delta =
          // sum_j P_ij dP_ij can be had from fp32 values.  From the rounded O it is off
          // by a rounding of O, which counts where O is not yet an average of many rows.
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            sum += 2 * e > cmax ? 0.f : P[e].x * dp[e].x;
            sum += 2 * e + 1 > cmax ? 0.f : P[e].y * dp[e].y;
          }
          float* xch = reinterpret_cast<float*>(smem + Cfg::OFF_X);
          xch[hh * 128 + r] = sum;
          named_bar_sync(2 + quarter, 64);  // the row's other half
          sum += xch[(hh ^ 1) * 128 + r];
          named_bar_sync(2 + quarter, 64);  // read before the next item writes
          dl2 = make_float2(sum, sum);
          if (live && hh == 0) p.delta[row] = sum;  // for the dK/dV kernel
        }
        auto grad = [&](auto masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t ds[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float2 s = fmul2(P[8 * c + e], fsub2(dp[8 * c + e], dl2));
              if (masked()) {
                s.x = 16 * c + 2 * e > cmax ? 0.f : s.x;
                s.y = 16 * c + 2 * e + 1 > cmax ? 0.f : s.y;
              }
              ds[e] = T::pack(s.x, s.y);
            }
            tmem_st8(lane_base + Cfg::DS_COL + 64 * (n & 1) + 32 * hh + 8 * c, ds);
          }
        };
        if (mask)
          grad(std::true_type());
        else
          grad(std::false_type());
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(dq_full, item & 1, g, 18));
      if (!ok) break;
      tc_fence_after();
      float2 dq[HD / 4];
      if constexpr (HD == 128) {
        tmem_load64(lane_base + Cfg::DQ_COL + 64 * hh, *reinterpret_cast<float2(*)[32]>(dq));
      } else {
        uint32_t v[32];
        tmem_load32(lane_base + Cfg::DQ_COL + 32 * hh, v);
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[e] = make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
      }
      tc_fence_before();
      mbar_arrive(dq_empty);
#pragma unroll
      for (int i = 0; i < out.rows(); ++i) {
        const int row_tok = token_of(p.d, out.row(i));
        out.off[i] = (row_tok * p.d.Hq + out.row(i) - row_tok * p.d.p) * p.d.N;
        out.live[i] = row_tok < w.t1 - t0;
      }
      uint16_t* tile = p.dq + ((long long)(w.seq0 + t0) * p.d.Hq + w.h0) * p.d.N;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) out.template store32<T>(dq + 16 * c, p.scale, tile, hh * (HD / 2) + 32 * c, p.d.N);
      feed.done(item, lane);
      ++item;
    }
    // The last two steps' ds_free have landed before this CTA's shared memory goes away.
    for (int m = n > 1 ? n - 2 : 0; ok && m < n; ++m) ok = __all_sync(0xffffffffu, mbar_wait(ds_free(m & 1), (m >> 1) & 1, g, 19));
    if (!ok) g.ok = false;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- dK, dV
template <int HD>
struct PackedDkvCfg {
  static constexpr int KVB = HD <= 64 ? 2 : 1;  // K/V buffers
  static constexpr int SB = HD <= 64 ? 2 : 1;   // S^T buffers in TMEM
  static constexpr int ST = HD <= 64 ? 4 : 2;   // Q/dO ring depth: S^T runs SB steps ahead of the stage's release
  static constexpr uint32_t TB = 128 * HD * 2;
  static constexpr uint32_t S_COL = 0, DP_COL = SB * 128, DV_COL = DP_COL + 128, DK_COL = DV_COL + HD;
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr int REG_SOFTMAX = 208, REG_REST = 88;  // 256 x 208 + 128 x 88 = 384 x 168
  static_assert(DK_COL + HD <= 512, "TMEM budget");
  static constexpr uint32_t OFF_Q = KVB * 2 * TB, OFF_ROW = OFF_Q + ST * 2 * TB, OFF_BAR = OFF_ROW + ST * 1024;
  static constexpr uint32_t OFF_OUT = OFF_BAR + 768;
  static constexpr size_t SMEM = 1024 + OFF_OUT + 8 * WarpRows<true>::BYTES;
};

// Part `part` of `splits` of a key tile's walk: steps [lo, hi) over the group's
// query tiles, `span` of them for each of `groups` sets of p heads.  A walk of
// fewer steps has fewer parts.
struct DkvItem {
  int seq0, len, k0, kvh, qt0, span, h0, part;
  int lo, hi;  // lo = hi: a part that a short walk does not have; lo < 0: no item
  __device__ DkvItem() {}
  __device__ DkvItem(const PackedDims& d, const PackedPlan& plan, int idx, int splits, int n_items) {
    lo = hi = -1;
    if (idx >= n_items) return;
    part = 0;
    if (splits > 1) {
      const int i = idx / splits;
      part = idx - i * splits;
      idx = i;
    }
    const PackedTile<false> it(plan.list[LIST_K], idx, d.Hkv, 128);  // the first tile takes longest
    kvh = it.head;
    seq0 = it.seq0;
    len = it.len;
    k0 = it.tile * 128;
    qt0 = k0 / d.tt;
    span = (len + d.tt - 1) / d.tt - qt0;
    h0 = kvh * (d.Hq / d.Hkv);
    lo = 0;
    hi = d.Hq / d.Hkv / d.p * span;
    if (splits > 1) {
      const int all = hi, n = parts(d, splits);
      lo = part < n ? int((long long)all * part / n) : 0;
      hi = part < n ? int((long long)all * (part + 1) / n) : 0;
    }
  }
  __device__ int parts(const PackedDims& d, int splits) const { return min(splits, d.Hq / d.Hkv / d.p * span); }
  __device__ int steps() const volatile { return hi - lo; }
  __device__ bool there() const volatile { return lo >= 0; }
};
// The query tile and head set of each step in turn.
struct DkvStep {
  int qt, gi;
  __device__ explicit DkvStep(const DkvItem& w) : qt(w.qt0), gi(0) {
    if (w.lo) {
      gi = w.lo / w.span;
      qt += w.lo - gi * w.span;
    }
  }
  __device__ void next(const DkvItem& w) {
    if (++qt == w.qt0 + w.span) {
      qt = w.qt0;
      ++gi;
    }
  }
};

// CUT: walks may come in parts (the parts' bookkeeping costs the whole walks some 8%).
template <int HD, class T, bool CUT>
__global__ void __launch_bounds__(384, 1) packed_dkv_kernel(const __grid_constant__ PackedBwdMaps maps,
                                                            const __grid_constant__ PackedBwdParams p) {
  using Cfg = PackedDkvCfg<HD>;
  using Tile = HeadTile<HD>;
  constexpr int KVB = Cfg::KVB, SB = Cfg::SB, ST = Cfg::ST;
  constexpr uint32_t TB = Cfg::TB;
  constexpr uint32_t IDESC_SS = idesc_16bit(T::FMT, 128, 128, 0, 0);
  constexpr uint32_t IDESC_KV = idesc_16bit(T::FMT, 128, HD, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  auto sK = [&](int b) { return base + 2 * TB * b; };
  auto sV = [&](int b) { return base + 2 * TB * b + TB; };
  auto sQ = [&](int s) { return base + Cfg::OFF_Q + 2 * TB * s; };
  auto sdO = [&](int s) { return base + Cfg::OFF_Q + 2 * TB * s + TB; };
  float* rows = reinterpret_cast<float*>(smem + Cfg::OFF_ROW);  // [ST][2][128]: -lse2, delta
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  const uint32_t b0 = smem_u32(bars);
  auto kv_full = [&](int b) { return b0 + 8u * b; };
  auto kv_empty = [&](int b) { return b0 + 8u * (2 + b); };
  auto qdo_full = [&](int s) { return b0 + 8u * (4 + s); };
  auto qdo_empty = [&](int s) { return b0 + 8u * (8 + s); };
  auto row_full = [&](int s) { return b0 + 8u * (12 + s); };
  // Per S^T buffer, because with two of them S^T runs a step ahead: a single
  // barrier could complete twice before its waiter looks.
  auto s_full = [&](int b) { return b0 + 8u * (16 + b); };        // S^T computed
  auto p_full = [&](int b) { return b0 + 8u * (18 + b); };        // P^T written over it
  const uint32_t dp_full = b0 + 8u * 20, ds_full = b0 + 8u * 21;  // dP^T computed / dS^T written over it
  const uint32_t acc_full = b0 + 8u * 22, acc_empty = b0 + 8u * 23;  // an item's dK, dV complete / read out
  const uint32_t raw_bar = b0 + 8u * 24, drain_bar = b0 + 8u * 25;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  const Feed<DkvItem> feed{b0 + 8u * 26, b0 + 8u * 30, reinterpret_cast<DkvItem*>(bars + 36)};

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 12; ++i) mbar_init(b0 + 8u * i, 1);
    for (int s = 0; s < ST; ++s) mbar_init(row_full(s), 32);
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(p_full(b), 256);
    }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 256);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 256);
    mbar_init(raw_bar, 1);
    mbar_init(drain_bar, 1);
    static_assert(8 * 36 + Feed<DkvItem>::BYTES <= 768, "barrier space");
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
  if (warp == 0 && p.d.p * p.d.tt < 128) {
    // Rows past p * tt are in no box: cleared once, they stay zero.
    for (int s = 0; s < ST; ++s) {
      zero_rows<HD>(sQ(s), p.d.p * p.d.tt, lane);
      zero_rows<HD>(sdO(s), p.d.p * p.d.tt, lane);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  const int splits = CUT ? p.plan.head->splits : 1;
  const int n_items = p.plan.head->n[LIST_K] * p.d.Hkv * splits;
  Guard g(p.status, KID_PACKED_DKV);

  auto finish = [&]() {  // TMEM is freed once every warp is done with it
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
      const bool lead = lane == 0;
      const uint32_t box = uint32_t(p.d.p * p.d.tt) * 128 * Tile::NCHUNK;
      int kvpar[2] = {-1, -1}, qpar[ST];
      for (int s = 0; s < ST; ++s) qpar[s] = -1;
      int n = 0, item = 0, raw = 0;
      auto draw = [&](int idx) {  // tile idx, or the next one that has steps
        DkvItem w(p.d, p.plan, idx, splits, n_items);
        while (CUT && w.there() && !w.steps()) {
          if (lead) idx = int(gridDim.x) + atomicAdd(p.next + LIST_K, 1);
          w = DkvItem(p.d, p.plan, __shfl_sync(0xffffffffu, idx, 0), splits, n_items);
        }
        return w;
      };
      DkvItem w = draw(blockIdx.x), next;
      if (lead) feed.put(0, w, g);
      while (w.there() && g.ok) {
        const int kb = item % KVB;
        if (lead && (item < KVB || mbar_wait(kv_empty(kb), uint32_t((item / KVB - 1) & 1), g, 1))) {
          mbar_expect_tx(kv_full(kb), 2 * TB);
#pragma unroll
          for (int c = 0; c < Tile::NCHUNK; ++c) {
            tma_load_3d(sK(kb) + c * 16384, &maps.k, kv_full(kb), c * 64, w.kvh, w.seq0 + w.k0);
            tma_load_3d(sV(kb) + c * 16384, &maps.v, kv_full(kb), c * 64, w.kvh, w.seq0 + w.k0);
          }
          kvpar[kb] = (item / KVB) & 1;
        }
        ++item;
        DkvStep at(w);
        for (int k = w.lo; k < w.hi; ++k, ++n, at.next(w)) {
          const int s = n % ST;
          const uint32_t ph = (n / ST) & 1;
          const int t0 = at.qt * p.d.tt;
          // Rows past the sequence's end: P and dS are zero there, but the dV and
          // dK products would still multiply them by whatever the rows hold.
          const int valid = min(w.len - t0, p.d.tt) * p.d.p;
          const bool tail = valid < p.d.p * p.d.tt;
          if (lead && mbar_wait(qdo_empty(s), ph ^ 1, g, 2)) {
            const uint32_t full = tail ? raw_bar : qdo_full(s);
            mbar_expect_tx(full, 2 * box);
#pragma unroll
            for (int c = 0; c < Tile::NCHUNK; ++c) {
              tma_load_3d(sQ(s) + c * 16384, &maps.q, full, c * 64, w.h0 + at.gi * p.d.p, w.seq0 + t0);
              tma_load_3d(sdO(s) + c * 16384, &maps.dO, full, c * 64, w.h0 + at.gi * p.d.p, w.seq0 + t0);
            }
            qpar[s] = int(ph);
          }
          if (k == max(w.hi - 3, w.lo)) {
            int idx = 0;
            if (lead) idx = int(gridDim.x) + atomicAdd(p.next + LIST_K, 1);
            next = draw(__shfl_sync(0xffffffffu, idx, 0));
            if (lead) feed.put(item, next, g);  // (item counts this one already)
          }
          g.ok = __all_sync(0xffffffffu, g.ok);
          if (!g.ok) break;
          if (tail) {
            g.ok = __all_sync(0xffffffffu, mbar_wait(raw_bar, raw & 1, g, 3));
            ++raw;
            if (!g.ok) break;
            zero_rows<HD>(sQ(s), valid, lane);
            zero_rows<HD>(sdO(s), valid, lane);
            fence_proxy_async_smem();
            __syncwarp();
            if (lead) mbar_arrive(qdo_full(s));
          }
        }
        w = next;
      }
      if (lead) {
        if (!g.ok) {
          for (int b = 0; b < KVB; ++b)
            if (kvpar[b] >= 0) mbar_drain(kv_full(b), uint32_t(kvpar[b]));
          for (int s = 0; s < ST; ++s)
            if (qpar[s] >= 0) mbar_drain(qdo_full(s), uint32_t(qpar[s]));
          mbar_drain(raw_bar, uint32_t(raw & 1));
        } else {
          for (int b = 0; b < KVB; ++b)
            if (kvpar[b] >= 0) mbar_wait(kv_empty(b), uint32_t(kvpar[b]), g, 4);
          for (int s = 0; s < ST; ++s)
            if (qpar[s] >= 0) mbar_wait(qdo_empty(s), uint32_t(qpar[s]), g, 5);
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      if (elect_one()) {
        bool any = false;
        // S^T and dP^T run ahead of dV and dK, across items: their next steps.
        // With two S^T buffers S^T may be an item ahead of dP^T, so the steps of up to
        // three items in a row are kept (0: no more).
        int item_steps[3], got = 0;
        auto steps_of = [&](int item) -> int {
          while (got <= item) {
            DkvItem w;
            const int st = feed.get(got, w, g) ? w.steps() : 0;
            if (got % 3 == 0) item_steps[0] = st;
            if (got % 3 == 1) item_steps[1] = st;
            if (got % 3 == 2) item_steps[2] = st;
            ++got;
            if (st == 0) break;
          }
          return item % 3 == 0 ? item_steps[0] : item % 3 == 1 ? item_steps[1] : item_steps[2];
        };
        struct Ahead {
          int n, item, left;  // left = 0: no more steps
        };
        auto advance = [&](Ahead& a) {
          ++a.n;
          if (--a.left == 0) a.left = steps_of(++a.item);
        };
        Ahead as{0, 0, steps_of(0)}, ad = as;
        auto issue_s = [&]() -> bool {  // S^T = K Q^T
          const int kb = as.item % KVB, s = as.n % ST;
          if (!mbar_wait(kv_full(kb), (as.item / KVB) & 1, g, 6)) return false;
          if (!mbar_wait(qdo_full(s), (as.n / ST) & 1, g, 7)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + Cfg::S_COL + 128 * (as.n % SB), Tile::kmajor(sK(kb), 128, kk), Tile::kmajor(sQ(s), 128, kk),
                   IDESC_SS, kk > 0 ? 1u : 0u);
          mma_commit(s_full(as.n % SB));
          any = true;
          advance(as);
          return true;
        };
        auto issue_dp = [&]() -> void {  // dP^T = V dO^T, after the same step's S^T: its operands are there
          const int kb = ad.item % KVB, s = ad.n % ST;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + Cfg::DP_COL, Tile::kmajor(sV(kb), 128, kk), Tile::kmajor(sdO(s), 128, kk), IDESC_SS,
                   kk > 0 ? 1u : 0u);
          mma_commit(dp_full);
          if (ad.left == 1) mma_commit(kv_empty(kb));  // the item's last read of K and V
          advance(ad);
        };
        int n = 0, item = 0;
        if (as.left && issue_s()) issue_dp();
        for (int steps = steps_of(0); steps && g.ok; steps = steps_of(++item)) {
          for (int k = 0; k < steps; ++k, ++n) {
            const int s = n % ST;
            const uint32_t pt = tmem + Cfg::S_COL + 128 * (n % SB), dst = tmem + Cfg::DP_COL;
            // Two S^T buffers: the next one is free once dV of the step before has been issued.
            if (SB == 2 && as.left && !issue_s()) break;
            if (!mbar_wait(p_full(n % SB), (n / SB) & 1, g, 8)) break;
            if (k == 0 && item > 0 && !mbar_wait(acc_empty, (item - 1) & 1, g, 9)) break;
            tc_fence_after();
            // dV += P^T dO: queries [64 hh, 64 hh + 64) of P^T start at column 64 hh.
#pragma unroll
            for (int kc = 0; kc < 8; ++kc)
              mma_ts(tmem + Cfg::DV_COL, pt + (kc >> 2) * 64 + (kc & 3) * 8, Tile::mnmajor(sdO(s), 128, kc), IDESC_KV,
                     (k > 0 || kc > 0) ? 1u : 0u);
            // One buffer: after dV, or after the item's last dK, which should not wait for the next K and V.
            const bool last = k + 1 == steps;
            if (SB == 1 && as.left && !last && !issue_s()) break;
            if (!mbar_wait(ds_full, n & 1, g, 10)) break;
            tc_fence_after();
            // dK += dS^T Q
#pragma unroll
            for (int kc = 0; kc < 8; ++kc)
              mma_ts(tmem + Cfg::DK_COL, dst + (kc >> 2) * 64 + (kc & 3) * 8, Tile::mnmajor(sQ(s), 128, kc), IDESC_KV,
                     (k > 0 || kc > 0) ? 1u : 0u);
            mma_commit(qdo_empty(s));
            if (last) mma_commit(acc_full);
            if (SB == 1 && as.left && last && !issue_s()) break;
            if (ad.left) issue_dp();
          }
        }
        if (!g.ok && any) {
          mma_commit(drain_bar);
          mbar_drain(drain_bar, 0);
        }
      }
    } else if (warp == 2) {
      // ---------------- -lse2 and delta of each step's 128 query rows ----------------
      // (in registers while the stage is still in use)
      int tok[4], head[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tok[i] = token_of(p.d, lane + 32 * i);
        head[i] = lane + 32 * i - tok[i] * p.d.p;
      }
      int n = 0;
      for (int item = 0; g.ok; ++item) {
        const volatile DkvItem& slot = *feed.look(item, g);
        if (!g.ok || !slot.there()) break;
        const DkvItem w = const_cast<const DkvItem&>(slot);
        feed.done(item, lane);
        DkvStep at(w);
        float l[4], d[4];
        auto fetch = [&]() {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = at.qt * p.d.tt + tok[i];
            const bool live = tok[i] < p.d.tt && t < w.len;
            const long long row = (long long)(w.seq0 + t) * p.d.Hq + w.h0 + at.gi * p.d.p + head[i];
            l[i] = live ? -__ldg(p.lse2 + row) : -INFINITY;  // P = 0 in rows that are not there
            d[i] = live ? p.delta[row] : 0.f;
          }
        };
        if (w.lo < w.hi) fetch();
        for (int k = w.lo; k < w.hi; ++k, ++n) {
          const int s = n % ST;
          g.ok = __all_sync(0xffffffffu, mbar_wait(qdo_empty(s), ((n / ST) & 1) ^ 1, g, 11));
          if (!g.ok) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            rows[s * 256 + lane + 32 * i] = l[i];
            rows[s * 256 + 128 + lane + 32 * i] = d[i];
          }
          mbar_arrive(row_full(s));
          at.next(w);
          if (k + 1 < w.hi) fetch();
        }
      }
    }
    finish();
    return;
  }
  reg_alloc<Cfg::REG_SOFTMAX>();
  {
    // ---------------- softmax warps 4..11: key row r, queries [64 hh, 64 hh + 64) ----------------
    const int quarter = warp & 3, hh = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = tmem + (uint32_t(quarter * 32) << 16);
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    WarpRows<true> out(base + Cfg::OFF_OUT + (warp - 4) * WarpRows<true>::BYTES, lane, quarter * 32);
#pragma unroll
    for (int i = 0; i < out.rows(); ++i) out.off[i] = out.row(i) * p.d.Hkv * p.d.N;
    bool ok = true;
    int n = 0, item = 0;
    while (ok) {
      const volatile DkvItem& w = *feed.look(item, g);
      ok = g.ok;
      if (!ok || !w.there()) break;
      const int k0 = w.k0, key = k0 + r, qt0 = w.qt0, qt_end = qt0 + w.span;
      int qt = qt0 + w.lo % w.span;
      for (int k = w.hi - w.lo; k > 0; --k, ++n, qt = qt + 1 == qt_end ? qt0 : qt + 1) {
        const int s = n % ST;
        ok = __all_sync(0xffffffffu, mbar_wait(row_full(s), (n / ST) & 1, g, 12));
        if (!ok) break;
        const int t0 = qt * p.d.tt;
        const bool mask = t0 < k0 + 127;
        const int cmin = p.d.p * (key - t0) - 64 * hh;  // first of this thread's columns that sees the key
        const uint32_t sa = lane_base + Cfg::S_COL + 128 * (n % SB) + 64 * hh;
        const uint32_t da = lane_base + Cfg::DP_COL + 64 * hh;
        // The columns' -lse2 and, below, delta come to registers before the waits for
        // S^T and dP^T: shared memory is busy with the MMAs' operands then.
        auto row_values = [&](int which, float2(&v)[32]) {
          const float4* q = reinterpret_cast<const float4*>(rows + s * 256 + 128 * which + 64 * hh);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float4 f = q[e];
            v[2 * e] = make_float2(f.x, f.y);
            v[2 * e + 1] = make_float2(f.z, f.w);
          }
        };
        float2 P[32], rv[32];
        row_values(0, rv);
        ok = __all_sync(0xffffffffu, mbar_wait(s_full(n % SB), (n / SB) & 1, g, 13));
        if (!ok) break;
        tc_fence_after();
        tmem_load64(sa, P);
#pragma unroll
        for (int e = 0; e < 32; ++e) P[e] = ffma2(P[e], sl2, rv[e]);
        auto probs = [&](auto masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float2 x = exp2_pair(P[8 * c + e], (kPolyPairsBwd >> e) & 1);
              if (masked()) {
                x.x = 16 * c + 2 * e < cmin ? 0.f : x.x;
                x.y = 16 * c + 2 * e + 1 < cmin ? 0.f : x.y;
              }
              P[8 * c + e] = x;
              pk[e] = T::pack(x.x, x.y);
            }
            tmem_st8(sa + 8 * c, pk);  // over columns this thread has read
          }
        };
        if (mask)
          probs(std::true_type());
        else
          probs(std::false_type());
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(n % SB));
        row_values(1, rv);
        ok = __all_sync(0xffffffffu, mbar_wait(dp_full, n & 1, g, 14));
        if (!ok) break;
        tc_fence_after();
        // (Masked entries have P = 0; keys of other sequences are other lanes, their rows of dO are cleared.)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[32], ds[16];
          tmem_load32(da + 32 * h, dp);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = fmul2(P[16 * h + e], fsub2(make_float2(__uint_as_float(dp[2 * e]), __uint_as_float(dp[2 * e + 1])),
                                                        rv[16 * h + e]));
            ds[e] = T::pack(x.x, x.y);
          }
          tmem_st16(da + 16 * h, ds);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full, item & 1, g, 15));
      if (!ok) break;
      tc_fence_after();
      // Warps 4..7 write dV, 8..11 dK.
      const uint32_t acc = lane_base + (hh ? Cfg::DK_COL : Cfg::DV_COL);
      const float sc = hh ? p.scale : 1.0f;
      const long long first = ((long long)(w.seq0 + k0) * p.d.Hkv + w.kvh) * p.d.N;  // of the tile's first row
#pragma unroll
      for (int i = 0; i < out.rows(); ++i) out.live[i] = k0 + out.row(i) < w.len;
#pragma unroll
      for (int c = 0; c < HD; c += 64) {
        float2 v[32];
        tmem_load64(acc + c, v);
        if (c + 64 == HD) {
          tc_fence_before();
          mbar_arrive(acc_empty);
        }
        if (!CUT || splits == 1) {
          uint16_t* tile = (hh ? p.dk : p.dv) + first;
          out.template store32<T>(v, sc, tile, c, p.d.N);
          out.template store32<T>(v + 16, sc, tile, c + 32, p.d.N);
        } else if (key < w.len) {
          float* row = p.parts + (2LL * w.part + (hh ? 0 : 1)) * p.d.total * p.d.Hkv * p.d.N + first + (long long)r * p.d.Hkv * p.d.N;
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            if (c + 2 * e < p.d.N)
              *reinterpret_cast<float4*>(row + c + 2 * e) = make_float4(v[e].x * sc, v[e].y * sc, v[e + 1].x * sc, v[e + 1].y * sc);
        }
      }
      feed.done(item, lane);
      ++item;
    }
    if (!ok) g.ok = false;
    finish();
  }
}

// dK and dV of cut walks: each key tile's parts added in their order and rounded
// once.  A block takes 16 rows of a (tile, key/value head) at a time; nothing to
// do where walks were not cut.
constexpr int SUM_ROWS = 16;
template <class T>
__global__ void __launch_bounds__(256) packed_dkv_sum_kernel(const __grid_constant__ PackedBwdParams p) {
  pdl_wait();
  const int splits = p.plan.head->splits;
  if (splits == 1) return;
  constexpr int CHUNKS = 128 / SUM_ROWS;
  const int n_items = p.plan.head->n[LIST_K] * p.d.Hkv * CHUNKS, vecs = p.d.N / 4;
  const long long set = (long long)p.d.total * p.d.Hkv * p.d.N;
  for (int idx = blockIdx.x; idx < n_items; idx += gridDim.x) {
    const DkvItem w(p.d, p.plan, idx / CHUNKS * splits, splits, n_items / CHUNKS * splits);
    const int row0 = w.k0 + idx % CHUNKS * SUM_ROWS, rows = min(SUM_ROWS, w.len - row0), parts = w.parts(p.d, splits);
    if (rows <= 0) continue;
    const long long first = ((long long)(w.seq0 + row0) * p.d.Hkv + w.kvh) * p.d.N;
    for (int i = threadIdx.x; i < 2 * rows * vecs; i += blockDim.x) {
      const int which = i >= rows * vecs, k = i - which * rows * vecs;
      const long long at = first + (long long)(k / vecs) * p.d.Hkv * p.d.N + 4 * (k % vecs);
      const float4* f = reinterpret_cast<const float4*>(p.parts + which * set + at);
      float4 a = __ldcs(f);
#pragma unroll 4
      for (int s = 1; s < parts; ++s) {
        const float4 g = __ldcs(f + s * (set / 2));  // (2 sets of `set` floats a part)
        a.x += g.x;
        a.y += g.y;
        a.z += g.z;
        a.w += g.w;
      }
      *reinterpret_cast<uint2*>((which ? p.dv : p.dk) + at) = make_uint2(T::pack(a.x, a.y), T::pack(a.z, a.w));
    }
  }
}

template <int HD, class T>
static int launch_packed_bwd(const PackedBwdMaps& maps, const PackedBwdParams& p, cudaStream_t st) {
  static_assert(PackedDqCfg<HD>::SMEM <= 232448 && PackedDkvCfg<HD>::SMEM <= 232448, "shared memory");
  auto dq = packed_dq_kernel<HD, T>;
  auto dkv = p.d.most_splits > 1 ? packed_dkv_kernel<HD, T, true> : packed_dkv_kernel<HD, T, false>;
  if (!smem_attr_set(reinterpret_cast<const void*>(dq), int(PackedDqCfg<HD>::SMEM)) ||
      !smem_attr_set(reinterpret_cast<const void*>(dkv), int(PackedDkvCfg<HD>::SMEM)))
    return set_error(MEA_ERR_CUDA, "cudaFuncSetAttribute(packed backward) failed");
  const int sms = num_sms();
  cudaLaunchAttribute attr;
  const long long nq = (long long)p.d.cap[LIST_Q] * p.d.hg, nk = (long long)p.d.cap[LIST_K] * p.d.Hkv * p.d.most_splits;
  cudaLaunchConfig_t cfg = packed_launch(int(nq < sms ? nq : sms), 384, PackedDqCfg<HD>::SMEM, st, &attr);
  cudaLaunchKernelEx(&cfg, dq, maps, p);
  int rc = check_launch("packed_dq_kernel");
  if (rc != MEA_OK) return rc;
  cfg = packed_launch(int(nk < sms ? nk : sms), 384, PackedDkvCfg<HD>::SMEM, st, &attr);
  cudaLaunchKernelEx(&cfg, dkv, maps, p);
  if ((rc = check_launch("packed_dkv_kernel")) != MEA_OK || p.d.most_splits == 1) return rc;
  const long long blocks = (long long)p.d.cap[LIST_K] * p.d.Hkv * (128 / SUM_ROWS);
  cfg = packed_launch(int(blocks < 8 * sms ? blocks : 8 * sms), 256, 0, st, &attr);
  cudaLaunchKernelEx(&cfg, packed_dkv_sum_kernel<T>, p);
  return check_launch("packed_dkv_sum_kernel");
}

}  // namespace mea

extern "C" int mea_packed_attention_backward(const mea_packed_dims* d, const void* q, const void* k, const void* v,
                                             const void* o, const void* dO, long long do_row, long long do_head,
                                             const float* lse2, const void* plan, size_t plan_bytes, void* workspace,
                                             size_t workspace_bytes, void* dq, void* dk, void* dv, int* status,
                                             void* stream) {
  using namespace mea;
  PackedDims pd;
  int rc = packed_dims(d, &pd);
  if (rc != MEA_OK) return rc;
  if (pd.total == 0) return MEA_OK;
  const long long wq = (long long)pd.Hq * pd.N, wk = (long long)pd.Hkv * pd.N;
  if ((rc = packed_check_rows("q", q, d->q_row, d->q_head, pd, pd.Hq)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("k", k, d->k_row, d->k_head, pd, pd.Hkv)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("v", v, d->v_row, d->v_head, pd, pd.Hkv)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("o", o, wq, pd.N, pd, pd.Hq)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("dO", dO, do_row, do_head, pd, pd.Hq)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("dq", dq, wq, pd.N, pd, pd.Hq)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("dk", dk, wk, pd.N, pd, pd.Hkv)) != MEA_OK) return rc;
  if ((rc = packed_check_rows("dv", dv, wk, pd.N, pd, pd.Hkv)) != MEA_OK) return rc;
  if (!lse2 || !plan || !workspace)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention backward: lse2, plan and workspace must be non-NULL");
  if (reinterpret_cast<uintptr_t>(lse2) & 3 || (reinterpret_cast<uintptr_t>(plan) | reinterpret_cast<uintptr_t>(workspace)) & 255)
    return set_error(MEA_ERR_ALIGNMENT,
                     "packed attention backward: lse2 must be 4-byte, plan and workspace 256-byte aligned");
  if (plan_bytes < packed_plan_bytes(pd))
    return set_error(MEA_ERR_WORKSPACE, "packed attention backward: plan has %zu bytes, needs %zu", plan_bytes,
                     packed_plan_bytes(pd));
  if (workspace_bytes < packed_backward_bytes(pd))
    return set_error(MEA_ERR_WORKSPACE, "packed attention backward: workspace has %zu bytes, needs %zu", workspace_bytes,
                     packed_backward_bytes(pd));
  int* next = static_cast<int*>(workspace);
  float* delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + PACKED_COUNTERS);
  auto st = static_cast<cudaStream_t>(stream);
  if (pd.n_seqs == 0) {  // no sequence owns a row
    if (cudaMemsetAsync(dq, 0, size_t(pd.total) * wq * 2, st) != cudaSuccess ||
        cudaMemsetAsync(dk, 0, size_t(pd.total) * wk * 2, st) != cudaSuccess ||
        cudaMemsetAsync(dv, 0, size_t(pd.total) * wk * 2, st) != cudaSuccess)
      return set_error(MEA_ERR_CUDA, "packed attention backward: clearing the gradients failed");
    return MEA_OK;
  }
  PackedBwdMaps maps;
  rc = packed_map(&maps.q, pd, d->dtype, q, d->q_row, d->q_head, pd.Hq, pd.p, pd.tt);
  rc |= packed_map(&maps.dO, pd, d->dtype, dO, do_row, do_head, pd.Hq, pd.p, pd.tt);
  rc |= packed_map(&maps.k, pd, d->dtype, k, d->k_row, d->k_head, pd.Hkv, 1, 128);
  rc |= packed_map(&maps.v, pd, d->dtype, v, d->v_row, d->v_head, pd.Hkv, 1, 128);
  if (rc) return set_error(MEA_ERR_CUDA, "packed attention backward: tensor map encode failed (%d)", rc);
  PackedBwdParams p;
  p.d = pd;
  p.plan = packed_plan_view(pd, const_cast<void*>(plan));  // read only
  p.scale = d->scale;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.lse2 = lse2;
  p.delta = delta;
  p.next = next;
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + PACKED_COUNTERS + packed_delta_bytes(pd));
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.status = status;
  const long long rows = (long long)pd.total * pd.Hq, blocks = (rows + DELTA_ROWS - 1) / DELTA_ROWS;
  if (blocks > 0x7fffffffLL)
    return set_error(MEA_ERR_UNSUPPORTED_SHAPE, "packed attention backward: %d rows x %d heads are too many", pd.total, pd.Hq);
  const bool bf = d->dtype == MEA_BF16;
  (bf ? packed_delta_kernel<Bf16> : packed_delta_kernel<Fp16>)<<<unsigned(blocks), 256, 0, st>>>(
      pd, p.plan.head, next, static_cast<const uint16_t*>(o), static_cast<const uint16_t*>(dO), do_row, do_head, delta,
      static_cast<uint4*>(dq), static_cast<uint4*>(dk), static_cast<uint4*>(dv));
  if ((rc = check_launch("packed_delta_kernel")) != MEA_OK) return rc;
  if (bf) return pd.N <= 64 ? launch_packed_bwd<64, Bf16>(maps, p, st) : launch_packed_bwd<128, Bf16>(maps, p, st);
  return pd.N <= 64 ? launch_packed_bwd<64, Fp16>(maps, p, st) : launch_packed_bwd<128, Fp16>(maps, p, st);
}
