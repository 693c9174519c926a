// What the packed-sequence attention kernels share: the work plan, element
// types, tile geometry and masks.
//
// Layout.  q, o are [total, Hq, N]; k, v are [total, Hkv, N]; sequence s owns
// rows cu[s] .. cu[s+1], and query head h reads key/value head h / G with
// G = Hq / Hkv.  A query tile holds `tt` consecutive tokens of one sequence
// times `p` neighbouring heads of one group (p divides G), token-major: tile
// row r is token r / p, head r % p.  One 3-D TMA box {64 elements, p heads, tt
// tokens} brings it in, so a group's heads share every K/V tile that is loaded
// and a short sequence still fills rows of the 128-row MMA.
//
// Head dims up to 64 run as HD = 64 and up to 128 as HD = 128: TMA fills the
// columns past N with zeros, which add nothing to a score or a product.
#pragma once
#include <cuda_fp16.h>

#include "attn_common.cuh"

namespace mea {

// ---- work plan (device memory, written by packed_plan_kernel) ----
// header, then three lists of int4 entries, one per tile: query tiles (the dQ
// kernel's), 128-row key tiles, and the forward's items of one or two query
// tiles.  An entry is {first row of the sequence, its length, z, by_tile}.
// Tile number idx of the whole list belongs to entry idx / heads.  by_tile = 1:
// the entry is tile z and the head idx % heads.  by_tile = 0: z tiles are listed
// before the sequence's own nt entries, and there idx - z * heads = head * nt + n
// for the n-th tile from the one that takes longest.
struct PackedHeader {
  int n[3];        // entries of each list
  int first, end;  // rows [first, end) belong to sequences
  int next;        // next forward item to be drawn
  int splits;      // parts that a key tile's walk is cut into
  int pad;
};

struct PackedDims {
  int total, n_seqs, Hq, Hkv, N;
  int p, tt;        // heads and tokens of a query tile
  int p_inv;        // ceil(2^16 / p)
  int hg;           // query tiles per token tile: Hq / p
  int streams;      // query tiles of a forward item
  int rows[3];      // tokens of a tile of each list
  int heads[3];     // tiles per entry: head groups, or key/value heads
  int cap[3];       // entries there can be
  int most_splits;  // parts that a key tile's walk may be cut into
};

// The token of a query tile's row: row / p, exact for rows below 128.
__device__ __forceinline__ int token_of(const PackedDims& d, int row) { return row * d.p_inv >> 16; }

enum PackedList { LIST_Q = 0, LIST_K = 1, LIST_FWD = 2 };
struct PackedPlan {
  PackedHeader* head;
  int4* list[3];
};

// ---- element types ----
struct Bf16 {
  static constexpr uint32_t FMT = 1;
  static constexpr uint32_t EXP = 0x7F80;  // exponent field: all ones is inf or NaN
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
  __device__ static __forceinline__ float lo(uint32_t v) { return bf16_lo(v); }
  __device__ static __forceinline__ float hi(uint32_t v) { return bf16_hi(v); }
  // acc + 0 * v per half: stays 0 unless v holds an inf or NaN.
  __device__ static __forceinline__ void probe(uint32_t& acc, uint32_t v) {
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0u));
  }
};
struct Fp16 {
  static constexpr uint32_t FMT = 0;
  static constexpr uint32_t EXP = 0x7C00;
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ float lo(uint32_t v) { return __half2float(__ushort_as_half(uint16_t(v))); }
  __device__ static __forceinline__ float hi(uint32_t v) { return __half2float(__ushort_as_half(uint16_t(v >> 16))); }
  __device__ static __forceinline__ void probe(uint32_t& acc, uint32_t v) {
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0u));
  }
};
template <class T>
__device__ __forceinline__ bool half_nonfinite(uint32_t h) {
  return (h & T::EXP) == T::EXP;
}

// ---- shared memory ----
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Rows [r0, 128) of a [128 x HD] tile (64-column chunks of 128-byte rows) to
// zero, by one warp.  A whole row is cleared, so the swizzle does not matter.
template <int HD>
__device__ __forceinline__ void zero_rows(uint32_t tile, int r0, int lane) {
  const int units = (128 - r0) * 8;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c)
    for (int u = lane; u < units; u += 32) sts128(tile + c * 16384 + r0 * 128 + u * 16, 0, 0, 0, 0);
}

// Tiles of a persistent CTA: warp 0 draws the next number from a counter (long
// tiles first, so the CTAs end together), works out where the tile lies, and hands
// that to the other roles through a ring of four slots, three steps before the
// present tile's last loads (drawn earlier, it would wait behind a long tile while
// other CTAs run out of work); each reader gives the slot back.  Working it out
// costs a read of the plan and two divisions; with every role doing that for itself
// 64 documents took 92 us forward instead of 85, 16384 tokens with 16/2 heads 1902
// us of dK/dV instead of 1804.  Which CTA takes a tile changes no result.
template <class Item>
struct Feed {
  static constexpr int SLOTS = 4, WORDS = sizeof(Item) / 4;
  static constexpr uint32_t BYTES = SLOTS * sizeof(Item);
  uint32_t full, empty;  // mbarriers, SLOTS each
  Item* slot;
  __device__ void put(int n, const Item& w, Guard& g) const {  // one thread
    if (!mbar_wait(empty + 8u * (n % SLOTS), ((n / SLOTS) & 1) ^ 1, g, 30)) return;
    slot[n % SLOTS] = w;
    mbar_arrive(full + 8u * (n % SLOTS));
  }
  __device__ bool get(int n, Item& w, Guard& g) const {  // one thread; false: no more tiles
    if (!mbar_wait(full + 8u * (n % SLOTS), (n / SLOTS) & 1, g, 31)) return false;
    w = slot[n % SLOTS];
    mbar_arrive(empty + 8u * (n % SLOTS));
    return w.there();
  }
  // A whole warp: the tile stays in its slot (where its fields cost no registers)
  // until done().
  __device__ const volatile Item* look(int n, Guard& g) const {
    g.ok = __all_sync(0xffffffffu, mbar_wait(full + 8u * (n % SLOTS), (n / SLOTS) & 1, g, 31));
    return slot + n % SLOTS;
  }
  __device__ void done(int n, int lane) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8u * (n % SLOTS));
  }
};

// Where tile idx of a list lies: sequence, head (group) and the tile in it.
// LAST_FIRST: a sequence's last tile takes longest (query tiles), else its first.
template <bool LAST_FIRST>
struct PackedTile {
  int seq0, len, head, tile;
  __device__ __forceinline__ PackedTile(const int4* items, int idx, int heads, int rows) {
    const int i = idx / heads;
    const int4 e = items[i];
    seq0 = e.x;
    len = e.y;
    head = idx - i * heads;
    tile = e.z;
    if (!e.w) {
      const int nt = (len + rows - 1) / rows, off = idx - e.z * heads;
      head = off / nt;
      tile = off - head * nt;
      if (LAST_FIRST) tile = nt - 1 - tile;
    }
  }
};

// 64 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_load64(uint32_t taddr, float2 (&v)[32]) {
  uint32_t a[32], b[32];
  tmem_ld32(taddr, a);
  tmem_ld32(taddr + 32, b);
  tmem_wait_ld_tied2x32(a, b);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    v[e] = make_float2(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1]));
    v[16 + e] = make_float2(__uint_as_float(b[2 * e]), __uint_as_float(b[2 * e + 1]));
  }
}

// A warp's 32 rows, one per lane, to global memory, 32 columns at a time.  STAGED:
// through 2 KB of shared memory.  With one row per lane a store instruction touches
// 32 rows (and takes as many passes); through shared memory it writes 64 bytes of
// each of eight, but shared memory is busy with the MMAs' operands.  Measured: the
// dK/dV kernel gains at both head dims (16 documents of up to 2048 tokens, 8 heads
// of 64: 144 -> 138 us; 16 x 2048 tokens, 16 heads of 128: 648 -> 623), the forward
// at 128 (377 -> 362), where 64 loses (92 -> 98).
template <bool STAGED>
struct WarpRows {
  static constexpr uint32_t BYTES = STAGED ? 2048 : 0;
  uint32_t buf;
  int lane, row0;
  int off[4];    // STAGED: element offsets of rows lane / 4 + 8 i; else [0]: of the lane's own row
  bool live[4];  // which of them are written
  __device__ WarpRows(uint32_t buf_, int lane_, int first_row) : buf(buf_), lane(lane_), row0(first_row) {}
  __device__ static constexpr int rows() { return STAGED ? 4 : 1; }
  __device__ int row(int i) const { return row0 + (STAGED ? (lane >> 2) + 8 * i : lane); }
  // Columns [col, col + 32) of this lane's row times `scale`, n columns in all.
  template <class T>
  __device__ __forceinline__ void store32(const float2* v, float scale, uint16_t* out, int col, int n) const {
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = T::pack(v[e].x * scale, v[e].y * scale);
    if constexpr (!STAGED) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (live[0] && col + 8 * u < n)
          st_global_v4(out + off[0] + col + 8 * u, w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    } else {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      sts128(buf + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4), w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    __syncwarp();
    const int unit = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + 8 * i;
      uint32_t x[4];
      lds128(buf + r * 64 + ((unit ^ ((r >> 1) & 3)) << 4), x);
      if (live[i] && col + 8 * unit < n) st_global_v4(out + off[i] + col + 8 * unit, x[0], x[1], x[2], x[3]);
    }
    __syncwarp();
    }
  }
};

// Rows of `width` 16-byte units outside [first, end) of a [total, width] output
// to zero, spread over the grid: no sequence owns them.
__device__ __forceinline__ void zero_outside(uint4* out, int total, int first, int end, long long width, int block,
                                             int blocks, int thread, int threads) {
  const int behind = total - end;
  for (int r = block; r < first + behind; r += blocks) {
    uint4* row = out + (long long)(r < first ? r : end + (r - first)) * width;
    for (long long u = thread; u < width; u += threads) row[u] = make_uint4(0, 0, 0, 0);
  }
}

}  // namespace mea
