// Layer norm over the last dimension, forward and backward.
//
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w,  xhat = (x - mean) rstd
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  dw = sum_rows dy xhat,  db = sum_rows dy
//
// Both directions are bound by HBM: the forward reads x and writes y, the
// backward reads x and dy and writes dx.  A row stays in the registers of the
// TPR threads that share it, so it is read once although the variance is taken
// about the mean (a second sum, not a difference of large ones).  In the
// backward each thread keeps its own columns for every row that its block takes,
// so dw and db grow in registers; each block writes one fp32 partial row and a
// second kernel adds those in a fixed order.  All sums are fp32.  Either way the
// next rows are on their way while the present ones are summed: forward in
// registers, backward in shared memory.  65536 x 2048 bf16 takes 92 us forward
// (5.8 TB/s; 106 us without the second row) and 138 us backward with its column
// sums (5.8 TB/s; 152 us with the second rows in registers, 185 without).
//
// Rows too long for that (above 512 x 8 16-byte vectors forward and 512 x 32
// elements backward; 16384 and 8192 elements where a row is no whole number of
// vectors) take kernels that walk the row several times,
// and a column-wise pass for dw and db.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "ptx.cuh"

namespace mea {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// VEC values at p (VEC = 1, or 16 bytes of T; weights of another type take two 16-byte loads).
template <int VEC, class T>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f(*p);
  } else {
    constexpr int PER = 16 / sizeof(T);
    static_assert(VEC % PER == 0, "");
#pragma unroll
    for (int i = 0; i < VEC / PER; ++i) {
      const uint4 r = reinterpret_cast<const uint4*>(p)[i];
      T t[PER];
      *reinterpret_cast<uint4*>(t) = r;
#pragma unroll
      for (int e = 0; e < PER; ++e) f[i * PER + e] = to_f(t[e]);
    }
  }
}
template <int VEC, class T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(f[0]);
  } else {
    T t[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = from_f<T>(f[e]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(t);
  }
}

// Sums K values (a power of two) over each group of TPR threads; every thread
// gets the sums.  Within a warp the values are folded onto each other first (each
// step halves the values a lane carries), so K sums cost about K + 5 shuffles
// instead of 5 K.  One block barrier when a group has several warps: `red` holds
// two sets, used in turn.
template <int TPR, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* red, int& turn) {
  const int lane = threadIdx.x & 31;
  int m = 16;
#pragma unroll
  for (int n = K / 2; n >= 1; n /= 2, m /= 2) {
    const bool upper = lane & m;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = upper ? v[i] : v[i + n];
      v[i] = (upper ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, give, m);
    }
  }
  float t = v[0];
#pragma unroll
  for (; m; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
  // Lane l now holds the sum of value l / (32 / K).
  if constexpr (TPR == 32) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = K == 1 ? t : __shfl_sync(0xffffffffu, t, k * (32 / K));
  } else {
    constexpr int WARPS = TPR / 32;
    const int warp = threadIdx.x >> 5, all = blockDim.x >> 5;
    float* r = red + turn * all * K;
    turn ^= 1;
    if (lane % (32 / K) == 0) r[warp * K + lane / (32 / K)] = t;
    named_bar_sync(1 + threadIdx.x / TPR, TPR);  // the group's own threads only
    const float* first = r + (warp / WARPS) * WARPS * K;
    t = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS * K; i += 32)
      if (i + lane < WARPS * K) t += first[i + lane];  // value lane % K of several warps
#pragma unroll
    for (int d = 16; d >= K; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = K == 1 ? t : __shfl_sync(0xffffffffu, t, k);
  }
}

template <int TPR>
constexpr int ln_threads() {
  return TPR > 256 ? TPR : 256;
}

// What one thread holds of a row, as it lies in memory: V vectors of 16 bytes, or
// V single elements.  pair(i) converts elements 2 i and 2 i + 1 (element v VEC + e
// is column (v TPR + lane) VEC + e); columns past C hold zero.
template <class T, int VEC, int TPR, int V>
struct Row {
  static constexpr int PAIRS = V * VEC / 2;
  static_assert(VEC > 1 || V % 2 == 0, "");
  typename std::conditional<VEC == 1, T, uint4>::type r[V];
  __device__ __forceinline__ void load(const T* row, int lane, int C, bool live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * TPR + lane) * VEC;
      if constexpr (VEC == 1)
        r[v] = live && c < C ? row[c] : from_f<T>(0.f);
      else
        r[v] = live && c < C ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (VEC == 1) {
      return make_float2(to_f(r[2 * i]), to_f(r[2 * i + 1]));
    } else {
      const uint4& q = r[2 * i / VEC];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      const int k = i % (VEC / 2);
      if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(bf16_lo(w[k]), bf16_hi(w[k]));
      return __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    }
  }
};
// Stores PAIRS pairs as T at the thread's columns of `row`.
template <class T, int VEC, int TPR, int V>
__device__ __forceinline__ void store_row(T* row, int lane, int C, const float2 (&f)[V * VEC / 2]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * TPR + lane) * VEC;
    if (c >= C) continue;
    if constexpr (VEC == 1) {
      row[c] = from_f<T>(v & 1 ? f[v / 2].y : f[v / 2].x);
    } else {
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        o[e] = f[(v * VEC + e) / 2].x;
        o[e + 1] = f[(v * VEC + e) / 2].y;
      }
      store_vec<VEC>(row + c, o);
    }
  }
}
// The thread's columns of a weight vector as pairs; `none` where there is no vector or no column.
template <class W, int VEC, int TPR, int V>
__device__ __forceinline__ void load_cols(const W* w, int lane, int C, float none, float2 (&f)[V * VEC / 2]) {
  float t[V * VEC];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * TPR + lane) * VEC;
    float x[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = none;
    if (w && c < C) load_vec<VEC>(w + c, x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[v * VEC + e] = x[e];
  }
#pragma unroll
  for (int i = 0; i < V * VEC / 2; ++i) f[i] = make_float2(t[2 * i], t[2 * i + 1]);
}
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }

template <int TPR, int ELEMS>
constexpr int ln_fwd_blocks() {
  constexpr int threads = ELEMS > 32 ? 640 : 768;
  return threads / ln_threads<TPR>() ? threads / ln_threads<TPR>() : 1;
}
template <class T, class W, int VEC, int TPR, int V>
__global__ void __launch_bounds__(ln_threads<TPR>(), ln_fwd_blocks<TPR, VEC * V>()) layernorm_fwd_kernel(long long rows, int C, float eps,
                                                                         const T* __restrict__ x,
                                                                         const W* __restrict__ w,
                                                                         const W* __restrict__ b, T* __restrict__ y,
                                                                         float* __restrict__ mean_out,
                                                                         float* __restrict__ rstd_out) {
  constexpr int THREADS = ln_threads<TPR>(), GROUPS = THREADS / TPR, PAIRS = V * VEC / 2;
  __shared__ float red[2 * THREADS / 32];
  int turn = 0;
  const int g = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const float inv_c = 1.0f / float(C);
  const long long step = (long long)gridDim.x * GROUPS;
  long long row0 = (long long)blockIdx.x * GROUPS;
  Row<T, VEC, TPR, V> next;
  next.load(x + (row0 + g) * C, lane, C, row0 + g < rows);
  for (; row0 < rows; row0 += step) {
    const long long row = row0 + g;
    const bool live = row < rows;
    const Row<T, VEC, TPR, V> a = next;
    next.load(x + (row + step) * C, lane, C, row + step < rows);  // on its way while this row is summed
    float2 acc = two(0.f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) acc = fadd2(acc, a.pair(i));
    float s[1] = {acc.x + acc.y};
    group_sum<TPR>(s, red, turn);
    const float mean = s[0] * inv_c;
    acc = two(0.f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      // columns past C (whole vectors, or single elements) stay out of the variance
      float2 d = fsub2(a.pair(i), two(mean));
      const int v = 2 * i / VEC;
      if ((v * TPR + lane) * VEC >= C) d.x = 0.f;
      if (((VEC == 1 ? v + 1 : v) * TPR + lane) * VEC >= C) d.y = 0.f;
      acc = ffma2(d, d, acc);
    }
    s[0] = acc.x + acc.y;
    group_sum<TPR>(s, red, turn);
    const float rstd = 1.0f / sqrtf(s[0] * inv_c + eps);
    if (!live) continue;  // the loop's trip count is the block's, not the group's
    if (lane == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * TPR + lane) * VEC;
      if (c >= C) continue;
      float ww[VEC], bb[VEC], o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        ww[e] = 1.f;
        bb[e] = 0.f;
      }
      if (w) load_vec<VEC>(w + c, ww);
      if (b) load_vec<VEC>(b + c, bb);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 f = a.pair((v * VEC + e) / 2);
        o[e] = fmaf((((v * VEC + e) & 1 ? f.y : f.x) - mean) * rstd, ww[e], bb[e]);
      }
      store_vec<VEC>(y + row * C + c, o);
    }
  }
}

// Asynchronous copies to shared memory; each thread waits for its own.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool live) {  // zeros if not live
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rounds of rows on their way in the backward: a ring of STAGES in shared memory,
// where every thread puts and finds its own vectors (no barrier), and every warp
// its rows' statistics.  Between 32 and 64 KB on their way an SM is best, more is
// slower: 131072 x 1024 bf16, two blocks of 16 KB stages an SM, takes 132 us with
// two stages, 144 with three, 148 with four; 32768 x 4096, one block of 32 KB
// stages, 142, 132 and 142.  A row that leaves room for one stage only (16384
// fp32) still gains by it: 163 us for 4096 rows, 351 through registers that spill.
// Rows of single elements have the next round in registers.
template <int VEC, int TPR, int V, int R>
struct LnRing {
  static constexpr int THREADS = ln_threads<TPR>(), SLOTS = 2 * R * V;  // 16-byte vectors of a thread and round
  static constexpr uint32_t ROWS = SLOTS * THREADS * 16, STAGE = ROWS + THREADS / 32 * 2 * R * 4;
  static constexpr bool USED = VEC > 1;
  static constexpr int STAGES = !USED || ROWS > 65536 ? 1 : THREADS > 256 && ROWS <= 32768 ? 3 : 2;
  static constexpr uint32_t BYTES = USED ? STAGES * STAGE : 0;
};

// R rows per group and round; block i takes every gridDim.x-th round, and the
// next rounds' rows are on their way while this one's are summed.  Partial sums of
// the block's rows: part[(2 i) C ..] for dw, part[(2 i + 1) C ..] for db.
// Columns past C hold dy = 0 and add nothing to any sum.
template <class T, class W, int VEC, int TPR, int V, int R>
__global__ void __launch_bounds__(ln_threads<TPR>(), 512 / ln_threads<TPR>()) layernorm_bwd_kernel(
    long long rows, int C, const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int THREADS = ln_threads<TPR>(), GROUPS = THREADS / TPR, PAIRS = V * VEC / 2;
  using Ring = LnRing<VEC, TPR, V, R>;
  constexpr bool AGAIN = Ring::USED && V * VEC > 16;  // rows and weights read again for dx, instead of 4 V VEC more registers
  __shared__ float red[2 * 2 * R * THREADS / 32];
  extern __shared__ __align__(16) char ring[];
  float* cols = reinterpret_cast<float*>(ring);  // [2][C] at the end, only with several groups
  pdl_launch();
  int turn = 0;
  const int g = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  const float inv_c = 1.0f / float(C);
  float2 ww[PAIRS], dw[PAIRS], db[PAIRS];
  load_cols<W, VEC, TPR, V>(w, lane, C, 1.f, ww);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) dw[i] = db[i] = two(0.f);
  struct Rows {
    Row<T, VEC, TPR, V> x[R], d[R];
    float mean[R], rstd[R];
  };
  const long long step = (long long)gridDim.x * GROUPS * R;
  long long row0 = (long long)blockIdx.x * GROUPS * R;
  auto fetch = [&](Rows& a, long long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + g * R + r;
      const bool live = row < rows;
      a.x[r].load(x + row * C, lane, C, live);
      a.d[r].load(dy + row * C, lane, C, live);
      a.mean[r] = live ? mean_in[row] : 0.f;
      a.rstd[r] = live ? rstd_in[row] : 0.f;  // xhat = 0 in rows that are not there
    }
  };
  auto start = [&](int stage, long long row0) {
    const uint32_t at = smem_u32(ring) + stage * Ring::STAGE + threadIdx.x * 16;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + g * R + r;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + lane) * VEC;
        const bool live = row < rows && c < C;
        const long long from = live ? row * C + c : 0;
        copy_async16(at + (2 * (r * V + v)) * THREADS * 16, x + from, live);
        copy_async16(at + (2 * (r * V + v) + 1) * THREADS * 16, dy + from, live);
      }
    }
    const int k = threadIdx.x & 31;
    if (k < 2 * R) {
      const long long row = row0 + g * R + (k >> 1);
      copy_async4(smem_u32(ring) + stage * Ring::STAGE + Ring::ROWS + (threadIdx.x >> 5) * 2 * R * 4 + k * 4,
                  (k & 1 ? rstd_in : mean_in) + (row < rows ? row : 0), row < rows);
    }
    copy_async_commit();
  };
  auto collect = [&](Rows& a, int stage) {
    const char* at = ring + stage * Ring::STAGE;
    const float* stats = reinterpret_cast<const float*>(at + Ring::ROWS) + (threadIdx.x >> 5) * 2 * R;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint4* q = reinterpret_cast<const uint4*>(at) + 2 * (r * V + v) * THREADS + threadIdx.x;
        if constexpr (Ring::USED) {
          a.x[r].r[v] = q[0];
          a.d[r].r[v] = q[THREADS];
        }
      }
      a.mean[r] = stats[2 * r];
      a.rstd[r] = stats[2 * r + 1];
    }
  };
  Rows a;
  int stage = 0;
  if constexpr (Ring::USED) {
#pragma unroll
    for (int s = 0; s < Ring::STAGES - 1; ++s) start(s, row0 + s * step);
  } else {
    if (row0 < rows) fetch(a, row0);
  }
  for (; row0 < rows; row0 += step) {
    Rows next;
    if constexpr (Ring::USED) {
      // Into the slot of the round before, which this warp has read.
      start(stage ? stage - 1 : Ring::STAGES - 1, row0 + (Ring::STAGES - 1) * step);
      copy_async_wait<Ring::STAGES - 1>();
      __syncwarp();
      collect(a, stage);
    } else if (row0 + step < rows) {
      fetch(next, row0 + step);
    }
    float sums[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float2 rs = two(a.rstd[r]), mr = two(-a.mean[r] * a.rstd[r]);
      float2 s1 = two(0.f), s2 = two(0.f);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 xh = ffma2(a.x[r].pair(i), rs, mr), d = a.d[r].pair(i), gg = fmul2(d, ww[i]);
        s1 = fadd2(s1, gg);
        s2 = ffma2(gg, xh, s2);
        dw[i] = ffma2(d, xh, dw[i]);
        db[i] = fadd2(db[i], d);
      }
      sums[2 * r] = s1.x + s1.y;
      sums[2 * r + 1] = s2.x + s2.y;
    }
    group_sum<TPR>(sums, red, turn);
    if constexpr (AGAIN) {
      collect(a, stage);
      load_cols<W, VEC, TPR, V>(w, lane, C, 1.f, ww);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + g * R + r;
      if (row >= rows) continue;
      const float2 rs = two(a.rstd[r]), mr = two(-a.mean[r] * a.rstd[r]);
      const float2 m1 = two(-sums[2 * r] * inv_c * a.rstd[r]), m2 = two(-sums[2 * r + 1] * inv_c * a.rstd[r]);
      float2 o[PAIRS];
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 xh = ffma2(a.x[r].pair(i), rs, mr);
        o[i] = ffma2(fmul2(a.d[r].pair(i), ww[i]), rs, ffma2(xh, m2, m1));
      }
      store_row<T, VEC, TPR, V>(dx + row * C, lane, C, o);
    }
    if constexpr (Ring::USED) {
      if constexpr (AGAIN) load_cols<W, VEC, TPR, V>(w, lane, C, 1.f, ww);
      if (++stage == Ring::STAGES) stage = 0;
      __syncwarp();  // the statistics are read before a lane copies over them
    } else {
      a = next;
    }
  }
  if constexpr (Ring::USED) {
    copy_async_wait<0>();
    __syncthreads();  // the ring becomes `cols`
  }
  if (!part) return;
  auto at = [](const float2* f, int i) { return i & 1 ? f[i >> 1].y : f[i >> 1].x; };
  float* out = part + (long long)blockIdx.x * 2 * C;
  if (GROUPS > 1) {  // the groups' sums, added in their order
    for (int k = 0; k < GROUPS; ++k) {
      if (g == k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = (v * TPR + lane) * VEC;
          if (c >= C) continue;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            cols[c + e] = (k ? cols[c + e] : 0.f) + at(dw, v * VEC + e);
            cols[C + c + e] = (k ? cols[C + c + e] : 0.f) + at(db, v * VEC + e);
          }
        }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * C; i += THREADS) out[i] = cols[i];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * TPR + lane) * VEC;
      if (c >= C) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        out[c + e] = at(dw, v * VEC + e);
        out[C + c + e] = at(db, v * VEC + e);
      }
    }
  }
}

// dw (blockIdx.y = 0) and db (1): column sums of `n` partial rows, 32 columns a
// block, 32 slices of rows added in order, then the slices in order.
template <class W>
__global__ void __launch_bounds__(1024) layernorm_cols_kernel(int n, int C, const float* __restrict__ part,
                                                              W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float s[32][33];
  pdl_wait();
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  float a = 0.f;
  if (c < C)
    for (int i = threadIdx.y; i < n; i += 32) a += part[((long long)2 * i + blockIdx.y) * C + c];
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += s[i][threadIdx.x];
    out[c] = from_f<W>(t);
  }
}

// ---- rows longer than the register path takes: one block per row, the row walked several times ----
__device__ __forceinline__ float block_sum(float v, float* red, int& turn) {
  float a[1] = {v};
  group_sum<1024>(a, red, turn);
  return a[0];
}
template <class T, class W>
__global__ void __launch_bounds__(1024) layernorm_fwd_long_kernel(long long rows, int C, float eps,
                                                                  const T* __restrict__ x, const W* __restrict__ w,
                                                                  const W* __restrict__ b, T* __restrict__ y,
                                                                  float* __restrict__ mean_out,
                                                                  float* __restrict__ rstd_out) {
  __shared__ float red[64];
  int turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * C;
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) s += to_f(xr[c]);
    const float mean = block_sum(s, red, turn) / float(C);
    s = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = to_f(xr[c]) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, red, turn) / float(C) + eps);
    if (threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int c = threadIdx.x; c < C; c += 1024)
      y[row * C + c] = from_f<T>((to_f(xr[c]) - mean) * rstd * (w ? to_f(w[c]) : 1.f) + (b ? to_f(b[c]) : 0.f));
  }
}
template <class T, class W>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_kernel(long long rows, int C, const T* __restrict__ dy,
                                                                  const T* __restrict__ x, const W* __restrict__ w,
                                                                  const float* __restrict__ mean_in,
                                                                  const float* __restrict__ rstd_in,
                                                                  T* __restrict__ dx) {
  __shared__ float red[64];
  int turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * C, *dr = dy + row * C;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float gg = to_f(dr[c]) * (w ? to_f(w[c]) : 1.f);
      s1 += gg;
      s2 += gg * ((to_f(xr[c]) - mean) * rstd);
    }
    const float m1 = block_sum(s1, red, turn) / float(C), m2 = block_sum(s2, red, turn) / float(C);
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float gg = to_f(dr[c]) * (w ? to_f(w[c]) : 1.f);
      dx[row * C + c] = from_f<T>(rstd * (gg - m1 - (to_f(xr[c]) - mean) * rstd * m2));
    }
  }
}
// Partial column sums: block (i, j) adds rows i, i + gridDim.y, ... of columns [256 j, 256 j + 256).
template <class T>
__global__ void __launch_bounds__(256) layernorm_part_long_kernel(long long rows, int C, const T* __restrict__ dy,
                                                                  const T* __restrict__ x,
                                                                  const float* __restrict__ mean_in,
                                                                  const float* __restrict__ rstd_in,
                                                                  float* __restrict__ part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = to_f(dy[row * C + c]);
    dw += d * ((to_f(x[row * C + c]) - mean_in[row]) * rstd_in[row]);
    db += d;
  }
  part[((long long)2 * blockIdx.y) * C + c] = dw;
  part[((long long)2 * blockIdx.y + 1) * C + c] = db;
}

// ---------------------------------------------------------------- host side
// Register path: TPR threads with V vectors of VEC elements each hold a row.
struct LnShape {
  int vec, tpr, v;  // v = 0: the long-row kernels
};
// Forward: one warp per row while it holds it in 8 vectors a lane, because then no
// barrier stands between the row's load and its store (65536 x 2048 bf16: 92 us
// with one warp of 8 vectors a lane, 102 with two of 4, 117 with four of 2);
// longer rows take more warps, and so do rows too few to give every SM a block.
static LnShape ln_fwd_shape(long long rows, int C, int elem, bool aligned) {
  LnShape s;
  s.vec = aligned && C % (16 / elem) == 0 ? 16 / elem : 1;
  const int units = (C + s.vec - 1) / s.vec, least = s.vec == 1 ? 8 : 1, most = 8;
  s.tpr = 32;
  while (s.tpr < 512 && s.tpr * most < units) s.tpr *= 2;
  s.v = least;
  while (s.tpr * s.v < units) s.v *= s.vec == 1 ? 4 : 2;
  if (s.v > (s.vec == 1 ? 32 : 8)) {
    s.v = 0;
    return s;
  }
  while (s.vec > 1 && s.v > least && s.tpr < 256 && rows * s.tpr < (long long)num_sms() * 256) {
    s.tpr *= 2;
    s.v /= 2;
  }
  return s;
}
// Backward: a thread also keeps two sums per column, so TPR grows before V.
static LnShape ln_bwd_shape(int C, int elem, bool aligned) {
  LnShape s;
  s.vec = aligned && C % (16 / elem) == 0 ? 16 / elem : 1;
  const int units = (C + s.vec - 1) / s.vec;
  s.tpr = 32;
  const int most = s.vec == 1 ? 8 : 1;  // vectors (or single elements) a thread takes before the next doubling of TPR
  while (s.tpr < 512 && s.tpr * most < units) s.tpr *= 2;
  s.v = most;
  while (s.tpr * s.v < units) s.v *= 2;
  if (s.vec * s.v > (s.vec == 1 ? 16 : 32)) s.v = 0;
  return s;
}
constexpr int LN_LONG_PARTS = 64;
constexpr int LN_MAX_PARTS = 2 * 160;  // partial rows of dw and db: one per block, two blocks an SM

static int ln_bwd_blocks(long long rows, const LnShape& s, int rows_per_round) {
  const int threads = s.tpr > 256 ? s.tpr : 256, groups = threads / s.tpr;
  const long long rounds = (rows + (long long)groups * rows_per_round - 1) / ((long long)groups * rows_per_round);
  return int(std::min<long long>(rounds, std::min(num_sms() * (threads > 256 ? 1 : 2), LN_MAX_PARTS)));
}
// Rows per group and round (131072 x 1024 bf16: two rows 132 us, one 142, four 144).
template <int VEC, int V>
constexpr int ln_rows() {
  return VEC * V > 8 ? 1 : 2;
}

template <class T, class W, int VEC, int TPR, int V>
static void ln_fwd(long long rows, int C, float eps, const void* x, const void* w, const void* b, void* y, float* mean,
                   float* rstd, cudaStream_t st) {
  constexpr int THREADS = ln_threads<TPR>(), GROUPS = THREADS / TPR;
  const long long rounds = (rows + GROUPS - 1) / GROUPS;
  const int grid = int(std::min<long long>(rounds, (long long)num_sms() * (2048 / THREADS)));
  layernorm_fwd_kernel<T, W, VEC, TPR, V><<<grid, THREADS, 0, st>>>(
      rows, C, eps, static_cast<const T*>(x), static_cast<const W*>(w), static_cast<const W*>(b), static_cast<T*>(y), mean,
      rstd);
}
template <class T, class W, int VEC, int TPR, int V>
static int ln_bwd(long long rows, int C, const void* dy, const void* x, const void* w, const float* mean,
                   const float* rstd, void* dx, float* part, int grid, cudaStream_t st) {
  constexpr int THREADS = ln_threads<TPR>();
  auto kernel = layernorm_bwd_kernel<T, W, VEC, TPR, V, ln_rows<VEC, V>()>;
  // (several groups: the block's sums are joined in [2][C] floats; they fit where a ring was)
  using Ring = LnRing<VEC, TPR, V, ln_rows<VEC, V>()>;
  static_assert(Ring::BYTES <= 227 * 1024, "");
  static_assert(!Ring::USED || THREADS == TPR || Ring::BYTES >= 8u * TPR * V * VEC, "");
  const size_t smem = Ring::USED ? Ring::BYTES : THREADS > TPR && part ? size_t(2) * C * sizeof(float) : 0;
  if (Ring::USED && !smem_attr_set(reinterpret_cast<const void*>(kernel), int(Ring::BYTES)))
    return set_error(MEA_ERR_CUDA, "cudaFuncSetAttribute(layer norm backward) failed");
  kernel<<<grid, THREADS, smem, st>>>(
      rows, C, static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const W*>(w), mean, rstd,
      static_cast<T*>(dx), part);
  return check_launch("layernorm_bwd_kernel");
}

// f(VEC, TPR, V) as compile-time constants for a shape of ln_fwd_shape.
template <int FULL, class F>
static void ln_fwd_dispatch(const LnShape& s, F&& f) {
  using std::integral_constant;
  auto tpr = [&](auto vec, auto v) {
    switch (s.tpr) {
      case 32: return f(vec, integral_constant<int, 32>(), v);
      case 64: return f(vec, integral_constant<int, 64>(), v);
      case 128: return f(vec, integral_constant<int, 128>(), v);
      case 256: return f(vec, integral_constant<int, 256>(), v);
      default: return f(vec, integral_constant<int, 512>(), v);
    }
  };
  if (s.vec == 1) return s.v == 8 ? tpr(integral_constant<int, 1>(), integral_constant<int, 8>())
                                  : tpr(integral_constant<int, 1>(), integral_constant<int, 32>());
  integral_constant<int, FULL> vec;
  switch (s.v) {
    case 1: return tpr(vec, integral_constant<int, 1>());
    case 2: return tpr(vec, integral_constant<int, 2>());
    case 4: return tpr(vec, integral_constant<int, 4>());
    default: return tpr(vec, integral_constant<int, 8>());
  }
}
// The same for ln_bwd_shape: V is above its least value at TPR = 512 only.
template <int FULL, class F>
static void ln_bwd_dispatch(const LnShape& s, F&& f) {
  using std::integral_constant;
  auto tpr = [&](auto vec, auto v) {
    switch (s.tpr) {
      case 32: return f(vec, integral_constant<int, 32>(), v);
      case 64: return f(vec, integral_constant<int, 64>(), v);
      case 128: return f(vec, integral_constant<int, 128>(), v);
      case 256: return f(vec, integral_constant<int, 256>(), v);
      default: return f(vec, integral_constant<int, 512>(), v);
    }
  };
  integral_constant<int, 512> all;
  if (s.vec == 1) {
    integral_constant<int, 1> one;
    if (s.v == 8) return tpr(one, integral_constant<int, 8>());
    return f(one, all, integral_constant<int, 16>());
  }
  integral_constant<int, FULL> vec;
  if (s.v == 1) return tpr(vec, integral_constant<int, 1>());
  if (s.v == 2) return f(vec, all, integral_constant<int, 2>());
  if (s.v == 4) return f(vec, all, integral_constant<int, 4>());
  if constexpr (FULL == 4) f(vec, all, integral_constant<int, 8>());
}

template <class T, class W>
static int layernorm_fwd(long long rows, int C, float eps, const void* x, const void* w, const void* b, void* y,
                         float* mean, float* rstd, const LnShape& s, cudaStream_t st) {
  if (s.v == 0) {
    const int grid = int(std::min<long long>(rows, (long long)num_sms() * 2));
    layernorm_fwd_long_kernel<T, W><<<grid, 1024, 0, st>>>(rows, C, eps, static_cast<const T*>(x),
                                                           static_cast<const W*>(w), static_cast<const W*>(b),
                                                           static_cast<T*>(y), mean, rstd);
  } else {
    ln_fwd_dispatch<16 / sizeof(T)>(s, [&](auto vec, auto tpr, auto v) {
      ln_fwd<T, W, vec(), tpr(), v()>(rows, C, eps, x, w, b, y, mean, rstd, st);
    });
  }
  return check_launch("layernorm_fwd_kernel");
}

static int ln_rows_of(const LnShape& s) { return s.vec * s.v > 8 ? 1 : 2; }

template <class T, class W>
static int layernorm_bwd(long long rows, int C, const void* dy, const void* x, const void* w, const float* mean,
                         const float* rstd, void* dx, void* dw, void* db, float* part, const LnShape& s,
                         cudaStream_t st) {
  int parts = 0;
  if (rows > 0) {
    int rc = MEA_OK;
    if (s.v == 0) {
      const int grid = int(std::min<long long>(rows, (long long)num_sms() * 2));
      layernorm_bwd_long_kernel<T, W><<<grid, 1024, 0, st>>>(rows, C, static_cast<const T*>(dy), static_cast<const T*>(x),
                                                             static_cast<const W*>(w), mean, rstd, static_cast<T*>(dx));
      if (part) {
        parts = int(std::min<long long>(rows, LN_LONG_PARTS));
        layernorm_part_long_kernel<T><<<dim3(unsigned((C + 255) / 256), unsigned(parts)), 256, 0, st>>>(
            rows, C, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, part);
      }
      rc = check_launch("layernorm_bwd_long_kernel");
    } else {
      parts = ln_bwd_blocks(rows, s, ln_rows_of(s));
      ln_bwd_dispatch<16 / sizeof(T)>(s, [&](auto vec, auto tpr, auto v) {
        rc = ln_bwd<T, W, vec(), tpr(), v()>(rows, C, dy, x, w, mean, rstd, dx, part, parts, st);
      });
    }
    if (rc != MEA_OK) return rc;
  }
  if (!part) return MEA_OK;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((C + 31) / 32), 2);
  cfg.blockDim = dim3(32, 32);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, layernorm_cols_kernel<W>, parts, C, static_cast<const float*>(part), static_cast<W*>(dw),
                     static_cast<W*>(db));
  return check_launch("layernorm_cols_kernel");
}

static int ln_check(long long rows, int C, int dtype, int wdtype) {
  if (rows < 0 || C <= 0)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm: rows=%lld must be >= 0 and C=%d positive", rows, C);
  if (dtype != MEA_BF16 && dtype != MEA_FP16 && dtype != MEA_FP32)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm: dtype %d is none of MEA_BF16, MEA_FP16, MEA_FP32", dtype);
  if (wdtype != dtype && wdtype != MEA_FP32)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm: the weight's dtype %d is neither x's (%d) nor MEA_FP32", wdtype,
                     dtype);
  return MEA_OK;
}
static int ln_align(std::initializer_list<const void*> ps, int elem) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % elem)
      return set_error(MEA_ERR_ALIGNMENT, "layer norm: a tensor is not aligned to its %d-byte elements", elem);
  return MEA_OK;
}
static bool ln_vector(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

}  // namespace mea

extern "C" size_t mea_layernorm_workspace_size(long long rows, int C) {
  if (rows < 0 || C <= 0) return 0;
  return size_t(2) * size_t(C) * sizeof(float) * mea::LN_MAX_PARTS;
}

extern "C" int mea_layernorm_forward(long long rows, int C, float eps, int dtype, int wdtype, const void* x, const void* w,
                                     const void* b, void* y, float* mean, float* rstd, void* stream) {
  using namespace mea;
  int rc = ln_check(rows, C, dtype, wdtype);
  if (rc != MEA_OK) return rc;
  if (!(eps >= 0.f) || !(eps < 3.0e38f)) return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm: eps=%g must be >= 0", eps);
  if (rows == 0) return MEA_OK;
  if (!x || !y || !mean || !rstd) return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm: x, y, mean and rstd must be non-NULL");
  const int elem = dtype == MEA_FP32 ? 4 : 2;
  if ((rc = ln_align({x, y}, elem)) != MEA_OK || (rc = ln_align({mean, rstd}, 4)) != MEA_OK ||
      (rc = ln_align({w, b}, wdtype == MEA_FP32 ? 4 : 2)) != MEA_OK)
    return rc;
  auto st = static_cast<cudaStream_t>(stream);
  const LnShape s = ln_fwd_shape(rows, C, elem, ln_vector({x, y, w, b}));
  if (dtype == MEA_FP32) return layernorm_fwd<float, float>(rows, C, eps, x, w, b, y, mean, rstd, s, st);
  if (dtype == MEA_BF16)
    return wdtype == MEA_FP32 ? layernorm_fwd<__nv_bfloat16, float>(rows, C, eps, x, w, b, y, mean, rstd, s, st)
                              : layernorm_fwd<__nv_bfloat16, __nv_bfloat16>(rows, C, eps, x, w, b, y, mean, rstd, s, st);
  return wdtype == MEA_FP32 ? layernorm_fwd<__half, float>(rows, C, eps, x, w, b, y, mean, rstd, s, st)
                            : layernorm_fwd<__half, __half>(rows, C, eps, x, w, b, y, mean, rstd, s, st);
}

extern "C" int mea_layernorm_backward(long long rows, int C, int dtype, int wdtype, const void* dy, const void* x,
                                      const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mea;
  int rc = ln_check(rows, C, dtype, wdtype);
  if (rc != MEA_OK) return rc;
  const bool sums = dw || db;
  if (rows == 0 && !sums) return MEA_OK;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx))
    return set_error(MEA_ERR_INVALID_ARGUMENT, "layer norm backward: dy, x, mean, rstd and dx must be non-NULL");
  const int elem = dtype == MEA_FP32 ? 4 : 2;
  if ((rc = ln_align({dy, x, dx}, elem)) != MEA_OK || (rc = ln_align({mean, rstd}, 4)) != MEA_OK ||
      (rc = ln_align({w, dw, db}, wdtype == MEA_FP32 ? 4 : 2)) != MEA_OK)
    return rc;
  if (sums && (!workspace || reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(MEA_ERR_ALIGNMENT, "layer norm backward: the workspace must be non-NULL and 16-byte aligned");
  if (sums && workspace_bytes < mea_layernorm_workspace_size(rows, C))
    return set_error(MEA_ERR_WORKSPACE, "layer norm backward: the workspace has %zu bytes, needs %zu", workspace_bytes,
                     mea_layernorm_workspace_size(rows, C));
  auto st = static_cast<cudaStream_t>(stream);
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  const LnShape s = ln_bwd_shape(C, elem, ln_vector({dy, x, dx, w}));
  if (dtype == MEA_FP32) return layernorm_bwd<float, float>(rows, C, dy, x, w, mean, rstd, dx, dw, db, part, s, st);
  if (dtype == MEA_BF16)
    return wdtype == MEA_FP32
               ? layernorm_bwd<__nv_bfloat16, float>(rows, C, dy, x, w, mean, rstd, dx, dw, db, part, s, st)
               : layernorm_bwd<__nv_bfloat16, __nv_bfloat16>(rows, C, dy, x, w, mean, rstd, dx, dw, db, part, s, st);
  return wdtype == MEA_FP32 ? layernorm_bwd<__half, float>(rows, C, dy, x, w, mean, rstd, dx, dw, db, part, s, st)
                            : layernorm_bwd<__half, __half>(rows, C, dy, x, w, mean, rstd, dx, dw, db, part, s, st);
}
