// The work plan of the packed-sequence attention, and its host side: shapes,
// strides, tensor maps and buffer sizes shared by the forward and backward.
//
// The lengths are device data, so the host only knows how many tiles there can
// be: total / tt + n_seqs.  A small kernel turns cu_seqlens into the list of
// tiles, in one of two orders; blocks past the list's end leave at once.
//  * By falling work, all heads of a tile together: the longest tiles start first
//    and the GPU's SMs end together.  All sequences and heads are in flight.
//  * By sequence (longest first), then head, then falling work: the tiles that run
//    at one time share a few heads' rows in L2.  Taken when the rows that the tiles
//    walk over are more than half of L2 and there are eight or more tiles to an
//    SM, so that the end still comes out even.
// Measured (N = 128): 16 x 2048 tokens with 16 heads (268 MB of K and V), forward
// 422 us by work, 354 by sequence, dQ 584 and 499; 12289 + 4095 tokens with 16
// query and 4 key/value heads, dK/dV 1169 us by work, 1514 by sequence (a tile of
// the first key rows alone walks 385 steps of 576 that an SM has).
// The plan belongs to the call, never to a later one: a captured call builds it
// again from the values cu_seqlens has at the replay.
#include <algorithm>

#include "attn_packed.h"
#include "attn_packed.cuh"

namespace mea {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_CLASSES = 1024;
constexpr int PLAN_SMEM_SEQS = 1024;  // up to this many sequences are sorted in shared memory

// Exclusive block-wide prefix sum of one value per thread; *sum is the total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // warp_sums of an earlier call are read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *sum = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// Last index s with pre[s] <= id (pre is non-decreasing, pre[0] = 0): the
// sequence that tile `id` lies in; sequences without tiles are passed over.
__device__ __forceinline__ int seq_of(const int* pre, int n_seqs, int id) {
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= id)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Block i makes list i.  `at_once`: up to this many entries of the list start
// together whatever their order, so they are not sorted; `wide`: the rows that its
// tiles walk over are more than half of L2.
struct PlanParams {
  PackedDims d;
  PackedPlan plan;
  int at_once[3], wide[3];
  int* scratch;
  int* status;
};

__global__ void __launch_bounds__(PLAN_THREADS) packed_plan_kernel(const int* __restrict__ cu, const PlanParams p) {
  __shared__ int seq_s[3 * PLAN_SMEM_SEQS];
  __shared__ int hist[PLAN_CLASSES];
  __shared__ int warp_sums[32];
  __shared__ int longest_s;
  const int tid = threadIdx.x, kind = blockIdx.x, n_seqs = p.d.n_seqs, tt = p.d.tt;
  pdl_launch();
  if (tid == 0) longest_s = 0;
  const int rows = p.d.rows[kind];  // tokens of a tile
  const bool keys = kind == LIST_K;
  // The sequences in the order they are taken: first row, length, tiles before it.
  const bool in_smem = n_seqs <= PLAN_SMEM_SEQS;
  int* begin = in_smem ? seq_s : p.scratch + size_t(3) * kind * n_seqs;
  int* len = begin + (in_smem ? PLAN_SMEM_SEQS : n_seqs);
  int* pre = len + (in_smem ? PLAN_SMEM_SEQS : n_seqs);
  int longest = 0, most_tiles = 0;
  bool good = true;
  for (int s = tid; s < n_seqs; s += PLAN_THREADS) {
    const int a = cu[s], b = cu[s + 1];
    good &= a >= 0 && a <= b && b <= p.d.total;
    if (good) {
      longest = max(longest, b - a);
      most_tiles += (b - a + rows - 1) / rows;
    }
  }
  hist[tid] = 0;
  longest = __reduce_max_sync(0xffffffffu, longest);
  if ((tid & 31) == 0) atomicMax(&longest_s, longest);
  // cu_seqlens must rise from >= 0 to <= total; otherwise no tile is made (every
  // output row is then zero) and the status word says so.
  if (!__syncthreads_and(good)) {
    if (tid == 0) {
      p.plan.head->n[kind] = 0;
      if (keys) p.plan.head->splits = 1;
      if (kind == 0) {
        record_error(p.status, KID_PACKED_PLAN, 1);
        p.plan.head->first = p.plan.head->end = 0;
      }
    }
    return;
  }
  longest = longest_s;
  int n;
  block_scan(most_tiles, warp_sums, &n);
  const int cap = p.d.cap[kind];
  if (tid == 0) {
    p.plan.head->n[kind] = min(n, cap);
    if (kind == LIST_FWD) p.plan.head->next = 0;
    if (kind == 0) {
      p.plan.head->first = cu[0];
      p.plan.head->end = cu[n_seqs];
    }
  }
  const int most = keys ? (longest + tt - 1) / tt : (longest + 127) >> 7;  // steps of the longest tile
  // A part of a key tile's walk should still be some eight steps.
  if (keys && tid == 0)
    p.plan.head->splits = max(1, min(p.d.most_splits, most * (p.d.Hq / p.d.Hkv / p.d.p) / 8));
  const bool by_seq = p.wide[kind] && n >= 8 * max(p.at_once[kind], 1);
  if (!by_seq) {
    for (int s = tid; s < n_seqs; s += PLAN_THREADS) {
      begin[s] = cu[s];
      len[s] = cu[s + 1] - cu[s];
    }
  } else {  // counting sort by falling length, 1024 classes; the order within a class is free
    int shift = 0;
    while ((longest >> shift) >= PLAN_CLASSES) ++shift;
    for (int s = tid; s < n_seqs; s += PLAN_THREADS) atomicAdd(&hist[(longest >> shift) - ((cu[s + 1] - cu[s]) >> shift)], 1);
    __syncthreads();
    int all;
    const int at = block_scan(hist[tid], warp_sums, &all);
    hist[tid] = at;
    __syncthreads();
    for (int s = tid; s < n_seqs; s += PLAN_THREADS) {
      const int l = cu[s + 1] - cu[s];
      const int slot = atomicAdd(&hist[(longest >> shift) - (l >> shift)], 1);
      begin[slot] = cu[s];
      len[slot] = l;
    }
  }
  __syncthreads();
  int sum = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += PLAN_THREADS) {
    const int s = s0 + tid;
    int part;
    const int at = block_scan(s < n_seqs ? (len[s] + rows - 1) / rows : 0, warp_sums, &part);
    if (s < n_seqs) pre[s] = sum + at;
    sum += part;
  }
  __syncthreads();
  int4* items = p.plan.list[kind];
  auto entry = [&](int id) {
    const int s = seq_of(pre, n_seqs, id);
    return make_int4(begin[s], len[s], by_seq ? pre[s] : id - pre[s], by_seq ? 0 : 1);
  };
  if (by_seq || n <= p.at_once[kind]) {
    for (int id = tid; id < min(n, cap); id += PLAN_THREADS) items[id] = entry(id);
    return;
  }
  // Counting sort by falling work, 1024 classes.
  int shift = 0;
  while ((most >> shift) >= PLAN_CLASSES) ++shift;
  auto cls = [&](const int4& e) {
    // steps: key tiles up to the query tile's last token, or query tiles from the key tile's first
    const int steps = keys ? (e.y + tt - 1) / tt - e.z * 128 / tt
                           : (int(min((long long)(e.z + 1) * rows, (long long)e.y)) + 127) >> 7;
    return (most >> shift) - (steps >> shift);
  };
  hist[tid] = 0;
  __syncthreads();
  for (int id = tid; id < n; id += PLAN_THREADS) atomicAdd(&hist[cls(entry(id))], 1);
  __syncthreads();
  int all;
  const int at = block_scan(hist[tid], warp_sums, &all);
  hist[tid] = at;
  __syncthreads();
  for (int id = tid; id < n; id += PLAN_THREADS) {
    const int4 e = entry(id);
    const int slot = atomicAdd(&hist[cls(e)], 1);  // order within a class is free: tiles are independent
    if (slot < cap) items[slot] = e;
  }
}
static_assert(PLAN_CLASSES == PLAN_THREADS, "one class per thread in the scan");

// ---------------------------------------------------------------- host side
static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

int packed_dims(const mea_packed_dims* d, PackedDims* out) {
  if (!d) return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: dims is NULL");
  if (d->total < 0 || d->n_seqs < 0)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: total=%d and n_seqs=%d must be >= 0", d->total,
                     d->n_seqs);
  if (d->total > (1 << 30))
    return set_error(MEA_ERR_UNSUPPORTED_SHAPE, "packed attention: total=%d is more than 2^30 rows", d->total);
  if (d->Hq <= 0 || d->Hkv <= 0 || d->Hq % d->Hkv)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: Hq=%d must be a positive multiple of Hkv=%d", d->Hq,
                     d->Hkv);
  if (d->N <= 0 || d->N > 128 || d->N % 8)
    return set_error(MEA_ERR_UNSUPPORTED_SHAPE, "packed attention: head dim N=%d must be a multiple of 8 up to 128", d->N);
  if (d->dtype != MEA_BF16 && d->dtype != MEA_FP16)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: dtype %d is neither MEA_BF16 nor MEA_FP16", d->dtype);
  if (!(d->scale > 0.f) || !(d->scale < 3.0e38f))
    return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: scale=%g must be positive and finite", d->scale);
  PackedDims o;
  o.total = d->total;
  o.n_seqs = d->n_seqs;
  o.Hq = d->Hq;
  o.Hkv = d->Hkv;
  o.N = d->N;
  // Heads per query tile: the divisor of the group size that fills most of the
  // 128 rows, the larger one at a tie (fewer K/V reads).
  const int G = d->Hq / d->Hkv;
  o.p = 1;
  o.tt = 128;
  for (int p = 2; p <= G && p <= 128; ++p)
    if (G % p == 0 && p * (128 / p) >= o.p * o.tt) {
      o.p = p;
      o.tt = 128 / p;
    }
  o.p_inv = (65536 + o.p - 1) / o.p;
  o.hg = d->Hq / o.p;
  // Two query tiles to a forward item where that still gives every SM one.
  o.streams = (long long)d->total / (2 * o.tt) * o.hg >= num_sms() ? 2 : 1;
  const int rows[3] = {o.tt, 128, o.tt * o.streams}, heads[3] = {o.hg, d->Hkv, o.hg};
  for (int i = 0; i < 3; ++i) {
    const long long cap = (long long)d->total / rows[i] + d->n_seqs;
    if (cap * heads[i] > 0x3fffffffLL)  // (the counters run on by one per SM)
      return set_error(MEA_ERR_UNSUPPORTED_SHAPE,
                       "packed attention: total=%d rows, %d sequences and %d heads make too many tiles", d->total,
                       d->n_seqs, d->Hq);
    o.rows[i] = rows[i];
    o.heads[i] = heads[i];
    o.cap[i] = int(cap);
  }
  // Few key tiles (few key/value heads, not many rows): each tile's walk over the
  // queries may be cut into parts, as many as make four for every SM.
  const long long k_tiles = std::max<long long>(1, (long long)d->total / 128 * d->Hkv);
  o.most_splits = int(std::min<long long>(16, std::max<long long>(1, 4LL * num_sms() / k_tiles)));
  *out = o;
  return MEA_OK;
}

size_t packed_delta_bytes(const PackedDims& d) { return up256(sizeof(float) * size_t(d.total) * d.Hq); }
size_t packed_backward_bytes(const PackedDims& d) {
  const size_t parts = d.most_splits > 1 ? size_t(d.most_splits) * 2 * sizeof(float) * d.total * d.Hkv * d.N : 0;
  return PACKED_COUNTERS + packed_delta_bytes(d) + up256(parts);
}

static size_t plan_scratch(const PackedDims& d) {  // offset of the plan kernel's own space
  size_t n = up256(sizeof(PackedHeader));
  for (int i = 0; i < 3; ++i) n += up256(sizeof(int4) * size_t(d.cap[i]));
  return n;
}

size_t packed_plan_bytes(const PackedDims& d) {
  return plan_scratch(d) + (d.n_seqs > PLAN_SMEM_SEQS ? up256(sizeof(int) * 9 * size_t(d.n_seqs)) : 0);
}

PackedPlan packed_plan_view(const PackedDims& d, void* plan) {
  char* b = static_cast<char*>(plan);
  PackedPlan v;
  v.head = reinterpret_cast<PackedHeader*>(b);
  b += up256(sizeof(PackedHeader));
  for (int i = 0; i < 3; ++i) {
    v.list[i] = reinterpret_cast<int4*>(b);
    b += up256(sizeof(int4) * size_t(d.cap[i]));
  }
  return v;
}

bool packed_wide(const PackedDims& d, int list) {  // Q and dO, or K and V
  return 4LL * d.total * (list == LIST_K ? d.Hq : d.Hkv) * d.N > (64LL << 20);
}

int run_packed_plan(const PackedDims& d, const int* cu, void* plan, int* status, cudaStream_t st) {
  PlanParams p;
  p.d = d;
  p.plan = packed_plan_view(d, plan);
  for (int i = 0; i < 3; ++i) {
    p.at_once[i] = num_sms() / d.heads[i];
    p.wide[i] = packed_wide(d, i);
  }
  p.scratch = reinterpret_cast<int*>(static_cast<char*>(plan) + plan_scratch(d));
  p.status = status;
  packed_plan_kernel<<<3, PLAN_THREADS, 0, st>>>(cu, p);
  return check_launch("packed_plan_kernel");
}

int packed_check_rows(const char* name, const void* base, long long tok, long long head, const PackedDims& d, int heads) {
  if (!base) return set_error(MEA_ERR_INVALID_ARGUMENT, "packed attention: %s is NULL", name);
  if (reinterpret_cast<uintptr_t>(base) & 15)
    return set_error(MEA_ERR_ALIGNMENT, "packed attention: %s must be 16-byte aligned", name);
  if ((d.total > 1 && (tok < d.N || tok % 8)) || (heads > 1 && (head < d.N || head % 8)))
    return set_error(MEA_ERR_ALIGNMENT,
                     "packed attention: the row and head strides of %s (%lld, %lld) must be multiples of 8 elements, "
                     "at least N=%d", name, tok, head, d.N);
  if ((d.total > 1 && tok >= (1LL << 38)) || (heads > 1 && head >= (1LL << 38)))
    return set_error(MEA_ERR_UNSUPPORTED_SHAPE, "packed attention: a stride of %s is too large", name);
  return MEA_OK;
}

int packed_map(CUtensorMap* map, const PackedDims& d, int dtype, const void* base, long long tok, long long head,
               int heads, int box_heads, int box_rows) {
  // The stride of a dimension of extent one is never used; it still has to be a legal one.
  if (heads == 1) head = d.N;
  if (d.total == 1) tok = (long long)heads * (head > d.N ? head : d.N);
  return make_tmap_3d(map, base, uint64_t(d.N), uint64_t(heads), uint64_t(head) * 2, uint64_t(d.total),
                      uint64_t(tok) * 2, 64, uint32_t(box_heads), uint32_t(box_rows), CU_TENSOR_MAP_SWIZZLE_128B,
                      dtype == MEA_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

cudaLaunchConfig_t packed_launch(int grid, int threads, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

}  // namespace mea

extern "C" size_t mea_packed_backward_workspace_size(const mea_packed_dims* d) {
  mea::PackedDims pd;
  if (mea::packed_dims(d, &pd) != MEA_OK) return 0;
  return mea::packed_backward_bytes(pd);
}
extern "C" size_t mea_packed_plan_size(const mea_packed_dims* d) {
  mea::PackedDims pd;
  if (mea::packed_dims(d, &pd) != MEA_OK) return 0;
  return mea::packed_plan_bytes(pd);
}
