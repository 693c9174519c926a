// The global norm of a list of gradients, and their clipping by it.
//
//   total = sqrt(sum over all tensors of sum g^2)   (or max |g|)
//   g *= min(1, max_norm / (total + 1e-6))
//
// Bound by HBM: each gradient is read once for the norm, and read and written
// once more only if the norm is above max_norm.  The list travels in the kernel's
// parameters (pointers, lengths, first chunks), so a call needs no copy to the
// device and can be captured; a launch takes up to GN_TENSORS tensors.  Tensors
// are cut into chunks of GN_CHUNK elements, dealt to the blocks in turn; every
// block writes one fp64 partial, and whoever needs the norm adds the partials in
// their order, so the result does not depend on the order of the blocks.  The
// scaling kernel walks the chunks backwards: what the norm read last may still be
// in L2.  268 MB of bf16 take 44 us for the norm (6.1 TB/s) and 87 us for the
// scaling (6.2 TB/s); 12 layers of width 2048 with MLPs (1.3 GB) 659 us for both.
//
// Squares are summed in fp32 over one thread's 16 bytes and in fp64 from there
// on; where such a group's sum leaves fp32's comfortable range it is formed again
// in fp64, so gradients of 1e25 or 1e-25 have their norm too.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <memory>
#include <new>

#include "launch.h"
#include "ptx.cuh"

namespace mea {

constexpr int GN_TENSORS = 512;
constexpr int GN_CHUNK = 32768;
constexpr int GN_THREADS = 512;

struct GradList {
  void* ptr[GN_TENSORS];
  long long n[GN_TENSORS];
  int chunk0[GN_TENSORS + 1];  // first chunk of each tensor
  uint8_t dtype[GN_TENSORS];
  int count;
};

__device__ __forceinline__ void unpack16(const uint4& r, int dtype, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == MEA_BF16) {
      f[2 * i] = bf16_lo(w[i]);
      f[2 * i + 1] = bf16_hi(w[i]);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

// The tensor that chunk `id` lies in.
__device__ __forceinline__ int tensor_of(const GradList& L, int id) {
  int lo = 0, hi = L.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.chunk0[mid] <= id)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float element(const void* p, int dtype, long long i) {
  if (dtype == MEA_FP32) return static_cast<const float*>(p)[i];
  if (dtype == MEA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Squares (or the largest magnitude, NaN if any is) of `N` values.
template <bool INF, int N>
__device__ __forceinline__ void take(double& acc, const float (&f)[N]) {
  if (INF) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max3f_nan(m, fabsf(f[i]), 0.f);
    acc = (m != m || acc != acc) ? __longlong_as_double(0x7ff8000000000000LL) : fmax(acc, double(m));
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(f[i], f[i], s);
    // Above 2^100 a square may have overflowed, below 2^-80 one may have lost bits.
    if (s < 1.2676506e30f && s > 8.2718061e-25f) {
      acc += double(s);
    } else {
      double d = 0.0;
#pragma unroll
      for (int i = 0; i < N; ++i) d = fma(double(f[i]), double(f[i]), d);
      acc += d;
    }
  }
}

template <bool INF>
__device__ __forceinline__ double merge(double a, double b) {
  if (!INF) return a + b;
  return (a != a || b != b) ? __longlong_as_double(0x7ff8000000000000LL) : fmax(a, b);
}

template <bool INF>
__device__ __forceinline__ double block_merge(double v, double* red) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v = merge<INF>(v, __shfl_xor_sync(0xffffffffu, v, m));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < int(blockDim.x >> 5); ++w) v = merge<INF>(v, red[w]);
  return v;
}

// The chunk's part of its tensor: elements [at, at + len); `head` of them before
// the first 16-byte boundary, then `vecs` vectors, then the rest.
struct Chunk {
  void* p;
  int dtype, len, head, vecs, per;
  __device__ Chunk(const GradList& L, int id) {
    const int t = tensor_of(L, id);
    const long long at = (long long)(id - L.chunk0[t]) * GN_CHUNK;
    dtype = L.dtype[t];
    const int elem = dtype == MEA_FP32 ? 4 : 2;
    p = static_cast<char*>(L.ptr[t]) + at * elem;
    len = int(min((long long)GN_CHUNK, L.n[t] - at));
    per = 16 / elem;
    head = min(len, int(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / elem));
    vecs = (len - head) / per;
  }
  __device__ uint4* vec() const { return reinterpret_cast<uint4*>(static_cast<char*>(p) + head * (16 / per)); }
};

template <bool INF>
__global__ void __launch_bounds__(GN_THREADS) grad_norm_kernel(const __grid_constant__ GradList L, double* part) {
  __shared__ double red[GN_THREADS / 32];
  pdl_launch();
  double acc = 0.0;
  for (int id = blockIdx.x; id < L.chunk0[L.count]; id += gridDim.x) {
    const Chunk c(L, id);
    const uint4* v = c.vec();
    constexpr int U = 4;
    for (int i0 = 0; i0 < c.vecs; i0 += U * GN_THREADS) {
      uint4 r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * GN_THREADS + threadIdx.x;
        r[u] = i < c.vecs ? v[i] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u * GN_THREADS + int(threadIdx.x) >= c.vecs) continue;
        if (c.dtype == MEA_FP32) {
          const float f[4] = {__uint_as_float(r[u].x), __uint_as_float(r[u].y), __uint_as_float(r[u].z), __uint_as_float(r[u].w)};
          take<INF>(acc, f);
        } else {
          float f[8];
          unpack16(r[u], c.dtype, f);
          take<INF>(acc, f);
        }
      }
    }
    const int rest = c.len - c.vecs * c.per;  // the elements before and behind the vectors
    if (int(threadIdx.x) < rest) {
      const int i = int(threadIdx.x) < c.head ? int(threadIdx.x) : c.vecs * c.per + int(threadIdx.x);
      const float f[1] = {element(c.p, c.dtype, i)};
      take<INF>(acc, f);
    }
  }
  acc = block_merge<INF>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The norm from n partials, the same in every block (each thread takes every
// blockDim.x-th, then the block merges in a fixed order).
template <bool INF>
__device__ __forceinline__ double norm_of(const double* part, int n, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v = merge<INF>(v, __ldcg(part + i));
  v = block_merge<INF>(v, red);
  return INF ? v : sqrt(v);
}

// total norm -> *norm (fp32), sum of squares (or the maximum) -> *sumsq; either may be NULL.
template <bool INF>
__global__ void __launch_bounds__(GN_THREADS) grad_norm_total_kernel(const double* part, int n, float* norm, double* sumsq) {
  __shared__ double red[GN_THREADS / 32];
  pdl_wait();
  const double v = norm_of<INF>(part, n, red);
  if (threadIdx.x == 0) {
    if (norm) *norm = float(v);
    if (sumsq) {
      double s = 0.0;
      if (INF) {
        s = v;
      } else {
        for (int w = 0; w < GN_THREADS / 32; ++w) s += red[w];
      }
      *sumsq = s;
    }
  }
}

template <bool INF>
__global__ void __launch_bounds__(GN_THREADS) grad_scale_kernel(const __grid_constant__ GradList L, const double* part,
                                                                int n_part, double max_norm, float* norm_out) {
  __shared__ double red[GN_THREADS / 32];
  pdl_wait();
  pdl_launch();
  const double norm = norm_of<INF>(part, n_part, red);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = float(norm);
  const float f = clip_factor(norm, max_norm);
  if (f == 1.0f) return;  // times one: every bit would stay
  const int chunks = L.chunk0[L.count];
  for (int k = blockIdx.x; k < chunks; k += gridDim.x) {
    const Chunk c(L, chunks - 1 - k);
    uint4* v = c.vec();
    constexpr int U = 4;
    for (int i0 = 0; i0 < c.vecs; i0 += U * GN_THREADS) {
      uint4 r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * GN_THREADS + threadIdx.x;
        if (i < c.vecs) r[u] = v[i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * GN_THREADS + threadIdx.x;
        if (i >= c.vecs) continue;
        uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
        if (c.dtype == MEA_FP32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
        } else {
          float x[8];
          unpack16(r[u], c.dtype, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (c.dtype == MEA_BF16) {
              w[e] = pack_bf16(x[2 * e] * f, x[2 * e + 1] * f);
            } else {
              const __half2 h = __floats2half2_rn(x[2 * e] * f, x[2 * e + 1] * f);
              w[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
        }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    const int rest = c.len - c.vecs * c.per;
    if (int(threadIdx.x) < rest) {
      const int i = int(threadIdx.x) < c.head ? int(threadIdx.x) : c.vecs * c.per + int(threadIdx.x);
      const float x = element(c.p, c.dtype, i) * f;
      if (c.dtype == MEA_FP32)
        static_cast<float*>(c.p)[i] = x;
      else if (c.dtype == MEA_BF16)
        static_cast<__nv_bfloat16*>(c.p)[i] = __float2bfloat16_rn(x);
      else
        static_cast<__half*>(c.p)[i] = __float2half_rn(x);
    }
  }
}

// ---------------------------------------------------------------- host side
constexpr int GN_BLOCKS_PER_SM = 4;

static int gn_check(int count, const void* const* grads, const long long* n, const int* dtypes, int kind) {
  if (count < 0 || (count > 0 && (!grads || !n || !dtypes)))
    return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient norm: count=%d must be >= 0 and its arrays non-NULL", count);
  if (kind != MEA_NORM_2 && kind != MEA_NORM_INF)
    return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient norm: kind %d is neither MEA_NORM_2 nor MEA_NORM_INF", kind);
  long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (dtypes[i] != MEA_BF16 && dtypes[i] != MEA_FP16 && dtypes[i] != MEA_FP32)
      return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient norm: tensor %d has dtype %d", i, dtypes[i]);
    if (n[i] < 0 || n[i] > (1LL << 44) || (n[i] > 0 && !grads[i]))
      return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient norm: tensor %d has %lld elements at a %s pointer", i, n[i],
                       grads[i] ? "non-NULL" : "NULL");
    if (reinterpret_cast<uintptr_t>(grads[i]) % (dtypes[i] == MEA_FP32 ? 4 : 2))
      return set_error(MEA_ERR_ALIGNMENT, "gradient norm: tensor %d is not aligned to its elements", i);
    chunks += (n[i] + GN_CHUNK - 1) / GN_CHUNK;
    if (chunks > 0x3fffffffLL)
      return set_error(MEA_ERR_UNSUPPORTED_SHAPE, "gradient norm: the tensors hold more than 2^30 chunks of %d elements", GN_CHUNK);
  }
  return MEA_OK;
}

// The next launch's list from tensor `i` on (tensors without elements are left out); false when none is left.
static bool gn_fill(GradList& L, int& i, int count, const void* const* grads, const long long* n, const int* dtypes) {
  L.count = 0;
  long long chunks = 0;
  for (; i < count && L.count < GN_TENSORS; ++i) {
    if (!n[i]) continue;
    const long long c = (n[i] + GN_CHUNK - 1) / GN_CHUNK;
    L.ptr[L.count] = const_cast<void*>(grads[i]);
    L.n[L.count] = n[i];
    L.dtype[L.count] = uint8_t(dtypes[i]);
    L.chunk0[L.count++] = int(chunks);
    chunks += c;
  }
  L.chunk0[L.count] = int(chunks);
  return L.count > 0;
}

static int gn_grid(const GradList& L) {
  return std::min(L.chunk0[L.count], num_sms() * GN_BLOCKS_PER_SM);
}

// Partials of every tensor; *n_part is how many there are.
template <bool INF>
static int gn_partials(int count, const void* const* grads, const long long* n, const int* dtypes, double* part,
                       long long cap, int* n_part, cudaStream_t st) {
  GradList L;
  int i = 0, at = 0;
  while (gn_fill(L, i, count, grads, n, dtypes)) {
    const int grid = gn_grid(L);
    if (at + grid > cap) return set_error(MEA_ERR_WORKSPACE, "gradient norm: workspace too small");
    grad_norm_kernel<INF><<<grid, GN_THREADS, 0, st>>>(L, part + at);
    const int rc = check_launch("grad_norm_kernel");
    if (rc != MEA_OK) return rc;
    at += grid;
  }
  *n_part = at;
  return MEA_OK;
}

static cudaLaunchConfig_t gn_launch(int grid, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(GN_THREADS);
  cfg.stream = st;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <bool INF>
static int gn_run(int count, const void* const* grads, const long long* n, const int* dtypes, bool scale, double max_norm,
                  float* norm, double* sumsq, double* part, long long cap, cudaStream_t st) {
  int n_part = 0;
  int rc = gn_partials<INF>(count, grads, n, dtypes, part, cap, &n_part, st);
  if (rc != MEA_OK) return rc;
  cudaLaunchAttribute attr;
  if (!scale || n_part == 0) {
    const cudaLaunchConfig_t cfg = gn_launch(1, st, &attr);
    cudaLaunchKernelEx(&cfg, grad_norm_total_kernel<INF>, static_cast<const double*>(part), n_part, norm, sumsq);
    return check_launch("grad_norm_total_kernel");
  }
  GradList L;
  int i = 0;
  float* out = norm;
  while (gn_fill(L, i, count, grads, n, dtypes)) {
    const cudaLaunchConfig_t cfg = gn_launch(gn_grid(L), st, &attr);
    cudaLaunchKernelEx(&cfg, grad_scale_kernel<INF>, L, static_cast<const double*>(part), n_part, max_norm, out);
    if ((rc = check_launch("grad_scale_kernel")) != MEA_OK) return rc;
    out = nullptr;
  }
  return MEA_OK;
}

static long long gn_cap(int count) {
  const long long launches = count <= 0 ? 1 : (count + GN_TENSORS - 1) / GN_TENSORS;
  return launches * 160 * GN_BLOCKS_PER_SM;
}

}  // namespace mea

extern "C" size_t mea_grad_norm_workspace_size(int count) { return size_t(mea::gn_cap(count)) * sizeof(double); }

static int gn_buffers(int count, const void* workspace, size_t workspace_bytes) {
  using namespace mea;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) & 7)
    return set_error(MEA_ERR_ALIGNMENT, "gradient norm: the workspace must be non-NULL and 8-byte aligned");
  if (workspace_bytes < mea_grad_norm_workspace_size(count))
    return set_error(MEA_ERR_WORKSPACE, "gradient norm: the workspace has %zu bytes, needs %zu", workspace_bytes,
                     mea_grad_norm_workspace_size(count));
  return MEA_OK;
}

extern "C" int mea_grad_norm(int count, const void* const* grads, const long long* n, const int* dtypes, int kind,
                             float* norm, double* sumsq, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mea;
  int rc = gn_check(count, grads, n, dtypes, kind);
  if (rc != MEA_OK) return rc;
  if (!norm && !sumsq) return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient norm: norm and sumsq are both NULL");
  if (reinterpret_cast<uintptr_t>(norm) & 3 || reinterpret_cast<uintptr_t>(sumsq) & 7)
    return set_error(MEA_ERR_ALIGNMENT, "gradient norm: norm must be 4-byte, sumsq 8-byte aligned");
  if ((rc = gn_buffers(count, workspace, workspace_bytes)) != MEA_OK) return rc;
  auto fn = kind == MEA_NORM_INF ? gn_run<true> : gn_run<false>;
  return fn(count, grads, n, dtypes, false, 0.0, norm, sumsq, static_cast<double*>(workspace), gn_cap(count),
            static_cast<cudaStream_t>(stream));
}

// Elements of two tensors at one address would be scaled once or twice as the blocks fall.
static int gn_apart(int count, void* const* grads, const long long* n, const int* dtypes) {
  using namespace mea;
  struct Span {
    uintptr_t begin, end;
  };
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[size_t(count) + 1]);
  if (!spans) return set_error(MEA_ERR_WORKSPACE, "gradient clipping: no host memory for %d tensors", count);
  int k = 0;
  for (int i = 0; i < count; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(grads[i]);
    if (n[i]) spans[k++] = {at, at + uintptr_t(n[i]) * (dtypes[i] == MEA_FP32 ? 4 : 2)};
  }
  std::sort(&spans[0], &spans[k], [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (int i = 1; i < k; ++i)
    if (spans[i].begin < spans[i - 1].end)
      return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient clipping: two of the tensors overlap in memory");
  return MEA_OK;
}

extern "C" int mea_clip_grad_norm(int count, void* const* grads, const long long* n, const int* dtypes, int kind,
                                  double max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mea;
  int rc = gn_check(count, grads, n, dtypes, kind);
  if (rc != MEA_OK) return rc;
  if (!(max_norm >= 0.0)) return set_error(MEA_ERR_INVALID_ARGUMENT, "gradient clipping: max_norm=%g must be >= 0", max_norm);
  if (!norm || reinterpret_cast<uintptr_t>(norm) & 3)
    return set_error(MEA_ERR_ALIGNMENT, "gradient clipping: norm must be non-NULL and 4-byte aligned");
  if ((rc = gn_buffers(count, workspace, workspace_bytes)) != MEA_OK) return rc;
  if ((rc = gn_apart(count, grads, n, dtypes)) != MEA_OK) return rc;
  auto fn = kind == MEA_NORM_INF ? gn_run<true> : gn_run<false>;
  return fn(count, grads, n, dtypes, true, max_norm, norm, nullptr, static_cast<double*>(workspace), gn_cap(count),
            static_cast<cudaStream_t>(stream));
}
