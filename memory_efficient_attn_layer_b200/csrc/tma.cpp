#include "tma.h"

#include <cudaTypedefs.h>
#include <mutex>

namespace mea {

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// cuTensorMapEncodeTiled needs a current context, which a thread that has made no
// runtime call yet (a new one, or autograd's) does not have: the device's primary
// context is then made current, as any runtime call would.
template <class Encode>
static CUresult with_context(Encode&& encode) {
  CUresult r = encode();
  int dev = 0;
  if ((r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) && cudaGetDevice(&dev) == cudaSuccess &&
      cudaSetDevice(dev) == cudaSuccess)
    r = encode();
  return r;
}

int make_tmap_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t row_bytes,
                 uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swizzle, CUtensorMapDataType dtype) {
  auto fn = encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = with_context([&] {
    return fn(map, dtype, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  return r == CUDA_SUCCESS ? 0 : int(r);
}

int make_tmap_3d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t n1, uint64_t s1, uint64_t n2, uint64_t s2,
                 uint32_t box0, uint32_t box1, uint32_t box2, CUtensorMapSwizzle swizzle, CUtensorMapDataType dtype) {
  auto fn = encode_fn();
  if (!fn) return -1;
  cuuint64_t dims[3] = {inner, n1, n2};
  cuuint64_t strides[2] = {s1, s2};
  cuuint32_t box[3] = {box0, box1, box2};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = with_context([&] {
    return fn(map, dtype, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  return r == CUDA_SUCCESS ? 0 : int(r);
}

}  // namespace mea
