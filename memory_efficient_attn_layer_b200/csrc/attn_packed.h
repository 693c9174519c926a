// Host-side interface between the packed-sequence attention's sources.
#pragma once
#include "launch.h"
#include "tma.h"

namespace mea {

struct PackedDims;
struct PackedPlan;

// Checks the sizes of *d and derives the tile shape and the plan's capacity.
int packed_dims(const mea_packed_dims* d, PackedDims* out);
size_t packed_plan_bytes(const PackedDims& d);
// The backward's workspace: its tile counters, delta [total, Hq], then the parts' dK and dV in fp32.
constexpr size_t PACKED_COUNTERS = 256;
size_t packed_delta_bytes(const PackedDims& d);
size_t packed_backward_bytes(const PackedDims& d);
PackedPlan packed_plan_view(const PackedDims& d, void* plan);
// The rows that a list's tiles walk over are more than half of L2.
bool packed_wide(const PackedDims& d, int list);
int run_packed_plan(const PackedDims& d, const int* cu, void* plan, int* status, cudaStream_t st);
// Pointer, alignment and stride checks of one [total, heads, N] tensor.
int packed_check_rows(const char* name, const void* base, long long tok, long long head, const PackedDims& d, int heads);
// Tensor map of a [total, heads, N] tensor with {64, box_heads, box_rows} boxes, 128-byte swizzle.
int packed_map(CUtensorMap* map, const PackedDims& d, int dtype, const void* base, long long tok, long long head,
               int heads, int box_heads, int box_rows);
// Launch configuration whose kernel may start while the one before it ends; the kernel calls pdl_wait().
cudaLaunchConfig_t packed_launch(int grid, int threads, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr);

}  // namespace mea
