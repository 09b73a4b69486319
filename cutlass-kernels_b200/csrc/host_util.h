// Host-side helpers shared by the C-ABI translation units: TMA descriptor encoding through the
// driver entry point (no link-time libcuda dependency), the per-device status block, and error text.
// The reference builds its TMA descriptors with CuTe's make_tma_copy inside each launcher
// (src/fmha-pipeline/fmha_forward.cu:144-252, src/cute-gemm-tma-gma/gemm.cu:363-384).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cfk_b200.h"

namespace cfk {

// Records the text of a CUDA runtime error for cfk_last_cuda_error(); returns its argument.
cudaError_t note_cuda(cudaError_t e, const char* what);

// Launch with programmatic stream serialization: the kernel may be set up on the device while the launch before it in
// the stream is still running, and waits for it with grid_dependency_wait() (common.cuh) before it touches memory.
// Plain back-to-back launches of a kernel of a few microseconds repeat every 4.1, 6.2 or 8.2 us on B200 (steps of 2.05 us
// whatever the kernel does); launched this way the period is the kernel's own work plus about 1.2 us, and the host side
// of a launch takes 2.1 us instead of 2.6.
// `cluster` > 1: in clusters of so many CTAs along x (for kernels without a cluster size of their own).
template <class... KArgs, class... Args>
inline cudaError_t launch_overlapped_in(int cluster, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                        cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}
template <class... KArgs, class... Args>
inline cudaError_t launch_overlapped(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                     const Args&... args) {
  return launch_overlapped_in(1, kern, grid, block, smem, stream, args...);
}

// Allows a kernel `bytes` of dynamic shared memory on the current device; asked once per thread and device.  Internal linkage: the
// record belongs to the kernel of this copy of the library.
template <class... KArgs>
static int allow_shared_memory(void (*kern)(KArgs...), int bytes) {
  static thread_local const void* kernel = nullptr;       // a translation unit instantiates this for one kernel or a few
  static thread_local int device = -1;
  int dev = 0;
  if (note_cuda(cudaGetDevice(&dev), "cudaGetDevice") != cudaSuccess) return CFK_ERR_NO_DRIVER;
  if (device == dev && kernel == reinterpret_cast<const void*>(kern)) return CFK_OK;
  if (note_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                "cudaFuncSetAttribute(shared memory)") != cudaSuccess)
    return CFK_ERR_LAUNCH;
  device = dev;
  kernel = reinterpret_cast<const void*>(kern);
  return CFK_OK;
}

// SMs of the one device this library is built for.  Only the choice between kernels and the sizes of grids follow from it.
constexpr int kSMs = 148;

// Device pointer to the 256-byte status block of the current device (int[64]; word 0 is the status
// word the kernels write).  nullptr (and *err set) if there is no usable device.
int* device_status_block(int* err);

// Device address of the fixed scratch array that cfk_fmha_forward_static uses (fmha_static.cu); allocates nothing.
int* static_scratch_for_current_device(int* err);

inline int dtype_size(int dt) { return dt == CFK_E4M3 || dt == CFK_INT8 ? 1 : (dt == CFK_FP32 ? 4 : 2); }

// Rows of a matrix as the feed-forward operators take them: at multiples of 16 bytes, not overlapping, within what a tensor map's
// stride field holds (2^40 bytes for all rows).
inline bool rows_ok(const void* base, int dt, int64_t cols, int64_t stride) {
  return ((uintptr_t)base & 15u) == 0 && stride >= cols && stride < (int64_t)1 << 31 && (stride * dtype_size(dt)) % 16 == 0;
}

// Rows of a matrix in memory: `rows` of `bytes` bytes, `stride` bytes apart.
struct RowSpan {
  const void* base;
  int64_t rows, bytes, stride;
};
// Whether two of them share memory (a null base shares none).  Finds it for matrices with the same distance of rows, as halves of a
// wider matrix have, and for those without gaps; of others it looks at the first row of the one that begins later.
inline bool share_memory(const RowSpan& a, const RowSpan& b) {
  if (!a.base || !b.base) return false;
  const bool a_first = (uintptr_t)a.base <= (uintptr_t)b.base;
  const RowSpan &lo = a_first ? a : b, &hi = a_first ? b : a;
  const int64_t d = (int64_t)((uintptr_t)hi.base - (uintptr_t)lo.base);
  const int64_t row = d / lo.stride, at = d % lo.stride;           // of lo; no product of sizes, which could pass 64 bits
  if (row >= lo.rows) return false;
  const int64_t run = hi.stride == hi.bytes ? hi.rows : 1;         // rows that hi covers without a gap
  return at < lo.bytes || (row + 1 < lo.rows && run > (lo.stride - at) / hi.bytes);
}

// Generic tiled descriptor.  dims/box are innermost first; strides_bytes has rank-1 entries.
// Returns CFK_OK, CFK_ERR_NO_DRIVER or CFK_ERR_DESCRIPTOR.
int encode_tiled(CUtensorMap* map, int dtype, int rank, const void* base, const uint64_t* dims,
                 const uint64_t* strides_bytes, const uint32_t* box, int swizzle_bytes /* 128, 64 or 0 */);

// [batch][seq][head][d] tensor (element strides sb, ss, sh; d contiguous) seen as the 5-D tensor
// {128-byte span, seq, spans per row, head, batch}; a box is {span, box_rows, all spans, 1, 1}, so
// one copy lands in shared memory as [span][row][128 B] with the 128-byte swizzle applied.  Rows of 64 bytes
// (e4m3, d = 64) are a single 64-byte span with the 64-byte swizzle.
int encode_bshd(CUtensorMap* map, int dtype, const void* base, int batch, int seq, int heads, int d, int64_t sb,
                int64_t ss, int64_t sh, int box_rows, int box_spans = 0 /* 0 = all spans of a row */);

}  // namespace cfk
