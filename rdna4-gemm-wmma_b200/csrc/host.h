// Host-side helpers of b2g_api.cu that the other translation units of libb2g_gemm.so use:
// error reporting, the options, the tensor-map cache, per-device facts and the stream-ordered
// workspace pool.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "../../include/b2g_gemm.h"

namespace b2g {

// Sets the calling thread's error message and returns `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
void clear_error();
// Path reported by b2g_last_path().
void set_path(int path);
void count_launch();

// Options (b2g_set_option) that every tensor-core launch obeys.
struct LaunchOptions {
  int cta_group, tile_n, split_k, raster_group, force_generic, fault_flags;
  bool tail_split, pdl, cluster_fixup, serial_fixup;
  int64_t timeout_ns;
};
LaunchOptions launch_options();

// Current device: ordinal, SM count and compute capability (looked up once per device).
int current_device(int* dev, int* sm_count, int* cc_major);

// Tensor map of a pure (address, type, dims, strides, box, swizzle, promotion), cached.
CUresult encode_cached(CUtensorMap* out, CUtensorMapDataType dt, cuuint32_t rank, void* addr,
                       const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                       CUtensorMapSwizzle swz, CUtensorMapL2promotion l2);

// Stream-ordered pool of the workspaces on the current device.
int split_pool(cudaMemPool_t* out);

// Error check and launch count of one kernel launch.
inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  count_launch();
  return B2G_OK;
}

// Operand classes of the 8-bit operators.
inline bool is_real(int dt) {
  return dt == B2G_DTYPE_F16 || dt == B2G_DTYPE_BF16 || dt == B2G_DTYPE_F32;
}
inline bool is_q8(int dt) { return dt == B2G_DTYPE_I8 || dt == B2G_DTYPE_E4M3; }

// Refuses pointers below the alignment of their element type, which the kernels' accesses rely on
// (null: an optional argument that is not given).
struct Operand {
  const char* name;
  const void* p;
  int dtype;
};
inline int check_alignment(std::initializer_list<Operand> ops) {
  for (const Operand& o : ops) {
    const uintptr_t size = o.dtype == B2G_DTYPE_F32 ? 4 : is_real(o.dtype) ? 2 : 1;
    if ((uintptr_t)o.p % size != 0)
      return fail(B2G_ERR_INVALID_ARG, "%s is not aligned to its element type", o.name);
  }
  return B2G_OK;
}

// b2g_dequantize_q8 without its argument checks (b2g_rows.cu).
int dequantize_rows(const void* Q, const float* scale, void* X, int64_t M, int64_t N, int64_t ldq,
                    int64_t ldx, int q_dtype, int dtype, cudaStream_t s);

// Stream-ordered workspace from that pool, given back on the same stream when it goes out of
// scope (the kernels queued before then keep it).
class Workspace {
 public:
  explicit Workspace(cudaStream_t stream) : stream_(stream) {}
  ~Workspace() {
    if (ptr_) cudaFreeAsync(ptr_, stream_);
  }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
  int alloc(size_t bytes, const char* what) {
    cudaMemPool_t pool = nullptr;
    const int rc = split_pool(&pool);
    if (rc != B2G_OK) return rc;
    const cudaError_t e = cudaMallocFromPoolAsync(&ptr_, bytes, pool, stream_);
    if (e != cudaSuccess) {
      ptr_ = nullptr;
      cudaGetLastError();
      return cuda_fail(e, what);
    }
    return B2G_OK;
  }
  void* get() const { return ptr_; }

 private:
  cudaStream_t stream_;
  void* ptr_ = nullptr;
};

}  // namespace b2g
