// Row operators of the 8-bit linear layer: rows into 8 bits and out again, the RMS norm with an
// 8-bit output, and its backward pass.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/b2g_gemm.h"
#include "errors.h"
#include "host.h"
#include "plan.h"
#include "ptx.cuh"
#include "q8.cuh"

namespace b2g {

// First bounded wait of the row kernels that gave up (0: none), merged into b2g_device_status().
static __device__ int g_rows_error;

int rows_device_error(int clear, int* value) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_rows_error, sizeof(int));
  if (e == cudaSuccess && clear) {
    const int z = 0;
    e = cudaMemcpyToSymbol(g_rows_error, &z, sizeof(int));
  }
  return (int)e;
}

namespace {

using namespace q8;

constexpr int ERR_WAIT_ROW = 8;  // a row's bulk copy did not arrive

constexpr int kRowThreads = 256;
constexpr int kLongThreads = 512;  // of a block that passes twice over a long row

// Sum over the block, returned to every thread.  `buf` holds one word per
// warp; the leading barrier lets consecutive calls share it.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) s += buf[i];
  return s;
}

struct NormArgs {
  const void *X, *R, *W;
  void *H, *Q;
  float *scale, *rstd;
  int64_t M, N, ldx, ldr, ldh, ldq;
  int dtype, w_dtype, q_dtype;
  float eps;
  bool norm, pow2;
  bool fault;  // test-only: a ring's copies are left out, so that its waits run out
};

// ------------------------------------------------------------------ vectors of a row
// VEC consecutive elements, loaded and stored as one piece.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T e[VEC];
};

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__half* d, float v) { *d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16* d, float v) { *d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float* d, float v) { *d = v; }

// Elements [n, n + VEC) of a row of N (a multiple of VEC), zeros past the row.  One predicated load: a
// branch with an element-wise end would make every load wait for the one before it.
// AGAIN: the row is read once more (otherwise it must not displace the weights from L1).
template <typename T, int VEC, bool AGAIN = false>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* row, int n, int N) {
  Vec<T, VEC> v;
  if constexpr (sizeof(v) == 16) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (n < N) u = AGAIN ? *reinterpret_cast<const uint4*>(row + n) : __ldcs(reinterpret_cast<const uint4*>(row + n));
    *reinterpret_cast<uint4*>(&v) = u;
  } else if constexpr (sizeof(v) == 8) {
    uint2 u = make_uint2(0, 0);
    if (n < N) u = __ldcs(reinterpret_cast<const uint2*>(row + n));
    *reinterpret_cast<uint2*>(&v) = u;
  } else {
    static_assert(VEC == 1 || sizeof(v) == 4, "vector size");
    if constexpr (sizeof(v) == 4) {
      uint32_t u = 0;
      if (n < N) u = *reinterpret_cast<const uint32_t*>(row + n);
      *reinterpret_cast<uint32_t*>(&v) = u;
    } else if constexpr (sizeof(v) == 2) {
      uint16_t u = 0;
      if (n < N) u = *reinterpret_cast<const uint16_t*>(row + n);
      *reinterpret_cast<uint16_t*>(&v) = u;
    } else {
      uint8_t u = 0;
      if (n < N) u = *reinterpret_cast<const uint8_t*>(row + n);
      *reinterpret_cast<uint8_t*>(&v) = u;
    }
  }
  return v;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* row, int n, int N, const Vec<T, VEC>& v) {
  if (n < N) *reinterpret_cast<Vec<T, VEC>*>(row + n) = v;
}

// VEC weights as fp32 (any type; cached in L1 for the block's next row).
template <int VEC>
__device__ __forceinline__ void load_weights(const void* W, int w_dtype, bool vec, int n, int N, float (&w)[VEC]) {
  if constexpr (VEC >= 4) {
    if (vec) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {  // four at a time: 16 bytes of fp32, 8 of the 16-bit types
        if (w_dtype == B2G_DTYPE_F32) {
          float4 x = make_float4(0, 0, 0, 0);
          if (n < N) x = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(W) + n + j));
          w[j] = x.x; w[j + 1] = x.y; w[j + 2] = x.z; w[j + 3] = x.w;
        } else {
          uint2 x = make_uint2(0, 0);
          if (n < N) x = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(W) + n + j));
          const uint32_t b[2] = {x.x, x.y};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (w_dtype == B2G_DTYPE_BF16) {
              w[j + 2 * k] = __uint_as_float(b[k] << 16);
              w[j + 2 * k + 1] = __uint_as_float(b[k] & 0xffff0000u);
            } else {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[k]));
              w[j + 2 * k] = f.x;
              w[j + 2 * k + 1] = f.y;
            }
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) {  // (no branch around the loads, which would then follow one another)
    uint32_t bits = 0;
    if (n + j < N && w_dtype == B2G_DTYPE_F32) bits = __ldg(static_cast<const uint32_t*>(W) + n + j);
    if (n + j < N && w_dtype != B2G_DTYPE_F32) bits = __ldg(static_cast<const uint16_t*>(W) + n + j);
    w[j] = w_dtype == B2G_DTYPE_F32    ? __uint_as_float(bits)
           : w_dtype == B2G_DTYPE_BF16 ? __uint_as_float(bits << 16)
                                       : __half2float(__ushort_as_half((unsigned short)bits));
  }
}

__device__ __forceinline__ bool weights_vec(const void* W, int w_dtype) {
  return (reinterpret_cast<uintptr_t>(W) & (w_dtype == B2G_DTYPE_F32 ? 15 : 7)) == 0;
}

// (sum, integer maximum) over the threads of a row: LANES consecutive lanes of a warp, or (LANES = 0)
// the block.  `buf` holds two words per warp for each parity of the row count, so consecutive rows
// need one barrier each.  SUM: whether the sum is wanted.
template <int LANES, bool SUM>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& top, float* buf, int parity) {
  constexpr int L = LANES ? LANES : 32;
  if constexpr (SUM) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if constexpr (L == 32) {
    top = __reduce_max_sync(0xffffffffu, top);
  } else {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if constexpr (LANES == 0) {
    float2* b = reinterpret_cast<float2*>(buf) + parity * 32;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = make_float2(sum, __uint_as_float(top));
    __syncthreads();
    const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
    const float2 x = lane < warps ? b[lane] : make_float2(0.0f, 0.0f);
    if constexpr (SUM) {
      sum = x.x;
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    top = __reduce_max_sync(0xffffffffu, __float_as_uint(x.y));
  }
}

// Rows into 8 bits, each row held in registers: one pass over the data.  A row belongs to LANES lanes of
// a warp (short rows) or, LANES = 0, to the block; a thread holds V vectors of VEC elements of it,
// `threads` vectors apart.  Blocks stride over the rows; where registers allow (AHEAD: blocks of up
// to 256 threads, and single elements) a row's loads are issued before the previous row is reduced,
// so that the reduction is not waited out with the memory idle, and the weights stay in registers.
//
// Per row: sum of squares and largest |h * w| (|x| without the norm).  The largest |y| is rstd
// times that, so one reduction serves both; rstd cancels from the 8-bit values (row_quant).
//
// Measured (us, bf16, graph): short rows, several a warp against one a block: quantize 16384 x 256 4.5
// against 5.8, 100000 x 64 6.0 against 22.6, norm with residual 16384 x 256 12.4 (2.4 TB/s, bound
// by instructions) against 14.0, 16384 x 512 22 against 27.  Few long rows (latency): quantize 1 x 8192
// 2.3, norm 148 x 4096 3.4.
template <typename T, bool NORM, int VEC, int V, int LANES, bool AHEAD>
__global__ void __launch_bounds__(LANES ? 128 : AHEAD ? 256 : 1024, LANES ? 7 : AHEAD ? 2 : 1)
    rows_to_q8_kernel(const NormArgs a) {
  __shared__ float buf[128];
  constexpr int PER = LANES ? 128 / LANES : 1;  // rows a block holds at once
  const int tid = LANES ? (int)threadIdx.x % (LANES ? LANES : 1) : (int)threadIdx.x;
  const int threads = LANES ? LANES : (int)blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * PER + (LANES ? (int)threadIdx.x / (LANES ? LANES : 1) : 0);
  const int64_t step = (int64_t)gridDim.x * PER;
  const T* X = static_cast<const T*>(a.X);
  const T* R = static_cast<const T*>(a.R);
  const int N = (int)a.N;
  const bool wvec = NORM && weights_vec(a.W, a.w_dtype);
  Vec<T, VEC> x[V], r[V];
  auto fetch = [&](int64_t m) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = load_vec<T, VEC>(X + m * a.ldx, (i * threads + tid) * VEC, N);
    if (NORM && R)
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = load_vec<T, VEC>(R + m * a.ldr, (i * threads + tid) * VEC, N);
  };
  if (AHEAD && first < a.M) fetch(first);
  float wreg[NORM && AHEAD ? V : 1][VEC];
  if constexpr (NORM && AHEAD)
#pragma unroll
    for (int i = 0; i < V; ++i) load_weights<VEC>(a.W, a.w_dtype, wvec, (i * threads + tid) * VEC, N, wreg[i]);
  int parity = 0;
  // (the lanes of a warp stay together: those whose rows have run out go on with the last row's
  // values until the warp's first row is past the end, and store nothing)
  const int64_t end = LANES ? a.M + (int64_t)(threadIdx.x % 32) / (LANES ? LANES : 1) : a.M;
  for (int64_t m = first; m < end; m += step, parity ^= 1) {
    const bool live = m < a.M;
    if (!AHEAD && live) fetch(m);
    float v[V][VEC];
    float ss = 0.0f, ftop = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = to_f(x[i].e[j]);
      if constexpr (NORM) {
        if (R) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += to_f(r[i].e[j]);
        }
        if (a.H && live) {
          Vec<T, VEC> h;
#pragma unroll
          for (int j = 0; j < VEC; ++j) from_f(&h.e[j], v[i][j]);
          store_vec<T, VEC>(static_cast<T*>(a.H) + m * a.ldh, n, N, h);
        }
        float w[VEC];
        if constexpr (!AHEAD) load_weights<VEC>(a.W, a.w_dtype, wvec, n, N, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ss = fmaf(v[i][j], v[i][j], ss);
          v[i][j] *= AHEAD ? wreg[NORM && AHEAD ? i : 0][j] : w[j];
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) ftop = max_abs(ftop, v[i][j]);
    }
    uint32_t top = __float_as_uint(ftop);
    if (AHEAD && m + step < a.M) fetch(m + step);
    row_reduce<LANES, NORM>(ss, top, buf, parity);
    if (!live) continue;
    const float rstd = NORM ? 1.0f / sqrtf(ss / (float)N + a.eps) : 1.0f;
    const RowQuant rq = row_quant(top, rstd, q_max(a.q_dtype), a.pow2);
    if (tid == 0) {
      a.scale[m] = rq.scale;
      if (NORM && a.rstd) a.rstd[m] = rstd;
    }
    const bool bad = rq.scale != rq.scale;
    uint8_t* q = static_cast<uint8_t*>(a.Q) + m * a.ldq;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Vec<uint8_t, VEC> o;
      pack_q8<VEC>(v[i], rq, a.q_dtype, bad, o.e);
      store_vec<uint8_t, VEC>(q, (i * threads + tid) * VEC, N, o);
    }
  }
}

// VEC 16-byte-aligned elements from shared memory as fp32.
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const uint8_t* p, float (&v)[VEC]) {
  const Vec<T, VEC> x = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = to_f(x.e[j]);
}

// A ring of row buffers in shared memory, filled by bulk copies.  `full` barriers count the bytes of each
// buffer; thread 0 refills a buffer once every thread has read it.  Copies run ahead of the rows by
// up to `stages`, which keeps the memory busy however long a row's reduction takes, and costs no
// registers.  A wait that runs out raises the block's flag, and every row from there on comes out as NaN:
// each thread looks at the flag after its wait, not at the wait's answer, because a buffer that is not
// refilled shows every other of its later phases as complete.
struct Ring {
  uint32_t base, bars, stage_bytes;
  int stages;
  volatile int* abort_flag;
  uint64_t limit_ns;
  __device__ __forceinline__ uint32_t stage(int k) const { return base + (uint32_t)(k % stages) * stage_bytes; }
  __device__ __forceinline__ uint32_t bar(int k) const { return bars + 8u * (uint32_t)(k % stages); }
  __device__ __forceinline__ bool wait(int k) const {
    return ptx::mbar_wait(bar(k), (uint32_t)(k / stages) & 1u, abort_flag, &g_rows_error, ERR_WAIT_ROW, limit_ns);
  }
  // After a wait gave up: no copy may be in flight when the shared memory goes away.
  __device__ __forceinline__ void drain(int issued) const {
    for (int i = max(0, issued - stages); i < issued; ++i)
      ptx::mbar_wait_drain(bar(i), (uint32_t)(i / stages) & 1u, &g_rows_error, ERR_WAIT_ROW, limit_ns);
  }
};

// A ring of `stages` buffers at the start of dynamic shared memory, its barriers behind them.
__device__ __forceinline__ Ring make_ring(uint8_t* smem, int stages, uint32_t stage_bytes, uint64_t limit_ns,
                                          int* abort_flag) {
  const uint32_t base = ptx::smem_u32(smem), bars = base + (uint32_t)stages * stage_bytes;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) ptx::mbar_init(bars + 8u * i, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  return {base, bars, stage_bytes, stages, abort_flag, limit_ns};
}

// rows_to_q8_kernel with its rows in a ring: rows of whole 16-byte vectors, one row at a time a block of
// up to THREADS threads, which hold V vectors each.  The norm's weights stay in registers where V <= 4.
// CTAS blocks share an SM, so that one's reduction overlaps the others' arithmetic.  Bound by memory: bf16,
// norm with residual 8192 x 8192 82 us and 16384 x 4096 82 us (5.7 TB/s), quantize 16384 x 8192 77 us
// (5.2 TB/s); rows of 1024 by instructions, norm 16384 x 1024 27.5 us (4.3 TB/s).
template <typename T, bool NORM, int V, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS)
    rows_ring_kernel(const NormArgs a, int stages, uint32_t row_bytes, uint64_t limit_ns) {
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr bool WREG = NORM && V <= 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float buf[128];
  __shared__ int abort_flag;
  const int tid = (int)threadIdx.x, threads = (int)blockDim.x;
  const int64_t first = blockIdx.x, step = gridDim.x;
  const T* X = static_cast<const T*>(a.X);
  const T* R = NORM ? static_cast<const T*>(a.R) : nullptr;
  const int N = (int)a.N;
  const uint32_t r_off = row_bytes;  // R's row follows X's in a stage
  const Ring ring = make_ring(smem, stages, R ? 2 * row_bytes : row_bytes, limit_ns, &abort_flag);
  auto fill = [&](int64_t m, int k) {
    const uint32_t bar = ring.bar(k), dst = ring.stage(k);
    ptx::mbar_arrive_expect_tx(bar, R ? 2 * row_bytes : row_bytes);
    ptx::bulk_load(dst, X + m * a.ldx, row_bytes, bar);
    if (R) ptx::bulk_load(dst + r_off, R + m * a.ldr, row_bytes, bar);
  };
  int issued = 0;
  if (tid == 0)
    for (int64_t m = first + (a.fault ? a.M : 0); m < a.M && issued < stages; m += step) fill(m, issued++);
  const bool wvec = NORM && weights_vec(a.W, a.w_dtype);
  float wreg[WREG ? V : 1][VEC];
  if constexpr (WREG)
#pragma unroll
    for (int i = 0; i < V; ++i) load_weights<VEC>(a.W, a.w_dtype, wvec, (i * threads + tid) * VEC, N, wreg[i]);
  int k = 0;
  for (int64_t m = first; m < a.M; m += step, ++k) {
    ring.wait(k);
    const uint8_t* st = smem + (uint32_t)(k % stages) * ring.stage_bytes;
    float v[V][VEC];
    F2 ss = f2(0.0f, 0.0f);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
      if (n < N) {
        unpack<T, VEC>(st + n * (int)sizeof(T), v[i]);
        if constexpr (NORM) {
          if (R) {
            float r[VEC];
            unpack<T, VEC>(st + r_off + n * (int)sizeof(T), r);
#pragma unroll
            for (int j = 0; j < VEC; j += 2)
              f2_get(f2_add(f2(v[i][j], v[i][j + 1]), f2(r[j], r[j + 1])), v[i][j], v[i][j + 1]);
          }
          if (a.H) {
            Vec<T, VEC> h;
#pragma unroll
            for (int j = 0; j < VEC; ++j) from_f(&h.e[j], v[i][j]);
            *reinterpret_cast<Vec<T, VEC>*>(static_cast<T*>(a.H) + m * a.ldh + n) = h;
          }
          float wl[VEC];
          if constexpr (!WREG) load_weights<VEC>(a.W, a.w_dtype, wvec, n, N, wl);
#pragma unroll
          for (int j = 0; j < VEC; j += 2) {
            const F2 h = f2(v[i][j], v[i][j + 1]);
            ss = f2_fma(h, h, ss);
            const F2 w = WREG ? f2(wreg[WREG ? i : 0][j], wreg[WREG ? i : 0][j + 1]) : f2(wl[j], wl[j + 1]);
            f2_get(f2_mul(h, w), v[i][j], v[i][j + 1]);
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) top = max_abs(top, v[i][j]);
      }
    }
    float s0, s1;
    f2_get(ss, s0, s1);
    float sum = s0 + s1;
    uint32_t bits = __float_as_uint(top);
    if (*ring.abort_flag) {
      bits = 0x7fffffffu;
      sum = __int_as_float(0x7fc00000);
    }
    row_reduce<0, NORM>(sum, bits, buf, k & 1);
    if (tid == 0 && m + step * stages < a.M && !*ring.abort_flag) {
      fill(m + step * stages, k + stages);  // every thread has read this row (row_reduce)
      ++issued;
    }
    const float rstd = NORM ? 1.0f / sqrtf(sum / (float)N + a.eps) : 1.0f;
    const RowQuant rq = row_quant(bits, rstd, q_max(a.q_dtype), a.pow2);
    if (tid == 0) {
      a.scale[m] = rq.scale;
      if (NORM && a.rstd) a.rstd[m] = rstd;
    }
    const bool bad = rq.scale != rq.scale;
    uint8_t* q = static_cast<uint8_t*>(a.Q) + m * a.ldq;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
      if (n < N) {
        Vec<uint8_t, VEC> o;
        pack_q8<VEC>(v[i], rq, a.q_dtype, bad, o.e);
        *reinterpret_cast<Vec<uint8_t, VEC>*>(q + n) = o;
      }
    }
  }
  if (NORM && a.H && *ring.abort_flag)  // H was stored before its row was known to be lost
    for (int64_t m = first; m < a.M; m += step)
      for (int n = tid; n < N; n += (int)blockDim.x) from_f(static_cast<T*>(a.H) + m * a.ldh + n, __int_as_float(0x7fc00000));
  if (tid == 0 && *ring.abort_flag) ring.drain(issued);
}

// Bulk copy of a row of `bytes` bytes without 16-byte alignment: the whole 16-byte pieces that hold it.
// The pieces at its ends reach up to 15 bytes into the neighbouring rows, whose bytes are not used;
// the matrix's first and last row, whose pieces could reach out of it, are never copied this way.
__device__ __forceinline__ uint32_t span_bytes(const void* row, uint32_t bytes) {
  return (((uint32_t)(uintptr_t)row & 15u) + bytes + 15u) & ~15u;
}
__device__ __forceinline__ void span_load(uint32_t dst, const void* row, uint32_t bytes, uint32_t bar) {
  ptx::bulk_load(dst, reinterpret_cast<const void*>((uintptr_t)row & ~(uintptr_t)15), span_bytes(row, bytes), bar);
}
__device__ __forceinline__ uint32_t low4(const void* p) { return (uint32_t)(uintptr_t)p & 15u; }

// rows_ring_kernel for rows of any alignment, element by element: element i * THREADS + tid of a row is a
// thread's, so that shared and global accesses of a warp are consecutive.  Q, H and the first and
// last row go through ordinary accesses.  Instructions are the limit here (one access an element and
// operand), so THREADS is a constant: every address is one base with a constant offset.  bf16, norm with
// residual 8192 x 8191 129 us (3.6 TB/s); 8192 x 8192 at an odd pitch 129 us, where rows_ring_kernel
// takes 82 for aligned rows, quantize 16384 x 8192 116 against 77.
template <typename T, bool NORM, int THREADS, int V>
__global__ void __launch_bounds__(THREADS, V <= 16 ? 1024 / THREADS : 1)
    rows_ring_elems_kernel(const NormArgs a, int stages, uint32_t slot, uint64_t limit_ns) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float buf[128];
  __shared__ int abort_flag;
  const int tid = (int)threadIdx.x;
  const int64_t first = blockIdx.x, step = gridDim.x;
  const T* X = static_cast<const T*>(a.X);
  const T* R = NORM ? static_cast<const T*>(a.R) : nullptr;
  const int N = (int)a.N;
  const uint32_t row_bytes = (uint32_t)N * (uint32_t)sizeof(T);
  const Ring ring = make_ring(smem, stages, R ? 2 * slot : slot, limit_ns, &abort_flag);
  auto at_end = [&](int64_t m) { return m == 0 || m == a.M - 1; };
  auto fill = [&](int64_t m, int k) {
    const uint32_t bar = ring.bar(k), dst = ring.stage(k);
    if (at_end(m)) {
      ptx::mbar_arrive(bar);  // read from global memory when its turn comes
      return;
    }
    const T* x = X + m * a.ldx;
    const T* r = R ? R + m * a.ldr : nullptr;
    ptx::mbar_arrive_expect_tx(bar, span_bytes(x, row_bytes) + (R ? span_bytes(r, row_bytes) : 0));
    span_load(dst, x, row_bytes, bar);
    if (R) span_load(dst + slot, r, row_bytes, bar);
  };
  int issued = 0;
  if (tid == 0)
    for (int64_t m = first + (a.fault ? a.M : 0); m < a.M && issued < stages; m += step) fill(m, issued++);
  float w[NORM ? V : 1];
  if constexpr (NORM)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float f[1];
      load_weights<1>(a.W, a.w_dtype, false, i * THREADS + tid, N, f);
      w[i] = f[0];
    }
  int k = 0;
  for (int64_t m = first; m < a.M; m += step, ++k) {
    ring.wait(k);
    const bool end = at_end(m);
    const uint8_t* st = smem + (uint32_t)(k % stages) * ring.stage_bytes;
    const T* gx = X + m * a.ldx;
    const T* gr = R ? R + m * a.ldr : nullptr;
    const T* sx = reinterpret_cast<const T*>(st + low4(gx));
    const T* sr = reinterpret_cast<const T*>(st + slot + low4(gr));
    float v[V];
    float sum = 0.0f, top = 0.0f;
    const int count = N - tid;  // element i is in the row if i * THREADS < count
    auto take = [&](const T* x, const T* r) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = i * THREADS < count ? to_f(x[i * THREADS]) : 0.0f;
      if (NORM && R)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += i * THREADS < count ? to_f(r[i * THREADS]) : 0.0f;
    };
    if (end)
      take(gx + tid, gr + tid);
    else
      take(sx + tid, sr + tid);
    if (NORM && a.H) {
      T* h = static_cast<T*>(a.H) + m * a.ldh + tid;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i * THREADS < count) from_f(h + i * THREADS, v[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (NORM) {
        sum = fmaf(v[i], v[i], sum);
        v[i] *= w[NORM ? i : 0];
      }
      top = max_abs(top, v[i]);
    }
    uint32_t bits = __float_as_uint(top);
    if (*ring.abort_flag) {
      bits = 0x7fffffffu;
      sum = __int_as_float(0x7fc00000);
    }
    row_reduce<0, NORM>(sum, bits, buf, k & 1);
    if (tid == 0 && m + step * stages < a.M && !*ring.abort_flag) {
      fill(m + step * stages, k + stages);  // every thread has read this row (row_reduce)
      ++issued;
    }
    const float rstd = NORM ? 1.0f / sqrtf(sum / (float)N + a.eps) : 1.0f;
    const RowQuant rq = row_quant(bits, rstd, q_max(a.q_dtype), a.pow2);
    if (tid == 0) {
      a.scale[m] = rq.scale;
      if (NORM && a.rstd) a.rstd[m] = rstd;
    }
    const bool bad = rq.scale != rq.scale;
    uint8_t* q = static_cast<uint8_t*>(a.Q) + m * a.ldq + tid;
    uint32_t o[V];
    round_q8<V>(v, rq, a.q_dtype, bad, o);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * THREADS < count) q[i * THREADS] = (uint8_t)o[i];
  }
  if (NORM && a.H && *ring.abort_flag)  // H was stored before its row was known to be lost
    for (int64_t m = first; m < a.M; m += step)
      for (int n = tid; n < N; n += (int)blockDim.x) from_f(static_cast<T*>(a.H) + m * a.ldh + n, __int_as_float(0x7fc00000));
  if (tid == 0 && *ring.abort_flag) ring.drain(issued);
}

// The same for rows too long for a block's registers (over 32768 16-bit or 16384 fp32 elements, aligned; over
// 16384, unaligned): two passes over the row, the second from L2.  Bound by its loads' latency: bf16,
// quantize 8192 x 40000 220 us (4.5 TB/s), norm with residual 8192 x 40960 858 us (2.7 TB/s).
template <typename T, bool NORM, int VEC>
__global__ void __launch_bounds__(kLongThreads, NORM ? 1 : 2) long_rows_to_q8_kernel(const NormArgs a) {
  constexpr int P = VEC == 1 ? 8 : NORM ? 2 : 4;  // vectors a thread has in flight
  constexpr int SPAN = kLongThreads * VEC * P;
  __shared__ float buf[128];
  const int tid = (int)threadIdx.x;
  const bool wvec = NORM && weights_vec(a.W, a.w_dtype);
  int parity = 0;
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x, parity ^= 1) {
    const T* X = static_cast<const T*>(a.X) + m * a.ldx;
    const T* R = NORM && a.R ? static_cast<const T*>(a.R) + m * a.ldr : nullptr;
    // h of the SPAN elements from n0 on (zeros past the row), and with the norm h * w
    auto take = [&](int64_t n0, int left, float (&h)[P][VEC], float (&v)[P][VEC]) {
      Vec<T, VEC> x[P], r[P];
#pragma unroll
      for (int i = 0; i < P; ++i) x[i] = load_vec<T, VEC, true>(X + n0, (i * kLongThreads + tid) * VEC, left);
      if (R)
#pragma unroll
        for (int i = 0; i < P; ++i) r[i] = load_vec<T, VEC, true>(R + n0, (i * kLongThreads + tid) * VEC, left);
#pragma unroll
      for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = to_f(x[i].e[j]);
        if (R)
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] += to_f(r[i].e[j]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = h[i][j];
        if constexpr (NORM) {
          float w[VEC];
          const char* wp = static_cast<const char*>(a.W) + n0 * (a.w_dtype == B2G_DTYPE_F32 ? 4 : 2);
          load_weights<VEC>(wp, a.w_dtype, wvec, (i * kLongThreads + tid) * VEC, left, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] *= w[j];
        }
      }
    };
    float ss = 0.0f, ftop = 0.0f;
    for (int64_t n0 = 0; n0 < a.N; n0 += SPAN) {
      float h[P][VEC], v[P][VEC];
      take(n0, (int)min(a.N - n0, (int64_t)SPAN), h, v);
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if constexpr (NORM) ss = fmaf(h[i][j], h[i][j], ss);
          ftop = max_abs(ftop, v[i][j]);
        }
    }
    uint32_t top = __float_as_uint(ftop);
    row_reduce<0, NORM>(ss, top, buf, parity);
    const float rstd = NORM ? 1.0f / sqrtf(ss / (float)a.N + a.eps) : 1.0f;
    const RowQuant rq = row_quant(top, rstd, q_max(a.q_dtype), a.pow2);
    if (tid == 0) {
      a.scale[m] = rq.scale;
      if (NORM && a.rstd) a.rstd[m] = rstd;
    }
    const bool bad = rq.scale != rq.scale;
    for (int64_t n0 = 0; n0 < a.N; n0 += SPAN) {
      const int left = (int)min(a.N - n0, (int64_t)SPAN);
      float h[P][VEC], v[P][VEC];
      take(n0, left, h, v);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int n = (i * kLongThreads + tid) * VEC;
        Vec<uint8_t, VEC> o;
        pack_q8<VEC>(v[i], rq, a.q_dtype, bad, o.e);
        store_vec<uint8_t, VEC>(static_cast<uint8_t*>(a.Q) + m * a.ldq + n0, n, left, o);
        if (NORM && a.H) {
          Vec<T, VEC> x;
#pragma unroll
          for (int j = 0; j < VEC; ++j) from_f(&x.e[j], h[i][j]);
          store_vec<T, VEC>(static_cast<T*>(a.H) + m * a.ldh + n0, n, left, x);
        }
      }
    }
  }
}

// Rows out of 8 bits.  Memory-bound: 1 byte in, 2 or 4 out.  VEC16: 16 values a vector, two vectors a
// thread, vectors numbered over the whole matrix (so that short rows fill a block); else single
// values, eight a thread, a block's width apart in one row.  All loads go before the first store.
// 16384 x 8192 into bf16 66 us (6.1 TB/s), the single values' way 145 us.
constexpr int kPiece = 2, kPieceElems = 8;

template <typename T, bool VEC16>
__global__ void __launch_bounds__(kRowThreads)
    dequantize_kernel(const uint8_t* Q, const float* scale, T* X, int64_t M, int64_t N, int64_t ldq,
                      int64_t ldx, int q_dtype, float top) {
  if constexpr (VEC16) {
    constexpr int OUT = 16 / (int)sizeof(T);
    const uint32_t per_row = (uint32_t)((N + 15) / 16);
    const int64_t total = M * per_row, span = (int64_t)gridDim.x * kRowThreads * kPiece;
    for (int64_t i0 = (int64_t)blockIdx.x * kRowThreads * kPiece + threadIdx.x; i0 < total; i0 += span) {
      uint4 c[kPiece];
      float s[kPiece];
      int64_t m[kPiece], n[kPiece];
#pragma unroll
      for (int k = 0; k < kPiece; ++k) {
        const int64_t i = i0 + k * kRowThreads;
        m[k] = i >> 32 ? i / per_row : (int64_t)((uint32_t)i / per_row);
        n[k] = (i - m[k] * per_row) * 16;
        s[k] = 0.0f;
        if (i < total) {
          s[k] = __ldg(scale + m[k]);
          if (n[k] + 16 <= N) c[k] = __ldcs(reinterpret_cast<const uint4*>(Q + m[k] * ldq + n[k]));
        }
      }
#pragma unroll
      for (int k = 0; k < kPiece; ++k) {
        if (i0 + k * kRowThreads >= total) break;
        T* x = X + m[k] * ldx + n[k];
        const float f = s[k];
        // (a value that may pass the type's range, or a NaN scale, goes the slower way)
        if (n[k] + 16 <= N && fabsf(f) * 448.0f <= top) {
          const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
          Vec<T, OUT> o[16 / OUT];
          T* d = o[0].e;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            F2 lo, hi;
            unpack_q8x4(w[j], q_dtype, lo, hi);
            float v[4];
            f2_get(f2_mul(lo, f2(f, f)), v[0], v[1]);
            f2_get(f2_mul(hi, f2(f, f)), v[2], v[3]);
#pragma unroll
            for (int l = 0; l < 4; ++l) from_f(d + 4 * j + l, v[l]);
          }
#pragma unroll
          for (int j = 0; j < 16 / OUT; ++j) *reinterpret_cast<Vec<T, OUT>*>(x + j * OUT) = o[j];
        } else {
          const int count = N - n[k] < 16 ? (int)(N - n[k]) : 16;
          for (int j = 0; j < count; ++j) from_f(x + j, clamp_to(load_elem(Q + m[k] * ldq + n[k], j, q_dtype) * f, top));
        }
      }
    }
  } else {
    constexpr int per_block = kRowThreads * kPieceElems;
    const int64_t bpr = (N + per_block - 1) / per_block;  // pieces of a row
    for (int64_t b = blockIdx.x; b < M * bpr; b += gridDim.x) {
      const int64_t m = b / bpr, n0 = (b - m * bpr) * per_block + threadIdx.x;
      const uint8_t* q = Q + m * ldq + n0;
      T* x = X + m * ldx + n0;
      const float s = __ldg(scale + m);
      const int64_t left = N - n0;
      uint8_t c[kPieceElems];
#pragma unroll
      for (int i = 0; i < kPieceElems; ++i) c[i] = i * kRowThreads < left ? q[i * kRowThreads] : 0;
#pragma unroll
      for (int i = 0; i < kPieceElems; ++i)
        if (i * kRowThreads < left) {
          const float v = q_dtype == B2G_DTYPE_I8 ? (float)(int8_t)c[i]
                                                  : float(*reinterpret_cast<const __nv_fp8_e4m3*>(&c[i]));
          from_f(x + i * kRowThreads, clamp_to(v * s, top));
        }
    }
  }
}

struct BwdArgs {
  const void *dY, *X, *W, *dR;
  const float *x_scale, *rstd;
  void* dX;
  float* part;  // [blocks][N] partial sums of dw, or null
  int64_t M, N, ldy, ldx, ldr, lddx;
  int dtype, x_dtype, w_dtype;
  bool fault;  // as NormArgs::fault
};

// Any size, alignment and checkpoint type, one block a row at a time, element by element: mean(g * xh), then
// dx, the second pass from L2.  X8: 8-bit checkpoint; else any 16- or 32-bit type.  The block's share of dw
// is added up in its row of partial sums.  Bound by its loads' latency (bf16, int8 checkpoint: 2048 x
// 32768 404 us, 4096 x 9001 215 us).

template <typename T, bool X8>
__global__ void __launch_bounds__(kLongThreads, 2) rmsnorm_bwd_kernel(const BwdArgs a) {
  constexpr int P = 8, SPAN = kLongThreads * P;  // elements a thread has in flight
  __shared__ float buf[kLongThreads / 32];
  const int tid = (int)threadIdx.x;
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const float rstd = __ldg(a.rstd + m), xs = a.x_scale ? __ldg(a.x_scale + m) * rstd : rstd;
    const T* dY = static_cast<const T*>(a.dY) + m * a.ldy;
    // dy, w and xh of the SPAN elements from n0 on (zeros past the row)
    auto take = [&](int64_t n0, int left, float (&dy)[P], float (&w)[P], float (&xh)[P]) {
#pragma unroll
      for (int i = 0; i < P; ++i) dy[i] = to_f(load_vec<T, 1>(dY + n0, i * kLongThreads + tid, left).e[0]);
      if constexpr (X8) {
        const uint8_t* X = static_cast<const uint8_t*>(a.X) + m * a.ldx + n0;
        uint8_t b[P];
#pragma unroll
        for (int i = 0; i < P; ++i) b[i] = load_vec<uint8_t, 1>(X, i * kLongThreads + tid, left).e[0];
#pragma unroll
        for (int i = 0; i < P; ++i) xh[i] = load_elem(&b[i], 0, a.x_dtype);
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const int n = i * kLongThreads + tid;
          xh[i] = n < left ? load_elem(a.X, m * a.ldx + n0 + n, a.x_dtype) : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float f[1];
        load_weights<1>(static_cast<const char*>(a.W) + n0 * (a.w_dtype == B2G_DTYPE_F32 ? 4 : 2), a.w_dtype, false,
                        i * kLongThreads + tid, left, f);
        w[i] = f[0];
        xh[i] *= xs;
      }
    };
    float c = 0.0f;
    for (int64_t n0 = 0; n0 < a.N; n0 += SPAN) {
      const int left = (int)min(a.N - n0, (int64_t)SPAN);
      float dy[P], w[P], xh[P];
      take(n0, left, dy, w, xh);
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (i * kLongThreads + tid < left) c = fmaf(dy[i] * w[i], xh[i], c);
    }
    c = block_sum(c, buf) / (float)a.N;
    for (int64_t n0 = 0; n0 < a.N; n0 += SPAN) {
      const int left = (int)min(a.N - n0, (int64_t)SPAN);
      float dy[P], w[P], xh[P], dr[P], dw[P];
      float* part = a.part ? a.part + (int64_t)blockIdx.x * a.N + n0 : nullptr;
      take(n0, left, dy, w, xh);
      if (a.dR) {
        const T* dR = static_cast<const T*>(a.dR) + m * a.ldr + n0;
#pragma unroll
        for (int i = 0; i < P; ++i) dr[i] = to_f(load_vec<T, 1>(dR, i * kLongThreads + tid, left).e[0]);
      }
      const bool add = part && m != blockIdx.x;
#pragma unroll
      for (int i = 0; i < P; ++i) dw[i] = add ? load_vec<float, 1>(part, i * kLongThreads + tid, left).e[0] : 0.0f;
      T* dX = static_cast<T*>(a.dX) + m * a.lddx + n0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int n = i * kLongThreads + tid;
        if (n < left) {
          float dx = rstd * (dy[i] * w[i] - xh[i] * c);
          if (a.dR) dx += dr[i];
          if (part) part[n] = fmaf(dy[i], xh[i], dw[i]);
          from_f(dX + n, dx);
        }
      }
    }
  }
}

// VEC checkpoint values from shared memory: 8-bit, or of the gradient's type.
template <typename T, bool X8>
struct XVec {
  static constexpr int VEC = 16 / (int)sizeof(T);
  static constexpr int SIZE = X8 ? VEC : 16;  // bytes
  alignas(16) uint32_t w[SIZE / 4];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (SIZE == 16)
      *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (SIZE == 8)
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else
      w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  __device__ __forceinline__ void get(int x_dtype, F2 (&v)[VEC / 2]) const {
    if constexpr (X8) {
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) unpack_q8x4(w[j], x_dtype, v[2 * j], v[2 * j + 1]);
    } else {
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) v[j] = f2(to_f(e[2 * j]), to_f(e[2 * j + 1]));
    }
  }
};

// rmsnorm_bwd_kernel over a ring of rows (dY, X and dR of whole 16-byte vectors).  A thread holds V
// vectors of a row, and its columns' share of dw in fp32 over all of the block's rows: dw costs no
// traffic but one partial row a block.  HOLD (up to 16 elements a thread): the weights, and a row's
// dy * w and xh, stay in fp32 registers; else a row stays packed between the reduction and the
// output and is unpacked twice, with the weights read from L1.  bf16, int8 checkpoint, residual:
// 8192 x 8192 86 us (5.5 TB/s), 8192 x 4096 52 us (packed, when compared, 102 against 50), 16384 x 1024 30 us
// (packed 57 against 31), 4096 x 16384, packed, 154 us (3.0 TB/s, instructions).
template <typename T, bool X8, int V, bool HOLD>
__global__ void __launch_bounds__(512, 1)
    rmsnorm_bwd_ring_kernel(const BwdArgs a, int stages, uint32_t y_bytes, uint32_t x_bytes,
                            uint64_t limit_ns) {
  using XV = XVec<T, X8>;
  constexpr int VEC = XV::VEC, P = VEC / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float buf[128];
  __shared__ int abort_flag;
  const int tid = (int)threadIdx.x, threads = (int)blockDim.x;
  const int64_t first = blockIdx.x, step = gridDim.x;
  const int N = (int)a.N;
  const T* dY = static_cast<const T*>(a.dY);
  const T* dR = static_cast<const T*>(a.dR);
  const uint8_t* X = static_cast<const uint8_t*>(a.X);
  const int64_t x_pitch = a.ldx * (X8 ? 1 : (int)sizeof(T));
  const uint32_t stage_bytes = (dR ? 2 * y_bytes : y_bytes) + x_bytes, r_off = y_bytes + x_bytes;
  const Ring ring = make_ring(smem, stages, stage_bytes, limit_ns, &abort_flag);
  auto fill = [&](int64_t m, int k) {
    const uint32_t bar = ring.bar(k), dst = ring.stage(k);
    ptx::mbar_arrive_expect_tx(bar, stage_bytes);
    ptx::bulk_load(dst, dY + m * a.ldy, y_bytes, bar);
    ptx::bulk_load(dst + y_bytes, X + m * x_pitch, x_bytes, bar);
    if (dR) ptx::bulk_load(dst + r_off, dR + m * a.ldr, y_bytes, bar);
  };
  int issued = 0;
  if (tid == 0)
    for (int64_t m = first + (a.fault ? a.M : 0); m < a.M && issued < stages; m += step) fill(m, issued++);
  const bool wvec = weights_vec(a.W, a.w_dtype);
  auto weights = [&](int i, F2 (&w)[P]) {
    float f[VEC];
    load_weights<VEC>(a.W, a.w_dtype, wvec, (i * threads + tid) * VEC, N, f);
#pragma unroll
    for (int j = 0; j < P; ++j) w[j] = f2(f[2 * j], f[2 * j + 1]);
  };
  F2 wreg[HOLD ? V : 1][P], g[HOLD ? V : 1][P], xh[HOLD ? V : 1][P];
  if constexpr (HOLD)
#pragma unroll
    for (int i = 0; i < V; ++i) weights(i, wreg[i]);
  F2 dw[V][P];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < P; ++j) dw[i][j] = f2(0.0f, 0.0f);
  // a row's two factors, loaded a row ahead
  float next_rstd = __ldg(a.rstd + first), next_scale = a.x_scale ? __ldg(a.x_scale + first) : 1.0f;
  int k = 0;
  for (int64_t m = first; m < a.M; m += step, ++k) {
    const float rstd = next_rstd, xs = next_scale * rstd;
    if (m + step < a.M) {
      next_rstd = __ldg(a.rstd + m + step);
      if (a.x_scale) next_scale = __ldg(a.x_scale + m + step);
    }
    const F2 xs2 = f2(xs, xs);
    ring.wait(k);
    const uint8_t* st = smem + (uint32_t)(k % stages) * stage_bytes;
    Vec<T, VEC> y[V], r[V];
    XV x[V];
    F2 c2 = f2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
      if (n < N) {
        y[i] = *reinterpret_cast<const Vec<T, VEC>*>(st + n * (int)sizeof(T));
        x[i].load(st + y_bytes + n * (X8 ? 1 : (int)sizeof(T)));
        if (dR) r[i] = *reinterpret_cast<const Vec<T, VEC>*>(st + r_off + n * (int)sizeof(T));
        F2 w[P], xv[P];
        if constexpr (!HOLD) weights(i, w);
        x[i].get(a.x_dtype, xv);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const F2 dy = f2(to_f(y[i].e[2 * j]), to_f(y[i].e[2 * j + 1]));
          xv[j] = f2_mul(xv[j], xs2);
          const F2 gj = f2_mul(dy, HOLD ? wreg[HOLD ? i : 0][j] : w[j]);
          c2 = f2_fma(gj, xv[j], c2);
          if constexpr (HOLD) {
            dw[i][j] = f2_fma(dy, xv[j], dw[i][j]);
            g[i][j] = gj;
            xh[i][j] = xv[j];
          }
        }
      }
    }
    float c0, c1;
    f2_get(c2, c0, c1);
    float c = c0 + c1;
    uint32_t late = (uint32_t)*ring.abort_flag;
    row_reduce<0, true>(c, late, buf, k & 1);
    if (tid == 0 && m + step * stages < a.M && !*ring.abort_flag) {
      fill(m + step * stages, k + stages);  // every thread holds its part of this row (row_reduce)
      ++issued;
    }
    c = late ? __int_as_float(0x7fc00000) : c / (float)N;
    const F2 nc = f2(-c * rstd, -c * rstd), rs2 = f2(rstd, rstd);
    T* dX = static_cast<T*>(a.dX) + m * a.lddx;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
      if (n < N) {
        F2 w[P], xv[P];
        if constexpr (!HOLD) {
          weights(i, w);
          x[i].get(a.x_dtype, xv);
        }
        Vec<T, VEC> o;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          F2 gj, xj;
          if constexpr (HOLD) {
            gj = g[i][j];
            xj = xh[i][j];
          } else {
            const F2 dy = f2(to_f(y[i].e[2 * j]), to_f(y[i].e[2 * j + 1]));
            xj = f2_mul(xv[j], xs2);
            dw[i][j] = f2_fma(dy, xj, dw[i][j]);
            gj = f2_mul(dy, w[j]);
          }
          F2 d = f2_fma(xj, nc, f2_mul(gj, rs2));
          if (dR) d = f2_add(d, f2(to_f(r[i].e[2 * j]), to_f(r[i].e[2 * j + 1])));
          float d0, d1;
          f2_get(d, d0, d1);
          from_f(&o.e[2 * j], d0);
          from_f(&o.e[2 * j + 1], d1);
        }
        *reinterpret_cast<Vec<T, VEC>*>(dX + n) = o;
      }
    }
  }
  if (a.part) {
    const bool lost = *ring.abort_flag;  // dw took in a row whose copy did not arrive
    float* p = a.part + (int64_t)blockIdx.x * a.N;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (i * threads + tid) * VEC;
      if (n < N)
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
          float4 v;
          f2_get(dw[i][j / 2], v.x, v.y);
          f2_get(dw[i][j / 2 + 1], v.z, v.w);
          if (lost) v.x = v.y = v.z = v.w = __int_as_float(0x7fc00000);
          *reinterpret_cast<float4*>(p + n + j) = v;
        }
    }
  }
  if (tid == 0 && *ring.abort_flag) ring.drain(issued);
}

// The same for rows of any alignment, element by element (as rows_ring_elems_kernel).  Bound by
// instructions: at an odd pitch 174 us at 8192 x 8192 (the kernel above, aligned, 86), 50 us at 16384 x 256
// (14).
template <typename T, bool X8, int THREADS, int V>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
    rmsnorm_bwd_elems_kernel(const BwdArgs a, int stages, uint32_t y_slot, uint32_t x_slot, uint64_t limit_ns) {
  using XT = typename std::conditional<X8, uint8_t, T>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float buf[128];
  __shared__ int abort_flag;
  const int tid = (int)threadIdx.x, N = (int)a.N;
  const int64_t first = blockIdx.x, step = gridDim.x;
  const T* dY = static_cast<const T*>(a.dY);
  const T* dR = static_cast<const T*>(a.dR);
  const XT* X = static_cast<const XT*>(a.X);
  const uint32_t y_bytes = (uint32_t)N * (uint32_t)sizeof(T), x_bytes = (uint32_t)N * (uint32_t)sizeof(XT);
  const Ring ring = make_ring(smem, stages, (dR ? 2 : 1) * y_slot + x_slot, limit_ns, &abort_flag);
  auto at_end = [&](int64_t m) { return m == 0 || m == a.M - 1; };
  auto fill = [&](int64_t m, int k) {
    const uint32_t bar = ring.bar(k), dst = ring.stage(k);
    if (at_end(m)) {
      ptx::mbar_arrive(bar);  // read from global memory when its turn comes
      return;
    }
    const T* y = dY + m * a.ldy;
    const XT* x = X + m * a.ldx;
    const T* r = dR ? dR + m * a.ldr : nullptr;
    ptx::mbar_arrive_expect_tx(bar, span_bytes(y, y_bytes) + span_bytes(x, x_bytes) + (dR ? span_bytes(r, y_bytes) : 0));
    span_load(dst, y, y_bytes, bar);
    span_load(dst + y_slot, x, x_bytes, bar);
    if (dR) span_load(dst + y_slot + x_slot, r, y_bytes, bar);
  };
  int issued = 0;
  if (tid == 0)
    for (int64_t m = first + (a.fault ? a.M : 0); m < a.M && issued < stages; m += step) fill(m, issued++);
  float w[V], dw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float f[1];
    load_weights<1>(a.W, a.w_dtype, false, i * THREADS + tid, N, f);
    w[i] = f[0];
    dw[i] = 0.0f;
  }
  // a row's two factors, loaded a row ahead
  float next_rstd = __ldg(a.rstd + first), next_scale = a.x_scale ? __ldg(a.x_scale + first) : 1.0f;
  int k = 0;
  for (int64_t m = first; m < a.M; m += step, ++k) {
    const float rstd = next_rstd, xs = next_scale * rstd;
    if (m + step < a.M) {
      next_rstd = __ldg(a.rstd + m + step);
      if (a.x_scale) next_scale = __ldg(a.x_scale + m + step);
    }
    ring.wait(k);
    const bool end = at_end(m);
    const uint8_t* st = smem + (uint32_t)(k % stages) * ring.stage_bytes;
    float g[V], xh[V], dr[V];
    float c = 0.0f;
    const int count = N - tid;  // element i is in the row if i * THREADS < count
    auto take = [&](const T* y, const XT* x, const T* r) {
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = i * THREADS < count ? to_f(y[i * THREADS]) : 0.0f;
      if constexpr (!X8) {
#pragma unroll
        for (int i = 0; i < V; ++i) xh[i] = i * THREADS < count ? to_f(x[i * THREADS]) : 0.0f;
      } else if (a.x_dtype == B2G_DTYPE_I8) {
#pragma unroll
        for (int i = 0; i < V; ++i)  // the byte, sign bit flipped, in the low byte of 2^23
          xh[i] = __uint_as_float(0x4b000000u | ((i * THREADS < count ? x[i * THREADS] : 0u) ^ 0x80u)) - 8388736.0f;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint8_t b = i * THREADS < count ? x[i * THREADS] : 0;
          xh[i] = float(*reinterpret_cast<const __nv_fp8_e4m3*>(&b));
        }
      }
      if (dR)
#pragma unroll
        for (int i = 0; i < V; ++i) dr[i] = i * THREADS < count ? to_f(r[i * THREADS]) : 0.0f;
    };
    const T* gy = dY + m * a.ldy;
    const XT* gx = X + m * a.ldx;
    const T* gr = dR ? dR + m * a.ldr : nullptr;
    if (end)
      take(gy + tid, gx + tid, gr + tid);
    else
      take(reinterpret_cast<const T*>(st + low4(gy)) + tid, reinterpret_cast<const XT*>(st + y_slot + low4(gx)) + tid,
           reinterpret_cast<const T*>(st + y_slot + x_slot + low4(gr)) + tid);
#pragma unroll
    for (int i = 0; i < V; ++i) {  // (a NaN scale must not reach elements past the row)
      xh[i] *= xs;
      if (i * THREADS >= count) xh[i] = 0.0f;
      dw[i] = fmaf(g[i], xh[i], dw[i]);
      g[i] *= w[i];
      c = fmaf(g[i], xh[i], c);
    }
    uint32_t late = (uint32_t)*ring.abort_flag;
    row_reduce<0, true>(c, late, buf, k & 1);
    if (tid == 0 && m + step * stages < a.M && !*ring.abort_flag) {
      fill(m + step * stages, k + stages);  // every thread holds its part of this row (row_reduce)
      ++issued;
    }
    c = late ? __int_as_float(0x7fc00000) : c / (float)N;
    T* dX = static_cast<T*>(a.dX) + m * a.lddx + tid;
    const float nc = -c * rstd;
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = fmaf(xh[i], nc, g[i] * rstd);
    if (dR)
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] += dr[i];
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * THREADS < count) from_f(dX + i * THREADS, g[i]);
  }
  const bool lost = *ring.abort_flag;
  if (a.part)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * THREADS + tid < N) a.part[(int64_t)blockIdx.x * N + i * THREADS + tid] = lost ? __int_as_float(0x7fc00000) : dw[i];
  if (tid == 0 && *ring.abort_flag) ring.drain(issued);
}

// dw[n] = the blocks' partial sums: a block sums COLS columns, 1024 / COLS rows at a time, and those sums
// of a column are added in a fixed order.
template <int COLS>
__global__ void __launch_bounds__(1024) dw_sum_kernel(const float* part, float* dw, int64_t N, int rows) {
  constexpr int R = 1024 / COLS;
  __shared__ float buf[R][COLS + 1];
  const int col = threadIdx.x % COLS, first = threadIdx.x / COLS;
  const int64_t n = (int64_t)blockIdx.x * COLS + col;
  float s = 0.0f;
  if (n < N)
#pragma unroll 8
    for (int b = first; b < rows; b += R) s += __ldcs(part + (int64_t)b * N + n);
  buf[first][col] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < COLS) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < R; i += 32) s += buf[i + lane][warp];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int64_t c = (int64_t)blockIdx.x * COLS + warp;
    if (lane == 0 && c < N) dw[c] = s;
  }
}

// Checks that every row operator shares: extents and leading dimensions.
int check_rows(int64_t M, int64_t N, std::initializer_list<int64_t> lds) {
  if (M < 0 || N < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  for (int64_t ld : lds)
    if (ld < std::max<int64_t>(N, 1))
      return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  return B2G_OK;
}

bool aligned(const void* p, int64_t pitch_bytes, int64_t rows, int to) {
  return ((uintptr_t)p % to) == 0 && (rows == 1 || pitch_bytes % to == 0);
}

// One launch of rows_to_q8_kernel: as many resident blocks as the GPU holds, at most one a row (set of rows).
template <typename T, bool NORM, int VEC, int V, int LANES, bool AHEAD = true>
int launch_rows(const NormArgs& a, int threads, int sms, cudaStream_t s) {
  if (LANES) threads = 128;
  const int per_block = LANES ? 128 / (LANES ? LANES : 1) : 1;
  const int64_t need = (a.M + per_block - 1) / per_block;
  const int64_t cap = (int64_t)sms * std::max(1, 1024 / threads);
  rows_to_q8_kernel<T, NORM, VEC, V, LANES, AHEAD><<<(unsigned)std::min(need, cap), threads, 0, s>>>(a);
  return launched("rows_to_q8_kernel");
}

// Raises a kernel's shared-memory limit once per device.
template <typename F>
int raise_smem(F fn, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingSmem);
    if (e == cudaSuccess) ready |= 1ull << dev;
  }
  return e == cudaSuccess ? (int)B2G_OK : cuda_fail(e, "cudaFuncSetAttribute(smem)");
}

// A launch of rows_ring_kernel, or false where its stages do not fit or a block would have too few rows (one
// with the norm, two without) for the ring to pay.  Against rows_to_q8_kernel (us, bf16, graph): norm with
// residual, 8192 rows of 8192 82 against 151, 16384 of 1024 27 against 51, 1000 of 4096 11.4 against
// 13.4, 296 of 8192 7.2 against 8.1, but 296 of 4096 4.8 against 3.9; quantize, 16384 of 8192 78
// against 99, 1000 of 4096 4.2 against 4.5, but 444 of 16384 8.6 against 6.6.
template <typename T, bool NORM, int V, int THREADS, int CTAS>
bool launch_ring(const NormArgs& a, int sms, cudaStream_t s, int* rc) {
  const uint32_t row_bytes = (uint32_t)(a.N * (int64_t)sizeof(T));
  const uint32_t stage = (a.R ? 2 : 1) * row_bytes;
  const int64_t nv = a.N * (int64_t)sizeof(T) / 16;
  const int threads = (int)((nv + V * 32 - 1) / (V * 32)) * 32;
  int ctas = 0, stages = 0;  // (blocks of fewer threads than THREADS leave registers for more of them)
  if (!ring_shape(stage, THREADS * CTAS / threads, &ctas, &stages) ||
      a.M < (int64_t)sms * ctas * (NORM ? 1 : 2))
    return false;
  auto fn = rows_ring_kernel<T, NORM, V, THREADS, CTAS>;
  static std::atomic<uint64_t> ready{0};
  *rc = raise_smem(fn, ready);
  if (*rc != B2G_OK) return true;
  fn<<<(unsigned)(sms * ctas), threads, ring_bytes(stages, stage), s>>>(
      a, stages, row_bytes, (uint64_t)launch_options().timeout_ns);
  *rc = launched("rows_ring_kernel");
  return true;
}

// A launch of rows_ring_elems_kernel, or false where its stages do not fit.
template <typename T, bool NORM, int THREADS, int V>
bool launch_ring_elems(const NormArgs& a, int sms, cudaStream_t s, int* rc) {
  const uint32_t slot = ((uint32_t)(a.N * (int64_t)sizeof(T)) + 30u) & ~15u, stage = (a.R ? 2 : 1) * slot;
  int ctas = V <= 16 ? 1024 / THREADS : 1, stages = 0;
  if (!ring_shape(stage, ctas, &ctas, &stages)) return false;
  auto fn = rows_ring_elems_kernel<T, NORM, THREADS, V>;
  static std::atomic<uint64_t> ready{0};
  *rc = raise_smem(fn, ready);
  if (*rc != B2G_OK) return true;
  fn<<<(unsigned)std::min<int64_t>(a.M, (int64_t)sms * ctas), THREADS, ring_bytes(stages, stage), s>>>(
      a, stages, slot, (uint64_t)launch_options().timeout_ns);
  *rc = launched("rows_ring_elems_kernel");
  return true;
}

// Vectors of 16 bytes where every address and pitch allows, else single elements (both sides: at
// rows_ring_elems_kernel).  Rows of up to 64
// vectors: two vectors a lane, several rows a warp; longer ones: a ring, or with few rows (latency
// counts then) one block a row with its loads in registers.
template <typename T, bool NORM>
int rows_of(const NormArgs& a, int sms, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int es = (int)sizeof(T);
  const bool vec = a.N % VEC == 0 && aligned(a.X, a.ldx * es, a.M, 16) &&
                   (!a.R || aligned(a.R, a.ldr * es, a.M, 16)) &&
                   (!a.H || aligned(a.H, a.ldh * es, a.M, 16)) && aligned(a.Q, a.ldq, a.M, VEC);
  if (vec) {
    const int64_t nv = a.N / VEC;
    if (nv <= 8) return launch_rows<T, NORM, VEC, 2, 4>(a, 0, sms, s);
    if (nv <= 16) return launch_rows<T, NORM, VEC, 2, 8>(a, 0, sms, s);
    if (nv <= 32) return launch_rows<T, NORM, VEC, 2, 16>(a, 0, sms, s);
    if (nv <= 64) return launch_rows<T, NORM, VEC, 2, 32>(a, 0, sms, s);
    int rc = B2G_OK;
    if (nv <= 128 ? launch_ring<T, NORM, 2, 64, 14>(a, sms, s, &rc)
        : nv <= 256 ? launch_ring<T, NORM, 2, 128, NORM ? 7 : 8>(a, sms, s, &rc)
        : nv <= 512 ? launch_ring<T, NORM, 4, 128, NORM ? 4 : 7>(a, sms, s, &rc)
        : nv <= 1024 ? launch_ring<T, NORM, 4, 256, NORM ? 2 : 4>(a, sms, s, &rc)
        : nv <= 2048 ? launch_ring<T, NORM, 4, 512, NORM ? 1 : 2>(a, sms, s, &rc)
        : nv <= 4096 ? launch_ring<T, NORM, 8, 512, 1>(a, sms, s, &rc)
                     : false)
      return rc;
    if (nv <= 256) return launch_rows<T, NORM, VEC, 1, 0>(a, (int)(nv + 31) / 32 * 32, sms, s);
    if (nv <= 512) return launch_rows<T, NORM, VEC, 2, 0>(a, (int)(nv + 63) / 64 * 32, sms, s);
    if (nv <= 1024) return launch_rows<T, NORM, VEC, 4, 0>(a, (int)(nv + 127) / 128 * 32, sms, s);
    if (nv <= 4096) return launch_rows<T, NORM, VEC, 4, 0, false>(a, (int)(nv + 127) / 128 * 32, sms, s);
  } else {
    if (a.N <= 32 * 8) return launch_rows<T, NORM, 1, 8, 32>(a, 0, sms, s);
    int rc = B2G_OK;
    if (a.N <= 128 * 8 ? launch_ring_elems<T, NORM, 128, 8>(a, sms, s, &rc)
        : a.N <= 128 * 16 ? launch_ring_elems<T, NORM, 128, 16>(a, sms, s, &rc)
        : a.N <= 256 * 16 ? launch_ring_elems<T, NORM, 256, 16>(a, sms, s, &rc)
        : a.N <= 512 * 16 ? launch_ring_elems<T, NORM, 512, 16>(a, sms, s, &rc)
        : a.N <= 512 * 32 ? launch_ring_elems<T, NORM, 512, 32>(a, sms, s, &rc)
                          : false)
      return rc;
  }
  const unsigned blocks = (unsigned)std::min<int64_t>(a.M, (int64_t)sms * 2);  // (what is resident at once)
  if (vec)
    long_rows_to_q8_kernel<T, NORM, VEC><<<blocks, kLongThreads, 0, s>>>(a);
  else
    long_rows_to_q8_kernel<T, NORM, 1><<<blocks, kLongThreads, 0, s>>>(a);
  return launched("long_rows_to_q8_kernel");
}

int rows_to_q8(const NormArgs& a, cudaStream_t s) {
  int dev = 0, sms = 0, cc = 0;
  const int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  switch (a.dtype) {
    case B2G_DTYPE_F16:
      return a.norm ? rows_of<__half, true>(a, sms, s) : rows_of<__half, false>(a, sms, s);
    case B2G_DTYPE_BF16:
      return a.norm ? rows_of<__nv_bfloat16, true>(a, sms, s) : rows_of<__nv_bfloat16, false>(a, sms, s);
    default:
      return a.norm ? rows_of<float, true>(a, sms, s) : rows_of<float, false>(a, sms, s);
  }
}

template <typename T>
int dequantize_to(const void* Q, const float* scale, T* X, int64_t M, int64_t N, int64_t ldq, int64_t ldx,
                  int q_dtype, float top, int sms, cudaStream_t s) {
  const uint8_t* q = static_cast<const uint8_t*>(Q);
  const bool vec = aligned(Q, ldq, M, 16) && aligned(X, ldx * (int64_t)sizeof(T), M, 16);
  const int64_t per_block = kRowThreads * (vec ? kPiece : kPieceElems);
  const int64_t need = vec ? (M * ((N + 15) / 16) + per_block - 1) / per_block : M * ((N + per_block - 1) / per_block);
  const int64_t blocks = std::min<int64_t>(need, (int64_t)sms * 1024);
  if (vec)
    dequantize_kernel<T, true><<<(unsigned)blocks, kRowThreads, 0, s>>>(q, scale, X, M, N, ldq, ldx, q_dtype, top);
  else
    dequantize_kernel<T, false><<<(unsigned)blocks, kRowThreads, 0, s>>>(q, scale, X, M, N, ldq, ldx, q_dtype, top);
  return launched("dequantize_kernel");
}

template <typename T, bool X8, int V, bool HOLD>
int launch_bwd_ring(const BwdArgs& a, int threads, unsigned blocks, int stages, cudaStream_t s) {
  const uint32_t yb = (uint32_t)(a.N * (int64_t)sizeof(T)), xb = X8 ? (uint32_t)a.N : yb;
  auto fn = rmsnorm_bwd_ring_kernel<T, X8, V, HOLD>;
  static std::atomic<uint64_t> ready{0};
  const int rc = raise_smem(fn, ready);
  if (rc != B2G_OK) return rc;
  fn<<<blocks, threads, ring_bytes(stages, (a.dR ? 2 : 1) * yb + xb), s>>>(
      a, stages, yb, xb, (uint64_t)launch_options().timeout_ns);
  return launched("rmsnorm_bwd_ring_kernel");
}

template <typename T, bool X8, int THREADS, int V>
int launch_bwd_elems(const BwdArgs& a, unsigned blocks, int stages, uint32_t y_slot, uint32_t x_slot,
                     cudaStream_t s) {
  auto fn = rmsnorm_bwd_elems_kernel<T, X8, THREADS, V>;
  static std::atomic<uint64_t> ready{0};
  const int rc = raise_smem(fn, ready);
  if (rc != B2G_OK) return rc;
  fn<<<blocks, THREADS, ring_bytes(stages, (a.dR ? 2 : 1) * y_slot + x_slot), s>>>(
      a, stages, y_slot, x_slot, (uint64_t)launch_options().timeout_ns);
  return launched("rmsnorm_bwd_elems_kernel");
}

template <typename T, bool X8>
int bwd_elems(const BwdArgs& a, int threads, unsigned blocks, int stages, uint32_t y_slot, uint32_t x_slot,
              cudaStream_t s) {
  if (threads == 128 && a.N <= 1024) return launch_bwd_elems<T, X8, 128, 8>(a, blocks, stages, y_slot, x_slot, s);
  if (threads == 128) return launch_bwd_elems<T, X8, 128, 16>(a, blocks, stages, y_slot, x_slot, s);
  if (threads == 256) return launch_bwd_elems<T, X8, 256, 16>(a, blocks, stages, y_slot, x_slot, s);
  return launch_bwd_elems<T, X8, 512, 16>(a, blocks, stages, y_slot, x_slot, s);
}

// Rows of whole 16-byte vectors whose stages fit shared memory run on the ring kernel; others of up to 8192
// elements element by element in registers; longer ones (and a checkpoint of another 16- or 32-bit
// type than dY's) in two passes.
template <typename T>
int bwd_of(BwdArgs a, bool x8, bool same, float* dw, int sms, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T), V = 16 / VEC;  // 16 elements a thread
  const int es = (int)sizeof(T), xe = x8 ? 1 : es;
  const int64_t nv = a.N / VEC;
  const bool hold = nv <= 512 * V;
  const int threads = (int)((nv + (hold ? V : 2 * V) * 32 - 1) / ((hold ? V : 2 * V) * 32)) * 32;
  int ctas = std::max(1, 512 / std::max(threads, 32)), stages = 0;
  const bool ring = (x8 || same) && a.N % VEC == 0 && a.N * xe % 16 == 0 && nv <= 1024 * V &&
                    aligned(a.dY, a.ldy * es, a.M, 16) && aligned(a.X, a.ldx * xe, a.M, 16) &&
                    aligned(a.dX, a.lddx * es, a.M, 16) && (!a.dR || aligned(a.dR, a.ldr * es, a.M, 16)) &&
                    ring_shape((uint32_t)(a.N * ((a.dR ? 2 : 1) * es + xe)), ctas, &ctas, &stages);
  const uint32_t y_slot = ((uint32_t)(a.N * es) + 30u) & ~15u, x_slot = ((uint32_t)(a.N * xe) + 30u) & ~15u;
  const int ethreads = a.N <= 2048 ? 128 : a.N <= 4096 ? 256 : 512;  // of the kernel for any alignment
  int ectas = 512 / ethreads, estages = 0;
  const bool elems = !ring && (x8 || same) && a.N >= 16 && a.N <= 8192 &&
                     ring_shape((a.dR ? 2 : 1) * y_slot + x_slot, ectas, &ectas, &estages);
  const unsigned blocks = ring || elems ? (unsigned)std::min<int64_t>(a.M, (int64_t)sms * (ring ? ctas : ectas))
                                        : (unsigned)std::min<int64_t>(a.M, (int64_t)sms * 2);
  Workspace ws(s);
  int rc = B2G_OK;
  if (dw) {
    rc = ws.alloc((size_t)blocks * (size_t)a.N * sizeof(float), "cudaMallocFromPoolAsync(dw partial sums)");
    if (rc != B2G_OK) return rc;
    a.part = static_cast<float*>(ws.get());
  }
  if (elems) {
    rc = x8 ? bwd_elems<T, true>(a, ethreads, blocks, estages, y_slot, x_slot, s)
            : bwd_elems<T, false>(a, ethreads, blocks, estages, y_slot, x_slot, s);
  } else if (!ring) {
    if (x8)
      rmsnorm_bwd_kernel<T, true><<<blocks, kLongThreads, 0, s>>>(a);
    else
      rmsnorm_bwd_kernel<T, false><<<blocks, kLongThreads, 0, s>>>(a);
    rc = launched("rmsnorm_bwd_kernel");
  } else if (hold) {
    rc = x8 ? launch_bwd_ring<T, true, V, true>(a, threads, blocks, stages, s)
            : launch_bwd_ring<T, false, V, true>(a, threads, blocks, stages, s);
  } else {
    rc = x8 ? launch_bwd_ring<T, true, 2 * V, false>(a, threads, blocks, stages, s)
            : launch_bwd_ring<T, false, 2 * V, false>(a, threads, blocks, stages, s);
  }
  if (rc != B2G_OK || !dw) return rc;
  // few columns: fewer a block, so that more blocks read the partial sums (16384 x 256 3 us faster with
  // 8; 8192 x 8192 2 us faster with 32)
  if (a.N < 4096)
    dw_sum_kernel<8><<<(unsigned)((a.N + 7) / 8), 1024, 0, s>>>(a.part, dw, a.N, (int)blocks);
  else
    dw_sum_kernel<32><<<(unsigned)((a.N + 31) / 32), 1024, 0, s>>>(a.part, dw, a.N, (int)blocks);
  return launched("dw_sum_kernel");
}

}  // namespace

int dequantize_rows(const void* Q, const float* scale, void* X, int64_t M, int64_t N, int64_t ldq,
                    int64_t ldx, int q_dtype, int dtype, cudaStream_t s) {
  int dev = 0, sms = 0, cc = 0;
  const int rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  switch (dtype) {
    case B2G_DTYPE_F16:
      return dequantize_to(Q, scale, static_cast<__half*>(X), M, N, ldq, ldx, q_dtype, 65504.0f, sms, s);
    case B2G_DTYPE_BF16:
      return dequantize_to(Q, scale, static_cast<__nv_bfloat16*>(X), M, N, ldq, ldx, q_dtype,
                           0x1.fep127f, sms, s);
    default:
      return dequantize_to(Q, scale, static_cast<float*>(X), M, N, ldq, ldx, q_dtype, 0x1.fffffep127f,
                           sms, s);
  }
}

}  // namespace b2g

// ==================================================================== C ABI
using namespace b2g;

extern "C" int b2g_quantize_q8(const void* X, void* Q, float* scale, int64_t M, int64_t N,
                               int64_t ldx, int64_t ldq, int dtype, int q_dtype, int pow2,
                               void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported input type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  int rc = check_rows(M, N, {ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (M == 0) return B2G_OK;
  if (N == 0) return fail(B2G_ERR_INVALID_ARG, "rows of no elements have no scale");
  if (!X || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, Q or scale is null");
  rc = check_alignment({{"X", X, dtype}, {"scale", scale, B2G_DTYPE_F32}});
  if (rc != B2G_OK) return rc;
  NormArgs a{};
  a.X = X;
  a.Q = Q;
  a.scale = scale;
  a.M = M; a.N = N; a.ldx = ldx; a.ldq = ldq;
  a.dtype = dtype; a.w_dtype = dtype; a.q_dtype = q_dtype;
  a.pow2 = pow2 != 0;
  a.fault = (launch_options().fault_flags & 1) != 0;
  return rows_to_q8(a, static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_dequantize_q8(const void* Q, const float* scale, void* X, int64_t M, int64_t N,
                                 int64_t ldq, int64_t ldx, int q_dtype, int dtype, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  int rc = check_rows(M, N, {ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (M == 0 || N == 0) return B2G_OK;
  if (!X || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, Q or scale is null");
  rc = check_alignment({{"X", X, dtype}, {"scale", scale, B2G_DTYPE_F32}});
  if (rc != B2G_OK) return rc;
  return dequantize_rows(Q, scale, X, M, N, ldq, ldx, q_dtype, dtype,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_rmsnorm_q8(const void* X, const void* R, const void* W, void* H, void* Q,
                              float* scale, float* rstd, int64_t M, int64_t N, int64_t ldx,
                              int64_t ldr, int64_t ldh, int64_t ldq, int dtype, int w_dtype,
                              int q_dtype, float eps, int pow2, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported input type code %d", dtype);
  if (!is_real(w_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported weight type code %d", w_dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  int rc = check_rows(M, N, {ldx, R ? ldr : ldx, H ? ldh : ldx, ldq});
  if (rc != B2G_OK) return rc;
  if (!(eps >= 0.0f)) return fail(B2G_ERR_INVALID_ARG, "eps is negative or NaN");
  if (M == 0) return B2G_OK;
  if (N == 0) return fail(B2G_ERR_INVALID_ARG, "rows of no elements have no norm");
  if (!X || !W || !Q || !scale) return fail(B2G_ERR_INVALID_ARG, "X, W, Q or scale is null");
  rc = check_alignment({{"X", X, dtype}, {"R", R, dtype}, {"W", W, w_dtype}, {"H", H, dtype},
                        {"scale", scale, B2G_DTYPE_F32}, {"rstd", rstd, B2G_DTYPE_F32}});
  if (rc != B2G_OK) return rc;
  if (H && ((H == X && ldh != ldx) || (H == R && ldh != ldr)))
    return fail(B2G_ERR_INVALID_ARG, "H in place needs the leading dimension of what it replaces");
  NormArgs a{};
  a.X = X; a.R = R; a.W = W; a.H = H; a.Q = Q;
  a.scale = scale; a.rstd = rstd;
  a.M = M; a.N = N; a.ldx = ldx; a.ldr = ldr; a.ldh = ldh; a.ldq = ldq;
  a.dtype = dtype; a.w_dtype = w_dtype; a.q_dtype = q_dtype;
  a.eps = eps;
  a.norm = true;
  a.pow2 = pow2 != 0;
  a.fault = (launch_options().fault_flags & 1) != 0;
  return rows_to_q8(a, static_cast<cudaStream_t>(stream));
}

extern "C" int b2g_rmsnorm_bwd_q8(const void* dY, const void* X, const float* x_scale, const void* W,
                                  const float* rstd, const void* dR, void* dX, float* dw, int64_t M,
                                  int64_t N, int64_t ldy, int64_t ldx, int64_t ldr, int64_t lddx,
                                  int dtype, int x_dtype, int w_dtype, void* stream) {
  clear_error();
  if (!is_real(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported gradient type code %d", dtype);
  if (!is_real(w_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported weight type code %d", w_dtype);
  if (!is_real(x_dtype) && !is_q8(x_dtype))
    return fail(B2G_ERR_INVALID_ARG, "unsupported checkpoint type code %d", x_dtype);
  int rc = check_rows(M, N, {ldy, ldx, dR ? ldr : ldy, lddx});
  if (rc != B2G_OK) return rc;
  if (N == 0) return B2G_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {  // no token: dw is a sum of nothing
    if (!dw) return B2G_OK;
    const cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)N * sizeof(float), s);
    return e == cudaSuccess ? B2G_OK : cuda_fail(e, "cudaMemsetAsync(dw)");
  }
  if (!dY || !X || !W || !rstd || !dX)
    return fail(B2G_ERR_INVALID_ARG, "dY, X, W, rstd or dX is null");
  if (is_q8(x_dtype) != (x_scale != nullptr))
    return fail(B2G_ERR_INVALID_ARG, "x_scale goes with an 8-bit checkpoint, and only with one");
  rc = check_alignment({{"dY", dY, dtype}, {"X", X, x_dtype}, {"x_scale", x_scale, B2G_DTYPE_F32},
                        {"W", W, w_dtype}, {"rstd", rstd, B2G_DTYPE_F32}, {"dR", dR, dtype}, {"dX", dX, dtype},
                        {"dw", dw, B2G_DTYPE_F32}});
  if (rc != B2G_OK) return rc;
  if ((dX == dY && lddx != ldy) || (dX == dR && lddx != ldr))
    return fail(B2G_ERR_INVALID_ARG, "dX in place needs the leading dimension of what it replaces");
  int dev = 0, sms = 0, cc = 0;
  rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  BwdArgs a{};
  a.dY = dY; a.X = X; a.W = W; a.dR = dR;
  a.x_scale = x_scale; a.rstd = rstd;
  a.dX = dX;
  a.M = M; a.N = N; a.ldy = ldy; a.ldx = ldx; a.ldr = ldr; a.lddx = lddx;
  a.dtype = dtype; a.x_dtype = x_dtype; a.w_dtype = w_dtype;
  a.fault = (launch_options().fault_flags & 1) != 0;
  const bool x8 = is_q8(x_dtype), same = x_dtype == dtype;
  switch (dtype) {
    case B2G_DTYPE_F16: return bwd_of<__half>(a, x8, same, dw, sms, s);
    case B2G_DTYPE_BF16: return bwd_of<__nv_bfloat16>(a, x8, same, dw, sms, s);
    default: return bwd_of<float>(a, x8, same, dw, sms, s);
  }
}
