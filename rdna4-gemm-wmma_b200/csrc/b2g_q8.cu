// Matrix products of the 8-bit linear layer: the scaled 8-bit product and the weight gradient from
// an 8-bit checkpoint.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

#include "../../include/b2g_gemm.h"
#include "errors.h"
#include "gemm_sm100.cuh"
#include "host.h"
#include "plan.h"
#include "q8.cuh"
#include "sched.h"
#include "skinny_sm100.cuh"

namespace b2g {

int q8_device_error(int clear, int* value) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (e == cudaSuccess && clear) {
    const int z = 0;
    e = cudaMemcpyToSymbol(g_device_error, &z, sizeof(int));
  }
  return (int)e;
}

namespace {

using namespace q8;

constexpr int kTile = 16;

// What the tensor-core kernels do not take (extents past 2^30, K = 0, option force_generic): 16 x 16 tiles
// of C through shared memory, one element per thread, 64-bit offsets.  int8 sums are int32; e4m3
// sums fp32, K in ascending order.  Bound by shared-memory loads: 1024^3 313 us (tensor cores 7.7).
template <bool I8>
__global__ void __launch_bounds__(kTile* kTile)
    gemm_q8_generic_kernel(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                           int64_t lda, int64_t ldb, int64_t ldc, const float* a_scale,
                           const float* b_scale, const float* bias, int c_dtype) {
  using T = typename std::conditional<I8, int, float>::type;
  __shared__ T as[kTile][kTile + 1], bs[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  const int dt = I8 ? B2G_DTYPE_I8 : B2G_DTYPE_E4M3;
  const int64_t tn = (N + kTile - 1) / kTile, tiles = tn * ((M + kTile - 1) / kTile);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / tn * kTile, n0 = t % tn * kTile;
    T acc = 0;
    for (int64_t k0 = 0; k0 < K; k0 += kTile) {
      as[ty][tx] = m0 + ty < M && k0 + tx < K ? (T)load_elem(A, (m0 + ty) * lda + k0 + tx, dt) : (T)0;
      bs[ty][tx] = n0 + ty < N && k0 + tx < K ? (T)load_elem(B, (n0 + ty) * ldb + k0 + tx, dt) : (T)0;
      __syncthreads();
      for (int k = 0; k < kTile; ++k) acc += as[ty][k] * bs[tx][k];
      __syncthreads();
    }
    const int64_t m = m0 + ty, n = n0 + tx;
    if (m < M && n < N) {
      float v = (float)acc;
      if (a_scale) v *= a_scale[m];
      if (b_scale) v *= b_scale[n];
      if (bias) v += bias[n];
      store_elem(C, m * ldc + n, c_dtype, v);
    }
  }
}

// The same for dW, tokens in ascending order: 1024^3 368 us (tensor cores 12.8).
__global__ void __launch_bounds__(kTile* kTile)
    wgrad_q8_generic_kernel(const void* dY, const void* Q, const float* scale, void* dW, int64_t M,
                            int64_t N, int64_t K, int64_t ldy, int64_t ldq, int64_t ldw, int dtype,
                            int q_dtype, bool accumulate, int c_dtype) {
  __shared__ float ys[kTile][kTile + 1], xs[kTile][kTile + 1];
  const int tx = threadIdx.x % kTile, ty = threadIdx.x / kTile;
  const int64_t tk = (K + kTile - 1) / kTile, tiles = tk * ((N + kTile - 1) / kTile);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t n0 = t / tk * kTile, k0 = t % tk * kTile;
    float acc = 0.0f;
    for (int64_t m0 = 0; m0 < M; m0 += kTile) {
      const bool in = m0 + ty < M;
      ys[ty][tx] = in && n0 + tx < N ? load_elem(dY, (m0 + ty) * ldy + n0 + tx, dtype) : 0.0f;
      float x = 0.0f;
      if (in && k0 + tx < K) {
        x = load_elem(Q, (m0 + ty) * ldq + k0 + tx, q_dtype) * scale[m0 + ty];
        x = clamp_to(x, largest(dtype));
        x = dtype == B2G_DTYPE_BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
      }
      xs[ty][tx] = x;
      __syncthreads();
      for (int m = 0; m < kTile; ++m) acc = fmaf(ys[m][ty], xs[m][tx], acc);
      __syncthreads();
    }
    const int64_t n = n0 + ty, k = k0 + tx;
    if (n < N && k < K) {
      if (accumulate) acc += static_cast<const float*>(dW)[n * ldw + k];
      store_elem(dW, n * ldw + k, c_dtype, acc);
    }
  }
}

unsigned tile_blocks(int64_t rows, int64_t cols, int sms) {
  const int64_t t = ((rows + kTile - 1) / kTile) * ((cols + kTile - 1) / kTile);
  return (unsigned)std::min<int64_t>(t, (int64_t)sms * 32);
}

// ------------------------------------------------------------------ few tokens
constexpr int kFewSteps = 4;  // 64-byte steps of K in a warp's turn

// D (16 x 8, 32-bit) += A (16 x 32 bytes) . B (32 bytes x 8): int8 into int32, or e4m3 into fp32.
template <bool I8>
__device__ __forceinline__ void mma_16x8x32(uint32_t (&d)[4], const uint32_t a0, const uint32_t a1,
                                            const uint32_t a2, const uint32_t a3, const uint32_t b0,
                                            const uint32_t b1) {
  if constexpr (I8)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Few tokens and few weights: latency counts, so the weights go from memory straight into the registers of
// warp-level MMAs, as their 16-row side (the tokens are its 8 columns), with no pipeline to fill and
// no tensor memory between.  The order of K inside a product does not matter, so a lane's fragments
// are whole 16-byte pieces: lane (g, t) of a warp takes bytes [16 t, 16 t + 16) of each 64-byte step
// of weight rows g and g + 8 and of token g, and feeds two MMAs from them.
//
// A block has 16 weight rows; its warps take K in turns of U steps and add their sums through shared
// memory, in warp order.  The next turn's weights are loaded before this turn's products.  Bound by
// latency: 1 token, 1024 x 4096 weights 2.7 us, 4096 x 2048 2.8 us (3.0 TB/s).
template <bool I8, int NT>
__global__ void __launch_bounds__(512, 1)
    gemm_q8_few_kernel(const int8_t* __restrict__ A, const int8_t* __restrict__ B, void* __restrict__ C,
                       int M, int64_t N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                       const float* __restrict__ a_scale, const float* __restrict__ b_scale,
                       const float* __restrict__ bias, int c_dtype) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  extern __shared__ uint32_t part[];  // [warps][16][NT * 8 + 1]
  constexpr int U = kFewSteps, PITCH = NT * 8 + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int8_t* w[2];  // rows past N read the last one; their sums are not stored
#pragma unroll
  for (int h = 0; h < 2; ++h) w[h] = B + min(n0 + h * 8 + g, N - 1) * ldb + t * 16;
  const int8_t* x[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) x[j] = A + (int64_t)min(j * 8 + g, M - 1) * lda + t * 16;
  uint32_t acc[NT][4] = {};
  uint4 cur[U][2], nxt[U][2];
  const int step = warps * U * 64;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  auto fetch = [&](int k, uint4 (&d)[U][2]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        d[u][h] = k + u * 64 + t * 16 < K ? __ldcs(reinterpret_cast<const uint4*>(w[h] + k + u * 64)) : zero;
  };
  int k = warp * U * 64;
  if (k < K) fetch(k, cur);
  for (; k < K; k += step) {
    if (k + step < K) fetch(k + step, nxt);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = k + u * 64 + t * 16 < K;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 b = in ? __ldg(reinterpret_cast<const uint4*>(x[j] + k + u * 64)) : zero;
        const uint4 p = cur[u][0], q = cur[u][1];
        mma_16x8x32<I8>(acc[j], p.x, q.x, p.y, q.y, b.x, b.y);
        mma_16x8x32<I8>(acc[j], p.z, q.z, p.w, q.w, b.z, b.w);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) cur[u][h] = nxt[u][h];
  }
  // rows g and g + 8 of the weights, tokens 2 t and 2 t + 1
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    uint32_t* p = part + (warp * 16 + g) * PITCH + j * 8 + 2 * t;
    p[0] = acc[j][0];
    p[1] = acc[j][1];
    p[8 * PITCH] = acc[j][2];
    p[8 * PITCH + 1] = acc[j][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * M; o += blockDim.x) {
    const int row = o % 16, m = o / 16;
    const int64_t n = n0 + row;
    if (n >= N) continue;
    const uint32_t* p = part + row * PITCH + m;
    float v;
    if constexpr (I8) {
      int s = 0;
      for (int i = 0; i < warps; ++i) s += (int)p[i * 16 * PITCH];
      v = (float)s;
    } else {
      v = 0.0f;
      for (int i = 0; i < warps; ++i) v += __uint_as_float(p[i * 16 * PITCH]);
    }
    if (a_scale) v *= a_scale[m];
    if (b_scale) v *= b_scale[n];
    if (bias) v += bias[n];
    store_elem(C, (int64_t)m * ldc + n, c_dtype, v);
  }
}

// A product whose weights are read once for all tokens.
struct FewArgs {
  const void *A, *B;
  void* C;
  int64_t M, N, K, lda, ldb, ldc;
  const float *a_scale, *b_scale, *bias;
  int c_dtype;
};

// gemm_q8_few_kernel takes up to 16 tokens where the weights are up to 12 Mi bytes (K a multiple of 16), as
// measured against gemm_q8_skinny_kernel (us a call, back to back in a graph, int8): 1 token, N x K =
// 1024 x 4096 2.7 against 5.4, 8192 x 1024 2.7 against 4.6, 4096 x 2048 2.8 against 5.4, 8192 x 8192
// 15.5 against 14.0; 16 tokens, 2048 x 2048 3.3 against 5.5, 4096 x 2048 3.3 against 5.6, 4096 x 4096
// 7.6 against 6.8.
bool is_few(const FewArgs& a) { return a.M <= 16 && a.K % 16 == 0 && a.N * a.K <= (int64_t)12 << 20; }

// Warps of a block: as many (4 to 16) as give the GPU about 16 an SM, each with a whole turn of K.
template <bool I8, int NT>
int launch_few(const FewArgs& a, int sms, cudaStream_t s) {
  const int64_t blocks = (a.N + 15) / 16;
  int warps = 4;
  while (warps < 16 && blocks * warps < (int64_t)sms * 16 && a.K >= (int64_t)warps * 2 * kFewSteps * 64) warps *= 2;
  const uint32_t smem = (uint32_t)(warps * 16 * (NT * 8 + 1)) * 4;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3((unsigned)warps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  if (launch_options().pdl) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, gemm_q8_few_kernel<I8, NT>, static_cast<const int8_t*>(a.A), static_cast<const int8_t*>(a.B), a.C,
      (int)a.M, a.N, (int)a.K, a.lda, a.ldb, a.ldc, a.a_scale, a.b_scale, a.bias, a.c_dtype);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_q8_few_kernel launch");
  count_launch();
  return B2G_OK;
}

template <bool I8>
int few_tokens(const FewArgs& a, int sms, cudaStream_t s) {
  return a.M <= 8 ? launch_few<I8, 1>(a, sms, s) : launch_few<I8, 2>(a, sms, s);
}

// ------------------------------------------------------------------ aligned copies
// Rows of `bytes` bytes from pitch `sp` to pitch `dp` (a multiple of 16), for operands whose base or
// pitch TMA cannot address: up to two matrices a launch.
struct RepackJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, bytes, sp, dp;
  uint32_t pieces;  // of a row
  int64_t items;    // rows * pieces (0: no matrix)
};

// A warp copies a piece of a row: each lane loads whole 4-byte words from the word that holds its first
// byte on, takes the next word from its neighbour and shifts the two together.  A row's piece may
// begin up to 3 bytes before the row and end as far behind it; in the rows from which that could reach out of
// the matrix (the first and the last, and more of them where pitches are below 3 bytes) words are put
// together from bytes where they would.  Memory-bound: all of a
// piece's loads are issued before the first is used.  It costs 30 us for 64 MiB of weights (4.4 TB/s, read
// and written), which a product of 16 tokens with them, 14.8 us, pays in every call.
constexpr int kRepackWords = 8;  // words a lane

__global__ void __launch_bounds__(256) repack_kernel(const RepackJob a, const RepackJob b) {
  constexpr int U = kRepackWords;
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < a.items + b.items; i += warps) {
    const RepackJob& g = i < a.items ? a : b;
    const uint64_t item = (uint64_t)(i < a.items ? i : i - a.items);
    const int64_t r = item >> 32 ? (int64_t)(item / g.pieces) : (int64_t)((uint32_t)item / g.pieces);
    const int64_t at0 = (int64_t)(item - (uint64_t)r * g.pieces) * (128 * U) + lane * 4;
    const uint8_t* row = g.src + r * g.sp;
    const uint32_t off = (uint32_t)(uintptr_t)row & 3u;  // (a piece is whole words: the same for all)
    const uint8_t* p = row - off + at0;
    const int64_t left = g.bytes + off - at0;  // bytes of the row from p on
    uint32_t w[U], last = 0;
    if (b2g_row_words_inside(r, g.rows, g.sp)) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        w[u] = u * 128 < left ? __ldcs(reinterpret_cast<const uint32_t*>(p + u * 128)) : 0u;
      if (lane == 31 && (U - 1) * 128 + 4 < left) last = __ldcs(reinterpret_cast<const uint32_t*>(p + (U - 1) * 128 + 4));
    } else {
      const uint8_t* const end = g.src + (g.rows - 1) * g.sp + g.bytes;
      auto word = [&](const uint8_t* q, int64_t here) -> uint32_t {
        if (here <= 0) return 0;
        if (q >= g.src && q + 4 <= end) return *reinterpret_cast<const uint32_t*>(q);
        uint32_t v = 0;
        for (int k = 0; k < 4; ++k)
          if (q + k >= g.src && q + k < end) v |= (uint32_t)q[k] << (8 * k);
        return v;
      };
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = word(p + u * 128, left - u * 128);
      if (lane == 31) last = word(p + (U - 1) * 128 + 4, left - (U - 1) * 128 - 4);
    }
    uint8_t* d = g.dst + r * g.dp + at0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t next = __shfl_down_sync(0xffffffffu, w[u], 1);
      const uint32_t wrap = u + 1 < U ? __shfl_sync(0xffffffffu, w[u + 1 < U ? u + 1 : u], 0) : last;
      if (lane == 31) next = wrap;
      if (at0 + u * 128 < g.bytes) *reinterpret_cast<uint32_t*>(d + u * 128) = __funnelshift_r(w[u], next, off * 8);
    }
  }
}

// An operand by its rows of bytes; `copy` where it needs a 16-byte aligned form.
struct Rows {
  const void* p;
  int64_t pitch, rows, bytes;
  bool copy() const { return (((uintptr_t)p | (uintptr_t)(rows > 1 ? pitch : 0)) & 15) != 0; }
  int64_t aligned_pitch() const { return (bytes + 15) / 16 * 16; }
  size_t copy_bytes() const { return copy() ? (size_t)(rows * aligned_pitch() + 255) / 256 * 256 : 0; }
};

// Turns the operands that need it into aligned copies in `mem` (the sum of their copy_bytes()).
int align_rows(Rows* a, Rows* b, void* mem, int sms, cudaStream_t s) {
  RepackJob jobs[2] = {};
  uint8_t* at = static_cast<uint8_t*>(mem);
  int n = 0;
  for (Rows* x : {a, b}) {
    if (!x || !x->copy()) continue;
    RepackJob& j = jobs[n++];
    j.src = static_cast<const uint8_t*>(x->p);
    j.dst = at;
    j.rows = x->rows;
    j.bytes = x->bytes;
    j.sp = x->pitch;
    j.dp = x->aligned_pitch();
    j.pieces = (uint32_t)((x->bytes + 128 * kRepackWords - 1) / (128 * kRepackWords));
    j.items = j.rows * j.pieces;
    at += x->copy_bytes();
    x->p = j.dst;
    x->pitch = j.dp;
  }
  if (n == 0) return B2G_OK;
  const int64_t blocks = std::min<int64_t>((jobs[0].items + jobs[1].items + 7) / 8, (int64_t)sms * 64);
  repack_kernel<<<(unsigned)blocks, 256, 0, s>>>(jobs[0], jobs[1]);
  return launched("repack_kernel");
}

// ------------------------------------------------------------------ tensor-core launch
// C (rows x cols, row-major) from a 128-byte-K-block product of gemm_tc_kernel.  Q_I8 / Q_FP8: A is
// rows x k, B cols x k, 8-bit, K contiguous.  Q_WGRAD: A is k x rows, B k x cols, 16-bit, rows and
// columns contiguous.  Bases and pitches of A and B are 16-byte aligned (align_rows).
//
// Tiles and splits are the plain product's.  Measured (graph): int8 8192^3 330 us (3.33 PFLOP/s, twice the
// 16-bit rate: bound by the tensor cores under the power limit), e4m3 380 to 409 us; weight gradient
// 4096 tokens x 8192 x 8192 with its conversion 370 us into bf16 (1.49 PFLOP/s), 490 to 550 us into fp32
// (kMaxTokens); an unaligned fp16 C of 3817 x 19967, K = 1888, 167 us against 131 us for an aligned one.
struct Product {
  int q;
  const void *A, *B;
  void* C;
  int64_t rows, cols, k;
  int64_t lda, ldb, ldc;  // elements
  int fmt;                // UMMA operand format of Q_WGRAD: 0 = fp16, 1 = bf16
  int c_type;             // 0 = fp32, 1 = fp16, 2 = bf16
  bool accumulate;
  const float *row_scale, *col_scale, *bias;
  int part_blocks;        // Q_WGRAD: K blocks that one accumulator may sum (0: any number)
  TileChoice tile;        // with part_blocks: the tile and the K splits of plan_parts()
  int splits;
};

using KernFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const GemmParams);

struct Variant {
  int cg, bn, threads;
  uint32_t smem;
  KernFn fn[4];  // Q_I8, Q_FP8, Q_WGRAD, Q_WGRAD_SUM (null for the 512-column tile)
};

template <int CG, int BN, int EW>
Variant make_variant() {
  using C = Cfg<CG, BN, kBM, EW>;
  KernFn sum = nullptr;
  if constexpr (BN <= 256) sum = gemm_tc_kernel<CG, BN, false, false, 2, kBM, EW, false, Q_WGRAD_SUM>;
  return {CG, BN, C::THREADS, C::SMEM_BYTES,
          {gemm_tc_kernel<CG, BN, true, false, 1, kBM, EW, false, Q_I8>,
           gemm_tc_kernel<CG, BN, true, false, 1, kBM, EW, false, Q_FP8>,
           gemm_tc_kernel<CG, BN, false, false, 2, kBM, EW, false, Q_WGRAD>, sum}};
}

const Variant* variants() {
  static const Variant v[4] = {make_variant<1, 128, 8>(), make_variant<1, 256, 8>(), make_variant<2, 256, 8>(),
                               make_variant<2, 512, 8>()};
  return v;
}
int variant_of(const TileChoice& tc) {
  return tc.cg == 1 ? (tc.bn == 128 ? 0 : 1) : (tc.bn == 256 ? 2 : 3);
}

// Clusters of `size` CTAs of a kernel resident at once on the current device, asked once per
// (device, variant, Q, size); also raises the kernel's shared-memory limit the first time.
int resident_clusters(int dev, int v, const Variant& var, int q, int size, int sms, int* out) {
  static std::mutex mu;
  static int known[64][4][4][9] = {};
  if (dev < 0 || dev >= 64) return fail(B2G_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
  std::lock_guard<std::mutex> lk(mu);
  int& n = known[dev][v][q - 1][size];
  if (n == 0) {
    KernFn fn = var.fn[q - 1];
    const cudaError_t e =
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)var.smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
    n = sms / size;
    if (size > 1) {
      cudaLaunchConfig_t qc = {};
      cudaLaunchAttribute qa[1];
      qa[0].id = cudaLaunchAttributeClusterDimension;
      qa[0].val.clusterDim.x = (unsigned)size;
      qa[0].val.clusterDim.y = qa[0].val.clusterDim.z = 1;
      qc.gridDim = dim3((unsigned)(size * (sms / size)), 1, 1);
      qc.blockDim = dim3((unsigned)var.threads, 1, 1);
      qc.dynamicSmemBytes = var.smem;
      qc.attrs = qa;
      qc.numAttrs = 1;
      int got = 0;
      if (cudaOccupancyMaxActiveClusters(&got, (void*)fn, &qc) == cudaSuccess && got > 0) {
        n = got;
      } else {
        cudaGetLastError();
        n = var.cg == size ? sms / size : -1;  // -1: never launched in clusters of this size
      }
    }
  }
  *out = n;
  return B2G_OK;
}

bool al16(uintptr_t x) { return (x & 15) == 0; }

int launch_product(const Product& g, int dev, int sms, cudaStream_t stream) {
  const LaunchOptions opt = launch_options();
  const int esz = g.q == Q_WGRAD ? 2 : 1, kb = kRowBytes / esz;
  const int64_t nmt = (g.rows + kBM - 1) / kBM, kit = (g.k + kb - 1) / kb;
  const TileChoice tc =
      g.part_blocks > 0 ? g.tile : choose_tiles(nmt, g.cols, kit, sms, opt.cta_group, opt.tile_n, 128);
  const int v = variant_of(tc);
  const Variant& var = variants()[v];
  const int cg = var.cg, bn = var.bn;

  // ---- tensor maps (dimensions of extent 1 get a stride that is never used)
  CUtensorMap tmA, tmB, tmC;
  const CUtensorMapDataType mt = esz == 1  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : g.fmt == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto up16 = [](int64_t bytes) -> cuuint64_t { return (cuuint64_t)((bytes + 15) & ~15LL); };
  auto pitch = [&](int64_t ld, int64_t n, int esize) -> cuuint64_t {
    return n == 1 ? up16(ld * esize) : (cuuint64_t)(ld * esize);
  };
  auto encode = [&](CUtensorMap* m, const void* base, int64_t inner, int64_t mid, int64_t outer,
                    int64_t ld, cuuint32_t b0, cuuint32_t b1, bool k_major, bool five) -> CUresult {
    // K-major: (k, 1, row[, 1, 1]); MN-major: (row, k, 1)
    if (k_major) {
      const cuuint64_t dims[5] = {(cuuint64_t)inner, 1, (cuuint64_t)outer, 1, 1};
      const cuuint64_t p = pitch(ld, outer, esz);
      const cuuint64_t st[4] = {up16(inner * esz), p, p, p};
      const cuuint32_t box[5] = {b0, 1, b1, 1, 1};
      return encode_cached(m, mt, five ? 5 : 3, const_cast<void*>(base), dims, st, box,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)mid, 1};
    const cuuint64_t st[2] = {pitch(ld, mid, esz), pitch(ld, mid, esz)};
    const cuuint32_t box[3] = {b0, b1, 1};
    return encode_cached(m, mt, 3, const_cast<void*>(base), dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  };
  const int bph = std::min(bn, 256) / cg;  // B columns of one N-half held by one CTA
  CUresult r;
  if (g.q == Q_WGRAD) {
    r = encode(&tmA, g.A, g.rows, g.k, 1, g.lda, 64, 64, false, false);
    if (r == CUDA_SUCCESS) r = encode(&tmB, g.B, g.cols, g.k, 1, g.ldb, 64, 64, false, false);
  } else {
    r = encode(&tmA, g.A, g.k, 1, g.rows, g.lda, 128, 128, true, true);
    if (r == CUDA_SUCCESS) r = encode(&tmB, g.B, g.k, 1, g.cols, g.ldb, 128, (cuuint32_t)bph, true, false);
  }
  if (r != CUDA_SUCCESS) return fail(B2G_ERR_CUDA, "tensor map of an 8-bit layer operand: CUresult %d", (int)r);
  const int csz = g.c_type == 0 ? 4 : 2;
  const bool direct = !al16((uintptr_t)g.C) || (g.rows > 1 && !al16((uintptr_t)(g.ldc * csz)));
  if (direct) {
    tmC = tmA;  // not used
  } else {
    const cuuint64_t dims[4] = {(cuuint64_t)g.cols, (cuuint64_t)g.rows, 1, 1};
    const cuuint64_t p0 = pitch(g.ldc, g.rows, csz), st[3] = {p0, p0, p0};
    const cuuint32_t box[4] = {32, 32, 1, 1};
    r = encode_cached(&tmC,
                      g.c_type == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                      : g.c_type == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      4, g.C, dims, st, box,
                      g.c_type == 0 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                      CU_TENSOR_MAP_L2_PROMOTION_NONE);
    if (r != CUDA_SUCCESS) return fail(B2G_ERR_CUDA, "tensor map of C: CUresult %d", (int)r);
  }

  GemmParams p{};
  p.i_size = (int)g.rows;
  p.b_size = p.a_size = 1;
  p.bi = kBM;
  p.bb = p.ba = 1;
  p.ti = (int)nmt;
  p.tb = 1;
  p.si = 32;
  p.sb = p.sa = 1;
  p.num_m_tiles = (int)nmt;
  p.num_pm_tiles = (int)((nmt + cg - 1) / cg);
  p.n_size = (int)g.cols;
  p.num_n_tiles = (int)((g.cols + bn - 1) / bn);
  p.k_blocks_per_j = (int)kit;
  p.k_iters = (int)kit;
  p.num_tiles = p.num_pm_tiles * p.num_n_tiles;
  p.raster_group = opt.raster_group > 0 ? opt.raster_group : (cg == 2 ? 8 : 16);
  p.accumulate = g.accumulate ? 1 : 0;
  p.alpha = 1.0f;
  p.c_type = g.c_type;
  p.bias = g.bias;
  p.ab_format = g.q == Q_WGRAD ? g.fmt : 0;  // e4m3 is format 0 of kind::f8f6f4
  p.timeout_ns = (unsigned long long)opt.timeout_ns;
  p.fault_flags = opt.fault_flags;
  p.row_scale = g.row_scale;
  p.col_scale = g.col_scale;
  // A TMA store whose row ends inside a 16-byte piece was seen to write zeros to the rest of that
  // piece (a 1-column bf16 C), so chunks at such an end are stored element by element.
  p.c_direct = direct || g.cols * csz % 16 != 0 ? g.C : nullptr;
  p.direct_all = direct ? 1 : 0;
  p.ldc = (long long)g.ldc;

  // ---- split-K, as the plain product plans it
  int group_cap = 0;
  int rc = resident_clusters(dev, v, var, g.q, cg, sms, &group_cap);
  if (rc != B2G_OK) return rc;
  const SplitChoice sc =
      g.part_blocks > 0 ? choose_splits(p.num_tiles, p.k_iters, group_cap, cg, g.splits, false)
                        : choose_splits(p.num_tiles, p.k_iters, group_cap, cg, opt.split_k, opt.tail_split);
  p.k_per_split = sc.k_per_split;
  p.k_splits = sc.k_splits;
  p.num_full = sc.num_full;
  p.k_parts = 1;
  const bool sum = g.part_blocks > 0 && p.k_splits == 1 && p.k_iters > g.part_blocks;
  const int q = sum ? (int)Q_WGRAD_SUM : g.q;
  if (sum) {
    p.k_per_part = part_length(p.k_iters, g.part_blocks);
    p.k_parts = (p.k_iters + p.k_per_part - 1) / p.k_per_part;
  }
  const int split_tiles = p.num_tiles - p.num_full;
  p.num_units = sum ? p.num_tiles * p.k_parts : p.num_full + split_tiles * p.k_splits;
  if (cg == 1 && p.k_splits > 1 && p.k_splits <= 8 && p.num_full == 0 && opt.cluster_fixup &&
      !opt.serial_fixup) {
    int nclu = 0;
    rc = resident_clusters(dev, v, var, g.q, p.k_splits, sms, &nclu);
    if (rc != B2G_OK) return rc;
    if (nclu > 0 && p.num_units <= nclu * p.k_splits) p.cluster_fixup = 1;
  }
  Workspace ws(stream);
  if (p.k_splits > 1 && !p.cluster_fixup) {
    // partial tiles, and one arrival counter per split tile and CTA (zeroed here: nothing of a
    // call outlives it, so captured graphs and streams share no counters)
    const size_t ctr = ((size_t)split_tiles * cg * sizeof(int) + 255) / 256 * 256;
    rc = ws.alloc(ctr + (size_t)split_tiles * p.k_splits * cg * kBM * bn * sizeof(float),
                  "cudaMallocFromPoolAsync(split-K workspace)");
    if (rc != B2G_OK) return rc;
    p.counters = static_cast<int*>(ws.get());
    p.ws = reinterpret_cast<float*>(static_cast<char*>(ws.get()) + ctr);
    const cudaError_t e = cudaMemsetAsync(p.counters, 0, ctr, stream);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(split-K counters)");
  }
  // parallel fix-up only when each CTA group holds at most one split unit: all of them then run at the
  // same time and wait for one another.  Without a cluster that co-schedules them the launch is
  // cooperative, so that no other stream's kernels can hold a part of the SMs it needs.
  const int groups = p.cluster_fixup ? p.num_units
                                     : std::max(1, std::min(group_cap, p.num_units / p.k_parts));
  p.fixup_parallel = p.k_splits > 1 && p.num_full % groups == 0 && p.num_units - p.num_full <= groups &&
                     !opt.serial_fixup;

  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3((unsigned)(groups * cg), 1, 1);
  cfg.blockDim = dim3((unsigned)(var.threads + 32 * (lead_warps(q) - 2)), 1, 1);
  cfg.dynamicSmemBytes = var.smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (cg == 2 || p.cluster_fixup) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = p.cluster_fixup ? (unsigned)p.k_splits : 2u;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (p.fixup_parallel && !p.cluster_fixup) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeCooperative;
    attr[cfg.numAttrs].val.cooperative = 1;
    ++cfg.numAttrs;
  } else if (opt.pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  if (sum) {  // raises the instance's shared-memory limit (its occupancy is the plain instance's)
    int n = 0;
    rc = resident_clusters(dev, v, var, q, cg, sms, &n);
    if (rc != B2G_OK) return rc;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, var.fn[q - 1], tmA, tmB, tmC, p);
  if (e != cudaSuccess) return cuda_fail(e, "8-bit layer tcgen05 kernel launch");
  count_launch();
  set_path(cg == 1 ? B2G_PATH_TC_1CTA : B2G_PATH_TC_2CTA);
  return B2G_OK;
}

// ------------------------------------------------------------------ decoding batches
// Up to this many tokens (the kernel's most columns) run on gemm_q8_skinny_kernel.  Measured against the
// tiles of larger batches (us a call, back to back in a graph, int8, N = K = 8192): 1 token 14.0
// against 23.6, 32 tokens 15.0 against 23.5, 64 tokens 16.3 against 23.6, 128 tokens 19.1 against
// 24.1; 10240 x 8192, 43 tokens 18.2 against 26.8; 28672 x 8192, 128 tokens 46.3 against 53.7;
// 1024 x 1024, 128 tokens 6.5 against 7.4.
constexpr int64_t kSkinnyTokens = 128;

template <bool I8, int NT>
int launch_skinny(const FewArgs& a, int sms, cudaStream_t s) {
  using C = SkinnyCfg<NT>;
  const LaunchOptions opt = launch_options();
  auto fn = gemm_q8_skinny_kernel<I8, NT>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM_BYTES);
    if (e == cudaSuccess) ready |= 1ull << dev;
  }
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
  CUtensorMap tmW, tmX;
  auto encode = [&](CUtensorMap* m, const void* base, int64_t rows, int64_t ld, cuuint32_t box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.K, 1, (cuuint64_t)rows};
    const cuuint64_t p = (cuuint64_t)(rows == 1 ? (ld + 15) / 16 * 16 : ld);
    const cuuint64_t st[2] = {(cuuint64_t)((a.K + 15) / 16 * 16), p};
    const cuuint32_t box[3] = {(cuuint32_t)kRowBytes, 1, box_rows};
    return encode_cached(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, st, box,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  };
  CUresult r = encode(&tmW, a.B, a.N, a.ldb, 128);
  if (r == CUDA_SUCCESS) r = encode(&tmX, a.A, a.M, a.lda, NT);
  if (r != CUDA_SUCCESS) return fail(B2G_ERR_CUDA, "tensor map of a decoding batch: CUresult %d", (int)r);
  SkinnyParams p{};
  p.M = (int)a.M;
  p.N = a.N;
  p.k_iters = (int)((a.K + kRowBytes - 1) / kRowBytes);
  const int tiles = (int)((a.N + 127) / 128);
  // splits: up to two CTAs an SM, each split keeping 8 K blocks (us, graph, by splits: 43 tokens x 10240 x
  // 8192, 1: 25.5, 2: 20.1, 3 (the rule): 18.3, 4: 25.2; 1 x 8192 x 8192, 2: 14.9, 4 (the rule): 14.3, 8:
  // 18.7; 32 x 28672 x 8192, 1 (the rule): 40.1, 2: 43.7; 128 x 4096 x 4096, 4 (the rule): 11.8, 8: 12.3)
  int splits = opt.split_k > 0 ? std::min(opt.split_k, 8)
                               : std::max(1, std::min({8, 2 * sms / tiles, p.k_iters / 8}));
  splits = std::min(splits, p.k_iters);
  p.k_per_split = (p.k_iters + splits - 1) / splits;
  p.splits = (p.k_iters + p.k_per_split - 1) / p.k_per_split;  // no empty split
  p.C = a.C;
  p.ldc = a.ldc;
  p.c_dtype = a.c_dtype;
  p.a_scale = a.a_scale;
  p.b_scale = a.b_scale;
  p.bias = a.bias;
  p.timeout_ns = (unsigned long long)opt.timeout_ns;
  p.fault_flags = opt.fault_flags;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3((unsigned)(tiles * p.splits), 1, 1);
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = s;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.numAttrs = 1;
  if (opt.pdl) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  e = cudaLaunchKernelEx(&cfg, fn, tmW, tmX, p);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_q8_skinny_kernel launch");
  count_launch();
  set_path(B2G_PATH_TC_1CTA);
  return B2G_OK;
}

template <bool I8>
int skinny(const FewArgs& a, int sms, cudaStream_t s) {
  if (a.M <= 32) return launch_skinny<I8, 32>(a, sms, s);
  if (a.M <= 64) return launch_skinny<I8, 64>(a, sms, s);
  return launch_skinny<I8, 128>(a, sms, s);
}

// Whether a product can run on the tensor-core kernel: an sm_100 device, and extents that its
// 32-bit coordinates hold.
bool tensor_ok(int cc, int64_t rows, int64_t cols, int64_t k) {
  const int64_t top = INT32_MAX / 2;
  return cc == 10 && !launch_options().force_generic && rows <= top && cols <= top && k > 0 && k <= top &&
         ((rows + 127) / 128) * ((cols + 127) / 128) <= INT32_MAX / 4;
}

int c_type_of(int c_dtype) { return c_dtype == B2G_DTYPE_F32 ? 0 : c_dtype == B2G_DTYPE_F16 ? 1 : 2; }

// Tokens that one tensor-core accumulator sums for an fp32 weight gradient.  The accumulator
// truncates, so its error grows with the number of terms.  Against 64 bits (2-norm, int8 rows of
// scales from 2^-6 to 2^1, fp32 library product 1.3e-7 to 5.8e-7): bf16 3.5e-7 over 512 tokens,
// 9.1e-7 over 1024, 1.8e-6 over 2048; fp16 6.2e-7, 1.2e-6, 2.4e-6.  Parts cost speed where they
// forbid the 512-column tile, whose operands need a quarter fewer L2 bytes.
constexpr int64_t kMaxTokens = 768;

}  // namespace
}  // namespace b2g

// ==================================================================== C ABI
using namespace b2g;

extern "C" int b2g_gemm_q8(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                           int64_t lda, int64_t ldb, int64_t ldc, int dtype, const float* a_scale,
                           const float* b_scale, const float* bias, int c_dtype, void* stream) {
  clear_error();
  if (!is_q8(dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", dtype);
  if (!is_real(c_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", c_dtype);
  if (M < 0 || N < 0 || K < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  if (lda < std::max<int64_t>(K, 1) || ldb < std::max<int64_t>(K, 1) || ldc < std::max<int64_t>(N, 1))
    return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  if (dtype == B2G_DTYPE_I8 && K > 131071)
    return fail(B2G_ERR_INVALID_ARG, "int8 sums of K = %lld products can overflow int32 (at most 131071)",
                (long long)K);
  if (M == 0 || N == 0) {
    set_path(B2G_PATH_EMPTY);
    return B2G_OK;
  }
  if (!C) return fail(B2G_ERR_INVALID_ARG, "C is null");
  if (K > 0 && (!A || !B)) return fail(B2G_ERR_INVALID_ARG, "A or B is null");
  if (M == 1) lda = std::max<int64_t>(K, 1), ldc = N;  // the pitch of a single row is not used: any is as good
  if (N == 1) ldb = std::max<int64_t>(K, 1);
  int rc = check_alignment({{"C", C, c_dtype}, {"a_scale", a_scale, B2G_DTYPE_F32},
                            {"b_scale", b_scale, B2G_DTYPE_F32}, {"bias", bias, B2G_DTYPE_F32}});
  if (rc != B2G_OK) return rc;
  int dev = 0, sms = 0, cc = 0;
  rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tensor_ok(cc, M, N, K)) {
    Workspace ws(s);
    Rows ra = {A, lda, M, K}, rb = {B, ldb, N, K};
    if (ra.copy() || rb.copy()) {
      rc = ws.alloc(ra.copy_bytes() + rb.copy_bytes(), "cudaMallocFromPoolAsync(aligned operands)");
      if (rc == B2G_OK) rc = align_rows(&ra, &rb, ws.get(), sms, s);
      if (rc != B2G_OK) return rc;
      A = ra.p; lda = ra.pitch;
      B = rb.p; ldb = rb.pitch;
    }
    const FewArgs f = {A, B, C, M, N, K, lda, ldb, ldc, a_scale, b_scale, bias, c_dtype};
    if (is_few(f)) {
      rc = dtype == B2G_DTYPE_I8 ? few_tokens<true>(f, sms, s) : few_tokens<false>(f, sms, s);
      if (rc == B2G_OK) set_path(B2G_PATH_FEW);
      return rc;
    }
    if (M <= kSkinnyTokens) return dtype == B2G_DTYPE_I8 ? skinny<true>(f, sms, s) : skinny<false>(f, sms, s);
    const Product g = {dtype == B2G_DTYPE_I8 ? Q_I8 : Q_FP8, A, B, C, M, N, K, lda, ldb, ldc, 0,
                       c_type_of(c_dtype), false, a_scale, b_scale, bias, 0, {}, 0};
    return launch_product(g, dev, sms, s);
  }
  const unsigned blocks = tile_blocks(M, N, sms);
  if (dtype == B2G_DTYPE_I8)
    gemm_q8_generic_kernel<true><<<blocks, kTile * kTile, 0, s>>>(A, B, C, M, N, K, lda, ldb, ldc, a_scale,
                                                                  b_scale, bias, c_dtype);
  else
    gemm_q8_generic_kernel<false><<<blocks, kTile * kTile, 0, s>>>(A, B, C, M, N, K, lda, ldb, ldc,
                                                                   a_scale, b_scale, bias, c_dtype);
  rc = launched("gemm_q8_generic_kernel");
  if (rc == B2G_OK) set_path(K == 0 ? B2G_PATH_ZERO : B2G_PATH_GENERIC);
  return rc;
}

extern "C" int b2g_wgrad_q8(const void* dY, const void* Q, const float* scale, void* dW, int64_t M,
                            int64_t N, int64_t K, int64_t ldy, int64_t ldq, int64_t ldw, int dtype,
                            int q_dtype, int accumulate, int c_dtype, void* stream) {
  clear_error();
  if (dtype != B2G_DTYPE_F16 && dtype != B2G_DTYPE_BF16)
    return fail(B2G_ERR_INVALID_ARG, "unsupported gradient type code %d", dtype);
  if (!is_q8(q_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported 8-bit type code %d", q_dtype);
  if (!is_real(c_dtype)) return fail(B2G_ERR_INVALID_ARG, "unsupported output type code %d", c_dtype);
  if (accumulate && c_dtype != B2G_DTYPE_F32)
    return fail(B2G_ERR_INVALID_ARG, "a 16-bit dW is overwritten, not added to");
  if (M < 0 || N < 0 || K < 0) return fail(B2G_ERR_INVALID_ARG, "negative dimension");
  if (ldy < std::max<int64_t>(N, 1) || ldq < std::max<int64_t>(K, 1) || ldw < std::max<int64_t>(K, 1))
    return fail(B2G_ERR_INVALID_ARG, "leading dimension smaller than the row length");
  if (N == 0 || K == 0) {
    set_path(B2G_PATH_EMPTY);
    return B2G_OK;
  }
  if (!dW) return fail(B2G_ERR_INVALID_ARG, "dW is null");
  if (M > 0 && (!dY || !Q || !scale)) return fail(B2G_ERR_INVALID_ARG, "dY, Q or scale is null");
  if (M == 1) ldy = N, ldq = K;  // as in b2g_gemm_q8
  if (N == 1) ldw = K;
  int rc = check_alignment({{"dY", dY, dtype}, {"scale", scale, B2G_DTYPE_F32}, {"dW", dW, c_dtype}});
  if (rc != B2G_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int dev = 0, sms = 0, cc = 0;
  rc = current_device(&dev, &sms, &cc);
  if (rc != B2G_OK) return rc;
  if (tensor_ok(cc, N, K, M)) {
    // the checkpoint's rows in dY's type, then the product of two token-major matrices
    Workspace ws(s);
    const int64_t ldx = (K + 7) / 8 * 8;
    const size_t x_bytes = ((size_t)(M * ldx) * 2 + 255) / 256 * 256;
    Rows ry = {dY, ldy * 2, M, N * 2};
    rc = ws.alloc(x_bytes + ry.copy_bytes(), "cudaMallocFromPoolAsync(dequantized checkpoint)");
    if (rc == B2G_OK) rc = dequantize_rows(Q, scale, ws.get(), M, K, ldq, ldx, q_dtype, dtype, s);
    if (rc == B2G_OK) rc = align_rows(&ry, nullptr, static_cast<char*>(ws.get()) + x_bytes, sms, s);
    if (rc != B2G_OK) return rc;
    const int64_t pitch = ry.pitch;
    const LaunchOptions opt = launch_options();
    const int part_blocks = c_dtype == B2G_DTYPE_F32 ? (int)(kMaxTokens / 64) : 0;
    int64_t per = M;
    PartPlan plan{};
    if (part_blocks) {
      const int64_t nmt = (N + kBM - 1) / kBM, kit = (M + 63) / 64;
      const TileChoice tc = choose_part_tiles(nmt, K, kit, sms, opt.cta_group, opt.tile_n, part_blocks);
      int cap = 0;
      rc = resident_clusters(dev, variant_of(tc), variants()[variant_of(tc)], Q_WGRAD, tc.cg, sms, &cap);
      if (rc != B2G_OK) return rc;
      plan = plan_parts(tc, nmt, K, kit, cap, opt.split_k, part_blocks);
      per = plan.blocks * 64;
    }
    for (int64_t m0 = 0; m0 < M && rc == B2G_OK; m0 += per) {
      const Product g = {Q_WGRAD, static_cast<const char*>(ry.p) + m0 * pitch,
                         static_cast<const char*>(ws.get()) + m0 * ldx * 2, dW, N, K,
                         std::min(per, M - m0), pitch / 2, ldx, ldw, dtype == B2G_DTYPE_F16 ? 0 : 1,
                         c_type_of(c_dtype), accumulate != 0 || m0 > 0, nullptr, nullptr, nullptr,
                         part_blocks, plan.tile, plan.splits};
      rc = launch_product(g, dev, sms, s);
    }
    return rc;
  }
  wgrad_q8_generic_kernel<<<tile_blocks(N, K, sms), kTile * kTile, 0, s>>>(
      dY, Q, scale, dW, M, N, K, ldy, ldq, ldw, dtype, q_dtype, accumulate != 0, c_dtype);
  rc = launched("wgrad_q8_generic_kernel");
  if (rc == B2G_OK) set_path(M == 0 ? B2G_PATH_ZERO : B2G_PATH_GENERIC);
  return rc;
}

extern "C" int b2g_call_q8(int call, const void* args) {
  clear_error();
  if (!args) return fail(B2G_ERR_INVALID_ARG, "args is null");
  const int64_t* a = static_cast<const int64_t*>(args);
  auto ptr = [a](int i) { return reinterpret_cast<void*>(static_cast<intptr_t>(a[i])); };
  auto vec = [ptr](int i) { return static_cast<float*>(ptr(i)); };
  auto num = [a](int i) { return static_cast<int>(a[i]); };
  switch (call) {
    case B2G_CALL_QUANTIZE_Q8:
      return b2g_quantize_q8(ptr(0), ptr(1), vec(2), a[3], a[4], a[5], a[6], num(7), num(8), num(9), ptr(10));
    case B2G_CALL_DEQUANTIZE_Q8:
      return b2g_dequantize_q8(ptr(0), vec(1), ptr(2), a[3], a[4], a[5], a[6], num(7), num(8), ptr(9));
    case B2G_CALL_RMSNORM_Q8: {
      double eps;
      std::memcpy(&eps, a + 16, sizeof(eps));
      return b2g_rmsnorm_q8(ptr(0), ptr(1), ptr(2), ptr(3), ptr(4), vec(5), vec(6), a[7], a[8], a[9], a[10],
                            a[11], a[12], num(13), num(14), num(15), (float)eps, num(17), ptr(18));
    }
    case B2G_CALL_GEMM_Q8:
      return b2g_gemm_q8(ptr(0), ptr(1), ptr(2), a[3], a[4], a[5], a[6], a[7], a[8], num(9), vec(10), vec(11),
                         vec(12), num(13), ptr(14));
    case B2G_CALL_WGRAD_Q8:
      return b2g_wgrad_q8(ptr(0), ptr(1), vec(2), ptr(3), a[4], a[5], a[6], a[7], a[8], a[9], num(10), num(11),
                          num(12), num(13), ptr(14));
    case B2G_CALL_RMSNORM_BWD_Q8:
      return b2g_rmsnorm_bwd_q8(ptr(0), ptr(1), vec(2), ptr(3), vec(4), ptr(5), ptr(6), vec(7), a[8], a[9],
                                a[10], a[11], a[12], a[13], num(14), num(15), num(16), ptr(17));
  }
  return fail(B2G_ERR_INVALID_ARG, "unknown call %d", call);
}
