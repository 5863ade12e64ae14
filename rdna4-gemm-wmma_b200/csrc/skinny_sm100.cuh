// Scaled 8-bit product of a decoding batch (up to 128 tokens), bound by the weights' bytes.
//
// C[m][n] = sum_k A[m][k] B[n][k] with few m.  The weights B are the 128-row side of the MMA and the tokens
// its NT columns, so that a CTA's accumulator is 128 x NT words, not 128 x 256: little to reduce
// when K is split, and little epilogue that nothing overlaps.  Pipeline as in gemm_tc_kernel (TMA
// into 128-byte-swizzled stages, one MMA-issuing thread, accumulator in TMEM), but at about 100 KB
// of shared memory, so that two CTAs share an SM: their loads keep about 190 KB an SM in flight,
// and a following launch can set up beside this one.
//
// K is split over the CTAs of a cluster.  Each leaves its accumulator in its (idle) stages, and CTA r of
// S sums columns r, r + S, ... of all of them through distributed shared memory in rank order.
//
// Measured (graph, int8): 1 x 8192 x 8192 14.0 us (4.8 TB/s), 43 x 10240 x 8192 18.2 us (4.6 TB/s), 32 x
// 28672 x 8192 40.1 us (5.9 TB/s), 128 x 28672 x 8192 46.3 us (5.2 TB/s).  A short product's fixed cost
// (set-up, first loads, epilogue: about 5 us) is what keeps it off the memory's rate.
//
// Nothing overlaps the epilogue, and a warp alone on its scheduler issues an instruction every few
// cycles: so eight warps share it, and loads from several CTAs are in flight together.
#pragma once
#include <type_traits>

#include "gemm_sm100.cuh"
#include "q8.cuh"

namespace b2g {

struct SkinnyParams {
  int M;                 // tokens (at most NT)
  int64_t N;             // weight rows
  int k_iters;           // 128-byte K blocks
  int k_per_split;
  int splits;            // CTAs of a cluster
  void* C;
  int64_t ldc;
  int c_dtype;
  const float *a_scale, *b_scale, *bias;
  unsigned long long timeout_ns;
  int fault_flags;       // test-only, as GemmParams::fault_flags
};

template <int NT>
struct SkinnyCfg {
  static constexpr uint32_t A_BYTES = 128 * kRowBytes;  // weights
  static constexpr uint32_t B_BYTES = NT * kRowBytes;   // tokens
  static constexpr int STAGES = (int)(100 * 1024 / (A_BYTES + B_BYTES));
  static constexpr uint32_t OFF_B = STAGES * A_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_B + STAGES * B_BYTES;
  static constexpr uint32_t OFF_MISC = OFF_BAR + (2 * STAGES + 2) * 8;
  static constexpr uint32_t OFF_SCALE = OFF_MISC + 16;
  static constexpr uint32_t SMEM_BYTES = OFF_SCALE + NT * 4 + 1024;
  static constexpr uint32_t TMEM_COLS = NT;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
};
static_assert(SkinnyCfg<32>::OFF_BAR >= 128 * 32 * 4 && SkinnyCfg<64>::OFF_BAR >= 128 * 64 * 4 &&
                  SkinnyCfg<128>::OFF_BAR >= 128 * 128 * 4,
              "an accumulator fits in the stages");

template <bool I8, int NT>
__global__ void __launch_bounds__(SkinnyCfg<NT>::THREADS, 2)
    gemm_q8_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                          const SkinnyParams p) {
  using C = SkinnyCfg<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint32_t base = ptx::smem_u32(smem_raw);
  const uint32_t pad = (1024u - (base & 1023u)) & 1023u;
  base += pad;
  uint8_t* smem = smem_raw + pad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto full_bar = [&](int s) { return base + C::OFF_BAR + 8u * s; };
  auto empty_bar = [&](int s) { return base + C::OFF_BAR + 8u * (C::STAGES + s); };
  const uint32_t tfull_bar = base + C::OFF_BAR + 8u * (2 * C::STAGES);
  const uint32_t done_bar = base + C::OFF_BAR + 8u * (2 * C::STAGES + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  float* scale = reinterpret_cast<float*>(smem + C::OFF_SCALE);
  int* err = &g_device_error;
  const unsigned long long lim = p.timeout_ns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(tfull_bar, 1);
    ptx::mbar_init(done_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    ptx::tma_prefetch_desc(&tmW);
    ptx::tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(base + C::OFF_MISC, C::TMEM_COLS);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::OFF_MISC);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();

  const int split = (int)(blockIdx.x % p.splits);
  const int64_t n0 = (int64_t)(blockIdx.x / p.splits) * 128;
  const int kb_lo = split * p.k_per_split, kb_hi = min(p.k_iters, kb_lo + p.k_per_split);

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int kb = kb_lo; kb < kb_hi; ++kb, ++it) {
        const int s = it % C::STAGES;
        if (!ptx::mbar_wait(empty_bar(s), ((uint32_t)(it / C::STAGES) & 1u) ^ 1u, abort_flag, err, ERR_WAIT_EMPTY, lim))
          break;
        ptx::mbar_arrive_expect_tx(full_bar(s), C::A_BYTES + C::B_BYTES);
        if (p.fault_flags & 1) continue;
        ptx::tma_load_3d<1>(base + s * C::A_BYTES, &tmW, full_bar(s), kb * kRowBytes, 0, (int)n0);
        ptx::tma_load_3d<1>(base + C::OFF_B + s * C::B_BYTES, &tmX, full_bar(s), kb * kRowBytes, 0, 0);
      }
      // every load must land before the CTA's shared memory goes away
      if (!(p.fault_flags & 1))
        for (int i = max(0, it - C::STAGES); i < it; ++i)
          ptx::mbar_wait_drain(full_bar(i % C::STAGES), (uint32_t)(i / C::STAGES) & 1u, err, ERR_WAIT_DRAIN, lim);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = I8 ? make_idesc_i8(128, NT) : make_idesc(128, NT, false, 0);
      bool ok = true;
      int it = 0;
      for (int kb = kb_lo; kb < kb_hi && ok; ++kb, ++it) {
        const int s = it % C::STAGES;
        ok = ptx::mbar_wait(full_bar(s), (uint32_t)(it / C::STAGES) & 1u, abort_flag, err, ERR_WAIT_FULL, lim);
        if (!ok) break;
        ptx::tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t ad = ptx::smem_desc_sw128(base + s * C::A_BYTES + 32u * k, 16u, 1024u);
          const uint64_t bd = ptx::smem_desc_sw128(base + C::OFF_B + s * C::B_BYTES + 32u * k, 16u, 1024u);
          if constexpr (I8)
            ptx::umma_i8<1>(tmem, ad, bd, idesc, (it | k) != 0 ? 1u : 0u);
          else
            ptx::umma<1, 1>(tmem, ad, bd, idesc, (it | k) != 0 ? 1u : 0u);
        }
        ptx::umma_commit<1>(empty_bar(s), 0);
      }
      if (ok) ptx::umma_commit<1>(tfull_bar, 0);
      ptx::umma_commit<1>(done_bar, 0);
      ptx::mbar_wait_drain(done_bar, 0u, err, ERR_WAIT_DRAIN, lim);
    }
  }

  // ------------------------------------------------------------ epilogue: warps 2..9
  const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter; which of its two warps
  const int row = 32 * q + lane;
  const bool mine = warp >= 2 && n0 + row < p.N;
  float ws = 1.0f, bias = 0.0f;
  if (warp >= 2) {
    // the row's (output channel's) scale and bias, and the tokens' scales, while the MMAs run
    if (mine && p.b_scale) ws = __ldg(p.b_scale + n0 + row);
    if (mine && p.bias) bias = __ldg(p.bias + n0 + row);
    for (int j = (int)threadIdx.x - 64; j < NT; j += 32 * C::EPI_WARPS) scale[j] = p.a_scale && j < p.M ? __ldg(p.a_scale + j) : 1.0f;
    ptx::named_barrier_sync(1, 32 * C::EPI_WARPS);
  }
  // COUNT results, of tokens m, m + step, ...: everything is computed before the first store (a store
  // could alias the scales as far as the compiler knows, and would wait for each of them in turn)
  auto store = [&](auto count, int m, int step, const uint32_t* acc) {
    constexpr int COUNT = decltype(count)::value;
    float v[COUNT];
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int at = m + j * step;
      const float x = I8 ? (float)(int)acc[j] : __uint_as_float(acc[j]);
      v[j] = x * (at < NT ? scale[at] : 0.0f) * ws + bias;
    }
    const int64_t first = (int64_t)m * p.ldc + n0 + row, pitch = (int64_t)step * p.ldc;
    auto out = [&](auto* c, auto put) {
      c += first;
#pragma unroll
      for (int j = 0; j < COUNT; ++j)
        if (mine && m + j * step < p.M) put(c + j * pitch, v[j]);
    };
    if (p.c_dtype == B2G_DTYPE_BF16)
      out(static_cast<__nv_bfloat16*>(p.C), [](__nv_bfloat16* c, float x) { *c = __float2bfloat16_rn(x); });
    else if (p.c_dtype == B2G_DTYPE_F16)
      out(static_cast<__half*>(p.C), [](__half* c, float x) { *c = __float2half_rn(x); });
    else
      out(static_cast<float*>(p.C), [](float* c, float x) { *c = x; });
  };
  if (warp >= 2) {
    const bool got = ptx::mbar_wait(tfull_bar, 0u, abort_flag, err, ERR_WAIT_TFULL, lim);
    if (__all_sync(0xffffffffu, got)) {
      ptx::tc_fence_after();
      const uint32_t t = tmem + ((uint32_t)(32 * q) << 16);
#pragma unroll 1
      for (int c = 16 * half; c < NT; c += 32) {
        if (c >= p.M) break;
        uint32_t v[16];
        ptx::tmem_ld_32x32b_x16(t + c, v);
        ptx::tmem_ld_wait();
        if (p.splits == 1) {
          store(std::integral_constant<int, 16>(), c, 1, v);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) ptx::st_shared_b32(base + 4u * (uint32_t)((c + j) * 128 + row), v[j]);
        }
      }
    }
  }
  if (p.splits > 1) {
    __syncwarp();
    ptx::cluster_sync();  // every CTA's accumulator is in its shared memory
    if (warp >= 2) {
      // eight tokens of a CTA's share, four of each half, and up to four CTAs' loads at a time
#pragma unroll 1
      for (int m = split + 4 * half * p.splits; m < p.M; m += 8 * p.splits) {
        const uint32_t at = base + 4u * (uint32_t)(m * 128 + row);
        uint32_t s[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
        for (int r0 = 0; r0 < p.splits; r0 += 4) {
          uint32_t x[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (r0 + r < p.splits && m + j * p.splits < p.M)
                x[r][j] = ptx::ld_shared_cluster_b32(ptx::mapa(at, (uint32_t)(r0 + r)) + 512u * (uint32_t)(j * p.splits));
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (r0 + r < p.splits && m + j * p.splits < p.M)
                s[j] = __float_as_uint(acc_add<I8>(__uint_as_float(s[j]), __uint_as_float(x[r][j])));
        }
        store(std::integral_constant<int, 4>(), m, p.splits, s);
      }
    }
    __syncwarp();
    ptx::cluster_sync();  // no CTA leaves while another reads its accumulator
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    ptx::tmem_dealloc<1>(tmem, C::TMEM_COLS);
  }
}

}  // namespace b2g
