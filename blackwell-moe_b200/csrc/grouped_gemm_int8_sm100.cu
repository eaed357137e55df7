// Grouped products in 8-bit integers on the 5th-generation tensor cores, a scale for each row and for each channel.
//
//   PLAIN  : out[m,n] = (sum_k a[m,k] * w[e,k,n]) * row_scale[m] * channel_scale[e,n]
//   SWIGLU : h[m,n]   = silu(gate) * up, gate and up being two such products of the same rows
//
// where e is the expert whose segment offsets[e] .. offsets[e+1] holds row m.  The sums are formed in 32-bit integers and
// are exact whatever their order (|a|, |w| <= 128 and K < 2^17); scales, SwiGLU and the one rounding to the output type
// happen in fp32 in the epilogue.
//
// Structure per CTA (320 threads, one CTA per SM, persistent): warp 0 TMA producer, warp 1 tcgen05.mma issuer
// (kind::i8, M=128 N=256 K=32, int32 accumulators in tensor memory, two 256-column buffers), warps 2..9 epilogue, two per
// tensor-memory lane quarter.  A tile is 128 rows of one expert x 256 accumulator columns (SWIGLU: 128 gate + 128 up
// columns); activations are read K-major, weights in the caller's [E, K, N] layout (N contiguous).  Tiles are ordered by
// expert, then column block, then row block, so that an expert's rows stay in L2 while its weights stream through once.
// Every wait is bounded as in the other GEMM kernels of this library.
#include "sm100_gemm.cuh"

namespace bwmoe {
namespace {
using namespace sm100;

// D = int32, A = B = signed 8-bit, A K-major, B MN-major, N = 256, M = 128
constexpr uint32_t IDESC_I8 = (2u << 4) | (1u << 7) | (1u << 10) | (0u << 15) | (1u << 16) | ((uint32_t)(BN >> 3) << 17) |
                              ((uint32_t)(BM >> 4) << 24);
constexpr int kMaxGroups = 256;
constexpr int EPI_WARPS = 8;
constexpr int I8_THREADS = 64 + 32 * EPI_WARPS;

__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct I8Params {
  const int32_t* offsets;   // [E+1]; nullptr: one segment with every row
  const float* row_scale;   // [M]
  const float* scale0;      // [E, N] (SWIGLU: gate)
  const float* scale1;      // [E, N] up
  void* out;                // [M, N]
  int32_t* status;
  int E, M, Kdim, N, n_tiles;
};

// Segment e, clamped to the rows there are: offsets are data from outside the kernel.
__device__ __forceinline__ void segment(const I8Params& p, int e, int& r0, int& r1) {
  r0 = p.offsets != nullptr ? min(max(p.offsets[e], 0), p.M) : 0;
  r1 = p.offsets != nullptr ? min(max(p.offsets[e + 1], r0), p.M) : p.M;
}

// s_first[0 .. E] and s_end[0 .. E-1]: the segments; s_cum[0 .. E]: tiles before each.  All threads of the block.
template <int THREADS>
__device__ __forceinline__ void tile_table(const I8Params& p, int tile_rows, int tiles_per_row_block, int* s_first, int* s_end,
                                           int* s_cum) {
  for (int e = threadIdx.x; e < kMaxGroups; e += THREADS) {
    int r0 = 0, r1 = 0;
    if (e < p.E) segment(p, e, r0, r1);
    s_first[e] = r0, s_end[e] = r1;
    s_cum[e + 1] = ((r1 - r0 + tile_rows - 1) / tile_rows) * tiles_per_row_block;
  }
  __syncthreads();
  if (threadIdx.x < 32) {       // inclusive scan: 8 values per lane, then a shuffle scan of the lanes' totals
    const int lane = threadIdx.x;
    int v[8], run = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      run += s_cum[1 + lane * 8 + j];
      v[j] = run;
    }
    int incl = run;
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s_cum[1 + lane * 8 + j] = incl - run + v[j];
    if (lane == 0) s_cum[0] = 0;
  }
}

// tile index -> (expert, first row, end of its segment, column block); every role walks the same rising sequence
struct I8Cursor {
  const int *first, *end, *cum;
  int E, tile_rows, e;
  __device__ bool locate(int tile, int& row0, int& row_end, int& n_idx) {
    while (e < E && tile >= cum[e + 1]) ++e;
    if (e >= E) return false;
    const int m_tiles = (end[e] - first[e] + tile_rows - 1) / tile_rows;
    const int within = tile - cum[e];
    n_idx = within / m_tiles;
    row0 = first[e] + (within - n_idx * m_tiles) * tile_rows;
    row_end = end[e];
    return true;
  }
};

// ---- output types: how many make 16 bytes, and the packing ----
template <class T> struct Out;
template <> struct Out<float> {
  static constexpr int kPer16 = 4;
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ float one(float v) { return v; }
};
template <> struct Out<__half> {
  static constexpr int kPer16 = 8;
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(two(v[0], v[1]), two(v[2], v[3]), two(v[4], v[5]), two(v[6], v[7]));
  }
  static __device__ __forceinline__ __half one(float v) { return __float2half_rn(v); }
};
template <> struct Out<__nv_bfloat16> {
  static constexpr int kPer16 = 8;
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(two(v[0], v[1]), two(v[2], v[3]), two(v[4], v[5]), two(v[6], v[7]));
  }
  static __device__ __forceinline__ __nv_bfloat16 one(float v) { return __float2bfloat16_rn(v); }
};
// fp32 results get the accurate exponential and division, 16-bit ones the fast forms (2^-21 against a rounding of 2^-9)
template <class T> __device__ __forceinline__ float swiglu(float g, float u) {
  if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g)) * u;
  else                          return silu_f(g) * u;
}

// Rows behind the last segment belong to no expert: zeros.  `part` of `parts` threads.
template <class T>
__device__ __forceinline__ void zero_tail_rows(const I8Params& p, int part, int parts) {
  if (p.offsets == nullptr) return;
  const int first = min(max(p.offsets[p.E], 0), p.M);
  const size_t n = (size_t)(p.M - first) * p.N / Out<T>::kPer16;
  uint4* at = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (size_t)first * p.N);
  for (size_t i = part; i < n; i += parts) at[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <bool SWIGLU, class T>
__global__ void __launch_bounds__(I8_THREADS, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b0,
                 const __grid_constant__ CUtensorMap map_b1, const I8Params p) {
  chain_wait();
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_first[kMaxGroups], s_end[kMaxGroups], s_cum[kMaxGroups + 1];
  __shared__ __align__(16) float s_scale[EPI_WARPS][BN / 2];      // each epilogue warp's channel scales of its tile
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const uint32_t tiles_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = tiles_base + STAGES * STAGE_BYTES;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * STAGES;
  const uint32_t bar_tfull = bars + 16 * STAGES, bar_tempty = bar_tfull + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < STAGES; ++s) mbar_init(bar_full + 8 * s, 1), mbar_init(bar_empty + 8 * s, 1);
    for (int b = 0; b < 2; ++b) mbar_init(bar_tfull + 8 * b, 1), mbar_init(bar_tempty + 8 * b, EPI_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tile_table<I8_THREADS>(p, BM, p.n_tiles, s_first, s_end, s_cum);
  if (warp == 1) tmem_alloc(smem_u32(&s_tmem_base), TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  const int total_tiles = s_cum[p.E], k_blocks = (p.Kdim + BK - 1) / BK;
  I8Cursor cur{s_first, s_end, s_cum, p.E, BM, 0};

  if (warp == 0) {
    // ===================== TMA producer =====================
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
        int row0, row_end, n_idx;
        if (!cur.locate(tile, row0, row_end, n_idx)) break;
        const int n0 = n_idx * (SWIGLU ? BN_HALF : BN);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status))) break;
          const uint32_t sa = tiles_base + stage * STAGE_BYTES, full = bar_full + 8 * stage;
          mbar_expect_tx(full, STAGE_BYTES);
          tma_load_2d(sa, &map_a, full, kb * BK, row0);
          tma_load_3d(sa + A_BYTES, &map_b0, full, n0, kb * BK, cur.e);
          if (SWIGLU) tma_load_3d(sa + A_BYTES + B_HALF_BYTES, &map_b1, full, n0, kb * BK, cur.e);
          else        tma_load_3d(sa + A_BYTES + B_HALF_BYTES, &map_b0, full, n0 + BN_HALF, kb * BK, cur.e);
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, local = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x, ++local) {
        const uint32_t buf = local & 1u, use = local >> 1;
        if (!(ok = mbar_wait(bar_tempty + 8 * buf, (use & 1u) ^ 1u, abort_flag, p.status))) break;
        tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!(ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status))) break;
          tc_fence_after();
          const uint32_t sa = tiles_base + stage * STAGE_BYTES;
          const uint64_t da = desc_kmajor(sa), db = desc_nmajor(sa + A_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)     // A: +32 bytes along K inside the swizzle atom; B: +32 K rows = 4096 bytes
            mma_i8(tmem_base + buf * BN, da + (uint64_t)(k * 2), db + (uint64_t)(k * 256), IDESC_I8, (kb | k) ? 1u : 0u);
          mma_commit(bar_empty + 8 * stage);
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
        if (ok) mma_commit(bar_tfull + 8 * buf);
      }
    }
  } else {
    // ===================== epilogue (warps 2..9) =====================
    const int quarter = warp & 3, half = (warp - 2) >> 2;      // tensor-memory lanes this warp may read; half of the columns
    float* my_scale = s_scale[warp - 2];
    uint32_t local = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x, ++local) {
      int row0, row_end, n_idx;
      if (!cur.locate(tile, row0, row_end, n_idx)) break;
      const uint32_t buf = local & 1u, use = local >> 1;
      const int row = row0 + quarter * 32 + lane;
      const bool row_ok = row < row_end;
      const float rs = row_ok ? p.row_scale[row] : 0.f;
      // channel scales of this warp's columns (SWIGLU: 64 of the gate, then 64 of the up product), zero past N
      const int n0 = n_idx * (SWIGLU ? BN_HALF : BN) + half * (SWIGLU ? BN_HALF / 2 : BN_HALF);
      {
        const float* s = (SWIGLU && lane >= 16 ? p.scale1 : p.scale0) + (size_t)cur.e * p.N;
        const int n = n0 + (SWIGLU ? (lane & 15) : lane) * 4;
        __syncwarp();                            // the tile before has read its scales
        // (N is a multiple of 16, scales of 16-byte alignment: four at a time)
        *reinterpret_cast<float4*>(my_scale + 4 * lane) =
            n < p.N ? *reinterpret_cast<const float4*>(s + n) : make_float4(0.f, 0.f, 0.f, 0.f);
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * buf, use & 1u, abort_flag, p.status));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * BN;
      const unsigned ok_rows = __ballot_sync(0xffffffffu, row_ok);
      unsigned long long row_ptr[8];
      group8_row_pointers(static_cast<T*>(p.out) + (size_t)row * p.N, lane, row_ptr);
      constexpr int PER = Out<T>::kPer16, COLS = SWIGLU ? BN_HALF / 2 : BN_HALF;       // columns of this warp
      // eight 16-byte pieces per lane at a time, exchanged so that a store writes 128 contiguous bytes of four rows
#pragma unroll 1
      for (int c0 = 0; c0 < COLS; c0 += 8 * PER) {
        uint4 v[8];
#pragma unroll
        for (int part = 0; part < 8 * PER / 32; ++part) {
          const int c = c0 + part * 32;
          uint32_t a[32], u[SWIGLU ? 32 : 1];
          tmem_ld32(t_row + half * COLS + c, a);
          if constexpr (SWIGLU) tmem_ld32(t_row + BN_HALF + half * COLS + c, u);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32 / PER; ++j) {
            float f[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int x = j * PER + i;
              f[i] = __int2float_rn((int)a[x]) * rs * my_scale[c + x];
              if constexpr (SWIGLU) f[i] = swiglu<T>(f[i], __int2float_rn((int)u[x]) * rs * my_scale[64 + c + x]);
            }
            v[part * (32 / PER) + j] = Out<T>::pack(f);
          }
        }
        group8_transpose(v, lane);
        const int col = n0 + c0 + (lane & 7) * PER;
        if (col < p.N) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if ((ok_rows >> ((lane & ~7) + k)) & 1u)
              *reinterpret_cast<uint4*>(static_cast<uintptr_t>(row_ptr[k]) + (size_t)col * sizeof(T)) = v[k];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
    }
    zero_tail_rows<T>(p, blockIdx.x * (32 * EPI_WARPS) + threadIdx.x - 64, gridDim.x * (32 * EPI_WARPS));
  }

  // ---- teardown ----
  if (*abort_flag) {            // copies that are still in flight land before the shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

template <bool SWIGLU, class T>
int run_large(const CUtensorMap& ma, const CUtensorMap& mb0, const CUtensorMap& mb1, const I8Params& p, cudaStream_t st) {
  static unsigned char smem_set[64] = {0};
  BWMOE_CUDA_OK(ensure_dynamic_smem(int8_gemm_kernel<SWIGLU, T>, SMEM_BYTES, smem_set));
  const long long max_tiles = (long long)(ceil_div(p.M, BM) + p.E) * p.n_tiles;
  const int grid = (int)std::min<long long>(gemm_sm_budget(), max_tiles);
  BWMOE_CUDA_OK(launch_chained(int8_gemm_kernel<SWIGLU, T>, dim3(grid), dim3(I8_THREADS), SMEM_BYTES, st, ma, mb0, mb1, p));
  return BWMOE_OK;
}

template <bool SWIGLU>
int run_typed(const CUtensorMap& ma, const CUtensorMap& mb0, const CUtensorMap& mb1, const I8Params& p, int dtype, cudaStream_t st) {
  if (dtype == BWMOE_F32) return run_large<SWIGLU, float>(ma, mb0, mb1, p, st);
  if (dtype == BWMOE_F16) return run_large<SWIGLU, __half>(ma, mb0, mb1, p, st);
  return run_large<SWIGLU, __nv_bfloat16>(ma, mb0, mb1, p, st);
}

}  // namespace

size_t int8_scratch_bytes(int /*M*/, int /*K*/, int /*N*/, int /*E*/) { return 256; }

int check_int8_gemm(const void* a, const float* row_scale, const int32_t* offsets, const void* w0, const void* w1,
                    const float* scale0, const float* scale1, int M, int K, int N, int E, int dtype, const void* out,
                    const int32_t* status) {
  const bool swiglu = w1 != nullptr;
  const char* who = swiglu ? "int_gateup_swiglu" : "int_grouped_gemm";
  BWMOE_REQUIRE(M > 0 && K > 0 && N > 0 && E > 0, BWMOE_ERR_BAD_SHAPE, "%s: M=%d K=%d N=%d E=%d", who, M, K, N, E);
  BWMOE_REQUIRE(K % 16 == 0 && N % 16 == 0, BWMOE_ERR_BAD_SHAPE, "%s: K=%d and N=%d must be multiples of 16", who, K, N);
  BWMOE_REQUIRE(E <= kMaxGroups, BWMOE_ERR_UNSUPPORTED, "%s: E=%d > %d", who, E, kMaxGroups);
  BWMOE_REQUIRE(K < (1 << 17), BWMOE_ERR_UNSUPPORTED, "%s: K=%d: sums of 2^17 products or more do not fit 32 bits", who, K);
  BWMOE_REQUIRE(dtype >= BWMOE_BF16 && dtype <= BWMOE_F32, BWMOE_ERR_UNSUPPORTED, "%s: unknown type %d", who, dtype);
  BWMOE_REQUIRE(a && row_scale && w0 && scale0 && out && status && (!swiglu || scale1), BWMOE_ERR_NULL, "%s: null pointer", who);
  BWMOE_REQUIRE(offsets != nullptr || E == 1, BWMOE_ERR_NULL, "%s: %d experts need offsets", who, E);
  BWMOE_REQUIRE(aligned16(a) && aligned16(w0) && aligned16(w1) && aligned16(scale0) && aligned16(scale1) && aligned16(out),
                BWMOE_ERR_BAD_ALIGN, "%s: codes, channel scales and the result must be 16-byte aligned", who);
  BWMOE_REQUIRE((long long)(ceil_div(M, BM) + E) * ceil_div(N, BN_HALF) < (1ll << 31), BWMOE_ERR_UNSUPPORTED, "%s: too many tiles", who);
  return BWMOE_OK;
}

int launch_int8_gemm(const void* a, const float* row_scale, const int32_t* offsets, const void* w0, const void* w1,
                     const float* scale0, const float* scale1, int M, int K, int N, int E, int dtype, void* out, int32_t* status,
                     cudaStream_t st, bool clear_status) {
  const bool swiglu = w1 != nullptr;
  if (int rc = check_int8_gemm(a, row_scale, offsets, w0, w1, scale0, scale1, M, K, N, E, dtype, out, status)) return rc;
  if (clear_status) BWMOE_CUDA_OK(cudaMemsetAsync(status, 0, 16, st));
  const int n_tiles = ceil_div(N, swiglu ? BN_HALF : BN);
  CUtensorMap ma, mb0, mb1;
  if (int rc = make_map_a(&ma, a, M, K)) return rc;
  if (int rc = make_map_b(&mb0, w0, E, K, N)) return rc;
  if (int rc = make_map_b(&mb1, swiglu ? w1 : w0, E, K, N)) return rc;
  const I8Params p{offsets, row_scale, scale0, scale1, out, status, E, M, K, N, n_tiles};
  return swiglu ? run_typed<true>(ma, mb0, mb1, p, dtype, st) : run_typed<false>(ma, mb0, mb1, p, dtype, st);
}

}  // namespace bwmoe
