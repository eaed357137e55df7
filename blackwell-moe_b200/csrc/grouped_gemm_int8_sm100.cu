// Grouped products in 8-bit integers on the 5th-generation tensor cores, a scale for each row and for each channel.
//
//   PLAIN  : out[m,n] = (sum_k a[m,k] * w[e,k,n]) * row_scale[m] * channel_scale[e,n]
//   SWIGLU : h[m,n]   = silu(gate) * up, gate and up being two such products of the same rows
//
// where e is the expert whose segment offsets[e] .. offsets[e+1] holds row m.  The sums are formed in 32-bit integers and
// are exact whatever their order (|a|, |w| <= 128 and K < 2^17); scales, SwiGLU and the one rounding to the output type
// happen in fp32 in the epilogue (scaled() says in which order).
//
// Two kernels, persistent, one CTA per SM, warp-specialised (TMA producer, tcgen05.mma kind::i8 issuer, epilogue warps);
// activations are read K-major, weights in the caller's [E, K, N] layout (N contiguous):
//   int8_gemm_kernel        128 rows x 256 channels per tile, the rows on the MMA's M side; or a CTA pair on 256 x 256
//   int8_gemm_small_kernel  32 rows x 256 channels per tile, the channels on the M side (decode batches)
// (SWIGLU: 128 gate + 128 up channels in the place of the 256.)
//
// Pieces.  Where the tiles do not fill the chip, their K loops are cut into slices.  A slice leaves its accumulators in the
// scratch, and the one of a tile that arrives last (a counter per tile and epilogue warp) adds them up and finishes the tile:
// nobody waits for anybody, no second kernel runs, and 32-bit integer sums are the same in every order.  Pieces (tile, slice)
// are ordered by expert, then slice, then channels, then rows, so that neighbouring CTAs read neighbouring bytes of the same
// rows of the weights at the same time and an expert's rows stay in L2 while its weights stream through once.  (Dealing the K
// blocks of all tiles out in equal contiguous shares instead, which keeps every CTA equally busy, reads scattered 256-byte
// pieces: 4.1 TB/s against 5.6 at 8 experts of 4096 x 14336.)
//
// Every wait is bounded as in the other GEMM kernels of this library.
#include <type_traits>

#include "sm100_gemm.cuh"

namespace bwmoe {
namespace {
using namespace sm100;

// D = int32, A = B = signed 8-bit, A K-major, B MN-major, N = 256, M = 128
constexpr uint32_t IDESC_I8 = (2u << 4) | (1u << 7) | (1u << 10) | (0u << 15) | (1u << 16) | ((uint32_t)(BN >> 3) << 17) |
                              ((uint32_t)(BM >> 4) << 24);
constexpr uint32_t IDESC_I8_HALF = (IDESC_I8 & ~(0x3fu << 17)) | ((uint32_t)(BN_HALF >> 3) << 17);      // N = 128: one weight box
constexpr uint32_t IDESC_I8_PAIR = (IDESC_I8 & ~(0x1fu << 24)) | ((uint32_t)((2 * BM) >> 4) << 24);        // M = 256: a CTA pair
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

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
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
  // The kernel in front is the one that quantised the rows, and it lets this one be scheduled beside it: weights, scales and
  // offsets are older than that kernel, so set-up and the first weight tiles do not wait for it.
  bool early;
  bool sectors;             // out is aligned to 32 bytes
};

// Segment e, clamped to the rows there are: offsets are data from outside the kernel.
__device__ __forceinline__ void segment(const I8Params& p, int e, int& r0, int& r1) {
  r0 = p.offsets != nullptr ? min(max(p.offsets[e], 0), p.M) : 0;
  r1 = p.offsets != nullptr ? min(max(p.offsets[e + 1], r0), p.M) : p.M;
}

// Segments in order have fewer tiles (the host checks); overlapping ones might not, and their count ends here.
constexpr unsigned kMostTiles = 0x7fffffffu;

// first / end: the segments; cum: tiles before each.  All threads of the block; read behind the next __syncthreads().
template <int THREADS>
__device__ __forceinline__ void tile_table(const I8Params& p, int tile_rows, int tiles_per_row_block, int* s_first, int* s_end,
                                           int* s_cum) {
  for (int e = threadIdx.x; e < kMaxGroups; e += THREADS) {
    int r0 = 0, r1 = 0;
    if (e < p.E) segment(p, e, r0, r1);
    s_first[e] = r0, s_end[e] = r1;
    s_cum[e + 1] = (int)min((long long)((r1 - r0 + tile_rows - 1) / tile_rows) * tiles_per_row_block, (long long)kMostTiles);
  }
  __syncthreads();
  if (threadIdx.x < 32) {       // inclusive scan: 8 values per lane, then a shuffle scan of the lanes' totals
    const int lane = threadIdx.x;
    auto sum = [](int a, int b) { return (int)min((unsigned)a + (unsigned)b, kMostTiles); };
    int v[8], run = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = run = sum(run, s_cum[1 + lane * 8 + j]);
    int incl = run;
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl = sum(incl, o);
    }
    const int before = __shfl_up_sync(0xffffffffu, incl, 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) s_cum[1 + lane * 8 + j] = lane > 0 ? sum(before, v[j]) : v[j];
    if (lane == 0) s_cum[0] = 0;
  }
}

// K blocks per slice (one warp).  In ns, a slicing takes the longer of all K blocks at the memory's rate (32 KiB of weights in
// 5.5, which is 6 TB/s) and of the longest CTA's blocks, and then the adding up: fixed, and per slice.  One K block of a CTA counts
// as 500.  Measured, weights from memory, by the difference between K = 32768 and 65536 and between 65536 and 131056: 32-row
// tiles 260 (64 CTAs) to 320 - 440 (100), 128-row tiles 350 - 450; the rest is for what the others on the chip take of the memory.
__device__ __forceinline__ int blocks_per_slice(int tiles, int k_blocks, int ctas, int max_pieces, int fixed_ns, int slice_ns) {
  const int lane = threadIdx.x & 31, per = (k_blocks + lane) / (lane + 1), slices = (k_blocks + per - 1) / per;
  const long long pieces = (long long)tiles * slices;
  unsigned cost = 0x7ffffffu;
  if (slices == 1 || pieces <= max_pieces) {
    const long long memory = (long long)tiles * k_blocks * 11 / 2, longest = (pieces + ctas - 1) / ctas * per * 500;
    cost = (unsigned)min((memory > longest ? memory : longest) + (slices > 1 ? fixed_ns + slice_ns * slices : 0), 0x7fffffell);
  }
  const unsigned best = __reduce_min_sync(0xffffffffu, cost * 32u + (unsigned)lane);      // (a tie: fewer slices)
  return __shfl_sync(0xffffffffu, per, best & 31u);
}

// The pieces' places: every role of a CTA walks the same rising sequence of piece numbers.
struct I8Pieces {
  const int *first, *end, *cum;
  int E, tile_rows, k_blocks, per, slices, e;
  long long total;
  int tile, row0, row_end, n_idx, slice, kb0, kb1;      // of the piece last located, an expert e's
  __device__ __forceinline__ I8Pieces(const int* first_, const int* end_, const int* cum_, int E_, int tile_rows_, int k_blocks_, int per_)
      : first(first_), end(end_), cum(cum_), E(E_), tile_rows(tile_rows_), k_blocks(k_blocks_), per(per_),
        slices((k_blocks_ + per_ - 1) / per_), e(0), total((long long)cum_[E_] * slices) {}
  __device__ __forceinline__ void locate(long long piece) {      // piece < total
    while (piece >= (long long)cum[e + 1] * slices) ++e;
    const int tiles = cum[e + 1] - cum[e], m_tiles = (end[e] - first[e] + tile_rows - 1) / tile_rows;
    int within = (int)(piece - (long long)cum[e] * slices);
    slice = slices > 1 ? within / tiles : 0;
    within -= slice * tiles;
    tile = cum[e] + within;
    n_idx = within / m_tiles;
    row0 = first[e] + (within - n_idx * m_tiles) * tile_rows;
    row_end = end[e];
    kb0 = slice * per, kb1 = min(k_blocks, kb0 + per);
  }
};

// The weights of the CTA's first stages (all stages are free then); the number of stages begun.
template <class Load>
__device__ __forceinline__ int first_weights(I8Pieces q, int stages, int first_piece, int piece_step, Load load_weights) {
  int n = 0;
  for (long long piece = first_piece; n < stages && piece < q.total; piece += piece_step) {
    q.locate(piece);
    for (int kb = q.kb0; n < stages && kb < q.kb1; ++kb, ++n) load_weights(q, kb, n);
  }
  return n;
}

// Slices of a tile meet here.  A slab holds the accumulators of one piece, 16 bytes per lane side by side.
struct I8Slices {
  uint32_t* arrivals;       // [tiles][8 epilogue warps], zero at the start and at the end
  int4* slabs;              // nullptr: no tile is cut
};
// N accumulators of every lane, at vector `at` of the warp's part of the slab
template <int N>
__device__ __forceinline__ void slab_store(int4* part, int at, int lane, const uint32_t* a) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    __stcg(part + (at + i) * 32 + lane, make_int4((int)a[4 * i], (int)a[4 * i + 1], (int)a[4 * i + 2], (int)a[4 * i + 3]));
}
// adds the other slices' accumulators; `stride`: vectors from one slice's slab to the next.  Up to 64 values are requested at once.
template <int N>
__device__ __forceinline__ void slab_add(const int4* part0, size_t stride, int slices, int mine, int at, int lane, uint32_t* a) {
  constexpr int AT_ONCE = 64 / N;
#pragma unroll 1
  for (int s0 = 0; s0 < slices; s0 += AT_ONCE) {
    int4 v[AT_ONCE][N / 4];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        v[j][i] = s0 + j < slices && s0 + j != mine ? __ldcg(part0 + (size_t)(s0 + j) * stride + (at + i) * 32 + lane) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        a[4 * i] += (uint32_t)v[j][i].x, a[4 * i + 1] += (uint32_t)v[j][i].y;
        a[4 * i + 2] += (uint32_t)v[j][i].z, a[4 * i + 3] += (uint32_t)v[j][i].w;
      }
  }
}
// The warp's accumulators are in the slab: whether all other slices' are, too.
__device__ __forceinline__ bool last_slice(uint32_t* counter, int slices, int lane) {
  __syncwarp();
  unsigned arrived = 0;
  if (lane == 0) {
    __threadfence();
    arrived = atomicAdd(counter, 1u);
    __threadfence();
  }
  const bool last = __shfl_sync(0xffffffffu, arrived, 0) == (unsigned)slices - 1;
  __syncwarp();                                   // (orders the other lanes' reads behind lane 0's fence)
  if (last && lane == 0) *counter = 0;            // for the next product with this scratch
  return last;
}

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
// 32 bytes at a 16-byte aligned address; at once where it is aligned to 32.
__device__ __forceinline__ void store_sector(void* p, const uint4& a, const uint4& b, bool aligned32) {
  if (aligned32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
                 "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = a;
    reinterpret_cast<uint4*>(p)[1] = b;
  }
}
// acc * channel * row in the order that ends in infinity only where the product itself does: |acc| < 2^31, so a factor of up
// to 2^96 can come first, and where that is the row's scale and not the channel's, the row's does.  (With both above it, any
// acc but 0 gives infinity.)  Nothing is lost at the other end: |acc| >= 1, so acc * scale is below the normal numbers only
// where the scale is, and then it is exact.
constexpr float kFirstScale = 7.922816251426434e28f;      // 2^96
__device__ __forceinline__ float scaled(uint32_t acc, float channel, float row) {
  return __int2float_rn((int)acc) * channel * row;
}
__device__ __forceinline__ float scaled_any(uint32_t acc, float channel, float row) {
  const bool row_first = channel > kFirstScale && row <= kFirstScale;
  return scaled(acc, row_first ? row : channel, row_first ? channel : row);
}

// silu(g) * u with the accurate exponential and a quotient that is rounded like a division's.  16-bit results get the quotient
// from the reciprocal and one Newton step on what is left over (Markstein's correction), which needs no branch per element: half
// a step and 2^-22 of one.  (What is left over is NaN where g or d is infinite; then the first estimate is the result.  From
// d = 2^126 on the reciprocal is 0, and so is the result instead of a number below 2^-119.)  With __expf and __fdividef, whose
// error of 2 + 1.16 |g| steps grows with the gate, one bf16 result in 120000 and one fp16 result in 22500 was rounded the other way
// (gates of ordinary size), and where it was a row's largest, every code of the row followed: a block of 2048 x 1408 experts was up to
// 3.6e-4 (2-norm) from the same steps by torch in 32 bits, at most 3.3e-5 now.  Cost at 64 experts of 2048 x 1408, 768 rows each: 212 -> 218 us (222 with the
// division); 384 rows 126 -> 128, decode batches and fp32 results nothing.
template <class T> __device__ __forceinline__ float swiglu(float g, float u) {
  const float d = 1.0f + expf(-g);
  if constexpr (sizeof(T) == 4) return g / d * u;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  const float q = g * r, rest = fmaf(-d, q, g);
  return (rest == rest ? fmaf(rest, r, q) : q) * u;
}

// Rows in front of the first segment and behind the last belong to no expert: zeros.  `part` of `parts` threads.
template <class T>
__device__ __forceinline__ void zero_other_rows(const I8Params& p, int part, int parts) {
  if (p.offsets == nullptr) return;
  const size_t row = (size_t)p.N / Out<T>::kPer16;      // 16-byte vectors
  const size_t head = min(max(p.offsets[0], 0), p.M) * row, tail = min(max(p.offsets[p.E], 0), p.M) * row, end = p.M * row;
  uint4* out = static_cast<uint4*>(p.out);
  for (size_t i = part; i < head; i += parts) out[i] = make_uint4(0u, 0u, 0u, 0u);
  for (size_t i = tail + part; i < end; i += parts) out[i] = make_uint4(0u, 0u, 0u, 0u);
}

constexpr int L_MAX_PIECES = 320;                                             // where tiles are cut: a slab for each
constexpr int L_PART = BN / 2 * 32 / 4;                                       // vectors of one epilogue warp's part of a slab
constexpr size_t L_SLAB = (size_t)EPI_WARPS * L_PART * sizeof(int4);          // 128 KiB

// PAIR: the CTAs of a two-CTA cluster share 256-row tiles (cta_group::2).  CTA `rank` of the pair loads rows rank * 128 .. of the
// tile and one of its two weight boxes (SWIGLU: rank 0 the gate's, rank 1 the up matrix's); the even CTA issues M = 256 MMAs
// that read both shared memories and write each CTA's 128 rows into that CTA's tensor memory.  Loads of both CTAs report to
// the even CTA's full barrier; the issuer commits to each CTA's empty and full-accumulator barriers in turn; the odd CTA's
// epilogue warps hand accumulator buffers back on the even CTA's barrier.  None of the loads is a multicast.
template <bool SWIGLU, class T, bool PAIR>
__global__ void __launch_bounds__(I8_THREADS, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b0,
                 const __grid_constant__ CUtensorMap map_b1, const I8Params p, const I8Slices sl) {
  if (!p.early) chain_wait();
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_first[kMaxGroups], s_end[kMaxGroups], s_cum[kMaxGroups + 1];
  __shared__ __align__(16) float s_scale[EPI_WARPS][BN / 2];      // each epilogue warp's channel scales of its tile
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_per;

  constexpr int NSTAGE = PAIR ? PAIR_STAGES : STAGES, STAGE_SZ = PAIR ? PAIR_STAGE_BYTES : STAGE_BYTES;
  const uint32_t tiles_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = tiles_base + NSTAGE * STAGE_SZ;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * NSTAGE;
  const uint32_t bar_tfull = bars + 16 * NSTAGE, bar_tempty = bar_tfull + 16;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;            // place in the pair
  const int first_piece = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, piece_step = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k_blocks = (p.Kdim + BK - 1) / BK;
  volatile int* abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < NSTAGE; ++s) mbar_init(bar_full + 8 * s, 1), mbar_init(bar_empty + 8 * s, 1);
    for (int b = 0; b < 2; ++b) mbar_init(bar_tfull + 8 * b, 1), mbar_init(bar_tempty + 8 * b, PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tile_table<I8_THREADS>(p, PAIR ? 2 * BM : BM, p.n_tiles, s_first, s_end, s_cum);
  if (warp == 0) {
    __syncwarp();
    const int per = PAIR || sl.slabs == nullptr ? k_blocks : blocks_per_slice(s_cum[p.E], k_blocks, gridDim.x, L_MAX_PIECES, 3000, 2200);
    if (lane == 0) s_per = per;
  }
  if (warp == 1) {
    if constexpr (PAIR) tmem_alloc_pair(smem_u32(&s_tmem_base), TMEM_COLS);
    else                tmem_alloc(smem_u32(&s_tmem_base), TMEM_COLS);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();       // the peer's barriers and tensor memory exist from here on
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  I8Pieces q(s_first, s_end, s_cum, p.E, PAIR ? 2 * BM : BM, k_blocks, s_per);

  // PLAIN: the last tile of a row may have one weight box of channels only; then the other is neither loaded nor multiplied
  auto one_box = [&](const I8Pieces& q) { return !SWIGLU && !PAIR && q.n_idx * BN + BN_HALF >= p.N; };
  auto load_weights = [&](const I8Pieces& q, int kb, uint32_t stage) {
    const uint32_t sb = tiles_base + stage * STAGE_SZ + A_BYTES, full = bar_full + 8 * stage;
    const int n0 = q.n_idx * (SWIGLU ? BN_HALF : BN);
    if constexpr (PAIR) {       // both CTAs' bytes are counted by the even CTA's barrier, which alone announces them
      if (rank == 0) mbar_expect_tx(full, 2 * PAIR_STAGE_BYTES);
      if (SWIGLU) tma_load_3d_pair(sb, rank ? &map_b1 : &map_b0, map_to_cta(full, 0), n0, kb * BK, q.e);
      else        tma_load_3d_pair(sb, &map_b0, map_to_cta(full, 0), n0 + (int)rank * BN_HALF, kb * BK, q.e);
      return;
    }
    const bool one = one_box(q);
    mbar_expect_tx(full, one ? STAGE_BYTES - B_HALF_BYTES : STAGE_BYTES);
    tma_load_3d(sb, &map_b0, full, n0, kb * BK, q.e);
    if (SWIGLU)    tma_load_3d(sb + B_HALF_BYTES, &map_b1, full, n0, kb * BK, q.e);
    else if (!one) tma_load_3d(sb + B_HALF_BYTES, &map_b0, full, n0 + BN_HALF, kb * BK, q.e);
  };
  int ahead = 0;                // stages whose weights are on their way already
  if (p.early) {
    if (threadIdx.x == 0) ahead = first_weights(q, NSTAGE, first_piece, piece_step, load_weights);
    chain_wait();
  }
  if (warp == 0) {
    // ===================== TMA producer =====================
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (long long piece = first_piece; ok && piece < q.total; piece += piece_step) {
        q.locate(piece);
        for (int kb = q.kb0; kb < q.kb1; ++kb) {
          if (ahead > 0) {
            --ahead;
          } else {
            if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status))) break;
            load_weights(q, kb, stage);
          }
          const uint32_t sa = tiles_base + stage * STAGE_SZ, full = bar_full + 8 * stage;
          if constexpr (PAIR) tma_load_2d_pair(sa, &map_a, map_to_cta(full, 0), kb * BK, q.row0 + (int)rank * BM);
          else                tma_load_2d(sa, &map_a, full, kb * BK, q.row0);
          if (++stage == NSTAGE) stage = 0, phase ^= 1u;
        }
      }
      if constexpr (PAIR) {
        // the issuer's last commits arrive on this CTA's empty barriers from the other CTA: let them land before this CTA can leave
        for (int i = 0; ok && i < NSTAGE; ++i) {
          ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status);
          if (++stage == NSTAGE) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    if (lane == 0 && rank == 0) {
      uint32_t stage = 0, phase = 0, local = 0;
      bool ok = true;
      for (long long piece = first_piece; ok && piece < q.total; piece += piece_step, ++local) {
        q.locate(piece);
        const uint32_t buf = local & 1u, use = local >> 1, desc = one_box(q) ? IDESC_I8_HALF : IDESC_I8;
        if (!(ok = mbar_wait(bar_tempty + 8 * buf, (use & 1u) ^ 1u, abort_flag, p.status))) break;
        tc_fence_after();
        for (int kb = q.kb0; kb < q.kb1; ++kb) {
          if (!(ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status))) break;
          tc_fence_after();
          const uint32_t sa = tiles_base + stage * STAGE_SZ;
          const uint64_t da = desc_kmajor(sa), db = desc_nmajor(sa + A_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) {   // A: +32 bytes along K inside the swizzle atom; B: +32 K rows = 4096 bytes
            const uint32_t acc = kb > q.kb0 || k > 0 ? 1u : 0u;
            if constexpr (PAIR) mma_i8_pair(tmem_base + buf * BN, da + (uint64_t)(k * 2), db + (uint64_t)(k * 256), IDESC_I8_PAIR, acc);
            else                mma_i8(tmem_base + buf * BN, da + (uint64_t)(k * 2), db + (uint64_t)(k * 256), desc, acc);
          }
          if constexpr (PAIR) mma_commit_pair(bar_empty + 8 * stage), mma_commit_pair(map_to_cta(bar_empty + 8 * stage, 1));
          else                mma_commit(bar_empty + 8 * stage);
          if (++stage == NSTAGE) stage = 0, phase ^= 1u;
        }
        if (ok) {
          if constexpr (PAIR) mma_commit_pair(bar_tfull + 8 * buf), mma_commit_pair(map_to_cta(bar_tfull + 8 * buf, 1));
          else                mma_commit(bar_tfull + 8 * buf);
        }
      }
    }
  } else {
    // ===================== epilogue (warps 2..9) =====================
    const int quarter = warp & 3, half = (warp - 2) >> 2;      // tensor-memory lanes this warp may read; half of the columns
    float* my_scale = s_scale[warp - 2];
    uint32_t local = 0;
    bool ok = true;
    for (long long piece = first_piece; ok && piece < q.total; piece += piece_step, ++local) {
      q.locate(piece);
      const uint32_t buf = local & 1u, use = local >> 1;
      const int row = q.row0 + (int)rank * BM + quarter * 32 + lane;
      const bool row_ok = row < q.row_end;
      const float rs = row_ok ? p.row_scale[row] : 0.f;
      // channel scales of this warp's columns (SWIGLU: 64 of the gate, then 64 of the up product), zero past N
      const int n0 = q.n_idx * (SWIGLU ? BN_HALF : BN) + half * (SWIGLU ? BN_HALF / 2 : BN_HALF);
      bool huge;                                 // a channel scale that may have to come second
      {
        const float* s = (SWIGLU && lane >= 16 ? p.scale1 : p.scale0) + (size_t)q.e * p.N;
        const int n = n0 + (SWIGLU ? (lane & 15) : lane) * 4;
        __syncwarp();                            // the tile before has read its scales
        // (N is a multiple of 16, scales of 16-byte alignment: four at a time)
        const float4 v = n < p.N ? *reinterpret_cast<const float4*>(s + n) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(my_scale + 4 * lane) = v;
        huge = __any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) > kFirstScale);
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * buf, use & 1u, abort_flag, p.status));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * BN;
      constexpr int PER = Out<T>::kPer16, COLS = SWIGLU ? BN_HALF / 2 : BN_HALF;       // columns of this warp
      const bool work = n0 < p.N;                                // (the second half of a tile may lie past N)
      bool complete = work;
      const int4* part0 = nullptr;                               // this warp's part of slice 0's slab
      if (q.slices > 1 && work) {
        part0 = sl.slabs + ((size_t)q.tile * q.slices * EPI_WARPS + (warp - 2)) * L_PART;
        int4* part = const_cast<int4*>(part0) + (size_t)q.slice * EPI_WARPS * L_PART;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32) {
          uint32_t a[32];
          tmem_ld32(t_row + half * COLS + c, a);
          tmem_ld_wait();
          slab_store<32>(part, c / 4, lane, a);
          if constexpr (SWIGLU) {
            tmem_ld32(t_row + BN_HALF + half * COLS + c, a);
            tmem_ld_wait();
            slab_store<32>(part, (COLS + c) / 4, lane, a);
          }
        }
        complete = last_slice(sl.arrivals + q.tile * EPI_WARPS + (warp - 2), q.slices, lane);
      }
      // A lane writes its row in whole 32-byte sectors.  (Pieces exchanged between lanes, so that a store covers 128 bytes of
      // four rows, cost shared-memory cycles that the MMAs' operands want: 64 experts of 2048 x 1408
      // with 768 rows each, SwiGLU: 255 -> 237 us, one product 142 -> 140)
      T* dst = static_cast<T*>(p.out) + (size_t)row * p.N + n0;
#pragma unroll 1
      for (int c = 0; complete && c < COLS; c += 32) {
        uint32_t a[32], u[SWIGLU ? 32 : 4];
        tmem_ld32(t_row + half * COLS + c, a);
        if constexpr (SWIGLU) tmem_ld32(t_row + BN_HALF + half * COLS + c, u);
        tmem_ld_wait();
        if (q.slices > 1) {
          slab_add<32>(part0, (size_t)EPI_WARPS * L_PART, q.slices, q.slice, c / 4, lane, a);
          if constexpr (SWIGLU) slab_add<32>(part0, (size_t)EPI_WARPS * L_PART, q.slices, q.slice, (COLS + c) / 4, lane, u);
        }
        auto store = [&](auto scale) {
#pragma unroll
          for (int j = 0; j < 32; j += 2 * PER) {
            uint4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float f[PER];
#pragma unroll
              for (int i = 0; i < PER; ++i) {
                const int x = j + h * PER + i;
                f[i] = scale(a[x], my_scale[c + x], rs);
                if constexpr (SWIGLU) f[i] = swiglu<T>(f[i], scale(u[x], my_scale[64 + c + x], rs));
              }
              v[h] = Out<T>::pack(f);
            }
            if (row_ok && n0 + c + j < p.N) store_sector(dst + c + j, v[0], v[1], p.sectors);       // (N is a multiple of 16)
          }
        };
        if (huge) store([](uint32_t acc, float channel, float row) { return scaled_any(acc, channel, row); });
        else      store([](uint32_t acc, float channel, float row) { return scaled(acc, channel, row); });
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR && rank != 0) mbar_arrive_cluster(map_to_cta(bar_tempty + 8 * buf, 0));
        else                   mbar_arrive(bar_tempty + 8 * buf);
      }
    }
    zero_other_rows<T>(p, blockIdx.x * (32 * EPI_WARPS) + threadIdx.x - 64, gridDim.x * (32 * EPI_WARPS));
  }

  // ---- teardown ----
  if (*abort_flag) {            // copies that are still in flight land before the shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();       // neither CTA leaves while the other may still signal it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else                tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- few rows per expert
// Few rows per expert (decode): bound by the weights' bytes.  The weight tile takes the M side of the MMA and the rows the N
// side, D^T[128 channels (tensor-memory lanes), 32 rows (columns)]: a stage is 32 KiB of weights and 4 KiB of rows, and six of
// them are in flight.  Two epilogue warps per lane quarter, 16 of the rows each; a thread owns a channel of either weight tile.
// NARROW: 128 channels per tile, one weight box per stage, where that still fits the SMs at once: twice the tiles, half the
// slices to add up (one row, 4096 x 14336: 17.5 -> 15.5 us, 2048 x 2048: 9.5 -> 8.6; 32 rows, 8192 x 1024: 16.5 -> 12.4).
constexpr int S_NT = 32;                                     // rows per tile
constexpr int S_THREADS = 64 + 32 * EPI_WARPS;
constexpr int S_STAGES = 6;
constexpr int S_W_BYTES = 2 * B_HALF_BYTES;
constexpr int S_STAGE_BYTES = S_W_BYTES + S_NT * BK;         // 36 KiB
constexpr int S_SMEM_BYTES = S_STAGES * S_STAGE_BYTES + 1024 /*alignment slack*/ + 512 /*barriers*/;
constexpr int S_BUF_COLS = 2 * S_NT;
constexpr int S_NBUF = TMEM_COLS / S_BUF_COLS;               // tiles in flight in tensor memory
constexpr int S_MAX_PIECES = 640;                            // where tiles are cut: a slab for each
constexpr int S_PART = 2 * (S_NT / 2) * 32 / 4;              // vectors of one epilogue warp's part of a slab
constexpr size_t S_SLAB = (size_t)EPI_WARPS * S_PART * sizeof(int4);        // 32 KiB
// D = int32, A = B = signed 8-bit, A MN-major (the weight tile), B K-major (the rows), N = 32, M = 128
constexpr uint32_t IDESC_I8_SMALL = (2u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | ((uint32_t)(S_NT >> 3) << 17) |
                                    ((uint32_t)(BM >> 4) << 24);

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[8]) { tmem_ld8(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

template <bool SWIGLU, class T, bool NARROW>
__global__ void __launch_bounds__(S_THREADS, 1)
int8_gemm_small_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                       const __grid_constant__ CUtensorMap map_w1, const I8Params p, const I8Slices sl) {
  if (!p.early) chain_wait();
  static_assert(!(SWIGLU && NARROW), "SwiGLU has two weight boxes");
  constexpr int CH = SWIGLU || NARROW ? BN_HALF : BN;             // channels of the result in a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_first[kMaxGroups], s_end[kMaxGroups], s_cum[kMaxGroups + 1];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_per;

  const uint32_t tiles_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = tiles_base + S_STAGES * S_STAGE_BYTES;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * S_STAGES;
  const uint32_t bar_tfull = bars + 16 * S_STAGES, bar_tempty = bar_tfull + 8 * S_NBUF;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k_blocks = (p.Kdim + BK - 1) / BK;
  volatile int* abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < S_STAGES; ++s) mbar_init(bar_full + 8 * s, 1), mbar_init(bar_empty + 8 * s, 1);
    for (int b = 0; b < S_NBUF; ++b) mbar_init(bar_tfull + 8 * b, 1), mbar_init(bar_tempty + 8 * b, EPI_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tile_table<S_THREADS>(p, S_NT, p.n_tiles, s_first, s_end, s_cum);
  if (warp == 0) {
    __syncwarp();
    const int per = blocks_per_slice(s_cum[p.E], k_blocks, gridDim.x, S_MAX_PIECES, 1500, 100);
    if (lane == 0) s_per = per;
  }
  if (warp == 1) tmem_alloc(smem_u32(&s_tmem_base), TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  I8Pieces q(s_first, s_end, s_cum, p.E, S_NT, k_blocks, s_per);

  auto load_weights = [&](const I8Pieces& q, int kb, uint32_t stage) {
    const uint32_t sw = tiles_base + stage * S_STAGE_BYTES, full = bar_full + 8 * stage;
    const int n0 = q.n_idx * CH;
    mbar_expect_tx(full, NARROW ? S_STAGE_BYTES - B_HALF_BYTES : S_STAGE_BYTES);
    tma_load_3d(sw, &map_w0, full, n0, kb * BK, q.e);
    if (SWIGLU)       tma_load_3d(sw + B_HALF_BYTES, &map_w1, full, n0, kb * BK, q.e);
    else if (!NARROW) tma_load_3d(sw + B_HALF_BYTES, &map_w0, full, n0 + BN_HALF, kb * BK, q.e);
  };
  int ahead = 0;                // stages whose weights are on their way already
  if (p.early) {
    if (threadIdx.x == 0) ahead = first_weights(q, S_STAGES, blockIdx.x, gridDim.x, load_weights);
    chain_wait();
  }
  if (warp == 0) {
    // ===================== TMA producer =====================
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (long long piece = blockIdx.x; ok && piece < q.total; piece += gridDim.x) {
        q.locate(piece);
        for (int kb = q.kb0; kb < q.kb1; ++kb) {
          if (ahead > 0) {
            --ahead;
          } else {
            if (!(ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status))) break;
            load_weights(q, kb, stage);
          }
          tma_load_2d(tiles_base + stage * S_STAGE_BYTES + S_W_BYTES, &map_x, bar_full + 8 * stage, kb * BK, q.row0);
          if (++stage == S_STAGES) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, it = 0;
      bool ok = true;
      for (long long piece = blockIdx.x; ok && piece < q.total; piece += gridDim.x, ++it) {
        q.locate(piece);
        const uint32_t buf = it % S_NBUF, use = it / S_NBUF;
        if (!(ok = mbar_wait(bar_tempty + 8 * buf, (use & 1u) ^ 1u, abort_flag, p.status))) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * S_BUF_COLS;
        for (int kb = q.kb0; kb < q.kb1; ++kb) {
          if (!(ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status))) break;
          tc_fence_after();
          const uint32_t sw = tiles_base + stage * S_STAGE_BYTES;
          const uint64_t db = desc_kmajor(sw + S_W_BYTES), da0 = desc_nmajor(sw), da1 = desc_nmajor(sw + B_HALF_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) {     // weights: +32 K rows = 4096 bytes; rows: +32 bytes along K
            mma_i8(d, da0 + (uint64_t)(k * 256), db + (uint64_t)(k * 2), IDESC_I8_SMALL, kb > q.kb0 || k > 0 ? 1u : 0u);
            if (!NARROW) mma_i8(d + S_NT, da1 + (uint64_t)(k * 256), db + (uint64_t)(k * 2), IDESC_I8_SMALL, kb > q.kb0 || k > 0 ? 1u : 0u);
          }
          mma_commit(bar_empty + 8 * stage);
          if (++stage == S_STAGES) stage = 0, phase ^= 1u;
        }
        if (ok) mma_commit(bar_tfull + 8 * buf);
      }
    }
  } else {
    // ===================== epilogue (warps 2..9) =====================
    const int quarter = warp & 3, c0 = ((warp - 2) >> 2) * (S_NT / 2), f = quarter * 32 + lane;
    uint32_t it = 0;
    bool ok = true;
    for (long long piece = blockIdx.x; ok && piece < q.total; piece += gridDim.x, ++it) {
      q.locate(piece);
      const uint32_t buf = it % S_NBUF, use = it / S_NBUF;
      const int n_valid = min(S_NT / 2, q.row_end - q.row0 - c0);       // this warp's rows; none: <= 0
      const int n = q.n_idx * CH + f, m = SWIGLU ? n : n + BN_HALF;      // the thread's two channels (NARROW: the first)
      const float s0 = n < p.N ? p.scale0[(size_t)q.e * p.N + n] : 0.f;
      const float s1 = !NARROW && m < p.N ? (SWIGLU ? p.scale1 : p.scale0)[(size_t)q.e * p.N + m] : 0.f;
      const float my_rs = lane < n_valid ? p.row_scale[q.row0 + c0 + lane] : 0.f;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * buf, use & 1u, abort_flag, p.status));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * S_BUF_COLS + c0;
      auto finish = [&](auto columns) {
        constexpr int NC = decltype(columns)::value;
        uint32_t a0[NC], a1[NC];
        tmem_ld_cols(t_row, a0);
        if (!NARROW) tmem_ld_cols(t_row + S_NT, a1);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
        if (q.slices > 1) {
          const int4* part0 = sl.slabs + ((size_t)q.tile * q.slices * EPI_WARPS + (warp - 2)) * S_PART;
          int4* part = const_cast<int4*>(part0) + (size_t)q.slice * EPI_WARPS * S_PART;
          slab_store<NC>(part, 0, lane, a0);
          if (!NARROW) slab_store<NC>(part, S_NT / 8, lane, a1);
          if (!last_slice(sl.arrivals + q.tile * EPI_WARPS + (warp - 2), q.slices, lane)) return;
          slab_add<NC>(part0, (size_t)EPI_WARPS * S_PART, q.slices, q.slice, 0, lane, a0);
          if (!NARROW) slab_add<NC>(part0, (size_t)EPI_WARPS * S_PART, q.slices, q.slice, S_NT / 8, lane, a1);
        }
        T* out = static_cast<T*>(p.out) + (size_t)(q.row0 + c0) * p.N;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float rs = __shfl_sync(0xffffffffu, my_rs, c);
          const float v0 = scaled_any(a0[c], s0, rs), v1 = NARROW ? 0.f : scaled_any(a1[c], s1, rs);
          if (c >= n_valid) continue;
          if (SWIGLU) {
            if (n < p.N) out[(size_t)c * p.N + n] = Out<T>::one(swiglu<T>(v0, v1));
          } else {
            if (n < p.N) out[(size_t)c * p.N + n] = Out<T>::one(v0);
            if (!NARROW && m < p.N) out[(size_t)c * p.N + m] = Out<T>::one(v1);
          }
        }
      };
      if (n_valid > 8) finish(std::integral_constant<int, 16>{});
      else if (n_valid > 0) finish(std::integral_constant<int, 8>{});
      else {                                            // the tile has no rows for this warp
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
      }
    }
    zero_other_rows<T>(p, blockIdx.x * (32 * EPI_WARPS) + threadIdx.x - 64, gridDim.x * (32 * EPI_WARPS));
  }

  if (*abort_flag) {            // copies that are still in flight land before the shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// Which kernel a product gets.  32-row tiles: few rows per expert, or tiles so few that they fit the SMs at once (and K blocks
// few enough that reading the weights again for every 32 rows does not count).  Measured, us, 32-row tiles against 128-row tiles
// (launched one after the other, weights from memory):
//   8 experts of 4096 x 14336 (SwiGLU):  1 row each 144 / 203,  32 rows 150 / 158,  48 rows 161 / 158,  128 rows 300 / 167
//   64 experts of 2048 x 1408:           8 rows each 35.6 / 40.6,  32 rows 37.2 / 38.6,  48 rows 43.8 / 39.4
//   one matrix 4096 x 14336:  1 row 17.4 / 24.5,  48 rows 17.7 / 23.1,  128 rows 29.0 / 23.4
//   one matrix 2048 x 2048:  512 rows 11.7 / 13.2;   14336 x 4096:  48 rows 22.5 / 32.5,  128 rows 28.5 / 32.9,  256 rows 44.6 / 32.3
bool small_applies(int M, int K, int n_tiles, int E) {
  if (M <= 32ll * E) return true;
  const long long tiles = ((long long)M / S_NT + E) * n_tiles;
  return tiles <= sm_count() && tiles * ceil_div(K, BK) <= 8192;
}
// 128 channels per tile: one product of one matrix (whose tiles are known here) and one or two row blocks (with three of K =
// 14336 the rows' boxes count: 33 us against 28).
bool narrow_applies(int M, int N, int E, bool swiglu) {
  return !swiglu && E == 1 && M <= 2 * S_NT && ceil_div(M, S_NT) * ceil_div(N, BN_HALF) <= sm_count();
}
// Whether the other kernel's tiles may leave SMs without work, so that slabs are worth their memory.
bool may_slice(int M, int n_tiles) { return (long long)ceil_div(M, BM) * n_tiles < sm_count(); }

// Scratch: the status word, the counters (tiles that are cut have two slices at least), the slabs.
constexpr size_t kArrivalsAt = 16;
constexpr size_t kSlabsAt = kArrivalsAt + (S_MAX_PIECES > L_MAX_PIECES ? S_MAX_PIECES : L_MAX_PIECES) / 2 * EPI_WARPS * sizeof(uint32_t);

// CTA pairs (256-row tiles, every weight byte enters one of the two shared memories).  A 128 x 256 tile reads 96 bytes of
// operands a cycle from shared memory and wants 96 more written by its loads, of the 128 there are: the tensor pipe is busy 65 to
// 78 % of the time.  A pair's tile needs 64 + 64 (94 %).  Against it: the rows past a segment's end (half a tile on average, 128
// instead of 64), a start across two SMs, and with SwiGLU an epilogue that keeps up with fewer of a pair's MMAs.  Measured, us,
// pairs / single CTAs (alternating, queued back to back):
//   one product, one matrix:  8192 rows, 8192 x 8192 349 / 449, 2048 x 8192 95 / 105, 1024 x 8192 67 / 67, 512 x 8192 59 / 56;
//     4096 rows, 4096 x 4096 50.5 / 56.3;  2048 rows, 8192 x 8192 92.5 / 98.6;  1024 rows, 4096 x 4096 (64 tiles) 25.7 / 22.1
//   one product, 64 experts:  768 rows each, 2048 x 1536 138 / 149, 1408 x 2048 149 / 155;  1024 rows, 173 / 190, 201 / 196
//   one product, 8 experts of 14336 x 4096:  512 rows each 244 / 208, 1024 rows 356 / 391, 4096 rows 1430 / 1620
//   SwiGLU:  8 experts of 4096 x 14336, 1024 rows each 800 / 783, 2048 rows 1460 / 1490, 4096 rows 2720 / 2895;
//     64 experts of 2048 x 1408, 1024 rows each 359 / 336, 2048 rows 580 / 624
// At the borders the two are within 4 % of each other (one product: 67 / 67, 149 / 155, 201 / 196; SwiGLU: 1460 / 1490, 359 / 336 just
// outside).
bool pair_applies(int M, int K, int N, int E, bool swiglu) {
  if (gemm_sm_budget() < 2) return false;
  if (swiglu) return M >= 2048ll * E && 2.0 * M * K * N >= 4e11;
  const long long tiles = (long long)(M / (2 * BM)) * (N / BN);
  return M >= 768ll * E && K >= 1408 && N % BN == 0 && tiles >= 3 * (sm_count() / 2);
}

template <class Kernel>
int run(Kernel kernel, dim3 grid, int threads, int smem, unsigned char (&smem_set)[64], const CUtensorMap& ma, const CUtensorMap& mb0,
        const CUtensorMap& mb1, const I8Params& p, const I8Slices& sl, cudaStream_t st) {
  BWMOE_CUDA_OK(ensure_dynamic_smem(kernel, smem, smem_set));
  BWMOE_CUDA_OK(launch_chained(kernel, grid, dim3(threads), smem, st, ma, mb0, mb1, p, sl));
  return BWMOE_OK;
}

template <class Kernel>
int run_pair(Kernel kernel, unsigned char (&smem_set)[64], int (&resident)[64], const CUtensorMap& ma, const CUtensorMap& mb0,
             const CUtensorMap& mb1, const I8Params& p, const I8Slices& sl, cudaStream_t st) {
  BWMOE_CUDA_OK(ensure_dynamic_smem(kernel, PAIR_SMEM_BYTES, smem_set));
  const long long max_tiles = (long long)(ceil_div(p.M, 2 * BM) + p.E) * p.n_tiles;
  int pairs = (int)std::min<long long>(gemm_sm_budget() / 2, max_tiles);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(I8_THREADS);
  cfg.dynamicSmemBytes = PAIR_SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;     // the kernel waits for the one in front
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  // pairs that can be resident at once (per device, asked once): the persistent loop needs no more
  int dev = 0;
  BWMOE_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64) {
    if (resident[dev] == 0) {
      int n = 0;
      cfg.gridDim = dim3(2 * (sm_count() / 2));
      BWMOE_CUDA_OK(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      BWMOE_REQUIRE(n >= 1, BWMOE_ERR_CUDA, "no CTA pair of the 8-bit integer product fits on this device");
      resident[dev] = n;
    }
    pairs = std::min(pairs, resident[dev]);
  }
  cfg.gridDim = dim3(2 * pairs);
  note_launch();
  BWMOE_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, ma, mb0, mb1, p, sl));
  return BWMOE_OK;
}

template <bool SWIGLU, class T>
int run_typed(bool small, const CUtensorMap& ma, const CUtensorMap& mb0, const CUtensorMap& mb1, const I8Params& p,
              const I8Slices& sl, cudaStream_t st) {
  static unsigned char smem_set[3][64] = {};
  static int resident[64] = {};
  if (!small && pair_applies(p.M, p.Kdim, p.N, p.E, SWIGLU))
    return run_pair(int8_gemm_kernel<SWIGLU, T, true>, smem_set[2], resident, ma, mb0, mb1, p, sl, st);
  const long long max_pieces = (long long)(ceil_div(p.M, small ? S_NT : BM) + p.E) * p.n_tiles * (sl.slabs ? ceil_div(p.Kdim, BK) : 1);
  const dim3 grid((unsigned)std::min<long long>(gemm_sm_budget(), max_pieces));
  if constexpr (!SWIGLU) {
    static unsigned char narrow_set[64] = {};
    if (small && p.n_tiles == ceil_div(p.N, BN_HALF) && p.n_tiles != ceil_div(p.N, BN))
      return run(int8_gemm_small_kernel<false, T, true>, grid, S_THREADS, S_SMEM_BYTES, narrow_set, ma, mb0, mb1, p, sl, st);
  }
  return small ? run(int8_gemm_small_kernel<SWIGLU, T, false>, grid, S_THREADS, S_SMEM_BYTES, smem_set[1], ma, mb0, mb1, p, sl, st)
               : run(int8_gemm_kernel<SWIGLU, T, false>, grid, I8_THREADS, SMEM_BYTES, smem_set[0], ma, mb0, mb1, p, sl, st);
}

// fn(type tag)
template <class F>
int for_type(int dtype, F fn) {
  if (dtype == BWMOE_F32) return fn(TypeTag<float>{});
  if (dtype == BWMOE_F16) return fn(TypeTag<__half>{});
  return fn(TypeTag<__nv_bfloat16>{});
}

}  // namespace

size_t int8_clear_bytes() { return kSlabsAt; }
size_t int8_scratch_bytes(int M, int K, int N, int E) {
  // for one product and for SwiGLU, which has more tiles
  size_t slabs = 0;
  for (const int n_tiles : {ceil_div(N, BN), ceil_div(N, BN_HALF)})
    slabs = std::max(slabs, small_applies(M, K, n_tiles, E) ? S_MAX_PIECES * S_SLAB : may_slice(M, n_tiles) ? L_MAX_PIECES * L_SLAB : 0);
  return kSlabsAt + slabs;
}

int check_int8_gemm(const void* a, const float* row_scale, const int32_t* offsets, const void* w0, const void* w1,
                    const float* scale0, const float* scale1, int M, int K, int N, int E, int dtype, const void* out,
                    const int32_t* status) {
  const bool swiglu = w1 != nullptr;
  const char* who = swiglu ? "int_gateup_swiglu" : "int_grouped_gemm";
  BWMOE_REQUIRE(M > 0 && K > 0 && N > 0 && E > 0, BWMOE_ERR_BAD_SHAPE, "%s: M=%d K=%d N=%d E=%d", who, M, K, N, E);
  BWMOE_REQUIRE(K % 16 == 0 && N % 16 == 0, BWMOE_ERR_BAD_SHAPE, "%s: K=%d and N=%d must be multiples of 16", who, K, N);
  BWMOE_REQUIRE(E <= kMaxGroups, BWMOE_ERR_UNSUPPORTED, "%s: E=%d > %d", who, E, kMaxGroups);
  BWMOE_REQUIRE(M <= kMaxRows, BWMOE_ERR_UNSUPPORTED, "%s: M=%d rows", who, M);
  BWMOE_REQUIRE(K < (1 << 17), BWMOE_ERR_UNSUPPORTED, "%s: K=%d: sums of 2^17 products or more do not fit 32 bits", who, K);
  BWMOE_REQUIRE(dtype >= BWMOE_BF16 && dtype <= BWMOE_F32, BWMOE_ERR_UNSUPPORTED, "%s: unknown type %d", who, dtype);
  BWMOE_REQUIRE(a && row_scale && w0 && scale0 && out && status && (!swiglu || scale1), BWMOE_ERR_NULL, "%s: null pointer", who);
  BWMOE_REQUIRE(offsets != nullptr || E == 1, BWMOE_ERR_NULL, "%s: %d experts need offsets", who, E);
  BWMOE_REQUIRE(aligned16(a) && aligned16(w0) && aligned16(w1) && aligned16(scale0) && aligned16(scale1) && aligned16(out),
                BWMOE_ERR_BAD_ALIGN, "%s: codes, channel scales and the result must be 16-byte aligned", who);
  // (32-row tiles where M <= 32 E: at most 2 E of them over the rows)
  BWMOE_REQUIRE((ceil_div(M, BM) + 2ll * E) * ceil_div(N, BN_HALF) < kMostTiles, BWMOE_ERR_UNSUPPORTED, "%s: too many tiles", who);
  return BWMOE_OK;
}

int launch_int8_gemm(const void* a, const float* row_scale, const int32_t* offsets, const void* w0, const void* w1,
                     const float* scale0, const float* scale1, int M, int K, int N, int E, int dtype, void* out, void* scratch,
                     cudaStream_t st, bool clear, int32_t* status, bool early) {
  const bool swiglu = w1 != nullptr;
  if (status == nullptr) status = static_cast<int32_t*>(scratch);
  if (int rc = check_int8_gemm(a, row_scale, offsets, w0, w1, scale0, scale1, M, K, N, E, dtype, out, status)) return rc;
  if (clear) BWMOE_CUDA_OK(cudaMemsetAsync(scratch, 0, kSlabsAt, st));
  const int n_tiles = ceil_div(N, swiglu ? BN_HALF : BN);
  const bool small = small_applies(M, K, n_tiles, E);
  CUtensorMap ma, mb0, mb1;
  if (int rc = small ? make_map_rows(&ma, a, M, K, S_NT) : make_map_a(&ma, a, M, K)) return rc;
  if (int rc = make_map_b(&mb0, w0, E, K, N)) return rc;
  if (int rc = make_map_b(&mb1, swiglu ? w1 : w0, E, K, N)) return rc;
  I8Params p{offsets, row_scale, scale0, scale1, out, status, E, M, K, N, n_tiles, early && !clear,
             reinterpret_cast<uintptr_t>(out) % 32 == 0};
  if (small && narrow_applies(M, N, E, swiglu)) p.n_tiles = ceil_div(N, BN_HALF);
  uint8_t* s = static_cast<uint8_t*>(scratch);
  const bool slabs = small || may_slice(M, n_tiles);
  const I8Slices sl{reinterpret_cast<uint32_t*>(s + kArrivalsAt), slabs ? reinterpret_cast<int4*>(s + kSlabsAt) : nullptr};
  return for_type(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    return swiglu ? run_typed<true, T>(small, ma, mb0, mb1, p, sl, st) : run_typed<false, T>(small, ma, mb0, mb1, p, sl, st);
  });
}

}  // namespace bwmoe
