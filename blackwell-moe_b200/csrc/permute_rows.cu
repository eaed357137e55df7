// Tokens into expert order and back, with gradients.  M = T * K rows; pos[t,k] is the row of slot (t,k), -1 where the
// slot's expert id was out of range, and the rows offsets[E] .. M-1 then belong to no slot.  (A plan made elsewhere may leave out
// any row.)
//
//   row slots          slots[pos[t,k]] = (t,k), else -1                  for plans made elsewhere (no_slot() reads it)
//   permute            rows[pos[t,k]] = x[t]                             its gradient:  dx[t] = sum_k drows[pos[t,k]]
//   unpermute          out[t] = sum_k w[t,k] * rows[pos[t,k]]            (w absent: 1)
//   unpermute backward drows[pos[t,k]] = w[t,k] * dout[t]                dw[t,k] = < rows[pos[t,k]], dout[t] >
//
// Sums are held in fp32 and added in the order of k (of the row's vectors, for dw), so results do not depend on the
// launch's timing; a 16-bit result is rounded once.  All of it is bound by memory: every kernel walks the batch by
// token, so that the token's side (x, out, dout) moves once and only the rows move K times.  Rows that no slot owns are
// written as zeros.
#include <type_traits>

#include "pieces.cuh"

namespace bwmoe {
namespace {

constexpr int kThreads = 256;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

template <class T, int BYTES>
union Values {
  typename Piece<BYTES>::type raw;
  T v[BYTES / sizeof(T)];
  __device__ Values() {}
};

template <int ROWS> constexpr int kPiecesPerThread = ROWS >= 4 ? 8 / ROWS : 2;

// Row of slot s; -1 where there is none.  A plan is data from outside the kernel: an entry past the rows is no row.
__device__ __forceinline__ int row_of(const int32_t* __restrict__ pos, long long s, int M) {
  const int p = pos[s];
  return (unsigned)p < (unsigned)M ? p : -1;
}

__global__ void __launch_bounds__(kThreads)
row_slots_kernel(const int32_t* __restrict__ pos, int M, int32_t* __restrict__ slots) {
  chain_wait();
  const long long s = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (s >= M) return;
  const int p = row_of(pos, s, M);
  if (p >= 0) slots[p] = (int)s;
}

// `lanes` threads (a power of two) stand side by side on one token's row, each with U pieces.
template <int BYTES>
__global__ void __launch_bounds__(kThreads)
permute_rows_kernel(const typename Piece<BYTES>::type* __restrict__ x, const int32_t* __restrict__ pos,
                    const int32_t* __restrict__ offsets, int E, int T, int K, int pieces, int lanes,
                    typename Piece<BYTES>::type* __restrict__ rows) {
  using P = typename Piece<BYTES>::type;
  constexpr int U = 2;
  chain_wait();
  const int t = blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes, c0 = blockIdx.y * lanes * U + threadIdx.x % lanes;
  if (t >= T) return;
  P v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + u * lanes < pieces) v[u] = x[(size_t)t * pieces + c0 + u * lanes];
  const int M = T * K, n_rows = E > 0 ? offsets[E] : 0;
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const int s = t * K + k, p = row_of(pos, s, M);
    const bool none = no_slot(offsets, E, n_rows, s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * lanes;
      if (c >= pieces) continue;
      if (p >= 0) rows[(size_t)p * pieces + c] = v[u];
      if (none) rows[(size_t)s * pieces + c] = zero_piece<P>();
    }
  }
}

// R rows at a time and U pieces of each per thread: their places first, then their pieces, all requested before the first
// is used.  Four or eight pieces in flight per thread, whatever K is: the registers that absent rows hold keep threads off the
// chip (R = 8 for two rows per token: 137 us for 16384 tokens x 2 rows of 4096, 65 with R = 2).  More than four rows come four
// at a time, two pieces of each (8192 tokens x 8 rows of 2048: 45 us, 49 eight at a time; 1003 x 8 rows of 2050 in fp32: 13 and
// 17), or, where the batch is too small to hide a second round trip, eight at a time (64 x 6 rows: 1.8 us, 2.4 with four).
// Blocks of 128 threads, and rows that are read once marked as such where many are in flight (16384 x 2 rows: 75 us with the
// mark, 70 without; 8192 x 8 rows of 2048: 50 and 58, 20000 x 4 rows of 1024: 30 and 35; 256 threads: 4 to 7 % more).
constexpr int kSumThreads = 128;
template <int R, class P> __device__ __forceinline__ P load_row(const P* p) {
  if constexpr (R >= 4) return __ldcs(p);
  else                  return *p;
}
template <class T, int BYTES, bool WEIGHTED, int R>
__global__ void __launch_bounds__(kSumThreads)
unpermute_rows_kernel(const typename Piece<BYTES>::type* __restrict__ rows, const int32_t* __restrict__ pos,
                      const float* __restrict__ weights, int n_tok, int K, int pieces, int lanes,
                      typename Piece<BYTES>::type* __restrict__ out) {
  constexpr int W = BYTES / (int)sizeof(T), U = kPiecesPerThread<R>;
  chain_wait();
  const int t = blockIdx.x * (kSumThreads / lanes) + threadIdx.x / lanes, c0 = blockIdx.y * lanes * U + threadIdx.x % lanes;
  if (t >= n_tok || c0 >= pieces) return;
  const int M = n_tok * K;
  float acc[U][W];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[u][i] = 0.f;
  for (int k0 = 0; k0 < K; k0 += R) {
    int p[R];
    float w[R];
    Values<T, BYTES> q[R][U];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      p[j] = k0 + j < K ? row_of(pos, (size_t)t * K + k0 + j, M) : -1;
      w[j] = WEIGHTED && k0 + j < K ? weights[(size_t)t * K + k0 + j] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p[j] >= 0 && c0 + u * lanes < pieces) q[j][u].raw = load_row<R>(rows + (size_t)p[j] * pieces + c0 + u * lanes);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (p[j] < 0) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < W; ++i)
          acc[u][i] = WEIGHTED ? fmaf(w[j], to_f32(q[j][u].v[i]), acc[u][i]) : acc[u][i] + to_f32(q[j][u].v[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (c0 + u * lanes >= pieces) continue;
    Values<T, BYTES> o;
#pragma unroll
    for (int i = 0; i < W; ++i) o.v[i] = from_f32<T>(acc[u][i]);
    out[(size_t)t * pieces + c0 + u * lanes] = o.raw;
  }
}

// wpt warps (1, 2, 4 or 8) share a token; lane l of them takes every (32 * wpt)-th piece of the row.
template <class T, int BYTES, bool DROWS, bool DW, int R>
__global__ void __launch_bounds__(kThreads)
unpermute_rows_backward_kernel(const typename Piece<BYTES>::type* __restrict__ dout,
                               const typename Piece<BYTES>::type* __restrict__ rows, const int32_t* __restrict__ pos,
                               const int32_t* __restrict__ offsets, int E, const float* __restrict__ weights, int n_tok,
                               int K, int pieces, int wpt, typename Piece<BYTES>::type* __restrict__ drows,
                               float* __restrict__ dweights) {
  using P = typename Piece<BYTES>::type;
  constexpr int W = BYTES / (int)sizeof(T);
  chain_wait();
  __shared__ float s_part[kThreads / 32][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kThreads / 32 / wpt) + warp / wpt, sub = warp % wpt;
  const bool live = t < n_tok;
  const int M = n_tok * K, n_rows = DROWS && E > 0 ? offsets[E] : 0;
  for (int k0 = 0; k0 < K; k0 += R) {
    int p[R];
    float w[R], dot[R];
    unsigned none = 0;                              // rows (of the slots' numbers) that no slot owns
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool slot = live && k0 + j < K;
      p[j] = slot ? row_of(pos, (size_t)t * K + k0 + j, M) : -1;
      w[j] = DROWS && slot ? weights[(size_t)t * K + k0 + j] : 0.f;
      dot[j] = 0.f;
      if (DROWS && slot && no_slot(offsets, E, n_rows, t * K + k0 + j)) none |= 1u << j;
    }
    for (int c = sub * 32 + lane; live && c < pieces; c += 32 * wpt) {
      Values<T, BYTES> d, q[R];
      d.raw = dout[(size_t)t * pieces + c];
      if constexpr (DW) {
#pragma unroll
        for (int j = 0; j < R; ++j)
          if (p[j] >= 0) q[j].raw = rows[(size_t)p[j] * pieces + c];
      }
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (DROWS && (none >> j & 1u)) drows[(size_t)(t * K + k0 + j) * pieces + c] = zero_piece<P>();
        if (p[j] < 0) continue;
        if constexpr (DW) {
#pragma unroll
          for (int i = 0; i < W; ++i) dot[j] = fmaf(to_f32(q[j].v[i]), to_f32(d.v[i]), dot[j]);
        }
        if constexpr (DROWS) {
          Values<T, BYTES> o;
#pragma unroll
          for (int i = 0; i < W; ++i) o.v[i] = from_f32<T>(w[j] * to_f32(d.v[i]));
          drows[(size_t)p[j] * pieces + c] = o.raw;
        }
      }
    }
    if constexpr (DW) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        for (int off = 16; off; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
      if (wpt == 1) {
#pragma unroll
        for (int j = 0; j < R; ++j)
          if (lane == j && live && k0 + j < K) dweights[(size_t)t * K + k0 + j] = dot[j];
      } else {                                     // (the same in the whole block)
#pragma unroll
        for (int j = 0; j < R; ++j)
          if (lane == j) s_part[warp][j] = dot[j];
        __syncthreads();
        if (sub == 0 && lane < R && live && k0 + lane < K) {
          float sum = 0.f;
          for (int i = 0; i < wpt; ++i) sum += s_part[warp + i][lane];
          dweights[(size_t)t * K + k0 + lane] = sum;
        }
        __syncthreads();
      }
    }
  }
}

int lanes_for(int pieces, int threads) {
  int lanes = 1;
  while (lanes < pieces && lanes < threads) lanes *= 2;
  return lanes;
}

int check_rows(const char* who, int T, int D, int K, int dtype) {
  BWMOE_REQUIRE(T > 0 && D > 0 && K > 0, BWMOE_ERR_BAD_SHAPE, "%s: T=%d D=%d K=%d", who, T, D, K);
  BWMOE_REQUIRE(K <= 32, BWMOE_ERR_UNSUPPORTED, "%s: K=%d > 32 slots per token", who, K);
  BWMOE_REQUIRE((long long)T * K <= kMaxRows, BWMOE_ERR_UNSUPPORTED, "%s: T*K too large", who);
  BWMOE_REQUIRE(D <= (1 << 24), BWMOE_ERR_UNSUPPORTED, "%s: D=%d too large", who, D);
  BWMOE_REQUIRE(dtype >= BWMOE_BF16 && dtype <= BWMOE_F32, BWMOE_ERR_UNSUPPORTED, "%s: unknown type %d", who, dtype);
  return BWMOE_OK;
}
int check_align(const char* who, int dtype, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    BWMOE_REQUIRE(reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype) == 0, BWMOE_ERR_BAD_ALIGN,
                  "%s: a pointer is not aligned to its type", who);
  return BWMOE_OK;
}

template <int BYTES>
int run_permute(const void* x, const int32_t* pos, const int32_t* offsets, int E, int T, int K, size_t row_bytes,
                void* rows, cudaStream_t st) {
  using P = typename Piece<BYTES>::type;
  const int pieces = (int)(row_bytes / BYTES), lanes = lanes_for(ceil_div(pieces, 2), kThreads);
  const dim3 grid((unsigned)ceil_div(T, kThreads / lanes), (unsigned)ceil_div(pieces, 2 * lanes));
  BWMOE_REQUIRE(grid.y <= 65535, BWMOE_ERR_UNSUPPORTED, "permute_rows: rows of %zu bytes", row_bytes);
  BWMOE_CUDA_OK(launch_chained(permute_rows_kernel<BYTES>, grid, dim3(kThreads), 0, st, static_cast<const P*>(x), pos, offsets,
                               E, T, K, pieces, lanes, static_cast<P*>(rows)));
  return BWMOE_OK;
}

template <class T, int BYTES>
int run_unpermute(const void* rows, const int32_t* pos, const float* weights, int n_tok, int K, size_t row_bytes, void* out,
                  cudaStream_t st) {
  using P = typename Piece<BYTES>::type;
  const int pieces = (int)(row_bytes / BYTES);
  auto run = [&](auto rows_at_once) {
    constexpr int R = decltype(rows_at_once)::value, U = kPiecesPerThread<R>;
    const int lanes = lanes_for(ceil_div(pieces, U), kSumThreads);
    const dim3 grid((unsigned)ceil_div(n_tok, kSumThreads / lanes), (unsigned)ceil_div(pieces, U * lanes));
    BWMOE_REQUIRE(grid.y <= 65535, BWMOE_ERR_UNSUPPORTED, "unpermute_rows: rows of %zu bytes", row_bytes);
    auto kernel = weights ? unpermute_rows_kernel<T, BYTES, true, R> : unpermute_rows_kernel<T, BYTES, false, R>;
    BWMOE_CUDA_OK(launch_chained(kernel, grid, dim3(kSumThreads), 0, st, static_cast<const P*>(rows), pos, weights, n_tok, K,
                                 pieces, lanes, static_cast<P*>(out)));
    return (int)BWMOE_OK;
  };
  const bool small = n_tok <= 4 * sm_count();
  return K <= 2            ? run(std::integral_constant<int, 2>{})
         : K <= 4 || !small ? run(std::integral_constant<int, 4>{})
                            : run(std::integral_constant<int, 8>{});
}

template <class T, int BYTES>
int run_unpermute_backward(const void* dout, const void* rows, const int32_t* pos, const int32_t* offsets, int E,
                           const float* weights, int n_tok, int K, size_t row_bytes, void* drows, float* dweights,
                           cudaStream_t st) {
  using P = typename Piece<BYTES>::type;
  const int pieces = (int)(row_bytes / BYTES);
  // warps per token: more while the row feeds them and the batch leaves the chip's warp slots empty
  int wpt = 1;
  while (wpt < 8 && 32 * wpt < pieces && (long long)n_tok * wpt < 16ll * sm_count()) wpt *= 2;
  const unsigned blocks = (unsigned)ceil_div(n_tok, kThreads / 32 / wpt);
  auto run = [&](auto rows_at_once) {
    constexpr int R = decltype(rows_at_once)::value;
    auto kernel = drows && dweights ? unpermute_rows_backward_kernel<T, BYTES, true, true, R>
                  : drows           ? unpermute_rows_backward_kernel<T, BYTES, true, false, R>
                                    : unpermute_rows_backward_kernel<T, BYTES, false, true, R>;
    BWMOE_CUDA_OK(launch_chained(kernel, dim3(blocks), dim3(kThreads), 0, st, static_cast<const P*>(dout),
                                 static_cast<const P*>(rows), pos, offsets, E, weights, n_tok, K, pieces, wpt,
                                 static_cast<P*>(drows), dweights));
    return (int)BWMOE_OK;
  };
  // eight rows at a time only where a piece is 16 bytes (8192 x 8 rows of 2048 in bf16: 98 us, 112 four at a time; with 8-byte
  // pieces, 1003 x 8 rows of 2050 in fp32: 34 and 28)
  return K <= 2                ? run(std::integral_constant<int, 2>{})
         : K <= 4 || BYTES < 16 ? run(std::integral_constant<int, 4>{})
                                : run(std::integral_constant<int, 8>{});
}

// fn(type tag, piece tag) for the element type and the widest piece
template <class F>
int for_type_and_piece(int dtype, int bytes, F fn) {
  auto by_piece = [&](auto tag) {
    using T = typename decltype(tag)::type;
    switch (bytes) {
      case 16: return fn(tag, std::integral_constant<int, 16>{});
      case 8: return fn(tag, std::integral_constant<int, 8>{});
      case 4: return fn(tag, std::integral_constant<int, 4>{});
      default: return fn(tag, std::integral_constant<int, sizeof(T)>{});     // an fp32 row is never split below 4 bytes
    }
  };
  if (dtype == BWMOE_F32) return by_piece(TypeTag<float>{});
  if (dtype == BWMOE_F16) return by_piece(TypeTag<__half>{});
  return by_piece(TypeTag<__nv_bfloat16>{});
}

}  // namespace

int launch_row_slots(const int32_t* pos, int T, int K, int32_t* row_slot, cudaStream_t st) {
  BWMOE_REQUIRE(T > 0 && K > 0, BWMOE_ERR_BAD_SHAPE, "plan_row_slots: T=%d K=%d", T, K);
  BWMOE_REQUIRE((long long)T * K <= kMaxRows, BWMOE_ERR_UNSUPPORTED, "plan_row_slots: T*K too large");
  BWMOE_REQUIRE(pos && row_slot, BWMOE_ERR_NULL, "plan_row_slots: null pointer");
  BWMOE_CUDA_OK(cudaMemsetAsync(row_slot, 0xff, sizeof(int32_t) * (size_t)T * K, st));
  BWMOE_CUDA_OK(launch_chained(row_slots_kernel, dim3((unsigned)ceil_div(T * K, kThreads)), dim3(kThreads), 0, st, pos, T * K, row_slot));
  return BWMOE_OK;
}

int launch_permute_rows(const void* x, const int32_t* pos, const int32_t* offsets, int T, int D, int E, int K, int dtype,
                        void* rows, cudaStream_t st) {
  if (int rc = check_rows("permute_rows", T, D, K, dtype)) return rc;
  BWMOE_REQUIRE(E >= 0, BWMOE_ERR_BAD_SHAPE, "permute_rows: E=%d", E);
  BWMOE_REQUIRE(x && pos && offsets && rows, BWMOE_ERR_NULL, "permute_rows: null pointer");
  if (int rc = check_align("permute_rows", dtype, {x, rows})) return rc;
  const size_t row_bytes = (size_t)D * dtype_bytes(dtype);
  switch (piece_bytes(row_bytes, {x, rows})) {
    case 16: return run_permute<16>(x, pos, offsets, E, T, K, row_bytes, rows, st);
    case 8: return run_permute<8>(x, pos, offsets, E, T, K, row_bytes, rows, st);
    case 4: return run_permute<4>(x, pos, offsets, E, T, K, row_bytes, rows, st);
    default: return run_permute<2>(x, pos, offsets, E, T, K, row_bytes, rows, st);
  }
}

int launch_unpermute_rows(const void* rows, const int32_t* pos, const float* weights, int T, int D, int K, int dtype, void* out,
                          cudaStream_t st) {
  if (int rc = check_rows("unpermute_rows", T, D, K, dtype)) return rc;
  BWMOE_REQUIRE(rows && pos && out, BWMOE_ERR_NULL, "unpermute_rows: null pointer");
  if (int rc = check_align("unpermute_rows", dtype, {rows, out})) return rc;
  const size_t row_bytes = (size_t)D * dtype_bytes(dtype);
  return for_type_and_piece(dtype, piece_bytes(row_bytes, {rows, out}), [&](auto type, auto bytes) {
    return run_unpermute<typename decltype(type)::type, decltype(bytes)::value>(rows, pos, weights, T, K, row_bytes, out, st);
  });
}

int launch_unpermute_rows_backward(const void* dout, const void* rows, const int32_t* pos, const int32_t* offsets,
                                   const float* weights, int T, int D, int E, int K, int dtype, void* drows, float* dweights,
                                   cudaStream_t st) {
  if (int rc = check_rows("unpermute_rows_backward", T, D, K, dtype)) return rc;
  BWMOE_REQUIRE(dout && pos && (drows || dweights), BWMOE_ERR_NULL, "unpermute_rows_backward: null pointer");
  BWMOE_REQUIRE(!drows || (offsets && weights && E >= 0), BWMOE_ERR_NULL,
                "unpermute_rows_backward: the rows' gradient needs offsets and weights");
  BWMOE_REQUIRE(!dweights || rows, BWMOE_ERR_NULL, "unpermute_rows_backward: the weights' gradient needs the rows");
  if (int rc = check_align("unpermute_rows_backward", dtype, {dout, rows, drows})) return rc;
  const size_t row_bytes = (size_t)D * dtype_bytes(dtype);
  return for_type_and_piece(dtype, piece_bytes(row_bytes, {dout, rows, drows}), [&](auto type, auto bytes) {
    return run_unpermute_backward<typename decltype(type)::type, decltype(bytes)::value>(dout, rows, pos, offsets, E, weights, T,
                                                                                         K, row_bytes, drows, dweights, st);
  });
}

}  // namespace bwmoe
