// Activations -> 8-bit integers, one scale per row:
//   scale = fl32(max|x| / 127)      code = x / scale rounded to the nearest whole number, ties to even
// The scale is rounded to fp32 once and the codes are exact for that scale.  A row of zeros has scale 0 and codes 0.  A row
// with an infinity or a NaN has no representation in 8 bits: its scale is NaN and its codes are 0, so that every product of
// the row is NaN.
//
// A product with the reciprocal may end on the wrong side of a border n + 1/2.  For 16-bit inputs that is settled per row:
// with p significant bits (8 or 11) the quotient 127 x / max|x| of two such numbers is either on a border or at least
// 2^-(p+9) of its value away from every border, and scale = max|x| / 127 * (1 + d), |d| <= 2^-24, moves the quotients on a
// border all to the same side, the one that the sign of d gives.  So the reciprocal is made 2^-21 smaller (d > 0) or larger
// (d < 0): more than its own roundings and d together (2^-22), and less than 2^-20.  With d = 0 borders are ties; they come
// out right where the reciprocal is exact, and the other rows (one in 100 in fp16) are divided one by one.  (16-bit inputs
// meet borders once in 500 values: with each checked and decided by itself 368 us for 32768 rows of 14336, 196 us for 16384
// x 4096 into two rows each.)  For fp32 inputs a piece with a quotient within 1e-5 of a border (one in 3000) is decided by
// the sign of x - (n + 1/2) * scale, which one fused multiply-add gives exactly.
//
// Bound by memory: a row is read once - each thread keeps its pieces of 16 elements in registers between the maximum and
// the codes - and written to all of the rows it is needed in (the K rows of its token, or one).  The conversion adds
// 1.5 * 2^23 instead of converting (the low byte of the sum is the code): at 3 bytes per element the conversion unit
// (16 results per cycle and SM) would be as busy as the memory.
#include "pieces.cuh"

namespace bwmoe {
namespace {

constexpr int kThreads = 256;
constexpr float kTinyScale = 7.888609052210118e-31f;     // 2^-100: below it products with the scale may lose bits

// x / scale, rounded exactly (ties to even); scale > 0
__device__ __noinline__ int exact_code(float x, float scale) {
  const float a = fabsf(x), f = floorf(fminf(__fdiv_rn(a, scale), 127.f));
  // the sign of a - (f + 1/2) * scale; doubled where the scale's last bits are the smallest there are
  const float r = scale >= kTinyScale ? fmaf(-(f + 0.5f), scale, a) : fmaf(-(2.f * f + 1.f), scale, 2.f * a);
  int q = (int)f;
  if (r > 0.f || (r == 0.f && (q & 1))) ++q;
  q = min(q, 127);
  return x < 0.f ? -q : q;
}

template <class T> struct Piece16;             // 16 elements
template <> struct Piece16<float> {
  float4 r[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = reinterpret_cast<const float4*>(p)[i];
  }
  __device__ __forceinline__ void values(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 * i] = r[i].x, f[4 * i + 1] = r[i].y, f[4 * i + 2] = r[i].z, f[4 * i + 3] = r[i].w;
  }
};
template <class T2, class T> __device__ __forceinline__ float2 pair_to_f32(uint32_t w);
template <> __device__ __forceinline__ float2 pair_to_f32<__half2, __half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 pair_to_f32<__nv_bfloat162, __nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T2, class T> struct Piece16Half {
  uint4 r[2];
  __device__ __forceinline__ void load(const T* p) {
    r[0] = reinterpret_cast<const uint4*>(p)[0], r[1] = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ void values(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = pair_to_f32<T2, T>(w[j]);
        f[8 * i + 2 * j] = v.x, f[8 * i + 2 * j + 1] = v.y;
      }
    }
  }
};
template <> struct Piece16<__half> : Piece16Half<__half2, __half> {};
template <> struct Piece16<__nv_bfloat16> : Piece16Half<__nv_bfloat162, __nv_bfloat16> {};

// Largest |x| of the piece as a bit pattern of the element's type: infinities and NaN are larger than every number.
__device__ __forceinline__ uint32_t piece_amax_bits(const Piece16<float>& p) {
  float f[16];
  p.values(f);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}
template <class T2, class T>
__device__ __forceinline__ uint32_t piece_amax_bits(const Piece16Half<T2, T>& p) {      // two at a time
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m = __vmaxu2(m, p.r[i].x & 0x7fff7fffu), m = __vmaxu2(m, p.r[i].y & 0x7fff7fffu);
    m = __vmaxu2(m, p.r[i].z & 0x7fff7fffu), m = __vmaxu2(m, p.r[i].w & 0x7fff7fffu);
  }
  return max(m & 0xffffu, m >> 16);
}
// the pattern's value; infinity and NaN stay what they are
__device__ __forceinline__ float bits_value(uint32_t m, float) { return __uint_as_float(m); }
__device__ __forceinline__ float bits_value(uint32_t m, __half) { return __half2float(__ushort_as_half((unsigned short)m)); }
__device__ __forceinline__ float bits_value(uint32_t m, __nv_bfloat16) { return __uint_as_float(m << 16); }

__device__ __forceinline__ uint4 pack_codes(const uint32_t (&b)[16]) {      // the low bytes
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// How a row's codes are formed.
struct RowScale {
  float scale, inv;
  bool none;          // zeros, or a row without a representation: all codes 0
  bool one_by_one;    // every quotient by itself
};
template <class T>
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const float amax = bits_value(amax_bits, T{});
  RowScale r;
  const bool finite = amax <= 3.402823466e38f;
  r.scale = finite ? __fdiv_rn(amax, 127.f) : __uint_as_float(0x7fc00000u);
  r.none = !(r.scale > 0.f);
  r.inv = __fdiv_rn(1.f, r.scale);
  r.one_by_one = r.scale < kTinyScale;
  if (sizeof(T) == 2) {
    const float d = fmaf(r.scale, 127.f, -amax);      // (its sign is exact)
    constexpr float kBias = 4.76837158203125e-7f;     // 2^-21
    if (d > 0.f) r.inv *= 1.f - kBias;
    if (d < 0.f) r.inv *= 1.f + kBias;
    if (d == 0.f && (__float_as_uint(r.scale) & 0x7fffffu) != 0u) r.one_by_one = true;
  }
  return r;
}

template <class T>
__device__ __forceinline__ uint4 piece_codes(const Piece16<T>& p, const RowScale& r) {
  if (r.none) return make_uint4(0u, 0u, 0u, 0u);
  constexpr float kMagic = 12582912.f;          // 1.5 * 2^23: the sum's last bit is worth 1
  float f[16];
  p.values(f);
  uint32_t b[16];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float m = fmaf(f[i], r.inv, kMagic);
    if (sizeof(T) == 4) far = fmaxf(far, fabsf(fmaf(f[i], r.inv, kMagic - m)));
    b[i] = __float_as_uint(m);
  }
  // fp32: f * inv is off by at most 127 * 2^-24 = 7.6e-6 (the reciprocal's rounding), its distance from the code by 2^-25 more
  if (r.one_by_one || (sizeof(T) == 4 && far > 0.49999f)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = (uint32_t)exact_code(f[i], r.scale);
  }
  return pack_codes(b);
}

// wpr warps (1, 2, 4 or 8) share a row.  pos == nullptr: row t is written to row t.
// next: the kernel behind is let in at once (a product that requests its weights meanwhile).
// kKept: pieces of a row that a thread keeps in registers - 4, or 2 for rows of up to 128 pieces, which then get more warps
// (1003 tokens of 2048 into 8 rows each: 7.5 -> 5.6 us, 8024 rows of 768: 9.4 -> 8.1; rows of 14336 with 2: 31 -> 38).
template <class T, int kKept>
__global__ void __launch_bounds__(kThreads)
quant_int8_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ pos, const int32_t* __restrict__ offsets, int E,
                       int n_tok, int K, int D, int wpr, int8_t* __restrict__ codes, float* __restrict__ scales,
                       uint32_t* __restrict__ zero, int zero_words, bool next) {
  chain_wait();
  if (next) chain_next();
  __shared__ uint32_t s_max[kThreads / 32];
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < zero_words; i += kThreads) zero[i] = 0u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * (kThreads / 32 / wpr) + warp / wpr, sub = warp % wpr;
  const bool live = t < n_tok;
  const int pieces = D / 16, step = 32 * wpr, c0 = sub * 32 + lane;
  const T* src = x + (size_t)t * D;
  Piece16<T> kept[kKept];
  uint32_t m = 0;
  if (live) {
#pragma unroll
    for (int i = 0; i < kKept; ++i)
      if (c0 + i * step < pieces) kept[i].load(src + (size_t)(c0 + i * step) * 16);
#pragma unroll
    for (int i = 0; i < kKept; ++i)
      if (c0 + i * step < pieces) m = max(m, piece_amax_bits(kept[i]));
    for (int c = c0 + kKept * step; c < pieces; c += step) {      // rows longer than the registers hold
      Piece16<T> q;
      q.load(src + (size_t)c * 16);
      m = max(m, piece_amax_bits(q));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (wpr > 1) {                                // (the same in the whole block)
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
    for (int i = 0; i < wpr; ++i) m = max(m, s_max[warp - sub + i]);
  }
  if (!live) return;
  const RowScale r = row_scale<T>(m);
  const int M = n_tok * K, n_rows = pos != nullptr && E > 0 ? offsets[E] : 0;
  auto store = [&](int c, uint4 o) {
    if (pos == nullptr) {
      reinterpret_cast<uint4*>(codes + (size_t)t * D)[c] = o;
      if (c == 0) scales[t] = r.scale;
      return;
    }
#pragma unroll 4
    for (int k = 0; k < K; ++k) {
      const int s = t * K + k, p = pos[s];
      if ((unsigned)p < (unsigned)M) {          // a plan is data from outside the kernel
        reinterpret_cast<uint4*>(codes + (size_t)p * D)[c] = o;
        if (c == 0) scales[p] = r.scale;
      }
      if (no_slot(offsets, E, n_rows, s)) {
        reinterpret_cast<uint4*>(codes + (size_t)s * D)[c] = make_uint4(0u, 0u, 0u, 0u);
        if (c == 0) scales[s] = 0.f;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (c0 + i * step < pieces) store(c0 + i * step, piece_codes(kept[i], r));
  for (int c = c0 + kKept * step; c < pieces; c += step) {
    Piece16<T> q;
    q.load(src + (size_t)c * 16);
    store(c, piece_codes(q, r));
  }
}

}  // namespace

int launch_quant_int8_rows(const void* x, const int32_t* pos, const int32_t* offsets, int T, int D, int E, int K, int dtype,
                           void* codes, float* scales, cudaStream_t st, void* zero, size_t zero_bytes) {
  BWMOE_REQUIRE(T > 0 && D > 0 && K > 0 && D % 16 == 0, BWMOE_ERR_BAD_SHAPE, "int_quant: T=%d D=%d K=%d (D a multiple of 16)", T, D, K);
  BWMOE_REQUIRE((long long)T * K <= kMaxRows, BWMOE_ERR_UNSUPPORTED, "int_quant: T*K too large");
  BWMOE_REQUIRE(dtype >= BWMOE_BF16 && dtype <= BWMOE_F32, BWMOE_ERR_UNSUPPORTED, "int_quant: unknown type %d", dtype);
  BWMOE_REQUIRE(x && codes && scales, BWMOE_ERR_NULL, "int_quant: null pointer");
  BWMOE_REQUIRE(pos == nullptr ? K == 1 : (offsets != nullptr && E >= 0), BWMOE_ERR_BAD_SHAPE,
                "int_quant: K=%d needs the slots' places and the segments' offsets", K);
  BWMOE_REQUIRE(aligned16(x) && aligned16(codes) && reinterpret_cast<uintptr_t>(scales) % 4 == 0, BWMOE_ERR_BAD_ALIGN,
                "int_quant: x and codes must be 16-byte aligned");
  const int pieces = D / 16;
  const int kept = pieces <= 128 ? 2 : 4;
  int wpr = 1;      // warps per row: until the row fits the registers, and more while the batch leaves the chip empty
  while (wpr < 8 && 32 * wpr < pieces && (32 * wpr * kept < pieces || (long long)T * wpr < 32ll * sm_count())) wpr *= 2;
  const dim3 grid((unsigned)ceil_div(T, kThreads / 32 / wpr));
  auto run = [&](auto tag) {
    using X = typename decltype(tag)::type;
    return launch_chained(kept == 2 ? quant_int8_rows_kernel<X, 2> : quant_int8_rows_kernel<X, 4>, grid, dim3(kThreads), 0, st, static_cast<const X*>(x), pos, offsets, E, T, K,
                          D, wpr, static_cast<int8_t*>(codes), scales, static_cast<uint32_t*>(zero), (int)(zero_bytes / 4), (int)grid.x <= 2 * sm_count());
  };
  BWMOE_CUDA_OK(dtype == BWMOE_F32 ? run(TypeTag<float>{}) : dtype == BWMOE_F16 ? run(TypeTag<__half>{}) : run(TypeTag<__nv_bfloat16>{}));
  return BWMOE_OK;
}

}  // namespace bwmoe
